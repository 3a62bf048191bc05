// A GDN layer's convolution and gated delta rule over a batch of sequences whose states lie in a pool.
//
// Reference arithmetic: model/qwen35_moe_dflash/fused/model.py:206-263 and fused/ops.py:36-71 (conv and, per token,
// S <- e^g S; u = beta (v - S^T k); S <- S + k u^T; o = S^T q).  Tokens [starts[b], starts[b + 1]) of the block are sequence
// b's; its conv history and state are slot slots[b] of the pool.  All three are read on the device, and whatever they
// hold leads to no address outside the block or the pool.
#include "kernels.h"

namespace dflash {
namespace {

constexpr int kTaps = 4;

template <bool kBf16>
__device__ __forceinline__ float to_f32(uint16_t v) {
  if constexpr (kBf16) return __uint_as_float(static_cast<uint32_t>(v) << 16);
  return static_cast<float>(__builtin_bit_cast(_Float16, v));
}
template <bool kBf16>
__device__ __forceinline__ uint16_t from_f32(float v) {
  if constexpr (kBf16) return f32_to_bf16(v);
  return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}
template <bool kBf16>
__device__ __forceinline__ void unpack8(uint4 w, float (&f)[8]) {
  const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = to_f32<kBf16>(static_cast<uint16_t>(d[i]));
    f[2 * i + 1] = to_f32<kBf16>(static_cast<uint16_t>(d[i] >> 16));
  }
}

struct Span {
  int start, tokens, slot;  // slot -1: none
  int count;                // tokens that the state advances by, 0: it stays
  bool fresh;               // the state before the block is zeros
};
__device__ __forceinline__ Span span_of(const PoolParams& p, int b) {
  Span s;
  s.start = clampi(p.starts[b], 0, p.T);
  s.tokens = clampi(p.starts[b + 1], s.start, p.T) - s.start;
  s.slot = p.slots[b];
  if (s.slot < 0 || s.slot >= p.pool_slots) s.slot = -1;
  s.count = p.counts ? clampi(p.counts[b], 0, s.tokens) : s.tokens;
  if (s.slot < 0) s.count = 0;
  s.fresh = s.slot < 0 || (p.fresh && p.fresh[b]);
  return s;
}

// Sequences whose block ends at or before token t (a wave's lanes together; the result is uniform).
__device__ __forceinline__ int ended_before(const int32_t* starts, int B, int t) {
  int n = 0;
  for (int i = 0; i < B; i += 64) {
    const int b = i + lane_id();
    n += __popcll(__ballot(b < B && starts[b + 1] <= t));
  }
  return __builtin_amdgcn_readfirstlane(n);
}

// ------------------------------------------------------------------ convolution
// Element j < 3 of a channel's history stands before the block's row 0 at row j - 3.
struct History {
  float c[8][kTaps - 1];
};
template <bool kBf16>
__device__ __forceinline__ History load_history(const PoolParams& p, const Span& s, int channel) {
  History h;
  if (s.fresh) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < kTaps - 1; ++j) h.c[i][j] = 0.f;
    return h;
  }
  const uint4* r = reinterpret_cast<const uint4*>(p.history + s.slot * p.history_stride + static_cast<int64_t>(channel) * (kTaps - 1));
  float f[3][8];
#pragma unroll
  for (int i = 0; i < 3; ++i) unpack8<kBf16>(r[i], f[i]);
#pragma unroll
  for (int i = 0; i < 24; ++i) h.c[i / 3][i % 3] = f[i / 8][i % 8];
  return h;
}

// The history after `count` >= 1 rows of the block.
template <bool kBf16>
__device__ __forceinline__ void store_history(const PoolParams& p, const Span& s, int channel, const History& h, const uint16_t* x,
                                              int64_t x_stride) {
  float rows[kTaps - 1][8];
#pragma unroll
  for (int j = 0; j < kTaps - 1; ++j) {
    const int r = s.count - (kTaps - 1) + j;
    if (r >= 0) {
      unpack8<kBf16>(*reinterpret_cast<const uint4*>(x + (s.start + r) * x_stride + channel), rows[j]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) rows[j][i] = s.count == 1 ? h.c[i][min(j + 1, 2)] : h.c[i][min(j + 2, 2)];
    }
  }
  uint16_t out[24];
#pragma unroll
  for (int i = 0; i < 24; ++i) out[i] = from_f32<kBf16>(rows[i % 3][i / 3]);
  uint4* to = reinterpret_cast<uint4*>(p.history + s.slot * p.history_stride + static_cast<int64_t>(channel) * (kTaps - 1));
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    uint4 w;
    w.x = out[8 * i] | static_cast<uint32_t>(out[8 * i + 1]) << 16;
    w.y = out[8 * i + 2] | static_cast<uint32_t>(out[8 * i + 3]) << 16;
    w.z = out[8 * i + 4] | static_cast<uint32_t>(out[8 * i + 5]) << 16;
    w.w = out[8 * i + 6] | static_cast<uint32_t>(out[8 * i + 7]) << 16;
    to[i] = w;
  }
}

// A workgroup per kRows tokens and 2048 channels, a thread eight neighbouring channels.  A block's first three rows read the
// history that the same thread replaces, so they go with the first of them, whichever tile they fall into.
template <bool kBf16, int kRows>
__global__ __launch_bounds__(256) void gdn_conv_kernel(ConvParams p) {
  const int t0 = blockIdx.x * kRows, channel = (blockIdx.y * 256 + threadIdx.x) * 8;
  int b = ended_before(p.pool.starts, p.pool.B, t0);
  if (channel >= p.channels) return;
  float w[8][kTaps];
  {
    const uint4* r = reinterpret_cast<const uint4*>(p.weight + static_cast<int64_t>(channel) * kTaps);
    float f[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack8<kBf16>(r[i], f[i]);
#pragma unroll
    for (int i = 0; i < 32; ++i) w[i / 4][i % 4] = f[i / 8][i % 8];
  }
  for (; b < p.pool.B; ++b) {
    const Span s = span_of(p.pool, b);
    if (s.start >= t0 + kRows) break;
    if (s.tokens == 0) continue;
    const bool first = s.start >= t0;
    const int lo = first ? s.start : max(t0, s.start + kTaps - 1);
    const int end = s.start + s.tokens;
    const int hi = min(end, first ? max(t0 + kRows, s.start + kTaps - 1) : t0 + kRows);
    if (lo >= hi) continue;
    History h;
    float past[kTaps - 1][8];
    if (first) {
      h = load_history<kBf16>(p.pool, s, channel);
#pragma unroll
      for (int j = 0; j < kTaps - 1; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) past[j][i] = h.c[i][j];
    } else {
#pragma unroll
      for (int j = 0; j < kTaps - 1; ++j)
        unpack8<kBf16>(*reinterpret_cast<const uint4*>(p.x + (lo - (kTaps - 1) + j) * p.x_stride + channel), past[j]);
    }
    for (int t = lo; t < hi; ++t) {
      float x[8];
      unpack8<kBf16>(*reinterpret_cast<const uint4*>(p.x + t * p.x_stride + channel), x);
      uint16_t o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = ((past[0][i] * w[i][0] + past[1][i] * w[i][1]) + past[2][i] * w[i][2]) + x[i] * w[i][3];
        o[i] = from_f32<kBf16>(y / (1.0f + __expf(-y)));
        past[0][i] = past[1][i];
        past[1][i] = past[2][i];
        past[2][i] = x[i];
      }
      uint4 v;
      v.x = o[0] | static_cast<uint32_t>(o[1]) << 16;
      v.y = o[2] | static_cast<uint32_t>(o[3]) << 16;
      v.z = o[4] | static_cast<uint32_t>(o[5]) << 16;
      v.w = o[6] | static_cast<uint32_t>(o[7]) << 16;
      *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(t) * p.channels + channel) = v;
    }
    if (first && s.count > 0) store_history<kBf16>(p.pool, s, channel, h, p.x, p.x_stride);
  }
}

// ------------------------------------------------------------------ the rule, token after token
__device__ __forceinline__ float gate_value(const void* data, int dtype, int64_t i) {
  if (dtype == 1) return static_cast<const float*>(data)[i];
  const uint16_t v = static_cast<const uint16_t*>(data)[i];
  return dtype == 0 ? to_f32<true>(v) : to_f32<false>(v);
}
// log decay and write strength of one token and head
__device__ __forceinline__ float2 gates_of(const RuleParams& p, int64_t token, int head) {
  float g = gate_value(p.decay, p.gates_dtype, token * p.decay_stride + head);
  float b = gate_value(p.beta, p.gates_dtype, token * p.beta_stride + head);
  if (p.a_log) {
    const float a = g + p.dt_bias[head];
    g = -expf(p.a_log[head]) * (a > 20.0f ? a : log1pf(expf(a)));
    b = 1.0f / (1.0f + expf(-b));
  }
  return make_float2(g, b);
}

// One workgroup per (sequence, value head), its state in registers: wave w holds columns [w D/4, (w + 1) D/4), a lane four
// columns of kPer rows, so a column's two products with the state (S^T k, S^T q) are sums over kGroups lanes of one wave
// and no token needs a barrier.  A slight decay is applied as S + (e^g - 1) S, one fma: e^g itself is off by half a step near 1,
// which a head that remembers thousands of tokens would sum up wherever its decay is a constant.  o = S_new^T q = e^g S_old^T q + u (k.q) takes both products from the old state.
constexpr float kStrong = 2.0f;  // no value of e^g - 1 for g <= 0: the decay is applied as e^g S

template <bool kBf16, int kDim, bool kOut>
__device__ __forceinline__ void rule_steps(const RuleParams& p, int b, int head, float* lds) {
  constexpr int kCols = kDim / 16, kGroups = 64 / kCols, kQuads = kDim / (4 * kGroups), kBlock = 16;
  float(*ks)[kDim] = reinterpret_cast<float(*)[kDim]>(lds);
  float(*qs)[kDim] = ks + kBlock;
  float(*vs)[kDim] = qs + (kOut ? kBlock : 0);
  float(*scalars)[4] = reinterpret_cast<float(*)[4]>(vs + kBlock);  // e^g, beta, k.q, e^g - 1 or kStrong
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int col = wave * (kDim / 4) + 4 * (lane % kCols), group = lane / kCols;
  const Span s = span_of(p.pool, b);
  const int limit = kOut ? s.tokens : s.count;
  if (limit == 0) return;
  float* place = p.pool.recurrent + s.slot * p.pool.recurrent_stride + static_cast<int64_t>(head) * kDim * kDim + col;
  f32x4 state[kQuads][4];  // rows 4 kGroups j + 4 group + e
#pragma unroll
  for (int j = 0; j < kQuads; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      state[j][e] = s.fresh ? f32x4{0.f, 0.f, 0.f, 0.f}
                            : *reinterpret_cast<const f32x4*>(place + (4 * kGroups * j + 4 * group + e) * kDim);
  const int khead = head / p.rep;
  for (int t0 = 0; t0 < limit; t0 += kBlock) {
    const int n = min(kBlock, limit - t0);
    if (t0) __syncthreads();
    for (int i = wave; i < n; i += 4) {
      const int64_t t = s.start + t0 + i;
      constexpr int kEach = kDim / 64;
      float k[kEach], q[kEach], kk = 0.f, qq = 0.f, kq = 0.f;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int d = lane * kEach + e;
        k[e] = to_f32<kBf16>(p.key[t * p.key_token + khead * p.key_head + d]);
        if constexpr (kOut) q[e] = to_f32<kBf16>(p.query[t * p.query_token + khead * p.query_head + d]);
        vs[i][d] = to_f32<kBf16>(p.value[t * p.value_token + head * p.value_head + d]);
        kk += k[e] * k[e];
        if constexpr (kOut) {
          qq += q[e] * q[e];
          kq += q[e] * k[e];
        }
      }
      float rk = 1.f, rq = p.scale;
      if (p.normalise) {
        rk = 1.0f / sqrtf(wave_sum(kk) + 1e-6f);
        if constexpr (kOut) rq *= 1.0f / sqrtf(wave_sum(qq) + 1e-6f);
      }
      if constexpr (kOut) kq = wave_sum(kq) * rk * rq;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        ks[i][lane * kEach + e] = k[e] * rk;
        if constexpr (kOut) qs[i][lane * kEach + e] = q[e] * rq;
      }
      const float2 g = gates_of(p, t, head);
      if (lane == 0) {
        scalars[i][0] = expf(g.x);
        scalars[i][1] = g.y;
        scalars[i][2] = kq;
        scalars[i][3] = g.x > -0.5f ? expm1f(g.x) : kStrong;
      }
    }
    __syncthreads();
    for (int i = 0; i < n; ++i) {
      f32x4 k[kQuads], q[kQuads], kd{0.f, 0.f, 0.f, 0.f}, qd{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kQuads; ++j) {
        k[j] = *reinterpret_cast<const f32x4*>(&ks[i][4 * kGroups * j + 4 * group]);
        if constexpr (kOut) q[j] = *reinterpret_cast<const f32x4*>(&qs[i][4 * kGroups * j + 4 * group]);
      }
#pragma unroll
      for (int j = 0; j < kQuads; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          kd += state[j][e] * k[j][e];
          if constexpr (kOut) qd += state[j][e] * q[j][e];
        }
#pragma unroll
      for (int o = kCols; o < 64; o <<= 1)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          kd[c] += __shfl_xor(kd[c], o, 64);
          if constexpr (kOut) qd[c] += __shfl_xor(qd[c], o, 64);
        }
      const float decay = scalars[i][0], beta = scalars[i][1];
      const f32x4 v = *reinterpret_cast<const f32x4*>(&vs[i][col]);
      const f32x4 u = beta * (v - decay * kd);
      if constexpr (kOut) {
        if (group == 0) {
          const f32x4 o = decay * qd + scalars[i][2] * u;
          ushort4 r;
          r.x = from_f32<kBf16>(o[0]);
          r.y = from_f32<kBf16>(o[1]);
          r.z = from_f32<kBf16>(o[2]);
          r.w = from_f32<kBf16>(o[3]);
          *reinterpret_cast<ushort4*>(p.out + (static_cast<int64_t>(s.start + t0 + i) * p.Hv + head) * kDim + col) = r;
        }
      }
      const float fade = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(scalars[i][3])));
      if (fade != kStrong) {
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) state[j][e] = (fade * state[j][e] + state[j][e]) + k[j][e] * u;
      } else {
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) state[j][e] = decay * state[j][e] + k[j][e] * u;
      }
      if (t0 + i + 1 == s.count)
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) *reinterpret_cast<f32x4*>(place + (4 * kGroups * j + 4 * group + e) * kDim) = state[j][e];
    }
  }
}

constexpr int rule_lds(int dim, bool out) { return 16 * ((out ? 3 : 2) * dim + 4); }

template <bool kBf16, int kDim>
__global__ __launch_bounds__(256) void gdn_rule_kernel(RuleParams p) {
  __shared__ __align__(16) float lds[rule_lds(kDim, true)];
  rule_steps<kBf16, kDim, true>(p, blockIdx.x / p.Hv, blockIdx.x % p.Hv, lds);
}

// States and conv histories after the part of the block that counts, one launch for both: the first B * Hv workgroups
// take the states, the others the histories.
template <bool kBf16, int kDim>
__global__ __launch_bounds__(256) void gdn_advance_kernel(RuleParams p, ConvParams c) {
  __shared__ __align__(16) float lds[rule_lds(kDim, false)];
  const int states = p.pool.B * p.Hv;
  if (static_cast<int>(blockIdx.x) < states) {
    rule_steps<kBf16, kDim, false>(p, blockIdx.x / p.Hv, blockIdx.x % p.Hv, lds);
    return;
  }
  const int across = (c.channels + 2047) / 2048, i = blockIdx.x - states;
  const int channel = (i % across * 256 + threadIdx.x) * 8;
  if (channel >= c.channels) return;
  const Span s = span_of(c.pool, i / across);
  if (s.count == 0) return;
  const History h = load_history<kBf16>(c.pool, s, channel);
  store_history<kBf16>(c.pool, s, channel, h, c.x, c.x_stride);
}

}  // namespace

void launch_gdn_conv(bool bf16, const ConvParams& p, hipStream_t stream) {
  const int across = (p.channels + 2047) / 2048;
  constexpr int kRows = 8;
  if (static_cast<int64_t>(p.pool.T) * across <= 4096) {
    const dim3 grid(p.pool.T, across);
    if (bf16) hipLaunchKernelGGL((gdn_conv_kernel<true, 1>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((gdn_conv_kernel<false, 1>), grid, dim3(256), 0, stream, p);
  } else {
    const dim3 grid((p.pool.T + kRows - 1) / kRows, across);
    if (bf16) hipLaunchKernelGGL((gdn_conv_kernel<true, kRows>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((gdn_conv_kernel<false, kRows>), grid, dim3(256), 0, stream, p);
  }
}

void launch_gdn_rule(int dim, bool bf16, const RuleParams& p, hipStream_t stream) {
  const dim3 grid(p.pool.B * p.Hv);
  if (dim == 128) {
    if (bf16) hipLaunchKernelGGL((gdn_rule_kernel<true, 128>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((gdn_rule_kernel<false, 128>), grid, dim3(256), 0, stream, p);
  } else {
    if (bf16) hipLaunchKernelGGL((gdn_rule_kernel<true, 64>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((gdn_rule_kernel<false, 64>), grid, dim3(256), 0, stream, p);
  }
}

void launch_gdn_advance(int dim, bool bf16, const RuleParams& p, const ConvParams& c, hipStream_t stream) {
  const dim3 grid(p.pool.B * p.Hv + p.pool.B * ((c.channels + 2047) / 2048));
  if (dim == 128) {
    if (bf16) hipLaunchKernelGGL((gdn_advance_kernel<true, 128>), grid, dim3(256), 0, stream, p, c);
    else hipLaunchKernelGGL((gdn_advance_kernel<false, 128>), grid, dim3(256), 0, stream, p, c);
  } else {
    if (bf16) hipLaunchKernelGGL((gdn_advance_kernel<true, 64>), grid, dim3(256), 0, stream, p, c);
    else hipLaunchKernelGGL((gdn_advance_kernel<false, 64>), grid, dim3(256), 0, stream, p, c);
  }
}

}  // namespace dflash
