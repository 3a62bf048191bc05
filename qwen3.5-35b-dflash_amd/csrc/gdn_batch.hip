// A GDN layer's convolution and gated delta rule over a batch of sequences whose states lie in a pool.
//
// Reference arithmetic: model/qwen35_moe_dflash/fused/model.py:206-263 and fused/ops.py:36-71 (conv and, per token,
// S <- e^g S; u = beta (v - S^T k); S <- S + k u^T; o = S^T q).  Tokens [starts[b], starts[b + 1]) of the block are sequence
// b's; its conv history and state are slot slots[b] of the pool.  All three are read on the device, and whatever they
// hold leads to no address outside the block or the pool.
//
// Times stand for heads of 128 (16 of keys, 32 of values) where nothing else is said.
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
// b is the same in every lane, and so is what stands in memory for it.
__device__ __forceinline__ Span span_of(const PoolParams& p, int b) {
  const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  Span s;
  s.start = clampi(one(p.starts[b]), 0, p.T);
  s.tokens = clampi(one(p.starts[b + 1]), s.start, p.T) - s.start;
  s.slot = one(p.slots[b]);
  if (s.slot < 0 || s.slot >= p.pool_slots) s.slot = -1;
  s.count = p.counts ? clampi(one(p.counts[b]), 0, s.tokens) : s.tokens;
  if (s.slot < 0) s.count = 0;
  s.fresh = s.slot < 0 || (p.fresh && one(p.fresh[b]));
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

// silu(sum of weight x row) of eight channels: four rows, the token's own last.
template <bool kBf16>
__device__ __forceinline__ uint4 conv8(const float (&r0)[8], const float (&r1)[8], const float (&r2)[8], const float (&r3)[8],
                                       const float (&w)[8][kTaps]) {
  uint16_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = ((r0[i] * w[i][0] + r1[i] * w[i][1]) + r2[i] * w[i][2]) + r3[i] * w[i][3];
    o[i] = from_f32<kBf16>(y * __builtin_amdgcn_rcpf(1.0f + __expf(-y)));  // exponential and reciprocal to a step: far under the result's rounding
  }
  return make_uint4(o[0] | static_cast<uint32_t>(o[1]) << 16, o[2] | static_cast<uint32_t>(o[3]) << 16,
                    o[4] | static_cast<uint32_t>(o[5]) << 16, o[6] | static_cast<uint32_t>(o[7]) << 16);
}

// A workgroup per kRows tokens and 2048 channels, a thread eight neighbouring channels.  A block's first three rows read the
// history that the same thread replaces, so they go with the first of them, whichever tile they fall into.  Bound by memory: tiles
// inside one sequence have all their rows in flight at once.  8869 tokens of five prompts, 8192 channels: 56 us, 5.2 TB/s; a token 3.3.
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
  if (kRows > 1 && b < p.pool.B) {
    const Span s = span_of(p.pool, b);
    if (s.start + kTaps - 1 <= t0 && t0 + kRows <= s.start + s.tokens) {
      uint4 x[kRows + kTaps - 1];
      const uint16_t* from = p.x + (t0 - (kTaps - 1)) * p.x_stride + channel;
#pragma unroll
      for (int i = 0; i < kRows + kTaps - 1; ++i) x[i] = *reinterpret_cast<const uint4*>(from + i * p.x_stride);
      float f[kTaps][8];
#pragma unroll
      for (int j = 0; j < kTaps - 1; ++j) unpack8<kBf16>(x[j], f[j]);
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        unpack8<kBf16>(x[i + kTaps - 1], f[(i + kTaps - 1) % kTaps]);
        *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(t0 + i) * p.channels + channel) =
            conv8<kBf16>(f[i % kTaps], f[(i + 1) % kTaps], f[(i + 2) % kTaps], f[(i + 3) % kTaps], w);
      }
      return;
    }
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
    // a whole tile, or a block's first three rows where it starts at the tile's last ones
    constexpr int kMost = kRows > kTaps - 1 ? kRows : kTaps - 1;
    uint4 x[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i) x[i] = *reinterpret_cast<const uint4*>(p.x + min(lo + i, hi - 1) * p.x_stride + channel);
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      float f[8];
      unpack8<kBf16>(x[i], f);
      if (lo + i < hi) *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(lo + i) * p.channels + channel) = conv8<kBf16>(past[0], past[1], past[2], f, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        past[0][j] = past[1][j];
        past[1][j] = past[2][j];
        past[2][j] = f[j];
      }
    }
    if (first && s.count > 0) store_history<kBf16>(p.pool, s, channel, h, p.x, p.x_stride);
  }
}

// ------------------------------------------------------------------ the rule over short blocks
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

// A state's decay by e^g as S <- by S + rest S.  A slight one is S + (e^g - 1) S: e^g itself is off by half a step near 1, which a head
// that remembers thousands of tokens would sum up wherever its decay is a constant, call after call (a steady state's norm by 1e-4).
struct Fade {
  float by, rest;
};
__device__ __forceinline__ Fade fade_of(float g) { return g > -0.5f ? Fade{expm1f(g), 1.0f} : Fade{expf(g), 0.0f}; }

// x as the sum of kParts bf16 numbers, each the rounding of what the ones before leave.
template <int kParts, int kN>
__device__ __forceinline__ void cut(const float (&x)[kN], uint32_t (&parts)[kParts][kN / 2]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  float rest[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) rest[i] = x[i];
#pragma unroll
  for (int p = 0; p < kParts; ++p)
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      parts[p][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{rest[2 * i], rest[2 * i + 1]}, bf16x2));
      rest[2 * i] -= __uint_as_float(parts[p][i] << 16);
      rest[2 * i + 1] -= __uint_as_float(parts[p][i] & 0xFFFF0000u);
    }
}
// Eight 16-bit values as bf16 parts: bf16 as they are, fp16 (11 bits) as two.
template <bool kBf16>
__device__ __forceinline__ void row_parts(uint4 w, uint4 (&parts)[kBf16 ? 1 : 2]) {
  if constexpr (kBf16) {
    parts[0] = w;
  } else {
    float f[8];
    unpack8<false>(w, f);
    uint32_t c[2][4];
    cut<2, 8>(f, c);
    parts[0] = make_uint4(c[0][0], c[0][1], c[0][2], c[0][3]);
    parts[1] = make_uint4(c[1][0], c[1][1], c[1][2], c[1][3]);
  }
}
template <bool kBf16>
__device__ __forceinline__ f32x4 mfma_rows(uint4 a, uint4 b, f32x4 c) {
  if constexpr (kBf16) return mfma16x16x32(a, b, c);
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16x16x16(uint2 a, uint2 b, f32x4 c) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}

__device__ __forceinline__ float2 buf_load8(buf_rsrc r, int lane_offset, int offset) {
  return __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(r, lane_offset, offset, 0));
}
__device__ __forceinline__ void buf_store8(buf_rsrc r, int lane_offset, int offset, float2 v) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v), r, lane_offset, offset, 0);
}

__device__ __forceinline__ void buf_store16(buf_rsrc r, int lane_offset, int offset, f32x4 v) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, lane_offset, offset, 0);
}

// Sum over groups of 8 or 16 neighbouring lanes, and over the four 16-lane rows of a wave: no LDS trip.
template <int kLanes>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp_f32<0xB1>(v);   // quad_perm [1,0,3,2]
  v += dpp_f32<0x4E>(v);   // quad_perm [2,3,0,1]
  v += dpp_f32<0x141>(v);  // row_half_mirror
  if constexpr (kLanes == 16) v += dpp_f32<0x140>(v);  // row_mirror
  return v;
}
__device__ __forceinline__ float rows_sum(float v) {
  auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// ------------------------------------------------------------------ the rule, token after token
// For blocks of a token or two, where reading and writing the state is all (a token's arithmetic takes as long whatever the block
// is).  One workgroup per (sequence, value head), its state in registers: wave w holds columns [w D/4, (w + 1) D/4), a lane four
// columns of kQuads x 4 rows, so a column's products with the state (S^T k, S^T q) are sums over kGroups lanes of one wave, and
// so are the norms: no LDS and no barrier, and between the sequence's place and the last store one round trip to memory.
// o = S_new^T q = e^g S_old^T q + u (k.q) takes both products from the old state.  64 sequences 57 us (4.7 TB/s; 45 where the last-level
// cache still holds their states from the call before), one 6 us, its latency.
template <int kGroups>
__device__ __forceinline__ float groups_sum(float v) {
  if constexpr (kGroups == 16) v += dpp_f32<0x124>(v);  // row_ror:4
  return rows_sum(v + dpp_f32<0x128>(v));               // row_ror:8
}

template <bool kBf16, int kDim>
__device__ __forceinline__ void rule_tokens(const RuleParams& p, const Span& s, int head) {
  constexpr int kCols = kDim / 16, kGroups = 64 / kCols, kQuads = kDim / (4 * kGroups);
  const int khead = head / p.rep, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int col = wave * (kDim / 4) + 4 * (lane % kCols), group = lane / kCols;
  const buf_rsrc place = make_rsrc(p.pool.recurrent + max(s.slot, 0) * p.pool.recurrent_stride + static_cast<int64_t>(head) * kDim * kDim,
                                   s.slot < 0 ? 0 : kDim * kDim * 4);
  const int at = (4 * group * kDim + col) * 4;
  const auto row_place = [](int j, int e) { return (4 * kGroups * j + e) * kDim * 4; };
  struct Token {
    uint2 k[kQuads], q[kQuads], v;
    float2 gates;
  };
  const auto load = [&](int i) {
    Token o;
    const int64_t t = s.start + i;
    const uint16_t* k = p.key + t * p.key_token + khead * p.key_head + 4 * group;
    const uint16_t* q = p.query + t * p.query_token + khead * p.query_head + 4 * group;
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
      o.k[j] = *reinterpret_cast<const uint2*>(k + 4 * kGroups * j);
      o.q[j] = *reinterpret_cast<const uint2*>(q + 4 * kGroups * j);
    }
    o.v = *reinterpret_cast<const uint2*>(p.value + t * p.value_token + head * p.value_head + col);
    o.gates = gates_of(p, t, head);
    return o;
  };
  const auto four = [](uint2 w) {
    return f32x4{to_f32<kBf16>(static_cast<uint16_t>(w.x)), to_f32<kBf16>(static_cast<uint16_t>(w.x >> 16)),
                 to_f32<kBf16>(static_cast<uint16_t>(w.y)), to_f32<kBf16>(static_cast<uint16_t>(w.y >> 16))};
  };
  f32x4 state[kQuads][4];  // rows 4 kGroups j + 4 group + e
  if (s.fresh) {
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) state[j][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  } else {
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) state[j][e] = __builtin_bit_cast(f32x4, buf_load16(place, at, row_place(j, e)));
  }
  Token token = load(0);
#pragma unroll 1
  for (int i = 0;; ++i) {
    f32x4 k[kQuads], kd{0.f, 0.f, 0.f, 0.f}, qd{0.f, 0.f, 0.f, 0.f};
    float kk = 0.f, qq = 0.f, kq = 0.f;
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
      k[j] = four(token.k[j]);
      const f32x4 q = four(token.q[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        kk += k[j][e] * k[j][e];
        qq += q[e] * q[e];
        kq += k[j][e] * q[e];
        kd += state[j][e] * k[j][e];
        qd += state[j][e] * q[e];
      }
    }
    kk = groups_sum<kGroups>(kk);
    qq = groups_sum<kGroups>(qq);
    kq = groups_sum<kGroups>(kq);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      kd[x] = groups_sum<kGroups>(kd[x]);
      qd[x] = groups_sum<kGroups>(qd[x]);
    }
    const float rk = p.normalise ? 1.0f / sqrtf(kk + 1e-6f) : 1.0f, rq = (p.normalise ? 1.0f / sqrtf(qq + 1e-6f) : 1.0f) * p.scale;
    const float g = token.gates.x, decay = expf(g);
    const f32x4 u = token.gates.y * (four(token.v) - (decay * rk) * kd);
    if (group == 0) {
      const f32x4 o = (decay * rq) * qd + (kq * rk * rq) * u;
      ushort4 w;
      w.x = from_f32<kBf16>(o[0]);
      w.y = from_f32<kBf16>(o[1]);
      w.z = from_f32<kBf16>(o[2]);
      w.w = from_f32<kBf16>(o[3]);
      *reinterpret_cast<ushort4*>(p.out + (static_cast<int64_t>(s.start + i) * p.Hv + head) * kDim + col) = w;
    }
    const bool last = i + 1 == s.tokens;
    if (last && s.count != s.tokens) break;  // nobody sees the state behind the last token
    if (!last) token = load(i + 1);
    const Fade fade = fade_of(g);
    const f32x4 write = rk * u;
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) state[j][e] = (fade.by * state[j][e] + fade.rest * state[j][e]) + k[j][e] * write;
    if (i + 1 == s.count)
#pragma unroll
      for (int j = 0; j < kQuads; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) buf_store16(place, at, row_place(j, e), state[j][e]);
    if (last) break;
  }
}
template <bool kBf16, int kDim>
__global__ __launch_bounds__(256, 3) void gdn_token_kernel(RuleParams p) {
  const Span s = span_of(p.pool, blockIdx.x / p.Hv);
  if (s.tokens > 0) rule_tokens<kBf16, kDim>(p, s, blockIdx.x % p.Hv);
}

// Blocks of up to so many tokens go token after token.  us a call, that way and 16 at a time: 64 sequences of one token 45 and 68, of two 51
// and 69, of three 60 and 68, of four 71 and 69; 32 of four both 42; one of one 5.4 and 12.5, of four 12.0 and 12.6; 16 heads of 64, 32
// sequences of two 8.1 and 11.2, of three 10.0 and 11.2, of four 12.3 and 11.3.
constexpr int kTokenSteps = 3;

// ------------------------------------------------------------------ the rule, 16 tokens at a time
// A workgroup holds one head's state of one sequence in registers, 32 columns a wave: register (i, x, e) of lane l is row
// 16 i + 4 (l >> 4) + e, column 2 (l & 15) + x, which is the layout of a matrix instruction's result (the columns of tile x are
// every other one, so that a lane loads two neighbours) and, when the sum over rows is taken in that order, of a B operand.  So
// the state takes part in products without leaving its registers.  Sub-blocks of up to 16 tokens with the formulas of a chunk (below):
//   X = V - diag(e^G r) K S,  U = T X,  O = diag(e^G rq) Q S + P U,  S <- e^G S + K^T diag(e^{G_end - G} r) U.
// 32 sequences of up to 16 tokens 35 us with the state left alone (74 MB: memory takes 14; the rest is the sub-block's chain of
// K K^T, the substitution, two products and the output, some 6 us behind the load of the state, in 1.3 rounds of three workgroups a CU),
// 40 us as gdn_advance, which writes it (139 MB).
template <bool kBf16, int kDim>
struct BlockShared {
  uint16_t k[16][kDim + 8], q[16][kDim + 8];
  float a[16][20], t[16][20], p[16][20];
  double total[16];           // G
  float gate[16], beta[16], rk[16], rq[16], key[16], query[16], write[16];
  Fade fade[16];              // by e^G
};

template <bool kBf16, int kDim, bool kOut>
__device__ __forceinline__ void rule_block(const RuleParams& p, const Span& s, int head, BlockShared<kBf16, kDim>& lds) {
  constexpr int kTiles = kDim / 16, kWaves = kDim / 32, kLanes = kDim / 8, kRowParts = kBf16 ? 1 : 2;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, lr = lane & 15, quarter = lane >> 4;
  const int col = 32 * wave + 2 * lr, khead = head / p.rep;
  const int limit = kOut ? s.tokens : s.count;
  if (limit == 0) return;
  // through a buffer, whose rows are uniform offsets: a lane's own 32 addresses would take 64 registers (no slot: nothing is read or written)
  const buf_rsrc place = make_rsrc(p.pool.recurrent + max(s.slot, 0) * p.pool.recurrent_stride + static_cast<int64_t>(head) * kDim * kDim,
                                   s.slot < 0 ? 0 : kDim * kDim * 4);
  const int at = (4 * quarter * kDim + col) * 4;
  const auto row_place = [](int i, int e) { return (16 * i + e) * kDim * 4; };
  float st[kTiles][4][2];
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 v = s.fresh ? make_float2(0.f, 0.f) : buf_load8(place, at, row_place(i, e));
      st[i][e][0] = v.x;
      st[i][e][1] = v.y;
    }
#pragma unroll 1
  for (int b0 = 0; b0 < limit; b0 += 16) {
    const int n = min(16, limit - b0), t0 = s.start + b0;
    if (b0) __syncthreads();
    {
      const int r = tid / kLanes, d = tid % kLanes * 8;  // a row each group of lanes
      const int64_t t = t0 + min(r, n - 1);
      uint4 k = *reinterpret_cast<const uint4*>(p.key + t * p.key_token + khead * p.key_head + d), q = make_uint4(0, 0, 0, 0);
      if constexpr (kOut) q = *reinterpret_cast<const uint4*>(p.query + t * p.query_token + khead * p.query_head + d);
      if (r >= n) k = q = make_uint4(0, 0, 0, 0);
      if (wave == kWaves - 1 && lane < 16) {
        float2 g = make_float2(0.f, 0.f);
        if (lane < n) g = gates_of(p, t0 + lane, head);
        lds.gate[lane] = g.x < -200.0f ? -200.0f : g.x;  // e^-200 is 0 in fp32, and what stands behind it keeps its bits
        lds.beta[lane] = g.y;
      }
      float f[8], h[8], kk = 0.f, qq = 0.f;
      unpack8<kBf16>(k, f);
      unpack8<kBf16>(q, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        kk += f[e] * f[e];
        qq += h[e] * h[e];
      }
      kk = group_sum<kLanes>(kk);
      const float rk = p.normalise ? 1.0f / sqrtf(kk + 1e-6f) : 1.0f;
      float rq = p.scale;
      if constexpr (kOut) {
        qq = group_sum<kLanes>(qq);
        if (p.normalise) rq *= 1.0f / sqrtf(qq + 1e-6f);
      }
      if (d == 0) {
        lds.rk[r] = rk;
        lds.rq[r] = rq;
      }
      *reinterpret_cast<uint4*>(&lds.k[r][d]) = k;
      if constexpr (kOut) *reinterpret_cast<uint4*>(&lds.q[r][d]) = q;
    }
    uint32_t v[4];  // two columns of tokens 4 quarter + e
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] = *reinterpret_cast<const uint32_t*>(p.value + (t0 + min(4 * quarter + e, n - 1)) * p.value_token + head * p.value_head + col);
    __syncthreads();

    // K S and Q S, 32 rows of the state an instruction
    f32x4 ks[2], qs[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) ks[x] = qs[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    // first what the others wait for: A on wave 0, P on the next
    if (wave < (kOut ? 2 : 1)) {
      f32x4 d{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < kDim / 32; ++m) {
        const uint4 other = *reinterpret_cast<const uint4*>(&lds.k[lr][32 * m + 8 * quarter]);
        const uint4 own = wave ? *reinterpret_cast<const uint4*>(&lds.q[lr][32 * m + 8 * quarter]) : other;
        d = mfma_rows<kBf16>(own, other, d);
      }
      // the running log decay in 64 bits, so that a decay e^{G_t - G_s} is as exact as its own exponent
      double sum = 0.0, here = 0.0, rows[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sum += static_cast<double>(lds.gate[i]);
        if (i == lr) here = sum;
        if (i >> 2 == quarter) rows[i & 3] = sum;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = 4 * quarter + e;
        const float decay = lr <= t ? __expf(static_cast<float>(rows[e] - here)) * lds.rk[lr] : 0.f;
        if (wave) lds.p[t][lr] = lds.rq[t] * decay * d[e];
        else lds.a[t][lr] = lr < t ? lds.beta[t] * lds.rk[t] * decay * d[e] : 0.f;
      }
      if (wave == 0) {
        if (lane < 16) {
          const float decay = expf(static_cast<float>(here));
          lds.key[lr] = decay * lds.rk[lr];
          lds.query[lr] = decay * lds.rq[lr];
          lds.write[lr] = expf(static_cast<float>(sum - here)) * lds.rk[lr];
          lds.total[lr] = here;
          lds.fade[lr] = fade_of(static_cast<float>(here));
        }
        // (I + A)^-1 diag(beta) by forward substitution, a column a lane (one wave wrote A and reads it)
        __builtin_amdgcn_wave_barrier();
        if (lane < 16) {
          float x[16];
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            float s0 = t == lr ? lds.beta[lr] : 0.f, s1 = 0.f;
#pragma unroll
            for (int i = 0; i < t; ++i) {
              const float f = lds.a[t][i];
              if (i & 1) s1 -= f * x[i];
              else s0 -= f * x[i];
            }
            x[t] = s0 + s1;
            lds.t[t][lr] = x[t];
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < kDim / 32; ++m) {
      uint4 k[kRowParts], q[kRowParts];
      const auto rows = [&](const uint16_t(&from)[16][kDim + 8], uint4(&to)[kRowParts]) {
        const uint2 lo = *reinterpret_cast<const uint2*>(&from[lr][32 * m + 4 * quarter]);
        const uint2 hi = *reinterpret_cast<const uint2*>(&from[lr][32 * m + 16 + 4 * quarter]);
        row_parts<kBf16>(make_uint4(lo.x, lo.y, hi.x, hi.y), to);
      };
      rows(lds.k, k);
      if constexpr (kOut) rows(lds.q, q);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float f[8] = {st[2 * m][0][x],     st[2 * m][1][x],     st[2 * m][2][x],     st[2 * m][3][x],
                            st[2 * m + 1][0][x], st[2 * m + 1][1][x], st[2 * m + 1][2][x], st[2 * m + 1][3][x]};
        uint32_t c[3][4];
        cut<3, 8>(f, c);
#pragma unroll
        for (int i = 2; i >= 0; --i) {
          const uint4 part = make_uint4(c[i][0], c[i][1], c[i][2], c[i][3]);
          if (!kBf16 && i < 2) ks[x] = mfma16x16x32(k[kRowParts - 1], part, ks[x]);
          ks[x] = mfma16x16x32(k[0], part, ks[x]);
          if constexpr (kOut) {
            if (!kBf16 && i < 2) qs[x] = mfma16x16x32(q[kRowParts - 1], part, qs[x]);
            qs[x] = mfma16x16x32(q[0], part, qs[x]);
          }
        }
      }
    }
    __syncthreads();
    const f32x4 key = *reinterpret_cast<const f32x4*>(&lds.key[4 * quarter]), t = *reinterpret_cast<const f32x4*>(&lds.t[lr][4 * quarter]);
    f32x4 u[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      u[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        u[x] = mfma16x16x4f32(t[e], to_f32<kBf16>(static_cast<uint16_t>(v[e] >> 16 * x)) - key[e] * ks[x][e], u[x]);
    }
    if constexpr (kOut) {
      const f32x4 query = *reinterpret_cast<const f32x4*>(&lds.query[4 * quarter]), w = *reinterpret_cast<const f32x4*>(&lds.p[lr][4 * quarter]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        qs[x] *= query;
#pragma unroll
        for (int e = 0; e < 4; ++e) qs[x] = mfma16x16x4f32(w[e], u[x][e], qs[x]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * quarter + e < n)
          *reinterpret_cast<uint32_t*>(p.out + (static_cast<int64_t>(t0 + 4 * quarter + e) * p.Hv + head) * kDim + col) =
              from_f32<kBf16>(qs[0][e]) | static_cast<uint32_t>(from_f32<kBf16>(qs[1][e])) << 16;
    }
    // the state after the first `part` tokens, into the pool or as the one that goes on
    const auto after = [&](int part, bool keep_it) {
      f32x4 write = *reinterpret_cast<const f32x4*>(&lds.write[4 * quarter]);
      if (part < n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * quarter + e;
          write[e] = r < part ? expf(static_cast<float>(lds.total[part - 1] - lds.total[r])) * lds.rk[r] : 0.f;
        }
      const Fade fade = lds.fade[part - 1];
      uint2 w[2][3];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float f[4] = {write[0] * u[x][0], write[1] * u[x][1], write[2] * u[x][2], write[3] * u[x][3]};
        uint32_t c[3][2];
        cut<3, 4>(f, c);
#pragma unroll
        for (int i = 0; i < 3; ++i) w[x][i] = make_uint2(c[i][0], c[i][1]);
      }
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        uint16_t r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = lds.k[4 * quarter + e][16 * i + lr];
        uint2 k[kRowParts];
        if constexpr (kBf16) {
          k[0] = make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
        } else {
          const float f[4] = {to_f32<false>(r[0]), to_f32<false>(r[1]), to_f32<false>(r[2]), to_f32<false>(r[3])};
          uint32_t c[2][2];
          cut<2, 4>(f, c);
          k[0] = make_uint2(c[0][0], c[0][1]);
          k[1] = make_uint2(c[1][0], c[1][1]);
        }
        f32x4 sum[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[x][e] = fade.by * st[i][e][x] + fade.rest * st[i][e][x];
#pragma unroll
          for (int j = 2; j >= 0; --j) {
            if (!kBf16 && j < 2) sum[x] = mfma16x16x16(k[kRowParts - 1], w[x][j], sum[x]);
            sum[x] = mfma16x16x16(k[0], w[x][j], sum[x]);
          }
        }
        if (keep_it) {
#pragma unroll
          for (int e = 0; e < 4; ++e) buf_store8(place, at, row_place(i, e), make_float2(sum[0][e], sum[1][e]));
        } else {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) st[i][e][x] = sum[x][e];
        }
      }
    };
    const int part = s.count - b0;
    if (part > 0 && (part <= n || b0 + 16 >= limit)) after(min(part, n), true);
    if (b0 + 16 >= limit) return;
    after(n, false);
  }
}

template <bool kBf16, int kDim>
__global__ __launch_bounds__(2 * kDim, 3) void gdn_rule_kernel(RuleParams p) {
  __shared__ __align__(16) BlockShared<kBf16, kDim> lds;
  const Span s = span_of(p.pool, blockIdx.x / p.Hv);
  if (p.most && s.tokens > p.most) return;
  if constexpr (kDim == 128) {  // four waves, as that way is cut
    if (s.tokens <= kTokenSteps) {
      if (s.tokens > 0) rule_tokens<kBf16, kDim>(p, s, blockIdx.x % p.Hv);
      return;
    }
  }
  rule_block<kBf16, kDim, true>(p, s, blockIdx.x % p.Hv, lds);
}

// States and conv histories after the part of the block that counts, one launch for both: the first B * Hv workgroups
// take the states, the others the histories.
template <bool kBf16, int kDim>
__global__ __launch_bounds__(2 * kDim, 3) void gdn_advance_kernel(RuleParams p, ConvParams c) {
  __shared__ __align__(16) BlockShared<kBf16, kDim> lds;
  const int states = p.pool.B * p.Hv;
  if (static_cast<int>(blockIdx.x) < states) {
    rule_block<kBf16, kDim, false>(p, span_of(p.pool, blockIdx.x / p.Hv), blockIdx.x % p.Hv, lds);
    return;
  }
  const int across = (c.channels + 16 * kDim - 1) / (16 * kDim), i = blockIdx.x - states;
  const int channel = (i % across * 2 * kDim + threadIdx.x) * 8;
  if (channel >= c.channels) return;
  const Span s = span_of(c.pool, i / across);
  if (s.count == 0) return;
  const History h = load_history<kBf16>(c.pool, s, channel);
  store_history<kBf16>(c.pool, s, channel, h, c.x, c.x_stride);
}

// ------------------------------------------------------------------ the rule, 64 tokens at a time
// With G the running sum of g in a chunk, r the keys' and q's norms' inverses (q's with the scale) and raw rows k, q, v:
//   A_ts = beta_t r_t r_s e^{G_t - G_s} k_t.k_s (s < t),   T = (I + A)^-1 diag(beta),
//   P_ts = rq_t r_s e^{G_t - G_s} q_t.k_s (s <= t),
//   X = V - diag(e^G r) K S,   U = T X,   O = diag(e^G rq) Q S + P U,   S <- e^{G_64} S + K^T diag(e^{G_64 - G} r) U.
// T and P do not depend on the state: gdn_chunk_kernel makes them for all chunks at once, and gdn_scan_kernel walks a
// sequence's chunks with a 16-column slice of the state per workgroup.
//
// Precision: the products take 16-bit operands of the matrix cores and sum in fp32.  Raw rows are 16 bits as they are (fp16:
// two bf16 parts, since states need bf16's range), norms and gates stand beside them as fp32 factors.  What meets them (S, X, U,
// T, P) is cut into three bf16 parts, 24 bits, and of their products those above 2^-24 of the whole are taken.  So states and outputs
// come out as from fp32 products, at 1/3 to 1/6 of the 16-bit rate instead of 1/16 of it.  (Two parts for what only an output sees
// would be exact enough for the output's own rounding, but not where its terms cancel: a prompt of 4096 tokens took 147 us so, 160 now.)
constexpr int kChunk = 64, kPitch = 68;     // tokens of a chunk; floats of an LDS row
constexpr int kTriangle = 6;                // 16 x 32 fragments of a lower triangle of 64 x 64
__device__ __forceinline__ int triangle(int block, int step) { return block < 2 ? block : 2 * block - 2 + step; }

// Chunks of a sequence, none of one with fewer than `least` tokens; and the sequence and chunk of an ordinal (a wave's lanes together),
// x = B: none.
__device__ __forceinline__ int chunks_of(const PoolParams& p, int least, int b) {
  const int start = clampi(p.starts[b], 0, p.T), tokens = clampi(p.starts[b + 1], start, p.T) - start;
  return tokens < least ? 0 : (tokens + kChunk - 1) / kChunk;
}
__device__ __forceinline__ int2 chunk_place(const PoolParams& p, int least, int ordinal) {
  int base = 0;
  for (int i = 0; i < p.B; i += 64) {
    const int b = i + lane_id();
    const int own = b < p.B ? chunks_of(p, least, b) : 0;
    int sum = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o, 64);
      if (lane_id() >= o) sum += v;
    }
    const uint64_t over = __ballot(base + sum > ordinal);
    if (over) {
      const int lane = __ffsll(static_cast<unsigned long long>(over)) - 1;
      return make_int2(__builtin_amdgcn_readfirstlane(i + lane),
                       __builtin_amdgcn_readfirstlane(ordinal - base - (__shfl(sum, lane, 64) - __shfl(own, lane, 64))));
    }
    base += __shfl(sum, 63, 64);
  }
  return make_int2(p.B, 0);
}
// The sequence with chunks that `ordinal` of them stand before, and the chunks before its own; x = B: none.
__device__ __forceinline__ int2 sequence_place(const PoolParams& p, int least, int ordinal) {
  int seen = 0, base = 0;
  for (int i = 0; i < p.B; i += 64) {
    const int lane = lane_id(), b = i + lane;
    const int own = b < p.B ? chunks_of(p, least, b) : 0;
    const uint64_t held = __ballot(own > 0);
    const int n = __popcll(held);
    if (seen + n > ordinal) {
      const uint64_t at = __ballot(own > 0 && __popcll(held & ((uint64_t{1} << lane) - 1)) == ordinal - seen);
      const int hit = __ffsll(static_cast<unsigned long long>(at)) - 1;
      const int before = wave_sum_int(lane < hit ? own : 0);
      return make_int2(__builtin_amdgcn_readfirstlane(i + hit), __builtin_amdgcn_readfirstlane(base + before));
    }
    seen += n;
    base = min(base + wave_sum_int(own), 1 << 24);  // bounded: starts that do not ascend may count a token many times
  }
  return make_int2(p.B, 0);
}

// One workgroup per (chunk, value head), wave w rows 16 w .. 16 w + 15 of the chunk's matrices: 2048 of them 49 us for 4096 tokens of one
// sequence, a chain of seven steps with barriers between, three workgroups a CU (LDS).  Rows come in whole (256 bytes a
// load of 16 lanes) and pass through LDS: what the scan reads eight times over, once a slice, it finds in the order of
// its operands, 1 KB a load (rows read straight into operands cost a cache line a lane).
template <bool kBf16, int kDim>
__global__ __launch_bounds__(256) void gdn_chunk_kernel(ChunkParams c) {
  const RuleParams& p = c.rule;
  constexpr int kSteps = kDim / 32, kRowParts = kBf16 ? 1 : 2, kRaw = kDim + 8;
  union Shared {
    uint16_t raw[kChunk][kRaw];
    float f[kChunk][kPitch];
  };
  __shared__ __align__(16) Shared keys_t, query_p;  // first the rows, then T and P
  __shared__ __align__(16) float am[kChunk][kPitch];
  __shared__ double gsum[kChunk];
  __shared__ float beta[kChunk], rk[kChunk], rq[kChunk];
  auto& tm = keys_t.f;
  auto& pm = query_p.f;
  const int ordinal = blockIdx.x / p.Hv, head = blockIdx.x % p.Hv, khead = head / p.rep;
  const int2 place = chunk_place(p.pool, c.least, ordinal);
  if (place.x == p.pool.B) return;
  const Span s = span_of(p.pool, place.x);
  const int t0 = s.start + place.y * kChunk, n = min(kChunk, s.start + s.tokens - t0);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int lr = lane & 15, quarter = lane >> 4;
  const int blocks = (n + 15) / 16;  // row blocks that hold tokens
  const int64_t at = static_cast<int64_t>(ordinal) * p.Hv + head;

  {
    constexpr int kLanes = kDim / 8, kRows = 256 / kLanes;  // lanes a row, rows a pass
    const int r0 = tid / kLanes, d = tid % kLanes * 8;
    uint4 k[kChunk / kRows], q[kChunk / kRows];
#pragma unroll
    for (int i = 0; i < kChunk / kRows; ++i) {
      const int r = r0 + i * kRows;
      const int64_t t = t0 + min(r, n - 1);
      k[i] = *reinterpret_cast<const uint4*>(p.key + t * p.key_token + khead * p.key_head + d);
      q[i] = *reinterpret_cast<const uint4*>(p.query + t * p.query_token + khead * p.query_head + d);
    }
    if (wave == 0) {
      float2 g = make_float2(0.f, 0.f);
      if (lane < n) g = gates_of(p, t0 + lane, head);
      // the running log decay in 64 bits, so that a decay e^{G_t - G_s} is as exact as its own exponent; bounded from below, so
      // that what stands behind a decay of -infinity keeps its bits (e^-200 is 0 in fp32 all the same)
      double sum = g.x < -200.0f ? -200.0f : g.x;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double x = __shfl_up(sum, o, 64);
        if (lane >= o) sum += x;
      }
      gsum[lane] = sum;
      beta[lane] = g.y;
    }
#pragma unroll
    for (int i = 0; i < kChunk / kRows; ++i) {
      const int r = r0 + i * kRows;
      if (r >= n) k[i] = q[i] = make_uint4(0, 0, 0, 0);
      float f[8], kk = 0.f, qq = 0.f;
      unpack8<kBf16>(k[i], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) kk += f[e] * f[e];
      unpack8<kBf16>(q[i], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) qq += f[e] * f[e];
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) {
        kk += __shfl_xor(kk, o, 64);
        qq += __shfl_xor(qq, o, 64);
      }
      if (d == 0) {
        rk[r] = p.normalise ? 1.0f / sqrtf(kk + 1e-6f) : 1.0f;
        rq[r] = (p.normalise ? 1.0f / sqrtf(qq + 1e-6f) : 1.0f) * p.scale;
      }
      *reinterpret_cast<uint4*>(&keys_t.raw[r][d]) = k[i];
      *reinterpret_cast<uint4*>(&query_p.raw[r][d]) = q[i];
    }
  }
  __syncthreads();

  // A and P of this wave's rows, without their factors
  f32x4 a[4], q[4];
  uint4 own_k[kSteps], own_q[kSteps];
#pragma unroll
  for (int m = 0; m < kSteps; ++m) {
    own_k[m] = *reinterpret_cast<const uint4*>(&keys_t.raw[16 * wave + lr][32 * m + 8 * quarter]);
    own_q[m] = *reinterpret_cast<const uint4*>(&query_p.raw[16 * wave + lr][32 * m + 8 * quarter]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    a[j] = q[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (j <= wave)
#pragma unroll
      for (int m = 0; m < kSteps; ++m) {
        const uint4 k = *reinterpret_cast<const uint4*>(&keys_t.raw[16 * j + lr][32 * m + 8 * quarter]);
        a[j] = mfma_rows<kBf16>(own_k[m], k, a[j]);
        q[j] = mfma_rows<kBf16>(own_q[m], k, q[j]);
      }
  }
  // the rows as operands: keys and queries, and the keys transposed, once for the value heads that share them
  if (head % p.rep == 0) {
    uint16_t* to = c.rows + (static_cast<int64_t>(ordinal) * (p.Hv / p.rep) + khead) * (2 * kDim * kChunk) + lane * 8;
#pragma unroll
    for (int m = 0; m < kSteps; ++m) {
      *reinterpret_cast<uint4*>(to + (wave * kSteps + m) * 512) = own_k[m];
      *reinterpret_cast<uint4*>(to + kDim * kChunk + (wave * kSteps + m) * 512) = own_q[m];
    }
    to = c.kt + (static_cast<int64_t>(ordinal) * (p.Hv / p.rep) + khead) * (kRowParts * kDim * kChunk) + lane * 8;
    for (int f = wave; f < kDim / 16 * 2; f += 4) {  // fragment: 16 features, 32 tokens
      uint16_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = keys_t.raw[32 * (f & 1) + 8 * quarter + i][16 * (f >> 1) + lr];
      uint4 parts[kRowParts];
      row_parts<kBf16>(make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16), parts);
#pragma unroll
      for (int i = 0; i < kRowParts; ++i) *reinterpret_cast<uint4*>(to + i * kDim * kChunk + f * 512) = parts[i];
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j > (wave | 1)) continue;  // never read
    const int col = 16 * j + lr;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 16 * wave + 4 * quarter + e;
      const float decay = col <= row ? __expf(static_cast<float>(gsum[row] - gsum[col])) * rk[col] : 0.f;
      am[row][col] = col < row ? beta[row] * rk[row] * decay * a[j][e] : 0.f;
      pm[row][col] = col <= row ? rq[row] * decay * q[j][e] : 0.f;
    }
  }
  __syncthreads();

  // (I + A)^-1: the diagonal blocks by forward substitution, a column a lane; then block column w on wave w:
  // T_ij = -T_ii sum_k A_ik T_kj.  A result's registers (rows 4 quarter + e) are the next product's B operand when the sum is
  // taken in that order.
  if (lane < 16) {
    float x[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      float sum0 = t == lr ? 1.f : 0.f, sum1 = 0.f;
#pragma unroll
      for (int i = 0; i < t; ++i) {
        const float f = am[16 * wave + t][16 * wave + i];
        if (i & 1) sum1 -= f * x[i];
        else sum0 -= f * x[i];
      }
      x[t] = sum0 + sum1;
      tm[16 * wave + t][16 * wave + lr] = x[t];
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j != wave) continue;
    f32x4 col[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) col[j][e] = tm[16 * j + 4 * quarter + e][16 * j + lr];
#pragma unroll
    for (int i = j + 1; i < 4; ++i) {
      f32x4 sum{0.f, 0.f, 0.f, 0.f}, next{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = j; k < i; ++k) {
        const f32x4 f = *reinterpret_cast<const f32x4*>(&am[16 * i + lr][16 * k + 4 * quarter]);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = mfma16x16x4f32(f[e], col[k][e], sum);
      }
      const f32x4 d = *reinterpret_cast<const f32x4*>(&tm[16 * i + lr][16 * i + 4 * quarter]);
#pragma unroll
      for (int e = 0; e < 4; ++e) next = mfma16x16x4f32(d[e], -sum[e], next);
      col[i] = next;
#pragma unroll
      for (int e = 0; e < 4; ++e) tm[16 * i + 4 * quarter + e][16 * j + lr] = next[e];
    }
    if (j & 1)  // above the diagonal in the same fragment
#pragma unroll
      for (int e = 0; e < 4; ++e) tm[16 * (j - 1) + 4 * quarter + e][16 * j + lr] = 0.f;
  }
  __syncthreads();

  // T and P as operands
  if (wave < blocks) {
    const int row = 16 * wave + lr;
    for (int m = 0; m <= wave / 2; ++m) {
      const int col = 32 * m + 8 * quarter, f = triangle(wave, m);
      float x[8], y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = tm[row][col + i] * beta[col + i];
        y[i] = pm[row][col + i];
      }
      uint32_t pp[3][4];
      cut<3, 8>(y, pp);
      float* t = c.t + (at * kTriangle + f) * 512 + lane * 4;
      *reinterpret_cast<float4*>(t) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(t + 256) = make_float4(x[4], x[5], x[6], x[7]);
#pragma unroll
      for (int i = 0; i < 3; ++i)
        *reinterpret_cast<uint4*>(c.p + ((at * 3 + i) * kTriangle + f) * 512 + lane * 8) = make_uint4(pp[i][0], pp[i][1], pp[i][2], pp[i][3]);
    }
  }
  if (tid < kChunk) {
    ChunkScalars* to = c.scalars + at;
    const bool in = tid < n;
    const float head_decay = expf(static_cast<float>(gsum[tid]));
    to->key[tid] = in ? head_decay * rk[tid] : 0.f;
    to->query[tid] = head_decay * rq[tid];
    to->write[tid] = in ? expf(static_cast<float>(gsum[kChunk - 1] - gsum[tid])) * rk[tid] : 0.f;
    to->norm[tid] = rk[tid];
    to->total[tid] = gsum[tid];
    if (tid == 0) {
      const Fade fade = fade_of(static_cast<float>(gsum[kChunk - 1]));
      to->fade = fade.by;
      to->rest = fade.rest;
    }
  }
}

// What the waves of gdn_scan_kernel leave for one another: S, X, U times its writes' decays, and U (of this chunk and the one before),
// as bf16 parts in the order of a B operand, per 16 columns.
template <int kDim, int kTiles>
struct ScanShared {
  uint4 state[kTiles][3][kDim * 2], x[kTiles][3][128], write[kTiles][3][128], u[2][kTiles][3][128];
};
// Four values of rows 16 tile + 4 quarter .. + 3 and a lane's column: half of a B operand's eight, per part.
template <int kParts>
__device__ __forceinline__ void put_parts(uint4* to, int part_stride, const float (&x)[4], int tile) {
  const int lane = lane_id(), lr = lane & 15, quarter = lane >> 4;
  uint32_t w[kParts][2];
  cut<kParts, 4>(x, w);
#pragma unroll
  for (int i = 0; i < kParts; ++i)
    reinterpret_cast<uint2*>(to + i * part_stride + (2 * tile + (quarter >> 1)) * 16 + lr)[quarter & 1] = make_uint2(w[i][0], w[i][1]);
}

// The chunk's place in a walk over a sequence.
struct ScanWalk {
  int base, count, head, slice;
};
// Column of tile x and lane column lr: with two tiles every other one, so that a lane's two are neighbours.
template <int kTiles>
__device__ __forceinline__ int scan_column(const ScanWalk& w, int lr) {
  return kTiles * (16 * w.slice + lr);
}

// Waves 0 to 3 of gdn_scan_kernel: X and U of 16 tokens.  In both kinds of waves loads stand in no branch but a first one (indices
// are bounded instead) and nothing is computed from them before they are needed, so that those of the two chunks ahead stay in flight.
template <bool kBf16, int kDim, int kTiles>
__device__ __forceinline__ void scan_solve(const ChunkParams& c, const Span& s, const ScanWalk& w, int block, ScanShared<kDim, kTiles>& lds) {
  const RuleParams& p = c.rule;
  constexpr int kSteps = kDim / 32, kRowParts = kBf16 ? 1 : 2;
  const int lane = lane_id(), quarter = lane >> 4, khead = w.head / p.rep, last = w.count - 1;
  const int col = scan_column<kTiles>(w, lane & 15);
  struct Ops {
    uint4 rows[kSteps];  // K
    float4 mat[2][2];    // T
    f32x4 scale, write;  // e^G r, e^{G_64 - G} r
    uint32_t v[4];       // V: a row's kTiles columns
  };
  const auto load = [&](int i, Ops& o) {
    const int64_t at = static_cast<int64_t>(w.base + i) * p.Hv + w.head;
    const float* mat = c.t + (at * kTriangle + triangle(block, 0)) * 512 + lane * 4;
    if (block > 1)
#pragma unroll
      for (int h = 0; h < 2; ++h) o.mat[1][h] = *reinterpret_cast<const float4*>(mat + 512 + 256 * h);
#pragma unroll
    for (int h = 0; h < 2; ++h) o.mat[0][h] = *reinterpret_cast<const float4*>(mat + 256 * h);
    const uint16_t* rows = c.rows + (static_cast<int64_t>(w.base + i) * (p.Hv / p.rep) + khead) * (2 * kDim * kChunk) + block * (kSteps * 512) + lane * 8;
#pragma unroll
    for (int m = 0; m < kSteps; ++m) o.rows[m] = *reinterpret_cast<const uint4*>(rows + m * 512);
    const ChunkScalars* f = c.scalars + at;
    o.scale = *reinterpret_cast<const f32x4*>(f->key + 16 * block + 4 * quarter);
    o.write = *reinterpret_cast<const f32x4*>(f->write + 16 * block + 4 * quarter);
    const int t0 = s.start + i * kChunk, n = min(kChunk, s.tokens - i * kChunk);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint16_t* v = p.value + (t0 + min(16 * block + 4 * quarter + e, n - 1)) * p.value_token + w.head * p.value_head + col;
      if constexpr (kTiles == 2) o.v[e] = *reinterpret_cast<const uint32_t*>(v);
      else o.v[e] = *v;
    }
  };
  uint4 mat[3][2];  // T of the chunk at hand, in parts
  const auto cut_mat = [&](const Ops& o) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const float f[8] = {o.mat[m][0].x, o.mat[m][0].y, o.mat[m][0].z, o.mat[m][0].w, o.mat[m][1].x, o.mat[m][1].y, o.mat[m][1].z, o.mat[m][1].w};
      uint32_t parts[3][4];
      cut<3, 8>(f, parts);
#pragma unroll
      for (int i = 0; i < 3; ++i) mat[i][m] = make_uint4(parts[i][0], parts[i][1], parts[i][2], parts[i][3]);
    }
  };
  const auto step = [&](int i, Ops& o, const Ops& next) {
    const int n = min(kChunk, s.tokens - i * kChunk);
    const bool active = 16 * block < n;
    lds_barrier();  // the state's parts are there
#pragma unroll
    for (int x = 0; x < kTiles; ++x) {
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (active) {
        f32x4 sum[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int m = 0; m < kSteps; ++m) {
          uint4 r[kRowParts], st[3];
          row_parts<kBf16>(o.rows[m], r);
#pragma unroll
          for (int i3 = 0; i3 < 3; ++i3) st[i3] = lds.state[x][i3][m * 64 + lane];
#pragma unroll
          for (int i3 = 2; i3 >= 0; --i3) {
            if (!kBf16 && i3 < 2) sum[m & 1] = mfma16x16x32(r[kRowParts - 1], st[i3], sum[m & 1]);
            sum[m & 1] = mfma16x16x32(r[0], st[i3], sum[m & 1]);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = to_f32<kBf16>(static_cast<uint16_t>(o.v[e] >> 16 * x)) - o.scale[e] * (sum[0][e] + sum[1][e]);
      }
      put_parts<3>(lds.x[x][0], 128, f, block);
    }
    lds_barrier();  // X is there
    float u[kTiles][4];
#pragma unroll
    for (int x = 0; x < kTiles; ++x) {
      float scaled[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) u[x][e] = 0.f;
      if (active) {
        f32x4 sum[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int m = 0; m < 2; ++m)
          if (m <= block / 2) {
            uint4 f[3];
#pragma unroll
            for (int i3 = 0; i3 < 3; ++i3) f[i3] = lds.x[x][i3][m * 64 + lane];
            sum[0] = mfma16x16x32(mat[2][m], f[0], sum[0]);
            sum[1] = mfma16x16x32(mat[1][m], f[1], sum[1]);
            sum[0] = mfma16x16x32(mat[0][m], f[2], sum[0]);
            sum[1] = mfma16x16x32(mat[1][m], f[0], sum[1]);
            sum[0] = mfma16x16x32(mat[0][m], f[1], sum[0]);
            sum[1] = mfma16x16x32(mat[0][m], f[0], sum[1]);
          }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u[x][e] = sum[0][e] + sum[1][e];
          scaled[e] = o.write[e] * u[x][e];
        }
      }
      put_parts<3>(lds.write[x][0], 128, scaled, block);
    }
#pragma unroll
    for (int x = 0; x < kTiles; ++x) put_parts<3>(lds.u[i & 1][x][0], 128, u[x], block);
    lds_barrier();  // U is there
    const int part = s.count - i * kChunk;
    if (part > 0 && part < n) {
      // the kept state ends inside this chunk: U once more, with the decays up to its last token
      const ChunkScalars* f = c.scalars + static_cast<int64_t>(w.base + i) * p.Hv + w.head;
      const double end = f->total[part - 1];
      float factor[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * block + 4 * quarter + e;
        factor[e] = r < part ? expf(static_cast<float>(end - f->total[r])) * f->norm[r] : 0.f;
      }
      lds_barrier();  // the whole chunk's is taken
#pragma unroll
      for (int x = 0; x < kTiles; ++x) {
        const float scaled[4] = {factor[0] * u[x][0], factor[1] * u[x][1], factor[2] * u[x][2], factor[3] * u[x][3]};
        put_parts<3>(lds.write[x][0], 128, scaled, block);
      }
      lds_barrier();
    }
    load(min(i + 2, last), o);
    cut_mat(next);
  };
  Ops o0, o1;
  load(0, o0);
  load(min(1, last), o1);
  wait_vmem();  // so that the loop, whose registers these loads may have passed through, starts with none in flight
  cut_mat(o0);
#pragma unroll 1
  for (int i = 0; i <= last; i += 2) {
    step(i, o0, o1);
    if (i < last) step(i + 1, o1, o0);
  }
}

// Waves 4 to 7: the outputs of 16 tokens and a quarter of the state's rows.  Q S follows the state at once; P U, which nobody waits
// for, a chunk later, while the others solve.
template <bool kBf16, int kDim, int kTiles>
__device__ __forceinline__ void scan_output(const ChunkParams& c, const Span& s, const ScanWalk& w, int block, ScanShared<kDim, kTiles>& lds) {
  const RuleParams& p = c.rule;
  constexpr int kSteps = kDim / 32, kRowParts = kBf16 ? 1 : 2, kHeld = kDim / 64;  // 16-row tiles of the state
  const int lane = lane_id(), lr = lane & 15, quarter = lane >> 4, khead = w.head / p.rep, last = w.count - 1;
  const int col = scan_column<kTiles>(w, lr);
  float* state = p.pool.recurrent + s.slot * p.pool.recurrent_stride +
                 (static_cast<int64_t>(w.head) * kDim + 16 * kHeld * block + 4 * quarter) * kDim + col;
  f32x4 st[kHeld][kTiles];
#pragma unroll
  for (int h = 0; h < kHeld; ++h)
#pragma unroll
    for (int x = 0; x < kTiles; ++x) st[h][x] = f32x4{0.f, 0.f, 0.f, 0.f};
  typedef float Columns __attribute__((ext_vector_type(kTiles)));
  if (!s.fresh)
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Columns v = *reinterpret_cast<const Columns*>(state + (16 * h + e) * kDim);
#pragma unroll
        for (int x = 0; x < kTiles; ++x) st[h][x][e] = v[x];
      }
  const auto keep_state = [&](const f32x4 (&from)[kHeld][kTiles]) {
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        Columns v;
#pragma unroll
        for (int x = 0; x < kTiles; ++x) v[x] = from[h][x][e];
        *reinterpret_cast<Columns*>(state + (16 * h + e) * kDim) = v;
      }
  };
  const auto put_state = [&]() {
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
#pragma unroll
      for (int x = 0; x < kTiles; ++x) {
        const float f[4] = {st[h][x][0], st[h][x][1], st[h][x][2], st[h][x][3]};
        put_parts<3>(lds.state[x][0], kDim * 2, f, kHeld * block + h);
      }
  };

  struct Ops {
    uint4 rows[kSteps], kt[kRowParts][kHeld][2];             // Q, the keys transposed
    f32x4 scale;                                             // e^G rq
    Fade fade;                                               // by e^G of the chunk
  };
  const auto load = [&](int i, Ops& o) {
    const int64_t at = static_cast<int64_t>(w.base + i) * p.Hv + w.head;
    const int64_t shared = static_cast<int64_t>(w.base + i) * (p.Hv / p.rep) + khead;
    const uint16_t* rows = c.rows + shared * (2 * kDim * kChunk) + kDim * kChunk + block * (kSteps * 512) + lane * 8;
#pragma unroll
    for (int m = 0; m < kSteps; ++m) o.rows[m] = *reinterpret_cast<const uint4*>(rows + m * 512);
    const ChunkScalars* f = c.scalars + at;
    o.scale = *reinterpret_cast<const f32x4*>(f->query + 16 * block + 4 * quarter);
    o.fade = Fade{f->fade, f->rest};
    const uint16_t* kt = c.kt + shared * (kRowParts * kDim * kChunk) + block * (kHeld * 1024) + lane * 8;
#pragma unroll
    for (int i3 = 0; i3 < kRowParts; ++i3)
#pragma unroll
      for (int h = 0; h < kHeld; ++h)
#pragma unroll
        for (int m = 0; m < 2; ++m) o.kt[i3][h][m] = *reinterpret_cast<const uint4*>(kt + i3 * kDim * kChunk + (2 * h + m) * 512);
  };
  uint4 mat[3][2];  // P of the chunk before, in parts
  const auto load_mat = [&](int i) {
    const uint16_t* from = c.p + (static_cast<int64_t>(w.base + i) * p.Hv + w.head) * (3 * kTriangle * 512) + triangle(block, 0) * 512 + lane * 8;
    if (block > 1)
#pragma unroll
      for (int i3 = 0; i3 < 3; ++i3) mat[i3][1] = *reinterpret_cast<const uint4*>(from + (i3 * kTriangle + 1) * 512);
#pragma unroll
    for (int i3 = 0; i3 < 3; ++i3) mat[i3][0] = *reinterpret_cast<const uint4*>(from + i3 * kTriangle * 512);
  };
  // S faded + K^T (the writes in LDS)
  const auto update = [&](const Ops& o, const Fade& fade, f32x4 (&sum)[kHeld][kTiles]) {
#pragma unroll
    for (int x = 0; x < kTiles; ++x) {
      uint4 u[2][3];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < 3; ++i) u[m][i] = lds.write[x][i][m * 64 + lane];
#pragma unroll
      for (int h = 0; h < kHeld; ++h) sum[h][x] = fade.by * st[h][x] + fade.rest * st[h][x];
#pragma unroll
      for (int i = 2; i >= 0; --i)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int h = 0; h < kHeld; ++h) {
            if (!kBf16 && i < 2) sum[h][x] = mfma16x16x32(o.kt[kRowParts - 1][h][m], u[m][i], sum[h][x]);
            sum[h][x] = mfma16x16x32(o.kt[0][h][m], u[m][i], sum[h][x]);
          }
    }
  };
  f32x4 seen[kTiles];  // e^G rq Q S of the chunk whose P U is still to come
  const auto write_out = [&](int i) {
    const int t0 = s.start + i * kChunk, n = min(kChunk, s.tokens - i * kChunk);
    if (16 * block >= n) return;
    f32x4 sum[kTiles];
#pragma unroll
    for (int x = 0; x < kTiles; ++x) {
      sum[x] = seen[x];
#pragma unroll
      for (int m = 0; m < 2; ++m)
        if (m <= block / 2) {
          uint4 f[3];
#pragma unroll
          for (int i3 = 0; i3 < 3; ++i3) f[i3] = lds.u[i & 1][x][i3][m * 64 + lane];
          sum[x] = mfma16x16x32(mat[2][m], f[0], sum[x]);
          sum[x] = mfma16x16x32(mat[1][m], f[1], sum[x]);
          sum[x] = mfma16x16x32(mat[0][m], f[2], sum[x]);
          sum[x] = mfma16x16x32(mat[1][m], f[0], sum[x]);
          sum[x] = mfma16x16x32(mat[0][m], f[1], sum[x]);
          sum[x] = mfma16x16x32(mat[0][m], f[0], sum[x]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = 16 * block + 4 * quarter + e;
      uint16_t* to = p.out + (static_cast<int64_t>(t0 + r) * p.Hv + w.head) * kDim + col;
      if (r < n) {
        if constexpr (kTiles == 2) *reinterpret_cast<uint32_t*>(to) = from_f32<kBf16>(sum[0][e]) | static_cast<uint32_t>(from_f32<kBf16>(sum[1][e])) << 16;
        else *to = from_f32<kBf16>(sum[0][e]);
      }
    }
  };

  const auto step = [&](int i, const Ops& o, Ops& next) {
    const int n = min(kChunk, s.tokens - i * kChunk);
    const bool active = 16 * block < n;
    lds_barrier();  // the state's parts are there
    f32x4 rows[kTiles];
#pragma unroll
    for (int x = 0; x < kTiles; ++x) rows[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (active)
#pragma unroll
      for (int x = 0; x < kTiles; ++x)
#pragma unroll
        for (int m = 0; m < kSteps; ++m) {
          uint4 r[kRowParts];
          row_parts<kBf16>(o.rows[m], r);
#pragma unroll
          for (int i3 = 2; i3 >= 0; --i3) {
            const uint4 f = lds.state[x][i3][m * 64 + lane];
            if (!kBf16 && i3 < 2) rows[x] = mfma16x16x32(r[kRowParts - 1], f, rows[x]);
            rows[x] = mfma16x16x32(r[0], f, rows[x]);
          }
        }
    load(min(i + 1, last), next);
    if (i > 0 && s.count == i * kChunk) keep_state(st);  // the kept state ends where this chunk begins
    lds_barrier();                                       // X is there
    if (i > 0) write_out(i - 1);
    load_mat(i);
#pragma unroll
    for (int x = 0; x < kTiles; ++x) seen[x] = o.scale * rows[x];
    lds_barrier();  // U is there
    f32x4 after[kHeld][kTiles];
    update(o, o.fade, after);
    const int part = s.count - i * kChunk;
    if (part > 0 && part < n) {
      const double end = c.scalars[static_cast<int64_t>(w.base + i) * p.Hv + w.head].total[part - 1];
      lds_barrier();
      lds_barrier();
      f32x4 kept[kHeld][kTiles];
      update(o, fade_of(static_cast<float>(end)), kept);
      keep_state(kept);
    }
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
#pragma unroll
      for (int x = 0; x < kTiles; ++x) st[h][x] = after[h][x];
    put_state();
  };

  Ops o0, o1;
  load(0, o0);
  put_state();
  wait_vmem();
#pragma unroll 1
  for (int i = 0; i <= last; i += 2) {
    step(i, o0, o1);
    if (i < last) step(i + 1, o1, o0);
  }
  write_out(last);
  if (s.count == s.tokens && s.count > 0) keep_state(st);
}

// One workgroup per (sequence, value head, 16 kTiles columns of the state), the sequence's chunks in turn.  Three barriers a chunk:
// S, then X, then U are there.  Bound by that chain: 2.0 us a chunk, 127 us for 4096 tokens of one sequence.
template <bool kBf16, int kDim, int kTiles>
__global__ __launch_bounds__(512) void gdn_scan_kernel(ChunkParams c) {
  const RuleParams& p = c.rule;
  constexpr int kSlices = kDim / (16 * kTiles);
  __shared__ __align__(16) ScanShared<kDim, kTiles> lds;
  const int group = blockIdx.x / (8 * kSlices), rest = blockIdx.x % (8 * kSlices);
  const int unit = group * 8 + rest % 8;  // a head's slices on one XCD, which share all but V
  if (unit >= c.sequences * p.Hv) return;
  const int2 place = sequence_place(p.pool, c.least, unit / p.Hv);
  if (place.x == p.pool.B) return;
  const Span s = span_of(p.pool, place.x);
  ScanWalk w;
  w.base = place.y;
  w.count = min((s.tokens + kChunk - 1) / kChunk, c.chunks - w.base);
  w.head = unit % p.Hv;
  w.slice = rest / 8;
  if (w.count <= 0) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave < 4) scan_solve<kBf16, kDim, kTiles>(c, s, w, wave, lds);
  else scan_output<kBf16, kDim, kTiles>(c, s, w, wave - 4, lds);
}

}  // namespace

void launch_gdn_conv(bool bf16, const ConvParams& p, hipStream_t stream) {
  const int across = (p.channels + 2047) / 2048;
  // Eight tokens a workgroup share the rows before them; where sequences have one token each they would only stand in line:
  // 64 single tokens 6.2 us one a workgroup, 15.9 eight; 512 blocks of two 32 and 20; 64 blocks of 16 29 and 10.
  constexpr int kRows = 8;
  if (p.pool.T < 2 * static_cast<int64_t>(p.pool.B)) {
    const dim3 grid(p.pool.T, across);
    if (bf16) hipLaunchKernelGGL((gdn_conv_kernel<true, 1>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((gdn_conv_kernel<false, 1>), grid, dim3(256), 0, stream, p);
  } else {
    const dim3 grid((p.pool.T + kRows - 1) / kRows, across);
    if (bf16) hipLaunchKernelGGL((gdn_conv_kernel<true, kRows>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((gdn_conv_kernel<false, kRows>), grid, dim3(256), 0, stream, p);
  }
}

template <bool kBf16, int kDim>
void launch_chunks(const ChunkParams& c, hipStream_t stream) {
  const RuleParams& p = c.rule;
  hipLaunchKernelGGL((gdn_chunk_kernel<kBf16, kDim>), dim3(c.chunks * p.Hv), dim3(256), 0, stream, c);
  const int units = (c.sequences * p.Hv + 7) / 8 * 8, typical = c.typical * p.Hv;
  // Registers let a CU hold one workgroup at head dim 128 (168 a lane at least, 512 threads; two would have to do with 128), so workgroups
  // are counted in rounds of the card.  With 32 columns one reads half as much a column and takes longer: it pays where that saves rounds.
  // us a call, 16 and 32 columns, by sequences of 1024 tokens: one 53 and 62, two 97 and 81, four 172 and 144; 16 heads of 64, of 512 tokens:
  // six both 39, twelve 66 and 69.
  const auto rounds = [&](int columns) { return (typical * (kDim / columns) + c.cus - 1) / c.cus; };
  if (5 * rounds(32) <= 3 * rounds(16))
    hipLaunchKernelGGL((gdn_scan_kernel<kBf16, kDim, 2>), dim3(units * (kDim / 32)), dim3(512), 0, stream, c);
  else
    hipLaunchKernelGGL((gdn_scan_kernel<kBf16, kDim, 1>), dim3(units * (kDim / 16)), dim3(512), 0, stream, c);
  if (c.least > 1) {
    RuleParams rest = p;
    rest.most = c.least - 1;
    hipLaunchKernelGGL((gdn_rule_kernel<kBf16, kDim>), dim3(p.pool.B * p.Hv), dim3(2 * kDim), 0, stream, rest);
  }
}

void launch_gdn_chunks(int dim, bool bf16, const ChunkParams& c, hipStream_t stream) {
  if (dim == 128) bf16 ? launch_chunks<true, 128>(c, stream) : launch_chunks<false, 128>(c, stream);
  else bf16 ? launch_chunks<true, 64>(c, stream) : launch_chunks<false, 64>(c, stream);
}

template <bool kBf16, int kDim>
void launch_rule(const RuleParams& p, int64_t longest, hipStream_t stream) {
  if (longest <= kTokenSteps) hipLaunchKernelGGL((gdn_token_kernel<kBf16, kDim>), dim3(p.pool.B * p.Hv), dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((gdn_rule_kernel<kBf16, kDim>), dim3(p.pool.B * p.Hv), dim3(2 * kDim), 0, stream, p);
}
template <bool kBf16, int kDim>
void launch_advance(const RuleParams& p, const ConvParams& c, hipStream_t stream) {
  const int across = (c.channels + 16 * kDim - 1) / (16 * kDim);
  hipLaunchKernelGGL((gdn_advance_kernel<kBf16, kDim>), dim3(p.pool.B * (p.Hv + across)), dim3(2 * kDim), 0, stream, p, c);
}

void launch_gdn_rule(int dim, bool bf16, const RuleParams& p, int64_t longest, hipStream_t stream) {
  if (dim == 128) bf16 ? launch_rule<true, 128>(p, longest, stream) : launch_rule<false, 128>(p, longest, stream);
  else bf16 ? launch_rule<true, 64>(p, longest, stream) : launch_rule<false, 64>(p, longest, stream);
}

void launch_gdn_advance(int dim, bool bf16, const RuleParams& p, const ConvParams& c, hipStream_t stream) {
  if (dim == 128) bf16 ? launch_advance<true, 128>(p, c, stream) : launch_advance<false, 128>(p, c, stream);
  else bf16 ? launch_advance<true, 64>(p, c, stream) : launch_advance<false, 64>(p, c, stream);
}

}  // namespace dflash
