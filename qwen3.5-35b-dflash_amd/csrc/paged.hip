// Paged-cache kernels: append with Q/K norm and position rotation, and attention of a batch of blocks over the pages.
//
// Append (model/qwen35_moe_dflash/fused/model.py:265-294 per sequence).  For a row x of the query or key:
//   n = x / sqrt(mean x^2 + eps) * (w + 1);  y_i = n_i cos a_i - n_{i+h} sin a_i, y_{i+h} = n_{i+h} cos a_i + n_i sin a_i
//   (i < h = rotary_dim / 2, a_i = position * inv_freq_i), the other features as they are; one rounding to 16 bits.
// K and V rows go to row (length - tokens + i) of their sequence.
//
// Attention.  Over keys j < visible(row): m = max s_j, l = sum e^{s_j - m}, o = sum e^{s_j - m} v_j, out = o / l, with
// s_j = scale q.k_j in fp32 from exact products of 16-bit values; a row that sees no key gives zeros.  Partial results
// over disjoint keys merge as m = max m_i, l = sum l_i e^{m_i - m}, o = sum o_i e^{m_i - m}: chunks of a long sequence, and a
// prefix that all sequences share, whose keys are taken once for the stacked rows of the whole batch.
// A probability is rounded to 16 bits for the product with V, as V itself is held; the sum l takes it unrounded.  Each is off by
// at most half a step, and its error is weighed as the value it multiplies: that leaves the sum about as far off as the output's own
// rounding does.
#include <algorithm>
#include <type_traits>

#include "kernels.h"

namespace dflash {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct Bf16 {
  typedef __bf16 Pair __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kExponent = 0x7F80;  // all ones: an infinity or NaN
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_f32(uint16_t v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ uint16_t from_f32(float v) { return f32_to_bf16(v); }
  static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
struct Fp16 {
  typedef _Float16 Pair __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kExponent = 0x7C00;
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_f32(uint16_t v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }
  static __device__ __forceinline__ uint16_t from_f32(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }
  static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <class E>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), typename E::Pair));
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

__device__ __forceinline__ SeqSpan load_span(const PagedParams& p, int b) {
  return seq_span(p.starts[b], p.starts[b + 1], p.own.lengths[b], p.T, p.own.capacity);
}

// Element offset of the page that holds a sequence's 16 rows from 16 * g on, and their first row inside the page.  Pages
// are multiples of 16 rows, or one page is the whole sequence, so 16 rows never lie in two.  An entry outside the pool
// is taken as the nearest page: nothing outside the pool is read.
struct PageAt {
  int page, row;
};
__device__ __forceinline__ PageAt page_at(const PagedSide& s, const int32_t* table, int g) {
  const int i = divide(g, s.groups_per_page);
  return {clampi(table[i], 0, s.pages - 1), (g - i * s.page_groups) * 16};
}

// ------------------------------------------------------------------ append
// One workgroup per (token, slice of its heads); D / 8 lanes a head row, 8 features a lane.  The token's cosines and sines are
// made once for all its heads: 64-bit products and reduction by 2 pi (positions reach 2^31, where a 32-bit angle is off by
// more than a turn), then fp32 functions of the remainder.
template <int D, class E>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p) {
  constexpr int L = D / 8, kHeads = 256 / L;
  __shared__ float cs[D / 2], sn[D / 2];
  const int t = blockIdx.x, tid = threadIdx.x;
  // the token's sequence: the first whose end lies past it (64 ends at a time, one a lane)
  int b = p.B;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int lane = tid & 63;
    const bool past = b0 + lane < p.B && p.starts[b0 + lane + 1] > t;
    const uint64_t m = __ballot(past);
    if (m) {
      b = b0 + __builtin_ctzll(m);
      break;
    }
  }
  b = uniform(b);
  if (b == p.B) return;
  const SeqSpan s = seq_span(p.starts[b], p.starts[b + 1], p.side.lengths[b], p.T, p.side.capacity);
  if (t < s.start || t >= s.start + s.tokens) return;
  const int row = s.keys - s.tokens + t - s.start;
  if (p.half) {
    const int position = p.positions ? p.positions[t] : row;
    for (int i = tid; i < p.half; i += 256) {
      const double a = static_cast<double>(position) * static_cast<double>(p.inv_freq[i]);
      const double turns = rint(a * 0.15915494309189535);
      const float r = static_cast<float>(fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, a)));
      cs[i] = cosf(r);
      sn[i] = sinf(r);
    }
  }
  __syncthreads();
  const int all = p.heads + 2 * p.kv, c = (tid % L) * 8;
  for (int j = blockIdx.y * kHeads + tid / L; j < all; j += gridDim.y * kHeads) {
    const bool is_q = j < p.heads, is_v = j >= p.heads + p.kv;
    const int h = is_q ? j : is_v ? j - p.heads - p.kv : j - p.heads;
    const uint16_t* src = is_q ? p.query + t * p.query_token + h * p.query_head
                        : is_v ? p.value + t * p.value_token + h * p.value_head
                               : p.key + t * p.key_token + h * p.key_head;
    const u32x4 raw = *reinterpret_cast<const u32x4*>(src + c);
    u32x4 out = raw;
    if (!is_v) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = E::to_f32(raw[i] & 0xFFFF);
        v[2 * i + 1] = E::to_f32(raw[i] >> 16);
      }
      const float* w = is_q ? p.q_norm : p.k_norm;
      if (w) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[i] * v[i];
#pragma unroll
        for (int o = 1; o < L; o <<= 1) sum += __shfl_xor(sum, o, 64);
        const float inv = rsqrtf(sum / D + p.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * (w[c + i] + 1.0f);
      }
      if (p.half) {  // a multiple of 8: a lane's features rotate with those of one other lane of its row
        const int lanes = p.half / 8, at = tid % L;
        const bool rot = at < 2 * lanes, first = at < lanes;
        const int other = rot ? (first ? tid + lanes : tid - lanes) : tid;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = __shfl(v[i], other & 63, 64);
          if (rot) {
            const int k = first ? c + i : c - p.half + i;
            v[i] = v[i] * cs[k] + (first ? -x : x) * sn[k];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = pack2<E>(v[2 * i], v[2 * i + 1]);
    }
    if (is_q) {
      *reinterpret_cast<u32x4*>(p.query_out + (static_cast<int64_t>(t) * p.heads + h) * D + c) = out;
    } else if (row >= 0) {
      const int i = divide(row >> 4, p.side.groups_per_page), page = p.side.table[b * p.side.table_stride + i];
      const int inside = row - i * p.side.page_groups * 16;
      if (page >= 0 && page < p.side.pages) {
        uint16_t* dst = is_v ? p.values + page * p.side.value_page + h * p.side.value_head + inside * p.side.value_row
                             : p.keys + page * p.side.key_page + h * p.side.key_head + inside * p.side.key_row;
        *reinterpret_cast<u32x4*>(dst + c) = out;
      }
    }
  }
}

// ------------------------------------------------------------------ a workgroup's share of the attention
struct Share {
  int start, tokens, keys;  // the rows' block (start: its first token) and the keys of its sequence
  int tile, chunk, chunks;  // row tile and chunk of its keys
  int partial;              // partial tile of the tile's first chunk (per KV head), or -1: the result is final
  int c;                    // units a chunk
  const int32_t* table;
};

// Share `id` of the own-keys stage: every wave finds it by itself, 64 sequences at a time, one a lane.
__device__ __forceinline__ bool own_share(const PagedParams& p, int id, int tile_rows, int unit, int least, Share* out) {
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    int64_t u = 0;
    if (b0 + lane < p.B) {
      const SeqSpan s = load_span(p, b0 + lane);
      u = static_cast<int64_t>(seq_tiles(s.tokens, p.group, tile_rows)) * seq_units(s.keys, unit);
    }
    for (int o = 1; o < 64; o <<= 1) u += __shfl_xor(u, o, 64);
    total += u;
  }
  const int c = uniform(chunk_units(total, p.kv, p.slots, least));
  int first = 0, held = 0;  // shares and partial tiles of the sequences before
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    SeqSpan s{0, 0, 0};
    int n = 0, k = 1;
    if (b0 + lane < p.B) {
      s = load_span(p, b0 + lane);
      k = tile_chunks(seq_units(s.keys, unit), c);
      n = seq_tiles(s.tokens, p.group, tile_rows) * k;
    }
    const int kept = k > 1 || p.merge_prefix ? n : 0;
    int sum = n, sum_kept = kept;
    for (int o = 1; o < 64; o <<= 1) {
      const int a = __shfl_up(sum, o, 64), d = __shfl_up(sum_kept, o, 64);
      if (lane >= o) {
        sum += a;
        sum_kept += d;
      }
    }
    const uint64_t m = __ballot(n > 0 && id < first + sum);
    if (m) {
      const int l = __builtin_ctzll(m);
      const int rest = id - (first + __builtin_amdgcn_readlane(sum - n, l));
      const int chunks = __builtin_amdgcn_readlane(k, l);
      out->start = __builtin_amdgcn_readlane(s.start, l);
      out->tokens = __builtin_amdgcn_readlane(s.tokens, l);
      out->keys = __builtin_amdgcn_readlane(s.keys, l);
      out->tile = uniform(rest / chunks);
      out->chunk = uniform(rest - out->tile * chunks);
      out->chunks = chunks;
      out->partial = chunks > 1 || p.merge_prefix
                         ? uniform(held + __builtin_amdgcn_readlane(sum_kept - kept, l) + out->tile * chunks) : -1;
      out->c = c;
      out->table = p.own.table + static_cast<int64_t>(b0 + l) * p.own.table_stride;
      return true;
    }
    first += __builtin_amdgcn_readlane(sum, 63);
    held += __builtin_amdgcn_readlane(sum_kept, 63);
  }
  return false;
}

// Share `id` of the prefix stage: one sequence whose block is the whole batch.
__device__ __forceinline__ bool prefix_share(const PagedParams& p, int id, int tile_rows, int unit, int least, Share* out) {
  const int keys = uniform(clampi(p.prefix.lengths[0], 0, p.prefix.capacity));
  const int tiles = seq_tiles(p.T, p.group, tile_rows), units = seq_units(keys, unit);
  const int c = chunk_units(static_cast<int64_t>(tiles) * units, p.kv, p.slots, least);
  const int chunks = tile_chunks(units, c);
  if (id >= tiles * chunks) return false;
  *out = Share{0, p.T, keys, id / chunks, id % chunks, chunks, id / chunks * chunks, c, p.prefix.table};
  return true;
}

// ------------------------------------------------------------------ 16 rows, four waves over the keys
// For blocks of few rows.  Scores transposed, S^T = K Q^T: lane l holds query row l & 15 and keys 4 (l >> 4) + e of each of two
// 16-key tiles, which, with those eight keys as the reduction's octet l >> 4, is the B operand of O^T = V^T P^T as it stands.  The A
// operand needs eight keys of one dim per lane: a lane loads D / 16 neighbouring dims of its eight keys and pairs halves in
// registers, so V needs no transpose and neither operand passes through LDS.
constexpr int kSmallRows = 16, kSmallUnit = 128;  // keys a round of the four waves
template <int D, class E, bool kPrefix>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_small_kernel(PagedParams p) {
  constexpr int NC = D / 16, KS = D / 32, VL = NC / 8, kPitch = D + 4;
  __shared__ __align__(16) float osum[4][16][kPitch];
  __shared__ float mx[4][16], ls[4][16];
  const int kvh = blockIdx.x % p.kv;
  Share w;
  if (!(kPrefix ? prefix_share(p, blockIdx.x / p.kv, kSmallRows, kSmallUnit, 1, &w)
                : own_share(p, blockIdx.x / p.kv, kSmallRows, kSmallUnit, 1, &w)))
    return;
  const PagedSide& side = kPrefix ? p.prefix : p.own;
  const bool causal = !kPrefix && p.causal;
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, lr = lane & 15, kq = lane >> 4;
  const int rows = w.tokens * p.group, nrows = min(16, rows - w.tile * 16);
  const int r = w.tile * 16 + min(lr, nrows - 1);  // this lane's row in its block
  const int tok = r / p.group, head = kvh * p.group + r - tok * p.group;
  const int visible = visible_keys(w.keys, w.tokens, tok, causal);
  const int tok0 = uniform(w.tile * 16 / p.group), tok1 = uniform((w.tile * 16 + nrows - 1) / p.group);
  const int least = visible_keys(w.keys, w.tokens, tok0, causal);  // keys that every row of the tile sees
  const int n = visible_keys(w.keys, w.tokens, tok1, causal);      // keys that some row sees
  const int k0 = w.chunk * w.c * kSmallUnit, k1 = min(k0 + w.c * kSmallUnit, n);

  u32x4 q[KS];
  {
    const uint16_t* qr = p.query + (w.start + tok) * p.query_token + head * p.query_head + 8 * kq;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const u32x4*>(qr + 32 * s);
  }
  const uint16_t* keys = side.keys + kvh * side.key_head;
  const uint16_t* vals = side.values + kvh * side.value_head;
  f32x4 o[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), l = 0.f;

  for (int j0 = k0 + 32 * wave; j0 < k1; j0 += kSmallUnit) {
    u32x4 kf[2][KS], vf[8][VL];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      // a group past the last key repeats the last group, a row past it the last row; both are masked below
      const int g = min(j0 / 16 + b, (n - 1) / 16), left = n - 1 - 16 * g;
      const PageAt at = page_at(side, w.table, g);
      const uint16_t* kr = keys + at.page * side.key_page + (at.row + min(lr, left)) * side.key_row + 8 * kq;
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[b][s] = *reinterpret_cast<const u32x4*>(kr + 32 * s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint16_t* vr = vals + at.page * side.value_page + (at.row + min(4 * kq + i, left)) * side.value_row + NC * lr;
#pragma unroll
        for (int h = 0; h < VL; ++h) vf[4 * b + i][h] = *reinterpret_cast<const u32x4*>(vr + 8 * h);
      }
    }
    float s8[8];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) acc = E::mfma16(kf[b][s], q[s], acc);
#pragma unroll
      for (int e = 0; e < 4; ++e) s8[4 * b + e] = j0 + 16 * b + 4 * kq + e < visible ? acc[e] : -__builtin_inff();
    }
    float mc = fmaxf(fmaxf(fmaxf(s8[0], s8[1]), fmaxf(s8[2], s8[3])), fmaxf(fmaxf(s8[4], s8[5]), fmaxf(s8[6], s8[7])));
    mc = fmaxf(mc, __shfl_xor(mc, 16, 64));
    mc = fmaxf(mc, __shfl_xor(mc, 32, 64));
    const float mn = fmaxf(m, mc);
    // a row that has seen no key keeps weights of 0 (the exponent is -inf); a NaN score, which the maximum skips, makes l and
    // o NaN, and so they stay
    const float ref = mn == -__builtin_inff() ? 0.f : mn * p.scale_log2;
    const float corr = __builtin_amdgcn_exp2f(__builtin_fmaf(m, p.scale_log2, -ref));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s8[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s8[i], p.scale_log2, -ref));
      sum += s8[i];
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    l = l * corr + sum;
    m = mn;
    u32x4 pf;
#pragma unroll
    for (int i = 0; i < 4; ++i) pf[i] = pack2<E>(s8[2 * i], s8[2 * i + 1]);
    const auto value = [&](int c, int i) {
      return __builtin_amdgcn_perm(vf[2 * i + 1][c >> 3][(c >> 1) & 3], vf[2 * i][c >> 3][(c >> 1) & 3],
                                   c & 1 ? 0x07060302u : 0x05040100u);
    };
#pragma unroll
    for (int c = 0; c < NC; ++c) o[c] *= corr;
    if (j0 + 32 <= least) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        u32x4 a;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = value(c, i);
        o[c] = E::mfma16(a, pf, o[c]);
      }
    } else {
      // Some row masks some of these keys: its weights there are 0, but 0 times an infinite or NaN value is not.  A column of the
      // product depends on no other column, so each token's columns take the product with the values past its own keys
      // as zeros.
      for (int token = tok0; token <= tok1; ++token) {
        const int seen = visible_keys(w.keys, w.tokens, token, causal);
        uint32_t keep[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = j0 + 16 * (i >> 1) + 4 * kq + 2 * (i & 1);
          keep[i] = (key < seen ? 0xFFFFu : 0u) | (key + 1 < seen ? 0xFFFF0000u : 0u);
        }
        const bool mine = tok == token;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          u32x4 a;
#pragma unroll
          for (int i = 0; i < 4; ++i) a[i] = value(c, i) & keep[i];
          const f32x4 t = E::mfma16(a, pf, o[c]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][e] = mine ? t[e] : o[c][e];
        }
      }
    }
  }
  // merge the four waves: each scales its sums to the workgroup's maximum (a wave without keys has sums of 0, not only a
  // maximum of -inf: with scores that are all NaN its sums are NaN and stay in)
  if (kq == 0) {
    mx[wave][lr] = m;
    ls[wave][lr] = l;
  }
  __syncthreads();
  const auto factor = [&](float mw, float M) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(mw, p.scale_log2, M == -__builtin_inff() ? 0.f : -M * p.scale_log2));
  };
  const float M = fmaxf(fmaxf(mx[0][lr], mx[1][lr]), fmaxf(mx[2][lr], mx[3][lr]));
  const float f = factor(m, M);
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int c = 0; c < NC; c += 4)
      *reinterpret_cast<f32x4*>(&osum[wave][lr][NC * (4 * kq + e) + c]) =
          f32x4{o[c][e] * f, o[c + 1][e] * f, o[c + 2][e] * f, o[c + 3][e] * f};
  __syncthreads();
  const int64_t held = (static_cast<int64_t>(w.partial + w.chunk) * p.kv + kvh) * 16;
  for (int i = tid; i < nrows * (D / 4); i += 256) {
    const int row = i / (D / 4), c = i % (D / 4) * 4;
    f32x4 v = *reinterpret_cast<const f32x4*>(&osum[0][row][c]);
#pragma unroll
    for (int x = 1; x < 4; ++x) v += *reinterpret_cast<const f32x4*>(&osum[x][row][c]);
    const float Mr = fmaxf(fmaxf(mx[0][row], mx[1][row]), fmaxf(mx[2][row], mx[3][row]));
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) sum += ls[x][row] * factor(mx[x][row], Mr);
    const int rr = w.tile * 16 + row, tk = rr / p.group, hd = kvh * p.group + rr - tk * p.group;
    const int64_t out = static_cast<int64_t>(w.start + tk) * p.heads + hd;
    if (w.partial >= 0) {
      *reinterpret_cast<f32x4*>(p.part + (held + row) * D + c) = v;
      if (c == 0) {
        p.ml[held + row] = make_float2(Mr, sum);
        if (w.chunk == 0) p.info[out] = make_int2(static_cast<int>(held) + row, w.chunks);
      }
    } else {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
      *reinterpret_cast<uint2*>(p.out + out * D + c) =
          make_uint2(pack2<E>(v[0] * inv, v[1] * inv), pack2<E>(v[2] * inv, v[3] * inv));
      if (c == 0 && w.chunk == 0) p.info[out] = make_int2(0, 0);
    }
  }
}

// ------------------------------------------------------------------ 128 rows, four waves of 32
// For blocks of many rows.  A workgroup takes 64 keys at a time through LDS, two stages of keys and values, loaded straight into
// it a step ahead; wave w has rows 32 w to 32 w + 31 for all of them.  Scores transposed again: lane l holds query row l & 31 and
// keys 8 (e / 4) + 4 (l >> 5) + e % 4 of a 32-key block (e: element of the 32x32 result), whose elements 8 s to 8 s + 7 are, as a
// reduction's octet l >> 5, the B operand of O^T = V^T P^T for keys 16 s of the block.  So a probability never leaves its lane.  V^T's
// operand needs eight keys of a dim: two transposing LDS reads of four keys each.
// The rows' running maximum is a reference that moves only when a score exceeds it by 8 (weights reach 2^8, their relative precision
// is the same): the accumulators are rescaled a few times a row instead of at every step.
// A run of n matrix instructions that take one operand each from LDS: use(i, read(i)) for all i, each read kAhead instructions ahead of
// its use.  Left to itself the compiler puts each read right before its use and waits for it (a read takes four times as long as
// the instruction), so the order is fixed.
template <int n, int kAhead, class Read, class Use>
__device__ __forceinline__ void feed(const Read& read, const Use& use) {
  u32x4 f[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) f[i] = read(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < n; ++i) {
    const u32x4 now = f[i % kAhead];
    use(i, now);
    if (i + kAhead < n) f[i % kAhead] = read(i + kAhead);
    __builtin_amdgcn_sched_barrier(0);
  }
}
// Four keys of one dim a lane: lane j of 16 gives the place of row j / 4, dims 4 (j % 4) on, and gets dim j of the four rows.
__device__ __forceinline__ uint2 read_turned(const char* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p)));
}
// 16 bytes a lane from global memory to 1 KB of LDS, lane by lane.
__device__ __forceinline__ void copy_to_lds(const char* src, char* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16,
                                   0, 0);
}
constexpr int kLargeRows = 128, kLargeUnit = 64, kLargeLeast = 4;
template <int D, class E, bool kPrefix>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_large_kernel(PagedParams p) {
  constexpr int KS = D / 16, NC = D / 32, SL = D / 8, KR = 256 / SL, KP = 64 / KR;
  constexpr int kStage = 64 * D * 2;  // bytes of a stage of keys or values
  constexpr int kAhead = D == 256 ? 4 : 3;
  __shared__ __align__(16) char lds[4 * kStage];  // keys of both stages, then values
  __shared__ int odd;  // a stage lacks values that are infinite or NaN
  const int kvh = blockIdx.x % p.kv;
  Share w;
  if (!(kPrefix ? prefix_share(p, blockIdx.x / p.kv, kLargeRows, kLargeUnit, kLargeLeast, &w)
                : own_share(p, blockIdx.x / p.kv, kLargeRows, kLargeUnit, kLargeLeast, &w)))
    return;
  const PagedSide& side = kPrefix ? p.prefix : p.own;
  const bool causal = !kPrefix && p.causal;
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, l31 = lane & 31, half = lane >> 5;
  const int rows = w.tokens * p.group, nrows = min(kLargeRows, rows - w.tile * kLargeRows);
  const int row0 = w.tile * kLargeRows;
  const int r = row0 + min(wave * 32 + l31, nrows - 1);
  const int tok = r / p.group, head = kvh * p.group + r - tok * p.group;
  const int visible = visible_keys(w.keys, w.tokens, tok, causal);
  const int least = visible_keys(w.keys, w.tokens, uniform(row0 / p.group), causal);
  const int n = visible_keys(w.keys, w.tokens, uniform((row0 + nrows - 1) / p.group), causal);
  const int k0 = w.chunk * w.c * kLargeUnit, k1 = min(k0 + w.c * kLargeUnit, n);
  const int steps = k1 > k0 ? (k1 - k0 + 63) / 64 : 0;

  u32x4 q[KS];
  {
    const uint16_t* qr = p.query + (w.start + tok) * p.query_token + head * p.query_head + 8 * half;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      q[s] = *reinterpret_cast<const u32x4*>(qr + 16 * s);
      // at head dim 256 the queries stay in the accumulation registers, where matrix instructions take them from
      if constexpr (D == 256) asm volatile("" : "+a"(q[s]));
    }
  }
  if (tid == 0) odd = 0;

  // Staging: thread tid loads 16-byte slot tid % SL of rows tid / SL, + KR, ... of keys and values.  A 16-row group's place is a 64-bit
  // offset that is found a step ahead, group g of the step in lane g; rows inside it are 32-bit offsets that do not change.
  // LDS: slot c of row r holds 16-byte piece c ^ (r % 16) of the keys, c ^ 4 (r % 8 or 4) of the values, so that neither kind of read
  // puts two of the lanes that read together on one bank; the loads permute the pieces, since their own order in LDS is fixed.
  const char* keys = reinterpret_cast<const char*>(side.keys + kvh * side.key_head);
  const char* vals = reinterpret_cast<const char*>(side.values + kvh * side.value_head);
  const int krow = static_cast<int>(2 * side.key_row), vrow = static_cast<int>(2 * side.value_row);  // bytes
  const int slot = tid % SL, tr = tid / SL;
  const uint32_t vcol = (slot ^ (tr & (D == 256 ? 7 : 3)) << 2) * 16;
  const auto kcol = [&](int i) { return static_cast<uint32_t>((slot ^ ((tr + i * KR) & 15)) * 16); };
  uint32_t koff[KP / 4], voff[KP / 4];
#pragma unroll
  for (int i = 0; i < KP / 4; ++i) {
    koff[i] = (tr + i * KR) * krow + kcol(i);
    voff[i] = (tr + i * KR) * vrow + vcol;
  }
  PageAt place = {0, 0}, ahead = {0, 0};  // of group lane % 4 of the step whose values, and whose keys, are loaded next
  const auto find = [&](int key0) {
    place = ahead;
    ahead = page_at(side, w.table, min(key0 / 16 + (lane & 3), (n - 1) / 16));
  };
  const auto load = [&](bool values, const PageAt& at, int stage, int key0) {
    const int stride = values ? vrow : krow;
    const int64_t offset = at.page * (2 * (values ? side.value_page : side.key_page)) + static_cast<int64_t>(at.row) * stride;
    char* to = lds + (stage + (values ? 2 : 0)) * kStage + wave * 1024;
    const bool tail = key0 + 64 > n;  // rows past the last key repeat it
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const int g = i / (KP / 4);
      const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(offset), g);
      const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(static_cast<uint64_t>(offset) >> 32), g);
      const char* base = (values ? vals : keys) + static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
      uint32_t off = values ? voff[i % (KP / 4)] : koff[i % (KP / 4)];
      if (tail)
        off = min((i * KR + tr) & 15, n - 1 - 16 * min(key0 / 16 + i * KR / 16, (n - 1) / 16)) * stride + (values ? vcol : kcol(i));
      copy_to_lds(base + off, to + i * 4096);
    }
  };
  // Some row masks some of a step's keys: its weights there are 0, but 0 times an infinite or NaN value is not.  Such values, and keys
  // past the last one, become zeros in the stage.
  const auto clean = [&](int stage, int key0) {
    bool wild = false;
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      u32x4* at = reinterpret_cast<u32x4*>(lds + (2 + stage) * kStage + i * 4096 + tid * 16);
      u32x4 v = *at;
      const bool in = key0 + i * KR + tr < n;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t x = in ? v[k] : 0, high = E::kExponent << 16;
        const bool a = (x & E::kExponent) == E::kExponent, b = (x & high) == high;
        wild |= a || b;
        v[k] = x & (a ? 0xFFFF0000u : ~0u) & (b ? 0xFFFFu : ~0u);
      }
      *at = v;
    }
    if (wild) odd = 1;
    lds_barrier();
  };
  uint32_t kr = l31 * (2 * D) + ((half ^ l31) & 15) * 16;
  const int j15 = lane & 15, turn = D == 256 ? 4 * half + (j15 >> 2) : j15 >> 2;
  uint32_t vr = 2 * kStage + (4 * half + (j15 >> 2)) * (2 * D) + (2 * (lane >> 4 & 1) + (j15 >> 1 & 1)) * 16 + (j15 & 1) * 8 + turn * 64;

  f32x16 o[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[c][e] = 0.f;
  float m = -__builtin_inff(), l = 0.f;  // reference of the row's weights, and the sum of this lane's weights

  // Step i multiplies its weights with its values, and before that the next step's keys with the queries: the exponentials of the one
  // stand between the matrix instructions of the other, and the maximum of the next scores between those of the values.  So keys are
  // loaded two steps ahead, values one.
  const auto fill = [&](int i) {  // what step i loads
    if (i + 1 < steps) load(true, place, ~i & 1, k0 + 64 * (i + 1));
    if (i + 2 < steps) load(false, ahead, i & 1, k0 + 64 * (i + 2));
    find(k0 + 64 * (i + 3));
  };
  const auto arrive = [&]() {
    wait_vmem();
    lds_barrier();
  };
  if (steps > 0) {
    find(k0);
    load(false, ahead, 0, k0);
    load(true, ahead, 0, k0);
    find(k0 + 64);
    if (steps > 1) load(false, ahead, 1, k0 + 64);
    find(k0 + 128);
  }
  arrive();
  if (wave * 32 >= nrows) {  // no rows: the wave only stages
    if (steps > 2) lds_barrier();
    for (int i = 0; i < steps; ++i) {
      fill(i);
      if (k0 + 64 * (i + 1) > least) clean(i & 1, k0 + 64 * i);
      arrive();
    }
    return;
  }
  f32x16 sc[2][2];  // scores of even and odd steps, 32 keys each
  const auto clear = [&](f32x16 (&t)[2]) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) t[b][e] = 0.f;
  };
  const auto hide = [&](f32x16 (&t)[2], int key0) {
    if (key0 + 64 <= least) return;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (key0 + 32 * b + 8 * (e >> 2) + 4 * half + (e & 3) >= visible) t[b][e] = -__builtin_inff();
  };
  const auto key_at = [&](int stage, int i) {
    return *reinterpret_cast<const u32x4*>(lds + ((kr ^ (32 * (i >> 1))) + (stage * kStage + (i & 1) * 64 * D)));
  };
  float mc = -__builtin_inff();  // maximum of the scores of the step to come
  if (steps > 0) {
    clear(sc[0]);
    feed<2 * KS, kAhead>([&](int i) { return key_at(0, i); },
                         [&](int i, u32x4 k) { sc[0][i & 1] = E::mfma32(k, q[i >> 1], sc[0][i & 1]); });
    hide(sc[0], k0);
#pragma unroll
    for (int e = 0; e < 32; ++e) mc = fmaxf(mc, sc[0][e >> 4][e & 15]);
    if (steps > 2) lds_barrier();  // step 0 loads step 2's keys where these were
  }
  const auto step = [&](auto stage_, auto last_, int i) {
    constexpr int stage = decltype(stage_)::value;
    constexpr bool more = !decltype(last_)::value;
    const int key0 = k0 + 64 * i;
    f32x16(&now)[2] = sc[stage];
    f32x16(&next)[2] = sc[stage ^ 1];
    fill(i);
    if (key0 + 64 > least) clean(stage, key0);
    if constexpr (D == 256) asm volatile("" : "+v"(kr), "+v"(vr));  // no two dozen registers of places kept over the steps
    mc = fmaxf(mc, __shfl_xor(mc, 32, 64));
    // a row that has seen no key keeps weights of 0 (the exponent is -inf); a NaN score, which the maximum skips, makes l and
    // o NaN, and so they stay
    const bool move = (mc - m) * p.scale_log2 > 8.f || (m == -__builtin_inff() && mc > m);
    if (__any(move)) {
      const float to = move ? mc : m;
      const float corr = __builtin_amdgcn_exp2f(__builtin_fmaf(m, p.scale_log2, to == -__builtin_inff() ? 0.f : -to * p.scale_log2));
      l *= move ? corr : 1.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[c][e] *= move ? corr : 1.f;
      m = to;
    }
    const float ref = m == -__builtin_inff() ? 0.f : m * p.scale_log2;
    u32x4 pf[4];
    float sum[2] = {0.f, 0.f};
    const auto weigh = [&](int e) {  // elements e and e + 1 of the step's 32
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(now[e >> 4][e & 15], p.scale_log2, -ref));
      const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(now[e >> 4][(e & 15) + 1], p.scale_log2, -ref));
      sum[0] += x;
      sum[1] += y;
      uint32_t both = pack2<E>(x, y);
      asm volatile("" : "+v"(both));  // made here, between the matrix instructions, not where it is used
      pf[e >> 3][(e & 7) >> 1] = both;
    };
    if constexpr (more) {
      clear(next);
      constexpr int kEach = KS / 8;  // instructions a pair of elements
      feed<2 * KS, kAhead>([&](int k) { return key_at(stage ^ 1, k); },
                           [&](int k, u32x4 v) {
                             next[k & 1] = E::mfma32(v, q[k >> 1], next[k & 1]);
                             if (k % kEach == 0) weigh(k / kEach * 2);
                           });
      hide(next, key0 + 64);
    } else {
#pragma unroll
      for (int e = 0; e < 32; e += 2) weigh(e);
    }
    l += sum[0] + sum[1];
    mc = -__builtin_inff();
    feed<4 * NC, kAhead>(
        [&](int k) {
          const char* at = lds + ((vr ^ (64 * (k % NC))) + (stage * kStage + k / NC * 32 * D));
          const uint2 a = read_turned(at), b = read_turned(at + 16 * D);
          return u32x4{a.x, a.y, b.x, b.y};
        },
        [&](int k, u32x4 v) {
          o[k % NC] = E::mfma32(v, pf[k / NC], o[k % NC]);
          constexpr int kEach = NC / 4;  // instructions a pair of elements of the next scores
          if (more && k % kEach == 0) {
            const int e = k / kEach * 2;
            mc = fmaxf(fmaxf(mc, next[e >> 4][e & 15]), next[e >> 4][(e & 15) + 1]);
          }
        });
    arrive();
  };
  if (steps > 0) {
    const std::integral_constant<int, 0> even{};
    const std::integral_constant<int, 1> uneven{};
    int i = 0;
    for (; i + 2 < steps; i += 2) {
      step(even, std::false_type{}, i);
      step(uneven, std::false_type{}, i + 1);
    }
    if (i + 1 < steps) {
      step(even, std::false_type{}, i);
      step(uneven, std::true_type{}, i + 1);
    } else {
      step(even, std::true_type{}, i);
    }
  }
  if (steps > 0 && odd) {
    // the values left out of the stages: infinite or NaN in the rows that see them, whatever their (positive) weight
    for (int key = k0 + max(0, (least - k0) / 64) * 64; key < k1; ++key) {
      const PageAt at = page_at(side, w.table, key / 16);
      const char* src = vals + 2 * at.page * side.value_page + static_cast<int64_t>(at.row + key % 16) * vrow;
      if (key >= visible) continue;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const uint2 v = *reinterpret_cast<const uint2*>(src + 2 * (32 * c + 2 * e + 4 * half));
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t x = (y < 2 ? v.x : v.y) >> (16 * (y & 1)) & 0xFFFF;
            if ((x & E::kExponent) == E::kExponent) o[c][e + y] += E::to_f32(x);
          }
        }
    }
  }

  l += __shfl_xor(l, 32, 64);
  if (wave * 32 + l31 >= nrows) return;
  const int64_t out = static_cast<int64_t>(w.start + tok) * p.heads + head;
  if (w.partial >= 0) {
    const int64_t held = (static_cast<int64_t>(w.partial + w.chunk) * p.kv + kvh) * kLargeRows + wave * 32 + l31;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4*>(p.part + held * D + 32 * c + 2 * e + 4 * half) = f32x4{o[c][e], o[c][e + 1], o[c][e + 2], o[c][e + 3]};
    if (half == 0) {
      p.ml[held] = make_float2(m, l);
      if (w.chunk == 0) p.info[out] = make_int2(static_cast<int>(held), w.chunks);
    }
  } else {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<uint2*>(p.out + out * D + 32 * c + 2 * e + 4 * half) =
            make_uint2(pack2<E>(o[c][e] * inv, o[c][e + 1] * inv), pack2<E>(o[c][e + 2] * inv, o[c][e + 3] * inv));
    if (half == 0 && w.chunk == 0) p.info[out] = make_int2(0, 0);
  }
}

// ------------------------------------------------------------------ merge
// kWaves waves per (token, head), D / 64 dims a lane; wave w takes the row's partial results w, w + kWaves, ...: first every maximum
// and sum, a partial a lane, then their rows, several in flight.  The order of the additions depends on the sizes alone.
template <int D, class E, int kWaves>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedParams p) {
  constexpr int F = D / 64, kFlight = 8, kRows = 4 / kWaves;
  __shared__ float om[4][D], lm[4];
  __shared__ float mm[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, part = wave % kWaves;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + wave / kWaves;
  const int t = static_cast<int>(row / p.heads);
  // rows of tokens in no sequence are not written (with one row a workgroup and several waves this holds for all of them)
  const bool covered = t < p.T && t >= p.starts[0] && t < p.starts[p.B];
  int2 range[2] = {make_int2(0, 0), make_int2(0, 0)};
  if (covered) {
    range[0] = p.info[row];
    if (p.merge_prefix) range[1] = p.prefix_info[row];
  }
  const bool any = covered && range[0].y > 0;
  if (kWaves == 1 && !any) return;
  if (kWaves > 1 && !any) return;  // the same for all waves: they share the row
  float M = -__builtin_inff();
  const int tile[2] = {p.own_tile_rows, p.prefix_tile_rows};
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    // whatever the sequences' starts held, nothing outside the partial results is read
    const int64_t last = range[g].x + static_cast<int64_t>(range[g].y - 1) * tile[g] * p.kv;
    if (range[g].x < 0 || range[g].y < 0 || last >= p.part_rows[g]) range[g].y = 0;
    const float2* ml = g ? p.prefix_ml : p.ml;
    for (int i = part + kWaves * lane; i < range[g].y; i += 64 * kWaves)
      M = fmaxf(M, ml[range[g].x + static_cast<int64_t>(i) * tile[g] * p.kv].x);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  const float ref = M == -__builtin_inff() ? 0.f : M * p.scale_log2;
  float l = 0.f, acc[F];
#pragma unroll
  for (int i = 0; i < F; ++i) acc[i] = 0.f;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float2* ml = g ? p.prefix_ml : p.ml;
    const float* rows = (g ? p.prefix_part : p.part) + lane * F;
    const int64_t step = static_cast<int64_t>(tile[g]) * p.kv * kWaves;
    const int64_t base = range[g].x + static_cast<int64_t>(part) * tile[g] * p.kv;
    const int count = (range[g].y - part + kWaves - 1) / kWaves;
    for (int i0 = 0; i0 < count; i0 += kFlight) {
      float x[kFlight][F];
      float2 v[kFlight];
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        const int64_t at = base + min(i0 + i, count - 1) * step;
        v[i] = ml[at];
#pragma unroll
        for (int f = 0; f < F; ++f) x[i][f] = rows[at * D + f];
      }
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        if (i0 + i >= count || v[i].y == 0.f) continue;  // no key of this row in that chunk
        const float f = __builtin_amdgcn_exp2f(__builtin_fmaf(v[i].x, p.scale_log2, -ref));
        l += v[i].y * f;
#pragma unroll
        for (int k = 0; k < F; ++k) acc[k] += x[i][k] * f;
      }
    }
  }
  if (kWaves > 1) {
    if (lane == 0) {
      lm[wave] = l;
      mm[wave] = M;
    }
#pragma unroll
    for (int k = 0; k < F; ++k) om[wave][lane * F + k] = acc[k];
    __syncthreads();
    if (wave) return;
    M = fmaxf(fmaxf(mm[0], mm[1]), fmaxf(mm[2], mm[3]));
    const float all = M == -__builtin_inff() ? 0.f : M * p.scale_log2;
    l = 0.f;
#pragma unroll
    for (int k = 0; k < F; ++k) acc[k] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(__builtin_fmaf(mm[w], p.scale_log2, -all));
      l += lm[w] * f;
#pragma unroll
      for (int k = 0; k < F; ++k) acc[k] += om[w][lane * F + k] * f;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint32_t* out = reinterpret_cast<uint32_t*>(p.out + row * D + lane * F);
#pragma unroll
  for (int k = 0; k < F; k += 2) out[k / 2] = pack2<E>(acc[k] * inv, acc[k + 1] * inv);
}

}  // namespace

// Rows of a stage's tiles, by the rows a sequence has on average: up to 32 take the kernel of 16 rows, whose waves share the
// keys out; more take the one of 128, whose waves share the keys' way through LDS.
int paged_tile_rows(int64_t tokens, int64_t sequences, int64_t group) {
  const int64_t blocks = std::max<int64_t>(1, std::min(tokens, sequences));
  return tokens * group > 32 * blocks ? kLargeRows : kSmallRows;
}
// Workgroups that a stage's work is cut for: as many as run at once.
int paged_slots(int tile_rows, int head_dim, int cus) { return tile_rows == kLargeRows && head_dim == 256 ? cus : 2 * cus; }

template <int D, class E>
static void launch_append(const AppendParams& p, hipStream_t stream) {
  // a token's heads over several workgroups while there are few tokens: each makes the token's angles itself
  constexpr int kHeads = 256 / (D / 8);
  const int all = (p.heads + 2 * p.kv + kHeads - 1) / kHeads;
  hipLaunchKernelGGL((paged_append_kernel<D, E>), dim3(p.T, p.T <= 256 ? all : 1), dim3(256), 0, stream, p);
}
void launch_paged_append(int head_dim, bool bf16, const AppendParams& p, hipStream_t stream) {
  if (head_dim == 256) bf16 ? launch_append<256, Bf16>(p, stream) : launch_append<256, Fp16>(p, stream);
  else bf16 ? launch_append<128, Bf16>(p, stream) : launch_append<128, Fp16>(p, stream);
}

template <int D, class E, bool kPrefix>
static void launch_stage(const PagedParams& p, int tile_rows, int64_t tiles, hipStream_t stream) {
  const dim3 grid(max_chunks(tiles, p.kv, p.slots) * p.kv);
  if (tile_rows == kLargeRows) hipLaunchKernelGGL((paged_large_kernel<D, E, kPrefix>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((paged_small_kernel<D, E, kPrefix>), grid, dim3(256), 0, stream, p);
}
template <int D, class E>
static void launch_attend(const PagedParams& p, const PagedParams& before, hipStream_t stream) {
  const int own = p.own_tile_rows, front = p.prefix_tile_rows;
  if (p.merge_prefix) launch_stage<D, E, true>(before, front, seq_tiles(p.T, p.group, front), stream);
  launch_stage<D, E, false>(p, own, max_tiles(p.T, p.B, p.group, own), stream);
  const int least = own == kLargeRows ? kLargeUnit * kLargeLeast : kSmallUnit;
  if (!p.merge_prefix && p.own.capacity <= least) return;  // one chunk a tile: nothing to merge
  const int64_t rows = static_cast<int64_t>(p.T) * p.heads;
  // few rows may be in many chunks: four waves a row
  if (rows <= 4096) hipLaunchKernelGGL((paged_merge_kernel<D, E, 4>), dim3(rows), dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((paged_merge_kernel<D, E, 1>), dim3((rows + 3) / 4), dim3(256), 0, stream, p);
}
void launch_paged_attention(int head_dim, bool bf16, const PagedParams& p, const PagedParams& before, hipStream_t stream) {
  if (head_dim == 256) bf16 ? launch_attend<256, Bf16>(p, before, stream) : launch_attend<256, Fp16>(p, before, stream);
  else bf16 ? launch_attend<128, Bf16>(p, before, stream) : launch_attend<128, Fp16>(p, before, stream);
}

}  // namespace dflash
