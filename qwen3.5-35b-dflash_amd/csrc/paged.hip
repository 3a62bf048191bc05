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
// A probability takes part in the product with V as two 16-bit parts, its rounding and the rounding of what that leaves: off by 2^-16 of
// itself in bf16, 2^-22 in fp16, so that what an output is off by is its own rounding (1.66e-3 of the norm in bf16, 2.0e-4 in fp16, for
// values from N(0, 1)).  With one part it would be 2.0e-3 to 2.3e-3 and 2.6e-4; the second costs matrix instructions, a third of those of
// the 128-row kernel: 322 instead of 237 us for its largest case below, 124 instead of 121 for decode of 64 sequences.
//
// The reference.  A probability is held as 2^(t_j - r), t_j = s_j log2 e in fp32, with a reference r of its row; partial results keep the
// r that their l and o belong to, and merge by it whatever it is.  Both roundings of t_j - r are those of one product and one difference,
// so that the largest score keeps the largest weight at any magnitude: with an fma the rounding of the row's maximum, which is more
// than a binade from 2^24 on, would be part of every weight.  In bf16, which has the range of fp32, r is a maximum.
// fp16 has its precision from 2^-14 to 2^16 only.  There r is lower, so that the largest weight is 2^kSmallBias or 2^kLargeBias and at
// most 2^15.9, and it follows the keys down as well as up: where all of a step's keys weigh less than 2^-kFall of the reference's, as
// those behind one key that takes nearly all of the softmax do, r falls to what their maximum asks for, and l and o, which have
// the range of fp32, are scaled up to it (at most kReach below the highest so far: with weights of 2^16, values of 2^16 and 2^30 keys
// the sums stay under 2^102).  So a weight is off by 2^-28 of the largest of the same 32 or 64 keys at most, and has 11 bits
// or more from 2^-17 of that one on.
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
  static constexpr bool kNarrow = false;         // the reference of weights never falls
  static constexpr int kRise = 8;                // 128-row kernel: how far scores may exceed the reference
  static constexpr int kSmallBias = 0, kLargeBias = 0;
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
  static constexpr bool kNarrow = true;
  static constexpr int kRise = 4;
  static constexpr int kSmallBias = 15, kLargeBias = 15 - kRise;
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

// What pack2 leaves of a and b, in 16 bits.
template <class E>
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t both) {
  return pack2<E>(a - E::to_f32(both & 0xFFFF), b - E::to_f32(both >> 16));
}

constexpr float kFall = 8.f, kReach = 40.f;
// A score in units of log2: a product of its own, never fused with the difference that follows.
__device__ __forceinline__ float scaled(float score, float scale_log2) {
#pragma clang fp contract(off)
  return score * scale_log2;
}
// The reference whose largest weight is about 2^bias: t - bias, or t where that would round to less than t - (bias + 0.9).
template <int bias>
__device__ __forceinline__ float reference_of(float t) {
  if constexpr (bias == 0) return t;
  const float r = t - bias;
  return t - r < bias + 0.9f ? r : t;
}
// The number that is subtracted: a row that has seen no key keeps weights of 0 (the exponent is -inf).
__device__ __forceinline__ float reference(float m) { return m == -__builtin_inff() ? 0.f : m; }

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
// Bound: memory, behind it the angles' latency, which the first heads' loads cover: 15005 tokens of 48 rows at head dim 128, 218 MB,
// 52.5 us (4.15 TB/s; a copy of 1 GB 5.16); few tokens: the launch and the chain starts - table - store, 5.1 us for one.
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
  // of the length as it stands, not the most that the table holds: rows past that have no page
  const int64_t row = static_cast<int64_t>(p.side.lengths[b]) - s.tokens + t - s.start;
  const int all = p.heads + 2 * p.kv, c = (tid % L) * 8, step = gridDim.y * kHeads;
  const auto read = [&](int j) {
    const bool is_q = j < p.heads, is_v = j >= p.heads + p.kv;
    const int h = is_q ? j : is_v ? j - p.heads - p.kv : j - p.heads;
    const uint16_t* src = is_q ? p.query + t * p.query_token + h * p.query_head
                        : is_v ? p.value + t * p.value_token + h * p.value_head
                               : p.key + t * p.key_token + h * p.key_head;
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + c));  // read once
  };
  // the first heads are on their way while the angles are made, the next while heads are turned
  int j = blockIdx.y * kHeads + tid / L;
  u32x4 next{0, 0, 0, 0};
  if (j < all) next = read(j);
  int page = -1, inside = 0;  // where the token's rows go; -1: nowhere
  if (row >= 0 && row < p.side.capacity) {
    const int i = divide(static_cast<uint32_t>(row) >> 4, p.side.groups_per_page);
    page = p.side.table[b * p.side.table_stride + i];
    inside = static_cast<int>(row) - i * p.side.page_groups * 16;
    if (page >= p.side.pages) page = -1;
  }
  if (p.half) {
    const int64_t position = p.positions ? p.positions[t] : row;
    for (int i = tid; i < p.half; i += 256) {
      const double a = static_cast<double>(position) * static_cast<double>(p.inv_freq[i]);
      const double turns = rint(a * 0.15915494309189535);
      const float r = static_cast<float>(fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, a)));
      cs[i] = cosf(r);
      sn[i] = sinf(r);
    }
  }
  __syncthreads();
  for (; j < all; j += step) {
    const bool is_q = j < p.heads, is_v = j >= p.heads + p.kv;
    const int h = is_q ? j : is_v ? j - p.heads - p.kv : j - p.heads;
    const u32x4 raw = next;
    if (j + step < all) next = read(j + step);
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
    } else if (page >= 0) {
      uint16_t* dst = is_v ? p.values + page * p.side.value_page + h * p.side.value_head + inside * p.side.value_row
                           : p.keys + page * p.side.key_page + h * p.side.key_head + inside * p.side.key_row;
      *reinterpret_cast<u32x4*>(dst + c) = out;
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

// Sum of a wave's 64 values and inclusive sums over its lanes, on the lanes' own data paths (a shuffle through LDS takes ten
// times as long, and the search below is part of every workgroup's start).
template <int kCtrl>
__device__ __forceinline__ int shifted(int v) {
  return __builtin_amdgcn_update_dpp(0, v, kCtrl, 0xF, 0xF, true);
}
__device__ __forceinline__ int wave_scan(int v) {
  v += shifted<0x111>(v);  // row_shr:1, within 16 lanes
  v += shifted<0x112>(v);
  v += shifted<0x114>(v);
  v += shifted<0x118>(v);
  const int a = __builtin_amdgcn_readlane(v, 15), b = __builtin_amdgcn_readlane(v, 31), c = __builtin_amdgcn_readlane(v, 47);
  const int row = (threadIdx.x >> 4) & 3;
  return v + (row > 0 ? a : 0) + (row > 1 ? b : 0) + (row > 2 ? c : 0);
}

// Row tiles of all sequences, and the (tile, unit of keys) pairs; `last` keeps what the lane found of the last 64 sequences.
struct Work {
  int tiles;
  double units;
};
__device__ __forceinline__ Work own_work(const PagedParams& p, int tile_rows, int unit, SeqSpan* last) {
  const int lane = threadIdx.x & 63;
  int tiles = 0;
  uint64_t units = 0;
#pragma unroll 4
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    *last = SeqSpan{0, 0, 0};
    if (b0 + lane < p.B) *last = load_span(p, b0 + lane);
    const int t = seq_tiles(last->tokens, p.group, tile_rows);
    tiles += t;
    units += static_cast<uint64_t>(t) * seq_units(last->keys, unit);
  }
  // in two parts whose sums stay in 31 bits
  const int lo = wave_scan(static_cast<int>(units & 0xFFFFFF)), hi = wave_scan(static_cast<int>(units >> 24));
  return Work{__builtin_amdgcn_readlane(wave_scan(tiles), 63),
              __builtin_amdgcn_readlane(hi, 63) * 16777216.0 + __builtin_amdgcn_readlane(lo, 63)};
}
// The prefix as a sequence whose block is the whole batch.
__device__ __forceinline__ Work front_work(const PagedParams& p, int tile_rows, int unit, int* keys) {
  *keys = uniform(clampi(p.prefix.lengths[0], 0, p.prefix.capacity));
  const int tiles = seq_tiles(p.T, p.group, tile_rows);
  return Work{tiles, static_cast<double>(static_cast<int64_t>(tiles) * seq_units(*keys, unit))};
}

// Share `id` of the sequences' own keys in chunks of c units: every wave finds it by itself, 64 sequences at a time, one a lane.
// `s`: what own_work left.  A sequence's last tiles come first: where the block's tokens mask what follows them, later tiles have more
// keys, and the longest should not start last.  (All sequences' tiles in one order by their place: 1% faster with prompts of 442 to
// 2222 tokens, not kept.)
__device__ __forceinline__ bool own_share(const PagedParams& p, int id, int tile_rows, int unit, int c, SeqSpan s, Share* out) {
  const int lane = threadIdx.x & 63;
  int first = 0, held = 0;  // shares of the sequences before; partial tiles of those that this lane had
  const auto at = [&](int b) { return b < p.B ? load_span(p, b) : SeqSpan{0, 0, 0}; };
  SeqSpan next = s;
  if (p.B > 64) next = at(lane);
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    s = next;
    if (b0 + 64 < p.B) next = at(b0 + 64 + lane);
    const int k = tile_chunks(seq_units(s.keys, unit), c), n = seq_tiles(s.tokens, p.group, tile_rows) * k;
    const int kept = k > 1 || p.merge_prefix ? n : 0;
    const int sum = wave_scan(n);
    const uint64_t m = __ballot(n > 0 && id < first + sum);
    if (m) {
      const int l = __builtin_ctzll(m);
      const int rest = id - (first + __builtin_amdgcn_readlane(sum - n, l));
      const int chunks = __builtin_amdgcn_readlane(k, l);
      const uint32_t tiles = __builtin_amdgcn_readlane(n, l) / static_cast<uint32_t>(chunks);
      const uint32_t before = static_cast<uint32_t>(rest) / static_cast<uint32_t>(chunks);
      const int chunk = rest - before * chunks;
      const int partial = __builtin_amdgcn_readlane(wave_scan(held + (lane < l ? kept : 0)), 63);
      out->start = __builtin_amdgcn_readlane(s.start, l);
      out->tokens = __builtin_amdgcn_readlane(s.tokens, l);
      out->keys = __builtin_amdgcn_readlane(s.keys, l);
      out->tile = uniform(static_cast<int>(tiles - 1 - before));
      out->chunk = uniform(chunk);
      out->chunks = chunks;
      out->partial = chunks > 1 || p.merge_prefix
                         ? uniform(partial + out->tile * chunks) : -1;
      out->c = c;
      out->table = p.own.table + static_cast<int64_t>(b0 + l) * p.own.table_stride;
      // blocks that overlap (starts that are no such thing) may have more tiles than there is room for
      return out->partial < 0 || static_cast<int64_t>(out->partial + chunk + 1) * p.kv * tile_rows <= p.part_rows[0];
    }
    first += __builtin_amdgcn_readlane(sum, 63);
    held += kept;
  }
  return false;
}

// The thread's number, with nothing that was computed from it before: for what is rarely needed and would else stay in registers.
__device__ __forceinline__ int thread_again() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// 16 bytes a lane from base + off to 1 KB of LDS at the wave's `dst`, lane by lane.  In assembly, so that the compiler does not put a
// wait for every load into LDS before every read of it: what a read needs has arrived at the barrier before (arrive() below).  No
// register is written but m0, which nothing else in this file uses.
__device__ __forceinline__ void copy_to_lds(const char* base, uint32_t off, char* dst) {
  const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(dst)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(off), "s"(base) : "memory");
}
// The same from a place of each lane's own.
__device__ __forceinline__ void copy_to_lds(const uint16_t* from, char* dst) {
  const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(dst)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory");
}

// ------------------------------------------------------------------ 16 rows, four waves over the keys
// For blocks of few rows.  Scores transposed, S^T = K Q^T: lane l holds query row l & 15 and keys 4 (l >> 4) + e of each of two
// 16-key tiles, which, with those eight keys as the reduction's octet l >> 4, is the B operand of O^T = V^T P^T as it stands.  The A
// operand needs eight keys of one dim per lane: a lane loads D / 16 neighbouring dims of its eight keys and pairs halves in
// registers, so V needs no transpose and neither operand passes through LDS.
// Bound: memory.  A wave has a round's 32 keys and values in flight, two workgroups a CU: 64 sequences of up to 8192 keys, 572 MB, 124 us
// (4.6 TB/s).  One workgroup a CU, with the registers of two: 10 us more; streaming loads 12, the rounds' places looked up eight rounds
// ahead 17.  At head dim 256 the queries wait in LDS: in registers 16 of them went through memory in every round, 135 us.  One row behind
// 131072 keys, 268 MB, both kernels: 62.7 us.  Few keys: latency.
constexpr int kSmallRows = 16, kSmallUnit = 128;  // keys a round of the four waves
template <int D>
constexpr int kSmallPitch = D + 4;
template <int D>
constexpr int kSmallArea = 16 * kSmallPitch<D> * 4;  // bytes a wave's sums take
// `areas`: LDS of kSmallArea bytes for each wave.
template <int D, class E>
__device__ __forceinline__ void small_share(const PagedParams& p, const Share& w, bool on_front, int kvh, char* const (&areas)[4], float (&mx)[4][16], float (&ls)[4][16]) {
  constexpr int NC = D / 16, KS = D / 32, VL = NC / 8, kPitch = kSmallPitch<D>;
  const PagedSide& side = on_front ? p.prefix : p.own;
  const bool causal = !on_front && p.causal;
  const int tid = thread_again(), wave = uniform(tid >> 6), lane = tid & 63, lr = lane & 15, kq = lane >> 4;
  const int rows = w.tokens * p.group, nrows = min(16, rows - w.tile * 16);
  const int r = w.tile * 16 + min(lr, nrows - 1);  // this lane's row in its block
  const int tok = divide(r, p.by_group), head = kvh * p.group + r - tok * p.group;
  const int visible = visible_keys(w.keys, w.tokens, tok, causal);
  const int tok0 = uniform(static_cast<int>(divide(w.tile * 16, p.by_group))), tok1 = uniform(static_cast<int>(divide(w.tile * 16 + nrows - 1, p.by_group)));
  const int least = visible_keys(w.keys, w.tokens, tok0, causal);  // keys that every row of the tile sees
  const int n = visible_keys(w.keys, w.tokens, tok1, causal);      // keys that some row sees
  const int k0 = w.chunk * w.c * kSmallUnit, k1 = chunk_end(k0, w.c, kSmallUnit, n);

  // At head dim 256 the queries wait in the wave's area of LDS, which it needs for its sums at the end only.
  constexpr bool kHeld = D == 256;
  char* const area = wave == 0 ? areas[0] : wave == 1 ? areas[1] : wave == 2 ? areas[2] : areas[3];
  u32x4 q[kHeld ? 1 : KS];
  if (!kHeld || k0 + 32 * wave < k1) {  // a wave without keys leaves its area alone
    const uint16_t* qr = p.query + (w.start + tok) * p.query_token + head * p.query_head + 8 * kq;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if constexpr (kHeld) copy_to_lds(qr + 32 * s, area + 1024 * s);
      else q[s] = *reinterpret_cast<const u32x4*>(qr + 32 * s);
    }
  }
  const uint16_t* keys = side.keys + kvh * side.key_head;
  const uint16_t* vals = side.values + kvh * side.value_head;
  f32x4 o[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), l = 0.f, peak = -__builtin_inff();  // the row's reference, sum of weights, highest reference

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
    uint32_t held_at = 16 * lane;
    if constexpr (kHeld) {
      if (j0 < k0 + kSmallUnit) wait_vmem();  // the wave's first round: the queries have arrived
      asm volatile("" : "+v"(held_at)::"memory");
    }
    f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      u32x4 qs;
      if constexpr (kHeld) qs = *reinterpret_cast<const u32x4*>(area + held_at + 1024 * s);
      else qs = q[s];
#pragma unroll
      for (int b = 0; b < 2; ++b) acc[b] = E::mfma16(kf[b][s], qs, acc[b]);
    }
    float s8[8];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) s8[4 * b + e] = j0 + 16 * b + 4 * kq + e < visible ? acc[b][e] : -__builtin_inff();
    float mc = fmaxf(fmaxf(fmaxf(s8[0], s8[1]), fmaxf(s8[2], s8[3])), fmaxf(fmaxf(s8[4], s8[5]), fmaxf(s8[6], s8[7])));
    mc = fmaxf(mc, __shfl_xor(mc, 16, 64));
    mc = fmaxf(mc, __shfl_xor(mc, 32, 64));
    const float want = reference_of<E::kSmallBias>(scaled(mc, p.scale_log2));
    float mn = fmaxf(m, want);
    if constexpr (E::kNarrow) {
      peak = fmaxf(peak, want);
      const bool fall = (m - want > kFall) & (want > -__builtin_inff());
      mn = fall ? fmaxf(want, peak - kReach) : mn;
    }
    // a NaN score, which the maximum skips, makes l and o NaN, and so they stay
    const float ref = reference(mn);
    const float corr = __builtin_amdgcn_exp2f(m - ref);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s8[i] = __builtin_amdgcn_exp2f(scaled(s8[i], p.scale_log2) - ref);
      sum += s8[i];
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    l = l * corr + sum;
    m = mn;
    u32x4 pf, pr;  // the weights' two parts
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pf[i] = pack2<E>(s8[2 * i], s8[2 * i + 1]);
      pr[i] = rest2<E>(s8[2 * i], s8[2 * i + 1], pf[i]);
    }
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
        o[c] = E::mfma16(a, pr, E::mfma16(a, pf, o[c]));
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
          const f32x4 t = E::mfma16(a, pr, E::mfma16(a, pf, o[c]));
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][e] = mine ? t[e] : o[c][e];
        }
      }
    }
  }
  // merge the four waves: each scales its sums to the workgroup's largest reference (a wave without keys has sums of 0, not only a
  // maximum of -inf: with scores that are all NaN its sums are NaN and stay in)
  if (kq == 0) {
    mx[wave][lr] = m;
    ls[wave][lr] = l;
  }
  __syncthreads();
  const auto factor = [&](float mw, float M) { return __builtin_amdgcn_exp2f(mw - reference(M)); };
  const float M = fmaxf(fmaxf(mx[0][lr], mx[1][lr]), fmaxf(mx[2][lr], mx[3][lr]));
  const float f = factor(m, M);
  float* const mine = reinterpret_cast<float*>(area) + lr * kPitch;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int c = 0; c < NC; c += 4)
      *reinterpret_cast<f32x4*>(mine + NC * (4 * kq + e) + c) =
          f32x4{o[c][e] * f, o[c + 1][e] * f, o[c + 2][e] * f, o[c + 3][e] * f};
  __syncthreads();
  const int64_t held = (static_cast<int64_t>(w.partial + w.chunk) * p.kv + kvh) * 16;
  for (int i = tid; i < nrows * (D / 4); i += 256) {
    const int row = i / (D / 4), c = i % (D / 4) * 4;
    const int at = 4 * (row * kPitch + c);
    f32x4 v = *reinterpret_cast<const f32x4*>(areas[0] + at);
#pragma unroll
    for (int x = 1; x < 4; ++x) v += *reinterpret_cast<const f32x4*>(areas[x] + at);
    const float Mr = fmaxf(fmaxf(mx[0][row], mx[1][row]), fmaxf(mx[2][row], mx[3][row]));
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) sum += ls[x][row] * factor(mx[x][row], Mr);
    const int rr = w.tile * 16 + row, tk = divide(rr, p.by_group), hd = kvh * p.group + rr - tk * p.group;
    const int64_t out = static_cast<int64_t>(w.start + tk) * p.heads + hd;
    if (w.partial >= 0) {
      *reinterpret_cast<f32x4*>((on_front ? p.prefix_part : p.part) + (held + row) * D + c) = v;
      if (c == 0) {
        (on_front ? p.prefix_ml : p.ml)[held + row] = make_float2(Mr, sum);
        if (w.chunk == 0) (on_front ? p.prefix_info : p.info)[out] = make_int2(static_cast<int>(held) + row, w.chunks);
      }
    } else {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
      *reinterpret_cast<uint2*>(p.out + out * D + c) =
          make_uint2(pack2<E>(v[0] * inv, v[1] * inv), pack2<E>(v[2] * inv, v[3] * inv));
      if (c == 0 && w.chunk == 0) (on_front ? p.prefix_info : p.info)[out] = make_int2(0, 0);
    }
  }
}

// ------------------------------------------------------------------ 128 rows, four waves of 32
// For blocks of many rows.  A workgroup takes 64 keys at a time through LDS, two stages of keys and values, loaded straight into
// it a step ahead; wave w has rows 32 w to 32 w + 31 for all of them.  Scores transposed again: lane l holds query row l & 31 and
// keys 8 (e / 4) + 4 (l >> 5) + e % 4 of a 32-key block (e: element of the 32x32 result), whose elements 8 s to 8 s + 7 are, as a
// reduction's octet l >> 5, the B operand of O^T = V^T P^T for keys 16 s of the block.  So a probability never leaves its lane.  V^T's
// operand needs eight keys of a dim: two transposing LDS reads of four keys each.
// Bound: matrix instructions, behind them LDS reads (a wave reads every key and value for its 32 rows; 64 rows a wave would halve
// the reads but need more than its 512 registers at head dim 256).  2048 tokens behind 6144 keys, 16 heads of 256: 313 to 328 us, 733 to
// 767 TFLOP/s of the formulas, 1.1 PFLOP/s of matrix instructions with the weights' second parts (a large library product 1.3); prompts
// of 442 to 2222 tokens, 32 heads of 128: 157 to 165 us.  Started cold, a launch spends about 14 us before and behind its
// steps, most of it fetching code that runs once.
// The rows' reference moves only when a score exceeds it by kRise (weights reach 2^kRise, their relative precision is the same): the
// accumulators are rescaled a few times a row instead of at every step.
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
constexpr int kLargeRows = 128, kLargeUnit = 64, kLargeLeast = 4;
template <int D>
constexpr int kStage = 64 * D * 2;  // bytes of a stage of keys or values
// `odd`: set where a stage lacks values that are infinite or NaN.
template <int D, class E, bool kPrefix>
__device__ __forceinline__ void large_share(const PagedParams& p, const Share& w, int kvh, char* const keys0, char* const keys1, char* const values0, char* const values1, int& odd) {
  constexpr int KS = D / 16, NC = D / 32, SL = D / 8, KR = 256 / SL, KP = 64 / KR;
  constexpr int kAhead = D == 256 ? 4 : 2;
  const PagedSide& side = kPrefix ? p.prefix : p.own;
  const bool causal = !kPrefix && p.causal;
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, l31 = lane & 31, half = lane >> 5;
  const int rows = w.tokens * p.group, nrows = min(kLargeRows, rows - w.tile * kLargeRows);
  const int row0 = w.tile * kLargeRows;
  const int r = row0 + min(wave * 32 + l31, nrows - 1);
  const int tok = divide(r, p.by_group), head = kvh * p.group + r - tok * p.group;
  const int visible = visible_keys(w.keys, w.tokens, tok, causal);
  const int least = visible_keys(w.keys, w.tokens, uniform(static_cast<int>(divide(row0, p.by_group))), causal);
  const int n = visible_keys(w.keys, w.tokens, uniform(static_cast<int>(divide(row0 + nrows - 1, p.by_group))), causal);
  const int k0 = w.chunk * w.c * kLargeUnit, k1 = chunk_end(k0, w.c, kLargeUnit, n);
  const int steps = k1 > k0 ? (k1 - k0 + 63) / 64 : 0;

  if (tid == 0) odd = 0;

  // Staging: thread tid loads 16-byte slot tid % SL of rows tid / SL, + KR, ... of keys and values.  A 16-row group's place is a 64-bit
  // offset, looked up many steps ahead; rows inside it are 32-bit offsets that do not change.
  // LDS: slot c of row r holds 16-byte piece c ^ (r % 16) of the keys, c ^ 4 (r % 8 or 4) of the values, so that neither kind of read
  // puts two of the lanes that read together on one bank; the loads permute the pieces, since their own order in LDS is fixed.
  const char* keys = reinterpret_cast<const char*>(side.keys + kvh * side.key_head);
  const char* vals = reinterpret_cast<const char*>(side.values + kvh * side.value_head);
  const int krow = static_cast<int>(2 * side.key_row), vrow = static_cast<int>(2 * side.value_row);  // bytes
  const auto vcol = [](int t) { return static_cast<uint32_t>((t % SL ^ (t / SL & (D == 256 ? 7 : 3)) << 2) * 16); };
  const auto kcol = [](int t, int i) { return static_cast<uint32_t>((t % SL ^ ((t / SL + i * KR) & 15)) * 16); };
  uint32_t koff[KP / 4], voff[KP / 4];
#pragma unroll
  for (int i = 0; i < KP / 4; ++i) {
    koff[i] = (tid / SL + i * KR) * krow + kcol(tid, i);
    voff[i] = (tid / SL + i * KR) * vrow + vcol(tid);
  }
  // Groups' places, 64 of them (16 steps) a lookup, group lane of its block of steps: byte offsets of keys and values.
  struct Places {
    int64_t k, v;
  };
  const auto find = [&](int block) {
    const PageAt at = page_at(side, w.table, min(k0 / 16 + 64 * block + (thread_again() & 63), (n - 1) / 16));
    return Places{at.page * (2 * side.key_page) + static_cast<int64_t>(at.row) * krow,
                  at.page * (2 * side.value_page) + static_cast<int64_t>(at.row) * vrow};
  };
  struct Bases {
    const char* g[4];  // of the step's four groups
  };
  const auto bases = [&](const char* from, int64_t places, int step) {
    Bases b;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(places), 4 * (step & 15) + g);
      const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(static_cast<uint64_t>(places) >> 32), 4 * (step & 15) + g);
      b.g[g] = from + static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
    }
    return b;
  };
  const auto piece = [&](auto values_, char* into, const Bases& b, int i) {
    copy_to_lds(b.g[i / (KP / 4)], (decltype(values_)::value ? voff : koff)[i % (KP / 4)], into + wave * 1024 + i * 4096);
  };
  const auto load = [&](auto values_, char* into, int64_t places, int step) {
    constexpr bool values = decltype(values_)::value;
    const int key0 = k0 + 64 * step;
    const Bases b = bases(values ? vals : keys, places, step);
    if (key0 + 64 <= n) {
#pragma unroll
      for (int i = 0; i < KP; ++i) piece(values_, into, b, i);
    } else {  // rows past the last key repeat it
      const int t = thread_again();
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const int row = min((i * KR + t / SL) & 15, n - 1 - 16 * min(key0 / 16 + i * KR / 16, (n - 1) / 16));
        copy_to_lds(b.g[i / (KP / 4)], row * (values ? vrow : krow) + (values ? vcol(t) : kcol(t, i)), into + wave * 1024 + i * 4096);
      }
    }
  };
  // Some row masks some of a step's keys: its weights there are 0, but 0 times an infinite or NaN value is not.  Such values, and keys
  // past the last one, become zeros in the stage.
  const auto clean = [&](char* stage, int key0) {
    bool wild = false;
    const int t = thread_again();
#pragma unroll 1
    for (int i = 0; i < KP; ++i) {
      u32x4* at = reinterpret_cast<u32x4*>(stage + i * 4096 + t * 16);
      u32x4 v = *at;
      const bool in = key0 + i * KR + t / SL < n;
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
  uint32_t vr = (4 * half + (j15 >> 2)) * (2 * D) + (2 * (lane >> 4 & 1) + (j15 >> 1 & 1)) * 16 + (j15 & 1) * 8 + turn * 64;

  f32x16 o[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[c][e] = 0.f;
  float m = -__builtin_inff(), l = 0.f;  // reference of the row's weights, and the sum of this lane's weights
  float peak = -__builtin_inff();        // the highest reference that its scores asked for, where it may fall

  // Step i multiplies the next step's keys with the queries, then its own weights with its values: the exponentials of its scores
  // stand between the matrix instructions of the one, the maximum of the next scores between those of the other.  Each half ends
  // with a barrier, after which the stage it read takes the keys, or values, of two steps on: every load has one and a half steps.
  const std::false_type of_keys{};
  const std::true_type of_values{};
  Places here{0, 0}, after{0, 0};  // of the steps whose keys are loaded, and of the next 16
  int64_t vhere = 0;               // of the step whose values are loaded, a step behind
  const auto turn_keys = [&](int t) {
    if (t > 0 && (t & 15) == 0) {
      here = after;
      after = find(t / 16 + 1);
    }
  };
  const auto turn_values = [&](int t) {
    if ((t & 15) == 0) vhere = here.v;
  };
  const auto load_keys = [&](char* into, int t) {
    if (t >= steps) return;
    turn_keys(t);
    load(of_keys, into, here.k, t);
  };
  const auto load_values = [&](char* into, int t) {
    if (t >= steps) return;
    turn_values(t);
    load(of_values, into, vhere, t);
  };
  // All but the last 2 KP loads have arrived, where that many are on their way behind the ones waited for; and every wave is here.
  const auto arrive = [&](bool behind) {
    if (behind) __builtin_amdgcn_s_waitcnt(KP == 8 ? 0x4F70 : 0x0F78);  // vmcnt(2 KP)
    else wait_vmem();
    lds_barrier();
  };
  u32x4 q[KS];
  if (steps > 0) {
    here = find(0);
    const uint16_t* qr = p.query + (w.start + tok) * p.query_token + head * p.query_head + 8 * half;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const u32x4*>(qr + 16 * s);
    load_keys(keys0, 0);
    load_keys(keys1, 1);
    load_values(values0, 0);
    after = find(1);
    // at head dim 256 the queries stay in the accumulation registers, where matrix instructions take them from
    if constexpr (D == 256) {
#pragma unroll
      for (int s = 0; s < KS; ++s) asm volatile("" : "+a"(q[s]));
    }
  }
  arrive(false);
  if (wave * 32 >= nrows) {  // no rows: the wave only stages
    if (steps > 0) lds_barrier();
    load_keys(keys0, 2);
    load_values(values1, 1);
    for (int i = 0; i < steps; ++i) {
      arrive(i + 2 < steps);
      load_keys(i & 1 ? keys0 : keys1, i + 3);
      if (k0 + 64 * (i + 1) > least) clean(i & 1 ? values1 : values0, k0 + 64 * i);
      arrive(i + 3 < steps);
      load_values(i & 1 ? values1 : values0, i + 2);
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
  const auto key_at = [&](const char* from, int i) {
    return *reinterpret_cast<const u32x4*>(from + ((kr ^ (32 * (i >> 1))) + (i & 1) * 64 * D));
  };
  float mc = -__builtin_inff();  // maximum of the scores of the step to come
  if (steps > 0) {
    clear(sc[0]);
    feed<2 * KS, kAhead>([&](int i) { return key_at(keys0, i); },
                         [&](int i, u32x4 k) { sc[0][i & 1] = E::mfma32(k, q[i >> 1], sc[0][i & 1]); });
    hide(sc[0], k0);
#pragma unroll
    for (int e = 0; e < 32; ++e) mc = fmaxf(mc, sc[0][e >> 4][e & 15]);
    lds_barrier();
    load_keys(keys0, 2);
  }
  const auto step = [&](auto stage_, auto inner_, int i) {
    constexpr int stage = decltype(stage_)::value;
    // Whole steps follow: the loads stand between the matrix instructions too.  And no row masks any of this step's keys or the next's:
    // a tile has 128 tokens at most, so that all rows see all but the last 127 keys, and five steps follow.
    constexpr bool inner = decltype(inner_)::value;
    char* const other = stage ? keys0 : keys1;      // the next step's keys
    char* const held = stage ? values1 : values0;   // this step's values
    const int key0 = k0 + 64 * i;
    f32x16(&now)[2] = sc[stage];
    f32x16(&next)[2] = sc[stage ^ 1];
    asm volatile("" : "+v"(kr), "+v"(vr));  // no two dozen registers of places kept over the steps
    mc = fmaxf(mc, __shfl_xor(mc, 32, 64));
    // a NaN score, which the maximum skips, makes l and o NaN, and so they stay
    const float top = scaled(mc, p.scale_log2);
    float to = reference_of<E::kLargeBias>(top);
    bool move = top - m > E::kRise + E::kLargeBias;  // the first key's too, from -inf; not where both are
    if constexpr (E::kNarrow) {
      peak = fmaxf(peak, to);
      move |= (m - to > kFall) & (to > -__builtin_inff()) & (m > peak - kReach);
      to = fmaxf(to, peak - kReach);
    }
    if (__any(move)) {
      if (!move) to = m;
      const float corr = __builtin_amdgcn_exp2f(m - reference(to));
      l *= move ? corr : 1.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[c][e] *= move ? corr : 1.f;
      m = to;
    }
    const float ref = reference(m);
    float sum[2] = {0.f, 0.f};
    const auto weigh = [&](int e) {  // elements e and e + 1 of the step's 32
      float x = __builtin_amdgcn_exp2f(scaled(now[e >> 4][e & 15], p.scale_log2) - ref);
      float y = __builtin_amdgcn_exp2f(scaled(now[e >> 4][(e & 15) + 1], p.scale_log2) - ref);
      asm volatile("" : "+v"(x), "+v"(y));  // made here, between the matrix instructions, not where they are used
      sum[0] += x;
      sum[1] += y;
      now[e >> 4][e & 15] = x;
      now[e >> 4][(e & 15) + 1] = y;
    };
    clear(next);
    constexpr int kPairK = KS / 8, kPairV = NC / 4;  // matrix instructions a pair of elements
    char* const ahead = stage ? values0 : values1;   // the next step's values
    Bases b;
    if constexpr (inner) {
      turn_values(i + 1);
      b = bases(vals, vhere, i + 1);
    }
    feed<2 * KS, kAhead>([&](int k) { return key_at(other, k); },
                         [&](int k, u32x4 v) {
                           next[k & 1] = E::mfma32(v, q[k >> 1], next[k & 1]);
                           if (k % kPairK == 0) weigh(k / kPairK * 2);
                           if constexpr (inner) {
                             if (k % 4 == 1) piece(of_values, ahead, b, k / 4);
                           }
                         });
    if constexpr (!inner) hide(next, key0 + 64);
    l += sum[0] + sum[1];
    mc = -__builtin_inff();
    arrive(inner || i + 2 < steps);
    if constexpr (inner) {
      turn_keys(i + 3);
      b = bases(keys, here.k, i + 3);
    } else {
      load_keys(other, i + 3);
    }
    if constexpr (!inner) {
      if (key0 + 64 > least) clean(held, key0);
    }
    u32x4 pf, pr;  // the two parts of the weights of 16 keys
    const auto split = [&](int part) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 8 * part + 2 * i;
        const float x = now[e >> 4][e & 15], y = now[e >> 4][(e & 15) + 1];
        pf[i] = pack2<E>(x, y);
        pr[i] = rest2<E>(x, y, pf[i]);
      }
    };
    feed<4 * NC, kAhead>(
        [&](int k) {
          const char* at = held + ((vr ^ (64 * (k % NC))) + k / NC * 32 * D);
          const uint2 a = read_turned(at), b = read_turned(at + 16 * D);
          return u32x4{a.x, a.y, b.x, b.y};
        },
        [&](int k, u32x4 v) {
          if (k % NC == 0) split(k / NC);
          o[k % NC] = E::mfma32(v, pf, o[k % NC]);
          o[k % NC] = E::mfma32(v, pr, o[k % NC]);
          if (k % kPairV == 0) {
            const int e = k / kPairV * 2;
            mc = fmaxf(fmaxf(mc, next[e >> 4][e & 15]), next[e >> 4][(e & 15) + 1]);
          }
          if constexpr (inner) {
            if (k % 4 == 1) piece(of_keys, other, b, k / 4);
          }
        });
    arrive(inner || i + 3 < steps);
    if constexpr (!inner) load_values(held, i + 2);
  };
  // the last step multiplies keys that are none: code of its own for it would cost more than that
  const std::integral_constant<int, 0> even{};
  const std::integral_constant<int, 1> uneven{};
  int i = 0;
  for (; i + 5 < steps; i += 2) {
    step(even, std::true_type{}, i);
    step(uneven, std::true_type{}, i + 1);
  }
  load_values(values1, i + 1);
  for (; i < steps; i += 2) {
    step(even, std::false_type{}, i);
    if (i + 1 < steps) step(uneven, std::false_type{}, i + 1);
  }
  const int again = thread_again();  // the lane's row once more
  const int part = again >> 5 & 1, mine = (again >> 6) * 32 + (again & 31), at_row = row0 + min(mine, nrows - 1);
  const int at_token = divide(at_row, p.by_group), at_head = kvh * p.group + at_row - at_token * p.group;
  if (steps > 0 && odd) {
    // the values left out of the stages: infinite or NaN in the rows that see them, whatever their (positive) weight
    for (int key = k0 + max(0, (least - k0) / 64) * 64; key < k1; ++key) {
      const PageAt at = page_at(side, w.table, key / 16);
      const char* src = vals + 2 * at.page * side.value_page + static_cast<int64_t>(at.row + key % 16) * vrow;
      if (key >= visible_keys(w.keys, w.tokens, at_token, causal)) continue;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const uint2 v = *reinterpret_cast<const uint2*>(src + 2 * (32 * c + 2 * e + 4 * part));
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t x = (y < 2 ? v.x : v.y) >> (16 * (y & 1)) & 0xFFFF;
            if ((x & E::kExponent) == E::kExponent) o[c][e + y] += E::to_f32(x);
          }
        }
    }
  }

  l += __shfl_xor(l, 32, 64);
  if (mine >= nrows) return;
  const int64_t out = static_cast<int64_t>(w.start + at_token) * p.heads + at_head;
  if (w.partial >= 0) {
    const int64_t held = (static_cast<int64_t>(w.partial + w.chunk) * p.kv + kvh) * kLargeRows + mine;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4*>((kPrefix ? p.prefix_part : p.part) + held * D + 32 * c + 2 * e + 4 * part) = f32x4{o[c][e], o[c][e + 1], o[c][e + 2], o[c][e + 3]};
    if (part == 0) {
      (kPrefix ? p.prefix_ml : p.ml)[held] = make_float2(m, l);
      if (w.chunk == 0) (kPrefix ? p.prefix_info : p.info)[out] = make_int2(static_cast<int>(held), w.chunks);
    }
  } else {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<uint2*>(p.out + out * D + 32 * c + 2 * e + 4 * part) =
            make_uint2(pack2<E>(o[c][e] * inv, o[c][e + 1] * inv), pack2<E>(o[c][e + 2] * inv, o[c][e + 3] * inv));
    if (part == 0 && w.chunk == 0) (kPrefix ? p.prefix_info : p.info)[out] = make_int2(0, 0);
  }
}

// ------------------------------------------------------------------ the kernels
template <int D, class E>
__global__ __launch_bounds__(256, 2) void paged_small_kernel(PagedParams p) {
  __shared__ __align__(16) char s0[kSmallArea<D>], s1[kSmallArea<D>], s2[kSmallArea<D>], s3[kSmallArea<D>];
  __shared__ float mx[4][16], ls[4][16];
  SeqSpan last{0, 0, 0};
  const int c = uniform(chunk_units(own_work(p, kSmallRows, kSmallUnit, &last).units, p.kv, p.per_slot, 1));
  Share w;
  if (!own_share(p, blockIdx.x / p.kv, kSmallRows, kSmallUnit, c, last, &w)) return;
  small_share<D, E>(p, w, false, uniform(static_cast<int>(blockIdx.x) % p.kv), {s0, s1, s2, s3}, mx, ls);
}
template <int D, class E>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_large_kernel(PagedParams p) {
  __shared__ __align__(16) char keys0[kStage<D>], keys1[kStage<D>], values0[kStage<D>], values1[kStage<D>];
  __shared__ int odd;
  SeqSpan last{0, 0, 0};
  const int c = uniform(chunk_units(own_work(p, kLargeRows, kLargeUnit, &last).units, p.kv, p.per_slot, kLargeLeast));
  Share w;
  if (!own_share(p, blockIdx.x / p.kv, kLargeRows, kLargeUnit, c, last, &w)) return;
  large_share<D, E, false>(p, w, uniform(static_cast<int>(blockIdx.x) % p.kv), keys0, keys1, values0, values1, odd);
}
// The prefix and the sequences' own keys in one launch: what multiplies much and what reads many bytes run side by side, and
// neither waits for the other's slowest share.  The workgroups that run at once are divided by the two sides' work; the prefix's
// shares, all alike, come first, and the sequences' take what places are left.
template <int D, class E, bool kOwnLarge, bool kFrontLarge>
__global__ __launch_bounds__(256, kFrontLarge && D == 256 ? 1 : 2) void paged_pair_kernel(PagedParams p) {
  static_assert(kFrontLarge || !kOwnLarge, "the prefix has the rows of all sequences");
  constexpr int kArea = kFrontLarge ? kStage<D> : kSmallArea<D>;
  static_assert(kArea >= kSmallArea<D>, "either fits");
  constexpr int kOwnRows = kOwnLarge ? kLargeRows : kSmallRows, kOwnUnit = kOwnLarge ? kLargeUnit : kSmallUnit;
  constexpr int kFrontRows = kFrontLarge ? kLargeRows : kSmallRows, kFrontUnit = kFrontLarge ? kLargeUnit : kSmallUnit;
  // Time of a unit of own keys, and of a row tile's start and end, in units of the prefix: a 128-row step takes about 2 us and its
  // kernel's start and end 14, a 16-row round 3 us or, when memory is the limit, 6, its start and end 8.  kUnitCost from 1.5 to
  // 4: 64 sequences behind 8192 shared keys 42.0 to 46.3 us (43.9 here), 256 behind 32768 254.7 to 258 (255).
  constexpr float kUnitCost = kOwnLarge == kFrontLarge ? 1.f : 3.f, kStartCost = kOwnLarge ? 8.f : kFrontLarge ? 4.5f : 2.f;
  __shared__ __align__(16) char s0[kArea], s1[kArea], s2[kArea], s3[kArea];
  __shared__ float mx[4][16], ls[4][16];
  __shared__ int odd;
  const int kvh = uniform(static_cast<int>(blockIdx.x) % p.kv), id = blockIdx.x / p.kv;
  int keys;
  SeqSpan last{0, 0, 0};
  const Work front = front_work(p, kFrontRows, kFrontUnit, &keys), own = own_work(p, kOwnRows, kOwnUnit, &last);
  const float for_own = own_places(own.units, own.tiles, front.units, p.kv, p.slots, kUnitCost, kStartCost);
  const int c0 = uniform(front_chunk(front.units, p.kv, p.slots, for_own, kFrontLarge ? kLargeLeast : 1));
  const int chunks = uniform(tile_chunks(seq_units(keys, kFrontUnit), c0)), shares = front.tiles * chunks;
  Share w;
  if (id < shares) {
    const int tile = uniform(static_cast<int>(static_cast<uint32_t>(id) / static_cast<uint32_t>(chunks)));
    w = Share{0, p.T, keys, tile, id - tile * chunks, chunks, tile * chunks, c0, p.prefix.table};
    if constexpr (kFrontLarge) {
      large_share<D, E, true>(p, w, kvh, s0, s1, s2, s3, odd);
      return;
    }
  } else {
    const int c1 = uniform(own_chunk(own.units, p.kv, for_own, kOwnLarge ? kLargeLeast : 1));
    if (!own_share(p, id - shares, kOwnRows, kOwnUnit, c1, last, &w)) return;
    if constexpr (kOwnLarge) large_share<D, E, false>(p, w, kvh, s0, s1, s2, s3, odd);
  }
  if constexpr (!kOwnLarge) small_share<D, E>(p, w, !kFrontLarge && id < shares, kvh, {s0, s1, s2, s3}, mx, ls);
}

// ------------------------------------------------------------------ merge
// kWaves waves per (token, head), D / 64 dims a lane; wave w takes the row's partial results w, w + kWaves, ..., eight in flight, and
// the waves' sums meet in LDS.  The order of the additions depends on the sizes alone.  A wave that has rows to itself (kWaves 1)
// looks at kRows of them at once and takes those that are in parts.
// Bound: latency (info, then the parts): 4.7 us where nothing is in parts, 6 to 9 where all is.  Eight waves a row instead of one: 62
// instead of 83 us for a row behind 131072 keys, 17.6 instead of 20.9 for 8 blocks of 2 behind 4096 (both kernels); sixteen rows a
// wave instead of one: 2 us less for 32768 rows that are in one part each.
template <int D, class E, int kWaves, int kRows>
__global__ __launch_bounds__(kWaves == 1 ? 256 : 64 * kWaves) void paged_merge_kernel(PagedParams p) {
  static_assert(kWaves == 1 || kRows == 1, "waves that share rows meet once");
  constexpr int F = D / 64, kFlight = 8;
  __shared__ float om[kWaves == 1 ? 1 : kWaves][D], lm[kWaves], mm[kWaves];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, part = kWaves == 1 ? 0 : wave;
  const int64_t row0 = kWaves == 1 ? (static_cast<int64_t>(blockIdx.x) * 4 + wave) * kRows : blockIdx.x;
  const int64_t rows = static_cast<int64_t>(p.T) * p.heads;
  // rows of tokens in no sequence are not written
  const int64_t from = static_cast<int64_t>(p.starts[0]) * p.heads, to = static_cast<int64_t>(p.starts[p.B]) * p.heads;
  int2 range[2] = {make_int2(0, 0), make_int2(0, 0)};
  {
    const int64_t row = row0 + lane % kRows;
    if (row < rows) {
      range[0] = p.info[row];
      if (p.merge_prefix) range[1] = p.prefix_info[row];
    }
    if (row < from || row >= to) range[0].y = 0;
  }
  uint64_t todo = __ballot(range[0].y > 0 && lane < kRows);
  for (; todo; todo &= todo - 1) {
    const int at = __builtin_ctzll(todo);
    const int64_t row = row0 + at;
    float M = -__builtin_inff(), l = 0.f, acc[F];
#pragma unroll
    for (int i = 0; i < F; ++i) acc[i] = 0.f;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      if (g == 1 && !p.merge_prefix) break;
      const int first = __builtin_amdgcn_readlane(range[g].x, at);
      int chunks = __builtin_amdgcn_readlane(range[g].y, at);
      // whatever the sequences' starts held, nothing outside the partial results is read
      const int64_t stride = static_cast<int64_t>(g ? p.prefix_tile_rows : p.own_tile_rows) * p.kv;
      if (first < 0 || chunks < 0 || first + (chunks - 1) * stride >= p.part_rows[g]) chunks = 0;
      const float2* ml = g ? p.prefix_ml : p.ml;
      const float* data = (g ? p.prefix_part : p.part) + lane * F;
      const int64_t step = stride * kWaves, base = first + part * stride;
      const int count = (chunks - part + kWaves - 1) / kWaves;
      for (int i0 = 0; i0 < count; i0 += kFlight) {
        float x[kFlight][F];
        float2 v[kFlight];
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
          const int64_t r = base + min(i0 + i, count - 1) * step;
          v[i] = ml[r];
          if (i0 + i >= count) v[i] = make_float2(-__builtin_inff(), 0.f);
#pragma unroll
          for (int f = 0; f < F; ++f) x[i][f] = data[r * D + f];
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < kFlight; ++i) top = fmaxf(top, v[i].x);
        const float ref = reference(top);
        const float corr = __builtin_amdgcn_exp2f(M - ref);
        M = top;
        l *= corr;
#pragma unroll
        for (int k = 0; k < F; ++k) acc[k] *= corr;
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
          if (v[i].y == 0.f) continue;  // no key of this row in that chunk, whose row may hold anything
          const float f = __builtin_amdgcn_exp2f(v[i].x - ref);
          l += v[i].y * f;
#pragma unroll
          for (int k = 0; k < F; ++k) acc[k] += x[i][k] * f;
        }
      }
    }
    if (kWaves > 1) {  // the same rows in all waves: they share one
      if (lane == 0) {
        lm[part] = l;
        mm[part] = M;
      }
#pragma unroll
      for (int k = 0; k < F; ++k) om[part][lane * F + k] = acc[k];
      __syncthreads();
      if (wave) return;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) M = fmaxf(M, mm[w]);
      const float ref = reference(M);
      l = 0.f;
#pragma unroll
      for (int k = 0; k < F; ++k) acc[k] = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(mm[w] - ref);
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
}

}  // namespace

// Rows of a side's tiles, by the rows a sequence has on average: up to 20 take the kernel of 16 rows, whose waves share the
// keys out; more, which would be two such tiles or several, take the one of 128, whose waves share the keys' way through LDS.  16 and
// 128 rows, us: 64 sequences behind 4096 keys, 16 rows each 109 and 108, 24 rows 163 and 110, 32 rows 164 and 111; 8 sequences,
// 16 rows 25 and 27, 24 rows 33 and 29, 75 rows on average 35 and 31; of unlike blocks, 64 of 18 rows on average 79 and 99, 8 of
// 21 27 and 25, 64 of 31 121 and 102; 16 sequences of 24 rows behind 1000 keys 19 and 23; one row 14 and 20.
int paged_tile_rows(int64_t tokens, int64_t sequences, int64_t group) {
  const int64_t blocks = std::max<int64_t>(1, std::min(tokens, sequences));
  return tokens * group > 20 * blocks ? kLargeRows : kSmallRows;
}
// Workgroups that a stage's work is cut for: as many as run at once.
int paged_slots(int tile_rows, int head_dim, int cus) { return tile_rows == kLargeRows && head_dim == 256 ? cus : 2 * cus; }

template <int D, class E>
static void launch_append(const AppendParams& p, hipStream_t stream) {
  // a token's heads over several workgroups while there are few tokens: each makes the token's angles itself
  constexpr int kHeads = 256 / (D / 8);
  const int all = (p.heads + 2 * p.kv + kHeads - 1) / kHeads;
  hipLaunchKernelGGL((paged_append_kernel<D, E>), dim3(p.T, p.T <= 1024 ? all : 1), dim3(256), 0, stream, p);
}
void launch_paged_append(int head_dim, bool bf16, const AppendParams& p, hipStream_t stream) {
  if (head_dim == 256) bf16 ? launch_append<256, Bf16>(p, stream) : launch_append<256, Fp16>(p, stream);
  else bf16 ? launch_append<128, Bf16>(p, stream) : launch_append<128, Fp16>(p, stream);
}

template <int D, class E>
static void launch_attend(const PagedParams& p, hipStream_t stream) {
  const int own = p.own_tile_rows, front = p.prefix_tile_rows;
  const int64_t tiles = max_tiles(p.T, p.B, p.group, own) + (p.merge_prefix ? seq_tiles(p.T, p.group, front) : 0);
  const dim3 grid(max_chunks(tiles, p.kv, p.slots) * p.kv), block(256);
  if (p.merge_prefix && own == kLargeRows) hipLaunchKernelGGL((paged_pair_kernel<D, E, true, true>), grid, block, 0, stream, p);
  else if (p.merge_prefix && front == kLargeRows) hipLaunchKernelGGL((paged_pair_kernel<D, E, false, true>), grid, block, 0, stream, p);
  else if (p.merge_prefix) hipLaunchKernelGGL((paged_pair_kernel<D, E, false, false>), grid, block, 0, stream, p);
  else if (own == kLargeRows) hipLaunchKernelGGL((paged_large_kernel<D, E>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((paged_small_kernel<D, E>), grid, block, 0, stream, p);
  const int least = own == kLargeRows ? kLargeUnit * kLargeLeast : kSmallUnit;
  if (!p.merge_prefix && p.own.capacity <= least) return;  // one chunk a tile: nothing to merge
  const int64_t rows = static_cast<int64_t>(p.T) * p.heads;
  // few rows may be in many chunks: eight waves a row; many rows are mostly in one: sixteen rows a wave
  if (rows <= 512) hipLaunchKernelGGL((paged_merge_kernel<D, E, 8, 1>), dim3(rows), dim3(512), 0, stream, p);
  else if (rows <= 16384) hipLaunchKernelGGL((paged_merge_kernel<D, E, 1, 1>), dim3((rows + 3) / 4), dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((paged_merge_kernel<D, E, 1, 16>), dim3((rows + 63) / 64), dim3(256), 0, stream, p);
}
void launch_paged_attention(int head_dim, bool bf16, const PagedParams& p, hipStream_t stream) {
  if (head_dim == 256) bf16 ? launch_attend<256, Bf16>(p, stream) : launch_attend<256, Fp16>(p, stream);
  else bf16 ? launch_attend<128, Bf16>(p, stream) : launch_attend<128, Fp16>(p, stream);
}

}  // namespace dflash
