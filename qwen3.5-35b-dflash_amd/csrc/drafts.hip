// Check of drafted tokens against the target's probabilities from given random numbers (speculative sampling).
//
// Sequence b has rows [starts[b], starts[b + 1]); row r predicts the token behind row r, and drafted[r] is the drafter's
// choice for it (the last row has none).  With p and q the softmaxes of the target's and the drafter's logits over the
// temperature, x = drafted[r] and u = uniforms[r]:  x is accepted iff u q(x) < p(x).  The first row r that is not accepted
// draws its token from max(p - q, 0), the last row from p, both by the inverse of the running sum with the uniform of the
// row behind (r + 1, which tests nothing then) or of the last row itself.  So the tokens follow the target's distribution
// whatever the drafter's is.
//
// A whole number hangs on a comparison, so what is compared carries 64 bits: the sums, and in the rows that tokens are drawn
// from each weight, since one of 2.5e5 running sums lies within 1e-7 of a given number once in forty times.  The
// acceptance test compares one number a row; its sums add 32-bit exponentials in 64 bits.
//
// Logits that are NaN count as -infinity, +infinity as the largest fp32 number.  A row without a logit above -infinity has no
// token to give.
#include "kernels.h"

#include <float.h>

namespace dflash {
namespace {

constexpr float kNone = -FLT_MAX;
constexpr int kNowhere = 0x7FFFFFFF;

// Logits as the caller has them: kType an enum dflash_dtype.
template <int kType>
struct Row {
  static constexpr int kSize = kType == 1 ? 4 : 2;
  const char* data;
  int V, ahead;  // ahead: tokens that the row's first eight start before the row itself, so that all but its ends are aligned

  __device__ Row(const void* base, int64_t stride, int row, int vocab)
      : data(static_cast<const char*>(base) + row * stride * kSize), V(vocab) {
    ahead = static_cast<int>((reinterpret_cast<uintptr_t>(data) & 15u) / kSize);
  }
  __device__ int eights() const { return (V + ahead + 7) / 8; }
  __device__ int first(int eight) const { return 8 * eight - ahead; }
  __device__ static float bounded(float v) { return fminf(fmaxf(v, -INFINITY), FLT_MAX); }
  __device__ float at(int64_t i) const {
    if constexpr (kType == 1) return bounded(reinterpret_cast<const float*>(data)[i]);
    const uint16_t w = reinterpret_cast<const uint16_t*>(data)[i];
    return bounded(kType == 0 ? bf16_to_f32(w) : static_cast<float>(__builtin_bit_cast(_Float16, w)));
  }
  struct Raw {
    uint4 w[kSize / 2];
  };
  // Eight tokens from an aligned place inside the row
  __device__ Raw raw(int64_t j) const {
    Raw r;
    const uint4* from = reinterpret_cast<const uint4*>(data + j * kSize);
#pragma unroll
    for (int i = 0; i < kSize / 2; ++i) r.w[i] = from[i];
    return r;
  }
  __device__ static void unpack(const Raw& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4& q = r.w[kType == 1 ? i / 4 : 0];
      const int k = kType == 1 ? i % 4 : i / 2;
      const uint32_t w = k == 0 ? q.x : k == 1 ? q.y : k == 2 ? q.z : q.w;
      if constexpr (kType == 1) f[i] = __uint_as_float(w);
      else if constexpr (kType == 0) f[i] = __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
      else f[i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(i & 1 ? w >> 16 : w)));
      f[i] = bounded(f[i]);
    }
  }
  // Tokens [j, j + 8), -infinity outside the row
  __device__ void eight(int64_t j, float (&f)[8]) const {
    if (j >= 0 && j + 8 <= V && (reinterpret_cast<uintptr_t>(data + j * kSize) & 15u) == 0) {
      unpack(raw(j), f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = j + i >= 0 && j + i < V ? at(j + i) : -INFINITY;
    }
  }
};

// The sequence of a row (a wave's lanes together), B: none.
__device__ __forceinline__ int sequence_of(const DraftParams& p, int row) {
  int n = 0;
  for (int i = 0; i < p.B; i += 64) {
    const int b = i + lane_id();
    n += __popcll(__ballot(b < p.B && p.starts[b + 1] <= row));
  }
  n = __builtin_amdgcn_readfirstlane(n);
  return n < p.B && p.starts[n] <= row ? n : p.B;
}
// 0: greedy (a temperature that is not above zero, NaN among them); bounded so that its inverse stays in fp32's range
__device__ __forceinline__ float temperature_of(const DraftParams& p, int b) {
  const float t = p.temperature ? p.temperature[b] : 1.0f;
  return t > 0.0f ? fminf(fmaxf(t, 1e-30f), 1e30f) : 0.0f;
}
// 2^((l - top) scale), scale = log2 e / temperature, in 64 bits: the power's whole part as an exponent, 2^f for |f| <= 1/2 by its
// Taylor series up to f^11 (what follows is under 7e-15 of it).  Zero for l = -infinity.
__device__ __forceinline__ double weight(float l, float top, double scale) {
  const double z = fmax((static_cast<double>(l) - static_cast<double>(top)) * scale, -1100.0);
  const double n = rint(z), f = z - n;
  constexpr double kLn2 = 0.6931471805599453;
  constexpr double k2 = kLn2 * kLn2 / 2, k3 = k2 * kLn2 / 3, k4 = k3 * kLn2 / 4, k5 = k4 * kLn2 / 5, k6 = k5 * kLn2 / 6,
                   k7 = k6 * kLn2 / 7, k8 = k7 * kLn2 / 8, k9 = k8 * kLn2 / 9, k10 = k9 * kLn2 / 10, k11 = k10 * kLn2 / 11;
  double y = fma(k11, f, k10);
  y = fma(y, f, k9);
  y = fma(y, f, k8);
  y = fma(y, f, k7);
  y = fma(y, f, k6);
  y = fma(y, f, k5);
  y = fma(y, f, k4);
  y = fma(y, f, k3);
  y = fma(y, f, k2);
  y = fma(y, f, kLn2);
  y = fma(y, f, 1.0);
  return ldexp(y, static_cast<int>(n));
}
__device__ __forceinline__ double scale_of(float temperature) { return 1.4426950408889634 / temperature; }

struct Best {
  float top;
  int at;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.top > a.top || (b.top == a.top && b.at < a.at) ? b : a; }
__device__ __forceinline__ Best wave_best(Best a) {
  for (int o = 1; o < 64; o <<= 1) a = better(a, Best{__shfl_xor(a.top, o, 64), __shfl_xor(a.at, o, 64)});
  return a;
}
__device__ __forceinline__ double wave_sum64(double v) {
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// ------------------------------------------------------------------ every row
// Largest logit and sum of exponentials of one part of one row; y: target or drafter.  One pass: a thread keeps the largest logit
// it has seen and the sum relative to it.
template <int kType>
__global__ __launch_bounds__(256) void draft_stats_kernel(DraftParams p) {
  __shared__ Best bests[4];
  __shared__ double sums[4];
  const int split = blockIdx.x % p.splits, row = blockIdx.x / p.splits, side = blockIdx.y;
  const int b = sequence_of(p, row);
  if (b == p.B) return;
  const float t = temperature_of(p, b);
  // no token is drafted behind a sequence's last row, and greedy rows do not ask the drafter
  if (side && (t == 0.0f || row + 1 == p.starts[b + 1])) return;
  const Row<kType> data(side ? p.draft : p.target, side ? p.draft_stride : p.target_stride, row, p.V);
  const int first = split * p.split_octets, last = min(first + p.split_octets, data.eights()), tid = threadIdx.x;
  float top = kNone, sum = 0.f;
  int at = kNowhere;
  const float c = t > 0.0f ? static_cast<float>(scale_of(t)) : 0.0f;
  const auto take = [&](int o, const float (&f)[8]) {
    float m = fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
    if (t == 0.0f) {
      if (m > top || (at == kNowhere && m == top)) {
        top = m;
#pragma unroll
        for (int i = 7; i >= 0; --i)
          if (f[i] == m) at = data.first(o) + i;
      }
      return;
    }
    if (m > top) {
      sum *= exp2f((top - m) * c);
      top = m;
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i & 1] += __builtin_amdgcn_exp2f((f[i] - top) * c);
    sum += s[0] + s[1];
  };
  // the eights inside the row, four loads in flight; its ends
  const int inner0 = max(first, data.ahead ? 1 : 0), inner1 = min(last, (p.V + data.ahead) / 8);
  int o = inner0 + tid;
  for (; o + 768 < inner1; o += 1024) {
    typename Row<kType>::Raw r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = data.raw(data.first(o + 256 * i));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[8];
      Row<kType>::unpack(r[i], f);
      take(o + 256 * i, f);
    }
  }
  for (; o < inner1; o += 256) {
    float f[8];
    Row<kType>::unpack(data.raw(data.first(o)), f);
    take(o, f);
  }
  for (int e = 0; e < 2; ++e) {
    const int end = e ? data.eights() - 1 : 0;
    const bool partial = end < inner0 || end >= inner1;  // not taken above
    if (tid == 64 * e && end >= first && end < last && partial && (e == 0 || end > 0)) {
      float f[8];
      data.eight(data.first(end), f);
      take(end, f);
    }
  }
  // join the threads
  Best best = wave_best(Best{top, at});
  if ((tid & 63) == 0) bests[tid >> 6] = best;
  __syncthreads();
  best = better(better(bests[0], bests[1]), better(bests[2], bests[3]));
  const double s = wave_sum64(static_cast<double>(sum) * static_cast<double>(exp2f((top - best.top) * c)));
  if ((tid & 63) == 0) sums[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    DraftStats r;
    r.top = best.top;
    r.at = best.at;
    r.sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    p.stats[(static_cast<int64_t>(side) * p.rows + row) * p.splits + split] = r;
  }
}

struct Whole {
  float top;
  int at;
  double sum;
};
// A row's parts joined by one wave.
__device__ __forceinline__ Whole joined(const DraftParams& p, int side, int row, float t) {
  const DraftStats* s = p.stats + (static_cast<int64_t>(side) * p.rows + row) * p.splits;
  Best best{kNone, kNowhere};
  for (int i = lane_id(); i < p.splits; i += 64) best = better(best, Best{s[i].top, s[i].at});
  best = wave_best(best);
  double sum = 0.0;
  if (t > 0.0f) {
    const double scale = scale_of(t);
    for (int i = lane_id(); i < p.splits; i += 64) sum += s[i].sum * weight(s[i].top, best.top, scale);
    sum = wave_sum64(sum);
  }
  return Whole{best.top, best.at, sum};
}

// One workgroup a sequence, a wave a row: how many drafted tokens are accepted, and the row that the next one is drawn from.
// Greedy sequences are done here.
constexpr int kChooseWaves = 16;
template <int kType>
__global__ __launch_bounds__(64 * kChooseWaves) void draft_choose_kernel(DraftParams p) {
  __shared__ int stop;
  const int b = blockIdx.x, wave = threadIdx.x >> 6;
  const int start = clampi(p.starts[b], 0, p.rows), n = clampi(p.starts[b + 1], start, p.rows) - start;
  const float t = temperature_of(p, b);
  if (n == 0) {
    if (threadIdx.x == 0) {
      p.accepted[b] = 0;
      p.token[b] = -1;
      p.choice[b].row = -1;
    }
    return;
  }
  if (threadIdx.x == 0) stop = n - 1;
  __syncthreads();
  for (int i0 = 0; i0 < n - 1; i0 += kChooseWaves) {
    const int i = i0 + wave, row = start + i;
    if (i < n - 1) {
      const int x = p.drafted[row];
      const bool inside = x >= 0 && x < p.V;
      const Whole target = joined(p, 0, row, t);
      bool accepted;
      if (t == 0.0f) {
        accepted = inside && x == target.at && p.uniforms[row] < 1.0f;
      } else {
        const double scale = scale_of(t);
        const auto chance = [&](const void* data, int64_t stride, const Whole& r) {
          return inside && r.sum > 0.0 ? weight(Row<kType>(data, stride, row, p.V).at(x), r.top, scale) / r.sum : 0.0;
        };
        const double px = chance(p.target, p.target_stride, target);
        const double qx = p.draft ? chance(p.draft, p.draft_stride, joined(p, 1, row, t)) : 1.0;
        accepted = static_cast<double>(p.uniforms[row]) * qx < px;
      }
      if (!accepted && lane_id() == 0) atomicMin(&stop, i);
    }
    __syncthreads();
    if (stop < i0 + kChooseWaves) break;
  }
  __syncthreads();
  const int row = start + stop;
  if (wave == 0) {
    const Whole target = joined(p, 0, row, t);
    const bool rejected = stop < n - 1;
    float draft_top = kNone;
    if (rejected && p.draft && t > 0.0f) draft_top = joined(p, 1, row, t).top;
    if (lane_id() == 0) {
      p.accepted[b] = stop;
      DraftChoice c;
      c.row = row;
      c.has_draft = rejected;
      c.target_top = target.top;
      c.draft_top = draft_top;
      if (t == 0.0f) {
        // the largest logit's first token; none where every logit is -infinity
        p.token[b] = target.at == kNowhere ? -1 : target.at;
        c.row = -1;
      }
      p.choice[b] = c;
    }
  }
}

// ------------------------------------------------------------------ the rows that tokens are drawn from
// Their norms in 64 bits, a part a workgroup; y: target or drafter.
template <int kType>
__global__ __launch_bounds__(256) void draft_norm_kernel(DraftParams p) {
  __shared__ double sums[4];
  const int part = blockIdx.x % p.parts, b = blockIdx.x / p.parts, side = blockIdx.y, tid = threadIdx.x;
  const DraftChoice c = p.choice[b];
  if (c.row < 0 || !c.has_draft) return;
  const double scale = scale_of(temperature_of(p, b));
  const Row<kType> data(side ? p.draft : p.target, side ? p.draft_stride : p.target_stride, c.row, p.V);
  const float top = side ? c.draft_top : c.target_top;
  double sum = 0.0;
  for (int o = part * p.part_octets + tid; o < min((part + 1) * p.part_octets, data.eights()); o += 256) {
    float f[8];
    data.eight(data.first(o), f);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += weight(f[i], top, scale);
  }
  sum = wave_sum64(sum);
  if ((tid & 63) == 0) sums[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) p.norms[(static_cast<int64_t>(side) * p.B + b) * p.parts + part] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// What a chosen row's tokens weigh: w_j = p_j - q_j where that is above zero.
template <int kType>
struct Residual {
  Row<kType> target, draft;
  float target_top, draft_top;
  double scale, by_target, by_draft;  // 1 / norm, 0 where the row has nothing
  bool both;                          // the drafter's distribution is taken off
  int one;                            // the token that the drafter chose outright, -1: none

  __device__ static double norm(const DraftParams& p, int side, int b) {
    const double* n = p.norms + (static_cast<int64_t>(side) * p.B + b) * p.parts;
    double sum = 0.0;
    for (int i = lane_id(); i < p.parts; i += 64) sum += n[i];
    return wave_sum64(sum);
  }
  __device__ Residual(const DraftParams& p, int b, const DraftChoice& c)
      : target(p.target, p.target_stride, c.row, p.V), draft(p.draft ? p.draft : p.target, p.draft ? p.draft_stride : p.target_stride, c.row, p.V),
        target_top(c.target_top), draft_top(c.draft_top), scale(scale_of(temperature_of(p, b))), by_target(1.0), by_draft(0.0),
        both(c.has_draft && p.draft), one(c.has_draft && !p.draft ? p.drafted[c.row] : -1) {
    if (both) {
      const double a = norm(p, 0, b), d = norm(p, 1, b);
      by_target = a > 0.0 ? 1.0 / a : 0.0;
      by_draft = d > 0.0 ? 1.0 / d : 0.0;
    }
  }
  // Weights of tokens [j, j + 8): the target's own and what is left of them.
  __device__ void eight(int64_t j, double (&whole)[8], double (&left)[8]) const {
    float f[8], g[8];
    target.eight(j, f);
    if (both) draft.eight(j, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      whole[i] = weight(f[i], target_top, scale) * by_target;
      left[i] = j + i == one ? 0.0 : whole[i];
      if (both) left[i] = fmax(whole[i] - weight(g[i], draft_top, scale) * by_draft, 0.0);
    }
  }
};

template <int kType>
__global__ __launch_bounds__(256) void draft_parts_kernel(DraftParams p) {
  __shared__ double sums[2][4];
  __shared__ int lasts[2][4];
  const int part = blockIdx.x % p.parts, b = blockIdx.x / p.parts, tid = threadIdx.x;
  const DraftChoice c = p.choice[b];
  if (c.row < 0) return;
  const Residual<kType> r(p, b, c);
  double sl = 0.0, sw = 0.0;
  int ll = -1, lw = -1;
  for (int o = part * p.part_octets + tid; o < min((part + 1) * p.part_octets, r.target.eights()); o += 256) {
    double whole[8], left[8];
    const int j = r.target.first(o);
    r.eight(j, whole, left);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sl += left[i];
      sw += whole[i];
      if (left[i] > 0.0) ll = j + i;
      if (whole[i] > 0.0) lw = j + i;
    }
  }
  sl = wave_sum64(sl);
  sw = wave_sum64(sw);
  for (int o = 1; o < 64; o <<= 1) {
    ll = max(ll, __shfl_xor(ll, o, 64));
    lw = max(lw, __shfl_xor(lw, o, 64));
  }
  if ((tid & 63) == 0) {
    sums[0][tid >> 6] = sl;
    sums[1][tid >> 6] = sw;
    lasts[0][tid >> 6] = ll;
    lasts[1][tid >> 6] = lw;
  }
  __syncthreads();
  if (tid == 0) {
    DraftPart d;
    d.left = (sums[0][0] + sums[0][1]) + (sums[0][2] + sums[0][3]);
    d.whole = (sums[1][0] + sums[1][1]) + (sums[1][2] + sums[1][3]);
    d.last_left = max(max(lasts[0][0], lasts[0][1]), max(lasts[0][2], lasts[0][3]));
    d.last_whole = max(max(lasts[1][0], lasts[1][1]), max(lasts[1][2], lasts[1][3]));
    p.part[static_cast<int64_t>(b) * p.parts + part] = d;
  }
}

// Running sum over a workgroup's 256 threads, a thread's own included, from `base` on; `waves`: its four waves' sums.
__device__ __forceinline__ double running_sum(double own, double base, double* waves) {
  double sum = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double v = __shfl_up(sum, o, 64);
    if (lane_id() >= o) sum += v;
  }
  __syncthreads();
  if (lane_id() == 63) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  for (int w = 0; w < static_cast<int>(threadIdx.x >> 6); ++w) base += waves[w];
  return base + sum;
}

// One workgroup a sequence: the part in which the running sum passes u times the whole, then the token in it.
template <int kType>
__global__ __launch_bounds__(256) void draft_token_kernel(DraftParams p) {
  __shared__ double waves[4];
  __shared__ double totals[2][4];
  __shared__ double base;
  __shared__ int lasts[4], found, chosen;
  const int b = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
  const DraftChoice c = p.choice[b];
  if (c.row < 0) return;
  const DraftPart* parts = p.part + static_cast<int64_t>(b) * p.parts;  // at most 256
  DraftPart own{0.0, 0.0, -1, -1};
  if (tid < p.parts) own = parts[tid];
  const double left = wave_sum64(own.left), whole = wave_sum64(own.whole);
  if ((tid & 63) == 0) {
    totals[0][wave] = left;
    totals[1][wave] = whole;
  }
  if (tid == 0) chosen = kNowhere;
  __syncthreads();
  const double all_left = (totals[0][0] + totals[0][1]) + (totals[0][2] + totals[0][3]);
  const bool use_left = all_left > 0.0;
  const double total = use_left ? all_left : (totals[1][0] + totals[1][1]) + (totals[1][2] + totals[1][3]);
  const double mine = use_left ? own.left : own.whole;
  int last = use_left ? own.last_left : own.last_whole;
  const int own_last = last;
  for (int o = 1; o < 64; o <<= 1) last = max(last, __shfl_xor(last, o, 64));
  if ((tid & 63) == 0) lasts[wave] = last;
  const double goal = static_cast<double>(p.uniforms[c.has_draft ? c.row + 1 : c.row]) * total;
  const double run = running_sum(mine, 0.0, waves);
  if (run > goal) atomicMin(&chosen, tid);
  __syncthreads();
  if (tid == chosen) {
    found = own_last;  // where rounding hides the place
    base = run - mine;
  }
  if (chosen == kNowhere && tid == 0) found = max(max(lasts[0], lasts[1]), max(lasts[2], lasts[3]));
  __syncthreads();
  if (chosen != kNowhere) {
    const Residual<kType> r(p, b, c);
    const int end = min((chosen + 1) * p.part_octets, r.target.eights());
    const int each = (p.part_octets + 255) / 256, first = chosen * p.part_octets + tid * each;
    double sum = 0.0;
    for (int o = first; o < min(first + each, end); ++o) {
      double w[8], l[8];
      r.eight(r.target.first(o), w, l);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += use_left ? l[i] : w[i];
    }
    const double until = running_sum(sum, base, waves);
    if (until > goal) {
      double at = until - sum;
      for (int o = first; o < min(first + each, end); ++o) {
        double w[8], l[8];
        const int j = r.target.first(o);
        r.eight(j, w, l);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double v = use_left ? l[i] : w[i];
          at += v;
          if (at > goal && v > 0.0) atomicMin(&found, j + i);
        }
      }
    }
    __syncthreads();
  }
  if (tid == 0) p.token[b] = found;
}

template <int kType>
void launch(const DraftParams& p, hipStream_t stream) {
  const int sides = p.draft ? 2 : 1;
  if (p.rows) hipLaunchKernelGGL(draft_stats_kernel<kType>, dim3(p.rows * p.splits, sides), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(draft_choose_kernel<kType>, dim3(p.B), dim3(64 * kChooseWaves), 0, stream, p);
  if (!p.rows) return;
  if (p.draft) hipLaunchKernelGGL(draft_norm_kernel<kType>, dim3(p.B * p.parts, 2), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(draft_parts_kernel<kType>, dim3(p.B * p.parts), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(draft_token_kernel<kType>, dim3(p.B), dim3(256), 0, stream, p);
}

}  // namespace

void launch_verify_drafts(const DraftParams& p, hipStream_t stream) {
  if (p.dtype == 0) launch<0>(p, stream);
  else if (p.dtype == 1) launch<1>(p, stream);
  else launch<2>(p, stream);
}

}  // namespace dflash
