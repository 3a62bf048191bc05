// Check of drafted tokens against the target's probabilities from given random numbers (speculative sampling).
//
// Sequence b has rows [starts[b], starts[b + 1]); row r predicts the token behind row r, and drafted[r] is the drafter's
// choice for it (the last row has none).  With p and q the softmaxes of the target's and the drafter's logits over the
// temperature, x = drafted[r] and u = uniforms[r]:  x is accepted iff u q(x) < p(x).  The first row r that is not accepted
// draws its token from max(p - q, 0), the last row from p, both by the inverse of the running sum with the uniform of the
// row behind (r + 1, which tests nothing then) or of the last row itself.  So the tokens follow the target's distribution
// whatever the drafter's is.
//
// A whole number hangs on a comparison, so what decides carries 64 bits, weights and sums.  In the rows that tokens are drawn
// from that is every weight, since one of 2.5e5 running sums lies within 1e-7 of a given number once in forty times.  The
// acceptance test compares one number a row: sums of 32-bit exponentials tell on which side it is, but once in 3e4 rows or so, and
// those rows are summed again.  So what is accepted depends on the row alone, not on how the rows of a call are cut.
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
// it has seen and the sum relative to `base`, which follows in steps of a factor of 2^16 at least, so that a row which rises all along
// does not round the sum again and again.  The exponentials have 32 bits, eight are added in 32 and those sums in 64.  How far a
// row's sum is off: an exponential of z = (l - base) c by the three roundings of z, 2.1 |z| 2^-24, and two of its own, the sum of eight by
// four; |z| is at most 32 (16 and `base`'s own rounding) or what the weight 2^-y of the token says, so up to y = 40 that is
// (6 + 2.1 * 40) 2^-24 < 2^-17, and all the tokens that weigh less add nothing to it.
// Bound by memory: 478 MB of logits (513 rows and their drafter's, 248 320 tokens in bf16) 86 us, 5.6 TB/s with what the last-level cache
// holds (83 with sums of 32 bits).
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
  float top = kNone, base = kNone;
  double sum = 0.0;
  int at = kNowhere;
  const float c = t > 0.0f ? static_cast<float>(scale_of(t)) : 0.0f, ahead = t > 0.0f ? 16.0f / c : 0.0f;
  const auto most = [](const float (&f)[8]) {
    return fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
  };
  const auto find = [&](int o, const float (&f)[8]) {
    const float m = most(f);
    if (m < top) return;
    int place = kNowhere;
#pragma unroll
    for (int i = 7; i >= 0; --i)
      if (f[i] == m) place = data.first(o) + i;
    // by places, not by the order of visits: a row's first eight, where it is not whole, is seen last
    if (m > top || place < at) at = place;
    top = m;
  };
  const auto add = [&](int, const float (&f)[8]) {
    const float m = most(f);
    top = fmaxf(top, m);
    if (m > base + ahead) {
      sum *= static_cast<double>(exp2f((base - m) * c));
      base = m;
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i & 1] += __builtin_amdgcn_exp2f((f[i] - base) * c);
    sum += static_cast<double>(s[0] + s[1]);
  };
  // the eights inside the row, four loads in flight; its ends
  const int inner0 = max(first, data.ahead ? 1 : 0), inner1 = min(last, (p.V + data.ahead) / 8);
  const auto walk = [&](auto take) {
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
    {
      typename Row<kType>::Raw r[3];
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (o + 256 * i < inner1) r[i] = data.raw(data.first(o + 256 * i));
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (o + 256 * i < inner1) {
          float f[8];
          Row<kType>::unpack(r[i], f);
          take(o + 256 * i, f);
        }
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
  };
  if (t == 0.0f) walk(find);
  else walk(add);
  // join the threads
  Best best = wave_best(Best{top, at});
  if ((tid & 63) == 0) bests[tid >> 6] = best;
  __syncthreads();
  best = better(better(bests[0], bests[1]), better(bests[2], bests[3]));
  const double s = t > 0.0f ? wave_sum64(sum * weight(base, best.top, scale_of(t))) : 0.0;
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
// Greedy sequences are done here.  A chain of dependent loads: one row 3.2 us, a block of 16 rows 6.3, 64 blocks 7.7; with a wave for each of
// 16 rows, since four waves take their rows in turn.  A row whose test the sums of 32-bit exponentials leave open is summed again in 64 bits by the
// whole workgroup, in an order of the tokens' places alone (50 us for a row of 248 320 tokens, the drafter's as long).
constexpr int kChooseWaves = 16;
constexpr double kDoubt = 0x1p-15;  // both sides' sums are off by less than 2^-17
enum Outcome : int { kAccepted, kRejected, kOpen };
template <int kType>
__global__ __launch_bounds__(64 * kChooseWaves) void draft_choose_kernel(DraftParams p) {
  __shared__ DraftChoice choices[kChooseWaves];
  __shared__ int largest[kChooseWaves], outcomes[kChooseWaves];
  __shared__ double sums[2][kChooseWaves];
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
  const double scale = t > 0.0f ? scale_of(t) : 0.0;
  // whether u q(x) < p(x), where the sums of the row's weights are known
  const auto test = [&](int row, int x, float target_top, double target_sum, bool ask, float draft_top, double draft_sum) {
    const auto chance = [&](const void* data, int64_t stride, float top, double sum) {
      return x >= 0 && x < p.V && sum > 0.0 ? weight(Row<kType>(data, stride, row, p.V).at(x), top, scale) / sum : 0.0;
    };
    const double px = chance(p.target, p.target_stride, target_top, target_sum);
    const double qx = (ask ? chance(p.draft, p.draft_stride, draft_top, draft_sum) : 1.0) * static_cast<double>(p.uniforms[row]);
    return fabs(px - qx) < kDoubt * fmax(px, qx) ? make_int2(qx < px, kOpen) : make_int2(qx < px, qx < px ? kAccepted : kRejected);
  };
  int i0 = 0, stop = -1;
  for (;; i0 += kChooseWaves) {
    const int i = i0 + wave, row = start + i;
    if (i < n) {
      const bool drafted = i < n - 1, ask = drafted && p.draft && t > 0.0f;
      const Whole target = joined(p, 0, row, t);
      Whole draft{kNone, kNowhere, 0.0};
      if (ask) draft = joined(p, 1, row, t);
      int outcome = kRejected;
      if (drafted) {
        const int x = p.drafted[row];
        if (t == 0.0f) outcome = x >= 0 && x < p.V && x == target.at && p.uniforms[row] < 1.0f ? kAccepted : kRejected;
        else outcome = test(row, x, target.top, target.sum, ask, draft.top, draft.sum).y;
      }
      if (lane_id() == 0) {
        choices[wave] = DraftChoice{row, drafted, target.top, draft.top};
        largest[wave] = target.at;
        outcomes[wave] = outcome;
      }
    }
    __syncthreads();
    const int own = lane_id() < min(kChooseWaves, n - i0) ? outcomes[lane_id()] : kAccepted;
    for (uint64_t held = __ballot(own != kAccepted); held; held &= held - 1) {  // the same in all waves
      const int w = __ffsll(static_cast<unsigned long long>(held)) - 1;
      const DraftChoice c = choices[w];
      bool accepted = false;
      if (__shfl(own, w, 64) == kOpen) {
        for (int side = 0; side < (p.draft ? 2 : 1); ++side) {
          const Row<kType> data(side ? p.draft : p.target, side ? p.draft_stride : p.target_stride, c.row, p.V);
          double sum = 0.0;
#pragma unroll 4
          for (int j = threadIdx.x; j < p.V; j += 64 * kChooseWaves) sum += weight(data.at(j), side ? c.draft_top : c.target_top, scale);
          sum = wave_sum64(sum);
          if (lane_id() == 0) sums[side][wave] = sum;
        }
        __syncthreads();
        double whole[2] = {0.0, 0.0};
        for (int k = 0; k < kChooseWaves; ++k) {
          whole[0] += sums[0][k];
          if (p.draft) whole[1] += sums[1][k];
        }
        accepted = test(c.row, p.drafted[c.row], c.target_top, whole[0], p.draft != nullptr, c.draft_top, whole[1]).x;
        __syncthreads();
      }
      if (!accepted) {  // at the last row at the latest
        stop = i0 + w;
        break;
      }
    }
    if (stop >= 0) break;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    DraftChoice c = choices[stop - i0];
    p.accepted[b] = stop;
    if (t == 0.0f) {
      // the largest logit's first token; none where every logit is -infinity
      const int at = largest[stop - i0];
      p.token[b] = at == kNowhere ? -1 : at;
      c.row = -1;
    }
    p.choice[b] = c;
  }
}

// ------------------------------------------------------------------ the rows that tokens are drawn from
// Their norms in 64 bits, four parts a workgroup; y: target or drafter.  Bound by the 64-bit exponentials, some twenty
// instructions each: 32 million of 64 sequences 28 us, as many again in the parts below 34.
template <int kType>
__global__ __launch_bounds__(256) void draft_norm_kernel(DraftParams p) {
  __shared__ double sums[4];
  const int groups = p.parts / 4, group = blockIdx.x % groups, b = blockIdx.x / groups, side = blockIdx.y, tid = threadIdx.x;
  const DraftChoice c = p.choice[b];
  if (c.row < 0 || !c.has_draft) return;
  const double scale = scale_of(temperature_of(p, b));
  const Row<kType> data(side ? p.draft : p.target, side ? p.draft_stride : p.target_stride, c.row, p.V);
  const float top = side ? c.draft_top : c.target_top;
  const int last = min(4 * (group + 1) * p.part_octets, data.eights());
  double sum = 0.0;
  for (int o = 4 * group * p.part_octets + tid; o < last; o += 256) {
    float f[8];
    data.eight(data.first(o), f);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += weight(f[i], top, scale);
  }
  sum = wave_sum64(sum);
  if (lane_id() == 0) sums[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) p.norms[(static_cast<int64_t>(side) * p.B + b) * groups + group] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// What a chosen row's tokens weigh, in units of its largest logit's weight: e_j - f_j norm(e) / norm(f) where that is above zero, e
// and f the target's and the drafter's weights.
template <int kType>
struct Residual {
  Row<kType> target, draft;
  float target_top, draft_top;
  double scale, ratio;  // norm(e) / norm(f), 0 where the drafter's row has nothing
  bool both;            // the drafter's distribution is taken off
  int one;              // the token that the drafter chose outright, -1: none

  __device__ Residual(const DraftParams& p, int b, const DraftChoice& c)
      : target(p.target, p.target_stride, c.row, p.V), draft(p.draft ? p.draft : p.target, p.draft ? p.draft_stride : p.target_stride, c.row, p.V),
        target_top(c.target_top), draft_top(c.draft_top), scale(scale_of(temperature_of(p, b))), ratio(0.0), both(c.has_draft && p.draft),
        one(c.has_draft && !p.draft ? p.drafted[c.row] : -1) {}
  // The ratio from the parts of the norms (a wave's lanes together)
  __device__ void find_ratio(const DraftParams& p, int b) {
    const int groups = p.parts / 4;  // at most 64
    const double* n = p.norms + static_cast<int64_t>(b) * groups;
    const int i = min(lane_id(), groups - 1);
    double e = n[i], f = n[static_cast<int64_t>(p.B) * groups + i];
    if (lane_id() >= groups) e = f = 0.0;
    for (int o = 1; o < 64; o <<= 1) {
      e += __shfl_xor(e, o, 64);
      f += __shfl_xor(f, o, 64);
    }
    ratio = f > 0.0 ? e / f : 0.0;
  }
  // Weight of one token: what is left of the target's, or its own.
  __device__ double one_of(float f, float g, int j, bool use_left) const {
    const double own = weight(f, target_top, scale);
    if (!use_left) return own;
    if (both) return fmax(fma(-ratio, weight(g, draft_top, scale), own), 0.0);
    return j == one ? 0.0 : own;
  }
  // Sum of what is left of a wave's eights o, o + 64, ... before `last`, by lanes.
  __device__ double sum(int o, int last) const {
    float f[8], g[8];
    double s[2] = {0.0, 0.0};
    if (both) {
      for (; o < last; o += 64) {
        target.eight(target.first(o), f);
        draft.eight(target.first(o), g);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i & 1] += fmax(fma(-ratio, weight(g[i], draft_top, scale), weight(f[i], target_top, scale)), 0.0);
      }
    } else {
      for (; o < last; o += 64) {
        const int j = target.first(o);
        target.eight(j, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i & 1] += j + i == one ? 0.0 : weight(f[i], target_top, scale);
      }
    }
    return s[0] + s[1];
  }
};

// Sums of what is left, a part a wave.
template <int kType>
__global__ __launch_bounds__(256) void draft_parts_kernel(DraftParams p) {
  const int unit = blockIdx.x * 4 + (threadIdx.x >> 6), part = unit % p.parts, b = unit / p.parts;
  const DraftChoice c = p.choice[b];
  if (c.row < 0) return;
  Residual<kType> r(p, b, c);
  if (r.both) r.find_ratio(p, b);
  if (part == 0 && lane_id() == 0) p.ratio[b] = r.ratio;
  const double sum = wave_sum64(r.sum(part * p.part_octets + lane_id(), min((part + 1) * p.part_octets, r.target.eights())));
  if (lane_id() == 0) p.left[static_cast<int64_t>(b) * p.parts + part] = sum;
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

// One workgroup a sequence: the part in which the running sum passes u times the whole, then the token in it.  Where nothing is
// left (the drafter's distribution is the target's, to the roundings) the same with the target's own weights, over the whole row.
// The chain of choice, parts, logits, 64-bit weights and the search: one row 8.9 us, one block 12.3, 64 blocks 14.5.
template <int kType>
__global__ __launch_bounds__(256) void draft_token_kernel(DraftParams p) {
  __shared__ double waves[4], base;
  __shared__ int found, last, chosen;
  __shared__ float logits[2][8][256];
  const int b = blockIdx.x, tid = threadIdx.x;
  const DraftChoice c = p.choice[b];
  if (c.row < 0) return;
  Residual<kType> r(p, b, c);
  r.ratio = p.ratio[b];
  const double u = static_cast<double>(p.uniforms[c.has_draft ? c.row + 1 : c.row]);
  // Walks over eights [from, to), 2048 tokens at a time, eight neighbours a thread, from the sum `before` on: the first token at
  // which the sum exceeds `goal` into `found`, the last that weighs anything into `last`; returns the sum at the end.  The
  // weights are made in loops that stay loops: straight code would run once, and fetching it takes longer than running it.
  const auto walk = [&](int from, int to, double before, double goal, bool use_left) {
    for (int o0 = from; o0 < to; o0 += 256) {
      const int o = o0 + tid, j = r.target.first(o);
      double sum = 0.0;
      int held = -1;
      if (o < to) {
        float f[8];
        r.target.eight(j, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) logits[0][i][tid] = f[i];
        if (r.both) {
          r.draft.eight(j, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) logits[1][i][tid] = f[i];
        }
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const double v = r.one_of(logits[0][i][tid], logits[1][i][tid], j + i, use_left);
          sum += v;
          if (v > 0.0) held = j + i;
        }
      }
      const double until = running_sum(sum, before, waves);
      if (held >= 0) atomicMax(&last, held);
      if (until > goal && held >= 0) {
        double at = until - sum;
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const double v = r.one_of(logits[0][i][tid], logits[1][i][tid], j + i, use_left);
          at += v;
          if ((at > goal && v > 0.0) || j + i == held) {  // its last one where rounding hides the place
            atomicMin(&found, j + i);
            break;
          }
        }
      }
      before += (waves[0] + waves[1]) + (waves[2] + waves[3]);
      if (before > goal) break;
    }
    __syncthreads();
    return before;
  };
  const int eights = r.target.eights();
  const double mine = tid < p.parts ? p.left[static_cast<int64_t>(b) * p.parts + tid] : 0.0;  // at most 256 parts
  if (tid == 0) {
    found = kNowhere;
    chosen = kNowhere;
    last = -1;
  }
  const double run = running_sum(mine, 0.0, waves);
  const double total = (waves[0] + waves[1]) + (waves[2] + waves[3]);
  if (total > 0.0) {
    const double goal = u * total;
    if (run > goal && mine > 0.0) atomicMin(&chosen, tid);
    __syncthreads();
    if (tid == chosen) base = run - mine;
    __syncthreads();
    // Added up token by token the part's end may come out a rounding lower than its sum, and not above the goal: then the part's last
    // token is the one, and `last` holds it.  Where no part's sum exceeds the goal (a random number of one or above) it is the row's.
    if (chosen != kNowhere) walk(chosen * p.part_octets, min((chosen + 1) * p.part_octets, eights), base, goal, true);
    else walk(0, eights, 0.0, INFINITY, true);
  } else {
    const double whole = walk(0, eights, 0.0, INFINITY, false);
    if (whole > 0.0) walk(0, eights, 0.0, u * whole, false);
  }
  if (tid == 0) p.token[b] = found != kNowhere ? found : last;
}

template <int kType>
void launch(const DraftParams& p, hipStream_t stream) {
  const int sides = p.draft ? 2 : 1;
  if (p.rows) hipLaunchKernelGGL(draft_stats_kernel<kType>, dim3(p.rows * p.splits, sides), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(draft_choose_kernel<kType>, dim3(p.B), dim3(64 * kChooseWaves), 0, stream, p);
  if (!p.rows) return;
  if (p.draft) hipLaunchKernelGGL(draft_norm_kernel<kType>, dim3(p.B * p.parts / 4, 2), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(draft_parts_kernel<kType>, dim3(p.B * p.parts / 4), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(draft_token_kernel<kType>, dim3(p.B), dim3(256), 0, stream, p);
}

}  // namespace

void launch_verify_drafts(const DraftParams& p, hipStream_t stream) {
  if (p.dtype == 0) launch<0>(p, stream);
  else if (p.dtype == 1) launch<1>(p, stream);
  else launch<2>(p, stream);
}

}  // namespace dflash
