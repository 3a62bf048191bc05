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

__device__ __forceinline__ float element(const void* row, int dtype, int64_t i) {
  float v;
  if (dtype == 1) {
    v = static_cast<const float*>(row)[i];
  } else {
    const uint16_t w = static_cast<const uint16_t*>(row)[i];
    v = dtype == 0 ? bf16_to_f32(w) : static_cast<float>(__builtin_bit_cast(_Float16, w));
  }
  return fminf(fmaxf(v, -INFINITY), FLT_MAX);
}

// Tokens [j, j + 8) of a row of V, -infinity outside it; 16-byte loads where they lie so.
__device__ __forceinline__ void load8(const void* row, int dtype, int64_t j, int V, float (&f)[8]) {
  const int size = dtype == 1 ? 4 : 2;
  const char* at = static_cast<const char*>(row) + j * size;
  if (j >= 0 && j + 8 <= V && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
    const uint4 a = *reinterpret_cast<const uint4*>(at);
    if (dtype == 1) {
      const uint4 b = *reinterpret_cast<const uint4*>(at + 16);
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    } else {
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (dtype == 0) {
          f[2 * i] = __uint_as_float(w[i] << 16);
          f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
          f[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i])));
          f[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] >> 16)));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = fminf(fmaxf(f[i], -INFINITY), FLT_MAX);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = j + i >= 0 && j + i < V ? element(row, dtype, j + i) : -INFINITY;
}

// Tokens that a row's first eight starts before the row itself, so that all but the first and last eights are aligned.
__device__ __forceinline__ int lead(const void* row, int dtype) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / (dtype == 1 ? 4 : 2));
}

__device__ __forceinline__ const void* row_of(const void* data, int dtype, int64_t stride, int row) {
  return static_cast<const char*>(data) + row * stride * (dtype == 1 ? 4 : 2);
}

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
// exp((l - top) / t) in 64 bits
__device__ __forceinline__ double weight(float l, float top, double inverse) {
  const double z = (static_cast<double>(l) - static_cast<double>(top)) * inverse;
  return l == top ? 1.0 : l == -INFINITY ? 0.0 : exp(z);
}

struct Best {
  float top;
  int at;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.top > a.top || (b.top == a.top && b.at < a.at) ? b : a; }

// Largest logit and sum of exponentials of one part of one row; y: target or drafter.
__global__ __launch_bounds__(256) void draft_stats_kernel(DraftParams p) {
  __shared__ float tops[4];
  __shared__ int ats[4];
  __shared__ double sums[4];
  const int split = blockIdx.x % p.splits, row = blockIdx.x / p.splits, side = blockIdx.y;
  const int b = sequence_of(p, row);
  if (b == p.B) return;
  const float t = temperature_of(p, b);
  // no token is drafted behind a sequence's last row, and greedy rows do not ask the drafter
  if (side && (t == 0.0f || row + 1 == p.starts[b + 1])) return;
  const void* data = row_of(side ? p.draft : p.target, p.dtype, side ? p.draft_stride : p.target_stride, row);
  const int first = split * p.split_octets, ahead = lead(data, p.dtype);
  const int last = min(first + p.split_octets, (p.V + ahead + 7) / 8);
  const int tid = threadIdx.x;
  float top = kNone;
  int at = 0x7FFFFFFF;
  float sum = 0.f;
  const float c = t > 0.0f ? static_cast<float>(1.4426950408889634 / t) : 0.0f;
  for (int o = first + tid; o < last; o += 256) {
    float f[8];
    load8(data, p.dtype, 8ll * o - ahead, p.V, f);
    float m = f[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, f[i]);
    if (t == 0.0f) {
      if (m > top || (at == 0x7FFFFFFF && m == top)) {
        top = m;
#pragma unroll
        for (int i = 7; i >= 0; --i)
          if (f[i] == m) at = 8 * o - ahead + i;
      }
    } else {
      if (m > top) {
        sum *= exp2f((top - m) * c);
        top = m;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += exp2f((f[i] - top) * c);
    }
  }
  // join the threads
  Best best{top, at};
  for (int o = 1; o < 64; o <<= 1) best = better(best, Best{__shfl_xor(best.top, o, 64), __shfl_xor(best.at, o, 64)});
  if ((tid & 63) == 0) {
    tops[tid >> 6] = best.top;
    ats[tid >> 6] = best.at;
  }
  __syncthreads();
  best = Best{tops[0], ats[0]};
#pragma unroll
  for (int w = 1; w < 4; ++w) best = better(best, Best{tops[w], ats[w]});
  double s = static_cast<double>(sum) * static_cast<double>(exp2f((top - best.top) * c));
  for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
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

struct Row {
  float top;
  int at;
  double sum;
};
// A row's parts joined by one wave.
__device__ __forceinline__ Row joined(const DraftParams& p, int side, int row, float t) {
  const DraftStats* s = p.stats + (static_cast<int64_t>(side) * p.rows + row) * p.splits;
  Best best{kNone, 0x7FFFFFFF};
  for (int i = lane_id(); i < p.splits; i += 64) best = better(best, Best{s[i].top, s[i].at});
  for (int o = 1; o < 64; o <<= 1) best = better(best, Best{__shfl_xor(best.top, o, 64), __shfl_xor(best.at, o, 64)});
  double sum = 0.0;
  if (t > 0.0f) {
    const double inverse = 1.0 / t;
    for (int i = lane_id(); i < p.splits; i += 64) sum += s[i].sum * weight(s[i].top, best.top, inverse);
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
  }
  return Row{best.top, best.at, sum};
}

// One workgroup a sequence: how many drafted tokens are accepted, and the row that the next one is drawn from.  Greedy
// sequences are done here.
__global__ __launch_bounds__(256) void draft_choose_kernel(DraftParams p) {
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
  for (int i0 = 0; i0 < n - 1; i0 += 4) {
    const int i = i0 + wave, row = start + i;
    if (i < n - 1) {
      const int x = p.drafted[row];
      const bool inside = x >= 0 && x < p.V;
      const Row target = joined(p, 0, row, t);
      bool accepted;
      if (t == 0.0f) {
        accepted = inside && x == target.at && p.uniforms[row] < 1.0f;
      } else {
        const double inverse = 1.0 / t;
        const auto chance = [&](const void* data, int64_t stride, const Row& r) {
          return inside && r.sum > 0.0 ? weight(element(row_of(data, p.dtype, stride, row), p.dtype, x), r.top, inverse) / r.sum : 0.0;
        };
        const double px = chance(p.target, p.target_stride, target);
        const double qx = p.draft ? chance(p.draft, p.draft_stride, joined(p, 1, row, t)) : 1.0;
        accepted = static_cast<double>(p.uniforms[row]) * qx < px;
      }
      if (!accepted && lane_id() == 0) atomicMin(&stop, i);
    }
    __syncthreads();
    if (stop < i0 + 4) break;
  }
  __syncthreads();
  const int row = start + stop;
  if (wave == 0) {
    const Row target = joined(p, 0, row, t);
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
        p.token[b] = target.at == 0x7FFFFFFF ? -1 : target.at;
        c.row = -1;
      }
      p.choice[b] = c;
    }
  }
}

// Norms of the chosen rows in 64 bits, a part a workgroup; y: target or drafter.
__global__ __launch_bounds__(256) void draft_norm_kernel(DraftParams p) {
  __shared__ double sums[4];
  const int part = blockIdx.x % p.parts, b = blockIdx.x / p.parts, side = blockIdx.y, tid = threadIdx.x;
  const DraftChoice c = p.choice[b];
  if (c.row < 0 || !c.has_draft) return;
  const double inverse = 1.0 / temperature_of(p, b);
  const void* data = row_of(side ? p.draft : p.target, p.dtype, side ? p.draft_stride : p.target_stride, c.row);
  const float top = side ? c.draft_top : c.target_top;
  const int ahead = lead(data, p.dtype);
  double sum = 0.0;
  for (int o = part * p.part_octets + tid; o < min((part + 1) * p.part_octets, (p.V + ahead + 7) / 8); o += 256) {
    float f[8];
    load8(data, p.dtype, 8ll * o - ahead, p.V, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += weight(f[i], top, inverse);
  }
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
  if ((tid & 63) == 0) sums[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) p.norms[(static_cast<int64_t>(side) * p.B + b) * p.parts + part] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// What a chosen row's tokens weigh: w_j = p_j - q_j where that is above zero.
struct Residual {
  const void *target, *draft;
  float target_top, draft_top;
  double inverse, by_target, by_draft;  // 1 / norm, 0 where the row has nothing
  int one;                              // the token that the drafter chose outright, -1: none
};
__device__ __forceinline__ double norm_of(const DraftParams& p, int side, int b) {
  const double* n = p.norms + (static_cast<int64_t>(side) * p.B + b) * p.parts;
  double sum = 0.0;
  for (int i = lane_id(); i < p.parts; i += 64) sum += n[i];
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
  return sum;
}
__device__ __forceinline__ Residual residual_of(const DraftParams& p, int b, const DraftChoice& c) {
  Residual r;
  r.target = row_of(p.target, p.dtype, p.target_stride, c.row);
  r.target_top = c.target_top;
  r.inverse = 1.0 / temperature_of(p, b);
  r.draft = nullptr;
  r.draft_top = c.draft_top;
  r.by_target = 1.0;
  r.by_draft = 0.0;
  r.one = -1;
  if (c.has_draft) {
    if (p.draft) {
      r.draft = row_of(p.draft, p.dtype, p.draft_stride, c.row);
      const double a = norm_of(p, 0, b), d = norm_of(p, 1, b);
      r.by_target = a > 0.0 ? 1.0 / a : 0.0;
      r.by_draft = d > 0.0 ? 1.0 / d : 0.0;
    } else {
      r.one = p.drafted[c.row];
    }
  }
  return r;
}
// Weights of tokens [j, j + 8): the target's own and what is left of them.
__device__ __forceinline__ void residual8(const DraftParams& p, const Residual& r, int64_t j, double (&whole)[8], double (&left)[8]) {
  float f[8];
  load8(r.target, p.dtype, j, p.V, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    whole[i] = weight(f[i], r.target_top, r.inverse) * r.by_target;
    left[i] = j + i == r.one ? 0.0 : whole[i];
  }
  if (r.draft) {
    load8(r.draft, p.dtype, j, p.V, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double d = whole[i] - weight(f[i], r.draft_top, r.inverse) * r.by_draft;
      left[i] = d > 0.0 ? d : 0.0;
    }
  }
}

__global__ __launch_bounds__(256) void draft_parts_kernel(DraftParams p) {
  __shared__ double sums[2][4];
  __shared__ int lasts[2][4];
  const int part = blockIdx.x % p.parts, b = blockIdx.x / p.parts, tid = threadIdx.x;
  const DraftChoice c = p.choice[b];
  if (c.row < 0) return;
  const Residual r = residual_of(p, b, c);
  const int ahead = lead(r.target, p.dtype);
  double sl = 0.0, sw = 0.0;
  int ll = -1, lw = -1;
  for (int o = part * p.part_octets + tid; o < min((part + 1) * p.part_octets, (p.V + ahead + 7) / 8); o += 256) {
    double whole[8], left[8];
    const int64_t j = 8ll * o - ahead;
    residual8(p, r, j, whole, left);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sl += left[i];
      sw += whole[i];
      if (left[i] > 0.0) ll = static_cast<int>(j) + i;
      if (whole[i] > 0.0) lw = static_cast<int>(j) + i;
    }
  }
  for (int o = 1; o < 64; o <<= 1) {
    sl += __shfl_xor(sl, o, 64);
    sw += __shfl_xor(sw, o, 64);
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

// One workgroup a sequence: the part in which the running sum passes u times the whole, then the token in it.
__global__ __launch_bounds__(256) void draft_token_kernel(DraftParams p) {
  __shared__ double before[256];
  __shared__ int found, chosen;
  __shared__ double base;
  const int b = blockIdx.x, tid = threadIdx.x;
  const DraftChoice c = p.choice[b];
  if (c.row < 0) return;
  const DraftPart* parts = p.part + static_cast<int64_t>(b) * p.parts;
  // every thread sums the parts alike: there are few
  double left = 0.0, whole = 0.0;
  int last_left = -1, last_whole = -1;
  for (int i = 0; i < p.parts; ++i) {
    left += parts[i].left;
    whole += parts[i].whole;
    last_left = max(last_left, parts[i].last_left);
    last_whole = max(last_whole, parts[i].last_whole);
  }
  const bool use_left = left > 0.0;
  const double total = use_left ? left : whole;
  const int last = use_left ? last_left : last_whole;
  if (last < 0) {
    if (tid == 0) p.token[b] = -1;
    return;
  }
  const double goal = static_cast<double>(p.uniforms[c.has_draft ? c.row + 1 : c.row]) * total;
  if (tid == 0) {
    int at = last;
    chosen = -1;
    double sum = 0.0;
    for (int i = 0; i < p.parts; ++i) {
      const double next = sum + (use_left ? parts[i].left : parts[i].whole);
      if (next > goal) {
        chosen = i;
        at = use_left ? parts[i].last_left : parts[i].last_whole;
        break;
      }
      sum = next;
    }
    base = sum;
    found = at;
  }
  __syncthreads();
  if (chosen >= 0) {
    const Residual r = residual_of(p, b, c);
    const int ahead = lead(r.target, p.dtype);
    const int end = min((chosen + 1) * p.part_octets, (p.V + ahead + 7) / 8);
    const int each = (p.part_octets + 255) / 256, first = chosen * p.part_octets + tid * each;
    double sum = 0.0;
    for (int o = first; o < min(first + each, end); ++o) {
      double w[8], l[8];
      residual8(p, r, 8ll * o - ahead, w, l);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += use_left ? l[i] : w[i];
    }
    before[tid] = sum;
    __syncthreads();
    double run = base;
    for (int i = 0; i < tid; ++i) run += before[i];
    if (run + sum > goal) {
      for (int o = first; o < min(first + each, end); ++o) {
        double w[8], l[8];
        residual8(p, r, 8ll * o - ahead, w, l);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double v = use_left ? l[i] : w[i];
          run += v;
          if (run > goal && v > 0.0) atomicMin(&found, static_cast<int>(8ll * o - ahead) + i);
        }
      }
    }
    __syncthreads();
  }
  if (tid == 0) p.token[b] = found;
}

}  // namespace

void launch_verify_drafts(const DraftParams& p, hipStream_t stream) {
  const int sides = p.draft ? 2 : 1;
  hipLaunchKernelGGL(draft_stats_kernel, dim3(p.rows * p.splits, sides), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(draft_choose_kernel, dim3(p.B), dim3(256), 0, stream, p);
  if (p.draft) hipLaunchKernelGGL(draft_norm_kernel, dim3(p.B * p.parts, 2), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(draft_parts_kernel, dim3(p.B * p.parts), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(draft_token_kernel, dim3(p.B), dim3(256), 0, stream, p);
}

}  // namespace dflash
