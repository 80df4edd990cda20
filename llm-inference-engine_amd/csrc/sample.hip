// One token per row of logits (ie_hip_sample_rows): temperature, top-k, min-p, top-p, then inverse
// CDF in index order at the caller's random number.
//
// A weight is exp((l - max) / T) in float64, taken to whole numbers of 2^-45 (fewer bits where n of
// them would pass 63: weight_bits): sums of whole numbers are exact, so no order of adding them
// changes a result, and a border of the sums lies where the 64-bit definition has it to within 2^-46
// of the largest weight per token.
//
// What is kept is a prefix of the tokens ordered by (logit descending, index ascending): its last key
// is found digit by digit (11 + 11 + 10 bits of the logit's ordered bit pattern) from histograms of
// counts and weights, its last index among equal logits by counting.
#include <algorithm>
#include <cmath>

#include "common.hpp"

namespace iehip {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;

// Bits of the largest weight, so that n of them stay under 2^63.
int weight_bits(int n) {
  int log2 = 0;
  while ((int64_t(1) << log2) < n) ++log2;
  return std::min(45, 63 - log2);
}

// Logits in their order as unsigned numbers; NaN below all, -0 with +0.
__device__ __forceinline__ uint32_t order_key(float l) {
  if (l != l) return 0;
  const uint32_t b = __float_as_uint(l + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Row {
  float top;     // the largest logit
  double t;      // temperature
  double least;  // min-p as a weight
  double one;    // the largest weight
};

__device__ __forceinline__ unsigned long long weight(float l, const Row& w) {
  if (!(l > -INFINITY)) return 0;
  if (w.top == INFINITY) return l == INFINITY ? static_cast<unsigned long long>(w.one) : 0ull;
  const double e = exp((double(l) - double(w.top)) / w.t);
  return e >= w.least ? static_cast<unsigned long long>(__double2ll_rn(e * w.one)) : 0ull;
}

struct Bins {
  uint32_t count[kBins];
  unsigned long long mass[kBins];
};

__global__ void __launch_bounds__(kThreads)
sample_rows_kernel(int32_t* __restrict__ out, const float* __restrict__ logits,
                   const float* __restrict__ temperature, const int32_t* __restrict__ top_k,
                   const float* __restrict__ top_p, const float* __restrict__ min_p,
                   const float* __restrict__ u, int n, double one) {
  __shared__ Bins bins;
  __shared__ float red_v[kWaves];
  __shared__ int red_i[kWaves];
  __shared__ unsigned long long red_m[kWaves];
  __shared__ uint32_t found_bin, found_left;
  __shared__ unsigned long long found_before;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* l = logits + size_t(row) * n;

  float best = -INFINITY;
  int at = 0x7fffffff;
  for (int i = tid; i < n; i += kThreads)
    if (l[i] > best) {
      best = l[i];
      at = i;
    }
  for (int off = 32; off > 0; off >>= 1) {
    const float v = __shfl_xor(best, off, 64);
    const int i = __shfl_xor(at, off, 64);
    if (v > best || (v == best && i < at)) best = v, at = i;
  }
  if (lane == 0) red_v[wave] = best, red_i[wave] = at;
  __syncthreads();
  best = red_v[0], at = red_i[0];
  for (int w = 1; w < kWaves; ++w)
    if (red_v[w] > best || (red_v[w] == best && red_i[w] < at)) best = red_v[w], at = red_i[w];
  if (at == 0x7fffffff) at = 0;
  const float temp = temperature[row];
  if (!(temp > 0.0f) || best == -INFINITY) {
    if (tid == 0) out[row] = at;
    return;
  }
  Row w;
  w.top = best;
  w.t = temp;
  w.one = one;
  const float mp = min_p ? min_p[row] : 0.0f;
  w.least = mp > 0.0f ? fmin(double(mp), 1.0) : 0.0;
  int k = top_k ? top_k[row] : 0;
  if (k <= 0 || k > n) k = n;
  const float tp = top_p ? top_p[row] : 1.0f;
  const bool by_mass = tp < 1.0f;
  if (by_mass && tp <= 0.0f) k = 1;

  // The kept prefix so far: keys above `key`, and those equal to it up to index `last`.
  uint32_t key = 0;
  int last = n - 1;
  auto kept = [&](float v, int i) {
    const uint32_t o = order_key(v);
    return o > key || (o == key && i <= last);
  };
  for (int pass = 0; pass < 2; ++pass) {  // by count, then by weight
    if (pass == 0 ? k >= n : !by_mass || tp <= 0.0f) continue;
    double goal = 0;
    if (pass == 1) {
      unsigned long long m = 0;
      for (int i = tid; i < n; i += kThreads)
        if (kept(l[i], i)) m += weight(l[i], w);
      for (int off = 32; off > 0; off >>= 1) m += __shfl_xor(m, off, 64);
      __syncthreads();
      if (lane == 0) red_m[wave] = m;
      __syncthreads();
      m = 0;
      for (int i = 0; i < kWaves; ++i) m += red_m[i];
      goal = double(tp) * double(m);
    }
    uint32_t prefix = 0, left = k;  // left: how many of the current digit's tokens stay
    unsigned long long before = 0;  // what stands above the current digit
    uint32_t count_before = 0;
    for (int d = 0; d < 3; ++d) {
      const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, bits = d == 2 ? 10 : 11;
      for (int i = tid; i < kBins; i += kThreads) bins.count[i] = 0, bins.mass[i] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const uint32_t o = order_key(l[i]);
        if (d > 0 && (o >> (shift + bits)) != prefix) continue;
        if (!kept(l[i], i)) continue;
        const uint32_t b = (o >> shift) & ((1u << bits) - 1);
        atomicAdd(&bins.count[b], 1u);
        if (pass == 1) atomicAdd(&bins.mass[b], weight(l[i], w));
      }
      __syncthreads();
      if (tid == 0) {
        for (int b = (1 << bits) - 1; b >= 0; --b) {
          if (!bins.count[b]) continue;
          const bool here = pass == 0 ? count_before + bins.count[b] >= uint32_t(k)
                                      : double(before + bins.mass[b]) >= goal;
          if (here) {
            found_bin = b;
            found_before = before;
            found_left = count_before;
            break;
          }
          before += bins.mass[b];
          count_before += bins.count[b];
        }
      }
      __syncthreads();
      prefix = (prefix << bits) | found_bin;
      before = found_before;
      count_before = found_left;
      left = bins.count[found_bin];
      __syncthreads();
    }
    // `left` tokens share the last key: how many of them stay, and the index of the last.
    uint32_t stay;
    if (pass == 0) {
      stay = k - count_before;
    } else {
      const unsigned long long one = bins.mass[found_bin] / left;
      const double need = (goal - double(before)) / double(one);
      stay = need <= 1.0 ? 1u : uint32_t(fmin(ceil(need), double(left)));
    }
    const int old_last = prefix == key ? last : n - 1;
    if (wave == 0) {
      uint32_t seen = 0;
      int end = n - 1;
      for (int i0 = 0; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        const bool eq = i < n && i <= old_last && order_key(l[i]) == prefix;
        const unsigned long long b = __ballot(eq);
        const uint32_t here = __popcll(b);
        if (seen + here >= stay) {
          const uint32_t rank = seen + __popcll(b & ((1ull << lane) - 1)) + 1;
          const unsigned long long hit = __ballot(eq && rank == stay);
          end = i0 + __ffsll(hit) - 1;
          break;
        }
        seen += here;
      }
      if (lane == 0) found_bin = uint32_t(end);
    }
    __syncthreads();
    key = prefix;
    last = int(found_bin);
    __syncthreads();
  }

  // The draw: each wave's stretch of the row, then the one the target falls in.
  const int per = (n + kWaves * 64 - 1) / (kWaves * 64) * 64;
  const int lo = min(n, wave * per), hi = min(n, lo + per);
  auto part = [&](int i) {
    return i < hi && kept(l[i], i) ? weight(l[i], w) : 0ull;
  };
  unsigned long long m = 0;
  for (int i = lo + lane; i < hi; i += 64) m += part(i);
  for (int off = 32; off > 0; off >>= 1) m += __shfl_xor(m, off, 64);
  __syncthreads();
  if (lane == 0) red_m[wave] = m;
  __syncthreads();
  unsigned long long total = 0, mine = 0;
  for (int i = 0; i < kWaves; ++i) {
    if (i == wave) mine = total;
    total += red_m[i];
  }
  float r = u[row];
  r = r > 0.0f ? fminf(r, 0x1.fffffep-1f) : 0.0f;
  const double target = double(r) * double(total);
  if (!(double(mine) <= target && target < double(mine + m))) return;
  unsigned long long sum = mine;
  for (int i0 = lo; i0 < hi; i0 += 64) {
    const unsigned long long p = part(i0 + lane);
    unsigned long long s = p;
    for (int off = 1; off < 64; off <<= 1) {
      const unsigned long long o = __shfl_up(s, off, 64);
      if (lane >= off) s += o;
    }
    const unsigned long long past = __ballot(double(sum + s) > target);
    if (past) {
      if (lane == 0) out[row] = i0 + __ffsll(past) - 1;
      return;
    }
    sum += __shfl(s, 63, 64);
  }
}

}  // namespace
}  // namespace iehip

using namespace iehip;

extern "C" size_t ie_hip_sample_rows_workspace_bytes(int R, int n) {
  (void)R;
  (void)n;
  return 0;
}

extern "C" int ie_hip_sample_rows(int32_t* out, const float* logits, const float* temperature,
                                  const int32_t* top_k, const float* top_p, const float* min_p,
                                  const float* u, int R, int n, void* workspace, hipStream_t stream) {
  clear_error();
  (void)workspace;
  if (R < 0 || n <= 0 || n > (1 << 30)) return fail(IE_HIP_EINVAL, "sample_rows: bad sizes");
  if (R == 0) return IE_HIP_OK;
  if (!out || !logits || !temperature || !u) return fail(IE_HIP_EINVAL, "sample_rows: null pointer");
  hipLaunchKernelGGL(sample_rows_kernel, dim3(R), dim3(kThreads), 0, stream, out, logits, temperature,
                     top_k, top_p, min_p, u, n, std::ldexp(1.0, weight_bits(n)));
  return check_launch("sample_rows");
}
