// One token per row of logits (ie_hip_sample_rows): temperature, top-k, min-p, top-p, then inverse
// CDF in index order at the caller's random number.
//
// A weight is exp((l - max) / T) in float64, taken to whole numbers of 2^-45 (fewer bits where n of
// them would pass 63: weight_bits): sums of whole numbers are exact, so no order of adding them
// changes a result, and a border of the sums lies where the 64-bit definition has it to within about
// 2^-45 of the largest weight per token. A row is cut into chunks of kChunk logits, whatever R is.
//
// What is kept is a prefix of the tokens ordered by (logit descending, index ascending). Four launches,
// two over (row, chunk) that fill the chip and two over rows:
//   chunks   the chunk's largest logit, its weight relative to that, and, for rows with a filter, a
//            histogram of counts and weights over bins of T / 15.75 in the logit, which every
//            chunk places alike (place())
//   border   the row's histogram: which few bins hold the filters' borders; greedy rows end here
//   collect  per chunk the weight of the bins above all borders; the tokens of the border bins go to
//            the row's list
//   draw     the borders, found digit by digit of the ordered bit pattern in that list (of at most
//            kHeld tokens, in LDS up to kList; the whole row where the bins hold more, as with a row of
//            equal logits), then the chunk and the token where the running sum passes the target
// (64 rows x 151,936, settings mixed: one workgroup a row through all of it took 1,440 us.)
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.hpp"

namespace iehip {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;  // of the launches over rows
constexpr int kChunkThreads = 512, kEach = 8;           // of those over chunks, and logits of a thread
constexpr int kChunk = kChunkThreads * kEach;
constexpr int kPlaces = 512;               // bins of the rows' histograms
// Border tokens of a row: in LDS, in the workspace (1 x 151,936 of logits in steps of a half, at T = 5
// with top-p: 12,000 in one bin, 60 us from the workspace, 646 by walks of the row).
constexpr int kList = 6144, kHeld = 32768;
constexpr int kDigits = 2048;
constexpr int kMaxTokens = 1 << 22, kMaxChunks = kMaxTokens / kChunk;
typedef unsigned long long u64;

// Bits of the largest weight, so that n of them stay under 2^63.
int weight_bits(int n) {
  int log2 = 0;
  while ((int64_t(1) << log2) < n) ++log2;
  return std::min(45, 63 - log2);
}

enum Mode { kDone, kAll, kFiltered };

// What the border launch leaves of a row. Bins below `sure` are kept whole; those in
// [outer_lo, outer_hi] hold the border of top-k or min-p, those in [inner_lo, inner_hi] top-p's.
struct RowState {
  int32_t mode, listed;
  float top;
  int32_t sure, outer_lo, outer_hi, inner_lo, inner_hi;
  int32_t top_left;      // top-k: how many of the outer bins' tokens stay (INT_MAX: no limit)
  int32_t pad;
  u64 outer_mass;        // of the bins below outer_lo
  u64 outer_pass;        // of the outer bins' tokens that min-p keeps, where top-k does not bind
  u64 total;             // of the row
};

struct Entry {
  float l;
  int32_t i;
};

struct Workspace {
  RowState* rows;    // [R]
  Entry* list;       // [R, kHeld]
  u64* mass;         // [R, chunks] relative to the chunk's own top; after `collect` its sure weight
  u64* top;          // [R, chunks] the largest logit and its place (candidate)
  u64* bin_mass;     // [R, chunks, kPlaces]
  uint32_t* bin_count;
};

size_t lay_out(Workspace* w, void* base, int R, int n) {
  const size_t chunks = (size_t(n) + kChunk - 1) / kChunk, rc = R * chunks;
  unsigned char* p = static_cast<unsigned char*>(base);
  auto take = [&](size_t bytes) {
    unsigned char* at = p;
    p += (bytes + 15) / 16 * 16;
    return at;
  };
  Workspace v;
  v.rows = reinterpret_cast<RowState*>(take(R * sizeof(RowState)));
  v.list = reinterpret_cast<Entry*>(take(R * size_t(kHeld) * sizeof(Entry)));
  v.mass = reinterpret_cast<u64*>(take(rc * 8));
  v.top = reinterpret_cast<u64*>(take(rc * 8));
  v.bin_mass = reinterpret_cast<u64*>(take(rc * kPlaces * 8));
  v.bin_count = reinterpret_cast<uint32_t*>(take(rc * kPlaces * 4));
  if (w) *w = v;
  return size_t(p - static_cast<unsigned char*>(base));
}

struct Settings {
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
};

// One row's settings, brought into their ranges.
struct Row {
  double inv, rate, scale, least, one;  // 1 / T, weight_of's, bins per logit, min-p, the largest weight
  int k;                          // n: no top-k
  float p;                        // 1: no top-p
  bool greedy;
  __device__ __forceinline__ Row(const Settings& s, int row, int n, double one_) : one(one_) {
    const float t = s.temperature[row];
    greedy = !(t > 0.0f);
    inv = 1.0 / double(t);
    rate = 92.33248261689366 * inv;
    scale = 15.75 * inv;
    const float m = s.min_p ? s.min_p[row] : 0.0f;
    least = m > 0.0f ? fmin(double(m), 1.0) : 0.0;
    k = s.top_k ? s.top_k[row] : 0;
    if (k <= 0 || k > n) k = n;
    p = s.top_p ? s.top_p[row] : 1.0f;
    if (!(p < 1.0f)) p = 1.0f;
    if (p <= 0.0f) {
      k = 1;
      p = 1.0f;
    }
    if (k == 1) p = 1.0f;
  }
  __device__ __forceinline__ bool filtered(int n) const { return k < n || p < 1.0f || least > 0.0; }
};

// Logits in their order as unsigned numbers, -0 with +0. (NaN was read as -inf.)
__device__ __forceinline__ uint32_t order_key(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// 2^(j / 64) rounded to float64, brought to LDS for weight_of.
__device__ const double kPowers[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};
__device__ __forceinline__ void fill_powers(double* powers) {
  if (threadIdx.x < 64) powers[threadIdx.x] = kPowers[threadIdx.x];
}

// exp((l - top) / T) in [0, 1]. With x = 64 (l - top) / (T ln 2), m = round(x) and r = x - m:
// 2^(m div 64) 2^(m mod 64 / 64) (1 + c1 r + .. + c5 r^5), ck = (ln2 / 64)^k / k!. The series is off by
// 2^-54.7, the product x by 2^-53 x, which is below 2^-53 of the largest weight where the weight is
// e^x: 16 instructions, most of the launches over chunks (with the library's exp 64 rows x 151,936 took
// half as long again). `rate` is 64 / (T ln 2).
__device__ __forceinline__ double weight_of(float l, float top, double rate, const double* powers) {
  const double d = double(l) - double(top);
  const double x = fmax(d * rate, -64.0 * 64.0);  // 2^-64: nothing. l = -inf, and then T = inf, too
  const double m = rint(x), r = x - m;
  double e = __builtin_fma(r, 0x1.5d87fe78a6731p-40, 0x1.3b2ab6fba4e77p-31);
  e = __builtin_fma(e, r, 0x1.c6b08d704a0c0p-23);
  e = __builtin_fma(e, r, 0x1.ebfbdff82c58fp-15);
  e = __builtin_fma(e, r, 0x1.62e42fefa39efp-7);
  e = __builtin_fma(e, r, 1.0);
  const int im = int(m);
  return ldexp(powers[im & 63] * e, im >> 6);
}

// A weight as a whole number: adding 2^52 leaves it, rounded, in the low bits.
__device__ __forceinline__ u64 whole(double e, double one) {
  return static_cast<u64>(__double_as_longlong(__builtin_fma(e, one, 0x1p52))) & 0xFFFFFFFFFFFFFull;
}

// Where logits stand on the bins' axis, one function of l for every chunk, and how many bins below
// another place that is (the last bin: that many or more).
__device__ __forceinline__ double place(float l, double scale) { return floor(double(l) * scale); }
__device__ __forceinline__ int bin_below(double top_place, float l, double scale) {
  return int(fmin(top_place - place(l, scale), double(kPlaces - 1)));
}

__device__ __forceinline__ float read_logit(float v) { return v == v ? v : -INFINITY; }
// In a row whose largest logit is +inf, as in one of zeros where it is and nothing elsewhere.
__device__ __forceinline__ float in_row(float v, bool infinite) {
  return infinite ? (v == INFINITY ? 0.0f : -INFINITY) : v;
}

// A thread's logits of a chunk: element e of vec4 u is number (u * kChunkThreads + tid) * 4 + e.
__device__ __forceinline__ int chunk_index(int j) {
  return ((j >> 2) * kChunkThreads + int(threadIdx.x)) * 4 + (j & 3);
}
// VEC: n is a multiple of 4. Every load is issued, at a place within the chunk, and what is past its end
// replaced: a load behind a condition would wait for the one before.
template <bool VEC>
__device__ __forceinline__ void load_chunk(float (&v)[kEach], const float* l, int len) {
#pragma unroll
  for (int u = 0; u < kEach / 4; ++u) {
    const int at = chunk_index(4 * u);
    if constexpr (VEC) {
      const float4 q = *reinterpret_cast<const float4*>(l + min(at, len - 4));
      v[4 * u] = q.x, v[4 * u + 1] = q.y, v[4 * u + 2] = q.z, v[4 * u + 3] = q.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * u + e] = l[min(at + e, len - 1)];
    }
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j) v[j] = chunk_index(j) < len ? read_logit(v[j]) : -INFINITY;
}

// Running sums and maxima over a wave's lanes with the VALU's lane shifts (each row of 16 by 1, 2, 4 and
// 8, then rows 0 into 1 and 2 into 3, then lane 31 into the upper half): a step takes a few cycles, a
// shuffle through LDS some hundred.
template <int CTRL, int ROWS, class T, class F>
__device__ __forceinline__ T lane_step(T x, const F& join) {
  T y;
  if constexpr (sizeof(T) == 8) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, int(uint32_t(x)), CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, int(uint32_t(x >> 32)), CTRL, ROWS, 0xF, false);
    y = T(hi) << 32 | lo;
  } else {
    y = __builtin_amdgcn_update_dpp(0, int(x), CTRL, ROWS, 0xF, false);
  }
  return join(x, y);  // lanes without a source join 0
}
template <class T, class F>
__device__ __forceinline__ T wave_scan(T x, const F& join) {
  x = lane_step<0x111, 0xF>(x, join);  // row_shr:1
  x = lane_step<0x112, 0xF>(x, join);
  x = lane_step<0x114, 0xF>(x, join);
  x = lane_step<0x118, 0xF>(x, join);
  x = lane_step<0x142, 0xA>(x, join);  // row_bcast:15 into rows 1 and 3
  return lane_step<0x143, 0xC>(x, join);  // row_bcast:31 into rows 2 and 3
}
template <class T>
__device__ __forceinline__ T wave_running(T x) {
  return wave_scan(x, [](T a, T b) { return a + b; });
}
__device__ __forceinline__ u64 last_lane(u64 x) {
  return u64(uint32_t(__builtin_amdgcn_readlane(int(x >> 32), 63))) << 32 |
         uint32_t(__builtin_amdgcn_readlane(int(x), 63));
}
__device__ __forceinline__ u64 wave_sum(u64 m) { return last_lane(wave_running(m)); }

// A logit and its place as one number: larger logits, then lower places, are larger; 0 is none.
__device__ __forceinline__ u64 candidate(float l, int i) {
  return l > -INFINITY ? u64(order_key(l)) << 32 | uint32_t(~i) : 0;
}
__device__ __forceinline__ u64 wave_best(u64 c) {
  return last_lane(wave_scan(c, [](u64 a, u64 b) { return a > b ? a : b; }));
}
__device__ __forceinline__ float candidate_logit(u64 c) {
  const uint32_t o = uint32_t(c >> 32);
  return !c ? -INFINITY : __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ int candidate_place(u64 c) { return int(~uint32_t(c)); }

template <bool VEC>
__global__ void __launch_bounds__(kChunkThreads)
sample_chunks_kernel(const float* __restrict__ logits, Settings s, Workspace w, int n, int chunks,
                     double one) {
  constexpr int kParts = kChunkThreads / 64;
  __shared__ uint32_t count[kPlaces];
  __shared__ u64 mass[kPlaces];
  __shared__ double powers[64];
  __shared__ u64 red_m[kParts], red_s[kParts];
  const int row = blockIdx.x / chunks, c = blockIdx.x - row * chunks;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int base = c * kChunk, len = min(kChunk, n - base);
  float v[kEach];
  load_chunk<VEC>(v, logits + size_t(row) * n + base, len);
  const Row r(s, row, n, one);
  for (int i = tid; i < kPlaces; i += kChunkThreads) count[i] = 0, mass[i] = 0;
  fill_powers(powers);
  float most = v[0];
  int where = 0;
#pragma unroll
  for (int j = 1; j < kEach; ++j)
    if (v[j] > most) most = v[j], where = j;  // a thread's places rise with j
  u64 found = candidate(most, base + chunk_index(where));
  found = wave_best(found);
  if (lane == 0) red_m[wave] = found;
  __syncthreads();
  found = 0;
#pragma unroll
  for (int i = 0; i < kParts; ++i) found = red_m[i] > found ? red_m[i] : found;
  float best = candidate_logit(found);
  const size_t rc = size_t(row) * chunks + c;
  if (tid == 0) w.top[rc] = found;
  const bool by_count = r.k < n, by_mass = r.p < 1.0f;
  if (r.greedy || (r.filtered(n) && !by_count && !by_mass)) return;  // min-p alone needs no sums here
  if (best == INFINITY) {
    best = 0.0f;
#pragma unroll
    for (int j = 0; j < kEach; ++j) v[j] = in_row(v[j], true);
  }
  u64 sum = 0;
  const double tp = place(best, r.scale);
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (v[j] == -INFINITY) continue;  // (a masked row's tokens, and what is past the row)
    const u64 m = by_count && !by_mass ? 0 : whole(weight_of(v[j], best, r.rate, powers), one);
    sum += m;
    if (!by_count && !by_mass) continue;
    const int b = bin_below(tp, v[j], r.scale);
    if (b == kPlaces - 1) continue;  // what the others leave
    if (by_count) atomicAdd(&count[b], 1u);
    if (by_mass) atomicAdd(&mass[b], m);
  }
  sum = wave_sum(sum);
  if (lane == 0) red_s[wave] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0;
#pragma unroll
    for (int i = 0; i < kParts; ++i) sum += red_s[i];
    w.mass[rc] = sum;
  }
  if (by_count)
    for (int i = tid; i < kPlaces; i += kChunkThreads) w.bin_count[rc * kPlaces + i] = count[i];
  if (by_mass)
    for (int i = tid; i < kPlaces; i += kChunkThreads) w.bin_mass[rc * kPlaces + i] = mass[i];
}

// A chunk's weight, kept relative to its own largest logit, on the row's scale.
__device__ __forceinline__ u64 rescale(u64 m, double factor) {
  return factor == 1.0 ? m : static_cast<u64>(rint(double(m) * factor));
}

// Running sums over the workgroup's threads, own value included.
template <class T, int WAVES>
__device__ __forceinline__ T running(u64 (&sh)[WAVES], T x) {
  const int wave = threadIdx.x >> 6;
  x = wave_running(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sh[wave] = x;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) x += i < wave ? T(sh[i]) : T(0);
  return x;
}

__global__ void __launch_bounds__(kThreads)
sample_border_kernel(int32_t* __restrict__ out, Settings s, Workspace w, int n, int chunks, double one) {
  static_assert(kThreads == 2 * kPlaces, "a bin is two threads'");
  __shared__ uint32_t count[kPlaces];
  __shared__ u64 mass[kPlaces];
  __shared__ double powers[64];
  __shared__ u64 sh[kWaves];
  __shared__ int found[3];
  __shared__ double factor[kMaxChunks];
  __shared__ int shift[kMaxChunks];
  __shared__ u64 sums[kMaxChunks];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Row r(s, row, n, one);
  const u64* tops = w.top + size_t(row) * chunks;
  if (tid < 3) found[tid] = kPlaces - 1;
  fill_powers(powers);
  u64 best = 0;
  for (int c = tid; c < chunks; c += kThreads) best = tops[c] > best ? tops[c] : best;
  best = wave_best(best);
  if (lane == 0) sh[wave] = best;
  __syncthreads();
  best = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) best = sh[i] > best ? sh[i] : best;
  const float largest = candidate_logit(best);
  const bool infinite = largest == INFINITY;
  const float top = infinite ? 0.0f : largest;
  RowState* st = w.rows + row;
  if (r.greedy || !best || !r.filtered(n)) {
    if (tid == 0) {
      const bool done = r.greedy || !best;
      st->mode = done ? kDone : kAll;
      st->top = largest;
      if (done) out[row] = best ? candidate_place(best) : 0;
    }
    return;
  }
  const double tp = place(top, r.scale);
  for (int c = tid; c < chunks; c += kThreads) {
    const float t = in_row(candidate_logit(tops[c]), infinite);
    factor[c] = weight_of(t, top, r.rate, powers);
    sums[c] = r.p < 1.0f ? rescale(w.mass[size_t(row) * chunks + c], factor[c]) : 0;
    shift[c] = t > -INFINITY ? bin_below(tp, t, r.scale) : kPlaces;
  }
  __syncthreads();
  // A bin over the chunks, every other one by each of two threads: a chunk has it further down by how far
  // its own top is below the row's. The last bin is what the others leave, so nothing is added up from
  // several bins.
  const bool by_count = r.k < n, by_mass = r.p < 1.0f;
  const int place_of = tid % kPlaces, half = tid / kPlaces;
  u64 own_m = 0, all = 0;
  uint32_t own_n = 0;
  auto gather = [&](auto with_mass, auto with_count) {
    constexpr bool MASS = decltype(with_mass)::value, COUNT = decltype(with_count)::value;
    constexpr int kBatch = 10;  // loads of either kind under way at once
    for (int c0 = half; c0 < chunks; c0 += 2 * kBatch) {
      u64 m[kBatch];
      uint32_t k[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int c = min(c0 + 2 * j, chunks - 1);
        const size_t at = (size_t(row) * chunks + c) * kPlaces + max(place_of - shift[c], 0);
        if constexpr (MASS) m[j] = w.bin_mass[at];
        if constexpr (COUNT) k[j] = w.bin_count[at];
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int c = min(c0 + 2 * j, chunks - 1);
        const bool in = c0 + 2 * j < chunks && place_of >= shift[c];
        if constexpr (MASS) own_m += in ? rescale(m[j], factor[c]) : 0;
        if constexpr (COUNT) own_n += in ? k[j] : 0;
      }
    }
  };
  if (by_mass && by_count)
    gather(std::true_type{}, std::true_type{});
  else if (by_mass)
    gather(std::true_type{}, std::false_type{});
  else if (by_count)
    gather(std::false_type{}, std::true_type{});
  if (half) count[place_of] = own_n, mass[place_of] = own_m;
  __syncthreads();
  own_n = half ? 0 : own_n + count[place_of];
  own_m = half ? 0 : own_m + mass[place_of];
  if (by_mass) {
    for (int c = lane; c < chunks; c += 64) all += sums[c];
    all = wave_sum(all);
  }
  if (tid == kPlaces - 1) own_m = 0, own_n = 0;
  u64 cm = by_mass ? running(sh, own_m) : 0;
  uint32_t cn = by_count ? running(sh, own_n) : 0;
  if (tid == kPlaces - 1) {
    own_m = all > cm ? all - cm : 0;
    own_n = uint32_t(n) - cn;
    cm += own_m;
    cn = uint32_t(n);
  }
  __syncthreads();
  if (!half) count[tid] = cn, mass[tid] = cm;  // running sums from here on
  const u64 bm = cm - own_m;
  const uint32_t bn = cn - own_n;
  // top-k's bin: the one in which the running count reaches k
  if (!half && bn < uint32_t(r.k) && cn >= uint32_t(r.k)) found[0] = tid;
  __syncthreads();
  // The last bin's weights are 0 (e^-32.38 of the largest is less than half of 2^-45), so nobody asks
  // which of its tokens are kept, and a border there is none.
  int lo = 0x7fffffff, hi = -1, left = 0x7fffffff;
  if (r.least > 0.0) {
    // min-p's: one bin to either side of where its logit falls, for the roundings of the two
    const double d = tp - floor((double(top) + log(r.least) / r.inv) * r.scale);
    const int b = d < double(kPlaces - 2) ? int(fmax(d, 0.0)) : kPlaces - 2;
    lo = max(b - 1, 0);
    hi = min(b + 1, kPlaces - 2);
  }
  if (by_count && found[0] < kPlaces - 1) {
    const int b = found[0];
    if (b < lo) {
      lo = hi = b;
    } else {
      hi = min(hi, b);
    }
    if (b <= hi) left = r.k - (lo ? int(count[lo - 1]) : 0);
  }
  const bool outer = hi >= 0;
  const u64 total = mass[kPlaces - 1];
  const u64 below = outer ? (lo ? mass[lo - 1] : 0) : total;
  const u64 above = outer ? mass[hi] : total;
  if (r.p < 1.0f) {
    const double glo = double(r.p) * double(below), ghi = double(r.p) * double(above);
    if (!half && (tid == 0 || double(bm) < glo) && double(cm) >= glo) found[1] = tid;
    if (!half && (tid == 0 || double(bm) < ghi) && double(cm) >= ghi) found[2] = tid;
  }
  __syncthreads();
  if (tid != 0) return;
  RowState o;
  o.top = largest;
  o.outer_lo = outer ? lo : kPlaces;
  o.outer_hi = outer ? hi : kPlaces;
  o.inner_lo = r.p < 1.0f ? found[1] : kPlaces;
  o.inner_hi = r.p < 1.0f ? min(outer ? min(found[2], hi) : found[2], kPlaces - 2) : kPlaces;
  if (o.inner_lo > o.inner_hi) o.inner_lo = o.inner_hi;
  o.sure = min(o.outer_lo, o.inner_lo);
  o.outer_mass = below;
  o.outer_pass = 0;
  o.total = total;
  o.top_left = left;
  o.pad = 0;
  o.listed = 0;
  o.mode = kFiltered;
  *st = o;
}

template <bool VEC>
__global__ void __launch_bounds__(kChunkThreads)
sample_collect_kernel(const float* __restrict__ logits, Settings s, Workspace w, int n, int chunks,
                      double one) {
  __shared__ double powers[64];
  __shared__ u64 red_m[kChunkThreads / 64];
  __shared__ int many, next;
  const int row = blockIdx.x / chunks, c = blockIdx.x - row * chunks;
  RowState* st = w.rows + row;
  if (st->mode != kFiltered) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t rc = size_t(row) * chunks + c;
  const int sure = st->sure, outer_lo = st->outer_lo, outer_hi = st->outer_hi;
  const int inner_lo = st->inner_lo, inner_hi = st->inner_hi;
  const bool infinite = st->top == INFINITY;
  const float top = infinite ? 0.0f : st->top, chunk_top = in_row(candidate_logit(w.top[rc]), infinite);
  const Row r(s, row, n, one);
  const double tp = place(top, r.scale);
  const int nearest = chunk_top > -INFINITY ? bin_below(tp, chunk_top, r.scale) : kPlaces;
  const int last = max(sure - 1, max(outer_hi < kPlaces ? outer_hi : -1, inner_hi < kPlaces ? inner_hi : -1));
  if (nearest > last) {
    if (tid == 0) w.mass[rc] = 0;
    return;
  }
  const int base = c * kChunk, len = min(kChunk, n - base);
  float v[kEach];
  load_chunk<VEC>(v, logits + size_t(row) * n + base, len);
  fill_powers(powers);
  if (tid == 0) many = 0;
  __syncthreads();
  // Where top-k does not bind, min-p decides its bins' tokens one by one, and only top-p's are listed.
  const bool free = st->top_left == 0x7fffffff;
  u64 sum = 0, pass = 0;
  uint32_t listed = 0;  // a bit per logit
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    v[j] = in_row(v[j], infinite);
    if (v[j] == -INFINITY) continue;
    const int b = bin_below(tp, v[j], r.scale);
    const bool outer = b >= outer_lo && b <= outer_hi, inner = b >= inner_lo && b <= inner_hi;
    if (b < sure || (outer && free)) {
      const double x = weight_of(v[j], top, r.rate, powers);
      if (b >= sure && x < r.least) continue;
      const u64 m = whole(x, one);
      if (outer) pass += m;
      if (inner)
        listed |= 1u << j;
      else if (b < inner_lo)
        sum += m;
    } else if (outer || inner) {
      listed |= 1u << j;
    }
  }
  sum = wave_sum(sum);
  if (lane == 0) red_m[wave] = sum;
  if (free && r.p < 1.0f) {
    pass = wave_sum(pass);
    if (lane == 0 && pass) atomicAdd(&st->outer_pass, pass);
  }
  int at = listed ? atomicAdd(&many, __popc(listed)) : 0;
  __syncthreads();
  if (tid == 0) {
    sum = 0;
    for (int i = 0; i < kChunkThreads / 64; ++i) sum += red_m[i];
    w.mass[rc] = sum;
    next = many ? atomicAdd(&st->listed, many) : 0;
  }
  __syncthreads();
  at += next;
  Entry* list = w.list + size_t(row) * kHeld;
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (listed >> j & 1) {
      if (at < kHeld) list[at] = Entry{v[j], base + chunk_index(j)};
      ++at;
    }
}

struct Digits {
  u64 mass[kDigits];
  uint32_t count[kDigits];
  u64 sums[kWaves];
  int bin;
  uint32_t in_count;
  u64 before;
};

// One digit over `items` tokens: digit(i, mass) gives a token's bin (-1: none) and weight. The bin in
// which reach(running sum) first holds, of the weights with MASS, of the counts otherwise, is left in d
// (d.bin = -1: in none) with the sum before it.
template <bool MASS, class Digit, class Reach>
__device__ __forceinline__ void digit_pass(Digits& d, int items, const Digit& digit, const Reach& reach) {
  const int tid = threadIdx.x;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kDigits / kThreads; ++i) {
    d.count[i * kThreads + tid] = 0;
    if (MASS) d.mass[i * kThreads + tid] = 0;
  }
  if (tid == 0) d.bin = -1;
  __syncthreads();
  for (int i0 = 0; i0 < items; i0 += kThreads) {
    u64 m = 0;
    const int i = i0 + tid, b = i < items ? digit(i, m) : -1;
    // Equal logits fall into one bin: a wave's as one.
    const int first = __builtin_amdgcn_readfirstlane(b);
    if (__all(b == first)) {
      if (first < 0) continue;
      if (MASS) m = wave_sum(m);
      if ((tid & 63) == 0) {
        atomicAdd(&d.count[first], 64u);
        if (MASS && m) atomicAdd(&d.mass[first], m);
      }
    } else if (b >= 0) {
      atomicAdd(&d.count[b], 1u);
      if (MASS && m) atomicAdd(&d.mass[b], m);
    }
  }
  __syncthreads();
  const uint32_t n0 = d.count[2 * tid], n1 = d.count[2 * tid + 1];
  const u64 s0 = MASS ? d.mass[2 * tid] : n0, s1 = MASS ? d.mass[2 * tid + 1] : n1;
  const u64 sum = running(d.sums, s0 + s1), before = sum - s0 - s1;
  const bool r0 = reach(before), r1 = reach(before + s0), r2 = reach(sum);
  if (!r0 && r1) d.bin = 2 * tid, d.before = before, d.in_count = n0;
  if (!r1 && r2) d.bin = 2 * tid + 1, d.before = before + s0, d.in_count = n1;
  __syncthreads();
}

__global__ void __launch_bounds__(kThreads)
sample_draw_kernel(int32_t* __restrict__ out, const float* __restrict__ logits, Settings s, Workspace w,
                   int n, int chunks, double one) {
  __shared__ Digits d;
  __shared__ Entry list[kList];
  __shared__ double powers[64];
  __shared__ u64 chunk_mass[kMaxChunks];
  __shared__ u64 red_m[kWaves];
  __shared__ u64 before_of;
  __shared__ int chosen;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  RowState st = w.rows[row];
  if (st.mode == kDone) return;
  const float* l = logits + size_t(row) * n;
  const Row r(s, row, n, one);
  const bool filtered = st.mode != kAll, all = filtered && st.listed > kHeld;
  const bool infinite = st.top == INFINITY;
  if (infinite) st.top = 0.0f;
  const double tp = place(st.top, r.scale);
  fill_powers(powers);
  if (all) {
    st.sure = 0, st.outer_lo = 0, st.outer_hi = kPlaces - 1, st.inner_lo = 0, st.inner_hi = kPlaces - 1;
    st.outer_mass = 0;
    st.top_left = r.k < n ? r.k : 0x7fffffff;
  }
  const int items = !filtered ? 0 : all ? n : st.listed;
  const bool in_lds = items <= kList;
  const Entry* held = w.list + size_t(row) * kHeld;
  if (!all && in_lds)
    for (int i = tid; i < items; i += kThreads) list[i] = held[i];
  for (int i = tid; i < chunks; i += kThreads) {
    const size_t rc = size_t(row) * chunks + i;
    chunk_mass[i] = filtered && !all ? w.mass[rc] : 0;
  }
  __syncthreads();
  // The list's logits agree in their leading bits, being of few bins: how many digits that leaves.
  int digits = 3;
  uint32_t common_prefix = 0;
  if (filtered && !all && items > 0) {
    const uint32_t o = order_key(held[0].l);
    uint32_t differ = 0;
    for (int i = tid; i < items; i += kThreads) differ |= order_key(in_lds ? list[i].l : held[i].l) ^ o;
    if (tid == 0) chosen = 0;
    __syncthreads();
    if (differ) atomicOr(&chosen, int(differ));
    __syncthreads();
    const uint32_t any = uint32_t(chosen);
    digits = any >> 21 ? 3 : any >> 10 ? 2 : 1;
    common_prefix = digits == 3 ? 0 : digits == 2 ? o >> 21 : o >> 10;
  }
  auto entry = [&](int i) {
    return all ? Entry{in_row(read_logit(l[i]), infinite), i} : in_lds ? list[i] : held[i];
  };
  auto bin_of = [&](float v) { return v > -INFINITY ? bin_below(tp, v, r.scale) : kPlaces - 1; };
  auto weight = [&](float v) { return weight_of(v, st.top, r.rate, powers); };

  // The kept part of the list: at or above (key, last index), in order, of bins up to `end`, with the
  // least weight where the bin is one of the outer ones.
  uint32_t key = 0;
  int last = 0x7fffffff, end = kPlaces - 1;
  auto above = [&](float v, int i) {
    const uint32_t o = order_key(v);
    return o > key || (o == key && i <= last);
  };
  auto outer = [&](int b) { return b >= st.outer_lo && b <= st.outer_hi; };
  auto stays = [&](float v, int i, int b, double e) {
    return b <= end && above(v, i) && (!outer(b) || e >= r.least);
  };
  // Moves (key, last) to the token at which reach() first holds of the running sums (of weights with
  // by_mass, else of tokens) over the tokens that `take` lets in; stay() says how many of the last key's
  // equal tokens that is.
  auto select = [&](auto by_mass, const auto& take, const auto& reach, const auto& stay) {
    constexpr bool MASS = decltype(by_mass)::value;
    uint32_t prefix = common_prefix;
    u64 sum = 0;
    for (int pass = 3 - digits; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      digit_pass<MASS>(
          d, items,
          [&](int i, u64& m) {
            const Entry e = entry(i);
            const uint32_t o = order_key(e.l);
            if (pass > 3 - digits && (o >> (shift + bits)) != prefix) return -1;
            return take(e.l, e.i, m) ? int(((1u << bits) - 1) - ((o >> shift) & ((1u << bits) - 1))) : -1;
          },
          [&](u64 s) { return reach(sum + s); });
      if (d.bin < 0) return;  // never: all stay
      prefix = (prefix << bits) | (((1u << bits) - 1) - uint32_t(d.bin));
      sum += d.before;
    }
    const uint32_t equal = d.in_count, keep = equal > 1 ? stay(equal, sum, prefix) : 1;
    int to = 0x7fffffff;
    if (keep < equal) {  // the index of the keep-th of them
      int high = 0;
      u64 c0 = 0;
      for (int pass = 0; pass < 2; ++pass) {
        digit_pass<false>(
            d, items,
            [&](int i, u64&) {
              const Entry e = entry(i);
              if (order_key(e.l) != prefix || (pass == 1 && e.i >> 11 != high)) return -1;
              u64 m;
              return take(e.l, e.i, m) ? (pass == 0 ? e.i >> 11 : e.i & 2047) : -1;
            },
            [&](u64 c) { return c0 + c >= keep; });
        if (pass == 0) high = d.bin, c0 = d.before;
      }
      to = (high << 11) | d.bin;
    }
    key = prefix;
    last = to;
  };

  if (filtered && st.top_left != 0x7fffffff) {
    const uint32_t left = uint32_t(st.top_left);
    select(
        std::false_type{}, [&](float v, int, u64&) { return outer(bin_of(v)); },
        [&](u64 c) { return c >= left; },
        [&](uint32_t, u64 c, uint32_t) { return left - uint32_t(c); });
  }
  if (filtered && r.p < 1.0f) {
    u64 of = st.total;
    if (st.outer_lo < kPlaces && !all && st.top_left == 0x7fffffff) {
      of = st.outer_mass + st.outer_pass;
    } else if (st.outer_lo < kPlaces) {
      u64 m = 0;
      for (int i = tid; i < items; i += kThreads) {
        const Entry e = entry(i);
        const int b = bin_of(e.l);
        const double x = weight(e.l);
        if (outer(b) && stays(e.l, e.i, b, x)) m += whole(x, one);
      }
      m = wave_sum(m);
      __syncthreads();
      if (lane == 0) red_m[wave] = m;
      __syncthreads();
      of = st.outer_mass;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) of += red_m[i];
    }
    const double goal = double(r.p) * double(of);
    // What the list's tokens come on top of: the chunks' sums so far.
    u64 base = 0;
    for (int i = lane; i < chunks; i += 64) base += chunk_mass[i];
    base = wave_sum(base);
    end = st.inner_hi;
    select(
        std::true_type{},
        [&](float v, int i, u64& m) {
          const int b = bin_of(v);
          const double x = weight(v);
          m = whole(x, one);
          return stays(v, i, b, x);
        },
        [&](u64 m) { return double(base + m) >= goal; },
        [&](uint32_t equal, u64 m, uint32_t o) {
          const float v = __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
          const double each = double(whole(weight(v), one));
          const double need = (goal - double(base + m)) / each;
          return need <= 1.0 ? 1u : uint32_t(fmin(ceil(need), double(equal)));
        });
  }
  // The kept weight of each chunk.
  if (!filtered) {
    for (int i = tid; i < chunks; i += kThreads) {
      const size_t rc = size_t(row) * chunks + i;
      chunk_mass[i] = rescale(w.mass[rc], weight(in_row(candidate_logit(w.top[rc]), infinite)));
    }
  }
  auto kept = [&](float v, int i) -> u64 {
    if (!(v > -INFINITY)) return 0;
    const double x = weight(v);
    if (filtered) {
      const int b = bin_of(v);
      const bool listed = outer(b) || (b >= st.inner_lo && b <= st.inner_hi);
      if (b >= st.sure && !(listed && stays(v, i, b, x))) return 0;
    }
    return whole(x, one);
  };
  __syncthreads();
  for (int i0 = 0; i0 < items; i0 += kThreads) {
    const int i = i0 + tid;
    const Entry e = i < items ? entry(i) : Entry{-INFINITY, 0};
    u64 m = kept(e.l, e.i);
    if (all) {  // a wave's tokens are of one chunk
      m = wave_sum(m);
      if (lane == 0 && m) atomicAdd(&chunk_mass[e.i / kChunk], m);
    } else if (m) {
      atomicAdd(&chunk_mass[e.i / kChunk], m);
    }
  }
  __syncthreads();
  const u64 own = tid < chunks ? chunk_mass[tid] : 0;
  const u64 cm = running(d.sums, own);
  if (tid == kThreads - 1) before_of = cm;
  __syncthreads();
  const u64 total = before_of;
  float u = s.u[row];
  u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
  // The first running sum above u * total, in whole numbers: the first that reaches `need`.
  const u64 need = min(static_cast<u64>(double(u) * double(total)) + 1, total);
  __syncthreads();
  if (cm - own < need && cm >= need) chosen = tid, before_of = cm - own;
  __syncthreads();
  const int base = chosen * kChunk, len = min(kChunk, n - base);
  u64 want = need - before_of;
  if (!filtered) {  // in the chunk's own units, whose sum is at hand
    const size_t rc = size_t(row) * chunks + chosen;
    const float chunk_top = in_row(candidate_logit(w.top[rc]), infinite);
    if (chunk_top != st.top) {
      const double f = weight(chunk_top);
      want = max(u64(1), min(w.mass[rc], static_cast<u64>(ceil(double(want) / f))));
      st.top = chunk_top;
    }
  }
  // A wave's stretch of the chunk, kPart weights a lane.
  constexpr int kPart = kChunk / kThreads;
  const int lo = wave * kPart * 64 + lane;
  float v[kPart];
#pragma unroll
  for (int j = 0; j < kPart; ++j) v[j] = in_row(lo + 64 * j < len ? read_logit(l[base + min(lo + 64 * j, len - 1)]) : -INFINITY, infinite);
  u64 p[kPart], m = 0;
#pragma unroll
  for (int j = 0; j < kPart; ++j) {
    p[j] = kept(v[j], base + lo + 64 * j);
    m += p[j];
  }
  m = wave_sum(m);
  __syncthreads();
  if (lane == 0) red_m[wave] = m;
  __syncthreads();
  u64 sum = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) sum += i < wave ? red_m[i] : 0;
  if (!(sum < want && sum + m >= want)) return;
  for (int j = 0; j < kPart; ++j) {
    u64 q = 0;
#pragma unroll
    for (int i = 0; i < kPart; ++i) q = i == j ? p[i] : q;
    q = wave_running(q);
    const u64 past = __ballot(sum + q >= want);
    if (past) {
      if (lane == 0) out[row] = base + wave * kPart * 64 + 64 * j + __ffsll(past) - 1;
      return;
    }
    sum += last_lane(q);
  }
}

}  // namespace
}  // namespace iehip

using namespace iehip;

extern "C" size_t ie_hip_sample_rows_workspace_bytes(int R, int n) {
  if (R <= 0 || n <= 0 || n > kMaxTokens) return 0;
  return lay_out(nullptr, nullptr, R, n);
}

extern "C" int ie_hip_sample_rows(int32_t* out, const float* logits, const float* temperature,
                                  const int32_t* top_k, const float* top_p, const float* min_p,
                                  const float* u, int R, int n, void* workspace, hipStream_t stream) {
  clear_error();
  if (R < 0 || n <= 0) return fail(IE_HIP_EINVAL, "sample_rows: bad sizes");
  if (n > kMaxTokens) return fail(IE_HIP_EINVAL, "sample_rows: more than 4,194,304 tokens");
  if (R == 0) return IE_HIP_OK;
  if (!out || !logits || !temperature || !u) return fail(IE_HIP_EINVAL, "sample_rows: null pointer");
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(IE_HIP_EINVAL, "sample_rows: needs a 16-byte aligned workspace");
  const int chunks = (n + kChunk - 1) / kChunk;
  if (int64_t(R) * std::max(chunks * kChunkThreads, kThreads) > int64_t(UINT32_MAX))
    return fail(IE_HIP_EINVAL, "sample_rows: too many rows");
  Workspace w;
  lay_out(&w, workspace, R, n);
  const Settings s{temperature, top_k, top_p, min_p, u};
  const double one = std::ldexp(1.0, weight_bits(n));
  const bool vec = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && n % 4 == 0;
  const dim3 every(unsigned(R) * chunks), rows(R), wide(kChunkThreads), block(kThreads);
  const auto each = vec ? sample_chunks_kernel<true> : sample_chunks_kernel<false>;
  const auto collect = vec ? sample_collect_kernel<true> : sample_collect_kernel<false>;
  hipLaunchKernelGGL(each, every, wide, 0, stream, logits, s, w, n, chunks, one);
  hipLaunchKernelGGL(sample_border_kernel, rows, block, 0, stream, out, s, w, n, chunks, one);
  if (top_k || top_p || min_p)
    hipLaunchKernelGGL(collect, every, wide, 0, stream, logits, s, w, n, chunks, one);
  hipLaunchKernelGGL(sample_draw_kernel, rows, block, 0, stream, out, logits, s, w, n, chunks, one);
  return check_launch("sample_rows");
}
