// A step's logits under each row's rules (ie_hip_adjust_logits): penalties for tokens of its
// history, biases, a grammar's mask.
//
//   l' = seen ? (l > 0 ? l / rep : l * rep) : l
//   l' = l' - freq * count - pres * (count > 0);  l' = l' + bias;  -inf where masked
//
// A workgroup takes SEG consecutive tokens of one row: their logits go to registers, then it reads the
// row's whole history (4 bytes an entry, from L2 after the first workgroup of the row) and counts its own
// tokens in LDS, applies the penalties, notes the last bias entry of each token in the same place and
// applies those, then the mask. The counting is by integer LDS atomics, so neither the order of the
// entries' arrival nor the launch shape changes a result, and nothing is kept between calls.
// Bound by the logits' way in and out; segments of 2,048 where 8,192 would leave compute units idle.
#include "common.hpp"

namespace iehip {
namespace {

constexpr uint32_t kSeen = 0x80000000u;  // in the history; the low bits count generated tokens

template <int SEG, int THREADS, bool VEC>
__global__ void __launch_bounds__(THREADS)
adjust_logits_kernel(float* out, const float* logits, ie_logit_rules u, int n, int segs) {
  constexpr int kQuads = SEG / THREADS / 4;  // of a thread
  __shared__ __attribute__((aligned(16))) uint32_t word[SEG];
  const int row = blockIdx.x / segs, base = (blockIdx.x - row * segs) * SEG;
  const int len = min(SEG, n - base), tid = threadIdx.x;
  const size_t at = size_t(row) * n + base;
  // Quad q of a thread: tokens quad(q) .. + 3 of the segment.
  auto quad = [&](int q) { return (q * THREADS + tid) * 4; };
  float4 l[kQuads];
#pragma unroll
  for (int q = 0; q < kQuads; ++q) {
    // (past the end: some logit of the segment, never stored; a load behind a condition would wait)
    const int i = quad(q);
    if constexpr (VEC)  // n and so len are multiples of 4
      l[q] = *reinterpret_cast<const float4*>(logits + at + min(i, len - 4));
    else
      l[q] = make_float4(logits[at + min(i, len - 1)], logits[at + min(i + 1, len - 1)],
                         logits[at + min(i + 2, len - 1)], logits[at + min(i + 3, len - 1)]);
  }
  auto clear = [&]() {
#pragma unroll
    for (int q = 0; q < kQuads; ++q) *reinterpret_cast<uint4*>(word + quad(q)) = make_uint4(0, 0, 0, 0);
    __syncthreads();
  };
  if (u.history) {
    const int64_t h0 = u.history_start[row], hn = u.history_len[row];
    const int64_t made = h0 + (u.prompt_len ? u.prompt_len[row] : 0);
    const float rep = u.repetition ? u.repetition[row] : 1.0f;
    const float pres = u.presence ? u.presence[row] : 0.0f;
    const float freq = u.frequency ? u.frequency[row] : 0.0f;
    const int64_t first = max(h0, int64_t(0)), end = min(h0 + hn, u.history_size);
    if (first < end) {  // the whole workgroup
      clear();
      for (int64_t e = first + tid; e < end; e += THREADS) {
        const int64_t t = int64_t(u.history[e]) - base;
        if (t < 0 || t >= len) continue;
        if (e < made)
          atomicOr(&word[t], kSeen);
        else
          atomicAdd(&word[t], 1u);
      }
      __syncthreads();
      auto penalty = [&](float& v, uint32_t c) {
        if (!c) return;
        const uint32_t times = c & ~kSeen;
        v = v > 0.0f ? v / rep : v * rep;
        v = v - freq * static_cast<float>(times);
        v = v - (times ? pres : 0.0f);
      };
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        const uint4 c = *reinterpret_cast<const uint4*>(word + quad(q));
        if (!(c.x | c.y | c.z | c.w)) continue;
        penalty(l[q].x, c.x);
        penalty(l[q].y, c.y);
        penalty(l[q].z, c.z);
        penalty(l[q].w, c.w);
      }
    }
  }
  if (u.bias_token) {
    const int64_t b0 = u.bias_start[row], bn = u.bias_len[row];
    const int64_t first = max(b0, int64_t(0)), end = min(b0 + bn, u.bias_size);
    if (first < end) {
      clear();  // a thread's own words, which it alone has read
      for (int64_t e = first + tid; e < end; e += THREADS) {
        const int64_t t = int64_t(u.bias_token[e]) - base;
        if (t >= 0 && t < len) atomicMax(&word[t], uint32_t(e - b0) + 1);
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        const uint4 c = *reinterpret_cast<const uint4*>(word + quad(q));
        if (c.x) l[q].x = l[q].x + u.bias_value[b0 + c.x - 1];
        if (c.y) l[q].y = l[q].y + u.bias_value[b0 + c.y - 1];
        if (c.z) l[q].z = l[q].z + u.bias_value[b0 + c.z - 1];
        if (c.w) l[q].w = l[q].w + u.bias_value[b0 + c.w - 1];
      }
    }
  }
  const uint32_t* mask = nullptr;
  if (u.mask) {
    const int m = u.mask_row ? u.mask_row[row] : row;
    if (m >= 0 && m < u.mask_rows) mask = u.mask + size_t(m) * ((n + 31) / 32);
  }
#pragma unroll
  for (int q = 0; q < kQuads; ++q) {
    const int i = quad(q);
    if (i >= len) continue;
    if (mask) {  // a quad's bits are of one word
      const uint32_t on = mask[(base + i) >> 5] >> ((base + i) & 31);
      if (!(on & 1)) l[q].x = -INFINITY;
      if (!(on & 2)) l[q].y = -INFINITY;
      if (!(on & 4)) l[q].z = -INFINITY;
      if (!(on & 8)) l[q].w = -INFINITY;
    }
    if constexpr (VEC) {
      *reinterpret_cast<float4*>(out + at + i) = l[q];
    } else {
      out[at + i] = l[q].x;
      if (i + 1 < len) out[at + i + 1] = l[q].y;
      if (i + 2 < len) out[at + i + 2] = l[q].z;
      if (i + 3 < len) out[at + i + 3] = l[q].w;
    }
  }
}

template <int SEG, int THREADS>
int launch_adjust(float* out, const float* logits, const ie_logit_rules& u, int R, int n, hipStream_t stream) {
  const int64_t segs = (int64_t(n) + SEG - 1) / SEG;
  if (segs * R * THREADS > int64_t(UINT32_MAX))
    return fail(IE_HIP_EINVAL, "adjust_logits: too many logits");
  const bool vec = ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(logits)) & 15) == 0 &&
                   n % 4 == 0;
  const dim3 grid(unsigned(segs * R)), block(THREADS);
  if (vec)
    hipLaunchKernelGGL((adjust_logits_kernel<SEG, THREADS, true>), grid, block, 0, stream, out, logits, u,
                       n, int(segs));
  else
    hipLaunchKernelGGL((adjust_logits_kernel<SEG, THREADS, false>), grid, block, 0, stream, out, logits, u,
                       n, int(segs));
  return check_launch("adjust_logits");
}

}  // namespace
}  // namespace iehip

using namespace iehip;

extern "C" int ie_hip_adjust_logits(float* out, const float* logits, ie_logit_rules u, int R, int n,
                                    hipStream_t stream) {
  clear_error();
  if (R < 0 || n <= 0) return fail(IE_HIP_EINVAL, "adjust_logits: bad sizes");
  if (R == 0) return IE_HIP_OK;
  if (!out || !logits) return fail(IE_HIP_EINVAL, "adjust_logits: null pointer");
  if (u.history && (!u.history_start || !u.history_len || u.history_size < 0))
    return fail(IE_HIP_EINVAL, "adjust_logits: a history needs its starts, lengths and size");
  if (!u.history && (u.repetition || u.presence || u.frequency || u.prompt_len))
    return fail(IE_HIP_EINVAL, "adjust_logits: penalties need a history");
  if (!u.bias_token != !u.bias_value ||
      (u.bias_token && (!u.bias_start || !u.bias_len || u.bias_size < 0)))
    return fail(IE_HIP_EINVAL, "adjust_logits: biases need tokens, values, starts, lengths and a size");
  if (u.mask && u.mask_rows < 0) return fail(IE_HIP_EINVAL, "adjust_logits: mask_rows < 0");
  if (!u.mask && u.mask_row) return fail(IE_HIP_EINVAL, "adjust_logits: mask rows without a mask");
  const int64_t wide = (int64_t(n) + 8191) / 8192 * R;
  return wide >= device_compute_units() ? launch_adjust<8192, 512>(out, logits, u, R, n, stream)
                                        : launch_adjust<2048, 256>(out, logits, u, R, n, stream);
}
