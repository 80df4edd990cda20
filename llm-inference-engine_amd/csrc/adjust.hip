// A step's logits under each row's rules (ie_hip_adjust_logits): penalties for tokens of its
// history, biases, a grammar's mask.
//
//   l' = seen ? (l > 0 ? l / rep : l * rep) : l
//   l' = l' - freq * count - pres * (count > 0);  l' = l' + bias;  -inf where masked
//
// A workgroup takes kSeg consecutive tokens of one row. It reads the row's whole history (4 bytes an
// entry, from L2 after the first workgroup of the row) and counts its own tokens in LDS, and notes
// the last bias entry of each in the same way: integer LDS atomics, so neither the order of the
// entries' arrival nor the launch shape changes a result, and nothing is kept between calls. Then one
// pass over the logits. The logits are loaded before the counting, which hides it.
#include "common.hpp"

namespace iehip {
namespace {

constexpr int kThreads = 256;
constexpr int kSeg = 8192;              // tokens of a workgroup
constexpr uint32_t kSeen = 0x80000000u;  // in the history; the low bits count generated tokens

__global__ void __launch_bounds__(kThreads)
adjust_logits_kernel(float* out, const float* logits, ie_logit_rules u, int n, int segs) {
  __shared__ uint32_t count[kSeg];
  __shared__ int32_t last[kSeg];  // 1 + the last bias entry's place in the row's list
  const int row = blockIdx.x / segs, base = (blockIdx.x - row * segs) * kSeg;
  const int len = min(kSeg, n - base);
  const size_t at = size_t(row) * n + base;
  const int tid = threadIdx.x;
  const bool history = u.history != nullptr, bias = u.bias_token != nullptr;
  int64_t h0 = 0, b0 = 0;
  int hn = 0, bn = 0;
  if (history) {
    h0 = u.history_start[row];
    hn = u.history_len[row];
  }
  if (bias) {
    b0 = u.bias_start[row];
    bn = u.bias_len[row];
  }
  if (history)
    for (int i = tid; i < kSeg; i += kThreads) count[i] = 0;
  if (bias)
    for (int i = tid; i < kSeg; i += kThreads) last[i] = 0;
  __syncthreads();
  if (history) {
    const int64_t made = h0 + (u.prompt_len ? u.prompt_len[row] : 0);
    const int64_t end = min(h0 + hn, u.history_size);
    for (int64_t e = max(h0, int64_t(0)) + tid; e < end; e += kThreads) {
      const int64_t t = int64_t(u.history[e]) - base;
      if (t < 0 || t >= len) continue;
      if (e < made)
        atomicOr(&count[t], kSeen);
      else
        atomicAdd(&count[t], 1u);
    }
  }
  if (bias) {
    const int64_t end = min(b0 + bn, u.bias_size);
    for (int64_t e = max(b0, int64_t(0)) + tid; e < end; e += kThreads) {
      const int64_t t = int64_t(u.bias_token[e]) - base;
      if (t >= 0 && t < len) atomicMax(&last[t], int32_t(e - b0) + 1);
    }
  }
  __syncthreads();
  const float rep = u.repetition ? u.repetition[row] : 1.0f;
  const float pres = u.presence ? u.presence[row] : 0.0f;
  const float freq = u.frequency ? u.frequency[row] : 0.0f;
  const uint32_t* mask = nullptr;
  if (u.mask) {
    const int m = u.mask_row ? u.mask_row[row] : row;
    if (m >= 0 && m < u.mask_rows) mask = u.mask + size_t(m) * ((n + 31) / 32);
  }
  for (int i = tid; i < len; i += kThreads) {
    float l = logits[at + i];
    if (history) {
      const uint32_t c = count[i];
      if (c) {
        const uint32_t times = c & ~kSeen;
        l = l > 0.0f ? l / rep : l * rep;
        l = l - freq * static_cast<float>(times);
        l = l - (times ? pres : 0.0f);
      }
    }
    if (bias && last[i]) l = l + u.bias_value[b0 + last[i] - 1];
    if (mask && !((mask[(base + i) >> 5] >> ((base + i) & 31)) & 1u)) l = -INFINITY;
    out[at + i] = l;
  }
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
  const int64_t segs = (int64_t(n) + kSeg - 1) / kSeg;
  if (segs * R * kThreads > int64_t(UINT32_MAX))
    return fail(IE_HIP_EINVAL, "adjust_logits: too many logits");
  hipLaunchKernelGGL(adjust_logits_kernel, dim3(unsigned(segs * R)), dim3(kThreads), 0, stream, out,
                     logits, u, n, int(segs));
  return check_launch("adjust_logits");
}
