// Products with 4-bit weights and group scales (gfx950): matmul_q4, qkv_proj_q4, gate_up_silu_q4.
//
//   y[t][o] = sum_g s[o][g] * sum_{k in g} (q[o][k] - z[o][g]) * x[t][k]  (+ bias, + y, SiLU product)
//
// on v_mfma_f32_16x16x32_f16. A weight enters the matrix cores as the whole number q - z, exact
// in f16 (|q - z| <= 255); its group's scale multiplies the group's f32 sum. An activation enters
// as two f16 parts of x / 2^e, hi + lo, with one power of two per token and block of 128 columns
// that puts the block's largest finite |x| in [2^14, 2^15): |x - (hi + lo) 2^e| <= 2^-23 |x| + 2^-40
// max|block|, one more rounding of float32's size. (Three bf16 parts, as the BF16 projections take
// them, would be exact without the power of two but cost half as many products again, and bf16 has
// no packed subtract to make q - z with.) Sums are f32 throughout: a group's over its products,
// then one fma per group and output into the slot's, then the slots in order.
//
// Order of the sums: the matrix's blocks of 128 columns are cut into 8 slots (slot_block), a slot's
// blocks are added in order, then the slots in order. It depends on the matrix's columns alone, so a
// token's result is the same bit for bit in whatever batch and by whichever kernel it is computed.
//
// Lane (g, r) of a tile of 16 rows x 16 tokens loads 16 bytes = 32 columns of row r at a time, and
// holds the results of tokens 4g .. 4g+3 and row r, so that a lane meets one scale per group.
#include <algorithm>

#include "common.hpp"
#include "matmul_tiled.hpp"
#include "mfma.hpp"

namespace iehip {
namespace {

constexpr int kBlock = 128;  // columns that share an activation scale: 4 products of 32
constexpr int kSlots = 8;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// First block of slot i of n blocks.
__host__ __device__ __forceinline__ int slot_block(int i, int n) { return int(int64_t(i) * n / kSlots); }

// One 4-bit matrix as a kernel sees it.
struct Q4View {
  const uint8_t* data;
  const void* scale;
  const uint8_t* zero;
};

// The scale of (row, group) and the pair of f16 constants that take a weight's zero point off.
__device__ __forceinline__ float q4_scale(const Q4View& w, int type, size_t at) {
  if (type == IE_KV_F32) return static_cast<const float*>(w.scale)[at];
  const uint16_t b = static_cast<const uint16_t*>(w.scale)[at];
  return type == IE_KV_F16 ? f16_bits_to_f32(b) : bf16_bits_to_f32(b);
}
__device__ __forceinline__ uint32_t q4_zero(const Q4View& w, size_t at) {
  return w.zero ? w.zero[at] : 8u;
}

// 8 weights of a word, less their zero point, as f16: element order 0, 4, 1, 5, 2, 6, 3, 7.
// A nibble in the low bits of an f16 of 1,024 reads 1024 + q; one four bits up reads 1024 + 16 q,
// which an fma with 1/16 brings down: every step is exact. (4 + 1 bit operations and 4 packed ones
// for 8 weights.)
__device__ __forceinline__ f16x8 unpack8(uint32_t w, uint32_t zero) {
  const uint32_t base = 0x64006400u;
  auto pair = [](uint32_t v) { return __builtin_bit_cast(f16x2, v); };
  const f16x2 z1024 = pair(base + zero * 0x10001u);                           // 1024 + z
  const _Float16 z = static_cast<_Float16>(-64.0f - static_cast<float>(zero));  // -(64 + z)
  const f16x2 z64 = {z, z};
  const f16x2 sixteenth = {_Float16(0.0625f), _Float16(0.0625f)};
  const uint32_t h = w >> 8;
  const f16x2 a = pair((w & 0x000F000Fu) | base) - z1024;
  const f16x2 b = __builtin_elementwise_fma(pair((w & 0x00F000F0u) | base), sixteenth, z64);
  const f16x2 c = pair((h & 0x000F000Fu) | base) - z1024;
  const f16x2 d = __builtin_elementwise_fma(pair((h & 0x00F000F0u) | base), sixteenth, z64);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 4x4 transpose of words over the lane groups: word j of group g becomes word g of group j.
__device__ __forceinline__ void transpose4(u32x4& v) {
  uint32_t a = v[0], b = v[1], c = v[2], d = v[3];
  asm volatile(
      "s_nop 1\n\tv_permlane32_swap_b32 %0, %2\n\tv_permlane32_swap_b32 %1, %3\n\t"
      "s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\tv_permlane16_swap_b32 %2, %3\n\ts_nop 1"
      : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
  v = u32x4{a, b, c, d};
}

// The power of two of a block from the bits of its largest finite |x|: `factor` takes x to f16's
// range, `back` is its inverse. Blocks below 2^-100 keep the factor of 2^-100.
__device__ __forceinline__ void block_scale(uint32_t largest, float& factor, float& back) {
  const uint32_t e = max(largest >> 23, 27u);
  factor = __uint_as_float((268u - e) << 23);
  back = __uint_as_float((e - 14u) << 23);
}

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t u = __float_as_uint(v) & 0x7FFFFFFFu;
  return u < 0x7F800000u ? u : 0u;
}

// 8 activations as hi + lo parts in unpack8's order. A value that is not finite is all in hi.
__device__ __forceinline__ void split8(const float (&x)[8], float factor, f16x8& hi, f16x8& lo) {
  constexpr int kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = x[kOrder[i]] * factor;
    _Float16 h, l;
    split16(v, h, l);
    hi[i] = h;
    lo[i] = finite_bits(v) == (__float_as_uint(v) & 0x7FFFFFFFu) ? l : _Float16(0.0f);
  }
}

// Where the part of columns 8 k8 .. 8 k8 + 7 of a block stands in LDS: 16 bytes per (step, lane
// group, token), tokens permuted by k8 so that the 16 lanes that write a token's block hit every bank.
// WIDE (groups of 128): step j holds columns 32 g + 8 j of lane group g, as the weights are loaded;
// otherwise step j is columns 32 j .. 32 j + 31 and the weights are transposed to it.
template <bool WIDE>
__device__ __forceinline__ int part_slot(int step, int g, int tok) {
  const int k8 = WIDE ? 4 * g + step : 4 * step + g;
  return step * 64 + 16 * g + (tok ^ k8);
}

struct Q4Out {
  float* y;
  const float* bias;
  int accumulate;
  RowSplit split;
};

__device__ __forceinline__ void q4_store(const Q4Out& o, int rows, int tok, int row, float v) {
  float* dst;
  if (row < o.split.split0)
    dst = o.y + size_t(tok) * o.split.split0 + row;
  else if (row < o.split.split1)
    dst = o.split.y1 + size_t(tok) * (o.split.split1 - o.split.split0) + (row - o.split.split0);
  else
    dst = o.split.y2 + size_t(tok) * (rows - o.split.split1) + (row - o.split.split1);
  if (o.bias) v += o.bias[row];
  if (o.accumulate) v += *dst;
  *dst = v;
}

// A workgroup: RT tiles of 16 rows (per matrix) by one tile of 16 tokens; wave i takes slot i. A wave
// splits its own blocks of activations through 8 KB of LDS of its own, so no wave waits for another
// before the slots are added.
template <bool GATE, int RT, int GROUP>
__global__ void __launch_bounds__(64 * kSlots)
q4_few_kernel(Q4Out out, const float* __restrict__ x, Q4View w0, Q4View w1, int scale_type, int T,
              int rows, int cols, int row_groups) {
  constexpr int NA = GATE ? 2 : 1, NT = NA * RT;
  constexpr bool WIDE = GROUP == 128;
  constexpr int kPer = kBlock / GROUP;  // groups of a block
  constexpr int kStage = 8192 + 64;
  constexpr int kLds = kSlots * kStage > kSlots * NT * 1024 ? kSlots * kStage : kSlots * NT * 1024;
  __shared__ __attribute__((aligned(16))) unsigned char lds[kLds];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int tok_tile = blockIdx.x / row_groups, row_group = blockIdx.x - tok_tile * row_groups;
  const int row0 = row_group * 16 * RT, tok0 = tok_tile * 16;
  const int nt = min(16, T - tok0);
  const int blocks = (cols + kBlock - 1) / kBlock, groups = (cols + GROUP - 1) / GROUP;
  unsigned char* stage = lds + wave * kStage;
  float* back_of = reinterpret_cast<float*>(stage + 8192);
  const Q4View w[2] = {w0, w1};

  f32x4 acc[NA][RT];
#pragma unroll
  for (int n = 0; n < NA; ++n)
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  int row[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) row[i] = min(row0 + 16 * i + r, rows - 1);

  const int b1 = slot_block(wave + 1, blocks);
  for (int b = slot_block(wave, blocks); b < b1; ++b) {
    const int kw = b * kBlock + 32 * g;  // this lane's 32 columns
    u32x4 q[NA][RT];
    float s[NA][RT][kPer];
    uint32_t z[NA][RT][kPer];
#pragma unroll
    for (int n = 0; n < NA; ++n)
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        q[n][i] = kw < cols ? *reinterpret_cast<const u32x4*>(w[n].data + size_t(row[i]) * (cols / 2) + kw / 2)
                            : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < kPer; ++p) {
          const size_t at = size_t(row[i]) * groups + min(b * kPer + p, groups - 1);
          s[n][i][p] = q4_scale(w[n], scale_type, at);
          z[n][i][p] = q4_zero(w[n], at);
        }
      }
    // Split the block's activations: 16 lanes per token, 8 columns each.
    for (int t = lane >> 4; t < nt; t += 4) {
      const int k8 = lane & 15, k = b * kBlock + 8 * k8;
      float v[8];
      uint32_t largest = 0;
      const float4* src = reinterpret_cast<const float4*>(x + size_t(tok0 + t) * cols + k);
      const float4 v0 = k < cols ? src[0] : make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 v1 = k < cols ? src[1] : make_float4(0.f, 0.f, 0.f, 0.f);
      v[0] = v0.x; v[1] = v0.y; v[2] = v0.z; v[3] = v0.w;
      v[4] = v1.x; v[5] = v1.y; v[6] = v1.z; v[7] = v1.w;
#pragma unroll
      for (int i = 0; i < 8; ++i) largest = max(largest, finite_bits(v[i]));
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) largest = max(largest, uint32_t(__shfl_xor(int(largest), off, 64)));
      float factor, back;
      block_scale(largest, factor, back);
      f16x8 hi, lo;
      split8(v, factor, hi, lo);
      const int step = WIDE ? k8 & 3 : k8 >> 2, kg = WIDE ? k8 >> 2 : k8 & 3;
      const int at = part_slot<WIDE>(step, kg, t) * 16;
      *reinterpret_cast<f16x8*>(stage + at) = hi;
      *reinterpret_cast<f16x8*>(stage + 4096 + at) = lo;
      if (k8 == 0) back_of[t] = back;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    f16x8 hi[4], lo[4];
    const int tr = min(r, nt - 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = part_slot<WIDE>(j, g, tr) * 16;
      hi[j] = *reinterpret_cast<const f16x8*>(stage + at);
      lo[j] = *reinterpret_cast<const f16x8*>(stage + 4096 + at);
    }
    f32x4 back;
#pragma unroll
    for (int e = 0; e < 4; ++e) back[e] = back_of[min(4 * g + e, nt - 1)];
#pragma unroll
    for (int n = 0; n < NA; ++n)
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        if constexpr (!WIDE) transpose4(q[n][i]);
        f32x4 part = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int p = j * kPer / 4;
          const f16x8 wq = unpack8(q[n][i][j], z[n][i][p]);
          part = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[j], wq, part, 0, 0, 0);
          part = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[j], wq, part, 0, 0, 0);
          if ((j + 1) % (4 / kPer) == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[n][i][e] = __builtin_fmaf(part[e], s[n][i][p] * back[e], acc[n][i][e]);
            part = f32x4{0.f, 0.f, 0.f, 0.f};
          }
        }
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  // The slots' tiles through LDS, added in slot order.
  __syncthreads();
  f32x4* sums = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int n = 0; n < NA; ++n)
#pragma unroll
    for (int i = 0; i < RT; ++i) sums[(wave * NT + n * RT + i) * 64 + lane] = acc[n][i];
  __syncthreads();
  for (int i = wave; i < RT; i += kSlots) {
    f32x4 v[NA];
#pragma unroll
    for (int n = 0; n < NA; ++n) {
      v[n] = sums[(n * RT + i) * 64 + lane];
#pragma unroll
      for (int sl = 1; sl < kSlots; ++sl) v[n] += sums[(sl * NT + n * RT + i) * 64 + lane];
    }
    const int at = row0 + 16 * i + r;
    if (at >= rows) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int tok = 4 * g + e;
      if (tok >= nt) break;
      float o = v[0][e];
      if constexpr (GATE) o = silu(o) * v[NA - 1][e];
      q4_store(out, rows, tok0 + tok, at, o);
    }
  }
}

// ---- many tokens: the activations are split once, by a launch of their own ----
//
// The workspace holds, per tile of 16 tokens and block of 128 columns, 8 KB of parts as the products
// take them (hi, then lo: 4 steps x 64 lanes x 16 bytes), then per tile and block the 16 powers of two.
struct Parts {
  unsigned char* parts;
  float* back;
};
constexpr int kPartBytes = 8192;
__host__ __device__ inline size_t part_tiles(int T) { return (size_t(T) + 15) / 16; }

template <bool WIDE>
__global__ void __launch_bounds__(256)
q4_split_kernel(Parts out, const float* __restrict__ x, int T, int cols, int blocks) {
  // 16 lanes per (token, block), so a workgroup is one tile and block.
  const size_t tile = blockIdx.x / blocks, b = blockIdx.x - tile * blocks;
  const int t = threadIdx.x >> 4, k8 = threadIdx.x & 15, k = int(b) * kBlock + 8 * k8;
  const size_t tok = tile * 16 + t;
  float v[8] = {};
  if (tok < size_t(T) && k < cols) {
    const float4* src = reinterpret_cast<const float4*>(x + tok * cols + k);
    const float4 v0 = src[0], v1 = src[1];
    v[0] = v0.x; v[1] = v0.y; v[2] = v0.z; v[3] = v0.w;
    v[4] = v1.x; v[5] = v1.y; v[6] = v1.z; v[7] = v1.w;
  }
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) largest = max(largest, finite_bits(v[i]));
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) largest = max(largest, uint32_t(__shfl_xor(int(largest), off, 64)));
  float factor, back;
  block_scale(largest, factor, back);
  f16x8 hi, lo;
  split8(v, factor, hi, lo);
  const int step = WIDE ? k8 & 3 : k8 >> 2, g = WIDE ? k8 >> 2 : k8 & 3;
  unsigned char* to = out.parts + (tile * blocks + b) * kPartBytes + (step * 64 + 16 * g + t) * 16;
  *reinterpret_cast<f16x8*>(to) = hi;
  *reinterpret_cast<f16x8*>(to + 4096) = lo;
  if (k8 == 0) out.back[(tile * blocks + b) * 16 + t] = back;
}

// A lane's weights, scales and zero points of one block.
template <int RT, int GROUP>
struct Q4Block {
  static constexpr int kPer = kBlock / GROUP;
  u32x4 q[RT];
  float s[RT][kPer];
  uint32_t z[RT][kPer];
  __device__ __forceinline__ void load(const Q4View& w, int scale_type, const int (&row)[RT], int b,
                                       int g, int cols, int groups) {
    const int kw = b * kBlock + 32 * g;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      q[i] = kw < cols ? *reinterpret_cast<const u32x4*>(w.data + size_t(row[i]) * (cols / 2) + kw / 2)
                       : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        const size_t at = size_t(row[i]) * groups + min(b * kPer + p, groups - 1);
        s[i][p] = q4_scale(w, scale_type, at);
        z[i][p] = q4_zero(w, at);
      }
    }
  }
};

// A few tiles of tokens: the slots' waves as in q4_few_kernel, each with its own blocks' parts straight
// from the workspace; CT tiles of 16 tokens share the weights.
template <bool GATE, int RT, int CT, int GROUP>
__global__ void __launch_bounds__(64 * kSlots)
q4_slots_kernel(Q4Out out, Parts x, Q4View w0, Q4View w1, int scale_type, int T, int rows, int cols,
                int row_groups) {
  constexpr int NA = GATE ? 2 : 1, NT = NA * RT * CT;
  constexpr int kPer = kBlock / GROUP;
  extern __shared__ __attribute__((aligned(16))) unsigned char dyn[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int tok_group = blockIdx.x / row_groups, row_group = blockIdx.x - tok_group * row_groups;
  const int row0 = row_group * 16 * RT, tok0 = tok_group * 16 * CT;
  const int blocks = (cols + kBlock - 1) / kBlock, groups = (cols + GROUP - 1) / GROUP;
  const int last_tile = (T - 1) / 16;
  int row[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) row[i] = min(row0 + 16 * i + r, rows - 1);
  f32x4 acc[NA][RT][CT];
#pragma unroll
  for (int n = 0; n < NA; ++n)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[n][i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  const Q4View w[2] = {w0, w1};
  const int b1 = slot_block(wave + 1, blocks);
  for (int b = slot_block(wave, blocks); b < b1; ++b) {
    Q4Block<RT, GROUP> wb[NA];
#pragma unroll
    for (int n = 0; n < NA; ++n) wb[n].load(w[n], scale_type, row, b, g, cols, groups);
    if constexpr (GROUP != 128) {
#pragma unroll
      for (int n = 0; n < NA; ++n)
#pragma unroll
        for (int i = 0; i < RT; ++i) transpose4(wb[n].q[i]);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const size_t at = size_t(min(tok0 / 16 + c, last_tile)) * blocks + b;
      const unsigned char* parts = x.parts + at * kPartBytes + lane * 16;
      f16x8 hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        hi[j] = *reinterpret_cast<const f16x8*>(parts + j * 1024);
        lo[j] = *reinterpret_cast<const f16x8*>(parts + 4096 + j * 1024);
      }
      const f32x4 back = *reinterpret_cast<const f32x4*>(x.back + at * 16 + 4 * g);
#pragma unroll
      for (int n = 0; n < NA; ++n)
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          f32x4 part = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int p = j * kPer / 4;
            const f16x8 wq = unpack8(wb[n].q[i][j], wb[n].z[i][p]);
            part = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[j], wq, part, 0, 0, 0);
            part = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[j], wq, part, 0, 0, 0);
            if ((j + 1) % (4 / kPer) == 0) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[n][i][c][e] = __builtin_fmaf(part[e], wb[n].s[i][p] * back[e], acc[n][i][c][e]);
              part = f32x4{0.f, 0.f, 0.f, 0.f};
            }
          }
        }
    }
  }
  f32x4* sums = reinterpret_cast<f32x4*>(dyn);
#pragma unroll
  for (int n = 0; n < NA; ++n)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int c = 0; c < CT; ++c)
        sums[(wave * NT + (n * RT + i) * CT + c) * 64 + lane] = acc[n][i][c];
  __syncthreads();
  for (int t = wave; t < RT * CT; t += kSlots) {
    f32x4 v[NA];
#pragma unroll
    for (int n = 0; n < NA; ++n) {
      v[n] = sums[(n * RT * CT + t) * 64 + lane];
#pragma unroll
      for (int sl = 1; sl < kSlots; ++sl) v[n] += sums[(sl * NT + n * RT * CT + t) * 64 + lane];
    }
    const int at = row0 + 16 * (t / CT) + r, tok1 = tok0 + 16 * (t % CT) + 4 * g;
    if (at >= rows) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (tok1 + e >= T) break;
      float o = v[0][e];
      if constexpr (GATE) o = silu(o) * v[NA - 1][e];
      q4_store(out, rows, tok1 + e, at, o);
    }
  }
}

// Prompts: 128 rows (64 of each matrix with GATE) x 128 tokens a workgroup, a wave 64 x 64 of them: 2 x 2
// waves, one to a SIMD. The tokens' parts of a block reach LDS by DMA (64 KB, two stages, the next under
// way while a block is multiplied); the weights go from memory to registers, where a wave unpacks them
// once for its 64 tokens. All blocks are walked in turn, the slots' sums folded at their ends.
template <bool GATE, int GROUP>
__global__ void __launch_bounds__(256, 1)
q4_tiles_kernel(Q4Out out, Parts x, Q4View w0, Q4View w1, int scale_type, int T, int rows, int cols,
                int row_tiles, int tok_tiles) {
  constexpr int NA = GATE ? 2 : 1, RT = 4, CT = 4, RM = RT / NA;  // RM: row tiles per matrix
  constexpr int kPer = kBlock / GROUP;
  constexpr int kStage = 8 * kPartBytes;
  extern __shared__ __attribute__((aligned(16))) unsigned char dyn[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15, wm = wave >> 1, wn = wave & 1;
  int row_tile, tok_tile;
  tile_of_block<GATE>(blockIdx.x, row_tiles, tok_tiles, row_tile, tok_tile);
  const int row0 = (row_tile * 2 + wm) * 16 * RM, tok0 = tok_tile * 128;
  const int blocks = (cols + kBlock - 1) / kBlock, groups = (cols + GROUP - 1) / GROUP;
  const int last_tile = (T - 1) / 16;
  int row[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) row[i] = min(row0 + 16 * i + r, rows - 1);
  const Q4View w[2] = {w0, w1};
  const unsigned base = lds_address(dyn);
  // Wave i brings token tiles 2i and 2i + 1 of a block: 16 transfers of 1 KB.
  auto stage = [&](int b, int s) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const size_t at = size_t(min(tok_tile * 8 + 2 * wave + c, last_tile)) * blocks + b;
      const unsigned char* src = x.parts + at * kPartBytes + lane * 16;
      const unsigned to = base + s * kStage + (2 * wave + c) * kPartBytes;
#pragma unroll
      for (int j = 0; j < 8; ++j) dma16(src + j * 1024, to + j * 1024);
    }
  };
  size_t tile_at[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) tile_at[c] = size_t(min(tok_tile * 8 + 4 * wn + c, last_tile)) * blocks;

  f32x4 total[RT][CT], acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      total[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
      acc[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  Q4Block<RM, GROUP> next[NA];
  f32x4 next_back[CT];
  auto fetch = [&](int b) {
#pragma unroll
    for (int n = 0; n < NA; ++n) next[n].load(w[n], scale_type, row, b, g, cols, groups);
#pragma unroll
    for (int c = 0; c < CT; ++c)
      next_back[c] = *reinterpret_cast<const f32x4*>(x.back + (tile_at[c] + b) * 16 + 4 * g);
  };
  stage(0, 0);
  fetch(0);
  int b = 0;
  for (int slot = 0; slot < kSlots; ++slot) {
    const int b1 = slot_block(slot + 1, blocks);
    for (; b < b1; ++b) {
      wait_vmcnt<0>();
      __syncthreads();
      Q4Block<RM, GROUP> wb[NA];
      f32x4 back[CT];
#pragma unroll
      for (int n = 0; n < NA; ++n) wb[n] = next[n];
#pragma unroll
      for (int c = 0; c < CT; ++c) back[c] = next_back[c];
      if (b + 1 < blocks) {
        fetch(b + 1);
        stage(b + 1, (b + 1) & 1);
      }
      if constexpr (GROUP != 128) {
#pragma unroll
        for (int n = 0; n < NA; ++n)
#pragma unroll
          for (int i = 0; i < RM; ++i) transpose4(wb[n].q[i]);
      }
      const unsigned char* parts = dyn + (b & 1) * kStage + 4 * wn * kPartBytes + lane * 16;
      f32x4 part[RT][CT];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int p = j * kPer / 4;
        f16x8 hi[CT], lo[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          hi[c] = *reinterpret_cast<const f16x8*>(parts + c * kPartBytes + j * 1024);
          lo[c] = *reinterpret_cast<const f16x8*>(parts + c * kPartBytes + 4096 + j * 1024);
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const Q4Block<RM, GROUP>& wi = wb[i / RM];
          const f16x8 wq = unpack8(wi.q[i % RM][j], wi.z[i % RM][p]);
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            if (j % (4 / kPer) == 0) part[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
            part[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[c], wq, part[i][c], 0, 0, 0);
          }
#pragma unroll
          for (int c = 0; c < CT; ++c)
            part[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[c], wq, part[i][c], 0, 0, 0);
          if ((j + 1) % (4 / kPer) == 0) {
            const float s = wi.s[i % RM][p];
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[i][c][e] = __builtin_fmaf(part[i][c][e], s * back[c][e], acc[i][c][e]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        total[i][c] = slot == 0 ? acc[i][c] : total[i][c] + acc[i][c];
        acc[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
  }
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int at = row0 + 16 * i + r;
    if (at >= rows) continue;
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int tok = tok0 + (4 * wn + c) * 16 + 4 * g + e;
        if (tok >= T) continue;
        float o = total[i][c][e];
        if constexpr (GATE) o = silu(o) * total[RM + i][c][e];
        q4_store(out, rows, tok, at, o);
      }
  }
}

int check_matrix_q4(const ie_matrix_q4& m, const char* who) {
  if (!m.data || !m.scale || m.rows <= 0 || m.cols <= 0)
    return fail(IE_HIP_EINVAL, std::string(who) + ": empty weight matrix");
  if (m.group != 32 && m.group != 64 && m.group != 128)
    return fail(IE_HIP_EINVAL, std::string(who) + ": groups must be of 32, 64 or 128 columns");
  if (m.cols % 32)
    return fail(IE_HIP_EINVAL, std::string(who) + ": cols must be a multiple of 32");
  if (m.scale_dtype != IE_KV_F32 && m.scale_dtype != IE_KV_F16 && m.scale_dtype != IE_KV_BF16)
    return fail(IE_HIP_EINVAL, std::string(who) + ": unknown scale_dtype " + std::to_string(m.scale_dtype));
  if (reinterpret_cast<uintptr_t>(m.data) & 15)
    return fail(IE_HIP_EINVAL, std::string(who) + ": the weights must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(m.scale) & (m.scale_dtype == IE_KV_F32 ? 3 : 1))
    return fail(IE_HIP_EINVAL, std::string(who) + ": the scales are not aligned to their type");
  return IE_HIP_OK;
}

// Tokens that a launch splits by itself; more are split once into the workspace.
constexpr int kFewTokens = 16;

struct Q4Launch {
  Q4Out out;
  const float* x;
  Q4View w0, w1;
  int scale_type, T, rows, cols;
  Parts parts;
  hipStream_t stream;
  const char* who;

  int too_many() const { return fail(IE_HIP_EINVAL, std::string(who) + ": too many rows or tokens"); }
  template <bool GATE, int RT, int GROUP>
  int few() const {
    const int64_t row_groups = (int64_t(rows) + 16 * RT - 1) / (16 * RT);
    if (row_groups * 64 * kSlots > int64_t(UINT32_MAX)) return too_many();
    hipLaunchKernelGGL((q4_few_kernel<GATE, RT, GROUP>), dim3(unsigned(row_groups)), dim3(64 * kSlots), 0,
                       stream, out, x, w0, w1, scale_type, T, rows, cols, int(row_groups));
    return IE_HIP_OK;
  }
  template <bool GATE, int RT, int CT, int GROUP>
  int slots() const {
    constexpr int kLds = kSlots * (GATE ? 2 : 1) * RT * CT * 1024;
    const auto kernel = q4_slots_kernel<GATE, RT, CT, GROUP>;
    if (kLds > 64 * 1024) {
      static const hipError_t attr = hipFuncSetAttribute(
          reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
      if (int rc = check_hip(attr, "hipFuncSetAttribute(q4)")) return rc;
    }
    const int64_t row_groups = (int64_t(rows) + 16 * RT - 1) / (16 * RT);
    const int64_t grid = row_groups * ((int64_t(T) + 16 * CT - 1) / (16 * CT));
    if (grid * 64 * kSlots > int64_t(UINT32_MAX)) return too_many();
    hipLaunchKernelGGL(kernel, dim3(unsigned(grid)), dim3(64 * kSlots), kLds, stream, out, parts, w0, w1,
                       scale_type, T, rows, cols, int(row_groups));
    return IE_HIP_OK;
  }
  template <bool GATE, int GROUP>
  int tiles() const {
    constexpr int kLds = 2 * 8 * kPartBytes, kRows = GATE ? 64 : 128;
    const auto kernel = q4_tiles_kernel<GATE, GROUP>;
    static const hipError_t attr = hipFuncSetAttribute(
        reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (int rc = check_hip(attr, "hipFuncSetAttribute(q4)")) return rc;
    const int64_t row_tiles = (int64_t(rows) + kRows - 1) / kRows, tok_tiles = (int64_t(T) + 127) / 128;
    if (row_tiles * tok_tiles * 256 > int64_t(UINT32_MAX)) return too_many();
    hipLaunchKernelGGL(kernel, dim3(unsigned(row_tiles * tok_tiles)), dim3(256), kLds, stream, out, parts,
                       w0, w1, scale_type, T, rows, cols, int(row_tiles), int(tok_tiles));
    return IE_HIP_OK;
  }
  template <bool GATE, int GROUP>
  int run() const {
    const int64_t row_tiles = (int64_t(rows) + 15) / 16;
    const int64_t cus = device_compute_units();
    if (T <= kFewTokens) {
      if (row_tiles >= 8 * cus) return few<GATE, 4, GROUP>();
      if (row_tiles >= 4 * cus) return few<GATE, 2, GROUP>();
      return few<GATE, 1, GROUP>();
    }
    const int64_t tok_tiles = (int64_t(T) + 15) / 16, blocks = (int64_t(cols) + kBlock - 1) / kBlock;
    if (tok_tiles * blocks * 256 > int64_t(UINT32_MAX)) return too_many();
    hipLaunchKernelGGL(q4_split_kernel<GROUP == 128>, dim3(unsigned(tok_tiles * blocks)), dim3(256), 0,
                       stream, parts, x, T, cols, int(blocks));
    const int64_t big = ((int64_t(rows) + (GATE ? 63 : 127)) / (GATE ? 64 : 128)) * ((int64_t(T) + 127) / 128);
    if (2 * big >= cus) return tiles<GATE, GROUP>();
    if (T <= 32) return row_tiles >= 4 * cus ? slots<GATE, 2, 2, GROUP>() : slots<GATE, 1, 2, GROUP>();
    if constexpr (!GATE)
      if (row_tiles >= 2 * cus) return slots<GATE, 2, 4, GROUP>();
    return slots<GATE, 1, 4, GROUP>();
  }
  template <bool GATE>
  int run(int group) const {
    return group == 128 ? run<GATE, 128>() : group == 64 ? run<GATE, 64>() : run<GATE, 32>();
  }
};

Parts parts_of(void* workspace, int T, int cols) {
  unsigned char* base = static_cast<unsigned char*>(workspace);
  const size_t n = part_tiles(T) * ((size_t(cols) + kBlock - 1) / kBlock);
  return Parts{base, reinterpret_cast<float*>(base + n * kPartBytes)};
}

int launch_q4(bool gate, float* y, const float* x, const ie_matrix_q4& w, const ie_matrix_q4* w2,
              const float* bias, int T, int accumulate, void* workspace, hipStream_t stream,
              const char* who, RowSplit split = RowSplit{nullptr, nullptr, 0, 0}) {
  if (split.split0 == 0 && split.split1 == 0) split.split0 = split.split1 = w.rows;
  if (int rc = check_matrix_q4(w, who)) return rc;
  if (w2) {
    if (int rc = check_matrix_q4(*w2, who)) return rc;
    if (w2->rows != w.rows || w2->cols != w.cols || w2->group != w.group ||
        w2->scale_dtype != w.scale_dtype)
      return fail(IE_HIP_EINVAL, std::string(who) + ": gate and up shapes or formats differ");
  }
  if (T < 0) return fail(IE_HIP_EINVAL, std::string(who) + ": T < 0");
  if (T == 0) return IE_HIP_OK;
  if (!y || !x) return fail(IE_HIP_EINVAL, std::string(who) + ": null pointer");
  if (reinterpret_cast<uintptr_t>(x) & 15)
    return fail(IE_HIP_EINVAL, std::string(who) + ": x must be 16-byte aligned");
  const size_t need = ie_hip_matmul_q4_workspace_bytes(T, w.cols);
  if (need && !workspace)
    return fail(IE_HIP_EINVAL, std::string(who) + ": " + std::to_string(T) +
                                   " tokens need a workspace (ie_hip_matmul_q4_workspace_bytes)");
  if (need && (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(IE_HIP_EINVAL, std::string(who) + ": the workspace must be 16-byte aligned");
  const Q4Launch launch{Q4Out{y, bias, accumulate, split},
                        x,
                        Q4View{static_cast<const uint8_t*>(w.data), w.scale,
                               static_cast<const uint8_t*>(w.zero)},
                        w2 ? Q4View{static_cast<const uint8_t*>(w2->data), w2->scale,
                                    static_cast<const uint8_t*>(w2->zero)}
                           : Q4View{nullptr, nullptr, nullptr},
                        w.scale_dtype,
                        T,
                        w.rows,
                        w.cols,
                        parts_of(workspace, T, w.cols),
                        stream,
                        who};
  if (int rc = gate ? launch.run<true>(w.group) : launch.run<false>(w.group)) return rc;
  return check_launch(who);
}

}  // namespace
}  // namespace iehip

using namespace iehip;

extern "C" size_t ie_hip_matmul_q4_workspace_bytes(int T, int cols) {
  if (T <= kFewTokens || cols <= 0) return 0;
  return part_tiles(T) * ((size_t(cols) + kBlock - 1) / kBlock) * (kPartBytes + 64);
}

extern "C" int ie_hip_matmul_q4(float* y, const float* x, ie_matrix_q4 w, const float* bias, int T,
                                int accumulate, void* workspace, hipStream_t stream) {
  clear_error();
  return launch_q4(false, y, x, w, nullptr, bias, T, accumulate, workspace, stream, "matmul_q4");
}

extern "C" int ie_hip_qkv_proj_q4(float* q, float* k, float* v, const float* x, ie_matrix_q4 w_qkv,
                                  const float* b_qkv, int T, int q_dim, int kv_dim, void* workspace,
                                  hipStream_t stream) {
  clear_error();
  if (q_dim <= 0 || kv_dim <= 0 || int64_t(w_qkv.rows) != q_dim + 2 * int64_t(kv_dim))
    return fail(IE_HIP_EINVAL, "qkv_proj_q4: weight rows must be q_dim + 2 kv_dim");
  if (T > 0 && (!q || !k || !v)) return fail(IE_HIP_EINVAL, "qkv_proj_q4: null pointer");
  return launch_q4(false, q, x, w_qkv, nullptr, b_qkv, T, 0, workspace, stream, "qkv_proj_q4",
                   RowSplit{k, v, q_dim, q_dim + kv_dim});
}

extern "C" int ie_hip_gate_up_silu_q4(float* out, const float* x, ie_matrix_q4 w_gate,
                                      ie_matrix_q4 w_up, int T, void* workspace, hipStream_t stream) {
  clear_error();
  return launch_q4(true, out, x, w_gate, &w_up, nullptr, T, 0, workspace, stream, "gate_up_silu_q4");
}
