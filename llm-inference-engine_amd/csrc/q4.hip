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
#include <atomic>

#include "common.hpp"
#include "matmul_tiled.hpp"
#include "mfma.hpp"

namespace iehip {
namespace {

constexpr int kBlock = 128;  // columns that share an activation scale: 4 products of 32
constexpr int kSlots = 8;
constexpr int kMaxCols = 1 << 24;  // a tile's byte offsets from its first row fit 32 bits

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// First block of slot i of n blocks.
__host__ __device__ __forceinline__ int slot_block(int i, int n) { return int(int64_t(i) * n / kSlots); }

// One 4-bit matrix as a kernel sees it.
struct Q4View {
  const uint8_t* data;
  const uint8_t* scale;
  const uint8_t* zero;  // null: 8 everywhere
};
__device__ const uint8_t kEight[4] = {8, 8, 8, 8};

// A group's zero point as the two pairs of f16 constants that take it off its weights.
struct Q4Zero {
  f16x2 low, high;  // 1024 + z; -(64 + z)
};
__device__ __forceinline__ Q4Zero q4_zero(uint32_t z) {
  const _Float16 h = static_cast<_Float16>(-64.0f - static_cast<float>(z));
  return Q4Zero{__builtin_bit_cast(f16x2, 0x64006400u + z * 0x10001u), f16x2{h, h}};
}

// 8 weights of a word, less their zero point, as f16: element order 0, 4, 1, 5, 2, 6, 3, 7.
// A nibble in the low bits of an f16 of 1,024 reads 1024 + q; one four bits up reads 1024 + 16 q,
// which an fma with 1/16 brings down: every step is exact, 9 instructions for 8 weights.
__device__ __forceinline__ f16x8 unpack8(uint32_t w, const Q4Zero& z) {
  uint32_t base = 0x64006400u;
  asm("" : "+v"(base));  // in a register: of two literals the compiler makes an and and an or
  const uint32_t h = w >> 8;
  auto pair = [&](uint32_t v, uint32_t mask) { return __builtin_bit_cast(f16x2, (v & mask) | base); };
  const f16x2 sixteenth = {_Float16(0.0625f), _Float16(0.0625f)};
  const f16x2 a = pair(w, 0x000F000Fu) - z.low;
  const f16x2 b = __builtin_elementwise_fma(pair(w, 0x00F000F0u), sixteenth, z.high);
  const f16x2 c = pair(h, 0x000F000Fu) - z.low;
  const f16x2 d = __builtin_elementwise_fma(pair(h, 0x00F000F0u), sixteenth, z.high);
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

// Columns 8 k8 .. 8 k8 + 7 of a block belong to step `step` of lane group g of the products. WIDE
// (groups of 128): step j holds columns 32 g + 8 j of lane group g, as the weights are loaded; otherwise
// step j is columns 32 j .. 32 j + 31 and the weights are transposed to it.
template <bool WIDE>
__device__ __forceinline__ int k8_of(int step, int g) {
  return WIDE ? 4 * g + step : 4 * step + g;
}

// A block's parts in LDS: 16 bytes per (k8, token), hi then lo, TP token places. Of 8 and 16 places they
// are permuted by k8, so that the 16 lanes that write a token's block hit every bank.
template <int TP>
struct Places {
  static constexpr int kHalf = 16 * TP * 16, kBytes = 2 * kHalf;
  __device__ __forceinline__ static int at(int k8, int tok) {
    return (k8 * TP + (TP >= 8 ? tok ^ (k8 % TP) : tok)) * 16;
  }
};

// A lane's 8 activations of a (token, block), split among the 16 lanes that hold the block.
__device__ __forceinline__ float split_lane(const float (&v)[8], f16x8& hi, f16x8& lo) {
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) largest = max(largest, finite_bits(v[i]));
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) largest = max(largest, uint32_t(__shfl_xor(int(largest), off, 64)));
  float factor, back;
  block_scale(largest, factor, back);
  split8(v, factor, hi, lo);
  return back;
}
__device__ __forceinline__ void load8(float (&v)[8], const float* src, bool in) {
  const float4* p = reinterpret_cast<const float4*>(src);
  const float4 a = in ? p[0] : make_float4(0.f, 0.f, 0.f, 0.f);
  const float4 b = in ? p[1] : make_float4(0.f, 0.f, 0.f, 0.f);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// A lane's rows of RT row tiles from row0 on: byte offsets from the first of them, which is uniform.
template <int RT, int GROUP, bool S32>
struct Q4Rows {
  static constexpr int kPer = kBlock / GROUP, kSize = S32 ? 4 : 2;
  const uint8_t *data, *scale, *zero;
  uint32_t q[RT], s[RT], z[RT];
  int last_word, groups, step;
  bool bf16;
  __device__ __forceinline__ Q4Rows(const Q4View& w, int scale_type, int row0, int rows, int cols, int r) {
    const int first = min(row0, rows - 1);
    groups = (cols + GROUP - 1) / GROUP;
    step = w.zero ? 1 : 0;
    bf16 = scale_type == IE_KV_BF16;
    last_word = cols / 2 - 16;
    data = w.data + size_t(first) * (cols / 2);
    scale = w.scale + size_t(first) * groups * kSize;
    zero = w.zero ? w.zero + size_t(first) * groups : kEight;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const uint32_t row = min(16 * i + r, rows - 1 - first);
      q[i] = row * (cols / 2);
      s[i] = row * groups * kSize;
      z[i] = row * groups * step;
    }
  }
};

// A lane's weights of one block, with the scale and zero point of the group that step g of the block
// falls into (so that the four lane groups hold a block's between them). Lanes past the last column take
// the columns before it: their activations are 0.
template <int RT, int GROUP, bool S32>
struct Q4Block {
  static constexpr int kPer = kBlock / GROUP;
  u32x4 q[RT];
  uint32_t s[RT], z[RT];
  __device__ __forceinline__ void load(const Q4Rows<RT, GROUP, S32>& w, int b, int g) {
    const uint32_t k = min(b * (kBlock / 2) + 16 * g, w.last_word);
    const uint32_t group = min(b * kPer + g * kPer / 4, w.groups - 1);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      q[i] = *reinterpret_cast<const u32x4*>(w.data + (w.q[i] + k));
      const uint8_t* at = w.scale + (w.s[i] + group * w.kSize);
      if constexpr (S32)
        s[i] = *reinterpret_cast<const uint32_t*>(at);
      else
        s[i] = *reinterpret_cast<const uint16_t*>(at);
      z[i] = w.zero[w.z[i] + group * w.step];
    }
  }
};

// One of its row tiles ready to multiply: the words' order and each step's scale and zero point.
template <int GROUP, bool S32>
struct Q4Tile {
  static constexpr int kPer = kBlock / GROUP;
  u32x4 q;
  float scale[kPer];
  Q4Zero zero[kPer];
  __device__ __forceinline__ void set(int p, uint32_t s, uint32_t z, bool bf16) {
    if constexpr (S32)
      scale[p] = __uint_as_float(s);
    else
      scale[p] = bf16 ? __uint_as_float(s << 16) : f16_bits_to_f32(uint16_t(s));
    zero[p] = q4_zero(z);
  }
  __device__ __forceinline__ Q4Tile(const u32x4& words, const uint32_t (&s)[kPer], const uint32_t (&z)[kPer],
                                    bool bf16)
      : q(words) {
    if constexpr (kPer > 1) transpose4(q);
#pragma unroll
    for (int p = 0; p < kPer; ++p) set(p, s[p], z[p], bf16);
  }
  template <int RT>
  __device__ __forceinline__ Q4Tile(const Q4Block<RT, GROUP, S32>& b, int i, bool bf16) : q(b.q[i]) {
    u32x4 s = u32x4(b.s[i]), z = u32x4(b.z[i]);
    if constexpr (kPer > 1) {
      transpose4(q);
      if constexpr (S32) {
        transpose4(s);
        transpose4(z);
      } else {
        s = u32x4(b.s[i] | b.z[i] << 16);
        transpose4(s);
        z = s >> 16;
        s &= 0xFFFF;
      }
    }
#pragma unroll
    for (int p = 0; p < kPer; ++p) set(p, s[p * 4 / kPer], z[p * 4 / kPer], bf16);
  }
  __device__ __forceinline__ f16x8 weights(int step) const { return unpack8(q[step], zero[step * kPer / 4]); }
  __device__ __forceinline__ void unpack(f16x8 (&wq)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) wq[j] = weights(j);
  }
  // The tile times one tile of tokens, added to acc group by group.
  __device__ __forceinline__ static void multiply(const f16x8 (&wq)[4], const float (&scale)[kPer],
                                                  const f16x8 (&hi)[4], const f16x8 (&lo)[4],
                                                  const f32x4& back, f32x4& acc) {
    f32x4 part = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      part = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[j], wq[j], part, 0, 0, 0);
      part = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[j], wq[j], part, 0, 0, 0);
      if ((j + 1) % (4 / kPer) == 0) {
        const float sc = scale[j * kPer / 4];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(part[e], sc * back[e], acc[e]);
        part = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  }
};

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

// Global -> LDS transfers of 4, 2 or 1 bytes a lane, widened to the lane's word at lds + 4 lane; as dma16.
template <int BYTES>
__device__ __forceinline__ void dma_word(const void* base, unsigned offset, unsigned lds) {
  if constexpr (BYTES == 4)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
                 :
                 : "v"(offset), "s"(base), "s"(lds)
                 : "memory", "m0");
  else if constexpr (BYTES == 2)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_ushort %0, %1"
                 :
                 : "v"(offset), "s"(base), "s"(lds)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_ubyte %0, %1"
                 :
                 : "v"(offset), "s"(base), "s"(lds)
                 : "memory", "m0");
}

__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// A barrier for data in LDS that leaves loads from memory under way.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// LDS of q4_few_kernel: two stages a wave, the slots' sums, the activations' parts and powers.
template <bool GATE, int GROUP, int TP, int SB, bool SPLIT>
struct FewShape {
  static constexpr int NA = GATE ? 2 : 1, kPer = kBlock / GROUP;
  static constexpr int kScales = (SB * kPer + 3) / 4;  // transfers of 4 groups' scales
  static constexpr int kUnit = SB * 1024 + kScales * 512, kStage = NA * kUnit;
  static constexpr int kLoads = NA * (SB + 2 * kScales);
  static constexpr int kSums = kSlots * 2 * kStage, kParts = kSums + (SPLIT ? kSlots * NA * 1024 : 0);
  static constexpr int64_t bytes(int64_t blocks) { return kParts + blocks * (Places<TP>::kBytes + 4 * TP); }
};

// Up to 16 tokens whose parts fit LDS beside the rest: a workgroup splits them once, then its waves stream
// weights past them through two stages of LDS each: SB blocks of 16 rows (of each matrix) by DMA, 64 SB
// contiguous bytes of a row a transfer, the next stage under way while one is multiplied. SPLIT: a
// workgroup takes row tiles in turn, wave i slot i, and the slots are added through LDS. Otherwise (row
// tiles enough for every wave) a wave takes row tiles of its own, all blocks, folding slots as it passes
// their ends, and waits for nobody. TP: token places, 1, 4, 8 or 16.
// Loads straight to registers touch 16 rows 64 bytes at a time, which bounds them (8,192 x 8,192 at 1
// token: 22 us so).
template <bool GATE, int GROUP, bool S32, int TP, int SB, bool SPLIT>
__global__ void __launch_bounds__(64 * kSlots)
q4_few_kernel(Q4Out out, const float* __restrict__ x, Q4View w0, Q4View w1, int scale_type, int T, int rows,
              int cols, int row_tiles) {
  using F = FewShape<GATE, GROUP, TP, SB, SPLIT>;
  using P = Places<TP>;
  constexpr int NA = F::NA, kPer = F::kPer, kSize = S32 ? 4 : 2, kWide = 4 * SB;  // kWide: words x 4 of a row
  constexpr int kShift = SB == 4 ? 0 : SB == 2 ? 1 : 2;
  constexpr bool WIDE = GROUP == kBlock;
  extern __shared__ __attribute__((aligned(16))) unsigned char dyn[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int blocks = (cols + kBlock - 1) / kBlock, groups = (cols + GROUP - 1) / GROUP;
  const int b0 = SPLIT ? slot_block(wave, blocks) : 0, b1 = SPLIT ? slot_block(wave + 1, blocks) : blocks;
  const int first = SPLIT ? blockIdx.x : blockIdx.x * kSlots + wave;
  const int hop = SPLIT ? gridDim.x : gridDim.x * kSlots;
  const bool bf16 = scale_type == IE_KV_BF16;
  unsigned char* ring = dyn + wave * 2 * F::kStage;
  const unsigned ring_lds = lds_address(ring);
  unsigned char* parts = dyn + F::kParts;
  float* backs = reinterpret_cast<float*>(parts + size_t(blocks) * P::kBytes);

  auto issue = [&](int tile, int b, int stage) {
    const int row0 = tile * 16, last_row = rows - 1 - row0;
#pragma unroll
    for (int n = 0; n < NA; ++n) {
      const Q4View& w = n ? w1 : w0;
      const unsigned to = ring_lds + stage * F::kStage + n * F::kUnit;
      const uint8_t* data = w.data + size_t(row0) * (cols / 2);
#pragma unroll
      for (int i = 0; i < SB; ++i) {
        const int row = 64 / kWide * i + lane / kWide;
        const int word = min(4 * b + ((lane % kWide) ^ (row >> kShift)), cols / 32 - 1);
        dma16_at(data, uint32_t(min(row, last_row)) * (cols / 2) + word * 16, to + i * 1024);
      }
      const uint32_t step = w.zero ? 1 : 0;
      const uint8_t* scale = w.scale + size_t(row0) * groups * kSize;
      const uint8_t* zero = w.zero ? w.zero + size_t(row0) * groups : kEight;
#pragma unroll
      for (int p = 0; p < F::kScales; ++p) {
        const uint32_t at = uint32_t(min(r, last_row)) * groups + min(b * kPer + 4 * p + g, groups - 1);
        dma_word<kSize>(scale, at * kSize, to + SB * 1024 + p * 256);
        dma_word<1>(zero, at * step, to + SB * 1024 + (F::kScales + p) * 256);
      }
    }
  };
  // One block a stage, which is a slot's whole share: two stages go out before the activations are split.
  // More blocks: the next stage goes out before a stage is multiplied (8,192 x 8,192 at 1 token 12.2 us,
  // two ahead and the next after it 13.0).
  constexpr bool kTwoAhead = SB == 1;
  int ahead_tile = first, ahead_b = b0;
  auto issue_next = [&](int stage) {
    if (ahead_tile >= row_tiles || b0 >= b1) return false;
    issue(ahead_tile, ahead_b, stage);
    ahead_b += SB;
    if (ahead_b >= b1) {
      ahead_b = b0;
      ahead_tile += hop;
    }
    return true;
  };
  issue_next(0);
  bool more = kTwoAhead && issue_next(1);  // whether the stage after the one at hand is under way
  int stage = 0;
  for (int u = threadIdx.x >> 4; u < blocks * T; u += 32) {
    const int b = u / T, tok = u - b * T, k8 = r, k = b * kBlock + 8 * k8;
    float v[8];
    load8(v, x + size_t(tok) * cols + (k < cols ? k : 0), k < cols);
    f16x8 hi, lo;
    const float back = split_lane(v, hi, lo);
    unsigned char* to = parts + b * P::kBytes + P::at(k8, tok);
    *reinterpret_cast<f16x8*>(to) = hi;
    *reinterpret_cast<f16x8*>(to + P::kHalf) = lo;
    if (k8 == 0) backs[b * TP + tok] = back;
  }
  lds_barrier();
  for (int tile = first; tile < row_tiles; tile += hop) {
    f32x4 total[NA], acc[NA];
#pragma unroll
    for (int n = 0; n < NA; ++n) total[n] = acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    int slot = 0;
    for (int b = b0; b < b1; b += SB) {
      if constexpr (!kTwoAhead) {
        wait_lds();  // the other stage has been read
        more = issue_next(stage ^ 1);
      }
      if (more)
        wait_vmcnt<F::kLoads>();
      else
        wait_vmcnt<0>();
      asm volatile("" ::: "memory");
      const unsigned char* from = ring + stage * F::kStage;
#pragma unroll
      for (int sb = 0; sb < SB; ++sb) {
        if (b + sb >= b1) break;
        const unsigned char* at = parts + size_t(b + sb) * P::kBytes;
        f16x8 hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned char* part = at + P::at(k8_of<WIDE>(j, g), TP == 1 ? 0 : min(r, T - 1));
          hi[j] = *reinterpret_cast<const f16x8*>(part);
          lo[j] = *reinterpret_cast<const f16x8*>(part + P::kHalf);
        }
        f32x4 back;
#pragma unroll
        for (int e = 0; e < 4; ++e) back[e] = backs[(b + sb) * TP + (TP == 1 ? 0 : min(4 * g + e, T - 1))];
#pragma unroll
        for (int n = 0; n < NA; ++n) {
          const unsigned char* unit = from + n * F::kUnit;
          const u32x4 q = *reinterpret_cast<const u32x4*>(unit + (r * kWide + ((4 * sb + g) ^ (r >> kShift))) * 16);
          const uint32_t* words = reinterpret_cast<const uint32_t*>(unit + SB * 1024);
          uint32_t sc[kPer], ze[kPer];
#pragma unroll
          for (int p = 0; p < kPer; ++p) {
            const int in = sb * kPer + p;
            sc[p] = words[in / 4 * 64 + in % 4 * 16 + r];
            if constexpr (!S32) sc[p] &= 0xFFFFu;
            ze[p] = words[(F::kScales + in / 4) * 64 + in % 4 * 16 + r] & 0xFFu;
          }
          const Q4Tile<GROUP, S32> t(q, sc, ze, bf16);
          f16x8 wq[4];
          t.unpack(wq);
          t.multiply(wq, t.scale, hi, lo, back, acc[n]);
        }
        if constexpr (!SPLIT)
          while (slot < kSlots && slot_block(slot + 1, blocks) <= b + sb + 1) {
#pragma unroll
            for (int n = 0; n < NA; ++n) {
              total[n] += acc[n];
              acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            ++slot;
          }
      }
      if constexpr (kTwoAhead) {
        wait_lds();  // the stage has been read
        more = issue_next(stage);
      }
      stage ^= 1;
    }
    if constexpr (SPLIT) {
      f32x4* sums = reinterpret_cast<f32x4*>(dyn + F::kSums);
      lds_barrier();  // the last tile's sums have been read
#pragma unroll
      for (int n = 0; n < NA; ++n) sums[(wave * NA + n) * 64 + lane] = acc[n];
      lds_barrier();
      if (wave != 0) continue;
#pragma unroll
      for (int n = 0; n < NA; ++n)
#pragma unroll
        for (int sl = 0; sl < kSlots; ++sl) total[n] += sums[(sl * NA + n) * 64 + lane];
    }
    const int at = tile * 16 + r;
    if (at >= rows) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int tok = 4 * g + e;
      if (tok >= T) break;
      float o = total[0][e];
      if constexpr (GATE) o = silu(o) * total[NA - 1][e];
      q4_store(out, rows, tok, at, o);
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
  const bool in = tok < size_t(T) && k < cols;
  float v[8];
  load8(v, x + (in ? tok * cols + k : 0), in);
  f16x8 hi, lo;
  const float back = split_lane(v, hi, lo);
  const int step = WIDE ? k8 & 3 : k8 >> 2, g = WIDE ? k8 >> 2 : k8 & 3;
  unsigned char* to = out.parts + (tile * blocks + b) * kPartBytes + (step * 64 + 16 * g + t) * 16;
  *reinterpret_cast<f16x8*>(to) = hi;
  *reinterpret_cast<f16x8*>(to + 4096) = lo;
  if (k8 == 0) out.back[(tile * blocks + b) * 16 + t] = back;
}

// What the split kernel leaves of a tile of tokens and a block, to the same bits, made by the wave itself:
// a lane has 32 columns of token `tok`.
template <bool WIDE>
__device__ __forceinline__ void split_tile(f16x8 (&hi)[4], f16x8 (&lo)[4], f32x4& back, const float* x,
                                           int tok, int T, int cols, int b, int g) {
  float v[4][8];
  uint32_t largest = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = b * kBlock + 8 * k8_of<WIDE>(j, g);
    const bool in = tok < T && k < cols;
    load8(v[j], x + (in ? size_t(tok) * cols + k : 0), in);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = max(largest, finite_bits(v[j][i]));
#pragma unroll
  for (int off = 32; off > 8; off >>= 1) largest = max(largest, uint32_t(__shfl_xor(int(largest), off, 64)));
  float factor, mine;
  block_scale(largest, factor, mine);
#pragma unroll
  for (int j = 0; j < 4; ++j) split8(v[j], factor, hi[j], lo[j]);
#pragma unroll
  for (int e = 0; e < 4; ++e) back[e] = __shfl(mine, 4 * g + e, 64);
}

// More tokens than q4_few_kernel's, fewer than fill the chip with q4_tiles_kernel's: wave i takes slot i of
// RT row tiles (of each matrix) by CT tiles of 16 tokens, the tokens' parts straight from the workspace
// (DIRECT: split by the wave) and held while the row tiles go past them, then the slots are added through
// LDS. What a launch reads over and over is the parts (once per group of row tiles), so row tiles come
// before token tiles: q/k/v of 300 tokens 1 x 4 tiles 10.1 us, 4 x 1 8.5; a workgroup's registers leave
// room for a second one.
template <bool GATE, int RT, int CT, int GROUP, bool S32, bool DIRECT>
__global__ void __launch_bounds__(64 * kSlots, 4)
q4_slots_kernel(Q4Out out, Parts x, const float* __restrict__ direct, Q4View w0, Q4View w1, int scale_type, int T, int rows, int cols,
                int row_groups, int tok_groups) {
  constexpr int NA = GATE ? 2 : 1, NT = NA * RT * CT;
  extern __shared__ __attribute__((aligned(16))) unsigned char dyn[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  int row_group, tok_group;
  tile_of_block<true>(blockIdx.x, row_groups, tok_groups, row_group, tok_group);
  const int row0 = row_group * 16 * RT, tok0 = tok_group * 16 * CT;
  const int blocks = (cols + kBlock - 1) / kBlock;
  const int last_tile = (T - 1) / 16;
  f32x4 acc[NA][RT][CT];
#pragma unroll
  for (int n = 0; n < NA; ++n)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[n][i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  const Q4Rows<RT, GROUP, S32> w[2] = {{w0, scale_type, row0, rows, cols, r},
                                       {GATE ? w1 : w0, scale_type, row0, rows, cols, r}};
  const int b0 = slot_block(wave, blocks), b1 = slot_block(wave + 1, blocks);
  struct Ahead {
    Q4Block<RT, GROUP, S32> w[NA];
    f16x8 hi[CT][4], lo[CT][4];
    f32x4 back[CT];
  };
  auto fetch = [&](Ahead& a, int b) {
#pragma unroll
    for (int n = 0; n < NA; ++n) a.w[n].load(w[n], b, g);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      if constexpr (DIRECT) {
        split_tile<GROUP == kBlock>(a.hi[c], a.lo[c], a.back[c], direct, tok0 + 16 * c + r, T, cols, b, g);
        continue;
      }
      const size_t at = size_t(min(tok0 / 16 + c, last_tile)) * blocks + b;
      const unsigned char* parts = x.parts + at * kPartBytes;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a.hi[c][j] = *reinterpret_cast<const f16x8*>(parts + (lane * 16 + j * 1024));
        a.lo[c][j] = *reinterpret_cast<const f16x8*>(parts + (lane * 16 + 4096 + j * 1024));
      }
      a.back[c] = *reinterpret_cast<const f32x4*>(x.back + at * 16 + 4 * g);
    }
  };
  constexpr bool kAhead = NA * RT == 1;  // one row tile leaves registers for the next block
  Ahead next;
  if (kAhead && b0 < b1) fetch(next, b0);
  for (int b = b0; b < b1; ++b) {
    if constexpr (!kAhead) fetch(next, b);
    const Ahead now = next;
    if (kAhead && b + 1 < b1) fetch(next, b + 1);
    const auto& wb = now.w;
    const auto &hi = now.hi, &lo = now.lo;
    const auto& back = now.back;
#pragma unroll
    for (int n = 0; n < NA; ++n)
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const Q4Tile<GROUP, S32> t(wb[n], i, w[0].bf16);
        f16x8 wq[4];
        t.unpack(wq);
#pragma unroll
        for (int c = 0; c < CT; ++c) t.multiply(wq, t.scale, hi[c], lo[c], back[c], acc[n][i][c]);
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
  // 4 RT CT quarter tiles, one value of a lane each.
  for (int q = wave; q < 4 * RT * CT; q += kSlots) {
    const int tile = q / 4, e = q % 4;
    const int at = row0 + 16 * (tile / CT) + r, tok = tok0 + 16 * (tile % CT) + 4 * g + e;
    float v[NA];
#pragma unroll
    for (int n = 0; n < NA; ++n) {
      v[n] = 0.f;
#pragma unroll
      for (int sl = 0; sl < kSlots; ++sl)
        v[n] += reinterpret_cast<const float*>(sums + (sl * NT + n * RT * CT + tile) * 64 + lane)[e];
    }
    if (at >= rows || tok >= T) continue;
    float o = v[0];
    if constexpr (GATE) o = silu(o) * v[NA - 1];
    q4_store(out, rows, tok, at, o);
  }
}

// q4_tiles_kernel's workgroup: WN waves of 32 tokens by 8 / WN of 64 rows (32 of each matrix with GATE), and
// its stage in LDS: the parts of 2 WN token tiles, their powers, 32 / WN row tiles' weights with their
// scales and zero points.
template <bool GATE, int WN>
struct TilesShape {
  static constexpr int WM = 8 / WN, kTokens = 32 * WN, kRows = (GATE ? 32 : 64) * WM;
  static constexpr int kTokTiles = 2 * WN, kRowTiles = 4 * WM;  // of both matrices
  static constexpr int kBacks = kTokTiles * kPartBytes, kWeights = kBacks + kTokTiles * 256;
  static constexpr int kUnit = 1024 + 512, kStage = kWeights + kRowTiles * kUnit;
};

// Prompts, and a decode batch against a matrix of many rows: a wave multiplies 64 rows (32 of each matrix)
// by 32 tokens, two waves to a SIMD, so that one's VALU work stands beside the other's products (4 waves
// of 64 x 64, which unpack half as often, one to a SIMD: 4,096 x 4,096 at 2,048 tokens 258 us). A block's
// parts and weights reach LDS by DMA (64 to 78 KB, two stages, the next under way while a block is
// multiplied: weights straight to registers 248 us, all of a block's transfers issued before its products
// 172, between them 158). All blocks are walked in turn, the slots' sums folded at their ends. WN: 4 waves
// of tokens (128), 2 up to 64 tokens, 1 up to 32.
template <bool GATE, int GROUP, bool S32, int WN>
__global__ void __launch_bounds__(512)
q4_tiles_kernel(Q4Out out, Parts x, Q4View w0, Q4View w1, int scale_type, int T, int rows, int cols,
                int row_tiles, int tok_tiles) {
  using F = TilesShape<GATE, WN>;
  constexpr int NA = GATE ? 2 : 1, RT = 4, CT = 2, RM = RT / NA;  // RM: row tiles per matrix
  constexpr int kPer = kBlock / GROUP, kSize = S32 ? 4 : 2, kMine = F::kRowTiles / 8;
  extern __shared__ __attribute__((aligned(16))) unsigned char dyn[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15, wm = wave / WN, wn = wave % WN;
  int row_tile, tok_tile;
  tile_of_block<GATE>(blockIdx.x, row_tiles, tok_tiles, row_tile, tok_tile);
  const int row0 = (row_tile * F::WM + wm) * 16 * RM, tok0 = tok_tile * F::kTokens;
  const int blocks = (cols + kBlock - 1) / kBlock, groups = (cols + GROUP - 1) / GROUP;
  const int last_tile = (T - 1) / 16;
  const bool bf16 = scale_type == IE_KV_BF16;
  const unsigned base = lds_address(dyn);
  // Of a block, a wave brings 2 WN of the parts' transfers of 1 KB, row tiles wave kMine .. of the
  // workgroup's (each a transfer of weights, of scales, of zero points), and a token tile's powers. Row
  // tile 4 wm + i is tile i of the waves wm: of matrix i / RM.
  const uint8_t *data[kMine], *scale[kMine], *zero[kMine];
  uint32_t data_row[kMine], scale_row[kMine], zero_step[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int t = wave * kMine + i;
    const Q4View& w = t % 4 >= RM ? w1 : w0;
    const int row = min((row_tile * F::WM + t / 4) * 16 * RM + t % RM * 16, rows - 1), last = rows - 1 - row;
    data[i] = w.data + size_t(row) * (cols / 2);
    scale[i] = w.scale + size_t(row) * groups * kSize;
    zero[i] = w.zero ? w.zero + size_t(row) * groups : kEight;
    zero_step[i] = w.zero ? 1 : 0;
    data_row[i] = uint32_t(min(lane / 4, last)) * (cols / 2);
    scale_row[i] = uint32_t(min(r, last)) * groups;
  }
  auto token_tile = [&](int t) { return size_t(min(tok_tile * F::kTokTiles + t, last_tile)) * blocks; };
  // In four parts, so that a block's products start before all of the next one's transfers are taken.
  auto issue = [&](int b, int s, int part) {
    const unsigned to = base + s * F::kStage;
#pragma unroll
    for (int j = part; j < 2 * WN; j += 4) {
      const int n = wave * 2 * WN + j;  // of the 16 WN transfers
      dma16_at(x.parts + (token_tile(n / 8) + b) * kPartBytes + n % 8 * 1024, lane * 16, to + n * 1024);
    }
    if (part == 3 && wave < F::kTokTiles)
      dma_word<4>(x.back + (token_tile(wave) + b) * 16, r * 4, to + F::kBacks + wave * 256);
    if (part < kMine) {
      const unsigned unit = to + F::kWeights + (wave * kMine + part) * F::kUnit;
      const int word = min(4 * b + ((lane & 3) ^ (lane >> 4)), cols / 32 - 1);
      dma16_at(data[part % kMine], data_row[part % kMine] + word * 16, unit);
      const uint32_t at = scale_row[part % kMine] + min(b * kPer + g * kPer / 4, groups - 1);
      dma_word<kSize>(scale[part % kMine], at * kSize, unit + 1024);
      dma_word<1>(zero[part % kMine], at * zero_step[part % kMine], unit + 1280);
    }
  };
  f32x4 total[RT][CT], acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      total[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
      acc[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
  for (int j = 0; j < 4; ++j) issue(0, 0, j);
  int b = 0;
  for (int slot = 0; slot < kSlots; ++slot) {
    const int b1 = slot_block(slot + 1, blocks);
    for (; b < b1; ++b) {
      // This wave's transfers have landed, then everyone's, and the other stage has been read.
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const unsigned char* from = dyn + (b & 1) * F::kStage;
      const unsigned char* parts = from + 2 * wn * kPartBytes + lane * 16;
      f16x8 hi[2][CT], lo[2][CT];
      auto read = [&](int j) {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          hi[j & 1][c] = *reinterpret_cast<const f16x8*>(parts + c * kPartBytes + j * 1024);
          lo[j & 1][c] = *reinterpret_cast<const f16x8*>(parts + c * kPartBytes + 4096 + j * 1024);
        }
      };
      read(0);
      using Tile = Q4Tile<GROUP, S32>;
      auto tile = [&](int i) {
        const unsigned char* unit = from + F::kWeights + (4 * wm + i) * F::kUnit;
        const u32x4 q = *reinterpret_cast<const u32x4*>(unit + (r * 4 + (g ^ (r >> 2))) * 16);
        uint32_t sc[kPer], ze[kPer];
#pragma unroll
        for (int p = 0; p < kPer; ++p) {
          sc[p] = reinterpret_cast<const uint32_t*>(unit + 1024)[p * 4 / kPer * 16 + r];
          if constexpr (!S32) sc[p] &= 0xFFFFu;
          ze[p] = reinterpret_cast<const uint32_t*>(unit + 1280)[p * 4 / kPer * 16 + r] & 0xFFu;
        }
        return Tile(q, sc, ze, bf16);
      };
      const Tile t[RT] = {tile(0), tile(1), tile(2), tile(3)};
      f32x4 part[RT][CT];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j < 3) read(j + 1);
        if (b + 1 < blocks) issue(b + 1, (b + 1) & 1, j);
        f16x8 wq[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) wq[i] = t[i].weights(j);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int c = 0; c < CT; ++c)
            part[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                hi[j & 1][c], wq[i], j % (4 / kPer) == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : part[i][c], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int c = 0; c < CT; ++c)
            part[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[j & 1][c], wq[i], part[i][c], 0, 0, 0);
        if ((j + 1) % (4 / kPer) == 0) {
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            const f32x4 back = *reinterpret_cast<const f32x4*>(from + F::kBacks + (2 * wn + c) * 256 + 16 * g);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[i][c][e] = __builtin_fmaf(part[i][c][e], t[i].scale[j * kPer / 4] * back[e], acc[i][c][e]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        total[i][c] += acc[i][c];
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
        const int tok = tok0 + (2 * wn + c) * 16 + 4 * g + e;
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
  if (m.cols % 32 || m.cols > kMaxCols)
    return fail(IE_HIP_EINVAL, std::string(who) + ": cols must be a multiple of 32 up to 16,777,216");
  if (m.scale_dtype != IE_KV_F32 && m.scale_dtype != IE_KV_F16 && m.scale_dtype != IE_KV_BF16)
    return fail(IE_HIP_EINVAL, std::string(who) + ": unknown scale_dtype " + std::to_string(m.scale_dtype));
  if (reinterpret_cast<uintptr_t>(m.data) & 15)
    return fail(IE_HIP_EINVAL, std::string(who) + ": the weights must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(m.scale) & (m.scale_dtype == IE_KV_F32 ? 3 : 1))
    return fail(IE_HIP_EINVAL, std::string(who) + ": the scales are not aligned to their type");
  return IE_HIP_OK;
}

constexpr int kFewLds = 160 * 1024;

// Whether the activations are split once into the workspace, by a launch of their own: more than 16
// tokens, or more than q4_few_kernel holds in LDS beside its smallest stages (95 KB of parts).
bool needs_parts(int T, int cols) {
  const int64_t places = T == 1 ? 1 : T <= 4 ? 4 : T <= 8 ? 8 : 16, blocks = (int64_t(cols) + kBlock - 1) / kBlock;
  return T > 16 || places * blocks > 184;
}

struct Q4Launch {
  Q4Out out;
  const float* x;
  Q4View w0, w1;
  int scale_type, T, rows, cols;
  Parts parts;
  hipStream_t stream;
  const char* who;

  int too_many() const { return fail(IE_HIP_EINVAL, std::string(who) + ": too many rows or tokens"); }
  // Raises a kernel's dynamic-LDS cap, once on each device: `done` is the kernel's own, a bit a device.
  template <class Kernel>
  int more_lds(Kernel kernel, int bytes, std::atomic<uint64_t>& done) const {
    int device = 0;
    if (int rc = check_hip(hipGetDevice(&device), "hipGetDevice")) return rc;
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (device < 64 && (done.load(std::memory_order_relaxed) & bit)) return IE_HIP_OK;
    if (int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, bytes),
                           "hipFuncSetAttribute(q4)"))
      return rc;
    done.fetch_or(bit, std::memory_order_relaxed);
    return IE_HIP_OK;
  }
  // False where the tokens' parts do not fit.
  template <bool GATE, int GROUP, bool S32, int TP, int SB, bool SPLIT>
  bool few_go(int64_t row_tiles, int64_t cus, int* rc) const {
    using F = FewShape<GATE, GROUP, TP, SB, SPLIT>;
    const int64_t lds = F::bytes((int64_t(cols) + kBlock - 1) / kBlock);
    if (lds > kFewLds) return false;
    const auto kernel = q4_few_kernel<GATE, GROUP, S32, TP, SB, SPLIT>;
    static std::atomic<uint64_t> done{0};
    if ((*rc = more_lds(kernel, kFewLds, done))) return true;
    const int64_t each = std::min<int64_t>(2, kFewLds / lds);  // workgroups of a compute unit
    const int64_t grid = std::min(SPLIT ? row_tiles : (row_tiles + kSlots - 1) / kSlots, each * cus);
    hipLaunchKernelGGL(kernel, dim3(unsigned(grid)), dim3(64 * kSlots), unsigned(lds), stream, out, x, w0,
                       w1, scale_type, T, rows, cols, int(row_tiles));
    return true;
  }
  template <bool GATE, int GROUP, bool S32, int TP>
  bool few(int64_t row_tiles, int64_t cus, int* rc) const {
    constexpr int kMost = GATE ? 2 : 4;  // blocks of a stage, fewer where the tokens' parts need the room
    if (row_tiles >= 8 * cus && few_go<GATE, GROUP, S32, TP, kMost, false>(row_tiles, cus, rc)) return true;
    if (cols <= kSlots * kBlock) return few_go<GATE, GROUP, S32, TP, 1, true>(row_tiles, cus, rc);
    return few_go<GATE, GROUP, S32, TP, kMost, true>(row_tiles, cus, rc) ||
           few_go<GATE, GROUP, S32, TP, kMost / 2, true>(row_tiles, cus, rc);
  }
  template <bool GATE, int RT, int CT, int GROUP, bool S32, bool DIRECT>
  int slots() const {
    constexpr int kLds = kSlots * (GATE ? 2 : 1) * RT * CT * 1024;
    static_assert(kLds <= 64 * 1024, "two workgroups of a compute unit");
    const int64_t row_groups = (int64_t(rows) + 16 * RT - 1) / (16 * RT);
    const int64_t tok_groups = (int64_t(T) + 16 * CT - 1) / (16 * CT);
    if (row_groups * tok_groups * 64 * kSlots > int64_t(UINT32_MAX)) return too_many();
    hipLaunchKernelGGL((q4_slots_kernel<GATE, RT, CT, GROUP, S32, DIRECT>), dim3(unsigned(row_groups * tok_groups)),
                       dim3(64 * kSlots), kLds, stream, out, parts, x, w0, w1, scale_type, T, rows, cols,
                       int(row_groups), int(tok_groups));
    return IE_HIP_OK;
  }
  // False where the tiles, one a compute unit, are so few that the slots take less time: theirs grows with
  // the launch, the tiles' hardly until every unit has one. Tiles and slots, us: 117 tiles of 896 columns
  // 27.8 and 26.3, 135 28.3 and 30.0; 96 tiles of 2,048 columns 42.4 and 42.6, 112 42.3 and 48.5; 112 of
  // 4,096 72.2 and 98.0.
  template <bool GATE, int GROUP, bool S32, int WN>
  bool tiles(int64_t cus, int* rc) const {
    using F = TilesShape<GATE, WN>;
    constexpr int kLds = 2 * F::kStage;
    static_assert(kLds <= 160 * 1024, "a compute unit's LDS");
    const int64_t row_tiles = (int64_t(rows) + F::kRows - 1) / F::kRows;
    const int64_t tok_tiles = (int64_t(T) + F::kTokens - 1) / F::kTokens;
    if ((cols < 2048 ? 2.0 : 2.5) * double(row_tiles * tok_tiles) < double(cus)) return false;
    const auto kernel = q4_tiles_kernel<GATE, GROUP, S32, WN>;
    static std::atomic<uint64_t> done{0};
    if ((*rc = more_lds(kernel, kLds, done))) return true;
    if (row_tiles * tok_tiles * 512 > int64_t(UINT32_MAX)) {
      *rc = too_many();
      return true;
    }
    hipLaunchKernelGGL(kernel, dim3(unsigned(row_tiles * tok_tiles)), dim3(512), kLds, stream, out, parts,
                       w0, w1, scale_type, T, rows, cols, int(row_tiles), int(tok_tiles));
    return true;
  }
  template <bool GATE, int GROUP, bool S32, bool DIRECT>
  int by_slots(int64_t row_tiles, int64_t tok_tiles, int64_t cus) const {
    constexpr int kMost = GATE ? 2 : 4;  // row tiles of a workgroup: as many as leave every unit one
    if ((row_tiles + kMost - 1) / kMost * tok_tiles >= cus) return slots<GATE, kMost, 1, GROUP, S32, DIRECT>();
    if (!GATE && (row_tiles + 1) / 2 * tok_tiles >= cus) return slots<GATE, 2, 1, GROUP, S32, DIRECT>();
    return slots<GATE, 1, 1, GROUP, S32, DIRECT>();
  }
  template <bool GATE, int GROUP, bool S32>
  int run() const {
    const int64_t row_tiles = (int64_t(rows) + 15) / 16;
    const int64_t cus = device_compute_units();
    int rc = IE_HIP_OK;
    if (!needs_parts(T, cols)) {
      if (T == 1 ? few<GATE, GROUP, S32, 1>(row_tiles, cus, &rc)
          : T <= 4 ? few<GATE, GROUP, S32, 4>(row_tiles, cus, &rc)
          : T <= 8 ? few<GATE, GROUP, S32, 8>(row_tiles, cus, &rc)
                   : few<GATE, GROUP, S32, 16>(row_tiles, cus, &rc))
        return rc;
      return fail(IE_HIP_EINVAL, std::string(who) + ": activations past a workgroup's memory");
    }
    const int64_t tok_tiles = (int64_t(T) + 15) / 16, blocks = (int64_t(cols) + kBlock - 1) / kBlock;
    // One block a slot, and a tile or less for each unit or one group of row tiles: the waves split what
    // they multiply, a launch less (us, parts first and not: 40 tokens of 896 columns by 1,152 rows 5.8 and
    // 5.5, 2,048 by 64 11.0 and 5.9). With more blocks a wave has nothing under way while it splits (20 of
    // 4,864 by 128 10.4 and 14.3), with more tiles it splits the same tokens too often (64 of 896 by 1,152
    // 6.5 and 7.6).
    if (cols <= kSlots * kBlock && (row_tiles <= (GATE ? 2 : 4) || row_tiles * tok_tiles <= cus))
      return by_slots<GATE, GROUP, S32, true>(row_tiles, tok_tiles, cus);
    if (tok_tiles * blocks * 256 > int64_t(UINT32_MAX)) return too_many();
    hipLaunchKernelGGL(q4_split_kernel<GROUP == kBlock>, dim3(unsigned(tok_tiles * blocks)), dim3(256), 0,
                       stream, parts, x, T, cols, int(blocks));
    if (T <= 32 ? tiles<GATE, GROUP, S32, 1>(cus, &rc)
                : T <= 64 ? tiles<GATE, GROUP, S32, 2>(cus, &rc) : tiles<GATE, GROUP, S32, 4>(cus, &rc))
      return rc;
    return by_slots<GATE, GROUP, S32, false>(row_tiles, tok_tiles, cus);
  }
  template <bool GATE, int GROUP>
  int run() const {
    return scale_type == IE_KV_F32 ? run<GATE, GROUP, true>() : run<GATE, GROUP, false>();
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

Q4View view_of(const ie_matrix_q4& w) {
  return Q4View{static_cast<const uint8_t*>(w.data), static_cast<const uint8_t*>(w.scale),
                static_cast<const uint8_t*>(w.zero)};
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
                        view_of(w),
                        w2 ? view_of(*w2) : Q4View{nullptr, nullptr, nullptr},
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
  if (T <= 0 || cols <= 0 || !needs_parts(T, cols)) return 0;
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
