// Products of few rows with 4-bit weights: y[m, n] = sum_g ws[n, g] sum_{k in g} x[m, k] wc[n, k] + bias[n].
//
// Packed weights.  Weights are laid out once in the order in which a warp feeds the tensor cores
// (m16n8k16, the weights as the 16-row operand): a tile is 16 weight rows x 64 inputs, 512 bytes, lane
// (g = lane / 4, t = lane % 4) owning 16 consecutive bytes.  Its word w = 2 h + s holds inputs
// 32 h + 8 t + 4 s + {0, 1, 2, 3} of rows g and g + 8; nibbles i and i + 4 of a word are the two halves of
// operand register i: (row g + 8 (i % 2), inputs 2 (i / 2) + {0, 1}).  Codes are stored plus 8.  Tiles are
// [row tile][input tile]; scales are [row tile][group][rows 0, 8, 1, 9, .. 7, 15].  Rows and inputs past the matrix hold the
// code 0 (stored 8), rows past it the scale 0.
//
// w4_product_kernel.  Bound: the weights' bytes, then instruction issue: unpacking takes 7 operations for 8 bf16 codes,
// 5 for fp16 ones.  A block has 16 weight rows (or 32, below) and all inputs, which its warps take in turn, 64 at a
// time, each through a ring of its own in shared memory that asynchronous copies fill with codes, scales and inputs: no
// barrier before the last tile, and the weights on their way hold no registers.  A group's sum of x * code is exact
// products in an fp32 accumulator, scaled once, added in fp32; the warps' sums are added in their order.  tcgen05 would
// want 128 weight rows a tile and unpacked codes in shared memory: at 32 rows and fewer the products are not the bound.
// Measured on the device, bf16, groups of 128: 16,384 x 8,192 1 row 20.9 us (3.3 TB/s of weights), 16 rows 27.4 us, 32
// rows 42 us; 4,096 x 4,096 1 row 5.2 us, 32 rows 8.6 us; 4,096 x 14,336 1 row 11.8 us.  At 1 row the issue slots bound
// it where blocks are many, and at 16,384 weight rows 512 blocks on 296 places leave some SMs idle at the end.
#include <algorithm>

#include "quant4.cuh"

namespace msb {
namespace {

__global__ void w4_pack_kernel(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scales, int64_t n,
                               int64_t k, int group, uint32_t* __restrict__ out, uint16_t* __restrict__ out_scales) {
  const int64_t tiles_n = (n + 15) / 16, tiles_k = (k + 63) / 64, groups = (k + group - 1) / group;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = first; i < tiles_n * tiles_k * 128; i += stride) {
    const int w = static_cast<int>(i & 3), lane = static_cast<int>((i >> 2) & 31);
    const int64_t tile = i >> 7;
    const int64_t k0 = (tile % tiles_k) * 64 + 32 * (w >> 1) + 8 * (lane & 3) + 4 * (w & 1);
    uint32_t word = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const int64_t row = (tile / tiles_k) * 16 + (lane >> 2) + 8 * (p & 1);
      const int64_t col = k0 + 2 * ((p & 3) >> 1) + (p >> 2);
      uint32_t u = 8;
      if (row < n && col < k) u = ((codes[row * (k / 2) + col / 2] >> (4 * (col & 1))) & 15) ^ 8;
      word |= u << (4 * p);
    }
    out[i] = word;
  }
  for (int64_t i = first; i < tiles_n * groups * 16; i += stride) {
    const int64_t row = (i / (16 * groups)) * 16 + ((i >> 1) & 7) + 8 * (i & 1), g = (i >> 4) % groups;
    out_scales[i] = row < n ? scales[row * groups + g] : 0;
  }
}

constexpr int kMaxWarps = 8;

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The four operand registers of a word, exact codes: a nibble is put into the last bits of a number whose last
// place is 1 (fp16: 1024, or 64 for bits four up; bf16: 128), and that number and the stored 8 are subtracted.
__device__ __forceinline__ void unpack(uint32_t (&a)[4], uint32_t w, __half) {
  const uint32_t v = w >> 8;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(a[0]) : "r"(w), "r"(0x64006400u));  // (a & b) | c
  asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(a[1]) : "r"(w), "r"(0x54005400u));
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(a[2]) : "r"(v), "r"(0x64006400u));
  asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(a[3]) : "r"(v), "r"(0x54005400u));
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(a[i]) : "r"(i & 1 ? 0x54805480u : 0x64086408u));
}
__device__ __forceinline__ void unpack(uint32_t (&a)[4], uint32_t w, __nv_bfloat16) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(a[i]) : "r"(w >> (4 * i)), "r"(0x43004300u));
    asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(a[i]) : "r"(0x43084308u));  // 136
  }
}

// 16 bytes (4 bytes) to shared memory, zeros where not `valid`.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// One input tile of a warp: codes of its row tiles, its inputs (rows of 128 bytes, 16-byte pieces), scales.
template <int kCols, int kRowTiles, bool kFine>
struct Stage {
  static constexpr int kParts = kFine ? 2 : 1;   // scales of a 64-input tile
  static constexpr int off_x = kRowTiles * 512;
  static constexpr int off_scales = off_x + kCols * 1024;
  static constexpr int kBytes = off_scales + kRowTiles * kParts * 32;
  // Tiles on their way: enough bytes in flight with 16 warps to an SM (8 with 32 input rows).
  static constexpr int kStages = kCols == 1 ? 8 / kRowTiles : 4;
};

// kCols column tiles of 8 input rows, kRowTiles tiles of 16 weight rows to a block, kFine: groups of 32.  The block's
// warps take the input tiles in turn, so that together they read consecutive bytes.
template <class T, int kCols, int kRowTiles, bool kFine>
__global__ void __launch_bounds__(kMaxWarps * 32, kCols < 4 ? 2 : 1) w4_product_kernel(W4View w, W4Product p) {
  using S = Stage<kCols, kRowTiles, kFine>;
  constexpr int kRows = 16 * kRowTiles, kPitch = 8 * kCols + 1;
  extern __shared__ __align__(128) unsigned char ring[];
  float(*sums)[kRows * kPitch] = reinterpret_cast<float(*)[kRows * kPitch]>(ring);  // after the last tile
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, warps = blockDim.x >> 5;
  const int tiles_n = static_cast<int>((w.n + 15) / 16), tiles_k = static_cast<int>((w.k + 63) / 64);
  const int groups = static_cast<int>((w.k + w.group - 1) / w.group), group_shift = w.group == 128 ? 1 : 0;
  const int tile0 = static_cast<int>(blockIdx.x) * kRowTiles;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * (8 * kCols);

  const uint4* codes[kRowTiles];
  const uint32_t* scales[kRowTiles];  // bfloat16 of rows g and g + 8: copied by the lanes with t = 0
#pragma unroll
  for (int r = 0; r < kRowTiles; ++r) {
    const int64_t tile = min(tile0 + r, tiles_n - 1);
    codes[r] = reinterpret_cast<const uint4*>(w.codes) + (tile * tiles_k + warp) * 32 + lane;
    scales[r] = reinterpret_cast<const uint32_t*>(w.scales) + tile * groups * 8 + g;
  }
  // Copies of inputs: lane l takes piece l % 8 of rows l / 8 and on, by fours; `limit`: the inputs past its piece.
  const int piece = lane & 7;
  const T* x[2 * kCols];
  int limit[2 * kCols];
#pragma unroll
  for (int c = 0; c < 2 * kCols; ++c) {
    const int64_t row = row0 + 4 * c + (lane >> 3);
    x[c] = static_cast<const T*>(p.x) + (row < p.rows ? row : 0) * p.x_stride + 8 * piece;
    limit[c] = row < p.rows ? static_cast<int>(w.k) - 8 * piece : 0;
  }
  unsigned char* const stages = ring + warp * (S::kStages * S::kBytes);
  const uint32_t stage_at = static_cast<uint32_t>(__cvta_generic_to_shared(stages));
  // Pieces of odd rows lie four on (of eight): the eight lanes that read together then meet no bank twice.
  const uint32_t x_dst = static_cast<uint32_t>(S::off_x + (lane >> 3) * 128 + ((piece ^ ((lane >> 3) & 1) << 2) << 4));
  auto copy_tile = [&](int kt, int stage) {
    if (kt < tiles_k) {
      const uint32_t dst = stage_at + stage * S::kBytes;
#pragma unroll
      for (int r = 0; r < kRowTiles; ++r) {
        copy16(dst + r * 512 + lane * 16, codes[r], true);
        codes[r] += warps * 32;
        if (t == 0) {
#pragma unroll
          for (int h = 0; h < S::kParts; ++h)
            copy4(dst + S::off_scales + (r * S::kParts + h) * 32 + g * 4,
                  scales[r] + (kFine ? min(2 * kt + h, groups - 1) : kt >> group_shift) * 8);
        }
      }
#pragma unroll
      for (int c = 0; c < 2 * kCols; ++c) {
        const bool valid = kt * 64 < limit[c];
        copy16(dst + x_dst + c * 512, valid ? x[c] + kt * 64 : x[c], valid);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  float2 acc[kRowTiles][kCols][2];  // rows g and g + 8, two columns each
#pragma unroll
  for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[r][c][0] = acc[r][c][1] = make_float2(0.0F, 0.0F);

#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) copy_tile(warp + i * warps, i);
  int stage = 0;
  for (int kt = warp; kt < tiles_k; kt += warps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
    __syncwarp();
    // Every lane has left the stage of the tile before: the next copies go there.
    copy_tile(kt + (S::kStages - 1) * warps, stage == 0 ? S::kStages - 1 : stage - 1);
    const unsigned char* const here = stages + stage * S::kBytes;
    stage = stage == S::kStages - 1 ? 0 : stage + 1;
    uint4 in[kCols][2];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        in[c][h] = *reinterpret_cast<const uint4*>(here + S::off_x + (8 * c + g) * 128 + (((4 * h + t) ^ ((g & 1) << 2)) << 4));
#pragma unroll
    for (int r = 0; r < kRowTiles; ++r) {
      const uint4 word = *reinterpret_cast<const uint4*>(here + r * 512 + lane * 16);
      const uint32_t words[4] = {word.x, word.y, word.z, word.w};
      float part[kCols][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i == 0 || (kFine && i == 2)) {
#pragma unroll
          for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[c][j] = 0.0F;
        }
        uint32_t a[4];
        unpack(a, words[i], T());
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const uint4 v = in[c][i >> 1];
          mma(part[c], a, i & 1 ? v.z : v.x, i & 1 ? v.w : v.y, T());
        }
        if (i == 3 || (kFine && i == 1)) {
          const uint32_t sc = *reinterpret_cast<const uint32_t*>(here + S::off_scales + (r * S::kParts + (kFine ? i >> 1 : 0)) * 32 + g * 4);
          const float lo = __uint_as_float(sc << 16), hi = __uint_as_float(sc & 0xFFFF0000u);
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            acc[r][c][0] = __ffma2_rn(make_float2(part[c][0], part[c][1]), make_float2(lo, lo), acc[r][c][0]);
            acc[r][c][1] = __ffma2_rn(make_float2(part[c][2], part[c][3]), make_float2(hi, hi), acc[r][c][1]);
          }
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();

  // The warps' sums, in their order, then the bias and the one rounding.
#pragma unroll
  for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float* to = &sums[warp][(r * 16 + g + 8 * h) * kPitch + c * 8 + 2 * t];
        to[0] = acc[r][c][h].x;
        to[1] = acc[r][c][h].y;
      }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * 8 * kCols; i += blockDim.x) {
    const int n = i % kRows, m = i / kRows;
    const int64_t out_n = static_cast<int64_t>(blockIdx.x) * kRows + n;
    if (out_n >= w.n || row0 + m >= p.rows) continue;
    float y = 0.0F;
    for (int k = 0; k < warps; ++k) y += sums[k][n * kPitch + m];
    if (p.bias) y += to_f32(static_cast<const T*>(p.bias)[out_n]);
    static_cast<T*>(p.y)[(row0 + m) * p.y_stride + out_n] = from_f32<T>(y);
  }
}

template <class T, int kCols, int kRowTiles, bool kFine>
void launch_stages(const W4View& w, const W4Product& p, dim3 grid, int warps, cudaStream_t stream) {
  using S = Stage<kCols, kRowTiles, kFine>;
  constexpr int kPerWarp = S::kStages * S::kBytes;
  static_assert(kPerWarp >= 16 * kRowTiles * (8 * kCols + 1) * static_cast<int>(sizeof(float)), "sums fit the ring");
  allow_dynamic_shared<w4_product_kernel<T, kCols, kRowTiles, kFine>>(kMaxWarps * kPerWarp, "shared memory of the 4-bit weight product kernel");
  w4_product_kernel<T, kCols, kRowTiles, kFine><<<grid, warps * 32, warps * kPerWarp, stream>>>(w, p);
}

template <class T, int kCols, int kRowTiles>
void launch_cols(const W4View& w, const W4Product& p, cudaStream_t stream) {
  const int64_t units = (w.n + 16 * kRowTiles - 1) / (16 * kRowTiles), tiles_k = (w.k + 63) / 64;
  // Eight warps to a block are through its inputs soonest; where blocks outnumber the SMs and the inputs' columns are
  // several, more blocks of fewer warps wait less.  (us with 2, 4 and 8 warps, bf16: 4,096 x 4,096, 16 rows 11.4, 7.3 and 6.3;
  // 16,384 x 8,192, 8 rows 23.3, 21.9 and 21.3, 16 rows 28.1, 27.4 and 28.0, 32 rows 42.0, 43.3 and 47.2.)
  int warps = kCols == 1 || units <= 148 ? 8 : kCols == 4 && units > 2 * 148 ? 2 : 4;
  while (warps > 1 && warps > tiles_k) warps >>= 1;
  const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>((p.rows + 8 * kCols - 1) / (8 * kCols)));
  if (w.group == 32) launch_stages<T, kCols, kRowTiles, true>(w, p, grid, warps, stream);
  else launch_stages<T, kCols, kRowTiles, false>(w, p, grid, warps, stream);
}

template <class T>
void launch_typed(const W4View& w, const W4Product& p, cudaStream_t stream) {
  // Two row tiles to a block share its inputs' loads, where that leaves blocks for three quarters of the SMs.  (us with one and
  // two, 8 warps: 4,096 x 4,096, 1 row 5.6 and 5.2, 32 rows 11.5 and 8.6; 2,048 x 4,096 4.0 and 4.7, 6.3 and 8.4.)
  const bool wide = 4 * w.n >= 3 * 148 * 32;
  if (p.rows <= 8) {
    if (wide) launch_cols<T, 1, 2>(w, p, stream);
    else launch_cols<T, 1, 1>(w, p, stream);
  } else if (p.rows <= 16) {
    if (wide) launch_cols<T, 2, 2>(w, p, stream);
    else launch_cols<T, 2, 1>(w, p, stream);
  } else {
    if (wide) launch_cols<T, 4, 2>(w, p, stream);
    else launch_cols<T, 4, 1>(w, p, stream);
  }
}

}  // namespace

void launch_w4_pack(const uint8_t* codes, const uint16_t* scales, int64_t n, int64_t k, int group, uint8_t* out,
                    uint16_t* out_scales, cudaStream_t stream) {
  w4_pack_kernel<<<148 * 8, 256, 0, stream>>>(codes, scales, n, k, group, reinterpret_cast<uint32_t*>(out),
                                              out_scales);
  count_launch();
  check(cudaGetLastError(), "launch weight pack kernel");
}

void launch_w4_product(const W4View& w, const W4Product& p, cudaStream_t stream) {
  // Row blocks (of 32 rows where rows are many) are a grid's second dimension, which ends at 65,535.
  constexpr int64_t kMostRows = int64_t{65535} * 32;
  for (int64_t row = 0; row < p.rows; row += kMostRows) {
    W4Product part = p;
    part.x = static_cast<const uint16_t*>(p.x) + row * p.x_stride;
    part.y = static_cast<uint16_t*>(p.y) + row * p.y_stride;
    part.rows = std::min(kMostRows, p.rows - row);
    if (p.type == kElemF16) launch_typed<__half>(w, part, stream);
    else launch_typed<__nv_bfloat16>(w, part, stream);
    count_launch();
    check(cudaGetLastError(), "launch 4-bit weight product kernel");
  }
}

}  // namespace msb
