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
// w4_product_kernel.  Bound: the weights' bytes; the integer pipe that unpacks them comes next (7 operations for 8
// bf16 codes, 5 for fp16).  A warp takes 16-row tiles over a slice of the inputs, its block's warps the slices;
// a group's sum of x * code is exact products in an fp32 accumulator, scaled once, added in fp32.  Inputs go to the
// 8-column operand straight from global memory, 8 consecutive elements a load.
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

constexpr int kWarps = 8;

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

// kCols column tiles of 8 input rows, kRowTiles tiles of 16 weight rows to a warp, kFine: groups of 32.
template <class T, int kCols, int kRowTiles, bool kFine>
__global__ void __launch_bounds__(kWarps * 32) w4_product_kernel(W4View w, W4Product p, int split, bool aligned) {
  constexpr int kParts = kFine ? 2 : 1;   // scales of a 64-input tile
  constexpr int kAhead = kCols * kRowTiles >= 8 ? 1 : kCols * kRowTiles >= 4 ? 2 : 4;  // input tiles loaded together
  constexpr int kPitch = 8 * kCols + 1;
  __shared__ float sums[kWarps][kRowTiles * 16 * kPitch];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int tiles_n = static_cast<int>((w.n + 15) / 16), tiles_k = static_cast<int>((w.k + 63) / 64);
  const int groups = static_cast<int>((w.k + w.group - 1) / w.group), group_shift = w.group == 128 ? 1 : 0;
  const int slice = warp % split;  // of the inputs
  const int tile0 = (static_cast<int>(blockIdx.x) * (kWarps / split) + warp / split) * kRowTiles;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * (8 * kCols);
  const int k_begin = static_cast<int>(static_cast<int64_t>(tiles_k) * slice / split);
  const int k_end = tile0 < tiles_n ? static_cast<int>(static_cast<int64_t>(tiles_k) * (slice + 1) / split) : k_begin;

  const uint4* codes[kRowTiles];
  const uint32_t* scales[kRowTiles];  // bfloat16 of rows g and g + 8
#pragma unroll
  for (int r = 0; r < kRowTiles; ++r) {
    const int64_t tile = min(tile0 + r, tiles_n - 1);
    codes[r] = reinterpret_cast<const uint4*>(w.codes) + tile * tiles_k * 32 + lane;
    scales[r] = reinterpret_cast<const uint32_t*>(w.scales) + tile * groups * 8 + g;
  }
  const T* x[kCols];
  bool live[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    live[c] = row0 + c * 8 + g < p.rows;
    x[c] = static_cast<const T*>(p.x) + (live[c] ? row0 + c * 8 + g : 0) * p.x_stride + 8 * t;
  }

  float acc[kRowTiles][kCols][4];
#pragma unroll
  for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][c][i] = 0.0F;

  for (int k0 = k_begin; k0 < k_end; k0 += kAhead) {
    uint4 word[kAhead][kRowTiles], in[kAhead][kCols][2];
    uint32_t scale[kAhead][kRowTiles][kParts];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int kt = min(k0 + u, k_end - 1);
#pragma unroll
      for (int r = 0; r < kRowTiles; ++r) {
        word[u][r] = __ldcs(codes[r] + static_cast<int64_t>(kt) * 32);
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
          const int at = kFine ? 2 * kt + h : kt >> group_shift;
          scale[u][r][h] = __ldg(scales[r] + min(at, groups - 1) * 8);
        }
      }
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          in[u][c][h] = make_uint4(0, 0, 0, 0);
          const int64_t k = static_cast<int64_t>(kt) * 64 + 32 * h;
          if (live[c] && k + 8 * t < w.k) {
            if (aligned) {
              in[u][c][h] = __ldg(reinterpret_cast<const uint4*>(x[c] + k));
            } else {
              __align__(16) T e[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) e[i] = x[c][k + i];
              in[u][c][h] = *reinterpret_cast<const uint4*>(e);
            }
          }
        }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (k0 + u >= k_end) break;
#pragma unroll
      for (int r = 0; r < kRowTiles; ++r) {
        const uint32_t words[4] = {word[u][r].x, word[u][r].y, word[u][r].z, word[u][r].w};
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
            const uint4 v = in[u][c][i >> 1];
            mma(part[c], a, i & 1 ? v.z : v.x, i & 1 ? v.w : v.y, T());
          }
          if (i == 3 || (kFine && i == 1)) {
            const uint32_t sc = scale[u][r][kFine ? i >> 1 : 0];
            const float lo = __uint_as_float(sc << 16), hi = __uint_as_float(sc & 0xFFFF0000u);
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              acc[r][c][0] = fmaf(part[c][0], lo, acc[r][c][0]);
              acc[r][c][1] = fmaf(part[c][1], lo, acc[r][c][1]);
              acc[r][c][2] = fmaf(part[c][2], hi, acc[r][c][2]);
              acc[r][c][3] = fmaf(part[c][3], hi, acc[r][c][3]);
            }
          }
        }
      }
    }
  }

  // The slices' sums, in their order, then the bias and the one rounding.
#pragma unroll
  for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sums[warp][(r * 16 + g + 8 * (i >> 1)) * kPitch + c * 8 + 2 * t + (i & 1)] = acc[r][c][i];
  __syncthreads();
  constexpr int kOutputs = kRowTiles * 16 * 8 * kCols;
  for (int i = threadIdx.x; i < kOutputs * (kWarps / split); i += kWarps * 32) {
    const int unit = i / kOutputs, n = i % (kRowTiles * 16), m = (i % kOutputs) / (kRowTiles * 16);
    const int64_t out_n = (static_cast<int64_t>(blockIdx.x) * (kWarps / split) + unit) * kRowTiles * 16 + n;
    if (out_n >= w.n || row0 + m >= p.rows) continue;
    float y = 0.0F;
    for (int k = 0; k < split; ++k) y += sums[unit * split + k][n * kPitch + m];
    if (p.bias) y += to_f32(static_cast<const T*>(p.bias)[out_n]);
    static_cast<T*>(p.y)[(row0 + m) * p.y_stride + out_n] = from_f32<T>(y);
  }
}

template <class T, int kCols, int kRowTiles>
void launch_cols(const W4View& w, const W4Product& p, cudaStream_t stream) {
  const int64_t units = (w.n + 16 * kRowTiles - 1) / (16 * kRowTiles);
  const int64_t tiles_k = (w.k + 63) / 64;
  int split = kWarps;
  while (split > 1 && split > tiles_k) split >>= 1;
  const bool aligned = ((reinterpret_cast<uintptr_t>(p.x) | static_cast<uint64_t>(p.x_stride) * sizeof(T)) & 15) == 0;
  const int per_block = kWarps / split;
  const dim3 grid(static_cast<unsigned>((units + per_block - 1) / per_block),
                  static_cast<unsigned>((p.rows + 8 * kCols - 1) / (8 * kCols)));
  if (w.group == 32) w4_product_kernel<T, kCols, kRowTiles, true><<<grid, kWarps * 32, 0, stream>>>(w, p, split, aligned);
  else w4_product_kernel<T, kCols, kRowTiles, false><<<grid, kWarps * 32, 0, stream>>>(w, p, split, aligned);
}

template <class T>
void launch_typed(const W4View& w, const W4Product& p, cudaStream_t stream) {
  if (p.rows <= 8) launch_cols<T, 1, 1>(w, p, stream);
  else if (p.rows <= 16) launch_cols<T, 2, 2>(w, p, stream);
  else launch_cols<T, 4, 2>(w, p, stream);
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
  if (p.rows <= 0) return;
  if (p.type == kElemF16) launch_typed<__half>(w, p, stream);
  else launch_typed<__nv_bfloat16>(w, p, stream);
  count_launch();
  check(cudaGetLastError(), "launch 4-bit weight product kernel");
}

}  // namespace msb
