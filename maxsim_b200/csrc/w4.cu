// Products of few rows with 4-bit weights: y[m, n] = sum_g ws[n, g] sum_{k in g} x[m, k] wc[n, k] + bias[n].
//
// Packed weights.  Weights are laid out once in the order in which a warp feeds the tensor cores
// (m16n8k16, the weights as the 16-row operand): a tile is 16 weight rows x 64 inputs, 512 bytes, lane
// (g = lane / 4, t = lane % 4) owning 16 consecutive bytes.  Its word w = 2 h + s holds inputs
// 32 h + 8 t + 4 s + {0, 1, 2, 3} of rows g and g + 8; nibbles i and i + 4 of a word are the two halves of
// operand register i: (row g + 8 (i % 2), inputs 2 (i / 2) + {0, 1}).  Codes are stored plus 8.  Tiles are
// [row tile][input tile]; scales are [row tile][group][16 rows].  Rows and inputs past the matrix hold the
// code 0 (stored 8), rows past it the scale 0.
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
    const int64_t row = (i / (16 * groups)) * 16 + (i & 15), g = (i >> 4) % groups;
    out_scales[i] = row < n ? scales[row * groups + g] : 0;
  }
}

// One warp per weight row and input row.
template <class T>
__global__ void w4_product_kernel(W4View w, W4Product p) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= w.n) return;
  const int64_t tiles_k = (w.k + 63) / 64, groups = (w.k + w.group - 1) / w.group;
  const T* x = static_cast<const T*>(p.x) + blockIdx.y * p.x_stride;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(w.codes);
  float sum = 0.0F;
  for (int64_t k = lane; k < w.k; k += 32) {
    const int in = static_cast<int>(k & 63), h = in >> 5, t = (in & 31) >> 3, s = (in & 7) >> 2, c = in & 3;
    const int g = static_cast<int>(row & 7), nib = ((c >> 1) << 1) + ((row & 8) ? 1 : 0) + 4 * (c & 1);
    const uint32_t word = words[(((row >> 4) * tiles_k + (k >> 6)) * 32 + g * 4 + t) * 4 + 2 * h + s];
    const float code = static_cast<float>(static_cast<int>((word >> (4 * nib)) & 15) - 8);
    const uint32_t bits = w.scales[((row >> 4) * groups + k / w.group) * 16 + (row & 15)];
    sum += code * __uint_as_float(bits << 16) * to_f32(x[k]);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
  if (lane == 0) {
    if (p.bias) sum += to_f32(static_cast<const T*>(p.bias)[row]);
    static_cast<T*>(p.y)[blockIdx.y * p.y_stride + row] = from_f32<T>(sum);
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
  if (p.rows <= 0) return;
  const dim3 grid(static_cast<unsigned>((w.n + 3) / 4), static_cast<unsigned>(p.rows));
  if (p.type == kElemF16) w4_product_kernel<__half><<<grid, 128, 0, stream>>>(w, p);
  else w4_product_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(w, p);
  count_launch();
  check(cudaGetLastError(), "launch 4-bit weight product kernel");
}

}  // namespace msb
