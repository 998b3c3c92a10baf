// The 4-bit key/value cache: quantising vectors as they are written, reading them back.
//
// One vector (a token's key or value of one head): s = fl(max|x| * fl(1/7)) (0 -> 1), codes
// clip(rint(fl(x / s)), -7, 7), in the nibble layout of the corpus format int4_per_token (prep.cu).  The
// scale is the product with fl(1/7), as torch divides a tensor by a number on the device, and so within two
// units in the last place of the corpus packer's quotient.  A vector with an element that is not finite
// stores scale NaN and codes 0: it reads back, and is attended to, as NaN, and nothing else changes.
#include <algorithm>

#include "quant4.cuh"

namespace msb {
namespace {

template <class T>
__global__ void kv4_append_kernel(Kv4View c, Kv4Append a) {
  const int64_t vec = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int which = blockIdx.y;
  if (vec >= a.tokens * c.heads) return;
  const int64_t token = vec / c.heads;
  const int head = static_cast<int>(vec % c.heads);
  const int64_t slot = a.slots[token];
  if (slot < 0 || slot >= (c.num_pages << c.page_shift)) return;
  const T* x = static_cast<const T*>(a.x[which]) + token * a.token_stride[which] + head * a.head_stride[which];
  float m = 0.0F;
  bool finite = true;
  for (int i = lane; i < c.dim; i += 32) {
    const float v = fabsf(to_f32(x[i]));
    finite = finite && isfinite(v);
    m = fmaxf(m, v);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
  finite = __all_sync(0xFFFFFFFFu, finite);
  float s = __fmul_rn(m, 1.0F / 7.0F);
  if (s == 0.0F) s = 1.0F;
  const int64_t at = c.vector(slot >> c.page_shift, head, static_cast<int>(slot & ((1 << c.page_shift) - 1)));
  if (lane == 0) c.scales[which][at] = finite ? s : __int_as_float(0x7FC00000);
  for (int p = lane; p < c.dim / 2; p += 32) {
    const int lo = finite ? static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(to_f32(x[2 * p]), s)), -7.0F), 7.0F)) : 0;
    const int hi = finite ? static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(to_f32(x[2 * p + 1]), s)), -7.0F), 7.0F)) : 0;
    c.codes[which][at * (c.dim / 2) + p] = static_cast<uint8_t>((lo & 15) | ((hi & 15) << 4));
  }
}

template <class T>
__global__ void kv4_read_kernel(Kv4View c, Kv4Read a) {
  const int64_t vec = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int which = blockIdx.y;
  if (vec >= a.tokens * c.heads) return;
  const int64_t token = vec / c.heads;
  const int head = static_cast<int>(vec % c.heads);
  const int64_t slot = a.slots[token];
  const bool held = slot >= 0 && slot < (c.num_pages << c.page_shift);
  const int64_t at =
      held ? c.vector(slot >> c.page_shift, head, static_cast<int>(slot & ((1 << c.page_shift) - 1))) : 0;
  const float s = held ? c.scales[which][at] : 0.0F;
  T* out = static_cast<T*>(a.out[which]) + vec * c.dim;
  for (int p = lane; p < c.dim / 2; p += 32) {
    const int byte = held ? c.codes[which][at * (c.dim / 2) + p] : 0;
    out[2 * p] = from_f32<T>(static_cast<float>(((byte & 15) ^ 8) - 8) * s);
    out[2 * p + 1] = from_f32<T>(static_cast<float>(((byte >> 4) ^ 8) - 8) * s);
  }
}

}  // namespace

void launch_kv4_append(const Kv4View& c, const Kv4Append& a, cudaStream_t stream) {
  if (a.tokens <= 0) return;
  const int64_t threads = a.tokens * c.heads * 32;
  const dim3 grid(static_cast<unsigned>((threads + 255) / 256), 2);
  if (a.type == kElemF32) kv4_append_kernel<float><<<grid, 256, 0, stream>>>(c, a);
  else if (a.type == kElemF16) kv4_append_kernel<__half><<<grid, 256, 0, stream>>>(c, a);
  else kv4_append_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(c, a);
  count_launch();
  check(cudaGetLastError(), "launch cache append kernel");
}

void launch_kv4_read(const Kv4View& c, const Kv4Read& a, cudaStream_t stream) {
  if (a.tokens <= 0) return;
  const int64_t threads = a.tokens * c.heads * 32;
  const dim3 grid(static_cast<unsigned>((threads + 255) / 256), 2);
  if (a.type == kElemF32) kv4_read_kernel<float><<<grid, 256, 0, stream>>>(c, a);
  else if (a.type == kElemF16) kv4_read_kernel<__half><<<grid, 256, 0, stream>>>(c, a);
  else kv4_read_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(c, a);
  count_launch();
  check(cudaGetLastError(), "launch cache read kernel");
}

}  // namespace msb
