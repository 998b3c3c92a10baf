// The 4-bit key/value cache: quantising vectors as they are written, reading them back.
//
// One vector (a token's key or value of one head): s = fl(max|x| * fl(1/7)) (0 -> 1), codes
// clip(rint(fl(x / s)), -7, 7), in the nibble layout of the corpus format int4_per_token (prep.cu).  The
// scale is the product with fl(1/7), as torch divides a tensor by a number on the device, and so within two
// units in the last place of the corpus packer's quotient.  A vector with an element that is not finite
// stores scale NaN and codes 0: it reads back, and is attended to, as NaN, and nothing else changes.
//
// Both kernels are bound by memory.  A thread has 8 dimensions (one word of codes, 16 bytes of 16-bit
// elements) of a token's key and value, D / 8 neighbouring threads a vector: loads and stores are whole
// 32-byte sectors in one pass, and a thread's two vectors are two independent loads.
#include <algorithm>

#include "quant4.cuh"

namespace msb {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Eight consecutive elements as fp32.
template <class T>
__device__ __forceinline__ void load8(float (&x)[8], const T* p, bool aligned) {
  if (aligned) {
    constexpr int kLoads = 8 * sizeof(T) / 16;
    uint4 v[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    const T* e = reinterpret_cast<const T*>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
  }
}

// rint(fl(x / s)) of eight elements with |x / s| <= 7.1, as a word of codes.
// For s of ordinary size the quotients share one reciprocal: with r = RN(1 / s), two steps of
// q += r (x - q s), each remainder exact in an FMA, give RN(x / s) (P. Markstein, "Computation of elementary
// functions on the IBM RISC System/6000 processor", 1990); elsewhere the division itself.  Adding 1.5 * 2^23 + 8
// rounds to the nearest integer, ties to even, and leaves code + 8 in the last bits; the words' sum by
// powers of 16 has the nibbles in place, the flip of each fourth bit makes them two's complement.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float s) {
  constexpr float kRound = 12582912.0F + 8.0F;
  uint32_t word = 0;
  if (s > 0x1p-100F && s < 0x1p100F) {
    const float r = __frcp_rn(s);
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      float q = __fmul_rn(x[i], r);
      q = __fmaf_rn(__fmaf_rn(-q, s, x[i]), r, q);
      q = __fmaf_rn(__fmaf_rn(-q, s, x[i]), r, q);
      word = word * 16u + __float_as_uint(__fadd_rn(q, kRound));
    }
  } else {
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      const float q = fminf(fmaxf(__fdiv_rn(x[i], s), -7.0F), 7.0F);
      word = word * 16u + __float_as_uint(__fadd_rn(q, kRound));
    }
  }
  // The bits of 1.5 * 2^23, 0x4B400000, came along with every power of 16.
  word -= 0x4B400000u * 0x11111111u;
  return word ^ 0x88888888u;
}

template <class T, int kDim>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(Kv4View c, Kv4Append a, bool aligned) {
  constexpr int kLanes = kDim / 8;  // threads of a vector
  const uint32_t vec = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool inside = vec < static_cast<uint32_t>(a.tokens) * c.heads;  // below 2^31
  const uint32_t token = inside ? vec / c.heads : 0, head = inside ? vec - token * c.heads : 0;
  const int64_t slot = inside ? __ldg(a.slots + token) : -1;
  const bool held = slot >= 0 && slot < (c.num_pages << c.page_shift);
  float x[2][8], m[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[w][i] = 0.0F;
    if (held)
      load8(x[w], static_cast<const T*>(a.x[w]) + token * a.token_stride[w] + head * a.head_stride[w] + lane * 8, aligned);
  }
  // The maximum keeps a NaN, and is infinite where an element is: both mark a vector that is not finite.
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    m[w] = 0.0F;
#pragma unroll
    for (int i = 0; i < 8; ++i) m[w] = max_nan(m[w], fabsf(x[w][i]));
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1) m[w] = max_nan(m[w], __shfl_xor_sync(0xFFFFFFFFu, m[w], d));
  }
  if (!held) return;
  const int64_t at = c.vector(slot >> c.page_shift, head, static_cast<int>(slot & ((1 << c.page_shift) - 1)));
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const bool finite = m[w] < INFINITY;
    float s = __fmul_rn(m[w], 1.0F / 7.0F);
    if (s == 0.0F) s = 1.0F;
    const uint32_t word = finite ? codes_of(x[w], s) : 0u;
    *reinterpret_cast<uint32_t*>(c.codes[w] + at * (kDim / 2) + lane * 4) = word;
    if (lane == 0) c.scales[w][at] = finite ? s : __int_as_float(0x7FC00000);
  }
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  __align__(16) T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(e) / 16); ++i)
    __stcs(reinterpret_cast<uint4*>(p) + i, reinterpret_cast<const uint4*>(e)[i]);
}

template <class T, int kDim>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(Kv4View c, Kv4Read a) {
  constexpr int kLanes = kDim / 8;
  const uint32_t vec = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  if (vec >= static_cast<uint32_t>(a.tokens) * c.heads) return;
  const uint32_t token = vec / c.heads, head = vec - token * c.heads;
  const int64_t slot = __ldg(a.slots + token);
  const bool held = slot >= 0 && slot < (c.num_pages << c.page_shift);
  uint32_t word[2] = {0, 0};
  float s[2] = {0.0F, 0.0F};
  if (held) {
    const int64_t at = c.vector(slot >> c.page_shift, head, static_cast<int>(slot & ((1 << c.page_shift) - 1)));
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      word[w] = __ldg(reinterpret_cast<const uint32_t*>(c.codes[w] + at * (kDim / 2) + lane * 4));
      s[w] = __ldg(c.scales[w] + at);
    }
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // 2^23 + (code + 8) as float bits, less 2^23 + 8
      const float u = __uint_as_float((((word[w] >> (4 * i)) & 15u) ^ 8u) | 0x4B000000u);
      x[i] = __fmul_rn(__fsub_rn(u, 8388616.0F), s[w]);
    }
    store8(static_cast<T*>(a.out[w]) + static_cast<int64_t>(vec) * kDim + lane * 8, x);
  }
}

template <class T>
void append_typed(const Kv4View& c, const Kv4Append& a, cudaStream_t stream) {
  // Rows start on 16 bytes where base and strides do (a vector's threads load 16 bytes each then).
  uint64_t starts = 0;
  for (int w = 0; w < 2; ++w)
    starts |= reinterpret_cast<uintptr_t>(a.x[w]) | static_cast<uint64_t>(a.token_stride[w]) * sizeof(T) |
              static_cast<uint64_t>(a.head_stride[w]) * sizeof(T);
  const bool aligned = (starts & 15) == 0;
  const int64_t vectors = a.tokens * c.heads, per_block = kThreads / (c.dim / 8);
  const unsigned blocks = static_cast<unsigned>((vectors + per_block - 1) / per_block);
  if (c.dim == 64) kv4_append_kernel<T, 64><<<blocks, kThreads, 0, stream>>>(c, a, aligned);
  else if (c.dim == 128) kv4_append_kernel<T, 128><<<blocks, kThreads, 0, stream>>>(c, a, aligned);
  else kv4_append_kernel<T, 256><<<blocks, kThreads, 0, stream>>>(c, a, aligned);
}

template <class T>
void read_typed(const Kv4View& c, const Kv4Read& a, cudaStream_t stream) {
  const int64_t vectors = a.tokens * c.heads, per_block = kThreads / (c.dim / 8);
  const unsigned blocks = static_cast<unsigned>((vectors + per_block - 1) / per_block);
  if (c.dim == 64) kv4_read_kernel<T, 64><<<blocks, kThreads, 0, stream>>>(c, a);
  else if (c.dim == 128) kv4_read_kernel<T, 128><<<blocks, kThreads, 0, stream>>>(c, a);
  else kv4_read_kernel<T, 256><<<blocks, kThreads, 0, stream>>>(c, a);
}

}  // namespace

void launch_kv4_append(const Kv4View& c, const Kv4Append& a, cudaStream_t stream) {
  if (a.tokens <= 0) return;
  if (a.type == kElemF32) append_typed<float>(c, a, stream);
  else if (a.type == kElemF16) append_typed<__half>(c, a, stream);
  else append_typed<__nv_bfloat16>(c, a, stream);
  count_launch();
  check(cudaGetLastError(), "launch cache append kernel");
}

void launch_kv4_read(const Kv4View& c, const Kv4Read& a, cudaStream_t stream) {
  if (a.tokens <= 0) return;
  if (a.type == kElemF32) read_typed<float>(c, a, stream);
  else if (a.type == kElemF16) read_typed<__half>(c, a, stream);
  else read_typed<__nv_bfloat16>(c, a, stream);
  count_launch();
  check(cudaGetLastError(), "launch cache read kernel");
}

}  // namespace msb
