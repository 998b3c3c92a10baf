// What the kernels of the 4-bit key/value cache and of the 4-bit weights share: element types, the cache's
// addressing and the host-side argument blocks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "common.cuh"

namespace msb {

enum ElementType : int { kElemF32 = 0, kElemF16 = 1, kElemBF16 = 2 };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Pages of `page_size` (a power of two) tokens: codes [pages, heads, page_size, dim / 2], scales
// [pages, heads, page_size].  Slot s is token s % page_size of page s / page_size.
struct Kv4View {
  uint8_t* codes[2];   // keys, values
  float* scales[2];
  int64_t num_pages;
  int page_shift;      // log2(page_size)
  int heads;
  int dim;
  // Index of a token's vector of one head, in vectors (64 bits: caches pass 2^31 vectors and 4 GB).
  __host__ __device__ __forceinline__ int64_t vector(int64_t page, int head, int at) const {
    return (((page * heads) + head) << page_shift) + at;
  }
};

struct Kv4Append {
  const void* x[2];           // keys, values [tokens, heads, dim]
  int64_t token_stride[2];    // in elements
  int64_t head_stride[2];
  const int64_t* slots;       // [tokens]; outside the cache: not written
  int64_t tokens;
  int type;
};

struct Kv4Read {
  void* out[2];               // [tokens, heads, dim], contiguous
  const int64_t* slots;       // outside the cache: zeros
  int64_t tokens;
  int type;
};

struct Kv4Attend {
  const void* query;          // [rows, heads, dim]
  int64_t q_row_stride, q_head_stride;
  int64_t rows;               // query rows of all sequences
  int heads;                  // query heads, a multiple of the cache's
  const int32_t* page_table;  // [batch, max_pages]
  int64_t table_stride;
  int max_pages;
  const int32_t* lengths;     // [batch] cached tokens
  const int32_t* offsets;     // [batch + 1] rows of each sequence, or nullptr: one row each
  int batch;
  int max_rows;               // the most rows of one sequence
  float scale;
  int causal;
  int window;                 // 0: none
  // What keeps sums of weights finite (set by the launch, see keep_sums_finite): the least log2 of a value scale that
  // references count, and the weight that none may pass.
  float least_exponent;
  float most_weight;
  void* out;                  // [rows, heads, dim], contiguous
  float* lse;                 // [rows, heads] or nullptr
  void* workspace;
  size_t workspace_bytes;
  int type;
  int engine;                 // 0 by size, 1 the kernel for few rows, 2 that for many
  int fill;                   // rows that are not worked on are written too (kv4_fill_rows)
};

// One sequence of an attention call, with what the device arrays say held to what the call can read:
// lengths to the table's pages, rows to the query's rows.  Of these the announced maximum is worked on; positions count
// from all of them.
struct Kv4Sequence {
  int64_t row0;
  int rows;
  int length;
  int pos0;   // position of row 0, negative where rows outnumber tokens
  int left;   // rows past the announced maximum
};
__device__ __forceinline__ Kv4Sequence kv4_sequence(const Kv4Attend& a, int page_shift, int b) {
  Kv4Sequence s;
  const int64_t most = static_cast<int64_t>(a.max_pages) << page_shift;
  s.length = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(a.lengths[b]), most)));
  if (a.offsets == nullptr) {
    s.row0 = b;
    s.rows = 1;
    s.pos0 = s.length - 1;
    s.left = 0;
  } else {
    const int64_t lo = max(0, a.offsets[b]);
    const int64_t hi = min(static_cast<int64_t>(a.offsets[b + 1]), a.rows);
    s.row0 = lo;
    const int all = static_cast<int>(max(static_cast<int64_t>(0), hi - lo));  // at most a.rows
    s.rows = min(all, a.max_rows);
    s.pos0 = s.length - all;
    s.left = all - s.rows;
  }
  return s;
}

// A block's `share` of `shares` of rows lo .. hi of an output (`width` elements a row) and of their log-sum-exp (`heads` a row)
// to one value each.  (Out of line, as seldom run: the kernels' own code then lies together.)
template <class T>
__device__ __noinline__ void set_rows(T* out, float* lse, int64_t width, int heads, int64_t lo, int64_t hi, float value,
                                      float lse_value, int share, int shares, int thread, int threads) {
  const int64_t first = lo + (hi - lo) * share / shares, last = lo + (hi - lo) * (share + 1) / shares;
#pragma unroll 1
  for (int64_t i = first * width + thread; i < last * width; i += threads) out[i] = from_f32<T>(value);
  if (lse == nullptr) return;
#pragma unroll 1
  for (int64_t i = first * heads + thread; i < last * heads; i += threads) lse[i] = lse_value;
}
// Where the caller's output is fresh memory, the rows that no block works on are written by the blocks that have sequence
// b (this one is `share` of `shares`): zeros and a log-sum-exp of -inf in the rows before the first sequence's and after
// the last's, NaN past a sequence's announced number of rows (that number was wrong, and it shows).
template <class T>
__device__ __forceinline__ void kv4_fill_rows(const Kv4Attend& a, int dim, int b, const Kv4Sequence& q, int share, int shares,
                                              int thread, int threads) {
  const int64_t end = q.row0 + q.rows + q.left;
  const bool before = b == 0 && q.row0 > 0, after = b == a.batch - 1 && end < a.rows;
  if (!before && !after && q.left == 0) return;
#pragma unroll 1
  for (int part = 0; part < 3; ++part) {  // one call in the code
    const int64_t lo = part == 0 ? 0 : part == 1 ? end - q.left : end;
    const int64_t hi = part == 0 ? (b == 0 ? min(q.row0, a.rows) : 0) : part == 1 ? end : b == a.batch - 1 ? a.rows : end;
    set_rows(static_cast<T*>(a.out), a.lse, static_cast<int64_t>(a.heads) * dim, a.heads, lo, max(lo, hi), part == 1 ? NAN : 0.0F,
             part == 1 ? NAN : -INFINITY, share, shares, thread, threads);
  }
}

// A weight p = 2^(s - reference) is as large as 1 / vs where the value scale vs is small, since references are maxima of
// s + log2(vs), less `lift`.  With log2(vs) held to -h and up, p stays at or below 2^(lift + h); h leaves as many of
// these as the table has tokens below 2^127.  Upwards the logarithm is held to lift + 109.5 (most_exponent): p vs of the
// largest scales, 2^125.2, stays at 2^15.7, which fp16 holds; p of these is 2^-109.5, and weights 2^-16 of it are the last
// that fp32 holds.  Scales below 2^-h lose digits in p vs, where that sinks below fp16's normal numbers.
constexpr float kExponents = 110.0F;  // h at most
constexpr float most_exponent(float lift) { return lift + 109.5F; }
inline void keep_sums_finite(Kv4Attend& a, int page_shift, float lift) {
  int bits = 0;
  while ((int64_t{1} << bits) < (static_cast<int64_t>(a.max_pages) << page_shift)) ++bits;
  a.least_exponent = -std::min(kExponents, 127.0F - static_cast<float>(bits) - lift);
  a.most_weight = std::ldexp(1.0F, 127 - bits);
}
// About log2 of a value scale, held to [least, most] (and so a number where the scale is 0, NaN or infinite).
__device__ __forceinline__ float scale_exponent(float s, float least, float most) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return fminf(fmaxf(r, least), most);
}
// Whether a vector's codes are all 0.  Such a vector is stored with scale 1 (append), which says nothing of its
// neighbours' size: it counts in the sum of weights, with a value scale of 0, but not in references.
template <int kDim>
__device__ __forceinline__ bool zero_codes(const uint8_t* codes) {
  uint32_t any = 0;
#pragma unroll 1  // seldom run, among kernels whose registers are all in use
  for (int i = 0; i < kDim / 8; ++i) any |= reinterpret_cast<const uint32_t*>(codes)[i];
  return any == 0;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// What sums with reference `from` are multiplied by to have reference `to` >= from.  Sums with reference -inf
// are 0, or NaN where a score was: they stay so.
__device__ __forceinline__ float fade_to(float from, float to) { return from == to ? 1.0F : exp2_fast(from - to); }
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Opts a kernel in to its dynamic shared memory, once per device.
template <auto kernel>
void allow_dynamic_shared(int bytes, const char* what) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  check(cudaGetDevice(&dev), "get device");
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return;
  check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), what);
  done.fetch_or(bit, std::memory_order_relaxed);
}

struct W4View {
  const uint8_t* codes;       // packed, see w4.cu
  const uint16_t* scales;     // bfloat16 bits [row tiles, groups, 16]
  int64_t n;
  int64_t k;
  int group;
};

struct W4Product {
  const void* x;              // [rows, k]
  int64_t x_stride;
  int64_t rows;
  const void* bias;           // [n] or nullptr
  void* y;                    // [rows, n]
  int64_t y_stride;
  int type;
};

}  // namespace msb
