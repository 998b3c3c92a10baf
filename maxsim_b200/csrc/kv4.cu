// The 4-bit key/value cache: quantising vectors as they are written, reading them back.
//
// One vector (a token's key or value of one head): s = fl(max|x| * fl(1/7)) (0 -> 1), codes
// clip(rint(fl(x / s)), -7, 7), in the nibble layout of the corpus format int4_per_token (prep.cu).  The
// scale is the product with fl(1/7), as torch divides a tensor by a number on the device, and so within two
// units in the last place of the corpus packer's quotient.  A vector with an element that is not finite
// stores scale NaN and codes 0: it reads back, and is attended to, as NaN, and nothing else changes.
//
// Both kernels are bound by memory.  Writing, a thread has 8 dimensions (one word of codes, 16 bytes of 16-bit
// elements) of a token's key and value, D / 8 neighbouring threads a vector; reading, 16 bytes of output.  A thread
// asks for several vectors before it works on the first: whole sectors, and enough of them on their way.
// Measured on the device, keys and values, 8 heads, D = 128: writing 32,768 tokens from bf16 38.3 us (4.4 TB/s; issue,
// the conversions and quotients), from fp32 46.2 us (6.6 TB/s); reading them to bf16 28.3 us (6.0 TB/s), to fp32
// 47.5 us (6.4 TB/s); either of 64 tokens 2.5 to 2.8 us.
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

// Eight consecutive elements as they lie.
template <class T>
struct Eight {
  uint4 raw[8 * sizeof(T) / 16];
  __device__ __forceinline__ float get(int i) const { return to_f32(reinterpret_cast<const T*>(raw)[i]); }
};
template <bool kAligned, class T>
__device__ __forceinline__ void load8(Eight<T>& x, const T* p) {
  if constexpr (kAligned) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(8 * sizeof(T) / 16); ++i) x.raw[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(x.raw)[i] = p[i];
  }
}

// rint(fl(x / s)) of eight elements with |x / s| <= 7.1, as a word of codes.
// For s of ordinary size the quotients share one reciprocal: with r = RN(1 / s) and q = RN(x r), one step
// q + r (x - q s), the remainder exact in an FMA, gives RN(x / s) (P. Markstein, "Computation of elementary
// functions on the IBM RISC System/6000 processor", 1990; checked for every significand of s at the seven x
// around each half-integer quotient); elsewhere the division itself.  Adding 1.5 * 2^23 + 8
// rounds to the nearest integer, ties to even, and leaves code + 8 in the last bits; the words' sum by
// powers of 16 has the nibbles in place, the flip of each fourth bit makes them two's complement.
template <bool kShared, class T>
__device__ __forceinline__ uint32_t codes_of(const Eight<T>& x, float s) {
  constexpr float kRound = 12582912.0F + 8.0F;
  const float r = kShared ? __frcp_rn(s) : 0.0F;
  uint32_t word = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    const float v = x.get(i);
    float q;
    if (kShared) {
      q = __fmul_rn(v, r);
      q = __fmaf_rn(__fmaf_rn(-q, s, v), r, q);
    } else {
      q = fminf(fmaxf(__fdiv_rn(v, s), -7.0F), 7.0F);
    }
    word = word * 16u + __float_as_uint(__fadd_rn(q, kRound));
  }
  // The bits of 1.5 * 2^23, 0x4B400000, came along with every power of 16.
  word -= 0x4B400000u * 0x11111111u;
  return word ^ 0x88888888u;
}

// A block has one head: its vectors are neighbours in the cache, and a vector's place needs no division.
constexpr int kWrites = 2;  // tokens of a thread, loaded together
template <class T, int kDim, bool kAligned>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(Kv4View c, Kv4Append a) {
  constexpr int kLanes = kDim / 8, kStep = kThreads / kLanes;  // threads of a vector, vectors at a time
  const int head = blockIdx.y, lane = threadIdx.x % kLanes;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kStep * kWrites) + threadIdx.x / kLanes;
  Eight<T> x[kWrites][2];
  int64_t slot[kWrites];
#pragma unroll
  for (int k = 0; k < kWrites; ++k) {
    const int64_t token = first + k * kStep, here = min(token, a.tokens - 1);
    slot[k] = token < a.tokens ? __ldg(a.slots + token) : -1;
#pragma unroll
    for (int w = 0; w < 2; ++w)
      load8<kAligned>(x[k][w], static_cast<const T*>(a.x[w]) + here * a.token_stride[w] + head * a.head_stride[w] + lane * 8);
  }
#pragma unroll
  for (int k = 0; k < kWrites; ++k) {
    // The maximum keeps a NaN, and is infinite where an element is: both mark a vector that is not finite.
    float m[2], s[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      m[w] = fabsf(x[k][w].get(0));
#pragma unroll
      for (int i = 1; i < 8; ++i) m[w] = max_nan(m[w], fabsf(x[k][w].get(i)));
#pragma unroll
      for (int d = 1; d < kLanes; d <<= 1) m[w] = max_nan(m[w], __shfl_xor_sync(0xFFFFFFFFu, m[w], d));
      s[w] = __fmul_rn(m[w], 1.0F / 7.0F);
    }
    if (slot[k] < 0 || slot[k] >= (c.num_pages << c.page_shift)) continue;
    const int64_t at = c.vector(slot[k] >> c.page_shift, head, static_cast<int>(slot[k] & ((1 << c.page_shift) - 1)));
    uint32_t word[2];
    // (False for a NaN.)
    if (fminf(s[0], s[1]) > 0x1p-100F && max_nan(s[0], s[1]) < 0x1p100F) {
      word[0] = codes_of<true>(x[k][0], s[0]);
      word[1] = codes_of<true>(x[k][1], s[1]);
    } else {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        if (s[w] == 0.0F) s[w] = 1.0F;
        const bool finite = m[w] < INFINITY;
        word[w] = finite ? codes_of<false>(x[k][w], s[w]) : 0u;
        if (!finite) s[w] = __int_as_float(0x7FC00000);
      }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      *reinterpret_cast<uint32_t*>(c.codes[w] + at * (kDim / 2) + lane * 4) = word[w];
      if (lane == 0) c.scales[w][at] = s[w];
    }
  }
}

// Vectors of a thread: their slots, then their codes, are asked for together.
constexpr int kReads = 4;

// A thread writes 16 bytes: 8 dimensions of a 16-bit type, 4 of fp32.
template <class T, int kDim>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(Kv4View c, Kv4Read a) {
  constexpr int kPer = 16 / sizeof(T), kLanes = kDim / kPer, kStep = kThreads / kLanes;
  const uint32_t first = blockIdx.x * (kStep * kReads) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const uint32_t vectors = static_cast<uint32_t>(a.tokens) * c.heads;  // below 2^31
  const int64_t slots = c.num_pages << c.page_shift;
  int64_t slot[kReads];
  uint32_t head[kReads];
#pragma unroll
  for (int k = 0; k < kReads; ++k) {
    const uint32_t vec = first + k * kStep, token = vec / c.heads;
    head[k] = vec - token * c.heads;
    slot[k] = vec < vectors ? __ldg(a.slots + token) : -1;
  }
  uint32_t word[kReads][2];
  float s[kReads][2];
#pragma unroll
  for (int k = 0; k < kReads; ++k) {
    const bool held = slot[k] >= 0 && slot[k] < slots;
    const int64_t at = held ? c.vector(slot[k] >> c.page_shift, head[k], static_cast<int>(slot[k] & ((1 << c.page_shift) - 1))) : 0;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const uint8_t* codes = c.codes[w] + at * (kDim / 2) + lane * (kPer / 2);
      word[k][w] = 0;
      s[k][w] = 0.0F;
      if (held) {
        word[k][w] = kPer == 8 ? __ldg(reinterpret_cast<const uint32_t*>(codes)) : __ldg(reinterpret_cast<const uint16_t*>(codes));
        s[k][w] = __ldg(c.scales[w] + at);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kReads; ++k) {
    const uint32_t vec = first + k * kStep;
    if (vec >= vectors) return;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      __align__(16) T e[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        // 2^23 + (code + 8) as float bits, less 2^23 + 8
        const float u = __uint_as_float((((word[k][w] >> (4 * i)) & 15u) ^ 8u) | 0x4B000000u);
        e[i] = from_f32<T>(__fmul_rn(__fsub_rn(u, 8388616.0F), s[k][w]));
      }
      __stcs(reinterpret_cast<uint4*>(static_cast<T*>(a.out[w]) + static_cast<int64_t>(vec) * kDim + lane * kPer),
             *reinterpret_cast<const uint4*>(e));
    }
  }
}

// Moving cached vectors: every source is read before a target is written, so that a token may be the one's target and
// the other's source (the accepted path of a tree of drafted tokens takes the places after the context's last one).
// Heads, and the parts of a vector, do not meet: where one block has all tokens of one part (32 bytes of codes, or the
// scales) of one head, a barrier between its reads and its writes is enough.  Bound: latency, a slot, then a vector; 256
// tokens of 8 heads with their read back 6.2 us.
constexpr int kMoveThreads = 512;
constexpr int kMoves = 2;                             // tokens of a thread
constexpr int kMostMoved = kMoveThreads * kMoves;     // of one launch
__device__ __forceinline__ int64_t moved_vector(const Kv4View& c, int64_t slot, int head) {
  return c.vector(slot >> c.page_shift, head, static_cast<int>(slot & ((1 << c.page_shift) - 1)));
}
__global__ void __launch_bounds__(kMoveThreads) kv4_move_kernel(Kv4View c, Kv4Move a) {
  const int parts = c.dim / 64 + 1, part = blockIdx.x % parts, which = blockIdx.x / parts, head = blockIdx.y;
  wait_for_previous();
  let_next_start();
  const int64_t slots = c.num_pages << c.page_shift;
  uint8_t* const codes = which ? c.codes[1] : c.codes[0];
  float* const scales = which ? c.scales[1] : c.scales[0];
  int64_t to[kMoves];
  uint4 x[kMoves][2];
#pragma unroll
  for (int k = 0; k < kMoves; ++k) {
    const int64_t i = threadIdx.x + k * kMoveThreads;
    to[k] = -1;
    if (i >= a.tokens) continue;
    const int64_t source = a.source[i], target = a.target[i];
    if (source < 0 || source >= slots || target < 0 || target >= slots) continue;
    to[k] = moved_vector(c, target, head);
    const int64_t from = moved_vector(c, source, head);
    if (part == 0) {
      x[k][0].x = __float_as_uint(scales[from]);
    } else {
      const uint4* p = reinterpret_cast<const uint4*>(codes + from * (c.dim / 2) + (part - 1) * 32);
      x[k][0] = p[0];
      x[k][1] = p[1];
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kMoves; ++k) {
    if (to[k] < 0) continue;
    if (part == 0) {
      scales[to[k]] = __uint_as_float(x[k][0].x);
    } else {
      uint4* p = reinterpret_cast<uint4*>(codes + to[k] * (c.dim / 2) + (part - 1) * 32);
      p[0] = x[k][0];
      p[1] = x[k][1];
    }
  }
}
// More tokens: out to a workspace, [key or value][head][token] codes, then scales alike, and back in a second launch, most
// of it through L2.  A thread has 16 bytes of codes of kManyMoves vectors, asked for together, a vector's first
// thread its scale too.  16,411 tokens of 8 heads, D = 128 (17.9 MB): either pass 9 us alone, both with the tokens' read back
// (25.4 us) 33.9, as the second starts while the first is at work and has its slots by then.
constexpr int kManyMoves = 4;
template <bool kOut, int kDim>
__global__ void __launch_bounds__(kThreads) kv4_move_many_kernel(Kv4View c, Kv4Move a) {
  constexpr int kLanes = kDim / 32, kStep = kThreads / kLanes;
  const int head = blockIdx.y, which = blockIdx.z, lane = threadIdx.x % kLanes;
  uint8_t* const codes = which ? c.codes[1] : c.codes[0];
  float* const scales = which ? c.scales[1] : c.scales[0];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kStep * kManyMoves) + threadIdx.x / kLanes;
  const int64_t slots = c.num_pages << c.page_shift, kept0 = (static_cast<int64_t>(which) * c.heads + head) * a.tokens;
  uint4* const kept = static_cast<uint4*>(a.workspace) + kept0 * kLanes + lane;
  float* const kept_scales = reinterpret_cast<float*>(static_cast<uint4*>(a.workspace) + 2 * c.heads * a.tokens * kLanes) + kept0;
  if (kOut) {  // what the second pass reads before it waits is there when it starts
    wait_for_previous();
    let_next_start();
  }
  int64_t here[kManyMoves];  // -1: none
#pragma unroll
  for (int k = 0; k < kManyMoves; ++k) {
    const int64_t i = first + k * kStep;
    here[k] = -1;
    if (i >= a.tokens) continue;
    const int64_t source = a.source[i], target = a.target[i];
    if (source < 0 || source >= slots || target < 0 || target >= slots) continue;
    here[k] = moved_vector(c, kOut ? source : target, head);
  }
  if (!kOut) wait_for_previous();
  uint4 x[kManyMoves];
  float s[kManyMoves];
#pragma unroll
  for (int k = 0; k < kManyMoves; ++k) {
    if (here[k] < 0) continue;
    const int64_t i = first + k * kStep;
    x[k] = kOut ? *(reinterpret_cast<const uint4*>(codes + here[k] * (kDim / 2)) + lane) : kept[i * kLanes];
    if (lane == 0) s[k] = kOut ? scales[here[k]] : kept_scales[i];
  }
#pragma unroll
  for (int k = 0; k < kManyMoves; ++k) {
    if (here[k] < 0) continue;
    const int64_t i = first + k * kStep;
    if (kOut) kept[i * kLanes] = x[k];
    else *(reinterpret_cast<uint4*>(codes + here[k] * (kDim / 2)) + lane) = x[k];
    if (lane == 0) (kOut ? kept_scales[i] : scales[here[k]]) = s[k];
  }
}
template <int kDim>
void launch_move_many(const Kv4View& c, const Kv4Move& a, cudaStream_t stream) {
  const int64_t per_block = kThreads / (kDim / 32) * kManyMoves;
  const dim3 blocks(static_cast<unsigned>((a.tokens + per_block - 1) / per_block), static_cast<unsigned>(c.heads), 2);
  launch_early(kv4_move_many_kernel<true, kDim>, blocks, kThreads, 0, stream, 0, "launch cache move kernel", c, a);
  // The second reads its slots while the first is at work: neither writes them.
  launch_early(kv4_move_many_kernel<false, kDim>, blocks, kThreads, 0, stream, 0, "launch cache move kernel", c, a);
}

template <class T, bool kAligned>
void append_aligned(const Kv4View& c, const Kv4Append& a, cudaStream_t stream) {
  const int64_t per_block = kThreads / (c.dim / 8) * kWrites;
  const dim3 blocks(static_cast<unsigned>((a.tokens + per_block - 1) / per_block), static_cast<unsigned>(c.heads));
  if (c.dim == 64) kv4_append_kernel<T, 64, kAligned><<<blocks, kThreads, 0, stream>>>(c, a);
  else if (c.dim == 128) kv4_append_kernel<T, 128, kAligned><<<blocks, kThreads, 0, stream>>>(c, a);
  else kv4_append_kernel<T, 256, kAligned><<<blocks, kThreads, 0, stream>>>(c, a);
}

template <class T>
void append_typed(const Kv4View& c, const Kv4Append& a, cudaStream_t stream) {
  // Rows start on 16 bytes where base and strides do (a vector's threads load 16 bytes each then).
  uint64_t starts = 0;
  for (int w = 0; w < 2; ++w)
    starts |= reinterpret_cast<uintptr_t>(a.x[w]) | static_cast<uint64_t>(a.token_stride[w]) * sizeof(T) |
              static_cast<uint64_t>(a.head_stride[w]) * sizeof(T);
  if ((starts & 15) == 0) append_aligned<T, true>(c, a, stream);
  else append_aligned<T, false>(c, a, stream);
}

template <class T>
void read_typed(const Kv4View& c, const Kv4Read& a, cudaStream_t stream) {
  const int64_t vectors = a.tokens * c.heads, per_block = kThreads / (c.dim * static_cast<int>(sizeof(T)) / 16) * kReads;
  const unsigned blocks = static_cast<unsigned>((vectors + per_block - 1) / per_block);
  if (c.dim == 64) kv4_read_kernel<T, 64><<<blocks, kThreads, 0, stream>>>(c, a);
  else if (c.dim == 128) kv4_read_kernel<T, 128><<<blocks, kThreads, 0, stream>>>(c, a);
  else kv4_read_kernel<T, 256><<<blocks, kThreads, 0, stream>>>(c, a);
}

}  // namespace

size_t kv4_move_workspace_bytes(const Kv4View& c, int64_t tokens) {
  return tokens > kMostMoved ? static_cast<size_t>(2) * c.heads * tokens * (c.dim / 2 + 4) : 0;
}

void launch_kv4_move(const Kv4View& c, const Kv4Move& a, cudaStream_t stream) {
  if (a.tokens <= 0) return;
  if (a.tokens <= kMostMoved) {
    launch_early(kv4_move_kernel, dim3(2 * (c.dim / 64 + 1), static_cast<unsigned>(c.heads)), kMoveThreads, 0, stream, 0,
                 "launch cache move kernel", c, a);
  } else {
    if (c.dim == 64) launch_move_many<64>(c, a, stream);
    else if (c.dim == 128) launch_move_many<128>(c, a, stream);
    else launch_move_many<256>(c, a, stream);
  }
}

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
