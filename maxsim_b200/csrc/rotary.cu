// Rotary positions with several axes: pairs of a head's dimensions turn by an angle of the token's position.
//
// Pair i of a token turns by pos[axis(i)] * f_i: (a, b) -> (a cos - b sin, a sin + b cos), inverse: the other way.
// Angles.  f_i is held in turns, F_i = round(f_i / 2 pi * 2^64): the product pos * F_i in 64 bits wraps at whole turns,
// so the fraction of a turn is exact to |pos| 2^-65 of one however far the position (the product of two fp32 numbers
// would be off by 2^-8 of a turn at 10^5).  The nearest quarter turn is taken off in integers; what is left, an eighth
// of a turn at most, becomes fp32 with all its bits.
//   Bound: memory, every element is read and written once.  A block has a few tokens: their sines and cosines are formed
//   once, in shared memory, for all heads, while the first vectors are on their way.
#include <algorithm>

#include "quant4.cuh"
#include "rotary.cuh"

namespace msb {
namespace {

constexpr int kThreads = 256;
constexpr int kTurns = 512;  // sines and cosines of a block, at most
constexpr int kBatch = 4;    // items of a thread on their way together

// kPer consecutive elements.
template <class T, int kPer>
struct Piece {
  __align__(sizeof(T) * kPer) T e[kPer];
};
template <class T, int kPer>
__device__ __forceinline__ void load_piece(Piece<T, kPer>& v, const T* p) {
  if constexpr (sizeof(T) * kPer == 16) *reinterpret_cast<uint4*>(v.e) = *reinterpret_cast<const uint4*>(p);
  else v.e[0] = *p;
}
template <class T, int kPer>
__device__ __forceinline__ void store_piece(T* p, const Piece<T, kPer>& v) {
  if constexpr (sizeof(T) * kPer == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v.e);
  else *p = v.e[0];
}

__device__ __forceinline__ float2 turn(const Rotate& a, int64_t token, int pair) {
  const int64_t at = a.axis[pair] * a.position_axis + token * a.position_token;
  const int64_t position = a.wide ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
  const uint64_t part = static_cast<uint64_t>(position) * a.turns[pair];
  const uint32_t quarter = static_cast<uint32_t>((part + (uint64_t{1} << 61)) >> 62);
  const int64_t rest = static_cast<int64_t>(part - (static_cast<uint64_t>(quarter) << 62));
  float s, c;
  sincospif(__ll2float_rn(rest) * 0x1p-63F, &s, &c);
  // cos and sin of (quarter / 4 + rest) turns
  float2 r = quarter & 1 ? make_float2(-s, c) : make_float2(c, s);
  if (quarter & 2) r = make_float2(-r.x, -r.y);
  if (a.inverse) r.y = -r.y;
  return r;
}

// kPer: elements that a thread has of either half of its pairs (halves), or in all (neighbours): 16 bytes, or, where
// something does not start on 16 bytes, one pair.
template <class T, int kPer, bool kNeighbours>
__global__ void __launch_bounds__(kThreads) rotate_kernel(Rotate a, int block_tokens, int pieces, int turning) {
  constexpr int kVec = kNeighbours && kPer == 1 ? 1 : kPer;
  __shared__ float2 turns[kTurns];
  const int heads = a.heads[0] + a.heads[1];
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * block_tokens;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(block_tokens), a.tokens - token0));
  const int items = tokens * heads * pieces;
  struct Item {
    int token, which, head, piece;
  };
  auto item_of = [&](int i) {
    Item r;
    const int vector = i / pieces;
    r.piece = i - vector * pieces;
    r.token = vector / heads;
    const int head = vector - r.token * heads;
    r.which = head >= a.heads[0];
    r.head = r.which ? head - a.heads[0] : head;
    return r;
  };
  // Where a piece's elements start in its vector, and how far its second part lies from its first.  Of the pieces the
  // first `turning` turn; the others are copied.
  auto place = [&](int piece) {
    if (kNeighbours && kPer == 1) return piece < turning ? 2 * piece : 2 * a.half + (piece - turning);
    if (kNeighbours) return piece * kPer;
    return piece < turning ? piece * kPer : 2 * a.half + (piece - turning) * kPer;
  };
  constexpr bool kTwoParts = !kNeighbours || kPer == 1;
  const int apart = kNeighbours ? 1 : a.half;
  Piece<T, kVec> x[kBatch][2];
  auto load = [&](int base) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = base + k * kThreads;
      if (i >= items) continue;
      const Item at = item_of(i);
      const T* p = static_cast<const T*>(a.x[at.which]) + (token0 + at.token) * a.x_token[at.which] +
                   at.head * a.x_head[at.which] + place(at.piece);
      load_piece(x[k][0], p);
      if (kTwoParts && at.piece < turning) load_piece(x[k][1], p + apart);
    }
  };
  load(threadIdx.x);
  for (int i = threadIdx.x; i < tokens * a.half; i += kThreads) {
    const int token = i / a.half;
    turns[i] = turn(a, token0 + token, i - token * a.half);
  }
  __syncthreads();
  for (int base = threadIdx.x; base < items; base += kBatch * kThreads) {
    if (base != threadIdx.x) load(base);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = base + k * kThreads;
      if (i >= items) continue;
      const Item at = item_of(i);
      T* p = static_cast<T*>(a.y[at.which]) + (token0 + at.token) * a.y_token[at.which] + at.head * a.y_head[at.which] +
             place(at.piece);
      if (at.piece < turning) {
        if constexpr (kTwoParts) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            const float2 t = turns[at.token * a.half + at.piece * kVec + e];
            const float u = to_f32(x[k][0].e[e]), v = to_f32(x[k][1].e[e]);
            x[k][0].e[e] = from_f32<T>(u * t.x - v * t.y);
            x[k][1].e[e] = from_f32<T>(u * t.y + v * t.x);
          }
          store_piece(p + apart, x[k][1]);
        } else {
#pragma unroll
          for (int e = 0; e < kVec; e += 2) {
            const float2 t = turns[at.token * a.half + (at.piece * kVec + e) / 2];
            const float u = to_f32(x[k][0].e[e]), v = to_f32(x[k][0].e[e + 1]);
            x[k][0].e[e] = from_f32<T>(u * t.x - v * t.y);
            x[k][0].e[e + 1] = from_f32<T>(u * t.y + v * t.x);
          }
        }
      }
      store_piece(p, x[k][0]);
    }
  }
}

template <class T, int kPer, bool kNeighbours>
void launch_pairs(const Rotate& a, cudaStream_t stream) {
  const int turned = 2 * a.half, heads = a.heads[0] + a.heads[1];
  const int turning = kNeighbours && kPer > 1 ? turned / kPer : a.half / kPer;
  const int pieces = turning + (a.dim - turned) / kPer;
  // As many tokens to a block as give each thread an item of sines or a batch of vectors, whichever is less.
  const int64_t items = static_cast<int64_t>(heads) * pieces;
  int block_tokens = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kThreads / a.half, kBatch * kThreads / items)));
  const int64_t blocks = (a.tokens + block_tokens - 1) / block_tokens;
  rotate_kernel<T, kPer, kNeighbours><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(a, block_tokens, pieces, turning);
}

template <class T>
void launch_typed(const Rotate& a, cudaStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  uint64_t starts = 0;
  for (int w = 0; w < 2; ++w) {
    if (a.heads[w] == 0) continue;
    starts |= reinterpret_cast<uintptr_t>(a.x[w]) | reinterpret_cast<uintptr_t>(a.y[w]);
    for (const int64_t stride : {a.x_token[w], a.x_head[w], a.y_token[w], a.y_head[w]})
      starts |= static_cast<uint64_t>(stride) * sizeof(T);
  }
  // What a thread has in one part: whole pieces of the half (halves) or of the pairs, and of what stays.
  const int part = a.neighbours ? 2 * a.half : a.half;
  const bool wide = (starts & 15) == 0 && part % kWide == 0 && (a.dim - 2 * a.half) % kWide == 0;
  if (a.neighbours) {
    if (wide) launch_pairs<T, kWide, true>(a, stream);
    else launch_pairs<T, 1, true>(a, stream);
  } else {
    if (wide) launch_pairs<T, kWide, false>(a, stream);
    else launch_pairs<T, 1, false>(a, stream);
  }
}

}  // namespace

void launch_rotate(const Rotate& a, cudaStream_t stream) {
  if (a.tokens <= 0 || a.heads[0] + a.heads[1] <= 0) return;
  if (a.type == kElemF32) launch_typed<float>(a, stream);
  else if (a.type == kElemF16) launch_typed<__half>(a, stream);
  else launch_typed<__nv_bfloat16>(a, stream);
  count_launch();
  check(cudaGetLastError(), "launch rotary kernel");
}

}  // namespace msb
