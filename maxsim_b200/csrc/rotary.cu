// Rotary positions with several axes: pairs of a head's dimensions turn by an angle of the token's position.
//
// Pair i of a token turns by pos[axis(i)] * f_i: (a, b) -> (a cos - b sin, a sin + b cos), inverse: the other way.
// Angles.  f_i is held in turns, F_i = round(f_i / 2 pi * 2^64): the product pos * F_i in 64 bits wraps at whole turns,
// so the fraction of a turn is exact to |pos| 2^-65 of one however far the position (the product of two fp32 numbers
// would be off by 2^-8 of a turn at 10^5).  The nearest quarter turn is taken off in integers; what is left, an eighth
// of a turn at most, becomes fp32 with all its bits.
//   Bound: memory, every element is read and written once.  A block has a few tokens: their sines and cosines are formed
//   once, in shared memory, for all heads, while the first vectors are on their way.  A thread keeps those of its piece of a
//   vector in registers and goes through heads; two vectors on their way leave registers for four blocks of 256 threads an
//   SM (four and one block's worth: 70 us where this takes 57; sines read from shared memory for every vector: 79).
//   Measured on the device: 16,384 tokens, 32 + 8 heads of 128, bf16, 56 to 57 us, 6.0 TB/s; 64 of them 2.5 us.
#include <algorithm>
#include <climits>

#include "quant4.cuh"
#include "rotary.cuh"

namespace msb {
namespace {

// Threads of a block, at most: a vector of 1,024 dimensions has as many pieces at most.
constexpr int most_threads(int per) { return per == 1 ? 1024 : 256; }
constexpr int kTurns = 1024;  // sines and cosines of a block, at most
constexpr int kBatch = 2;     // vectors of a thread on their way together
constexpr int kHeads = 4;     // of a thread, about

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

// How a call's blocks share its vectors: those before `blocks` of the first have queries, the others keys.
struct Split {
  int64_t blocks;
  int tokens[2];      // of a block
  int head_lanes[2];
  int pieces;         // of a vector
  int turning;        // the first of these turn, the others are copied
};
// A thread has one piece of one token's vectors, in every `head_lanes`-th head: its sines and cosines stay in registers.
// kPer: elements of a piece, of either half of its pairs (halves), or in all (neighbours): 16 bytes, or, where something
// does not start on 16 bytes, one pair.
template <class T, int kPer, bool kNeighbours>
__global__ void __launch_bounds__(most_threads(kPer), kPer == 1 ? 1 : 4)
    rotate_kernel(const __grid_constant__ Rotate a, const __grid_constant__ Split c) {
  constexpr bool kTwoParts = !kNeighbours || kPer == 1;   // a piece's elements lie in two places
  constexpr int kPairs = kTwoParts ? kPer : kPer / 2;     // of a piece
  __shared__ float2 turns[kTurns];
  wait_for_previous();
  let_next_start();
  const int which = blockIdx.x >= c.blocks;
  const int heads = a.heads[which], head_lanes = c.head_lanes[which], block_tokens = c.tokens[which];
  const int64_t token0 = (static_cast<int64_t>(blockIdx.x) - (which ? c.blocks : 0)) * block_tokens;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(block_tokens), a.tokens - token0));
  const int vector = threadIdx.x / c.pieces, piece = threadIdx.x - vector * c.pieces;
  const int my_token = vector / head_lanes, head0 = vector - my_token * head_lanes;
  const bool turns_it = piece < c.turning;
  const int start = turns_it ? (kTwoParts && kNeighbours ? 2 * piece : piece * kPer) : 2 * a.half + (piece - c.turning) * kPer;
  const int apart = kNeighbours ? 1 : a.half;
  const T* x = static_cast<const T*>(a.x[which]) + (token0 + my_token) * a.x_token[which] + head0 * a.x_head[which] + start;
  T* y = static_cast<T*>(a.y[which]) + (token0 + my_token) * a.y_token[which] + head0 * a.y_head[which] + start;
  const int64_t x_step = head_lanes * a.x_head[which], y_step = head_lanes * a.y_head[which];
  int left = my_token < tokens ? (heads - head0 + head_lanes - 1) / head_lanes : 0;  // heads of this thread
  Piece<T, kPer> v[kBatch][2];
  auto load = [&]() {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (k >= left) break;
      load_piece(v[k][0], x);
      if (kTwoParts && turns_it) load_piece(v[k][1], x + apart);
      x += x_step;
    }
  };
  load();
  for (int i = threadIdx.x; i < tokens * a.half; i += blockDim.x) {
    const int token = i / a.half;
    turns[i] = turn(a, token0 + token, i - token * a.half);
  }
  __syncthreads();
  if (left <= 0) return;
  float2 t[kPairs];
#pragma unroll
  for (int e = 0; e < kPairs; ++e) t[e] = turns_it ? turns[my_token * a.half + piece * kPairs + e] : make_float2(1.0F, 0.0F);
#pragma unroll 1
  for (;;) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (k >= left) break;
      if (turns_it) {
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          T& u = kTwoParts ? v[k][0].e[e] : v[k][0].e[2 * e];
          T& w = kTwoParts ? v[k][1].e[e] : v[k][0].e[2 * e + 1];
          const float fu = to_f32(u), fw = to_f32(w);
          u = from_f32<T>(fu * t[e].x - fw * t[e].y);
          w = from_f32<T>(fu * t[e].y + fw * t[e].x);
        }
        if (kTwoParts) store_piece(y + apart, v[k][1]);
      }
      store_piece(y, v[k][0]);
      y += y_step;
    }
    left -= kBatch;
    if (left <= 0) return;
    load();
  }
}

template <class T, int kPer, bool kNeighbours>
void launch_pairs(const Rotate& a, cudaStream_t stream) {
  const int turned = 2 * a.half;
  Split c{};
  c.turning = kNeighbours && kPer > 1 ? turned / kPer : a.half / kPer;
  c.pieces = c.turning + (a.dim - turned) / kPer;
  // Heads of a thread: some batches; few tokens spread over the SMs, one to a block.
  const bool few = a.tokens <= 2 * sm_count();
  constexpr int kWanted = 256;
  int threads = std::min(kWanted, a.half);
  int64_t blocks[2];
  for (int w = 0; w < 2; ++w) {
    c.head_lanes[w] = std::max(1, std::min(few ? a.heads[w] : (a.heads[w] + kHeads - 1) / kHeads, kWanted / c.pieces));
    const int per_token = c.pieces * c.head_lanes[w];  // at most most_threads(kPer)
    c.tokens[w] = few ? 1 : std::max(1, std::min(kWanted / per_token, kTurns / a.half));
    blocks[w] = a.heads[w] > 0 ? (a.tokens + c.tokens[w] - 1) / c.tokens[w] : 0;
    if (blocks[w] > 0) threads = std::max(threads, per_token * c.tokens[w]);
  }
  if (blocks[0] + blocks[1] > INT_MAX) throw InvalidArgument("tokens are too many for one call");
  c.blocks = blocks[0];
  threads = (threads + 31) / 32 * 32;
  launch_early(rotate_kernel<T, kPer, kNeighbours>, dim3(static_cast<unsigned>(blocks[0] + blocks[1])), threads, 0, stream, 0,
               "launch rotary kernel", a, c);
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
}

}  // namespace msb
