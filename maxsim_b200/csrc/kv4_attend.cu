// Attention over the 4-bit key/value cache.
//
// Row (query token i of sequence b, query head h) sees cached tokens j <= pos (causal) and
// j > pos - window, pos = length - rows + i.  With s_j = scale * ks_j * <q, kc_j>, its output is
// sum_j e^(s_j - m) vs_j vc_j / sum_j e^(s_j - m) in one pass with a running reference m, sums in fp32; a row
// that sees nothing writes zeros and a log-sum-exp of -inf.
//
// kv4_attend_kernel: few rows a sequence (decode, drafted tokens).
//   Bound: the codes' bytes, D + 8 per token and head, then the integer pipe that unpacks them.
//   Products.  m16n8k16 fp16 products with the tokens as the 16-row operand: S^T = K Q^T, O^T = V^T P^T, so
//   8 query rows (the heads that share a key/value head, times the query tokens) fill a column tile instead
//   of half a row tile.  tcgen05 wants 128 rows of queries, which decode has not.
//   Operands straight from global memory: the order of the summed index is free, so lane (g, t) = (lane / 4,
//   lane % 4) takes D / 4 consecutive dimensions of key tokens g and g + 8 (a 16-byte load each at D = 128),
//   and D / 8 consecutive dimensions of value tokens 2t, 2t + 1, 2t + 8, 2t + 9; nothing passes through shared
//   memory.  A 16-token tile lies in one page (pages are powers of two >= 16), so a tile has one page lookup.
//   Unpacking.  Nibble n of a code is code & 15; (w & 0x00f000f0) ^ 0x54805480 is the fp16 pair 72 + code in
//   one logic operation.  Keys keep the 72: accumulators start at -72 sum(q).  Values subtract it (their sum
//   over tokens would lose digits to it): both are exact.
//   Queries are fp16 after a power of two per row that puts their maximum in [1, 2): exact for fp16 inputs and
//   for bf16 ones down to 2^-24 of the row's maximum.  Probabilities are fp16 (11 bits): they enter one sum
//   that is rounded to the output's type, of as many bits or fewer.
//   Reference.  Probabilities carry the values' scales, p_j vs_j, so the running reference is the maximum of
//   s_j + e_j with vs_j in 2^(e_j + [0, 1)): p_j vs_j stays in fp16's range whatever the scales are.  e_j is
//   held to +-110, so the fp32 sum of the p_j stays finite.
//   Work split.  The 128-token tiles of all (sequence, head, row block) segments form one line, cut into equal
//   ranges, one per resident block, from the lengths on the device: no plan, no host copy, no imbalance.
//   A segment cut by a range's end leaves partial sums in the workspace (at most two per block), which
//   kv4_join_kernel adds in a fixed order; it is launched early (programmatic dependent launch).
#include <algorithm>

#include "quant4.cuh"

namespace msb {
namespace {

constexpr int kWarps = 4;
constexpr int kStep = 32;              // tokens a warp takes at a time
constexpr int kTile = kWarps * kStep;  // tokens of one unit of the work line
constexpr float kLift = 8.0F;          // references lie 2^8 below the maximum: probabilities of 2^-22 are normal in fp16

template <class T>
__device__ __forceinline__ T load_stream(const void* p);
template <>
__device__ __forceinline__ uint4 load_stream<uint4>(const void* p) {
  uint4 r;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
template <>
__device__ __forceinline__ uint2 load_stream<uint2>(const void* p) {
  uint2 r;
  asm("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}
template <>
__device__ __forceinline__ uint32_t load_stream<uint32_t>(const void* p) {
  uint32_t r;
  asm("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}
// kWords consecutive words (a power of two; the address is aligned to their size or to 16 bytes).
template <int kWords>
__device__ __forceinline__ void load_words(uint32_t (&r)[kWords], const uint8_t* p) {
  if constexpr (kWords == 1) {
    r[0] = load_stream<uint32_t>(p);
  } else if constexpr (kWords == 2) {
    const uint2 v = load_stream<uint2>(p);
    r[0] = v.x, r[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const uint4 v = load_stream<uint4>(p + 4 * i);
      r[i] = v.x, r[i + 1] = v.y, r[i + 2] = v.z, r[i + 3] = v.w;
    }
  }
}

// fp16 pair 72 + code of nibbles i and i + 4 of a word.
template <int kI>
__device__ __forceinline__ uint32_t codes_plus72(uint32_t w) {
  const uint32_t at = kI == 0 ? w << 4 : w >> (4 * kI - 4);
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x54805480, 0x6a;" : "=r"(r) : "r"(at));  // (a & b) ^ c
  return r;
}
template <int kI>
__device__ __forceinline__ uint32_t codes_exact(uint32_t w) {
  const uint32_t v = codes_plus72<kI>(w);
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x54805480u));  // 0x5480 is 72
  return r;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// What sums with reference `from` are multiplied by to have reference `to` >= from.  Sums with reference -inf
// are 0, or NaN where a score was: they stay so.
__device__ __forceinline__ float fade_to(float from, float to) { return from == to ? 1.0F : exp2_fast(from - to); }
__device__ __forceinline__ float log_sum(float m, float l) {
  return l == 0.0F ? -INFINITY : (m - kLift + __log2f(l)) * 0.693147181F;
}
// Exponent of a scale (the e of 2^(e + [0, 1))), held to +-110.
__device__ __forceinline__ float scale_exponent(float s) {
  const int e = static_cast<int>((__float_as_uint(s) >> 23) & 255) - 127;
  return static_cast<float>(max(-110, min(110, e)));
}

// The work line: units of kTile tokens of every (sequence, key/value head, row block).
struct Line {
  int heads;        // of the cache
  int shared;       // query heads per cache head
  int block_rows;   // rows of a row block
  int page_shift;
};
struct SequenceWork {
  Kv4Sequence q;
  int begin;        // first token that a row may see, down to a multiple of 16
  int tiles;        // units of one segment
  int blocks;       // row blocks
  __device__ __forceinline__ int64_t units(const Line& l) const {
    return static_cast<int64_t>(l.heads) * blocks * tiles;
  }
};
__device__ __forceinline__ SequenceWork sequence_work(const Kv4Attend& a, const Line& l, int b) {
  SequenceWork w;
  w.q = kv4_sequence(a, l.page_shift, b);
  w.begin = 0;
  if (a.window > 0) w.begin = max(0, max(0, w.q.length - w.q.rows) - a.window + 1) & ~15;
  // A sequence of no tokens keeps one empty unit: its rows are written as zeros.
  w.tiles = max(1, (w.q.length - w.begin + kTile - 1) / kTile);
  w.blocks = (w.q.rows * l.shared + l.block_rows - 1) / l.block_rows;
  return w;
}

// Units of all sequences, and those before sequence b: every thread of the block gets both.  kWarps * 32
// sequences at a time.
struct Place {
  int64_t total;
  int64_t before;   // units before the found sequence
  int sequence;
};
// Finds the sequence that holds unit (range start) `first(total)`, or sums up to sequence `want` if want >= 0.
template <class F>
__device__ __forceinline__ Place find_place(const Kv4Attend& a, const Line& l, int want, F first, int64_t* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kBlock = kWarps * 32;
  int64_t mine = 0, total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kBlock) {
    mine = b0 + threadIdx.x < a.batch ? sequence_work(a, l, b0 + threadIdx.x).units(l) : 0;
    total += mine;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, d);
  if (lane == 0) scratch[warp] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += scratch[w];
  Place p{total, 0, want >= 0 ? want : a.batch};
  const int64_t target = want >= 0 ? -1 : first(total);
  int64_t carry = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kBlock) {
    if (a.batch > kBlock) mine = b0 + threadIdx.x < a.batch ? sequence_work(a, l, b0 + threadIdx.x).units(l) : 0;
    int64_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
      if (lane >= d) upto += o;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = upto;
    if (threadIdx.x == 0) scratch[kWarps] = -1;
    __syncthreads();
    int64_t base = carry, chunk = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += scratch[w];
      chunk += scratch[w];
    }
    const int64_t before = base + upto - mine;
    const bool hit = want >= 0 ? b0 + static_cast<int>(threadIdx.x) == want : target >= before && target < before + mine;
    if (hit) {
      scratch[kWarps] = before;
      scratch[kWarps + 1] = b0 + threadIdx.x;
    }
    __syncthreads();
    if (scratch[kWarps] >= 0) {
      p.before = scratch[kWarps];
      p.sequence = static_cast<int>(scratch[kWarps + 1]);
      break;
    }
    carry += chunk;
  }
  __syncthreads();
  return p;
}
// Of n = min(blocks, total) ranges, range c is [c total / n, (c + 1) total / n): none is empty.
__device__ __forceinline__ int64_t ranges(int64_t total, int64_t blocks) {
  return total < blocks ? (total > 0 ? total : 1) : blocks;
}
__device__ __forceinline__ int64_t range_start(int64_t total, int64_t c, int64_t n) { return c * total / n; }
// The range that holds unit u.
__device__ __forceinline__ int64_t range_of(int64_t total, int64_t u, int64_t n) { return ((u + 1) * n - 1) / total; }

// Partial sums of one segment's row block: rows x dim unnormalised outputs, then (reference, sum) per row.
__host__ __device__ constexpr int partial_floats(int rows, int dim) { return rows * dim + 2 * rows; }

template <class T, int kDim, int kTiles>
__global__ void __launch_bounds__(kWarps * 32) kv4_attend_kernel(Kv4View c, Kv4Attend a, Line line) {
  constexpr int kRows = 8 * kTiles;      // rows of a row block
  constexpr int kKeyWords = kDim / 32;   // of one token, per lane
  constexpr int kValueWords = kDim / 64;
  constexpr int kOut = kDim / 16;        // 16-dimension tiles of the output
  constexpr int kPitch = kDim + 4;       // floats between rows in shared memory
  __shared__ float merge[kWarps][kRows * kPitch / 2];
  __shared__ float stats[kWarps][2][kRows];
  __shared__ int64_t scratch[kWarps + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;

  const int64_t block = blockIdx.x;
  const Place place = find_place(
      a, line, -1, [&](int64_t total) { return range_start(total, block, ranges(total, gridDim.x)); }, scratch);
  const int64_t n = ranges(place.total, gridDim.x);
#if __CUDA_ARCH__ >= 900
  cudaTriggerProgrammaticLaunchCompletion();
#endif
  if (block >= n) return;
  int64_t unit = range_start(place.total, block, n);
  const int64_t unit_end = range_start(place.total, block + 1, n);
  int64_t before = place.before;
  int b = place.sequence;
  SequenceWork w{};
  if (unit < unit_end) w = sequence_work(a, line, b);

  while (unit < unit_end) {
    while (unit >= before + w.units(line)) {
      before += w.units(line);
      w = sequence_work(a, line, ++b);
    }
    // The segment (head, row block) that holds `unit`, and this block's part of it.
    const int64_t inside = unit - before;
    const int64_t segment = inside / w.tiles;
    const int tile0 = static_cast<int>(inside - segment * w.tiles);
    const int tile1 = static_cast<int>(min(static_cast<int64_t>(w.tiles), tile0 + (unit_end - unit)));
    const int head = static_cast<int>(segment / w.blocks), row0 = static_cast<int>(segment % w.blocks) * kRows;
    const int all_rows = w.q.rows * line.shared;

    // Queries: lane (g, t) holds row g of each column tile, dimensions t * kDim / 4 and on.
    uint32_t q[kTiles][2 * kKeyWords][2];
    float lift[kTiles][2];   // -72 sum(q) of columns 2t, 2t + 1
    float factor[kTiles][2]; // scale * log2(e) * the row's power of two
    int last[kTiles][2], first[kTiles][2];  // tokens that columns 2t, 2t + 1 see: first <= j <= last
    int every_last = INT_MAX, every_first = 0, any_last = -1, any_first = INT_MAX;
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      const int r = row0 + nt * 8 + g;
      float x[kKeyWords * 8], top = 0.0F;
      if (r < all_rows) {
        const T* p = static_cast<const T*>(a.query) + (w.q.row0 + r / line.shared) * a.q_row_stride +
                     static_cast<int64_t>(head * line.shared + r % line.shared) * a.q_head_stride + t * (kDim / 4);
#pragma unroll
        for (int d = 0; d < kKeyWords * 8; ++d) x[d] = to_f32(p[d]);
      } else {
#pragma unroll
        for (int d = 0; d < kKeyWords * 8; ++d) x[d] = 0.0F;
      }
#pragma unroll
      for (int d = 0; d < kKeyWords * 8; ++d) top = fmaxf(top, fabsf(x[d]));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      const int e = max(-126, min(126, static_cast<int>(__float_as_uint(top) >> 23) - 127));
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      float sum = 0.0F;
#pragma unroll
      for (int word = 0; word < kKeyWords; ++word) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t v = pack_half2(x[8 * word + i] * down, x[8 * word + 4 + i] * down);
          q[nt][2 * word + (i >> 1)][i & 1] = v;
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
          sum += f.x + f.y;
        }
      }
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
      const float up = a.scale * 1.44269504F * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
      for (int k = 0; k < 2; ++k) {  // from the lanes that hold row 2t + k to the column's lanes
        lift[nt][k] = -72.0F * __shfl_sync(0xFFFFFFFFu, sum, 4 * (2 * t + k));
        factor[nt][k] = __shfl_sync(0xFFFFFFFFu, up, 4 * (2 * t + k));
        const int rr = row0 + nt * 8 + 2 * t + k;
        first[nt][k] = 0;
        last[nt][k] = INT_MAX;  // rows past the block are not written: no reason to mask for them
        if (rr < all_rows) {
          const int pos = w.q.length - w.q.rows + rr / line.shared;
          last[nt][k] = a.causal ? pos : w.q.length - 1;
          first[nt][k] = a.window > 0 ? max(0, pos - a.window + 1) : 0;
          every_last = min(every_last, last[nt][k]);
          every_first = max(every_first, first[nt][k]);
          any_last = max(any_last, last[nt][k]);
          any_first = min(any_first, first[nt][k]);
        }
      }
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      every_last = min(every_last, __shfl_xor_sync(0xFFFFFFFFu, every_last, d));
      every_first = max(every_first, __shfl_xor_sync(0xFFFFFFFFu, every_first, d));
      any_last = max(any_last, __shfl_xor_sync(0xFFFFFFFFu, any_last, d));
      any_first = min(any_first, __shfl_xor_sync(0xFFFFFFFFu, any_first, d));
    }

    float o[kOut][kTiles][4];
    float top[kTiles][2], sum[kTiles][2];
#pragma unroll
    for (int i = 0; i < kOut; ++i)
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][nt][k] = 0.0F;
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) top[nt][0] = top[nt][1] = -INFINITY, sum[nt][0] = sum[nt][1] = 0.0F;

    // This warp's steps of 32 tokens, those that some row sees.
    const int from = w.begin + tile0 * kTile, upto = min(w.begin + tile1 * kTile, any_last + 1);
    int j0 = from + warp * kStep;
    if (any_first > j0) j0 += (any_first - j0) / kTile * kTile;

    uint32_t key[2][2][kKeyWords], value[2][4][kValueWords];
    float key_scale[2][2], value_scale[2][2];
    bool held[2];
    auto tile_vector = [&](int j, bool& ok) -> int64_t {
      ok = false;
      if (j > any_last) return 0;
      const int page = a.page_table[b * a.table_stride + (j >> c.page_shift)];
      ok = page >= 0 && page < c.num_pages;
      return ok ? c.vector(page, head, j & ((1 << c.page_shift) - 1)) : 0;
    };
    int64_t vector[2];
    auto load_keys = [&](int j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        vector[i] = tile_vector(j + 16 * i, held[i]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          load_words(key[i][k], c.codes[0] + (vector[i] + g + 8 * k) * (kDim / 2) + t * (kDim / 8));
          key_scale[i][k] = c.scales[0][vector[i] + g + 8 * k];
          value_scale[i][k] = c.scales[1][vector[i] + g + 8 * k];
        }
      }
    };
    auto load_values = [&]() {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          load_words(value[i][k],
                     c.codes[1] + (vector[i] + 2 * t + (k & 1) + 8 * (k >> 1)) * (kDim / 2) + g * (kDim / 16));
    };
    if (j0 < upto) {
      load_keys(j0);
      load_values();
    }
    for (; j0 < upto; j0 += kTile) {
      // Scores of the step: s[i][nt][0, 1] of token g, [2, 3] of token g + 8, columns 2t, 2t + 1.
      float s[2][kTiles][4];
      float ks[2][2], vs[2][2];
      bool seen[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[i][nt][k] = lift[nt][k & 1];
#pragma unroll
        for (int word = 0; word < kKeyWords; ++word) {
          const uint32_t x = key[i][0][word], y = key[i][1][word];
          const uint32_t x0 = codes_plus72<0>(x), x1 = codes_plus72<1>(x), x2 = codes_plus72<2>(x), x3 = codes_plus72<3>(x);
          const uint32_t y0 = codes_plus72<0>(y), y1 = codes_plus72<1>(y), y2 = codes_plus72<2>(y), y3 = codes_plus72<3>(y);
#pragma unroll
          for (int nt = 0; nt < kTiles; ++nt) {
            mma(s[i][nt], x0, y0, x1, y1, q[nt][2 * word][0], q[nt][2 * word][1]);
            mma(s[i][nt], x2, y2, x3, y3, q[nt][2 * word + 1][0], q[nt][2 * word + 1][1]);
          }
        }
        ks[i][0] = key_scale[i][0], ks[i][1] = key_scale[i][1];
        vs[i][0] = value_scale[i][0], vs[i][1] = value_scale[i][1];
        seen[i] = held[i];
      }
      uint32_t p[2][kTiles][2];
      // Values of this step were loaded with its keys; the next keys are asked for before the softmax.
      uint32_t now[2][4][kValueWords];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int word = 0; word < kValueWords; ++word) now[i][k][word] = value[i][k][word];
      if (j0 + kTile < upto) {
        load_keys(j0 + kTile);
        load_values();
      }
      float e[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        e[i][0] = scale_exponent(vs[i][0]);
        e[i][1] = scale_exponent(vs[i][1]);
      }
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[i][nt][k] *= ks[i][k >> 1] * factor[nt][k & 1];
      }
      bool masked[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = j0 + 16 * i;
        masked[i] = !seen[i] || j < every_first || j + 15 > every_last;
        if (masked[i]) {
#pragma unroll
          for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int at = j + g + 8 * (k >> 1);
              if (!seen[i] || at < first[nt][k & 1] || at > last[nt][k & 1]) s[i][nt][k] = -INFINITY;
            }
        }
      }
      bool moved = false;
      float fade[kTiles][2], ref[kTiles][2];
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float m = fmaxf(fmaxf(s[0][nt][k] + e[0][0], s[0][nt][k + 2] + e[0][1]),
                          fmaxf(s[1][nt][k] + e[1][0], s[1][nt][k + 2] + e[1][1]));
          m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 16));
          m = fmaxf(m, top[nt][k]);
          moved = moved || m > top[nt][k];
          ref[nt][k] = m == -INFINITY ? 0.0F : m - kLift;
          fade[nt][k] = fade_to(top[nt][k], m);
          top[nt][k] = m;
        }
      }
      if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
        for (int nt = 0; nt < kTiles; ++nt) {
          sum[nt][0] *= fade[nt][0];
          sum[nt][1] *= fade[nt][1];
#pragma unroll
          for (int i = 0; i < kOut; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[i][nt][k] *= fade[nt][k & 1];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int nt = 0; nt < kTiles; ++nt) {
          float pv[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float pr = exp2_fast(s[i][nt][k] - ref[nt][k & 1]);
            sum[nt][k & 1] += pr;
            pv[k] = pr * vs[i][k >> 1];
          }
          if (masked[i]) {  // an unseen token's scale may be NaN or infinite
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (s[i][nt][k] == -INFINITY) pv[k] = 0.0F;
          }
          p[i][nt][0] = transpose8x8(pack_half2(pv[0], pv[1]));
          p[i][nt][1] = transpose8x8(pack_half2(pv[2], pv[3]));
        }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int word = 0; word < kValueWords; ++word) {
          const uint32_t va = now[i][0][word], vb = now[i][1][word], vc = now[i][2][word], vd = now[i][3][word];
          const uint32_t x0 = __byte_perm(va, vb, 0x5410), y0 = __byte_perm(va, vb, 0x7632);
          const uint32_t x1 = __byte_perm(vc, vd, 0x5410), y1 = __byte_perm(vc, vd, 0x7632);
#pragma unroll
          for (int nib = 0; nib < 4; ++nib) {
            uint32_t a0, a1, a2, a3;
            if (nib == 0) a0 = codes_exact<0>(x0), a1 = codes_exact<0>(y0), a2 = codes_exact<0>(x1), a3 = codes_exact<0>(y1);
            else if (nib == 1) a0 = codes_exact<1>(x0), a1 = codes_exact<1>(y0), a2 = codes_exact<1>(x1), a3 = codes_exact<1>(y1);
            else if (nib == 2) a0 = codes_exact<2>(x0), a1 = codes_exact<2>(y0), a2 = codes_exact<2>(x1), a3 = codes_exact<2>(y1);
            else a0 = codes_exact<3>(x0), a1 = codes_exact<3>(y0), a2 = codes_exact<3>(x1), a3 = codes_exact<3>(y1);
#pragma unroll
            for (int nt = 0; nt < kTiles; ++nt) mma(o[4 * word + nib][nt], a0, a1, a2, a3, p[i][nt][0], p[i][nt][1]);
          }
        }
    }

    // The warps' parts, joined in the order of the warps.
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float l = sum[nt][k];
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 4);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 8);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 16);
        if (g == 0) {
          stats[warp][0][nt * 8 + 2 * t + k] = top[nt][k];
          stats[warp][1][nt * 8 + 2 * t + k] = l;
        }
      }
    const bool whole = tile0 == 0 && tile1 == w.tiles;
    float* partial = nullptr;
    if (!whole)
      partial = static_cast<float*>(a.workspace) + (2 * block + (tile0 == 0 ? 1 : 0)) * partial_floats(kRows, kDim);
    constexpr int kHalf = kDim / 2;      // dimensions of one pass through shared memory
    constexpr int kHalfPitch = kPitch / 2;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
      // Lanes with g / 4 == half hold dimensions of this half: tile word * 4 + nib of lane g is dimension
      // g * kDim / 8 + 8 word + nib (and + 4).
      if ((g >> 2) == half) {
#pragma unroll
        for (int word = 0; word < kValueWords; ++word)
#pragma unroll
          for (int nib = 0; nib < 4; ++nib)
#pragma unroll
            for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                merge[warp][(nt * 8 + 2 * t + (k & 1)) * kHalfPitch + (g & 3) * (kDim / 8) + 8 * word + nib +
                            4 * (k >> 1)] = o[4 * word + nib][nt][k];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < kRows * kHalf; i += kWarps * 32) {
        const int r = i / kHalf, d = i - r * kHalf;
        if (row0 + r >= all_rows) continue;
        float m = -INFINITY, l = 0.0F, v = 0.0F;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) m = fmaxf(m, stats[k][0][r]);
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          const float f = fade_to(stats[k][0][r], m);
          l += f * stats[k][1][r];
          v += f * merge[k][r * kHalfPitch + d];
        }
        if (whole) {
          const int64_t row = (w.q.row0 + (row0 + r) / line.shared) * a.heads + head * line.shared + (row0 + r) % line.shared;
          static_cast<T*>(a.out)[row * kDim + half * kHalf + d] = from_f32<T>(l == 0.0F ? 0.0F : v / l);
          if (a.lse && half == 0 && d == 0)
            a.lse[row] = log_sum(m, l);
        } else {
          partial[r * kDim + half * kHalf + d] = v;
          if (half == 0 && d == 0) {
            partial[kRows * kDim + 2 * r] = m;
            partial[kRows * kDim + 2 * r + 1] = l;
          }
        }
      }
    }
    __syncthreads();
    unit += tile1 - tile0;
  }
}

// Adds the partial sums of the segments that were cut, in the order of the line.
template <class T, int kDim, int kTiles>
__global__ void __launch_bounds__(kWarps * 32) kv4_join_kernel(Kv4View c, Kv4Attend a, Line line, int64_t blocks) {
  constexpr int kRows = 8 * kTiles;
  __shared__ int64_t scratch[kWarps + 2];
  const int b = blockIdx.x;
  const Place place = find_place(a, line, b, [](int64_t) { return int64_t{0}; }, scratch);
  const SequenceWork w = sequence_work(a, line, b);
#if __CUDA_ARCH__ >= 900
  cudaGridDependencySynchronize();
#endif
  const int64_t n = ranges(place.total, blocks);
  for (int64_t segment = blockIdx.y; segment < static_cast<int64_t>(c.heads) * w.blocks; segment += gridDim.y) {
    const int64_t u0 = place.before + segment * w.tiles, u1 = u0 + w.tiles;
    const int64_t c0 = range_of(place.total, u0, n), c1 = range_of(place.total, u1 - 1, n);
    if (c0 == c1) continue;
    const int head = static_cast<int>(segment / w.blocks), row0 = static_cast<int>(segment % w.blocks) * kRows;
    const float* base = static_cast<const float*>(a.workspace);
    for (int i = threadIdx.x; i < kRows * kDim; i += kWarps * 32) {
      const int r = i / kDim, d = i - r * kDim;
      if (row0 + r >= w.q.rows * line.shared) continue;
      float m = -INFINITY, l = 0.0F, v = 0.0F;
      for (int64_t k = c0; k <= c1; ++k) {
        // Where the segment starts, it is the block's last; elsewhere its first.
        const float* p = base + (2 * k + (range_start(place.total, k, n) <= u0 ? 1 : 0)) * partial_floats(kRows, kDim);
        const float pm = p[kRows * kDim + 2 * r], pl = p[kRows * kDim + 2 * r + 1];
        const float next = fmaxf(m, pm);
        const float f0 = fade_to(m, next), f1 = fade_to(pm, next);
        l = l * f0 + pl * f1;
        v = v * f0 + p[i] * f1;
        m = next;
      }
      const int64_t row = (w.q.row0 + (row0 + r) / line.shared) * a.heads + head * line.shared + (row0 + r) % line.shared;
      static_cast<T*>(a.out)[row * kDim + d] = from_f32<T>(l == 0.0F ? 0.0F : v / l);
      if (a.lse && d == 0) a.lse[row] = log_sum(m, l);
    }
  }
}

struct Shape {
  int tiles;        // column tiles of 8 rows
  int64_t blocks;   // blocks of the main kernel
};
constexpr int kResident = 148 * 4;

Shape shape_of(const Kv4View& c, const Kv4Attend& a) {
  const int shared = a.heads / c.heads;
  const int64_t rows = static_cast<int64_t>(a.max_rows) * shared;
  Shape s;
  s.tiles = rows > 8 && c.dim < 256 ? 2 : 1;
  const int64_t most = static_cast<int64_t>(a.max_pages) << c.page_shift;
  const int64_t units = std::max<int64_t>(1, (most + kTile - 1) / kTile) * a.batch * c.heads *
                        ((rows + 8 * s.tiles - 1) / (8 * s.tiles));
  s.blocks = std::max<int64_t>(1, std::min<int64_t>(kResident, units));
  return s;
}

template <class T, int kDim, int kTiles>
void launch_shape(const Kv4View& c, const Kv4Attend& a, const Shape& s, cudaStream_t stream) {
  const Line line{c.heads, a.heads / c.heads, 8 * kTiles, c.page_shift};
  kv4_attend_kernel<T, kDim, kTiles><<<static_cast<unsigned>(s.blocks), kWarps * 32, 0, stream>>>(c, a, line);
  count_launch();
  check(cudaGetLastError(), "launch cache attention kernel");
  if ((static_cast<int64_t>(a.max_pages) << c.page_shift) <= kTile) return;  // no segment can be cut
  const int64_t segments = c.heads * ((static_cast<int64_t>(a.max_rows) * line.shared + line.block_rows - 1) / line.block_rows);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch), static_cast<unsigned>(std::min<int64_t>(segments, 65535)));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  check(cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, kDim, kTiles>, c, a, line, s.blocks), "launch cache attention join kernel");
  count_launch();
}

template <class T>
void launch_typed(const Kv4View& c, const Kv4Attend& a, const Shape& s, cudaStream_t stream) {
  if (c.dim == 64) {
    if (s.tiles == 1) launch_shape<T, 64, 1>(c, a, s, stream);
    else launch_shape<T, 64, 2>(c, a, s, stream);
  } else if (c.dim == 128) {
    if (s.tiles == 1) launch_shape<T, 128, 1>(c, a, s, stream);
    else launch_shape<T, 128, 2>(c, a, s, stream);
  } else {
    launch_shape<T, 256, 1>(c, a, s, stream);
  }
}

}  // namespace

size_t kv4_attend_workspace_bytes(const Kv4View& c, const Kv4Attend& a) {
  if (a.rows <= 0 || a.batch <= 0 || a.max_rows <= 0) return 0;
  if ((static_cast<int64_t>(a.max_pages) << c.page_shift) <= kTile) return 0;
  const Shape s = shape_of(c, a);
  return sizeof(float) * 2 * static_cast<size_t>(s.blocks) * partial_floats(8 * s.tiles, c.dim);
}

void launch_kv4_attend(const Kv4View& c, const Kv4Attend& a, cudaStream_t stream) {
  if (a.rows <= 0 || a.batch <= 0 || a.max_rows <= 0) return;
  const Shape s = shape_of(c, a);
  if (a.type == kElemF16) launch_typed<__half>(c, a, s, stream);
  else launch_typed<__nv_bfloat16>(c, a, s, stream);
}

}  // namespace msb
