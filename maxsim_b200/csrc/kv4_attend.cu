// Attention over the 4-bit key/value cache.
//
// Row (query token i of sequence b, query head h) sees cached tokens j <= pos (causal) and
// j > pos - window, pos = length - rows + i.  With s_j = scale * ks_j * <q, kc_j>, its output is
// sum_j e^(s_j - m) vs_j vc_j / sum_j e^(s_j - m) in one pass with a running reference m, sums in fp32; a row
// that sees nothing writes zeros and a log-sum-exp of -inf.
//
// kv4_attend_kernel: few rows a sequence (decode, drafted tokens).
//   Bound: the codes' bytes, D + 8 per token and head; then latency, a warp's chain a step (unpacking, products, maximum,
//   vote, exponentials, products): of 16 warps an SM it leaves 57% of the issue slots and of the memory's rate used.
//   Products.  m16n8k16 fp16 products with the tokens as the 16-row operand: S^T = K Q^T, O^T = V^T P^T, so
//   8 query rows (the heads that share a key/value head, times the query tokens) fill a column tile instead
//   of half a row tile.  tcgen05 wants 128 rows of queries, which decode has not.
//   Loads.  A warp takes steps of 32 tokens through a ring of its own in shared memory, three steps deep, filled by
//   asynchronous copies: no barrier between warps, and the bytes on their way hold no registers.  A 16-token tile lies
//   in one page (pages are powers of two >= 16), so a tile has one page lookup.
//   Operands.  The order of the summed index is free, so lane (g, t) = (lane / 4, lane % 4) reads D / 4 consecutive
//   dimensions of key tokens g and g + 8 (16 bytes at D = 128), and D / 8 consecutive dimensions of value tokens 2t,
//   2t + 1, 2t + 8, 2t + 9; probabilities become operands by an 8 x 8 transpose in registers.
//   Unpacking.  Nibbles i and i + 4 of a word are an fp16 pair in one logic operation: 1032 + code where they lie in
//   a half's last bits, 72 + code where four above; a subtraction makes them exact codes.  Keys keep the 72:
//   accumulators start at -72 sum(q) of those dimensions, exact products that cancel in fp32.  Values subtract
//   both (their sum over all tokens would lose digits to them).  (As fp16 subnormals codes would need neither, but the
//   products then lost 6 to 10 bits.)
//   Queries are fp16 after a power of two per row that puts their maximum in [2^10, 2^11): exact for fp16 inputs
//   down to 2^-34 of the row's maximum, and so for bf16 ones, up to their largest.  Probabilities are fp16 (11 bits): they enter one sum
//   that is rounded to the output's type, of as many bits or fewer.
//   Reference.  Probabilities carry the values' scales, p_j vs_j, so the running reference is the maximum of
//   s_j + log2 vs_j less 8: the largest p_j vs_j is about 2^8 whatever the scales are, and those 2^-22 of it are
//   normal in fp16.  Vectors of zeros are left out of it (zero_codes); keep_sums_finite has what holds the fp32 sum of
//   the p_j.
//   Work split.  The 128-token units of all (sequence, head, row block) segments form one line, cut into equal
//   ranges, one per resident block, from the lengths on the device: no plan, no host copy, no imbalance.
//   A segment cut by a range's end leaves partial sums in the workspace (at most two per block), which
//   kv4_join_kernel adds in a fixed order; it is launched early (programmatic dependent launch).
//   Short contexts (shape_of has the rule) take a cluster of 2 to 8 blocks a segment instead, whose parts are
//   joined over distributed shared memory: one launch.
//   Measured on the device, D = 128, 8 heads, 4 query heads each: 64 sequences of 4,096 tokens 77 us (3.7 TB/s of
//   codes, 57% of a copy's rate), 2 of 115,000 66 us (3.8 TB/s), 1 of 16,384 17 us, 1 of 1,030 6.9 us; of the first 4 to
//   5 us are the join and both launches' ends.  D = 256: the first 134 us (4.1 TB/s).
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <climits>

#include "quant4.cuh"

namespace msb {
bool kv4_chunk_supported(const Kv4View&);
void launch_kv4_chunk(const Kv4View&, const Kv4Attend&, cudaStream_t);

namespace {

constexpr int kWarps = 4;
constexpr int kStep = 32;              // tokens a warp takes at a time
constexpr int kTile = kWarps * kStep;  // tokens of one unit of the work line
constexpr int kStages = 3;             // steps in a warp's ring: one worked on, two on their way
constexpr float kLift = 8.0F;          // references lie 2^8 below the maximum: probabilities of 2^-22 are normal in fp16

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
// kWords consecutive words of shared memory (aligned to their size or to 16 bytes).
template <int kWords>
__device__ __forceinline__ void load_words(uint32_t (&r)[kWords], const unsigned char* p) {
  if constexpr (kWords == 1) {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (kWords == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r[0] = v.x, r[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      r[i] = v.x, r[i + 1] = v.y, r[i + 2] = v.z, r[i + 3] = v.w;
    }
  }
}

// Nibbles kI and kI + 4 of a word as an fp16 pair: 1032 + code (kI even) or 72 + code (kI odd), the nibbles in
// the last bits of 1024's mantissa or four above the last of 64's.
template <int kI>
__device__ __forceinline__ uint32_t codes_raised(uint32_t w) {
  constexpr uint32_t kMask = kI & 1 ? 0x00f000f0u : 0x000f000fu, kFlip = kI & 1 ? 0x54805480u : 0x64086408u;
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(kI < 2 ? w : w >> 8), "n"(kMask), "r"(kFlip));  // (a & b) ^ c
  return r;
}
template <int kI>
__device__ __forceinline__ uint32_t codes_exact(uint32_t w) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(codes_raised<kI>(w)), "r"(kI & 1 ? 0x54805480u : 0x64086408u));
  return r;
}
// Key codes: the 72 of odd nibbles stays, and the accumulators start at -72 times the sum of their queries.
template <int kI>
__device__ __forceinline__ uint32_t codes_key(uint32_t w) {
  return kI & 1 ? codes_raised<kI>(w) : codes_exact<kI>(w);
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Consecutive elements from anywhere.
template <int kRaw, class T>
__device__ __noinline__ void load_scattered(uint4 (&raw)[kRaw], const T* p) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(kRaw * 16 / sizeof(T)); ++i) reinterpret_cast<T*>(raw)[i] = p[i];
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float log_sum(float m, float l) {
  return l == 0.0F ? -INFINITY : (m - kLift + __log2f(l)) * 0.693147181F;
}

// The work line: units of kTile tokens of every (sequence, key/value head, row block).
struct Line {
  int heads;        // of the cache
  int shared;       // query heads per cache head
  int block_rows;   // rows of a row block
  int page_shift;
  int aligned;      // query rows of every head start on 16 bytes
  int most_blocks;  // row blocks of the largest sequence
};
constexpr int kMostCluster = 8;
struct SequenceWork {
  Kv4Sequence q;
  int begin;        // first token that a row may see, down to a multiple of kStep
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
  if (a.window > 0) w.begin = max(0, max(0, w.q.pos0) - a.window + 1) & ~(kStep - 1);
  // A sequence of no tokens keeps one empty unit: its rows are written as zeros.
  w.tiles = max(1, (w.q.length - w.begin + kTile - 1) / kTile);
  w.blocks = (w.q.rows * l.shared + l.block_rows - 1) / l.block_rows;
  return w;
}

// The workspace: where each sequence starts on the line ([batch + 1], the last is the line's end), then the blocks'
// partial sums.
__host__ __device__ __forceinline__ size_t starts_bytes(int64_t batch) {
  return (static_cast<size_t>(batch + 1) * sizeof(int64_t) + 127) & ~static_cast<size_t>(127);
}
__device__ __forceinline__ float* line_parts(const Kv4Attend& a) {
  return reinterpret_cast<float*>(static_cast<char*>(a.workspace) + starts_bytes(a.batch));
}

// Units of all sequences, the sequence that holds unit `first(total)` and the units before it, by all threads of
// the block, as many sequences at a time as it has threads.  The first block writes the sequences' starts where a
// join follows (else there is no workspace to write to).
struct Place {
  int64_t total;
  int64_t before;
  int sequence;
};
// For 32 sequences and fewer each warp finds them by itself: units up to and of sequence `lane`.
constexpr int kWarpBatch = 32;
__device__ __forceinline__ void warp_line(const Kv4Attend& a, const Line& l, int64_t& before, int64_t& mine, int64_t& total) {
  const int lane = threadIdx.x & 31;
  mine = lane < a.batch ? sequence_work(a, l, lane).units(l) : 0;
  int64_t upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += o;
  }
  before = upto - mine;
  total = __shfl_sync(0xFFFFFFFFu, upto, 31);
}
template <class F>
__device__ __forceinline__ Place find_place(const Kv4Attend& a, const Line& l, F first, int64_t* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (a.batch <= kWarpBatch) {
    int64_t before, mine, total;
    warp_line(a, l, before, mine, total);
    const int64_t target = first(total);
    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, target >= before && target < before + mine);
    const int at = hit ? __ffs(hit) - 1 : 0;
    return Place{total, __shfl_sync(0xFFFFFFFFu, before, at), hit ? at : a.batch};
  }
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
  Place p{total, 0, a.batch};
  const int64_t target = first(total);
  const bool writes = blockIdx.x == 0 && a.workspace != nullptr;
  int64_t* starts = static_cast<int64_t*>(a.workspace);
  if (writes && threadIdx.x == 0) starts[a.batch] = total;
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
    if (writes && b0 + threadIdx.x < a.batch) starts[b0 + threadIdx.x] = before;
    if (target >= before && target < before + mine) {
      scratch[kWarps] = before;
      scratch[kWarps + 1] = b0 + threadIdx.x;
    }
    __syncthreads();
    if (scratch[kWarps] >= 0) {
      p.before = scratch[kWarps];
      p.sequence = static_cast<int>(scratch[kWarps + 1]);
      if (!writes) break;
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

// Resident blocks per SM that the registers are held to (128 threads, 65,536 registers).
__host__ __device__ constexpr int resident_blocks(int dim, int tiles) {
  return dim == 256 ? 2 : dim == 128 ? (tiles == 1 ? 4 : 3) : (tiles == 1 ? 5 : 4);
}

// The warps' rings: codes of keys and values and both scales of kStages steps.
__host__ __device__ constexpr int ring_bytes(int dim) { return kWarps * kStages * (kStep * dim + 2 * kStep * 4); }

// kCluster: instead of the line, a cluster of blocks has each segment (sequence, head, row block) and adds its parts
// over distributed shared memory.
template <class T, int kDim, int kTiles, bool kCluster>
__global__ void __launch_bounds__(kWarps * 32, resident_blocks(kDim, kTiles)) kv4_attend_kernel(Kv4View c, Kv4Attend a, Line line) {
  constexpr int kRows = 8 * kTiles;      // rows of a row block
  constexpr int kKeyWords = kDim / 32;   // of one token, per lane
  constexpr int kValueWords = kDim / 64;
  constexpr int kOut = kDim / 16;        // 16-dimension tiles of the output
  constexpr int kPitch = kDim + 4;                  // floats between rows of the warps' sums
  constexpr int kCodeBytes = kStep * kDim / 2;      // one step's keys, or values
  constexpr int kStageBytes = 2 * kCodeBytes + 2 * kStep * 4;
  extern __shared__ __align__(128) unsigned char ring[];
  float(*merge)[kRows * kPitch] = reinterpret_cast<float(*)[kRows * kPitch]>(ring);  // after the last step
  __shared__ float stats[kWarps][2][kRows];
  __shared__ int64_t scratch[kWarps + 2];
  __shared__ float2 part_stats[kRows];   // of the block, for its cluster
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;

  const int64_t block = blockIdx.x;
  int64_t unit = 0, unit_end = 1, before = 0;
  int b = 0;
  SequenceWork w{};
  uint32_t cluster_segment = 0, cluster_rank = 0, cluster_size = 1;
  if constexpr (kCluster) {
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    cluster_rank = cluster.block_rank();
    cluster_size = cluster.num_blocks();
    const uint32_t here = blockIdx.x / cluster_size;
    b = here / (line.heads * line.most_blocks);
    cluster_segment = here - b * (line.heads * line.most_blocks);
    w = sequence_work(a, line, b);
    if (static_cast<int>(cluster_segment % line.most_blocks) >= w.blocks) unit_end = 0;  // nothing for the whole cluster
  } else {
    const Place place = find_place(
        a, line, [&](int64_t total) { return range_start(total, block, ranges(total, gridDim.x)); }, scratch);
    const int64_t n = ranges(place.total, gridDim.x);
#if __CUDA_ARCH__ >= 900
    cudaTriggerProgrammaticLaunchCompletion();
#endif
    // Without a join, which has time for it, the rows left over are filled here.
    if (a.fill && a.workspace == nullptr) {
      for (int s = blockIdx.x; s < a.batch; s += gridDim.x)
        kv4_fill_rows<T>(a, kDim, s, kv4_sequence(a, c.page_shift, s), 0, 1, threadIdx.x, kWarps * 32);
    }
    if (block >= n) return;
    unit = range_start(place.total, block, n);
    unit_end = range_start(place.total, block + 1, n);
    before = place.before;
    b = place.sequence;
    if (unit < unit_end) w = sequence_work(a, line, b);
  }

  while (unit < unit_end) {
    // The segment (head, row block) that holds `unit`, and this block's part of it.
    int head, row0, tile0, tile1;
    if constexpr (kCluster) {
      head = cluster_segment / line.most_blocks;
      row0 = (cluster_segment - head * line.most_blocks) * kRows;
      tile0 = static_cast<int>(static_cast<int64_t>(w.tiles) * cluster_rank / cluster_size);
      tile1 = static_cast<int>(static_cast<int64_t>(w.tiles) * (cluster_rank + 1) / cluster_size);
    } else {
      while (unit >= before + w.units(line)) {
        before += w.units(line);
        w = sequence_work(a, line, ++b);
      }
      const int64_t inside = unit - before;
      const int64_t segment = inside / w.tiles;
      tile0 = static_cast<int>(inside - segment * w.tiles);
      tile1 = static_cast<int>(min(static_cast<int64_t>(w.tiles), tile0 + (unit_end - unit)));
      head = static_cast<int>(segment / w.blocks);
      row0 = static_cast<int>(segment % w.blocks) * kRows;
    }
    const int all_rows = w.q.rows * line.shared;

    // Rows: which tokens they see; lane (g, t) loads row g of each column tile, dimensions t * kDim / 4 and on.
    constexpr int kRaw = kKeyWords * 8 * sizeof(T) / 16;
    uint4 raw[kTiles][kRaw];
    int last[kTiles][2], first[kTiles][2];  // tokens that columns 2t, 2t + 1 see: first <= j <= last
    int every_last = INT_MAX, every_first = 0, any_last = -1, any_first = INT_MAX;
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      const int r = row0 + nt * 8 + g;
#pragma unroll
      for (int i = 0; i < kRaw; ++i) raw[nt][i] = make_uint4(0, 0, 0, 0);
      if (r < all_rows) {
        const T* p = static_cast<const T*>(a.query) + (w.q.row0 + r / line.shared) * a.q_row_stride +
                     static_cast<int64_t>(head * line.shared + r % line.shared) * a.q_head_stride + t * (kDim / 4);
        if (line.aligned) {
#pragma unroll
          for (int i = 0; i < kRaw; ++i) raw[nt][i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
        } else {
          load_scattered(raw[nt], p);
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int rr = row0 + nt * 8 + 2 * t + k;
        first[nt][k] = 0;
        last[nt][k] = INT_MAX;  // rows past the block are not written: no reason to mask for them
        if (rr < all_rows) {
          const int pos = w.q.pos0 + rr / line.shared;
          last[nt][k] = a.causal ? pos : w.q.length - 1;
          first[nt][k] = a.window > 0 ? max(0, max(0, pos) - a.window + 1) : 0;
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

    // This warp's steps of 32 tokens, those that some row sees.
    const int upto = min(w.begin + tile1 * kTile, any_last + 1);
    int j0 = w.begin + tile0 * kTile + warp * kStep;
    if (any_first > j0) j0 += (any_first - j0) / kTile * kTile;

    const int32_t* pages = a.page_table + b * a.table_stride;
    const bool two_pages = c.page_shift == 4;  // else 32 aligned tokens lie in one
    const int page_mask = (1 << c.page_shift) - 1;
    unsigned char* const stages = ring + warp * (kStages * kStageBytes);
    const uint32_t lane_stage = static_cast<uint32_t>(__cvta_generic_to_shared(stages)) + lane * 16;
    const unsigned char* lane_codes[2] = {c.codes[0] + lane * 16, c.codes[1] + lane * 16};
    const float* lane_scales = (lane & 8 ? c.scales[1] : c.scales[0]) + (lane & 3) * 4;
    int next_page[2];  // the pages of the next step to be copied, -1 past the last token seen
    uint32_t seen_queue = 0;  // two bits a step, the oldest lowest: its 16-token tiles lie on pages of the cache
    auto ask_pages = [&](int j) {
      next_page[0] = j < upto ? __ldg(pages + (j >> c.page_shift)) : -1;
      next_page[1] = !two_pages ? next_page[0] : j + 16 < upto ? __ldg(pages + ((j + 16) >> c.page_shift)) : -1;
    };
    // Copies the step at j into a stage; tiles without a page copy the cache's first vectors.
    auto copy_step = [&](int j, int stage, int slot) {
      if (j < upto) {
        const uint32_t dst = lane_stage + stage * kStageBytes;
        auto tile_of = [&](int i) -> int64_t {
          if (static_cast<uint32_t>(next_page[i]) >= static_cast<uint32_t>(c.num_pages)) return 0;
          seen_queue |= (!two_pages ? 3u : 1u << i) << (2 * slot);
          return (static_cast<int64_t>(static_cast<uint32_t>(next_page[i]) * c.heads + head) << c.page_shift) +
                 ((j + 16 * i) & page_mask);
        };
        const int64_t tile = tile_of(0);
        const uint8_t* src[2] = {lane_codes[0] + tile * (kDim / 2), lane_codes[1] + tile * (kDim / 2)};
        if (!two_pages) {
#pragma unroll
          for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int k = 0; k < kDim / 32; ++k) copy16(dst + which * kCodeBytes + k * 512, src[which] + k * 512);
          if (lane < 16) copy16(dst + 2 * kCodeBytes, lane_scales + tile + ((lane >> 2) & 1) * 16);
        } else {
          const int64_t other = tile_of(1), step = (other - tile) * (kDim / 2);
#pragma unroll
          for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int k = 0; k < kDim / 64; ++k) {
              copy16(dst + which * kCodeBytes + k * 512, src[which] + k * 512);
              copy16(dst + which * kCodeBytes + kCodeBytes / 2 + k * 512, src[which] + step + k * 512);
            }
          if (lane < 16) copy16(dst + 2 * kCodeBytes, lane_scales + ((lane >> 2) & 1 ? other : tile));
        }
      }
      copies_commit();
    };
    ask_pages(j0);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      copy_step(j0 + i * kTile, i, i);
      ask_pages(j0 + (i + 1) * kTile);
    }
    // Queries, while the first copies are on their way.
    uint32_t q[kTiles][2 * kKeyWords][2];
    float2 lift[kTiles];     // what columns 2t, 2t + 1 start at (codes_key)
    float2 factor[kTiles];   // scale * log2(e) * the row's power of two
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      const T* const x = reinterpret_cast<const T*>(raw[nt]);
      float top = 0.0F;
#pragma unroll
      for (int d = 0; d < kKeyWords * 8; ++d) top = fmaxf(top, fabsf(to_f32(x[d])));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      const int e = max(-110, min(127, static_cast<int>(__float_as_uint(top) >> 23) - 127));
      const float down = __uint_as_float(static_cast<uint32_t>(127 + 10 - e) << 23);
      float sum[4] = {0.0F, 0.0F, 0.0F, 0.0F};
#pragma unroll
      for (int word = 0; word < kKeyWords; ++word) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          q[nt][2 * word + (i >> 1)][i & 1] = pack_half2(to_f32(x[8 * word + i]) * down, to_f32(x[8 * word + 4 + i]) * down);
        // -72 (0xD480) times the queries of odd nibbles, summed where the scores will be
        mma(sum, 0u, 0u, 0xD480D480u, 0xD480D480u, q[nt][2 * word][0], q[nt][2 * word][1]);
        mma(sum, 0u, 0u, 0xD480D480u, 0xD480D480u, q[nt][2 * word + 1][0], q[nt][2 * word + 1][1]);
      }
      const float up = a.scale * 1.44269504F * __uint_as_float(static_cast<uint32_t>(127 - 10 + e) << 23);
      lift[nt] = make_float2(sum[0], sum[1]);
      // from the lanes that hold rows 2t, 2t + 1 to the columns' lanes
      factor[nt] = make_float2(__shfl_sync(0xFFFFFFFFu, up, 8 * t), __shfl_sync(0xFFFFFFFFu, up, 8 * t + 4));
    }

    float o[kOut][kTiles][4];
    float top[kTiles][2];
    float2 sum[kTiles];
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < kOut; ++i) o[i][nt][k] = 0.0F;
      top[nt][0] = top[nt][1] = -INFINITY;
      sum[nt] = make_float2(0.0F, 0.0F);
    }

    int stage = 0;
    for (; j0 < upto; j0 += kTile) {
      copies_wait<kStages - 2>();
      __syncwarp();
      // Every lane has left the stage of the step before: the copies two steps ahead go there.
      const unsigned char* here = stages + stage * kStageBytes;
      const uint32_t seen = seen_queue & 3u;
      seen_queue >>= 2;
      copy_step(j0 + (kStages - 1) * kTile, stage == 0 ? kStages - 1 : stage - 1, kStages - 2);
      ask_pages(j0 + kStages * kTile);
      stage = stage == kStages - 1 ? 0 : stage + 1;
      // Scores of the step: s[i][nt][0] of token g, [1] of token g + 8, columns 2t, 2t + 1.
      float2 s[2][kTiles][2];
      float2 vs[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float d[kTiles][4];
#pragma unroll
        for (int nt = 0; nt < kTiles; ++nt) {
          d[nt][0] = d[nt][2] = lift[nt].x;
          d[nt][1] = d[nt][3] = lift[nt].y;
        }
        uint32_t key[2][kKeyWords];
#pragma unroll
        for (int k = 0; k < 2; ++k) load_words(key[k], here + (16 * i + g + 8 * k) * (kDim / 2) + t * (kDim / 8));
#pragma unroll
        for (int word = 0; word < kKeyWords; ++word) {
          const uint32_t x = key[0][word], y = key[1][word];
          const uint32_t x0 = codes_key<0>(x), x1 = codes_key<1>(x), x2 = codes_key<2>(x), x3 = codes_key<3>(x);
          const uint32_t y0 = codes_key<0>(y), y1 = codes_key<1>(y), y2 = codes_key<2>(y), y3 = codes_key<3>(y);
#pragma unroll
          for (int nt = 0; nt < kTiles; ++nt) {
            mma(d[nt], x0, y0, x1, y1, q[nt][2 * word][0], q[nt][2 * word][1]);
            mma(d[nt], x2, y2, x3, y3, q[nt][2 * word + 1][0], q[nt][2 * word + 1][1]);
          }
        }
        const float* scales = reinterpret_cast<const float*>(here + 2 * kCodeBytes) + 16 * i + g;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float ks = scales[8 * k], v = scales[kStep + 8 * k];
          vs[i][k] = make_float2(v, v);
#pragma unroll
          for (int nt = 0; nt < kTiles; ++nt)
            s[i][nt][k] = __fmul2_rn(make_float2(d[nt][2 * k], d[nt][2 * k + 1]), __fmul2_rn(factor[nt], make_float2(ks, ks)));
        }
      }
      const bool one = vs[0][0].x == 1.0F || vs[0][1].x == 1.0F || vs[1][0].x == 1.0F || vs[1][1].x == 1.0F;
      const bool masked = seen != 3u || j0 < every_first || j0 + kStep - 1 > every_last || one;
      if (masked) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (vs[i][k].x == 1.0F && zero_codes<kDim>(here + kCodeBytes + (16 * i + g + 8 * k) * (kDim / 2)))
              vs[i][k] = make_float2(0.0F, 0.0F);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int j = j0 + 16 * i + g + 8 * k;
              const bool off = !((seen >> i) & 1u);
              if (off || j < first[nt][0] || j > last[nt][0]) s[i][nt][k].x = -INFINITY;
              if (off || j < first[nt][1] || j > last[nt][1]) s[i][nt][k].y = -INFINITY;
            }
      }
      float2 raise[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float e = scale_exponent(vs[i][k].x, a.least_exponent, most_exponent(kLift));
          raise[i][k] = make_float2(e, e);
        }
      bool moved = false;
      float2 fade[kTiles], ref[kTiles];
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt) {
        const float2 v0 = __fadd2_rn(s[0][nt][0], raise[0][0]), v1 = __fadd2_rn(s[0][nt][1], raise[0][1]);
        const float2 v2 = __fadd2_rn(s[1][nt][0], raise[1][0]), v3 = __fadd2_rn(s[1][nt][1], raise[1][1]);
        float2 m = make_float2(fmax3(v0.x, v1.x, fmaxf(v2.x, v3.x)), fmax3(v0.y, v1.y, fmaxf(v2.y, v3.y)));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          const float2 other = make_float2(__shfl_xor_sync(0xFFFFFFFFu, m.x, d), __shfl_xor_sync(0xFFFFFFFFu, m.y, d));
          m.x = d < 16 ? fmaxf(m.x, other.x) : fmax3(m.x, other.x, top[nt][0]);
          m.y = d < 16 ? fmaxf(m.y, other.y) : fmax3(m.y, other.y, top[nt][1]);
        }
        moved = moved || m.x > top[nt][0] || m.y > top[nt][1];
        ref[nt] = make_float2(m.x == -INFINITY ? 0.0F : kLift - m.x, m.y == -INFINITY ? 0.0F : kLift - m.y);
        fade[nt] = m;
      }
      if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
        for (int nt = 0; nt < kTiles; ++nt) {
          const float2 m = fade[nt], f = make_float2(fade_to(top[nt][0], m.x), fade_to(top[nt][1], m.y));
          top[nt][0] = m.x;
          top[nt][1] = m.y;
          sum[nt] = __fmul2_rn(sum[nt], f);
#pragma unroll
          for (int i = 0; i < kOut; ++i) {
            const float2 lo = __fmul2_rn(make_float2(o[i][nt][0], o[i][nt][1]), f);
            const float2 hi = __fmul2_rn(make_float2(o[i][nt][2], o[i][nt][3]), f);
            o[i][nt][0] = lo.x, o[i][nt][1] = lo.y, o[i][nt][2] = hi.x, o[i][nt][3] = hi.y;
          }
        }
      }
      uint32_t p[2][kTiles][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 x = __fadd2_rn(s[i][nt][k], ref[nt]);
            const float2 pr = make_float2(exp2_fast(x.x), exp2_fast(x.y));
            sum[nt] = __fadd2_rn(sum[nt], pr);
            float2 pv = __fmul2_rn(pr, vs[i][k]);
            if (masked) {  // an unseen token's scale may be NaN or infinite
              if (s[i][nt][k].x == -INFINITY) pv.x = 0.0F;
              if (s[i][nt][k].y == -INFINITY) pv.y = 0.0F;
            }
            p[i][nt][k] = transpose8x8(pack_half2(pv.x, pv.y));
          }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t value[4][kValueWords];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          load_words(value[k], here + kCodeBytes + (16 * i + 2 * t + (k & 1) + 8 * (k >> 1)) * (kDim / 2) + g * (kDim / 16));
#pragma unroll
        for (int word = 0; word < kValueWords; ++word) {
          const uint32_t va = value[0][word], vb = value[1][word], vc = value[2][word], vd = value[3][word];
          const uint32_t x0 = __byte_perm(va, vb, 0x5410), y0 = __byte_perm(va, vb, 0x7632);
          const uint32_t x1 = __byte_perm(vc, vd, 0x5410), y1 = __byte_perm(vc, vd, 0x7632);
#pragma unroll
          for (int nt = 0; nt < kTiles; ++nt) {
            mma(o[4 * word][nt], codes_exact<0>(x0), codes_exact<0>(y0), codes_exact<0>(x1), codes_exact<0>(y1), p[i][nt][0], p[i][nt][1]);
            mma(o[4 * word + 1][nt], codes_exact<1>(x0), codes_exact<1>(y0), codes_exact<1>(x1), codes_exact<1>(y1), p[i][nt][0], p[i][nt][1]);
            mma(o[4 * word + 2][nt], codes_exact<2>(x0), codes_exact<2>(y0), codes_exact<2>(x1), codes_exact<2>(y1), p[i][nt][0], p[i][nt][1]);
            mma(o[4 * word + 3][nt], codes_exact<3>(x0), codes_exact<3>(y0), codes_exact<3>(x1), codes_exact<3>(y1), p[i][nt][0], p[i][nt][1]);
          }
        }
      }
    }
    copies_wait<0>();

    // The warps' parts, joined in the order of the warps.
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float l = k ? sum[nt].y : sum[nt].x;
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 4);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 8);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 16);
        const int r = nt * 8 + 2 * t + k;
        if (g == 0) {
          stats[warp][0][r] = top[nt][k];
          stats[warp][1][r] = l;
        }
        // Lane g holds dimensions g * kDim / 8 and on: tile 4 word + nib is 8 word + nib, and + 4.
#pragma unroll
        for (int word = 0; word < kValueWords; ++word)
#pragma unroll
          for (int hi = 0; hi < 2; ++hi)
            *reinterpret_cast<float4*>(&merge[warp][r * kPitch + g * (kDim / 8) + 8 * word + 4 * hi]) =
                make_float4(o[4 * word][nt][2 * hi + k], o[4 * word + 1][nt][2 * hi + k], o[4 * word + 2][nt][2 * hi + k],
                            o[4 * word + 3][nt][2 * hi + k]);
      }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == w.tiles;
    float* partial = nullptr;
    if constexpr (!kCluster) partial = line_parts(a) + (2 * block + (tile0 == 0 ? 1 : 0)) * partial_floats(kRows, kDim);
    auto write_out = [&](int r, int d, float m, float l, const float4& v) {
      const float inv = l == 0.0F ? 0.0F : 1.0F / l;
      const int64_t row = (w.q.row0 + (row0 + r) / line.shared) * a.heads + head * line.shared + (row0 + r) % line.shared;
      T* out = static_cast<T*>(a.out) + row * kDim + d;
      out[0] = from_f32<T>(v.x * inv);
      out[1] = from_f32<T>(v.y * inv);
      out[2] = from_f32<T>(v.z * inv);
      out[3] = from_f32<T>(v.w * inv);
      if (a.lse && d == 0) a.lse[row] = log_sum(m, l);
    };
    for (int i = threadIdx.x; i < kRows * kDim / 4; i += kWarps * 32) {
      const int r = i / (kDim / 4), d = i % (kDim / 4) * 4;
      if (row0 + r >= all_rows) continue;
      float m = stats[0][0][r], l = 0.0F;
#pragma unroll
      for (int k = 1; k < kWarps; ++k) m = fmaxf(m, stats[k][0][r]);
      float4 v = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float f = fade_to(stats[k][0][r], m);
        const float4 x = *reinterpret_cast<const float4*>(&merge[k][r * kPitch + d]);
        l += f * stats[k][1][r];
        v.x += f * x.x;
        v.y += f * x.y;
        v.z += f * x.z;
        v.w += f * x.w;
      }
      if constexpr (kCluster) {
        *reinterpret_cast<float4*>(&merge[0][r * kPitch + d]) = v;  // only this thread reads that place
        if (d == 0) part_stats[r] = make_float2(m, l);
      } else if (whole) {
        write_out(r, d, m, l, v);
      } else {
        *reinterpret_cast<float4*>(partial + r * kDim + d) = v;
        if (d == 0) {
          partial[kRows * kDim + 2 * r] = m;
          partial[kRows * kDim + 2 * r + 1] = l;
        }
      }
    }
    if constexpr (kCluster) {
      // The blocks' parts, in the order of their ranks; each block writes its share of the rows' dimensions.
      const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
      cluster.sync();
      for (int i = cluster_rank * (kWarps * 32) + threadIdx.x; i < kRows * kDim / 4; i += cluster_size * (kWarps * 32)) {
        const int r = i / (kDim / 4), d = i % (kDim / 4) * 4;
        if (row0 + r >= all_rows) continue;
        float2 st[kMostCluster];
        float4 x[kMostCluster];
        float m = -INFINITY, l = 0.0F;
#pragma unroll
        for (int k = 0; k < kMostCluster; ++k) {
          st[k] = make_float2(-INFINITY, 0.0F);
          x[k] = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
          if (k < static_cast<int>(cluster_size)) {
            st[k] = *cluster.map_shared_rank(&part_stats[r], k);
            x[k] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(&merge[0][r * kPitch + d], k));
          }
          m = fmaxf(m, st[k].x);
        }
        float4 v = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
#pragma unroll
        for (int k = 0; k < kMostCluster; ++k) {
          const float f = fade_to(st[k].x, m);
          l += f * st[k].y;
          v.x += f * x[k].x;
          v.y += f * x[k].y;
          v.z += f * x[k].z;
          v.w += f * x[k].w;
        }
        write_out(r, d, m, l, v);
      }
      cluster.sync();  // before a block's shared memory goes
      unit = unit_end;
    } else {
      __syncthreads();
      unit += tile1 - tile0;
    }
  }
  if constexpr (kCluster) {
    // Last: ahead of the first loads it costs 0.1 us of 6.9.
    if (a.fill)
      kv4_fill_rows<T>(a, kDim, b, w.q, cluster_segment * cluster_size + cluster_rank, line.heads * line.most_blocks * cluster_size,
                       threadIdx.x, kWarps * 32);
  }
}

// Adds the partial sums of the segments that were cut.  A warp adds the parts of one output row, or, where
// segments have many parts, each of a block's kJoinWarps warps adds every kJoinWarps-th of one row's and the first
// adds the warps' sums: in either case in an order that the cut alone decides.
constexpr int kJoinWarps = 8;
template <class T, int kDim, int kTiles>
__global__ void __launch_bounds__(kJoinWarps * 32) kv4_join_kernel(Kv4View c, Kv4Attend a, Line line, int64_t blocks,
                                                                  int warps_per_row) {
  constexpr int kRows = 8 * kTiles, kPer = kDim / 32;
  __shared__ float sums[kJoinWarps][kDim + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x;
  const SequenceWork w = sequence_work(a, line, b);
  int64_t before = 0, total = 0;
  if (a.batch <= kWarpBatch) {
    int64_t mine;
    warp_line(a, line, before, mine, total);
    before = __shfl_sync(0xFFFFFFFFu, before, b);
  }
  if (a.fill) kv4_fill_rows<T>(a, kDim, b, w.q, blockIdx.y, gridDim.y, threadIdx.x, kJoinWarps * 32);
#if __CUDA_ARCH__ >= 900
  cudaGridDependencySynchronize();
#endif
  if (a.batch > kWarpBatch) {
    const int64_t* line_starts = reinterpret_cast<const int64_t*>(a.workspace);
    before = line_starts[b];
    total = line_starts[a.batch];
  }
  const int64_t n = ranges(total, blocks);
  const float* base = line_parts(a);
  const int rows_per_block = kJoinWarps / warps_per_row, group = warp % warps_per_row;
  const int64_t rows = static_cast<int64_t>(w.q.rows) * a.heads;
  for (int64_t i0 = static_cast<int64_t>(blockIdx.y) * rows_per_block; i0 < rows; i0 += static_cast<int64_t>(gridDim.y) * rows_per_block) {
    // Output row i is query row i / heads, head i % heads.
    const int64_t i = i0 + warp / warps_per_row;
    const bool mine = i < rows;
    const int row = static_cast<int>(mine ? i / a.heads : 0), q_head = static_cast<int>(mine ? i % a.heads : 0);
    const int r = row * line.shared + q_head % line.shared;
    const int64_t segment = static_cast<int64_t>(q_head / line.shared) * w.blocks + r / kRows;
    const int64_t u0 = before + segment * w.tiles, u1 = u0 + w.tiles;
    const int64_t c0 = range_of(total, u0, n), c1 = range_of(total, u1 - 1, n);
    float m = -INFINITY, l = 0.0F, v[kPer];
#pragma unroll
    for (int d = 0; d < kPer; ++d) v[d] = 0.0F;
    if (mine && c0 != c1) {
      // Part k of the segment: the last of the block where the segment starts, the first of the others.
      const float* first = base + (2 * c0 + 1) * partial_floats(kRows, kDim);
      const float* other = base + 2 * c0 * partial_floats(kRows, kDim);
      const int parts = static_cast<int>(c1 - c0) + 1, rr = r % kRows;
      for (int k0 = group; k0 < parts; k0 += 32 * warps_per_row) {
        // 32 parts at a time: lane k holds the k-th's reference and sum.
        const int k = k0 + lane * warps_per_row;
        const float* p = k == 0 ? first : other + 2 * static_cast<int64_t>(k) * partial_floats(kRows, kDim);
        float2 st = make_float2(-INFINITY, 0.0F);
        if (k < parts) st = *reinterpret_cast<const float2*>(p + kRows * kDim + 2 * rr);
        float next = st.x;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) next = fmaxf(next, __shfl_xor_sync(0xFFFFFFFFu, next, d));
        next = fmaxf(next, m);
        const float old = fade_to(m, next), f = fade_to(st.x, next);
        l *= old;
        m = next;
#pragma unroll
        for (int d = 0; d < kPer; ++d) v[d] *= old;
        const int here = min(32, (parts - k0 + warps_per_row - 1) / warps_per_row);
#pragma unroll 8
        for (int j = 0; j < here; ++j) {
          const int64_t at = k0 + static_cast<int64_t>(j) * warps_per_row;
          const float* x = (at == 0 ? first : other + 2 * at * partial_floats(kRows, kDim)) + rr * kDim + lane * kPer;
          const float fj = __shfl_sync(0xFFFFFFFFu, f, j);
          l += fj * __shfl_sync(0xFFFFFFFFu, st.y, j);
          float e[kPer];
          if constexpr (kPer == 2) {
            *reinterpret_cast<float2*>(e) = *reinterpret_cast<const float2*>(x);
          } else {
#pragma unroll
            for (int d = 0; d < kPer; d += 4) *reinterpret_cast<float4*>(e + d) = *reinterpret_cast<const float4*>(x + d);
          }
#pragma unroll
          for (int d = 0; d < kPer; ++d) v[d] += fj * e[d];
        }
      }
    }
    if (warps_per_row > 1) {
      __syncthreads();
#pragma unroll
      for (int d = 0; d < kPer; ++d) sums[warp][lane * kPer + d] = v[d];
      if (lane == 0) sums[warp][kDim] = m, sums[warp][kDim + 1] = l;
      __syncthreads();
      if (group != 0) continue;
      float top = m;
      for (int k = 1; k < warps_per_row; ++k) top = fmaxf(top, sums[warp + k][kDim]);
      const float f0 = fade_to(m, top);
      l *= f0;
#pragma unroll
      for (int d = 0; d < kPer; ++d) v[d] *= f0;
      for (int k = 1; k < warps_per_row; ++k) {
        const float f = fade_to(sums[warp + k][kDim], top);
        l += f * sums[warp + k][kDim + 1];
#pragma unroll
        for (int d = 0; d < kPer; ++d) v[d] += f * sums[warp + k][lane * kPer + d];
      }
      m = top;
    }
    if (mine && c0 != c1) {
      const float inv = l == 0.0F ? 0.0F : 1.0F / l;
      const int64_t at = (w.q.row0 + row) * a.heads + q_head;
      T* out = static_cast<T*>(a.out) + at * kDim + lane * kPer;
#pragma unroll
      for (int d = 0; d < kPer; ++d) out[d] = from_f32<T>(v[d] * inv);
      if (a.lse && lane == 0) a.lse[at] = log_sum(m, l);
    }
  }
}

struct Shape {
  int tiles;        // column tiles of 8 rows
  int64_t blocks;   // blocks of the main kernel
  int cluster;      // blocks to a segment, 0: the work line
  int row_blocks;   // of the largest sequence
};
int sm_count() {
  static std::atomic<int> known{0};
  int n = known.load(std::memory_order_relaxed);
  if (n == 0) {
    int dev = 0;
    check(cudaGetDevice(&dev), "get device");
    check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "SM count");
    known.store(n, std::memory_order_relaxed);
  }
  return n;
}

Shape shape_of(const Kv4View& c, const Kv4Attend& a) {
  const int shared = a.heads / c.heads;
  const int64_t rows = static_cast<int64_t>(a.max_rows) * shared;
  Shape s;
  s.tiles = rows > 8 && c.dim < 256 ? 2 : 1;
  const int64_t most = static_cast<int64_t>(a.max_pages) << c.page_shift;
  const int64_t units = std::max<int64_t>(1, (most + kTile - 1) / kTile) * a.batch * c.heads *
                        ((rows + 8 * s.tiles - 1) / (8 * s.tiles));
  const int64_t slots = sm_count() * resident_blocks(c.dim, s.tiles);
  s.blocks = std::max<int64_t>(1, std::min<int64_t>(slots, units));
  // Short contexts and few segments: a cluster to a segment, joined without a second kernel, where every block is
  // resident at once and walks four tiles at most.  (One sequence of 1,030 tokens, 8 heads: 9.6 us on the line, 6.9 us so; eight of
  // 2,048: 18.0 and 11.9 us.)
  const int64_t row_blocks = (rows + 8 * s.tiles - 1) / (8 * s.tiles), segments = row_blocks * a.batch * c.heads;
  int64_t seen = most;  // tokens of a segment, at most
  if (a.window > 0) seen = std::min<int64_t>(seen, static_cast<int64_t>(a.window) + a.max_rows + kStep);
  const int64_t tiles = (seen + kTile - 1) / kTile;
  s.cluster = 0;
  s.row_blocks = static_cast<int>(std::min<int64_t>(row_blocks, INT_MAX));
  for (int size = 2; size <= kMostCluster; size *= 2)
    if (size < 2 * tiles && tiles <= 4 * size && segments * size <= slots) s.cluster = size;
  return s;
}

// Whether the line may cut a segment: one of a single unit never is.
bool needs_join(const Kv4View& c, const Kv4Attend& a) { return (static_cast<int64_t>(a.max_pages) << c.page_shift) > kTile; }

template <class T, int kDim, int kTiles>
void launch_shape(const Kv4View& c, const Kv4Attend& given, const Shape& s, cudaStream_t stream) {
  Kv4Attend a = given;
  // What the call did not ask for (kv4_attend_workspace_bytes) is not its to write, whatever the caller passed.
  if (!needs_join(c, a)) a.workspace = nullptr;
  keep_sums_finite(a, c.page_shift, kLift);
  const uint64_t starts = reinterpret_cast<uintptr_t>(a.query) | static_cast<uint64_t>(a.q_row_stride) * sizeof(T) |
                          static_cast<uint64_t>(a.q_head_stride) * sizeof(T);
  const Line line{c.heads, a.heads / c.heads, 8 * kTiles, c.page_shift, (starts & 15) == 0, s.row_blocks};
  constexpr int kShared = ring_bytes(kDim);
  static_assert(kShared >= static_cast<int>(sizeof(float)) * kWarps * 8 * kTiles * (kDim + 4), "sums fit the ring");
  if (s.cluster > 0) {
    allow_dynamic_shared<kv4_attend_kernel<T, kDim, kTiles, true>>(kShared, "shared memory of the cache attention kernel");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(s.row_blocks) * a.batch * c.heads * s.cluster));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = kShared;
    cfg.stream = stream;
    cudaLaunchAttribute size{};
    size.id = cudaLaunchAttributeClusterDimension;
    size.val.clusterDim.x = static_cast<unsigned>(s.cluster);
    size.val.clusterDim.y = size.val.clusterDim.z = 1;
    cfg.attrs = &size;
    cfg.numAttrs = 1;
    check(cudaLaunchKernelEx(&cfg, kv4_attend_kernel<T, kDim, kTiles, true>, c, a, line), "launch cache attention kernel");
    count_launch();
    return;
  }
  allow_dynamic_shared<kv4_attend_kernel<T, kDim, kTiles, false>>(kShared, "shared memory of the cache attention kernel");
  kv4_attend_kernel<T, kDim, kTiles, false><<<static_cast<unsigned>(s.blocks), kWarps * 32, kShared, stream>>>(c, a, line);
  count_launch();
  check(cudaGetLastError(), "launch cache attention kernel");
  if (!needs_join(c, a)) return;
  const int64_t rows = static_cast<int64_t>(a.max_rows) * a.heads;
  const int64_t segments = c.heads * ((static_cast<int64_t>(a.max_rows) * line.shared + line.block_rows - 1) / line.block_rows);
  // Eight warps a row where a segment has 16 parts or more on average, each adding two or more.
  const int warps_per_row = s.blocks >= 16 * segments * a.batch ? kJoinWarps : 1;
  const int64_t blocks_y = (rows * warps_per_row + kJoinWarps - 1) / kJoinWarps;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch), static_cast<unsigned>(std::min<int64_t>(blocks_y, 65535)));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  check(cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, kDim, kTiles>, c, a, line, s.blocks, warps_per_row),
        "launch cache attention join kernel");
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

// Which kernel: this file's takes a time in proportion to the row blocks of 16, kv4_chunk.cu's to the waves of blocks
// of 256 rows over the SMs, whatever fills them.  Measured per 128 tokens: 6.6 ns a row block over the whole device,
// 2.8 us a wave (2.2 us with 128 rows or fewer) and 20 us, which the factors of 440 and 350 spread over contexts of some
// thousand tokens.  (4 sequences of 4,096 tokens, 8 heads: 63 and 81 us at 128 rows a head, 111 and 100 at 256; 32 of
// 2,000: 73 and 93 at 32, 125 and 93 at 64.)  Rows are those announced, for every sequence: what the device arrays hold
// is not known here, and a call that announces far more than there are gets the kernel for many.
bool many_rows(const Kv4View& c, const Kv4Attend& a) {
  if (!kv4_chunk_supported(c) || a.engine == 1) return false;
  if (a.engine == 2) return true;
  const int64_t rows = static_cast<int64_t>(a.max_rows) * (a.heads / c.heads);
  const int64_t heads = static_cast<int64_t>(a.batch) * c.heads, sms = sm_count();
  const int64_t waves = (heads * ((rows + 255) / 256) + sms - 1) / sms;
  return heads * ((rows + 15) / 16) >= waves * (rows > 128 ? 440 : 350);
}

}  // namespace

size_t kv4_attend_workspace_bytes(const Kv4View& c, const Kv4Attend& a) {
  if (a.rows <= 0 || a.batch <= 0 || a.max_rows <= 0 || many_rows(c, a) || !needs_join(c, a)) return 0;
  const Shape s = shape_of(c, a);
  if (s.cluster > 0) return 0;
  return starts_bytes(a.batch) + sizeof(float) * 2 * static_cast<size_t>(s.blocks) * partial_floats(8 * s.tiles, c.dim);
}

void launch_kv4_attend(const Kv4View& c, const Kv4Attend& a, cudaStream_t stream) {
  if (a.rows <= 0 || a.batch <= 0 || a.max_rows <= 0) return;
  if (many_rows(c, a)) {
    launch_kv4_chunk(c, a, stream);
    return;
  }
  const Shape s = shape_of(c, a);
  if (a.type == kElemF16) launch_typed<__half>(c, a, s, stream);
  else launch_typed<__nv_bfloat16>(c, a, s, stream);
}

}  // namespace msb
