// Attention of many query rows over the 4-bit key/value cache (prompt chunks), on the 5th-generation tensor cores.
//
// The operator and its formulas: kv4_attend.cu.  A block owns one sequence, one key/value head and 256 rows (query
// tokens times the query heads that share the head), and walks the 128-token tiles that its rows see.
//   Bound: the exponentials (16 a clock and SM) and the products (two of 128 x 128 x D per 128 rows), about equal at
//   D = 128; then instruction issue.
//   Products.  S = Q K^T from shared memory (tcgen05.mma, fp16, 128 x 128 x D, fp32 in tensor memory), O += P V with P
//   (fp16) read back from tensor memory over S.  The 256 rows are two tiles of 128: while one's softmax runs, the
//   other's products do.
//   Operands.  Four warps unpack keys and values, each code once per block, to exact fp16 integers in the
//   128-byte-swizzled layout of the products: keys as [token][dimension] (dimensions in the order of a word's nibble
//   pairs, queries alike), values as [dimension][token] - their nibbles are paired by tokens (byte permutes of two
//   tokens' words), so nothing is transposed.  Codes are loaded a tile ahead into registers.
//   Softmax.  Sixteen warps, eight to a row tile: a warp has 16 rows, a thread two of them and a quarter of their
//   columns, in blocks of 32 columns.  (With half the warps, a row to a thread: 206 us where this took 184.)
//   Scales of keys and values are fp32 factors of scores and probabilities (they would lose digits in fp16 operands);
//   the reference is the running maximum of s_j + log2(vs_j) (without vectors of zeros) as in kv4_attend.cu, set 2^2
//   below it and moved (and the sums rescaled) only when some p vs would pass 60,000, which fp16 just holds, or p what
//   keep_sums_finite allows (a test of the block's sums that costs 4 us of the 172 below: it waits for the exponentials).
//   2^2 leaves the maximum 2^14 to grow before sums are read and rescaled; p vs below 2^-16 of the maximum are
//   subnormal in fp16 then, each off by at most 2^-27 of the maximum.
//   Two further warps issue the products, one for each row tile.
//   Measured: 4 sequences of 1,500 to 4,096 tokens, the last 512 of each as rows, 32 heads (8 of the cache), D = 128:
//   171 us on the device, 173 with the host's call (12 us more before the scores were formed in halves, below).  A
//   tile of 256 rows takes about 5,000 cycles, of which the exponentials need 2,048 and the products as much: what bounds
//   it is the softmax warps' chain of loads, conversions and stores, 1,000 cycles and more for 32 columns whatever waits
//   beside it.  Half of the issue slots are used.  Reading the queries takes about 7,000 cycles of a block and writing the rows
//   5,000.  And the blocks' order: 256 of them start by row block, then by sequence, whatever their length.  Replayed on
//   148 SMs from these cycles that ends after 153 to 156 us; longest first would end after 116, evenly spread after 105.
//   Sparse rows (sinks, trees of drafted tokens) have instances of their own, in which a block works through a range of a
//   line of tiles of all segments (find_place), since segments of 2 to 70 tiles fill 148 SMs badly one to a block (trees:
//   234 us so, 127 on the line; a part of a segment costs about 10 us beside its tiles: reading queries 4, the first tile's
//   chain, writing 3).  Their softmax and unpacking warps take 88 registers, from two warps that only make the block whole
//   warpgroups: with 80 a few words more spilled, and as the codes' loads pass through what is left of L1 beside 205 KB of shared
//   memory, every reload went to L2 (5.3 us a tile of 256 rows where this takes 3.3; what still spills is 0.4% of the instructions).  Measured: 16 trees of 25 to 64 nodes
//   after 100 to 8,192 tokens, 32 heads (8 of the cache), D = 128, 127 us with the join; chunks of 512 rows of 4 sequences up
//   to 16,000 tokens, a window of 2,048 and 100 sinks, 142 us.  A tile takes 6,300 cycles there, 3,400 of them in the
//   columns' loops (exponentials alone: 2,048); the rest are its products' and barriers' latencies.  (The next tile's first
//   scores asked for before the last probabilities are written: 3% slower.)
// Every wait is bounded; a block that gives up writes NaN rows.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "quant4.cuh"

namespace msb {
namespace {

constexpr int kTokens = 128;         // of a tile
constexpr int kRowsTile = 128;       // rows of one accumulator
constexpr int kBlockRows = 256;
constexpr int kSoftWarps = 16;       // eight to a row tile: warp w has 16 rows, half (w / 4) % 2 of lane quarter w % 4
constexpr int kUnpackWarp0 = 16;     // warps 16-19: keys, the tiles' scales, values
constexpr int kMmaWarp = 20;         // warps 20, 21: a row tile's products each
constexpr int kThreads = 22 * 32;
constexpr int kLineThreads = 24 * 32;  // of a line's block: whole warpgroups, whose registers can be shared out
constexpr int kStages = 2;
constexpr float kLift = 2.0F;        // a reference is set 2^2 below the largest p vs seen
constexpr float kMostP = 60000.0F;   // and kept while p vs stays in fp16
constexpr int kCols = 32;            // columns of a softmax block
constexpr int kMetaPitch = 12;       // floats between the columns of a block that neighbouring lanes read (8 each)
constexpr int kMetaFloats = kTokens / kCols * 4 * kMetaPitch;
constexpr uint64_t kTimeoutNs = 4000000000ull;

template <int kDim>
struct Layout {
  static constexpr int kQBytes = kRowsTile * kDim * 2;         // one row tile
  static constexpr int kTileBytes = kTokens * kDim * 2;        // one tile of keys, or of values
  static constexpr int off_q = 0;
  static constexpr int off_k = off_q + 2 * kQBytes;
  static constexpr int off_v = off_k + kStages * kTileBytes;
  static constexpr int off_meta = off_v + kStages * kTileBytes;  // [stage][3]: key scales, value scales, their log2
  static constexpr int off_flags = off_meta + kStages * 3 * kMetaFloats * 4;  // [stage][4]: some token is not seen
  static constexpr int off_rows = off_flags + kStages * 16;      // [256] the rows' factors
  static constexpr int off_seen = off_rows + kBlockRows * 4;     // [256] what sparse rows see
  static constexpr int off_bars = off_seen + kBlockRows * 8;
  static constexpr int kUsed = off_bars + 24 * 8 + 1024;        // and room to align to 1024
  // A block takes all of an SM's tensor memory: more than half of its shared memory keeps a second one away.
  static constexpr int kBytes = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint64_t global_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
// False when the wait was given up (here or elsewhere in the block).
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  // A try sleeps in hardware until the phase ends or a while has passed; the clock, slow to read, comes after some.
#pragma unroll 1
  for (int i = 0; i < 16; ++i)
    if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  for (uint32_t it = 0;; ++it) {
    if (mbar_try(bar, parity)) return true;
    if ((it & 7u) == 7u) {
      if (*abort_flag) return false;
      if (global_ns() - t0 > kTimeoutNs) {
        *abort_flag = 1;
        return false;
      }
    }
  }
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// K-major, 128-byte swizzle: 1024 bytes between groups of 8 rows.
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Issued by the one lane whose `leader` is not 0, in converged code: operands stay warp-uniform.
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar)), "r"(leader)
      : "memory");
}
__device__ __forceinline__ uint32_t elect() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r;
}
// A block of 16 lanes x 32 columns: thread t has, for j = 0..3, columns 8j + 2 (t % 4) + {0, 1} of lane t / 4 in f[4j],
// f[4j + 1] and of lane t / 4 + 8 in f[4j + 2], f[4j + 3]; as fp16 pairs, 16 columns, r[2j] and r[2j + 1].
__device__ __forceinline__ void tmem_ld_block(uint32_t taddr, float (&f)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      " tcgen05.wait::ld.sync.aligned;"
      : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]),
        "=f"(f[8]), "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_block(uint32_t taddr, const float (&f)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
      :
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]),
        "f"(f[8]), "f"(f[9]), "f"(f[10]), "f"(f[11]), "f"(f[12]), "f"(f[13]), "f"(f[14]), "f"(f[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_pairs(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x128b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_pairs(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x4.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
      :
      : "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Nibbles kI and kI + 4 of a word as an exact fp16 pair (kv4_attend.cu).
template <int kI>
__device__ __forceinline__ uint32_t codes_exact(uint32_t w) {
  constexpr uint32_t kMask = kI & 1 ? 0x00f000f0u : 0x000f000fu, kFlip = kI & 1 ? 0x54805480u : 0x64086408u;
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;\n sub.rn.f16x2 %0, %0, %3;" : "=&r"(r) : "r"(kI < 2 ? w : w >> 8), "n"(kMask), "r"(kFlip));
  return r;
}
// Byte of 16-byte chunk `chunk` of row `row` in a tile of 128-byte rows, 128-byte swizzle.
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) {
  return static_cast<uint32_t>((row >> 3) * 1024 + (row & 7) * 128 + ((chunk ^ (row & 7)) << 4));
}
__device__ __forceinline__ void store16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Where column `c` of a tile keeps its scale: those of a block that one lane reads lie together.
__device__ __forceinline__ int meta_at(int c) {
  return c / kCols * (4 * kMetaPitch) + ((c >> 1) & 3) * kMetaPitch + (c % kCols >> 3) * 2 + (c & 1);
}

// What a thread keeps of its two rows, lane / 4 and + 8 of its warp's 16.
struct Rows {
  float2 factor[2];   // scale * log2(e) * the row's power of two, twice
  float2 ref[2];      // 2^-(reference), as an exponent, twice
  float2 sum[2];      // of p, the thread's columns
  int last[2];        // the last token seen
  int window;         // and how many up to it (INT_MAX: all)
  float top[2];       // the reference, -inf before there is one
};

// Scores (f: two rows x 8 columns) to probabilities times value scales, fp16 pairs; the largest into `most`.  Of sparse
// rows, `seen` has what each sees of the block, shifted to the thread's first column.
template <bool kMasked, bool kSparse>
__device__ __forceinline__ void probabilities(const float (&f)[16], const float* meta, int j0, const Rows& rows,
                                              const uint32_t (&seen)[2], uint32_t (&p)[8], float2 (&add)[2], float (&most)[2]) {
  add[0] = add[1] = make_float2(0.0F, 0.0F);
  most[0] = most[1] = 0.0F;
#pragma unroll
  for (int j = 0; j < kCols / 8; j += 2) {
    const float4 ks4 = *reinterpret_cast<const float4*>(meta + 2 * j);
    const float4 vs4 = *reinterpret_cast<const float4*>(meta + kMetaFloats + 2 * j);
    float4 e4 = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
    if (kMasked && !kSparse) e4 = *reinterpret_cast<const float4*>(meta + 2 * kMetaFloats + 2 * j);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 ks = h ? make_float2(ks4.z, ks4.w) : make_float2(ks4.x, ks4.y);
      const float2 vs = h ? make_float2(vs4.z, vs4.w) : make_float2(vs4.x, vs4.y);
      const float2 e = h ? make_float2(e4.z, e4.w) : make_float2(e4.x, e4.y);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int at = 4 * (j + h) + 2 * r;
        const float2 x = __ffma2_rn(__fmul2_rn(make_float2(f[at], f[at + 1]), ks), rows.factor[r], rows.ref[r]);
        float2 pr = make_float2(exp2_fast(x.x), exp2_fast(x.y));
        float2 pv = __fmul2_rn(pr, vs);
        if (kMasked) {
          const int c = j0 + 8 * (j + h);
          if (kSparse ? !(seen[r] & (1u << (8 * (j + h)))) : e.x == -INFINITY || c > rows.last[r] || rows.last[r] - c >= rows.window)
            pr.x = pv.x = 0.0F;
          if (kSparse ? !(seen[r] & (2u << (8 * (j + h))))
                      : e.y == -INFINITY || c + 1 > rows.last[r] || rows.last[r] - c - 1 >= rows.window)
            pr.y = pv.y = 0.0F;
        }
        add[r] = __fadd2_rn(add[r], pr);
        most[r] = fmax3(most[r], pv.x, pv.y);
        p[2 * (j + h) + r] = pack_half2(pv.x, pv.y);
      }
    }
  }
}
// The largest s + log2(vs) of the thread's seen columns, per row; -inf where there are none (or nothing but NaN).
template <bool kSparse>
__device__ __forceinline__ void references(const float (&f)[16], const float* meta, int j0, const Rows& rows,
                                           const uint32_t (&seen)[2], float (&best)[2]) {
  best[0] = best[1] = -INFINITY;
#pragma unroll
  for (int j = 0; j < kCols / 8; ++j)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float ks = meta[2 * j + k], e = meta[2 * kMetaFloats + 2 * j + k];
      const int c = j0 + 8 * j + k;
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (kSparse ? (seen[r] & (1u << (8 * j + k))) != 0u
                    : e != -INFINITY && c <= rows.last[r] && rows.last[r] - c < rows.window)
          best[r] = fmaxf(best[r], f[4 * j + 2 * r + k] * ks * rows.factor[r].x + e);
    }
}

// Whether token j's value is a vector of zeros.  Out of line: in the unpacking warps' loop it cost 5 us of 170.
template <int kDim, bool kSparse>
__device__ __noinline__ bool zero_value(const uint8_t* codes, const int32_t* pages, int heads, int head, int page_shift, int j) {
  const int64_t page = load_input<kSparse>(pages + (j >> page_shift));
  return zero_codes<kDim>(codes + (((page * heads + head) << page_shift) + (j & ((1 << page_shift) - 1))) * (kDim / 2));
}

// What a block does of one segment (sequence, head, 256 rows).
struct Work {
  Kv4Sequence q;
  int b, head;
  uint32_t block_row0;
  int row_count, tiles_m;
  int any_first, any_last;  // tokens that some row sees
  int begin, front;         // the tiles over them start at `begin`; sparse rows: `front` tiles over the sinks come first
  int tile0, tiles;         // this block's tiles
  bool whole;               // which are the segment's
  // Of the block's segments before: tiles, those of either row tile, and segments with tiles (the phases of barriers).
  int done, row_done[2], segments;
  template <bool kSparse>
  __device__ __forceinline__ int tile_start(int i) const {
    if (!kSparse) return begin + i * kTokens;
    return tile0 + i < front ? (tile0 + i) * kTokens : begin + (tile0 + i - front) * kTokens;
  }
};
template <bool kSparse>
__device__ __forceinline__ Work work_of(const Kv4Attend& a, uint32_t shared, const Kv4Sequence& q, int b, int head, int block) {
  Work w;
  w.q = q;
  w.b = b;
  w.head = head;
  w.block_row0 = static_cast<uint32_t>(block) * kBlockRows;  // below 2^31
  w.row_count = static_cast<int>(min(static_cast<uint32_t>(kBlockRows), static_cast<uint32_t>(q.rows) * shared - w.block_row0));
  w.tiles_m = w.row_count > kRowsTile ? 2 : 1;
  const int pos0 = q.pos0 + static_cast<int>(w.block_row0 / shared);
  const int pos1 = q.pos0 + static_cast<int>((w.block_row0 + w.row_count - 1) / shared);
  const bool tree = kSparse && a.ancestors != nullptr;
  w.any_last = a.causal && !tree ? pos1 : q.length - 1;
  // (Rows before the sequence's first token have negative positions; less a window these would pass 32 bits.)
  w.any_first = a.window > 0 ? max(0, max(0, tree ? q.pos0 - 1 : pos0) - a.window + 1) : 0;
  w.begin = w.any_first & ~15;
  w.front = 0;
  if constexpr (kSparse) {
    w.front = a.window > 0 ? (a.sinks + kTokens - 1) / kTokens : 0;
    if (w.front * kTokens >= w.begin) w.front = w.begin = 0;  // sinks that reach the window: one run
  }
  w.tile0 = 0;
  w.tiles = w.any_last >= w.any_first ? w.front + (w.any_last - w.begin) / kTokens + 1 : 0;
  w.whole = true;
  return w;
}

// Sparse rows' segments lie on a line: units of one tile, of every (sequence, head, row block), cut into equal ranges, one a
// block.  Every segment of a sequence has as many units as the largest could have tiles, and some for what a segment costs
// beside its tiles (reading queries, the first tile's chain, writing rows: about 10 us and the join, a tile 3 to 3.5).
constexpr int kSegmentUnits = 4;
// Segments are cut where there are fewer than blocks, into ranges of kLeastUnits and more (a part of one has its 10 us
// too).  The workspace: of each block the segment that starts in its range and ends in another, for the join, then the parts.
constexpr int kLeastUnits = 8;
struct Cut {
  int64_t row0;         // of the sequence
  uint32_t block_row0;
  int row_count;
  int head;
  int parts;            // 0: none
  int unused[2];
};
__host__ __device__ __forceinline__ size_t cut_bytes(int64_t blocks) {
  return (static_cast<size_t>(blocks) * sizeof(Cut) + 127) & ~static_cast<size_t>(127);
}
__device__ __forceinline__ float* chunk_parts(const Kv4Attend& a, int64_t blocks) {
  return reinterpret_cast<float*>(static_cast<char*>(a.workspace) + cut_bytes(blocks));
}
// Quotients of numbers that are mostly below 2^32 (a division in 64 bits takes several hundred cycles of a block's start).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}
struct Line {
  int units;   // of a segment
  int blocks;  // row blocks
  __device__ __forceinline__ int64_t all(int heads) const { return static_cast<int64_t>(heads) * blocks * units; }
};
__device__ __forceinline__ Line line_of(const Kv4Attend& a, const Kv4Sequence& q, uint32_t shared) {
  Line l;
  l.blocks = static_cast<int>((static_cast<uint32_t>(q.rows) * shared + kBlockRows - 1) / kBlockRows);
  l.units = max(1, (q.length + kTokens - 1) / kTokens);
  if (a.window > 0) {
    // A block's rows are those of this many query tokens (of a tree: all see the same tiles); a window that starts up
    // to 15 tokens early, and a tree's that starts one early.
    const int64_t tokens = a.ancestors ? static_cast<int64_t>(q.rows) + q.left + 1
                                       : min(static_cast<int64_t>(q.rows), static_cast<int64_t>((kBlockRows - 1) / shared + 2));
    const int64_t seen = (a.sinks + kTokens - 1) / kTokens + (tokens - 1 + a.window + 14) / kTokens + 1;
    l.units = static_cast<int>(min(static_cast<int64_t>(l.units), seen));
  }
  l.units += kSegmentUnits;
  return l;
}
// Segment `segment` of a sequence.
__device__ __forceinline__ Work segment_of(const Kv4Attend& a, uint32_t shared, const Kv4Sequence& q, const Line& l, int b,
                                           int64_t segment) {
  const int64_t head = quotient(segment, l.blocks);
  return work_of<true>(a, shared, q, b, static_cast<int>(head), static_cast<int>(segment - head * l.blocks));
}
// Where a block is on the line.
struct Place {
  int64_t unit, unit_end, before;  // before: units of the sequences before b
  int64_t total, ranges;
  int b;
};
// The block's next segments, up to `most`, into a list, and the one that is cut at its range's end for the join; by one
// thread.  A part past a segment's tiles is nobody's.
__device__ __forceinline__ int next_works(const Kv4View& c, const Kv4Attend& a, uint32_t shared, Place& p, Work* works, int most) {
  int count = 0, done = 0, row_done[2] = {0, 0}, segments = 0;
  const Work* const last_work = works + most - 1;
  if (p.unit < p.unit_end && p.before >= 0) {
    // (Counters go on from the list before, whose last entry is still there.)
    if (most > 0 && last_work->segments >= 0) {
      done = last_work->done + last_work->tiles;
      segments = last_work->segments + (last_work->tiles > 0);
      row_done[0] = last_work->row_done[0] + last_work->tiles;
      row_done[1] = last_work->row_done[1] + (last_work->tiles_m > 1 ? last_work->tiles : 0);
    }
    Kv4Sequence q = kv4_sequence(a, c.page_shift, p.b);
    Line l = line_of(a, q, shared);
    while (p.unit < p.unit_end && count < most) {
      while (p.unit >= p.before + l.all(c.heads)) {
        p.before += l.all(c.heads);
        q = kv4_sequence(a, c.page_shift, ++p.b);
        l = line_of(a, q, shared);
      }
      const int64_t inside = p.unit - p.before, segment = quotient(inside, l.units);
      const int first = static_cast<int>(inside - segment * l.units);
      const int last = static_cast<int>(min(static_cast<int64_t>(l.units), first + (p.unit_end - p.unit)));
      p.unit += last - first;
      Work w = segment_of(a, shared, q, l, p.b, segment);
      if (first >= max(1, w.tiles)) continue;
      w.whole = first == 0 && last >= w.tiles;
      if (first == 0 && !w.whole) {  // its tiles' last unit is so many ranges on
        const int64_t end = p.before + segment * l.units + w.tiles - 1;
        const int64_t on = quotient((end + 1) * p.ranges - 1, p.total) - blockIdx.x;
        static_cast<Cut*>(a.workspace)[blockIdx.x] =
            Cut{q.row0, w.block_row0, w.row_count, w.head, static_cast<int>(on) + 1, {0, 0}};
      }
      w.tile0 = first;
      w.tiles = max(0, min(last, w.tiles) - first);
      w.done = done;
      w.row_done[0] = row_done[0];
      w.row_done[1] = row_done[1];
      w.segments = segments;
      done += w.tiles;
      row_done[0] += w.tiles;
      row_done[1] += w.tiles_m > 1 ? w.tiles : 0;
      segments += w.tiles > 0;
      works[count++] = w;
    }
  }
  return count;
}
// The block's range, by all of its threads.
__device__ __noinline__ Place find_place(const Kv4View& c, const Kv4Attend& a, uint32_t shared) {
  __shared__ int64_t sums[kLineThreads / 32];
  __shared__ int64_t found[2];
  constexpr int kWarps = kLineThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto units_of = [&](int b) {
    if (b >= a.batch) return int64_t{0};
    return line_of(a, kv4_sequence(a, c.page_shift, b), shared).all(c.heads);
  };
  __shared__ int64_t segment_sums[kLineThreads / 32];
  int64_t total = 0, segments = 0;
  for (int b = threadIdx.x; b < a.batch; b += kLineThreads) {
    const Line l = line_of(a, kv4_sequence(a, c.page_shift, b), shared);
    total += l.all(c.heads);
    segments += static_cast<int64_t>(c.heads) * l.blocks;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    total += __shfl_xor_sync(0xFFFFFFFFu, total, d);
    segments += __shfl_xor_sync(0xFFFFFFFFu, segments, d);
  }
  if (lane == 0) sums[warp] = total, segment_sums[warp] = segments;
  __syncthreads();
  total = segments = 0;
  for (int i = 0; i < kWarps; ++i) total += sums[i], segments += segment_sums[i];
  const int64_t n = ranges(total, min(static_cast<int64_t>(gridDim.x), max(segments, total / kLeastUnits))), c0 = blockIdx.x;
  Place p{0, 0, 0, total, n, 0};
  if (c0 < n) {
    p.unit = quotient(c0 * total, n);
    p.unit_end = min(quotient((c0 + 1) * total, n), total);
  }
  int64_t carry = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kLineThreads) {
    const int b = b0 + threadIdx.x;
    const int64_t mine = units_of(b);
    int64_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
      if (lane >= d) upto += o;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int64_t base = carry;
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) base += sums[i];
      carry += sums[i];
    }
    const int64_t before = base + upto - mine;
    if (p.unit >= before && p.unit < before + mine) {
      found[0] = before;
      found[1] = b;
    }
  }
  if (threadIdx.x == 0) static_cast<Cut*>(a.workspace)[c0].parts = 0;  // until next_works finds one
  __syncthreads();
  if (p.unit < p.unit_end) {
    p.before = found[0];
    p.b = static_cast<int>(found[1]);
  }
  return p;
}

template <int kCount>
__device__ __forceinline__ void registers_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kCount));
}
template <int kCount>
__device__ __forceinline__ void registers_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCount));
}
// Bits 0 .. n - 1, of any n.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }
// Which of the 32 tokens from j on a row sees, but for its tree's (kv4_tree_bits).
__device__ __forceinline__ uint32_t run_bits(const Kv4Seen& run, int sinks, int j) {
  return low_bits(run.last + 1 - j) & (~low_bits(run.first - j) | low_bits(sinks - j));
}

// kSparse: rows that see sinks past their window, or a tree of drafted tokens (kv4_seen), by ranges of the line: a block
// has one segment after the other, of the first and the last perhaps a part, whose sums go to the workspace.  Its roles
// pass from a segment to the next by themselves, as barriers' phases count on.
template <class T, int kDim, bool kSparse>
__global__ void __launch_bounds__(kSparse ? kLineThreads : kThreads, 1)
    kv4_chunk_kernel(const __grid_constant__ Kv4View c, const __grid_constant__ Kv4Attend a, uint32_t shared, int row_blocks, bool aligned) {
  using L = Layout<kDim>;
  extern __shared__ unsigned char raw_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // On a line: the block's next segments, and how many.  (In shared memory: read once a tile, in registers they would cost
  // those of the loops.)
  constexpr int kList = kSparse ? 32 : 1;
  __shared__ Work works[kList];
  __shared__ Place place;
  __shared__ int work_count;
  Work only{};
  int share = 0, shares = 1;
  if constexpr (!kSparse) {
    // Later row blocks see more tokens under a causal mask: they start first.
    const int64_t per_block = static_cast<int64_t>(a.batch) * c.heads;
    const int block = row_blocks - 1 - static_cast<int>(blockIdx.x / per_block);
    const int b = static_cast<int>(blockIdx.x % per_block / c.heads), head = static_cast<int>(blockIdx.x % c.heads);
    const Kv4Sequence q = kv4_sequence(a, c.page_shift, b);
    share = block * c.heads + head, shares = row_blocks * c.heads;  // of the sequence's blocks
    if (static_cast<uint32_t>(block) * kBlockRows >= static_cast<uint32_t>(q.rows) * shared) {
      if (a.fill) kv4_fill_rows<T>(a, kDim, b, q, share, shares, threadIdx.x, kThreads);
      return;
    }
    only = work_of<false>(a, shared, q, b, head, block);
  }
  const bool tree = kSparse && a.ancestors != nullptr;

  unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t{1023});
  const uint32_t base = smem_u32(smem);
  float* const meta = reinterpret_cast<float*>(smem + L::off_meta);
  uint32_t* const flags = reinterpret_cast<uint32_t*>(smem + L::off_flags);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + L::off_bars);
  uint64_t* const k_full = bars;           // [stage] keys and scales written
  uint64_t* const k_empty = bars + 2;      // [stage] products over the keys done
  uint64_t* const v_full = bars + 4;
  uint64_t* const v_empty = bars + 6;
  uint64_t* const meta_empty = bars + 8;   // [stage] scales read by every softmax warp
  uint64_t* const s_full = bars + 10;      // [row tile] all scores ready (and the sums of the tile before)
  uint64_t* const p_full = bars + 12;      // [row tile] probabilities written
  uint64_t* const o_full = bars + 14;      // all sums done
  uint64_t* const q_full = bars + 15;
  uint64_t* const s_half = bars + 16;      // [row tile] scores of the half that comes first ready
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(bars + 19);
  // Row tiles that arrive: on a line always two; where a segment has one, that one's warps arrive for both.
  const int row_tiles = kSparse ? 2 : only.tiles_m;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&k_empty[s], row_tiles);
      mbar_init(&v_full[s], 4);
      mbar_init(&v_empty[s], row_tiles);
      mbar_init(&meta_empty[s], 8 * row_tiles);
    }
    for (int m = 0; m < 2; ++m) {
      mbar_init(&s_half[m], 1);
      mbar_init(&s_full[m], 1);
      mbar_init(&p_full[m], 8);
    }
    mbar_init(o_full, row_tiles);
    mbar_init(q_full, 8 * row_tiles);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if constexpr (kSparse) {  // nothing of what is above reads what the kernel before may write
    wait_for_previous();
    let_next_start();
    const Place start = find_place(c, a, shared);
    if (threadIdx.x == 0) {
      place = start;
      works[kList - 1].segments = -1;
      work_count = next_works(c, a, shared, place, works, kList);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
  // Tensor memory: scores of the row tiles at columns 0 and 128 (probabilities over them), sums at 256 and 384.
  // Half h of a tile's scores, 64 tokens, is in columns 64 h and on.  Of tile i the half i % 2 comes first and the
  // probabilities of both go to its columns, so that the other half's are free for the half of tile i + 1 that
  // comes first: its product does not wait for this tile's sums, nor its softmax.

  const int page_mask = (1 << c.page_shift) - 1;
  // Vector of token j's 16-token group on page p (-1: none), and whether the page is the cache's.
  auto ask_page = [&](const Work& w, int j) {
    return j <= w.any_last ? load_input<kSparse>(a.page_table + w.b * a.table_stride + (j >> c.page_shift)) : -1;
  };
  auto vector_of = [&](const Work& w, int page, int j) {
    return static_cast<uint32_t>(page) < static_cast<uint32_t>(c.num_pages)
               ? (static_cast<int64_t>(static_cast<uint32_t>(page) * c.heads + w.head) << c.page_shift) + (j & page_mask)
               : int64_t{0};
  };

  auto work = [&](int k) -> const Work& {
    if constexpr (kSparse) return works[k];
    return only;
  };
  int count = 1;
  if constexpr (kSparse) count = work_count;
  // The next list, after a full one: every role comes here (with the loop over lists around the roles, what one of them
  // needs would be formed before it and held through all).
  auto next_list = [&](bool writes) {
    if (!kSparse || count < kList) return false;
    asm volatile("bar.sync 0;" ::: "memory");
    if constexpr (kSparse)
      if (writes && threadIdx.x == (kMmaWarp + 2) * 32) work_count = next_works(c, a, shared, place, works, kList);
    asm volatile("bar.sync 0;" ::: "memory");
    count = work_count;
    return count > 0;
  };
  // Of the 24 x 32 x 80 registers that a line's block is launched with: 20 warps' 88 and 4 warps' 40.  (Each role asks for its
  // own: after a common place the compiler would not know which it has.  96, 64 and 32: 1% faster with two row tiles, 10%
  // slower with one, which the unpacking bounds then; 88, 72 and 56: 4% slower.)
  if (warp < kSoftWarps) {
    if constexpr (kSparse) registers_inc<88>();
    // =================== softmax: a warp has 16 rows, a thread two of them and a quarter of their columns ===================
    const int m = warp >> 3;
    bool ok = true;
    do {
      for (int segment = 0; segment < count; ++segment) {
        const Work& w = work(segment);
        const int row0 = (warp & 3) * 32 + ((warp >> 2) & 1) * 16;  // of the row tile, and its lane of tensor memory
        if (kSparse ? m * kRowsTile + row0 >= w.row_count : m >= w.tiles_m) {
          // No rows for this warp.  On a line it passes the segment with the others all the same, as no wait may fall a phase
          // behind, and arrives for what it does not do (its rows' products are never read): the warps that have rows get
          // its share of the issue slots.
          if constexpr (kSparse) {
            if (w.tiles == 0) continue;
            if (lane == 0) mbar_arrive(q_full);
            for (int i = 0; i < w.tiles && m < w.tiles_m && ok; ++i) {
              ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s_full[m], (w.row_done[m] + i) & 1, abort_flag));
              if (lane == 0 && ok) {
                uint64_t* const bar = &meta_empty[(w.done + i) & 1];
                mbar_arrive(bar);
                if (w.tiles_m == 1) mbar_arrive(bar);
                mbar_arrive(&p_full[m]);
              }
            }
            ok = ok && mbar_wait(o_full, w.segments & 1, abort_flag);
            ok = __all_sync(0xFFFFFFFFu, ok);
          }
          continue;
        }
        float* const row_factor = reinterpret_cast<float*>(smem + L::off_rows) + m * kRowsTile + row0;
        constexpr int kRowLanes = kDim / 8, kRowsAtOnce = 32 / kRowLanes, kLoads = 16 / kRowsAtOnce;
        // The warp's rows of the query tile, 8 dimensions a lane: scaled by a power of two to a maximum in [2^10, 2^11),
        // fp16, in the codes' order.  In a short loop, two loads ahead: what runs once a segment is fetched from memory, and
        // eight rows' code straight on took 4.3 us of each.
        constexpr int kBatch = 2;
        const int first_row = m * kRowsTile + row0 + lane / kRowLanes;
        uint32_t token = (w.block_row0 + first_row) / shared, in_group = w.block_row0 + first_row - token * shared;
        int r = first_row;  // the next row to be asked for, query head in_group of the row's token
        auto ask = [&](uint4 (&x)[kBatch]) {
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            x[k] = make_uint4(0, 0, 0, 0);
            if (r < w.row_count) {
              const T* src = static_cast<const T*>(a.query) + (w.q.row0 + token) * a.q_row_stride +
                             static_cast<int64_t>(w.head * shared + in_group) * a.q_head_stride + (lane % kRowLanes) * 8;
              if (aligned) {
                x[k] = load_input<kSparse>(reinterpret_cast<const uint4*>(src));
              } else {
                __align__(16) T e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = src[i];
                x[k] = *reinterpret_cast<const uint4*>(e);
              }
            }
            r += kRowsAtOnce;
            in_group += kRowsAtOnce;
            while (in_group >= shared) in_group -= shared, ++token;
          }
        };
        uint4 x[kBatch], next[kBatch];
        ask(next);
#pragma unroll 1
        for (int k0 = 0; k0 < kLoads; k0 += kBatch) {
#pragma unroll
          for (int k = 0; k < kBatch; ++k) x[k] = next[k];
          if (k0 + kBatch < kLoads) ask(next);
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            const T* const v = reinterpret_cast<const T*>(&x[k]);
            float top = 0.0F;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(to_f32(v[i])));
#pragma unroll
            for (int d = 1; d < kRowLanes; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
            const int e = max(-110, min(127, static_cast<int>(__float_as_uint(top) >> 23) - 127));
            const float down = __uint_as_float(static_cast<uint32_t>(127 + 10 - e) << 23);
            const int here = (k0 + k) * kRowsAtOnce + lane / kRowLanes, piece = lane % kRowLanes;
            store16(base + L::off_q + m * L::kQBytes + (piece >> 3) * (kRowsTile * 128) + swizzled(row0 + here, piece & 7),
                    pack_half2(to_f32(v[0]) * down, to_f32(v[4]) * down), pack_half2(to_f32(v[1]) * down, to_f32(v[5]) * down),
                    pack_half2(to_f32(v[2]) * down, to_f32(v[6]) * down), pack_half2(to_f32(v[3]) * down, to_f32(v[7]) * down));
            if (piece == 0) row_factor[here] = a.scale * 1.44269504F * __uint_as_float(static_cast<uint32_t>(127 - 10 + e) << 23);
          }
        }
        fence_proxy_async();
        if (kSparse) tc_fence_before();  // the sums of the segment before have been read
        __syncwarp();
        if (lane == 0 && (!kSparse || w.tiles > 0)) mbar_arrive(q_full);

        Rows rows;
        int every_first = 0, every_last = 0;
        Kv4Seen* const row_seen = reinterpret_cast<Kv4Seen*>(smem + L::off_seen) + m * kRowsTile + row0;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          // Rows past the last do as it does: what they compute is not written.
          const int mine = 8 * k + (lane >> 2), at = min(m * kRowsTile + row0 + mine, w.row_count - 1);
          const int pos = w.q.pos0 + static_cast<int>((w.block_row0 + at) / shared);
          rows.factor[k] = make_float2(row_factor[mine], row_factor[mine]);
          rows.ref[k] = rows.sum[k] = make_float2(0.0F, 0.0F);
          rows.last[k] = a.causal ? pos : w.q.length - 1;
          rows.top[k] = -INFINITY;
          if constexpr (kSparse) {
            const Kv4Seen seen = kv4_seen(a, w.q, pos - w.q.pos0);
            every_first = k ? max(every_first, seen.first) : seen.first;
            every_last = k ? min(every_last, seen.last) : seen.last;
            row_seen[mine] = seen;  // (four lanes write the same)
          }
        }
        if constexpr (kSparse) __syncwarp();
        rows.window = a.window > 0 ? a.window : INT_MAX;
        if constexpr (!kSparse) {
          every_last = min(rows.last[0], rows.last[1]);
          every_first = a.window > 0 ? max(0, max(rows.last[0], rows.last[1])) - a.window + 1 : 0;
        }
        const uint32_t s_at = tmem + (static_cast<uint32_t>(row0) << 16) + m * 128, o_at = s_at + 256;
        for (int i = 0; i < w.tiles; ++i) {
          const int it = kSparse ? w.done + i : i, s = it & 1, j0 = w.tile_start<kSparse>(i);
          const int im = kSparse ? w.row_done[m] + i : i;
          ok = (!kSparse || ok) && mbar_wait(&k_full[s], (it >> 1) & 1, abort_flag) && mbar_wait(&s_half[m], im & 1, abort_flag);
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint4 flag = *reinterpret_cast<const uint4*>(flags + 4 * s);
          const bool masked = __any_sync(0xFFFFFFFFu, (flag.x | flag.y | flag.z | flag.w) != 0u || j0 < every_first ||
                                                         j0 + kTokens - 1 > every_last);
          const uint32_t p_at = s_at + s * (kTokens / 2);
          // A block of 32 columns.  kMode: without masks, with them, or as `masked` says.
          auto columns = [&](int part, auto mode) {
            constexpr int kMode = decltype(mode)::value;
            const bool with_masks = kMode == 2 ? masked : kMode == 1;
            const int piece = part ^ (2 * s);  // the block of columns
            const float* const my_meta = meta + s * 3 * kMetaFloats + (4 * piece + (lane & 3)) * kMetaPitch;
            const int my_j0 = j0 + kCols * piece + 2 * (lane & 3);
            if (part == kTokens / kCols / 2) {
              ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s_full[m], im & 1, abort_flag));
              if (!ok) return;
              tc_fence_after();
            }
            uint32_t seen[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
            if (kSparse && with_masks) {
              const int j = j0 + kCols * piece;
              const uint32_t absent = flags[4 * s + piece];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int mine = 8 * k + (lane >> 2);
                seen[k] = run_bits(row_seen[mine], a.sinks, j);
                if (tree && j + kCols > w.q.pos0)
                  seen[k] |= kv4_tree_bits(
                      a, w.q, static_cast<int>((w.block_row0 + min(m * kRowsTile + row0 + mine, w.row_count - 1)) / shared), j);
                seen[k] = (seen[k] & ~absent) >> (2 * (lane & 3));
              }
            }
            float f[16], most[2];
            float2 add[2];
            uint32_t p[8];
            tmem_ld_block(s_at + kCols * piece, f);
            if (with_masks) probabilities<true, kSparse>(f, my_meta, my_j0, rows, seen, p, add, most);
            else probabilities<false, kSparse>(f, my_meta, my_j0, rows, seen, p, add, most);
            // A row without a reference yet, or one whose reference has become too low: for p vs, or for p, which value
            // scales near zero let grow unseen by p vs (an infinite p among either).
            const float weights = fmax3(fmaxf(add[0].x, add[0].y), add[1].x, add[1].y);
            const bool low = fminf(rows.top[0], rows.top[1]) == -INFINITY || fmaxf(most[0], most[1]) > kMostP || weights > a.most_weight;
            if (__any_sync(0xFFFFFFFFu, low)) {
              tmem_wait_st();  // what was written before is read below, the sums of the tiles before too
              ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s_full[m], im & 1, abort_flag));
              if (!ok) return;
              tc_fence_after();
              float best[2], fade[2];
              tmem_ld_block(s_at + kCols * piece, f);
              references<kSparse>(f, my_meta, my_j0, rows, seen, best);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                best[k] = fmaxf(best[k], __shfl_xor_sync(0xFFFFFFFFu, best[k], 1));
                best[k] = fmaxf(best[k], __shfl_xor_sync(0xFFFFFFFFu, best[k], 2));
                const float next = fmaxf(rows.top[k], best[k]);
                fade[k] = fade_to(rows.top[k], next);
                rows.top[k] = next;
                const float ref = next == -INFINITY ? 0.0F : kLift - next;
                rows.ref[k] = make_float2(ref, ref);
                rows.sum[k] = __fmul2_rn(rows.sum[k], make_float2(fade[k], fade[k]));
              }
              probabilities<true, kSparse>(f, my_meta, my_j0, rows, seen, p, add, most);
              if (i > 0) {  // the sums of the tiles before
#pragma unroll 1
                for (int d = 0; d < kDim; d += kCols) {
                  tmem_ld_block(o_at + d, f);
#pragma unroll
                  for (int k = 0; k < 16; ++k) f[k] *= fade[(k >> 1) & 1];
                  tmem_st_block(o_at + d, f);
                }
              }
#pragma unroll 1
              for (int d = 0; d < part; ++d) {  // and the probabilities of the columns before
                uint32_t w[8];
                tmem_ld_pairs(p_at + kCols / 2 * d, w);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
                  w[k] = pack_half2(v.x * fade[k & 1], v.y * fade[k & 1]);
                }
                tmem_st_pairs(p_at + kCols / 2 * d, w);
              }
            }
            rows.sum[0] = __fadd2_rn(rows.sum[0], add[0]);
            rows.sum[1] = __fadd2_rn(rows.sum[1], add[1]);
            tmem_st_pairs(p_at + kCols / 2 * part, p);
          };
          // Blocks in one short loop: its instructions stay near, the other three warps of a scheduler fill its waits.
          // (Sparse rows' masks are selects in the same steps: as one loop with both, the compiler joined the two, and every
          // tile paid for them.)
          if constexpr (!kSparse) {
#pragma unroll 1
            for (int part = 0; part < kTokens / kCols; ++part) {
              columns(part, std::integral_constant<int, 2>{});
              if (!ok) break;
            }
          } else if (masked) {
#pragma unroll 1
            for (int part = 0; part < kTokens / kCols; ++part) {
              columns(part, std::integral_constant<int, 1>{});
              if (!ok) break;
            }
          } else {
#pragma unroll 1
            for (int part = 0; part < kTokens / kCols; ++part) {
              columns(part, std::integral_constant<int, 0>{});
              if (!ok) break;
            }
          }
          if (!ok) break;
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (kSparse) {  // (a segment's last probabilities end it: what is counted on comes before)
              mbar_arrive(&meta_empty[s]);
              if (w.tiles_m == 1) mbar_arrive(&meta_empty[s]);
            }
            mbar_arrive(&p_full[m]);
            if (!kSparse) mbar_arrive(&meta_empty[s]);
          }
        }
        // The rows' outputs, through the query tile's shared memory to 16 bytes a lane.
        if (ok && w.tiles > 0) ok = mbar_wait(o_full, kSparse ? w.segments & 1 : 0, abort_flag);
        ok = __all_sync(0xFFFFFFFFu, ok) && !*abort_flag;
        tc_fence_after();
        float inv[2], sum[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float l = rows.sum[k].x + rows.sum[k].y;
          l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
          l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
          sum[k] = l;
          inv[k] = l == 0.0F ? 0.0F : 1.0F / l;
        }
        if constexpr (kSparse) {
          if (!w.whole) {  // a part of a segment: its sums as they are, and their references
            float* const part =
                chunk_parts(a, gridDim.x) + (2 * static_cast<int64_t>(blockIdx.x) + (w.tile0 == 0 ? 1 : 0)) * partial_floats(kBlockRows, kDim);
            float* const sums = part + (m * kRowsTile + row0 + (lane >> 2)) * kDim + 2 * (lane & 3);
#pragma unroll 1
            for (int d = 0; d < kDim && w.tiles > 0; d += kCols) {
              float f[16];
              if (ok) tmem_ld_block(o_at + d, f);
#pragma unroll
              for (int k = 0; k < 8; ++k)
                *reinterpret_cast<float2*>(sums + (k & 1) * 8 * kDim + d + 8 * (k >> 1)) = make_float2(f[2 * k], f[2 * k + 1]);
            }
            if ((lane & 3) == 0) {
#pragma unroll
              for (int k = 0; k < 2; ++k)
                *reinterpret_cast<float2*>(part + kBlockRows * kDim + 2 * (m * kRowsTile + row0 + 8 * k + (lane >> 2))) =
                    ok ? make_float2(rows.top[k], w.tiles > 0 ? sum[k] : 0.0F) : make_float2(0.0F, NAN);
            }
            continue;
          }
        }
#pragma unroll 1
        for (int d = 0; d < kDim; d += kCols) {
          float f[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) f[k] = 0.0F;
          if (ok && w.tiles > 0) tmem_ld_block(o_at + d, f);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float scale = inv[k & 1];
            T e[2];
            e[0] = from_f32<T>(!ok ? NAN : sum[k & 1] == 0.0F ? 0.0F : f[2 * k] * scale);
            e[1] = from_f32<T>(!ok ? NAN : sum[k & 1] == 0.0F ? 0.0F : f[2 * k + 1] * scale);
            const int r = row0 + 8 * (k & 1) + (lane >> 2), piece = (d >> 3) + (k >> 1);
            uint32_t v;
            memcpy(&v, e, 4);
            *reinterpret_cast<uint32_t*>(smem + L::off_q + m * L::kQBytes + (piece >> 3) * (kRowsTile * 128) +
                                         swizzled(r, piece & 7) + 4 * (lane & 3)) = v;
          }
        }
        __syncwarp();
        const bool out_aligned = (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
#pragma unroll 4
        for (int k = 0; k < kLoads; ++k) {
          const int in_warp = k * kRowsAtOnce + lane / kRowLanes, r = m * kRowsTile + row0 + in_warp, piece = lane % kRowLanes;
          if (r >= w.row_count) continue;
          const uint32_t token = (w.block_row0 + r) / shared, in_group = w.block_row0 + r - token * shared;
          const int64_t out_row = (w.q.row0 + token) * a.heads + w.head * shared + in_group;
          const uint4 v = *reinterpret_cast<const uint4*>(smem + L::off_q + m * L::kQBytes + (piece >> 3) * (kRowsTile * 128) +
                                                          swizzled(row0 + in_warp, piece & 7));
          T* const out = static_cast<T*>(a.out) + out_row * kDim + piece * 8;
          if (out_aligned) {
            *reinterpret_cast<uint4*>(out) = v;
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) out[i] = reinterpret_cast<const T*>(&v)[i];
          }
        }
        if (a.lse && (lane & 3) == 0) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int r = m * kRowsTile + row0 + 8 * k + (lane >> 2);
            if (r >= w.row_count) continue;
            const uint32_t token = (w.block_row0 + r) / shared, in_group = w.block_row0 + r - token * shared;
            const float reference = rows.top[k] == -INFINITY ? 0.0F : rows.top[k] - kLift;
            a.lse[(w.q.row0 + token) * a.heads + w.head * shared + in_group] =
                !ok ? NAN : sum[k] == 0.0F ? -INFINITY : (reference + __log2f(sum[k])) * 0.693147181F;
          }
        }
      }
    } while (next_list(false));
  } else if (warp < kMmaWarp) {
    if constexpr (kSparse) registers_inc<88>();
    // =================== unpacking ===================
    // Keys: lane (g, t) takes 16 bytes t (at D = 128) of tokens g, g + 8, .. of its warp's 32.
    const int uw = warp - kUnpackWarp0, g = lane >> 2, t = lane & 3;
    constexpr int kWords = kDim / 32;                       // of a token, per lane
    uint32_t word[4][kWords];
    float ks = 0.0F, vs = 0.0F;
    bool seen = false;
    int page[2] = {-1, -1};
    auto load_keys = [&](const Work& w, int i) {
      const int j = w.tile_start<kSparse>(i) + 32 * uw;
      const int64_t v[2] = {vector_of(w, page[0], j), vector_of(w, page[1], j + 16)};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint8_t* src = c.codes[0] + (v[k >> 1] + 8 * (k & 1) + g) * (kDim / 2) + t * (kDim / 8);
        if constexpr (kWords == 4) {
          const uint4 u = load_input<kSparse>(reinterpret_cast<const uint4*>(src));
          word[k][0] = u.x, word[k][1] = u.y, word[k][2] = u.z, word[k][3] = u.w;
        } else {
          const uint2 u = load_input<kSparse>(reinterpret_cast<const uint2*>(src));
          word[k][0] = u.x, word[k][1] = u.y;
        }
      }
      const int mine = j + lane;
      const int64_t at = (lane < 16 ? v[0] : v[1]) + (lane & 15);
      seen = static_cast<uint32_t>(lane < 16 ? page[0] : page[1]) < static_cast<uint32_t>(c.num_pages) &&
             (mine >= w.any_first || (kSparse && mine < a.sinks)) && mine <= w.any_last;
      ks = load_input<kSparse>(c.scales[0] + at);
      vs = load_input<kSparse>(c.scales[1] + at);
      const int next = kSparse ? w.tile_start<kSparse>(i + 1) + 32 * uw : j + kTokens;
      page[0] = ask_page(w, next);
      page[1] = ask_page(w, next + 16);
    };
    // Values: a lane takes 8 tokens and 8 or 16 dimensions.
    constexpr int kValueWords = kDim / 64;                  // 8-dimension words of a token, per lane
    const int group = (uw >> 1) * 8 + (lane & 7);           // its 8 tokens
    const int piece = (uw & 1) * 4 + (lane >> 3);           // its words: piece * kValueWords and on
    uint32_t value[8][kValueWords];
    int value_page = -1;
    auto load_values = [&](const Work& w, int i) {
      const int j = w.tile_start<kSparse>(i) + (group >> 1) * 16;
      const uint8_t* src = c.codes[1] + (vector_of(w, value_page, j) + 8 * (group & 1)) * (kDim / 2) + piece * (4 * kValueWords);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if constexpr (kValueWords == 2) {
          const uint2 u = load_input<kSparse>(reinterpret_cast<const uint2*>(src + k * (kDim / 2)));
          value[k][0] = u.x, value[k][1] = u.y;
        } else {
          value[k][0] = load_input<kSparse>(reinterpret_cast<const uint32_t*>(src + k * (kDim / 2)));
        }
      }
      value_page = ask_page(w, kSparse ? w.tile_start<kSparse>(i + 1) + (group >> 1) * 16 : j + kTokens);
    };
    bool ok = true;
    do {
      for (int segment = 0; segment < count && ok; ++segment) {
        const Work& w = work(segment);
        if (w.tiles > 0) {
          page[0] = ask_page(w, w.tile_start<kSparse>(0) + 32 * uw);
          page[1] = ask_page(w, w.tile_start<kSparse>(0) + 32 * uw + 16);
          value_page = ask_page(w, w.tile_start<kSparse>(0) + (group >> 1) * 16);
          load_keys(w, 0);
          load_values(w, 0);
        }
        for (int i = 0; i < w.tiles; ++i) {
          const int it = kSparse ? w.done + i : i, s = it & 1;
          const uint32_t parity = ((it >> 1) - 1) & 1;
          if (it >= kStages) {
            ok = mbar_wait(&k_empty[s], parity, abort_flag) && mbar_wait(&meta_empty[s], parity, abort_flag);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
          }
          const uint32_t key_dst = base + L::off_k + s * L::kTileBytes;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int token = 32 * uw + 8 * k + g;
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
              // Lanes two apart lie in the two halves of a row: they take their words in another order, off the same banks.
              const int jj = kWords == 4 ? j ^ (t & 2) : j;
              uint32_t w = word[k][j];
              if constexpr (kWords == 4) w = (t & 2) ? word[k][j ^ 2] : w;
              const int at = t * kWords + jj;  // word of the row
              store16(key_dst + (at >> 3) * (kTokens * 128) + swizzled(token, at & 7), codes_exact<0>(w), codes_exact<1>(w),
                      codes_exact<2>(w), codes_exact<3>(w));
            }
          }
          float* const ms = meta + s * 3 * kMetaFloats + meta_at(32 * uw + lane);
          if (seen && vs == 1.0F &&
              zero_value<kDim, kSparse>(c.codes[1], a.page_table + w.b * a.table_stride, c.heads, w.head, c.page_shift,
                               w.tile_start<kSparse>(i) + 32 * uw + lane))
            vs = 0.0F;
          ms[0] = seen ? ks : 0.0F;
          ms[kMetaFloats] = seen ? vs : 0.0F;
          ms[2 * kMetaFloats] = seen ? scale_exponent(vs, a.least_exponent, most_exponent(kLift)) : -INFINITY;
          const uint32_t all = __ballot_sync(0xFFFFFFFFu, seen);
          if (lane == 0) flags[4 * s + uw] = ~all;
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&k_full[s]);
          if (i + 1 < w.tiles) load_keys(w, i + 1);

          if (it >= kStages) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(&v_empty[s], parity, abort_flag));
            if (!ok) break;
          }
          // Row of a dimension: 64 tokens, 128 bytes; this lane's 8 tokens are one 16-byte chunk.
          const uint32_t dst = base + L::off_v + s * L::kTileBytes + (group >> 3) * (kDim * 128);
#pragma unroll
          for (int j = 0; j < kValueWords; ++j) {
            uint32_t x[4], y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              x[k] = __byte_perm(value[2 * k][j], value[2 * k + 1][j], 0x5410);
              y[k] = __byte_perm(value[2 * k][j], value[2 * k + 1][j], 0x7632);
            }
            const int d = (piece * kValueWords + j) * 8, chunk = group & 7;
            store16(dst + swizzled(d + 0, chunk), codes_exact<0>(x[0]), codes_exact<0>(x[1]), codes_exact<0>(x[2]), codes_exact<0>(x[3]));
            store16(dst + swizzled(d + 1, chunk), codes_exact<1>(x[0]), codes_exact<1>(x[1]), codes_exact<1>(x[2]), codes_exact<1>(x[3]));
            store16(dst + swizzled(d + 2, chunk), codes_exact<2>(x[0]), codes_exact<2>(x[1]), codes_exact<2>(x[2]), codes_exact<2>(x[3]));
            store16(dst + swizzled(d + 3, chunk), codes_exact<3>(x[0]), codes_exact<3>(x[1]), codes_exact<3>(x[2]), codes_exact<3>(x[3]));
            store16(dst + swizzled(d + 4, chunk), codes_exact<0>(y[0]), codes_exact<0>(y[1]), codes_exact<0>(y[2]), codes_exact<0>(y[3]));
            store16(dst + swizzled(d + 5, chunk), codes_exact<1>(y[0]), codes_exact<1>(y[1]), codes_exact<1>(y[2]), codes_exact<1>(y[3]));
            store16(dst + swizzled(d + 6, chunk), codes_exact<2>(y[0]), codes_exact<2>(y[1]), codes_exact<2>(y[2]), codes_exact<2>(y[3]));
            store16(dst + swizzled(d + 7, chunk), codes_exact<3>(y[0]), codes_exact<3>(y[1]), codes_exact<3>(y[2]), codes_exact<3>(y[3]));
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_full[s]);
          if (i + 1 < w.tiles) load_values(w, i + 1);
      }
      }
    } while (next_list(false));
    // These warps are done first.
    if (a.fill) {
      constexpr int kFillThreads = (kMmaWarp - kUnpackWarp0) * 32;
      const int thread = threadIdx.x - kUnpackWarp0 * 32;
      if constexpr (kSparse) {
        for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
          kv4_fill_rows<T>(a, kDim, b, kv4_sequence(a, c.page_shift, b), 0, 1, thread, kFillThreads);
      } else {
        kv4_fill_rows<T>(a, kDim, only.b, kv4_sequence(a, c.page_shift, only.b), share, shares, thread, kFillThreads);
      }
    }
  } else {
    if constexpr (kSparse) registers_dec<40>();
    if (warp >= kMmaWarp + 2) {
      // They make a line's block whole warpgroups, and its lists.
      while (next_list(true)) {
      }
    } else if (kSparse || (warp - kMmaWarp < only.tiles_m && only.tiles > 0)) {
      // =================== products of a row tile: one lane issues ===================
      const int m = warp - kMmaWarp;
      const uint32_t leader = elect();
      constexpr uint32_t kInstrS = (1u << 4) | (static_cast<uint32_t>(kTokens / 2 >> 3) << 17) | (8u << 24);
      constexpr uint32_t kInstrO = (1u << 4) | (static_cast<uint32_t>(kDim >> 3) << 17) | (8u << 24);
      const uint32_t s_tmem = tmem + m * 128, o_tmem = s_tmem + 256;
      const uint64_t q_desc = operand_desc(base + L::off_q + m * L::kQBytes), k_desc = operand_desc(base + L::off_k);
      const uint64_t v_desc = operand_desc(base + L::off_v);
      auto scores = [&](int s, int half) {
#pragma unroll
        for (int k = 0; k < kDim / 16; ++k) {  // 16 dimensions: 32 bytes of a 128-byte row
          const uint32_t at = ((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4;
          const uint32_t rows = half * (kTokens / 2 * 128) >> 4;
          mma_ss(leader, s_tmem + half * (kTokens / 2), q_desc + at, k_desc + (s * L::kTileBytes >> 4) + rows + at, kInstrS, k > 0);
        }
      };
      // (For both row tiles, where a segment of a line has one.)
      uint32_t alone = 0;
      auto commit_both = [&](uint64_t* bar) {
        mma_commit(leader, bar);
        if (kSparse) mma_commit(leader & alone, bar);
      };
      auto first_half = [&](int s) {
        scores(s, s);
        mma_commit(leader, &s_half[m]);
      };
      auto other_half = [&](int s) {
        scores(s, s ^ 1);
        mma_commit(leader, &s_full[m]);
        commit_both(&k_empty[s]);
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag)) != 0;
      };
      bool ok = true;
      do {
        for (int segment = 0; segment < count && ok; ++segment) {
          const Work& w = work(segment);
          if (kSparse && w.tiles == 0) continue;
          alone = w.tiles_m == 1;
          ok = wait(q_full, kSparse ? w.segments & 1 : 0);
          if (kSparse && m >= w.tiles_m) {
            // Nothing to do but to have seen this phase: the next one's arrivals come after o_full, which waits for this.
            if (ok && lane == 0) mbar_arrive(o_full);
            continue;
          }
          const int start = kSparse ? w.done : 0;
          ok = ok && wait(&k_full[start & 1], (start >> 1) & 1);
          if (ok) {
            tc_fence_after();
            first_half(start & 1);
            other_half(start & 1);
          }
          for (int i = 0; i < w.tiles && ok; ++i) {
            const int it = kSparse ? w.done + i : i, s = it & 1;
            const bool more = i + 1 < w.tiles;
            // Operands first, which are early: nothing but the products is then between probabilities and scores.
            ok = wait(&v_full[s], (it >> 1) & 1) && (!more || wait(&k_full[s ^ 1], ((it + 1) >> 1) & 1)) &&
                 wait(&p_full[m], (kSparse ? w.row_done[m] + i : i) & 1);
            if (!ok) break;
            tc_fence_after();
            if (more) first_half(s ^ 1);
            const uint32_t p_tmem = s_tmem + s * (kTokens / 2);
#pragma unroll
            for (int k = 0; k < kTokens / 16; ++k) {  // 16 tokens
              const uint32_t at = ((k >> 2) * (kDim * 128) + (k & 3) * 32) >> 4;
              mma_ts(leader, o_tmem, p_tmem + 8 * (k ^ (4 * s)), v_desc + (s * L::kTileBytes >> 4) + at, kInstrO, i > 0 || k > 0);
            }
            commit_both(&v_empty[s]);
            if (more) other_half(s ^ 1);
          }
          if (ok) mma_commit(leader, o_full);
        }
        __syncwarp();
      } while (next_list(false));
    }
  }
  __syncwarp();
  // After a wait was given up, products under way end by themselves: time for that before the tensor memory is freed.
  if (warp >= kMmaWarp && *abort_flag) {
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 2000000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Adds the parts of the segments that a line's ranges cut, a block to a range, in which one starts that ends in another, and a
// share of its rows: a warp has a row, the parts come in their order.
constexpr int kJoinWarps = 8;
constexpr int kJoinShares = 16;
template <class T, int kDim>
__global__ void __launch_bounds__(kJoinWarps * 32) kv4_chunk_join_kernel(Kv4Attend a, uint32_t shared, int64_t blocks) {
  constexpr int kPer = kDim / 32;
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Cut w = static_cast<const Cut*>(a.workspace)[blockIdx.x];
  const int64_t c0 = blockIdx.x, c1 = c0 + w.parts - 1;
  const float* const base = chunk_parts(a, blocks);
  for (int r = blockIdx.y * kJoinWarps + warp; r < (w.parts > 1 ? w.row_count : 0); r += kJoinShares * kJoinWarps) {
    float m = -INFINITY, sum = 0.0F, v[kPer];
#pragma unroll
    for (int d = 0; d < kPer; ++d) v[d] = 0.0F;
    for (int64_t k = c0; k <= c1; ++k) {
      const float* const part = base + (2 * k + (k == c0 ? 1 : 0)) * partial_floats(kBlockRows, kDim);
      const float2 st = *reinterpret_cast<const float2*>(part + kBlockRows * kDim + 2 * r);
      if (st.y == 0.0F) continue;  // the part's tiles had nothing for the row: its sums may not have been written
      float x[kPer];
      if constexpr (kPer == 2) *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(part + r * kDim + lane * kPer);
      else *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(part + r * kDim + lane * kPer);
      const float next = fmaxf(m, st.x), old = fade_to(m, next), f = fade_to(st.x, next);
      m = next;
      sum = sum * old + f * st.y;
#pragma unroll
      for (int d = 0; d < kPer; ++d) v[d] = v[d] * old + f * x[d];
    }
    const float inv = sum == 0.0F ? 0.0F : 1.0F / sum;
    const uint32_t token = (w.block_row0 + r) / shared, in_group = w.block_row0 + r - token * shared;
    const int64_t at = (w.row0 + token) * a.heads + w.head * shared + in_group;
    T* const out = static_cast<T*>(a.out) + at * kDim + lane * kPer;
#pragma unroll
    for (int d = 0; d < kPer; ++d) out[d] = from_f32<T>(v[d] * inv);
    if (a.lse && lane == 0) a.lse[at] = sum == 0.0F ? -INFINITY : ((m == -INFINITY ? 0.0F : m - kLift) + __log2f(sum)) * 0.693147181F;
  }
}

// Blocks of a line: one an SM, and no more than there can be tiles.
int64_t line_blocks(const Kv4View& c, const Kv4Attend& a) {
  const int64_t row_blocks = (static_cast<int64_t>(a.max_rows) * (a.heads / c.heads) + kBlockRows - 1) / kBlockRows;
  const int64_t tiles = std::max<int64_t>(1, ((static_cast<int64_t>(a.max_pages) << c.page_shift) + kTokens - 1) / kTokens);
  const int64_t segments = row_blocks * a.batch * c.heads;
  return segments >= sm_count() ? sm_count() : std::min<int64_t>(sm_count(), segments * tiles);
}

template <class T, int kDim, bool kSparse>
void launch_dim(const Kv4View& c, const Kv4Attend& given, cudaStream_t stream) {
  Kv4Attend a = given;
  keep_sums_finite(a, c.page_shift, kLift);
  const int shared = a.heads / c.heads;
  const int64_t row_blocks = (static_cast<int64_t>(a.max_rows) * shared + kBlockRows - 1) / kBlockRows;
  const int64_t blocks = kSparse ? line_blocks(c, a) : row_blocks * a.batch * c.heads;
  if (row_blocks * a.batch * c.heads > INT_MAX) throw InvalidArgument("batch * heads * query rows are too many for one call");
  const uint64_t starts = reinterpret_cast<uintptr_t>(a.query) | static_cast<uint64_t>(a.q_row_stride) * sizeof(T) |
                          static_cast<uint64_t>(a.q_head_stride) * sizeof(T);
  allow_dynamic_shared<kv4_chunk_kernel<T, kDim, kSparse>>(Layout<kDim>::kBytes, "shared memory of the chunk attention kernel");
  if constexpr (kSparse) {
    launch_early(kv4_chunk_kernel<T, kDim, true>, dim3(static_cast<unsigned>(blocks)), kLineThreads, Layout<kDim>::kBytes, stream, 0,
                 "launch chunk attention kernel", c, a, static_cast<uint32_t>(shared), static_cast<int>(row_blocks), (starts & 15) == 0);
    if (blocks > 1)
      launch_early(kv4_chunk_join_kernel<T, kDim>, dim3(static_cast<unsigned>(blocks - 1), kJoinShares), kJoinWarps * 32, 0, stream, 0,
                   "launch chunk attention join kernel", a, static_cast<uint32_t>(shared), blocks);
  } else {
    kv4_chunk_kernel<T, kDim, false><<<static_cast<unsigned>(blocks), kThreads, Layout<kDim>::kBytes, stream>>>(
        c, a, shared, static_cast<int>(row_blocks), (starts & 15) == 0);
    count_launch();
    check(cudaGetLastError(), "launch chunk attention kernel");
  }
}

template <class T>
void launch_typed(const Kv4View& c, const Kv4Attend& a, cudaStream_t stream) {
  const bool sparse = a.sinks > 0 || a.ancestors;
  if (c.dim == 64) sparse ? launch_dim<T, 64, true>(c, a, stream) : launch_dim<T, 64, false>(c, a, stream);
  else sparse ? launch_dim<T, 128, true>(c, a, stream) : launch_dim<T, 128, false>(c, a, stream);
}

}  // namespace

// Head dimension 256 would need 768 columns of tensor memory.
bool kv4_chunk_supported(const Kv4View& c) { return c.dim <= 128; }

size_t kv4_chunk_workspace_bytes(const Kv4View& c, const Kv4Attend& a) {
  if (a.sinks == 0 && !a.ancestors) return 0;
  return cut_bytes(line_blocks(c, a)) + sizeof(float) * 2 * static_cast<size_t>(line_blocks(c, a)) * partial_floats(kBlockRows, c.dim);
}

void launch_kv4_chunk(const Kv4View& c, const Kv4Attend& a, cudaStream_t stream) {
  if (a.type == kElemF16) launch_typed<__half>(c, a, stream);
  else launch_typed<__nv_bfloat16>(c, a, stream);
}

}  // namespace msb
