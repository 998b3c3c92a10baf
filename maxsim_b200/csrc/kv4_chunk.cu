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
//   172 us on the device, 174 to 176 with the host's call (12 us more before the scores were formed in halves, below).  A
//   tile of 256 rows takes about 5,000 cycles, of which the exponentials need 2,048 and the products as much: what bounds
//   it is the softmax warps' chain of loads, conversions and stores, 1,000 cycles and more for 32 columns whatever waits
//   beside it.  Half of the issue slots are used.  Reading the queries takes 8,000 cycles of a block and writing the rows
//   5,000.  And the blocks' order: 256 of them start by row block, then by sequence, whatever their length.  Replayed on
//   148 SMs from these cycles that ends after 153 to 156 us; longest first would end after 116, evenly spread after 105.
// Every wait is bounded; a block that gives up writes NaN rows.
#include <algorithm>
#include <climits>

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
  static constexpr int off_bars = off_rows + kBlockRows * 4;
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
  int first[2];       // of sparse rows: the first one,
  int sinks;          // those before it that are seen too,
  uint32_t bits[2];   // and of the 32 columns at hand those that the row sees whatever else (a tree of drafted tokens)
  float top[2];       // the reference, -inf before there is one
};

// Whether row r does not see token c, the j-th column of its lane's eight (of four lanes') of a block.
template <bool kSparse>
__device__ __forceinline__ bool not_seen(const Rows& rows, int r, int c, int column) {
  if constexpr (!kSparse) return c > rows.last[r] || rows.last[r] - c >= rows.window;
  const bool run = c <= rows.last[r] && (c >= rows.first[r] || c < rows.sinks);
  return !run && !((rows.bits[r] >> column) & 1u);
}
// Scores (f: two rows x 8 columns) to probabilities times value scales, fp16 pairs; the largest into `most`.
template <bool kMasked, bool kSparse>
__device__ __forceinline__ void probabilities(const float (&f)[16], const float* meta, int j0, const Rows& rows, uint32_t (&p)[8],
                                              float2 (&add)[2], float (&most)[2]) {
  add[0] = add[1] = make_float2(0.0F, 0.0F);
  most[0] = most[1] = 0.0F;
#pragma unroll
  for (int j = 0; j < kCols / 8; j += 2) {
    const float4 ks4 = *reinterpret_cast<const float4*>(meta + 2 * j);
    const float4 vs4 = *reinterpret_cast<const float4*>(meta + kMetaFloats + 2 * j);
    float4 e4 = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
    if (kMasked) e4 = *reinterpret_cast<const float4*>(meta + 2 * kMetaFloats + 2 * j);
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
          const int column = 8 * (j + h) + 2 * (threadIdx.x & 3);
          if (e.x == -INFINITY || not_seen<kSparse>(rows, r, c, column)) pr.x = pv.x = 0.0F;
          if (e.y == -INFINITY || not_seen<kSparse>(rows, r, c + 1, column + 1)) pr.y = pv.y = 0.0F;
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
__device__ __forceinline__ void references(const float (&f)[16], const float* meta, int j0, const Rows& rows, float (&best)[2]) {
  best[0] = best[1] = -INFINITY;
#pragma unroll
  for (int j = 0; j < kCols / 8; ++j)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float ks = meta[2 * j + k], e = meta[2 * kMetaFloats + 2 * j + k];
      const int c = j0 + 8 * j + k;
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (e != -INFINITY && !not_seen<kSparse>(rows, r, c, 8 * j + k + 2 * (threadIdx.x & 3)))
          best[r] = fmaxf(best[r], f[4 * j + 2 * r + k] * ks * rows.factor[r].x + e);
    }
}

// Whether token j's value is a vector of zeros.  Out of line: in the unpacking warps' loop it cost 5 us of 170.
template <int kDim>
__device__ __noinline__ bool zero_value(const uint8_t* codes, const int32_t* pages, int heads, int head, int page_shift, int j) {
  const int64_t page = __ldg(pages + (j >> page_shift));
  return zero_codes<kDim>(codes + (((page * heads + head) << page_shift) + (j & ((1 << page_shift) - 1))) * (kDim / 2));
}

// kSparse: rows that see sinks past their window, or a tree of drafted tokens (kv4_seen): tiles over the sinks come first.
template <class T, int kDim, bool kSparse>
__global__ void __launch_bounds__(kThreads, 1) kv4_chunk_kernel(Kv4View c, Kv4Attend a, uint32_t shared, int row_blocks,
                                                                bool aligned) {
  using L = Layout<kDim>;
  extern __shared__ unsigned char raw_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // Later row blocks see more tokens under a causal mask: they start first.
  const int64_t per_block = static_cast<int64_t>(a.batch) * c.heads;
  const int block = row_blocks - 1 - static_cast<int>(blockIdx.x / per_block);
  const int b = static_cast<int>(blockIdx.x % per_block / c.heads), head = static_cast<int>(blockIdx.x % c.heads);
  const Kv4Sequence q = kv4_sequence(a, c.page_shift, b);
  const uint32_t all_rows = static_cast<uint32_t>(q.rows) * shared, block_row0 = static_cast<uint32_t>(block) * kBlockRows;  // below 2^31
  const int share = block * c.heads + head, shares = row_blocks * c.heads;  // of the sequence's blocks
  if (block_row0 >= all_rows) {
    if (a.fill) kv4_fill_rows<T>(a, kDim, b, q, share, shares, threadIdx.x, kThreads);
    return;
  }
  const int row_count = static_cast<int>(min(static_cast<uint32_t>(kBlockRows), all_rows - block_row0));
  const int tiles_m = row_count > kRowsTile ? 2 : 1;
  // Tokens that some row of the block sees, and the tiles over them.
  const int pos0 = q.pos0 + static_cast<int>(block_row0 / shared);
  const int pos1 = q.pos0 + static_cast<int>((block_row0 + row_count - 1) / shared);
  const bool tree = kSparse && a.ancestors != nullptr;
  const int any_last = a.causal && !tree ? pos1 : q.length - 1;
  // (Rows before the sequence's first token have negative positions; less a window these would pass 32 bits.)
  const int any_first = a.window > 0 ? max(0, max(0, tree ? q.pos0 - 1 : pos0) - a.window + 1) : 0;
  int begin = any_first & ~15;
  // The tiles over the sinks; where these reach the window, all is one run.
  int front = 0;
  if constexpr (kSparse) {
    front = a.window > 0 ? (a.sinks + kTokens - 1) / kTokens : 0;
    if (front * kTokens >= begin) front = begin = 0;
  }
  const int tiles = any_last >= any_first ? front + (any_last - begin) / kTokens + 1 : 0;
  auto tile_start = [&](int i) { return kSparse && i < front ? i * kTokens : begin + (i - front) * kTokens; };

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
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&k_empty[s], tiles_m);
      mbar_init(&v_full[s], 4);
      mbar_init(&v_empty[s], tiles_m);
      mbar_init(&meta_empty[s], 8 * tiles_m);
    }
    for (int m = 0; m < 2; ++m) {
      mbar_init(&s_half[m], 1);
      mbar_init(&s_full[m], 1);
      mbar_init(&p_full[m], 8);
    }
    mbar_init(o_full, tiles_m);
    mbar_init(q_full, 8 * tiles_m);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
  // Tensor memory: scores of the row tiles at columns 0 and 128 (probabilities over them), sums at 256 and 384.
  // Half h of a tile's scores, 64 tokens, is in columns 64 h and on.  Of tile i the half i % 2 comes first and the
  // probabilities of both go to its columns, so that the other half's are free for the half of tile i + 1 that
  // comes first: its product does not wait for this tile's sums, nor its softmax.

  const int32_t* const pages = a.page_table + b * a.table_stride;
  const int page_mask = (1 << c.page_shift) - 1;
  // Vector of token j's 16-token group on page p (-1: none), and whether the page is the cache's.
  auto ask_page = [&](int j) { return j <= any_last ? __ldg(pages + (j >> c.page_shift)) : -1; };
  auto vector_of = [&](int page, int j) {
    return static_cast<uint32_t>(page) < static_cast<uint32_t>(c.num_pages)
               ? (static_cast<int64_t>(static_cast<uint32_t>(page) * c.heads + head) << c.page_shift) + (j & page_mask)
               : int64_t{0};
  };

  if (warp < kSoftWarps) {
    // =================== softmax: a warp has 16 rows, a thread two of them and a quarter of their columns ===================
    const int m = warp >> 3;
    if (m < tiles_m) {
      const int row0 = (warp & 3) * 32 + ((warp >> 2) & 1) * 16;  // of the row tile, and its lane of tensor memory
      float* const row_factor = reinterpret_cast<float*>(smem + L::off_rows) + m * kRowsTile + row0;
      constexpr int kRowLanes = kDim / 8, kRowsAtOnce = 32 / kRowLanes, kLoads = 16 / kRowsAtOnce;
      // The warp's rows of the query tile, 8 dimensions a lane: scaled by a power of two to a maximum in [2^10, 2^11),
      // fp16, in the codes' order.  (In a loop: straight code would be fetched from memory and used once.)
      constexpr int kBatch = 4;
#pragma unroll 1
      for (int k0 = 0; k0 < kLoads; k0 += kBatch) {
        uint4 x[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int r = m * kRowsTile + row0 + (k0 + k) * kRowsAtOnce + lane / kRowLanes;
          x[k] = make_uint4(0, 0, 0, 0);
          if (r < row_count) {
            const uint32_t token = (block_row0 + r) / shared, in_group = block_row0 + r - token * shared;
            const T* src = static_cast<const T*>(a.query) + (q.row0 + token) * a.q_row_stride +
                           static_cast<int64_t>(head * shared + in_group) * a.q_head_stride + (lane % kRowLanes) * 8;
            if (aligned) {
              x[k] = __ldg(reinterpret_cast<const uint4*>(src));
            } else {
              __align__(16) T e[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) e[i] = src[i];
              x[k] = *reinterpret_cast<const uint4*>(e);
            }
          }
        }
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
          const int r = (k0 + k) * kRowsAtOnce + lane / kRowLanes, piece = lane % kRowLanes;
          store16(base + L::off_q + m * L::kQBytes + (piece >> 3) * (kRowsTile * 128) + swizzled(row0 + r, piece & 7),
                  pack_half2(to_f32(v[0]) * down, to_f32(v[4]) * down), pack_half2(to_f32(v[1]) * down, to_f32(v[5]) * down),
                  pack_half2(to_f32(v[2]) * down, to_f32(v[6]) * down), pack_half2(to_f32(v[3]) * down, to_f32(v[7]) * down));
          if (piece == 0) row_factor[r] = a.scale * 1.44269504F * __uint_as_float(static_cast<uint32_t>(127 - 10 + e) << 23);
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);

      Rows rows;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        // Rows past the last do as it does: what they compute is not written.
        const int mine = 8 * k + (lane >> 2), at = min(m * kRowsTile + row0 + mine, row_count - 1);
        const int pos = q.pos0 + static_cast<int>((block_row0 + at) / shared);
        rows.factor[k] = make_float2(row_factor[mine], row_factor[mine]);
        rows.ref[k] = rows.sum[k] = make_float2(0.0F, 0.0F);
        rows.last[k] = a.causal ? pos : q.length - 1;
        rows.top[k] = -INFINITY;
        if constexpr (kSparse) {
          const Kv4Seen seen = kv4_seen(a, q, pos - q.pos0);
          rows.first[k] = seen.first;
          rows.last[k] = seen.last;
          rows.bits[k] = 0;
        }
      }
      rows.sinks = a.sinks;
      rows.window = a.window > 0 ? a.window : INT_MAX;
      const int every_last = min(rows.last[0], rows.last[1]);
      const int every_first = kSparse        ? max(rows.first[0], rows.first[1])
                              : a.window > 0 ? max(0, max(rows.last[0], rows.last[1])) - a.window + 1
                                             : 0;
      const uint32_t s_at = tmem + (static_cast<uint32_t>(row0) << 16) + m * 128, o_at = s_at + 256;
      bool ok = true;
      for (int i = 0; i < tiles; ++i) {
        const int s = i & 1, j0 = tile_start(i);
        ok = mbar_wait(&k_full[s], (i >> 1) & 1, abort_flag) && mbar_wait(&s_half[m], i & 1, abort_flag);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint4 flag = *reinterpret_cast<const uint4*>(flags + 4 * s);
        const bool masked = __any_sync(0xFFFFFFFFu, (flag.x | flag.y | flag.z | flag.w) != 0u || j0 < every_first ||
                                                       j0 + kTokens - 1 > every_last);
        const uint32_t p_at = s_at + s * (kTokens / 2);
        // Blocks of 32 columns in one short loop: its instructions stay near, the other three warps of a scheduler
        // fill its waits.
#pragma unroll 1
        for (int part = 0; part < kTokens / kCols; ++part) {
          const int piece = part ^ (2 * s);  // the block of columns
          const float* const my_meta = meta + s * 3 * kMetaFloats + (4 * piece + (lane & 3)) * kMetaPitch;
          const int my_j0 = j0 + kCols * piece + 2 * (lane & 3);
          if (part == kTokens / kCols / 2) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s_full[m], i & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
          }
          if (tree && masked) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int at = min(m * kRowsTile + row0 + 8 * k + (lane >> 2), row_count - 1);
              rows.bits[k] = kv4_tree_bits(a, q, static_cast<int>((block_row0 + at) / shared), j0 + kCols * piece);
            }
          }
          float f[16], most[2];
          float2 add[2];
          uint32_t p[8];
          tmem_ld_block(s_at + kCols * piece, f);
          if (masked) probabilities<true, kSparse>(f, my_meta, my_j0, rows, p, add, most);
          else probabilities<false, kSparse>(f, my_meta, my_j0, rows, p, add, most);
          // A row without a reference yet, or one whose reference has become too low: for p vs, or for p, which value
          // scales near zero let grow unseen by p vs (an infinite p among either).
          const float weights = fmax3(fmaxf(add[0].x, add[0].y), add[1].x, add[1].y);
          const bool low = fminf(rows.top[0], rows.top[1]) == -INFINITY || fmaxf(most[0], most[1]) > kMostP || weights > a.most_weight;
          if (__any_sync(0xFFFFFFFFu, low)) {
            tmem_wait_st();  // what was written before is read below, the sums of the tiles before too
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s_full[m], i & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            float best[2], fade[2];
            tmem_ld_block(s_at + kCols * piece, f);
            references<kSparse>(f, my_meta, my_j0, rows, best);
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
            probabilities<true, kSparse>(f, my_meta, my_j0, rows, p, add, most);
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
        }
        if (!ok) break;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&p_full[m]);
          mbar_arrive(&meta_empty[s]);
        }
      }
      // The rows' outputs, through the query tile's shared memory to 16 bytes a lane.
      if (ok && tiles > 0) ok = mbar_wait(o_full, 0, abort_flag);
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
#pragma unroll 1
      for (int d = 0; d < kDim; d += kCols) {
        float f[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) f[k] = 0.0F;
        if (ok && tiles > 0) tmem_ld_block(o_at + d, f);
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
        if (r >= row_count) continue;
        const uint32_t token = (block_row0 + r) / shared, in_group = block_row0 + r - token * shared;
        const int64_t out_row = (q.row0 + token) * a.heads + head * shared + in_group;
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
          if (r >= row_count) continue;
          const uint32_t token = (block_row0 + r) / shared, in_group = block_row0 + r - token * shared;
          const float reference = rows.top[k] == -INFINITY ? 0.0F : rows.top[k] - kLift;
          a.lse[(q.row0 + token) * a.heads + head * shared + in_group] =
              !ok ? NAN : sum[k] == 0.0F ? -INFINITY : (reference + __log2f(sum[k])) * 0.693147181F;
        }
      }
    }
  } else if (warp < kMmaWarp) {
    // =================== unpacking ===================
    // Keys: lane (g, t) takes 16 bytes t (at D = 128) of tokens g, g + 8, .. of its warp's 32.
    const int uw = warp - kUnpackWarp0, g = lane >> 2, t = lane & 3;
    constexpr int kWords = kDim / 32;                       // of a token, per lane
    uint32_t word[4][kWords];
    float ks = 0.0F, vs = 0.0F;
    bool seen = false;
    int page[2] = {ask_page(tile_start(0) + 32 * uw), ask_page(tile_start(0) + 32 * uw + 16)};
    auto load_keys = [&](int i) {
      const int j = tile_start(i) + 32 * uw;
      const int64_t v[2] = {vector_of(page[0], j), vector_of(page[1], j + 16)};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint8_t* src = c.codes[0] + (v[k >> 1] + 8 * (k & 1) + g) * (kDim / 2) + t * (kDim / 8);
        if constexpr (kWords == 4) {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(src));
          word[k][0] = u.x, word[k][1] = u.y, word[k][2] = u.z, word[k][3] = u.w;
        } else {
          const uint2 u = __ldg(reinterpret_cast<const uint2*>(src));
          word[k][0] = u.x, word[k][1] = u.y;
        }
      }
      const int mine = j + lane;
      const int64_t at = (lane < 16 ? v[0] : v[1]) + (lane & 15);
      seen = static_cast<uint32_t>(lane < 16 ? page[0] : page[1]) < static_cast<uint32_t>(c.num_pages) &&
             (mine >= any_first || (kSparse && mine < a.sinks)) && mine <= any_last;
      ks = __ldg(c.scales[0] + at);
      vs = __ldg(c.scales[1] + at);
      const int next = kSparse ? tile_start(i + 1) + 32 * uw : j + kTokens;
      page[0] = ask_page(next);
      page[1] = ask_page(next + 16);
    };
    // Values: a lane takes 8 tokens and 8 or 16 dimensions.
    constexpr int kValueWords = kDim / 64;                  // 8-dimension words of a token, per lane
    const int group = (uw >> 1) * 8 + (lane & 7);           // its 8 tokens
    const int piece = (uw & 1) * 4 + (lane >> 3);           // its words: piece * kValueWords and on
    uint32_t value[8][kValueWords];
    int value_page = ask_page(tile_start(0) + (group >> 1) * 16);
    auto load_values = [&](int i) {
      const int j = tile_start(i) + (group >> 1) * 16;
      const uint8_t* src = c.codes[1] + (vector_of(value_page, j) + 8 * (group & 1)) * (kDim / 2) + piece * (4 * kValueWords);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if constexpr (kValueWords == 2) {
          const uint2 u = __ldg(reinterpret_cast<const uint2*>(src + k * (kDim / 2)));
          value[k][0] = u.x, value[k][1] = u.y;
        } else {
          value[k][0] = __ldg(reinterpret_cast<const uint32_t*>(src + k * (kDim / 2)));
        }
      }
      value_page = ask_page(kSparse ? tile_start(i + 1) + (group >> 1) * 16 : j + kTokens);
    };
    if (tiles > 0) {
      load_keys(0);
      load_values(0);
    }
    for (int i = 0; i < tiles; ++i) {
      const int s = i & 1;
      const uint32_t parity = ((i >> 1) - 1) & 1;
      if (i >= kStages) {
        const bool ok = mbar_wait(&k_empty[s], parity, abort_flag) && mbar_wait(&meta_empty[s], parity, abort_flag);
        if (!__all_sync(0xFFFFFFFFu, ok)) break;
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
          zero_value<kDim>(c.codes[1], pages, c.heads, head, c.page_shift, tile_start(i) + 32 * uw + lane))
        vs = 0.0F;
      ms[0] = seen ? ks : 0.0F;
      ms[kMetaFloats] = seen ? vs : 0.0F;
      ms[2 * kMetaFloats] = seen ? scale_exponent(vs, a.least_exponent, most_exponent(kLift)) : -INFINITY;
      const uint32_t all = __ballot_sync(0xFFFFFFFFu, seen);
      if (lane == 0) flags[4 * s + uw] = ~all;
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[s]);
      if (i + 1 < tiles) load_keys(i + 1);

      if (i >= kStages) {
        const bool ok = mbar_wait(&v_empty[s], parity, abort_flag);
        if (!__all_sync(0xFFFFFFFFu, ok)) break;
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
      if (i + 1 < tiles) load_values(i + 1);
    }
    // These warps are done first.
    if (a.fill)
      kv4_fill_rows<T>(a, kDim, b, kv4_sequence(a, c.page_shift, b), share, shares, threadIdx.x - kUnpackWarp0 * 32,
                       (kMmaWarp - kUnpackWarp0) * 32);
  } else if (warp - kMmaWarp < tiles_m && tiles > 0) {
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
    auto first_half = [&](int s) {
      scores(s, s);
      mma_commit(leader, &s_half[m]);
    };
    auto other_half = [&](int s) {
      scores(s, s ^ 1);
      mma_commit(leader, &s_full[m]);
      mma_commit(leader, &k_empty[s]);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag)) != 0;
    };
    bool ok = wait(q_full, 0) && wait(&k_full[0], 0);
    if (ok) {
      tc_fence_after();
      first_half(0);
      other_half(0);
    }
    for (int i = 0; i < tiles && ok; ++i) {
      const int s = i & 1;
      const bool more = i + 1 < tiles;
      // Operands first, which are early: nothing but the products is then between probabilities and scores.
      ok = wait(&v_full[s], (i >> 1) & 1) && (!more || wait(&k_full[s ^ 1], ((i + 1) >> 1) & 1)) && wait(&p_full[m], i & 1);
      if (!ok) break;
      tc_fence_after();
      if (more) first_half(s ^ 1);
      const uint32_t p_tmem = s_tmem + s * (kTokens / 2);
#pragma unroll
      for (int k = 0; k < kTokens / 16; ++k) {  // 16 tokens
        const uint32_t at = ((k >> 2) * (kDim * 128) + (k & 3) * 32) >> 4;
        mma_ts(leader, o_tmem, p_tmem + 8 * (k ^ (4 * s)), v_desc + (s * L::kTileBytes >> 4) + at, kInstrO, i > 0 || k > 0);
      }
      mma_commit(leader, &v_empty[s]);
      if (more) other_half(s ^ 1);
    }
    if (ok) mma_commit(leader, o_full);
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

template <class T, int kDim, bool kSparse>
void launch_dim(const Kv4View& c, const Kv4Attend& given, cudaStream_t stream) {
  Kv4Attend a = given;
  keep_sums_finite(a, c.page_shift, kLift);
  const int shared = a.heads / c.heads;
  const int64_t row_blocks = (static_cast<int64_t>(a.max_rows) * shared + kBlockRows - 1) / kBlockRows;
  const int64_t blocks = row_blocks * a.batch * c.heads;
  if (blocks > INT_MAX) throw InvalidArgument("batch * heads * query rows are too many for one call");
  const uint64_t starts = reinterpret_cast<uintptr_t>(a.query) | static_cast<uint64_t>(a.q_row_stride) * sizeof(T) |
                          static_cast<uint64_t>(a.q_head_stride) * sizeof(T);
  allow_dynamic_shared<kv4_chunk_kernel<T, kDim, kSparse>>(Layout<kDim>::kBytes, "shared memory of the chunk attention kernel");
  kv4_chunk_kernel<T, kDim, kSparse><<<static_cast<unsigned>(blocks), kThreads, Layout<kDim>::kBytes, stream>>>(
      c, a, shared, static_cast<int>(row_blocks), (starts & 15) == 0);
  count_launch();
  check(cudaGetLastError(), "launch chunk attention kernel");
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

void launch_kv4_chunk(const Kv4View& c, const Kv4Attend& a, cudaStream_t stream) {
  if (a.type == kElemF16) launch_typed<__half>(c, a, stream);
  else launch_typed<__nv_bfloat16>(c, a, stream);
}

}  // namespace msb
