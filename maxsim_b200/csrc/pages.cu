// Page tables of the 4-bit key/value cache, kept on the device: pages taken from a stack of free ones as sequences
// grow, given back as they shrink, and the slots and positions of a step's rows; and the masks of drafted trees.
//
// extend.  With L_b tokens held, n_b = max(tokens_b, 0) new ones and pages of P tokens, sequence b holds
// have_b = ceil(L_b / P) pages and wants ceil((L_b + n_b) / P).  Its rows are E_b .. E_b + n_b of the step, E the
// exclusive sums of n.  Of the sequences whose pages fit their row of the table and whose rows fit the step, U_b is the
// inclusive sum of the pages they lack; b is served where it lacks none or U_b <= free.  Its page of column c >= have_b
// is entry free - 1 - (U_b - lacks_b + c - have_b) of the stack.  Row i of b is at position L_b + i.
// truncate.  Pages past ceil(L'_b / P) go back, the first sequence's first one on top: what extend took lies as before.
//   Bound: latency.  One block forms the sums (plan); where rows or sequences are many a second kernel with four rows (or a
//   page given back) to a thread does the rest, launched early, else the same block does it, from shared memory.
//   A row whose position starts a page enters that page in the table: each new page has one such row.
//   Measured on the device: a token for each of 64 sequences, and back, 5.9 us; 128,000 rows of 500 sequences in 8,000 new
//   pages, and back, 12.7 us (launch_pages_extend has what chooses between the forms).
#include <cooperative_groups.h>

#include <algorithm>

#include "pages.cuh"

namespace msb {
namespace {

constexpr int kMostThreads = 1024;
constexpr int kSmall = 1024;      // sequences that one block keeps in shared memory
constexpr int kSmallRows = 8192;  // rows that a cluster does by itself
constexpr int kRowThreads = 256;
constexpr int kRows = 4;          // rows of a thread

// What the sums leave for the rows: of each sequence the row (or page) where it starts, its length before (-1: refused)
// and its first entry of the stack.
struct Plan {
  int64_t* start;   // [sequences + 1]
  int32_t* length;  // [sequences]
  int32_t* entry;   // [sequences]
};
__host__ __device__ __forceinline__ size_t plan_bytes(int64_t sequences) {
  return static_cast<size_t>(sequences + 1) * 8 + static_cast<size_t>(sequences) * 8;
}
__host__ __device__ __forceinline__ Plan plan_at(void* p, int64_t sequences) {
  Plan r;
  r.start = static_cast<int64_t*>(p);
  r.length = reinterpret_cast<int32_t*>(r.start + sequences + 1);
  r.entry = r.length + sequences;
  return r;
}

// Inclusive sums of two numbers over the block; the block's totals too.
struct Two {
  int64_t a, b;
};
template <int kThreads>
__device__ __forceinline__ Two block_sum(Two v, Two* scratch, Two& total) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t oa = __shfl_up_sync(0xFFFFFFFFu, v.a, d), ob = __shfl_up_sync(0xFFFFFFFFu, v.b, d);
    if (lane >= d) v.a += oa, v.b += ob;
  }
  __syncthreads();  // the sums before have been read
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  Two s = lane < kWarps ? scratch[lane] : Two{0, 0};
#pragma unroll
  for (int d = 1; d < kWarps; d <<= 1) {
    const int64_t oa = __shfl_up_sync(0xFFFFFFFFu, s.a, d), ob = __shfl_up_sync(0xFFFFFFFFu, s.b, d);
    if (lane >= d) s.a += oa, s.b += ob;
  }
  total = Two{__shfl_sync(0xFFFFFFFFu, s.a, kWarps - 1), __shfl_sync(0xFFFFFFFFu, s.b, kWarps - 1)};
  const int64_t ba = __shfl_sync(0xFFFFFFFFu, s.a, max(0, warp - 1)), bb = __shfl_sync(0xFFFFFFFFu, s.b, max(0, warp - 1));
  return warp > 0 ? Two{v.a + ba, v.b + bb} : v;
}

__device__ __forceinline__ int64_t held_length(const Pages& p, int b) {
  return max(int64_t{0}, min(static_cast<int64_t>(p.lengths[b]), static_cast<int64_t>(p.max_pages) << p.page_shift));
}
__device__ __forceinline__ int64_t pages_of(const Pages& p, int64_t tokens) {
  return (tokens + (int64_t{1} << p.page_shift) - 1) >> p.page_shift;
}
__device__ __forceinline__ int64_t free_pages(const Pages& p) {
  return max(int64_t{0}, min(static_cast<int64_t>(*p.free_count), p.num_pages));
}
// The sequence that holds `at`: the last whose start is not past it (some start is).
__device__ __forceinline__ int sequence_of(const int64_t* start, int sequences, int64_t at) {
  int lo = 0, hi = sequences;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= at) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Forms the plan; reads the state only.  What is taken from the stack comes back.
template <int kThreads>
__device__ __forceinline__ int extend_plan(const Pages& p, const PagesExtend& e, const Plan& plan, Two* scratch, int64_t free) {
  __shared__ int taken;
  if (threadIdx.x == 0) taken = 0;
  Two before{0, 0};  // rows, pages
  for (int b0 = 0; b0 < p.sequences; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int64_t length = 0, n = 0;
    if (b < p.sequences) {
      length = held_length(p, b);
      n = max(0, e.tokens[b]);
    }
    const int64_t have = pages_of(p, length), want = pages_of(p, length + n);
    bool fits = want <= p.max_pages;
    int64_t lacks = fits ? want - have : 0;
    Two total, upto = block_sum<kThreads>(Two{n, lacks}, scratch, total);
    const int64_t end = before.a + upto.a;
    if (before.a + total.a > e.rows) {  // rows run out: whose do not fit asks for no pages
      fits = fits && end <= e.rows;
      lacks = fits ? lacks : 0;
      Two again;
      upto.b = block_sum<kThreads>(Two{0, lacks}, scratch, again).b;
      total.b = again.b;
    }
    const int64_t pages = before.b + upto.b;
    const bool served = fits && (lacks == 0 || pages <= free);
    if (b < p.sequences) {
      plan.start[b] = end - n;
      plan.length[b] = served ? static_cast<int32_t>(length) : -1;
      plan.entry[b] = static_cast<int32_t>(max(int64_t{0}, free - 1 - (pages - lacks)));
      // Those that lack pages and are served are the first that lack some: the largest of their sums is all that is taken.
      if (served && lacks > 0) atomicMax(&taken, static_cast<int>(pages));
    }
    before.a += total.a;
    before.b += total.b;
  }
  if (threadIdx.x == 0) plan.start[p.sequences] = before.a;
  __syncthreads();
  return taken;
}
// The new state and the rows' starts, once every block has read the old one.
template <int kThreads>
__device__ __forceinline__ void extend_state(const Pages& p, const PagesExtend& e, const Plan& plan, int64_t free, int taken) {
  for (int b = threadIdx.x; b <= p.sequences; b += kThreads) {
    const int64_t start = plan.start[b];
    e.offsets[b] = static_cast<int32_t>(min(start, e.rows));
    if (b == p.sequences) break;
    const int64_t n = plan.start[b + 1] - start;
    if (plan.length[b] >= 0 && n > 0) p.lengths[b] = static_cast<int32_t>(plan.length[b] + n);
  }
  if (threadIdx.x == 0) *p.free_count = static_cast<int32_t>(free - taken);
}

// Slot and position of a row of sequence b (which starts at `start`).
__device__ __forceinline__ void place_row(const Pages& p, const Plan& plan, int b, int64_t start, int64_t row, int64_t& slot,
                                          int32_t& position) {
  slot = -1;
  position = -1;
  const int32_t length = plan.length[b];
  if (length < 0) return;
  position = static_cast<int32_t>(length + (row - start));
  const int column = position >> p.page_shift, have = static_cast<int>(pages_of(p, length));
  const int at = position & ((1 << p.page_shift) - 1);
  int32_t* const cell = p.table + static_cast<int64_t>(b) * p.max_pages + column;
  int32_t page;
  if (column < have) {
    page = *cell;
  } else {
    page = p.free[max(0, plan.entry[b] - (column - have))];
    if (at == 0) *cell = page;
  }
  if (page >= 0) slot = (static_cast<int64_t>(page) << p.page_shift) + at;
}

// kRows consecutive rows.
__device__ __forceinline__ void place_rows(const Pages& p, const PagesExtend& e, const Plan& plan, int64_t row0) {
  const int64_t all = plan.start[p.sequences];
  int b = row0 < all ? sequence_of(plan.start, p.sequences, row0) : 0;
  int64_t slot[kRows];
  int32_t position[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    slot[k] = -1;
    position[k] = -1;
    if (row0 + k >= all) continue;
    while (row0 + k >= plan.start[b + 1]) ++b;
    place_row(p, plan, b, plan.start[b], row0 + k, slot[k], position[k]);
  }
  if (row0 + kRows <= e.rows) {  // arrays of rows start on 16 bytes
    reinterpret_cast<longlong2*>(e.slots + row0)[0] = make_longlong2(slot[0], slot[1]);
    reinterpret_cast<longlong2*>(e.slots + row0)[1] = make_longlong2(slot[2], slot[3]);
    *reinterpret_cast<int4*>(e.positions + row0) = make_int4(position[0], position[1], position[2], position[3]);
  } else {
#pragma unroll
    for (int k = 0; k < kRows; ++k)
      if (row0 + k < e.rows) e.slots[row0 + k] = slot[k], e.positions[row0 + k] = position[k];
  }
}

// Up to kSmall sequences: every block of a cluster (or one block) forms the same plan, and has its share of the rows.
template <int kThreads, bool kCluster>
__global__ void __launch_bounds__(kThreads) extend_kernel(Pages p, PagesExtend e) {
  constexpr int kMost = kCluster ? kSmall : kThreads;
  __shared__ __align__(8) unsigned char plan_memory[(kMost + 1) * 8 + kMost * 8];
  __shared__ Two scratch[kThreads / 32];
  const Plan plan = plan_at(plan_memory, p.sequences);
  wait_for_previous();
  let_next_start();
  const int64_t free = free_pages(p);
  const int taken = extend_plan<kThreads>(p, e, plan, scratch, free);
  if constexpr (kCluster) cooperative_groups::this_cluster().sync();
  if (blockIdx.x == 0) extend_state<kThreads>(p, e, plan, free, taken);
  if constexpr (kCluster) {
    for (int64_t row = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * kRows; row < e.rows;
         row += static_cast<int64_t>(gridDim.x) * kThreads * kRows)
      place_rows(p, e, plan, row);
  } else {  // few rows: one a thread
    const int64_t all = plan.start[p.sequences];
    for (int64_t row = threadIdx.x; row < e.rows; row += kThreads) {
      int64_t slot = -1;
      int32_t position = -1;
      if (row < all) {
        const int b = sequence_of(plan.start, p.sequences, row);
        place_row(p, plan, b, plan.start[b], row, slot, position);
      }
      e.slots[row] = slot;
      e.positions[row] = position;
    }
  }
}
__global__ void __launch_bounds__(kMostThreads) extend_plan_kernel(Pages p, PagesExtend e) {
  __shared__ Two scratch[kMostThreads / 32];
  wait_for_previous();
  let_next_start();
  const Plan plan = plan_at(e.workspace, p.sequences);
  const int64_t free = free_pages(p);
  const int taken = extend_plan<kMostThreads>(p, e, plan, scratch, free);
  extend_state<kMostThreads>(p, e, plan, free, taken);
}
__global__ void __launch_bounds__(kRowThreads) extend_rows_kernel(Pages p, PagesExtend e) {
  __shared__ __align__(8) unsigned char plan_memory[(kSmall + 1) * 8 + kSmall * 8];
  Plan plan = plan_at(e.workspace, p.sequences);
  wait_for_previous();
  if (p.sequences <= kSmall) {  // all that the plan has, at once
    const Plan here = plan_at(plan_memory, p.sequences);
    for (int b = threadIdx.x; b < p.sequences; b += kRowThreads) {
      here.start[b] = plan.start[b];
      here.length[b] = plan.length[b];
      here.entry[b] = plan.entry[b];
    }
    if (threadIdx.x == 0) here.start[p.sequences] = plan.start[p.sequences];
    __syncthreads();
    plan = here;
  }
  const int64_t row0 = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) * kRows;
  if (row0 < e.rows) place_rows(p, e, plan, row0);
}

// Forms the plan; reads the state only.
template <int kThreads>
__device__ __forceinline__ void truncate_plan(const Pages& p, const int32_t* to, const Plan& plan, Two* scratch, int64_t free) {
  int64_t before = 0;
  for (int b0 = 0; b0 < p.sequences; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int64_t length = 0, left = 0;
    if (b < p.sequences) {
      length = held_length(p, b);
      left = max(int64_t{0}, min(static_cast<int64_t>(to[b]), length));
    }
    const int64_t keep = pages_of(p, left), back = pages_of(p, length) - keep;
    Two total;
    const int64_t upto = before + block_sum<kThreads>(Two{back, 0}, scratch, total).a;
    if (b < p.sequences) {
      plan.start[b] = upto - back;
      plan.length[b] = static_cast<int32_t>(keep);  // the first column given back
      if (b > 0) plan.entry[b] = static_cast<int32_t>(left);
    }
    before += total.a;
  }
  if (threadIdx.x == 0) {
    plan.start[p.sequences] = before;
    plan.entry[0] = static_cast<int32_t>(free);
  }
  __syncthreads();
}
// The new state, once every block has read the old one.  (The first sequence's length is formed again.)
template <int kThreads>
__device__ __forceinline__ void truncate_state(const Pages& p, const int32_t* to, const Plan& plan, int64_t free) {
  for (int b = threadIdx.x; b < p.sequences; b += kThreads)
    p.lengths[b] =
        b > 0 ? plan.entry[b] : static_cast<int32_t>(max(int64_t{0}, min(static_cast<int64_t>(to[0]), held_length(p, 0))));
  if (threadIdx.x == 0) *p.free_count = static_cast<int32_t>(min(free + plan.start[p.sequences], p.num_pages));
}
// Page k of those given back goes to entry free + all - 1 - k.  A thread (`first` of `step`) has kRows consecutive ones at a
// time: one search, and their cells are asked for together.
__device__ __forceinline__ void truncate_pages(const Pages& p, const Plan& plan, int64_t first, int64_t step) {
  const int64_t all = plan.start[p.sequences], top = plan.entry[0] + all - 1;
  for (int64_t k0 = first * kRows; k0 < all; k0 += step * kRows) {
    int b = sequence_of(plan.start, p.sequences, k0);
    int32_t* cell[kRows];
    int32_t page[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t k = k0 + i;
      if (k >= all) continue;
      while (k >= plan.start[b + 1]) ++b;
      cell[i] = p.table + static_cast<int64_t>(b) * p.max_pages + plan.length[b] + static_cast<int>(k - plan.start[b]);
      page[i] = *cell[i];
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t k = k0 + i;
      if (k >= all) continue;
      if (top - k < p.num_pages) p.free[top - k] = page[i];
      *cell[i] = -1;
    }
  }
}
template <int kThreads, bool kCluster>
__global__ void __launch_bounds__(kThreads) truncate_kernel(Pages p, const int32_t* to) {
  constexpr int kMost = kCluster ? kSmall : kThreads;
  __shared__ __align__(8) unsigned char plan_memory[(kMost + 1) * 8 + kMost * 8];
  __shared__ Two scratch[kThreads / 32];
  const Plan plan = plan_at(plan_memory, p.sequences);
  wait_for_previous();
  let_next_start();
  const int64_t free = free_pages(p);
  truncate_plan<kThreads>(p, to, plan, scratch, free);
  if constexpr (kCluster) cooperative_groups::this_cluster().sync();
  if (blockIdx.x == 0) truncate_state<kThreads>(p, to, plan, free);
  truncate_pages(p, plan, static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, static_cast<int64_t>(gridDim.x) * kThreads);
}
__global__ void __launch_bounds__(kMostThreads) truncate_plan_kernel(Pages p, const int32_t* to, void* workspace) {
  __shared__ Two scratch[kMostThreads / 32];
  wait_for_previous();
  let_next_start();
  const Plan plan = plan_at(workspace, p.sequences);
  const int64_t free = free_pages(p);
  truncate_plan<kMostThreads>(p, to, plan, scratch, free);
  truncate_state<kMostThreads>(p, to, plan, free);
}
__global__ void __launch_bounds__(kRowThreads) truncate_pages_kernel(Pages p, void* workspace) {
  wait_for_previous();
  truncate_pages(p, plan_at(workspace, p.sequences), static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x,
                 static_cast<int64_t>(gridDim.x) * kRowThreads);
}

// Ancestors of the nodes of drafted trees: a block a sequence, its parents in shared memory, a thread a node's
// word of 64 nodes; it walks the node's path up, which ends, as a parent has a lower index.
constexpr int kTreeThreads = 128;
__global__ void __launch_bounds__(kTreeThreads) draft_ancestors_kernel(DraftTrees t) {
  __shared__ int16_t parent[kMostTreeRows];
  wait_for_previous();
  let_next_start();
  const int b = blockIdx.x;
  // Sequences' rows held to the call's; the rows before the first and after the last, and past the announced number, 0.
  const int64_t lo = max(0, t.offsets[b]), hi = min(static_cast<int64_t>(t.offsets[b + 1]), t.rows);
  const int all = static_cast<int>(max(int64_t{0}, hi - lo)), rows = min(all, t.max_rows);
  for (int i = threadIdx.x; i < rows; i += kTreeThreads) {
    const int p = t.parents[lo + i];
    parent[i] = static_cast<int16_t>(p >= 0 && p < i ? p : -1);
  }
  __syncthreads();
  // Words with nodes, and those past them (a caller's rows may be wider, up to 2^24 words: their number passes 32 bits).
  const int words = min(t.words, kMostTreeRows / 64);
  for (int k = threadIdx.x; k < rows * words; k += kTreeThreads) {
    const int i = k / words, word = k - i * words;
    uint64_t bits = 0;
    int depth = -1;
    for (int at = i; at >= 0; at = parent[at]) {
      if (at >> 6 == word) bits |= uint64_t{1} << (at & 63);
      ++depth;
    }
    t.ancestors[(lo + i) * t.words + word] = static_cast<int64_t>(bits);
    if (word == 0) t.depths[lo + i] = depth;
  }
  for (int i = threadIdx.x / 32; i < rows; i += kTreeThreads / 32)
    for (int word = words + threadIdx.x % 32; word < t.words; word += 32) t.ancestors[(lo + i) * t.words + word] = 0;
  auto clear = [&](int64_t from, int64_t to) {
    for (int64_t k = from * t.words + threadIdx.x; k < to * t.words; k += kTreeThreads) t.ancestors[k] = 0;
    for (int64_t i = from + threadIdx.x; i < to; i += kTreeThreads) t.depths[i] = 0;
  };
  clear(lo + rows, lo + all);
  if (b == 0) clear(0, min(lo, t.rows));
  if (b == t.batch - 1) clear(min(lo + all, t.rows), t.rows);
}

}  // namespace

size_t pages_workspace_bytes(const Pages& p, int64_t rows) {
  return p.sequences > kSmall || rows > kSmallRows ? plan_bytes(p.sequences) : 0;
}

// Up to 256 sequences one block of as many threads does it all (extend: up to 1,024 rows): for 64 sequences, a token each,
// 2 us less a call than a cluster.  (How many pages go back the host does not know: some thousand
// at once, which end many long sequences, take a block longer, 11 us for 8,000.)  Up to 1,024 sequences and 8,192 rows a
// cluster: giving back 8,000 pages of 500 sequences 6.9 us.  More, two kernels: 128,000 rows 10 us, which are 21 in a
// cluster, bound by the loads and stores of its eight SMs.
constexpr int kFewThreads = 256;
constexpr int kClusterThreads = 512;
constexpr int kCluster = 8;

void launch_pages_extend(const Pages& p, const PagesExtend& e, cudaStream_t stream) {
  constexpr const char* kWhat = "launch page table kernel";
  if (pages_workspace_bytes(p, e.rows) > 0) {
    launch_early(extend_plan_kernel, dim3(1), kMostThreads, 0, stream, 0, kWhat, p, e);
    constexpr int kPerBlock = kRowThreads * kRows;
    if (e.rows > 0)
      launch_early(extend_rows_kernel, dim3(static_cast<unsigned>((e.rows + kPerBlock - 1) / kPerBlock)), kRowThreads, 0, stream,
                   0, kWhat, p, e);
  } else if (p.sequences <= kFewThreads && e.rows <= 4 * kFewThreads) {
    launch_early(extend_kernel<kFewThreads, false>, dim3(1), kFewThreads, 0, stream, 0, kWhat, p, e);
  } else {
    launch_early(extend_kernel<kClusterThreads, true>, dim3(kCluster), kClusterThreads, 0, stream, kCluster, kWhat, p, e);
  }
}

void launch_pages_truncate(const Pages& p, const int32_t* to, void* workspace, cudaStream_t stream) {
  constexpr const char* kWhat = "launch page return kernel";
  if (pages_workspace_bytes(p, 0) > 0) {
    launch_early(truncate_plan_kernel, dim3(1), kMostThreads, 0, stream, 0, kWhat, p, to, workspace);
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(512, (p.num_pages + kRowThreads - 1) / kRowThreads));
    launch_early(truncate_pages_kernel, dim3(static_cast<unsigned>(blocks)), kRowThreads, 0, stream, 0, kWhat, p, workspace);
  } else if (p.sequences <= kFewThreads) {
    launch_early(truncate_kernel<kFewThreads, false>, dim3(1), kFewThreads, 0, stream, 0, kWhat, p, to);
  } else {
    launch_early(truncate_kernel<kClusterThreads, true>, dim3(kCluster), kClusterThreads, 0, stream, kCluster, kWhat, p,
                 to);
  }
}

void launch_draft_ancestors(const DraftTrees& t, cudaStream_t stream) {
  launch_early(draft_ancestors_kernel, dim3(static_cast<unsigned>(t.batch)), kTreeThreads, 0, stream, 0, "launch draft tree kernel", t);
}

}  // namespace msb
