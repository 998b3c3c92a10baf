// Page tables of the 4-bit key/value cache, kept on the device: pages taken from a stack of free ones as sequences
// grow, given back as they shrink, and the slots and positions of a step's rows; and the masks of drafted trees.
//
// extend.  With L_b tokens held, n_b = max(tokens_b, 0) new ones and pages of P tokens, sequence b holds
// have_b = ceil(L_b / P) pages and wants ceil((L_b + n_b) / P).  Its rows are E_b .. E_b + n_b of the step, E the
// exclusive sums of n.  Of the sequences whose pages fit their row of the table and whose rows fit the step, U_b is the
// inclusive sum of the pages they lack; b is served where it lacks none or U_b <= free.  Its page of column c >= have_b
// is entry free - 1 - (U_b - lacks_b + c - have_b) of the stack.  Row i of b is at position L_b + i.
// truncate.  Pages past ceil(L'_b / P) go back, the first sequence's first one on top: what extend took lies as before.
//   Bound: latency.  One block forms the sums (plan); where rows or sequences are many a second kernel with a thread a
//   row (or a page given back) does the rest, launched early, else the same block does it, from shared memory.
//   A row whose position starts a page enters that page in the table: each new page has one such row.
#include <algorithm>

#include "pages.cuh"

namespace msb {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kSmall = 1024;      // sequences that one block keeps in shared memory
constexpr int kSmallRows = 8192;  // rows that it does by itself
constexpr int kRowThreads = 256;

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

// Inclusive sums over the block; the block's total too.
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* scratch, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xFFFFFFFFu, v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();  // the sums before have been read
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  int64_t s = lane < kWarps ? scratch[lane] : 0;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xFFFFFFFFu, s, d);
    if (lane >= d) s += o;
  }
  total = __shfl_sync(0xFFFFFFFFu, s, 31);
  const int64_t before = __shfl_sync(0xFFFFFFFFu, s, warp > 0 ? warp - 1 : 0);
  return v + (warp > 0 ? before : 0);
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

__device__ void extend_plan(const Pages& p, const PagesExtend& e, const Plan& plan, int64_t* scratch) {
  const int64_t free = free_pages(p);
  int64_t rows_before = 0, pages_before = 0, taken = 0;
  for (int b0 = 0; b0 < p.sequences; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int64_t length = 0, n = 0;
    if (b < p.sequences) {
      length = held_length(p, b);
      n = max(0, e.tokens[b]);
    }
    int64_t rows, pages;
    const int64_t end = rows_before + block_sum(n, scratch, rows);
    const int64_t have = pages_of(p, length), want = pages_of(p, length + n);
    const bool fits = want <= p.max_pages && end <= e.rows;
    const int64_t lacks = fits ? want - have : 0;
    const int64_t upto = pages_before + block_sum(lacks, scratch, pages);
    const bool served = fits && (lacks == 0 || upto <= free);
    if (b < p.sequences) {
      plan.start[b] = end - n;
      plan.length[b] = served ? static_cast<int32_t>(length) : -1;
      plan.entry[b] = static_cast<int32_t>(max(int64_t{0}, free - 1 - (upto - lacks)));
      e.offsets[b] = static_cast<int32_t>(min(end - n, e.rows));
      if (served) p.lengths[b] = static_cast<int32_t>(length + n);
    }
    // Those that lack pages and are served are the first that lack some: the largest of their sums is all that is taken.
    taken = max(taken, served && lacks > 0 ? upto : int64_t{0});
    rows_before += rows;
    pages_before += pages;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) taken = max(taken, __shfl_xor_sync(0xFFFFFFFFu, taken, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = taken;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) taken = max(taken, scratch[w]);
    plan.start[p.sequences] = rows_before;
    e.offsets[p.sequences] = static_cast<int32_t>(min(rows_before, e.rows));
    *p.free_count = static_cast<int32_t>(free - taken);
  }
}

__device__ __forceinline__ void extend_row(const Pages& p, const PagesExtend& e, const Plan& plan, int64_t row) {
  int64_t slot = -1;
  int32_t position = -1;
  if (row < plan.start[p.sequences]) {
    const int b = sequence_of(plan.start, p.sequences, row);
    const int32_t length = plan.length[b];
    if (length >= 0) {
      position = static_cast<int32_t>(length + (row - plan.start[b]));
      const int column = position >> p.page_shift, have = static_cast<int>(pages_of(p, length));
      int32_t* const cell = p.table + static_cast<int64_t>(b) * p.max_pages + column;
      int32_t page;
      if (column < have) {
        page = *cell;
      } else {
        page = p.free[max(0, plan.entry[b] - (column - have))];
        if ((position & ((1 << p.page_shift) - 1)) == 0) *cell = page;
      }
      slot = (static_cast<int64_t>(page) << p.page_shift) + (position & ((1 << p.page_shift) - 1));
      if (page < 0) slot = -1;
    }
  }
  e.slots[row] = slot;
  e.positions[row] = position;
}

__global__ void __launch_bounds__(kThreads) extend_small_kernel(Pages p, PagesExtend e) {
  __shared__ __align__(8) unsigned char plan_memory[(kSmall + 1) * 8 + kSmall * 8];
  __shared__ int64_t scratch[kWarps];
  const Plan plan = plan_at(plan_memory, p.sequences);
  extend_plan(p, e, plan, scratch);
  __syncthreads();
  for (int64_t row = threadIdx.x; row < e.rows; row += kThreads) extend_row(p, e, plan, row);
}
__global__ void __launch_bounds__(kThreads) extend_plan_kernel(Pages p, PagesExtend e) {
  __shared__ int64_t scratch[kWarps];
  extend_plan(p, e, plan_at(e.workspace, p.sequences), scratch);
}
__global__ void __launch_bounds__(kRowThreads) extend_rows_kernel(Pages p, PagesExtend e) {
#if __CUDA_ARCH__ >= 900
  cudaGridDependencySynchronize();
#endif
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
  if (row < e.rows) extend_row(p, e, plan_at(e.workspace, p.sequences), row);
}

__device__ void truncate_plan(const Pages& p, const int32_t* to, const Plan& plan, int64_t* scratch) {
  const int64_t free = free_pages(p);
  int64_t before = 0;
  for (int b0 = 0; b0 < p.sequences; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int64_t length = 0, left = 0;
    if (b < p.sequences) {
      length = held_length(p, b);
      left = max(int64_t{0}, min(static_cast<int64_t>(to[b]), length));
    }
    const int64_t keep = pages_of(p, left), back = pages_of(p, length) - keep;
    int64_t total;
    const int64_t upto = before + block_sum(back, scratch, total);
    if (b < p.sequences) {
      plan.start[b] = upto - back;
      plan.length[b] = static_cast<int32_t>(keep);  // the first column given back
      p.lengths[b] = static_cast<int32_t>(left);
    }
    before += total;
  }
  if (threadIdx.x == 0) {
    plan.start[p.sequences] = before;
    plan.entry[0] = static_cast<int32_t>(free);
    *p.free_count = static_cast<int32_t>(min(free + before, p.num_pages));
  }
}
// Page k of those given back goes to entry free + all - 1 - k.
__device__ __forceinline__ void truncate_page(const Pages& p, const Plan& plan, int64_t k) {
  const int b = sequence_of(plan.start, p.sequences, k);
  int32_t* const cell =
      p.table + static_cast<int64_t>(b) * p.max_pages + plan.length[b] + static_cast<int>(k - plan.start[b]);
  const int64_t entry = plan.entry[0] + plan.start[p.sequences] - 1 - k;
  if (entry < p.num_pages) p.free[entry] = *cell;
  *cell = -1;
}
__global__ void __launch_bounds__(kThreads) truncate_small_kernel(Pages p, const int32_t* to) {
  __shared__ __align__(8) unsigned char plan_memory[(kSmall + 1) * 8 + kSmall * 8];
  __shared__ int64_t scratch[kWarps];
  const Plan plan = plan_at(plan_memory, p.sequences);
  truncate_plan(p, to, plan, scratch);
  __syncthreads();
  for (int64_t k = threadIdx.x; k < plan.start[p.sequences]; k += kThreads) truncate_page(p, plan, k);
}
__global__ void __launch_bounds__(kThreads) truncate_plan_kernel(Pages p, const int32_t* to, void* workspace) {
  __shared__ int64_t scratch[kWarps];
  truncate_plan(p, to, plan_at(workspace, p.sequences), scratch);
}
__global__ void __launch_bounds__(kRowThreads) truncate_pages_kernel(Pages p, void* workspace) {
#if __CUDA_ARCH__ >= 900
  cudaGridDependencySynchronize();
#endif
  const Plan plan = plan_at(workspace, p.sequences);
  const int64_t all = plan.start[p.sequences];
  for (int64_t k = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x; k < all;
       k += static_cast<int64_t>(gridDim.x) * kRowThreads)
    truncate_page(p, plan, k);
}

template <class... Args>
void launch_early(void (*kernel)(Args...), int64_t blocks, int threads, cudaStream_t stream, const char* what, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = stream;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  check(cudaLaunchKernelEx(&cfg, kernel, args...), what);
  count_launch();
}

// Ancestors of the nodes of drafted trees: a block a sequence, its parents in shared memory, a thread a node's
// word of 64 nodes; it walks the node's path up, which ends, as a parent has a lower index.
constexpr int kTreeThreads = 128;
__global__ void __launch_bounds__(kTreeThreads) draft_ancestors_kernel(DraftTrees t) {
  __shared__ int16_t parent[kMostTreeRows];
  const int b = blockIdx.x;
  // Sequences' rows held to the call's; the rows before the first and after the last, and past the announced number, 0.
  const int64_t lo = max(0, t.offsets[b]), hi = min(static_cast<int64_t>(t.offsets[b + 1]), t.rows);
  const int all = static_cast<int>(max(int64_t{0}, hi - lo)), rows = min(all, t.max_rows);
  for (int i = threadIdx.x; i < rows; i += kTreeThreads) {
    const int p = t.parents[lo + i];
    parent[i] = static_cast<int16_t>(p >= 0 && p < i ? p : -1);
  }
  __syncthreads();
  for (int k = threadIdx.x; k < rows * t.words; k += kTreeThreads) {
    const int i = k / t.words, word = k - i * t.words;
    uint64_t bits = 0;
    int depth = -1;
    for (int at = i; at >= 0; at = parent[at]) {
      if (at >> 6 == word) bits |= uint64_t{1} << (at & 63);
      ++depth;
    }
    t.ancestors[(lo + i) * t.words + word] = static_cast<int64_t>(bits);
    if (word == 0) t.depths[lo + i] = depth;
  }
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

void launch_pages_extend(const Pages& p, const PagesExtend& e, cudaStream_t stream) {
  if (pages_workspace_bytes(p, e.rows) == 0) {
    extend_small_kernel<<<1, kThreads, 0, stream>>>(p, e);
    count_launch();
    check(cudaGetLastError(), "launch page table kernel");
    return;
  }
  extend_plan_kernel<<<1, kThreads, 0, stream>>>(p, e);
  count_launch();
  check(cudaGetLastError(), "launch page table kernel");
  if (e.rows > 0)
    launch_early(extend_rows_kernel, (e.rows + kRowThreads - 1) / kRowThreads, kRowThreads, stream, "launch slot kernel", p, e);
}

void launch_pages_truncate(const Pages& p, const int32_t* to, void* workspace, cudaStream_t stream) {
  if (pages_workspace_bytes(p, 0) == 0) {
    truncate_small_kernel<<<1, kThreads, 0, stream>>>(p, to);
    count_launch();
    check(cudaGetLastError(), "launch page return kernel");
    return;
  }
  truncate_plan_kernel<<<1, kThreads, 0, stream>>>(p, to, workspace);
  count_launch();
  check(cudaGetLastError(), "launch page return kernel");
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(512, (p.num_pages + kRowThreads - 1) / kRowThreads));
  launch_early(truncate_pages_kernel, blocks, kRowThreads, stream, "launch page return kernel", p, workspace);
}

void launch_draft_ancestors(const DraftTrees& t, cudaStream_t stream) {
  draft_ancestors_kernel<<<static_cast<unsigned>(t.batch), kTreeThreads, 0, stream>>>(t);
  count_launch();
  check(cudaGetLastError(), "launch draft tree kernel");
}

}  // namespace msb
