// Attention over the 4-bit key/value cache.
//
// Row (query token i of sequence b, query head h) sees cached tokens j <= pos (causal) and
// j > pos - window, pos = length - rows + i.  With s_j = scale * ks_j * <q, kc_j>, the row's output is
// sum_j exp(s_j - m) vs_j vc_j / sum_j exp(s_j - m), kept in fp32 with the running maximum m; a row that sees
// nothing writes zeros and a log-sum-exp of -inf.
#include <algorithm>

#include "quant4.cuh"

namespace msb {
namespace {

// One warp per row and head; lane l holds dimensions l * dim / 32 and on.
template <class T, int kDim>
__global__ void kv4_attend_kernel(Kv4View c, Kv4Attend a) {
  constexpr int kPer = kDim / 32;
  const int lane = threadIdx.x & 31;
  const int head = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int b = blockIdx.z;
  if (head >= a.heads) return;
  const Kv4Sequence q = kv4_sequence(a, c.page_shift, b);
  for (int i = blockIdx.y; i < q.rows; i += gridDim.y) {
    const int64_t row = q.row0 + i;
    const T* x = static_cast<const T*>(a.query) + row * a.q_row_stride + head * a.q_head_stride + lane * kPer;
    float qv[kPer], o[kPer], m = -INFINITY, l = 0.0F;
#pragma unroll
    for (int d = 0; d < kPer; ++d) {
      qv[d] = to_f32(x[d]) * a.scale;
      o[d] = 0.0F;
    }
    const int pos = q.length - q.rows + i;
    const int end = a.causal ? pos + 1 : q.length;
    const int begin = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const int kv_head = head / (a.heads / c.heads);
    for (int j = begin; j < end; ++j) {
      const int page = a.page_table[b * a.table_stride + (j >> c.page_shift)];
      if (page < 0 || page >= c.num_pages) continue;
      const int64_t at = c.vector(page, kv_head, j & ((1 << c.page_shift) - 1));
      float s = 0.0F, v[kPer];
#pragma unroll
      for (int d = 0; d < kPer; d += 2) {
        const int64_t byte = at * (kDim / 2) + (lane * kPer + d) / 2;
        const int kb = c.codes[0][byte], vb = c.codes[1][byte];
        s += qv[d] * static_cast<float>(((kb & 15) ^ 8) - 8) + qv[d + 1] * static_cast<float>(((kb >> 4) ^ 8) - 8);
        v[d] = static_cast<float>(((vb & 15) ^ 8) - 8);
        v[d + 1] = static_cast<float>(((vb >> 4) ^ 8) - 8);
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
      s *= c.scales[0][at];
      const float next = fmaxf(m, s);
      const float fade = __expf(m - next), p = __expf(s - next), pv = p * c.scales[1][at];
      m = next;
      l = l * fade + p;
#pragma unroll
      for (int d = 0; d < kPer; ++d) o[d] = o[d] * fade + pv * v[d];
    }
    T* out = static_cast<T*>(a.out) + (row * a.heads + head) * kDim + lane * kPer;
#pragma unroll
    for (int d = 0; d < kPer; ++d) out[d] = from_f32<T>(l == 0.0F ? 0.0F : o[d] / l);
    if (a.lse && lane == 0) a.lse[row * a.heads + head] = l == 0.0F ? -INFINITY : m + logf(l);
  }
}

template <class T>
void launch_typed(const Kv4View& c, const Kv4Attend& a, cudaStream_t stream) {
  const dim3 grid((a.heads + 3) / 4, std::min(a.max_rows, 32768), a.batch);
  if (c.dim == 64) kv4_attend_kernel<T, 64><<<grid, 128, 0, stream>>>(c, a);
  else if (c.dim == 128) kv4_attend_kernel<T, 128><<<grid, 128, 0, stream>>>(c, a);
  else kv4_attend_kernel<T, 256><<<grid, 128, 0, stream>>>(c, a);
}

}  // namespace

size_t kv4_attend_workspace_bytes(const Kv4View&, const Kv4Attend&) { return 0; }

void launch_kv4_attend(const Kv4View& c, const Kv4Attend& a, cudaStream_t stream) {
  if (a.rows <= 0 || a.batch <= 0) return;
  if (a.type == kElemF16) launch_typed<__half>(c, a, stream);
  else launch_typed<__nv_bfloat16>(c, a, stream);
  count_launch();
  check(cudaGetLastError(), "launch cache attention kernel");
}

}  // namespace msb
