// Attention of one token per row over the pages of a cache (paged.py has the definition).
//
// The keys of a row are cut into splits over as many blocks; each leaves the maximum of its scores, the sum of their
// exponentials and the weighted sum of values, which a second kernel joins, gates and rounds.
#include <algorithm>
#include <climits>
#include "../api.h"
#include "../common/common.cuh"

namespace {

using bf16 = __nv_bfloat16;
constexpr int WARPS = 4, MAX_SPLITS = 64;

struct AttendArgs {
  const bf16* pool;
  int pages, panels, first, kv_heads, page, rows, width, splits;
  const int* table;
  const int* lengths;
  const bf16* q;
  long q_row, q_head;
  int heads;
  const bf16* gate;
  long gate_row, gate_head;
  float scale;
  bf16* out;
  float* sums;     // [rows, heads, splits, dim]
  float2* stats;   // [rows, heads, splits]: maximum, sum of exponentials
};

// One warp per (query head, row, split): keys one after another.
template <int D>
__global__ void __launch_bounds__(WARPS * 32) attend_kernel(const AttendArgs a) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x % 32;
  const long item = (long)blockIdx.x * WARPS + threadIdx.x / 32;
  if (item >= (long)a.rows * a.heads * a.splits) return;
  const int split = item % a.splits, head = item / a.splits % a.heads, row = item / a.splits / a.heads;
  const int panel = a.first + head / (a.heads / a.kv_heads);
  const int n = min(max(a.lengths[row], 0), a.width * a.page);
  const int lo = (int)((long)n * split / a.splits), hi = (int)((long)n * (split + 1) / a.splits);
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = rt::to_f(a.q[row * a.q_row + head * a.q_head + e * 32 + lane]) * a.scale;
    o[e] = 0.f;
  }
  for (int t = lo; t < hi; ++t) {
    const int p = a.table[(long)row * a.width + t / a.page];
    if (p < 0 || p >= a.pages) continue;
    const bf16* k = a.pool + (((long)p * a.panels + panel) * a.page + t % a.page) * D;
    const bf16* v = k + (long)a.kv_heads * a.page * D;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += q[e] * rt::to_f(k[e * 32 + lane]);
    s = rt::warp_sum(s);
    const float top = fmaxf(m, s), keep = expf(m - top), w = expf(s - top);
    m = top;
    l = l * keep + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * keep + w * rt::to_f(v[e * 32 + lane]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) a.sums[item * D + e * 32 + lane] = o[e];
  if (lane == 0) a.stats[item] = make_float2(m, l);
}

// Block per (row, query head), a thread per component.
__global__ void join_kernel(const AttendArgs a, int D) {
  const long rh = blockIdx.x;
  const int head = rh % a.heads, row = rh / a.heads, c = threadIdx.x;
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int i = 0; i < a.splits; ++i) m = fmaxf(m, a.stats[rh * a.splits + i].x);
  for (int i = 0; i < a.splits; ++i) {
    const float2 st = a.stats[rh * a.splits + i];
    if (st.y == 0.f) continue;
    const float w = expf(st.x - m);
    l += w * st.y;
    o += w * a.sums[(rh * a.splits + i) * D + c];
  }
  o = l == 0.f ? 0.f : o / l;
  if (a.gate) o *= rt::sigmoidf_(rt::to_f(a.gate[row * a.gate_row + head * a.gate_head + c]));
  a.out[rh * D + c] = __float2bfloat16_rn(o);
}

int splits_for(const RtPool* p, int heads) {
  const long keys = (long)p->width * p->page, warps = (long)p->rows * heads;
  return (int)std::max(1L, std::min({keys / 64, (148 * 16 + warps - 1) / warps, (long)MAX_SPLITS}));
}

}  // namespace

extern "C" long rt_paged_attention_workspace_floats(const RtPool* p, int heads, int group) {
  return (long)p->rows * heads * splits_for(p, heads) * (p->dim + 2);
}

extern "C" cudaError_t rt_paged_attention(const RtPool* p, int block, const int* table, const int* lengths,
                                          const void* q, long q_row, long q_head, int heads, const void* gate,
                                          long gate_row, long gate_head, int group, void* out, float* work,
                                          cudaStream_t s) {
  if (block < 0 || block >= p->blocks || heads < 1 || heads % p->heads || group < 1 || p->rows % group ||
      (long)p->width * p->page > INT_MAX)
    return cudaErrorInvalidValue;
  AttendArgs a{};
  a.pool = static_cast<const bf16*>(p->pool);
  a.pages = p->pages;
  a.panels = p->blocks * 2 * p->heads;
  a.first = block * 2 * p->heads;
  a.kv_heads = p->heads;
  a.page = p->page;
  a.rows = p->rows;
  a.width = p->width;
  a.splits = splits_for(p, heads);
  a.table = table;
  a.lengths = lengths;
  a.q = static_cast<const bf16*>(q);
  a.q_row = q_row;
  a.q_head = q_head;
  a.heads = heads;
  a.gate = static_cast<const bf16*>(gate);
  a.gate_row = gate_row;
  a.gate_head = gate_head;
  a.scale = 1.f / sqrtf((float)p->dim);
  a.out = static_cast<bf16*>(out);
  const long items = (long)p->rows * heads * a.splits;
  if ((items + WARPS - 1) / WARPS > INT_MAX) return cudaErrorInvalidValue;
  a.stats = reinterpret_cast<float2*>(work);
  a.sums = work + 2 * items;
  const unsigned blocks = (unsigned)((items + WARPS - 1) / WARPS);
  if (p->dim == 64) attend_kernel<64><<<blocks, WARPS * 32, 0, s>>>(a);
  else if (p->dim == 128) attend_kernel<128><<<blocks, WARPS * 32, 0, s>>>(a);
  else if (p->dim == 256) attend_kernel<256><<<blocks, WARPS * 32, 0, s>>>(a);
  else return cudaErrorInvalidValue;
  RT_CUDA_CHECK(cudaGetLastError());
  join_kernel<<<(unsigned)(p->rows * heads), p->dim, 0, s>>>(a, p->dim);
  return cudaGetLastError();
}
