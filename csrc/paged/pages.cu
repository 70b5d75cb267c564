// Bookkeeping and copies of a paged key/value cache (paged.py has the definitions).
//
// A pool holds pages [pages, blocks, 2, heads, page, dim] bf16; table [rows, width], lengths [rows] and refs [pages]
// (int32) say who holds them. Every decision is taken on the device by one block (a few thousand integers: bound by
// its barriers and reads: 5-6 us for up to 256 rows), which leaves a list of copies for a second kernel (bound by memory:
// 34 MB copied in 15 us from memory, 10 us from L2; 404 MB of whole pages in 134 us, 6.0 TB/s). Nothing depends on the
// order of an atomic: counts are sums, and free pages are numbered by their position.
#include <algorithm>
#include <climits>
#include "../api.h"
#include "../common/common.cuh"

namespace {

using bf16 = __nv_bfloat16;
constexpr int MAX_ROWS = 1024, SMALL_POOL = 5120;

// Exclusive prefix sum over the block and its total. Two barriers.
template <int WARPS>
__device__ __forceinline__ int block_prefix(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll 8
  for (int w = 0; w < WARPS; ++w) {
    before += w < warp ? warp_sums[w] : 0;
    total += warp_sums[w];
  }
  return before + x - v;
}

struct AdvanceArgs {
  const int* table;
  const int* lengths;
  const int* refs;
  int* new_table;  // may be the arrays above
  int* new_lengths;
  int* new_refs;
  int* status;
  int keep_status;
  const long* parents;  // [rows / K, K] or null
  const bool* live;     // [rows] or null
  int rows, K, width, pages, page, tokens;
  int4* copies;         // [rows]: (from, to, tokens, -)
  int* count;           // of them
};

// SMALL: the counts fit shared memory, which takes three waits for memory out of the chain that this kernel is bound by.
template <bool SMALL, int THREADS>
__global__ void __launch_bounds__(THREADS) advance_kernel(const AdvanceArgs a) {
  constexpr int WARPS = THREADS / 32, ROWS = THREADS;
  __shared__ int source[ROWS];  // row whose history a row takes over, -1: none (not live)
  __shared__ int before[ROWS];  // its last slot (of the partly filled page), -1: none
  __shared__ int last[ROWS];    // partly filled page that a row appends to, -1: none
  __shared__ int wants[ROWS];   // exclusive prefix of the pages that rows take
  __shared__ int slot[ROWS];    // where a row's first taken page goes
  __shared__ int target[ROWS];  // that page, -1: none found
  __shared__ int counts[SMALL ? SMALL_POOL : 1];
  __shared__ int warp_sums[WARPS];
  __shared__ int bits;
  const int tid = threadIdx.x, R = a.rows;
  int* refs = SMALL ? counts : a.new_refs;
  auto count_of = [&](int p) { return SMALL ? counts[p] : __ldcg(&a.new_refs[p]); };
  if (tid == 0) bits = 0;
  if (SMALL || a.new_refs != a.refs)
    for (int p = tid; p < a.pages; p += THREADS) refs[p] = a.refs[p];
  __syncthreads();
  int length = 0, row_source = -1;
  if (tid < R) {
    int from = tid;
    if (a.parents) {
      const long p = a.parents[tid];
      if (p >= 0 && p < a.K) from = tid / a.K * a.K + (int)p;
      else atomicOr(&bits, 4);
    }
    if (!a.live || a.live[tid]) {
      row_source = from;
      length = min(max(a.lengths[from], 0), a.width * a.page);
    }
  }
  const int fill = length % a.page, have = (length + a.page - 1) / a.page;
  const long need = ((long)length + a.tokens + a.page - 1) / a.page;
  bool grows = row_source >= 0 && a.tokens > 0;
  if (grows && need > a.width) {
    atomicOr(&bits, 2);
    grows = false;
  }
  if (tid < R) {
    source[tid] = row_source;
    before[tid] = grows && fill ? have - 1 : -1;
    last[tid] = -1;
  }
  __syncthreads();

  // ---- histories: all rows of some columns are read before any is written
  const int columns = THREADS / R, c_in = tid / R, r_in = tid - c_in * R;
  const bool busy = c_in < columns;
  const int from = busy ? source[r_in] : -1, at = busy ? before[r_in] : -1;
  constexpr int U = 4;
  for (int c0 = 0; c0 < a.width; c0 += U * columns) {
    int old[U], now[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int c = c0 + k * columns + c_in;
      const bool on = busy && c < a.width;
      old[k] = on ? a.table[(long)r_in * a.width + c] : -1;
      now[k] = on && from >= 0 && from != r_in ? a.table[(long)from * a.width + c] : -1;
      if (from == r_in) now[k] = old[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int c = c0 + k * columns + c_in;
      if (!busy || c >= a.width) continue;
      if (now[k] != old[k]) {
        if (old[k] >= 0 && old[k] < a.pages) atomicSub(&refs[old[k]], 1);
        if (now[k] >= 0 && now[k] < a.pages) atomicAdd(&refs[now[k]], 1);
      }
      a.new_table[(long)r_in * a.width + c] = now[k];
      if (c == at && now[k] < a.pages) last[r_in] = now[k];
    }
  }
  __threadfence_block();
  __syncthreads();

  // ---- what each row takes: a page of its own for a shared partly filled one, and the pages behind it
  const int mine = tid < R ? last[tid] : -1;
  bool copy = false;
  if (mine >= 0) {
    int earlier = 0;  // rows above that share it: each has left it by then
    for (int r = 0; r < tid; ++r) earlier += last[r] == mine;
    copy = count_of(mine) - earlier > 1;
  }
  const int takes = grows ? (int)copy + (int)need - have : 0;
  int total = 0;
  const int prefix = block_prefix<WARPS>(takes, warp_sums, total);
  if (tid < R) {
    wants[tid] = prefix;
    slot[tid] = have - (int)copy;
    target[tid] = -1;
  }
  for (int i = 0; i < takes; ++i) a.new_table[(long)tid * a.width + have - (int)copy + i] = -1;  // until found
  if (copy) atomicSub(&refs[mine], 1);
  __syncthreads();

  // ---- the lowest free pages, to rows in order (a page is looked at once, so taking one disturbs no other)
  int found = 0;
  for (int p0 = 0; p0 < a.pages && found < total; p0 += THREADS) {
    const int p = p0 + tid;
    const bool free = p < a.pages && count_of(p) <= 0;
    int here;
    const int n = found + block_prefix<WARPS>(free, warp_sums, here);
    if (free && n < total) {
      int lo = 0, hi = R - 1;  // the last row whose prefix is at most n: of equal ones only the last takes pages
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (wants[mid] <= n) lo = mid;
        else hi = mid - 1;
      }
      const int k = n - wants[lo];
      refs[p] = 1;
      a.new_table[(long)lo * a.width + slot[lo] + k] = p;
      if (k == 0) target[lo] = p;
    }
    found += here;
  }
  __syncthreads();
  if (tid < R) a.new_lengths[tid] = length + (grows ? a.tokens : 0);
  const bool copies = copy && target[tid] >= 0;
  int listed;
  const int at_copy = block_prefix<WARPS>(copies, warp_sums, listed);
  if (copies) a.copies[at_copy] = make_int4(mine, target[tid], fill, 0);
  if (tid == 0) *a.count = listed;
  if (SMALL)
    for (int p = tid; p < a.pages; p += THREADS) a.new_refs[p] = counts[p];
  if (tid == 0) {
    if (found < total) bits |= 1;
    *a.status = bits | (a.keep_status ? *a.status : 0);
  }
}

// Copies of a warp's or block's vectors, several in flight per thread.
template <int U>
__device__ __forceinline__ void copy_vectors(uint4* to, const uint4* from, long n, int first, int step) {
  long i = first;
  for (; i + (U - 1) * (long)step < n; i += U * (long)step) {
    uint4 v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) v[k] = from[i + k * (long)step];
#pragma unroll
    for (int k = 0; k < U; ++k) to[i + k * (long)step] = v[k];
  }
  for (; i < n; i += step) to[i] = from[i];
}

// The first tokens of a page in every block and head, for each listed copy. Blocks walk (copy, panel, half) and load the
// next one's vectors before they store this one's.
__global__ void __launch_bounds__(256) copy_tokens_kernel(bf16* pool, const int4* copies, const int* count, int panels,
                                                          int page, int dim) {
  constexpr int U = 4;  // 64 tokens of 256 components are 2 x 4 vectors per thread
  const int size = page * dim / 8;  // vectors of a panel: one block's keys or values of one head
  const int items = *count * panels * 2;
  uint4* base = reinterpret_cast<uint4*>(pool);
  uint4 v[U];
  auto load = [&](int item, uint4*& to) {
    int n = 0;
    if (item < items) {
      const int half = item & 1, pair = item >> 1, which = pair / panels, panel = pair - which * panels;
      const int4 c = copies[which];
      const int all = c.z * dim / 8, first = half ? (all + 1) / 2 : 0;
      n = half ? all - first : (all + 1) / 2;
      const uint4* from = base + ((long)c.x * panels + panel) * size + first;
      to = base + ((long)c.y * panels + panel) * size + first;
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (k * 256 + (int)threadIdx.x < n) v[k] = from[k * 256 + threadIdx.x];
    }
    return n;
  };
  uint4* to = nullptr;
  int n = load(blockIdx.x, to);
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    uint4 now[U];
#pragma unroll
    for (int k = 0; k < U; ++k) now[k] = v[k];
    uint4* here = to;
    const int m = n;
    n = load(item + gridDim.x, to);
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (k * 256 + (int)threadIdx.x < m) here[k * 256 + threadIdx.x] = now[k];
  }
}

struct CompactArgs {
  const int* table;
  const int* refs;
  int* new_table;  // may be the arrays above
  int* new_refs;
  int* used;
  int pages;
  long entries;
  int* place;   // [pages]: where each page goes
  int* holes;   // [pages]: free pages before the last that stays, in order
  int2* moves;  // [pages]: (from, to)
  int* count;
};

__global__ void __launch_bounds__(1024) compact_kernel(const CompactArgs a) {
  constexpr int THREADS = 1024, WARPS = THREADS / 32;
  __shared__ int warp_sums[WARPS];
  const int tid = threadIdx.x;
  int mine = 0, used;
  for (int p = tid; p < a.pages; p += THREADS) mine += a.refs[p] > 0;
  block_prefix<WARPS>(mine, warp_sums, used);
  int holes = 0, moves = 0;
  for (int p0 = 0; p0 < used; p0 += THREADS) {
    const int p = p0 + tid;
    const bool hole = p < used && a.refs[p] <= 0;
    int here;
    const int n = holes + block_prefix<WARPS>(hole, warp_sums, here);
    if (hole) a.holes[n] = p;
    if (p < used) a.place[p] = p;
    holes += here;
  }
  __syncthreads();
  for (int p0 = used; p0 < a.pages; p0 += THREADS) {
    const int p = p0 + tid;
    const int count = p < a.pages ? a.refs[p] : 0;
    int here;
    const int n = moves + block_prefix<WARPS>(count > 0, warp_sums, here);
    if (count > 0) {
      const int to = a.holes[n];
      a.place[p] = to;
      a.moves[n] = make_int2(p, to);
    } else if (p < a.pages) {
      a.place[p] = p;
    }
    moves += here;
  }
  __syncthreads();
  // in place or not: a hole's count is read from the page that fills it, which nothing else writes before
  if (a.new_refs != a.refs)
    for (int p = tid; p < a.pages; p += THREADS) a.new_refs[p] = a.refs[p];
  __syncthreads();
  for (int i = tid; i < moves; i += THREADS) {
    const int2 m = a.moves[i];
    a.new_refs[m.y] = a.refs[m.x];
    a.new_refs[m.x] = 0;
  }
  for (long i = tid; i < a.entries; i += THREADS) {
    const int e = a.table[i];
    a.new_table[i] = e >= 0 && e < a.pages ? a.place[e] : e;
  }
  if (tid == 0) {
    *a.used = used;
    *a.count = moves;
  }
}

// Whole pages of `vectors` 16-byte words; blocks walk the (page, part) pairs of the list.
__global__ void __launch_bounds__(256) copy_pages_kernel(uint4* pool, const int2* moves, const int* count, long vectors,
                                                         int parts) {
  const long work = (long)*count * parts;
  for (long w = blockIdx.x; w < work; w += gridDim.x) {
    const int2 m = moves[w / parts];
    const long lo = vectors * (w % parts) / parts, hi = vectors * (w % parts + 1) / parts;
    copy_vectors<8>(pool + m.y * vectors + lo, pool + m.x * vectors + lo, hi - lo, threadIdx.x, blockDim.x);
  }
}

struct Place {
  const int* table;
  const int* lengths;
  int width, pages, panels, page, dim;
};

// Where token `position` of a row lies within a panel (block * 2 heads + ...), in elements of the pool; -1: nowhere.
__device__ __forceinline__ long place_of(const Place& a, int row, long position, int panel) {
  if (position < 0 || position >= (long)a.width * a.page) return -1;
  const int p = a.table[(long)row * a.width + position / a.page];
  if (p < 0 || p >= a.pages) return -1;
  return (((long)p * a.panels + panel) * a.page + position % a.page) * a.dim;
}

struct StoreArgs {
  Place at;
  const bf16* x[2];               // keys, values [rows / every, T, heads, dim], unit stride of the last
  long batch[2], time[2], head[2];
  bf16* pool;
  int first;                      // panel of the block's keys of head 0
  int T, heads, every;
  long items;                     // rows / every * T * heads
};

// One warp per (row, token, head): its key, then its value.
__global__ void __launch_bounds__(256) store_kernel(const StoreArgs a) {
  const long item = (long)blockIdx.x * 8 + threadIdx.x / 32;
  if (item >= a.items) return;
  const int h = item % a.heads, lane = threadIdx.x % 32;
  const long rt = item / a.heads;
  const int t = rt % a.T, n = rt / a.T, row = n * a.every;
  for (int kind = 0; kind < 2; ++kind) {
    const long to = place_of(a.at, row, (long)a.at.lengths[row] - a.T + t, a.first + kind * a.heads + h);
    if (to < 0) continue;
    const bf16* x = a.x[kind] + n * a.batch[kind] + t * a.time[kind] + h * a.head[kind];
    if ((reinterpret_cast<uintptr_t>(x) & 15) == 0) {
      const int c = lane * 8;
      if (c < a.at.dim) *reinterpret_cast<uint4*>(a.pool + to + c) = *reinterpret_cast<const uint4*>(x + c);
    } else {
      for (int c = lane; c < a.at.dim; c += 32) a.pool[to + c] = x[c];
    }
  }
}

struct AppendArgs {
  Place at;
  const bf16* x;
  long ld;
  const float* q_weight;
  const float* k_weight;
  const float* inv_freq;
  bf16* q;      // [rows, heads, dim]
  bf16* pool;
  int first;    // panel of the block's keys of head 0
  int rows, heads, kv_heads, half;
  float eps;
  int vec;      // rows of x are 16-byte aligned
};

// One warp per (row, head): the query heads, then keys, then values (4 us for 64 rows of 24 + 4 heads of 256, of which the
// 8 MB would take 1: two dependent reads and the launch). The angle position * frequency is reduced to a
// turn in fp64 (in fp32 it is 0.01 off at position 2^17 already), its sine and cosine are fp32.
__global__ void __launch_bounds__(128) append_kernel(const AppendArgs a) {
  __shared__ __align__(16) float buf[4][256];
  const int lane = threadIdx.x % 32, D = a.at.dim, per = a.heads + 2 * a.kv_heads;
  const long item = (long)blockIdx.x * 4 + threadIdx.x / 32;
  if (item >= (long)a.rows * per) return;
  const int row = item / per, h = item % per, kind = h < a.heads ? 0 : h < a.heads + a.kv_heads ? 1 : 2;
  const bf16* x = a.x + row * a.ld + (kind == 0 ? 2L * h * D : (long)(h + a.heads) * D);
  const long position = (long)a.at.lengths[row] - 1;
  bf16* out;
  if (kind == 0) {
    out = a.q + ((long)row * a.heads + h) * D;
  } else {
    const long to = place_of(a.at, row, position, a.first + h - a.heads);
    if (to < 0) return;
    out = a.pool + to;
    if (kind == 2) {
      if (a.vec) {
        if (lane * 8 < D) *reinterpret_cast<uint4*>(out + lane * 8) = *reinterpret_cast<const uint4*>(x + lane * 8);
      } else {
        for (int c = lane; c < D; c += 32) out[c] = x[c];
      }
      return;
    }
  }
  float* s = buf[threadIdx.x / 32];
  const float* w = kind == 0 ? a.q_weight : a.k_weight;
  float sum = 0.f;
  if (a.vec) {  // eight components of each lane
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, g[8];
    const int c = lane * 8;
    if (c < D) {
      rt::unpack8(*reinterpret_cast<const uint4*>(x + c), v);
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = w[c + k];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += v[k] * v[k];
    const float inv = rsqrtf(rt::warp_sum(sum) / D + a.eps);
    if (c < D)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[c + k] = v[k] * inv * (1.f + g[k]);
  } else {
    for (int c = lane; c < D; c += 32) {
      const float v = rt::to_f(x[c]);
      s[c] = v;
      sum += v * v;
    }
    const float inv = rsqrtf(rt::warp_sum(sum) / D + a.eps);
    for (int c = lane; c < D; c += 32) s[c] *= inv * (1.f + w[c]);
  }
  __syncwarp();
  for (int i = lane; i < a.half; i += 32) {
    const double turns = (double)max(position, 0L) * a.inv_freq[i] * 0.15915494309189535;
    float sn, cs;
    sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
    const float x0 = s[i], x1 = s[i + a.half];
    s[i] = x0 * cs - x1 * sn;
    s[i + a.half] = x1 * cs + x0 * sn;
  }
  __syncwarp();
  if (a.vec) {
    if (lane * 8 < D) *reinterpret_cast<uint4*>(out + lane * 8) = rt::pack8(s + lane * 8);
  } else {
    for (int c = lane; c < D; c += 32) out[c] = __float2bfloat16_rn(s[c]);
  }
}

bool pool_fits(const RtPool* p) {
  return p->pages > 0 && p->blocks > 0 && p->heads > 0 && (p->page == 16 || p->page == 32 || p->page == 64) &&
         (p->dim == 64 || p->dim == 128 || p->dim == 256) && p->rows > 0 && p->rows <= MAX_ROWS && p->width > 0 &&
         (long)p->width * p->page <= INT_MAX && (long)p->blocks * 2 * p->heads <= INT_MAX &&
         reinterpret_cast<uintptr_t>(p->pool) % 16 == 0;
}
Place place(const RtPool* p, const int* table, const int* lengths) {
  return {table, lengths, p->width, p->pages, p->blocks * 2 * p->heads, p->page, p->dim};
}

}  // namespace

extern "C" long rt_advance_workspace_bytes(int rows) { return (rows + 1) * (long)sizeof(int4); }

// parents [rows / K, K] or null; live [rows] or null; the outputs may be the inputs. work: 16-byte aligned.
extern "C" cudaError_t rt_advance_pages(const RtPool* p, const int* table, const int* lengths, const int* refs,
                                        int tokens, const long* parents, int K, const bool* live, int* new_table,
                                        int* new_lengths, int* new_refs, int* status, int keep_status, void* work,
                                        cudaStream_t s) {
  if (!pool_fits(p) || tokens < 0 || K < 1 || p->rows % K) return cudaErrorInvalidValue;
  const int panels = p->blocks * 2 * p->heads;
  const long items = (long)panels * 2 * p->rows;  // of the copies at most, and the blocks' next ones stay in range
  if (items > INT_MAX - 65536) return cudaErrorInvalidValue;
  AdvanceArgs a{table, lengths, refs, new_table, new_lengths, new_refs, status, keep_status, parents, live,
                p->rows, K, p->width, p->pages, p->page, tokens, static_cast<int4*>(work) + 1, static_cast<int*>(work)};
  // (few rows: the barriers of a smaller block are cheaper)
  if (p->rows <= 256 && p->pages <= SMALL_POOL) advance_kernel<true, 256><<<1, 256, 0, s>>>(a);
  else if (p->pages <= SMALL_POOL) advance_kernel<true, 1024><<<1, 1024, 0, s>>>(a);
  else advance_kernel<false, 1024><<<1, 1024, 0, s>>>(a);
  RT_CUDA_CHECK(cudaGetLastError());
  if (tokens == 0) return cudaSuccess;
  copy_tokens_kernel<<<(unsigned)std::min(items, 148L * 6), 256, 0, s>>>(static_cast<bf16*>(p->pool), a.copies, a.count,
                                                                       panels, p->page, p->dim);
  return cudaGetLastError();
}

extern "C" long rt_compact_workspace_bytes(int pages) { return pages * 16L + 16; }

extern "C" cudaError_t rt_compact_pages(const RtPool* p, const int* table, const int* refs, int* new_table,
                                        int* new_refs, int* used, void* work, cudaStream_t s) {
  if (!pool_fits(p)) return cudaErrorInvalidValue;
  CompactArgs a{};
  a.table = table;
  a.refs = refs;
  a.new_table = new_table;
  a.new_refs = new_refs;
  a.used = used;
  a.pages = p->pages;
  a.entries = (long)p->rows * p->width;
  a.moves = static_cast<int2*>(work);
  a.place = reinterpret_cast<int*>(a.moves + p->pages);
  a.holes = a.place + p->pages;
  a.count = a.holes + p->pages;
  compact_kernel<<<1, 1024, 0, s>>>(a);
  RT_CUDA_CHECK(cudaGetLastError());
  const long vectors = (long)p->blocks * 2 * p->heads * p->page * p->dim / 8;
  const int parts = (int)std::min((vectors + 2047) / 2048, 4096L);  // 32 KB: eight vectors per thread
  copy_pages_kernel<<<148 * 8, 256, 0, s>>>(static_cast<uint4*>(p->pool), a.moves, a.count, vectors, parts);
  return cudaGetLastError();
}

// keys, values [rows / every, T, heads, dim] bf16 with unit inner stride; strides {batch, time, head} in elements.
extern "C" cudaError_t rt_store_pages(const RtPool* p, int block, const int* table, const int* lengths,
                                      const void* keys, const long* key_strides, const void* values,
                                      const long* value_strides, int T, int every, cudaStream_t s) {
  if (!pool_fits(p) || block < 0 || block >= p->blocks || every < 1 || p->rows % every || T < 0)
    return cudaErrorInvalidValue;
  StoreArgs a{place(p, table, lengths)};
  a.x[0] = static_cast<const bf16*>(keys);
  a.x[1] = static_cast<const bf16*>(values);
  for (int i = 0; i < 2; ++i) {
    const long* st = i ? value_strides : key_strides;
    a.batch[i] = st[0];
    a.time[i] = st[1];
    a.head[i] = st[2];
  }
  a.pool = static_cast<bf16*>(p->pool);
  a.first = block * 2 * p->heads;
  a.T = T;
  a.heads = p->heads;
  a.every = every;
  a.items = (long)(p->rows / every) * T * p->heads;
  if (a.items == 0) return cudaSuccess;
  if ((a.items + 7) / 8 > INT_MAX) return cudaErrorInvalidValue;
  store_kernel<<<(unsigned)((a.items + 7) / 8), 256, 0, s>>>(a);
  return cudaGetLastError();
}

// x [rows, (2 heads + 2 kv heads) dim] bf16 with row stride ld; q [rows, heads, dim]; half = rotated components / 2.
extern "C" cudaError_t rt_append_heads(const RtPool* p, int block, const int* table, const int* lengths, const void* x,
                                       long ld, const float* q_weight, const float* k_weight, const float* inv_freq,
                                       int half, int heads, float eps, void* q, cudaStream_t s) {
  if (!pool_fits(p) || block < 0 || block >= p->blocks || heads < 1 || half < 0 || 2 * half > p->dim)
    return cudaErrorInvalidValue;
  AppendArgs a{place(p, table, lengths), static_cast<const bf16*>(x), ld, q_weight, k_weight, inv_freq,
               static_cast<bf16*>(q), static_cast<bf16*>(p->pool), block * 2 * p->heads, p->rows, heads, p->heads, half,
               eps, (reinterpret_cast<uintptr_t>(x) | (uintptr_t)(ld * 2)) % 16 == 0};
  const long items = (long)p->rows * (heads + 2 * p->heads);
  append_kernel<<<(unsigned)((items + 3) / 4), 128, 0, s>>>(a);
  return cudaGetLastError();
}
