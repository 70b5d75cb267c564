// One step of beam search: of a group's K beams x V tokens the K candidates with the largest rank.
//
//   value(b, v) = score_b + z_bv - log sum_w exp z_bw    (running beams)
//   rank        = value / max(length_b + 1, 1)^penalty
//
// Within a beam the order is that of its logits, so a block per (beam, segment of the vocabulary) needs no softmax to
// find the segment's K best: it holds the segment in registers, forms the segment's maximum and sum of exponentials
// (terms in fp32, added up over threads in fp64), takes the K-th largest of its threads' maxima as a bound that K
// values reach, and sorts the few values that do. A second kernel, one block per group, joins the sums, ranks the
// segments' candidates in fp64 and draws the K best. Ranks of different beams differ by the fp32 exponentials' error
// at worst (about 1e-7), those of one beam only by their logits.
//
// A finished beam is a list of its own: itself at the end token, then nothing (-inf) at the other tokens; a beam
// without a finite score or sum is all -inf. So every group has K candidates whatever its logits hold.
#include <algorithm>
#include <climits>
#include "../api.h"
#include "../common/common.cuh"

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int LIST = 1024;            // candidates of a segment
constexpr int SEGMENT = 16384 - 64;   // values of a segment at most (its ends need not be aligned)
constexpr int MAX_SEGMENTS = 256;
constexpr int MERGE_THREADS = 256, MERGE_WARPS = MERGE_THREADS / 32;

// Order-preserving 32-bit key of a logit: -0 equals +0; 0 is below all of them. (Of a NaN any: its beam has no rank.)
__device__ __forceinline__ unsigned order_key(float v) {
  const unsigned b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ unsigned long long entry(unsigned key, int index) {
  return (unsigned long long)key << 32 | (unsigned)~index;
}
__device__ __forceinline__ unsigned long long rank_key(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

__device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) { rt::unpack8(u, f); }
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
  f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}

struct SelectArgs {
  const void* logits;
  long ld_group, ld_beam;
  int K, V, segments;
  const float* scores;
  const int* lengths;
  const bool* finished;
  int end_token;
  double penalty;
  unsigned long long* entries;  // [rows, segments, K], zeros behind a short segment's values
  double* sums;                 // [rows, segments]
  float* tops;                  // [rows, segments]
  long* tokens;
  long* parents;
  float* out_scores;
  int* out_lengths;
  bool* out_finished;
};

__device__ __forceinline__ bool running(const SelectArgs& a, long row) {
  return !a.finished[row] && isfinite(a.scores[row]);
}

// Sum over the block of a per-thread count. Two barriers.
__device__ __forceinline__ int block_count(int n, int* counter) {
  __syncthreads();
  if (threadIdx.x == 0) *counter = 0;
  __syncthreads();
  n = __reduce_add_sync(~0u, n);
  if ((threadIdx.x & 31) == 0 && n) atomicAdd(counter, n);
  __syncthreads();
  return *counter;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) select_rows_kernel(const SelectArgs a) {
  constexpr int VEC = 16 / sizeof(T), NV = 16384 / (THREADS * VEC);
  __shared__ unsigned long long list[LIST];
  __shared__ unsigned maxima[THREADS];
  __shared__ float warp_top[WARPS];
  __shared__ double warp_sum[WARPS];
  __shared__ unsigned bound;
  __shared__ int found;
  const long row = blockIdx.x / a.segments;
  const int seg = blockIdx.x % a.segments, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (!running(a, row)) return;
  const int lo = (int)((long)a.V * seg / a.segments), n = (int)((long)a.V * (seg + 1) / a.segments) - lo;
  const T* z = static_cast<const T*>(a.logits) + row / a.K * a.ld_group + row % a.K * a.ld_beam + lo;
  // aligned vectors, and the few values before and behind them, one per thread
  const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / (int)sizeof(T));
  const int nvec = (n - head) / VEC, tail = n - head - nvec * VEC;
  const uint4* zv = reinterpret_cast<const uint4*>(z + head);
  int single = -1;
  if (tid < head) single = tid;
  else if (tid >= 16 && tid < 16 + tail) single = n - tail + (tid - 16);
  uint4 u[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * THREADS + tid < nvec) u[i] = __ldg(zv + i * THREADS + tid);
  const float one = single >= 0 ? rt::to_f<T>(z[single]) : -INFINITY;
  if (tid == 0) found = 0;

  // ---- maximum, and whether the segment holds what gives a beam no rank
  float top = one;
  bool bad = !(one < INFINITY);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * THREADS + tid < nvec) {
      float f[VEC];
      unpack(u[i], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        top = fmaxf(top, f[j]);
        bad |= !(f[j] < INFINITY);
      }
    }
  maxima[tid] = single >= 0 || tid < nvec ? order_key(top) : 0u;
  float m = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  if (lane == 0) warp_top[warp] = m;
  bad = __syncthreads_or(bad);
  m = warp_top[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) m = fmaxf(m, warp_top[w]);
  const long at = row * a.segments + seg;
  if (bad) {
    if (tid == 0) {
      a.tops[at] = INFINITY;
      a.sums[at] = NAN;
    }
    return;
  }

  // ---- sum of exponentials
  float s = 0.f;
  if (m > -INFINITY) {
    if (one > -INFINITY) s = expf(one - m);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * THREADS + tid < nvec) {
        float f[VEC];
        unpack(u[i], f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += expf(f[j] - m);
      }
  }
  double d = s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(~0u, d, o);
  if (lane == 0) warp_sum[warp] = d;

  // ---- bound: the K-th largest of the threads' maxima, bit by bit (1, which every value reaches, where fewer have one)
  if (warp == 0) {
    unsigned key[WARPS];
#pragma unroll
    for (int i = 0; i < WARPS; ++i) key[i] = maxima[i * 32 + lane];
    unsigned t = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned c = t | 1u << bit;
      int reach = 0;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) reach += key[i] >= c;
      if (__reduce_add_sync(~0u, reach) >= a.K) t = c;
    }
    if (lane == 0) bound = max(t, 1u);
  }
  __syncthreads();
  if (tid == 0) {
    double total = 0.0;
    for (int w = 0; w < WARPS; ++w) total += warp_sum[w];
    a.tops[at] = m;
    a.sums[at] = total;
  }

  // ---- candidates
  auto each = [&](auto&& take) {
    if (single >= 0) take(entry(order_key(one), lo + single));
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * THREADS + tid < nvec) {
        float f[VEC];
        unpack(u[i], f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) take(entry(order_key(f[j]), lo + head + (i * THREADS + tid) * VEC + j));
      }
  };
  unsigned long long least = (unsigned long long)bound << 32;
  auto collect = [&]() {
    if (maxima[tid] >= (unsigned)(least >> 32) && maxima[tid])
      each([&](unsigned long long e) {
        if (e >= least) {
          const int to = atomicAdd(&found, 1);
          if (to < LIST) list[to] = e;
        }
      });
    __syncthreads();
  };
  collect();
  if (found > LIST) {  // many equal values: the K-th largest of the unique entries, bit by bit
    __shared__ int counter;
    unsigned long long t = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const unsigned long long c = t | 1ull << bit;
      int reach = 0;
      each([&](unsigned long long e) { reach += e >= c; });
      if (block_count(reach, &counter) >= a.K) t = c;
    }
    least = t;
    if (tid == 0) found = 0;
    __syncthreads();
    collect();
  }
  const int have = found;
  unsigned long long* out = a.entries + at * a.K;
  for (int i = tid; i < have; i += THREADS) {  // place = number of larger entries
    const unsigned long long e = list[i];
    int rank = 0;
    for (int j = 0; j < have; ++j) rank += list[j] > e;
    if (rank < a.K) out[rank] = e;
  }
  for (int i = have + tid; i < a.K; i += THREADS) out[i] = 0;
}

// Block per group. Its lists (one per beam and segment, sorted) are drawn from K times: the best of their heads.
__global__ void __launch_bounds__(MERGE_THREADS) select_group_kernel(const SelectArgs a) {
  extern __shared__ unsigned char taken[];  // of each list
  __shared__ double base[32], norm[32];     // value = base + (z - top); rank = value / norm
  __shared__ float row_top[32];
  __shared__ int kind[32];                  // 0 running, 1 finished, 2 nothing
  __shared__ unsigned long long warp_rank[MERGE_WARPS];
  __shared__ long warp_flat[MERGE_WARPS];
  __shared__ unsigned long long best_rank;
  __shared__ long best_flat, chosen[32];
  __shared__ double values[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.K, S = a.segments, lists = K * S;
  const long first = (long)blockIdx.x * K;
  for (int i = tid; i < lists; i += MERGE_THREADS) taken[i] = 0;
  for (int b = warp; b < K; b += MERGE_WARPS) {
    const long row = first + b;
    const bool run = running(a, row);
    float top = -INFINITY;
    if (run)
      for (int i = lane; i < S; i += 32) top = fmaxf(top, a.tops[row * S + i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    double sum = 0.0;
    if (run && top > -INFINITY)
      for (int i = lane; i < S; i += 32) {
        const float t = a.tops[row * S + i];
        if (t > -INFINITY) sum += a.sums[row * S + i] * exp((double)t - (double)top);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) {
      const double score = a.scores[row];
      const bool fit = sum > 0.0 && isfinite(sum) && isfinite(top);
      kind[b] = run && fit ? 0 : a.finished[row] && isfinite(score) ? 1 : 2;
      base[b] = score - (kind[b] == 0 ? log(sum) : 0.0);
      row_top[b] = top;
      const int length = a.lengths[row] + (a.finished[row] ? 0 : 1);
      norm[b] = pow((double)max(length, 1), a.penalty);
    }
  }
  __syncthreads();
  // head of list i (rank key 0: none left)
  auto head = [&](int i, unsigned long long& rank, long& flat, double& value) {
    const int b = i / S, seg = i % S;
    int j = taken[i];
    rank = 0;
    flat = LONG_MAX;
    if (j >= K) return;
    int token;
    value = -INFINITY;
    if (kind[b] == 0) {
      const unsigned long long e = a.entries[((first + b) * S + seg) * K + j];
      if (e == 0) return;
      token = (int)~(unsigned)e;
      const float z = key_value((unsigned)(e >> 32));
      if (z > -INFINITY) value = base[b] + ((double)z - (double)row_top[b]);
    } else {
      if (seg > 0) return;
      token = j;
      if (kind[b] == 1 && a.end_token >= 0) {  // the end token first, then the others in order
        if (j == 0) value = base[b];
        token = j == 0 ? a.end_token : j - 1 + (j - 1 >= a.end_token);
      }
      if (token >= a.V) return;
    }
    rank = rank_key(value / norm[b]);
    flat = (long)b * a.V + token;
  };
  unsigned long long rank = 0;
  long flat = LONG_MAX;
  int mine = -1;
  double value = 0.0;
  auto refresh = [&]() {
    rank = 0;
    flat = LONG_MAX;
    mine = -1;
    for (int i = tid; i < lists; i += MERGE_THREADS) {
      unsigned long long r;
      long f;
      double v = 0.0;
      head(i, r, f, v);
      if (r > rank || (r == rank && f < flat)) {
        rank = r;
        flat = f;
        mine = i;
        value = v;
      }
    }
  };
  refresh();
  for (int n = 0; n < K; ++n) {
    unsigned long long r = rank;
    long f = flat;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long r2 = __shfl_xor_sync(~0u, r, o);
      const long f2 = __shfl_xor_sync(~0u, f, o);
      if (r2 > r || (r2 == r && f2 < f)) {
        r = r2;
        f = f2;
      }
    }
    if (lane == 0) {
      warp_rank[warp] = r;
      warp_flat[warp] = f;
    }
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < MERGE_WARPS; ++w)
        if (warp_rank[w] > r || (warp_rank[w] == r && warp_flat[w] < f)) {
          r = warp_rank[w];
          f = warp_flat[w];
        }
      best_rank = r;
      best_flat = f;
    }
    __syncthreads();
    if (mine >= 0 && flat == best_flat && rank == best_rank) {
      chosen[n] = flat;
      values[n] = value;
      ++taken[mine];
      refresh();
    }
  }
  __syncthreads();
  if (warp != 0) return;
  // ---- slots: a parent's best child keeps the parent's, the others fill what is left in order
  const bool in = lane < K;
  const unsigned all = K == 32 ? ~0u : (1u << K) - 1;
  const int parent = in ? (int)(chosen[lane] / a.V) : 32 + lane;
  const unsigned siblings = __match_any_sync(~0u, parent);
  const bool keeps = in && __ffs(siblings) - 1 == lane;
  unsigned left = all & ~__reduce_or_sync(~0u, in ? 1u << parent : 0u);
  const unsigned others = __ballot_sync(~0u, in && !keeps);
  if (!in) return;
  int slot = parent;
  if (!keeps) {
    for (int skip = __popc(others & ((1u << lane) - 1)); skip > 0; --skip) left &= left - 1;
    slot = __ffs(left) - 1;
  }
  const long token = chosen[lane] % a.V, to = first + slot, from = first + parent;
  a.tokens[to] = token;
  a.parents[to] = parent;
  a.out_scores[to] = (float)values[lane];
  a.out_lengths[to] = a.lengths[from] + (a.finished[from] ? 0 : 1);
  a.out_finished[to] = a.finished[from] || token == a.end_token;
}

// Segments of a beam's vocabulary: enough to fill the SMs twice, of 2048 values at least.
int segments_for(long rows, long V) {
  const long least = (V + SEGMENT - 1) / SEGMENT;
  const long spread = std::min((296 + rows - 1) / rows, V / 2048);
  return (int)std::max({1L, least, spread});
}

}  // namespace

extern "C" long rt_beam_select_workspace_bytes(long groups, int K, long V) {
  const long lists = groups * K * segments_for(groups * K, V);
  return lists * (8L * K + 8 + 4);
}

// dtype 1 = bf16, 0 = fp32; logits [groups, K, V] with strides in elements; everything else [groups, K], contiguous.
// The outputs must not overlap the inputs. work: rt_beam_select_workspace_bytes, 8-byte aligned.
extern "C" cudaError_t rt_beam_select(int dtype, const void* logits, long groups, int K, long V, long ld_group,
                                      long ld_beam, const float* scores, const int* lengths, const bool* finished,
                                      int end_token, double penalty, long* tokens, long* parents, float* out_scores,
                                      int* out_lengths, bool* out_finished, void* work, cudaStream_t s) {
  if (groups < 0 || K < 1 || K > 32 || V < 1 || V > (long)SEGMENT * MAX_SEGMENTS || end_token >= V)
    return cudaErrorInvalidValue;
  if (groups == 0) return cudaSuccess;
  const long rows = groups * K;
  SelectArgs a{};
  a.segments = segments_for(rows, V);
  if (groups > INT_MAX / 32 || rows * a.segments > INT_MAX) return cudaErrorInvalidValue;
  a.logits = logits;
  a.ld_group = ld_group;
  a.ld_beam = ld_beam;
  a.K = K;
  a.V = (int)V;
  a.scores = scores;
  a.lengths = lengths;
  a.finished = finished;
  a.end_token = end_token;
  a.penalty = penalty;
  a.entries = static_cast<unsigned long long*>(work);
  a.sums = reinterpret_cast<double*>(a.entries + rows * a.segments * K);
  a.tops = reinterpret_cast<float*>(a.sums + rows * a.segments);
  a.tokens = tokens;
  a.parents = parents;
  a.out_scores = out_scores;
  a.out_lengths = out_lengths;
  a.out_finished = out_finished;
  const unsigned blocks = (unsigned)(rows * a.segments);
  if (dtype == 1) select_rows_kernel<__nv_bfloat16><<<blocks, THREADS, 0, s>>>(a);
  else select_rows_kernel<float><<<blocks, THREADS, 0, s>>>(a);
  RT_CUDA_CHECK(cudaGetLastError());
  select_group_kernel<<<(unsigned)groups, MERGE_THREADS, K * a.segments, s>>>(a);
  return cudaGetLastError();
}
