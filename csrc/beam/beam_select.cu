// One step of beam search: of a group's K beams x V tokens the K candidates with the largest rank.
//
//   value(b, v) = score_b + z_bv - log sum_w exp z_bw    (running beams)
//   rank        = value / max(length_b + 1, 1)^penalty
//
// Equal ranks go by the beam, then the logit, then the token. So within a beam the order is that of its logits, and a block
// per (beam, segment of the vocabulary) needs no softmax to find the segment's K best: it holds the segment in registers,
// forms the segment's maximum and sum of exponentials (terms in fp32, added up over threads in fp64), takes a bound from its
// threads' maxima that K values reach, and sorts the few values that do. A second kernel, one block per group, joins the
// sums, ranks the segments' candidates in fp64 and keeps the K best. Ranks of different beams are off by the fp32
// exponentials' error at worst (about 1e-7), those of one beam differ by their logits alone.
//
// Eight groups of eight beams x 248077 fp32 logits (a sixth of them ended, 53 MB): 17 us for the segments, bound by half
// of the issue slots and the phases of a block, 6 us for the groups, a chain of reads, barriers and code that each block
// passes once (17 k cycles with a division and an exponential inlined at each use and all lists' entries read, 11-12 k so).
// Four beams x 4096: 5 and 6 us.
//
// A finished beam is a list of its own: itself at the end token, then nothing (-inf) at the other tokens; a beam
// without a finite score or sum is all -inf. So every group has K candidates whatever its logits hold.
#include <algorithm>
#include <climits>
#include "../api.h"
#include "../common/common.cuh"

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int LIST = 512;            // candidates of a segment
constexpr int HELD = 8192;           // values of a block in registers
constexpr int SEGMENT = HELD - 64;   // of a segment at most (its ends need not be aligned)
constexpr int MAX_SEGMENTS = 512;
constexpr int MERGE_LIST = 1024;     // candidates of a group
static_assert((long)SEGMENT * MAX_SEGMENTS <= 1 << 22, "a token has 22 bits");
constexpr float LOG2E = 1.4426950408889634f;

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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
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

// The K largest entries of z[0, n) into list, unsorted (many equal values): they are unique, so the K-th largest is found
// bit by bit, with a read of the segment for each. Returns how many there are.
template <typename T>
__device__ __noinline__ int take_by_bits(const T* z, int lo, int n, int K, unsigned long long* list) {
  __shared__ int counter;
  unsigned long long least = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const unsigned long long c = least | 1ull << bit;
    int reach = 0;
    for (int v = threadIdx.x; v < n; v += THREADS) reach += entry(order_key(rt::to_f<T>(z[v])), lo + v) >= c;
    if (block_count(reach, &counter) >= K) least = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) counter = 0;
  __syncthreads();
  for (int v = threadIdx.x; v < n; v += THREADS) {
    const unsigned long long e = entry(order_key(rt::to_f<T>(z[v])), lo + v);
    if (e >= least) list[atomicAdd(&counter, 1)] = e;
  }
  __syncthreads();
  return counter;
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 5) select_rows_kernel(const SelectArgs a) {
  constexpr int VEC = 16 / sizeof(T), NV = HELD / (THREADS * VEC);
  __shared__ unsigned long long list[LIST];
  __shared__ float warp_top[WARPS];
  __shared__ double warp_sum[WARPS];
  __shared__ unsigned warp_bound[WARPS];
  __shared__ int found;
  // (32-bit divisions: those of 64 bits were half of this kernel's instructions; V x segments is below 2^32)
  const unsigned segments = a.segments, row = blockIdx.x / segments, seg = blockIdx.x - row * segments;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (!running(a, row)) return;
  const int lo = (int)((unsigned)a.V * seg / segments), n = (int)((unsigned)a.V * (seg + 1) / segments) - lo;
  const unsigned group = row / (unsigned)a.K;
  const T* z = static_cast<const T*>(a.logits) + group * a.ld_group + (row - group * a.K) * a.ld_beam + lo;
  // aligned vectors, and the few values before and behind them, one per thread
  const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / (int)sizeof(T));
  const int nvec = (n - head) / VEC, tail = n - head - nvec * VEC;
  const uint4* zv = reinterpret_cast<const uint4*>(z + head);
  int single = -1;
  if (tid < head) single = tid;
  else if (tid >= 16 && tid < 16 + tail) single = n - tail + (tid - 16);
  uint4 u[NV];  // -inf behind the last vector
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
    u[i] = i * THREADS + tid < nvec ? __ldg(zv + i * THREADS + tid) : make_uint4(none, none, none, none);
  }
  const float one = single >= 0 ? rt::to_f<T>(z[single]) : -INFINITY;
  if (tid == 0) found = 0;

  // ---- maximum (of the numbers: a NaN or +inf, which leaves its beam without a rank, makes the sum below NaN)
  float top = one;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float f[VEC];
    unpack(u[i], f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) top = fmaxf(top, f[j]);
  }
  const unsigned mine = single >= 0 || tid < nvec ? order_key(top) : 0u;
  float m = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  // ---- bound: of the warps whose threads all have values, each one's k-th largest of its threads' maxima, the smallest
  // of which K values reach (none where there is no such warp)
  const int whole = min(nvec / 32, WARPS);
  if (warp < whole) {
    unsigned key = mine, t = 0;
    for (int k = (a.K + whole - 1) / whole; k > 0; --k) {
      t = __reduce_max_sync(~0u, key);
      const unsigned equal = __ballot_sync(~0u, key == t);
      if (lane == __ffs(equal) - 1) key = 0;
    }
    if (lane == 0) warp_bound[warp] = t;
  }
  if (lane == 0) warp_top[warp] = m;
  __syncthreads();
  m = warp_top[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) m = fmaxf(m, warp_top[w]);
  const long at = blockIdx.x;

  // ---- sum of exponentials (differences before products: a mask of the type's lowest value may leave fp32's range)
  float2 sum2 = make_float2(0.f, 0.f);
  if (m > -INFINITY) {
    if (single >= 0) sum2.x = ex2((one - m) * LOG2E);
    const float2 less = make_float2(-m, -m), scale = make_float2(LOG2E, LOG2E);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[VEC];
      unpack(u[i], f);
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        const float2 y = mul2(add2(make_float2(f[j], f[j + 1]), less), scale);
        sum2 = add2(sum2, make_float2(ex2(y.x), ex2(y.y)));
      }
    }
  } else {  // no number above -inf, but a NaN leaves the beam without a rank here too
    bool none = single >= 0 && one != one;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[VEC];
      unpack(u[i], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) none |= f[j] != f[j];
    }
    if (none) sum2.x = NAN;
  }
  double d = (double)sum2.x + (double)sum2.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(~0u, d, o);
  if (lane == 0) warp_sum[warp] = d;
  unsigned bound = 0;
  for (int w = 0; w < whole; ++w) bound = w ? min(bound, warp_bound[w]) : warp_bound[0];

  // ---- candidates
  if (mine && mine >= bound) {
    const float least = bound ? key_value(bound) : -INFINITY;
    auto take = [&](float f, int index) {
      if (f >= least) {
        const int to = atomicAdd(&found, 1);
        if (to < LIST) list[to] = entry(order_key(f), index);
      }
    };
    if (single >= 0) take(one, lo + single);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[VEC], best = -INFINITY;
      unpack(u[i], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) best = fmaxf(best, f[j]);
      if (best >= least && i * THREADS + tid < nvec)
#pragma unroll
        for (int j = 0; j < VEC; ++j) take(f[j], lo + head + (i * THREADS + tid) * VEC + j);
    }
  }
  __syncthreads();
  if (tid == 0) {
    double total = 0.0;
    for (int w = 0; w < WARPS; ++w) total += warp_sum[w];
    a.tops[at] = m;
    a.sums[at] = total;
  }
  const int have = found <= LIST ? found : take_by_bits(z, lo, n, a.K, list);
  unsigned long long* out = a.entries + at * a.K;
  for (int i = tid; i < have; i += THREADS) {  // place = number of larger entries
    const unsigned long long e = list[i];
    int rank = 0;
    for (int j = 0; j < have; ++j) rank += list[j] > e;
    if (rank < a.K) out[rank] = e;
  }
  for (int i = have + tid; i < a.K; i += THREADS) out[i] = 0;
}

// (One copy of each: a block passes its code once, and the larger it is the longer it waits for instructions.)
__device__ __noinline__ double exp_of(double x) { return exp(x); }

// Block per group: the K best of its lists (one per beam and segment, sorted, K entries each). Their
// heads give a bound that K candidates reach; the candidates that do are few, and each counts those before it. Where
// equal heads make them too many, the best head is drawn K times instead.
template <int MERGE_THREADS>
__global__ void __launch_bounds__(MERGE_THREADS) select_group_kernel(const SelectArgs a) {
  constexpr int MERGE_WARPS = MERGE_THREADS / 32;
  extern __shared__ unsigned char taken[];  // of each list
  __shared__ double base[32], norm[32];     // value = base + (z - top); rank = value / norm
  __shared__ float row_top[32];
  __shared__ int kind[32];                  // 0 running, 1 finished, 2 nothing
  __shared__ int next_length[32];
  __shared__ bool ended[32];
  __shared__ unsigned long long list_rank[MERGE_LIST], best_rank, warp_rank[MERGE_WARPS];
  __shared__ long list_flat[MERGE_LIST], best_flat, warp_flat[MERGE_WARPS], chosen[32];
  __shared__ double list_value[MERGE_LIST];
  __shared__ unsigned warp_bound[MERGE_WARPS], heads[MERGE_THREADS];
  __shared__ float row_least[32];
  __shared__ int found, reaching;
  __shared__ double values[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.K, S = a.segments, lists = K * S;
  const long first = (long)blockIdx.x * K;
  if (tid == 0) found = reaching = 0;
  if (tid < K) chosen[tid] = (long)tid << 54;
  const int whole = min((lists + 31) / 32, MERGE_WARPS), mine = lane * whole + warp;  // this thread's first list
  const float per_list = 1.f / S;
  // (floor of i / S: i < 2^14 and S <= 512, so the half keeps the quotient 2^-10 off any whole number, 2^6 times its error)
  auto row_of = [&](int i) { return __float2int_rd((i + 0.5f) * per_list); };
  const unsigned long long first_head = warp < whole && mine < lists ? a.entries[(first * S + mine) * K] : 0ull;
  for (int b = warp; b < K; b += MERGE_WARPS) {
    const long row = first + b;
    // (what rows that do not run leave unwritten is loaded with the rest, in one wait for memory, and not used)
    float t[4], top = -INFINITY;
    double s[4], sum = 0.0;
    auto load = [&](int i0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * 32 + lane;
        t[j] = i < S ? a.tops[row * S + i] : -INFINITY;
        s[j] = i < S ? a.sums[row * S + i] : 0.0;
      }
    };
    load(0);
    const float score = a.scores[row];
    const bool finished = a.finished[row], run = !finished && isfinite(score);
    const int length = a.lengths[row] + (finished ? 0 : 1);
    for (int i0 = 0; i0 < S && run; i0 += 128) {
      if (i0) load(i0);
      float more = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) more = fmaxf(more, __shfl_xor_sync(~0u, more, o));
      if (more > top) {
        sum *= top == -INFINITY ? 0.0 : exp_of((double)top - (double)more);
        top = more;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (s[j] != 0.0) sum += s[j] * (t[j] == top ? 1.0 : exp_of((double)t[j] - (double)top));  // NaN stays
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) {
      const bool fit = sum > 0.0 && isfinite(sum) && isfinite(top);
      kind[b] = run && fit ? 0 : finished && isfinite(score) ? 1 : 2;
      base[b] = (double)score - (kind[b] == 0 ? log(sum) : 0.0);
      row_top[b] = top;
      next_length[b] = length;
      ended[b] = finished;
      norm[b] = a.penalty == 0.0 ? 1.0 : pow((double)max(length, 1), a.penalty);
    }
  }
  __syncthreads();
  auto entry_of = [&](int i, int j) { return kind[row_of(i)] == 0 && j < K ? a.entries[(first * S + i) * K + j] : 0ull; };
  // j-th entry of list i, which is e where its row runs (rank key 0: there is none)
  auto item = [&](int i, int j, unsigned long long e, unsigned long long& rank, long& flat, double& value) {
    const int b = row_of(i), seg = i - b * S;
    rank = 0;
    flat = LONG_MAX;
    value = -INFINITY;
    if (j >= K) return;
    int token;
    unsigned below = 0;  // falls with the logit
    if (kind[b] == 0) {
      if (e == 0) return;
      token = (int)~(unsigned)e;
      below = ~(unsigned)(e >> 32);
      const float z = key_value(~below);
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
    flat = (long)b << 54 | (long)below << 22 | token;  // equal ranks: beam, logit, token (of 22 bits)
  };
  // the upper half of a rank's key keeps its order. A warp's lists are spread over all beams, as they are not alike
  // (a thread may stand for several lists); each warp's k-th largest head, as in a segment
  unsigned best_head = 0;  // of this thread's lists
  if (warp < whole) {
    unsigned head = 0, t = 0;
    for (int i = mine; i < lists; i += 32 * whole) {
      unsigned long long r;
      long f;
      double v;
      item(i, 0, i == mine ? first_head : entry_of(i, 0), r, f, v);
      head = max(head, (unsigned)(r >> 32));
    }
    best_head = head;
    for (int k = (K + whole - 1) / whole; k > 0; --k) {
      t = __reduce_max_sync(~0u, head);
      const unsigned equal = __ballot_sync(~0u, head == t);
      if (lane == __ffs(equal) - 1) head = 0;
    }
    if (lane == 0) warp_bound[warp] = t;
    heads[warp * 32 + lane] = best_head;
  }
  __syncthreads();
  unsigned least = __reduce_min_sync(~0u, lane < whole ? warp_bound[lane] : ~0u);
  if (whole > 4) {  // many lists: a bound that is theirs and not each warp's (of fewer it would cost more than it saves)
    if (warp == 0) {
      unsigned key[MERGE_WARPS], above = 0;
#pragma unroll
      for (int i = 0; i < MERGE_WARPS; ++i) {
        key[i] = i < whole ? heads[i * 32 + lane] : 0u;
        above = max(above, key[i]);
      }
      unsigned below = least;  // K heads reach it
      above = __reduce_max_sync(~0u, above) + 1;
      while (above - below > 1) {
        const unsigned mid = below + (above - below) / 2;
        int reach = 0;
#pragma unroll
        for (int i = 0; i < MERGE_WARPS; ++i) reach += key[i] >= mid;
        reach = __reduce_add_sync(~0u, reach);
        if (reach < K) {
          above = mid;
        } else {
          below = mid;
          if (reach <= K + K / 4) break;
        }
      }
      if (lane == 0) warp_bound[0] = below;
    }
    __syncthreads();
    least = warp_bound[0];
  }
  least = max(least, 1u);
  auto offer = [&](int i, int j, unsigned long long e) {
    const int to = atomicAdd(&found, 1);
    if (to < MERGE_LIST) {
      list_rank[to] = e;
      list_flat[to] = i << 5 | j;
    }
  };
  // A row's candidates that can reach the bound have a logit of about (bound norm - base) + top; they are few, and only
  // they are ranked. Rank, value and the terms here are rounded by 2^-53 of one of the three terms each (a score of -3e38,
  // which a mask's lowest value leaves, swallows logits whole): the margin of 2^-48 of all, and of more than the logit's own
  // rounding, is far above that, and what it lets through is ranked in vain.
  if (tid < K) {
    const unsigned long long key = (unsigned long long)least << 32;
    const double rank = __longlong_as_double((long long)(key >> 63 ? key & ~(1ull << 63) : ~key));
    const double reach = rank * norm[tid], at_least = reach - base[tid] + (double)row_top[tid];
    const double margin = (fabs(reach) + fabs(base[tid]) + fabs((double)row_top[tid])) * 0x1p-48;
    // (NaN, of a bound below all numbers, lets everything through)
    row_least[tid] = __double2float_rd(at_least - margin - fabs(at_least) * 1e-6 - 1e-3);
  }
  // only lists whose head reaches the bound are read on: of 608 lists of 32 beams some 40, and 10 KB of 156
  unsigned* reached = heads;  // (which nobody reads any more)
  if (warp < whole && best_head >= least) reached[atomicAdd(&reaching, 1)] = mine;
  __syncthreads();
  // a lane per entry, 32 / K lists per warp
  const int per = 32 / K, sub = lane / K, j = lane - sub * K, slots = reaching;
  for (int more = 0; more < lists; more += 32 * whole)
    for (int w0 = warp * per + sub; w0 < slots; w0 += 2 * MERGE_WARPS * per) {
      unsigned long long in[2];
      int at[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int w = w0 + k * MERGE_WARPS * per;
        at[k] = w < slots ? (int)reached[w] + more : lists;
        in[k] = sub < per && at[k] < lists ? a.entries[(first * S + at[k]) * K + j] : 0ull;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int b = row_of(min(at[k], lists - 1));
        if (in[k] && kind[b] == 0 && !(key_value((unsigned)(in[k] >> 32)) < row_least[b])) offer(at[k], j, in[k]);
      }
    }
  const bool none_reach = least <= (unsigned)(rank_key(-INFINITY) >> 32);  // the bound is -inf
  for (int e = tid; e < K * K; e += MERGE_THREADS) {
    const int b = e / K;
    if (kind[b] != 0 && (none_reach || (kind[b] == 1 && e == b * K))) offer(b * S, e - b * K, 0ull);
  }
  __syncthreads();
  const int have = found;
  if (have <= MERGE_LIST) {
    for (int i = tid; i < have; i += MERGE_THREADS) {
      const int at = (int)list_flat[i];
      unsigned long long r;
      long f;
      double v;
      item(at >> 5, at & 31, list_rank[i], r, f, v);
      list_rank[i] = r;
      list_flat[i] = f;
      list_value[i] = v;
    }
    __syncthreads();
    for (int i = tid; i < have; i += MERGE_THREADS) {
      const unsigned long long r = list_rank[i];
      const long f = list_flat[i];
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < have; ++j) {  // (both are read whatever they say, so that the reads do not wait for one another)
        const unsigned long long other = list_rank[j];
        const long at = list_flat[j];
        place += (other > r) | ((other == r) & (at < f));
      }
      if (place < K) {
        chosen[place] = f;
        values[place] = list_value[i];
      }
    }
  } else {
    for (int i = tid; i < lists; i += MERGE_THREADS) taken[i] = 0;
    unsigned long long rank;
    long flat;
    int best;
    double value;
    auto refresh = [&]() {  // the best head of this thread's lists
      rank = 0;
      flat = LONG_MAX;
      best = -1;
      for (int i = tid; i < lists; i += MERGE_THREADS) {
        unsigned long long r;
        long f;
        double v;
        item(i, taken[i], entry_of(i, taken[i]), r, f, v);
        if (r > rank || (r == rank && f < flat)) {
          rank = r;
          flat = f;
          best = i;
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
      if (best >= 0 && flat == best_flat && rank == best_rank) {
        chosen[n] = flat;
        values[n] = value;
        ++taken[best];
        refresh();
      }
    }
  }
  __syncthreads();
  if (warp != 0) return;
  // ---- slots: a parent's best child keeps the parent's, the others fill what is left in order
  const bool in = lane < K;
  const unsigned all = K == 32 ? ~0u : (1u << K) - 1;
  const int parent = in ? (int)(chosen[lane] >> 54) : 32 + lane;
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
  const long token = chosen[lane] & ((1 << 22) - 1), to = first + slot;
  a.tokens[to] = token;
  a.parents[to] = parent;
  a.out_scores[to] = (float)values[lane];
  a.out_lengths[to] = next_length[parent];
  a.out_finished[to] = ended[parent] || token == a.end_token;
}

// Segments of a beam's vocabulary: enough for four blocks per SM, of 1024 values at least.
int segments_for(long rows, long V) {
  const long least = (V + SEGMENT - 1) / SEGMENT;
  const long spread = std::min({(592 + rows - 1) / rows, V / 1024, 128L});
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
  // (a warp per beam and a thread per list are enough: the barriers of a smaller block are cheaper)
  if (K <= 8 && K * a.segments <= 256) select_group_kernel<256><<<(unsigned)groups, 256, K * a.segments, s>>>(a);
  else select_group_kernel<1024><<<(unsigned)groups, 1024, K * a.segments, s>>>(a);
  return cudaGetLastError();
}
