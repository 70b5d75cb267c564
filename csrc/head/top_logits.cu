// The k largest log-probabilities of each row of logits, largest first, equal logits by the lowest index.
//
// One read of the logits. A row is streamed in groups of 8 or 32 values, whose maxima stay in shared memory, while the
// softmax's denominator is summed. A value t that k of the maxima reach is reached by k logits at least, so the result
// lies in the groups whose maximum reaches t. t is the k-th largest of 1.5 k maxima or more over several groups each,
// found by one warp's bisection of their order-preserving keys; the groups that reach it (about 1.4 k at most) are read
// again, and their values from t up are sorted as unique 64-bit keys (value above, lower index first below). Rows whose
// equal or special values defeat the bounds (thousands of equal maxima, infinities, NaN) take a radix descent over the
// whole row instead.
//
// Bound by memory: per value one packed maximum's half, unpacking, packed subtraction, product and sum, and ex2
// (about 5.5 issue slots of the 11 that the bandwidth leaves). Several blocks per SM, so that one streams while
// another selects. Few rows are cut into segments over as many blocks, whose k candidates a second kernel merges.
#include <algorithm>
#include <atomic>
#include <climits>
#include "../api.h"
#include "../common/common.cuh"

namespace {

constexpr int THREADS = 384, WARPS = THREADS / 32;
constexpr int MAX_KEYS = 8192;     // group maxima of a segment
constexpr int MAX_GROUPS = 2048;   // groups read again
constexpr int BATCH = 4;           // vectors of 16 bytes in flight per thread
constexpr float LOG2E = 1.4426950408889634f;

// Order-preserving 32-bit key of a logit: -0 equals +0, NaN is above every number; 0 is below all of them.
__device__ __forceinline__ unsigned order_key(float v) {
  if (v != v) return 0xffffffffu;
  const unsigned b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// Of a maximum, which is no NaN.
__device__ __forceinline__ unsigned max_key(float v) {
  const int b = __float_as_int(v + 0.f);
  return (unsigned)b ^ ((unsigned)(b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ unsigned long long entry(unsigned key, int index) {
  return (unsigned long long)key << 32 | (unsigned)~index;
}

// Group maxima in shared memory: a bf16's key fits the upper half of its 32-bit key.
template <typename T> struct Key { using type = unsigned; };
template <> struct Key<__nv_bfloat16> { using type = unsigned short; };
template <typename T> __device__ __forceinline__ typename Key<T>::type pack_key(unsigned key) {
  return (typename Key<T>::type)(sizeof(T) == 2 ? key >> 16 : key);
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

// (max of logits, sum of exp2(c (logit - max))).
__device__ __forceinline__ float2 merge(float2 a, float2 b, float c) {
  const float m = fmaxf(a.x, b.x);
  const float fa = a.x == m ? 1.f : exp2f((a.x - m) * c), fb = b.x == m ? 1.f : exp2f((b.x - m) * c);
  return make_float2(m, a.y * fa + b.y * fb);
}

__device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) { rt::unpack8(u, f); }
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
  f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ float vec_max(const uint4& u, const __nv_bfloat16*) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&u);
  const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float vec_max(const uint4& u, const float*) {
  float f[4];
  unpack(u, f);
  return fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
}

// Sum over the block of a per-thread count (every thread gets it). `slot` cycles over three counters.
__device__ __forceinline__ int block_count(int n, int* counters, int& slot) {
  n = __reduce_add_sync(~0u, n);
  if ((threadIdx.x & 31) == 0 && n) atomicAdd(&counters[slot], n);
  if (threadIdx.x == 0) counters[slot == 2 ? 0 : slot + 1] = 0;
  __syncthreads();
  const int total = counters[slot];
  slot = slot == 2 ? 0 : slot + 1;
  return total;
}

// By one warp: the largest t found that at least k of maxima[0, 32 each) reach and, as far as they differ, few more (0
// where fewer than k are above 0). `top` is their largest.
template <typename K>
__device__ __forceinline__ unsigned reached_by(const K* maxima, int each, int k, unsigned top) {
  constexpr int HELD = 16;  // per lane in registers, which serves records of up to 256
  const int lane = threadIdx.x & 31;
  unsigned r[HELD], least = top;
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    r[j] = j < each ? (unsigned)maxima[j * 32 + lane] : 0u;
    if (j < each) least = min(least, r[j]);
  }
  for (int j = HELD; j < each; ++j) least = min(least, (unsigned)maxima[j * 32 + lane]);
  unsigned below = __reduce_min_sync(~0u, least), above = top + 1;  // all of them reach `below`
  while (above - below > 1) {
    const unsigned mid = below + (above - below) / 2;
    int count = 0;
#pragma unroll
    for (int j = 0; j < HELD; ++j) count += r[j] >= mid;
    for (int j = HELD; j < each; ++j) count += (unsigned)maxima[j * 32 + lane] >= mid;
    count = __reduce_add_sync(~0u, count);
    if (count < k) {
      above = mid;
    } else {
      below = mid;
      if (count <= k + k / 8) break;
    }
  }
  return below;
}

// Keys of 16 bytes at once: their maximum, and the j-th.
template <typename K> struct KeyVec;
template <> struct KeyVec<unsigned short> {
  static constexpr int N = 8;
  static __device__ __forceinline__ unsigned max(const uint4& u) {
    const unsigned m = __vmaxu2(__vmaxu2(u.x, u.y), __vmaxu2(u.z, u.w));
    return ::max(m & 0xffffu, m >> 16);
  }
  static __device__ __forceinline__ unsigned at(const uint4& u, int j) {
    const unsigned w = j < 4 ? (j < 2 ? u.x : u.y) : (j < 6 ? u.z : u.w);
    return j & 1 ? w >> 16 : w & 0xffffu;
  }
};
template <> struct KeyVec<unsigned> {
  static constexpr int N = 4;
  static __device__ __forceinline__ unsigned max(const uint4& u) { return ::max(::max(u.x, u.y), ::max(u.z, u.w)); }
  static __device__ __forceinline__ unsigned at(const uint4& u, int j) {
    return j < 2 ? (j < 1 ? u.x : u.y) : (j < 3 ? u.z : u.w);
  }
};

// list[0, n) sorted downwards; its capacity is a power of two of at least n. Entries are unique but for zeros.
__device__ void sort_down(unsigned long long* list, int n) {
  int np = 1;
  while (np < n) np <<= 1;
  for (int i = n + threadIdx.x; i < np; i += blockDim.x) list[i] = 0;
  __syncthreads();
  for (int size = 2; size <= np; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int i = threadIdx.x; i < np / 2; i += blockDim.x) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const unsigned long long a = list[lo], b = list[hi];
        if ((a < b) == ((lo & size) == 0)) {
          list[lo] = b;
          list[hi] = a;
        }
      }
      __syncthreads();
    }
}

// The k largest entries of z[0, n) into list, unsorted, by a radix descent over the keys' bytes: five reads of the row.
template <typename T>
__device__ __noinline__ void descend(const T* z, int n, int k, unsigned long long* list) {
  __shared__ int hist[256];
  __shared__ int found, need, digit, wsum[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned prefix = 0, seen = 0;
  int left = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
    __syncthreads();
    for (int v = tid; v < n; v += THREADS) {
      const unsigned key = order_key(rt::to_f<T>(z[v]));
      if ((key & seen) == prefix) atomicAdd(&hist[key >> shift & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255;
      while (d > 0 && left > hist[d]) left -= hist[d--];
      digit = d;
      need = left;
    }
    __syncthreads();
    prefix |= (unsigned)digit << shift;
    seen |= 255u << shift;
    left = need;
    __syncthreads();
  }
  if (tid == 0) found = 0;
  __syncthreads();
  int equal = 0;  // entries above the threshold in any order, the first `left` equal ones in index order
  for (int base = 0; base < n; base += THREADS) {
    const int v = base + tid;
    const unsigned key = v < n ? order_key(rt::to_f<T>(z[v])) : 0u;
    if (v < n && key > prefix) list[atomicAdd(&found, 1)] = entry(key, v);
    const bool same = v < n && key == prefix;
    const unsigned ballot = __ballot_sync(~0u, same);
    if (lane == 0) wsum[warp] = __popc(ballot);
    __syncthreads();
    int before = equal + __popc(ballot & ((1u << lane) - 1)), all = 0;
    for (int w = 0; w < WARPS; ++w) {
      before += w < warp ? wsum[w] : 0;
      all += wsum[w];
    }
    if (same && before < left) list[k - left + before] = entry(key, v);
    equal += all;
    __syncthreads();
  }
}

struct TopArgs {
  long ld;
  int V, k, segments, capacity;  // capacity of the list, a power of two of at least 2 k
  float scale;
  float* logp;                   // [rows, k]
  long* index;
  unsigned long long* entries;   // segments > 1: [rows, segments, k], zeros behind a short segment's values
  float2* sums;                  // [rows, segments]
};

// list[0, n), n >= min(k, available): the row's result from its candidates and denominator.
__device__ void write_row(const TopArgs& a, long row, unsigned long long* list, int n, float2 ms) {
  const float log_sum = logf(ms.y);
  auto put = [&](int rank, unsigned long long e) {
    a.index[row * a.k + rank] = (long)(int)~(unsigned)e;
    a.logp[row * a.k + rank] = (key_value((unsigned)(e >> 32)) - ms.x) * a.scale - log_sum;
  };
  if (n <= 512) {  // place = number of larger entries
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const unsigned long long e = list[i];
      int rank = 0;
      const ulonglong2* two = reinterpret_cast<const ulonglong2*>(list);
#pragma unroll 8
      for (int j = 0; j < n / 2; ++j) rank += (two[j].x > e) + (two[j].y > e);
      if (n & 1) rank += list[n - 1] > e;
      if (rank < a.k) put(rank, e);
    }
    return;
  }
  sort_down(list, n);
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) put(i, list[i]);
}

// Block (segment, row). U = vectors of a group: 1, or BATCH for long segments.
template <typename T, int U>
__global__ void __launch_bounds__(THREADS, 4) top_kernel(const T* __restrict__ logits, const TopArgs a) {
  constexpr int VEC = 16 / sizeof(T);
  using K = typename Key<T>::type;
  extern __shared__ __align__(16) uint8_t smem[];
  unsigned long long* list = reinterpret_cast<unsigned long long*>(smem);
  K* keys = reinterpret_cast<K*>(list + a.capacity);
  K* maxima = reinterpret_cast<K*>(list);  // until candidates are listed
  __shared__ int picked, found;
  __shared__ unsigned bound;
  __shared__ float2 warps[WARPS];
  __shared__ unsigned short groups[MAX_GROUPS];
  const int tid = threadIdx.x, lane = tid & 31;
  const long row = blockIdx.y;
  const int lo = (int)((long)a.V * blockIdx.x / a.segments), n = (int)((long)a.V * (blockIdx.x + 1) / a.segments) - lo;
  const T* z = logits + row * a.ld + lo;
  const float c = a.scale * LOG2E;
  // aligned vectors, and the few values before and behind them, one per thread
  const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / (int)sizeof(T));
  const int nvec = (n - head) / VEC, tail = n - head - nvec * VEC;
  const uint4* zv = reinterpret_cast<const uint4*>(z + head);
  int single = -1;
  if (tid < head) single = tid;
  else if (tid >= 16 && tid < 16 + tail) single = n - tail + (tid - 16);
  if (tid == 0) picked = found = 0;

  float m = -INFINITY, s = 0.f;
  bool special = false;  // NaN or +inf: left to the descent
  unsigned single_key = 0;
  if (single >= 0) {
    const float v = rt::to_f<T>(z[single]);
    single_key = order_key(v);
    special = !(v < INFINITY);
    if (v > -INFINITY) {
      m = v;
      s = 1.f;
    }
    if (special) s = NAN;
  }
  const int steps = (nvec + BATCH * THREADS - 1) / (BATCH * THREADS);
  auto step = [&](int it, bool whole) {
    uint4 u[BATCH];
    float g[BATCH];
    const int v0 = it * BATCH * THREADS + tid;
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;  // -inf
      if (whole || v0 + b * THREADS < nvec) u[b] = __ldg(zv + v0 + b * THREADS);
      else u[b] = make_uint4(none, none, none, none);
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b) g[b] = vec_max(u[b], (const T*)nullptr);
    const float top = fmaxf(fmaxf(g[0], g[1]), fmaxf(g[2], g[3]));
    if (U == 1) {
#pragma unroll
      for (int b = 0; b < BATCH; ++b)
        keys[(it * BATCH + b) * THREADS + tid] =
            whole || v0 + b * THREADS < nvec ? pack_key<T>(max_key(g[b])) : (K)0;
    } else {
      keys[it * THREADS + tid] = whole || v0 < nvec ? pack_key<T>(max_key(top)) : (K)0;
    }
    if (top > m) {
      s *= m == -INFINITY ? 0.f : ex2((m - top) * c);
      m = top;
    }
    // c (f - m) and not c f - c m: a mask of the type's lowest value times c is beyond fp32
    const float less = m == -INFINITY ? 0.f : -m;
    float2 sum = make_float2(0.f, 0.f);
    const float2 c2 = make_float2(c, c), less2 = make_float2(less, less);
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      float f[VEC];
      unpack(u[b], f);
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        const float2 y = mul2(add2(make_float2(f[j], f[j + 1]), less2), c2);
        sum = add2(sum, make_float2(ex2(y.x), ex2(y.y)));
      }
    }
    s += sum.x + sum.y;
  };
  const int whole = nvec / (BATCH * THREADS);
  for (int it = 0; it < whole; ++it) step(it, true);
  if (whole < steps) step(whole, false);
  float2 o = make_float2(m, s);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    o = merge(o, make_float2(__shfl_xor_sync(~0u, o.x, off), __shfl_xor_sync(~0u, o.y, off)), c);
  if (lane == 0) warps[tid >> 5] = o;
  __syncthreads();
  o = warps[0];
  for (int w = 1; w < WARPS; ++w) o = merge(o, warps[w], c);

  // ---- threshold: THREADS x parts maxima, each of one thread's every parts-th group; the k-th largest of them
  const int slots = steps * THREADS * (U == 1 ? BATCH : 1), vecs = slots / KeyVec<K>::N;
  const uint4* kv = reinterpret_cast<const uint4*>(keys);
  unsigned threshold = 0;  // every value, where there are few groups
  // NaN and +inf make the sum NaN; a row of -inf has nothing above it
  bool ok = !special && o.y == o.y && o.x > -INFINITY;
  ok = !__syncthreads_or(!ok);
  if (ok && slots > max(2 * a.k, 128)) {
    // (by 16 bytes of keys, or by single keys where the row is too short for that many)
    const bool wide = nvec / (U * KeyVec<K>::N) >= 2 * a.k;
    int parts = 1;
    while (parts < 8 && parts * THREADS * 2 < 3 * a.k) parts <<= 1;
    for (int p = 0; p < parts; ++p) {
      unsigned best = 0;
      if (wide) {
#pragma unroll 2
        for (int i = tid + p * THREADS; i < vecs; i += parts * THREADS) best = max(best, KeyVec<K>::max(kv[i]));
      } else {
        for (int i = tid + p * THREADS; i < slots; i += parts * THREADS) best = max(best, (unsigned)keys[i]);
      }
      maxima[p * THREADS + tid] = (K)best;
    }
    __syncthreads();
    if (tid < 32) {
      const int shift = sizeof(T) == 2 ? 16 : 0;
      const unsigned t = reached_by(maxima, WARPS * parts, a.k, order_key(o.x) >> shift) << shift;
      if (lane == 0) bound = t;
    }
    __syncthreads();
    threshold = bound;
  }
  // ---- candidates
  if (ok) {
    const unsigned tk = max((unsigned)pack_key<T>(threshold), 1u);
#pragma unroll 2
    for (int i = tid; i < vecs; i += THREADS) {
      const uint4 u = kv[i];
      if (KeyVec<K>::max(u) < tk) continue;
#pragma unroll
      for (int j = 0; j < KeyVec<K>::N; ++j)
        if (KeyVec<K>::at(u, j) >= tk) {
          const int at = atomicAdd(&picked, 1);
          if (at < MAX_GROUPS) groups[at] = (unsigned short)(i * KeyVec<K>::N + j);
        }
    }
    if (single >= 0 && single_key >= threshold) {
      const int at = atomicAdd(&found, 1);
      if (at < a.capacity) list[at] = entry(single_key, lo + single);
    }
    __syncthreads();
    ok = picked <= MAX_GROUPS;
    const int lines = ok ? picked * U : 0;
    for (int i = tid; i < lines; i += 2 * THREADS) {
      int v[2];
      uint4 u[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = i + h * THREADS, g = at < lines ? groups[at / U] : 0;
        v[h] = U == 1 ? g : (g / THREADS) * BATCH * THREADS + (at % U) * THREADS + g % THREADS;
        if (at >= lines || v[h] >= nvec) v[h] = -1;
        if (v[h] >= 0) u[h] = __ldg(zv + v[h]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (v[h] < 0) continue;
        float f[VEC];
        unpack(u[h], f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const unsigned key = order_key(f[j]);
          if (key >= threshold) {
            const int at = atomicAdd(&found, 1);
            if (at < a.capacity) list[at] = entry(key, lo + head + v[h] * VEC + j);
          }
        }
      }
    }
    __syncthreads();
    ok = ok && found <= a.capacity;
  }
  int have = found;
  if (!ok) {
    have = min(n, a.k);
    __syncthreads();
    descend<T>(z, n, have, list);
    __syncthreads();
    for (int i = tid; i < have; i += THREADS) list[i] -= (unsigned)lo;  // ~(index + lo) = ~index - lo
    __syncthreads();
  }
  if (a.segments == 1) {
    write_row(a, row, list, have, o);
    return;
  }
  const long at = row * a.segments + blockIdx.x;
  if (tid == 0) a.sums[at] = o;
  if (have > a.k) sort_down(list, have);
  for (int i = tid; i < a.k; i += THREADS) a.entries[at * a.k + i] = i < have ? list[i] : 0ull;
}

constexpr int MERGE_THREADS = 512, MERGE_EACH = 16;

// Block per row: the segments' candidates, at most MERGE_THREADS x MERGE_EACH. The threshold is found as above, from
// the maxima of one or a few candidates each; where too many are equal to it, by bisection of the unique 64-bit keys.
__global__ void __launch_bounds__(MERGE_THREADS) top_merge_kernel(const TopArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  unsigned long long* list = reinterpret_cast<unsigned long long*>(smem);
  unsigned* maxima = reinterpret_cast<unsigned*>(smem);  // until candidates are listed
  __shared__ int counters[3], found;
  __shared__ unsigned peak, bound;
  __shared__ float2 sums[MERGE_THREADS / 32];
  const long row = blockIdx.x;
  const int tid = threadIdx.x, total = a.segments * a.k, parts = a.k <= MERGE_THREADS / 2 ? 1 : 4;
  const unsigned long long* in = a.entries + row * total;
  unsigned long long e[MERGE_EACH];
  unsigned top = 0, part_top = 0;
#pragma unroll
  for (int j = 0; j < MERGE_EACH; ++j) {
    e[j] = j * MERGE_THREADS + tid < total ? in[j * MERGE_THREADS + tid] : 0ull;
    part_top = max(part_top, (unsigned)(e[j] >> 32));
    if (parts == 1 ? j == MERGE_EACH - 1 : j % 4 == 3) {
      maxima[(parts == 1 ? 0 : j / 4) * MERGE_THREADS + tid] = part_top;
      top = max(top, part_top);
      part_top = 0;
    }
  }
  const float c = a.scale * LOG2E;
  float2 ms = make_float2(-INFINITY, 0.f);
  for (int i = tid; i < a.segments; i += MERGE_THREADS) ms = merge(ms, a.sums[row * a.segments + i], c);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    ms = merge(ms, make_float2(__shfl_xor_sync(~0u, ms.x, off), __shfl_xor_sync(~0u, ms.y, off)), c);
  top = __reduce_max_sync(~0u, top);
  if (tid == 0) counters[0] = counters[1] = counters[2] = found = peak = 0;
  __syncthreads();
  if ((tid & 31) == 0) {
    atomicMax(&peak, top);
    sums[tid >> 5] = ms;
  }
  __syncthreads();
  ms = sums[0];
#pragma unroll
  for (int w = 1; w < MERGE_THREADS / 32; ++w) ms = merge(ms, sums[w], c);
  if (tid < 32) {
    // a NaN's key is the largest there is: one less, as its successor has to exist
    const unsigned t = reached_by(maxima, parts * MERGE_THREADS / 32, a.k, min(peak, 0xfffffffeu));
    if (tid == 0) bound = t;
  }
  __syncthreads();
  unsigned long long below = max(1ull, (unsigned long long)bound << 32);
  int count = 0, slot = 0;
#pragma unroll
  for (int j = 0; j < MERGE_EACH; ++j) count += e[j] >= below;
  count = block_count(count, counters, slot);
  if (count > a.capacity) {
    unsigned long long above = ~0ull;  // no entry: its index would be 0 and its key a NaN's, and it alone reaches it
    while (above - below > 1) {
      const unsigned long long mid = below + (above - below) / 2;
      count = 0;
#pragma unroll
      for (int j = 0; j < MERGE_EACH; ++j) count += e[j] >= mid;
      count = block_count(count, counters, slot);
      if (count < a.k) {
        above = mid;
      } else {
        below = mid;
        if (count <= a.capacity) break;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < MERGE_EACH; ++j)
    if (e[j] >= below) list[atomicAdd(&found, 1)] = e[j];
  __syncthreads();
  write_row(a, row, list, found, ms);
}

constexpr int capacity_for(int k) {
  int c = 1024;
  while (c < 4 * k) c <<= 1;
  return c;
}
// Dynamic shared memory of a block whose segment has `vecs` vectors.
template <typename T, int U>
constexpr size_t smem_for(int capacity, long vecs) {
  const long steps = (vecs + BATCH * THREADS - 1) / (BATCH * THREADS);
  return (size_t)capacity * 8 + (size_t)steps * THREADS * (U == 1 ? BATCH : 1) * sizeof(typename Key<T>::type);
}

// Segments of a row. One block takes a row of 32003 values in 10 us and of 248077 in 20 us, and merging segments costs
// another launch of about 8 us, so only a few long rows are cut (8 segments of 1 x 248077 bf16, k 64: 18.7 us), and
// rows with more vectors than a segment's maxima have room for (past a million values, a long record may not fit: 0).
int segments_for(int dtype, long rows, long V, int k) {
  const int vec = dtype == 1 ? 8 : 4;
  const long least = (V / vec + (long)MAX_KEYS * BATCH - 1) / ((long)MAX_KEYS * BATCH);
  const long spread = rows <= 16 && k <= 128 && V / vec >= 7 * MAX_KEYS * BATCH / 8 ? 8 : 1;
  const long segments = std::max({1L, least, spread});
  return segments == 1 || segments * k <= MERGE_THREADS * MERGE_EACH ? (int)segments : 0;
}

template <typename T, int U>
cudaError_t launch(const T* logits, long rows, const TopArgs& a, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  const long longest = (a.V + a.segments - 1) / a.segments;
  const size_t smem = smem_for<T, U>(a.capacity, longest / VEC);
  // The longest segment and record; the limit belongs to the device and not to the call, so it is raised once.
  constexpr size_t most = smem_for<T, U>(capacity_for(RT_HEAD_MAX_RECORD), (long)MAX_KEYS * (U == 1 ? 1 : BATCH) + 1);
  if (smem > most) return cudaErrorInvalidValue;
  static std::atomic<uint64_t> set{0};  // devices
  int dev = 0;
  RT_CUDA_CHECK(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!bit || !(set.load(std::memory_order_acquire) & bit)) {
    RT_CUDA_CHECK(cudaFuncSetAttribute(top_kernel<T, U>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    set.fetch_or(bit, std::memory_order_acq_rel);
  }
  for (long r = 0; r < rows; r += 65535) {
    const long some = std::min(rows - r, 65535L);
    TopArgs b = a;
    b.logp += r * a.k;
    b.index += r * a.k;
    b.entries += r * a.segments * a.k;
    b.sums += r * a.segments;
    top_kernel<T, U><<<dim3((unsigned)a.segments, (unsigned)some), THREADS, smem, s>>>(logits + r * a.ld, b);
  }
  return cudaGetLastError();
}

}  // namespace

extern "C" long rt_top_workspace_bytes(int dtype, long rows, long V, int k) {
  const int s = segments_for(dtype, rows, V, k);
  return s > 1 ? rows * s * (8L * k + 8) : s - 1;  // -1: too many logits for a record of this length
}

// dtype 1 = bf16, 0 = fp32; logits [rows, V] with row stride ld; logp, index [rows, k]; work: rt_top_workspace_bytes,
// 16-byte aligned.
extern "C" cudaError_t rt_top_log_probs(int dtype, const void* logits, long rows, long V, long ld, int k, float scale,
                                        float* logp, long* index, void* work, cudaStream_t s) {
  if (rows < 0 || rows > INT_MAX || V < 1 || V > INT_MAX / 2 || k < 1 || k > V || k > RT_HEAD_MAX_RECORD)
    return cudaErrorInvalidValue;
  if (rows == 0) return cudaSuccess;
  TopArgs a{};
  a.ld = ld;
  a.V = (int)V;
  a.k = k;
  a.segments = segments_for(dtype, rows, V, k);
  a.capacity = capacity_for(k);
  a.scale = scale;
  a.logp = logp;
  a.index = index;
  if (a.segments == 0 || (a.segments > 1 && !work)) return cudaErrorInvalidValue;
  if (a.segments > 1) {
    a.entries = static_cast<unsigned long long*>(work);
    a.sums = reinterpret_cast<float2*>(a.entries + rows * a.segments * k);
  }
  const long values = (V + a.segments - 1) / a.segments;
  if (dtype == 1) {
    const auto* z = static_cast<const __nv_bfloat16*>(logits);
    RT_CUDA_CHECK((values / 8 <= MAX_KEYS ? launch<__nv_bfloat16, 1>(z, rows, a, s)
                                          : launch<__nv_bfloat16, BATCH>(z, rows, a, s)));
  } else {
    const auto* z = static_cast<const float*>(logits);
    RT_CUDA_CHECK((values / 4 <= MAX_KEYS ? launch<float, 1>(z, rows, a, s) : launch<float, BATCH>(z, rows, a, s)));
  }
  if (a.segments > 1) top_merge_kernel<<<(unsigned)rows, MERGE_THREADS, a.capacity * 8, s>>>(a);
  return cudaGetLastError();
}
