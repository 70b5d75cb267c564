// The k largest log-probabilities of each row of logits, largest first, equal logits by the lowest index.
#include <climits>
#include "../api.h"
#include "../common/common.cuh"

namespace {

// Order-preserving 32-bit key of a logit: -0 equals +0, and NaN is above every number.
__device__ __forceinline__ unsigned order_key(float v) {
  if (v != v) return 0xffffffffu;
  const unsigned b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int THREADS = 512, WARPS = THREADS / 32;

// Block per row: the k-th largest key by a radix descent over its four bytes, then the entries above it and the first
// ones equal to it, sorted. The first sweep also sums the softmax's denominator.
template <typename T>
__global__ void __launch_bounds__(THREADS) top_kernel(const T* __restrict__ logits, long ld, int V, int k, int kp,
                                                      float scale, float* __restrict__ logp, long* __restrict__ index) {
  extern __shared__ unsigned long long pick[];  // kp entries: key above, ~index below
  __shared__ int hist[256];
  __shared__ int found, need, digit, wsum[WARPS];
  __shared__ float2 warps[WARPS];
  __shared__ float lse;
  const T* z = logits + blockIdx.x * ld;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned prefix = 0, seen = 0;
  int left = k;
  float m = -INFINITY, s = 0.f;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
    __syncthreads();
    for (int v = tid; v < V; v += THREADS) {
      const float x = rt::to_f<T>(z[v]);
      const unsigned key = order_key(x);
      if ((key & seen) == prefix) atomicAdd(&hist[key >> shift & 255], 1);
      if (shift == 24) {
        const float y = x * scale;
        if (y > m) {
          s *= expf(m - y);
          m = y;
        }
        s += y == -INFINITY && m == -INFINITY ? 0.f : expf(y - m);
      }
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
  auto merge = [](float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    const float fa = a.x == -INFINITY ? 1.f : expf(a.x - m), fb = b.x == -INFINITY ? 1.f : expf(b.x - m);
    return make_float2(m, a.y * fa + b.y * fb);
  };
  float2 o = make_float2(m, s);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    o = merge(o, make_float2(__shfl_xor_sync(~0u, o.x, off), __shfl_xor_sync(~0u, o.y, off)));
  if (lane == 0) warps[warp] = o;
  for (int i = tid; i < kp; i += THREADS) pick[i] = 0;
  if (tid == 0) found = 0;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < WARPS; ++w) o = merge(o, warps[w]);
    lse = o.x + logf(o.y);
  }
  // entries above the threshold in any order, the first `left` equal ones in index order
  int equal = 0;
  for (int base = 0; base < V; base += THREADS) {
    const int v = base + tid;
    const unsigned key = v < V ? order_key(rt::to_f<T>(z[v])) : 0u;
    const unsigned long long entry = (unsigned long long)key << 32 | (unsigned)~v;
    if (v < V && key > prefix) pick[atomicAdd(&found, 1)] = entry;
    const bool same = v < V && key == prefix;
    const unsigned ballot = __ballot_sync(~0u, same);
    if (lane == 0) wsum[warp] = __popc(ballot);
    __syncthreads();
    int before = equal + __popc(ballot & ((1u << lane) - 1)), all = 0;
    for (int w = 0; w < WARPS; ++w) {
      before += w < warp ? wsum[w] : 0;
      all += wsum[w];
    }
    if (same && before < left) pick[k - left + before] = entry;
    equal += all;
    __syncthreads();
  }
  for (int size = 2; size <= kp; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int i = tid; i < kp / 2; i += THREADS) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const bool down = (lo & size) == 0;
        const unsigned long long a = pick[lo], b = pick[hi];
        if ((a < b) == down) {
          pick[lo] = b;
          pick[hi] = a;
        }
      }
      __syncthreads();
    }
  for (int i = tid; i < k; i += THREADS) {
    const int v = (int)~(unsigned)pick[i];
    index[(long)blockIdx.x * k + i] = v;
    logp[(long)blockIdx.x * k + i] = rt::to_f<T>(z[v]) * scale - lse;
  }
}

}  // namespace

// dtype 1 = bf16, 0 = fp32; logits [rows, V] with row stride ld; logp, index [rows, k].
extern "C" cudaError_t rt_top_log_probs(int dtype, const void* logits, long rows, long V, long ld, int k, float scale,
                                        float* logp, long* index, cudaStream_t s) {
  if (rows < 0 || rows > INT_MAX || V < 1 || V > INT_MAX - THREADS || k < 1 || k > V || k > RT_HEAD_MAX_RECORD)
    return cudaErrorInvalidValue;
  if (rows == 0) return cudaSuccess;
  int kp = 1;
  while (kp < k) kp <<= 1;
  if (dtype == 1)
    top_kernel<__nv_bfloat16><<<(unsigned)rows, THREADS, kp * 8, s>>>((const __nv_bfloat16*)logits, ld, (int)V, k, kp,
                                                                     scale, logp, index);
  else
    top_kernel<float><<<(unsigned)rows, THREADS, kp * 8, s>>>((const float*)logits, ld, (int)V, k, kp, scale, logp,
                                                             index);
  return cudaGetLastError();
}
