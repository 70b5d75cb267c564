// Losses of the vocabulary head from hidden states: next-token cross entropy and the KL from a teacher's recorded top
// log-probabilities, with the gradients of the hidden states and of the head's weight. The logits are formed in pieces
// of the vocabulary and never kept.
//
// With z_tv = scale x_t . W_v, a row's record is a set S of held entries (v, log p_v); the cross entropy's record is
// its target with p = 1. With P = sum_S p, r = max(0, 1 - P) (the rest as one more class, or 0 without it), w = P + r,
// Z = sum_v exp z_v and Z_rest = sum_{v not in S} exp z_v:
//   loss  = sum_S p (log p - z_v + log Z) + r (log r - log Z_rest + log Z)
//   d/dz_v = w exp(z_v) / Z - p_v                       (v in S)
//          = exp(z_v) / Z (w - r Z / Z_rest)            (v not in S)
// Z_rest is summed without the held entries instead of as Z minus them, so a row that is sure of its target keeps the
// relative precision of 1 - q. All sums and row statistics are fp32 (the few held terms of a row: double).
#include <algorithm>
#include <climits>
#include "../api.h"
#include "../common/common.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// ---------------------------------------------------------------- records
// One block per row: held entries sorted by vocabulary index (entries outside the record last, as INT_MAX), their
// log-probabilities in the same order, and the row's kind: 0 no entry (no loss), 1 valid, 2 an index outside the
// vocabulary (its loss is NaN and its gradient zero). K is padded to a power of two in shared memory.
__global__ void records_kernel(const long* __restrict__ idx, const float* __restrict__ logp, int K, int Kp, long V,
                               long ignore, int* __restrict__ sidx, float* __restrict__ slogp,
                               int* __restrict__ kind) {
  extern __shared__ unsigned long long keys[];
  const long row = blockIdx.x;
  __shared__ int bad, held;
  if (threadIdx.x == 0) bad = held = 0;
  __syncthreads();
  for (int k = threadIdx.x; k < Kp; k += blockDim.x) {
    int v = INT_MAX;
    float lp = 0.f;
    if (k < K) {
      const long id = idx[row * K + k];
      const bool none = logp ? id < 0 : id == ignore;
      if (!none) {
        if (id < 0 || id >= V) atomicOr(&bad, 1);
        else {
          v = (int)id;
          lp = logp ? logp[row * K + k] : 0.f;
          atomicOr(&held, 1);
        }
      }
    }
    keys[k] = ((unsigned long long)v << 32) | __float_as_uint(lp);
  }
  __syncthreads();
  for (int size = 2; size <= Kp; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int i = threadIdx.x; i < Kp / 2; i += blockDim.x) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const bool up = (lo & size) == 0;
        const unsigned long long a = keys[lo], b = keys[hi];
        if ((a > b) == up) {
          keys[lo] = b;
          keys[hi] = a;
        }
      }
      __syncthreads();
    }
  for (int k = threadIdx.x; k < K; k += blockDim.x) {
    sidx[row * K + k] = (int)(keys[k] >> 32);
    slogp[row * K + k] = __uint_as_float((unsigned)keys[k]);
  }
  if (threadIdx.x == 0) kind[row] = bad ? 2 : held;
}

// count[0] = rows with a loss (valid or NaN).
__global__ void count_kernel(const int* __restrict__ kind, long rows, int* __restrict__ count) {
  __shared__ float scratch[32];
  int n = 0;
  for (long t = threadIdx.x; t < rows; t += blockDim.x) n += kind[t] != 0;
  const float total = rt::block_sum((float)n, scratch);
  if (threadIdx.x == 0) count[0] = (int)total;
}

// ---------------------------------------------------------------- logits of the held entries
// hit[row, k] = scale2 x_row . W_sidx (units of log2), one warp per entry. These logits enter the loss with a weight
// of about one, where all others enter it through the sum of exponentials, so they are summed by fp32 fused
// multiply-adds, which round, instead of on the tensor cores, which truncate (see mma_gain).
__global__ void __launch_bounds__(256) held_logits_kernel(const __nv_bfloat16* __restrict__ x, long ldx,
                                                          const __nv_bfloat16* __restrict__ w, long ldw, int C,
                                                          long entries, int K, const int* __restrict__ sidx,
                                                          float scale2, float* __restrict__ hit) {
  const long e = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (e >= entries) return;
  const int v = sidx[e];
  if (v == INT_MAX) return;
  const uint4* xr = reinterpret_cast<const uint4*>(x + e / K * ldx);
  const uint4* wr = reinterpret_cast<const uint4*>(w + (long)v * ldw);
  float sum = 0.f;
  for (int c = lane; c < C / 8; c += 32) {
    float a[8], b[8];
    rt::unpack8(__ldg(xr + c), a);
    rt::unpack8(__ldg(wr + c), b);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(a[j], b[j], sum);
  }
  sum = rt::warp_sum(sum);
  if (lane == 0) hit[e] = sum * scale2;
}

// ---------------------------------------------------------------- statistics of one vocabulary piece
// Block per row over z [rows, width] (columns [first, first + width) of the vocabulary): part[row] = (max, sum of
// exp2 relative to it) of the row's logits outside the record, in units of log2.
__global__ void __launch_bounds__(256) piece_stats_kernel(const float* __restrict__ z, int width, int first, int K,
                                                          const int* __restrict__ sidx, float scale2,
                                                          float2* __restrict__ part) {
  extern __shared__ unsigned mask[];  // one bit per column: held
  __shared__ float2 warps[8];
  const long row = blockIdx.x;
  const float* zr = z + row * (long)width;
  for (int i = threadIdx.x; i < (width + 31) / 32; i += blockDim.x) mask[i] = 0;
  __syncthreads();
  for (int k = threadIdx.x; k < K; k += blockDim.x) {
    const int c = sidx[row * K + k] - first;
    if (c >= 0 && c < width) atomicOr(&mask[c >> 5], 1u << (c & 31));
  }
  __syncthreads();
  float m = -INFINITY, s = 0.f;
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    if (mask[c >> 5] >> (c & 31) & 1) continue;
    const float v = zr[c] * scale2;
    if (v > m) {
      s *= exp2f(m - v);
      m = v;
    }
    s += v == -INFINITY ? 0.f : exp2f(v - m);
  }
  auto merge = [](float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    const float fa = a.x == -INFINITY ? 1.f : exp2f(a.x - m), fb = b.x == -INFINITY ? 1.f : exp2f(b.x - m);
    return make_float2(m, a.y * fa + b.y * fb);
  };
  float2 o = make_float2(m, s);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    o = merge(o, make_float2(__shfl_xor_sync(~0u, o.x, off), __shfl_xor_sync(~0u, o.y, off)));
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = o;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < (int)blockDim.x / 32; ++w) o = merge(o, warps[w]);
    part[row] = o;
  }
}

// ---------------------------------------------------------------- rows
// Warp per row: merges the pieces' statistics in a fixed order, forms the loss and the row's gradient coefficients:
// d/dz_v = tail[row] exp2(z_v - lse[row]) outside the record, coef[k] for its held entries, both times scale and the
// row's upstream gradient (given per row, or 1, or 1 / rows with a loss).
__global__ void rows_kernel(const float2* __restrict__ part, int pieces, long rows, int K, int tail_class,
                            const int* __restrict__ kind, const int* __restrict__ sidx,
                            const float* __restrict__ slogp, const float* __restrict__ hit, float scale,
                            const float* __restrict__ grad, int mean, const int* __restrict__ count,
                            float* __restrict__ loss, float* __restrict__ lse2, float* __restrict__ tail,
                            float* __restrict__ coef) {
  const long row = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  if (kind[row] != 1) {
    if (lane == 0) {
      loss[row] = kind[row] ? NAN : 0.f;
      lse2[row] = 0.f;
      tail[row] = 0.f;
    }
    for (int k = lane; k < K; k += 32) coef[row * K + k] = 0.f;
    return;
  }
  float m = -INFINITY, top = -INFINITY;
  for (int i = lane; i < pieces; i += 32) m = fmaxf(m, part[i * rows + row].x);
  for (int k = lane; k < K; k += 32)
    if (sidx[row * K + k] != INT_MAX) top = fmaxf(top, hit[row * K + k]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(~0u, m, off));
    top = fmaxf(top, __shfl_xor_sync(~0u, top, off));
  }
  const float peak = fmaxf(m, top);
  float rest = 0.f, heldz = 0.f;
  for (int i = lane; i < pieces; i += 32) {
    const float2 p = part[i * rows + row];
    rest += p.x == -INFINITY ? p.y : p.y * exp2f(p.x - m);
  }
  double P = 0., L = 0.;
  for (int k = lane; k < K; k += 32) {
    if (sidx[row * K + k] == INT_MAX) continue;
    const float z2 = hit[row * K + k], lp = slogp[row * K + k];
    heldz += exp2f(z2 - peak);
    const double p = exp((double)lp);
    P += p;
    if (!(p <= 0.)) L += p * ((double)lp - (double)z2 * 0.6931471805599453);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    rest += __shfl_xor_sync(~0u, rest, off);
    heldz += __shfl_xor_sync(~0u, heldz, off);
    P += __shfl_xor_sync(~0u, P, off);
    L += __shfl_xor_sync(~0u, L, off);
  }
  // rest is relative to m, heldz to peak
  const float Z = heldz + (m == -INFINITY ? rest : rest * exp2f(m - peak));
  const double l2 = (double)peak + log2((double)Z);
  const double lse = l2 * 0.6931471805599453;
  const double r = tail_class && P < 1. ? 1. - P : 0.;
  const bool has_rest = !(rest <= 0.f);  // an empty rest of the vocabulary has no class
  double w = P, a = P;
  double value = L + P * lse;
  if (tail_class) {
    w = P + r;
    a = w;
    if (r > 0. && has_rest) {
      const double lr = ((double)m + log2((double)rest)) * 0.6931471805599453 - lse;  // log of the student's rest
      value += r * (log(r) - lr);
      a = w - r * exp(-lr);
    }
  }
  const float g = scale * (grad ? grad[row] : (mean ? 1.f / (float)max(count[0], 1) : 1.f));
  if (lane == 0) {
    loss[row] = (float)value;
    lse2[row] = (float)l2;
    tail[row] = g * (float)a;
  }
  for (int k = lane; k < K; k += 32) {
    float c = 0.f;
    if (sidx[row * K + k] != INT_MAX) {
      // for one held entry with p = 1 (cross entropy) q - 1 = -Z_rest / Z without cancellation
      const double p = exp((double)slogp[row * K + k]);
      const double q = exp2((double)hit[row * K + k] - l2);
      c = K == 1 && p == 1. ? -g * (m == -INFINITY ? rest : rest * exp2f((float)((double)m - l2))) : g * (float)(w * q - p);
    }
    coef[row * K + k] = c;
  }
}

// out[0] = sum (or mean over rows with a loss) of loss, in a fixed order.
__global__ void total_kernel(const float* __restrict__ loss, long rows, int mean, const int* __restrict__ count,
                             float* __restrict__ out) {
  __shared__ double part[32];
  double s = 0.;
  for (long t = threadIdx.x; t < rows; t += blockDim.x) s += (double)loss[t];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(~0u, s, off);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < (int)blockDim.x / 32; ++w) s += part[w];
    out[0] = (float)(mean ? s / (double)max(count[0], 1) : s);
  }
}

// ---------------------------------------------------------------- gradient of one vocabulary piece
// dz [rows, ld] bf16 from z [rows, width] fp32; rows without a gradient are zero whatever their logits hold.
__global__ void __launch_bounds__(256) piece_grad_kernel(const float* __restrict__ z, int width, int first, int ld,
                                                         int K, const int* __restrict__ sidx, float scale2,
                                                         const float* __restrict__ lse2,
                                                         const float* __restrict__ tail,
                                                         const float* __restrict__ coef, const int* __restrict__ kind,
                                                         __nv_bfloat16* __restrict__ dz) {
  const long row = blockIdx.x;
  const float* zr = z + row * (long)width;
  __nv_bfloat16* out = dz + row * (long)ld;
  const float l = lse2[row], a = tail[row];
  const bool live = kind[row] == 1;
  for (int c = threadIdx.x; c < ld; c += blockDim.x)
    out[c] = __float2bfloat16_rn(live && c < width ? a * exp2f(zr[c] * scale2 - l) : 0.f);
  __syncthreads();
  for (int k = threadIdx.x; k < K; k += blockDim.x) {
    const int c = sidx[row * K + k] - first;
    if (c >= 0 && c < width && live) out[c] = __float2bfloat16_rn(coef[row * K + k]);
  }
}

// out = x with the rows that have no gradient zero (they may hold anything: 0 times NaN would reach every weight row).
__global__ void live_rows_kernel(const __nv_bfloat16* __restrict__ x, long ld, int C, const int* __restrict__ kind,
                                 __nv_bfloat16* __restrict__ out) {
  const long row = blockIdx.x;
  const bool live = kind[row] == 1;
  for (int c = threadIdx.x; c < C; c += blockDim.x)
    out[row * (long)C + c] = live ? x[row * ld + c] : __float2bfloat16_rn(0.f);
}

// x *= *factor, nothing at all for a factor of one (the usual upstream gradient of a training loss).
__global__ void scale_kernel(__nv_bfloat16* __restrict__ x, const float* __restrict__ factor, long n) {
  const float f = *factor;
  if (f == 1.f) return;
  const long step = (long)gridDim.x * blockDim.x, n8 = n / 8;
  uint4* x8 = reinterpret_cast<uint4*>(x);
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += step) {
    float v[8];
    rt::unpack8(x8[i], v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= f;
    x8[i] = rt::pack8(v);
  }
  for (long i = 8 * n8 + (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step)
    x[i] = __float2bfloat16_rn(__bfloat162float(x[i]) * f);
}

// The tensor cores round each of the C / 16 partial sums of a logit towards zero. Given the sum z, the partial sums are
// (k / n) z on average, each loses half a unit in its last place, and the expected loss is n 2^-26 z (measured: 4.84e-6
// z at width 5120, 1.82e-6 at 2048, 0.86e-6 at 1024, on random operands; the rest of the error has no preferred side).
// Undoing it takes the error of log Z from 9.6e-6 to 2e-7 at width 5120.
float mma_gain(int C) { return 1.f + (float)(C / 16) * 0x1p-26f; }

long up(long n, long to) { return (n + to - 1) / to * to; }

// Columns of a vocabulary piece: a multiple of 64 whose fp32 logits take about 64 MB, at most 8192.
int piece_columns(long rows, long V) {
  const long fit = (16L << 20) / std::max(rows, 1L) / 64 * 64;
  return (int)std::min(up(V, 64), std::max(256L, std::min(8192L, fit)));
}

struct Layout {  // offsets in floats, each 16-byte aligned
  long sidx, slogp, hit, coef, kind, count, lse2, tail, part, z, dz, dx, x, total;
};
Layout layout(long rows, long V, int C, int K, bool grad_h, bool grad_w) {
  Layout l;
  long at = 0;
  auto take = [&](long n) {
    const long o = at;
    at += up(n, 4);
    return o;
  };
  const int cols = piece_columns(rows, V);
  const long pieces = (V + cols - 1) / cols;
  l.sidx = take(rows * K);
  l.slogp = take(rows * K);
  l.hit = take(rows * K);
  l.coef = take(rows * K);
  l.kind = take(rows);
  l.count = take(4);
  l.lse2 = take(rows);
  l.tail = take(rows);
  l.part = take(2 * rows * pieces);
  l.z = take(rows * cols);
  l.dz = take(grad_h || grad_w ? rows * cols / 2 + 4 : 0);
  l.dx = take(grad_h ? rows * C : 0);
  l.x = take(grad_w ? rows * C / 2 + 4 : 0);
  l.total = at;
  return l;
}

}  // namespace

extern "C" long rt_head_loss_workspace_floats(long rows, long V, int C, int K, int grad_h, int grad_w) {
  return layout(rows, V, C, K, grad_h != 0, grad_w != 0).total;
}

extern "C" cudaError_t rt_head_loss(const RtHeadLoss* p, float* work, cudaStream_t s) {
  if (!p || !work) return cudaErrorInvalidValue;
  const long T = p->rows, V = p->vocab;
  const int C = p->width, K = p->K;
  if (T < 0 || V < 1 || V > INT_MAX - 1 || T > (1 << 24) || C < 1 || C % 8 || K < 1 || K > RT_HEAD_MAX_RECORD ||
      (reinterpret_cast<uintptr_t>(work) & 15))
    return cudaErrorInvalidValue;
  if (T == 0) {
    if (p->reduction) RT_CUDA_CHECK(cudaMemsetAsync(p->loss, 0, sizeof(float), s));
    if (p->dweight) RT_CUDA_CHECK(cudaMemsetAsync(p->dweight, 0, (size_t)V * C * 2, s));
    return cudaSuccess;
  }
  const Layout l = layout(T, V, C, K, p->dhidden != nullptr, p->dweight != nullptr);
  int* sidx = reinterpret_cast<int*>(work + l.sidx);
  float* slogp = work + l.slogp;
  float* hit = work + l.hit;
  float* coef = work + l.coef;
  int* kind = reinterpret_cast<int*>(work + l.kind);
  int* count = reinterpret_cast<int*>(work + l.count);
  float2* part = reinterpret_cast<float2*>(work + l.part);
  float* z = work + l.z;
  __nv_bfloat16* dz = reinterpret_cast<__nv_bfloat16*>(work + l.dz);
  const float scale2 = p->scale * LOG2E;
  const float scale2_mma = scale2 * mma_gain(C);
  int Kp = 1;
  while (Kp < K) Kp <<= 1;
  const int threads = std::min(256, std::max(32, Kp / 2));
  records_kernel<<<(unsigned)T, threads, Kp * 8, s>>>(p->index, p->log_probs, K, Kp, V, p->ignore, sidx, slogp, kind);
  count_kernel<<<1, 1024, 0, s>>>(kind, T, count);
  const int cols = piece_columns(T, V);
  const int pieces = (int)((V + cols - 1) / cols);
  const __nv_bfloat16* W = reinterpret_cast<const __nv_bfloat16*>(p->weight);
  held_logits_kernel<<<(unsigned)((T * K * 32 + 255) / 256), 256, 0, s>>>(
      reinterpret_cast<const __nv_bfloat16*>(p->hidden), p->ld_hidden, W, p->ld_weight, C, T * K, K, sidx, scale2, hit);
  for (int i = 0; i < pieces; ++i) {
    const int first = i * cols, width = (int)std::min<long>(cols, V - first);
    RT_CUDA_CHECK(rt_gemm_bf16(p->hidden, p->ld_hidden, 0, W + (long)first * p->ld_weight, p->ld_weight, 0, z, width,
                               (int)T, width, C, 1, 1.f, nullptr, s));
    piece_stats_kernel<<<(unsigned)T, 256, (width + 31) / 32 * 4, s>>>(z, width, first, K, sidx, scale2_mma,
                                                                       part + (long)i * T);
  }
  rows_kernel<<<(unsigned)((T * 32 + 127) / 128), 128, 0, s>>>(part, pieces, T, K, p->tail, kind, sidx, slogp, hit,
                                                               p->scale, p->row_grad, p->reduction == 2, count,
                                                               p->row_loss, work + l.lse2, work + l.tail, coef);
  if (p->reduction) total_kernel<<<1, 1024, 0, s>>>(p->row_loss, T, p->reduction == 2, count, p->loss);
  RT_CUDA_CHECK(cudaGetLastError());
  if (!p->dhidden && !p->dweight) return cudaSuccess;
  float* dx = work + l.dx;
  if (p->dhidden) RT_CUDA_CHECK(rt_zero_f32(dx, T * C, s));
  __nv_bfloat16* x = reinterpret_cast<__nv_bfloat16*>(work + l.x);
  if (p->dweight)
    live_rows_kernel<<<(unsigned)T, 256, 0, s>>>(reinterpret_cast<const __nv_bfloat16*>(p->hidden), p->ld_hidden, C,
                                                 kind, x);
  for (int i = 0; i < pieces; ++i) {
    const int first = i * cols, width = (int)std::min<long>(cols, V - first);
    const int ld = (int)up(width, 8);
    RT_CUDA_CHECK(rt_gemm_bf16(p->hidden, p->ld_hidden, 0, W + (long)first * p->ld_weight, p->ld_weight, 0, z, width,
                               (int)T, width, C, 1, 1.f, nullptr, s));
    piece_grad_kernel<<<(unsigned)T, 256, 0, s>>>(z, width, first, ld, K, sidx, scale2_mma, work + l.lse2, work + l.tail,
                                                  coef, kind, dz);
    if (p->dhidden)
      RT_CUDA_CHECK(rt_gemm_bf16(dz, ld, 0, W + (long)first * p->ld_weight, p->ld_weight, 1, dx, C, (int)T, C, width,
                                 2, 1.f, nullptr, s));
    if (p->dweight)
      RT_CUDA_CHECK(rt_gemm_bf16(dz, ld, 1, x, C, 1,
                                 reinterpret_cast<__nv_bfloat16*>(p->dweight) + (long)first * C, C, width, C, (int)T,
                                 0, 1.f, nullptr, s));
  }
  if (p->dhidden) RT_CUDA_CHECK(rt_to_bf16(dx, p->dhidden, T * C, s));
  return cudaGetLastError();
}

// x [n] bf16 *= *factor (device scalar).
extern "C" cudaError_t rt_scale_bf16(void* x, const float* factor, long n, cudaStream_t s) {
  if (n <= 0) return cudaSuccess;
  if (reinterpret_cast<uintptr_t>(x) & 15) return cudaErrorInvalidValue;
  const long blocks = std::min((n / 8 + 255) / 256 + 1, 148L * 8);
  scale_kernel<<<(unsigned)blocks, 256, 0, s>>>(reinterpret_cast<__nv_bfloat16*>(x), factor, n);
  return cudaGetLastError();
}
