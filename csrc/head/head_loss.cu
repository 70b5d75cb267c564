// Losses of the vocabulary head from hidden states: next-token cross entropy and the KL from a teacher's recorded top
// log-probabilities, with the gradients of the hidden states and of the head's weight.
//
// With z_tv = scale x_t . W_v, a row's record is a set S of held entries (v, log p_v); the cross entropy's record is
// its target with p = 1. With P = sum_S p, r = max(0, 1 - P) (the rest as one more class; 0 without that class, or
// where S is the whole vocabulary), w = P + r, Z = sum_v exp z_v and Z_rest = sum_{v not in S} exp z_v:
//   loss  = sum_S p (log p - z_v + log Z) + r (log r - log Z_rest + log Z)
//   d/dz_v = w exp(z_v) / Z - p_v                       (v in S)
//          = exp(z_v) / Z_rest (w Z_rest / Z - r)       (v not in S, r > 0)
//          = exp(z_v) / Z w                             (v not in S, r = 0)
// Z_rest is summed without the held entries instead of as Z minus them, so a row that is sure of its target keeps the
// relative precision of 1 - q. The second form has factors of at most one however small Z_rest / Z is; as exp(z_v) / Z
// (w - r Z / Z_rest) its factors leave fp32's range at Z_rest / Z = e^-87.
// Sums within a tile and over a row's tiles are fp32. What joins a row's rest and its held entries (Z, log Z, the loss
// and the gradient's coefficients) and the sum of the rows' losses are fp64: a KL is a small difference of these.
//
// Launches of one call: the rows that have a loss are counted and packed (gather_kernel: their hidden states, sorted
// records and held logits), z = X W^T leaves per row and 256-column tile its maximum and sum of exponentials
// (head_gemm.cuh), merge_kernel forms the losses. With gradients the same product also leaves each logit's depth below
// its tile's maximum in 16 bits; gradient_kernel turns them into dz (bf16) in place, and dX = dz W, dW = dz^T X follow.
// That is 6 T V C operations, against 8 T V C where the logits are formed a second time, for T V 16-bit values of
// workspace; CHUNK_VALUES bounds it, and more rows run in chunks whose dW adds up in fp32. Rows without a loss cost
// nothing but their packing, and what they hold never meets the other rows. The cross entropy of a few rows without
// gradients is not packed and takes two launches. A product that gave up a bounded wait leaves NaN in all that is
// formed after it: the losses, dX, and the first 16 bytes of dW.
#include <algorithm>
#include <atomic>
#include <climits>
#include "../api.h"
#include "../common/common.cuh"
#include "head_gemm.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453;

// ---------------------------------------------------------------- rows with a loss
// Kind of each row: 0 no entry (no loss), 1 valid, 2 an index outside the vocabulary (loss NaN, gradient zero).
__device__ __forceinline__ int entry_kind(long id, bool record, long ignore, long V) {
  if (record ? id < 0 : id == ignore) return 0;
  return id < 0 || id >= V ? 2 : 1;
}
// From its entries' kinds or'd.
__device__ __forceinline__ int row_kind(int entries) { return entries & 2 ? 2 : entries; }

// One warp per row: kind[row] of a record of K entries.
__global__ void kinds_kernel(const long* __restrict__ idx, long rows, int K, long V, int* __restrict__ kind) {
  const long row = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (row >= rows) return;
  int any = 0;
  for (int k = threadIdx.x & 31; k < K; k += 32) any |= entry_kind(idx[row * K + k], true, 0, V);
  any = __reduce_or_sync(~0u, any);
  if ((threadIdx.x & 31) == 0) kind[row] = row_kind(any);
}

// What the rows' losses and gradients are taken over: valid rows, rows with a loss, a product that gave up a wait
// (where the caller has no status word), and blocks of merge_kernel that are done.
// `factor` is what all rows' gradients have in common (scale, the mean's 1 / rows with a loss, the largest upstream
// gradient of a row): dX and dW are multiplied by it in fp32. In dz it would round the target entries of all rows,
// which are nearly -factor, the same way: up to 0.4% of the whole gradient. `unit`: the upstream gradient that counts
// as one.
struct Counts {
  int valid, counted, failed, done;
  float factor, unit;
};

struct Upstream {
  float scale;
  int mean;
  const float* rows;  // or null
  __device__ __forceinline__ float of(long row) const { return rows ? fabsf(rows[row]) : 0.f; }
  // top: the largest of the valid rows
  __device__ __forceinline__ Counts counts(int valid, int counted, float top) const {
    const float unit = top > 0.f && top < INFINITY ? top : 1.f;
    return Counts{valid, counted, 0, 0, rows ? scale * unit : mean ? scale / (float)max(counted, 1) : scale, unit};
  }
};

// One block: slot[row] = place of a valid row among the valid ones, or -1 (no loss), -2 (outside the vocabulary). The
// kinds come from `kind`, or from targets.
__global__ void __launch_bounds__(1024) pack_kernel(const int* __restrict__ kind, const long* __restrict__ targets,
                                                    long ignore, long V, long rows, const Upstream up,
                                                    int* __restrict__ slot, Counts* __restrict__ counts) {
  __shared__ int warps[2][32], top_bits;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int valid = 0, bad = 0;
  float top = 0.f;
  if (threadIdx.x == 0) top_bits = 0;
  for (long base = 0; base < rows; base += 1024) {
    const long t = base + threadIdx.x;
    const int k = t >= rows ? 0 : kind ? kind[t] : entry_kind(targets[t], false, ignore, V);
    if (k == 1) top = fmaxf(top, up.of(t));
    const unsigned good = __ballot_sync(~0u, k == 1), outside = __ballot_sync(~0u, k == 2);
    if (lane == 0) {
      warps[0][warp] = __popc(good);
      warps[1][warp] = __popc(outside);
    }
    __syncthreads();
    int at = valid + __popc(good & ((1u << lane) - 1));
    const int g = warps[0][lane], b = warps[1][lane];
    at += __reduce_add_sync(~0u, lane < warp ? g : 0);
    valid += __reduce_add_sync(~0u, g);
    bad += __reduce_add_sync(~0u, b);
    if (t < rows) slot[t] = k == 1 ? at : -k - (k == 0);
    __syncthreads();
  }
  if (up.rows) atomicMax(&top_bits, __float_as_int(top));  // not negative: ordered like the numbers
  __syncthreads();
  if (threadIdx.x == 0) *counts = up.counts(valid, valid + bad, __int_as_float(top_bits));
}

// The same for the block of one row of a short call (at most SHORT_ENTRIES in all its records), which counts the rows
// before its own itself: the place or -1 / -2, and the number of valid rows. Saves one or two launches.
// (16 targets: 3.4 us against 1.9 + 3.0 in two launches; 1024 targets: 27 against 2.2 + 18.5.)
constexpr int SHORT_ENTRIES = 512;
__device__ __forceinline__ int place_in_short(const long* idx, bool record, int K, long rows, long row, long ignore,
                                              long V, const Upstream& up, Counts* counts, int* scratch, int& valid) {
  int before = 0, all = 0, bad = 0;
  float top = 0.f;
  for (long t = threadIdx.x; t < rows; t += blockDim.x) {
    int any = 0;
    for (int k = 0; k < K; ++k) any |= entry_kind(idx[t * K + k], record, ignore, V);
    const int kind = row_kind(any);
    before += t < row && kind == 1;
    all += kind == 1;
    bad += kind == 2;
    if (t == row) scratch[3] = kind;
    if (row == 0 && kind == 1) top = fmaxf(top, up.of(t));
  }
  if (threadIdx.x < 3) scratch[threadIdx.x] = 0;
  if (threadIdx.x == 3) scratch[4] = 0;
  __syncthreads();
  before = __reduce_add_sync(~0u, before);
  all = __reduce_add_sync(~0u, all);
  bad = __reduce_add_sync(~0u, bad);
  if ((threadIdx.x & 31) == 0) {
    atomicAdd(&scratch[0], before);
    atomicAdd(&scratch[1], all);
    atomicAdd(&scratch[2], bad);
  }
  if (row == 0 && up.rows) atomicMax(&scratch[4], __float_as_int(top));
  __syncthreads();
  valid = scratch[1];
  if (row == 0 && threadIdx.x == 0) *counts = up.counts(valid, valid + scratch[2], __int_as_float(scratch[4]));
  if (row >= rows) return 0;
  const int kind = scratch[3];
  return kind == 1 ? scratch[0] : -kind - (kind == 0);
}

// One warp: x . w over 8 c8 values by fp32 fused multiply-adds.
__device__ __forceinline__ float row_dot(const uint4* x, const uint4* w, int c8, int lane) {
  float sum = 0.f;
#pragma unroll 4
  for (int c = lane; c < c8; c += 32) {
    float a[8], b[8];
    rt::unpack8(__ldg(x + c), a);
    rt::unpack8(__ldg(w + c), b);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(a[j], b[j], sum);
  }
  return rt::warp_sum(sum);
}

// One block per row, and 64 more for the zero rows that fill the packed rows' last block of 64. A valid row's hidden
// state goes to its place in `x`; its entries are sorted by vocabulary index (INT_MAX behind the last) with their
// log-probabilities, and their logits in units of log2 are summed here: they enter the loss with a weight of about one,
// where all others enter it through the sum of exponentials, so they come from fp32 fused multiply-adds, which round,
// instead of from the tensor cores, which truncate (see mma_gain). Rows without a gradient get their zeros here. Where
// there are few rows, the entries of a row are shared out over the blocks of its y index.
__global__ void __launch_bounds__(256) gather_kernel(const long* __restrict__ idx, const float* __restrict__ logp,
                                                     int K, int Kp, long rows, const __nv_bfloat16* __restrict__ hidden,
                                                     long ldh, const __nv_bfloat16* __restrict__ w, long ldw, int C,
                                                     float scale2, long V, long ignore, bool brief,
                                                     const Upstream up, const int* __restrict__ slot,
                                                     Counts* __restrict__ counts, int* __restrict__ row_of,
                                                     uint4* __restrict__ x,
                                                     int* __restrict__ sidx, float* __restrict__ slogp,
                                                     float* __restrict__ hit, float* __restrict__ row_loss,
                                                     uint4* __restrict__ dhidden) {
  extern __shared__ unsigned long long keys[];
  const long row = blockIdx.x;
  const int C8 = C / 8;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  __shared__ int scratch[5];
  int valid;
  long place;
  if (brief) {
    place = place_in_short(idx, logp != nullptr, K, rows, row, ignore, V, up, counts, scratch, valid);
  } else {
    valid = counts->valid;
    place = row < rows ? slot[row] : 0;
  }
  const bool lead = blockIdx.y == 0;
  if (row >= rows) {
    if (!lead) return;
    const long n = valid, fill = n + (row - rows);
    if (fill < max((n + 63) / 64 * 64, 64L))
      for (int c = threadIdx.x; c < C8; c += blockDim.x) x[fill * C8 + c] = zero;
    return;
  }
  if (place < 0) {
    if (!lead) return;
    if (threadIdx.x == 0) row_loss[row] = place == -1 ? 0.f : NAN;
    if (dhidden)
      for (int c = threadIdx.x; c < C8; c += blockDim.x) dhidden[row * C8 + c] = zero;
    return;
  }
  if (lead && threadIdx.x == 0) row_of[place] = (int)row;
  const uint4* src = reinterpret_cast<const uint4*>(hidden + row * ldh);
  for (int c = threadIdx.x; lead && c < C8; c += blockDim.x) x[place * C8 + c] = __ldg(src + c);
  for (int k = threadIdx.x; k < Kp; k += blockDim.x) {
    int v = INT_MAX;
    float lp = 0.f;
    if (k < K && idx[row * K + k] >= 0) {
      v = (int)idx[row * K + k];
      lp = logp ? logp[row * K + k] : 0.f;
    }
    keys[k] = ((unsigned long long)v << 32) | __float_as_uint(lp);
  }
  __syncthreads();
  for (int size = 2; size <= Kp; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int i = threadIdx.x; i < Kp / 2; i += blockDim.x) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const unsigned long long a = keys[lo], b = keys[hi];
        if ((a > b) == ((lo & size) == 0)) {
          keys[lo] = b;
          keys[hi] = a;
        }
      }
      __syncthreads();
    }
  const int lane = threadIdx.x & 31;
  for (int k = (threadIdx.x >> 5) + 8 * blockIdx.y; k < K; k += 8 * gridDim.y) {
    const int v = (int)(keys[k] >> 32);
    const float sum = v == INT_MAX ? 0.f : row_dot(src, reinterpret_cast<const uint4*>(w + (long)v * ldw), C8, lane);
    if (lane == 0) {
      sidx[place * K + k] = v;
      slogp[place * K + k] = __uint_as_float((unsigned)keys[k]);
      hit[place * K + k] = sum * scale2;
    }
  }
}

// ---------------------------------------------------------------- losses of the valid rows of a chunk
// Block of ROWS rows (four, or one of the few rows whose statistics are finer): its threads merge the tiles' statistics
// (in a fixed order: each row's tiles go round-robin to MERGE_THREADS / ROWS threads), then one warp per row forms the
// loss and the gradient's coefficients: d/dz_v = tail exp2(z_v - base2) outside the record (base2 = log2 Z_rest with a
// rest's class, else log2 Z), coef[k] for its held entries, both times the row's upstream gradient in units of the
// call's (see Counts).
constexpr int MERGE_THREADS = 256;
struct MergeArgs {
  const float2* part;
  long part_ld;
  int tiles, row0, rows, K, tail_class, mean;
  int blocks;  // of all chunks
  long all_rows;
  Counts* counts;
  const int* failed;  // a product gave up a wait
  const int* row_of;
  const int* sidx;
  const float* slogp;
  const float* hit;
  const float* grad;  // upstream gradients of the rows, or null
  float* row_loss;
  float* loss;  // null: the rows' losses are the result
  float* base2;
  float* tail;
  float* coef;
};

// (max, sum of exponentials relative to it) of two sets.
__device__ __forceinline__ float2 merge2(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  return make_float2(m, (a.x == m ? a.y : a.y * exp2f(a.x - m)) + (b.x == m ? b.y : b.y * exp2f(b.x - m)));
}

template <int ROWS>
__device__ __forceinline__ void merge_rows(const MergeArgs& p) {
  constexpr int GROUPS = MERGE_THREADS / ROWS;
  __shared__ float2 merged[GROUPS][ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = min(max(p.counts->valid - p.row0, 0), p.rows);
  const int first = blockIdx.x * ROWS;
  if (first < n) {
    const int j = threadIdx.x % ROWS, group = threadIdx.x / ROWS;
    const float2* part = p.part + min(first + j, n - 1);
    float2 sum = make_float2(-INFINITY, 0.f);
    for (int i = group; i < p.tiles; i += 4 * GROUPS) {
      float2 t[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        t[u] = i + u * GROUPS < p.tiles ? part[(i + u * GROUPS) * p.part_ld] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int u = 0; u < 4; ++u) sum = merge2(sum, t[u]);
    }
    merged[group][j] = sum;
  }
  __syncthreads();
  const int j = warp;
  if (j < ROWS && first + j < n) {
    const int r = first + j;
    const long place = p.row0 + r, row = p.row_of[place];
    const int* sidx = p.sidx + place * p.K;
    const float* slogp = p.slogp + place * p.K;
    const float* hit = p.hit + place * p.K;
    float2 all = merged[lane][j];
#pragma unroll
    for (int i = 32; i < GROUPS; i += 32) all = merge2(all, merged[lane + i][j]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
      all = merge2(all, make_float2(__shfl_xor_sync(~0u, all.x, off), __shfl_xor_sync(~0u, all.y, off)));
    const float m = all.x, rest = all.y;
    float top = -INFINITY;
    for (int k = lane; k < p.K; k += 32)
      if (sidx[k] != INT_MAX) top = fmaxf(top, hit[k]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, off));
    const float peak = fmaxf(m, top);
    double heldz = 0., P = 0., L = 0.;
    for (int k = lane; k < p.K; k += 32) {
      if (sidx[k] == INT_MAX) continue;
      const float z2 = hit[k], lp = slogp[k];
      heldz += exp2((double)z2 - (double)peak);
      const double q = exp((double)lp);
      P += q;
      if (!(q <= 0.)) L += q * ((double)lp - (double)z2 * LN2);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      heldz += __shfl_xor_sync(~0u, heldz, off);
      P += __shfl_xor_sync(~0u, P, off);
      L += __shfl_xor_sync(~0u, L, off);
    }
    // rest is relative to m, heldz to peak. In fp64: a KL is a small difference of these, and fp32's exp2f alone put
    // -4e-8 on a mean of 0.018.
    const double Z = heldz + (m == -INFINITY ? rest : rest * exp2((double)m - (double)peak));
    const double l2 = (double)peak + log2(Z);
    const double lse = l2 * LN2;
    const double r1 = p.tail_class && P < 1. && !(rest <= 0.f) ? 1. - P : 0.;  // an empty rest has no class
    const double weight = P + r1;
    double a = Z == Z ? weight : NAN, value = L + P * lse, base = l2;  // NaN logits: also where a tile has no maximum
    if (r1 > 0.) {
      base = (double)m + log2((double)rest);
      const double lr = base * LN2 - lse;  // log of the student's rest
      value += r1 * (log(r1) - lr);
      a = weight * exp(lr) - r1;
    }
    const float g = p.grad ? p.grad[row] / p.counts->unit : 1.f;
    if (lane == 0) {
      p.row_loss[row] = *p.failed ? NAN : (float)value;
      p.base2[place] = (float)base;
      p.tail[place] = g * (float)a;
    }
    if (!p.coef) return;
    for (int k = lane; k < p.K; k += 32) {
      float c = 0.f;
      if (sidx[k] != INT_MAX) {
        // for one held entry with p = 1 (cross entropy) q - 1 = -Z_rest / Z without cancellation
        const double q = exp((double)slogp[k]);
        c = p.K == 1 && q == 1. ? -g * (m == -INFINITY ? rest : rest * exp2f((float)((double)m - l2)))
                                : g * (float)(weight * exp2((double)hit[k] - l2) - q);
      }
      p.coef[place * p.K + k] = c;
    }
  }
}

// The last block to finish also adds up the rows' losses, in a fixed order (mean: over rows with a loss).
template <int ROWS>
__global__ void __launch_bounds__(MERGE_THREADS) merge_kernel(const MergeArgs p) {
  __shared__ double part[MERGE_THREADS / 32];
  __shared__ bool last;
  merge_rows<ROWS>(p);
  if (!p.loss) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&p.counts->done, 1) == p.blocks - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.;
  for (long t = threadIdx.x; t < p.all_rows; t += blockDim.x) s += (double)__ldcg(p.row_loss + t);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(~0u, s, off);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < (int)blockDim.x / 32; ++w) s += part[w];
    *p.loss = (float)(p.mean ? s / (double)max(p.counts->counted, 1) : s);
  }
}

// Cross entropy of a few rows without gradients, whose rows were not gathered: block per row, whose last warp sums its
// target's logit beside the merge. Same operations in the same order as merge_kernel<1>, and so the same bits. The last
// block adds up the rows' losses as in merge_kernel.
struct ScoreArgs {
  const float2* part;
  long part_ld;
  int tiles, mean;
  const long* targets;
  long ignore, V;
  const __nv_bfloat16* hidden;
  long ldh;
  const __nv_bfloat16* w;
  long ldw;
  int C;
  float scale2;
  Counts* counts;
  const int* failed;
  float* row_loss;
  float* loss;
};
__global__ void __launch_bounds__(MERGE_THREADS + 32) score_kernel(const ScoreArgs p) {
  __shared__ float2 merged[MERGE_THREADS];
  __shared__ float target_z2;
  __shared__ bool last;
  const int tid = threadIdx.x, lane = tid & 31, row = blockIdx.x, rows = gridDim.x;
  const long target = p.targets[row];
  const int kind = entry_kind(target, false, p.ignore, p.V);
  if (kind == 1 && tid >= MERGE_THREADS) {
    const float dot = row_dot(reinterpret_cast<const uint4*>(p.hidden + row * p.ldh),
                              reinterpret_cast<const uint4*>(p.w + target * p.ldw), p.C / 8, lane);
    if (lane == 0) target_z2 = dot * p.scale2;
  } else if (kind == 1) {
    float2 sum = make_float2(-INFINITY, 0.f);
    for (int i = tid; i < p.tiles; i += 8 * MERGE_THREADS) {
      float2 t[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        t[u] = i + u * MERGE_THREADS < p.tiles ? p.part[(i + u * MERGE_THREADS) * p.part_ld + row]
                                               : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int u = 0; u < 8; ++u) sum = merge2(sum, t[u]);
    }
    merged[tid] = sum;
  }
  __syncthreads();
  if (tid < 32) {
    float value = kind ? NAN : 0.f;
    if (kind == 1) {
      float2 all = merged[lane];
#pragma unroll
      for (int i = 32; i < MERGE_THREADS; i += 32) all = merge2(all, merged[lane + i]);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1)
        all = merge2(all, make_float2(__shfl_xor_sync(~0u, all.x, off), __shfl_xor_sync(~0u, all.y, off)));
      const float z2 = target_z2, peak = fmaxf(all.x, z2);
      const double Z = exp2((double)z2 - (double)peak) +
                       (all.x == -INFINITY ? all.y : all.y * exp2((double)all.x - (double)peak));
      if (!*p.failed) value = (float)(((double)peak + log2(Z)) * LN2 - (double)z2 * LN2);
    }
    if (lane == 0) p.row_loss[row] = value;
  }
  if (!p.loss) return;
  __threadfence();
  __syncthreads();
  if (tid == 0) last = atomicAdd(&p.counts->done, 1) == rows - 1;
  __syncthreads();
  if (!last || tid >= 32) return;
  __threadfence();
  double s = 0.;
  int counted = 0;
  for (int t = lane; t < rows; t += 32) {
    s += (double)__ldcg(p.row_loss + t);
    counted += p.targets[t] != p.ignore;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(~0u, s, off);
  counted = __reduce_add_sync(~0u, counted);
  if (lane == 0) *p.loss = (float)(p.mean ? s / (double)max(counted, 1) : s);
}

// ---------------------------------------------------------------- gradient of the logits
// In place: depths of a chunk's logits (below the maximum of their `group` columns) -> dz, one warp per row and 256
// columns; the block of 32 such tiles also puts their held entries in their places; rows that fill the last block of 64
// become zero. A read and a write of every value: 0.16 ms for 992 x 248077 (6.0 TB/s), where forming the logits again
// would cost 1.8 ms. dz is rounded to bf16 here, once: it is a tensor-core operand next.
__global__ void __launch_bounds__(256) gradient_kernel(__nv_bfloat16* __restrict__ e, long ld, int V, int row0,
                                                       int rows, const Counts* __restrict__ counts,
                                                       const float2* __restrict__ part, long part_ld, int group,
                                                       const float* __restrict__ base2, const float* __restrict__ tail,
                                                       int K, const int* __restrict__ sidx,
                                                       const float* __restrict__ coef) {
  const int n = min(max(counts->valid - row0, 0), rows), r = blockIdx.y;
  if (r >= max((n + 63) / 64 * 64, 64)) return;
  const int lane = threadIdx.x & 31;
  const bool live = r < n;
  const float l = live ? base2[row0 + r] : 0.f, a = live ? tail[row0 + r] : 0.f;
  sidx += (long)(row0 + r) * K;
  coef += (long)(row0 + r) * K;
  __nv_bfloat16* out = e + r * ld;
  uint4 depths[4];
  float m[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {  // all loads first: nothing says that the stores leave them alone
    const int c = ((blockIdx.x * 4 + u) * 8 + (threadIdx.x >> 5)) * 256 + lane * 8;
    if (live && c < V) {
      depths[u] = *reinterpret_cast<const uint4*>(out + c);
      m[u] = part[c / group * part_ld + r].x;
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int c = ((blockIdx.x * 4 + u) * 8 + (threadIdx.x >> 5)) * 256 + lane * 8;
    if (c >= ld) continue;
    float v[8] = {};
    if (live && c < V) {
      const float top = m[u] == -INFINITY ? m[u] : m[u] - l;
      const uint32_t w[4] = {depths[u].x, depths[u].y, depths[u].z, depths[u].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // 2^23 + depth as a float, and back
        const uint32_t word = __byte_perm(w[j / 2], 0x4b000000u, j & 1 ? 0x7632 : 0x7610);
        const float d = __uint_as_float(word) - head::DEPTH_BASE;
        v[j] = a * head::ex2(fmaf(d, -1.f / head::DEPTH_STEPS, top));
      }
    }
    *reinterpret_cast<uint4*>(out + c) = rt::pack8(v);
  }
  if (!live) return;
  __syncthreads();
  const int first = blockIdx.x * 32 * 256;
  for (int k = threadIdx.x; k < K; k += blockDim.x) {
    const int s = sidx[k];
    if (s >= first && s - first < 32 * 256 && s < V) e[r * ld + s] = __float2bfloat16_rn(coef[k]);
  }
}

// dhidden[row_of[place]] = bf16 of factor times the row's partial sums, added in order.
__global__ void __launch_bounds__(256) dhidden_kernel(const float* __restrict__ partial, int splits, long split_rows,
                                                      int C, int row0, int rows, const Counts* __restrict__ counts,
                                                      const int* failed, const int* __restrict__ row_of,
                                                      __nv_bfloat16* __restrict__ out) {
  const int n = min(max(counts->valid - row0, 0), rows), r = blockIdx.x;
  if (r >= n) return;
  const float factor = *failed ? NAN : counts->factor;  // a product gave up a wait
  uint4* dst = reinterpret_cast<uint4*>(out + (long)row_of[row0 + r] * C);
  for (int c = threadIdx.x; c < C / 8; c += blockDim.x) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    for (int s = 0; s < splits; ++s) {
      const float4* src = reinterpret_cast<const float4*>(partial + ((long)s * split_rows + r) * C) + 2 * c;
      const float4 x = __ldg(src), y = __ldg(src + 1);
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
      v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= factor;
    dst[c] = rt::pack8(v);
  }
}

// The weight's gradient where a product gave up a wait (the one-chunk kernel leaves its NaN itself).
__global__ void failed_kernel(const int* failed, __nv_bfloat16* __restrict__ dweight) {
  if (*failed && threadIdx.x < 8) dweight[threadIdx.x] = __float2bfloat16_rn(NAN);
}

// x *= *factor for up to two tensors, nothing at all for a factor of one (the usual upstream gradient of a loss). A
// factor that is no power of two rounds the gradients to bf16 a second time: it is only known in backward, and fp32
// gradients kept until then would take twice the weight's memory (5 GB at the 27B head).
struct ScaleArgs {
  __nv_bfloat16* x[2];
  long n[2];
};
__global__ void scale_kernel(const ScaleArgs p, const float* __restrict__ factor) {
  const float f = *factor;
  if (f == 1.f) return;
  const long step = (long)gridDim.x * blockDim.x, at = (long)blockIdx.x * blockDim.x + threadIdx.x;
  for (int t = 0; t < 2; ++t) {
    const long n8 = p.n[t] / 8;
    uint4* x8 = reinterpret_cast<uint4*>(p.x[t]);
    for (long i = at; i < n8; i += step) {
      float v[8];
      rt::unpack8(x8[i], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= f;
      x8[i] = rt::pack8(v);
    }
    for (long i = 8 * n8 + at; i < p.n[t]; i += step)
      p.x[t][i] = __float2bfloat16_rn(__bfloat162float(p.x[t][i]) * f);
  }
}

// The tensor cores round each of the C / 16 partial sums of a logit towards zero. Given the sum z, the partial sums are
// (k / n) z on average, each loses half a unit in its last place, and the expected loss is n 2^-26 z (measured: 4.84e-6
// z at width 5120, 1.82e-6 at 2048, 0.86e-6 at 1024, on random operands; the rest of the error has no preferred side).
// Undoing it takes the error of log Z from 9.6e-6 to 2e-7 at width 5120. Where the products add up exactly (one-hot
// hidden states, small whole numbers) there is nothing to undo, and n 2^-26 of the logit is the error: 4.8e-6 at width
// 5120, as large as without the correction on other operands.
float mma_gain(int C) { return 1.f + (float)(C / 16) * 0x1p-26f; }

constexpr long up(long n, long to) { return (n + to - 1) / to * to; }

// Rows of a chunk: with gradients their logits' depths take up to 2 GiB, without their statistics take 8 bytes per
// row and tile.
constexpr long CHUNK_VALUES = 1L << 30, CHUNK_ROWS = 32768;
constexpr long SCORE_ROWS = 16384;

int pairs() {
  static const int n = [] {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return std::max(1, sms / 2);
  }();
  return n;
}

// Calls of up to this many rows run the products as W . X^T, with the rows as the tiles' columns (head_gemm.cuh).
constexpr long NARROW_ROWS = 128;

// Parts of K = V for dX. A wave of tiles takes kblocks / S blocks of 512 cycles (700 to read W, for few rows) and fills
// `pairs` pairs, or part of them in the last wave; each part adds a write and a read of rows x C fp32 partial sums (16
// bytes per value at about 5 TB/s = 2800 bytes a cycle).
int dx_splits(long rows, long V, int C) {
  const long tiles = up(rows, 256) / 256 * (up(C, 256) / 256), kblocks = up(V, 64) / 64;
  const double block = rows <= NARROW_ROWS ? 700 : 512;
  int best = 1;
  double least = 1e300;
  for (int S = 1; S <= 64 && S <= std::max(1L, kblocks / 16); ++S) {
    const long waves = (tiles * S + pairs() - 1) / pairs();
    const double cycles = waves * ((double)kblocks / S * block + 3000) + (double)S * rows * C * 16 / 2800;
    if (cycles < least * 0.995) {
      least = cycles;
      best = S;
    }
  }
  return best;
}

// Offsets in floats. Each is a multiple of 1 KB: a TMA box row of 128 bytes that straddles two lines costs twice the L2
// accesses (dW of 1024 tokens: 2.8 ms from a 16-byte aligned dz, 1.8 ms from an aligned one).
struct Layout {
  // rows of a chunk, row stride of the depths and of dz, 256-wide tiles of the vocabulary, groups of columns with
  // statistics and values between them, and for dX the parts of K and the rows between their partial sums
  long rows, ld_e, tiles, groups, part_ld, splits, split_rows;
  bool dw32;
  long kind, slot, row_of, counts, x, sidx, slogp, hit, coef, base2, tail, part, e, dx, dw, total;
};
Layout layout(long T, long V, int C, int K, bool grad_h, bool grad_w) {
  Layout l;
  long at = 0;
  auto take = [&](long floats) {
    const long o = at;
    at += up(floats, 256);
    return o;
  };
  const bool grad = grad_h || grad_w;
  l.ld_e = up(V, 64);
  l.tiles = up(V, 256) / 256;
  l.groups = T <= NARROW_ROWS ? l.tiles * 8 : l.tiles;
  l.rows = std::min(up(T, 64),
                    grad ? std::min(CHUNK_ROWS, std::max(256L, CHUNK_VALUES / l.ld_e / 256 * 256)) : SCORE_ROWS);
  l.dw32 = grad_w && l.rows < T;
  l.splits = grad_h ? dx_splits(l.rows, V, C) : 0;
  l.split_rows = up(l.rows, 256);
  l.kind = take(T);
  l.slot = take(T);
  l.row_of = take(T);
  l.counts = take(sizeof(Counts) / 4);
  l.x = take(up(T, 64) * C / 2);
  l.sidx = take(T * K);
  l.slogp = take(T * K);
  l.hit = take(T * K);
  l.coef = take(grad ? T * K : 0);
  l.base2 = take(T);
  l.tail = take(T);
  l.part_ld = std::min(T, l.rows);  // one row x 7760 groups: score_kernel 12 us, with values 512 bytes apart 21 us
  l.part = take(2 * l.groups * l.part_ld);
  l.e = take(grad ? l.rows * l.ld_e / 2 : 0);
  l.dx = take(l.splits * l.split_rows * C);
  l.dw = take(l.dw32 ? V * C : 0);
  l.total = at;
  return l;
}

bool map2d(CUtensorMap* map, bool f32, const void* base, long inner, long outer, long row_bytes, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)inner, (uint64_t)outer}, strides[1] = {(uint64_t)row_bytes};
  const uint32_t box[2] = {f32 ? 32u : 64u, (uint32_t)box_rows};
  return tmap::encode(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims,
                      strides, box);
}

template <int MODE, int NT = head::TILE>
cudaError_t launch(const head::Maps& maps, const head::Args& args, long units, cudaStream_t s) {
  static std::atomic<uint64_t> set{0};  // per device: the shared-memory size has been raised
  int dev = 0;
  RT_CUDA_CHECK(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!bit || !(set.load(std::memory_order_acquire) & bit)) {
    RT_CUDA_CHECK(cudaFuncSetAttribute(head::pair_kernel<MODE, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       head::Cfg<MODE, NT>::SMEM_BYTES));
    set.fetch_or(bit, std::memory_order_acq_rel);
  }
  const unsigned grid = 2 * (unsigned)std::min<long>(units, pairs());
  head::pair_kernel<MODE, NT><<<grid, head::THREADS, head::Cfg<MODE, NT>::SMEM_BYTES, s>>>(maps, args);
  return cudaGetLastError();
}

}  // namespace

extern "C" long rt_head_loss_workspace_floats(long rows, long V, int C, int K, int grad_h, int grad_w) {
  return layout(rows, V, C, K, grad_h != 0, grad_w != 0).total;
}

extern "C" cudaError_t rt_head_loss(const RtHeadLoss* p, float* work, cudaStream_t s) {
  return rt_head_loss_status(p, work, nullptr, s);
}

extern "C" cudaError_t rt_head_loss_status(const RtHeadLoss* p, float* work, int* status, cudaStream_t s) {
  if (!p || !work) return cudaErrorInvalidValue;
  const long T = p->rows, V = p->vocab;
  const int C = p->width, K = p->K;
  if (T < 0 || V < 1 || V > INT_MAX - 512 || T > (1 << 24) || C < 1 || C % 8 || K < 1 || K > RT_HEAD_MAX_RECORD ||
      (!p->log_probs && K != 1) || p->ld_hidden % 8 || p->ld_weight % 8 || (T && !p->hidden) || !p->weight ||
      ((reinterpret_cast<uintptr_t>(work) | reinterpret_cast<uintptr_t>(p->hidden) |
        reinterpret_cast<uintptr_t>(p->weight) | reinterpret_cast<uintptr_t>(p->dhidden) |
        reinterpret_cast<uintptr_t>(p->dweight)) & 15))
    return cudaErrorInvalidValue;
  if (T == 0) {
    if (p->reduction) RT_CUDA_CHECK(cudaMemsetAsync(p->loss, 0, sizeof(float), s));
    if (p->dweight) RT_CUDA_CHECK(cudaMemsetAsync(p->dweight, 0, (size_t)V * C * 2, s));
    return cudaSuccess;
  }
  const bool grad = p->dhidden || p->dweight;
  const Layout l = layout(T, V, C, K, p->dhidden != nullptr, p->dweight != nullptr);
  auto ints = [&](long at) { return reinterpret_cast<int*>(work + at); };
  Counts* counts = reinterpret_cast<Counts*>(work + l.counts);
  int* failed = status ? status : &counts->failed;
  __nv_bfloat16* x = reinterpret_cast<__nv_bfloat16*>(work + l.x);
  __nv_bfloat16* e = reinterpret_cast<__nv_bfloat16*>(work + l.e);
  float2* part = reinterpret_cast<float2*>(work + l.part);
  const float scale2 = p->scale * LOG2E;
  const bool narrow = T <= NARROW_ROWS, few = T <= 32;  // one chunk
  if (narrow && !grad && !p->log_probs) {  // scores: two launches, the rows where they are
    head::Maps maps;
    head::Args args{};
    args.rows = (int)T;
    args.V = (int)V;
    args.C = C;
    args.K = 1;
    args.scale2 = scale2 * mma_gain(C);
    args.part = part;
    args.part_ld = l.part_ld;
    args.targets = p->index;
    args.counts = &counts->valid;
    args.status = failed;
    if (!map2d(&maps.a, false, p->weight, C, V, 2 * p->ld_weight, 128) ||
        !map2d(&maps.b, false, p->hidden, C, T, 2 * p->ld_hidden, few ? 16 : 64) ||
        !map2d(&maps.out, false, p->hidden, C, T, 2 * p->ld_hidden, 32))
      return cudaErrorInvalidValue;
    RT_CUDA_CHECK((few ? launch<head::LOGITS_N, 32>(maps, args, l.tiles, s)
                       : launch<head::LOGITS_N, 128>(maps, args, l.tiles, s)));
    const ScoreArgs score{part, l.part_ld, (int)l.groups, p->reduction == 2, p->index, p->ignore, V,
                          reinterpret_cast<const __nv_bfloat16*>(p->hidden), p->ld_hidden,
                          reinterpret_cast<const __nv_bfloat16*>(p->weight), p->ld_weight, C, scale2, counts,
                          failed, p->row_loss, p->reduction ? p->loss : nullptr};
    score_kernel<<<(unsigned)T, MERGE_THREADS + 32, 0, s>>>(score);
    return cudaGetLastError();
  }
  const bool brief = T * K <= SHORT_ENTRIES;
  const Upstream upstream{p->scale, p->reduction == 2, p->row_grad};
  if (!brief) {
    if (p->log_probs) kinds_kernel<<<(unsigned)((T * 32 + 255) / 256), 256, 0, s>>>(p->index, T, K, V, ints(l.kind));
    pack_kernel<<<1, 1024, 0, s>>>(p->log_probs ? ints(l.kind) : nullptr, p->index, p->ignore, V, T, upstream,
                                   ints(l.slot), counts);
  }
  int Kp = 1;
  while (Kp < K) Kp <<= 1;
  const unsigned share = (unsigned)std::max(1L, std::min((K + 7L) / 8, 296 / T));  // blocks of a row: two per SM in all
  gather_kernel<<<dim3((unsigned)(T + 64), share), 256, Kp * 8, s>>>(
      p->index, p->log_probs, K, Kp, T, reinterpret_cast<const __nv_bfloat16*>(p->hidden), p->ld_hidden,
      reinterpret_cast<const __nv_bfloat16*>(p->weight), p->ld_weight, C, scale2, V, p->ignore, brief, upstream,
      ints(l.slot), counts, ints(l.row_of), reinterpret_cast<uint4*>(x), ints(l.sidx), work + l.slogp, work + l.hit,
      p->row_loss, reinterpret_cast<uint4*>(p->dhidden));
  RT_CUDA_CHECK(cudaGetLastError());

  head::Maps logits, dx, dw;
  head::Args args{};
  args.live = &counts->valid;
  args.V = (int)V;
  args.C = C;
  args.K = K;
  args.scale2 = scale2 * mma_gain(C);
  args.part = part;
  args.e = reinterpret_cast<unsigned short*>(e);
  args.ld_e = l.ld_e;
  args.dx = work + l.dx;
  args.part_ld = l.part_ld;
  args.store_e = grad;
  args.splits = (int)std::max(1L, l.splits);
  args.split_rows = (int)l.split_rows;
  args.status = failed;
  int merge_blocks = 0;
  for (long row0 = 0; row0 < T; row0 += l.rows)
    merge_blocks += (int)(std::min(l.rows, up(T - row0, 64)) / (narrow ? 1 : 4));  // multiples of 64
  for (long row0 = 0; row0 < T; row0 += l.rows) {
    const long rows = std::min(l.rows, up(T - row0, 64));  // packed rows of x are filled up to a block of 64
    __nv_bfloat16* xc = x + row0 * C;
    args.row0 = (int)row0;
    args.rows = (int)l.rows;
    args.sidx = ints(l.sidx) + row0 * K;
    args.add = row0 > 0;
    const long tiles_m = up(rows, 256) / 256, tiles_c = up(C, 256) / 256;
    CUtensorMap* of_x = narrow ? &logits.b : &logits.a;
    if (!map2d(of_x, false, xc, C, rows, 2L * C, few ? 16 : narrow ? 64 : 128) ||
        !map2d(narrow ? &logits.a : &logits.b, false, p->weight, C, V, 2 * p->ld_weight, 128) ||
        !map2d(&logits.out, false, grad ? (void*)e : (void*)xc, grad ? V : C, rows, 2 * (grad ? l.ld_e : C), 32))
      return cudaErrorInvalidValue;
    RT_CUDA_CHECK((few      ? launch<head::LOGITS_N, 32>(logits, args, l.tiles, s)
                   : narrow ? launch<head::LOGITS_N, 128>(logits, args, l.tiles, s)
                            : launch<head::LOGITS>(logits, args, tiles_m * l.tiles, s)));
    MergeArgs m{part, l.part_ld, (int)l.groups, (int)row0, (int)l.rows, K, p->tail, p->reduction == 2, merge_blocks, T,
                counts, failed, ints(l.row_of), ints(l.sidx), work + l.slogp, work + l.hit, p->row_grad, p->row_loss,
                p->reduction ? p->loss : nullptr, work + l.base2, work + l.tail,
                grad ? work + l.coef : nullptr};
    if (narrow) merge_kernel<1><<<(unsigned)rows, MERGE_THREADS, 0, s>>>(m);
    else merge_kernel<4><<<(unsigned)(rows + 3) / 4, MERGE_THREADS, 0, s>>>(m);
    if (grad)
      gradient_kernel<<<dim3((unsigned)((l.tiles + 31) / 32), (unsigned)rows), 256, 0, s>>>(
          e, l.ld_e, (int)V, (int)row0, (int)l.rows, counts, part, l.part_ld, narrow ? 32 : 256,
          work + l.base2, work + l.tail, K, ints(l.sidx), work + l.coef);
    RT_CUDA_CHECK(cudaGetLastError());
    if (p->dhidden) {
      if (!map2d(narrow ? &dx.b : &dx.a, false, e, V, rows, 2 * l.ld_e, few ? 16 : narrow ? 64 : 128) ||
          !map2d(narrow ? &dx.a : &dx.b, false, p->weight, C, V, 2 * p->ld_weight, 64) ||
          !map2d(&dx.out, true, work + l.dx, C, l.splits * l.split_rows, 4L * C, 32))
        return cudaErrorInvalidValue;
      RT_CUDA_CHECK((few      ? launch<head::DX_N, 32>(dx, args, tiles_c * l.splits, s)
                     : narrow ? launch<head::DX_N, 128>(dx, args, tiles_c * l.splits, s)
                              : launch<head::DX>(dx, args, tiles_m * tiles_c * l.splits, s)));
      dhidden_kernel<<<(unsigned)rows, 256, 0, s>>>(work + l.dx, (int)l.splits, l.split_rows, C, (int)row0, (int)l.rows,
                                                    counts, failed, ints(l.row_of),
                                                    reinterpret_cast<__nv_bfloat16*>(p->dhidden));
    }
    if (p->dweight) {
      void* out = l.dw32 ? (void*)(work + l.dw) : p->dweight;
      if (!map2d(&dw.a, false, e, V, rows, 2 * l.ld_e, 64) || !map2d(&dw.b, false, xc, C, rows, 2L * C, 64) ||
          !map2d(&dw.out, l.dw32, out, C, V, (l.dw32 ? 4L : 2L) * C, 32))
        return cudaErrorInvalidValue;
      const long units = l.tiles * tiles_c;
      args.poison = static_cast<uint4*>(p->dweight);
      args.factor = &counts->factor;
      RT_CUDA_CHECK(l.dw32 ? launch<head::DW32>(dw, args, units, s) : launch<head::DW>(dw, args, units, s));
    }
  }
  if (l.dw32) {
    RT_CUDA_CHECK(rt_to_bf16(work + l.dw, p->dweight, V * C, s));
    failed_kernel<<<1, 32, 0, s>>>(failed, reinterpret_cast<__nv_bfloat16*>(p->dweight));
  }
  return cudaGetLastError();
}

// x[t] [n[t]] bf16 *= *factor (device scalar), t = 0, 1 (n = 0: none).
extern "C" cudaError_t rt_scale_bf16(void* const x[2], const long n[2], const float* factor, cudaStream_t s) {
  const long most = std::max(n[0], n[1]);
  if (most <= 0) return cudaSuccess;
  ScaleArgs p;
  for (int t = 0; t < 2; ++t) {
    if (reinterpret_cast<uintptr_t>(x[t]) & 15) return cudaErrorInvalidValue;
    p.x[t] = reinterpret_cast<__nv_bfloat16*>(x[t]);
    p.n[t] = n[t];
  }
  scale_kernel<<<(unsigned)std::min((most / 8 + 255) / 256 + 1, 148L * 8), 256, 0, s>>>(p, factor);
  return cudaGetLastError();
}
