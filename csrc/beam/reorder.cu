// Rows of many tensors replaced by their parents' rows, in place, in one launch.
//
// A block takes a range of columns of one group of one tensor: each thread reads its columns of every row that another
// slot takes over, then writes them to the slots that do. All reads of a column precede its writes and no other thread
// touches it, so any indices are safe without scratch memory, cycles and rows taken more than once included. Rows that
// stay are neither read (unless a slot takes them over) nor written.
//
// Bound by memory: one read of each row that moves and one write of each that changes. 128 states of 172 MB per row, two of
// four rows moving in two groups (1.4 GB): 225 us, 6.2 TB/s.
#include <algorithm>
#include <climits>
#include "../api.h"
#include "../common/common.cuh"

namespace {

constexpr int THREADS = 256, MAX_ITEMS = 128;

struct Item {
  char* base;
  long bytes;   // of a row
  long chunks;  // blocks of this tensor and all before it
};
struct ReorderArgs {
  Item item[MAX_ITEMS];
  const long* parents;
  int items, K, width;  // bytes that a thread moves at once
};

template <int N> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<4> { using type = unsigned; };
template <> struct Word<1> { using type = unsigned char; };

// Columns of a thread: as many as fit some 32 words of 16 bytes in flight.
constexpr int columns(int beams) { return beams >= 16 ? 1 : 16 / beams; }

template <int B, int WIDTH>
__device__ __forceinline__ void move(char* rows, long bytes, long chunk, const unsigned* children, int K) {
  using W = typename Word<WIDTH>::type;
  constexpr int U = columns(B);
  const long words = bytes / WIDTH;
  const long c0 = chunk * (THREADS * U) + threadIdx.x;
  W v[B][U];
#pragma unroll
  for (int j = 0; j < B; ++j)
    if (j < K && children[j])
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (c0 + i * THREADS < words) v[j][i] = *reinterpret_cast<const W*>(rows + j * bytes + (c0 + i * THREADS) * WIDTH);
#pragma unroll
  for (int j = 0; j < B; ++j) {
    if (j >= K) break;
    for (unsigned to = children[j]; to; to &= to - 1) {
      const int k = __ffs(to) - 1;
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (c0 + i * THREADS < words) *reinterpret_cast<W*>(rows + k * bytes + (c0 + i * THREADS) * WIDTH) = v[j][i];
    }
  }
}

// Grid (chunks of all tensors, groups).
template <int B>
__global__ void __launch_bounds__(THREADS) reorder_kernel(const __grid_constant__ ReorderArgs a) {
  __shared__ unsigned children[B];  // slots other than itself that take a slot's row over
  const int tid = threadIdx.x, K = a.K;
  const long group = blockIdx.y;
  if (tid < B) children[tid] = 0;
  __syncthreads();
  if (tid < K) {
    const long p = a.parents[group * K + tid];
    if (p >= 0 && p < K && p != tid) atomicOr(&children[p], 1u << tid);
  }
  __syncthreads();
  int lo = 0, hi = a.items - 1;  // first tensor whose blocks end behind this one
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.item[mid].chunks > (long)blockIdx.x) hi = mid;
    else lo = mid + 1;
  }
  const Item it = a.item[lo];
  const long chunk = blockIdx.x - (lo ? a.item[lo - 1].chunks : 0);
  char* rows = it.base + group * K * it.bytes;
  if (a.width == 16) move<B, 16>(rows, it.bytes, chunk, children, K);
  else if (a.width == 4) move<B, 4>(rows, it.bytes, chunk, children, K);
  else move<B, 1>(rows, it.bytes, chunk, children, K);
}

template <int B>
cudaError_t launch(ReorderArgs& a, long groups, cudaStream_t s) {
  const long per = (long)THREADS * columns(B) * a.width;
  long chunks = 0;
  for (int i = 0; i < a.items; ++i) a.item[i].chunks = chunks += (a.item[i].bytes + per - 1) / per;
  if (chunks > INT_MAX) return cudaErrorInvalidValue;
  for (long g = 0; g < groups; g += 65535) {
    ReorderArgs b = a;
    b.parents += g * a.K;
    for (int i = 0; i < a.items; ++i) b.item[i].base += g * a.K * a.item[i].bytes;
    reorder_kernel<B><<<dim3((unsigned)chunks, (unsigned)std::min(groups - g, 65535L)), THREADS, 0, s>>>(b);
  }
  return cudaGetLastError();
}

cudaError_t launch(ReorderArgs& a, long groups, cudaStream_t s) {
  if (a.K <= 2) return launch<2>(a, groups, s);
  if (a.K <= 4) return launch<4>(a, groups, s);
  if (a.K <= 8) return launch<8>(a, groups, s);
  if (a.K <= 16) return launch<16>(a, groups, s);
  return launch<32>(a, groups, s);
}

}  // namespace

// n tensors of groups * K rows of bytes[i] > 0 each, disjoint; parents [groups, K].
extern "C" cudaError_t rt_reorder_rows(void* const* base, const long* bytes, int n, const long* parents, long groups,
                                       int K, cudaStream_t s) {
  if (n < 0 || groups < 0 || K < 1 || K > 32) return cudaErrorInvalidValue;
  if (n == 0 || groups == 0) return cudaSuccess;
  // tensors of a width together: those that 16-byte words divide, then 4-byte words, then single bytes
  for (int width : {16, 4, 1}) {
    ReorderArgs a{};
    a.parents = parents;
    a.K = K;
    a.width = width;
    for (int i = 0; i < n; ++i) {
      const unsigned long bits = reinterpret_cast<uintptr_t>(base[i]) | (unsigned long)bytes[i];
      if (bytes[i] <= 0) return cudaErrorInvalidValue;
      if ((bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1) != width) continue;
      a.item[a.items++] = {static_cast<char*>(base[i]), bytes[i], 0};
      if (a.items == MAX_ITEMS) {
        RT_CUDA_CHECK(launch(a, groups, s));
        a.items = 0;
      }
    }
    if (a.items) RT_CUDA_CHECK(launch(a, groups, s));
  }
  return cudaGetLastError();
}
