// Rows of many tensors replaced by their parents' rows, in place, in one launch.
//
// A block takes a range of columns of one group of one tensor: each thread reads its columns of every row that another
// slot takes over, then writes them to the slots that do. All reads of a column precede its writes and no other thread
// touches it, so any indices are safe without scratch memory, cycles and rows taken more than once included. Rows that
// stay are neither read (unless a slot takes them over) nor written.
//
// Bound by memory: one read of each row that moves and one write of each that changes. What is held in registers follows the
// rows that are taken over, not the beams: few of many leave room for more columns of each. 128 states of 172 MB per row, two
// of four rows moving in two groups (1.4 GB): 217 us, 6.5 TB/s; 20 of 27 rows of 7.5 MB: 42 us, 4.8 TB/s (80 us with registers
// for every beam).
#include <algorithm>
#include <climits>
#include "../api.h"
#include "../common/common.cuh"

namespace {

constexpr int THREADS = 256, MAX_ITEMS = 128, ENOUGH = 592;  // blocks: four per SM

struct Item {
  char* base;
  long bytes;   // of a row
  long chunks;  // blocks of this tensor and all before it
};
struct ReorderArgs {
  Item item[MAX_ITEMS];
  const long* parents;
  int items, K, width;  // bytes that a thread moves at once
  long columns;         // words of a row that a block moves
};

template <int N> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = unsigned; };
template <> struct Word<1> { using type = unsigned char; };

// Columns [c0, end) of the rows that are taken over (N of them at most, held), U columns of each in a thread's registers.
template <int N, int U, int WIDTH>
__device__ __forceinline__ void move(char* rows, long bytes, long c0, long end, const int* from, const unsigned* children,
                                     int held) {
  using W = typename Word<WIDTH>::type;
#pragma unroll 1
  for (; c0 < end; c0 += THREADS * U) {
    W v[N][U];
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < held) {
        const W* row = reinterpret_cast<const W*>(rows + from[j] * bytes);
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (c0 + i * THREADS < end) v[j][i] = row[c0 + i * THREADS];
      }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j >= held) break;
      for (unsigned to = children[j]; to; to &= to - 1) {
        W* row = reinterpret_cast<W*>(rows + (__ffs(to) - 1) * bytes);
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (c0 + i * THREADS < end) row[c0 + i * THREADS] = v[j][i];
      }
    }
  }
}

// As many columns of each row as keep 16 words in flight per thread (of half the size where 32 rows may be held: registers
// for two blocks per SM).
template <int B, int CAP, int WIDTH, int N = 1>
__device__ __forceinline__ void move_held(char* rows, long bytes, long c0, long end, const int* from,
                                          const unsigned* children, int held) {
  if constexpr (N < B) {
    if (held > N) return move_held<B, CAP, WIDTH, 2 * N>(rows, bytes, c0, end, from, children, held);
  }
  if constexpr (N == 32 && WIDTH == 16)
    move<N, 1, 8>(rows, bytes, 2 * (c0 - threadIdx.x) + threadIdx.x, 2 * end, from, children, held);
  else
    move<N, N >= 16 ? 1 : N * CAP >= 16 ? 16 / N : CAP, WIDTH>(rows, bytes, c0, end, from, children, held);
}

// Grid (chunks of all tensors, groups).
template <int B, int CAP>
__global__ void __launch_bounds__(THREADS) reorder_kernel(const __grid_constant__ ReorderArgs a) {
  __shared__ int from[THREADS / 32][B];           // the rows that other slots take over (each warp finds them for itself,
  __shared__ unsigned children[THREADS / 32][B];  // which takes no barrier), and those slots
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.K;
  const long group = blockIdx.y;
  const long p = lane < K ? a.parents[group * K + lane] : -1;
  const bool moves = p >= 0 && p < K && p != lane;
  const unsigned siblings = __match_any_sync(~0u, moves ? (int)p : 32 + lane);
  const bool first = moves && __ffs(siblings) - 1 == lane;
  const unsigned firsts = __ballot_sync(~0u, first);
  const int held = __popc(firsts);
  if (held == 0) return;
  if (first) {
    const int at = __popc(firsts & ((1u << lane) - 1));
    from[warp][at] = (int)p;
    children[warp][at] = siblings;
  }
  __syncwarp();
  int lo = 0, hi = a.items - 1;  // first tensor whose blocks end behind this one
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.item[mid].chunks > (long)blockIdx.x) hi = mid;
    else lo = mid + 1;
  }
  const Item it = a.item[lo];
  const long chunk = blockIdx.x - (lo ? a.item[lo - 1].chunks : 0);
  char* rows = it.base + group * K * it.bytes;
  const long c0 = chunk * a.columns + tid, end = min((chunk + 1) * a.columns, it.bytes / a.width);
  if (a.width == 16) move_held<B, CAP, 16>(rows, it.bytes, c0, end, from[warp], children[warp], held);
  else if (a.width == 4) move_held<B, CAP, 4>(rows, it.bytes, c0, end, from[warp], children[warp], held);
  else move_held<B, CAP, 1>(rows, it.bytes, c0, end, from[warp], children[warp], held);
}

template <int B>
cudaError_t launch(ReorderArgs& a, long groups, cudaStream_t s) {
  // 16 words per thread, fewer where the blocks would be too few for the SMs; from four on a block's own start costs more
  // (three rows of 1.9 MB: 9 us with blocks of four words and 13 with blocks of one). Its code takes no more than four at once
  // then: a block waits for its code as well (four rows of 1.9 MB: 6 us).
  int words = 16;
  long chunks = 0;
  for (;; words /= 2) {
    a.columns = (long)THREADS * words;
    const long per = a.columns * a.width;
    chunks = 0;
    for (int i = 0; i < a.items; ++i) a.item[i].chunks = chunks += (a.item[i].bytes + per - 1) / per;
    if (words == 4 || chunks * groups >= ENOUGH) break;
  }
  if (chunks > INT_MAX) return cudaErrorInvalidValue;
  for (long g = 0; g < groups; g += 65535) {
    ReorderArgs b = a;
    b.parents += g * a.K;
    for (int i = 0; i < a.items; ++i) b.item[i].base += g * a.K * a.item[i].bytes;
    const dim3 grid((unsigned)chunks, (unsigned)std::min(groups - g, 65535L));
    if (words == 4) reorder_kernel<B, 4><<<grid, THREADS, 0, s>>>(b);
    else reorder_kernel<B, 16><<<grid, THREADS, 0, s>>>(b);
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
