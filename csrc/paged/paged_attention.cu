// Attention of one token per row over the pages of a cache (paged.py has the definition).
//
// Bound by memory: every page that a row or its group's other beams hold has to be read once. So a block takes the
// rows of a group together (one key head, every splits-th tile of 64 keys): of each tile it loads the pages that
// differ between the rows, and each of them meets the queries of all rows that hold it (up to 64 queries; rows that do
// not hold it are left out). Roles (128 threads):
//   warp 2      finds the tile's distinct pages (a lane per row) and brings their keys and values into a ring with TMA
//               (128-byte swizzle, boxes of 64 components);
//   warp 3      issues S = Q K^T (M = 128, N = 64) into one of two TMEM buffers and O += P V (N = dim), V read MN-major.
//               The queries are rows 0-63 of the tile; what the products make of the rows behind them, which are whatever
//               lies in shared memory there, stays in TMEM lanes that nobody reads;
//   warps 0, 1  softmax, a thread per query: scores against the query's reference, which is raised (O rescaled in TMEM)
//               only where a score exceeds it by 2^8; P in bf16 (2^-8 of each weight at most, which the product needs; sums
//               and outputs are fp32) in place of the scores. With two threads per query every unit needs their agreement.
//
// Eight beams of 32 k shared tokens, 24 / 4 heads of 256 (135 MB): 34 us, of which 4 until the first tile, 25 for the tiles
// (5.3 TB/s; about 1900 cycles each from L2: scores 730, then weights and their product, which follow one another) and 2-3
// for the results, then 5 us to join them. The same with mma.sync (16 keys x 8 queries per instruction) took 76 us: its
// operand loads alone are 2300 cycles of shared memory per tile, against 2700 that the tile's bytes leave. Queries of a row
// of 24 / 4 heads are 6 of a tile's 128 rows; a block's time does not depend on how many there are, as the tile's bytes and
// the products' latency bound it. Tried without gain: one copy for a tile's keys instead of one per 64 components, a
// shorter way to the classes of rows that are all alike (40 us in all against 39).
//
// Keys that a row does not see (behind its last token, or in a missing page) get the weight 0 whatever they hold:
// their scores are replaced, their values zeroed in shared memory.
#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>
#include <cuda.h>
#include "../api.h"
#include "../common/common.cuh"
#include "../common/sm100.cuh"
#include "../common/tmap.cuh"

namespace {

using bf16 = __nv_bfloat16;
constexpr int TILE = 64, QUERIES = 64, THREADS = 128;  // keys of a unit, queries of a block
constexpr int MAX_SPLITS = 296, UNITS = 8;
constexpr int AHEAD = 8, APART = 16;  // tiles whose pages are looked up together; last tiles that may be dealt out by units
constexpr float HEADROOM = 8.f;  // log2 that a score may exceed its reference by before that is raised

struct AttendArgs {
  int pages, panels, first, kv_heads, page, width, splits;
  int rows, group, together, subgroups;  // rows of a block at most, blocks per group of beams
  int heads, per_kv;
  const int* table;
  const int* lengths;
  const bf16* q;
  long q_row, q_head;
  int q_vec;       // rows of q are 16-byte aligned
  const bf16* gate;
  long gate_row, gate_head;
  float scale_log2;
  bf16* out;
  float* sums;     // [rows, heads, splits, dim]
  float2* stats;   // [rows, heads, splits]: reference in log2 units, sum of exponentials
};

// A unit: a tile's pages as some rows hold them.
struct Unit {
  uint32_t members;  // rows; 0: no more units
  int valid;         // keys before the rows' end
  uint32_t there;    // 16-key blocks whose page exists
  uint64_t queries;  // of the members
};

static_assert(sizeof(Unit) == 24, "room for the units");

template <int D> struct Shape {
  // TMEM: O, two buffers of scores (whose weights replace them), and the queries where they fit beside them (D / 2 columns;
  // products then read 4 KB less of shared memory each, which is what bounds them at N = 64). Two blocks per SM below 256.
  static constexpr uint32_t COLUMNS = D == 256 ? 512 : 256, S = D, Q_COLUMN = S + 2 * TILE;
  static constexpr bool Q_TMEM = Q_COLUMN + D / 2 <= COLUMNS;
  static constexpr int BOX = TILE * 128;                            // 64 components of a tile's keys or values
  static constexpr int HALF = TILE * D * 2;                         // all of them
  static constexpr int RING = D == 256 ? 6 : D == 128 ? 5 : 8;      // tiles of keys or values
  // products read 64 rows more than a tile of queries in shared memory has: what follows has to be as long
  static constexpr int Q = 0;                                       // [D / 64][64][64]
  static constexpr int KV = Q + (Q_TMEM ? 0 : QUERIES * D * 2);
  static constexpr int TABLE = KV + RING * HALF;                    // [32 rows][4][AHEAD tiles]
  static constexpr int TAIL = TABLE + 32 * 4 * AHEAD * 4;           // [32 rows][4][APART tiles]
  static constexpr int UNIT = TAIL + 32 * 4 * APART * 4;
  static constexpr int BARS = UNIT + UNITS * 24;
  static constexpr int BYTES = BARS + 8 * (2 * RING + UNITS + 8) + 16 + 1024;
  static constexpr uint32_t IDESC_S = sm100::idesc_bf16(128, TILE, false, false);
  static constexpr uint32_t IDESC_O = sm100::idesc_bf16(128, D, false, true);
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// D = A B (+ D) with A in TMEM: two bf16 per column of its row's lane.
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D += A B in the TMEM lanes whose bit is set among the first 64 (the others are not written, whatever the product is).
__device__ __forceinline__ void mma_lanes(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t lo, uint32_t hi) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %7, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%4, %5, %6, %6}, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(~lo), "r"(~hi), "r"(~0u), "r"(1u)
      : "memory");
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Grid (splits, key heads, groups x subgroups).
template <int D>
__global__ void __launch_bounds__(THREADS) attend_kernel(const __grid_constant__ CUtensorMap map, const AttendArgs a) {
  using Sh = Shape<D>;
  constexpr int RING = Sh::RING, HALF = Sh::HALF, BOX = Sh::BOX, BOXES = D / 64;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = sm100::align_smem_1024(raw);
  uint8_t *sQ = smem + Sh::Q, *sKV = smem + Sh::KV;
  int *sTable = reinterpret_cast<int*>(smem + Sh::TABLE), *sTail = reinterpret_cast<int*>(smem + Sh::TAIL);
  Unit* units = reinterpret_cast<Unit*>(smem + Sh::UNIT);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Sh::BARS);  // a tile of the ring has landed
  uint64_t* empty = full + RING;                                  // its products are done
  uint64_t* known = empty + RING;                                 // [UNITS] a unit's description is there
  uint64_t* q_full = known + UNITS;
  uint64_t* s_full = q_full + 1;  // [2]
  uint64_t* p_full = s_full + 2;  // [2]
  uint64_t* o_done = p_full + 2;  // [2]
  uint64_t* drain = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x, kv = blockIdx.y, g = blockIdx.z / a.subgroups, sub = blockIdx.z % a.subgroups;
  const int row0 = g * a.group + sub * a.together, rows = min(a.together, a.group - sub * a.together);
  const int capacity = a.width * a.page, span = TILE / a.page;  // pages of a tile
  int length = 0;  // of row0 + lane, for the loads
  if (warp == 2) {
    sm100::prefetch_tmap(&map);
    if (lane < rows) length = min(max(a.lengths[row0 + lane], 0), capacity);
  }
  if (tid == 0) {
    for (int i = 0; i < RING; ++i) {
      sm100::mbar_init(&full[i], 1);
      sm100::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < UNITS; ++i) sm100::mbar_init(&known[i], 1);
    sm100::mbar_init(q_full, QUERIES);
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(&s_full[i], 1);
      sm100::mbar_init(&p_full[i], QUERIES);
      sm100::mbar_init(&o_done[i], 1);
    }
    sm100::mbar_init(drain, 1);
    *abort = 0;
    sm100::fence_barrier_init();
  }
  if (warp == 3) {
    sm100::tmem_alloc(tmem_slot, Sh::COLUMNS);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 2) {
    // ------------------------------------------------------------ loads
    const int longest = __reduce_max_sync(~0u, length);
    const int count = (longest + TILE - 1) / TILE;
    // The rows' pages of N tiles, a lane per tile, so that their loads wait for memory together (-1: no such page);
    // to[(row * 4 + j) * N + tile]. Returns whether the lane's tile is another one for some row than for the first.
    auto look_up = [&](auto tiles, int first, int step, int* to) {
      constexpr int N = decltype(tiles)::value;
      const int i = first + lane * step;
      const int n0 = min(max(__shfl_sync(~0u, length, 0) - i * TILE, 0), TILE);
      int e0[4];
      bool apart = false;
      for (int r0 = 0; r0 < rows; r0 += 8) {
        int e[8][4];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int n = __shfl_sync(~0u, length, (r0 + r) & 31);  // 0 behind the last row
          const int* table = a.table + (long)(row0 + r0 + r) * a.width;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            e[r][j] = lane < N && j < span && i < count && i * TILE + j * a.page < n ? table[i * span + j] : -1;
          apart |= r0 + r < rows && min(max(n - i * TILE, 0), TILE) != n0;
        }
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int page = e[r][j] < a.pages ? max(e[r][j], -1) : -1;
            if (r == 0 && r0 == 0) e0[j] = page;
            apart |= r0 + r < rows && page != e0[j];
            if (lane < N) to[((r0 + r) * 4 + j) * N + lane] = page;
          }
      }
      __syncwarp();
      return apart && lane < N && i < count;
    };
    const uint64_t one = a.per_kv == 64 ? ~0ull : (1ull << a.per_kv) - 1;  // the queries of row 0
    int entry = 0, unit = 0;  // tiles of the ring (keys, values, keys, ...) and units so far
    bool ok = true;
    // The tiles are dealt out to the splits in turn; from the first of the last APART on where rows have gone apart, the
    // units one by one.
    const int window = max(count - APART, 0);
    const unsigned apart = __ballot_sync(~0u, look_up(std::integral_constant<int, APART>{}, window, 1, sTail));
    const int tail = apart ? window + __ffs(apart) - 1 : count;
    int dealt = tail;  // units before the next one, where they are dealt out
    for (int i = split < tail ? split : tail, t = 0; i < count && ok; t = (t + 1) % AHEAD) {
      const bool single = i >= tail;
      if (!single && i < window && t == 0) look_up(std::integral_constant<int, AHEAD>{}, i, a.splits, sTable);
      int e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        e[j] = lane >= rows  ? -1
               : i >= window ? sTail[(lane * 4 + j) * APART + i - window]
                             : sTable[(lane * 4 + j) * AHEAD + t];
      const int valid = min(max(length - i * TILE, 0), TILE);
      unsigned same = __match_any_sync(~0u, valid);
      bool any = false;
      unsigned there = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        same &= __match_any_sync(~0u, e[j]);
        any |= e[j] >= 0;
        if (e[j] >= 0) there |= ((1u << (a.page / 16)) - 1) << (j * (a.page / 16));
      }
      unsigned left = __ballot_sync(~0u, any && valid > 0);
      while (left && ok) {
        const int leader = __ffs(left) - 1;
        Unit u;
        u.members = __shfl_sync(~0u, same, leader);
        u.valid = __shfl_sync(~0u, valid, leader);
        u.there = __shfl_sync(~0u, there, leader);
        left &= ~u.members;
        if (single && dealt++ % a.splits != split) continue;
        u.queries = 0;
        for (uint32_t k = u.members; k; k &= k - 1) u.queries |= one << ((__ffs(k) - 1) * a.per_kv);
        int p[4], here = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[j] = __shfl_sync(~0u, e[j], leader);
          here += p[j] >= 0;
        }
        for (int kind = 0; kind < 2; ++kind) {
          const int slot = entry % RING;
          ok = __all_sync(~0u, entry < RING || sm100::mbar_wait(&empty[slot], (entry / RING - 1) & 1, abort));
          if (!ok) break;
          if (lane == 0) {
            if (kind == 0) {
              // eight units before this one the softmax is done: the ring holds four at most
              units[unit % UNITS] = u;
              sm100::mbar_arrive(&known[unit % UNITS]);
            }
            sm100::mbar_expect_tx(&full[slot], here * a.page * D * 2);
          }
          __syncwarp();
          const int j = lane / BOXES, box = lane % BOXES;  // a copy per lane
          const int page = j == 0 ? p[0] : j == 1 ? p[1] : j == 2 ? p[2] : p[3];
          if (j < span && page >= 0) {
            const int y = (page * a.panels + a.first + kind * a.kv_heads + kv) * a.page;
            sm100::tma_load_2d(sKV + slot * HALF + box * BOX + j * a.page * 128, &map, &full[slot], box * 64, y);
          }
          __syncwarp();
          ++entry;
        }
        ++unit;
      }
      __syncwarp();
      if (single) ++i;
      else i = min(i + a.splits, tail);
    }
    if (ok && lane == 0) {
      units[unit % UNITS].members = 0;
      sm100::mbar_arrive(&known[unit % UNITS]);
    }
    // copies in flight have to land before the block ends (all have where the products were done)
    if (!ok)
      for (int i = max(entry - RING, 0); i < entry; ++i) sm100::mbar_wait_bounded(&full[i % RING], (i / RING) & 1);
  } else if (warp == 3) {
    // ------------------------------------------------------------ products
    if (sm100::elect_one()) {
      const uint32_t qb = sm100::smem_u32(sQ);
      bool ok = sm100::mbar_wait(q_full, 0, abort), last = false;
      sm100::tc_fence_after();
      auto scores = [&](int u) {  // of unit u, unless there is none
        if (!sm100::mbar_wait(&known[u % UNITS], (u / UNITS) & 1, abort)) return false;
        if (units[u % UNITS].members == 0) {
          last = true;
          return true;
        }
        const int entry = 2 * u, slot = entry % RING;
        if (!sm100::mbar_wait(&full[slot], (entry / RING) & 1, abort)) return false;
        sm100::tc_fence_after();
        const uint32_t kb = sm100::smem_u32(sKV + slot * HALF);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t d = tmem + Sh::S + (u & 1) * TILE;
          const uint64_t bd = sm100::smem_desc(kb + (k >> 2) * BOX + (k & 3) * 32, 16, 1024);
          if (Sh::Q_TMEM)
            mma_tmem(d, tmem + Sh::Q_COLUMN + k * 8, bd, Sh::IDESC_S, k > 0);
          else
            sm100::mma_bf16(d, sm100::smem_desc(qb + (k >> 2) * BOX + (k & 3) * 32, 16, 1024), bd, Sh::IDESC_S, k > 0);
        }
        sm100::mma_commit(&s_full[u & 1]);
        sm100::mma_commit(&empty[slot]);
        return true;
      };
      if (ok) ok = scores(0);
      int end = last ? 0 : 1;  // units whose scores are formed
      if (ok && !last) {
        ok = scores(1);
        end += !last;
      }
      for (int u = 0; ok && u < end; ++u) {
        const int entry = 2 * u + 1, slot = entry % RING;
        if (!sm100::mbar_wait(&p_full[u & 1], (u >> 1) & 1, abort)) break;
        if (!sm100::mbar_wait(&full[slot], (entry / RING) & 1, abort)) break;
        sm100::tc_fence_after();
        const uint64_t queries = units[u % UNITS].queries;
        const uint32_t vb = sm100::smem_u32(sKV + slot * HALF);
#pragma unroll
        for (int k = 0; k < TILE / 16; ++k) {
          const uint64_t bd = sm100::smem_desc(vb + k * 2048, BOX, 1024);
          mma_lanes(tmem, tmem + Sh::S + (u & 1) * TILE + k * 8, bd, Sh::IDESC_O, (uint32_t)queries, (uint32_t)(queries >> 32));
        }
        sm100::mma_commit(&o_done[u & 1]);
        sm100::mma_commit(&empty[slot]);
        if (!last) {
          // the next scores take the weights' columns, which this product reads
          ok = sm100::mbar_wait(&o_done[u & 1], (u >> 1) & 1, abort) && scores(u + 2);
          end += !last;
        }
      }
      sm100::mma_commit(drain);
      sm100::mbar_wait_bounded(drain, 0);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax
    const int n = tid, row = n / a.per_kv, h = n % a.per_kv;
    const bool used = row < rows;  // a query, of row0 + row
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    // queries into the product's layout (zeros where there is none)
    if (Sh::Q_TMEM) {
      const bf16* x = a.q + (row0 + row) * a.q_row + (long)(kv * a.per_kv + h) * a.q_head;
#pragma unroll 2
      for (int c = 0; c < D; c += 64) {
        uint4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          v[k] = make_uint4(0, 0, 0, 0);
          if (used && a.q_vec) {
            v[k] = *reinterpret_cast<const uint4*>(x + c + k * 8);
          } else if (used) {
            bf16* e = reinterpret_cast<bf16*>(&v[k]);
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = x[c + k * 8 + j];
          }
        }
        float w[32];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          w[4 * k] = __uint_as_float(v[k].x);
          w[4 * k + 1] = __uint_as_float(v[k].y);
          w[4 * k + 2] = __uint_as_float(v[k].z);
          w[4 * k + 3] = __uint_as_float(v[k].w);
        }
        sm100::tmem_st32(lanes + Sh::Q_COLUMN + c / 2, w);
      }
      sm100::tmem_wait_st();
    } else {
      constexpr int EACH = QUERIES * D / 8 / 64;  // 16-byte words of a thread
#pragma unroll
      for (int k0 = 0; k0 < EACH; k0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int i = (k0 + k) * 64 + tid, m = i / (D / 8), c = i % (D / 8), r = m / a.per_kv;
          v[k] = make_uint4(0, 0, 0, 0);
          if (k0 + k < EACH && r < rows) {
            const bf16* x = a.q + (row0 + r) * a.q_row + (long)(kv * a.per_kv + m % a.per_kv) * a.q_head + c * 8;
            if (a.q_vec) {
              v[k] = *reinterpret_cast<const uint4*>(x);
            } else {
              bf16* e = reinterpret_cast<bf16*>(&v[k]);
#pragma unroll
              for (int j = 0; j < 8; ++j) e[j] = x[j];
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int i = (k0 + k) * 64 + tid, m = i / (D / 8), c = i % (D / 8);
          if (k0 + k < EACH) *reinterpret_cast<uint4*>(sQ + (c >> 3) * BOX + m * 128 + (((c & 7) ^ (m & 7)) << 4)) = v[k];
        }
      }
      fence_proxy_async();
    }
    sm100::tc_fence_before();
    sm100::mbar_arrive(q_full);
    {  // products add to O from the first on (the first product waits for these threads' first weights)
      float zero[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) zero[i] = 0.f;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) sm100::tmem_st32(lanes + c, zero);
      sm100::tmem_wait_st();
    }
    float m = -INFINITY, l = 0.f;
    int u = 0;
    bool bad = false;
    for (;; ++u) {
      const int st = u & 1;
      if (__any_sync(~0u, !sm100::mbar_wait(&known[u % UNITS], (u / UNITS) & 1, abort))) bad = true;
      const Unit unit = units[u % UNITS];
      if (bad || unit.members == 0) break;
      bad = __any_sync(~0u, !sm100::mbar_wait(&s_full[st], (u >> 1) & 1, abort));
      if (bad) break;
      const bool member = used && (unit.members >> row & 1), partial = unit.valid < TILE || unit.there != 15u;
      float s[2][32];
      sm100::tc_fence_after();
      sm100::tmem_ld32(lanes + Sh::S + st * TILE, s[0]);
      sm100::tmem_ld32(lanes + Sh::S + st * TILE + 32, s[1]);
      sm100::tmem_wait_ld();
      if (partial) {
#pragma unroll
        for (int i = 0; i < TILE; ++i)
          if (i >= unit.valid || !(unit.there >> (i / 16) & 1)) s[i / 32][i % 32] = -INFINITY;
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < TILE; ++i) {
        s[i / 32][i % 32] *= a.scale_log2;
        top[i & 3] = fmaxf(top[i & 3], s[i / 32][i % 32]);
      }
      const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      // a score far above the reference, or the first: the maximum is the reference from now on
      const bool higher = member && !(most - m <= HEADROOM);
      if (__any_sync(~0u, higher)) {
        const float keep = higher && most > m ? ex2(m - most) : 1.f;  // (m of -inf: sums and outputs are 0 so far)
        if (higher && most > m) {
          m = most;
          l *= keep;
        }
        if (u > 0) {  // O must hold what came before it is rescaled
          bad = __any_sync(~0u, !sm100::mbar_wait(&o_done[(u - 1) & 1], ((u - 1) >> 1) & 1, abort));
          if (!bad && __any_sync(~0u, keep != 1.f)) {
            sm100::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              float o[32];
              sm100::tmem_ld32(lanes + c, o);
              sm100::tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= keep;
              sm100::tmem_st32(lanes + c, o);
            }
            sm100::tmem_wait_st();
          }
        }
      }
      if (partial) {  // values that nobody sees
        const int entry = 2 * u + 1, slot = entry % RING;
        bad |= __any_sync(~0u, !sm100::mbar_wait(&full[slot], (entry / RING) & 1, abort));
        for (int i = tid; i < TILE * D / 8; i += QUERIES) {  // boxes of 64 rows of 8 words
          const int r = i / 8 % TILE;
          if (r >= unit.valid || !(unit.there >> (r / 16) & 1))
            *reinterpret_cast<uint4*>(sKV + slot * HALF + i * 16) = make_uint4(0, 0, 0, 0);
        }
      }
      if (bad) break;
      const float base = m == -INFINITY ? 0.f : m;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      float w[32];  // two weights each (rows that do not hold the page: of no consequence)
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float x = ex2(s[i / 16][i % 16 * 2] - base), y = ex2(s[i / 16][i % 16 * 2 + 1] - base);
        sum[i & 3] += x + y;
        w[i] = __uint_as_float(pack(x, y));
      }
      if (member) l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      sm100::tmem_st32(lanes + Sh::S + st * TILE, w);
      sm100::tmem_wait_st();
      if (partial) fence_proxy_async();
      sm100::tc_fence_before();
      sm100::mbar_arrive(&p_full[st]);
    }
    // ---- result: u units were seen (bad: it is none)
    if (u > 0 && !bad) bad = __any_sync(~0u, !sm100::mbar_wait(&o_done[(u - 1) & 1], ((u - 1) >> 1) & 1, abort));
    sm100::tc_fence_after();
    const long at = ((long)(row0 + row) * a.heads + kv * a.per_kv + h) * a.splits + split;
    if (used) a.stats[at] = make_float2(m, bad ? NAN : l);
    // rows through shared memory (16 bytes apart beyond their size), one copy each; the ring has had its use
    float* line = reinterpret_cast<float*>(sKV) + n * (D + 4);
#pragma unroll 1
    for (int c = 0; c < D && !bad; c += 32) {
      float o[32];
      sm100::tmem_ld32(lanes + c, o);
      sm100::tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; i += 4)
        *reinterpret_cast<float4*>(line + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
    }
    fence_proxy_async();
    if (used && !bad) {
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(a.sums + at * D),
                   "r"(sm100::smem_u32(line)), "r"(D * 4)
                   : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 3) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, Sh::COLUMNS);
  }
}

// Four components of a result: normalised, gated, rounded.
__device__ __forceinline__ void finish(const AttendArgs& a, long rh, int D, int c, float4 o, float l,
                                       const float (&gate)[4]) {
  const float scale = l == 0.f ? 0.f : 1.f / l;  // nothing seen: zeros
  float v[4] = {o.x * scale, o.y * scale, o.z * scale, o.w * scale};
  if (a.gate)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= rt::sigmoidf_(gate[j]);
  __nv_bfloat162 r[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
  *reinterpret_cast<uint2*>(a.out + rh * D + c) = *reinterpret_cast<const uint2*>(r);
}

// Up to FEW splits: a thread per four components of a (row, query head), several of them per block, no barrier (1536 of
// them with two splits: 15 us by the kernel below, one block each).
constexpr int FEW = 8;
__global__ void __launch_bounds__(256) join_few_kernel(const AttendArgs a, int D, long items) {
  const int wide = D / 4;
  const long rh = (long)blockIdx.x * (256 / wide) + threadIdx.x / wide;
  if (rh >= items) return;
  const int c = threadIdx.x % wide * 4, head = rh % a.heads, row = rh / a.heads;
  float gate[4] = {0.f, 0.f, 0.f, 0.f};
  if (a.gate)
#pragma unroll
    for (int j = 0; j < 4; ++j) gate[j] = rt::to_f(a.gate[row * a.gate_row + head * a.gate_head + c + j]);
  float4 x[FEW];
  float2 st[FEW];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < FEW; ++i) {
    const bool on = i < a.splits;
    st[i] = on ? a.stats[rh * a.splits + i] : make_float2(-INFINITY, 0.f);
    x[i] = on ? *reinterpret_cast<const float4*>(a.sums + (rh * a.splits + i) * D + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    m = fmaxf(m, st[i].x);
  }
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < FEW; ++i) {
    // (a split that saw nothing has the sum 0 and the reference -inf)
    const float w = st[i].y == 0.f ? 0.f : st[i].x == m ? 1.f : ex2(st[i].x - m);
    l += w * st[i].y;
    o.x += w * x[i].x;
    o.y += w * x[i].y;
    o.z += w * x[i].z;
    o.w += w * x[i].w;
  }
  finish(a, rh, D, c, o, l, gate);
}

// Block of 256 threads per (row, query head), a thread per four components of every (1024 / dim)-th split. Everything is
// loaded at once: each warp forms the splits' weights for itself, so that one barrier is left, before the threads' sums
// are added.
__global__ void __launch_bounds__(256) join_kernel(const AttendArgs a, int D) {
  constexpr int EACH = (MAX_SPLITS + 31) / 32, AHEAD = 10;
  __shared__ float weights[8][MAX_SPLITS];
  __shared__ float4 parts[256];
  const long rh = blockIdx.x;
  const int head = rh % a.heads, row = rh / a.heads, tid = threadIdx.x, lane = tid & 31, wide = D / 4;
  const int c = tid % wide, first = tid / wide, step = 256 / wide;
  const float4* sums = reinterpret_cast<const float4*>(a.sums) + rh * a.splits * wide + c;
  float4 x[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    x[k] = first + k * step < a.splits ? sums[(long)(first + k * step) * wide] : make_float4(0.f, 0.f, 0.f, 0.f);
  float gate[4] = {0.f, 0.f, 0.f, 0.f};
  if (a.gate && tid < wide)
#pragma unroll
    for (int j = 0; j < 4; ++j) gate[j] = rt::to_f(a.gate[row * a.gate_row + head * a.gate_head + tid * 4 + j]);
  float2 st[EACH];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int i = j * 32 + lane;
    st[j] = i < a.splits ? a.stats[rh * a.splits + i] : make_float2(-INFINITY, 0.f);
    m = fmaxf(m, st[j].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  float* weight = weights[tid >> 5];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const float w = st[j].y == 0.f ? 0.f : st[j].x == m ? 1.f : ex2(st[j].x - m);
    if (j * 32 + lane < a.splits) weight[j * 32 + lane] = w;
    l += w * st[j].y;
  }
  l = rt::warp_sum(l);
  __syncwarp();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](int i, const float4& v) {
    const float w = weight[i];
    o.x += w * v.x;
    o.y += w * v.y;
    o.z += w * v.z;
    o.w += w * v.w;
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (first + k * step < a.splits) add(first + k * step, x[k]);
  for (int i = first + AHEAD * step; i < a.splits; i += step) add(i, sums[(long)i * wide]);
  parts[tid] = o;
  __syncthreads();
  if (tid >= wide) return;
  for (int i = 1; i < step; ++i) {
    const float4 v = parts[i * wide + tid];
    o.x += v.x;
    o.y += v.y;
    o.z += v.z;
    o.w += v.w;
  }
  finish(a, rh, D, tid * 4, o, l, gate);
}

// How a call is cut: rows of a group that fit a block's queries (and a lane each) together, evenly; splits of the keys
// so that the blocks fill the SMs once, but no finer than the cache's tiles.
struct Plan {
  int together, subgroups, splits;
};
Plan plan_for(const RtPool* p, int heads, int group) {
  Plan x;
  const int most = std::min(32, QUERIES / (heads / p->heads));
  x.subgroups = (group + most - 1) / most;
  x.together = (group + x.subgroups - 1) / x.subgroups;
  x.subgroups = (group + x.together - 1) / x.together;
  const long blocks = (long)(p->rows / group) * x.subgroups * p->heads;
  const long tiles = ((long)p->width * p->page + TILE - 1) / TILE;
  x.splits = (int)std::max(1L, std::min({tiles, (p->dim == 256 ? 148 : 296) / blocks, (long)MAX_SPLITS}));
  return x;
}

template <int D>
cudaError_t launch(const CUtensorMap& map, const AttendArgs& a, const Plan& x, cudaStream_t s) {
  constexpr int bytes = Shape<D>::BYTES;
  static_assert(bytes <= (D == 256 ? 227 : 113) * 1024, "shared memory of a block");
  // The limit belongs to the device and not to the call, so it is raised once.
  static std::atomic<uint64_t> set{0};  // devices
  int dev = 0;
  RT_CUDA_CHECK(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!bit || !(set.load(std::memory_order_acquire) & bit)) {
    RT_CUDA_CHECK(cudaFuncSetAttribute(attend_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    set.fetch_or(bit, std::memory_order_acq_rel);
  }
  const dim3 grid((unsigned)x.splits, (unsigned)a.kv_heads, (unsigned)(a.rows / a.group * x.subgroups));
  attend_kernel<D><<<grid, THREADS, bytes, s>>>(map, a);
  return cudaGetLastError();
}

}  // namespace

extern "C" long rt_paged_attention_workspace_floats(const RtPool* p, int heads, int group) {
  return (long)p->rows * heads * plan_for(p, heads, group).splits * (p->dim + 2);
}

// q [rows, heads, dim] and gate (or null) with strides in elements, unit inner stride; out contiguous; work:
// rt_paged_attention_workspace_floats, 16-byte aligned. Results are NaN if a bounded wait gave up.
extern "C" cudaError_t rt_paged_attention(const RtPool* p, int block, const int* table, const int* lengths,
                                          const void* q, long q_row, long q_head, int heads, const void* gate,
                                          long gate_row, long gate_head, int group, void* out, float* work,
                                          cudaStream_t s) {
  if (block < 0 || block >= p->blocks || heads < 1 || heads % p->heads || heads > QUERIES * p->heads || group < 1 ||
      p->rows < 1 || p->rows % group || p->heads > 65535 || (p->page != 16 && p->page != 32 && p->page != 64) ||
      (long)p->width * p->page > INT_MAX - TILE || reinterpret_cast<uintptr_t>(p->pool) % 16)
    return cudaErrorInvalidValue;
  const long panels = (long)p->blocks * 2 * p->heads, lines = p->pages * panels * p->page;
  if (lines > INT_MAX) return cudaErrorInvalidValue;
  const Plan x = plan_for(p, heads, group);
  AttendArgs a{};
  a.pages = p->pages;
  a.panels = (int)panels;
  a.first = block * 2 * p->heads;
  a.kv_heads = p->heads;
  a.page = p->page;
  a.width = p->width;
  a.splits = x.splits;
  a.rows = p->rows;
  a.group = group;
  a.together = x.together;
  a.subgroups = x.subgroups;
  a.heads = heads;
  a.per_kv = heads / p->heads;
  a.table = table;
  a.lengths = lengths;
  a.q = static_cast<const bf16*>(q);
  a.q_row = q_row;
  a.q_head = q_head;
  a.q_vec = (reinterpret_cast<uintptr_t>(q) | (uintptr_t)(q_row * 2) | (uintptr_t)(q_head * 2)) % 16 == 0;
  a.gate = static_cast<const bf16*>(gate);
  a.gate_row = gate_row;
  a.gate_head = gate_head;
  a.scale_log2 = 1.4426950408889634f / sqrtf((float)p->dim);
  a.out = static_cast<bf16*>(out);
  a.sums = work;
  a.stats = reinterpret_cast<float2*>(work + (long)p->rows * heads * x.splits * p->dim);
  // the pool as rows of one token's key or value in one head; a box is a page's rows of 64 components
  CUtensorMap map;
  const uint64_t dims[2] = {(uint64_t)p->dim, (uint64_t)lines}, strides[1] = {(uint64_t)p->dim * 2};
  const uint32_t box[2] = {64, (uint32_t)p->page};
  if (!tmap::encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p->pool, dims, strides, box)) return cudaErrorInvalidValue;
  if (p->dim == 64) RT_CUDA_CHECK(launch<64>(map, a, x, s));
  else if (p->dim == 128) RT_CUDA_CHECK(launch<128>(map, a, x, s));
  else if (p->dim == 256) RT_CUDA_CHECK(launch<256>(map, a, x, s));
  else return cudaErrorInvalidValue;
  const long items = (long)p->rows * heads, together = 1024 / p->dim;
  if (x.splits <= FEW) join_few_kernel<<<(unsigned)((items + together - 1) / together), 256, 0, s>>>(a, p->dim, items);
  else join_kernel<<<(unsigned)items, 256, 0, s>>>(a, p->dim);
  return cudaGetLastError();
}
