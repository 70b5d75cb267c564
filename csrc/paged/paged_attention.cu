// Attention of one token per row over the pages of a cache (paged.py has the definition).
//
// Bound by memory: every page that a row or its group's other beams hold has to be read once. So a block takes the
// rows of a group together (one key head, every splits-th tile of 64 keys): of each tile it loads the pages that
// differ between the rows, and each of them meets the queries of all rows that hold it. Roles:
//   warp 8      finds the tile's distinct pages (a lane per row) and brings their keys and values in with TMA (128-byte
//               swizzle, boxes of 64 components) into a ring of tiles;
//   warps 0-3, 4-7   two groups, which take the ring's units (a tile of keys and of values) in turn, each with its own
//               running maximum, sum and output, so that one group's barriers hide behind the other's products.
// The products are transposed: S^T = K Q^T has the keys as the 16 rows of a matrix instruction and the (up to 8) query
// heads of one row as its 8 columns, so a tile in registers serves all rows that hold its page and rows that do not
// cost nothing; O^T = V^T P^T likewise, V^T by transposing loads. A warp forms the scores of 16 keys for all queries and
// the outputs of a quarter of the components; P goes through shared memory in bf16 (2^-8 of each weight at most, the
// rounding that the operands of the product need), sums and outputs stay fp32. At 8 queries these are mma.sync's
// shapes: with 128 rows of queries a tcgen05 tile would be padded 16-fold, and its transposed form would need P in the
// swizzled layout and the outputs rescaled in TMEM, for products that take half of the time that the loads take.
//
// Keys that a row does not see (behind its last token, or in a missing page) get the weight 0 whatever they hold:
// their scores are replaced, their values zeroed in shared memory.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cuda.h>
#include "../api.h"
#include "../common/common.cuh"
#include "../common/sm100.cuh"
#include "../common/tmap.cuh"

namespace {

using bf16 = __nv_bfloat16;
constexpr int TILE = 64, MAX_TILES = 8;  // keys of a unit; 8-query tiles of a block
constexpr int MAX_SPLITS = 148;

struct AttendArgs {
  int pages, panels, first, kv_heads, page, width, splits;
  int rows, group, together, subgroups;  // rows of a block at most, blocks per group of beams
  int heads, per_kv, tiles_per_row;
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
  float2* stats;   // [rows, heads, splits]: maximum, sum of exponentials
};

template <int D> struct Shape {
  static constexpr int HALF = TILE * D * 2;                    // bytes of a tile of keys or of values
  static constexpr int SLOTS = D == 256 ? 5 : D == 128 ? 6 : 8;
  static constexpr int MTILES = D / 64;                        // of 16 components per warp
};
// Eight tiles of queries need more registers than an even split gives (168): there the loading warp's warpgroup is
// whole and hands some of its registers over, 4 x 40 + 8 x 232 of the 12 x 168 that the block has.
constexpr int threads(int NT) { return NT == 8 ? 384 : 288; }
constexpr int GIVEN = 40, TAKEN = 232;
static_assert(4 * GIVEN + 8 * TAKEN <= 12 * 168, "registers handed over");
template <int D, int NT> constexpr int smem_bytes() {
  return Shape<D>::SLOTS * Shape<D>::HALF + NT * 8 * D * 2 + 2 * NT * 8 * TILE * 2 + 2 * 4 * NT * 8 * 4 +
         Shape<D>::SLOTS * 32 + 64 + 1024;
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void stsm2_t(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1,%2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Barrier of a group of 128 threads.
__device__ __forceinline__ void group_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void both_sync() { asm volatile("bar.sync 3, 256;" ::: "memory"); }
// A group's, and whether any of them says so.
__device__ __forceinline__ bool group_any(int id, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "bar.red.or.pred q, %1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)v)
      : "memory");
  return r != 0;
}

// A unit of the ring, in the slot of its keys.
struct Unit {
  uint32_t tiles;  // of queries that hold its page; 0: no more units
  int valid;       // keys before the rows' end
  uint32_t there;  // 16-key blocks whose page exists
};

// Grid (splits, key heads, groups x subgroups). NT: 8-query tiles.
template <int D, int NT>
__global__ void __launch_bounds__(threads(NT), 1) attend_kernel(const __grid_constant__ CUtensorMap map, const AttendArgs a) {
  constexpr int THREADS = threads(NT);
  constexpr int SLOTS = Shape<D>::SLOTS, HALF = Shape<D>::HALF, MT = Shape<D>::MTILES, BOXES = D / 64;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = sm100::align_smem_1024(raw);
  uint8_t* sQ = smem + SLOTS * HALF;                                   // [NT * 8][D], 16-byte chunks swizzled by row
  uint8_t* sP = sQ + NT * 8 * D * 2;                                   // per group [NT * 8][64 keys], likewise
  float* sMax = reinterpret_cast<float*>(sP + 2 * NT * 8 * TILE * 2);  // per group [4 warps][NT * 8]
  Unit* units = reinterpret_cast<Unit*>(sMax + 2 * 4 * NT * 8);        // [SLOTS]
  uint64_t* full = reinterpret_cast<uint64_t*>(units + SLOTS + (SLOTS & 1));
  uint64_t* empty = full + SLOTS;
  volatile int* abort = reinterpret_cast<volatile int*>(empty + SLOTS);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x, kv = blockIdx.y, g = blockIdx.z / a.subgroups, sub = blockIdx.z % a.subgroups;
  const int row0 = g * a.group + sub * a.together, rows = min(a.together, a.group - sub * a.together);
  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      sm100::mbar_init(&full[i], 1);
      sm100::mbar_init(&empty[i], 4);
    }
    *abort = 0;
    sm100::fence_barrier_init();
  }
  // queries: row r's head h is query r * tiles_per_row * 8 + h; the others are zero
  const int row_queries = a.tiles_per_row * 8;
  for (int i = tid; i < NT * 8 * (D / 8); i += THREADS) {
    const int n = i / (D / 8), c = i % (D / 8), r = n / row_queries, h = n % row_queries;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < rows && h < a.per_kv) {
      const bf16* x = a.q + (row0 + r) * a.q_row + (long)(kv * a.per_kv + h) * a.q_head + c * 8;
      if (a.q_vec) {
        v = *reinterpret_cast<const uint4*>(x);
      } else {
        bf16* e = reinterpret_cast<bf16*>(&v);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = x[j];
      }
    }
    *reinterpret_cast<uint4*>(sQ + n * D * 2 + ((c ^ (n & 7)) << 4)) = v;
  }
  __syncthreads();

  if (warp >= 8) {
    if (NT == 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(GIVEN));
    if (warp > 8) return;
    // ------------------------------------------------------------ producer
    const int capacity = a.width * a.page, span = TILE / a.page;  // pages of a tile
    const int length = lane < rows ? min(max(a.lengths[row0 + lane], 0), capacity) : 0;
    const int longest = __reduce_max_sync(~0u, length);
    const int* table = a.table + (long)(row0 + (lane < rows ? lane : 0)) * a.width;
    const int count = (longest + TILE - 1) / TILE;
    auto entries = [&](int i, int (&e)[4]) {  // this row's pages of a tile, -1: none
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e[j] = -1;
        if (j < span && i < count && i * TILE + j * a.page < length) {
          const int p = table[i * span + j];
          if (p >= 0 && p < a.pages) e[j] = p;
        }
      }
    };
    if (lane == 0) sm100::prefetch_tmap(&map);
    int next[4], entry = 0;
    entries(split, next);
    bool ok = true;
    auto wait_empty = [&](int slot) {
      if (entry >= SLOTS && !sm100::mbar_wait(&empty[slot], (entry / SLOTS - 1) & 1, abort)) ok = false;
      ok = __all_sync(~0u, ok);
    };
    for (int i = split; i < count && ok; i += a.splits) {
      int e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = next[j];
      entries(i + a.splits, next);
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
        const unsigned members = __shfl_sync(~0u, same, leader);
        left &= ~members;
        Unit u;
        u.valid = __shfl_sync(~0u, valid, leader);
        u.there = __shfl_sync(~0u, there, leader);
        u.tiles = 0;
        for (unsigned r = members; r; r &= r - 1)
          u.tiles |= ((1u << a.tiles_per_row) - 1) << ((__ffs(r) - 1) * a.tiles_per_row);
        int p[4], here = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[j] = __shfl_sync(~0u, e[j], leader);
          here += p[j] >= 0;
        }
        for (int kind = 0; kind < 2 && ok; ++kind, ++entry) {
          const int slot = entry % SLOTS;
          wait_empty(slot);
          if (!ok) break;
          if (lane == 0) {
            if (kind == 0) units[slot] = u;
            sm100::mbar_expect_tx(&full[slot], here * a.page * D * 2);
          }
          __syncwarp();
          const int j = lane / BOXES, box = lane % BOXES;  // a copy per lane
          const int page = j == 0 ? p[0] : j == 1 ? p[1] : j == 2 ? p[2] : p[3];
          if (j < span && page >= 0) {
            const int y = (page * a.panels + a.first + kind * a.kv_heads + kv) * a.page;
            sm100::tma_load_2d(smem + slot * HALF + box * (TILE * 128) + j * a.page * 128, &map, &full[slot], box * 64, y);
          }
          __syncwarp();
        }
      }
    }
    // both groups' ends
    for (int i = 0; i < 2 && ok; ++i) {
      const int slot = entry % SLOTS;
      wait_empty(slot);
      if (ok && lane == 0) {
        units[slot].tiles = 0;
        sm100::mbar_arrive(&full[slot]);
      }
      entry += 2;
    }
    if (!ok)  // copies in flight have to land before the block ends
      for (int i = max(entry - SLOTS, 0); i < entry; ++i) sm100::mbar_wait_bounded(&full[i % SLOTS], (i / SLOTS) & 1);
    return;
  }

  // -------------------------------------------------------------- groups
  if (NT == 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TAKEN));
  const int grp = warp >> 2, w = warp & 3;
  float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int t = 0; t < MT; ++t) o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.f;
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
  }
  {
    const uint32_t q_base = sm100::smem_u32(sQ), p_base = sm100::smem_u32(sP) + grp * NT * 8 * TILE * 2;
    float* top = sMax + grp * 4 * NT * 8;
    const int bar = 1 + grp, t2 = 2 * (lane & 3);
    for (int u = grp;; u += 2) {
      const int ke = 2 * u, ks = ke % SLOTS, vs = (ke + 1) % SLOTS;
      // what ends the loop is agreed on at the group's first barrier, whichever thread's wait gives up
      bool bad = __any_sync(~0u, !sm100::mbar_wait(&full[ks], (ke / SLOTS) & 1, abort));
      const Unit unit = units[ks];
      const bool done = bad || unit.tiles == 0;
      const uint32_t k_base = sm100::smem_u32(smem) + ks * HALF, v_base = sm100::smem_u32(smem) + vs * HALF;
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      if (!done) {
        const int r = w * 16 + (lane & 15);
        const uint32_t row = k_base + r * 128;
#pragma unroll 4
        for (int kk = 0; kk < D / 32; ++kk) {
          uint32_t a0[4], a1[4];
          const uint32_t box = row + (kk >> 1) * (TILE * 128);
          const int c = (kk & 1) * 4 + (lane >> 4);
          ldsm4(a0, box + ((c ^ (r & 7)) << 4));
          ldsm4(a1, box + (((c + 2) ^ (r & 7)) << 4));
#pragma unroll
          for (int n = 0; n < NT; ++n)
            if (unit.tiles >> n & 1) {
              uint32_t b[4];
              const int x = lane & 7;
              ldsm4(b, q_base + (n * 8 + x) * D * 2 + (((kk * 4 + (lane >> 3)) ^ x) << 4));
              mma(s[n], a0, b[0], b[1]);
              mma(s[n], a1, b[2], b[3]);
            }
        }
      }
      if (!done) {
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&empty[ks]);
        // keys lane / 4 and lane / 4 + 8 of this warp's 16, queries t2 and t2 + 1 of each tile
        const int key = w * 16 + (lane >> 2);
        const bool block = unit.there >> w & 1, see0 = block && key < unit.valid, see1 = block && key + 8 < unit.valid;
#pragma unroll
        for (int n = 0; n < NT; ++n)
          if (unit.tiles >> n & 1) {
            if (!see0) s[n][0] = s[n][1] = -INFINITY;
            if (!see1) s[n][2] = s[n][3] = -INFINITY;
            float x = fmaxf(s[n][0], s[n][2]), y = fmaxf(s[n][1], s[n][3]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
              x = fmaxf(x, __shfl_xor_sync(~0u, x, off));
              y = fmaxf(y, __shfl_xor_sync(~0u, y, off));
            }
            if (lane < 4) *reinterpret_cast<float2*>(top + w * NT * 8 + n * 8 + t2) = make_float2(x, y);
          }
        bad = !sm100::mbar_wait(&full[vs], ((ke + 1) / SLOTS) & 1, abort);
      }
      if (group_any(bar, done || bad)) break;
      const bool partial = unit.valid < TILE || unit.there != 15u;
      if (partial) {
        const int t = tid & 127;
        for (int i = t; i < TILE * D / 8; i += 128) {  // boxes of 64 rows of 8 chunks
          const int r = i / 8 % TILE;
          if (r >= unit.valid || !(unit.there >> (r / 16) & 1))
            *reinterpret_cast<uint4*>(smem + vs * HALF + i * 16) = make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (unit.tiles >> n & 1) {
          float2 mx = make_float2(m[n][0], m[n][1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 x = *reinterpret_cast<const float2*>(top + i * NT * 8 + n * 8 + t2);
            mx.x = fmaxf(mx.x, x.x);
            mx.y = fmaxf(mx.y, x.y);
          }
          // (relative to 0 while nothing is seen: every weight is 0 then)
          const float bx = mx.x == -INFINITY ? 0.f : mx.x, by = mx.y == -INFINITY ? 0.f : mx.y;
          const float kx = ex2((m[n][0] - bx) * a.scale_log2), ky = ex2((m[n][1] - by) * a.scale_log2);
          m[n][0] = mx.x;
          m[n][1] = mx.y;
          s[n][0] = ex2((s[n][0] - bx) * a.scale_log2);
          s[n][1] = ex2((s[n][1] - by) * a.scale_log2);
          s[n][2] = ex2((s[n][2] - bx) * a.scale_log2);
          s[n][3] = ex2((s[n][3] - by) * a.scale_log2);
          l[n][0] = l[n][0] * kx + (s[n][0] + s[n][2]);
          l[n][1] = l[n][1] * ky + (s[n][1] + s[n][3]);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            o[n][t][0] *= kx;
            o[n][t][1] *= ky;
            o[n][t][2] *= kx;
            o[n][t][3] *= ky;
          }
          // transposed: row = query, column = key
          const int x = lane & 7;
          stsm2_t(p_base + (n * 8 + x) * TILE * 2 + (((w * 2 + ((lane >> 3) & 1)) ^ x) << 4), pack(s[n][0], s[n][1]),
                  pack(s[n][2], s[n][3]));
        }
      group_sync(bar);
#pragma unroll
      for (int kp = 0; kp < 2; ++kp) {
        uint32_t v[2][MT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const int d = w * (D / 4) + t * 16, r = (kp * 2 + h) * 16 + (lane & 7) + (lane >> 4) * 8;
            const int c = (d & 63) / 8 + ((lane >> 3) & 1);
            ldsm4_t(v[h][t], v_base + (d >> 6) * (TILE * 128) + r * 128 + ((c ^ (r & 7)) << 4));
          }
#pragma unroll
        for (int n = 0; n < NT; ++n)
          if (unit.tiles >> n & 1) {
            uint32_t b[4];
            const int x = lane & 7;
            ldsm4(b, p_base + (n * 8 + x) * TILE * 2 + (((kp * 4 + (lane >> 3)) ^ x) << 4));
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              mma(o[n][t], v[0][t], b[0], b[1]);
              mma(o[n][t], v[1][t], b[2], b[3]);
            }
          }
      }
      if (partial) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // zeros, then the next copy
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&empty[vs]);
    }
  }
  both_sync();
  if (*abort)
#pragma unroll
    for (int n = 0; n < NT; ++n) l[n][0] = l[n][1] = NAN;  // a wait that gave up: no result

  // ---- the groups' results joined: the second's through shared memory, sums over the warps' keys
  float* out1 = reinterpret_cast<float*>(smem);                   // [NT * 8][D] of the second group
  float2* ml = reinterpret_cast<float2*>(smem + NT * 8 * D * 4);  // [2 groups][4 warps][NT * 8]: maximum, sum
  {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = l[n][j];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) x += __shfl_xor_sync(~0u, x, off);
        if (lane < 4) ml[(grp * 4 + w) * NT * 8 + n * 8 + 2 * lane + j] = make_float2(m[n][j], x);
      }
    }
    if (grp == 1)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = w * (D / 4) + t * 16 + (lane >> 2) + (i >> 1) * 8, q = n * 8 + 2 * (lane & 3) + (i & 1);
            out1[q * D + d] = o[n][t][i];
          }
  }
  both_sync();
  if (grp == 1) return;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int q = n * 8 + 2 * (lane & 3) + j, r = q / row_queries, h = q % row_queries;
      if (r >= rows || h >= a.per_kv) continue;
      const float m0 = ml[q].x, m1 = ml[4 * NT * 8 + q].x, mx = fmaxf(m0, m1), base = mx == -INFINITY ? 0.f : mx;
      const float w0 = ex2((m0 - base) * a.scale_log2), w1 = ex2((m1 - base) * a.scale_log2);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += w0 * ml[i * NT * 8 + q].y + w1 * ml[(4 + i) * NT * 8 + q].y;
      const long at = ((long)(row0 + r) * a.heads + kv * a.per_kv + h) * a.splits + split;
      if (w == 0 && (lane >> 2) == 0) a.stats[at] = make_float2(mx, sum);
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int d = w * (D / 4) + t * 16 + (lane >> 2) + i * 8;
          a.sums[at * D + d] = w0 * o[n][t][2 * i + j] + w1 * out1[q * D + d];
        }
    }
}

// Block per (row, query head), a thread per component.
__global__ void join_kernel(const AttendArgs a, int D) {
  const long rh = blockIdx.x;
  const int head = rh % a.heads, row = rh / a.heads, c = threadIdx.x;
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int i = 0; i < a.splits; ++i) m = fmaxf(m, a.stats[rh * a.splits + i].x);
  for (int i = 0; i < a.splits; ++i) {
    const float2 st = a.stats[rh * a.splits + i];
    if (st.y == 0.f) continue;
    const float w = st.x == m ? 1.f : ex2((st.x - m) * a.scale_log2);
    l += w * st.y;
    o += w * a.sums[(rh * a.splits + i) * D + c];
  }
  o = l == 0.f ? 0.f : o / l;
  if (a.gate) o *= rt::sigmoidf_(rt::to_f(a.gate[row * a.gate_row + head * a.gate_head + c]));
  a.out[rh * D + c] = __float2bfloat16_rn(o);
}

// How a call is cut: rows of a group that fit a block's query tiles together, evenly; splits of the keys so that the
// blocks fill the SMs once (one block each), but no finer than the cache's tiles.
struct Plan {
  int tiles_per_row, together, subgroups, splits;
};
Plan plan_for(const RtPool* p, int heads, int group) {
  Plan x;
  x.tiles_per_row = (heads / p->heads + 7) / 8;
  const int most = std::max(1, MAX_TILES / x.tiles_per_row);
  x.subgroups = (group + most - 1) / most;
  x.together = (group + x.subgroups - 1) / x.subgroups;
  x.subgroups = (group + x.together - 1) / x.together;
  const long blocks = (long)(p->rows / group) * x.subgroups * p->heads;
  const long tiles = ((long)p->width * p->page + TILE - 1) / TILE;
  x.splits = (int)std::max(1L, std::min({tiles, 148 / blocks, (long)MAX_SPLITS}));
  return x;
}

template <int D, int NT>
cudaError_t launch(const CUtensorMap& map, const AttendArgs& a, const Plan& x, cudaStream_t s) {
  constexpr int bytes = smem_bytes<D, NT>();
  static_assert(bytes <= 227 * 1024, "shared memory of a block");
  static_assert(NT * 8 * D * 4 + 8 * NT * 8 * 8 <= Shape<D>::SLOTS * Shape<D>::HALF, "the join fits the ring");
  // The limit belongs to the device and not to the call, so it is raised once.
  static std::atomic<uint64_t> set{0};  // devices
  int dev = 0;
  RT_CUDA_CHECK(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!bit || !(set.load(std::memory_order_acquire) & bit)) {
    RT_CUDA_CHECK(cudaFuncSetAttribute(attend_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    set.fetch_or(bit, std::memory_order_acq_rel);
  }
  const dim3 grid((unsigned)x.splits, (unsigned)a.kv_heads, (unsigned)(a.rows / a.group * x.subgroups));
  attend_kernel<D, NT><<<grid, threads(NT), bytes, s>>>(map, a);
  return cudaGetLastError();
}
template <int D>
cudaError_t launch(const CUtensorMap& map, const AttendArgs& a, const Plan& x, cudaStream_t s) {
  const int tiles = x.together * x.tiles_per_row;
  if (tiles <= 1) return launch<D, 1>(map, a, x, s);
  if (tiles <= 2) return launch<D, 2>(map, a, x, s);
  if (tiles <= 4) return launch<D, 4>(map, a, x, s);
  return launch<D, 8>(map, a, x, s);
}

}  // namespace

extern "C" long rt_paged_attention_workspace_floats(const RtPool* p, int heads, int group) {
  return (long)p->rows * heads * plan_for(p, heads, group).splits * (p->dim + 2);
}

// q [rows, heads, dim] and gate (or null) with strides in elements, unit inner stride; out contiguous; work:
// rt_paged_attention_workspace_floats, 8-byte aligned. Results are NaN if a bounded wait gave up.
extern "C" cudaError_t rt_paged_attention(const RtPool* p, int block, const int* table, const int* lengths,
                                          const void* q, long q_row, long q_head, int heads, const void* gate,
                                          long gate_row, long gate_head, int group, void* out, float* work,
                                          cudaStream_t s) {
  if (block < 0 || block >= p->blocks || heads < 1 || heads % p->heads || heads > 64 * p->heads || group < 1 ||
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
  a.tiles_per_row = x.tiles_per_row;
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
  a.stats = reinterpret_cast<float2*>(work);
  a.sums = work + 2L * p->rows * heads * x.splits;
  // the pool as rows of one token's key or value in one head; a box is a page's rows of 64 components
  CUtensorMap map;
  const uint64_t dims[2] = {(uint64_t)p->dim, (uint64_t)lines}, strides[1] = {(uint64_t)p->dim * 2};
  const uint32_t box[2] = {64, (uint32_t)p->page};
  if (!tmap::encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p->pool, dims, strides, box)) return cudaErrorInvalidValue;
  if (p->dim == 64) RT_CUDA_CHECK(launch<64>(map, a, x, s));
  else if (p->dim == 128) RT_CUDA_CHECK(launch<128>(map, a, x, s));
  else if (p->dim == 256) RT_CUDA_CHECK(launch<256>(map, a, x, s));
  else return cudaErrorInvalidValue;
  join_kernel<<<(unsigned)(p->rows * heads), p->dim, 0, s>>>(a, p->dim);
  return cudaGetLastError();
}
