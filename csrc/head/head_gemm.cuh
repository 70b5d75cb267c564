// The three matrix products of the vocabulary-head losses on CTA pairs: tiles of 256 x 256 (256 x NT for few rows),
// fp32 accumulators in TMEM, one persistent kernel each.
//
//   LOGITS  z = X . W^T              X [n, C] live rows, W [V, C]; z stays on chip: per row and tile the epilogue
//                                    leaves (max, sum of exponentials) and, for gradients, how far each logit lies
//                                    below that maximum (see depth)
//   DX      dX = dz . W              dz [n, V]; K = V is cut into `splits` parts, each an fp32 partial sum
//   DW      dW = dz^T . X            bf16, or fp32 added up over chunks of rows
//   LOGITS_N, DX_N                   the first two for up to NT = 32 or 128 rows, as z^T = W . X^T and
//                                    dX^T = W^T . dz^T: the rows are the tile's columns, so the tensor cores do 1/8 or
//                                    1/2 of the work of a 256-row tile that is mostly padding. These calls are bound by
//                                    reading W; with padded tiles the 1 kW power cap held the clock at 1.25 GHz and the
//                                    bandwidth at 4.7 TB/s (one row x 248077 x 5120 in a loop: 540 us; now 405 us).
//
// n, the number of rows that have a loss, is only known on the device (`live`): the kernels read it there.
//
// Roles (192 threads per CTA): warp 0 loads tiles by TMA (128-byte swizzle, no multicast) into a ring of STAGES stages
// of 64-deep K blocks; warp 1 of the even CTA issues the pair's MMAs (M = 256, N = 256, K = 16: each CTA holds 128
// rows of A and 128 columns of B, so an operand byte in shared memory feeds twice the products of a one-CTA tile);
// warps 2-5 drain the double-buffered accumulators. Outputs leave through swizzled staging buffers by TMA stores of 32
// rows, one warp at a time (LOGITS_N, DX_N: by coalesced stores). All waits are bounded (sm100.cuh); one that gives up
// sets *status.
#pragma once
#include <climits>
#include "../common/common.cuh"
#include "../common/sm100_pair.cuh"
#include "../common/tmap.cuh"

namespace head {

enum Mode : int { LOGITS = 0, DX = 1, DW = 2, DW32 = 3, LOGITS_N = 4, DX_N = 5 };

constexpr int TILE = 256, BK = 64, THREADS = 192;
constexpr int HALF_BYTES = 128 * BK * 2;           // one CTA's half of a 256-wide operand block
constexpr int MN_CHUNK_BYTES = 64 * BK * 2;        // MN-major operands: 64-wide chunks of BK rows x 128 bytes
constexpr int STAGING_BYTES = 32 * 128;            // 32 rows of 128 bytes, one buffer per epilogue warp
constexpr int MASK_BYTES = 4 * 8 * 32 * 4;         // held columns of a tile: 8 words per row

template <int MODE, int NT>
struct Cfg {
  static constexpr bool NARROW = MODE == LOGITS_N || MODE == DX_N;
  static_assert(NARROW ? NT == 32 || NT == 128 : NT == TILE, "tile widths");
  static constexpr bool A_MN = MODE == DW || MODE == DW32 || MODE == DX_N;
  static constexpr bool B_MN = MODE == DX || MODE == DW || MODE == DW32;
  static constexpr int STAGE_BYTES = HALF_BYTES + NT / 2 * BK * 2;  // A half and B half
  // narrow tiles only stream W: their ring holds about as many bytes of it as fit. 256 x 256 tiles: 6 stages and one
  // staging buffer per warp took 1.90 / 2.05 / 2.01 ms (dW, dX, logits of 1024 rows in a loop), 5 stages and two
  // buffers 1.97 / 2.06 / 2.02.
  static constexpr int STAGES = NT == 32 ? 11 : NT == 128 ? 8 : 6;
  static constexpr int STAGING = NARROW ? 0 : 4 * STAGING_BYTES, MASKS = MODE == LOGITS ? MASK_BYTES : 0;
  static constexpr int BAR_BYTES = 512;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + STAGING + MASKS + BAR_BYTES + 1024;
  static constexpr int ACC_COLS = NT, TMEM_COLS = 2 * NT;
  static constexpr uint32_t IDESC = sm100::idesc_bf16(256, NT, A_MN, B_MN);
};

struct Args {
  const int* live;  // rows with a loss, all chunks (null: `rows` rows, whether they have one or not)
  int row0, rows;   // this chunk: live rows [row0, row0 + rows)
  int V, C;
  int splits, split_rows;  // DX: parts of K, and rows between their partial sums
  // LOGITS
  float scale2;     // logits to units of log2
  int K;            // held entries per row
  const int* sidx;  // [rows, K] ascending, INT_MAX behind the last
  const long* targets;  // LOGITS_N without `live`: the rows' targets in their place, and
  int* counts;      // four counters that the call's next kernel finds zero
  float2* part;     // [tiles of the vocabulary, part_ld]
  long part_ld;
  int store_e;
  unsigned short* e; // LOGITS_N: the logits' depths, [rows, ld_e]
  long ld_e;
  float* dx;        // DX_N: the partial sums
  int add;          // DW32: add to what is there
  const float* factor;  // DW, DW32: of the whole product
  int* status;
  uint4* poison;    // DW: the gradient's first 16 bytes, NaN if a wait of this or of an earlier product gave up
};

struct Maps {
  CUtensorMap a, b, out;
};

// Of a logit below its tile's or row's maximum: off by 2^-22 at most, and zero from 126 octaves below it on.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A tile's maximum m in units of log2, rounded up: fmaf(v, scale2, -m2) is then never above 0 for v <= m, where depth()
// would wrap around (rounded to nearest it is, from logits of 1e4 on). 0 for a tile of -inf.
__device__ __forceinline__ float tile_top(float m, float scale2) {
  return m == -INFINITY ? 0.f : __fmul_ru(m, scale2);
}

// A logit t <= 0 octaves (units of log2) from its tile's maximum as a 16-bit number of 1/512 octaves: the exponential
// it stands for is off by 7e-4 at most, a fifth of bf16's rounding, down to 2^-128. Here as the low half of an fp32
// word (2^23 + depth, so that one fused multiply-add rounds).
constexpr float DEPTH_STEPS = 512.f, DEPTH_BASE = 8388608.f;
__device__ __forceinline__ uint32_t depth(float t) {
  return __float_as_uint(fminf(fmaf(t, -DEPTH_STEPS, DEPTH_BASE), DEPTH_BASE + 65535.f));
}
__device__ __forceinline__ uint4 pack_depths(const float* t) {
  uint4 u;
  u.x = __byte_perm(depth(t[0]), depth(t[1]), 0x5410);
  u.y = __byte_perm(depth(t[2]), depth(t[3]), 0x5410);
  u.z = __byte_perm(depth(t[4]), depth(t[5]), 0x5410);
  u.w = __byte_perm(depth(t[6]), depth(t[7]), 0x5410);
  return u;
}

template <int MODE>
struct Work {
  int tiles_m, tiles_n, units, kblocks, splits, unit, stride;
  __device__ Work(const Args& a, int n) {
    const int rows_m = (n + TILE - 1) / TILE;
    if (MODE == LOGITS) {
      tiles_m = rows_m;
      tiles_n = (a.V + TILE - 1) / TILE;
      kblocks = (a.C + BK - 1) / BK;
    } else if (MODE == DX) {
      tiles_m = rows_m;
      tiles_n = (a.C + TILE - 1) / TILE;
      kblocks = (a.V + BK - 1) / BK;
    } else if (MODE == LOGITS_N) {
      tiles_m = n ? (a.V + TILE - 1) / TILE : 0;
      tiles_n = 1;
      kblocks = (a.C + BK - 1) / BK;
    } else if (MODE == DX_N) {
      tiles_m = n ? (a.C + TILE - 1) / TILE : 0;
      tiles_n = 1;
      kblocks = (a.V + BK - 1) / BK;
    } else {
      tiles_m = (a.V + TILE - 1) / TILE;
      tiles_n = (a.C + TILE - 1) / TILE;
      kblocks = max(1, (n + BK - 1) / BK);  // no live row: one block of zeros
    }
    splits = MODE == DX || MODE == DX_N ? a.splits : 1;
    units = tiles_m * tiles_n * splits;
    if (MODE == DW32 && n == 0 && a.add) units = 0;
    unit = blockIdx.x >> 1;
    stride = gridDim.x >> 1;
  }
  __device__ bool next(int& tm, int& tn, int& split, int& k0, int& k1) {
    if (unit >= units) return false;
    int t = unit;
    split = 0;
    if (MODE == DX || MODE == DX_N) {  // one part of K at a time: the pairs running together share its rows of W in L2
      const int tiles = tiles_m * tiles_n;
      split = t / tiles;
      t %= tiles;
    }
    if (MODE != DW && MODE != DW32) {  // rows fastest: the tiles running together share their part of W
      tm = t % tiles_m;
      tn = t / tiles_m;
    } else {  // columns fastest: they share the larger dz
      tn = t % tiles_n;
      tm = t / tiles_n;
    }
    k0 = (int)((long)kblocks * split / splits);
    k1 = (int)((long)kblocks * (split + 1) / splits);
    unit += stride;
    return true;
  }
};

// Held columns of row `row` in [col0, col0 + 256), and the columns past the vocabulary, as bits in this thread's eight
// words (word c at mask[c * 32]). Returns whether any row of the warp has one.
__device__ __forceinline__ bool held_mask(const Args& a, int row, int n, int col0, uint32_t* mask) {
  int lo = 0, first = INT_MAX;
  const int* s = a.sidx + (long)row * a.K;
  if (row < n) {
    int hi = a.K;
    while (hi - lo > 1) {  // lo: the last entry below col0, or 0
      const int mid = (lo + hi) >> 1;
      if (s[mid] < col0) lo = mid; else hi = mid;
    }
    first = s[lo];
    if (first < col0) first = ++lo < a.K ? s[lo] : INT_MAX;
  }
  const int end = min(col0 + TILE, a.V);
  const bool edge = col0 + TILE > a.V;
  if (!__any_sync(~0u, first < end) && !edge) return false;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const int over = edge ? min(max(col0 + 32 * c + 32 - a.V, 0), 32) : 0;  // columns of the word past the vocabulary
    mask[c * 32] = over >= 32 ? ~0u : over ? ~0u << (32 - over) : 0u;
  }
  while (first < end) {
    const int d = first - col0;
    mask[(d >> 5) * 32] |= 1u << (d & 31);
    first = ++lo < a.K ? s[lo] : INT_MAX;
  }
  return true;
}

// Entries of one row's record in [first, first + 32), as bits.
__device__ __forceinline__ uint32_t held_word(const int* s, int K, int first) {
  int lo = 0, hi = K;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] < first) lo = mid; else hi = mid;
  }
  uint32_t word = 0;
  for (; lo < K; ++lo) {
    const int d = s[lo] - first;
    if (d >= 32) break;
    if (d >= 0) word |= 1u << d;
  }
  return word;
}

// Lane j: op over the lanes of v[j]. Each step halves the columns a lane holds: 31 shuffles for 32 columns.
template <typename Op>
__device__ __forceinline__ float columns(float (&v)[32], int lane, Op op) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const bool upper = lane & s;
#pragma unroll
    for (int i = 0; i < s; ++i) {
      const float send = upper ? v[i] : v[i + s], keep = upper ? v[i + s] : v[i];
      v[i] = op(keep, __shfl_xor_sync(~0u, send, s));
    }
  }
  return v[0];
}

__device__ __forceinline__ void drop_held(float (&v)[32], uint32_t word) {
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = word >> i & 1 ? -INFINITY : v[i];
}

// 16-byte chunk q of staging row `lane` (128-byte swizzle).
__device__ __forceinline__ uint4* staged(uint8_t* buf, int lane, int q) {
  return reinterpret_cast<uint4*>(buf + lane * 128 + ((q ^ (lane & 7)) << 4));
}

template <int MODE, int NT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
pair_kernel(const __grid_constant__ Maps maps, const Args args) {
  using C_ = Cfg<MODE, NT>;
  constexpr bool A_MN = C_::A_MN, B_MN = C_::B_MN;
  constexpr int STAGES = C_::STAGES, STAGE_BYTES = C_::STAGE_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = sm100::align_smem_1024(smem_raw);
  uint8_t* staging = smem + STAGES * STAGE_BYTES;
  uint32_t* masks = reinterpret_cast<uint32_t*>(staging + C_::STAGING);
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + C_::STAGING + C_::MASKS);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = (int)sm100::cluster_rank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      sm100::mbar_init(&tfull[a], 1);
      sm100::mbar_init(&tempty[a], 8);  // four epilogue warps of each CTA
    }
    sm100::mbar_init(drain, 1);
    *abort = 0;
    sm100::fence_barrier_init();
    sm100::prefetch_tmap(&maps.a);
    sm100::prefetch_tmap(&maps.b);
    sm100::prefetch_tmap(&maps.out);
  }
  if (warp == 1) {
    sm100::tmem_alloc_pair(tmem_slot, C_::TMEM_COLS);
    sm100::tmem_relinquish_pair();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::cluster_sync();
  sm100::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const bool direct = MODE == LOGITS_N && !args.live;
  if (direct && blockIdx.x == 0 && threadIdx.x < 4) args.counts[threadIdx.x] = 0;
  const int n = direct ? args.rows : min(max(*args.live - args.row0, 0), args.rows);
  Work<MODE> work(args, n);
  int tm, tn, split, k0, k1;

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer (both CTAs)
    if (sm100::elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && work.next(tm, tn, split, k0, k1)) {
        const int am = tm * TILE + cta * 128, bn = tn * NT + cta * (NT / 2);
        for (int kb = k0; kb < k1; ++kb) {
          if (!sm100::mbar_wait(&empty[stage], phase ^ 1, abort)) {
            ok = false;
            break;
          }
          uint8_t* a_dst = smem + stage * STAGE_BYTES;
          uint8_t* b_dst = a_dst + HALF_BYTES;
          const uint32_t bar = sm100::map_rank(&full[stage], 0);
          if (cta == 0) sm100::mbar_expect_tx(&full[stage], 2 * STAGE_BYTES);  // both CTAs' bytes
          if (!A_MN) {
            sm100::tma_load_2d_pair(a_dst, &maps.a, bar, kb * BK, am);
          } else {
            sm100::tma_load_2d_pair(a_dst, &maps.a, bar, am, kb * BK);
            sm100::tma_load_2d_pair(a_dst + MN_CHUNK_BYTES, &maps.a, bar, am + 64, kb * BK);
          }
          if (!B_MN) {
            sm100::tma_load_2d_pair(b_dst, &maps.b, bar, kb * BK, bn);
          } else {
            sm100::tma_load_2d_pair(b_dst, &maps.b, bar, bn, kb * BK);
            sm100::tma_load_2d_pair(b_dst + MN_CHUNK_BYTES, &maps.b, bar, bn + 64, kb * BK);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      for (int s = 0; s < STAGES; ++s) {  // every loaded stage has been consumed before shared memory goes away
        if (!sm100::mbar_wait_bounded(&empty[stage], phase ^ 1)) break;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer (even CTA)
    if (cta == 0 && sm100::elect_one()) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      while (ok && work.next(tm, tn, split, k0, k1)) {
        if (!sm100::mbar_wait(&tempty[acc], acc_phase ^ 1, abort)) break;
        sm100::tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * C_::ACC_COLS;
        for (int kb = k0; kb < k1; ++kb) {
          if (!sm100::mbar_wait(&full[stage], phase, abort)) {
            ok = false;
            break;
          }
          sm100::tc_fence_after();
          const uint32_t a_base = sm100::smem_u32(smem + stage * STAGE_BYTES);
          const uint32_t b_base = a_base + HALF_BYTES;
#pragma unroll
          for (int ks = 0; ks < BK / 16; ++ks) {
            const uint64_t adesc = A_MN ? sm100::smem_desc(a_base + ks * 2048, MN_CHUNK_BYTES, 1024)
                                        : sm100::smem_desc(a_base + ks * 32, 16, 1024);
            const uint64_t bdesc = B_MN ? sm100::smem_desc(b_base + ks * 2048, MN_CHUNK_BYTES, 1024)
                                        : sm100::smem_desc(b_base + ks * 32, 16, 1024);
            sm100::mma_bf16_pair(d_tmem, adesc, bdesc, C_::IDESC, kb != k0 || ks != 0);
          }
          sm100::mma_commit_pair(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        sm100::mma_commit_pair(&tfull[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      sm100::mma_commit_pair(drain);
      sm100::mbar_wait_bounded(drain, 0);
    } else if (cta == 1 && lane == 0) {
      sm100::mbar_wait_bounded(drain, 0);  // the last arrival from the other CTA lands before shared memory goes away
    }
  } else {
    // ---------------------------------------------------------------- epilogue (warps 2..5, both CTAs)
    const int quarter = warp & 3;
    uint8_t* buf = staging + quarter * STAGING_BYTES;
    uint32_t* mask = masks + quarter * 8 * 32 + lane;
    const float factor = MODE == DW || MODE == DW32 ? *args.factor : 1.f;
    int acc = 0;
    uint32_t acc_phase = 0;
    while (work.next(tm, tn, split, k0, k1)) {
      const int row0 = tm * TILE + cta * 128 + quarter * 32;  // this warp's first row of the tile
      const int col0 = tn * TILE;
      bool masked = false;
      if (MODE == LOGITS) masked = held_mask(args, row0 + lane, n, col0, mask);
      if (!__all_sync(~0u, sm100::mbar_wait(&tfull[acc], acc_phase, abort))) break;
      sm100::tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * C_::ACC_COLS;
      // staging buffer of the next store: its previous store has been read
      auto next_buffer = [&]() {
        if (lane == 0) sm100::bulk_wait_read<0>();
        __syncwarp();
        return buf;
      };
      auto send = [&](uint8_t* b, int x, int y, bool add) {
        sm100::fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          if (add) sm100::tma_add_2d(&maps.out, b, x, y);
          else sm100::tma_store_2d(&maps.out, b, x, y);
          sm100::bulk_commit();
        }
      };
      if (MODE == LOGITS_N) {
        const int v_at = row0 + lane;  // this thread's entry of the vocabulary; the columns are rows of X
#pragma unroll 1
        for (int g = 0; g < NT / 32 && 32 * g < n; ++g) {
          const int j = 32 * g + lane;
          uint32_t word = 0;
          if (direct) {
            const long d = j < n ? args.targets[j] - row0 : -1;
            if (d >= 0 && d < 32) word = 1u << d;
          } else if (j < n) {
            word = held_word(args.sidx + (long)j * args.K, args.K, row0);
          }
          const bool held = __any_sync(~0u, word != 0);
          float v[32], t[32];
          sm100::tmem_ld32(t_row + 32 * g, v);
          sm100::tmem_wait_ld();
          if (held) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (__shfl_sync(~0u, word, i) >> lane & 1) v[i] = -INFINITY;
          }
          if (v_at >= args.V) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) t[i] = v[i];
          const float m = columns(t, lane, [](float a, float b) { return fmaxf(a, b); });
          const float m2 = tile_top(m, args.scale2);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            v[i] = fmaf(v[i], args.scale2, -__shfl_sync(~0u, m2, i));
            if (args.store_e && 32 * g + i < n && v_at < args.V)
              args.e[(32 * g + i) * args.ld_e + v_at] = (unsigned short)depth(v[i]);
            v[i] = ex2(v[i]);
          }
          const float sum = columns(v, lane, [](float a, float b) { return a + b; });
          if (j < n) args.part[(row0 / 32) * args.part_ld + j] = make_float2(m == -INFINITY ? m : m2, sum);
        }
      } else if (MODE == DX_N) {
        const int c_at = row0 + lane;
#pragma unroll 1
        for (int g = 0; g < NT / 32 && 32 * g < n; ++g) {
          float v[32];
          sm100::tmem_ld32(t_row + 32 * g, v);
          sm100::tmem_wait_ld();
          float* out = args.dx + ((long)split * args.split_rows + 32 * g) * args.C + c_at;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (32 * g + i < n && c_at < args.C) out[(long)i * args.C] = v[i];
        }
      } else if (MODE == LOGITS) {
        float m = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {
          float v[32];
          sm100::tmem_ld32(t_row + c * 32, v);
          sm100::tmem_wait_ld();
          if (masked) drop_held(v, mask[c * 32]);
#pragma unroll
          for (int i = 0; i < 32; ++i) m = fmaxf(m, v[i]);
        }
        const float m2 = tile_top(m, args.scale2);
        float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll 1
        for (int c = 0; c < 8; c += 2) {
          const bool store = args.store_e && row0 < n && col0 + 32 * c < args.V;
          uint8_t* b = store ? next_buffer() : nullptr;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[32];
            sm100::tmem_ld32(t_row + (c + h) * 32, v);
            sm100::tmem_wait_ld();
            if (masked) drop_held(v, mask[(c + h) * 32]);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = fmaf(v[i], args.scale2, -m2);
            if (store) {
#pragma unroll
              for (int q = 0; q < 4; ++q) *staged(b, lane, 4 * h + q) = pack_depths(v + 8 * q);
            }
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              s0 += ex2(v[i]);
              s1 += ex2(v[i + 1]);
              s2 += ex2(v[i + 2]);
              s3 += ex2(v[i + 3]);
            }
          }
          if (store) send(b, col0 + 32 * c, row0, false);
        }
        if (row0 + lane < n)
          args.part[tn * args.part_ld + row0 + lane] = make_float2(m == -INFINITY ? m : m2, (s0 + s1) + (s2 + s3));
      } else if (MODE == DW) {
#pragma unroll 1
        for (int c = 0; c < 8; c += 2) {
          if (col0 + 32 * c >= args.C || row0 >= args.V) break;
          uint8_t* b = next_buffer();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[32];
            sm100::tmem_ld32(t_row + (c + h) * 32, v);
            sm100::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= factor;
#pragma unroll
            for (int q = 0; q < 4; ++q) *staged(b, lane, 4 * h + q) = rt::pack8(v + 8 * q);
          }
          send(b, col0 + 32 * c, row0, false);
        }
      } else {
        const int y = MODE == DX ? split * args.split_rows + row0 : row0;
        const bool inside = MODE == DX ? row0 < n : row0 < args.V;
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {
          if (col0 + 32 * c >= args.C || !inside) break;
          uint8_t* b = next_buffer();
          float v[32];
          sm100::tmem_ld32(t_row + c * 32, v);
          sm100::tmem_wait_ld();
          if (MODE == DW32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= factor;
          }
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *staged(b, lane, q) = make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]),
                                             __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3]));
          send(b, col0 + 32 * c, y, MODE == DW32 && args.add);
        }
      }
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive_cluster(sm100::map_rank(&tempty[acc], 0));
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (lane == 0) sm100::bulk_wait<0>();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::cluster_sync();  // neither CTA's shared memory or TMEM is used by the other any more
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc_pair(tmem_base, C_::TMEM_COLS);
  }
  if (threadIdx.x == 0) {
    const bool gave_up = *abort;
    if (gave_up) atomicExch(args.status, 1);
    if (MODE == DW && (gave_up || blockIdx.x == 0)) {
      // Block 0 has stored the tile with these bytes. It looks at the status after that, and a block that gave up sets
      // the status before it writes them: whichever comes last leaves NaN.
      __threadfence();
      if (gave_up || *reinterpret_cast<volatile int*>(args.status))
        *args.poison = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
    }
  }
}

}  // namespace head
