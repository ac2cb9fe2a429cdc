// Matrix products grouped by expert: rows offsets[g] .. offsets[g+1] of A are multiplied by matrix g
// of B (forward and input gradient), or the rows of X and Y that belong to g are multiplied with
// each other (weight gradient), in one launch whose sizes stay on the device.
//
//   ROWS_NK   C[r, n]    = sum_k A[r, k] B[g, n, k]      B K-contiguous
//   ROWS_KN   C[r, n]    = sum_k A[r, k] B[g, k, n]      B N-contiguous (input gradient of the former)
//   WGRAD     D[g, m, n] = sum_r X[r, m] Y[r, n]         the ragged dimension is summed
//
// Every CTA reads the offsets once, clamps them to 0 <= offsets[g] <= offsets[g+1] <= rows (so no
// value of theirs reaches outside the operands) and walks the same list of output tiles. A tile of
// ROWS_* starts at its group's first row, whatever that is: TMA rows have no alignment rule. Rows
// past the group's end are multiplied too (they belong to the next group, and fall into
// accumulator rows of their own) but not stored. In WGRAD they would be summed, so the last k-slab
// of a group is cut: whole k-steps behind the end are not issued, and a warp clears the rows
// between the end and the k-step's border in shared memory (both operands: a NaN or infinity there
// must not meet a zero). The tensor maps of B are 3-D, so a k-slab that reaches over K reads zeros, not
// the next matrix.
#pragma once
#include "bw_gemm_kernel.cuh"

namespace bw {

enum class GMode : int { ROWS_NK = 0, ROWS_KN = 1, WGRAD = 2 };

constexpr int kMaxGroups = 1024;
constexpr int kGroupedThreads = 224;  // producer, MMA, 4 epilogue warps, tail warp
constexpr int kGroupedMaxStages = 10;

struct GroupedParams {
  void* C;                   // WGRAD: D
  const int* offsets;        // groups + 1
  const float* row_scale;    // one a row of A, or null
  const float* group_scale;  // one a group, or null
  long long ldc;             // elements between C rows
  int groups;
  int rows;                  // rows of A (X, Y)
  int m, n, k;               // WGRAD: m x n outputs a group; else n columns, k summed
  int W;                     // tile width
  int stages, stage_bytes;
  int group_m;               // raster: tile rows a band
  int vec;                   // store width in bytes: 32, 16, or the element's
  uint32_t fmt;              // operand format of the instruction descriptor
  int* status;
  unsigned long long budget_ns;
};

// 3-D TMA load (no multicast).
__device__ __forceinline__ void tma_load_3d(const CUtensorMap* m, uint64_t* bar, void* dst, int x, int y, int z,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "l"(policy)
      : "memory");
}

// mbar_wait by a whole warp with one answer for all its lanes, so that a timeout takes the warp
// out of its loop together.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, const WaitCtl& w, int where) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, w, where));
}

// Waits for a load of this CTA's own that is still in flight when a timeout ends the kernel early.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity, uint64_t budget_ns) {
  const uint32_t a = smem_u32(bar);
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(a, parity) && globaltimer_ns() - t0 < budget_ns) {
  }
}

// bounds[g] = first row of group g (bounds[groups] = end of the last), clamped and made
// non-decreasing; tiles[g] = output tiles of the groups before g, `per_row` of them per tm rows.
// Executed by one warp.
__device__ __forceinline__ void grouped_schedule(const int* offsets, int groups, int rows, int tm, int per_row,
                                                 int* bounds, int* tiles) {
  const int lane = threadIdx.x & 31;
  int high = 0;
  for (int base = 0; base <= groups; base += 32) {
    const int g = base + lane;
    int v = g <= groups ? min(max(__ldg(offsets + g), 0), rows) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v = max(v, u);
    }
    v = max(v, high);
    if (g <= groups) bounds[g] = v;
    high = __shfl_sync(0xffffffffu, v, 31);
  }
  if (tiles == nullptr) return;
  __syncwarp();
  int sum = 0;
  for (int base = 0; base < groups; base += 32) {
    const int g = base + lane;
    int v = g < groups ? (bounds[g + 1] - bounds[g] + tm - 1) / tm * per_row : 0;
    const int own = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (g < groups) tiles[g] = sum + v - own;
    sum += __shfl_sync(0xffffffffu, v, 31);
  }
  if (lane == 0) tiles[groups] = sum;
}

// One output tile: its group, first output row and column, output rows that exist (ROWS_*: of the
// group; WGRAD: of m), and the summed extent.
struct GTile {
  int g, row0, rows, col0, kbase, k;
};

template <GMode MODE, int TM>
struct GWalk {
  const int* bounds;
  const int* tiles;
  int groups, tiles_n, group_m, per;  // per: WGRAD tiles a group
  int m, k, W;
  int g = 0;

  __device__ __forceinline__ GWalk(const GroupedParams& p, const int* b, const int* t)
      : bounds(b), tiles(t), groups(p.groups), tiles_n((p.n + p.W - 1) / p.W), group_m(p.group_m), m(p.m), k(p.k), W(p.W) {
    per = (p.m + TM - 1) / TM * tiles_n;
  }
  __device__ __forceinline__ int count() const {
    if constexpr (MODE == GMode::WGRAD) return per * groups;
    else return tiles[groups];
  }
  // t must not decrease from call to call
  __device__ __forceinline__ GTile at(int t) {
    GTile o;
    int tm, tn;
    if constexpr (MODE == GMode::WGRAD) {
      g = t / per;
      tile_coords(t - g * per, (m + TM - 1) / TM, tiles_n, group_m, tm, tn);
      o.row0 = tm * TM;
      o.rows = min(TM, m - o.row0);
      o.kbase = bounds[g];
      o.k = bounds[g + 1] - o.kbase;
    } else {
      while (t >= tiles[g + 1]) ++g;
      const int first = bounds[g], n = bounds[g + 1] - first;
      tile_coords(t - tiles[g], (n + TM - 1) / TM, tiles_n, group_m, tm, tn);
      o.row0 = first + tm * TM;
      o.rows = min(TM, n - tm * TM);
      o.kbase = 0;
      o.k = k;
    }
    o.g = g;
    o.col0 = tn * W;
    return o;
  }
};

// Stores up to 32 columns of one row; `vec` bytes at a time where all of them exist.
template <Out OUT>
__device__ __forceinline__ void store_cols(void* base, long long at, const uint32_t (&r)[32], float alpha, int ncols,
                                           int vec) {
  if constexpr (OUT == Out::F32) {
    float* dst = static_cast<float*>(base) + at;
    if (vec >= 16 && ncols >= 32) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __float_as_uint(__uint_as_float(r[8 * g + j]) * alpha);
        if (vec == 32) {
          st_global_v8(dst + 8 * g, v);
        } else {
          st_global_v4(dst + 8 * g, make_uint4(v[0], v[1], v[2], v[3]));
          st_global_v4(dst + 8 * g + 4, make_uint4(v[4], v[5], v[6], v[7]));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < ncols) dst[j] = __uint_as_float(r[j]) * alpha;
    }
  } else {
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(base) + at;
    if (vec >= 16 && ncols >= 32) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(r[16 * g + 2 * j]) * alpha,
                                                         __uint_as_float(r[16 * g + 2 * j + 1]) * alpha);
          v[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        if (vec == 32) {
          st_global_v8(dst + 16 * g, v);
        } else {
          st_global_v4(dst + 16 * g, make_uint4(v[0], v[1], v[2], v[3]));
          st_global_v4(dst + 16 * g + 8, make_uint4(v[4], v[5], v[6], v[7]));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < ncols) dst[j] = __float2bfloat16_rn(__uint_as_float(r[j]) * alpha);
    }
  }
}

// One warp's 32 rows x W columns of a finished accumulator (zeros where nothing was summed).
// `release` runs after the last read of the accumulator.
template <GMode MODE, Out OUT, typename Release>
__device__ __forceinline__ void grouped_epilogue(const GroupedParams& p, const GTile& t, uint32_t tbase, int first,
                                                 int lane, Release release) {
  if (first >= t.rows) {  // none of this warp's rows exists
    release();
    return;
  }
  const int r = first + lane;
  const bool live = r < t.rows;
  long long at;
  float alpha = 1.f;
  if constexpr (MODE == GMode::WGRAD) {
    at = (static_cast<long long>(t.g) * p.m + t.row0 + r) * p.ldc + t.col0;
  } else {
    at = static_cast<long long>(t.row0 + r) * p.ldc + t.col0;
    if (p.group_scale && t.k > 0) alpha *= __ldg(p.group_scale + t.g);
    if (p.row_scale && t.k > 0 && live) alpha *= __ldg(p.row_scale + t.row0 + r);
  }
  const int width = min(p.W, p.n - t.col0);
#pragma unroll 1
  for (int c = 0; c < width; c += 32) {
    uint32_t v[32];
    if (t.k > 0) {
      tmem_ld_32x32b_x32(tbase + c, v);
      tmem_ld_wait();
      if (c + 32 >= width) release();
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = 0;
    }
    if (live) store_cols<OUT>(p.C, at + c, v, alpha, width - c, p.vec);
  }
}

__host__ __device__ constexpr int grouped_tail_bytes(int groups) {
  // barriers (full, empty, tailfull, fixed per stage; accfull, accempty x 2; teardown), TMEM slot and abort
  // flag, bounds and tiles, alignment slack
  return (4 * kGroupedMaxStages + 5) * 8 + 16 + 2 * (groups + 1) * 4 + 1024;
}

// WGRAD: a slab with `left` rows of its group left ends inside a k-step of 16.
__device__ __forceinline__ bool slab_is_cut(int left, int slab) { return left < slab && (left & 15) != 0; }

// One CTA a tile of 128 x W (W = 64, 128 or 256).
template <Kind KIND, GMode MODE, Out OUT>
__global__ void __launch_bounds__(kGroupedThreads, 1)
    bw_tc_gemm_grouped_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                              const GroupedParams p) {
  constexpr int KE = KindTraits<KIND>::kElemsPerSlab;   // K elements a slab (WGRAD: rows)
  constexpr bool A_MN = MODE == GMode::WGRAD, B_MN = MODE != GMode::ROWS_NK;
  constexpr int kABytes = kBM * kSlabBytes;
  constexpr int kBoxBytes = 64 * kSlabBytes;            // one 64 x 64 box of an MN-major operand
  static_assert(KIND == Kind::F16 || (KIND == Kind::F8 && MODE == GMode::ROWS_NK), "8-bit operands are K-contiguous");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int S = p.stages;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + static_cast<size_t>(S) * p.stage_bytes);
  uint64_t* empty = full + kGroupedMaxStages;
  uint64_t* tailfull = empty + kGroupedMaxStages;  // WGRAD: a cut slab has landed, its rows behind the end still to clear
  uint64_t* fixed = tailfull + kGroupedMaxStages;  // ... and are cleared
  uint64_t* accfull = fixed + kGroupedMaxStages;
  uint64_t* accempty = accfull + 2;
  uint64_t* teardown = accempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(teardown + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* bounds = reinterpret_cast<int*>(tmem_slot + 4);
  int* tiles = bounds + p.groups + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const WaitCtl wc{abort_flag, p.status, p.budget_ns};
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&tailfull[s], 1);
      mbar_init(&fixed[s], 1);
    }
    for (int b = 0; b < 2; ++b) { mbar_init(&accfull[b], 1); mbar_init(&accempty[b], kEpiWarps * 32); }
    mbar_init(teardown, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  // nothing is loaded (and the maps are empty) where nothing is summed
  if (warp == 0 && lane == 0 && (MODE == GMode::WGRAD ? p.rows : p.k) > 0) { tma_prefetch_desc(&tmA); tma_prefetch_desc(&tmB); }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  if (warp == 2)
    grouped_schedule(p.offsets, p.groups, p.rows, kBM, (p.n + p.W - 1) / p.W, bounds,
                     MODE == GMode::WGRAD ? nullptr : tiles);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  GWalk<MODE, kBM> walk(p, bounds, tiles);
  const int num_tiles = walk.count();

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      const uint64_t pol = l2_policy_evict_normal();
      int s = 0;
      uint32_t ph = 0;
      long long issued = 0;
      uint32_t cut_last = 0, cut_ph = 0;  // a bit a stage: its last slab was cut; parity of its next cut slab
      bool ok = true;
      for (int t = blockIdx.x; t < num_tiles && ok; t += gridDim.x) {
        const GTile o = walk.at(t);
        const int nk = (o.k + KE - 1) / KE;
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait(&empty[s], ph ^ 1, wc, 21)) { ok = false; break; }
          uint8_t* sA = smem + static_cast<size_t>(s) * p.stage_bytes;
          uint8_t* sB = sA + kABytes;
          if constexpr (A_MN) {
            // A cut slab lands on a barrier of its own, which the tail warp waits for: it follows
            // only these (on full[s] it could fall two phases behind). full[s] completes at once.
            uint64_t* bar = &full[s];
            if (slab_is_cut(o.k - kb * KE, KE)) {
              mbar_arrive(bar);
              bar = &tailfull[s];
              cut_last |= 1u << s;
              cut_ph ^= 1u << s;
            } else {
              cut_last &= ~(1u << s);
            }
            mbar_arrive_expect_tx(bar, p.stage_bytes);
            tma_load_2d(&tmA, bar, sA, o.row0, o.kbase + kb * KE, pol);
            tma_load_2d(&tmA, bar, sA + kBoxBytes, o.row0 + 64, o.kbase + kb * KE, pol);
            for (int j = 0; j < p.W / 64; ++j)
              tma_load_2d(&tmB, bar, sB + j * kBoxBytes, o.col0 + 64 * j, o.kbase + kb * KE, pol);
          } else {
            mbar_arrive_expect_tx(&full[s], p.stage_bytes);
            tma_load_2d(&tmA, &full[s], sA, kb * KE, o.row0, pol);
            if constexpr (B_MN) {
              for (int j = 0; j < p.W / 64; ++j)
                tma_load_3d(&tmB, &full[s], sB + j * kBoxBytes, o.col0 + 64 * j, kb * KE, o.g, pol);
            } else {
              tma_load_3d(&tmB, &full[s], sB, kb * KE, o.col0, o.g, pol);
            }
          }
          ++issued;
          if (++s == S) { s = 0; ph ^= 1; }
        }
      }
      if (!ok)  // a timeout: loads in flight must land before the CTA gives its shared memory back
        for (long long i = issued > S ? issued - S : 0; i < issued; ++i) {
          const int st = static_cast<int>(i % S);
          if ((cut_last >> st) & 1u) mbar_drain(&tailfull[st], ((cut_ph >> st) & 1u) ^ 1u, p.budget_ns);
          else mbar_drain(&full[st], static_cast<uint32_t>(i / S) & 1u, p.budget_ns);
        }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      const uint32_t idesc = idesc_dense(p.fmt, p.fmt, B_MN, kBM, p.W) | (A_MN ? 1u << 15 : 0u);
      int s = 0;
      uint32_t ph = 0, fixed_ph = 0;  // fixed_ph: one parity bit a stage
      int local = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < num_tiles && ok; t += gridDim.x) {
        const GTile o = walk.at(t);
        const int nk = (o.k + KE - 1) / KE;
        if (nk == 0) continue;
        const int b = local & 1;
        const uint32_t aph = (local >> 1) & 1;
        ++local;
        if (!mbar_wait(&accempty[b], aph ^ 1, wc, 22)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + b * 256;
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait(&full[s], ph, wc, 23)) { ok = false; break; }
          int steps = 4;
          if constexpr (MODE == GMode::WGRAD) {
            const int left = o.k - kb * KE;
            if (left < KE) {
              steps = (left + 15) / 16;
              if (slab_is_cut(left, KE)) {
                if (!mbar_wait(&fixed[s], (fixed_ph >> s) & 1u, wc, 24)) { ok = false; break; }
                fixed_ph ^= 1u << s;
              }
            }
          }
          tc_fence_after();
          const uint32_t aaddr = smem_u32(smem + static_cast<size_t>(s) * p.stage_bytes);
          const uint32_t baddr = aaddr + kABytes;
          for (int kk = 0; kk < steps; ++kk) {
            const uint32_t acc = (kb > 0 || kk > 0) ? 1u : 0u;
            uint64_t adesc, bdesc;
            if constexpr (A_MN) adesc = sdesc_sw128(aaddr + kk * 16 * kSlabBytes, kBoxBytes, 1024);
            else adesc = sdesc_sw128(aaddr + kk * 32, 16, 1024);
            if constexpr (B_MN) bdesc = sdesc_sw128(baddr + kk * 16 * kSlabBytes, kBoxBytes, 1024);
            else bdesc = sdesc_sw128(baddr + kk * 32, 16, 1024);
            if constexpr (KIND == Kind::F16) umma_f16(d_tmem, adesc, bdesc, idesc, acc);
            else umma_f8f6f4(d_tmem, adesc, bdesc, idesc, acc);
          }
          umma_commit(&empty[s]);
          if (++s == S) { s = 0; ph ^= 1; }
        }
        if (ok) umma_commit(&accfull[b]);
      }
      umma_commit(teardown);
      mbar_drain(teardown, 0, p.budget_ns);
    }
  } else if (warp < 6) {
    // ---------------- epilogue ----------------
    const int q = warp & 3;
    int local = 0;
    for (int t = blockIdx.x; t < num_tiles; t += gridDim.x) {
      const GTile o = walk.at(t);
      if (o.k == 0) {
        grouped_epilogue<MODE, OUT>(p, o, 0, q * 32, lane, [] {});
        continue;
      }
      const int b = local & 1;
      const uint32_t aph = (local >> 1) & 1;
      ++local;
      if (!mbar_wait_warp(&accfull[b], aph, wc, 25)) break;
      tc_fence_after();
      grouped_epilogue<MODE, OUT>(p, o, tmem_base + (static_cast<uint32_t>(q * 32) << 16) + b * 256, q * 32, lane, [&] {
        tc_fence_before();
        mbar_arrive(&accempty[b]);
      });
    }
  } else if (MODE == GMode::WGRAD) {
    // ---------------- tail: clears rows between a group's end and the k-step's border ----------------
    long long issue = 0;   // k-slabs before this tile
    uint32_t cut_ph = 0;   // one parity bit a stage
    for (int t = blockIdx.x; t < num_tiles; t += gridDim.x) {
      const GTile o = walk.at(t);
      const int nk = (o.k + KE - 1) / KE;
      const int left = o.k - (nk - 1) * KE;
      issue += nk;
      if (nk == 0 || !slab_is_cut(left, KE)) continue;
      const int s = static_cast<int>((issue - 1) % S);
      if (!mbar_wait_warp(&tailfull[s], (cut_ph >> s) & 1u, wc, 26)) break;
      cut_ph ^= 1u << s;
      const uint32_t base = smem_u32(smem + static_cast<size_t>(s) * p.stage_bytes);
      const int nz = ((left + 15) & ~15) - left;  // 1..15 rows of 128 bytes in each box
      for (int i = lane; i < (2 + p.W / 64) * nz * 8; i += 32) {
        const int box = i / (nz * 8), rest = i - box * nz * 8;
        st_shared_v4(base + box * kBoxBytes + (left + rest / 8) * kSlabBytes + (rest & 7) * 16, 0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&fixed[s]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace bw
