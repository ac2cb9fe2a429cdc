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
#include <type_traits>

#include "bw_gemm_kernel.cuh"

namespace bw {

enum class GMode : int { ROWS_NK = 0, ROWS_KN = 1, WGRAD = 2 };

constexpr int kMaxGroups = 1024;
constexpr int kGroupedEpiWarps = 8;   // two for each 32 lanes of Tensor Memory
constexpr int kGroupedThreads = 32 * (2 + kGroupedEpiWarps + 1);  // producer, MMA, epilogue, tail warp
constexpr int kGroupedChunkBytes = 64;                             // of a row, staged at a time
constexpr int kGroupedStageBytes = 32 * kGroupedChunkBytes;        // staging of one epilogue warp
constexpr int kGroupedMaxStages = 6;

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
  int sub;                   // K atoms a stage (single-CTA kernel)
  int stages, stage_bytes;
  int group_m;               // raster: tile rows a band
  int vec;                   // store width in bytes: 16, or the element's
  uint32_t fmt;              // operand format of the instruction descriptor
  int* status;
  unsigned long long budget_ns;
  // self-test of the waits (instances with STALL only): the first CTA's (pair's) MMA thread waits for nothing in front of
  // k-slab `stall`, its producers (leader, peer) take the wait in front of slab `stop` as timed out
  int stall, stop[2];
  int* landed;               // ... number of the CTA's stages whose last load was seen to land
};

// One lane of a converged warp. elect.sync (not a comparison of the lane index) tells the compiler
// that a single thread runs what follows, which tcgen05 and TMA instructions with their uniform
// operands need to be issued without a loop over lanes.
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}

// 3-D TMA load (no multicast).
__device__ __forceinline__ void tma_load_3d(const CUtensorMap* m, uint64_t* bar, void* dst, int x, int y, int z,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "l"(policy)
      : "memory");
}

// Bounded wait like mbar_wait, which reads the global timer as soon as its first try fails; that read
// takes longer than the wait of a running pipeline, so the timer starts after 64 tries here.
__device__ __forceinline__ bool mbar_poll(uint64_t* bar, uint32_t parity, const WaitCtl& w, int where) {
  const uint32_t a = smem_u32(bar);
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(a, parity)) return true;
  return mbar_wait(bar, parity, w, where);
}

// The same by a whole warp with one answer for all its lanes, so that a timeout takes the warp
// out of its loop together.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, const WaitCtl& w, int where) {
  return __all_sync(0xffffffffu, mbar_poll(bar, parity, w, where));
}

// Takes `bytes` off what a barrier's current phase still expects.
__device__ __forceinline__ void mbar_complete_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.shared::cluster.relaxed.cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
               : "memory");
}

// bounds[g] = first row of group g (bounds[groups] = end of the last), clamped and made
// non-decreasing; tiles[g] = output tiles of the groups before g, `per_row` of them per tm rows.
// All threads fetch the offsets (one trip to memory, past L1: the kernel before may just have written
// them); warp 2 scans them.
__device__ __forceinline__ void grouped_fetch(const int* offsets, int groups, int rows, int* bounds) {
  for (int g = threadIdx.x; g <= groups; g += kGroupedThreads) bounds[g] = min(max(__ldcg(offsets + g), 0), rows);
}
// Each lane takes a run of consecutive entries, so both scans cross the warp once whatever `groups` is
// (32 groups at a time, 64 of them took about 1300 cycles).
__device__ __forceinline__ void grouped_scan(int groups, int tm, int per_row, int* bounds, int* tiles) {
  const int lane = threadIdx.x & 31;
  const int run = groups / 32 + 1;  // of the groups + 1 bounds
  const int first = min(lane * run, groups + 1), last = min(first + run, groups + 1);
  int high = 0;  // largest bound of the run
  for (int g = first; g < last; ++g) high = max(high, bounds[g]);
  int before = high;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before = max(before, u);
  }
  before = __shfl_up_sync(0xffffffffu, before, 1);  // largest bound in front of the run
  if (lane == 0) before = 0;
  int v = before, sum = 0;
  for (int g = first; g < last; ++g) {
    const int u = max(v, bounds[g]);
    bounds[g] = u;
    if (g > 0) sum += (u - v + tm - 1) / tm * per_row;  // tiles of group g - 1
    v = u;
  }
  if (tiles == nullptr) return;
  int at = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at += u;
  }
  at -= sum;  // tiles in front of the run
  v = before;
  for (int g = first; g < last; ++g) {
    const int u = bounds[g];
    if (g > 0) at += (u - v + tm - 1) / tm * per_row;
    tiles[g] = at;
    v = u;
  }
}

// One output tile: its group, first output row and column, output rows that exist (ROWS_*: of the
// group; WGRAD: of m), and the summed extent.
struct GTile {
  int g, row0, rows, col0, kbase, k;
  bool b_once;  // no other tile reads this one's columns of B
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
      o.b_once = true;
    } else {
      while (t >= tiles[g + 1]) ++g;
      const int first = bounds[g], n = bounds[g + 1] - first;
      tile_coords(t - tiles[g], (n + TM - 1) / TM, tiles_n, group_m, tm, tn);
      o.row0 = first + tm * TM;
      o.rows = min(TM, n - tm * TM);
      o.kbase = 0;
      o.k = k;
      o.b_once = n <= TM;
    }
    o.g = g;
    o.col0 = tn * W;
    return o;
  }
};

// TMEM -> registers: 32 lanes x 16 consecutive 32-bit columns.
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// One warp's share of 32 rows x W columns of a finished accumulator (zeros where nothing was summed): every other
// chunk of 64 bytes of each row, from chunk `part`. A chunk goes registers -> the warp's 2 KB of shared memory
// (16-byte pieces, XOR-swizzled over the banks) -> 4 lanes a row, so that a store instruction covers whole
// sectors of 8 rows. A lane storing its own row straight from registers touches 32 lines an instruction; tiles that
// sum little (a gradient of few rows a group, short K) are bound by that, and by the latency of one
// warp's chain: hence two warps for the same rows. `release` runs after the last read of the accumulator.
template <GMode MODE, Out OUT, typename Release>
__device__ __forceinline__ void grouped_epilogue(const GroupedParams& p, const GTile& t, uint32_t tbase, int first,
                                                 int part, int lane, uint32_t stage, Release release) {
  constexpr int kElem = OUT == Out::F32 ? 4 : 2;
  constexpr int kCols = kGroupedChunkBytes / kElem;    // columns of a chunk
  constexpr int kPiece = 16 / kElem;
  const int width = min(p.W, p.n - t.col0);
  if (first >= t.rows || part * kCols >= width) {  // none of this warp's rows or columns exists
    release();
    return;
  }
  const int nrows = min(32, t.rows - first);
  const bool summed = t.k > 0;
  uint32_t v[kCols];
  auto load = [&](int c) {
    if constexpr (kCols == 32) tmem_ld_32x32b_x32(tbase + c, v);
    else tmem_ld_32x32b_x16(tbase + c, v);
  };
  if (summed) load(part * kCols);  // on its way beside the scales
  long long row;
  float alpha = 1.f;
  bool twice = false;  // the scales' product leaves FP32's normal range in one of this warp's rows
  if constexpr (MODE == GMode::WGRAD) {
    row = static_cast<long long>(t.g) * p.m + t.row0 + first;
  } else {
    row = t.row0 + first;
    if (t.k > 0) {
      if (p.group_scale) alpha *= __ldcg(p.group_scale + t.g);
      if (p.row_scale && lane < nrows) alpha *= __ldcg(p.row_scale + row + lane);
      if (p.group_scale && p.row_scale)  // exponent field 0 or 255
        twice = __any_sync(0xffffffffu, (__float_as_uint(alpha) << 1) - 0x01000000u >= 0xfe000000u);
    }
  }
  const long long pitch = p.ldc * kElem;
  char* out = static_cast<char*>(p.C) + row * pitch + static_cast<long long>(t.col0) * kElem;
  // the pieces that this lane stores: piece jj of rows rr + 8 i
  const int rr = lane >> 2, jj = lane & 3;
  const uint32_t from = stage + rr * kGroupedChunkBytes + ((jj ^ ((rr >> 1) & 3)) << 4);
  const uint32_t to = stage + lane * kGroupedChunkBytes;
  const int swz = (lane >> 1) & 3;
  float beta = 1.f;
  auto store = [&](auto scaled_twice) {
#pragma unroll 1
    for (int c = part * kCols; c < width; c += 2 * kCols) {
      uint32_t w[16];
      if (summed) tmem_ld_wait();
      if constexpr (decltype(scaled_twice)::value) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * beta);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if constexpr (OUT == Out::F32) {
          w[j] = __float_as_uint(__uint_as_float(v[j]) * alpha);
        } else {
          const __nv_bfloat162 two =
              __floats2bfloat162_rn(__uint_as_float(v[2 * j]) * alpha, __uint_as_float(v[2 * j + 1]) * alpha);
          w[j] = *reinterpret_cast<const uint32_t*>(&two);
        }
        if (!summed) w[j] = 0;
      }
      if (summed) {  // the next columns come while these are stored
        if (c + 2 * kCols < width) load(c + 2 * kCols);
        else release();
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) st_shared_v4(to + ((j ^ swz) << 4), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
      __syncwarp();
      const int have = width - c - jj * kPiece;  // columns of this lane's pieces that exist
      char* dst = out + rr * pitch + (c + jj * kPiece) * kElem;
      if (p.vec == 16 && width - c >= kCols) {
        uint4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ld_shared_v4(from + i * 8 * kGroupedChunkBytes);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (rr + 8 * i < nrows) st_global_v4(dst + 8 * i * pitch, x[i]);
      } else {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          if (rr + 8 * i >= nrows || have <= 0) continue;
          const uint4 x = ld_shared_v4(from + i * 8 * kGroupedChunkBytes);
          char* at = dst + 8 * i * pitch;
          if (p.vec == 16 && have >= kPiece) {
            st_global_v4(at, x);
          } else {
            const uint32_t e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < kPiece; ++k) {
              if (k >= have) break;
              if constexpr (OUT == Out::F32) reinterpret_cast<uint32_t*>(at)[k] = e[k];
              else reinterpret_cast<uint16_t*>(at)[k] = static_cast<uint16_t>(e[k / 2] >> (16 * (k & 1)));
            }
          }
        }
      }
      __syncwarp();
    }
  };
  if (MODE != GMode::WGRAD && twice) {
    // alpha becomes the smaller scale, and the sums are multiplied by the larger one, beta, first (a loop of its own: 32
    // products more, or a branch around them, take 4% of a call that is bound by this loop)
    const float g = __ldcg(p.group_scale + t.g), r = lane < nrows ? __ldcg(p.row_scale + row + lane) : 1.f;
    if (g != 0.f && r != 0.f) {
      alpha = fabsf(g) > fabsf(r) ? r : g;
      beta = fabsf(g) > fabsf(r) ? g : r;
    }
    store(std::true_type{});
  } else {
    store(std::false_type{});
  }
}

__host__ __device__ constexpr int grouped_tail_bytes(int groups) {
  // barriers (full, empty, tailfull, fixed per stage; accfull, accempty x 2; teardown), TMEM slot, abort flags and
  // the pair's record of its loads, bounds and tiles, the epilogue's staging, alignment slack
  return (4 * kGroupedMaxStages + 5) * 8 + 32 + 2 * (groups + 1) * 4 + kGroupedEpiWarps * kGroupedStageBytes + 1024;
}

// A tile of few rows loads them in boxes of 16 (a box of 128 rows would fetch its neighbours' too, and
// one that lies mostly behind the tensor's end is slow: 8 rows of 4096 x 2048 E4M3 times 8
// matrices took 66 us with it, 19 us without).
constexpr int kFewRows = 64;
__device__ __forceinline__ int a_load_bytes(int valid) {
  return valid > kFewRows ? kBM * kSlabBytes : (valid + 15) / 16 * 16 * kSlabBytes;
}

// Clears n (1..15) rows of 128 bytes: a warp, 4 rows at a time.
__device__ __forceinline__ void clear_rows(uint32_t at, int n, int lane) {
  const uint32_t mine = at + (lane >> 3) * kSlabBytes + (lane & 7) * 16;
#pragma unroll
  for (int r = 0; r < 16; r += 4)
    if ((lane >> 3) + r < n) st_shared_v4(mine + r * kSlabBytes, 0, 0, 0, 0);
}

// WGRAD: a slab with `left` rows of its group left ends inside a k-step of 16.
__device__ __forceinline__ bool slab_is_cut(int left, int slab) { return left < slab && (left & 15) != 0; }

// Groups of few rows: bound by HBM, which every weight leaves once (64 matrices of 4096 x 2048 E4M3, 16 rows each:
// 85-90 us, 6.0-6.5 TB/s of the measured 6.5). Persistent, one CTA an SM: warp 0 streams k-slabs into
// a ring of 3 to 6 stages, warp 1 multiplies, warps 2-9 store one tile while the next is summed in the
// other half of Tensor Memory. A tile has 128 rows however few count: their products cost nothing while the weights
// arrive, and narrower tiles would read them again.
// One CTA a tile of 128 x W (W <= 256; a multiple of 16, for an N-contiguous B of 64).
template <Kind KIND, GMode MODE, Out OUT, bool STALL = false>
__global__ void __launch_bounds__(kGroupedThreads, 1)
    bw_tc_gemm_grouped_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA16,
                              const __grid_constant__ CUtensorMap tmB, const GroupedParams p) {
  constexpr int KA = KindTraits<KIND>::kElemsPerSlab;   // K elements a swizzle atom (WGRAD: rows)
  const int KE = KA * p.sub;                            // ... a stage
  constexpr bool A_MN = MODE == GMode::WGRAD, B_MN = MODE != GMode::ROWS_NK;
  constexpr int kABytes = kBM * kSlabBytes;             // an atom of A
  const int b_bytes = p.W * kSlabBytes;                 // an atom of B
  constexpr int kBoxBytes = 64 * kSlabBytes;            // one 64 x 64 box of an MN-major operand
  static_assert(KIND == Kind::F16 || (KIND == Kind::F8 && MODE == GMode::ROWS_NK), "8-bit operands are K-contiguous");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int S = p.stages;
  uint8_t* staging = smem + static_cast<size_t>(S) * p.stage_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + kGroupedEpiWarps * kGroupedStageBytes);
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
    for (int b = 0; b < 2; ++b) { mbar_init(&accfull[b], 1); mbar_init(&accempty[b], kGroupedEpiWarps * 32); }
    mbar_init(teardown, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  // nothing is loaded (and the maps are empty) where nothing is summed
  if (warp == 0 && lane == 0 && (MODE == GMode::WGRAD ? p.rows : p.k) > 0) { tma_prefetch_desc(&tmA); tma_prefetch_desc(&tmB); }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  grid_dependency_wait();
  grouped_fetch(p.offsets, p.groups, p.rows, bounds);
  __syncthreads();
  if (warp == 2) grouped_scan(p.groups, kBM, (p.n + p.W - 1) / p.W, bounds, MODE == GMode::WGRAD ? nullptr : tiles);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  GWalk<MODE, kBM> walk(p, bounds, tiles);
  const int num_tiles = walk.count();

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (elect_one()) {
      // A's rows are read by every tile of their group, B's columns (the weights) once where a group
      // has one tile row: these then leave L2 first (64 matrices of 4096 x 2048 E4M3 and 1024 rows: 90.6 -> 84.8 us;
      // for groups of more rows it costs 3%). WGRAD: Y's, which measured the same or 5-10% faster.
      const uint64_t pol = l2_policy_evict_last(), pol_once = l2_policy_evict_first(), pol_more = l2_policy_evict_normal();
      int s = 0;
      uint32_t ph = 0;
      long long issued = 0;
      uint32_t cut_last = 0, cut_ph = 0;  // a bit a stage: its last slab was cut; parity of its next cut slab
      bool ok = true;
      for (int t = blockIdx.x; t < num_tiles && ok; t += gridDim.x) {
        const GTile o = walk.at(t);
        const int nk = (o.k + KE - 1) / KE;
        const uint64_t pol_b = o.b_once ? pol_once : pol_more;
        for (int kb = 0; kb < nk; ++kb) {
          if (STALL && blockIdx.x == 0 && issued == p.stop[0]) { ok = false; break; }
          if (!mbar_poll(&empty[s], ph ^ 1, wc, 21)) { ok = false; break; }
          uint8_t* sA = smem + static_cast<size_t>(s) * p.stage_bytes;
          uint8_t* sB = sA + p.sub * kABytes;
          const int left = o.k - kb * KE;
          const int atoms = left > KA ? p.sub : 1;  // the others lie behind the end
          if constexpr (A_MN) {
            // A cut slab lands on a barrier of its own, which the tail warp waits for: it follows
            // only these (on full[s] it could fall two phases behind). full[s] completes at once.
            uint64_t* bar = &full[s];
            if (slab_is_cut(left, KE)) {
              mbar_arrive(bar);
              bar = &tailfull[s];
              cut_last |= 1u << s;
              cut_ph ^= 1u << s;
            } else {
              cut_last &= ~(1u << s);
            }
            mbar_arrive_expect_tx(bar, atoms * (kABytes + b_bytes));
            for (int a = 0; a < atoms; ++a) {
              const int y = o.kbase + kb * KE + a * KA;
              tma_load_2d(&tmA, bar, sA + a * kABytes, o.row0, y, pol);
              tma_load_2d(&tmA, bar, sA + a * kABytes + kBoxBytes, o.row0 + 64, y, pol);
              for (int j = 0; j < p.W / 64; ++j)
                tma_load_2d(&tmB, bar, sB + a * b_bytes + j * kBoxBytes, o.col0 + 64 * j, y, pol_b);
            }
          } else {
            mbar_arrive_expect_tx(&full[s], atoms * (a_load_bytes(o.rows) + b_bytes));
            for (int a = 0; a < atoms; ++a) {
              const int x = kb * KE + a * KA;
              if (o.rows > kFewRows) {
                tma_load_2d(&tmA, &full[s], sA + a * kABytes, x, o.row0, pol);
              } else {
                for (int r = 0; r < o.rows; r += 16)
                  tma_load_2d(&tmA16, &full[s], sA + a * kABytes + r * kSlabBytes, x, o.row0 + r, pol);
              }
              if constexpr (B_MN) {
                for (int j = 0; j < p.W / 64; ++j)
                  tma_load_3d(&tmB, &full[s], sB + a * b_bytes + j * kBoxBytes, o.col0 + 64 * j, x, o.g, pol_b);
              } else {
                tma_load_3d(&tmB, &full[s], sB + a * b_bytes, x, o.col0, o.g, pol_b);
              }
            }
          }
          ++issued;
          if (++s == S) { s = 0; ph ^= 1; }
        }
      }
      // Every load lands before the CTA gives its shared memory back, whichever thread's wait may have
      // timed out: this one has issued its last slabs long before the others are done with them.
      for (int i = 0; i < S && i < issued; ++i) {
        if (--s < 0) { s = S - 1; ph ^= 1; }
        const bool cut = (cut_last >> s) & 1u;
        const bool in = mbar_drain(cut ? &tailfull[s] : &full[s], cut ? ((cut_ph >> s) & 1u) ^ 1u : ph);
        if (STALL && blockIdx.x == 0 && in) atomicAdd(p.landed, 1);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (elect_one()) {
      const uint32_t idesc = idesc_dense(p.fmt, p.fmt, B_MN, kBM, p.W) | (A_MN ? 1u << 15 : 0u);
      int s = 0;
      uint32_t ph = 0, fixed_ph = 0;  // fixed_ph: one parity bit a stage
      int local = 0;
      bool ok = true;
      [[maybe_unused]] int slab = 0;
      for (int t = blockIdx.x; t < num_tiles && ok; t += gridDim.x) {
        const GTile o = walk.at(t);
        const int nk = (o.k + KE - 1) / KE;
        if (nk == 0) continue;
        const int b = local & 1;
        const uint32_t aph = (local >> 1) & 1;
        ++local;
        if (!mbar_poll(&accempty[b], aph ^ 1, wc, 22)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + b * 256;
        for (int kb = 0; kb < nk; ++kb) {
          if constexpr (STALL)
            if (blockIdx.x == 0 && slab++ == p.stall && !mbar_poll(teardown, 0, wc, 27)) { ok = false; break; }
          if (!mbar_poll(&full[s], ph, wc, 23)) { ok = false; break; }
          const int left = o.k - kb * KE;
          // WGRAD: k-steps with rows of the group; else whole atoms (zeros behind K)
          int steps = 4 * p.sub;
          if (left < KE) steps = MODE == GMode::WGRAD ? (left + 15) / 16 : (left > KA ? 4 * p.sub : 4);
          if (MODE == GMode::WGRAD && slab_is_cut(left, KE)) {
            if (!mbar_poll(&fixed[s], (fixed_ph >> s) & 1u, wc, 24)) { ok = false; break; }
            fixed_ph ^= 1u << s;
          }
          tc_fence_after();
          const uint32_t abase = smem_u32(smem + static_cast<size_t>(s) * p.stage_bytes);
          const uint32_t bbase = abase + p.sub * kABytes;
          for (int kk = 0; kk < steps; ++kk) {
            const uint32_t acc = (kb > 0 || kk > 0) ? 1u : 0u;
            const uint32_t aaddr = abase + (kk >> 2) * kABytes, baddr = bbase + (kk >> 2) * b_bytes;
            uint64_t adesc, bdesc;
            if constexpr (A_MN) adesc = sdesc_sw128(aaddr + (kk & 3) * 16 * kSlabBytes, kBoxBytes, 1024);
            else adesc = sdesc_sw128(aaddr + (kk & 3) * 32, 16, 1024);
            if constexpr (B_MN) bdesc = sdesc_sw128(baddr + (kk & 3) * 16 * kSlabBytes, kBoxBytes, 1024);
            else bdesc = sdesc_sw128(baddr + (kk & 3) * 32, 16, 1024);
            if constexpr (KIND == Kind::F16) umma_f16(d_tmem, adesc, bdesc, idesc, acc);
            else umma_f8f6f4(d_tmem, adesc, bdesc, idesc, acc);
          }
          umma_commit(&empty[s]);
          if (++s == S) { s = 0; ph ^= 1; }
        }
        if (ok) umma_commit(&accfull[b]);
      }
      umma_commit(teardown);
      mbar_drain(teardown, 0);
    }
  } else if (warp < 2 + kGroupedEpiWarps) {
    // ---------------- epilogue ----------------
    const int q = warp & 3, part = (warp - 2) >> 2;  // lanes of Tensor Memory, every other chunk of columns
    const uint32_t stage = smem_u32(staging) + (warp - 2) * kGroupedStageBytes;
    int local = 0;
    for (int t = blockIdx.x; t < num_tiles; t += gridDim.x) {
      const GTile o = walk.at(t);
      if (o.k == 0) {
        grouped_epilogue<MODE, OUT>(p, o, 0, q * 32, part, lane, stage, [] {});
        continue;
      }
      const int b = local & 1;
      const uint32_t aph = (local >> 1) & 1;
      ++local;
      if (!mbar_wait_warp(&accfull[b], aph, wc, 25)) break;
      tc_fence_after();
      grouped_epilogue<MODE, OUT>(p, o, tmem_base + (static_cast<uint32_t>(q * 32) << 16) + b * 256, q * 32, part, lane, stage,
                                  [&] {
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
      const int j = left / KA, at = left - j * KA;  // atom and row of the first row behind the end
      const uint32_t a0 = base + j * kABytes, b0 = base + p.sub * kABytes + j * b_bytes;
      const int nz = ((left + 15) & ~15) - left;    // 1..15 rows in each box
      for (int box = 0; box < 2; ++box) clear_rows(a0 + box * kBoxBytes + at * kSlabBytes, nz, lane);
      for (int box = 0; box < p.W / 64; ++box) clear_rows(b0 + box * kBoxBytes + at * kSlabBytes, nz, lane);
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

// ------------------------------------------------------------------------------------
// CTA pairs: 256 x 256 tiles for groups with many rows, bound by the tensor cores (91-92% of the active cycles; 8 x
// 4096 rows of 4096 x 2048 BF16 348 us = 1581 TFLOP/s at 1.47 GHz, E4M3 8 x 2048 of 8192 x 4096 371 us = 2967 at 1.43): a pair
// moves a third less per product than two single CTAs, which L2 cannot feed at that rate. As in bw_gemm_pair.cuh, each CTA of a pair
// loads its 128 rows of A and 128 columns of B, the leader's MMA thread multiplies both halves, and a
// pipeline stage holds two swizzle atoms of K. Barriers: full[s], fixed[s] and accempty[b] count in
// the leader; empty[s], accfull[b] and tailfull[s] exist in both CTAs.
// ------------------------------------------------------------------------------------
constexpr int kPairStages = 3, kPairSub = 2;  // stages, K atoms a stage
constexpr int kPairAtom = 128 * kSlabBytes;
constexpr int kPairStageBytes = 2 * kPairSub * kPairAtom;

__device__ __forceinline__ void tma_load_3d_pair(const CUtensorMap* m, uint32_t bar_cluster, void* dst, int x, int y,
                                                 int z, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar_cluster), "r"(x), "r"(y), "r"(z), "l"(policy)
      : "memory");
}
// Bounded wait that also acquires what the other CTA's threads wrote before they arrived.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, const WaitCtl& w, int where) {
  const uint32_t a = smem_u32(bar);
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(a), "r"(parity)
        : "memory");
    if (ok) return true;
    if (*w.abort_flag) return false;
    if (globaltimer_ns() - t0 > w.budget_ns) {
      *w.abort_flag = 1;
      atomicCAS(w.status, kDevOk, kDevTimeout * 256 + (where & 255));
      return false;
    }
  }
}

template <Kind KIND, GMode MODE, Out OUT, bool STALL = false>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGroupedThreads, 1)
    bw_tc_gemm_grouped_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA16,
                                   const __grid_constant__ CUtensorMap tmB, const GroupedParams p) {
  constexpr int KA = KindTraits<KIND>::kElemsPerSlab;  // K elements an atom (WGRAD: rows)
  constexpr int KE = KA * kPairSub;                    // ... a stage
  constexpr bool A_MN = MODE == GMode::WGRAD, B_MN = MODE != GMode::ROWS_NK;
  constexpr int kBoxBytes = 64 * kSlabBytes;
  constexpr int S = kPairStages;
  static_assert(KIND == Kind::F16 || (KIND == Kind::F8 && MODE == GMode::ROWS_NK), "8-bit operands are K-contiguous");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + S * kPairStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + kGroupedEpiWarps * kGroupedStageBytes);
  uint64_t* empty = full + kGroupedMaxStages;
  uint64_t* tailfull = empty + kGroupedMaxStages;
  uint64_t* fixed = tailfull + kGroupedMaxStages;
  uint64_t* accfull = fixed + kGroupedMaxStages;
  uint64_t* accempty = accfull + 2;
  uint64_t* teardown = accempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(teardown + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);
  volatile int* peer_abort = reinterpret_cast<volatile int*>(tmem_slot + 3);  // the other CTA's abort flag, written at the end
  uint32_t* loads = tmem_slot + 4;  // what this CTA's producer leaves: slabs issued, bytes of `peer_units`
  int* bounds = reinterpret_cast<int*>(tmem_slot + 8);
  int* tiles = bounds + p.groups + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
  const int half = static_cast<int>(rank) * 128;  // this CTA's first row and column of a tile
  const WaitCtl wc{abort_flag, p.status, p.budget_ns};
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&tailfull[s], 1);
      mbar_init(&fixed[s], 2);
    }
    for (int b = 0; b < 2; ++b) { mbar_init(&accfull[b], 1); mbar_init(&accempty[b], 2 * kGroupedEpiWarps); }
    mbar_init(teardown, 1);
    *abort_flag = 0;
    *peer_abort = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0 && (MODE == GMode::WGRAD ? p.rows : p.k) > 0) { tma_prefetch_desc(&tmA); tma_prefetch_desc(&tmB); }
  if (warp == 1) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
  grid_dependency_wait();
  grouped_fetch(p.offsets, p.groups, p.rows, bounds);
  __syncthreads();
  if (warp == 2) grouped_scan(p.groups, 256, (p.n + 255) / 256, bounds, MODE == GMode::WGRAD ? nullptr : tiles);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  GWalk<MODE, 256> walk(p, bounds, tiles);
  const int num_tiles = walk.count();

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    if (elect_one()) {
      const uint64_t pol = l2_policy_evict_last();
      const uint32_t full_leader = mapa_shared(smem_u32(full), 0);
      int s = 0;
      uint32_t ph = 0;
      uint32_t issued = 0;
      uint32_t peer_units = 0;  // a byte a stage: what the peer's loads of its last slab add to full, in units of 2 KB
      uint32_t cut_last = 0, cut_ph = 0;
      bool ok = true;
      for (int t = cluster; t < num_tiles && ok; t += nclusters) {
        const GTile o = walk.at(t);
        const int nk = (o.k + KE - 1) / KE;
        const int arow = o.row0 + half, bcol = o.col0 + half;
        const int valid = min(128, o.rows - half);  // ROWS: this CTA's rows of the tile (may be <= 0)
        const uint32_t peer_a = o.rows > 128 ? a_load_bytes(o.rows - 128) : 0;
        const uint32_t a_bytes = a_load_bytes(min(128, o.rows)) + peer_a;
        for (int kb = 0; kb < nk; ++kb) {
          if (STALL && cluster == 0 && issued == static_cast<uint32_t>(p.stop[rank])) { ok = false; break; }
          if (!mbar_poll(&empty[s], ph ^ 1, wc, 61)) { ok = false; break; }
          uint8_t* sA = smem + s * kPairStageBytes;
          uint8_t* sB = sA + kPairSub * kPairAtom;
          uint32_t bar = full_leader + s * 8;
          const int left = o.k - kb * KE;
          const int atoms = left > KA ? 2 : 1;
          const bool cut = A_MN && slab_is_cut(left, KE);
          const uint32_t units = cut ? 0u : atoms * (A_MN ? 2 * kPairAtom : peer_a + kPairAtom) / 2048;
          peer_units = (peer_units & ~(255u << (8 * s))) | units << (8 * s);
          if constexpr (A_MN) {
            // a cut slab's two halves land on barriers of their own CTA's (see the single-CTA kernel)
            if (cut) {
              if (leader) mbar_arrive(&full[s]);
              bar = smem_u32(&tailfull[s]);
              mbar_arrive_expect_tx(&tailfull[s], atoms * 2 * kPairAtom);
              cut_last |= 1u << s;
              cut_ph ^= 1u << s;
            } else {
              if (leader) mbar_arrive_expect_tx(&full[s], atoms * 4 * kPairAtom);
              cut_last &= ~(1u << s);
            }
            for (int j = 0; j < atoms; ++j) {
              const int y = o.kbase + kb * KE + j * KA;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                tma_load_2d_pair(&tmA, bar, sA + j * kPairAtom + i * kBoxBytes, arow + 64 * i, y, pol);
                tma_load_2d_pair(&tmB, bar, sB + j * kPairAtom + i * kBoxBytes, bcol + 64 * i, y, pol);
              }
            }
          } else {
            if (leader) mbar_arrive_expect_tx(&full[s], atoms * (a_bytes + 2 * kPairAtom));
            for (int j = 0; j < atoms; ++j) {
              const int x = kb * KE + j * KA;
              if (valid > kFewRows) {
                tma_load_2d_pair(&tmA, bar, sA + j * kPairAtom, x, arow, pol);
              } else {
                for (int r = 0; r < valid; r += 16)
                  tma_load_2d_pair(&tmA16, bar, sA + j * kPairAtom + r * kSlabBytes, x, arow + r, pol);
              }
              if constexpr (B_MN) {
                tma_load_3d_pair(&tmB, bar, sB + j * kPairAtom, bcol, x, o.g, pol);
                tma_load_3d_pair(&tmB, bar, sB + j * kPairAtom + kBoxBytes, bcol + 64, x, o.g, pol);
              } else {
                tma_load_3d_pair(&tmB, bar, sB + j * kPairAtom, x, bcol, o.g, pol);
              }
            }
          }
          ++issued;
          if (++s == S) { s = 0; ph ^= 1; }
        }
      }
      // cut slabs land on barriers of this CTA's own; the others are waited for at the end, where it is known
      // whether both CTAs issued them
      for (int st = 0; st < S; ++st)
        if ((cut_last >> st) & 1u) {
          const bool in = mbar_drain(&tailfull[st], ((cut_ph >> st) & 1u) ^ 1u);
          if (STALL && cluster == 0 && in) atomicAdd(p.landed, 1);
        }
      loads[0] = issued;
      loads[1] = peer_units;
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (leader CTA only) ----------------
    if (leader && elect_one()) {
      const uint32_t idesc = idesc_dense(p.fmt, p.fmt, B_MN, 256, 256) | (A_MN ? 1u << 15 : 0u);
      const uint32_t empty_own = smem_u32(empty), empty_peer = mapa_shared(smem_u32(empty), 1);
      const uint32_t accfull_own = smem_u32(accfull), accfull_peer = mapa_shared(smem_u32(accfull), 1);
      int s = 0;
      uint32_t ph = 0, fixed_ph = 0;
      int local = 0;
      bool ok = true;
      [[maybe_unused]] int slab = 0;
      for (int t = cluster; t < num_tiles && ok; t += nclusters) {
        const GTile o = walk.at(t);
        const int nk = (o.k + KE - 1) / KE;
        if (nk == 0) continue;
        const int b = local & 1;
        const uint32_t aph = (local >> 1) & 1;
        ++local;
        if (!mbar_poll(&accempty[b], aph ^ 1, wc, 62)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + b * 256;
        for (int kb = 0; kb < nk; ++kb) {
          if constexpr (STALL)
            if (cluster == 0 && slab++ == p.stall && !mbar_poll(teardown, 0, wc, 67)) { ok = false; break; }
          if (!mbar_poll(&full[s], ph, wc, 63)) { ok = false; break; }
          const int left = o.k - kb * KE;
          // WGRAD: k-steps with rows of the group; else whole atoms (zeros behind K)
          int steps = 4 * kPairSub;
          if (left < KE) steps = MODE == GMode::WGRAD ? (left + 15) / 16 : (left > KA ? 8 : 4);
          if (MODE == GMode::WGRAD && slab_is_cut(left, KE)) {
            if (!mbar_wait_cluster(&fixed[s], (fixed_ph >> s) & 1u, wc, 64)) { ok = false; break; }
            fixed_ph ^= 1u << s;
          }
          tc_fence_after();
          const uint32_t aaddr = smem_u32(smem + s * kPairStageBytes);
          const uint32_t baddr = aaddr + kPairSub * kPairAtom;
          auto step = [&](int kk) {
            const int j = kk >> 2, k = kk & 3;
            const uint32_t acc = (kb > 0 || kk > 0) ? 1u : 0u;
            uint64_t adesc, bdesc;
            if constexpr (A_MN) adesc = sdesc_sw128(aaddr + j * kPairAtom + k * 16 * kSlabBytes, kBoxBytes, 1024);
            else adesc = sdesc_sw128(aaddr + j * kPairAtom + k * 32, 16, 1024);
            if constexpr (B_MN) bdesc = sdesc_sw128(baddr + j * kPairAtom + k * 16 * kSlabBytes, kBoxBytes, 1024);
            else bdesc = sdesc_sw128(baddr + j * kPairAtom + k * 32, 16, 1024);
            if constexpr (KIND == Kind::F16) umma_f16_pair(d_tmem, adesc, bdesc, idesc, acc);
            else umma_f8f6f4_pair(d_tmem, adesc, bdesc, idesc, acc);
          };
          if (steps == 4 * kPairSub) {
#pragma unroll
            for (int kk = 0; kk < 4 * kPairSub; ++kk) step(kk);
          } else {
            for (int kk = 0; kk < steps; ++kk) step(kk);
          }
          umma_commit_pair(empty_own + s * 8);
          umma_commit_pair(empty_peer + s * 8);
          if (++s == S) { s = 0; ph ^= 1; }
        }
        if (ok) {
          umma_commit_pair(accfull_own + b * 8);
          umma_commit_pair(accfull_peer + b * 8);
        }
      }
      umma_commit_pair(smem_u32(teardown));
      mbar_drain(teardown, 0);
    }
  } else if (warp < 2 + kGroupedEpiWarps) {
    // ---------------- epilogue (both CTAs) ----------------
    const int q = warp & 3, part = (warp - 2) >> 2;  // lanes of Tensor Memory, every other chunk of columns
    const uint32_t accempty_leader = mapa_shared(smem_u32(accempty), 0);
    const uint32_t stage = smem_u32(staging) + (warp - 2) * kGroupedStageBytes;
    int local = 0;
    for (int t = cluster; t < num_tiles; t += nclusters) {
      const GTile o = walk.at(t);
      if (o.k == 0) {
        grouped_epilogue<MODE, OUT>(p, o, 0, half + q * 32, part, lane, stage, [] {});
        continue;
      }
      const int b = local & 1;
      const uint32_t aph = (local >> 1) & 1;
      ++local;
      if (!mbar_wait_warp(&accfull[b], aph, wc, 65)) break;
      tc_fence_after();
      grouped_epilogue<MODE, OUT>(p, o, tmem_base + (static_cast<uint32_t>(q * 32) << 16) + b * 256, half + q * 32, part,
                                  lane, stage, [&] {
                                    tc_fence_before();
                                    __syncwarp();
                                    if (lane == 0) mbar_arrive_remote_cta(accempty_leader + b * 8);
                                  });
    }
  } else if (MODE == GMode::WGRAD) {
    // ---------------- tail (both CTAs, each its own halves) ----------------
    const uint32_t fixed_leader = mapa_shared(smem_u32(fixed), 0);
    long long issue = 0;
    uint32_t cut_ph = 0;
    for (int t = cluster; t < num_tiles; t += nclusters) {
      const GTile o = walk.at(t);
      const int nk = (o.k + KE - 1) / KE;
      const int left = o.k - (nk - 1) * KE;
      issue += nk;
      if (nk == 0 || !slab_is_cut(left, KE)) continue;
      const int s = static_cast<int>((issue - 1) % S);
      if (!mbar_wait_warp(&tailfull[s], (cut_ph >> s) & 1u, wc, 66)) break;
      cut_ph ^= 1u << s;
      const int j = left / KA, at = left - j * KA;  // atom and row of the first row behind the end
      const uint32_t base = smem_u32(smem + s * kPairStageBytes) + j * kPairAtom + at * kSlabBytes;
      const int nz = ((left + 15) & ~15) - left;
#pragma unroll
      for (int box = 0; box < 2; ++box) {
        clear_rows(base + box * kBoxBytes, nz, lane);                          // A
        clear_rows(base + kPairSub * kPairAtom + box * kBoxBytes, nz, lane);  // B
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(fixed_leader + s * 8);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) st_shared_cluster(mapa_shared(smem_u32(const_cast<int*>(peer_abort)), rank ^ 1), 1);
  __syncwarp();
  cluster_sync();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
  if (*reinterpret_cast<volatile unsigned long long*>(tmem_slot + 2) != 0) {  // both flags
    // A wait timed out in one of the CTAs: both come here. The loads of both land before either ends. They are counted on
    // the leader's full[s], which expects a slab's bytes from both CTAs as soon as the leader issues its half; where only one
    // has issued the stage's last slab, the phase is made to expect that one's bytes alone. (The two are
    // at most a slab a stage apart: the MMA thread frees no stage that lacks a half.)
    if (leader && threadIdx.x == 0) {
      const uint32_t theirs = mapa_shared(smem_u32(loads), 1);
      const uint32_t n0 = loads[0], n1 = ld_shared_cluster(theirs), units0 = loads[1], units1 = ld_shared_cluster(theirs + 4);
      for (int s = 0; s < S; ++s) {
        const uint32_t u0 = (n0 + S - 1 - s) / S, u1 = (n1 + S - 1 - s) / S;  // times that the stage was filled
        if (u1 > u0) mbar_arrive_expect_tx(&full[s], ((units1 >> (8 * s)) & 255u) * 2048);
        else if (u0 > u1 && ((units0 >> (8 * s)) & 255u)) mbar_complete_tx(&full[s], ((units0 >> (8 * s)) & 255u) * 2048);
        const uint32_t u = max(u0, u1);
        const bool in = u == 0 || mbar_drain(&full[s], (u - 1) & 1u);
        if (STALL && cluster == 0 && u > 0 && in) atomicAdd(p.landed, 256);
      }
    }
    __syncthreads();
    cluster_sync();
  }
}

}  // namespace bw
