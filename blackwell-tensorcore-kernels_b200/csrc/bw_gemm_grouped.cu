// Entry points of the products grouped by expert: argument checks, TMA descriptors, tile choice and
// launch of the kernels in bw_gemm_grouped.cuh.
#include <atomic>

#include "bw_gemm_grouped.cuh"
#include "bw_runtime.cuh"

namespace bw {
namespace {

constexpr int kMaxSmem = 232448;
constexpr int kMaxExtent = 0x7fffffff - 1024;  // tile coordinates round up and stay ints

struct Operands {  // what the tensor maps are made of
  const void* A;
  const void* B;
  long long lda, ldb;  // elements between rows of A (X) and, in WGRAD, Y
};

CUtensorMapDataType map_type(int dtype) {
  return dtype == BW_DTYPE_FP8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
         : dtype == BW_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// K atoms a stage and stages of the single-CTA kernel. Narrow tiles hold two atoms a stage: the issuing threads take about
// 450 cycles a stage, and an atom of such a tile less to load and multiply (one group of 300 x 4096 x 4096, W = 96: E4M3
// 17.5 -> 14.4 us, BF16 29.0 -> 23.2).
constexpr int atoms_a_stage(int W) { return W <= 128 ? 2 : 1; }
constexpr int stage_bytes(int W) { return atoms_a_stage(W) * (kBM + W) * kSlabBytes; }
constexpr int stages_of(int W, int groups) { return (kMaxSmem - grouped_tail_bytes(groups)) / stage_bytes(W); }
constexpr bool stages_within(int lo, int hi) {
  for (int W = 64; W <= 256; W += 16)
    if (stages_of(W, kMaxGroups) < lo || stages_of(W, 1) > hi) return false;
  return true;
}
static_assert(stages_within(3, kGroupedMaxStages) && !stages_within(4, kGroupedMaxStages) && !stages_within(3, kGroupedMaxStages - 1),
              "3 to kGroupedMaxStages stages");

// Tile rows that the output can have at most, and that it has when the rows spread evenly.
long long max_tile_rows(int rows, int groups, int tm) {
  return rows / tm + (groups < rows ? groups : rows);
}
long long even_tile_rows(int rows, int groups, int tm) {
  const long long active = groups < rows ? groups : rows;
  const long long each = (rows + active - 1) / active;
  return active * ((each + tm - 1) / tm);
}

// Tile width of the single-CTA kernel: the multiple of `gran` from 64 to 256 with the least work on the
// busiest SM, ceil(tiles / SMs) x (W + c): a tile reads W columns of B and (in c) its rows of A, and
// costs a start and an end. Ties go to the wider tile. 8 tokens' rows over 8 matrices of 4096 x 2048
// E4M3: W = 240 (144 tiles, one wave).
int tile_width(const GroupedParams& p, long long tile_rows, int gran, bool wgrad, const DeviceState& d, long long* work = nullptr) {
  const int forced = env_int("BW_GROUPED_W", 0);
  if (forced >= 64 && forced <= 256 && forced % gran == 0) return forced;
  const long long active = p.groups < p.rows ? p.groups : p.rows;
  const long long each = wgrad || active == 0 ? kBM : p.rows / active;
  const long long c = 32 + (each < kBM ? each : kBM);
  long long best = -1;
  int W = 64;
  for (int w = 64; w <= 256; w += gran) {
    const long long tiles = tile_rows * ((p.n + w - 1) / w);
    const long long cost = (tiles + d.sms - 1) / d.sms * (w + c);
    if (best < 0 || cost <= best) {
      best = cost;
      W = w;
    }
  }
  if (work) *work = best;
  return W;
}

// CTA pairs with 256 x 256 tiles where the groups have rows enough for them, and the tiles SMs enough:
// measured against the single-CTA kernel over 32 groups of 2048 x 2048, E4M3 (BF16), by rows a group on
// average: 96 35.6 / 35.3 us (62.3 / 60.7), 160 37.8 / 42.1 (64.9 / 74.2), 320 57.2 / 59.5, 640 86.8 / 96.4; weight gradient of
// 1024 x 2048: 160 44.2 / 42.5, 224 49.4 / 51.0, 640 88.4 / 98.1, and of
// 2008 x 2464, 60 groups of 187 213 / 234. One group of 4096 x 4096 E4M3: 32 tiles (512
// rows) 16.9 / 14.9 us, 64 tiles (1024 rows) 17.4 / 19.9. A weight gradient of one or two rounds of pairs takes the kernel
// with less work on the busiest SM, a pair's tile counting 354 on the scale of tile_width (256 + 160, less what it saves
// in loads): 3 groups of 4005 rows, 3992 x 336 BF16 57.0 / 40.2 us.
bool use_pair(const GroupedParams& p, bool wgrad, const DeviceState& d) {
  const int forced = env_int("BW_GROUPED_PAIR", -1);
  if (forced >= 0) return forced != 0;
  const long long active = p.groups < p.rows ? p.groups : p.rows;
  if (active == 0 || p.rows / active < (wgrad ? 160 : 144)) return false;
  const long long tm = wgrad ? p.groups * ((p.m + 255LL) / 256) : even_tile_rows(p.rows, p.groups, 256);
  const long long tiles = tm * ((p.n + 255LL) / 256), rounds = (2 * tiles + d.sms - 1) / d.sms;
  if (tiles * 5 < 2LL * d.sms) return false;
  if (!wgrad || rounds > 2) return true;
  long long single;
  tile_width(p, p.groups * ((p.m + 127LL) / 128), 64, true, d, &single);
  return rounds * 354 <= single;
}

// STALL: the self-test of the waits, on the kernel that `pair_asked` names.
template <Kind KIND, GMode MODE, Out OUT, bool STALL = false>
int launch(const Operands& o, int dtype, GroupedParams p, cudaStream_t s, const DeviceState& d, bool pair_asked = false) {
  constexpr bool wgrad = MODE == GMode::WGRAD;
  constexpr int KE = KindTraits<KIND>::kElemsPerSlab;
  const int es = dtype == BW_DTYPE_FP8 ? 1 : 2;
  const bool pair = STALL ? pair_asked : use_pair(p, wgrad, d);
  const int tm = pair ? 256 : kBM;
  const long long mt = wgrad ? static_cast<long long>(p.groups) * ((p.m + tm - 1) / tm) : even_tile_rows(p.rows, p.groups, tm);
  p.W = pair ? 256 : tile_width(p, mt, MODE == GMode::ROWS_NK ? 16 : 64, wgrad, d);
  const long long most = (wgrad ? mt : max_tile_rows(p.rows, p.groups, tm)) * ((p.n + p.W - 1) / p.W);
  if (most >= (1LL << 31) - 4096) return set_error(BW_ERR_INVALID, "grouped GEMM: %lld output tiles exceed the index range", most);
  p.sub = atoms_a_stage(p.W);
  p.stage_bytes = pair ? kPairStageBytes : stage_bytes(p.W);
  p.stages = pair ? kPairStages : stages_of(p.W, p.groups);
  const int smem = p.stages * p.stage_bytes + grouped_tail_bytes(p.groups);
  CUtensorMap ta{}, ta16{}, tb{};
  if ((wgrad ? p.rows : p.k) > 0) {
    const CUtensorMapDataType ty = map_type(dtype);
    const int b_box = pair ? 128 : p.W;  // a CTA of a pair loads its half of the tile's columns
    int r;
    if (wgrad) {
      r = make_tmap_2d(&ta, ty, o.A, p.m, p.rows, uint64_t(o.lda) * es, 64, 64);
      if (r == BW_OK) r = make_tmap_2d(&tb, ty, o.B, p.n, p.rows, uint64_t(o.ldb) * es, 64, 64);
    } else {
      r = make_tmap_2d(&ta, ty, o.A, p.k, p.rows, uint64_t(o.lda) * es, KE, kBM);
      if (r == BW_OK) r = make_tmap_2d(&ta16, ty, o.A, p.k, p.rows, uint64_t(o.lda) * es, KE, 16);
      const uint64_t matrix = uint64_t(p.k) * p.n * es;
      if (r == BW_OK)
        r = MODE == GMode::ROWS_NK ? make_tmap_3d(&tb, ty, o.B, p.k, p.n, p.groups, uint64_t(p.k) * es, matrix, KE, b_box)
                                   : make_tmap_3d(&tb, ty, o.B, p.n, p.k, p.groups, uint64_t(p.n) * es, matrix, 64, 64);
    }
    if (r != BW_OK) return r;
  }
  int dev = 0;
  BW_CUDA(cudaGetDevice(&dev));
  auto one = bw_tc_gemm_grouped_kernel<KIND, MODE, OUT, STALL>;
  auto two = bw_tc_gemm_grouped_pair_kernel<KIND, MODE, OUT, STALL>;
  static std::atomic<int> resident[64] = {};  // co-resident CTA pairs; 0: kernels not set up on this device
  int clusters = resident[dev & 63].load(std::memory_order_acquire);
  if (clusters == 0) {
    BW_CUDA(cudaFuncSetAttribute(one, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    BW_CUDA(cudaFuncSetAttribute(two, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    clusters = pair_clusters_resident(two, kGroupedThreads,
                                      kPairStages * kPairStageBytes + grouped_tail_bytes(kMaxGroups), d);
    resident[dev & 63].store(clusters, std::memory_order_release);
  }
  long long room = pair ? clusters : d.sms;
  const int cap = env_int("BW_MAX_CTAS", 0);
  if (cap > 0 && room > cap / (pair ? 2 : 1)) room = cap / (pair ? 2 : 1) > 0 ? cap / (pair ? 2 : 1) : 1;
  const int n = static_cast<int>(most < room ? most : room);
  BW_CUDA(launch_dependent(pair ? two : one, dim3(pair ? 2 * n : n), kGroupedThreads, smem, s, ta, ta16, tb, p));
  return BW_OK;
}

template <Kind KIND, GMode MODE>
int launch_out(const Operands& o, int dtype, int out_dtype, const GroupedParams& p, cudaStream_t s, const DeviceState& d) {
  if (out_dtype == BW_OUT_F32) return launch<KIND, MODE, Out::F32>(o, dtype, p, s, d);
  return launch<KIND, MODE, Out::BF16>(o, dtype, p, s, d);
}

int check_grouped(const char* name, int dtype, bool fp8, int out_dtype, const int* offsets, int groups, int rows, int a,
                  int b) {
  if (dtype != BW_DTYPE_F16 && dtype != BW_DTYPE_BF16 && !(fp8 && dtype == BW_DTYPE_FP8))
    return set_error(BW_ERR_INVALID, "%s: bad dtype %d", name, dtype);
  if (out_dtype != BW_OUT_F32 && out_dtype != BW_OUT_BF16)
    return set_error(BW_ERR_INVALID, "%s: bad out_dtype %d", name, out_dtype);
  if (rows < 0 || a < 0 || b < 0) return set_error(BW_ERR_INVALID, "%s: negative size", name);
  if (rows > kMaxExtent || a > kMaxExtent || b > kMaxExtent)
    return set_error(BW_ERR_INVALID, "%s: a size exceeds %d", name, kMaxExtent);
  if (groups < 1 || groups > kMaxGroups) return set_error(BW_ERR_INVALID, "%s: groups = %d (1..%d)", name, groups, kMaxGroups);
  if (!offsets || (reinterpret_cast<uintptr_t>(offsets) & 3u))
    return set_error(BW_ERR_INVALID, "%s: offsets is null or not aligned to an int", name);
  return BW_OK;
}

int check_operand(const char* name, const char* what, const void* p, long long ld, long long rows, int cols, int es) {
  if (!p) return set_error(BW_ERR_INVALID, "%s: %s is null", name, what);
  if (ld < cols && rows > 1) return set_error(BW_ERR_INVALID, "%s: %s's row pitch %lld is below %d", name, what, ld, cols);
  if (!aligned16(p) || (rows > 1 && ld * es % 16 != 0))
    return set_error(BW_ERR_INVALID, "%s: %s and its row pitch must be multiples of 16 bytes", name, what);
  return BW_OK;
}

// The widest store that every row of C allows.
int store_width(const void* C, long long ldc, int elem) {
  return aligned16(C) && ldc * elem % 16 == 0 ? 16 : elem;
}

GroupedParams base(const DeviceState& d, int dtype, void* C, long long ldc, int out_dtype, const int* offsets, int groups,
                   int rows) {
  GroupedParams p{};
  p.C = C;
  p.ldc = ldc;
  p.offsets = offsets;
  p.groups = groups;
  p.rows = rows;
  p.group_m = 16;
  p.vec = store_width(C, ldc, out_dtype == BW_OUT_F32 ? 4 : 2);
  p.fmt = dtype == BW_DTYPE_BF16 ? 1u : 0u;  // kind::f16: 0 FP16, 1 BF16; kind::f8f6f4: 0 E4M3
  p.status = d.status;
  p.budget_ns = wait_budget_ns();
  return p;
}

}  // namespace
}  // namespace bw

using namespace bw;

extern "C" {

int bw_gemm_grouped(int dtype, const void* A, long long lda, const void* B, int b_transposed, const int* offsets,
                    int groups, const float* row_scale, const float* group_scale, void* C, long long ldc,
                    int out_dtype, int rows, int N, int K, void* stream) {
  const char* name = "grouped GEMM";
  int r = check_grouped(name, dtype, true, out_dtype, offsets, groups, rows, N, K);
  if (r != BW_OK) return r;
  if (dtype == BW_DTYPE_FP8 && !b_transposed)
    return set_error(BW_ERR_INVALID, "%s: E4M3 takes a K-contiguous B (b_transposed)", name);
  if (rows == 0 || N == 0) return BW_OK;
  const int oe = out_dtype == BW_OUT_F32 ? 4 : 2, es = dtype == BW_DTYPE_FP8 ? 1 : 2;
  if (!C || reinterpret_cast<uintptr_t>(C) % oe) return set_error(BW_ERR_INVALID, "%s: C is null or not aligned to its element", name);
  if (rows > 1 && ldc < N) return set_error(BW_ERR_INVALID, "%s: C's row pitch %lld is below N = %d", name, ldc, N);
  if (((reinterpret_cast<uintptr_t>(row_scale) | reinterpret_cast<uintptr_t>(group_scale)) & 3u))
    return set_error(BW_ERR_INVALID, "%s: scales are not aligned to a float", name);
  if (C == A || C == B) return set_error(BW_ERR_INVALID, "%s: C over an operand", name);
  if (rows == 1) { lda = (K + 15LL) / 16 * 16; ldc = ldc < N ? N : ldc; }  // a single row has no pitch
  if (K > 0) {
    if ((r = check_operand(name, "A", A, lda, rows, K, es)) != BW_OK) return r;
    const int inner = b_transposed ? K : N;
    if ((r = check_operand(name, "B", B, inner, 2, inner, es)) != BW_OK) return r;
  }
  DeviceState* d;
  if ((r = ensure_device(&d)) != BW_OK) return r;
  GroupedParams p = base(*d, dtype, C, ldc, out_dtype, offsets, groups, rows);
  p.row_scale = row_scale;
  p.group_scale = group_scale;
  p.n = N;
  p.k = K;
  const Operands o{A, B, lda, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BW_DTYPE_FP8) return launch_out<Kind::F8, GMode::ROWS_NK>(o, dtype, out_dtype, p, s, *d);
  if (b_transposed) return launch_out<Kind::F16, GMode::ROWS_NK>(o, dtype, out_dtype, p, s, *d);
  return launch_out<Kind::F16, GMode::ROWS_KN>(o, dtype, out_dtype, p, s, *d);
}

int bw_gemm_grouped_wgrad(int dtype, const void* X, long long ldx, const void* Y, long long ldy, const int* offsets,
                          int groups, void* D, int out_dtype, int rows, int M, int N, void* stream) {
  const char* name = "grouped weight gradient";
  int r = check_grouped(name, dtype, false, out_dtype, offsets, groups, rows, M, N);
  if (r != BW_OK) return r;
  if (M == 0 || N == 0) return BW_OK;
  const int oe = out_dtype == BW_OUT_F32 ? 4 : 2;
  if (!D || reinterpret_cast<uintptr_t>(D) % oe) return set_error(BW_ERR_INVALID, "%s: D is null or not aligned to its element", name);
  if (D == X || D == Y) return set_error(BW_ERR_INVALID, "%s: D over an operand", name);
  if (rows == 1) { ldx = (M + 7LL) / 8 * 8; ldy = (N + 7LL) / 8 * 8; }
  if (rows > 0 && ((r = check_operand(name, "X", X, ldx, rows, M, 2)) != BW_OK ||
                   (r = check_operand(name, "Y", Y, ldy, rows, N, 2)) != BW_OK))
    return r;
  DeviceState* d;
  if ((r = ensure_device(&d)) != BW_OK) return r;
  GroupedParams p = base(*d, dtype, D, N, out_dtype, offsets, groups, rows);
  p.m = M;
  p.n = N;
  const Operands o{X, Y, ldx, ldy};
  return launch_out<Kind::F16, GMode::WGRAD>(o, dtype, out_dtype, p, static_cast<cudaStream_t>(stream), *d);
}

int bw_selftest_grouped_wait(int pair, int wgrad, const void* A, const void* B, const int* offsets, int groups, void* C,
                             int rows, int N, int K, int stall, int stop_leader, int stop_peer,
                             unsigned long long budget_ns, int* landed, void* stream) {
  const char* name = "self-test of the grouped products";
  int r = check_grouped(name, BW_DTYPE_BF16, false, BW_OUT_BF16, offsets, groups, rows, N, K);
  if (r != BW_OK) return r;
  if (budget_ns == 0 || budget_ns > 1000000000ull) return set_error(BW_ERR_INVALID, "%s: budget must be in (0, 1 s]", name);
  if (stall < 0 || stop_leader < 0 || stop_peer < 0) return set_error(BW_ERR_INVALID, "%s: negative slab", name);
  if (rows == 0 || N == 0 || K == 0 || !C || !landed || !aligned16(C))
    return set_error(BW_ERR_INVALID, "%s: empty size, or C or landed is null or not aligned", name);
  if ((r = check_operand(name, "A", A, wgrad ? N : K, 2, wgrad ? N : K, 2)) != BW_OK || (r = check_operand(name, "B", B, K, 2, K, 2)) != BW_OK)
    return r;
  DeviceState* d;
  if ((r = ensure_device(&d)) != BW_OK) return r;
  GroupedParams p = base(*d, BW_DTYPE_BF16, C, wgrad ? K : N, BW_OUT_BF16, offsets, groups, rows);
  (wgrad ? p.m : p.n) = N;
  (wgrad ? p.n : p.k) = K;
  p.budget_ns = budget_ns;
  p.stall = stall;
  p.stop[0] = stop_leader;
  p.stop[1] = stop_peer;
  p.landed = landed;
  const Operands o{A, B, wgrad ? N : K, K};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  r = wgrad ? launch<Kind::F16, GMode::WGRAD, Out::BF16, true>(o, BW_DTYPE_BF16, p, s, *d, pair != 0)
            : launch<Kind::F16, GMode::ROWS_NK, Out::BF16, true>(o, BW_DTYPE_BF16, p, s, *d, pair != 0);
  if (r != BW_OK) return r;
  int st = 0;
  return bw_device_status(stream, &st);
}

}  // extern "C"
