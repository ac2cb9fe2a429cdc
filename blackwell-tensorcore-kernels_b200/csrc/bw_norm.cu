// Root-mean-square norm in front of a low-precision product, and its gradient.
//
//   h    = x + residual                      held in x's type: what the next layer and the gradient read
//   rstd = (mean_j h_j^2 + eps)^(-1/2)
//   y_j  = h_j w_j rstd                      written in x's type, or as E4M3 with one scale a row:
//   s    = max_j |y_j| / 448,  q_j = e4m3(y_j * (448 / max))      (s = 1 where the maximum is 0 or not finite)
//
// and for the gradient, with n = h rstd:
//   dx_j = rstd (dy_j w_j - n_j mean_i(dy_i w_i n_i)) + dresidual_j,      dw_j = sum over rows of dy_j n_j
//
// Both are bound by memory: every input is read once and every output written once. A row stays
// in registers (packed in its own type: h is rounded to it anyway) between its reduction and its
// output. max |y| needs no second reduction: y_j = (h_j w_j) rstd and rounding is monotonic, so
// max |y| = max |h w| * rstd exactly, and both sums travel through one reduction. Statistics and
// sums are FP32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>

#include "bw_runtime.cuh"

namespace bw {
namespace {

constexpr float kE4m3Max = 448.f;

// ------------------------------------------------------------------ element access
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VE consecutive elements, moved as one access of VE * sizeof(T) bytes.
template <typename T, int VE>
struct alignas(sizeof(T) * VE) Pack {
  T v[VE];
};
template <int BYTES>
struct RawOf;
template <> struct RawOf<1> { using type = uint8_t; };
template <> struct RawOf<2> { using type = uint16_t; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };
template <typename T, int VE>
__device__ __forceinline__ Pack<T, VE> load_pack(const T* p) {
  using Raw = typename RawOf<sizeof(T) * VE>::type;
  const Raw raw = *reinterpret_cast<const Raw*>(p);
  Pack<T, VE> v;
  __builtin_memcpy(&v, &raw, sizeof(v));
  return v;
}
template <typename T, int VE>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VE>& v) {
  using Raw = typename RawOf<sizeof(T) * VE>::type;
  Raw raw;
  __builtin_memcpy(&raw, &v, sizeof(v));
  *reinterpret_cast<Raw*>(p) = raw;
}

// VE weights from column c, of x's type or FP32.
template <typename T, int VE>
__device__ __forceinline__ void load_weight(const void* w, int w_f32, long long c, float (&out)[VE]) {
  if (w_f32) {
    constexpr int F = VE < 4 ? VE : 4;
#pragma unroll
    for (int i = 0; i < VE / F; ++i) {
      const Pack<float, F> f = load_pack<float, F>(static_cast<const float*>(w) + c + F * i);
#pragma unroll
      for (int j = 0; j < F; ++j) out[F * i + j] = f.v[j];
    }
  } else {
    const Pack<T, VE> f = load_pack<T, VE>(static_cast<const T*>(w) + c);
#pragma unroll
    for (int j = 0; j < VE; ++j) out[j] = to_f32(f.v[j]);
  }
}

// Reduction over the `tpr` threads of a row: part of a warp (tpr <= 32), or the whole block.
// `slot` alternates between two halves of `sm`, so one barrier a call is enough.
struct SumMax {
  float sum, max;
};
__device__ __forceinline__ SumMax reduce_row(SumMax v, int tpr, SumMax* sm) {
  for (int o = (tpr < 32 ? tpr : 32) / 2; o > 0; o >>= 1) {
    v.sum += __shfl_xor_sync(0xffffffffu, v.sum, o);
    v.max = fmaxf(v.max, __shfl_xor_sync(0xffffffffu, v.max, o));
  }
  if (tpr > 32) {
    const int warps = tpr >> 5;
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sm[(threadIdx.x & 31) % warps];  // warps is a power of two: every lane ends with the whole
    for (int o = warps / 2; o > 0; o >>= 1) {
      v.sum += __shfl_xor_sync(0xffffffffu, v.sum, o);
      v.max = fmaxf(v.max, __shfl_xor_sync(0xffffffffu, v.max, o));
    }
  }
  return v;
}

struct NormParams {
  const void* x;
  const void* res;     // or null
  const void* w;
  int w_f32;
  void* h;             // or null
  void* y;             // T, or E4M3 bytes
  float* row_scale;    // E4M3 only
  float* rstd;         // or null
  long long ldx, ldr, ldh, ldy;  // row pitches in elements
  long long rows;
  int cols;
  float eps;
};

// Scale of an E4M3 row by its maximum, and the factor that quantises it. A maximum so small that
// 448 / max overflows counts as zero.
__device__ __forceinline__ void e4m3_row_scale(float amax, float& mul, float& s) {
  mul = 1.f;
  s = 1.f;
  if (amax > 0.f && amax < INFINITY) {
    const float m = kE4m3Max / amax;
    if (m < INFINITY) {
      mul = m;
      s = amax / kE4m3Max;
    }
  }
}

template <int VE>
__device__ __forceinline__ Pack<uint8_t, VE> encode_e4m3(const float (&y)[VE], float mul) {
  Pack<uint8_t, VE> q;
  if constexpr (VE % 2 == 0) {
#pragma unroll
    for (int j = 0; j < VE; j += 2) {
      const __nv_fp8x2_storage_t two =
          __nv_cvt_float2_to_fp8x2(make_float2(y[j] * mul, y[j + 1] * mul), __NV_SATFINITE, __NV_E4M3);
      q.v[j] = static_cast<uint8_t>(two & 0xff);
      q.v[j + 1] = static_cast<uint8_t>(two >> 8);
    }
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j) q.v[j] = static_cast<uint8_t>(__nv_cvt_float_to_fp8(y[j] * mul, __NV_SATFINITE, __NV_E4M3));
  }
  return q;
}

template <typename T, bool Q8, int VE>
__device__ __forceinline__ void write_out(const NormParams& p, long long row, long long c, const Pack<T, VE>& h,
                                          float rstd, float mul) {
  float w[VE], y[VE];
  load_weight<T, VE>(p.w, p.w_f32, c, w);
#pragma unroll
  for (int j = 0; j < VE; ++j) y[j] = to_f32(h.v[j]) * w[j] * rstd;
  if constexpr (Q8) {
    store_pack<uint8_t, VE>(static_cast<uint8_t*>(p.y) + row * p.ldy + c, encode_e4m3<VE>(y, mul));
  } else {
    Pack<T, VE> o;
#pragma unroll
    for (int j = 0; j < VE; ++j) o.v[j] = from_f32<T>(y[j]);
    store_pack<T, VE>(static_cast<T*>(p.y) + row * p.ldy + c, o);
  }
}

// h of one vector: x, or x + residual rounded to T and stored.
template <typename T, int VE>
__device__ __forceinline__ void add_residual(Pack<T, VE>& h, const Pack<T, VE>& r) {
#pragma unroll
  for (int j = 0; j < VE; ++j) h.v[j] = from_f32<T>(to_f32(h.v[j]) + to_f32(r.v[j]));
}

template <typename T, bool Q8, int VE>
__device__ __forceinline__ void accumulate(const NormParams& p, long long c, const Pack<T, VE>& h, SumMax& a) {
  float w[VE];
  if constexpr (Q8) load_weight<T, VE>(p.w, p.w_f32, c, w);
#pragma unroll
  for (int j = 0; j < VE; ++j) {
    const float v = to_f32(h.v[j]);
    a.sum = fmaf(v, v, a.sum);
    if constexpr (Q8) a.max = fmaxf(a.max, fabsf(v * w[j]));
  }
}

template <bool Q8>
__device__ __forceinline__ float finish_row(const NormParams& p, long long row, const SumMax& a, bool first,
                                            float& mul) {
  const float rstd = 1.f / sqrtf(a.sum / static_cast<float>(p.cols) + p.eps);
  mul = 1.f;
  float s = 1.f;
  if constexpr (Q8) e4m3_row_scale(a.max * rstd, mul, s);
  if (first) {
    if (p.rstd) p.rstd[row] = rstd;
    if constexpr (Q8) p.row_scale[row] = s;
  }
  return rstd;
}

// tpr threads a row (a power of two), NV vectors of VE elements a thread: the row is read once
// and kept. blockDim.x = tpr for tpr > 32, else a block holds blockDim.x / tpr rows.
template <typename T, bool Q8, int VE, int NV>
__global__ void __launch_bounds__(1024) k_rmsnorm(const NormParams p, int tpr) {
  __shared__ SumMax sm[32];
  const int t = threadIdx.x & (tpr - 1);
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x / tpr) + threadIdx.x / tpr;
  const bool live = row < p.rows;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* r = p.res ? static_cast<const T*>(p.res) + row * p.ldr : nullptr;
  Pack<T, VE> h[NV], res[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + t) * VE;
    if (live && c < p.cols) h[i] = load_pack<T, VE>(x + c);
  }
  if (r) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VE;
      if (live && c < p.cols) res[i] = load_pack<T, VE>(r + c);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VE;
      if (live && c < p.cols) add_residual<T, VE>(h[i], res[i]);
    }
  }
  SumMax a{0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + t) * VE;
    if (!live || c >= p.cols) continue;
    if (p.h) store_pack<T, VE>(static_cast<T*>(p.h) + row * p.ldh + c, h[i]);
    accumulate<T, Q8, VE>(p, c, h[i], a);
  }
  a = reduce_row(a, tpr, sm);
  if (!live) return;
  float mul;
  const float rstd = finish_row<Q8>(p, row, a, t == 0, mul);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + t) * VE;
    if (c < p.cols) write_out<T, Q8, VE>(p, row, c, h[i], rstd, mul);
  }
}

// Rows too long for the registers of one block: one block a row, which reads its row twice (the
// second time from L2).
template <typename T, bool Q8, int VE>
__global__ void __launch_bounds__(1024) k_rmsnorm_wide(const NormParams p) {
  __shared__ SumMax sm[32];
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* r = p.res ? static_cast<const T*>(p.res) + row * p.ldr : nullptr;
  T* hr = p.h ? static_cast<T*>(p.h) + row * p.ldh : nullptr;
  SumMax a{0.f, 0.f};
  for (long long c = static_cast<long long>(threadIdx.x) * VE; c < p.cols; c += 1024LL * VE) {
    Pack<T, VE> h = load_pack<T, VE>(x + c);
    if (r) add_residual<T, VE>(h, load_pack<T, VE>(r + c));
    if (hr) store_pack<T, VE>(hr + c, h);
    accumulate<T, Q8, VE>(p, c, h, a);
  }
  a = reduce_row(a, 1024, sm);
  float mul;
  const float rstd = finish_row<Q8>(p, row, a, threadIdx.x == 0, mul);
  for (long long c = static_cast<long long>(threadIdx.x) * VE; c < p.cols; c += 1024LL * VE) {
    // this thread wrote h[c] itself; where h is not kept, the sum is taken again. x and the
    // residual still hold their values then: h and y are written at this thread's own columns,
    // and a column's y after its last read.
    Pack<T, VE> h;
    if (hr) {
      h = load_pack<T, VE>(hr + c);
    } else {
      h = load_pack<T, VE>(x + c);
      if (r) add_residual<T, VE>(h, load_pack<T, VE>(r + c));
    }
    write_out<T, Q8, VE>(p, row, c, h, rstd, mul);
  }
}

// ------------------------------------------------------------------ gradient
struct NormGradParams {
  const void* dy;
  const void* h;
  const void* w;
  int w_f32;
  const float* rstd;
  const void* dres;    // or null
  void* dx;
  float* partial;      // [slabs][cols], summed into dw by k_sum_slabs
  long long lddy, ldh, lddr, lddx;
  long long rows;
  int cols;
  int slabs;           // blocks (each adds up the rows it takes)
};

// A block takes row groups blockIdx.x, + gridDim.x, ...; each thread keeps the weight gradient of
// its own columns in registers over all of them.
template <int VE>
constexpr int kGradThreads = VE == 1 ? 1024 : 512;  // 64 / 128 registers a thread
template <typename T, int VE>
constexpr int kGradMaxNv = VE == 1 ? 16 : sizeof(T) == 4 ? 8 : 4;
template <typename T, int VE, int NV>
__global__ void __launch_bounds__(kGradThreads<VE>) k_rmsnorm_grad(const NormGradParams p, int tpr) {
  __shared__ SumMax sm[2][32];
  extern __shared__ float cols_sum[];  // tpr <= 32: [row of the block][cols]
  const int t = threadIdx.x & (tpr - 1);
  const int per_block = blockDim.x / tpr, mine = threadIdx.x / tpr;
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  float dw[NV][VE];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) dw[i][j] = 0.f;
  int half = 0;
  for (long long r0 = static_cast<long long>(blockIdx.x) * per_block; r0 < p.rows;
       r0 += static_cast<long long>(gridDim.x) * per_block) {
    const long long row = r0 + mine;
    const bool live = row < p.rows;
    const T* dyr = static_cast<const T*>(p.dy) + row * p.lddy;
    const T* hr = static_cast<const T*>(p.h) + row * p.ldh;
    Pack<T, VE> dy[NV], h[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VE;
      if (live && c < p.cols) {
        dy[i] = load_pack<T, VE>(dyr + c);
        h[i] = load_pack<T, VE>(hr + c);
      }
    }
    const float rstd = live ? p.rstd[row] : 0.f;
    SumMax a{0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VE;
      if (!live || c >= p.cols) continue;
      float w[VE];
      load_weight<T, VE>(p.w, p.w_f32, c, w);
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float n = to_f32(h[i].v[j]) * rstd, d = to_f32(dy[i].v[j]);
        a.sum = fmaf(d * w[j], n, a.sum);
        dw[i][j] = fmaf(d, n, dw[i][j]);
      }
    }
    a = reduce_row(a, tpr, sm[half]);
    half ^= 1;
    const float mean = a.sum * inv_cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VE;
      if (!live || c >= p.cols) continue;
      float w[VE];
      load_weight<T, VE>(p.w, p.w_f32, c, w);
      Pack<T, VE> o, dr;
      if (p.dres) dr = load_pack<T, VE>(static_cast<const T*>(p.dres) + row * p.lddr + c);
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float n = to_f32(h[i].v[j]) * rstd;
        float g = rstd * (to_f32(dy[i].v[j]) * w[j] - n * mean);
        if (p.dres) g += to_f32(dr.v[j]);
        o.v[j] = from_f32<T>(g);
      }
      store_pack<T, VE>(static_cast<T*>(p.dx) + row * p.lddx + c, o);
    }
  }
  float* out = p.partial + static_cast<long long>(blockIdx.x) * p.cols;
  if (tpr > 32) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VE;
      if (c >= p.cols) continue;
#pragma unroll
      for (int j = 0; j < VE; ++j) out[c + j] = dw[i][j];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + t) * VE;
    if (c >= p.cols) continue;
#pragma unroll
    for (int j = 0; j < VE; ++j) cols_sum[mine * p.cols + c + j] = dw[i][j];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    float s = 0.f;
    for (int g = 0; g < per_block; ++g) s += cols_sum[g * p.cols + c];
    out[c] = s;
  }
}

// Rows too long for registers: dx with the row read twice, and the weight gradient's slabs by
// columns in a kernel of their own.
template <typename T>
__global__ void __launch_bounds__(1024) k_rmsnorm_grad_wide(const NormGradParams p) {
  __shared__ SumMax sm[32];
  const long long row = blockIdx.x;
  const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
  const T* h = static_cast<const T*>(p.h) + row * p.ldh;
  const float rstd = p.rstd[row];
  SumMax a{0.f, 0.f};
  for (long long c = threadIdx.x; c < p.cols; c += 1024) {
    float w[1];
    load_weight<T, 1>(p.w, p.w_f32, c, w);
    a.sum = fmaf(to_f32(dy[c]) * w[0], to_f32(h[c]) * rstd, a.sum);
  }
  a = reduce_row(a, 1024, sm);
  const float mean = a.sum / static_cast<float>(p.cols);
  for (long long c = threadIdx.x; c < p.cols; c += 1024) {
    float w[1];
    load_weight<T, 1>(p.w, p.w_f32, c, w);
    float g = rstd * (to_f32(dy[c]) * w[0] - to_f32(h[c]) * rstd * mean);
    if (p.dres) g += to_f32(static_cast<const T*>(p.dres)[row * p.lddr + c]);
    static_cast<T*>(p.dx)[row * p.lddx + c] = from_f32<T>(g);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) k_rmsnorm_dw_wide(const NormGradParams p) {
  const long long c = blockIdx.x * 256LL + threadIdx.x;
  if (c >= p.cols) return;
  for (int slab = blockIdx.y; slab < p.slabs; slab += gridDim.y) {
    float s = 0.f;
    for (long long row = slab; row < p.rows; row += p.slabs)
      s = fmaf(to_f32(static_cast<const T*>(p.dy)[row * p.lddy + c]),
               to_f32(static_cast<const T*>(p.h)[row * p.ldh + c]) * p.rstd[row], s);
    p.partial[static_cast<long long>(slab) * p.cols + c] = s;
  }
}

// dw[c] = sum over slabs in a fixed order: 32 columns a block, 32 warps over the slabs.
__global__ void __launch_bounds__(1024) k_sum_slabs(const float* __restrict__ partial, float* __restrict__ dw,
                                                    int slabs, int cols) {
  __shared__ float sm[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long c = blockIdx.x * 32LL + lane;
  float s = 0.f;
  if (c < cols)
    for (int i = warp; i < slabs; i += 32) s += partial[static_cast<long long>(i) * cols + c];
  sm[warp][lane] = s;
  __syncthreads();
  s = sm[lane][warp];  // column blockIdx.x * 32 + warp, partial sum `lane`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const long long cw = blockIdx.x * 32LL + warp;
  if (lane == 0 && cw < cols) dw[cw] = s;
}

// ------------------------------------------------------------------ launch shapes
int elem_bytes(int dtype) { return dtype == BW_DTYPE_F32 ? 4 : 2; }

bool norm_dtype_ok(int dtype) { return dtype == BW_DTYPE_F32 || dtype == BW_DTYPE_F16 || dtype == BW_DTYPE_BF16; }

bool multiple_of(const void* p, long long ld, int elem, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && (ld * elem) % bytes == 0;
}

struct Shape {
  int tpr, nv;  // nv = 0: too long for registers
};

// Threads a row and vectors a thread: NV vectors a thread where there are rows enough to fill the
// GPU, more threads and fewer vectors otherwise (each load waits once, so a short chain per thread).
Shape row_shape(long long rows, int cols, int ve, int max_tpr, int max_nv) {
  const long long nvec = (static_cast<long long>(cols) + ve - 1) / ve;
  const int want = rows >= 1024 ? 4 : 1;
  int tpr = 1;
  while (tpr < max_tpr && static_cast<long long>(tpr) * want < nvec) tpr *= 2;
  int nv = 1;
  while (nv <= max_nv && static_cast<long long>(nv) * tpr < nvec) nv *= 2;
  if (nv > max_nv) nv = 0;
  return {tpr, nv};
}

template <typename T, bool Q8, int VE>
int launch_norm(const NormParams& p, cudaStream_t s) {
  const Shape sh = row_shape(p.rows, p.cols, VE, 1024, VE == 1 ? 8 : 4);
  const int block = sh.tpr > 32 ? sh.tpr : 256;
  const long long per = block / sh.tpr;
  const long long grid = (p.rows + per - 1) / per;
  if (sh.nv == 0) {
    k_rmsnorm_wide<T, Q8, VE><<<static_cast<unsigned>(p.rows), 1024, 0, s>>>(p);
  } else {
    const unsigned g = static_cast<unsigned>(grid);
    switch (sh.nv) {
      case 1: k_rmsnorm<T, Q8, VE, 1><<<g, block, 0, s>>>(p, sh.tpr); break;
      case 2: k_rmsnorm<T, Q8, VE, 2><<<g, block, 0, s>>>(p, sh.tpr); break;
      case 4: k_rmsnorm<T, Q8, VE, 4><<<g, block, 0, s>>>(p, sh.tpr); break;
      default:
        if constexpr (VE == 1) k_rmsnorm<T, Q8, 1, 8><<<g, block, 0, s>>>(p, sh.tpr);
        break;
    }
  }
  BW_CUDA(cudaGetLastError());
  return BW_OK;
}

template <typename T, bool Q8>
int dispatch_norm(const NormParams& p, cudaStream_t s) {
  constexpr int VE = 16 / sizeof(T);
  const int e = sizeof(T);
  // 16-byte vectors need every row of every tensor to start on its vector's boundary
  const bool vec = p.cols % VE == 0 && multiple_of(p.x, p.ldx, e, 16) && (!p.res || multiple_of(p.res, p.ldr, e, 16)) &&
                   (!p.h || multiple_of(p.h, p.ldh, e, 16)) && multiple_of(p.y, p.ldy, Q8 ? 1 : e, Q8 ? VE : 16) &&
                   multiple_of(p.w, 0, 1, 16);
  return vec ? launch_norm<T, Q8, VE>(p, s) : launch_norm<T, Q8, 1>(p, s);
}

int check_pitch(const char* what, long long ld, long long rows, int cols) {
  if (rows > 1 && ld < cols) return set_error(BW_ERR_INVALID, "%s: row pitch %lld is below cols = %d", what, ld, cols);
  return BW_OK;
}

int check_ptr(const char* what, const void* p, int align) {
  if (!p) return set_error(BW_ERR_INVALID, "%s is null", what);
  if (reinterpret_cast<uintptr_t>(p) % align) return set_error(BW_ERR_INVALID, "%s is not aligned to its element", what);
  return BW_OK;
}

int check_norm_common(int dtype, int weight_dtype, int rows, int cols) {
  if (!norm_dtype_ok(dtype)) return set_error(BW_ERR_INVALID, "rmsnorm takes F32, F16 or BF16 (dtype %d)", dtype);
  if (weight_dtype != dtype && weight_dtype != BW_DTYPE_F32)
    return set_error(BW_ERR_INVALID, "rmsnorm weight has x's type or F32 (weight_dtype %d)", weight_dtype);
  if (rows < 0 || cols < 0) return set_error(BW_ERR_INVALID, "negative size rows=%d cols=%d", rows, cols);
  if (rows > 0 && cols == 0) return set_error(BW_ERR_INVALID, "rmsnorm of rows without elements");
  return BW_OK;
}

int norm_impl(const void* x, long long ldx, const void* residual, long long ldr, const void* weight, int dtype,
              int weight_dtype, float eps, bool q8, void* y, long long ldy, float* row_scale, void* h, long long ldh,
              float* rstd, int rows, int cols, void* stream) {
  int r = check_norm_common(dtype, weight_dtype, rows, cols);
  if (r != BW_OK) return r;
  if (!(eps >= 0.f) || std::isinf(eps)) return set_error(BW_ERR_INVALID, "eps must be finite and not negative");
  if (rows == 0) return BW_OK;
  const int e = elem_bytes(dtype);
  if ((r = check_ptr("x", x, e)) != BW_OK || (r = check_ptr("weight", weight, elem_bytes(weight_dtype))) != BW_OK ||
      (r = check_ptr(q8 ? "q" : "y", y, q8 ? 1 : e)) != BW_OK)
    return r;
  if (residual && (r = check_ptr("residual", residual, e)) != BW_OK) return r;
  if (h && (r = check_ptr("h", h, e)) != BW_OK) return r;
  if (q8 && (r = check_ptr("row_scale", row_scale, 4)) != BW_OK) return r;
  if (rstd && (r = check_ptr("rstd", rstd, 4)) != BW_OK) return r;
  if ((r = check_pitch("x", ldx, rows, cols)) != BW_OK || (r = check_pitch(q8 ? "q" : "y", ldy, rows, cols)) != BW_OK)
    return r;
  if (residual && (r = check_pitch("residual", ldr, rows, cols)) != BW_OK) return r;
  if (h && (r = check_pitch("h", ldh, rows, cols)) != BW_OK) return r;
  DeviceState* d;
  if ((r = ensure_device(&d)) != BW_OK) return r;
  NormParams p{};
  p.x = x;
  p.res = residual;
  p.w = weight;
  p.w_f32 = weight_dtype == BW_DTYPE_F32;
  p.h = h;
  p.y = y;
  p.row_scale = row_scale;
  p.rstd = rstd;
  p.ldx = ldx;
  p.ldr = ldr;
  p.ldh = ldh;
  p.ldy = ldy;
  p.rows = rows;
  p.cols = cols;
  p.eps = eps;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BW_DTYPE_F32) return q8 ? dispatch_norm<float, true>(p, s) : dispatch_norm<float, false>(p, s);
  if (dtype == BW_DTYPE_F16) return q8 ? dispatch_norm<__half, true>(p, s) : dispatch_norm<__half, false>(p, s);
  return q8 ? dispatch_norm<__nv_bfloat16, true>(p, s) : dispatch_norm<__nv_bfloat16, false>(p, s);
}

// Slabs of the weight gradient: a function of the sizes alone, so that the sums (and the
// workspace) are the same on every device.
constexpr int kMaxSlabs = 296;
int grad_slabs(long long rows) { return static_cast<int>(rows < kMaxSlabs ? rows : kMaxSlabs); }

template <typename T, int VE>
int launch_grad(NormGradParams p, float* dw, cudaStream_t s) {
  const Shape sh = row_shape(p.rows, p.cols, VE, kGradThreads<VE>, kGradMaxNv<T, VE>);
  if (sh.nv == 0) {
    // the weight gradient first: dx may be written over dy or h
    k_rmsnorm_dw_wide<T><<<dim3(static_cast<unsigned>((p.cols + 255LL) / 256), p.slabs), 256, 0, s>>>(p);
    BW_CUDA(cudaGetLastError());
    k_rmsnorm_grad_wide<T><<<static_cast<unsigned>(p.rows), 1024, 0, s>>>(p);
  } else {
    const int block = sh.tpr > 32 ? sh.tpr : 256;
    const long long per = block / sh.tpr;
    const long long groups = (p.rows + per - 1) / per;
    if (groups < p.slabs) p.slabs = static_cast<int>(groups);
    const size_t smem = sh.tpr > 32 ? 0 : static_cast<size_t>(per) * p.cols * sizeof(float);
    switch (sh.nv) {
      case 1: k_rmsnorm_grad<T, VE, 1><<<p.slabs, block, smem, s>>>(p, sh.tpr); break;
      case 2: k_rmsnorm_grad<T, VE, 2><<<p.slabs, block, smem, s>>>(p, sh.tpr); break;
      case 4: k_rmsnorm_grad<T, VE, 4><<<p.slabs, block, smem, s>>>(p, sh.tpr); break;
      case 8:
        if constexpr (kGradMaxNv<T, VE> >= 8) k_rmsnorm_grad<T, VE, 8><<<p.slabs, block, smem, s>>>(p, sh.tpr);
        break;
      default:
        if constexpr (kGradMaxNv<T, VE> >= 16) k_rmsnorm_grad<T, VE, 16><<<p.slabs, block, smem, s>>>(p, sh.tpr);
        break;
    }
  }
  BW_CUDA(cudaGetLastError());
  k_sum_slabs<<<static_cast<unsigned>((p.cols + 31LL) / 32), 1024, 0, s>>>(p.partial, dw, p.slabs, p.cols);
  BW_CUDA(cudaGetLastError());
  return BW_OK;
}

template <typename T>
int dispatch_grad(const NormGradParams& p, float* dw, cudaStream_t s) {
  constexpr int VE = 16 / sizeof(T);
  const int e = sizeof(T);
  const bool vec = p.cols % VE == 0 && multiple_of(p.dy, p.lddy, e, 16) && multiple_of(p.h, p.ldh, e, 16) &&
                   (!p.dres || multiple_of(p.dres, p.lddr, e, 16)) && multiple_of(p.dx, p.lddx, e, 16) &&
                   multiple_of(p.w, 0, 1, 16);
  return vec ? launch_grad<T, VE>(p, dw, s) : launch_grad<T, 1>(p, dw, s);
}

}  // namespace
}  // namespace bw

using namespace bw;

extern "C" {

int bw_rmsnorm(const void* x, long long ldx, const void* residual, long long ldr, const void* weight, int dtype,
               int weight_dtype, float eps, void* y, long long ldy, void* h, long long ldh, float* rstd, int rows,
               int cols, void* stream) {
  return norm_impl(x, ldx, residual, ldr, weight, dtype, weight_dtype, eps, false, y, ldy, nullptr, h, ldh, rstd, rows,
                   cols, stream);
}

int bw_rmsnorm_fp8(const void* x, long long ldx, const void* residual, long long ldr, const void* weight, int dtype,
                   int weight_dtype, float eps, uint8_t* q, long long ldq, float* row_scale, void* h, long long ldh,
                   float* rstd, int rows, int cols, void* stream) {
  return norm_impl(x, ldx, residual, ldr, weight, dtype, weight_dtype, eps, true, q, ldq, row_scale, h, ldh, rstd, rows,
                   cols, stream);
}

size_t bw_rmsnorm_backward_workspace(int rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return static_cast<size_t>(grad_slabs(rows)) * cols * sizeof(float);
}

int bw_rmsnorm_backward(const void* dy, long long lddy, const void* h, long long ldh, const void* weight, int dtype,
                        int weight_dtype, const float* rstd, const void* dresidual, long long lddr, void* dx,
                        long long lddx, float* dweight, void* workspace, size_t workspace_bytes, int rows, int cols,
                        void* stream) {
  int r = check_norm_common(dtype, weight_dtype, rows, cols);
  if (r != BW_OK) return r;
  if (cols == 0) return BW_OK;
  if ((r = check_ptr("dweight", dweight, 4)) != BW_OK) return r;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DeviceState* d;
  if (rows == 0) {
    if ((r = ensure_device(&d)) != BW_OK) return r;
    BW_CUDA(cudaMemsetAsync(dweight, 0, sizeof(float) * static_cast<size_t>(cols), s));
    return BW_OK;
  }
  const int e = elem_bytes(dtype);
  if ((r = check_ptr("dy", dy, e)) != BW_OK || (r = check_ptr("h", h, e)) != BW_OK ||
      (r = check_ptr("weight", weight, elem_bytes(weight_dtype))) != BW_OK ||
      (r = check_ptr("rstd", rstd, 4)) != BW_OK || (r = check_ptr("dx", dx, e)) != BW_OK ||
      (r = check_ptr("workspace", workspace, 4)) != BW_OK)
    return r;
  if (dresidual && (r = check_ptr("dresidual", dresidual, e)) != BW_OK) return r;
  if ((r = check_pitch("dy", lddy, rows, cols)) != BW_OK || (r = check_pitch("h", ldh, rows, cols)) != BW_OK ||
      (r = check_pitch("dx", lddx, rows, cols)) != BW_OK)
    return r;
  if (dresidual && (r = check_pitch("dresidual", lddr, rows, cols)) != BW_OK) return r;
  const size_t need = bw_rmsnorm_backward_workspace(rows, cols);
  if (workspace_bytes < need)
    return set_error(BW_ERR_INVALID, "workspace holds %zu bytes, rmsnorm backward needs %zu", workspace_bytes, need);
  if ((r = ensure_device(&d)) != BW_OK) return r;
  NormGradParams p{};
  p.dy = dy;
  p.h = h;
  p.w = weight;
  p.w_f32 = weight_dtype == BW_DTYPE_F32;
  p.rstd = rstd;
  p.dres = dresidual;
  p.dx = dx;
  p.partial = static_cast<float*>(workspace);
  p.lddy = lddy;
  p.ldh = ldh;
  p.lddr = lddr;
  p.lddx = lddx;
  p.rows = rows;
  p.cols = cols;
  p.slabs = grad_slabs(rows);
  if (dtype == BW_DTYPE_F32) return dispatch_grad<float>(p, dweight, s);
  if (dtype == BW_DTYPE_F16) return dispatch_grad<__half>(p, dweight, s);
  return dispatch_grad<__nv_bfloat16>(p, dweight, s);
}

}  // extern "C"
