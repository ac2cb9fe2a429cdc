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
// in registers (packed in its own type: h is rounded to it anyway, and h w in FP32) between its
// reduction and its output. max |y| needs no second reduction: y_j = (h_j w_j) rstd and rounding is
// monotonic, so max |y| = max |h w| * rstd exactly, and both sums travel through one reduction.
// Statistics and sums are FP32. Measured, 16384 x 8192 BF16 with residual: to E4M3 137 us alone (6.9 TB/s of
// the 7 bytes an element), 143 called one by one, 150 back to back in a graph; gradient 155 us (6.9 TB/s of 8 bytes); 131072 x
// 128 BF16 to BF16 10.4 us (6.5 TB/s); 16384 x 8191 to E4M3, rows at every alignment, 144 us; one row of 8192 2.6 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>
#include <cmath>
#include <type_traits>

#include "bw_ptx.cuh"
#include "bw_runtime.cuh"

namespace bw {
namespace {

constexpr float kE4m3Max = 448.f;

// ------------------------------------------------------------------ element access
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// VE consecutive elements in whole registers, moved as one access of VE * sizeof(T) bytes (an array
// of 16-bit elements would take a register each).
template <int BYTES>
struct Words {
  static_assert(BYTES == 4 || BYTES == 8 || BYTES == 16 || BYTES == 32, "a power of two of words");
  uint32_t u[BYTES / 4];
};
template <>
struct Words<2> {
  uint32_t u[1];
};
template <>
struct Words<1> {
  uint32_t u[1];
};
template <typename T, int VE>
using Vec = Words<sizeof(T) * VE>;

template <int BYTES>
__device__ __forceinline__ Words<BYTES> load_words(const void* p) {
  Words<BYTES> v;
  if constexpr (BYTES == 1) {
    v.u[0] = *static_cast<const uint8_t*>(p);
  } else if constexpr (BYTES == 2) {
    v.u[0] = *static_cast<const uint16_t*>(p);
  } else if constexpr (BYTES == 4) {
    v.u[0] = *static_cast<const uint32_t*>(p);
  } else if constexpr (BYTES == 8) {
    const uint2 x = *static_cast<const uint2*>(p);
    v.u[0] = x.x;
    v.u[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 x = static_cast<const uint4*>(p)[i];
      v.u[4 * i] = x.x;
      v.u[4 * i + 1] = x.y;
      v.u[4 * i + 2] = x.z;
      v.u[4 * i + 3] = x.w;
    }
  }
  return v;
}
template <int BYTES>
__device__ __forceinline__ void store_words(void* p, const Words<BYTES>& v) {
  if constexpr (BYTES == 1) *static_cast<uint8_t*>(p) = static_cast<uint8_t>(v.u[0]);
  else if constexpr (BYTES == 2) *static_cast<uint16_t*>(p) = static_cast<uint16_t>(v.u[0]);
  else if constexpr (BYTES == 4) *static_cast<uint32_t*>(p) = v.u[0];
  else if constexpr (BYTES == 8) *static_cast<uint2*>(p) = make_uint2(v.u[0], v.u[1]);
  else *static_cast<uint4*>(p) = make_uint4(v.u[0], v.u[1], v.u[2], v.u[3]);
}
template <int BYTES>
__device__ __forceinline__ Words<BYTES> zero_words() {
  Words<BYTES> v;
#pragma unroll
  for (int i = 0; i < (BYTES + 3) / 4; ++i) v.u[i] = 0;
  return v;
}
// Element j of a vector as FP32, and two FP32 values as elements 2 i, 2 i + 1.
template <typename T, int BYTES>
__device__ __forceinline__ float elem(const Words<BYTES>& v, int j) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(v.u[j]);
  } else if constexpr (std::is_same_v<T, __half>) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(v.u[j / 2] >> (16 * (j & 1)))));
  } else {
    return __uint_as_float(j & 1 ? v.u[j / 2] & 0xffff0000u : v.u[j / 2] << 16);
  }
}
// Two FP32 operations an instruction (these kernels issue 5 to 10 instructions an element, enough to
// show beside the memory's time).
__device__ __forceinline__ uint64_t pack2(float2 a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t r) {
  float2 a;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(r));
  return a;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
  return unpack2(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)), "l"(pack2(c)));
  return unpack2(r);
}
// Elements 2 i and 2 i + 1.
template <typename T, int BYTES>
__device__ __forceinline__ float2 elems2(const Words<BYTES>& v, int i) {
  if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&v.u[i]));
  else return make_float2(elem<T>(v, 2 * i), elem<T>(v, 2 * i + 1));
}
template <typename T>
__device__ __forceinline__ uint32_t two_elems(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T, int VE>
__device__ __forceinline__ Vec<T, VE> from_floats(const float (&f)[VE]) {
  Vec<T, VE> v;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < VE; ++j) v.u[j] = __float_as_uint(f[j]);
  } else if constexpr (VE == 1) {
    v.u[0] = two_elems<T>(f[0], 0.f);
  } else {
#pragma unroll
    for (int j = 0; j < VE; j += 2) v.u[j / 2] = two_elems<T>(f[j], f[j + 1]);
  }
  return v;
}

// What a thread holds of a row: vectors i at columns col(i) .. col(i) + VE - 1, all of them whole. Where the
// row starts behind a vector's boundary (SHIFT), the elements in front of the first boundary and behind
// the last are left, at most VE - 1 each: 16 threads of the row hold one of them each, at column
// `single`. (Edge vectors of which parts count cost the two threads that had them, and with them
// the whole row, three times as long as everything else.)
template <int VE, bool SHIFT>
struct Columns {
  int tpr, t, front, vecs, single;
  __device__ __forceinline__ Columns(int tpr_, int t_, int phase, int cols) : tpr(tpr_), t(t_), front(0), single(-1) {
    if constexpr (SHIFT) front = min((VE - phase) & (VE - 1), cols);
    vecs = (cols - front) / VE;
    if constexpr (SHIFT) {
      const int behind = front + vecs * VE + t - 8;
      if (t < front) single = t;
      else if (t >= 8 && t < 16 && behind < cols) single = behind;
    }
  }
  __device__ __forceinline__ int col(int i) const { return front + (i * tpr + t) * VE; }
  __device__ __forceinline__ bool has(int i) const { return i * tpr + t < vecs; }
};
template <typename T, int VE, int NV, bool SHIFT>
struct Part {
  Vec<T, VE> v[NV];
  float one;  // the single element
};

template <typename T, int VE, int NV, bool SHIFT>
__device__ __forceinline__ void load_row(const T* row, const Columns<VE, SHIFT>& c, Part<T, VE, NV, SHIFT>& o) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
    o.v[i] = c.has(i) ? load_words<sizeof(T) * VE>(row + c.col(i)) : zero_words<sizeof(T) * VE>();
  if constexpr (SHIFT) o.one = c.single >= 0 ? to_f32(row[c.single]) : 0.f;
}
template <typename T, int VE, int NV, bool SHIFT>
__device__ __forceinline__ void store_row(T* row, const Columns<VE, SHIFT>& c, const Part<T, VE, NV, SHIFT>& o) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (c.has(i)) store_words<sizeof(T) * VE>(row + c.col(i), o.v[i]);
  if constexpr (SHIFT)
    if (c.single >= 0) row[c.single] = from_f32<T>(o.one);
}
// The weights have an alignment of their own: SHIFT reads them one by one (once for all rows of a
// thread, unless they do not fit its registers).
template <typename WT, int VE, bool SHIFT>
__device__ __forceinline__ Vec<WT, VE> load_weight(const void* w, const Columns<VE, SHIFT>& c, int i) {
  Vec<WT, VE> v = zero_words<sizeof(WT) * VE>();
  if (!c.has(i)) return v;
  const WT* p = static_cast<const WT*>(w) + c.col(i);
  if constexpr (SHIFT) {
#pragma unroll
    for (int j = 0; j < VE; ++j)
      v.u[j * sizeof(WT) / 4] |= load_words<sizeof(WT)>(p + j).u[0] << (8 * (j * sizeof(WT) % 4));
  } else {
    v = load_words<sizeof(WT) * VE>(p);
  }
  return v;
}

// Reduction over the `tpr` threads of a row: part of a warp (a power of two up to 32), or the whole
// block (up to 32 warps). All threads get the result. A caller in a loop alternates between two `sm`,
// so one barrier a call is enough.
struct SumMax {
  float sum, max;
};
template <bool MAX>
__device__ __forceinline__ SumMax reduce_lanes(SumMax v, int width) {
  for (int o = width / 2; o > 0; o >>= 1) {
    v.sum += __shfl_xor_sync(0xffffffffu, v.sum, o);
    if constexpr (MAX) v.max = fmaxf(v.max, __shfl_xor_sync(0xffffffffu, v.max, o));
  }
  return v;
}
// The whole warp: maxima of magnitudes order as integers.
template <bool MAX>
__device__ __forceinline__ SumMax reduce_warp(SumMax v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v.sum += __shfl_xor_sync(0xffffffffu, v.sum, o);
  if constexpr (MAX) v.max = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v.max)));
  return v;
}
template <bool MAX>
__device__ __forceinline__ SumMax reduce_row(SumMax v, int tpr, SumMax* sm) {
  if (tpr < 32) return reduce_lanes<MAX>(v, tpr);
  v = reduce_warp<MAX>(v);
  if (tpr > 32) {
    const int warps = tpr >> 5, lane = threadIdx.x & 31;
    if (lane == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? sm[lane] : SumMax{0.f, 0.f};  // maxima are of magnitudes
    v = reduce_warp<MAX>(v);
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
  float eps, inv_cols;
  int phase;           // elements between a vector's boundary and the first row (SHIFT)
  int depth;           // rows in flight (staged kernels)
  int* status;
  unsigned long long budget_ns;
};

// Scale of an E4M3 row by its maximum, and the factor that quantises it. A maximum so small that
// 448 / max overflows counts as zero.
__device__ __forceinline__ void e4m3_row_scale(float amax, float& mul, float& s) {
  mul = 1.f;
  s = 1.f;
  if (amax > 0.f && amax < INFINITY) {
    const float m = amax < 0x1p125f ? __fdividef(kE4m3Max, amax) : kE4m3Max / amax;  // the former gives 0 from 2^126 on
    if (m < INFINITY) {
      mul = m;
      s = amax / kE4m3Max;
    }
  }
}

template <int VE>
__device__ __forceinline__ void scale(const float (&a)[VE], float f, float (&o)[VE]) {
  if constexpr (VE == 1) {
    o[0] = a[0] * f;
  } else {
#pragma unroll
    for (int j = 0; j < VE; j += 2) {
      const float2 q = mul2(make_float2(a[j], a[j + 1]), make_float2(f, f));
      o[j] = q.x;
      o[j + 1] = q.y;
    }
  }
}

template <int VE>
__device__ __forceinline__ Words<VE> encode_e4m3(const float (&y)[VE], float mul) {
  Words<VE> q = zero_words<VE>();
  if constexpr (VE % 2 == 0) {
#pragma unroll
    for (int j = 0; j < VE; j += 2) {
      const __nv_fp8x2_storage_t two =
          __nv_cvt_float2_to_fp8x2(mul2(make_float2(y[j], y[j + 1]), make_float2(mul, mul)), __NV_SATFINITE, __NV_E4M3);
      q.u[j / 4] |= static_cast<uint32_t>(two) << (8 * (j % 4));
    }
  } else {
    q.u[0] = __nv_cvt_float_to_fp8(y[0] * mul, __NV_SATFINITE, __NV_E4M3);
  }
  return q;
}

// h + r, rounded once; 16-bit elements two an instruction. (Through FP32 the result is the same, 7 instructions for 2
// elements: in the register kernel 4% less to 3% more time over 32 widths and sizes, without a pattern. 16384 x 8192 BF16 to
// E4M3 140 us so and 145-149 packed as a captured graph, 146.5 and 143 called one by one; 26214 x 5120 144 / 141.)
template <typename T, int VE>
__device__ __forceinline__ void add_residual(Vec<T, VE>& h, const Vec<T, VE>& r) {
  if constexpr (std::is_same_v<T, float>) {
    float f[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) f[j] = elem<T>(h, j) + elem<T>(r, j);
    h = from_floats<T, VE>(f);
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(h.u) / 4); ++i) {
      const T2 sum = __hadd2(*reinterpret_cast<const T2*>(&h.u[i]), *reinterpret_cast<const T2*>(&r.u[i]));
      h.u[i] = *reinterpret_cast<const uint32_t*>(&sum);
    }
  }
}
__device__ __forceinline__ float add_as(float, float a, float b) { return a + b; }
template <typename T>
__device__ __forceinline__ float add_as(T, float a, float b) {
  return to_f32(__hadd(from_f32<T>(a), from_f32<T>(b)));
}

// p = h w, and its share of the row's sums.
template <bool Q8, typename T, typename WT, int VE>
__device__ __forceinline__ void accumulate(const Vec<T, VE>& h, const Vec<WT, VE>& w, float (&p)[VE], SumMax& a) {
  if constexpr (VE == 1) {
    const float v = elem<T>(h, 0);
    p[0] = v * elem<WT>(w, 0);
    a.sum = fmaf(v, v, a.sum);
    if constexpr (Q8) a.max = fmaxf(a.max, fabsf(p[0]));
  } else {
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) {
      const float2 v = elems2<T>(h, i);
      const float2 q = mul2(v, elems2<WT>(w, i));
      s = fma2(v, v, s);
      if constexpr (Q8) a.max = fmaxf(fmaxf(a.max, fabsf(q.x)), fabsf(q.y));
      p[2 * i] = q.x;
      p[2 * i + 1] = q.y;
    }
    a.sum += s.x + s.y;
  }
}

// v^(-1/2): CUDA's rsqrtf (2 steps off at most) and a Newton step. All threads of a row take it, in front of
// their output: a square root and a division are 40 instructions more.
__device__ __forceinline__ float inv_sqrt(float v) {
  const float y = rsqrtf(v);
  const float better = fmaf(0.5f * y, fmaf(-v * y, y, 1.f), y);
  return better < INFINITY && better > 0.f ? better : y;  // v = 0, infinite, NaN or so small that a product overflows
}

// Writes a row's rstd (and scale). Returns the factor from h w to y, or to the code's value; where that
// overflows (a row of tiny values), `pre` is a first factor of its own, else 1.
template <bool Q8>
__device__ __forceinline__ float finish_row(const NormParams& p, long long row, const SumMax& a, bool first, float& pre) {
  const float rstd = inv_sqrt(fmaf(a.sum, p.inv_cols, p.eps));
  float mul = 1.f, s = 1.f;
  if constexpr (Q8) e4m3_row_scale(a.max * rstd, mul, s);
  if (first) {
    if (p.rstd) p.rstd[row] = rstd;
    if constexpr (Q8) p.row_scale[row] = s;
  }
  const float f = rstd * mul;
  pre = 1.f;
  if (!Q8 || f < INFINITY) return f;
  pre = rstd;
  return mul;
}

template <typename T, bool Q8, int VE>
__device__ __forceinline__ auto output(const float (&hw)[VE], float f, float pre) {
  if constexpr (Q8) {
    if (pre == 1.f) return encode_e4m3<VE>(hw, f);
    float y[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) y[j] = hw[j] * pre;
    return encode_e4m3<VE>(y, f);
  } else {
    float y[VE];
    scale<VE>(hw, f, y);
    return from_floats<T, VE>(y);
  }
}

// Bytes of a row that one thread holds, an element of 16 bits alone taking a register.
template <typename T, int VE, int NV>
constexpr int kThreadBytes = NV * (sizeof(T) * VE < 4 ? 4 : sizeof(T) * VE);

// tpr threads take a row, NV vectors of VE elements each: a whole block for tpr > 32, else (a power of two)
// one of blockDim.x / tpr groups of a block. A group walks the rows with a stride of all groups, keeps its columns' weights in
// registers, and fetches its next row as soon as this one's h is summed, so that loads are in
// flight during the reduction and the stores (neither where a thread holds over 64 bytes of a row).
// SHIFT: rows start `phase` elements behind a vector's boundary, a different number from row to
// row; the group stride is a multiple of VE rows then, so a group's rows all have the same phase.
template <typename T, typename WT, bool Q8, int VE, int NV, bool SHIFT>
__global__ void __launch_bounds__(512) k_rmsnorm(const NormParams p, int tpr) {
  constexpr bool kKeep = kThreadBytes<T, VE, NV> <= 64;
  grid_dependency_wait();
  __shared__ SumMax sm[2][32];
  const int per_block = blockDim.x / tpr;
  const int t = threadIdx.x % tpr;
  const long long stride = static_cast<long long>(gridDim.x) * per_block;
  long long row0 = static_cast<long long>(blockIdx.x) * per_block;  // of the block: its loop is uniform
  long long row = row0 + threadIdx.x / tpr;
  const Columns<VE, SHIFT> c(tpr, t, static_cast<int>((p.phase + row * p.ldx) & (VE - 1)), p.cols);
  const T* x = static_cast<const T*>(p.x);
  const T* r = static_cast<const T*>(p.res);
  using O = std::conditional_t<Q8, uint8_t, T>;
  Part<T, VE, NV, SHIFT> h, res;
  Vec<WT, VE> w[kKeep ? NV : 1];
  float w1 = 0.f;
  auto fetch = [&](long long rw) {
    if (rw >= p.rows) return;
    load_row(x + rw * p.ldx, c, h);
    if (r) load_row(r + rw * p.ldr, c, res);
  };
  if constexpr (kKeep) {
    fetch(row);
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i] = load_weight<WT, VE, SHIFT>(p.w, c, i);
  }
  if (SHIFT && c.single >= 0) w1 = to_f32(static_cast<const WT*>(p.w)[c.single]);
  int half = 0;
  for (; row0 < p.rows; row0 += stride, row += stride) {
    const bool live = row < p.rows;
    float hw[NV][VE], hw1 = 0.f;
    SumMax a{0.f, 0.f};
    if (live) {
      if constexpr (!kKeep) fetch(row);
      if (r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) add_residual<T, VE>(h.v[i], res.v[i]);
        if constexpr (SHIFT) h.one = add_as(T{}, h.one, res.one);
      }
      if (p.h) store_row(static_cast<T*>(p.h) + row * p.ldh, c, h);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (!kKeep) w[0] = load_weight<WT, VE, SHIFT>(p.w, c, i);
        accumulate<Q8, T, WT, VE>(h.v[i], w[kKeep ? i : 0], hw[i], a);
      }
      if constexpr (SHIFT) {
        hw1 = h.one * w1;
        a.sum = fmaf(h.one, h.one, a.sum);
        if constexpr (Q8) a.max = fmaxf(a.max, fabsf(hw1));
      }
      if constexpr (kKeep) fetch(row + stride);
    }
    a = reduce_row<Q8>(a, tpr, sm[half]);
    half ^= 1;
    if (live) {
      float pre;
      const float f = finish_row<Q8>(p, row, a, t == 0, pre);
      O* y = static_cast<O*>(p.y) + row * p.ldy;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (c.has(i)) store_words<sizeof(O) * VE>(y + c.col(i), output<T, Q8, VE>(hw[i], f, pre));
      if constexpr (SHIFT) {
        const float one[1] = {hw1};
        if (c.single >= 0) store_words<sizeof(O)>(y + c.single, output<T, Q8, 1>(one, f, pre));
      }
    }
  }
}

// Rows on their way to a block: the whole vectors of TENSORS rows a slot, `depth` slots, copied by the TMA unit while
// the block is at earlier rows. So the bytes in flight depend neither on registers nor on idle lanes. One
// thread of the row's own issues the copies (a warp for that alone takes the place of one that
// computes: 37476 x 3519 gradient 208 us, 241 with such a warp).
constexpr int kMaxDepth = 4;
template <int TENSORS>  // of which the last may be absent
struct RowRing {
  uint64_t* full;   // [depth], shared
  uint8_t* data;
  int depth, pitch;  // bytes between the rows of a slot
  int slot = 0;
  uint32_t parity = 0;
  const char* src[TENSORS];        // null: absent
  long long step[TENSORS];         // bytes between a block's rows
  uint32_t bytes;
  int issued = 0;                  // rows, by the thread that issues them

  __device__ __forceinline__ int tensors() const { return src[TENSORS - 1] ? TENSORS : TENSORS - 1; }
  __device__ __forceinline__ uint8_t* at(int s, int tensor) const { return data + (s * tensors() + tensor) * pitch; }
  __device__ __forceinline__ void issue(int s, long long n) {  // the block's n-th row
    ++issued;
    mbar_arrive_expect_tx(&full[s], tensors() * bytes);
#pragma unroll
    for (int i = 0; i < TENSORS; ++i)
      if (src[i] && bytes) bulk_load(at(s, i), src[i] + n * step[i], bytes, &full[s]);
  }
  __device__ __forceinline__ void advance() {
    if (++slot == depth) { slot = 0; parity ^= 1; }
  }
  // After a timeout the copies in flight land before the block gives its shared memory back, however
  // short the wait budget is.
  __device__ __forceinline__ void drain() const {
    for (int i = issued > depth ? issued - depth : 0; i < issued; ++i)
      mbar_drain(&full[i % depth], static_cast<uint32_t>(i / depth) & 1u);
  }
};
template <typename T, int VE, int NV, bool SHIFT>
__device__ __forceinline__ void load_staged(const uint8_t* row, const Columns<VE, SHIFT>& c, Part<T, VE, NV, SHIFT>& o) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
    o.v[i] = c.has(i) ? load_words<sizeof(T) * VE>(row + (i * c.tpr + c.t) * (sizeof(T) * VE)) : zero_words<sizeof(T) * VE>();
}

// k_rmsnorm for rows over 128 vectors which leave lanes idle there, which start behind a boundary, or which are
// too long for its registers: a block takes one row at a time out of its ring. Both measured, us, in registers / staged
// (BF16 to E4M3 with residual): behind a boundary 19407 x 2498 75 / 59, 3564 x 9553 78 / 40; whole vectors 15252 x 8800 186 / 165 (one
// block an SM), 16384 x 8192 147 / 164, 26214 x 5120 142 / 160. Where the line lies for whole vectors (1700 of an SM's 2048 in use, below):
// time in registers over time staged, 12 to 128 million elements at 33 widths from 1088 to 16384, both outputs. With a
// residual 0.86-1.03 (mean 0.96) above the line and 0.83-1.22 (0.99) under it; without one 0.93-1.27 (1.07) and 0.86-1.61 (1.12).
template <typename T, typename WT, bool Q8, int VE, int NV, bool SHIFT>
__global__ void __launch_bounds__(512) k_rmsnorm_staged(const NormParams p) {
  constexpr bool kKeep = kThreadBytes<T, VE, NV> <= 64;
  extern __shared__ __align__(128) uint8_t ring_data[];
  __shared__ uint64_t full[kMaxDepth];
  __shared__ volatile int abort_flag;
  __shared__ SumMax sm[2][32];
  const int tpr = blockDim.x, t = threadIdx.x;
  const long long stride = gridDim.x;
  long long row = blockIdx.x;
  const Columns<VE, SHIFT> c(tpr, t, static_cast<int>((p.phase + row * p.ldx) & (VE - 1)), p.cols);
  const T* x = static_cast<const T*>(p.x);
  const T* r = static_cast<const T*>(p.res);
  RowRing<2> ring;
  ring.full = full;
  ring.data = ring_data;
  ring.depth = p.depth;
  ring.pitch = p.cols / VE * 16;
  ring.src[0] = reinterpret_cast<const char*>(x + row * p.ldx + c.front);
  ring.src[1] = r ? reinterpret_cast<const char*>(r + row * p.ldr + c.front) : nullptr;
  ring.step[0] = stride * p.ldx * sizeof(T);
  ring.step[1] = stride * p.ldr * sizeof(T);
  ring.bytes = c.vecs * 16;
  const WaitCtl wc{&abort_flag, p.status, p.budget_ns};
  if (t == 0) {
    for (int d = 0; d < p.depth; ++d) mbar_init(&full[d], 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  grid_dependency_wait();
  if (t == 0)
    for (int d = 0; d < p.depth && row + d * stride < p.rows; ++d) ring.issue(d, d);
  using O = std::conditional_t<Q8, uint8_t, T>;
  Part<T, VE, NV, SHIFT> h, res;
  Vec<WT, VE> w[kKeep ? NV : 1];
  float w1 = 0.f, one = 0.f, one_res = 0.f;
  auto fetch_single = [&](long long rw) {
    if (!SHIFT || c.single < 0 || rw >= p.rows) return;
    one = to_f32(x[rw * p.ldx + c.single]);
    if (r) one_res = to_f32(r[rw * p.ldr + c.single]);
  };
  fetch_single(row);
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i] = load_weight<WT, VE, SHIFT>(p.w, c, i);
  }
  if (SHIFT && c.single >= 0) w1 = to_f32(static_cast<const WT*>(p.w)[c.single]);
  __syncthreads();  // the barriers are set up
  int half = 0;
  for (long long n = 0; row < p.rows; ++n, row += stride) {
    float hw[NV][VE], hw1 = 0.f;
    SumMax a{0.f, 0.f};
    mbar_wait(&full[ring.slot], ring.parity, wc, 71);  // after a timeout the block goes on, with wrong values and the status set
    load_staged(ring.at(ring.slot, 0), c, h);
    if (r) {
      load_staged(ring.at(ring.slot, 1), c, res);
#pragma unroll
      for (int i = 0; i < NV; ++i) add_residual<T, VE>(h.v[i], res.v[i]);
    }
    if constexpr (SHIFT) {
      h.one = r ? add_as(T{}, one, one_res) : one;
      fetch_single(row + stride);
    }
    if (p.h) store_row(static_cast<T*>(p.h) + row * p.ldh, c, h);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (!kKeep) w[0] = load_weight<WT, VE, SHIFT>(p.w, c, i);
      accumulate<Q8, T, WT, VE>(h.v[i], w[kKeep ? i : 0], hw[i], a);
    }
    if constexpr (SHIFT) {
      hw1 = h.one * w1;
      a.sum = fmaf(h.one, h.one, a.sum);
      if constexpr (Q8) a.max = fmaxf(a.max, fabsf(hw1));
    }
    __syncwarp();
    a = reduce_row<Q8>(a, tpr, sm[half]);
    half ^= 1;
    // every thread has read its part of the slot
    if (t == 0 && row + p.depth * stride < p.rows && !abort_flag) ring.issue(ring.slot, n + p.depth);
    ring.advance();
    float pre;
    const float f = finish_row<Q8>(p, row, a, t == 0, pre);
    O* y = static_cast<O*>(p.y) + row * p.ldy;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (c.has(i)) store_words<sizeof(O) * VE>(y + c.col(i), output<T, Q8, VE>(hw[i], f, pre));
    if constexpr (SHIFT) {
      const float last[1] = {hw1};
      if (c.single >= 0) store_words<sizeof(O)>(y + c.single, output<T, Q8, 1>(last, f, pre));
    }
  }
  if (t == 0 && abort_flag) ring.drain();
}

// Rows too long for the registers of one block: one block a row, which reads its row twice (the
// second time from L2).
template <typename T, typename WT, bool Q8, int VE>
__global__ void __launch_bounds__(1024) k_rmsnorm_wide(const NormParams p) {
  __shared__ SumMax sm[32];
  grid_dependency_wait();
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* r = p.res ? static_cast<const T*>(p.res) + row * p.ldr : nullptr;
  T* hr = p.h ? static_cast<T*>(p.h) + row * p.ldh : nullptr;
  SumMax a{0.f, 0.f};
  const WT* w = static_cast<const WT*>(p.w);
  float hw[VE];
  for (long long c = static_cast<long long>(threadIdx.x) * VE; c < p.cols; c += 1024LL * VE) {
    Vec<T, VE> h = load_words<sizeof(T) * VE>(x + c);
    if (r) add_residual<T, VE>(h, load_words<sizeof(T) * VE>(r + c));
    if (hr) store_words<sizeof(T) * VE>(hr + c, h);
    accumulate<Q8, T, WT, VE>(h, load_words<sizeof(WT) * VE>(w + c), hw, a);
  }
  a = reduce_row<Q8>(a, 1024, sm);
  float pre;
  const float f = finish_row<Q8>(p, row, a, threadIdx.x == 0, pre);
  for (long long c = static_cast<long long>(threadIdx.x) * VE; c < p.cols; c += 1024LL * VE) {
    // this thread wrote h[c] itself; where h is not kept, the sum is taken again. x and the
    // residual still hold their values then: h and y are written at this thread's own columns,
    // and a column's y after its last read.
    Vec<T, VE> h;
    if (hr) {
      h = load_words<sizeof(T) * VE>(hr + c);
    } else {
      h = load_words<sizeof(T) * VE>(x + c);
      if (r) add_residual<T, VE>(h, load_words<sizeof(T) * VE>(r + c));
    }
    SumMax unused{0.f, 0.f};
    accumulate<false, T, WT, VE>(h, load_words<sizeof(WT) * VE>(w + c), hw, unused);
    using O = std::conditional_t<Q8, uint8_t, T>;
    store_words<sizeof(O) * VE>(static_cast<O*>(p.y) + row * p.ldy + c, output<T, Q8, VE>(hw, f, pre));
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
  int phase;           // elements between a vector's boundary and the first row (SHIFT)
  int depth;           // rows in flight (staged kernels)
  int* status;
  unsigned long long budget_ns;
};

// A vector's share of sum(g h) and of the weight gradient.
template <typename T, typename WT, int VE>
__device__ __forceinline__ void grad_sums(const Vec<T, VE>& dy, const Vec<T, VE>& h, const Vec<WT, VE>& w, float rstd,
                                          float& sum, float (&dw)[VE]) {
  if constexpr (VE == 1) {
    const float d = elem<T>(dy, 0), v = elem<T>(h, 0);
    sum = fmaf(d * elem<WT>(w, 0), v, sum);
    dw[0] = fmaf(d * rstd, v, dw[0]);
  } else {
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) {
      const float2 d = elems2<T>(dy, i), v = elems2<T>(h, i);
      s = fma2(mul2(d, elems2<WT>(w, i)), v, s);
      const float2 t = fma2(mul2(d, make_float2(rstd, rstd)), v, make_float2(dw[2 * i], dw[2 * i + 1]));
      dw[2 * i] = t.x;
      dw[2 * i + 1] = t.y;
    }
    sum += s.x + s.y;
  }
}
template <typename T, typename WT, int VE>
__device__ __forceinline__ Vec<T, VE> grad_output(const Vec<T, VE>& dy, const Vec<T, VE>& h, const Vec<WT, VE>& w,
                                                  const Vec<T, VE>& dres, float rstd, float m) {
  float o[VE];
  if constexpr (VE == 1) {
    o[0] = fmaf(rstd, fmaf(-m, elem<T>(h, 0) * rstd, elem<T>(dy, 0) * elem<WT>(w, 0)), elem<T>(dres, 0));
  } else {
    const float2 r2 = make_float2(rstd, rstd), m2 = make_float2(-m, -m);
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) {
      const float2 g = mul2(elems2<T>(dy, i), elems2<WT>(w, i)), n = mul2(elems2<T>(h, i), r2);
      const float2 t = fma2(r2, fma2(m2, n, g), elems2<T>(dres, i));
      o[2 * i] = t.x;
      o[2 * i + 1] = t.y;
    }
  }
  return from_floats<T, VE>(o);
}

template <int VE>
__device__ __forceinline__ void store_sums(float* at, const float (&dw)[VE]) {
  if (VE % 4 == 0 && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
#pragma unroll
    for (int j = 0; j + 3 < VE; j += 4) *reinterpret_cast<float4*>(at + j) = make_float4(dw[j], dw[j + 1], dw[j + 2], dw[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j) at[j] = dw[j];
  }
}

// Rows, columns and phases as in k_rmsnorm; each thread keeps the weight gradient of its own
// columns in registers over all its rows, and stores it four columns at a time (64 x 8192 BF16 10.6 us one
// by one, 6.6 us so; through shared memory, for columns behind a boundary, measured slower). With g = dy w:
//   dx = rstd (g - n m) + dresidual,   n = h rstd,   m = rstd sum(g h) / cols,   dw += (dy rstd) h
// (one product more an element than rstd g - h rstd^3 sum / cols, whose cube leaves FP32 for rows of
// 10^13 or 10^-13).
// Where a thread holds up to 32 bytes of a row it keeps its weights and fetches the next row during this
// one's reduction; else it reads the weights again and dresidual late.
template <typename T, typename WT, int VE, int NV, bool SHIFT>
__global__ void __launch_bounds__(512) k_rmsnorm_grad(const NormGradParams p, int tpr) {
  constexpr bool kKeep = kThreadBytes<T, VE, NV> <= 32;
  grid_dependency_wait();
  __shared__ SumMax sm[2][32];
  extern __shared__ float cols_sum[];  // tpr <= 32: [group of the block][cols]
  const int per_block = blockDim.x / tpr, mine = threadIdx.x / tpr;
  const int t = threadIdx.x - mine * tpr;
  const long long stride = static_cast<long long>(gridDim.x) * per_block;
  long long row0 = static_cast<long long>(blockIdx.x) * per_block;
  long long row = row0 + mine;
  const Columns<VE, SHIFT> c(tpr, t, static_cast<int>((p.phase + row * p.ldh) & (VE - 1)), p.cols);
  const T* dys = static_cast<const T*>(p.dy);
  const T* hs = static_cast<const T*>(p.h);
  const T* drs = static_cast<const T*>(p.dres);
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  using Row = Part<T, VE, NV, SHIFT>;
  Row dy, h, dr;
  Vec<WT, VE> w[kKeep ? NV : 1];
  float dw[NV][VE], dw1 = 0.f, w1 = 0.f;
  float rstd = 0.f;
  auto fetch = [&](long long rw, Row& dyv, Row& hv, Row& drv, float& rs) {
    if (rw >= p.rows) return;
    load_row(dys + rw * p.lddy, c, dyv);
    load_row(hs + rw * p.ldh, c, hv);
    if constexpr (kKeep)
      if (drs) load_row(drs + rw * p.lddr, c, drv);
    rs = p.rstd[rw];
  };
  if constexpr (kKeep) {
    fetch(row, dy, h, dr, rstd);
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i] = load_weight<WT, VE, SHIFT>(p.w, c, i);
  }
  if (SHIFT && c.single >= 0) w1 = to_f32(static_cast<const WT*>(p.w)[c.single]);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) dw[i][j] = 0.f;
  int half = 0;
  for (; row0 < p.rows; row0 += stride, row += stride) {
    const bool live = row < p.rows;
    Row dy2, h2, dr2;
    float rstd2 = 0.f;
    if (live) {
      if constexpr (kKeep) fetch(row + stride, dy2, h2, dr2, rstd2);
      else fetch(row, dy, h, dr, rstd);
    }
    SumMax a{0.f, 0.f};
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (!kKeep) w[0] = load_weight<WT, VE, SHIFT>(p.w, c, i);
        grad_sums<T, WT, VE>(dy.v[i], h.v[i], w[kKeep ? i : 0], rstd, a.sum, dw[i]);
      }
      if constexpr (SHIFT) {
        a.sum = fmaf(dy.one * w1, h.one, a.sum);
        dw1 = fmaf(dy.one * rstd, h.one, dw1);
      }
    }
    a = reduce_row<false>(a, tpr, sm[half]);
    half ^= 1;
    if (live) {
      const float m = rstd * (a.sum * inv_cols);
      if constexpr (!kKeep)
        if (drs) load_row(drs + row * p.lddr, c, dr);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (!kKeep) w[0] = load_weight<WT, VE, SHIFT>(p.w, c, i);
        dy.v[i] = grad_output<T, WT, VE>(dy.v[i], h.v[i], w[kKeep ? i : 0], drs ? dr.v[i] : zero_words<sizeof(T) * VE>(), rstd, m);
      }
      if constexpr (SHIFT) {
        dy.one = rstd * (dy.one * w1 - h.one * rstd * m);
        if (drs) dy.one += dr.one;
      }
      store_row(static_cast<T*>(p.dx) + row * p.lddx, c, dy);
      if constexpr (kKeep) {
        dy = dy2;
        h = h2;
        dr = dr2;
        rstd = rstd2;
      }
    }
  }
  float* out = p.partial + static_cast<long long>(blockIdx.x) * p.cols;
  float* mine_out = tpr > 32 ? out : cols_sum + mine * p.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (c.has(i)) store_sums<VE>(mine_out + c.col(i), dw[i]);
  if (SHIFT && c.single >= 0) mine_out[c.single] = dw1;
  if (tpr > 32) return;
  __syncthreads();
  for (int j = threadIdx.x; j < p.cols; j += blockDim.x) {
    float s = 0.f;
    for (int g = 0; g < per_block; ++g) s += cols_sum[g * p.cols + j];
    out[j] = s;
  }
}

// k_rmsnorm_grad for many rows over 64 vectors: a block takes one row at a time out of its ring. In registers / staged, us, BF16
// with a residual's gradient: 16384 x 8192 175 / 155, 23786 x 4608 195 / 129, 37476 x 3519 267 / 202, 6629 x 10184 166 / 104,
// 31373 x 950 63 / 53; with few rows a block the first copies and barriers cost more than they save (1000 x 2050 FP32 11.1 / 12-18).
template <typename T, typename WT, int VE, int NV, bool SHIFT>
__global__ void __launch_bounds__(512) k_rmsnorm_grad_staged(const NormGradParams p) {
  constexpr bool kKeep = kThreadBytes<T, VE, NV> <= 32;
  extern __shared__ __align__(128) uint8_t ring_data[];
  __shared__ uint64_t full[kMaxDepth];
  __shared__ volatile int abort_flag;
  __shared__ SumMax sm[2][32];
  const int tpr = blockDim.x, t = threadIdx.x;
  const long long stride = gridDim.x;
  long long row = blockIdx.x;
  const Columns<VE, SHIFT> c(tpr, t, static_cast<int>((p.phase + row * p.ldh) & (VE - 1)), p.cols);
  const T* dys = static_cast<const T*>(p.dy);
  const T* hs = static_cast<const T*>(p.h);
  const T* drs = static_cast<const T*>(p.dres);
  RowRing<3> ring;
  ring.full = full;
  ring.data = ring_data;
  ring.depth = p.depth;
  ring.pitch = p.cols / VE * 16;
  ring.src[0] = reinterpret_cast<const char*>(dys + row * p.lddy + c.front);
  ring.src[1] = reinterpret_cast<const char*>(hs + row * p.ldh + c.front);
  ring.src[2] = drs ? reinterpret_cast<const char*>(drs + row * p.lddr + c.front) : nullptr;
  ring.step[0] = stride * p.lddy * sizeof(T);
  ring.step[1] = stride * p.ldh * sizeof(T);
  ring.step[2] = stride * p.lddr * sizeof(T);
  ring.bytes = c.vecs * 16;
  const WaitCtl wc{&abort_flag, p.status, p.budget_ns};
  if (t == 0) {
    for (int d = 0; d < p.depth; ++d) mbar_init(&full[d], 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  grid_dependency_wait();
  if (t == 0)
    for (int d = 0; d < p.depth && row + d * stride < p.rows; ++d) ring.issue(d, d);
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  Part<T, VE, NV, SHIFT> dy, h, dr;
  Vec<WT, VE> w[kKeep ? NV : 1];
  float dw[NV][VE], dw1 = 0.f, w1 = 0.f;
  float rstd = 0.f, one_dy = 0.f, one_h = 0.f, one_dr = 0.f;
  auto fetch_rest = [&](long long rw) {
    if (rw >= p.rows) return;
    rstd = p.rstd[rw];
    if (!SHIFT || c.single < 0) return;
    one_dy = to_f32(dys[rw * p.lddy + c.single]);
    one_h = to_f32(hs[rw * p.ldh + c.single]);
    if (drs) one_dr = to_f32(drs[rw * p.lddr + c.single]);
  };
  fetch_rest(row);
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i] = load_weight<WT, VE, SHIFT>(p.w, c, i);
  }
  if (SHIFT && c.single >= 0) w1 = to_f32(static_cast<const WT*>(p.w)[c.single]);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) dw[i][j] = 0.f;
  __syncthreads();  // the barriers are set up
  int half = 0;
  for (long long n = 0; row < p.rows; ++n, row += stride) {
    mbar_wait(&full[ring.slot], ring.parity, wc, 72);  // after a timeout the block goes on, with wrong values and the status set
    load_staged(ring.at(ring.slot, 0), c, dy);
    load_staged(ring.at(ring.slot, 1), c, h);
    if (drs) load_staged(ring.at(ring.slot, 2), c, dr);
    const float rs = rstd;
    dy.one = one_dy;
    h.one = one_h;
    dr.one = one_dr;
    fetch_rest(row + stride);
    SumMax a{0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (!kKeep) w[0] = load_weight<WT, VE, SHIFT>(p.w, c, i);
      grad_sums<T, WT, VE>(dy.v[i], h.v[i], w[kKeep ? i : 0], rs, a.sum, dw[i]);
    }
    if constexpr (SHIFT) {
      a.sum = fmaf(dy.one * w1, h.one, a.sum);
      dw1 = fmaf(dy.one * rs, h.one, dw1);
    }
    __syncwarp();
    a = reduce_row<false>(a, tpr, sm[half]);
    half ^= 1;
    // every thread has read its part of the slot
    if (t == 0 && row + p.depth * stride < p.rows && !abort_flag) ring.issue(ring.slot, n + p.depth);
    ring.advance();
    const float m = rs * (a.sum * inv_cols);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (!kKeep) w[0] = load_weight<WT, VE, SHIFT>(p.w, c, i);
      dy.v[i] = grad_output<T, WT, VE>(dy.v[i], h.v[i], w[kKeep ? i : 0], drs ? dr.v[i] : zero_words<sizeof(T) * VE>(), rs, m);
    }
    if constexpr (SHIFT) {
      dy.one = rs * (dy.one * w1 - h.one * rs * m);
      if (drs) dy.one += dr.one;
    }
    store_row(static_cast<T*>(p.dx) + row * p.lddx, c, dy);
  }
  if (t == 0 && abort_flag) ring.drain();
  float* out = p.partial + static_cast<long long>(blockIdx.x) * p.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (c.has(i)) store_sums<VE>(out + c.col(i), dw[i]);
  if (SHIFT && c.single >= 0) out[c.single] = dw1;
}

// Rows too long for registers: dx with the row read twice, and the weight gradient's slabs by
// columns in a kernel of their own.
template <typename T, typename WT>
__global__ void __launch_bounds__(1024) k_rmsnorm_grad_wide(const NormGradParams p) {
  __shared__ SumMax sm[32];
  grid_dependency_wait();
  const long long row = blockIdx.x;
  const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
  const T* h = static_cast<const T*>(p.h) + row * p.ldh;
  const WT* w = static_cast<const WT*>(p.w);
  const float rstd = p.rstd[row];
  SumMax a{0.f, 0.f};
  for (long long c = threadIdx.x; c < p.cols; c += 1024) a.sum = fmaf(to_f32(dy[c]) * to_f32(w[c]), to_f32(h[c]), a.sum);
  a = reduce_row<false>(a, 1024, sm);
  const float m = rstd * (a.sum / static_cast<float>(p.cols));
  for (long long c = threadIdx.x; c < p.cols; c += 1024) {
    float g = rstd * (to_f32(dy[c]) * to_f32(w[c]) - to_f32(h[c]) * rstd * m);
    if (p.dres) g += to_f32(static_cast<const T*>(p.dres)[row * p.lddr + c]);
    static_cast<T*>(p.dx)[row * p.lddx + c] = from_f32<T>(g);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) k_rmsnorm_dw_wide(const NormGradParams p) {
  grid_dependency_wait();
  const long long c = blockIdx.x * 256LL + threadIdx.x;
  if (c >= p.cols) return;
  for (int slab = blockIdx.y; slab < p.slabs; slab += gridDim.y) {
    float s = 0.f;
    for (long long row = slab; row < p.rows; row += p.slabs)
      s = fmaf(to_f32(static_cast<const T*>(p.dy)[row * p.lddy + c]) * p.rstd[row],
               to_f32(static_cast<const T*>(p.h)[row * p.ldh + c]), s);
    p.partial[static_cast<long long>(slab) * p.cols + c] = s;
  }
}

// dw[c] = sum over slabs in a fixed order: 32 columns a block, 32 warps over the slabs.
__global__ void __launch_bounds__(1024) k_sum_slabs(const float* partial, float* dw, int slabs, int cols) {
  __shared__ float sm[32][33];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long c = blockIdx.x * 32LL + lane;
  float s = 0.f;
  if (c < cols)
    for (int i = warp; i < slabs; i += 32) s += __ldcg(partial + static_cast<long long>(i) * cols + c);
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

struct Shape {
  int tpr, nv;  // nv = 0: too long for registers
  int block;
  long long groups;  // a block
};

// Threads a row (at least min_tpr) and vectors a thread (1, 2, 4, ... up to max_nv): `want` vectors, so that a
// block is small and each thread has more loads in flight, but one where that still gives every
// resident thread (512 an SM) at most one (BF16 to E4M3 with one / four: 150 x 512 2.3 / 3.0 us, 150 x 2048
// 2.6 / 2.8, 300 x 2048 3.2 / 3.2, 150 x 8192 4.6 / 3.8, 1200 x 8192 16.2 / 12.9); fewer also where a warp's
// granularity would leave over an eighth more of them idle.
constexpr int kMaxThreads = 512;
Shape row_shape(long long rows, long long nvec, int want, int max_nv, int min_tpr, int sms) {
  if (rows * nvec <= sms * 512LL) want = 1;
  int nv = want;
  while (nv <= max_nv && nvec > static_cast<long long>(nv) * kMaxThreads) nv *= 2;
  if (nv > max_nv) return {0, 0, 0, 0};
  if (nvec <= 32 * nv) {  // groups inside warps
    int tpr = min_tpr;
    while (tpr * nv < nvec) tpr *= 2;
    return {tpr, nv, 256, 256 / tpr};
  }
  auto threads = [&](int n) { return static_cast<int>((nvec + 32 * n - 1) / (32 * n)) * 32; };
  for (int n = nv / 2; n >= 1 && threads(n) <= kMaxThreads; n /= 2)
    if (8 * threads(nv) * nv > 9 * threads(n) * n) nv = n;
  return {threads(nv), nv, threads(nv), 1};
}

// How a call's rows are read: 16-byte vectors from a boundary, vectors behind one (every tensor's
// row at the same distance, which contiguous tensors have whatever cols is), or element by element.
enum class Access { ALIGNED, SHIFTED, SCALAR };
struct RowsOf {  // one tensor: address, pitch in elements, element size
  const void* p;
  long long ld;
  int elem;
};
template <int N>
Access row_access(const RowsOf (&t)[N], int ve, long long cols, int* phase) {
  // element offset from a vector's boundary of the tensor's first row
  auto first = [&](const RowsOf& o) { return static_cast<long long>(reinterpret_cast<uintptr_t>(o.p) / o.elem % ve); };
  const RowsOf& a = t[0];
  bool same = true, aligned = cols % ve == 0;
  for (const RowsOf& o : t) {
    if (!o.p) continue;
    same = same && first(o) == first(a) && (o.ld - a.ld) % ve == 0;
    aligned = aligned && first(o) == 0 && o.ld % ve == 0;
  }
  *phase = static_cast<int>(first(a));
  return aligned ? Access::ALIGNED : same ? Access::SHIFTED : Access::SCALAR;
}

// As many blocks as are resident at once (16384 x 8192 BF16: one more a SM takes 1% longer, a few left over twice as long),
// each with its share of the rows.
template <auto KERN, bool SHIFT>
int launch_rows(const NormParams& p, const Shape& sh, cudaStream_t s, const DeviceState& d) {
  static std::atomic<int> resident[kMaxThreads / 32 + 1] = {};  // by block size, of this kernel; 0: not asked yet
  std::atomic<int>& known = resident[sh.block / 32];
  int per_sm = known.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    BW_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, KERN, sh.block, 0));
    known.store(per_sm, std::memory_order_relaxed);
  }
  long long grid = (p.rows + sh.groups - 1) / sh.groups;
  long long cap = static_cast<long long>(d.sms) * per_sm;
  if (SHIFT) cap = cap / 8 * 8;  // a stride of whole phases
  if (grid > cap) grid = cap;
  BW_CUDA(launch_dependent(KERN, dim3(static_cast<unsigned>(grid)), sh.block, 0, s, p, sh.tpr));
  return BW_OK;
}

// A staged kernel's block (one row at a time, `want` vectors a thread or more), rows in flight and dynamic shared
// memory, where an SM holds `resident` threads by their registers. depth = 0: the row is too long.
struct Staging {
  int nv, block, depth;
  size_t smem;
};
constexpr int kRingBytes = 160 << 10, kRingMost = 200 << 10;  // of an SM; where two rows need more than the former
Staging row_staging(long long nvec, int want, int max_nv, int tensors, int resident) {
  Staging g{want, 0, 0, 0};
  while (nvec > static_cast<long long>(g.nv) * kMaxThreads) g.nv *= 2;
  if (nvec == 0 || g.nv > max_nv) return g;
  g.block = static_cast<int>((nvec + 32 * g.nv - 1) / (32 * g.nv)) * 32;
  const long long slot = tensors * nvec * 16;
  int blocks = resident / g.block;
  if (blocks < 1) blocks = 1;
  while (blocks > 1 && kRingBytes / blocks < 2 * slot) --blocks;
  long long depth = kRingBytes / blocks / slot;
  if (depth < 2) depth = kRingMost / blocks / slot;
  g.depth = static_cast<int>(depth > kMaxDepth ? kMaxDepth : depth);
  g.smem = static_cast<size_t>(g.depth) * slot;
  return g;
}
constexpr int kMaxDynamic = 225 << 10;

// Blocks of a staged kernel that an SM holds.
template <auto KERN>
int staged_resident(const Staging& g, int* per_sm) {
  static std::atomic<int> known[64][kMaxThreads / 32 + 1] = {};  // by device and block size, without the ring
  int dev = 0;
  BW_CUDA(cudaGetDevice(&dev));
  std::atomic<int>& k = known[dev & 63][g.block / 32];
  int n = k.load(std::memory_order_acquire);
  if (n == 0) {
    BW_CUDA(cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynamic));
    BW_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERN, g.block, 0));
    k.store(n, std::memory_order_release);
  }
  const int fit = static_cast<int>((228u << 10) / (g.smem + 2048));  // 1 KB of the system's, 1 KB static
  *per_sm = n < fit ? n : fit;
  return BW_OK;
}

template <auto KERN, bool SHIFT>
int launch_staged(NormParams p, const Staging& g, cudaStream_t s, const DeviceState& d) {
  int per_sm = 0;
  const int r = staged_resident<KERN>(g, &per_sm);
  if (r != BW_OK) return r;
  long long grid = static_cast<long long>(d.sms) * per_sm;
  if (SHIFT) grid = grid / 8 * 8;
  if (grid > p.rows) grid = p.rows;
  p.depth = g.depth;
  BW_CUDA(launch_dependent(KERN, dim3(static_cast<unsigned>(grid)), g.block, g.smem, s, p));
  return BW_OK;
}

template <typename T, typename WT, bool Q8, int VE, bool SHIFT>
int launch_norm(const NormParams& p, cudaStream_t s, const DeviceState& d) {
  constexpr int kMaxNv = VE == 1 ? 16 : sizeof(T) == 4 ? 8 : 4;
  const long long nvec = SHIFT ? p.cols / VE : (p.cols + VE - 1LL) / VE;
  if constexpr (VE > 1) {
    const Shape sh = row_shape(p.rows, nvec, 4, kMaxNv, 1, d.sms);
    // rows of whole vectors whose blocks leave few of an SM's 512 x 4 vectors unused
    const bool full = !SHIFT && sh.nv == 4 && kMaxThreads / sh.block * nvec >= 1700;
    if (nvec > 128 && p.rows * nvec > d.sms * 512LL && !full) {
      const Staging g = row_staging(nvec, 4, sizeof(T) == 4 ? 8 : 4, p.res ? 2 : 1, 768);
      if (g.depth > 0 && g.nv == 4) return launch_staged<k_rmsnorm_staged<T, WT, Q8, VE, 4, SHIFT>, SHIFT>(p, g, s, d);
      if constexpr (sizeof(T) == 4)
        if (g.depth > 0) return launch_staged<k_rmsnorm_staged<T, WT, Q8, VE, 8, SHIFT>, SHIFT>(p, g, s, d);
    }
  }
  const Shape sh = row_shape(p.rows, nvec, SHIFT && nvec <= 32 ? 1 : 4, kMaxNv, SHIFT ? 16 : 1, d.sms);
  if (sh.nv == 0) {
    constexpr int WVE = SHIFT ? 1 : VE;
    BW_CUDA(launch_dependent(k_rmsnorm_wide<T, WT, Q8, WVE>, dim3(static_cast<unsigned>(p.rows)), 1024, 0, s, p));
    return BW_OK;
  }
  switch (sh.nv) {
    case 1: return launch_rows<k_rmsnorm<T, WT, Q8, VE, 1, SHIFT>, SHIFT>(p, sh, s, d);
    case 2: return launch_rows<k_rmsnorm<T, WT, Q8, VE, 2, SHIFT>, SHIFT>(p, sh, s, d);
    case 4: return launch_rows<k_rmsnorm<T, WT, Q8, VE, 4, SHIFT>, SHIFT>(p, sh, s, d);
    case 8:
      if constexpr (kMaxNv >= 8) return launch_rows<k_rmsnorm<T, WT, Q8, VE, 8, SHIFT>, SHIFT>(p, sh, s, d);
      [[fallthrough]];
    default:
      if constexpr (kMaxNv >= 16) return launch_rows<k_rmsnorm<T, WT, Q8, VE, 16, SHIFT>, SHIFT>(p, sh, s, d);
      return BW_OK;  // row_shape gives no more than kMaxNv
  }
}

template <typename T, typename WT, bool Q8>
int dispatch_norm(NormParams p, cudaStream_t s, const DeviceState& d) {
  constexpr int VE = 16 / sizeof(T);
  const int e = sizeof(T);
  const RowsOf t[] = {{p.x, p.ldx, e}, {p.res, p.ldr, e}, {p.h, p.ldh, e}, {p.y, p.ldy, Q8 ? 1 : e}};
  switch (row_access(t, VE, p.cols, &p.phase)) {
    case Access::ALIGNED:
      if (aligned16(p.w)) return launch_norm<T, WT, Q8, VE, false>(p, s, d);
      [[fallthrough]];
    case Access::SHIFTED: return launch_norm<T, WT, Q8, VE, true>(p, s, d);
    default: return launch_norm<T, WT, Q8, 1, false>(p, s, d);
  }
}

template <typename T>
int dispatch_weight(const NormParams& p, bool q8, cudaStream_t s, const DeviceState& d) {
  if constexpr (sizeof(T) < 4)
    if (p.w_f32) return q8 ? dispatch_norm<T, float, true>(p, s, d) : dispatch_norm<T, float, false>(p, s, d);
  return q8 ? dispatch_norm<T, T, true>(p, s, d) : dispatch_norm<T, T, false>(p, s, d);
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

// An output over an input: row by row, so both need one pitch.
int check_in_place(const char* out, const void* o, long long ldo, const char* in, const void* i, long long ldi, int rows) {
  if (o && o == i && rows > 1 && ldo != ldi)
    return set_error(BW_ERR_INVALID, "%s over %s: row pitches %lld and %lld differ", out, in, ldo, ldi);
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
  if (y == h) return set_error(BW_ERR_INVALID, "%s and h are one buffer", q8 ? "q" : "y");
  if (q8 && (y == x || y == residual)) return set_error(BW_ERR_INVALID, "q over an input: elements of different size");
  if ((r = check_in_place("y", y, ldy, "x", x, ldx, rows)) != BW_OK ||
      (r = check_in_place("y", y, ldy, "residual", residual, ldr, rows)) != BW_OK ||
      (r = check_in_place("h", h, ldh, "x", x, ldx, rows)) != BW_OK ||
      (r = check_in_place("h", h, ldh, "residual", residual, ldr, rows)) != BW_OK)
    return r;
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
  p.inv_cols = 1.f / static_cast<float>(cols);
  p.status = d->status;
  p.budget_ns = wait_budget_ns();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BW_DTYPE_F32) return dispatch_weight<float>(p, q8, s, *d);
  if (dtype == BW_DTYPE_F16) return dispatch_weight<__half>(p, q8, s, *d);
  return dispatch_weight<__nv_bfloat16>(p, q8, s, *d);
}

// Slabs of the weight gradient that the workspace has room for, one a block: a function of the sizes alone, so that the
// workspace is the same on every device and for every layout. 512 threads are resident on an SM (of 148) with this
// kernel's registers (640 with the staged one's), and a block has one for 16 columns, or 256 for short rows; more
// slabs wait for those to end (a whole second wave, 37476 x 3519 BF16: 267 us with 296, 411 with 338) and write more partial
// sums (16384 x 8192 BF16: 180 us with 148, 199 with 592).
int grad_slabs(long long rows, long long cols) {
  long long most = 296;
  constexpr int kSms = 148;
  if (cols > 512 && cols <= 16384) {
    const int threads = cols > 8192 ? 512 : static_cast<int>((cols + 511) / 512 * 32);
    most = kSms * ((threads > 256 ? 640 : 512) / threads);
  }
  if (cols <= 16384 && most > rows / 4) most = rows / 4 > kSms ? rows / 4 : kSms;
  return static_cast<int>(rows < most ? rows : most);
}

int sum_slabs(const NormGradParams& p, float* dw, cudaStream_t s) {
  BW_CUDA(launch_dependent(k_sum_slabs, dim3(static_cast<unsigned>((p.cols + 31LL) / 32)), 1024, 0, s,
                           static_cast<const float*>(p.partial), dw, p.slabs, p.cols));
  return BW_OK;
}

// A slab (block) for every row up to the workspace's slabs, and no more blocks than one wave holds by its
// ring and registers.
template <auto KERN, bool SHIFT>
int launch_grad_staged(NormGradParams p, const Staging& g, float* dw, cudaStream_t s, const DeviceState& d) {
  int per_sm = 0;
  const int r = staged_resident<KERN>(g, &per_sm);
  if (r != BW_OK) return r;
  int most = d.sms * per_sm;
  if (most > p.slabs) most = p.slabs;
  if (SHIFT && most > 8) most = most / 8 * 8;
  p.slabs = p.rows < most ? static_cast<int>(p.rows) : most;
  p.depth = g.depth;
  BW_CUDA(launch_dependent(KERN, dim3(p.slabs), g.block, g.smem, s, p));
  return sum_slabs(p, dw, s);
}

template <typename T, typename WT, int VE, bool SHIFT>
int launch_grad(NormGradParams p, float* dw, cudaStream_t s, const DeviceState& d) {
  constexpr int kMaxNv = VE == 1 ? 16 : sizeof(T) == 4 ? 8 : 4;
  const long long nvec = SHIFT ? p.cols / VE : (p.cols + VE - 1LL) / VE;
  if constexpr (VE > 1) {
    if (nvec > 64 && p.rows >= 8LL * p.slabs) {
      constexpr int kNv = sizeof(T) == 4 ? 4 : 2;
      const Staging g = row_staging(nvec, kNv, 4, p.dres ? 3 : 2, 512);
      if (g.depth > 0 && g.nv == kNv) return launch_grad_staged<k_rmsnorm_grad_staged<T, WT, VE, kNv, SHIFT>, SHIFT>(p, g, dw, s, d);
      if constexpr (kNv == 2)
        if (g.depth > 0) return launch_grad_staged<k_rmsnorm_grad_staged<T, WT, VE, 4, SHIFT>, SHIFT>(p, g, dw, s, d);
    }
  }
  // 32 bytes of a row a thread (it fetches ahead then), 64 for long sums in FP32
  const Shape sh = row_shape(p.rows, nvec, sizeof(T) == 4 && p.rows >= 2048 ? 4 : 2, kMaxNv, SHIFT ? 16 : 1, d.sms);
  if (sh.nv == 0) {
    // the weight gradient first: dx may be written over dy or h
    BW_CUDA(launch_dependent(k_rmsnorm_dw_wide<T>, dim3(static_cast<unsigned>((p.cols + 255LL) / 256), p.slabs), 256, 0, s, p));
    BW_CUDA(launch_dependent(k_rmsnorm_grad_wide<T, WT>, dim3(static_cast<unsigned>(p.rows)), 1024, 0, s, p));
  } else {
    if (sh.tpr > 32 && p.slabs > d.sms * (kMaxThreads / sh.block)) p.slabs = d.sms * (kMaxThreads / sh.block);
    const long long groups = (p.rows + sh.groups - 1) / sh.groups;
    if (groups <= p.slabs) p.slabs = static_cast<int>(groups);  // a row each
    else if (SHIFT && sh.groups < 8) p.slabs = p.slabs / 8 * 8;  // a stride of whole phases
    const size_t smem = sh.tpr > 32 ? 0 : static_cast<size_t>(sh.groups) * p.cols * sizeof(float);
    auto go = [&](auto kern) { return launch_dependent(kern, dim3(p.slabs), sh.block, smem, s, p, sh.tpr); };
    switch (sh.nv) {
      case 1: BW_CUDA(go(k_rmsnorm_grad<T, WT, VE, 1, SHIFT>)); break;
      case 2: BW_CUDA(go(k_rmsnorm_grad<T, WT, VE, 2, SHIFT>)); break;
      case 4: BW_CUDA(go(k_rmsnorm_grad<T, WT, VE, 4, SHIFT>)); break;
      case 8:
        if constexpr (kMaxNv >= 8) BW_CUDA(go(k_rmsnorm_grad<T, WT, VE, 8, SHIFT>));
        break;
      default:
        if constexpr (kMaxNv >= 16) BW_CUDA(go(k_rmsnorm_grad<T, WT, VE, 16, SHIFT>));
        break;
    }
  }
  return sum_slabs(p, dw, s);
}

template <typename T, typename WT>
int dispatch_grad(NormGradParams p, float* dw, cudaStream_t s, const DeviceState& d) {
  constexpr int VE = 16 / sizeof(T);
  const int e = sizeof(T);
  const RowsOf t[] = {{p.h, p.ldh, e}, {p.dy, p.lddy, e}, {p.dres, p.lddr, e}, {p.dx, p.lddx, e}};
  switch (row_access(t, VE, p.cols, &p.phase)) {
    case Access::ALIGNED:
      if (aligned16(p.w)) return launch_grad<T, WT, VE, false>(p, dw, s, d);
      [[fallthrough]];
    case Access::SHIFTED: return launch_grad<T, WT, VE, true>(p, dw, s, d);
    default: return launch_grad<T, WT, 1, false>(p, dw, s, d);
  }
}

template <typename T>
int dispatch_grad_weight(const NormGradParams& p, float* dw, cudaStream_t s, const DeviceState& d) {
  if constexpr (sizeof(T) < 4)
    if (p.w_f32) return dispatch_grad<T, float>(p, dw, s, d);
  return dispatch_grad<T, T>(p, dw, s, d);
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
  return static_cast<size_t>(grad_slabs(rows, cols)) * cols * sizeof(float);
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
  if ((r = check_in_place("dx", dx, lddx, "dy", dy, lddy, rows)) != BW_OK ||
      (r = check_in_place("dx", dx, lddx, "h", h, ldh, rows)) != BW_OK ||
      (r = check_in_place("dx", dx, lddx, "dresidual", dresidual, lddr, rows)) != BW_OK)
    return r;
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
  p.slabs = grad_slabs(rows, cols);
  p.status = d->status;
  p.budget_ns = wait_budget_ns();
  if (dtype == BW_DTYPE_F32) return dispatch_grad_weight<float>(p, dweight, s, *d);
  if (dtype == BW_DTYPE_F16) return dispatch_grad_weight<__half>(p, dweight, s, *d);
  return dispatch_grad_weight<__nv_bfloat16>(p, dweight, s, *d);
}

}  // extern "C"
