// Shared pieces of the sequence operators (seq_norm.hip, seq_linear.hip, seq_conv.hip, seq_scan.hip): element types fp16 / bf16 / fp32,
// row access in pieces of eight at aligned and at any addresses, activations, and the ordered reduction of per-block partial rows.
#pragma once
#include "seg_common.h"
#include <math.h>
#include <type_traits>

namespace {

typedef __bf16 bf16_t;
typedef bf16_t b8 __attribute__((ext_vector_type(8)));

// eight consecutive elements <-> eight floats.  VEC: 16-byte accesses (32 bytes in fp32: two) at aligned addresses, all or none (n <= 0)
// of the eight; else the first n (<= 8) exist - the others read as zero and are not written - and the address is any element's: whole
// eights are still one or two accesses (this card takes them at any address; element by element 8 x 4096 x 2050 f16 rows took the
// causal convolution 230 us instead of 74), the ends of rows go one by one
template <typename T, bool VEC> __device__ __forceinline__ auto raw_load8(const T* p, int n) {
  typedef T tv __attribute__((ext_vector_type(8)));
  tv v = tv{};
  if constexpr (VEC) {
    if (n > 0) v = *reinterpret_cast<const tv*>(p);
  } else if (n >= 8) {
    __builtin_memcpy(&v, p, sizeof(v));
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) v[j] = p[j];
  }
  return v;
}
template <typename T> __device__ __forceinline__ void vload8(const T* p, float* f) {
  if constexpr (std::is_same<T, float>::value) {
    load8<float>(p, f);
  } else if constexpr (std::is_same<T, half_t>::value) {
    unpack8(ld16(p), f);
  } else {
    const u4 v = ld16(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(v[i] << 16);
      f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
}
template <typename T> __device__ __forceinline__ void vstore8(T* p, const float* f) {
  if constexpr (std::is_same<T, float>::value) {
    store8<float>(p, f);
  } else if constexpr (std::is_same<T, half_t>::value) {
    st16(p, pack8(f));
  } else {
    b8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (bf16_t)f[i];
    st16(p, __builtin_bit_cast(u4, v));
  }
}
template <typename T, bool VEC> __device__ __forceinline__ void row_load8(const T* p, int n, float* f) {
  if constexpr (VEC) {
    if (n > 0) {
      vload8(p, f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = 0.f;
    }
  } else {
    const auto v = raw_load8<T, false>(p, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
  }
}
template <typename T, bool VEC> __device__ __forceinline__ void row_store8(T* p, int n, const float* f) {
  if constexpr (VEC) {
    if (n > 0) vstore8(p, f);
  } else {
    typedef T tv __attribute__((ext_vector_type(8)));
    tv v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (T)f[i];                // (rounded in front of the branch, as above: rows of either kind get the same bits)
    if (n >= 8) {
      __builtin_memcpy(p, &v, sizeof(v));
    } else {
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < n) p[i] = v[i];
    }
  }
}

// relative error, measured over |v| <= 80 in half steps of 2^-24: 3 for |v| < 1, about |v| in the left tail (the exponential's argument is
// rounded), 2 to the right; silu the same.  The slope s (1 + v (1 - s)) is off by up to 16 of these absolutely (1 - s loses its low bits to the right)
__device__ __forceinline__ float sigmoid_f(float v) { return __builtin_amdgcn_rcpf(1.f + __expf(-v)); }
// At +-inf the activations and their slopes take their limits: a factor v meets one that is 0 in 32 bits from |v| = 100 on, and inf * 0
// would be NaN.  The factor is cut far behind that - no finite v changes its result -, and a NaN stays one by way of the other factor.
constexpr float ACT_FAR = 128.f;
__device__ __forceinline__ float silu_f(float v) { return __builtin_amdgcn_fmed3f(v, -ACT_FAR, INFINITY) * sigmoid_f(v); }
__device__ __forceinline__ float silu_slope_f(float v) {
  const float s = sigmoid_f(v);
  float far = ACT_FAR;
  asm("" : "+s"(far));                                         // (one scalar register for both ends: as literals either end costs a move each time)
  return s * (1.f + __builtin_amdgcn_fmed3f(v, -far, far) * (1.f - s));
}
// Phi(-|v|) = erfc(|v| / sqrt 2) / 2 = Q e with e = exp(-v^2 / 2), and ve = |v| e.  erfc(x) exp(x^2) = t P(t) with t = 1 / (1 + 0.3 x), P of degree 8
// fitted to a relative error of 2e-8 on 0 <= x <= 9.5 (behind it both factors are 0 in 32 bits), at about 20 instructions - half of the
// library's erff, and the derivative's Gaussian comes with it.  GELU's relative error as evaluated, in half steps of 2^-24: 9 for |v| < 1,
// 16 to -4, 53 to -8, 134 to -13 (v^2 is rounded in front of the exponential), where 1 + erf has no bits left; 2 to the right of 1.
// 0 <= ve <= 0.61: cut to [0, 1] - a modifier of the product's instruction - it is what it was, but for inf * 0, which becomes 0.
__device__ __forceinline__ float phi_neg(float v, float& e, float& ve) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.21213203435596426f, fabsf(v), 1.f));
  e = __builtin_amdgcn_exp2f(-0.72134752044448170f * v * v);
  ve = __builtin_amdgcn_fmed3f(fabsf(v) * e, 0.f, 1.f);
  float P = -0.12943415125844135f;
  P = fmaf(P, t, 0.48509680347354195f);
  P = fmaf(P, t, -0.5112271909366609f);
  P = fmaf(P, t, 0.5463959258695201f);
  P = fmaf(P, t, -0.09363188029990382f);
  P = fmaf(P, t, 0.2144365590320213f);
  P = fmaf(P, t, 0.1484823543501283f);
  P = fmaf(P, t, 0.17069194623730768f);
  P = fmaf(P, t, 0.16918961408577482f);
  return 0.5f * t * P;
}

__device__ __forceinline__ float seq_act(float v, int act, float alpha) {
  switch (act) {
    case SEG_ACT_RELU: return v <= 0.f ? 0.f : v;              // (a NaN stays one, here and in the slope: the gradient passes, as torch's)
    case SEG_ACT_LEAKY: return v > 0.f ? v : v * alpha;
    case SEG_ACT_SIGMOID: return sigmoid_f(v);
    case SEG_ACT_SILU: return silu_f(v);
    case SEG_ACT_GELU: { float e, ve; const float Q = phi_neg(v, e, ve); return fmaf(-Q, ve, fmaxf(v, 0.f)); }      // v Phi(v)
    default: return v;
  }
}
// derivative from the activation's INPUT
__device__ __forceinline__ float seq_act_slope(float v, int act, float alpha) {
  switch (act) {
    case SEG_ACT_RELU: return v <= 0.f ? 0.f : 1.f;
    case SEG_ACT_LEAKY: return v > 0.f ? 1.f : alpha;
    case SEG_ACT_SIGMOID: { const float s = sigmoid_f(v); return s * (1.f - s); }
    case SEG_ACT_SILU: return silu_slope_f(v);
    case SEG_ACT_GELU: {                                       // g: the slope at -|v|; the two add up to 1
      float e, ve;
      const float Q = phi_neg(v, e, ve), g = fmaf(ve, -0.39894228040143268f, Q * e);
      return v < 0.f ? g : 1.f - g;
    }
    default: return 1.f;
  }
}

// eight at a time, the (launch-uniform) choice taken once
#define SEQ_ACT8_CASES(F)                                                                        \
  switch (act) {                                                                                 \
    case SEG_ACT_RELU: F(SEG_ACT_RELU) break;                                                    \
    case SEG_ACT_LEAKY: F(SEG_ACT_LEAKY) break;                                                  \
    case SEG_ACT_SIGMOID: F(SEG_ACT_SIGMOID) break;                                              \
    case SEG_ACT_SILU: F(SEG_ACT_SILU) break;                                                    \
    case SEG_ACT_GELU: F(SEG_ACT_GELU) break;                                                    \
    default: break;                                                                              \
  }
__device__ __forceinline__ void act8(float* v, int act, float alpha) {
#define SEQ_F(A) { _Pragma("unroll") for (int t = 0; t < 8; ++t) v[t] = seq_act(v[t], A, alpha); }
  SEQ_ACT8_CASES(SEQ_F)
#undef SEQ_F
}
__device__ __forceinline__ void slope8(float* v, const float* z, int act, float alpha) {
#define SEQ_F(A) { _Pragma("unroll") for (int t = 0; t < 8; ++t) v[t] *= seq_act_slope(z[t], A, alpha); }
  SEQ_ACT8_CASES(SEQ_F)
#undef SEQ_F
}
#undef SEQ_ACT8_CASES

// out[c] = sum over parts of part[p * ld + c], in a fixed order: 16 columns x R rows of threads per block, a thread adds its parts in turn
// (four running sums), the rows are added in order.  Up to two sets of columns in one launch.
struct ColsumSet { const float* part; int64_t nparts, ld, cols; float* out; };
template <int R>
__global__ __launch_bounds__(16 * R) void colsum_parts_kernel(const ColsumSet s0, const ColsumSet s1, int64_t blocks0) {
  const bool second = (int64_t)blockIdx.x >= blocks0;
  const ColsumSet s = second ? s1 : s0;
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int64_t col = ((int64_t)blockIdx.x - (second ? blocks0 : 0)) * 16 + c;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (col < s.cols) {
    const float* p = s.part + col;
    int64_t k = r;
    for (; k + 3 * R < s.nparts; k += 4 * R) {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += p[(k + q * R) * s.ld];
    }
    for (int q = 0; k < s.nparts; k += R, ++q) v[q] += p[k * s.ld];
  }
  __shared__ float sh[R][17];
  sh[r][c] = (v[0] + v[1]) + (v[2] + v[3]);
  __syncthreads();
  if (r == 0 && col < s.cols) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) t += sh[i][c];
    s.out[col] = t;
  }
}
inline void launch_colsum_sets(const ColsumSet& s0, const ColsumSet& s1, hipStream_t st) {
  // (2^21 blocks of 1024 threads: more columns go by pieces, see grid_takes below)
  constexpr int64_t MOST = (int64_t)1 << 24;
  if (s0.cols + s1.cols > 2 * MOST) {
    for (const ColsumSet* s : {&s0, &s1})
      for (int64_t c = 0; c < s->cols; c += MOST)
        launch_colsum_sets({s->part == nullptr ? nullptr : s->part + c, s->nparts, s->ld, s->cols - c < MOST ? s->cols - c : MOST, s->out + c}, {nullptr, 0, 0, 0, nullptr}, st);
    return;
  }
  const int64_t b0 = (s0.cols + 15) / 16, b1 = (s1.cols + 15) / 16, most = s0.nparts > s1.nparts ? s0.nparts : s1.nparts;
  if (b0 + b1 == 0) return;
  // many parts: four times the threads on the same columns (1024 parts of 128 columns: 20 us with 16 rows of threads)
  if (most > 64) hipLaunchKernelGGL(colsum_parts_kernel<64>, dim3((unsigned)(b0 + b1)), dim3(1024), 0, st, s0, s1, b0);
  else hipLaunchKernelGGL(colsum_parts_kernel<16>, dim3((unsigned)(b0 + b1)), dim3(256), 0, st, s0, s1, b0);
}
// part rows hold n0 + n1 neighbouring columns that belong to out0 and out1 (either may be NULL): one set where the outputs are neighbours too
inline void launch_colsum_pair(const float* part, int64_t nparts, int64_t ld, int64_t n0, float* out0, int64_t n1, float* out1, hipStream_t st) {
  ColsumSet a{part, nparts, ld, out0 != nullptr ? n0 : 0, out0}, b{part == nullptr ? nullptr : part + n0, nparts, ld, out1 != nullptr ? n1 : 0, out1};
  if (out0 != nullptr && out1 == out0 + n0) { a.cols = n0 + n1; b.cols = 0; }
  launch_colsum_sets(a, b, st);
}

// an axis of a grid takes fewer than 2^32 threads: a larger one comes out as its low 32 bits, without an error
inline bool grid_takes(int64_t threads) { return threads < (int64_t)1 << 32; }
inline size_t dt_size(int dt) { return dt == SEG_DT_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// whether 8-element vector accesses fit a tensor's rows (NULL: not there, fits)
inline bool vec_ok(const void* p, int64_t ld, int64_t bs, int dt) {
  const int64_t u = dt == SEG_DT_F32 ? 4 : 8;
  return p == nullptr || (aligned16(p) && ld % u == 0 && bs % u == 0);
}

template <typename F>
inline int seq_dispatch_dtype(int dt, F&& f) {
  if (dt == SEG_DT_F16) f((half_t*)nullptr);
  else if (dt == SEG_DT_BF16) f((bf16_t*)nullptr);
  else f((float*)nullptr);
  return 0;
}

}  // namespace
