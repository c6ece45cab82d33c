// Layer normalisation of rows of channels, forward and backward (seg_layernorm_fwd / _bwd).
//
//   mean = sum x / C,  var = sum (x - mean)^2 / C,  y = (x - mean) rstd gamma + beta
//   dx = rstd (g - sum g / C - xhat sum (g xhat) / C),  g = dy gamma;   dgamma = sum_rows dy xhat,  dbeta = sum_rows dy
//
// Bandwidth bounds both: the row is read ONCE and kept in registers, so the variance is the two-pass one (no cancellation of
// sum x^2 - mean^2) at no traffic.  LPR lanes share a row - 8 lanes for the 64-channel rows of a full-resolution level, a wave, or
// the whole block - with NCH chunks of 8 channels per lane; rows longer than a block's registers are walked in a loop.
//
// Measured: forward 4096 x 1024 f16 6.6 us (2.5 TB/s: one memory latency per block is what is left); backward 1 048 576 x 64 f16 75 us
// (5.4 TB/s; a large copy reaches 4.9) and 4.7 us for the blocks' sums; 5003 x 1111 f32, 4-byte accesses, 17.6 us (3.8 TB/s) and 4.3 us.
#include "seq_common.h"

namespace {

constexpr int TPB = 256;
constexpr int64_t LN_REG_MAX = 256 * 8 * 8;      // longest row held in registers: 256 lanes x 8 chunks x 8 channels

// sum over the LPR lanes of a row (LPR <= 64: inside the wave; 256: the block, through `sh`)
template <int LPR> __device__ __forceinline__ float row_sum(float v, float* sh) {
#pragma unroll
  for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (LPR > 64) {
    const int w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[w] = v;
    __syncthreads();
    v = sh[0] + sh[1] + sh[2] + sh[3];
  }
  return v;
}
template <int LPR> __device__ __forceinline__ void row_sum2(float& a, float& b, float* sh) {
#pragma unroll
  for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1) {
    a += __shfl_xor(a, o);
    b += __shfl_xor(b, o);
  }
  if constexpr (LPR > 64) {
    const int w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { sh[w] = a; sh[4 + w] = b; }
    __syncthreads();
    a = sh[0] + sh[1] + sh[2] + sh[3];
    b = sh[4] + sh[5] + sh[6] + sh[7];
  }
}

// The mean's sum rounds: it is off by a few steps of the row's offset, which counts where the row's spread is small against that.  Such a row
// (spread below 1 / 16 of the mean) adds up what is left, sum (x - mean) - differences that are exact, or nearly so, there - and takes the
// variance about the corrected mean: a row of constants has exactly its value for a mean, and y is exactly beta.  The other rows pay for one
// comparison (8192 x 4096 f16 26 us; with the sum of the differences taken for every row 28.5).
__device__ __forceinline__ bool far_row(float mean, float var) { return mean * mean * (1.f / 256.f) > var; }

// chunk i of a lane covers channels c0 .. c0 + n: with VEC 8 consecutive ones per lane, else the lanes' channels interleave (j LPR apart)
// so that scalar accesses of neighbouring lanes stay neighbours (5003 x 1111 f32 backward 17.4 us; eight neighbours per lane at any address 26)
template <typename T, bool VEC, int LPR> struct Chunk {
  int l;
  __device__ __forceinline__ int chan(int i, int j) const { return VEC ? (l + LPR * i) * 8 + j : l + LPR * (i * 8 + j); }
  __device__ __forceinline__ void load(const T* row, int i, int C, float* f) const {
    if constexpr (VEC) {
      row_load8<T, true>(row + (l + LPR * i) * 8, C - (l + LPR * i) * 8, f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = chan(i, j) < C ? (float)row[chan(i, j)] : 0.f;
    }
  }
  __device__ __forceinline__ void loadf(const float* p, float none, int i, int C, float* f) const {
    if (p == nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = none;
    } else if constexpr (VEC) {
      const int c = (l + LPR * i) * 8;
      if (c < C) {
        load8<float>(p + c, f);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = chan(i, j) < C ? p[chan(i, j)] : 0.f;
    }
  }
  template <typename U> __device__ __forceinline__ void store(U* row, int i, int C, const float* f) const {
    if constexpr (VEC) {
      row_store8<U, true>(row + (l + LPR * i) * 8, C - (l + LPR * i) * 8, f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (chan(i, j) < C) row[chan(i, j)] = (U)f[j];
    }
  }
};

template <typename T, bool VEC, int LPR, int NCH>
__global__ __launch_bounds__(TPB) void ln_fwd_kernel(const T* x, int64_t x_ld, T* y, int64_t y_ld, int64_t rows, int C, const float* gamma,
                                                     const float* beta, float eps, float* mean_o, float* rstd_o) {
  constexpr int RPB = TPB / LPR;
  __shared__ float sh[8];
  const Chunk<T, VEC, LPR> ck{(int)(threadIdx.x % LPR)};
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + threadIdx.x / LPR;
    const bool live = row < rows;                 // (always where a row takes the whole block)
    float v[NCH][8];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      ck.load(x + row * x_ld, i, live ? C : 0, v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[i][j];
    }
    float mean = row_sum<LPR>(s, sh) / (float)C;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] -= mean;
        if (ck.chan(i, j) < C) q = fmaf(v[i][j], v[i][j], q);
      }
    float var = row_sum<LPR>(q, sh) / (float)C;
    if (far_row(mean, var)) {                                  // (the same for all lanes of a row)
      float r = 0.f;
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) r += ck.chan(i, j) < C ? v[i][j] : 0.f;
      const float m0 = mean;
      mean += row_sum<LPR>(r, sh) / (float)C;
      const float shift = mean - m0;
      q = 0.f;
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[i][j] -= shift;
          if (ck.chan(i, j) < C) q = fmaf(v[i][j], v[i][j], q);
        }
      var = row_sum<LPR>(q, sh) / (float)C;
    }
    const float rstd = 1.f / sqrtf(var + eps);
    if (live) {
      if (ck.l == 0) {
        if (mean_o != nullptr) mean_o[row] = mean;
        if (rstd_o != nullptr) rstd_o[row] = rstd;
      }
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        float g[8], b[8];
        ck.loadf(gamma, 1.f, i, C, g);
        ck.loadf(beta, 0.f, i, C, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = fmaf(v[i][j] * rstd, g[j], b[j]);
        ck.store(y + row * y_ld, i, C, g);
      }
    }
  }
}

// eight channels of a long row per thread and turn, at any address
template <typename T> struct LongRow {
  __device__ __forceinline__ int first(int i) const { return ((int)threadIdx.x + TPB * i) * 8; }
  __device__ __forceinline__ void load(const T* row, int i, int C, float* f) const { row_load8<T, false>(row + first(i), C - first(i), f); }
  __device__ __forceinline__ void loadf(const float* p, float none, int i, int C, float* f) const {
    if (p == nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = none;
    } else {
      row_load8<float, false>(p + first(i), C - first(i), f);
    }
  }
  __device__ __forceinline__ void store(T* row, int i, int C, const float* f) const { row_store8<T, false>(row + first(i), C - first(i), f); }
};

// rows longer than LN_REG_MAX: one block per row, three walks over it (the second and third from the L2;
// 2000 x 20000 f16 51 us, 4 x 1048576 434)
template <typename T>
__global__ __launch_bounds__(TPB) void ln_fwd_long_kernel(const T* x, int64_t x_ld, T* y, int64_t y_ld, int64_t rows, int C, const float* gamma,
                                                          const float* beta, float eps, float* mean_o, float* rstd_o) {
  __shared__ float sh[8];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * x_ld;
    const LongRow<T> ck;
    float s = 0.f;
#pragma unroll 4
    for (int i = 0; ck.first(i) < C; ++i) {
      float v[8];
      ck.load(xr, i, C, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    float mean = row_sum<256>(s, sh) / (float)C, q = 0.f;
#pragma unroll 4
    for (int i = 0; ck.first(i) < C; ++i) {
      float v[8];
      ck.load(xr, i, C, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] -= mean;
        if (ck.first(i) + j < C) q = fmaf(v[j], v[j], q);
      }
    }
    float var = row_sum<256>(q, sh) / (float)C;
    if (far_row(mean, var)) {                                  // (two more walks)
      float r = 0.f;
      for (int i = 0; ck.first(i) < C; ++i) {
        float v[8];
        ck.load(xr, i, C, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) r += ck.first(i) + j < C ? v[j] - mean : 0.f;
      }
      mean += row_sum<256>(r, sh) / (float)C;
      q = 0.f;
      for (int i = 0; ck.first(i) < C; ++i) {
        float v[8];
        ck.load(xr, i, C, v);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (ck.first(i) + j < C) q = fmaf(v[j] - mean, v[j] - mean, q);
      }
      var = row_sum<256>(q, sh) / (float)C;
    }
    const float rstd = 1.f / sqrtf(var + eps);
    if (threadIdx.x == 0) {
      if (mean_o != nullptr) mean_o[row] = mean;
      if (rstd_o != nullptr) rstd_o[row] = rstd;
    }
    T* yr = y + row * y_ld;
    for (int i = 0; ck.first(i) < C; ++i) {
      float v[8], g[8], b[8];
      ck.load(xr, i, C, v);
      ck.loadf(gamma, 1.f, i, C, g);
      ck.loadf(beta, 0.f, i, C, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fmaf((v[j] - mean) * rstd, g[j], b[j]);
      ck.store(yr, i, C, v);
    }
  }
}

// A block walks rows blockIdx.x * RPB + gridDim.x * RPB * k and keeps its share of dgamma / dbeta in registers: one partial row pair
// per block at the end, part[block][2][C], added up in order by a second launch.
template <typename T, bool VEC, int LPR, int NCH>
__global__ __launch_bounds__(TPB) void ln_bwd_kernel(const T* dy, int64_t dy_ld, const T* x, int64_t x_ld, T* dx, int64_t dx_ld, int64_t rows, int C,
                                                     const float* mean_i, const float* rstd_i, const float* gamma, float* part) {
  constexpr int RPB = TPB / LPR;
  __shared__ float sh[8];
  __shared__ float comb[LPR < 256 ? (LPR <= 64 ? 4 * LPR * 16 : 1) : 1];
  const Chunk<T, VEC, LPR> ck{(int)(threadIdx.x % LPR)};
  const float inv = 1.f / (float)C;
  float g[NCH][8], dg[NCH][8], db[NCH][8];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    ck.loadf(gamma, 1.f, i, C, g[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dg[i][j] = db[i][j] = 0.f;
  }
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + threadIdx.x / LPR;
    const bool live = row < rows;
    const float mean = live ? mean_i[row] : 0.f, rstd = live ? rstd_i[row] : 0.f;
    float xh[NCH][8], d[NCH][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      ck.load(x + row * x_ld, i, live ? C : 0, xh[i]);
      ck.load(dy + row * dy_ld, i, live ? C : 0, d[i]);
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[i][j] = (xh[i][j] - mean) * rstd;
        dg[i][j] = fmaf(d[i][j], xh[i][j], dg[i][j]);        // (a channel that is not there has d = 0)
        db[i][j] += d[i][j];
        d[i][j] *= g[i][j];
        s1 += d[i][j];
        s2 = fmaf(d[i][j], xh[i][j], s2);
      }
    if (dx != nullptr) {                                     // (kernel-uniform)
      row_sum2<LPR>(s1, s2, sh);
      s1 *= inv;
      s2 *= inv;
      if (live) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
#pragma unroll
          for (int j = 0; j < 8; ++j) d[i][j] = rstd * (d[i][j] - s1 - xh[i][j] * s2);
          ck.store(dx + row * dx_ld, i, C, d[i]);
        }
      }
    }
  }
  if (part == nullptr) return;
  // rows of one wave, then the four waves (LPR = 256: a channel has one owner)
  float* out = part + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if constexpr (LPR <= 64) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1) {
          dg[i][j] += __shfl_xor(dg[i][j], o);
          db[i][j] += __shfl_xor(db[i][j], o);
        }
      __syncthreads();
      if ((threadIdx.x & 63) < LPR) {
        float* c = comb + ((threadIdx.x >> 6) * LPR + ck.l) * 16;
#pragma unroll
        for (int j = 0; j < 8; ++j) { c[j] = dg[i][j]; c[8 + j] = db[i][j]; }
      }
      __syncthreads();
      if (threadIdx.x < LPR) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          dg[i][j] = db[i][j] = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            dg[i][j] += comb[(w * LPR + ck.l) * 16 + j];
            db[i][j] += comb[(w * LPR + ck.l) * 16 + 8 + j];
          }
        }
      }
    }
    if (LPR == 256 || threadIdx.x < LPR) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (ck.chan(i, j) < C) {
          out[ck.chan(i, j)] = dg[i][j];
          out[C + ck.chan(i, j)] = db[i][j];
        }
    }
  }
}

// rows longer than LN_REG_MAX: dx by one block per row; dgamma / dbeta by columns, a block takes 256 channels x a range of rows
template <typename T>
__global__ __launch_bounds__(TPB) void ln_bwd_long_dx_kernel(const T* dy, int64_t dy_ld, const T* x, int64_t x_ld, T* dx, int64_t dx_ld, int64_t rows,
                                                             int C, const float* mean_i, const float* rstd_i, const float* gamma) {
  __shared__ float sh[8];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float mean = mean_i[row], rstd = rstd_i[row], inv = 1.f / (float)C;
    const T *xr = x + row * x_ld, *dr = dy + row * dy_ld;
    T* o = dx + row * dx_ld;
    const LongRow<T> ck;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll 2
    for (int i = 0; ck.first(i) < C; ++i) {
      float v[8], d[8], g[8];
      ck.load(xr, i, C, v);
      ck.load(dr, i, C, d);
      ck.loadf(gamma, 1.f, i, C, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) {                            // (a channel that is not there has d = 0)
        d[j] *= g[j];
        s1 += d[j];
        s2 = fmaf(d[j], (v[j] - mean) * rstd, s2);
      }
    }
    row_sum2<256>(s1, s2, sh);
    s1 *= inv;
    s2 *= inv;
    for (int i = 0; ck.first(i) < C; ++i) {
      float v[8], d[8], g[8];
      ck.load(xr, i, C, v);
      ck.load(dr, i, C, d);
      ck.loadf(gamma, 1.f, i, C, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = rstd * (d[j] * g[j] - s1 - (v[j] - mean) * rstd * s2);
      ck.store(o, i, C, d);
    }
  }
}
template <typename T>
__global__ __launch_bounds__(TPB) void ln_bwd_long_param_kernel(const T* dy, int64_t dy_ld, const T* x, int64_t x_ld, int64_t rows, int C,
                                                                const float* mean_i, const float* rstd_i, float* part) {
  const int c = blockIdx.x * TPB + threadIdx.x;
  if (c >= C) return;
  float dg = 0.f, db = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float d = (float)dy[r * dy_ld + c];
    db += d;
    dg = fmaf(d, ((float)x[r * x_ld + c] - mean_i[r]) * rstd_i[r], dg);
  }
  part[((int64_t)blockIdx.y * 2) * C + c] = dg;
  part[((int64_t)blockIdx.y * 2 + 1) * C + c] = db;
}

// lanes per row and chunks per lane for C channels: the fewest lanes that keep a row's chunks at four or fewer, a wave first
struct LnShape { int lpr, nch; };
inline LnShape ln_shape(int C) {
  const int chunks = (C + 7) / 8;
  for (int lpr : {8, 16, 32, 64})
    if (chunks <= lpr) return {lpr, 1};
  if (chunks <= 128) return {64, 2};
  if (chunks <= 256) return {64, 4};
  if (chunks <= 512) return {256, 2};
  if (chunks <= 1024) return {256, 4};
  return {256, 8};
}
// backward: five row-sized arrays per lane instead of one - rows of more than 512 channels take the whole block
inline LnShape ln_bwd_shape(int C) {
  const int chunks = (C + 7) / 8;
  return chunks <= 64 ? ln_shape(C) : chunks <= 256 ? LnShape{256, 1} : ln_shape(C);
}
template <typename F>
inline void ln_dispatch(const LnShape& s, F&& f) {
  using std::integral_constant;
#define LN_CASE(L, N) \
  if (s.lpr == L && s.nch == N) return f(integral_constant<int, L>{}, integral_constant<int, N>{});
  LN_CASE(8, 1) LN_CASE(16, 1) LN_CASE(32, 1) LN_CASE(64, 1) LN_CASE(64, 2) LN_CASE(64, 4) LN_CASE(256, 1) LN_CASE(256, 2) LN_CASE(256, 4) LN_CASE(256, 8)
#undef LN_CASE
}
// the kernels walk rows with the grid as stride: more blocks than this gain nothing
inline unsigned ln_grid(int64_t blocks) { return (unsigned)(blocks < (1 << 20) ? blocks : 1 << 20); }
inline int64_t ln_bwd_blocks(int64_t rows, int C) {
  if (C > LN_REG_MAX) return rows < 64 ? rows : 64;
  const int64_t rpb = TPB / ln_bwd_shape(C).lpr, groups = (rows + rpb - 1) / rpb;
  // every block leaves a partial row pair in 32 bits: at least eight rows per block keep that below a tenth of the traffic
  // (but a block per CU first: 1000 x 8192 f16 39 us with 125 blocks, 33 with 250)
  const int64_t most = 1024, share = rpb >= 4 ? 2 : 8 / rpb, want = (groups + share - 1) / share, least = groups < 256 ? groups : 256;
  return want < least ? least : want < most ? want : most;
}

bool ln_vec(std::initializer_list<const void*> ps, std::initializer_list<int64_t> lds, int C, int dt) {
  if (C % 8 != 0) return false;
  for (const void* p : ps)
    if (p != nullptr && !aligned16(p)) return false;
  for (int64_t l : lds)
    if (l % (dt == SEG_DT_F32 ? 4 : 8) != 0) return false;
  return true;
}

}  // namespace

extern "C" int seg_layernorm_fwd(const void* x, int64_t x_ld, void* y, int64_t y_ld, int64_t rows, int32_t C, int32_t dtype, const float* gamma,
                                 const float* beta, float eps, float* mean, float* rstd, seg_stream_t stream) {
  SEG_CHECK_ARG(dtype >= SEG_DT_F16 && dtype <= SEG_DT_F32, "layernorm_fwd: dtype %d", dtype);
  SEG_CHECK_ARG(rows >= 0 && C > 0 && C <= (1 << 30), "layernorm_fwd: rows %lld, C %d (2^30 at most)", (long long)rows, C);
  SEG_CHECK_ARG(rows <= 1 || (x_ld >= C && y_ld >= C), "layernorm_fwd: row strides below the %d channels", C);
  if (rows == 0) return SEG_OK;
  SEG_CHECK_ARG(x != nullptr && y != nullptr, "layernorm_fwd: x / y is NULL");
  SEG_CHECK_ARG(y != x || rows == 1 || y_ld == x_ld, "layernorm_fwd: y in place of x has another row stride");
  hipStream_t st = (hipStream_t)stream;
  seq_dispatch_dtype(dtype, [&](auto* tp) {
    typedef typename std::remove_pointer<decltype(tp)>::type T;
    if (C > LN_REG_MAX) {
      hipLaunchKernelGGL((ln_fwd_long_kernel<T>), dim3(ln_grid(rows)), dim3(TPB), 0, st, (const T*)x, x_ld, (T*)y, y_ld, rows, C, gamma, beta, eps, mean, rstd);
      return;
    }
    const LnShape s = ln_shape(C);
    const unsigned grid = ln_grid((rows + TPB / s.lpr - 1) / (TPB / s.lpr));
    ln_dispatch(s, [&](auto L, auto N) {
      if (ln_vec({x, y, gamma, beta}, {x_ld, y_ld}, C, dtype))
        hipLaunchKernelGGL((ln_fwd_kernel<T, true, L(), N()>), dim3(grid), dim3(TPB), 0, st, (const T*)x, x_ld, (T*)y, y_ld, rows, C, gamma, beta, eps, mean, rstd);
      else
        hipLaunchKernelGGL((ln_fwd_kernel<T, false, L(), N()>), dim3(grid), dim3(TPB), 0, st, (const T*)x, x_ld, (T*)y, y_ld, rows, C, gamma, beta, eps, mean, rstd);
    });
  });
  SEG_CHECK_LAUNCH("layernorm_fwd");
  return SEG_OK;
}

extern "C" int64_t seg_layernorm_bwd_workspace_bytes(int64_t rows, int32_t C, int32_t dtype) {
  (void)dtype;
  if (rows <= 0 || C <= 0) return 0;
  return ln_bwd_blocks(rows, C) * 2 * C * 4 + 2 * (int64_t)C * 4;
}

extern "C" int seg_layernorm_bwd(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, void* dx, int64_t dx_ld, int64_t rows, int32_t C,
                                 int32_t dtype, const float* mean, const float* rstd, const float* gamma, float* dgamma, float* dbeta,
                                 void* workspace, seg_stream_t stream) {
  SEG_CHECK_ARG(dtype >= SEG_DT_F16 && dtype <= SEG_DT_F32, "layernorm_bwd: dtype %d", dtype);
  SEG_CHECK_ARG(rows >= 0 && C > 0 && C <= (1 << 30), "layernorm_bwd: rows %lld, C %d (2^30 at most)", (long long)rows, C);
  SEG_CHECK_ARG(rows <= 1 || (x_ld >= C && dy_ld >= C && (dx == nullptr || dx_ld >= C)), "layernorm_bwd: row strides below the %d channels", C);
  const bool params = dgamma != nullptr || dbeta != nullptr;
  SEG_CHECK_ARG(rows == 0 || (dy != nullptr && x != nullptr && mean != nullptr && rstd != nullptr), "layernorm_bwd: dy / x / mean / rstd is NULL");
  SEG_CHECK_ARG(rows == 0 || !params || workspace != nullptr, "layernorm_bwd: dgamma / dbeta need the workspace");
  SEG_CHECK_ARG(rows <= 1 || dx == nullptr || ((dx != dy || dx_ld == dy_ld) && (dx != x || dx_ld == x_ld)), "layernorm_bwd: dx in place of dy / x has another row stride");
  hipStream_t st = (hipStream_t)stream;
  float* part = params ? (float*)workspace : nullptr;
  const int64_t nblk = rows > 0 ? ln_bwd_blocks(rows, C) : 0;
  if (rows > 0 && (params || dx != nullptr))
    seq_dispatch_dtype(dtype, [&](auto* tp) {
      typedef typename std::remove_pointer<decltype(tp)>::type T;
      if (C > LN_REG_MAX) {
        if (params)                               // (in front of dx, which may be dy or x)
          hipLaunchKernelGGL((ln_bwd_long_param_kernel<T>), dim3((C + TPB - 1) / TPB, (unsigned)nblk), dim3(TPB), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, rows, C, mean, rstd, part);
        if (dx != nullptr)
          hipLaunchKernelGGL((ln_bwd_long_dx_kernel<T>), dim3(ln_grid(rows)), dim3(TPB), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (T*)dx, dx_ld, rows, C, mean, rstd, gamma);
        return;
      }
      ln_dispatch(ln_bwd_shape(C), [&](auto L, auto N) {
        if (ln_vec({x, dy, dx, gamma}, {x_ld, dy_ld, dx == nullptr ? 0 : dx_ld}, C, dtype))
          hipLaunchKernelGGL((ln_bwd_kernel<T, true, L(), N()>), dim3((unsigned)nblk), dim3(TPB), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (T*)dx, dx_ld, rows, C, mean, rstd, gamma, part);
        else
          hipLaunchKernelGGL((ln_bwd_kernel<T, false, L(), N()>), dim3((unsigned)nblk), dim3(TPB), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (T*)dx, dx_ld, rows, C, mean, rstd, gamma, part);
      });
    });
  launch_colsum_pair(part, nblk, 2 * (int64_t)C, C, dgamma, C, dbeta, st);
  SEG_CHECK_LAUNCH("layernorm_bwd");
  return SEG_OK;
}
