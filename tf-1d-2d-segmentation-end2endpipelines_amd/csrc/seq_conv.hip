// Short causal convolution per channel, for prompts, training and single rows (seg_causal_conv_fwd / _bwd / _step).
//
//   xx = [state (K - 1 rows); x],  v[t] = bias + sum_k w[k] xx[t + k],  y[t] = act(v[t])
//   dv = dy act'(v),  dxx[r] = sum_k w[k] dv[r - k] (+ dstate_out on the rows the final state took),  dw[k] = sum dv[t] xx[t + k]
//
// Bandwidth bounds all three.  A thread owns 8 neighbouring channels (one 16-byte access per row) and walks a run of rows with the
// window of K rows in registers, so every row is read once per run plus K - 1 rows at its edges.
//
// Measured: forward 8 x 4096 x 2048 bf16, K = 4, half of the sequences shorter, 49 us (the bytes' floor 41, with whole sequences 55);
// backward 16 x 1024 x 512 f16 21 us for 50 MB: 57 instructions per element (11 rows recomputed for 8) are 12 us of the vector ALUs, and
// its 227 registers leave two waves per SIMD to hide the loads behind them.  K = 8 takes 313 us for 8 x 4096 x 2048 (120 with K = 4, the bytes 82).
#include "seq_common.h"

namespace {

constexpr int RUN = 16, RUN_SMALL = 8;          // rows per thread, forward / backward and small grids
constexpr int MAXK = 8;

// eight channels of a row in their memory format; n <= 0: zeros
template <typename T, bool VEC> struct Raw {
  typedef T tv __attribute__((ext_vector_type(8)));
  tv v;
  __device__ __forceinline__ void load(const T* p, int n) { v = raw_load8<T, VEC>(p, n); }
  __device__ __forceinline__ float operator[](int j) const { return (float)v[j]; }
};
// rows of xx = [state; x]: r < 0 is state row K - 1 + r.  x rows at or behind the length are not read
template <typename T, bool VEC, int K>
__device__ __forceinline__ void load_xx(const seg_causal_conv_args& p, int b, int r, int len, int c, Raw<T, VEC>& f) {
  if (r >= 0) f.load((const T*)p.x + b * p.x_bs + r * p.x_ld + c, r < len ? p.D - c : 0);
  else f.load((const T*)p.state + ((int64_t)b * (K - 1) + K - 1 + r) * p.D + c, p.state != nullptr ? p.D - c : 0);
}
template <bool VEC> __device__ __forceinline__ void load_par(const float* p, int n, float* f) {
  if (p == nullptr) n = 0;
  row_load8<float, VEC>(p, n, f);
}
__device__ __forceinline__ int conv_len(const seg_causal_conv_args& p, int b) {
  if (p.lengths == nullptr) return p.L;
  const int n = p.lengths[b];
  return n < 0 ? 0 : n > p.L ? p.L : n;
}
__device__ __forceinline__ float conv_act(float v, int act) { return act == SEG_ACT_SILU ? silu_f(v) : v; }

__device__ __forceinline__ unsigned conv_row_block(int split) { return (blockIdx.z & ((1u << split) - 1)) * gridDim.y + blockIdx.y; }

// threads: 32 channel groups of 8 x 8 runs of RUNS rows; grid (channels / 256, blocks of 8 runs, B).  An axis
// ends at 65535 blocks: more of them are cut into 2^split pieces, which share the third axis with B (on one axis with the channels, by a
// division: the prompt 54.5 us instead of 51.5).  A run's rows are all on their way before the
// first is used: one memory latency per run
template <typename T, bool VEC, int K, int RUNS>
__global__ __launch_bounds__(256) void conv_fwd_kernel(const seg_causal_conv_args p, int split) {
  const int c = (blockIdx.x * 32 + (threadIdx.x & 31)) * 8, b = blockIdx.z >> split;
  const int64_t run = (int64_t)conv_row_block(split) * 8 + (threadIdx.x >> 5);
  if (c >= p.D) return;
  const int len = conv_len(p, b), n = p.D - c;
  const int64_t t0l = run * RUNS;
  if (run == 0 && p.state_out != nullptr && K > 1) {          // one thread per channel group carries the state on
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      Raw<T, VEC> f;
      load_xx<T, VEC, K>(p, b, len - (K - 1) + k, len, c, f);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = f[j];
      row_store8<T, VEC>((T*)p.state_out + ((int64_t)b * (K - 1) + k) * p.D + c, n, v);
    }
  }
  if (t0l >= p.L) return;
  const int t0 = (int)t0l, t1 = t0 + RUNS < p.L ? t0 + RUNS : p.L;
  Raw<T, VEC> x[RUNS + K - 1];                                 // x[i]: row t0 - (K - 1) + i of xx
#pragma unroll
  for (int i = 0; i < RUNS + K - 1; ++i) load_xx<T, VEC, K>(p, b, t0 - (K - 1) + i, len, c, x[i]);
  float w[K][8], bias[8];
#pragma unroll
  for (int k = 0; k < K; ++k) load_par<VEC>(p.w + (int64_t)k * p.D + c, n, w[k]);
  load_par<VEC>(p.bias == nullptr ? nullptr : p.bias + c, n, bias);
  T* y = (T*)p.y + b * p.y_bs + c;
#pragma unroll
  for (int i = 0; i < RUNS; ++i) {
    const int t = t0 + i;
    if (t < t1) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = bias[j];
#pragma unroll
        for (int k = 0; k < K; ++k) v[j] = fmaf(w[k][j], x[i + k][j], v[j]);
        v[j] = t < len ? conv_act(v[j], p.act) : 0.f;
      }
      row_store8<T, VEC>(y + t * p.y_ld, n, v);
    }
  }
}

// The same run of rows backward: dv of rows t0 .. t0 + RUNS + K - 2 (each from its own window), dx[t] from the K dv behind it; dw / db
// from the run's own rows only, summed over the block's eight runs in LDS: part[block along rows and B][K + 1][D].
template <typename T, bool VEC, int K>
__global__ __launch_bounds__(256) void conv_bwd_kernel(const seg_causal_conv_args p, int split, float* part) {
  constexpr int RUNS = RUN_SMALL;
  const int cg = threadIdx.x & 31, c = (blockIdx.x * 32 + cg) * 8, b = blockIdx.z >> split;
  const int64_t run = (int64_t)conv_row_block(split) * 8 + (threadIdx.x >> 5), t0l = run * RUNS;
  const int len = conv_len(p, b), n = c < p.D ? p.D - c : 0;
  float dw[K + 1][8];
#pragma unroll
  for (int k = 0; k <= K; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[k][j] = 0.f;
  // rows of dx this thread writes: [t0, t1); the first run also owns the carried state's rows -(K - 1) .. -1
  if (n > 0 && (t0l < p.L || run == 0)) {
    const int t0 = (int)t0l, t1 = t0 + RUNS < p.L ? t0 + RUNS : p.L;
    Raw<T, VEC> x[RUNS + 2 * K - 2], dy[RUNS + K - 1];         // x[i]: row t0 - (K - 1) + i of xx;  dy[i]: row t0 + i
#pragma unroll
    for (int i = 0; i < RUNS + 2 * K - 2; ++i) load_xx<T, VEC, K>(p, b, t0 - (K - 1) + i, len, c, x[i]);
#pragma unroll
    for (int i = 0; i < RUNS + K - 1; ++i) dy[i].load((const T*)p.dy + b * p.dy_bs + (t0 + i) * p.dy_ld + c, t0 + i < len ? n : 0);
    float w[K][8], bias[8], dv[K][8];                          // dv[k] = dv of row r - (K - 1) + k
#pragma unroll
    for (int k = 0; k < K; ++k) load_par<VEC>(p.w + (int64_t)k * p.D + c, n, w[k]);
    load_par<VEC>(p.bias == nullptr ? nullptr : p.bias + c, n, bias);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) dv[k][j] = 0.f;
#pragma unroll
    for (int i = 0; i < RUNS + K - 1; ++i) {
      const int r = t0 + i;                                    // the row whose dv is computed; dx of row r - (K - 1) is complete then
      if (r < t1 + K - 1) {
        float d[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
          for (int k = 0; k + 1 < K; ++k) dv[k][j] = dv[k + 1][j];
          d[j] = dy[i][j];
          if (p.act == SEG_ACT_SILU) {
            float v = bias[j];
#pragma unroll
            for (int k = 0; k < K; ++k) v = fmaf(w[k][j], x[i + k][j], v);
            d[j] *= silu_slope_f(v);
          }
          d[j] = r < len ? d[j] : 0.f;
          dv[K - 1][j] = d[j];
        }
        if (r < t1 && r < len) {                               // (a padded row's 0 would meet whatever its window holds)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            dw[K][j] += d[j];
#pragma unroll
            for (int k = 0; k < K; ++k) dw[k][j] = fmaf(d[j], x[i + k][j], dw[k][j]);
          }
        }
        const int t = r - (K - 1);                             // dxx row t + K - 1: sum_k w[k] dv[t + K - 1 - k]
        const bool own = t >= t0 || (run == 0);                // (run 0: t >= -(K - 1))
        if (own && t < t1 && (t >= 0 ? p.dx != nullptr : p.dstate != nullptr)) {
          float g[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            g[j] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) g[j] = fmaf(w[k][j], dv[K - 1 - k][j], g[j]);
          }
          const int e = t - (len - (K - 1));                   // the final state's row that is xx row t
          if (K > 1 && p.dstate_out != nullptr && e >= 0 && e < K - 1) {
            float s[8];
            row_load8<T, VEC>((const T*)p.dstate_out + ((int64_t)b * (K - 1) + e) * p.D + c, n, s);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] += s[j];
          }
          if (t >= 0) row_store8<T, VEC>((T*)p.dx + b * p.dx_bs + t * p.dx_ld + c, n, g);
          else row_store8<T, VEC>((T*)p.dstate + ((int64_t)b * (K - 1) + K - 1 + t) * p.D + c, n, g);
        }
      }
    }
  }
  if (part == nullptr) return;
  __shared__ float sh[8][32][9];
  const int64_t row = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * (K + 1);
  const int ol = threadIdx.x >> 3, oj = threadIdx.x & 7, oc = (blockIdx.x * 32 + ol) * 8 + oj;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) sh[threadIdx.x >> 5][cg][j] = dw[k][j];
    __syncthreads();
    if (oc < p.D) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) v += sh[q][ol][oj];
      part[(row + k) * p.D + oc] = v;
    }
    __syncthreads();
  }
}

template <typename T, bool VEC, int K>
__global__ __launch_bounds__(256) void conv_step_kernel(const seg_causal_conv_args p) {
  const int groups = (p.D + 7) / 8;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= (int64_t)p.B * groups) return;
  const int b = (int)(e / groups), c = (int)(e % groups) * 8, n = p.D - c;
  float win[K][8], v[8];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) row_load8<T, VEC>((const T*)p.state + ((int64_t)b * (K - 1) + k) * p.D + c, p.state != nullptr ? n : 0, win[k]);
  row_load8<T, VEC>((const T*)p.x + b * p.x_bs + c, n, win[K - 1]);
  load_par<VEC>(p.bias == nullptr ? nullptr : p.bias + c, n, v);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float w[8];
    load_par<VEC>(p.w + (int64_t)k * p.D + c, n, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fmaf(w[j], win[k][j], v[j]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = conv_act(v[j], p.act);
  row_store8<T, VEC>((T*)p.y + b * p.y_bs + c, n, v);
  if (p.state_out != nullptr) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) row_store8<T, VEC>((T*)p.state_out + ((int64_t)b * (K - 1) + k) * p.D + c, n, win[k + 1]);
  }
}

template <typename F>
inline void conv_dispatch(const seg_causal_conv_args& a, bool vec, F&& f) {
  seq_dispatch_dtype(a.dtype, [&](auto* tp) {
    typedef typename std::remove_pointer<decltype(tp)>::type T;
#define CONV_K(k)                                                                        \
  case k:                                                                                \
    if (vec) f((T*)nullptr, std::true_type{}, std::integral_constant<int, k>{});         \
    else f((T*)nullptr, std::false_type{}, std::integral_constant<int, k>{});            \
    break;
    switch (a.K) { CONV_K(1) CONV_K(2) CONV_K(3) CONV_K(4) CONV_K(5) CONV_K(6) CONV_K(7) CONV_K(8) }
#undef CONV_K
  });
}
inline bool conv_vec(const seg_causal_conv_args& a, bool bwd) {
  if (a.D % 8 != 0 || !aligned16(a.w) || !aligned16(a.bias)) return false;
  bool ok = vec_ok(a.x, a.x_ld, a.x_bs, a.dtype) && vec_ok(a.state, 0, 0, a.dtype);
  if (bwd) return ok && vec_ok(a.dy, a.dy_ld, a.dy_bs, a.dtype) && vec_ok(a.dx, a.dx_ld, a.dx_bs, a.dtype) && vec_ok(a.dstate, 0, 0, a.dtype) && vec_ok(a.dstate_out, 0, 0, a.dtype);
  return ok && vec_ok(a.y, a.y_ld, a.y_bs, a.dtype) && vec_ok(a.state_out, 0, 0, a.dtype);
}
struct ConvGrid {
  dim3 blocks;
  int split;
  int64_t parts() const { return (int64_t)blocks.y * blocks.z; }           // partial rows of dw / db
};
inline ConvGrid conv_grid(const seg_causal_conv_args& a, int run) {
  const int64_t runs = ((int64_t)a.L + run - 1) / run, blocks = runs <= 8 ? 1 : (runs + 7) / 8;
  int split = 0;
  while (blocks > (int64_t)65535 << split) ++split;
  return {dim3((unsigned)(((int64_t)a.D + 255) / 256), (unsigned)((blocks + (1 << split) - 1) >> split), (unsigned)a.B << split), split};
}

int check_conv(const seg_causal_conv_args* a, const char* name) {
  SEG_CHECK_ARG(a != nullptr, "%s: args is NULL", name);
  SEG_CHECK_ARG(a->dtype >= SEG_DT_F16 && a->dtype <= SEG_DT_F32, "%s: dtype %d", name, a->dtype);
  SEG_CHECK_ARG(a->B >= 0 && a->L >= 0 && a->D > 0 && a->D <= (1 << 30), "%s: B %d, L %d, D %d (2^30 at most)", name, a->B, a->L, a->D);
  SEG_CHECK_ARG(a->K >= 1 && a->K <= MAXK, "%s: K = %d (1 .. %d)", name, a->K, MAXK);
  SEG_CHECK_ARG(a->act == SEG_ACT_NONE || a->act == SEG_ACT_SILU, "%s: activation %d (none or silu)", name, a->act);
  SEG_CHECK_ARG(a->B <= 65535, "%s: %d sequences in one call (65535 at most)", name, a->B);
  SEG_CHECK_ARG(a->L <= (1 << 30), "%s: %d rows in one call (2^30 at most)", name, a->L);
  SEG_CHECK_ARG((int64_t)a->B << conv_grid(*a, RUN_SMALL).split <= 65535, "%s: %d sequences of %d rows in one call (65535 for each 2^22 rows begun)", name, a->B, a->L);
  SEG_CHECK_ARG(a->w != nullptr, "%s: w is NULL", name);
  return SEG_OK;
}

}  // namespace

extern "C" int seg_causal_conv_fwd(const seg_causal_conv_args* a, seg_stream_t stream) {
  if (int rc = check_conv(a, "causal_conv_fwd")) return rc;
  SEG_CHECK_ARG(a->B == 0 || a->L == 0 || (a->x != nullptr && a->y != nullptr), "causal_conv_fwd: x / y is NULL");
  SEG_CHECK_ARG(a->L <= 1 || (a->x_ld >= a->D && a->y_ld >= a->D), "causal_conv_fwd: row strides below the %d channels", a->D);
  SEG_CHECK_ARG(a->state_out == nullptr || a->state_out != a->state, "causal_conv_fwd: state_out may not be state");
  if (a->B == 0 || (a->L == 0 && a->state_out == nullptr)) return SEG_OK;
  conv_dispatch(*a, conv_vec(*a, false), [&](auto* tp, auto V, auto Kc) {
    typedef typename std::remove_pointer<decltype(tp)>::type T;
    // runs of 16 rows read the window's edges half as often as runs of 8; too few of them to fill the card are halved
    const ConvGrid g = conv_grid(*a, RUN), small = conv_grid(*a, RUN_SMALL);
    if (g.blocks.x * g.parts() >= 1024) hipLaunchKernelGGL((conv_fwd_kernel<T, V(), Kc(), RUN>), g.blocks, dim3(256), 0, (hipStream_t)stream, *a, g.split);
    else hipLaunchKernelGGL((conv_fwd_kernel<T, V(), Kc(), RUN_SMALL>), small.blocks, dim3(256), 0, (hipStream_t)stream, *a, small.split);
  });
  SEG_CHECK_LAUNCH("causal_conv_fwd");
  return SEG_OK;
}

extern "C" int64_t seg_causal_conv_bwd_workspace_bytes(const seg_causal_conv_args* a) {
  if (a == nullptr || a->B <= 0 || a->L < 0 || a->D <= 0 || a->K < 1) return 0;
  return conv_grid(*a, RUN_SMALL).parts() * (a->K + 1) * a->D * 4;
}

extern "C" int seg_causal_conv_bwd(const seg_causal_conv_args* a, seg_stream_t stream) {
  if (int rc = check_conv(a, "causal_conv_bwd")) return rc;
  SEG_CHECK_ARG(a->B == 0 || a->L == 0 || (a->x != nullptr && a->dy != nullptr), "causal_conv_bwd: x / dy is NULL");
  SEG_CHECK_ARG(a->L <= 1 || (a->x_ld >= a->D && a->dy_ld >= a->D && (a->dx == nullptr || a->dx_ld >= a->D)), "causal_conv_bwd: row strides below the %d channels", a->D);
  const bool params = a->dw != nullptr || a->db != nullptr;
  SEG_CHECK_ARG(a->B == 0 || !params || a->workspace != nullptr, "causal_conv_bwd: dw / db need the workspace");
  SEG_CHECK_ARG(a->dx == nullptr || (a->dx != a->dy && a->dx != a->x), "causal_conv_bwd: dx may not be dy or x");
  hipStream_t st = (hipStream_t)stream;
  float* part = params ? (float*)a->workspace : nullptr;
  const ConvGrid g = conv_grid(*a, RUN_SMALL);
  if (a->B > 0)
    conv_dispatch(*a, conv_vec(*a, true), [&](auto* tp, auto V, auto Kc) {
      typedef typename std::remove_pointer<decltype(tp)>::type T;
      hipLaunchKernelGGL((conv_bwd_kernel<T, V(), Kc()>), g.blocks, dim3(256), 0, st, *a, g.split, part);
    });
  const int64_t parts = a->B > 0 ? g.parts() : 0, ld = (int64_t)(a->K + 1) * a->D;
  launch_colsum_pair(part, parts, ld, (int64_t)a->K * a->D, a->dw, a->D, a->db, st);
  SEG_CHECK_LAUNCH("causal_conv_bwd");
  return SEG_OK;
}

extern "C" int seg_causal_conv_step(const seg_causal_conv_args* a, seg_stream_t stream) {
  if (int rc = check_conv(a, "causal_conv_step")) return rc;
  if (a->B == 0) return SEG_OK;
  SEG_CHECK_ARG(a->x != nullptr && a->y != nullptr, "causal_conv_step: x / y is NULL");
  SEG_CHECK_ARG(a->B == 1 || (a->x_bs >= a->D && a->y_bs >= a->D), "causal_conv_step: row strides below the %d channels", a->D);
  const int64_t n = (int64_t)a->B * (((int64_t)a->D + 7) / 8);
  SEG_CHECK_ARG(grid_takes(n + 255), "causal_conv_step: %d sequences of %d channels are too many for one call (2^35 elements)", a->B, a->D);
  conv_dispatch(*a, conv_vec(*a, false), [&](auto* tp, auto V, auto Kc) {
    typedef typename std::remove_pointer<decltype(tp)>::type T;
    hipLaunchKernelGGL((conv_step_kernel<T, V(), Kc()>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, *a);
  });
  SEG_CHECK_LAUNCH("causal_conv_step");
  return SEG_OK;
}
