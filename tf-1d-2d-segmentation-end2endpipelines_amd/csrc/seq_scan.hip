// Selective state space scan: prompts, training, single rows (seg_selective_scan_fwd / _bwd / _step).
//
//   h[t] = a[t] h[t-1] + delta[t] B[t] u[t],  a[t] = exp(delta[t] A),  y[t] = (C[t] . h[t] + D u[t]) silu(z[t])
//
// The vector ALUs bound it: one exponential (a quarter-rate instruction) and four operations per state and row, against 8 bytes of
// rows per S states.  Layout: G = S / 4 lanes (rounded up to a power of two) share a channel, four states each in registers; a block
// walks its channels' rows in tiles of TT rows that all threads stage into LDS first - softplus, gate and products of rows computed
// once per element there, 8 channels per access - so that the recurrence itself reads LDS only.
//
// Few channels leave the card empty, so the rows can be cut into chunks that run side by side: one launch computes every chunk's last
// state from a zero start and the chunk's sum of delta (its decay is exp(A sum delta): no product of the a is kept), a small launch
// walks the chunks in order, and the main launch starts each chunk from its true state.
//
// Backward: with dp = dy silu(z) the adjoint g[t] = C[t] dp[t] + a[t+1] g[t+1] runs from the end, over the same chunks in the same way
// (a chunk's own part of the adjoint in front of it is sum_t (prod_{k<=t} a[k]) C[t] dp[t], which a walk FORWARD in t adds up).  The
// states are not kept: the forward call saves h in front of every tile, each tile is recomputed from there into registers.
#include "seq_common.h"

namespace {

constexpr int TT = 32;            // rows per tile = distance of the saved states
constexpr int SUB = 16;           // rows whose a and h the backward pass holds in registers
constexpr int MAXS = 64;
constexpr float LOG2E = 1.4426950408889634f;

template <int G> struct Lay {
  static constexpr int CB = G <= 4 ? 64 : 256 / G;             // channels per block
  static constexpr int NT = CB * G;                            // threads
  static constexpr int NW = NT / 64;
  static constexpr int SP = 4 * G;                             // states, padded
  static constexpr int CHUNKS = CB / 8;                        // 8-channel pieces of a row
  static constexpr int TASKS = TT * CHUNKS;
};

__device__ __forceinline__ float exp2_f(float v) { return __builtin_amdgcn_exp2f(v); }
// max(v, 0) + log(1 + e), e = exp(-|v|), with a small RELATIVE error: 1 + e loses low bits of e, which the logarithm gets back to first
// order (log(1 + e) = log(w) + (e - (w - 1)) / w, w the rounded sum); where e is small the series is used
__device__ __forceinline__ float softplus_f(float v) {
  const float e = __expf(-fabsf(v)), w = 1.f + e;
  const float l = e < 0.03125f ? e * (1.f - e * (0.5f - e * (0.33333333f - e * (0.25f - e * 0.2f)))) : __logf(w) + (e - (w - 1.f)) * __frcp_rn(w);
  return fmaxf(v, 0.f) + l;
}
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140, DPP_ROR4 = 0x124, DPP_ROR8 = 0x128;
// sum over the G neighbouring lanes of a channel
template <int G> __device__ __forceinline__ float group_sum(float v) {
  if constexpr (G >= 2) v += dpp<DPP_XOR1>(v);
  if constexpr (G >= 4) v += dpp<DPP_XOR2>(v);
  if constexpr (G >= 8) v += dpp<DPP_HALF_MIRROR>(v);
  if constexpr (G >= 16) v += dpp<DPP_MIRROR>(v);
  return v;
}

__device__ __forceinline__ int scan_len(const seg_scan_args& p, int b) {
  if (p.lengths == nullptr) return p.L;
  const int n = p.lengths[b];
  return n < 0 ? 0 : n > p.L ? p.L : n;
}
// four states of a channel: [.., S] rows of fp32, states at or behind S read as zero and are not written
__device__ __forceinline__ f4 load_states(const float* row, int s0, int S) {
  f4 h = {0.f, 0.f, 0.f, 0.f};
  if ((S & 3) == 0) {
    if (s0 < S) h = *reinterpret_cast<const f4*>(row + s0);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (s0 + i < S) h[i] = row[s0 + i];
  }
  return h;
}
__device__ __forceinline__ void store_states(float* row, int s0, int S, f4 h) {
  if ((S & 3) == 0) {
    if (s0 < S) *reinterpret_cast<f4*>(row + s0) = h;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (s0 + i < S) row[s0 + i] = h[i];
  }
}
// rows t0 .. t0 + TT of Bm / Cm as fp32 [TT][SP]; zero behind the length and behind S
template <typename T, int G>
__device__ __forceinline__ void stage_states(const T* m, int64_t bs, int64_t ld, int b, int t0, int len, int S, float* dst) {
  for (int e = threadIdx.x; e < TT * Lay<G>::SP; e += Lay<G>::NT) {
    const int t = t0 + e / Lay<G>::SP, s = e % Lay<G>::SP;
    dst[e] = (t < len && s < S) ? (float)m[b * bs + t * ld + s] : 0.f;
  }
}
template <bool VEC> __device__ __forceinline__ void load_chan(const float* p, int c, int n, float* f) {
  row_load8<float, VEC>(p + c, p != nullptr ? n : 0, f);
}
template <typename T, bool VEC>
__device__ __forceinline__ void stage_delta(const seg_scan_args& p, int b, int t, int len, int c, int n, const float* bias, float* delta) {
  row_load8<T, VEC>((const T*)p.dt + b * p.dt_bs + t * p.dt_ld + c, t < len ? n : 0, delta);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = delta[j] + bias[j];
    delta[j] = t < len ? (p.softplus ? softplus_f(v) : v) : 0.f;
  }
}

// MAIN: y, saved states and the last state from the chunk's true start; else the chunk's last state from zero and its sum of delta
template <typename T, bool VEC, int G, bool MAIN>
__global__ __launch_bounds__(Lay<G>::NT) void scan_fwd_kernel(const seg_scan_args p, int clen, float* start, float* sumd) {
  typedef Lay<G> Y;
  __shared__ float2 sdu[TT][Y::CB];
  __shared__ __align__(16) float sB[TT * Y::SP], sC[MAIN ? TT * Y::SP : 1];
  __shared__ __align__(16) float sy[MAIN ? TT : 1][Y::CB];
  const int tid = threadIdx.x, g = tid % G, c = tid / G, b = blockIdx.z, chunk = blockIdx.y, nch = gridDim.y;
  const int c0 = blockIdx.x * Y::CB, d = c0 + c, len = scan_len(p, b);
  const bool live = d < p.D;
  const int tbeg = chunk * clen, tend = tbeg + clen < p.L ? tbeg + clen : p.L;
  const int q0c = (tid % Y::CHUNKS) * 8, tc = c0 + q0c, tn = tc < p.D ? p.D - tc : 0;      // this thread's channels when staging rows
  float bias[8], skip[8];
  load_chan<VEC>(p.dt_bias, tc, tn, bias);
  if constexpr (MAIN) load_chan<VEC>(p.Dskip, tc, tn, skip);
  f4 A2 = {0.f, 0.f, 0.f, 0.f}, h = A2;
  if (live) {
    A2 = load_states(p.A + (int64_t)d * p.S, 4 * g, p.S) * LOG2E;
    if constexpr (MAIN) {
      if (start != nullptr) h = load_states(start + (((int64_t)b * nch + chunk) * p.D + d) * p.S, 4 * g, p.S);
      else if (p.state != nullptr) h = load_states(p.state + ((int64_t)b * p.D + d) * p.S, 4 * g, p.S);
    }
  }
  float dsum = 0.f;
  const int64_t nck = (p.L + TT - 1) / TT;
  for (int t0 = tbeg; t0 < tend; t0 += TT) {
    if constexpr (MAIN) {
      if (p.saved != nullptr && live) store_states(p.saved + (((int64_t)b * nck + t0 / TT) * p.D + d) * p.S, 4 * g, p.S, h);
    }
    for (int q = tid; q < Y::TASKS; q += Y::NT) {
      const int r = q / Y::CHUNKS, t = t0 + r;
      float delta[8], u[8];
      stage_delta<T, VEC>(p, b, t, len, tc, tn, bias, delta);
      row_load8<T, VEC>((const T*)p.u + b * p.u_bs + t * p.u_ld + tc, t < len ? tn : 0, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) sdu[r][q0c + j] = float2{delta[j], delta[j] * u[j]};
    }
    stage_states<T, G>((const T*)p.Bm, p.Bm_bs, p.Bm_ld, b, t0, len, p.S, sB);
    if constexpr (MAIN) stage_states<T, G>((const T*)p.Cm, p.Cm_bs, p.Cm_ld, b, t0, len, p.S, sC);
    __syncthreads();
#pragma unroll 4
    for (int r = 0; r < TT; ++r) {
      const float2 dd = sdu[r][c];
      const f4 B4 = *reinterpret_cast<const f4*>(sB + r * Y::SP + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = fmaf(exp2_f(dd.x * A2[i]), h[i], dd.y * B4[i]);
      if constexpr (MAIN) {
        const f4 C4 = *reinterpret_cast<const f4*>(sC + r * Y::SP + 4 * g);
        const float y = group_sum<G>(fmaf(C4[3], h[3], fmaf(C4[2], h[2], fmaf(C4[1], h[1], C4[0] * h[0]))));
        if (g == 0) sy[r][c] = y;
      } else {
        dsum += dd.x;
      }
    }
    __syncthreads();
    if constexpr (MAIN) {
      for (int q = tid; q < Y::TASKS; q += Y::NT) {
        const int r = q / Y::CHUNKS, t = t0 + r;
        if (t < tend && tn > 0) {
          float u[8], z[8], y[8];
          row_load8<T, VEC>((const T*)p.u + b * p.u_bs + t * p.u_ld + tc, t < len ? tn : 0, u);
          if (p.z != nullptr) row_load8<T, VEC>((const T*)p.z + b * p.z_bs + t * p.z_ld + tc, t < len ? tn : 0, z);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            y[j] = fmaf(skip[j], u[j], sy[r][q0c + j]);
            if (p.z != nullptr) y[j] *= z[j] * sigmoid_f(z[j]);
            if (t >= len) y[j] = 0.f;
          }
          row_store8<T, VEC>((T*)p.y + b * p.y_bs + t * p.y_ld + tc, tn, y);
        }
      }
      // (the next tile's staging writes sdu / sB / sC, whose readers are past the barrier above; sy is written behind its own next barrier)
    }
  }
  if (!live) return;
  if constexpr (MAIN) {
    if (p.state_out != nullptr && chunk == nch - 1) store_states(p.state_out + ((int64_t)b * p.D + d) * p.S, 4 * g, p.S, h);
  } else {
    const int64_t o = ((int64_t)b * nch + chunk) * p.D + d;
    store_states(start + o * p.S, 4 * g, p.S, h);
    if (g == 0) sumd[o] = dsum;
  }
}

// the chunks in order: in place, a chunk's own last state becomes the state in front of it
__global__ __launch_bounds__(256) void scan_join_kernel(const seg_scan_args p, int nch, float* start, const float* sumd) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)p.D * p.S;
  const int b = blockIdx.y;
  if (e >= n) return;
  const int64_t d = e / p.S;
  const float A2 = p.A[e] * LOG2E;
  float h = p.state != nullptr ? p.state[b * n + e] : 0.f;
  for (int k = 0; k < nch; ++k) {
    const int64_t o = (int64_t)b * nch + k;
    const float own = start[o * n + e];
    start[o * n + e] = h;
    h = fmaf(exp2_f(A2 * sumd[o * p.D + d]), h, own);
  }
}
// the same for the adjoint, from the last chunk: a chunk's own part becomes the adjoint that enters it from behind
__global__ __launch_bounds__(256) void scan_join_bwd_kernel(const seg_scan_args p, int nch, float* adj, const float* sumd) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)p.D * p.S;
  const int b = blockIdx.y;
  if (e >= n) return;
  const int64_t d = e / p.S;
  const float A2 = p.A[e] * LOG2E;
  float q = p.dstate_out != nullptr ? p.dstate_out[b * n + e] : 0.f;
  for (int k = nch - 1; k >= 0; --k) {
    const int64_t o = (int64_t)b * nch + k;
    const float own = adj[o * n + e];
    adj[o * n + e] = q;
    q = fmaf(exp2_f(A2 * sumd[o * p.D + d]), q, own);
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void stage_dp(const seg_scan_args& p, int b, int t, int len, int c, int n, float* dp, float* z) {
  row_load8<T, VEC>((const T*)p.dy + b * p.dy_bs + t * p.dy_ld + c, t < len ? n : 0, dp);
  if (p.z != nullptr) {
    row_load8<T, VEC>((const T*)p.z + b * p.z_bs + t * p.z_ld + c, t < len ? n : 0, z);
#pragma unroll
    for (int j = 0; j < 8; ++j) dp[j] *= z[j] * sigmoid_f(z[j]);
  }
}

// a chunk's own part of the adjoint in front of it, and its sum of delta
template <typename T, bool VEC, int G>
__global__ __launch_bounds__(Lay<G>::NT) void scan_bwd_local_kernel(const seg_scan_args p, int clen, float* adj, float* sumd) {
  typedef Lay<G> Y;
  __shared__ float2 sdp[TT][Y::CB];
  __shared__ __align__(16) float sC[TT * Y::SP];
  const int tid = threadIdx.x, g = tid % G, c = tid / G, b = blockIdx.z, chunk = blockIdx.y, nch = gridDim.y;
  const int c0 = blockIdx.x * Y::CB, d = c0 + c, len = scan_len(p, b);
  const bool live = d < p.D;
  const int tbeg = chunk * clen, tend = tbeg + clen < p.L ? tbeg + clen : p.L;
  const int q0c = (tid % Y::CHUNKS) * 8, tc = c0 + q0c, tn = tc < p.D ? p.D - tc : 0;
  float bias[8];
  load_chan<VEC>(p.dt_bias, tc, tn, bias);
  f4 A2 = {0.f, 0.f, 0.f, 0.f}, P = {1.f, 1.f, 1.f, 1.f}, q = A2;
  if (live) A2 = load_states(p.A + (int64_t)d * p.S, 4 * g, p.S) * LOG2E;
  float dsum = 0.f;
  for (int t0 = tbeg; t0 < tend; t0 += TT) {
    for (int k = tid; k < Y::TASKS; k += Y::NT) {
      const int r = k / Y::CHUNKS, t = t0 + r;
      float delta[8], dp[8], z[8];
      stage_delta<T, VEC>(p, b, t, len, tc, tn, bias, delta);
      stage_dp<T, VEC>(p, b, t, len, tc, tn, dp, z);
#pragma unroll
      for (int j = 0; j < 8; ++j) sdp[r][q0c + j] = float2{delta[j], dp[j]};
    }
    stage_states<T, G>((const T*)p.Cm, p.Cm_bs, p.Cm_ld, b, t0, len, p.S, sC);
    __syncthreads();
#pragma unroll 4
    for (int r = 0; r < TT; ++r) {
      const float2 dd = sdp[r][c];
      const f4 C4 = *reinterpret_cast<const f4*>(sC + r * Y::SP + 4 * g);
      dsum += dd.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        P[i] *= exp2_f(dd.x * A2[i]);
        q[i] = fmaf(P[i], C4[i] * dd.y, q[i]);
      }
    }
    __syncthreads();
  }
  if (!live) return;
  const int64_t o = ((int64_t)b * nch + chunk) * p.D + d;
  store_states(adj + o * p.S, 4 * g, p.S, q);
  if (g == 0) sumd[o] = dsum;
}

// sum the eight values v over the lanes of a wave that share lane % G; lanes with bit 5 clear end with v[0..3], the others with
// v[4..7]; of these bit 4 chooses the first or the last two: w[0..1]
template <int G> __device__ __forceinline__ void lane_sums(const float* v, float* w) {
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v[i]), __builtin_bit_cast(unsigned, v[4 + i]), false, false);
    x[i] = __builtin_bit_cast(float, (unsigned)s[0]) + __builtin_bit_cast(float, (unsigned)s[1]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto s = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x[i]), __builtin_bit_cast(unsigned, x[2 + i]), false, false);
    w[i] = __builtin_bit_cast(float, (unsigned)s[0]) + __builtin_bit_cast(float, (unsigned)s[1]);
    if constexpr (G <= 8) w[i] += dpp<DPP_ROR8>(w[i]);
    if constexpr (G <= 4) w[i] += dpp<DPP_ROR4>(w[i]);
    if constexpr (G <= 2) w[i] += dpp<DPP_XOR2>(w[i]);
    if constexpr (G <= 1) w[i] += dpp<DPP_XOR1>(w[i]);
  }
}

// the gradients of a chunk.  adj: the adjoint that enters each chunk from behind (NULL: one chunk, dstate_out).  Partial sums:
// pbc[channel block][B][L][2][S] (dB, dC), pA[B nch][D][S], pD[B nch][2][D] (dD, ddt_bias)
template <typename T, bool VEC, int G>
__global__ __launch_bounds__(Lay<G>::NT) void scan_bwd_kernel(const seg_scan_args p, int clen, const float* adj, float* pbc, float* pA, float* pD) {
  typedef Lay<G> Y;
  __shared__ f4 sx[TT][Y::CB];                               // delta, u -> sum g B, dp -> sum g a h A, -> C . h
  __shared__ __align__(16) float sB[TT * Y::SP], sC[TT * Y::SP];
  __shared__ __align__(16) float sbc[Y::NW][SUB][2][Y::SP];
  const int tid = threadIdx.x, g = tid % G, c = tid / G, b = blockIdx.z, chunk = blockIdx.y, nch = gridDim.y;
  const int lane = tid & 63, wave = tid >> 6;
  const int c0 = blockIdx.x * Y::CB, d = c0 + c, len = scan_len(p, b);
  const bool live = d < p.D;
  const int tbeg = chunk * clen, tend = tbeg + clen < p.L ? tbeg + clen : p.L;
  const int q0c = (tid % Y::CHUNKS) * 8, tc = c0 + q0c, tn = tc < p.D ? p.D - tc : 0;
  float bias[8], skip[8], accD[8], accB[8];
  load_chan<VEC>(p.dt_bias, tc, tn, bias);
  load_chan<VEC>(p.Dskip, tc, tn, skip);
#pragma unroll
  for (int j = 0; j < 8; ++j) accD[j] = accB[j] = 0.f;
  f4 A = {0.f, 0.f, 0.f, 0.f}, A2 = A, q = A, dA = A;
  if (live) {
    A = load_states(p.A + (int64_t)d * p.S, 4 * g, p.S);
    A2 = A * LOG2E;
    if (adj != nullptr) q = load_states(adj + (((int64_t)b * nch + chunk) * p.D + d) * p.S, 4 * g, p.S);
    else if (p.dstate_out != nullptr) q = load_states(p.dstate_out + ((int64_t)b * p.D + d) * p.S, 4 * g, p.S);
  }
  const int64_t nck = (p.L + TT - 1) / TT;
  const int ntile = tend > tbeg ? (tend - tbeg + TT - 1) / TT : 0;
  for (int tile = ntile - 1; tile >= 0; --tile) {
    const int t0 = tbeg + tile * TT;
    f4 hs = {0.f, 0.f, 0.f, 0.f};
    if (live) hs = load_states(p.saved + (((int64_t)b * nck + t0 / TT) * p.D + d) * p.S, 4 * g, p.S);
    for (int k = tid; k < Y::TASKS; k += Y::NT) {
      const int r = k / Y::CHUNKS, t = t0 + r;
      float delta[8], u[8], dp[8], z[8];
      stage_delta<T, VEC>(p, b, t, len, tc, tn, bias, delta);
      row_load8<T, VEC>((const T*)p.u + b * p.u_bs + t * p.u_ld + tc, t < len ? tn : 0, u);
      stage_dp<T, VEC>(p, b, t, len, tc, tn, dp, z);
#pragma unroll
      for (int j = 0; j < 8; ++j) sx[r][q0c + j] = f4{delta[j], u[j], dp[j], 0.f};
    }
    stage_states<T, G>((const T*)p.Bm, p.Bm_bs, p.Bm_ld, b, t0, len, p.S, sB);
    stage_states<T, G>((const T*)p.Cm, p.Cm_bs, p.Cm_ld, b, t0, len, p.S, sC);
    __syncthreads();
    f4 hmid = hs;                                            // the state in front of the tile's second half
#pragma unroll 4
    for (int r = 0; r < SUB; ++r) {
      const f4 x = sx[r][c];
      const f4 B4 = *reinterpret_cast<const f4*>(sB + r * Y::SP + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) hmid[i] = fmaf(exp2_f(x[0] * A2[i]), hmid[i], x[0] * x[1] * B4[i]);
    }
#pragma unroll 1
    for (int half = TT / SUB - 1; half >= 0; --half) {
      f4 a[SUB], hp[SUB], h = half ? hmid : hs;
#pragma unroll
      for (int k = 0; k < SUB; ++k) {
        const int r = half * SUB + k;
        const f4 x = sx[r][c];
        const f4 B4 = *reinterpret_cast<const f4*>(sB + r * Y::SP + 4 * g), C4 = *reinterpret_cast<const f4*>(sC + r * Y::SP + 4 * g);
        const float du = x[0] * x[1];
        hp[k] = h;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[k][i] = exp2_f(x[0] * A2[i]);
          h[i] = fmaf(a[k][i], h[i], du * B4[i]);
        }
        const float y = group_sum<G>(fmaf(C4[3], h[3], fmaf(C4[2], h[2], fmaf(C4[1], h[1], C4[0] * h[0]))));
        if (g == 0) sx[r][c][3] = y;
      }
#pragma unroll
      for (int k = SUB - 1; k >= 0; --k) {
        const int r = half * SUB + k;
        const f4 x = sx[r][c];
        const f4 B4 = *reinterpret_cast<const f4*>(sB + r * Y::SP + 4 * g), C4 = *reinterpret_cast<const f4*>(sC + r * Y::SP + 4 * g);
        const float du = x[0] * x[1];
        float v[8], w[2], sgB = 0.f, sA = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float gi = fmaf(C4[i], x[2], q[i]);
          const float ga = gi * a[k][i], gh = ga * hp[k][i];
          sgB = fmaf(gi, B4[i], sgB);
          sA = fmaf(gh, A[i], sA);
          dA[i] = fmaf(gh, x[0], dA[i]);
          v[i] = gi * du;
          v[4 + i] = x[2] * h[i];
          q[i] = ga;
        }
        h = hp[k];
        sgB = group_sum<G>(sgB);
        sA = group_sum<G>(sA);
        if (g == 0) { sx[r][c][1] = sgB; sx[r][c][2] = sA; }
        lane_sums<G>(v, w);
        if ((lane & 15) < G) {
          float* o = &sbc[wave][k][lane >> 5][4 * g + 2 * ((lane >> 4) & 1)];
          o[0] = w[0];
          o[1] = w[1];
        }
      }
      __syncthreads();
      if (pbc != nullptr) {
        for (int e = tid; e < SUB * 2 * Y::SP; e += Y::NT) {
          const int k = e / (2 * Y::SP), wh = (e / Y::SP) & 1, s = e % Y::SP, t = t0 + half * SUB + k;
          if (t < tend && s < p.S) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < Y::NW; ++w) v += sbc[w][k][wh][s];
            pbc[((((int64_t)blockIdx.x * p.B + b) * p.L + t) * 2 + wh) * p.S + s] = v;
          }
        }
      }
      __syncthreads();
    }
    for (int k = tid; k < Y::TASKS; k += Y::NT) {
      const int r = k / Y::CHUNKS, t = t0 + r;
      if (t < tend && tn > 0) {
        float u[8], dp[8], z[8], dtv[8], dout[8], o[8];
        const int n = t < len ? tn : 0;
        row_load8<T, VEC>((const T*)p.u + b * p.u_bs + t * p.u_ld + tc, n, u);
        row_load8<T, VEC>((const T*)p.dt + b * p.dt_bs + t * p.dt_ld + tc, n, dtv);
        row_load8<T, VEC>((const T*)p.dy + b * p.dy_bs + t * p.dy_ld + tc, n, dout);
        stage_dp<T, VEC>(p, b, t, len, tc, tn, dp, z);
        f4 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = sx[r][q0c + j];
        if (p.du != nullptr) {
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = t < len ? fmaf(skip[j], dp[j], x[j][0] * x[j][1]) : 0.f;
          row_store8<T, VEC>((T*)p.du + b * p.du_bs + t * p.du_ld + tc, tn, o);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[j] = fmaf(x[j][1], u[j], x[j][2]);
          if (p.softplus) o[j] *= sigmoid_f(dtv[j] + bias[j]);
          if (t >= len) o[j] = 0.f;
          accB[j] += o[j];
          accD[j] = fmaf(dp[j], u[j], accD[j]);
        }
        if (p.ddt != nullptr) row_store8<T, VEC>((T*)p.ddt + b * p.ddt_bs + t * p.ddt_ld + tc, tn, o);
        if (p.dz != nullptr) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float s = sigmoid_f(z[j]);
            o[j] = t < len ? dout[j] * fmaf(skip[j], u[j], x[j][3]) * s * (1.f + z[j] * (1.f - s)) : 0.f;
          }
          row_store8<T, VEC>((T*)p.dz + b * p.dz_bs + t * p.dz_ld + tc, tn, o);
        }
      }
    }
    __syncthreads();
  }
  const int64_t o = (int64_t)b * nch + chunk;
  if (live && pA != nullptr) store_states(pA + (o * p.D + d) * p.S, 4 * g, p.S, dA);
  if (live && p.dstate != nullptr && chunk == 0) store_states(p.dstate + ((int64_t)b * p.D + d) * p.S, 4 * g, p.S, q);
  if (pD != nullptr) {
    // the threads of a channel piece: NT / CHUNKS rows of CB values, added by the block's first CB threads, dD and then ddt_bias
    float* sh = reinterpret_cast<float*>(&sx[0][0]);
    constexpr int R = Y::NT / Y::CHUNKS;
    static_assert(R * Y::CB * 4 <= (int)sizeof(sx), "the rows fit the tile's LDS");
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sh[(tid / Y::CHUNKS) * Y::CB + q0c + j] = k == 0 ? accD[j] : accB[j];
      __syncthreads();
      if (tid < Y::CB && c0 + tid < p.D) {
        float v = 0.f;
        for (int r = 0; r < R; ++r) v += sh[r * Y::CB + tid];
        pD[(o * 2 + k) * p.D + c0 + tid] = v;
      }
      __syncthreads();
    }
  }
}

// dB / dC: the channel blocks' parts in order
template <typename T>
__global__ __launch_bounds__(256) void scan_bc_kernel(const seg_scan_args p, int nblk, const float* pbc) {
  const int64_t n = (int64_t)p.B * p.L * 2 * p.S;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int k = 0; k < nblk; ++k) v += pbc[k * n + e];
    const int s = (int)(e % p.S), wh = (int)(e / p.S) & 1;
    const int64_t bt = e / (2 * p.S), b = bt / p.L, t = bt - b * p.L;
    if (wh == 0) { if (p.dBm != nullptr) ((T*)p.dBm)[b * p.dBm_bs + t * p.dBm_ld + s] = (T)v; }
    else if (p.dCm != nullptr) ((T*)p.dCm)[b * p.dCm_bs + t * p.dCm_ld + s] = (T)v;
  }
}

template <typename T, int G>
__global__ __launch_bounds__(256) void scan_step_kernel(const seg_scan_args p) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, bd = e / G;
  const int g = (int)(e % G);
  const bool live = bd < (int64_t)p.B * p.D;                   // (whole groups of lanes; the sum below needs all of a group)
  const int b = live ? (int)(bd / p.D) : 0, d = live ? (int)(bd - (int64_t)b * p.D) : 0;
  float y = 0.f, u = 0.f;
  if (live) {
    u = (float)((const T*)p.u)[b * p.u_bs + d];
    float delta = (float)((const T*)p.dt)[b * p.dt_bs + d] + (p.dt_bias != nullptr ? p.dt_bias[d] : 0.f);
    if (p.softplus) delta = softplus_f(delta);
    const int64_t so = ((int64_t)b * p.D + d) * p.S;
    f4 h = {0.f, 0.f, 0.f, 0.f};
    if (p.state != nullptr) h = load_states(p.state + so, 4 * g, p.S);
    const f4 A2 = load_states(p.A + (int64_t)d * p.S, 4 * g, p.S) * LOG2E;
    const T *Bm = (const T*)p.Bm + b * p.Bm_bs, *Cm = (const T*)p.Cm + b * p.Cm_bs;
    const float du = delta * u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = 4 * g + i;
      if (s < p.S) {
        h[i] = fmaf(exp2_f(delta * A2[i]), h[i], du * (float)Bm[s]);
        y = fmaf((float)Cm[s], h[i], y);
      }
    }
    if (p.state_out != nullptr) store_states(p.state_out + so, 4 * g, p.S, h);
  }
  y = group_sum<G>(y);
  if (live && g == 0) {
    if (p.Dskip != nullptr) y = fmaf(p.Dskip[d], u, y);
    if (p.z != nullptr) {
      const float z = (float)((const T*)p.z)[b * p.z_bs + d];
      y *= z * sigmoid_f(z);
    }
    ((T*)p.y)[b * p.y_bs + d] = (T)y;
  }
}

inline int scan_group(int S) { return S <= 4 ? 1 : S <= 8 ? 2 : S <= 16 ? 4 : S <= 32 ? 8 : 16; }
inline int scan_cb(int S) { const int G = scan_group(S); return G <= 4 ? 64 : 256 / G; }

struct ScanPlan { int nblk, nch, clen; };
inline ScanPlan scan_plan(const seg_scan_args& a) {
  ScanPlan s;
  const int cb = scan_cb(a.S);
  s.nblk = (a.D + cb - 1) / cb;
  const int64_t blocks = (int64_t)s.nblk * a.B;
  int64_t nch = blocks >= 512 ? 1 : (1024 + blocks - 1) / (blocks < 1 ? 1 : blocks);
  const int64_t most = (a.L + 63) / 64;
  if (nch > most) nch = most;
  if (nch < 1) nch = 1;
  int64_t clen = ((int64_t)a.L + nch - 1) / nch;
  clen = (clen + TT - 1) / TT * TT;
  if (clen < TT) clen = TT;
  s.clen = (int)clen;
  s.nch = (int)(((int64_t)a.L + clen - 1) / clen);
  if (s.nch < 1) s.nch = 1;
  return s;
}
struct ScanBwdSpace { int64_t adj, sumd, pbc, pA, pD, total; };          // offsets in floats
inline ScanBwdSpace scan_bwd_space(const seg_scan_args& a, const ScanPlan& s) {
  ScanBwdSpace w;
  const int64_t bn = (int64_t)a.B * s.nch, st = (int64_t)a.D * a.S;
  auto up = [](int64_t v) { return (v + 3) / 4 * 4; };
  int64_t o = 0;
  w.adj = o; o += s.nch > 1 ? up(bn * st) : 0;
  w.sumd = o; o += s.nch > 1 ? up(bn * a.D) : 0;
  w.pbc = o; o += up((int64_t)s.nblk * a.B * a.L * 2 * a.S);
  w.pA = o; o += up(bn * st);
  w.pD = o; o += up(bn * 2 * a.D);
  w.total = o;
  return w;
}

template <typename F>
inline void scan_dispatch(const seg_scan_args& a, F&& f) {
  seq_dispatch_dtype(a.dtype, [&](auto* tp) {
    typedef typename std::remove_pointer<decltype(tp)>::type T;
    switch (scan_group(a.S)) {
      case 1: f((T*)nullptr, std::integral_constant<int, 1>{}); break;
      case 2: f((T*)nullptr, std::integral_constant<int, 2>{}); break;
      case 4: f((T*)nullptr, std::integral_constant<int, 4>{}); break;
      case 8: f((T*)nullptr, std::integral_constant<int, 8>{}); break;
      default: f((T*)nullptr, std::integral_constant<int, 16>{}); break;
    }
  });
}
inline bool scan_vec(const seg_scan_args& a, bool bwd) {
  if (a.D % 8 != 0 || !aligned16(a.dt_bias) || !aligned16(a.Dskip)) return false;
  const bool ok = vec_ok(a.u, a.u_ld, a.u_bs, a.dtype) && vec_ok(a.dt, a.dt_ld, a.dt_bs, a.dtype) && vec_ok(a.z, a.z_ld, a.z_bs, a.dtype);
  if (!bwd) return ok && vec_ok(a.y, a.y_ld, a.y_bs, a.dtype);
  return ok && vec_ok(a.dy, a.dy_ld, a.dy_bs, a.dtype) && vec_ok(a.du, a.du_ld, a.du_bs, a.dtype) && vec_ok(a.ddt, a.ddt_ld, a.ddt_bs, a.dtype) &&
         vec_ok(a.dz, a.dz_ld, a.dz_bs, a.dtype);
}

int check_scan(const seg_scan_args* a, const char* name) {
  SEG_CHECK_ARG(a != nullptr, "%s: args is NULL", name);
  SEG_CHECK_ARG(a->dtype >= SEG_DT_F16 && a->dtype <= SEG_DT_F32, "%s: dtype %d", name, a->dtype);
  SEG_CHECK_ARG(a->B >= 0 && a->L >= 0 && a->D > 0, "%s: B %d, L %d, D %d", name, a->B, a->L, a->D);
  SEG_CHECK_ARG(a->S >= 1 && a->S <= MAXS, "%s: %d states (1 .. %d)", name, a->S, MAXS);
  SEG_CHECK_ARG(a->B <= 65535, "%s: %d sequences in one call (65535 at most)", name, a->B);
  SEG_CHECK_ARG(a->L <= (1 << 30), "%s: %d rows in one call (2^30 at most)", name, a->L);
  SEG_CHECK_ARG(a->A != nullptr, "%s: A is NULL", name);
  SEG_CHECK_ARG(((uintptr_t)a->A & 15) == 0 && ((uintptr_t)a->state & 15) == 0 && ((uintptr_t)a->state_out & 15) == 0 && ((uintptr_t)a->saved & 15) == 0 &&
                ((uintptr_t)a->dstate_out & 15) == 0 && ((uintptr_t)a->dstate & 15) == 0, "%s: A / state / saved need 16-byte alignment", name);
  SEG_CHECK_ARG(aligned16(a->workspace), "%s: workspace needs 16-byte alignment", name);
  return SEG_OK;
}
bool scan_rows_ok(const seg_scan_args& a) {
  return a.L <= 1 || (a.u_ld >= a.D && a.dt_ld >= a.D && (a.z == nullptr || a.z_ld >= a.D) && a.Bm_ld >= a.S && a.Cm_ld >= a.S);
}

}  // namespace

extern "C" int64_t seg_selective_scan_saved_bytes(const seg_scan_args* a) {
  if (a == nullptr || a->B <= 0 || a->L <= 0 || a->D <= 0 || a->S <= 0) return 0;
  return (int64_t)a->B * ((a->L + TT - 1) / TT) * a->D * a->S * 4;
}
extern "C" int64_t seg_selective_scan_fwd_workspace_bytes(const seg_scan_args* a) {
  if (a == nullptr || a->B <= 0 || a->L <= 0 || a->D <= 0 || a->S <= 0) return 0;
  const ScanPlan s = scan_plan(*a);
  if (s.nch <= 1) return 0;
  return ((int64_t)a->B * s.nch * a->D * a->S + 3) / 4 * 16 + (int64_t)a->B * s.nch * a->D * 4;
}
extern "C" int64_t seg_selective_scan_bwd_workspace_bytes(const seg_scan_args* a) {
  if (a == nullptr || a->B <= 0 || a->L <= 0 || a->D <= 0 || a->S <= 0) return 0;
  return scan_bwd_space(*a, scan_plan(*a)).total * 4;
}

extern "C" int seg_selective_scan_fwd(const seg_scan_args* a, seg_stream_t stream) {
  if (int rc = check_scan(a, "selective_scan_fwd")) return rc;
  SEG_CHECK_ARG(a->B == 0 || a->L == 0 || (a->u != nullptr && a->dt != nullptr && a->Bm != nullptr && a->Cm != nullptr && a->y != nullptr), "selective_scan_fwd: u / dt / Bm / Cm / y is NULL");
  SEG_CHECK_ARG(scan_rows_ok(*a) && (a->L <= 1 || a->y_ld >= a->D), "selective_scan_fwd: row strides below the channels / states");
  SEG_CHECK_ARG(a->state_out == nullptr || a->state_out != a->state, "selective_scan_fwd: state_out may not be state");
  if (a->B == 0 || (a->L == 0 && a->state_out == nullptr)) return SEG_OK;
  const ScanPlan s = scan_plan(*a);
  SEG_CHECK_ARG(s.nch <= 1 || a->workspace != nullptr, "selective_scan_fwd: workspace is NULL (%lld bytes are needed)", (long long)seg_selective_scan_fwd_workspace_bytes(a));
  hipStream_t st = (hipStream_t)stream;
  float* start = s.nch > 1 ? (float*)a->workspace : nullptr;
  float* sumd = s.nch > 1 ? start + ((int64_t)a->B * s.nch * a->D * a->S + 3) / 4 * 4 : nullptr;
  const dim3 grid((unsigned)s.nblk, (unsigned)s.nch, (unsigned)a->B);
  const bool vec = scan_vec(*a, false);
  scan_dispatch(*a, [&](auto* tp, auto Gc) {
    typedef typename std::remove_pointer<decltype(tp)>::type T;
    constexpr int G = Gc(), NT = Lay<G>::NT;
    if (s.nch > 1) {
      if (vec) hipLaunchKernelGGL((scan_fwd_kernel<T, true, G, false>), grid, dim3(NT), 0, st, *a, s.clen, start, sumd);
      else hipLaunchKernelGGL((scan_fwd_kernel<T, false, G, false>), grid, dim3(NT), 0, st, *a, s.clen, start, sumd);
      const int64_t n = (int64_t)a->D * a->S;
      hipLaunchKernelGGL(scan_join_kernel, dim3((unsigned)((n + 255) / 256), (unsigned)a->B), dim3(256), 0, st, *a, s.nch, start, sumd);
    }
    if (vec) hipLaunchKernelGGL((scan_fwd_kernel<T, true, G, true>), grid, dim3(NT), 0, st, *a, s.clen, start, sumd);
    else hipLaunchKernelGGL((scan_fwd_kernel<T, false, G, true>), grid, dim3(NT), 0, st, *a, s.clen, start, sumd);
  });
  SEG_CHECK_LAUNCH("selective_scan_fwd");
  return SEG_OK;
}

extern "C" int seg_selective_scan_bwd(const seg_scan_args* a, seg_stream_t stream) {
  if (int rc = check_scan(a, "selective_scan_bwd")) return rc;
  const bool none = a->B == 0 || a->L == 0;
  SEG_CHECK_ARG(none || (a->u != nullptr && a->dt != nullptr && a->Bm != nullptr && a->Cm != nullptr && a->dy != nullptr && a->saved != nullptr),
                "selective_scan_bwd: u / dt / Bm / Cm / dy / saved is NULL");
  SEG_CHECK_ARG(scan_rows_ok(*a) && (a->L <= 1 || (a->dy_ld >= a->D && (a->du == nullptr || a->du_ld >= a->D) && (a->ddt == nullptr || a->ddt_ld >= a->D) &&
                (a->dz == nullptr || a->dz_ld >= a->D) && (a->dBm == nullptr || a->dBm_ld >= a->S) && (a->dCm == nullptr || a->dCm_ld >= a->S))),
                "selective_scan_bwd: row strides below the channels / states");
  SEG_CHECK_ARG(a->dz == nullptr || a->z != nullptr, "selective_scan_bwd: dz without z");
  SEG_CHECK_ARG(none || a->workspace != nullptr, "selective_scan_bwd: workspace is NULL (%lld bytes are needed)", (long long)seg_selective_scan_bwd_workspace_bytes(a));
  hipStream_t st = (hipStream_t)stream;
  const ScanPlan s = scan_plan(*a);
  const ScanBwdSpace w = scan_bwd_space(*a, s);
  float* ws = (float*)a->workspace;
  const int64_t n = (int64_t)a->D * a->S;
  float *adj = s.nch > 1 && !none ? ws + w.adj : nullptr, *sumd = ws + w.sumd;
  const bool bc = a->dBm != nullptr || a->dCm != nullptr, pd = a->dD != nullptr || a->ddt_bias != nullptr;
  const dim3 grid((unsigned)s.nblk, (unsigned)s.nch, (unsigned)a->B);
  if (a->B > 0 && (!none || a->dstate != nullptr)) {
    const bool vec = scan_vec(*a, true);
    scan_dispatch(*a, [&](auto* tp, auto Gc) {
      typedef typename std::remove_pointer<decltype(tp)>::type T;
      constexpr int G = Gc(), NT = Lay<G>::NT;
      if (s.nch > 1) {
        if (vec) hipLaunchKernelGGL((scan_bwd_local_kernel<T, true, G>), grid, dim3(NT), 0, st, *a, s.clen, adj, sumd);
        else hipLaunchKernelGGL((scan_bwd_local_kernel<T, false, G>), grid, dim3(NT), 0, st, *a, s.clen, adj, sumd);
        hipLaunchKernelGGL(scan_join_bwd_kernel, dim3((unsigned)((n + 255) / 256), (unsigned)a->B), dim3(256), 0, st, *a, s.nch, adj, sumd);
      }
      float *pbc = bc && !none ? ws + w.pbc : nullptr, *pA = a->dA != nullptr && !none ? ws + w.pA : nullptr, *pD = pd && !none ? ws + w.pD : nullptr;
      if (vec) hipLaunchKernelGGL((scan_bwd_kernel<T, true, G>), grid, dim3(NT), 0, st, *a, s.clen, adj, pbc, pA, pD);
      else hipLaunchKernelGGL((scan_bwd_kernel<T, false, G>), grid, dim3(NT), 0, st, *a, s.clen, adj, pbc, pA, pD);
      if (pbc != nullptr) {
        const int64_t blocks = ((int64_t)a->B * a->L * 2 * a->S + 255) / 256;
        hipLaunchKernelGGL((scan_bc_kernel<T>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st, *a, s.nblk, pbc);
      }
    });
  }
  const int64_t parts = none ? 0 : (int64_t)a->B * s.nch;
  if (a->dA != nullptr) launch_colsum_parts(ws + (none ? 0 : w.pA), parts, n, n, a->dA, st);
  if (a->dD != nullptr) launch_colsum_parts(ws + (none ? 0 : w.pD), parts, 2 * (int64_t)a->D, a->D, a->dD, st);
  if (a->ddt_bias != nullptr) launch_colsum_parts(none ? ws : ws + w.pD + a->D, parts, 2 * (int64_t)a->D, a->D, a->ddt_bias, st);
  SEG_CHECK_LAUNCH("selective_scan_bwd");
  return SEG_OK;
}

extern "C" int seg_selective_scan_step(const seg_scan_args* a, seg_stream_t stream) {
  if (int rc = check_scan(a, "selective_scan_step")) return rc;
  if (a->B == 0) return SEG_OK;
  SEG_CHECK_ARG(a->u != nullptr && a->dt != nullptr && a->Bm != nullptr && a->Cm != nullptr && a->y != nullptr, "selective_scan_step: u / dt / Bm / Cm / y is NULL");
  SEG_CHECK_ARG(a->B == 1 || (a->u_bs >= a->D && a->dt_bs >= a->D && (a->z == nullptr || a->z_bs >= a->D) && a->Bm_bs >= a->S && a->Cm_bs >= a->S && a->y_bs >= a->D),
                "selective_scan_step: row strides below the channels / states");
  scan_dispatch(*a, [&](auto* tp, auto Gc) {
    typedef typename std::remove_pointer<decltype(tp)>::type T;
    constexpr int G = Gc();
    const int64_t n = (int64_t)a->B * a->D * G;
    hipLaunchKernelGGL((scan_step_kernel<T, G>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, *a);
  });
  SEG_CHECK_LAUNCH("selective_scan_step");
  return SEG_OK;
}
