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
//
// Measured: 8 prompts of up to 2048 rows x 2048 channels x 16 states, bf16: main launch 150 us, the chunks' first pass 98 (the main loop
// issues 35 slots per four states and row - the floor of one exponential and four operations is 32 - and staging another fifth); training
// step 8 x 1024 x 1024 x 16, f16: forward 33 + 47, backward 36 + 160 us at two waves per SIMD (255 registers); one row of 64 x 2048 x 16
// 7.7 us (2.2 TB/s of states).
#include "seq_common.h"

namespace {

constexpr int TT = 32;            // rows per tile = distance of the saved states
constexpr int SUB = 8;            // rows whose a and h the backward pass holds in registers
constexpr int MAXS = 64;
constexpr float LOG2E = 1.4426950408889634f;

template <int G> struct Lay {
  static constexpr int CB = G <= 4 ? 64 : 256 / G;             // channels per block
  static constexpr int NT = CB * G;                            // threads
  static constexpr int NW = NT / 64;
  static constexpr int SP = 4 * G;                             // states, padded
  static constexpr int CHUNKS = CB / 8;                        // 8-channel pieces of a row
  static constexpr int TASKS = TT * CHUNKS;                    // pieces of a tile
  static constexpr int PIECES = TASKS > NT ? TASKS / NT : 1;   // of these per thread (G > 4: the first TASKS threads, one each)
  static constexpr int ROWS = NT / CHUNKS;                     // rows between a thread's pieces
};

__device__ __forceinline__ float exp2_f(float v) { return __builtin_amdgcn_exp2f(v); }
// max(v, 0) + log(1 + e), e = exp(-|v|) in (0, 1]: log(1 + e) = e P(e), P of degree 8 fitted to 3e-8 on [0, 1] - half the instructions of a
// logarithm whose argument's lost bits are corrected.  Relative error, measured in half steps of 2^-24: 3 around zero, about |v| in the left
// tail (the exponential's argument is rounded: 15 at -16, 61 at -80), 1 to the right
__device__ __forceinline__ float softplus_f(float v) {
  const float e = __expf(-fabsf(v));
  float P = 0.0052326812f;
  P = fmaf(P, e, -0.0295051865f);
  P = fmaf(P, e, 0.0782258667f);
  P = fmaf(P, e, -0.136632386f);
  P = fmaf(P, e, 0.191060034f);
  P = fmaf(P, e, -0.248429813f);
  P = fmaf(P, e, 0.333190967f);
  P = fmaf(P, e, -0.499994931f);
  P = fmaf(P, e, 0.99999997f);
  return fmaf(P, e, fmaxf(v, 0.f));
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

// y[0..3]: a channel's parts of four rows in each of its G lanes.  Stores the rows' sums at o[row * ld]: lane g & 3 the row of that number,
// no lane waits for another's branch (in two halvings for G = 4: a lane keeps what it will store and sends the rest)
template <int G> __device__ __forceinline__ void store_rows4(const float* y, int g, float* o, int ld) {
  if constexpr (G == 4) {
    const bool odd = g & 1, up = g & 2;
    const float a = (odd ? y[1] : y[0]) + dpp<DPP_XOR1>(odd ? y[0] : y[1]), b = (odd ? y[3] : y[2]) + dpp<DPP_XOR1>(odd ? y[2] : y[3]);
    o[g * ld] = (up ? b : a) + dpp<DPP_XOR2>(up ? a : b);
  } else if constexpr (G > 4) {
    float s[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = group_sum<G>(y[k]);
    o[(g & 3) * ld] = (g & 2) ? ((g & 1) ? s[3] : s[2]) : ((g & 1) ? s[1] : s[0]);       // (lanes of one number store the same value)
  } else {
#pragma unroll
    for (int k = 0; k < 4; k += G) {
      float s[G];
#pragma unroll
      for (int j = 0; j < G; ++j) s[j] = group_sum<G>(y[k + j]);
      o[(k + g) * ld] = G == 1 ? s[0] : g ? s[G - 1] : s[0];
    }
  }
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
template <bool VEC> __device__ __forceinline__ void load_chan(const float* p, int c, int n, float* f) {
  row_load8<float, VEC>(p + c, p != nullptr ? n : 0, f);
}
// A tile's rows on their way: every thread fetches its 8-channel pieces (PIECES of them: one row each) and its share of the tile's
// Bm / Cm elements a tile ahead, in their memory format, so that no wave waits for memory between two tiles.
template <typename T, bool VEC> struct Raw {
  typedef T tv __attribute__((ext_vector_type(8)));
  tv v;
  __device__ __forceinline__ void load(const T* p, int n) { v = raw_load8<T, VEC>(p, n); }
  __device__ __forceinline__ float operator[](int j) const { return (float)v[j]; }
};
template <typename T, int G> struct RawStates {
  static constexpr int N = TT * Lay<G>::SP / Lay<G>::NT;
  T v[N];
  __device__ __forceinline__ void load(const T* m, int64_t bs, int64_t ld, int b, int t0, int len, int S) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = threadIdx.x + i * Lay<G>::NT, t = t0 + e / Lay<G>::SP, s = e % Lay<G>::SP;
      v[i] = (t < len && s < S) ? m[b * bs + t * ld + s] : (T)0.f;
    }
  }
  __device__ __forceinline__ void put(float* dst) const {
#pragma unroll
    for (int i = 0; i < N; ++i) dst[threadIdx.x + i * Lay<G>::NT] = (float)v[i];
  }
};
// delta of eight channels from the raw step; 0 behind the length
__device__ __forceinline__ float delta_of(const seg_scan_args& p, float dt, float bias, bool on) {
  const float v = dt + bias;
  return on ? (p.softplus ? softplus_f(v) : v) : 0.f;
}

// MAIN: y, saved states and the last state from the chunk's true start; else the chunk's last state from zero and its sum of delta
template <typename T, bool VEC, int G, bool MAIN>
__global__ __launch_bounds__(Lay<G>::NT) void scan_fwd_kernel(const seg_scan_args p, int clen, int nch, float* start, float* sumd) {
  typedef Lay<G> Y;
  __shared__ __align__(16) float2 sdu[TT][Y::CB];              // (written two channels, 16 bytes, at a time)
  __shared__ __align__(16) float sB[TT * Y::SP], sC[MAIN ? TT * Y::SP : 1];
  __shared__ __align__(16) float sy[MAIN ? TT : 1][Y::CB];
  const int tid = threadIdx.x, g = tid % G, c = tid / G, b = blockIdx.z, chunk = blockIdx.y;
  const int c0 = blockIdx.x * Y::CB, d = c0 + c, len = scan_len(p, b);
  const bool live = d < p.D;
  const int tbeg = chunk * clen, tend = tbeg + clen < p.L ? tbeg + clen : p.L;
  const int row0 = tid / Y::CHUNKS, q0c = (tid % Y::CHUNKS) * 8, tc = c0 + q0c, tn = tc < p.D ? p.D - tc : 0;      // this thread's piece of the rows
  const bool worker = tid < Y::TASKS;
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
  Raw<T, VEC> ru[Y::PIECES], rt[Y::PIECES], rz[MAIN ? Y::PIECES : 1], cu[Y::PIECES], cz[MAIN ? Y::PIECES : 1];
  RawStates<T, G> rB, rC;
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < Y::PIECES; ++i) {
      const int t = t0 + row0 + i * Y::ROWS, n = worker && t < len ? tn : 0;
      ru[i].load((const T*)p.u + b * p.u_bs + t * p.u_ld + tc, n);
      rt[i].load((const T*)p.dt + b * p.dt_bs + t * p.dt_ld + tc, n);
      if constexpr (MAIN) rz[i].load((const T*)p.z + b * p.z_bs + t * p.z_ld + tc, p.z != nullptr ? n : 0);
    }
    rB.load((const T*)p.Bm, p.Bm_bs, p.Bm_ld, b, t0, len, p.S);
    if constexpr (MAIN) rC.load((const T*)p.Cm, p.Cm_bs, p.Cm_ld, b, t0, len, p.S);
  };
  const int tlive = tend < len ? tend : len;                   // rows from here on leave the state as it is: their y is 0
  if (tbeg < tlive) fetch(tbeg);
  for (int t0 = tbeg; t0 < tend; t0 += TT) {
    if constexpr (MAIN) {
      if (p.saved != nullptr && live) store_states(p.saved + (((int64_t)b * nck + t0 / TT) * p.D + d) * p.S, 4 * g, p.S, h);
    }
    if (t0 < tlive) {                                          // (block-uniform)
#pragma unroll
      for (int i = 0; i < Y::PIECES; ++i) {
        const int r = row0 + i * Y::ROWS;
        cu[i] = ru[i];
        if constexpr (MAIN) cz[i] = rz[i];
        if (worker) {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float d0 = delta_of(p, rt[i][j], bias[j], t0 + r < len), d1 = delta_of(p, rt[i][j + 1], bias[j + 1], t0 + r < len);
            *reinterpret_cast<f4*>(&sdu[r][q0c + j]) = f4{d0, d0 * ru[i][j], d1, d1 * ru[i][j + 1]};
          }
        }
      }
      rB.put(sB);
      if constexpr (MAIN) rC.put(sC);
      if (t0 + TT < tlive) fetch(t0 + TT);
      __syncthreads();
      // four rows at a time, the next four rows' operands on their way from the LDS meanwhile
      float2 dn[4];
      f4 Bn[4], Cn[4];
      auto ahead = [&](int r) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          dn[k] = sdu[r + k][c];
          Bn[k] = *reinterpret_cast<const f4*>(sB + (r + k) * Y::SP + 4 * g);
          if constexpr (MAIN) Cn[k] = *reinterpret_cast<const f4*>(sC + (r + k) * Y::SP + 4 * g);
        }
      };
      ahead(0);
#pragma unroll 2
      for (int r = 0; r < TT; r += 4) {
        float2 dd[4];
        f4 B4[4], C4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) { dd[k] = dn[k]; B4[k] = Bn[k]; C4[k] = Cn[k]; }
        if (r + 4 < TT) ahead(r + 4);
        float y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
          for (int i = 0; i < 4; ++i) h[i] = fmaf(exp2_f(dd[k].x * A2[i]), h[i], dd[k].y * B4[k][i]);
          if constexpr (MAIN) y[k] = fmaf(C4[k][3], h[3], fmaf(C4[k][2], h[2], fmaf(C4[k][1], h[1], C4[k][0] * h[0])));
          else dsum += dd[k].x;
        }
        if constexpr (MAIN) store_rows4<G>(y, g, &sy[r][c], Y::CB);
      }
      __syncthreads();
    }
    if constexpr (MAIN) {
      if (worker && tn > 0) {
#pragma unroll
        for (int i = 0; i < Y::PIECES; ++i) {
          const int r = row0 + i * Y::ROWS, t = t0 + r;
          if (t < tend) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = 0.f;
            if (t < len) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                y[j] = fmaf(skip[j], cu[i][j], sy[r][q0c + j]);
                if (p.z != nullptr) y[j] *= silu_f(cz[i][j]);
              }
            }
            row_store8<T, VEC>((T*)p.y + b * p.y_bs + t * p.y_ld + tc, tn, y);
          }
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

// A chunk's whole factor lies past 32 bits where states grow (softplus off and steps of the wrong sign): what is still zero stays zero there
__device__ __forceinline__ float carried(float factor, float h, float own) { return h != 0.f ? fmaf(factor, h, own) : own; }
// the chunks in order: in place, a chunk's own last state becomes the state in front of it
constexpr int JOIN = 8;          // chunks whose parts are on their way together (1 x 100000 x 64 x 16, 1563 chunks: 535 us one at a time, 200)
__global__ __launch_bounds__(256) void scan_join_kernel(const seg_scan_args p, int nch, float* start, const float* sumd) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)p.D * p.S;
  const int b = blockIdx.y;
  if (e >= n) return;
  const int64_t d = e / p.S;
  const float A2 = p.A[e] * LOG2E;
  float h = p.state != nullptr ? p.state[b * n + e] : 0.f;
  const int64_t o0 = (int64_t)b * nch;
  for (int k0 = 0; k0 < nch - 1; k0 += JOIN) {
    float own[JOIN], a[JOIN];
#pragma unroll
    for (int k = 0; k < JOIN; ++k)
      if (k0 + k < nch - 1) {
        own[k] = start[(o0 + k0 + k) * n + e];
        a[k] = sumd[(o0 + k0 + k) * p.D + d];
      }
#pragma unroll
    for (int k = 0; k < JOIN; ++k)
      if (k0 + k < nch - 1) {
        start[(o0 + k0 + k) * n + e] = h;
        h = carried(exp2_f(A2 * a[k]), h, own[k]);
      }
  }
  start[(o0 + nch - 1) * n + e] = h;                           // (the last chunk's own last state was not computed: nothing starts behind it)
}
// the same for the adjoint, from the last chunk: a chunk's own part becomes the adjoint that enters it from behind
__global__ __launch_bounds__(256) void scan_join_bwd_kernel(const seg_scan_args p, int nch, float* adj, const float* sumd) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)p.D * p.S;
  const int b = blockIdx.y;
  if (e >= n) return;
  const int64_t d = e / p.S;
  const float A2 = p.A[e] * LOG2E;
  float q = p.dstate_out != nullptr ? p.dstate_out[b * n + e] : 0.f;
  const int64_t o0 = (int64_t)b * nch;
  for (int k0 = nch - 1; k0 > 0; k0 -= JOIN) {
    float own[JOIN], a[JOIN];
#pragma unroll
    for (int k = 0; k < JOIN; ++k)
      if (k0 - k > 0) {
        own[k] = adj[(o0 + k0 - k) * n + e];
        a[k] = sumd[(o0 + k0 - k) * p.D + d];
      }
#pragma unroll
    for (int k = 0; k < JOIN; ++k)
      if (k0 - k > 0) {
        adj[(o0 + k0 - k) * n + e] = q;
        q = carried(exp2_f(A2 * a[k]), q, own[k]);
      }
  }
  adj[o0 * n + e] = q;                                         // (the first chunk's own part was not computed: nothing lies in front of it)
}

// dp = dy silu(z) of a piece
template <typename T, bool VEC>
__device__ __forceinline__ float dp_of(const seg_scan_args& p, const Raw<T, VEC>& dy, const Raw<T, VEC>& z, int j) {
  return p.z != nullptr ? dy[j] * silu_f(z[j]) : dy[j];
}

// a chunk's own part of the adjoint in front of it, and its sum of delta (chunks 1 ..: blockIdx.y + 1)
template <typename T, bool VEC, int G>
__global__ __launch_bounds__(Lay<G>::NT) void scan_bwd_local_kernel(const seg_scan_args p, int clen, int nch, float* adj, float* sumd) {
  typedef Lay<G> Y;
  __shared__ __align__(16) float2 sdp[TT][Y::CB];              // (written two channels, 16 bytes, at a time)
  __shared__ __align__(16) float sC[TT * Y::SP];
  const int tid = threadIdx.x, g = tid % G, c = tid / G, b = blockIdx.z, chunk = blockIdx.y + 1;
  const int c0 = blockIdx.x * Y::CB, d = c0 + c, len = scan_len(p, b);
  const bool live = d < p.D;
  const int tbeg = chunk * clen, tend = tbeg + clen < p.L ? tbeg + clen : p.L, tlive = tend < len ? tend : len;
  const int row0 = tid / Y::CHUNKS, q0c = (tid % Y::CHUNKS) * 8, tc = c0 + q0c, tn = tc < p.D ? p.D - tc : 0;
  const bool worker = tid < Y::TASKS;
  float bias[8];
  load_chan<VEC>(p.dt_bias, tc, tn, bias);
  f4 A2 = {0.f, 0.f, 0.f, 0.f}, P = {1.f, 1.f, 1.f, 1.f}, q = A2;
  if (live) A2 = load_states(p.A + (int64_t)d * p.S, 4 * g, p.S) * LOG2E;
  float dsum = 0.f;
  Raw<T, VEC> rt[Y::PIECES], ry[Y::PIECES], rz[Y::PIECES];
  RawStates<T, G> rC;
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < Y::PIECES; ++i) {
      const int t = t0 + row0 + i * Y::ROWS, n = worker && t < len ? tn : 0;
      rt[i].load((const T*)p.dt + b * p.dt_bs + t * p.dt_ld + tc, n);
      ry[i].load((const T*)p.dy + b * p.dy_bs + t * p.dy_ld + tc, n);
      rz[i].load((const T*)p.z + b * p.z_bs + t * p.z_ld + tc, p.z != nullptr ? n : 0);
    }
    rC.load((const T*)p.Cm, p.Cm_bs, p.Cm_ld, b, t0, len, p.S);
  };
  // GROWN: the factors from their logarithms' sum, terms of zero left out
  auto walk = [&](auto GROWN) {
    if (tbeg < tlive) fetch(tbeg);
    for (int t0 = tbeg; t0 < tlive; t0 += TT) {
      if (worker) {
#pragma unroll
        for (int i = 0; i < Y::PIECES; ++i) {
          const int r = row0 + i * Y::ROWS;
#pragma unroll
          for (int j = 0; j < 8; j += 2)
            *reinterpret_cast<f4*>(&sdp[r][q0c + j]) = f4{delta_of(p, rt[i][j], bias[j], t0 + r < len), dp_of<T, VEC>(p, ry[i], rz[i], j),
                                                         delta_of(p, rt[i][j + 1], bias[j + 1], t0 + r < len), dp_of<T, VEC>(p, ry[i], rz[i], j + 1)};
        }
      }
      rC.put(sC);
      if (t0 + TT < tlive) fetch(t0 + TT);
      __syncthreads();
#pragma unroll 4
      for (int r = 0; r < TT; ++r) {
        const float2 dd = sdp[r][c];
        const f4 C4 = *reinterpret_cast<const f4*>(sC + r * Y::SP + 4 * g);
        dsum += dd.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = C4[i] * dd.y;
          if constexpr (GROWN()) {
            if (x != 0.f) q[i] = fmaf(exp2_f(dsum * A2[i]), x, q[i]);
          } else {
            P[i] *= exp2_f(dd.x * A2[i]);
            q[i] = fmaf(P[i], x, q[i]);
          }
        }
      }
      __syncthreads();
    }
  };
  walk(std::false_type{});
  // (a product that has left 32 bits stays outside of them; the block's other lanes keep what they have)
  const bool far = !(P[0] + P[1] + P[2] + P[3] < INFINITY);
  if (__syncthreads_or(far)) {
    const f4 near = q;
    dsum = 0.f;
    q = f4{0.f, 0.f, 0.f, 0.f};
    walk(std::true_type{});
    if (!far) q = near;
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
__global__ __launch_bounds__(Lay<G>::NT, 2) void scan_bwd_kernel(const seg_scan_args p, int clen, const float* adj, float* pbc, float* pA, float* pD) {
  typedef Lay<G> Y;
  __shared__ f4 sx[TT][Y::CB];                               // delta, u -> sum g B, dp -> sum g a h A, -> C . h
  __shared__ __align__(16) float sB[TT * Y::SP], sC[TT * Y::SP];
  __shared__ __align__(16) float sbc[Y::NW][SUB][2][Y::SP];
  __shared__ f4 shs[TT / SUB - 1][Y::NT];                    // the states in front of every SUB rows of the tile but the first
  const int tid = threadIdx.x, g = tid % G, c = tid / G, b = blockIdx.z, chunk = blockIdx.y, nch = gridDim.y;
  const int lane = tid & 63, wave = tid >> 6;
  const int c0 = blockIdx.x * Y::CB, d = c0 + c, len = scan_len(p, b);
  const bool live = d < p.D;
  const int tbeg = chunk * clen, tend = tbeg + clen < p.L ? tbeg + clen : p.L, tlive = tend < len ? tend : len;
  const int row0 = tid / Y::CHUNKS, q0c = (tid % Y::CHUNKS) * 8, tc = c0 + q0c, tn = tc < p.D ? p.D - tc : 0;
  const bool worker = tid < Y::TASKS;
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
  // rows behind the length: gradients are 0, the adjoint passes
  for (int t = (tlive > tbeg ? tlive : tbeg) + row0; worker && tn > 0 && t < tend; t += (Y::ROWS < TT ? Y::ROWS : TT)) {
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = 0.f;
    if (p.du != nullptr) row_store8<T, VEC>((T*)p.du + b * p.du_bs + t * p.du_ld + tc, tn, o);
    if (p.ddt != nullptr) row_store8<T, VEC>((T*)p.ddt + b * p.ddt_bs + t * p.ddt_ld + tc, tn, o);
    if (p.dz != nullptr) row_store8<T, VEC>((T*)p.dz + b * p.dz_bs + t * p.dz_ld + tc, tn, o);
  }
  if (pbc != nullptr) {
    const int t1 = tlive > tbeg ? tlive : tbeg;
    for (int64_t e = tid; e < (int64_t)(tend - t1) * 2 * p.S; e += Y::NT) pbc[(((int64_t)blockIdx.x * p.B + b) * p.L + t1) * 2 * p.S + e] = 0.f;
  }
  Raw<T, VEC> ru[Y::PIECES], rt[Y::PIECES], rz[Y::PIECES], ry[Y::PIECES];
  RawStates<T, G> rB, rC;
  f4 rh = {0.f, 0.f, 0.f, 0.f};
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < Y::PIECES; ++i) {
      const int t = t0 + row0 + i * Y::ROWS, n = worker && t < len ? tn : 0;
      ru[i].load((const T*)p.u + b * p.u_bs + t * p.u_ld + tc, n);
      rt[i].load((const T*)p.dt + b * p.dt_bs + t * p.dt_ld + tc, n);
      rz[i].load((const T*)p.z + b * p.z_bs + t * p.z_ld + tc, p.z != nullptr ? n : 0);
      ry[i].load((const T*)p.dy + b * p.dy_bs + t * p.dy_ld + tc, n);
    }
    rB.load((const T*)p.Bm, p.Bm_bs, p.Bm_ld, b, t0, len, p.S);
    rC.load((const T*)p.Cm, p.Cm_bs, p.Cm_ld, b, t0, len, p.S);
    if (live) rh = load_states(p.saved + (((int64_t)b * nck + t0 / TT) * p.D + d) * p.S, 4 * g, p.S);
  };
  const int ntile = tlive > tbeg ? (tlive - tbeg + TT - 1) / TT : 0;
  if (ntile > 0) fetch(tbeg + (ntile - 1) * TT);
  for (int tile = ntile - 1; tile >= 0; --tile) {
    const int t0 = tbeg + tile * TT;
    Raw<T, VEC> cu[Y::PIECES], ct[Y::PIECES], cz[Y::PIECES], cy[Y::PIECES];
    f4 h = rh;
#pragma unroll
    for (int i = 0; i < Y::PIECES; ++i) {
      const int r = row0 + i * Y::ROWS;
      cu[i] = ru[i]; ct[i] = rt[i]; cz[i] = rz[i]; cy[i] = ry[i];
      if (worker) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sx[r][q0c + j] = f4{delta_of(p, rt[i][j], bias[j], t0 + r < len), ru[i][j], dp_of<T, VEC>(p, ry[i], rz[i], j), 0.f};
      }
    }
    rB.put(sB);
    rC.put(sC);
    __syncthreads();
    // (a row's LDS reads are issued one row ahead, no further: left alone the compiler moves all of a sub-tile's reads to its front, and
    // their registers leave one wave per SIMD)
    const f4 h0 = h;
#pragma unroll 1
    for (int s = 1; s < TT / SUB; ++s) {
      const int r0 = (s - 1) * SUB;
      float2 x = *reinterpret_cast<const float2*>(&sx[r0][c]);
      f4 B4 = *reinterpret_cast<const f4*>(sB + r0 * Y::SP + 4 * g);
#pragma unroll
      for (int k = 0; k < SUB; ++k) {
        const float2 xc = x;
        const f4 Bc = B4;
        if (k + 1 < SUB) {
          x = *reinterpret_cast<const float2*>(&sx[r0 + k + 1][c]);
          B4 = *reinterpret_cast<const f4*>(sB + (r0 + k + 1) * Y::SP + 4 * g);
        }
        const float du = xc.x * xc.y;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = fmaf(exp2_f(xc.x * A2[i]), h[i], du * Bc[i]);
        __builtin_amdgcn_sched_barrier(0);
      }
      shs[s - 1][tid] = h;
    }
#pragma unroll 1
    for (int s = TT / SUB - 1; s >= 0; --s) {
      f4 a[SUB], hp[SUB];
      const int r0 = s * SUB;
      h = s > 0 ? shs[s - 1][tid] : h0;
      {
        float2 x = *reinterpret_cast<const float2*>(&sx[r0][c]);
        f4 B4 = *reinterpret_cast<const f4*>(sB + r0 * Y::SP + 4 * g), C4 = *reinterpret_cast<const f4*>(sC + r0 * Y::SP + 4 * g);
#pragma unroll
        for (int k = 0; k < SUB; ++k) {
          const float2 xc = x;
          const f4 Bc = B4, Cc = C4;
          if (k + 1 < SUB) {
            x = *reinterpret_cast<const float2*>(&sx[r0 + k + 1][c]);
            B4 = *reinterpret_cast<const f4*>(sB + (r0 + k + 1) * Y::SP + 4 * g);
            C4 = *reinterpret_cast<const f4*>(sC + (r0 + k + 1) * Y::SP + 4 * g);
          }
          const float du = xc.x * xc.y;
          hp[k] = h;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            a[k][i] = exp2_f(xc.x * A2[i]);
            h[i] = fmaf(a[k][i], h[i], du * Bc[i]);
          }
          const float y = group_sum<G>(fmaf(Cc[3], h[3], fmaf(Cc[2], h[2], fmaf(Cc[1], h[1], Cc[0] * h[0]))));
          sx[r0 + k][c][3] = y;                                // (every lane of the channel holds and stores the same sum: no branch)
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      f4 x = sx[r0 + SUB - 1][c];
      f4 B4 = *reinterpret_cast<const f4*>(sB + (r0 + SUB - 1) * Y::SP + 4 * g), C4 = *reinterpret_cast<const f4*>(sC + (r0 + SUB - 1) * Y::SP + 4 * g);
#pragma unroll
      for (int k = SUB - 1; k >= 0; --k) {
        const f4 xc = x, Bc = B4, Cc = C4;
        if (k > 0) {
          x = sx[r0 + k - 1][c];
          B4 = *reinterpret_cast<const f4*>(sB + (r0 + k - 1) * Y::SP + 4 * g);
          C4 = *reinterpret_cast<const f4*>(sC + (r0 + k - 1) * Y::SP + 4 * g);
        }
        const float du = xc[0] * xc[1];
        float v[8], w[2], sgB = 0.f, sA = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float gi = fmaf(Cc[i], xc[2], q[i]);
          const float ga = gi * a[k][i], gh = ga * hp[k][i];
          sgB = fmaf(gi, Bc[i], sgB);
          sA = fmaf(gh, A[i], sA);
          dA[i] = fmaf(gh, xc[0], dA[i]);
          v[i] = gi * du;
          v[4 + i] = xc[2] * h[i];
          q[i] = ga;
        }
        h = hp[k];
        sgB = group_sum<G>(sgB);
        sA = group_sum<G>(sA);
        sx[r0 + k][c][1] = sgB;
        sx[r0 + k][c][2] = sA;
        lane_sums<G>(v, w);
        *reinterpret_cast<float2*>(&sbc[wave][k][lane >> 5][4 * g + 2 * ((lane >> 4) & 1)]) = float2{w[0], w[1]};
        __builtin_amdgcn_sched_barrier(0);
      }
      __syncthreads();
      if (pbc != nullptr) {
        for (int e = tid; e < SUB * 2 * Y::SP; e += Y::NT) {
          const int k = e / (2 * Y::SP), wh = (e / Y::SP) & 1, st = e % Y::SP, t = t0 + s * SUB + k;
          if (t < tlive && st < p.S) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < Y::NW; ++w) v += sbc[w][k][wh][st];
            pbc[((((int64_t)blockIdx.x * p.B + b) * p.L + t) * 2 + wh) * p.S + st] = v;
          }
        }
      }
      __syncthreads();
    }
    if (tile > 0) fetch(t0 - TT);
    if (worker && tn > 0) {
#pragma unroll
      for (int i = 0; i < Y::PIECES; ++i) {
        const int r = row0 + i * Y::ROWS, t = t0 + r;
        if (t < tlive) {
          float o[8];
          f4 x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = sx[r][q0c + j];
          if (p.du != nullptr) {
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = fmaf(skip[j], dp_of<T, VEC>(p, cy[i], cz[i], j), x[j][0] * x[j][1]);
            row_store8<T, VEC>((T*)p.du + b * p.du_bs + t * p.du_ld + tc, tn, o);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            o[j] = fmaf(x[j][1], cu[i][j], x[j][2]);
            if (p.softplus) o[j] *= sigmoid_f(ct[i][j] + bias[j]);
            accB[j] += o[j];
            accD[j] = fmaf(dp_of<T, VEC>(p, cy[i], cz[i], j), cu[i][j], accD[j]);
          }
          if (p.ddt != nullptr) row_store8<T, VEC>((T*)p.ddt + b * p.ddt_bs + t * p.ddt_ld + tc, tn, o);
          if (p.dz != nullptr) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              o[j] = cy[i][j] * fmaf(skip[j], cu[i][j], x[j][3]) * silu_slope_f(cz[i][j]);
            }
            row_store8<T, VEC>((T*)p.dz + b * p.dz_bs + t * p.dz_ld + tc, tn, o);
          }
        }
      }
    }
    __syncthreads();
  }
  const int64_t o = (int64_t)b * nch + chunk;
  if (live && pA != nullptr) store_states(pA + (o * p.D + d) * p.S, 4 * g, p.S, dA);
  if (live && p.dstate != nullptr && chunk == 0) store_states(p.dstate + ((int64_t)b * p.D + d) * p.S, 4 * g, p.S, q);
  if (pD != nullptr) {
    // the threads of a channel piece: ROWS rows of CB values, added by the block's first CB threads, dD and then ddt_bias
    float* sh = reinterpret_cast<float*>(&sx[0][0]);
    constexpr int R = Y::ROWS;
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
      y *= silu_f(z);
    }
    ((T*)p.y)[b * p.y_bs + d] = (T)y;
  }
}

inline int scan_group(int S) { return S <= 4 ? 1 : S <= 8 ? 2 : S <= 16 ? 4 : S <= 32 ? 8 : 16; }
inline int scan_cb(int S) { const int G = scan_group(S); return G <= 4 ? 64 : 256 / G; }

struct ScanPlan { int nblk, nch, clen; };
inline ScanPlan scan_plan(const seg_scan_args& a, bool bwd) {
  ScanPlan s;
  const int cb = scan_cb(a.S);
  s.nblk = (a.D + cb - 1) / cb;
  const int64_t blocks = (int64_t)s.nblk * a.B;
  // chunks until this many blocks are there.  Forward: 256 / 512 / 1024 / 2048 blocks took 353 / 313 / 273 / 255 us (8 prompts of up to
  // 2048 rows, 2048 channels, 16 states, bf16: short sequences leave early, many blocks level that); backward: a block keeps two waves
  // per SIMD busy at most, and every chunk adds partial rows of dA - 256 / 512 / 1024: 423 / 326 / 325 us (8 x 1024 x 1024 x 16, f16)
  const int64_t want = bwd ? 512 : 2048;
  int64_t nch = (want + blocks - 1) / (blocks < 1 ? 1 : blocks);
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
  SEG_CHECK_ARG(a->B >= 0 && a->L >= 0 && a->D > 0 && a->D <= (1 << 30), "%s: B %d, L %d, D %d (2^30 at most)", name, a->B, a->L, a->D);
  SEG_CHECK_ARG(a->S >= 1 && a->S <= MAXS, "%s: %d states (1 .. %d)", name, a->S, MAXS);
  SEG_CHECK_ARG(a->B <= 65535, "%s: %d sequences in one call (65535 at most)", name, a->B);
  SEG_CHECK_ARG(a->L <= (1 << 30), "%s: %d rows in one call (2^30 at most)", name, a->L);
  const int64_t G = scan_group(a->S), cb = scan_cb(a->S);
  SEG_CHECK_ARG(grid_takes((a->D + cb - 1) / cb * cb * G), "%s: %d channels of %d states are too many for one call (2^32 pieces of four states)", name, a->D, a->S);
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
  const ScanPlan s = scan_plan(*a, false);
  if (s.nch <= 1) return 0;
  return ((int64_t)a->B * s.nch * a->D * a->S + 3) / 4 * 16 + (int64_t)a->B * s.nch * a->D * 4;
}
extern "C" int64_t seg_selective_scan_bwd_workspace_bytes(const seg_scan_args* a) {
  if (a == nullptr || a->B <= 0 || a->L <= 0 || a->D <= 0 || a->S <= 0) return 0;
  return scan_bwd_space(*a, scan_plan(*a, true)).total * 4;
}

extern "C" int seg_selective_scan_fwd(const seg_scan_args* a, seg_stream_t stream) {
  if (int rc = check_scan(a, "selective_scan_fwd")) return rc;
  SEG_CHECK_ARG(a->B == 0 || a->L == 0 || (a->u != nullptr && a->dt != nullptr && a->Bm != nullptr && a->Cm != nullptr && a->y != nullptr), "selective_scan_fwd: u / dt / Bm / Cm / y is NULL");
  SEG_CHECK_ARG(scan_rows_ok(*a) && (a->L <= 1 || a->y_ld >= a->D), "selective_scan_fwd: row strides below the channels / states");
  SEG_CHECK_ARG(a->state_out == nullptr || a->state_out != a->state, "selective_scan_fwd: state_out may not be state");
  if (a->B == 0 || (a->L == 0 && a->state_out == nullptr)) return SEG_OK;
  const ScanPlan s = scan_plan(*a, false);
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
      const dim3 front((unsigned)s.nblk, (unsigned)s.nch - 1, (unsigned)a->B);           // (the last chunk's own last state starts nothing)
      if (vec) hipLaunchKernelGGL((scan_fwd_kernel<T, true, G, false>), front, dim3(NT), 0, st, *a, s.clen, s.nch, start, sumd);
      else hipLaunchKernelGGL((scan_fwd_kernel<T, false, G, false>), front, dim3(NT), 0, st, *a, s.clen, s.nch, start, sumd);
      const int64_t n = (int64_t)a->D * a->S;
      hipLaunchKernelGGL(scan_join_kernel, dim3((unsigned)((n + 255) / 256), (unsigned)a->B), dim3(256), 0, st, *a, s.nch, start, sumd);
    }
    if (vec) hipLaunchKernelGGL((scan_fwd_kernel<T, true, G, true>), grid, dim3(NT), 0, st, *a, s.clen, s.nch, start, sumd);
    else hipLaunchKernelGGL((scan_fwd_kernel<T, false, G, true>), grid, dim3(NT), 0, st, *a, s.clen, s.nch, start, sumd);
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
  const ScanPlan s = scan_plan(*a, true);
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
        const dim3 back((unsigned)s.nblk, (unsigned)s.nch - 1, (unsigned)a->B);          // (nothing lies in front of the first chunk)
        if (vec) hipLaunchKernelGGL((scan_bwd_local_kernel<T, true, G>), back, dim3(NT), 0, st, *a, s.clen, s.nch, adj, sumd);
        else hipLaunchKernelGGL((scan_bwd_local_kernel<T, false, G>), back, dim3(NT), 0, st, *a, s.clen, s.nch, adj, sumd);
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
  // dA and, their columns being neighbours, dD / ddt_bias in one launch; outputs that are not neighbours take another
  const float *pAs = none ? nullptr : ws + w.pA, *pDs = none ? nullptr : ws + w.pD;
  const int64_t D2 = 2 * (int64_t)a->D;
  ColsumSet sa{pAs, parts, n, a->dA != nullptr ? n : 0, a->dA}, sd{pDs, parts, D2, 0, a->dD};
  if (a->dD != nullptr && a->ddt_bias == a->dD + a->D) {
    sd.cols = D2;
    launch_colsum_sets(sa, sd, st);
  } else {
    launch_colsum_sets(sa, sd, st);
    launch_colsum_pair(pDs, parts, D2, a->D, a->dD, a->D, a->ddt_bias, st);
  }
  SEG_CHECK_LAUNCH("selective_scan_bwd");
  return SEG_OK;
}

extern "C" int seg_selective_scan_step(const seg_scan_args* a, seg_stream_t stream) {
  if (int rc = check_scan(a, "selective_scan_step")) return rc;
  if (a->B == 0) return SEG_OK;
  SEG_CHECK_ARG(a->u != nullptr && a->dt != nullptr && a->Bm != nullptr && a->Cm != nullptr && a->y != nullptr, "selective_scan_step: u / dt / Bm / Cm / y is NULL");
  SEG_CHECK_ARG(a->B == 1 || (a->u_bs >= a->D && a->dt_bs >= a->D && (a->z == nullptr || a->z_bs >= a->D) && a->Bm_bs >= a->S && a->Cm_bs >= a->S && a->y_bs >= a->D),
                "selective_scan_step: row strides below the channels / states");
  SEG_CHECK_ARG(grid_takes((int64_t)a->B * a->D * scan_group(a->S) + 255), "selective_scan_step: %d sequences of %d channels of %d states are too many for one call (2^32 pieces of four states)",
                a->B, a->D, a->S);
  scan_dispatch(*a, [&](auto* tp, auto Gc) {
    typedef typename std::remove_pointer<decltype(tp)>::type T;
    constexpr int G = Gc();
    const int64_t n = (int64_t)a->B * a->D * G;
    hipLaunchKernelGGL((scan_step_kernel<T, G>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, *a);
  });
  SEG_CHECK_LAUNCH("selective_scan_step");
  return SEG_OK;
}
