// Matrix product with its epilogue and its two gradients (seg_linear_fwd / _bwd_data / _bwd_weight).  All three are
//   C[i][j] = sum_k A(i, k) B(j, k)
// with the operands as the caller stores them:
//   pass            i        j        k       A             B
//   fwd             rows     units    inputs  x  [i][k]     w [j][k]      z = C + bias, y = act(z) + residual
//   bwd_data        rows     inputs   units   dy [i][k]     w [k][j]      y = C act'(z) + residual
//   bwd_weight      units    inputs   rows    dy [k][i]     x [k][j]      dw = C (fp32)
#include "seq_common.h"
#include "igemm_common.h"

namespace {

constexpr int TPB = 256;
typedef short s4v __attribute__((__vector_size__(4 * sizeof(short))));
typedef __attribute__((address_space(3))) s4v* lds_s4v_ptr;
typedef __attribute__((address_space(3))) unsigned char* lds_byte_ptr;

struct GemmArgs {
  const void *A, *B;
  int64_t a_ld, b_ld;
  int64_t I, Kd;
  int J;
  int ti, tj;                    // tiles along i and j
  int splits;                    // ranges of k contracted by different blocks
  int64_t kper;                  // their length (a multiple of the K step)
  float* part;                   // [splits][I][jp] when splits > 1
  int jp;                        // J in whole pieces of 8
  int act;
  float alpha;
  const float* bias;
  const void* res; int64_t res_ld;
  void* z; int64_t z_ld;
  void* out; int64_t out_ld;
  float* db;                     // bwd_weight: column sums of dy (NULL: not wanted)
  float* part_db;                // [splits][I]
  int vecio;                     // rows of z, residual and out take 16-byte accesses
};

// one element of the result through the pass's epilogue
template <int PASS, typename T> __device__ __forceinline__ void epilogue1(const GemmArgs& p, int64_t i, int j, float v) {
  if constexpr (PASS == SEG_LINEAR_BWD_WEIGHT) {
    ((float*)p.out)[i * p.out_ld + j] = v;
  } else {
    if constexpr (PASS == SEG_LINEAR_FWD) {
      if (p.bias != nullptr) v += p.bias[j];
      if (p.z != nullptr) ((T*)p.z)[i * p.z_ld + j] = (T)v;
      v = seq_act(v, p.act, p.alpha);
    } else {
      if (p.z != nullptr) v *= seq_act_slope((float)((const T*)p.z)[i * p.z_ld + j], p.act, p.alpha);
    }
    if (p.res != nullptr) v += (float)((const T*)p.res)[i * p.res_ld + j];
    ((T*)p.out)[i * p.out_ld + j] = (T)v;
  }
}

template <typename T> __device__ __forceinline__ f16v mfma16(u4 a, u4 b, f16v c) {
  if constexpr (std::is_same<T, half_t>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}
template <typename T> __device__ __forceinline__ u4 ones16() {
  const uint32_t one = std::is_same<T, half_t>::value ? 0x3c003c00u : 0x3f803f80u;
  return u4{one, one, one, one};
}
// a product with ones: every column of the 32 x 32 tile holds the rows' sums
__device__ __forceinline__ void store_sums(const GemmArgs& p, const f16v& acc, int64_t ib, int lane) {
  if ((lane & 31) != 0) return;
  float* o = p.splits > 1 ? p.part_db + blockIdx.y * p.I : p.db;
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const int64_t i = ib + (q & 3) + 8 * (q >> 2) + 4 * (lane >> 5);
    if (i < p.I) o[i] = acc[q];
  }
}

// ---- the kernel for every size, stride and type: 64 x 64 tiles, four waves of one 32 x 32 tile each, operands through registers into the
// LDS in the order they have in memory - rows of BK along k (LD elements apart), or BK rows of 64 along i / j (LDT apart: the four rows of
// a transposing 16-bit read fall into four 64-byte quarters of the banks; 32-bit fragments are single elements there, rows that are four
// apart lie in different halves of them).  VEC: 16-byte rows; otherwise the same accesses at
// any element's address.  The ends of rows and of k go element by element.
template <typename T> struct AnyStep { static constexpr int BK = 32, EPT = 8, LD = 40, LDT = 96, SIZE = 32 * 96; };
template <> struct AnyStep<float> { static constexpr int BK = 16, EPT = 4, LD = 20, LDT = 72, SIZE = 64 * 20; };

// 16 bytes of elements, kept in their memory format until they are put into the LDS (unpacked earlier they would be waited for earlier)
template <typename T, bool VEC> __device__ __forceinline__ u4 load_elems(const T* p) {
  if constexpr (VEC) return ld16(p);
  u4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

template <int PASS, typename T, bool VEC>
__global__ __launch_bounds__(TPB) void gemm_any_kernel(const GemmArgs p) {
  typedef AnyStep<T> S;
  constexpr bool AKC = PASS != SEG_LINEAR_BWD_WEIGHT, BKC = PASS == SEG_LINEAR_FWD;
  static_assert(S::SIZE >= 64 * S::LD && S::SIZE >= S::BK * S::LDT, "either order fits");
  __shared__ __align__(16) T smem[2][2][S::SIZE];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 31, fh = lane >> 5;
  const int t = xcd_remap(blockIdx.x, p.ti * p.tj);
  const int64_t i0 = (int64_t)(t / p.tj) * 64;
  const int j0 = (t % p.tj) * 64;
  const int64_t kbeg = blockIdx.y * p.kper, kend = kbeg + p.kper < p.Kd ? kbeg + p.kper : p.Kd;
  constexpr int KCH = S::BK / S::EPT, ICH = 64 / S::EPT;       // chunks per k-contiguous / i-contiguous row
  const T *A = (const T*)p.A, *B = (const T*)p.B;
  typedef T tv __attribute__((ext_vector_type(S::EPT)));
  u4 ra[2], rb[2];                                             // two steps on their way
  // A whole step's chunk without a branch: a row that is not there is read from the last one (its results are dropped), and so is a chunk
  // along i / j where chunks lie inside the operand or outside as a whole.  (Guards here cost the prefetch: the compiler waits for the
  // loads where the guarded and the unguarded path meet - 22 us instead of 14 for 1111 x 333 x 700, f16.)
  auto fetch = [&](const T* base, int64_t ld, bool kc, int64_t r0, int64_t rend, int64_t k) -> u4 {
    const int64_t row = r0 + tid / KCH;
    const int64_t col = r0 + (tid % ICH) * S::EPT;
    return kc ? load_elems<T, VEC>(base + (row < rend ? row : rend - 1) * ld + k + (tid % KCH) * S::EPT)
              : load_elems<T, VEC>(base + (k + tid / ICH) * ld + (col < rend ? col : rend - S::EPT));
  };
  // element by element, what is not there reads as zero: the end of k, and tiles that reach over the operand's columns
  auto fetch_edge = [&](const T* base, int64_t ld, bool kc, int64_t r0, int64_t rend, int64_t k) -> u4 {
    const int64_t row = kc ? r0 + tid / KCH : r0 + (tid % ICH) * S::EPT, kk = kc ? k + (tid % KCH) * S::EPT : k + tid / ICH;
    const T* p0 = kc ? base + row * ld + kk : base + kk * ld + row;
    const int64_t n = kc ? (row < rend ? kend - kk : 0) : (kk < kend ? rend - row : 0);
    tv r;
#pragma unroll
    for (int t = 0; t < S::EPT; ++t) r[t] = t < n ? p0[t] : (T)0.f;
    return __builtin_bit_cast(u4, r);
  };
  auto put = [&](T* s, bool kc, u4 r) {
    st16(kc ? s + (tid / KCH) * S::LD + (tid % KCH) * S::EPT : s + (tid / ICH) * S::LDT + (tid % ICH) * S::EPT, r);
  };
  // a wave's 32 rows from row0, k step ks
  auto frag = [&](const T* s, bool kc, int row0, int ks) -> u4 {
    if (kc) return ld16(s + (row0 + fr) * S::LD + ks * 16 + fh * 8);
    const int tg = lane >> 4, tt = lane & 15;
    const T* a = s + (ks * 16 + 8 * (tg >> 1) + (tt >> 2)) * S::LDT + row0 + 16 * (tg & 1) + 4 * (tt & 3);
    const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v_ptr)a), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v_ptr)(a + 4 * S::LDT));
    const u2 l = __builtin_bit_cast(u2, lo), h = __builtin_bit_cast(u2, hi);
    return u4{l[0], l[1], h[0], h[1]};
  };
  // fp32: four of k, the two halves of a wave taking k0 + 0 .. 3 and k0 + 4 .. 7 (both operands in the same order): 16-byte reads, where
  // single elements took 172 us instead of 149 (2048 x 2048 x 2048, fp32; the matrix rate's floor 112)
  auto elem4 = [&](const T* s, bool kc, int row0, int k0) -> f4 {
    if (kc) return __builtin_bit_cast(f4, ld16(s + (row0 + fr) * S::LD + k0 + 4 * fh));
    f4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = s[(k0 + 4 * fh + e) * S::LDT + row0 + fr];
    return v;
  };
  f16v acc, accb;
#pragma unroll
  for (int q = 0; q < 16; ++q) acc[q] = accb[q] = 0.f;
  const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
  // the sums of dy's columns ride on the first tile column's waves as one more product, with ones
  const bool sums = PASS == SEG_LINEAR_BWD_WEIGHT && p.db != nullptr && j0 == 0 && wj == 0;
  auto step = [&](int buf) {                                   // (buf is a literal at every call: the registers are named at compile time)
    const T *sa = smem[buf][0], *sb = smem[buf][1];
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int ks = 0; ks < S::BK / 8; ++ks) {
        const f4 a = elem4(sa, AKC, wi, 8 * ks), b = elem4(sb, BKC, wj, 8 * ks);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
          if (PASS == SEG_LINEAR_BWD_WEIGHT && sums) accb = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], 1.f, accb, 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const u4 a = frag(sa, AKC, wi, ks);
        acc = mfma16<T>(a, frag(sb, BKC, wj, ks), acc);
        if (PASS == SEG_LINEAR_BWD_WEIGHT && sums) accb = mfma16<T>(a, ones16<T>(), accb);
      }
    }
  };
  auto stage = [&](int buf) {                                  // (the buffer written next is the one whose readers passed the barrier)
    put(smem[buf][0], AKC, ra[buf]);
    put(smem[buf][1], BKC, rb[buf]);
    __syncthreads();
  };
  const bool inside = (AKC || i0 + 64 <= p.I || p.I % S::EPT == 0) && (BKC || j0 + 64 <= p.J || p.J % S::EPT == 0);
  const int64_t kfull = inside ? kbeg + (kend - kbeg) / S::BK * S::BK : kbeg;
  auto fetch2 = [&](int set, int64_t k) {
    ra[set] = fetch(A, p.a_ld, AKC, i0, p.I, k);
    rb[set] = fetch(B, p.b_ld, BKC, j0, p.J, k);
  };
  int64_t k = kbeg;
  if (kbeg < kfull) {
    const int64_t last = kfull - S::BK;                        // (steps behind the last one fetch it again: no branch)
    fetch2(0, kbeg);
    fetch2(1, kbeg + S::BK < last ? kbeg + S::BK : last);
    for (; k + S::BK < kfull; k += 2 * S::BK) {
      stage(0);
      fetch2(0, k + 2 * S::BK < last ? k + 2 * S::BK : last);
      step(0);
      stage(1);
      fetch2(1, k + 3 * S::BK < last ? k + 3 * S::BK : last);
      step(1);
    }
  }
  if (k < kfull) {
    stage(0);
    step(0);
    k += S::BK;
    __syncthreads();
  }
  for (; k < kend; k += S::BK) {
    ra[0] = fetch_edge(A, p.a_ld, AKC, i0, p.I, k);
    rb[0] = fetch_edge(B, p.b_ld, BKC, j0, p.J, k);
    stage(0);
    step(0);
    __syncthreads();                                           // (one buffer here)
  }
  if (sums) store_sums(p, accb, i0 + wi, lane);
  const int j = j0 + wj + fr;
  if (j < p.J) {
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int64_t i = i0 + wi + (q & 3) + 8 * (q >> 2) + 4 * fh;
      if (i < p.I) {
        if (p.splits > 1) p.part[((int64_t)blockIdx.y * p.I + i) * p.jp + j] = acc[q];
        else epilogue1<PASS, T>(p, i, j, acc[q]);
      }
    }
  }
}

// ---- the tile kernel for 16-bit operands whose rows take 16-byte accesses: BM x BN tiles, 64 of k per step, both operands by LDS-DMA in
// the layout they have in memory - k-contiguous rows of 128 bytes, or rows of one k with BM / BN columns, which the transposing LDS
// reads turn into the same fragments - NST stages in a ring: a step's loads are in flight while NST - 1 steps before it are contracted.  Two
// stages where other blocks of the CU hide a load's latency (or the tile fills the LDS), four where a block has its CU to itself:
// 2048 x 2048 x 2048 f16 25 us and 28 with two, 256 x 16384 x 4096 43 and 49, weight gradient of 1048576 x 64 x 64 46 and 57.
//
// LDS swizzle (the DMA writes lane i's 16 bytes at 16 i, so the lane chooses the memory chunk instead): k-contiguous rows keep chunk c of
// row r at c ^ ((r >> 1) & 7), so that the 16 rows a ds_read_b128 group touches lie on 16 different 16-byte slots; rows of one k keep it at
// c ^ ((k & 3) << 2), so that the four k rows of a transposing read lie in four different 64-byte quarters (rows of 64 columns: two of them
// fill the banks, c ^ ((k & 2) << 1)).
//
// The matrix cores bound it: 63 % of their cycles busy at 16384 x 4096 x 4096 (1.2 PFLOP/s bf16; the library's own product 1.55), the LDS 25 %.
// Measured against and dropped: 128 x 256 and 256 x 128 in three stages of 32 at two blocks per CU (4 - 6 % slower: half again the operand
// traffic), 128 x 128 per wave (the accumulators leave no registers), four stages of 32 (2 % slower).
constexpr int BK = 64;
template <int ROWS> __device__ __forceinline__ int k_swizzle(int k) { return ROWS == 64 ? (k & 2) << 1 : (k & 3) << 2; }

// one operand's side of the ring: ROWS tile rows (along i or j) x BK of k, loaded by NWV waves
template <bool KC, int ROWS, int NWV> struct TileLoader {
  static constexpr int NI = ROWS * BK * 2 / 1024 / NWV;        // DMA instructions (1 KiB) per wave and step
  unsigned voff[NI];
  int kchunk[2];                                               // KC: the k chunk a lane fetches in even / odd instructions
  i4v rsrc;
  const unsigned char* base;
  int64_t ld2;
  int cols2;
  __device__ __forceinline__ void init(const void* ptr, int64_t ld, int64_t r0, int64_t rend, int64_t Kd, int wave, int lane) {
    ld2 = ld * 2;
    const int64_t left = rend - r0;
    const int rows = left < ROWS ? (int)left : ROWS;
    if constexpr (KC) {
      static_assert(NI % 2 == 0, "the swizzle of an instruction depends on its parity only");
      base = (const unsigned char*)ptr + r0 * ld2;
      rsrc = make_rsrc(base, (int)((rows - 1) * ld2 + (Kd + 7) / 8 * 16));          // rows behind the operand's end start behind this
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int row = (wave * NI + i) * 8 + (lane >> 3);
        const int ch = (lane & 7) ^ ((row >> 1) & 7);
        kchunk[i & 1] = ch;
        voff[i] = (unsigned)(row * ld2 + ch * 16);
      }
    } else {
      base = (const unsigned char*)ptr + r0 * 2;
      cols2 = ((int)left * 2 + 3) / 4 * 4;                     // (bounds are checked by 4 bytes)
      constexpr int RPI = 512 / ROWS, LPR = 64 / RPI;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int k = (wave * NI + i) * RPI + lane / LPR;
        const int ch = (lane % LPR) ^ k_swizzle<ROWS>(k);
        voff[i] = (unsigned)(k * ld2 + ch * 16);
      }
    }
  }
  // k0 .. k0 + BK (to kend) into the LDS at dst; what is not there reads as zero (the buffer's bounds, or a masked offset)
  __device__ __forceinline__ void issue(unsigned dst, int64_t k0, int64_t kend, int wave) {
    if constexpr (KC) {
      const bool tail = kend - k0 < BK;
      const int rem = (int)(kend - k0);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        unsigned v = voff[i];
        if (tail && kchunk[i & 1] * 8 >= rem) v = 0x80000000u;
        lds_dma16(rsrc, dst + (wave * NI + i) * 1024, v, (int)(k0 * 2));
      }
    } else {
      const int64_t left = kend - k0;
      const int rows = left < BK ? (int)left : BK;
      const i4v r = make_rsrc(base + k0 * ld2, (int)((rows - 1) * ld2 + cols2));
#pragma unroll
      for (int i = 0; i < NI; ++i) lds_dma16(r, dst + (wave * NI + i) * 1024, voff[i], 0);
    }
  }
};
// 32 rows from row0 of an operand's tile, k step ks
template <bool KC, int ROWS> __device__ __forceinline__ u4 tile_frag(const unsigned char* s, int row0, int ks, int lane) {
  if constexpr (KC) {
    const int fr = lane & 31, fh = lane >> 5;
    return *reinterpret_cast<const u4*>(s + (row0 + fr) * (BK * 2) + (((ks * 2 + fh) ^ ((fr >> 1) & 7)) << 4));
  } else {
    const int tg = lane >> 4, tt = lane & 15, tq = tt >> 2, tp = tt & 3;
    const int ch = (row0 >> 3) + 2 * (tg & 1) + (tp >> 1);
    const unsigned char* a = s + (ks * 16 + 8 * (tg >> 1) + tq) * (ROWS * 2) + ((ch ^ k_swizzle<ROWS>(tq)) << 4) + (tp & 1) * 8;
    const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v_ptr)a);
    const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v_ptr)(a + 4 * ROWS * 2));
    const u2 l = __builtin_bit_cast(u2, lo), h = __builtin_bit_cast(u2, hi);
    return u4{l[0], l[1], h[0], h[1]};
  }
}
// eight neighbouring elements of the result (n of them exist; vec: all, and 16-byte accesses fit) through the pass's epilogue; f: the row
// of z (bwd_data), r: of the residual, fetched before
template <int PASS, typename T> __device__ __forceinline__ void epilogue8(const GemmArgs& p, int64_t i, int j, const float* bias, float* v, const float* f,
                                                                          const float* r, int n, bool vec) {
  if constexpr (PASS == SEG_LINEAR_BWD_WEIGHT) {
    float* o = (float*)p.out + i * p.out_ld + j;
    if (vec) store8<float>(o, v);
    else row_store8<float, false>(o, n, v);
  } else {
    if constexpr (PASS == SEG_LINEAR_FWD) {
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] += bias[t];
      if (p.z != nullptr) {
        if (vec) row_store8<T, true>((T*)p.z + i * p.z_ld + j, 8, v);
        else row_store8<T, false>((T*)p.z + i * p.z_ld + j, n, v);
      }
      act8(v, p.act, p.alpha);
    } else if (p.z != nullptr) {
      slope8(v, f, p.act, p.alpha);
    }
    if (p.res != nullptr) {
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] += r[t];
    }
    if (vec) row_store8<T, true>((T*)p.out + i * p.out_ld + j, 8, v);
    else row_store8<T, false>((T*)p.out + i * p.out_ld + j, n, v);
  }
}
template <typename T> struct Row8 {                            // eight elements of a row in their memory format
  typedef T tv __attribute__((ext_vector_type(8)));
  tv v;
  __device__ __forceinline__ void load(const T* p, int n, bool vec) {
    if (vec) v = *reinterpret_cast<const tv*>(p);
    else v = raw_load8<T, false>(p, n);
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int t = 0; t < 8; ++t) f[t] = (float)v[t];
  }
};

// until at most `left` more stages of PER loads each are on their way (the DMA's loads land in order; left < NST)
template <int PER, int NST> __device__ __forceinline__ void wait_stages(int left) {
  if (NST > 3 && left >= 3) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * PER) : "memory");
  else if (NST > 2 && left == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PER) : "memory");
  else if (left == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}
template <int PASS, typename T, int BM, int BN, int WM, int WN, int NST>
__global__ __launch_bounds__(64 * WM * WN, NST == 2 ? 2 : 1) void gemm_tile_kernel(const GemmArgs p) {
  constexpr bool AKC = PASS != SEG_LINEAR_BWD_WEIGHT, BKC = PASS == SEG_LINEAR_FWD;
  constexpr int NWV = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, STAGE = (BM + BN) * BK * 2, SLAB = 32 * 68 * 4;
  static_assert(TN % 2 == 0 && NWV * SLAB <= NST * STAGE && NST <= 4, "the epilogue's slabs take 64 columns and fit the ring");
  __shared__ __align__(1024) unsigned char smem[NST * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // tiles in groups of eight rows of tiles, column by column: the blocks of one XCD share operand panels in both directions
  const int t = xcd_remap(blockIdx.x, p.ti * p.tj);
  const int grp = t / (8 * p.tj), in = t - grp * 8 * p.tj, gh = p.ti - grp * 8 < 8 ? p.ti - grp * 8 : 8;
  const int64_t i0 = (int64_t)(grp * 8 + in % gh) * BM;
  const int j0 = in / gh * BN;
  const int64_t kbeg = blockIdx.y * p.kper, kend = kbeg + p.kper < p.Kd ? kbeg + p.kper : p.Kd;
  const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(lds_byte_ptr)smem);
  TileLoader<AKC, BM, NWV> la;
  TileLoader<BKC, BN, NWV> lb;
  la.init(p.A, p.a_ld, i0, p.I, p.Kd, wave, lane);
  lb.init(p.B, p.b_ld, j0, p.J, p.Kd, wave, lane);
  f16v acc[TM][TN];
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[a][b][q] = 0.f;
  const int wr = (wave / WN) * TM * 32, wc = (wave % WN) * TN * 32;
  // The fragments of a k step are read while the step before is contracted (two register sets); across the ring's barrier the last
  // step of a stage is: the barrier stands in front of its MFMAs, and the next stage's first reads and the DMA that refills this stage
  // are issued there, so that neither latency is waited for.
  u4 af[2][TM], bf[2][TN];
  auto frags = [&](int set, const unsigned char* sa, int ks) {
#pragma unroll
    for (int a = 0; a < TM; ++a) af[set][a] = tile_frag<AKC, BM>(sa, wr + a * 32, ks, lane);
#pragma unroll
    for (int b = 0; b < TN; ++b) bf[set][b] = tile_frag<BKC, BN>(sa + BM * BK * 2, wc + b * 32, ks, lane);
  };
  auto contract = [&](int set) {
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
      for (int b = 0; b < TN; ++b) acc[a][b] = mfma16<T>(af[set][a], bf[set][b], acc[a][b]);
  };
  auto issue = [&](int st, int64_t k) {
    const unsigned d = lds0 + st * STAGE;
    la.issue(d, k, kend, wave);
    lb.issue(d + BM * BK * 2, k, kend, wave);
  };
  const int steps = (int)((kend - kbeg + BK - 1) / BK);
  constexpr int PER = TileLoader<AKC, BM, NWV>::NI + TileLoader<BKC, BN, NWV>::NI;
  const int ahead = steps < NST ? steps : NST;
#pragma unroll
  for (int st = 0; st < NST; ++st)
    if (st < ahead) issue(st, kbeg + st * BK);
  wait_stages<PER, NST>(ahead - 1);
  ring_release_barrier();
  frags(0, smem, 0);
  int64_t knext = kbeg + NST * BK;
  int stage = 0;
  for (int it = 0; it < steps; ++it, knext += BK) {
    const unsigned char* sa = smem + stage * STAGE;
    const int next = stage + 1 < NST ? stage + 1 : 0;
#pragma unroll
    for (int ks = 1; ks < BK / 16; ++ks) {
      frags(ks & 1, sa, ks);
      contract((ks - 1) & 1);
    }
    if (it + 1 < steps) {
      wait_stages<PER, NST>(steps - it - 2 < NST - 2 ? steps - it - 2 : NST - 2);
      ring_release_barrier();                                  // the next stage has landed for every wave, this one has no readers left
      frags(0, smem + next * STAGE, 0);
      if (it + NST < steps) issue(stage, knext);
    }
    contract((BK / 16 - 1) & 1);
    stage = next;
  }
  // Results leave through wave-private slabs of 32 rows x 64 columns in the ring's LDS, so that a store covers whole 128-byte lines:
  // stores straight from the accumulators (32-byte pieces of 32 rows) took 221 us instead of 172 where two tensors are written
  // (16384 x 4096 x 1024, y and z).
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  ring_release_barrier();
  float* slab = reinterpret_cast<float*>(smem + wave * SLAB);
  const int fr = lane & 31, fh = lane >> 5;
  const bool vecio = p.vecio != 0;
  // what the epilogue reads (z of bwd_data, the residual) is fetched a 32 x 64 piece ahead of its use
  constexpr int PIECES = TN / 2 * TM;
  constexpr bool READS = PASS != SEG_LINEAR_BWD_WEIGHT;
  Row8<T> zr[2][4], rr[2][4];
  auto fetch = [&](int u) {
    const int j = j0 + wc + (u / TM) * 64 + (lane & 7) * 8, n = p.J - j;
    const bool vec = vecio && n >= 8;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t i = i0 + wr + (u % TM) * 32 + (lane >> 3) + r * 8;
      if (j < p.J && i < p.I && p.splits == 1) {
        if (PASS == SEG_LINEAR_BWD_DATA && p.z != nullptr) zr[u & 1][r].load((const T*)p.z + i * p.z_ld + j, n, vec);
        if (p.res != nullptr) rr[u & 1][r].load((const T*)p.res + i * p.res_ld + j, n, vec);
      }
    }
  };
  if constexpr (READS) fetch(0);
  float bias[8];
#pragma unroll
  for (int u = 0; u < PIECES; ++u) {
    const int bp = u / TM, a = u % TM;
    const int j = j0 + wc + bp * 64 + (lane & 7) * 8;
    const int n = p.J - j;
    const bool jn = n > 0, vec = vecio && n >= 8;
    if (a == 0) {
#pragma unroll
      for (int q = 0; q < 8; ++q) bias[q] = (PASS == SEG_LINEAR_FWD && p.bias != nullptr && q < n) ? p.bias[j + q] : 0.f;
    }
    if constexpr (READS) {
      if (u + 1 < PIECES) fetch(u + 1);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 16; ++q) slab[((q & 3) + 8 * (q >> 2) + 4 * fh) * 68 + h * 32 + fr] = acc[a][2 * bp + h][q];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t i = i0 + wr + a * 32 + (lane >> 3) + r * 8;
      float v[8], f[8], g[8];
      load8<float>(slab + ((lane >> 3) + r * 8) * 68 + (lane & 7) * 8, v);
      if (i < p.I && jn) {
        if (p.splits > 1) {
          store8<float>(p.part + ((int64_t)blockIdx.y * p.I + i) * p.jp + j, v);         // (whole pieces: jp)
        } else {
          if (PASS == SEG_LINEAR_BWD_DATA && p.z != nullptr) zr[u & 1][r].get(f);
          if (READS && p.res != nullptr) rr[u & 1][r].get(g);
          epilogue8<PASS, T>(p, i, j, bias, v, f, g, n, vec);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- a copy of an operand whose rows no 16-byte access fits, in rows of whole 16 bytes with zeros at their ends
template <typename T>
__global__ __launch_bounds__(TPB) void pack_rows_kernel(const T* x, int64_t ld, int64_t rows, int64_t cols, T* o, int64_t ld8) {
  const int64_t n = rows * (ld8 / 8);
  for (int64_t e = (int64_t)blockIdx.x * TPB + threadIdx.x; e < n; e += (int64_t)gridDim.x * TPB) {
    const int64_t r = e / (ld8 / 8), c = (e - r * (ld8 / 8)) * 8;
    const auto v = raw_load8<T, false>(x + r * ld + c, (int)(cols - c));
    st16(o + r * ld8 + c, __builtin_bit_cast(u4, v));
  }
}

// ---- a few rows against all the weights (forward, up to 64 rows): the weights' bytes and one memory latency bound it, so they go straight
// into the matrix instructions' registers, once, with no LDS in between.  A block owns 16 units; its waves share k in steps of 64 bytes per
// row (lane l: row l % 16, 16 bytes at chunk l / 16), keep four steps' loads in flight and add their sums in the LDS.  MT x 16 rows of x.
// 4 x 4096 x 1024 bf16: 4.2 us (2 TB/s of weights); the tiled kernel with split sums took 12.
template <typename T, int MT, int WK>
__global__ __launch_bounds__(64 * WK) void gemm_rows_kernel(const GemmArgs p) {
  constexpr int EPC = 16 / (int)sizeof(T), STEP = 4 * EPC, UN = MT <= 2 ? 4 : 2;
  __shared__ float red[WK][MT * 16][17];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, ch = lane >> 4, j0 = blockIdx.x * 16, M = (int)p.I;
  const T* w = (const T*)p.B + (int64_t)(j0 + r < p.J ? j0 + r : p.J - 1) * p.b_ld + ch * EPC;     // (rows that are not there: results dropped)
  const T* x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) x[m] = (const T*)p.A + (int64_t)(m * 16 + r < M ? m * 16 + r : M - 1) * p.a_ld + ch * EPC;
  f4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = f4{0.f, 0.f, 0.f, 0.f};
  const u4 zero = {0u, 0u, 0u, 0u};
  const int K = (int)p.Kd, steps = (K + STEP - 1) / STEP;
  for (int s0 = wave; s0 < steps; s0 += WK * UN) {
    u4 wv[UN], xv[MT][UN];
#pragma unroll
    for (int q = 0; q < UN; ++q) {
      const int k = (s0 + q * WK) * STEP;
      const bool in = k + ch * EPC < K;
      wv[q] = in ? ld16(w + k) : zero;
#pragma unroll
      for (int m = 0; m < MT; ++m) xv[m][q] = in ? ld16(x[m] + k) : zero;
    }
#pragma unroll
    for (int q = 0; q < UN; ++q)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if constexpr (std::is_same<T, float>::value) {
          const f4 a = __builtin_bit_cast(f4, wv[q]), b = __builtin_bit_cast(f4, xv[m][q]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], acc[m], 0, 0, 0);
        } else if constexpr (std::is_same<T, half_t>::value) {
          acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, wv[q]), __builtin_bit_cast(h8, xv[m][q]), acc[m], 0, 0, 0);
        } else {
          acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, wv[q]), __builtin_bit_cast(b8, xv[m][q]), acc[m], 0, 0, 0);
        }
      }
  }
  // lane: row of x l % 16, units 4 (l / 16) + 0 .. 3
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[wave][m * 16 + r][ch * 4 + e] = acc[m][e];
  __syncthreads();
  for (int o = tid; o < MT * 256; o += 64 * WK) {
    const int i = o >> 4, j = o & 15;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < WK; ++k) v += red[k][i][j];
    if (i < M && j0 + j < p.J) epilogue1<SEG_LINEAR_FWD, T>(p, i, j0 + j, v);
  }
}

// the split ranges of k added in a fixed order, then the epilogue: R threads per element, thread r adds ranges r, r + R, ..
template <int PASS, typename T, int R>
__global__ __launch_bounds__(TPB) void gemm_join_kernel(const GemmArgs p) {
  constexpr int EPB = TPB / R;
  __shared__ float sh[R > 1 ? TPB : 1];
  const int r = threadIdx.x / EPB, c = threadIdx.x % EPB;
  const int64_t n = p.I * p.J, all = n + (p.db != nullptr ? p.I : 0);
  for (int64_t e0 = (int64_t)blockIdx.x * EPB; e0 < all; e0 += (int64_t)gridDim.x * EPB) {
    const int64_t e = e0 + c, i = e / p.J;
    const int j = (int)(e - i * p.J);
    const bool bias = PASS == SEG_LINEAR_BWD_WEIGHT && e >= n;
    float v = 0.f;
    if (e < all) {
      const float* q = bias ? p.part_db + (e - n) : p.part + i * p.jp + j;
      const int64_t ld = bias ? p.I : p.I * p.jp;
#pragma unroll 4
      for (int s = r; s < p.splits; s += R) v += q[s * ld];
    }
    if constexpr (R > 1) {
      __syncthreads();
      sh[threadIdx.x] = v;
      __syncthreads();
      if (r == 0) {
#pragma unroll
        for (int k = 1; k < R; ++k) v += sh[k * EPB + c];
      }
    }
    if (r == 0 && e < all) {
      if (bias) p.db[e - n] = v;
      else epilogue1<PASS, T>(p, i, j, v);
    }
  }
}

// ---- the bias gradient where gemm_any_kernel does not carry it (no weight gradient wanted; the tile kernels, whose registers the extra
// product overflows: 133 -> 213 us): column sums of dy, rows in ranges of blocks (part[range][N], added up in order by colsum_parts_kernel)
template <typename T, bool VEC>
__global__ __launch_bounds__(TPB) void colsum_rows_kernel(const T* dy, int64_t ld, int64_t rows, int cols, int64_t per, float* part) {
  const int l = threadIdx.x & 31, r = threadIdx.x >> 5, c = (blockIdx.x * 32 + l) * 8;
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = 0.f;
  const int64_t beg = blockIdx.y * per, end = beg + per < rows ? beg + per : rows;
  if (c < cols)
    for (int64_t i = beg + r; i < end; i += 8) {
      float f[8];
      row_load8<T, VEC>(dy + i * ld + c, cols - c, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += f[j];
    }
  __shared__ float sh[8][32][9];
#pragma unroll
  for (int j = 0; j < 8; ++j) sh[r][l][j] = s[j];
  __syncthreads();
  const int ol = threadIdx.x >> 3, oj = threadIdx.x & 7, oc = (blockIdx.x * 32 + ol) * 8 + oj;
  if (oc < cols) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) v += sh[q][ol][oj];
    part[(int64_t)blockIdx.y * cols + oc] = v;
  }
}
struct ColsumPlan { int64_t per, parts; };
inline ColsumPlan colsum_plan(int64_t rows, int cols) {
  const int64_t cb = (cols + 255) / 256, want = (1024 + cb - 1) / cb;
  int64_t per = (rows + want - 1) / want;
  per = (per + 31) / 32 * 32;
  return {per, (rows + per - 1) / per};
}

// ---- plans
enum { TILE_ANY = 0, TILE_128 = 1, TILE_256 = 2, FEW_ROWS = 3, TILE_NARROW = 4 };
inline bool tiled(int kind) { return kind == TILE_128 || kind == TILE_256 || kind == TILE_NARROW; }
struct GemmPlan { int kind; int ti, tj, splits; int64_t kper; };
inline GemmPlan gemm_plan(int64_t I, int J, int64_t Kd, int dtype, bool dma) {
  GemmPlan g;
  // 128 x 64 for up to 64 columns (1048576 x 64 x 64, f16: 69 us, 157 with 128 x 128, the bytes' floor 55); 256 x 256 where such tiles
  // (with k split in ranges of 4096) fill three quarters of the 256 CUs: 233 us against 250 with 128 x 128
  // for 16384 x 4096 x 1024 (f16, GELU, pre-activation kept), 375 against 402 for the backward pass of 16384 x 1024 x 4096 (bf16)
  const int64_t t256 = ((I + 255) / 256) * ((J + 255) / 256);
  g.kind = !dma ? TILE_ANY : J <= 64 ? TILE_NARROW : t256 * (Kd > 4096 * 64 ? 64 : (Kd + 4095) / 4096) >= 192 ? TILE_256 : TILE_128;
  const int si = g.kind == TILE_ANY ? 64 : g.kind == TILE_256 ? 256 : 128, sj = g.kind == TILE_NARROW ? 64 : si;
  g.ti = (int)((I + si - 1) / si);
  g.tj = (J + sj - 1) / sj;
  const int64_t tiles = (int64_t)g.ti * g.tj, room = g.kind == TILE_ANY ? 1024 : 256, most = Kd / 512;
  // fewer tiles than the card has room for: k is split, down to 512 of it per block, and a second launch joins the parts (1111 x 333 x 700,
  // f16: 14 us in one launch, 16 in two).  Half a microsecond per step of 64 and block against 5 us for the second launch and 8 bytes
  // per element and range written and read again (at 4 TB/s): as many ranges as level the two.  Against filling every CU twice
  // (f16): 2048 x 2048 x 2048 42 -> 25 us, 1024 x 1024 x 1024 18.6 -> 14.3, 128 x 4096 x 4096 21.1 -> 19.2
  int64_t s = tiles * 2 > room || tiles == 0 ? 1 : room / tiles;
  if (s > most) s = most;
  if (s > 256) s = 256;
  if (g.kind == TILE_128 || g.kind == TILE_NARROW) {
    const double us = 0.55 * (double)Kd / 64, join = (double)I * J * 2e-6;
    const int64_t level = (int64_t)(sqrt(us / join) + 0.5);
    if (s > level) s = level;
    if (s > 1 && us / s + 5 + s * join > us) s = 1;
  }
  if (s < 1) s = 1;
  const int64_t step = g.kind != TILE_ANY ? 64 : dtype == SEG_DT_F32 ? 16 : 32;
  g.kper = ((Kd + s - 1) / s + step - 1) / step * step;
  g.splits = g.kper > 0 ? (int)((Kd + g.kper - 1) / g.kper) : 1;
  if (g.splits < 1) g.splits = 1;
  return g;
}

struct Extents { int64_t I, Kd; int J; };
inline Extents extents(const seg_linear_args& a, int pass) {
  if (pass == SEG_LINEAR_BWD_WEIGHT) return {a.N, a.M, a.K};
  return {a.M, a.K, a.N};
}

// What the LDS-DMA tile kernels take of a pass: 16-bit operands in 16-byte rows (k-contiguous ones also a whole number of 8 inputs),
// offsets inside a tile below 2 GiB.  A large product whose operands do not fit is worth a packed copy of them (16384 x 4095 x 4095 f16:
// 2012 us without, 553 with; its gradients 2439 and 550, 2838 and 598).  dma: 0 no, 1 as they are, 2 with copies (a, b: which)
struct Operand { const void* p; int64_t ld, rows, cols; bool kc; };
struct DmaPlan { int dma; bool a, b; int64_t a_elems, b_elems; };
inline Operand operand_a(const seg_linear_args& a, int pass) {
  if (pass == SEG_LINEAR_BWD_WEIGHT) return {a.dy, a.dy_ld, a.M, a.N, false};
  return {a.x, a.x_ld, a.M, a.K, true};
}
inline Operand operand_b(const seg_linear_args& a, int pass) {
  if (pass == SEG_LINEAR_BWD_WEIGHT) return {a.x, a.x_ld, a.M, a.K, false};
  return pass == SEG_LINEAR_FWD ? Operand{a.w, a.w_ld, a.N, a.K, true} : Operand{a.w, a.w_ld, a.K, a.N, false};
}
inline DmaPlan dma_plan(const seg_linear_args& a, int pass) {
  DmaPlan d = {0, false, false, 0, 0};
  const Extents e = extents(a, pass);
  // (tiles far larger than the result waste the matrix cores)
  if (a.dtype == SEG_DT_F32 || e.I < 64 || e.J < 48 || e.Kd < 1) return d;
  const Operand A = operand_a(a, pass), B = operand_b(a, pass);
  if (A.ld > (1 << 21) || B.ld > (1 << 21) || A.cols > (1 << 21) || B.cols > (1 << 21)) return d;
  auto fits = [](const Operand& o) { return aligned16(o.p) && o.ld % 8 == 0 && (!o.kc || o.cols % 8 == 0); };
  d.a = !fits(A);
  d.b = !fits(B);
  if (!d.a && !d.b) { d.dma = 1; return d; }
  // A copy pays where enough products share it, sooner for operands along i / j, which the other kernel transposes at a quarter of the
  // tile kernel's pace.  Without and with (f16): forward 8192 x 519 x 523 24 and 28 us, 16384 x 1001 x 1003 103 and 59, 16384 x 63 x 4001
  // 43 and 77; data gradients 2000 x 1001 x 777 37 and 25, 500 x 301 x 1203 14 and 17; weight gradients 46 and 27, 18 and 19
  const double products = (double)e.I * e.J * e.Kd;
  if (pass == SEG_LINEAR_FWD ? e.I < 256 || products < 4294967296.0 : products < 1073741824.0) return d;
  if (e.J < 256) return d;
  d.dma = 2;
  auto elems = [](const Operand& o) { return o.rows * ((o.cols + 7) / 8 * 8); };
  d.a_elems = d.a ? elems(A) : 0;
  d.b_elems = d.b ? elems(B) : 0;
  return d;
}
// Up to 64 rows forward, every row of both operands in 16-byte pieces, go to gemm_rows_kernel where one launch gains more than its blocks
// lose: a block walks all of k (16 rows f16: 1.7 us per 1024 of it, four times that for 64 rows) and reads all of x again.  Against the
// kernels with split sums (f16): 16 x 4096 x 4096 10 us and 14, 32 x 1024 x 4096 13 and 14, 64 x 4096 x 1024 10 and 13.4; beyond the two
// limits 64 x 64 x 65536 276 and 14, 32 x 256 x 16384 44 and 14, 64 x 16384 x 4096 74 and 31, 32 x 8192 x 8192 45 and 27.  fp32 has
// no faster way for many units: 1 x 16384 x 4096 57 and 89, 16 x 4096 x 16384 69 and 96 (up to 2^26: blocks of 512 threads own 16 units,
// and an axis of a grid takes fewer than 2^32 threads).
inline bool rows_ok(const seg_linear_args& a, int pass) {
  if (pass != SEG_LINEAR_FWD || a.M > 64) return false;
  const int64_t u = a.dtype == SEG_DT_F32 ? 4 : 8;
  if (!(aligned16(a.x) && aligned16(a.w) && a.x_ld % u == 0 && a.w_ld % u == 0 && a.K % u == 0)) return false;
  const int64_t groups = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
  if (a.dtype == SEG_DT_F32 && groups == 1 && a.N >= 2048 && a.N <= 1 << 26) return true;
  return groups * a.K * (int64_t)dt_size(a.dtype) <= 16384 && groups * a.K * a.N <= (int64_t)1 << 25;
}
inline GemmPlan plan_of(const seg_linear_args& a, int pass) {
  const Extents e = extents(a, pass);
  if (rows_ok(a, pass)) return {FEW_ROWS, 1, (e.J + 15) / 16, 1, e.Kd};
  return gemm_plan(e.I, e.J, e.Kd, a.dtype, dma_plan(a, pass).dma != 0);
}

// bwd_weight: whether db is part of the product's launch, and the floats of the product's split sums (whole 16 bytes)
inline bool sums_ride(const seg_linear_args& a) { return a.dw != nullptr && plan_of(a, SEG_LINEAR_BWD_WEIGHT).kind == TILE_ANY; }
inline int64_t weight_parts(const seg_linear_args& a) {
  const GemmPlan g = plan_of(a, SEG_LINEAR_BWD_WEIGHT);
  if (a.dw == nullptr || g.splits <= 1) return 0;
  return ((int64_t)g.splits * a.N * ((a.K + 7) / 8 * 8 + (a.db != nullptr && g.kind == TILE_ANY ? 1 : 0)) + 3) / 4 * 4;
}

inline int64_t gemm_parts(const seg_linear_args& a, int pass) {            // floats in front of the packed copies
  if (pass == SEG_LINEAR_BWD_WEIGHT) return weight_parts(a) + (a.db != nullptr && !sums_ride(a) ? (colsum_plan(a.M, a.N).parts * a.N + 3) / 4 * 4 : 0);
  const GemmPlan g = plan_of(a, pass);
  const Extents e = extents(a, pass);
  return g.splits > 1 ? (int64_t)g.splits * e.I * ((e.J + 7) / 8 * 8) : 0;
}
inline int64_t pack_offset(const seg_linear_args& a, int pass) { return (gemm_parts(a, pass) * 4 + 15) / 16 * 16; }
inline int64_t gemm_workspace(const seg_linear_args& a, int pass) {
  const bool product = pass != SEG_LINEAR_BWD_WEIGHT || a.dw != nullptr;
  const GemmPlan g = plan_of(a, pass);
  const DmaPlan d = product && tiled(g.kind) ? dma_plan(a, pass) : DmaPlan{0, false, false, 0, 0};
  return d.dma == 2 ? pack_offset(a, pass) + (d.a_elems + d.b_elems) * 2 : gemm_parts(a, pass) * 4;
}

template <int PASS>
int run_gemm(const seg_linear_args& a, GemmArgs& p, hipStream_t st) {
  const Extents e = extents(a, PASS);
  const GemmPlan g = plan_of(a, PASS);
  p.I = e.I; p.J = e.J; p.Kd = e.Kd;
  p.ti = g.ti; p.tj = g.tj; p.splits = g.splits; p.kper = g.kper;
  p.part = (float*)a.workspace;
  p.jp = (e.J + 7) / 8 * 8;
  p.part_db = p.part + (int64_t)g.splits * e.I * p.jp;
  p.act = a.act; p.alpha = a.alpha;
  p.vecio = PASS == SEG_LINEAR_BWD_WEIGHT ? vec_ok(p.out, p.out_ld, 0, SEG_DT_F32)
                                          : vec_ok(p.out, p.out_ld, 0, a.dtype) && vec_ok(p.z, p.z_ld, 0, a.dtype) && vec_ok(p.res, p.res_ld, 0, a.dtype);
  const DmaPlan d = tiled(g.kind) ? dma_plan(a, PASS) : DmaPlan{0, false, false, 0, 0};
  if (d.dma == 2) {
    uint16_t* to = (uint16_t*)((char*)a.workspace + pack_offset(a, PASS));
    auto pack = [&](const Operand& o, uint16_t* dst) {         // (bit copies: either 16-bit type)
      const int64_t ld8 = (o.cols + 7) / 8 * 8, blocks = (o.rows * (ld8 / 8) + TPB - 1) / TPB;
      hipLaunchKernelGGL((pack_rows_kernel<half_t>), dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(TPB), 0, st, (const half_t*)o.p, o.ld, o.rows, o.cols, (half_t*)dst, ld8);
      return ld8;
    };
    if (d.a) { p.a_ld = pack(operand_a(a, PASS), to); p.A = to; }
    if (d.b) { p.b_ld = pack(operand_b(a, PASS), to + d.a_elems); p.B = to + d.a_elems; }
  }
  const dim3 grid((unsigned)(g.ti * g.tj), (unsigned)g.splits);
  const bool vec = vec_ok(p.A, p.a_ld, 0, a.dtype) && vec_ok(p.B, p.b_ld, 0, a.dtype);
  seq_dispatch_dtype(a.dtype, [&](auto* tp) {
    typedef typename std::remove_pointer<decltype(tp)>::type T;
    if (g.kind == FEW_ROWS) {
      if constexpr (PASS == SEG_LINEAR_FWD) {
        // 16 waves per block where the blocks alone do not fill the card
        const bool deep = g.tj < 256;
#define ROWS_CASE(m, wk) hipLaunchKernelGGL((gemm_rows_kernel<T, m, wk>), dim3((unsigned)g.tj), dim3(64 * wk), 0, st, p)
        if (p.I <= 16) { if (deep) ROWS_CASE(1, 16); else ROWS_CASE(1, 8); }
        else if (p.I <= 32) { if (deep) ROWS_CASE(2, 16); else ROWS_CASE(2, 8); }
        else ROWS_CASE(4, 8);
#undef ROWS_CASE
      }
    } else if (g.kind != TILE_ANY) {
      if constexpr (!std::is_same<T, float>::value) {
        // a block that has its CU to itself keeps three steps on their way instead of one
        const bool deep = (int64_t)g.ti * g.tj * g.splits <= 256;
#define TILE_CASE(bm, bn, wm, wn, nst) hipLaunchKernelGGL((gemm_tile_kernel<PASS, T, bm, bn, wm, wn, nst>), grid, dim3(64 * wm * wn), 0, st, p)
        if (g.kind == TILE_256) TILE_CASE(256, 256, 2, 4, 2);
        else if (g.kind == TILE_NARROW) { if (deep) TILE_CASE(128, 64, 2, 1, 4); else TILE_CASE(128, 64, 2, 1, 2); }
        else { if (deep) TILE_CASE(128, 128, 2, 2, 4); else TILE_CASE(128, 128, 2, 2, 2); }
#undef TILE_CASE
      }
    } else if (vec) hipLaunchKernelGGL((gemm_any_kernel<PASS, T, true>), grid, dim3(TPB), 0, st, p);
    else hipLaunchKernelGGL((gemm_any_kernel<PASS, T, false>), grid, dim3(TPB), 0, st, p);
    if (g.splits > 1) {
      const bool wide = g.splits >= 32;
      const int64_t per = wide ? TPB / 8 : TPB, blocks = (p.I * (p.J + (p.db != nullptr ? 1 : 0)) + per - 1) / per;
      const dim3 jg((unsigned)(blocks < 4096 ? blocks : 4096));
      if (wide) hipLaunchKernelGGL((gemm_join_kernel<PASS, T, 8>), jg, dim3(TPB), 0, st, p);
      else hipLaunchKernelGGL((gemm_join_kernel<PASS, T, 1>), jg, dim3(TPB), 0, st, p);
    }
  });
  return SEG_OK;
}

int check_linear(const seg_linear_args* a, int pass, const char* name) {
  SEG_CHECK_ARG(a != nullptr, "%s: args is NULL", name);
  SEG_CHECK_ARG(a->dtype >= SEG_DT_F16 && a->dtype <= SEG_DT_F32, "%s: dtype %d", name, a->dtype);
  SEG_CHECK_ARG(a->M >= 0 && a->N > 0 && a->K > 0, "%s: M %lld, N %d, K %d", name, (long long)a->M, a->N, a->K);
  SEG_CHECK_ARG(a->act == SEG_ACT_NONE || a->act == SEG_ACT_RELU || a->act == SEG_ACT_LEAKY || a->act == SEG_ACT_SIGMOID || a->act == SEG_ACT_SILU || a->act == SEG_ACT_GELU,
                "%s: activation %d", name, a->act);
  const Extents e = extents(*a, pass);
  SEG_CHECK_ARG(((e.I + 63) / 64) * ((int64_t)(e.J + 63) / 64) < (int64_t)1 << 24, "%s: result of %lld x %d is too large for one call", name, (long long)e.I, e.J);
  SEG_CHECK_ARG(aligned16(a->workspace), "%s: workspace needs 16-byte alignment", name);
  SEG_CHECK_ARG(a->M == 0 || a->workspace != nullptr || gemm_workspace(*a, pass) == 0, "%s: workspace is NULL (%lld bytes are needed)", name,
                (long long)gemm_workspace(*a, pass));
  return SEG_OK;
}

}  // namespace

extern "C" int64_t seg_linear_workspace_bytes(const seg_linear_args* a, int32_t pass) {
  if (a == nullptr || a->M <= 0 || a->N <= 0 || a->K <= 0 || pass < SEG_LINEAR_FWD || pass > SEG_LINEAR_BWD_WEIGHT) return 0;
  return gemm_workspace(*a, pass);
}

extern "C" int seg_linear_fwd(const seg_linear_args* a, seg_stream_t stream) {
  if (int rc = check_linear(a, SEG_LINEAR_FWD, "linear_fwd")) return rc;
  if (a->M == 0) return SEG_OK;
  SEG_CHECK_ARG(a->x != nullptr && a->w != nullptr && a->y != nullptr, "linear_fwd: x / w / y is NULL");
  SEG_CHECK_ARG((a->M == 1 || a->x_ld >= a->K) && (a->N == 1 || a->w_ld >= a->K), "linear_fwd: row strides below K = %d", a->K);
  SEG_CHECK_ARG(a->M == 1 || (a->y_ld >= a->N && (a->z == nullptr || a->z_ld >= a->N) && (a->residual == nullptr || a->residual_ld >= 0)),
                "linear_fwd: row strides below N = %d", a->N);
  SEG_CHECK_ARG(a->M == 1 || a->residual != a->y || a->residual_ld == a->y_ld, "linear_fwd: y in place of the residual has another row stride");
  GemmArgs p = {};
  p.A = a->x; p.a_ld = a->x_ld; p.B = a->w; p.b_ld = a->w_ld;
  p.bias = a->bias; p.res = a->residual; p.res_ld = a->residual_ld; p.z = a->z; p.z_ld = a->z_ld; p.out = a->y; p.out_ld = a->y_ld;
  run_gemm<SEG_LINEAR_FWD>(*a, p, (hipStream_t)stream);
  SEG_CHECK_LAUNCH("linear_fwd");
  return SEG_OK;
}

extern "C" int seg_linear_bwd_data(const seg_linear_args* a, seg_stream_t stream) {
  if (int rc = check_linear(a, SEG_LINEAR_BWD_DATA, "linear_bwd_data")) return rc;
  SEG_CHECK_ARG(a->bias == nullptr, "linear_bwd_data: takes no bias");
  if (a->M == 0) return SEG_OK;
  SEG_CHECK_ARG(a->x != nullptr && a->w != nullptr && a->y != nullptr, "linear_bwd_data: x / w / y is NULL");
  SEG_CHECK_ARG((a->M == 1 || a->x_ld >= a->K) && (a->K == 1 || a->w_ld >= a->N), "linear_bwd_data: row strides of x below %d or of w below %d", a->K, a->N);
  SEG_CHECK_ARG(a->M == 1 || (a->y_ld >= a->N && (a->z == nullptr || a->z_ld >= a->N) && (a->residual == nullptr || a->residual_ld >= 0)),
                "linear_bwd_data: row strides below N = %d", a->N);
  SEG_CHECK_ARG(a->M == 1 || a->residual != a->y || a->residual_ld == a->y_ld, "linear_bwd_data: y in place of the residual has another row stride");
  GemmArgs p = {};
  p.A = a->x; p.a_ld = a->x_ld; p.B = a->w; p.b_ld = a->w_ld;
  p.res = a->residual; p.res_ld = a->residual_ld; p.z = a->z; p.z_ld = a->z_ld; p.out = a->y; p.out_ld = a->y_ld;
  run_gemm<SEG_LINEAR_BWD_DATA>(*a, p, (hipStream_t)stream);
  SEG_CHECK_LAUNCH("linear_bwd_data");
  return SEG_OK;
}

extern "C" int seg_linear_bwd_weight(const seg_linear_args* a, seg_stream_t stream) {
  if (int rc = check_linear(a, SEG_LINEAR_BWD_WEIGHT, "linear_bwd_weight")) return rc;
  SEG_CHECK_ARG(a->M == 0 || (a->dy != nullptr && (a->dw == nullptr || a->x != nullptr)), "linear_bwd_weight: dy / x is NULL");
  SEG_CHECK_ARG(a->M <= 1 || (a->dy_ld >= a->N && (a->dw == nullptr || a->x_ld >= a->K)), "linear_bwd_weight: row strides below N = %d / K = %d", a->N, a->K);
  SEG_CHECK_ARG(a->dw == nullptr || a->N == 1 || a->dw_ld >= a->K, "linear_bwd_weight: dw_ld below K = %d", a->K);
  hipStream_t st = (hipStream_t)stream;
  if (a->dw != nullptr) {
    GemmArgs p = {};
    p.A = a->dy; p.a_ld = a->dy_ld; p.B = a->x; p.b_ld = a->x_ld; p.out = a->dw; p.out_ld = a->dw_ld; p.db = sums_ride(*a) ? a->db : nullptr;
    run_gemm<SEG_LINEAR_BWD_WEIGHT>(*a, p, st);       // (M = 0: an empty sum, zeros are stored)
  }
  if (a->db != nullptr && !sums_ride(*a)) {
    float* part = (float*)a->workspace + weight_parts(*a);
    const ColsumPlan c = a->M > 0 ? colsum_plan(a->M, a->N) : ColsumPlan{0, 0};
    if (a->M > 0)
      seq_dispatch_dtype(a->dtype, [&](auto* tp) {
        typedef typename std::remove_pointer<decltype(tp)>::type T;
        const dim3 grid((a->N + 255) / 256, (unsigned)c.parts);
        if (a->N % 8 == 0 && vec_ok(a->dy, a->dy_ld, 0, a->dtype))
          hipLaunchKernelGGL((colsum_rows_kernel<T, true>), grid, dim3(TPB), 0, st, (const T*)a->dy, a->dy_ld, a->M, a->N, c.per, part);
        else
          hipLaunchKernelGGL((colsum_rows_kernel<T, false>), grid, dim3(TPB), 0, st, (const T*)a->dy, a->dy_ld, a->M, a->N, c.per, part);
      });
    launch_colsum_pair(part, c.parts, a->N, a->N, a->db, 0, nullptr, st);
  }
  SEG_CHECK_LAUNCH("linear_bwd_weight");
  return SEG_OK;
}

namespace {
template <typename T, bool VEC>
__global__ __launch_bounds__(TPB) void act_bwd_kernel(const T* dy, int64_t dy_ld, const T* z, int64_t z_ld, T* dx, int64_t dx_ld, int64_t rows, int C,
                                                      int act, float alpha) {
  const int chunks = (int)(((int64_t)C + 7) / 8);
  const int64_t n = rows * chunks;
  for (int64_t e = (int64_t)blockIdx.x * TPB + threadIdx.x; e < n; e += (int64_t)gridDim.x * TPB) {
    const int64_t r = e / chunks;
    const int c = (int)(e - r * chunks) * 8;
    float d[8], v[8];
    row_load8<T, VEC>(dy + r * dy_ld + c, C - c, d);
    row_load8<T, VEC>(z + r * z_ld + c, C - c, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] *= seq_act_slope(v[j], act, alpha);
    row_store8<T, VEC>(dx + r * dx_ld + c, C - c, d);
  }
}
}  // namespace

extern "C" int seg_linear_act_bwd(const void* dy, int64_t dy_ld, const void* z, int64_t z_ld, void* dx, int64_t dx_ld, int64_t rows, int32_t C,
                                  int32_t dtype, int32_t act, float alpha, seg_stream_t stream) {
  SEG_CHECK_ARG(dtype >= SEG_DT_F16 && dtype <= SEG_DT_F32, "linear_act_bwd: dtype %d", dtype);
  SEG_CHECK_ARG(rows >= 0 && C > 0, "linear_act_bwd: rows %lld, C %d", (long long)rows, C);
  SEG_CHECK_ARG(act == SEG_ACT_NONE || act == SEG_ACT_RELU || act == SEG_ACT_LEAKY || act == SEG_ACT_SIGMOID || act == SEG_ACT_SILU || act == SEG_ACT_GELU,
                "linear_act_bwd: activation %d", act);
  if (rows == 0) return SEG_OK;
  SEG_CHECK_ARG(dy != nullptr && z != nullptr && dx != nullptr, "linear_act_bwd: dy / z / dx is NULL");
  SEG_CHECK_ARG(rows == 1 || (dy_ld >= C && z_ld >= C && dx_ld >= C), "linear_act_bwd: row strides below the %d channels", C);
  SEG_CHECK_ARG(rows == 1 || dx != dy || dx_ld == dy_ld, "linear_act_bwd: dx in place of dy has another row stride");
  seq_dispatch_dtype(dtype, [&](auto* tp) {
    typedef typename std::remove_pointer<decltype(tp)>::type T;
    const int64_t blocks = (rows * (((int64_t)C + 7) / 8) + TPB - 1) / TPB;
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
    if (C % 8 == 0 && vec_ok(dy, dy_ld, 0, dtype) && vec_ok(z, z_ld, 0, dtype) && vec_ok(dx, dx_ld, 0, dtype))
      hipLaunchKernelGGL((act_bwd_kernel<T, true>), grid, dim3(TPB), 0, (hipStream_t)stream, (const T*)dy, dy_ld, (const T*)z, z_ld, (T*)dx, dx_ld, rows, C, act, alpha);
    else
      hipLaunchKernelGGL((act_bwd_kernel<T, false>), grid, dim3(TPB), 0, (hipStream_t)stream, (const T*)dy, dy_ld, (const T*)z, z_ld, (T*)dx, dx_ld, rows, C, act, alpha);
  });
  SEG_CHECK_LAUNCH("linear_act_bwd");
  return SEG_OK;
}
