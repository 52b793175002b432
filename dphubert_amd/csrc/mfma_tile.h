// Tile products of byte rows for the matrix cores: C[m][n] = sum_k A[m][k] B[n][k], both operands k-contiguous, of
// 8-bit integers (32-bit integer sums) or fp16 (fp32 sums).  The two types share everything but the instruction:
// v_mfma_i32_16x16x64_i8 and v_mfma_f32_16x16x32_f16 both take 16 bytes of a row per lane and run at 16 cycles, so a
// 128-byte step along k is 128 integers or 64 fp16 with the same staging, LDS image and fragment reads.
//
// LDS image of an operand step: rows of 128 bytes, 16-byte chunk p of row r holds the k-chunk p ^ ((r >> 1) & 7) (no
// bank conflict for the 16-lane groups of ds_read_b128); the swizzle is applied to the source address, since an LDS
// DMA writes its 1 KB in lane order.
//
// F16T: fp16 operands that lie the other way round, sum_k A[k][m] B[k][n], so that a Gram matrix needs no transposed
// copy: a step is 64 rows of k, the image [64][R] (R = 64 or 128 of the operand's columns), and the fragments come out
// of it by the hardware's transposing read (ds_read_b64_tr_b16, two a fragment).
#pragma once
#include "gemm_core.h"

#include <type_traits>

namespace dph {
namespace {
namespace mt {

typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;

// 16 bytes at any alignment of the element: one access, which the hardware takes
__device__ __forceinline__ uint4 ld16(const void* p) {
  uint4 r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
__device__ __forceinline__ void st16(void* p, uint4 r) { __builtin_memcpy(p, &r, 16); }

struct I8 {
  static constexpr bool TR = false;
  typedef i32x4_t acc_t;
  static constexpr int ESIZE = 1;
  static __device__ __forceinline__ acc_t mfma(i32x4_t a, i32x4_t b, acc_t c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
};
struct F16 {
  static constexpr bool TR = false;
  typedef f32x4_t acc_t;
  static constexpr int ESIZE = 2;
  static __device__ __forceinline__ acc_t mfma(i32x4_t a, i32x4_t b, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  }
};

struct F16T : F16 {
  static constexpr bool TR = true;
};

// One operand: rows of ld bytes, `rows` of them; ld and the base are multiples of 16.  F16T: `rows` columns (a multiple of
// 8) of k-rows ld bytes apart
struct Rows {
  const char* p;
  int64_t ld;
  int32_t rows;
};

// the transposed image [64][R]: 16-byte chunk c of k-row r stands at c ^ swz(r), which puts the 8 k-rows x 2 chunks of a
// half-wave's transposing read on different banks
template <int R>
__device__ __forceinline__ int tr_swz(int r) {
  return (2 * ((r >> 1) & 1) + 4 * ((r >> 3) & 1) + 8 * (r & 1)) & (R / 8 - 1);
}
// where the fragment of columns c0 .. c0 + 15 (c0 a multiple of 16) starts for a lane; substep s is 64 R bytes further
template <int R>
__device__ __forceinline__ int tr_off(int c0, int lane) {
  const int i = lane & 15, q = i >> 2, p = i & 3, k0 = 8 * (lane >> 4) + q, c = (c0 >> 3) + (p >> 1);
  return k0 * (2 * R) + ((c ^ tr_swz<R>(k0)) << 4) + ((p & 1) << 3);
}
// Both substeps' fragments of N column groups (c0, c0 + 16, ...), read and waited for.  Written as one block each: to the
// compiler the builtin of this read may alias every LDS DMA in flight, and it waits for all of them before it, which leaves
// nothing in flight across a step (the Gram matrices of 24 matrices of 1024 x 4096: 151 us with the builtin, 134 so; of one
// of 768 x 768 11 and 8.  Two workgroups a CU hide it: 45 and 47 us for 48 of 768 x 768)
template <int R, int N>
__device__ __forceinline__ void tr_frags(const char* img, int c0, int lane, i32x4_t (&f)[N][2]) {
  typedef __attribute__((ext_vector_type(2))) int i32x2_t;
  static_assert(N == 1 || N == 2 || N == 4, "column groups of a block");
  constexpr int O1 = 8 * R, O2 = 64 * R, O3 = 72 * R;
  uint32_t a[N];
  i32x2_t v[N][4];
#pragma unroll
  for (int i = 0; i < N; ++i)
    a[i] = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)img + (uint32_t)tr_off<R>(c0 + 16 * i, lane);
#define DPH_TR4(d0, d1, d2, d3, s)                                                                        \
  "ds_read_b64_tr_b16 %" d0 ", %" s "\n\tds_read_b64_tr_b16 %" d1 ", %" s " offset:%c[o1]\n\t"            \
  "ds_read_b64_tr_b16 %" d2 ", %" s " offset:%c[o2]\n\tds_read_b64_tr_b16 %" d3 ", %" s " offset:%c[o3]\n\t"
#define DPH_TRO(i) "=&v"(v[i][0]), "=&v"(v[i][1]), "=&v"(v[i][2]), "=&v"(v[i][3])
  if constexpr (N == 1)
    asm volatile(DPH_TR4("0", "1", "2", "3", "4") "s_waitcnt lgkmcnt(0)"
                 : DPH_TRO(0)
                 : "v"(a[0]), [o1] "i"(O1), [o2] "i"(O2), [o3] "i"(O3)
                 : "memory");
  else if constexpr (N == 2)
    asm volatile(DPH_TR4("0", "1", "2", "3", "8") DPH_TR4("4", "5", "6", "7", "9") "s_waitcnt lgkmcnt(0)"
                 : DPH_TRO(0), DPH_TRO(1)
                 : "v"(a[0]), "v"(a[1]), [o1] "i"(O1), [o2] "i"(O2), [o3] "i"(O3)
                 : "memory");
  else
    asm volatile(DPH_TR4("0", "1", "2", "3", "16") DPH_TR4("4", "5", "6", "7", "17") DPH_TR4("8", "9", "10", "11", "18")
                     DPH_TR4("12", "13", "14", "15", "19") "s_waitcnt lgkmcnt(0)"
                 : DPH_TRO(0), DPH_TRO(1), DPH_TRO(2), DPH_TRO(3)
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), [o1] "i"(O1), [o2] "i"(O2), [o3] "i"(O3)
                 : "memory");
#undef DPH_TR4
#undef DPH_TRO
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int s = 0; s < 2; ++s) f[i][s] = i32x4_t{v[i][2 * s][0], v[i][2 * s][1], v[i][2 * s + 1][0], v[i][2 * s + 1][1]};
}

// WR x WC waves, a ring of S steps in the LDS
template <int BM_, int BN_, int WR_, int WC_, int S_>
struct Tile {
  static constexpr bool DUO = false;
  static constexpr int BM = BM_, BN = BN_, WR = WR_, WC = WC_, NW = WR_ * WC_, NT = NW * 64, S = S_;
  static constexpr int WTM = BM / WR, WTN = BN / WC, FM = WTM / 16, FN = WTN / 16;
  static constexpr int GA = BM / 8 / NW, GB = BN / 8 / NW;   // LDS DMA instructions of a wave per step
  static constexpr int BUF = (BM + BN) * 128, LDS = S * BUF, WPE = 2;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && 2 * LDS <= 160 * 1024, "two workgroups a CU");
};

__device__ __forceinline__ i32x4_t frag(const char* img, int row0, int s, int lane) {
  const int row = row0 + (lane & 15);
  return *reinterpret_cast<const i32x4_t*>(img + row * 128 + (((s * 4 + (lane >> 4)) ^ ((row >> 1) & 7)) << 4));
}

// the first nb (may be negative or above 16) bytes of a fragment, zeros behind them
__device__ __forceinline__ i32x4_t keep_bytes(i32x4_t v, int nb) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int k = nb - 4 * d;
    v[d] &= k >= 4 ? -1 : (k <= 0 ? 0 : (1 << (8 * k)) - 1);
  }
  return v;
}

// acc(i, j) of wave (wr, wc), lane l: rows m0 + wr WTM + 16 i + (l & 15), columns n0 + wc WTN + 16 j + 4 (l >> 4) + r
// (B goes in as the first operand).  Rows past the operand's end read its last row, chunks past kbytes (rounded up to
// 16) the row's first one; where kbytes is no multiple of 128, A's bytes from kbytes on are zeroed in the registers,
// so what stands behind a row of either operand has no effect -- for integers; fp16 rows are zero-padded to 128 bytes,
// F16T's k-rows to a multiple of 64 (kbytes: 2 bytes a k-row).  The product is added to what init() puts into acc while
// the first steps are on their way; it ends with a barrier, so another may follow.  S - 1 steps are in flight: with few
// tiles a step is a load's latency unless several are.  (Seven in flight, one workgroup a CU, were slower than three: 6.2
// against 4.9 us at 499 x 768 x 768; the next step's fragments read before this one's products changed nothing.  Two wave
// groups with half of the steps each, where a CU has one tile, took 6 % off the iteration of one 768 x 768, but a result
// would then depend on how many tiles a call has.)
template <class T, class C, class Init>
__device__ __forceinline__ void product(const Rows& A, const Rows& B, int32_t kbytes, int32_t m0, int32_t n0,
                                        typename T::acc_t (&acc)[C::FM][C::FN], char* smem, int wave, int lane,
                                        Init init) {
  const int wr = wave / C::WC, wc = wave % C::WC;
  const int nk = (kbytes + 127) >> 7, kend = (kbytes + 15) & ~15;
  const char *pa[C::GA], *pb[C::GB];
  int ca[C::GA], cb[C::GB];                       // logical chunk (bytes) of this lane in its row
#pragma unroll
  for (int g = 0; g < C::GA; ++g) {
    const int w = g * C::NW + wave;
    if constexpr (T::TR) {
      const int kr = w * (512 / C::BM) + lane / (C::BM / 8), c = ((lane % (C::BM / 8)) ^ tr_swz<C::BM>(kr)) * 8;
      pa[g] = A.p + (int64_t)kr * A.ld + min(m0 + c, A.rows - 8) * 2;
    } else {
      const int row = w * 8 + (lane >> 3);
      pa[g] = A.p + (int64_t)min(m0 + row, A.rows - 1) * A.ld;
      ca[g] = ((lane & 7) ^ ((row >> 1) & 7)) << 4;
    }
  }
#pragma unroll
  for (int g = 0; g < C::GB; ++g) {
    const int w = g * C::NW + wave;
    if constexpr (T::TR) {
      const int kr = w * (512 / C::BN) + lane / (C::BN / 8), c = ((lane % (C::BN / 8)) ^ tr_swz<C::BN>(kr)) * 8;
      pb[g] = B.p + (int64_t)kr * B.ld + min(n0 + c, B.rows - 8) * 2;
    } else {
      const int row = w * 8 + (lane >> 3);
      pb[g] = B.p + (int64_t)min(n0 + row, B.rows - 1) * B.ld;
      cb[g] = ((lane & 7) ^ ((row >> 1) & 7)) << 4;
    }
  }
  auto stage = [&](int kt, int slot) {
    char* buf = smem + slot * C::BUF;
#pragma unroll
    for (int g = 0; g < C::GA; ++g) {
      const char* p;
      if constexpr (T::TR) p = pa[g] + (int64_t)kt * 64 * A.ld;
      else p = pa[g] + (kt * 128 + ca[g] < kend ? kt * 128 + ca[g] : 0);
      ring::dma16(reinterpret_cast<const bf16_t*>(p), buf + (g * C::NW + wave) * 1024);
    }
#pragma unroll
    for (int g = 0; g < C::GB; ++g) {
      const char* p;
      if constexpr (T::TR) p = pb[g] + (int64_t)kt * 64 * B.ld;
      else p = pb[g] + (kt * 128 + cb[g] < kend ? kt * 128 + cb[g] : 0);
      ring::dma16(reinterpret_cast<const bf16_t*>(p), buf + C::BM * 128 + (g * C::NW + wave) * 1024);
    }
  };
  constexpr int G = C::GA + C::GB;
#pragma unroll
  for (int k = 0; k < C::S - 1; ++k)
    if (k < nk) stage(k, k);
  init();
  int slot = 0;
  for (int kt = 0; kt < nk; ++kt) {
    // step kt is there: the S - 2 behind it may be in flight
    if (nk - 1 - kt >= C::S - 2) pp::vm_wait<(C::S - 2) * G>();
    else pp::vm_wait<0>();
    pp::bar();
    // the slot that was read in the last step (every wave is past it)
    if (kt + C::S - 1 < nk) stage(kt + C::S - 1, slot == 0 ? C::S - 1 : slot - 1);
    const char* buf = smem + slot * C::BUF;
    i32x4_t ta[C::FM][2], tb[C::FN][2];
    if constexpr (T::TR) {
      tr_frags<C::BM>(buf, wr * C::WTM, lane, ta);
      tr_frags<C::BN>(buf + C::BM * 128, wc * C::WTN, lane, tb);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      i32x4_t fa[C::FM], fb[C::FN];
#pragma unroll
      for (int i = 0; i < C::FM; ++i) fa[i] = T::TR ? ta[i][s] : frag(buf, wr * C::WTM + 16 * i, s, lane);
#pragma unroll
      for (int j = 0; j < C::FN; ++j) fb[j] = T::TR ? tb[j][s] : frag(buf + C::BM * 128, wc * C::WTN + 16 * j, s, lane);
      if (T::ESIZE == 1 && kt * 128 + 128 > kbytes) {
        const int nb = kbytes - kt * 128 - (s * 4 + (lane >> 4)) * 16;
#pragma unroll
        for (int i = 0; i < C::FM; ++i) fa[i] = keep_bytes(fa[i], nb);
      }
#pragma unroll
      for (int i = 0; i < C::FM; ++i)
#pragma unroll
        for (int j = 0; j < C::FN; ++j) acc[i][j] = T::mfma(fb[j], fa[i], acc[i][j]);
    }
    pp::lgkm0();   // (this step's image is read: the next step's barrier lets it be overwritten)
    slot = slot + 1 == C::S ? 0 : slot + 1;
  }
  pp::bar();
}

// ---- two wave groups in turn --------------------------------------------------------------------------------------
// The same product by 8 waves, 2 along m and 4 along n, in two groups (the two rows of waves; a SIMD holds one wave of
// each) that run one barrier interval apart: while one multiplies, the other reads its next fragments from the LDS and
// issues the next LDS DMAs, so the matrix core and the LDS work at once.  A 128-byte step along k is staged as four
// half-tiles with lifetimes of their own -- A-lo / A-hi: the first / last FM / 2 fragment rows of both rows of waves;
// B-0 / B-1: the first ceil(FN / 2) / other fragment columns of every wave -- and takes four intervals:
//   0: read B-0 (and A-lo), stage B-1(u+1); A-lo x B-0       1: read B-1, stage A-hi(u+1); A-lo x B-1
//   2: read A-hi, stage A-lo(u+2); A-hi x B-1                3: (read A-lo(u+1)), stage B-0(u+2); A-hi x B-0
// Every half-tile is overwritten two intervals after its last read and read one interval after the wait that retires
// it, and one step's DMAs (G a thread) stay in flight across the barriers.  acc as product's.  A row distance of less
// than 2^23 bytes (32-bit offsets inside a tile); fp16 rows of at least 256 bytes.
template <int BM_, int BN_, int MINB_>
struct Duo {
  static constexpr bool DUO = true;
  static constexpr int BM = BM_, BN = BN_, NW = 8, NT = 512, WC = 4;
  static constexpr int WTM = BM / 2, WTN = BN / 4, FM = WTM / 16, FN = WTN / 16;
  static constexpr int FM2 = FM / 2, FN0 = (FN + 1) / 2, FN1 = FN / 2;
  static constexpr int RA = BM / 2, RB0 = 64 * FN0, RB1 = 64 * FN1;
  static constexpr int GA = RA / 64, GB0 = RB0 / 64, GB1 = RB1 / 64, G = 2 * GA + GB0 + GB1;
  static constexpr int O_ALO = 0, O_AHI = RA * 128, O_B0 = 2 * RA * 128, O_B1 = O_B0 + RB0 * 128;
  static constexpr int BUF = (BM + BN) * 128, LDS = 2 * BUF;
  static constexpr int WPE = 2 * MINB_;                    // waves per SIMD: MINB_ workgroups a CU
  static constexpr bool SPLITA = BM_ == 256 || BN_ == 128; // A-lo of the next step is read in the last interval
  static_assert(FM % 2 == 0 && FN >= 2 && RA % 64 == 0 && MINB_ * LDS <= 160 * 1024, "geometry");
};

template <class T, class C, class Init>
__device__ __forceinline__ void product_duo(const Rows& A, const Rows& B, int32_t kbytes, int32_t m0, int32_t n0,
                                            typename T::acc_t (&acc)[C::FM][C::FN], char* smem, int wave, int lane,
                                            Init init) {
  const int wr = wave >> 2, wc = wave & 3;
  const int nk = max((kbytes + 127) >> 7, 2), kend = (kbytes + 15) & ~15;
  const bool part = T::ESIZE == 1 && kbytes < nk * 128;    // (a step past kbytes: all of it masked)
  const char* Ab = A.p + (T::TR ? (int64_t)m0 * 2 : (int64_t)m0 * A.ld);
  const char* Bb = B.p + (T::TR ? (int64_t)n0 * 2 : (int64_t)n0 * B.ld);
  const int32_t ml = A.rows - 1 - m0, nl = B.rows - 1 - n0, lda = (int32_t)A.ld, ldb = (int32_t)B.ld;
  constexpr int HA = C::WTM / 2;
  // wave instruction g * 8 + wave fills half-tile rows (g * 8 + wave) * 8 .. + 7; lane -> row lane / 8, chunk lane % 8
  const int rw = wave * 8 + (lane >> 3);
  const int lc = ((lane & 7) ^ ((rw >> 1) & 7)) << 4;      // ((row >> 1) & 7 does not depend on g)
  // F16T: row rw of the half-tile image is a k-row, its chunk 8 operand columns
  auto tr_row = [&](int g, int R) { return (g * 8 + wave) * (512 / R) + lane / (R / 8); };
  uint32_t oal[C::GA], oah[C::GA], ob0[C::GB0], ob1[C::GB1];
#pragma unroll
  for (int g = 0; g < C::GA; ++g) {
    int rho = g * 64 + rw;
    if constexpr (T::TR) rho = ((lane % (C::RA / 8)) ^ tr_swz<C::RA>(tr_row(g, C::RA))) * 8;
    const int row = (rho / HA) * C::WTM + rho % HA;
    if constexpr (T::TR) {
      const uint32_t k = (uint32_t)(tr_row(g, C::RA) * lda);
      oal[g] = k + 2 * min(row, ml - 7);
      oah[g] = k + 2 * min(row + HA, ml - 7);
    } else {
      oal[g] = (uint32_t)(min(row, ml) * lda);
      oah[g] = (uint32_t)(min(row + HA, ml) * lda);
    }
  }
#pragma unroll
  for (int g = 0; g < C::GB0; ++g) {
    int rho = g * 64 + rw;
    if constexpr (T::TR) rho = ((lane % (C::RB0 / 8)) ^ tr_swz<C::RB0>(tr_row(g, C::RB0))) * 8;
    const int row = (rho / (16 * C::FN0)) * C::WTN + rho % (16 * C::FN0);
    if constexpr (T::TR) ob0[g] = (uint32_t)(tr_row(g, C::RB0) * ldb) + 2 * min(row, nl - 7);
    else ob0[g] = (uint32_t)(min(row, nl) * ldb);
  }
#pragma unroll
  for (int g = 0; g < C::GB1; ++g) {
    int rho = g * 64 + rw;
    if constexpr (T::TR) rho = ((lane % (C::RB1 / 8)) ^ tr_swz<C::RB1>(tr_row(g, C::RB1))) * 8;
    const int row = (rho / (16 * C::FN1)) * C::WTN + 16 * C::FN0 + rho % (16 * C::FN1);
    if constexpr (T::TR) ob1[g] = (uint32_t)(tr_row(g, C::RB1) * ldb) + 2 * min(row, nl - 7);
    else ob1[g] = (uint32_t)(min(row, nl) * ldb);
  }
  auto buf = [&](int u) -> char* { return smem + (u & 1) * C::BUF; };
  auto koff = [&](int u) -> uint32_t {
    if (T::TR) return 0u;
    if (T::ESIZE == 1) return u * 128 + lc < kend ? (uint32_t)(u * 128 + lc) : 0u;
    return (uint32_t)(u * 128 + lc);
  };
  auto base = [&](const char* p, int64_t ld, int u) { return T::TR ? p + (int64_t)u * 64 * ld : p; };
  auto dma = [&](const char* p, uint32_t off, char* to) { ring::dma16(reinterpret_cast<const bf16_t*>(p + off), to); };
  auto st_alo = [&](int u) {
    const uint32_t k = koff(u);
    const char* p = base(Ab, A.ld, u);
#pragma unroll
    for (int g = 0; g < C::GA; ++g) dma(p, oal[g] + k, buf(u) + C::O_ALO + (g * 8 + wave) * 1024);
  };
  auto st_ahi = [&](int u) {
    const uint32_t k = koff(u);
    const char* p = base(Ab, A.ld, u);
#pragma unroll
    for (int g = 0; g < C::GA; ++g) dma(p, oah[g] + k, buf(u) + C::O_AHI + (g * 8 + wave) * 1024);
  };
  auto st_b0 = [&](int u) {
    const uint32_t k = koff(u);
    const char* p = base(Bb, B.ld, u);
#pragma unroll
    for (int g = 0; g < C::GB0; ++g) dma(p, ob0[g] + k, buf(u) + C::O_B0 + (g * 8 + wave) * 1024);
  };
  auto st_b1 = [&](int u) {
    const uint32_t k = koff(u);
    const char* p = base(Bb, B.ld, u);
#pragma unroll
    for (int g = 0; g < C::GB1; ++g) dma(p, ob1[g] + k, buf(u) + C::O_B1 + (g * 8 + wave) * 1024);
  };
  i32x4_t falo[C::FM2][2], fah_[C::FM2][2], fb0[C::FN0][2], fb1[C::FN1][2];
  i32x4_t(&fahi)[C::FM2][2] = C::SPLITA ? fah_ : falo;
  // the fragments of N groups of 16 rows from r0 on
  auto rd = [&](const char* ht, int r0, auto& f, auto R) {
    if constexpr (T::TR) {
      tr_frags<decltype(R)::value>(ht, r0, lane, f);
    } else {
      constexpr int N = sizeof(f) / sizeof(f[0]);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s) f[i][s] = frag(ht, r0 + 16 * i, s, lane);
    }
  };
  auto rd_a = [&](const char* ht, i32x4_t(&fa)[C::FM2][2]) { rd(ht, wr * HA, fa, std::integral_constant<int, C::RA>{}); };
  auto rd_b0 = [&](const char* bu) {
    rd(bu + C::O_B0, wc * 16 * C::FN0, fb0, std::integral_constant<int, C::RB0>{});
  };
  auto rd_b1 = [&](const char* bu) {
    rd(bu + C::O_B1, wc * 16 * C::FN1, fb1, std::integral_constant<int, C::RB1>{});
  };
  auto mask = [&](int u, i32x4_t(&fa)[C::FM2][2]) {
    if (!part) return;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int nb = kbytes - u * 128 - (s * 4 + (lane >> 4)) * 16;
#pragma unroll
      for (int i = 0; i < C::FM2; ++i) fa[i][s] = keep_bytes(fa[i][s], nb);
    }
  };
  auto mm0 = [&](int i0, const i32x4_t(&fa)[C::FM2][2]) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < C::FM2; ++i)
#pragma unroll
        for (int j = 0; j < C::FN0; ++j) acc[i0 + i][j] = T::mfma(fb0[j][s], fa[i][s], acc[i0 + i][j]);
    __builtin_amdgcn_s_setprio(0);
  };
  auto mm1 = [&](int i0, const i32x4_t(&fa)[C::FM2][2]) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < C::FM2; ++i)
#pragma unroll
        for (int j = 0; j < C::FN1; ++j) acc[i0 + i][C::FN0 + j] = T::mfma(fb1[j][s], fa[i][s], acc[i0 + i][C::FN0 + j]);
    __builtin_amdgcn_s_setprio(0);
  };
  constexpr int G = C::G;
  auto go = [&]() {          // the reads of this interval are in registers
    pp::bar();
    pp::lgkm0();
    __builtin_amdgcn_sched_barrier(0);
  };
  st_alo(0);
  st_b0(0);
  st_b1(0);
  st_ahi(0);
  st_alo(1);
  st_b0(1);
  init();
  pp::vm_wait<G>();
  pp::bar();
  if constexpr (C::SPLITA) rd_a(buf(0) + C::O_ALO, falo);
  if (wr == 1) pp::bar();    // group 1 runs one interval behind group 0
  int u = 0;
#pragma unroll 1
  for (; u + 2 < nk; ++u) {
    const char* bu = buf(u);
    rd_b0(bu);
    if constexpr (!C::SPLITA) rd_a(bu + C::O_ALO, falo);
    st_b1(u + 1);
    pp::vm_wait<G>();
    go();
    mm0(0, falo);
    pp::bar();
    rd_b1(bu);
    st_ahi(u + 1);
    pp::vm_wait<G>();
    go();
    mm1(0, falo);
    pp::bar();
    rd_a(bu + C::O_AHI, fahi);
    st_alo(u + 2);
    pp::vm_wait<G>();
    go();
    mm1(C::FM2, fahi);
    pp::bar();
    if constexpr (C::SPLITA) rd_a(buf(u + 1) + C::O_ALO, falo);
    st_b0(u + 2);
    pp::vm_wait<G>();
    pp::bar();
    mm0(C::FM2, fahi);
    pp::bar();
  }
  // the last two steps: nothing is staged past nk - 1, the waits drain
#pragma unroll
  for (int t = 0; t < 2; ++t, ++u) {
    const char* bu = buf(u);
    rd_b0(bu);
    if constexpr (!C::SPLITA) rd_a(bu + C::O_ALO, falo);
    if (t == 0) {
      st_b1(u + 1);
      pp::vm_wait<G>();
    } else {
      pp::vm_wait<C::GA>();
    }
    go();
    mask(u, falo);
    mm0(0, falo);
    pp::bar();
    rd_b1(bu);
    if (t == 0) {
      st_ahi(u + 1);
      pp::vm_wait<G>();
    } else {
      pp::vm_wait<0>();
    }
    go();
    mm1(0, falo);
    pp::bar();
    rd_a(bu + C::O_AHI, fahi);
    if (t == 0) pp::vm_wait<G - C::GA>();
    else pp::vm_wait<0>();
    go();
    mask(u, fahi);
    mm1(C::FM2, fahi);
    pp::bar();
    if (t == 0) {
      if constexpr (C::SPLITA) rd_a(buf(u + 1) + C::O_ALO, falo);
      pp::vm_wait<C::GB1 + C::GA>();
    } else {
      pp::vm_wait<0>();
    }
    pp::bar();
    mm0(C::FM2, fahi);
    pp::bar();
  }
  if (wr == 0) pp::bar();    // pairs with group 1's first one
}

template <class T, class C>
__device__ __forceinline__ void clear(typename T::acc_t (&acc)[C::FM][C::FN]) {
#pragma unroll
  for (int i = 0; i < C::FM; ++i)
#pragma unroll
    for (int j = 0; j < C::FN; ++j) acc[i][j] = typename T::acc_t{0, 0, 0, 0};
}

template <class T, class C, class Init>
__device__ __forceinline__ void product_of(const Rows& A, const Rows& B, int32_t kbytes, int32_t m0, int32_t n0,
                                           typename T::acc_t (&acc)[C::FM][C::FN], char* smem, int wave, int lane,
                                           Init init) {
  if constexpr (C::DUO) product_duo<T, C>(A, B, kbytes, m0, n0, acc, smem, wave, lane, init);
  else product<T, C>(A, B, kbytes, m0, n0, acc, smem, wave, lane, init);
}

// ---- 16 bytes of a row in a lane -------------------------------------------------------------------------------------
// A wave's 16 x 16 FN strip of acc has 4 columns of each fragment in a lane: 16-byte accesses of 64-byte runs if they are
// stored in 32 bits, but 8-byte ones of 32-byte runs in 16.  Exchanging the columns of two fragments between the groups
// of 16 lanes (by lane swaps; its own inverse) gives a lane 8 consecutive ones, and 64-byte runs of 16-bit numbers.
// (16 columns a lane, two 16-byte accesses a lane, stored 7984 x 4096 at 2.4 TB/s: what counts is one access's run.)
template <int FN, int W_>
struct Strip {
  static constexpr int W = W_, NG = 4 * FN / W;   // NG groups of W columns a lane
  static_assert(W == 4 || (W == 8 && FN % 2 == 0) || (W == 16 && FN % 4 == 0), "whole exchanges");
  // first column of group q in the strip
  static __device__ __forceinline__ int col(int q, int lane) {
    return W == 4    ? 16 * q + 4 * (lane >> 4)
           : W == 8  ? 32 * q + 16 * ((lane >> 4) & 1) + 8 * (lane >> 5)
                     : 64 * q + 16 * (lane >> 4);
  }
  static __device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
  }
  static __device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
  }
  // v[4 j + r]: fragment j's column 4 (lane / 16) + r  <->  v[W q + c]: column col(q) + c
  static __device__ __forceinline__ void exchange(uint32_t (&v)[4 * FN]) {
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        uint32_t* a = v + W * q + r;
        if constexpr (W == 16) {
          swap32(a[0], a[8]);
          swap32(a[4], a[12]);
          swap16(a[0], a[4]);
          swap16(a[8], a[12]);
        } else if constexpr (W == 8) {
          swap16(a[0], a[4]);
        }
      }
  }
};

// Workgroups go to the 8 XCDs in turn: block b of n works on a contiguous range of tiles per XCD, so the tiles of one
// L2 share their operands' rows (reverse: each XCD its own range backwards)
__device__ __forceinline__ int xcd_tile(int b, int n, bool reverse = false) {
  const int q = n >> 3, r = n & 7, x = b & 7, i = b >> 3, size = q + (x < r ? 1 : 0);
  return x * q + min(x, r) + (reverse ? size - 1 - i : i);
}

// Which tiles a product of so many of each takes: 256 x 256 (one workgroup a CU), 128 x 128 or 64 x 64 (two).  A CU's work
// is counted in rounds of 256 CUs: a 256 x 256 tile 1, two tiles of 128 x 128 side by side 0.58 and one alone 0.36, of 64 x
// 64 0.33 and 0.22 (measured on K of 512 to 4096: the larger the tile, the fewer bytes pass the LDS a product, but the
// more of the chip idles in the last round).  A negative count: not available.
struct C256 : Duo<256, 256, 1> {};
struct C128 : Duo<128, 128, 2> {};
struct C64 : Tile<64, 64, 2, 2, 4> {};
inline double pairs(int64_t tiles, double two, double one) {
  const int64_t n = cdiv(tiles, 256);
  return tiles < 0 ? 1e30 : (double)(n / 2) * two + (double)(n % 2) * one;
}
inline int choose_tile(int64_t t256, int64_t t128, int64_t t64) {
  const double c256 = (double)cdiv(t256, 256), c128 = pairs(t128, 0.58, 0.36), c64 = pairs(t64, 0.33, 0.22);
  return c64 < c128 && c64 < c256 ? 64 : c128 < c256 ? 128 : 256;
}

}  // namespace mt
}  // namespace
}  // namespace dph
