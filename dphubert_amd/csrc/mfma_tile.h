// Tile products of byte rows for the matrix cores: C[m][n] = sum_k A[m][k] B[n][k], both operands k-contiguous, of
// 8-bit integers (32-bit integer sums) or fp16 (fp32 sums).  The two types share everything but the instruction:
// v_mfma_i32_16x16x64_i8 and v_mfma_f32_16x16x32_f16 both take 16 bytes of a row per lane and run at 16 cycles, so a
// 128-byte step along k is 128 integers or 64 fp16 with the same staging, LDS image and fragment reads.
//
// LDS image of an operand step: rows of 128 bytes, 16-byte chunk p of row r holds the k-chunk p ^ ((r >> 1) & 7) (no
// bank conflict for the 16-lane groups of ds_read_b128); the swizzle is applied to the source address, since an LDS
// DMA writes its 1 KB in lane order.
#pragma once
#include "gemm_core.h"

namespace dph {
namespace {
namespace mt {

typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;

struct I8 {
  typedef i32x4_t acc_t;
  static constexpr int ESIZE = 1;
  static __device__ __forceinline__ acc_t mfma(i32x4_t a, i32x4_t b, acc_t c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
};
struct F16 {
  typedef f32x4_t acc_t;
  static constexpr int ESIZE = 2;
  static __device__ __forceinline__ acc_t mfma(i32x4_t a, i32x4_t b, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  }
};

// One operand: rows of ld bytes, `rows` of them; ld and the base are multiples of 16
struct Rows {
  const char* p;
  int64_t ld;
  int32_t rows;
};

template <int BM_, int BN_, int WR_, int WC_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WR = WR_, WC = WC_, NW = WR_ * WC_, NT = NW * 64;
  static constexpr int WTM = BM / WR, WTN = BN / WC, FM = WTM / 16, FN = WTN / 16;
  static constexpr int GA = BM / 8 / NW, GB = BN / 8 / NW;   // LDS DMA instructions of a wave per step
  static constexpr int BUF = (BM + BN) * 128, LDS = 2 * BUF;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "whole DMA instructions");
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
// so what stands behind a row of either operand has no effect -- for integers; fp16 rows are zero-padded to 128 bytes.
// The product is added to acc; it ends with a barrier, so another may follow.
template <class T, class C>
__device__ __forceinline__ void product(const Rows& A, const Rows& B, int32_t kbytes, int32_t m0, int32_t n0,
                                        typename T::acc_t (&acc)[C::FM][C::FN], char* smem, int wave, int lane) {
  const int wr = wave / C::WC, wc = wave % C::WC;
  const int nk = (kbytes + 127) >> 7, kend = (kbytes + 15) & ~15;
  const char *pa[C::GA], *pb[C::GB];
  const int lrow = lane >> 3;
#pragma unroll
  for (int g = 0; g < C::GA; ++g) pa[g] = A.p + (int64_t)min(m0 + (g * C::NW + wave) * 8 + lrow, A.rows - 1) * A.ld;
#pragma unroll
  for (int g = 0; g < C::GB; ++g) pb[g] = B.p + (int64_t)min(n0 + (g * C::NW + wave) * 8 + lrow, B.rows - 1) * B.ld;
  // ((row >> 1) & 7 of row = 8 (..) + lrow)
  auto stage = [&](int kt) {
    char* buf = smem + (kt & 1) * C::BUF;
#pragma unroll
    for (int g = 0; g < C::GA; ++g) {
      const int row = (g * C::NW + wave) * 8 + lrow;
      const int off = kt * 128 + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
      ring::dma16(reinterpret_cast<const bf16_t*>(pa[g] + (off < kend ? off : 0)), buf + (g * C::NW + wave) * 1024);
    }
#pragma unroll
    for (int g = 0; g < C::GB; ++g) {
      const int row = (g * C::NW + wave) * 8 + lrow;
      const int off = kt * 128 + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
      ring::dma16(reinterpret_cast<const bf16_t*>(pb[g] + (off < kend ? off : 0)),
                  buf + C::BM * 128 + (g * C::NW + wave) * 1024);
    }
  };
  stage(0);
  for (int kt = 0; kt < nk; ++kt) {
    pp::vm_wait<0>();
    pp::bar();
    if (kt + 1 < nk) stage(kt + 1);
    const char* buf = smem + (kt & 1) * C::BUF;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      i32x4_t fa[C::FM], fb[C::FN];
#pragma unroll
      for (int i = 0; i < C::FM; ++i) fa[i] = frag(buf, wr * C::WTM + 16 * i, s, lane);
#pragma unroll
      for (int j = 0; j < C::FN; ++j) fb[j] = frag(buf + C::BM * 128, wc * C::WTN + 16 * j, s, lane);
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
  }
  pp::bar();
}

template <class T, class C>
__device__ __forceinline__ void clear(typename T::acc_t (&acc)[C::FM][C::FN]) {
#pragma unroll
  for (int i = 0; i < C::FM; ++i)
#pragma unroll
    for (int j = 0; j < C::FN; ++j) acc[i][j] = typename T::acc_t{0, 0, 0, 0};
}

// Workgroups go to the 8 XCDs in turn: block b of n works on a contiguous range of tiles per XCD, so the tiles of one
// L2 share their operands' rows
__device__ __forceinline__ int xcd_tile(int b, int n) {
  const int q = n >> 3, r = n & 7, x = b & 7, i = b >> 3;
  return x * q + min(x, r) + i;
}

}  // namespace mt
}  // namespace
}  // namespace dph
