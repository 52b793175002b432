// Products in 8-bit integers with one scale a row of either operand (a token's, an output channel's):
//
//   y[m][n] = act( xs[m] ws[n] sum_k q[m][k] w[n][k] + bias[n] ) + residual[m][n]
//
// q[m][k] = x[m][k] / xs[m] to the nearest integer, ties to even, xs[m] = max_k |x[m][k]| (1 / 127) -- the activations are
// quantised on the way in, a row at a time, either as they stand or as the output of a LayerNorm.
#include "mfma_tile.h"

#include <type_traits>

namespace dph {
namespace {

constexpr float SCALE_MIN = 1.17549435e-38f;   // 2^-126: the scale of a row of zeros (its inverse is finite)

// x / s to the nearest integer, ties to even, of the EXACT quotient: t = x inv is within one of it, and d = x - t s is
// exact (one fma; a multiple of s's last place, at most 24 bits), so comparing 2 d with s decides the rounding -- five
// instructions instead of a division
__device__ __forceinline__ int quant1(float x, float inv, float s) {
  float t = rintf(x * inv);
  const float d = fmaf(-t, s, x), a = fabsf(d), h = 0.5f * s;
  const int i = (int)t, off = (int)(a > h) | ((int)(a == h) & i);
  return i + (off & 1 ? (d > 0.f ? 1 : -1) : 0);
}

// 8 elements as they are in memory (bf16: 16 bytes, fp32: 32), zeros past K
template <typename XT>
struct Raw8 {
  uint4 a, b;   // (b: fp32 only)
  __device__ __forceinline__ void load(const XT* row, int c, int K) {
    constexpr bool F = std::is_same_v<XT, float>;
    if (c + 8 <= K) {
      a = mt::ld16(row + c);
      if constexpr (F) b = mt::ld16(row + c + 4);
    } else {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = 0;
        if (c + i < K) {
          if constexpr (F) w[i] = __float_as_uint(row[c + i]);
          else w[i] = row[c + i];
        }
      }
      if constexpr (F) {
        a = make_uint4(w[0], w[1], w[2], w[3]);
        b = make_uint4(w[4], w[5], w[6], w[7]);
      } else {
        a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (std::is_same_v<XT, float>) v[i] = __uint_as_float(w[i]);
      else v[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    }
  }
};
template <typename XT>
__device__ __forceinline__ void load8(const XT* row, int c, int K, float (&v)[8]) {
  Raw8<XT> r;
  r.load(row, c, K);
  r.get(v);
}

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  return v;
}

// scale of a row from the largest |x| as bits (so that a NaN, or an infinity, counts as the largest)
__device__ __forceinline__ float row_scale(uint32_t amax_bits) {
  return amax_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(amax_bits) * (1.0f / 127.0f), SCALE_MIN);
}

// 8 integers of a row.  Adding 1.5 2^23 rounds x inv to an integer and leaves it in the low bits; unless a remainder is half a
// step or more (x / s so near a half that x inv may be on its other side: 1 of 30000 numbers), that is the quotient's: 5
// instructions a number instead of 13 (7984 x 4096 from bf16 22.5 -> 19.8 us)
__device__ __forceinline__ uint2 pack8(const float (&v)[8], float inv, float s) {
  constexpr float UP = 12582912.f;
  float r[8], m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    r[i] = fmaf(v[i], inv, UP);
    m = fmaxf(m, fabsf(fmaf(UP - r[i], s, v[i])));
  }
  if (__builtin_expect(m < 0.5f * s, 1)) {
    auto four = [&](int i) {
      const uint32_t a = __builtin_amdgcn_perm(__float_as_uint(r[i + 1]), __float_as_uint(r[i]), 0x0c0c0400u);
      const uint32_t b = __builtin_amdgcn_perm(__float_as_uint(r[i + 3]), __float_as_uint(r[i + 2]), 0x04000c0cu);
      return a | b;
    };
    return make_uint2(four(0), four(4));
  }
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i >> 2] |= ((uint32_t)quant1(v[i], inv, s) & 0xffu) << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}

// exact-erf GELU as common.h's (Abramowitz & Stegun 7.1.26, 1.5e-7), in the form max(x, 0) - |x| erfc(|x| / sqrt 2) / 2: no
// comparison, and the halves and square roots are in the constants (58 -> 56 us at 7984 x 4096 x 1024, where it is a third).
// An infinite |x| is cut off where it meets the erfc's zero (a NaN stays one: it comes through t)
__device__ __forceinline__ float gelu_i8(float x) {
  const float ax = fabsf(x), t = __builtin_amdgcn_rcpf(fmaf(0.23164189f, ax, 1.0f));
  const float p = t * (0.127414796f + t * (-0.142248368f + t * (0.7107068705f + t * (-0.7265760135f + t * 0.5307027145f))));
  return fmaf(-fminf(ax, 1e30f), p * __builtin_amdgcn_exp2f(x * x * -0.72134752f), fmaxf(x, 0.f));
}

__device__ __forceinline__ uint32_t umax8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

// One wave a row, read once: NV chunks of 8 elements a lane stay in registers (NV 512 columns); longer rows are read
// again for their integers (NV = 0).  ldq is a multiple of 16; the row's bytes from K on are written as zeros.  Bound by
// memory: 7984 x 4096 in 25.8 us from fp32 (164 MB, 6.4 TB/s) and in 19.8 us from bf16 (98 MB, 5.0 TB/s).
template <typename XT, int NV>
__global__ void __launch_bounds__(256) quant_rows_kernel(const XT* __restrict__ x, int64_t rows, int32_t K, int64_t ldx,
                                                         int8_t* __restrict__ q, int64_t ldq,
                                                         float* __restrict__ scale) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const XT* xr = x + r * ldx;
  int8_t* qr = q + r * ldq;
  float v[8];
  uint32_t m = 0;
  if constexpr (NV > 0) {
    Raw8<XT> raw[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) raw[j].load(xr, j * 512 + lane * 8, K);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      raw[j].get(v);
      m = max(m, umax8(v));
    }
    const float s = row_scale(wave_umax(m)), inv = 1.0f / s;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = j * 512 + lane * 8;
      raw[j].get(v);
      if (c < ldq) *reinterpret_cast<uint2*>(qr + c) = s == s ? pack8(v, inv, s) : make_uint2(0, 0);
    }
    if (lane == 0) scale[r] = s;
  } else {
    for (int c = lane * 8; c < K; c += 512) {
      load8(xr, c, K, v);
      m = max(m, umax8(v));
    }
    const float s = row_scale(wave_umax(m)), inv = 1.0f / s;
    for (int c = lane * 8; c < ldq; c += 512) {
      load8(xr, c, K, v);
      *reinterpret_cast<uint2*>(qr + c) = s == s ? pack8(v, inv, s) : make_uint2(0, 0);
    }
    if (lane == 0) scale[r] = s;
  }
}

// LayerNorm of a row (fp32 two-pass statistics) into v; the values go to yr in bf16 too where the residual branch wants
// them.  One wave; NV chunks of 8 columns a lane.  Returns the largest |v| as bits.
template <int NV, typename XT>
__device__ __forceinline__ uint32_t norm_row(const XT* xr, const float* __restrict__ gamma,
                                             const float* __restrict__ beta, int K, float eps, bf16_t* yr,
                                             int lane, float (&v)[NV][8]) {
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load8(xr, j * 512 + lane * 8, K, v[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += v[j][i];
  }
  const float mean = wave_sum(sum) / (float)K;
  float sq = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = j * 512 + lane * 8 + i < K ? v[j][i] - mean : 0.f;
      sq += d * d;
    }
  const float rstd = rsqrtf(wave_sum(sq) / (float)K + eps);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * 512 + lane * 8;
    float g[8], b[8];
    load8(gamma, c, K, g);
    load8(beta, c, K, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = c + i < K ? (v[j][i] - mean) * rstd * g[i] + b[i] : 0.f;
    m = max(m, umax8(v[j]));
    if (yr) {
      if (c + 8 <= K) {
        mt::st16(yr + c, make_uint4(pack2bf(v[j][0], v[j][1]), pack2bf(v[j][2], v[j][3]),
                                 pack2bf(v[j][4], v[j][5]), pack2bf(v[j][6], v[j][7])));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < K) yr[c + i] = f2bf(v[j][i]);
      }
    }
  }
  return wave_umax(m);
}

// The LayerNorm's rows as integers: one wave a row, read once, everything between the read and the integers in its registers.
// Bound by memory and, about as much, by its instructions: 7984 x 1024 from fp32 in 10.6 us (41 MB, 3.9 TB/s).
template <typename XT, int NV>
__global__ void __launch_bounds__(256) ln_quant_kernel(const XT* __restrict__ x, const float* __restrict__ gamma,
                                                       const float* __restrict__ beta, int64_t rows, int32_t K,
                                                       int64_t ldx, float eps, bf16_t* __restrict__ y, int64_t ldy,
                                                       int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  float v[NV][8];
  const float s = row_scale(norm_row<NV>(x + r * ldx, gamma, beta, K, eps, y ? y + r * ldy : nullptr, lane, v));
  const float inv = 1.0f / s;
  int8_t* qr = q + r * ldq;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * 512 + lane * 8;
    if (c < ldq) *reinterpret_cast<uint2*>(qr + c) = s == s ? pack8(v[j], inv, s) : make_uint2(0, 0);
  }
  if (lane == 0) scale[r] = s;
}

// ---- the product --------------------------------------------------------------------------------------------------
struct LinearI8 {
  mt::Rows x, w;
  int32_t M, N, K;
  const float *xs, *ws, *bias;
  const void* res;
  void* out;
  int64_t ldr, ldo;
  int32_t ntn, ntiles;
};

// W consecutive columns of the residual's row m from n on, as they are in memory: VEC in one read (at any alignment), else
// one by one, the last column's past N.  RES: 0 none, 1 bf16, 2 fp32
template <int W, int RES>
struct Resid {
  uint32_t w[RES == 2 ? W : W / 2];
  template <bool VEC>
  __device__ __forceinline__ void load(const LinearI8& a, int64_t m, int n) {
    const int64_t o = m * a.ldr + n;
    [[maybe_unused]] const int last = a.N - 1 - n;      // (may be negative: the row's last column all the same)
    if constexpr (VEC) {
      const uint4 r = mt::ld16(reinterpret_cast<const char*>(a.res) + o * (RES == 2 ? 4 : 2));
      w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
    } else if constexpr (RES == 1) {
      const bf16_t* p = reinterpret_cast<const bf16_t*>(a.res) + o;
#pragma unroll
      for (int c = 0; c < W; c += 2) w[c / 2] = (uint32_t)p[min(c, last)] | (uint32_t)p[min(c + 1, last)] << 16;
    } else if constexpr (RES == 2) {
      const float* p = reinterpret_cast<const float*>(a.res) + o;
#pragma unroll
      for (int c = 0; c < W; ++c) w[c] = __float_as_uint(p[min(c, last)]);
    }
  }
  __device__ __forceinline__ float get(int c) const {
    if constexpr (RES == 0) return 0.f;
    if constexpr (RES == 2) return __uint_as_float(w[c]);
    return __uint_as_float(c & 1 ? w[c / 2] & 0xffff0000u : w[c / 2] << 16);
  }
};

// The row's W sums v, finished and stored (the output has the residual's type; without one it is bf16, or fp32 with OUT32)
template <int W, bool GELU, int RES, bool OUT32, bool VEC>
__device__ __forceinline__ void finish(const LinearI8& a, int64_t m, int n, float xs, const float* ws, const float* bias,
                                       const Resid<W, RES>& t, float* v) {
  static_assert(W == (OUT32 ? 4 : 8), "16 bytes");
  const int64_t o = m * a.ldo + n;
#pragma unroll
  for (int c = 0; c < W; ++c) {
    v[c] = fmaf(v[c] * xs, ws[c], bias[c]);
    if (GELU) v[c] = gelu_i8(v[c]);
    if constexpr (RES != 0) v[c] += t.get(c);
  }
  if constexpr (OUT32) {
    float* p = reinterpret_cast<float*>(a.out) + o;
    if constexpr (VEC) {
      mt::st16(p, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
    } else {
#pragma unroll
      for (int c = 0; c < W; ++c)
        if (n + c < a.N) p[c] = v[c];
    }
  } else {
    bf16_t* p = reinterpret_cast<bf16_t*>(a.out) + o;
    if constexpr (VEC) {
      mt::st16(p, make_uint4(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7])));
    } else {
#pragma unroll
      for (int c = 0; c < W; ++c)
        if (n + c < a.N) p[c] = f2bf(v[c]);
    }
  }
}

// A tile's scales and biases: asked for before the product, in the LDS after it (read from memory between the stores they
// cost a latency a fragment row: the stores might write them, for all the compiler knows)
template <class C>
struct Scales {
  float xs[C::BM], ws[C::BN], bias[C::BN];
};
template <class C>
struct ScaleRegs {
  static_assert(C::NT >= C::BM && C::NT >= C::BN, "one of each a thread");
  float xs, ws, bias;
  __device__ __forceinline__ void load(const LinearI8& a, int m0, int n0) {
    const int t = threadIdx.x, n = min(n0 + t, a.N - 1);
    if (t < C::BM) xs = a.xs[min(m0 + t, a.M - 1)];
    if (t < C::BN) {
      ws = a.ws[n];
      bias = a.bias ? a.bias[n] : 0.f;
    }
  }
  __device__ __forceinline__ void store(Scales<C>& s) const {
    const int t = threadIdx.x;
    if (t < C::BM) s.xs[t] = xs;
    if (t < C::BN) s.ws[t] = ws, s.bias[t] = bias;
    __syncthreads();
  }
};

template <class C, bool GELU, int RES, bool OUT32>
__device__ __forceinline__ void store_tile(const LinearI8& a, const mt::i32x4_t (&acc)[C::FM][C::FN],
                                           const Scales<C>& sc, int m0, int n0, int wave, int lane) {
  using V = mt::Strip<C::FN, OUT32 ? 4 : 8>;
  const int wn = wave % C::WC * C::WTN, mt0 = wave / C::WC * C::WTM + (lane & 15);
  auto rows = [&](auto vec) {
    constexpr bool VEC = decltype(vec)::value;
#pragma unroll
    for (int i = 0; i < C::FM; ++i) {
      const int mt = mt0 + 16 * i, m = m0 + mt;
      // (a fragment row's residual when the row before is stored: asked for two, four or eight rows early, reads and writes
      // come in bursts, 86, 89 and 98 us against 86 at 7984 x 4096 x 1024 in fp32)
      Resid<V::W, RES> t[V::NG];
      if constexpr (RES != 0) {
#pragma unroll
        for (int q = 0; q < V::NG; ++q) t[q].template load<VEC>(a, min(m, a.M - 1), n0 + wn + V::col(q, lane));
      }
      uint32_t b[4 * C::FN];
#pragma unroll
      for (int r = 0; r < 4 * C::FN; ++r) b[r] = (uint32_t)acc[i][r >> 2][r & 3];
      V::exchange(b);
      const float xs = sc.xs[mt];
#pragma unroll
      for (int q = 0; q < V::NG; ++q) {
        const int nt = wn + V::col(q, lane);
        float v[V::W];
#pragma unroll
        for (int r = 0; r < V::W; ++r) v[r] = (float)(int32_t)b[V::W * q + r];
        if (m < a.M) finish<V::W, GELU, RES, OUT32, VEC>(a, m, n0 + nt, xs, sc.ws + nt, sc.bias + nt, t[q], v);
      }
    }
  };
  // a wave's strip of whole vectors has no branch but the one on the row (a read inside a branch is waited for there, alone:
  // 109 us instead of 86)
  if (n0 + wn + C::WTN <= a.N) rows(std::true_type{});
  else rows(std::false_type{});
}

// The tiles of mfma_tile.h with the scales, the activation and the residual in the epilogue.  8192 x 8192 x 8192 398 us (2760
// TOP/s; 455 us on a device that clocks lower); 7984 x 1024 x 4096 36 us (1860 TOP/s), with an fp32 residual 41; 7984 x 4096 x 1024 39 us, with GELU 51, with an
// fp32 residual 84 (262 MB).  Long sums are bound by the passage of operands through the LDS; short ones by the epilogue,
// 14 instructions an element for GELU or memory, which a CU's one workgroup does not overlap with products, and two
// workgroups, whose smaller tiles move more through the LDS, overlap in part.
template <class C, bool GELU, int RES, bool OUT32>
__global__ void __launch_bounds__(C::NT, C::WPE) linear_i8_kernel(const LinearI8 a) {
  __shared__ __align__(1024) char smem[C::LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // tiles of one XCD: GM rows of tiles, column by column, so that its L2 holds both operands of what runs there
  constexpr int GM = C::BM > 128 ? 4 : 8;
  const int t = mt::xcd_tile((int)blockIdx.x, a.ntiles), per = GM * a.ntn, ntm = a.ntiles / a.ntn;
  const int first = t / per * GM, h = min(GM, ntm - first), l = t % per;
  const int m0 = (first + l % h) * C::BM, n0 = l / h * C::BN;
  mt::i32x4_t acc[C::FM][C::FN];
  ScaleRegs<C> sr;
  mt::product_of<mt::I8, C>(a.x, a.w, a.K, m0, n0, acc, smem, wave, lane, [&]() {
    sr.load(a, m0, n0);
    mt::clear<mt::I8, C>(acc);
  });
  Scales<C>& sc = *reinterpret_cast<Scales<C>*>(smem);    // (the product is through with its images)
  sr.store(sc);
  store_tile<C, GELU, RES, OUT32>(a, acc, sc, m0, n0, wave, lane);
}

// Up to 16 rows of x in one launch: a workgroup quantises all of them for itself (they come from the L2), into the LDS,
// and multiplies 16 channels of W, read once and straight into the registers, a quarter of K a wave.  What bounds it is
// the latency of one read of x, the quantiser's reductions and one read of W, asked for before them: 4.1 us for one row of
// 1024 and 4096 channels in a replayed graph, 4.9 by the kernel trace (W's 4.2 MB at a copy's rate: 0.9 us).
struct SmallI8 {
  LinearI8 l;
  const void* x;
  int64_t ldx;
  const float *gamma, *beta;
  bf16_t* norm;
  int64_t ldn;
  float eps;
  int32_t lds_ld;      // bytes of a row of q in the LDS
};

template <typename XT, int NV>
__device__ __forceinline__ float small_quant(const SmallI8& a, int r, int8_t* qr, int lane) {
  const int K = a.l.K;
  const XT* xr = reinterpret_cast<const XT*>(a.x) + r * a.ldx;
  float s;
  if constexpr (NV > 0) {       // LayerNorm
    float v[NV][8];
    bf16_t* yr = a.norm && blockIdx.x == 0 ? a.norm + r * a.ldn : nullptr;
    s = row_scale(norm_row<NV>(xr, a.gamma, a.beta, K, a.eps, yr, lane, v));
    const float inv = 1.0f / s;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = j * 512 + lane * 8;
      if (c < a.lds_ld) *reinterpret_cast<uint2*>(qr + c) = s == s ? pack8(v[j], inv, s) : make_uint2(0, 0);
    }
  } else {
    uint32_t m = 0;
    float v[8];
    for (int c = lane * 8; c < K; c += 512) {
      load8(xr, c, K, v);
      m = max(m, umax8(v));
    }
    s = row_scale(wave_umax(m));
    const float inv = 1.0f / s;
    for (int c = lane * 8; c < a.lds_ld; c += 512) {
      load8(xr, c, K, v);
      *reinterpret_cast<uint2*>(qr + c) = s == s ? pack8(v, inv, s) : make_uint2(0, 0);
    }
  }
  return s;
}

constexpr int SMALL_M = 16, SMALL_LDS = 56 * 1024;   // (static and dynamic LDS within 64 KB)
// bytes of a row of q in the LDS: whole steps of 64, and 16 more so that the rows start on different banks
constexpr int64_t small_ld(int64_t K) { return ((K + 63) & ~(int64_t)63) + 16; }

template <typename XT, int NV, bool GELU, int RES, bool OUT32>
__global__ void __launch_bounds__(256) small_i8_kernel(const SmallI8 a) {
  extern __shared__ __align__(16) char sq[];     // [M][lds_ld] integers
  __shared__ float scale[SMALL_M];
  __shared__ int32_t part[4][SMALL_M][17];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int M = a.l.M, n0 = blockIdx.x * 16;
  // W's first chunks are asked for before x is looked at
  const int steps = (a.l.K + 63) >> 6, per = (steps + 3) >> 2, k0 = wave * per, k1 = min(steps, k0 + per);
  const int kend = (a.l.K + 15) & ~15;
  const char* wr = a.l.w.p + (int64_t)min(n0 + (lane & 15), a.l.N - 1) * a.l.w.ld;
  auto ldw = [&](int k) {
    const int off = k * 64 + (lane >> 4) * 16;
    return *reinterpret_cast<const mt::i32x4_t*>(wr + (off < kend ? off : 0));
  };
  constexpr int AHEAD = 4;
  mt::i32x4_t w[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (k0 + i < k1) w[i] = ldw(k0 + i);
  for (int r = wave; r < M; r += 4) {
    const float s = small_quant<XT, NV>(a, r, reinterpret_cast<int8_t*>(sq) + r * a.lds_ld, lane);
    if (lane == 0) scale[r] = s;
  }
  __syncthreads();
  // (rows past M: the last one's, never stored; chunks past K are zeros in the LDS)
  const char* qr = sq + min(lane & 15, M - 1) * a.lds_ld + (lane >> 4) * 16;
  mt::i32x4_t acc = {0, 0, 0, 0};
  for (int k = k0; k < k1; k += AHEAD) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (k + i >= k1) break;
      const mt::i32x4_t now = w[i];
      if (k + i + AHEAD < k1) w[i] = ldw(k + i + AHEAD);
      acc = mt::I8::mfma(now, *reinterpret_cast<const mt::i32x4_t*>(qr + (k + i) * 64), acc);
    }
  }
  // acc: channel n0 + 4 (lane / 16) + r of row lane % 16
#pragma unroll
  for (int r = 0; r < 4; ++r) part[wave][lane & 15][4 * (lane >> 4) + r] = acc[r];
  __syncthreads();
  const int m = threadIdx.x >> 4, c = threadIdx.x & 15, n = n0 + c;
  if (m < M && n < a.l.N) {
    float v = (float)(part[0][m][c] + part[1][m][c] + part[2][m][c] + part[3][m][c]);
    v = fmaf(v * scale[m], a.l.ws[n], a.l.bias ? a.l.bias[n] : 0.f);
    if (GELU) v = gelu_i8(v);
    if constexpr (RES == 1) v += bf2f(reinterpret_cast<const bf16_t*>(a.l.res)[m * a.l.ldr + n]);
    if constexpr (RES == 2) v += reinterpret_cast<const float*>(a.l.res)[m * a.l.ldr + n];
    if constexpr (OUT32) reinterpret_cast<float*>(a.l.out)[m * a.l.ldo + n] = v;
    else reinterpret_cast<bf16_t*>(a.l.out)[m * a.l.ldo + n] = f2bf(v);
  }
}

template <typename F>
void with_epilogue(bool gelu, int res, bool out32, F f) {
  auto go = [&](auto g) {
    using std::integral_constant;
    if (res == 1) f(g, integral_constant<int, 1>{}, std::false_type{});
    else if (res == 2) f(g, integral_constant<int, 2>{}, std::true_type{});
    else if (out32) f(g, integral_constant<int, 0>{}, std::true_type{});
    else f(g, integral_constant<int, 0>{}, std::false_type{});
  };
  if (gelu) go(std::true_type{});
  else go(std::false_type{});
}

template <class C>
void launch_linear(const LinearI8& a, bool gelu, int res, bool out32, hipStream_t stream) {
  with_epilogue(gelu, res, out32, [&](auto g, auto r, auto o) {
    hipLaunchKernelGGL((linear_i8_kernel<C, decltype(g)::value, decltype(r)::value, decltype(o)::value>),
                       dim3((unsigned)a.ntiles), dim3(C::NT), 0, stream, a);
  });
}

// f(chunks of 512 columns in the registers)
template <typename F>
void with_chunks(int64_t K, F f) {
  if (K <= 512) f(std::integral_constant<int, 1>{});
  else if (K <= 1024) f(std::integral_constant<int, 2>{});
  else f(std::integral_constant<int, 4>{});
}

template <typename XT>
void launch_small(const SmallI8& a, bool gelu, int res, bool out32, hipStream_t stream) {
  const dim3 g((unsigned)cdiv(a.l.N, 16));
  const size_t lds = (size_t)a.l.M * a.lds_ld;
  with_epilogue(gelu, res, out32, [&](auto ge, auto re, auto o) {
    auto go = [&](auto nv) {
      hipLaunchKernelGGL((small_i8_kernel<XT, decltype(nv)::value, decltype(ge)::value, decltype(re)::value,
                                          decltype(o)::value>),
                         g, dim3(256), lds, stream, a);
    };
    if (a.gamma) {
      if constexpr (decltype(re)::value == 0 && !decltype(o)::value) with_chunks(a.l.K, go);
    } else {
      go(std::integral_constant<int, 0>{});
    }
  });
}

template <typename XT>
int quant_rows(const void* x, int64_t rows, int64_t K, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
               hipStream_t stream) {
  auto go = [&](auto nv) {
    hipLaunchKernelGGL((quant_rows_kernel<XT, decltype(nv)::value>), dim3((unsigned)cdiv(rows, 4)), dim3(256), 0, stream,
                       reinterpret_cast<const XT*>(x), rows, (int32_t)K, ldx, q, ldq, scale);
  };
  if (ldq <= 2048) with_chunks(ldq, go);
  else if (ldq <= 4096) go(std::integral_constant<int, 8>{});
  else go(std::integral_constant<int, 0>{});
  return check_launch("dph_quant_rows_i8");
}

template <typename XT>
int ln_quant(const DphLinearI8Args& a, hipStream_t stream) {
  with_chunks(a.K, [&](auto nv) {
    hipLaunchKernelGGL((ln_quant_kernel<XT, decltype(nv)::value>), dim3((unsigned)cdiv(a.M, 4)), dim3(256), 0, stream,
                       reinterpret_cast<const XT*>(a.x), a.ln_weight, a.ln_bias, a.M, (int32_t)a.K, a.ldx, a.ln_eps,
                       reinterpret_cast<bf16_t*>(a.norm_out), a.ld_norm, a.q, a.ldq, a.q_scale);
  });
  return check_launch("dph_linear_i8 (LayerNorm)");
}

constexpr int64_t I32MAX = 0x7fffffff;
constexpr int64_t ROWS_MAX = (int64_t)1 << 25;   // rows of one launch (a wave each: fewer than 2^32 threads)

}  // namespace
}  // namespace dph

using namespace dph;

extern "C" int dph_quant_rows_i8(const void* x, int x_f32, int64_t rows, int64_t K, int64_t ldx, int8_t* q, int64_t ldq,
                                 float* scale, hipStream_t stream) {
  DPH_REQUIRE(rows >= 0 && K >= 1, "dph_quant_rows_i8: rows >= 0 and K >= 1 (got %lld x %lld)", (long long)rows,
              (long long)K);
  if (rows == 0) return DPH_OK;
  DPH_REQUIRE(x && q && scale, "dph_quant_rows_i8: null pointer");
  DPH_REQUIRE(K <= DPH_I8_K_MAX && rows <= ROWS_MAX, "dph_quant_rows_i8: K up to %d, rows up to 2^25", DPH_I8_K_MAX);
  DPH_REQUIRE(ldx >= K || rows == 1, "dph_quant_rows_i8: rows overlap");
  DPH_REQUIRE(ldq >= K && ldq % 16 == 0 && ldq <= I32MAX && reinterpret_cast<uintptr_t>(q) % 16 == 0,
              "dph_quant_rows_i8: rows of q start 16 bytes apart or a multiple of it");
  return x_f32 ? quant_rows<float>(x, rows, K, ldx, q, ldq, scale, stream)
               : quant_rows<bf16_t>(x, rows, K, ldx, q, ldq, scale, stream);
}

// whether x (given, not its integers) goes through the kernel of up to 16 rows, which needs no q.  All its workgroups read
// x while some have written their part of out: where these lie over each other x is quantised first
static bool small_i8(const DphLinearI8Args& a) {
  if (!a.x || a.M > SMALL_M || a.M * small_ld(a.K) > SMALL_LDS || a.N <= 0) return false;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.x), o = reinterpret_cast<uintptr_t>(a.out);
  const int64_t nx = ((a.M - 1) * a.ldx + a.K) * (a.x_f32 ? 4 : 2),
                no = ((a.M - 1) * a.ldo + a.N) * (a.out_dtype == DPH_OUT_F32 ? 4 : 2);
  return !o || x + nx <= o || o + no <= x;
}

extern "C" int64_t dph_linear_i8_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N < 0 || K <= 0) return 0;
  DphLinearI8Args a = {};
  a.M = M, a.N = N, a.K = K, a.x = &a;
  return small_i8(a) ? 0 : M * (((K + 15) & ~(int64_t)15) + 4);
}

extern "C" int dph_linear_i8(const DphLinearI8Args* args, hipStream_t stream) {
  DPH_REQUIRE(args, "dph_linear_i8: null args");
  const DphLinearI8Args& a = *args;
  DPH_REQUIRE(a.M >= 0 && a.N >= 0 && a.K >= 1, "dph_linear_i8: M, N >= 0 and K >= 1");
  DPH_REQUIRE(a.M <= ROWS_MAX && a.N <= ROWS_MAX && a.K <= DPH_I8_K_MAX,
              "dph_linear_i8: M and N up to 2^25, K up to %d (32-bit sums)", DPH_I8_K_MAX);
  if (a.M == 0) return DPH_OK;
  DPH_REQUIRE(a.act == DPH_ACT_NONE || a.act == DPH_ACT_GELU, "dph_linear_i8: act is none or gelu");
  const bool out32 = a.out_dtype == DPH_OUT_F32;
  DPH_REQUIRE(out32 || a.out_dtype == DPH_OUT_BF16, "dph_linear_i8: out is bf16 or fp32");
  DPH_REQUIRE(!a.residual || (a.residual_f32 != 0) == out32, "dph_linear_i8: out has the residual's type");
  DPH_REQUIRE(!a.residual || a.ldr >= a.N || a.M == 1, "dph_linear_i8: rows of the residual overlap");
  const bool small = small_i8(a);
  if (!small) {
    DPH_REQUIRE(a.q && a.q_scale, "dph_linear_i8: null operand");
    DPH_REQUIRE(a.ldq >= a.K && a.ldq % 16 == 0 && reinterpret_cast<uintptr_t>(a.q) % 16 == 0,
                "dph_linear_i8: rows of q start 16 bytes apart or a multiple of it");
  }
  auto tiles = [&](int b) { return cdiv(a.M, b) * cdiv(a.N, b); };
  if (a.N > 0) {
    DPH_REQUIRE(a.w && a.w_scale && a.out, "dph_linear_i8: null operand");
    DPH_REQUIRE(a.ldw >= a.K && a.ldw % 16 == 0 && reinterpret_cast<uintptr_t>(a.w) % 16 == 0,
                "dph_linear_i8: rows of w start 16 bytes apart or a multiple of it");
    DPH_REQUIRE(a.ldo >= a.N || a.M == 1, "dph_linear_i8: rows of out overlap");
    DPH_REQUIRE((small || a.ldq < (1 << 23)) && a.ldw < (1 << 23),
                "dph_linear_i8: rows of q and w less than 2^23 bytes apart");
    DPH_REQUIRE(tiles(256) < (1 << 22), "dph_linear_i8: too many tiles");
  }
  if (a.x) {
    DPH_REQUIRE(a.ldx >= a.K || a.M == 1, "dph_linear_i8: rows of x overlap");
    if (a.ln_weight) {
      DPH_REQUIRE(a.ln_bias, "dph_linear_i8: LayerNorm without a bias");
      DPH_REQUIRE(a.K <= DPH_I8_LN_MAX, "dph_linear_i8: LayerNorm of up to %d columns", DPH_I8_LN_MAX);
      DPH_REQUIRE(!a.norm_out || a.ld_norm >= a.K, "dph_linear_i8: rows of norm_out overlap");
      DPH_REQUIRE(!a.residual && !out32, "dph_linear_i8: the LayerNorm form gives bf16 without a residual");
    }
    if (!small) {
      if (a.ln_weight) {
        DPH_REQUIRE(a.ldq <= (a.K <= 512 ? 512 : a.K <= 1024 ? 1024 : 2048), "dph_linear_i8: ldq of the LayerNorm form");
        DPH_TRY(a.x_f32 ? ln_quant<float>(a, stream) : ln_quant<bf16_t>(a, stream));
      } else {
        DPH_TRY(dph_quant_rows_i8(a.x, a.x_f32, a.M, a.K, a.ldx, a.q, a.ldq, a.q_scale, stream));
      }
    }
  }
  if (a.N == 0) return DPH_OK;
  const int res = a.residual ? (out32 ? 2 : 1) : 0;
  LinearI8 p{{reinterpret_cast<const char*>(a.q), a.ldq, (int32_t)a.M},
             {reinterpret_cast<const char*>(a.w), a.ldw, (int32_t)a.N},
             (int32_t)a.M, (int32_t)a.N, (int32_t)a.K, a.q_scale, a.w_scale, a.bias, a.residual, a.out, a.ldr, a.ldo,
             0, 0};
  const bool gelu = a.act == DPH_ACT_GELU;
  if (small) {
    SmallI8 sm{p, a.x, a.ldx, a.ln_weight, a.ln_bias, reinterpret_cast<bf16_t*>(a.norm_out), a.ld_norm, a.ln_eps,
               (int32_t)small_ld(a.K)};
    if (a.x_f32) launch_small<float>(sm, gelu, res, out32, stream);
    else launch_small<bf16_t>(sm, gelu, res, out32, stream);
    return check_launch("dph_linear_i8");
  }
  // Measured on tiles of 256 / 128 / 64, the product alone: 7984 x 1024 x 4096 62 / 45 / 66 us, 8192 x 8192 x 8192 398 / 518 us
  // / -, 7984 x 2304 x 768 32 / 24 / 36 us, 1497 x 768 x 1533 37 / 16 / 15 us
  auto go = [&](auto c) {
    using C = decltype(c);
    p.ntn = (int32_t)cdiv(a.N, C::BN);
    p.ntiles = (int32_t)tiles(C::BM);
    launch_linear<C>(p, gelu, res, out32, stream);
  };
  const int tile = mt::choose_tile(tiles(256), tiles(128), tiles(64));
  if (tile == 64) go(mt::C64{});
  else if (tile == 128) go(mt::C128{});
  else go(mt::C256{});
  return check_launch("dph_linear_i8");
}
