// Products in 8-bit integers with one scale a row of either operand (a token's, an output channel's):
//
//   y[m][n] = act( xs[m] ws[n] sum_k q[m][k] w[n][k] + bias[n] ) + residual[m][n]
//
// q[m][k] = x[m][k] / xs[m] to the nearest integer, ties to even, xs[m] = max_k |x[m][k]| (1 / 127) -- the activations are
// quantised on the way in, a row at a time, either as they stand or as the output of a LayerNorm.
#include "mfma_tile.h"

#include <stdlib.h>

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
  const bool odd = ((int)t & 1) != 0;
  if (a > h || (a == h && odd)) t += d > 0.f ? 1.f : -1.f;
  return (int)t;
}

template <typename XT>
__device__ __forceinline__ float ld1(const XT* p) {
  if constexpr (std::is_same_v<XT, float>) return *p;
  else return bf2f(*p);
}

// 8 consecutive elements, 16-byte aligned
__device__ __forceinline__ void ld8v(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void ld8v(const bf16_t* p, float (&v)[8]) {
  const uint4 r = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

template <bool VEC, typename XT>
__device__ __forceinline__ void load8(const XT* row, int c, int K, float (&v)[8]) {
  if (VEC && c + 8 <= K) {
    ld8v(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? ld1(row + c + i) : 0.f;
  }
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

__device__ __forceinline__ uint2 pack8(const float (&v)[8], float inv, float s) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i >> 2] |= ((uint32_t)quant1(v[i], inv, s) & 0xffu) << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}

// One wave a row: the largest |x|, then the integers (the row's second reading comes from the L2).  ldq is a multiple
// of 16 and the row's bytes from K on are written as zeros.
template <typename XT, bool VEC>
__global__ void __launch_bounds__(256) quant_rows_kernel(const XT* __restrict__ x, int64_t rows, int32_t K, int64_t ldx,
                                                         int8_t* __restrict__ q, int64_t ldq,
                                                         float* __restrict__ scale) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const XT* xr = x + r * ldx;
  uint32_t m = 0;
  for (int c = lane * 8; c < K; c += 512) {
    float v[8];
    load8<VEC>(xr, c, K, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  const float s = row_scale(wave_umax(m));
  const bool ok = s == s;
  const float inv = 1.0f / s;
  int8_t* qr = q + r * ldq;
  for (int c = lane * 8; c < ldq; c += 512) {
    float v[8];
    load8<VEC>(xr, c, K, v);
    *reinterpret_cast<uint2*>(qr + c) = ok ? pack8(v, inv, s) : make_uint2(0, 0);
  }
  if (lane == 0) scale[r] = s;
}

// LayerNorm of a row (fp32 two-pass statistics) quantised from its fp32 values, and the values themselves in bf16 where
// the residual branch wants them.  One wave a row; rows of up to 2048 columns stay in registers (NV chunks of 8 a lane).
template <typename XT, bool VEC, int NV>
__global__ void __launch_bounds__(256) ln_quant_kernel(const XT* __restrict__ x, const float* __restrict__ gamma,
                                                       const float* __restrict__ beta, int64_t rows, int32_t K,
                                                       int64_t ldx, float eps, bf16_t* __restrict__ y, int64_t ldy,
                                                       int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const XT* xr = x + r * ldx;
  float v[NV][8];
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load8<VEC>(xr, j * 512 + lane * 8, K, v[j]);
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
    load8<VEC>(gamma, c, K, g);
    load8<VEC>(beta, c, K, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[j][i] = c + i < K ? (v[j][i] - mean) * rstd * g[i] + b[i] : 0.f;
      m = max(m, __float_as_uint(v[j][i]) & 0x7fffffffu);
    }
    if (y) {
      bf16_t* yr = y + r * ldy + c;
      if (VEC && c + 8 <= K) {
        *reinterpret_cast<uint4*>(yr) = make_uint4(pack2bf(v[j][0], v[j][1]), pack2bf(v[j][2], v[j][3]),
                                                   pack2bf(v[j][4], v[j][5]), pack2bf(v[j][6], v[j][7]));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < K) yr[i] = f2bf(v[j][i]);
      }
    }
  }
  const float s = row_scale(wave_umax(m));
  const bool ok = s == s;
  const float inv = 1.0f / s;
  int8_t* qr = q + r * ldq;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * 512 + lane * 8;
    if (c < ldq) *reinterpret_cast<uint2*>(qr + c) = ok ? pack8(v[j], inv, s) : make_uint2(0, 0);
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
  int32_t vec;      // 4 consecutive columns of res and out are one aligned access
};

// RES: 0 none, 1 bf16, 2 fp32 (the output has the residual's type; without one it is bf16, or fp32 with OUT32)
template <class C, bool GELU, int RES, bool OUT32>
__device__ __forceinline__ void store_tile(const LinearI8& a, const mt::i32x4_t (&acc)[C::FM][C::FN], int mw, int nw,
                                           int lane) {
  const int ml = mw + (lane & 15), nl = nw + 4 * (lane >> 4);
  float ws[C::FN][4], bias[C::FN][4];
#pragma unroll
  for (int j = 0; j < C::FN; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = min(nl + 16 * j + r, a.N - 1);
      ws[j][r] = a.ws[n];
      bias[j][r] = a.bias ? a.bias[n] : 0.f;
    }
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    const int m = ml + 16 * i;
    if (m >= a.M) continue;
    const float xs = a.xs[m];
#pragma unroll
    for (int j = 0; j < C::FN; ++j) {
      const int n = nl + 16 * j;
      if (n >= a.N) continue;
      const int64_t o = (int64_t)m * a.ldo + n, ro = (int64_t)m * a.ldr + n;
      const bool vec = a.vec && n + 4 <= a.N;
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[r] = fmaf((float)acc[i][j][r] * xs, ws[j][r], bias[j][r]);
        if (GELU) v[r] = gelu_f(v[r]);
      }
      if constexpr (RES == 1) {
        const bf16_t* p = reinterpret_cast<const bf16_t*>(a.res) + ro;
        if (vec) {
          float t[4];
          ring::unpack_bf16x4(*reinterpret_cast<const uint2*>(p), t);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += t[r];
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += n + r < a.N ? bf2f(p[r]) : 0.f;
        }
      } else if constexpr (RES == 2) {
        const float* p = reinterpret_cast<const float*>(a.res) + ro;
        if (vec) {
          const float4 t = *reinterpret_cast<const float4*>(p);
          v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += n + r < a.N ? p[r] : 0.f;
        }
      }
      if constexpr (OUT32) {
        float* p = reinterpret_cast<float*>(a.out) + o;
        if (vec) {
          *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < a.N) p[r] = v[r];
        }
      } else {
        bf16_t* p = reinterpret_cast<bf16_t*>(a.out) + o;
        if (vec) {
          *reinterpret_cast<uint2*>(p) = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]));
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < a.N) p[r] = f2bf(v[r]);
        }
      }
    }
  }
}

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
  mt::product_of<mt::I8, C>(a.x, a.w, a.K, m0, n0, acc, smem, wave, lane, [&]() { mt::clear<mt::I8, C>(acc); });
  store_tile<C, GELU, RES, OUT32>(a, acc, m0 + wave / C::WC * C::WTM, n0 + wave % C::WC * C::WTN, lane);
}

template <class C>
void launch_linear(const LinearI8& a, bool gelu, int res, bool out32, hipStream_t stream) {
  const dim3 g((unsigned)a.ntiles), b(C::NT);
#define DPH_LIN(G, R, O) hipLaunchKernelGGL((linear_i8_kernel<C, G, R, O>), g, b, 0, stream, a)
  if (gelu) {
    if (res == 1) DPH_LIN(true, 1, false);
    else if (res == 2) DPH_LIN(true, 2, true);
    else if (out32) DPH_LIN(true, 0, true);
    else DPH_LIN(true, 0, false);
  } else {
    if (res == 1) DPH_LIN(false, 1, false);
    else if (res == 2) DPH_LIN(false, 2, true);
    else if (out32) DPH_LIN(false, 0, true);
    else DPH_LIN(false, 0, false);
  }
#undef DPH_LIN
}

template <typename XT>
int quant_rows(const void* x, int64_t rows, int64_t K, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
               hipStream_t stream) {
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * sizeof(XT) % 16 == 0;
  const dim3 g((unsigned)cdiv(rows, 4));
  const XT* xp = reinterpret_cast<const XT*>(x);
  if (vec) hipLaunchKernelGGL((quant_rows_kernel<XT, true>), g, dim3(256), 0, stream, xp, rows, (int32_t)K, ldx, q, ldq, scale);
  else hipLaunchKernelGGL((quant_rows_kernel<XT, false>), g, dim3(256), 0, stream, xp, rows, (int32_t)K, ldx, q, ldq, scale);
  return check_launch("dph_quant_rows_i8");
}

template <typename XT>
int ln_quant(const DphLinearI8Args& a, hipStream_t stream) {
  const uintptr_t al = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.ln_weight) |
                       reinterpret_cast<uintptr_t>(a.ln_bias) | reinterpret_cast<uintptr_t>(a.norm_out) |
                       (uintptr_t)(a.ldx * sizeof(XT)) | (uintptr_t)(a.norm_out ? a.ld_norm * 2 : 0);
  const bool vec = al % 16 == 0;
  const dim3 g((unsigned)cdiv(a.M, 4));
  auto go = [&](auto vc, auto nv) {
    hipLaunchKernelGGL((ln_quant_kernel<XT, decltype(vc)::value, decltype(nv)::value>), g, dim3(256), 0, stream,
                       reinterpret_cast<const XT*>(a.x), a.ln_weight, a.ln_bias, a.M, (int32_t)a.K, a.ldx, a.ln_eps,
                       reinterpret_cast<bf16_t*>(a.norm_out), a.ld_norm, a.q, a.ldq, a.q_scale);
  };
  auto nvs = [&](auto vc) {
    if (a.K <= 512) go(vc, std::integral_constant<int, 1>{});
    else if (a.K <= 1024) go(vc, std::integral_constant<int, 2>{});
    else go(vc, std::integral_constant<int, 4>{});
  };
  if (vec) nvs(std::true_type{});
  else nvs(std::false_type{});
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

extern "C" int dph_linear_i8(const DphLinearI8Args* args, hipStream_t stream) {
  DPH_REQUIRE(args, "dph_linear_i8: null args");
  const DphLinearI8Args& a = *args;
  DPH_REQUIRE(a.M >= 0 && a.N >= 0 && a.K >= 1, "dph_linear_i8: M, N >= 0 and K >= 1");
  DPH_REQUIRE(a.M <= ROWS_MAX && a.N <= ROWS_MAX && a.K <= DPH_I8_K_MAX,
              "dph_linear_i8: M and N up to 2^25, K up to %d (32-bit sums)", DPH_I8_K_MAX);
  if (a.M == 0) return DPH_OK;
  DPH_REQUIRE(a.q && a.q_scale, "dph_linear_i8: null operand");
  DPH_REQUIRE(a.ldq >= a.K && a.ldq % 16 == 0 && reinterpret_cast<uintptr_t>(a.q) % 16 == 0,
              "dph_linear_i8: rows of q start 16 bytes apart or a multiple of it");
  DPH_REQUIRE(a.act == DPH_ACT_NONE || a.act == DPH_ACT_GELU, "dph_linear_i8: act is none or gelu");
  const bool out32 = a.out_dtype == DPH_OUT_F32;
  DPH_REQUIRE(out32 || a.out_dtype == DPH_OUT_BF16, "dph_linear_i8: out is bf16 or fp32");
  DPH_REQUIRE(!a.residual || (a.residual_f32 != 0) == out32, "dph_linear_i8: out has the residual's type");
  if (a.x) {
    DPH_REQUIRE(a.ldx >= a.K || a.M == 1, "dph_linear_i8: rows of x overlap");
    if (a.ln_weight) {
      DPH_REQUIRE(a.ln_bias, "dph_linear_i8: LayerNorm without a bias");
      DPH_REQUIRE(a.K <= DPH_I8_LN_MAX, "dph_linear_i8: LayerNorm of up to %d columns", DPH_I8_LN_MAX);
      DPH_REQUIRE(a.ldq <= (a.K <= 512 ? 512 : a.K <= 1024 ? 1024 : 2048), "dph_linear_i8: ldq of the LayerNorm form");
      DPH_TRY(a.x_f32 ? ln_quant<float>(a, stream) : ln_quant<bf16_t>(a, stream));
    } else {
      DPH_TRY(dph_quant_rows_i8(a.x, a.x_f32, a.M, a.K, a.ldx, a.q, a.ldq, a.q_scale, stream));
    }
  }
  if (a.N == 0) return DPH_OK;
  DPH_REQUIRE(a.w && a.w_scale && a.out, "dph_linear_i8: null operand");
  DPH_REQUIRE(a.ldw >= a.K && a.ldw % 16 == 0 && reinterpret_cast<uintptr_t>(a.w) % 16 == 0,
              "dph_linear_i8: rows of w start 16 bytes apart or a multiple of it");
  DPH_REQUIRE(a.ldo >= a.N || a.M == 1, "dph_linear_i8: rows of out overlap");
  DPH_REQUIRE(a.ldq < (1 << 23) && a.ldw < (1 << 23), "dph_linear_i8: rows of q and w less than 2^23 bytes apart");
  const int es = out32 ? 4 : 2;
  const uintptr_t al = reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.residual) |
                       (uintptr_t)(a.ldo * es) | (uintptr_t)(a.residual ? a.ldr * es : 0);
  LinearI8 p{{reinterpret_cast<const char*>(a.q), a.ldq, (int32_t)a.M},
             {reinterpret_cast<const char*>(a.w), a.ldw, (int32_t)a.N},
             (int32_t)a.M, (int32_t)a.N, (int32_t)a.K, a.q_scale, a.w_scale, a.bias, a.residual, a.out, a.ldr, a.ldo,
             0, 0, al % (4 * es) == 0};
  auto go = [&](auto c) -> int {
    using C = decltype(c);
    const int64_t ntm = cdiv(a.M, C::BM), ntn = cdiv(a.N, C::BN);
    DPH_REQUIRE(ntm * ntn < (1 << 22), "dph_linear_i8: too many tiles");
    p.ntn = (int32_t)ntn;
    p.ntiles = (int32_t)(ntm * ntn);
    launch_linear<C>(p, a.act == DPH_ACT_GELU, a.residual ? (out32 ? 2 : 1) : 0, out32, stream);
    return DPH_OK;
  };
  const char* ev = getenv("DPH_I8_TILE");
  const int sel = ev ? atoi(ev) : 0;
  if (sel == 0) DPH_TRY(go(mt::Tile<128, 128, 2, 2, 2>{}));
  if (sel == 1) DPH_TRY(go(mt::Duo<256, 256, 1>{}));
  if (sel == 2) DPH_TRY(go(mt::Duo<128, 256, 1>{}));
  if (sel == 3) DPH_TRY(go(mt::Duo<128, 192, 2>{}));
  if (sel == 4) DPH_TRY(go(mt::Duo<128, 128, 2>{}));
  if (sel == 5) DPH_TRY(go(mt::Tile<64, 64, 2, 2, 4>{}));
  if (sel == 6) DPH_TRY(go(mt::Duo<256, 128, 1>{}));
  if (sel == 7) DPH_TRY(go(mt::Duo<128, 192, 1>{}));
  return check_launch("dph_linear_i8");
}
