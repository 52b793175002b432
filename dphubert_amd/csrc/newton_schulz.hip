// Orthogonal factors of a list of matrices by the quintic Newton-Schulz iteration (Muon's update direction):
//
//   X0 = G / (|G|_F + eps);   A = X X^T;   X <- a X + (b A + c A^2) X        (X [m][n], m <= n; transposed otherwise)
//
// Every step is three matrix products over all matrices at once (a launch each, whatever the shapes): the Gram matrix
// and its square, of which only the tiles on and below the diagonal are computed and the others mirrored, and the
// product with X.
//
// Numbers.  The operands are fp16, the sums fp32.  fp16 has 8 times bf16's resolution and its range suffices: X's
// singular values stay near or below 1, and X is held times a power of two s that puts its mean entry at about 1/4.
// Two things keep the operands' rounding (2^-12) from growing through the steps; rounding errors of the result against
// 64 bits (2-norm, 5 steps, sizes 64 to 1533, of noise / of a few directions 100 times above the rest): plain fp16
// 1.3e-3 / 1.1e-2, as built 0.8e-3 / 1.3e-3, bf16 in place of fp16 1.0e-2 / 9e-2.
//   * While singular values grow, a X dominates the step: X is held in 16 bits and more for that term (fp16, and what it
//     leaves in e4m3), so weak directions are not lost in the rounding of strong ones.  The products read the fp16 alone.
//   * In the last two steps the singular values are near 1 and a X + b A X + c A^2 X cancel by a factor of 5.  There the
//     polynomial is expanded about d = 1:  E = A - d I,  F = (b + 2 c d) E + c E^2,  X <- (a + b d + c d^2) X + F X,
//     the same products on numbers near 0, whose roundings are small (the last coefficient is put into F's diagonal).
// In large matrices an operand's roundings average out; up to NS_SPLIT rows they need not (a 1 x 1 matrix is off by
// 8e-3), and there every operand is two fp16 and every product three: h h + l h + h l.  Such matrices are a few tiles:
// launches, not products, set their time.
//
// Layout.  What is stored is Y = X^T ([n][m], the long side first), and only that: Y F has both operands contiguous
// along k, and the Gram matrix reads Y through the transposing LDS read.  A step then moves Y in and out once (and its 8
// more bits while they are held) -- with a transposed copy kept, and 16 bits more, the update of 24 matrices of 4096 x
// 1024 took 487 us instead of 262.
//
// What bounds it.  24 matrices of 1024 x 4096, a step: Gram matrix 133 us (103 GFLOP, 240 tiles: one round of CUs, 55 % of
// the matrix cores' cycles in use), square 45 us (26 GFLOP), product with Y 254 us (206 GFLOP and 600 MB) while the 8 bits
// are held and 191 us after (400 MB): reading Y, products and writing take turns in a CU, whose registers hold one tile's
// sums and nothing of the next.  (Workgroups started in a staggered order, so that some multiply while others store, gained
// what the staggering cost.)  One matrix of 768 x 768: 17 launches of 5 to 8 us, each a chain of 12 latencies.
#include "mfma_tile.h"

#include <type_traits>

namespace dph {
namespace {

typedef uint16_t f16_t;
constexpr int NS_GROUPS = 16;      // groups of equal shapes in one launch
constexpr int NS_MATS = 64;        // matrices of one packing launch
constexpr float NS_E = 64.f;       // E and F are held times 64 (entries of a few 1e-5 stay normal fp16 numbers)
constexpr int NS_PARTS = 64;       // partial sums of a matrix's squares
constexpr int NS_SPLIT = 128;      // rows up to which all operands are held in two parts
// The Gram matrix of few rows and many columns is few tiles and a long sum: up to NS_DEEP rows, from NS_LONG columns on,
// the sum is cut into parts of a fixed number of steps (by the shape alone, so that a result does not depend on what else
// is in the list), whose tiles are added in their order by a launch of their own.  4 matrices of 128 x 4000: 617 -> 195 us.
constexpr int NS_DEEP = 256, NS_LONG = 1024;

__device__ __forceinline__ f16_t f2h(float v) { return __builtin_bit_cast(f16_t, (_Float16)v); }
__device__ __forceinline__ float h2f(f16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
__device__ __forceinline__ uint32_t pack2h(float a, float b) {
  typedef __attribute__((ext_vector_type(2))) float f2;
  typedef __attribute__((ext_vector_type(2))) _Float16 h2;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), h2));
}
__device__ __forceinline__ void unpack4h(uint2 r, float* v) {
  v[0] = h2f((f16_t)(r.x & 0xffff)); v[1] = h2f((f16_t)(r.x >> 16));
  v[2] = h2f((f16_t)(r.y & 0xffff)); v[3] = h2f((f16_t)(r.y >> 16));
}

// what 4 numbers have beyond their fp16 halves h, as fp16
__device__ __forceinline__ uint2 low4h(const float* v, uint2 h) {
  float q[4];
  unpack4h(h, q);
  return make_uint2(pack2h(v[0] - q[0], v[1] - q[1]), pack2h(v[2] - q[2], v[3] - q[3]));
}
// the same in e4m3, times 2^13: half a place of a mean entry (1/4) counts 1/2; what entries above 900 times that leave is
// cut off at e4m3's 448
constexpr float LO_UP = 8192.f;
__device__ __forceinline__ uint32_t low4q(const float* v, uint2 h) {
  float q[4];
  unpack4h(h, q);
#pragma unroll
  for (int r = 0; r < 4; ++r) q[r] = fminf(fmaxf(fmaf(q[r], -LO_UP, v[r] * LO_UP), -448.f), 448.f);
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
}
// v = (v + what w holds) scale
__device__ __forceinline__ void add_low4q(float* v, uint32_t w, float scale) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  const float l = scale * (1.f / LO_UP);
  v[0] = fmaf(v[0], scale, a[0] * l);
  v[1] = fmaf(v[1], scale, a[1] * l);
  v[2] = fmaf(v[2], scale, b[0] * l);
  v[3] = fmaf(v[3], scale, b[1] * l);
}

// Matrices of one shape: cnt of them, Y n x m (m <= n) in rows padded with zeros to multiples of 64 (np, mp)
struct Group {
  int32_t m, n, mp, np, cnt, wide;    // wide: the caller's matrices are m x n
  float s;                            // Y is held times s
  int32_t pad;
  char *y[2], *lo, *yl[2];            // [cnt][np][mp]: fp16 x 2, then e4m3, or (split) two fp16 halves more
  char *e, *f, *el, *fl;              // [cnt][mp][mp]; the lower halves (split) or null
  double* part;                       // [cnt][NS_PARTS]
  bf16_t* out;                        // [cnt] matrices as the caller has them, dense
  float* slab;                        // [cnt][tiles of the Gram matrix][parts][64 x 64] sums
  int32_t parts, part_steps;          // of the Gram matrix's sum (1: none)
};
struct Groups {
  int32_t ng;
  int32_t first[NS_GROUPS + 1];       // first tile of each group
  Group g[NS_GROUPS];
};
struct Mat {
  const void* p;
  int64_t ns, ms;                     // strides of Y's row and column index; one of them is 1
  int32_t group, index, first, pad;   // group, place in it, first block of the launch
};
struct Mats {
  int32_t n, pad;
  Mat m[NS_MATS];
};
struct Step {
  float d, fe, fq, mu, fd; // E = A - d I;  F = fe E + fq E^2 + fd I;  Y <- mu Y + Y F
  int32_t reverse;         // tiles from the last to the first
  int32_t cur;             // which y is read
  int32_t lo_out;          // Y's 8 bits more are written (they are read where mu is not 0)
};
struct PackGroup {
  int32_t m, n, mp, np, in_f32;
  float s;
  char *y, *lo, *yl;
  double* part;
};
struct PackGroups {
  PackGroup g[NS_GROUPS];
};
static_assert(sizeof(Groups) + sizeof(Step) <= 4096 && sizeof(Mats) + sizeof(PackGroups) + 8 <= 4096, "kernel arguments");

__device__ __forceinline__ float ldg(const void* p, int64_t i, int f32) {
  return f32 ? reinterpret_cast<const float*>(p)[i] : bf2f(reinterpret_cast<const bf16_t*>(p)[i]);
}

__device__ __forceinline__ int find_mat(const Mats& a, int b) {
  int k = 0;
  while (k + 1 < a.n && a.m[k + 1].first <= b) ++k;
  return k;
}

// Sums of squares in 64 bits, NS_PARTS parts of a matrix, added in a fixed order later.  A matrix without gaps is read
// as one run of 16-byte vectors, another line by line.  Bound by memory: 403 MB in 93 us, 4.3 TB/s.
__global__ void __launch_bounds__(256) ns_sumsq_kernel(const Mats a, const PackGroups pg) {
  const int k = find_mat(a, (int)blockIdx.x);
  const Mat& t = a.m[k];
  const PackGroup& g = pg.g[t.group];
  const int part = (int)blockIdx.x - t.first;
  const bool by_n = t.ms == 1;
  const int64_t lines = by_n ? g.n : g.m, len = by_n ? g.m : g.n, gap = by_n ? t.ns : t.ms;
  const int esize = g.in_f32 ? 4 : 2, ve = 16 / esize;
  double s0 = 0.0, s1 = 0.0;
  auto add4 = [&](float4 v) {
    s0 += (double)v.x * v.x + (double)v.y * v.y;
    s1 += (double)v.z * v.z + (double)v.w * v.w;
  };
  if (gap == len && (reinterpret_cast<uintptr_t>(t.p) & 15) == 0) {
    const int64_t total = lines * len, nv = total / ve, per = cdiv(nv, NS_PARTS);
    const int64_t i1 = min(nv, (part + 1) * per);
    const uint4* p = reinterpret_cast<const uint4*>(t.p);
    auto add = [&](uint4 r) {
      if (g.in_f32) {
        add4(make_float4(__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z), __uint_as_float(r.w)));
      } else {
        add4(make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                         __uint_as_float(r.y & 0xffff0000u)));
        add4(make_float4(__uint_as_float(r.z << 16), __uint_as_float(r.z & 0xffff0000u), __uint_as_float(r.w << 16),
                         __uint_as_float(r.w & 0xffff0000u)));
      }
    };
    int64_t i = part * per + threadIdx.x;
    for (; i + 768 < i1; i += 1024) {
      const uint4 r0 = p[i], r1 = p[i + 256], r2 = p[i + 512], r3 = p[i + 768];
      add(r0);
      add(r1);
      add(r2);
      add(r3);
    }
    for (; i < i1; i += 256) add(p[i]);
    if (part == NS_PARTS - 1)
      for (int64_t q = nv * ve + threadIdx.x; q < total; q += 256) {
        const double v = ldg(t.p, q, g.in_f32);
        s0 += v * v;
      }
  } else {
    for (int64_t l = part; l < lines; l += NS_PARTS)
      for (int64_t q = threadIdx.x; q < len; q += 256) {
        const double v = ldg(t.p, l * gap + q, g.in_f32);
        s0 += v * v;
      }
  }
  double s = s0 + s1;
  __shared__ double red[4];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) g.part[(int64_t)t.index * NS_PARTS + part] = (red[0] + red[1]) + (red[2] + red[3]);
}

// Y0, 64 x 64 tiles through the LDS; reads run along whichever stride of the input is 1.  Bound by memory: 403 MB read and
// 302 written in 123 us, 5.7 TB/s.
__global__ void __launch_bounds__(256) ns_pack_kernel(const Mats a, const PackGroups pg, float eps) {
  __shared__ float tile[64][65];
  __shared__ float scale;                // s / (|G| + eps) = scale 2^up: as one fp32 number it overflows for the smallest G
  __shared__ int up;
  const int k = find_mat(a, (int)blockIdx.x);
  const Mat& t = a.m[k];
  const PackGroup& g = pg.g[t.group];
  if (threadIdx.x < 64) {
    double s = g.part[(int64_t)t.index * NS_PARTS + threadIdx.x];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (threadIdx.x == 0) {
      int e;
      scale = (float)frexp((double)g.s / (sqrt(s) + (double)eps), &e);
      up = e;
    }
  }
  const int b = (int)blockIdx.x - t.first, tm = g.mp >> 6;
  const int r0 = b / tm * 64, c0 = b % tm * 64;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  float in[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = r0 + (t.ms == 1 ? 4 * i + ty : tx), c = c0 + (t.ms == 1 ? tx : 4 * i + ty);
    in[i] = r < g.n && c < g.m ? ldg(t.p, r * t.ns + c * t.ms, g.in_f32) : 0.f;
  }
  __syncthreads();
  const float sc = scale;
  const int e = up;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float v = ldexpf(in[i], e) * sc;
    if (t.ms == 1) tile[4 * i + ty][tx] = v;
    else tile[tx][4 * i + ty] = v;
  }
  __syncthreads();
  const int64_t mat = (int64_t)t.index * g.np * g.mp;
  const int x4 = (threadIdx.x & 15) * 4;
#pragma unroll
  for (int i = threadIdx.x >> 4; i < 64; i += 16) {
    const float v[4] = {tile[i][x4], tile[i][x4 + 1], tile[i][x4 + 2], tile[i][x4 + 3]};
    const int64_t o = mat + (int64_t)(r0 + i) * g.mp + c0 + x4;
    const uint2 h = make_uint2(pack2h(v[0], v[1]), pack2h(v[2], v[3]));
    *reinterpret_cast<uint2*>(g.y + 2 * o) = h;
    if (g.yl) *reinterpret_cast<uint2*>(g.yl + 2 * o) = low4h(v, h);
    else *reinterpret_cast<uint32_t*>(g.lo + o) = low4q(v, h);
  }
}

// ---- the products -------------------------------------------------------------------------------------------------
enum { GRAM, POLY, UPDATE, LAST };

// 4 x 4 transpose inside a quad of lanes: lane q of the quad has element (row q, column r) as the r-th of 4 16-bit
// numbers and leaves with (row r, column q)
__device__ __forceinline__ uint2 quad_transpose(uint2 x, int lane) {
  // (byte permutes with a lane's own selector: written as conditions, they are compiled to branches)
  const uint32_t s1 = lane & 1 ? 0x03020706u : 0x05040100u, s2 = lane & 2 ? 0x07060504u : 0x03020100u;
  const uint32_t y0 = (uint32_t)__builtin_amdgcn_mov_dpp((int)x.x, 0xb1, 0xf, 0xf, true);   // lane ^ 1
  const uint32_t y1 = (uint32_t)__builtin_amdgcn_mov_dpp((int)x.y, 0xb1, 0xf, 0xf, true);
  const uint32_t a0 = __builtin_amdgcn_perm(y0, x.x, s1), a1 = __builtin_amdgcn_perm(y1, x.y, s1);
  const uint32_t b0 = (uint32_t)__builtin_amdgcn_mov_dpp((int)a0, 0x4e, 0xf, 0xf, true);    // lane ^ 2
  const uint32_t b1 = (uint32_t)__builtin_amdgcn_mov_dpp((int)a1, 0x4e, 0xf, 0xf, true);
  return make_uint2(__builtin_amdgcn_perm(b1, a0, s2), __builtin_amdgcn_perm(a1, b0, s2));
}

// FINISH: the Gram matrix's parts are added, and no product is made
template <int KIND, bool SPLIT, class C, bool FINISH>
__global__ void __launch_bounds__(C::NT, C::WPE) ns_product_kernel(const Groups gs, const Step st) {
  __shared__ __align__(16) char smem[C::LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // every other launch goes through the matrices backwards: it starts with what the last one wrote last, which the
  // caches still hold (each XCD keeps its own matrices: its L2 has them)
  int t = mt::xcd_tile((int)blockIdx.x, (int)gridDim.x, st.reverse != 0);
  int k = 0;
  while (k + 1 < gs.ng && gs.first[k + 1] <= t) ++k;
  const Group& g = gs.g[k];
  t -= gs.first[k];
  constexpr bool SYM = KIND == GRAM || KIND == POLY;
  using T = std::conditional_t<KIND == GRAM, mt::F16T, mt::F16>;
  int ti, tj, z, kp = 0;
  float* slab = nullptr;
  constexpr bool PARTS = KIND == GRAM && C::BM == 64 && C::BN == 64;
  if (SYM) {
    static_assert(!SYM || C::BM == C::BN, "square tiles");
    const int tm = (g.m + C::BM - 1) / C::BM, per = tm * (tm + 1) / 2;
    if (PARTS && g.parts > 1) {
      slab = g.slab + (int64_t)t * (FINISH ? g.parts : 1) * 4096;
      if (!FINISH) {
        kp = t % g.parts;
        t /= g.parts;
      }
    }
    z = t / per;
    t -= z * per;
    ti = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > t) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    tj = t - ti * (ti + 1) / 2;
  } else {
    const int tm = (g.m + C::BN - 1) / C::BN, tn = (g.n + C::BM - 1) / C::BM, per = tm * tn;
    z = t / per;
    t -= z * per;
    ti = t / tm;         // (consecutive tiles share rows of Y)
    tj = t % tm;
  }
  // the last product in the caller's order: a wide matrix is F Y^T (the operands change places), so that a lane has columns
  // of it next to each other
  const bool flip = KIND == LAST && g.wide;
  if (flip) {
    static_assert(KIND != LAST || C::BM == C::BN, "square tiles");
    const int x = ti;
    ti = tj, tj = x;
  }
  const int m0 = ti * C::BM, n0 = tj * C::BN;
  const int64_t yoff = (int64_t)z * g.np * g.mp * 2, eoff = (int64_t)z * g.mp * g.mp * 2;
  int kbytes = (KIND == GRAM ? g.np : g.mp) * 2;
  const int64_t ld = (int64_t)g.mp * 2;
  int64_t koff = 0;                   // bytes of the part's first k-row
  if (PARTS && slab) {
    koff = (int64_t)kp * g.part_steps * 64 * ld;
    kbytes = min(g.part_steps * 128, kbytes - kp * g.part_steps * 128);
  }
  using V = mt::Strip<C::FN, C::FN % 4 == 0 ? 16 : 8>;
  constexpr int NV = 4 * C::FN;
  f32x4_t acc[C::FM][C::FN];
  const int mw = m0 + wave / C::WC * C::WTM + (lane & 15), nw = n0 + wave % C::WC * C::WTN;
  [[maybe_unused]] const int M = SYM ? g.mp : g.np, N = g.mp;      // (what lies past m and n is zero, and stays zero)
  // the sums start from 0, or from mu Y, whose rows are about to be read as an operand anyway.  All its reads are asked for
  // before the first is used, and rows past the end read the last one instead of none (a read inside a branch is waited
  // for there, 32 latencies one after the other: all steps of 24 matrices of 1024 x 4096 took 2546 us instead of 2260)
  auto init = [&]() {
    if constexpr (KIND != UPDATE) {
      mt::clear<T, C>(acc);
    } else if (st.mu == 0.f) {
      mt::clear<T, C>(acc);
    } else {
      const float mu = st.mu * NS_E;
      using Low = std::conditional_t<SPLIT, uint4, uint2>;
      uint4 h[C::FM][NV / 8];
      Low l[C::FM][NV / 8];
#pragma unroll
      for (int i = 0; i < C::FM; ++i) {
        const int64_t row = yoff / 2 + (int64_t)min(mw + 16 * i, M - 1) * N;
#pragma unroll
        for (int c = 0; c < NV; c += 8) {
          const int64_t o = row + min(nw + V::col(c / V::W, lane), N - V::W) + c % V::W;
          h[i][c / 8] = *reinterpret_cast<const uint4*>(g.y[st.cur] + 2 * o);
          if constexpr (SPLIT) l[i][c / 8] = *reinterpret_cast<const uint4*>(g.yl[st.cur] + 2 * o);
          else l[i][c / 8] = *reinterpret_cast<const uint2*>(g.lo + o);
        }
      }
#pragma unroll
      for (int i = 0; i < C::FM; ++i) {
        float x[NV];
#pragma unroll
        for (int c = 0; c < NV; c += 8) {
          const uint4 hi = h[i][c / 8];
          const Low lo = l[i][c / 8];
          unpack4h(make_uint2(hi.x, hi.y), x + c);
          unpack4h(make_uint2(hi.z, hi.w), x + c + 4);
          if constexpr (SPLIT) {
            float f[8];
            unpack4h(make_uint2(lo.x, lo.y), f);
            unpack4h(make_uint2(lo.z, lo.w), f + 4);
#pragma unroll
            for (int r = 0; r < 8; ++r) x[c + r] = (x[c + r] + f[r]) * mu;
          } else {
            add_low4q(x + c, lo.x, mu);
            add_low4q(x + c + 4, lo.y, mu);
          }
        }
        uint32_t b[NV];
#pragma unroll
        for (int r = 0; r < NV; ++r) b[r] = __float_as_uint(x[r]);
        V::exchange(b);
#pragma unroll
        for (int r = 0; r < NV; ++r) acc[i][r >> 2][r & 3] = __uint_as_float(b[r]);
      }
    }
  };
  const auto at = [&](int i, int j) { return ((wave * C::FM + i) * C::FN + j) * 256 + lane * 4; };   // in a part's tile
  if constexpr (FINISH) {
    init();
    for (int p = 0; p < g.parts; ++p)
#pragma unroll
      for (int i = 0; i < C::FM; ++i)
#pragma unroll
        for (int j = 0; j < C::FN; ++j) acc[i][j] += *reinterpret_cast<const f32x4_t*>(slab + (int64_t)p * 4096 + at(i, j));
  }
#pragma unroll 1
  for (int part = 0; part < (FINISH ? 0 : SPLIT ? 3 : 1); ++part) {   // h h, l h, h l
    const bool la = part == 1, lb = part == 2;
    mt::Rows A, B;
    if constexpr (KIND == GRAM) {
      A = mt::Rows{(la ? g.yl[st.cur] : g.y[st.cur]) + yoff + koff, ld, g.mp};
      B = mt::Rows{(lb ? g.yl[st.cur] : g.y[st.cur]) + yoff + koff, ld, g.mp};
    } else if constexpr (KIND == POLY) {
      A = mt::Rows{(la ? g.el : g.e) + eoff, ld, g.mp};
      B = mt::Rows{(lb ? g.el : g.e) + eoff, ld, g.mp};
    } else {
      A = mt::Rows{(la ? g.yl[st.cur] : g.y[st.cur]) + yoff, ld, g.np};
      B = mt::Rows{(lb ? g.fl : g.f) + eoff, ld, g.mp};
      if (flip) {
        const mt::Rows x = A;
        A = B, B = x;
      }
    }
    mt::product_of<T, C>(A, B, kbytes, m0, n0, acc, smem, wave, lane, [&]() {
      if (!SPLIT || part == 0) init();
    });
  }
  if (PARTS && !FINISH && slab) {
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int j = 0; j < C::FN; ++j) *reinterpret_cast<f32x4_t*>(slab + at(i, j)) = acc[i][j];
    return;
  }

  // (the lane anew: what init() worked out from it is not kept through the product, where every register is taken)
  int le = lane;
  asm volatile("" : "+v"(le));
  const int me = m0 + wave / C::WC * C::WTM + (le & 15);
  // (E, like Y above: all of the tile before the first store)
  constexpr int NE = KIND == POLY ? NV / 4 : 1;
  uint2 e_hi[C::FM][NE], e_lo[C::FM][SPLIT ? NE : 1];
  if constexpr (KIND == POLY) {
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int c = 0; c < NV; c += 4) {
        const int64_t o = (int64_t)min(me + 16 * i, M - 1) * N + min(nw + V::col(c / V::W, le), N - V::W) + c % V::W;
        e_hi[i][c / 4] = *reinterpret_cast<const uint2*>(g.e + eoff + o * 2);
        if constexpr (SPLIT) e_lo[i][c / 4] = *reinterpret_cast<const uint2*>(g.el + eoff + o * 2);
      }
  }
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    const int m = me + 16 * i;
    uint32_t b[NV];
#pragma unroll
    for (int r = 0; r < NV; ++r) b[r] = __float_as_uint(acc[i][r >> 2][r & 3]);
    V::exchange(b);
#pragma unroll
    for (int q = 0; q < V::NG; ++q) {
      const int n0q = nw + V::col(q, le);
      [[maybe_unused]] const bool in = m < M && n0q < N;
      float v[V::W];
      uint2 h[V::W / 4];
      [[maybe_unused]] uint2 l[V::W / 4];
#pragma unroll
      for (int r = 0; r < V::W; ++r) v[r] = __uint_as_float(b[V::W * q + r]);
      if constexpr (SYM) {
        char* to = (KIND == GRAM ? g.e : g.f) + eoff;
        char* tl = (KIND == GRAM ? g.el : g.fl) + eoff;
        const int64_t o = (int64_t)m * N + n0q;
        if constexpr (KIND == GRAM) {
          const float sc = NS_E / (g.s * g.s);
#pragma unroll
          for (int r = 0; r < V::W; ++r) v[r] *= sc;
        } else {
#pragma unroll
          for (int r = 0; r < V::W; ++r) v[r] *= st.fq / NS_E;
#pragma unroll
          for (int c = 0; c < V::W; c += 4) {
            float e[4];
            unpack4h(e_hi[i][(V::W * q + c) / 4], e);
            if constexpr (SPLIT) {
              float lo[4];
              unpack4h(e_lo[i][(V::W * q + c) / 4], lo);
#pragma unroll
              for (int r = 0; r < 4; ++r) e[r] += lo[r];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) v[c + r] += st.fe * e[r];
          }
        }
        if (ti == tj) {
          const uint32_t diag = __float_as_uint(m < g.m ? NS_E * (KIND == GRAM ? -st.d : st.fd) : 0.f);
#pragma unroll
          for (int r = 0; r < V::W; ++r) v[r] += __uint_as_float(diag & -(uint32_t)(m == n0q + r));
        }
#pragma unroll
        for (int c = 0; c < V::W / 4; ++c) {
          h[c] = make_uint2(pack2h(v[4 * c], v[4 * c + 1]), pack2h(v[4 * c + 2], v[4 * c + 3]));
          if constexpr (SPLIT) l[c] = low4h(v + 4 * c, h[c]);
        }
        // a tile below the diagonal is stored a second time, transposed
        uint2 ht[V::W / 4], lt[V::W / 4];
        const int64_t ot = (int64_t)(n0q + (le & 3)) * M + (m & ~3);
        if (ti != tj) {
#pragma unroll
          for (int c = 0; c < V::W / 4; ++c) {
            ht[c] = quad_transpose(h[c], le);
            if constexpr (SPLIT) lt[c] = quad_transpose(l[c], le);
          }
        }
        if (in) {
#pragma unroll
          for (int c = 0; c < V::W / 4; c += 2) {
            *reinterpret_cast<uint4*>(to + (o + 4 * c) * 2) = make_uint4(h[c].x, h[c].y, h[c + 1].x, h[c + 1].y);
            if constexpr (SPLIT)
              *reinterpret_cast<uint4*>(tl + (o + 4 * c) * 2) = make_uint4(l[c].x, l[c].y, l[c + 1].x, l[c + 1].y);
          }
          if (ti != tj) {
#pragma unroll
            for (int c = 0; c < V::W / 4; ++c) {
              *reinterpret_cast<uint2*>(to + (ot + 4 * c * (int64_t)M) * 2) = ht[c];
              if constexpr (SPLIT) *reinterpret_cast<uint2*>(tl + (ot + 4 * c * (int64_t)M) * 2) = lt[c];
            }
          }
        }
      } else if constexpr (KIND == UPDATE) {
        if (in) {
          const int64_t o = yoff / 2 + (int64_t)m * N + n0q;
#pragma unroll
          for (int r = 0; r < V::W; ++r) v[r] *= 1.f / NS_E;
#pragma unroll
          for (int c = 0; c < V::W / 4; ++c) {
            h[c] = make_uint2(pack2h(v[4 * c], v[4 * c + 1]), pack2h(v[4 * c + 2], v[4 * c + 3]));
            if constexpr (SPLIT) *reinterpret_cast<uint2*>(g.yl[st.cur ^ 1] + 2 * (o + 4 * c)) = low4h(v + 4 * c, h[c]);
            else if (st.lo_out) l[c].x = low4q(v + 4 * c, h[c]);
          }
#pragma unroll
          for (int c = 0; c < V::W / 4; c += 2)
            *reinterpret_cast<uint4*>(g.y[st.cur ^ 1] + 2 * (o + 4 * c)) =
                make_uint4(h[c].x, h[c].y, h[c + 1].x, h[c + 1].y);
          if (!SPLIT && st.lo_out) {
            if constexpr (V::W == 16) *reinterpret_cast<uint4*>(g.lo + o) = make_uint4(l[0].x, l[1].x, l[2].x, l[3].x);
            else *reinterpret_cast<uint2*>(g.lo + o) = make_uint2(l[0].x, l[1].x);
          }
        }
      } else {
        const float inv = 1.0f / (g.s * NS_E);
        const int rows = flip ? g.m : g.n, cols = flip ? g.n : g.m;
        uint32_t w[V::W / 2];
#pragma unroll
        for (int r = 0; r < V::W / 2; ++r) w[r] = pack2bf(v[2 * r] * inv, v[2 * r + 1] * inv);
        bf16_t* p = g.out + (int64_t)z * rows * cols + (int64_t)m * cols + n0q;
        if (m < rows) {
          if (nw + C::WTN <= cols) {
#pragma unroll
            for (int r = 0; r < V::W / 2; r += 4) mt::st16(p + 2 * r, make_uint4(w[r], w[r + 1], w[r + 2], w[r + 3]));
          } else {
#pragma unroll
            for (int r = 0; r < V::W; ++r)
              if (n0q + r < cols) p[r] = (bf16_t)(w[r >> 1] >> (16 * (r & 1)));
          }
        }
      }
    }
  }
}

int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }

// a group's part of the workspace
int64_t group_bytes(const DphNsGroup& g, char* at, Group* out) {
  const int64_t m = g.rows < g.cols ? g.rows : g.cols, n = g.rows < g.cols ? g.cols : g.rows;
  const int64_t mp = up64(m), np = up64(n), y = g.count * np * mp * 2, e = g.count * mp * mp * 2;
  const int64_t part = g.count * NS_PARTS * (int64_t)sizeof(double);
  const bool split = m <= NS_SPLIT;
  // parts of at least 4 steps of 64 columns, 32 at most
  const int64_t steps = np / 64, want = m <= NS_DEEP && n >= NS_LONG ? (steps / 4 < 32 ? steps / 4 : 32) : 1;
  const int64_t part_steps = cdiv(steps, want), parts = cdiv(steps, part_steps), tm = mp / 64;
  const int64_t slab = parts > 1 ? g.count * (tm * (tm + 1) / 2) * parts * 4096 * (int64_t)sizeof(float) : 0;
  if (out) {
    out->part = reinterpret_cast<double*>(at);
    at += part;
    auto take = [&](bool want, int64_t bytes) -> char* {
      char* p = want ? at : nullptr;
      if (want) at += bytes;
      return p;
    };
    out->y[0] = take(true, y);
    out->y[1] = take(true, y);
    out->e = take(true, e);
    out->f = take(true, e);
    out->lo = take(!split, y / 2);
    out->yl[0] = take(split, y);
    out->yl[1] = take(split, y);
    out->el = take(split, e);
    out->fl = take(split, e);
    out->slab = reinterpret_cast<float*>(take(slab > 0, slab));
    out->parts = (int32_t)parts;
    out->part_steps = (int32_t)part_steps;
  }
  return part + 2 * y + 2 * e + (split ? 2 * y + 2 * e : y / 2) + slab;
}

int check_groups(const DphNsGroup* groups, int64_t n, const char* who) {
  DPH_REQUIRE(n >= 0 && (n == 0 || groups), "%s: null groups", who);
  for (int64_t i = 0; i < n; ++i) {
    const DphNsGroup& g = groups[i];
    DPH_REQUIRE(g.rows >= 1 && g.cols >= 1 && g.count >= 1, "%s: group %lld: empty matrices", who, (long long)i);
    DPH_REQUIRE(g.rows <= DPH_NS_MAX && g.cols <= DPH_NS_MAX && g.count <= DPH_NS_MAX, "%s: group %lld: %lld x %lld (%lld): up to %d",
                who, (long long)i, (long long)g.rows, (long long)g.cols, (long long)g.count, DPH_NS_MAX);
  }
  return DPH_OK;
}

}  // namespace
}  // namespace dph

using namespace dph;

extern "C" int64_t dph_newton_schulz_workspace(const DphNsGroup* groups, int64_t n_groups) {
  if (check_groups(groups, n_groups, "dph_newton_schulz_workspace") != DPH_OK) return -1;
  int64_t most = 0;
  for (int64_t g0 = 0; g0 < n_groups; g0 += NS_GROUPS) {
    int64_t b = 0;
    for (int64_t i = g0; i < n_groups && i < g0 + NS_GROUPS; ++i) b += group_bytes(groups[i], nullptr, nullptr);
    if (b > most) most = b;
  }
  return most;
}

namespace dph {
namespace {

// Kinds of groups: operands split or not, the Gram matrix's sum in parts or not
enum { SHALLOW = 1, DEEP = 2 };

// the groups that are split, or the others, of these kinds, and how many workgroups their tiles of C take
template <int KIND, bool SPLIT, class C, bool FINISH>
int64_t choose(const Groups& all, int kinds, Groups* gs) {
  int64_t tiles = 0;
  gs->ng = 0;
  for (int i = 0; i < all.ng; ++i) {
    const Group& g = all.g[i];
    if ((g.el != nullptr) != SPLIT || !(kinds & (g.parts > 1 ? DEEP : SHALLOW))) continue;
    const int64_t tm = cdiv(g.m, C::BN), tn = cdiv(g.n, C::BM);
    gs->first[gs->ng] = (int32_t)tiles;
    gs->g[gs->ng++] = g;
    tiles += (KIND == GRAM || KIND == POLY ? tm * (tm + 1) / 2 : tm * tn) * g.cnt *
             (KIND == GRAM && C::BM == 64 && !FINISH ? g.parts : 1);
    if (tiles >= (1 << 22)) return -1;
  }
  return tiles;
}
template <int KIND, bool SPLIT, class C, bool FINISH = false>
int launch_tiles(const Groups& all, int kinds, const Step& st, hipStream_t stream) {
  Groups gs = {};
  const int64_t tiles = choose<KIND, SPLIT, C, FINISH>(all, kinds, &gs);
  DPH_REQUIRE(tiles >= 0, "dph_newton_schulz: too many tiles");
  if (tiles == 0) return DPH_OK;
  hipLaunchKernelGGL((ns_product_kernel<KIND, SPLIT, C, FINISH>), dim3((unsigned)tiles), dim3(C::NT), 0, stream, gs, st);
  return check_launch("dph_newton_schulz");
}

// Measured, a whole call with all products on tiles of 256 / 128 / 64: 24 of 1024 x 4096 2.63 / 2.88 / 4.61 ms, 48 of 768 x
// 768 1.11 / 0.88 / 1.20 ms, one of 768 x 768 472 / 221 / 147 us, 8 of 448 x 768 396 / 188 / 152 us.
template <int KIND>
int launch_product(const Groups& gs, const Step& st, hipStream_t stream) {
  // (sums in parts: tiles of 64 x 64 only)
  const int any = KIND == GRAM ? SHALLOW : SHALLOW | DEEP;
  DPH_TRY((launch_tiles<KIND, true, mt::C64>(gs, SHALLOW | DEEP, st, stream)));
  if constexpr (KIND == GRAM) {
    DPH_TRY((launch_tiles<KIND, false, mt::C64>(gs, DEEP, st, stream)));
    DPH_TRY((launch_tiles<KIND, true, mt::C64, true>(gs, DEEP, st, stream)));
    DPH_TRY((launch_tiles<KIND, false, mt::C64, true>(gs, DEEP, st, stream)));
  }
  Groups some = {};
  const int64_t t256 = choose<KIND, false, mt::C256, false>(gs, any, &some),
                t128 = choose<KIND, false, mt::C128, false>(gs, any, &some),
                t64 = choose<KIND, false, mt::C64, false>(gs, any, &some);
  const int tile = t256 < 0 ? 256 : mt::choose_tile(t256, t128, t64);
  if (tile == 64) return launch_tiles<KIND, false, mt::C64>(gs, any, st, stream);
  if (tile == 128) return launch_tiles<KIND, false, mt::C128>(gs, any, st, stream);
  return launch_tiles<KIND, false, mt::C256>(gs, any, st, stream);
}

// up to NS_GROUPS groups, whose matrices start at mats
int run_groups(const DphNsMat* mats, const DphNsGroup* groups, int ng, int steps, const float* c, float eps, char* ws,
               hipStream_t stream) {
  Groups gs = {};
  PackGroups pg = {};
  gs.ng = ng;
  for (int i = 0; i < ng; ++i) {
    const DphNsGroup& in = groups[i];
    Group& g = gs.g[i];
    g.wide = in.rows < in.cols;
    g.m = (int32_t)(g.wide ? in.rows : in.cols);
    g.n = (int32_t)(g.wide ? in.cols : in.rows);
    g.mp = (int32_t)up64(g.m);
    g.np = (int32_t)up64(g.n);
    g.cnt = (int32_t)in.count;
    g.out = reinterpret_cast<bf16_t*>(in.out);
    // entries of X0 have the mean square 1 / (m n): s is the power of two next below sqrt(m n) / 4, at most 2^14 so
    // that an entry of 1.5 times s is a finite fp16 number
    g.s = 1.f;
    while (g.s < 16384.f && (double)g.s * g.s * 64.0 <= (double)g.m * g.n) g.s *= 2.f;
    ws += group_bytes(in, ws, &g);
    pg.g[i] = PackGroup{g.m, g.n, g.mp, g.np, in.f32, g.s, g.y[0], g.lo, g.yl[0], g.part};
  }
  // both packing passes, NS_MATS matrices at a time
  int gi = 0;
  int64_t idx = 0, at = 0;
  while (gi < ng) {
    Mats sum = {}, pack = {};
    int64_t bs = 0, bp = 0;
    while (gi < ng && sum.n < NS_MATS) {
      const Group& g = gs.g[gi];
      const DphNsMat& in = mats[at++];
      const int64_t ns = g.wide ? in.col_stride : in.row_stride, ms = g.wide ? in.row_stride : in.col_stride;
      sum.m[sum.n++] = Mat{in.p, ns, ms, gi, (int32_t)idx, (int32_t)bs, 0};
      pack.m[pack.n++] = Mat{in.p, ns, ms, gi, (int32_t)idx, (int32_t)bp, 0};
      bs += NS_PARTS;
      bp += (int64_t)(g.mp / 64) * (g.np / 64);
      DPH_REQUIRE(bp < (1 << 24), "dph_newton_schulz: too many tiles");
      if (++idx == g.cnt) ++gi, idx = 0;
    }
    hipLaunchKernelGGL(ns_sumsq_kernel, dim3((unsigned)bs), dim3(256), 0, stream, sum, pg);
    hipLaunchKernelGGL(ns_pack_kernel, dim3((unsigned)bp), dim3(256), 0, stream, pack, pg, eps);
  }
  DPH_TRY(check_launch("dph_newton_schulz (packing)"));
  Step st = {};
  for (int i = 0; i < steps; ++i) {
    const bool late = steps - i <= 2 && steps >= 4;    // the last two steps of a run that has got there
    st.d = late ? 1.f : 0.f;
    st.fe = c[1] + 2.f * c[2] * st.d;
    st.fq = c[2];
    // near the end mu is below 1 and goes into F's diagonal, whose rounding it does not make worse, and Y is read as an
    // operand only; before, mu Y is added in as many bits as Y has.  (In the last step of a short run too: its fp16 rounding
    // is an eighth of the result's to bf16)
    const float mu = c[0] + c[1] * st.d + c[2] * st.d * st.d;
    const bool diag = late || i + 1 == steps;
    st.mu = diag ? 0.f : mu;
    st.fd = diag ? mu : 0.f;
    st.cur = i & 1;
    st.lo_out = steps - i - 1 > (steps >= 4 ? 2 : 1);
    DPH_TRY(launch_product<GRAM>(gs, st, stream));
    st.reverse ^= 1;
    DPH_TRY(launch_product<POLY>(gs, st, stream));
    st.reverse ^= 1;
    if (i + 1 < steps) DPH_TRY(launch_product<UPDATE>(gs, st, stream));
    else DPH_TRY(launch_product<LAST>(gs, st, stream));
    st.reverse ^= 1;
  }
  return DPH_OK;
}

}  // namespace
}  // namespace dph

extern "C" int dph_newton_schulz(const DphNsMat* mats, const DphNsGroup* groups, int64_t n_groups, int64_t steps,
                                 const float* coeffs, float eps, void* workspace, int64_t workspace_bytes,
                                 hipStream_t stream) {
  DPH_TRY(check_groups(groups, n_groups, "dph_newton_schulz"));
  if (n_groups == 0) return DPH_OK;
  DPH_REQUIRE(mats && coeffs && workspace, "dph_newton_schulz: null pointer");
  DPH_REQUIRE(steps >= 1 && steps <= 64, "dph_newton_schulz: 1 to 64 steps (got %lld)", (long long)steps);
  for (int i = 0; i < 3; ++i)      // (F's entries times 64 are finite fp16 numbers)
    DPH_REQUIRE(coeffs[i] >= -DPH_NS_COEFF_MAX && coeffs[i] <= DPH_NS_COEFF_MAX, "dph_newton_schulz: coefficients up to %g",
                DPH_NS_COEFF_MAX);
  DPH_REQUIRE(workspace_bytes >= dph_newton_schulz_workspace(groups, n_groups) &&
                  reinterpret_cast<uintptr_t>(workspace) % 256 == 0,
              "dph_newton_schulz: workspace of %lld bytes, 256-byte aligned, wanted",
              (long long)dph_newton_schulz_workspace(groups, n_groups));
  int64_t at = 0;
  for (int64_t i = 0; i < n_groups; ++i) {
    const DphNsGroup& g = groups[i];
    DPH_REQUIRE(g.out && reinterpret_cast<uintptr_t>(g.out) % 8 == 0, "dph_newton_schulz: out is 8-byte aligned");
    for (int64_t k = 0; k < g.count; ++k, ++at) {
      const DphNsMat& t = mats[at];
      DPH_REQUIRE(t.p, "dph_newton_schulz: matrix %lld: null", (long long)at);
      DPH_REQUIRE((t.col_stride == 1 && (t.row_stride >= g.cols || g.rows == 1)) ||
                      (t.row_stride == 1 && (t.col_stride >= g.rows || g.cols == 1)),
                  "dph_newton_schulz: matrix %lld: one of the strides is 1 and the lines do not overlap", (long long)at);
    }
  }
  at = 0;
  for (int64_t i = 0; i < n_groups; i += NS_GROUPS) {
    const int ng = (int)(n_groups - i < NS_GROUPS ? n_groups - i : NS_GROUPS);
    DPH_TRY(run_groups(mats + at, groups + i, ng, (int)steps, coeffs, eps, reinterpret_cast<char*>(workspace), stream));
    for (int k = 0; k < ng; ++k) at += groups[i + k].count;
  }
  return DPH_OK;
}
