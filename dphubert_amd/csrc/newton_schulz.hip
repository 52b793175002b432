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
//   * While singular values grow, a X dominates the step: X is held as two fp16 (22 bits) for that term, so weak
//     directions are not lost in the rounding of strong ones.  The products read the upper half alone.
//   * In the last two steps the singular values are near 1 and a X + b A X + c A^2 X cancel by a factor of 5.  There the
//     polynomial is expanded about d = 1:  E = A - d I,  F = (b + 2 c d) E + c E^2,  X <- (a + b d + c d^2) X + F X,
//     the same products on numbers near 0, whose roundings are small.
// In large matrices an operand's roundings average out; up to NS_SPLIT rows they need not (a 1 x 1 matrix is off by
// 8e-3), and there every operand is two fp16 and every product three: h h + l h + h l.  Such a matrix is one row of
// tiles: launches, not products, set its time.
#include "mfma_tile.h"


namespace dph {
namespace {

typedef uint16_t f16_t;
constexpr int NS_GROUPS = 16;      // groups of equal shapes in one launch
constexpr int NS_MATS = 64;        // matrices of one packing launch
constexpr float NS_E = 64.f;       // E and F are held times 64 (entries of a few 1e-5 stay normal fp16 numbers)
constexpr int NS_PARTS = 64;       // partial sums of a matrix's squares
constexpr int NS_SPLIT = 128;      // rows up to which all operands are held in two parts

__device__ __forceinline__ f16_t f2h(float v) { return __builtin_bit_cast(f16_t, (_Float16)v); }
__device__ __forceinline__ float h2f(f16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
__device__ __forceinline__ uint32_t pack2h(float a, float b) { return (uint32_t)f2h(a) | ((uint32_t)f2h(b) << 16); }
__device__ __forceinline__ void unpack4h(uint2 r, float (&v)[4]) {
  v[0] = h2f((f16_t)(r.x & 0xffff)); v[1] = h2f((f16_t)(r.x >> 16));
  v[2] = h2f((f16_t)(r.y & 0xffff)); v[3] = h2f((f16_t)(r.y >> 16));
}

// what 4 numbers have beyond their fp16 halves h
__device__ __forceinline__ uint2 low4h(const float (&v)[4], uint2 h) {
  float q[4];
  unpack4h(h, q);
  return make_uint2(pack2h(v[0] - q[0], v[1] - q[1]), pack2h(v[2] - q[2], v[3] - q[3]));
}

// Matrices of one shape: cnt of them, each m x n (m <= n) in rows padded with zeros to multiples of 64 (mp, np)
struct Group {
  int32_t m, n, mp, np, cnt, trans;   // trans: the caller's matrices are n x m
  float s;                            // X is held times s
  int32_t in_f32;
  char *xh, *xl, *xt[2], *e, *f;      // [cnt][mp][np] x 2, [cnt][np][mp] x 2, [cnt][mp][mp] x 2
  char *xtl[2], *el, *fl;             // the lower halves of xt, e, f (split) or null
  double* part;                       // [cnt][NS_PARTS]
  bf16_t* out;                        // [cnt] matrices as the caller has them, dense
};
struct Groups {
  int32_t ng;
  int32_t first[NS_GROUPS + 1];       // first tile of each group
  Group g[NS_GROUPS];
};
struct Mat {
  const void* p;
  int64_t rs, cs;                     // strides of the row and the column index of the m x n orientation
  int32_t group, index, first, pad;   // group, place in it, first block of the launch
};
struct Mats {
  int32_t n, pad;
  Mat m[NS_MATS];
};
struct Step {
  float d, fe, fq, mu;     // E = A - d I;  F = fe E + fq E^2;  X <- mu X + F X
  int32_t cur;             // which xt is read
  int32_t lo_in, lo_out;   // X's lower half is read, written
};

struct PackGroup {
  int32_t m, n, mp, np, in_f32;
  float s;
  char *xh, *xl, *xt, *xtl;
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

// Sums of squares in 64 bits, NS_PARTS strips of rows a matrix (in its memory order), added in a fixed order later
__global__ void __launch_bounds__(256) ns_sumsq_kernel(const Mats a, const PackGroups pg) {
  const int k = find_mat(a, (int)blockIdx.x);
  const Mat& t = a.m[k];
  const PackGroup& g = pg.g[t.group];
  const int part = (int)blockIdx.x - t.first;
  // walk along the unit stride
  const bool by_row = t.cs == 1;
  const int32_t R = by_row ? g.m : g.n, L = by_row ? g.n : g.m;
  const int64_t rs = by_row ? t.rs : t.cs, cs = by_row ? t.cs : t.rs;
  double s = 0.0;
  const int64_t total = (int64_t)R * L, per = cdiv(total, NS_PARTS);
  const int64_t i1 = min(total, (part + 1) * per);
  for (int64_t i = part * per + threadIdx.x; i < i1; i += 256) {
    const int64_t r = i / L, c = i - r * L;
    const double v = ldg(t.p, r * rs + c * cs, g.in_f32);
    s += v * v;
  }
  __shared__ double red[4];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) g.part[(int64_t)t.index * NS_PARTS + part] = (red[0] + red[1]) + (red[2] + red[3]);
}

// X0 in both orders, 64 x 64 tiles through the LDS; reads run along whichever stride of the input is 1
__global__ void __launch_bounds__(256) ns_pack_kernel(const Mats a, const PackGroups pg, float eps) {
  __shared__ float tile[64][65];
  __shared__ float scale;
  const int k = find_mat(a, (int)blockIdx.x);
  const Mat& t = a.m[k];
  const PackGroup& g = pg.g[t.group];
  if (threadIdx.x < 64) {
    double s = g.part[(int64_t)t.index * NS_PARTS + threadIdx.x];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (threadIdx.x == 0) scale = (float)((double)g.s / (sqrt(s) + (double)eps));
  }
  const int b = (int)blockIdx.x - t.first, tn = g.np >> 6;
  const int r0 = b / tn * 64, c0 = b % tn * 64;
  __syncthreads();
  const float sc = scale;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  if (t.cs == 1) {
    for (int i = ty; i < 64; i += 4)
      tile[i][tx] = r0 + i < g.m && c0 + tx < g.n ? ldg(t.p, (int64_t)(r0 + i) * t.rs + c0 + tx, g.in_f32) * sc : 0.f;
  } else {
    for (int i = ty; i < 64; i += 4)
      tile[tx][i] = r0 + tx < g.m && c0 + i < g.n ? ldg(t.p, (int64_t)(r0 + tx) * t.rs + (int64_t)(c0 + i) * t.cs, g.in_f32) * sc : 0.f;
  }
  __syncthreads();
  const int64_t mat = (int64_t)t.index * g.mp * g.np;
  // 4 consecutive elements a thread
  const int x4 = (threadIdx.x & 15) * 4, y = threadIdx.x >> 4;
  for (int i = y; i < 64; i += 16) {
    float v[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = tile[i][x4 + j];
      lo[j] = v[j] - h2f(f2h(v[j]));
    }
    const int64_t o = mat + (int64_t)(r0 + i) * g.np + c0 + x4;
    *reinterpret_cast<uint2*>(reinterpret_cast<f16_t*>(g.xh) + o) = make_uint2(pack2h(v[0], v[1]), pack2h(v[2], v[3]));
    *reinterpret_cast<uint2*>(reinterpret_cast<f16_t*>(g.xl) + o) = make_uint2(pack2h(lo[0], lo[1]), pack2h(lo[2], lo[3]));
    const int64_t ot = mat + (int64_t)(c0 + i) * g.mp + r0 + x4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = tile[x4 + j][i];
      lo[j] = v[j] - h2f(f2h(v[j]));
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<f16_t*>(g.xt) + ot) = make_uint2(pack2h(v[0], v[1]), pack2h(v[2], v[3]));
    if (g.xtl)
      *reinterpret_cast<uint2*>(reinterpret_cast<f16_t*>(g.xtl) + ot) = make_uint2(pack2h(lo[0], lo[1]), pack2h(lo[2], lo[3]));
  }
}

// ---- the products -------------------------------------------------------------------------------------------------
enum { GRAM, POLY, UPDATE, LAST };

// 4 x 4 transpose inside a quad of lanes: lane q of the quad has element (row q, column r) as the r-th of 4 16-bit
// numbers and leaves with (row r, column q)
__device__ __forceinline__ uint2 quad_transpose(uint2 x, int lane) {
  const bool o1 = lane & 1, o2 = lane & 2;
  const uint32_t y0 = (uint32_t)__builtin_amdgcn_mov_dpp((int)x.x, 0xb1, 0xf, 0xf, true);   // lane ^ 1
  const uint32_t y1 = (uint32_t)__builtin_amdgcn_mov_dpp((int)x.y, 0xb1, 0xf, 0xf, true);
  const uint32_t a0 = o1 ? (y0 >> 16) | (x.x & 0xffff0000u) : (x.x & 0xffffu) | (y0 << 16);
  const uint32_t a1 = o1 ? (y1 >> 16) | (x.y & 0xffff0000u) : (x.y & 0xffffu) | (y1 << 16);
  const uint32_t b0 = (uint32_t)__builtin_amdgcn_mov_dpp((int)a0, 0x4e, 0xf, 0xf, true);    // lane ^ 2
  const uint32_t b1 = (uint32_t)__builtin_amdgcn_mov_dpp((int)a1, 0x4e, 0xf, 0xf, true);
  return o2 ? make_uint2(b1, a1) : make_uint2(a0, b0);
}

template <int KIND, class C>
__global__ void __launch_bounds__(C::NT, 2) ns_product_kernel(const Groups gs, const Step st) {
  __shared__ __align__(16) char smem[C::LDS];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int t = mt::xcd_tile((int)blockIdx.x, (int)gridDim.x);
  int k = 0;
  while (k + 1 < gs.ng && gs.first[k + 1] <= t) ++k;
  const Group& g = gs.g[k];
  t -= gs.first[k];
  constexpr bool SYM = KIND == GRAM || KIND == POLY;
  const int tm = (g.m + C::BM - 1) / C::BM;
  int ti, tj, z;
  if (SYM) {
    static_assert(C::BM == C::BN && C::BM >= NS_SPLIT, "square tiles, one of them where operands are split");
    const int per = tm * (tm + 1) / 2;
    z = t / per;
    t -= z * per;
    ti = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > t) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    tj = t - ti * (ti + 1) / 2;
  } else {
    const int tn = (g.n + C::BN - 1) / C::BN, per = tm * tn;
    z = t / per;
    t -= z * per;
    tj = t / tm;         // (consecutive tiles share rows of X^T)
    ti = t % tm;
  }
  const int m0 = ti * C::BM, n0 = tj * C::BN;
  const int64_t xoff = (int64_t)z * g.mp * g.np * 2, eoff = (int64_t)z * g.mp * g.mp * 2;
  const bool split = g.el != nullptr;
  f32x4_t acc[C::FM][C::FN];
  mt::clear<mt::F16, C>(acc);
  for (int part = 0; part < (split ? 3 : 1); ++part) {   // h h, l h, h l
    const bool la = part == 1, lb = part == 2;
    mt::Rows A, B;
    int kbytes;
    if constexpr (KIND == GRAM) {
      kbytes = g.np * 2;
      A = mt::Rows{(la ? g.xl : g.xh) + xoff, kbytes, g.mp};
      B = mt::Rows{(lb ? g.xl : g.xh) + xoff, kbytes, g.mp};
    } else if constexpr (KIND == POLY) {
      kbytes = g.mp * 2;
      A = mt::Rows{(la ? g.el : g.e) + eoff, kbytes, g.mp};
      B = mt::Rows{(lb ? g.el : g.e) + eoff, kbytes, g.mp};
    } else {
      kbytes = g.mp * 2;
      A = mt::Rows{(la ? g.fl : g.f) + eoff, kbytes, g.mp};
      B = mt::Rows{(lb ? g.xtl[st.cur] : g.xt[st.cur]) + xoff, kbytes, g.np};
    }
    mt::product<mt::F16, C>(A, B, kbytes, m0, n0, acc, smem, wave, lane);
  }

  const int ml = m0 + wave / C::WC * C::WTM + (lane & 15), nl = n0 + wave % C::WC * C::WTN + 4 * (lane >> 4);
  const int M = g.mp, N = SYM ? g.mp : g.np;      // (what lies past m and n is zero, and stays zero)
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
#pragma unroll
    for (int j = 0; j < C::FN; ++j) {
      const int m = ml + 16 * i, n = nl + 16 * j;
      const bool in = m < M && n < N;
      // rows of the quad's transpose: n + (lane & 3), columns 4 (m / 4) ..
      const int tr = n + (lane & 3), tc = m & ~3;
      float v[4];
      if constexpr (SYM) {
        if constexpr (KIND == GRAM) {
          const float sc = NS_E / (g.s * g.s);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = acc[i][j][r] * sc - (m == n + r && m < g.m ? NS_E * st.d : 0.f);
        } else {
          float e[4] = {0.f, 0.f, 0.f, 0.f};
          if (in) {
            unpack4h(*reinterpret_cast<const uint2*>(g.e + eoff + ((int64_t)m * M + n) * 2), e);
            if (split) {
              float lo[4];
              unpack4h(*reinterpret_cast<const uint2*>(g.el + eoff + ((int64_t)m * M + n) * 2), lo);
#pragma unroll
              for (int r = 0; r < 4; ++r) e[r] += lo[r];
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = st.fe * e[r] + st.fq / NS_E * acc[i][j][r];
        }
        const uint2 h = make_uint2(pack2h(v[0], v[1]), pack2h(v[2], v[3]));
        char* o = (KIND == GRAM ? g.e : g.f) + eoff;
        if (in) *reinterpret_cast<uint2*>(o + ((int64_t)m * M + n) * 2) = h;
        const uint2 ht = quad_transpose(h, lane);
        if (ti != tj && in) *reinterpret_cast<uint2*>(o + ((int64_t)tr * M + tc) * 2) = ht;
        if (split && in)       // (a single tile: its own mirror image)
          *reinterpret_cast<uint2*>((KIND == GRAM ? g.el : g.fl) + eoff + ((int64_t)m * M + n) * 2) = low4h(v, h);
      } else {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        const int64_t o = xoff + ((int64_t)m * N + n) * 2;
        if (in) {
          unpack4h(*reinterpret_cast<const uint2*>(g.xh + o), x);
          if (st.lo_in || split) {
            float lo[4];
            unpack4h(*reinterpret_cast<const uint2*>(g.xl + o), lo);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] += lo[r];
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = st.mu * x[r] + acc[i][j][r] / NS_E;
        if constexpr (KIND == UPDATE) {
          const uint2 h = make_uint2(pack2h(v[0], v[1]), pack2h(v[2], v[3]));
          if (in) {
            *reinterpret_cast<uint2*>(g.xh + o) = h;
            if (st.lo_out || split) *reinterpret_cast<uint2*>(g.xl + o) = low4h(v, h);
          }
          const uint2 ht = quad_transpose(h, lane);
          if (in) *reinterpret_cast<uint2*>(g.xt[st.cur ^ 1] + xoff + ((int64_t)tr * g.mp + tc) * 2) = ht;
          if (split) {
            const uint2 lt = quad_transpose(low4h(v, h), lane);
            if (in) *reinterpret_cast<uint2*>(g.xtl[st.cur ^ 1] + xoff + ((int64_t)tr * g.mp + tc) * 2) = lt;
          }
        } else {
          const float inv = 1.0f / g.s;
          uint2 h = make_uint2(pack2bf(v[0] * inv, v[1] * inv), pack2bf(v[2] * inv, v[3] * inv));
          // the caller's order: rows of n, or of m where the matrix was transposed
          int row = m, col = n, cols = g.n, rows = g.m;
          if (g.trans) {
            h = quad_transpose(h, lane);
            row = tr, col = tc, cols = g.m, rows = g.n;
          }
          bf16_t* p = g.out + (int64_t)z * g.m * g.n + (int64_t)row * cols + col;
          if (row < rows) {
            if (col + 4 <= cols && (cols & 3) == 0) {
              *reinterpret_cast<uint2*>(p) = h;
            } else {
              const uint32_t w[2] = {h.x, h.y};
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (col + r < cols) p[r] = (bf16_t)(w[r >> 1] >> (16 * (r & 1)));
            }
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
  const int64_t mp = up64(m), np = up64(n), x = g.count * mp * np * 2, e = g.count * mp * mp * 2;
  const int64_t part = g.count * NS_PARTS * (int64_t)sizeof(double);
  const bool split = m <= NS_SPLIT;
  if (out) {
    out->part = reinterpret_cast<double*>(at);
    at += part;
    out->xh = at;
    out->xl = at + x;
    out->xt[0] = at + 2 * x;
    out->xt[1] = at + 3 * x;
    out->e = at + 4 * x;
    out->f = at + 4 * x + e;
    at += 4 * x + 2 * e;
    out->xtl[0] = split ? at : nullptr;
    out->xtl[1] = split ? at + x : nullptr;
    out->el = split ? at + 2 * x : nullptr;
    out->fl = split ? at + 2 * x + e : nullptr;
  }
  return part + 4 * x + 2 * e + (split ? 2 * x + 2 * e : 0);
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

using NsTile = mt::Tile<128, 128, 2, 2>;

template <int KIND>
int launch_product(const Groups& gs0, const Step& st, hipStream_t stream) {
  Groups gs = gs0;
  int64_t tiles = 0;
  for (int i = 0; i < gs.ng; ++i) {
    const Group& g = gs.g[i];
    const int64_t tm = cdiv(g.m, NsTile::BM), tn = cdiv(g.n, NsTile::BN);
    gs.first[i] = (int32_t)tiles;
    tiles += (KIND == GRAM || KIND == POLY ? tm * (tm + 1) / 2 : tm * tn) * g.cnt;
    DPH_REQUIRE(tiles < (1 << 24), "dph_newton_schulz: too many tiles");
  }
  hipLaunchKernelGGL((ns_product_kernel<KIND, NsTile>), dim3((unsigned)tiles), dim3(NsTile::NT), 0, stream, gs, st);
  return check_launch("dph_newton_schulz");
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
    g.trans = in.rows > in.cols;
    g.m = (int32_t)(g.trans ? in.cols : in.rows);
    g.n = (int32_t)(g.trans ? in.rows : in.cols);
    g.mp = (int32_t)up64(g.m);
    g.np = (int32_t)up64(g.n);
    g.cnt = (int32_t)in.count;
    g.in_f32 = in.f32;
    g.out = reinterpret_cast<bf16_t*>(in.out);
    // entries of X0 have the mean square 1 / (m n): s is the power of two next below sqrt(m n) / 4, at most 2^14 so
    // that an entry of 1.5 times s is a finite fp16 number
    g.s = 1.f;
    while (g.s < 16384.f && (double)g.s * g.s * 64.0 <= (double)g.m * g.n) g.s *= 2.f;
    ws += group_bytes(in, ws, &g);
    pg.g[i] = PackGroup{g.m, g.n, g.mp, g.np, g.in_f32, g.s, g.xh, g.xl, g.xt[0], g.xtl[0], g.part};
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
      const int64_t rs = g.trans ? in.col_stride : in.row_stride, cs = g.trans ? in.row_stride : in.col_stride;
      sum.m[sum.n++] = Mat{in.p, rs, cs, gi, (int32_t)idx, (int32_t)bs, 0};
      pack.m[pack.n++] = Mat{in.p, rs, cs, gi, (int32_t)idx, (int32_t)bp, 0};
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
    st.mu = c[0] + c[1] * st.d + c[2] * st.d * st.d;
    st.cur = i & 1;
    st.lo_in = !late;
    st.lo_out = !(steps - i - 1 <= 2 && steps >= 4);
    DPH_TRY(launch_product<GRAM>(gs, st, stream));
    DPH_TRY(launch_product<POLY>(gs, st, stream));
    if (i + 1 < steps) DPH_TRY(launch_product<UPDATE>(gs, st, stream));
    else DPH_TRY(launch_product<LAST>(gs, st, stream));
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
