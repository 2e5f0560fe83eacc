// The orthogonal factor of a matrix by Newton-Schulz products:  X = G / |G|_F, then for every step with coefficients (a, b, c)
//
//   S = X X',   X <- a X + (b S + c S S) X        (s = the shorter side, l = the longer one; X stands as s x l)
//
// which drives every singular value of X towards one and leaves its singular vectors.  Small singular values grow by a in each step, so
// does a rounding error made early: everything is carried to 32-bit accuracy or better.
//
//   s <= 96: the polynomials of several steps are polynomials of their first S.  One pass over X makes S in 64 bits, one workgroup per matrix
//     iterates on s x s matrices in LDS in 64 bits (S <- P S P, Q <- Q P), a second pass applies Q.  Two reads and a write of G.  (Five steps on
//     90 x 20000: 131 us, the other form 192; 60 of 96 x 3000: 234 and 465; one of 96 x 96, where the iteration is all there is: 114 and 105.  Fourteen:
//     359 and 493, 647 and 1220, 315 and 279.  Beyond, three matrices do not fit into LDS.)
//     What is iterated is not X: a rounding error e = 2^-53 in an eigenvalue of S near zero, which may make it negative, grows by growth^2 (growth: the
//     product of the steps' largest a + b S + c S S), and from some 1e-2 on it takes over -- where rows of G depend on each other, the default steps leave
//     the right place after 12 steps and every bound after 16.  So the steps are taken in groups of growth up to 2048 (5e-10), X is formed after
//     each (in fp32: in O, or for 16-bit types in the workspace, some matrices at a time), and the next group starts from the S of that X.
//   s > 96: products on the 16-bit matrix pipes.  An entry x is kept as two fp16 numbers, hi + lo (22 significant bits), scaled by a power of
//     two that the growth bound of the step allows; a product is hi hi + hi lo + lo hi, summed in 32 bits (what is dropped is 2^-22 of it).
#include <type_traits>

#include "nmfk_matrix.h"

using namespace nmfk_mat;

namespace {

constexpr int SMALL = 96;
constexpr double GROWTH32 = 512;  // up to which s <= 96 applies its factor in 32 bits: five of the default steps, 3e-5 of |G| in the directions that grow so
constexpr double GROWTH = 2048;   // ... and up to which one factor holds: six of the default steps
constexpr int64_t PORTION = (int64_t)1 << 26;  // bytes of X between the factors of 16-bit matrices
constexpr int64_t BATCH = 32768;  // matrices a launch
constexpr double TINY = 1e-20;    // bounds below it are not followed any further

struct Strided {
  char *p;
  int64_t batch, row, col;  // strides in entries: row along s, col along l
};

template <typename T>
__device__ __forceinline__ float read_at(const Strided &g, int64_t b, int64_t i, int64_t j) {
  return to_f32(((const T *)g.p)[b * g.batch + i * g.row + j * g.col]);
}

// ---- s <= 96 ---------------------------------------------------------------------------------------------------------------------
//
// The fp64 matrix instruction (16 x 16 x 4) leaves entry [4 r + g][c] of its result in register r of lane 16 g + c, and takes, for its k-th step,
// entry [c][4 k + g] of the first and [4 k + g][c] of the second operand there.  All matrices of the iteration are polynomials of S, hence
// symmetric and commuting: register r of a result IS the operand of step r, on either side.  Products chain without moving an entry.

struct SmallArgs {
  Strided g, o;
  double *part;  // [batch][chunks][s][s]
  double *q;     // s > 16, [batch][small_q_size]: Q / |G| in the order in which small_apply_kernel takes it, then the exponent left out of it
  int s, chunks, steps;
  int first;         // X is G / |G|; otherwise it is taken as it is
  int q64;           // Q is applied in 64 bits
  int64_t l, chunk;  // entries of l per workgroup
  int gvec, ovec;    // the side that is walked is contiguous: four entries at once
};

struct Coefs {
  double v[3 * 32];
};

template <typename T, bool WIDE>
__device__ __forceinline__ void small_load4(const Strided &g, const T *p, int s, int64_t l, int vec, int i, int64_t j, float (&out)[4]) {
  const T *q = p + i * g.row + j * g.col;
  const bool whole = WIDE ? i < s && j + 4 <= l : j < l && i + 4 <= s;
  if (vec && whole) {
    read4(q, out);
  } else {
    const int64_t step = WIDE ? g.col : g.row;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = (WIDE ? i < s && j + e < l : j < l && i + e < s) ? to_f32(q[e * step]) : 0.f;
  }
}

// Partial S over a chunk of l, in 64 bits.  What bounds it is the read of G, so a lane holds an entry in the place where the matrix
// instruction wants it on both sides, straight from memory.  With s <= 8 the instruction's 16 rows take 16 / s columns of X at once (the
// diagonal blocks of the result add up to S).  480 of 8192 x 16 in fp32: 60 us, 4.2 TB/s.
template <typename T, int TT, bool WIDE>
__global__ __launch_bounds__(256) void small_gram_kernel(SmallArgs a) {
  __shared__ double sum[4][256];
  const int64_t b = blockIdx.y;
  const int64_t l0 = blockIdx.x * a.chunk, l1 = min(a.l, l0 + a.chunk);
  const int s = a.s, t = threadIdx.x, w = t >> 6, lane = t & 63, c = lane & 15, g = lane >> 4;
  const int packed = TT == 1 ? max(1, 16 / s) : 1, grp = TT == 1 ? c / s : 0, row = TT == 1 ? c - grp * s : c;
  const bool live = grp < packed;
  const T *p = (const T *)a.g.p + b * a.g.batch;
  f64x4 acc[TT * (TT + 1) / 2];
#pragma unroll
  for (int k = 0; k < TT * (TT + 1) / 2; ++k) acc[k] = (f64x4){0, 0, 0, 0};
  constexpr int U = TT == 1 ? 8 : TT == 2 ? 4 : 2;  // loads in flight
  if (WIDE) {
    constexpr int UW = TT == 1 ? 4 : TT == 2 ? 2 : 1;
    const int span = 16 * packed;
    for (int64_t base = l0 + (int64_t)w * UW * span; base < l1; base += 4 * UW * span) {
      float x[UW][TT][4];
#pragma unroll
      for (int u = 0; u < UW; ++u)
#pragma unroll
        for (int k = 0; k < TT; ++k) small_load4<T, true>(a.g, p, live ? s : 0, l1, a.gvec, 16 * k + row, base + u * span + grp * 16 + 4 * g, x[u][k]);
#pragma unroll
      for (int u = 0; u < UW; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          double v[TT];
#pragma unroll
          for (int k = 0; k < TT; ++k) v[k] = (double)x[u][k][e];
#pragma unroll
          for (int i = 0; i < TT; ++i)
#pragma unroll
            for (int j = 0; j <= i; ++j) acc[i * (i + 1) / 2 + j] = __builtin_amdgcn_mfma_f64_16x16x4f64(v[i], v[j], acc[i * (i + 1) / 2 + j], 0, 0, 0);
        }
    }
  } else {
    // TT == 1: two sums take turns, an fp64 instruction waits for its predecessor's result otherwise
    f64x4 odd = {0, 0, 0, 0};
    const int span = 4 * packed, mine = g * packed + grp;
    const int64_t step = span * a.g.col;
    auto multiply = [&](const float (&x)[U][TT]) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        double v[TT];
#pragma unroll
        for (int k = 0; k < TT; ++k) v[k] = (double)x[u][k];
        if (TT == 1 && (u & 1)) {
          odd = __builtin_amdgcn_mfma_f64_16x16x4f64(v[0], v[0], odd, 0, 0, 0);
          continue;
        }
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
          for (int j = 0; j <= i; ++j) acc[i * (i + 1) / 2 + j] = __builtin_amdgcn_mfma_f64_16x16x4f64(v[i], v[j], acc[i * (i + 1) / 2 + j], 0, 0, 0);
      }
    };
    int64_t base = l0 + (int64_t)w * U * span;
    const T *q[TT];
    bool here[TT];
#pragma unroll
    for (int k = 0; k < TT; ++k) {
      here[k] = live && 16 * k + row < s;
      q[k] = p + (here[k] ? (16 * k + row) * a.g.row + (base + mine) * a.g.col : 0);
    }
    float x[U][TT], next[U][TT];
    auto load = [&](float (&to)[U][TT], bool whole) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < TT; ++k) to[u][k] = here[k] && (whole || base + u * span + mine < l1) ? to_f32(q[k][u * step]) : 0.f;
#pragma unroll
      for (int k = 0; k < TT; ++k) q[k] += 4 * U * step;
      base += 4 * U * span;
    };
    // the next entries are on their way while these are multiplied
    if (base + U * span <= l1) {
      load(x, true);
      while (base + U * span <= l1) {
        load(next, true);
        multiply(x);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int k = 0; k < TT; ++k) x[u][k] = next[u][k];
      }
      multiply(x);
    }
    if (base < l1) {
      load(x, false);
      multiply(x);
    }
    if (TT == 1) acc[0] += odd;
  }
  double *out = a.part + ((int64_t)blockIdx.y * a.chunks + blockIdx.x) * s * s;
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j <= i; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[w][(4 * r + g) * 16 + c] = acc[i * (i + 1) / 2 + j][r];
      __syncthreads();
      if (TT == 1) {
        if (t < s * s) {
          const int y = t / s, x = t - y * s;
          double v = 0;
          for (int k = 0; k < packed; ++k) {
            const int e = (k * s + y) * 16 + k * s + x;
            v += (sum[0][e] + sum[1][e]) + (sum[2][e] + sum[3][e]);
          }
          out[t] = v;
        }
      } else {
        const int y = 16 * i + (t >> 4), x = 16 * j + (t & 15);
        const double v = (sum[0][t] + sum[1][t]) + (sum[2][t] + sum[3][t]);
        if (y < s && x < s) {
          out[y * s + x] = v;
          if (i != j) out[x * s + y] = v;
        }
      }
      __syncthreads();
    }
}

// 1 / |G|^2 and 1 / |G| as the iteration uses them: 0 for a matrix of zeros, NaN for one that is not finite; 1 behind the first group of steps
__device__ __forceinline__ void small_norm(double &norm2, int first, double &inv2, double &inv) {
  if (!first) {
    norm2 = inv2 = inv = 1.0;
    return;
  }
  const double nan = __longlong_as_double(0x7ff8000000000000ll);
  const bool finite = norm2 <= 1.7e308;
  inv2 = !finite ? nan : norm2 > 0 ? 1.0 / norm2 : 0.0;
  inv = !finite ? nan : norm2 > 0 ? 1.0 / sqrt(norm2) : 0.0;
}

// Q / |G| goes up to growth / |G|, which 32 bits do not hold for a very small |G|, nor its bits for a very large one: there the power of two stays out of Q,
// and G is multiplied by it (exactly).
__device__ __forceinline__ int small_exponent(double norm2, int q64) {
  const int e = (__double2hiint(norm2) >> 20) - 1023;  // (zero and what is not finite are far outside)
  return !q64 && (e < -200 || e > 200) && e > -400 && e < 400 ? -e >> 1 : 0;
}

// Where small_apply_kernel looks for Q[y, x]: the operand of step k of tile (i, j) for lane 16 g + c at [((i TT + j) 4 + k) 64 + 16 g + c].  The fp64 instruction
// leaves entry [4 r + g] where the fp32 one leaves [4 g + r]: its rows are dealt so that a lane gets row 4 g + r, too.
template <int TT>
__host__ __device__ constexpr int small_q_size() {
  return TT * TT * 256 + 32;
}
template <int TT>
__device__ __forceinline__ int small_q_at(int y, int x, int q64) {
  const int c = q64 ? ((y & 3) << 2) + ((y >> 2) & 3) : y & 15;
  return (((y >> 4) * TT + (x >> 4)) * 4 + (x & 3)) * 64 + ((x & 12) << 2) + c;
}

__device__ __forceinline__ f64x4 sym_product(f64x4 x, f64x4 y) {
  f64x4 d = {0, 0, 0, 0};
#pragma unroll
  for (int r = 0; r < 4; ++r) d = __builtin_amdgcn_mfma_f64_16x16x4f64(x[r], y[r], d, 0, 0, 0);
  return d;
}

// s > 16: the chunks' partial S, added in their order and left in the place of the first
__global__ __launch_bounds__(256) void small_join_kernel(SmallArgs a) {
  const int ss = a.s * a.s, e = blockIdx.x * 256 + threadIdx.x;
  if (e >= ss) return;
  double *part = a.part + (int64_t)blockIdx.y * a.chunks * ss + e, v = 0;
#pragma unroll 16
  for (int k = 0; k < a.chunks; ++k) v += part[(int64_t)k * ss];
  *part = v;
}

// s > 16: the iteration by one workgroup per matrix.  What bounds it is the fp64 matrix instruction (64 cycles) on one CU, so only the tiles on and
// below the diagonal are computed, by a wave each (s > 80: two), and kept in LDS: rows of a tile 17 entries apart, so that a tile can be read
// as its transpose, too.  Above s = 80 there is no room for a fourth matrix, and U takes the place of S.  Five steps: 29 us at s = 64, 46 at 80, 82 at 96
// (every tile computed, partial sums added by this workgroup: 76 at s = 64).
constexpr int small_tiles(int tt) { return tt * (tt + 1) / 2; }
constexpr int small_waves(int tt) { return tt > 5 ? (small_tiles(tt) + 1) / 2 : small_tiles(tt); }
constexpr int small_lds(int tt) { return (tt > 5 ? 3 : 4) * small_tiles(tt) * 16 * 17 * 8; }
constexpr int SUMS = 4;  // partial S that the iteration adds itself; more of them are joined before
template <int TT>
__global__ __launch_bounds__(64 * small_waves(TT)) void small_iterate_kernel(SmallArgs a, Coefs cf, int parts) {
  extern __shared__ double mats[];
  constexpr int TILE = 16 * 17, NT = small_tiles(TT), N = NT * TILE, W = small_waves(TT), OWN = (NT + W - 1) / W;
  constexpr bool TIGHT = TT > 5;
  const int s = a.s, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  double *S = mats, *P = S + N, *Q = P + N, *U = TIGHT ? S : Q + N;
  const double *part = a.part + (int64_t)blockIdx.x * a.chunks * s * s;
  int ti[OWN], tj[OWN];
#pragma unroll
  for (int o = 0; o < OWN; ++o) {
    const int id = min(w + o * W, NT - 1);  // (the last tile twice: the same numbers to the same place)
    ti[o] = id < 1 ? 0 : id < 3 ? 1 : id < 6 ? 2 : id < 10 ? 3 : id < 15 ? 4 : 5;
    tj[o] = id - ti[o] * (ti[o] + 1) / 2;
  }
  const int down = 17 * g + c, across = 17 * c + g;  // entry [4 r + g][c] of a tile: 68 r further; of its transpose: 4 r further
  auto put = [&](double *m, const f64x4 (&d)[OWN]) {
#pragma unroll
    for (int o = 0; o < OWN; ++o)
#pragma unroll
      for (int r = 0; r < 4; ++r) m[(ti[o] * (ti[o] + 1) / 2 + tj[o]) * TILE + down + 68 * r] = d[o][r];
  };
  auto product = [&](const double *m, const double *n, f64x4 (&d)[OWN]) {
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      d[o] = (f64x4){0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < TT; ++k) {
        const int ui = k >= ti[o] ? (k * (k + 1) / 2 + ti[o]) * TILE + down : (ti[o] * (ti[o] + 1) / 2 + k) * TILE + across, si = k >= ti[o] ? 68 : 4;
        const int uj = k >= tj[o] ? (k * (k + 1) / 2 + tj[o]) * TILE + down : (tj[o] * (tj[o] + 1) / 2 + k) * TILE + across, sj = k >= tj[o] ? 68 : 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) d[o] = __builtin_amdgcn_mfma_f64_16x16x4f64(m[ui + r * si], n[uj + r * sj], d[o], 0, 0, 0);
      }
    }
  };
  f64x4 sv[OWN], p[OWN], q[OWN], u[OWN];
#pragma unroll
  for (int o = 0; o < OWN; ++o) {
    sv[o] = (f64x4){0, 0, 0, 0};
    const int x = 16 * tj[o] + c;
#pragma unroll
    for (int k = 0; k < SUMS; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int y = 16 * ti[o] + 4 * r + g;
        if (k < parts && y < s && x < s) sv[o][r] += part[(int64_t)k * s * s + y * s + x];
      }
  }
  put(S, sv);
  __syncthreads();
  double norm2 = 0;
  for (int i = lane; i < 16 * TT; i += 64) {  // zero behind s
    const int k = i >> 4, e = i & 15;
    norm2 += S[(k * (k + 1) / 2 + k) * TILE + 18 * e];
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) norm2 += __shfl_xor(norm2, o);
  double inv2, inv;
  small_norm(norm2, a.first, inv2, inv);
  __syncthreads();
#pragma unroll
  for (int o = 0; o < OWN; ++o) sv[o] *= inv2;
  put(S, sv);
  __syncthreads();
  for (int k = 0; k < a.steps; ++k) {
    product(S, S, p);
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      p[o] = cf.v[3 * k + 1] * sv[o] + cf.v[3 * k + 2] * p[o];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (ti[o] == tj[o] && 4 * r + g == c) p[o][r] += cf.v[3 * k];
    }
    put(P, p);
    __syncthreads();
    if (k == 0) {
#pragma unroll
      for (int o = 0; o < OWN; ++o) q[o] = p[o];
    } else {
      product(Q, P, q);
    }
    if (k + 1 == a.steps) break;
    product(S, P, u);
    if (TIGHT) __syncthreads();
    put(U, u);
    __syncthreads();
    put(Q, q);
    product(U, P, sv);
    if (TIGHT) __syncthreads();
    put(S, sv);
    __syncthreads();
  }
  const int e = small_exponent(norm2, a.q64);
  inv = ldexp(inv, -e);
  double *out = a.q + (int64_t)blockIdx.x * small_q_size<TT>();
  if (threadIdx.x == 0) out[TT * TT * 256] = e;
#pragma unroll
  for (int o = 0; o < OWN; ++o) {
    const int x = 16 * tj[o] + c;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int y = 16 * ti[o] + 4 * r + g;
      const double v = y < s && x < s ? q[o][r] * inv : 0.0;
      out[small_q_at<TT>(y, x, a.q64)] = v;
      if (ti[o] != tj[o]) out[small_q_at<TT>(x, y, a.q64)] = v;
    }
  }
}

// O = Q G over a chunk of l, on the fp32 matrix pipe (16 x 16 x 4: entry [c][.] of the first, [.][c] of the second operand in lane 16 g + c, result
// [4 g + r][c] in register r) or on the fp64 one.  Which four of the sum's entries a step takes is free: a lane's four consecutive entries of G or of Q
// serve four steps, or four columns, and its four results stand next to each other in O.  s <= 16: every workgroup iterates for itself, a wave in registers
// (about 2 microseconds, less than a launch), while the first entries of G are on their way.  480 of 8192 x 16 in fp32: 86 us, 5.9 TB/s.
//
// A = float: Q in registers, rounded to 32 bits, which puts an error of growth * 2^-24 |G| into O like the same steps in fp32 would.  A = double where that is
// too much: O is off by its own rounding (to fp32, then to its type).  Q stands in LDS, which is quick enough for an instruction of 64 cycles.  60 of 96 x 3000:
// 67 us in 32 bits, 123 in 64.
__device__ __forceinline__ f32x4 small_multiply(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f64x4 small_multiply(double a, double b, f64x4 c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }

template <typename T, typename O, typename A, int TT, bool WIDE>
__global__ __launch_bounds__(256, TT == 1 ? 4 : (std::is_same<A, double>::value && (TT < 4 || !WIDE) ? 2 : 1)) void small_apply_kernel(SmallArgs a, Coefs cf) {
  constexpr bool Q64 = std::is_same<A, double>::value, LDS = Q64 && TT > 1;
  using vec = typename std::conditional<Q64, f64x4, f32x4>::type;
  __shared__ double sum[TT == 1 ? 256 : 1];
  __shared__ A own[TT == 1 ? 256 : 1];
  __shared__ int exponent;
  extern __shared__ __attribute__((aligned(16))) double qs[];  // LDS: the operands of Q as in memory
  const int by = gridDim.y - 1 - blockIdx.y;  // the matrices read last are still in the last-level cache: take them first
  const int64_t l0 = blockIdx.x * a.chunk, l1 = min(a.l, l0 + a.chunk);
  const int s = a.s, t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, c = lane & 15, g = lane >> 4;
  const T *p = (const T *)a.g.p + by * a.g.batch;
  O *o = (O *)a.o.p + by * a.o.batch;
  constexpr int U = WIDE ? 4 : TT == 1 ? 4 : TT == 2 ? 2 : 1, SPAN = 16 * U;  // columns a wave takes at a time
  float x[WIDE ? TT : U][WIDE ? 4 : TT][4];
  // the strides as the compiler cannot know them from the round before: it would keep the addresses of all entries in registers otherwise
  auto afresh = [](Strided v) {
    asm volatile("" : "+s"(v.row), "+s"(v.col));
    return v;
  };
  auto load = [&](int64_t base) {
    const Strided from = afresh(a.g);
    if (WIDE) {
#pragma unroll
      for (int k = 0; k < TT; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) small_load4<T, true>(from, p, s, l1, a.gvec, 16 * k + 4 * g + r, base + 4 * c, x[k][r]);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < TT; ++k) small_load4<T, false>(from, p, s, l1, a.gvec, 16 * k + 4 * g, base + 16 * u + c, x[u][k]);
    }
  };
  const int64_t base0 = l0 + (int64_t)w * SPAN;
  if (TT == 1) load(base0);  // on its way during the iteration
  A mine[LDS ? 1 : TT][LDS ? 1 : TT][4];
  int ex = 0;
  if constexpr (TT == 1) {
    const double *part = a.part + (int64_t)by * a.chunks * s * s;
    const int y = t >> 4, x = t & 15;
    double v[4] = {0, 0, 0, 0};
    if (y < s && x < s) {
      const double *e = part + y * s + x;
      int k = 0;
      for (; k + 16 <= a.chunks; k += 16) {  // sixteen loads in flight
        double u[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) u[r] = e[(int64_t)(k + r) * s * s];
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r & 3] += u[r];
      }
      for (; k + 4 <= a.chunks; k += 4)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += e[(int64_t)(k + r) * s * s];
      for (; k < a.chunks; ++k) v[0] += e[(int64_t)k * s * s];
    }
    sum[t] = (v[0] + v[1]) + (v[2] + v[3]);
    __syncthreads();
    if (w == 0) {
      f64x4 S, P, Q = {0, 0, 0, 0};
      double norm2 = 0, inv2, inv;
#pragma unroll
      for (int r = 0; r < 4; ++r) S[r] = sum[(4 * r + g) * 16 + c];
#pragma unroll
      for (int i = 0; i < 16; ++i) norm2 += sum[i * 17];
      small_norm(norm2, a.first, inv2, inv);
      S *= inv2;
      for (int k = 0; k < a.steps; ++k) {
        P = cf.v[3 * k + 1] * S + cf.v[3 * k + 2] * sym_product(S, S);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (4 * r + g == c) P[r] += cf.v[3 * k];
        if (k + 1 < a.steps) S = sym_product(sym_product(S, P), P);
        Q = k == 0 ? P : sym_product(Q, P);
      }
      const int e = small_exponent(norm2, Q64);
      inv = ldexp(inv, -e);
      if (lane == 0) exponent = e;
#pragma unroll
      for (int r = 0; r < 4; ++r) own[small_q_at<1>(4 * r + g, c, Q64)] = (A)(Q[r] * inv);
    }
    __syncthreads();
    ex = __builtin_amdgcn_readfirstlane(exponent);
#pragma unroll
    for (int k = 0; k < 4; ++k) mine[0][0][k] = own[k * 64 + lane];
  } else {
    const double *m = a.q + (int64_t)by * small_q_size<TT>();
    if constexpr (LDS) {
      for (int e = t; e < TT * TT * 128; e += 256) ((i32x4 *)qs)[e] = ((const i32x4 *)m)[e];
      __syncthreads();
    } else {
      ex = __builtin_amdgcn_readfirstlane((int)m[TT * TT * 256]);
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) mine[i][j][k] = (A)m[((i * TT + j) * 4 + k) * 64 + lane];
    }
  }
  auto q = [&](int i, int j, int k) -> A {
    if constexpr (LDS)
      return qs[((i * TT + j) * 4 + k) * 64 + lane];
    else
      return mine[i][j][k];
  };
  auto scale = [&]() {
#pragma unroll
    for (int i = 0; i < (WIDE ? TT : U); ++i)
#pragma unroll
      for (int k = 0; k < (WIDE ? 4 : TT); ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][k][e] = ldexpf(x[i][k][e], ex);
  };
  Strided to = a.o;
  auto store_wide = [&](int row, int64_t j, float v0, float v1, float v2, float v3) {  // entries j .. j + 3 of a row
    if (row >= s) return;
    O *z = o + row * to.row + j * to.col;
    if (a.ovec && j + 4 <= l1) {
      write4(z, v0, v1, v2, v3);
    } else {
      const float v[4] = {v0, v1, v2, v3};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e < l1) z[e * to.col] = from_f32<O>(v[e]);
    }
  };
  auto store_tall = [&](int row, int64_t j, const vec &v) {  // entries row .. row + 3 of a column
    O *z = o + row * to.row + j * to.col;
    if (a.ovec && row + 4 <= s) {
      write4(z, (float)v[0], (float)v[1], (float)v[2], (float)v[3]);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (row + r < s) z[r * to.row] = from_f32<O>((float)v[r]);
    }
  };
  for (int64_t base = base0; base < l1; base += 4 * SPAN) {
    if (TT > 1) load(base);
    to = afresh(a.o);
    if (!Q64 && ex) scale();
    if constexpr (LDS) asm volatile("" ::: "memory");  // Q is read in every round: it would not fit into the registers
    if constexpr (WIDE && LDS) {
      // a column of the lane's four at a time, all rows: O's entries take the places of G's, whose column is no longer needed
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        vec d[TT];
#pragma unroll
        for (int i = 0; i < TT; ++i) d[i] = (vec){0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < TT; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const A v = (A)x[k][r][e];
#pragma unroll
            for (int i = 0; i < TT; ++i) d[i] = small_multiply(q(i, k, r), v, d[i]);
          }
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[i][r][e] = (float)d[i][r];
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) store_wide(16 * i + 4 * g + r, base + 4 * c, x[i][r][0], x[i][r][1], x[i][r][2], x[i][r][3]);
    } else if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        vec d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = (vec){0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < TT; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = small_multiply(q(i, k, r), (A)x[k][r][e], d[e]);
        if (TT == 1) load(base + 4 * SPAN);
#pragma unroll
        for (int r = 0; r < 4; ++r) store_wide(16 * i + 4 * g + r, base + 4 * c, (float)d[0][r], (float)d[1][r], (float)d[2][r], (float)d[3][r]);
        if (TT > 1) __builtin_amdgcn_sched_barrier(0);  // (rows of tiles one after the other: all at once take twice the registers)
      }
    } else {
      vec d[U][TT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < TT; ++i) d[u][i] = (vec){0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < TT; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const A v = (A)x[u][k][r];
#pragma unroll
            for (int i = 0; i < TT; ++i) d[u][i] = small_multiply(q(i, k, r), v, d[u][i]);
          }
      }
      if (TT == 1) load(base + 4 * SPAN);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t j = base + 16 * u + c;
        if (j >= l1) continue;
#pragma unroll
        for (int i = 0; i < TT; ++i) store_tall(16 * i + 4 * g, j, d[u][i]);
      }
    }
  }
}

// ---- s > 96 ----------------------------------------------------------------------------------------------------------------------
//
// A split matrix: rows of 128-byte blocks, a block = the hi parts of 32 consecutive entries, then their lo parts; zeros behind the last entry.

struct Split {
  char *p;
  int64_t batch, ld;  // bytes
};

__device__ __forceinline__ void split4(f32x4 v, f16x4 &hi, f16x4 &lo) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    hi[r] = (_Float16)v[r];
    lo[r] = (_Float16)(v[r] - (float)hi[r]);
  }
}
// entries col .. col + 3 of a row (col a multiple of 4)
__device__ __forceinline__ void put4(char *row, int col, f32x4 v) {
  f16x4 hi, lo;
  split4(v, hi, lo);
  char *q = row + (col >> 5) * 128 + (col & 31) * 2;
  *(f16x4 *)q = hi;
  *(f16x4 *)(q + 64) = lo;
}
__device__ __forceinline__ void put1(char *row, int col, float v) {
  const _Float16 hi = (_Float16)v, lo = (_Float16)(v - (float)hi);
  char *q = row + (col >> 5) * 128 + (col & 31) * 2;
  *(_Float16 *)q = hi;
  *(_Float16 *)(q + 64) = lo;
}
__device__ __forceinline__ f32x4 get4(const char *row, int col) {
  const char *q = row + (col >> 5) * 128 + (col & 31) * 2;
  const f16x4 hi = *(const f16x4 *)q, lo = *(const f16x4 *)(q + 64);
  f32x4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = (float)hi[r] + (float)lo[r];
  return v;
}

constexpr int NORM_PARTS = 256;  // at most: one for each thread of split_kernel

// |G|^2 in 64 bits, as partial sums of gridDim.x workgroups per matrix: a wave walks rows along the contiguous side, four entries a lane
template <typename T>
__global__ __launch_bounds__(256) void norm_kernel(Strided g, int64_t b0, int s, int64_t l, double *part, int vec) {
  const int64_t b = b0 + blockIdx.y;
  const bool flip = g.row == 1;
  const int64_t outer = flip ? l : s, inner = flip ? s : l;
  const int64_t so = flip ? g.col : g.row, si = flip ? g.row : g.col;
  const T *p = (const T *)g.p + b * g.batch;
  double v = 0;
  const int lane = threadIdx.x & 63;
  for (int64_t o = blockIdx.x + gridDim.x * (threadIdx.x >> 6); o < outer; o += 4 * gridDim.x) {
    const T *q = p + o * so;
#pragma unroll 4
    for (int64_t e = lane * 4; e < inner; e += 256) {
      float x[4];
      if (vec && e + 4 <= inner) {
        read4(q + e, x);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = e + k < inner ? to_f32(q[(e + k) * si]) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) v = fma((double)x[k], (double)x[k], v);
    }
  }
  __shared__ double sum[4];
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = ((sum[0] + sum[1]) + sum[2]) + sum[3];
}

// X' = (G * (1 / |G|) * 2^e)', split: l rows of s entries, and rows of zeros up to a multiple of 32.  A 64 x 64 tile per workgroup, turned in LDS.
template <typename T>
__global__ __launch_bounds__(256) void split_kernel(Strided g, int64_t b0, int s, int64_t l, const double *part, int parts, double pow2, Split xt) {
  __shared__ float tile[64][65];
  const int t = threadIdx.x;
  const int64_t b = b0 + blockIdx.z;
  __shared__ double sums[4];
  double norm2 = t < parts ? part[(int64_t)blockIdx.z * parts + t] : 0.0;
#pragma unroll
  for (int o = 32; o; o >>= 1) norm2 += __shfl_xor(norm2, o);
  if ((t & 63) == 0) sums[t >> 6] = norm2;
  __syncthreads();
  norm2 = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  const double scale = !(norm2 <= 1.7e308) ? __longlong_as_double(0x7ff8000000000000ll) : norm2 > 0 ? pow2 / sqrt(norm2) : 0.0;
  const int64_t j0 = (int64_t)blockIdx.x * 64;
  const int i0 = blockIdx.y * 64;
  const int64_t lp = (l + 31) & ~(int64_t)31;
  const int sp = (s + 31) & ~31;
#pragma unroll 4
  for (int k = 0; k < 16; ++k) {
    const int e = t + k * 256, u = e >> 6, v = e & 63;
    const int i = g.row == 1 ? v : u, j = g.row == 1 ? u : v;
    tile[i][j] = i0 + i < s && j0 + j < l ? (float)(scale * (double)read_at<T>(g, b, i0 + i, j0 + j)) : 0.f;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int e = t + k * 256, u = e >> 4, v = (e & 15) * 4;
    if (j0 + u < lp && i0 + v < sp)
      put4(xt.p + blockIdx.z * xt.batch + (j0 + u) * xt.ld, i0 + v, (f32x4){tile[v][u], tile[v + 1][u], tile[v + 2][u], tile[v + 3][u]});
  }
}

enum { GRAM = 0, SYM = 1, APPLY = 2, LAST = 3 };

struct GemmArgs {
  Split p, q;    // C[i, j] = sum_k P[i, k] Q[j, k]; GRAM: sum_k P[k, i] P[k, j]
  int m, n, kb;  // kb: blocks of 32
  float mul, add;  // result = mul * C + add * D
  Split d;           // read where add is not zero; SYM: [i, j], APPLY and LAST: [j, i]
  Split out;         // GRAM and SYM: [i, j] and [j, i], APPLY: [j, i]
  int tiles_n;
  // GRAM and SYM: the workgroups from `whole` on are the rest of the tiles, `splits` workgroups for each; partial sums as [tile of the rest][split][side][side]
  float *part;
  int tiles, whole, rest, splits, kb_split;
  Strided o;  // LAST
  int64_t b0;
  int vec;
};

__device__ __forceinline__ void sym_tile(int id, int &ti, int &tj) {  // the tiles on and below the diagonal, row by row
  ti = (int)((sqrtf(8.f * id + 1.f) - 1.f) * 0.5f);
  while ((ti + 1) * (ti + 2) / 2 <= id) ++ti;
  while (ti * (ti + 1) / 2 > id) --ti;
  tj = id - ti * (ti + 1) / 2;
}

// Operands of GRAM: the hi and lo parts of a tile's columns, eight entries a lane, each out of two reads that turn 4 x 16 entries (OFF: bytes from the first
// four rows to the next).  In assembly with their wait, because the compiler puts a wait for all copies into LDS before the builtin.
using pair64 = __attribute__((ext_vector_type(2))) uint32_t;
struct Turned {
  f16x8 hi, lo;
};
__device__ __forceinline__ f16x8 join8(pair64 a, pair64 b) {
  const i32x4 v = {(int)a[0], (int)a[1], (int)b[0], (int)b[1]};
  return __builtin_bit_cast(f16x8, v);
}
template <int OFF>
__device__ __forceinline__ Turned read_turned(uint32_t hi, uint32_t lo) {
  pair64 a, b, c, d;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\tds_read_b64_tr_b16 %2, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d)
      : "v"(hi), "v"(lo), "n"(OFF)
      : "memory");
  return {join8(a, b), join8(c, d)};
}
template <int OFF>
__device__ __forceinline__ void read_turned2(uint32_t h0, uint32_t l0, uint32_t h1, uint32_t l1, Turned &x, Turned &y) {
  pair64 a, b, c, d, e, f, g, h;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\tds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\tds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d), "=&v"(e), "=&v"(f), "=&v"(g), "=&v"(h)
      : "v"(h0), "v"(l0), "v"(h1), "v"(l1), "n"(OFF)
      : "memory");
  x = {join8(a, b), join8(c, d)};
  y = {join8(e, f), join8(g, h)};
}

// BM x BN outputs a workgroup, WM x WN waves.  GRAM and SYM: the result is symmetric, only the tiles on and below the diagonal are computed and each is
// written to both places.
// What bounds it is the matrix pipes: per block of 32 a 16 x 16 tile takes three instructions of 16 cycles (4096 x 4096: 1.1 .. 1.25 PFLOP/s of these, where a
// large fp16 product of the vendor's library runs at 1.4 on the same card).  Two buffers in LDS; a wave holds Q's operands of a block in
// registers, so Q's half of a buffer is free after the first row of tiles and P's before the last one: at these two places the waves meet and
// start the copies of the block after the next.  The operands of a row are requested a row ahead.
//
// GRAM sums over l, and X stands as l rows of s: X is kept in this one orientation, half of the memory traffic of keeping both.  32 rows of a block are
// copied as they are, a row's 32-byte segment q (16 hi or 16 lo parts) at segment q ^ f(row); ds_read_b64_tr_b16 turns 4 rows x 16 columns for 16
// lanes, so that a lane gets eight entries of its column.  f takes the 16 rows that an instruction touches to 16 (at a side of 64: 8) segments.
// APPLY: a lane's four results are neighbours along s, which is how X' stands.
template <int MODE, typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void gemm_kernel(GemmArgs a) {
  constexpr int STAGE = (BM + BN) * 128, WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr bool TURNED = MODE == GRAM, HALF = MODE == GRAM || MODE == SYM;
  static_assert(!HALF || BM == BN, "");
  static_assert(TM >= 4, "Q is copied between row 1 and row TM - 2");
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  int ti, tj, kb0 = 0, kb1 = a.kb;
  int64_t b = blockIdx.z;
  bool partial = false;
  int slot = 0;
  if (HALF) {
    int id = blockIdx.x;
    if (id < a.whole) {
      id = xcd_order(id, a.whole);
    } else {
      // an XCD gets tiles of one matrix and one part of the sum: they share rows
      id = xcd_order(id - a.whole, a.rest * a.splits);
      const int k = id / (a.tiles * a.splits), left = id - k * a.tiles * a.splits, here = min(a.tiles, a.rest - k * a.tiles), split = left / here;
      const int tile = k * a.tiles + left - split * here;
      partial = a.splits > 1;
      slot = tile * a.splits + split;
      kb0 = split * a.kb_split;
      kb1 = min(a.kb, kb0 + a.kb_split);
      id = a.whole + tile;
    }
    b = id / a.tiles;
    sym_tile(id - (int)b * a.tiles, ti, tj);
  } else {
    tile_at(xcd_order(blockIdx.x, gridDim.x), (a.m + BM - 1) / BM, a.tiles_n, BM == 256 ? 4 : 8, ti, tj);
  }
  const int i0 = ti * BM, j0 = tj * BN;
  constexpr int CP = BM / 8 / WAVES, CQ = BN / 8 / WAVES;  // copies of 1024 bytes a wave
  static_assert(CP * 8 * WAVES == BM && CQ * 8 * WAVES == BN, "");
  const char *pp, *pq;
  int64_t advance;
  uint32_t off_p[CP], off_q[CQ];
  if (TURNED) {
    // A copy is 1024 / (4 BM) rows.  Columns behind the last block repeat the first (their results are not stored); rows are whole blocks of 32.  An
    // offset: at most 32 rows of 2^17 bytes.
    constexpr int ROW = BM * 4, PER = 64 / (ROW / 16);
    pp = a.p.p + b * a.p.batch + (int64_t)kb0 * 32 * a.p.ld;
    pq = pp;
    advance = 32 * a.p.ld;
    const int row = lane / (ROW / 16), chunk = lane % (ROW / 16);
    auto offset = [&](int k, int c0) {
      const int r = k * PER + row, seg = (chunk >> 1) ^ (((r & 3) | ((r >> 3) & 3) << 2) & (ROW / 32 - 1));
      const int at = c0 * 4 + seg * 32;
      return (uint32_t)(r * (int)a.p.ld + (at < (int)a.p.ld ? at : 0) + (chunk & 1) * 16);
    };
#pragma unroll
    for (int k = 0; k < CP; ++k) off_p[k] = offset(k * WAVES + w, i0);
#pragma unroll
    for (int k = 0; k < CQ; ++k) off_q[k] = offset(k * WAVES + w, j0);
  } else {
    // rows behind the last one repeat it.  A lane's offset from its tile's first row: at most 256 rows of 2^17 bytes
    const int lr = lane >> 3, lc = ((lane & 7) ^ lr) << 4;
    pp = a.p.p + b * a.p.batch + i0 * a.p.ld + (int64_t)kb0 * 128;
    pq = a.q.p + b * a.q.batch + j0 * a.q.ld + (int64_t)kb0 * 128;
    advance = 128;
#pragma unroll
    for (int k = 0; k < CP; ++k) off_p[k] = (uint32_t)min((k * WAVES + w) * 8 + lr, a.m - 1 - i0) * (uint32_t)a.p.ld + lc;
#pragma unroll
    for (int k = 0; k < CQ; ++k) off_q[k] = (uint32_t)min((k * WAVES + w) * 8 + lr, a.n - 1 - j0) * (uint32_t)a.q.ld + lc;
  }
  auto stage_p = [&](int buf) {
#pragma unroll
    for (int k = 0; k < CP; ++k) stage8(pp + off_p[k], lds + buf * STAGE + (k * WAVES + w) * 1024);
    pp += advance;
  };
  auto stage_q = [&](int buf) {
#pragma unroll
    for (int k = 0; k < CQ; ++k) stage8(pq + off_q[k], lds + buf * STAGE + BM * 128 + (k * WAVES + w) * 1024);
    pq += advance;
  };
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int fr = lane & 15, fg = lane >> 4, wi = (w / WN) * (BM / WM), wj = (w % WN) * (BN / WN);
  const int turn_row = 8 * fg + (fr >> 2), turn_seg = ((fr >> 2) | fg << 2) & (BM * 4 / 32 - 1), turn_at = turn_row * (BM * 4) + (fr & 3) * 8;
  auto turned = [&](int part, int tile, int half) {  // part: byte offset of the operand in LDS, tile: its first column
    const int seg = (tile >> 5) * 4 + half * 2 + ((tile >> 4) & 1);
    return (uint32_t)(uintptr_t)(lvoid *)(lds + part + turn_at + ((seg ^ turn_seg) << 5));
  };
  auto read_p = [&](int buf, int i, f16x8 &h, f16x8 &l) {
    const int part = buf * STAGE, tile = wi + i * 16;
    if (TURNED) {
      const Turned v = read_turned<16 * BM>(turned(part, tile, 0), turned(part, tile, 1));
      h = v.hi, l = v.lo;
    } else {
      h = __builtin_bit_cast(f16x8, lds_chunk(lds + part, tile + fr, fg));
      l = __builtin_bit_cast(f16x8, lds_chunk(lds + part, tile + fr, fg + 4));
    }
  };
  auto frag_q = [&](int buf, int j, int half) { return __builtin_bit_cast(f16x8, lds_chunk(lds + buf * STAGE + BM * 128, wj + j * 16 + fr, fg + 4 * half)); };
  auto turn_q = [&](int buf, f16x8 (&h)[TN], f16x8 (&l)[TN]) {
    const int part = buf * STAGE + BM * 128;
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
      Turned x, y;
      read_turned2<16 * BM>(turned(part, wj + j * 16, 0), turned(part, wj + j * 16, 1), turned(part, wj + j * 16 + 16, 0), turned(part, wj + j * 16 + 16, 1), x, y);
      h[j] = x.hi, l[j] = x.lo, h[j + 1] = y.hi, l[j + 1] = y.lo;
    }
  };
  auto multiply = [&](const f16x8 &p, const f16x8 &q, f32x4 c) {
    return HALF ? __builtin_amdgcn_mfma_f32_16x16x32_f16(q, p, c, 0, 0, 0) : __builtin_amdgcn_mfma_f32_16x16x32_f16(p, q, c, 0, 0, 0);
  };
  if (kb0 < kb1) {
    stage_p(0);
    stage_q(0);
    staged();
    meet();
    if (kb0 + 1 < kb1) {
      stage_p(1);
      stage_q(1);
    }
    f16x8 qh[TN], ql[TN], ph, pl;
    read_p(0, 0, ph, pl);
    if (TURNED) {
      turn_q(0, qh, ql);
    } else {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        qh[j] = frag_q(0, j, 0);
        ql[j] = frag_q(0, j, 1);
      }
    }
    int buf = 0;
    for (int kb = kb0; kb < kb1; ++kb) {  // (behind the last block the operands of "the next" are whatever stands in LDS, unused)
      const bool copy = kb + 2 < kb1;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if (i == 1 && copy) {
          meet();
          stage_q(buf);
        }
        f16x8 ph_next, pl_next;
        if (i < TM - 1) {
          read_p(buf, i + 1, ph_next, pl_next);
        } else {
          if (copy) {
            staged_but<CQ>();  // of the block after the next, Q may still be on its way
            meet();
            stage_p(buf);
          } else {
            staged();
            meet();
          }
          read_p(buf ^ 1, 0, ph_next, pl_next);
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = multiply(ph, ql[j], acc[i][j]);
        if (i == TM - 1 && !TURNED) {
#pragma unroll
          for (int j = 0; j < TN; ++j) ql[j] = frag_q(buf ^ 1, j, 1);
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = multiply(pl, qh[j], acc[i][j]);
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = multiply(ph, qh[j], acc[i][j]);
        if (i == TM - 1) {
          if (TURNED) {
            turn_q(buf ^ 1, qh, ql);
          } else {
#pragma unroll
            for (int j = 0; j < TN; ++j) qh[j] = frag_q(buf ^ 1, j, 0);
          }
        }
        ph = ph_next;
        pl = pl_next;
        __builtin_amdgcn_sched_barrier(0);
      }
      buf ^= 1;
    }
  }
  const int mp = (a.m + 31) & ~31, np = (a.n + 31) & ~31;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      f32x4 v = acc[i][j];
      f32x4 d = {0.f, 0.f, 0.f, 0.f};
      if (HALF) {
        const int m = i0 + wi + i * 16 + fr, n = j0 + wj + j * 16 + fg * 4;
        if (partial) {
          *(f32x4 *)(a.part + (int64_t)slot * (BM * BN) + (m - i0) * BN + (n - j0)) = v;
          continue;
        }
        if (a.add != 0.f && m < a.m && n < np) d = get4(a.d.p + b * a.d.batch + (int64_t)m * a.d.ld, n);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = m < a.m && n + r < a.n ? fmaf(a.mul, v[r], a.add * d[r]) : 0.f;
        if (m < a.m && n < np) put4(a.out.p + b * a.out.batch + (int64_t)m * a.out.ld, n, v);
        if (ti == tj || m >= mp) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < a.n) put1(a.out.p + b * a.out.batch + (int64_t)(n + r) * a.out.ld, m, v[r]);
      } else {
        const int m = i0 + wi + i * 16 + fg * 4, n = j0 + wj + j * 16 + fr;
        if (m >= mp || n >= np) continue;
        if (n < a.n) d = get4(a.d.p + b * a.d.batch + (int64_t)n * a.d.ld, m);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = m + r < a.m && n < a.n ? fmaf(a.mul, v[r], a.add * d[r]) : 0.f;
        if (MODE == APPLY) {
          put4(a.out.p + b * a.out.batch + (int64_t)n * a.out.ld, m, v);
        } else if (n < a.n) {
          T *q = (T *)a.o.p + (a.b0 + b) * a.o.batch + m * a.o.row + (int64_t)n * a.o.col;
          if (a.vec && m + 4 <= a.m) {
            write4(q, v[0], v[1], v[2], v[3]);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (m + r < a.m) q[r * a.o.row] = from_f32<T>(v[r]);
          }
        }
      }
    }
  }
}

// The tiles whose sum was split: the partial sums in the order of the splits, then what the tile's own workgroup would have done.  32 x 32 results
// a workgroup, turned in LDS for the place across the diagonal.
template <int TS>
__global__ __launch_bounds__(256) void sym_join_kernel(GemmArgs a) {
  __shared__ float turn[32][33];
  const int t = threadIdx.x, y = t >> 3, x = (t & 7) * 4;
  const int id = a.whole + blockIdx.x, b = id / a.tiles;
  int ti, tj;
  sym_tile(id - b * a.tiles, ti, tj);
  const int u0 = blockIdx.y / (TS / 32) * 32, v0 = blockIdx.y % (TS / 32) * 32;
  const int m0 = ti * TS + u0, n0 = tj * TS + v0, m = m0 + y, n = n0 + x, mp = (a.m + 31) & ~31;
  if (m0 >= mp || n0 >= mp) return;
  const float *p = a.part + (int64_t)blockIdx.x * a.splits * (TS * TS) + (u0 + y) * TS + v0 + x;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 0; k < a.splits; ++k) v += *(const f32x4 *)(p + (int64_t)k * (TS * TS));
  f32x4 d = {0.f, 0.f, 0.f, 0.f};
  if (a.add != 0.f && m < a.m) d = get4(a.d.p + b * a.d.batch + (int64_t)m * a.d.ld, n);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    v[r] = m < a.m && n + r < a.m ? fmaf(a.mul, v[r], a.add * d[r]) : 0.f;
    turn[y][x + r] = v[r];
  }
  if (m < a.m) put4(a.out.p + b * a.out.batch + (int64_t)m * a.out.ld, n, v);
  if (ti == tj) return;
  __syncthreads();
  if (n0 + y < a.m) put4(a.out.p + b * a.out.batch + (int64_t)(n0 + y) * a.out.ld, m0 + x, (f32x4){turn[x][y], turn[x + 1][y], turn[x + 2][y], turn[x + 3][y]});
}

// ---- host ------------------------------------------------------------------------------------------------------------------------

// Which tiles a product is cut into.  Small tiles fill the 256 CUs where there is little to do, large ones read less for each operation.  The estimate, in
// microseconds, measured: `places` tiles of a side run at a time (LDS: 128, 64, 32 KB a workgroup); such a round takes `step` for each block of
// 32 of the sum, and `rest` to begin and to write.  A round that is not full takes less of `step`: GRAM and SYM the part of it that is filled, but at
// least `alone`; APPLY and LAST `base` and the filled part of what remains (1000 x 1000 in 256 tiles of 64: 18 us, in 64 tiles of 128: 27).
struct TileCost {
  int side;
  int64_t places;
  double step, alone, base, rest, part;  // part: a partial sum to write and read again
};
constexpr TileCost COST[3] = {{64, 1024, 0.95, 0.85, 0.2, 4, 0.008}, {128, 512, 1.35, 0.55, 0, 6, 0.03}, {256, 256, 2.6, 1.0, 0, 16, 0}};

double tiles_cost(const TileCost &c, int64_t tiles, int64_t kb, bool sym) {
  const int64_t full = tiles / c.places, rest = tiles - full * c.places;
  const double filled = (double)nmfk_div_up(rest, 256) * 256.0 / (double)c.places, share = sym ? std::max(filled, c.alone) : c.base + (1 - c.base) * filled;
  return (double)full * (c.step * (double)kb + c.rest) + (rest ? c.step * share * (double)kb + c.rest : 0.0);
}

// A symmetric product: the last round of tiles is rarely full, so the sums of its tiles may be split (the launch that joins them costs 4).  4096 x 4096 with
// 528 tiles of 128: the 16 of the second round in 16 parts, 226 -> 185.
struct SymPlan {
  int side;
  int tiles;  // a matrix
  int whole, rest, splits, kb_split;
};

SymPlan sym_plan(int64_t m, int64_t batch, int64_t kb) {
  SymPlan best = {};
  double least = 1e30;
  for (const TileCost &c : COST) {
    if (c.side == 256) continue;
    const int64_t tm = nmfk_div_up(m, c.side), tiles = tm * (tm + 1) / 2, total = tiles * batch;
    if (total > 0x7fffffff / 64) continue;
    const int64_t whole = total / c.places * c.places, rest = total - whole;
    const double before = tiles_cost(c, whole, kb, true);
    for (int64_t s = 1; s <= 64 && (s == 1 || (s * 4 <= kb && s * rest <= 3 * c.places)); ++s) {
      const double cost = before + tiles_cost(c, rest * s, nmfk_div_up(kb, s), true) + (s > 1 ? c.part * (double)(rest * s) + 4.0 : 0.0);
      if (cost >= least) continue;
      least = cost;
      best = {c.side, (int)tiles, (int)whole, (int)rest, (int)s, (int)nmfk_div_up(kb, s)};
    }
  }
  best.splits = (int)nmfk_div_up(kb, best.kb_split);
  if (best.splits == 1) best.whole += best.rest, best.rest = 0;
  return best;
}

int full_side(int64_t m, int64_t n, int64_t batch, int64_t kb) {
  int side = 0;
  double least = 1e30;
  for (const TileCost &c : COST) {
    const double cost = tiles_cost(c, nmfk_div_up(m, c.side) * nmfk_div_up(n, c.side) * batch, kb, false);
    if (cost < least) least = cost, side = c.side;
  }
  return side;
}

struct Layout {
  int64_t s, l, batch;
  int64_t chunks, chunk, portion, x;    // small; portion: matrices of 16 bits that more than one group of steps works on at a time
  int64_t xt[2], sq[2], norm, part, q;  // byte offsets
  int64_t ldt, lp;
  int64_t bytes;
};

int64_t small_q_bytes(int64_t s) { return s <= 16 ? 0 : (nmfk_div_up(s, 16) * nmfk_div_up(s, 16) * 256 + 32) * 8; }

Layout ortho_layout(int64_t batch, int64_t rows, int64_t cols) {
  Layout y = {};
  y.s = std::min(rows, cols);
  y.l = std::max(rows, cols);
  y.batch = batch;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += nmfk_round_up(bytes, 256);
    return o;
  };
  if (y.s <= SMALL) {
    // Workgroups a matrix.  Two for each CU while the matrices are few: what a workgroup does whatever its share (partial S, the iteration, Q) is 2 .. 6
    // microseconds of every round (20 of 30000 x 16: 33 us, with 2048 workgroups 61; 250 of 1000 x 48: 79 and 96).  Many matrices are a stream through
    // memory, where a short last round counts (480 of 8192 x 16 in 1920 workgroups 155, in 480 186; 600 of 3000 x 32 in 1800 244, in 600 270).
    const int64_t most = y.s <= 16 ? 256 : 128;
    y.chunks = batch <= 256 ? std::min(nmfk_div_up(y.l, most), 512 / batch) : std::min(nmfk_div_up(y.l, 1024), 2048 / batch);
    y.chunks = std::max<int64_t>(1, std::min(y.chunks, most));
    y.chunk = nmfk_round_up(nmfk_div_up(y.l, y.chunks), 64);
    y.chunks = nmfk_div_up(y.l, y.chunk);
    y.part = take(batch * y.chunks * y.s * y.s * 8);
    y.q = take(batch * small_q_bytes(y.s));
    y.portion = std::max<int64_t>(1, std::min(BATCH, PORTION / (4 * y.s * y.l)));
    y.x = take(4 * y.s * y.l * std::min(y.portion, batch));
  } else {
    y.lp = nmfk_round_up(y.l, 32);
    y.ldt = nmfk_round_up(y.s, 32) * 4;
    y.xt[0] = take(batch * y.lp * y.ldt);
    y.xt[1] = take(batch * y.lp * y.ldt);
    for (int k = 0; k < 2; ++k) y.sq[k] = take(batch * y.s * y.ldt);
    y.norm = take(batch * NORM_PARTS * 8);
    int64_t part = 0;
    for (int64_t b0 = 0; b0 < batch; b0 += BATCH)
      for (int64_t k : {y.l, y.s}) {
        const SymPlan q = sym_plan(y.s, std::min<int64_t>(BATCH, batch - b0), nmfk_div_up(k, 32));
        if (q.splits > 1) part = std::max<int64_t>(part, (int64_t)q.rest * q.splits * q.side * q.side * 4);
      }
    y.part = take(part);
  }
  y.bytes = at;
  return y;
}

enum { ODD = 1, EVEN = 0 };

// the largest |t (a + b t^2 + c t^4)| (ODD) or |a + b t^2 + c t^4| (EVEN) for 0 <= t <= u
double peak(double a, double b, double c, double u, int odd) {
  auto f = [&](double t) { return fabs((odd ? t : 1.0) * (a + t * t * (b + c * t * t))); };
  double best = std::max(f(0.0), f(u));
  auto at = [&](double x) {  // an extremum at t = sqrt(x)
    if (x > 0 && x < u * u) best = std::max(best, f(sqrt(x)));
  };
  if (!odd) {
    if (c != 0) at(-b / (2 * c));
  } else {
    // a + 3 b x + 5 c x^2 = 0: one root from the sum without cancellation, the other one from the roots' product
    const double disc = 9 * b * b - 20 * a * c;
    if (disc >= 0) {
      const double q = -0.5 * (3 * b + copysign(sqrt(disc), b));
      if (c != 0) at(q / (5 * c));
      if (q != 0) at(a / q);
    }
  }
  return best;
}

// What a step can multiply a singular value of at most u by, and then u itself
double step_growth(const double *c, double &u) {
  const double g = std::max(1.0, peak(c[0], c[1], c[2], u, EVEN));
  u = std::max(peak(c[0], c[1], c[2], u, ODD), TINY);
  return g;
}

// the power of two that brings `bound` to at most 2^15: an entry is never larger than the norm, and 65504 stays out of reach
int exponent(double bound) {
  int e;
  (void)frexp(bound, &e);  // bound < 2^e
  return std::min(15 - e, 100);
}

template <typename T, typename O, int TT, bool WIDE>
void small_launch(const SmallArgs &a, const Coefs &cf, unsigned nb, hipStream_t st) {
  const dim3 grid((unsigned)a.chunks, nb);
  small_gram_kernel<T, TT, WIDE><<<grid, 256, 0, st>>>(a);
  if (TT > 1) {
    constexpr int BYTES = small_lds(TT);
    static std::atomic<uint64_t> done{0};
    nmfk_allow_dynamic_lds((const void *)small_iterate_kernel<TT>, done, BYTES);
    if (a.chunks > SUMS) small_join_kernel<<<dim3((unsigned)nmfk_div_up((int64_t)a.s * a.s, 256), nb), 256, 0, st>>>(a);
    small_iterate_kernel<TT><<<dim3(nb), 64 * small_waves(TT), BYTES, st>>>(a, cf, a.chunks > SUMS ? 1 : a.chunks);
  }
  if constexpr (std::is_same<T, O>::value)
    if (!a.q64) {
      small_apply_kernel<T, O, float, TT, WIDE><<<grid, 256, 0, st>>>(a, cf);
      return;
    }
  constexpr int Q = TT > 1 ? TT * TT * 2048 : 0;
  if (TT > 1) {
    static std::atomic<uint64_t> done{0};
    nmfk_allow_dynamic_lds((const void *)small_apply_kernel<T, O, double, TT, WIDE>, done, Q);
  }
  small_apply_kernel<T, O, double, TT, WIDE><<<grid, 256, Q, st>>>(a, cf);
}

// one group of steps on nb matrices: O = Q G
template <typename T, typename O>
void small_group(SmallArgs a, const Strided &g, const Strided &o, int steps, const double *coef, unsigned nb, hipStream_t st) {
  Coefs cf = {};
  for (int k = 0; k < 3 * steps; ++k) cf.v[k] = coef[k];
  const bool wide = g.col == 1 && g.row != 1;
  a.g = g;
  a.o = o;
  a.steps = steps;
  a.gvec = wide || g.row == 1;
  a.ovec = (wide ? o.col : o.row) == 1;
#define NMFK_SMALL(TT) (wide ? small_launch<T, O, TT, true>(a, cf, nb, st) : small_launch<T, O, TT, false>(a, cf, nb, st))
  if (a.s <= 16)
    NMFK_SMALL(1);
  else if (a.s <= 32)
    NMFK_SMALL(2);
  else if (a.s <= 48)
    NMFK_SMALL(3);
  else if (a.s <= 64)
    NMFK_SMALL(4);
  else if (a.s <= 80)
    NMFK_SMALL(5);
  else
    NMFK_SMALL(6);
#undef NMFK_SMALL
}

template <typename T>
int ortho_small(const Layout &y, const Strided &g, const Strided &o, int steps, const double *coef, char *work, hipStream_t st) {
  constexpr bool F32 = std::is_same<T, float>::value;
  int end[32], groups = 0;
  double growth = 1, u = 1;
  for (int k = 0; k < steps; ++k) {
    const double by = step_growth(coef + 3 * k, u);
    if (k > (groups ? end[groups - 1] : 0) && growth * by > GROWTH) {
      end[groups++] = k;
      growth = 1;
    }
    growth *= by;
  }
  end[groups++] = steps;
  const int64_t most = groups > 1 && !F32 ? y.portion : BATCH;
  for (int64_t b0 = 0; b0 < y.batch; b0 += most) {
    const unsigned nb = (unsigned)std::min<int64_t>(most, y.batch - b0);
    SmallArgs a = {};
    a.part = (double *)(work + y.part) + b0 * y.chunks * y.s * y.s;
    a.q = (double *)(work + y.q + b0 * small_q_bytes(y.s));
    a.s = (int)y.s;
    a.chunks = (int)y.chunks;
    a.l = y.l;
    a.chunk = y.chunk;
    a.first = 1;
    a.q64 = groups > 1 || growth > GROWTH32;
    Strided from = g, to = o;
    from.p += b0 * g.batch * (int64_t)sizeof(T);
    to.p += b0 * o.batch * (int64_t)sizeof(T);
    if (groups == 1) {
      small_group<T, T>(a, from, to, steps, coef, nb, st);
      continue;
    }
    // between the groups X is O itself, or stands in the workspace along the side that is contiguous in G
    Strided x = to;
    if (!F32) x = g.col == 1 && g.row != 1 ? Strided{work + y.x, y.s * y.l, y.l, 1} : Strided{work + y.x, y.s * y.l, 1, y.s};
    small_group<T, float>(a, from, x, end[0], coef, nb, st);
    a.first = 0;
    for (int k = 1; k + 1 < groups; ++k) small_group<float, float>(a, x, x, end[k] - end[k - 1], coef + 3 * end[k - 1], nb, st);
    small_group<float, T>(a, x, to, steps - end[groups - 2], coef + 3 * end[groups - 2], nb, st);
  }
  return nmfk_launched("nmfk_orthogonalize");
}

template <int MODE, typename T, int BM, int BN, int WM, int WN>
void gemm_tile(const GemmArgs &a, dim3 grid, hipStream_t st) {
  constexpr int BYTES = 2 * (BM + BN) * 128;
  static std::atomic<uint64_t> done{0};
  nmfk_allow_dynamic_lds((const void *)gemm_kernel<MODE, T, BM, BN, WM, WN>, done, BYTES);
  gemm_kernel<MODE, T, BM, BN, WM, WN><<<grid, 64 * WM * WN, BYTES, st>>>(a);
}

// GRAM or SYM: the tiles on and below the diagonal
template <int MODE>
void gemm_sym(GemmArgs a, unsigned batch, hipStream_t st) {
  const SymPlan q = sym_plan(a.m, batch, a.kb);
  a.n = a.m;
  a.tiles = q.tiles;
  a.whole = q.whole;
  a.rest = q.rest;
  a.splits = q.splits;
  a.kb_split = q.kb_split;
  const dim3 grid((unsigned)(q.whole + q.rest * q.splits));
  if (q.side == 64)
    gemm_tile<MODE, float, 64, 64, 1, 2>(a, grid, st);
  else
    gemm_tile<MODE, float, 128, 128, 2, 2>(a, grid, st);
  if (!q.rest) return;
  if (q.side == 64)
    sym_join_kernel<64><<<dim3((unsigned)q.rest, 4), 256, 0, st>>>(a);
  else
    sym_join_kernel<128><<<dim3((unsigned)q.rest, 16), 256, 0, st>>>(a);
}

template <int MODE, typename T>
void gemm_full(GemmArgs a, unsigned batch, hipStream_t st) {
  const int side = full_side(a.m, a.n, batch, a.kb);
  a.tiles_n = (int)nmfk_div_up(a.n, side);
  const dim3 grid((unsigned)(nmfk_div_up(a.m, side) * a.tiles_n), 1, batch);
  if (side == 256)
    gemm_tile<MODE, T, 256, 256, 2, 4>(a, grid, st);
  else if (side == 128)
    gemm_tile<MODE, T, 128, 128, 2, 2>(a, grid, st);
  else
    gemm_tile<MODE, T, 64, 64, 1, 2>(a, grid, st);
}

// Each step forms S = X X', its polynomial P = b S + c S S and X <- a X + P X.  (The S of a later step could be had from the first one, S <- (a + P) S (a + P),
// which is cheaper for long rows; but then an error in a small eigenvalue grows by a^2 a step instead of a.  Measured on 100 x 66 with
// singular values 0.005 .. 0.84: 1.1e-4 after three such steps against 3e-7 of plain fp32.)
template <typename T>
int ortho_large(const Layout &y, const Strided &g, const Strided &o, int steps, const double *coef, char *work, hipStream_t st) {
  const int s = (int)y.s, l = (int)y.l, ks = (int)nmfk_div_up(s, 32), kl = (int)nmfk_div_up(l, 32);
  const int64_t bt = y.lp * y.ldt, bs = y.s * y.ldt;
  for (int64_t b0 = 0; b0 < y.batch; b0 += BATCH) {
    const unsigned nb = (unsigned)std::min<int64_t>(BATCH, y.batch - b0);
    Split X = {work + y.xt[0] + b0 * bt, bt, y.ldt}, N = {work + y.xt[1] + b0 * bt, bt, y.ldt};  // X', l rows of s
    Split S = {work + y.sq[0] + b0 * bs, bs, y.ldt}, P = {work + y.sq[1] + b0 * bs, bs, y.ldt};
    double *norm = (double *)(work + y.norm) + b0 * NORM_PARTS;
    double u = 1.0;  // bound of the singular values of X; e?: the power of two a matrix is scaled by
    int ex = exponent(1.01 * u);
    const unsigned parts = (unsigned)std::max<int64_t>(1, std::min<int64_t>(NORM_PARTS, 2048 / nb));  // 424 of 78 x 351: 82 us with 256 parts each, 16 so
    norm_kernel<T><<<dim3(parts, nb), 256, 0, st>>>(g, b0, s, l, norm, g.row == 1 || g.col == 1);
    split_kernel<T><<<dim3((unsigned)nmfk_div_up(l, 64), (unsigned)nmfk_div_up(s, 64), nb), 256, 0, st>>>(g, b0, s, l, norm, (int)parts, ldexp(1.0, ex), X);
    for (int k = 0; k < steps; ++k) {
      const double ca = coef[3 * k], cb = coef[3 * k + 1], cc = coef[3 * k + 2];
      const int es = exponent(1.02 * u * u), ep = exponent(1.02 * std::max(peak(0, cb, cc, u, EVEN), TINY));
      GemmArgs a = {};
      a.part = (float *)(work + y.part);  // (a launch's own: the next one starts behind the join)
      a.m = s;
      a.p = X;
      a.kb = kl;
      a.mul = (float)ldexp(1.0, es - 2 * ex);
      a.out = S;
      gemm_sym<GRAM>(a, nb, st);
      a.p = a.q = a.d = S;
      a.kb = ks;
      a.mul = (float)(cc * ldexp(1.0, ep - 2 * es));
      a.add = (float)(cb * ldexp(1.0, ep - es));
      a.out = P;
      gemm_sym<SYM>(a, nb, st);
      u = std::max(peak(ca, cb, cc, u, ODD), TINY);
      const bool last = k + 1 == steps;
      const int nx = last ? 0 : exponent(1.02 * u);
      a.p = P;
      a.q = a.d = X;
      a.n = l;
      a.mul = (float)ldexp(1.0, nx - ep - ex);
      a.add = (float)(ca * ldexp(1.0, nx - ex));
      a.out = N;
      if (last) {
        a.o = o;
        a.b0 = b0;
        a.vec = o.row == 1;
        gemm_full<LAST, T>(a, nb, st);
      } else {
        gemm_full<APPLY, float>(a, nb, st);
      }
      std::swap(X, N);
      ex = nx;
    }
  }
  return nmfk_launched("nmfk_orthogonalize");
}

int ortho_sizes(int64_t batch, int64_t rows, int64_t cols, const char *who) {
  if (batch < 0 || rows < 0 || cols < 0) return fail(NMFK_ERR_BAD_ARG, std::string(who) + ": negative size");
  if (batch > ((int64_t)1 << 22) || std::max(rows, cols) > ((int64_t)1 << 22)) return fail(NMFK_ERR_UNSUPPORTED, std::string(who) + ": a size above 2^22");
  if (std::min(rows, cols) > 32768) return fail(NMFK_ERR_UNSUPPORTED, std::string(who) + ": both sides above 32768");
  if (rows && cols && batch > ((int64_t)1 << 38) / (rows * cols)) return fail(NMFK_ERR_UNSUPPORTED, std::string(who) + ": more than 2^38 entries");
  return NMFK_OK;
}

}  // namespace

NMFK_EXPORT int nmfk_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols, int64_t *bytes) {
  if (!bytes) return fail(NMFK_ERR_BAD_ARG, "nmfk_orthogonalize_workspace: null pointer");
  if (int rc = ortho_sizes(batch, rows, cols, "nmfk_orthogonalize_workspace")) return rc;
  *bytes = batch && rows && cols ? ortho_layout(batch, rows, cols).bytes : 0;
  return NMFK_OK;
}

NMFK_EXPORT int nmfk_orthogonalize(int device, void *stream, int dtype, int64_t batch, int64_t rows, int64_t cols, const void *G,
                                   int64_t g_batch, int64_t g_row, int64_t g_col, void *O, int64_t o_batch, int64_t o_row, int64_t o_col,
                                   int steps, const double *coefficients, void *work, int64_t work_bytes) {
  if (int rc = ortho_sizes(batch, rows, cols, "nmfk_orthogonalize")) return rc;
  if (dtype < NMFK_F32 || dtype > NMFK_F16) return fail(NMFK_ERR_BAD_ARG, "nmfk_orthogonalize: dtype must be NMFK_F32, NMFK_BF16 or NMFK_F16");
  if (steps < 1 || steps > 32) return fail(NMFK_ERR_BAD_ARG, "nmfk_orthogonalize: 1 to 32 steps");
  if (!coefficients) return fail(NMFK_ERR_BAD_ARG, "nmfk_orthogonalize: null pointer");
  double u = 1.0;
  for (int k = 0; k < steps; ++k) {
    const double *c = coefficients + 3 * k;
    if (!(fabs(c[0]) <= 1e3 && fabs(c[1]) <= 1e3 && fabs(c[2]) <= 1e3)) return fail(NMFK_ERR_BAD_ARG, "nmfk_orthogonalize: a coefficient is not finite or above 1000");
    u = peak(c[0], c[1], c[2], u, ODD);
    if (u > 64.0) return fail(NMFK_ERR_BAD_ARG, "nmfk_orthogonalize: these coefficients let a singular value grow beyond 64");
  }
  if (batch == 0 || rows == 0 || cols == 0) return NMFK_OK;
  if (!G || !O) return fail(NMFK_ERR_BAD_ARG, "nmfk_orthogonalize: null pointer");
  const Layout y = ortho_layout(batch, rows, cols);
  if (!work || work_bytes < y.bytes || (uintptr_t)work % 256)
    return fail(NMFK_ERR_BAD_ARG, "nmfk_orthogonalize: the workspace is too small or not 256-byte aligned (nmfk_orthogonalize_workspace)");
  NmfkDeviceGuard guard(device);
  if (guard.status) return guard.status;
  const bool flip = rows > cols;
  const Strided g = {(char *)G, g_batch, flip ? g_col : g_row, flip ? g_row : g_col};
  const Strided o = {(char *)O, o_batch, flip ? o_col : o_row, flip ? o_row : o_col};
  hipStream_t st = (hipStream_t)stream;
  const bool small = y.s <= SMALL;
#define NMFK_ORTHO(T) (small ? ortho_small<T>(y, g, o, steps, coefficients, (char *)work, st) : ortho_large<T>(y, g, o, steps, coefficients, (char *)work, st))
  if (dtype == NMFK_F32) return NMFK_ORTHO(float);
  if (dtype == NMFK_BF16) return NMFK_ORTHO(bf16);
  return NMFK_ORTHO(_Float16);
#undef NMFK_ORTHO
}
