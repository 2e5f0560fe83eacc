// Y = A * B' for matrices in 8 bits with a scale per block of 128 entries (nmfk_quant.hip):
//
//   Y[i, j] = sum over blocks b of  sA[i, b] * sB[j, b] * (sum over the block's t of a[i, t] * b[j, t])
//
// A block's sum starts from zero in the matrix pipe and a vector instruction adds it, scaled, to the 32-bit sum.  The order in which an
// instruction takes the 128 entries does not matter as long as both operands use the same one.
//
// Two matrix pipes, chosen by the type of Y:
//   Y in 16 bits: one v_mfma_f32_16x16x128_f8f6f4 per block (4.2 PFLOP/s measured alone).  It adds 16 products at a time after aligning them to the
//     largest, and what falls more than 13 bits below that is cut off: on normal entries the block's sum is 1.4e-5 of its norm away from
//     the exact one, 1/35 of half a step of fp16, 1/280 of bf16.
//   Y in fp32: that would show, so the entries are converted to fp16 (exact) and go through four v_mfma_f32_16x16x32_f16 (a block's sum 1e-8
//     away), at half the rate.  v_mfma_f32_16x16x32_fp8_fp8 has the rate of the latter and the error of the former.
#include <type_traits>

#include "nmfk_matrix.h"

using namespace nmfk_mat;

namespace {

struct ProdArgs {
  const char *a, *b;  // rows of lda / ldb bytes, whole blocks of 128 (zeros behind the last entry)
  int64_t lda, ldb;
  const float *sa, *sb;  // scale of (row, block) at [block * ldsa + (row >> ashift)]
  int64_t ldsa, ldsb;
  int ashift, bshift;  // 0: a scale per row, 7: per tile of 128 rows
  void *y;             // [m][ldy]; split sums: float [splits][m][n]
  int64_t ldy;
  int m, n, kb;     // blocks of 128
  int kb_split;     // blocks per workgroup along the sum
  int tiles_m, tiles_n;
};

template <typename T>
__device__ __forceinline__ void store4(T *p, f32x4 v, int left) {
  if (left >= 4) {
    write4(p, v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < left) p[r] = from_f32<T>(v[r]);
  }
}

// A lane's operand for a block: 32 of its row's 128 entries.
struct Bytes {
  static constexpr int STEPS = 1;
  i32x8 v;
  __device__ __forceinline__ Bytes() {}
  __device__ __forceinline__ Bytes(i32x4 lo, i32x4 hi) { v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
};
struct Halves {
  static constexpr int STEPS = 4;
  f16x8 v[4];
  __device__ __forceinline__ Halves() {}
  __device__ __forceinline__ Halves(i32x4 lo, i32x4 hi) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int x = q < 2 ? lo[2 * q + w] : hi[2 * (q - 2) + w];
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true);
        v[q][4 * w] = a[0], v[q][4 * w + 1] = a[1], v[q][4 * w + 2] = b[0], v[q][4 * w + 3] = b[1];
      }
  }
};
// One step of a block's sum for a 16 x 16 tile: step 0 starts from zero.
__device__ __forceinline__ f32x4 block_step(const Bytes &x, const Bytes &y, f32x4, int) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x.v, y.v, zero, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 block_step(const Halves &x, const Halves &y, f32x4 part, int q) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(x.v[q], y.v[q], q ? part : zero, 0, 0, 0);
}

// Which scales change inside a wave's part of a tile: with tiles of 128 x 128 on one side that side's scale is one number, and a block costs one
// vector instruction for an output instead of two.
enum { ROWS_ROWS = 0, B_TILES = 1, A_TILES = 2 };

// A workgroup's tile of BM x BN outputs over its range of blocks: WM x WN waves, each (BM / WM) x (BN / WN).
// Two buffers of 128-byte rows in LDS; the copies into one are in flight while the other is multiplied.  A wave holds B's operands of a block in
// registers, so B's half of a buffer is free after the first row of tiles and A's before the last two: at these two places the waves meet, and
// the copies of the block after the next start, spread over the rows (all at once: 6 % slower).  The operands of the next block are read while the matrix
// pipe is still busy with the last row of this one.
// What bounds it at 8192^3 (256 x 256, 447 .. 465 microseconds, 2.4 PFLOP/s): the matrix and vector instructions of a block alone, without any memory,
// take 413, the additions about 35 of these; copies and stores add 40.  The same in 32 x 32 x 64 instructions: 7 % slower.
// The first operand of the matrix instruction is B, so that a lane's four outputs are neighbours in a row of Y.
template <int BM, int BN, int WM, int WN, int MODE, typename F, typename T, bool SPLIT>
__device__ __forceinline__ void prod_tile(const ProdArgs &p, int id, int split) {
  constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int STAGE = (BM + BN) * 128, SC = (BM + BN) * 4;
  static_assert(TM >= 4 && TN >= 2 && BM / WM <= 128 && BN / WN <= 128, "B is copied between row 1 and row TM - 2, the scales behind the last use of the old ones");
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int wm = w / WN, wn = w % WN;
  int tm, tn;
  tile_at(id, p.tiles_m, p.tiles_n, BM == 256 ? 4 : 8, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int kb0 = split * p.kb_split, kb1 = min(p.kb, kb0 + p.kb_split);

  // this wave's share of the copies; rows behind the last one repeat it (their outputs are not stored).  A lane's offset from its tile's
  // first row fits 32 bits: 256 rows of at most 2^23 bytes.
  const int lr = lane >> 3, lc = ((lane & 7) ^ lr) << 4;
  constexpr int CA = BM / 8 / WAVES, CB = BN / 8 / WAVES;
  static_assert(CA * 8 * WAVES == BM && CB * 8 * WAVES == BN, "");
  const char *pa = p.a + (int64_t)m0 * p.lda + (int64_t)kb0 * 128, *pb = p.b + (int64_t)n0 * p.ldb + (int64_t)kb0 * 128;
  uint32_t off_a[CA], off_b[CB];
#pragma unroll
  for (int i = 0; i < CA; ++i) off_a[i] = (uint32_t)min((i * WAVES + w) * 8 + lr, p.m - 1 - m0) * (uint32_t)p.lda + lc;
#pragma unroll
  for (int i = 0; i < CB; ++i) off_b[i] = (uint32_t)min((i * WAVES + w) * 8 + lr, p.n - 1 - n0) * (uint32_t)p.ldb + lc;
  // scales of rows: 64 at a time, by the waves in turn (a wave without a share of its own repeats another's)
  constexpr int CS = ((BM + BN) / 64 + WAVES - 1) / WAVES;
  const float *ps[CS];
  int64_t ps_ld[CS];
  int ps_row[CS];
#pragma unroll
  for (int i = 0; i < CS; ++i) {
    const int row = (i * WAVES + w) % ((BM + BN) / 64) * 64;
    const bool is_a = row < BM;
    ps_row[i] = row;
    ps_ld[i] = is_a ? p.ldsa : p.ldsb;
    ps[i] = (is_a ? p.sa + (min(m0 + row + lane, p.m - 1) >> p.ashift) : p.sb + (min(n0 + row - BM + lane, p.n - 1) >> p.bshift)) + kb0 * ps_ld[i];
  }
  // the copies of the next block in order: B's one by one, A's in two halves
  auto copy_b = [&](int buf, int i) {
    stage8(pb + off_b[i], lds + buf * STAGE + BM * 128 + (i * WAVES + w) * 1024);
    if (i == CB - 1) pb += 128;
  };
  auto copy_a_first = [&](int buf) {
#pragma unroll
    for (int i = 0; i < CA / 2; ++i) stage8(pa + off_a[i], lds + buf * STAGE + (i * WAVES + w) * 1024);
  };
  auto copy_a_second = [&](int buf) {
#pragma unroll
    for (int i = CA / 2; i < CA; ++i) stage8(pa + off_a[i], lds + buf * STAGE + (i * WAVES + w) * 1024);
    pa += 128;
    float *sc = (float *)(lds + 2 * STAGE + buf * SC);
#pragma unroll
    for (int i = 0; i < CS; ++i) {
      stage_f32(ps[i], sc + ps_row[i]);
      ps[i] += ps_ld[i];
    }
  };
  const int fr = lane & 15, fg = lane >> 4;
  const int rm = wm * (BM / WM) + fr, rn = wn * (BN / WN) + fr;
  auto scales = [&](int buf) { return (const float *)(lds + 2 * STAGE + buf * SC); };
  // the scale that is one number in this wave's part (through LDS like the others: a wait for a load into a register would be a wait for
  // the copies that started after it, too)
  auto one = [&](int buf) { return scales(buf)[MODE == B_TILES ? BM + wn * (BN / WN) : wm * (BM / WM)]; };
  auto frag_a = [&](int buf, int i) {
    const char *la = lds + buf * STAGE;
    return F(lds_chunk(la, rm + i * 16, fg), lds_chunk(la, rm + i * 16, fg + 4));
  };
  auto frag_b = [&](int buf, int j) {
    const char *lb = lds + buf * STAGE + BM * 128;
    return F(lds_chunk(lb, rn + j * 16, fg), lds_chunk(lb, rn + j * 16, fg + 4));
  };
  auto scale_b = [&](int buf, int j) { return *(const f32x4 *)(scales(buf) + BM + wn * (BN / WN) + j * 16 + fg * 4); };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int blocks = kb1 - kb0;
  if (blocks > 0) {
    auto copy_all = [&](int buf) {
      copy_a_first(buf);
      copy_a_second(buf);
#pragma unroll
      for (int i = 0; i < CB; ++i) copy_b(buf, i);
    };
    copy_all(0);
    staged();
    meet();
    if (blocks > 1) copy_all(1);
    // The matrix instructions of a block are one sequence n = i * TN + j.  The vector instructions add the tile LAG places behind the one the
    // matrix pipe has begun, and the operands of row i + 2 are requested when row i begins.
    constexpr int LAG = 2, LEN = TM * TN;
    F fb[TN], fa[3];
    f32x4 sb[TN], part[LEN];
    float sa[3] = {0.f, 0.f, 0.f}, so = 0.f, so_next = 0.f, s_old = 0.f;
    if (MODE != ROWS_ROWS) so = one(0);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      fb[j] = frag_b(0, j);
      if (MODE != B_TILES) sb[j] = MODE == A_TILES ? so * scale_b(0, j) : scale_b(0, j);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fa[i] = frag_a(0, i);
      if (MODE != A_TILES) sa[i] = scales(0)[rm + i * 16];
    }
#pragma unroll
    for (int n = LEN - LAG; n < LEN; ++n) part[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    int buf = 0;
    for (int kb = kb0; kb < kb1; ++kb) {  // (behind the last block the operands of "the next" are whatever stands in LDS, unused)
      const bool copy = kb + 2 < kb1;
      if (MODE == B_TILES) sa[0] *= so;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if (i == 1 && copy) meet();
        if (i >= 1 && i < TM - 2 && copy) {  // B's copies, spread over the rows 1 .. TM - 3
          constexpr int PER = (CB + TM - 4) / (TM - 3);
#pragma unroll
          for (int c = (i - 1) * PER; c < i * PER && c < CB; ++c) copy_b(buf, c);
        }
        if (i == TM - 2) {
          if (copy) {
            staged_but<CB>();  // of the block after the next, B may still be on its way
            meet();
            copy_a_first(buf);
          } else {
            staged();
            meet();
          }
          if (MODE != ROWS_ROWS) so_next = one(buf ^ 1);
        }
        if (i == TM - 1 && copy) copy_a_second(buf);
        const int from = i + 2 < TM ? buf : buf ^ 1, row = (i + 2) % TM;
        fa[2] = frag_a(from, row);
        if (MODE != A_TILES) sa[2] = scales(from)[rm + row * 16];
#pragma unroll
        for (int u = 0; u < TN * F::STEPS; ++u) {
          const int j = u % TN, q = u / TN, n = i * TN + j;
          part[n] = block_step(fb[j], fa[0], part[n], q);
          if (q < F::STEPS - 1) continue;
          if (i == TM - 1) fb[j] = frag_b(buf ^ 1, j);
          const int o = (n + LEN - LAG) % LEN, oi = o / TN, oj = o % TN;
          const float s = oi == i ? sa[0] : s_old;
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[oi][oj][r] = fmaf(part[o][r], MODE == B_TILES ? s : MODE == A_TILES ? sb[oj][r] : s * sb[oj][r], acc[oi][oj][r]);
          asm volatile("" : "+v"(acc[oi][oj]));  // the additions do not move behind a branch
          if (MODE != ROWS_ROWS && F::STEPS == 1) {  // a matrix instruction, a read from LDS, the additions
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);
          }
          if (MODE != B_TILES && oi == TM - 1) {  // the last use of this scale: the next block's
            const f32x4 v = scale_b(i == 0 ? buf : buf ^ 1, oj);
            sb[oj] = MODE == A_TILES ? (i == 0 ? so : so_next) * v : v;
          }
        }
        s_old = sa[0];
        sa[0] = MODE == B_TILES && i < TM - 1 ? sa[1] * so : sa[1];
        sa[1] = sa[2];
        fa[0] = fa[1];
        fa[1] = fa[2];
        __builtin_amdgcn_sched_barrier(0);
      }
      so = so_next;
      buf ^= 1;
    }
#pragma unroll
    for (int n = LEN - LAG; n < LEN; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[TM - 1][n % TN][r] = fmaf(part[n][r], MODE == B_TILES ? s_old : MODE == A_TILES ? sb[n % TN][r] : s_old * sb[n % TN][r], acc[TM - 1][n % TN][r]);
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + rm + i * 16;
    if (m >= p.m) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + wn * (BN / WN) + j * 16 + fg * 4;
      if (n >= p.n) continue;
      if (SPLIT)
        store4<float>((float *)p.y + ((int64_t)split * p.m + m) * p.n + n, acc[i][j], p.n - n);
      else
        store4<T>((T *)p.y + m * p.ldy + n, acc[i][j], p.n - n);
    }
  }
}

template <int BM, int BN, int WM, int WN, int MODE, typename F, typename T, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN) void prod_tile_kernel(ProdArgs p) {
  prod_tile<BM, BN, WM, WN, MODE, F, T, SPLIT>(p, xcd_order(blockIdx.x, gridDim.x), blockIdx.y);
}

// Two products that do not wait for each other in one launch, the one with the longer sums first: the second fills the CUs that the first one leaves idle
// at its end.  The first operands have a scale for each row.
struct ProdPair {
  ProdArgs p[2];
};
template <int BM, int BN, int WM, int WN, typename F, typename T>
__global__ __launch_bounds__(64 * WM * WN) void prod_pair_kernel(ProdPair a) {
  const int first = a.p[0].tiles_m * a.p[0].tiles_n, which = (int)blockIdx.x >= first;
  const ProdArgs &p = a.p[which];
  const int id = which ? xcd_order(blockIdx.x - first, gridDim.x - first) : xcd_order(blockIdx.x, first);
  if (p.bshift)
    prod_tile<BM, BN, WM, WN, B_TILES, F, T, false>(p, id, 0);
  else
    prod_tile<BM, BN, WM, WN, ROWS_ROWS, F, T, false>(p, id, 0);
}

// Few rows of A (m <= 16 TA): what bounds it is the one read of B.  A workgroup owns 16 TB columns of Y; its eight waves take the blocks of the sum in
// turn, the operands go from memory straight into registers (a row's 128 bytes are read by four lanes), and the waves' sums are added in
// their order through LDS.  One row against 4096 x 4096: 7 us with the call itself, 3.4 of them the read at copy speed.
template <int TA, int TB, typename F, typename T, bool SPLIT>
__global__ __launch_bounds__(512) void prod_rows_kernel(ProdArgs p) {
  __shared__ __attribute__((aligned(16))) float sum[8][TA * TB * 256];
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, fr = lane & 15, fg = lane >> 4;
  const int n0 = blockIdx.x * 16 * TB;
  const int kb0 = blockIdx.y * p.kb_split, kb1 = min(p.kb, kb0 + p.kb_split);
  const char *pa[TA], *pb[TB];
  const float *sa[TA], *sb[TB][4];
#pragma unroll
  for (int i = 0; i < TA; ++i) {
    const int r = min(16 * i + fr, p.m - 1);
    pa[i] = p.a + (int64_t)r * p.lda + fg * 16;
    sa[i] = p.sa + (r >> p.ashift);
  }
#pragma unroll
  for (int j = 0; j < TB; ++j) {
    pb[j] = p.b + (int64_t)min(n0 + 16 * j + fr, p.n - 1) * p.ldb + fg * 16;
#pragma unroll
    for (int r = 0; r < 4; ++r) sb[j][r] = p.sb + (min(n0 + 16 * j + fg * 4 + r, p.n - 1) >> p.bshift);
  }
  f32x4 acc[TA][TB];
#pragma unroll
  for (int i = 0; i < TA; ++i)
#pragma unroll
    for (int j = 0; j < TB; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll(TA * TB <= 2 ? 4 : 2)
  for (int kb = kb0 + w; kb < kb1; kb += 8) {
    const int64_t o = (int64_t)kb * 128;
    F fb[TB];
    float s[TB][4];
#pragma unroll
    for (int j = 0; j < TB; ++j) {
      fb[j] = F(*(const i32x4 *)(pb[j] + o), *(const i32x4 *)(pb[j] + o + 64));
#pragma unroll
      for (int r = 0; r < 4; ++r) s[j][r] = sb[j][r][kb * p.ldsb];
    }
#pragma unroll
    for (int i = 0; i < TA; ++i) {
      const F fa(*(const i32x4 *)(pa[i] + o), *(const i32x4 *)(pa[i] + o + 64));
      const float x = sa[i][kb * p.ldsa];
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < F::STEPS; ++q) part = block_step(fb[j], fa, part, q);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(part[r], x * s[j][r], acc[i][j][r]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TA; ++i)
#pragma unroll
    for (int j = 0; j < TB; ++j) *(f32x4 *)&sum[w][((i * TB + j) * 64 + lane) * 4] = acc[i][j];
  __syncthreads();
  for (int e = t; e < TA * TB * 64; e += 512) {
    f32x4 v = *(const f32x4 *)&sum[0][e * 4];
#pragma unroll
    for (int k = 1; k < 8; ++k) v += *(const f32x4 *)&sum[k][e * 4];
    const int l = e & 63, i = (e >> 6) / TB, j = (e >> 6) % TB;
    const int m = 16 * i + (l & 15), n = n0 + 16 * j + (l >> 4) * 4;
    if (m >= p.m || n >= p.n) continue;
    if (SPLIT)
      store4<float>((float *)p.y + ((int64_t)blockIdx.y * p.m + m) * p.n + n, v, p.n - n);
    else
      store4<T>((T *)p.y + m * p.ldy + n, v, p.n - n);
  }
}

// Joins the parts of split sums: a wave adds every fourth part of 64 V results, then the four waves' sums are added in their order, so the bits are
// the same on every run.  What bounds it is the latency of the reads, hence many small workgroups (2048 x 64 in 32 parts: 4.8 us;
// 128 x 128 x 65536 with its join 13.3 us, with a whole sum a thread 14.9).
template <typename T, int V>
__global__ __launch_bounds__(256) void prod_join_kernel(const float *part, int splits, int64_t m, int64_t n, T *y, int64_t ldy) {
  using vec = __attribute__((ext_vector_type(V))) float;
  __shared__ vec sum[3][64];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t i = ((int64_t)blockIdx.x * 64 + lane) * V, mn = m * n;
  vec s = 0.f;
  if (i < mn) {
#pragma unroll 8
    for (int k = w; k < splits; k += 4) s += *(const vec *)(part + k * mn + i);
  }
  if (w) sum[w - 1][lane] = s;
  __syncthreads();
  if (w || i >= mn) return;
  s = ((s + sum[0][lane]) + sum[1][lane]) + sum[2][lane];
  const int64_t r = i / n;
  T *z = y + r * ldy + (i - r * n);
#pragma unroll
  for (int e = 0; e < V; ++e) z[e] = from_f32<T>(s[e]);
}

template <typename T>
__global__ __launch_bounds__(256) void prod_zero_kernel(T *y, int64_t m, int64_t n, int64_t ldy) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < m * n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / n;
    y[r * ldy + (i - r * n)] = from_f32<T>(0.f);
  }
}

struct Plan {
  int bm, bn;  // bn <= 32: prod_rows_kernel, bm rows and bn columns a workgroup; otherwise prod_tile_kernel
  int splits, kb_split;
};

Plan prod_plan(int64_t m, int64_t n, int64_t kb, bool bytes) {
  Plan q;
  int64_t splits = 1;
  if (m <= 64 && n > m) {
    q.bm = m <= 16 ? 16 : m <= 32 ? 32 : 64;
    q.bn = q.bm > 16 && n >= 8192 ? 32 : 16;
    const int64_t groups = nmfk_div_up(n, q.bn);  // of eight waves: two for each CU, and at least two blocks for each wave
    if (groups < 256) splits = std::min<int64_t>(512 / groups, kb / 16);
  } else {
    q.bm = q.bn = 128;
    if (n <= 64)
      q.bn = 64;
    else if (bytes && nmfk_div_up(m, 256) * nmfk_div_up(n, 256) >= 200)
      q.bm = q.bn = 256;
    // Tiles of 64 x 64 where those of 128 x 128 would not give every CU one
    if (q.bn == 128 && nmfk_div_up(m, 128) * nmfk_div_up(n, 128) < 256) q.bm = q.bn = 64;
    const int64_t tiles = nmfk_div_up(m, q.bm) * nmfk_div_up(n, q.bn);
    // Few tiles leave many of the 256 CUs without one: split the sum, as long as a workgroup keeps six blocks (about 5 microseconds; the join of
    // the partial sums costs 3).  One workgroup for each CU, or two where both keep sixteen blocks: 1024 x 64 x 65536 in 32 parts 23 us, in 64
    // parts 27; 4096 x 64 x 65536 in 16 parts 62, in 8 parts 67.
    if (tiles < 192) splits = std::min<int64_t>(kb / 6, std::max<int64_t>(nmfk_div_up(256, tiles), std::min<int64_t>(512 / tiles, kb / 16)));
  }
  q.kb_split = (int)nmfk_div_up(kb, std::max<int64_t>(1, splits));
  q.splits = (int)std::max<int64_t>(1, nmfk_div_up(kb, q.kb_split));
  return q;
}

template <int BM, int BN, int WM, int WN, int MODE, typename F, typename T, bool SPLIT>
void prod_tile_mode(const ProdArgs &p, int splits, hipStream_t st) {
  constexpr int BYTES = 2 * (BM + BN) * 132;
  static std::atomic<uint64_t> done{0};
  nmfk_allow_dynamic_lds((const void *)prod_tile_kernel<BM, BN, WM, WN, MODE, F, T, SPLIT>, done, BYTES);
  prod_tile_kernel<BM, BN, WM, WN, MODE, F, T, SPLIT><<<dim3((unsigned)(p.tiles_m * p.tiles_n), (unsigned)splits), 64 * WM * WN, BYTES, st>>>(p);
}

template <int BM, int BN, int WM, int WN, typename F, typename T, bool SPLIT>
void prod_tile_side(const ProdArgs &p, int splits, hipStream_t st) {
  if (p.bshift)
    prod_tile_mode<BM, BN, WM, WN, B_TILES, F, T, SPLIT>(p, splits, st);
  else if (p.ashift)
    prod_tile_mode<BM, BN, WM, WN, A_TILES, F, T, SPLIT>(p, splits, st);
  else
    prod_tile_mode<BM, BN, WM, WN, ROWS_ROWS, F, T, SPLIT>(p, splits, st);
}

template <typename F, typename T, bool SPLIT>
void prod_launch(const ProdArgs &p, const Plan &q, hipStream_t st) {
  if (q.bn <= 32) {
    const dim3 grid((unsigned)nmfk_div_up(p.n, q.bn), (unsigned)q.splits);
    if constexpr (!SPLIT)  // (32 columns a workgroup: 8192 columns and more, whose workgroups are many)
      if (q.bn == 32) {
        if (q.bm == 32)
          prod_rows_kernel<2, 2, F, T, false><<<grid, 512, 0, st>>>(p);
        else
          prod_rows_kernel<4, 2, F, T, false><<<grid, 512, 0, st>>>(p);
        return;
      }
    if (q.bm == 16)
      prod_rows_kernel<1, 1, F, T, SPLIT><<<grid, 512, 0, st>>>(p);
    else if (q.bm == 32)
      prod_rows_kernel<2, 1, F, T, SPLIT><<<grid, 512, 0, st>>>(p);
    else
      prod_rows_kernel<4, 1, F, T, SPLIT><<<grid, 512, 0, st>>>(p);
    return;
  }
  if constexpr (!SPLIT) {  // (tiles of 128 x 128 and larger are many: prod_plan splits no sum of theirs)
    if constexpr (std::is_same<F, Bytes>::value)
      if (q.bn == 256) {
        prod_tile_side<256, 256, 2, 4, F, T, false>(p, 1, st);
        return;
      }
    if (q.bn == 128) {
      prod_tile_side<128, 128, 2, 2, F, T, false>(p, 1, st);
      return;
    }
  }
  if (q.bm == 64)
    prod_tile_side<64, 64, 1, 2, F, T, SPLIT>(p, q.splits, st);
  else
    prod_tile_side<128, 64, 2, 2, F, T, SPLIT>(p, q.splits, st);
}

template <typename F, typename T>
int prod_run(ProdArgs p, const Plan &q, void *work, hipStream_t st) {
  const int64_t mn = (int64_t)p.m * p.n;
  T *y = (T *)p.y;
  if (p.kb == 0) {
    prod_zero_kernel<T><<<dim3((unsigned)std::min<int64_t>(nmfk_div_up(mn, 256), 1 << 16)), 256, 0, st>>>(y, p.m, p.n, p.ldy);
    return nmfk_launched("nmfk_product");
  }
  p.tiles_m = (int)nmfk_div_up(p.m, q.bm);
  p.tiles_n = (int)nmfk_div_up(p.n, q.bn);
  p.kb_split = q.kb_split;
  if (q.splits > 1) {
    p.y = work;
    prod_launch<F, float, true>(p, q, st);
    if (p.n % 4 == 0)
      prod_join_kernel<T, 4><<<dim3((unsigned)nmfk_div_up(mn, 256)), 256, 0, st>>>((const float *)work, q.splits, p.m, p.n, y, p.ldy);
    else
      prod_join_kernel<T, 1><<<dim3((unsigned)nmfk_div_up(mn, 64)), 256, 0, st>>>((const float *)work, q.splits, p.m, p.n, y, p.ldy);
  } else {
    prod_launch<F, T, false>(p, q, st);
  }
  return nmfk_launched("nmfk_product");
}

template <int BM, int BN, int WM, int WN, typename F, typename T>
int prod_pair_side(ProdPair a, hipStream_t st) {
  constexpr int BYTES = 2 * (BM + BN) * 132;
  static std::atomic<uint64_t> done{0};
  nmfk_allow_dynamic_lds((const void *)prod_pair_kernel<BM, BN, WM, WN, F, T>, done, BYTES);
  unsigned tiles = 0;
  for (ProdArgs &p : a.p) {
    p.tiles_m = (int)nmfk_div_up(p.m, BM);
    p.tiles_n = (int)nmfk_div_up(p.n, BN);
    p.kb_split = p.kb;
    tiles += (unsigned)(p.tiles_m * p.tiles_n);
  }
  prod_pair_kernel<BM, BN, WM, WN, F, T><<<dim3(tiles), 64 * WM * WN, BYTES, st>>>(a);
  return nmfk_launched("nmfk_product_grads");
}

template <typename F, typename T>
int prod_pair(const ProdPair &a, int side, hipStream_t st) {
  if constexpr (std::is_same<F, Bytes>::value)
    if (side == 256) return prod_pair_side<256, 256, 2, 4, F, T>(a, st);
  if (side == 128) return prod_pair_side<128, 128, 2, 2, F, T>(a, st);
  return prod_pair_side<64, 64, 1, 2, F, T>(a, st);
}

// The side of the tiles with which two products go in one launch, by prod_plan's rule for both together; 0: one behind the other, because one of them
// is better off with another kernel or a split sum
int pair_side(int64_t m0, int64_t n0, int64_t kb0, int64_t m1, int64_t n1, int64_t kb1, bool bytes) {
  for (const Plan &q : {prod_plan(m0, n0, kb0, bytes), prod_plan(m1, n1, kb1, bytes)})
    if (q.splits > 1 || q.bm != q.bn || q.bm < 64) return 0;
  auto tiles = [&](int64_t side) { return nmfk_div_up(m0, side) * nmfk_div_up(n0, side) + nmfk_div_up(m1, side) * nmfk_div_up(n1, side); };
  return bytes && tiles(256) >= 200 ? 256 : tiles(128) >= 256 ? 128 : 64;
}

int prod_sizes(int64_t m, int64_t n, int64_t k, const char *who) {
  if (m < 0 || n < 0 || k < 0) return fail(NMFK_ERR_BAD_ARG, std::string(who) + ": negative size");
  if (m > ((int64_t)1 << 22) || n > ((int64_t)1 << 22) || k > ((int64_t)1 << 22))
    return fail(NMFK_ERR_UNSUPPORTED, std::string(who) + ": a size above 2^22");
  if (nmfk_div_up(m, 128) * nmfk_div_up(n, 64) > 0x7fffffff / 2) return fail(NMFK_ERR_UNSUPPORTED, std::string(who) + ": too many outputs");
  return NMFK_OK;
}

// the arguments of a product, checked; m = 0 or n = 0 is nothing to do
int prod_args(int64_t m, int64_t n, int64_t k, const uint8_t *A, int64_t lda, const float *sA, int64_t ldsa, int a_tiles, const uint8_t *B, int64_t ldb,
              const float *sB, int64_t ldsb, int b_tiles, int dtype, void *Y, int64_t ldy, ProdArgs &p) {
  if (int rc = prod_sizes(m, n, k, "nmfk_product")) return rc;
  if (dtype < NMFK_F32 || dtype > NMFK_F16) return fail(NMFK_ERR_BAD_ARG, "nmfk_product: dtype must be NMFK_F32, NMFK_BF16 or NMFK_F16");
  if (m == 0 || n == 0) return NMFK_OK;
  const int64_t kb = nmfk_div_up(k, 128);
  if (!Y || ldy < n) return fail(NMFK_ERR_BAD_ARG, "nmfk_product: Y is needed, with ldy >= n");
  if (kb > 0) {
    if (!A || !B || !sA || !sB) return fail(NMFK_ERR_BAD_ARG, "nmfk_product: null pointer");
    if (((uintptr_t)A | (uintptr_t)B | (uintptr_t)lda | (uintptr_t)ldb) & 15 || lda < kb * 128 || ldb < kb * 128 || lda > ((int64_t)1 << 23) || ldb > ((int64_t)1 << 23))
      return fail(NMFK_ERR_BAD_ARG, "nmfk_product: rows must be 16-byte aligned, hold whole blocks of 128 and be at most 2^23 bytes apart");
    if (ldsa < (a_tiles ? nmfk_div_up(m, 128) : m) || ldsb < (b_tiles ? nmfk_div_up(n, 128) : n))
      return fail(NMFK_ERR_BAD_ARG, "nmfk_product: the leading dimension of the scales is too small");
  }
  p = {(const char *)A, (const char *)B, lda, ldb, sA, sB, ldsa, ldsb, a_tiles ? 7 : 0, b_tiles ? 7 : 0, Y, ldy, (int)m, (int)n, (int)kb, 0, 0, 0};
  return NMFK_OK;
}

}  // namespace

NMFK_EXPORT int nmfk_product_workspace(int64_t m, int64_t n, int64_t k, int dtype, int64_t *bytes) {
  if (!bytes) return fail(NMFK_ERR_BAD_ARG, "nmfk_product_workspace: null pointer");
  if (int rc = prod_sizes(m, n, k, "nmfk_product_workspace")) return rc;
  if (dtype < NMFK_F32 || dtype > NMFK_F16) return fail(NMFK_ERR_BAD_ARG, "nmfk_product_workspace: dtype must be NMFK_F32, NMFK_BF16 or NMFK_F16");
  *bytes = 0;
  if (m == 0 || n == 0 || k == 0) return NMFK_OK;
  const Plan q = prod_plan(m, n, nmfk_div_up(k, 128), dtype != NMFK_F32);
  if (q.splits > 1) *bytes = (int64_t)q.splits * m * n * 4;
  return NMFK_OK;
}

NMFK_EXPORT int nmfk_product(int device, void *stream, int64_t m, int64_t n, int64_t k, const uint8_t *A, int64_t lda, const float *sA,
                             int64_t ldsa, int a_tiles, const uint8_t *B, int64_t ldb, const float *sB, int64_t ldsb, int b_tiles, int dtype,
                             void *Y, int64_t ldy, void *work, int64_t work_bytes) {
  ProdArgs p;
  if (int rc = prod_args(m, n, k, A, lda, sA, ldsa, a_tiles, B, ldb, sB, ldsb, b_tiles, dtype, Y, ldy, p)) return rc;
  if (m == 0 || n == 0) return NMFK_OK;
  const int64_t kb = p.kb;
  const Plan q = prod_plan(m, n, std::max<int64_t>(1, kb), dtype != NMFK_F32);
  if (kb > 0 && q.splits > 1 && (!work || work_bytes < (int64_t)q.splits * m * n * 4 || (uintptr_t)work % 16))
    return fail(NMFK_ERR_BAD_ARG, "nmfk_product: the workspace is too small or not 16-byte aligned (nmfk_product_workspace)");
  NmfkDeviceGuard guard(device);
  if (guard.status) return guard.status;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NMFK_F32) return prod_run<Halves, float>(p, q, work, st);
  if (dtype == NMFK_BF16) return prod_run<Bytes, bf16>(p, q, work, st);
  return prod_run<Bytes, _Float16>(p, q, work, st);
}

// ---- the backward pass -------------------------------------------------------------------------------------------------------------

namespace {

struct GradLayout {
  int64_t ldq, ldt;                   // bytes of a row of dY and of its transpose in 8 bits
  int64_t q, qs, t, ts, work, bytes;  // byte offsets: dY in 8 bits and its scales, its transpose and its, what the two products need (in turn)
};

int grad_layout(int64_t m, int64_t n, int64_t k, int dtype, GradLayout &y) {
  int64_t wa = 0, wb = 0;
  if (int rc = nmfk_product_workspace(m, k, n, dtype, &wa)) return rc;
  if (int rc = nmfk_product_workspace(n, k, m, dtype, &wb)) return rc;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += nmfk_round_up(bytes, 256);
    return o;
  };
  y.ldq = nmfk_round_up(n, 128);
  y.ldt = nmfk_round_up(m, 128);
  y.q = take(m * y.ldq);
  y.qs = take(4 * m * (y.ldq / 128));
  y.t = take(n * y.ldt);
  y.ts = take(4 * n * (y.ldt / 128));
  y.work = take(std::max(wa, wb));
  y.bytes = at;
  return NMFK_OK;
}

}  // namespace

NMFK_EXPORT int nmfk_product_grads_workspace(int64_t m, int64_t n, int64_t k, int dtype, int64_t *bytes) {
  if (!bytes) return fail(NMFK_ERR_BAD_ARG, "nmfk_product_grads_workspace: null pointer");
  GradLayout y;
  if (int rc = grad_layout(m, n, k, dtype, y)) return rc;
  *bytes = y.bytes;
  return NMFK_OK;
}

NMFK_EXPORT int nmfk_product_grads(int device, void *stream, int64_t m, int64_t n, int64_t k, int dy_dtype, const void *dY, int64_t row_stride,
                                   int64_t col_stride, const uint8_t *At, int64_t ldat, const float *sAt, int64_t ldsat, int at_tiles,
                                   const uint8_t *Bt, int64_t ldbt, const float *sBt, int64_t ldsbt, int bt_tiles, int dtype, void *dA,
                                   int64_t ldda, void *dB, int64_t lddb, void *work, int64_t work_bytes) {
  GradLayout y;
  if (int rc = grad_layout(m, n, k, dtype, y)) return rc;
  if (work_bytes < y.bytes || (y.bytes && (!work || (uintptr_t)work % 256)))
    return fail(NMFK_ERR_BAD_ARG, "nmfk_product_grads: the workspace is too small or not 256-byte aligned (nmfk_product_grads_workspace)");
  char *w = (char *)work;
  uint8_t *q = (uint8_t *)(w + y.q), *t = (uint8_t *)(w + y.t);
  float *qs = (float *)(w + y.qs), *ts = (float *)(w + y.ts);
  ProdPair pair;
  if (int rc = prod_args(m, k, n, q, y.ldq, qs, m, 0, Bt, ldbt, sBt, ldsbt, bt_tiles, dtype, dA, ldda, pair.p[0])) return rc;
  if (int rc = prod_args(n, k, m, t, y.ldt, ts, n, 0, At, ldat, sAt, ldsat, at_tiles, dtype, dB, lddb, pair.p[1])) return rc;
  if (m && n)
    if (int rc = nmfk_quantize(device, stream, dy_dtype, dY, m, n, row_stride, col_stride, 0, q, y.ldq, qs, m, t, y.ldt, ts, n)) return rc;
  const int side = m && n && k ? pair_side(m, k, nmfk_div_up(n, 128), n, k, nmfk_div_up(m, 128), dtype != NMFK_F32) : 0;
  if (side) {
    NmfkDeviceGuard guard(device);
    if (guard.status) return guard.status;
    if (m > n) std::swap(pair.p[0], pair.p[1]);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == NMFK_F32) return prod_pair<Halves, float>(pair, side, st);
    if (dtype == NMFK_BF16) return prod_pair<Bytes, bf16>(pair, side, st);
    return prod_pair<Bytes, _Float16>(pair, side, st);
  }
  if (int rc = nmfk_product(device, stream, m, k, n, q, y.ldq, qs, m, 0, Bt, ldbt, sBt, ldsbt, bt_tiles, dtype, dA, ldda, w + y.work, y.bytes - y.work)) return rc;
  return nmfk_product(device, stream, n, k, m, t, y.ldt, ts, n, 0, At, ldat, sAt, ldsat, at_tiles, dtype, dB, lddb, w + y.work, y.bytes - y.work);
}
