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
  int vec;          // four outputs may be stored at once
};

template <typename T>
__device__ __forceinline__ void store4(T *p, f32x4 v, int left, int vec) {
  if (left >= 4 && vec) {
    vec4<T> q;
#pragma unroll
    for (int r = 0; r < 4; ++r) q.v[r] = from_f32<T>(v[r]);
    *(vec4<T> *)p = q;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < left) p[r] = from_f32<T>(v[r]);
  }
}

// A lane's operand for a block: 32 of its row's 128 entries.
struct Bytes {
  i32x8 v;
  __device__ __forceinline__ Bytes() {}
  __device__ __forceinline__ Bytes(i32x4 lo, i32x4 hi) { v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
};
struct Halves {
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
// the block's sums of TN tiles against one: the instructions of different tiles are independent and alternate
template <int TN>
__device__ __forceinline__ void block_products(const Bytes (&x)[TN], const Bytes &y, f32x4 (&part)[TN]) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < TN; ++j) part[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x[j].v, y.v, zero, 0, 0, 0, 0, 0, 0);
}
template <int TN>
__device__ __forceinline__ void block_products(const Halves (&x)[TN], const Halves &y, f32x4 (&part)[TN]) {
#pragma unroll
  for (int j = 0; j < TN; ++j) part[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int j = 0; j < TN; ++j) part[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[j].v[q], y.v[q], part[j], 0, 0, 0);
}

// A workgroup's tile of BM x BN outputs over its range of blocks: WM x WN waves, each (BM / WM) x (BN / WN).
// Two buffers of 128-byte rows in LDS; the copies into one are in flight while the other is multiplied.
// The first operand of the matrix instruction is B, so that a lane's four outputs are neighbours in a row of Y.
template <int BM, int BN, int WM, int WN, typename F, typename T, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN) void prod_tile_kernel(ProdArgs p) {
  constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int STAGE = (BM + BN) * 128, SC = (BM + BN) * 4;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int wm = w / WN, wn = w % WN;
  const int id = xcd_order(blockIdx.x, gridDim.x);
  int tm, tn;
  tile_at(id, p.tiles_m, p.tiles_n, BM == 256 ? 4 : 8, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int kb0 = blockIdx.y * p.kb_split, kb1 = min(p.kb, kb0 + p.kb_split);

  // this wave's share of the copies; rows behind the last one repeat it (their outputs are not stored)
  const int lr = lane >> 3, lc = ((lane & 7) ^ lr) << 4;
  const char *src[(BM + BN) / 8 / WAVES];
#pragma unroll
  for (int i = 0; i < (BM + BN) / 8 / WAVES; ++i) {
    const int row = (i * WAVES + w) * 8;
    src[i] = row < BM ? p.a + (int64_t)min(m0 + row + lr, p.m - 1) * p.lda + lc : p.b + (int64_t)min(n0 + row - BM + lr, p.n - 1) * p.ldb + lc;
  }
  constexpr int SW = (BM + BN) / 64;  // waves' worth of scales
  auto stage = [&](int kb, int buf) {
    char *base = lds + buf * STAGE;
#pragma unroll
    for (int i = 0; i < (BM + BN) / 8 / WAVES; ++i) stage8(src[i] + (int64_t)kb * 128, base + (i * WAVES + w) * 1024);
    float *sc = (float *)(lds + 2 * STAGE + buf * SC);
#pragma unroll
    for (int i = w; i < SW; i += WAVES) {
      const int row = i * 64;
      const float *g = row < BM ? p.sa + kb * p.ldsa + (min(m0 + row + lane, p.m - 1) >> p.ashift)
                                : p.sb + kb * p.ldsb + (min(n0 + row - BM + lane, p.n - 1) >> p.bshift);
      stage_f32(g, sc + row);
    }
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  if (kb0 < kb1) {
    stage(kb0, 0);
    staged();
  }
  __syncthreads();
  const int fr = lane & 15, fg = lane >> 4;
  for (int kb = kb0, buf = 0; kb < kb1; ++kb, buf ^= 1) {
    if (kb + 1 < kb1) stage(kb + 1, buf ^ 1);
    const char *la = lds + buf * STAGE, *lb = la + BM * 128;
    const float *sc = (const float *)(lds + 2 * STAGE + buf * SC);
    F fb[TN];
    f32x4 sb[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int row = wn * (BN / WN) + j * 16;
      fb[j] = F(lds_chunk(lb, row + fr, fg), lds_chunk(lb, row + fr, fg + 4));
      sb[j] = *(const f32x4 *)(sc + BM + row + fg * 4);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = wm * (BM / WM) + i * 16;
      const F fa(lds_chunk(la, row + fr, fg), lds_chunk(la, row + fr, fg + 4));
      const float sa = sc[row + fr];
      f32x4 part[TN];
      block_products<TN>(fb, fa, part);
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(part[j][r], sa * sb[j][r], acc[i][j][r]);
    }
    staged();
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * (BM / WM) + i * 16 + fr;
    if (m >= p.m) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + wn * (BN / WN) + j * 16 + fg * 4;
      if (n >= p.n) continue;
      if (SPLIT)
        store4<float>((float *)p.y + ((int64_t)blockIdx.y * p.m + m) * p.n + n, acc[i][j], p.n - n, p.vec);
      else
        store4<T>((T *)p.y + m * p.ldy + n, acc[i][j], p.n - n, p.vec);
    }
  }
}

// sums the splits in their order: the same bits on every run
template <typename T>
__global__ __launch_bounds__(256) void prod_join_kernel(const float *part, int splits, int64_t m, int64_t n, T *y, int64_t ldy) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= m * n) return;
  float s = 0.f;
  for (int k = 0; k < splits; ++k) s += part[(int64_t)k * m * n + i];
  const int64_t r = i / n;
  y[r * ldy + (i - r * n)] = from_f32<T>(s);
}

template <typename T>
__global__ __launch_bounds__(256) void prod_zero_kernel(T *y, int64_t m, int64_t n, int64_t ldy) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= m * n) return;
  const int64_t r = i / n;
  y[r * ldy + (i - r * n)] = from_f32<T>(0.f);
}

struct Plan {
  int bm, bn;
  int splits, kb_split;
};

Plan prod_plan(int64_t m, int64_t n, int64_t kb) {
  Plan q;
  q.bm = q.bn = 128;
  if (n <= 64)
    q.bn = 64;
  else if (nmfk_div_up(m, 256) * nmfk_div_up(n, 256) >= 200)
    q.bm = q.bn = 256;
  const int64_t tiles = nmfk_div_up(m, q.bm) * nmfk_div_up(n, q.bn);
  // Few tiles leave most of the 256 CUs without one: split the sum, as long as a workgroup keeps four blocks.
  int64_t splits = tiles >= 256 ? 1 : std::min<int64_t>(512 / tiles, nmfk_div_up(kb, 4));
  q.kb_split = (int)nmfk_div_up(kb, std::max<int64_t>(1, splits));
  q.splits = (int)std::max<int64_t>(1, nmfk_div_up(kb, q.kb_split));
  return q;
}

template <int BM, int BN, int WM, int WN, typename F, typename T, bool SPLIT>
void prod_tile(const ProdArgs &p, int splits, hipStream_t st) {
  constexpr int BYTES = 2 * (BM + BN) * 132;
  static std::atomic<uint64_t> done{0};
  nmfk_allow_dynamic_lds((const void *)prod_tile_kernel<BM, BN, WM, WN, F, T, SPLIT>, done, BYTES);
  prod_tile_kernel<BM, BN, WM, WN, F, T, SPLIT><<<dim3((unsigned)(p.tiles_m * p.tiles_n), (unsigned)splits), 64 * WM * WN, BYTES, st>>>(p);
}

template <typename F, typename T>
int prod_run(ProdArgs p, const Plan &q, void *work, hipStream_t st) {
  const int64_t mn = (int64_t)p.m * p.n;
  T *y = (T *)p.y;
  if (p.kb == 0) {
    prod_zero_kernel<T><<<dim3((unsigned)nmfk_div_up(mn, 256)), 256, 0, st>>>(y, p.m, p.n, p.ldy);
    return nmfk_launched("nmfk_product");
  }
  p.tiles_m = (int)nmfk_div_up(p.m, q.bm);
  p.tiles_n = (int)nmfk_div_up(p.n, q.bn);
  p.kb_split = q.kb_split;
  if (q.splits > 1) {
    p.y = work;
    p.vec = p.n % 4 == 0;
    if (q.bn == 64)
      prod_tile<128, 64, 4, 1, F, float, true>(p, q.splits, st);
    else
      prod_tile<128, 128, 2, 2, F, float, true>(p, q.splits, st);
    prod_join_kernel<T><<<dim3((unsigned)nmfk_div_up(mn, 256)), 256, 0, st>>>((const float *)work, q.splits, p.m, p.n, y, p.ldy);
  } else {
    p.vec = p.ldy % 4 == 0 && (uintptr_t)y % (4 * sizeof(T)) == 0;
    if (q.bn == 256)
      prod_tile<256, 256, 2, 4, F, T, false>(p, 1, st);
    else if (q.bn == 64)
      prod_tile<128, 64, 4, 1, F, T, false>(p, 1, st);
    else
      prod_tile<128, 128, 2, 2, F, T, false>(p, 1, st);
  }
  return nmfk_launched("nmfk_product");
}

int prod_sizes(int64_t m, int64_t n, int64_t k, const char *who) {
  if (m < 0 || n < 0 || k < 0) return fail(NMFK_ERR_BAD_ARG, std::string(who) + ": negative size");
  if (m > ((int64_t)1 << 22) || n > ((int64_t)1 << 22) || k > ((int64_t)1 << 22))
    return fail(NMFK_ERR_UNSUPPORTED, std::string(who) + ": a size above 2^22");
  if (nmfk_div_up(m, 128) * nmfk_div_up(n, 64) > 0x7fffffff / 2) return fail(NMFK_ERR_UNSUPPORTED, std::string(who) + ": too many outputs");
  return NMFK_OK;
}

}  // namespace

NMFK_EXPORT int nmfk_product_workspace(int64_t m, int64_t n, int64_t k, int64_t *bytes) {
  if (!bytes) return fail(NMFK_ERR_BAD_ARG, "nmfk_product_workspace: null pointer");
  if (int rc = prod_sizes(m, n, k, "nmfk_product_workspace")) return rc;
  *bytes = 0;
  if (m == 0 || n == 0 || k == 0) return NMFK_OK;
  const Plan q = prod_plan(m, n, nmfk_div_up(k, 128));
  if (q.splits > 1) *bytes = (int64_t)q.splits * m * n * 4;
  return NMFK_OK;
}

NMFK_EXPORT int nmfk_product(int device, void *stream, int64_t m, int64_t n, int64_t k, const uint8_t *A, int64_t lda, const float *sA,
                             int64_t ldsa, int a_tiles, const uint8_t *B, int64_t ldb, const float *sB, int64_t ldsb, int b_tiles, int dtype,
                             void *Y, int64_t ldy, void *work, int64_t work_bytes) {
  if (int rc = prod_sizes(m, n, k, "nmfk_product")) return rc;
  if (dtype < NMFK_F32 || dtype > NMFK_F16) return fail(NMFK_ERR_BAD_ARG, "nmfk_product: dtype must be NMFK_F32, NMFK_BF16 or NMFK_F16");
  if (m == 0 || n == 0) return NMFK_OK;
  const int64_t kb = nmfk_div_up(k, 128);
  if (!Y || ldy < n) return fail(NMFK_ERR_BAD_ARG, "nmfk_product: Y is needed, with ldy >= n");
  if (kb > 0) {
    if (!A || !B || !sA || !sB) return fail(NMFK_ERR_BAD_ARG, "nmfk_product: null pointer");
    if (((uintptr_t)A | (uintptr_t)B | (uintptr_t)lda | (uintptr_t)ldb) & 15 || lda < kb * 128 || ldb < kb * 128)
      return fail(NMFK_ERR_BAD_ARG, "nmfk_product: rows must be 16-byte aligned and hold whole blocks of 128");
    if (ldsa < (a_tiles ? nmfk_div_up(m, 128) : m) || ldsb < (b_tiles ? nmfk_div_up(n, 128) : n))
      return fail(NMFK_ERR_BAD_ARG, "nmfk_product: the leading dimension of the scales is too small");
  }
  const Plan q = prod_plan(m, n, std::max<int64_t>(1, kb));
  if (kb > 0 && q.splits > 1 && (!work || work_bytes < (int64_t)q.splits * m * n * 4 || (uintptr_t)work % 16))
    return fail(NMFK_ERR_BAD_ARG, "nmfk_product: the workspace is too small or not 16-byte aligned (nmfk_product_workspace)");
  NmfkDeviceGuard guard(device);
  if (guard.status) return guard.status;
  ProdArgs p = {(const char *)A, (const char *)B, lda, ldb, sA, sB, ldsa, ldsb, a_tiles ? 7 : 0, b_tiles ? 7 : 0, Y, ldy, (int)m, (int)n, (int)kb, 0, 0, 0, 0};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NMFK_F32) return prod_run<Halves, float>(p, q, work, st);
  if (dtype == NMFK_BF16) return prod_run<Bytes, bf16>(p, q, work, st);
  return prod_run<Bytes, _Float16>(p, q, work, st);
}
