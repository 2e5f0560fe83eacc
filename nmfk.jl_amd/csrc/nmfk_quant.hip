// Matrices in 8-bit floating point (e4m3) with a scale for each block of 128 entries of a row, or for each 128 x 128 tile.
//
//   scale = max(max |x| / 448, 2^-126)   over the finite entries of the block, in 32 bits
//   value = e4m3(x / scale)              the quotient rounded to 32 bits, then to e4m3, ties to even; NaN where x is not finite
//
// What bounds it: memory.  An fp32 matrix in both orientations is 4 bytes read and 2 written for each entry, so the entries are read ONCE:
// a workgroup holds a 128 x 128 tile in registers, has the maxima of its rows, of its columns and of the whole, and writes the tile and
// its transpose (the latter turned in LDS, so that whole 128-byte lines leave).  65536 x 2048 of fp32 in tiles, both orientations: 141 us, 5.7 TB/s.
#include <algorithm>

#include "nmfk_matrix.h"

using namespace nmfk_mat;

namespace {

struct QuantArgs {
  const void *x;  // entry (r, c) at x[r * ld + c]
  int64_t rows, cols, ld;
  uint8_t *v;  // [rows][ldv], or null
  int64_t ldv;
  float *s;  // [blocks of a row][sld]: sld >= rows (blocks of rows) or blocks of rows (tiles)
  int64_t sld;
  uint8_t *tv;  // the transpose: [cols][ldtv], or null
  int64_t ldtv;
  float *ts;
  int64_t tsld;
};

__device__ __forceinline__ float block_scale(float top) { return fmaxf(top / 448.0f, 1.17549435e-38f); }
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// x / s rounded to nearest, for the many x of a block: with r = 1 / s rounded to nearest, q0 = x r, one correction q0 + r (x - q0 s) gives the
// correctly rounded quotient (Markstein's theorem) unless the significand of s is all ones.  The residual has to be exact: s in [2^-80, 2^80] makes
// it so for every quotient that does not round to zero in e4m3.  Elsewhere (EASY = false; a wave takes that path as a whole): the division, 11
// instructions instead of 3.  NaN and infinities come out of the short form as NaN by themselves, zeros with their sign (so a block with
// nothing else in it, as behind the last row, takes it, too).
__device__ __forceinline__ bool easy_divisor(float top, float s) {
  return top == 0.f || (s >= 0x1p-80f && s <= 0x1p80f && (__float_as_uint(s) & 0x7fffffu) != 0x7fffffu);
}
template <bool EASY>
__device__ __forceinline__ float quotient(float x, float s, float r) {
  if (EASY) {
    const float q = x * r;
    return fmaf(-fmaf(q, s, -x), r, q);
  }
  return fabsf(x) <= 3.402823466e38f ? x / s : __uint_as_float(0x7fc00000u);
}
template <bool EASY>
__device__ __forceinline__ uint32_t quotients(float a, float b, float c, float d, float s, float r) {
  return pack4(quotient<EASY>(a, s, r), quotient<EASY>(b, s, r), quotient<EASY>(c, s, r), quotient<EASY>(d, s, r));
}
// the largest of 32 lanes, in all of them: rotations within 16 lanes on the vector unit, then one exchange
template <int CTRL>
__device__ __forceinline__ float rotate(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float largest32(float m) {
  m = fmaxf(m, rotate<0x128>(m));  // row_ror:8
  m = fmaxf(m, rotate<0x124>(m));
  m = fmaxf(m, rotate<0x122>(m));
  m = fmaxf(m, rotate<0x121>(m));
  return fmaxf(m, __shfl_xor(m, 16));
}
template <typename T>
__device__ __forceinline__ void load4(const QuantArgs &a, int64_t r, int64_t c, float (&out)[4]) {
  const T *p = (const T *)a.x + r * a.ld + c;
  if (r < a.rows && c + 4 <= a.cols) {
    read4(p, out);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = r < a.rows && c + j < a.cols ? to_f32(p[j]) : 0.f;
  }
}

// blocks of rows, one orientation: a half wave per block, four entries a lane
template <typename T>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantArgs a, int64_t blocks, int64_t per_row) {
  const int64_t b = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (b >= blocks) return;
  const int64_t r = b / per_row, kb = b - r * per_row;
  const int64_t c = kb * 128 + (threadIdx.x & 31) * 4;
  float x[4];
  load4<T>(a, r, c, x);
  const float top = largest32(fmaxf(fmaxf(finite_abs(x[0]), finite_abs(x[1])), fmaxf(finite_abs(x[2]), finite_abs(x[3]))));
  const float s = block_scale(top), inv = 1.0f / s;
  *(uint32_t *)(a.v + r * a.ldv + c) = __all(easy_divisor(top, s)) ? quotients<true>(x[0], x[1], x[2], x[3], s, inv) : quotients<false>(x[0], x[1], x[2], x[3], s, inv);
  if ((threadIdx.x & 31) == 0) a.s[kb * a.sld + r] = s;
}

// A 128 x 128 tile per workgroup of 1024: lane group g = thread / 32 owns the rows 4 g .. 4 g + 3, thread % 32 four columns.  (With 256 threads and 16 rows each the
// code is four times as long, and a small matrix pays for fetching it: 35 tiles of fp32 in both orientations 12.3 us instead of 8.5.)  Scales of rows and
// columns are made by 256 of the threads, once each: two divisions, which in every thread that needs them cost as much as the quotients (4096 x 4096 of
// bf16 23 us instead of 16, the 35 tiles 8.5 instead of 5).
// `rs`, `cs`: the scales of the thread's rows and columns and their reciprocals (TILES: the one of the tile).
template <bool TILES, bool EASY>
__device__ __forceinline__ void quant_tile_values(const QuantArgs &a, const float (&x)[4][4], const float (&rs)[4], const float (&rr)[4], const float (&cs)[4],
                                                  const float (&cr)[4], char *turn, int64_t r0, int64_t c0) {
  const int t = threadIdx.x, g = t >> 5, cg = t & 31;
  uint32_t q[4];  // TILES: the values serve both orientations
  if (a.v || TILES) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      q[i] = quotients<EASY>(x[i][0], x[i][1], x[i][2], x[i][3], rs[TILES ? 0 : i], rr[TILES ? 0 : i]);
      if (a.v && r0 + g * 4 + i < a.rows) *(uint32_t *)(a.v + (r0 + g * 4 + i) * a.ldv + c0 + cg * 4) = q[i];
    }
  }
  if (!a.tv) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t w;
    if (TILES) {  // byte j of four rows: two permutations of register pairs
      const uint32_t sel = 0x0c0c0400u + 0x0101u * j;
      w = __builtin_amdgcn_perm(q[1], q[0], sel) | __builtin_amdgcn_perm(q[3], q[2], sel) << 16;
    } else {
      w = quotients<EASY>(x[0][j], x[1][j], x[2][j], x[3][j], cs[j], cr[j]);
    }
    *(uint32_t *)(turn + (cg * 4 + j) * 128 + (((g >> 2) ^ (cg & 7)) << 4) + (g & 3) * 4) = w;
  }
  __syncthreads();
  const int c = t >> 3, slot = t & 7;
  if (c0 + c < a.cols) *(i32x4 *)(a.tv + (c0 + c) * a.ldtv + r0 + slot * 16) = *(const i32x4 *)(turn + c * 128 + ((slot ^ ((c >> 2) & 7)) << 4));
}

template <typename T, bool TILES>
__global__ __launch_bounds__(1024) void quant_tile_kernel(QuantArgs a) {
  __shared__ __attribute__((aligned(16))) char turn[128 * 128];
  __shared__ __attribute__((aligned(16))) float ctop[16][128], rtop[2 * 128];
  __shared__ int hard;
  const int t = threadIdx.x, g = t >> 5, cg = t & 31;
  const int64_t r0 = (int64_t)blockIdx.y * 128, c0 = (int64_t)blockIdx.x * 128;
  float x[4][4];
  if (t == 0) hard = 0;
  if (r0 + 128 <= a.rows && c0 + 128 <= a.cols) {
    const T *p = (const T *)a.x + (r0 + g * 4) * a.ld + c0 + cg * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) read4(p + i * a.ld, x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) load4<T>(a, r0 + g * 4 + i, c0 + cg * 4, x[i]);
  }
  float cmax[4] = {0.f, 0.f, 0.f, 0.f}, rmax[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float f = finite_abs(x[i][j]);
      m = fmaxf(m, f);
      cmax[j] = fmaxf(cmax[j], f);
    }
    rmax[i] = m;
  }
  // columns: the two lane groups of a wave, then the sixteen waves
#pragma unroll
  for (int j = 0; j < 4; ++j) cmax[j] = fmaxf(cmax[j], __shfl_xor(cmax[j], 32));
  if (!(g & 1)) *(f32x4 *)&ctop[g >> 1][cg * 4] = (f32x4){cmax[0], cmax[1], cmax[2], cmax[3]};
  if (!TILES) {
#pragma unroll
    for (int i = 0; i < 4; ++i) rmax[i] = largest32(rmax[i]);
    if (cg == 0) *(f32x4 *)&rtop[g * 4] = (f32x4){rmax[0], rmax[1], rmax[2], rmax[3]};
  }
  __syncthreads();
  if (t < 128) {
    float m = ctop[0][t];
#pragma unroll
    for (int h = 1; h < 16; ++h) m = fmaxf(m, ctop[h][t]);
    if (TILES) {
      ctop[0][t] = m;
    } else {  // a column's scale and its reciprocal; two divisions, so once for each
      const float s = block_scale(m);
      ctop[0][t] = s;
      ctop[1][t] = 1.0f / s;
      if (!easy_divisor(m, s)) hard = 1;
      if (a.tv && c0 + t < a.cols) a.ts[(int64_t)blockIdx.y * a.tsld + c0 + t] = s;
    }
  } else if (!TILES && t < 256) {
    const int r = t - 128;
    const float m = rtop[r], s = block_scale(m);
    rtop[r] = s;
    rtop[128 + r] = 1.0f / s;
    if (!easy_divisor(m, s)) hard = 1;
    if (a.v && r0 + r < a.rows) a.s[(int64_t)blockIdx.x * a.sld + r0 + r] = s;
  }
  __syncthreads();
  float rs[4], rr[4], cs[4], cr[4];
  bool easy;
  const f32x4 top = *(const f32x4 *)&ctop[0][cg * 4];
  if (TILES) {
    const float m = largest32(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
    rs[0] = block_scale(m);
    rr[0] = 1.0f / rs[0];
    easy = easy_divisor(m, rs[0]);  // the same for all
    if (t == 0) {
      if (a.v) a.s[(int64_t)blockIdx.x * a.sld + blockIdx.y] = rs[0];
      if (a.tv) a.ts[(int64_t)blockIdx.y * a.tsld + blockIdx.x] = rs[0];
    }
  } else {
    const f32x4 inv = *(const f32x4 *)&ctop[1][cg * 4], row = *(const f32x4 *)&rtop[g * 4], row_inv = *(const f32x4 *)&rtop[128 + g * 4];
#pragma unroll
    for (int i = 0; i < 4; ++i) rs[i] = row[i], rr[i] = row_inv[i], cs[i] = top[i], cr[i] = inv[i];
    easy = !hard;
  }
  if (easy)
    quant_tile_values<TILES, true>(a, x, rs, rr, cs, cr, turn, r0, c0);
  else
    quant_tile_values<TILES, false>(a, x, rs, rr, cs, cr, turn, r0, c0);
}

template <typename T>
void quant_launch(QuantArgs a, bool tiles, hipStream_t st) {
  const int64_t kb = nmfk_div_up(a.cols, 128), rb = nmfk_div_up(a.rows, 128);
  if (!tiles && !a.tv) {
    // a launch holds fewer than 2^32 threads, 32 for each block
    const int64_t rows = a.rows, most = ((int64_t)1 << 26) / kb;
    for (int64_t r = 0; r < rows; r += most) {
      a.rows = std::min(most, rows - r);
      quant_rows_kernel<T><<<dim3((unsigned)nmfk_div_up(a.rows * kb, 8)), 256, 0, st>>>(a, a.rows * kb, kb);
      a.x = (const T *)a.x + a.rows * a.ld;
      a.v += a.rows * a.ldv;
      a.s += a.rows;
    }
  } else if (tiles) {
    quant_tile_kernel<T, true><<<dim3((unsigned)kb, (unsigned)rb), 1024, 0, st>>>(a);
  } else {
    quant_tile_kernel<T, false><<<dim3((unsigned)kb, (unsigned)rb), 1024, 0, st>>>(a);
  }
}

bool aligned16(const void *p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && (ld & 15) == 0; }

}  // namespace

NMFK_EXPORT int nmfk_quantize(int device, void *stream, int dtype, const void *X, int64_t rows, int64_t cols, int64_t row_stride,
                              int64_t col_stride, int tiles, uint8_t *values, int64_t ldv, float *scales, int64_t lds, uint8_t *tvalues,
                              int64_t ldtv, float *tscales, int64_t ldts) {
  if (rows < 0 || cols < 0) return fail(NMFK_ERR_BAD_ARG, "nmfk_quantize: negative size");
  if (dtype < NMFK_F32 || dtype > NMFK_F16) return fail(NMFK_ERR_BAD_ARG, "nmfk_quantize: dtype must be NMFK_F32, NMFK_BF16 or NMFK_F16");
  if (rows > ((int64_t)1 << 22) || cols > ((int64_t)1 << 22)) return fail(NMFK_ERR_UNSUPPORTED, "nmfk_quantize: more than 2^22 rows or columns");
  if (rows == 0 || cols == 0) return NMFK_OK;
  const int64_t kb = nmfk_div_up(cols, 128), rb = nmfk_div_up(rows, 128);
  if (!X || !values || !scales || (tvalues != nullptr) != (tscales != nullptr))
    return fail(NMFK_ERR_BAD_ARG, "nmfk_quantize: X, values and scales are needed, tvalues and tscales both or neither");
  if (!(col_stride == 1 && (row_stride >= cols || rows == 1)) && !(row_stride == 1 && (col_stride >= rows || cols == 1)))
    return fail(NMFK_ERR_BAD_ARG, "nmfk_quantize: the entries of a row or those of a column must be contiguous");
  if (!aligned16(values, ldv) || ldv < kb * 128 || lds < (tiles ? rb : rows))
    return fail(NMFK_ERR_BAD_ARG, "nmfk_quantize: values must be 16-byte aligned with ldv a multiple of 16 that holds whole blocks of 128; lds is too small");
  if (tvalues && (!aligned16(tvalues, ldtv) || ldtv < rb * 128 || ldts < (tiles ? kb : cols)))
    return fail(NMFK_ERR_BAD_ARG, "nmfk_quantize: tvalues must be 16-byte aligned with ldtv a multiple of 16 that holds whole blocks of 128; ldts is too small");
  NmfkDeviceGuard guard(device);
  if (guard.status) return guard.status;
  // the kernels walk the matrix as it stands in memory: if its columns are contiguous they see the transpose, and the outputs change places
  QuantArgs a;
  const bool as_is = col_stride == 1 && (row_stride >= cols || rows == 1);
  a.x = X;
  if (as_is)
    a = {X, rows, cols, rows == 1 ? cols : row_stride, values, ldv, scales, lds, tvalues, ldtv, tscales, ldts};
  else
    a = {X, cols, rows, cols == 1 ? rows : col_stride, tvalues, ldtv, tscales, ldts, values, ldv, scales, lds};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NMFK_F32)
    quant_launch<float>(a, tiles != 0, st);
  else if (dtype == NMFK_BF16)
    quant_launch<bf16>(a, tiles != 0, st);
  else
    quant_launch<_Float16>(a, tiles != 0, st);
  return nmfk_launched("nmfk_quantize");
}
