// Shared by the operators on plain matrices (nmfk_quant.hip, nmfk_prod8.hip, nmfk_ortho.hip): element types, the device guard of an entry
// point, and the staging of 128-byte rows into LDS that the tiled products use.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "nmfk_ctx.h"

// An entry point works on the device it is told and leaves the calling thread's current device as it was.  An error that another call of the runtime has
// left behind is not this call's: nmfk_launched would take it for its own.
struct NmfkDeviceGuard {
  int before = -1, status = 0;
  explicit NmfkDeviceGuard(int device) {
    int count = 0;
    (void)hipGetLastError();
    hipError_t e = hipGetDevice(&before);
    if (e == hipSuccess && before != device) {
      e = hipGetDeviceCount(&count);
      if (e == hipSuccess && (device < 0 || device >= count)) e = hipErrorInvalidDevice;
      if (e == hipSuccess) e = hipSetDevice(device);
    } else if (e == hipSuccess) {
      before = -1;  // nothing to restore
    }
    if (e != hipSuccess) {
      (void)hipGetLastError();
      status = fail(NMFK_ERR_NO_DEVICE, std::string("no usable gfx950 device for this call: ") + hipGetErrorString(e));
    }
  }
  ~NmfkDeviceGuard() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

static inline int nmfk_launched(const char *what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(NMFK_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
  return NMFK_OK;
}

static inline int64_t nmfk_div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline int64_t nmfk_round_up(int64_t a, int64_t b) { return nmfk_div_up(a, b) * b; }

namespace nmfk_mat {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using f64x4 = __attribute__((ext_vector_type(4))) double;
using i32x4 = __attribute__((ext_vector_type(4))) int;
using i32x8 = __attribute__((ext_vector_type(8))) int;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using f16x4 = __attribute__((ext_vector_type(4))) _Float16;

struct bf16 {
  uint16_t bits;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __uint_as_float((uint32_t)x.bits << 16); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ _Float16 from_f32<_Float16>(float x) {
  return (_Float16)x;  // to nearest, ties to even; beyond 65504 + half a step: infinity
}
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) {
  const uint32_t u = __float_as_uint(x);
  bf16 r;  // to nearest, ties to even; a NaN keeps its sign and stays one
  r.bits = (u & 0x7fffffffu) > 0x7f800000u ? (uint16_t)((u >> 16) | 0x40u) : (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
  return r;
}

// Four consecutive entries, loaded or stored at once.  The GPU takes them at any address that suits one entry.
template <typename T>
struct vec4 {
  T v[4];
};
template <typename T>
__device__ __forceinline__ void read4(const T *p, float (&out)[4]) {
  struct __attribute__((packed, aligned(sizeof(T)))) raw {
    uint32_t w[sizeof(T)];
  };
  const vec4<T> q = __builtin_bit_cast(vec4<T>, *(const raw *)p);
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = to_f32(q.v[e]);
}
template <typename T>
__device__ __forceinline__ void write4(T *p, float a, float b, float c, float d) {
  // (a vector, not a struct: the compiler would share a struct's last entry with the branch that stores entry by entry, and store in two pieces)
  typedef uint32_t raw __attribute__((ext_vector_type(sizeof(T)), aligned(sizeof(T))));
  *(raw *)p = __builtin_bit_cast(raw, (vec4<T>{from_f32<T>(a), from_f32<T>(b), from_f32<T>(c), from_f32<T>(d)}));
}

typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

// A wave copies 8 rows of 128 bytes from memory into LDS, 16 bytes a lane, past the registers.  LDS takes them in lane order, so the
// rows are 128 bytes apart there; the 16-byte chunk c of row r stands at slot c ^ (r & 7), which spreads a column of chunks -- what the
// matrix instructions' operands read, 16 rows at a time -- over all banks.  `g`: this lane's source (row lane / 8, chunk (lane & 7) ^ (lane / 8)).
__device__ __forceinline__ void stage8(const char *g, char *lds) {
  __builtin_amdgcn_global_load_lds((gvoid *)g, (lvoid *)lds, 16, 0, 0);
}
__device__ __forceinline__ void stage_f32(const float *g, float *lds) {
  __builtin_amdgcn_global_load_lds((gvoid *)g, (lvoid *)lds, 4, 0, 0);
}
__device__ __forceinline__ i32x4 lds_chunk(const char *lds, int row, int c) {
  return *(const i32x4 *)(lds + row * 128 + ((c ^ (row & 7)) << 4));
}
// every copy into LDS that this wave started has landed
__device__ __forceinline__ void staged() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ... all but the last N of them
template <int N>
__device__ __forceinline__ void staged_but() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// The workgroup's waves meet; what a wave has read from LDS it has received.  Unlike __syncthreads this does not wait for copies in flight.
__device__ __forceinline__ void meet() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Workgroups are dealt to the 8 XCDs in turn, each with an L2 of its own: renumber them so that an XCD gets consecutive numbers.
__device__ __forceinline__ int xcd_order(int id, int total) {
  const int per = total >> 3, rest = total & 7, x = id & 7, i = id >> 3;
  return x * per + (x < rest ? x : rest) + i;
}

// ... and walk the tiles in bands of `band` tile rows, column by column, so that the tiles which an XCD has in work at a time share rows of both operands
__device__ __forceinline__ void tile_at(int id, int tiles_m, int tiles_n, int band, int &tm, int &tn) {
  const int per = band * tiles_n, k = id / per, first = k * band, rows = min(band, tiles_m - first), in = id - k * per;
  tn = in / rows;
  tm = first + in - tn * rows;
}

}  // namespace nmfk_mat
