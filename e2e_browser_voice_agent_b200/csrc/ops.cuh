// What the stand-alone 8-bit serving operators (kv8.cu, kv8_att.cu, i8mm.cu) share: error reporting at the C entries,
// once-per-device kernel attributes, the record of expired waits, and loads and stores of activations of any type.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/h2cuda.h"

namespace h2 {

// Record the message of a failed call (h2c_last_error(NULL)) and return `code`. Never throws.
int op_error(int code, const char* fmt, ...) noexcept __attribute__((format(printf, 2, 3)));
// H2C_OK, or H2C_ERR_CUDA with "<who>: launch failed: ..." when the last launch of this thread failed.
int op_launched(const char* who) noexcept;
// Four device words of the current device in which a kernel whose bounded wait expired leaves {1, CTA, role, 0}
// (read by h2c_ops_check); nullptr when the device cannot be queried.
int* op_err_words() noexcept;

// An argument's memory: its name, the bytes from its lowest to its highest, and the alignment that it needs.
struct OpRange {
  const char* name;
  const void* p;
  uint64_t bytes;
  unsigned align = 1;
};
// H2C_OK, or H2C_ERR_INVALID with "<who>: X must be aligned to N bytes" when one is not, or "<who>: X must not share memory with Y"
// when one of the `n_out` ranges that a call writes shares bytes with one of the `n_in` that it reads, or two that it writes do.
int op_check_ranges(const char* who, const OpRange* out, int n_out, const OpRange* in, int n_in) noexcept;

// Rows of `bytes` bytes, `stride` bytes apart (of either sign, or 0).
struct OpRows {
  const void* p;
  int64_t rows, stride, bytes;
};
OpRange op_range(const char* name, const OpRows& r) noexcept;
// Whether two sets of rows share bytes: exact for the same stride (columns of one buffer) and for one row, else by their ranges.
bool op_rows_meet(const OpRows& a, const OpRows& b) noexcept;
// Whether of rows x heads vectors of `len` elements, `row` and `head` elements apart, two share elements (exact).
bool op_vectors_overlap(int64_t rows, int64_t row, int64_t heads, int64_t head, int64_t len) noexcept;

// Most rows of a call: kernels count past the last by up to a grid's stride.
constexpr int OP_MAX_ROWS = 0x7fffffff - (1 << 16);
constexpr int OP_MAX_DEVICES = 64;
// Run fn() once per device (kernel attributes); its status, or H2C_OK when it has already run on this device.
template <class F>
int op_once(const char* who, unsigned char* done, F fn) noexcept {
  int dev = -1;
  cudaError_t c = cudaGetDevice(&dev);
  if (c != cudaSuccess || dev < 0 || dev >= OP_MAX_DEVICES)
    return op_error(H2C_ERR_CUDA, "%s: cudaGetDevice: %s", who,
                    c != cudaSuccess ? cudaGetErrorString(c) : "device index out of range");
  if (__atomic_load_n(done + dev, __ATOMIC_ACQUIRE)) return H2C_OK;
  c = fn();  // idempotent: two threads that get here together both set the same attributes
  if (c != cudaSuccess) return op_error(H2C_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", who, cudaGetErrorString(c));
  __atomic_store_n(done + dev, 1, __ATOMIC_RELEASE);
  return H2C_OK;
}

inline size_t op_elem_size(int type) { return type == H2C_TYPE_F32 ? 4 : 2; }
inline bool op_type_ok(int type) { return type == H2C_TYPE_F32 || type == H2C_TYPE_F16 || type == H2C_TYPE_BF16; }

#ifdef __CUDACC__
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Four values with |v| < 2^22, rounded to integers (halves to even), as the low bytes of their two's complements: adding 1.5 x 2^23
// leaves the integer in the low bits of the sum. (Conversions to integers run at a quarter of the rate of additions.)
__device__ __forceinline__ uint32_t round_bytes(float a, float b, float c, float d) {
  const uint32_t x = __float_as_uint(__fadd_rn(a, 12582912.f)), y = __float_as_uint(__fadd_rn(b, 12582912.f)),
                 z = __float_as_uint(__fadd_rn(c, 12582912.f)), w = __float_as_uint(__fadd_rn(d, 12582912.f));
  return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}

// four consecutive values; VEC: the address is aligned to four of them
template <bool VEC>
__device__ __forceinline__ void load4(const float* p, float* v) {
  if (VEC) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = p[i];
  }
}
template <bool VEC, class T>
__device__ __forceinline__ void load4(const T* p, float* v) {
  static_assert(sizeof(T) == 2, "16-bit types");
  if (VEC) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    const T* h = reinterpret_cast<const T*>(&a);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = to_f(h[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = to_f(p[i]);
  }
}

// Four consecutive values as they lie in memory.
template <class T, bool VEC>
struct Raw4 {
  uint32_t w[sizeof(T)];
  __device__ __forceinline__ void load(const T* p) {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); i += 2) {
        const uint2 x = reinterpret_cast<const uint2*>(p)[i / 2];
        w[i] = x.x, w[i + 1] = x.y;
      }
    } else {
      T v[4];
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = p[i];
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); i++) w[i] = reinterpret_cast<const uint32_t*>(v)[i];
    }
  }
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = to_f(reinterpret_cast<const T*>(w)[i]);
  }
  // Magnitudes order as their bits do, infinities and NaN above every number: 16-bit ones two at a time. merge() joins the largest
  // so far with these; bits() makes the bits of a float32 of it.
  __device__ __forceinline__ unsigned merge(unsigned m) const {
    if (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); i++) m = max(m, w[i] & 0x7fffffffu);
      return m;
    }
    return __vmaxu2(m, __vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu));
  }
  static __device__ __forceinline__ unsigned bits(unsigned m) {
    if (sizeof(T) == 4) return m;
    const unsigned short u = (unsigned short)max(m & 0xffffu, m >> 16);
    return __float_as_uint(to_f(*reinterpret_cast<const T*>(&u)));
  }
};
#endif

}  // namespace h2
