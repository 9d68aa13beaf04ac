// The residual's addition, the root-mean-square norm and the 8-bit codes that a product takes, in one pass (h2c_i8_norm), and codes
// back to values (h2c_i8_values). The formulas are stated in include/h2cuda.h.
#include "ops.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace h2 {
namespace {

// ---------------------------------------------------------------- norm
//
// A CTA a row: each thread holds its units of eight values in registers between the three steps (sum of squares, largest
// magnitude, codes), so every input is read once. Rows longer than the CTA's registers hold read their sums again (a thread
// its own, from L2).
// Squares are summed in 64 bits and 1 / sqrt(mean + eps) is rounded once, so it does not depend on the order of the additions
// (but for one in 10^7 rows, whose rounding lies at a border); what follows are single float32 operations. So the codes
// are the formula's, whatever the division of a row among threads.
constexpr int NORM_V = 8, NORM_U = 2;  // values of a unit, units that a thread keeps

struct NormArgs {
  const void *x, *res;
  void* sum;
  long long x_row, res_row, sum_row, q_row;
  const float* w;
  double eps;
  int rows, k, k_pad;
  int8_t* q;
  float* scale;
};

// eight values from p; n of them exist (the others are 0)
template <bool VEC, class T>
__device__ __forceinline__ void load8(const T* p, int n, float* v) {
  if (VEC && n >= NORM_V) {
    constexpr int W = NORM_V * sizeof(T) / 16;
    uint4 raw[W];
#pragma unroll
    for (int i = 0; i < W; i++) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    const T* h = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < NORM_V; i++) v[i] = to_f(h[i]);
  } else {
#pragma unroll
    for (int i = 0; i < NORM_V; i++) v[i] = i < n ? to_f(p[i]) : 0.f;
  }
}
template <bool VEC, class T>
__device__ __forceinline__ void store8(T* p, int n, const float* v) {
  if (VEC && n >= NORM_V) {
    constexpr int W = NORM_V * sizeof(T) / 16;
    alignas(16) T h[NORM_V];
#pragma unroll
    for (int i = 0; i < NORM_V; i++) h[i] = from_f<T>(v[i]);
#pragma unroll
    for (int i = 0; i < W; i++) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(h)[i];
  } else {
#pragma unroll
    for (int i = 0; i < NORM_V; i++)
      if (i < n) p[i] = from_f<T>(v[i]);
  }
}

// TX: type of x; TR: of the residual and the sum, void without a residual
template <class TX, class TR, bool VEC>
__global__ void __launch_bounds__(1024) k_i8_norm(const NormArgs a) {
  constexpr bool RES = !std::is_void<TR>::value;
  using R = typename std::conditional<RES, TR, TX>::type;
  __shared__ double part[32];
  __shared__ unsigned most[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5, NT = blockDim.x;
  const int units = a.k_pad / NORM_V, row = blockIdx.x;
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_row;
  const R* res = static_cast<const R*>(a.res) + row * a.res_row;
  R* sum = static_cast<R*>(a.sum) + row * a.sum_row;
  const R* again = RES ? sum : reinterpret_cast<const R*>(x);  // where the values that registers do not hold are read again

  float s[NORM_U][NORM_V];
  double acc = 0;
  auto take = [&](int u, float* v) {
    const int at = u * NORM_V, n = a.k - at;
    load8<VEC>(x + at, n, v);
    if (RES) {
      float r[NORM_V];
      load8<VEC>(res + at, n, r);
#pragma unroll
      for (int i = 0; i < NORM_V; i++) v[i] = to_f(from_f<R>(__fadd_rn(v[i], r[i])));
    }
  };
  auto square = [&](const float* v) {
    double t = 0;
#pragma unroll
    for (int i = 0; i < NORM_V; i++) {
      const double d = v[i];
      t = fma(d, d, t);
    }
    acc += t;
  };
#pragma unroll
  for (int i = 0; i < NORM_U; i++) {
    const int u = tid + i * NT;
    if (u < units) take(u, s[i]);
  }
#pragma unroll
  for (int i = 0; i < NORM_U; i++) {
    const int u = tid + i * NT;
    if (u < units) {
      if (RES) store8<VEC>(sum + u * NORM_V, a.k - u * NORM_V, s[i]);
      square(s[i]);
    }
  }
  for (int u = tid + NORM_U * NT; u < units; u += NT) {
    float v[NORM_V];
    take(u, v);
    if (RES) store8<VEC>(sum + u * NORM_V, a.k - u * NORM_V, v);
    square(v);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0) part[warp] = acc;
  __syncthreads();
  acc = lane < warps ? part[lane] : 0.;
#pragma unroll
  for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  const float r = (float)(1. / sqrt(acc / a.k + a.eps));

  unsigned m = 0;
  auto normed = [&](int u, float* v) {
    float w[NORM_V];
    load8<VEC>(a.w + u * NORM_V, a.k - u * NORM_V, w);
#pragma unroll
    for (int i = 0; i < NORM_V; i++) {
      v[i] = __fmul_rn(__fmul_rn(v[i], r), w[i]);
      // (what lies past the row is no part of it, whatever r is)
      m = max(m, u * NORM_V + i < a.k ? __float_as_uint(v[i]) & 0x7fffffffu : 0u);
    }
  };
#pragma unroll
  for (int i = 0; i < NORM_U; i++) {
    const int u = tid + i * NT;
    if (u < units) normed(u, s[i]);
  }
  for (int u = tid + NORM_U * NT; u < units; u += NT) {
    float v[NORM_V];
    load8<VEC>(again + u * NORM_V, a.k - u * NORM_V, v);
    normed(u, v);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) most[warp] = m;
  __syncthreads();
  const RowScale rs = row_scale_of(__reduce_max_sync(0xffffffffu, lane < warps ? most[lane] : 0u));
  if (tid == 0) a.scale[row] = rs.scale;
  const bool fine = rs.scale == rs.scale;

  uint2* q = reinterpret_cast<uint2*>(a.q + row * a.q_row);
  auto code = [&](int u, const float* v) {
    float c[NORM_V];
#pragma unroll
    for (int i = 0; i < NORM_V; i++) c[i] = fine && u * NORM_V + i < a.k ? __fmul_rn(v[i], rs.inv) : 0.f;
    q[u] = make_uint2(round_bytes(c[0], c[1], c[2], c[3]), round_bytes(c[4], c[5], c[6], c[7]));
  };
#pragma unroll
  for (int i = 0; i < NORM_U; i++) {
    const int u = tid + i * NT;
    if (u < units) code(u, s[i]);
  }
  for (int u = tid + NORM_U * NT; u < units; u += NT) {
    float v[NORM_V];
    load8<VEC>(again + u * NORM_V, a.k - u * NORM_V, v);
    normed(u, v);
    code(u, v);
  }
}

template <class TX, class TR>
void launch_norm(const NormArgs& a, bool vec, cudaStream_t st) {
  const int units = a.k_pad / NORM_V;
  const int threads = std::min(1024, std::max(32, ((units + NORM_U - 1) / NORM_U + 31) / 32 * 32));
  if (vec) k_i8_norm<TX, TR, true><<<a.rows, threads, 0, st>>>(a);
  else k_i8_norm<TX, TR, false><<<a.rows, threads, 0, st>>>(a);
}
template <class TX>
void launch_norm_of(const NormArgs& a, int res_type, bool vec, cudaStream_t st) {
  if (!a.res) launch_norm<TX, void>(a, vec, st);
  else if (res_type == H2C_TYPE_F32) launch_norm<TX, float>(a, vec, st);
  else launch_norm<TX, TX>(a, vec, st);  // (the same type: the entry refuses others)
}

// ---------------------------------------------------------------- values
//
// A thread takes eight codes of a row; where rows of values do not begin at 16 bytes, one code.
template <class T, bool VEC>
__global__ void __launch_bounds__(256) k_i8_values(const int8_t* __restrict__ q, long long q_row, const float* __restrict__ scale,
                                                   int rows, int k, T* __restrict__ y) {
  const int per = VEC ? k / NORM_V : k;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)rows * per; i += (long long)gridDim.x * 256) {
    const int row = (int)(i / per), u = (int)(i - (long long)row * per);
    const float f = scale[row];
    if (VEC) {
      const uint2 w = *reinterpret_cast<const uint2*>(q + row * q_row + u * NORM_V);
      float v[NORM_V];
#pragma unroll
      for (int j = 0; j < NORM_V; j++) v[j] = (float)(int8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3))) * f;
      store8<true>(y + (long long)row * k + u * NORM_V, NORM_V, v);
    } else {
      y[i] = from_f<T>((float)q[row * q_row + u] * f);
    }
  }
}

template <class T>
void launch_values(const int8_t* q, long long q_row, const float* scale, int rows, int k, void* y, bool vec, cudaStream_t st) {
  const long long work = vec ? (long long)rows * (k / NORM_V) : (long long)rows * k;
  const int ctas = (int)std::min<long long>((work + 255) / 256, 148 * 16);
  if (vec) k_i8_values<T, true><<<ctas, 256, 0, st>>>(q, q_row, scale, rows, k, static_cast<T*>(y));
  else k_i8_values<T, false><<<ctas, 256, 0, st>>>(q, q_row, scale, rows, k, static_cast<T*>(y));
}

}  // namespace
}  // namespace h2

using namespace h2;

extern "C" {

int h2c_i8_norm(int32_t x_type, const void* x, int64_t x_row, int32_t res_type, const void* residual, int64_t res_row, void* sum,
                int64_t sum_row, const float* weight, double eps, int32_t rows, int32_t k, void* q, int64_t q_row, float* scale,
                void* stream) {
  const char* who = "h2c_i8_norm";
  if (!op_type_ok(x_type)) return op_error(H2C_ERR_BAD_TYPE, "%s: element type %d of x", who, x_type);
  if (residual && res_type != x_type && res_type != H2C_TYPE_F32)
    return op_error(H2C_ERR_BAD_TYPE, "%s: element type %d of the residual (x's type or float32 is wanted)", who, res_type);
  if (rows < 0 || rows > OP_MAX_ROWS || k < 1 || k > H2C_I8_MAX_K) return op_error(H2C_ERR_INVALID, "%s: %d rows of %d", who, rows, k);
  if (!(eps >= 0)) return op_error(H2C_ERR_INVALID, "%s: eps %g", who, eps);
  if (rows == 0) return H2C_OK;
  if (!x || !weight || !q || !scale || !residual != !sum) return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  const int64_t xs = (int64_t)op_elem_size(x_type), rs = residual ? (int64_t)op_elem_size(res_type) : 1, k_pad = (k + 15) / 16 * 16;
  if ((uintptr_t)x & (xs - 1)) return op_error(H2C_ERR_INVALID, "%s: x must be aligned to its elements", who);
  if (((uintptr_t)residual | (uintptr_t)sum) & (rs - 1))
    return op_error(H2C_ERR_INVALID, "%s: residual and sum must be aligned to their elements", who);
  if (((uintptr_t)q & 15) || (q_row & 15) || q_row < k)
    return op_error(H2C_ERR_INVALID, "%s: q must be 16-byte aligned with rows of a multiple of 16 bytes, at least k", who);
  const OpRows tx{x, rows, x_row * xs, k * xs}, tr{residual, rows, res_row * rs, k * rs}, ts{sum, rows, sum_row * rs, k * rs};
  const OpRows codes{q, rows, q_row, k_pad};
  const OpRange weights = {"weight", weight, 4ull * k, 4}, scales = {"scale", scale, 4ull * rows, 4}, q_range = op_range("q", codes);
  if (residual) {
    if (rows > 1 && (sum_row < 0 ? -sum_row : sum_row) < k)
      return op_error(H2C_ERR_INVALID, "%s: rows of sum overlap (%lld elements apart, %d long)", who, (long long)sum_row, k);
    // (in place: a thread reads its values before it writes their sum)
    auto apart = [&](const OpRows& in, bool same_type) {
      return (same_type && in.p == sum && (in.stride == ts.stride || rows == 1)) || !op_rows_meet(in, ts);
    };
    if (!apart(tx, x_type == res_type)) return op_error(H2C_ERR_INVALID, "%s: sum must be x itself or share no memory with it", who);
    if (!apart(tr, true)) return op_error(H2C_ERR_INVALID, "%s: sum must be residual itself or share no memory with it", who);
    const OpRange out[] = {op_range("sum", ts), scales}, in[] = {weights, op_range("residual", tr)};
    if (int rc = op_check_ranges(who, out, 1, in, 1)) return rc;
    if (int rc = op_check_ranges(who, out + 1, 1, in + 1, 1)) return rc;
    if (int rc = op_check_ranges(who, out, 2, in, 0)) return rc;
    if (op_rows_meet(tr, codes)) return op_error(H2C_ERR_INVALID, "%s: q must not share memory with residual", who);
    if (op_rows_meet(ts, codes)) return op_error(H2C_ERR_INVALID, "%s: q must not share memory with sum", who);
  }
  if (op_rows_meet(tx, codes)) return op_error(H2C_ERR_INVALID, "%s: q must not share memory with x", who);
  {
    const OpRange out[] = {q_range, scales}, in[] = {weights, op_range("x", tx)};
    if (int rc = op_check_ranges(who, out, 2, in, 1)) return rc;
    if (int rc = op_check_ranges(who, out + 1, 1, in + 1, 1)) return rc;
  }
  const NormArgs a{x, residual, sum, x_row, res_row, sum_row, q_row, weight, eps, rows, k, (int)k_pad, static_cast<int8_t*>(q), scale};
  auto wide = [&](const void* p, int64_t stride) { return !(((uintptr_t)p | (rows > 1 ? stride : 0)) & 15); };
  const bool vec = wide(x, tx.stride) && wide(weight, 0) && (!residual || (wide(residual, tr.stride) && wide(sum, ts.stride)));
  cudaStream_t st = (cudaStream_t)stream;
  if (x_type == H2C_TYPE_F32) launch_norm_of<float>(a, res_type, vec, st);
  else if (x_type == H2C_TYPE_F16) launch_norm_of<__half>(a, res_type, vec, st);
  else launch_norm_of<__nv_bfloat16>(a, res_type, vec, st);
  return op_launched(who);
}

int h2c_i8_values(const void* q, int64_t q_row, const float* scale, int32_t rows, int32_t k, int32_t type, void* y, void* stream) {
  const char* who = "h2c_i8_values";
  if (!op_type_ok(type)) return op_error(H2C_ERR_BAD_TYPE, "%s: element type %d", who, type);
  if (rows < 0 || rows > OP_MAX_ROWS || k < 1 || k > H2C_I8_MAX_K) return op_error(H2C_ERR_INVALID, "%s: %d rows of %d", who, rows, k);
  if (rows == 0) return H2C_OK;
  if (!q || !scale || !y) return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  if (((uintptr_t)q & 15) || (q_row & 15) || q_row < k)
    return op_error(H2C_ERR_INVALID, "%s: q must be 16-byte aligned with rows of a multiple of 16 bytes, at least k", who);
  const uint64_t es = op_elem_size(type);
  const OpRange in[] = {op_range("q", OpRows{q, rows, q_row, k}), {"scale", scale, 4ull * rows, 4}};
  const OpRange out[] = {{"y", y, (uint64_t)rows * k * es, (unsigned)es}};
  if (int rc = op_check_ranges(who, out, 1, in, 2)) return rc;
  const bool vec = !((uintptr_t)y & 15) && k % NORM_V == 0;
  const int8_t* c = static_cast<const int8_t*>(q);
  cudaStream_t st = (cudaStream_t)stream;
  if (type == H2C_TYPE_F32) launch_values<float>(c, q_row, scale, rows, k, y, vec, st);
  else if (type == H2C_TYPE_F16) launch_values<__half>(c, q_row, scale, rows, k, y, vec, st);
  else launch_values<__nv_bfloat16>(c, q_row, scale, rows, k, y, vec, st);
  return op_launched(who);
}

}  // extern "C"
