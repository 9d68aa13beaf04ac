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
// Squares are summed in 64 bits and 1 / sqrt(mean + eps) is rounded once, so it does not depend on the order of the additions (but for
// one in 10^7 rows, whose rounding lies at a border); what follows are single float32 operations. So the codes are the formula's,
// whatever the division of a row among threads.
// Rows of aligned units of four values, up to 8,192 units (k_i8_norm): one warp a row to 32, a few short rows a CTA, each thread holding
// up to eight units in registers between the three steps (sum of squares, largest magnitude, codes), so every input is read once and
// all of a row is on its way together. The sizes are the compiler's: with loops over sizes known at run time the instructions were what
// bound it (16,392 x 3,584 bfloat16 with a float32 residual: 146 us; now 97, 6.7 TB/s). Few rows: two units a thread, four times
// the warps, as latency is what counts (k_i8_norm's launch below). Other rows (k_i8_norm_any): a CTA each, whose values that do not fit
// its registers are read again.
// Bound: bandwidth for many rows (16,392 x 3,584 with a bfloat16 residual 63 us, 6.5 TB/s; float32 x 896 31 us, 6.1 TB/s). Rows without a
// residual have half the bytes on their way for each thread and are bound by latency: 47 us (3.7 TB/s) with 5 CTAs an SM, for which the compiler
// spills 8-16 bytes a thread, 86 with one. One row: 2.3 us, a launch.
// k_i8_norm_any, a CTA of 1,024 threads a row however short, is far from that: 16,392 rows of 10 or 100 bfloat16 values 190 us, of 1,001
// 200 (250 with a residual), of 3,586 275 (310), whose bytes would take 0.1, 0.8, 8 and 27; 4,000 rows of 40,000 380 (560), 73 by bytes.
constexpr int NORM_V = 4;        // values of a unit: 16 bytes of float32, so that a warp's accesses are whole lines
constexpr int NORM_WARPS = 8;    // of a CTA whose rows take fewer
constexpr int NORM_MOST = 32768; // values of a row that registers hold

struct NormArgs {
  const void *x, *res;
  void* sum;
  long long x_row, res_row, sum_row, q_row;
  const float* w;
  double eps, inv_k;
  int rows, k, k_pad;
  int8_t* q;
  float* scale;
};

// V values from p. VEC: all exist and p is aligned to V of them; else n of them exist, and the others are 0.
template <bool VEC, int V, class T>
__device__ __forceinline__ void load_unit(const T* p, int n, float* v) {
  using Word = typename std::conditional<V * sizeof(T) == 8, uint2, uint4>::type;
  constexpr int W = V * sizeof(T) / sizeof(Word);
  if (VEC) {
    Word raw[W];
#pragma unroll
    for (int i = 0; i < W; i++) raw[i] = reinterpret_cast<const Word*>(p)[i];
    const T* h = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = to_f(h[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = i < n ? to_f(p[i]) : 0.f;
  }
}
template <bool VEC, int V, class T>
__device__ __forceinline__ void store_unit(T* p, int n, const float* v) {
  using Word = typename std::conditional<V * sizeof(T) == 8, uint2, uint4>::type;
  constexpr int W = V * sizeof(T) / sizeof(Word);
  if (VEC) {
    alignas(16) T h[V];
#pragma unroll
    for (int i = 0; i < V; i++) h[i] = from_f<T>(v[i]);
#pragma unroll
    for (int i = 0; i < W; i++) reinterpret_cast<Word*>(p)[i] = reinterpret_cast<const Word*>(h)[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i < n) p[i] = from_f<T>(v[i]);
  }
}

// the largest magnitude, NaN if one is
__device__ __forceinline__ float max_mag(float m, float x, float y) {
  asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(x), "f"(y));
  return m;
}

// 1 / sqrt(x) as float32: float32's, made exact to 2^-51 by two of Newton's steps in 64 bits, so that the rounding is that of the value but
// where that lies as near to a border between two float32 numbers.
__device__ __forceinline__ float inverse_root(double x) {
  if (!(x > 1e-30 && x < 1e30)) return (float)rsqrt(x);
  double y = rsqrtf((float)x);
  const double h = 0.5 * x;
  y = fma(y, fma(-h * y, y, 0.5), y);
  y = fma(y, fma(-h * y, y, 0.5), y);
  return (float)y;
}

// Four values as they lie in memory: as float32, and float32 rounded to them.
template <class T>
struct Quad;
template <>
struct Quad<float> {
  float4 w;
  __device__ __forceinline__ void get(float* v) const { v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w; }
  __device__ __forceinline__ void set(const float* v) { w = make_float4(v[0], v[1], v[2], v[3]); }
};
template <>
struct Quad<__half> {
  __half2 w[2];
  __device__ __forceinline__ void get(float* v) const {
    const float2 a = __half22float2(w[0]), b = __half22float2(w[1]);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
  __device__ __forceinline__ void set(const float* v) { w[0] = __floats2half2_rn(v[0], v[1]), w[1] = __floats2half2_rn(v[2], v[3]); }
};
template <>
struct Quad<__nv_bfloat16> {
  uint32_t w[2];
  __device__ __forceinline__ void get(float* v) const {
    v[0] = __uint_as_float(w[0] << 16), v[1] = __uint_as_float(w[0] & 0xffff0000u);
    v[2] = __uint_as_float(w[1] << 16), v[3] = __uint_as_float(w[1] & 0xffff0000u);
  }
  __device__ __forceinline__ void set(const float* v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    w[0] = *reinterpret_cast<const uint32_t*>(&a), w[1] = *reinterpret_cast<const uint32_t*>(&b);
  }
};
template <class T>
__device__ __forceinline__ Quad<T> quad_at(const T* p) {
  Quad<T> q;
  if constexpr (sizeof(T) == 4) q.w = *reinterpret_cast<const float4*>(p);
  else *reinterpret_cast<uint2*>(q.w) = *reinterpret_cast<const uint2*>(p);
  return q;
}
// The same where `on`, without a branch, and not put off to where it is used: so that a thread's are on their way together (without a
// residual, 16,392 x 3,584 bfloat16: 82 us as plain loads, which the compiler moves down one by one).
template <class T>
__device__ __forceinline__ Quad<T> quad_if(const T* p, bool on) {
  uint32_t w[sizeof(T)];
  if constexpr (sizeof(T) == 4)
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n @p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n}\n"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "l"(p), "r"((int)on));
  else
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %3, 0;\n @p ld.global.v2.b32 {%0, %1}, [%2];\n}\n"
                 : "=r"(w[0]), "=r"(w[1])
                 : "l"(p), "r"((int)on));
  Quad<T> q;
  if constexpr (sizeof(T) == 4) q.w = make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]));
  else *reinterpret_cast<uint2*>(q.w) = make_uint2(w[0], w[1]);
  return q;
}
template <class T>
__device__ __forceinline__ void put_quad(T* p, const Quad<T>& q) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = q.w;
  else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(q.w);
}

// The steps of a row among `W` warps of which this is one; `part` and `most` have a place for each.
template <int W>
__device__ __forceinline__ double sum_of_row(double x, double* part, int warp, int lane, int barrier) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (W > 1) {
    if (lane == 0) part[warp] = x;
    asm volatile("barrier.sync %0, %1;" ::"r"(barrier), "n"(32 * W) : "memory");
    x = part[lane % W];
#pragma unroll
    for (int o = W / 2; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  }
  return x;
}
template <int W>
__device__ __forceinline__ float max_of_row(float m, unsigned* most, int warp, int lane, int barrier) {
  unsigned u = __reduce_max_sync(0xffffffffu, __float_as_uint(m));  // (not negative: ordered as their bits are, NaN above all)
  if (W > 1) {
    if (lane == 0) most[warp] = u;
    asm volatile("barrier.sync %0, %1;" ::"r"(barrier), "n"(32 * W) : "memory");
    u = __reduce_max_sync(0xffffffffu, most[lane % W]);
  }
  return __uint_as_float(u);
}

// TX: type of x; TR: of the residual and the sum, void without a residual; W warps a row, U units a thread. CTAs an SM: as many as ran
// fastest, which is what the compiler makes of the registers (16,392 x 3,584, 1, 4 and 5 of them: bfloat16 with a residual 68, 63 and 68
// us, with a float32 residual 97, 98 and 118, without one 86, 70 and 46).
template <class TX, class TR, int W, int U>
__global__ void __launch_bounds__(32 * (W < NORM_WARPS ? NORM_WARPS : W),
                                  W >= NORM_WARPS || U < 8 ? 1 : std::is_void<TR>::value ? 5 : std::is_same<TR, float>::value ? 1 : 4)
    k_i8_norm(const NormArgs a) {
  constexpr bool RES = !std::is_void<TR>::value;
  using R = typename std::conditional<RES, TR, TX>::type;
  constexpr int NT = 32 * W, GROUPS = W < NORM_WARPS ? NORM_WARPS / W : 1;
  __shared__ double part[GROUPS][W];
  __shared__ unsigned most[GROUPS][W];
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % W, group = threadIdx.x / NT, tid = threadIdx.x % NT;
  const long long row = (long long)blockIdx.x * GROUPS + group;
  if (row >= a.rows) return;
  const int units = a.k / NORM_V, mine = (units - tid + NT - 1) / NT;  // units of the row, of this thread
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_row + NORM_V * tid;
  const R* res = static_cast<const R*>(a.res) + row * a.res_row + NORM_V * tid;
  R* sum = static_cast<R*>(a.sum) + row * a.sum_row + NORM_V * tid;
  Quad<TX> qx[U];
  Quad<R> qr[RES ? U : 1];
#pragma unroll
  for (int i = 0; i < U; i++) {  // (all of them before the first store, which may be over the residual)
    qx[i] = quad_if(x + i * NT * NORM_V, i < mine);
    if (RES) qr[i % (RES ? U : 1)] = quad_if(res + i * NT * NORM_V, i < mine);
  }
  float s[U][NORM_V];
  double t[2] = {0., 0.};
#pragma unroll
  for (int i = 0; i < U; i++)
    if (i < mine) {
      qx[i].get(s[i]);
      if (RES) {
        float r[NORM_V];
        Quad<R>& q = qr[i % (RES ? U : 1)];
        q.get(r);
#pragma unroll
        for (int j = 0; j < NORM_V; j++) s[i][j] = __fadd_rn(s[i][j], r[j]);
        q.set(s[i]);
        put_quad(sum + i * NT * NORM_V, q);
        q.get(s[i]);
      }
#pragma unroll
      for (int j = 0; j < NORM_V; j++) {
        const double d = s[i][j];
        t[j & 1] = fma(d, d, t[j & 1]);
      }
    }
  const float f = inverse_root(fma(sum_of_row<W>(t[0] + t[1], part[group], warp, lane, 1 + group), a.inv_k, a.eps));
  float m = 0.f;
  const float* weight = a.w + NORM_V * tid;
#pragma unroll
  for (int i = 0; i < U; i++)
    if (i < mine) {
      float w[NORM_V];
      quad_at(weight + i * NT * NORM_V).get(w);
#pragma unroll
      for (int j = 0; j < NORM_V; j++) s[i][j] = __fmul_rn(__fmul_rn(s[i][j], f), w[j]);
      m = max_mag(max_mag(m, s[i][0], s[i][1]), s[i][2], s[i][3]);
    }
  m = max_of_row<W>(m, most[group], warp, lane, 1 + group);
  const float inv = row_scale_of(__float_as_uint(m)).inv;
  if (tid == 0) a.scale[row] = row_scale_of(__float_as_uint(m)).scale;
  uint32_t* q = reinterpret_cast<uint32_t*>(a.q + row * a.q_row) + tid;
#pragma unroll
  for (int i = 0; i < U; i++)
    if (i < mine)
      q[i * NT] = round_bytes(__fmul_rn(s[i][0], inv), __fmul_rn(s[i][1], inv), __fmul_rn(s[i][2], inv), __fmul_rn(s[i][3], inv));
  if (tid < a.k_pad / NORM_V - units) q[units] = 0;  // (zeros to 16 bytes: up to three units)
}

// The same for rows of any length and alignment; VEC: they are whole aligned units all the same
template <class TX, class TR, bool VEC>
__global__ void __launch_bounds__(1024) k_i8_norm_any(const NormArgs a) {
  constexpr bool RES = !std::is_void<TR>::value;
  using R = typename std::conditional<RES, TR, TX>::type;
  constexpr int W = 32, NT = 32 * W, U = 4;
  __shared__ double part[W];
  __shared__ unsigned most[W];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, units = a.k_pad / NORM_V;
  const long long row = blockIdx.x;
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_row;
  const R* res = static_cast<const R*>(a.res) + row * a.res_row;
  R* sum = static_cast<R*>(a.sum) + row * a.sum_row;
  const R* again = RES ? sum : reinterpret_cast<const R*>(x);  // where the values that registers do not hold are read again
  auto left = [&](int u) { return VEC && (u + 1) * NORM_V <= a.k ? NORM_V : a.k - u * NORM_V; };  // values of unit u
  auto load = [&](const auto* p, int u, float* v) {
    if (VEC && left(u) == NORM_V) load_unit<true, NORM_V>(p + u * NORM_V, NORM_V, v);
    else load_unit<false, NORM_V>(p + u * NORM_V, left(u), v);
  };
  double acc = 0;
  auto take = [&](int u, float* v) {  // the unit's sum with its residual, stored and squared
    load(x, u, v);
    if (RES) {
      float r[NORM_V];
      load(res, u, r);
#pragma unroll
      for (int i = 0; i < NORM_V; i++) v[i] = to_f(from_f<R>(__fadd_rn(v[i], r[i])));
      if (VEC && left(u) == NORM_V) store_unit<true, NORM_V>(sum + u * NORM_V, NORM_V, v);
      else store_unit<false, NORM_V>(sum + u * NORM_V, left(u), v);
    }
#pragma unroll
    for (int i = 0; i < NORM_V; i++) {
      const double d = v[i];
      acc = fma(d, d, acc);
    }
  };
  float s[U][NORM_V];
#pragma unroll
  for (int i = 0; i < U; i++)
    if (tid + i * NT < units) take(tid + i * NT, s[i]);
  for (int u = tid + U * NT; u < units; u += NT) {
    float v[NORM_V];
    take(u, v);
  }
  const float f = inverse_root(fma(sum_of_row<W>(acc, part, warp, lane, 1), a.inv_k, a.eps));
  float m = 0.f;
  auto norm = [&](float* v, int u) {
    float w[NORM_V];
    load(a.w, u, w);
#pragma unroll
    for (int i = 0; i < NORM_V; i++) v[i] = i < left(u) ? __fmul_rn(__fmul_rn(v[i], f), w[i]) : 0.f;  // (past the row: 0 whatever f is)
  };
#pragma unroll
  for (int i = 0; i < U; i++)
    if (tid + i * NT < units) {
      norm(s[i], tid + i * NT);
      m = max_mag(max_mag(m, s[i][0], s[i][1]), s[i][2], s[i][3]);
    }
  for (int u = tid + U * NT; u < units; u += NT) {
    float v[NORM_V];
    load(again, u, v);
    norm(v, u);
    m = max_mag(max_mag(m, v[0], v[1]), v[2], v[3]);
  }
  m = max_of_row<W>(m, most, warp, lane, 1);
  const RowScale rs = row_scale_of(__float_as_uint(m));
  if (tid == 0) a.scale[row] = rs.scale;
  uint32_t* q = reinterpret_cast<uint32_t*>(a.q + row * a.q_row);
  auto code = [&](const float* v, int u) {
    q[u] = round_bytes(__fmul_rn(v[0], rs.inv), __fmul_rn(v[1], rs.inv), __fmul_rn(v[2], rs.inv), __fmul_rn(v[3], rs.inv));
    if (left(u) < NORM_V) q[u] &= left(u) > 0 ? (1u << (8 * left(u))) - 1 : 0u;  // (0 times what may be an infinity)
  };
#pragma unroll
  for (int i = 0; i < U; i++)
    if (tid + i * NT < units) code(s[i], tid + i * NT);
  for (int u = tid + U * NT; u < units; u += NT) {
    float v[NORM_V];
    load(again, u, v);
    norm(v, u);
    code(v, u);
  }
}

template <class TX, class TR, int W, int U>
void launch_norm_w(const NormArgs& a, cudaStream_t st) {
  constexpr int groups = W < NORM_WARPS ? NORM_WARPS / W : 1;
  k_i8_norm<TX, TR, W, U><<<(a.rows + groups - 1) / groups, 32 * W * groups, 0, st>>>(a);
}
template <class TX, class TR>
void launch_norm(const NormArgs& a, bool vec, cudaStream_t st) {
  // Few rows, some 3 of them an SM: more warps each. us with more and with fewer warps, bfloat16 with a residual: 896 wide 32 rows 2.2
  // and 3.0, 600 rows 2.8 and 3.3, 1,200 rows 4.0 and 3.8; 3,584 wide 32 rows 2.7 and 3.4, 400 rows 3.7 and 4.1, 600 rows 5.1 and 4.7;
  // 8,192 wide 32 rows 3.6 and 3.6, 200 rows 4.7 and 4.1, so there all rows take 8 warps.
  const bool few = a.rows <= 148 * 3;
  if (!vec || a.k > NORM_MOST) {
    if (vec) k_i8_norm_any<TX, TR, true><<<a.rows, 1024, 0, st>>>(a);
    else k_i8_norm_any<TX, TR, false><<<a.rows, 1024, 0, st>>>(a);
  } else if (a.k <= 1024) {
    if (few) launch_norm_w<TX, TR, 4, 2>(a, st);
    else launch_norm_w<TX, TR, 1, 8>(a, st);
  } else if (a.k <= 4096) {
    if (few) launch_norm_w<TX, TR, 16, 2>(a, st);
    else launch_norm_w<TX, TR, 4, 8>(a, st);
  } else if (a.k <= 8192) {
    launch_norm_w<TX, TR, 8, 8>(a, st);
  } else {
    launch_norm_w<TX, TR, 32, 8>(a, st);
  }
}
template <class TX>
void launch_norm_of(const NormArgs& a, int res_type, bool vec, cudaStream_t st) {
  if (!a.res) launch_norm<TX, void>(a, vec, st);
  else if (res_type == H2C_TYPE_F32) launch_norm<TX, float>(a, vec, st);
  else launch_norm<TX, TX>(a, vec, st);  // (the same type: the entry refuses others)
}

// ---------------------------------------------------------------- values
//
// A thread takes eight codes of a row at a time, two of them under way; where rows of values do not begin at 16 bytes, one code.
constexpr int VALUES_V = 8;
template <class T, bool VEC>
__global__ void __launch_bounds__(256) k_i8_values(const int8_t* __restrict__ q, long long q_row, const float* __restrict__ scale,
                                                   int rows, int k, T* __restrict__ y) {
  constexpr int V = VEC ? VALUES_V : 1, AHEAD = 2;
  const unsigned per = k / V, magic = 0xffffffffu / per;
  const long long all = (long long)rows * per, step = (long long)gridDim.x * 256;
  for (long long i0 = (long long)blockIdx.x * 256 + threadIdx.x; i0 < all; i0 += AHEAD * step) {
    uint2 w[AHEAD];
    float f[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; n++) {
      const long long i = i0 + n * step;
      if (i >= all) break;
      long long row;
      unsigned u;
      if (all <= 0x7fffffff) {
        unsigned r = __umulhi((unsigned)i, magic);  // (one too few at most)
        u = (unsigned)i - r * per;
        if (u >= per) r++, u -= per;
        row = r;
      } else {
        row = i / per;
        u = (unsigned)(i - row * per);
      }
      const int8_t* p = q + row * q_row + u * V;
      if (VEC) w[n] = *reinterpret_cast<const uint2*>(p);
      else w[n].x = (uint8_t)*p;
      f[n] = scale[row];
    }
#pragma unroll
    for (int n = 0; n < AHEAD; n++) {
      const long long i = i0 + n * step;
      if (i >= all) break;
      float v[VALUES_V];
#pragma unroll
      for (int j = 0; j < V; j++) v[j] = (float)(int8_t)((j < 4 ? w[n].x : w[n].y) >> (8 * (j & 3))) * f[n];
      if constexpr (VEC) store_unit<true, VALUES_V>(y + i * V, V, v);  // (rows of y follow each other)
      else y[i] = from_f<T>(v[0]);
    }
  }
}

template <class T>
void launch_values(const int8_t* q, long long q_row, const float* scale, int rows, int k, void* y, bool vec, cudaStream_t st) {
  const long long work = vec ? (long long)rows * (k / VALUES_V) : (long long)rows * k;
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
  const NormArgs a{x, residual, sum, x_row, res_row, sum_row, q_row, weight, eps, 1. / k, rows, k, (int)k_pad, static_cast<int8_t*>(q), scale};
  auto wide = [&](const void* p, int64_t stride) { return !(((uintptr_t)p | (rows > 1 ? stride : 0)) & 15); };
  const bool vec = k % NORM_V == 0 && wide(x, tx.stride) && wide(weight, 0) && (!residual || (wide(residual, tr.stride) && wide(sum, ts.stride)));
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
  const bool vec = !((uintptr_t)y & 15) && k % VALUES_V == 0;
  const int8_t* c = static_cast<const int8_t*>(q);
  cudaStream_t st = (cudaStream_t)stream;
  if (type == H2C_TYPE_F32) launch_values<float>(c, q_row, scale, rows, k, y, vec, st);
  else if (type == H2C_TYPE_F16) launch_values<__half>(c, q_row, scale, rows, k, y, vec, st);
  else launch_values<__nv_bfloat16>(c, q_row, scale, rows, k, y, vec, st);
  return op_launched(who);
}

}  // extern "C"
