// Attention over the paged 8-bit cache: what the kernels of kv8_att.cu share.
#pragma once
#include "ops.cuh"

namespace h2 {

struct AttArgs {
  const void* q;
  long long q_row, q_head;
  void* out;
  long long out_row, out_head;
  float* lse;
  const int8_t* kv;
  const float* kv_scale;
  const int* table;
  const int *q_start, *kv_len;
  int n_pages, page_log, kv_heads, heads, group;  // group = heads / kv_heads
  int table_cols, n_req, rows, max_q, window;
  unsigned group_magic;   // see token_of
  int q_vec, out_vec;     // four-element loads of q, stores of out are aligned
  int q_vec16, out_vec16; // rows of q, of out begin at multiples of 16 bytes
  float scale_log2;       // scale * log2(e): scores are kept in powers of two
};

#ifdef __CUDACC__

namespace {

constexpr float P_SHIFT = 8.f;     // weights are kept as 2^(y - m + P_SHIFT), so that small ones stay normal float16 numbers
constexpr float M_SLACK = 6.f;     // the running maximum moves only when a score passes it by this much (2^14 < 65504)

struct Span {  // the division of a row tile's keys (lo .. hi) into spans of `blocks` blocks of `keys` keys, from a multiple of 16
  int first, n_blocks, used;
};
__device__ __forceinline__ Span spans_of(int lo, int hi, int splits, int blocks, int keys) {
  Span s;
  s.first = lo & ~15;
  s.n_blocks = hi > lo ? (hi - s.first + keys - 1) / keys : 0;
  s.used = max(1, min(splits, (s.n_blocks + blocks - 1) / blocks));
  return s;
}

// A request's queries and keys, clamped to what the arrays hold.
struct Request {
  int first, n_q, len;  // first row of q, queries, cached positions
};
__device__ __forceinline__ Request request_of(const AttArgs& a, int r, int* n_all) {  // n_all: the queries, max_q or not
  Request R;
  const int s0 = a.q_start[r], s1 = a.q_start[r + 1];
  *n_all = s1 - s0;
  R.first = max(s0, 0);
  R.n_q = max(0, min(max(0, min(s1, a.rows)) - R.first, a.max_q));  // (not negative: products with the group must not wrap around)
  const long long room = (long long)a.table_cols << a.page_log;
  R.len = max(0, (int)min((long long)a.kv_len[r], room));
  return R;
}

// The first key that the query at position pos sees. (Before position 0 it sees none; with the largest windows the difference would
// not fit there.)
__device__ __forceinline__ int first_key_of(const AttArgs& a, int pos) { return a.window > 0 ? max(pos, 0) + 1 - a.window : 0; }

// The keys that queries t0 .. t1 of a request may attend to: [lo, hi), hi <= lo when there are none.
__device__ __forceinline__ void key_range(const AttArgs& a, const Request& R, int n_all, int t0, int t1, int* lo, int* hi) {
  const int p0 = R.len - n_all + t0, p1 = R.len - n_all + t1;
  *hi = min(p1 + 1, R.len);
  *lo = max(0, first_key_of(a, p0));
}

__device__ __forceinline__ float exp2_fast(float x) {  // ex2.approx: 2 ulp, 0 for -infinity
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// four signed codes (bytes of w, sign bits already flipped) as two pairs of float16: 0x6400 | u is the float16 1024 + u, and
// u = code + 128, so subtracting 1152 leaves the code exactly
__device__ __forceinline__ uint32_t half2_of(uint32_t bytes) {
  const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&bytes), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// What the softmax needs of 16 keys: the scale of K, the term of V's scale in the exponent, the factor that this leaves, and what
// turns a weight back into the softmax's.
struct __align__(16) KeyInfo {
  float k, e, mant, inv;
};
// The scale of V is split as mantissa * 2^e: the exponent joins the score before the running maximum is taken, so that the
// weights that enter the tensor cores never leave float16's range however the pages' scales differ; the mantissa
// multiplies the weight. e is bounded so that 2^-e stays a normal number.
__device__ __forceinline__ void split_scale(float s, float* e, float* mant, float* inv_pow) {
  if (!(fabsf(s) < INFINITY)) {  // a lost page: NaN through the exponent, so that keys a row does not see stay without effect
    *e = __int_as_float(0x7fc00000);
    *mant = *inv_pow = 1.f;
    return;
  }
  const int x = max(-62, min(63, (int)((__float_as_uint(s) >> 23) & 255u) - 127));
  const float inv = __int_as_float((127 - x) << 23);
  *e = (float)x;
  *inv_pow = inv;
  *mant = s * inv;
}

template <class T>
__device__ __forceinline__ void store4(T* dst, const float* v, bool vec) {
  if (vec) {
    alignas(16) T o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = from_f<T>(v[i]);
    if (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(o);
    else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) dst[i] = from_f<T>(v[i]);
  }
}

// row / group, and the head of the group, by a multiplication: group_magic = 2^32 / group, so the quotient is off by at most one
// for rows below 2^31
__device__ __forceinline__ int token_of(const AttArgs& a, int row, int* head) {
  int t = (int)__umulhi((unsigned)row, a.group_magic), r = row - t * a.group;
  if (r >= a.group) t++, r -= a.group;
  if (r < 0) t--, r += a.group;
  *head = r;
  return t;
}

}  // namespace
#endif
}  // namespace h2
