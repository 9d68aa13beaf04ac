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
  int q_vec, out_vec;     // four-element loads of q, stores of out are aligned
  float scale_log2;       // scale * log2(e): scores are kept in powers of two
};

#ifdef __CUDACC__

// A request's queries and keys, clamped to what the arrays hold.
struct Request {
  int first, n_q, len;  // first row of q, queries, cached positions
};
__device__ __forceinline__ Request request_of(const AttArgs& a, int r) {
  Request R;
  const int s0 = a.q_start[r], s1 = a.q_start[r + 1];
  R.first = max(s0, 0);
  R.n_q = min(min(s1, a.rows) - R.first, a.max_q);
  const long long room = (long long)a.table_cols << a.page_log;
  R.len = max(0, (int)min((long long)a.kv_len[r], room));
  return R;
}

// The keys that queries t0 .. t1 of a request may attend to: [lo, hi), hi <= lo when there are none.
__device__ __forceinline__ void key_range(const AttArgs& a, const Request& R, int n_all, int t0, int t1, int* lo, int* hi) {
  const int p0 = R.len - n_all + t0, p1 = R.len - n_all + t1;
  *hi = min(p1 + 1, R.len);
  *lo = a.window > 0 ? max(0, p0 + 1 - a.window) : 0;
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
// The scale of V is split as mantissa * 2^e: the exponent joins the score before the running maximum is taken, so that the
// weights that enter the tensor cores never leave float16's range however the pages' scales differ; the mantissa
// multiplies the weight. e is bounded so that 2^-e stays a normal number.
__device__ __forceinline__ void split_scale(float s, float* e, float* mant, float* inv_pow) {
  const int x = max(-62, min(63, (int)((__float_as_uint(s) >> 23) & 255u) - 127));
  const float inv = __int_as_float((127 - x) << 23);
  *e = (float)x;
  *inv_pow = inv;
  *mant = s * inv;
}

#endif
}  // namespace h2
