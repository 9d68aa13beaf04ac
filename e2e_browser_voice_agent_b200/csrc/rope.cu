// Rotary positions of queries and keys (h2c_rope; the formula is stated in include/h2cuda.h).
//
// A CTA takes a few tokens: the angles of each token's pairs are the same for every head, so a thread makes one cosine and sine for
// all of them into shared memory, and then the CTA's vectors are turned with 16-byte loads and stores where the layout has them.
// The angle is formed in turns: position * (frequency / 2 pi) in 64 bits, whose whole turns are dropped before it becomes a
// float32, so far positions are as exact as near ones.
#include "ops.cuh"

#include <algorithm>
#include <climits>

namespace h2 {
namespace {

constexpr int ROPE_THREADS = 256, ROPE_PAIRS = 1024;  // pairs that a CTA holds angles of

struct RopeSide {  // queries or keys
  const void* in;
  void* out;
  long long in_row, in_head, out_row, out_head;
  int heads, copy;  // copy: the part that is not turned goes to out as it is
};
struct RopeArgs {
  RopeSide side[2];
  const int* position;
  const double* frequency;
  float magnitude;
  int tokens, head_dim, half, per_cta;  // half = pairs of a head; tokens of a CTA
};

// A pair turned: one product rounded, the other exact within its addition, whatever the layout.
__device__ __forceinline__ float turned_a(float a, float b, float2 cs) { return fmaf(a, cs.x, -__fmul_rn(b, cs.y)); }
__device__ __forceinline__ float turned_b(float a, float b, float2 cs) { return fmaf(b, cs.x, __fmul_rn(a, cs.y)); }

// W values as they lie in memory
template <class T, int W>
struct Piece {
  static constexpr int B = W * (int)sizeof(T);
  T v[W];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (B % 16 == 0) {
#pragma unroll
      for (int i = 0; i < B / 16; i++) {
        const uint4 x = reinterpret_cast<const uint4*>(p)[i];
        memcpy(reinterpret_cast<char*>(v) + 16 * i, &x, 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; i++) v[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (B % 16 == 0) {
#pragma unroll
      for (int i = 0; i < B / 16; i++) {
        uint4 x;
        memcpy(&x, reinterpret_cast<const char*>(v) + 16 * i, 16);
        reinterpret_cast<uint4*>(p)[i] = x;
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; i++) p[i] = v[i];
    }
  }
};

// One unit of work: W neighbouring values and, in the half layout, the W that are their partners. PAIR: values of a unit that
// hold whole pairs (interleaved).
template <class T, int W, bool INTER>
__global__ void __launch_bounds__(ROPE_THREADS) k_rope(const RopeArgs a) {
  extern __shared__ float2 turn[];  // [token][pair]: cosine and sine, times the magnitude
  constexpr int PP = INTER ? (W == 1 ? 1 : W / 2) : W;  // pairs of a unit
  const int t0 = blockIdx.x * a.per_cta, n = min(a.per_cta, a.tokens - t0);
  for (int i = threadIdx.x; i < n * a.half; i += ROPE_THREADS) {
    const int t = i / a.half, j = i - t * a.half, pos = a.position[t0 + t];
    const double turns = (double)max(pos, 0) * (a.frequency[j] * 0.15915494309189533577);
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    // (a token without a position is copied; an infinite frequency gives NaN, and so does every use of it)
    turn[i] = make_float2(c * a.magnitude, s * a.magnitude);
  }
  __syncthreads();
  const int rot = a.half / PP, rest = (a.head_dim - 2 * a.half) / W, units = rot + rest;  // of a head
  const int heads = a.side[0].heads + a.side[1].heads, all = n * heads * units;
  for (int i = threadIdx.x; i < all; i += ROPE_THREADS) {
    const int th = i / units, u = i - th * units, t = th / heads;
    int h = th - t * heads;
    const bool keys = h >= a.side[0].heads;
    const RopeSide& s = a.side[keys];
    if (keys) h -= a.side[0].heads;
    const T* in = static_cast<const T*>(s.in) + (t0 + t) * s.in_row + h * s.in_head;
    T* out = static_cast<T*>(s.out) + (t0 + t) * s.out_row + h * s.out_head;
    if (u >= rot) {
      if (!s.copy) continue;
      Piece<T, W> p;
      const int d = 2 * a.half + (u - rot) * W;
      p.load(in + d);
      p.store(out + d);
      continue;
    }
    const float2* cs = turn + t * a.half + u * PP;
    const bool turned = a.position[t0 + t] >= 0;
    if (!turned && !s.copy) continue;
    if constexpr (INTER) {
      Piece<T, 2 * PP> p;
      p.load(in + u * 2 * PP);
      if (turned) {
#pragma unroll
        for (int k = 0; k < PP; k++) {
          const float x = to_f(p.v[2 * k]), y = to_f(p.v[2 * k + 1]);
          p.v[2 * k] = from_f<T>(turned_a(x, y, cs[k]));
          p.v[2 * k + 1] = from_f<T>(turned_b(x, y, cs[k]));
        }
      }
      p.store(out + u * 2 * PP);
    } else {
      Piece<T, W> p, q;
      p.load(in + u * W);
      q.load(in + a.half + u * W);
      if (turned) {
#pragma unroll
        for (int k = 0; k < W; k++) {
          const float x = to_f(p.v[k]), y = to_f(q.v[k]);
          p.v[k] = from_f<T>(turned_a(x, y, cs[k]));
          q.v[k] = from_f<T>(turned_b(x, y, cs[k]));
        }
      }
      p.store(out + u * W);
      q.store(out + a.half + u * W);
    }
  }
}

template <class T>
void launch_rope(const RopeArgs& a, bool interleaved, bool vec, cudaStream_t st) {
  constexpr int W = 16 / (int)sizeof(T);
  const int ctas = (a.tokens + a.per_cta - 1) / a.per_cta;
  const size_t smem = (size_t)a.per_cta * a.half * sizeof(float2);
  if (interleaved)
    vec ? k_rope<T, W, true><<<ctas, ROPE_THREADS, smem, st>>>(a) : k_rope<T, 1, true><<<ctas, ROPE_THREADS, smem, st>>>(a);
  else
    vec ? k_rope<T, W, false><<<ctas, ROPE_THREADS, smem, st>>>(a) : k_rope<T, 1, false><<<ctas, ROPE_THREADS, smem, st>>>(a);
}

}  // namespace
}  // namespace h2

using namespace h2;

extern "C" int h2c_rope(int32_t type, const void* q, int64_t q_row, int64_t q_head, void* q_out, int64_t q_out_row, int64_t q_out_head,
                        int32_t q_heads, const void* k, int64_t k_row, int64_t k_head, void* k_out, int64_t k_out_row,
                        int64_t k_out_head, int32_t k_heads, int32_t tokens, int32_t head_dim, const int32_t* position,
                        const double* frequency, int32_t rotary_dim, int32_t interleaved, float magnitude, void* stream) {
  const char* who = "h2c_rope";
  if (!op_type_ok(type)) return op_error(H2C_ERR_BAD_TYPE, "%s: element type %d", who, type);
  if (tokens < 0 || tokens > OP_MAX_ROWS || q_heads < 0 || k_heads < 0 || q_heads > 65536 || k_heads > 65536)
    return op_error(H2C_ERR_INVALID, "%s: %d tokens of %d and %d heads", who, tokens, q_heads, k_heads);
  if (head_dim < 2 || head_dim > 1024 || rotary_dim < 2 || rotary_dim > head_dim || (rotary_dim & 1))
    return op_error(H2C_ERR_INVALID, "%s: rotary_dim (%d) must be even and at most head_dim (%d), which is 2 to 1024", who, rotary_dim, head_dim);
  if (interleaved != 0 && interleaved != 1) return op_error(H2C_ERR_INVALID, "%s: interleaved must be 0 or 1, not %d", who, interleaved);
  if (tokens == 0 || (q_heads == 0 && k_heads == 0)) return H2C_OK;
  if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || !position || !frequency)
    return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  const int64_t es = (int64_t)op_elem_size(type);
  RopeArgs a = {};
  a.position = position; a.frequency = frequency; a.magnitude = magnitude;
  a.tokens = tokens; a.head_dim = head_dim; a.half = rotary_dim / 2;
  a.side[0] = {q, q_out, q_row, q_head, q_out_row, q_out_head, q_heads, 0};
  a.side[1] = {k, k_out, k_row, k_head, k_out_row, k_out_head, k_heads, 0};
  const char* in_name[] = {"q", "k"};
  const char* out_name[] = {"q_out", "k_out"};
  // a token's vectors as one row, between the lowest and the highest
  auto rows_of = [&](const void* at, int64_t row, int64_t head, int heads) {
    const int64_t span = (heads - 1LL) * head;
    return OpRows{static_cast<const uint8_t*>(at) + std::min<int64_t>(0, span) * es, tokens, row * es, (std::abs(span) + head_dim) * es};
  };
  OpRows in[2], out[2];
  bool vec = head_dim * es % 16 == 0 && rotary_dim / (interleaved ? 1 : 2) * es % 16 == 0;
  for (int i = 0; i < 2; i++) {
    RopeSide& s = a.side[i];
    if (!s.heads) continue;
    if (((uintptr_t)s.in | (uintptr_t)s.out) & (es - 1))
      return op_error(H2C_ERR_INVALID, "%s: %s and %s must be aligned to their elements", who, in_name[i], out_name[i]);
    if (op_vectors_overlap(tokens, s.out_row, s.heads, s.out_head, head_dim))
      return op_error(H2C_ERR_INVALID, "%s: vectors of %s overlap (rows %lld elements apart, heads %lld)", who, out_name[i],
                      (long long)s.out_row, (long long)s.out_head);
    in[i] = rows_of(s.in, s.in_row, s.in_head, s.heads);
    out[i] = rows_of(s.out, s.out_row, s.out_head, s.heads);
    const bool in_place = s.in == s.out && (s.in_row == s.out_row || tokens == 1) && (s.in_head == s.out_head || s.heads == 1);
    s.copy = !in_place;
    if (!in_place && op_rows_meet(in[i], out[i]))
      return op_error(H2C_ERR_INVALID, "%s: %s must be %s itself or share no memory with it", who, out_name[i], in_name[i]);
    const OpRange written = op_range(out_name[i], out[i]);
    const OpRange read[] = {{"position", position, 4ull * tokens, 4}, {"frequency", frequency, 4ull * rotary_dim, 8}};
    if (int rc = op_check_ranges(who, &written, 1, read, 2)) return rc;
    auto wide = [&](const void* p, int64_t row, int64_t head) {
      return !(((uintptr_t)p | (tokens > 1 ? row * es : 0) | (s.heads > 1 ? head * es : 0)) & 15);
    };
    vec = vec && wide(s.in, s.in_row, s.in_head) && wide(s.out, s.out_row, s.out_head);
  }
  if (q_heads && k_heads) {
    for (int i = 0; i < 2; i++)
      if (op_rows_meet(out[i], in[1 - i]))
        return op_error(H2C_ERR_INVALID, "%s: %s must not share memory with %s", who, out_name[i], in_name[1 - i]);
    if (op_rows_meet(out[0], out[1])) return op_error(H2C_ERR_INVALID, "%s: q_out must not share memory with k_out", who);
  }
  const long long per_token = ((long long)q_heads + k_heads) * head_dim;
  // tokens of a CTA: some 8 vectors a thread, while that leaves every SM a CTA
  long long per = std::min<long long>({std::max(1LL, 16384 / per_token), ROPE_PAIRS / a.half, (tokens + 295LL) / 296});
  a.per_cta = (int)std::max(1LL, per);
  cudaStream_t st = (cudaStream_t)stream;
  if (type == H2C_TYPE_F32) launch_rope<float>(a, interleaved, vec, st);
  else if (type == H2C_TYPE_F16) launch_rope<__half>(a, interleaved, vec, st);
  else launch_rope<__nv_bfloat16>(a, interleaved, vec, st);
  return op_launched(who);
}
