// Rotary positions of queries and keys (h2c_rope; the formula is stated in include/h2cuda.h).
//
// A warp takes a token, or some of its heads where tokens are few: its lanes make the cosines and sines of the token's pairs, once for all
// heads, and hand them around through shared memory. A lane then has the same few pairs of every head that it turns, so it keeps their
// cosines and sines, and goes from head to head with loads and stores of 16 bytes where the layout has them.
// Bound: bandwidth for many tokens (16,392 of 32 heads of 128, bfloat16: 44 us, 6.0 TB/s), the launch and the 64-bit angles of a warp for
// few (one token 2.5 us).
// The angle is formed in turns: position * frequency / 2 pi, of which the product's remainder and the factor's are kept, too, so that what
// is left without the whole turns is exact to 2^-52 at any position. Its cosine and sine are taken in 64 bits and rounded once, times the
// magnitude (angles and functions in 32 bits: 0.93 x 2^-24 of a vector for 0.62, and 0.1-0.2 us less).
#include "ops.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace h2 {
namespace {

constexpr int ROPE_WARPS = 8, ROPE_AHEAD = 4;  // of a CTA; heads that a lane has under way

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
  int tokens, head_dim, half, parts;  // half = pairs of a head; parts: warps that share a token's heads
};

// A pair turned: one product rounded, the other exact within its addition, whatever the layout.
__device__ __forceinline__ float turned_a(float a, float b, float2 cs) { return fmaf(a, cs.x, -__fmul_rn(b, cs.y)); }
__device__ __forceinline__ float turned_b(float a, float b, float2 cs) { return fmaf(b, cs.x, __fmul_rn(a, cs.y)); }

// Cosine and sine of position * frequency, times the magnitude, rounded once.
__device__ __forceinline__ float2 turn_of(double position, double frequency, double magnitude) {
  constexpr double HI = 0.15915494309189535, LO = -9.839338337591243e-18;  // 1 / 2 pi
  const double angle = position * frequency, angle_rest = fma(position, frequency, -angle);
  const double turns = angle * HI, rest = fma(angle, HI, -turns) + fma(angle, LO, angle_rest * HI);
  double s, c;
  sincospi(2. * ((turns - rint(turns)) + rest), &s, &c);
  return make_float2((float)(c * magnitude), (float)(s * magnitude));
}

// W values as they lie in memory
template <class T, int W>
struct Piece {
  static constexpr int B = W * (int)sizeof(T);
  alignas(W * sizeof(T) >= 16 ? 16 : W * sizeof(T)) T v[W];
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

// Two 16-bit values of a word as float32, and float32 rounded to them.
template <class T>
__device__ __forceinline__ float2 two_of(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <class T>
__device__ __forceinline__ uint32_t word_of(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
// A unit's pairs turned: (p[i], q[i]), or the neighbours of p.
template <bool INTER, class T, int N, int W>
__device__ __forceinline__ void turn_unit(Piece<T, N>& p, Piece<T, W>& q, const float2* cs) {
  if constexpr (sizeof(T) == 2 && W > 1) {
    uint32_t* pw = reinterpret_cast<uint32_t*>(p.v);
    uint32_t* qw = reinterpret_cast<uint32_t*>(q.v);
#pragma unroll
    for (int i = 0; i < W / 2; i++) {
      const float2 x = two_of<T>(pw[i]);
      if constexpr (INTER) {
        const float2 c = cs[i];
        pw[i] = word_of<T>(turned_a(x.x, x.y, c), turned_b(x.x, x.y, c));
      } else {
        const float2 y = two_of<T>(qw[i]);
        const float4 c = reinterpret_cast<const float4*>(cs)[i];
        const float2 c0 = make_float2(c.x, c.y), c1 = make_float2(c.z, c.w);
        pw[i] = word_of<T>(turned_a(x.x, y.x, c0), turned_a(x.y, y.y, c1));
        qw[i] = word_of<T>(turned_b(x.x, y.x, c0), turned_b(x.y, y.y, c1));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < (INTER ? N / 2 : W); i++) {
      T& a = INTER ? p.v[2 * i] : p.v[i];
      T& b = INTER ? p.v[2 * i + 1] : q.v[i];
      const float x = to_f(a), y = to_f(b);
      a = from_f<T>(turned_a(x, y, cs[i]));
      b = from_f<T>(turned_b(x, y, cs[i]));
    }
  }
}

// One unit of work is W neighbouring values and, in the half layout, the W that are their partners; of the part that is not turned, W
// values: W is what 16 bytes hold, or 1 where a pointer, a stride or a head's parts are not multiples of 16 bytes (2,050 tokens of
// 36 heads of 128, bfloat16: 7.2 us, and 39 with 62 of the 128 values turned, which have to go one by one; interleaved 8.0 and 58).
// FEW: a head has at most 32 units, so a lane has one of them, of several heads at a time, and keeps its cosines and sines; else the
// lanes go through a head's units together.
template <class T, int W, bool INTER, bool FEW>
__global__ void __launch_bounds__(32 * ROPE_WARPS, 3) k_rope(const RopeArgs a) {
  extern __shared__ __align__(16) float2 turn[];  // [warp][pair]: cosine and sine, times the magnitude
  constexpr int PP = INTER ? (W == 1 ? 1 : W / 2) : W;  // pairs of a unit
  constexpr int IW = INTER ? 2 * PP : W;                // values of its first piece
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long job = (long long)blockIdx.x * ROPE_WARPS + warp;
  const int t = (int)(job / a.parts), part = (int)(job - (long long)t * a.parts);
  if (t >= a.tokens) return;
  float2* cs = turn + warp * ((a.half + 1) & ~1);
  const int pos = a.position[t];
  for (int j = lane; j < a.half; j += 32) {
    // (a token without a position is copied; an infinite frequency gives NaN, and so does every use of it)
    cs[j] = turn_of((double)max(pos, 0), a.frequency[j], a.magnitude);
  }
  __syncwarp();
  const int rot = a.half / PP, units = rot + (a.head_dim - 2 * a.half) / W, heads = a.side[0].heads + a.side[1].heads;
  // heads at a time, and what of them this lane has; it goes from its first head by as many as all warps of the token take at a time
  const int at_once = FEW ? 32 / units : 1, mine = FEW ? lane / units : 0, step = at_once * a.parts;
  if (mine >= at_once) return;
  auto go = [&](int u, const float2* c) {
    const bool pair = u < rot, turned = pair && pos >= 0;
    const int d = pair ? u * IW : 2 * a.half + (u - rot) * W;
    for (int h0 = part * at_once + mine; h0 < heads; h0 += ROPE_AHEAD * step) {
      Piece<T, IW> p[ROPE_AHEAD];
      Piece<T, W> q[ROPE_AHEAD];
      auto side_of = [&](int h) -> const RopeSide& { return a.side[h >= a.side[0].heads]; };
      auto in_side = [&](int h) { return h >= a.side[0].heads ? h - a.side[0].heads : h; };
#pragma unroll
      for (int k = 0; k < ROPE_AHEAD; k++) {
        const int h = h0 + k * step;
        if (h >= heads) break;
        const RopeSide& s = side_of(h);
        const T* in = static_cast<const T*>(s.in) + t * s.in_row + in_side(h) * s.in_head + d;
        if (!turned && !s.copy) continue;
        if (IW == W || pair) p[k].load(in);
        else p[k].v[0] = in[0];
        if (!INTER && pair) q[k].load(in + a.half);
      }
#pragma unroll
      for (int k = 0; k < ROPE_AHEAD; k++) {
        const int h = h0 + k * step;
        if (h >= heads) break;
        const RopeSide& s = side_of(h);
        T* out = static_cast<T*>(s.out) + t * s.out_row + in_side(h) * s.out_head + d;
        if (!turned && !s.copy) continue;
        if (turned) turn_unit<INTER>(p[k], q[k], c);
        if (IW == W || pair) p[k].store(out);
        else out[0] = p[k].v[0];
        if (!INTER && pair) q[k].store(out + a.half);
      }
    }
  };
  if (FEW) {
    const int u = lane - mine * units;
    alignas(16) float2 kept[PP];
#pragma unroll
    for (int i = 0; i < PP; i++) kept[i] = u < rot ? cs[u * PP + i] : make_float2(1.f, 0.f);
    go(u, kept);
  } else {
    for (int u = lane; u < units; u += 32) go(u, cs + (u < rot ? u * PP : 0));
  }
}

template <class T, int W, bool INTER>
void launch_rope_w(const RopeArgs& a, cudaStream_t st) {
  const int units = a.half / (INTER ? (W == 1 ? 1 : W / 2) : W) + (a.head_dim - 2 * a.half) / W;
  const unsigned ctas = (unsigned)(((long long)a.tokens * a.parts + ROPE_WARPS - 1) / ROPE_WARPS);
  const size_t smem = ROPE_WARPS * ((a.half + 1) & ~1) * sizeof(float2);
  if (units <= 32) k_rope<T, W, INTER, true><<<ctas, 32 * ROPE_WARPS, smem, st>>>(a);
  else k_rope<T, W, INTER, false><<<ctas, 32 * ROPE_WARPS, smem, st>>>(a);
}
template <class T>
void launch_rope(const RopeArgs& a, bool interleaved, bool vec, cudaStream_t st) {
  constexpr int W = 16 / (int)sizeof(T);
  if (interleaved) vec ? launch_rope_w<T, W, true>(a, st) : launch_rope_w<T, 1, true>(a, st);
  else vec ? launch_rope_w<T, W, false>(a, st) : launch_rope_w<T, 1, false>(a, st);
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
  // warps of a token: as many as give every SM 16, at most one for every four heads, since each makes the cosines again. us at 36 heads of
  // 128, bfloat16, with 16 and 32 warps an SM and with one warp a token: 32 tokens 2.9, 2.9 and 4.9, 600 tokens 4.1, 5.8 and 5.0, 2,050
  // tokens 9.3, 10.2 and 9.3. With a warp for every two, four and eight heads: 4 tokens 2.7, 2.7 and 3.1, 150 tokens 3.7, 3.4 and 3.3.
  a.parts = (int)std::max<long long>(1, std::min<long long>((q_heads + k_heads + 3) / 4, 148 * 16 / tokens));
  cudaStream_t st = (cudaStream_t)stream;
  if (type == H2C_TYPE_F32) launch_rope<float>(a, interleaved, vec, st);
  else if (type == H2C_TYPE_F16) launch_rope<__half>(a, interleaved, vec, st);
  else launch_rope<__nv_bfloat16>(a, interleaved, vec, st);
  return op_launched(who);
}
