// Penalties for repeated tokens, biases and masks of allowed tokens on a step's logits (h2c_logits_adjust; the formula is
// stated in include/h2cuda.h).
//
// A CTA takes a chunk of one row's vocabulary, whose logits are on their way to registers while it counts the row's earlier tokens that
// fall there in shared memory (whole numbers, so the order does not matter) and its first warp looks for the biased tokens among
// them and adds the biases of each up in the list's order. Then it changes, masks and writes the logits, and at last the few biased ones.
// Bound: bandwidth for many rows, and the instructions of the pass: a token that was said is found in nearly every warp's 256 logits, so
// its division is one of five multiplications where it can be. Each chunk goes through the row's history (from L2), so chunks are long.
// 32 rows of 151,936 float32: 15.3 us (2.6 TB/s); 256 rows behind up to 16,384 tokens, bfloat16: 57 us; one row: 3.6 us.
// A chunk's biased tokens are compared with each other, which counts where many fall into one chunk: 1,024 biases on 151,936 float32
// tokens take 12 us a row (32 rows 45), on 4,096 tokens 150, on 2,048 490; 128 biases 4, 10 and 17; 16 biases 3-4 everywhere.
#include "ops.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace h2 {
namespace {

constexpr int LG_THREADS = 512, LG_PER_SM = 3, LG_BIASES = H2C_LOGITS_MAX_BIASES;
constexpr int LG_AHEAD = 4;                     // units of 16 bytes that a thread has on their way
constexpr int LG_UNITS = LG_AHEAD * LG_THREADS;  // of the longest chunk
constexpr int LG_SAID = 2;                      // units of 4 earlier tokens that a thread has on their way

struct LogitArgs {
  const void* in;
  void* out;
  long long in_row, out_row, tokens_row, bias_row, allowed_row;
  int vocab, chunk, chunks, columns, n_bias;  // chunk: at most LG_UNITS units
  const int *tokens, *length;
  const float *repetition, *presence, *frequency;
  const int* bias_id;
  const float* bias;
  const unsigned* allowed;
};

struct Strength {
  float rep, pres, freq;
  float inv;  // 1 / rep, rounded; 0: quotients are formed by division
};
__device__ __forceinline__ Strength strength_of(const LogitArgs& a, int row) {
  Strength s{a.repetition ? a.repetition[row] : 1.f, a.presence ? a.presence[row] : 0.f, a.frequency ? a.frequency[row] : 0.f, 0.f};
  if (s.rep >= 0x1p-20f && s.rep <= 0x1p20f) s.inv = __fdiv_rn(1.f, s.rep);
  return s;
}
// x / rep as division rounds it. An approximation q is corrected by its remainder, which fma gives exactly: once makes q the quotient
// or one of its neighbours, and from there a correction with the rounded reciprocal rounds right (Markstein 1990), as long as no
// term leaves the normal numbers.
__device__ __forceinline__ float quotient(float x, const Strength& s) {
  if (!(s.inv > 0.f && x > 0x1p-60f && x < 0x1p60f)) return __fdiv_rn(x, s.rep);
  float q = __fmul_rn(x, s.inv);
  q = __fmaf_rn(__fmaf_rn(-q, s.rep, x), s.inv, q);
  return __fmaf_rn(__fmaf_rn(-q, s.rep, x), s.inv, q);
}
// the logit of a token that was said `count` times (single float32 operations)
__device__ __forceinline__ float penalized(float x, unsigned count, const Strength& s) {
  x = x > 0.f ? quotient(x, s) : __fmul_rn(x, s.rep);
  return __fsub_rn(x, __fadd_rn(__fmul_rn(s.freq, (float)count), s.pres));
}

// -infinity's bits, in each logit of a word
template <class T>
constexpr uint32_t MINUS_INF = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;

// Logit i of a word as a number, and put into it.
template <class T>
__device__ __forceinline__ float value_of(uint32_t w, int i) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(w);
  } else {
    const unsigned short u = (unsigned short)(i ? w >> 16 : w);
    return to_f(*reinterpret_cast<const T*>(&u));
  }
}
template <class T>
__device__ __forceinline__ void put_value(uint32_t* w, int i, T x) {
  if constexpr (sizeof(T) == 4) *w = __float_as_uint(x);
  else *w = __byte_perm(*w, *reinterpret_cast<const unsigned short*>(&x), i ? 0x5410 : 0x3254);
}

// The biased tokens of a chunk, in the list's order, in shared memory: their places in the chunk and their entries, and for a token's
// first entry the sum of its biases and its logit.
struct Biased {
  int *n, *at, *entry;
  float *sum, *x;
  int* first;
  __device__ __forceinline__ Biased(uint8_t* p, int most) {
    n = reinterpret_cast<int*>(p);
    at = n + 4, entry = at + most;
    sum = reinterpret_cast<float*>(entry + most), x = sum + most;
    first = reinterpret_cast<int*>(x + most);
  }
  static size_t bytes(int most) { return most ? 16 + 20 * (size_t)most : 0; }
};

// C: type of the counts
template <class T, class C, bool VEC>
__global__ void __launch_bounds__(LG_THREADS, LG_PER_SM) k_logits(const LogitArgs a) {
  extern __shared__ __align__(16) uint8_t sm[];
  constexpr int V = 16 / (int)sizeof(T), UN = LG_AHEAD, CPW = 4 / (int)sizeof(C);  // logits of 16 bytes, counts of a word
  const int tid = threadIdx.x, lane = tid & 31, row = blockIdx.x / a.chunks, c0 = (blockIdx.x - row * a.chunks) * a.chunk;
  const int n = min(a.chunk, a.vocab - c0);
  unsigned* counts = reinterpret_cast<unsigned*>(sm);
  const Biased biased(sm + (a.tokens ? a.chunk * sizeof(C) : 0), a.n_bias);
  const T* in = static_cast<const T*>(a.in) + row * a.in_row + c0;
  T* out = static_cast<T*>(a.out) + row * a.out_row + c0;
  const unsigned* allowed = a.allowed ? a.allowed + row * a.allowed_row + (c0 >> 5) : nullptr;
  auto is_allowed = [&](int i) { return !allowed || (allowed[i >> 5] >> (i & 31) & 1u); };
  // the units of V logits are on their way while the history is counted
  const int units = VEC ? n / V : 0;
  uint4 raw[UN];
#pragma unroll
  for (int k = 0; k < UN; k++) {
    const int u = tid + k * LG_THREADS;
    if (u < units) raw[k] = reinterpret_cast<const uint4*>(in)[u];
  }
  const Strength s = strength_of(a, row);
  auto count_of = [&](unsigned i) { return CPW == 1 ? counts[i] : counts[i >> 1] >> (16 * (i & 1)) & 0xffffu; };
  if (a.tokens) {
    const int* history = a.tokens + row * a.tokens_row;
    const int len = max(0, min(a.length[row], a.columns)), skip = min(len, (int)(((16 - ((uintptr_t)history & 15)) & 15) >> 2));
    const int quads = (len - skip) >> 2, ends = skip + ((len - skip) & 3);  // (at most 6 before the first 16 bytes and after the last)
    const int4* history4 = reinterpret_cast<const int4*>(history + skip);
    // (by all warps but the first where that has biases to look for)
    const int busy = a.n_bias ? 32 : 0, threads = LG_THREADS - busy, me = tid - busy;
    int4 t[LG_SAID];
    auto load = [&](int i0) {
#pragma unroll
      for (int k = 0; k < LG_SAID; k++)
        if (me >= 0 && i0 + k * threads < quads) t[k] = history4[i0 + k * threads];
    };
    load(me);
    const int rest = me >= 0 && me < ends ? history[me < skip ? me : len - ends + me] : -1;
    for (int i = tid; i < a.chunk * (int)sizeof(C) / 16; i += LG_THREADS) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    auto add = [&](int token) {
      const unsigned i = (unsigned)token - (unsigned)c0;
      if (i < (unsigned)n) atomicAdd(counts + i / CPW, CPW == 1 ? 1u : 1u << (16 * (i & 1)));  // (up to 65,535: no carry)
    };
    if (me >= 0) {
      if (me < ends) add(rest);
      for (int i = me; i < quads; i += LG_SAID * threads) {
        if (i != me) load(i);
#pragma unroll
        for (int k = 0; k < LG_SAID; k++)
          if (i + k * threads < quads) add(t[k].x), add(t[k].y), add(t[k].z), add(t[k].w);
      }
    }
  }
  if (a.n_bias && tid < 32) {
    int m = 0;
    for (int e0 = 0; e0 < a.n_bias; e0 += 32) {
      const int e = e0 + lane, token = e < a.n_bias ? a.bias_id[row * a.bias_row + e] : -1, at = token - c0;
      const bool here = token >= c0 && at < n;
      const unsigned b = __ballot_sync(0xffffffffu, here);
      if (here) {
        const int k = m + __popc(b & ((1u << lane) - 1));
        biased.at[k] = at;
        biased.entry[k] = e;
      }
      m += __popc(b);
    }
    if (lane == 0) *biased.n = m;
    __syncwarp();
    const float* b = a.bias + row * a.bias_row;
    for (int k = lane; k < m; k += 32) {
      const int at = biased.at[k];
      const float x = to_f(in[at]);  // (before it is written, where out is in)
      float sum = b[biased.entry[k]];
      bool first = true;
      for (int j = 0; first && j < k; j++) first = biased.at[j] != at;
      for (int j = k + 1; first && j < m; j++)
        if (biased.at[j] == at) sum = __fadd_rn(sum, b[biased.entry[j]]);
      biased.sum[k] = sum;
      biased.x[k] = x;
      biased.first[k] = first;
    }
  }
  __syncthreads();
  // (most units hold no token that was said: their counts are looked at together)
  constexpr int CW = V * (int)sizeof(C) / 4, PER = 4 / (int)sizeof(T);  // words of a unit's counts; logits of a word
#pragma unroll
  for (int k = 0; k < UN; k++) {
    const int u = tid + k * LG_THREADS;
    if (u >= units) break;
    uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
    if (a.tokens) {
      uint32_t c[CW], any = 0;
#pragma unroll
      for (int i = 0; i < CW; i += 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(counts + u * CW + i);
        c[i] = x.x, c[i + 1] = x.y;
        any |= x.x | x.y;
      }
      if (any) {
#pragma unroll
        for (int i = 0; i < V; i++) {
          const unsigned said = CPW == 1 ? c[i / CPW] : i % CPW ? c[i / CPW] >> 16 : c[i / CPW] & 0xffffu;
          if (said) {
            const T x = from_f<T>(penalized(value_of<T>(w[i / PER], i % PER), said, s));
            put_value<T>(&w[i / PER], i % PER, x);
          }
        }
      }
    }
    if (allowed) {
      const unsigned bits = ~(allowed[u * V >> 5] >> (u * V & 31));  // of those that may not come
#pragma unroll
      for (int i = 0; i < 4; i++) {
        uint32_t m;
        if (sizeof(T) == 4) m = bits >> i & 1u ? ~0u : 0u;
        else m = (bits >> (2 * i) & 1u ? 0xffffu : 0u) | (bits >> (2 * i + 1) & 1u ? 0xffff0000u : 0u);
        w[i] = (w[i] & ~m) | (MINUS_INF<T> & m);
      }
    }
    reinterpret_cast<uint4*>(out)[u] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  for (int i = units * V + tid; i < n; i += LG_THREADS) {
    const unsigned said = a.tokens ? count_of(i) : 0u;
    if (!is_allowed(i)) out[i] = from_f<T>(-INFINITY);
    else if (said) out[i] = from_f<T>(penalized(to_f(in[i]), said, s));
    else out[i] = in[i];
  }
  if (a.n_bias) {
    __syncthreads();
    for (int k = tid; k < *biased.n; k += LG_THREADS) {
      const int at = biased.at[k];
      if (!biased.first[k] || !is_allowed(at)) continue;
      const unsigned said = a.tokens ? count_of(at) : 0u;
      out[at] = from_f<T>(__fadd_rn(said ? penalized(biased.x[k], said, s) : biased.x[k], biased.sum[k]));
    }
  }
}

template <class T, class C>
int launch_logits(const char* who, const LogitArgs& a, int rows, bool vec, cudaStream_t st) {
  static unsigned char done[OP_MAX_DEVICES];
  constexpr int most = LG_UNITS * (16 / (int)sizeof(T)) * (int)sizeof(C) + 16 + 20 * LG_BIASES;
  if (int rc = op_once(who, done, [] {
        const cudaError_t c = cudaFuncSetAttribute(k_logits<T, C, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        return c != cudaSuccess ? c : cudaFuncSetAttribute(k_logits<T, C, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
      }))
    return rc;
  const size_t smem = (a.tokens ? (size_t)a.chunk * sizeof(C) : 0) + Biased::bytes(a.n_bias);
  if (vec) k_logits<T, C, true><<<rows * a.chunks, LG_THREADS, smem, st>>>(a);
  else k_logits<T, C, false><<<rows * a.chunks, LG_THREADS, smem, st>>>(a);
  return op_launched(who);
}

}  // namespace
}  // namespace h2

using namespace h2;

extern "C" int h2c_logits_adjust(int32_t type, const void* logits, int64_t in_row, void* out, int64_t out_row, int32_t rows,
                                 int32_t vocab, const int32_t* tokens, int64_t tokens_row, int32_t columns, const int32_t* length,
                                 const float* repetition, const float* presence, const float* frequency, const int32_t* bias_id,
                                 const float* bias, int32_t n_bias, const int32_t* allowed, int64_t allowed_row, void* stream) {
  const char* who = "h2c_logits_adjust";
  if (!op_type_ok(type)) return op_error(H2C_ERR_BAD_TYPE, "%s: element type %d", who, type);
  if (rows < 0 || rows > OP_MAX_ROWS || vocab < 1 || vocab > (1 << 30) || columns < 0)
    return op_error(H2C_ERR_INVALID, "%s: %d rows of %d, %d columns of tokens", who, rows, vocab, columns);
  if (n_bias < 0 || n_bias > LG_BIASES)
    return op_error(H2C_ERR_INVALID, "%s: n_bias must be 0 to %d, not %d", who, LG_BIASES, n_bias);
  if (rows == 0) return H2C_OK;
  if (!logits || !out || (n_bias && (!bias_id || !bias)) || !tokens != !length) return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  if (!tokens && (repetition || presence || frequency))
    return op_error(H2C_ERR_INVALID, "%s: penalties need the tokens that they are for", who);
  const int64_t es = (int64_t)op_elem_size(type), words = (vocab + 31LL) / 32;
  if (((uintptr_t)logits | (uintptr_t)out) & (es - 1))
    return op_error(H2C_ERR_INVALID, "%s: logits and out must be aligned to their elements", who);
  if (rows > 1 && (out_row < 0 ? -out_row : out_row) < vocab)
    return op_error(H2C_ERR_INVALID, "%s: rows of out overlap (%lld elements apart, %d long)", who, (long long)out_row, vocab);
  const OpRows from{logits, rows, in_row * es, vocab * es}, to{out, rows, out_row * es, vocab * es};
  const bool in_place = logits == out && (in_row == out_row || rows == 1);
  if (!in_place && op_rows_meet(from, to))
    return op_error(H2C_ERR_INVALID, "%s: out must be logits itself or share no memory with it", who);
  {
    auto lines = [&](const char* name, const void* p, int64_t row, int64_t len) {  // of 32-bit values
      OpRange r = op_range(name, OpRows{p, rows, row * 4, len * 4});
      if (!p || !len) r.bytes = 0;
      r.align = 4;
      return r;
    };
    const OpRange written = op_range("out", to);
    const OpRange in[] = {lines("tokens", tokens, tokens_row, columns), lines("length", length, 1, 1),
                          lines("repetition", repetition, 1, 1), lines("presence", presence, 1, 1),
                          lines("frequency", frequency, 1, 1), lines("bias_id", bias_id, n_bias, n_bias),
                          lines("bias", bias, n_bias, n_bias), lines("allowed", allowed, allowed_row, words)};
    if (int rc = op_check_ranges(who, &written, 1, in, 8)) return rc;
  }
  LogitArgs a{};
  a.in = logits; a.out = out; a.in_row = in_row; a.out_row = out_row; a.tokens_row = tokens_row; a.bias_row = n_bias;
  a.allowed_row = allowed_row; a.vocab = vocab; a.columns = columns; a.n_bias = n_bias;
  a.tokens = columns ? tokens : nullptr; a.length = length;
  a.repetition = repetition; a.presence = presence; a.frequency = frequency; a.bias_id = bias_id; a.bias = bias;
  a.allowed = reinterpret_cast<const unsigned*>(allowed);
  const bool wide = columns > 65535;  // counts of 32 bits
  // The longest chunks that leave every SM two CTAs, one behind long histories, through which every chunk goes: us with one, two and three
  // CTAs an SM, 151,936 logits, float32: 8 rows 6.5, 5.8 and 6.8, 16 rows 7.8, 7.9 and 9.2; 3 rows behind 16,384 tokens 8.0, 9.9 and 9.9,
  // 12 such 11.1, 12.8 and 12.8.
  const int ctas = columns > 8192 ? 148 : 148 * 2;
  a.chunk = LG_UNITS * (int)(16 / es);
  while (a.chunk > 1024 && rows * ((vocab + a.chunk - 1LL) / a.chunk) < ctas) a.chunk /= 2;
  const long long chunks = (vocab + a.chunk - 1LL) / a.chunk;
  if (chunks * rows > INT_MAX) return op_error(H2C_ERR_INVALID, "%s: too many logits for one call", who);
  a.chunks = (int)chunks;
  const bool vec = !(((uintptr_t)logits | (uintptr_t)out | (rows > 1 ? in_row * es | out_row * es : 0)) & 15);
  cudaStream_t st = (cudaStream_t)stream;
#define H2_LOGITS(T) (wide ? launch_logits<T, uint32_t>(who, a, rows, vec, st) : launch_logits<T, uint16_t>(who, a, rows, vec, st))
  if (type == H2C_TYPE_F32) return H2_LOGITS(float);
  if (type == H2C_TYPE_F16) return H2_LOGITS(__half);
  return H2_LOGITS(__nv_bfloat16);
#undef H2_LOGITS
}
