// Penalties for repeated tokens, biases and masks of allowed tokens on a step's logits (h2c_logits_adjust; the formula is
// stated in include/h2cuda.h).
//
// A CTA takes one row's tokens c0 .. c1 of the vocabulary: it counts the row's earlier tokens that fall there in shared memory
// (whole numbers, so the order of the counting does not matter), and then passes over its logits once. The few biased tokens of
// the chunk are computed beside the pass, each by one thread that adds the token's biases up in the list's order, and written
// after it. Bound: bandwidth for many rows; each chunk reads the row's history again (from L2), so chunks are long where histories are.
#include "ops.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace h2 {
namespace {

constexpr int LG_THREADS = 512, LG_BIASES = H2C_LOGITS_MAX_BIASES, LG_OWN = (LG_BIASES + LG_THREADS - 1) / LG_THREADS;
constexpr int LG_CHUNK = 32768;  // the longest chunk (of 16-bit counts)
constexpr int LG_SMEM = 2 * LG_CHUNK + 4 * LG_BIASES;

struct LogitArgs {
  const void* in;
  void* out;
  long long in_row, out_row, tokens_row, bias_row, allowed_row;
  int vocab, chunk, chunks, columns, n_bias;
  const int *tokens, *length;
  const float *repetition, *presence, *frequency;
  const int* bias_id;
  const float* bias;
  const unsigned* allowed;
};

struct Strength {
  float rep, pres, freq;
};
// the logit of a token that was said `count` times (single float32 operations)
__device__ __forceinline__ float penalized(float x, unsigned count, const Strength& s) {
  if (count) {
    x = x > 0.f ? __fdiv_rn(x, s.rep) : __fmul_rn(x, s.rep);
    x = __fsub_rn(x, __fadd_rn(__fmul_rn(s.freq, (float)count), s.pres));
  }
  return x;
}

// C: type of the counts
template <class T, class C, bool VEC>
__global__ void __launch_bounds__(LG_THREADS) k_logits(const LogitArgs a) {
  extern __shared__ __align__(16) uint8_t sm[];
  constexpr int V = 16 / (int)sizeof(T);
  const int tid = threadIdx.x, row = blockIdx.x / a.chunks, c0 = (blockIdx.x - row * a.chunks) * a.chunk, n = min(a.chunk, a.vocab - c0);
  C* count = reinterpret_cast<C*>(sm);
  int* id = reinterpret_cast<int*>(sm + (a.tokens ? a.chunk * sizeof(C) : 0));
  const T* in = static_cast<const T*>(a.in) + row * a.in_row + c0;
  T* out = static_cast<T*>(a.out) + row * a.out_row + c0;
  const unsigned* allowed = a.allowed ? a.allowed + row * a.allowed_row + (c0 >> 5) : nullptr;
  const Strength s{a.repetition ? a.repetition[row] : 1.f, a.presence ? a.presence[row] : 0.f, a.frequency ? a.frequency[row] : 0.f};
  if (a.tokens) {
    for (int i = tid; i < a.chunk * (int)sizeof(C) / 16; i += LG_THREADS) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int* said = a.tokens + row * a.tokens_row;
    const int len = max(0, min(a.length[row], a.columns));
#pragma unroll 4
    for (int i = tid; i < len; i += LG_THREADS) {
      const unsigned t = (unsigned)said[i] - (unsigned)c0;
      if (t < (unsigned)n) {
        if (sizeof(C) == 4) atomicAdd(reinterpret_cast<unsigned*>(count) + t, 1u);
        else atomicAdd(reinterpret_cast<unsigned*>(count) + (t >> 1), 1u << (16 * (t & 1)));  // (up to 65,535: no carry)
      }
    }
  }
  for (int i = tid; i < a.n_bias; i += LG_THREADS) id[i] = a.bias_id[row * a.bias_row + i];
  __syncthreads();
  auto count_of = [&](int i) { return a.tokens ? (unsigned)count[i] : 0u; };
  auto is_allowed = [&](int i) { return !allowed || (allowed[i >> 5] >> (i & 31) & 1u); };
  // a biased token is the thread's that has its first entry
  float own[LG_OWN];
  unsigned mine = 0;
  if (a.n_bias) {
    const float* b = a.bias + row * a.bias_row;
#pragma unroll
    for (int k = 0; k < LG_OWN; k++) {
      const int e = tid + k * LG_THREADS, t = e < a.n_bias ? id[e] : -1;
      bool first = t >= c0 && t - c0 < n;
      for (int j = 0; first && j < e; j++) first = id[j] != t;
      if (!first) continue;
      float sum = b[e];
      for (int j = e + 1; j < a.n_bias; j++)
        if (id[j] == t) sum = __fadd_rn(sum, b[j]);
      own[k] = is_allowed(t - c0) ? __fadd_rn(penalized(to_f(in[t - c0]), count_of(t - c0), s), sum) : -INFINITY;
      mine |= 1u << k;
    }
    __syncthreads();  // (out may be in: they are read before any is written)
  }
  if (VEC) {
    for (int i = tid * V; i + V <= n; i += LG_THREADS * V) {
      const uint4 raw = *reinterpret_cast<const uint4*>(in + i);
      const T* h = reinterpret_cast<const T*>(&raw);
      alignas(16) T o[V];
      const unsigned bits = allowed ? allowed[i >> 5] >> (i & 31) : ~0u;
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float x = penalized(to_f(h[k]), count_of(i + k), s);
        o[k] = from_f<T>(bits >> k & 1u ? x : -INFINITY);
      }
      *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(o);
    }
  }
  for (int i = (VEC ? n / V * V : 0) + tid; i < n; i += LG_THREADS)
    out[i] = from_f<T>(is_allowed(i) ? penalized(to_f(in[i]), count_of(i), s) : -INFINITY);
  if (a.n_bias) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < LG_OWN; k++)
      if (mine >> k & 1u) out[id[tid + k * LG_THREADS] - c0] = from_f<T>(own[k]);
  }
}

template <class T, class C>
int launch_logits(const char* who, const LogitArgs& a, int rows, int chunks, bool vec, cudaStream_t st) {
  static unsigned char done[OP_MAX_DEVICES];
  if (int rc = op_once(who, done, [] {
        const cudaError_t c = cudaFuncSetAttribute(k_logits<T, C, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, LG_SMEM);
        return c != cudaSuccess ? c : cudaFuncSetAttribute(k_logits<T, C, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, LG_SMEM);
      }))
    return rc;
  const size_t smem = (a.tokens ? (size_t)a.chunk * sizeof(C) : 0) + 4 * a.n_bias;
  if (vec) k_logits<T, C, true><<<rows * chunks, LG_THREADS, smem, st>>>(a);
  else k_logits<T, C, false><<<rows * chunks, LG_THREADS, smem, st>>>(a);
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
  // the longest chunks that leave every SM a few CTAs
  a.chunk = wide ? LG_CHUNK / 2 : LG_CHUNK;
  while (a.chunk > 1024 && rows * ((vocab + a.chunk - 1LL) / a.chunk) < 148 * 4) a.chunk /= 2;
  const long long chunks = (vocab + a.chunk - 1LL) / a.chunk;
  if (chunks * rows > INT_MAX) return op_error(H2C_ERR_INVALID, "%s: too many logits for one call", who);
  a.chunks = (int)chunks;
  const bool vec = !(((uintptr_t)logits | (uintptr_t)out | (rows > 1 ? in_row * es | out_row * es : 0)) & 15);
  cudaStream_t st = (cudaStream_t)stream;
#define H2_LOGITS(T) (wide ? launch_logits<T, uint32_t>(who, a, rows, a.chunks, vec, st) : launch_logits<T, uint16_t>(who, a, rows, a.chunks, vec, st))
  if (type == H2C_TYPE_F32) return H2_LOGITS(float);
  if (type == H2C_TYPE_F16) return H2_LOGITS(__half);
  return H2_LOGITS(__nv_bfloat16);
#undef H2_LOGITS
}
