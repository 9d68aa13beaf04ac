// Attention over the paged 8-bit cache for many queries (prompts, long continuations): the tensor-core kernel of
// h2c_kv8_attention. Included by kv8_att.cu.
//
// A CTA takes 256 rows (query, head of the kv head's group) of one request and kv head, as two tiles of 128, and one span of
// its keys, 64 keys at a time:
//   warps 0-3, 4-7     softmax of row tile 0, 1: a thread owns a row; S from TMEM, P back into S's columns as float16
//   warps 8-11, 12-15  converters of K and of V: 8-bit codes from their pages to float16 tiles in shared memory (exact:
//                      codes are integers up to 127), the next tile's loads in flight meanwhile; both row tiles use them
//   warps 16, 17       tcgen05.mma (kind::f16): S = Q K^T of row tile 0, 1 into TMEM
//   warps 18, 19       O += P V of row tile 0, 1, with P read from TMEM
// The block starts with 96 registers a thread (20 warps); the softmax warps take 136, the converters 64, the last four 56:
// 8 x 136 + 8 x 64 + 4 x 56 = 1,824 of 20 x 96 = 1,920.
// TMEM per row tile: two S slots of 64 columns (P takes its S slot's place) and O. S of the next keys is issued before O's
// update with the present ones, so the tensor cores work while the softmax does.
// * A page's scale of K multiplies its scores; its scale of V joins the exponent (see split_scale), so a row's weights
//   are powers of two relative to one running maximum, which moves only when a score passes it by M_SLACK: only then is
//   O rescaled (by the softmax warps, in TMEM).
// * float32 queries and float32 and float16 rows' weights are two float16 terms each (22 bits), one tcgen05.mma per term.
// * The tensor cores' sums are added up outside them every few tiles of keys (see FOLD).
// * V lies in shared memory as its rows come, [key][dimension]: the second product's B operand in MN-major form.
// * The softmaxes of the two row tiles take turns at the exponentials, so that one's wait for its scores falls into the
//   other's turn (385 us in step with each other, 370 so).
// Bound: a key tile of 256 rows needs 1,024 cycles of exponentials (16 a cycle) and about 1,280 of the tensor cores (the S
// products' operands of 64 keys take 1.5 times their multiply time to read from shared memory). It takes about 2,350: the
// softmax warps issue what lies between a score and its weight (maximum, scale, conversion, TMEM both ways) one after the
// other, and each hand-over between warps costs 115-175 cycles (2.0 stalls an issue at barriers, 1.8 for fixed latencies; tensor
// pipe 27%, issue 45% busy). That is where this form stands, not a bound of the hardware. A CTA spends about 12,500 cycles more
// on its first scores and its last outputs. Measured (4 prompts of 2,064-4,099 tokens, 28 heads over 4, 128 wide, bfloat16): 382
// us, 662 TFLOP/s of the products that the mask leaves. Slower: tiles of 128 keys with one S slot (412), two threads a row (405).
// Waits for data are bounded; the allocation of TMEM waits for an SM's other CTAs, which free theirs at their end in any case.
#pragma once
#include "kv8_att.cuh"
#include "tc5_ptx.cuh"

#include <type_traits>

namespace h2 {
namespace {

constexpr int PR_ROWS = 256, PR_KEYS = 64, PR_THREADS = 5 * 128, PR_INFO = 32;
constexpr int PR_SLOTS = 192;  // places for spilled sums
enum { PR_CONVERT = 21, PR_MMA = 22, PR_SOFTMAX = 23, PR_SLOT = 24 };

// The row tiles of all requests, the spans that each is cut into, and the 64-key tiles of a span.
struct PromptShape {
  int tiles, splits, blocks;
};
// Spans: as many as fill `units` CTAs once, of at least `least` key tiles.
__host__ __device__ inline PromptShape prompt_shape(int tiles, int kv_heads, int key_tiles, int units, int least) {
  PromptShape s{tiles, 1, key_tiles < 1 ? 1 : key_tiles};
  const int ctas = tiles * kv_heads;
  if (ctas > 0 && ctas <= units / 2 && key_tiles >= 2 * least) {
    const int most = units / ctas, n = most < key_tiles / least ? most : key_tiles / least;
    s.blocks = (key_tiles + n - 1) / n;
    s.splits = (key_tiles + s.blocks - 1) / s.blocks;
  }
  return s;
}

struct PromptArgs {
  AttArgs a;
  int min_rows;       // requests of fewer rows are k_att_rows'
  PromptShape shape;  // as the host knows it: exact, or a bound of the row tiles, which are one span each
  int key_tiles;      // bound of a history's 64-key tiles
  int units;          // above 0: the shape is found here, for up to so many CTAs
  float* part;
  float2* ml;
  float* sums;        // (PromptCfg::SPILL) PR_SLOTS places of 256 rows' sums; nullptr where no row tile has more than FOLD tiles of keys
  int* err;
};

// The host knows a single request's row tiles. Those of several depend on how their queries are spread (one chunk of a prompt
// beside many single tokens has few), and are counted here by whole warps, as is the longest history among them. Spans of 512
// keys or more: shorter ones take from k_att_rows' CTAs what they gain (31 single tokens of 100-4,096 and a chunk of 256 on 4,096, 28
// heads over 4 of 128: 115 us in one span, 74 in 5; with a chunk of 512 on 512 instead: 50 us, 65 in two spans of 256 keys, and
// 55 with the count that finds none).
__device__ __forceinline__ PromptShape shape_of_call(const PromptArgs& pa) {
  if (!pa.units) return pa.shape;
  const AttArgs& a = pa.a;
  int n = 0, keys = 0;
#pragma unroll 4
  for (int r = threadIdx.x & 31; r < a.n_req; r += 32) {
    int n_all;
    const Request R = request_of(a, r, &n_all);
    const int rows = R.n_q * a.group;
    if (rows >= pa.min_rows) {
      n += (rows + PR_ROWS - 1) / PR_ROWS;
      keys = max(keys, R.len);
    }
  }
  n = min(pa.shape.tiles, __reduce_add_sync(0xffffffffu, n));
  keys = min(pa.key_tiles, __reduce_max_sync(0xffffffffu, keys) / PR_KEYS + 1);
  return prompt_shape(n, a.kv_heads, keys, pa.units, 8);
}

// The idx-th row tile over all requests: its request (r = -1 beyond the last), what it holds, and the tile's first row. Called
// by whole warps.
struct TileAt {
  int r, row0, n_all;  // n_all: the request's queries, max_q or not
  Request R;
};
__device__ __forceinline__ TileAt tile_at(const PromptArgs& pa, int idx) {
  const AttArgs& a = pa.a;
  const int lane = threadIdx.x & 31;
  TileAt t{-1, 0, 0, {0, 0, 0}};
  int before = 0;
  for (int base = 0; base < a.n_req; base += 32) {
    const int r = base + lane;
    int n = 0, n_all = 0;
    Request R{0, 0, 0};
    if (r < a.n_req) {
      R = request_of(a, r, &n_all);
      const int rows = R.n_q * a.group;
      if (rows >= pa.min_rows) n = (rows + PR_ROWS - 1) / PR_ROWS;
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += u;
    }
    const int at = idx - before;  // among these requests' tiles
    const unsigned in = __ballot_sync(0xffffffffu, at >= sum - n && at < sum);
    if (in) {
      const int l = __ffs(in) - 1;
      t.r = base + l;
      t.row0 = (at - __shfl_sync(0xffffffffu, sum - n, l)) * PR_ROWS;
      t.n_all = __shfl_sync(0xffffffffu, n_all, l);
      t.R.first = __shfl_sync(0xffffffffu, R.first, l);
      t.R.n_q = __shfl_sync(0xffffffffu, R.n_q, l);
      t.R.len = __shfl_sync(0xffffffffu, R.len, l);
      return t;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return t;
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]),
      "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]),
      "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
      : "memory");
}
// packed pairs of float32
__device__ __forceinline__ unsigned long long pair(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(unsigned long long v, float* a, float* b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(v));
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// D (TMEM, float32) (+)= A B with float16 operands: both in shared memory, or A in TMEM
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
// A wait of a warpgroup: its first thread polls (many pollers slow every barrier operation of the SM down: measured 250
// cycles per completed wait with 17 warps polling), the others stand at a named barrier. `go` holds the outcome for two waits
// in turn, so that every thread of the group takes the same way; false when the wait expired.
__device__ __forceinline__ bool wait_group(uint64_t* b, unsigned parity, const Abort& a, int role, int id, volatile int* go, int j) {
  if ((threadIdx.x & 127) == 0) go[j & 1] = wait_phase(b, parity, a, role);
  asm volatile("barrier.sync %0, 128;" ::"r"(id) : "memory");  // (a warp need not have come together)
  return go[j & 1] != 0;
}
// whether the phase has completed, without waiting
__device__ __forceinline__ bool bar_test(uint64_t* b, unsigned parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok)
               : "r"(su32(b)), "r"(parity)
               : "memory");
  return ok != 0;
}
// both phases (their tests in flight together: a test takes over 100 cycles)
__device__ __forceinline__ bool wait_two(uint64_t* b0, unsigned p0, uint64_t* b1, unsigned p1, const Abort& a, int role) {
  const bool d0 = bar_test(b0, p0), d1 = bar_test(b1, p1);
  return (d0 || wait_phase(b0, p0, a, role)) && (d1 || wait_phase(b1, p1, a, role));
}
// a 128-byte-swizzled tile of 64-element (128-byte) rows: byte address of the 16-byte piece c of row r
__device__ __forceinline__ uint32_t sw128(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

template <class T, int HD>
struct PromptCfg {
  static constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  static constexpr int Q_TERMS = sizeof(T) == 4 ? 2 : 1;  // float16 terms of queries
  // ... and of weights. One where the output is bfloat16: 2^-12 of each weight, an eighth of that rounding. With float16 outputs one
  // term's error would be as large as theirs (some 1.2 times the error in all; 445 us for the prompts below, 543 with two).
  static constexpr int P_TERMS = BF16 ? 1 : 2;
  static constexpr int BLKS = HD / 64;                   // 64-dimension blocks of a row
  static constexpr int Q_TILE = 128 * HD * 2;            // one row tile, one term
  static constexpr int KV_TILE = PR_KEYS * HD * 2;
  static constexpr int OUT_LD = 256 + 16;                // bytes per row of a row tile's output staging: up to 256 of the row
  // a row tile's queries, later the staging of its output
  static constexpr int Q_AREA = Q_TERMS * Q_TILE > 128 * OUT_LD ? Q_TERMS * Q_TILE : 128 * OUT_LD;
  // Tensor cores cut off what their float32 sums cannot hold, so a sum over many tiles of keys shrinks with each. O therefore
  // holds FOLD tiles' sum and is then added to the sum so far by the softmax warps, which round. 64 wide that lies beside O in
  // TMEM; 128 wide there is no room, and it lies in a place of the workspace (SPILL, claim_slot). One span of 4,000 and 131,072 keys,
  // relative to the output: off by 7e-6 and 4.5e-4 without (16-bit types, before their rounding: 5e-6 and 4e-4). Float32 4e-7 and
  // 1.5e-6 so 64 wide (a chunk of 256 on 4,096 tokens takes 30 us for 27.6), 8e-7 and 1.6e-6 128 wide (that chunk, 28 heads over 4, 62
  // us for 53, prompts of 2,064-4,099 797 for 650: the places' way to L2. 4 tiles: 63 and 830 us, 4e-7 and 1.4e-6; CTAs of one row
  // tile, whose sum fits into the other's TMEM: 78 and 1,071). 16-bit types 1.2e-5 and less, a twentieth of float16's rounding: chunks
  // on 32,000 and more keys take 2-3% longer.
  static constexpr int FOLD = sizeof(T) == 4 ? (HD == 64 ? 4 : 8) : HD == 64 ? 32 : BF16 ? 128 : 64;
  static constexpr bool SPILL = HD == 128;
  static constexpr int OFF_K = 2 * Q_AREA;
  static constexpr int STAGES = Q_TERMS * HD > 128 ? 2 : 3;   // K and V tiles each
  static constexpr int OFF_V = OFF_K + STAGES * KV_TILE;
  static constexpr int SMEM = OFF_V + STAGES * KV_TILE + 1024;
  static_assert(Q_AREA % 1024 == 0 && SMEM <= 226 * 1024, "shared memory budget");
};

// The weights of one tile of keys for one row: scores s (products of codes) to p = 2^(s f + e - m), times V's mantissa where the
// exponent does not hold it (MANT), packed as float16 (and the remainders when two terms are kept); the sum of the softmax's weights
// is added to l. base = P_SHIFT - m.
template <int TERMS, bool MANT, bool EDGE>
__device__ __forceinline__ void weights(const float* s, const KeyInfo* in, float base, int key0, int first_key,
                                        int pos, uint32_t* p, uint32_t* rest, float* l) {
#pragma unroll
  for (int g = 0; g < PR_KEYS / 16; g++) {
    const float f = in[g].k, e = in[g].e + base;
    const unsigned long long ff = pair(f, f), ee = pair(e, e);
    unsigned long long sum = 0;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      float w0, w1;
      unpair(fma2(pair(s[16 * g + i], s[16 * g + i + 1]), ff, ee), &w0, &w1);
      if (EDGE) {
        const int key = key0 + 16 * g + i;
        w0 = key <= pos && key >= first_key ? w0 : -INFINITY;
        w1 = key + 1 <= pos && key + 1 >= first_key ? w1 : -INFINITY;
      }
      w0 = exp2_fast(w0);
      w1 = exp2_fast(w1);
      sum = add2(sum, pair(w0, w1));
      if (MANT) {
        w0 *= in[g].mant;
        w1 *= in[g].mant;
      }
      if (TERMS == 2) {
        const __half2 t = __floats2half2_rn(w0, w1);
        p[8 * g + i / 2] = *reinterpret_cast<const uint32_t*>(&t);
        rest[8 * g + i / 2] = pack_half2(w0 - __low2float(t), w1 - __high2float(t));
      } else {
        p[8 * g + i / 2] = pack_half2(w0, w1);
      }
    }
    float s0, s1;
    unpair(sum, &s0, &s1);
    *l = fmaf(s0 + s1, in[g].inv, *l);
  }
}

// Eight values as they lie in memory, and as float32.
template <class T>
struct Raw8 {
  uint32_t w[2 * sizeof(T)];
  __device__ __forceinline__ float at(int i) const { return to_f(reinterpret_cast<const T*>(w)[i]); }
  // the largest magnitude's bits as a float32 (infinities and NaN above every number)
  __device__ __forceinline__ unsigned largest() const {
    unsigned m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; i++) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      m = max(m & 0xffffu, m >> 16);
      const unsigned short u = (unsigned short)m;
      return __float_as_uint(to_f(*reinterpret_cast<const T*>(&u)));
    }
  }
};

// A warp's 32 rows of a row tile's queries (from row r0 of the tile, which begins at row tile0 of the request): HD / 8 lanes a
// row; lane i has the place of row i in q (row_at). Rows past the last are zeros, and not read: all of them from one place took
// a chunk of 10 float32 tokens on 16,000 positions from 19 to 35 us. A row is scaled by a power of two so that its largest magnitude lies in
// [2^13, 2^14) and split into one or two float16 terms; what undoes the scaling, times the softmax scale, goes to row_scale.
// The raw values are copied to where their terms will lie (8 of them take as many bytes as their terms do) and replaced
// there by the same lane. Rolled loops: code that runs once waits for its own fetching.
template <class T, int HD>
__device__ __forceinline__ void put_queries(const AttArgs& a, long long row_at, int n_rows, int tile0, int r0, uint8_t* qt,
                                            float* row_scale) {
  using C = PromptCfg<T, HD>;
  constexpr int LPR = HD / 8, RPP = 32 / LPR, PASSES = 32 / RPP, NB = 4;
  const int lane = threadIdx.x & 31, sub = lane / LPR, piece = lane % LPR;
  const T* q = static_cast<const T*>(a.q) + 8 * piece;
  uint8_t* blk = qt + (piece >> 3) * (128 * 128);
  if (a.q_vec16) {
#pragma unroll 2
    for (int p = 0; p < PASSES; p++) {
      const T* src = q + __shfl_sync(0xffffffffu, row_at, p * RPP + sub);
      const uint32_t dst = su32(blk + sw128(r0 + p * RPP + sub, piece & 7));
      const int bytes = tile0 + r0 + p * RPP + sub < n_rows ? 16 : 0;  // (what is not copied is filled with zeros)
#pragma unroll
      for (int t = 0; t < C::Q_TERMS; t++)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + t * C::Q_TILE), "l"(src + t * 4), "r"(bytes)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
  } else {
#pragma unroll 1
    for (int p = 0; p < PASSES; p++) {
      const T* src = q + __shfl_sync(0xffffffffu, row_at, p * RPP + sub);
      uint8_t* dst = blk + sw128(r0 + p * RPP + sub, piece & 7);
      const bool live = tile0 + r0 + p * RPP + sub < n_rows;
#pragma unroll
      for (int i = 0; i < 8; i++)
        *reinterpret_cast<T*>(dst + (i * (int)sizeof(T) >> 4) * C::Q_TILE + (i * (int)sizeof(T) & 15)) =
            live ? src[i] : from_f<T>(0.f);
    }
  }
#pragma unroll 1
  for (int p0 = 0; p0 < PASSES; p0 += NB) {
    Raw8<T> v[NB];
    unsigned m[NB];
    // (each step for all passes, so that their latencies overlap)
#pragma unroll
    for (int b = 0; b < NB; b++) {
      const uint8_t* at = blk + sw128(r0 + (p0 + b) * RPP + sub, piece & 7);
#pragma unroll
      for (int t = 0; t < C::Q_TERMS; t++) {
        const uint4 x = *reinterpret_cast<const uint4*>(at + t * C::Q_TILE);
        v[b].w[4 * t] = x.x, v[b].w[4 * t + 1] = x.y, v[b].w[4 * t + 2] = x.z, v[b].w[4 * t + 3] = x.w;
      }
    }
#pragma unroll
    for (int b = 0; b < NB; b++) m[b] = v[b].largest();
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1)
#pragma unroll
      for (int b = 0; b < NB; b++) m[b] = max(m[b], __shfl_xor_sync(0xffffffffu, m[b], o));
#pragma unroll
    for (int b = 0; b < NB; b++) {
      const int r = r0 + (p0 + b) * RPP + sub;
      const int e = (int)(m[b] >> 23);
      const int up = e == 255 || m[b] == 0 ? 127 : min(253, 267 - e);
      // (the sign of the softmax scale goes into the query, so that larger products are larger scores)
      const float mul = copysignf(__int_as_float(up << 23), a.scale_log2);
      if (piece == 0) row_scale[r] = __int_as_float((254 - up) << 23) * fabsf(a.scale_log2);
      uint32_t h[4], rest[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float x0 = v[b].at(2 * i) * mul, x1 = v[b].at(2 * i + 1) * mul;
        const __half2 t = __floats2half2_rn(x0, x1);
        h[i] = *reinterpret_cast<const uint32_t*>(&t);
        if (C::Q_TERMS == 2) rest[i] = pack_half2(x0 - __low2float(t), x1 - __high2float(t));
      }
      uint8_t* at = blk + sw128(r, piece & 7);
      *reinterpret_cast<uint4*>(at) = make_uint4(h[0], h[1], h[2], h[3]);
      if (C::Q_TERMS == 2) *reinterpret_cast<uint4*>(at + C::Q_TILE) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

// A place for spilled sums that no other CTA at work holds, for a whole CTA until release_slot: by one thread. An SM has one CTA
// of k_att_prompt at a time (its shared memory), so there are more places than CTAs at work in all streams together, and the first
// that is tried, the SM's number, is nearly always free. -1 (and the abort flag) if none was within the time limit.
__device__ int g_slot_held[PR_SLOTS];  // 0 between kernels
__device__ __forceinline__ int claim_slot(const Abort& a) {
  unsigned sm;
  asm volatile("mov.u32 %0, %smid;" : "=r"(sm));
  int at = (int)(sm % PR_SLOTS);
  const unsigned long long t0 = now_ns();
  for (unsigned it = 1;; it++) {
    if (atomicCAS(g_slot_held + at, 0, 1) == 0) break;
    at = at + 1 == PR_SLOTS ? 0 : at + 1;
    if (it % PR_SLOTS == 0 && now_ns() - t0 > TIMEOUT_NS) {
      raise_abort(a, PR_SLOT);
      return -1;
    }
  }
  __threadfence();
  return at;
}
__device__ __forceinline__ void release_slot(int slot) {
  __threadfence();
  atomicExch(g_slot_held + slot, 0);
}

// The place of a thread's columns col .. col + 3 in a row tile's spilled sums: [columns / 4][128 rows], so that a warp's accesses are
// whole lines. (Read and written in L2: the place was another SM's before.)
__device__ __forceinline__ float4* spill_at(float* sums, int trow, int col) {
  return reinterpret_cast<float4*>(sums) + (col >> 2) * 128 + trow;
}
// A row's O (128 columns) added to its spilled sum, which is multiplied by f first; the first time there is none.
__device__ __forceinline__ void spill_row(float* sums, int trow, uint32_t o_at, float f, bool first) {
#pragma unroll 1
  for (int c = 0; c < 128; c += 32) {
    float4 sum[8];
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] = first ? make_float4(0.f, 0.f, 0.f, 0.f) : __ldcg(spill_at(sums, trow, c + 4 * i));
    float o[32];
    tmem_ld32(o_at + c, o);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 8; i++)
      __stcg(spill_at(sums, trow, c + 4 * i), make_float4(fmaf(sum[i].x, f, o[4 * i]), fmaf(sum[i].y, f, o[4 * i + 1]),
                                                          fmaf(sum[i].z, f, o[4 * i + 2]), fmaf(sum[i].w, f, o[4 * i + 3])));
  }
}

// A thread's row of O (and of the sum of what it held before: at sum_at in TMEM if that is not 0, or spilled, times f, if sums is
// not null), scaled, as NC values of type U at dst (a row of the warp's staging; columns col .. col + NC of the row).
template <class U, int NC>
__device__ __forceinline__ void stage_row(uint8_t* dst, uint32_t o_at, bool any, float inv, uint32_t sum_at, float* sums, int trow,
                                          int col, float f) {
#pragma unroll 1
  for (int c = 0; c < NC; c += 32) {
    float o[32];
    if (any) {
      tmem_ld32(o_at + c, o);
      tc_wait_ld();
      if (sum_at) {
#pragma unroll
        for (int h = 0; h < 32; h += 16) {
          uint32_t sum[16];
          tmem_ld16(sum_at + c + h, sum);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i++) o[h + i] += __uint_as_float(sum[i]);
        }
      }
      if (sums) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float4 x = __ldcg(spill_at(sums, trow, col + c + 4 * i));
          o[4 * i] = fmaf(x.x, f, o[4 * i]);
          o[4 * i + 1] = fmaf(x.y, f, o[4 * i + 1]);
          o[4 * i + 2] = fmaf(x.z, f, o[4 * i + 2]);
          o[4 * i + 3] = fmaf(x.w, f, o[4 * i + 3]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; i++) o[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 32; i += 16 / (int)sizeof(U)) {
      alignas(16) U x[16 / sizeof(U)];
#pragma unroll
      for (int k = 0; k < 16 / (int)sizeof(U); k++) x[k] = from_f<U>(o[i + k] * inv);
      *reinterpret_cast<uint4*>(dst + (c + i) * sizeof(U)) = *reinterpret_cast<const uint4*>(x);
    }
  }
}
// The staged NC values to global memory, where `store` says so: one bulk copy when both sides are 16-byte aligned. On return
// the staging can be written again.
template <class U, int NC>
__device__ __forceinline__ void copy_row(U* dst, const uint8_t* src, bool store, bool bulk) {
  if (bulk) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %3, 0;\n @p cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n}\n" ::"l"(
            __cvta_generic_to_global(dst)),
        "r"(su32(src)), "r"(NC * (int)sizeof(U)), "r"((int)store)
        : "memory");
    asm volatile("cp.async.bulk.commit_group;\ncp.async.bulk.wait_group.read 0;" ::: "memory");
  } else if (store) {
#pragma unroll 1
    for (int i = 0; i < NC; i++) dst[i] = reinterpret_cast<const U*>(src)[i];
  }
  if (!bulk) __syncwarp();
}

// The largest score of one tile of keys among those the row sees, with the exponent of V's scale.
template <bool EDGE>
__device__ __forceinline__ float tile_max(const float* s, const KeyInfo* in, int key0, int first_key, int pos) {
  float mx = -INFINITY;
#pragma unroll
  for (int g = 0; g < PR_KEYS / 16; g++) {
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float x0 = s[16 * g + i + 2 * h], x1 = s[16 * g + i + 2 * h + 1];
        if (EDGE) {
          const int key = key0 + 16 * g + i + 2 * h;
          x0 = key <= pos && key >= first_key ? x0 : -INFINITY;
          x1 = key + 1 <= pos && key + 1 >= first_key ? x1 : -INFINITY;
        }
        top[h] = fmaxf(fmaxf(x0, x1), top[h]);
      }
    }
    const float x = fmaxf(top[0], top[1]);
    // (no key seen: stays -infinity whatever the page's scale is)
    mx = fmaxf(mx, x == -INFINITY ? x : fmaf(x, in[g].k, in[g].e));
  }
  return mx;
}

template <class T, int HD>
__global__ void __launch_bounds__(PR_THREADS, 1) k_att_prompt(const PromptArgs pa) {
  using C = PromptCfg<T, HD>;
  constexpr int STG = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (su32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t k_full[STG], k_empty[STG], v_full[STG], v_empty[STG], i_full[2];
  __shared__ uint64_t s_full[2][2], p_full[2][2], pv_done[2][2], q_full[2], mma_end[4];  // ([row tile][tile of keys & 1])
  __shared__ KeyInfo info[2][PR_INFO][PR_KEYS / 16];  // of two batches of PR_INFO tiles in turn
  __shared__ int go[2][2];
  __shared__ float row_scale[PR_ROWS];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_s, slot_s;
  const AttArgs& a = pa.a;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (k_att_rows or the joining kernel; both wait for this one's end)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PromptShape shape = shape_of_call(pa);
  const int split = (int)blockIdx.x % shape.splits, head = ((int)blockIdx.x / shape.splits) % a.kv_heads;
  // the last tiles of a causal prompt have the most keys and go first
  const int idx = shape.tiles - 1 - (int)blockIdx.x / (shape.splits * a.kv_heads);
  if (idx < 0) return;
  const TileAt at = tile_at(pa, idx);
  if (at.r < 0) return;
  const Request R = at.R;
  const int n_all = at.n_all, n_rows = R.n_q * a.group;
  int lo, hi;
  key_range(a, R, n_all, at.row0 / a.group, min(at.row0 + PR_ROWS - 1, n_rows - 1) / a.group, &lo, &hi);
  const Span sp = spans_of(lo, hi, shape.splits, shape.blocks, PR_KEYS);
  if (split >= sp.used) return;
  const int t_begin = split * shape.blocks, t_end = split == sp.used - 1 ? sp.n_blocks : t_begin + shape.blocks;
  const int n_tiles = t_end - t_begin, key_begin = sp.first + t_begin * PR_KEYS;
  const int n_q_tiles = n_rows - at.row0 > 128 ? 2 : 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STG; s++) {
      bar_init(k_full + s, 4);
      bar_init(k_empty + s, n_q_tiles);
      bar_init(v_full + s, 4);
      bar_init(v_empty + s, n_q_tiles);
    }
    bar_init(i_full, 1);
    bar_init(i_full + 1, 1);
    for (int q = 0; q < 2; q++) {
      bar_init(q_full + q, 4);
      bar_init(mma_end + q, 1);
      bar_init(mma_end + 2 + q, 1);
      bar_init(&s_full[q][0], 1);
      bar_init(&s_full[q][1], 1);
      for (int i = 0; i < 2; i++) {  // (two: a warp may be one tile of keys ahead of another, or of O's update)
        bar_init(&p_full[q][i], 4);
        bar_init(&pv_done[q][i], 1);
      }
    }
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (C::SPILL) slot_s = pa.sums && n_tiles > C::FOLD ? claim_slot(Abort{&abort_s, pa.err}) : -1;
  }
  __syncwarp();
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const Abort ab{&abort_s, pa.err};
  const int fold = C::SPILL && slot_s < 0 ? n_tiles : C::FOLD;  // (at least n_tiles: never)

  if (warp >= 8 && warp < 16) {  // ---------------- converters: warps 8-11 for K, warps 12-15 for V
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    constexpr int CPR = HD / 16;             // 16-code pieces of a row
    constexpr int RPI = 128 / CPR;           // rows that 128 threads take at once
    constexpr int NI = PR_KEYS / RPI;
    const int which = (warp - 8) >> 2, tid = threadIdx.x & 127, piece = tid % CPR, row = tid / CPR;
    const size_t head_bytes = (size_t)HD << a.page_log;
    const int page_mask = (1 << a.page_log) - 1;
    const int* table = a.table + (size_t)at.r * a.table_cols;
    const int8_t* src = a.kv + ((size_t)which * a.kv_heads + head) * head_bytes + piece * 16;
    const size_t page_bytes = 2 * a.kv_heads * head_bytes;
    uint64_t* full = which ? v_full : k_full;
    uint64_t* empty = which ? v_empty : k_empty;
    uint8_t* tiles = sm + (which ? C::OFF_V : C::OFF_K) + (piece >> 2) * (PR_KEYS * 128);
    // a tile is read while the one before it is converted, its page numbers another tile before that
    uint4 raw[NI];
    int id[NI];
    auto pages_of = [&](int j) {
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int key = key_begin + j * PR_KEYS + row + RPI * i;
        id[i] = -1;  // past the last key: code 0
        if (j < n_tiles && (key & ~15) < hi) {
          const int pg = table[key >> a.page_log];
          id[i] = (unsigned)pg < (unsigned)a.n_pages ? pg : 0;
        }
      }
    };
    auto load = [&](int j) {
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int key = key_begin + j * PR_KEYS + row + RPI * i;
        raw[i] = make_uint4(0, 0, 0, 0);
        if (id[i] >= 0) raw[i] = *reinterpret_cast<const uint4*>(src + id[i] * page_bytes + (size_t)(key & page_mask) * HD);
      }
    };
    // (warp 12) the scales of the 16-key groups of PR_INFO tiles, the batch-th such. Its place held batch - 2: this is called
    // 16 tiles before the batch begins, and a tile of V is not converted before the softmax is done with the tile STG before
    auto publish_info = [&](int batch) {
      const int g0 = batch * PR_INFO * (PR_KEYS / 16);
      float sk[4], sv[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int key = key_begin + 16 * (g0 + lane + 32 * i);
        sk[i] = sv[i] = 0.f;
        if (key < min(hi, key_begin + n_tiles * PR_KEYS)) {
          int pg = table[key >> a.page_log];
          pg = (unsigned)pg < (unsigned)a.n_pages ? pg : 0;
          const float* s = a.kv_scale + (size_t)pg * 2 * a.kv_heads + head;
          sk[i] = s[0];
          sv[i] = s[a.kv_heads];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        KeyInfo ki;
        ki.k = sk[i];
        split_scale(sv[i], &ki.e, &ki.mant, &ki.inv);
        if (sizeof(T) == 2) {  // the whole scale goes into the exponent (its logarithm is off by 2^-22 of the result)
          const float mant = fmaxf(ki.mant, 1.f);  // (a scale below 2^-62, or 0, counts as 2^-62)
          ki.e += __log2f(mant);
          ki.inv = __fdividef(ki.inv, mant);
        }
        info[batch & 1][(lane + 32 * i) / (PR_KEYS / 16)][lane % (PR_KEYS / 16)] = ki;
      }
      __syncwarp();
      if (lane == 0) bar_arrive(i_full + (batch & 1));
    };
    if (n_tiles > 0) {
      pages_of(0);
      load(0);
      pages_of(1);
      if (warp == 12) publish_info(0);
    }
    for (int j = 0; j < n_tiles; j++) {
      const int s = j % STG;
      if (!wait_group(empty + s, ((j / STG) & 1) ^ 1, ab, PR_CONVERT, 1 + which, go[which], j)) break;
      if (warp == 12 && j % PR_INFO == PR_INFO - 16 && j + 16 < n_tiles) publish_info(j / PR_INFO + 1);
      uint8_t* tile = tiles + s * C::KV_TILE;
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t u = w[k] ^ 0x80808080u;
          h[2 * k] = half2_of(__byte_perm(u, 0x64646464u, 0x4140));
          h[2 * k + 1] = half2_of(__byte_perm(u, 0x64646464u, 0x4342));
        }
        const int rr = row + RPI * i, c = (piece & 3) * 2;
        *reinterpret_cast<uint4*>(tile + sw128(rr, c)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(tile + sw128(rr, c + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(full + s);
      if (j + 1 < n_tiles) {
        load(j + 1);
        pages_of(j + 2);
      }
    }
  } else if (warp >= 16) {  // ---------------- products
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const int q = (warp - 16) & 1, what = (warp - 16) >> 1;  // row tile; scores, or O's update
    if (q < n_q_tiles && lane == 0) {
      const uint32_t base = tmem + q * 256;
      if (what == 0) {
        const uint32_t id_s = (1u << 4) | ((uint32_t)(PR_KEYS >> 3) << 17) | (8u << 24);
        const uint64_t q_desc = desc_sw128(su32(sm + q * C::Q_AREA), 1024);
        const uint64_t k_desc = desc_sw128(su32(sm + C::OFF_K), 1024);
        if (n_tiles == 0 || wait_phase(q_full + q, 0, ab, PR_MMA))
          for (int j = 0; j < n_tiles; j++) {
            // the slot held the weights of tile j - 2
            const int s = j % STG;
            if (!wait_two(k_full + s, (j / STG) & 1, &pv_done[q][j & 1], ((j >> 1) & 1) ^ 1, ab, PR_MMA)) break;
            tc_fence_after();
            const uint64_t kd = k_desc + s * (C::KV_TILE >> 4);
#pragma unroll
            for (int t = C::Q_TERMS - 1; t >= 0; t--)  // (the small term first: the sum is small while it is added)
#pragma unroll
              for (int k = 0; k < HD / 16; k++)
                mma_f16(base + (j & 1) * PR_KEYS, q_desc + ((t * C::Q_TILE + (k >> 2) * (128 * 128) + (k & 3) * 32) >> 4),
                        kd + (((k >> 2) * (PR_KEYS * 128) + (k & 3) * 32) >> 4), id_s, t < C::Q_TERMS - 1 || k > 0);
            mma_commit(&s_full[q][j & 1]);
            mma_commit(k_empty + s);
          }
      } else {
        const uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);  // B in MN-major form
        // (V's blocks of 64 dimensions lie PR_KEYS rows apart)
        const uint64_t v_desc = desc_sw128(su32(sm + C::OFF_V), 1024) + ((uint64_t)(((PR_KEYS * 128) >> 4) - 1) << 16);
        int anew = 0;  // the tile with which O begins anew
        for (int j = 0; j < n_tiles; j++) {
          const int s = j % STG;
          const bool add = j != anew;
          if (!add) anew += fold;
          if (!wait_two(v_full + s, (j / STG) & 1, &p_full[q][j & 1], (j >> 1) & 1, ab, PR_MMA)) break;
          tc_fence_after();
          const uint64_t vd = v_desc + s * (C::KV_TILE >> 4);
#pragma unroll
          for (int t = 0; t < C::P_TERMS; t++)
#pragma unroll
            for (int k = 0; k < PR_KEYS / 16; k++)
              mma_f16_ts(base + 128, base + (j & 1) * PR_KEYS + t * (PR_KEYS / 2) + 8 * k, vd + k * (2048 >> 4), id_o,
                         add || t > 0 || k > 0);
          mma_commit(&pv_done[q][j & 1]);
          mma_commit(v_empty + s);
        }
      }
      mma_commit(mma_end + 2 * what + q);
      drain_phase(mma_end + 2 * what + q, 0);
    }
  } else if ((warp >> 2) < n_q_tiles) {  // ---------------- softmax: one thread, one row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
    const int q = warp >> 2, w4 = warp & 3;
    const int trow = 32 * w4 + lane, row = at.row0 + q * 128 + trow;
    const bool live = row < n_rows;
    const int rr = live ? row : n_rows - 1;  // (rows past the last compute on zeros and are not stored)
    int hq;
    const int tok = token_of(a, rr, &hq);
    hq += head * a.group;
    const int pos = R.len - n_all + tok, first_key = first_key_of(a, pos);
    bool ok = true;
    if (n_tiles > 0) {
      put_queries<T, HD>(a, (long long)(R.first + tok) * a.q_row + hq * a.q_head, n_rows, at.row0 + q * 128, 32 * w4,
                         sm + q * C::Q_AREA, row_scale + q * 128);
      if (lane == 0) bar_arrive(q_full + q);
    }
    const float f_row = n_tiles > 0 ? row_scale[q * 128 + trow] : 0.f;
    const uint32_t tl = tmem + ((uint32_t)(32 * w4) << 16) + q * 256, to = tl + 128;
    float m_run = -INFINITY, l_run = 0.f;
    float m_sum = -INFINITY;  // (spilled sums) the maximum that they are relative to
    auto sums = [&] { return pa.sums + (slot_s * 2 + q) * (128 * HD); };
    int anew = fold;
    auto add_up = [&](int j) {  // O to the sum so far: the product with the weights of tile j begins it anew
      anew += fold;
      if (!wait_phase_warp(&pv_done[q][(j - 1) & 1], ((j - 1) >> 1) & 1, ab, PR_SOFTMAX)) ok = false;
      tc_fence_after();
      if (C::SPILL) {
        spill_row(sums(), trow, to, m_sum == m_run ? 1.f : exp2_fast(m_sum - m_run), j == C::FOLD);
        m_sum = m_run;
      }
#pragma unroll 1
      for (int c = 0; c < (C::SPILL ? 0 : HD); c += 16) {
        uint32_t o[16], sum[16];
        tmem_ld16(to + c, o);
        tmem_ld16(to + HD + c, sum);  // (what lies there before the first time is not used)
        tc_wait_ld();
        if (j > C::FOLD) {
#pragma unroll
          for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) + __uint_as_float(sum[i]));
        }
        tmem_st16(to + HD + c, o);
      }
      tc_wait_st();
    };
    bool ready = false;
    for (int j = 0; j < n_tiles; j++) {
      if (C::FOLD % PR_INFO && j == anew) add_up(j);
      if (__builtin_expect(j % PR_INFO == 0, 0)) {
        if (C::FOLD % PR_INFO == 0 && j == anew) add_up(j);
        if (!wait_phase_warp(i_full + (j / PR_INFO & 1), (j / PR_INFO >> 1) & 1, ab, PR_SOFTMAX)) ok = false;
      }
      KeyInfo in[PR_KEYS / 16];
#pragma unroll
      for (int g = 0; g < PR_KEYS / 16; g++) {
        const float4 x = *reinterpret_cast<const float4*>(&info[j / PR_INFO & 1][j % PR_INFO][g]);
        in[g] = {x.x * f_row, x.y, x.z, x.w};
      }
      // (no way out of the loop when a wait expires: the other row tile's warp counts the turns; waits are short then)
      if (!ready && !wait_phase_warp(&s_full[q][j & 1], (j >> 1) & 1, ab, PR_SOFTMAX)) ok = false;
      tc_fence_after();
      float s[PR_KEYS];
      const uint32_t ts = tl + (j & 1) * PR_KEYS;
      tmem_ld32(ts, s);
      tmem_ld32(ts + 32, s + 32);
      tc_wait_ld();
      const int key0 = key_begin + j * PR_KEYS;
      const bool edge = __any_sync(0xffffffffu, key0 + PR_KEYS - 1 > pos || key0 < first_key);
      float mx;
      if (edge) mx = tile_max<true>(s, in, key0, first_key, pos);
      else mx = tile_max<false>(s, in, key0, first_key, pos);
      if (__any_sync(0xffffffffu, mx > m_run + M_SLACK)) {
        const float m_new = mx > m_run + M_SLACK ? mx : m_run;  // (a row's result does not depend on its neighbours)
        const float f_old = m_new == m_run ? 1.f : m_run == -INFINITY ? 0.f : exp2_fast(m_run - m_new);
        m_run = m_new;
        l_run *= f_old;
        if (j > 0) {
          if (!wait_phase_warp(&pv_done[q][(j - 1) & 1], ((j - 1) >> 1) & 1, ab, PR_SOFTMAX)) ok = false;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            float o[32];
            tmem_ld32(to + c, o);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] *= f_old;
            tmem_st32(to + c, reinterpret_cast<const uint32_t*>(o));
          }
          if (!C::SPILL && j >= C::FOLD) {
#pragma unroll 1
            for (int c = HD; c < 2 * HD; c += 32) {
              float o[32];
              tmem_ld32(to + c, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; i++) o[i] *= f_old;
              tmem_st32(to + c, reinterpret_cast<const uint32_t*>(o));
            }
          }
          tc_wait_st();
        }
      }
      const float base = P_SHIFT - (m_run == -INFINITY ? 0.f : m_run);
      uint32_t p[PR_KEYS / 2], rest[C::P_TERMS == 2 ? PR_KEYS / 2 : 1];
      // The two row tiles take turns at the exponentials (the two warps of a scheduler, which share its unit for them): each has
      // the other's turn for everything else. Both at once, they also do everything else at once.
      if (n_q_tiles == 2 && (q || j)) asm volatile("bar.sync %0, 64;" ::"r"(3 + 4 * q + w4) : "memory");
      if (edge) weights<C::P_TERMS, sizeof(T) == 4, true>(s, in, base, key0, first_key, pos, p, rest, &l_run);
      else weights<C::P_TERMS, sizeof(T) == 4, false>(s, in, base, key0, first_key, pos, p, rest, &l_run);
      if (n_q_tiles == 2 && (!q || j + 1 < n_tiles)) asm volatile("bar.arrive %0, 64;" ::"r"(7 - 4 * q + w4) : "memory");
      tmem_st32(ts, p);
      if (C::P_TERMS == 2) tmem_st32(ts + 32, rest);
      // (the next scores are most often there: their test is under way while the stores are)
      const bool next = bar_test(&s_full[q][(j + 1) & 1], ((j + 1) >> 1) & 1);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&p_full[q][j & 1]);
      ready = __all_sync(0xffffffffu, next);  // (which also brings the warp together for the next aligned instruction)
    }
    // ---- the rows' output: each thread stages its row in the place of the row tile's queries (their last product was issued
    // before the last update of O, whose completion is waited for; without keys they were not written) and copies it out
    if (ok && n_tiles > 0) {
      ok = wait_phase_warp(&pv_done[q][(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1, ab, PR_SOFTMAX);
      tc_fence_after();
    }
    if (ok) {
      const bool whole = sp.used == 1;
      const float inv = whole && l_run != 0.f ? 1.f / l_run : 1.f;
      const size_t unit = ((size_t)idx * a.kv_heads + head) * shape.splits + split;
      uint8_t* stage = sm + q * C::Q_AREA + trow * C::OUT_LD;
      const bool folded = n_tiles > fold;
      const uint32_t sum_at = folded && !C::SPILL ? to + HD : 0;
      float* spilled = folded && C::SPILL ? sums() : nullptr;
      const float f_sum = m_sum == m_run ? 1.f : exp2_fast(m_sum - m_run);
      if (whole) {
        constexpr int NC = 256 / (int)sizeof(T) < HD ? 256 / (int)sizeof(T) : HD;
        T* dst = static_cast<T*>(a.out) + (long long)(R.first + tok) * a.out_row + hq * a.out_head;
#pragma unroll 1
        for (int c = 0; c < HD; c += NC) {
          stage_row<T, NC>(stage, to + c, n_tiles > 0, inv, sum_at ? sum_at + c : 0, spilled, trow, c, f_sum);
          copy_row<T, NC>(dst + c, stage, live, a.out_vec16);
        }
      } else {
        float* dst = pa.part + (unit * PR_ROWS + q * 128 + trow) * HD;
#pragma unroll 1
        for (int c = 0; c < HD; c += 64) {
          stage_row<float, 64>(stage, to + c, n_tiles > 0, 1.f, sum_at ? sum_at + c : 0, spilled, trow, c, f_sum);
          copy_row<float, 64>(dst + c, stage, live, true);
        }
      }
      if (live) {
        if (!whole) pa.ml[unit * PR_ROWS + q * 128 + trow] = make_float2(m_run, l_run);
        else if (a.lse)
          a.lse[(size_t)(R.first + tok) * a.heads + hq] =
              l_run == 0.f ? -INFINITY : 0.69314718055994531f * (log2f(l_run) + m_run - P_SHIFT);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (C::SPILL && threadIdx.x == 0 && slot_s >= 0) release_slot(slot_s);
  if (warp == 16) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

}  // namespace
}  // namespace h2
