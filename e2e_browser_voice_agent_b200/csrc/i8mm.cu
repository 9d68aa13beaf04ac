// Matrix products in 8-bit integers with a scale for each token and each output channel (h2c_i8_quantize, h2c_i8_matmul;
// the formulas are stated in include/h2cuda.h): y[m][n] = (sum_k xq[m][k] w[n][k]) * x_scale[m] * w_scale[n] + bias[n].
//
// The sums are exact (int32 in TMEM), so neither the tile shape nor the division of K changes a result. A CTA computes
// D[128 or 256 weight rows][NT tokens] with tcgen05.mma kind::i8: weights are the M side, so that one instruction shape serves
// one token (NT = 16) and a prompt (NT up to 256), and a warp of the epilogue holds 32 consecutive outputs of a token.
// Tiles of 256 rows (two products per operand of tokens) are for prompts, where the operands' way from L2 is the bound: all SMs
// together read about 50 bytes a cycle each, and a 128 x 208 tile wants 103 a cycle at the tensor cores' rate.
//   warp 0     TMA loads of both operands, 128 bytes of K per stage, 128-byte swizzle
//   warp 1     tcgen05.mma, four per stage
//   warps 4-7  epilogue: TMEM -> registers -> scaled outputs; with tiles of 128 rows there are two in TMEM, so it overlaps the
//              next tile's products
// Few tiles (few tokens on a small matrix): a cluster of up to 8 CTAs divides K and adds its partial tiles through
// distributed shared memory, each CTA finishing a share of the tokens.
// The tokens are quantized by a kernel of their own; the product is launched with it (programmatic dependent launch) and
// has its weights under way before it waits for the codes. One or two tokens are quantized by every CTA for itself, its share
// of K into shared memory while the weights come: one launch.
// Bound and measured: 1 x 896 by 1152 rows, float32: latency, 5.9 us. 32 x 3584 by 37888, bfloat16: the weights' bytes, 33 us with
// the codes of the tokens (136 MB, 4.4 TB/s over the product's 31). 4099 x 18944 by 3584: 270 us with the codes, the product alone
// 227 (2,455 Top/s): the operands' way from L2. (In bursts of ten; in a run of seconds the power limit brings the SMs to 1,695 MHz,
// and it takes 301 us.)
// Waits for data are bounded (1 s): on expiry the CTA records it (h2c_ops_check), drains its copies and returns. The allocation of
// TMEM waits for the SM's other CTAs to free theirs, which they do at their end, whether their own waits expire or not.
#include "ops.cuh"
#include "tc5_ptx.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace h2 {
namespace {

constexpr int TN = 128;          // weight rows per product
constexpr int KCH = 128;         // bytes of K per stage
constexpr int FUSE_TOKENS = 2, FUSE_VALUES = 4096;  // bounds of the form that quantizes its tokens itself
constexpr int X_CHUNK = 16 * KCH;  // its codes of one stage of K: 16 rows
constexpr int MAX_STAGES = 12;
constexpr int SMEM_RING = 220 * 1024;
static_assert(FUSE_VALUES / KCH * X_CHUNK + 2 * TN * KCH <= SMEM_RING, "all of such a call's codes, and two stages of weights");
constexpr int MM_THREADS = 256;
enum { I8_PRODUCER = 11, I8_MMA = 12, I8_EPILOGUE = 13 };

// ---------------------------------------------------------------- quantize rows
//
// A CTA a row, read twice (the second time from L2), four loads ahead. Bound: bandwidth for many rows (4,099 x 18,944 bfloat16, 233
// MB: 54 us, 4.3 TB/s), latency for few (32 x 3,584: 2.4 us). Rows of more than 4,096 get 1,024 threads while there are too few to
// fill the SMs (32 x 18,944 with its product through 3,584 rows: 36.9 us, with 256 threads 39.1; 4,099 rows: 270 with 256, 289).

// A row's scale and what its values are multiplied by, from its largest magnitude's bits (magnitudes order as their bits do,
// infinities and NaN above every number: they make the scale NaN). 127 / a overflows for denormal rows, whose largest code is then
// below 127.
struct RowScale {
  float scale, inv;
};
__device__ __forceinline__ RowScale row_scale_of(unsigned m) {
  const float a = __uint_as_float(m);
  return {m >= 0x7f800000u ? __int_as_float(0x7fc00000) : __fdiv_rn(a, 127.f),
          a > 0.f ? fminf(__fdiv_rn(127.f, a), 3.4028234663852886e38f) : 0.f};
}

template <class T, bool VEC>
__global__ void __launch_bounds__(1024) k_i8_quantize(const T* __restrict__ x, long long x_row, int k, int8_t* __restrict__ q,
                                                      long long q_row, int k_pad, float* __restrict__ scale) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ unsigned red[32];
  const T* src = x + (long long)blockIdx.x * x_row;
  const int units = k >> 2, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned m = 0;
#pragma unroll 4
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    Raw4<T, VEC> v;
    v.load(src + 4 * u);
    m = v.merge(m);
  }
  m = Raw4<T, VEC>::bits(m);
  if ((int)threadIdx.x < (k & 3)) m = max(m, __float_as_uint(to_f(src[4 * units + threadIdx.x])) & 0x7fffffffu);
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = __reduce_max_sync(0xffffffffu, lane < (int)(blockDim.x >> 5) ? red[lane] : 0u);
  const RowScale rs = row_scale_of(m);
  const float inv = rs.inv;
  if (threadIdx.x == 0) scale[blockIdx.x] = rs.scale;
  uint32_t* dst = reinterpret_cast<uint32_t*>(q + (long long)blockIdx.x * q_row);
#pragma unroll 4
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    Raw4<T, VEC> r;
    float v[4];
    r.load(src + 4 * u);
    r.get(v);
    dst[u] = round_bytes(__fmul_rn(v[0], inv), __fmul_rn(v[1], inv), __fmul_rn(v[2], inv), __fmul_rn(v[3], inv));
  }
  for (int u = units + threadIdx.x; u < k_pad >> 2; u += blockDim.x) {  // the row's end, and zeros to 16 bytes
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = 4 * u + i < k ? to_f(src[4 * u + i]) : 0.f;
    dst[u] = round_bytes(__fmul_rn(v[0], inv), __fmul_rn(v[1], inv), __fmul_rn(v[2], inv), __fmul_rn(v[3], inv));
  }
}

// ---------------------------------------------------------------- the product

struct MmArgs {
  int n, m, chunks;          // outputs per token, tokens, stages of K
  int nt, mt, stages, splits;  // tokens per tile, products of 128 rows per tile, ring depth, CTAs that divide K (the cluster)
  int tiles_n, tiles_m;
  const float *xs, *ws, *bias;
  void* y;
  long long y_row;
  int* err;
  // tokens as values (the form that quantizes them itself)
  const void* x;
  long long x_row;
  int k, x_vec;
};

__device__ __forceinline__ void dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The codes of the CTA's share of K (chunks c0 .. c1) of all a.m <= FUSE_TOKENS tokens, as k_i8_quantize makes them, in the layout
// that a TMA load with 128-byte swizzle leaves: 16 rows, those past the last token zeros. By all threads.
template <class TX>
__device__ __forceinline__ void quantize_here(const MmArgs& a, int c0, int c1, uint8_t* x_sm, float* scale) {
  __shared__ unsigned red[FUSE_TOKENS][MM_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, units = a.k >> 2;
  for (int t = 0; t < a.m; t++) {
    const TX* src = static_cast<const TX*>(a.x) + t * a.x_row;
    unsigned m = 0;
    auto most = [&](auto vec) {
#pragma unroll 4
      for (int u = tid; u < units; u += MM_THREADS) {
        float v[4];
        load4<decltype(vec)::value>(src + 4 * u, v);
#pragma unroll
        for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
      }
    };
    if (a.x_vec) most(std::true_type());
    else most(std::false_type());
    if (tid < (a.k & 3)) m = max(m, __float_as_uint(to_f(src[4 * units + tid])) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) red[t][warp] = m;
  }
  const int chunks = c1 - c0, words = chunks * (KCH / 4);
  for (int i = tid; i < chunks * 16 * (KCH / 16); i += MM_THREADS)  // the rows past the last token
    if (((i >> 3) & 15) >= a.m) reinterpret_cast<uint4*>(x_sm)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  for (int t = 0; t < a.m; t++) {
    const TX* src = static_cast<const TX*>(a.x) + t * a.x_row;
    const RowScale rs = row_scale_of(__reduce_max_sync(0xffffffffu, red[t][lane & (MM_THREADS / 32 - 1)]));
    if (tid == 0) scale[t] = rs.scale;
#pragma unroll 2
    for (int w = tid; w < words; w += MM_THREADS) {
      const int k = c0 * KCH + 4 * w;
      uint32_t q = 0;
      if (k < a.k) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (a.x_vec && k + 4 <= a.k) load4<true>(src + k, v);
        else
          for (int i = 0; i < 4 && k + i < a.k; i++) v[i] = to_f(src[k + i]);
        q = round_bytes(__fmul_rn(v[0], rs.inv), __fmul_rn(v[1], rs.inv), __fmul_rn(v[2], rs.inv), __fmul_rn(v[3], rs.inv));
      }
      const int b = 4 * (w & 31);  // byte of the chunk's row
      *reinterpret_cast<uint32_t*>(x_sm + (w >> 5) * X_CHUNK + t * KCH + ((((b >> 4) ^ (t & 7)) << 4) | (b & 15))) = q;
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Tiles in groups of up to 8 token tiles: within a group the token tile changes fastest, so that the CTAs at work at one
// time share few weight rows and few token tiles, and both stay in L2.
__device__ __forceinline__ void tile_at(const MmArgs& a, int i, int* tn, int* tm) {
  const int per = 8 * a.tiles_n, grp = i / per, in = i - grp * per;
  const int wide = min(8, a.tiles_m - 8 * grp);
  *tn = in / wide;
  *tm = 8 * grp + in % wide;
}

template <class T>
__device__ __forceinline__ void put(const MmArgs& a, int tok, int row, int acc, float xs, float ws, float b) {
  const float v = (float)acc * xs * ws + b;
  static_cast<T*>(a.y)[(long long)tok * a.y_row + row] = from_f<T>(v);
}

// TX: the tokens' type in the form that quantizes them itself, else void.
template <class T, class TX>
__global__ void __launch_bounds__(MM_THREADS, 1)
    k_i8_matmul(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const MmArgs a) {
  constexpr bool FUSE = !std::is_void<TX>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (su32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t bars[2 * MAX_STAGES + 5];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_s;
  __shared__ float fused_scale[FUSE_TOKENS];
  uint64_t* full = bars;
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* tfull = empty + MAX_STAGES;  // a TMEM tile is complete
  uint64_t* tempty = tfull + 2;          // a TMEM tile has been read
  uint64_t* done = tempty + 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int w_bytes = a.mt * TN * KCH, stage_bytes = w_bytes + (FUSE ? 0 : a.nt * KCH);
  const int tile_cols = a.mt * a.nt, slots = a.mt == 1 ? 2 : 1;  // TMEM tiles
  int cols = 32;
  while (cols < slots * tile_cols) cols *= 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; s++) {
      bar_init(full + s, 1);
      bar_init(empty + s, 1);
    }
    for (int t = 0; t < 2; t++) {
      bar_init(tfull + t, 1);
      bar_init(tempty + t, 4);
    }
    bar_init(done, 1);
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&tmem_slot)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int rank = blockIdx.x % a.splits, first = blockIdx.x / a.splits, step = gridDim.x / a.splits;
  const int n_tiles = a.tiles_n * a.tiles_m;
  const int c0 = (int)((long long)a.chunks * rank / a.splits), c1 = (int)((long long)a.chunks * (rank + 1) / a.splits);
  uint8_t* x_sm = sm + a.stages * stage_bytes;  // (FUSE) [chunk][16 tokens][128 bytes, swizzled]
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const Abort ab{&abort_s, a.err};

  // the weights of the first stages do not wait for the codes
  const int early = first < n_tiles ? min(a.stages, c1 - c0) : 0;
  if (threadIdx.x == 0 && early) {
    int tn, tm;
    tile_at(a, first, &tn, &tm);
    for (int s = 0; s < early; s++) {
      bar_expect(full + s, stage_bytes);
      tma2d(sm + s * stage_bytes, &tm_w, (c0 + s) * KCH, tn * a.mt * TN, full + s);
    }
  }
  __syncwarp();
  if constexpr (FUSE) {
    quantize_here<TX>(a, c0, c1, x_sm, fused_scale);
    __syncthreads();
  }

  if (warp == 0) {
    if (lane == 0) {  // ---------------- loads
      uint32_t issued = 0;
      dep_wait();
      for (int tile = first; tile < n_tiles; tile += step) {
        int tn, tm;
        tile_at(a, tile, &tn, &tm);
        for (int c = c0; c < c1; c++, issued++) {
          const int s = issued % a.stages;
          uint8_t* stg = sm + s * stage_bytes;
          if ((int)issued >= early) {
            if (!wait_phase(empty + s, ((issued / a.stages) & 1) ^ 1, ab, I8_PRODUCER)) goto loads_done;
            bar_expect(full + s, stage_bytes);
            tma2d(stg, &tm_w, c * KCH, tn * a.mt * TN, full + s);
          }
          if (!FUSE) tma2d(stg + w_bytes, &tm_x, c * KCH, tm * a.nt, full + s);
        }
      }
    loads_done:
      for (uint32_t k = issued > (uint32_t)a.stages ? issued - a.stages : 0; k < issued; k++)
        drain_phase(full + k % a.stages, (k / a.stages) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {  // ---------------- products
      const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(a.nt >> 3) << 17) | (8u << 24);
      uint32_t ci = 0, ti = 0;
      for (int tile = first; tile < n_tiles; tile += step, ti++) {
        const int t = slots == 2 ? ti & 1 : 0;
        if (!wait_phase(tempty + t, ((slots == 2 ? ti >> 1 : ti) & 1) ^ 1, ab, I8_MMA)) goto mma_done;
        tc_fence_after();
        for (int c = c0; c < c1; c++, ci++) {
          const int s = ci % a.stages;
          if (!wait_phase(full + s, (ci / a.stages) & 1, ab, I8_MMA)) goto mma_done;
          tc_fence_after();
          const uint32_t wb = su32(sm + s * stage_bytes), xb = FUSE ? su32(x_sm) + (c - c0) * X_CHUNK : wb + w_bytes;
          for (int h = 0; h < a.mt; h++)
#pragma unroll
            for (int j = 0; j < KCH / 32; j++)
              mma_i8(tmem + t * tile_cols + h * a.nt, desc_sw128(wb + h * (TN * KCH) + 32 * j, 1024),
                     desc_sw128(xb + 32 * j, 1024), idesc, c > c0 || j > 0);
          mma_commit(empty + s);
        }
        mma_commit(tfull + t);
      }
    mma_done:
      mma_commit(done);
      drain_phase(done, 0);
    }
  } else if (warp >= 4 && a.splits == 1) {  // ---------------- epilogue
    dep_wait();
    const int q = warp & 3;
    uint32_t ti = 0;
    for (int tile = first; tile < n_tiles; tile += step, ti++) {
      const int t = slots == 2 ? ti & 1 : 0;
      int tn, tm;
      tile_at(a, tile, &tn, &tm);
      const int tok0 = tm * a.nt;
      if (!wait_phase_warp(tfull + t, (slots == 2 ? ti >> 1 : ti) & 1, ab, I8_EPILOGUE)) break;
      tc_fence_after();
      for (int h = 0; h < a.mt; h++) {
        const int row = (tn * a.mt + h) * TN + 32 * q + lane;
        const float ws = row < a.n ? a.ws[row] : 0.f, b = a.bias && row < a.n ? a.bias[row] : 0.f;
        const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16) + t * tile_cols + h * a.nt;
        for (int c = 0; c < a.nt; c += 16) {
          if (tok0 + c >= a.m) break;
          uint32_t u[16];
          tmem_ld16(tl + c, u);
          tc_wait_ld();
          if (row < a.n) {
            if (!FUSE && tok0 + c + 16 <= a.m) {  // (without bounds inside: the stores need nothing but a moving address)
              const float* xs = a.xs + tok0 + c;
              T* y = static_cast<T*>(a.y) + (tok0 + c) * a.y_row + row;
#pragma unroll
              for (int i = 0; i < 16; i++, y += a.y_row) *y = from_f<T>((float)(int)u[i] * xs[i] * ws + b);
            } else {
#pragma unroll
              for (int i = 0; i < 16; i++)
                if (tok0 + c + i < a.m)
                  put<T>(a, tok0 + c + i, row, (int)u[i], FUSE ? fused_scale[i & (FUSE_TOKENS - 1)] : a.xs[tok0 + c + i], ws, b);
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(tempty + t);
    }
  }
  __syncwarp();
  if (a.splits > 1) {  // ---------------- one tile per cluster: partial tiles through distributed shared memory
    int* part = reinterpret_cast<int*>(sm);  // [nt][128] (the ring is idle: the tile's products are done)
    int tn, tm;
    tile_at(a, first, &tn, &tm);
    const int tok0 = tm * a.nt, live = min(a.nt, a.m - tok0);
    if (warp >= 4) {
      const int q = warp & 3;
      if (wait_phase_warp(tfull, 0, ab, I8_EPILOGUE)) {
        tc_fence_after();
        for (int c = 0; c < live; c += 16) {
          uint32_t u[16];
          tmem_ld16(tmem + ((uint32_t)(32 * q) << 16) + c, u);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i++) part[(c + i) * TN + 32 * q + lane] = (int)u[i];
        }
        tc_fence_before();
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    dep_wait();
    const int row = tn * TN + (threadIdx.x & (TN - 1));
    const float ws = row < a.n ? a.ws[row] : 0.f, b = a.bias && row < a.n ? a.bias[row] : 0.f;
    for (int c = rank + a.splits * (threadIdx.x / TN); c < live; c += a.splits * (MM_THREADS / TN)) {
      const uint32_t at = su32(part + c * TN + (threadIdx.x & (TN - 1)));
      int acc = 0;
      for (int k = 0; k < a.splits; k++) {
        uint32_t remote;
        int v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(k));
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
        acc += v;
      }
      if (row < a.n) put<T>(a, tok0 + c, row, acc, FUSE ? fused_scale[c & (FUSE_TOKENS - 1)] : a.xs[tok0 + c], ws, b);
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
  }
}

// ---------------------------------------------------------------- host

bool u8_map(CUtensorMap* out, const void* ptr, uint64_t inner, uint64_t rows, uint64_t stride, uint32_t box_rows) {
  auto fn = tma_encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {inner, rows}, strides[1] = {stride};
  const cuuint32_t box[2] = {KCH, box_rows}, estr[2] = {1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tokens and 128-row products per tile, CTAs that divide K. With few tokens one tile holds them all. With many, the tile that makes
// the least of (waves of tiles over the 148 SMs) x (time of a tile): a stage takes 2 cycles of the tensor cores per token and
// product, and its bytes at 50 a cycle from L2; a tile takes about 1,500 cycles around its stages, and its outputs at 80 cycles a
// token and product where no second TMEM tile lets that overlap (256 tokens through 37888 x 3584: tiles of 128 rows 50 us, of 256
// rows 60; 4099 through 3584 x 18944: 317 and 277).
void shape_of(int m, int n, int chunks, int* nt, int* mt, int* splits) {
  long long best = LLONG_MAX;
  for (int h = 1; h <= 2; h++)
    for (int w = 16; w <= 256; w += 16) {
      const int tn = (n + h * TN - 1) / (h * TN), tm = (m + w - 1) / w;
      if (w > 16 && tm == (m + w - 17) / (w - 16)) continue;  // a narrower tile gives as many
      const long long waves = ((long long)tn * tm + 147) / 148;
      const long long stage = std::max(2 * w * h, (h * TN + w) * KCH / 50);
      const long long t = waves * (chunks * stage + 1500 + (h == 2 ? 80 * h * w : 0)) + (h == 1 ? 80 * w : 0);
      if (t < best) best = t, *nt = w, *mt = h;
    }
  const int tiles = (n + *mt * TN - 1) / (*mt * TN) * ((m + *nt - 1) / *nt);
  *splits = *mt > 1 ? 1 : std::max(1, std::min(std::min(8, chunks), 148 / tiles));
}

// Whether the product quantizes its tokens itself: few of them, and a CTA's share of K small enough for shared memory. Through
// 1152 x 896, bfloat16, in us on the device and per call: one token 5.8 and 15.7 (two launches: 6.2 and 19.5), two 6.4 and 14.6 (6.2
// and 17.2), four 7.6 (6.2).
bool fused(int x_type, int m, int k) { return x_type != H2C_TYPE_I8 && m <= FUSE_TOKENS && (long long)m * k <= FUSE_VALUES; }

template <class T>
int launch_quantize(const char* who, const void* x, long long x_row, int rows, int k, void* q, long long q_row, int k_pad,
                    float* scale, bool vec, cudaStream_t st) {
  const int threads = k > 4096 && rows < 592 ? 1024 : 256;
  const T* p = static_cast<const T*>(x);
  if (vec) k_i8_quantize<T, true><<<rows, threads, 0, st>>>(p, x_row, k, static_cast<int8_t*>(q), q_row, k_pad, scale);
  else k_i8_quantize<T, false><<<rows, threads, 0, st>>>(p, x_row, k, static_cast<int8_t*>(q), q_row, k_pad, scale);
  return op_launched(who);
}

int quantize(const char* who, int type, const void* x, long long x_row, int rows, int k, void* q, long long q_row,
             float* scale, cudaStream_t st) {
  const size_t es = op_elem_size(type);
  const bool vec = !((uintptr_t)x & (4 * es - 1)) && !(x_row & 3);
  const int k_pad = (k + 15) / 16 * 16;
  if (type == H2C_TYPE_F32) return launch_quantize<float>(who, x, x_row, rows, k, q, q_row, k_pad, scale, vec, st);
  if (type == H2C_TYPE_F16) return launch_quantize<__half>(who, x, x_row, rows, k, q, q_row, k_pad, scale, vec, st);
  return launch_quantize<__nv_bfloat16>(who, x, x_row, rows, k, q, q_row, k_pad, scale, vec, st);
}

template <class T, class TX>
int launch_matmul(const char* who, const CUtensorMap& tw, const CUtensorMap& tx, const MmArgs& a, bool dependent,
                  cudaStream_t st) {
  static unsigned char done[OP_MAX_DEVICES];
  constexpr int smem = SMEM_RING + 1024;
  if (int rc = op_once(who, done, [] {
        return cudaFuncSetAttribute(k_i8_matmul<T, TX>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      }))
    return rc;
  const int tiles = a.tiles_n * a.tiles_m;
  const bool fuse = !std::is_void<TX>::value;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.splits > 1 ? tiles * a.splits : std::min(tiles, 148));
  cfg.blockDim = dim3(MM_THREADS);
  cfg.dynamicSmemBytes = a.stages * (a.mt * TN * KCH + (fuse ? 0 : a.nt * KCH)) + 1024 +
                         (fuse ? (a.chunks + a.splits - 1) / a.splits * X_CHUNK : 0);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (a.splits > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim = {(unsigned)a.splits, 1, 1};
    na++;
  }
  if (dependent) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    na++;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  const cudaError_t c = cudaLaunchKernelEx(&cfg, k_i8_matmul<T, TX>, tw, tx, a);
  if (c != cudaSuccess) {
    cudaGetLastError();
    return op_error(H2C_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(c));
  }
  return H2C_OK;
}

template <class T>
int launch_matmul_of(const char* who, int x_type, bool fuse, const CUtensorMap& tw, const CUtensorMap& tx, const MmArgs& a,
                     cudaStream_t st) {
  if (!fuse) return launch_matmul<T, void>(who, tw, tx, a, x_type != H2C_TYPE_I8, st);
  if (x_type == H2C_TYPE_F32) return launch_matmul<T, float>(who, tw, tx, a, false, st);
  if (x_type == H2C_TYPE_F16) return launch_matmul<T, __half>(who, tw, tx, a, false, st);
  return launch_matmul<T, __nv_bfloat16>(who, tw, tx, a, false, st);
}

uint64_t codes_bytes(int m, int k) { return ((uint64_t)m * ((k + 15) / 16 * 16) + 255) / 256 * 256; }

}  // namespace
}  // namespace h2

using namespace h2;

extern "C" {

int h2c_i8_quantize(int32_t type, const void* x, int64_t x_row, int32_t rows, int32_t k, void* q, int64_t q_row,
                    float* scale, void* stream) {
  const char* who = "h2c_i8_quantize";
  if (!op_type_ok(type)) return op_error(H2C_ERR_BAD_TYPE, "%s: element type %d", who, type);
  if (rows < 0 || rows > OP_MAX_ROWS || k < 1 || k > H2C_I8_MAX_K) return op_error(H2C_ERR_INVALID, "%s: %d rows of %d", who, rows, k);
  if (rows == 0) return H2C_OK;
  if (!x || !q || !scale) return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  if ((uintptr_t)x & (op_elem_size(type) - 1)) return op_error(H2C_ERR_INVALID, "%s: x must be aligned to its elements", who);
  if (((uintptr_t)q & 15) || (q_row & 15) || q_row < k)
    return op_error(H2C_ERR_INVALID, "%s: q must be 16-byte aligned with rows of a multiple of 16 bytes, at least k", who);
  const int64_t es = (int64_t)op_elem_size(type), k_pad = (k + 15) / 16 * 16;
  const OpRows values{x, rows, x_row * es, k * es}, codes{q, rows, q_row, k_pad};
  const OpRange in = op_range("x", values), out[] = {op_range("q", codes), {"scale", scale, 4ull * rows, 4}};
  if (op_rows_meet(values, codes)) return op_error(H2C_ERR_INVALID, "%s: q must not share memory with x", who);
  if (int rc = op_check_ranges(who, out, 2, &in, 0)) return rc;
  if (int rc = op_check_ranges(who, out + 1, 1, &in, 1)) return rc;
  return quantize(who, type, x, x_row, rows, k, q, q_row, scale, (cudaStream_t)stream);
}

uint64_t h2c_i8_matmul_workspace(int32_t x_type, int32_t m, int32_t k) {
  if (m <= 0 || k <= 0 || x_type == H2C_TYPE_I8) return 0;
  return codes_bytes(m, k) + ((uint64_t)m * 4 + 255) / 256 * 256;
}

int h2c_i8_matmul(int32_t x_type, const void* x, int64_t x_row, const float* x_scale, const void* w, int64_t w_row,
                  const float* w_scale, int32_t m, int32_t n, int32_t k, int32_t y_type, void* y, int64_t y_row,
                  const float* bias, void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* who = "h2c_i8_matmul";
  const bool codes = x_type == H2C_TYPE_I8;
  if (!codes && !op_type_ok(x_type)) return op_error(H2C_ERR_BAD_TYPE, "%s: element type %d of x", who, x_type);
  if (!op_type_ok(y_type)) return op_error(H2C_ERR_BAD_TYPE, "%s: element type %d of y", who, y_type);
  if (m < 0 || n < 0 || m > OP_MAX_ROWS || n > OP_MAX_ROWS || k < 1 || k > H2C_I8_MAX_K)
    return op_error(H2C_ERR_INVALID, "%s: sizes m %d, n %d, k %d (k is 1 to %d)", who, m, n, k, H2C_I8_MAX_K);
  if (m == 0 || n == 0) return H2C_OK;
  if (!x || !w || !w_scale || !y || (codes && !x_scale)) return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  if (((uintptr_t)w & 15) || (w_row & 15) || w_row < k)
    return op_error(H2C_ERR_INVALID, "%s: w must be 16-byte aligned with rows of a multiple of 16 bytes, at least k", who);
  if (codes && (((uintptr_t)x & 15) || (x_row & 15) || x_row < k))
    return op_error(H2C_ERR_INVALID, "%s: codes must be 16-byte aligned with rows of a multiple of 16 bytes, at least k", who);
  if (!codes && ((uintptr_t)x & (op_elem_size(x_type) - 1)))
    return op_error(H2C_ERR_INVALID, "%s: x must be aligned to its elements", who);
  if ((uintptr_t)y & (op_elem_size(y_type) - 1))
    return op_error(H2C_ERR_INVALID, "%s: y must be aligned to its elements", who);
  const uint64_t need = h2c_i8_matmul_workspace(x_type, m, k);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
    return op_error(H2C_ERR_INVALID, "%s: needs %llu bytes of 16-byte aligned workspace, got %llu", who,
                    (unsigned long long)need, (unsigned long long)(workspace ? workspace_bytes : 0));
  const int64_t es = codes ? 1 : (int64_t)op_elem_size(x_type), ys = (int64_t)op_elem_size(y_type);
  if (m > 1 && (y_row < 0 ? -y_row : y_row) < n)
    return op_error(H2C_ERR_INVALID, "%s: rows of y overlap (%lld elements apart, %d long)", who, (long long)y_row, n);
  const OpRows tokens{x, m, x_row * es, k * es}, out{y, m, y_row * ys, n * ys};
  {
    const OpRange in[] = {{"w", w, (uint64_t)(n - 1) * w_row + k}, {"w_scale", w_scale, 4ull * n, 4}, {"bias", bias, bias ? 4ull * n : 0, 4},
                          {"x_scale", x_scale, codes ? 4ull * m : 0, 4}};
    const OpRange written[] = {op_range("y", out), {"workspace", workspace, need}};
    if (int rc = op_check_ranges(who, written, 2, in, 4)) return rc;
    const OpRange x_range = op_range("x", tokens);
    if (int rc = op_check_ranges(who, written + 1, 1, &x_range, 1)) return rc;
    if (codes && op_rows_meet(tokens, out)) return op_error(H2C_ERR_INVALID, "%s: y must not share memory with the codes x", who);
  }
  cudaStream_t st = (cudaStream_t)stream;
  MmArgs a = {};
  a.err = op_err_words();
  if (!a.err) return op_error(H2C_ERR_CUDA, "%s: no device", who);
  a.n = n; a.m = m; a.k = k; a.chunks = (k + KCH - 1) / KCH;
  shape_of(m, n, a.chunks, &a.nt, &a.mt, &a.splits);
  // (a CTA of that form may write its outputs while another still reads the tokens, so y in their memory takes two kernels)
  const bool fuse = fused(x_type, m, k) && !op_rows_meet(tokens, out);
  if (fuse) {  // (one tile of 16 tokens)
    a.nt = 16;
    a.mt = 1;
  }
  const int x_smem = fuse ? (a.chunks + a.splits - 1) / a.splits * X_CHUNK : 0;
  const int stage_bytes = a.mt * TN * KCH + (fuse ? 0 : a.nt * KCH);
  a.stages = std::min(MAX_STAGES, (SMEM_RING - x_smem) / stage_bytes);
  if (a.splits > 1)  // as deep as a CTA's share of K, and room for its partial tile
    a.stages = std::max(std::min(a.stages, (a.chunks + a.splits - 1) / a.splits),
                        (a.nt * TN * 4 + stage_bytes - 1) / stage_bytes);
  a.tiles_n = (n + a.mt * TN - 1) / (a.mt * TN); a.tiles_m = (m + a.nt - 1) / a.nt;
  if ((long long)a.tiles_n * a.tiles_m > INT_MAX / 16) return op_error(H2C_ERR_INVALID, "%s: too many outputs", who);
  a.ws = w_scale; a.bias = bias; a.y = y; a.y_row = y_row;
  const int k_pad = (k + 15) / 16 * 16;
  CUtensorMap tw, tx;
  const void* xq = codes ? x : workspace;
  a.xs = codes ? x_scale : reinterpret_cast<const float*>(static_cast<const uint8_t*>(workspace) + codes_bytes(m, k));
  if (fuse) {
    a.x = x;
    a.x_row = x_row;
    a.x_vec = !((uintptr_t)x & (4 * op_elem_size(x_type) - 1)) && !(x_row & 3);
  }
  if (!u8_map(&tw, w, k, n, w_row, a.mt * TN) || (!fuse && !u8_map(&tx, xq, k, m, codes ? x_row : k_pad, a.nt)))
    return op_error(H2C_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed", who);
  if (fuse) tx = tw;  // (not used)
  if (!codes && !fuse)
    if (int rc = quantize(who, x_type, x, x_row, m, k, workspace, k_pad, const_cast<float*>(a.xs), st)) return rc;
  if (y_type == H2C_TYPE_F32) return launch_matmul_of<float>(who, x_type, fuse, tw, tx, a, st);
  if (y_type == H2C_TYPE_F16) return launch_matmul_of<__half>(who, x_type, fuse, tw, tx, a, st);
  return launch_matmul_of<__nv_bfloat16>(who, x_type, fuse, tw, tx, a, st);
}

}  // extern "C"
