// Matrix products in 8-bit integers with a scale for each token and each output channel (h2c_i8_quantize, h2c_i8_matmul;
// the formulas are stated in include/h2cuda.h): y[m][n] = (sum_k xq[m][k] w[n][k]) * x_scale[m] * w_scale[n] + bias[n].
//
// The sums are exact (int32 in TMEM), so neither the tile shape nor the division of K changes a result. A CTA computes
// D[128 weight rows][NT tokens] with tcgen05.mma kind::i8: weights are the M side, so that one instruction shape serves
// one token (NT = 16) and a prompt (NT up to 256), and a warp of the epilogue holds 32 consecutive outputs of a token.
//   warp 0     TMA loads of both operands, 128 bytes of K per stage, 128-byte swizzle
//   warp 1     tcgen05.mma, four per stage
//   warps 4-7  epilogue: TMEM -> registers -> scaled outputs; two TMEM tiles, so it overlaps the next tile's products
// Few tiles (few tokens on a small matrix): a cluster of up to 8 CTAs divides K and adds its partial tiles through
// distributed shared memory, each CTA finishing a share of the tokens.
// The tokens are quantized by a kernel of their own; the product is launched with it (programmatic dependent launch) and
// has its weights under way before it waits for the codes.
// Waits are bounded (1 s): on expiry the CTA records it (h2c_ops_check), drains its copies and returns.
#include "ops.cuh"
#include "tc5_ptx.cuh"

#include <algorithm>
#include <climits>

namespace h2 {
namespace {

constexpr int TN = 128;          // weight rows per tile
constexpr int KCH = 128;         // bytes of K per stage
constexpr int W_STAGE = TN * KCH;
constexpr int MAX_STAGES = 12;
constexpr int SMEM_RING = 220 * 1024;
constexpr int MM_THREADS = 256;
enum { I8_PRODUCER = 11, I8_MMA = 12, I8_EPILOGUE = 13 };

// ---------------------------------------------------------------- quantize rows

template <class T, bool VEC>
__global__ void __launch_bounds__(1024) k_i8_quantize(const T* __restrict__ x, long long x_row, int k, int8_t* __restrict__ q,
                                                      long long q_row, int k_pad, float* __restrict__ scale) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ unsigned red[32];
  const T* src = x + (long long)blockIdx.x * x_row;
  const int units = k >> 2, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned m = 0;  // magnitudes order as their bits do
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    float v[4];
    load4<VEC>(src + 4 * u, v);
#pragma unroll
    for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  if ((int)threadIdx.x < (k & 3)) m = max(m, __float_as_uint(to_f(src[4 * units + threadIdx.x])) & 0x7fffffffu);
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = __reduce_max_sync(0xffffffffu, lane < (int)(blockDim.x >> 5) ? red[lane] : 0u);
  const float a = __uint_as_float(m);
  // 127 / a overflows for denormal rows, whose largest code is then below 127; infinities and NaN make the scale NaN
  const float inv = a > 0.f ? fminf(__fdiv_rn(127.f, a), 3.4028234663852886e38f) : 0.f;
  if (threadIdx.x == 0) scale[blockIdx.x] = m >= 0x7f800000u ? __int_as_float(0x7fc00000) : __fdiv_rn(a, 127.f);
  uint32_t* dst = reinterpret_cast<uint32_t*>(q + (long long)blockIdx.x * q_row);
  for (int u = threadIdx.x; u < k_pad >> 2; u += blockDim.x) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (u < units) {
      load4<VEC>(src + 4 * u, v);
    } else {
      for (int i = 0; i < 4; i++)
        if (4 * u + i < k) v[i] = to_f(src[4 * u + i]);
    }
    dst[u] = round_bytes(__fmul_rn(v[0], inv), __fmul_rn(v[1], inv), __fmul_rn(v[2], inv), __fmul_rn(v[3], inv));
  }
}

// ---------------------------------------------------------------- the product

struct MmArgs {
  int n, m, chunks;          // outputs per token, tokens, stages of K
  int nt, stages, splits;    // tokens per tile, ring depth, CTAs that divide K (the cluster)
  int tiles_n, tiles_m;
  const float *xs, *ws, *bias;
  void* y;
  long long y_row;
  int* err;
};

__device__ __forceinline__ void dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Tiles in groups of up to 8 token tiles: within a group the token tile changes fastest, so that the CTAs at work at one
// time share few weight rows and few token tiles, and both stay in L2.
__device__ __forceinline__ void tile_at(const MmArgs& a, int i, int* tn, int* tm) {
  const int per = 8 * a.tiles_n, grp = i / per, in = i - grp * per;
  const int wide = min(8, a.tiles_m - 8 * grp);
  *tn = in / wide;
  *tm = 8 * grp + in % wide;
}

template <class T>
__device__ __forceinline__ void put(const MmArgs& a, int tok, int row, int acc, float ws, float b) {
  const float v = (float)acc * a.xs[tok] * ws + b;
  static_cast<T*>(a.y)[(long long)tok * a.y_row + row] = from_f<T>(v);
}

template <class T>
__global__ void __launch_bounds__(MM_THREADS, 1)
    k_i8_matmul(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const MmArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (su32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t bars[2 * MAX_STAGES + 5];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_s;
  uint64_t* full = bars;
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* tfull = empty + MAX_STAGES;  // a TMEM tile is complete
  uint64_t* tempty = tfull + 2;          // a TMEM tile has been read
  uint64_t* done = tempty + 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stage_bytes = W_STAGE + a.nt * KCH;
  int cols = 32;
  while (cols < 2 * a.nt) cols *= 2;

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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const Abort ab{&abort_s, a.err};
  const int rank = blockIdx.x % a.splits, first = blockIdx.x / a.splits, step = gridDim.x / a.splits;
  const int n_tiles = a.tiles_n * a.tiles_m;
  const int c0 = (int)((long long)a.chunks * rank / a.splits), c1 = (int)((long long)a.chunks * (rank + 1) / a.splits);

  if (warp == 0) {
    if (lane == 0) {  // ---------------- loads
      int tn = 0, tm = 0;
      uint32_t issued = 0;
      // the weights of the first stages do not wait for the codes
      int early = 0;
      if (first < n_tiles) {
        tile_at(a, first, &tn, &tm);
        early = min(a.stages, c1 - c0);
        for (int s = 0; s < early; s++) {
          bar_expect(full + s, stage_bytes);
          tma2d(sm + s * stage_bytes, &tm_w, (c0 + s) * KCH, tn * TN, full + s);
        }
      }
      dep_wait();
      for (int tile = first; tile < n_tiles; tile += step) {
        tile_at(a, tile, &tn, &tm);
        for (int c = c0; c < c1; c++, issued++) {
          const int s = issued % a.stages;
          uint8_t* stg = sm + s * stage_bytes;
          if ((int)issued >= early) {
            if (!wait_phase(empty + s, ((issued / a.stages) & 1) ^ 1, ab, I8_PRODUCER)) goto loads_done;
            bar_expect(full + s, stage_bytes);
            tma2d(stg, &tm_w, c * KCH, tn * TN, full + s);
          }
          tma2d(stg + W_STAGE, &tm_x, c * KCH, tm * a.nt, full + s);
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
        const int t = ti & 1;
        if (!wait_phase(tempty + t, ((ti >> 1) & 1) ^ 1, ab, I8_MMA)) goto mma_done;
        tc_fence_after();
        for (int c = c0; c < c1; c++, ci++) {
          const int s = ci % a.stages;
          if (!wait_phase(full + s, (ci / a.stages) & 1, ab, I8_MMA)) goto mma_done;
          tc_fence_after();
          const uint32_t wb = su32(sm + s * stage_bytes), xb = wb + W_STAGE;
#pragma unroll
          for (int j = 0; j < KCH / 32; j++)
            mma_i8(tmem + t * a.nt, desc_sw128(wb + 32 * j, 1024), desc_sw128(xb + 32 * j, 1024), idesc,
                   c > c0 || j > 0);
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
      const int t = ti & 1;
      int tn, tm;
      tile_at(a, tile, &tn, &tm);
      const int row = tn * TN + 32 * q + lane, tok0 = tm * a.nt;
      const float ws = row < a.n ? a.ws[row] : 0.f, b = a.bias && row < a.n ? a.bias[row] : 0.f;
      if (!wait_phase_warp(tfull + t, (ti >> 1) & 1, ab, I8_EPILOGUE)) break;
      tc_fence_after();
      const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16) + t * a.nt;
      for (int c = 0; c < a.nt; c += 16) {
        if (tok0 + c >= a.m) break;
        uint32_t u[16];
        tmem_ld16(tl + c, u);
        tc_wait_ld();
        if (row < a.n) {
#pragma unroll
          for (int i = 0; i < 16; i++)
            if (tok0 + c + i < a.m) put<T>(a, tok0 + c + i, row, (int)u[i], ws, b);
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
      if (row < a.n) put<T>(a, tok0 + c, row, acc, ws, b);
    }
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

// Tokens per tile, CTAs that divide K. With few tokens one tile holds them all. With many, the tile that makes the least
// of (waves of tiles over the 148 SMs) x (time of a tile): a stage takes 2 NT cycles of the tensor cores and at least
// (128 + NT) cycles of shared-memory reads (128 bytes a cycle), and a tile about 1,500 cycles around its stages.
void shape_of(int m, int n, int chunks, int* nt, int* splits) {
  const int tiles_n = (n + TN - 1) / TN;
  long long best = LLONG_MAX;
  for (int w = 16; w <= 256; w += 16) {
    const int tm = (m + w - 1) / w;
    if (w > 16 && tm == (m + w - 17) / (w - 16)) continue;  // a narrower tile gives as many
    const long long waves = ((long long)tiles_n * tm + 147) / 148;
    const long long t = waves * ((long long)chunks * std::max(2 * w, TN + w) + 1500);
    if (t < best) best = t, *nt = w;
  }
  const int tiles = tiles_n * ((m + *nt - 1) / *nt);
  *splits = std::max(1, std::min(std::min(8, chunks), 148 / tiles));
}

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

template <class T>
int launch_matmul(const char* who, const CUtensorMap& tw, const CUtensorMap& tx, const MmArgs& a, bool dependent,
                  cudaStream_t st) {
  static unsigned char done[OP_MAX_DEVICES];
  constexpr int smem = SMEM_RING + 1024;
  if (int rc = op_once(who, done, [] {
        return cudaFuncSetAttribute(k_i8_matmul<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      }))
    return rc;
  const int tiles = a.tiles_n * a.tiles_m;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.splits > 1 ? tiles * a.splits : std::min(tiles, 148));
  cfg.blockDim = dim3(MM_THREADS);
  cfg.dynamicSmemBytes = a.stages * (W_STAGE + a.nt * KCH) + 1024;
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
  const cudaError_t c = cudaLaunchKernelEx(&cfg, k_i8_matmul<T>, tw, tx, a);
  if (c != cudaSuccess) {
    cudaGetLastError();
    return op_error(H2C_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(c));
  }
  return H2C_OK;
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
  if (rows < 0 || k < 1 || k > H2C_I8_MAX_K) return op_error(H2C_ERR_INVALID, "%s: %d rows of %d", who, rows, k);
  if (rows == 0) return H2C_OK;
  if (!x || !q || !scale) return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  if ((uintptr_t)x & (op_elem_size(type) - 1)) return op_error(H2C_ERR_INVALID, "%s: x must be aligned to its elements", who);
  if (((uintptr_t)q & 15) || (q_row & 15) || q_row < k)
    return op_error(H2C_ERR_INVALID, "%s: q must be 16-byte aligned with rows of a multiple of 16 bytes, at least k", who);
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
  if (m < 0 || n < 0 || k < 1 || k > H2C_I8_MAX_K)
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
  cudaStream_t st = (cudaStream_t)stream;
  MmArgs a;
  a.err = op_err_words();
  if (!a.err) return op_error(H2C_ERR_CUDA, "%s: no device", who);
  a.n = n; a.m = m; a.chunks = (k + KCH - 1) / KCH;
  shape_of(m, n, a.chunks, &a.nt, &a.splits);
  const int stage_bytes = W_STAGE + a.nt * KCH;
  a.stages = std::min(MAX_STAGES, SMEM_RING / stage_bytes);
  if (a.splits > 1)  // as deep as a CTA's share of K, and room for its partial tile
    a.stages = std::max(std::min(a.stages, (a.chunks + a.splits - 1) / a.splits),
                        (a.nt * TN * 4 + stage_bytes - 1) / stage_bytes);
  a.tiles_n = (n + TN - 1) / TN; a.tiles_m = (m + a.nt - 1) / a.nt;
  if ((long long)a.tiles_n * a.tiles_m > INT_MAX / 16) return op_error(H2C_ERR_INVALID, "%s: too many outputs", who);
  a.ws = w_scale; a.bias = bias; a.y = y; a.y_row = y_row;
  const int k_pad = (k + 15) / 16 * 16;
  CUtensorMap tw, tx;
  const void* xq = codes ? x : workspace;
  a.xs = codes ? x_scale : reinterpret_cast<const float*>(static_cast<const uint8_t*>(workspace) + codes_bytes(m, k));
  if (!u8_map(&tw, w, k, n, w_row, TN) || !u8_map(&tx, xq, k, m, codes ? x_row : k_pad, a.nt))
    return op_error(H2C_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed", who);
  if (!codes)
    if (int rc = quantize(who, x_type, x, x_row, m, k, workspace, k_pad, const_cast<float*>(a.xs), st)) return rc;
  if (y_type == H2C_TYPE_F32) return launch_matmul<float>(who, tw, tx, a, !codes, st);
  if (y_type == H2C_TYPE_F16) return launch_matmul<__half>(who, tw, tx, a, !codes, st);
  return launch_matmul<__nv_bfloat16>(who, tw, tx, a, !codes, st);
}

}  // extern "C"
