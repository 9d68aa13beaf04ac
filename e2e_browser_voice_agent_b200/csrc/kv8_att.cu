// Attention over the paged 8-bit cache (h2c_kv8_attention; the formula is stated in include/h2cuda.h).
//
// Few queries: k_att_rows (kv8_rows.cuh). Many queries: k_att_prompt (kv8_prompt.cuh). Here: the kernel that joins the parts of
// spans, and the entry.
#include "kv8_rows.cuh"

#include <algorithm>
#include <climits>
#include <cstdlib>

namespace h2 {
namespace {

// Joins the spans of one row: the weights of span s relative to the common maximum are 2^(m_s - m). Span s of the row has
// its sums at part + s * part_step and its (m, l) at ml + s * ml_step. `n_warps` share it, `w` is the warp's turn (see JOIN_WARPS).
template <class T, int HD>
__device__ __forceinline__ void join_row(const AttArgs& a, const float* part, size_t part_step, const float2* ml, size_t ml_step,
                                         int used, int tok, int hq, int w, int n_warps) {
  constexpr int V = HD / 32;  // dimensions per lane
  __shared__ float acc[JOIN_WARPS][HD], acc_l[JOIN_WARPS];
  const int lane = threadIdx.x & 31;
  auto load = [&](int s, float* o) {
    if (V == 4) *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(part + s * part_step + V * lane);
    else *reinterpret_cast<float2*>(o) = *reinterpret_cast<const float2*>(part + s * part_step + V * lane);
  };
  float m = -INFINITY, v[V], l = 0.f;
#pragma unroll
  for (int i = 0; i < V; i++) v[i] = 0.f;
  auto add = [&](float2 x, const float* o) {
    const float f = x.x == -INFINITY ? 0.f : exp2_fast(x.x - m);
    l += f * x.y;
#pragma unroll
    for (int i = 0; i < V; i++) v[i] += f * o[i];
  };
  if (n_warps == 1) {  // everything on its way at once (a chunk of 256 on 4,096 tokens, 10 spans: 3 us less)
    float2 x[JOIN_WARP_SPANS];
    float o[JOIN_WARP_SPANS][V];
#pragma unroll
    for (int s = 0; s < JOIN_WARP_SPANS; s++)
      if (s < used) {
        x[s] = ml[s * ml_step];
        load(s, o[s]);
      }
#pragma unroll
    for (int s = 0; s < JOIN_WARP_SPANS; s++)
      if (s < used) m = fmaxf(m, x[s].x);
#pragma unroll
    for (int s = 0; s < JOIN_WARP_SPANS; s++)
      if (s < used) add(x[s], o[s]);
  } else {
    for (int s = lane; s < used; s += 32) m = fmaxf(m, ml[s * ml_step].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll 4
    for (int s = w; s < used; s += n_warps) {
      float o[V];
      load(s, o);
      add(ml[s * ml_step], o);
    }
  }
  if (n_warps > 1) {
#pragma unroll
    for (int i = 0; i < V; i++) acc[w][V * lane + i] = v[i];
    if (lane == 0) acc_l[w] = l;
    __syncthreads();
    if (w) return;
    for (int k = 1; k < n_warps; k++) {
      l += acc_l[k];
#pragma unroll
      for (int i = 0; i < V; i++) v[i] += acc[k][V * lane + i];
    }
  }
  const float inv = l != 0.f ? 1.f / l : 1.f;
  T* dst = static_cast<T*>(a.out) + (long long)tok * a.out_row + hq * a.out_head + V * lane;
#pragma unroll
  for (int i = 0; i < V; i++) v[i] *= inv;
  if (V == 4) {
    store4(dst, v, a.out_vec);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) dst[i] = from_f<T>(v[i]);
  }
  if (lane == 0 && a.lse)
    a.lse[(size_t)tok * a.heads + hq] = l == 0.f ? -INFINITY : 0.69314718055994531f * (log2f(l) + m - P_SHIFT);
}

// Row `i` of the CTAs that join, for this warp: its turn and the warps that share the row.
struct JoinTurn {
  int i, w, n;
};
__device__ __forceinline__ JoinTurn join_turn(int cta, int splits) {
  const int warp = threadIdx.x >> 5;
  if (splits <= JOIN_WARP_SPANS) return {cta * JOIN_WARPS + warp, 0, 1};
  return {cta, warp, JOIN_WARPS};
}
// The first row_ctas CTAs join k_att_rows' spans, per_req of them a request's; the others k_att_prompt's.
template <class T, int HD>
__device__ __forceinline__ void join_rows_at(const RowArgs& ra, int r, int cta) {
  const AttArgs& a = ra.a;
  const JoinTurn t = join_turn(cta, ra.splits);
  const int jr = t.i % RW_ROWS, th = t.i / RW_ROWS, head = th % a.kv_heads, tile = th / a.kv_heads;
  int n_all;
  const Request R = request_of(a, r, &n_all);
  const int row0 = tile * RW_ROWS, n_rows = R.n_q * a.group, row = row0 + jr;
  if (row >= n_rows || n_rows > ra.max_rows) return;
  int lo, hi;
  key_range(a, R, n_all, row0 / a.group, min(row0 + RW_ROWS - 1, n_rows - 1) / a.group, &lo, &hi);
  const Span sp = spans_of(lo, hi, ra.splits, ra.blocks, RW_BLK);
  if (sp.used == 1) return;  // (written by its only span)
  const size_t at = (((size_t)r * a.kv_heads + head) * ra.tiles + tile) * ra.splits * RW_ROWS + jr;
  int hq;
  const int tok = token_of(a, row, &hq);
  join_row<T, HD>(a, ra.part + at * HD, (size_t)RW_ROWS * HD, ra.ml + at, RW_ROWS, sp.used, R.first + tok, head * a.group + hq,
                  t.w, t.n);
}
template <class T, int HD>
__device__ __forceinline__ void join_prompts_at(const PromptArgs& pa, int cta) {
  const AttArgs& a = pa.a;
  const PromptShape shape = shape_of_call(pa);
  if (shape.splits == 1) return;
  const JoinTurn t = join_turn(cta, shape.splits);
  const int jr = t.i % PR_ROWS, th = t.i / PR_ROWS, head = th % a.kv_heads, idx = th / a.kv_heads;
  if (idx >= shape.tiles) return;
  const TileAt at = tile_at(pa, idx);
  if (at.r < 0) return;
  const Request R = at.R;
  const int n_all = at.n_all, n_rows = R.n_q * a.group, row = at.row0 + jr;
  if (row >= n_rows) return;
  int lo, hi;
  key_range(a, R, n_all, at.row0 / a.group, min(at.row0 + PR_ROWS - 1, n_rows - 1) / a.group, &lo, &hi);
  const Span sp = spans_of(lo, hi, shape.splits, shape.blocks, PR_KEYS);
  if (sp.used == 1) return;
  const size_t u = ((size_t)idx * a.kv_heads + head) * shape.splits * PR_ROWS + jr;
  int hq;
  const int tok = token_of(a, row, &hq);
  join_row<T, HD>(a, pa.part + u * HD, (size_t)PR_ROWS * HD, pa.ml + u, PR_ROWS, sp.used, R.first + tok, head * a.group + hq, t.w,
                  t.n);
}
template <class T, int HD>
__global__ void __launch_bounds__(32 * JOIN_WARPS) k_att_join(const RowArgs ra, const PromptArgs pa, int row_ctas, int per_req) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.x;
  if (b < row_ctas) join_rows_at<T, HD>(ra, b / per_req, b % per_req);
  else join_prompts_at<T, HD>(pa, b - row_ctas);
}

// ---------------------------------------------------------------- host

template <class T, int HD>
int launch(const char* who, const WorkPlan& p, AttArgs a, void* workspace, cudaStream_t st) {
  float* part = static_cast<float*>(workspace);
  float* p_part = part + p.units * RW_ROWS * HD;
  float* sums = p_part + (size_t)p.p_units * PR_ROWS * HD;
  float2* ml = reinterpret_cast<float2*>(sums + (p.spill ? (size_t)PR_SLOTS * PR_ROWS * HD : 0));
  int* err = p.prompt ? op_err_words() : nullptr;
  if (p.prompt && !err) return op_error(H2C_ERR_CUDA, "%s: no device", who);
  const PromptArgs pa{a, p.min_rows, p.shape, p.p_keys, p.counted ? p.p_units : 0, p_part, ml + p.units * RW_ROWS, p.spill ? sums : nullptr, err};
  const RowArgs ra{a, p.splits, p.blocks, p.tiles, p.max_rows, p.cluster, part, ml};
  // a kernel that may start while the one before it still runs waits for that one's end itself
  cudaLaunchAttribute dependent;
  dependent.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  dependent.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.stream = st;
  cfg.attrs = attr;
  cudaError_t c = cudaSuccess;
  if (p.prompt) {
    static unsigned char done[OP_MAX_DEVICES];
    constexpr int smem = PromptCfg<T, HD>::SMEM;
    if (int rc = op_once(who, done, [] {
          return cudaFuncSetAttribute(k_att_prompt<T, HD, AttArgs>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        }))
      return rc;
    k_att_prompt<T, HD, AttArgs><<<std::max(p.shape.tiles * a.kv_heads, p.p_units), PR_THREADS, smem, st>>>(pa);
    if (int rc = op_launched(who)) return rc;
  }
  if (p.rows) {
    static unsigned char done[OP_MAX_DEVICES];
    constexpr int smem = RowSmem<HD>::BYTES;
    if (int rc = op_once(who, done, [] {
          return cudaFuncSetAttribute(k_att_rows<T, HD, AttArgs>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        }))
      return rc;
    cfg.gridDim = dim3((unsigned)p.splits * a.kv_heads * p.tiles, a.n_req);
    cfg.blockDim = dim3(RW_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    if (p.cluster) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attr[cfg.numAttrs++].val.clusterDim = {(unsigned)p.splits, 1, 1};
    }
    if (p.prompt) attr[cfg.numAttrs++] = dependent;
    c = cudaLaunchKernelEx(&cfg, k_att_rows<T, HD, AttArgs>, ra);
  }
  const int per_req = p.rows && p.splits > 1 && !p.cluster ? (int)join_ctas((long long)RW_ROWS * a.kv_heads * p.tiles, p.splits) : 0;
  if (c == cudaSuccess && (per_req || p.p_join)) {
    cfg.gridDim = dim3((unsigned)per_req * a.n_req + p.p_join);
    cfg.blockDim = dim3(32 * JOIN_WARPS);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    attr[0] = dependent;
    c = cudaLaunchKernelEx(&cfg, k_att_join<T, HD>, ra, pa, per_req * a.n_req, std::max(1, per_req));
  }
  if (c == cudaSuccess) return H2C_OK;
  cudaGetLastError();
  return op_error(H2C_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(c));
}

template <class T>
int launch_typed(const char* who, int head_dim, const WorkPlan& p, const AttArgs& a, void* workspace, cudaStream_t st) {
  return head_dim == 64 ? launch<T, 64>(who, p, a, workspace, st) : launch<T, 128>(who, p, a, workspace, st);
}

}  // namespace
}  // namespace h2

using namespace h2;

extern "C" {

uint64_t h2c_kv8_attention_workspace(const h2c_kv8_attention_args* g) {
  if (check_args("h2c_kv8_attention_workspace", g) || nothing_to_do(g)) return 0;
  return plan_work(g).bytes;
}

int h2c_kv8_attention(const h2c_kv8_attention_args* g, void* stream) {
  const char* who = "h2c_kv8_attention";
  if (int rc = check_args(who, g)) return rc;
  if (nothing_to_do(g)) return H2C_OK;
  if (!g->q || !g->out || !g->kv || !g->kv_scale || !g->q_start || !g->kv_len || (g->table_cols && !g->block_table))
    return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  const size_t es = op_elem_size(g->type);
  if ((uintptr_t)g->kv & 15) return op_error(H2C_ERR_INVALID, "%s: the cache must be 16-byte aligned", who);
  if (((uintptr_t)g->q | (uintptr_t)g->out) & (es - 1))
    return op_error(H2C_ERR_INVALID, "%s: q and out must be aligned to their elements", who);
  const WorkPlan p = plan_work(g);
  if (p.bytes && (!g->workspace || g->workspace_bytes < p.bytes || ((uintptr_t)g->workspace & 15)))
    return op_error(H2C_ERR_INVALID, "%s: needs %llu bytes of 16-byte aligned workspace, got %llu", who,
                    (unsigned long long)p.bytes, (unsigned long long)(g->workspace ? g->workspace_bytes : 0));
  const uint64_t n4 = 4ull * g->n_req;
  const OpRange in[] = {{"block_table", g->block_table, n4 * g->table_cols, 4}, {"q_start", g->q_start, n4 + 4, 4}, {"kv_len", g->kv_len, n4, 4}};
  if (int rc = check_memory(who, g, in, 3, p.bytes)) return rc;
  const long long most = std::max((long long)p.splits * p.tiles * RW_ROWS, (long long)p.shape.tiles * PR_ROWS);
  if (most * g->kv_heads > INT_MAX) return op_error(H2C_ERR_INVALID, "%s: too many rows for one call", who);
  const AttArgs a = args_of(g);
  cudaStream_t st = (cudaStream_t)stream;
  if (g->type == H2C_TYPE_F32) return launch_typed<float>(who, g->head_dim, p, a, g->workspace, st);
  if (g->type == H2C_TYPE_F16) return launch_typed<__half>(who, g->head_dim, p, a, g->workspace, st);
  return launch_typed<__nv_bfloat16>(who, g->head_dim, p, a, g->workspace, st);
}

}  // extern "C"
