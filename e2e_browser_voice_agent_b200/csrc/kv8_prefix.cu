// Attention of requests that share prefixes over the paged 8-bit cache (h2c_kv8_prefix_attention; the formula is stated in
// include/h2cuda.h).
//
// Two passes and a join. All rows of a group of requests attend to the group's prefix together, as one request whose rows see every
// position: its keys are read once for 8 (k_att_rows) or 256 (k_att_prompt) rows of a kv head instead of once for each request.
// Each request attends to its own positions as in h2c_kv8_attention. Both passes leave (sum, maximum, weight) of each span of keys in
// the workspace, and k_prefix_join adds up what belongs to a row: the softmax over all its positions. The kernels are launched one
// behind the other without waiting for each other's end (programmatic dependent launch), those with tensor memory first; the
// single tokens' CTAs take the SMs that they leave.
#include "kv8_rows.cuh"

namespace h2 {
namespace {

struct Pass {
  RowArgsOf<SharedArgs> ra;
  PromptArgsOf<SharedArgs> pa;
  int rows, prompt;  // whether k_att_rows, k_att_prompt take part
};

// Where the spans of a row lie: span s has its sums at part + s * part_step and its (m, l) at ml + s * ml_step.
struct Parts {
  const float* part;
  const float2* ml;
  size_t part_step, ml_step;
  int used;  // 0: the row is in no request (group)
};

// The parts of row t (of q) and head hq. By whole warps: 32 requests at a time, until the one that has the row; the row tiles of
// k_att_prompt before it are counted on the way.
template <int HD>
__device__ __forceinline__ Parts parts_of(const Pass& p, int t, int hq) {
  const SharedArgs& a = p.ra.a;
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int base = 0; base < a.n_req; base += 32) {
    const int r = base + lane;
    int n = 0, n_all = 0;
    Request R{0, 0, 0};
    if (r < a.n_req) {
      R = request_of(a, r, &n_all);
      const int rows = R.n_q * a.group;
      if (p.prompt && rows >= p.pa.min_rows) n = (rows + PR_ROWS - 1) / PR_ROWS;
    }
    const unsigned in = __ballot_sync(0xffffffffu, t >= R.first && t - R.first < R.n_q);
    if (!in) {
      before += __reduce_add_sync(0xffffffffu, n);
      continue;
    }
    const int l = __ffs(in) - 1;
    before += __reduce_add_sync(0xffffffffu, lane < l ? n : 0);
    n_all = __shfl_sync(0xffffffffu, n_all, l);
    R.first = __shfl_sync(0xffffffffu, R.first, l);
    R.n_q = __shfl_sync(0xffffffffu, R.n_q, l);
    R.len = __shfl_sync(0xffffffffu, R.len, l);
    const int head = hq / a.group, row = (t - R.first) * a.group + (hq - head * a.group), n_rows = R.n_q * a.group;
    int lo, hi;
    if (p.prompt && n_rows >= p.pa.min_rows) {
      const PromptShape shape = shape_of_call(p.pa);
      const int idx = before + row / PR_ROWS, row0 = row / PR_ROWS * PR_ROWS;
      if (idx >= shape.tiles) break;  // (starts of requests without sense: not computed)
      key_range(a, R, n_all, row0 / a.group, min(row0 + PR_ROWS - 1, n_rows - 1) / a.group, &lo, &hi);
      const size_t u = ((size_t)idx * a.kv_heads + head) * shape.splits * PR_ROWS + (row - row0);
      return {p.pa.part + u * HD, p.pa.ml + u, (size_t)PR_ROWS * HD, PR_ROWS, spans_of(lo, hi, shape.splits, shape.blocks, PR_KEYS).used};
    }
    const int tile = row / RW_ROWS, row0 = tile * RW_ROWS;
    if (tile >= p.ra.tiles) break;
    key_range(a, R, n_all, row0 / a.group, min(row0 + RW_ROWS - 1, n_rows - 1) / a.group, &lo, &hi);
    const size_t u = (((size_t)(base + l) * a.kv_heads + head) * p.ra.tiles + tile) * p.ra.splits * RW_ROWS + (row - row0);
    return {p.ra.part + u * HD, p.ra.ml + u, (size_t)RW_ROWS * HD, RW_ROWS, spans_of(lo, hi, p.ra.splits, p.ra.blocks, RW_BLK).used};
  }
  return {nullptr, nullptr, 0, 0, 0};
}

// NW warps (1 or JOIN_WARPS) a row and head: see JOIN_WARPS.
template <class T, int HD, int NW>
__global__ void __launch_bounds__(32 * JOIN_WARPS) k_prefix_join(const Pass prefix, const Pass own) {
  constexpr int V = HD / 32, UN = 4;
  __shared__ float acc[NW][HD], acc_l[NW];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const AttArgs& a = own.ra.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = NW > 1 ? warp : 0;
  const long long i = NW > 1 ? blockIdx.x : (long long)blockIdx.x * JOIN_WARPS + warp;
  const int t = (int)(i / a.heads), hq = (int)(i - (long long)t * a.heads);
  if (t >= a.rows) return;
  const Parts o = parts_of<HD>(own, t, hq);
  if (o.used == 0) return;  // (a row of no request is not touched)
  const Parts p = parts_of<HD>(prefix, t, hq);
  const int all = p.used + o.used;
  auto ml_of = [&](int s) { return s < p.used ? p.ml[s * p.ml_step] : o.ml[(s - p.used) * o.ml_step]; };
  float m = -INFINITY;
  for (int s = lane; s < all; s += 32) m = fmaxf(m, ml_of(s).x);
#pragma unroll
  for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  float v[V], l = 0.f;
#pragma unroll
  for (int k = 0; k < V; k++) v[k] = 0.f;
  for (int s0 = w; s0 < all; s0 += UN * NW) {
    float x[UN][V];
    float2 ml[UN];
#pragma unroll
    for (int k = 0; k < UN; k++) {
      const int s = s0 + k * NW;
      if (s < all) {
        const float* src = (s < p.used ? p.part + s * p.part_step : o.part + (s - p.used) * o.part_step) + V * lane;
        ml[k] = ml_of(s);
        if (V == 4) *reinterpret_cast<float4*>(x[k]) = *reinterpret_cast<const float4*>(src);
        else *reinterpret_cast<float2*>(x[k]) = *reinterpret_cast<const float2*>(src);
      }
    }
#pragma unroll
    for (int k = 0; k < UN; k++)
      if (s0 + k * NW < all) {
        const float f = ml[k].x == -INFINITY ? 0.f : exp2_fast(ml[k].x - m);
        l = fmaf(f, ml[k].y, l);
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = fmaf(f, x[k][j], v[j]);
      }
  }
  if (NW > 1) {
#pragma unroll
    for (int k = 0; k < V; k++) acc[w][V * lane + k] = v[k];
    if (lane == 0) acc_l[w] = l;
    __syncthreads();
    if (w) return;
    for (int n = 1; n < NW; n++) {
      l += acc_l[n];
#pragma unroll
      for (int k = 0; k < V; k++) v[k] += acc[n][V * lane + k];
    }
  }
  const float inv = l != 0.f ? 1.f / l : 1.f;
  T* dst = static_cast<T*>(a.out) + (long long)t * a.out_row + hq * a.out_head + V * lane;
#pragma unroll
  for (int k = 0; k < V; k++) v[k] *= inv;
  if (V == 4) {
    store4(dst, v, a.out_vec);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) dst[k] = from_f<T>(v[k]);
  }
  if (lane == 0 && a.lse)
    a.lse[(size_t)t * a.heads + hq] = l == 0.f ? -INFINITY : 0.69314718055994531f * (log2f(l) + m - P_SHIFT);
}

// ---------------------------------------------------------------- host

// The prefix pass as a call of its own, whose requests are the groups: each may have all rows.
h2c_kv8_attention_args groups_of(const h2c_kv8_prefix_args* g) {
  h2c_kv8_attention_args p = g->own;
  p.block_table = g->prefix_table;
  p.table_cols = g->prefix_cols;
  p.n_req = g->n_groups;
  p.kv_len = g->prefix_len;
  p.max_q = p.rows;
  p.max_kv = g->max_prefix;
  return p;
}

struct PrefixPlan {
  WorkPlan own, prefix;
  bool shared;      // whether there is a prefix pass
  size_t bytes;
};
PrefixPlan plan_prefix(const h2c_kv8_prefix_args* g) {
  PrefixPlan p = {};
  p.own = plan_work(&g->own, true);
  p.shared = g->n_groups > 0 && g->prefix_cols > 0;
  if (p.shared) {
    const h2c_kv8_attention_args groups = groups_of(g);
    p.prefix = plan_work(&groups, true);
  }
  // (a CTA holds its place of spilled sums alone, whichever kernel it is of: one set of them)
  const size_t sums = (size_t)PR_SLOTS * PR_ROWS * g->own.head_dim * 4;
  p.bytes = p.own.bytes + p.prefix.bytes - (p.own.spill && p.prefix.spill ? sums : 0);
  return p;
}
long long tiles_of(const WorkPlan& p) { return std::max((long long)p.splits * p.tiles * RW_ROWS, (long long)p.shape.tiles * PR_ROWS * std::max(1, p.shape.splits)); }

template <class T, int HD>
int launch(const char* who, const PrefixPlan& plan, const h2c_kv8_prefix_args* g, cudaStream_t st) {
  float* at = static_cast<float*>(g->own.workspace);
  float* sums = nullptr;
  if (plan.own.spill || plan.prefix.spill) {
    sums = at;
    at += (size_t)PR_SLOTS * PR_ROWS * HD;
  }
  auto take = [&](size_t units, int rows) {
    float* p = at;
    at += units * rows * HD;
    return p;
  };
  int* err = plan.own.prompt || plan.prefix.prompt ? op_err_words() : nullptr;
  if ((plan.own.prompt || plan.prefix.prompt) && !err) return op_error(H2C_ERR_CUDA, "%s: no device", who);
  Pass pass[2] = {};  // prefix, own
  for (int i = 0; i < 2; i++) {
    const WorkPlan& p = i ? plan.own : plan.prefix;
    SharedArgs a{};
    const h2c_kv8_attention_args groups = groups_of(g);
    static_cast<AttArgs&>(a) = args_of(i ? &g->own : &groups);
    if (!i) {
      a.group_start = g->group_start;
      a.n_own = g->own.n_req;
      if (!plan.shared) a.n_req = 0;
    }
    float* part = take(p.units, RW_ROWS);
    float* p_part = take(p.p_units, PR_ROWS);
    pass[i].rows = p.rows;
    pass[i].prompt = p.prompt;
    pass[i].ra = {a, p.splits, p.blocks, p.tiles, p.max_rows, 0, part, nullptr};
    pass[i].pa = {a, p.min_rows, p.shape, p.p_keys, p.counted ? 148 : 0, p_part, nullptr, p.spill ? sums : nullptr, err};
  }
  for (int i = 0; i < 2; i++) {
    const WorkPlan& p = i ? plan.own : plan.prefix;
    pass[i].ra.ml = reinterpret_cast<float2*>(at);
    at += p.units * RW_ROWS * 2;
    pass[i].pa.ml = reinterpret_cast<float2*>(at);
    at += (size_t)p.p_units * PR_ROWS * 2;
  }

  static unsigned char done[OP_MAX_DEVICES];
  constexpr int p_smem = PromptCfg<T, HD>::SMEM, r_smem = RowSmem<HD>::BYTES;
  if (int rc = op_once(who, done, [] {
        const cudaError_t c = cudaFuncSetAttribute(k_att_prompt<T, HD, SharedArgs>, cudaFuncAttributeMaxDynamicSharedMemorySize, p_smem);
        return c != cudaSuccess ? c : cudaFuncSetAttribute(k_att_rows<T, HD, SharedArgs>, cudaFuncAttributeMaxDynamicSharedMemorySize, r_smem);
      }))
    return rc;
  // each kernel but the first may start while the one before it still runs, and ends after it
  cudaLaunchAttribute dependent;
  dependent.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  dependent.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cfg.attrs = &dependent;
  cudaError_t c = cudaSuccess;
  for (int i = 0; i < 2 && c == cudaSuccess; i++) {
    const WorkPlan& p = i ? plan.own : plan.prefix;
    if (!p.prompt) continue;
    cfg.gridDim = dim3((unsigned)std::max(p.shape.tiles * g->own.kv_heads * p.shape.splits, p.counted ? 148 : 0));
    cfg.blockDim = dim3(PR_THREADS);
    cfg.dynamicSmemBytes = p_smem;
    c = cudaLaunchKernelEx(&cfg, k_att_prompt<T, HD, SharedArgs>, pass[i].pa);
    cfg.numAttrs = 1;
  }
  for (int i = 0; i < 2 && c == cudaSuccess; i++) {
    const WorkPlan& p = i ? plan.own : plan.prefix;
    if (!p.rows) continue;
    cfg.gridDim = dim3((unsigned)p.splits * g->own.kv_heads * p.tiles, pass[i].ra.a.n_req);
    cfg.blockDim = dim3(RW_WARPS * 32);
    cfg.dynamicSmemBytes = r_smem;
    c = cudaLaunchKernelEx(&cfg, k_att_rows<T, HD, SharedArgs>, pass[i].ra);
    cfg.numAttrs = 1;
  }
  if (c == cudaSuccess) {
    auto most = [&](const WorkPlan& p) {  // spans of a row
      return std::max(p.rows ? p.splits : 0, p.prompt ? p.counted ? 148 / g->own.kv_heads : p.shape.splits : 0);
    };
    const long long rows = (long long)g->own.rows * g->own.heads;
    const int spans = most(plan.own) + most(plan.prefix);
    cfg.gridDim = dim3(join_ctas(rows, spans));
    cfg.blockDim = dim3(32 * JOIN_WARPS);
    cfg.dynamicSmemBytes = 0;
    c = spans <= JOIN_WARP_SPANS ? cudaLaunchKernelEx(&cfg, k_prefix_join<T, HD, 1>, pass[0], pass[1])
                                 : cudaLaunchKernelEx(&cfg, k_prefix_join<T, HD, JOIN_WARPS>, pass[0], pass[1]);
  }
  if (c == cudaSuccess) return H2C_OK;
  cudaGetLastError();
  return op_error(H2C_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(c));
}

template <class T>
int launch_typed(const char* who, const PrefixPlan& p, const h2c_kv8_prefix_args* g, cudaStream_t st) {
  return g->own.head_dim == 64 ? launch<T, 64>(who, p, g, st) : launch<T, 128>(who, p, g, st);
}

int check_prefix(const char* who, const h2c_kv8_prefix_args* g) {
  if (!g) return op_error(H2C_ERR_INVALID, "%s: null arguments", who);
  if (int rc = check_args(who, &g->own)) return rc;
  if (g->own.window) return op_error(H2C_ERR_INVALID, "%s: there is no window behind shared prefixes (%d)", who, g->own.window);
  if (g->n_groups < 0 || g->n_groups > H2C_KV8_MAX_REQUESTS)
    return op_error(H2C_ERR_INVALID, "%s: n_groups must be 0 to %d, not %d", who, H2C_KV8_MAX_REQUESTS, g->n_groups);
  if (g->prefix_cols < 0 || g->max_prefix < 0) return op_error(H2C_ERR_INVALID, "%s: a size is negative", who);
  if ((long long)g->own.rows * (g->own.heads / g->own.kv_heads) > INT_MAX / 2)
    return op_error(H2C_ERR_INVALID, "%s: rows %d out of range", who, g->own.rows);
  return H2C_OK;
}

}  // namespace
}  // namespace h2

using namespace h2;

extern "C" {

uint64_t h2c_kv8_prefix_attention_workspace(const h2c_kv8_prefix_args* g) {
  if (check_prefix("h2c_kv8_prefix_attention_workspace", g) || nothing_to_do(&g->own)) return 0;
  return plan_prefix(g).bytes;
}

int h2c_kv8_prefix_attention(const h2c_kv8_prefix_args* g, void* stream) {
  const char* who = "h2c_kv8_prefix_attention";
  if (int rc = check_prefix(who, g)) return rc;
  const h2c_kv8_attention_args* o = &g->own;
  if (nothing_to_do(o)) return H2C_OK;
  if (!o->q || !o->out || !o->kv || !o->kv_scale || !o->q_start || !o->kv_len || (o->table_cols && !o->block_table) ||
      (g->n_groups && (!g->prefix_len || !g->group_start || (g->prefix_cols && !g->prefix_table))))
    return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  const size_t es = op_elem_size(o->type);
  if ((uintptr_t)o->kv & 15) return op_error(H2C_ERR_INVALID, "%s: the cache must be 16-byte aligned", who);
  if (((uintptr_t)o->q | (uintptr_t)o->out) & (es - 1))
    return op_error(H2C_ERR_INVALID, "%s: q and out must be aligned to their elements", who);
  const PrefixPlan p = plan_prefix(g);
  if (p.bytes && (!o->workspace || o->workspace_bytes < p.bytes || ((uintptr_t)o->workspace & 15)))
    return op_error(H2C_ERR_INVALID, "%s: needs %llu bytes of 16-byte aligned workspace, got %llu", who, (unsigned long long)p.bytes,
                    (unsigned long long)(o->workspace ? o->workspace_bytes : 0));
  const uint64_t n4 = 4ull * o->n_req, g4 = 4ull * g->n_groups;
  const OpRange in[] = {{"block_table", o->block_table, n4 * o->table_cols, 4}, {"q_start", o->q_start, n4 + 4, 4},
                        {"kv_len", o->kv_len, n4, 4},                          {"prefix_table", g->prefix_table, g4 * g->prefix_cols, 4},
                        {"prefix_len", g->prefix_len, g4, 4},                  {"group_start", g->group_start, g4 ? g4 + 4 : 0, 4}};
  if (int rc = check_memory(who, o, in, 6, p.bytes)) return rc;
  if (std::max(tiles_of(p.own), p.shared ? tiles_of(p.prefix) : 0LL) * o->kv_heads > INT_MAX || (long long)o->rows * o->heads > INT_MAX)
    return op_error(H2C_ERR_INVALID, "%s: too many rows for one call", who);
  cudaStream_t st = (cudaStream_t)stream;
  if (o->type == H2C_TYPE_F32) return launch_typed<float>(who, p, g, st);
  if (o->type == H2C_TYPE_F16) return launch_typed<__half>(who, p, g, st);
  return launch_typed<__nv_bfloat16>(who, p, g, st);
}

}  // extern "C"
