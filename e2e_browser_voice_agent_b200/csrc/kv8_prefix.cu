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

// The request (group) that has row t of q, and the row tiles of k_att_prompt before its own. By all threads of the CTA, which test as
// many requests at a time.
struct Owner {
  int r, n_all, before;  // r = -1: no request has it
  Request R;
};
__device__ __forceinline__ void find_owner(const Pass& p, int t, Owner* owner, int* sums) {
  const SharedArgs& a = p.ra.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int base = 0;; base += 32 * JOIN_WARPS) {
    const int r = base + threadIdx.x;
    int n = 0, n_all = 0;
    Request R{0, 0, 0};
    if (r < a.n_req) {
      R = request_of(a, r, &n_all);
      const int rows = R.n_q * a.group;
      if (p.prompt && rows >= p.pa.min_rows) n = (rows + PR_ROWS - 1) / PR_ROWS;
    }
    const bool in = t >= R.first && t - R.first < R.n_q;
    int first = __reduce_min_sync(0xffffffffu, in ? r : INT_MAX);  // (of several, the first)
    const int sum = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) sums[warp] = sum, sums[JOIN_WARPS + warp] = first;
    __syncthreads();
    int all = 0, mine = before;
    first = INT_MAX;
#pragma unroll
    for (int w = 0; w < JOIN_WARPS; w++) {
      first = min(first, sums[JOIN_WARPS + w]);
      if (w < warp) mine += sums[w];
      all += sums[w];
    }
    if (first != INT_MAX) {
      if (first >> 5 == r >> 5) {  // (its warp)
        mine += __reduce_add_sync(0xffffffffu, r < first ? n : 0);
        if (r == first) *owner = {r, n_all, mine, R};
      }
    } else if (base + 32 * JOIN_WARPS >= a.n_req) {
      if (threadIdx.x == 0) owner->r = -1;
    }
    __syncthreads();
    if (first != INT_MAX || base + 32 * JOIN_WARPS >= a.n_req) return;
    before += all;
  }
}

// The parts of row t of q, which `o` has, and head hq. (idx, tile: beyond what was computed only with starts of requests without sense.)
template <int HD>
__device__ __forceinline__ Parts parts_of(const Pass& p, const PromptShape& shape, const Owner& o, int t, int hq) {
  if (o.r < 0) return {nullptr, nullptr, 0, 0, 0};
  const SharedArgs& a = p.ra.a;
  const Request& R = o.R;
  const int head = hq / a.group, row = (t - R.first) * a.group + (hq - head * a.group), n_rows = R.n_q * a.group;
  int lo, hi;
  if (p.prompt && n_rows >= p.pa.min_rows) {
    const int idx = o.before + row / PR_ROWS, row0 = row / PR_ROWS * PR_ROWS;
    if (idx >= shape.tiles) return {nullptr, nullptr, 0, 0, 0};
    key_range(a, R, o.n_all, row0 / a.group, min(row0 + PR_ROWS - 1, n_rows - 1) / a.group, &lo, &hi);
    const size_t u = ((size_t)idx * a.kv_heads + head) * shape.splits * PR_ROWS + (row - row0);
    return {p.pa.part + u * HD, p.pa.ml + u, (size_t)PR_ROWS * HD, PR_ROWS, spans_of(lo, hi, shape.splits, shape.blocks, PR_KEYS).used};
  }
  const int tile = row / RW_ROWS, row0 = tile * RW_ROWS;
  if (tile >= p.ra.tiles) return {nullptr, nullptr, 0, 0, 0};
  key_range(a, R, o.n_all, row0 / a.group, min(row0 + RW_ROWS - 1, n_rows - 1) / a.group, &lo, &hi);
  const size_t u = (((size_t)o.r * a.kv_heads + head) * p.ra.tiles + tile) * p.ra.splits * RW_ROWS + (row - row0);
  return {p.ra.part + u * HD, p.ra.ml + u, (size_t)RW_ROWS * HD, RW_ROWS, spans_of(lo, hi, p.ra.splits, p.ra.blocks, RW_BLK).used};
}

// A CTA takes `heads` heads of one token, NW warps (1 or JOIN_WARPS, see there) a head. What it looks up needs nothing of the passes and
// goes on while they end.
template <class T, int HD, int NW>
__global__ void __launch_bounds__(32 * JOIN_WARPS) k_prefix_join(const Pass prefix, const Pass own, int heads) {
  constexpr int V = HD / 32, UN = 6;
  __shared__ float acc[NW][HD];
  __shared__ float2 acc_ml[NW];
  __shared__ Owner owner[2];
  __shared__ int sums[2 * JOIN_WARPS];
  const AttArgs& a = own.ra.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = NW > 1 ? warp : 0, t = blockIdx.x;
  const int h0 = blockIdx.y * heads, h1 = min(h0 + heads, a.heads);
  find_owner(own, t, &owner[1], sums);
  find_owner(prefix, t, &owner[0], sums);
  const PromptShape own_shape = shape_of_call(own.pa), prefix_shape = shape_of_call(prefix.pa);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int hq = h0 + (NW > 1 ? 0 : warp); hq < h1; hq += NW > 1 ? 1 : JOIN_WARPS) {
    const Parts o = parts_of<HD>(own, own_shape, owner[1], t, hq);
    if (o.used == 0) return;  // (a row of no request is not touched)
    const Parts p = parts_of<HD>(prefix, prefix_shape, owner[0], t, hq);
    const int all = p.used + o.used;
    // UN spans at a time, everything of them on its way at once; the sums are relative to the largest maximum so far
    float m = -INFINITY, v[V], l = 0.f;
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = 0.f;
    for (int s0 = w; s0 < all; s0 += UN * NW) {
      float x[UN][V];
      float2 ml[UN];
#pragma unroll
      for (int k = 0; k < UN; k++) {
        const int s = s0 + k * NW;
        ml[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int j = 0; j < V; j++) x[k][j] = 0.f;
        if (s < all) {
          const bool shared = s < p.used;
          const int i = shared ? s : s - p.used;
          const float* src = (shared ? p.part + i * p.part_step : o.part + i * o.part_step) + V * lane;
          ml[k] = shared ? p.ml[i * p.ml_step] : o.ml[i * o.ml_step];
          if (V == 4) *reinterpret_cast<float4*>(x[k]) = *reinterpret_cast<const float4*>(src);
          else *reinterpret_cast<float2*>(x[k]) = *reinterpret_cast<const float2*>(src);
        }
      }
      float top = m;
#pragma unroll
      for (int k = 0; k < UN; k++) top = fmaxf(top, ml[k].x);
      const float f_old = m == -INFINITY ? 0.f : exp2_fast(m - top);
      m = top;
      l *= f_old;
#pragma unroll
      for (int j = 0; j < V; j++) v[j] *= f_old;
#pragma unroll
      for (int k = 0; k < UN; k++) {
        const float f = ml[k].x == -INFINITY ? 0.f : exp2_fast(ml[k].x - m);
        l = fmaf(f, ml[k].y, l);
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = fmaf(f, x[k][j], v[j]);
      }
    }
    if (NW > 1) {
#pragma unroll
      for (int k = 0; k < V; k++) acc[w][V * lane + k] = v[k];
      if (lane == 0) acc_ml[w] = make_float2(m, l);
      __syncthreads();
      if (w == 0) {
        for (int n = 1; n < NW; n++) m = fmaxf(m, acc_ml[n].x);
        l = 0.f;
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = 0.f;
        for (int n = 0; n < NW; n++) {
          const float f = acc_ml[n].x == -INFINITY ? 0.f : exp2_fast(acc_ml[n].x - m);
          l = fmaf(f, acc_ml[n].y, l);
#pragma unroll
          for (int k = 0; k < V; k++) v[k] = fmaf(f, acc[n][V * lane + k], v[k]);
        }
      }
      __syncthreads();
    }
    if (w == 0) {
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
  }
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
    // eight warps a head where spans are many and rows few; else a warp a head, eight heads a CTA or, of many tokens, all
    const long long all = (long long)g->own.rows * g->own.heads;
    const bool many = most(plan.own) + most(plan.prefix) > JOIN_WARP_SPANS && all <= 148 * 8;
    const int heads = many ? 1 : all <= 148 * 64 ? JOIN_WARPS : g->own.heads;
    cfg.gridDim = dim3(g->own.rows, (g->own.heads + heads - 1) / heads);
    cfg.blockDim = dim3(32 * JOIN_WARPS);
    cfg.dynamicSmemBytes = 0;
    c = many ? cudaLaunchKernelEx(&cfg, k_prefix_join<T, HD, JOIN_WARPS>, pass[0], pass[1], heads)
             : cudaLaunchKernelEx(&cfg, k_prefix_join<T, HD, 1>, pass[0], pass[1], heads);
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
