// Attention of requests that share prefixes over the paged 8-bit cache (h2c_kv8_prefix_attention; the formula is stated in
// include/h2cuda.h).
//
// Two passes and a join. All rows of a group of requests attend to the group's prefix together, as one request whose rows see every
// position: its keys are read once for 8 (k_att_rows) or 256 (k_att_prompt) rows of a kv head instead of once for each request.
// Each request attends to its own positions as in h2c_kv8_attention. Both passes leave (sum, maximum, weight) of each span of keys in
// the workspace, and k_prefix_join adds up what belongs to a row: the softmax over all its positions. The kernels are launched one
// behind the other without waiting for each other's end (programmatic dependent launch), those with tensor memory first; the
// single tokens' first CTAs take the SMs that they leave, and keep them until the kernel before is over (EndAfterTheOthers).
// Bound, 28 heads over 4 of 128, bfloat16: 256 single tokens with 16-2,000 positions of their own behind 16,385: 154 us, of which some 105 are
// k_att_prompt's rate on the prefix (28 row tiles of 257 tiles of keys, see there; with weights of one term 86); the own positions would take
// 54 alone, and 43 behind the prefix. Turns of 63 tokens of 26 requests in three groups, float16, 182 us: 160 that rate with the starts of
// some 540 CTAs of up to 22 tiles of keys, 20 the join of 65 MB (3.3 TB/s). 4 single tokens behind a prefix: 8.8 us, two launches and the
// latency of a span.
// Without the sharing, kv8.attention over tables that name the prefix reads its keys for each request (256 of 20-200 positions of their own
// behind 16,384: 731 us, 117 so), in one launch where there are few: it is the faster until the keys that it reads again are some 32 MB (32
// behind 640 18 us, 16 so; 8 behind 640 10 and 12).
// Where k_att_prompt takes part, its grid is a bound of the spans that its rows can have; CTAs without one look through the requests and end.
// With hundreds of groups of few rows these are thousands (1,024 groups of two single tokens behind 320 positions each: 660 us, 254 by
// kv8.attention over whole tables).
#include "kv8_rows.cuh"

namespace h2 {
namespace {

struct Pass {
  RowArgsOf<SharedArgs> ra;
  PromptArgsOf<SharedArgs> pa;
  int rows, prompt;  // whether k_att_rows, k_att_prompt take part
};

// k_att_rows of both passes in one launch: the groups, then the requests (4 sessions 9.1 us, 9.8 in two launches; 8 long requests 42 and
// 48; with a grid of both passes' largest axes, whose CTAs without work cost more than the launch, 54).
struct BothRows {
  RowArgsOf<SharedArgs> ra[2];
  unsigned across[2], first_own;  // CTAs that a request's rows take; the requests' first CTA
};
template <class T, int HD>
__global__ void __launch_bounds__(RW_WARPS * 32, HD == 128 ? 3 : 5) k_prefix_rows(const __grid_constant__ BothRows both) {
  const EndAfterTheOthers<true> end;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int own = blockIdx.x >= both.first_own;
  const unsigned at = own ? blockIdx.x - both.first_own : blockIdx.x, across = both.across[own], rz = at / across, n = both.ra[own].a.n_req;
  att_rows<T, HD>(both.ra[own], at - rz * across, rz % n, rz / n);
}

// Where the spans of a row lie: span s is row `first` + s * |`step`| of the sums and of the (m, l) of one of a pass's two kernels: of
// k_att_prompt where step is negative.
struct Parts {
  long long first;
  int used, step;  // spans; 0: the row is in no request (group)
};

// Quotients of numbers below 2^31 by multiplication: the joining kernel would spend most of its instructions on divisions else.
struct Divisor {
  unsigned d, magic;
  __device__ __forceinline__ explicit Divisor(int n) : d(n), magic(0xffffffffu / (unsigned)n) {}
  __device__ __forceinline__ Divisor(int n, unsigned m) : d(n), magic(m) {}
  __device__ __forceinline__ int quotient(int n) const {
    const unsigned q = __umulhi((unsigned)n, magic);  // (one too few at most)
    return (int)(q + ((unsigned)n - q * d >= d));
  }
  __device__ __forceinline__ int rounded_up(int n) const { return quotient(n + (int)d - 1); }
};

// The request (group) that has a row of q, and k_att_prompt's spans and rows of parts before its own, `blocks` tiles of keys each.
struct Owner {
  int r, n_all;      // r = -1: no request has it
  long long before, part;  // (part: its first row there)
  Request R;
  int tiles, spans;  // its row tiles in k_att_prompt, if it takes them, the spans of each and the tiles of keys of a span
  Divisor blocks;
};
// Those of rows t0 + i, for i = i0, i0 + step and so on below nt, to to[2 * i]. By whole warps, in one pass over the requests.
__device__ __forceinline__ void owners_of(const Pass& p, int t0, int i0, int step, int nt, Owner* to) {
  const SharedArgs& a = p.ra.a;
  const int lane = threadIdx.x & 31, blocks = p.prompt ? blocks_of_call(p.pa) : 1;
  for (int i = i0 + lane * step; i < nt; i += 32 * step) to[2 * i].r = -1;
  __syncwarp();
  long long before = 0, rows_before = 0;  // spans; rows of this lane's requests
  unsigned left = 0;  // rows to be found: bit m for i0 + m * step (JOIN_TOKENS at most)
  for (int i = i0, m = 0; i < nt; i += step, m++) left |= 1u << m;
  for (int base = 0; base < a.n_req && left; base += 32) {
    const int r = base + lane;
    int n = 0, n_all = 0, tiles = 0, spans = 1;
    long long rows = 0;
    Request R{0, 0, 0};
    if (r < a.n_req) {
      R = request_of(a, r, &n_all);
      if (p.prompt) {
        tiles = row_tiles_of(p.pa, R);
        spans = spans_of_len(p.pa, R.len, blocks);
        n = units_of(p.pa, tiles, spans);
        rows = part_rows_of(p.pa, R, tiles, spans);
      }
    }
    for (unsigned todo = left; todo; todo &= todo - 1) {
      const int m = __ffs(todo) - 1, i = i0 + m * step, t = t0 + i;
      const unsigned in = __ballot_sync(0xffffffffu, t >= R.first && t - R.first < R.n_q);
      if (!in) continue;
      const int l = __ffs(in) - 1;  // (of several, the first)
      const long long at = before + __reduce_add_sync(0xffffffffu, lane < l ? n : 0);
      const long long part = p.prompt ? sum_of_warp(rows_before + (lane < l ? rows : 0)) : 0;
      // (without room for its parts nothing of it was computed)
      if (lane == l && (!tiles || part + rows <= p.pa.part_rows))
        to[2 * i] = {r, n_all, at, part, R, tiles, spans, Divisor(tiles ? even_blocks(p.pa, R.len, spans) : 1)};
      left &= ~(1u << m);
    }
    before += __reduce_add_sync(0xffffffffu, n);
    rows_before += rows;
  }
}

// The parts of row t of q, which `o` has, and head h of kv head `head`'s group. row_blocks: blocks of k_att_rows' spans. (None where starts
// of requests without sense would lead beyond what was computed.)
__device__ __forceinline__ Parts parts_of(const Pass& p, const Divisor& row_blocks, const Owner& o, int t, int head, int h) {
  if (o.r < 0) return {0, 0, 0};
  const SharedArgs& a = p.ra.a;
  const Divisor group(a.group, a.group_magic);
  const int row = (t - o.R.first) * a.group + h;
  // the keys before the end of what the tile's last row sees
  auto end_of = [&](int last_row) {
    const int last = group.quotient(min(last_row, o.R.n_q * a.group - 1));
    return min(position_of(a, o.R, o.n_all, last) + 1, o.R.len);
  };
  if (o.tiles) {
    const int tile = row / PR_ROWS, n_blocks = (max(0, end_of(tile * PR_ROWS + PR_ROWS - 1)) + PR_KEYS - 1) / PR_KEYS;
    const long long unit = o.before + ((o.tiles - 1LL - tile) * a.kv_heads + head) * o.spans;
    if (unit + o.spans > p.pa.cap) return {0, 0, 0};
    const int n_rows = o.R.n_q * a.group;
    return {o.part + (long long)head * o.spans * n_rows + row, max(1, min(o.spans, o.blocks.rounded_up(n_blocks))), -n_rows};
  }
  const int tile = row / RW_ROWS, n_blocks = (max(0, end_of(tile * RW_ROWS + RW_ROWS - 1)) + RW_BLK - 1) / RW_BLK;
  if (tile >= p.ra.tiles) return {0, 0, 0};
  const long long unit = (((long long)o.r * a.kv_heads + head) * p.ra.tiles + tile) * p.ra.splits;
  return {unit * RW_ROWS + (row - tile * RW_ROWS), max(1, min(p.ra.splits, row_blocks.rounded_up(n_blocks))), RW_ROWS};
}
// The same for all lanes as lane j has them.
__device__ __forceinline__ Parts of_lane(const Parts& p, int j) {
  return {__shfl_sync(0xffffffffu, p.first, j), __shfl_sync(0xffffffffu, p.used, j), __shfl_sync(0xffffffffu, p.step, j)};
}

// A CTA takes `heads` heads (at most JOIN_WARPS) of `tokens` (at most JOIN_TOKENS) rows of q, L lanes (or NW = JOIN_WARPS warps, for one
// row) a head. What it looks up, whose row and request are shared by all warps and whose places by a warp's lanes, needs nothing of
// the passes and goes on while they end; the host makes no more CTAs than the SMs hold where it can.
constexpr int JOIN_TOKENS = 32, JOIN_PER_SM = 3, JOIN_CTAS = 148 * JOIN_PER_SM;
template <class T, int HD, int NW, int L>
__global__ void __launch_bounds__(32 * JOIN_WARPS, JOIN_PER_SM) k_prefix_join(const Pass prefix, const Pass own, int tokens, int heads) {
  constexpr int V = HD / L, UN = V > 4 ? 4 : 6;
  __shared__ float acc[NW][HD];
  __shared__ float2 acc_ml[NW];
  __shared__ __align__(16) uint8_t owner_s[JOIN_TOKENS * 2 * sizeof(Owner)];
  Owner(*owner)[2] = reinterpret_cast<Owner(*)[2]>(owner_s);
  const AttArgs& a = own.ra.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = NW > 1 ? warp : 0, t0 = blockIdx.x * tokens, ln = lane % L;
  const int h0 = blockIdx.y * heads, nh = min(heads, a.heads - h0), nt = min(tokens, a.rows - t0), n = nt * nh;
  // (every second warp the rows' requests, the others their prefixes' groups)
  owners_of(warp & 1 ? own : prefix, t0, warp >> 1, JOIN_WARPS / 2, nt, &owner[0][warp & 1]);
  __syncthreads();
  const Divisor by_heads(nh), by_group(a.group, a.group_magic);
  const Divisor prefix_row_blocks(max(1, prefix.ra.blocks)), own_row_blocks(max(1, own.ra.blocks));
  // lane j: of the warp's j-th row and head
  Parts o_of{0, 0, 0}, p_of{0, 0, 0};
  const int mine = NW > 1 ? lane : warp + lane * JOIN_WARPS;
  if (mine < n) {
    const int k_t = by_heads.quotient(mine), t = t0 + k_t, hq = h0 + mine - k_t * nh, head = by_group.quotient(hq), h = hq - head * a.group;
    o_of = parts_of(own, own_row_blocks, owner[k_t][1], t, head, h);
    p_of = parts_of(prefix, prefix_row_blocks, owner[k_t][0], t, head, h);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int j0 = 0; (NW > 1 ? j0 : warp + j0 * JOIN_WARPS) < n; j0 += 32 / L) {
    const int j = j0 + lane / L, i = NW > 1 ? j : warp + j * JOIN_WARPS;
    const Parts o = of_lane(o_of, j), p = of_lane(p_of, j);
    if (o.used == 0) continue;  // (a row of no request is not touched; nor is what lies past the warp's last)
    const int k_t = by_heads.quotient(i), t = t0 + k_t, hq = h0 + i - k_t * nh;
    const float* o_part = (o.step < 0 ? own.pa.part : own.ra.part) + o.first * HD + V * ln;
    const float2* o_ml = (o.step < 0 ? own.pa.ml : own.ra.ml) + o.first;
    const float* p_part = (p.step < 0 ? prefix.pa.part : prefix.ra.part) + p.first * HD + V * ln;
    const float2* p_ml = (p.step < 0 ? prefix.pa.ml : prefix.ra.ml) + p.first;
    const unsigned o_step = abs(o.step), p_step = abs(p.step);
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
          const size_t at = shared ? (size_t)s * p_step : (size_t)(s - p.used) * o_step;
          const float* src = (shared ? p_part : o_part) + at * HD;
          ml[k] = (shared ? p_ml : o_ml)[at];
          if (V == 2) {
            *reinterpret_cast<float2*>(x[k]) = *reinterpret_cast<const float2*>(src);
          } else {
#pragma unroll
            for (int j = 0; j < V; j += 4) *reinterpret_cast<float4*>(x[k] + j) = *reinterpret_cast<const float4*>(src + j);
          }
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
      for (int k = 0; k < V; k++) acc[w][V * ln + k] = v[k];
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
          for (int k = 0; k < V; k++) v[k] = fmaf(f, acc[n][V * ln + k], v[k]);
        }
      }
      __syncthreads();
    }
    if (w == 0) {
      const float inv = l != 0.f ? 1.f / l : 1.f;
      T* dst = static_cast<T*>(a.out) + (long long)t * a.out_row + hq * a.out_head + V * ln;
#pragma unroll
      for (int k = 0; k < V; k++) v[k] *= inv;
      if (V == 2) {
#pragma unroll
        for (int k = 0; k < V; k++) dst[k] = from_f<T>(v[k]);
      } else {
#pragma unroll
        for (int k = 0; k < V; k += 4) store4(dst + k, v + k, a.out_vec);
      }
      if (ln == 0 && a.lse)
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
    p.prefix = plan_work(&groups, true, true);
  }
  // (a CTA holds its place of spilled sums alone, whichever kernel it is of: one set of them)
  const size_t sums = (size_t)PR_SLOTS * PR_ROWS * g->own.head_dim * 4;
  p.bytes = p.own.bytes + p.prefix.bytes - (p.own.spill && p.prefix.spill ? sums : 0);
  return p;
}
// Whether a pass's counts fit their types: CTAs and rows of the workspace.
bool fits(const WorkPlan& p, long long kv_heads, long long requests) {
  return (long long)p.splits * p.tiles * RW_ROWS * kv_heads <= INT_MAX &&
         (p.tiles * kv_heads / RW_WARPS + 1) * requests * p.splits <= INT_MAX / 2 &&
         spans_at_most((long long)p.shape.tiles * kv_heads, p.p_keys) * PR_ROWS <= INT_MAX;
}

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
    float* p_part = take(p.p_rows, 1);
    pass[i].rows = p.rows;
    pass[i].prompt = p.prompt;
    pass[i].ra = {a, p.splits, p.blocks, p.tiles, p.max_rows, 0, part, nullptr};
    pass[i].pa = {a, p.min_rows, p.shape, p.p_keys, p.counted, p_part, nullptr, p.spill ? sums : nullptr, err, p.p_units, p.p_rows};
  }
  for (int i = 0; i < 2; i++) {
    const WorkPlan& p = i ? plan.own : plan.prefix;
    pass[i].ra.ml = reinterpret_cast<float2*>(at);
    at += p.units * RW_ROWS * 2;
    pass[i].pa.ml = reinterpret_cast<float2*>(at);
    at += (size_t)p.p_rows * 2;
  }

  static unsigned char done[OP_MAX_DEVICES];
  constexpr int p_smem = PromptCfg<T, HD, true>::SMEM, r_smem = RowSmem<HD>::BYTES;
  if (int rc = op_once(who, done, [] {
        const cudaError_t c = cudaFuncSetAttribute(k_att_prompt<T, HD, SharedArgs>, cudaFuncAttributeMaxDynamicSharedMemorySize, p_smem);
        return c != cudaSuccess ? c : cudaFuncSetAttribute(k_prefix_rows<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, r_smem);
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
    cfg.gridDim = dim3(p.p_units);
    cfg.blockDim = dim3(PR_THREADS);
    cfg.dynamicSmemBytes = p_smem;
    c = cudaLaunchKernelEx(&cfg, k_att_prompt<T, HD, SharedArgs>, pass[i].pa);
    cfg.numAttrs = 1;
  }
  if (c == cudaSuccess && (plan.own.rows || plan.prefix.rows)) {
    BothRows both{{pass[0].ra, pass[1].ra}, {1, 1}, 0};
    unsigned ctas = 0;
    for (int i = 0; i < 2; i++) {
      const WorkPlan& p = i ? plan.own : plan.prefix;
      both.first_own = i ? ctas : 0;
      if (!p.rows) continue;
      both.across[i] = (unsigned)(g->own.kv_heads * p.tiles + RW_WARPS - 1) / RW_WARPS;
      ctas += both.across[i] * pass[i].ra.a.n_req * p.splits;
    }
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(RW_WARPS * 32);
    cfg.dynamicSmemBytes = r_smem;
    c = cudaLaunchKernelEx(&cfg, k_prefix_rows<T, HD>, both);
    cfg.numAttrs = 1;
  }
  if (c == cudaSuccess) {
    auto most = [&](const WorkPlan& p) {  // spans of a row
      return std::max(p.rows ? p.splits : 0, p.prompt ? p.p_units / (p.shape.tiles * g->own.kv_heads) : 0);
    };
    // Eight warps a head where spans are many and rows few (28 heads over 4 of 128: 8 requests of up to 30,000 of their own behind 2,000
    // 42 us, 64 by a warp a head; 2 behind 300 10.2 and 11.5); else a warp a head, and no more CTAs than the SMs hold at a time, so that
    // all look up their places while the passes end (256 single tokens behind 16,385, weights of one term: 137 us, 140 with a CTA for each
    // token's eight heads).
    const bool many = most(plan.own) + most(plan.prefix) > JOIN_WARP_SPANS && (long long)g->own.rows * g->own.heads <= 148 * 8;
    const int heads = many ? 1 : std::min(JOIN_WARPS, g->own.heads);
    const long long ctas = (long long)g->own.rows * ((g->own.heads + heads - 1) / heads);
    const int tokens = many ? 1 : (int)std::min<long long>(JOIN_TOKENS, (ctas + JOIN_CTAS - 1) / JOIN_CTAS);
    cfg.gridDim = dim3((g->own.rows + tokens - 1) / tokens, (g->own.heads + heads - 1) / heads);
    cfg.blockDim = dim3(32 * JOIN_WARPS);
    cfg.dynamicSmemBytes = 0;
    // Where a warp has more than four rows and heads, two at a time: most instructions are then for both, and twice as much is on its way
    // (turns of 63 tokens of 26 requests 180 us, 184 one by one, of 200 484 and 511; 256 single tokens, two of whose rows and heads a
    // warp has, 135.5 and 134, when their weights had one term).
    const bool two = (long long)g->own.rows * g->own.heads > JOIN_CTAS * JOIN_WARPS * 4;
    c = many  ? cudaLaunchKernelEx(&cfg, k_prefix_join<T, HD, JOIN_WARPS, 32>, pass[0], pass[1], tokens, heads)
        : two ? cudaLaunchKernelEx(&cfg, k_prefix_join<T, HD, 1, 16>, pass[0], pass[1], tokens, heads)
              : cudaLaunchKernelEx(&cfg, k_prefix_join<T, HD, 1, 32>, pass[0], pass[1], tokens, heads);
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
  if (!fits(p.own, o->kv_heads, o->n_req) || !fits(p.prefix, o->kv_heads, g->n_groups) || (long long)o->rows * o->heads > INT_MAX)
    return op_error(H2C_ERR_INVALID, "%s: too many rows for one call", who);
  cudaStream_t st = (cudaStream_t)stream;
  if (o->type == H2C_TYPE_F32) return launch_typed<float>(who, p, g, st);
  if (o->type == H2C_TYPE_F16) return launch_typed<__half>(who, p, g, st);
  return launch_typed<__nv_bfloat16>(who, p, g, st);
}

}  // extern "C"
