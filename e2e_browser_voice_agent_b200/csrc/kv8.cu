// The paged 8-bit KV cache: block tables and slot maps from request lengths (h2c_kv8_plan), K and V rows into pages
// (h2c_kv8_append), and back out (h2c_kv8_read). The formulas are stated in include/h2cuda.h.
#include "ops.cuh"

#include <algorithm>
#include <climits>
#include <cstdlib>

namespace h2 {
namespace {

// ---------------------------------------------------------------- plan
//
// Three prefix sums over the requests (new tokens, pages taken, pages given back), then independent writes: one thread
// per new token, per page taken and per page given back finds its request by a search in the sums. Nothing that one
// thread writes is read by another (the tables' new entries are resolved through the ring, and the ring's new entries
// lie behind its tail), so every CTA forms the sums for itself from the 8 bytes per request and no grid-wide step is
// needed. Sums saturate at SUM_LIM, so that lengths without sense cannot wrap around to valid ones.
// Bound: latency (launch, two dependent reads, the sums); the bytes are 8 per request, token and page. 32 requests: 3.8 us;
// 2,048 requests with prompts among them: 9.1 us, most of it the sums, which every CTA forms again.
constexpr unsigned SUM_LIM = 0x3FFFFFFFu;
constexpr int PLAN_THREADS = 512;

__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b) { return min(a + b, SUM_LIM); }

struct PlanArgs {
  int n_req, page_log, table_cols, n_pages, max_tokens;
  const int *cached, *total;
  int *table, *ring;
  const long long* state;
  long long* state_out;
  int *kv_len, *q_start, *slot, *position, *status;
};

// the request whose range [sum[r], sum[r + 1]) holds i (sum[0] = 0, i < sum[n])
__device__ __forceinline__ int find_request(const unsigned* sum, int n, unsigned i) {
  int lo = 0, hi = n;  // sum[lo] <= i < sum[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sum[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) k_kv8_plan(const PlanArgs a) {
  extern __shared__ unsigned sums[];  // [3][n_req + 1]: new tokens, pages taken, pages given back
  const int n = a.n_req, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned* s_new = sums;
  unsigned* s_take = sums + n + 1;
  unsigned* s_back = sums + 2 * (n + 1);
  __shared__ unsigned part[3][PLAN_THREADS / 32];
  __shared__ int any_bad;
  if (tid == 0) {
    any_bad = 0;
    s_new[0] = s_take[0] = s_back[0] = 0;
  }
  const long long head = a.state[0], tail = a.state[1];
  const long long room = (long long)a.table_cols << a.page_log;
  const int round_up = (1 << a.page_log) - 1;
  __syncthreads();
  unsigned carry[3] = {0, 0, 0};
  for (int base = 0; base < n; base += PLAN_THREADS) {
    const int r = base + tid;
    unsigned v[3] = {0, 0, 0};
    if (r < n) {
      const int c = a.cached[r], t = a.total[r];
      if (c < 0 || t < 0 || c > room || t > room) {
        any_bad = 1;
      } else {
        const int have = (int)(((long long)c + round_up) >> a.page_log), want = (int)(((long long)t + round_up) >> a.page_log);
        v[0] = min((unsigned)max(t - c, 0), SUM_LIM);
        v[1] = min((unsigned)max(want - have, 0), SUM_LIM);
        v[2] = min((unsigned)max(have - want, 0), SUM_LIM);
      }
    }
#pragma unroll
    for (int k = 0; k < 3; k++) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned u = __shfl_up_sync(0xffffffffu, v[k], o);
        if (lane >= o) v[k] = sat_add(v[k], u);
      }
      if (lane == 31) part[k][warp] = v[k];
    }
    __syncthreads();
    if (warp < 3) {  // warp k sums the 16 warps' parts of sum k
      unsigned u = lane < PLAN_THREADS / 32 ? part[warp][lane] : 0u;
#pragma unroll
      for (int o = 1; o < PLAN_THREADS / 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, u, o);
        if (lane >= o) u = sat_add(u, x);
      }
      if (lane < PLAN_THREADS / 32) part[warp][lane] = u;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; k++) {
      const unsigned before = sat_add(carry[k], warp ? part[k][warp - 1] : 0u);
      if (r < n) sums[k * (n + 1) + r + 1] = sat_add(before, v[k]);
      carry[k] = sat_add(carry[k], part[k][PLAN_THREADS / 32 - 1]);
    }
    __syncthreads();
  }
  const unsigned n_new = carry[0], n_take = carry[1], n_back = carry[2];
  const long long avail = tail - head;
  const bool bad = any_bad || n_new > (unsigned)a.max_tokens || head < 0 || avail < 0 || avail + n_back > a.n_pages;
  const bool shortage = !bad && (long long)n_take > avail + n_back;
  const bool ok = !bad && !shortage;
  const int head_at = ok ? (int)(head % a.n_pages) : 0, tail_at = ok ? (int)(tail % a.n_pages) : 0;
  const int stride = gridDim.x * PLAN_THREADS, first = blockIdx.x * PLAN_THREADS + tid;

  auto pages_of = [&](int len) { return (int)(((long long)len + round_up) >> a.page_log); };
  auto given_back = [&](unsigned i) {  // the i-th page given back
    const int r = find_request(s_back, n, i);
    return a.table[(size_t)r * a.table_cols + pages_of(a.total[r]) + (i - s_back[r])];
  };
  auto taken = [&](unsigned i) {  // the i-th page taken
    if ((long long)i >= avail) return given_back(i - (unsigned)avail);
    unsigned at = head_at + i;
    if (at >= (unsigned)a.n_pages) at -= a.n_pages;
    return a.ring[at];
  };
  for (int t = first; t < a.max_tokens; t += stride) {
    int slot = -1, pos = -1;
    if (ok && (unsigned)t < n_new) {
      const int r = find_request(s_new, n, t), c = a.cached[r];
      pos = c + (t - (int)s_new[r]);
      const int have = pages_of(c), j = pos >> a.page_log;
      const int page = j < have ? a.table[(size_t)r * a.table_cols + j] : taken(s_take[r] + (j - have));
      slot = (page << a.page_log) + (pos & round_up);
    }
    a.slot[t] = slot;
    a.position[t] = pos;
  }
  if (ok) {
    for (unsigned i = first; i < n_take; i += stride) {
      const int r = find_request(s_take, n, i);
      a.table[(size_t)r * a.table_cols + pages_of(a.cached[r]) + (i - s_take[r])] = taken(i);
    }
    for (unsigned i = first; i < n_back; i += stride) {
      unsigned at = tail_at + i;
      if (at >= (unsigned)a.n_pages) at -= a.n_pages;
      a.ring[at] = given_back(i);
    }
  }
  for (int r = first; r <= n; r += stride) {
    a.q_start[r] = ok ? (int)s_new[r] : 0;
    if (r < n) {
      const int c = a.cached[r];
      a.kv_len[r] = ok ? a.total[r] : (c < 0 || c > room ? 0 : c);
    }
  }
  if (first == 0) {
    a.state_out[0] = head + (ok ? (long long)n_take : 0);
    a.state_out[1] = tail + (ok ? (long long)n_back : 0);
    a.status[0] = bad ? 2 : shortage ? 1 : 0;
    a.status[1] = shortage ? (int)(n_take - (avail + n_back)) : 0;
  }
}

// ---------------------------------------------------------------- append
//
// The rows that one call brings to one page form a run; its (K or V, head) part is quantized together because it shares
// a scale. grid.x covers windows of rows, grid.y K and V and the heads: a CTA takes the runs that start in its window
// (a run longer than the window reaches beyond it). Runs of up to SHORT rows (decode steps: one row) take a warp each,
// longer ones the whole CTA. A thread holds its values in registers between the maximum and the codes, so each input
// is read once. Bound: latency: one row, or a prompt's chain of slots, run, loads, maximum and codes, which 5 CTAs an SM (4: 21
// us, 6: 24) hide in part. 32 rows of 4 heads of 128, bfloat16: 4.5 us; 16,392 rows: 19.5 us, 50 MB at 2.6 TB/s. Float32 rows, which
// take twice the registers, 2 CTAs an SM: 4.2 and 31 us (4, which spill: 4.6 and 27; 200 prompts of 20 rows 11.8 and 12.7).
constexpr int APP_THREADS = 256, APP_WIN = 16, APP_MAX_WIN = 128, APP_SHORT = 2;
constexpr float SCALE_MIN = 0x1p-62f, SCALE_MAX = 0x1p63f;

struct AppendArgs {
  int8_t* kv;
  float* scale;
  int n_slots, page_log, kv_heads, rows, win;
  const void *k, *v;
  long long k_row, k_head, v_row, v_head;
  const int* slot;
};

// the scale after a run: a the largest magnitude (NaN or infinity: the page is lost), s0 the scale so far
__device__ __forceinline__ float grown_scale(float a, float s0, bool finite) {
  if (!finite || s0 != s0) return __int_as_float(0x7fc00000);
  if (s0 != 0.f && !(a > 127.5f * s0)) return s0;
  return fminf(fmaxf(fmaxf(__fdiv_rn(a, 127.f), 1.25f * s0), SCALE_MIN), SCALE_MAX);
}
__device__ __forceinline__ uint32_t codes_of(const float* x, float inv, bool clip) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[i] = __fmul_rn(x[i], inv);
    if (clip) v[i] = fminf(fmaxf(v[i], -127.f), 127.f);
  }
  return round_bytes(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = __fmul_rn((float)(int8_t)(w >> (8 * i)), ratio);
  return round_bytes(v[0], v[1], v[2], v[3]);
}

// One run of one (K or V, head) by the threads i0 = 0 .. NT-1 of a warp (NT = 32) or of the CTA; reduce() combines the
// largest magnitude bits over them. MAXU: units of 4 values that a thread keeps. A thread stays in one column of four.
template <class T, bool VEC, int HD, int NT, int MAXU, class R>
__device__ __forceinline__ void append_run(const T* src, long long row_stride, int len, int8_t* page, int off,
                                           float* scale, int i0, R reduce) {
  constexpr int UPR = HD / 4, RPS = NT / UPR;  // units per row, rows per step of all threads
  static_assert(NT % UPR == 0, "a thread's column must not change");
  const int row0 = i0 / UPR, col = (i0 % UPR) * 4;
  const float s0 = off == 0 ? 0.f : *scale;
  const T* p = src + row0 * row_stride + col;
  const long long step = RPS * row_stride;
  Raw4<T, VEC> v[MAXU];
#pragma unroll
  for (int k = 0; k < MAXU; k++)
    if (row0 + k * RPS < len) v[k].load(p + k * step);
  unsigned m = 0;
#pragma unroll
  for (int k = 0; k < MAXU; k++)
    if (row0 + k * RPS < len) m = v[k].merge(m);
  for (int r = row0 + MAXU * RPS; r < len; r += RPS) {  // (what does not fit the registers is read again below)
    Raw4<T, VEC> x;
    x.load(src + r * row_stride + col);
    m = x.merge(m);
  }
  m = reduce(Raw4<T, VEC>::bits(m));
  const bool finite = m < 0x7f800000u;
  const float s = grown_scale(__uint_as_float(m), s0, finite);
  const bool lost = s != s;
  const float inv = lost ? 0.f : __fdiv_rn(1.f, s);
  if (off && s != s0 && !lost) {
    const float ratio = __fdiv_rn(s0, s);
    for (int u = i0; u < off * UPR; u += NT) {
      uint32_t* w = reinterpret_cast<uint32_t*>(page) + u;
      *w = rescale4(*w, ratio);
    }
  }
  uint32_t* dst = reinterpret_cast<uint32_t*>(page + (size_t)off * HD) + i0;
  auto put = [&](bool clip) {
#pragma unroll
    for (int k = 0; k < MAXU; k++)
      if (row0 + k * RPS < len) {
        float x[4];
        v[k].get(x);
        dst[k * NT] = lost ? 0u : codes_of(x, inv, clip);
      }
    for (int r = row0 + MAXU * RPS; r < len; r += RPS) {
      Raw4<T, VEC> y;
      float x[4];
      y.load(src + r * row_stride + col);
      y.get(x);
      dst[(r - row0) * UPR] = lost ? 0u : codes_of(x, inv, clip);
    }
  };
  // (codes above 127 arise only where the largest magnitude is above 127 steps, and the scale did not grow for it)
  if (!lost && __fmul_rn(__uint_as_float(m), inv) > 127.25f) put(true);
  else put(false);
  if (i0 == 0 && s != s0) *scale = s;  // (also when s is NaN; every thread has read s0: reduce() synchronises them)
}

template <class T, bool VEC, int HD>
__global__ void __launch_bounds__(APP_THREADS, VEC && sizeof(T) == 2 ? 5 : 2) k_kv8_append(const AppendArgs a) {
  static_assert(APP_MAX_WIN + 128 <= APP_THREADS, "a thread per slot");
  __shared__ int run_row[APP_MAX_WIN], run_len[APP_MAX_WIN];
  __shared__ int slots[APP_MAX_WIN + 128];  // of the window and of the rows that its last run may reach
  __shared__ int n_runs;
  __shared__ unsigned red[APP_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = 1 << a.page_log;
  const int w0 = blockIdx.x * a.win;
  if (tid < a.win + 128) slots[tid] = w0 + tid < a.rows ? a.slot[w0 + tid] : -1;
  const int before = w0 > 0 && tid == 0 ? a.slot[w0 - 1] : -2;
  __syncthreads();
  if (warp == 0) {
    // a row starts a run unless the row before it is at the offset before its own in the same page
    const int last = __shfl_sync(0xffffffffu, before, 0);
    int n = 0;
    for (int t0 = 0; t0 < a.win; t0 += 32) {
      const int t = t0 + lane;
      bool lead = false;
      if (t < a.win) {
        const int s = slots[t];
        lead = s >= 0 && s < a.n_slots && ((s & (P - 1)) == 0 || (t ? slots[t - 1] : last) != s - 1);
      }
      const unsigned b = __ballot_sync(0xffffffffu, lead);
      if (lead) run_row[n + __popc(b & ((1u << lane) - 1))] = t;
      n += __popc(b);
    }
    if (lane == 0) n_runs = n;
  }
  __syncthreads();
  const int runs = n_runs;
  for (int i = warp; i < runs; i += APP_THREADS / 32) {  // run lengths, a warp per run
    const int t = run_row[i], s = slots[t], most = P - (s & (P - 1));
    int len = most;
    for (int b = 0; b < most; b += 32) {
      const bool in = b + lane < most && slots[t + b + lane] == s + b + lane;
      const unsigned in_all = __ballot_sync(0xffffffffu, in);
      if (in_all != 0xffffffffu) {
        len = min(most, b + __ffs(~in_all) - 1);
        break;
      }
    }
    if (lane == 0) run_len[i] = len;
  }
  __syncthreads();
  const int which = (int)blockIdx.y >= a.kv_heads, head = (int)blockIdx.y - which * a.kv_heads;
  const T* src = static_cast<const T*>(which ? a.v : a.k) + head * (which ? a.v_head : a.k_head);
  const long long row_stride = which ? a.v_row : a.k_row;
  auto page_of = [&](int s) {
    return a.kv + (((size_t)(s >> a.page_log) * 2 + which) * a.kv_heads + head) * ((size_t)P * HD);
  };
  auto scale_of = [&](int s) { return a.scale + ((size_t)(s >> a.page_log) * 2 + which) * a.kv_heads + head; };
  for (int i = warp; i < runs; i += APP_THREADS / 32) {
    if (run_len[i] > APP_SHORT) continue;
    const int t = w0 + run_row[i], s = slots[run_row[i]];
    append_run<T, VEC, HD, 32, APP_SHORT * HD / 128>(src + t * row_stride, row_stride, run_len[i], page_of(s),
                                                     s & (P - 1), scale_of(s), lane, [](unsigned m) {
                                                       m = __reduce_max_sync(0xffffffffu, m);
                                                       __syncwarp();  // (every lane has read the old scale)
                                                       return m;
                                                     });
  }
  for (int i = 0; i < runs; i++) {
    if (run_len[i] <= APP_SHORT) continue;
    const int t = w0 + run_row[i], s = slots[run_row[i]];
    append_run<T, VEC, HD, APP_THREADS, 8>(src + t * row_stride, row_stride, run_len[i], page_of(s), s & (P - 1),
                                           scale_of(s), tid, [&](unsigned m) {
                                             m = __reduce_max_sync(0xffffffffu, m);
                                             __syncthreads();  // (the run before is done with red[])
                                             if (lane == 0) red[warp] = m;
                                             __syncthreads();
                                             unsigned x = red[lane % (APP_THREADS / 32)];
                                             return __reduce_max_sync(0xffffffffu, x);
                                           });
  }
}

// ---------------------------------------------------------------- read

// A thread takes four consecutive codes of a row (blockDim.x threads across the row's K heads, then V heads) and goes from row to
// row: its 16 or 8 bytes of output join its neighbours'. Four rows in flight (16,392 rows of 4 heads of 128 to float32, 84 MB: 19
// us, 4.5 TB/s; one at a time 31). Bound: bandwidth; 32 rows: latency, 2.2 us.
template <class T>
__global__ void __launch_bounds__(256) k_kv8_read(const int8_t* __restrict__ kv, const float* __restrict__ scale, int n_slots,
                                                  int page_log, int kv_heads, int hd_log, const int* __restrict__ slot, int rows,
                                                  T* __restrict__ k_out, T* __restrict__ v_out) {
  constexpr int NR = 4;
  const int half = kv_heads << (hd_log - 2);  // units of four in a row's K
  const int page_mask = (1 << page_log) - 1, step = gridDim.x * blockDim.y;
  for (int u = threadIdx.x; u < 2 * half; u += blockDim.x) {
    const int which = u >= half, w = u - which * half;
    const int head = w >> (hd_log - 2), d = (w & ((1 << (hd_log - 2)) - 1)) * 4;
    T* out = (which ? v_out : k_out) + (head << hd_log) + d;
    const size_t row_len = (size_t)kv_heads << hd_log;
    for (int t0 = blockIdx.x * blockDim.y + threadIdx.y; t0 < rows; t0 += NR * step) {
      int sl[NR];
      uint32_t q[NR];
      float f[NR];
#pragma unroll
      for (int i = 0; i < NR; i++) {
        const int t = t0 + i * step;
        sl[i] = t < rows ? slot[t] : -1;
      }
#pragma unroll
      for (int i = 0; i < NR; i++) {
        q[i] = 0;
        f[i] = 0.f;
        if (sl[i] >= 0 && sl[i] < n_slots) {
          const size_t ph = ((size_t)(sl[i] >> page_log) * 2 + which) * kv_heads + head;
          q[i] = *reinterpret_cast<const uint32_t*>(kv + (((ph << page_log) + (sl[i] & page_mask)) << hd_log) + d);
          f[i] = scale[ph];
        }
      }
#pragma unroll
      for (int i = 0; i < NR; i++) {
        const int t = t0 + i * step;
        if (t >= rows) break;
        alignas(16) T o[4];
#pragma unroll
        for (int k = 0; k < 4; k++) o[k] = from_f<T>((float)(int8_t)(q[i] >> (8 * k)) * f[i]);
        if (sizeof(T) == 4) *reinterpret_cast<uint4*>(out + t * row_len) = *reinterpret_cast<const uint4*>(o);
        else *reinterpret_cast<uint2*>(out + t * row_len) = *reinterpret_cast<const uint2*>(o);
      }
    }
  }
}

int log2_of(int x) {
  int l = 0;
  while ((1 << l) < x) l++;
  return l;
}

int cache_ok(const char* who, const void* kv, const float* scale, int n_pages, int page_size, int kv_heads,
             int head_dim) {
  if (!kv || !scale) return op_error(H2C_ERR_INVALID, "%s: null cache", who);
  if ((uintptr_t)kv & 15) return op_error(H2C_ERR_INVALID, "%s: the cache must be 16-byte aligned", who);
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    return op_error(H2C_ERR_INVALID, "%s: page_size must be 16, 32, 64 or 128, not %d", who, page_size);
  if (head_dim != 64 && head_dim != 128)
    return op_error(H2C_ERR_INVALID, "%s: head_dim must be 64 or 128, not %d", who, head_dim);
  if (n_pages < 1 || (long long)n_pages * page_size > INT_MAX)
    return op_error(H2C_ERR_INVALID, "%s: n_pages %d out of range", who, n_pages);
  if (kv_heads < 1 || kv_heads > 4096) return op_error(H2C_ERR_INVALID, "%s: kv_heads %d out of range", who, kv_heads);
  return H2C_OK;
}

template <class T, bool VEC>
void launch_append(const AppendArgs& a, int head_dim, cudaStream_t st) {
  const dim3 grid((a.rows + a.win - 1) / a.win, 2 * a.kv_heads);
  if (head_dim == 64) k_kv8_append<T, VEC, 64><<<grid, APP_THREADS, 0, st>>>(a);
  else k_kv8_append<T, VEC, 128><<<grid, APP_THREADS, 0, st>>>(a);
}

}  // namespace
}  // namespace h2

using namespace h2;

extern "C" {

int h2c_kv8_plan(int32_t n_req, int32_t page_size, const int32_t* cached, const int32_t* total, int32_t* block_table,
                 int32_t table_cols, int32_t* free_ring, int32_t n_pages, const int64_t* free_state,
                 int64_t* free_state_out, int32_t* kv_len, int32_t* q_start, int32_t* slot, int32_t* position,
                 int32_t max_tokens, int32_t* status, void* stream) {
  const char* who = "h2c_kv8_plan";
  if (n_req < 0 || n_req > H2C_KV8_MAX_REQUESTS)
    return op_error(H2C_ERR_INVALID, "%s: n_req must be 0 to %d, not %d", who, H2C_KV8_MAX_REQUESTS, n_req);
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    return op_error(H2C_ERR_INVALID, "%s: page_size must be 16, 32, 64 or 128, not %d", who, page_size);
  if (!free_ring || !free_state || !free_state_out || !q_start || !status ||
      (n_req && (!cached || !total || !block_table || !kv_len)) || (max_tokens && (!slot || !position)))
    return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  if (free_state == free_state_out) return op_error(H2C_ERR_INVALID, "%s: free_state_out must not be free_state", who);
  if (n_pages < 1 || n_pages >= (int)SUM_LIM || (long long)n_pages * page_size > INT_MAX)
    return op_error(H2C_ERR_INVALID, "%s: n_pages %d out of range", who, n_pages);
  if (table_cols < 0 || (n_req && table_cols < 1))
    return op_error(H2C_ERR_INVALID, "%s: table_cols %d out of range", who, table_cols);
  if (max_tokens < 0 || max_tokens >= (int)SUM_LIM)
    return op_error(H2C_ERR_INVALID, "%s: max_tokens %d out of range", who, max_tokens);
  // (every CTA reads all of the inputs while others write)
  const uint64_t n4 = 4ull * n_req, t4 = 4ull * max_tokens;
  const OpRange in[] = {{"cached", cached, n4, 4}, {"total", total, n4, 4}, {"free_state", free_state, 16, 8}};
  const OpRange out[] = {{"block_table", block_table, n4 * table_cols, 4}, {"free_ring", free_ring, 4ull * n_pages, 4},
                         {"free_state_out", free_state_out, 16, 8}, {"kv_len", kv_len, n4, 4}, {"q_start", q_start, n4 + 4, 4},
                         {"slot", slot, t4, 4}, {"position", position, t4, 4}, {"status", status, 8, 4}};
  if (int rc = op_check_ranges(who, out, 8, in, 3)) return rc;
  static unsigned char done[OP_MAX_DEVICES];
  const int smem_max = 3 * (H2C_KV8_MAX_REQUESTS + 1) * (int)sizeof(unsigned);
  if (int rc = op_once(who, done, [&] {
        return cudaFuncSetAttribute(k_kv8_plan, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_max);
      }))
    return rc;
  PlanArgs a{n_req, log2_of(page_size), table_cols, n_pages, max_tokens, cached, total, block_table, free_ring,
             reinterpret_cast<const long long*>(free_state), reinterpret_cast<long long*>(free_state_out), kv_len, q_start,
             slot, position, status};
  const int work = std::max(max_tokens, n_req + 1);
  const int ctas = std::min(148, (work + PLAN_THREADS - 1) / PLAN_THREADS);
  k_kv8_plan<<<ctas, PLAN_THREADS, 3 * (n_req + 1) * sizeof(unsigned), (cudaStream_t)stream>>>(a);
  return op_launched(who);
}

int h2c_kv8_append(void* kv, float* kv_scale, int32_t n_pages, int32_t page_size, int32_t kv_heads, int32_t head_dim,
                   int32_t type, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row,
                   int64_t v_head, int32_t rows, const int32_t* slot, void* stream) {
  const char* who = "h2c_kv8_append";
  if (int rc = cache_ok(who, kv, kv_scale, n_pages, page_size, kv_heads, head_dim)) return rc;
  if (!op_type_ok(type)) return op_error(H2C_ERR_BAD_TYPE, "%s: element type %d", who, type);
  if (rows < 0 || rows > OP_MAX_ROWS) return op_error(H2C_ERR_INVALID, "%s: rows %d", who, rows);
  if (rows == 0) return H2C_OK;
  if (!k || !v || !slot) return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  const size_t es = op_elem_size(type);
  if (((uintptr_t)k | (uintptr_t)v) & (es - 1))
    return op_error(H2C_ERR_INVALID, "%s: k and v must be aligned to their elements", who);
  {
    auto range = [&](const char* name, const void* at, long long row, long long head) {  // of all rows and heads
      const long long r = (rows - 1LL) * row, h = (kv_heads - 1LL) * head;
      return OpRange{name, static_cast<const uint8_t*>(at) + (std::min(0LL, r) + std::min(0LL, h)) * (long long)es,
                     (uint64_t)(std::abs(r) + std::abs(h) + head_dim) * es};
    };
    const OpRange in[] = {range("k", k, k_row, k_head), range("v", v, v_row, v_head), {"slot", slot, 4ull * rows, 4}};
    const OpRange out[] = {{"kv", kv, 2ull * n_pages * kv_heads * page_size * head_dim},
                           {"kv_scale", kv_scale, 8ull * n_pages * kv_heads, 4}};
    if (int rc = op_check_ranges(who, out, 2, in, 3)) return rc;
  }
  // few rows (decode steps): windows of 16, so that few single rows wait in line for a warp; many: windows of a page, so that
  // every CTA of a prompt finds a run (16,392 rows into pages of 64: 19.6 us; with windows of 16, of which most begin no run, 29)
  const int win = (long long)(rows + APP_WIN - 1) / APP_WIN * 2 * kv_heads > 1184 ? std::max(APP_WIN, page_size) : APP_WIN;
  const AppendArgs a{static_cast<int8_t*>(kv), kv_scale, n_pages * page_size, log2_of(page_size), kv_heads, rows, win, k, v,
                     k_row, k_head, v_row, v_head, slot};
  // loads of four elements where every row and head starts at a multiple of four
  const bool vec = !(((uintptr_t)k | (uintptr_t)v) & (4 * es - 1)) && !((k_row | k_head | v_row | v_head) & 3);
  cudaStream_t st = (cudaStream_t)stream;
  if (type == H2C_TYPE_F32) vec ? launch_append<float, true>(a, head_dim, st) : launch_append<float, false>(a, head_dim, st);
  else if (type == H2C_TYPE_F16) vec ? launch_append<__half, true>(a, head_dim, st) : launch_append<__half, false>(a, head_dim, st);
  else vec ? launch_append<__nv_bfloat16, true>(a, head_dim, st) : launch_append<__nv_bfloat16, false>(a, head_dim, st);
  return op_launched(who);
}

int h2c_kv8_read(const void* kv, const float* kv_scale, int32_t n_pages, int32_t page_size, int32_t kv_heads,
                 int32_t head_dim, const int32_t* slot, int32_t rows, int32_t type, void* k_out, void* v_out,
                 void* stream) {
  const char* who = "h2c_kv8_read";
  if (int rc = cache_ok(who, kv, kv_scale, n_pages, page_size, kv_heads, head_dim)) return rc;
  if (!op_type_ok(type)) return op_error(H2C_ERR_BAD_TYPE, "%s: element type %d", who, type);
  if (rows < 0 || rows > OP_MAX_ROWS) return op_error(H2C_ERR_INVALID, "%s: rows %d", who, rows);
  if (rows == 0) return H2C_OK;
  if (!slot || !k_out || !v_out) return op_error(H2C_ERR_INVALID, "%s: null pointer", who);
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 15)
    return op_error(H2C_ERR_INVALID, "%s: k_out and v_out must be 16-byte aligned", who);
  const uint64_t bytes = (uint64_t)rows * kv_heads * head_dim * op_elem_size(type);
  const OpRange in[] = {{"kv", kv, 2ull * n_pages * kv_heads * page_size * head_dim},
                        {"kv_scale", kv_scale, 8ull * n_pages * kv_heads, 4}, {"slot", slot, 4ull * rows, 4}};
  const OpRange out[] = {{"k_out", k_out, bytes}, {"v_out", v_out, bytes}};
  if (int rc = op_check_ranges(who, out, 2, in, 3)) return rc;
  const int across = std::min(256, (2 * kv_heads * (head_dim / 4) + 31) / 32 * 32);
  const dim3 block(across, 256 / across);
  const int ctas = std::min((rows + (int)block.y - 1) / (int)block.y, 148 * 8);
  const int8_t* c = static_cast<const int8_t*>(kv);
  cudaStream_t st = (cudaStream_t)stream;
  const int n_slots = n_pages * page_size, pl = log2_of(page_size), hl = log2_of(head_dim);
  if (type == H2C_TYPE_F32)
    k_kv8_read<<<ctas, block, 0, st>>>(c, kv_scale, n_slots, pl, kv_heads, hl, slot, rows, (float*)k_out, (float*)v_out);
  else if (type == H2C_TYPE_F16)
    k_kv8_read<<<ctas, block, 0, st>>>(c, kv_scale, n_slots, pl, kv_heads, hl, slot, rows, (__half*)k_out, (__half*)v_out);
  else
    k_kv8_read<<<ctas, block, 0, st>>>(c, kv_scale, n_slots, pl, kv_heads, hl, slot, rows, (__nv_bfloat16*)k_out,
                                       (__nv_bfloat16*)v_out);
  return op_launched(who);
}

}  // extern "C"
