// Attention over the paged 8-bit cache (h2c_kv8_attention; the formula is stated in include/h2cuda.h).
//
// Many queries (k_att_prompt): kv8_prompt.cuh. Few queries (k_att_rows): a CTA takes 8 rows (query, head of the kv head's
// group) of one request and kv head and one span of its keys; 4 warps take blocks of 16 keys in turn, each with its own
// running maximum, sum and output, joined at the end; up to 8 spans are joined by their cluster, more by a second kernel.
// * Tensor cores (mma.sync m16n8k16, float16 in, float32 sums): codes are integers up to 127 and exact in float16. The
//   16 rows of an operand tile hold 8 rows twice: a float16 term in rows 0-7 and the remainder in rows 8-15, for the
//   queries (scaled by a power of two per row) and for the softmax weights, so the products carry 22 bits, whatever the
//   element type, at the price of one. The group of 7 or fewer heads of a single token fills no more than 8 rows anyway.
// * The tensor cores cut off what a float32 sum cannot hold, so a sum kept there shrinks with every addition (16,000 keys in
//   one span: 6e-6 of the output, 131,072: 9e-5). Each block's product with V starts from zero and is added to the output
//   outside them, with rounding (1e-7 at any length).
// * The cache is the traffic: each lane copies its own 16-byte pieces of a block with cp.async into a ring that only it
//   reads, so the ring needs no barrier; the order of dimensions inside a product is free as long as both operands use
//   it, which lets a lane take 16 consecutive bytes of a key (QK) or of 4 keys (PV) without a transpose.
// * Bound: long histories (28 heads over 4, 128 wide, bfloat16; 8 requests of 69,224-131,072 tokens, 876 MB: 193 us, 4.5 TB/s)
//   not by the bytes that can be on their way (12 warps an SM, 3 blocks of 4 KB each), nor by DRAM (48% of its cycles), but by
//   what the warps wait for between them: shared memory (1.6 stalls an issue), fixed latencies (1.2), the matrix pipe (0.6);
//   the loads alone take 179 us in this ring. The time goes with the SMs' clock: 210 us in a run of seconds, in which the power
//   limit brings it to 1,750 MHz. Short ones by latency (32 requests of 120-4,096 tokens, 51 MB: 19 us and 5 to join; one of
//   641 tokens, 14 heads over 2, 64 wide, float32: 5.9 us, of which a launch is 2-3).
#include "kv8_att.cuh"
#include "kv8_prompt.cuh"

#include <algorithm>
#include <climits>
#include <cstdlib>

namespace h2 {
namespace {

constexpr int RW_WARPS = 4, RW_ROWS = 8, RW_BLK = 16, RW_STAGES = 4, RW_CLUSTER = 8;
struct RowArgs {
  AttArgs a;
  int splits, blocks, tiles;  // spans per row tile, blocks per span, row tiles per (request, kv head)
  int max_rows;               // requests of more rows are k_att_prompt's
  int cluster;                // the spans of a row tile are a cluster, which joins them itself
  float* part;                // (without clusters) [request][kv head][tile][span][8][HD] sums, then the same without HD for m and l
  float2* ml;
};

__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the product alone
__device__ __forceinline__ void mma16816_new(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

template <int HD>
struct RowSmem {
  static constexpr int STAGE = RW_BLK * HD * 2;                       // a warp's block: K, then V
  static constexpr int RING = RW_WARPS * RW_STAGES * STAGE;
  static constexpr int JOIN = (RW_WARPS + 1) * RW_ROWS * (HD + 2) * 4;  // (reuses the ring) the warps' parts, then the CTA's
  static constexpr int SCALES = RW_WARPS * 64 * 16;                   // KeyInfo of 64 blocks per warp
  static constexpr int BYTES = (RING > JOIN ? RING : JOIN) + SCALES;
};

// In a call that launches k_att_prompt too, k_att_rows follows it by programmatic dependent launch: it uses nothing of it and
// takes the SMs that its last CTAs leave (31 single tokens of 100-4,096 beside 2 prompts of 2,048: 134 -> 130 us). Its CTAs end after that one's, so that what follows on the stream finds both done. (They
// start when all of the kernel before have started, so none waits for a CTA that needs its place.)
struct EndAfterThePrompts {
  __device__ __forceinline__ ~EndAfterThePrompts() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
};

// (the CTAs an SM that shared memory has room for 128 wide, and registers 64 wide: without the bound the compiler spills for one more)
template <class T, int HD>
__global__ void __launch_bounds__(RW_WARPS * 32, HD == 128 ? 3 : 5) k_att_rows(const RowArgs ra) {
  const EndAfterThePrompts end;
  using S = RowSmem<HD>;
  constexpr int KC = HD / 64;   // 16-byte pieces of a key per lane
  constexpr int VB = HD / 8;    // bytes of a value row per lane (16 or 8)
  constexpr int NT = HD / 8;    // output tiles of 8 dimensions
  extern __shared__ __align__(16) uint8_t sm[];
  const AttArgs& a = ra.a;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (the joining kernel, which waits for this one's end)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x % ra.splits, th = blockIdx.x / ra.splits, head = th % a.kv_heads, tile = th / a.kv_heads;
  const int r = blockIdx.y;
  int n_all;
  const Request R = request_of(a, r, &n_all);
  const int row0 = tile * RW_ROWS, n_rows = R.n_q * a.group;
  if (row0 >= n_rows || n_rows > ra.max_rows) return;
  int lo, hi;
  key_range(a, R, n_all, row0 / a.group, min(row0 + RW_ROWS - 1, n_rows - 1) / a.group, &lo, &hi);
  const Span sp = spans_of(lo, hi, ra.splits, ra.blocks, RW_BLK);
  if (split >= sp.used && !ra.cluster) return;
  // (in a cluster a span without keys has its part in the join)
  const int b_begin = split * ra.blocks;
  const int b_end = split >= sp.used ? b_begin : split == sp.used - 1 ? sp.n_blocks : b_begin + ra.blocks;

  // ---- this lane's row: query dimensions 64j + 16c .. +15, as float16 terms
  const int row = row0 + g;
  const bool live = row < n_rows;
  int hq;
  const int tok = token_of(a, live ? row : row0, &hq);
  hq += head * a.group;
  const int pos = R.len - n_all + tok;               // its position, and the keys it may see: [first_key, pos]
  const int first_key = first_key_of(a, pos);
  uint32_t qa[KC * 4][4];
  float q_scale;  // what a product of codes is multiplied by: power of two of the row, softmax scale
  {
    float v[KC][16];
    const T* src = static_cast<const T*>(a.q) + (long long)(R.first + tok) * a.q_row + hq * a.q_head + 16 * c;
#pragma unroll
    for (int j = 0; j < KC; j++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (live) {
          if (a.q_vec) load4<true>(src + 64 * j + 4 * i, &v[j][4 * i]);
          else load4<false>(src + 64 * j + 4 * i, &v[j][4 * i]);
        } else {
          v[j][4 * i] = v[j][4 * i + 1] = v[j][4 * i + 2] = v[j][4 * i + 3] = 0.f;
        }
      }
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < KC; j++)
#pragma unroll
      for (int i = 0; i < 16; i++) m = max(m, __float_as_uint(v[j][i]) & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    // the largest magnitude to [2^13, 2^14): the remainders stay normal float16 numbers
    const int e = (int)(m >> 23);
    const int up = e == 255 || m == 0 ? 127 : min(253, 267 - e);
    const float mul = __int_as_float(up << 23);
    q_scale = __int_as_float((254 - up) << 23) * a.scale_log2;
#pragma unroll
    for (int j = 0; j < KC; j++)
#pragma unroll
      for (int s = 0; s < 4; s++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float x0 = v[j][4 * s + 2 * h] * mul, x1 = v[j][4 * s + 2 * h + 1] * mul;
          const __half2 t = __floats2half2_rn(x0, x1);
          qa[4 * j + s][2 * h] = *reinterpret_cast<const uint32_t*>(&t);
          qa[4 * j + s][2 * h + 1] = pack_half2(x0 - __low2float(t), x1 - __high2float(t));
        }
  }

  unsigned long long o[NT];  // (two dimensions)
#pragma unroll
  for (int t = 0; t < NT; t++) o[t] = 0;
  float m_run = -INFINITY, l_run = 0.f;

  // ---- the warp's blocks: b_begin + warp + 4 it
  const int n_it = max(0, (b_end - b_begin - warp + RW_WARPS - 1) / RW_WARPS);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm) + warp * RW_STAGES * S::STAGE;
  KeyInfo* info = reinterpret_cast<KeyInfo*>(sm + S::BYTES - S::SCALES) + warp * 64;
  const int P = 1 << a.page_log;
  const size_t head_bytes = (size_t)P * HD;
  const size_t v_off = a.kv_heads * head_bytes;
  const int8_t* k_lane = a.kv + head * head_bytes + g * HD + 16 * c;              // this lane's pieces of a block at offset 0
  const int8_t* v_lane = a.kv + head * head_bytes + v_off + 2 * c * HD + VB * g;
  const uint32_t k_dst = ring + lane * 16, v_dst = ring + RW_BLK * HD + lane * VB;
  unsigned long long i_off = 0;
  auto issue = [&](int it) {
    if (it < n_it) {
      if ((it & 31) == 0) {  // places and scales of the next 32 blocks, one per lane
        const int b = b_begin + warp + RW_WARPS * (it + lane);
        if (b < b_end) {
          const int key = sp.first + b * RW_BLK;
          int pg = a.table[(size_t)r * a.table_cols + (key >> a.page_log)];
          pg = (unsigned)pg < (unsigned)a.n_pages ? pg : 0;
          i_off = (size_t)pg * 2 * v_off + (key & (P - 1)) * HD;
          const float* s = a.kv_scale + (size_t)pg * 2 * a.kv_heads + head;
          KeyInfo ki;
          ki.k = s[0];
          split_scale(s[a.kv_heads], &ki.e, &ki.mant, &ki.inv);
          info[(it + lane) & 63] = ki;  // (the block that was there 64 turns before is done with)
        }
      }
      const size_t off = __shfl_sync(0xffffffffu, i_off, it & 31);
      const uint32_t st = (it % RW_STAGES) * S::STAGE;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int j = 0; j < KC; j++) copy_async<16>(k_dst + st + (t * KC + j) * 512, k_lane + off + 8 * t * HD + 64 * j);
#pragma unroll
      for (int i = 0; i < 4; i++)
        copy_async<VB>(v_dst + st + i * 32 * VB, v_lane + off + ((i & 1) + 8 * (i >> 1)) * HD);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // blocks that every row of the tile sees whole need no masks
  const int clear_from = __reduce_max_sync(0xffffffffu, live ? first_key : 0);
  const int clear_to = __reduce_min_sync(0xffffffffu, live ? pos : INT_MAX);
#pragma unroll
  for (int it = 0; it < RW_STAGES - 1; it++) issue(it);

  for (int it = 0; it < n_it; it++) {
    asm volatile("cp.async.wait_group %0;" ::"n"(RW_STAGES - 2) : "memory");
    __syncwarp();
    const int stage = it % RW_STAGES;
    const uint8_t* kst = sm + warp * RW_STAGES * S::STAGE + stage * S::STAGE + lane * 16;
    const uint8_t* vst = sm + warp * RW_STAGES * S::STAGE + stage * S::STAGE + RW_BLK * HD + lane * VB;
    const KeyInfo ki = info[it & 63];
    const int blk0 = sp.first + (b_begin + warp + RW_WARPS * it) * RW_BLK, key0 = blk0 + 2 * c;
    // scores of 8 rows x 16 keys: this lane has keys key0, key0 + 1 (tile 0), key0 + 8, key0 + 9 (tile 1) of its row
    float y[4];
    const float f = q_scale * ki.k;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KC; j++) {
        const uint4 w4 = *reinterpret_cast<const uint4*>(kst + (t * KC + j) * 512);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int s = 0; s < 4; s++) {
          const uint32_t u = w[s] ^ 0x80808080u;
          mma16816(d, qa[4 * j + s][0], qa[4 * j + s][1], qa[4 * j + s][2], qa[4 * j + s][3],
                   half2_of(__byte_perm(u, 0x64646464u, 0x4140)), half2_of(__byte_perm(u, 0x64646464u, 0x4342)));
        }
      }
      y[2 * t] = fmaf(d[0] + d[2], f, ki.e);
      y[2 * t + 1] = fmaf(d[1] + d[3], f, ki.e);
    }
    if (blk0 < clear_from || blk0 + RW_BLK - 1 > clear_to) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int key = key0 + 8 * (i >> 1) + (i & 1);
        if (!(live && key <= pos && key >= first_key)) y[i] = -INFINITY;
      }
    }
    float mx = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
    if (__any_sync(0xffffffffu, mx > m_run + M_SLACK)) {
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = mx > m_run + M_SLACK ? mx : m_run;  // (a row's result does not depend on its neighbours)
      const float f_old = m_new == m_run ? 1.f : m_run == -INFINITY ? 0.f : exp2_fast(m_run - m_new);
      m_run = m_new;
      l_run *= f_old;
#pragma unroll
      for (int t = 0; t < NT; t++) o[t] = mul2(o[t], pair(f_old, f_old));
    }
    const float m_use = (m_run == -INFINITY ? 0.f : m_run) - P_SHIFT;
    float p[4], rest[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float w = exp2_fast(y[i] - m_use);
      l_run = fmaf(w, ki.inv, l_run);
      p[i] = w * ki.mant;
    }
    const uint32_t a0 = pack_half2(p[0], p[1]), a2 = pack_half2(p[2], p[3]);
    {
      const __half2 h0 = *reinterpret_cast<const __half2*>(&a0), h1 = *reinterpret_cast<const __half2*>(&a2);
      rest[0] = p[0] - __low2float(h0); rest[1] = p[1] - __high2float(h0);
      rest[2] = p[2] - __low2float(h1); rest[3] = p[3] - __high2float(h1);
    }
    const uint32_t a1 = pack_half2(rest[0], rest[1]), a3 = pack_half2(rest[2], rest[3]);
    // values: 4 keys x VB consecutive dimensions; tile t of the output takes dimension VB * n + t at column n
    uint32_t vw[4][VB / 4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (VB == 16) *reinterpret_cast<uint4*>(vw[i]) = *reinterpret_cast<const uint4*>(vst + i * 32 * VB);
      else *reinterpret_cast<uint2*>(vw[i]) = *reinterpret_cast<const uint2*>(vst + i * 32 * VB);
    }
#pragma unroll
    for (int w = 0; w < VB / 4; w++) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; i++) u[i] = vw[i][w] ^ 0x80808080u;
#pragma unroll
      for (int hpair = 0; hpair < 2; hpair++) {
        const uint32_t k01 = __byte_perm(u[0], u[1], hpair ? 0x7362 : 0x5140);
        const uint32_t k23 = __byte_perm(u[2], u[3], hpair ? 0x7362 : 0x5140);
        float d0[4], d1[4];
        mma16816_new(d0, a0, a1, a2, a3, half2_of(__byte_perm(k01, 0x64646464u, 0x4140)),
                     half2_of(__byte_perm(k23, 0x64646464u, 0x4140)));
        mma16816_new(d1, a0, a1, a2, a3, half2_of(__byte_perm(k01, 0x64646464u, 0x4342)),
                     half2_of(__byte_perm(k23, 0x64646464u, 0x4342)));
        unsigned long long* sum = &o[4 * w + 2 * hpair];
        sum[0] = add2(sum[0], add2(pair(d0[0], d0[1]), pair(d0[2], d0[3])));
        sum[1] = add2(sum[1], add2(pair(d1[0], d1[1]), pair(d1[2], d1[3])));
      }
    }
    issue(it + RW_STAGES - 1);
  }
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);

  // ---- join the warps: [warp][8][HD] sums, [warp][8] maxima, [warp][8] sums of weights
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* js = reinterpret_cast<float*>(sm);
  float* jm = js + RW_WARPS * RW_ROWS * HD;
  float* jl = jm + RW_WARPS * RW_ROWS;
  if (c == 0) {
    jm[warp * RW_ROWS + g] = m_run;
    jl[warp * RW_ROWS + g] = l_run;
  }
#pragma unroll
  for (int t = 0; t < NT; t += 4) {
    float v[4][2];
#pragma unroll
    for (int i = 0; i < 4; i++) unpair(o[t + i], &v[i][0], &v[i][1]);
#pragma unroll
    for (int i = 0; i < 2; i++)
      *reinterpret_cast<float4*>(js + (warp * RW_ROWS + g) * HD + VB * (2 * c + i) + t) =
          make_float4(v[0][i], v[1][i], v[2][i], v[3][i]);
  }
  __syncthreads();
  constexpr int TPR = RW_WARPS * 32 / RW_ROWS;  // threads per row
  const int jr = threadIdx.x / TPR, jt = threadIdx.x % TPR, orow = row0 + jr;
  float mm = -INFINITY, ll = 0.f, fw[RW_WARPS];
#pragma unroll
  for (int w = 0; w < RW_WARPS; w++) mm = fmaxf(mm, jm[w * RW_ROWS + jr]);
#pragma unroll
  for (int w = 0; w < RW_WARPS; w++) {
    const float mw = jm[w * RW_ROWS + jr];
    fw[w] = mw == -INFINITY ? 0.f : exp2_fast(mw - mm);
    ll += fw[w] * jl[w * RW_ROWS + jr];
  }
  const size_t unit = (((size_t)r * a.kv_heads + head) * ra.tiles + tile) * ra.splits + split;
  const bool whole = sp.used == 1 && !ra.cluster;
  const float inv = whole && ll != 0.f ? 1.f / ll : 1.f;
  int oh;
  const int otok = token_of(a, orow, &oh);
  oh += head * a.group;
  float* cs = jl + RW_WARPS * RW_ROWS;  // (cluster) this CTA's rows: sums, then (m, l) pairs
#pragma unroll
  for (int k = 0; k < HD / 4 / TPR; k++) {
    const int d = (jt + k * TPR) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < RW_WARPS; w++) {
      const float4 x = *reinterpret_cast<const float4*>(js + (w * RW_ROWS + jr) * HD + d);
      v[0] += fw[w] * x.x; v[1] += fw[w] * x.y; v[2] += fw[w] * x.z; v[3] += fw[w] * x.w;
    }
    if (ra.cluster) {
      *reinterpret_cast<float4*>(cs + jr * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (orow >= n_rows) {
    } else if (whole) {
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] *= inv;
      store4(static_cast<T*>(a.out) + (long long)(R.first + otok) * a.out_row + oh * a.out_head + d, v, a.out_vec);
    } else {
      *reinterpret_cast<float4*>(ra.part + (unit * RW_ROWS + jr) * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  if (jt == 0) {
    if (ra.cluster) reinterpret_cast<float2*>(cs + RW_ROWS * HD)[jr] = make_float2(mm, ll);
    else if (orow >= n_rows) {
    } else if (!whole) ra.ml[unit * RW_ROWS + jr] = make_float2(mm, ll);
    else if (a.lse)
      a.lse[(size_t)(R.first + otok) * a.heads + oh] =
          ll == 0.f ? -INFINITY : 0.69314718055994531f * (log2f(ll) + mm - P_SHIFT);
  }
  if (!ra.cluster) return;
  __syncwarp();

  // ---- the cluster's spans, each CTA a share of the rows' pieces of four dimensions, through distributed shared memory
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const uint32_t c_at = (uint32_t)__cvta_generic_to_shared(cs);
  for (int u = split * RW_WARPS * 32 + threadIdx.x; u < RW_ROWS * HD / 4; u += ra.splits * RW_WARPS * 32) {
    const int cr = u / (HD / 4), d = (u % (HD / 4)) * 4, row_c = row0 + cr;
    if (row_c >= n_rows) break;
    float2 ml[RW_CLUSTER];
    float4 x[RW_CLUSTER];
#pragma unroll
    for (int k = 0; k < RW_CLUSTER; k++)
      if (k < ra.splits) {
        uint32_t at;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(c_at), "r"(k));
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                     : "=f"(ml[k].x), "=f"(ml[k].y)
                     : "r"(at + RW_ROWS * HD * 4 + cr * 8)
                     : "memory");
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(x[k].x), "=f"(x[k].y), "=f"(x[k].z), "=f"(x[k].w)
                     : "r"(at + (cr * HD + d) * 4)
                     : "memory");
      }
    float m = -INFINITY, l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < RW_CLUSTER; k++)
      if (k < ra.splits) m = fmaxf(m, ml[k].x);
#pragma unroll
    for (int k = 0; k < RW_CLUSTER; k++)
      if (k < ra.splits) {
        const float f = ml[k].x == -INFINITY ? 0.f : exp2_fast(ml[k].x - m);
        l += f * ml[k].y;
        v[0] += f * x[k].x; v[1] += f * x[k].y; v[2] += f * x[k].z; v[3] += f * x[k].w;
      }
    const float c_inv = l != 0.f ? 1.f / l : 1.f;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] *= c_inv;
    int ch;
    const int ctok = token_of(a, row_c, &ch);
    ch += head * a.group;
    store4(static_cast<T*>(a.out) + (long long)(R.first + ctok) * a.out_row + ch * a.out_head + d, v, a.out_vec);
    if (d == 0 && a.lse)
      a.lse[(size_t)(R.first + ctok) * a.heads + ch] = l == 0.f ? -INFINITY : 0.69314718055994531f * (log2f(l) + m - P_SHIFT);
  }
  __syncwarp();
  // (the others may still read this CTA's part)
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Joins the spans of one row: the weights of span s relative to the common maximum are 2^(m_s - m). Span s of the row has
// its sums at part + s * part_step and its (m, l) at ml + s * ml_step. By a warp for few spans (8 rows a CTA), by 8 warps for many,
// each taking every 8th span: `n_warps`, `w` the warp's turn; the order of the additions goes by the spans' number alone. A warp up
// to 12 spans (a chunk of 256 on 4,096, 10 spans: 30 us, 41 by 8 warps, 33 with room for 24 in a warp's registers; 32 single tokens,
// 7 spans: 19, 21, 19; a chunk of 100 on 16,000, 18 spans: 43 by 8 warps, 39 by one with room for 24).
constexpr int JOIN_WARPS = 8, JOIN_WARP_SPANS = 12;
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
inline unsigned join_ctas(long long rows, int splits) {
  return (unsigned)(splits <= JOIN_WARP_SPANS ? (rows + JOIN_WARPS - 1) / JOIN_WARPS : rows);
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

// k_att_rows reads a request's keys again for every 8 rows and starts in half the time; k_att_prompt takes 256 rows at once. A call
// that visits few keys altogether (row tiles of 8 x keys, as many as max_q and max_kv allow; a tile's start counts as 256 keys)
// is k_att_rows' whole: up to 2^17 visits 128 wide, 2^19 64 wide. In a call of more, each CTA looks at its request's rows on the
// device: up to 16 (32) are k_att_rows', others k_att_prompt's, and the host launches the one kernel or both by max_q.
// Measured, k_att_rows and k_att_prompt in us. bfloat16 128 wide, 28 heads over 4, one request of 4,000 keys: 35 rows (80,000
// visits) 14 and 21, 70 rows (144,000) 21 and 22, 126 rows (256,000) 31 and 23; of 16,000, 35 rows (320,000) 32 and 26. Several
// requests, whose spans are longer, cross later: 2 of 4,000 keys, 35 rows (160,000) 24 and 32, 70 rows (288,000) 36 and 33, 252 rows
// (1,024,000) 67 and 38. float32: 70 rows of one 21 and 26, 126 rows 31 and 28. 64 wide, 14 over 2, bfloat16 and float32: one of
// 4,000 keys, 504 rows (504,000) 23, 22 and 27, 1,008 rows (1,008,000) 36, 27 and 32; of 16,000, 126 rows (512,000) 24, 18 and 22;
// 8 of 4,000 keys, 63 rows (512,000) 23, 28 and 34, 126 rows (1,024,000) 35, 29 and 35.
struct WorkPlan {
  bool rows, prompt, cluster, counted;
  int max_rows, splits, blocks, tiles;         // k_att_rows
  int min_rows, p_keys, p_units;               // k_att_prompt (see PromptArgs; p_units also without counting)
  PromptShape shape;
  unsigned p_join;                             // CTAs of its joining kernel, 0 without one
  size_t units;                                // row tiles x spans in the workspace
  bool spill;                                  // its sums go through the workspace
  size_t bytes;
};
// Tiles of keys after which k_att_prompt's sums go to the workspace.
int spill_after(int type, int head_dim) {
  if (head_dim == 64) return INT_MAX;
  return type == H2C_TYPE_F32 ? PromptCfg<float, 128>::FOLD
         : type == H2C_TYPE_F16 ? PromptCfg<__half, 128>::FOLD
                                : PromptCfg<__nv_bfloat16, 128>::FOLD;
}
WorkPlan plan_work(const h2c_kv8_attention_args* g) {
  WorkPlan p = {};
  const long long group = g->heads / g->kv_heads, most_rows = g->max_q * group;
  long long keys = g->max_kv;
  if (g->window > 0) keys = std::min(keys, (long long)g->window + g->max_q);
  const long long visits = (most_rows + RW_ROWS - 1) / RW_ROWS * g->n_req * g->kv_heads * std::max(keys, 256LL);
  const int few = g->head_dim == 64 ? 32 : 16;
  p.prompt = most_rows > few && visits > (g->head_dim == 64 ? 1 << 19 : 1 << 17);
  p.rows = !p.prompt || g->n_req > 1;
  if (p.rows) {
    p.max_rows = p.prompt ? few : INT_MAX;
    p.tiles = (int)((std::min<long long>(most_rows, p.max_rows) + RW_ROWS - 1) / RW_ROWS);
    // spans: enough CTAs for two waves of three per SM (28 heads over 4, 128 wide, bfloat16; 888, half and one and a half times as
    // many in us: 32 requests of 100-4,096 keys 19, 23 and 19; 64 of them 33, 44 and 35; 2 of 30,000-60,000 42, 38 and 47; 8 of
    // 60,000-131,072 175, 176 and 164; 32 of 4,000-16,000 89, 81 and 75). Up to 8 are one cluster, whose join costs little: spans of 128 keys (2
    // blocks per warp) or more. More of them, for few rows over long histories, leave their parts in the workspace for a
    // second kernel: spans of 256 keys or more, below which a span's start-up costs more than it shares out
    const long long groups = (long long)g->n_req * g->kv_heads * p.tiles, want = (888 + groups - 1) / groups;
    const int n_blocks = (int)((keys + RW_BLK - 1) / RW_BLK) + (g->window > 0 ? 1 : 0);
    p.cluster = groups * RW_CLUSTER <= 444 && n_blocks / 16 <= RW_CLUSTER;
    p.splits = (int)std::max(1LL, p.cluster ? std::min<long long>({(long long)RW_CLUSTER, want, (n_blocks + 7LL) / 8})
                                            : std::min<long long>(want, n_blocks / 16));
    p.blocks = std::max(RW_WARPS, ((n_blocks + p.splits - 1) / p.splits + RW_WARPS - 1) / RW_WARPS * RW_WARPS);
    p.splits = std::max(1, (n_blocks + p.blocks - 1) / p.blocks);
    p.cluster = p.cluster && p.splits > 1;
    p.units = p.splits > 1 && !p.cluster ? (size_t)groups * p.splits : 0;
  }
  if (p.prompt) {
    p.min_rows = p.rows ? few + 1 : 0;
    const int tiles = (int)std::min<long long>({(long long)g->n_req * ((most_rows + PR_ROWS - 1) / PR_ROWS),
                                                (long long)g->rows * group / PR_ROWS + g->n_req, (long long)INT_MAX / g->kv_heads});
    p.p_keys = (int)((keys + PR_KEYS - 1) / PR_KEYS) + (g->window > 0 ? 1 : 0);
    p.shape = prompt_shape(tiles, g->kv_heads, p.p_keys, g->n_req == 1 ? 148 : 0, 4);
    if (g->n_req == 1) {
      p.p_units = p.shape.splits > 1 ? tiles * g->kv_heads * p.shape.splits : 0;
      p.p_join = p.p_units ? join_ctas((long long)tiles * g->kv_heads * PR_ROWS, p.shape.splits) : 0;
    } else if (g->n_req <= 256 && (long long)g->rows * group / PR_ROWS * g->kv_heads <= 74 && g->kv_heads <= 74 && p.p_keys >= 16) {
      // all rows together leave half of the SMs or more idle: each CTA counts. A chunk of 256 on 4,096 beside 31, 127, 255 and 511 single
      // tokens (28 heads over 4 of 128, bfloat16): 72, 97, 138 and 270 us, without the count 121, 137, 176 and 270, so up to 256 requests.
      // On histories of 16 tiles of keys or more: 128 beside 7 on 768, 1,024 and 1,536 tokens: 36, 40 and 41, without 31, 37 and 47
      p.counted = true;
      p.p_units = 148;
      // rows that the joining kernel may find: of one in 2 .. JOIN_WARP_SPANS units (a warp each), or in more (a CTA each)
      const long long groups = (long long)tiles * g->kv_heads;
      p.p_join = std::max(join_ctas(std::min(groups, 148LL / 2) * PR_ROWS, 2),
                          join_ctas(std::min(groups, 148LL / (JOIN_WARP_SPANS + 1)) * PR_ROWS, JOIN_WARP_SPANS + 1));
    }
  }
  // whether a row tile can have more tiles of keys than a sum may take, whatever max_kv says
  const long long room = (long long)g->table_cols * g->page_size;
  const long long most_keys = g->window > 0 ? std::min(room, (long long)g->window + PR_ROWS + 16) : room;
  p.spill = p.prompt && (most_keys + PR_KEYS - 1) / PR_KEYS + 1 > spill_after(g->type, g->head_dim);
  p.bytes = (p.units * RW_ROWS + (size_t)p.p_units * PR_ROWS) * ((size_t)g->head_dim * 4 + 8) +
            (p.spill ? (size_t)PR_SLOTS * PR_ROWS * g->head_dim * 4 : 0);
  return p;
}

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
          return cudaFuncSetAttribute(k_att_prompt<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        }))
      return rc;
    k_att_prompt<T, HD><<<std::max(p.shape.tiles * a.kv_heads, p.p_units), PR_THREADS, smem, st>>>(pa);
    if (int rc = op_launched(who)) return rc;
  }
  if (p.rows) {
    static unsigned char done[OP_MAX_DEVICES];
    constexpr int smem = RowSmem<HD>::BYTES;
    if (int rc = op_once(who, done, [] {
          return cudaFuncSetAttribute(k_att_rows<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
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
    c = cudaLaunchKernelEx(&cfg, k_att_rows<T, HD>, ra);
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

int check_args(const char* who, const h2c_kv8_attention_args* g) {
  if (!g) return op_error(H2C_ERR_INVALID, "%s: null arguments", who);
  if (g->page_size != 16 && g->page_size != 32 && g->page_size != 64 && g->page_size != 128)
    return op_error(H2C_ERR_INVALID, "%s: page_size must be 16, 32, 64 or 128, not %d", who, g->page_size);
  if (g->head_dim != 64 && g->head_dim != 128)
    return op_error(H2C_ERR_INVALID, "%s: head_dim must be 64 or 128, not %d", who, g->head_dim);
  if (g->n_pages < 1 || (long long)g->n_pages * g->page_size > INT_MAX)
    return op_error(H2C_ERR_INVALID, "%s: n_pages %d out of range", who, g->n_pages);
  if (g->kv_heads < 1 || g->kv_heads > 4096 || g->heads < g->kv_heads || g->heads > 65536 || g->heads % g->kv_heads)
    return op_error(H2C_ERR_INVALID, "%s: heads (%d) must be a multiple of kv_heads (%d)", who, g->heads, g->kv_heads);
  if (!op_type_ok(g->type)) return op_error(H2C_ERR_BAD_TYPE, "%s: element type %d", who, g->type);
  if (g->n_req < 0 || g->n_req > H2C_KV8_MAX_REQUESTS)
    return op_error(H2C_ERR_INVALID, "%s: n_req must be 0 to %d, not %d", who, H2C_KV8_MAX_REQUESTS, g->n_req);
  if (g->rows < 0 || g->max_q < 0 || g->max_kv < 0 || g->window < 0 || g->table_cols < 0)
    return op_error(H2C_ERR_INVALID, "%s: a size is negative", who);
  if (g->rows > OP_MAX_ROWS) return op_error(H2C_ERR_INVALID, "%s: rows %d out of range", who, g->rows);
  if ((long long)g->max_q * (g->heads / g->kv_heads) > INT_MAX / 2)
    return op_error(H2C_ERR_INVALID, "%s: max_q %d out of range", who, g->max_q);
  return H2C_OK;
}

bool nothing_to_do(const h2c_kv8_attention_args* g) { return g->n_req == 0 || g->rows == 0 || g->max_q == 0; }

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
  const long long hd = g->head_dim;
  if (op_vectors_overlap(g->rows, g->out_row, g->heads, g->out_head, hd))
    return op_error(H2C_ERR_INVALID, "%s: vectors of out overlap (rows %lld elements apart, heads %lld)", who,
                    (long long)g->out_row, (long long)g->out_head);
  {
    // a token's vectors as one row, between the lowest and the highest
    auto rows_of = [&](const void* at, long long row, long long head) {
      const long long span = (g->heads - 1) * head;
      return OpRows{static_cast<const uint8_t*>(at) + std::min(0LL, span) * (long long)es, g->rows, row * (long long)es,
                    (std::abs(span) + hd) * (long long)es};
    };
    const OpRows q = rows_of(g->q, g->q_row, g->q_head), out = rows_of(g->out, g->out_row, g->out_head);
    // (in place is safe: the CTAs that read a vector are done with it before one of them writes it)
    const bool in_place = g->out == g->q && (g->out_row == g->q_row || g->rows == 1) && (g->out_head == g->q_head || g->heads == 1);
    if (!in_place && op_rows_meet(q, out))
      return op_error(H2C_ERR_INVALID, "%s: out must be q itself or share no memory with it", who);
    const uint64_t kv_bytes = 2ull * g->n_pages * g->kv_heads * g->page_size * g->head_dim;
    const OpRange in[] = {{"kv", g->kv, kv_bytes}, {"kv_scale", g->kv_scale, 8ull * g->n_pages * g->kv_heads, 4},
                          {"block_table", g->block_table, 4ull * g->n_req * g->table_cols, 4},
                          {"q_start", g->q_start, 4ull * g->n_req + 4, 4}, {"kv_len", g->kv_len, 4ull * g->n_req, 4}};
    const OpRange written[] = {op_range("out", out), {"lse", g->lse, g->lse ? 4ull * g->rows * g->heads : 0, 4},
                               {"workspace", g->workspace, p.bytes}};
    if (int rc = op_check_ranges(who, written, 3, in, 5)) return rc;
    const OpRange q_range = op_range("q", q);
    if (int rc = op_check_ranges(who, written + 1, 2, &q_range, 1)) return rc;
  }
  const long long most = std::max((long long)p.splits * p.tiles * RW_ROWS, (long long)p.shape.tiles * PR_ROWS);
  if (most * g->kv_heads > INT_MAX) return op_error(H2C_ERR_INVALID, "%s: too many rows for one call", who);
  AttArgs a;
  a.q = g->q; a.q_row = g->q_row; a.q_head = g->q_head;
  a.out = g->out; a.out_row = g->out_row; a.out_head = g->out_head;
  a.lse = g->lse;
  a.kv = static_cast<const int8_t*>(g->kv); a.kv_scale = g->kv_scale;
  a.table = g->block_table; a.q_start = g->q_start; a.kv_len = g->kv_len;
  a.n_pages = g->n_pages; a.kv_heads = g->kv_heads; a.heads = g->heads; a.group = g->heads / g->kv_heads;
  a.group_magic = 0xffffffffu / (unsigned)a.group;
  a.page_log = g->page_size == 16 ? 4 : g->page_size == 32 ? 5 : g->page_size == 64 ? 6 : 7;
  a.table_cols = g->table_cols; a.n_req = g->n_req; a.rows = g->rows; a.max_q = g->max_q; a.window = g->window;
  a.q_vec = !((uintptr_t)g->q & (4 * es - 1)) && !((g->q_row | g->q_head) & 3);
  a.out_vec = !((uintptr_t)g->out & (4 * es - 1)) && !((g->out_row | g->out_head) & 3);
  a.q_vec16 = !((uintptr_t)g->q & 15) && !((g->q_row * es | g->q_head * es) & 15);
  a.out_vec16 = !((uintptr_t)g->out & 15) && !((g->out_row * es | g->out_head * es) & 15);
  a.scale_log2 = g->scale * 1.4426950408889634f;
  cudaStream_t st = (cudaStream_t)stream;
  if (g->type == H2C_TYPE_F32) return launch_typed<float>(who, g->head_dim, p, a, g->workspace, st);
  if (g->type == H2C_TYPE_F16) return launch_typed<__half>(who, g->head_dim, p, a, g->workspace, st);
  return launch_typed<__nv_bfloat16>(who, g->head_dim, p, a, g->workspace, st);
}

}  // extern "C"
