/* h2cuda: the B200 (sm_100a) backend of the H2 engine's Qwen2 Q4_0 token loop, as a plain C ABI.
 *
 * This is the drop-in boundary. It replaces the reference's WebAssembly kernel exports
 * (h2-own-inference-engine/engine/kernels.c:418-496: set_config / set_tensor / set_buffers / run /
 * profile_* / run_read_test), which its CPU backend host binds (cpu-worker.js:85-137, 169-182), and it
 * implements the backend object contract of cpu.js:52-68 / webgpu.js:616-620 one layer up:
 *   forward(ids, pos, {temperature, seed, wantLogits}) -> next token id   => h2c_forward
 *   readLogits()                                                          => h2c_read_logits
 *   profile(ids, pos)                                                     => h2c_profile
 *   destroy()                                                             => h2c_destroy
 *
 * Ownership differs from the reference on purpose: there, JavaScript owns all memory (set_buffers); here the
 * library owns the device weights, the KV cache, the scratch buffers and the CUDA graph of a decode step, and
 * callers pass only host pointers. No torch types cross this boundary.
 *
 * Every call returns a status (H2C_OK = 0, negative on error) and never aborts; h2c_last_error() gives the
 * message of the last failing call on that engine. Calls on one engine must be serialised by the caller (the
 * reference keeps a single outstanding request per backend, cpu.js:33-50).
 */
#ifndef H2CUDA_H
#define H2CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* status codes */
#define H2C_OK 0
#define H2C_ERR_INVALID (-1)      /* bad argument or call order */
#define H2C_ERR_CONTEXT_FULL (-2) /* pos + n >= ctx: "context full", cpu-worker.js:173, webgpu.js:552 */
#define H2C_ERR_BAD_TYPE (-3)     /* unsupported tensor type: cpu-worker.js:105, 112, 126 */
#define H2C_ERR_CUDA (-4)         /* a CUDA runtime call failed */
#define H2C_ERR_NOT_READY (-5)    /* forward before every tensor was set */
#define H2C_ERR_NO_MEMORY (-6)    /* device or pinned allocation failed */
#define H2C_ERR_TIMEOUT (-7)      /* a bounded device-side wait expired (persistent decode kernel, tcgen05 matmul) or a
                                     tensor-parallel peer did not answer within the engine's deadline */
#define H2C_ERR_UNSUPPORTED (-8)  /* tensor parallelism without an NCCL library (libnccl.so.2) in the process */

/* GGML tensor types accepted by h2c_set_tensor (gguf.js:6) */
#define H2C_GGML_F32 0
#define H2C_GGML_Q4_0 2
#define H2C_GGML_Q8_0 8

/* tensor kinds: the numbering of the reference's set_tensor (kernels.c:422-430) */
#define H2C_KIND_QKV 0         /* [Wq; Wk; Wv] rows concatenated, Q4_0 (cpu-worker.js:60, 108-115) */
#define H2C_KIND_O 1           /* attn_output, Q4_0 */
#define H2C_KIND_GATE_UP 2     /* [Wgate; Wup] rows concatenated, Q4_0 */
#define H2C_KIND_DOWN 3        /* ffn_down, Q4_0 */
#define H2C_KIND_ATTN_NORM 4   /* F32 [dim] */
#define H2C_KIND_FFN_NORM 5    /* F32 [dim] */
#define H2C_KIND_QKV_BIAS 6    /* F32 [dim + 2*kv_heads*head_dim]: [bq; bk; bv] */
#define H2C_KIND_EMBED 7       /* token_embd, Q4_0 [vocab][dim] */
#define H2C_KIND_OUTPUT 8      /* output.weight, Q8_0 (the reference's only type) or Q4_0; unset = tied to EMBED */
#define H2C_KIND_OUTPUT_NORM 9 /* F32 [dim] */

/* Model and runtime configuration: set_config(dim, layers, ffn, heads, kvh, vocab, ctx, mt, eps)
 * (kernels.c:418-421) plus the RoPE base the reference host uses for its table (cpu-worker.js:131-135). */
typedef struct h2c_config {
  int32_t dim, layers, ffn, heads, kv_heads, vocab;
  int32_t ctx;        /* positions per sequence (KV cache length); forward needs pos + n < ctx */
  int32_t max_chunk;  /* tokens per prefill pass (the reference's mt / prefillChunk: cpu.js:46) */
  int32_t max_seqs;   /* independent sequences (sessions), each with its own KV cache; >= 1 */
  float eps;          /* RMSNorm epsilon */
  double rope_theta;  /* RoPE frequency base (gguf.js:82) */
} h2c_config;

typedef struct h2c_engine h2c_engine;

/* Per-operation device time of one forward pass, in the reference's profile order (cpu-worker.js:32). */
#define H2C_NPROF 11
/* 0 embed, 1 norm+quantize, 2 matvec qkv, 3 rope+kv, 4 attention, 5 quantize, 6 matvec o, 7 matvec gate+up,
 * 8 swiglu+quantize, 9 matvec down, 10 matvec output */

/* Create an engine on CUDA device `device`: allocates the KV cache and scratch (replaces set_config +
 * set_buffers, kernels.c:418-437 and the layout of cpu-worker.js:52-88). With max_chunk >= 32 the scratch includes
 * the score buffer of prompt passes: heads x max_chunk x ctx floats, at most 256 MB (the environment variable
 * H2C_PROMPT_SCORES_MB, read here, sets another cap; longer passes then run in query blocks, same results). */
int h2c_create(int device, const h2c_config* cfg, h2c_engine** out);

/* Tensor parallelism over G GPUs of one node, one process (or thread) per GPU: the 7B configuration split so that
 * each rank reads 1/G of the weights per token (no reference counterpart: the reference runs one CPU process).
 * Every matrix is split by output rows, so each output value is computed whole, in the reference's order, by one
 * rank, and the results stay bit-identical to one GPU's: rank r owns query heads [r*H/G, (r+1)*H/G) with their
 * kv heads (and that part of the KV cache), rows [r*D/G, (r+1)*D/G) of O and of down, rows [r*F/G, (r+1)*F/G) of
 * gate and of up, and rows [r*Vp, r*Vp + Vp) of the lm_head (Vp = vocab / G rounded up to 32 rows). NCCL
 * all-gathers of the attention output, of the residual after O and after down, of the quantized FFN activation and
 * of the logits give every rank the full vectors in between; every rank computes the same token. Requires
 * kv_heads, dim / 32 and ffn / 32 divisible by G (Qwen2-7B: G = 1, 2 or 4; 4 kv heads cannot be split 8 ways).
 *
 * h2c_tp_unique_id: rank 0 creates the group's id (H2C_TP_ID_BYTES bytes) and the host hands it to every rank.
 * h2c_create_tp: every rank calls it at about the same time with the same cfg and id; the engine then takes the
 * FULL tensors in h2c_set_tensor and keeps this rank's rows. Every rank must then make the same calls with the same
 * arguments (h2c_forward, h2c_generate, h2c_profile). timeout_ms (<= 0: 120 s) bounds the group's set-up and each
 * call's wait: a peer that never joins or stops answering ends in H2C_ERR_TIMEOUT with the communicator aborted
 * (the engine then only accepts h2c_destroy). Not available with tensor parallelism: h2c_forward_batch,
 * h2c_generate_batch, the persistent decode kernel (steps run on the CUDA graph path), h2c_trace_decode. NCCL is
 * loaded at run time (libnccl.so.2 of the process, else the system's): H2C_ERR_UNSUPPORTED without one. G = 1
 * behaves as h2c_create. */
#define H2C_TP_ID_BYTES 128
int h2c_tp_unique_id(uint8_t* id);
int h2c_create_tp(int device, const h2c_config* cfg, int32_t world, int32_t rank, const uint8_t* id,
                  int32_t timeout_ms, h2c_engine** out);
/* This engine's rank and group size (0 and 1 without tensor parallelism). */
int32_t h2c_tp_rank(const h2c_engine* e);
int32_t h2c_tp_world(const h2c_engine* e);

/* Upload one tensor from host memory holding raw GGUF bytes of `ggml_type` (blocks for Q4_0 / Q8_0, floats for
 * F32). Replaces set_tensor (kernels.c:423-431) and the repack of cpu-worker.js:97-128: the library splits
 * GGUF blocks into its own device layout. `layer` is ignored for kinds 7..9. */
int h2c_set_tensor(h2c_engine* e, int kind, int layer, int ggml_type, const void* data, uint64_t nbytes);

/* Run ids[0..n) of sequence `seq` at positions pos..pos+n-1 (prefill when n > 1, one decode step when n == 1)
 * and return the next token in *next: greedy argmax (ties to the lowest id) when temperature <= 0, else a
 * sample of softmax(logits / temperature) with mulberry32 seeded by (seed + pos) (cpu-worker.js:154-180), drawn on
 * the device (the logits never leave it). temperature is a double, as the reference's JavaScript number is.
 * Prompts run in chunks of max_chunk tokens; logits exist for the last token only (kernels.c:404-414).
 * Replaces run() (kernels.c:454-465) plus the host loop of cpu-worker.js:169-182. */
int h2c_forward(h2c_engine* e, int seq, const int32_t* ids, int32_t n, int32_t pos, double temperature,
                uint32_t seed, int32_t* next);

/* One decode step of n sessions at once (the multi-session serving form, forwardBatch of the CUDA backend; no
 * reference counterpart: the reference serves one session per backend, cpu.js:33-50). Token ids[m] of sequence
 * seqs[m] (distinct) is processed at position pos[m]; next[m] receives its next token, chosen as by h2c_forward
 * (greedy, or sampled with seed + pos[m]). Each weight byte is read once for the whole batch; every token's
 * arithmetic is the single-token arithmetic, so the results equal n separate h2c_forward calls bit for bit.
 * 1 <= n <= min(max_chunk, 256). h2c_read_logits(seqs[m]) returns token m's logits afterwards. */
int h2c_forward_batch(h2c_engine* e, int32_t n, const int32_t* seqs, const int32_t* ids, const int32_t* pos,
                      double temperature, uint32_t seed, int32_t* next);

/* Greedy decode of `steps` tokens of each of n sessions entirely on the device: batched steps as h2c_forward_batch,
 * each step's tokens fed to the next without a host round trip. out_tokens (nullable) receives [n][steps] ids;
 * device_ms (nullable) the CUDA-event time of the steps. Needs pos[m] + steps < ctx. */
int h2c_generate_batch(h2c_engine* e, int32_t n, const int32_t* seqs, const int32_t* ids, const int32_t* pos,
                       int32_t steps, int32_t* out_tokens, float* device_ms);

/* Greedy decode of `steps` tokens of sequence `seq` entirely on the device: first_id is processed at `pos`, each
 * step's argmax becomes the next step's input without a host round trip (the WebGPU backend keeps its sampled
 * token on the GPU the same way, webgpu.js:391, 553-574). out_tokens (nullable) receives the `steps` generated
 * ids; device_ms (nullable) the CUDA-event time of the steps on the engine's stream. Needs pos + steps < ctx.
 * Equivalent to steps calls of h2c_forward(e, seq, &id, 1, pos + i, 0, 0, &id). */
int h2c_generate(h2c_engine* e, int seq, int32_t first_id, int32_t pos, int32_t steps, int32_t* out_tokens,
                 float* device_ms);

/* Decode-step implementations. AUTO (default) uses the persistent kernel when the model fits it (one cooperative
 * launch runs every layer of one or more tokens; weights stream into shared memory ahead of use) and otherwise
 * the CUDA graph of per-operation kernels. Both give bit-identical results. */
#define H2C_DECODE_AUTO 0
#define H2C_DECODE_GRAPH 1
#define H2C_DECODE_PERSISTENT 2
/* Select the decode path; H2C_DECODE_PERSISTENT fails with H2C_ERR_INVALID if the model does not fit it. */
int h2c_set_decode_mode(h2c_engine* e, int mode);
/* The path single-token steps will take: H2C_DECODE_GRAPH or H2C_DECODE_PERSISTENT (< 0 on error). */
int h2c_decode_path(h2c_engine* e);

/* The kernel of passes of several tokens (prompt chunks, batched decode steps), process-wide (no reference
 * counterpart: the reference has one CPU matmul). TCGEN05 takes the Blackwell tensor-core form (tcgen05.mma into
 * TMEM) for Q4_0 matrices, MMA_SYNC the warp-level int8 mma.sync form; AUTO (default) the tcgen05 form for passes of
 * 64 or more tokens and the mma.sync form for fewer (the faster of the two at each size on B200). All are
 * bit-identical to the reference. Takes effect for passes enqueued afterwards (a batch step's CUDA graph keeps the
 * kernel it was captured with). */
#define H2C_MATMUL_AUTO 0
#define H2C_MATMUL_MMA_SYNC 1
#define H2C_MATMUL_TCGEN05 2
int h2c_set_matmul_kernel(int kind);
/* The current setting (H2C_MATMUL_AUTO, _MMA_SYNC or _TCGEN05). */
int h2c_matmul_kernel(void);

/* Profiling aid for the persistent decode kernel: runs h2c_generate's device-side greedy decode once with
 * %globaltimer stamps (nanoseconds) taken at the stage boundaries of every CTA. out receives
 * h2c_decode_ctas(e) * steps * (layers + 1) * 16 entries: [cta][step][layer or lm_head][point], 0 where a point
 * does not apply. The per-operation profile of the reference (profile_start/get, kernels.c:481-483) for this
 * path. Allocates a temporary device buffer. */
int h2c_trace_decode(h2c_engine* e, int seq, int32_t first_id, int32_t pos, int32_t steps, uint64_t* out, int64_t n);

/* Grid size (CTAs) of the persistent decode kernel, 0 when the model takes the graph path; < 0 on error. */
int h2c_decode_ctas(h2c_engine* e);

/* Test aid for the persistent kernel's failure detection (no reference counterpart): every bounded wait of the
 * kernel gives up after timeout_ns (default 2 s), and with stall_cta >= 0 that CTA never publishes its QKV rows,
 * so the CTAs that need them wait until the limit, record the error and every CTA returns; the next
 * h2c_forward / h2c_generate then fails with H2C_ERR_TIMEOUT and the engine stays usable (the affected positions
 * of the KV cache must be recomputed). stall_cta = -1 restores normal operation. No fault, trap or hang. */
int h2c_set_decode_fault(h2c_engine* e, int stall_cta, int64_t timeout_ns);

/* Self-test of the decode kernels' correctly rounded arithmetic (no reference counterpart): compares the fast
 * division by 127 and by 896, reciprocal and square root used on the quantization and RMSNorm paths with CUDA's
 * IEEE-rounded __fdiv_rn / __fsqrt_rn over all 2^32 float bit patterns on `device` and writes the four mismatch
 * counts (all 0 when the fast forms are exact on this GPU) to mismatches[0..3]. */
int h2c_selftest_math(int device, uint64_t* mismatches);

/* Number of kernels one batched decode step of n sessions launches (the kernel nodes of its CUDA graph, which the
 * first h2c_forward_batch / h2c_generate_batch of that size builds); 0 before that; < 0 on error. */
int h2c_batch_kernels(h2c_engine* e, int32_t n);

/* Number of kernels one decode step launches (the kernel nodes of the decode-step CUDA graph); < 0 on error. */
int h2c_decode_kernels(h2c_engine* e);

/* Copy the logits of the last forward of `seq` (vocab floats) to host memory (cpu.js:60-62, webgpu.js:605-611). */
int h2c_read_logits(h2c_engine* e, int seq, float* out, int64_t n);

/* One forward pass like h2c_forward with greedy sampling, timing each operation with CUDA events (no graph):
 * ms[H2C_NPROF] receives milliseconds per operation class (profile_start/get/stop, kernels.c:481-483). */
int h2c_profile(h2c_engine* e, int seq, const int32_t* ids, int32_t n, int32_t pos, double* ms);

/* Free everything the engine owns (cpu.js:67 destroy). Safe on NULL. */
int h2c_destroy(h2c_engine* e);

/* Message of the last error on this engine; with e NULL, of the last failed call on this thread that has no engine
 * (h2c_create, h2c_q4_matvec, h2c_q4_matvec_noalloc). */
const char* h2c_last_error(const h2c_engine* e);

/* Bytes of device memory the engine holds (cpu.js:53 memoryBytes / webgpu.js uploadedBytes). */
int64_t h2c_device_bytes(const h2c_engine* e);

/* ---- Q4_0 matvec, the reference's matmul_q4 (kernels.c:200-273) with its quantize_row (kernels.c:90-114)
 * as a stand-alone device operation: the Q4_0 matvec microbench. Pointers are DEVICE pointers. ---- */

/* Bytes of the device layout of an N x K Q4_0 matrix (values, then fp16 scales). */
uint64_t h2c_q4_matrix_bytes(int32_t n_rows, int32_t k);
/* Convert raw GGUF Q4_0 blocks (host) to the device layout (host buffer of h2c_q4_matrix_bytes). */
int h2c_q4_pack(const void* gguf_blocks, int32_t n_rows, int32_t k, void* packed_host);
/* Scratch bytes h2c_q4_matvec needs for m tokens of length k (the int8 activations and their scales). */
uint64_t h2c_q4_matvec_scratch_bytes(int32_t m, int32_t k);
/* y[m][n] (op)= W[n] . quantize(x[m]) for m < M on `stream` (a cudaStream_t, 0 = default).
 * op: 0 store, 1 add bias[n], 2 accumulate into y (the reference's put(): kernels.c:190-194).
 * w: packed matrix (h2c_q4_pack layout) on the device; x: float32 [M][K]; y: float32 [M][N]; bias: float32 [N]
 * or NULL; scratch: h2c_q4_matvec_scratch_bytes(M, K) bytes of device memory, 16-byte aligned. */
int h2c_q4_matvec(const void* w, int32_t n_rows, int32_t k, const float* x, int32_t m, float* y, int32_t op,
                  const float* bias, void* scratch, void* stream);

/* h2c_q4_matvec without any allocation, for callers that cannot call cudaMalloc (a host that owns all device
 * memory through its own pool, or a latency-critical thread such as a voice pipeline's audio callback, where
 * cudaMalloc can block and synchronize the device). This entry point has no counterpart in the reference.
 * Same arguments and result as h2c_q4_matvec, minus `scratch`: the scratch lives in a fixed 256 KiB
 * __device__ array inside this library (held on every GPU that loads it until the process exits), so m and k are
 * limited to h2c_q4_matvec_scratch_bytes(m, k) <= 262144 (for example m = 32 tokens of k = 4864); larger inputs
 * are rejected with H2C_ERR_INVALID and a message in h2c_last_error(NULL). The first call on a device looks the
 * array's device address up (make it before any stream capture). All calls share the array: calls that overlap
 * on the GPU race and must be serialised by the caller. */
int h2c_q4_matvec_noalloc(const void* w, int32_t n_rows, int32_t k, const float* x, int32_t m, float* y,
                          int32_t op, const float* bias, void* stream);

/* ---- 8-bit serving operators: a paged 8-bit KV cache and matrix products in 8-bit integers. Stand-alone device
 * operations (no engine): every pointer is a DEVICE pointer unless said otherwise, `stream` is a cudaStream_t of the
 * current device (0 = default) and a call only enqueues work on it, nothing is allocated, and a call whose arguments
 * do not fit (sizes, alignment to their elements, outputs over other arguments) returns a status with a message in
 * h2c_last_error(NULL) before anything is enqueued. Sizes of zero (requests, rows) are valid and do nothing; more than
 * 2^31 - 65537 rows are refused. A call's results do not depend on the stream, on what else runs, or on earlier calls.
 *
 * The cache: `kv` holds int8 codes [n_pages][2][kv_heads][page_size][head_dim] (index 0 of the second axis: K, 1: V;
 * 16-byte aligned), `kv_scale` float32 [n_pages][2][kv_heads], not negative; a cached value is code * scale. page_size is
 * 16, 32, 64 or
 * 128, head_dim 64 or 128, n_pages * page_size < 2^31. A slot is page * page_size + offset. A request's position p lies
 * in page block_table[request][p / page_size] at offset p % page_size; no page belongs to two requests. ---- */

/* element types of activations */
#define H2C_TYPE_F32 0
#define H2C_TYPE_F16 1
#define H2C_TYPE_BF16 2

#define H2C_KV8_MAX_REQUESTS 8192

/* H2C_OK, or H2C_ERR_TIMEOUT when a bounded wait inside one of these operators' kernels expired on the current device
 * since the last check (its output is then not valid; this never happens in normal operation). Waits for `stream`. */
int h2c_ops_check(void* stream);

/* Block tables and slot maps from request lengths, on the device. Request r holds cached[r] tokens and will hold total[r]
 * after the step: more (its new tokens are cached[r] .. total[r]-1, pages are taken for them), as many, or fewer (it is
 * cut back, or ends at 0, and the pages beyond are given back).
 *   cached, total    int32 [n_req], n_req <= H2C_KV8_MAX_REQUESTS
 *   block_table      int32 [n_req][table_cols], in place: the entries of the pages taken are written; entries past a
 *                    request's length keep what they held and mean nothing
 *   free_ring        int32 [n_pages], in place: a ring of free page numbers; free_state int64 [2] = {head, tail}
 *                    (both only grow): the free pages are free_ring[head % n_pages] .. free_ring[(tail - 1) % n_pages].
 *                    Pages are taken at the head in request order, those given back are appended at the tail in
 *                    request order, and can be taken in the same call once the older ones are used up
 *   free_state_out   int64 [2], the ring after the step (not the same memory as free_state: a call with the same
 *                    inputs again gives the same results)
 *   kv_len           int32 [n_req]: total[r];  q_start int32 [n_req + 1]: prefix sums of the new tokens
 *   slot, position   int32 [max_tokens]: slot and position of each new token, in request order; -1 beyond the last
 *   status           int32 [2]: {0, 0}; {1, missing} when the free pages do not suffice; {2, 0} when a length is negative
 *                    or above table_cols * page_size, the new tokens are more than max_tokens, or the ring's state is
 *                    not that of n_pages pages. With a non-zero status nothing is taken or given back: kv_len is
 *                    cached (0 where that is invalid), q_start all 0, slot and position all -1, free_state_out =
 *                    free_state.
 * What is written shares no memory with what is read or with another output (refused): a loop that feeds kv_len back as the
 * next step's cached keeps two sets of outputs in turn. */
int h2c_kv8_plan(int32_t n_req, int32_t page_size, const int32_t* cached, const int32_t* total, int32_t* block_table,
                 int32_t table_cols, int32_t* free_ring, int32_t n_pages, const int64_t* free_state,
                 int64_t* free_state_out, int32_t* kv_len, int32_t* q_start, int32_t* slot, int32_t* position,
                 int32_t max_tokens, int32_t* status, void* stream);

/* Append rows of K and V (element type `type`, row t of head h at k + t * k_row + h * k_head elements, head_dim values
 * each, likewise v) to the cache at slot[t]; rows whose slot is not in the cache (-1) are skipped. The rows of one page
 * must be consecutive rows at consecutive offsets, as h2c_kv8_plan orders them. Per (page, K or V, head), with a the
 * largest magnitude of the rows that go there and s0 the scale so far (0 when they start at offset 0, which makes the
 * page new whatever it held): if a > 127.5 s0 the scale becomes s = max(a / 127, 1.25 s0), within [2^-62, 2^63], and the
 * codes at earlier offsets become round(code * (s0 / s)); else s = s0. The new codes are round(x * (1 / s)), within
 * [-127, 127] (float32 operations, halves to even). A code is re-rounded only when the scale grows, which it does by at
 * least 1.25 each time, so a cached value is off by at most 2.5 final steps (magnitudes above 127 * 2^63 become that). A
 * row with an infinity or NaN makes its
 * page's scale NaN until the page is new again: every read of that page and head gives NaN. The cache shares no memory
 * with k, v or
 * slot (refused). */
int h2c_kv8_append(void* kv, float* kv_scale, int32_t n_pages, int32_t page_size, int32_t kv_heads, int32_t head_dim,
                   int32_t type, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row,
                   int64_t v_head, int32_t rows, const int32_t* slot, void* stream);

/* The cached values at slot[t], t < rows: k_out and v_out [rows][kv_heads][head_dim] of element type `type` (16-byte
 * aligned, sharing no memory with the cache, slot or each other); zeros where the slot is not in the cache. To move a
 * session elsewhere, or to look at what the cache holds. */
int h2c_kv8_read(const void* kv, const float* kv_scale, int32_t n_pages, int32_t page_size, int32_t kv_heads,
                 int32_t head_dim, const int32_t* slot, int32_t rows, int32_t type, void* k_out, void* v_out,
                 void* stream);

/* Grouped-query attention of a ragged batch over the cache. Request r's queries are rows q_start[r] .. q_start[r + 1]-1 of
 * q, its last query at position kv_len[r] - 1: query i of n sits at position p = kv_len[r] - n + i and attends to the cached
 * positions 0 .. p, or p - window + 1 .. p with window > 0. Head h reads kv head h / (heads / kv_heads).
 *   x = scale * (q . k),  out = sum softmax(x) v  (rounded once to `type`),  lse = log sum exp x  (natural logarithm)
 * A query with no position to attend to (p < 0) gives zeros and lse = -infinity. Rows of q that belong to no request are
 * not touched. out may be q itself (the same address and strides); otherwise what is written (out, lse, the workspace)
 * shares no
 * memory with another argument, nor do two vectors of out (refused).
 * Scores, softmax statistics and sums are float32. Codes and 16-bit queries enter the tensor cores exactly, float32 queries
 * as two float16 terms (22 bits), the softmax's weights as two, too, save in bfloat16 prompts, which round each weight to 11
 * bits (2^-12 of it; the output's own rounding is 2^-9 of itself). 16-bit prompts take V's scales through their logarithm
 * (2^-22), and one below 2^-62 as 2^-62. Prompts' sums are the tensor cores' for 4 to 128 tiles of 64 keys, which cut off
 * what float32 does not hold, and are rounded between: that puts float32 outputs off by some 1e-6 of their size at any
 * length of the history, 16-bit outputs by 2e-5 beside their rounding. How a call is divided (n_req, max_q, max_kv,
 * window, and so the
 * requests beside a request) moves results within these errors; the same call gives the same bits every time. */
typedef struct h2c_kv8_attention_args {
  const void* q;          /* row t of head h at t * q_row + h * q_head elements, head_dim values */
  int64_t q_row, q_head;
  void* out;              /* the same with out_row, out_head */
  int64_t out_row, out_head;
  float* lse;             /* [rows][heads], or NULL */
  const void* kv;
  const float* kv_scale;
  int32_t n_pages, page_size, kv_heads, head_dim;
  int32_t heads, type;    /* heads a multiple of kv_heads; element type of q and out */
  const int32_t* block_table; /* [n_req][table_cols] */
  int32_t table_cols, n_req;
  const int32_t* q_start; /* [n_req + 1] */
  const int32_t* kv_len;  /* [n_req] */
  int32_t rows;           /* rows of q and out */
  int32_t max_q, max_kv;  /* bounds of the requests' query counts and kv_len, for the division of the work: a request with
                             more than max_q queries has only its first max_q computed; kv_len above max_kv costs time */
  int32_t window;         /* 0: none */
  float scale;
  void* workspace;        /* h2c_kv8_attention_workspace(args) bytes, 16-byte aligned; NULL when that is 0 */
  uint64_t workspace_bytes;
} h2c_kv8_attention_args;
/* Bytes of device workspace a call with these sizes needs (pointers are not looked at). Host only. */
uint64_t h2c_kv8_attention_workspace(const h2c_kv8_attention_args* args);
int h2c_kv8_attention(const h2c_kv8_attention_args* args, void* stream);

/* Attention of requests that share prefixes (a system prompt of many sessions): as h2c_kv8_attention, with the positions of a prefix
 * before a request's own. Requests group_start[g] .. group_start[g + 1]-1 share prefix g, the first prefix_len[g] positions of the
 * pages prefix_table[g] (which no request's own table needs to name: a prefix is held like a session of its own, and may end
 * anywhere in a page); requests of no group have none. Request r's queries see all positions of its prefix and, causally, its own: query
 * i of n its own positions 0 .. kv_len[r] - n + i. The softmax is over both, and a prefix's keys are read once for all of a group's
 * rows of a kv head, or for every 256 of them. A query that sees nothing gives zeros and lse = -infinity.
 * own.window must be 0. What is rounded where is as in h2c_kv8_attention, where a group's rows count as one prompt for the prefix, but
 * that the softmax's weights have 22 bits in bfloat16 prompts, too; the parts are joined in float32. group_start is clamped to
 * 0 .. own.n_req and must not decrease: where groups overlap, a row has the prefix of one of its groups or, when their rows are more
 * than the call's, of none. The workspace is h2c_kv8_prefix_attention_workspace bytes. */
typedef struct h2c_kv8_prefix_args {
  h2c_kv8_attention_args own;
  const int32_t* prefix_table; /* [n_groups][prefix_cols] */
  const int32_t* prefix_len;   /* [n_groups] */
  const int32_t* group_start;  /* [n_groups + 1] */
  int32_t prefix_cols, n_groups;
  int32_t max_prefix;          /* bounds the prefixes' lengths, for the division of the work */
} h2c_kv8_prefix_args;
uint64_t h2c_kv8_prefix_attention_workspace(const h2c_kv8_prefix_args* args);
int h2c_kv8_prefix_attention(const h2c_kv8_prefix_args* args, void* stream);

/* Matrix products in 8-bit integers, with a scale for each token and each output channel. */
#define H2C_TYPE_I8 3         /* codes, where an entry says so */
#define H2C_I8_MAX_K 131072   /* (sums of k products of two codes stay within 32 bits) */

/* Rows of x (element type `type`, row r at x + r * x_row elements, k values) as codes q[r][0 .. k) and scale[r]: with a the
 * row's largest magnitude, scale = a / 127 and q = round(x * min(127 / a, FLT_MAX)) (float32 operations, halves to even;
 * a row of zeros gives zeros). Rows of q start q_row bytes apart (a multiple of 16, at least k, q 16-byte aligned); the
 * bytes from k to the next multiple of 16 become 0. A row with an infinity or NaN has the scale NaN (and codes without
 * meaning): every product with it is NaN. q and scale share no memory with x or each other (refused). For weights (rows =
 * output channels), once, and for activations that
 * several products share. */
int h2c_i8_quantize(int32_t type, const void* x, int64_t x_row, int32_t rows, int32_t k, void* q, int64_t q_row,
                    float* scale, void* stream);

/* y[i][j] = (sum over k of xq[i][k] * w[j][k]) * xs[i] * w_scale[j] + bias[j], i < m, j < n, rounded to y_type; the integer
 * sum is exact. xq and xs are the codes and scales of h2c_i8_quantize for row i of x: x_type F32, F16 or BF16 makes them
 * in the workspace (x_scale is not looked at), x_type H2C_TYPE_I8 takes x as codes (x_row bytes apart) with x_scale.
 * w: int8 [n] rows w_row bytes apart. Codes and w are 16-byte aligned with rows a multiple of 16 bytes apart, at least k;
 * what lies beyond k is not looked at. y: row i at y + i * y_row elements. bias: float32 [n] or NULL. workspace:
 * h2c_i8_matmul_workspace bytes, 16-byte aligned (NULL when that is 0). m = 0 or n = 0 does nothing. y may lie in the memory of
 * x's values, which are read before it is written; it shares none with another argument, nor do its rows (refused). */
uint64_t h2c_i8_matmul_workspace(int32_t x_type, int32_t m, int32_t k);
int h2c_i8_matmul(int32_t x_type, const void* x, int64_t x_row, const float* x_scale, const void* w, int64_t w_row,
                  const float* w_scale, int32_t m, int32_t n, int32_t k, int32_t y_type, void* y, int64_t y_row,
                  const float* bias, void* workspace, uint64_t workspace_bytes, void* stream);

/* ---- The operators of a serving step beside its cache and its products, to the same rules as those above: device pointers, the
 * caller's stream, nothing allocated, arguments that do not fit refused before anything is enqueued. ---- */

/* Norm and codes of rows r < rows of k <= H2C_I8_MAX_K values, in one pass. With a residual:
 *   s = x + residual, rounded to the residual's type and written to sum (row r at sum + r * sum_row elements)
 * else s = x (residual and sum NULL, res_type and the strides not looked at). Then, with the mean over the row in 64 bits,
 *   f = 1 / sqrt(mean(s^2) + eps) rounded to float32,  y = (s * f) * weight
 * and q, scale are the codes and scales that h2c_i8_quantize has for y: a = max |y|, scale = a / 127, q = round(y * min(127 / a,
 * FLT_MAX)), single float32 operations, halves to even; q as there (rows a multiple of 16 bytes apart, zeros from k to the next
 * multiple of 16), ready for h2c_i8_matmul with x_type H2C_TYPE_I8. A row whose y holds an infinity or NaN has the scale NaN.
 * x_type F32, F16 or BF16; res_type x_type or F32; weight float32 [k]; eps not negative. sum may be residual itself or x itself (same
 * address, strides and type); beside that what is written shares no memory with another argument, nor do rows of sum (refused). */
int h2c_i8_norm(int32_t x_type, const void* x, int64_t x_row, int32_t res_type, const void* residual, int64_t res_row, void* sum,
                int64_t sum_row, const float* weight, double eps, int32_t rows, int32_t k, void* q, int64_t q_row, float* scale,
                void* stream);

/* What codes stand for: y[r][i] = q[r][i] * scale[r], rounded to `type`, rows of y k elements apart. q as above, of which the bytes
 * from k on are not looked at; y shares no memory with q or scale (refused). */
int h2c_i8_values(const void* q, int64_t q_row, const float* scale, int32_t rows, int32_t k, int32_t type, void* y, void* stream);

/* Rotary positions. Token t's vectors of q_heads queries (row t of head h at q + t * q_row + h * q_head elements, head_dim values, 2
 * to 1024) and of k_heads keys (likewise; either may be 0) go to q_out and k_out with the first rotary_dim (even) values turned and
 * the others as they are. Pair j < rotary_dim / 2 is (x[j], x[j + rotary_dim / 2]), or with `interleaved` (x[2j], x[2j + 1]):
 *   (a, b) -> (a c - b s, b c + a s),  c = magnitude * cos(u), s = magnitude * sin(u),  u = position[t] * frequency[j]
 * frequency: float64 [rotary_dim / 2], radians per position. The angle's whole turns are dropped from a product that keeps its
 * remainder, so it is as exact far out as near 0; c and s are taken in 64 bits and rounded to float32 once, the rest is float32. A token whose position is negative (h2c_kv8_plan's beyond the last) is not turned,
 * magnitude included. q_out may be q itself (same address and strides), k_out k; beside that what is written shares no memory with
 * another argument, nor do two vectors of it (refused). */
int h2c_rope(int32_t type, const void* q, int64_t q_row, int64_t q_head, void* q_out, int64_t q_out_row, int64_t q_out_head,
             int32_t q_heads, const void* k, int64_t k_row, int64_t k_head, void* k_out, int64_t k_out_row, int64_t k_out_head,
             int32_t k_heads, int32_t tokens, int32_t head_dim, const int32_t* position, const double* frequency,
             int32_t rotary_dim, int32_t interleaved, float magnitude, void* stream);

#define H2C_LOGITS_MAX_BIASES 1024

/* Penalties, biases and masks on the logits of `rows` rows, `vocab` each (row r at logits + r * in_row elements of `type`, out
 * likewise). With c the number of times that token i stands among the row's tokens so far (tokens[r * tokens_row + 0 ..
 * length[r] - 1], at most `columns`; numbers outside the vocabulary count for none), in single float32 operations:
 *   c > 0:  x = x > 0 ? x / repetition[r] : x * repetition[r],  then  x = x - (frequency[r] * c + presence[r])
 *   i among bias_id[r][0 .. n_bias):  x = x + the sum of its biases, in the list's order (an id outside the vocabulary, as -1, is
 *                                     skipped)
 *   bit i % 32 of allowed[r * allowed_row + i / 32] is 0:  x = -infinity, whatever it was (a row may be left with nothing)
 * and rounded to `type`. tokens and length NULL: no penalties (repetition, presence and frequency then NULL, too, each of which
 * may be NULL otherwise: 1, 0 and 0); bias_id and bias int32 and float32 [rows][n_bias], n_bias <= H2C_LOGITS_MAX_BIASES, 0: none;
 * allowed NULL: all. out may be logits itself (same address and stride); beside that it shares no memory with another argument, nor do
 * its rows (refused). */
int h2c_logits_adjust(int32_t type, const void* logits, int64_t in_row, void* out, int64_t out_row, int32_t rows, int32_t vocab,
                      const int32_t* tokens, int64_t tokens_row, int32_t columns, const int32_t* length, const float* repetition,
                      const float* presence, const float* frequency, const int32_t* bias_id, const float* bias, int32_t n_bias,
                      const int32_t* allowed, int64_t allowed_row, void* stream);

#ifdef __cplusplus
}
#endif
#endif
