// Host side shared by the stand-alone 8-bit serving operators (ops.cuh).
#include "ops.cuh"

#include <cstdarg>
#include <cstdio>
#include <mutex>

namespace h2 {

void set_last_error(const char* msg) noexcept;  // h2cuda.cu: the message of h2c_last_error(NULL)

int op_error(int code, const char* fmt, ...) noexcept {
  char buf[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}

int op_launched(const char* who) noexcept {
  const cudaError_t c = cudaGetLastError();
  return c == cudaSuccess ? H2C_OK : op_error(H2C_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(c));
}

int op_check_ranges(const char* who, const OpRange* out, int n_out, const OpRange* in, int n_in) noexcept {
  auto meet = [](const OpRange& a, const OpRange& b) {
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    return a.bytes && b.bytes && (x < y ? y - x < a.bytes : x - y < b.bytes);
  };
  for (int i = 0; i < n_out; i++) {
    for (int j = 0; j < n_in; j++)
      if (meet(out[i], in[j])) return op_error(H2C_ERR_INVALID, "%s: %s must not share memory with %s", who, out[i].name, in[j].name);
    for (int j = 0; j < i; j++)
      if (meet(out[i], out[j])) return op_error(H2C_ERR_INVALID, "%s: %s must not share memory with %s", who, out[i].name, out[j].name);
  }
  for (int i = 0; i < n_out + n_in; i++) {
    const OpRange& r = i < n_out ? out[i] : in[i - n_out];
    if (r.bytes && (uintptr_t)r.p % r.align) return op_error(H2C_ERR_INVALID, "%s: %s must be aligned to %u bytes", who, r.name, r.align);
  }
  return H2C_OK;
}

OpRange op_range(const char* name, const OpRows& r) noexcept {
  const int64_t span = (r.rows - 1) * r.stride;
  return {name, static_cast<const uint8_t*>(r.p) + (span < 0 ? span : 0), (uint64_t)((span < 0 ? -span : span) + r.bytes)};
}

bool op_rows_meet(const OpRows& a, const OpRows& b) noexcept {
  const OpRange x = op_range("", a), y = op_range("", b);
  const uintptr_t xp = (uintptr_t)x.p, yp = (uintptr_t)y.p;
  if (xp + x.bytes <= yp || yp + y.bytes <= xp) return false;
  int64_t s = a.rows == 1 ? b.stride : a.stride;
  if ((a.rows > 1 && b.rows > 1 && a.stride != b.stride) || (a.rows == 1 && b.rows == 1)) return true;
  if (s < 0) s = -s;
  if (a.bytes > s || b.bytes > s) return true;
  const uint64_t d = (yp > xp ? yp - xp : (uint64_t)s - (xp - yp) % s) % s;  // from a row of a to the next of b
  return d < (uint64_t)a.bytes || (uint64_t)s - d < (uint64_t)b.bytes;
}

bool op_vectors_overlap(int64_t rows, int64_t row, int64_t heads, int64_t head, int64_t len) noexcept {
  if (row < 0) row = -row;
  if (head < 0) head = -head;
  if ((rows > 1 && row < len) || (heads > 1 && head < len)) return true;
  if (rows <= 1 || heads <= 1 || row >= (heads - 1) * head + len || head >= (rows - 1) * row + len) return false;
  for (int64_t h = 1; h < heads; h++) {  // vectors h heads apart, and the rows' distance that comes nearest
    const int64_t r = h * head / row, over = h * head - r * row;
    if ((r < rows && over < len) || (r + 1 < rows && row - over < len)) return true;
  }
  return false;
}

namespace {
__device__ int g_op_err[4];
int* g_op_err_ptr[OP_MAX_DEVICES];
}  // namespace

int* op_err_words() noexcept {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= OP_MAX_DEVICES) return nullptr;
  int* p = __atomic_load_n(&g_op_err_ptr[dev], __ATOMIC_ACQUIRE);
  if (!p) {
    void* q = nullptr;
    if (cudaGetSymbolAddress(&q, g_op_err) != cudaSuccess) return nullptr;
    p = static_cast<int*>(q);
    __atomic_store_n(&g_op_err_ptr[dev], p, __ATOMIC_RELEASE);
  }
  return p;
}

}  // namespace h2

extern "C" int h2c_ops_check(void* stream) {
  using namespace h2;
  int* d = op_err_words();
  if (!d) return op_error(H2C_ERR_CUDA, "h2c_ops_check: no device");
  int w[4] = {0, 0, 0, 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t c = cudaMemcpyAsync(w, d, sizeof w, cudaMemcpyDeviceToHost, st);
  if (c == cudaSuccess) c = cudaStreamSynchronize(st);
  if (c == cudaSuccess && w[0]) {
    c = cudaMemsetAsync(d, 0, sizeof w, st);
    if (c == cudaSuccess) c = cudaStreamSynchronize(st);
  }
  if (c != cudaSuccess) return op_error(H2C_ERR_CUDA, "h2c_ops_check: %s", cudaGetErrorString(c));
  if (w[0]) return op_error(H2C_ERR_TIMEOUT, "a wait inside an operator expired (CTA %d, role %d): its output is not valid", w[1], w[2]);
  return H2C_OK;
}
