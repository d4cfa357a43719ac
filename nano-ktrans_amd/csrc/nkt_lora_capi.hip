// C ABI of the adapters (declared in include/nkt_lora.h).
#include <stdarg.h>
#include <stdio.h>

#include <new>

#include "../../include/nkt_lora.h"
#include "nkt_lora_internal.h"

namespace {

using namespace nkt;

struct LoraHandle {
  LoraView view;
  bool bound;
};

void set_err(char* err, size_t len, const char* fmt, ...) {
  if (!err || len == 0) return;
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(err, len, fmt, ap);
  va_end(ap);
}

bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Tokens of a call, columns of a projection, values of a buffer's adapter.
constexpr int kMaxTokens = 1 << 22;
constexpr int64_t kMaxColumns = 1 << 20;
constexpr int64_t kMaxValues = (int64_t)1 << 31;

bool check_tokens(int num_tokens, char* err, size_t len) {
  if (num_tokens >= 0 && num_tokens <= kMaxTokens) return true;
  set_err(err, len, "num_tokens=%d outside [0, 2^22]", num_tokens);
  return false;
}

// Whether [a, a_bytes) and [b, b_bytes) share a byte.
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  return (uintptr_t)a < (uintptr_t)b + b_bytes && (uintptr_t)b < (uintptr_t)a + a_bytes;
}

}  // namespace

extern "C" {

void* nkt_lora_create(int num_adapters, int in_features, const int* out_features, int num_parts, int max_rank,
                      char* err, size_t err_len) {
  if (num_adapters < 1 || num_adapters > 4096) {
    set_err(err, err_len, "num_adapters=%d outside [1, 4096]", num_adapters);
    return nullptr;
  }
  if (in_features < 64 || in_features % 64) {
    set_err(err, err_len, "in_features=%d: a multiple of 64 wanted", in_features);
    return nullptr;
  }
  if (!out_features || num_parts < 1 || num_parts > NKT_LORA_MAX_PARTS) {
    set_err(err, err_len, "num_parts=%d: 1 to %d parts with their out_features wanted", num_parts, NKT_LORA_MAX_PARTS);
    return nullptr;
  }
  if (max_rank < 1 || max_rank > NKT_LORA_MAX_RANK) {
    set_err(err, err_len, "max_rank=%d outside [1, %d]", max_rank, NKT_LORA_MAX_RANK);
    return nullptr;
  }
  LoraView v = {};
  v.adapters = num_adapters;
  v.parts = num_parts;
  v.in = in_features;
  v.rank = max_rank <= 16 ? 16 : max_rank <= 32 ? 32 : max_rank <= 64 ? 64 : 128;
  v.row_blocks = (num_parts * v.rank + 31) / 32;
  int64_t columns = 0;
  for (int p = 0; p < NKT_LORA_MAX_PARTS; ++p) {
    if (p < num_parts) {
      if (out_features[p] < 64 || out_features[p] % 64) {
        set_err(err, err_len, "out_features[%d]=%d: a multiple of 64 wanted", p, out_features[p]);
        return nullptr;
      }
      columns += out_features[p];
    }
    v.part_end[p] = p < num_parts ? (int)(columns / 64) : INT32_MAX;
  }
  if (columns > kMaxColumns) {
    set_err(err, err_len, "out_features of %lld in all: over 2^20", (long long)columns);
    return nullptr;
  }
  if (columns * v.rank > kMaxValues || (int64_t)in_features * v.row_blocks * 32 > kMaxValues) {
    set_err(err, err_len, "in_features=%d, out_features of %lld in all: over 2^31 values of an adapter", in_features,
            (long long)columns);
    return nullptr;
  }
  v.columns = (int)columns;
  LoraHandle* h = new (std::nothrow) LoraHandle();
  if (!h) {
    set_err(err, err_len, "out of host memory");
    return nullptr;
  }
  h->view = v;
  return h;
}

void nkt_lora_destroy(void* handle) { delete (LoraHandle*)handle; }

int nkt_lora_buffer_bytes(void* handle, int buffer, size_t* bytes, char* err, size_t err_len) {
  const LoraHandle* h = (LoraHandle*)handle;
  if (!h || !bytes) {
    set_err(err, err_len, "null handle or output pointer");
    return NKT_LORA_ERR;
  }
  const LoraView& v = h->view;
  const size_t n = v.adapters;
  switch (buffer) {
    case NKT_LORA_BUF_A: *bytes = n * v.row_blocks * 32 * v.in * 2; break;
    case NKT_LORA_BUF_B: *bytes = n * v.columns * v.rank * 2; break;
    case NKT_LORA_BUF_SCALES:
    case NKT_LORA_BUF_RANKS: *bytes = n * v.parts * 4; break;
    case NKT_LORA_BUF_STATUS: *bytes = 4; break;
    default:
      set_err(err, err_len, "buffer=%d outside [0, %d)", buffer, NKT_LORA_NUM_BUFS);
      return NKT_LORA_ERR;
  }
  return NKT_LORA_OK;
}

int nkt_lora_bind(void* handle, void* const* ptrs, char* err, size_t err_len) {
  LoraHandle* h = (LoraHandle*)handle;
  if (!h || !ptrs) {
    set_err(err, err_len, "bad arguments");
    return NKT_LORA_ERR;
  }
  for (int i = 0; i < NKT_LORA_NUM_BUFS; ++i) {
    if (!ptrs[i] || !aligned(ptrs[i], i == NKT_LORA_BUF_STATUS ? 4 : 16)) {
      set_err(err, err_len, "buffer %d: null or not 16-byte aligned", i);
      return NKT_LORA_ERR;
    }
  }
  h->view.a = (const uint16_t*)ptrs[NKT_LORA_BUF_A];
  h->view.b = (const uint16_t*)ptrs[NKT_LORA_BUF_B];
  h->view.scales = (const float*)ptrs[NKT_LORA_BUF_SCALES];
  h->view.ranks = (const int32_t*)ptrs[NKT_LORA_BUF_RANKS];
  h->view.status = (uint32_t*)ptrs[NKT_LORA_BUF_STATUS];
  h->bound = true;
  return NKT_LORA_OK;
}

int nkt_lora_workspace_bytes(void* handle, int num_tokens, size_t* bytes, char* err, size_t err_len) {
  const LoraHandle* h = (LoraHandle*)handle;
  if (!h || !bytes) {
    set_err(err, err_len, "null handle or output pointer");
    return NKT_LORA_ERR;
  }
  if (!check_tokens(num_tokens, err, err_len)) return NKT_LORA_ERR;
  *bytes = lora_workspace_bytes(h->view, num_tokens);
  return NKT_LORA_OK;
}

int nkt_lora_forward(void* handle, const void* x, int64_t x_stride, const void* base, int64_t base_stride,
                     const int64_t* index, int num_tokens, void* out, int64_t out_stride, void* workspace,
                     size_t workspace_bytes, void* stream, char* err, size_t err_len) {
  const LoraHandle* h = (LoraHandle*)handle;
  if (!h) {
    set_err(err, err_len, "null handle");
    return NKT_LORA_ERR;
  }
  if (!h->bound) {
    set_err(err, err_len, "no buffers bound (nkt_lora_bind)");
    return NKT_LORA_ERR;
  }
  if (!check_tokens(num_tokens, err, err_len)) return NKT_LORA_ERR;
  if (num_tokens == 0) return NKT_LORA_OK;
  const LoraView& v = h->view;
  if (!x || !base || !index || !out) {
    set_err(err, err_len, "null x, base, index or out");
    return NKT_LORA_ERR;
  }
  if (!aligned(x, 16) || !aligned(base, 16) || !aligned(out, 16) || x_stride % 8 || base_stride % 8 ||
      out_stride % 8) {
    set_err(err, err_len, "x, base and out (and their strides) must be 16-byte aligned");
    return NKT_LORA_ERR;
  }
  const int64_t most = (int64_t)1 << 27;
  if (num_tokens > 1 && (x_stride < 0 || x_stride > most || base_stride < 0 || base_stride > most ||
                         out_stride < v.columns || out_stride > most)) {
    set_err(err, err_len, "strides of x=%lld, base=%lld, out=%lld: 0 to 2^27 wanted, out's at least %d",
            (long long)x_stride, (long long)base_stride, (long long)out_stride, v.columns);
    return NKT_LORA_ERR;
  }
  auto span = [&](int64_t stride, int64_t width) { return ((num_tokens - 1) * stride + width) * 2; };
  const int64_t out_bytes = span(out_stride, v.columns);
  const bool same = out == base && (out_stride == base_stride || num_tokens == 1);
  if ((!same && overlap(out, out_bytes, base, span(base_stride, v.columns))) ||
      overlap(out, out_bytes, x, span(x_stride, v.in))) {
    set_err(err, err_len, "out overlaps base or x: pass base itself, or another array");
    return NKT_LORA_ERR;
  }
  const size_t need = lora_workspace_bytes(v, num_tokens);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) {
    set_err(err, err_len, "workspace of %zu bytes, 16-byte aligned, needed; got %zu", need, workspace_bytes);
    return NKT_LORA_ERR;
  }
  LoraArgs a = {};
  a.x = (const uint16_t*)x;
  a.base = (const uint16_t*)base;
  a.out = (uint16_t*)out;
  a.x_stride = x_stride;
  a.base_stride = base_stride;
  a.out_stride = out_stride;
  a.index = index;
  a.tokens = num_tokens;
  const hipError_t e = launch_lora(v, a, workspace, (hipStream_t)stream);
  if (e != hipSuccess) {
    set_err(err, err_len, "adapter kernel: %s", hipGetErrorString(e));
    return NKT_LORA_ERR;
  }
  return NKT_LORA_OK;
}

}  // extern "C"
