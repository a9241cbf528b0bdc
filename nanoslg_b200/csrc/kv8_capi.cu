// extern "C" entry points of the 8-bit KV cache (include/nslg_b200.h): argument checks and
// the choice of kernel. Nothing is thrown across the boundary.
#include <algorithm>
#include <string>

#include "launch.h"

using namespace nslg;

namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Sizes and pointers every entry point of the cache shares.
int check_cache(const std::string& what, int dtype, int batch, int hkv, int d, int page_size,
                const Kv8Cache& c) {
  if (dtype != NSLG_DTYPE_BF16 && dtype != NSLG_DTYPE_F16 && dtype != NSLG_DTYPE_F32)
    return set_error(NSLG_ERR_ARG, what + ": bad dtype");
  if (batch < 0) return set_error(NSLG_ERR_ARG, what + ": batch < 0");
  if (hkv <= 0 || hkv > 65535) return set_error(NSLG_ERR_ARG, what + ": bad num_kv_heads");
  if (d <= 0 || d % 32 || d > 256)
    return set_error(NSLG_ERR_UNSUPPORTED, what + ": head_dim must be a multiple of 32, at most 256");
  if (page_size <= 0 || page_size > 65536 || c.num_pages <= 0)
    return set_error(NSLG_ERR_ARG, what + ": page_size and num_pages must be positive");
  if (static_cast<int64_t>(page_size) * hkv * d >= (int64_t{1} << 31))
    return set_error(NSLG_ERR_UNSUPPORTED, what + ": a page of 2^31 elements or more");
  if (!c.codes_k || !c.codes_v || !c.scale_k || !c.scale_v)
    return set_error(NSLG_ERR_ARG, what + ": null cache pointer");
  if (!c.kv_indptr || !c.kv_indices || !c.kv_lpl)
    return set_error(NSLG_ERR_ARG, what + ": null page list");
  if (!aligned(c.codes_k, 16) || !aligned(c.codes_v, 16) || !aligned(c.scale_k, 4) ||
      !aligned(c.scale_v, 4))
    return set_error(NSLG_ERR_ARG, what + ": the codes must be 16-byte aligned");
  return NSLG_OK;
}

int check_rows(const std::string& what, const char* name, const void* p, int64_t stride,
               int64_t width, int dtype) {
  const int64_t es = dtype_bytes(dtype);
  if (!aligned(p, 16) || (stride * es) % 16 || stride < width)
    return set_error(NSLG_ERR_ARG, what + ": " + name +
                                       " rows must be 16-byte aligned and its stride cover a row");
  return NSLG_OK;
}

int check_attention(const std::string& what, int dtype, const Kv8AttnParams& p) {
  int rc = check_cache(what, dtype, p.batch, p.hkv, p.d, p.page_size, p);
  if (rc) return rc;
  if (p.hq <= 0 || p.hq % p.hkv)
    return set_error(NSLG_ERR_ARG, what + ": need num_qo_heads % num_kv_heads == 0");
  if (!p.q || !p.out) return set_error(NSLG_ERR_ARG, what + ": null pointer");
  if (!(p.sm_scale > 0.f)) return set_error(NSLG_ERR_ARG, what + ": sm_scale must be > 0");
  const int64_t width = static_cast<int64_t>(p.hq) * p.d;
  if ((rc = check_rows(what, "q", p.q, p.q_stride, width, dtype))) return rc;
  if ((rc = check_rows(what, "out", p.out, p.out_stride, width, dtype))) return rc;
  return NSLG_OK;
}

template <typename F>
int guarded(F&& f) {
  try {
    clear_error();
    return f();
  } catch (...) {
    return NSLG_ERR_CUDA;
  }
}

}  // namespace

extern "C" {

int nslg_rope_kv8_append(int dtype, int batch, int num_qo_heads, int num_kv_heads, int head_dim,
                         int page_size, const void* q, int64_t q_stride, const void* k,
                         int64_t k_stride, const void* v, int64_t v_stride, int64_t num_rows,
                         void* q_out, const float* cos_table, const float* sin_table,
                         int64_t table_rows, void* codes_k, void* codes_v, float* scale_k,
                         float* scale_v, int64_t num_pages, const int32_t* qo_indptr,
                         const int32_t* q_row_start, int max_qo_len, const int32_t* kv_indptr,
                         const int32_t* kv_indices, const int32_t* kv_last_page_len,
                         uint32_t* dev_status, void* stream) {
  return guarded([&]() -> int {
    const std::string what = "rope_kv8_append";
    Kv8AppendParams p{};
    p.codes_k = codes_k;
    p.codes_v = codes_v;
    p.scale_k = scale_k;
    p.scale_v = scale_v;
    p.num_pages = num_pages;
    p.kv_indptr = kv_indptr;
    p.kv_indices = kv_indices;
    p.kv_lpl = kv_last_page_len;
    if (batch == 0 || max_qo_len == 0) return NSLG_OK;
    int rc = check_cache(what, dtype, batch, num_kv_heads, head_dim, page_size, p);
    if (rc) return rc;
    if (max_qo_len < 0 || num_rows < 0)
      return set_error(NSLG_ERR_ARG, what + ": negative max_qo_len or num_rows");
    if (num_qo_heads <= 0 || num_qo_heads % num_kv_heads)
      return set_error(NSLG_ERR_ARG, what + ": need num_qo_heads % num_kv_heads == 0");
    if (!k || !v || !qo_indptr) return set_error(NSLG_ERR_ARG, what + ": null pointer");
    if (q_out != nullptr && q == nullptr)
      return set_error(NSLG_ERR_ARG, what + ": q_out given without q");
    if ((cos_table == nullptr) != (sin_table == nullptr) || (cos_table && table_rows <= 0))
      return set_error(NSLG_ERR_ARG, what + ": the rotation needs both cos and sin tables");
    const int64_t kvw = static_cast<int64_t>(num_kv_heads) * head_dim;
    const int64_t qw = static_cast<int64_t>(num_qo_heads) * head_dim;
    if ((rc = check_rows(what, "k", k, k_stride, kvw, dtype))) return rc;
    if ((rc = check_rows(what, "v", v, v_stride, kvw, dtype))) return rc;
    if (q_out && (rc = check_rows(what, "q", q, q_stride, qw, dtype))) return rc;
    if (q_out && (rc = check_rows(what, "q_out", q_out, qw, qw, dtype))) return rc;
    if (!aligned(cos_table, 16) || !aligned(sin_table, 16))
      return set_error(NSLG_ERR_ARG, what + ": cos/sin tables must be 16-byte aligned");
    p.q = q_out ? q : nullptr;
    p.k = k;
    p.v = v;
    p.q_out = q_out;
    p.cos_t = cos_table;
    p.sin_t = sin_table;
    p.qo_indptr = qo_indptr;
    p.q_row_start = q_row_start;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.num_rows = num_rows;
    p.table_rows = table_rows;
    p.batch = batch;
    p.hq = num_qo_heads;
    p.hkv = num_kv_heads;
    p.d = head_dim;
    p.page_size = page_size;
    p.group = num_qo_heads / num_kv_heads;
    if (static_cast<int64_t>(page_size) * p.group * head_dim >= (int64_t{1} << 31))
      return set_error(NSLG_ERR_UNSUPPORTED, what + ": a page's query rows of 2^31 elements or more");
    if (num_rows == 0) return NSLG_OK;
    p.max_qo_len = static_cast<int>(std::min<int64_t>(max_qo_len, num_rows));   // more never fit
    p.pages_per_seq = static_cast<int>((static_cast<int64_t>(p.max_qo_len) + page_size - 2) / page_size) + 1;
    p.status = dev_status;
    return launch_kv8_append(dtype, p, static_cast<cudaStream_t>(stream));
  });
}

int nslg_kv8_gather(int dtype, int batch, int num_kv_heads, int head_dim, int page_size,
                    const void* codes_k, const void* codes_v, const float* scale_k,
                    const float* scale_v, int64_t num_pages, const int32_t* kv_indptr,
                    const int32_t* kv_indices, const int32_t* kv_last_page_len,
                    int64_t num_indices, void* out_k, void* out_v, uint32_t* dev_status,
                    void* stream) {
  return guarded([&]() -> int {
    const std::string what = "kv8_gather";
    Kv8GatherParams p{};
    p.codes_k = const_cast<void*>(codes_k);
    p.codes_v = const_cast<void*>(codes_v);
    p.scale_k = const_cast<float*>(scale_k);
    p.scale_v = const_cast<float*>(scale_v);
    p.num_pages = num_pages;
    p.kv_indptr = kv_indptr;
    p.kv_indices = kv_indices;
    p.kv_lpl = kv_last_page_len;
    if (batch == 0 || num_indices == 0) return NSLG_OK;
    const int rc = check_cache(what, dtype, batch, num_kv_heads, head_dim, page_size, p);
    if (rc) return rc;
    if (num_indices < 0 || num_indices > 0x7fffffff)
      return set_error(NSLG_ERR_ARG, what + ": num_indices out of range");
    if (!out_k || !out_v) return set_error(NSLG_ERR_ARG, what + ": null pointer");
    if (!aligned(out_k, 16) || !aligned(out_v, 16))
      return set_error(NSLG_ERR_ARG, what + ": the outputs must be 16-byte aligned");
    p.out_k = out_k;
    p.out_v = out_v;
    p.num_indices = num_indices;
    p.batch = batch;
    p.hkv = num_kv_heads;
    p.d = head_dim;
    p.page_size = page_size;
    p.status = dev_status;
    return launch_kv8_gather(dtype, p, static_cast<cudaStream_t>(stream));
  });
}

int64_t nslg_decode_kv8_workspace_bytes(int batch, int num_qo_heads, int num_kv_heads,
                                        int head_dim) {
  if (batch < 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      num_qo_heads % num_kv_heads)
    return 0;
  return kv8_attn_tc_workspace_bytes(num_qo_heads / num_kv_heads, 1, head_dim);
}

int nslg_paged_decode_kv8(int dtype, int batch, int num_qo_heads, int num_kv_heads, int head_dim,
                          int page_size, const void* q, int64_t q_stride, void* out,
                          int64_t out_stride, const void* codes_k, const void* codes_v,
                          const float* scale_k, const float* scale_v, int64_t num_pages,
                          const int32_t* kv_indptr, const int32_t* kv_indices,
                          const int32_t* kv_last_page_len, float sm_scale, void* workspace,
                          int64_t workspace_bytes, uint32_t* dev_status, void* stream) {
  return guarded([&]() -> int {
    if (batch == 0) return NSLG_OK;
    Kv8AttnParams p{};
    p.codes_k = const_cast<void*>(codes_k);
    p.codes_v = const_cast<void*>(codes_v);
    p.scale_k = const_cast<float*>(scale_k);
    p.scale_v = const_cast<float*>(scale_v);
    p.num_pages = num_pages;
    p.kv_indptr = kv_indptr;
    p.kv_indices = kv_indices;
    p.kv_lpl = kv_last_page_len;
    p.q = q;
    p.out = out;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.num_rows = batch;
    p.batch = batch;
    p.hq = num_qo_heads;
    p.hkv = num_kv_heads;
    p.d = head_dim;
    p.page_size = page_size;
    p.max_qo_len = 1;
    p.causal = 0;
    p.sm_scale = sm_scale;
    p.status = dev_status;
    const int rc = check_attention("paged_decode_kv8", dtype, p);
    if (rc) return rc;
    if (kv8_attn_tc_supported(dtype, p))
      return launch_kv8_attention_tc(dtype, p, workspace, workspace_bytes,
                                     static_cast<cudaStream_t>(stream));
    return launch_kv8_attention_simt(dtype, p, static_cast<cudaStream_t>(stream));
  });
}

int64_t nslg_prefill_kv8_workspace_bytes(int num_qo_heads, int num_kv_heads, int head_dim,
                                         int max_qo_len) {
  if (num_qo_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || max_qo_len < 0 ||
      num_qo_heads % num_kv_heads)
    return 0;
  return kv8_attn_tc_workspace_bytes(num_qo_heads / num_kv_heads, max_qo_len, head_dim);
}

int nslg_paged_prefill_kv8(int dtype, int batch, int num_qo_heads, int num_kv_heads, int head_dim,
                           int page_size, const void* q, int64_t q_stride, int64_t q_rows,
                           void* out, int64_t out_stride, const int32_t* qo_indptr,
                           const int32_t* q_row_start, int max_qo_len, const void* codes_k,
                           const void* codes_v, const float* scale_k, const float* scale_v,
                           int64_t num_pages, const int32_t* kv_indptr, const int32_t* kv_indices,
                           const int32_t* kv_last_page_len, float sm_scale, int causal,
                           void* workspace, int64_t workspace_bytes, uint32_t* dev_status,
                           void* stream) {
  return guarded([&]() -> int {
    const std::string what = "paged_prefill_kv8";
    if (batch == 0 || max_qo_len == 0) return NSLG_OK;
    if (max_qo_len < 0 || q_rows <= 0)
      return set_error(NSLG_ERR_ARG, what + ": bad max_qo_len or q_rows");
    if (!qo_indptr) return set_error(NSLG_ERR_ARG, what + ": null pointer");
    Kv8AttnParams p{};
    p.codes_k = const_cast<void*>(codes_k);
    p.codes_v = const_cast<void*>(codes_v);
    p.scale_k = const_cast<float*>(scale_k);
    p.scale_v = const_cast<float*>(scale_v);
    p.num_pages = num_pages;
    p.kv_indptr = kv_indptr;
    p.kv_indices = kv_indices;
    p.kv_lpl = kv_last_page_len;
    p.q = q;
    p.out = out;
    p.qo_indptr = qo_indptr;
    p.q_row_start = q_row_start;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.num_rows = q_rows;
    p.batch = batch;
    p.hq = num_qo_heads;
    p.hkv = num_kv_heads;
    p.d = head_dim;
    p.page_size = page_size;
    p.max_qo_len = static_cast<int>(std::min<int64_t>(max_qo_len, q_rows));   // more never fit
    p.causal = causal ? 1 : 0;
    p.sm_scale = sm_scale;
    p.status = dev_status;
    const int rc = check_attention(what, dtype, p);
    if (rc) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (kv8_prefill_tc_supported(dtype, p) &&
        (kv8_prefill_tc_faster(p) || !kv8_attn_tc_supported(dtype, p)))
      return launch_kv8_prefill_tc(dtype, p, st);
    if (kv8_attn_tc_supported(dtype, p))
      return launch_kv8_attention_tc(dtype, p, workspace, workspace_bytes, st);
    return launch_kv8_attention_simt(dtype, p, st);
  });
}

int nslg_stream_capture_id(void* stream, uint64_t* id) {
  return guarded([&]() -> int {
    if (id == nullptr) return set_error(NSLG_ERR_ARG, "stream_capture_id: null pointer");
    *id = 0;
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    unsigned long long n = 0;
    const cudaError_t err = cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &st, &n);
    if (err != cudaSuccess) return set_error(NSLG_ERR_CUDA, cudaGetErrorString(err));
    if (st == cudaStreamCaptureStatusActive) *id = n;
    return NSLG_OK;
  });
}

}  // extern "C"
