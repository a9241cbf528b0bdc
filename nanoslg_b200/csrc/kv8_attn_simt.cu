// Attention over the 8-bit paged cache on CUDA cores: one warp per (query row, query
// head), online softmax in fp32 over the row's visible positions, lanes splitting head_dim.
// The kernel for fp32 activations (a tensor-core product would round q) and for the shapes
// the tensor-core kernels do not take (page sizes other than 16, head_dim other than 64
// and 128, groups above 16). Decode is the qo_len == 1 case without qo_indptr.
//
// s_j = sm_scale * scale_k * (q . code_k[j]);  o = sum_j p_j scale_v code_v[j] / sum_j p_j
#include "kv8.cuh"
#include "launch.h"

namespace nslg {
namespace {

template <typename T, int DV>
__global__ void __launch_bounds__(128) kv8_attn_simt_kernel(const Kv8AttnParams p) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int hgroups = (p.hq + 3) / 4;
  const int h = static_cast<int>(blockIdx.x % hgroups) * 4 + warp;
  const int64_t bi = blockIdx.x / hgroups;
  const int i = static_cast<int>(bi % p.max_qo_len);
  const int b = static_cast<int>(bi / p.max_qo_len);
  if (h >= p.hq) return;
  const int qo0 = p.qo_indptr != nullptr ? p.qo_indptr[b] : b;
  const int qo_len = p.qo_indptr != nullptr ? p.qo_indptr[b + 1] - qo0 : 1;
  if (i >= qo_len) return;
  const int kv_beg = p.kv_indptr[b];
  const int np = p.kv_indptr[b + 1] - kv_beg;
  const int kv_len = np > 0 ? (np - 1) * p.page_size + p.kv_lpl[b] : 0;
  const int limit = p.causal ? min(kv_len, kv_len - qo_len + i + 1) : kv_len;
  const int64_t row = static_cast<int64_t>(p.q_row_start != nullptr ? p.q_row_start[b] : qo0) + i;
  if (row < 0 || row >= p.num_rows || qo_len > p.max_qo_len) {
    if (lane == 0) report(p.status, NSLG_DEV_BAD_PLAN);
    return;
  }
  const int kvh = h / (p.hq / p.hkv);
  const int d0 = lane * DV;

  float qv[DV], acc[DV];
  const T* qp = static_cast<const T*>(p.q) + row * p.q_stride + static_cast<int64_t>(h) * p.d;
#pragma unroll
  for (int e = 0; e < DV; ++e) {
    qv[e] = Elem<T>::to_f(qp[d0 + e]);
    acc[e] = 0.f;
  }
  const uint8_t* ck = static_cast<const uint8_t*>(p.codes_k);
  const uint8_t* cv = static_cast<const uint8_t*>(p.codes_v);
  auto value = [](uint8_t c) { return f32x2_from_e4m3x2(c).x; };
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < limit; ++j) {
    const int page = p.kv_indices[kv_beg + j / p.page_size];
    if (page < 0 || page >= p.num_pages) {
      if (lane == 0) report(p.status, NSLG_DEV_BAD_PAGE);
      continue;
    }
    const int64_t blk = static_cast<int64_t>(page) * p.hkv + kvh;
    const int64_t off = (blk * p.page_size + j % p.page_size) * p.d + d0;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < DV; ++e) s = fmaf(qv[e], value(ck[off + e]), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s = s * p.scale_k[blk] * p.sm_scale;
    const float m_new = fmaxf(m, s);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = expf(m - base);
    const float pw = expf(s - base);
    const float pv = pw * p.scale_v[blk];
    l = l * alpha + pw;
#pragma unroll
    for (int e = 0; e < DV; ++e) acc[e] = fmaf(pv, value(cv[off + e]), acc[e] * alpha);
    m = m_new;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* op = static_cast<T*>(p.out) + row * p.out_stride + static_cast<int64_t>(h) * p.d;
#pragma unroll
  for (int e = 0; e < DV; ++e) op[d0 + e] = Elem<T>::from_f(acc[e] * inv);
}

template <typename T>
int launch_typed(const Kv8AttnParams& p, cudaStream_t stream) {
  const int64_t blocks = static_cast<int64_t>((p.hq + 3) / 4) * p.max_qo_len * p.batch;
  if (blocks > 0x7fffffff)
    return set_error(NSLG_ERR_UNSUPPORTED, "kv8 attention: too many query rows in one call");
  const dim3 grid(static_cast<unsigned>(blocks));
  switch (p.d / 32) {
    case 1: kv8_attn_simt_kernel<T, 1><<<grid, 128, 0, stream>>>(p); break;
    case 2: kv8_attn_simt_kernel<T, 2><<<grid, 128, 0, stream>>>(p); break;
    case 3: kv8_attn_simt_kernel<T, 3><<<grid, 128, 0, stream>>>(p); break;
    case 4: kv8_attn_simt_kernel<T, 4><<<grid, 128, 0, stream>>>(p); break;
    case 5: kv8_attn_simt_kernel<T, 5><<<grid, 128, 0, stream>>>(p); break;
    case 6: kv8_attn_simt_kernel<T, 6><<<grid, 128, 0, stream>>>(p); break;
    case 7: kv8_attn_simt_kernel<T, 7><<<grid, 128, 0, stream>>>(p); break;
    default: kv8_attn_simt_kernel<T, 8><<<grid, 128, 0, stream>>>(p); break;
  }
  return check_launch("kv8_attn_simt");
}

}  // namespace

int launch_kv8_attention_simt(int dtype, const Kv8AttnParams& p, cudaStream_t stream) {
  if (dtype == NSLG_DTYPE_BF16) return launch_typed<__nv_bfloat16>(p, stream);
  if (dtype == NSLG_DTYPE_F16) return launch_typed<__half>(p, stream);
  return launch_typed<float>(p, stream);
}

}  // namespace nslg
