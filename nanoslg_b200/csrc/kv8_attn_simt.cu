// Attention over the 8-bit paged cache on CUDA cores: a block per (query row, query head), its
// warps taking the row's visible positions kStep at a time in turn, each with an online
// softmax of its own in fp32, lanes splitting head_dim; the warps' parts are joined at the end.
// The kernel for fp32 activations (a tensor-core product would round q) and for the shapes
// the tensor-core kernels do not take (page sizes other than 16, head_dim other than 64
// and 128). Decode is the qo_len == 1 case without qo_indptr.
//
// s_j = sm_scale * scale_k * (q . code_k[j]);  o = sum_j p_j scale_v code_v[j] / sum_j p_j
//
// Bound by the latency of a step's loads and by its instructions, every query head reading its
// kv head's codes again: it is there to be right. Decode of 513 tokens, fp32, 32 / 8 heads of
// 128: 26 us (238 with a warp to a head and a position at a time); of 64 sequences of 768
// 325 us, in bf16 and pages of 32 339; prompts of 8 x 512 in fp32 5.8 ms.
#include "kv8.cuh"
#include "launch.h"

namespace nslg {
namespace {

constexpr int kWarps = 8;
constexpr int kStep = 4;                 // positions whose loads are under way at once

template <typename T, int DV>
__global__ void __launch_bounds__(kWarps * 32) kv8_attn_simt_kernel(const Kv8AttnParams p) {
  __shared__ float s_m[kWarps], s_l[kWarps], s_acc[kWarps][DV * 32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int h = static_cast<int>(blockIdx.x % p.hq);
  const int64_t bi = blockIdx.x / p.hq;
  const int i = static_cast<int>(bi % p.max_qo_len);
  const int b = static_cast<int>(bi / p.max_qo_len);
  const int qo0 = p.qo_indptr != nullptr ? p.qo_indptr[b] : b;
  const int qo_len = p.qo_indptr != nullptr ? p.qo_indptr[b + 1] - qo0 : 1;
  if (i >= qo_len) return;
  const int kv_beg = p.kv_indptr[b];
  const int np = p.kv_indptr[b + 1] - kv_beg;
  const int lpl = p.kv_lpl[b];
  const int kv_len = np > 0 ? (np - 1) * p.page_size + lpl : 0;
  const int limit = p.causal ? min(kv_len, kv_len - qo_len + i + 1) : kv_len;
  const int64_t row = static_cast<int64_t>(p.q_row_start != nullptr ? p.q_row_start[b] : qo0) + i;
  if (row < 0 || row >= p.num_rows || qo_len > p.max_qo_len ||
      (np > 0 && (lpl < 1 || lpl > p.page_size))) {
    if (threadIdx.x == 0) report(p.status, NSLG_DEV_BAD_PLAN);
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
  for (int j0 = warp * kStep; j0 < limit; j0 += kWarps * kStep) {
    uint8_t kc[kStep][DV], vc[kStep][DV];
    float sk[kStep], sv[kStep];
    bool has[kStep];
#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      const int j = j0 + u;
      const int page = j < limit ? p.kv_indices[kv_beg + j / p.page_size] : -1;
      has[u] = page >= 0 && page < p.num_pages;
      if (j < limit && !has[u] && lane == 0) report(p.status, NSLG_DEV_BAD_PAGE);
      const int64_t blk = static_cast<int64_t>(has[u] ? page : 0) * p.hkv + kvh;
      const int64_t off = (blk * p.page_size + j % p.page_size) * p.d + d0;
      sk[u] = p.scale_k[blk];
      sv[u] = p.scale_v[blk];
#pragma unroll
      for (int e = 0; e < DV; ++e) {
        kc[u][e] = ck[off + e];
        vc[u][e] = cv[off + e];
      }
    }
    float s[kStep], top = m;
#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      s[u] = 0.f;
#pragma unroll
      for (int e = 0; e < DV; ++e) s[u] = fmaf(qv[e], value(kc[u][e]), s[u]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < kStep; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], o);
#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      s[u] = s[u] * sk[u] * p.sm_scale;
      if (has[u]) top = fmaxf(top, s[u]);
    }
    const float base = top == -INFINITY ? 0.f : top;
    const float alpha = expf(m - base);
    l *= alpha;
#pragma unroll
    for (int e = 0; e < DV; ++e) acc[e] *= alpha;
#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      if (!has[u]) continue;
      const float pw = expf(s[u] - base), pv = pw * sv[u];
      l += pw;
#pragma unroll
      for (int e = 0; e < DV; ++e) acc[e] = fmaf(pv, value(vc[u][e]), acc[e]);
    }
    m = top;
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < DV; ++e) s_acc[warp][d0 + e] = acc[e];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
  const float base = top == -INFINITY ? 0.f : top;
  float part[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    part[w] = expf(s_m[w] - base);
    sum = fmaf(part[w], s_l[w], sum);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* op = static_cast<T*>(p.out) + row * p.out_stride + static_cast<int64_t>(h) * p.d;
  for (int e = threadIdx.x; e < DV * 32; e += kWarps * 32) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) o = fmaf(part[w], s_acc[w][e], o);
    op[e] = Elem<T>::from_f(o * inv);
  }
}

template <typename T>
int launch_typed(const Kv8AttnParams& p, cudaStream_t stream) {
  const int64_t blocks = static_cast<int64_t>(p.hq) * p.max_qo_len * p.batch;
  if (blocks > 0x7fffffff)
    return set_error(NSLG_ERR_UNSUPPORTED, "kv8 attention: too many query rows in one call");
  const dim3 grid(static_cast<unsigned>(blocks));
  switch (p.d / 32) {
    case 1: kv8_attn_simt_kernel<T, 1><<<grid, kWarps * 32, 0, stream>>>(p); break;
    case 2: kv8_attn_simt_kernel<T, 2><<<grid, kWarps * 32, 0, stream>>>(p); break;
    case 3: kv8_attn_simt_kernel<T, 3><<<grid, kWarps * 32, 0, stream>>>(p); break;
    case 4: kv8_attn_simt_kernel<T, 4><<<grid, kWarps * 32, 0, stream>>>(p); break;
    case 5: kv8_attn_simt_kernel<T, 5><<<grid, kWarps * 32, 0, stream>>>(p); break;
    case 6: kv8_attn_simt_kernel<T, 6><<<grid, kWarps * 32, 0, stream>>>(p); break;
    case 7: kv8_attn_simt_kernel<T, 7><<<grid, kWarps * 32, 0, stream>>>(p); break;
    default: kv8_attn_simt_kernel<T, 8><<<grid, kWarps * 32, 0, stream>>>(p); break;
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
