// RoPE + quantising append to the 8-bit paged cache, and reading it back.
//
// Append. The new rows of sequence b take its last qo_len positions, so the pages that a
// call writes, and the tokens that were in them before, follow from the page list alone.
// One block per (sequence, written page, kv head) owns the page's K and V block of that
// head: it needs the largest magnitude over all of the block's new tokens before the first
// code can be rounded, and the codes of older tokens change where the scale grows. No two
// blocks of a call touch the same bytes, so nothing is atomic and the result does not
// depend on any order. A page that starts at a new token takes no account of what was in
// it (neither codes nor scale), so a page handed out again needs no clearing.
//
//   k' = rot(k, p), v' = v            (fp32: every product and the sum rounded once)
//   s  = max(s_old if the page has older tokens, scale(max |new|))
//   code = e4m3(x / s);  older codes: e4m3(code * s_old / s) where s grew
//   q_out = rot(q, p), rounded once to the activation type
#include "kv8.cuh"
#include "launch.h"

namespace nslg {
namespace {

// Element e of a rotated row (rotate-half: dimension e is paired with e +- d / 2).
template <typename T>
__device__ __forceinline__ float rotated(const T* row, int e, int d, const float* c,
                                         const float* s) {
  const int half = d / 2;
  const float x = Elem<T>::to_f(row[e]);
  const float y = Elem<T>::to_f(row[e < half ? e + half : e - half]);
  const float yr = __fmul_rn(y, s[e]);
  return e < half ? __fsub_rn(__fmul_rn(x, c[e]), yr) : __fadd_rn(__fmul_rn(x, c[e]), yr);
}

constexpr int kAppendThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const Kv8AppendParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t s_amax[2];
  const int b = blockIdx.x / p.pages_per_seq;
  const int h = blockIdx.y;
  const int tid = threadIdx.x;
  const int qo0 = p.qo_indptr[b];
  const int qo_len = p.qo_indptr[b + 1] - qo0;
  const int ip0 = p.kv_indptr[b];
  const int np = p.kv_indptr[b + 1] - ip0;
  const int kv_len = np > 0 ? (np - 1) * p.page_size + p.kv_lpl[b] : 0;
  const int start = kv_len - qo_len;
  const int64_t row0 = p.q_row_start != nullptr ? p.q_row_start[b] : qo0;
  if (qo_len <= 0) return;
  if (start < 0 || qo_len > p.max_qo_len || row0 < 0 || row0 + qo_len > p.num_rows) {
    if (tid == 0) report(p.status, NSLG_DEV_BAD_PLAN);
    return;
  }
  const int pi = start / p.page_size + blockIdx.x % p.pages_per_seq;
  const int base = pi * p.page_size;                  // position of the page's first slot
  if (base >= kv_len) return;
  const int t0 = max(start, base), t1 = min(kv_len, base + p.page_size);
  const int d = p.d, nt = t1 - t0;
  const int64_t row = row0 + (t0 - start);

  bool rot = p.cos_t != nullptr;
  if (rot && t1 > p.table_rows) {
    if (tid == 0) report(p.status, NSLG_DEV_BAD_POSITION);
    rot = false;
  }
  const float* ct = p.cos_t + static_cast<int64_t>(t0) * d;
  const float* st = p.sin_t + static_cast<int64_t>(t0) * d;

  // the query heads that read this kv head
  if (p.q_out != nullptr) {
    const int per_tok = p.group * d;
    for (int i = tid; i < nt * per_tok; i += kAppendThreads) {
      const int t = i / per_tok, g = i % per_tok / d, e = i % d;
      const T* src = static_cast<const T*>(p.q) + (row + t) * p.q_stride +
                     static_cast<int64_t>(h * p.group + g) * d;
      T* dst = static_cast<T*>(p.q_out) +
               ((row + t) * p.hq + h * p.group + g) * static_cast<int64_t>(d);
      dst[e] = rot ? Elem<T>::from_f(rotated(src, e, d, ct + t * d, st + t * d)) : src[e];
    }
  }

  const int page = p.kv_indices[ip0 + pi];
  if (page < 0 || page >= p.num_pages) {
    if (tid == 0) report(p.status, NSLG_DEV_BAD_PAGE);
    return;
  }
  const int64_t blk = static_cast<int64_t>(page) * p.hkv + h;
  auto value = [&](int kv, int t, int e) -> float {
    if (kv == 0) {
      const T* src = static_cast<const T*>(p.k) + (row + t) * p.k_stride + static_cast<int64_t>(h) * d;
      return rot ? rotated(src, e, d, ct + t * d, st + t * d) : Elem<T>::to_f(src[e]);
    }
    return Elem<T>::to_f(
        static_cast<const T*>(p.v)[(row + t) * p.v_stride + static_cast<int64_t>(h) * d + e]);
  };
  if (tid < 2) s_amax[tid] = 0u;
  __syncthreads();
  for (int kv = 0; kv < 2; ++kv) {
    uint32_t m = 0u;
    for (int i = tid; i < nt * d; i += kAppendThreads) m = max(m, abs_bits(value(kv, i / d, i % d)));
    m = __reduce_max_sync(0xffffffffu, m);
    if (tid % 32 == 0) atomicMax(&s_amax[kv], m);
  }
  __syncthreads();
  const int older = t0 - base;
  float was[2], now[2];
  for (int kv = 0; kv < 2; ++kv) {
    const float* sc = kv == 0 ? p.scale_k : p.scale_v;
    was[kv] = older > 0 ? sc[blk] : 0.f;
    now[kv] = scale_max(was[kv], scale_from_amax(s_amax[kv]));
  }
  __syncthreads();   // every thread has read the old scales
  for (int kv = 0; kv < 2; ++kv) {
    uint8_t* codes = static_cast<uint8_t*>(kv == 0 ? p.codes_k : p.codes_v) +
                     blk * p.page_size * d;
    if (tid == 0) (kv == 0 ? p.scale_k : p.scale_v)[blk] = now[kv];
    // a block that is not finite: every code 0, its NaN is the scale
    const bool nan = now[kv] != now[kv];
    if (older > 0 && !(now[kv] == was[kv])) {
      const float ratio = was[kv] * scale_inverse(now[kv]);
      uint16_t* c2 = reinterpret_cast<uint16_t*>(codes);
      for (int i = tid; i < older * d / 2; i += kAppendThreads) c2[i] = nan ? 0 : e4m3x2_rescale(c2[i], ratio);
    }
    const float inv = scale_inverse(now[kv]);
    uint16_t* dst = reinterpret_cast<uint16_t*>(codes + static_cast<int64_t>(older) * d);
    for (int i = tid; i < nt * d / 2; i += kAppendThreads) {
      const int t = i / (d / 2), e = i % (d / 2) * 2;
      dst[i] = nan ? 0 : e4m3x2_from_f32(value(kv, t, e) * inv, value(kv, t, e + 1) * inv);
    }
  }
}

// Reading back: one block per listed page, [page_size, hkv, d] values of type T in list
// order; slots behind the sequence's last token are zeros. Rows of pages behind the last
// listed one are left as they are. A thread takes 16 codes of one head row: 16-byte loads,
// 16-byte stores, consecutive threads along the output. Bound by its bytes (one read and two
// or four written per element).
//
// kStage: the pages staged for the 16-bit prefill kernel, which reads them through an
// identity page list (`ids`). There the value of a masked position still meets a probability
// of 0 in a product, so the NaN of a V block is moved to its K block, whose scores are masked
// by selection; and rows that see no position, which that kernel does not visit, are zeroed.
constexpr int kGatherThreads = 256;

template <typename T>
__device__ __forceinline__ void store16(T* dst, const uint4& c, float sc) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  constexpr int kPer = 16 / sizeof(T);           // elements per 16-byte store
  alignas(16) T v[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = f32x2_from_e4m3x2(static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1))));
    v[2 * i] = from_cache<T>(f.x * sc);
    v[2 * i + 1] = from_cache<T>(f.y * sc);
  }
#pragma unroll
  for (int i = 0; i < 16; i += kPer)
    *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<const uint4*>(v + i);
}

template <typename T, bool kStage>
__global__ void __launch_bounds__(kGatherThreads) kv8_gather_kernel(const Kv8GatherParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ int s_fill;
  const int64_t j = blockIdx.x;
  const int tid = threadIdx.x;
  if constexpr (kStage) {
    for (int64_t b = j; b < p.batch; b += gridDim.x) {
      const int q0 = p.qo_indptr[b], len = p.qo_indptr[b + 1] - q0;
      const int np = p.kv_indptr[b + 1] - p.kv_indptr[b];
      const int kv_len = np > 0 ? (np - 1) * p.page_size + p.kv_lpl[b] : 0;
      const int none = kv_len == 0 ? len : p.causal ? len - kv_len : 0;
      const int64_t row0 = p.q_row_start != nullptr ? p.q_row_start[b] : q0;
      if (none <= 0 || len > p.max_qo_len || row0 < 0 || row0 + len > p.num_rows) continue;
      const int words = p.hq * p.d * static_cast<int>(sizeof(T)) / 16;
      for (int64_t i = tid; i < static_cast<int64_t>(none) * words; i += kGatherThreads)
        reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (row0 + i / words) * p.out_stride)[i % words] =
            make_uint4(0u, 0u, 0u, 0u);
    }
    if (tid == 0) p.ids[j] = static_cast<int32_t>(j);
  }
  if (j >= p.kv_indptr[p.batch]) return;
  const int64_t page = p.kv_indices[j];
  for (int b = tid; b < p.batch; b += kGatherThreads) {
    const int lo = p.kv_indptr[b], hi = p.kv_indptr[b + 1];
    if (lo <= j && j < hi) s_fill = j == hi - 1 ? p.kv_lpl[b] : p.page_size;
  }
  __syncthreads();
  const int fill = s_fill;
  const bool bad = page < 0 || page >= p.num_pages;
  if (bad && tid == 0) report(p.status, NSLG_DEV_BAD_PAGE);
  const int chunks = p.d / 16, per_slot = p.hkv * chunks, n = p.page_size * per_slot;
  const int64_t blk0 = page * p.hkv;
  for (int i = tid; i < n; i += kGatherThreads) {
    const int s = i / per_slot, r = i - s * per_slot, h = r / chunks, c = r - h * chunks;
    uint4 ck = make_uint4(0u, 0u, 0u, 0u), cv = ck;
    float sk = 0.f, sv = 0.f;
    if (!bad && s < fill) {
      const int64_t off = ((blk0 + h) * p.page_size + s) * p.d + c * 16;
      ck = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.codes_k) + off);
      cv = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.codes_v) + off);
      sk = p.scale_k[blk0 + h];
      sv = p.scale_v[blk0 + h];
      if (kStage && sv != sv) {
        sk = sv;
        sv = 0.f;
      }
    }
    const int64_t dst = (j * n + i) * 16;
    store16(static_cast<T*>(p.out_k) + dst, ck, sk);
    store16(static_cast<T*>(p.out_v) + dst, cv, sv);
  }
}

}  // namespace

int launch_kv8_append(int dtype, const Kv8AppendParams& p, cudaStream_t stream) {
  const int64_t blocks = static_cast<int64_t>(p.batch) * p.pages_per_seq;
  if (blocks > 0x7fffffff)
    return set_error(NSLG_ERR_UNSUPPORTED, "rope_kv8_append: too many pages in one call");
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(p.hkv));
  const dim3 block(kAppendThreads);
  if (dtype == NSLG_DTYPE_BF16)
    return launch_pdl("kv8_append", kv8_append_kernel<__nv_bfloat16>, grid, block, 0, stream, p);
  if (dtype == NSLG_DTYPE_F16)
    return launch_pdl("kv8_append", kv8_append_kernel<__half>, grid, block, 0, stream, p);
  return launch_pdl("kv8_append", kv8_append_kernel<float>, grid, block, 0, stream, p);
}

int launch_kv8_gather(int dtype, const Kv8GatherParams& p, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.num_indices)), block(kGatherThreads);
  if (dtype == NSLG_DTYPE_BF16)
    return launch_pdl("kv8_gather", kv8_gather_kernel<__nv_bfloat16, false>, grid, block, 0, stream, p);
  if (dtype == NSLG_DTYPE_F16)
    return launch_pdl("kv8_gather", kv8_gather_kernel<__half, false>, grid, block, 0, stream, p);
  return launch_pdl("kv8_gather", kv8_gather_kernel<float, false>, grid, block, 0, stream, p);
}

int launch_kv8_stage(int dtype, const Kv8GatherParams& p, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.num_indices)), block(kGatherThreads);
  if (dtype == NSLG_DTYPE_BF16)
    return launch_pdl("kv8_stage", kv8_gather_kernel<__nv_bfloat16, true>, grid, block, 0, stream, p);
  return launch_pdl("kv8_stage", kv8_gather_kernel<__half, true>, grid, block, 0, stream, p);
}

}  // namespace nslg
