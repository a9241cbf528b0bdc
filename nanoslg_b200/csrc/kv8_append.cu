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
//
// What bounds it: the bytes of the rows, read once, of q_out and of the codes, written once.
// Measured (bf16, 32 / 8 heads of 128, graphs of 60 calls): prompts of 64 x 512 tokens 139 us,
// 5.3 TB/s, 0.81 of a copy's rate (181 with the reading back of what was written); 16 x 128
// behind 1024 11.4 us (46 MB: 7.0); one token for each of 64 sequences 2.9 us, most of it the
// launch and the chain plan, page, scale, codes.
#include <algorithm>

#include "kv8.cuh"
#include "launch.h"

namespace nslg {
namespace {

// Element e of a rotated row, x and y being the pair (e, e + d / 2) it belongs to (rotate-half).
template <typename T>
__device__ __forceinline__ float rotated(T x, T y, const float* c, const float* s, int e, int half) {
  const float a = Elem<T>::to_f(x), b = Elem<T>::to_f(y);
  return e < half ? __fsub_rn(__fmul_rn(a, c[e]), __fmul_rn(b, s[e]))
                  : __fadd_rn(__fmul_rn(b, c[e]), __fmul_rn(a, s[e]));
}

// The new rows of sequence b and where they start (row0: row of the first one in the row
// tensors). False, with the status set, where the plan does not fit.
struct NewRows {
  int start, kv_len, first;      // positions [start, kv_len); first entry of the page list
  int64_t row0;
};
__device__ __forceinline__ bool new_rows(const Kv8AppendParams& p, int b, bool reports, NewRows& r) {
  const int qo0 = p.qo_indptr[b], qo1 = p.qo_indptr[b + 1];
  const int ip0 = p.kv_indptr[b], ip1 = p.kv_indptr[b + 1];
  const int lpl = p.kv_lpl[b];
  const int64_t row0 = p.q_row_start != nullptr ? p.q_row_start[b] : qo0;
  const int len = qo1 - qo0;
  if (len <= 0) return false;
  r.first = ip0;
  r.kv_len = ip1 > ip0 ? (ip1 - ip0 - 1) * p.page_size + lpl : 0;
  r.start = r.kv_len - len;
  r.row0 = row0;
  if (r.start < 0 || (ip1 > ip0 && (lpl < 1 || lpl > p.page_size)) || len > p.max_qo_len || row0 < 0 ||
      row0 + len > p.num_rows) {
    if (reports) report(p.status, NSLG_DEV_BAD_PLAN);
    return false;
  }
  return true;
}

// ---------------------------------------------------------------- 16-bit rows, head_dim 64 / 128
// A thread owns 8 dims of each half of a head row (16-byte loads; rotate-half pairs them), so a
// row takes D / 16 threads.
struct Row16 {
  uint4 lo, hi;                  // dims 8c .. 8c + 7 and the same of the second half
};
struct Turn {                    // cos and sin of those dims
  float c1[8], s1[8], c2[8], s2[8];
};

template <int D>
__device__ __forceinline__ void load_turn(const float* ct, const float* st, int c, Turn& t) {
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    *reinterpret_cast<float4*>(t.c1 + i) = *reinterpret_cast<const float4*>(ct + 8 * c + i);
    *reinterpret_cast<float4*>(t.s1 + i) = *reinterpret_cast<const float4*>(st + 8 * c + i);
    *reinterpret_cast<float4*>(t.c2 + i) = *reinterpret_cast<const float4*>(ct + D / 2 + 8 * c + i);
    *reinterpret_cast<float4*>(t.s2 + i) = *reinterpret_cast<const float4*>(st + D / 2 + 8 * c + i);
  }
}

template <typename T, int D>
__device__ __forceinline__ Row16 load_row(const T* row, int c) {
  return Row16{*reinterpret_cast<const uint4*>(row + 8 * c),
               *reinterpret_cast<const uint4*>(row + D / 2 + 8 * c)};
}

// The row in fp32: v[0 .. 7] first half, v[8 .. 15] second, rotated.
template <typename T>
__device__ __forceinline__ void widen(const Row16& r, bool rot, const Turn& t, float (&v)[16]) {
  const T* x = reinterpret_cast<const T*>(&r.lo);
  const T* y = reinterpret_cast<const T*>(&r.hi);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = Elem<T>::to_f(x[i]), b = Elem<T>::to_f(y[i]);
    v[i] = rot ? __fsub_rn(__fmul_rn(a, t.c1[i]), __fmul_rn(b, t.s1[i])) : a;
    v[8 + i] = rot ? __fadd_rn(__fmul_rn(b, t.c2[i]), __fmul_rn(a, t.s2[i])) : b;
  }
}

template <typename T, int D>
__device__ __forceinline__ void store_row(T* row, int c, const float (&v)[16]) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = Mma16<T>::pack(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(row + 8 * c) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(row + D / 2 + 8 * c) = make_uint4(w[4], w[5], w[6], w[7]);
}

__device__ __forceinline__ uint32_t top_of(const float (&v)[16]) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, abs_bits(v[i]));
  return m;
}

// Codes of a row at scale s (1 / s = inv; a block that is not finite has codes of 0).
template <int D>
__device__ __forceinline__ void store_codes(uint8_t* row, int c, const float (&v)[16], float s) {
  const float inv = scale_inverse(s);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = s != s ? 0u
                  : e4m3x2_from_f32(v[4 * i] * inv, v[4 * i + 1] * inv) |
                        static_cast<uint32_t>(e4m3x2_from_f32(v[4 * i + 2] * inv, v[4 * i + 3] * inv)) << 16;
  *reinterpret_cast<uint2*>(row + 8 * c) = make_uint2(w[0], w[1]);
  *reinterpret_cast<uint2*>(row + D / 2 + 8 * c) = make_uint2(w[2], w[3]);
}

// Four codes rounded again.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio, bool nan) {
  return nan ? 0u
             : e4m3x2_rescale(static_cast<uint16_t>(w), ratio) |
                   static_cast<uint32_t>(e4m3x2_rescale(static_cast<uint16_t>(w >> 16), ratio)) << 16;
}

// Whole pages (prompts; from two new tokens on): a block owns (sequence, page) for `heads_per_block` kv heads with the
// query heads that read them; a thread owns slot tid / (D / 16) of the page for all of those
// heads, so cos and sin are read once. A head costs one barrier: the largest magnitudes of
// the 16 tokens meet in one of two rows of shared memory, used in turn. Room for 4 blocks of
// 128 threads an SM: 64 x 512 tokens take 180 us, 193 with 2 or 3 (too few loads under way),
// 186 with 5 (spills).
template <typename T, int D>
__global__ void __launch_bounds__(D, 512 / D)
    kv8_append_pages_kernel(const Kv8AppendParams p) {
  constexpr int kRow = D / 16;           // threads a row
  constexpr int kWarps = D / 32;         // 16 slots x kRow threads
  __shared__ uint32_t s_top[2][kWarps][2];
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x / p.pages_per_seq;
  const int tid = threadIdx.x, slot = tid / kRow, c = tid % kRow;
  NewRows r;
  if (!new_rows(p, b, tid == 0, r)) return;
  const int pi = r.start / 16 + static_cast<int>(blockIdx.x) % p.pages_per_seq;
  const int base = pi * 16;
  if (base >= r.kv_len) return;
  const int page = p.kv_indices[r.first + pi];
  const bool paged = page >= 0 && page < p.num_pages;
  const int pos = base + slot;
  const bool fresh = pos >= r.start && pos < r.kv_len;   // this thread's slot takes a new token
  const int older = max(r.start - base, 0);              // slots filled before this call
  const int64_t row = r.row0 + (pos - r.start);
  bool rot = p.cos_t != nullptr;
  if (rot && min(r.kv_len, base + 16) > p.table_rows) {
    if (tid == 0) report(p.status, NSLG_DEV_BAD_POSITION);
    rot = false;
  }
  Turn turn;
  if (rot && fresh)
    load_turn<D>(p.cos_t + static_cast<int64_t>(pos) * D, p.sin_t + static_cast<int64_t>(pos) * D, c, turn);
  const int h0 = blockIdx.y * p.heads_per_block, h1 = min(p.hkv, h0 + p.heads_per_block);
  for (int h = h0; h < h1; ++h) {
    float v[2][16];
    if (fresh) {
      const Row16 rk = load_row<T, D>(static_cast<const T*>(p.k) + row * p.k_stride + static_cast<int64_t>(h) * D, c);
      const Row16 rv = load_row<T, D>(static_cast<const T*>(p.v) + row * p.v_stride + static_cast<int64_t>(h) * D, c);
      if (p.q_out != nullptr) {
        const T* src = static_cast<const T*>(p.q) + row * p.q_stride + static_cast<int64_t>(h) * p.group * D;
        T* dst = static_cast<T*>(p.q_out) + (row * p.hq + static_cast<int64_t>(h) * p.group) * D;
        for (int g0 = 0; g0 < p.group; g0 += 4) {
          Row16 rq[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (g0 + i < p.group) rq[i] = load_row<T, D>(src + (g0 + i) * D, c);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (g0 + i < p.group) {
              float x[16];
              widen<T>(rq[i], rot, turn, x);
              store_row<T, D>(dst + (g0 + i) * D, c, x);
            }
        }
      }
      widen<T>(rk, rot, turn, v[0]);
      widen<T>(rv, false, turn, v[1]);
    }
    if (!paged) continue;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, fresh ? top_of(v[kv]) : 0u);
      if (tid % 32 == 0) s_top[h & 1][tid / 32][kv] = top;
    }
    const int64_t blk = static_cast<int64_t>(page) * p.hkv + h;
    const float was[2] = {older > 0 ? p.scale_k[blk] : 0.f, older > 0 ? p.scale_v[blk] : 0.f};
    __syncthreads();               // also: every thread has read the old scales
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint32_t top = 0u;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = max(top, s_top[h & 1][w][kv]);
      const float now = scale_max(was[kv], scale_from_amax(top));
      uint8_t* dst = static_cast<uint8_t*>(kv ? p.codes_v : p.codes_k) + (blk * 16 + slot) * D;
      if (fresh) {
        store_codes<D>(dst, c, v[kv], now);
      } else if (slot < older && !(now == was[kv])) {
        uint4* w = reinterpret_cast<uint4*>(dst) + c;
        const float ratio = was[kv] * scale_inverse(now);
        const bool nan = now != now;
        const uint4 x = *w;
        *w = make_uint4(rescale4(x.x, ratio, nan), rescale4(x.y, ratio, nan),
                        rescale4(x.z, ratio, nan), rescale4(x.w, ratio, nan));
      }
      if (tid == 0) (kv ? p.scale_v : p.scale_k)[blk] = now;
    }
  }
  // here, so that no row waits for the page's number
  if (!paged && tid == 0) report(p.status, NSLG_DEV_BAD_PAGE);
}

// One new token a sequence (decode): a block owns a sequence and all its heads; D / 16 lanes
// own a head row, so a row's largest magnitude is a few shuffles, and where a block's scale
// grows the same lanes round its older codes again.
template <typename T, int D>
__global__ void __launch_bounds__(512) kv8_append_token_kernel(const Kv8AppendParams p) {
  constexpr int kRow = D / 16;
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x;
  const int tid = threadIdx.x, c = tid % kRow;
  NewRows r;
  if (!new_rows(p, b, tid == 0, r)) return;
  const int pos = r.kv_len - 1, pi = pos / 16, slot = pos % 16;
  bool rot = p.cos_t != nullptr;
  if (rot && r.kv_len > p.table_rows) {
    if (tid == 0) report(p.status, NSLG_DEV_BAD_POSITION);
    rot = false;
  }
  Turn turn;
  if (rot)
    load_turn<D>(p.cos_t + static_cast<int64_t>(pos) * D, p.sin_t + static_cast<int64_t>(pos) * D, c, turn);
  const int page = p.kv_indices[r.first + pi];
  const bool paged = page >= 0 && page < p.num_pages;
  if (!paged && tid == 0) report(p.status, NSLG_DEV_BAD_PAGE);
  // rows: kv heads of K, of V, then the query heads; every lane of a warp stays in the loop
  const int rows = 2 * p.hkv + (p.q_out != nullptr ? p.hq : 0);
  const int step = blockDim.x / kRow;
  for (int i0 = 0; i0 < rows; i0 += step) {
    const int i = i0 + tid / kRow;
    const bool live = i < rows, is_q = i >= 2 * p.hkv;
    const int kv = i >= p.hkv ? 1 : 0, h = is_q ? i - 2 * p.hkv : i - kv * p.hkv;
    const int64_t blk = static_cast<int64_t>(page) * p.hkv + h;
    float* sc = (kv ? p.scale_v : p.scale_k) + blk;
    const bool writes = live && !is_q && paged;
    const float was = writes && slot > 0 ? *sc : 0.f;
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = 0.f;
    if (live) {
      const T* src = is_q ? static_cast<const T*>(p.q) + r.row0 * p.q_stride
                     : kv ? static_cast<const T*>(p.v) + r.row0 * p.v_stride
                          : static_cast<const T*>(p.k) + r.row0 * p.k_stride;
      const Row16 x = load_row<T, D>(src + static_cast<int64_t>(h) * D, c);
      widen<T>(x, rot && (is_q || kv == 0), turn, v);
    }
    uint32_t top = top_of(v);
#pragma unroll
    for (int o = 1; o < kRow; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    __syncwarp();                  // every lane of the row has read the old scale
    if (live && is_q) {
      store_row<T, D>(static_cast<T*>(p.q_out) + (r.row0 * p.hq + h) * D, c, v);
    } else if (writes) {
      uint8_t* codes = static_cast<uint8_t*>(kv ? p.codes_v : p.codes_k) + blk * 16 * D;
      const float now = scale_max(was, scale_from_amax(top));
      if (!(now == was)) {
        const float ratio = was * scale_inverse(now);
        const bool nan = now != now;
#pragma unroll 4
        for (int s = 0; s < slot; ++s) {
          uint4* w = reinterpret_cast<uint4*>(codes + s * D) + c;
          const uint4 x = *w;
          *w = make_uint4(rescale4(x.x, ratio, nan), rescale4(x.y, ratio, nan),
                          rescale4(x.z, ratio, nan), rescale4(x.w, ratio, nan));
        }
      }
      // a page that starts here takes its scale even where that is 0: its last owner's is in memory
      if (c == 0 && (slot == 0 || !(now == was))) *sc = now;
      store_codes<D>(codes + slot * D, c, v, now);
    }
  }
}

// ---------------------------------------------------------------- any shape and type
// A block a page and kv head, two codes a store, every element of K rotated twice (for the
// block's largest magnitude and for the codes): there to be right. 16 x 128 rows behind 1024, 32 / 8
// heads: 55 us for fp32, 47 at head_dim 96, 92 in pages of 32 (11 by the kernel above).
constexpr int kAppendThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const Kv8AppendParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t s_amax[2];
  const int b = blockIdx.x / p.pages_per_seq;
  const int h = blockIdx.y;
  const int tid = threadIdx.x;
  NewRows r;
  if (!new_rows(p, b, tid == 0, r)) return;
  const int start = r.start, kv_len = r.kv_len;
  const int pi = start / p.page_size + blockIdx.x % p.pages_per_seq;
  const int base = pi * p.page_size;                  // position of the page's first slot
  if (base >= kv_len) return;
  const int t0 = max(start, base), t1 = min(kv_len, base + p.page_size);
  const int d = p.d, nt = t1 - t0;
  const int64_t row = r.row0 + (t0 - start);

  bool rot = p.cos_t != nullptr;
  if (rot && t1 > p.table_rows) {
    if (tid == 0) report(p.status, NSLG_DEV_BAD_POSITION);
    rot = false;
  }
  const float* ct = p.cos_t + static_cast<int64_t>(t0) * d;
  const float* st = p.sin_t + static_cast<int64_t>(t0) * d;

  // the query heads that read this kv head
  if (p.q_out != nullptr) {
    const int half = d / 2, per_tok = p.group * half;
    for (int i = tid; i < nt * per_tok; i += kAppendThreads) {
      const int t = i / per_tok, g = i % per_tok / half, e = i % half;
      const T* src = static_cast<const T*>(p.q) + (row + t) * p.q_stride +
                     static_cast<int64_t>(h * p.group + g) * d;
      T* dst = static_cast<T*>(p.q_out) +
               ((row + t) * p.hq + h * p.group + g) * static_cast<int64_t>(d);
      // both of a rotated pair are read before either is written: dst may be src
      const float* c = ct + t * d;
      const float* s = st + t * d;
      const T x = src[e], y = src[e + half];
      dst[e] = rot ? Elem<T>::from_f(rotated(x, y, c, s, e, half)) : x;
      dst[e + half] = rot ? Elem<T>::from_f(rotated(x, y, c, s, e + half, half)) : y;
    }
  }

  const int page = p.kv_indices[r.first + pi];
  if (page < 0 || page >= p.num_pages) {
    if (tid == 0) report(p.status, NSLG_DEV_BAD_PAGE);
    return;
  }
  const int64_t blk = static_cast<int64_t>(page) * p.hkv + h;
  auto value = [&](int kv, int t, int e) -> float {
    if (kv == 0) {
      const T* src = static_cast<const T*>(p.k) + (row + t) * p.k_stride + static_cast<int64_t>(h) * d;
      const int e0 = e < d / 2 ? e : e - d / 2;
      return rot ? rotated(src[e0], src[e0 + d / 2], ct + t * d, st + t * d, e, d / 2)
                 : Elem<T>::to_f(src[e]);
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

// Reading back: the listed pages as [page_size, hkv, d] values of type T in list order; slots
// behind the sequence's last token are zeros. Rows of list entries of no sequence are left as
// they are. A thread takes 16 codes of one head row: 16-byte loads, 16-byte stores, consecutive
// threads along the output. Bound by its bytes (one read and two or four written per element):
// 16 sequences of 1152 tokens (8 heads of 128, bf16) 24.4 us, 4.6 TB/s, 2 of it the launch, fp32
// output 45 us; 1, 2 or 4 chunks a thread at a time take the same within 7 %. What holds it below a copy's rate is likely the stores: a thread's chunk is
// 32 bytes of output in two stores, so a warp's store touches 32 sectors by halves (counted).
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

// kBatch: chunks a thread holds at a time.
template <typename T, int kBatch>
__global__ void __launch_bounds__(kGatherThreads) kv8_gather_kernel(const Kv8GatherParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ int s_fill;
  const int64_t j = blockIdx.x;
  const int tid = threadIdx.x;
  if (j < p.kv_indptr[0] || j >= p.kv_indptr[p.batch]) return;
  const int64_t page = p.kv_indices[j];
  for (int b = tid; b < p.batch; b += kGatherThreads) {
    const int lo = p.kv_indptr[b], hi = p.kv_indptr[b + 1];
    if (lo <= j && j < hi) s_fill = j == hi - 1 ? p.kv_lpl[b] : p.page_size;
  }
  const bool bad = page < 0 || page >= p.num_pages;
  if (bad && tid == 0) report(p.status, NSLG_DEV_BAD_PAGE);
  const int chunks = p.d / 16, per_slot = p.hkv * chunks, n = p.page_size * per_slot;
  const int64_t blk0 = page * p.hkv;
  bool synced = false;
  const int step = kBatch * kGatherThreads * static_cast<int>(gridDim.y);
  for (int i0 = blockIdx.y * kBatch * kGatherThreads + tid; i0 - tid < n; i0 += step) {
    uint4 ck[kBatch], cv[kBatch];
    float sk[kBatch], sv[kBatch];
    int slot[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {             // every load before the first store
      const int i = i0 + u * kGatherThreads;
      slot[u] = i / per_slot;
      ck[u] = cv[u] = make_uint4(0u, 0u, 0u, 0u);
      sk[u] = sv[u] = 0.f;
      if (!bad && i < n) {
        const int r = i - slot[u] * per_slot, h = r / chunks, c = r - h * chunks;
        const int64_t off = ((blk0 + h) * p.page_size + slot[u]) * p.d + c * 16;
        ck[u] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.codes_k) + off);
        cv[u] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.codes_v) + off);
        sk[u] = p.scale_k[blk0 + h];
        sv[u] = p.scale_v[blk0 + h];
      }
    }
    if (!synced) __syncthreads();                  // s_fill
    synced = true;
    const int fill = s_fill;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = i0 + u * kGatherThreads;
      if (i >= n) break;
      const bool held = slot[u] < fill;
      const uint4 none = make_uint4(0u, 0u, 0u, 0u);
      const int64_t dst = (j * n + i) * 16;
      store16(static_cast<T*>(p.out_k) + dst, held ? ck[u] : none, held ? sk[u] : 0.f);
      store16(static_cast<T*>(p.out_v) + dst, held ? cv[u] : none, held ? sv[u] : 0.f);
    }
  }
}

}  // namespace

template <typename T, int D>
static int launch_append16(Kv8AppendParams p, cudaStream_t stream) {
  if (p.max_qo_len == 1) {
    const int64_t want = (2ll * p.hkv + (p.q_out != nullptr ? p.hq : 0)) * (D / 16);
    const int threads = static_cast<int>(want < 512 ? (want + 31) / 32 * 32 : 512);
    return launch_pdl("kv8_append", kv8_append_token_kernel<T, D>, dim3(p.batch), dim3(threads), 0,
                      stream, p);
  }
  // kv heads a block: all of them (one table read for all) while that leaves about six blocks an
  // SM; three or twelve time the same within 2 % at 16 x 128 and 64 x 512 tokens
  const int64_t pages = static_cast<int64_t>(p.batch) * p.pages_per_seq;
  const int64_t per = pages * p.hkv / (6ll * sm_count());
  p.heads_per_block = static_cast<int>(per < 1 ? 1 : per > p.hkv ? p.hkv : per);
  const dim3 grid(static_cast<unsigned>(pages), (p.hkv + p.heads_per_block - 1) / p.heads_per_block);
  return launch_pdl("kv8_append", kv8_append_pages_kernel<T, D>, grid, dim3(D), 0, stream, p);
}

int launch_kv8_append(int dtype, const Kv8AppendParams& p, cudaStream_t stream) {
  const int64_t blocks = static_cast<int64_t>(p.batch) * p.pages_per_seq;
  if (blocks > 0x7fffffff)
    return set_error(NSLG_ERR_UNSUPPORTED, "rope_kv8_append: too many pages in one call");
  if (p.page_size == 16 && (p.d == 128 || p.d == 64)) {
    if (dtype == NSLG_DTYPE_BF16)
      return p.d == 128 ? launch_append16<__nv_bfloat16, 128>(p, stream)
                        : launch_append16<__nv_bfloat16, 64>(p, stream);
    if (dtype == NSLG_DTYPE_F16)
      return p.d == 128 ? launch_append16<__half, 128>(p, stream)
                        : launch_append16<__half, 64>(p, stream);
  }
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(p.hkv));
  const dim3 block(kAppendThreads);
  if (dtype == NSLG_DTYPE_BF16)
    return launch_pdl("kv8_append", kv8_append_kernel<__nv_bfloat16>, grid, block, 0, stream, p);
  if (dtype == NSLG_DTYPE_F16)
    return launch_pdl("kv8_append", kv8_append_kernel<__half>, grid, block, 0, stream, p);
  return launch_pdl("kv8_append", kv8_append_kernel<float>, grid, block, 0, stream, p);
}

namespace {

// A page is shared by several blocks where the list is short (up to about 8 blocks an SM), down to
// a chunk a thread for lists of fewer pages than SMs. Us for 19 / 144 / 300 / 1184 pages of 8
// heads of 128: a block a page 4.4 / 5.1 / 9.3 / 25.5; shared, two chunks a thread 3.2 / 5.1 /
// 9.9 / 25.5; one chunk 2.6 / 4.9 / 11.2 / 27.4.
template <typename T, int kBatch>
int launch_gather(const Kv8GatherParams& p, cudaStream_t stream) {
  const int64_t chunks = static_cast<int64_t>(p.page_size) * p.hkv * (p.d / 16);
  const int64_t most = std::min<int64_t>((chunks + kBatch * kGatherThreads - 1) / (kBatch * kGatherThreads), 65535);
  const int64_t parts = std::max<int64_t>(std::min(8ll * sm_count() / p.num_indices, static_cast<long long>(most)), 1);
  const dim3 grid(static_cast<unsigned>(p.num_indices), static_cast<unsigned>(parts));
  return launch_pdl("kv8_gather", kv8_gather_kernel<T, kBatch>, grid, dim3(kGatherThreads), 0, stream, p);
}

template <typename T>
int launch_gather_typed(const Kv8GatherParams& p, cudaStream_t stream) {
  return p.num_indices < sm_count() ? launch_gather<T, 1>(p, stream) : launch_gather<T, 2>(p, stream);
}

}  // namespace

int launch_kv8_gather(int dtype, const Kv8GatherParams& p, cudaStream_t stream) {
  if (dtype == NSLG_DTYPE_BF16) return launch_gather_typed<__nv_bfloat16>(p, stream);
  if (dtype == NSLG_DTYPE_F16) return launch_gather_typed<__half>(p, stream);
  return launch_gather_typed<float>(p, stream);
}

}  // namespace nslg
