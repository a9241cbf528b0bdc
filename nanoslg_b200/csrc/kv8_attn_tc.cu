// Split-KV attention over the 8-bit paged cache for decode steps and for a few new rows on
// a long context: page_size 16, head_dim 64 or 128, 16-bit activations, any head counts.
//
// What bounds it: the bytes of the cache, one per element, read once. So every SM streams
// an equal share of them whatever the sequences' lengths, and the arithmetic per byte is
// kept below what an SM can issue in the time its share of the bandwidth takes. Measured
// (bf16, 32 / 8 heads of 128, graphs of 60 calls): 64 sequences of 512 to 8192 tokens 103 us,
// 5.8 TB/s, 0.89 of a copy's rate (110 us over seconds); 64 of 513 to 768 24.4 us (87 MB: 13.3
// at that rate, and about 10 us of launch, plan, first loads and joining, none of which the
// batch's size changes); one of 513 9.0 us. The page list is read behind the kernel in front,
// like all else: reading it ahead of that saved 0.7 to 1.4 us a call and took a list that the
// kernel in front had yet to write.
//
// Work split. A unit is one page of one kv head: 16 tokens, K and V blocks of 16 * head_dim
// bytes each, contiguous, with one scale each. A "virtual sequence" is (sequence, kv head,
// tile of 8 NT query rows), its rows being the (new token, query head of the group) pairs that
// read this kv head. The units of all virtual sequences form one flat list (U = pages x kv
// heads x tiles), and CTA c of n takes [U c / n, U (c + 1) / n), each of its W warps an
// equal contiguous part of that, n = min(#SMs, U / W). It is computed on the device from kv_indptr:
// no host-side plan, replayable in a CUDA graph. Splitting by kv head (not only by pages)
// spreads one short sequence over as many warps as it has units, and keeps a partial to one
// group's rows, so a batch costs about one partial per CTA boundary.
//
// A warp is a pipeline of its own: lane i & 31 holds the page id and the scales of unit i,
// issues the two TMA loads (2 KiB each at head_dim 128, 128-byte swizzle, no multicast) into
// one of the warp's `stages` slots, and refills a slot as soon as the warp has read it, so
// there is no producer warp and no barrier between warps before the end.
//
// Mathematics of a unit, transposed so that a short group wastes little of an mma: the 16
// tokens (of K) and 16-dim chunks (of V) are the rows of m16n8k16 products, the query rows
// their 8 columns (one or two column tiles, NT):
//   s^T = code_k . q^T  (16 tokens x 8 NT rows)
//   t = s F + E          F = scale_k sm_scale log2(e) / (the row's q factor), E = log2 scale_v
//   p = 2^(t - M)        M: running reference, raised only when t passes it by 8 (p <= 2^8)
//   o^T = o^T + code_v^T . p^T;  l = l + 2^-E sum p;  out = o / l
// The scales cost nothing per element: K's is a factor the score needs anyway, V's joins the
// exponent, so p is what multiplies the code and M follows the largest of these weights.
// p is rounded to f16 (2^-11, whatever the activation type) relative to that, so the scales
// of neighbouring pages may differ by any factor. Blocks of zeros in V, which have no E, stand
// at kZeroE.
// Against rows-first products (16 query rows, 4 of them in use at a group of 4) this halves
// the products, the accumulators (32 registers instead of 64 at head_dim 128, so 12 warps
// fit an SM instead of 8) and the exponentials.
// Codes become f16 exactly (one cvt per two). q of bf16 becomes f16 exactly too: each row is
// first multiplied by the power of two that brings its largest magnitude to [2^14, 2^15)
// (elements 2^-38 below it vanish).
// Operand layouts: the order of head_dim inside a k step of K.q is free as long as q and K
// agree, so K fragments are plain ldmatrix words (4 codes = dims 4t .. 4t + 3 of a 16-dim
// chunk) and q is loaded to match. V^T comes from ldmatrix.trans of 16-bit units (two dims
// of one token); one byte permute pairs the tokens, and row g / g + 8 of the chunk's product
// is dim 2g / 2g + 1. p^T is the scores' fragment transposed by movmatrix.
// A block whose scale is NaN reads as NaN: its NaN is put on the scores (masked like them),
// so a row that sees nothing of the block is not touched. Codes behind a sequence's last
// token may be anything, NaN codes too: they are cleared in V and masked in the scores.
//
// Joining. A virtual sequence inside one warp's part is written straight to `out`. Pieces of
// the warps of one CTA meet in shared memory. One that spans CTAs leaves a partial (o, m, l)
// per CTA in the workspace; the CTA that arrives last, by a count per first CTA, joins them in
// CTA order and puts the count back to zero. No CTA waits for another, and the sums do not
// depend on who is last.
#include <cuda.h>

#include <string>
#include <type_traits>

#include "kv8.cuh"
#include "launch.h"

namespace nslg {
namespace {

constexpr int kPS = 16;
constexpr int kMaxStages = 8;
constexpr int kStaticSmem = 2048;     // at least the kernel's __shared__ arrays
constexpr int kMaxSmem = 232448;      // 227 KiB
constexpr int kSmemBatch = 2048;      // batches up to this size keep the page list's bounds in smem
constexpr float kHeadroom = 8.f;      // log2 of the largest probability before m is raised

struct TcParams : Kv8AttnParams {
  float* part_o;        // [2 * grid][rows][D]
  float* part_ml;       // [2 * grid][rows][2]
  uint32_t* arrive;     // [grid]
  int group, tiles, rows, stages, grid, smem_csr;
  float scale_log2;
};

// W warps a CTA, one CTA an SM. With 12 the rings of a full SM are 192 KiB in 4 stages; at 8
// query rows a warp (times of short bursts) 8 / 12 / 16 warps took 119 / 98.7 / 100 us for 64 sequences of up to 8192 tokens
// (8 kv heads of 128), 16.9 / 16.2 / 17.2 for 32 of up to 4096 (2 kv heads). The 16 rows of two
// column tiles need more than the 168 registers of 12 warps.
template <int NT>
struct Shape {
  static constexpr int kWarps = NT == 1 ? 12 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kRows = 8 * NT;
};

// The 8 x 8 matrix of 16-bit elements held two a lane (row lane / 4), transposed.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Rows of one virtual sequence's tile in q and out, and what they see.
struct Tile {
  int b, h, r0;           // sequence, kv head, first (token, head) pair of the tile
  int qo_len, kv_len, pages;
  int64_t row0;           // row of the sequence's first new token
};

// [0, total) in n contiguous parts, the first total % n of them one longer.
struct Split {
  int q, r;
  __device__ __forceinline__ Split(int total, int n) : q(total / n), r(total % n) {}
  __device__ __forceinline__ int begin(int c) const { return q * c + min(c, r); }
  __device__ __forceinline__ int part_of(int u) const {
    const int cut = r * (q + 1);
    return u < cut ? u / (q + 1) : r + (u - cut) / q;
  }
};

// The sequence that holds flat page x.
__device__ __forceinline__ int seq_of(const int32_t* indptr, int batch, int x) {
  int lo = 1, hi = batch;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (indptr[mid] > x) hi = mid; else lo = mid + 1;
  }
  return lo - 1;
}

// New rows of sequence b (0 where the plan does not fit the row tensors).
__device__ __forceinline__ int new_rows(const TcParams& p, int b, int64_t* row0) {
  if (p.qo_indptr == nullptr) {
    *row0 = b;
    return 1;
  }
  const int q0 = p.qo_indptr[b];
  const int len = p.qo_indptr[b + 1] - q0;
  *row0 = p.q_row_start != nullptr ? p.q_row_start[b] : q0;
  if (len <= 0) return 0;
  if (len > p.max_qo_len || *row0 < 0 || *row0 + len > p.num_rows) {
    report(p.status, NSLG_DEV_BAD_PLAN);
    return 0;
  }
  return len;
}

__device__ __forceinline__ void tma_load_2d(void* dst, const void* tmap, uint64_t* bar, int c0,
                                            int c1, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(smem_u32(dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "l"(policy)
      : "memory");
}

// Joined pieces of one row: sums relative to the running maximum m of their references.
struct Sum {
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  // the first min(N, count) of N pieces (x = m, l; a = four values); the others are repeats
  template <int N>
  __device__ __forceinline__ void add(const float2 (&x)[N], const float4 (&a)[N], int count) {
    float mn = m;
#pragma unroll
    for (int i = 0; i < N; ++i) mn = fmaxf(mn, x[i].x);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float old = fast_exp2(m - base);       // 0 for m = -inf: nothing has been added yet
    m = mn;
    l *= old;
    acc.x *= old;
    acc.y *= old;
    acc.z *= old;
    acc.w *= old;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i < count) {
        const float w = fast_exp2(x[i].x - base);
        l = fmaf(w, x[i].y, l);
        acc.x = fmaf(w, a[i].x, acc.x);
        acc.y = fmaf(w, a[i].y, acc.y);
        acc.z = fmaf(w, a[i].z, acc.z);
        acc.w = fmaf(w, a[i].w, acc.w);
      }
    }
  }
};

// Where the rows of a virtual sequence's tile go: new row (r0 + r) / group of its sequence,
// query head head0 + (r0 + r) % group.
struct Group {
  int b, head0, r0, len, part;
  int64_t row0;
};

// A virtual sequence that spans CTAs cf .. cf + cnt - 1 (vid -1: none).
struct Join {
  int vid, cf, cnt;
  Group to;
};

// Sequences without pages: their rows are zeros. CTA c takes sequences c, c + grid, ...
template <typename T, int kThreads>
__device__ void zero_empty(const TcParams& p, const int32_t* indptr) {
  const int words = p.hq * p.d / 8;
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (indptr[b] != indptr[b + 1]) continue;
    int64_t row0;
    const int len = new_rows(p, b, &row0);
    for (int i = 0; i < len; ++i) {
      uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (row0 + i) * p.out_stride);
      for (int e = threadIdx.x; e < words; e += kThreads) o[e] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

// Byte offset of 16-byte chunk c of token t inside a block's tile: the block is rows of 128
// bytes (two tokens a row at head_dim 64), TMA's 128-byte swizzle.
template <int D>
__device__ __forceinline__ uint32_t tile_offset(int t, int c) {
  if (D == 128) return t * 128 + ((c ^ (t & 7)) << 4);
  const int row = t >> 1, cc = (t & 1) * 4 + c;
  return row * 128 + ((cc ^ (row & 7)) << 4);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Shape<NT>::kThreads, 1)
    kv8_attn_tc_kernel(const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const TcParams p) {
  constexpr int kWarps = Shape<NT>::kWarps, kThreads = Shape<NT>::kThreads;
  constexpr int KS = D / 16;             // 16-dim chunks: k steps of K.q, row tiles of V^T.p^T
  constexpr int kBlock = kPS * D;        // bytes of one K (or V) block
  constexpr int kSlot = 2 * kBlock;
  constexpr int kBoxRows = kBlock / 128;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_vid[2 * kWarps];      // virtual sequence of each warp's head / tail piece
  __shared__ int s_piece[2 * kWarps];    // pieces in unit order: offset in floats from `smem`
  __shared__ int s_group[2 * kWarps + 1];
  __shared__ Group s_info[2 * kWarps];
  __shared__ Join s_join[2];
  __shared__ int s_ngroups, s_last[2];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stages = p.stages;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  constexpr int kPR = D + 8;             // row stride of a piece: its stores hit every bank
  const int piece_floats = (p.rows * (kPR + 2) + 3) & ~3;
  uint8_t* ring = smem + static_cast<size_t>(warp) * stages * kSlot;
  float* heads = reinterpret_cast<float*>(smem + static_cast<size_t>(kWarps) * stages * kSlot);
  uint64_t* bars = reinterpret_cast<uint64_t*>(
      heads + static_cast<size_t>(kWarps) * piece_floats);
  uint64_t* full = bars + warp * stages;

  if (lane < stages) mbar_init(&full[lane], 1);
  fence_barrier_init();
  if (threadIdx.x < 2 * kWarps) s_vid[threadIdx.x] = -1;
  // the kernel before may have written anything this one reads, the page list too
  pdl_wait();
  pdl_trigger();

  const int32_t* indptr = p.kv_indptr;
  const int32_t* lpl = p.kv_lpl;
  if (p.smem_csr) {
    int32_t* s_ip = reinterpret_cast<int32_t*>(bars + kWarps * stages);
    int32_t* s_lpl = s_ip + p.batch + 1;
    for (int i = threadIdx.x; i <= p.batch; i += kThreads) s_ip[i] = p.kv_indptr[i];
    for (int i = threadIdx.x; i < p.batch; i += kThreads) s_lpl[i] = p.kv_lpl[i];
    indptr = s_ip;
    lpl = s_lpl;
  }
  __syncthreads();

  const int hm = p.hkv * p.tiles;        // virtual sequences per sequence
  // units are numbered from the list's first entry on, which may be one of a longer list
  const int64_t from = static_cast<int64_t>(indptr[0]) * hm, to = static_cast<int64_t>(indptr[p.batch]) * hm;
  const bool fits = from >= 0 && to >= from && to < (int64_t{1} << 31) - kWarps;
  const int ufirst = fits ? static_cast<int>(from) : 0;
  const int total = fits ? static_cast<int>(to - from) : 0;
  const int n = min((total + kWarps - 1) / kWarps, p.grid);
  const int c = blockIdx.x;
  if (c >= n) {
    if (!fits && threadIdx.x == 0) report(p.status, NSLG_DEV_BAD_PLAN);
    zero_empty<T, kThreads>(p, indptr);
    return;
  }
  const Split ctas(total, n);
  const int u0 = ufirst + ctas.begin(c), u1 = ufirst + ctas.begin(c + 1);
  const Split parts(u1 - u0, kWarps);
  const int ua = u0 + parts.begin(warp), ub = u0 + parts.begin(warp + 1);
  const int units = ub - ua;

  // ---- metadata of 32 units at a time, one per lane
  struct Meta {
    int blk, vid, j;       // block (page * kv heads + head; -1: a bad page), sequence, page of it
    float sk, sv;          // scale_k and scale_v as loaded; then what weigh() makes of them
    float iv;
  };
  auto locate = [&](int u, int& vid, int& first) {   // unit u: its sequence and page list entry
    const int b = seq_of(indptr, p.batch, u / hm);
    first = indptr[b];
    const int np = indptr[b + 1] - first;
    const int loc = u - first * hm;
    const int vs = loc / np;
    vid = b * hm + vs;
    return loc - vs * np;
  };
  auto look_up = [&](int i, Meta& m) {
    m.blk = -1;
    m.vid = -1;
    m.j = 0;
    if (i < units) {
      int first;
      m.j = locate(ua + i, m.vid, first);
      const int page = p.kv_indices[first + m.j];
      if (page < 0 || page >= p.num_pages)
        report(p.status, NSLG_DEV_BAD_PAGE);
      else
        m.blk = page * p.hkv + m.vid % hm / p.tiles;
    }
  };
  auto load_scales = [&](Meta& m) {
    m.sk = m.blk >= 0 ? p.scale_k[m.blk] : 0.f;
    m.sv = m.blk >= 0 ? p.scale_v[m.blk] : 0.f;
  };
  // sv becomes E = log2 scale_v, NaN where V is zeros or not finite, and iv 2^-E; sk becomes NaN
  // where scale_v is (the NaN rides on the scores). Once for 32 units, when they are begun.
  auto weigh = [&](Meta& m) {
    const bool plain = has_exponent(m.sv);
    if (m.sv != m.sv) m.sk = m.sv;
    m.sv = plain ? __log2f(m.sv) : NAN;   // any value near the logarithm will do: iv is its inverse
    m.iv = fast_exp2(-m.sv);
  };
  const uint64_t policy = p.tiles > 1 ? l2_policy_evict_last() : l2_policy_evict_first();
  auto issue = [&](const Meta& m, int i) {   // by the lane that holds unit i
    const int s = i % stages;
    const int row = m.blk * kBoxRows;   // a bad page: a box before the first row, which reads as zeros
    mbar_arrive_expect_tx(&full[s], kSlot);
    tma_load_2d(ring + s * kSlot, &tmap_k, &full[s], 0, row, policy);
    tma_load_2d(ring + s * kSlot + kBlock, &tmap_v, &full[s], 0, row, policy);
  };

  Meta cur, nxt;
  look_up(lane, nxt);
  load_scales(nxt);   // before the bulk loads, which would queue in front of them
  if (lane < stages && lane < units) issue(nxt, lane);
  zero_empty<T, kThreads>(p, indptr);

  const int g = lane >> 2, tq = lane & 3;
  const int mi = lane >> 3, lr = lane & 7;
  // ldmatrix row addresses: K matrices (tokens 0-7 | 8-15) x (chunk, chunk + 1)
  const int ltok = (mi & 1) * 8 + lr, lch = mi >> 1;

  uint32_t qb[NT][KS][2];                // q^T fragments: row g of column tile nt
  float o[NT][KS][4];                    // rows 2tq, 2tq + 1 (c 0/1), dims 2g (0, 1), 2g + 1 (2, 3)
  float m[NT][2], nb[NT][2], l[NT][2], f[NT][2];   // of rows 2tq, 2tq + 1
  int pos[NT][2];                        // last position they see
  int low = 0;                           // ... the least of all the tile's rows
  float ev = 0.f;                        // E of the last page that had one
  bool seen = false;                     // ... whether there was one
  int vid = -1;
  Tile t{};
  bool ok = true;

  auto begin = [&](int v) {
    vid = v;
    t.b = v / hm;
    const int vs = v % hm;
    t.h = vs / p.tiles;
    t.r0 = vs % p.tiles * Shape<NT>::kRows;
    t.qo_len = new_rows(p, t.b, &t.row0);
    t.pages = indptr[t.b + 1] - indptr[t.b];
    int last = lpl[t.b];
    if (last < 1 || last > kPS) {
      report(p.status, NSLG_DEV_BAD_PLAN);
      last = kPS;
    }
    t.kv_len = (t.pages - 1) * kPS + last;
    low = 0x7fffffff;
    ev = 0.f;
    seen = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int pair = t.r0 + nt * 8 + g;
      const int tok = pair / p.group;
      const bool live = nt * 8 + g < p.rows && tok < t.qo_len;
      const T* src = static_cast<const T*>(p.q) + (t.row0 + tok) * p.q_stride +
                     static_cast<int64_t>(t.h * p.group + pair % p.group) * D + 4 * tq;
      uint2 raw[KS];
#pragma unroll
      for (int k = 0; k < KS; ++k)
        raw[k] = live ? *reinterpret_cast<const uint2*>(src + 16 * k) : make_uint2(0u, 0u);
      // a row of no sequence sees everything: it is never written, and no page is an edge for it
      const int lim = !live ? 0x7fffffff : p.causal ? t.kv_len - t.qo_len + tok : t.kv_len - 1;
      float sc = p.scale_log2;
      if constexpr (Mma16<T>::kFormat == 1) {      // bf16 -> f16 by a power of two
        uint32_t top = 0u;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          top = max(max(top, (raw[k].x & 0x7FFFu)), (raw[k].x >> 16) & 0x7FFFu);
          top = max(max(top, (raw[k].y & 0x7FFFu)), (raw[k].y >> 16) & 0x7FFFu);
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // magnitude in [2^(e - 127), 2^(e - 126)): times 2^(141 - e) is in [2^14, 2^15)
        const int e = static_cast<int>(top >> 7);
        float up = 1.f;
        if (e > 14 && e < 255) {       // smaller rows, zeros, infinities and NaN: as they are
          up = __uint_as_float(static_cast<uint32_t>(268 - e) << 23);
          sc *= 1.f / up;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          qb[nt][k][0] = pack_f16x2(__uint_as_float(raw[k].x << 16) * up,
                                    __uint_as_float(raw[k].x & 0xFFFF0000u) * up);
          qb[nt][k][1] = pack_f16x2(__uint_as_float(raw[k].y << 16) * up,
                                    __uint_as_float(raw[k].y & 0xFFFF0000u) * up);
        }
      } else {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          qb[nt][k][0] = raw[k].x;
          qb[nt][k][1] = raw[k].y;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {    // row r's values are in the lanes 4r .. 4r + 3
        f[nt][e] = __shfl_sync(0xffffffffu, sc, (2 * tq + e) * 4);
        pos[nt][e] = __shfl_sync(0xffffffffu, lim, (2 * tq + e) * 4);
        m[nt][e] = -INFINITY;
        nb[nt][e] = l[nt][e] = 0.f;
      }
      low = min(low, __reduce_min_sync(0xffffffffu, lim));
#pragma unroll
      for (int k = 0; k < KS; ++k) o[nt][k][0] = o[nt][k][1] = o[nt][k][2] = o[nt][k][3] = 0.f;
    }
  };

  auto segment = [&](int v, int& beg, int& end) {   // units of virtual sequence v
    const int b = v / hm;
    const int first = indptr[b], np = indptr[b + 1] - first;
    beg = first * hm + (v - b * hm) * np;
    end = beg + np;
  };
  auto group_of = [&](int v) {           // where the rows of virtual sequence v go
    Group gi;
    gi.b = v / hm;
    const int vs = v - gi.b * hm, h = vs / p.tiles;
    gi.head0 = h * p.group;
    gi.r0 = (vs - h * p.tiles) * Shape<NT>::kRows;
    gi.len = new_rows(p, gi.b, &gi.row0);
    return gi;
  };
  auto out_row = [&](const Group& gi, int r) -> T* {   // row r of the tile, null: none
    const int pair = gi.r0 + r, tok = pair / p.group;
    if (tok >= gi.len) return nullptr;
    return static_cast<T*>(p.out) + (gi.row0 + tok) * p.out_stride +
           static_cast<int64_t>(gi.head0 + pair - tok * p.group) * D;
  };

  // The virtual sequences this CTA shares with others, worked out while the first loads are
  // under way: [0] one that began in an earlier CTA, [1] one that begins here and goes on.
  if (warp < 2 && lane == 0) {
    Join jn;
    int first;
    locate(warp == 0 ? u0 : u1 - 1, jn.vid, first);
    int beg, end;
    segment(jn.vid, beg, end);
    if (warp == 0 ? beg < u0 : (beg >= u0 && end > u1)) {
      jn.cf = ctas.part_of(beg - ufirst);
      jn.cnt = ctas.part_of(end - 1 - ufirst) - jn.cf + 1;
      jn.to = group_of(jn.vid);
    } else {
      jn.vid = -1;
    }
    s_join[warp] = jn;
  }

  // The warp's state of virtual sequence `vid`, finished: to out, or as a piece.
  auto finish = [&]() {
    int beg, end;
    segment(vid, beg, end);
    const bool whole = beg >= ua && end <= ub;
    const bool tail = end > ub;
    float* piece = tail ? reinterpret_cast<float*>(ring) : heads + warp * piece_floats;
    if (!whole && lane == 0) s_vid[2 * warp + (tail ? 1 : 0)] = vid;
    Group to{};
    if (whole) to = group_of(vid);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float ls = l[nt][e];
        ls += __shfl_xor_sync(0xffffffffu, ls, 4);
        ls += __shfl_xor_sync(0xffffffffu, ls, 8);
        ls += __shfl_xor_sync(0xffffffffu, ls, 16);
        const int row = nt * 8 + 2 * tq + e;
        if (row >= p.rows) continue;
        if (whole) {
          T* dst = out_row(to, row);
          if (dst == nullptr) continue;
          const float inv = ls == 0.f ? 0.f : 1.f / ls;
#pragma unroll
          for (int k = 0; k < KS; ++k)
            *reinterpret_cast<uint32_t*>(dst + 16 * k + 2 * g) =
                Mma16<T>::pack(o[nt][k][e] * inv, o[nt][k][2 + e] * inv);
        } else {
#pragma unroll
          for (int k = 0; k < KS; ++k)
            *reinterpret_cast<float2*>(piece + row * kPR + 16 * k + 2 * g) =
                make_float2(o[nt][k][e], o[nt][k][2 + e]);
          if (g == 0) {
            piece[p.rows * kPR + 2 * row] = m[nt][e];
            piece[p.rows * kPR + 2 * row + 1] = ls;
          }
        }
      }
  };

  int left = 0, tok0 = 0;                // units of `vid` to come, the first token of this one
  int slot = 0;
  uint32_t phase = 0;
  for (int base = 0; base < units && ok; base += 32) {
    cur = nxt;
    weigh(cur);
    look_up(base + 32 + lane, nxt);
    load_scales(nxt);
    const int stop = min(32, units - base);
    for (int i = 0; i < stop; ++i) {
      if (left == 0) {             // the next virtual sequence
        if (vid >= 0) finish();
        begin(__shfl_sync(0xffffffffu, cur.vid, i));
        const int j = __shfl_sync(0xffffffffu, cur.j, i);
        tok0 = j * kPS;
        left = t.pages - j;
      }
      const float sk = __shfl_sync(0xffffffffu, cur.sk, i);
      float eu = __shfl_sync(0xffffffffu, cur.sv, i), iu = __shfl_sync(0xffffffffu, cur.iv, i);
      const bool plain = eu == eu;
      const bool anew = plain && !seen;
      if (plain) {
        ev = eu;
        seen = true;
      } else {
        eu = seen ? fmaxf(ev - kZeroE, kLeastE) : 0.f;
        iu = fast_exp2(-eu);
      }
      ok = __all_sync(0xffffffffu, mbar_wait(&full[slot], phase));
      if (!ok) {
        if (lane == 0) report(p.status, NSLG_DEV_WAIT_TIMEOUT);
        // issue nothing more; wait (bounded) for the loads in flight before leaving
        for (int k = 1; k < stages; ++k) {
          const int s = (slot + k) % stages;
          if (base + i + k < units) (void)mbar_wait(&full[s], s > slot ? phase : phase ^ 1);
        }
        break;
      }
      const uint32_t kb = smem_u32(ring + slot * kSlot), vb = kb + kBlock;
      // ---- scores of the page's 16 tokens
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; k += 2) {
        uint32_t w[4];
        ldmatrix_x4(kb + tile_offset<D>(ltok, k + lch), w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t a[4] = {f16x2_from_e4m3x2(static_cast<uint16_t>(w[2 * e])),
                                 f16x2_from_e4m3x2(static_cast<uint16_t>(w[2 * e + 1])),
                                 f16x2_from_e4m3x2(static_cast<uint16_t>(w[2 * e] >> 16)),
                                 f16x2_from_e4m3x2(static_cast<uint16_t>(w[2 * e + 1] >> 16))};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_f16_16816(s[nt], a, qb[nt][k + e][0], qb[nt][k + e][1]);
        }
      }
      // a page some row does not see whole, or that ends the sequence
      const int held = t.kv_len - tok0;
      const bool edge = low < tok0 + kPS - 1 || held < kPS;
      bool raise = anew;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][e] = fmaf(s[nt][e], f[nt][e & 1] * sk, eu);
          if (edge && tok0 + (e >> 1) * 8 + g > pos[nt][e & 1]) s[nt][e] = -INFINITY;
          raise |= s[nt][e] > m[nt][e & 1] + kHeadroom;
        }
      }
      // ---- the running reference, raised when a score passes it by kHeadroom
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(s[nt][e], s[nt][2 + e]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            // anew: o is all zeros, M may go down (where the row sees the page)
            const float mn = anew && x > -INFINITY ? fmaxf(x, m[nt][e] - kMostDown) : fmaxf(m[nt][e], x);
            const float cf = mn == -INFINITY || m[nt][e] == -INFINITY ? 1.f : fast_exp2(m[nt][e] - mn);
            m[nt][e] = mn;
            nb[nt][e] = mn == -INFINITY ? 0.f : -mn;
            l[nt][e] *= cf;
            if (!anew)
#pragma unroll
              for (int k = 0; k < KS; ++k) {
                o[nt][k][e] *= cf;
                o[nt][k][2 + e] *= cf;
              }
          }
      }
      uint32_t pb[NT][2];      // p^T: tokens 0-7, 8-15
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float pr[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[e] = fast_exp2(s[nt][e] + nb[nt][e & 1]);
        l[nt][0] = fmaf(pr[0] + pr[2], iu, l[nt][0]);
        l[nt][1] = fmaf(pr[1] + pr[3], iu, l[nt][1]);
        pb[nt][0] = movmatrix_trans(pack_f16x2(pr[0], pr[1]));
        pb[nt][1] = movmatrix_trans(pack_f16x2(pr[2], pr[3]));
      }
      // ---- o^T += V^T . p^T
      // selectors that pair the bytes of tokens 2tq and 2tq + 1 (+ 8 for the second); codes
      // behind the last token, and of a scale of 0 or NaN, count as 0 (byte 4)
      uint32_t sel[2] = {0x3120u, 0x3120u};
      if (held < kPS || !plain) {
        const int live = plain ? held : 0;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          sel[e] = (tq * 2 + 8 * e < live ? 0x0100u : 0x0404u) |
                   (tq * 2 + 8 * e + 1 < live ? 0x3020u : 0x4040u);
      }
#pragma unroll
      for (int k = 0; k < KS; k += 2) {
        uint32_t w[4];
        ldmatrix_x4_trans(vb + tile_offset<D>(ltok, k + lch), w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = __byte_perm(w[e], 0u, sel[e & 1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t a[4] = {f16x2_from_e4m3x2(static_cast<uint16_t>(w[2 * e])),
                                 f16x2_from_e4m3x2(static_cast<uint16_t>(w[2 * e] >> 16)),
                                 f16x2_from_e4m3x2(static_cast<uint16_t>(w[2 * e + 1])),
                                 f16x2_from_e4m3x2(static_cast<uint16_t>(w[2 * e + 1] >> 16))};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_f16_16816(o[nt][k + e], a, pb[nt][0], pb[nt][1]);
        }
      }
      __syncwarp();        // the slot has been read by every lane
      const int ahead = i + stages;
      if (base + ahead < units && lane == (ahead & 31)) issue(ahead < 32 ? cur : nxt, base + ahead);
      tok0 += kPS;
      --left;
      if (++slot == stages) {
        slot = 0;
        phase ^= 1;
      }
    }
  }
  // after a wait that gave up: the pieces are garbage (the status says so), but the joining
  // below keeps its control flow, so the counts return to zero
  if (vid >= 0) finish();
  __syncthreads();

  // ---- the pieces of this CTA, in unit order, grouped by virtual sequence
  if (warp == 0) {
    const int v = lane < 2 * kWarps ? s_vid[lane] : -1;
    const uint32_t have = __ballot_sync(0xffffffffu, v >= 0);
    const uint32_t before = have & ((1u << lane) - 1u);
    // the piece before this one, if it is of the same sequence, is not a start
    const int prev = __shfl_sync(0xffffffffu, v, before != 0u ? 31 - __clz(before) : 0);
    const bool starts = v >= 0 && (before == 0u || prev != v);
    const uint32_t st = __ballot_sync(0xffffffffu, starts);
    if (v >= 0) {
      const int w = lane >> 1;
      s_piece[__popc(before)] =
          (lane & 1) ? w * stages * (kSlot / 4) : kWarps * stages * (kSlot / 4) + w * piece_floats;
    }
    if (starts) {
      const int gr = __popc(st & ((1u << lane) - 1u));
      s_group[gr] = __popc(before);
      Group gi = group_of(v);
      int beg, end;
      segment(v, beg, end);
      // whole in this CTA: to out; else to the partial of the one that began before (2c) or
      // begins here (2c + 1)
      gi.part = beg >= u0 && end <= u1 ? -1 : 2 * c + (beg >= u0 ? 1 : 0);
      s_info[gr] = gi;
    }
    if (lane == 0) {
      s_ngroups = __popc(st);
      s_group[__popc(st)] = __popc(have);
      s_last[0] = s_last[1] = 0;
    }
  }
  __syncthreads();
  const int ngroups = s_ngroups;
  // a CTA that others wait to count arrives even where its warps gave up before they had a piece
  if (ngroups == 0 && s_join[0].vid < 0 && s_join[1].vid < 0) return;
  constexpr int DQ = D / 4;
  const float* pieces = reinterpret_cast<const float*>(smem);
  const int ml = p.rows * kPR;           // (m, l) of a piece's rows lie behind its values
  auto store_out = [&](T* dst, const float4& a, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(Mma16<T>::pack(a.x * inv, a.y * inv), Mma16<T>::pack(a.z * inv, a.w * inv));
  };
  const int per_group = p.rows * DQ;
  for (int e = threadIdx.x; e < ngroups * per_group; e += kThreads) {
    const int gr = e / per_group, row = (e - gr * per_group) / DQ, dq = e % DQ;
    const int k0 = s_group[gr], k1 = s_group[gr + 1];
    Sum sum;
    for (int k = k0; k < k1; k += 4) {
      float2 x[4];
      float4 a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* pc = pieces + s_piece[min(k + i, k1 - 1)];
        x[i] = *reinterpret_cast<const float2*>(pc + ml + 2 * row);
        a[i] = *reinterpret_cast<const float4*>(pc + row * kPR + 4 * dq);
      }
      sum.add<4>(x, a, k1 - k);
    }
    const Group& gi = s_info[gr];
    if (gi.part < 0) {
      T* dst = out_row(gi, row);
      if (dst != nullptr) store_out(dst + 4 * dq, sum.acc, sum.l);
    } else {
      const int64_t r = static_cast<int64_t>(gi.part) * p.rows + row;
      *reinterpret_cast<float4*>(p.part_o + r * D + 4 * dq) = sum.acc;
      if (dq == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * r) = make_float2(sum.m, sum.l);
    }
  }
  __syncthreads();

  // ---- virtual sequences that span CTAs
  if (warp < 2 && lane == 0 && s_join[warp].vid >= 0) {
    uint32_t* count = &p.arrive[s_join[warp].cf];
    const uint32_t prev = atom_add_acq_rel_u32(count, 1u);
    if (prev + 1u == static_cast<uint32_t>(s_join[warp].cnt)) {
      atomicExch(count, 0u);
      s_last[warp] = 1;
    }
  }
  __syncthreads();
  for (int k = 0; k < 2; ++k) {
    if (!s_last[k]) continue;
    const Join& jn = s_join[k];
    const int cnt = jn.cnt;
    // kBatch partials at a time, every load of a batch in flight at once: 4 where that is all (a
    // batch of sequences; the loads that repeat the last one cost: 12 for all of them took 0.6 us
    // more on one of 513 tokens), 12 for a few that are spread over many CTAs (5 rows on
    // 4001 tokens 19.8 us with 8, 18.3 with 12). Partial i is CTA cf + i's: the one that begins
    // there for the first, the one that began before else.
    auto join = [&](auto batch) {
      constexpr int kBatch = decltype(batch)::value;
      for (int e = threadIdx.x; e < per_group; e += kThreads) {
        const int row = e / DQ, dq = e % DQ;
        Sum sum;
        for (int i0 = 0; i0 < cnt; i0 += kBatch) {
          float2 x[kBatch];
          float4 a[kBatch];
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int at = min(i0 + i, cnt - 1);
            const int64_t r = (2ll * (jn.cf + at) + (at == 0 ? 1 : 0)) * p.rows + row;
            x[i] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + 2 * r));
            a[i] = __ldcg(reinterpret_cast<const float4*>(p.part_o + r * D + 4 * dq));
          }
          sum.template add<kBatch>(x, a, cnt - i0);
        }
        T* dst = out_row(jn.to, row);
        if (dst != nullptr) store_out(dst + 4 * dq, sum.acc, sum.l);
      }
    };
    if (cnt <= 4)
      join(std::integral_constant<int, 4>{});
    else
      join(std::integral_constant<int, 12>{});
  }
}

int64_t arrive_bytes(int grid) { return (static_cast<int64_t>(grid) * 4 + 255) / 256 * 256; }

int tile_rows(int group, int max_qo_len) {
  const int64_t pairs = static_cast<int64_t>(group) * max_qo_len;
  return pairs < 16 ? static_cast<int>(pairs) : 16;
}

template <typename T, int D, int NT>
int launch_typed(TcParams p, cudaStream_t stream) {
  constexpr int kWarps = Shape<NT>::kWarps, kThreads = Shape<NT>::kThreads;
  CUtensorMap tk, tv;
  const uint64_t rows = static_cast<uint64_t>(p.num_pages) * p.hkv * kPS * D / 128;
  int rc = encode_tiled_2d_bytes(&tk, p.codes_k, 128, rows, kPS * D / 128);
  if (rc == NSLG_OK) rc = encode_tiled_2d_bytes(&tv, p.codes_v, 128, rows, kPS * D / 128);
  if (rc != NSLG_OK) return rc;
  constexpr size_t kSlot = 2 * kPS * D;
  p.smem_csr = p.batch <= kSmemBatch ? 1 : 0;
  const size_t piece = static_cast<size_t>((p.rows * (D + 10) + 3) & ~3) * 4;
  const size_t heads = kWarps * piece;
  const size_t csr = p.smem_csr ? static_cast<size_t>(2 * p.batch + 1) * 4 : 0;
  const size_t fixed = 1024 + heads + csr + kWarps * kMaxStages * 8 + kStaticSmem;
  int stages = static_cast<int>((kMaxSmem - fixed) / (kWarps * kSlot));
  if (stages > kMaxStages) stages = kMaxStages;
  if (static_cast<size_t>(stages) * kSlot < piece)
    // a warp's tail piece is put into its part of the ring
    return set_error(NSLG_ERR_UNSUPPORTED, "kv8 attention: no room for the pipeline");
  p.stages = stages;
  const size_t smem = 1024 + heads + csr + static_cast<size_t>(kWarps) * stages * (kSlot + 8);
  auto kern = kv8_attn_tc_kernel<T, D, NT>;
  const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem));
  if (err != cudaSuccess) return set_error(NSLG_ERR_CUDA, cudaGetErrorString(err));
  return launch_pdl("kv8_attn_tc", kern, dim3(p.grid), dim3(kThreads), smem, stream, tk, tv, p);
}

template <typename T>
int launch_dim(const TcParams& p, cudaStream_t stream) {
  if (p.rows <= 8)
    return p.d == 128 ? launch_typed<T, 128, 1>(p, stream) : launch_typed<T, 64, 1>(p, stream);
  return p.d == 128 ? launch_typed<T, 128, 2>(p, stream) : launch_typed<T, 64, 2>(p, stream);
}

}  // namespace

bool kv8_attn_tc_supported(int dtype, const Kv8AttnParams& p) {
  if (dtype != NSLG_DTYPE_BF16 && dtype != NSLG_DTYPE_F16) return false;
  if (p.page_size != kPS || (p.d != 64 && p.d != 128)) return false;
  const int64_t tiles = (static_cast<int64_t>(p.hq / p.hkv) * p.max_qo_len + 15) / 16;
  // TMA row coordinates and the virtual sequences' numbers are 32-bit
  return p.num_pages * p.hkv * kPS < (int64_t{1} << 31) &&
         static_cast<int64_t>(p.batch) * p.hkv * tiles < (int64_t{1} << 31);
}

int64_t kv8_attn_tc_workspace_bytes(int group, int max_qo_len, int d) {
  const int grid = sm_count();
  return arrive_bytes(grid) + 2ll * grid * tile_rows(group, max_qo_len) * (d + 2) * 4 + 256;
}

int launch_kv8_attention_tc(int dtype, const Kv8AttnParams& a, void* workspace,
                            int64_t workspace_bytes, cudaStream_t stream) {
  TcParams p{};
  static_cast<Kv8AttnParams&>(p) = a;
  p.group = a.hq / a.hkv;
  const int64_t need = kv8_attn_tc_workspace_bytes(p.group, a.max_qo_len, a.d);
  if (workspace == nullptr || workspace_bytes < need)
    return set_error(NSLG_ERR_WORKSPACE, "kv8 attention: the workspace needs " + std::to_string(need) + " bytes");
  p.grid = sm_count();
  p.rows = tile_rows(p.group, a.max_qo_len);
  p.tiles = static_cast<int>((static_cast<int64_t>(p.group) * a.max_qo_len + 15) / 16);
  p.scale_log2 = a.sm_scale * 1.4426950408889634f;
  const uintptr_t ws = (reinterpret_cast<uintptr_t>(workspace) + 255) & ~static_cast<uintptr_t>(255);
  p.arrive = reinterpret_cast<uint32_t*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + arrive_bytes(p.grid));
  p.part_ml = p.part_o + 2ll * p.grid * p.rows * a.d;
  if (dtype == NSLG_DTYPE_F16) return launch_dim<__half>(p, stream);
  return launch_dim<__nv_bfloat16>(p, stream);
}

}  // namespace nslg
