// Causal prefill / extend attention over the 8-bit paged cache on the 5th-generation tensor
// cores (tcgen05.mma, accumulators in TMEM): page_size 16, head_dim 128, bf16 or fp16 q.
//
// What bounds it: 4 * 128 flop and one exponential per (query row, head, position). At 16
// exponentials a clock and SM they take as long as the products at full rate, so everything
// else has to stay off the softmax warps. The codes are therefore not dequantised: they are
// only widened to f16, which is exact and one instruction per two, and the blocks' scales
// join the exponent, where they cost nothing per element:
//   t_j = s_j F_g + E_g      s = q . code_k, F = scale_k sm_scale log2(e) / (row's q factor),
//                            E = log2(scale_v), g = j's page (16 positions share F and E)
//   p_j = 2^(t_j - M)        M: running maximum of t, raised when passed by 8
//   o   = sum_j p_j code_v[j];  l = sum_g 2^-E_g sum_{j in g} p_j;  out = o / l
// so p is what multiplies the code in the f16 product, M follows the largest of these
// weights, and no ratio of scales between pages can underflow what matters (a block of zeros
// in V has no E, only a part in l: it takes one kZeroE below the tile's least, so that it
// raises M only where it outweighs the row's other pages by 2^60; the first tile with an E of
// its own sets M anew). F >= 0 makes the
// maximum of t over a page a function of the maximum of s. bf16 q becomes f16 exactly after
// each row is multiplied by the power of two that brings its largest magnitude to [2^14, 2^15).
//
// Work item: two query tiles of 128 rows ("halves" A and B) of one sequence and kv head, each
// 128 / G new tokens times the G query heads that share the kv head; both read the same K and
// V tiles of 128 positions (N = 128: at N = 64 an m128 product reads its operands from shared
// memory for longer than it computes). A persistent grid, one CTA an SM, takes the items,
// longest causal spans first.
//
// Roles (16 warps; registers moved to the softmax warps by setmaxnreg):
//   producer warp   bulk copies of the tile's page blocks (2 KiB each, contiguous) into raw
//                   buffers, TMA boxes of Q; the pages' F and E factors into a ring of 4.
//   converters (4)  raw codes -> f16 tiles in the 128-byte swizzled layout (rings of 2 for K
//                   and for V), zeros behind the sequence's end and for bad pages; bf16 Q ->
//                   f16 in place, with the rows' factors.
//   MMA warp        per tile: P_A.V, S_A(t+1), P_B.V, S_B(t+1): while the softmax of one half
//                   runs, the pipe does the other half's products. P is written over S
//                   (tcgen05.mma of one thread execute in the order of issue, so S(t+1) may
//                   follow P(t).V into the same columns).
//   softmax A, B    one thread a row: S from TMEM, p to TMEM as f16, o rescaled there when M is
//                   raised; at the end of an item o / l straight to `out`.
// TMEM per half: S (and P over it) 128 + O 128 columns; 512 in all.
//
// A block whose scale is NaN (K's or V's) gives NaN to the rows that see it: its F is NaN, and
// masked positions are left out by selection. Every mbarrier wait is bounded; on a timeout
// the kernel records NSLG_DEV_WAIT_TIMEOUT, waits (bounded) for what it issued, frees its
// TMEM and returns.
#include <cuda.h>

#include <string>

#include "kv8.cuh"
#include "launch.h"
#include "tcgen05.cuh"

namespace nslg {
namespace {

constexpr int kD = 128;
constexpr int kBM = 128;              // rows per half
constexpr int kBN = 128;              // positions per tile
constexpr int kPS = 16;
constexpr int kPages = kBN / kPS;
constexpr int kThreads = 512;         // warps 0-3 converters, 4 producer, 5 MMA, 8-11 / 12-15 softmax
constexpr int kTmemCols = 512;
constexpr int kHalfCols = 256;        // S / P at +0, O at +128
constexpr int kColO = 128;
constexpr int kDimHalf = 128 * 128;   // [128 rows][128 bytes]: 64 dims of a Q half or a K / V tile
constexpr int kTileBytes = 2 * kDimHalf;
constexpr int kRaw = kBN * kD;        // codes of a tile
constexpr int kBlockBytes = kPS * kD;
constexpr float kZeroE = 60.f;
constexpr int kFactors = 4;           // ring of the pages' factors
constexpr int kSmemBytes = 1024 + 2 * kTileBytes /* Q */ + 4 * kTileBytes /* K, V rings */ +
                           2 * kRaw + 1536;   // and the factors, barriers and row_up

struct PrefillParams : Kv8AttnParams {
  int group, tokens_per_tile, n_items;
  float scale_log2;
};

// The factors of a tile's pages.
struct Factors {
  float f[kPages];      // scale_k (NaN where the block of K or V is not finite)
  float e[kPages];      // log2 scale_v
  float inv[kPages];    // 2^-e
  uint32_t valid;       // pages with codes
  uint32_t plain;       // pages with an e of their own
};

struct Half {
  int i0;               // first new token
  int64_t row0;         // its row
  bool any;
};
struct Item {
  int b, h, qo_len, kv_beg, npages, kv_len, ntiles;
  Half x[2];
};

// Item (pair of query tiles counted from the end, sequence, kv head). False: nothing to
// compute; `rows` then says whether the item has rows, which see no position.
__device__ __forceinline__ bool load_item(const PrefillParams& p, int item, Item& it, bool& rows) {
  const int per = p.batch * p.hkv;
  const int back = item / per;
  const int rem = item - back * per;
  it.b = rem / p.hkv;
  it.h = rem - it.b * p.hkv;
  const int qo0 = p.qo_indptr[it.b], qo1 = p.qo_indptr[it.b + 1];
  const int ip0 = p.kv_indptr[it.b], ip1 = p.kv_indptr[it.b + 1], lpl = p.kv_lpl[it.b];
  const int64_t start = p.q_row_start != nullptr ? p.q_row_start[it.b] : qo0;
  rows = false;
  it.qo_len = qo1 - qo0;
  if (it.qo_len <= 0) return false;
  if (it.qo_len > p.max_qo_len || start < 0 || start + it.qo_len > p.num_rows) {
    report(p.status, NSLG_DEV_BAD_PLAN);
    return false;
  }
  const int tpt = p.tokens_per_tile;
  const int pairs = ((it.qo_len + tpt - 1) / tpt + 1) / 2;
  const int pk = pairs - 1 - back;
  if (pk < 0) return false;
  rows = true;
  it.kv_beg = ip0;
  it.npages = ip1 - ip0;
  it.kv_len = it.npages > 0 ? (it.npages - 1) * kPS + lpl : 0;
  int last = 0;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    Half& hx = it.x[x];
    hx.i0 = (2 * pk + x) * tpt;
    hx.row0 = start + hx.i0;
    hx.any = hx.i0 < it.qo_len;
    if (hx.any) last = min(hx.i0 + tpt, it.qo_len) - 1;
  }
  const int span = p.causal ? min(it.kv_len, it.kv_len - it.qo_len + last + 1) : it.kv_len;
  it.ntiles = (span + kBN - 1) / kBN;
  return it.ntiles > 0;
}

// The next item with work from `item` on.
__device__ __forceinline__ int find_item(const PrefillParams& p, int item, Item& it) {
  bool rows;
  while (item < p.n_items && !load_item(p, item, it, rows)) item += gridDim.x;
  return item;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

template <int kRegs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    kv8_prefill_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const PrefillParams p) {
  constexpr bool kWiden = Mma16<T>::kFormat == 1;     // q has to become f16
  const int G = p.group;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sq = smem;                                 // [half][64-dim half][128 rows][128 B]
  uint8_t* sk = sq + 2 * kTileBytes;                  // [2][64-dim half][128 positions][128 B]
  uint8_t* sv = sk + 2 * kTileBytes;
  uint8_t* raw = sv + 2 * kTileBytes;                 // [K, V][128 positions][128 codes]
  Factors* fac = reinterpret_cast<Factors*>(raw + 2 * kRaw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(fac) + 512);
  uint64_t* q_full = bars + 0;       // [half] Q arrived
  uint64_t* q_ready = bars + 2;      // [half] ... and is f16
  uint64_t* q_empty = bars + 4;      // [half] last S of the item done
  uint64_t* raw_full = bars + 6;     // [K, V]
  uint64_t* raw_empty = bars + 8;    // [K, V]
  uint64_t* k_full = bars + 10;      // [2]
  uint64_t* k_empty = bars + 12;
  uint64_t* v_full = bars + 14;
  uint64_t* v_empty = bars + 16;
  uint64_t* s_full = bars + 18;      // [half]
  uint64_t* p_full = bars + 20;      // [half]
  uint64_t* pv_done = bars + 22;     // [half]
  uint64_t* o_free = bars + 24;      // [half]
  uint64_t* f_full = bars + 26;      // [kFactors]
  uint64_t* drain = bars + 30;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 31);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 32);
  int8_t* row_up = reinterpret_cast<int8_t*>(bars + 33);   // [item parity][half][row]: q was times 2^row_up

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_ready[i], 4);
      mbar_init(&q_empty[i], 1);
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 4);
      mbar_init(&k_full[i], 4);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 4);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_free[i], 128);
    }
    for (int i = 0; i < kFactors; ++i) mbar_init(&f_full[i], 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto gone = [&]() { return *abort_flag != 0; };
  auto give_up = [&]() {
    report(p.status, NSLG_DEV_WAIT_TIMEOUT);
    *abort_flag = 1;
  };

  // 128 registers a thread at launch: 2 x 128 x 184 + 128 x 72 + 128 x 64 of them are given out
  if (warp < 4) {
    // -------------------------------------------------------------- converters
    regs_dec<72>();
    const int tid = threadIdx.x;
    const int c = tid & 7, t0 = tid >> 3;              // 16-code chunk, first position
    int nk = 0, nv = 0, n_it = 0;                      // K tiles, V tiles, items
    bool ok = true;
    auto all_wait = [&](uint64_t* bar, uint32_t par) {
      return static_cast<bool>(__all_sync(0xffffffffu, !gone() && mbar_wait(bar, par)));
    };
    // one tile of codes to f16: kv 0 K, 1 V; tile number n, positions `held` of it exist
    auto convert = [&](int kv, int n, int held) -> bool {
      uint64_t* full = kv ? v_full : k_full;
      uint64_t* empty = kv ? v_empty : k_empty;
      const int s = n & 1;
      if (!all_wait(&raw_full[kv], n & 1)) return false;
      if (!all_wait(&empty[s], ((n >> 1) & 1) ^ 1)) return false;
      // pages whose codes count (V: not those of a scale of 0 or NaN)
      const uint32_t valid = kv ? fac[n % kFactors].plain : fac[n % kFactors].valid;
      const uint8_t* src = raw + kv * kRaw + t0 * 128 + c * 16;
      uint8_t* dst = (kv ? sv : sk) + s * kTileBytes + (c >> 2) * kDimHalf;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = t0 + 16 * i;                     // page i of the tile
        uint4 w = *reinterpret_cast<const uint4*>(src + 16 * i * 128);
        if (t >= held || !((valid >> i) & 1u)) w = make_uint4(0u, 0u, 0u, 0u);
        const uint4 lo = make_uint4(f16x2_from_e4m3x2(static_cast<uint16_t>(w.x)),
                                    f16x2_from_e4m3x2(static_cast<uint16_t>(w.x >> 16)),
                                    f16x2_from_e4m3x2(static_cast<uint16_t>(w.y)),
                                    f16x2_from_e4m3x2(static_cast<uint16_t>(w.y >> 16)));
        const uint4 hi = make_uint4(f16x2_from_e4m3x2(static_cast<uint16_t>(w.z)),
                                    f16x2_from_e4m3x2(static_cast<uint16_t>(w.z >> 16)),
                                    f16x2_from_e4m3x2(static_cast<uint16_t>(w.w)),
                                    f16x2_from_e4m3x2(static_cast<uint16_t>(w.w >> 16)));
        // 16-byte chunks 2 (c & 3) and the next of the row's 128 bytes; the lanes of the upper
        // 64 dims write theirs in the other order, so that eight lanes meet eight banks
        const int c0 = 2 * (c & 3), odd = c >> 2;
        uint8_t* row = dst + t * 128;
        *reinterpret_cast<uint4*>(row + (((c0 + odd) ^ (t & 7)) << 4)) = odd ? hi : lo;
        *reinterpret_cast<uint4*>(row + (((c0 + 1 - odd) ^ (t & 7)) << 4)) = odd ? lo : hi;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&raw_empty[kv]);
        mbar_arrive(&full[s]);
      }
      return true;
    };
    auto widen_q = [&](int x) -> bool {                // thread tid: row tid of the half
      if (!all_wait(&q_full[x], n_it & 1)) return false;
      uint8_t* row = sq + x * kTileBytes + tid * 128;
      uint32_t top = 0u;
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(row + (i >> 3) * kDimHalf +
                                                        (((i & 7) ^ (tid & 7)) << 4));
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) top = max(max(top, v[k] & 0x7FFFu), (v[k] >> 16) & 0x7FFFu);
      }
      // magnitude in [2^(e - 127), 2^(e - 126)): times 2^(141 - e) is in [2^14, 2^15)
      const int e = static_cast<int>(top >> 7);
      // (smaller rows, zeros, infinities and NaN: as they are)
      const int by = e > 14 && e < 255 ? 141 - e : 0;
      const float up = __uint_as_float(static_cast<uint32_t>(by + 127) << 23);
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        uint4* at = reinterpret_cast<uint4*>(row + (i >> 3) * kDimHalf + (((i & 7) ^ (tid & 7)) << 4));
        const uint4 w = *at;
        auto two = [&](uint32_t v) {
          return pack_f16x2(__uint_as_float(v << 16) * up, __uint_as_float(v & 0xFFFF0000u) * up);
        };
        *at = make_uint4(two(w.x), two(w.y), two(w.z), two(w.w));
      }
      row_up[((n_it & 1) * 2 + x) * kBM + tid] = static_cast<int8_t>(by);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[x]);
      return true;
    };
    Item it;
    int item = find_item(p, blockIdx.x, it);
    while (ok && item < p.n_items) {
      ok = convert(0, nk++, it.kv_len);
      if constexpr (kWiden)
        for (int x = 0; ok && x < 2; ++x) ok = widen_q(x);
      for (int j = 0; ok && j < it.ntiles; ++j) {
        ok = convert(1, nv++, it.kv_len - j * kBN);
        if (ok && j + 1 < it.ntiles) ok = convert(0, nk++, it.kv_len - (j + 1) * kBN);
      }
      ++n_it;
      item = find_item(p, item + gridDim.x, it);
    }
    if (!ok && lane == 0) give_up();
  } else if (warp < 8) {
    regs_dec<64>();
    if (warp == 4) {
      // -------------------------------------------------------------- producer
      int nk = 0, nv = 0, n_it = 0, nq = 0;
      float carry = 0.f;                               // e of this item's last tile that had one
      bool ok = true;
      auto all_wait = [&](uint64_t* bar, uint32_t par) {
        return static_cast<bool>(__all_sync(0xffffffffu, !gone() && mbar_wait(bar, par)));
      };
      // lane i < kPages: page i of the tile
      auto page_of = [&](const Item& it, int j) {
        const int pi = j * kPages + lane;
        return lane < kPages && j < it.ntiles && pi < it.npages ? p.kv_indices[it.kv_beg + pi] : -2;
      };
      auto load = [&](int kv, int n, const Item& it, int page) -> bool {
        if (!all_wait(&raw_empty[kv], (n & 1) ^ 1)) return false;
        const bool has = page >= 0 && page < p.num_pages;
        if (page != -2 && !has) report(p.status, NSLG_DEV_BAD_PAGE);
        const uint32_t valid = __ballot_sync(0xffffffffu, has);
        const int64_t blk = static_cast<int64_t>(page) * p.hkv + it.h;
        if (has)
          bulk_load(raw + kv * kRaw + lane * kBlockBytes,
                    static_cast<const uint8_t*>(kv ? p.codes_v : p.codes_k) + blk * kBlockBytes,
                    kBlockBytes, &raw_full[kv]);
        if (kv == 0) {
          float f = has ? p.scale_k[blk] : 0.f;
          const float v = has ? p.scale_v[blk] : 0.f;
          if (v != v) f = v;                           // NaN rides on the scores
          float e = log2f(v);
          const bool plain = v > 0.f && v < INFINITY;
          float least = plain ? e : INFINITY;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
          if (least != INFINITY) carry = least;
          if (!plain) e = fmaxf(carry - kZeroE, -120.f);
          const uint32_t own = __ballot_sync(0xffffffffu, plain);
          if (lane < kPages) {
            Factors& fc = fac[n % kFactors];
            fc.f[lane] = f;
            fc.e[lane] = e;
            fc.inv[lane] = exp2f(-e);
            if (lane == 0) {
              fc.valid = valid;
              fc.plain = own;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&f_full[n % kFactors]);
        }
        if (lane == 0) mbar_arrive_expect_tx(&raw_full[kv], __popc(valid) * kBlockBytes);
        __syncwarp();
        return true;
      };
      Item it;
      int item = find_item(p, blockIdx.x, it);
      int page = item < p.n_items ? page_of(it, 0) : -2;
      const uint64_t keep = l2_policy_evict_last();
      while (ok && item < p.n_items) {
        carry = 0.f;
        if (!(ok = load(0, nk, it, page))) break;
        ++nk;
        for (int x = 0; ok && x < 2; ++x) {
          if (!(ok = all_wait(&q_empty[x], (n_it & 1) ^ 1))) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[x], kTileBytes);
            uint8_t* dst = sq + x * kTileBytes;
            const int row = static_cast<int>(it.x[x].row0);
            tma_load_3d(dst, &tmap_q, &q_full[x], 0, it.h * G, row, keep);
            tma_load_3d(dst + kDimHalf, &tmap_q, &q_full[x], 64, it.h * G, row, keep);
          }
          ++nq;
          __syncwarp();
        }
        for (int j = 0; ok && j < it.ntiles; ++j) {
          const int next = page_of(it, j + 1);
          if (!(ok = load(1, nv, it, page))) break;
          ++nv;
          page = next;
          if (j + 1 < it.ntiles) {
            if (!(ok = load(0, nk, it, page))) break;
            ++nk;
          }
        }
        if (!ok) break;
        ++n_it;
        item = find_item(p, item + gridDim.x, it);
        page = item < p.n_items ? page_of(it, 0) : -2;
      }
      if (!ok) {
        if (lane == 0) give_up();
        // no copy may still be writing shared memory when the CTA leaves (bounded waits)
        if (nk > 0) (void)mbar_wait(&raw_full[0], (nk - 1) & 1);
        if (nv > 0) (void)mbar_wait(&raw_full[1], (nv - 1) & 1);
        for (int x = 0; x < 2; ++x) {
          const int loads = (nq + 1 - x) / 2;
          if (loads > 0) (void)mbar_wait(&q_full[x], (loads - 1) & 1);
        }
      }
    } else if (warp == 5 && lane == 0) {
      // -------------------------------------------------------------- MMA issuer
      constexpr uint32_t kIdescS = idesc_f16(0, kBN, false);
      constexpr uint32_t kIdescO = idesc_f16(0, kD, true);
      constexpr uint32_t kDescHi = smem_desc_hi(1024);
      const uint32_t q_lo0 = smem_desc_lo(smem_u32(sq), 16);
      const uint32_t k_lo0 = smem_desc_lo(smem_u32(sk), 16);
      const uint32_t v_lo0 = smem_desc_lo(smem_u32(sv), kDimHalf);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t par) { return !gone() && mbar_wait(bar, par); };
      // S_x(u) = Q_x . K(u)^T; behind P_x(u - 1).V in the pipe, which reads the same columns
      auto issue_s = [&](int u, int x, bool last) -> bool {
        const int slot = u & 1;
        if (x == 0 && !wait(&k_full[slot], (u >> 1) & 1)) return false;
        tc_fence_after();
        const uint32_t q_lo = q_lo0 + x * (kTileBytes >> 4);
        const uint32_t k_lo = k_lo0 + slot * (kTileBytes >> 4);
        const uint32_t dcol = tmem + x * kHalfCols;
#pragma unroll
        for (int ks = 0; ks < kD / 16; ++ks) {
          const uint32_t off = ((ks >> 2) * kDimHalf + (ks & 3) * 32) >> 4;
          mma_ss_w(dcol, q_lo + off, k_lo + off, kDescHi, kIdescS, ks > 0 ? 1u : 0u);
        }
        mma_commit(&s_full[x]);
        if (x == 1) mma_commit(&k_empty[slot]);
        if (last) mma_commit(&q_empty[x]);
        return true;
      };
      int t = 0, n_it = 0;
      Item it;
      int item = find_item(p, blockIdx.x, it);
      while (ok && item < p.n_items) {
        const int nt = it.ntiles;
        for (int x = 0; ok && x < 2; ++x)
          ok = wait(kWiden ? &q_ready[x] : &q_full[x], n_it & 1) && issue_s(t, x, nt == 1);
        Item nx;                                       // found while the pipe works
        const int nitem = find_item(p, item + gridDim.x, nx);
        for (int j = 0; ok && j < nt; ++j, ++t) {
          const int slot = t & 1;
          if (!(ok = wait(&v_full[slot], (t >> 1) & 1))) break;
          const uint32_t v_lo = v_lo0 + slot * (kTileBytes >> 4);
          for (int x = 0; x < 2; ++x) {
            if (!(ok = wait(&p_full[x], t & 1))) break;
            if (j == 0 && n_it > 0 && !(ok = wait(&o_free[x], (n_it - 1) & 1))) break;
            tc_fence_after();
            const uint32_t hb = tmem + x * kHalfCols;
#pragma unroll
            for (int kt = 0; kt < kBN / 16; ++kt)
              mma_ts_w(hb + kColO, hb + kt * 8, v_lo + (kt * 2048 >> 4), kDescHi, kIdescO,
                       (j > 0 || kt > 0) ? 1u : 0u);
            mma_commit(&pv_done[x]);
            if (x == 1) mma_commit(&v_empty[slot]);
            if (j + 1 < nt && !(ok = issue_s(t + 1, x, j + 2 == nt))) break;
          }
          if (!ok) break;
        }
        ++n_it;
        it = nx;
        item = nitem;
      }
      if (!ok) give_up();
      mma_commit(drain);                               // everything issued has completed (bounded)
      (void)mbar_wait(drain, 0);
    }
  } else {
    // -------------------------------------------------------------- softmax warpgroups
    regs_inc<184>();
    const int x = (warp - 8) / 4;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;                 // row = TMEM lane
    const int tok = r / G, hd = r - tok * G;
    const uint32_t base = tmem + x * kHalfCols + (static_cast<uint32_t>(quarter * 32) << 16);
    int t = 0, n_it = 0;
    bool ok = true;
    auto all_wait = [&](uint64_t* bar, uint32_t par) {
      return static_cast<bool>(__all_sync(0xffffffffu, !gone() && mbar_wait(bar, par)));
    };
    for (int item = blockIdx.x; ok && item < p.n_items; item += gridDim.x) {
      Item it;
      bool rows;
      const bool work = load_item(p, item, it, rows);
      if (!rows) continue;
      const Half& hx = it.x[x];
      const bool live = hx.i0 + tok < it.qo_len;
      T* dst = static_cast<T*>(p.out) + (hx.row0 + tok) * p.out_stride +
               static_cast<int64_t>(it.h * G + hd) * kD;
      if (!work) {                                     // rows that see no position
        if (live)
#pragma unroll
          for (int i = 0; i < kD / 8; ++i) reinterpret_cast<uint4*>(dst)[i] = make_uint4(0u, 0u, 0u, 0u);
        continue;
      }
      // last position the row sees; a row of no sequence sees everything and is not written
      const int lim = !live ? 0x7fffffff
                      : p.causal ? min(it.kv_len - it.qo_len + hx.i0 + tok, it.kv_len - 1)
                                 : it.kv_len - 1;
      float rf = p.scale_log2;
      if constexpr (kWiden) {
        if (!(ok = all_wait(&q_ready[x], n_it & 1))) break;
        rf *= __uint_as_float(static_cast<uint32_t>(127 - row_up[((n_it & 1) * 2 + x) * kBM + r]) << 23);
      }
      float m = -INFINITY, l = 0.f;
      bool seen = false;                               // a tile with an E of its own
      for (int j = 0; j < it.ntiles; ++j, ++t) {
        if (!(ok = all_wait(&f_full[t % kFactors], (t / kFactors) & 1))) break;
        const Factors& fc = fac[t % kFactors];
        if (!(ok = all_wait(&s_full[x], t & 1))) break;
        tc_fence_after();
        float s[2][64];
        tmem_ld64(base, s[0]);
        tmem_ld64(base + 64, s[1]);
        tmem_wait_ld();
        const int kbase = j * kBN;
        const bool edge = !__all_sync(0xffffffffu, kbase + kBN - 1 <= lim);
        if (edge) {
#pragma unroll
          for (int c = 0; c < kBN; ++c)
            if (kbase + c > lim) s[c >> 6][c & 63] = -INFINITY;
        }
        float F[kPages], A[kPages];
        float mt = -INFINITY;
#pragma unroll
        for (int g = 0; g < kPages; ++g) {
          const float* sg = &s[g >> 2][(g & 3) * 16];
          float a = fmaxf(fmaxf(sg[0], sg[1]), fmaxf(sg[2], sg[3]));
          float b = fmaxf(fmaxf(sg[4], sg[5]), fmaxf(sg[6], sg[7]));
          float c = fmaxf(fmaxf(sg[8], sg[9]), fmaxf(sg[10], sg[11]));
          float d = fmaxf(fmaxf(sg[12], sg[13]), fmaxf(sg[14], sg[15]));
          F[g] = rf * fc.f[g];
          A[g] = fc.e[g];
          mt = fmaxf(mt, fmaf(fmaxf(fmaxf(a, b), fmaxf(c, d)), F[g], A[g]));   // NaN is ignored
        }
        const bool anew = !seen && fc.plain != 0u;     // O is all zeros so far: M may go down too
        seen = seen || fc.plain != 0u;
        const bool raise = (anew && mt > -INFINITY) || mt > m + 8.f;   // and on the first finite maximum
        const float alpha =
            raise && m != -INFINITY && mt != -INFINITY ? fast_exp2(m - mt) : 1.f;
        if (raise) m = mt;
        const float nb = m == -INFINITY ? 0.f : -m;
        float sum = 0.f;
        uint32_t pk[2][32];
#pragma unroll
        for (int g = 0; g < kPages; ++g) {
          const float* sg = &s[g >> 2][(g & 3) * 16];
          const float add = A[g] + nb;
          float gs0 = 0.f, gs1 = 0.f;
#pragma unroll
          for (int c = 0; c < 16; c += 2) {
            float p0 = fast_exp2(fmaf(sg[c], F[g], add));
            float p1 = fast_exp2(fmaf(sg[c + 1], F[g], add));
            if (edge) {                                // F = 0 or NaN times -inf is NaN
              if (kbase + g * 16 + c > lim) p0 = 0.f;
              if (kbase + g * 16 + c + 1 > lim) p1 = 0.f;
            }
            gs0 += p0;
            gs1 += p1;
            pk[g >> 2][(g & 3) * 8 + c / 2] = pack_f16x2(p0, p1);
          }
          sum = fmaf(gs0 + gs1, fc.inv[g], sum);
        }
        // O may only be rescaled once P(t-1).V(t-1) is done (tcgen05.ld / st are
        // warp-collective; rows with alpha == 1 multiply by 1)
        if (j > 0 && !anew && __any_sync(0xffffffffu, alpha != 1.f)) {
          if (!(ok = all_wait(&pv_done[x], (t - 1) & 1))) break;
          tc_fence_after();
#pragma unroll 1
          for (int cb = 0; cb < kD; cb += 32) {
            float o[32];
            tmem_ld32(base + kColO + cb, o);
            tmem_wait_ld();
            uint32_t w[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) w[c] = __float_as_uint(o[c] * alpha);
            tmem_st32(base + kColO + cb, w);
          }
        }
        l = fmaf(l, alpha, sum);
        tmem_st32(base, pk[0]);                        // P over S
        tmem_st32(base + 32, pk[1]);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[x]);
      }
      if (!ok) break;
      const int tl = t - 1;
      if (!(ok = all_wait(&pv_done[x], tl & 1))) break;
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int cb = 0; cb < kD; cb += 64) {
        float o[64];
        tmem_ld64(base + kColO + cb, o);
        tmem_wait_ld();
        if (cb + 64 == kD) {
          tc_fence_before();
          mbar_arrive(&o_free[x]);                     // O may be overwritten now
        }
        if (live) {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            reinterpret_cast<uint4*>(dst + cb)[c] =
                make_uint4(Mma16<T>::pack(o[8 * c] * inv, o[8 * c + 1] * inv),
                           Mma16<T>::pack(o[8 * c + 2] * inv, o[8 * c + 3] * inv),
                           Mma16<T>::pack(o[8 * c + 4] * inv, o[8 * c + 5] * inv),
                           Mma16<T>::pack(o[8 * c + 6] * inv, o[8 * c + 7] * inv));
        }
      }
      ++n_it;
    }
    if (!ok && lane == 0) give_up();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
  }
}

}  // namespace

bool kv8_prefill_tc_supported(int dtype, const Kv8AttnParams& p) {
  if ((dtype != NSLG_DTYPE_BF16 && dtype != NSLG_DTYPE_F16) || p.d != kD || p.page_size != kPS)
    return false;
  const int g = p.hq / p.hkv;
  if (g > 16 || kBM % g != 0 || p.num_rows >= (int64_t{1} << 31)) return false;
  const int64_t pairs = (static_cast<int64_t>(p.max_qo_len) * g + 2 * kBM - 1) / (2 * kBM) + 1;
  return pairs * p.batch * p.hkv < (int64_t{1} << 30);
}

int launch_kv8_prefill_tc(int dtype, const Kv8AttnParams& a, cudaStream_t stream) {
  PrefillParams p{};
  static_cast<Kv8AttnParams&>(p) = a;
  p.group = a.hq / a.hkv;
  p.tokens_per_tile = kBM / p.group;
  p.scale_log2 = a.sm_scale * 1.4426950408889634f;
  CUtensorMap tq;
  const int rc = encode_tiled_3d_bf16(&tq, a.q, kD, a.hq, a.num_rows, static_cast<uint64_t>(kD) * 2,
                                      static_cast<uint64_t>(a.q_stride) * 2, 64, p.group,
                                      p.tokens_per_tile);
  if (rc != NSLG_OK) return rc;
  const int64_t tiles = (static_cast<int64_t>(a.max_qo_len) + p.tokens_per_tile - 1) / p.tokens_per_tile;
  const int64_t items = (tiles + 1) / 2 * a.batch * a.hkv;
  p.n_items = static_cast<int>(items);
  const int sms = sm_count();
  const unsigned grid = static_cast<unsigned>(items < sms ? items : sms);
  auto kern = dtype == NSLG_DTYPE_F16 ? kv8_prefill_tc_kernel<__half> : kv8_prefill_tc_kernel<__nv_bfloat16>;
  const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (err != cudaSuccess) return set_error(NSLG_ERR_CUDA, cudaGetErrorString(err));
  kern<<<grid, kThreads, kSmemBytes, stream>>>(tq, p);
  return check_launch("kv8_prefill_tc");
}

}  // namespace nslg
