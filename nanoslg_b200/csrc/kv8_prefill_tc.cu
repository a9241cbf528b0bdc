// Causal prefill / extend attention over the 8-bit paged cache on the 5th-generation tensor
// cores (tcgen05.mma, accumulators in TMEM): page_size 16, head_dim 64 or 128, bf16 or fp16 q.
//
// What bounds it: 4 * head_dim flop and one exponential per (query row, head, position). At 16
// exponentials a clock and SM they take as long as the products at full rate (0.55 us for 256
// rows and 64 positions at head_dim 128), so everything else has to stay off the softmax
// warps. Measured (bf16, 32 / 8 heads of 128, graphs of 60 calls): prompts of 64 x 512 tokens
// 256 us (540 TFLOP/s; 182 us at head_dim 64), 16 suffixes of 128 behind 1024 57 us (640): 1.1 to
// 1.2 us for such a tile, the chain of one half's scores, maximum, exponentials and weights, and
// 2 us at an item's end. The steps quoted below were measured in bursts of a few calls, before
// the power limit lowers the clocks; there the prompts take 226 us.
//
// The codes are not dequantised: they are only widened, which is exact (K to q's type, V to
// f16), and the blocks' scales join the exponent, where they cost nothing per element:
//   t_j = s_j F_g + E_g      s = q . code_k, F = scale_k sm_scale log2(e), E = log2 scale_v,
//                            g = j's page (16 positions share F and E)
//   p_j = 2^(t_j - M)        M: running maximum of t, raised when passed by 8
//   o   = sum_j p_j code_v[j];  l = sum_g 2^-E_g sum_{j in g} p_j;  out = o / l
// so p is what multiplies the code in the f16 product, M follows the largest of these weights,
// and no ratio of scales between pages can underflow what matters (blocks of zeros in V, which
// have no E, stand at kZeroE). F > 0 makes the maximum of t over a page a function of the
// maximum of s. p is f16 (2^-11) for both activation types.
//
// Work item: two query tiles of 128 rows ("halves" A and B) of one sequence and kv head, each
// 128 / G new tokens times the G query heads that share the kv head; both read the same K and
// V tiles of 64 positions. A persistent grid, one CTA an SM, takes the items,
// longest causal spans first.
//
// Roles (16 warps; registers moved to the softmax warps by setmaxnreg):
//   producer warp   the items and, per tile, the pages' blocks and factors F and E into rings.
//   Q warp          TMA boxes of Q.
//   converters (4)  a thread fetches its 16-byte pieces of the raw codes two tiles ahead
//                   (cp.async into places of its own, so nothing but its own wait is needed),
//                   widens them into 16-bit tiles in the 128-byte swizzled layout (rings of 3
//                   for K and for V); zeros behind the sequence's end and for bad pages.
//   MMA A, B        one warp a half, per tile: P(t).V, S(t+2), across items. P is written
//                   over S (tcgen05.mma of one thread execute in the order of issue, so S(t+2)
//                   may follow P(t).V into the same columns), and each half has two such
//                   buffers, so its softmax goes from tile to tile without waiting for the pipe.
//                   With one buffer of 128 positions the scores of a half waited for its
//                   softmax and the other way round: 2.9 us per 128 positions.
//   softmax A, B    one thread a row: S from TMEM, p to TMEM as f16, o rescaled there when M is
//                   raised. o / l of an item is written behind the next item's first tile, when
//                   its last P.V is done (251 -> 234 us for 64 x 512). The warps of A and B that
//                   share a scheduler take turns at the exponentials, so that one's are under
//                   way while the other waits for its next scores (234 -> 228).
// TMEM per half: two S (and P over it) of 64 + O 128 columns; 512 in all.
//
// A block whose scale is NaN (K's or V's) gives NaN to the rows that see it: their scores of
// the page are set to NaN. Every mbarrier wait is bounded; on a timeout the kernel records
// NSLG_DEV_WAIT_TIMEOUT, waits (bounded) for what it issued, frees its TMEM and returns.
#include <cuda.h>

#include <string>
#include <type_traits>

#include "kv8.cuh"
#include "launch.h"
#include "tcgen05.cuh"

namespace nslg {
namespace {

constexpr int kBM = 128;              // rows per half
constexpr int kBN = 64;               // positions per tile
constexpr int kPS = 16;
constexpr int kPages = kBN / kPS;
constexpr int kThreads = 512;         // warps 0-3 converters, 4 producer, 5 / 6 MMA, 7 Q, 8-11 / 12-15 softmax
constexpr int kTmemCols = 512;
constexpr int kHalfCols = 256;        // S / P of even tiles at +0, of odd ones at +64, O at +128
constexpr int kColO = 128;
constexpr int kQDimHalf = kBM * 128;  // 16-bit tiles are [64 dims][rows][128 bytes]
constexpr int kDimHalf = kBN * 128;
constexpr int kRing = 3;              // K tiles, V tiles
constexpr int kRawRing = 2;
constexpr int kFactors = 8;           // ring of the pages' factors
constexpr int kItems = 4;             // ring of published items
template <int D>
struct Shape {
  static constexpr int kQBytes = kBM * D * 2;       // a Q half
  static constexpr int kTileBytes = kBN * D * 2;    // a K or V tile
  static constexpr int kRaw = kBN * D;              // codes of a tile
  static constexpr int kBlockBytes = kPS * D;
  static constexpr int kRows = 128 * 16 / D;        // positions the converters take at once
  static constexpr int kSmemBytes = 1024 + 2 * kQBytes + 2 * kRing * kTileBytes + 2 * kRawRing * kRaw +
                                    1536;   // and the factors, barriers and items
};

struct PrefillParams : Kv8AttnParams {
  int group, tokens_per_tile, n_items;
  float scale_log2;
};

// What a tile's pages are.
struct alignas(16) Factors {
  float f[kPages];      // scale_k sm_scale log2(e), above 0: a masked score, -inf, stays one
  float e[kPages];      // log2 scale_v
  float inv[kPages];    // 2^-e
  int blk[kPages];      // block (page * kv heads + head), -1: none
  uint32_t plain;       // pages with an e of their own
  uint32_t nan;         // pages whose block of K or V is not finite
  int held;             // positions that exist, maybe more than the tile's; -1: no more tiles
};

// A work item as the producer publishes it. ntiles -1: no more.
struct Item {
  int h, qo_len, kv_len, ntiles;
  int i0, row0;         // half A's first new token and its row; half B's: tokens_per_tile on
  int kv_beg, npages;
};

// The per-sequence values of an item, read one item ahead, so that their latency overlaps
// the item before.
struct ItemLoads {
  int b, h, back;
  int qo0, qo1, ip0, ip1, lpl, start;
};

__device__ __forceinline__ void issue_item(const PrefillParams& p, int item, ItemLoads& L) {
  if (item >= p.n_items) return;
  const int per = p.batch * p.hkv;
  L.back = item / per;                 // pair of query tiles, counted from the sequence's end
  const int rem = item - L.back * per;
  L.b = rem / p.hkv;
  L.h = rem - L.b * p.hkv;
  L.qo0 = p.qo_indptr[L.b];
  L.qo1 = p.qo_indptr[L.b + 1];
  L.ip0 = p.kv_indptr[L.b];
  L.ip1 = p.kv_indptr[L.b + 1];
  L.lpl = p.kv_lpl[L.b];
  L.start = p.q_row_start != nullptr ? p.q_row_start[L.b] : L.qo0;
}

// False: no rows.
__device__ __forceinline__ bool finish_item(const PrefillParams& p, const ItemLoads& L, Item& it) {
  it.h = L.h;
  it.qo_len = L.qo1 - L.qo0;
  if (it.qo_len <= 0) return false;
  if (it.qo_len > p.max_qo_len || L.start < 0 || (L.ip1 > L.ip0 && (L.lpl < 1 || L.lpl > kPS)) ||
      static_cast<int64_t>(L.start) + it.qo_len > p.num_rows) {
    report(p.status, NSLG_DEV_BAD_PLAN);
    return false;
  }
  const int tpt = p.tokens_per_tile;
  const int pairs = ((it.qo_len + tpt - 1) / tpt + 1) / 2;
  const int pk = pairs - 1 - L.back;
  if (pk < 0) return false;
  it.kv_beg = L.ip0;
  it.npages = L.ip1 - L.ip0;
  it.kv_len = it.npages > 0 ? (it.npages - 1) * kPS + L.lpl : 0;
  it.i0 = 2 * pk * tpt;
  it.row0 = L.start + it.i0;
  const int last = min(it.i0 + 2 * tpt, it.qo_len) - 1;
  const int span = p.causal ? min(it.kv_len, it.kv_len - it.qo_len + last + 1) : it.kv_len;
  it.ntiles = span > 0 ? (span + kBN - 1) / kBN : 0;
  return true;
}

// 16 bytes, or zeros.
__device__ __forceinline__ void copy16(void* dst, const void* src, bool full) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(full ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {   // all but the last N groups
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// True in one lane of the (converged) warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0u;
}

// Pairs of fp32 values: one instruction for two of the softmax's products or sums.
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void from_f32x2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int kRegs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    kv8_prefill_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const PrefillParams p) {
  constexpr int kQBytes = Shape<D>::kQBytes, kTileBytes = Shape<D>::kTileBytes;
  constexpr int kRaw = Shape<D>::kRaw, kBlockBytes = Shape<D>::kBlockBytes;
  const int G = p.group;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sq = smem;                                 // [half]
  uint8_t* sk = sq + 2 * kQBytes;                     // [kRing]
  uint8_t* sv = sk + kRing * kTileBytes;              // [kRing]
  uint8_t* raw = sv + kRing * kTileBytes;             // [K, V][kRawRing][64 positions][128 codes]
  Factors* fac = reinterpret_cast<Factors*>(raw + 2 * kRawRing * kRaw);
  Item* items = reinterpret_cast<Item*>(fac + kFactors);   // [kItems]
  uint64_t* bars = reinterpret_cast<uint64_t*>(items + kItems);
  uint64_t* q_full = bars + 0;       // [half] Q arrived
  uint64_t* q_empty = bars + 2;      // [half] last S of the item done
  uint64_t* k_full = bars + 4;       // [kRing]
  uint64_t* k_empty = bars + 8;
  uint64_t* v_full = bars + 12;
  uint64_t* v_empty = bars + 16;
  uint64_t* s_full = bars + 20;      // [half][2]
  uint64_t* p_full = bars + 24;      // [half][2]
  uint64_t* pv_done = bars + 28;     // [half][2]
  uint64_t* o_free = bars + 32;      // [half]
  uint64_t* f_full = bars + 34;      // [kFactors]
  uint64_t* f_empty = bars + 42;     // [kFactors] P.V of the tile done: all have read them
  uint64_t* item_full = bars + 50;   // [kItems]
  uint64_t* item_empty = bars + 54;  // [kItems] read by the Q, MMA and softmax warps
  uint64_t* drain = bars + 58;
  uint64_t* turn = bars + 60;        // [half][quarter] the exponentials' turn
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 59);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&o_free[i], 128);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&k_empty[i], 2);
      mbar_init(&v_full[i], 4);
      mbar_init(&v_empty[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < kFactors; ++i) {
      mbar_init(&f_full[i], 1);
      mbar_init(&f_empty[i], 2);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 1 + 2 + 8);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&turn[i], 1);
    mbar_init(drain, 2);
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
  auto all_wait = [&](uint64_t* bar, uint32_t par) {   // by a converged warp
    return static_cast<bool>(__all_sync(0xffffffffu, mbar_wait(bar, par)));
  };
  // item number n as published, copied out of its slot; false: a wait gave up
  auto take_item = [&](int n, Item& it) -> bool {
    const int s = n % kItems;
    if (!all_wait(&item_full[s], (n / kItems) & 1)) return false;
    it = items[s];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[s]);
    return true;
  };
  // after a wait that gave up a role leaves, and the waits of the others for it give up too
  auto give_up = [&]() { report(p.status, NSLG_DEV_WAIT_TIMEOUT); };

  // 128 registers a thread at launch: 2 x 128 x 184 + 2 x 128 x 72 = 512 x 128
  if (warp < 4) {
    // -------------------------------------------------------------- converters
    regs_dec<72>();
    const int tid = threadIdx.x;
    // 16-code chunk c of positions t0 + kRows i. At head_dim 128 the lanes of the upper 64 dims
    // take the neighbouring position: the swizzle then puts the eight lanes that store
    // together into eight banks (at 64 two positions share them anyway)
    constexpr int kChunks = D / 16, kRows = Shape<D>::kRows, kSteps = kBN / kRows;
    const int c = tid % kChunks, t0 = (tid / kChunks) ^ (c >> 2);
    bool ok = true;
    const uint32_t row0 = (c >> 2) * kDimHalf + t0 * 128;
    const uint32_t at0 = row0 + (((2 * (c & 3)) ^ (t0 & 7)) << 4);
    const uint32_t at1 = row0 + (((2 * (c & 3) + 1) ^ (t0 & 7)) << 4);
    const uint32_t from = t0 % kPS * D + c * 16;       // in a page's block
    const uint32_t put = t0 * D + c * 16;              // in a raw tile
    bool more = true;                                  // tiles to come behind those fetched
    // starts the copies of tile n's codes: a group of K, a group of V (empty behind the last tile)
    auto fetch = [&](int n) -> bool {
      if (more) {
        const int fs = n % kFactors;
        if (!all_wait(&f_full[fs], (n / kFactors) & 1)) return false;
        const int held = fac[fs].held;
        more = held >= 0;
        if (more) {
          const uint32_t plain = fac[fs].plain;
          const uint8_t* ck = static_cast<const uint8_t*>(p.codes_k);
          const uint8_t* cv = static_cast<const uint8_t*>(p.codes_v);
          uint8_t* dst = raw + (n % kRawRing) * kRaw + put;
          bool has[kSteps];
          int64_t at[kSteps];
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            const int page = (t0 + kRows * i) / kPS;   // of the tile
            const int blk = fac[fs].blk[page];
            has[i] = blk >= 0 && t0 + kRows * i < held;
            at[i] = has[i] ? static_cast<int64_t>(blk) * kBlockBytes + from : 0;
            copy16(dst + i * kRows * D, ck + at[i], has[i]);
            has[i] = has[i] && ((plain >> page) & 1u); // no codes of a scale of 0 or NaN in V
          }
          copy_commit();
#pragma unroll
          for (int i = 0; i < kSteps; ++i)
            copy16(dst + kRawRing * kRaw + i * kRows * D, cv + at[i], has[i]);
          copy_commit();
          return true;
        }
      }
      copy_commit();
      copy_commit();
      return true;
    };
    // one tile of codes to 16 bits: K to q's type, V to f16
    auto convert = [&](auto kind, int n) -> bool {
      constexpr int kv = decltype(kind)::value;
      const int s = n % kRing;
      if (!all_wait(&(kv ? v_empty : k_empty)[s], ((n / kRing) & 1) ^ 1)) return false;
      const uint8_t* src = raw + (kv * kRawRing + n % kRawRing) * kRaw + put;
      uint8_t* dst = (kv ? sv : sk) + s * kTileBytes;
      auto two = [&](uint32_t codes) -> uint32_t {     // the low two codes
        const uint32_t h = f16x2_from_e4m3x2(static_cast<uint16_t>(codes));
        if constexpr (kv == 1 || Mma16<T>::kFormat == 0) {
          return h;
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
          return pack_bf16x2(f.x, f.y);
        }
      };
      uint4 w[kSteps];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) w[i] = *reinterpret_cast<const uint4*>(src + i * kRows * D);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const uint4 lo = make_uint4(two(w[i].x), two(w[i].x >> 16), two(w[i].y), two(w[i].y >> 16));
        const uint4 hi = make_uint4(two(w[i].z), two(w[i].z >> 16), two(w[i].w), two(w[i].w >> 16));
        *reinterpret_cast<uint4*>(dst + at0 + i * kRows * 128) = lo;
        *reinterpret_cast<uint4*>(dst + at1 + i * kRows * 128) = hi;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&(kv ? v_full : k_full)[s]);
      return true;
    };
    constexpr std::integral_constant<int, 0> kK{};
    constexpr std::integral_constant<int, 1> kV{};
    int tiles = 0;                                     // fetched
    for (int i = 0; ok && i < kRawRing; ++i) {
      ok = fetch(i);
      tiles += more ? 1 : 0;                           // false once a fetch has found the end
    }
    for (int n = 0; ok && n < tiles; ++n) {
      copy_wait<2 * kRawRing - 1>();
      if (!(ok = convert(kK, n))) break;
      copy_wait<2 * kRawRing - 2>();
      if (!(ok = convert(kV, n))) break;
      ok = fetch(tiles);
      tiles += more ? 1 : 0;
    }
    copy_wait<0>();                                    // none may still be writing shared memory
    if (!ok && lane == 0) give_up();
  } else if (warp < 8) {
    regs_dec<72>();
    if (warp == 4) {
      // -------------------------------------------------------------- producer
      // Pages are looked up 32 at a time (a group: 8 tiles of an item), one a lane, two groups
      // ahead: their numbers, then their scales, then the factors. Tile by tile
      // the loads' latency was 1.5 us a tile, more than all the rest of it.
      struct Group {
        int n, j0, page;                               // item (-1: none), first tile, the lane's page (-1: none)
        float sk, sv;
      };
      int n = 0;                                       // tiles published
      float carry = INFINITY;                          // least e of this item's last tile that had one
      int item = blockIdx.x, n_items = 0;              // items with tiles
      int j_next = 0, nt = 0, kv_beg = 0, npages = 0;  // of the item being looked up
      ItemLoads ahead;
      issue_item(p, item, ahead);
      auto fetch = [&](Group& gr) -> bool {
        while (j_next >= nt) {                         // the next item with tiles
          if (item >= p.n_items) {
            gr.n = -1;
            return true;
          }
          const ItemLoads L = ahead;
          item += gridDim.x;
          issue_item(p, item, ahead);
          Item it;
          if (!finish_item(p, L, it)) continue;
          if (it.ntiles == 0) {                        // rows that see no position
            const int rows = min(2 * p.tokens_per_tile, it.qo_len - it.i0);
            for (int i = 0; i < rows; ++i) {
              uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) +
                                                    (static_cast<int64_t>(it.row0) + i) * p.out_stride +
                                                    static_cast<int64_t>(it.h) * G * D);
              for (int e = lane; e < G * (D / 8); e += 32) dst[e] = make_uint4(0u, 0u, 0u, 0u);
            }
            continue;
          }
          // what has been published is at most two items behind: the roles get on to the item
          // that held this slot
          const int s = n_items % kItems;
          if (!all_wait(&item_empty[s], ((n_items / kItems) & 1) ^ 1)) return false;
          if (lane == 0) items[s] = it;
          __syncwarp();
          ++n_items;
          j_next = 0;
          nt = it.ntiles;
          kv_beg = it.kv_beg;
          npages = it.npages;
        }
        gr.n = n_items - 1;
        gr.j0 = j_next;
        const int pi = j_next * kPages + lane;
        gr.page = -1;
        if (pi < min(npages, nt * kPages)) {
          gr.page = p.kv_indices[kv_beg + pi];
          if (gr.page < 0) gr.page = -2;
        }
        j_next += 32 / kPages;
        return true;
      };
      auto load_scales = [&](Group& gr) {
        gr.sk = gr.sv = 0.f;
        if (gr.n < 0) return;
        if (gr.page < -1 || gr.page >= p.num_pages) {
          report(p.status, NSLG_DEV_BAD_PAGE);
          gr.page = -1;
        }
        if (gr.page >= 0) {
          const int64_t blk = static_cast<int64_t>(gr.page) * p.hkv + items[gr.n % kItems].h;
          gr.sk = p.scale_k[blk];
          gr.sv = p.scale_v[blk];
        }
      };
      auto publish = [&](const Group& gr) -> bool {
        const int s = gr.n % kItems;
        const int h = items[s].h, tiles = min(32 / kPages, items[s].ntiles - gr.j0);
        if (gr.j0 == 0) carry = INFINITY;              // none yet
        // ---- the factors of the lane's page
        const uint32_t nan = __ballot_sync(0xffffffffu, gr.sk != gr.sk || gr.sv != gr.sv);
        const bool plain = has_exponent(gr.sv);
        float e = log2f(gr.sv);
        const uint32_t own = __ballot_sync(0xffffffffu, plain);
        float least = plain ? e : INFINITY;            // of the tile's pages
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, 1));
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, 2));
        if (own != 0xffffffffu) {                      // the last tile, this one included, that has one
          const uint32_t upto = own & ((2u << (lane | (kPages - 1))) - 1u);
          const float last = __shfl_sync(0xffffffffu, least, upto != 0u ? 31 - __clz(upto) : 0);
          const float before = upto != 0u ? last : carry;
          if (!plain) e = before == INFINITY ? 0.f : fmaxf(before - kZeroE, kLeastE);
        }
        if (own != 0u) carry = __shfl_sync(0xffffffffu, least, 31 - __clz(own));
        const float inv = exp2f(-e), f_log2 = fmaxf(gr.sk * p.scale_log2, 1e-37f);
        const int blk = gr.page >= 0 ? gr.page * p.hkv + h : -1;
        for (int j = 0; j < tiles; ++j, ++n) {
          const int fs = n % kFactors;
          if (!all_wait(&f_empty[fs], ((n / kFactors) & 1) ^ 1)) return false;
          Factors& fc = fac[fs];
          if (lane / kPages == j) {
            fc.f[lane % kPages] = f_log2;
            fc.e[lane % kPages] = e;
            fc.inv[lane % kPages] = inv;
            fc.blk[lane % kPages] = blk;
            if (lane % kPages == 0) {
              fc.plain = (own >> lane) & ((1u << kPages) - 1u);
              fc.nan = (nan >> lane) & ((1u << kPages) - 1u);
              fc.held = items[s].kv_len - (gr.j0 + j) * kBN;
            }
          }
          const bool first = gr.j0 == 0 && j == 0;
          __syncwarp();
          if (lane == 0) {
            if (first) mbar_arrive(&item_full[s]);
            mbar_arrive(&f_full[fs]);
          }
        }
        return true;
      };
      Group g0, g1, g2;
      bool ok = fetch(g0);
      if (ok) {
        load_scales(g0);
        ok = fetch(g1);
      }
      while (ok && g0.n >= 0) {
        load_scales(g1);
        if (!(ok = fetch(g2)) || !(ok = publish(g0))) break;
        g0 = g1;
        g1 = g2;
      }
      if (ok) {
        const int s = n_items % kItems, fs = n % kFactors;
        ok = all_wait(&item_empty[s], ((n_items / kItems) & 1) ^ 1) &&
             all_wait(&f_empty[fs], ((n / kFactors) & 1) ^ 1);
        if (ok && lane == 0) {
          items[s].ntiles = -1;
          mbar_arrive(&item_full[s]);
          fac[fs].held = -1;
          mbar_arrive(&f_full[fs]);
        }
      }
      if (!ok && lane == 0) give_up();
    } else if (warp == 7) {
      // -------------------------------------------------------------- Q
      // a warp of its own: the rows of an item may be copied only when the last scores of the
      // one before are done, and the producer is tiles ahead of that
      const uint64_t keep = l2_policy_evict_last();
      bool ok = true;
      int nq = 0;                                      // halves copied
      Item it;
      for (int n = 0; (ok = take_item(n, it)) && it.ntiles >= 0; ++n) {
#pragma unroll 1
        for (int x = 0; ok && x < 2; ++x) {
          if (!(ok = all_wait(&q_empty[x], (n & 1) ^ 1))) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[x], kQBytes);
            uint8_t* dst = sq + x * kQBytes;
            const int row = it.row0 + x * p.tokens_per_tile;
            tma_load_3d(dst, &tmap_q, &q_full[x], 0, it.h * G, row, keep);
            if constexpr (D == 128) tma_load_3d(dst + kQDimHalf, &tmap_q, &q_full[x], 64, it.h * G, row, keep);
          }
          ++nq;
          __syncwarp();
        }
        if (!ok) break;
      }
      if (!ok) {
        if (lane == 0) give_up();
        // no copy may still be writing shared memory when the CTA leaves (bounded waits)
        for (int x = 0; x < 2; ++x) {
          const int loads = (nq + 1 - x) / 2;
          if (loads > 0) (void)mbar_wait(&q_full[x], (loads - 1) & 1);
        }
      }
    } else {
      // -------------------------------------------------------------- MMA issuers, one per half
      // The whole warp runs the loop and one elected lane issues: the descriptors then stay
      // warp-uniform. With the loop in one lane an MMA costs enough instructions that the
      // softmax warps on the same scheduler held it to 118 clocks an m128n128k16 instead of 64
      // (71 this way, FMA-bound warps beside it); and one warp for both halves spent 2.1 us of
      // issuing and waiting on a tile whose products take 0.7.
      const int x = warp - 5;
      constexpr uint32_t kIdescS = idesc_f16(Mma16<T>::kFormat, kBN, false);
      constexpr uint32_t kIdescO = idesc_f16(0, D, true);
      constexpr uint32_t kDescHi = smem_desc_hi(1024);
      const uint32_t q_lo = smem_desc_lo(smem_u32(sq + x * kQBytes), 16);
      const uint32_t k_lo0 = smem_desc_lo(smem_u32(sk), 16);
      const uint32_t v_lo0 = smem_desc_lo(smem_u32(sv), kDimHalf);
      const uint32_t hb = tmem + x * kHalfCols;
      bool ok = true;
      // The tiles of all items form one stream. S(u) goes into the buffer of P(u - 2), right
      // behind P(u - 2).V in the pipe, so it is there when the softmax has done tile u - 1, and
      // an item's first scores are computed while the rows before are written.
      int u = 0, sj = 0, snt = 0, n = 0;     // tiles scored; tile of the item being scored; items
      bool end = false;
      int nts[3] = {0, 0, 0};                // tiles of the items between P.V and S, oldest first
      int held = 0;                          // ... how many
      // S of the tiles up to t + 2 (t + 1 where Q is not there yet)
      auto score = [&](int t) {
        while (!end && u <= t + 2) {
          if (sj == snt) {                   // the next item with tiles
            Item it;
            if (!(ok = take_item(n, it)) || it.ntiles < 0) {
              end = true;
              return;
            }
            ++n;
            snt = it.ntiles;
            sj = 0;
            if (held == 0) nts[0] = snt;
            else if (held == 1) nts[1] = snt;
            else nts[2] = snt;
            ++held;
          }
          const uint32_t q_par = (n - 1) & 1;
          if (sj == 0) {
            if (u > t + 1 && !__all_sync(0xffffffffu, mbar_try_wait(&q_full[x], q_par))) return;
            if (!(ok = all_wait(&q_full[x], q_par))) return;
          }
          const int slot = u % kRing;
          if (!(ok = all_wait(&k_full[slot], (u / kRing) & 1))) return;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t k_lo = k_lo0 + slot * (kTileBytes >> 4), dcol = hb + 64 * (u & 1);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              mma_ss_w(dcol, q_lo + (((ks >> 2) * kQDimHalf + (ks & 3) * 32) >> 4),
                       k_lo + (((ks >> 2) * kDimHalf + (ks & 3) * 32) >> 4), kDescHi, kIdescS,
                       ks > 0 ? 1u : 0u);
            mma_commit(&s_full[x * 2 + (u & 1)]);
            mma_commit(&k_empty[slot]);
            if (sj + 1 == snt) mma_commit(&q_empty[x]);
          }
          __syncwarp();
          ++sj;
          ++u;
        }
      };
      int t = -2, pj = 0, n_o = 0;           // tile, its place in its item, items whose O was begun
#pragma unroll 1
      for (; ok && t < 0; ++t) score(t);
      for (t = 0; ok && t < u; ++t) {
        const int slot = t % kRing, b = t & 1;
        if (!(ok = all_wait(&v_full[slot], (t / kRing) & 1))) break;
        if (!(ok = all_wait(&p_full[x * 2 + b], (t >> 1) & 1))) break;
        if (pj == 0 && n_o++ > 0 && !(ok = all_wait(&o_free[x], n_o & 1))) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t v_lo = v_lo0 + slot * (kTileBytes >> 4);
#pragma unroll
          for (int kt = 0; kt < kBN / 16; ++kt)
            mma_ts_w(hb + kColO, hb + 64 * b + kt * 8, v_lo + (kt * 2048 >> 4), kDescHi, kIdescO,
                     (pj > 0 || kt > 0) ? 1u : 0u);
          mma_commit(&pv_done[x * 2 + b]);
          mma_commit(&v_empty[slot]);
          mma_commit(&f_empty[t % kFactors]);
        }
        __syncwarp();
        if (++pj == nts[0]) {
          pj = 0;
          nts[0] = nts[1];
          nts[1] = nts[2];
          --held;
        }
        score(t);
      }
      if (!ok && lane == 0) give_up();
      if (elect_one()) mma_commit(drain);              // everything issued has completed (bounded)
      __syncwarp();
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
    const bool wide = ((reinterpret_cast<uintptr_t>(p.out) | static_cast<uintptr_t>(p.out_stride) * sizeof(T)) & 31) == 0;
    int t = 0;
    bool ok = true;
    // The rows of the item before, whose o is written behind this item's first tile of
    // softmax: its last P.V has been done by then.
    bool due = false;
    T* due_dst = nullptr;                              // null: a row of no sequence
    float due_l = 0.f;
    Item it, nx;
    ok = take_item(0, nx);
    for (int n = 1; ok && (nx.ntiles >= 0 || due); ++n) {
      it = nx;
      const bool end = it.ntiles < 0;                  // no more: only o is due
      const int i0 = it.i0 + x * p.tokens_per_tile + tok;   // the row's new token
      const bool live = i0 < it.qo_len;
      // last position the row sees; a row of no sequence sees everything and is not written
      const int lim = !live      ? 0x7fffffff
                      : p.causal ? min(it.kv_len - it.qo_len + i0, it.kv_len - 1)
                                 : it.kv_len - 1;
      const int low = __reduce_min_sync(0xffffffffu, lim);
      float m = -INFINITY, l = 0.f;
      bool seen = false;                               // a tile with an E of its own
      // one tile; edge: some row of the warp does not see all of it
      auto softmax = [&](bool edge, int j) -> bool {
        const Factors& fc = fac[t % kFactors];
        const int gap = lim - j * kBN;                 // last column the row sees
        const int b = t & 1;
        float s[kBN];
        tmem_ld64(base + 64 * b, s);
        tmem_wait_ld();
        if (edge || fc.nan != 0u) {
          const uint32_t nan = fc.nan;
#pragma unroll
          for (int c = 0; c < kBN; ++c) {
            if ((nan >> (c / kPS)) & 1u) s[c] = NAN;
            if (c > gap) s[c] = -INFINITY;
          }
        }
        auto page_max = [&](int g) {                   // of t over the page; NaN is ignored
          const float* sg = s + g * 16;
          float a = fmaxf(fmaxf(sg[0], sg[1]), sg[2]), b2 = fmaxf(fmaxf(sg[3], sg[4]), sg[5]);
          a = fmaxf(fmaxf(a, sg[6]), sg[7]);
          b2 = fmaxf(fmaxf(b2, sg[8]), sg[9]);
          a = fmaxf(fmaxf(a, sg[10]), sg[11]);
          b2 = fmaxf(fmaxf(b2, sg[12]), sg[13]);
          a = fmaxf(fmaxf(a, sg[14]), sg[15]);
          return fmaf(fmaxf(a, b2), fc.f[g], fc.e[g]);
        };
        float alpha = 1.f;
        auto raise_to = [&](float mt) {
          if (m != -INFINITY && mt != -INFINITY) alpha = fast_exp2(m - mt);
          m = mt;
        };
        const bool own = fc.plain != 0u, anew = !seen && own;   // anew: O is all zeros so far,
        seen = seen || own;                            // M may go down too
        float mt = -INFINITY;
#pragma unroll
        for (int g = 0; g < kPages; ++g) mt = fmaxf(mt, page_max(g));
        if (anew && mt > -INFINITY)
          raise_to(fmaxf(mt, m - kMostDown));
        else if (mt > m + 8.f)
          raise_to(mt);
        const float nb = m == -INFINITY ? 0.f : -m;
        if (!all_wait(&turn[x * 4 + quarter], (t & 1) ^ 1 ^ x)) return false;
#pragma unroll
        for (int g = 0; g < kPages; ++g) {
          const float add = fc.e[g] + nb;
          const uint64_t F2 = f32x2(fc.f[g], fc.f[g]), add2_ = f32x2(add, add);
#pragma unroll
          for (int c = g * 16; c < g * 16 + 16; c += 2) {
            from_f32x2(fma2(f32x2(s[c], s[c + 1]), F2, add2_), s[c], s[c + 1]);
            s[c] = fast_exp2(s[c]);
            s[c + 1] = fast_exp2(s[c + 1]);
          }
        }
        float sum = 0.f;
        uint32_t pk[32];
#pragma unroll
        for (int g = 0; g < kPages; ++g) {
          uint64_t gs = f32x2(s[g * 16], s[g * 16 + 1]);
#pragma unroll
          for (int c = 0; c < 16; c += 2) {
            if (c > 0) gs = add2(gs, f32x2(s[g * 16 + c], s[g * 16 + c + 1]));
            pk[g * 8 + c / 2] = pack_f16x2(s[g * 16 + c], s[g * 16 + c + 1]);
          }
          float a, b2;
          from_f32x2(gs, a, b2);
          sum = fmaf(a + b2, fc.inv[g], sum);
        }
        tmem_st32(base + 64 * b, pk);                  // P over S
        if (lane == 0) mbar_arrive(&turn[(x ^ 1) * 4 + quarter]);
        __syncwarp();
        // O may only be rescaled once P(t-1).V(t-1) is done (tcgen05.ld / st are
        // warp-collective; rows with alpha == 1 multiply by 1)
        if (j > 0 && !anew && __any_sync(0xffffffffu, alpha != 1.f)) {
          if (!all_wait(&pv_done[x * 2 + (b ^ 1)], ((t - 1) >> 1) & 1)) return false;
          tc_fence_after();
#pragma unroll 1
          for (int cb = 0; cb < D; cb += 32) {
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
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[x * 2 + b]);
        return true;
      };
      for (int j = 0; j == 0 || j < it.ntiles; ++j) {
        if (!end) {
          if (j + 1 == it.ntiles && !(ok = take_item(n, nx))) break;
          // S(t) is made of K(t), which was fetched with the factors: they are there
          if (!(ok = all_wait(&s_full[x * 2 + (t & 1)], (t >> 1) & 1))) break;
          tc_fence_after();
          if (!(ok = softmax(!__all_sync(0xffffffffu, (j + 1) * kBN - 1 <= lim), j))) break;
        }
        if (j == 0 && due) {
          const int tl = t - 1;                        // the last tile of the item before
          if (!(ok = all_wait(&pv_done[x * 2 + (tl & 1)], (tl >> 1) & 1))) break;
          tc_fence_after();
          const float inv = due_l == 0.f ? 0.f : 1.f / due_l;
#pragma unroll 1
          for (int cb = 0; cb < D; cb += 64) {
            float o[64];
            tmem_ld64(base + kColO + cb, o);
            tmem_wait_ld();
            if (cb + 64 == D) {
              tc_fence_before();
              mbar_arrive(&o_free[x]);                 // O may be overwritten now
            }
            if (due_dst != nullptr) {
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  w[e] = Mma16<T>::pack(o[16 * c + 2 * e] * inv, o[16 * c + 2 * e + 1] * inv);
                T* at = due_dst + cb + 16 * c;
                if (wide) {
                  // a thread's row against the others' is a line each: fewer, wider stores
                  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at),
                               "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                               "r"(w[6]), "r"(w[7])
                               : "memory");
                } else {
                  reinterpret_cast<uint4*>(at)[0] = make_uint4(w[0], w[1], w[2], w[3]);
                  reinterpret_cast<uint4*>(at)[1] = make_uint4(w[4], w[5], w[6], w[7]);
                }
              }
            }
          }
        }
        if (!end) ++t;
      }
      if (end) break;
      due = true;
      due_l = l;
      due_dst = live ? static_cast<T*>(p.out) +
                           (static_cast<int64_t>(it.row0) + x * p.tokens_per_tile + tok) * p.out_stride +
                           static_cast<int64_t>(it.h * G + hd) * D
                     : nullptr;
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

namespace {

template <typename T, int D>
int launch_typed(const PrefillParams& p, cudaStream_t stream) {
  CUtensorMap tq;
  const int rc = encode_tiled_3d_bf16(&tq, p.q, D, p.hq, p.num_rows, static_cast<uint64_t>(D) * 2,
                                      static_cast<uint64_t>(p.q_stride) * 2, 64, p.group,
                                      p.tokens_per_tile);
  if (rc != NSLG_OK) return rc;
  constexpr int kSmemBytes = Shape<D>::kSmemBytes;
  const int sms = sm_count();
  const unsigned grid = static_cast<unsigned>(p.n_items < sms ? p.n_items : sms);
  auto kern = kv8_prefill_tc_kernel<T, D>;
  const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (err != cudaSuccess) return set_error(NSLG_ERR_CUDA, cudaGetErrorString(err));
  kern<<<grid, kThreads, kSmemBytes, stream>>>(tq, p);
  return check_launch("kv8_prefill_tc");
}

// Pairs of query tiles of the longest sequence.
int64_t pairs_of(int group, int max_qo_len) {
  return (static_cast<int64_t>(max_qo_len) * group + 2 * kBM - 1) / (2 * kBM);
}

}  // namespace

bool kv8_prefill_tc_supported(int dtype, const Kv8AttnParams& p) {
  if ((dtype != NSLG_DTYPE_BF16 && dtype != NSLG_DTYPE_F16) || (p.d != 64 && p.d != 128) ||
      p.page_size != kPS)
    return false;
  const int g = p.hq / p.hkv;
  if (g > 16 || kBM % g != 0 || p.num_rows >= (int64_t{1} << 31)) return false;
  if (p.num_pages * p.hkv >= (int64_t{1} << 31)) return false;   // blocks are 32-bit numbers
  return pairs_of(g, p.max_qo_len) * p.batch * p.hkv < (int64_t{1} << 30);
}

// Against the split-KV kernel (kv8_attn_tc): that one streams the cache once per 16 query rows,
// spread over all SMs; this one streams it once per 256, an SM to each item. A round of items
// takes what the split kernel takes for about two tiles of 16 rows an SM, whatever the
// lengths. Measured (us, this kernel against split; bf16, 32 / 8 heads of 128; sequences x
// context, query rows a kv head):
//   1 x 4096, 256 rows    80 : 43      16 x 1024, 48 rows    26 : 39
//   4 x 4096, 128 rows    81 : 74      64 x 4096, 32 rows   305 : 257
//   4 x 4096, 192 rows    81 : 103     64 x 4096, 48 rows   315 : 378
bool kv8_prefill_tc_faster(const Kv8AttnParams& p) {
  const int g = p.hq / p.hkv, sms = sm_count();
  const int64_t vs = static_cast<int64_t>(p.batch) * p.hkv;
  const int64_t rounds = (pairs_of(g, p.max_qo_len) * vs + sms - 1) / sms;
  return vs * ((static_cast<int64_t>(p.max_qo_len) * g + 15) / 16) > 2 * rounds * sms;
}

int launch_kv8_prefill_tc(int dtype, const Kv8AttnParams& a, cudaStream_t stream) {
  PrefillParams p{};
  static_cast<Kv8AttnParams&>(p) = a;
  p.group = a.hq / a.hkv;
  p.tokens_per_tile = kBM / p.group;
  p.scale_log2 = a.sm_scale * 1.4426950408889634f;
  p.n_items = static_cast<int>(pairs_of(p.group, a.max_qo_len) * a.batch * a.hkv);
  if (dtype == NSLG_DTYPE_F16)
    return a.d == 128 ? launch_typed<__half, 128>(p, stream) : launch_typed<__half, 64>(p, stream);
  return a.d == 128 ? launch_typed<__nv_bfloat16, 128>(p, stream)
                    : launch_typed<__nv_bfloat16, 64>(p, stream);
}

}  // namespace nslg
