// Attention of a ragged batch's new tokens over the paged cache for many rows per
// kv head (prompt chunks, long drafted blocks): the tensor-core form of the
// mathematics in paged_attn.cu.
//
// Bound: the two products, 4 * head_dim flops for each visible (row, key) pair, on
// tcgen05; the keys and values come from L2 after the first row tile of a head.
//
// One persistent CTA per SM walks its items (paged_plan.h) with warp roles:
//   warp 8       producer: q tiles (TMA), then 128-key tiles of K and V: UMMA pages
//                as one bulk copy each, row pages as TMA boxes (128-byte swizzle)
//   warp 9       MMA issuer (one thread): S = Q K^T and O += P V, 128 x 128 x 16
//                steps, S and O in TMEM, P written over S as 16-bit A operand
//   warp 10      (16-bit pages) zeroes the value rows of a span's first and last tile
//                that no row sees: a weight of 0 would still turn a NaN there into NaN
//   warps 0-7    two softmax warpgroups, thread = row = TMEM lane
//   warps 10, 11 (e4m3 pages) look for NaN codes in the landed tiles
//   warps 12-15  (e4m3 pages) widen the landed 8-bit tiles, scale included, into the
//                bf16 tiles the products read; exact, see paged.cuh
// The two warpgroups ("streams") alternate on the tensor core: while one turns S
// into P the other's products run. A unit of more rows than one tile gives each
// stream a q tile of its own against the same keys; a unit of at most one tile
// gives both the same rows and every other key tile (`split`), joined at the end
// through TMEM, so few rows do not leave half of the machine idle.
// A q tile is floor(128 / G) tokens times the G heads of the kv head, so any G
// works; the rows behind them hold whatever the buffer held and are never written.
//
// Online softmax in the log2 domain with a lazy maximum: O is rescaled in TMEM
// only when the running maximum grows by more than 8 (f16: 4). Weights are rounded to
// nearest for the second product; their fp32 values go into the sum. f16 weights are
// taken 2^11 times as large, up to 2^15: what lies below 2^-14 is subnormal, so they
// are off by 2^-11 relative down to 2^-25 of the row's largest, and below that by at
// most 2^-36 of it (a prompt of 8192 tokens in f16 takes 482 us so, 483 with weights of
// up to 2^8, and 509 with rescaling from 2 on and a factor of 2^13). Tiles that every
// row sees whole skip the mask; the others take
// each score's minimum with an infinity of the sign that the row's [lo, hi) gives it.
//
// Measured, as calls among others (32 / 8 heads of 128, bf16; of 1657 TFLOP/s of a
// library product in a burst, 1395 under the power cap): a prompt of 8192 tokens 540 us =
// 1019 TFLOP/s = 0.61 (0.73). The chain of one q tile -- softmax, P V, the next
// Q K^T and two hand-offs -- is as long as the other tile's, which it passes under, so
// the tensor pipe is active for 53% of the time and the exponential unit for 54%.
// Heads of 64 have half the product per tile and the same softmax. 16 blocks of 16
// tokens over 2k to 16k keys 150 us = 0.67 of the copy rate, 9 us of it the joining
// kernel (134 us a call where calls follow at once and the next one starts under it); over
// e4m3 pages, half of the bytes, 234 us: the widening is the chain. Chunks under a window
// of 128 are two tiles each: the start and end of a unit are most of its 7 us (six
// chunks 79 us a call).
#include <atomic>
#include <string>
#include <type_traits>

#include "paged_attn.cuh"

namespace d2sd {
namespace paged {
namespace {

enum { kNative = 0, kRows = 1, kE4m3 = 2 };

constexpr int kTmaWarp = 8, kMmaWarp = 9, kFixWarp = 10;
constexpr uint32_t kTmemCols = 512;
constexpr int kPanelBytes = 128 * 128;  // 128 rows x 64 16-bit values

// SPLIT: no unit of the launch has a second q tile, and its room goes to more stages
// (16 blocks of 16 tokens against 2k to 16k keys, back to back: 134 us against 146).
template <int D, int MODE, bool SPLIT>
struct Cfg {
  static constexpr int kThreads = MODE == kE4m3 ? 512 : 384;
  // registers: with 384 threads the launch's 168 a thread are shared out between
  // the softmax warpgroups and the third (setmaxnreg); with 512 every thread has 128
  static constexpr int kLaunchRegs = 168, kSoftmaxRegs = 192, kSideRegs = 112;
  static_assert(256 * kSoftmaxRegs + 128 * kSideRegs <= 384 * kLaunchRegs,
                "register split above the launch's registers");
  static constexpr int kPanels = D / 64;
  static constexpr int kTileBytes = 128 * D * 2;
  // of K and of V
  static constexpr int kStages = MODE != kE4m3 && SPLIT ? (D == 128 ? 3 : 6) : (D == 128 ? 2 : 4);
  static constexpr int kSmemQ = 0;
  static constexpr int kSmemK = kSmemQ + (SPLIT ? 1 : 2) * kTileBytes;
  static constexpr int kSmemV = kSmemK + kStages * kTileBytes;
  static constexpr int kSmemLand = kSmemV + kStages * kTileBytes;  // 8-bit K, V tiles, their scales
  static constexpr int kLandBytes = 128 * D;
  // 8-bit tiles on their way in: one of K and V each, more where there is room (a
  // widened tile's buffer is filled again only after it, a latency of about 2 us; 16
  // blocks of 16 tokens over e4m3 223 us with one)
  static constexpr int kLand = MODE != kE4m3 ? 0 : (D == 128 ? (SPLIT ? 2 : 1) : 3);
  static_assert(kLand <= kStages, "a tile lands only when the stage's last tile has been counted (nan_finder)");
  static constexpr int kSmemScales = kSmemLand + kLand * 2 * kLandBytes;  // [kLand][K, V][128]
  static constexpr int kSmemJoin = kSmemScales + kLand * 256;
  static constexpr int kSmemBar = kSmemJoin + 128 * 8;  // [128] (m, l) of stream 1
  static constexpr int B_QFULL = 0, B_QFREE = 1, B_KFULL = 2, B_VFULL = B_KFULL + kStages,
                       B_KEMPTY = B_VFULL + kStages, B_VEMPTY = B_KEMPTY + kStages,
                       B_SFULL = B_VEMPTY + kStages, B_PHALF = B_SFULL + 2, B_PFULL = B_PHALF + 2,
                       B_OFINAL = B_PFULL + 2, B_OFREE = B_OFINAL + 2, B_VREADY = B_OFREE + 2,
                       B_LFULL = B_VREADY + kStages, B_LEMPTY = B_LFULL + 2 * kLand, B_WIDE = B_LEMPTY + 2 * kLand,
                       kNumBars = B_WIDE + 2 * kLand;
  static constexpr int kSmemBytes = kSmemBar + kNumBars * 8 + 32 + 1024;  // + alignment slack
  static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");
};

__device__ __forceinline__ void prefetch_l1(const void* p) {
  asm volatile("prefetch.global.L1 [%0];" ::"l"(p));
}
__device__ __forceinline__ uint32_t s_col(int i) { return static_cast<uint32_t>(i * 128); }
__device__ __forceinline__ uint32_t o_col(int i) { return static_cast<uint32_t>(256 + i * 128); }

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  const bool ok = mbar_wait(bar, parity, abort);
  return __all_sync(0xffffffffu, ok);
}
// One lane of the warp. The compiler knows that a branch on it runs a single
// thread, so what tcgen05 takes from uniform registers is computed there; behind
// `lane == 0` every operand of every product is moved over one by one.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// Lanes `step` apart exchange: the lower keeps a and takes the other's a as b, the
// upper (up = 1) keeps b and takes the other's b as a.
__device__ __forceinline__ void quad_swap(uint4& a, uint4& b, int up, int step) {
  uint4 s = up ? a : b;
  s.x = __shfl_xor_sync(0xffffffffu, s.x, step);
  s.y = __shfl_xor_sync(0xffffffffu, s.y, step);
  s.z = __shfl_xor_sync(0xffffffffu, s.z, step);
  s.w = __shfl_xor_sync(0xffffffffu, s.w, step);
  if (up) a = s; else b = s;
}
// a shared-memory descriptor moved by `bytes` (its start address is the low 14
// bits, address >> 4; shared addresses are below 256 KB, so nothing is carried)
__device__ __forceinline__ uint64_t desc_at(uint64_t d, uint32_t bytes) {
  uint32_t lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(d));
  lo += bytes >> 4;
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}

// What every role derives from an item. rG = 1 / G: the unit's rows are at most 256
// and a multiple of G, so the rounded product is their number of tokens.
struct Item {
  int head, tok0, tokb, ntok, key0, key1, pos0, window, kv_len, parts, slot, page_off;
  int tiles;
  bool split;  // both streams on the same q tile, every other key tile
  Item() = default;
  __device__ __forceinline__ Item(const int32_t* items, int it, float rG, int TT) {
    const int4* p = reinterpret_cast<const int4*>(items + it * kItemInts);
    const int4 a = __ldg(p), b = __ldg(p + 1), c = __ldg(p + 2), d = __ldg(p + 3);
    static_assert(P_HEAD == 1 && P_TOK0 == 2 && P_NROWS == 4 && P_KEY0 == 5 && P_KEY1 == 6 && P_POS0 == 7 &&
                      P_WINDOW == 8 && P_PAGE_OFF == 9 && P_KV_LEN == 10 && P_SLOT == 11 && P_PARTS == 12 &&
                      P_FIRST_TOKEN == 13 && kItemInts == 16,
                  "the layout read here");
    head = a.y, tok0 = a.z, key0 = b.y, key1 = b.z, pos0 = b.w, window = c.x, page_off = c.y, kv_len = c.z;
    slot = c.w, parts = d.x, tokb = d.y;
    ntok = __float2int_rn(b.x * rG);
    tiles = (key1 - key0 + kTileKeys - 1) / kTileKeys;
    split = ntok <= TT;
  }
  __device__ __forceinline__ int row_hi(int t) const { return max(0, min(kv_len, pos0 + t + 1)); }
  __device__ __forceinline__ int row_lo(int t) const { return window ? max(0, pos0 + t + 1 - window) : 0; }
  // keys [lo, hi) that some row of the unit sees
  __device__ __forceinline__ int hi_max() const { return row_hi(tokb + ntok - 1); }
  __device__ __forceinline__ int lo_min() const { return row_lo(tokb); }
  __device__ __forceinline__ bool fix(int t) const {  // tile t has values no row sees
    const int k = key0 + t * kTileKeys;
    return k + kTileKeys > hi_max() || k < lo_min();
  }
  __device__ __forceinline__ int count(int i) const { return split ? (tiles + 1 - i) / 2 : tiles; }
  __device__ __forceinline__ int tile(int i, int j) const { return split ? 2 * j + i : j; }
};

// ---------------------------------------------------------------------------
template <int D, int MODE, bool SPLIT>
__device__ void producer(const CUtensorMap* tm_q, const CUtensorMap* tm_k, const CUtensorMap* tm_v,
                         const AttnArgs& a, uint8_t* smem, uint64_t* bars, volatile int* abort,
                         const int32_t* items, int item0, int item1, int G, float rG, int TT, int rpb) {
  using C = Cfg<D, MODE, SPLIT>;
  const int lane = threadIdx.x & 31;
  const int boxes = kTileKeys / rpb;  // copies of a K or V tile (<= 8 ... 16)
  uint32_t kt = 0, kitem = 0;
  bool alive = true;
  for (int it = item0; it < item1 && alive; ++it) {
    const Item I(items, it, rG, TT);
    if (it + 2 < item1) prefetch_l1(items + (it + 2) * kItemInts);  // for every role
    if (I.tiles == 0) continue;
    // lane b: the page of box b of tile t (slots behind the last position are
    // filled from the last page and masked), clamped to the pool
    const int last = (I.kv_len - 1) / rpb;
    auto box_page = [&](int t) -> int {
      int b = (I.key0 + t * kTileKeys) / rpb + lane;
      if (b > last) b = last;
      const int64_t e = I.page_off + static_cast<int64_t>(b) * rpb / a.g.page_size;
      if (lane >= boxes || e >= a.page_table_len) return 0;
      if (!a.page_table) return static_cast<int>(e - a.first_entry);  // widened pages
      const int64_t id = a.page_table[e];
      return static_cast<int>(id < 0 ? 0 : (id >= a.g.num_pages ? a.g.num_pages - 1 : id));
    };
    auto box_slot = [&](int t, int b) -> int {
      int x = (I.key0 + t * kTileKeys) / rpb + b;
      if (x > last) x = last;
      return static_cast<int>(static_cast<int64_t>(x) * rpb % a.g.page_size);
    };
    int page = box_page(0);
    for (int t = 0; t < I.tiles && alive; ++t, ++kt) {
      const int next = (t + 1 < I.tiles) ? box_page(t + 1) : 0;
      const uint32_t st = kt % C::kStages, use = kt / C::kStages;
      for (int kv = 0; kv < 2; ++kv) {
        uint64_t* full;
        bool ok = true;
        uint8_t* land = nullptr;
        uint8_t* scales = nullptr;
        if constexpr (MODE == kE4m3) {
          const uint32_t ls = kt % C::kLand, lu = kt / C::kLand;
          full = &bars[C::B_LFULL + 2 * ls + kv];
          land = smem + C::kSmemLand + (2 * ls + kv) * C::kLandBytes;
          scales = smem + C::kSmemScales + (2 * ls + kv) * 128;
          if (lane == 0 && lu > 0) ok = mbar_wait(&bars[C::B_LEMPTY + 2 * ls + kv], (lu - 1) & 1, abort);
        } else {
          full = &bars[(kv ? C::B_VFULL : C::B_KFULL) + st];
          if (lane == 0 && use > 0)
            ok = mbar_wait(&bars[(kv ? C::B_VEMPTY : C::B_KEMPTY) + st], (use - 1) & 1, abort);
        }
        alive = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (!alive) break;
        if (MODE == kRows) {
          if (lane == 0) mbar_arrive_expect_tx(full, C::kTileBytes);
          uint8_t* dst = smem + (kv ? C::kSmemV : C::kSmemK) + st * C::kTileBytes;
          __syncwarp();
          if (lane < boxes) {
            const int slot = box_slot(t, lane);
#pragma unroll
            for (int pn = 0; pn < C::kPanels; ++pn)
              tma_load_4d(dst + pn * kPanelBytes + lane * rpb * 128, kv ? tm_v : tm_k, full, pn * 64, slot,
                          I.head, page);
          }
        } else {
          constexpr int kBlock = 16 * D * (MODE == kE4m3 ? 1 : 2);  // a page of one head
          uint8_t* dst = MODE == kE4m3 ? land
                                       : smem + (kv ? C::kSmemV : C::kSmemK) + st * C::kTileBytes;
          if (lane == 0) mbar_arrive_expect_tx(full, 8 * (kBlock + (MODE == kE4m3 ? 16 : 0)));
          __syncwarp();
          if (lane < 8) {
            const int64_t p = page;
            bulk_load(dst + lane * kBlock, (kv ? a.v_pool : a.k_pool) + p * a.g.stride_page + I.head * a.g.stride_head,
                      kBlock, full);
            if (MODE == kE4m3)
              bulk_load(scales + lane * 16,
                        (kv ? a.v_scale : a.k_scale) + p * a.g.scale_page + I.head * a.g.scale_head, 16, full);
          }
        }
      }
      page = next;
      if (t > 0) continue;
      // q behind the first tile's keys and values: its buffer is free only when the
      // previous item's last S is done, and their copies need not wait for that
      if (lane == 0) {
        if (kitem > 0 && !mbar_wait(&bars[C::B_QFREE], (kitem - 1) & 1, abort)) alive = false;
        if (alive) {
          const int nq = I.split ? 1 : 2;
          mbar_arrive_expect_tx(&bars[C::B_QFULL], nq * C::kPanels * TT * G * 128);
          for (int i = 0; i < nq; ++i)
            for (int pn = 0; pn < C::kPanels; ++pn)
              tma_load_3d(smem + C::kSmemQ + i * C::kTileBytes + pn * kPanelBytes, tm_q,
                          &bars[C::B_QFULL], pn * 64, I.head * G, I.tok0 + I.tokb + i * TT);
        }
      }
      ++kitem;
      alive = __shfl_sync(0xffffffffu, alive ? 1 : 0, 0) != 0;
    }
  }
}

// S = Q K^T: N = 128 keys, D in steps of 16 (descriptors as in prefix_attn.cu: q
// and row pages are 128-byte-swizzled panels, UMMA pages core matrices).
template <int D, bool SWZ>
__device__ __forceinline__ void issue_qk(uint32_t tmem_s, uint64_t qd, uint64_t kd, uint32_t idesc) {
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    const uint32_t off = (ks / 4) * kPanelBytes + (ks % 4) * 32;
    umma_ss(tmem_s, desc_at(qd, off), desc_at(kd, SWZ ? off : ks * 256), idesc, ks > 0 ? 1u : 0u);
  }
}
// O (+)= P V for the 16-key steps [KS0, KS1)
template <int D, bool SWZ, int KS0, int KS1>
__device__ __forceinline__ void issue_pv(uint32_t tmem_o, uint32_t tmem_p, uint64_t vd, uint32_t idesc,
                                         bool accumulate) {
  constexpr uint32_t kGroup = (D / 8) * 128;
#pragma unroll
  for (int ks = KS0; ks < KS1; ++ks)
    umma_ts(tmem_o, tmem_p + ks * 8, desc_at(vd, SWZ ? ks * 16 * 128 : ks * 2 * kGroup), idesc,
            (accumulate || ks > 0) ? 1u : 0u);
}

template <typename T, int D, int MODE, bool SPLIT>
__device__ void mma_issuer(uint8_t* smem, uint64_t* bars, uint32_t tmem, volatile int* abort,
                           const int32_t* items, int item0, int item1, float rG, int TT) {
  using C = Cfg<D, MODE, SPLIT>;
  constexpr bool SWZ = MODE == kRows;
  constexpr uint32_t kFmt = std::is_same<T, __half>::value ? 0u : 1u;
  constexpr uint32_t qk_desc = umma_idesc(128, 128, false, kFmt), pv_desc = umma_idesc(128, D, true, kFmt);
  constexpr uint32_t kGroup = (D / 8) * 128;
  const uint64_t qd0 = umma_desc_sw128(smem_u32(smem + C::kSmemQ), 16, 1024);
  const uint64_t kd0 = SWZ ? umma_desc_sw128(smem_u32(smem + C::kSmemK), 16, 1024)
                           : umma_desc_noswz(smem_u32(smem + C::kSmemK), 128, kGroup);
  const uint64_t vd0 = SWZ ? umma_desc_sw128(smem_u32(smem + C::kSmemV), kPanelBytes, 1024)
                           : umma_desc_noswz(smem_u32(smem + C::kSmemV), kGroup, 128);
  uint32_t kt = 0, kitem = 0;
  uint32_t pcount[2] = {0, 0};
  for (int it = item0; it < item1; ++it) {
    const Item I(items, it, rG, TT);
    if (I.tiles == 0) continue;
    const int n = I.tiles;
    // S of stream i's step j
    auto qk = [&](int i, int j) -> bool {
      const int t = I.tile(i, j);
      const uint32_t st = (kt + t) % C::kStages;
      if (!mbar_wait(&bars[C::B_KFULL + st], ((kt + t) / C::kStages) & 1, abort)) return false;
      tc_fence_after();
      issue_qk<D, SWZ>(tmem + s_col(i), desc_at(qd0, SPLIT || I.split ? 0 : i * C::kTileBytes),
                       desc_at(kd0, st * C::kTileBytes), qk_desc);
      umma_commit(&bars[C::B_SFULL + i]);
      if (I.split || i == 1) {
        umma_commit(&bars[C::B_KEMPTY + st]);
        if (t == n - 1) umma_commit(&bars[C::B_QFREE]);
      }
      return true;
    };
    if (!mbar_wait(&bars[C::B_QFULL], kitem & 1, abort)) return;
    tc_fence_after();
    if (!qk(0, 0)) return;
    if (I.count(1) > 0 && !qk(1, 0)) return;
    for (int j = 0; j < I.count(0); ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // O of the previous item has been read (waited for in every item, so that
        // the barrier's phases are followed one by one)
        if (j == 0 && kitem > 0 && !mbar_wait(&bars[C::B_OFREE + i], (kitem - 1) & 1, abort)) return;
        if (j >= I.count(i)) continue;
        const int t = I.tile(i, j);
        const uint32_t st = (kt + t) % C::kStages;
        if (!mbar_wait(&bars[C::B_VFULL + st], ((kt + t) / C::kStages) & 1, abort)) return;
        if (MODE != kE4m3 && !mbar_wait(&bars[C::B_VREADY + st], ((kt + t) / C::kStages) & 1, abort)) return;
        const uint64_t vd = desc_at(vd0, st * C::kTileBytes);
        const uint32_t ts = tmem + s_col(i), to = tmem + o_col(i);
        if (!mbar_wait(&bars[C::B_PHALF + i], pcount[i] & 1, abort)) return;
        tc_fence_after();
        issue_pv<D, SWZ, 0, 4>(to, ts, vd, pv_desc, j > 0);
        if (!mbar_wait(&bars[C::B_PFULL + i], pcount[i] & 1, abort)) return;
        ++pcount[i];
        tc_fence_after();
        issue_pv<D, SWZ, 4, 8>(to, ts, vd, pv_desc, true);
        if (I.split || i == 1) umma_commit(&bars[C::B_VEMPTY + st]);
        if (j + 1 < I.count(i) && !qk(i, j + 1)) return;
      }
    }
    umma_commit(&bars[C::B_OFINAL + 0]);
    umma_commit(&bars[C::B_OFINAL + 1]);
    kt += n;
    ++kitem;
  }
}

// Zeroes the value rows that no row of the unit sees, and passes every value tile
// on to the MMA issuer (a barrier for each stage, so that no phase is skipped).
template <int D, int MODE, bool SPLIT>
__device__ void fixer(uint8_t* smem, uint64_t* bars, volatile int* abort, const int32_t* items, int item0,
                      int item1, float rG, int TT) {
  using C = Cfg<D, MODE, SPLIT>;
  const int lane = threadIdx.x & 31;
  uint32_t kt = 0;
  for (int it = item0; it < item1; ++it) {
    const Item I(items, it, rG, TT);
    for (int t = 0; t < I.tiles; ++t, ++kt) {
      const uint32_t st = kt % C::kStages;
      if (!warp_wait(&bars[C::B_VFULL + st], (kt / C::kStages) & 1, abort)) return;
      if (I.fix(t)) {
        uint8_t* v = smem + C::kSmemV + st * C::kTileBytes;
        const int k = I.key0 + t * kTileKeys, hi = I.hi_max(), lo = I.lo_min();
        for (int x = lane; x < 128 * (D / 8); x += 32) {
          const int r = x & 127, c = x >> 7;  // row, 16-byte chunk
          if (k + r >= hi || k + r < lo) {
            uint8_t* at = MODE == kRows ? v + (c >> 3) * kPanelBytes + r * 128 + (c & 7) * 16
                                        : v + (r >> 4) * (32 * D) + (((r >> 3) & 1) * (D / 8) + c) * 128 + (r & 7) * 16;
            *reinterpret_cast<uint4*>(at) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(&bars[C::B_VREADY + st]);
    }
  }
}

// 8-bit tiles from the landing buffers into the bf16 tiles of the products. A
// thread takes 16-byte chunks: 16 elements of one row.
template <int D, bool SPLIT>
__device__ void widener(uint8_t* smem, uint64_t* bars, volatile int* abort, const int32_t* items, int item0,
                        int item1, float rG, int TT) {
  using C = Cfg<D, kE4m3, SPLIT>;
  const int tid = threadIdx.x - 384, lane = threadIdx.x & 31;
  // a page is D chunks; this thread's chunk of a page: row group, chunk, row
  constexpr int kPagesPer = 128 / D;  // pages that the 128 threads take at once
  const int y = tid % D, g = y / (D / 2), c = (y / 8) % (D / 16), r = y % 8;
  const int row0 = tid / D * 16 + g * 8 + r;
  const int dst0 = tid / D * (32 * D) + (g * (D / 8) + 2 * c) * 128 + r * 16;
  uint32_t kt = 0;
  for (int it = item0; it < item1; ++it) {
    const Item I(items, it, rG, TT);
    const int hi = I.hi_max(), lo = I.lo_min();
    for (int t = 0; t < I.tiles; ++t, ++kt) {
      const uint32_t st = kt % C::kStages, use = kt / C::kStages;
      const int key = I.key0 + t * kTileKeys;
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t ls = kt % C::kLand;
        if (!warp_wait(&bars[C::B_LFULL + 2 * ls + kv], (kt / C::kLand) & 1, abort)) return;
        if (use > 0 && !warp_wait(&bars[(kv ? C::B_VEMPTY : C::B_KEMPTY) + st], (use - 1) & 1, abort)) return;
        const uint8_t* src = smem + C::kSmemLand + (2 * ls + kv) * C::kLandBytes + tid * 16;
        const uint8_t* scales = smem + C::kSmemScales + (2 * ls + kv) * 128 + row0;
        uint8_t* dst = smem + (kv ? C::kSmemV : C::kSmemK) + st * C::kTileBytes + dst0;
        const bool fix = kv == 1 && (key + kTileKeys > hi || key < lo);
#pragma unroll 2
        for (int x = 0; x < D / 16; ++x) {  // chunk tid + 128 x: kPagesPer pages further on
          const uint4 w = *reinterpret_cast<const uint4*>(src + x * 2048);
          const uint32_t byte = scales[x * kPagesPer * 16];
          // 2^(120 + e) as a bf16; the exponent field ends at 254, the rest of a
          // scale above 2^7 is a second factor
          uint32_t f0 = min(byte + 120u, 254u) << 7;
          if (byte == 0u) f0 = 0u;
          if (byte == 255u) f0 = 0x7fc0u;  // NaN
          if (fix) {
            const int k = key + row0 + x * kPagesPer * 16;
            if (k >= hi || k < lo) f0 = 0u;  // a value no row sees
          }
          f0 |= f0 << 16;
          uint32_t o[8];
          const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t b = __byte_perm(in[i], 0u, h ? 0x3424 : 0x1404);  // bytes into the high halves
              uint32_t v = (b & 0x80008000u) | ((b & 0x7f007f00u) >> 4);
              asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(f0));
              o[2 * i + h] = v;
            }
          }
          if (byte > 134u && byte < 255u) {
            uint32_t f1 = (byte + 120u - 254u + 127u) << 7;
            f1 |= f1 << 16;
#pragma unroll
            for (int i = 0; i < 8; ++i) asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(o[i]) : "r"(f1));
          }
          uint8_t* at = dst + x * kPagesPer * (32 * D);
          *reinterpret_cast<uint4*>(at) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(at + 128) = make_uint4(o[4], o[5], o[6], o[7]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          // the landing buffer last: its next tile is what lets any role go on, which then
          // finds the other barriers' phases of this tile counted
          mbar_arrive(&bars[C::B_WIDE + 2 * ls + kv]);
          mbar_arrive(&bars[(kv ? C::B_VFULL : C::B_KFULL) + st]);
          mbar_arrive(&bars[C::B_LEMPTY + 2 * ls + kv]);
        }
      }
    }
  }
}

// e4m3's NaN (all ones but the sign) is no number of the bits that the widener moves.
// These two warps, idle otherwise, look for it in the landed tiles and put NaN over what
// the widener has written in its place (in the widener's own loop the search cost 17%: 16
// blocks of 16 tokens 274 us against 235).
template <int D, bool SPLIT>
__device__ void nan_finder(uint8_t* smem, uint64_t* bars, volatile int* abort, const int32_t* items, int item0,
                           int item1, float rG, int TT) {
  using C = Cfg<D, kE4m3, SPLIT>;
  const int tid = threadIdx.x - kFixWarp * 32, lane = threadIdx.x & 31;
  constexpr int kChunks = 128 * D / 16 / 64;  // of a thread
  uint32_t kt = 0;
  for (int it = item0; it < item1; ++it) {
    const Item I(items, it, rG, TT);
    const int hi = I.hi_max(), lo = I.lo_min();
    for (int t = 0; t < I.tiles; ++t, ++kt) {
      const uint32_t st = kt % C::kStages, ls = kt % C::kLand;
      const int key = I.key0 + t * kTileKeys;
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv) {
        if (!warp_wait(&bars[C::B_LFULL + 2 * ls + kv], (kt / C::kLand) & 1, abort)) return;
        const uint8_t* src = smem + C::kSmemLand + (2 * ls + kv) * C::kLandBytes;
        uint32_t found = 0u;  // a byte's carry into its sign bit
#pragma unroll 4
        for (int x = 0; x < kChunks; ++x) {
          const uint4 w = *reinterpret_cast<const uint4*>(src + (x * 64 + tid) * 16);
          found |= (w.x ^ (w.x + 0x01010101u)) | (w.y ^ (w.y + 0x01010101u));
          found |= (w.z ^ (w.z + 0x01010101u)) | (w.w ^ (w.w + 0x01010101u));
        }
        if (__any_sync(0xffffffffu, (found & 0x80808080u) != 0u)) {
          if (!warp_wait(&bars[C::B_WIDE + 2 * ls + kv], (kt / C::kLand) & 1, abort)) return;
          uint8_t* dst = smem + (kv ? C::kSmemV : C::kSmemK) + st * C::kTileBytes;
          for (int x = 0; x < kChunks; ++x) {
            // page, row group, chunk and row of the 16 bytes (as in the widener)
            const int i = x * 64 + tid, y = i % D, g = y / (D / 2), c = (y / 8) % (D / 16), r = y % 8;
            const int k = key + i / D * 16 + g * 8 + r;
            if (kv == 1 && (k >= hi || k < lo)) continue;  // zeroed
            uint16_t* row = reinterpret_cast<uint16_t*>(dst + i / D * (32 * D) + (g * (D / 8) + 2 * c) * 128 + r * 16);
            for (int e = 0; e < 16; ++e)
              if ((src[i * 16 + e] & 0x7f) == 0x7f) row[e / 8 * 64 + e % 8] = 0x7fff;
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) {
          mbar_arrive(&bars[(kv ? C::B_VFULL : C::B_KFULL) + st]);
          mbar_arrive(&bars[C::B_LEMPTY + 2 * ls + kv]);  // last, as there
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
template <typename T, int D, int MODE, bool SPLIT>
__device__ void softmax_role(const AttnArgs& a, uint8_t* smem, uint64_t* bars, uint32_t tmem,
                             volatile int* abort, const int32_t* items, int item0,
                             int item1, int G, float rG, int TT) {
  using C = Cfg<D, MODE, SPLIT>;
  constexpr bool kTwoPass = MODE == kE4m3;
  const int i = threadIdx.x / 128, wq = (threadIdx.x / 32) & 3, lane = threadIdx.x & 31;
  const int row = wq * 32 + lane;
  const uint32_t lane_base = tmem + (static_cast<uint32_t>(wq * 32) << 16);
  const float sl2 = a.scale_log2;
  constexpr bool kF16 = std::is_same<T, __half>::value;
  constexpr float kLag = kF16 ? 4.f : 8.f, kTop = kF16 ? 11.f : 0.f;
  float2* join = reinterpret_cast<float2*>(smem + C::kSmemJoin);
  uint32_t scount = 0, kitem = 0;
  const int row_tok = row / G, row_g = row % G;
  // tokens of the warp's first and last row
  const int warp_tok0 = wq * 32 / G, warp_tok1 = min(wq * 32 + 31, TT * G - 1) / G;
  // a wait ran out of time: the warp does no more work, but goes through the
  // named barriers, which the other warps may be waiting at
  bool dead = false;
  for (int it = item0; it < item1; ++it) {
    const Item I(items, it, rG, TT);
    const int base = I.tokb + (I.split ? 0 : i * TT);  // first token of the tile, inside the request
    const int tok = base + row_tok;
    const int tok_end = I.tokb + (I.split ? I.ntok : min(I.ntok, (i + 1) * TT));
    const bool valid = row < TT * G && tok < tok_end;
    const int hq = I.head * G + row_g;
    const float sink = a.sinks && valid ? a.sinks[hq] : 0.f;
    const int hi = valid ? I.row_hi(tok) : 0, lo = valid ? I.row_lo(tok) : 0;
    // keys that every row, and that some row, of this warp sees
    const bool warp_any = wq * 32 < TT * G && base + warp_tok0 < tok_end;
    const int w0 = base + warp_tok0, w1 = min(base + warp_tok1, tok_end - 1);
    const int all_hi = warp_any ? I.row_hi(w0) : 0, any_hi = warp_any ? I.row_hi(w1) : 0;
    const int any_lo = I.row_lo(w0), all_lo = I.row_lo(w1);
    float m_run = -INFINITY, l_run = 0.f;
    const int steps = I.count(i);
    for (int j = 0; j < steps && !dead; ++j) {
      if (!warp_wait(&bars[C::B_SFULL + i], scount & 1, abort)) {
        dead = true;
        break;
      }
      ++scount;
      tc_fence_after();
      if (!warp_any) {  // rows that are not there: whatever S holds may be their P
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars[C::B_PHALF + i]);
          mbar_arrive(&bars[C::B_PFULL + i]);
        }
        continue;
      }
      const int key = I.key0 + I.tile(i, j) * kTileKeys;
      const bool edge = key + kTileKeys > all_hi || key < all_lo;
      // In a tile that not every row of the warp sees whole, chunks of 32 keys that
      // no row sees are skipped and those between are masked: key e is kept by a
      // minimum with (h - e) * inf, which is +inf below h and -inf above (h half an
      // integer), and likewise at the window's end -- two operations of the idle FMA
      // pipe for two keys, where comparing and selecting costs more operations of the
      // pipe that also takes the row maximum.
      const float h = static_cast<float>(hi - key) - 0.5f, l = static_cast<float>(lo - key) - 0.5f;
      auto skip = [&](int c) { return key + c * 32 >= any_hi || key + c * 32 + 32 <= any_lo; };
      auto bound = [](uint32_t* v, float first, float step) {  // element e against first + e step
        const uint64_t inf2 = f2_pack(INFINITY, INFINITY), two = f2_pack(2.f * step, 2.f * step);
        uint64_t x = f2_pack(first, first + step);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float t0, t1;
          f2_unpack(f2_mul(x, inf2), t0, t1);
          v[e] = __float_as_uint(fminf(__uint_as_float(v[e]), t0));
          v[e + 1] = __float_as_uint(fminf(__uint_as_float(v[e + 1]), t1));
          x = f2_add(x, two);
        }
      };
      auto cut_hi = [&](int c) { return key + c * 32 + 32 > all_hi; };
      auto cut_lo = [&](int c) { return key + c * 32 < all_lo; };
      auto mask = [&](int c, uint32_t* v) {
        if (cut_hi(c)) bound(v, h - c * 32, -1.f);
        if (cut_lo(c)) bound(v, c * 32 - l, 1.f);
      };
      float f = 1.f, neg_m = 0.f;
      bool early = true;
      // the row's maximum of this tile (raw) -> reference and rescaling factor
      auto new_max = [&](float (&mx)[8]) {
        mx[0] = fmax3(mx[0], mx[1], mx[2]);
        mx[3] = fmax3(mx[3], mx[4], mx[5]);
        mx[6] = fmaxf(mx[6], mx[7]);
        const float m_tile = fmax3(mx[0], mx[3], mx[6]) * sl2;
        if (j == 0) {
          m_run = m_tile;
        } else if (m_tile > m_run + kLag) {
          f = fast_exp2(m_run - m_tile);  // 0 while the row has seen no key
          m_run = m_tile;
        }
        neg_m = m_run == -INFINITY ? 0.f : kTop - m_run;
        // the first half of P is released early, unless a lane must rescale O first
        early = __all_sync(0xffffffffu, f == 1.f);
      };
      uint64_t acc2[4] = {0ull, 0ull, 0ull, 0ull};
      auto weights = [&](const uint32_t* v, uint32_t (&pk)[16], uint64_t sc2, uint64_t nm2) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), sc2, nm2);
          float x0, x1;
          f2_unpack(x2, x0, x1);
          const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
          acc2[e & 3] = f2_add(acc2[e & 3], f2_pack(p0, p1));
          pk[e] = pack2(p0, p1, T());
        }
      };
      auto store_p = [&](int c, const uint32_t (&pk)[16]) {
        tmem_st16(lane_base + s_col(i) + c * 16, pk);
        if (c == 1 && early) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars[C::B_PHALF + i]);
        }
      };
      auto max32 = [&](const uint32_t* v, float (&mx)[8]) {
#pragma unroll
        for (int e = 0; e < 32; e += 16) {
#pragma unroll
          for (int k = 0; k < 8; ++k) mx[k] = fmax3(mx[k], __uint_as_float(v[e + k]), __uint_as_float(v[e + 8 + k]));
        }
      };
      float mx[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) mx[e] = -INFINITY;
      if (kTwoPass || (edge && I.window)) {
        // 32 scores at a time, twice, so that chunks no row sees are skipped (a
        // window leaves many; 117 us against 137 with the masks below at six chunks
        // of about 850 tokens, window 128) and no more than 32 are in registers
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          if (edge && skip(c)) continue;
          uint32_t v[32];
          tmem_ld32_wait(lane_base + s_col(i) + c * 32, v);
          if (edge && (cut_hi(c) || cut_lo(c))) {  // masked once, for the second pass too
            mask(c, v);
            tmem_st32(lane_base + s_col(i) + c * 32, v);
          }
          max32(v, mx);
        }
        tmem_st_wait();
        new_max(mx);
        const uint64_t sc2 = f2_pack(sl2, sl2), nm2 = f2_pack(neg_m, neg_m);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
          if (edge && skip(c)) {
#pragma unroll
            for (int e = 0; e < 16; ++e) pk[e] = 0u;
          } else {
            uint32_t v[32];
            tmem_ld32_wait(lane_base + s_col(i) + c * 32, v);
            weights(v, pk, sc2, nm2);
          }
          store_p(c, pk);
        }
      } else if constexpr (!kTwoPass) {
        uint32_t s[128];
        tmem_ld128_wait(lane_base + s_col(i), s);
        if (edge) {
#pragma unroll
          for (int c = 0; c < 4; ++c) mask(c, s + c * 32);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) max32(s + c * 32, mx);
        new_max(mx);
        const uint64_t sc2 = f2_pack(sl2, sl2), nm2 = f2_pack(neg_m, neg_m);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
          weights(s + c * 32, pk, sc2, nm2);
          store_p(c, pk);
        }
      }
      if (!early) {
        // TMEM access is warp-collective: the whole warp rescales, lanes with f = 1
        // unchanged. O is complete up to the previous tile (its P V precedes this
        // tile's S in issue order)
        l_run *= f;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32_wait(lane_base + o_col(i) + c * 32, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st32(lane_base + o_col(i) + c * 32, o);
        }
      }
      float a0, a1, b0, b1, c0, c1, d0, d1;
      f2_unpack(acc2[0], a0, a1);
      f2_unpack(acc2[1], b0, b1);
      f2_unpack(acc2[2], c0, c1);
      f2_unpack(acc2[3], d0, d1);
      l_run += ((a0 + a1) + (b0 + b1)) + ((c0 + c1) + (d0 + d1));
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (!early) mbar_arrive(&bars[C::B_PHALF + i]);
        mbar_arrive(&bars[C::B_PFULL + i]);
      }
    }
    m_run -= kTop;  // what the weights are relative to
    // while the last products run: the row's factor, and the next item
    auto factor = [&](float m, float l, float& lse2) {
      float f = row_factor(m, l, lse2);
      if (a.sinks) f *= sink_factor(lse2, sink, a.sink_mode);
      return f;
    };
    float lse_own = 0.f, f_row = 0.f;
    if (valid) f_row = factor(m_run, l_run, lse_own);
    const Item& cur = I;
    if (cur.tiles > 0) {
      if (!dead && !warp_wait(&bars[C::B_OFINAL + i], kitem & 1, abort)) dead = true;
      tc_fence_after();
    }

    // ---- a split unit: stream 0 takes over stream 1's state ----
    float f_own = 1.f, f_other = 0.f;  // factors of this stream's O and of stream 1's
    float m = m_run, l = l_run;
    if (cur.split) {
      if (i == 1) {
        join[row] = make_float2(m_run, l_run);
        named_sync(3, 256);
        named_sync(3, 256);  // it is read
        if (cur.tiles > 0) ++kitem;
        continue;  // stream 0 reads O1 and frees it
      }
      named_sync(3, 256);
      const float2 o1 = join[row];
      named_sync(3, 256);
      m = fmaxf(m_run, o1.x);
      const float mr = m == -INFINITY ? 0.f : m;
      f_own = fast_exp2(m_run - mr);
      f_other = cur.count(1) > 0 ? fast_exp2(o1.x - mr) : 0.f;
      l = l_run * f_own + o1.y * f_other;
    }
    const bool has_other = cur.split && cur.count(1) > 0;
    // 32 columns of this row's (joined, unnormalised) O
    auto load_o = [&](int c, float (&o)[32]) {
      uint32_t r[32];
      if (cur.tiles == 0) {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0.f;
        return;
      }
      tmem_ld32_wait(lane_base + o_col(i) + c * 32, r);
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(r[e]) * f_own;
      if (has_other) {
        tmem_ld32_wait(lane_base + o_col(1) + c * 32, r);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = fmaf(__uint_as_float(r[e]), f_other, o[e]);
      }
    };
    auto free_o = [&] {
      if (cur.tiles == 0) return;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars[C::B_OFREE + i]);
        if (cur.split) mbar_arrive(&bars[C::B_OFREE + 1]);
      }
      ++kitem;
    };
    const int64_t gtok = static_cast<int64_t>(cur.tok0) + tok;
    // 32 columns of the warp's rows. A thread has its own row; four neighbours
    // exchange 16-byte pieces, so that a store covers 64 bytes of a row each four
    // lanes and touches 8 lines instead of 32.
    auto store_o = [&](int c, const float (&o)[32], float f, const int64_t (&at)[4]) {
      uint4 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e].x = pack2(o[8 * e + 0] * f, o[8 * e + 1] * f, T());
        v[e].y = pack2(o[8 * e + 2] * f, o[8 * e + 3] * f, T());
        v[e].z = pack2(o[8 * e + 4] * f, o[8 * e + 5] * f, T());
        v[e].w = pack2(o[8 * e + 6] * f, o[8 * e + 7] * f, T());
      }
      quad_swap(v[0], v[1], lane & 1, 1);
      quad_swap(v[2], v[3], lane & 1, 1);
      quad_swap(v[0], v[2], (lane >> 1) & 1, 2);
      quad_swap(v[1], v[3], (lane >> 1) & 1, 2);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (at[k] >= 0)
          *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at[k] + c * 32 + (lane & 3) * 8) = v[k];
    };
    if (cur.parts == 1) {
      if (cur.split && valid) f_row = factor(m, l, lse_own);
      int64_t at[4];  // where the quad's rows go, -1: not a row
      const int64_t own = valid ? gtok * a.o_st + hq * a.o_sh : -1;
#pragma unroll
      for (int k = 0; k < 4; ++k) at[k] = __shfl_sync(0xffffffffu, own, (lane & ~3) + k);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        load_o(c, o);
        store_o(c, o, f_row, at);
      }
      if (valid && a.lse) a.lse[gtok * a.lse_st + hq] = lse_own;
      free_o();
      continue;
    }
    // ---- a span of a unit: leave the state in its slot (join_kernel) ----
    float* own = a.slots + static_cast<int64_t>(cur.slot * 2 + i) * tile_slot_floats(D);
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      float o[32];
      load_o(c, o);
      if (valid) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          reinterpret_cast<float4*>(own)[(c * 8 + e) * 128 + row] =
              make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
      }
    }
    if (valid) {
      own[128 * D + row] = m;
      own[128 * D + 128 + row] = l;
    }
    free_o();
  }
}

template <typename T, int D, int MODE, bool SPLIT>
__global__ void __launch_bounds__(Cfg<D, MODE, SPLIT>::kThreads, 1)
    tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const AttnArgs a, const int rpb) {
  using C = Cfg<D, MODE, SPLIT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kSmemBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bars[C::B_QFULL], 1);
    mbar_init(&bars[C::B_QFREE], 1);
    for (int s = 0; s < C::kStages; ++s) {
      // e4m3: full when the widener's four warps have written the tile and the two
      // that look for NaN have looked at it
      mbar_init(&bars[C::B_KFULL + s], MODE == kE4m3 ? 6 : 1);
      mbar_init(&bars[C::B_VFULL + s], MODE == kE4m3 ? 6 : 1);
      mbar_init(&bars[C::B_KEMPTY + s], 1);
      mbar_init(&bars[C::B_VEMPTY + s], 1);
      mbar_init(&bars[C::B_VREADY + s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[C::B_SFULL + i], 1);
      mbar_init(&bars[C::B_PHALF + i], 4);
      mbar_init(&bars[C::B_PFULL + i], 4);
      mbar_init(&bars[C::B_OFINAL + i], 1);
      mbar_init(&bars[C::B_OFREE + i], 4);
    }
    for (int i = 0; i < 2 * C::kLand; ++i) {
      mbar_init(&bars[C::B_LFULL + i], 1);
      mbar_init(&bars[C::B_LEMPTY + i], 6);
      mbar_init(&bars[C::B_WIDE + i], 4);
    }
    *abort = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == kTmaWarp && lane == 0) {
    tma_prefetch_desc(&tm_q);
    if (MODE == kRows) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_wait();

  const int32_t* sec = a.plan + H_SECTION + kSectionInts;
  const int G = a.plan[H_GROUP];
  const int TT = 128 / G;
  const float rG = 1.f / G;
  const bool spare = static_cast<int>(blockIdx.x) >= sec[S_CTAS];  // of a fixed grid
  const int item0 = spare ? 0 : a.plan[sec[S_OFF_CTA] + blockIdx.x];
  const int item1 = spare ? 0 : a.plan[sec[S_OFF_CTA] + blockIdx.x + 1];
  const int32_t* items = a.plan + sec[S_OFF_ITEMS];

  if (warp >= 8) {
    if constexpr (MODE != kE4m3) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kSideRegs));
    if (warp == kTmaWarp) {
      producer<D, MODE, SPLIT>(&tm_q, &tm_k, &tm_v, a, smem, bars, abort, items, item0, item1, G, rG, TT, rpb);
      __syncwarp();
    } else if (warp == kMmaWarp) {
      if (elect_one()) mma_issuer<T, D, MODE, SPLIT>(smem, bars, tmem, abort, items, item0, item1, rG, TT);
      __syncwarp();
    } else if (MODE == kE4m3 && (warp == kFixWarp || warp == kFixWarp + 1)) {
      if constexpr (MODE == kE4m3) nan_finder<D, SPLIT>(smem, bars, abort, items, item0, item1, rG, TT);
      __syncwarp();
    } else if (warp == kFixWarp) {
      fixer<D, MODE, SPLIT>(smem, bars, abort, items, item0, item1, rG, TT);
      __syncwarp();
    } else if (warp >= 12) {
      if constexpr (MODE == kE4m3) widener<D, SPLIT>(smem, bars, abort, items, item0, item1, rG, TT);
      __syncwarp();
    }
  } else {
    if constexpr (MODE != kE4m3) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
    softmax_role<T, D, MODE, SPLIT>(a, smem, bars, tmem, abort, items, item0, item1, G, rG, TT);
  }

  tc_fence_before();
  __syncthreads();
  if (*abort) {  // let the copies and products in flight end (1 ms)
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 1000000ull) {
    }
    __syncthreads();
  }
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (threadIdx.x == 0 && *abort && a.status) atomicExch(a.status, 1);
}

template <typename T, int D, int MODE, bool SPLIT>
int launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const AttnArgs& a, int rpb,
           int ctas, cudaStream_t stream) {
  using C = Cfg<D, MODE, SPLIT>;
  static std::atomic<uint64_t> configured{0};  // bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !((configured.load() >> dev) & 1)) {
    cudaError_t e = cudaFuncSetAttribute(tiles_kernel<T, D, MODE, SPLIT>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess)
      return fail(D2SD_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
    if (dev < 64) configured.fetch_or(1ull << dev);
  }
  return launch_pdl(tiles_kernel<T, D, MODE, SPLIT>, dim3(ctas), dim3(C::kThreads), C::kSmemBytes, stream,
                    "tiles_kernel", tq, tk, tv, a, rpb);
}

}  // namespace

int encode_pages(CUtensorMap* tk, CUtensorMap* tv, const AttnArgs& a, int32_t dtype, int32_t head_dim,
                 int32_t num_kv_heads) {
  const CUtensorMapDataType type =
      dtype == D2SD_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t dims[4] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(a.g.page_size),
                            static_cast<uint64_t>(num_kv_heads), static_cast<uint64_t>(a.g.num_pages)};
  const uint64_t strides[3] = {static_cast<uint64_t>(a.g.stride_slot), static_cast<uint64_t>(a.g.stride_head),
                               static_cast<uint64_t>(a.g.stride_page)};
  const uint32_t box[4] = {64, 16, 1, 1};
  int rc = encode_tensor_map(tk, type, a.k_pool, 4, dims, strides, box, "k");
  return rc ? rc : encode_tensor_map(tv, type, a.v_pool, 4, dims, strides, box, "v");
}

int launch_tiles(const AttnArgs& a, int32_t dtype, int32_t head_dim, bool scaled, int64_t num_tokens,
                 int32_t num_qo_heads, int32_t num_kv_heads, bool split, int ctas, void* stream) {
  const int G = num_qo_heads / num_kv_heads;
  const CUtensorMapDataType type =
      dtype == D2SD_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tq, tk, tv;
  {
    const uint64_t dims[3] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(num_qo_heads),
                              static_cast<uint64_t>(num_tokens)};
    const uint64_t strides[2] = {static_cast<uint64_t>(a.q_sh) * 2, static_cast<uint64_t>(a.q_st) * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(G), static_cast<uint32_t>(128 / G)};
    int rc = encode_tensor_map(&tq, type, a.q, 3, dims, strides, box, "q");
    if (rc) return rc;
  }
  constexpr int rpb = 16;  // rows of a box: a span starts at any multiple of 16 keys
  tk = tv = tq;  // unused with UMMA pages
  if (!a.g.umma) {
    int rc = encode_pages(&tk, &tv, a, dtype, head_dim, num_kv_heads);
    if (rc) return rc;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto t, auto mode) {
    using T = decltype(t);
    constexpr int M = decltype(mode)::value;
    if (head_dim == 128)
      return split ? launch<T, 128, M, true>(tq, tk, tv, a, rpb, ctas, st)
                   : launch<T, 128, M, false>(tq, tk, tv, a, rpb, ctas, st);
    return split ? launch<T, 64, M, true>(tq, tk, tv, a, rpb, ctas, st)
                 : launch<T, 64, M, false>(tq, tk, tv, a, rpb, ctas, st);
  };
  using Native = std::integral_constant<int, kNative>;
  using Rows = std::integral_constant<int, kRows>;
  if (scaled) return go(__nv_bfloat16(), std::integral_constant<int, kE4m3>());
  if (dtype == D2SD_DTYPE_BF16) return a.g.umma ? go(__nv_bfloat16(), Native()) : go(__nv_bfloat16(), Rows());
  return a.g.umma ? go(__half(), Native()) : go(__half(), Rows());
}

}  // namespace paged
}  // namespace d2sd
