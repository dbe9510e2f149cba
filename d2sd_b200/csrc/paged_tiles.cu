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
//   warp 10      zeroes the value rows of a span's first and last tile that no row
//                sees: a weight of 0 would still turn a NaN there into NaN
//   warps 0-7    two softmax warpgroups, thread = row = TMEM lane
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
// only when the running maximum grows by more than 8 (weights stay below 2^8,
// inside f16). Weights are rounded to nearest for the second product; their fp32
// values go into the sum. Tiles that every row sees whole skip
// the mask; the others compare each key with the row's [lo, hi).
#include <atomic>
#include <string>

#include "paged_attn.cuh"

namespace d2sd {
namespace paged {
namespace {

enum { kNative = 0, kRows = 1, kE4m3 = 2 };

constexpr int kTmaWarp = 8, kMmaWarp = 9, kFixWarp = 10;
constexpr uint32_t kTmemCols = 512;
constexpr int kPanelBytes = 128 * 128;  // 128 rows x 64 16-bit values

template <int D, int MODE>
struct Cfg {
  static constexpr int kThreads = MODE == kE4m3 ? 512 : 384;
  // registers: with 384 threads the launch's 168 a thread are shared out between
  // the softmax warpgroups and the third (setmaxnreg); with 512 every thread has 128
  static constexpr int kLaunchRegs = 168, kSoftmaxRegs = 192, kSideRegs = 112;
  static_assert(256 * kSoftmaxRegs + 128 * kSideRegs <= 384 * kLaunchRegs,
                "register split above the launch's registers");
  static constexpr int kPanels = D / 64;
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr int kStages = D == 128 ? 2 : 4;  // of K and of V
  static constexpr int kSmemQ = 0;
  static constexpr int kSmemK = kSmemQ + 2 * kTileBytes;
  static constexpr int kSmemV = kSmemK + kStages * kTileBytes;
  static constexpr int kSmemLand = kSmemV + kStages * kTileBytes;  // 8-bit K, V tiles, their scales
  static constexpr int kLandBytes = 128 * D;
  static constexpr int kSmemJoin = kSmemLand + (MODE == kE4m3 ? 2 * kLandBytes + 256 : 0);
  static constexpr int kSmemBar = kSmemJoin + 128 * 8;  // [128] (m, l) of stream 1
  static constexpr int B_QFULL = 0, B_QFREE = 1, B_KFULL = 2, B_VFULL = B_KFULL + kStages,
                       B_KEMPTY = B_VFULL + kStages, B_VEMPTY = B_KEMPTY + kStages,
                       B_SFULL = B_VEMPTY + kStages, B_PHALF = B_SFULL + 2, B_PFULL = B_PHALF + 2,
                       B_OFINAL = B_PFULL + 2, B_OFREE = B_OFINAL + 2, B_VREADY = B_OFREE + 2,
                       B_LFULL = B_VREADY + kStages, B_LEMPTY = B_LFULL + 2, kNumBars = B_LEMPTY + 2;
  static constexpr int kSmemBytes = kSmemBar + kNumBars * 8 + 32 + 1024;  // + alignment slack
  static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");
};

__device__ __forceinline__ float fmin3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
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

// What every role derives from an item.
struct Item {
  int head, tok0, tokb, ntok, key0, key1, pos0, window, kv_len, parts, slot, first_slot, ticket;
  int64_t page_off;
  int tiles;
  bool split;  // both streams on the same q tile, every other key tile
  __device__ __forceinline__ Item(const int32_t* I, int G, int TT) {
    head = I[P_HEAD], tok0 = I[P_TOK0], key0 = I[P_KEY0], key1 = I[P_KEY1], pos0 = I[P_POS0];
    window = I[P_WINDOW], kv_len = I[P_KV_LEN], parts = I[P_PARTS], slot = I[P_SLOT];
    first_slot = I[P_FIRST_SLOT], ticket = I[P_TICKET], page_off = I[P_PAGE_OFF];
    tokb = I[P_ROW0] / G;        // first token of the unit, inside the request
    ntok = I[P_NROWS] / G;       // tokens of the unit
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
template <int D, int MODE>
__device__ void producer(const CUtensorMap* tm_q, const CUtensorMap* tm_k, const CUtensorMap* tm_v,
                         const AttnArgs& a, uint8_t* smem, uint64_t* bars, volatile int* abort,
                         const int32_t* items, int item0, int item1, int G, int TT, int rpb) {
  using C = Cfg<D, MODE>;
  const int lane = threadIdx.x & 31;
  const int boxes = kTileKeys / rpb;  // copies of a K or V tile (<= 8 ... 16)
  uint32_t kt = 0, kitem = 0;
  bool alive = true;
  for (int it = item0; it < item1 && alive; ++it) {
    const Item I(items + it * kItemInts, G, TT);
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
        if (MODE == kE4m3) {  // one landing buffer each
          full = &bars[C::B_LFULL + kv];
          if (lane == 0 && kt > 0) ok = mbar_wait(&bars[C::B_LEMPTY + kv], (kt - 1) & 1, abort);
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
          uint8_t* dst = MODE == kE4m3 ? smem + C::kSmemLand + kv * C::kLandBytes
                                       : smem + (kv ? C::kSmemV : C::kSmemK) + st * C::kTileBytes;
          if (lane == 0) mbar_arrive_expect_tx(full, 8 * (kBlock + (MODE == kE4m3 ? 16 : 0)));
          __syncwarp();
          if (lane < 8) {
            const int64_t p = page;
            bulk_load(dst + lane * kBlock, (kv ? a.v_pool : a.k_pool) + p * a.g.stride_page + I.head * a.g.stride_head,
                      kBlock, full);
            if (MODE == kE4m3)
              bulk_load(smem + C::kSmemLand + 2 * C::kLandBytes + kv * 128 + lane * 16,
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

template <typename T, int D, int MODE>
__device__ void mma_issuer(uint8_t* smem, uint64_t* bars, uint32_t tmem, volatile int* abort,
                           const int32_t* items, int item0, int item1, int G, int TT) {
  using C = Cfg<D, MODE>;
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
    const Item I(items + it * kItemInts, G, TT);
    if (I.tiles == 0) continue;
    const int n = I.tiles;
    // S of stream i's step j
    auto qk = [&](int i, int j) -> bool {
      const int t = I.tile(i, j);
      const uint32_t st = (kt + t) % C::kStages;
      if (!mbar_wait(&bars[C::B_KFULL + st], ((kt + t) / C::kStages) & 1, abort)) return false;
      tc_fence_after();
      issue_qk<D, SWZ>(tmem + s_col(i), desc_at(qd0, I.split ? 0 : i * C::kTileBytes),
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
template <int D, int MODE>
__device__ void fixer(uint8_t* smem, uint64_t* bars, volatile int* abort, const int32_t* items, int item0,
                      int item1, int G, int TT) {
  using C = Cfg<D, MODE>;
  const int lane = threadIdx.x & 31;
  uint32_t kt = 0;
  for (int it = item0; it < item1; ++it) {
    const Item I(items + it * kItemInts, G, TT);
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
template <int D>
__device__ void widener(uint8_t* smem, uint64_t* bars, volatile int* abort, const int32_t* items, int item0,
                        int item1, int G, int TT) {
  using C = Cfg<D, kE4m3>;
  const int tid = threadIdx.x - 384, lane = threadIdx.x & 31;
  uint32_t kt = 0;
  for (int it = item0; it < item1; ++it) {
    const Item I(items + it * kItemInts, G, TT);
    const int hi = I.hi_max(), lo = I.lo_min();
    for (int t = 0; t < I.tiles; ++t, ++kt) {
      const uint32_t st = kt % C::kStages, use = kt / C::kStages;
      const int key = I.key0 + t * kTileKeys;
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv) {
        if (!warp_wait(&bars[C::B_LFULL + kv], kt & 1, abort)) return;
        if (use > 0 && !warp_wait(&bars[(kv ? C::B_VEMPTY : C::B_KEMPTY) + st], (use - 1) & 1, abort)) return;
        const uint8_t* src = smem + C::kSmemLand + kv * C::kLandBytes;
        const uint8_t* scales = smem + C::kSmemLand + 2 * C::kLandBytes + kv * 128;
        uint8_t* dst = smem + (kv ? C::kSmemV : C::kSmemK) + st * C::kTileBytes;
#pragma unroll 4
        for (int x = tid; x < 128 * (D / 16); x += 128) {
          const int page = x / D, y = x % D;  // D chunks of a 16-row page
          const int g = y / (D / 2), c = (y / 8) % (D / 16), r = y % 8;
          const int row = page * 16 + g * 8 + r;
          const uint4 w = *reinterpret_cast<const uint4*>(src + x * 16);
          // 2^(120 + e) as bf16, in two factors where it is above 2^127
          const int byte = scales[row];
          int e0 = byte == 0 ? 0 : byte + 120, e1 = 127;  // exponent fields
          if (e0 > 254) e1 = e0 - 254 + 127, e0 = 254;
          uint32_t f0 = static_cast<uint32_t>(e0) << 7, f1 = static_cast<uint32_t>(e1) << 7;
          if (byte == 255) f0 = 0x7fc0u;                                     // NaN
          if (kv == 1 && (key + row >= hi || key + row < lo)) f0 = 0u;       // seen by no row
          f0 |= f0 << 16;
          f1 |= f1 << 16;
          uint32_t o[8];
          const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t b = __byte_perm(in[i], 0u, h ? 0x3424 : 0x1404);  // bytes into the high halves
              uint32_t v = (b & 0x80008000u) | ((b & 0x7f007f00u) >> 4);
              asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(f0));
              if (e1 != 127) asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(f1));
              o[2 * i + h] = v;
            }
          }
          uint8_t* at = dst + page * (32 * D) + (g * (D / 8) + 2 * c) * 128 + r * 16;
          *reinterpret_cast<uint4*>(at) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(at + 128) = make_uint4(o[4], o[5], o[6], o[7]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars[C::B_LEMPTY + kv]);
          mbar_arrive(&bars[(kv ? C::B_VFULL : C::B_KFULL) + st]);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
template <typename T, int D, int MODE>
__device__ void softmax_role(const AttnArgs& a, uint8_t* smem, uint64_t* bars, uint32_t tmem,
                             volatile int* abort, volatile int* last_flag, const int32_t* items, int item0,
                             int item1, int G, int TT) {
  using C = Cfg<D, MODE>;
  constexpr bool kTwoPass = MODE == kE4m3;
  const int i = threadIdx.x / 128, wq = (threadIdx.x / 32) & 3, lane = threadIdx.x & 31;
  const int row = wq * 32 + lane;
  const uint32_t lane_base = tmem + (static_cast<uint32_t>(wq * 32) << 16);
  const float sl2 = a.scale_log2;
  float2* join = reinterpret_cast<float2*>(smem + C::kSmemJoin);
  uint32_t scount = 0, kitem = 0;
  const int row_tok = row / G, row_g = row % G;
  // a wait ran out of time: the warp does no more work, but goes through the
  // named barriers, which the other warps may be waiting at
  bool dead = false;
  for (int it = item0; it < item1; ++it) {
    const Item I(items + it * kItemInts, G, TT);
    const int tok = I.tokb + (I.split ? 0 : i * TT) + row_tok;  // inside the request
    const int tok_end = I.tokb + (I.split ? I.ntok : min(I.ntok, (i + 1) * TT));
    const bool valid = row < TT * G && tok < tok_end;
    const int hq = I.head * G + row_g;
    const float sink = a.sinks && valid ? a.sinks[hq] : 0.f;
    const int hi = valid ? I.row_hi(tok) : 0, lo = valid ? I.row_lo(tok) : 0;
    // keys every valid row of this tile sees
    const int first_tok = I.tokb + (I.split ? 0 : i * TT);
    const int hi_all = I.row_hi(first_tok), lo_all = I.row_lo(tok_end - 1);
    float m_run = -INFINITY, l_run = 0.f;
    const int steps = I.count(i);
    for (int j = 0; j < steps && !dead; ++j) {
      if (!warp_wait(&bars[C::B_SFULL + i], scount & 1, abort)) {
        dead = true;
        break;
      }
      ++scount;
      tc_fence_after();
      const int key = I.key0 + I.tile(i, j) * kTileKeys;
      const bool edge = key + kTileKeys > hi_all || key < lo_all;
      // The scores of 32 keys, those the row does not see at -inf: key e is kept by
      // a minimum with (h - e) * inf, which is +inf below h and -inf above (h half
      // an integer), and likewise for the window's end -- two multiplications on
      // the idle FMA pipe and one three-way minimum, where comparing and selecting
      // costs three operations of the pipe that also takes the row maximum. Two
      // passes over TMEM where there are no registers for all 128 keys.
      const float h = static_cast<float>(hi - key) - 0.5f, l = static_cast<float>(lo - key) - 0.5f;
      uint32_t s[kTwoPass ? 32 : 128];
      auto mask = [&](int c, uint32_t* v) {
        const float hc = h - c * 32, lc = c * 32 - l;
        if (I.window) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            v[e] = __float_as_uint(fmin3(__uint_as_float(v[e]), (hc - e) * INFINITY, (lc + e) * INFINITY));
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            v[e] = __float_as_uint(fminf(__uint_as_float(v[e]), (hc - e) * INFINITY));
        }
      };
      float mx[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) mx[e] = -INFINITY;
      if constexpr (!kTwoPass) {
        tmem_ld128_wait(lane_base + s_col(i), s);
        if (edge) {
#pragma unroll
          for (int c = 0; c < 4; ++c) mask(c, s + c * 32);
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t* v = kTwoPass ? s : s + c * 32;
        if constexpr (kTwoPass) {
          tmem_ld32_wait(lane_base + s_col(i) + c * 32, s);
          if (edge) mask(c, s);
        }
#pragma unroll
        for (int e = 0; e < 32; e += 16) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mx[k] = fmax3(mx[k], __uint_as_float(v[e + k]), __uint_as_float(v[e + 8 + k]));
        }
      }
      mx[0] = fmax3(mx[0], mx[1], mx[2]);
      mx[3] = fmax3(mx[3], mx[4], mx[5]);
      mx[6] = fmaxf(mx[6], mx[7]);
      const float m_tile = fmax3(mx[0], mx[3], mx[6]) * sl2;
      float f = 1.f;
      if (j == 0) {
        m_run = m_tile;
      } else if (m_tile > m_run + 8.f) {
        f = fast_exp2(m_run - m_tile);  // 0 while the row has seen no key
        m_run = m_tile;
      }
      const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
      // the first half of P is released early, unless a lane must rescale O first
      const bool early = __all_sync(0xffffffffu, f == 1.f);
      const uint64_t sc2 = f2_pack(sl2, sl2), nm2 = f2_pack(neg_m, neg_m);
      uint64_t acc2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
        const uint32_t* v = kTwoPass ? s : s + c * 32;
        if constexpr (kTwoPass) {
          tmem_ld32_wait(lane_base + s_col(i) + c * 32, s);
          if (edge) mask(c, s);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), sc2, nm2);
          float x0, x1;
          f2_unpack(x2, x0, x1);
          const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
          acc2[e & 3] = f2_add(acc2[e & 3], f2_pack(p0, p1));
          pk[e] = pack2(p0, p1, T());
        }
        tmem_st16(lane_base + s_col(i) + c * 16, pk);
        if (c == 1 && early) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars[C::B_PHALF + i]);
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
    if (I.tiles > 0) {
      if (!dead && !warp_wait(&bars[C::B_OFINAL + i], kitem & 1, abort)) dead = true;
      tc_fence_after();
    }

    // ---- a split unit: stream 0 takes over stream 1's state ----
    float f_own = 1.f, f_other = 0.f;  // factors of this stream's O and of stream 1's
    float m = m_run, l = l_run;
    if (I.split) {
      if (i == 1) {
        join[row] = make_float2(m_run, l_run);
        named_sync(3, 256);
        named_sync(3, 256);  // it is read
        if (I.tiles > 0) ++kitem;
        continue;  // stream 0 reads O1 and frees it
      }
      named_sync(3, 256);
      const float2 o1 = join[row];
      named_sync(3, 256);
      m = fmaxf(m_run, o1.x);
      const float mr = m == -INFINITY ? 0.f : m;
      f_own = fast_exp2(m_run - mr);
      f_other = I.count(1) > 0 ? fast_exp2(o1.x - mr) : 0.f;
      l = l_run * f_own + o1.y * f_other;
    }
    const bool has_other = I.split && I.count(1) > 0;
    // 32 columns of this row's (joined, unnormalised) O
    auto load_o = [&](int c, float (&o)[32]) {
      uint32_t r[32];
      if (I.tiles == 0) {
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
      if (I.tiles == 0) return;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars[C::B_OFREE + i]);
        if (I.split) mbar_arrive(&bars[C::B_OFREE + 1]);
      }
      ++kitem;
    };
    const int64_t gtok = static_cast<int64_t>(I.tok0) + tok;
    auto factor = [&](float m, float l, float& lse2) {
      lse2 = l > 0.f ? m + log2f(l) : (l == 0.f ? -INFINITY : l);
      float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      if (a.sinks) f *= sink_factor(lse2, sink, a.sink_mode);
      return f;
    };
    auto store_o = [&](int c, const float (&o)[32], float f) {
      T* op = static_cast<T*>(a.out) + gtok * a.o_st + hq * a.o_sh + c * 32;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint4 v;
        v.x = pack2(o[8 * e + 0] * f, o[8 * e + 1] * f, T());
        v.y = pack2(o[8 * e + 2] * f, o[8 * e + 3] * f, T());
        v.z = pack2(o[8 * e + 4] * f, o[8 * e + 5] * f, T());
        v.w = pack2(o[8 * e + 6] * f, o[8 * e + 7] * f, T());
        *reinterpret_cast<uint4*>(op + e * 8) = v;
      }
    };
    if (I.parts == 1) {
      float lse2 = 0.f, f = 0.f;
      if (valid) f = factor(m, l, lse2);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        load_o(c, o);
        if (valid) store_o(c, o, f);
      }
      if (valid && a.lse) a.lse[gtok * a.lse_st + hq] = lse2;
      free_o();
      continue;
    }
    // ---- a span of a unit: leave the state in its slot; the last span joins ----
    // slot: [D / 4][128 rows] of four columns, then m and l of the rows
    constexpr int kSlot = 128 * (D + 2);
    const int per = 2;  // slots of an item: one for each q tile
    float* own = a.slots + static_cast<int64_t>(I.slot * per + i) * kSlot;
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
    named_sync(1 + i, 128);
    if (row == 0)
      last_flag[i] = atom_add_acq_rel_gpu(&a.tickets[I.ticket * 2 + i], 1u) == static_cast<uint32_t>(I.parts - 1);
    named_sync(1 + i, 128);
    const bool last = last_flag[i] != 0;
    named_sync(1 + i, 128);  // the flag is read before the next item writes it
    if (!last) continue;
    if (row == 0) a.tickets[I.ticket * 2 + i] = 0;
    if (!valid) continue;
    const float* s0 = a.slots + static_cast<int64_t>(I.first_slot * per + i) * kSlot;
    const int64_t step = static_cast<int64_t>(per) * kSlot;
    float M = -INFINITY, L = 0.f;
    for (int p = 0; p < I.parts; ++p) M = fmaxf(M, __ldcg(s0 + p * step + 128 * D + row));
    const float Mr = M == -INFINITY ? 0.f : M;
    for (int p = 0; p < I.parts; ++p)
      L += __ldcg(s0 + p * step + 128 * D + 128 + row) * fast_exp2(__ldcg(s0 + p * step + 128 * D + row) - Mr);
    float lse2;
    const float f = factor(M, L, lse2);
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      float o[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = 0.f;
#pragma unroll 1
      for (int p = 0; p < I.parts; ++p) {
        const float w = fast_exp2(__ldcg(s0 + p * step + 128 * D + row) - Mr);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(s0 + p * step) + (c * 8 + e) * 128 + row);
          o[4 * e] = fmaf(v.x, w, o[4 * e]);
          o[4 * e + 1] = fmaf(v.y, w, o[4 * e + 1]);
          o[4 * e + 2] = fmaf(v.z, w, o[4 * e + 2]);
          o[4 * e + 3] = fmaf(v.w, w, o[4 * e + 3]);
        }
      }
      store_o(c, o, f);
    }
    if (a.lse) a.lse[gtok * a.lse_st + hq] = lse2;
  }
}

template <typename T, int D, int MODE>
__global__ void __launch_bounds__(Cfg<D, MODE>::kThreads, 1)
    tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const AttnArgs a, const int rpb) {
  using C = Cfg<D, MODE>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kSmemBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* last_flag = abort + 1;  // one for each stream
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bars[C::B_QFULL], 1);
    mbar_init(&bars[C::B_QFREE], 1);
    for (int s = 0; s < C::kStages; ++s) {
      // e4m3: full when the widener's four warps have written the tile
      mbar_init(&bars[C::B_KFULL + s], MODE == kE4m3 ? 4 : 1);
      mbar_init(&bars[C::B_VFULL + s], MODE == kE4m3 ? 4 : 1);
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
      mbar_init(&bars[C::B_LFULL + i], 1);
      mbar_init(&bars[C::B_LEMPTY + i], 4);
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
  const bool spare = static_cast<int>(blockIdx.x) >= sec[S_CTAS];  // of a fixed grid
  const int item0 = spare ? 0 : a.plan[sec[S_OFF_CTA] + blockIdx.x];
  const int item1 = spare ? 0 : a.plan[sec[S_OFF_CTA] + blockIdx.x + 1];
  const int32_t* items = a.plan + sec[S_OFF_ITEMS];

  if (warp >= 8) {
    if constexpr (MODE != kE4m3) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kSideRegs));
    if (warp == kTmaWarp) {
      producer<D, MODE>(&tm_q, &tm_k, &tm_v, a, smem, bars, abort, items, item0, item1, G, TT, rpb);
      __syncwarp();
    } else if (warp == kMmaWarp) {
      if (elect_one()) mma_issuer<T, D, MODE>(smem, bars, tmem, abort, items, item0, item1, G, TT);
      __syncwarp();
    } else if (warp == kFixWarp && MODE != kE4m3) {
      fixer<D, MODE>(smem, bars, abort, items, item0, item1, G, TT);
      __syncwarp();
    } else if (warp >= 12) {
      if constexpr (MODE == kE4m3) widener<D>(smem, bars, abort, items, item0, item1, G, TT);
      __syncwarp();
    }
  } else {
    if constexpr (MODE != kE4m3) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
    softmax_role<T, D, MODE>(a, smem, bars, tmem, abort, last_flag, items, item0, item1, G, TT);
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

template <typename T, int D, int MODE>
int launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const AttnArgs& a, int rpb,
           int ctas, cudaStream_t stream) {
  using C = Cfg<D, MODE>;
  static std::atomic<uint64_t> configured{0};  // bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !((configured.load() >> dev) & 1)) {
    cudaError_t e = cudaFuncSetAttribute(tiles_kernel<T, D, MODE>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess)
      return fail(D2SD_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
    if (dev < 64) configured.fetch_or(1ull << dev);
  }
  return launch_pdl(tiles_kernel<T, D, MODE>, dim3(ctas), dim3(C::kThreads), C::kSmemBytes, stream,
                    "tiles_kernel", tq, tk, tv, a, rpb);
}

}  // namespace

int launch_tiles(const AttnArgs& a, int32_t dtype, int32_t head_dim, bool scaled, int64_t num_tokens,
                 int32_t num_qo_heads, int32_t num_kv_heads, int ctas, void* stream) {
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
  int rpb = 16;
  tk = tv = tq;  // unused with UMMA pages
  if (!a.g.umma) {
    // the largest power of two up to 128 that divides the page: boxes of a tile
    // are whole and lie in one page
    while (rpb < 128 && a.g.page_size % (2 * rpb) == 0) rpb *= 2;
    const uint64_t dims[4] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(a.g.page_size),
                              static_cast<uint64_t>(num_kv_heads), static_cast<uint64_t>(a.g.num_pages)};
    const uint64_t strides[3] = {static_cast<uint64_t>(a.g.stride_slot), static_cast<uint64_t>(a.g.stride_head),
                                 static_cast<uint64_t>(a.g.stride_page)};
    const uint32_t box[4] = {64, static_cast<uint32_t>(rpb), 1, 1};
    int rc = encode_tensor_map(&tk, type, a.k_pool, 4, dims, strides, box, "k");
    if (rc) return rc;
    rc = encode_tensor_map(&tv, type, a.v_pool, 4, dims, strides, box, "v");
    if (rc) return rc;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool d128 = head_dim == 128;
  if (scaled) return d128 ? launch<__nv_bfloat16, 128, kE4m3>(tq, tk, tv, a, rpb, ctas, st)
                          : launch<__nv_bfloat16, 64, kE4m3>(tq, tk, tv, a, rpb, ctas, st);
  if (dtype == D2SD_DTYPE_BF16) {
    if (a.g.umma) return d128 ? launch<__nv_bfloat16, 128, kNative>(tq, tk, tv, a, rpb, ctas, st)
                              : launch<__nv_bfloat16, 64, kNative>(tq, tk, tv, a, rpb, ctas, st);
    return d128 ? launch<__nv_bfloat16, 128, kRows>(tq, tk, tv, a, rpb, ctas, st)
                : launch<__nv_bfloat16, 64, kRows>(tq, tk, tv, a, rpb, ctas, st);
  }
  if (a.g.umma) return d128 ? launch<__half, 128, kNative>(tq, tk, tv, a, rpb, ctas, st)
                            : launch<__half, 64, kNative>(tq, tk, tv, a, rpb, ctas, st);
  return d128 ? launch<__half, 128, kRows>(tq, tk, tv, a, rpb, ctas, st)
              : launch<__half, 64, kRows>(tq, tk, tv, a, rpb, ctas, st);
}

}  // namespace paged
}  // namespace d2sd
