// Attention of a ragged batch's new tokens over the paged cache (causal, window,
// sinks; 16-bit and e4m3 pages), for few rows per kv head: single tokens and
// drafted blocks.
//
// Row (token, g) of a kv head sees the keys j of its request with
// pos - window < j <= pos. With s_j = scale * log2e * (q . k_j):
//   m = max s_j, l = sum 2^(s_j - m), o = sum 2^(s_j - m) v_j / l, lse2 = m + log2 l
// in one pass over the keys (running maximum and sum). A row without a key gets
// o = 0 and lse2 = -inf.
//
// rows_kernel: a CTA takes up to 16 query rows of one kv head against a span of keys
// (paged_plan.h); its warps take the span's 16-key pages in turn, each with a ring of
// pages of its own in shared memory, so the loop has no CTA barrier and 190 KB of loads
// are in flight per SM -- the bound is HBM. The products are m16n8k16 matrix
// instructions: one 16-row tile is all the rows there are, and a 128-row tensor-core
// tile would be mostly padding. A page is stored as 8-row x 16-byte core matrices,
// exactly what ldmatrix fetches, without bank conflicts and without a swizzle; pages of
// plain rows are fetched as TMA boxes with a 128-byte swizzle, which serves ldmatrix as
// well. At the end the warps' states are joined in shared memory; a unit of several spans
// is joined inside its cluster of CTAs, or by join_kernel.
// Measured (32 / 8 heads of 128, bf16; of 6.54 TB/s of a plain copy): 64 requests of 512
// to 8191 keys, one token each, 1133 MB, 187 us = 0.92; over e4m3 pages, 571 MB, 113 us =
// 0.77 (instruction issue and the chain of one page share the rest); one request of 1000
// keys 8.3 us on the GPU, the latency of one launch (a call from Python is 12.7 us, its
// host time).
//
// e4m3 pages: their values are widened to f16 in registers (one conversion for two,
// exact) and both products are f16. A 16-byte row of a core matrix holds 16 elements
// of d; ldmatrix hands a lane four neighbouring ones, and since the order of the
// summed index is free, q's fragment takes the same four (K); for V the lane's four
// bytes are two keys by two neighbouring columns. f16's range is met by powers of
// two, which cost no precision: q's rows are scaled to 2^14 .. 2^15, and with e_j
// the exponent of value row j the weights are
//   w_j = 2^(s_j - m) 2^(e_j), m the running maximum of s_j + max(e_j, -60),
// at most 1 whatever the rows' sizes are, and the sum takes 2^(s_j - m) <= 2^60 (a
// value row under 2^-60 is below what f16 weights resolve). The key's scale
// multiplies the score in fp32.
// Weights are rounded to 16 bits for the second product: bf16 2^-8 relative, f16
// 2^-11. An f16 below 2^-14 is subnormal, so f16 weights are taken 2^15 times as large
// (and the state is taken back): relative down to 2^-29 of the row's largest, and off
// by at most 2^-40 of it below that (fp32's own end, 2^-126, is met before that only
// where value rows are above 2^108: with e = 119 at 2^-22 of the largest). Maximum, sum
// and output stay in fp32.
#include <atomic>
#include <string>
#include <type_traits>

#include "paged_attn.cuh"

namespace d2sd {
namespace {

using namespace paged;

template <int D, int ELEM>
struct RowsCfg {
  // Four small CTAs share an SM, so that one's start and end (an item's entry, its q
  // and its first pages come one after another, about 5 us, and then the join) pass
  // under the others' loads (one CTA of 8 warps per SM: 200 requests of about 1000 keys
  // 130 us, now 77). 8-bit pages take half of the bytes and more instructions: twice the
  // warps, with q's fragments in shared memory (unless R8) so that 128 registers suffice.
  static constexpr int kWarps = ELEM == 1 ? 4 : 2;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kPageBytes = 16 * D * ELEM;        // one of K, V
  static constexpr int kStageBytes = 2 * kPageBytes + (ELEM == 1 ? 32 : 0);  // + 16 + 16 scale bytes
  static constexpr int kRing = ELEM == 1 ? 12416 : 24576;  // bytes of a warp's ring
  static constexpr int kStages = (kRing / kStageBytes) < 8 ? (kRing / kStageBytes) : 8;
  static constexpr int kState = 16 * D * 4;               // a warp's O, over its ring at the end
  static constexpr int kSmemMl = kWarps * kRing;          // [warps][16] m, then l
  static constexpr int kSmemQ = kSmemMl + 2 * kWarps * 16 * 4;  // [D / 16][32 lanes][16 bytes] (8-bit)
  static constexpr int kSmemBars = kSmemQ + (ELEM == 1 ? 16 * D * 2 : 0);
  static constexpr int kSmemFlags = kSmemBars + kWarps * 8 * 8;
  static constexpr int kSmemBytes = kSmemFlags + 16 + 1024;
  static_assert(kState + 128 <= kRing, "the state fits the ring");
  static_assert(kRowsCtas * (kSmemBytes + 1024) <= 227 * 1024 + 1024, "the CTAs of an SM");
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                 uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 2^e of a scale byte (a row marked NaN, 255, here 2^128, has NaN values too, so the
// product is NaN), and e from -60 on, the weights' reference.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float exponent_of(uint32_t byte) {
  return __uint_as_float(0x4b000000u | max(byte, 67u)) - (8388608.f + 127.f);
}

// The four e4m3 values of x as two pairs of f16 (bytes 0 and 1, bytes 2 and 3).
__device__ __forceinline__ void e4m3x4_f16(uint32_t x, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(x));
}

// The 8 x 8 matrix of 16-bit values of the warp (lane: row lane / 4, two columns), transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Byte offset of (row, 16-byte chunk) of a page in shared memory: core matrices, or
// (rows fetched as TMA boxes) 128-byte-swizzled panels of 64 values. ldmatrix reads
// eight rows of a chunk without bank conflicts in both.
template <int CHUNKS, bool UMMA>
__device__ __forceinline__ uint32_t page_at(int row, int chunk) {
  return UMMA ? static_cast<uint32_t>(((row >> 3) * CHUNKS + chunk) * 128 + (row & 7) * 16)
              : static_cast<uint32_t>((chunk >> 3) * 2048 + row * 128 + (((chunk ^ row) & 7) << 4));
}

// Shared memory of the cluster's CTA `rank` at this CTA's address, and the barrier of
// all its threads.
__device__ __forceinline__ uint32_t peer_addr(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float peer_float(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 peer_float4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Zeroes rows [r0, r1) of a page in shared memory (the whole warp).
template <int D, int ELEM, bool UMMA>
__device__ __forceinline__ void zero_rows(uint8_t* page, int r0, int r1) {
  constexpr int C = D * ELEM / 16;
  const int lane = threadIdx.x & 31;
  for (int i = lane; i < 16 * C; i += 32) {
    const int r = i & 15, c = i >> 4;
    if (r >= r0 && r < r1) *reinterpret_cast<uint4*>(page + page_at<C, UMMA>(r, c)) = make_uint4(0, 0, 0, 0);
  }
}

// ELEM: bytes of a cached value (2: T, 1: e4m3); UMMA: pages in core-matrix order,
// fetched with one bulk copy each (else rows, TMA boxes); R8: no unit has more than 8
// rows, and the products are transposed, keys and columns of v in the instruction's 16
// rows and the query rows in its 8 columns: half the products, exponentials and
// accumulators (64 tokens over e4m3 pages 111 us, 123 without).
template <typename T, int D, int ELEM, bool UMMA, bool R8>
__global__ void __launch_bounds__(RowsCfg<D, ELEM>::kThreads, kRowsCtas) rows_kernel(
    const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const AttnArgs a) {
  using C = RowsCfg<D, ELEM>;
  constexpr int kWarps = C::kWarps, kThreads = C::kThreads;
  constexpr int kChunks = D * ELEM / 16;  // 16-byte chunks of a row
  // log2 of the largest weight (2^-15 takes it back): 15 in f16, which holds up to 2^16
  constexpr float kTop = ELEM == 1 || std::is_same<T, __half>::value ? 15.f : 0.f;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));  // of the swizzle
  float* sm_m = reinterpret_cast<float*>(smem + C::kSmemMl);
  float* sm_l = sm_m + kWarps * 16;
  uint4* sm_q = reinterpret_cast<uint4*>(smem + C::kSmemQ);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kSmemBars);
  volatile int* flags = reinterpret_cast<volatile int*>(smem + C::kSmemFlags);  // abort
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * C::kRing;
  uint64_t* full = bars + warp * 8;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kWarps * 8; ++i) mbar_init(&bars[i], ELEM == 1 ? 3 : 1);
    flags[0] = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  grid_dep_wait();

  const int32_t* sec = a.plan + H_SECTION;
  const int G = a.plan[H_GROUP];
  // the join's blocks wait beside this kernel (without one, the next kernel may be
  // any, and one that reads this kernel's output before it waits must not start early)
  if (sec[S_JOINS] > 0) grid_dep_launch();
  if (static_cast<int>(blockIdx.x) >= sec[S_CTAS]) return;  // a fixed grid's spare CTA
  const int item0 = a.plan[sec[S_OFF_CTA] + blockIdx.x], item1 = a.plan[sec[S_OFF_CTA] + blockIdx.x + 1];
  const int qr = lane >> 2, qc = lane & 3;
  // ring positions of this warp: the stage to fill next; the stage to read next and
  // the parity of its phase
  uint32_t fill = 0, read = 0, parity = 0;

  for (int it = item0; it < item1; ++it) {
    const int32_t* I = a.plan + sec[S_OFF_ITEMS] + it * kItemInts;
    const int head = I[P_HEAD], tok0 = I[P_TOK0], row0 = I[P_ROW0], nrows = I[P_NROWS];
    const int key0 = I[P_KEY0], key1 = I[P_KEY1], pos0 = I[P_POS0], window = I[P_WINDOW];
    const int kv_len = I[P_KV_LEN];
    const int64_t page_off = I[P_PAGE_OFF];
    // keys a row sees: [lo, hi)
    auto row_hi = [&](int r) { return r < nrows ? max(0, min(kv_len, pos0 + (row0 + r) / G + 1)) : 0; };
    auto row_lo = [&](int r) { return window ? max(0, pos0 + (row0 + r) / G + 1 - window) : 0; };
    // the two rows whose scores this lane has
    const int row_a = R8 ? 2 * qc : qr, row_b = R8 ? 2 * qc + 1 : qr + 8;
    const int hi0 = row_hi(row_a), hi1 = row_hi(row_b), lo0 = row_lo(row_a), lo1 = row_lo(row_b);
    const int hi_min = row_hi(0), hi_max = row_hi(nrows - 1);
    const int lo_min = row_lo(0), lo_max = row_lo(nrows - 1);

    // ---- q fragments (A operand, 16 rows x 16 of d per step) ----
    const T* q0 = nullptr;
    const T* q1 = nullptr;
    {
      const T* qb = static_cast<const T*>(a.q);
      if (qr < nrows)
        q0 = qb + (tok0 + static_cast<int64_t>((row0 + qr) / G)) * a.q_st + (head * G + (row0 + qr) % G) * a.q_sh;
      if (qr + 8 < nrows)
        q1 = qb + (tok0 + static_cast<int64_t>((row0 + qr + 8) / G)) * a.q_st +
             (head * G + (row0 + qr + 8) % G) * a.q_sh;
    }
    uint32_t qf[ELEM == 2 && !R8 ? D / 16 : 1][4];
    if constexpr (ELEM == 2 && !R8) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int d = ks * 16 + qc * 2;
        qf[ks][0] = q0 ? *reinterpret_cast<const uint32_t*>(q0 + d) : 0u;
        qf[ks][1] = q1 ? *reinterpret_cast<const uint32_t*>(q1 + d) : 0u;
        qf[ks][2] = q0 ? *reinterpret_cast<const uint32_t*>(q0 + d + 8) : 0u;
        qf[ks][3] = q1 ? *reinterpret_cast<const uint32_t*>(q1 + d + 8) : 0u;
      }
    }
    float row_scale[2] = {a.scale_log2, a.scale_log2};
    uint32_t qt[R8 ? D / 16 : 1][2];  // row qr, as the second operand
    if constexpr (R8 && ELEM == 2) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qt[ks][0] = q0 ? *reinterpret_cast<const uint32_t*>(q0 + ks * 16 + qc * 2) : 0u;
        qt[ks][1] = q0 ? *reinterpret_cast<const uint32_t*>(q0 + ks * 16 + qc * 2 + 8) : 0u;
      }
    } else if constexpr (R8) {
      float m = 0.f;
      uint2 x[D / 16];
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        x[ks] = q0 ? *reinterpret_cast<const uint2*>(q0 + ks * 16 + qc * 4) : make_uint2(0u, 0u);
        const T* e = reinterpret_cast<const T*>(&x[ks]);
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, fabsf(Num<T>::to_f(e[i])));
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const int k = min(141 - static_cast<int>(__float_as_uint(m) >> 23), 126);
      const float sc = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
      const float inv = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
      row_scale[0] = __shfl_sync(0xffffffffu, inv, 8 * qc);
      row_scale[1] = __shfl_sync(0xffffffffu, inv, 8 * qc + 4);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const T* e = reinterpret_cast<const T*>(&x[ks]);
        qt[ks][0] = pack2(Num<T>::to_f(e[0]) * sc, Num<T>::to_f(e[1]) * sc, __half());
        qt[ks][1] = pack2(Num<T>::to_f(e[2]) * sc, Num<T>::to_f(e[3]) * sc, __half());
      }
    } else if constexpr (ELEM == 1) {
      // rows scaled by 2^k to 2^14 <= max|q| < 2^15 and their scores by 2^-k
      float q_scale[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const T* qp = h ? q1 : q0;
        float m = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint2 x = qp ? *reinterpret_cast<const uint2*>(qp + ks * 16 + qc * 4) : make_uint2(0u, 0u);
          const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
          for (int i = 0; i < 4; ++i) m = fmaxf(m, fabsf(Num<T>::to_f(e[i])));
        }
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int e = static_cast<int>(__float_as_uint(m) >> 23);  // 2^(e - 127) <= m
        const int k = min(141 - e, 126);
        q_scale[h] = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
        row_scale[h] *= __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
      }
      for (int ks = warp; ks < D / 16; ks += kWarps) {  // the four elements a lane's K bytes belong to
        const int d = ks * 16 + qc * 4;
        uint4 f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const T* qp = h ? q1 : q0;
          const uint2 x = qp ? *reinterpret_cast<const uint2*>(qp + d) : make_uint2(0u, 0u);
          const T* e = reinterpret_cast<const T*>(&x);
          const float sc = q_scale[h];
          (h ? f.y : f.x) = pack2(Num<T>::to_f(e[0]) * sc, Num<T>::to_f(e[1]) * sc, __half());
          (h ? f.w : f.z) = pack2(Num<T>::to_f(e[2]) * sc, Num<T>::to_f(e[3]) * sc, __half());
        }
        sm_q[ks * 32 + lane] = f;
      }
    }
    constexpr int kO = R8 ? D / 16 : D / 8;
    float o[kO][4];
#pragma unroll
    for (int i = 0; i < kO; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    // ---- this warp's pages of 16 keys: b0 + warp, b0 + warp + 8, ... ----
    const int b0 = key0 / 16, nb = (key1 - key0 + 15) / 16;
    const int mine = nb > warp ? (nb - warp + kWarps - 1) / kWarps : 0;
    int ids = 0;  // lane j: the page of block `base + j` of mine
    auto fetch_ids = [&](int base) {
      const int64_t pos = static_cast<int64_t>(b0 + warp + (base + lane) * kWarps) * 16;
      const int64_t e = page_off + pos / a.g.page_size;
      ids = 0;
      if (base + lane < mine && e < a.page_table_len) {
        const int64_t id = a.page_table[e];
        ids = static_cast<int>(id < 0 ? 0 : (id >= a.g.num_pages ? a.g.num_pages - 1 : id));
      }
    };
    auto issue = [&](int j) {  // fetch block j of mine into its stage
      if ((j & 31) == 0) fetch_ids(j);
      const int64_t page = __shfl_sync(0xffffffffu, ids, j & 31);
      const uint32_t st = fill;
      fill = fill + 1 == C::kStages ? 0 : fill + 1;
      uint8_t* dst = ring + st * C::kStageBytes;
      const int64_t off = page * a.g.stride_page + head * a.g.stride_head;
      if (UMMA) {
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[st], 2 * C::kPageBytes);
          bulk_load(dst, a.k_pool + off, C::kPageBytes, &full[st]);
          bulk_load(dst + C::kPageBytes, a.v_pool + off, C::kPageBytes, &full[st]);
        }
        if (ELEM == 1 && lane < 2) {  // the scales: two more bulk copies would cost as much as the pages
          cp_async16(smem_u32(dst + 2 * C::kPageBytes + lane * 16),
                     (lane ? a.v_scale : a.k_scale) + page * a.g.scale_page + head * a.g.scale_head);
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[st])) : "memory");
        }
      } else {
        if (lane < 2 * (D / 64)) {  // a box of 16 rows by 64 values each
          const int slot0 = (b0 + warp + j * kWarps) * 16 % a.g.page_size;
          const int kv = lane & 1, pn = lane >> 1;
          if (lane == 0) mbar_arrive_expect_tx(&full[st], 2 * C::kPageBytes);
          __syncwarp((1u << (2 * (D / 64))) - 1u);
          tma_load_4d(dst + kv * C::kPageBytes + pn * 2048, kv ? &tm_v : &tm_k, &full[st], pn * 64, slot0, head,
                      static_cast<int>(page));
        }
      }
    };
    for (int j = 0; j < C::kStages - 1; ++j) {
      if (j < mine) issue(j);
    }
    if (ELEM == 1 && !R8) __syncthreads();  // q is in shared memory
    bool alive = true;
    int j = 0;
    for (; j < mine; ++j) {
      // the stage freed by block j - 1 takes block j + kStages - 1
      if (j + C::kStages - 1 < mine) issue(j + C::kStages - 1);
      const uint32_t st = read;
      const bool ok = mbar_wait(&full[st], parity, flags);
      if (!__all_sync(0xffffffffu, ok)) {
        alive = false;
        break;
      }
      uint8_t* kp = ring + st * C::kStageBytes;
      uint8_t* vp = kp + C::kPageBytes;
      const int key = (b0 + warp + j * kWarps) * 16;
      const bool edge = key + 16 > hi_min || key < lo_max;
      if (edge && (key + 16 > hi_max || key < lo_min)) {
        // values no row of the unit sees may be anything; a weight of 0 would
        // still turn a NaN or an infinity there into NaN
        zero_rows<D, ELEM, UMMA>(vp, max(0, hi_max - key), 16);
        zero_rows<D, ELEM, UMMA>(vp, 0, min(16, lo_min - key));
        fence_proxy_async_smem();  // before the next copy into this stage
        __syncwarp();
      }
      // ---- scores ----
      float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      const uint32_t ka = smem_u32(kp);
      const int mt = lane >> 3, r8 = lane & 7;  // matrix of an x4 this lane addresses, and its row
      // R8: c[0] has keys qr (0, 1) and qr + 8 (2, 3) by rows a and b
      if constexpr (R8 && ELEM == 2) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint32_t k[4];  // (keys 0-7, d lo), (8-15, lo), (0-7, hi), (8-15, hi)
          ldsm4(ka + page_at<kChunks, UMMA>((mt & 1) * 8 + r8, ks * 2 + (mt >> 1)), k);
          mma16816<T>(c[ks & 1], k, qt[ks][0], qt[ks][1]);  // two chains
        }
      } else if constexpr (R8) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ks += 2) {
          uint32_t b[4];  // (keys 0-7, chunk ks), (8-15, ks), (0-7, ks + 1), (8-15, ks + 1)
          ldsm4(ka + page_at<kChunks, UMMA>((mt & 1) * 8 + r8, ks + (mt >> 1)), b);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t k[4];
            e4m3x4_f16(b[2 * h], k[0], k[2]);
            e4m3x4_f16(b[2 * h + 1], k[1], k[3]);
            mma16816<__half>(c[h], k, qt[ks + h][0], qt[ks + h][1]);  // two chains
          }
        }
      } else if (ELEM == 2) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint32_t b[4];  // (keys 0-7, d lo), (0-7, hi), (8-15, lo), (8-15, hi)
          ldsm4(ka + page_at<kChunks, UMMA>((mt >> 1) * 8 + r8, ks * 2 + (mt & 1)), b);
          mma16816<T>(c[0], qf[ks], b[0], b[1]);
          mma16816<T>(c[1], qf[ks], b[2], b[3]);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < D / 16; ks += 2) {
          uint32_t b[4];  // (keys 0-7, chunk ks), (8-15, ks), (0-7, ks + 1), (8-15, ks + 1)
          ldsm4(ka + page_at<kChunks, UMMA>((mt & 1) * 8 + r8, ks + (mt >> 1)), b);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 q = sm_q[(ks + h) * 32 + lane];
            const uint32_t qa[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              uint32_t lo, hi;
              e4m3x4_f16(b[2 * h + n], lo, hi);
              mma16816<__half>(c[n], qa, lo, hi);
            }
          }
        }
      }
      float x0, x1;    // the rows' maxima of s_j (e4m3: s_j + e_j)
      float vs[2][2];  // 2^e_j
      if constexpr (R8) {
        const uint8_t* sp = kp + 2 * C::kPageBytes + qr;
        float ve[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float ks = ELEM == 1 ? scale_of(sp[n * 8]) : 1.f;
          uint32_t vb = ELEM == 1 ? sp[16 + n * 8] : 127u;
          c[0][2 * n] = (c[0][2 * n] + c[1][2 * n]) * (row_scale[0] * ks);
          c[0][2 * n + 1] = (c[0][2 * n + 1] + c[1][2 * n + 1]) * (row_scale[1] * ks);
          if (edge) {
            const int x = key + n * 8 + qr;
            if (x >= hi0 || x < lo0) c[0][2 * n] = -INFINITY;
            if (x >= hi1 || x < lo1) c[0][2 * n + 1] = -INFINITY;
            if (ELEM == 1 && (x >= hi_max || x < lo_min)) vb = 0u;  // a scale byte no row sees
          }
          vs[n][0] = scale_of(vb);
          ve[n] = ELEM == 1 ? exponent_of(vb) : 0.f;
        }
        x0 = fmaxf(c[0][0] + ve[0], c[0][2] + ve[1]);
        x1 = fmaxf(c[0][1] + ve[0], c[0][3] + ve[1]);
#pragma unroll
        for (int step = 4; step < 32; step *= 2) {  // over the eight lanes of a row
          x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, step));
          x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, step));
        }
      } else {
        uint32_t vb[2] = {0u, 0u};  // value scale bytes of this lane's four keys
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          float k0 = 1.f, k1 = 1.f;
          if (ELEM == 1) {
            const uint8_t* sp = kp + 2 * C::kPageBytes + n * 8 + qc * 2;
            const uint32_t kb = *reinterpret_cast<const uint16_t*>(sp);
            vb[n] = *reinterpret_cast<const uint16_t*>(sp + 16);
            k0 = scale_of(kb & 255u);
            k1 = scale_of(kb >> 8);
          }
          c[n][0] *= row_scale[0] * k0;
          c[n][1] *= row_scale[0] * k1;
          c[n][2] *= row_scale[1] * k0;
          c[n][3] *= row_scale[1] * k1;
        }
        if (edge) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int x = key + n * 8 + qc * 2 + e;
              if (x >= hi0 || x < lo0) c[n][e] = -INFINITY;
              if (x >= hi1 || x < lo1) c[n][2 + e] = -INFINITY;
              // a scale byte no row sees
              if (ELEM == 1 && (x >= hi_max || x < lo_min)) vb[n] &= e ? 0x00ffu : 0xff00u;
            }
        }
        // ---- running maximum and sum; o is rescaled only when the maximum grew ----
        auto row_max = [](float x) {  // over the four lanes of a row
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
          return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        };
        if (ELEM == 1) {
          float ve[2][2];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t byte = (vb[n] >> (8 * e)) & 255u;
              vs[n][e] = scale_of(byte);
              ve[n][e] = exponent_of(byte);
            }
          x0 = fmaxf(fmaxf(c[0][0] + ve[0][0], c[0][1] + ve[0][1]), fmaxf(c[1][0] + ve[1][0], c[1][1] + ve[1][1]));
          x1 = fmaxf(fmaxf(c[0][2] + ve[0][0], c[0][3] + ve[0][1]), fmaxf(c[1][2] + ve[1][0], c[1][3] + ve[1][1]));
        } else {
          x0 = fmaxf(fmaxf(c[0][0], c[0][1]), fmaxf(c[1][0], c[1][1]));
          x1 = fmaxf(fmaxf(c[0][2], c[0][3]), fmaxf(c[1][2], c[1][3]));
        }
        x0 = row_max(x0);
        x1 = row_max(x1);
      }
      if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        const float f0 = m0 == n0 ? 1.f : fast_exp2(m0 - n0), f1 = m1 == n1 ? 1.f : fast_exp2(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int i = 0; i < kO; ++i) {
          o[i][0] *= f0;
          o[i][R8 ? 2 : 1] *= f0;
          o[i][R8 ? 1 : 2] *= f1;
          o[i][3] *= f1;
        }
      }
      const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
      // the headroom is added last: x is exact for the largest weight (for 8-bit values a
      // whole number, -e), where m - 15 and what is relative to it would round by more
      auto weight = [](float x) { return fast_exp2(kTop > 0.f ? x + kTop : x); };
      uint32_t p[4];
      if constexpr (R8) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = weight(c[0][2 * n] - r0), p1 = weight(c[0][2 * n + 1] - r1);
          l0 += p0;
          l1 += p1;
          // row qr, keys 2 qc and 2 qc + 1
          p[n] = transpose8(ELEM == 1 ? pack2(p0 * vs[n][0], p1 * vs[n][0], __half()) : pack2(p0, p1, T()));
        }
      } else {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = weight(c[n][0] - r0), p1 = weight(c[n][1] - r0);
          const float p2 = weight(c[n][2] - r1), p3 = weight(c[n][3] - r1);
          l0 += p0 + p1;
          l1 += p2 + p3;
          if (ELEM == 1) {
            p[2 * n] = pack2(p0 * vs[n][0], p1 * vs[n][1], __half());
            p[2 * n + 1] = pack2(p2 * vs[n][0], p3 * vs[n][1], __half());
          } else {
            p[2 * n] = pack2(p0, p1, T());
            p[2 * n + 1] = pack2(p2, p3, T());
          }
        }
      }
      // ---- o += p v ----
      const uint32_t va = smem_u32(vp);
      if constexpr (R8 && ELEM == 2) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t v[4];  // (chunk 2 i, keys 0-7), (2 i + 1, 0-7), (2 i, 8-15), (2 i + 1, 8-15), transposed
          ldsm4_t(va + page_at<kChunks, UMMA>((mt >> 1) * 8 + r8, 2 * i + (mt & 1)), v);
          mma16816<T>(o[i], v, p[0], p[1]);
        }
      } else if constexpr (R8) {
#pragma unroll
        for (int i = 0; i < D / 16; i += 2) {
          uint32_t b[4];  // pairs of neighbouring d, transposed
          ldsm4_t(va + page_at<kChunks, UMMA>((mt & 1) * 8 + r8, i + (mt >> 1)), b);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v[4];  // even d's pairs of keys, odd d's; keys 0-7, 8-15
            e4m3x4_f16(__byte_perm(b[2 * h], 0u, 0x3120), v[0], v[1]);
            e4m3x4_f16(__byte_perm(b[2 * h + 1], 0u, 0x3120), v[2], v[3]);
            mma16816<__half>(o[i + h], v, p[0], p[1]);
          }
        }
      } else if (ELEM == 2) {
#pragma unroll
        for (int i = 0; i < D / 8; i += 2) {
          uint32_t b[4];  // (keys 0-7, chunk i), (8-15, i), (0-7, i + 1), (8-15, i + 1), transposed
          ldsm4_t(va + page_at<kChunks, UMMA>((mt & 1) * 8 + r8, i + (mt >> 1)), b);
          mma16816<T>(o[i], p, b[0], b[1]);
          mma16816<T>(o[i + 1], p, b[2], b[3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 16; i += 2) {
          uint32_t b[4];  // pairs of neighbouring d, transposed
          ldsm4_t(va + page_at<kChunks, UMMA>((mt & 1) * 8 + r8, i + (mt >> 1)), b);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // (key, d): bytes (0, 0) (0, 1) (1, 0) (1, 1) -> even d's pair of keys, odd d's
            uint32_t e0, d0, e1, d1;
            e4m3x4_f16(__byte_perm(b[2 * h], 0u, 0x3120), e0, d0);
            e4m3x4_f16(__byte_perm(b[2 * h + 1], 0u, 0x3120), e1, d1);
            mma16816<__half>(o[2 * (i + h)], p, e0, e1);
            mma16816<__half>(o[2 * (i + h) + 1], p, d0, d1);
          }
        }
      }
      __syncwarp();  // the stage is free for block j + kStages
      if (++read == C::kStages) read = 0, parity ^= 1;
    }
    if (!alive) {
      // give up: wait (bounded) for the copies in flight, so that none lands in
      // another block's shared memory
      flags[0] = 1;
      for (int x = j; x < min(j + C::kStages, mine); ++x) {
        const uint64_t t0 = global_timer_ns();
        while (!mbar_try_wait(&full[read], parity) && global_timer_ns() - t0 < kWaitTimeoutNs) {
        }
        if (++read == C::kStages) read = 0, parity ^= 1;
      }
    }
    if constexpr (kTop > 0.f) {
      l0 *= 0x1p-15f;
      l1 *= 0x1p-15f;
#pragma unroll
      for (int i = 0; i < kO; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= 0x1p-15f;
    }
#pragma unroll
    for (int step = R8 ? 4 : 1; step < (R8 ? 32 : 4); step *= 2) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, step);
      l1 += __shfl_xor_sync(0xffffffffu, l1, step);
    }

    // ---- join the warps: O over the warp's own ring, m and l beside it ----
    __syncwarp();
    float* os = reinterpret_cast<float*>(ring);
    if constexpr (R8) {
#pragma unroll
      for (int i = 0; i < kO; ++i) {  // rows a and b
        if (ELEM == 2) {  // columns 16 i + qr and 16 i + 8 + qr
          os[row_a * D + i * 16 + qr] = o[i][0];
          os[row_b * D + i * 16 + qr] = o[i][1];
          os[row_a * D + i * 16 + 8 + qr] = o[i][2];
          os[row_b * D + i * 16 + 8 + qr] = o[i][3];
          continue;
        }
        // columns 16 i + 2 qr and the next
        *reinterpret_cast<float2*>(os + row_a * D + i * 16 + qr * 2) = make_float2(o[i][0], o[i][2]);
        *reinterpret_cast<float2*>(os + row_b * D + i * 16 + qr * 2) = make_float2(o[i][1], o[i][3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        // 16-bit: columns of tile i are d = 8 i + n. 8-bit: tiles 2 j, 2 j + 1 hold
        // the even and the odd d of chunk j
        const int d0 = ELEM == 2 ? i * 8 + qc * 2 : (i >> 1) * 16 + qc * 4 + (i & 1);
        const int d1 = ELEM == 2 ? d0 + 1 : d0 + 2;
        os[qr * D + d0] = o[i][0];
        os[qr * D + d1] = o[i][1];
        os[(qr + 8) * D + d0] = o[i][2];
        os[(qr + 8) * D + d1] = o[i][3];
      }
    }
    if (R8 ? qr == 0 : qc == 0) {
      sm_m[warp * 16 + row_a] = m0;
      sm_m[warp * 16 + row_b] = m1;
      sm_l[warp * 16 + row_a] = l0;
      sm_l[warp * 16 + row_b] = l1;
    }
    fence_proxy_async_smem();  // before the next item's copies into the ring
    __syncthreads();
    constexpr int kPer = 16 * D / kThreads;  // outputs of a thread, neighbours in a row
    const int row = threadIdx.x / (kThreads / 16), dcol = (threadIdx.x % (kThreads / 16)) * kPer;
    float M = -INFINITY, L = 0.f, acc[kPer];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w * 16 + row]);
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
    const float Mr = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = fast_exp2(sm_m[w * 16 + row] - Mr);
      L += sm_l[w * 16 + row] * f;
      const float* ow = reinterpret_cast<const float*>(smem + w * C::kRing) + row * D + dcol;
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] = fmaf(ow[e], f, acc[e]);
    }
    if (I[P_PARTS] > 1 && sec[S_JOINS] == 0) {
      // a unit of one cluster: every CTA leaves its state in its shared memory, and
      // takes its share of the columns from all of them, in order
      __syncthreads();  // the rings are read
      float* state = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int e = 0; e < kPer; e += 4)
        *reinterpret_cast<float4*>(state + row * D + dcol + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
      if (dcol == 0) {
        state[16 * D + row] = M;
        state[16 * D + 16 + row] = L;
      }
      cluster_sync();
      auto join = [&](auto n) {
        constexpr int kSize = decltype(n)::value, kVecs = D / kSize / 4;  // kVecs of a row
        const int rank = blockIdx.x % kSize;
        for (int x = threadIdx.x; x < 16 * kVecs; x += kThreads) {
          const int r = x / kVecs, c = rank * (D / kSize) + x % kVecs * 4;
          if (r >= nrows) break;
          float m[kSize], top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int p = 0; p < kSize; ++p) {
            m[p] = peer_float(peer_addr(state + 16 * D + r, p));
            top = fmaxf(top, m[p]);
          }
          const float ref = top == -INFINITY ? 0.f : top;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int p = 0; p < kSize; ++p) {
            const float w = fast_exp2(m[p] - ref);
            const float4 v = peer_float4(peer_addr(state + r * D + c, p));
            sum = fmaf(peer_float(peer_addr(state + 16 * D + 16 + r, p)), w, sum);
            o.x = fmaf(v.x, w, o.x);
            o.y = fmaf(v.y, w, o.y);
            o.z = fmaf(v.z, w, o.z);
            o.w = fmaf(v.w, w, o.w);
          }
          const int64_t tok = tok0 + static_cast<int64_t>((row0 + r) / G);
          const int hq = head * G + (row0 + r) % G;
          float lse2;
          float f = row_factor(top, sum, lse2);
          if (a.sinks) f *= sink_factor(lse2, a.sinks[hq], a.sink_mode);
          uint2 v;
          v.x = pack2(o.x * f, o.y * f, T());
          v.y = pack2(o.z * f, o.w * f, T());
          *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + tok * a.o_st + hq * a.o_sh + c) = v;
          if (a.lse && c == 0) a.lse[tok * a.lse_st + hq] = lse2;
        }
      };
      if (I[P_PARTS] == 8) join(std::integral_constant<int, 8>());
      else if (I[P_PARTS] == 4) join(std::integral_constant<int, 4>());
      else join(std::integral_constant<int, 2>());
      cluster_sync();  // the states are read
    } else if (I[P_PARTS] > 1) {  // a span of a unit: leave the state in its slot (join_kernel)
      float* own = a.slots + static_cast<int64_t>(I[P_SLOT]) * rows_slot_floats(D);
      if (row < nrows) {
#pragma unroll
        for (int e = 0; e < kPer; e += 2)
          reinterpret_cast<float2*>(own)[((dcol + e) / 4 * 16 + row) * 2 + (dcol + e) / 2 % 2] =
              make_float2(acc[e], acc[e + 1]);
        if (dcol == 0) {
          own[16 * D + row] = M;
          own[16 * D + 16 + row] = L;
        }
      }
    } else if (row < nrows) {
      const int64_t tok = tok0 + static_cast<int64_t>((row0 + row) / G);
      const int hq = head * G + (row0 + row) % G;
      float lse2;
      float f = row_factor(M, L, lse2);
      if (a.sinks) f *= sink_factor(lse2, a.sinks[hq], a.sink_mode);
      T* op = static_cast<T*>(a.out) + tok * a.o_st + hq * a.o_sh + dcol;
#pragma unroll
      for (int e = 0; e < kPer; e += 2)
        *reinterpret_cast<uint32_t*>(op + e) = pack2(acc[e] * f, acc[e + 1] * f, T());
      if (a.lse && dcol == 0) a.lse[tok * a.lse_st + hq] = lse2;
    }
    __syncthreads();  // the rings are read; the next item's copies may land
    if (flags[0]) break;
  }
  if (threadIdx.x == 0 && flags[0] && a.status) atomicExch(a.status, 1);
}

// Joins the spans of split units: an entry of the join list is RB rows (or fewer)
// whose partial states lie `step` slots apart,
//   M = max m_p, L = sum l_p 2^(m_p - M), o = sum o_p 2^(m_p - M) / L,
// in slot order. A thread takes four columns of a row; few rows go to a block, and
// GROUPS groups of threads share the spans (joined in shared memory, in order), so
// that a unit of many spans has many loads in flight (32 tokens over 32k keys: 63 us for
// the whole attention with one group, 48 with them). Bound by the states' way through L2,
// 66 KB a span and q tile, and by its own start, which passes under the end of the rows
// kernel; the tiles kernel does not let it start early.
template <typename T, int D, int SECTION, int GROUPS>
__global__ void __launch_bounds__(kJoinRows[SECTION] * D / 4 * GROUPS) join_kernel(const AttnArgs a) {
  constexpr int RB = kJoinRows[SECTION], kThreads = RB * D / 4;  // of a group
  constexpr int kSlotRows = SECTION == 0 ? kRowsTile : 128;
  constexpr int64_t kSlot = SECTION == 0 ? rows_slot_floats(D) : tile_slot_floats(D);
  __shared__ float4 sm_o[GROUPS > 1 ? GROUPS * kThreads : 1];
  __shared__ float2 sm_ml[GROUPS > 1 ? GROUPS * RB : 1];
  const int group = threadIdx.x / kThreads, t = threadIdx.x % kThreads;
  const int r = t % RB, col = t / RB;
  grid_dep_wait();
  const int32_t* sec = a.plan + H_SECTION + SECTION * kSectionInts;
  const int G = a.plan[H_GROUP], n = sec[S_JOINS];
  const int32_t* list = a.plan + sec[S_OFF_JOINS];
  for (int b = blockIdx.x; b < n; b += gridDim.x) {
    const int32_t* J = list + b * kJoinInts;
    const bool live = r < J[J_ROWS];
    const int parts = J[J_PARTS], rq = J[J_ROW0] + r;
    const int p0 = parts * group / GROUPS, p1 = live ? parts * (group + 1) / GROUPS : p0;
    const float* s0 = a.slots + J[J_SLOT] * kSlot;
    const int64_t step = J[J_STEP] * kSlot;
    const int at = J[J_SLOT_ROW] + r;
    float M = -INFINITY, L = 0.f;
#pragma unroll 8
    for (int p = p0; p < p1; ++p) M = fmaxf(M, s0[p * step + kSlotRows * D + at]);
    float ref = M == -INFINITY ? 0.f : M;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int p = p0; p < p1; ++p) {
      const float* sp = s0 + p * step;
      const float4 v = reinterpret_cast<const float4*>(sp)[col * kSlotRows + at];
      const float w = fast_exp2(sp[kSlotRows * D + at] - ref);
      L = fmaf(sp[kSlotRows * D + kSlotRows + at], w, L);
      acc.x = fmaf(v.x, w, acc.x);
      acc.y = fmaf(v.y, w, acc.y);
      acc.z = fmaf(v.z, w, acc.z);
      acc.w = fmaf(v.w, w, acc.w);
    }
    if (GROUPS > 1) {
      sm_o[threadIdx.x] = acc;
      if (col == 0) sm_ml[group * RB + r] = make_float2(M, L);
      __syncthreads();
      if (group == 0) {
        M = -INFINITY;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) M = fmaxf(M, sm_ml[g * RB + r].x);
        ref = M == -INFINITY ? 0.f : M;
        L = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const float2 ml = sm_ml[g * RB + r];
          const float4 v = sm_o[g * kThreads + t];
          const float w = fast_exp2(ml.x - ref);
          L = fmaf(ml.y, w, L);
          acc.x = fmaf(v.x, w, acc.x);
          acc.y = fmaf(v.y, w, acc.y);
          acc.z = fmaf(v.z, w, acc.z);
          acc.w = fmaf(v.w, w, acc.w);
        }
      }
      __syncthreads();
    }
    if (group > 0 || !live) continue;
    const int64_t tok = J[J_TOK0] + static_cast<int64_t>(rq / G);
    const int hq = J[J_HEAD] * G + rq % G;
    float lse2;
    float f = row_factor(M, L, lse2);
    if (a.sinks) f *= sink_factor(lse2, a.sinks[hq], a.sink_mode);
    uint2 v;
    v.x = pack2(acc.x * f, acc.y * f, T());
    v.y = pack2(acc.z * f, acc.w * f, T());
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + tok * a.o_st + hq * a.o_sh + col * 4) = v;
    if (a.lse && col == 0) a.lse[tok * a.lse_st + hq] = lse2;
  }
}

template <int SECTION, int GROUPS>
int launch_join(const AttnArgs& a, int32_t dtype, int32_t head_dim, int blocks, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(blocks));
  const dim3 block(static_cast<unsigned>(kJoinRows[SECTION] * head_dim / 4 * GROUPS));
  auto go = [&](auto kernel) { return launch_pdl(kernel, grid, block, 0, st, "join_kernel", a); };
  if (dtype == D2SD_DTYPE_BF16)
    return head_dim == 128 ? go(join_kernel<__nv_bfloat16, 128, SECTION, GROUPS>)
                           : go(join_kernel<__nv_bfloat16, 64, SECTION, GROUPS>);
  return head_dim == 128 ? go(join_kernel<__half, 128, SECTION, GROUPS>)
                         : go(join_kernel<__half, 64, SECTION, GROUPS>);
}

// Groups share the spans where a unit has more of them than one thread keeps in
// flight (one token against 32k keys: 74 spans a unit).
template <int SECTION>
int run_join(const AttnArgs& a, int32_t dtype, int32_t head_dim, const int32_t* sec, int num_ctas,
             bool fixed_grid, cudaStream_t st) {
  const int most = 16 * num_ctas;
  // a fixed grid takes what fits the SMs at once (blocks of 1024 threads) and goes on from there
  const int blocks = fixed_grid ? 2 * num_ctas : (sec[S_JOINS] < most ? sec[S_JOINS] : most);
  if (fixed_grid || sec[S_PARTS] > 8) return launch_join<SECTION, SECTION == 0 ? 8 : 4>(a, dtype, head_dim, blocks, st);
  return launch_join<SECTION, 1>(a, dtype, head_dim, blocks, st);
}

template <typename T, int D, int ELEM, bool UMMA, bool R8>
int launch_rows(const AttnArgs& a, const CUtensorMap& tk, const CUtensorMap& tv, int ctas, int cluster,
                cudaStream_t stream) {
  using C = RowsCfg<D, ELEM>;
  static std::atomic<uint64_t> configured{0};  // bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !((configured.load() >> dev) & 1)) {
    cudaError_t e = cudaFuncSetAttribute(rows_kernel<T, D, ELEM, UMMA, R8>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess)
      return fail(D2SD_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
    if (dev < 64) configured.fetch_or(1ull << dev);
  }
  return launch_pdl_clusters(cluster, rows_kernel<T, D, ELEM, UMMA, R8>, dim3(ctas), dim3(C::kThreads),
                             C::kSmemBytes, stream, "rows_kernel", tk, tv, a);
}

int run_rows(const AttnArgs& a, int32_t dtype, int32_t head_dim, int32_t num_kv_heads, bool scaled, int ctas,
             int cluster, bool r8, cudaStream_t st) {
  CUtensorMap tk = {}, tv = {};  // of pages of rows only
  if (!a.g.umma) {
    int rc = encode_pages(&tk, &tv, a, dtype, head_dim, num_kv_heads);
    if (rc) return rc;
  }
  auto go = [&](auto t, auto elem, auto umma, auto few) {
    using T = decltype(t);
    constexpr int E = decltype(elem)::value;
    constexpr bool U = decltype(umma)::value, F = decltype(few)::value;
    return head_dim == 128 ? launch_rows<T, 128, E, U, F>(a, tk, tv, ctas, cluster, st)
                           : launch_rows<T, 64, E, U, F>(a, tk, tv, ctas, cluster, st);
  };
  const auto no = std::false_type();
  const auto yes = std::true_type();
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  auto rows = [&](auto t, auto elem, auto umma) { return r8 ? go(t, elem, umma, yes) : go(t, elem, umma, no); };
  if (scaled) return rows(__nv_bfloat16(), One(), yes);
  if (dtype == D2SD_DTYPE_BF16)
    return a.g.umma ? rows(__nv_bfloat16(), Two(), yes) : rows(__nv_bfloat16(), Two(), no);
  return a.g.umma ? rows(__half(), Two(), yes) : rows(__half(), Two(), no);
}

}  // namespace
}  // namespace d2sd

extern "C" int64_t d2sd_paged_workspace_bytes(int32_t num_ctas, int32_t head_dim) {
  if (num_ctas <= 0 || (head_dim != 64 && head_dim != 128)) return -1;
  return d2sd::paged::workspace_bytes(num_ctas, head_dim);
}

extern "C" int d2sd_paged_attention(
    const void* q, int64_t q_stride_token, int64_t q_stride_head, int64_t num_tokens, int32_t dtype,
    const void* k_pool,
    const void* v_pool, int64_t cache_stride_page, int64_t cache_stride_slot, int64_t cache_stride_head,
    int32_t page_size, int64_t num_pages, int32_t cache_format, const void* k_scale, const void* v_scale,
    int64_t scale_stride_page, int64_t scale_stride_head, const int32_t* page_table,
    int64_t page_table_len, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, float sm_scale,
    const int32_t* plan, const int32_t* sections, int32_t num_ctas, int32_t fixed_grid, void* workspace, int64_t workspace_bytes,
    void* wide_k, void* wide_v, const float* sinks, int32_t sink_mode, void* out, int64_t out_stride_token, int64_t out_stride_head,
    float* lse, int64_t lse_stride_token, int32_t* status, void* stream) {
  using namespace d2sd;
  using namespace d2sd::paged;
  const char* const w = "d2sd_paged_attention";
  if (!plan || !sections || num_qo_heads <= 0 || num_kv_heads <= 0 || num_qo_heads % num_kv_heads)
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": invalid argument");
  const int32_t* tiles = sections + kSectionInts;
  if (sections[S_ITEMS] == 0 && tiles[S_ITEMS] == 0 && !fixed_grid) return D2SD_OK;  // no query rows
  if (!(sm_scale > 0.f))
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": sm_scale must be positive");
  if (!q || !out || !k_pool || !v_pool || !page_table || page_table_len < 0 || num_tokens <= 0)
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": invalid argument");
  if (head_dim != 64 && head_dim != 128)
    return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": head_dim must be 64 or 128");
  if (dtype != D2SD_DTYPE_BF16 && dtype != D2SD_DTYPE_F16)
    return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": q must be bf16 or fp16");
  const bool scaled = k_scale != nullptr;
  if (scaled != (v_scale != nullptr))
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": k_scale and v_scale go together");
  if (scaled && dtype != D2SD_DTYPE_BF16)
    return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": 8-bit pages take bf16 queries");
  if ((wide_k != nullptr) != (wide_v != nullptr) || (wide_k && !scaled) || !aligned16(wide_k) || !aligned16(wide_v))
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": wide_k and wide_v go together, with an 8-bit cache");
  if (sinks && sink_mode != D2SD_SINK_REFERENCE && sink_mode != D2SD_SINK_EXACT)
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": unknown sink_mode");
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_pool) || !aligned16(v_pool) ||
      !aligned16(k_scale) || !aligned16(v_scale) || q_stride_token % 8 || q_stride_head % 8 ||
      out_stride_token % 8 || out_stride_head % 8 || scale_stride_page % 16 || scale_stride_head % 16)
    return fail(D2SD_ERR_INVALID_ARGUMENT,
                std::string(w) + ": rows must be 16-byte aligned, strides multiples of 8");
  const int cluster = sections[S_PARTS] > 1 && sections[S_JOINS] == 0 ? sections[S_PARTS] : 1;
  if (cluster > 1 && (fixed_grid || cluster > kCluster || sections[S_CTAS] % cluster))
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": a plan of clusters does not take a fixed grid");
  bool fits = num_ctas > 0;
  for (int s = 0; s < kSections; ++s) {
    const int32_t* sec = sections + s * kSectionInts;
    fits = fits && sec[S_CTAS] <= section_ctas(s, num_ctas) && sec[S_SLOTS] <= 2 * section_ctas(s, num_ctas);
  }
  if (!fits)
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": the plan is for another grid");
  if (workspace_bytes < d2sd_paged_workspace_bytes(num_ctas, head_dim) || !workspace ||
      !aligned16(workspace))
    return fail(D2SD_ERR_WORKSPACE, std::string(w) + ": workspace too small or unaligned");
  AttnArgs a{};
  int rc = make_page_geom(&a.g, w, head_dim, scaled ? 1 : 2, cache_stride_page, cache_stride_slot,
                          cache_stride_head, page_size, num_pages, cache_format, scaled,
                          scale_stride_page, scale_stride_head);
  if (rc) return rc;
  if (page_size % 16)
    return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": page_size must be a multiple of 16");
  a.q = q, a.out = out, a.lse = lse;
  a.q_st = q_stride_token, a.q_sh = q_stride_head, a.o_st = out_stride_token, a.o_sh = out_stride_head,
  a.lse_st = lse_stride_token;
  a.k_pool = static_cast<const uint8_t*>(k_pool), a.v_pool = static_cast<const uint8_t*>(v_pool);
  a.k_scale = static_cast<const uint8_t*>(k_scale), a.v_scale = static_cast<const uint8_t*>(v_scale);
  a.page_table = page_table, a.page_table_len = page_table_len;
  a.plan = plan;
  a.slots = static_cast<float*>(workspace);
  a.sinks = sinks, a.sink_mode = sink_mode;
  a.status = status;
  a.scale_log2 = sm_scale * kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int32_t kinds = sections[kSections * kSectionInts + 3];  // of units (paged_plan.cpp)
  const bool few_rows = (fixed_grid & (D2SD_GRID_FEW_ROWS | D2SD_GRID_EIGHT_ROWS)) != 0;
  if ((few_rows && tiles[S_ITEMS] > 0) || ((fixed_grid & D2SD_GRID_EIGHT_ROWS) && (kinds & 2)))
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": the plan has more rows than fixed_grid says");
  AttnArgs t = a;  // the tiles kernel's half of the workspace
  t.slots += tile_slots_at(num_ctas, head_dim);
  if (sections[S_ITEMS] > 0 || fixed_grid) {
    rc = run_rows(a, dtype, head_dim, num_kv_heads, scaled, fixed_grid ? section_ctas(0, num_ctas) : sections[S_CTAS],
                  cluster, fixed_grid ? (fixed_grid & D2SD_GRID_EIGHT_ROWS) != 0 : !(kinds & 2), st);
    if (rc) return rc;
  }
  const bool any_tiles = fixed_grid ? !few_rows : tiles[S_ITEMS] > 0;
  if (any_tiles) {
    if (wide_k) {  // 8-bit pages that many row tiles go over: widened once
      const int32_t lo = sections[kSections * kSectionInts + 1], hi = sections[kSections * kSectionInts + 2];
      if (lo < 0 || hi <= lo || hi > page_table_len)
        return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": the page table is shorter than the plan's");
      rc = launch_widen(a.k_pool, a.v_pool, a.k_scale, a.v_scale, a.g, page_table + lo, hi - lo, num_kv_heads,
                        head_dim, wide_k, wide_v, stream);
      if (rc) return rc;
      t.k_pool = static_cast<const uint8_t*>(wide_k), t.v_pool = static_cast<const uint8_t*>(wide_v);
      t.k_scale = t.v_scale = nullptr;
      t.page_table = nullptr;
      t.first_entry = lo;
      t.g.stride_head = 32 * static_cast<int64_t>(head_dim);
      t.g.stride_page = num_kv_heads * t.g.stride_head;
      t.g.num_pages = hi - lo;
    }
    rc = launch_tiles(t, dtype, head_dim, scaled && !wide_k, num_tokens, num_qo_heads, num_kv_heads,
                      !fixed_grid && !(kinds & 1),
                      fixed_grid ? num_ctas : tiles[S_CTAS], stream);
    if (rc) return rc;
  }
  if (sections[S_JOINS] > 0 || fixed_grid) {
    rc = run_join<0>(a, dtype, head_dim, sections, num_ctas, fixed_grid != 0, st);
    if (rc) return rc;
  }
  if (any_tiles && (tiles[S_JOINS] > 0 || fixed_grid)) rc = run_join<1>(t, dtype, head_dim, tiles, num_ctas, fixed_grid != 0, st);
  return rc;
}
