// Writing new tokens into the paged cache and reading rows back out of it.
//
// append_kernel: the step between a layer's projections and its attention, for a
// ragged batch of new tokens, in one pass: per-head RMSNorm of q and k
// (optional), the rotary position of q and k (optional), and the write of k and v
// into the cache's pages, in their own type or as e4m3 rows with a scale byte
// (paged.cuh). With c, s = cos, sin of the token's position (fp32 tables, so any
// scaling of the angles for long contexts is the table's):
//   y = x * rsqrt(mean(x^2) + eps) * w
//   (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s)
// with pairs (i, i + rotary/2) or (2i, 2i + 1), i < rotary/2; the rest of the head
// stays. All of it in fp32 and rounded once, into q_out and into the cache; an 8-bit k
// value next to a border between two of them is decided in 64 bits (exact_row).
// read_kernel: rows back out of the pages, 8-bit values times their scale.
// commit_e4m3_kernel: the accepted branch's rows (commit.cu) into an 8-bit cache.
//
// head_dim / 8 lanes hold one (token, head) row, 8 elements each: the norm's sum
// and the row's largest magnitude are shuffles inside that group, and the rotary
// partner is either in the lane (interleaved) or rotary/16 lanes away. A group
// stays with one token and takes its heads in turn, four rows' loads in flight:
// the chain of dependent loads that finds a token's page (request, position, page
// table) and its cos and sin are paid once for all its heads, and a warp's
// neighbouring tokens fill whole 32-byte sectors of the pages, whose rows of eight
// values lie 16 bytes apart. Few tokens spread their heads over several blocks.
//
// Bound: HBM, each row read once and written once. Measured (GPU time; of 6.54 TB/s of a
// plain copy): 9 prompts of 7 to 3001 tokens, 64 / 8 heads of 64, f16, 389 MB, 74 us =
// 0.80; about 13,000 tokens of 32 / 8 heads of 128 into e4m3 pages 77 us = 0.59 (rows of 128
// bytes written as 8-byte pieces), and their rows back 16 us; 32,768 rows of 8 e4m3
// heads of 128 read into bf16, 202 MB, 36.6 us = 0.84 (37.2 with four rows in flight);
// one new token of 64 requests 4.4 us on the GPU (a call from Python is 13 us, its host
// time).
// One group per row (the head inside the row index) took 84 us for that read: the chain
// of loads for each row, and sectors filled by half.
#include <string>
#include <type_traits>

#include "paged.cuh"

namespace d2sd {

int make_page_geom(PageGeom* g, const char* what, int32_t head_dim, int32_t elem, int64_t stride_page,
                   int64_t stride_slot, int64_t stride_head, int32_t page_size, int64_t num_pages,
                   int32_t cache_format, bool scaled, int64_t scale_stride_page,
                   int64_t scale_stride_head) {
  const std::string w(what);
  if (page_size <= 0 || num_pages <= 0)
    return fail(D2SD_ERR_INVALID_ARGUMENT, w + ": invalid page size or pool size");
  if (cache_format != D2SD_KV_ROWS && cache_format != D2SD_KV_UMMA_PAGES)
    return fail(D2SD_ERR_INVALID_ARGUMENT, w + ": unknown cache_format");
  const bool umma = cache_format == D2SD_KV_UMMA_PAGES;
  if (umma && (page_size != 16 || elem > 2))
    return fail(D2SD_ERR_UNSUPPORTED, w + ": UMMA pages hold 16 rows of 8- or 16-bit values");
  if (scaled && !umma)
    return fail(D2SD_ERR_UNSUPPORTED, w + ": 8-bit rows are kept in UMMA pages");
  const int64_t ve = 16 / elem;
  if (stride_page % ve || stride_head % ve || (!umma && stride_slot % ve))
    return fail(D2SD_ERR_INVALID_ARGUMENT, w + ": cache strides must keep rows 16-byte aligned");
  g->stride_page = stride_page * elem;
  g->stride_slot = stride_slot * elem;
  g->stride_head = stride_head * elem;
  g->scale_page = scale_stride_page;
  g->scale_head = scale_stride_head;
  g->num_pages = num_pages;
  g->page_size = page_size;
  g->umma = umma ? 1 : 0;
  return D2SD_OK;
}

namespace {

constexpr int kThreads = 256;

template <int W>  // sum / max over the W lanes of a row's group
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
template <int W>
__device__ __forceinline__ float group_max(float x) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// 1 / sqrt(x) with a Newton step, e = 1 - x r^2 from the exact product x r: to about
// half a last place (rsqrtf alone: 2). 0 and infinity keep rsqrtf's answers.
__device__ __forceinline__ float exact_rsqrt(float x) {
  const float r = rsqrtf(x);
  if (!(x > 0.f && x <= 3.402823466e38f)) return r;
  const float h = x * r, l = fmaf(x, r, -h);
  const float e = fmaf(-l, r, fmaf(-h, r, 1.f));
  return fmaf(0.5f * r, e, r);
}

// Lane `part` of a row's group holds elements 8 part .. 8 part + 7. Writes them to
// `at` (this lane's 8 bytes of the page) and the row's scale byte. The whole warp
// calls it; rows with store == false only take part in the shuffles. Returns (with
// kNear) whether a value lies so near a border between two e4m3 values, or the row's
// largest so near the scale's, that the fp32 f may have it on the wrong side. What f can
// be off: 10 * 2^-24 relative from the norm's factor and the last products, and from a
// rotation 2^-24 of the product that is rounded before the sum, of which `product` is
// the lane's largest. Values are taken 12 * 2^-24 of themselves and 1.25 * 2^-24 of the
// product up and down (inexact; rows as they came are not); where both round alike the
// exact value does too.
template <int D, bool kNear>
__device__ __forceinline__ bool store_e4m3(const float (&f)[8], int part, uint8_t* at, uint8_t* scale,
                                           bool store, bool inexact = false, float product = 0.f) {
  float m = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m = fmaxf(m, fabsf(f[i]));
    bad |= !(fabsf(f[i]) <= 3.402823466e38f);
  }
  m = group_max<D / 8>(bad ? INFINITY : m);
  const bool finite = m <= 3.402823466e38f;
  const uint32_t byte = finite ? e4m3_scale_byte(m) : 255u;
  const float inv = finite ? e4m3_inv_scale(byte) : 0.f;
  float u[8], d[8];
  const float rel = inexact ? 0x1.8p-21f : 0.f;
  // (2^-23 of the scale for rows whose f are subnormal)
  const float least = inexact ? fmaf(product * inv, 0x1.4p-24f, 0x1p-23f) : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    u[i] = f[i] * inv;
    d[i] = kNear ? fmaf(fabsf(u[i]), rel, least) : 0.f;
  }
  auto pack = [&](float sign) {
    auto x = [&](int i) { return fmaf(d[i], sign, u[i]); };
    return make_uint2(e4m3x2(x(0), x(1)) | (e4m3x2(x(2), x(3)) << 16),
                      e4m3x2(x(4), x(5)) | (e4m3x2(x(6), x(7)) << 16));
  };
  uint2 q = pack(kNear ? 1.f : 0.f);
  bool near = false;
  if (kNear) {
    const uint2 down = pack(-1.f);
    const float top = m * inv;  // 224 to 448
    near = (((q.x ^ down.x) | (q.y ^ down.y)) & 0x7f7f7f7fu) != 0u  // (a zero's sign aside)
           || top > 448.f - 0x1p-10f || (top < 224.f + 0x1p-10f && byte > 1u);
    near = near && inexact && finite && store;
  }
  if (!finite) q.x = q.y = 0x7f7f7f7fu;
  if (!store) return false;
  *reinterpret_cast<uint2*>(at) = q;
  if (part == 0) *scale = static_cast<uint8_t>(byte);
  return near;
}

struct AppendArgs {
  const void *q, *k, *v;
  void* q_out;
  int64_t q_st, q_sh, o_st, o_sh, k_st, k_sh, v_st, v_sh;  // element strides
  const void *q_weight, *k_weight;
  const float *cos, *sin;
  int64_t table_stride, table_rows;
  const int32_t *token_start, *first_pos;
  const int32_t *page_table, *page_bounds;
  int64_t page_table_len;
  uint8_t *k_pool, *v_pool, *k_scale, *v_scale;
  int32_t* status;
  int64_t tokens;
  PageGeom g;
  float eps;
  int32_t R, Hq, Hk, half, interleaved;  // half: rotary_dim / 2, 0 without rotation
};

// What a group knows of its token.
struct Place {
  int64_t pos, page;
  int slot, err;  // err < 0: the token belongs to no request
};

// The places of a warp's tokens: lane group t % (32 / W) has token t. Every lane of
// the warp calls it.
template <int W>
__device__ __forceinline__ Place find_place(int64_t t, int64_t tokens, const int32_t* token_start,
                                            const int32_t* first_pos, int R, const int32_t* page_table,
                                            int64_t page_table_len, const int32_t* page_bounds,
                                            const PageGeom& g) {
  int r = R;
#pragma unroll
  for (int k = 0; k < 32 / W; ++k) {
    const int64_t tk = __shfl_sync(0xffffffffu, t, k * W);
    const int rk = find_request(token_start, R, tk);
    if ((threadIdx.x & 31) / W == k) r = rk;
  }
  Place p{0, 0, 0, -1};
  if (t >= tokens || r >= R) return p;
  const int64_t start = token_start[r];
  if (t < start) return p;
  const int64_t lo = page_bounds[r], n = page_bounds[r + 1] - lo;
  p.pos = static_cast<int64_t>(first_pos[r]) + (t - start);
  p.err = kStatusPosition;
  const int64_t index = p.pos / g.page_size;
  if (p.pos < 0 || index >= n || lo < 0 || lo + index >= page_table_len) return p;
  p.page = page_table[lo + index];
  p.slot = static_cast<int>(p.pos % g.page_size);
  p.err = p.page < 0 || p.page >= g.num_pages ? kStatusPage : 0;
  return p;
}

__device__ __forceinline__ uint64_t warp_or(uint64_t x) {
  const uint32_t lo = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(x));
  const uint32_t hi = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(x >> 32));
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// A lane's eight elements of a k row once more, in 64 bits, with the scale. The whole
// warp calls it, after the other rows, and only rows with ok are written: what a token's
// rows become is theirs alone. About one row in 230 needs it, which costs 1 us of the 77
// of 13,000 tokens; in the rows' own loop its registers would cost all of them (116 us
// for the same tokens written and read back, 93 so).
template <typename T, int D>
__device__ __forceinline__ void exact_row(bool ok, const T* row, const T* weight, const float* cos, const float* sin,
                                          int half, int interleaved, float eps, uint8_t* at, uint8_t* scale) {
  constexpr int W = D / 8;
  const int lane = threadIdx.x & 31, part = lane % W, rot_lanes = half / 4;
  const bool rotated = part < rot_lanes, first = part < rot_lanes / 2;
  const int from = rotated ? (first ? lane + rot_lanes / 2 : lane - rot_lanes / 2) : lane;
  float g[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  Vec8<T> in;
  if (ok) {
    in.load(row);
    in.get(g);
  }
  double root = 1.;
  if (weight) {
    double ss = 0.;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fma(static_cast<double>(g[i]), static_cast<double>(g[i]), ss);
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    ss = ss * (1. / D) + static_cast<double>(eps);
    root = rsqrtf(static_cast<float>(ss));  // to 2^-22, and 2^-43 and 2^-52 after a step
    root *= fma(-0.5 * ss * root, root, 1.5);
    root *= fma(-0.5 * ss * root, root, 1.5);
    float w[8];
    in.load(weight);
    in.get(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] *= w[i];  // exact
  }
  double y[8], top = 0.;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = interleaved ? g[i ^ 1] : __shfl_sync(0xffffffffu, g[i], from);
    y[i] = g[i];
    if (cos) {
      const int col = interleaved ? part * 4 + i / 2 : part * 8 - (first ? 0 : half) + i;
      const double s = sin[col];
      y[i] = y[i] * cos[col] + static_cast<double>(x) * ((interleaved ? i % 2 == 0 : first) ? -s : s);
    }
    y[i] *= root;
    top = fmax(top, fabs(y[i]));
  }
  // rounded up to fp32: above the scale's border, an fp32 value, where the exact one is
  const uint32_t byte = e4m3_scale_byte(group_max<W>(__double2float_ru(top)));
  uint32_t q[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] *= e4m3_inv_scale(byte);
    float u = static_cast<float>(y[i]);
    // not onto a border from beside it: borders have four bits at most behind the first
    if ((__float_as_uint(u) & 0x7ffffu) == 0u && y[i] != u && u != 0.f)
      u = __uint_as_float(__float_as_uint(u) + ((y[i] > u) == (u > 0.f) ? 1u : -1u));
    q[i / 4] |= (e4m3x2(u, 0.f) & 255u) << (i % 4 * 8);
  }
  if (!ok) return;
  *reinterpret_cast<uint2*>(at) = make_uint2(q[0], q[1]);
  if (part == 0) *scale = static_cast<uint8_t>(byte);
}

template <typename T, int D, bool Q8>
__global__ void __launch_bounds__(kThreads, 3) append_kernel(const AppendArgs a, const int rows_per_block) {
  constexpr int W = D / 8;               // lanes of a row
  constexpr int kGroups = kThreads / W;  // tokens of a block
  const int part = threadIdx.x % W;
  const int64_t t = blockIdx.x * static_cast<int64_t>(kGroups) + threadIdx.x / W;
  const int rows = a.Hq + 2 * a.Hk;
  const int row0 = blockIdx.y * rows_per_block, row1 = min(rows, row0 + rows_per_block);
  grid_dep_wait();
  Place p = find_place<W>(t, a.tokens, a.token_start, a.first_pos, a.R, a.page_table, a.page_table_len,
                            a.page_bounds, a.g);
  if (p.err == 0 && a.half && p.pos >= a.table_rows) p.err = kStatusTable;
  if (p.err > 0 && part == 0 && row0 == 0) report(a.status, p.err);
  const bool ok = p.err == 0;  // else the token's rows are not written at all
  if (!__any_sync(0xffffffffu, ok)) return;
  // this lane's cos and sin: columns of its 8 elements' pairs
  float c[8], s[8];
  const int rot_lanes = a.half / 4;  // lanes that hold rotated elements
  const bool rotated = part < rot_lanes, first = part < rot_lanes / 2;
  const int lane = threadIdx.x & 31;
  const int from = rotated ? (first ? lane + rot_lanes / 2 : lane - rot_lanes / 2) : lane;
  if (rotated && ok && row0 < a.Hq + a.Hk) {
    const float* cr = a.cos + p.pos * a.table_stride;
    const float* sr = a.sin + p.pos * a.table_stride;
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[2 * i] = c[2 * i + 1] = __ldg(cr + part * 4 + i);
        s[2 * i + 1] = __ldg(sr + part * 4 + i);
        s[2 * i] = -s[2 * i + 1];
      }
    } else {
      const int col = part * 8 - (first ? 0 : a.half);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = __ldg(cr + col + i);
        s[i] = __ldg(sr + col + i);
        if (first) s[i] = -s[i];
      }
    }
  }
  // heads h0 .. h1 - 1 of q (0), k (1) or v (2): four rows' loads, then their work
  constexpr int kAhead = sizeof(T) == 4 ? 2 : 4;
  uint64_t redo = 0;  // (8-bit) k heads with a value of this lane near a border; bit 63: 63 on
  auto heads = [&](auto kind, int h0, int h1, const void* src_p, int64_t st, int64_t sh, const void* weight,
                   uint8_t* dst, int64_t dst_sh, uint8_t* scale) {
    constexpr int kKind = decltype(kind)::value;
    if (h0 >= h1) return;
    const T* src = static_cast<const T*>(src_p) + t * st + h0 * sh + part * 8;
    dst += h0 * dst_sh;
    if (Q8 && kKind != 0) scale += h0 * a.g.scale_head;
    float w[8];
    if (kKind != 2 && weight) {
      Vec8<T> wv;
      wv.load(static_cast<const T*>(weight) + part * 8);
      wv.get(w);
    }
    for (int h = h0; h < h1; h += kAhead) {
      Vec8<T> in[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (ok && h + u < h1) in[u].load(src + u * sh);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (h + u >= h1) break;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (ok) in[u].get(f);
        float inv = 1.f, product = 0.f;
        if (kKind != 2 && weight) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
          inv = exact_rsqrt(group_sum<W>(ss) * (1.f / D) + a.eps);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] *= w[i];
        }
        if (kKind != 2 && a.half) {
          float x[8];  // the partners
          if (a.interleaved) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = f[i ^ 1];
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __shfl_sync(0xffffffffu, f[i], from);
          }
          if (rotated) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float xs = x[i] * s[i];
              f[i] = fmaf(f[i], c[i], xs);
              if (Q8 && kKind == 1) product = fmaxf(product, fabsf(xs));
            }
          }
        }
        // last, as one rounding (x w is exact in fp32 for 16-bit types)
        if (kKind != 2 && weight) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] *= inv;
        }
        if (Q8 && kKind != 0) {
          if (store_e4m3<D, kKind == 1>(f, part, dst + u * dst_sh, scale + u * a.g.scale_head, ok,
                                            a.half || a.k_weight, product * inv))
            redo |= 1ull << min(h + u, 63);
        } else if (ok) {
          Vec8<T> v;
          v.set(f);
          v.store(dst + u * dst_sh);
        }
      }
      src += kAhead * sh;
      dst += kAhead * dst_sh;
      if (Q8 && kKind != 0) scale += kAhead * a.g.scale_head;
    }
  };
  // this lane's part of the token's row of head 0 in a page
  const int64_t at = page_chunk(a.g, p.page, 0, p.slot, Q8 ? part >> 1 : part * static_cast<int>(sizeof(T)) / 2,
                                (Q8 ? 1 : static_cast<int>(sizeof(T))) * D / 16) + (Q8 ? (part & 1) * 8 : 0);
  const int64_t sat = Q8 ? p.page * a.g.scale_page + p.slot : 0;
  heads(std::integral_constant<int, 0>(), row0, min(row1, a.Hq), a.q, a.q_st, a.q_sh, a.q_weight,
        static_cast<uint8_t*>(a.q_out) + (t * a.o_st + part * 8) * static_cast<int64_t>(sizeof(T)),
        a.o_sh * static_cast<int64_t>(sizeof(T)), nullptr);
  const int k0 = max(row0, a.Hq) - a.Hq, k1 = min(row1, a.Hq + a.Hk) - a.Hq;
  heads(std::integral_constant<int, 1>(), k0, k1, a.k, a.k_st, a.k_sh, a.k_weight, a.k_pool + at, a.g.stride_head,
        a.k_scale + sat);
  heads(std::integral_constant<int, 2>(), max(row0, a.Hq + a.Hk) - a.Hq - a.Hk, row1 - a.Hq - a.Hk, a.v, a.v_st,
        a.v_sh, nullptr, a.v_pool + at, a.g.stride_head, a.v_scale + sat);
  if constexpr (Q8) {
    if (!a.half && !a.k_weight) return;  // k itself, exact
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) redo |= __shfl_xor_sync(0xffffffffu, redo, o);  // the row's
    const uint64_t any = warp_or(redo);
    for (int h = k0; h < k1; ++h) {
      if (!(any >> min(h, 63) & 1)) continue;
      exact_row<T, D>(redo >> min(h, 63) & 1, static_cast<const T*>(a.k) + t * a.k_st + h * a.k_sh + part * 8,
                      a.k_weight ? static_cast<const T*>(a.k_weight) + part * 8 : nullptr,
                      rotated && ok ? a.cos + p.pos * a.table_stride : nullptr,
                      rotated && ok ? a.sin + p.pos * a.table_stride : nullptr, a.half, a.interleaved, a.eps,
                      a.k_pool + at + h * a.g.stride_head, a.k_scale + sat + h * a.g.scale_head);
    }
  }
}

// Heads of a token that one block takes: all of them when there are tokens enough
// for four blocks on each SM, else as few as fill them.
int rows_per_block(int64_t token_blocks, int rows) {
  const int64_t want = static_cast<int64_t>(current_sm_count()) * 4;
  int64_t splits = (want + token_blocks - 1) / token_blocks;
  if (splits > rows) splits = rows;
  return static_cast<int>((rows + splits - 1) / splits);
}

struct ReadArgs {
  const uint8_t *k_pool, *v_pool, *k_scale, *v_scale;
  void *k_out, *v_out;
  int64_t ko_st, ko_sh, vo_st, vo_sh;  // element strides
  const int32_t *token_start, *first_pos, *page_table, *page_bounds;
  int64_t page_table_len;
  int32_t* status;
  int64_t tokens;
  PageGeom g;
  int32_t R, Hk;
};

template <typename T, int D, bool Q8>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadArgs a, const int rows_per_block) {
  constexpr int W = D / 8;
  constexpr int kGroups = kThreads / W;
  constexpr int kAhead = 8;  // rows in flight
  const int part = threadIdx.x % W;
  const int64_t t = blockIdx.x * static_cast<int64_t>(kGroups) + threadIdx.x / W;
  const int row0 = blockIdx.y * rows_per_block, row1 = min(2 * a.Hk, row0 + rows_per_block);
  grid_dep_wait();
  const Place p =
      find_place<W>(t, a.tokens, a.token_start, a.first_pos, a.R, a.page_table, a.page_table_len,
                            a.page_bounds, a.g);
  if (p.err > 0 && part == 0 && row0 == 0) report(a.status, p.err);
  if (p.err != 0) return;
  for (int r0 = row0; r0 < row1; r0 += kAhead) {
    Vec8<T> x[kAhead];
    uint2 q[kAhead];
    uint32_t byte[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int row = r0 + u;
      if (row >= row1) break;
      const bool is_k = row < a.Hk;
      const int head = is_k ? row : row - a.Hk;
      const uint8_t* pool = is_k ? a.k_pool : a.v_pool;
      if (Q8) {
        q[u] = *reinterpret_cast<const uint2*>(pool + page_chunk(a.g, p.page, head, p.slot, part >> 1, D / 16) +
                                               (part & 1) * 8);
        byte[u] = (is_k ? a.k_scale : a.v_scale)[p.page * a.g.scale_page + head * a.g.scale_head + p.slot];
      } else {
        x[u].load(pool + (sizeof(T) == 2 ? page_chunk(a.g, p.page, head, p.slot, part, D / 8)
                                         : page_chunk(a.g, p.page, head, p.slot, part * 2, D / 4)));
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int row = r0 + u;
      if (row >= row1) break;
      const bool is_k = row < a.Hk;
      const int head = is_k ? row : row - a.Hk;
      if (Q8) {
        const float sc = e4m3_scale(byte[u]);
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = e4m3x2_to_f((i < 2 ? q[u].x : q[u].y) >> ((i & 1) * 16));
          f[2 * i] = v.x * sc;
          f[2 * i + 1] = v.y * sc;
        }
        x[u].set(f);
      }
      x[u].store(static_cast<T*>(is_k ? a.k_out : a.v_out) + t * (is_k ? a.ko_st : a.vo_st) +
                 head * (is_k ? a.ko_sh : a.vo_sh) + part * 8);
    }
  }
}

// The 8-bit pages of page-table entries [0, entries) as bf16 UMMA pages, entry e at
// page e: a 16-byte core-matrix row becomes two (exact, see paged.cuh). For attention
// that goes over the same keys many times. 32k positions of 8 heads of 128, 201 MB moved,
// 30 us = 1.0 of a plain copy's rate (the write stays in L2).
__global__ void __launch_bounds__(kThreads)
    widen_kernel(const uint8_t* k_pool, const uint8_t* v_pool, const uint8_t* k_scale, const uint8_t* v_scale,
                 const PageGeom g, const int32_t* __restrict__ page_table, int64_t entries, int Hk, int D,
                 uint8_t* k_out, uint8_t* v_out) {
  grid_dep_wait();
  const int chunks = D;  // 16-byte chunks of a (page, head) block of 16 * D bytes
  const int64_t total = entries * Hk * chunks;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int x = static_cast<int>(i % chunks);
    const int64_t eh = i / chunks;
    const int h = static_cast<int>(eh % Hk);
    const int64_t e = eh / Hk;
    int64_t page = page_table[e];
    page = page < 0 ? 0 : (page >= g.num_pages ? g.num_pages - 1 : page);
    const int row_chunks = D / 16;
    const int row = x / (8 * row_chunks) * 8 + x % 8, c = x / 8 % row_chunks;
    const int64_t src = page * g.stride_page + h * g.stride_head + x * 16;
    const int64_t sc = page * g.scale_page + h * g.scale_head + row;
    const int64_t dst = eh * (32 * D) + ((row >> 3) * (D / 8) + 2 * c) * 128 + (row & 7) * 16;
    const uint4 in[2] = {*reinterpret_cast<const uint4*>(k_pool + src), *reinterpret_cast<const uint4*>(v_pool + src)};
    const float f[2] = {e4m3_scale(k_scale[sc]), e4m3_scale(v_scale[sc])};
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint32_t w[4] = {in[kv].x, in[kv].y, in[kv].z, in[kv].w};
      uint32_t o[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 lo = e4m3x2_to_f(w[j]), hi = e4m3x2_to_f(w[j] >> 16);
        o[2 * j] = pack_bf16x2(lo.x * f[kv], lo.y * f[kv]);
        o[2 * j + 1] = pack_bf16x2(hi.x * f[kv], hi.y * f[kv]);
      }
      uint8_t* at = (kv ? v_out : k_out) + dst;
      *reinterpret_cast<uint4*>(at) = make_uint4(o[0], o[1], o[2], o[3]);
      *reinterpret_cast<uint4*>(at + 128) = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

struct CommitArgs8 {
  const void* const* layer_ptrs;  // [L][6] {new_k, new_v, cache_k, cache_v, k_scale, v_scale}
  int64_t n_sr, n_sb, n_sh, n_st;
  const int32_t *page_table, *page_bounds, *accept_results, *cache_lens;
  int64_t page_table_len;
  int32_t* status;
  PageGeom g;
  int32_t R, L, Hk, TB;
};

// One group per (request, layer, K | V, head): the accepted rows one after another. A few
// rows for each layer; bound by latency.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) commit_e4m3_kernel(const CommitArgs8 a) {
  constexpr int W = D / 8;
  const int part = threadIdx.x % W;
  grid_dep_wait();
  const int64_t total = static_cast<int64_t>(a.R) * a.L * 2 * a.Hk;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / W);
  const int64_t first = blockIdx.x * static_cast<int64_t>(kThreads / W) + threadIdx.x / W;
  // every group of a warp runs the same number of rounds (the shuffles are the whole warp's)
  for (int64_t i0 = 0; i0 < total; i0 += step) {
    const int64_t id = i0 + first;
    const bool live = id < total;
    const int64_t x = live ? id : 0;
    const int h = static_cast<int>(x % a.Hk);
    const int kv = static_cast<int>(x / a.Hk % 2);
    const int l = static_cast<int>(x / a.Hk / 2 % a.L);
    const int r = static_cast<int>(x / a.Hk / 2 / a.L);
    const int acc = live ? min(max(a.accept_results[2 * r], 0), a.TB) : 0;
    const int branch = a.accept_results[2 * r + 1];
    const int64_t len = a.cache_lens[r];
    const int64_t lo = a.page_bounds[r], n = a.page_bounds[r + 1] - lo;
    const T* src = static_cast<const T*>(a.layer_ptrs[6 * l + kv]) + r * a.n_sr + branch * a.n_sb +
                   h * a.n_sh + part * 8;
    uint8_t* pool = static_cast<uint8_t*>(const_cast<void*>(a.layer_ptrs[6 * l + 2 + kv]));
    uint8_t* scale = static_cast<uint8_t*>(const_cast<void*>(a.layer_ptrs[6 * l + 4 + kv]));
    int most = acc;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    for (int t = 0; t < most; ++t) {
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      bool ok = t < acc;
      int64_t page = 0;
      const int64_t pos = len + t;
      if (ok) {
        int err = 0;
        if (pos < 0 || pos / 16 >= n || lo < 0 || lo + pos / 16 >= a.page_table_len) {
          err = kStatusPosition;
        } else {
          page = a.page_table[lo + pos / 16];
          if (page < 0 || page >= a.g.num_pages) err = kStatusPage;
        }
        if (err) {
          ok = false;
          if (part == 0) report(a.status, err);
        } else {
          Vec8<T> v;
          v.load(src + t * a.n_st);
          v.get(f);
        }
      }
      const int slot = static_cast<int>(pos & 15);
      store_e4m3<D, false>(f, part, pool + page_chunk(a.g, page, h, slot, part >> 1, D / 16) + (part & 1) * 8,
                    scale + page * a.g.scale_page + h * a.g.scale_head + slot, ok);
    }
  }
}

bool aligned_rows(int64_t a, int64_t b) { return a % 8 == 0 && b % 8 == 0; }

}  // namespace

int launch_widen(const uint8_t* k_pool, const uint8_t* v_pool, const uint8_t* k_scale, const uint8_t* v_scale,
                 const PageGeom& g, const int32_t* page_table, int64_t entries, int num_kv_heads, int head_dim,
                 void* k_out, void* v_out, void* stream) {
  const int64_t total = entries * num_kv_heads * head_dim;
  const int64_t blocks = (total + kThreads - 1) / kThreads, most = static_cast<int64_t>(current_sm_count()) * 32;
  return launch_pdl(widen_kernel, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(kThreads), 0,
                    static_cast<cudaStream_t>(stream), "widen_kernel", k_pool, v_pool, k_scale, v_scale, g,
                    page_table, entries, num_kv_heads, head_dim, static_cast<uint8_t*>(k_out),
                    static_cast<uint8_t*>(v_out));
}
}  // namespace d2sd

extern "C" int d2sd_append_kv(
    const void* q, int64_t q_stride_token, int64_t q_stride_head, void* q_out,
    int64_t q_out_stride_token, int64_t q_out_stride_head, int32_t num_qo_heads, const void* k,
    int64_t k_stride_token, int64_t k_stride_head, const void* v, int64_t v_stride_token,
    int64_t v_stride_head, int32_t num_kv_heads, int64_t num_tokens, int32_t head_dim, int32_t dtype,
    const void* q_weight, const void* k_weight, float eps, const float* cos_table,
    const float* sin_table, int64_t table_stride, int64_t table_rows, int32_t rotary_dim,
    int32_t interleaved, const int32_t* token_start, const int32_t* first_pos, int32_t num_requests,
    void* k_pool, void* v_pool, int64_t cache_stride_page, int64_t cache_stride_slot,
    int64_t cache_stride_head, int32_t page_size, int64_t num_pages, int32_t cache_format,
    void* k_scale, void* v_scale, int64_t scale_stride_page, int64_t scale_stride_head,
    const int32_t* page_table, int64_t page_table_len, const int32_t* page_bounds, int32_t* status,
    void* stream) {
  using namespace d2sd;
  const char* const w = "d2sd_append_kv";
  if (num_tokens < 0 || num_requests < 0 || num_kv_heads <= 0 || num_qo_heads < 0 || !token_start ||
      !first_pos || !k_pool || !v_pool || !page_table || page_table_len < 0 || !page_bounds ||
      (num_tokens > 0 && (!k || !v || (num_qo_heads > 0 && (!q || !q_out)))))
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": invalid argument");
  if (num_tokens == 0 || num_requests == 0) return D2SD_OK;
  if (head_dim != 64 && head_dim != 128)
    return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": head_dim must be 64 or 128");
  if (dtype != D2SD_DTYPE_BF16 && dtype != D2SD_DTYPE_F16 && dtype != D2SD_DTYPE_F32)
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": unknown dtype");
  const bool scaled = k_scale != nullptr;
  if (scaled != (v_scale != nullptr))
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": k_scale and v_scale go together");
  if ((q_weight != nullptr) != (k_weight != nullptr) && num_qo_heads > 0)
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": q_weight and k_weight go together");
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16 != 0)
    return fail(D2SD_ERR_UNSUPPORTED,
                std::string(w) + ": rotary_dim must be a multiple of 16 up to head_dim");
  if (rotary_dim > 0 && (!cos_table || !sin_table || table_rows <= 0 || table_stride < rotary_dim / 2))
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": the rotary tables do not fit rotary_dim");
  const int elem = dtype == D2SD_DTYPE_F32 ? 4 : 2;
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_pool) || !aligned16(v_pool) ||
      !aligned16(q_weight) || !aligned16(k_weight) || !aligned_rows(k_stride_token, k_stride_head) ||
      !aligned_rows(v_stride_token, v_stride_head) ||
      (num_qo_heads > 0 && (!aligned16(q) || !aligned16(q_out) ||
                            !aligned_rows(q_stride_token, q_stride_head) ||
                            !aligned_rows(q_out_stride_token, q_out_stride_head))))
    return fail(D2SD_ERR_INVALID_ARGUMENT,
                std::string(w) + ": rows must be 16-byte aligned, strides multiples of 8");
  AppendArgs a{};
  int rc = make_page_geom(&a.g, w, head_dim, scaled ? 1 : elem, cache_stride_page, cache_stride_slot,
                          cache_stride_head, page_size, num_pages, cache_format, scaled,
                          scale_stride_page, scale_stride_head);
  if (rc) return rc;
  if (scaled && elem != 2)
    return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": 8-bit rows are written from 16-bit values");
  a.q = q, a.k = k, a.v = v, a.q_out = q_out;
  a.q_st = q_stride_token, a.q_sh = q_stride_head, a.o_st = q_out_stride_token,
  a.o_sh = q_out_stride_head, a.k_st = k_stride_token, a.k_sh = k_stride_head, a.v_st = v_stride_token,
  a.v_sh = v_stride_head;
  a.q_weight = q_weight, a.k_weight = k_weight;
  a.cos = cos_table, a.sin = sin_table, a.table_stride = table_stride, a.table_rows = table_rows;
  a.token_start = token_start, a.first_pos = first_pos;
  a.page_table = page_table, a.page_table_len = page_table_len, a.page_bounds = page_bounds;
  a.k_pool = static_cast<uint8_t*>(k_pool), a.v_pool = static_cast<uint8_t*>(v_pool);
  a.k_scale = static_cast<uint8_t*>(k_scale), a.v_scale = static_cast<uint8_t*>(v_scale);
  a.status = status;
  a.tokens = num_tokens;
  a.eps = eps;
  a.R = num_requests, a.Hq = num_qo_heads, a.Hk = num_kv_heads, a.half = rotary_dim / 2,
  a.interleaved = interleaved;
  const int rows = num_qo_heads + 2 * num_kv_heads;
  const int64_t per = kThreads / (head_dim / 8), blocks = (num_tokens + per - 1) / per;
  if (blocks > 0x7fffffff) return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": too many tokens");
  const int rpb = rows_per_block(blocks, rows);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((rows + rpb - 1) / rpb));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel) { return launch_pdl(kernel, grid, dim3(kThreads), 0, st, w, a, rpb); };
  if (dtype == D2SD_DTYPE_F32) return head_dim == 128 ? go(append_kernel<float, 128, false>) : go(append_kernel<float, 64, false>);
  if (dtype == D2SD_DTYPE_BF16) {
    if (scaled) return head_dim == 128 ? go(append_kernel<__nv_bfloat16, 128, true>) : go(append_kernel<__nv_bfloat16, 64, true>);
    return head_dim == 128 ? go(append_kernel<__nv_bfloat16, 128, false>) : go(append_kernel<__nv_bfloat16, 64, false>);
  }
  if (scaled) return head_dim == 128 ? go(append_kernel<__half, 128, true>) : go(append_kernel<__half, 64, true>);
  return head_dim == 128 ? go(append_kernel<__half, 128, false>) : go(append_kernel<__half, 64, false>);
}

extern "C" int d2sd_read_kv(const void* k_pool, const void* v_pool, int64_t cache_stride_page,
                            int64_t cache_stride_slot, int64_t cache_stride_head, int32_t page_size,
                            int64_t num_pages, int32_t cache_format, const void* k_scale,
                            const void* v_scale, int64_t scale_stride_page, int64_t scale_stride_head,
                            const int32_t* page_table, int64_t page_table_len,
                            const int32_t* page_bounds, const int32_t* token_start, const int32_t* first_pos, int32_t num_requests,
                            int64_t num_tokens, int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                            void* k_out, int64_t k_out_stride_token, int64_t k_out_stride_head,
                            void* v_out, int64_t v_out_stride_token, int64_t v_out_stride_head,
                            int32_t* status, void* stream) {
  using namespace d2sd;
  const char* const w = "d2sd_read_kv";
  if (num_tokens < 0 || num_requests < 0 || num_kv_heads <= 0 || !token_start || !first_pos || !k_pool ||
      !v_pool || !page_table || page_table_len < 0 || !page_bounds || (num_tokens > 0 && (!k_out || !v_out)))
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": invalid argument");
  if (num_tokens == 0 || num_requests == 0) return D2SD_OK;
  if (head_dim != 64 && head_dim != 128)
    return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": head_dim must be 64 or 128");
  if (dtype != D2SD_DTYPE_BF16 && dtype != D2SD_DTYPE_F16 && dtype != D2SD_DTYPE_F32)
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": unknown dtype");
  const bool scaled = k_scale != nullptr;
  if (scaled != (v_scale != nullptr))
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": k_scale and v_scale go together");
  if (!aligned16(k_pool) || !aligned16(v_pool) || !aligned16(k_out) || !aligned16(v_out) ||
      !aligned_rows(k_out_stride_token, k_out_stride_head) ||
      !aligned_rows(v_out_stride_token, v_out_stride_head))
    return fail(D2SD_ERR_INVALID_ARGUMENT,
                std::string(w) + ": rows must be 16-byte aligned, strides multiples of 8");
  const int elem = dtype == D2SD_DTYPE_F32 ? 4 : 2;
  if (scaled && elem != 2)
    return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": 8-bit rows are read into 16-bit values");
  ReadArgs a{};
  int rc = make_page_geom(&a.g, w, head_dim, scaled ? 1 : elem, cache_stride_page, cache_stride_slot,
                          cache_stride_head, page_size, num_pages, cache_format, scaled,
                          scale_stride_page, scale_stride_head);
  if (rc) return rc;
  a.k_pool = static_cast<const uint8_t*>(k_pool), a.v_pool = static_cast<const uint8_t*>(v_pool);
  a.k_scale = static_cast<const uint8_t*>(k_scale), a.v_scale = static_cast<const uint8_t*>(v_scale);
  a.k_out = k_out, a.v_out = v_out;
  a.ko_st = k_out_stride_token, a.ko_sh = k_out_stride_head, a.vo_st = v_out_stride_token,
  a.vo_sh = v_out_stride_head;
  a.token_start = token_start, a.first_pos = first_pos, a.page_table = page_table,
  a.page_table_len = page_table_len, a.page_bounds = page_bounds;
  a.status = status;
  a.tokens = num_tokens;
  a.R = num_requests, a.Hk = num_kv_heads;
  const int rows = 2 * num_kv_heads;
  const int64_t per = kThreads / (head_dim / 8), blocks = (num_tokens + per - 1) / per;
  if (blocks > 0x7fffffff) return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": too many tokens");
  const int rpb = rows_per_block(blocks, rows);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((rows + rpb - 1) / rpb));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel) { return launch_pdl(kernel, grid, dim3(kThreads), 0, st, w, a, rpb); };
  if (dtype == D2SD_DTYPE_F32) return head_dim == 128 ? go(read_kernel<float, 128, false>) : go(read_kernel<float, 64, false>);
  if (dtype == D2SD_DTYPE_BF16) {
    if (scaled) return head_dim == 128 ? go(read_kernel<__nv_bfloat16, 128, true>) : go(read_kernel<__nv_bfloat16, 64, true>);
    return head_dim == 128 ? go(read_kernel<__nv_bfloat16, 128, false>) : go(read_kernel<__nv_bfloat16, 64, false>);
  }
  if (scaled) return head_dim == 128 ? go(read_kernel<__half, 128, true>) : go(read_kernel<__half, 64, true>);
  return head_dim == 128 ? go(read_kernel<__half, 128, false>) : go(read_kernel<__half, 64, false>);
}

extern "C" int d2sd_commit_kv_e4m3(const void* const* layer_ptrs, int32_t num_layers,
                                   int32_t num_requests, int32_t num_kv_heads, int32_t head_dim,
                                   int32_t dtype, int32_t block_len, int64_t new_stride_request,
                                   int64_t new_stride_branch, int64_t new_stride_head,
                                   int64_t new_stride_token, int64_t cache_stride_page,
                                   int64_t cache_stride_head, int64_t num_pages,
                                   int64_t scale_stride_page, int64_t scale_stride_head,
                                   const int32_t* page_table, int64_t page_table_len,
                                   const int32_t* page_bounds, const int32_t* accept_results,
                                   const int32_t* cache_lens,
                                   int32_t* status, void* stream) {
  using namespace d2sd;
  const char* const w = "d2sd_commit_kv_e4m3";
  if (!layer_ptrs || num_layers <= 0 || num_requests <= 0 || num_kv_heads <= 0 || block_len <= 0 ||
      !page_table || page_table_len < 0 || !page_bounds || !accept_results || !cache_lens)
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": invalid argument");
  if (head_dim != 64 && head_dim != 128)
    return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": head_dim must be 64 or 128");
  if (dtype != D2SD_DTYPE_BF16 && dtype != D2SD_DTYPE_F16)
    return fail(D2SD_ERR_UNSUPPORTED, std::string(w) + ": 8-bit rows are written from 16-bit values");
  if (!aligned_rows(new_stride_request, new_stride_branch) ||
      !aligned_rows(new_stride_head, new_stride_token))
    return fail(D2SD_ERR_INVALID_ARGUMENT, std::string(w) + ": strides must be multiples of 8");
  CommitArgs8 a{};
  int rc = make_page_geom(&a.g, w, head_dim, 1, cache_stride_page, 0, cache_stride_head, 16, num_pages,
                          D2SD_KV_UMMA_PAGES, true, scale_stride_page, scale_stride_head);
  if (rc) return rc;
  a.layer_ptrs = layer_ptrs;
  a.n_sr = new_stride_request, a.n_sb = new_stride_branch, a.n_sh = new_stride_head,
  a.n_st = new_stride_token;
  a.page_table = page_table, a.page_table_len = page_table_len, a.page_bounds = page_bounds,
  a.accept_results = accept_results,
  a.cache_lens = cache_lens, a.status = status;
  a.R = num_requests, a.L = num_layers, a.Hk = num_kv_heads, a.TB = block_len;
  const int64_t groups = static_cast<int64_t>(num_requests) * num_layers * 2 * num_kv_heads;
  const int64_t per = kThreads / (head_dim / 8);
  int64_t blocks = (groups + per - 1) / per;
  const int64_t cap = static_cast<int64_t>(current_sm_count()) * 8;
  if (blocks > cap) blocks = cap;
  const dim3 grid(static_cast<unsigned>(blocks));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel) { return launch_pdl(kernel, grid, dim3(kThreads), 0, st, w, a); };
  if (dtype == D2SD_DTYPE_BF16)
    return head_dim == 128 ? go(commit_e4m3_kernel<__nv_bfloat16, 128>) : go(commit_e4m3_kernel<__nv_bfloat16, 64>);
  return head_dim == 128 ? go(commit_e4m3_kernel<__half, 128>) : go(commit_e4m3_kernel<__half, 64>);
}
