// Addressing of the paged cache and its 8-bit rows, shared by the kernels that
// write it, read it back and attend it.
//
// 8-bit rows. A row x of one (token, head) is held as e4m3 values and one scale
// byte: e = the smallest integer >= -126 with amax|x| <= 448 * 2^e, the byte is
// e + 127, and element i is the e4m3 value nearest to x_i * 2^-e (ties to even).
// The scale is a power of two because a finer one buys nothing (e4m3 is a
// floating format: its relative step is 2^-3 of the binade wherever a value
// lies), and it makes the division and every value read back exact (4 bits of
// significand fit bf16). That rounding, 2^-4 of the value at most, is the one
// choice of precision here; the row's maximum and the division are in fp32.
// A row that holds a NaN or an infinity gets the byte 255 and NaN values, and
// reads back as NaN. A byte of 0 (a pool that was never written) reads as 0.
#pragma once

#include "common.cuh"

namespace d2sd {

constexpr int kStatusPosition = 4;  // a position outside the request's pages
constexpr int kStatusPage = 5;      // a page id outside the pool
constexpr int kStatusTable = 6;     // a position outside the rotary tables

// The smallest code of a launch stays, whichever token reports first.
__device__ __forceinline__ void report(int32_t* status, int code) {
  if (status && atomicCAS(status, 0, code) > code) atomicMin(status, code);
}

// One pool (K and V alike): byte strides, so 8- and 16-bit values share it.
struct PageGeom {
  int64_t stride_page, stride_slot, stride_head;  // bytes
  int64_t scale_page, scale_head;                 // bytes of the scale pool
  int64_t num_pages;
  int32_t page_size;
  int32_t umma;  // core-matrix pages (16 slots) instead of rows
};

// Byte offset of 16-byte chunk c of slot s of (page, head).
__device__ __forceinline__ int64_t page_chunk(const PageGeom& g, int64_t page, int head, int s, int c,
                                              int chunks) {
  const int64_t base = page * g.stride_page + head * g.stride_head;
  return base + (g.umma ? static_cast<int64_t>(((s >> 3) * chunks + c) * 128 + (s & 7) * 16)
                        : s * g.stride_slot + c * 16);
}

// The scale exponent byte of a row with largest magnitude amax (finite).
__device__ __forceinline__ uint32_t e4m3_scale_byte(float amax) {
  // amax = m * 2^x, 1 <= m < 2 (x from the exponent field; a subnormal amax
  // ends at the smallest exponent). 448 = 1.75 * 2^8.
  const uint32_t bits = __float_as_uint(amax);
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(max(e, 1));
}
__device__ __forceinline__ float e4m3_scale(uint32_t byte) {  // 2^e; NaN for 255
  return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}
__device__ __forceinline__ float e4m3_inv_scale(uint32_t byte) {  // 2^-e, byte 1..253
  return __uint_as_float((254u - byte) << 23);
}
// Two fp32 values to e4m3 (round to nearest even), lo in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two e4m3 values (low 16 bits) to fp32.
__device__ __forceinline__ float2 e4m3x2_to_f(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(v)));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// Request of token t: the number of requests whose end is at or before t, found
// by the whole warp (token_start [R + 1] ascending). A t at or behind the last
// end gives R.
__device__ __forceinline__ int find_request(const int32_t* __restrict__ token_start, int R, int64_t t) {
  const int lane = threadIdx.x & 31;
  int r = 0;
  for (int base = 0; base < R; base += 32) {
    const bool before = base + lane < R && token_start[base + lane + 1] <= t;
    r += __popc(__ballot_sync(0xffffffffu, before));
  }
  return r;
}

// Eight consecutive elements of a row in fp32, loaded and stored as vectors.
template <typename T>
struct Vec8 {
  uint4 v;
  __device__ __forceinline__ void load(const void* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(void* p) const { *reinterpret_cast<uint4*>(p) = v; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Num<T>::to_f(e[i]);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = Num<T>::from_f(f[i]);
  }
};
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const void* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void store(void* p) const {
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    a = make_float4(f[0], f[1], f[2], f[3]);
    b = make_float4(f[4], f[5], f[6], f[7]);
  }
};

// Widen 8-bit pages into bf16 ones, one for each page-table entry (paged_kv.cu).
int launch_widen(const uint8_t* k_pool, const uint8_t* v_pool, const uint8_t* k_scale, const uint8_t* v_scale,
                 const PageGeom& g, const int32_t* page_table, int64_t entries, int num_kv_heads, int head_dim,
                 void* k_out, void* v_out, void* stream);

// Fill a PageGeom from the C arguments (strides in elements), or report what is
// wrong with them. elem is the bytes of a cached value.
int make_page_geom(PageGeom* g, const char* what, int32_t head_dim, int32_t elem, int64_t stride_page,
                   int64_t stride_slot, int64_t stride_head, int32_t page_size, int64_t num_pages,
                   int32_t cache_format, bool scaled, int64_t scale_stride_page,
                   int64_t scale_stride_head);

}  // namespace d2sd
