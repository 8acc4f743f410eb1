// Element types, vector loads and the 8-bit checkpoint format of the row operators (LayerNorm, the gated norm's
// checkpoint, the linear recurrence).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "umma.cuh"

namespace mek {

enum : int { kTypeBf16 = 0, kTypeFp16 = 1, kTypeFp32 = 2 };

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }

// N neighbouring elements of T moved as one access.
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T e[N];
};

template <typename T, int N>
__device__ __forceinline__ void unpack(const Vec<T, N>& raw, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = to_float(raw.e[i]);
}
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> pack(const float (&v)[N]) {
  Vec<T, N> raw;
#pragma unroll
  for (int i = 0; i < N; ++i) raw.e[i] = from_float<T>(v[i]);
  return raw;
}

// Two FP32 numbers in one register pair: the packed operations halve the instructions of a lane's two channels.
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float x, float y) {
  Two v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ Two two(float x) { return two(x, x); }
__device__ __forceinline__ float2 split(Two v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ Two sub2(Two a, Two b) {
  Two d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <typename T>
__device__ __forceinline__ Two widened(const Vec<T, 2>& v) { return two(to_float(v.e[0]), to_float(v.e[1])); }
template <typename T>
__device__ __forceinline__ Vec<T, 2> narrowed(Two v) {
  const float2 f = split(v);
  const float a[2] = {f.x, f.y};
  return pack<T, 2>(a);
}

// Element i of a parameter vector in one of the three types (a launch-uniform switch).
__device__ __forceinline__ float load_param(const void* p, int type, int64_t i) {
  if (type == kTypeBf16) return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (type == kTypeFp16) return to_float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_param(void* p, int type, int64_t i, float v) {
  if (type == kTypeBf16) static_cast<__nv_bfloat16*>(p)[i] = from_float<__nv_bfloat16>(v);
  else if (type == kTypeFp16) static_cast<__half*>(p)[i] = from_float<__half>(v);
  else static_cast<float*>(p)[i] = v;
}

// e4m3 codes (4 exponent bits, 3 mantissa bits, largest 448, NaN but no infinity), rounded to nearest even: off by at
// most 2^-4 of the value for magnitudes in [2^-6, 448], by 2^-10 below.  N of them, in whole words where there are that
// many (a register a byte otherwise).
template <int N>
struct Codes {
  static_assert(N % 4 == 0, "words");
  uint32_t word[N / 4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) word[i] = 0;
  }
};
template <>
struct Codes<1> {
  uint8_t byte;
  __device__ __forceinline__ void clear() { byte = 0; }
};
template <int N>
__device__ __forceinline__ Codes<N> load_codes(const uint8_t* p) {
  Codes<N> c;
  if constexpr (N == 1) c.byte = *p;
  else if constexpr (N == 4) c.word[0] = *reinterpret_cast<const uint32_t*>(p);
  else {
    static_assert(N == 8, "one access");
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    c.word[0] = w.x, c.word[1] = w.y;
  }
  return c;
}
template <int N>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&v)[N]) {
  if constexpr (N == 1) {
    *p = __nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
  } else {
    uint32_t word[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      word[i] = uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]), __NV_SATFINITE, __NV_E4M3)) |
                uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]), __NV_SATFINITE, __NV_E4M3)) << 16;
    if constexpr (N == 4) *reinterpret_cast<uint32_t*>(p) = word[0];
    else *reinterpret_cast<uint2*>(p) = make_uint2(word[0], word[1]);
  }
}
// Codes 2 q and 2 q + 1.
template <int N>
__device__ __forceinline__ float2 code_pair(const Codes<N>& c, int q) {
  const __nv_fp8x2_storage_t two = __nv_fp8x2_storage_t(c.word[q / 2] >> (q % 2 * 16));
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
}
__device__ __forceinline__ float code_value(uint8_t code) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
}

// How long the row operators' kernels wait, and, for the tests of a wait that runs out, what is not sent
// (mek_selftest_row_waits; as a rule one second, and everything is).
struct RowWaits {
  uint32_t limit_ns;
  uint32_t tiles_withheld;  // linear recurrence: bit w: the tokens of warp w of each tile; kWithholdWords: the tiles' words
  int64_t rows_served;      // LayerNorm: rows from here on are not copied where rows are streamed
};
constexpr uint32_t kWithholdWords = 1u << 8;
RowWaits row_waits();  // what the next launch takes

// A wait for copies that are on their way as a rule: the first looks go without the timer, whose reading costs more than
// a look (and is shared by the SM).
__device__ __forceinline__ bool mbar_wait_soon(uint64_t* bar, uint32_t parity, uint32_t limit_ns) {
  for (int looks = 0; looks < 256; ++looks)
    if (mbar_try_wait(bar, parity)) return true;
  const uint64_t began = global_timer_ns();
  for (;;) {
    if (mbar_try_wait(bar, parity)) return true;
    if (global_timer_ns() - began > limit_ns) return false;
  }
}

// After a wait that ran out: copies that are still in flight may write to this block's shared memory.
__device__ __forceinline__ void let_copies_land() {
  const uint64_t t0 = global_timer_ns();
  while (global_timer_ns() - t0 < 100000) __nanosleep(1000);
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}

}  // namespace mek
