// The 8-bit paged KV format and the device helpers that its kernels share.
//
// A cached row (token, KV head) of K or V is head_dim e4m3 codes and one scale
// byte (e8m0): the stored value is code * 2^(byte - 127).  The exponent is the
// smallest e in [-127, 119] with max|row| <= 448 * 2^e, so the largest element lands
// in (224, 448] and dividing by the scale is exact: the codes are the
// round-to-nearest-even e4m3 of x * 2^-e whatever precision that is done in.
// (Magnitudes above 448 * 2^119 = 2.98e38 saturate there, which keeps every stored
// value of a finite row finite in fp32 and bf16.)
// A row with an infinity or a NaN is stored as NaN codes with byte 255.
//
// Why a power of two and one byte per row: e4m3 is itself a floating-point format,
// so a finer scale would not add precision (only where in the octave the largest
// element lies), and a power of two multiplies bf16 / fp32 values without rounding,
// so attention can apply it to a score, a weight or a code alike.
#pragma once

#include "common.cuh"

namespace bpkv {
namespace q8 {

constexpr int kNanByte = 255;

// 2^(byte - 127); byte 0 is the subnormal 2^-127, byte 255 gives +inf (its codes are NaN).
__device__ __forceinline__ float scale_of(int byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : static_cast<uint32_t>(byte) << 23);
}

// Scale byte of a row whose largest magnitude has the bits `amax` (sign cleared).
// amax = 1.m * 2^x: 448 = 1.75 * 2^8, so e = x - 8, plus one when 1.m > 1.75.
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return kNanByte;
  const int e = static_cast<int>(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, -127), 119) + 127;
}

// 2^-qe, what a query row whose largest magnitude has the bits `amax` is multiplied by.  A row with an infinity or a NaN
// becomes NaN: whatever its scores are (with one infinite element all of them can be -inf), they have no softmax.
__device__ __forceinline__ float q_factor(uint32_t amax, int qe) {
  return __uint_as_float(amax >= 0x7f800000u ? 0x7fc00000u : static_cast<uint32_t>(127 - qe) << 23);
}

// Two floats -> two e4m3 codes (a in the low byte), round to nearest even.
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// Four e4m3 codes -> fp16, bytes 0 and 1 in `lo`, 2 and 3 in `hi`.  Exact: 4 significant bits, 2^-9..448.
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

// 32 bytes to a 32-byte boundary: a whole sector, where two 16-byte stores would write it in halves.
__device__ __forceinline__ void stg256(void* dst, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Page of request row `bt_row`, logical index j; -1 where the table has no such
// page of the pool (past the table's width, negative as of an offloaded page, or
// past the pool's end): such a page is never read or written.
__device__ __forceinline__ int page_of(const int32_t* bt_row, int j, int max_blocks, int num_pages) {
  if (j < 0 || j >= max_blocks) return -1;
  const int page = __ldg(bt_row + j);
  return (page >= 0 && page < num_pages) ? page : -1;
}

// Request of packed token i: the b with cu[b] <= i < cu[b+1], or -1 (before the first or past the last sequence).
__device__ __forceinline__ int request_of(const int32_t* cu, int batch, int i) {
  if (i < __ldg(cu) || i >= __ldg(cu + batch)) return -1;
  int lo = 0, hi = batch;  // cu[lo] <= i < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= i) lo = mid; else hi = mid;
  }
  return lo;
}

}  // namespace q8
}  // namespace bpkv
