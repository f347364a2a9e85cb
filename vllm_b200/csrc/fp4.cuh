// A key-value cache in 4 bits.  A row (a token's keys or values of one head, D = 16 n values y = x / factor) is n scales e = e4m3(max |y| / 6) and D codes
// e2m1(y / e), and stands for code * e * factor.  code * e has at most six significant bits and lies in [2^-10, 2688]: exact in bf16 and in fp16.
//
// Cache [blocks, 2, kv heads, page, D / 2 + D / 16] bytes: a page of one head is its rows' codes (D / 2 bytes a row, the even value in the low half of a
// byte), then its rows' scales (D / 16 bytes a row), so both are contiguous runs for any run of rows.
#pragma once
#include "common.cuh"

namespace fp4 {

VB_DEVICE int64_t page_bytes(int BS, int D) { return (int64_t)BS * (D / 2 + D / 16); }

// eight codes: pairs of fp16 in the order of the values
VB_DEVICE void unpack8(uint32_t codes, uint32_t (&r)[4]) {
  asm("{\n\t.reg .b8 x0, x1, x2, x3;\n\tmov.b32 {x0, x1, x2, x3}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, x0;\n\tcvt.rn.f16x2.e2m1x2 %1, x1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, x2;\n\tcvt.rn.f16x2.e2m1x2 %3, x3;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(codes));
}
// two scales as fp16
VB_DEVICE uint32_t scales2(uint32_t two) { uint32_t r; asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two)); return r; }
VB_DEVICE uint32_t mul2(uint32_t a, uint32_t b) { uint32_t r; asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
VB_DEVICE uint32_t low2(uint32_t x) { return __byte_perm(x, x, 0x1010); }
VB_DEVICE uint32_t high2(uint32_t x) { return __byte_perm(x, x, 0x3232); }
// scale byte of a group whose largest |y| is `top` (NaN: NaN), and as a number
VB_DEVICE uint32_t scale_of(float top) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %1;" : "=h"(r) : "f"(__fdiv_rn(top, 6.f)));
  return r & 0xff;
}
VB_DEVICE float scale_value(uint32_t byte) { const uint32_t h = scales2(byte); return __half2float(__ushort_as_half((unsigned short)(h & 0xffff))); }
// codes of eight quotients, the first in the lowest bits
VB_DEVICE uint32_t pack8(const float (&f)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 x0, x1, x2, x3;\n\tcvt.rn.satfinite.e2m1x2.f32 x0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 x1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 x2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 x3, %8, %7;\n\tmov.b32 %0, {x0, x1, x2, x3};\n\t}"
      : "=r"(r) : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return r;
}

}  // namespace fp4
