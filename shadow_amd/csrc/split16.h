// fp32 operands for the 16-bit matrix instructions: x * 2^e = hi + lo, two fp16 numbers each rounded to
// nearest, 22 bits of x; the power of two is common to all that one sum runs over.
#ifndef SHADOW_AMD_CSRC_SPLIT16_H_
#define SHADOW_AMD_CSRC_SPLIT16_H_

#include "device_common.h"

#pragma clang fp contract(off)

namespace shdw {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

SHDW_DEVICE float power2(int e) { return __int_as_float((e + 127) << 23); }  // -126 .. 127
SHDW_DEVICE int exponent_of(float v) { return static_cast<int>((__float_as_uint(v) >> 23) & 255u) - 127; }
// e such that 2^e times the largest of some numbers is in [2^13, 2^14), as far as 2^e and 2^-e are normal.
SHDW_DEVICE int lift_of(float largest) { return max(-126, min(126, 13 - exponent_of(largest))); }
// The same up to 140, which makes subnormal numbers whole multiples of 2^-9: what is lifted by it is multiplied twice, and
// 2^-e is subnormal too.
SHDW_DEVICE int far_lift_of(float largest) { return max(-126, 13 - exponent_of(largest)); }
SHDW_DEVICE float lifted(float v, int e) { return v * power2(min(e, 126)) * power2(max(e - 126, 0)); }
SHDW_DEVICE float lift_undone(int e) { return __builtin_ldexpf(1.f, -e); }
SHDW_DEVICE float larger(float a, float b) { return __builtin_fmaxf(a, b); }  // a NaN loses
SHDW_DEVICE float larger_or_nan(float a, float b) { return b <= a || a != a ? a : b; }

// Two at a time: four instructions, the back conversion being part of the subtraction.
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
SHDW_DEVICE void split2(float a, float b, v2h& hi, v2h& lo) {
  hi = __builtin_convertvector(v2f{a, b}, v2h);
  float ra, rb;  // a - hi[0], b - hi[1]
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(hi), "v"(a));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(hi), "v"(b));
  lo = __builtin_convertvector(v2f{ra, rb}, v2h);
}
SHDW_DEVICE void split8(const float (&x)[8], v8h& hi, v8h& lo) {
  v2h h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) split2(x[2 * i], x[2 * i + 1], h[i], l[i]);
  hi = v8h{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
  lo = v8h{l[0][0], l[0][1], l[1][0], l[1][1], l[2][0], l[2][1], l[3][0], l[3][1]};
}

// 16 bytes a lane from memory to LDS, from the lane's own address to 16 bytes a lane from `to` on.
SHDW_DEVICE void to_lds16(const void* from, void* to) {
  __builtin_amdgcn_global_load_lds(
      reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(from)),
      (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}
SHDW_DEVICE void to_lds4(const void* from, void* to) {  // 4 bytes a lane
  __builtin_amdgcn_global_load_lds(
      reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(from)),
      (__attribute__((address_space(3))) void*)to, 4, 0, 0);
}
// All of a workgroup's copies but each wave's last LATER have arrived, and all its reads of LDS are done.
template <int LATER = 0>
SHDW_DEVICE void copies_done() {
  static_assert(LATER >= 0 && LATER < 64, "what the counter holds");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((LATER & 15) | (LATER >> 4 << 14) | 7 << 4);  // vmcnt(LATER) lgkmcnt(0), where the compiler sees it
  asm volatile("s_barrier" ::: "memory");
}

// Waits for all loads where the compiler sees it, so that it does not wait later, where a rare path joins the others or a store may
// not be made: there it would be for copies or stores that are under way.
SHDW_DEVICE void loads_done() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0);
}

}  // namespace shdw

#endif  // SHADOW_AMD_CSRC_SPLIT16_H_
