// Splitting fp32 values in two fp16 halves for the split-operand matrix products (device code only).
#pragma once
#include <hip/hip_runtime.h>

namespace danra {

// The remainders below are written as arithmetic and not as asm statements of the mixed-precision FMAs that write fp16
// halves (which would be one instruction less): a matrix instruction has to stay two wait states behind the VALU
// instruction that writes one of its operands, and a register that it still reads must not be overwritten early.  The
// compiler keeps those distances for its own instructions and for none inside an asm statement.

// c * h + s of the two halves of h, each rounded to nearest fp16: the product and the sum are exact in fp32 where these
// splits use them, so the one rounding is the conversion's.
__device__ __forceinline__ unsigned fma_pair_f16(unsigned h, float c, float s0, float s1) {
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    const f16x2_t hv = __builtin_bit_cast(f16x2_t, h);
    const f16x2_t l = {(_Float16)__builtin_fmaf((float)hv[0], c, s0), (_Float16)__builtin_fmaf((float)hv[1], c, s1)};
    return __builtin_bit_cast(unsigned, l);
}

// (x0, x1) -> hi = the pair rounded towards zero to fp16 (one packed conversion), lo = fp16(x - hi), rounded to nearest:
// x = hi + lo to 22 significant bits while |x| is in [2^-3, 65504]; for a smaller |x| lo is an fp16 subnormal and x is
// kept to an absolute 2^-25.  Four instructions per pair: the mixed-precision FMA reads the fp16 half of `hi` as an fp32
// operand, and one conversion packs both remainders.
__device__ __forceinline__ void split_pair_f16(float x0, float x1, unsigned& hi, unsigned& lo) {
    typedef __fp16 fp16x2_t __attribute__((ext_vector_type(2)));
    hi = __builtin_bit_cast(unsigned, (fp16x2_t)__builtin_amdgcn_cvt_pkrtz(x0, x1));
    float minus_one = -1.f;
    asm("" : "+s"(minus_one));  // (no instruction: hides the value, or the FMA becomes a conversion and a subtraction)
    lo = fma_pair_f16(hi, minus_one, x0, x1);
}

// (x0, x1) -> h = the pair rounded towards zero to fp16, l = fp16(2^11 (x - h)): x = h + 2^-11 l, the split of the
// attention core's K and V (the scaled remainder stays a normal fp16 number for |x| down to 2^-14).  Six instructions
// per pair.
__device__ __forceinline__ void split_scaled_pair_f16(float x0, float x1, unsigned& h, unsigned& l) {
    typedef __fp16 fp16x2_t __attribute__((ext_vector_type(2)));
    h = __builtin_bit_cast(unsigned, (fp16x2_t)__builtin_amdgcn_cvt_pkrtz(x0, x1));
    l = fma_pair_f16(h, -2048.f, x0 * 2048.f, x1 * 2048.f);
}

}  // namespace danra
