// Correctly rounded reciprocals and quotients of ordinary numbers, without a look at all others, so that several of a lane overlap.
#pragma once

namespace ep {

// 1 / x, correctly rounded, for 1 <= x < 2^118: an estimate, and one step with its residual (P. W. Markstein, Computation of elementary functions on the
// IBM RISC System/6000 processor, 1990).  The bits of __frcp_rn for every one of these numbers.
__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return fmaf(r, fmaf(-x, r, 1.f), r);
}

// a / x, correctly rounded, of 2^-100 <= a <= 1 and 1 <= x <= 2^20 with x's correctly rounded reciprocal: a quotient that is off by less than its last place
// and one step with its exact residual round as the quotient does (the same work's theorem on division)
__device__ __forceinline__ float quotient(float a, float x, float inverse) {
    float q = a * inverse;
    q = fmaf(fmaf(-q, x, a), inverse, q);
    return fmaf(fmaf(-q, x, a), inverse, q);
}

}  // namespace ep
