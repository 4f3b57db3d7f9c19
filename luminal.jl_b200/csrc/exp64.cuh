// The exponential in 64 bits with which the token is chosen from a row of logits (verify.cu).
#pragma once
#include <cuda_runtime.h>
#include <float.h>

namespace lmb {

__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 32) table[threadIdx.x] = exp2(threadIdx.x / 32.0);
}

// exp((x - top) / T) for a logit x <= top: y = (x - top) log2(e) / T = k / 32 + f, |f| <= 1 / 64, and 2^y = 2^(k / 32) 2^f with the first factor from a table and the second by its power series
// (P. T. P. Tang, Table-driven implementation of the exponential function in IEEE floating-point arithmetic, ACM TOMS 15, 1989; here to base 2, so nothing is split for the reduction).
// Relative error: the series' first term left out, (ln 2 / 64)^6 / 720 = 2.2e-15; its and the table's roundings, 6 x 2^-53; those of y, four in a row, 4 x 2^-53 |y| ln 2.
struct Power {
  const double* table;                       // [32] in shared memory: 2^(k / 32)
  double slope, top;                         // log2(e) / T
  float least;                               // logits below it count for nothing: less than 2^-900 of the top's
  __device__ __forceinline__ Power(const double* t, float m, double inv_T) : table(t), slope(inv_T * 1.4426950408889634), top(m) {
    least = __double2float_ru(fmax(top - 900.0 / slope, -(double)FLT_MAX));        // upwards, never to a logit below it: the exponent field has no room for that
  }
  __device__ __forceinline__ double operator()(float x) const {
    asm("min.NaN.f32 %0, %0, 0f7f7fffff;" : "+f"(x));                    // +infinity as the largest float; NaN stays, and fails the comparison
    if (!(x >= least)) return 0.0;
    constexpr double kInt = 6755399441055744.0;                          // 1.5 2^52: a small number added to it leaves its rint in the low bits
    const double y = ((double)x - top) * slope, shifted = fma(y, 32.0, kInt), f = fma(shifted - kInt, -0.03125, y);
    const int k = __double2loint(shifted);
    // ln(2)^n / n!
    const double e = fma(fma(fma(fma(fma(f, 1.3333558146428443e-3, 9.618129107628477e-3), f, 5.550410866482158e-2), f, 0.24022650695910072), f, 0.6931471805599453), f, 1.0) *
                     table[k & 31];
    return __hiloint2double(__double2hiint(e) + (k >> 5) * 1048576, __double2loint(e));
  }
};

}  // namespace lmb
