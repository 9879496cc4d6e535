// Constants of 2^x on the fma pipe, without CUDA headers, so that the host can go over its whole range too.
//   x = n + f, n the nearest integer (found by adding EXP2_ROUND = 1.5 * 2^23, whose last place is 1), |f| <= 1/2;
//   2^f = ((((C4 f + C3) f + C2) f + C1) f + C0, a least-squares fit of the relative error, reweighted towards its
// peaks: at most 2.7e-6 = 2^-18.5 off; n is added to the exponent.
#pragma once

namespace lng {

constexpr float EXP2_ROUND = 12582912.f, EXP2_LOW = -126.f;  // below EXP2_LOW the result is 2^EXP2_LOW
constexpr float EXP2_C0 = 0.9999992847442627f, EXP2_C1 = 0.6931217908859253f, EXP2_C2 = 0.240247443318367f,
                EXP2_C3 = 0.05591785907745361f, EXP2_C4 = 0.009570100344717503f;

}  // namespace lng
