// Rotary angles in 64 bits (gfx950), shared by the rope operator and by the
// attention over caches that keep a table of rotary frequencies.
//
// A table holds, per pair of dims, how many turns (2 pi radians) one position
// adds to the pair's angle. position * turns is one 64-bit product, its whole
// turns are dropped exactly, and cosine and sine follow from the rest: at
// position 2^20 the angle is off by at most 2^20 * 0.16 * 2^-53 turns = 1.2e-10
// radians, where a 32-bit product is off by up to 0.06. f64 FMAs issue at the
// rate of f32 ones here, so the 25 of them a pair takes cost less than the
// argument reduction of a 32-bit sincosf does.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ribn_amd {

struct Rot64 {
    double s, c;
};

// Sine and cosine of `turns` turns: the quarter turn k nearest is taken off
// (both subtractions are exact), and the Taylor series at the remaining
// |x| <= pi / 4 are cut where the next term is below 2^-53: x^17 / 17! and
// x^18 / 18! at pi / 4 are 5e-17 and 2e-18.
__device__ __forceinline__ Rot64 turn_sincos(double turns) {
    const double t = turns - __builtin_rint(turns);
    const double k = __builtin_rint(4.0 * t);
    const double x = __builtin_fma(-0.25, k, t) * 6.283185307179586477;
    const double z = x * x;
    double s = -1.0 / 1307674368000.0;  // 1 / 15!
    s = __builtin_fma(s, z, 1.0 / 6227020800.0);
    s = __builtin_fma(s, z, -1.0 / 39916800.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    s = __builtin_fma(s, z, -1.0 / 6.0);
    s = __builtin_fma(s * z, x, x);
    double c = 1.0 / 20922789888000.0;  // 1 / 16!
    c = __builtin_fma(c, z, -1.0 / 87178291200.0);
    c = __builtin_fma(c, z, 1.0 / 479001600.0);
    c = __builtin_fma(c, z, -1.0 / 3628800.0);
    c = __builtin_fma(c, z, 1.0 / 40320.0);
    c = __builtin_fma(c, z, -1.0 / 720.0);
    c = __builtin_fma(c, z, 1.0 / 24.0);
    c = __builtin_fma(c, z, -0.5);
    c = __builtin_fma(c, z, 1.0);
    const int q = (int)k & 3;
    Rot64 r;
    r.s = (q & 1) ? c : s;
    r.c = (q & 1) ? s : c;
    if (q & 2) r.s = -r.s;
    if (q == 1 || q == 2) r.c = -r.c;
    return r;
}

// The rotation of pair `i` at `position`, gain included: a table is
// turns[pairs] followed by the gain of cosine and sine.
__device__ __forceinline__ Rot64 table_rot(const double* table, int pairs, int i, int position) {
    Rot64 r = turn_sincos((double)position * table[i]);
    const double gain = table[pairs];
    r.s *= gain;
    r.c *= gain;
    return r;
}

}  // namespace ribn_amd
