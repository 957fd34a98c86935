// A row in 8 bits: q = the integer nearest to 127 x / a with a = max |x|, scale = a / 127.
#pragma once
#include "lowp.h"

namespace rexsc {

constexpr float Q8_SMALL = 7.888609052210118e-31f; // 2^-100: below it 127 / a could overflow
constexpr float Q8_LIFT = 1.2676506002282294e30f;  // 2^100

// The integer nearest to 127 x / a, ties to even, exactly.  x * inv with inv = fl(127 / a) is off by less than 1e-4;
// where that could decide, 127 x is compared with (the half-way point) * a in 64 bits, where both are exact.
__device__ __forceinline__ int nearest127(float x, float a, float inv)
{
    const float t = x * inv, r = rintf(t), d = t - r;
    int q = (int)r;
    if (fabsf(fabsf(d) - 0.5f) < 1e-3f) {
        const int o = d >= 0.f ? q + 1 : q - 1;
        const double v = 127.0 * (double)x, half = 0.5 * (double)(q + o) * (double)a;
        const int lo = q < o ? q : o, hi = q < o ? o : q;
        q = v < half ? lo : v > half ? hi : (lo & 1) ? hi : lo;
    }
    return q;
}

struct RowScale { float a, inv, lift, scale; };

// From the bits of the row's largest magnitude.  A row with a NaN or an infinity: scale NaN and zeros.
__device__ __forceinline__ RowScale row_scale(unsigned top)
{
    RowScale r;
    const float a = __uint_as_float(top);
    if (top >= 0x7f800000u) { r.a = 1.f; r.inv = 0.f; r.lift = 0.f; r.scale = __uint_as_float(0x7fc00000u); return r; }
    r.scale = a / 127.f;
    r.lift = a < Q8_SMALL ? Q8_LIFT : 1.f; // exact: both powers of two
    r.a = a * r.lift;
    r.inv = a > 0.f ? 127.f / r.a : 0.f;
    return r;
}
__device__ __forceinline__ int quant8(float x, const RowScale &r)
{
    return r.inv == 0.f ? 0 : nearest127(x * r.lift, r.a, r.inv);
}

} // namespace rexsc
