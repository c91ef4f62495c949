/* rounded_math.c -- the correctly rounded functions that the oracle links, for
 * a checkout without the reference tree (whose CORE-MATH shim, entry points
 * crates/chelis-crmath/csrc/crmath_ffi.c:15-45, oracle/Makefile prefers).
 * A correctly rounded result is one number, so both give the same bits.
 *
 * binary64: the function in gcc's binary128 (113 bits, error near one unit in
 * the last place), rounded once.  What would be rounded the wrong way lies
 * within 2^-111 or so of the middle between two doubles, which no result of
 * these functions is expected to be unless it is that middle exactly; of these
 * functions pow alone reaches it (a power of few bits), and is put back on it.
 * binary32: libm in binary64 decides unless the numbers within 2^-47 of its
 * result (a hundred times the error of these functions in glibc) round to two
 * different floats, then binary128 does.
 */
#include <math.h>
#include <quadmath.h>
#include <stdint.h>
#include <string.h>

#define MARGIN 0x1p-47

/* Every NaN is the canonical quiet one, as CORE-MATH's entry points give it. */
static double quiet64(double v) { return v != v ? __builtin_nan("") : v; }
static float quiet32(float v) { return v != v ? __builtin_nanf("") : v; }

/* q to nearest, where q within 2^-111 of the middle of two numbers is that
 * middle (ties to the even one).  The square root of 1 - 2^-53 is as near as 2^-109
 * and is none. */
static double middle64(__float128 q) {
    const double v = (double)q;
    if (!isfinite(v) || q == v) return v;
    const double o = nextafter(v, q > v ? INFINITY : -INFINITY);
    if (!isfinite(o)) return v;
    const __float128 m = ((__float128)v + o) / 2;
    if (fabsq(q - m) > fabsq(m) * 0x1p-111Q) return v;
    uint64_t bits;
    memcpy(&bits, &v, 8);
    return bits & 1 ? o : v;
}
static float middle32(__float128 q) {
    const float v = (float)q;
    if (!isfinite(v) || q == v) return v;
    const float o = nextafterf(v, q > v ? INFINITY : -INFINITY);
    if (!isfinite(o)) return v;
    const __float128 m = ((__float128)v + o) / 2;
    if (fabsq(q - m) > fabsq(m) * 0x1p-111Q) return v;
    uint32_t bits;
    memcpy(&bits, &v, 4);
    return bits & 1 ? o : v;
}

#define UNARY(name)                                                                       \
    double chelis_crmath_ffi_##name(double x) { return quiet64((double)name##q(x)); }   \
    float chelis_crmath_ffi_##name##f(float x) {                                          \
        const double y = name((double)x);                                                 \
        const float lo = (float)(y * (1 - MARGIN)), hi = (float)(y * (1 + MARGIN));       \
        return quiet32(lo == hi || y != y ? lo : (float)name##q(x));                         \
    }
UNARY(exp)
UNARY(log)
UNARY(sin)
UNARY(cos)
UNARY(tan)
UNARY(atan)
UNARY(tanh)
UNARY(erf)
UNARY(erfc)

/* A signaling NaN makes every power NaN, pow(x, 0) and pow(1, y) too. */
double chelis_crmath_ffi_pow(double x, double y) {
    if (issignaling(x) || issignaling(y)) return __builtin_nan("");
    return quiet64(middle64(powq(x, y)));
}
float chelis_crmath_ffi_powf(float x, float y) {
    if (issignaling(x) || issignaling(y)) return __builtin_nanf("");
    const double p = pow((double)x, (double)y);
    const float lo = (float)(p * (1 - MARGIN)), hi = (float)(p * (1 + MARGIN));
    return quiet32(lo == hi || p != p ? lo : middle32(powq(x, y)));
}
