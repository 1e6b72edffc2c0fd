// nirrt_libm_host.hpp - the host's libm, called function by function.  Through volatile pointers: a compiler that sees sin(t) and
// cos(t) side by side may merge them into one sincos(t), whose last bits need not be those of the two functions the reference calls.
#pragma once
#include <math.h>

namespace nirrt_libm_host {
static double (*volatile p_atan2)(double, double) = static_cast<double (*)(double, double)>(&::atan2);
static double (*volatile p_sin)(double) = static_cast<double (*)(double)>(&::sin);
static double (*volatile p_cos)(double) = static_cast<double (*)(double)>(&::cos);
}   // namespace nirrt_libm_host
