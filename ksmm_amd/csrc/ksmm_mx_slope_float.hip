// Gradients of what activations were applied to, of products of microscaled 4-bit numbers: fp32.  (Of three d_i its four waves and the library's exponentials take
// longer than a launch for z and one for dz: a pass of (2,96,72,3), 25088 rows, 283 us for 263.)
#include "ksmm_mx_slope.h"

namespace ksmm {

int mx_slope_float(const MxProduct &p, bool last, bool gated, int act, hipStream_t s)
{
    if (last) return mx_slope<float, true, 1>(p, gated, act, s);
    switch (p.d) {
    case 1: return mx_slope<float, false, 1>(p, gated, act, s);
    case 2: return mx_slope<float, false, 2>(p, gated, act, s);
    default: return KSMM_ERR_BAD_ALGO;
    }
}

}  // namespace ksmm
