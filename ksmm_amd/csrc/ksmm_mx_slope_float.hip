// Gradients of what activations were applied to, of products of microscaled 4-bit numbers: fp32.  (Two d_i of dy take more LDS than there is.)
#include "ksmm_mx_slope.h"

namespace ksmm {

int mx_slope_float(const MxProduct &p, bool last, bool gated, int act, hipStream_t s)
{
    if (last) return mx_slope<float, true, 1>(p, gated, act, s);
    return p.d == 1 ? mx_slope<float, false, 1>(p, gated, act, s) : KSMM_ERR_BAD_ALGO;
}

}  // namespace ksmm
