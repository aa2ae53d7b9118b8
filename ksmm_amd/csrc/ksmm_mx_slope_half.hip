// Gradients of what activations were applied to, of products of microscaled 4-bit numbers: fp16.
#include "ksmm_mx_slope.h"

namespace ksmm {

int mx_slope_half(const MxProduct &p, bool last, bool gated, int act, hipStream_t s)
{
    if (last) return mx_slope<half_t, true, 1>(p, gated, act, s);
    switch (p.d) {
    case 1: return mx_slope<half_t, false, 1>(p, gated, act, s);
    case 2: return mx_slope<half_t, false, 2>(p, gated, act, s);
    case 3: return mx_slope<half_t, false, 3>(p, gated, act, s);
    case 4: return mx_slope<half_t, false, 4>(p, gated, act, s);
    default: return KSMM_ERR_BAD_ALGO;
    }
}

}  // namespace ksmm
