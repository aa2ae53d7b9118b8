// Products of microscaled 4-bit numbers: fp32, batch-size-last, gated.
#include "ksmm_mx_product.h"

namespace ksmm {

int mx_float_last_gated(const MxProduct &p, int act, hipStream_t s) { return mx_last<float, true>(p, act, s); }

}  // namespace ksmm
