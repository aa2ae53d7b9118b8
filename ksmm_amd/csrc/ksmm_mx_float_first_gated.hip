// Products of microscaled 4-bit numbers: fp32, batch-size-first, gated.
#include "ksmm_mx_product.h"

namespace ksmm {

int mx_float_first_gated(const MxProduct &p, int act, hipStream_t s) { return mx_first<float, true>(p, act, s); }

}  // namespace ksmm
