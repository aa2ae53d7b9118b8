// Products of microscaled 4-bit numbers: fp32, batch-size-last.
#include "ksmm_mx_product.h"

namespace ksmm {

int mx_float_last_plain(const MxProduct &p, int act, hipStream_t s) { return mx_last<float, false>(p, act, s); }

}  // namespace ksmm
