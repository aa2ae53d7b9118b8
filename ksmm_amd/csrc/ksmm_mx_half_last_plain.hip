// Products of microscaled 4-bit numbers: fp16, batch-size-last.
#include "ksmm_mx_product.h"

namespace ksmm {

int mx_half_last_plain(const MxProduct &p, int act, hipStream_t s) { return mx_last<half_t, false>(p, act, s); }

}  // namespace ksmm
