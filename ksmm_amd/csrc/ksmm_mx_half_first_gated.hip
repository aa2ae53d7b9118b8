// Products of microscaled 4-bit numbers: fp16, batch-size-first, gated.
#include "ksmm_mx_product.h"

namespace ksmm {

int mx_half_first_gated(const MxProduct &p, int act, hipStream_t s) { return mx_first<half_t, true>(p, act, s); }

}  // namespace ksmm
