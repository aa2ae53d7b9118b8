// Products of microscaled 4-bit numbers on fp32 activations.
#include "ksmm_mx_product.h"

namespace ksmm {

int mx_run_float(MxProduct p, bool last, bool gated, int act, hipStream_t s) { return mx_run<float>(p, last, gated, act, s); }

}  // namespace ksmm
