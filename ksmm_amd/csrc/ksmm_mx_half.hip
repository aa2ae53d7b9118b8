// Products of microscaled 4-bit numbers on fp16 activations.
#include "ksmm_mx_product.h"

namespace ksmm {

int mx_run_half(MxProduct p, bool last, bool gated, int act, hipStream_t s) { return mx_run<half_t>(p, last, gated, act, s); }

bool mx_in_lds(int c, int d, int bs_last) { return mx_lds(1, bs_last ? 1 : mx_run_of(d), (int)mx_blocks(c)) <= MX_LDS_MOST; }

}  // namespace ksmm
