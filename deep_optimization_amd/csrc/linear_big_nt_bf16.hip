#include "linear_big.h"

namespace dopt {

void lin_big_nt_bf16(const LinArgs& p, int bm, int n_cu, hipStream_t s) {
    if (bm == 160) lin_big_launch<160, false, false>(p, n_cu, s);
    else lin_big_launch<256, false, false>(p, n_cu, s);
}

}  // namespace dopt
