// fa_fp4_prefill.hip -- the prefill kernel over 4-bit codes (fa_quant_prefill.h).
#include "fa_quant_prefill.h"

namespace fa {

namespace {

template <int HD, int RB>
void launch_c(const QuantFwdArgs& a, int grid, hipStream_t stream) {
    if (a.bf16) launch_r<DT_BF16, CT_FP4, HD, RB>(a, grid, stream);
    else launch_r<DT_FP16, CT_FP4, HD, RB>(a, grid, stream);
}

}  // namespace

hipError_t launch_fp4_prefill(const QuantFwdArgs& a, int, int kd, int rows, int grid, hipStream_t stream) {
    if (kd == 64 && rows == 256) launch_c<64, 2>(a, grid, stream);
    else if (kd == 64) launch_c<64, 1>(a, grid, stream);
    else if (kd == 128 && rows == 256) launch_c<128, 2>(a, grid, stream);
    else if (kd == 128) launch_c<128, 1>(a, grid, stream);
    else launch_c<256, 1>(a, grid, stream);
    return hipGetLastError();
}

}  // namespace fa
