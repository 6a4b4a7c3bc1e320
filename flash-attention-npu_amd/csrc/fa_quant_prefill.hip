// fa_quant_prefill.hip -- the prefill kernel over 8-bit codes (fa_quant_prefill.h).
#include "fa_quant_prefill.h"

namespace fa {

namespace {

template <int HD, int RB>
void launch_c(const QuantFwdArgs& a, int ct, int grid, hipStream_t stream) {
    if (a.bf16) {
        if (ct == CT_INT8) launch_r<DT_BF16, CT_INT8, HD, RB>(a, grid, stream);
        else launch_r<DT_BF16, CT_E4M3, HD, RB>(a, grid, stream);
    } else {
        if (ct == CT_INT8) launch_r<DT_FP16, CT_INT8, HD, RB>(a, grid, stream);
        else launch_r<DT_FP16, CT_E4M3, HD, RB>(a, grid, stream);
    }
}

}  // namespace

// Rows of an item: 128, or as many as the registers take where sequences have them.
int quant_prefill_rows(int kd, bool many) { return many && kd < 256 ? 256 : 128; }

hipError_t launch_quant_prefill(const QuantFwdArgs& a, int ct, int kd, int rows, int grid, hipStream_t stream) {
    if (kd == 64 && rows == 256) launch_c<64, 2>(a, ct, grid, stream);
    else if (kd == 64) launch_c<64, 1>(a, ct, grid, stream);
    else if (kd == 128 && rows == 256) launch_c<128, 2>(a, ct, grid, stream);
    else if (kd == 128) launch_c<128, 1>(a, ct, grid, stream);
    else launch_c<256, 1>(a, ct, grid, stream);
    return hipGetLastError();
}

}  // namespace fa
