// ce_f32.hip — the linear cross entropy's products of f32 operands (ce_gemm.hpp).
#include "ce_gemm.hpp"

namespace mlxhip {

int ce_gemm_f32(int which, bool large, const ce::Args& a, hipStream_t s) {
    return ce::dispatch<MLXHIP_DTYPE_BF16, MLXHIP_DTYPE_F32, 3>(which, large, a, s);
}

}  // namespace mlxhip
