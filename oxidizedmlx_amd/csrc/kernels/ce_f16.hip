// ce_f16.hip — the linear cross entropy's products of f16 operands (ce_gemm.hpp).
#include "ce_gemm.hpp"

namespace mlxhip {

int ce_gemm_f16(int which, bool large, const ce::Args& a, hipStream_t s) {
    return ce::dispatch<MLXHIP_DTYPE_F16>(which, large, a, s);
}

}  // namespace mlxhip
