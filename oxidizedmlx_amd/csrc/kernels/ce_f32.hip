// ce_f32.hip — the linear cross entropy's products of f32 operands, as two f16
// planes each for the logits and three bf16 ones for the gradients (ce_gemm.hpp).
#include "ce_gemm.hpp"

namespace mlxhip {

int ce_gemm_f32(int which, bool large, const ce::Args& a, hipStream_t s) {
    return ce::dispatch<MLXHIP_DTYPE_F32>(which, large, a, s);
}

}  // namespace mlxhip
