// packed_attn_f32.hip — attention of packed sequences, its gradient, and attention over pages: f32.
#include "packed_attn_impl.hpp"
#include "packed_attn_vjp_impl.hpp"

namespace mlxhip {
namespace attn {
template int fwd<MLXHIP_DTYPE_F32>(const FwdArgs&, bool, bool, hipStream_t);
template int bwd<MLXHIP_DTYPE_F32>(const BwdArgs&, hipStream_t);
}  // namespace attn
}  // namespace mlxhip
