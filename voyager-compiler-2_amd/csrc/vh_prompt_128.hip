// Packed causal attention of heads of 128 channels.
#include "vh_prompt_backward.h"
#include "vh_prompt_forward.h"

namespace prompt {
template int forward<128>(const Args& a, bool bf16, hipStream_t s);
template int backward<128>(const Args& a, bool bf16, const int32_t* q_order, const int32_t* k_order, hipStream_t s);
}  // namespace prompt
