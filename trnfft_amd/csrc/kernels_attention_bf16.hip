// Linear attention in blocks of tokens (attention_blocks.h): bf16 operands.
#include "attention_blocks.h"

namespace tfa {

hipError_t launch_attn_blocks_bf16(const AttnPass& p) { return blocks_modes<__bf16>(p); }

}  // namespace tfa
