// Linear attention in blocks of tokens (attention_blocks.h): fp16 operands.
#include "attention_blocks.h"

namespace tfa {

hipError_t launch_attn_blocks_f16(const AttnPass& p) { return blocks_modes<_Float16>(p); }

}  // namespace tfa
