// Linear attention in blocks of tokens (attention_blocks.h): fp32 operands.
#include "attention_blocks.h"

namespace tfa {

hipError_t launch_attn_blocks_f32(const AttnPass& p) { return blocks_modes<float>(p); }

}  // namespace tfa
