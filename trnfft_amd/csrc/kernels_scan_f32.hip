// The selective scan over whole sequences (scan_blocks.h, scan_pairs.h): fp32 operands.
#include "scan_pairs.h"

namespace tfa {

hipError_t scan_f32(const ScanArgs& p, ScanMode mode) { return scan_typed<float>(p, mode); }

}  // namespace tfa
