// The selective scan over whole sequences (scan_blocks.h, scan_pairs.h): bf16 operands.
#include "scan_pairs.h"

namespace tfa {

hipError_t scan_bf16(const ScanArgs& p, ScanMode mode) { return scan_typed<__bf16>(p, mode); }

}  // namespace tfa
