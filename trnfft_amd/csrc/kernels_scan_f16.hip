// The selective scan over whole sequences (scan_blocks.h, scan_pairs.h): fp16 operands.
#include "scan_pairs.h"

namespace tfa {

hipError_t scan_f16(const ScanArgs& p, ScanMode mode) { return scan_typed<_Float16>(p, mode); }

}  // namespace tfa
