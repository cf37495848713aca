// Bits of the device status word, shared by the kernels that set them and the
// host that reports them.
#pragma once

#include <stdint.h>

namespace esmb200 {

// Device status bits written by kernels that wait on barriers.  A wait that
// runs past its bound records kStatusTimeout and the kernel unwinds instead
// of spinning forever; the host turns the bit into ESMCU_ERR_TIMEOUT.
constexpr uint32_t kStatusTimeout = 1u;
// Set by the paged-cache kernels when a length, position or page id that they
// read on the device lies outside the cache, its page table or the RoPE
// tables.  The access is skipped; the host turns the bit into
// ESMCU_ERR_OUT_OF_RANGE.
constexpr uint32_t kStatusBadIndex = 2u;

}  // namespace esmb200
