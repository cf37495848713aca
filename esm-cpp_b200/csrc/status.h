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

// A look at the status word, after which every bit that it held is the looker's
// and no other's.  `read` copies the word, nearly always 0; only then `take`
// exchanges it for 0, in one step, because kernels on other streams of the
// device may set bits at any time: what they set in between is taken too, what
// they set later stays.  Both return an error code (0: none) and give the word
// through their argument.
template <typename Read, typename Take>
int take_status(Read read, Take take, uint32_t& st) {
  const int rc = read(st);
  return rc != 0 || st == 0 ? rc : take(st);
}

}  // namespace esmb200
