// Index arithmetic of the paged K/V cache, shared by the kernels and by a host
// check of it: every page id, position and length that a kernel reads on the
// device passes through here before it becomes an address.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define ESMB_HD __host__ __device__ __forceinline__
#else
#define ESMB_HD inline
#endif

namespace esmb200 {

// Where a token of an append goes.
struct Place {
  int page;  // -1: nothing is written for this token
  int slot;
  int pos;
  int bad;  // its length, position or page id is out of range
};

// The b in [0, B) with cu[b] <= t < cu[b + 1], for cu[0] <= t < cu[B], cu not
// decreasing.
ESMB_HD int sequence_of(const int* cu, int B, int t) {
  // One token per sequence, as a decoding batch has: no search.
  if (t < B && cu[t] <= t && t < cu[t + 1]) return t;
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Token t of a packed append: position lens[b] + t - cu[b] of its sequence.
// Tokens outside [cu[0], cu[B]) belong to no sequence and are no error;
// rows = the RoPE table's, or a negative number when nothing is rotated.
ESMB_HD Place append_place(const int* cu, int B, const int* lens, const int* table,
                           long table_stride, int max_pages, int page_size, int num_pages, int rows,
                           int t) {
  Place p = {-1, 0, 0, 0};
  if (B <= 0 || t < cu[0] || t >= cu[B]) return p;
  const int b = sequence_of(cu, B, t);
  const long len = lens[b];
  const long pos = len + t - cu[b];
  const long entry = pos / page_size;
  p.bad = 1;
  if (len < 0 || pos < 0 || pos > 0x7fffffffL || entry >= max_pages || (rows >= 0 && pos >= rows)) return p;
  const int page = table[b * table_stride + entry];
  if (page < 0 || page >= num_pages) return p;
  p.bad = 0;
  p.page = page;
  p.slot = static_cast<int>(pos - entry * page_size);
  p.pos = static_cast<int>(pos);
  return p;
}

// The keys [first, end) that a query at the end of a sequence sees.
struct KeyRange {
  int first, end;
  int bad;  // the length is negative or beyond the page table
};

ESMB_HD KeyRange key_range(int len, int max_pages, int page_size, int window) {
  const long capacity = static_cast<long>(max_pages) * page_size;
  KeyRange r = {0, len, 0};
  if (len < 0) {
    r.end = 0;
    r.bad = 1;
  } else if (len > capacity) {
    r.end = static_cast<int>(capacity);
    r.bad = 1;
  }
  if (window > 0 && r.end > window) r.first = r.end - window;
  return r;
}

// Tiles of 16 keys that hold the range.  They start at multiples of 16, so that
// one never straddles a page whose size is a multiple of 16.
ESMB_HD int tiles_of(const KeyRange& r) {
  return r.end > r.first ? ((r.end - 1) >> 4) - (r.first >> 4) + 1 : 0;
}

}  // namespace esmb200
