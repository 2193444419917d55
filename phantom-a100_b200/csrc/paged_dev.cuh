#pragma once
// Device-side view of ragged sequences in a paged cache: lengths and page ids are device data and are bounded here, so
// that no value of theirs makes a kernel read or write outside the arrays it was given. What is out of range is recorded
// in the status word (PHANTOM_ATTN_STATUS_PAGE).
#include "paged.h"

namespace phantom {

// One sequence: its first packed token, new tokens, cached tokens.
struct Seq {
  int tok0, n, len;
};

__device__ __forceinline__ Seq seq_of(const PagedSeqs& s, int b) {
  const int c0 = s.cu_new[b], c1 = s.cu_new[b + 1], len = s.kv_lens[b];
  const long long room = (long long)s.width << s.page_log2;
  Seq x;
  x.tok0 = min(max(c0, 0), s.total);
  x.n = min(max(c1, x.tok0), s.total) - x.tok0;
  x.len = (int)min((long long)max(len, 0), min(room, 0x7fffff00LL));
  if (x.tok0 != c0 || x.tok0 + x.n != c1 || x.len != len) atomicOr(s.status, PHANTOM_ATTN_STATUS_PAGE);
  return x;
}

// Page id of entry i of sequence b; -1 where there is none.
__device__ __forceinline__ int page_of(const PagedSeqs& s, int b, int i) {
  int id = (unsigned)i < (unsigned)s.width ? s.table[(long long)b * s.table_stride + i] : -1;
  if ((unsigned)id >= (unsigned)s.num_pages) {
    atomicOr(s.status, PHANTOM_ATTN_STATUS_PAGE);
    id = -1;
  }
  return id;
}

// Sequence of packed token `tok` (whole warp, one token): how many sequences end at or before it.
__device__ __forceinline__ int seq_index(const PagedSeqs& s, int tok) {
  const int lane = threadIdx.x & 31;
  int b = 0;
  for (int i0 = 0; i0 < s.batch; i0 += 32) {
    const int i = i0 + lane;
    b += __popc(__ballot_sync(0xffffffffu, i < s.batch && s.cu_new[min(i, s.batch - 1) + 1] <= tok));
  }
  return b;
}

}  // namespace phantom
