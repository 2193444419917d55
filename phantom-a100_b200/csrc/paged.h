#pragma once
// Internal interface between the C ABI (capi.cu) and the kernels of the paged key/value cache. Torch-free.
#include <cuda_runtime.h>

#include "../../include/phantom_attn.h"

namespace phantom {

// Sequences and the pages they are cached in, as the kernels read them. Every length, offset and page id is device
// data, so the kernels bound each one before they use it (paged_dev.cuh) and the host launches without a copy.
struct PagedSeqs {
  const int* table;    // (batch, width) page ids
  const int* kv_lens;  // (batch) tokens cached, the new ones among them
  const int* cu_new;   // (batch + 1) offsets of each sequence's new tokens in the packed (total, ...) arrays
  int batch, width, table_stride;
  int total;           // packed new tokens
  int num_pages, page_log2, heads;
  int* status;
};

// Element strides of a (page, head, token) array; the innermost dimension, if any, is contiguous.
struct Strides3 {
  long long page, head, token;
};

struct PagedCopyArgs {
  PagedSeqs s;
  void *k, *v;              // packed (total, heads, d), 16-bit: read by append, written by read
  long long k_token, k_head, v_token, v_head;  // element strides
  void *kc, *vc;            // caches (page, head, token, d)
  float *ks, *vs;           // scales (page, head, token) of an 8-bit cache
  Strides3 kcs, vcs, kss, vss;
  int d;
  bool bf16, int8;
  bool wide;                // k and v are 32-byte aligned
  cudaStream_t stream;
};

cudaError_t launch_paged_append(const PagedCopyArgs& a);
cudaError_t launch_paged_read(const PagedCopyArgs& a);

struct PagedAttnArgs {
  PagedSeqs s;
  const void* q;            // packed (total, heads * group, d), 16-bit
  long long q_token, q_head;
  void* o;                  // (total, heads * group, d), contiguous
  const void *kc, *vc;
  const float *ks, *vs;
  Strides3 kcs, vcs, kss, vss;
  int group;                // query heads of one key head
  int d;
  bool bf16, int8, causal;
  float scale;              // of the scores
  cudaStream_t stream;
};

// Few query rows for each key head (decoding): attn_paged.cu. Right for any number of them.
// `wide` (8-bit caches): units of 16 rows instead of 8.
cudaError_t launch_paged_attn_rows(const PagedAttnArgs& a, int dev, bool wide);
// Many query rows (chunks of prompts): attn_paged_tc_sm100.cu.
cudaError_t launch_paged_attn_chunk(const PagedAttnArgs& a, int dev);

// Shared host-side pieces (attn_tc_sm100.cu).
cudaError_t sm_count(int dev, int* n);
// Stream-ordered scratch from the library's pool of device `dev`, released with cudaFreeAsync on the same stream.
cudaError_t scratch_alloc(int dev, size_t bytes, cudaStream_t stream, void** out);
// A number unique to a call in this process, never 0.
unsigned long long next_call();
// TMA map of a (page, head, token, d) cache as (columns of a swizzled row, token, block of such columns, head, page): boxes
// of `cols` elements of `elem` bytes (64 or 128 bytes, the swizzle's width) by `rows` tokens by `blocks` column blocks of
// one head and `pages` pages.
bool make_paged_map(void* map, const void* base, int num_pages, int heads, int page, int d, const Strides3& st, int elem,
                    bool bf16, int cols, int rows, int blocks, int pages);

}  // namespace phantom
