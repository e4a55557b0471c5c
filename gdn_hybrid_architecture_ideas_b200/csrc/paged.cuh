// What the kernels over the paged key/value cache share: the description of a batch of rows, its checks, and the 4-bit
// format. The cache is a pool of pages, [page, KV head, slot, channels]; 4 bits: E2M1 codes (two channels a byte, the
// even one low) with one E4M3 scale for 16 channels. Row b's packed new tokens are q_start[b] .. q_start[b + 1]; they are
// its last cached positions before lens[b].
//
// Metadata lives on the device, so the host cannot check its values. Every kernel checks what it is about to use (row
// ranges, lengths, page ids, rotary positions), writes a code to the status word where something is wrong and leaves the
// access out, so that a wrong table is an error the host reads, not a fault.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace ghb {

enum PagedStatus { ST_Q_START = 301, ST_LENS = 302, ST_START = 303, ST_PAGE = 304, ST_ROPE = 305, ST_DRAFTS = 306, ST_TOKEN = 307 };

struct Row { int q0, nq, len, start; };

// Row b's ranges, checked. A row whose range of packed tokens is wrong counts as having none; one whose length or
// start is wrong keeps its tokens but sees nothing (len 0).
__device__ __forceinline__ Row load_row(const PagedRows& r, int b) {
  Row o;
  o.q0 = r.q_start[b];
  const int q1 = r.q_start[b + 1];
  o.nq = q1 - o.q0;
  o.len = r.lens[b];
  o.start = r.start ? r.start[b] : 0;
  if (o.q0 < 0 || q1 < o.q0 || q1 > r.n) {
    *r.err = ST_Q_START;
    o.q0 = 0; o.nq = 0; o.len = 0; o.start = 0;
  } else if (o.len < o.nq || static_cast<long>(o.len) > (static_cast<long>(r.width) << r.page_shift)) {
    *r.err = ST_LENS;
    o.len = 0; o.start = 0;
  } else if (o.start < 0 || o.start > o.len) {
    *r.err = ST_START;
    o.len = 0; o.start = 0;
  }
  return o;
}

// The entry of (row b, position t, head h) as an index into [page, head, slot], or -1 where the page id is none.
__device__ __forceinline__ long entry_of(const PagedRows& r, int b, int t, int h) {
  const int page = r.pages[b * r.pages_stride + (t >> r.page_shift)];
  if (page < 0 || page >= r.n_pages) { *r.err = ST_PAGE; return -1; }
  return ((static_cast<long>(page) * r.Hkv + h) << r.page_shift) + (t & ((1 << r.page_shift) - 1));
}

// The row that packed token j belongs to: the last b with q_start[b] <= j < q_start[b + 1], or -1 (padding; in a table out of order
// perhaps a token that a row does own). qs is q_start, in shared memory where it fits.
__device__ __forceinline__ int row_of(const int* qs, int B, int j) {
  int lo = 0, hi = B;                  // rows lo .. hi - 1 may hold j
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (qs[mid + 1] <= j) lo = mid + 1; else hi = mid;
  }
  return lo < B && qs[lo] <= j ? lo : -1;
}

__device__ __forceinline__ float e4m3_to_float(uint8_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

}  // namespace ghb
