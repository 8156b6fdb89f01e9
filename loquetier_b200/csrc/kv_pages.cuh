// Copies of cache pages: whole pages (a pool that is drawn together) or the first entries of each (the last page of a
// prompt that several continuations go on from).
//
// A page is [layers, 2, kv_heads, page_size, 128]: its first e entries are layers * 2 * kv_heads runs of e * 256 bytes,
// page_size * 256 bytes apart.  Bound by HBM: every byte is read once and written once, eight 16-byte loads of a thread in
// flight before its first store.  Measured: 280 pages of 2 MB 167 us (7.0 TB/s read and written), the filled parts of 24 last
// pages to four continuations each (113 MB, 17 us at the copy rate) 20.5 us; 23.2 with a division per 16 bytes.
#pragma once
#include "paged_kv.cuh"

namespace smlm {

constexpr int kCpThreads = 256;
constexpr int kCpUnroll = 8;
constexpr int kCpChunks = kCpThreads * kCpUnroll;   // 16-byte chunks a CTA moves per step

struct CopyPagesArgs {
  const void* const* dst;     // [n] page addresses
  const void* const* src;     // [n]
  const int32_t* entries;     // [n] positions to copy; null: all
  int* err;
  int n, runs, page_size;     // runs: layers * 2 * kv_heads
};

// grid: (chunks of a page, pages)
__global__ void __launch_bounds__(kCpThreads) copy_pages_kernel(const CopyPagesArgs a) {
  pdl_wait();
  pdl_trigger();
  for (int i = blockIdx.y; i < a.n; i += gridDim.y) {
    uint4* dst = static_cast<uint4*>(const_cast<void*>(a.dst[i]));
    const uint4* src = static_cast<const uint4*>(a.src[i]);
    const int e = a.entries == nullptr ? a.page_size : a.entries[i];
    const bool bad_ptr = dst == nullptr || src == nullptr ||
                         ((reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(src)) & 15) != 0;
    if (bad_ptr || e < 0 || e > a.page_size) {
      if (blockIdx.x == 0 && threadIdx.x == 0 && a.err != nullptr) atomicOr(a.err, bad_ptr ? kErrBadPointer : kErrBadIndptr);
      continue;
    }
    const unsigned run = e * 16, gap = a.page_size * 16;   // chunks of a run, and from one run to the next
    const unsigned total = run * a.runs;
    const unsigned hop = kCpThreads / max(run, 1u), rest = kCpThreads % max(run, 1u);   // runs and chunks of a thread's step
    for (unsigned c0 = blockIdx.x * kCpChunks + threadIdx.x; c0 < total; c0 += gridDim.x * kCpChunks) {
      uint4 v[kCpUnroll];
      unsigned at[kCpUnroll];
      unsigned r = c0 / run, j = c0 % run;   // (one division per step of eight)
#pragma unroll
      for (int u = 0; u < kCpUnroll; ++u) {
        at[u] = r * gap + j;
        v[u] = make_uint4(0u, 0u, 0u, 0u);
        if (c0 + u * kCpThreads < total) v[u] = __ldg(src + at[u]);
        r += hop;
        j += rest;
        if (j >= run) {
          j -= run;
          ++r;
        }
      }
#pragma unroll
      for (int u = 0; u < kCpUnroll; ++u)
        if (c0 + u * kCpThreads < total) dst[at[u]] = v[u];
    }
  }
}

}  // namespace smlm
