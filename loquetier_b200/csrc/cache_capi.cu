// C ABI of the operators around a cache that several continuations share: attention of a chunk of new tokens, norms of
// queries and keys per head, page copies.  Declarations: include/smlm_b200_kv.h, include/smlm_b200.h.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/smlm_b200.h"
#include "../../include/smlm_b200_kv.h"
#include "head_norm.cuh"
#include "kv_pages.cuh"
#include "paged_extend.cuh"
#include "smlm_launch.cuh"

namespace {

// base^(-2 i / 128) / pi as pairs of floats; the last base's table is kept per thread (64 powers take a microsecond)
const RotTable& rot_table(double base) {
  thread_local RotTable table;
  thread_local double of = 0.0;
  if (of != base) {
    for (int i = 0; i < 64; ++i) {
      const double f = std::pow(base, -i / 64.0) / 3.14159265358979323846;
      table.hi[i] = static_cast<float>(f);
      table.lo[i] = static_cast<float>(f - static_cast<double>(table.hi[i]));
    }
    of = base;
  }
  return table;
}

// How an extend launch is laid out: everything follows from sizes the host knows, so that the workspace query and the launch
// agree.
struct ExPlan {
  int qt;          // quarters of 32 rows of a row tile
  int shares;      // CTAs per kv head
  int min_tiles;   // key tiles of a share at least
  bool dense;      // the keys are rotated once, in front
  bool fits;       // the work counts in 31 bits
  size_t state;    // bytes of cuts and softmax states
  size_t bytes;    // and of rotated keys
};

// Rows of a row tile, by the mean number of rows (new tokens x query heads per kv head) of a request.  A tile's rows cost
// softmax work and queries; rows that do not fit one tile walk the keys again.  32 requests with contexts 512..4096, 32 / 8
// heads, bf16, us with tiles of 32 / 64 / 128 rows, by rows per request:
//   4 and 8  87 / 95 / 101    32  91 / 99 / 103    40  155 / 97 / 110    64  153 / 101 / 114    80  214 / 167 / 116
// Keys rotated once in front (three more passes over them) or by every row tile that meets them, us, in place / in front, 32 / 8
// heads, by rows per request:
//   1 request on 16 k keys    128  50 / 56    256  69 / 69      320  81 / 73      512  97 / 83      1024  156 / 118    4096  490 / 308
//   8 requests on 4 k keys    128  73 / 87    256  106 / 103    320  136 / 124    512  165 / 141    1024  288 / 226    4096  1070 / 767
ExPlan extend_plan(int batch, int total_q, int total_pages, int page_size, int num_kv_heads, int group) {
  ExPlan p;
  const long long all_rows = static_cast<long long>(total_q) * group;
  const long long mean = (all_rows + batch - 1) / batch;
  p.qt = mean <= 32 ? 1 : mean <= 64 ? 2 : 4;
  p.dense = mean > 256;
  p.min_tiles = 4;   // (a share pays for its start: 18 us for 300 keys in shares of 4 tiles as of 8)
  const int rows = 32 * p.qt;
  // all the CTAs that are resident, but no more than the work can hold
  const long long key_tiles = static_cast<long long>(total_pages) * page_size / kXtKeys + batch;
  const long long most = (all_rows / rows + batch) * key_tiles / p.min_tiles + 1;
  p.fits = (all_rows / rows + batch) * key_tiles < 0x7fffff00LL;
  p.shares = static_cast<int>(std::min<long long>(std::max(1, kXtCtasPerSm * kNumSMs / num_kv_heads), most));
  p.state = p.shares > 1 ? static_cast<size_t>(p.shares) * num_kv_heads * (sizeof(ExCut) + 2 * rows * kPdRec * sizeof(float)) : 0;
  p.bytes = p.state + (p.dense ? static_cast<size_t>(total_pages) * page_size * num_kv_heads * kPdDim * 2 : 0);
  return p;
}

template <typename T, int QT, bool DENSE = false>
int launch_extend(const ExArgs& a, const ExPlan& p, cudaStream_t stream) {
  using X = Xt<QT, DENSE>;
  const unsigned heads = static_cast<unsigned>(a.num_kv_heads);
  if (DENSE) {
    const int rc = launch(extend_rotate_kernel<T>, dim3(a.total_pages, 1, 1), 128, 1, 0, stream, a);
    if (rc != SMLM_OK) return rc;
  }
  const int rc = launch(paged_extend_kernel<T, QT, DENSE>, dim3(p.shares * heads, 1, 1), X::kThreads, 1, X::kSmem, stream, a);
  if (rc != SMLM_OK || p.shares == 1) return rc;
  return launch(paged_extend_merge_kernel<T, QT>, dim3((p.shares - 1) * heads, kXtMergeSplit, 1), kXtMergeThreads, 1, 0, stream, a);
}

template <typename T>
int dispatch_extend(const ExArgs& a, const ExPlan& p, cudaStream_t stream) {
  switch (p.qt) {
    case 1: return launch_extend<T, 1>(a, p, stream);
    case 2: return launch_extend<T, 2>(a, p, stream);
    default: return p.dense ? launch_extend<T, 4, true>(a, p, stream) : launch_extend<T, 4>(a, p, stream);
  }
}

// Warps that share a token's heads: few tokens are spread over the machine (2368 warps, two CTAs per SM), four heads per warp at
// least.  bf16, us of one launch among others, by this rule / one warp per token / a warp per four heads always:
//   32 / 8 heads, forward    1 token  1.8 / 3.4 / 1.8    181  3.3 / 5.0 / 3.3    600  5.3 / 6.1 / 6.2    2048  10.5 / 8.9 / 16.1
//                 8192  31 / 31 / 62        backward    64  4.5 / 7.8 / 4.6    600  9.7 / 9.1 / 9.7    8192  50 / 51 / 58
//   32 / 32 heads, into the cache    64  3.2 / 9.5 / 3.2    600  6.6 / 12.2 / 7.5    2048  20.1 / 20.0 / 22.3
inline int head_splits(int T, int heads) {
  const int want = (8 * kNumSMs * 2 + T - 1) / std::max(T, 1);
  return std::max(1, std::min(want, (heads + 3) / 4));
}

// the streams of queries and keys, a unit per warp
void qk_streams(HeadNormArgs& a, int Nq, int Nk) {
  const int heads[2] = {Nq, Nk};
  for (int i = 0; i < 2; ++i) {
    a.s[i].heads = heads[i];
    a.s[i].splits = head_splits(a.T, heads[i]);
    a.s[i].ctas = static_cast<int>((static_cast<long long>(a.T) * a.s[i].splits + kHnWarps - 1) / kHnWarps);
  }
}

// the backward pass: as many CTAs as are resident at most, shared out by the numbers of heads
void qk_bwd_streams(HeadNormArgs& a, int Nq, int Nk) {
  qk_streams(a, Nq, Nk);
  const int resident = 2 * kNumSMs;
  const int k_most = std::max(1, static_cast<int>(static_cast<long long>(resident) * Nk / (Nq + Nk)));
  a.s[1].ctas = std::min(a.s[1].ctas, k_most);
  a.s[0].ctas = std::min(a.s[0].ctas, std::max(1, resident - k_most));
}

template <typename T>
int launch_qk_fwd(const HeadNormArgs& a, cudaStream_t stream) {
  const bool norm = a.s[0].w != nullptr, rope = a.positions != nullptr;
  const dim3 grid(a.s[0].ctas + a.s[1].ctas, 1, 1);
  if (norm) return rope ? launch(qk_norm_rope_kernel<T, true, true>, grid, kHnThreads, 1, 0, stream, a)
                        : launch(qk_norm_rope_kernel<T, true, false>, grid, kHnThreads, 1, 0, stream, a);
  return launch(qk_norm_rope_kernel<T, false, true>, grid, kHnThreads, 1, 0, stream, a);
}

template <typename T>
int launch_qk_bwd(const HeadNormArgs& a, void* dwq, void* dwk, cudaStream_t stream) {
  const bool norm = a.s[0].w != nullptr, rope = a.positions != nullptr;
  const dim3 grid(a.s[0].ctas + a.s[1].ctas, 1, 1);
  if (!norm) return launch(qk_norm_rope_bwd_kernel<T, false, true>, grid, kHnThreads, 1, kHnSmem, stream, a);
  const int rc = rope ? launch(qk_norm_rope_bwd_kernel<T, true, true>, grid, kHnThreads, 1, kHnSmem, stream, a)
                      : launch(qk_norm_rope_bwd_kernel<T, true, false>, grid, kHnThreads, 1, kHnSmem, stream, a);
  if (rc != SMLM_OK || dwq == nullptr) return rc;
  return launch(head_norm_dw_kernel<T>, dim3(2 * kPdDim / 8, 1, 1), 256, 1, 0, stream, dwq, dwk, a.partial, a.s[0].ctas,
                static_cast<int>(grid.x));
}

// the checks that both directions share; rows that are strided have to keep the 16-byte alignment of every head
int qk_check(const void* q, const void* k, const void* wq, const void* wk, const void* positions, long long q_stride,
             long long k_stride, int T, int Nq, int Nk, int head_dim, double rope_theta, int dtype) {
  if (T < 0 || Nq <= 0 || Nk <= 0 || (wq == nullptr) != (wk == nullptr) || (wq == nullptr && positions == nullptr) ||
      (positions != nullptr && !(rope_theta > 0.0)))
    return SMLM_ERR_INVALID_ARGUMENT;
  if (dtype != SMLM_F16 && dtype != SMLM_BF16) return SMLM_ERR_DTYPE;
  if (head_dim != kPdDim) return SMLM_ERR_NO_KERNEL;
  if (T == 0) return SMLM_OK;
  if (q == nullptr || k == nullptr) return SMLM_ERR_INVALID_ARGUMENT;
  if (q_stride < static_cast<long long>(Nq) * kPdDim || k_stride < static_cast<long long>(Nk) * kPdDim)
    return SMLM_ERR_INVALID_ARGUMENT;   // rows that overlap
  if (!aligned16(q) || !aligned16(k) || !aligned16(wq) || !aligned16(wk) || q_stride % 8 != 0 || k_stride % 8 != 0)
    return SMLM_ERR_MISALIGNED;
  return SMLM_OK;
}

}  // namespace

extern "C" {

size_t smlm_b200_batch_extend_workspace_bytes(int batch_size, int total_q, int total_pages, int page_size,
                                              int num_qo_heads, int num_kv_heads) {
  if (batch_size <= 0 || total_q <= 0 || total_pages < 0 || page_size <= 0 || num_kv_heads <= 0 ||
      num_qo_heads < num_kv_heads)
    return 0;
  return extend_plan(batch_size, total_q, total_pages, page_size, num_kv_heads, num_qo_heads / num_kv_heads).bytes;
}

int smlm_b200_batch_extend(void* o, const void* q, const int32_t* qo_indptr, const void* const* kv_ptrs,
                           const int32_t* kv_indptr, const int32_t* last_page_offset, void* workspace,
                           size_t workspace_bytes, int* status_word, int batch_size, int total_q, int total_pages,
                           int num_qo_heads, int num_kv_heads, int head_dim, int num_layers, int layer_idx, int page_size,
                           double rope_theta, int dtype, void* stream) {
  if (batch_size < 0 || total_q < 0 || total_pages < 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || num_layers <= 0 ||
      layer_idx < 0 || layer_idx >= num_layers || !(rope_theta > 0.0))
    return SMLM_ERR_INVALID_ARGUMENT;
  if (dtype != SMLM_F16 && dtype != SMLM_BF16) return SMLM_ERR_DTYPE;
  if (num_qo_heads % num_kv_heads != 0 || !kv_shape_ok(head_dim, page_size)) return SMLM_ERR_NO_KERNEL;
  const int group = num_qo_heads / num_kv_heads;
  if (group != 1 && group != 2 && group != 4 && group != 8) return SMLM_ERR_NO_KERNEL;
  if (batch_size == 0 || total_q == 0) return SMLM_OK;
  if (o == nullptr || q == nullptr || qo_indptr == nullptr || kv_indptr == nullptr || last_page_offset == nullptr ||
      (kv_ptrs == nullptr && total_pages > 0))
    return SMLM_ERR_INVALID_ARGUMENT;
  if (!aligned16(o) || !aligned16(q)) return SMLM_ERR_MISALIGNED;
  if (static_cast<long long>(total_q) * num_qo_heads > 0x7fffffffLL ||
      static_cast<long long>(total_pages) * page_size > 0x7fffffffLL ||
      static_cast<long long>(num_layers) * 2 * num_kv_heads * page_size * kPdDim * 2 > 0x7fffffffLL)   // a page of 2 GB
    return SMLM_ERR_INVALID_ARGUMENT;
  const ExPlan p = extend_plan(batch_size, total_q, total_pages, page_size, num_kv_heads, group);
  if (!p.fits) return SMLM_ERR_INVALID_ARGUMENT;
  if (p.bytes > 0) {
    if (workspace == nullptr || workspace_bytes < p.bytes) return SMLM_ERR_WORKSPACE;
    if (!aligned16(workspace)) return SMLM_ERR_MISALIGNED;
  }
  // (a row tile's queries may be read after another share has written its results)
  const uintptr_t o_at = reinterpret_cast<uintptr_t>(o), q_at = reinterpret_cast<uintptr_t>(q);
  const uintptr_t q_bytes = static_cast<uintptr_t>(total_q) * num_qo_heads * kPdDim * 2;
  if (o_at - q_at < q_bytes || q_at - o_at < q_bytes) return SMLM_ERR_INVALID_ARGUMENT;
  ExArgs a;
  a.o = o; a.q = q; a.qo_indptr = qo_indptr; a.kv_ptrs = kv_ptrs; a.kv_indptr = kv_indptr;
  a.last_page_offset = last_page_offset; a.err = status_word;
  a.cuts = p.state > 0 ? static_cast<ExCut*>(workspace) : nullptr;
  a.dense = p.dense ? static_cast<char*>(workspace) + p.state : nullptr;
  a.partial = reinterpret_cast<float*>(a.cuts + static_cast<size_t>(p.shares) * num_kv_heads);
  a.batch = batch_size; a.total_q = total_q; a.total_pages = total_pages; a.num_kv_heads = num_kv_heads;
  a.num_layers = num_layers; a.layer_idx = layer_idx; a.page_size = page_size;
  a.lg = group == 1 ? 0 : group == 2 ? 1 : group == 4 ? 2 : 3;
  a.shares = p.shares; a.min_tiles = p.min_tiles;
  a.rot = rot_table(rope_theta);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == SMLM_F16 ? dispatch_extend<__half>(a, p, st) : dispatch_extend<__nv_bfloat16>(a, p, st);
}

int smlm_b200_copy_pages(const void* const* dst_ptrs, const void* const* src_ptrs, const int32_t* entries,
                         int* status_word, int n, int num_layers, int num_kv_heads, int head_dim, int page_size, int dtype,
                         void* stream) {
  if (n < 0 || num_layers <= 0 || num_kv_heads <= 0) return SMLM_ERR_INVALID_ARGUMENT;
  if (dtype != SMLM_F16 && dtype != SMLM_BF16) return SMLM_ERR_DTYPE;
  if (!kv_shape_ok(head_dim, page_size)) return SMLM_ERR_NO_KERNEL;
  if (n == 0) return SMLM_OK;
  if (dst_ptrs == nullptr || src_ptrs == nullptr) return SMLM_ERR_INVALID_ARGUMENT;
  const long long chunks = static_cast<long long>(num_layers) * 2 * num_kv_heads * page_size * 16;
  if (chunks > 0x7fffffffLL) return SMLM_ERR_INVALID_ARGUMENT;   // a page of 32 GB
  CopyPagesArgs a;
  a.dst = dst_ptrs; a.src = src_ptrs; a.entries = entries; a.err = status_word;
  a.n = n; a.runs = num_layers * 2 * num_kv_heads; a.page_size = page_size;
  const dim3 grid(static_cast<unsigned>((chunks + kCpChunks - 1) / kCpChunks), std::min(n, 65535), 1);
  return launch(copy_pages_kernel, grid, kCpThreads, 1, 0, static_cast<cudaStream_t>(stream), a);
}

int smlm_b200_norm_append_kv(void* yq, const void* q, const void* k, const void* v, const void* wq, const void* wk,
                             const void* const* kv_ptrs, const int32_t* kv_indptr, const int32_t* last_page_offset,
                             const int32_t* seqlen_indptr, int* status_word, long long q_stride, long long k_stride,
                             long long v_stride, int batch_size, int total_tokens, int total_pages, int num_qo_heads,
                             int num_kv_heads, int head_dim, int num_layers, int layer_idx, int page_size, float eps,
                             int dtype, void* stream) {
  if (batch_size < 0 || total_tokens < 0 || total_pages < 0 || num_layers <= 0 || layer_idx < 0 ||
      layer_idx >= num_layers || (seqlen_indptr == nullptr && total_tokens != batch_size) || wq == nullptr || wk == nullptr)
    return SMLM_ERR_INVALID_ARGUMENT;
  const int rc = qk_check(q, k, wq, wk, nullptr, q_stride, k_stride, total_tokens, num_qo_heads, num_kv_heads, head_dim, 1.0,
                          dtype);
  if (rc != SMLM_OK) return rc;
  if (!kv_shape_ok(head_dim, page_size)) return SMLM_ERR_NO_KERNEL;
  if (batch_size == 0 || total_tokens == 0) return SMLM_OK;
  if (yq == nullptr || v == nullptr || kv_indptr == nullptr || last_page_offset == nullptr ||
      (kv_ptrs == nullptr && total_pages > 0) || v_stride < static_cast<long long>(num_kv_heads) * kPdDim)
    return SMLM_ERR_INVALID_ARGUMENT;
  if (!aligned16(yq) || !aligned16(v) || v_stride % 8 != 0) return SMLM_ERR_MISALIGNED;
  NormAppendArgs a;
  a.q = q; a.k = k; a.v = v; a.wq = wq; a.wk = wk; a.yq = yq; a.kv_ptrs = kv_ptrs; a.kv_indptr = kv_indptr;
  a.last_page_offset = last_page_offset; a.append_indptr = seqlen_indptr; a.err = status_word;
  a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.T = total_tokens; a.batch = batch_size; a.Nq = num_qo_heads; a.Nk = num_kv_heads; a.num_layers = num_layers;
  a.layer_idx = layer_idx; a.page_size = page_size; a.total_pages = total_pages; a.eps = eps;
  a.splits = head_splits(total_tokens, std::max(num_qo_heads, num_kv_heads));
  const dim3 grid(static_cast<unsigned>((static_cast<long long>(a.T) * a.splits + kHnWarps - 1) / kHnWarps), 1, 1);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == SMLM_F16 ? launch(norm_append_kernel<__half>, grid, kHnThreads, 1, 0, st, a)
                           : launch(norm_append_kernel<__nv_bfloat16>, grid, kHnThreads, 1, 0, st, a);
}

int smlm_b200_qk_norm_rope(void* yq, void* yk, const void* q, const void* k, const void* wq, const void* wk,
                           const void* positions, long long q_stride, long long k_stride, int T, int num_qo_heads,
                           int num_kv_heads, int head_dim, int positions_64, double rope_theta, float eps, int dtype,
                           void* stream) {
  const int rc = qk_check(q, k, wq, wk, positions, q_stride, k_stride, T, num_qo_heads, num_kv_heads, head_dim,
                          rope_theta, dtype);
  if (rc != SMLM_OK || T == 0) return rc;
  if (yq == nullptr || yk == nullptr) return SMLM_ERR_INVALID_ARGUMENT;
  if (!aligned16(yq) || !aligned16(yk)) return SMLM_ERR_MISALIGNED;
  HeadNormArgs a = {};
  a.positions = positions; a.T = T; a.pos64 = positions_64; a.eps = eps;
  a.s[0].x = q; a.s[0].w = wq; a.s[0].y = yq; a.s[0].stride = q_stride;
  a.s[1].x = k; a.s[1].w = wk; a.s[1].y = yk; a.s[1].stride = k_stride;
  qk_streams(a, num_qo_heads, num_kv_heads);
  if (positions != nullptr) a.rot = rot_table(rope_theta);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == SMLM_F16 ? launch_qk_fwd<__half>(a, st) : launch_qk_fwd<__nv_bfloat16>(a, st);
}

size_t smlm_b200_qk_norm_rope_bwd_workspace_bytes(int T, int num_qo_heads, int num_kv_heads) {
  if (T <= 0 || num_qo_heads <= 0 || num_kv_heads <= 0) return 0;
  HeadNormArgs a = {};
  a.T = T;
  qk_bwd_streams(a, num_qo_heads, num_kv_heads);
  return static_cast<size_t>(a.s[0].ctas + a.s[1].ctas) * kPdDim * sizeof(float);
}

int smlm_b200_qk_norm_rope_bwd(void* dq, void* dk, void* dwq, void* dwk, const void* gq, const void* gk, const void* q,
                               const void* k, const void* wq, const void* wk, const void* positions, void* workspace,
                               size_t workspace_bytes, long long q_stride, long long k_stride, int T, int num_qo_heads,
                               int num_kv_heads, int head_dim, int positions_64, double rope_theta, float eps, int dtype,
                               void* stream) {
  const int rc = qk_check(q, k, wq, wk, positions, q_stride, k_stride, T, num_qo_heads, num_kv_heads, head_dim,
                          rope_theta, dtype);
  if (rc != SMLM_OK) return rc;
  if (T == 0) return SMLM_ERR_INVALID_ARGUMENT;   // a sum over no rows: the caller zeroes the weight gradients itself
  if (dq == nullptr || dk == nullptr || gq == nullptr || gk == nullptr) return SMLM_ERR_INVALID_ARGUMENT;
  if (!aligned16(dq) || !aligned16(dk) || !aligned16(gq) || !aligned16(gk)) return SMLM_ERR_MISALIGNED;
  const bool dw = wq != nullptr && (dwq != nullptr || dwk != nullptr);
  if (dw) {
    if (dwq == nullptr || dwk == nullptr) return SMLM_ERR_INVALID_ARGUMENT;
    if (workspace == nullptr ||
        workspace_bytes < smlm_b200_qk_norm_rope_bwd_workspace_bytes(T, num_qo_heads, num_kv_heads))
      return SMLM_ERR_WORKSPACE;
    if (!aligned16(workspace)) return SMLM_ERR_MISALIGNED;
  }
  HeadNormArgs a = {};
  a.positions = positions; a.T = T; a.pos64 = positions_64; a.eps = eps; a.partial = dw ? static_cast<float*>(workspace) : nullptr;
  a.s[0].x = q; a.s[0].w = wq; a.s[0].g = gq; a.s[0].y = dq; a.s[0].stride = q_stride;
  a.s[1].x = k; a.s[1].w = wk; a.s[1].g = gk; a.s[1].y = dk; a.s[1].stride = k_stride;
  qk_bwd_streams(a, num_qo_heads, num_kv_heads);
  if (positions != nullptr) a.rot = rot_table(rope_theta);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == SMLM_F16 ? launch_qk_bwd<__half>(a, dw ? dwq : nullptr, dwk, st)
                           : launch_qk_bwd<__nv_bfloat16>(a, dw ? dwq : nullptr, dwk, st);
}

}  // extern "C"
