// Norms of queries and keys over each head's 128 dimensions, with the rotary position embedding in the same pass
// (training rows, forward and backward) or on the way into the paged cache (served rows; the cache keeps keys
// un-rotated).
//
//   s = rsqrt(mean(x^2) + eps)     n = x s w     y = R(p) n
//   R(p): dimensions i and i + 64 turned by the angle p base^(-2 i / 128)
//   backward:  dn = R(-p) dy     dw = sum over rows of x s dn     dx = s (w dn - x s^2 mean(w dn x))
//
// Everything is bound by HBM: a value is read once and written once, the norm's factor and the rotation are made in
// registers.  Eight lanes share a head - lane c holds dimensions 8 c .. 8 c + 7 and their partners 64 dimensions on, two
// 16-byte loads, no exchange for the rotation and three shuffles for the sum - so a warp has four heads in flight per
// step, and a lane meets the same eight frequencies for every head of its token: their sines are made once per token.
#pragma once
#include "paged_kv.cuh"
#include "rms_norm.cuh"
#include "rotary.cuh"

namespace smlm {

constexpr int kHnThreads = 256;
constexpr int kHnWarps = kHnThreads / 32;

// Queries and keys are two streams of (token, heads) units; a CTA works on one of them, so that its warps hold one set of
// weights (and, in the backward pass, of their gradients) in registers.
struct HeadNormStream {
  const void* x;            // [T, heads, 128], rows `stride` elements apart
  const void* w;            // [128], null: no norm
  const void* g;            // backward: gradient of the result, contiguous
  void* y;                  // forward: the result, backward: the gradient of x; contiguous
  long long stride;
  int heads;
  int splits;               // warps that share a token's heads
  int ctas;
};

struct HeadNormArgs {
  HeadNormStream s[2];      // queries, keys: the first s[0].ctas CTAs work on the queries
  const void* positions;    // int32 or int64 [T], null: no rotation
  float* partial;           // backward: [gridDim.x][128] shares of the weights' gradients
  int T, pos64;
  float eps;
  RotTable rot;
};

// the lane's eight cosines and sines at a token's position; freq: the table in shared memory
template <bool ROPE>
__device__ __forceinline__ void token_rotation(const HeadNormArgs& a, const float* freq, int t, int c, float (&cs)[8],
                                               float (&sn)[8]) {
  if (ROPE) {
    const float pos = a.pos64 ? static_cast<float>(static_cast<const long long*>(a.positions)[t])
                              : static_cast<float>(static_cast<const int*>(a.positions)[t]);
#pragma unroll
    for (int i = 0; i < 8; ++i) rot_sincos(pos, freq[c * 8 + i], freq[64 + c * 8 + i], &sn[i], &cs[i]);
  }
}

__device__ __forceinline__ float sum8(float v) {   // over the eight lanes of a head
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  return v;
}

// forward of the heads first .. first + 3, then `step` further on, of one token; x and y point at the token's first head,
// hl is the lane's head within four
template <typename T, bool NORM, bool ROPE, int U>
__device__ __forceinline__ void heads_forward(const T* x, T* y, int heads, int first, int step, const float (&w)[16],
                                              const float (&cs)[8], const float (&sn)[8], int c, int hl, float eps) {
  for (int h0 = first; h0 < heads; h0 += U * step) {   // uniform over the warp
    uint4 lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + hl + u * step;
      lo[u] = hi[u] = make_uint4(0u, 0u, 0u, 0u);
      if (h < heads) {
        lo[u] = __ldg(reinterpret_cast<const uint4*>(x + h * kPdDim + c * 8));
        hi[u] = __ldg(reinterpret_cast<const uint4*>(x + h * kPdDim + 64 + c * 8));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + hl + u * step;
      float p[8], q[8];
      unpack8<T>(lo[u], p);
      unpack8<T>(hi[u], q);
      if (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += p[i] * p[i] + q[i] * q[i];
        const float s = rsqrtf(sum8(ss) * (1.0f / kPdDim) + eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] *= s * w[i];
          q[i] *= s * w[8 + i];
        }
      }
      if (ROPE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float r = p[i] * cs[i] - q[i] * sn[i];
          q[i] = q[i] * cs[i] + p[i] * sn[i];
          p[i] = r;
        }
      }
      if (h < heads) {
        *reinterpret_cast<uint4*>(y + h * kPdDim + c * 8) = pack8<T>(p);
        *reinterpret_cast<uint4*>(y + h * kPdDim + 64 + c * 8) = pack8<T>(q);
      }
    }
  }
}

// the lane's sixteen weights of a head
template <typename T, bool NORM>
__device__ __forceinline__ void load_weight(const void* w, int c, float (&f)[16]) {
  if (NORM) {
    float a[8], b[8];
    unpack8<T>(__ldg(static_cast<const uint4*>(w) + c), a);
    unpack8<T>(__ldg(static_cast<const uint4*>(w) + 8 + c), b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] = a[i];
      f[8 + i] = b[i];
    }
  }
}

// One warp per (token, share of its heads).  Measured, 8192 tokens of 32 / 8 heads, bf16 (168 MB, 26 us at the copy rate):
// 31 us; 37 with both sets of weights in registers (two CTAs per SM instead of three).
template <typename T, bool NORM, bool ROPE>
__global__ void __launch_bounds__(kHnThreads, 3) qk_norm_rope_kernel(const __grid_constant__ HeadNormArgs a) {
  __shared__ __align__(16) float freq[ROPE ? 128 : 4];
  const int lane = threadIdx.x & 31, c = lane & 7, hl = lane >> 3;
  if (ROPE) {
    load_rot_table(a.rot, freq);
    __syncthreads();
  }
  pdl_wait();
  pdl_trigger();
  const bool keys = blockIdx.x >= a.s[0].ctas;
  const HeadNormStream& st = a.s[keys];
  const unsigned unit = (blockIdx.x - (keys ? a.s[0].ctas : 0)) * kHnWarps + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / st.splits), sp = static_cast<int>(unit % st.splits);
  if (t >= a.T) return;
  float w[16], cs[8], sn[8];
  load_weight<T, NORM>(st.w, c, w);
  token_rotation<ROPE>(a, freq, t, c, cs, sn);
  heads_forward<T, NORM, ROPE, 2>(static_cast<const T*>(st.x) + t * st.stride,
                                  static_cast<T*>(st.y) + static_cast<size_t>(t) * st.heads * kPdDim, st.heads, sp * 4,
                                  4 * st.splits, w, cs, sn, c, hl, a.eps);
}

constexpr int kHnAhead = 3;                          // fours of heads on their way per warp
constexpr int kHnStage = 4 * 512;                    // of four heads: gradient and input, two halves of a head's row each
constexpr int kHnRing = (kHnAhead + 1) * kHnStage;
constexpr int kHnSmem = kHnWarps * kHnRing;

// eight 16-bit values as four packed pairs of fp32, and back
template <typename T>
__device__ __forceinline__ void pairs8(const uint4& u, uint64_t* f) {
  const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y), c = unpack2<T>(u.z), d = unpack2<T>(u.w);
  f[0] = pack_f32x2(a.x, a.y);
  f[1] = pack_f32x2(b.x, b.y);
  f[2] = pack_f32x2(c.x, c.y);
  f[3] = pack_f32x2(d.x, d.y);
}
template <typename T>
__device__ __forceinline__ uint4 packed8(const uint64_t* f) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    unpack_f32x2(f[i], a, b);
    r[i] = pack2<T>(a, b);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// Warps walk over (token, share of its heads) with a fixed stride, four heads at a time, and keep their share of dw in fp32
// registers; the CTA adds its warps' in warp order and parks one row, which head_norm_dw_kernel adds in row order: the same
// result each time.  Bound by HBM, so by what is in flight: a warp has the next kHnAhead fours on their way, as asynchronous
// copies into a ring of its own in shared memory (a lane reads back what it copied: no barrier).  Measured, 8192 tokens of
// 32 / 8 heads, bf16 (252 MB, 39 us at the copy rate): 82 us with both sets of weights and gradients in registers (one CTA
// per SM), 50 with one stream per CTA and the next four heads requested ahead, 48 with the ring and packed arithmetic.
template <typename T, bool NORM, bool ROPE>
__global__ void __launch_bounds__(kHnThreads, 2) qk_norm_rope_bwd_kernel(const __grid_constant__ HeadNormArgs a) {
  extern __shared__ __align__(16) unsigned char hn_ring[];
  __shared__ __align__(8) float red[NORM ? kHnWarps : 1][kPdDim];
  __shared__ __align__(16) float freq[ROPE ? 128 : 4];
  const int lane = threadIdx.x & 31, c = lane & 7, hl = lane >> 3, warp = threadIdx.x >> 5;
  if (ROPE) {
    load_rot_table(a.rot, freq);
    __syncthreads();
  }
  pdl_wait();
  pdl_trigger();
  const bool keys = blockIdx.x >= a.s[0].ctas;
  const HeadNormStream& st = a.s[keys];
  const int heads = st.heads, step = 4 * st.splits;
  uint64_t w[8], dw[8] = {}, cs[4], sn[4];   // pairs
  if (NORM) {
    pairs8<T>(__ldg(static_cast<const uint4*>(st.w) + c), w);
    pairs8<T>(__ldg(static_cast<const uint4*>(st.w) + 8 + c), w + 4);
  }
  // (few tokens are split, many are not: the numbers of units stay below 2^32)
  const unsigned units = static_cast<unsigned>(a.T) * st.splits, stride = static_cast<unsigned>(st.ctas) * kHnWarps;
  unsigned unit = (blockIdx.x - (keys ? a.s[0].ctas : 0)) * kHnWarps + warp;
  int t = static_cast<int>(unit / st.splits), h0 = static_cast<int>(unit % st.splits) * 4;   // where the loads are
  const uint32_t ring = smem_u32(hn_ring) + warp * kHnRing + lane * 16;
  auto request = [&](int stage) {
    const int h = h0 + hl;
    const bool ok = unit < units && h < heads;
    const T* g = static_cast<const T*>(st.g);
    if (ok) g += (static_cast<size_t>(t) * heads + h) * kPdDim + c * 8;
    const uint32_t dst = ring + stage * kHnStage;
    cp_async16(dst, g, ok);
    cp_async16(dst + 512, g + (ok ? 64 : 0), ok);
    if (NORM) {
      const T* x = static_cast<const T*>(st.x);
      if (ok) x += t * st.stride + h * kPdDim + c * 8;
      cp_async16(dst + 1024, x, ok);
      cp_async16(dst + 1536, x + (ok ? 64 : 0), ok);
    }
    cp_async_commit();
  };
  auto advance = [&](unsigned& u, int& tok, int& head) {
    head += step;
    if (head >= heads) {
      u += stride;
      tok = static_cast<int>(u / st.splits);
      head = static_cast<int>(u % st.splits) * 4;
    }
  };
  unsigned cu = unit;   // where the work is
  int ct = t, ch = h0, stage = 0;
#pragma unroll
  for (int i = 0; i < kHnAhead; ++i) {
    request(i);
    advance(unit, t, h0);
  }
  int at = -1;   // the token that the cosines and sines belong to
  while (cu < units) {   // uniform over the warp
    const int h = ch + hl, tok = ct;
    const int free_stage = stage == 0 ? kHnAhead : stage - 1;   // of the four before this one
    request(free_stage);
    advance(unit, t, h0);
    cp_async_wait<kHnAhead>();
    // pairs of neighbouring dimensions, [0..3] of the lane's eight and [4..7] of their partners: the gradient in front of
    // the rotation, and the input
    uint64_t d[8], x[8];
    const unsigned char* from = hn_ring + warp * kHnRing + stage * kHnStage + lane * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      pairs8<T>(*reinterpret_cast<const uint4*>(from + i * 512), d + 4 * i);
      if (NORM) pairs8<T>(*reinterpret_cast<const uint4*>(from + 1024 + i * 512), x + 4 * i);
    }
    stage = stage == kHnAhead ? 0 : stage + 1;
    advance(cu, ct, ch);
    if (ROPE && tok != at) {
      float c8[8], s8[8];
      token_rotation<ROPE>(a, freq, tok, c, c8, s8);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cs[i] = pack_f32x2(c8[2 * i], c8[2 * i + 1]);
        sn[i] = pack_f32x2(s8[2 * i], s8[2 * i + 1]);
      }
      at = tok;
    }
    constexpr uint64_t kNeg2 = 0x8000000080000000ull;   // flips the sign of both halves
    if (ROPE) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t r = fma_f32x2(d[i], cs[i], mul_f32x2(d[4 + i], sn[i]));
        d[4 + i] = fma_f32x2(d[4 + i], cs[i], mul_f32x2(d[i], sn[i] ^ kNeg2));
        d[i] = r;
      }
    }
    if (NORM) {
      uint64_t ss2 = 0ull, dot2 = 0ull, wd[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss2 = fma_f32x2(x[i], x[i], ss2);
        wd[i] = mul_f32x2(w[i], d[i]);
        dot2 = fma_f32x2(wd[i], x[i], dot2);
      }
      float u, v;
      unpack_f32x2(ss2, u, v);
      const float mean = sum8(u + v) * (1.0f / kPdDim) + a.eps;
      // (lanes behind the last head hold zeros: without an epsilon their factor would be infinite, and their share of dw a NaN)
      const float s = h < heads ? rsqrtf(mean) : 0.f;
      unpack_f32x2(dot2, u, v);
      const float coef = -sum8(u + v) * s * s * (1.0f / kPdDim);
      const uint64_t s2 = pack_f32x2(s, s), coef2 = pack_f32x2(coef, coef);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint64_t xs = mul_f32x2(x[i], s2);
        dw[i] = fma_f32x2(xs, d[i], dw[i]);
        d[i] = fma_f32x2(xs, coef2, mul_f32x2(wd[i], s2));
      }
    }
    if (h < heads) {
      T* dx = static_cast<T*>(st.y) + (static_cast<size_t>(tok) * heads + h) * kPdDim + c * 8;
      __stcs(reinterpret_cast<uint4*>(dx), packed8<T>(d));
      __stcs(reinterpret_cast<uint4*>(dx + 64), packed8<T>(d + 4));
    }
  }
  cp_async_wait<0>();
  if (NORM && a.partial != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float u, v;
      unpack_f32x2(dw[i], u, v);
#pragma unroll
      for (int m = 8; m < 32; m <<= 1) {
        u += __shfl_xor_sync(0xffffffffu, u, m);
        v += __shfl_xor_sync(0xffffffffu, v, m);
      }
      if (hl == 0) *reinterpret_cast<float2*>(&red[warp][(i >> 2) * 64 + c * 8 + (i & 3) * 2]) = make_float2(u, v);
    }
    __syncthreads();
    if (threadIdx.x < kPdDim) {
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < kHnWarps; ++v) sum += red[v][threadIdx.x];
      a.partial[static_cast<size_t>(blockIdx.x) * kPdDim + threadIdx.x] = sum;
    }
  }
}

// dwq and dwk: the parked rows of each added in a fixed order.  A CTA owns eight of the 256 columns; thread (r, col) adds the
// rows r, r + 32, ... and the 32 sums of a column are added in a tree over the lanes that hold them.
template <typename T>
__global__ void __launch_bounds__(256) head_norm_dw_kernel(void* dwq, void* dwk, const float* __restrict__ partial, int q_rows,
                                                           int rows) {
  __shared__ float red[32][9];
  const int col = threadIdx.x & 7, r = threadIdx.x >> 3;
  const bool keys = blockIdx.x >= kPdDim / 8;
  const int dim0 = (blockIdx.x % (kPdDim / 8)) * 8;
  pdl_wait();
  pdl_trigger();
  float t = 0.f;
  for (int i = (keys ? q_rows : 0) + r; i < (keys ? rows : q_rows); i += 32)
    t += __ldcg(partial + static_cast<size_t>(i) * kPdDim + dim0 + col);
  red[r][col] = t;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float v = red[lane][warp];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (lane == 0) static_cast<T*>(keys ? dwk : dwq)[dim0 + warp] = static_cast<T>(v);
}

// ---------------------------------------------------------------------------------------------
// the served rows: normalised queries out, normalised keys and the values into the pages
// ---------------------------------------------------------------------------------------------

struct NormAppendArgs {
  const void* q;            // [T, Nq, 128], rows q_stride elements apart
  const void* k;            // [T, Nk, 128]
  const void* v;
  const void* wq;
  const void* wk;
  void* yq;                 // [T, Nq, 128] contiguous
  const void* const* kv_ptrs;
  const int32_t* kv_indptr;
  const int32_t* last_page_offset;
  const int32_t* append_indptr;   // [B + 1]; null: one token per request
  int* err;
  long long q_stride, k_stride, v_stride;
  int T, batch, Nq, Nk, num_layers, layer_idx, page_size, total_pages, splits;
  float eps;
};

// One warp per (token, share of its heads).  Measured: 10622 tokens of 32 / 8 heads in 12 prompts, fp16 (261 MB, 40 us at the
// copy rate): 39 us; 64 single tokens: 6 us, latency.
template <typename T>
__global__ void __launch_bounds__(kHnThreads) norm_append_kernel(const NormAppendArgs a) {
  const int lane = threadIdx.x & 31, c = lane & 7, hl = lane >> 3;
  pdl_wait();
  pdl_trigger();
  const unsigned unit = blockIdx.x * kHnWarps + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / a.splits), sp = static_cast<int>(unit % a.splits);
  if (t >= a.T) return;
  // the request of the token: how many of them start at or before it (every lane looks at some, all loads at once)
  int b = t, t0 = t, n = 1;
  if (a.append_indptr != nullptr) {
    int before = 0;
    for (int i0 = 0; i0 < a.batch; i0 += 32) {
      const int i = i0 + lane;
      before += __popc(__ballot_sync(0xffffffffu, i < a.batch && a.append_indptr[i] <= t));
    }
    b = before - 1;
    if (b < 0) return;                       // a row in front of the first request
    t0 = a.append_indptr[b];
    n = a.append_indptr[b + 1] - t0;
    if (t - t0 >= n) return;                 // a row behind the last one
  }
  float wq[16], wk[16];
  const float none[8] = {};
  load_weight<T, true>(a.wq, c, wq);
  load_weight<T, true>(a.wk, c, wk);
  const int first = sp * 4, step = 4 * a.splits;
  heads_forward<T, true, false, 2>(static_cast<const T*>(a.q) + t * a.q_stride,
                                   static_cast<T*>(a.yq) + static_cast<size_t>(t) * a.Nq * kPdDim, a.Nq, first, step, wq,
                                   none, none, c, hl, a.eps);
  const int p0 = a.kv_indptr[b], p1 = a.kv_indptr[b + 1], P = a.page_size;
  const int len = p1 > p0 ? (p1 - p0 - 1) * P + a.last_page_offset[b] : 0;
  const int pos = len - n + (t - t0);
  if (p0 < 0 || p1 > a.total_pages || pos < 0 || n > len || pos >= (p1 - p0) * P) {   // the pages do not hold the token
    if (lane == 0 && a.err != nullptr) atomicOr(a.err, kErrBadIndptr);
    return;
  }
  T* page = static_cast<T*>(const_cast<void*>(a.kv_ptrs[p0 + pos / P]));
  if (page == nullptr || (reinterpret_cast<uintptr_t>(page) & 15) != 0) {
    if (lane == 0 && a.err != nullptr) atomicOr(a.err, kErrBadPointer);
    return;
  }
  // a head's place: [layer][key | value][head][entry][128]
  const size_t head_step = static_cast<size_t>(P) * kPdDim;
  T* kd = page + static_cast<size_t>(a.layer_idx) * 2 * a.Nk * head_step + static_cast<size_t>(pos % P) * kPdDim + c * 8;
  const T* ks = static_cast<const T*>(a.k) + t * a.k_stride + c * 8;
  const T* vs = static_cast<const T*>(a.v) + t * a.v_stride + c * 8;
  for (int h0 = first; h0 < a.Nk; h0 += step) {
    const int h = h0 + hl;
    uint4 kl = make_uint4(0u, 0u, 0u, 0u), kh = kl, vl = kl, vh = kl;
    if (h < a.Nk) {
      kl = __ldg(reinterpret_cast<const uint4*>(ks + h * kPdDim));
      kh = __ldg(reinterpret_cast<const uint4*>(ks + h * kPdDim + 64));
      vl = __ldg(reinterpret_cast<const uint4*>(vs + h * kPdDim));
      vh = __ldg(reinterpret_cast<const uint4*>(vs + h * kPdDim + 64));
    }
    float p[8], q[8];
    unpack8<T>(kl, p);
    unpack8<T>(kh, q);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += p[i] * p[i] + q[i] * q[i];
    const float s = rsqrtf(sum8(ss) * (1.0f / kPdDim) + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] *= s * wk[i];
      q[i] *= s * wk[8 + i];
    }
    if (h < a.Nk) {
      T* dst = kd + h * head_step;
      *reinterpret_cast<uint4*>(dst) = pack8<T>(p);
      *reinterpret_cast<uint4*>(dst + 64) = pack8<T>(q);
      dst += a.Nk * head_step;
      *reinterpret_cast<uint4*>(dst) = vl;
      *reinterpret_cast<uint4*>(dst + 64) = vh;
    }
  }
}

}  // namespace smlm
