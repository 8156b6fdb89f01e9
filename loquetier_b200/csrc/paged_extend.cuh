// Attention of a chunk of new tokens per request over its paged cache: between the decode kernel (one token) and the
// prefill kernels (whole prompts, which copy the batch's cache into a dense workspace first).
//
//   o[i, h] = sum_{j <= p_i} softmax_j( R(p_i) q[i, h] . R(j) k_j / sqrt(128) ) v_j,     p_i = L - n + i
//
// for the n new tokens of a request of L keys, which the cache already holds, un-rotated.  The pages are read in place.
// The rows of a request and kv head are its n * G (query, head) pairs, row = query * G + head of the group; they are cut into
// tiles, and the keys of a tile into ranges where there are too few tiles to fill the machine (few new tokens on a
// long cache).  A CTA owns one (tile, kv head, range).  Which one it finds for itself: the lengths live on the device.  The
// ranges follow from the lengths alone, so the same batch gives the same result; parked softmax states of a tile
// with several ranges are merged by a second launch, in range order.
#pragma once
#include "paged_kv.cuh"
#include "rotary.cuh"

namespace smlm {

constexpr int kExThreads = 128;

struct ExArgs {
  void* o;                        // [total_q, Nq, 128]
  const void* q;                  // [total_q, Nq, 128]
  const int32_t* qo_indptr;       // [B + 1]
  const void* const* kv_ptrs;
  const int32_t* kv_indptr;       // [B + 1]
  const int32_t* last_page_offset;  // [B]
  float* partial;                 // [slots * Nkv][rows of a tile][kPdRec]
  int* err;                       // error word, may be null
  int batch, total_q, total_pages, num_kv_heads, num_layers, layer_idx, page_size;
  int lg;                         // log2 of the query heads per kv head, G
  int target;                     // ranges aimed at per kv head
  int min_tiles;                  // a range has this many key tiles at least
  int slots;                      // (tile, range) pairs per kv head that the launch and the workspace provide for
  RotTable rot;
};

struct ExItem {
  int b;          // request; negative: the slot is not used
  int tile;       // of its rows
  int range, ranges;
  int slot0;      // the slot of the tile's first range
  int qo0, n;     // first row of q, new tokens
  int p0, len;    // first page in the table, keys
  int per;        // key tiles of a range
  int bad;        // error bits of its entries in the index arrays
};

// a request's rows and keys, with the index arrays checked
__device__ __forceinline__ void ex_request(const ExArgs& a, int b, ExItem& r) {
  const int q0 = a.qo_indptr[b], q1 = a.qo_indptr[b + 1];
  const int p0 = a.kv_indptr[b], p1 = a.kv_indptr[b + 1];
  const int last = a.last_page_offset[b];
  r.bad = 0;
  r.qo0 = q0;
  r.n = q1 - q0;
  if (q0 < 0 || q1 < q0 || q1 > a.total_q) {
    r.n = 0;
    r.bad = kErrBadIndptr;
  }
  r.p0 = p0;
  r.len = p1 > p0 ? (p1 - p0 - 1) * a.page_size + last : 0;
  if (p0 < 0 || p1 < p0 || p1 > a.total_pages || (p1 > p0 && (last < 0 || last > a.page_size))) {
    r.len = 0;
    r.bad = kErrBadIndptr;
  }
  if (r.len < r.n) r.bad = kErrBadIndptr;   // more queries than keys
}

// The (tile, range) that slot `slot` stands for.  ROWS rows and KEYS keys are a tile.  Requests come in order, a request's
// tiles in order, a tile's ranges in order.  Two passes over the requests: the batch's work gives the length of a range, the
// numbers of ranges the places.  Every thread of the CTA takes part; `report`: one of them writes down what is wrong with the
// index arrays.
template <int ROWS, int KEYS, int NT>
__device__ __forceinline__ ExItem ex_find(const ExArgs& a, int slot, bool report) {
  __shared__ long long s_sum[NT / 32];
  __shared__ int s_scan[NT / 32];
  __shared__ ExItem s_item;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  ExItem r;
  long long work = 0;
  for (int b = tid; b < a.batch; b += NT) {
    ex_request(a, b, r);
    if (report && r.bad != 0 && a.err != nullptr) atomicOr(a.err, r.bad);
    if (r.n > 0) work += static_cast<long long>(((r.n << a.lg) + ROWS - 1) / ROWS) * ((r.len + KEYS - 1) / KEYS);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) work += __shfl_xor_sync(0xffffffffu, work, d);
  if (lane == 0) s_sum[warp] = work;
  if (tid == 0) s_item.b = -1;
  __syncthreads();
  work = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) work += s_sum[w];
  const long long even = (work + a.target - 1) / a.target;
  const int per = static_cast<int>(even > a.min_tiles ? even : a.min_tiles);
  int before = 0;
  for (int b0 = 0; b0 < a.batch && before <= slot; b0 += NT) {
    const int b = b0 + tid;
    int tiles = 0, ranges = 0;
    if (b < a.batch) {
      if (a.batch > NT) ex_request(a, b, r);   // (else r still holds it)
      tiles = ((r.n << a.lg) + ROWS - 1) / ROWS;
      ranges = max(1, ((r.len + KEYS - 1) / KEYS + per - 1) / per);
    }
    const int mine = tiles * ranges;
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += up;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    int base = before, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      if (w < warp) base += s_scan[w];
      all += s_scan[w];
    }
    const int excl = base + incl - mine;
    if (mine > 0 && slot >= excl && slot - excl < mine) {
      const int local = slot - excl;
      r.b = b;
      r.tile = local / ranges;
      r.range = local % ranges;
      r.ranges = ranges;
      r.slot0 = slot - r.range;
      r.per = per;
      s_item = r;
    }
    before += all;
    __syncthreads();
  }
  return s_item;
}

// ---------------------------------------------------------------------------------------------
// few rows: mma.sync with the keys as the rows of the tile
// ---------------------------------------------------------------------------------------------

constexpr int kExRing = kPdWarps * kPdWarpRing;
constexpr int ex_rows(int nt) { return 8 * nt; }       // rows of a tile
// ring, queries, turns by 64 and by 8 keys, frequencies
constexpr int ex_smem(int nt) { return kExRing + ex_rows(nt) * kPdDim * 2 + 2 * 512 + 512; }
constexpr int ex_ctas_per_sm(int nt) { return nt >= 4 ? 2 : 3; }

// Like the decode kernel, with 8 NT rows in place of the heads of one token:
//   S^T[16 keys, 8 NT rows] = K . Q^T      O^T[128, 8 NT rows] += V^T . P^T       mma.sync m16n8k16
// Each warp streams every fourth tile of 16 keys through a ring of its own; a key is rotated once, in registers, for all
// rows.  Rotated keys and queries and the weights are rounded to 16 bits, the operands of the products; scores, maxima and
// sums are fp32.
template <typename T, int NT>
__global__ void __launch_bounds__(kExThreads, ex_ctas_per_sm(NT)) paged_extend_kernel(const __grid_constant__ ExArgs a) {
  extern __shared__ __align__(128) unsigned char ex_smem_buf[];
  constexpr int ROWS = 8 * NT;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;       // MMA fragment coordinates: row g, column pair t
  const uint32_t sbase = smem_u32(ex_smem_buf);
  const uint32_t qs = sbase + kExRing;
  float* rot = reinterpret_cast<float*>(ex_smem_buf + kExRing + ROWS * kPdDim * 2);
  float* freq = rot + 256;
  load_rot_table(a.rot, freq);

  pdl_wait();
  pdl_trigger();
  const int kvh = blockIdx.x % a.num_kv_heads, slot = blockIdx.x / a.num_kv_heads;
  const ExItem it = ex_find<ROWS, kPdTile, kExThreads>(a, slot, blockIdx.x == 0);
  if (it.b < 0) return;
  const int gmask = (1 << a.lg) - 1;
  const int Nq = a.num_kv_heads << a.lg, P = a.page_size;
  const int row0 = it.tile * ROWS;                    // of the request's n * G rows
  const int nrows = min(ROWS, (it.n << a.lg) - row0);
  const int pos0 = it.len - it.n;                     // position of the request's first new token
  const int pos_first = pos0 + (row0 >> a.lg), pos_last = pos0 + ((row0 + nrows - 1) >> a.lg);
  const int nkeys = max(0, min(it.len, pos_last + 1));
  const int ntiles = (nkeys + kPdTile - 1) / kPdTile;
  const int tile0 = it.range * it.per;
  const int ntl = max(0, min(ntiles, tile0 + it.per) - tile0);                      // tiles of this CTA
  const int ntw = ntl > warp ? (ntl - warp + kPdWarps - 1) / kPdWarps : 0;          // tiles of this warp

  // ---- the rotated, pre-scaled queries, the B operand: [ROWS][128] in shared memory ----
  {
    const int d0 = (tid & 15) * 4;            // dims d0..d0+3 and their partners d0+64..
    const float qscale = 1.4426950408889634f * rsqrtf(static_cast<float>(kPdDim));   // log2(e) / sqrt(d)
    uint2 uo[NT], up[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = (tid >> 4) + 8 * i;
      uo[i] = up[i] = make_uint2(0u, 0u);
      if (r < nrows) {
        const int rr = row0 + r;
        const T* qp = static_cast<const T*>(a.q) + (static_cast<size_t>(it.qo0 + (rr >> a.lg)) * Nq + (kvh << a.lg) + (rr & gmask)) * kPdDim + d0;
        uo[i] = __ldg(reinterpret_cast<const uint2*>(qp));
        up[i] = __ldg(reinterpret_cast<const uint2*>(qp + 64));
      }
    }
    // (the table is in shared memory since the barriers of ex_find)
    if (tid < 64) {
      float sn, cs;
      float* r = rot + (tid >> 1) * 4 + (tid & 1);
      rot_sincos(static_cast<float>(kPdStep), freq[tid], freq[64 + tid], &sn, &cs);
      r[0] = cs;
      r[2] = sn;
      rot_sincos(8.0f, freq[tid], freq[64 + tid], &sn, &cs);
      r[128] = cs;
      r[130] = sn;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = (tid >> 4) + 8 * i;
      const float pos = static_cast<float>(pos0 + ((row0 + r) >> a.lg));
      const float2 o0 = unpack2<T>(uo[i].x), o1 = unpack2<T>(uo[i].y), q0 = unpack2<T>(up[i].x), q1 = unpack2<T>(up[i].y);
      const float own[4] = {o0.x, o0.y, o1.x, o1.y}, par[4] = {q0.x, q0.y, q1.x, q1.y};
      float ro[4], rp[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float sn, cs;
        rot_sincos(pos, freq[d0 + k], freq[64 + d0 + k], &sn, &cs);
        ro[k] = (own[k] * cs - par[k] * sn) * qscale;
        rp[k] = (par[k] * cs + own[k] * sn) * qscale;
      }
      const int c_own = d0 >> 3, c_par = (d0 + 64) >> 3;
      const uint32_t off = (d0 & 7) * 2;
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(qs + r * 256 + ((c_own ^ (r & 7)) << 4) + off),
                   "r"(pack2<T>(ro[0], ro[1])), "r"(pack2<T>(ro[2], ro[3])) : "memory");
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(qs + r * 256 + ((c_par ^ (r & 7)) << 4) + off),
                   "r"(pack2<T>(rp[0], rp[1])), "r"(pack2<T>(rp[2], rp[3])) : "memory");
    }
  }
  __syncthreads();
  // B operand of k step ks (dimensions 16 ks ..) and of its partner ks + 4, rows 8 nt + g
  const uint32_t q_row = (lane & 7) * 256;
  const int q_chunk = ((lane >> 3) & 1) + ((lane >> 4) << 3);
  auto load_q = [&](int nt, int ks, uint32_t (&f)[4]) {
    ldsm_x4(f, qs + nt * 2048 + q_row + (((q_chunk + 2 * ks) ^ (lane & 7)) << 4));
  };
  uint32_t qf[NT == 1 ? 4 : 1][4];   // one column tile: kept in registers
  if (NT == 1) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) load_q(0, ks, qf[NT == 1 ? ks : 0]);
  }

  // ---- this warp's ring and its loader ----
  const uint32_t ring = sbase + warp * kPdWarpRing;
  const size_t head_off = (static_cast<size_t>(a.layer_idx) * 2 * a.num_kv_heads + kvh) * P * kPdDim;
  const size_t kv_delta = static_cast<size_t>(a.num_kv_heads) * P * kPdDim;
  bool bad_ptr = false;
  const int lp = 31 - __clz(P);   // the page size is a power of two (checked by the host)
  // The two halves of a tile (keys 0-7 and 8-15) each lie inside one page.  Their addresses are looked up one tile ahead, so
  // that the loads of the page table never sit in front of the copies.
  const T* half_ptr[2] = {nullptr, nullptr};
  auto lookup = [&](int j) {
    half_ptr[0] = half_ptr[1] = nullptr;
    if (j < ntw) {
      const int key0 = (tile0 + warp + j * kPdWarps) * kPdTile;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int gk = key0 + 8 * h;
        if (gk < nkeys) {
          const T* page = static_cast<const T*>(a.kv_ptrs[it.p0 + (gk >> lp)]);
          if (page == nullptr || (reinterpret_cast<uintptr_t>(page) & 15) != 0) bad_ptr = true;
          else half_ptr[h] = page + head_off + static_cast<size_t>(gk & (P - 1)) * kPdDim;
        }
      }
    }
  };
  // lane l copies chunk l & 15 of the keys 2 k + (l >> 4); chunk c of key e sits at slot c ^ (e & 7)
  const int cch = lane & 15, ckey = lane >> 4;
  const uint32_t dst_row = ckey * 256;
  auto issue = [&](int j) {   // j-th tile of this warp; its addresses were looked up before
    if (j < ntw) {
      const int key0 = (tile0 + warp + j * kPdWarps) * kPdTile;
      const uint32_t kst = ring + (j % kPdStages) * (2 * kPdTileBytes) + dst_row;
      const int valid = nkeys - key0 - ckey;   // key 2 k of this lane exists if 2 k < valid
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool have = half_ptr[h] != nullptr;
        const T* src = have ? half_ptr[h] + ckey * kPdDim + cch * 8 : static_cast<const T*>(a.q);
        const T* vsrc = have ? src + kv_delta : src;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool ok = have && 8 * h + 2 * k < valid;                    // keys past the end read as zeros
          const int step = ok ? 2 * k * kPdDim : 0;
          const uint32_t dst = kst + (8 * h + 2 * k) * 256 + ((cch ^ (2 * k + ckey)) << 4);
          cp_async16(dst, src + step, ok);
          cp_async16(dst + kPdTileBytes, vsrc + step, ok);
        }
      }
    }
    cp_async_commit();
    lookup(j + 1);
  };
  lookup(0);
#pragma unroll
  for (int j = 0; j < kPdStages - 1; ++j) issue(j);

  // cosines and sines of key g of the tile: pair p = 2 ks + h holds the frequencies 16 ks + 8 h + 2 t and the next
  uint64_t cc[8], ss[8];
  float m_run[NT][2], l_run[NT][2];          // rows 8 nt + 2 t and the next
  float o[NT][8][4];                         // dims 16 i + g and + 8 of those rows
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m_run[n][0] = m_run[n][1] = -INFINITY;
    l_run[n][0] = l_run[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
  }
  const int lm = lane >> 3, lr = lane & 7;
  const uint32_t k_row = ((lm & 1) * 8 + lr) * 256, k_x = ((lm >> 1) ^ lr) << 4;             // matrices: key half, dim half
  const uint32_t v_row = kPdTileBytes + ((lm >> 1) * 8 + lr) * 256, v_x = ((lm & 1) ^ lr) << 4;  // dim half, key half

  for (int j = 0; j < ntw; ++j) {
    issue(j + kPdStages - 1);
    const int key0 = (tile0 + warp + j * kPdWarps) * kPdTile;
    if (j % kPdReseed == 0) {
      const float pos = static_cast<float>(key0 + g);
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        float s0, s1, c0, c1;
        const int f = 8 * p + 2 * t;
        rot_sincos(pos, freq[f], freq[64 + f], &s0, &c0);
        rot_sincos(pos, freq[f + 1], freq[64 + f + 1], &s1, &c1);
        cc[p] = pack_f32x2(c0, c1);
        ss[p] = pack_f32x2(s0, s1);
      }
    }
    cp_async_wait<kPdStages - 1>();
    __syncwarp();
    const uint32_t kst = ring + (j % kPdStages) * (2 * kPdTileBytes);
    // S^T = K . Q^T with the keys rotated on the way
    float sc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      uint32_t own[4], par[4];
      const uint32_t ka = kst + k_row + (k_x ^ (ks << 5));
      ldsm_x4(own, ka);
      ldsm_x4(par, ka + 128);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int p = 2 * ks + h;
        const ulonglong2 t8 = *reinterpret_cast<const ulonglong2*>(rot + 128 + (4 * p + t) * 4);
        const ulonglong2 tw = *reinterpret_cast<const ulonglong2*>(rot + (4 * p + t) * 4);
        uint64_t c = cc[p], s = ss[p];
#pragma unroll
        for (int e = 0; e < 2; ++e) {   // key g, then key g + 8
          const float2 x = unpack2<T>(own[2 * h + e]), y = unpack2<T>(par[2 * h + e]);
          const uint64_t ko = pack_f32x2(x.x, x.y), kp = pack_f32x2(y.x, y.y);
          float a0, a1, b0, b1;
          unpack_f32x2(fma_f32x2(ko, c, mul_f32x2(kp, s ^ 0x8000000080000000ull)), a0, a1);   // ko c - kp s
          unpack_f32x2(fma_f32x2(kp, c, mul_f32x2(ko, s)), b0, b1);                           // kp c + ko s
          own[2 * h + e] = pack2<T>(a0, a1);
          par[2 * h + e] = pack2<T>(b0, b1);
          if (e == 0) turn_f32x2(c, s, t8.x, t8.y);
        }
        turn_f32x2(cc[p], ss[p], tw.x, tw.y);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t f[4];
        if (NT == 1) {
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = qf[NT == 1 ? ks : 0][i];
        } else {
          load_q(n, ks, f);
        }
        mma16816<T>(sc[n], own, f[0], f[1]);
        mma16816<T>(sc[n], par, f[2], f[3]);
      }
    }
    // running softmax: keys g and g + 8 of rows 8 n + 2 t and the next
    if (key0 + kPdTile - 1 > pos_first) {   // a row of the tile does not see all of these keys
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = row0 + 8 * n + 2 * t + (i & 1);
          if (key0 + g + (i >> 1) * 8 > min(pos0 + (row >> a.lg), pos_last)) sc[n][i] = -INFINITY;
        }
    }
    bool up = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
      up |= fmaxf(sc[n][0], sc[n][2]) > m_run[n][0] || fmaxf(sc[n][1], sc[n][3]) > m_run[n][1];
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float mx = fmaxf(sc[n][q], sc[n][q + 2]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float mn = fmaxf(m_run[n][q], mx);
          const float rescale = mn == -INFINITY ? 1.0f : exp2f(m_run[n][q] - mn);   // exp2f(-inf) = 0 on the first key
          m_run[n][q] = mn;
          l_run[n][q] *= rescale;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            o[n][i][q] *= rescale;
            o[n][i][q + 2] *= rescale;
          }
        }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float pr[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float m = m_run[n][i & 1];
        pr[i] = exp2f(sc[n][i] - (m == -INFINITY ? 0.f : m));   // a row that has seen no key yet: zeros
      }
      l_run[n][0] += pr[0] + pr[2];
      l_run[n][1] += pr[1] + pr[3];
      pb[n][0] = movm_t(pack2<T>(pr[0], pr[1]));
      pb[n][1] = movm_t(pack2<T>(pr[2], pr[3]));
    }
    // O^T += V^T . P^T ; P comes as [key][rows] and was transposed into the B operand
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t vf[4];
      ldsm_x4_t(vf, kst + v_row + ((i >> 2) << 7) + (v_x ^ ((i & 3) << 5)));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma16816<T>(o[n][i], vf, pb[n][0], pb[n][1]);
    }
    __syncwarp();   // the stage is free for the copy issued in the next iteration
  }
  cp_async_wait<0>();
  if (__any_sync(0xffffffffu, bad_ptr) && lane == 0 && a.err != nullptr) atomicOr(a.err, kErrBadPointer);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l_run[n][q] += __shfl_xor_sync(0xffffffffu, l_run[n][q], d);

  // ---- merge the warps in warp order, eight rows at a time: per (warp, row) m, l, 2 unused, o[128]; thread = dim ----
  float* red = reinterpret_cast<float*>(ex_smem_buf);
  constexpr int REC = kPdRec;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    __syncthreads();   // the rings, then the previous eight rows, are done with
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float* r = red + (warp * 8 + 2 * t + q) * REC;
      if (g == 0) {
        r[0] = m_run[n][q];
        r[1] = l_run[n][q];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        r[4 + 16 * i + g] = o[n][i][q];
        r[4 + 16 * i + 8 + g] = o[n][i][q + 2];
      }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 8; ++h) {
      const int row = 8 * n + h;
      if (row >= nrows) break;
      float m = -INFINITY, l = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < kPdWarps; ++w) {
        const float* r = red + (w * 8 + h) * REC;
        if (r[1] != 0.f) m = fmaxf(m, r[0]);   // an empty state carries no information
      }
#pragma unroll
      for (int w = 0; w < kPdWarps; ++w) {
        const float* r = red + (w * 8 + h) * REC;
        if (r[1] != 0.f) {
          const float wt = exp2f(r[0] - m);
          l += r[1] * wt;
          acc += r[4 + tid] * wt;
        }
      }
      if (it.ranges == 1) {
        const int rr = row0 + row;
        static_cast<T*>(a.o)[(static_cast<size_t>(it.qo0 + (rr >> a.lg)) * Nq + (kvh << a.lg) + (rr & gmask)) * kPdDim + tid] =
            static_cast<T>(l == 0.f ? 0.f : acc * (1.0f / l));   // no keys: zeros; a NaN stays one
      } else {
        float* r = a.partial + ((static_cast<size_t>(slot) * a.num_kv_heads + kvh) * ROWS + row) * REC;
        if (tid == 0) {
          r[0] = m;
          r[1] = l;
        }
        r[4 + tid] = acc;
      }
    }
  }
}

// Merges the parked states of tiles with several ranges, in range order.  The CTA of range r serves the tile's rows
// r, r + ranges, ...; thread = dim.
template <typename T, int ROWS, int KEYS>
__global__ void __launch_bounds__(kExThreads) paged_extend_merge_kernel(const __grid_constant__ ExArgs a) {
  // The index arrays were complete before the kernel in front started (it waited for them itself), so the search
  // needs no wait; the parked states do.
  const int kvh = blockIdx.x % a.num_kv_heads, slot = blockIdx.x / a.num_kv_heads;
  const ExItem it = ex_find<ROWS, KEYS, kExThreads>(a, slot, false);
  pdl_wait();
  pdl_trigger();
  if (it.b < 0 || it.ranges == 1) return;
  const int gmask = (1 << a.lg) - 1;
  const int Nq = a.num_kv_heads << a.lg;
  const int row0 = it.tile * ROWS;
  const int nrows = min(ROWS, (it.n << a.lg) - row0);
  const int ranges = min(it.ranges, a.slots - it.slot0);   // (an unsound table may ask for more than there is)
  const size_t next = static_cast<size_t>(a.num_kv_heads) * ROWS * kPdRec;
  for (int row = it.range; row < nrows; row += it.ranges) {
    const float* r = a.partial + ((static_cast<size_t>(it.slot0) * a.num_kv_heads + kvh) * ROWS + row) * kPdRec;
    float m = -INFINITY, l = 0.f, acc = 0.f;
    constexpr int U = 8;
    for (int z0 = 0; z0 < ranges; z0 += U) {   // eight states are requested together
      float mz[U], lz[U], oz[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        mz[u] = lz[u] = oz[u] = 0.f;
        if (z0 + u < ranges) {
          mz[u] = __ldcg(r + (z0 + u) * next);
          lz[u] = __ldcg(r + (z0 + u) * next + 1);
          oz[u] = __ldcg(r + (z0 + u) * next + 4 + threadIdx.x);
        }
      }
      float mn = m;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (lz[u] != 0.f) mn = fmaxf(mn, mz[u]);
      if (l != 0.f) {
        const float wt = exp2f(m - mn);
        l *= wt;
        acc *= wt;
      }
      m = mn;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (lz[u] != 0.f) {
          const float wt = exp2f(mz[u] - m);
          l += lz[u] * wt;
          acc += oz[u] * wt;
        }
      }
    }
    const int rr = row0 + row;
    static_cast<T*>(a.o)[(static_cast<size_t>(it.qo0 + (rr >> a.lg)) * Nq + (kvh << a.lg) + (rr & gmask)) * kPdDim + threadIdx.x] =
        static_cast<T>(l == 0.f ? 0.f : acc * (1.0f / l));
  }
}

}  // namespace smlm
