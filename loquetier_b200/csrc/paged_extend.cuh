// Attention of a chunk of new tokens per request over its paged cache: between the decode kernel (one token) and the
// prefill kernels (whole prompts, which copy the batch's cache into a dense workspace first).
//
//   o[i, h] = sum_{j <= p_i} softmax_j( R(p_i) q[i, h] . R(j) k_j / sqrt(128) ) v_j,     p_i = L - n + i
//
// for the n new tokens of a request of L keys, which the cache already holds, un-rotated.
//
// The rows of a request and kv head are its n * G (query, head) pairs, row = query * G + head of the group, cut into tiles
// of 32 QT rows; the keys are cut into tiles of 64.  All (request, row tile, key tile) triples of a kv head, in this order,
// are the work, and every CTA of that head takes an even, contiguous share of it: a long cache is spread over many CTAs,
// several short ones follow one another in one, and the launch is one wave that ends everywhere at once whatever the
// lengths.  A CTA finds its share itself, because the lengths live on the device.  A row tile that lies in one share is finished
// there; one that is cut leaves a softmax state per share, merged by a second launch in the order of the keys.  The cuts
// follow from the lengths alone: the same batch gives the same result.
//
//   S[128, 64]   = Q . K_tile^T    tcgen05.mma, both operands K-major in shared memory, two accumulators in tensor memory
//   P            = exp2(S - m)     a row is a tensor-memory lane, two threads per row (one where the keys are rotated in front)
//   O[128, 128] += P . V_tile      A = P in tensor memory, B = V MN-major as the cache stores it
//
// The products and the softmax are those of the prefill kernel (paged_prefill.cuh).  What differs is where the tiles come
// from: that kernel has the batch's cache copied into a dense workspace first, three times the bytes.  Here two warps, one for K
// and one for V, fetch the tiles from the pages themselves with 16-byte asynchronous copies, straight into the swizzled
// places the products read, and run ahead across row tiles and requests; four warps rotate the keys in place.  A rotator thread
// has eight frequencies (dimensions 8 c .. 8 c + 7 and their partners) and a fixed distance between its keys, so its cosines
// and sines go on from key to key by one turn and are computed afresh every 16 tiles: 63 turns at most, after which they are off
// by 2^-15.5 (measured; 2^-20.4 afresh), a twentieth of the rounding that an fp16 key gets next.
// Chunks of several row tiles would rotate every key several times: for them the keys are rotated once, in front, into a
// dense copy (DENSE; the values stay where they are).
//
// The products always have 128 rows; what lies behind the tile's rows in shared memory feeds accumulator lanes that nobody
// reads.  Softmax warps are those whose tensor-memory lanes hold the tile's rows, and warps of an empty quarter only pass
// hand-offs on.  Every wait is bounded.
//
// Rounded to 16 bits, as the operands of the products: rotated queries and keys and the softmax weights; with the result's own
// rounding the error against 64 bits is 3.3e-3 (bf16) and 4.1e-4 (fp16) of the result, where the result's rounding alone is
// 1.7e-3 and 2.1e-4.  Keeping the lower halves too (products of twice the depth) would take the shared memory of a stage
// of the rings and half of the tensor cores' time again.  Scores, maxima, sums and parked states are fp32.
//
// What bounds it (32 / 8 heads, B200).  32 requests, 512..4096 keys, 4 to 8 new tokens (285 MB, 44 us at the copy rate), 82 us a
// pass: the launch 76, of which 5 are the search for the share and cold instructions, 5 the first tile, and the loop runs at
// about the rate the pages arrive; the merge 5.  One request, 65 k keys, 17 tokens (269 MB): 81 us.  16 requests of 20 to 120
// tokens, 32 heads (695 MB): 200 to 208.  With the rotation, the softmax and most of the products taken out, the copies and the
// hand-offs between the roles alone take 73, 73 and 151 us (5.4 TB/s behind the start and in front of the merge), the hand-offs
// without copies 45, 43 and 94: what is left to gain in this form lies in the copies and the start, not in the arithmetic, but
// for tiles of 128 rows, where rotation, softmax and products each lengthen a tile's way through the rings by 10 to 25 us.  Copies
// started early, into L2, gain nothing.  4 requests of 400 to 512 tokens on 4 k to 12 k keys, 32 / 8 heads (160 GFLOP, 98 us): 241 to 247 where the inputs change
// from pass to pass, 219 on the same ones; by the launch 20 for the keys' rotation in front, 197, 12 for the merge.  The tensor
// pipe is active 47 %, between hand-offs of P and S.
// History on the first: one CTA per (row tile, range of keys) 146 us (CTAs of unequal length); even shares 100; roles whose
// registers fit (spills in the loaders' loop) 94; copies and rotation in warps of their own 91; descriptors formed by one
// addition, one barrier fewer, waits that sleep 84; key tiles counted exactly 82.  Waits that spin cost 5-15 % (they take
// issue slots), eight rotator warps measured the same as four, mma.sync with 8, 16 or 32 rows per tile 130-166 us.
#pragma once
#include "paged_prefill.cuh"
#include "rms_norm.cuh"
#include "rotary.cuh"

namespace smlm {

constexpr int kXtKeys = 64;
constexpr int kXtCtasPerSm = 2;
constexpr int kXtTileBytes = kXtKeys * kPdDim * 2;      // two 64-dim panels of [64 keys][128 B]
constexpr int kXtPanel = kXtKeys * 128;
constexpr int kXtOCol = 2 * kXtKeys;                    // tensor memory: two S buffers, then O
constexpr int kXtTmemCols = 256;
constexpr int kXtHalf = kXtKeys / 2;                    // columns of S per softmax thread
constexpr int kXtReseed = 16;                           // tiles after which the rotation is computed afresh

struct ExCut;

struct ExArgs {
  void* o;                        // [total_q, Nq, 128]
  const void* q;                  // [total_q, Nq, 128]
  const int32_t* qo_indptr;       // [B + 1]
  const void* const* kv_ptrs;
  const int32_t* kv_indptr;       // [B + 1]
  const int32_t* last_page_offset;  // [B]
  float* partial;                 // states [shares][2][Nkv][rows of a tile][kPdRec]: a share cuts two row tiles at most
  ExCut* cuts;                    // [shares][Nkv]
  void* dense;                    // rotated keys [Nkv][total_pages * page_size][128], or null
  int* err;                       // error word, may be null
  int batch, total_q, total_pages, num_kv_heads, num_layers, layer_idx, page_size;
  int lg;                         // log2 of the query heads per kv head, G
  int shares;                     // CTAs per kv head
  int min_tiles;                  // a share has this many key tiles at least
  RotTable rot;
};

struct ExRequest {
  int qo0, n;     // first row of q, new tokens
  int p0, len;    // first page in the table, keys
  int bad;        // error bits of its entries in the index arrays
};

__device__ __forceinline__ ExRequest ex_request(const ExArgs& a, int b) {
  const int q0 = a.qo_indptr[b], q1 = a.qo_indptr[b + 1];
  const int p0 = a.kv_indptr[b], p1 = a.kv_indptr[b + 1];
  const int last = a.last_page_offset[b];
  ExRequest r;
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
  return r;
}
template <int ROWS>
__device__ __forceinline__ int ex_row_tiles(const ExArgs& a, const ExRequest& r) {
  return ((r.n << a.lg) + ROWS - 1) / ROWS;
}
// Key tiles of a request's row tiles in front of row tile x, together: the keys that the last row of each sees, in tiles of
// 64.  Row tile t ends with query (t + 1) q - 1, q the queries of a row tile, and sees pos0 + (t + 1) q keys, the last one
// all; q is a power of two, so the sum has a closed form.  A request with more queries than keys (an error) counts all of its
// keys for every row tile, one tile at least: its rows have to be written.
template <int ROWS>
__device__ __forceinline__ int ex_before(const ExArgs& a, const ExRequest& r, int x) {
  const int all = ex_row_tiles<ROWS>(a, r);
  const int most = max(1, (r.len + kXtKeys - 1) / kXtKeys);
  if (r.len < r.n) return x * most;
  const int y = min(x, all - 1);                      // of these the closed form holds
  const int lq = 31 - __clz(ROWS) - a.lg;             // log2 of q
  const int first = r.len - r.n + (1 << lq) + kXtKeys - 1;   // row tile t: (first + t q) / 64, rounded down
  int sum;
  if (lq >= 6) {
    sum = y * (first >> 6) + static_cast<int>((static_cast<unsigned>(y) * (y - 1)) >> 1 << (lq - 6));
  } else {                                            // the quotients go up by one every m = 64 / q row tiles
    const int lm = 6 - lq, f = first >> lq;
    auto steps = [&](unsigned i) {                    // sum of j >> lm for j < i, modulo 2^32: the difference is what counts
      const unsigned t = i >> lm;
      return (((t & 1) ? t * ((t - 1) >> 1) : (t >> 1) * (t - 1)) << lm) + t * (i - (t << lm));
    };
    sum = static_cast<int>(steps(f + y) - steps(f));
  }
  return x == all ? sum + most : sum;
}
template <int ROWS>
__device__ __forceinline__ int ex_work(const ExArgs& a, const ExRequest& r) {
  return r.n > 0 ? ex_before<ROWS>(a, r, ex_row_tiles<ROWS>(a, r)) : 0;
}

// A run of key tiles of one row tile.
struct ExSeg {
  int qo0, row0, nrows;   // first row of q of the request; of its rows, the tile's first and their number
  int pos0, p0;           // position of the request's first new token; first page in the table
  int nkeys;              // keys that a row of the tile sees
  int tile0, ntiles;      // the run
  int part;               // where its state goes: 0, 1, or negative: the row tile is finished here
};

template <int SEGS>
struct ExScratch {
  long long sum[16];
  int begin, end, next;         // of the share's work; where the next round of runs starts
  int count;
  unsigned bad_v;               // runs with a value that is not finite behind some of the rows
  ExSeg seg[SEGS];              // runs of the share that are laid out at a time
};

// Running sums over the CTA's threads in their order: returns what the threads before this one hold, `all` the whole.  Where only
// the first warp's threads hold anything (up to 32 requests) it does without the others, for whom `all` is nothing: whatever
// follows from it is the first warp's as well.
template <int NT, typename S>
__device__ __forceinline__ long long ex_scan(long long v, long long& all, S& sc, bool one_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (one_warp) {
    all = __shfl_sync(0xffffffffu, incl, 31);
    return incl - v;
  }
  __syncthreads();
  if (lane == 31) sc.sum[warp] = incl;
  __syncthreads();
  long long base = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) base += sc.sum[w];
    all += sc.sum[w];
  }
  return base + incl - v;
}

// What the merge of the row tile that a share starts inside of needs to know.
struct ExCut {
  int qo0, row0, nrows;   // as in ExSeg; no rows: the share starts a row tile, or holds no work
  int first, shares;      // the row tile's first share, and how many more it lies in: that many CTAs merge
  int part;               // where the first share has its state; the others have it at 0
  int pos0;               // as in ExSeg
  int pad;
};

// keys that a row of row tile `tile` of the request sees
template <int ROWS>
__device__ __forceinline__ int ex_visible(const ExArgs& a, const ExRequest& r, int tile) {
  const int last = min((r.n << a.lg), (tile + 1) * ROWS) - 1;
  return max(0, min(r.len, r.len - r.n + (last >> a.lg) + 1));
}

// What a row of weight sum l at position pos is multiplied by.  A row that sees no key is zeros; one that sees keys, but none whose
// score is above -inf (products that leave fp32's range), has no answer, and a NaN says so.  A NaN stays one.
__device__ __forceinline__ float row_scale(float l, int pos) {
  return l != 0.f ? 1.0f / l : pos < 0 ? 0.f : __int_as_float(0x7fffffff);
}

// A thread's request of those that the CTA looks at together, its work and its place in the head's work.
struct ExMine {
  ExRequest r;
  int work, at;
};

// Requests b0 + thread; `before`: the work in front of them, and behind them on return
template <int ROWS, int NT, typename S>
__device__ __forceinline__ ExMine ex_mine(const ExArgs& a, int b0, long long& before, S& sc) {
  const int b = b0 + threadIdx.x;
  ExMine m = {};
  if (b < a.batch) {
    m.r = ex_request(a, b);
    m.work = ex_work<ROWS>(a, m.r);
  }
  long long all;
  const long long at = before + ex_scan<NT>(m.work, all, sc, a.batch <= 32);
  before += all;
  m.at = static_cast<int>(min(at, 0x7fffffffLL));   // (more work than that is refused, see ex_share)
  return m;
}

// Key tiles of a share, 0 where the index arrays make no sense together.  m: the first NT requests.  `report`: what is wrong
// with the index arrays is written down.
template <int ROWS, int NT, typename S>
__device__ __forceinline__ int ex_share(const ExArgs& a, bool report, ExMine& m, S& sc) {
  long long work = 0;
  int bad = 0;
  for (int b0 = 0; b0 < a.batch; b0 += NT) {
    const ExMine next = ex_mine<ROWS, NT>(a, b0, work, sc);
    bad |= next.r.bad;
    if (b0 == 0) m = next;
  }
  if (work > 0x7fffffffLL - kXtKeys) bad |= kErrBadIndptr;   // sound arrays stay below: the host has checked their sizes
  if (report && bad != 0 && a.err != nullptr) atomicOr(a.err, bad);
  if (work > 0x7fffffffLL - kXtKeys) return 0;
  const unsigned w = static_cast<unsigned>(work);
  return max(static_cast<int>((w + a.shares - 1) / a.shares), a.min_tiles);
}

// Lays out the share's runs from `w0` on, in order, as many as fit.  m: the first NT requests.  The first round also writes
// down the cut that the share starts with (cut: its place, null for other rounds).
template <int ROWS, int NT, int SEGS>
__device__ __forceinline__ void ex_layout(const ExArgs& a, int w0, unsigned per, const ExMine& m0, ExCut* cut,
                                          ExScratch<SEGS>& sc) {
  const int w_begin = sc.begin, w_end = sc.end;
  if (threadIdx.x == 0) sc.bad_v = 0;
  long long before = 0, segs = 0;
  bool wrote = false;
  for (int b0 = 0; b0 < a.batch && before < w_end && segs < SEGS; b0 += NT) {
    const ExMine m = a.batch <= NT ? m0 : ex_mine<ROWS, NT>(a, b0, before, sc);
    const int from = max(w0, m.at) - m.at, to = min(w_end - m.at, m.work);   // of the request's work
    int first = 0, n = 0;   // its row tiles in the share
    if (from < to) {
      const int all = ex_row_tiles<ROWS>(a, m.r);
      auto tile_at = [&](int w) {   // the row tile that holds w
        int lo = 0, hi = all;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (ex_before<ROWS>(a, m.r, mid) <= w) lo = mid; else hi = mid;
        }
        return lo;
      };
      first = tile_at(from);
      n = tile_at(to - 1) - first + 1;
    }
    long long all_segs;
    int i = static_cast<int>(min(segs + ex_scan<NT>(n, all_segs, sc, a.batch <= 32), static_cast<long long>(SEGS)));
    for (int tile = first; tile < first + n && i < SEGS; ++tile, ++i) {
      const int start = ex_before<ROWS>(a, m.r, tile), nt = ex_before<ROWS>(a, m.r, tile + 1) - start;
      const int k0 = max(from, start) - start, k1 = min(to, start + nt) - start;
      ExSeg s;
      s.qo0 = m.r.qo0;
      s.row0 = tile * ROWS;
      s.nrows = min(ROWS, (m.r.n << a.lg) - s.row0);
      s.pos0 = m.r.len - m.r.n;
      s.p0 = m.r.p0;
      s.nkeys = ex_visible<ROWS>(a, m.r, tile);
      s.tile0 = k0;
      s.ntiles = k1 - k0;
      s.part = k0 == 0 && k1 == nt ? -1 : m.at + start + k0 == w_begin ? 0 : 1;
      sc.seg[i] = s;
      if (i == SEGS - 1) sc.next = m.at + start + k1;
      if (cut != nullptr && i == 0 && k0 > 0) {
        const unsigned begin = m.at + start;
        ExCut c;
        c.qo0 = s.qo0; c.row0 = s.row0; c.nrows = s.nrows;
        c.first = begin / per;
        c.shares = (begin + nt - 1) / per - c.first;
        c.part = begin == c.first * per ? 0 : 1;
        c.pos0 = s.pos0;
        c.pad = 0;
        *cut = c;
        wrote = true;
      }
    }
    segs += all_segs;
  }
  if (cut != nullptr && !__syncthreads_or(wrote) && threadIdx.x == 0) cut->nrows = 0;
  __syncthreads();
  if (threadIdx.x == 0) {
    sc.count = static_cast<int>(min(segs, static_cast<long long>(SEGS)));
    if (segs < SEGS) sc.next = w_end;   // (otherwise whoever laid out the last run has stored it: one writer in either case)
  }
  __syncthreads();
}

template <int QT, bool DENSE = false>
struct Xt {
  static constexpr int kRows = 32 * QT;
  static constexpr int kKStages = 3, kVStages = QT == 4 ? 2 : 3;   // of the rings
  static constexpr int kSegs = QT == 1 ? 16 : 4;
  static constexpr int kRotWarps = DENSE ? 0 : 4;
  static constexpr int kHalves = DENSE ? 1 : 2;         // threads of a row
  static constexpr int kSoft = 32 * QT * kHalves;       // softmax threads
  static constexpr int kThreads = kSoft + 32 * (kRotWarps + 4);
  static constexpr int kQPanel = kRows * 128;           // Q: two 64-dim panels of [rows][128 B]
  static constexpr int kKOff = 2 * kQPanel;
  static constexpr int kVOff = kKOff + kKStages * kXtTileBytes;
  static constexpr int kBarOff = kVOff + kVStages * kXtTileBytes;
  static constexpr int kBars = 3 * kKStages + 2 * kVStages + 7;
  static constexpr int kTurnOff = (kBarOff + kBars * 8 + 8 + 15) / 16 * 16;
  static constexpr int kScratchOff = kTurnOff + 512;
  static constexpr int kSmem = kScratchOff + static_cast<int>(sizeof(ExScratch<kSegs>));
  static_assert(kXtCtasPerSm * (kSmem + 1024) <= 228 * 1024, "shared memory budget");
  static_assert(kQPanel + 128 * 128 <= kBarOff, "the products read 128 rows of each panel of Q");
};

// Eight keys of a tile, E the group's number: a lane copies 16 bytes of each second one, 512 bytes apart in the page, to the
// four places of the group in `dst` (the same in every group but for 1024 bytes)
template <int E>
__device__ __forceinline__ void copy_eight(const uint32_t (&dst)[4], uint32_t off, uint64_t src) {
  asm volatile("cp.async.cg.shared.global [%0 + %5], [%4], 16;\n"
               "cp.async.cg.shared.global [%1 + %5], [%4 + 512], 16;\n"
               "cp.async.cg.shared.global [%2 + %5], [%4 + 1024], 16;\n"
               "cp.async.cg.shared.global [%3 + %5], [%4 + 1536], 16;\n"
               ::"r"(dst[0] + off), "r"(dst[1] + off), "r"(dst[2] + off), "r"(dst[3] + off), "l"(src), "n"(E * 1024) : "memory");
}
// Replaces what is not finite in two 16-bit values by zero; true where something was.
template <typename T>
__device__ __forceinline__ bool drop_nonfinite(uint32_t& w) {
  constexpr uint32_t kExp = TcFormat<T>::value ? 0x7f80u : 0x7c00u;   // bf16, fp16
  const bool lo = (w & kExp) == kExp, hi = (w >> 16 & kExp) == kExp;
  if (lo) w &= 0xffff0000u;
  if (hi) w &= 0x0000ffffu;
  return lo || hi;
}
__device__ __forceinline__ void lds128(uint32_t at, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t at, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// The same for what a lane copied of the groups of eight keys e0 .. e1 - 1 of a tile of values: four pieces in each.
template <typename T>
__device__ __noinline__ bool drop_copied(uint32_t d0, uint32_t d1, uint32_t d2, uint32_t d3, int e0, int e1) {
  constexpr uint32_t kExp = TcFormat<T>::value ? 0x7f80u : 0x7c00u;
  const uint32_t at[4] = {d0, d1, d2, d3};
  bool found = false;
#pragma unroll 1
  for (int e = e0; e < e1; ++e) {
    uint32_t w[4][4], most = 0;   // the largest absolute value as integers, per half
#pragma unroll
    for (int i = 0; i < 4; ++i) lds128(at[i] + e * 1024, w[i]);
#pragma unroll
    for (int i = 0; i < 16; ++i) most = __vmaxu2(most, w[i >> 2][i & 3] & 0x7fff7fffu);
    if ((most & 0xffffu) < kExp && (most >> 16) < kExp) continue;
    found = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bool here = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) here |= drop_nonfinite<T>(w[i][k]);
      if (here) sts128(at[i] + e * 1024, w[i]);
    }
  }
  return found;
}
// The values that were taken out, for a thread's row, which sees the keys up to `pos`: added to its 64 dimensions of the result
// or, where that is null, of the state.  (Out of line, like the function above: nothing of the ordinary loops should make room
// for them.)
template <typename T>
__device__ __noinline__ void add_nonfinite(const ExArgs& a, const ExSeg& s, int kvh, int half, int pos, T* result, float* state) {
  const int P = a.page_size;
  const int from = max(s.tile0 * kXtKeys, (s.pos0 + (s.row0 >> a.lg) + 1) / 8 * 8);   // the first key that was looked at
  const int to = min(min(s.nkeys, (s.tile0 + s.ntiles) * kXtKeys), pos + 1);
  for (int key = from; key < to; ++key) {
    const T* page = static_cast<const T*>(a.kv_ptrs[s.p0 + key / P]);
    if (page == nullptr || (reinterpret_cast<uintptr_t>(page) & 15) != 0) continue;
    const uint32_t* v = reinterpret_cast<const uint32_t*>(
        page + (static_cast<size_t>((a.layer_idx * 2 + 1) * a.num_kv_heads + kvh) * P + key % P) * kPdDim + half * 64);
    for (int i = 0; i < 32; ++i) {
      const uint32_t w = v[i];
      uint32_t finite = w;
      if (!drop_nonfinite<T>(finite)) continue;
      const float2 x = unpack2<T>(w), y = unpack2<T>(finite);   // (a finite one: the same, nothing is added)
      if (result != nullptr) {
        result[2 * i] = static_cast<T>(static_cast<float>(result[2 * i]) + (x.x - y.x));
        result[2 * i + 1] = static_cast<T>(static_cast<float>(result[2 * i + 1]) + (x.y - y.y));
      } else {
        state[2 * i] += x.x - y.x;
        state[2 * i + 1] += x.y - y.y;
      }
    }
  }
}
// A run's queries, rotated and scaled by log2(e) / sqrt(d), as the A operand, K-major, where a thread has a row: a warp fetches its
// 32 rows and rotates them in place.  Short loops, out of line: code that a warp comes to once per run waits for its
// instructions (unrolled, with the rows in registers, this took 8000 cycles the first time and 1200 the second).  Eight prompts
// of 512 tokens: 110 us instead of 118, of 1024: 230 instead of 259.  Where two threads share a row, and registers are
// scarce, the same costs more in the loop over the keys than it gives: 229 us instead of 204 for 16 requests of 20 to 120 new
// tokens, 32 heads.
template <typename T>
__device__ __noinline__ void bring_queries(const ExArgs& a, const ExSeg& s, uint32_t qs, int panel, int kvh, int wq) {
  const int lg = a.lg, gmask = (1 << lg) - 1, row0 = s.row0 + wq * 32, nrows = s.nrows - wq * 32;
  const int lane = threadIdx.x & 31;
  qs += wq * 32 * 128;
  const T* q = static_cast<const T*>(a.q);
  const int Nq = a.num_kv_heads << lg;
#pragma unroll 1
  for (int i = lane; i < 32 * 16; i += 32) {
    const int r = i >> 4, at = row0 + r, c = i & 7;   // a row's chunks of 16 bytes; eight to a panel
    const T* src = q + (static_cast<size_t>(s.qo0 + (at >> lg)) * Nq + (kvh << lg) + (at & gmask)) * kPdDim + (i & 15) * 8;
    cp_async16(qs + r * 128 + ((c ^ (r & 7)) << 4) + (i & 8 ? panel : 0), r < nrows ? src : q, r < nrows);
  }
  cp_async_commit();
  cp_async_wait<0>();
  __syncwarp();
  // a thread turns eight dimensions and their partners of rows one after the other: the heads of a query share the sines
  const int c = lane & 7;
  float sn[8], cs[8];
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const int r = (lane >> 3) * 8 + i;
    if ((i & gmask) == 0) {
      const float scale = 1.4426950408889634f * rsqrtf(static_cast<float>(kPdDim));
      const float pos = static_cast<float>(s.pos0 + ((row0 + r) >> lg));
      const float *hi = rot_at(a.rot.hi) + c * 8, *lo = rot_at(a.rot.lo) + c * 8;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        rot_sincos(pos, hi[k], lo[k], &sn[k], &cs[k]);
        sn[k] *= scale;
        cs[k] *= scale;
      }
    }
    const uint32_t at = qs + r * 128 + ((c ^ (r & 7)) << 4);
    uint32_t own[4], par[4];
    lds128(at, own);
    lds128(at + panel, par);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = unpack2<T>(own[k]), y = unpack2<T>(par[k]);
      own[k] = pack2<T>(x.x * cs[2 * k] - y.x * sn[2 * k], x.y * cs[2 * k + 1] - y.y * sn[2 * k + 1]);
      par[k] = pack2<T>(y.x * cs[2 * k] + x.x * sn[2 * k], y.y * cs[2 * k + 1] + x.y * sn[2 * k + 1]);
    }
    sts128(at, own);
    sts128(at + panel, par);
  }
}
// an entry of the page table, zero where there is none to read; without a branch, so that nothing waits for it here
__device__ __forceinline__ uint64_t load_if(const void* const* at, bool yes) {
  uint64_t v;
  asm volatile("{\n.reg .pred p;\nsetp.ne.s32 p, %2, 0;\nmov.b64 %0, 0;\n@p ld.global.nc.b64 %0, [%1];\n}\n"
               : "=l"(v) : "l"(at), "r"(static_cast<int>(yes)));
  return v;
}

// grid: shares * Nkv
template <typename T, int QT, bool DENSE>
__global__ void __launch_bounds__(Xt<QT, DENSE>::kThreads, kXtCtasPerSm) paged_extend_kernel(const __grid_constant__ ExArgs a) {
  using X = Xt<QT, DENSE>;
  constexpr int H = X::kHalves;
  constexpr int ROWS = X::kRows, NK = X::kKStages, NV = X::kVStages, ROTATORS = 32 * X::kRotWarps;
  extern __shared__ __align__(1024) unsigned char xt_smem[];
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t sbase = smem_u32(xt_smem);
  // (cos, cos, sin, sin) of the turn from one of a loader's keys to the next, two frequencies each
  float* turn = reinterpret_cast<float*>(xt_smem + X::kTurnOff);
  ExScratch<X::kSegs>& sc = *reinterpret_cast<ExScratch<X::kSegs>*>(xt_smem + X::kScratchOff);
  if (!DENSE && tid < 64) {
    float sn, cs;
    rot_sincos(static_cast<float>(ROTATORS / 8), a.rot.hi[tid], a.rot.lo[tid], &sn, &cs);
    turn[(tid >> 1) * 4 + (tid & 1)] = cs;
    turn[(tid >> 1) * 4 + (tid & 1) + 2] = sn;
  }

  pdl_wait();
  pdl_trigger();
  if ((sbase & 1023u) != 0) {   // the swizzled layouts need the 1024-byte alignment asked for above
    if (tid == 0 && a.err != nullptr) atomicOr(a.err, kErrBadPointer);
    return;
  }
  const int kvh = blockIdx.x % a.num_kv_heads, share = blockIdx.x / a.num_kv_heads;
  const uint32_t qs = sbase, ks0 = sbase + X::kKOff, vs0 = sbase + X::kVOff, bars = sbase + X::kBarOff;
  const uint32_t k_raw = bars, k_full = k_raw + NK * 8, k_empty = k_full + NK * 8, v_full = k_empty + NK * 8, v_empty = v_full + NV * 8;
  // two each, used by alternate tiles: a softmax warp may be a tile ahead of another, and looks at the completion of a tile
  // after it has handed on the next
  const uint32_t s_full = v_empty + NV * 8, p_full = s_full + 16, o_done = s_full + 32;
  const uint32_t q_full = s_full + 48, tmem_slot = s_full + 56;
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(xt_smem + (tmem_slot - sbase));
  // roles: softmax warps w < 8 with w mod 4 < QT; of the others, in the order of their numbers, the rotators, a loader of K,
  // one of V, the issuers of S and of O
  const bool softmax = warp < 4 * H && (warp & 3) < QT;
  const int other = warp - (warp < 4 ? min(warp, QT) : H == 2 && warp < 8 ? QT + min(warp - 4, QT) : H * QT);
  const int role = softmax ? -1 : max(0, other - X::kRotWarps + 1);   // 0 rotator, 1 K, 2 V, 3 S, 4 O

  if (tid == 0) {
    for (int i = 0; i < NK; ++i) {
      mbar_init(k_raw + i * 8, 32);
      mbar_init(k_full + i * 8, DENSE ? 32 : ROTATORS);
      mbar_init(k_empty + i * 8, 1);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(v_full + i * 8, 32);
      mbar_init(v_empty + i * 8, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i * 8, 1);
      mbar_init(p_full + i * 8, X::kSoft);
      mbar_init(o_done + i * 8, 1);   // also: the S buffer, where P lives, is free
    }
    mbar_init(q_full, X::kSoft);
    fence_mbar_init();
  }
  if (role == 3) {
    tc_alloc(tmem_slot, kXtTmemCols);
    tc_relinquish();
  }
  tc_fence_before();   // (the search for the share has barriers enough, and hides what this takes)
  ExMine mine;
  const int per = ex_share<ROWS, X::kThreads>(a, blockIdx.x == 0, mine, sc);
  if (tid == 0) {
    const long long begin = static_cast<long long>(share) * per;
    sc.begin = static_cast<int>(min(begin, 0x7fffffffLL));
    sc.end = static_cast<int>(min(begin + per, 0x7fffffffLL));
  }
  __syncthreads();
  const int gmask = (1 << a.lg) - 1;
  const int Nq = a.num_kv_heads << a.lg, P = a.page_size;

  ex_layout<ROWS, X::kThreads>(a, sc.begin, per, mine, a.cuts == nullptr ? nullptr : a.cuts + blockIdx.x, sc);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot_ptr;
  if (sc.count == 0) {   // nothing left for this share (uniform over the CTA)
    if (role == 3) tc_dealloc(tmem, kXtTmemCols);
    return;
  }
  bool dead = false;
  int g = 0, gs = 0;   // tiles and row tiles so far, of the warp's role

  for (;;) {
    const int count = sc.count;
    if (!DENSE && role == 0) {
      // ---------------- rotators: thread = (chunk c of 8 dims and its partner, every STEP-th key) ----------------
      constexpr int STEP = 32 * Xt<QT>::kRotWarps / 8, KPT = kXtKeys / STEP;   // KPT: keys of a thread per tile
      const int rt = other * 32 + lane, c = rt & 7, kr = rt >> 3;
      const ulonglong2* my_turn = reinterpret_cast<const ulonglong2*>(turn) + c * 4;
      uint64_t cc[4] = {}, ss[4] = {};   // cosines and sines of key kr + STEP i, two frequencies each
      for (int seg = 0; seg < count; ++seg) {
        const int tile0 = sc.seg[seg].tile0, ntiles = sc.seg[seg].ntiles;
        for (int j = 0; j < ntiles; ++j, ++g) {
          if (j % kXtReseed == 0) {
            const float pos = static_cast<float>((tile0 + j) * kXtKeys + kr);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float s0, sx, c0, cx;
              rot_sincos(pos, a.rot.hi[c * 8 + 2 * k], a.rot.lo[c * 8 + 2 * k], &s0, &c0);
              rot_sincos(pos, a.rot.hi[c * 8 + 2 * k + 1], a.rot.lo[c * 8 + 2 * k + 1], &sx, &cx);
              cc[k] = pack_f32x2(c0, cx);
              ss[k] = pack_f32x2(s0, sx);
            }
          }
          const int st = g % NK;
          pf_wait_role(k_raw + st * 8, (g / NK) & 1, a.err, dead);
          // row kr of a panel; rows STEP further on are swizzled alike
          uint32_t at = ks0 + st * kXtTileBytes + kr * 128 + ((c ^ (kr & 7)) << 4);
#pragma unroll 1
          for (int i0 = 0; i0 < KPT; i0 += 2, at += 2 * STEP * 128) {   // two keys at a time: both are read before either is written
            uint32_t own[2][4], par[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              lds128(at + i * (STEP * 128), own[i]);
              lds128(at + i * (STEP * 128) + kXtPanel, par[i]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const ulonglong2 t1 = my_turn[k];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float2 x = unpack2<T>(own[i][k]), y = unpack2<T>(par[i][k]);
                const uint64_t ko = pack_f32x2(x.x, x.y), kq = pack_f32x2(y.x, y.y);
                const uint64_t ns = ss[k] ^ 0x8000000080000000ull;
                float a0, a1, b0, b1;
                unpack_f32x2(fma_f32x2(ko, cc[k], mul_f32x2(kq, ns)), a0, a1);      // own c - partner s
                unpack_f32x2(fma_f32x2(kq, cc[k], mul_f32x2(ko, ss[k])), b0, b1);   // partner c + own s
                own[i][k] = pack2<T>(a0, a1);
                par[i][k] = pack2<T>(b0, b1);
                // the next of the thread's keys; after the last of them the tile's 64 keys are passed
                const uint64_t n = fma_f32x2(cc[k], t1.x, mul_f32x2(ns, t1.y));
                ss[k] = fma_f32x2(ss[k], t1.x, mul_f32x2(cc[k], t1.y));
                cc[k] = n;
              }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              sts128(at + i * (STEP * 128), own[i]);
              sts128(at + i * (STEP * 128) + kXtPanel, par[i]);
            }
          }
          fence_proxy_async();   // the products read through the async proxy
          mbar_arrive(k_full + st * 8);
        }
      }
    } else if (role == 1 || role == 2) {
      // ---------------- loaders: a warp copies a tile, a lane chunk lane & 15 of the keys 2 i + (lane >> 4) ----------------
      const uint32_t ring = role == 1 ? ks0 : vs0, full = role == 2 ? v_full : DENSE ? k_full : k_raw, empty = role == 1 ? k_empty : v_empty;
      const int lp = 31 - __clz(P);   // the page size is a power of two (checked by the host)
      const uint32_t head_off =
          static_cast<uint32_t>(((a.layer_idx * 2 + role - 1) * a.num_kv_heads + kvh) * P) * 256u;   // bytes
      const uint32_t lane_off = (lane >> 4) * 256 + (lane & 15) * 16;
      uint32_t dst[4];   // of the keys 2 i + (lane >> 4) of a group of eight: panel, row, swizzled chunk
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 2 * i + (lane >> 4);
        dst[i] = ring + ((lane & 8) ? kXtPanel : 0) + row * 128 + (((lane & 7) ^ row) << 4);
      }
      const int stages = role == 1 ? NK : NV;
      int st = g % stages;                       // stage of the next tile
      uint32_t phase = (g / stages - 1) & 1;     // of its last use
      bool bad_ptr = false;
      // eight keys lie in one page: lane e looks after the keys 8 e .. 8 e + 7 of the tile, a tile ahead of the copies
      const int e8 = (lane & 7) * 8;
      const bool rows = DENSE && role == 1;   // rotated keys lie one after the other, the pages' places for them in order
      auto entry = [&](const ExSeg& s, int tile) -> uint64_t {
        const int key = tile * kXtKeys + e8;
        if (rows)
          return key < s.nkeys ? reinterpret_cast<uint64_t>(a.dense) +
                                     ((static_cast<uint64_t>(kvh) * a.total_pages + s.p0) * P + key) * 256u : 0;
        return load_if(a.kv_ptrs + s.p0 + (key >> lp), key < s.nkeys);
      };
      uint64_t page = entry(sc.seg[0], sc.seg[0].tile0);
      for (int seg = 0; seg < count && !dead; ++seg) {
        const int tile0 = sc.seg[seg].tile0, ntiles = sc.seg[seg].ntiles, nkeys = sc.seg[seg].nkeys;
        const int next = seg + 1;
        const int seen = role == 1 ? nkeys : sc.seg[seg].pos0 + (sc.seg[seg].row0 >> a.lg) + 1;   // keys that all rows see
        for (int j = 0; j < ntiles; ++j, ++g) {
          const int key0 = (tile0 + j) * kXtKeys;
          const bool ok = page != 0 && (page & 15) == 0;
          bad_ptr |= key0 + e8 < nkeys && !ok;
          const uint64_t base = rows ? page : page + head_off + ((key0 + e8) & (P - 1)) * 256u;
          const bool whole = __all_sync(0xffffffffu, ok) && key0 + kXtKeys <= nkeys;
          const uint64_t mine = ok ? base : 0;
          page = j + 1 < ntiles ? entry(sc.seg[seg], tile0 + j + 1) : next < count ? entry(sc.seg[next], sc.seg[next].tile0) : 0;
          if (g >= stages) pf_wait_role(empty + st * 8, phase, a.err, dead);
          if (dead) break;
          const uint32_t off = st * kXtTileBytes;
          if (whole) {
            auto src = [&](int e) { return __shfl_sync(0xffffffffu, mine, e) + lane_off; };
            copy_eight<0>(dst, off, src(0));
            copy_eight<1>(dst, off, src(1));
            copy_eight<2>(dst, off, src(2));
            copy_eight<3>(dst, off, src(3));
            copy_eight<4>(dst, off, src(4));
            copy_eight<5>(dst, off, src(5));
            copy_eight<6>(dst, off, src(6));
            copy_eight<7>(dst, off, src(7));
          } else {
#pragma unroll 1
            for (int e = 0; e < 8; ++e) {   // keys that do not exist read as zeros
              const uint64_t src = __shfl_sync(0xffffffffu, mine, e) + lane_off;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const bool have = src != lane_off && key0 + 8 * e + 2 * i + (lane >> 4) < nkeys;
                cp_async16(dst[i] + off + e * 1024, have ? reinterpret_cast<const void*>(src + i * 512) : a.q, have);
              }
            }
          }
          if (key0 + kXtKeys <= seen || role == 1) {
            cp_async_arrive(full + st * 8);   // when this lane's copies have landed
          } else {
            // The rows that do not see all of the tile weigh the rest with zeros, but zero times a value that is not finite is
            // none: such values are taken out, and added at the end to the rows that see them.  (With tiles of 128 rows, whose
            // ring has two stages, this is on the products' way: 204 us instead of 194 at 16 requests of 20 to 120 new tokens,
            // 32 heads.  A warp that takes the values out just before their product costs 211, the loader's lanes with the code
            // in line 204, but then 93 us instead of 84 at drafts.  Tiles that every row sees whole pay nothing.)
            cp_async_commit();
            cp_async_wait<0>();
            if (drop_copied<T>(dst[0] + off, dst[1] + off, dst[2] + off, dst[3] + off, max(seen - key0, 0) / 8,
                               (min(nkeys - key0, kXtKeys) + 7) / 8))
              atomicOr(&sc.bad_v, 1u << seg);
            mbar_arrive(full + st * 8);
          }
          if (++st == stages) {
            st = 0;
            phase ^= 1;
          }
        }
      }
      cp_async_wait<0>();
      if (__any_sync(0xffffffffu, bad_ptr) && lane == 0 && a.err != nullptr) atomicOr(a.err, kErrBadPointer);
    } else if (role == 3) {
      // ---------------- issuer of S = Q . K^T: runs up to two tiles ahead of the softmax ----------------
      if (lane == 0) {
        const uint32_t idesc_s = tc_idesc<T>(kXtKeys, false);
        const uint64_t qdesc = desc_kmajor(qs), kdesc = desc_kmajor(ks0);   // (addresses are added below: no field overflows)
        for (int seg = 0; seg < count; ++seg) {
          const int ntiles = sc.seg[seg].ntiles;
          pf_wait_role(q_full, gs & 1, a.err, dead);
          for (int j = 0; j < ntiles; ++j, ++g) {
            const int st = g % NK, sb = g & 1;
            pf_wait_role(k_full + st * 8, (g / NK) & 1, a.err, dead);
            if (DENSE) fence_proxy_async();   // K came by the loader's ordinary copies
            if (g >= 2) pf_wait_role(o_done + sb * 8, ((g >> 1) - 1) & 1, a.err, dead);   // P . V has read this S buffer
            tc_fence_after();
            if (!dead) {
              const uint64_t kd = kdesc + st * (kXtTileBytes >> 4);
#pragma unroll
              for (int kk = 0; kk < 8; ++kk)
                tc_mma(tmem + sb * kXtKeys, qdesc + (((kk >> 2) * X::kQPanel + (kk & 3) * 32) >> 4),
                       kd + (((kk >> 2) * kXtPanel + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
            }
            tc_commit(s_full + sb * 8);
            tc_commit(k_empty + st * 8);
          }
          ++gs;
        }
      }
    } else if (role == 4) {
      // ---------------- issuer of O += P . V ----------------
      if (lane == 0) {
        const uint32_t idesc_o = tc_idesc<T>(kPdDim, true);
        const uint64_t vdesc = desc_mnmajor(vs0, kXtPanel);
        for (int seg = 0; seg < count; ++seg) {
          const int ntiles = sc.seg[seg].ntiles;
          for (int j = 0; j < ntiles; ++j, ++g) {
            const int st = g % NV, sb = g & 1;
            pf_wait_role(v_full + st * 8, (g / NV) & 1, a.err, dead);
            fence_proxy_async();   // V came by the loader's ordinary copies
            pf_wait_role(p_full + sb * 8, (g >> 1) & 1, a.err, dead);
            tc_fence_after();
            if (!dead) {
              const uint64_t vd = vdesc + st * (kXtTileBytes >> 4);
              const uint32_t pa = tmem + sb * kXtKeys + kXtHalf / 2;
#pragma unroll
              for (int kk = 0; kk < kXtKeys / 16; ++kk)   // keys 16 kk .. 16 kk + 15: eight columns in the upper half of the
                                                          // columns of the thread that made them
                tc_mma_ts(tmem + kXtOCol, pa + (kk >> 1) * kXtHalf + (kk & 1) * 8, vd + kk * (2048 >> 4), idesc_o,
                          (j > 0 || kk > 0) ? 1u : 0u);
            }
            tc_commit(o_done + sb * 8);
            tc_commit(v_empty + st * 8);
          }
        }
      }
    } else {
      // ---------------- softmax warps: thread = (row, half of the columns), or a row ----------------
      // H = 2: warps w and w + 4 (w < QT) hold the same 32 rows, the first takes columns 0-31 of a tile of S and 0-63 of O, the
      // second the rest, and the two threads of a row agree on its maximum through tensor memory, as in the prefill kernel.
      // H = 1: a thread has the row, and nothing is exchanged: with four warps in place of eight, and 128 registers a thread where
      // nobody rotates, 230 us instead of 245 for 4 requests of 400 to 512 new tokens on 4 k to 12 k keys.  Beside rotators, with 80
      // registers, 249 instead of 208 for 16 requests of 20 to 120 new tokens.
      const int half = H == 2 ? warp >> 2 : 0;
      const int wq = warp & 3;
      const int row = wq * 32 + lane;
      const uint32_t my_tmem = tmem + (static_cast<uint32_t>(wq * 32) << 16);
      const uint32_t o_tmem = my_tmem + kXtOCol + half * 64;
      for (int seg = 0; seg < count; ++seg) {
        const ExSeg s = sc.seg[seg];
        const int rr = s.row0 + row;
        // rows past the end behave like the last one
        const int my_pos = s.pos0 + (min(rr, s.row0 + s.nrows - 1) >> a.lg);
        // ---- the rotated, pre-scaled queries: A operand, K-major.  16 threads per row ----
        if (H == 1) {
          bring_queries<T>(a, sc.seg[seg], qs, X::kQPanel, kvh, wq);
        } else {
          const int qt = (half * QT + wq) * 32 + lane;
          const int d0 = (qt & 15) * 4;
          const float qscale = 1.4426950408889634f * rsqrtf(static_cast<float>(kPdDim));   // log2(e) / sqrt(d)
          constexpr int PASS = 4 * QT;   // rows per pass
          uint2 uo[8], up[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = (qt >> 4) + PASS * i;
            uo[i] = up[i] = make_uint2(0u, 0u);
            if (r < s.nrows) {
              const T* qp = static_cast<const T*>(a.q) +
                            (static_cast<size_t>(s.qo0 + ((s.row0 + r) >> a.lg)) * Nq + (kvh << a.lg) + ((s.row0 + r) & gmask)) *
                                kPdDim + d0;
              uo[i] = __ldg(reinterpret_cast<const uint2*>(qp));
              up[i] = __ldg(reinterpret_cast<const uint2*>(qp + 64));
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = (qt >> 4) + PASS * i;
            const float pos = static_cast<float>(s.pos0 + ((s.row0 + r) >> a.lg));
            const float2 o0 = unpack2<T>(uo[i].x), o1 = unpack2<T>(uo[i].y), q0 = unpack2<T>(up[i].x), q1 = unpack2<T>(up[i].y);
            const float own[4] = {o0.x, o0.y, o1.x, o1.y}, par[4] = {q0.x, q0.y, q1.x, q1.y};
            float ro[4], rp[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float sn, cs;
              rot_sincos(pos, a.rot.hi[d0 + k], a.rot.lo[d0 + k], &sn, &cs);
              ro[k] = (own[k] * cs - par[k] * sn) * qscale;
              rp[k] = (par[k] * cs + own[k] * sn) * qscale;
            }
            const uint32_t addr = qs + r * 128 + (((d0 >> 3) ^ (r & 7)) << 4) + (d0 & 7) * 2;
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(addr), "r"(pack2<T>(ro[0], ro[1])), "r"(pack2<T>(ro[2], ro[3]))
                         : "memory");
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(addr + X::kQPanel), "r"(pack2<T>(rp[0], rp[1])),
                         "r"(pack2<T>(rp[2], rp[3])) : "memory");
          }
        }
        fence_proxy_async();   // the products read Q through the async proxy
        mbar_arrive(q_full);
        if (wq * 32 >= s.nrows) {   // no row of the tile: hands on what the others make
          for (int j = 0; j < s.ntiles; ++j, ++g) {
            pf_wait_role(s_full + (g & 1) * 8, (g >> 1) & 1, a.err, dead);
            mbar_arrive(p_full + (g & 1) * 8);
          }
          continue;
        }

        float m_ref = -INFINITY;
        uint64_t l2 = pack_f32x2(0.f, 0.f);   // this thread's share of the row sum, two lanes
        for (int j = 0; j < s.ntiles; ++j, ++g) {
          const int sb = g & 1;
          pf_wait_role(s_full + sb * 8, (g >> 1) & 1, a.err, dead);
          tc_fence_after();
          const uint32_t my_s = my_tmem + sb * kXtKeys + half * kXtHalf;
          const int lim = my_pos - (s.tile0 + j) * kXtKeys - half * kXtHalf;   // columns above lim are later keys
          uint32_t sv[3 - H][32];
#pragma unroll
          for (int h = 0; h < 3 - H; ++h) tc_ld32(my_s + h * kXtHalf, sv[h]);
          tc_wait_ld();
          if (lim < 64 / H - 1) {
#pragma unroll
            for (int i = 0; i < 64 / H; ++i)
              if (i > lim) sv[i >> 5][i & 31] = __float_as_uint(-INFINITY);
          }
          auto max_half = [](const uint32_t (&v)[32]) {
            float ma = max3(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]));
            float mb = max3(__uint_as_float(v[3]), __uint_as_float(v[4]), __uint_as_float(v[5]));
#pragma unroll
            for (int i = 6; i < 30; i += 4) {
              ma = max3(ma, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
              mb = max3(mb, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
            }
            return fmaxf(max3(ma, __uint_as_float(v[30]), __uint_as_float(v[31])), mb);
          };
          float mx = max_half(sv[0]);
          if (H == 1) {
            mx = fmaxf(mx, max_half(sv[2 - H]));
          } else {
            // exchange with the other half's thread: own maximum into the first column of the own half
            tc_st1(my_s, __float_as_uint(mx));
            tc_wait_st();
            tc_fence_before();
            pair_barrier(wq);
            tc_fence_after();
            mx = fmaxf(mx, __uint_as_float(tc_ld1(my_tmem + sb * kXtKeys + (half ^ 1) * kXtHalf)));
          }
          float rescale = 1.0f;
          bool raise = false;
          if (mx > m_ref + kPfRaise || m_ref == -INFINITY) {   // (-inf + 8 = -inf: the first visible key always raises)
            if (mx != -INFINITY) {
              raise = m_ref != -INFINITY;
              rescale = exp2f(m_ref - mx);   // 0 when nothing was accumulated yet
              m_ref = mx;
            }
          }
          const float nm = m_ref == -INFINITY ? 0.f : -m_ref;
          const uint64_t nm2 = pack_f32x2(nm, nm);
          uint64_t sum2 = pack_f32x2(0.f, 0.f);
          // P overwrites the upper half of the S columns that it was made of (the lower half keeps the exchanged maximum); the
          // other thread of the row has read its own columns before the exchange
          auto weights = [&](const uint32_t (&v)[32], int h) {
            uint32_t pw[kXtHalf / 2];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float x0, x1;
              unpack_f32x2(add_f32x2(pack_f32x2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), nm2), x0, x1);
              const float e0 = exp2f(x0), e1 = exp2f(x1);
              sum2 = add_f32x2(sum2, pack_f32x2(e0, e1));
              pw[i >> 1] = pack2<T>(e0, e1);
            }
            tc_st16(my_s + h * kXtHalf + kXtHalf / 2, pw);
          };
          weights(sv[0], 0);
          if (H == 1) weights(sv[2 - H], 1);
          l2 = add_f32x2(mul_f32x2(l2, pack_f32x2(rescale, rescale)), sum2);
          bool waited = j == 0;
          auto wait_prev = [&]() {   // P . V of the previous tile has completed: O is stable
            if (!waited) {
              pf_wait_role(o_done + (sb ^ 1) * 8, ((g - 1) >> 1) & 1, a.err, dead);
              tc_fence_after();
              waited = true;
            }
          };
          if (j > 0 && __any_sync(0xffffffffu, raise)) {
            wait_prev();
#pragma unroll 1
            for (int q = 0; q < 4 / H; ++q) {
              uint32_t ov[32];
              tc_ld32(o_tmem + q * 32, ov);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * rescale);
              tc_st32(o_tmem + q * 32, ov);
            }
            tc_wait_st();
          }
          tc_wait_st();
          tc_fence_before();
          mbar_arrive(p_full + sb * 8);
          wait_prev();   // every phase of the barrier is consumed, so that its parity stays readable
        }

        // ---- the result O / l, or the state; the two halves' sums meet through tensor memory as the maxima did ----
        pf_wait_role(o_done + ((g - 1) & 1) * 8, ((g - 1) >> 1) & 1, a.err, dead);
        tc_fence_after();
        float la, lb;
        unpack_f32x2(l2, la, lb);
        const float l_mine = la + lb;
        float l_run = l_mine;
        if (H == 2) {
          tc_st1(my_tmem + half * kXtHalf, __float_as_uint(l_mine));   // S buffer 0: the next product waits for this warp's queries
          tc_wait_st();
          tc_fence_before();
          pair_barrier(wq);
          tc_fence_after();
          l_run = l_mine + __uint_as_float(tc_ld1(my_tmem + (half ^ 1) * kXtHalf));
        }
        const float inv = row_scale(l_run, my_pos);
        T* orow = static_cast<T*>(a.o) + (static_cast<size_t>(s.qo0 + (rr >> a.lg)) * Nq + (kvh << a.lg) + (rr & gmask)) * kPdDim;
        float* rec = a.partial + (((static_cast<size_t>(share) * 2 + max(s.part, 0)) * a.num_kv_heads + kvh) * ROWS + row) * kPdRec;
        const bool write = row < s.nrows && !dead;
        if (write && s.part >= 0 && half == 0) {
          rec[0] = m_ref;
          rec[1] = l_run;
        }
#pragma unroll 1
        for (int q = 0; q < 4 / H; ++q) {
          uint32_t ov[32];
          tc_ld32(o_tmem + q * 32, ov);
          tc_wait_ld();
          if (!write) continue;
          if (s.part >= 0) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(rec + 4 + half * 64 + q * 32 + i) = make_uint4(ov[i], ov[i + 1], ov[i + 2], ov[i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              float f[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(ov[i + k]) * inv;
              *reinterpret_cast<uint4*>(orow + half * 64 + q * 32 + i) =
                  make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
            }
          }
        }
        if (write && (sc.bad_v >> seg & 1)) {
          for (int h = half; h < half + 3 - H; ++h)
            add_nonfinite<T>(a, sc.seg[seg], kvh, h, my_pos, s.part >= 0 ? nullptr : orow + h * 64, rec + 4 + h * 64);
        }
        tc_fence_before();   // the next row tile's products overwrite O after this warp has handed on a P
      }
    }
    if (sc.next >= sc.end) break;
    const int w0 = sc.next;
    __syncthreads();   // everyone is done with these runs
    long long before = 0;
    if (a.batch <= X::kThreads) mine = ex_mine<ROWS, X::kThreads>(a, 0, before, sc);
    ex_layout<ROWS, X::kThreads>(a, w0, 1u, mine, nullptr, sc);
    if (sc.count == 0) break;
  }

  // everyone is done with tensor memory: hand it back
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (role == 3) tc_dealloc(tmem, kXtTmemCols);
}

// The keys of all pages rotated, for chunks of several row tiles, which would each rotate them again: one CTA per page, a
// thread (entry, chunk of 8 dims and its partner), whose sines serve all kv heads.
template <typename T>
__global__ void __launch_bounds__(128) extend_rotate_kernel(const __grid_constant__ ExArgs a) {
  __shared__ __align__(16) float freq[128];
  load_rot_table(a.rot, freq);
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int pg = blockIdx.x, P = a.page_size;
  int lo = 0, hi = a.batch;   // the request of the page: the last one that starts at or before it
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.kv_indptr[mid] <= pg) lo = mid; else hi = mid;
  }
  const ExRequest r = ex_request(a, lo);
  const int first = (pg - r.p0) * P;   // position of the page's first entry
  if (r.n == 0 || first < 0 || first >= r.len) return;
  const T* page = static_cast<const T*>(a.kv_ptrs[pg]);
  if (page == nullptr || (reinterpret_cast<uintptr_t>(page) & 15) != 0) page = nullptr;   // (reported by the loader of V)
  T* out = static_cast<T*>(a.dense) + static_cast<size_t>(pg) * P * kPdDim;
  const size_t head_step = static_cast<size_t>(a.total_pages) * P * kPdDim;
  for (int i = threadIdx.x; i < P * 8; i += 128) {
    const int e = i >> 3, c = i & 7;
    if (first + e >= r.len) break;
    float cs[8], sn[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      rot_sincos(static_cast<float>(first + e), freq[c * 8 + k], freq[64 + c * 8 + k], &sn[k], &cs[k]);
    const T* src = page + (static_cast<size_t>(a.layer_idx) * 2 * a.num_kv_heads * P + e) * kPdDim + c * 8;
    T* dst = out + static_cast<size_t>(e) * kPdDim + c * 8;
    for (int h = 0; h < a.num_kv_heads; ++h, src += P * kPdDim, dst += head_step) {
      float x[8], y[8], u[8], v[8];
      uint4 xo = make_uint4(0u, 0u, 0u, 0u), yo = xo;
      if (page != nullptr) {
        xo = __ldcs(reinterpret_cast<const uint4*>(src));
        yo = __ldcs(reinterpret_cast<const uint4*>(src + 64));
      }
      unpack8<T>(xo, x);
      unpack8<T>(yo, y);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        u[k] = x[k] * cs[k] - y[k] * sn[k];
        v[k] = y[k] * cs[k] + x[k] * sn[k];
      }
      *reinterpret_cast<uint4*>(dst) = pack8<T>(u);
      *reinterpret_cast<uint4*>(dst + 64) = pack8<T>(v);
    }
  }
}

// adds one softmax state to another; an empty one (no weight) carries no information
__device__ __forceinline__ void add_state(float m1, float l1, const float4& o1, float& m, float& l, float4& acc) {
  if (l1 == 0.f) return;
  const float mn = fmaxf(m, m1), w0 = l == 0.f ? 0.f : exp2f(m - mn), w1 = exp2f(m1 - mn);
  m = mn;
  l = l * w0 + l1 * w1;
  acc.x = acc.x * w0 + o1.x * w1;
  acc.y = acc.y * w0 + o1.y * w1;
  acc.z = acc.z * w0 + o1.z * w1;
  acc.w = acc.w * w0 + o1.w * w1;
}

constexpr int kXtMergeThreads = 256;
constexpr int kXtMergeSplit = 2;   // (four to eight times as many CTAs of fewer rows measured the same or slower)

// Merges the states of the row tiles that are cut, in the order of the keys.  grid: ((shares - 1) * Nkv, kXtMergeSplit); a
// CTA stands for the cut at the start of a share and serves some of the rows of the tile that it goes through, a warp a row
// at a time, a lane four dimensions.
template <typename T, int QT>
__global__ void __launch_bounds__(kXtMergeThreads) paged_extend_merge_kernel(const __grid_constant__ ExArgs a) {
  constexpr int ROWS = Xt<QT>::kRows, WARPS = kXtMergeThreads / 32;
  pdl_wait();
  pdl_trigger();
  const int kvh = blockIdx.x % a.num_kv_heads, share = blockIdx.x / a.num_kv_heads + 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int4* rec = reinterpret_cast<const int4*>(a.cuts + blockIdx.x + a.num_kv_heads);
  const int4 c0 = __ldcg(rec), c1 = __ldcg(rec + 1);
  const int qo0 = c0.x, row0 = c0.y, nrows = c0.z, first = c0.w, shares = c1.x, part = c1.y, pos0 = c1.z;
  const int gmask = (1 << a.lg) - 1, Nq = a.num_kv_heads << a.lg;
  const size_t share_step = static_cast<size_t>(2) * a.num_kv_heads * ROWS * kPdRec;
  if (nrows == 0) return;
  const int count = shares + 1;
  // the states z0 .. z1 - 1 of a row, in order, added to (m, l, acc)
  auto add_states = [&](int row, int z0, int z1, float& m, float& l, float4& acc) {
    const float* base = a.partial + ((static_cast<size_t>(first) * 2 * a.num_kv_heads + kvh) * ROWS + row) * kPdRec;
    constexpr int U = 4;
    for (; z0 < z1; z0 += U) {   // four states are requested together
      float2 ml[U];
      float4 o[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ml[u] = make_float2(0.f, 0.f);
        o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (z0 + u < z1) {
          const float* r = base + (z0 + u) * share_step +
                           (z0 + u == 0 && part ? static_cast<size_t>(a.num_kv_heads) * ROWS * kPdRec : 0);
          ml[u] = __ldcg(reinterpret_cast<const float2*>(r));
          o[u] = __ldcg(reinterpret_cast<const float4*>(r + 4) + lane);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) add_state(ml[u].x, ml[u].y, o[u], m, l, acc);
    }
  };
  auto write_row = [&](int row, float l, const float4& acc) {
    const int rr = row0 + row;
    const float inv = row_scale(l, pos0 + (rr >> a.lg));
    T* op = static_cast<T*>(a.o) + (static_cast<size_t>(qo0 + (rr >> a.lg)) * Nq + (kvh << a.lg) + (rr & gmask)) * kPdDim;
    reinterpret_cast<uint2*>(op)[lane] = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
  };
  if (count <= 2 * WARPS) {   // a warp per row
    for (int i = blockIdx.y * WARPS + warp; ; i += kXtMergeSplit * WARPS) {
      const int row = i * shares + share - first - 1;
      if (row >= nrows) return;
      float m = -INFINITY, l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      add_states(row, 0, count, m, l, acc);
      write_row(row, l, acc);
    }
  }
  // few rows of many states (a long cache): the CTA's warps take a run of a row's states each
  __shared__ float4 s_acc[WARPS][32];
  __shared__ float2 s_ml[WARPS];
  const int run = (count + WARPS - 1) / WARPS;
  for (int i = blockIdx.y; ; i += kXtMergeSplit) {
    const int row = i * shares + share - first - 1;   // the same in every warp
    if (row >= nrows) return;
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    add_states(row, warp * run, min(count, (warp + 1) * run), m, l, acc);
    s_acc[warp][lane] = acc;
    if (lane == 0) s_ml[warp] = make_float2(m, l);
    __syncthreads();
    if (warp == 0) {
      m = -INFINITY;
      l = 0.f;
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int v = 0; v < WARPS; ++v) add_state(s_ml[v].x, s_ml[v].y, s_acc[v][lane], m, l, acc);
      write_row(row, l, acc);
    }
    __syncthreads();
  }
}

}  // namespace smlm
