// Paged key/value cache in 4 bits: geometry of a page, the batch of a call, and the division of an attention's work.
//
// A page holds P tokens (P = 16, 32 ... 256).  Its block for one key/value head is P * (d + 8) bytes:
//     key codes [P][d / 2]    element 2i of the head in the low half of byte i, 2i + 1 in the high half
//     value codes [P][d / 2]
//     key (scale, zero) [P][2] fp16, value (scale, zero) [P][2] fp16
// and a code c stands for scale * c + zero.  Codes, scales and zeros of consecutive tokens are contiguous, so a tile of
// tokens arrives in four bulk copies per page, and 16 tokens (the smallest page) fill whole 32-byte sectors.
#pragma once
#include <cuda_fp16.h>

#include "dq_common.h"
#include "dq_ptx.cuh"

namespace dq {

constexpr int kKv4Far = 1 << 30;  // positions, windows and sinks are cut here: sums of two of them stay in 32 bits

struct Kv4Batch {
  uint8_t* pages;
  int64_t page_stride;      // bytes from page to page
  int64_t num_pages;
  const int32_t* table;     // [B][table_stride]: page of tokens P * i ... of a sequence
  int64_t table_stride;
  const int32_t* kv_len;    // [B] tokens of a sequence, the new ones among them
  const int32_t* cu_new;    // [B + 1] first row of a sequence's new tokens, or null: T / B rows each
  int B, T, hkv, page_shift, capacity;  // capacity: tokens that a table row has room for
};

// Rows and length of sequence b.  Whatever the device arrays hold, rows stay in [0, T).
struct Kv4Seq {
  int row0, n, kv;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Batch& c, int b) {
  Kv4Seq s;
  if (c.cu_new != nullptr) {
    const int r0 = min(max(c.cu_new[b], 0), c.T), r1 = min(max(c.cu_new[b + 1], 0), c.T);
    s.row0 = r0;
    s.n = max(r1 - r0, 0);
  } else {
    s.n = c.T / c.B;
    s.row0 = b * s.n;
  }
  s.kv = min(max(c.kv_len[b], 0), kKv4Far);
  return s;
}

// Sequence of a token row (c.B: none), found by a whole warp: one round of loads for every 32 sequences.
__device__ __forceinline__ int kv4_seq_of_row(const Kv4Batch& c, int row, int lane) {
  if (c.cu_new == nullptr) return row / (c.T / c.B);
  int b = 0;
  for (int base = 0; base < c.B; base += 32) {
    const bool before = base + lane < c.B && c.cu_new[base + lane + 1] <= row;
    b += __popc(__ballot_sync(0xFFFFFFFFu, before));
  }
  return b;
}

// ------------------------------------------------------------------------------------------------------------------
// Division of the work.  A segment is (sequence, key/value head, tile of query rows); its rows are (token, query head of
// the group) pairs, token-major.  It reads the tokens that any of its rows sees, in tiles of TK tokens: with a window, first
// the tiles of the sinks, then those of the window.  All tiles of a call form one line, (sequence, head, row tile, token
// tile) with the last index running fastest, and CTA c takes the tiles [c * share, (c + 1) * share) of it: equal work
// whatever the lengths are, from lengths that only the device knows.  A CTA holds at most two segments that it shares with
// others, its first and its last; their sums go to the workspace and kv4_combine_kernel joins them, in the order of the CTAs.
// ------------------------------------------------------------------------------------------------------------------
struct Kv4Mask {
  int window, sinks;  // window 0: no window
};

struct Kv4Span {      // token tiles of a segment
  int count;          // at least one: a segment whose rows see nothing still has its rows written
  int sink_tiles, first;
  int p_lo, p_hi;     // positions of its first and last token
  __device__ __forceinline__ int tile(int u) const { return u < sink_tiles ? u : first + (u - sink_tiles); }
};

template <int TK>
__device__ __forceinline__ Kv4Span kv4_span(const Kv4Batch& c, const Kv4Seq& s, const Kv4Mask& m, int G, int row_tile, int R) {
  Kv4Span r;
  const int rows = s.n * G;
  const int i0 = row_tile * R / G, i1 = (min((row_tile + 1) * R, rows) - 1) / G;
  r.p_lo = s.kv - s.n + i0;
  r.p_hi = s.kv - s.n + i1;
  const int hi = min(min(r.p_hi + 1, s.kv), c.capacity);
  r.first = 0;
  r.sink_tiles = 0;
  if (hi <= 0) {
    r.count = 1;
    return r;
  }
  if (m.window > 0) {
    const int lo = max(0, r.p_lo - m.window + 1);
    r.first = min(lo, hi - 1) / TK;
    r.sink_tiles = min((m.sinks + TK - 1) / TK, r.first);
  }
  r.count = r.sink_tiles + (hi + TK - 1) / TK - r.first;
  return r;
}

__device__ __forceinline__ int kv4_row_tiles(const Kv4Seq& s, int G, int R) { return (s.n * G + R - 1) / R; }

template <int TK>
__device__ __forceinline__ long long kv4_units_per_head(const Kv4Batch& c, const Kv4Seq& s, const Kv4Mask& m, int G, int R) {
  long long n = 0;
  const int tiles = kv4_row_tiles(s, G, R);
  for (int rt = 0; rt < tiles; ++rt) n += kv4_span<TK>(c, s, m, G, rt, R).count;
  return n;
}

// Where a CTA is on the line of tiles.
struct Kv4Cursor {
  int b, h, rt;
  Kv4Seq seq;
  Kv4Span span;
  int u0, u1;      // this CTA's tiles of the segment
  long long left;  // tiles of the CTA behind this segment
};

// Steps over to the next segment that has tiles; false: none of the CTA's tiles are left.
template <int TK>
__device__ __forceinline__ bool kv4_next_segment(const Kv4Batch& c, const Kv4Mask& m, int G, int R, Kv4Cursor& k) {
  if (k.left <= 0) return false;
  if (++k.rt >= kv4_row_tiles(k.seq, G, R)) {
    k.rt = 0;
    if (++k.h >= c.hkv) {
      k.h = 0;
      do {
        if (++k.b >= c.B) return false;
        k.seq = kv4_seq(c, k.b);
      } while (k.seq.n == 0);
    }
  }
  k.span = kv4_span<TK>(c, k.seq, m, G, k.rt, R);
  k.u0 = 0;
  k.u1 = static_cast<int>(min(static_cast<long long>(k.span.count), k.left));
  k.left -= k.u1;
  return true;
}

struct Kv4Share {
  long long total, share;  // tiles of the call, tiles of a CTA
};

// Whole block of THREADS threads.  s_scan: THREADS + 1 long longs.  least: tiles that a CTA takes at least.
template <int TK, int THREADS>
__device__ __forceinline__ long long kv4_scan_units(const Kv4Batch& c, const Kv4Mask& m, int G, int R, int base,
                                                    long long* s_scan) {
  const int b = base + threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long n = 0;
  if (b < c.B) {
    const Kv4Seq s = kv4_seq(c, b);
    n = c.hkv * kv4_units_per_head<TK>(c, s, m, G, R);
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long v = __shfl_up_sync(0xFFFFFFFFu, n, d);
    if (lane >= d) n += v;
  }
  __shared__ long long s_warp[THREADS / 32];
  __syncthreads();
  if (lane == 31) s_warp[warp] = n;
  __syncthreads();
  for (int w = 0; w < warp; ++w) n += s_warp[w];
  s_scan[threadIdx.x + 1] = n;
  if (threadIdx.x == 0) s_scan[0] = 0;
  __syncthreads();
  return s_scan[THREADS];
}

template <int TK, int THREADS>
__device__ __forceinline__ Kv4Share kv4_share(const Kv4Batch& c, const Kv4Mask& m, int G, int R, int least, long long* s_scan) {
  Kv4Share r;
  r.total = 0;
  for (int base = 0; base < c.B; base += THREADS) r.total += kv4_scan_units<TK, THREADS>(c, m, G, R, base, s_scan);
  r.share = (r.total + gridDim.x - 1) / gridDim.x;
  if (r.share < least) r.share = least;
  return r;
}

// The segment that holds tile `at` (< total), with the tiles [at, at + want) of it and behind it.  Returns the number of the
// segment's first tile on the line.  Whole block; s_scan as kv4_share left it (its last round of sequences).
template <int TK, int THREADS>
__device__ __forceinline__ long long kv4_locate(const Kv4Batch& c, const Kv4Mask& m, int G, int R, long long at, long long want,
                                                long long* s_scan, Kv4Cursor& k) {
  long long before = 0;
  int base = 0;
  if (c.B > THREADS) {
    for (;; base += THREADS) {
      const long long n = kv4_scan_units<TK, THREADS>(c, m, G, R, base, s_scan);
      if (before + n > at || base + THREADS >= c.B) break;
      before += n;
    }
  }
  const long long rest = at - before;
  int lo = 0, hi = THREADS - 1;  // the last sequence whose tiles begin at or before `rest`: empty ones share a beginning
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_scan[mid] <= rest) lo = mid;
    else hi = mid - 1;
  }
  k.b = base + lo;
  k.seq = kv4_seq(c, k.b);
  long long in = rest - s_scan[lo];
  const long long per_head = (s_scan[lo + 1] - s_scan[lo]) / c.hkv;
  k.h = static_cast<int>(in / per_head);
  in -= k.h * per_head;
  k.rt = 0;
  k.span = kv4_span<TK>(c, k.seq, m, G, 0, R);
  while (in >= k.span.count) {
    in -= k.span.count;
    ++k.rt;
    k.span = kv4_span<TK>(c, k.seq, m, G, k.rt, R);
  }
  k.u0 = static_cast<int>(in);
  k.u1 = static_cast<int>(min(static_cast<long long>(k.span.count), in + want));
  k.left = want - (k.u1 - k.u0);
  return at - in;
}

// Sums of a segment that a CTA shares with others: [cta][0: its first segment, 1: its last][R rows: m, l, then O[d]]
__host__ __device__ constexpr size_t kv4_partial_floats(int R, int hd) { return static_cast<size_t>(R) * (hd + 2); }

int kv4_batch_of(const dq_kv4_batch* in, Kv4Batch* out);

struct Kv4AttnArgs {
  Kv4Batch c;
  Kv4Mask m;
  const unsigned short* q;  // bf16
  int64_t q_row, q_head;    // strides in elements
  unsigned short* out;      // bf16 [T][hq][d]
  float* partial;
  int G;
  float scale2;             // softmax scale * log2(e)
};

}  // namespace dq
