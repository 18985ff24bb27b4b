// Paged key/value cache in 4 bits: geometry of a page, the batch of a call, and the division of an attention's work.
//
// A page holds P tokens (P = 16, 32 ... 256).  Its block for one key/value head is P * (d + 8) bytes:
//     key codes [P][d / 2]    element 2i of the head in the low half of byte i, 2i + 1 in the high half
//     value codes [P][d / 2]
//     key (scale, zero) [P][2] fp16, value (scale, zero) [P][2] fp16
// and a code c stands for scale * c + zero.  Codes, scales and zeros of consecutive tokens are contiguous: a
// tile of tokens is four runs of bytes per page, and 16 tokens (the smallest page) fill whole 32-byte sectors of each.
#pragma once
#include <cuda_fp16.h>

#include "dq_common.h"
#include "dq_ptx.cuh"

namespace dq {

constexpr int kKv4Far = 1 << 30;  // positions, windows and sinks are cut here: sums of two of them stay in 32 bits

// Division by a number that the host knows: a product and a shift instead of the 150 cycles of an integer division, of which
// looking up a CTA's share alone took nine in a row.  n in [0, 2^31).
struct Kv4Div {
  uint32_t mul;
  int shift;
  __device__ __forceinline__ int operator()(int n) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift);
  }
};
inline Kv4Div kv4_div(int d) {
  int s = 0;
  while ((1ll << s) < d) ++s;
  // 2^31 <= mul < 2^32 for every d, and n * (mul * d - 2^(31 + s)) < 2^(31 + s): exact
  return {static_cast<uint32_t>((1ull << (31 + s)) / static_cast<uint32_t>(d) + 1), 31 + s};
}

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

// Sequence and position of a token row (c.B: it belongs to none), found by a whole warp with one round of loads for every 32
// sequences.
__device__ __forceinline__ int kv4_find(const Kv4Batch& c, int row, int lane, int* pos) {
  if (c.cu_new == nullptr) {
    const int n = c.T / c.B, b = row / n;
    *pos = min(max(c.kv_len[b], 0), kKv4Far) - n + (row - b * n);
    return b;
  }
  for (int base = 0; base < c.B; base += 32) {
    const int b = base + lane;
    Kv4Seq s = {0, 0, 0};
    if (b < c.B) s = kv4_seq(c, b);
    const uint32_t mine = __ballot_sync(0xFFFFFFFFu, row >= s.row0 && row - s.row0 < s.n);
    if (mine != 0) {
      const int l = __ffs(mine) - 1;
      *pos = __shfl_sync(0xFFFFFFFFu, s.kv - s.n + (row - s.row0), l);
      return base + l;
    }
  }
  *pos = -1;
  return c.B;
}

// The same for the lanes of a warp that have N rows from `row` on, each its `mine`-th; rows behind the last are none.
template <int N>
__device__ __forceinline__ void kv4_find_rows(const Kv4Batch& c, int row, int lane, int mine, int* b, int* pos) {
  if (c.cu_new == nullptr) {
    const int n = c.T / c.B;
    if (row + mine < c.T) {
      *b = (row + mine) / n;
      *pos = min(max(c.kv_len[*b], 0), kKv4Far) - n + (row + mine - *b * n);
    }
    return;
  }
  for (int base = 0; base < c.B; base += 32) {
    Kv4Seq s = {0, 0, 0};
    if (base + lane < c.B) s = kv4_seq(c, base + lane);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t has = __ballot_sync(0xFFFFFFFFu, row + i >= s.row0 && row + i - s.row0 < s.n);
      const int l = (__ffs(has) - 1) & 31, p = __shfl_sync(0xFFFFFFFFu, s.kv - s.n + (row + i - s.row0), l);
      if (has != 0 && i == mine && *b == c.B) *b = base + l, *pos = p;
    }
    if (__all_sync(0xFFFFFFFFu, *b < c.B)) break;
  }
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

struct Kv4Group {  // query heads of a key/value head
  int G;
  Kv4Div by;
};

struct Kv4Span {      // token tiles of a segment
  int count;          // at least one: a segment whose rows see nothing still has its rows written
  int sink_tiles, first;
  int p_lo, p_hi;     // positions of its first and last token
  __device__ __forceinline__ int tile(int u) const { return u < sink_tiles ? u : first + (u - sink_tiles); }
};

template <int TK>
__device__ __forceinline__ Kv4Span kv4_span(const Kv4Batch& c, const Kv4Seq& s, const Kv4Mask& m, const Kv4Group& g, int row_tile, int R) {
  Kv4Span r;
  const int rows = s.n * g.G;
  const int i0 = g.by(row_tile * R), i1 = g.by(min((row_tile + 1) * R, rows) - 1);
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

__device__ __forceinline__ int kv4_row_tiles(const Kv4Seq& s, const Kv4Group& g, int R) { return (s.n * g.G + R - 1) / R; }

template <int TK>
__device__ __forceinline__ int kv4_units_per_head(const Kv4Batch& c, const Kv4Seq& s, const Kv4Mask& m, const Kv4Group& g, int R) {
  int n = 0;
  const int tiles = kv4_row_tiles(s, g, R);
#pragma unroll 1
  for (int rt = 0; rt < tiles; ++rt) n += kv4_span<TK>(c, s, m, g, rt, R).count;
  return n;
}

// Where a CTA is on the line of tiles.
struct Kv4Cursor {
  int b, h, rt;
  Kv4Seq seq;
  Kv4Span span;
  int u0, u1;  // this CTA's tiles of the segment
  int left;    // tiles of the CTA behind this segment
};

// Steps over to the next segment that has tiles; false: none of the CTA's tiles are left.
template <int TK>
__device__ __forceinline__ bool kv4_next_segment(const Kv4Batch& c, const Kv4Mask& m, const Kv4Group& g, int R, Kv4Cursor& k) {
  if (k.left <= 0) return false;
  if (++k.rt >= kv4_row_tiles(k.seq, g, R)) {
    k.rt = 0;
    if (++k.h >= c.hkv) {
      k.h = 0;
      do {
        if (++k.b >= c.B) return false;
        k.seq = kv4_seq(c, k.b);
      } while (k.seq.n == 0);
    }
  }
  k.span = kv4_span<TK>(c, k.seq, m, g, k.rt, R);
  k.u0 = 0;
  k.u1 = min(k.span.count, k.left);
  k.left -= k.u1;
  return true;
}

struct Kv4Start {
  Kv4Cursor k;  // the CTA's first segment
  int share;    // tiles of every CTA
  bool any;     // false: the CTA has no tile
};
// Finds a CTA's share of the line and its first segment.  One warp.  grid: divides by gridDim.x; least: tiles a CTA takes at
// least.  Tile numbers are 32-bit; the host refuses batches that could pass that.
//
// The instructions of a kernel are cold when it starts (a pass through kv4_begin_any took 5000 cycles, a second one 1400), and
// what is read ahead ends at the next jump: batches of up to 128 sequences with one row tile each, the decode step, have a path
// without a loop, all others a function of their own.
__device__ __forceinline__ int kv4_warp_scan(int v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xFFFFFFFFu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}
__device__ __forceinline__ int kv4_share_of(int total, int least, Kv4Div grid) {
  // (the sum passes 31 bits for a total within gridDim.x of 2^31)
  const int g = static_cast<int>(gridDim.x);
  return max(total < 0x7FFF0000 ? grid(total + g - 1) : total / g + 1, least);
}
// in / per_head, below 1024: the quotient of floats is off by less than one
__device__ __forceinline__ int kv4_head_of(int in, int per_head) {
  int h = static_cast<int>(__fdividef(static_cast<float>(in), static_cast<float>(per_head)));
  if (h * per_head > in) --h;
  if ((h + 1) * per_head <= in) ++h;
  return h;
}

// a / b of positive numbers: the quotient of floats, put right
__device__ __forceinline__ int kv4_quotient(int a, int b) {
  int q = static_cast<int>(__fdividef(static_cast<float>(a), static_cast<float>(b)));
  q -= static_cast<long long>(q) * b > a ? 1 : 0;
  q += static_cast<long long>(q + 1) * b <= a ? 1 : 0;
  return q;
}

// Any batch: a lane adds up B / 32 neighbouring sequences, and the sequences of the lane that holds the first tile are added up
// once more, one a lane (two rounds of loads for up to 1024).
template <int TK>
__device__ __forceinline__ Kv4Start kv4_begin_any(const Kv4Batch& c, const Kv4Mask& m, const Kv4Group& g, int R, int least,
                                                  Kv4Div grid, int lane) {
  Kv4Start r;
  Kv4Cursor& k = r.k;
  const int each = (c.B + 31) / 32;
  int n = 0, rows = 0;
#pragma unroll 1
  for (int i = 0; i < each; ++i) {
    const int b = lane * each + i;
    if (b < c.B) {
      const Kv4Seq s = kv4_seq(c, b);
      rows = min(rows + s.n, c.T + 1);
      n += kv4_units_per_head<TK>(c, s, m, g, R) * c.hkv;
    }
  }
  // Row offsets that overlap: more tiles than the host's limit counted on, whose numbers could pass 32 bits.  Nothing is done.
  const uint64_t rows_hi = __reduce_add_sync(0xFFFFFFFFu, static_cast<uint32_t>(rows) >> 16);
  const uint64_t rows_lo = __reduce_add_sync(0xFFFFFFFFu, static_cast<uint32_t>(rows) & 0xFFFFu);
  r.any = (rows_hi << 16) + rows_lo <= static_cast<uint64_t>(c.T);
  if (!r.any) return r;
  const int upto = kv4_warp_scan(n, lane), total = __shfl_sync(0xFFFFFFFFu, upto, 31);
  r.share = kv4_share_of(total, least, grid);
  const long long at = static_cast<long long>(blockIdx.x) * r.share;
  r.any = at < total;
  if (!r.any) return r;
  const int begin = static_cast<int>(at);
  int owner = __ffs(__ballot_sync(0xFFFFFFFFu, upto > begin)) - 1;
  int in = begin - __shfl_sync(0xFFFFFFFFu, upto - n, owner);
  k.b = owner * each;
  int per_head = 0, u = 0, v = 0;
  uint32_t past = 0;
#pragma unroll 1
  for (int base = 0; base < each; base += 32) {
    const int b = owner * each + base + lane;
    per_head = 0;
    if (base + lane < each && b < c.B) per_head = kv4_units_per_head<TK>(c, kv4_seq(c, b), m, g, R);
    v = per_head * c.hkv;
    u = kv4_warp_scan(v, lane);
    past = __ballot_sync(0xFFFFFFFFu, u > in);
    if (past != 0) break;  // (one of them holds the tile)
    k.b += 32;
    in -= __shfl_sync(0xFFFFFFFFu, u, 31);
  }
  owner = (__ffs(past) - 1) & 31;
  k.b += owner;
  in -= __shfl_sync(0xFFFFFFFFu, u - v, owner);
  per_head = __shfl_sync(0xFFFFFFFFu, per_head, owner);
  k.seq = kv4_seq(c, k.b);
  k.h = kv4_head_of(in, per_head);
  in -= k.h * per_head;
  k.rt = 0;
  k.span = kv4_span<TK>(c, k.seq, m, g, 0, R);
#pragma unroll 1
  while (in >= k.span.count) {
    in -= k.span.count;
    ++k.rt;
    k.span = kv4_span<TK>(c, k.seq, m, g, k.rt, R);
  }
  const int want = min(r.share, total - begin);
  k.u0 = in;
  k.u1 = min(k.span.count, in + want);
  k.left = want - (k.u1 - k.u0);
  return r;
}

template <int TK>
__device__ __noinline__ Kv4Start kv4_begin_apart(const Kv4Batch& c, const Kv4Mask& m, const Kv4Group& g, int R, int least,
                                                 Kv4Div grid, int lane) {
  return kv4_begin_any<TK>(c, m, g, R, least, grid, lane);
}

template <int TK>
__device__ __forceinline__ Kv4Start kv4_begin(const Kv4Batch& c, const Kv4Mask& m, const Kv4Group& g, int R, int least, Kv4Div grid,
                                              int lane) {
  constexpr int N = 4;  // sequences of a lane
  const int each = c.B <= 32 ? 1 : N;
  Kv4Seq seq[N];
  bool one = c.B <= 32 * N;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    seq[i] = {0, 0, 0};
    const int b = lane * each + i;
    if (i < each && b < c.B) seq[i] = kv4_seq(c, b);
    one &= seq[i].n * g.G <= R;
  }
  if (!__all_sync(0xFFFFFFFFu, one)) return kv4_begin_apart<TK>(c, m, g, R, least, grid, lane);
  Kv4Start r;
  int weight[N], units = 0, segments = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    weight[i] = seq[i].n > 0 ? kv4_span<TK>(c, seq[i], m, g, 0, R).count : 0;
    units += weight[i];
    segments += seq[i].n > 0 ? 1 : 0;
  }
  const int total_units = __reduce_add_sync(0xFFFFFFFFu, units) * c.hkv;
  segments = __reduce_add_sync(0xFFFFFFFFu, segments) * c.hkv;
  // Few segments (a batch of one): each is cut into parts of `share` tiles for itself, at most `gridDim.x` in all, so that no CTA
  // begins a second segment when the others are done.  One sequence of 100000 tokens, 8 heads: 30.0 us, 30.9 on one line.  Shares
  // are up to a 31st larger, which is why more segments stay on the line: there a second one is the smaller loss.
  const int spare = static_cast<int>(gridDim.x) - segments;
  const bool cut = segments * 32 <= static_cast<int>(gridDim.x);
  if (cut) {
    r.share = max(kv4_quotient(total_units + spare - 1, spare), least);
#pragma unroll
    for (int i = 0; i < N; ++i) weight[i] = kv4_quotient(weight[i] + r.share - 1, r.share);
  } else {
    r.share = kv4_share_of(total_units, least, grid);
  }
  int upto[N], n = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    n += weight[i] * c.hkv;
    upto[i] = n;
  }
  const int all = kv4_warp_scan(n, lane), total = __shfl_sync(0xFFFFFFFFu, all, 31);
  const long long at = cut ? blockIdx.x : static_cast<long long>(blockIdx.x) * r.share;
  r.any = at < total;
  const int begin = static_cast<int>(at);
  const int owner = (__ffs(__ballot_sync(0xFFFFFFFFu, all > begin)) - 1) & 31;
  int in = begin - (all - n), which = 0;  // of use in the owner
  Kv4Seq s = seq[0];
#pragma unroll
  for (int i = 1; i < N; ++i)
    if (in >= upto[i - 1]) {
      s = seq[i];
      weight[0] = weight[i];
      which = i;
    }
#pragma unroll
  for (int i = N - 1; i > 0; --i)
    if (which == i) in -= upto[i - 1];
  Kv4Cursor& k = r.k;
  in = __shfl_sync(0xFFFFFFFFu, in, owner);
  const int per_head = __shfl_sync(0xFFFFFFFFu, weight[0], owner);
  k.b = owner * each + __shfl_sync(0xFFFFFFFFu, which, owner);
  k.rt = 0;
  k.seq.row0 = __shfl_sync(0xFFFFFFFFu, s.row0, owner);
  k.seq.n = __shfl_sync(0xFFFFFFFFu, s.n, owner);
  k.seq.kv = __shfl_sync(0xFFFFFFFFu, s.kv, owner);
  k.span = kv4_span<TK>(c, k.seq, m, g, 0, R);
  k.h = kv4_head_of(in, per_head);
  in -= k.h * per_head;
  const int want = cut ? r.share : min(r.share, total - begin);
  k.u0 = cut ? in * r.share : in;
  k.u1 = min(k.span.count, k.u0 + want);
  k.left = cut ? 0 : want - (k.u1 - k.u0);
  return r;
}

// Workspace: a Kv4Join for every CTA, then the sums of segments that it shares with others, [cta][0: its first segment, 1: its
// last][m, l of R rows, then O of R rows].
struct Kv4Join {
  int parts;     // CTAs from this one on that hold a part of the segment which begins in this one; 0: none goes on
  int slot;      // where this CTA's part is
  int rows, first_row, row0, h;
};
__host__ __device__ constexpr size_t kv4_partial_floats(int R, int hd) { return static_cast<size_t>(R) * (hd + 2); }

// Tiles of the two attention kernels: tokens, query rows, and the least tiles of a CTA.
constexpr int kDecTile = 32, kDecLeast = 4;                    // 8 or 16 rows
constexpr int kPreTile = 128, kPreLeast = 2;                 // 128 or 256
constexpr float kKv4NoMax = -1e30f;  // reference point of a row that has seen no token

// A query row as fp16: times +-2^p, which brings its largest element to [2^14, 2^15) and gives it the scale's sign (0: a scale of
// zero); scores of such elements are to be multiplied with `back`, which is positive.
// Where the largest element times the scale would pass 2^64, `back` is taken of 2^64: scores stay finite and above kKv4NoMax, and
// the row's weights are what they would be, one at the largest score and zero elsewhere (of scores of 2^64 keys fp32 resolves
// 2^40 keys, and a key's smallest step is 2^-24).
struct Kv4RowScale {
  float up, back;
};
// big: bits of the row's largest bf16 element, 0 for a row that is not finite
__device__ __forceinline__ Kv4RowScale kv4_row_scale(uint32_t big, float scale2) {
  const int e = big > 0 ? static_cast<int>(big >> 7) - 127 : 0;
  const int p = min(14 - e, 126);  // -113 ... 126
  const int over = max(e + static_cast<int>((__float_as_uint(scale2) >> 23) & 255u) - 127 - 63, 0);
  // (over > 0 only where e > -64: p + over lies in [-113, 126] or, with over, up to 78)
  const float up = __uint_as_float(static_cast<uint32_t>(127 + p) << 23);
  const float back = fabsf(scale2) * __uint_as_float(static_cast<uint32_t>(127 - p - over) << 23);
  return {scale2 > 0.0f ? up : scale2 < 0.0f ? -up : 0.0f, scale2 != 0.0f ? fmaxf(back, 1.2e-38f) : 1.0f};
}

// Weights are 2^(s mul - m) with one fused operation, whose product is not rounded as m once was: from |m| = 2^27 on they could
// pass what fp16 holds, or all be zero.  From 2^24 on a row goes on in units 2^k of scores that keep |m| below that (m and mul divided by
// it, `unit` multiplied: m * unit is the score).  Scores that such units bring together differ by less than 2^-19 of their size,
// which a sum of 128 products in fp32 may not tell apart either.
__device__ __forceinline__ void kv4_units(float& m, float& mul, float& unit) {
  if (fabsf(m) >= 16777216.0f && m != kKv4NoMax) {
    const uint32_t e = (__float_as_uint(m) >> 23) & 255u;  // 151 ... 215
    const float by = __uint_as_float((277u - e) << 23);
    m *= by;
    mul *= by;
    unit *= __uint_as_float((e - 23u) << 23);
  }
}

int kv4_batch_of(const dq_kv4_batch* in, Kv4Batch* out);

struct Kv4AttnArgs {
  Kv4Batch c;
  Kv4Mask m;
  const unsigned short* q;  // bf16
  int64_t q_row, q_head;    // strides in elements
  unsigned short* out;      // bf16 [T][hq][d]
  Kv4Join* join;
  float* partial;
  Kv4Group g;
  Kv4Div grid;              // by the number of CTAs
  float scale2;             // softmax scale * log2(e)
};

int kv4_decode_resident(int hd, int R);  // CTAs per SM
int launch_kv4_decode(const Kv4AttnArgs& a, int hd, int R, int grid, cudaStream_t s);
int launch_kv4_prefill(const Kv4AttnArgs& a, int hd, int R, int grid, cudaStream_t s, DeviceState* st);

}  // namespace dq
