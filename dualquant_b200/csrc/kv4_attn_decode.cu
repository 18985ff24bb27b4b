// Attention of a few query rows per sequence over the paged 4-bit cache (decode steps, drafted tokens).
//
//   o = sum_j p_j (s_j c_j + z_j) / sum_j p_j,   p_j = 2^(x_j - m),   x_j = scale log2(e) q . (s'_j c'_j + z'_j)
// with the scales outside of the matrix products:
//   q . (s c + z) = s (q . c) + z (q . 1),   sum_j p_j (s_j c_j + z_j) = sum_j (p_j s_j) c_j + sum_j p_j z_j
// so that the products run on the bare codes.  A 4-bit code in the low bits of an fp16 word IS an fp16 number, the subnormal
// c * 2^-24 (in bits 4 to 7: c * 2^-20): an AND makes two operands of mma.sync.m16n8k16, with no conversion, and the powers
// of two go into the row's factor, into every other query element, and into the last factor of the output.  A code costs
// 0.6 (keys) and 0.75 (values) instructions.
//
// Both products are taken transposed, keys or head elements along the 16 rows and up to eight query rows along the columns
// (S' = K Q', O' = V' P'), which wastes nothing on groups of up to eight query rows.  movmatrix turns the weights of S' into
// the operand of O'.  Query elements are permuted to the order in which nibbles come out of a 16-byte load.
//
// Each warp has a ring of its own of two tiles of 32 tokens in shared memory, which it fills with asynchronous 16-byte copies,
// and takes every fourth tile of its CTA's share; the warps meet once per segment, in the halves of their rings that are free
// then.  (Bulk copies, four a tile and page, issued by one lane with a barrier to wait for: 32.4 us where these take 30.6 on 16
// sequences of up to 8000 tokens, 265 and 257 on the batch below, at that stage.)
// Weights and sums:
//   * p_j s_j is fp16 (an mma operand, 2^-11 relative, in the row's own scale): the reference point m is taken of
//     x_j + exponent(s_j), so that p_j s_j stays below 2^10 and what counts stays normal whatever the scales are.  The rounding
//     meets codes 0 ... 15 and not the centred values: outputs are up to 17 % further from 64 bits than their bf16 rounding is;
//   * m moves only where a row would pass 2^8 above it; l, sum p z and O are fp32.
// Query rows are fp16 times a power of two of the row: an element is exact down to 2^-27 of the row's largest one (fp16 has its
// 8 bits down to 2^-17, every other element is taken times 1 / 16), and no row knows of its neighbours.
//
// 64 sequences of up to 16384 tokens, 8 heads of 128, four rows each, 1.14 GB: 220 us replayed from a graph (5.2 TB/s, 80 % of
// what a plain copy moves), 249 us a call when the inputs change from call to call (71 %).  No unit is at its end (integer pipe 60 %
// of its cycles, issue slots 56 %, memory 61 %): the twelve warps of an SM wait for their own results of fixed latency, 1.4
// cycles an issue.  Small batches pay for the launch, a first look at cold instructions, three
// dependent loads (lengths, pages, codes) and the second kernel: 9.3 us for one row over 300 tokens.  Four CTAs an SM at 128
// registers, three stages at two CTAs an SM, and tiles of 64 tokens were no faster.
#include "kv4.cuh"

namespace dq {

constexpr int kDecWarps = 4;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kDecStages = 2;    // tiles of a warp's ring
constexpr int kPieces = kDecTile / 16;
constexpr int kDecQueries = kDecStages + 1;  // query rows of a segment are copied when its predecessor's last tile is

template <int HD>
constexpr int kQPitch = 2 * HD + 16;  // bytes

template <int HD, int NT>
struct DecSmem {
  static constexpr int R = 8 * NT;
  static constexpr int kStage = kDecTile * (HD + 8);
  // Where the warps' outputs meet: up to eight rows in the half of a warp's ring that it fills next, sixteen in a place of
  // their own.
  static constexpr int kPitch = HD + 8;  // floats per row
  static constexpr int kRing = kDecWarps * kDecStages * kStage;
  static constexpr bool kMeetInRing = R * kPitch * 4 <= kStage;
  static constexpr int kOffMl = kRing + (kMeetInRing ? 0 : kDecWarps * R * kPitch * 4);
  static constexpr int kQBytes = R * kQPitch<HD>;
  static constexpr int kOffHalf = kOffMl + kDecWarps * R * 2 * 4;
  static constexpr int kOffQ = kOffHalf + 16;
  static constexpr int kOffCursor = kOffQ + kDecQueries * kQBytes;
  static constexpr int kBytes = kOffCursor + static_cast<int>(sizeof(Kv4Cursor)) + 8;
  static_assert(kOffQ % 16 == 0 && kOffCursor % 4 == 0, "alignment");
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst, const void* src, bool is) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(is ? 16 : 0) : "memory");
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// The query rows of a segment as the second operand of S' = K Q'.
template <int HD, int NT>
struct DecQuery {
  static constexpr int KS = HD / 16;  // steps of 16 head elements
  uint32_t f[NT][KS][2];
  // of query rows 2t and 2t + 1:
  float2 mul[NT];    // what s S' + z zq has to be multiplied with to be scores in base 2; positive
  float2 zq[NT];     // sum of a row's elements, in units of S'; NaN for a row that is not finite
  int pos[NT][2];    // the row's position; -1: no such row

  // rows: the segment's query rows in shared memory, bf16, kQPitch bytes apart; rows that do not exist are zero
  __device__ __forceinline__ void load(const Kv4AttnArgs& a, const Kv4Cursor& k, const uint8_t* q_rows, int lane) {
    constexpr int R = 8 * NT, W = HD / 32;  // W: 32-bit words of codes per lane
    const int g = lane >> 2, t = lane & 3, rows = k.seq.n * a.g.G;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint8_t* src = q_rows + (nt * 8 + g) * kQPitch<HD> + t * (W * 16);
      uint32_t raw[W * 4];  // pairs of bf16
      uint32_t big = 0;     // largest size of an element, as bf16 bits
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint4 v = *reinterpret_cast<const uint4*>(src + 16 * w);
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          raw[4 * w + j] = u[j];
          big = __vmaxu2(big, u[j] & 0x7FFF7FFFu);
        }
      }
      big = max(big & 0xFFFFu, big >> 16);
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, d));
      const bool fine = big < 0x7F80u;  // no infinity and no NaN in the row
      if (!fine) {
#pragma unroll
        for (int j = 0; j < W * 4; ++j) raw[j] = 0;
      }
      const Kv4RowScale by = kv4_row_scale(fine ? big : 0, a.scale2);
      float2 s[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
      for (int j = 0; j < W * 4; ++j)
        s[j & 1] = __ffma2_rn(make_float2(__uint_as_float(raw[j] << 16), __uint_as_float(raw[j] & 0xFFFF0000u)), both(by.up), s[j & 1]);
      s[0] = __fadd2_rn(s[0], s[1]);
      float total = s[0].x + s[0].y;
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, d);
      const float sum = fine ? total * 0x1p-24f : __int_as_float(0x7FC00000), back = by.back * 16777216.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          // elements 2u, 2u + 1 and 2u + 4, 2u + 5 of eight: the order of the nibbles (0, 4), (1, 5) ... of a word
          const uint32_t p = raw[4 * w + u], r = raw[4 * w + u + 2];
          const float2 even = __fmul2_rn(make_float2(__uint_as_float(p << 16), __uint_as_float(r << 16)), both(by.up));
          const float2 odd = __fmul2_rn(make_float2(__uint_as_float(p & 0xFFFF0000u), __uint_as_float(r & 0xFFFF0000u)),
                                        both(by.up * 0.0625f));
          f[nt][2 * w + u][0] = half2_bits(even.x, even.y);
          f[nt][2 * w + u][1] = half2_bits(odd.x, odd.y);
        }
      }
      mul[nt] = make_float2(__shfl_sync(0xFFFFFFFFu, back, 8 * t), __shfl_sync(0xFFFFFFFFu, back, 8 * t + 4));
      zq[nt] = make_float2(__shfl_sync(0xFFFFFFFFu, sum, 8 * t), __shfl_sync(0xFFFFFFFFu, sum, 8 * t + 4));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = k.rt * R + nt * 8 + 2 * t + i;
        pos[nt][i] = r < rows ? k.seq.kv - k.seq.n + a.g.by(r) : -1;
      }
    }
  }
};

template <int HD, int NT>
__global__ void __launch_bounds__(kDecThreads, NT == 1 ? 3 : 2)
kv4_decode_kernel(const __grid_constant__ Kv4AttnArgs a) {
  grid_dep_launch_dependents();
  extern __shared__ __align__(128) uint8_t smem[];
  using L = DecSmem<HD, NT>;
  constexpr int R = L::R, MT = HD / 16, W = HD / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * kDecStages * L::kStage;
  grid_dep_wait();
  // One warp looks up the CTA's share: its loads go to lines that every CTA wants at once.
  Kv4Cursor& found = *reinterpret_cast<Kv4Cursor*>(smem + L::kOffCursor);
  int* s_share = reinterpret_cast<int*>(&found + 1);  // tiles of a CTA; 0: none for this one
  if (warp == 0) {
    const Kv4Start k = kv4_begin<kDecTile>(a.c, a.m, a.g, R, kDecLeast, a.grid, lane);
    if (lane == 0) {
      if (k.any) found = k.k;
      else a.join[blockIdx.x].parts = 0;
      *s_share = k.any ? k.share : 0;
    }
  }
  __syncthreads();
  const int share = *s_share;
  if (share == 0) return;
  Kv4Cursor at = found;
  Kv4Cursor ahead = at;  // where the copies are
  const int P = 1 << a.c.page_shift;

  // A tile arrives in pieces of 16 tokens, each of one page, or from one page: lane l copies every 32nd 16 bytes of the codes,
  // lanes 0 to 7 the pairs of keys, 8 to 15 of values.  The page of piece i is kept by lane i, one tile ahead.
  bool more = true;
  int next_u = ahead.u0 + warp, next_page = -1, next_tok = 0;
  const uint8_t *src_codes = nullptr, *src_pairs = nullptr;  // the lane's 16 bytes of the head's block in page 0
  const int32_t* table_row = nullptr;                        // the sequence's pages
  int there = 0;                                             // the sequence's tokens that the table has room for
  int q_ahead = 0;
  auto seek_segment = [&]() {
    const uint8_t* block = a.c.pages + static_cast<int64_t>(ahead.h) * P * (HD + 8);
    src_codes = block + lane * 16;
    src_pairs = block + P * HD + ((lane >> 3) & 1) * 4 * P + (lane & 7) * 16;
    table_row = a.c.table + ahead.b * a.c.table_stride;
    there = min(ahead.seq.kv, a.c.capacity);
  };
  auto copy_queries = [&]() {
    if (warp == 0) {
      const int first_row = ahead.rt * R, rows = ahead.seq.n * a.g.G;
      const uint32_t to = smem_u32(smem + L::kOffQ) + q_ahead * L::kQBytes;
      for (int c = lane; c < R * HD / 8; c += 32) {
        const int row = c / (HD / 8), col = c % (HD / 8), r = first_row + row;
        const bool is = r < rows;
        const int i = is ? a.g.by(r) : 0, head = ahead.h * a.g.G + (is ? r - i * a.g.G : 0);
        cp_async_16_or_zero(to + row * kQPitch<HD> + col * 16,
                            a.q + static_cast<int64_t>(ahead.seq.row0 + i) * a.q_row + static_cast<int64_t>(head) * a.q_head + col * 8,
                            is);
      }
      if (++q_ahead == kDecQueries) q_ahead = 0;
    }
  };
  auto seek = [&]() {  // the warp's next tile, and its pages
    bool other = false;
    while (next_u >= ahead.u1) {
      other = true;
      more = kv4_next_segment<kDecTile>(a.c, a.m, a.g, R, ahead);
      if (!more) return;
      next_u = ahead.u0 + warp;
      seek_segment();
    }
    next_tok = ahead.span.tile(next_u) * kDecTile;
    const int tok = next_tok + lane * 16;
    next_page = lane < kPieces && tok < there ? table_row[tok >> a.c.page_shift] : -1;
    if (other) copy_queries();
  };
  const uint32_t dst_codes = smem_u32(ring) + lane * 16;
  const uint32_t dst_pairs = smem_u32(ring) + kDecTile * HD + ((lane >> 3) & 1) * kDecTile * 4 + (lane & 7) * 16;
  const uint32_t page_bytes = static_cast<uint32_t>(a.c.page_stride);
  auto fetch = [&](int stage) {  // which pieces of the tile are there
    uint32_t got = 0;
    if (more) {
      got = __ballot_sync(0xFFFFFFFFu, static_cast<uint32_t>(next_page) < static_cast<uint32_t>(a.c.num_pages));
      if (P >= kDecTile) {  // one page
        if (got & 1u) {
          const uint64_t off = static_cast<uint64_t>(static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, next_page, 0))) * page_bytes;
          const int slot = next_tok & (P - 1);
          const uint8_t* codes = src_codes + off + slot * (HD / 2);
          const uint32_t to = dst_codes + stage * L::kStage;
#pragma unroll
          for (int j = 0; j < HD / 32; ++j) {
            cp_async_16(to + j * 512, codes + j * 512);
            cp_async_16(to + kDecTile * (HD / 2) + j * 512, codes + P * (HD / 2) + j * 512);
          }
          if (lane < 16) cp_async_16(dst_pairs + stage * L::kStage, src_pairs + off + slot * 4);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const uint32_t page = static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, next_page, i));
          if ((got >> i) & 1u) {
            const uint64_t off = static_cast<uint64_t>(page) * page_bytes;
            const int slot = (next_tok + 16 * i) & (P - 1);
            const uint8_t* codes = src_codes + off + slot * (HD / 2);
            const uint32_t to = dst_codes + stage * L::kStage + i * 16 * (HD / 2);
#pragma unroll
            for (int j = 0; j < HD / 64; ++j) {
              cp_async_16(to + j * 512, codes + j * 512);
              cp_async_16(to + kDecTile * (HD / 2) + j * 512, codes + P * (HD / 2) + j * 512);
            }
            if ((lane & 7) < 4 && lane < 16) cp_async_16(dst_pairs + stage * L::kStage + i * 64, src_pairs + off + slot * 4);
          }
        }
      }
      next_u += kDecWarps;
      seek();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");  // (an empty one too: groups are counted)
    return got;
  };
  seek_segment();
  seek();
  copy_queries();
  asm volatile("cp.async.commit_group;" ::: "memory");
  static_assert(kDecStages == 2, "a tile is fetched while its predecessor is worked on");
  uint32_t got_next = fetch(0);
  // the first segment's queries have arrived (the others': see kDecQueries)
  asm volatile("cp.async.wait_group %0;" ::"n"(kDecStages - 1) : "memory");
  __syncthreads();

  int stage = 0, q_at = 0;
  bool is_first = true, goes_on = false;
  for (;; is_first = false) {
    DecQuery<HD, NT> q;
    q.load(a, at, smem + L::kOffQ + q_at * L::kQBytes, lane);
    if (++q_at == kDecQueries) q_at = 0;
    float o[NT][MT][4];
    float2 m[NT], l[NT], z[NT], unit[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < MT; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.0f;
      m[nt] = make_float2(kKv4NoMax, kKv4NoMax);
      l[nt] = z[nt] = make_float2(0.0f, 0.0f);
      unit[nt] = make_float2(1.0f, 1.0f);
    }
    const int kv = min(at.seq.kv, a.c.capacity);
    // tiles from these tokens on are seen whole by every row
    const int whole_hi = min(kv, at.span.p_lo + 1) - kDecTile, whole_lo = a.m.window > 0 ? at.span.p_hi - a.m.window : -1,
              whole_sinks = a.m.window > 0 ? a.m.sinks - kDecTile : -1;
    for (int u = at.u0 + warp; u < at.u1; u += kDecWarps) {
      const uint8_t* buf = ring + stage * L::kStage;
      const int base = at.span.tile(u) * kDecTile;
      const uint32_t got = got_next;
      got_next = fetch(stage ^ 1);  // into the tile that was read last
      asm volatile("cp.async.wait_group %0;" ::"n"(kDecStages - 1) : "memory");
      __syncwarp();
      const bool whole = got == (1u << kPieces) - 1 && base <= whole_hi && (base > whole_lo || base <= whole_sinks);
      const __half2* kpar = reinterpret_cast<const __half2*>(buf + kDecTile * HD);
      const __half2* vpar = kpar + kDecTile;
      // S' = K Q': rows g and g + 8 are tokens.  Two chains of sums for each 16 tokens: a chain's products wait for one another
      float2 x[kPieces][NT][2];  // scores of tokens 16 i + g and 16 i + g + 8, query rows 2t and 2t + 1, over q.mul
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        uint32_t ka[W], kb[W];
        const uint8_t* row = buf + (i * 16 + g) * (HD / 2) + t * (HD / 8);
        if constexpr (W == 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(row), v = *reinterpret_cast<const uint4*>(row + 8 * (HD / 2));
          ka[0] = u.x, ka[1] = u.y, ka[2] = u.z, ka[3] = u.w;
          kb[0] = v.x, kb[1] = v.y, kb[2] = v.z, kb[3] = v.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(row), v = *reinterpret_cast<const uint2*>(row + 8 * (HD / 2));
          ka[0] = u.x, ka[1] = u.y;
          kb[0] = v.x, kb[1] = v.y;
        }
        float s[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][0][e] = s[nt][1][e] = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const uint32_t xa = ka[w] >> (8 * v), xb = kb[w] >> (8 * v);
            const uint32_t a0 = xa & 0x000F000Fu, a1 = xb & 0x000F000Fu, a2 = xa & 0x00F000F0u, a3 = xb & 0x00F000F0u;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt][v], a0, a1, a2, a3, q.f[nt][2 * w + v][0], q.f[nt][2 * w + v][1]);
          }
        const float2 k0 = __half22float2(kpar[i * 16 + g]), k1 = __half22float2(kpar[i * 16 + g + 8]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 s0 = __fadd2_rn(make_float2(s[nt][0][0], s[nt][0][1]), make_float2(s[nt][1][0], s[nt][1][1]));
          const float2 s1 = __fadd2_rn(make_float2(s[nt][0][2], s[nt][0][3]), make_float2(s[nt][1][2], s[nt][1][3]));
          // (one query tile: scalars, which need no pair made of a scale; two: pairs.  The other way round 222.3 us where this
          // takes 220.1 on the batch above, and 61.2 where 60.4 for four tokens of 16 x 30000, 16 heads of 64 over 2)
          if constexpr (NT == 1) {
            x[i][nt][0] = make_float2(fmaf(k0.x, s0.x, k0.y * q.zq[nt].x), fmaf(k0.x, s0.y, k0.y * q.zq[nt].y));
            x[i][nt][1] = make_float2(fmaf(k1.x, s1.x, k1.y * q.zq[nt].x), fmaf(k1.x, s1.y, k1.y * q.zq[nt].y));
          } else {
            x[i][nt][0] = __ffma2_rn(both(k0.x), s0, __fmul2_rn(both(k0.y), q.zq[nt]));
            x[i][nt][1] = __ffma2_rn(both(k1.x), s1, __fmul2_rn(both(k1.y), q.zq[nt]));
          }
        }
      }
      // value scales and zeros, and the exponents of the scales
      float2 vp[kPieces][2];
      float ve[kPieces][2];
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          __half2 h = vpar[i * 16 + 8 * j + g];
          // slots that hold no token may hold anything
          if (!whole && (base + i * 16 + 8 * j + g >= kv || !((got >> i) & 1u))) h = __half2half2(__ushort_as_half(0));
          vp[i][j] = __half22float2(h);
          ve[i][j] = static_cast<float>(static_cast<int>((__half_as_ushort(__low2half(h)) >> 10) & 31u) - 15);
        }
      if (!whole) {
        auto see = [&](int i, int j, int p) {
          return ((got >> i) & 1u) && j < kv && j <= p && (a.m.window == 0 || j > p - a.m.window || j < a.m.sinks);
        };
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int tok = base + i * 16 + 8 * j + g;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (!see(i, tok, q.pos[nt][0])) x[i][nt][j].x = -INFINITY;
              if (!see(i, tok, q.pos[nt][1])) x[i][nt][j].y = -INFINITY;
            }
          }
      }
      bool lift = false;
      float2 high[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        high[nt] = make_float2(-INFINITY, -INFINITY);
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 v = __ffma2_rn(x[i][nt][j], q.mul[nt], both(ve[i][j]));
            high[nt] = make_float2(fmaxf(high[nt].x, v.x), fmaxf(high[nt].y, v.y));
          }
        lift |= high[nt].x > m[nt].x + 8.0f || high[nt].y > m[nt].y + 8.0f;
      }
      if (__any_sync(0xFFFFFFFFu, lift)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            high[nt].x = fmaxf(high[nt].x, __shfl_xor_sync(0xFFFFFFFFu, high[nt].x, d));
            high[nt].y = fmaxf(high[nt].y, __shfl_xor_sync(0xFFFFFFFFu, high[nt].y, d));
          }
          high[nt] = make_float2(fmaxf(high[nt].x, m[nt].x), fmaxf(high[nt].y, m[nt].y));
          const float2 by = make_float2(exp2_approx(m[nt].x - high[nt].x), exp2_approx(m[nt].y - high[nt].y));
          m[nt] = high[nt];
          kv4_units(m[nt].x, q.mul[nt].x, unit[nt].x);
          kv4_units(m[nt].y, q.mul[nt].y, unit[nt].y);
          l[nt] = __fmul2_rn(l[nt], by);
          z[nt] = __fmul2_rn(z[nt], by);
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            o[nt][j][0] *= by.x, o[nt][j][1] *= by.y;
            o[nt][j][2] *= by.x, o[nt][j][3] *= by.y;
          }
        }
      }
      // weights
      uint32_t pb[kPieces][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float2 low = make_float2(-m[nt].x, -m[nt].y);
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 y = __ffma2_rn(x[i][nt][j], q.mul[nt], low);
            const float2 p = make_float2(exp2_approx(y.x), exp2_approx(y.y));
            l[nt] = __fadd2_rn(l[nt], p);
            z[nt] = __ffma2_rn(p, both(vp[i][j].y), z[nt]);
            const float2 w = __fmul2_rn(p, both(vp[i][j].x));
            pb[i][nt][j] = transpose_8x8(half2_bits(w.x, w.y));
          }
      }
      // O' += V' P': rows g and g + 8 are head elements, columns of V' the tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        constexpr int VW = HD / 64;  // words of a token's value codes per lane
        const uint8_t* row = buf + kDecTile * (HD / 2) + (i * 16 + 2 * t) * (HD / 2) + g * (HD / 16);
        uint32_t v[4][VW];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint8_t* p = row + ((c & 1) + 8 * (c >> 1)) * (HD / 2);
          if constexpr (VW == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            v[c][0] = u.x, v[c][1] = u.y;
          } else {
            v[c][0] = *reinterpret_cast<const uint32_t*>(p);
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t lo = __byte_perm(v[0][w], v[1][w], h ? 0x7632 : 0x5410);
            const uint32_t hi = __byte_perm(v[2][w], v[3][w], h ? 0x7632 : 0x5410);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t ls = lo >> (8 * c), hs = hi >> (8 * c);
              const uint32_t a0 = ls & 0x000F000Fu, a1 = ls & 0x00F000F0u, a2 = hs & 0x000F000Fu, a3 = hs & 0x00F000F0u;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_f16(o[nt][(w * 2 + h) * 2 + c], a0, a1, a2, a3, pb[i][nt][0], pb[i][nt][1]);
            }
          }
      }
      __syncwarp();  // every lane has read the tile
      stage ^= 1;
    }
    // the warps' sums meet
    // (a warp's tiles in flight are in half `stage` of its ring, and the halves change alike or not at all: the others' are told)
    auto meet_of = [&](int w, int free_half) {
      return reinterpret_cast<float*>(smem + (L::kMeetInRing ? (w * kDecStages + free_half) * L::kStage
                                                             : L::kRing + w * R * L::kPitch * 4));
    };
    float* const mine = meet_of(warp, stage ^ 1);
    float* ml = reinterpret_cast<float*>(smem + L::kOffMl);
    int* half_of = reinterpret_cast<int*>(smem + L::kOffHalf);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float ls = i ? l[nt].y : l[nt].x, zs = i ? z[nt].y : z[nt].x;
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          ls += __shfl_xor_sync(0xFFFFFFFFu, ls, d);
          zs += __shfl_xor_sync(0xFFFFFFFFu, zs, d);
        }
        const int r = nt * 8 + 2 * t + i;
        float* dst = mine + r * L::kPitch + g * (2 * MT);
#pragma unroll
        for (int j = 0; j < MT / 2; ++j)
          reinterpret_cast<float4*>(dst)[j] =
              make_float4(fmaf(o[nt][2 * j][i], 16777216.0f, zs), fmaf(o[nt][2 * j][2 + i], 1048576.0f, zs),
                          fmaf(o[nt][2 * j + 1][i], 16777216.0f, zs), fmaf(o[nt][2 * j + 1][2 + i], 1048576.0f, zs));
        if (g == 0) {
          ml[(warp * R + r) * 2] = i ? m[nt].y * unit[nt].y : m[nt].x * unit[nt].x;
          ml[(warp * R + r) * 2 + 1] = ls;
        }
      }
    if (lane == 0) half_of[warp] = stage ^ 1;
    __syncthreads();
    const int rows = min(R, at.seq.n * a.g.G - at.rt * R);
    const bool whole_segment = at.u0 == 0 && at.u1 == at.span.count;
    if (at.u0 == 0 && at.u1 < at.span.count && threadIdx.x == 0) {
      // (the segment reaches the end of this CTA's share, and share tiles a CTA from there on)
      Kv4Join j;
      j.parts = 1 + (at.span.count - at.u1 + share - 1) / share;
      j.slot = is_first ? 0 : 1;
      j.rows = rows;
      j.first_row = at.rt * R;
      j.row0 = at.seq.row0;
      j.h = at.h;
      a.join[blockIdx.x] = j;
    }
    goes_on |= at.u0 == 0 && at.u1 < at.span.count;
    float* part_out = a.partial + (static_cast<size_t>(blockIdx.x) * 2 + (is_first ? 0 : 1)) * kv4_partial_floats(R, HD);
    for (int r = threadIdx.x / HD; r < rows; r += kDecThreads / HD) {
      const int d = threadIdx.x % HD;
      float top = kKv4NoMax, sum = 0.0f, acc = 0.0f;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) top = fmaxf(top, ml[(w * R + r) * 2]);
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) {
        const float by = exp2_approx(ml[(w * R + r) * 2] - top);
        sum = fmaf(by, ml[(w * R + r) * 2 + 1], sum);
        acc = fmaf(by, meet_of(w, half_of[w])[r * L::kPitch + d], acc);
      }
      if (whole_segment) {
        const int at_row = at.rt * R + r, i = a.g.by(at_row), head = at.h * a.g.G + (at_row - i * a.g.G);
        // no token seen: zero (and not 0 / 0); a row that is not finite stays NaN
        const float val = sum == 0.0f ? 0.0f : __fdividef(acc, sum);
        unsigned short bits;
        asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(bits) : "f"(val));
        a.out[(static_cast<int64_t>(at.seq.row0 + i) * a.c.hkv * a.g.G + head) * HD + d] = bits;
      } else {
        part_out[2 * R + r * HD + d] = acc;
        if (d == 0) {
          part_out[2 * r] = top;
          part_out[2 * r + 1] = sum;
        }
      }
    }
    if (!kv4_next_segment<kDecTile>(a.c, a.m, a.g, R, at)) break;
    __syncthreads();
  }
  if (threadIdx.x == 0 && !goes_on) a.join[blockIdx.x].parts = 0;
}

static int g_resident[2][2];  // CTAs per SM of kv4_decode_kernel<64 or 128, 1 or 2>

template <int HD, int NT>
static int init_decode() {
  int n = 0;
  DQ_CHECK_CUDA(cudaFuncSetAttribute(kv4_decode_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     DecSmem<HD, NT>::kBytes));
  DQ_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kv4_decode_kernel<HD, NT>, kDecThreads,
                                                              DecSmem<HD, NT>::kBytes));
  g_resident[HD == 128][NT - 1] = n < 1 ? 1 : n;
  return DQ_OK;
}
int init_kv4_decode_kernels() {
  int rc = init_decode<64, 1>();
  if (rc == DQ_OK) rc = init_decode<64, 2>();
  if (rc == DQ_OK) rc = init_decode<128, 1>();
  if (rc == DQ_OK) rc = init_decode<128, 2>();
  return rc;
}

int kv4_decode_resident(int hd, int R) { return g_resident[hd == 128][R / 8 - 1]; }

template <int HD, int NT>
static int launch_decode(const Kv4AttnArgs& a, int grid, cudaStream_t s) {
  DQ_CHECK_CUDA(launch_pdl(kv4_decode_kernel<HD, NT>, dim3(grid), dim3(kDecThreads), DecSmem<HD, NT>::kBytes, s, a));
  return DQ_OK;
}
int launch_kv4_decode(const Kv4AttnArgs& a, int hd, int R, int grid, cudaStream_t s) {
  if (hd == 128) return R == 8 ? launch_decode<128, 1>(a, grid, s) : launch_decode<128, 2>(a, grid, s);
  return R == 8 ? launch_decode<64, 1>(a, grid, s) : launch_decode<64, 2>(a, grid, s);
}

}  // namespace dq
