// Attention of many query rows per sequence over the paged 4-bit cache (prompts, pieces of prompts) on tcgen05.
//
// A segment has up to 256 query rows, (token, query head) pairs of one key/value head: two tiles of 128 rows against the same
// keys and values, tiles of 128 tokens (ROWS = 128: one row tile, whose warps 4-7 do nothing).  One persistent CTA per SM, sixteen warps:
//   warps 0-3, 4-7   softmax of row tile 0 / 1, a thread per row: scores out of tensor memory, the running maximum and sum,
//                    weights back to tensor memory, at the end the output
//   warps 8-11       codes from the pages to fp16 keys and values (fma(c, scale, zero), one rounding) in shared memory
//   warp 12          issues the products: S = Q K' (both from shared memory), O += P V (P from tensor memory)
//   warps 13-15      queries of the next segment into shared memory as soon as its predecessor's last scores are computed; the
//                    softmax warps make operands of them before they write their outputs
// Softmax goes by halves of a token tile, whose 64 scores a thread holds in registers; their weights are multiplied while the
// other half's are taken.  Tensor memory (512 columns): 128 scores for each row tile (the weights of a half take the first half
// of its scores' columns) and the outputs of both.
//
// Operands are fp16: a key or value of the cache is c * scale + zero with fp16 scale and zero, and 11 bits keep that to 2^-11
// where bf16 would give 2^-8; queries (bf16) are exact in fp16 times a power of two of their row; weights lie in [0, 2^8].
// Keys, values and queries hold the elements of each group of eight in the order 0 4 1 5 2 6 3 7, in which nibbles come out of a
// word two at a time; outputs undo it.  The running maximum m moves only where a row would pass 2^8 above it.
//
// Eight prompts of 2048 tokens, 32 heads of 128 over 8, 275 GFLOP: 409 us replayed from a graph (670 TFLOP/s, 41 % of the rate of
// a plain matrix product), 432 us a call when the inputs change from call to call (640, 39 %).  Neither memory (8 %) nor the
// tensor cores (36 % of their cycles) nor issue slots (51 %) are at their end: what bounds it is the dependent way of a tile,
// score, maximum, weight, product, of which a row tile has one at a time.  Without any arithmetic on the scores the
// same waits and products take 305 us.  The first tile of a segment waits for its queries and the last for its output, 10000
// cycles a segment: the softmax warps therefore convert the next queries before they write outputs.  Scores of a whole tile in
// a thread's registers spilled and left the instruction cache; they are taken by halves, and loops are kept short.
#include "kv4.cuh"

namespace dq {

constexpr int kPreThreads = 512;
constexpr int kPreStages = 2;
constexpr int kPreRaw = 3;        // keys or values of a converting warp's tiles that are on their way
constexpr int kPreLoaders = 3;    // warps that bring the queries

template <int HD>
struct PreSmem {
  static constexpr int kHalf = 128 * 128;              // 128 rows of 64 fp16 elements, 128-byte swizzle
  static constexpr int kOperand = HD / 64 * kHalf;     // one tile of queries, keys or values
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = 2 * kOperand;
  static constexpr int kOffV = kOffK + kPreStages * kOperand;
  static constexpr int kRaw = 32 * (HD / 2 + 4);       // a converting warp's codes and pairs of 32 keys or values
  static constexpr int kOffRaw = kOffV + kPreStages * kOperand;
  static constexpr int kOffBar = kOffRaw + 4 * kPreRaw * kRaw;
  static constexpr int kBars = 6 + 4 * kPreStages + 10;
  static constexpr int kOffValid = kOffBar + kBars * 8;
  static constexpr int kOffMul = kOffValid + 4 * 4;            // [256] what a row's scores have to be multiplied with
  static constexpr int kOffCursor = kOffMul + 256 * 4;
  static constexpr int kOffTmem = kOffCursor + static_cast<int>((sizeof(Kv4Cursor) + 8 + 15) / 16 * 16);
  static constexpr int kBytes = kOffTmem + 16 + 1024;  // (the operands start at a multiple of 1024)
};

// Instruction descriptor, kind::f16: fp16 A and B, fp32 accumulator.  b_rows: B's rows (the sum's index) are contiguous in N.
__host__ __device__ constexpr uint32_t pre_idesc(int m, int n, bool b_rows) {
  return (1u << 4) | (b_rows ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// Shared-memory descriptor of values as B of O += P V: rows are tokens (the sum's index), 64 head elements of a row are 128
// swizzled bytes; eight tokens are 1024 bytes, the next 64 elements kHalf bytes away.
__device__ __forceinline__ uint64_t pre_desc_rows(uint32_t smem_addr, uint32_t next_block) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(next_block >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
__device__ __forceinline__ void pre_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pre_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pre_tmem_st_x16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void pre_cp_async_16(uint32_t dst, const void* src, int bytes = 16) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float pre_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pre_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pre_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// eight codes -> fp16 c * scale + zero, elements 0 4 1 5 2 6 3 7
__device__ __forceinline__ uint4 pre_expand(uint32_t w, __half2 s, __half2 z) {
  const __half2 k1024 = __half2half2(__ushort_as_half(0x6400)), k16th = __half2half2(__ushort_as_half(0x2C00)),
                m64 = __half2half2(__ushort_as_half(0xD400));
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t v = w >> (8 * i);
    const uint32_t lo = (v & 0x000F000Fu) | 0x64006400u, hi = (v & 0x00F000F0u) | 0x64006400u;  // 1024 + c, 1024 + 16 c
    const __half2 c0 = __hsub2(*reinterpret_cast<const __half2*>(&lo), k1024);                   // exact
    const __half2 c1 = __hfma2(*reinterpret_cast<const __half2*>(&hi), k16th, m64);              // exact
    const __half2 x0 = __hfma2(c0, s, z), x1 = __hfma2(c1, s, z);
    r[2 * i] = *reinterpret_cast<const uint32_t*>(&x0);
    r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&x1);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// Groups of 64 tokens of a segment's share of tiles: the last tile's second group may lie behind all that the rows see.
__device__ __forceinline__ int pre_groups(const Kv4Batch& c, const Kv4Cursor& k) {
  const int n = 2 * (k.u1 - k.u0);
  const int hi = min(min(k.span.p_hi + 1, k.seq.kv), c.capacity);
  return k.u1 == k.span.count && hi <= k.span.tile(k.u1 - 1) * kPreTile + 64 ? n - 1 : n;
}

template <int HD, int ROWS>
__global__ void __launch_bounds__(kPreThreads, 1)
kv4_prefill_kernel(const __grid_constant__ Kv4AttnArgs a, int* status) {
  using L = PreSmem<HD>;
  constexpr bool kOne = ROWS == 128;  // segments of one row tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ volatile int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* q_full = bar;                       // [2] a row tile's queries are in shared memory, as operands
  uint64_t* q_empty = bar + 2;                  // [2] its last scores have been computed
  uint64_t* q_raw = bar + 4;                    // [2] they are as they came
  uint64_t* k_full = bar + 6;                   // [stage]
  uint64_t* k_empty = k_full + kPreStages;
  uint64_t* v_full = k_empty + kPreStages;
  uint64_t* v_empty = v_full + kPreStages;
  uint64_t* s_full = v_empty + kPreStages;      // [row tile] scores of a token tile are in tensor memory
  // (Of a row tile by itself, scores of the next token tile follow the first half's weights: a warp may bring a second half while
  // another has yet to bring the one before, and arrivals are counted, not named.  Its second halves therefore take two barriers
  // in turn, 1 and 3; that of the second half but one is through, since there are scores of this token tile.)
  uint64_t* p_full = s_full + 2;                // [row tile][half] weights of 64 tokens are
  uint64_t* o_done = p_full + 4;                // [row tile][half] the values of its weights are in the output
  float* q_mul = reinterpret_cast<float*>(smem + L::kOffMul);
  // pieces of 16 tokens that are there, of the last four tiles: two bits in each of four bytes (warps 8 to 11)
  volatile uint32_t* valid = reinterpret_cast<volatile uint32_t*>(smem + L::kOffValid);
  Kv4Cursor& found = *reinterpret_cast<Kv4Cursor*>(smem + L::kOffCursor);
  int* s_share = reinterpret_cast<int*>(&found + 1);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + L::kOffTmem);
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 128);
      mbar_init(q_raw + i, 32 * kPreLoaders);
      mbar_init(q_empty + i, 1);
      mbar_init(s_full + i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(o_done + i, 1);
      mbar_init(p_full + i, 128);
    }
    for (int i = 0; i < kPreStages; ++i) {
      mbar_init(k_full + i, 128);
      mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 128);
      mbar_init(v_empty + i, 1);
    }
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(s_tmem, 512);
    tmem_relinquish();
    // Behind the allocation: a kernel that came first on this SM could hold tensor memory until this one is done.
    grid_dep_launch_dependents();
  }
  grid_dep_wait();
  if (warp == 0) {
    const Kv4Start k = kv4_begin_any<kPreTile>(a.c, a.m, a.g, ROWS, kPreLeast, a.grid, lane);
    if (lane == 0) {
      if (k.any) found = k.k;
      else a.join[blockIdx.x].parts = 0;
      *s_share = k.any ? k.share : 0;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const int share = *s_share;
  const uint32_t base = smem_u32(smem);
  if (share == 0) {
    if (warp == 12) tmem_dealloc(tmem, 512);
    return;
  }
  Kv4Cursor at = found;
  bool ok = true;  // no wait has run out

  if (warp < 8) {
    // ------------------------------------------------------------------------------------------------ softmax
    const int tile = warp >> 2, row_in = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's lanes, in the upper half of an address
    const uint32_t t_s = tmem + lanes + tile * 128, t_o = tmem + lanes + 256 + tile * HD;
    uint32_t count[2] = {0, 0};  // first and second halves of token tiles so far
    auto second = [&](uint32_t n) { return kOne ? 1 + 2 * (n & 1) : 2 * tile + 1; };  // barrier of second half n, and its phase
    auto second_phase = [&](uint32_t n) { return (kOne ? n >> 1 : n) & 1; };
    int seen = 0;          // token tiles of the call, both row tiles'
    uint32_t q_uses = 0;
    bool is_first = true, goes_on = false, fresh = true, more = true;
    Kv4Cursor next = at;
    float mul = 1.0f, m = kKv4NoMax, unit = 1.0f;
    float2 l2 = make_float2(0.0f, 0.0f);
    bool finite = true;
    // One round: the queries of the next segment, so that its scores are computed meanwhile; the output of this segment; the
    // groups of the next.  (First round: no output.)
    for (;;) {
      float mul_next = 1.0f;
      if (more && ok && (tile == 0 || (!kOne && next.seq.n * a.g.G - next.rt * ROWS > 128))) {
        // A row as fp16 times a power of two that brings its largest element to [2^14, 2^15): HD / 16 lanes a row, in place
        constexpr int kRowLanes = HD / 16, kRowsAtOnce = 32 / kRowLanes;
        const int l = lane % kRowLanes;
        uint8_t* const dst = smem + L::kOffQ + tile * L::kOperand + (l >> 2) * L::kHalf;
        auto place = [&](int row, int c) { return dst + row * 128 + (((((2 * l) & 7) + c) ^ (row & 7)) << 4); };
        float* mul_out = q_mul + tile * 128;
        ok = mbar_wait(q_raw + tile, q_uses++ & 1, &s_abort, 56);
#pragma unroll 1
        for (int row = (warp & 3) * 32 + lane / kRowLanes; row < (warp & 3) * 32 + 32; row += kRowsAtOnce) {
          const uint4 v[2] = {*reinterpret_cast<const uint4*>(place(row, 0)), *reinterpret_cast<const uint4*>(place(row, 1))};
          uint32_t big = 0;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            big = __vmaxu2(big, __vmaxu2(__vmaxu2(v[i].x & 0x7FFF7FFFu, v[i].y & 0x7FFF7FFFu),
                                         __vmaxu2(v[i].z & 0x7FFF7FFFu, v[i].w & 0x7FFF7FFFu)));
          big = max(big & 0xFFFFu, big >> 16);
          // Ordinary rows, largest element in [2^-10, 2^15), are fp16 as they are (what lies below 2^-14 of them is off by 2^-25
          // at most); if one of the warp's rows is not, or the scale is huge, the factors of all of them are looked up.
          const uint32_t small = __ballot_sync(0xFFFFFFFFu, big < 0x3A80u);
          constexpr uint32_t kRowMask = (1u << kRowLanes) - 1u;
          const bool odd = big >= 0x4700u || ((small >> (lane & ~(kRowLanes - 1))) & kRowMask) == kRowMask || fabsf(a.scale2) > 1e12f;
          bool finite_row = true;
          float by = a.scale2 > 0.0f ? 1.0f : a.scale2 < 0.0f ? -1.0f : 0.0f;  // (the maximum is taken of scores times |scale|)
          float mul_row = a.scale2 != 0.0f ? fmaxf(fabsf(a.scale2), 1.2e-38f) : 1.0f;
          if (__any_sync(0xFFFFFFFFu, odd)) {
#pragma unroll
            for (int d = 1; d < kRowLanes; d <<= 1) big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, d));
            finite_row = big < 0x7F80u;  // no infinity and no NaN; rows that are not finite are made zero here
            const Kv4RowScale f = kv4_row_scale(finite_row ? big : 0, a.scale2);
            by = f.up;
            mul_row = f.back;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {  // elements 2j, 2j + 1 and 2j + 4, 2j + 5
              const uint32_t p = finite_row ? x[j] : 0u, q = finite_row ? x[j + 2] : 0u;
              h[2 * j] = pre_half2(__uint_as_float(p << 16) * by, __uint_as_float(q << 16) * by);
              h[2 * j + 1] = pre_half2(__uint_as_float(p & 0xFFFF0000u) * by, __uint_as_float(q & 0xFFFF0000u) * by);
            }
            *reinterpret_cast<uint4*>(place(row, i)) = make_uint4(h[0], h[1], h[2], h[3]);
          }
          if (l == 0) mul_out[row] = finite_row ? mul_row : __int_as_float(0x7FC00000);
        }
        fence_proxy_async_smem();
        mbar_arrive(q_full + tile);
        __syncwarp();
        mul_next = mul_out[row_in];
      }
      if (!fresh) {
        const int rows = at.seq.n * a.g.G - at.rt * ROWS;
        if (tile == 0 || (!kOne && rows > 128)) {
          const int r = at.rt * ROWS + tile * 128 + row_in;
          const bool there = tile * 128 + row_in < rows;
          const int i_tok = there ? a.g.by(r) : 0, head = at.h * a.g.G + (there ? r - i_tok * a.g.G : 0);
          const int64_t out_at = (static_cast<int64_t>(at.seq.row0 + i_tok) * a.c.hkv * a.g.G + head) * HD;
          // output of the row
          const float l = l2.x + l2.y;
          const int last_half = (pre_groups(a.c, at) - 1) & 1;
          ok = ok && mbar_wait(o_done + (last_half ? second(count[1] - 1) : 2 * tile),
                               last_half ? second_phase(count[1] - 1) : (count[0] - 1) & 1, &s_abort, 44);
          tc_fence_after();
          const bool whole_segment = at.u0 == 0 && at.u1 == at.span.count;
          // a row that sees no token is zero (and not 0 / 0), one that is not finite NaN
          float by = whole_segment ? (l == 0.0f ? 0.0f : __fdividef(1.0f, l)) : 1.0f;
          if (!finite && l != 0.0f) by = __int_as_float(0x7FC00000);
          float* part = a.partial + (static_cast<size_t>(blockIdx.x) * 2 + (is_first ? 0 : 1)) * kv4_partial_floats(ROWS, HD);
          float* part_o = part + 2 * ROWS + (tile * 128 + row_in) * HD;
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tmem_ld_x32(t_o + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int g = 0; g < 32; g += 8) {  // elements into their own order
              float v[8];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                v[e] = __uint_as_float(o[g + 2 * e]) * by;
                v[e + 4] = __uint_as_float(o[g + 2 * e + 1]) * by;
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) o[g + e] = __float_as_uint(l == 0.0f ? 0.0f : v[e]);
            }
            if (whole_segment) {
              // four lanes exchange their 64 bytes so that they store one row together, then the next
              uint4 x[4];
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const float* v = reinterpret_cast<const float*>(o + 8 * g);
                x[g] = make_uint4(pre_bf16x2(v[0], v[1]), pre_bf16x2(v[2], v[3]), pre_bf16x2(v[4], v[5]), pre_bf16x2(v[6], v[7]));
              }
#pragma unroll
              for (int d = 1; d < 4; d <<= 1) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                  if (g & d) continue;
                  const bool up = lane & d;  // gives x[g], keeps x[g + d]
                  const uint4 give = up ? x[g] : x[g + d];
                  const uint4 take = make_uint4(__shfl_xor_sync(0xFFFFFFFFu, give.x, d), __shfl_xor_sync(0xFFFFFFFFu, give.y, d),
                                                __shfl_xor_sync(0xFFFFFFFFu, give.z, d), __shfl_xor_sync(0xFFFFFFFFu, give.w, d));
                  if (up) x[g] = take;
                  else x[g + d] = take;
                }
              }
#pragma unroll
              for (int g = 0; g < 4; ++g) {  // 16 bytes lane % 4 of the row of lane (lane & ~3) + g
                const long long row_at = __shfl_sync(0xFFFFFFFFu, there ? static_cast<long long>(out_at) : -1ll, (lane & ~3) + g);
                if (row_at >= 0 && ok) *reinterpret_cast<uint4*>(a.out + row_at + c + 8 * (lane & 3)) = x[g];
              }
            } else if (there && ok) {
#pragma unroll
              for (int g = 0; g < 32; g += 4)
                *reinterpret_cast<uint4*>(part_o + c + g) = make_uint4(o[g], o[g + 1], o[g + 2], o[g + 3]);
            }
          }
          if (!whole_segment && there) {
            part[2 * (tile * 128 + row_in)] = m * unit;
            part[2 * (tile * 128 + row_in) + 1] = l;
          }
          tc_fence_before();  // (the next segment's products over O come behind this row's next arrival)
        }
        seen += at.u1 - at.u0;
        const bool begins = at.u0 == 0 && at.u1 < at.span.count;
        if (begins && threadIdx.x == 0) {
          Kv4Join j;
          j.parts = 1 + (at.span.count - at.u1 + share - 1) / share;
          j.slot = is_first ? 0 : 1;
          j.rows = min(rows, ROWS);
          j.first_row = at.rt * ROWS;
          j.row0 = at.seq.row0;
          j.h = at.h;
          a.join[blockIdx.x] = j;
        }
        goes_on |= begins;
        is_first = false;
      }
      if (!more || !ok) break;
      at = next;
      fresh = false;
      const int rows = at.seq.n * a.g.G - at.rt * ROWS;
      if (tile == 0 || (!kOne && rows > 128)) {
        const int n_groups = pre_groups(a.c, at);
        const bool there = tile * 128 + row_in < rows;
        const int i_tok = there ? a.g.by(at.rt * ROWS + tile * 128 + row_in) : 0;
        const int kv = min(at.seq.kv, a.c.capacity);
        const int p_row = at.seq.kv - at.seq.n + i_tok;
        const int hi = there ? min(p_row + 1, kv) : 0;                   // tokens lo ... hi - 1 and those below `first`
        const int lo = a.m.window > 0 ? p_row - a.m.window + 1 : 0;
        const int first = a.m.window > 0 ? min(a.m.sinks, hi) : 0;
        m = kKv4NoMax;
        l2 = make_float2(0.0f, 0.0f);
        finite = !isnan(mul_next);
        mul = finite ? mul_next : 1.0f;
        unit = 1.0f;
        // groups from these tokens on are seen whole by every row
        const int whole_hi = min(kv, at.span.p_lo + 1) - 64, whole_lo = a.m.window > 0 ? at.span.p_hi - a.m.window : -1,
                  whole_sinks = a.m.window > 0 ? a.m.sinks - 64 : -1;
        for (int j = 0; j < n_groups && ok; ++j) {
          const int tok = at.span.tile(at.u0 + (j >> 1)) * kPreTile + 64 * (j & 1);
          const int half = j & 1;
          const uint32_t t_b = t_s + ((kOne ? (j << 6) & 128 : 0) | (half << 6));
          if (half == 0) {
            ok = mbar_wait(s_full + tile, count[0]++ & 1, &s_abort, 42);
            tc_fence_after();
          } else {
            ++count[1];
          }
          const uint32_t got = (valid[(seen + (j >> 1)) & 3] >> (16 * (j & 1))) & 0xFFFFu;
          const bool whole = got == 0x0303u && tok <= whole_hi && (tok > whole_lo || tok <= whole_sinks);
          auto below = [](int n) { return n >= 32 ? 0xFFFFFFFFu : (1u << max(n, 0)) - 1u; };
          uint32_t s[64];
          tmem_ld_x32(t_b, s);
          tmem_ld_x32(t_b + 32, s + 32);
          tmem_ld_wait();
          if (!whole) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int t0 = tok + 32 * h;
              const uint32_t pieces = got >> (8 * h);
              const uint32_t see = below(hi - t0) & (~below(lo - t0) | below(first - t0)) &
                                   ((pieces & 1u ? 0xFFFFu : 0u) | (pieces & 2u ? 0xFFFF0000u : 0u));
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((see >> e) & 1u)) s[32 * h + e] = 0xFF800000u;
            }
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 64; e += 8)
#pragma unroll
            for (int f = 0; f < 4; ++f) top[f] = max3(top[f], __uint_as_float(s[e + f]), __uint_as_float(s[e + f + 4]));
          const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * mul;
          if (__any_sync(0xFFFFFFFFu, high > m + 8.0f)) {
            const float to = fmaxf(m, high), by = pre_exp2(m - to);
            m = to;
            kv4_units(m, mul, unit);
            l2 = make_float2(l2.x * by, l2.y * by);
            if (j > 0) {
              // the groups before are in O: of two row tiles those of earlier tiles are since there are scores of this one
              if (half == 1 || kOne)
                ok = ok && mbar_wait(o_done + (half == 1 ? 2 * tile : second(count[1] - 1)),
                                     half == 1 ? (count[0] - 1) & 1 : second_phase(count[1] - 1), &s_abort, 43);
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < HD; c += 16) {
                uint32_t o[16];
                tmem_ld_x16(t_o + c, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * by);
                pre_tmem_st_x16(t_o + c, o);
              }
            }
          }
          const float2 mul2 = make_float2(mul, mul), low = make_float2(-m, -m);
          // 64 scores into 32 columns of weights, over the scores.  Sixteen at a time; sums and stores are a batch behind, or they
          // would wait for every exponential: 662 cycles for 64 scores of a warp by itself, 1097 with sums in the order of the
          // scores.
          float2 w[2][8];
          uint32_t p[16];
#pragma unroll
          for (int b = 0; b < 5; ++b) {
            if (b < 4) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float2 x = __ffma2_rn(
                    make_float2(__uint_as_float(s[16 * b + 2 * e]), __uint_as_float(s[16 * b + 2 * e + 1])), mul2, low);
                w[b & 1][e] = make_float2(pre_exp2(x.x), pre_exp2(x.y));
              }
            }
            if (b > 0) {
              const float2(&v)[8] = w[(b - 1) & 1];
#pragma unroll
              for (int e = 0; e < 8; ++e) p[8 * ((b - 1) & 1) + e] = pre_half2(v[e].x, v[e].y);
              l2 = __fadd2_rn(l2, __fadd2_rn(__fadd2_rn(__fadd2_rn(v[0], v[1]), __fadd2_rn(v[2], v[3])),
                                             __fadd2_rn(__fadd2_rn(v[4], v[5]), __fadd2_rn(v[6], v[7]))));
              if (((b - 1) & 1) == 1) pre_tmem_st_x16(t_b + 8 * (b - 2), p);
            }
          }
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(p_full + (half == 0 ? 2 * tile : second(count[1] - 1)));
        }
      }
      more = kv4_next_segment<kPreTile>(a.c, a.m, a.g, ROWS, next);
    }
    if (threadIdx.x == 0 && !goes_on) a.join[blockIdx.x].parts = 0;
  } else if (warp < 12) {
    // ------------------------------------------------------------------------------------------------ keys and values
    constexpr int kLanes = HD / 32;           // lanes with 16 bytes of codes each to a token
    constexpr int kStep = 32 / kLanes;        // tokens of a warp per load
    constexpr int kLoads = 32 / kStep;        // loads for the warp's 32 tokens
    const int w = warp - 8, q = lane % kLanes, in = lane / kLanes;
    const int P = 1 << a.c.page_shift;
    // The tile that is copied next (`got`: this warp's two pieces of 16 tokens that are there, `left`: tokens of the tile from
    // this warp's first one on), and the page numbers of the one behind it, which are on their way.
    bool more = true, coming = true;
    int u = at.u0, h_next = 0, tok_next = 0, left_next = 0;
    uint32_t page_next[2];
    uint32_t got = 0;
    const uint8_t* block[2];
    int slot[2], left = 0;
    auto look_up = [&]() {
      while (coming && u >= at.u1) {
        coming = kv4_next_segment<kPreTile>(a.c, a.m, a.g, ROWS, at);
        u = at.u0;
      }
      if (!coming) return;
      tok_next = at.span.tile(u) * kPreTile + w * 32;
      left_next = min(at.seq.kv, a.c.capacity) - tok_next;
      h_next = at.h;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        page_next[i] = 0xFFFFFFFFu;
        if (16 * i < left_next)
          page_next[i] = static_cast<uint32_t>(a.c.table[at.b * a.c.table_stride + ((tok_next + 16 * i) >> a.c.page_shift)]);
      }
      ++u;
    };
    auto seek = [&]() {
      more = coming;
      if (!more) return;
      got = 0;
      left = left_next;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool is = page_next[i] < static_cast<uint32_t>(a.c.num_pages);
        got |= is ? 1u << i : 0u;
        block[i] = a.c.pages + static_cast<uint64_t>(is ? page_next[i] : 0u) * static_cast<uint32_t>(a.c.page_stride) +
                   static_cast<int64_t>(h_next) * P * (HD + 8);
        slot[i] = (tok_next + 16 * i) & (P - 1);
      }
      look_up();
    };
    // codes [32][HD / 2] and pairs [32] of the warp's tokens; pieces that are not there are left as they are in shared memory
    uint8_t* const raw = smem + L::kOffRaw + w * kPreRaw * L::kRaw;
    auto copy = [&](bool values, int place) {
      if (more) {
        const uint32_t dst = smem_u32(raw) + place * L::kRaw;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if ((got >> i) & 1u) {
            const uint8_t* src = block[i] + (values ? P * (HD / 2) : 0) + slot[i] * (HD / 2) + lane * 16;
#pragma unroll
            for (int e = 0; e < HD / 64; ++e) pre_cp_async_16(dst + i * 16 * (HD / 2) + e * 512 + lane * 16, src + e * 512);
            if (lane < 4)
              pre_cp_async_16(dst + 32 * (HD / 2) + i * 64 + lane * 16,
                              block[i] + P * HD + (values ? 4 * P : 0) + slot[i] * 4 + lane * 16);
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // The lane's place in an operand: token w * 32 + in, its four 16-byte columns.  Lanes of the second 64 elements take their
    // words in the order 2 3 0 1: the eight lanes that store together hit eight different columns.
    const int turned = q & 2;
    const uint32_t to_lane = (q >> 1) * L::kHalf + (w * 32 + in) * 128;
    uint32_t column[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) column[e] = ((((q & 1) << 2) + (e ^ turned)) ^ (in & 7)) << 4;
    // keys of tile 0, values of tile 0, keys of tile 1 ...: one is converted while the next ones are on the way
    static_assert(kPreRaw == 3, "keys of the next tile are asked for before this one is converted");
    look_up();
    seek();
    copy(false, 0);
    copy(true, 1);
    uint32_t got_now = got;
    int left_now = left, place = 0;
    seek();
    copy(false, 2);
    bool values = false, last = false;
    for (uint32_t n = 0; ok && !last;) {
      const int stage = n % kPreStages;
      asm volatile("cp.async.wait_group %0;" ::"n"(kPreRaw - 1) : "memory");
      __syncwarp();
      ok = mbar_wait((values ? v_empty : k_empty) + stage, ((n / kPreStages) & 1) ^ 1, &s_abort, 45);
      // (slot n % 4 was last read for tile n - 4: the products of tile n - 2, which are done, waited for that)
      if (!values && lane == 0)
        reinterpret_cast<volatile uint8_t*>(smem + L::kOffValid)[(n & 3) * 4 + w] = static_cast<uint8_t>(got_now);
      uint8_t* const from = raw + place * L::kRaw;
      // tokens that are not there become zeros: their weights are zero, and zero times what a slot may hold is not
      if (left_now < 32 || got_now != 3u) {
        if (lane >= left_now || !((got_now >> (lane >> 4)) & 1u)) reinterpret_cast<uint32_t*>(from + 32 * (HD / 2))[lane] = 0;
        __syncwarp();
      }
      const uint8_t *src = from + in * (HD / 2) + q * 16, *pairs = from + 32 * (HD / 2) + in * 4;
      uint8_t* const to = smem + (values ? L::kOffV : L::kOffK) + stage * L::kOperand + to_lane;
      // Beside one row tile these warps are what a tile waits for, and all loads come first, which the compiler cannot move over
      // stores; beside two row tiles that took their softmax's issue slots (409 to 411 us).
      constexpr int kAtOnce = kOne ? kLoads : 1;
#pragma unroll
      for (int i0 = 0; i0 < kLoads; i0 += kAtOnce) {
        uint2 c01[kAtOnce], c23[kAtOnce];
        __half2 pair[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          c01[i] = *reinterpret_cast<const uint2*>(src + (i0 + i) * kStep * (HD / 2) + 4 * turned);
          c23[i] = *reinterpret_cast<const uint2*>(src + (i0 + i) * kStep * (HD / 2) + (8 - 4 * turned));
          pair[i] = *reinterpret_cast<const __half2*>(pairs + (i0 + i) * kStep * 4);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          const __half2 sc = __low2half2(pair[i]), ze = __high2half2(pair[i]);
          const uint32_t c[4] = {c01[i].x, c01[i].y, c23[i].x, c23[i].y};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint4*>(to + column[e] + (i0 + i) * kStep * 128) = pre_expand(c[e], sc, ze);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive((values ? v_full : k_full) + stage);
      __syncwarp();  // every lane has read the codes
      if (values) {  // the tile behind this one is next, and the one behind that is asked for
        last = !more;
        got_now = got;
        left_now = left;
        ++n;
        seek();
      }
      copy(!values, place);
      place = place == kPreRaw - 1 ? 0 : place + 1;
      values = !values;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (warp == 12) {
    // ------------------------------------------------------------------------------------------------ products
    if (elect_one()) {
      constexpr uint32_t kIdescS = pre_idesc(128, 128, false), kIdescO = pre_idesc(128, HD, true);
      uint32_t q_phase[2] = {0, 0}, p_phase[2][2] = {{0, 0}, {0, 0}}, n = 0;  // n: token tiles so far
      auto scores = [&](int t, int at_s, uint32_t tile_number, bool last) {
        const uint32_t qa = base + L::kOffQ + t * L::kOperand, ka = base + L::kOffK + tile_number % kPreStages * L::kOperand;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          pre_mma_ss(tmem + at_s * 128, umma_desc_k_sw128(qa + (k >> 2) * L::kHalf + (k & 3) * 32),
                     umma_desc_k_sw128(ka + (k >> 2) * L::kHalf + (k & 3) * 32), kIdescS, k > 0);
        umma_commit(s_full + t);
        if (last) umma_commit(q_empty + t);
      };
      auto values = [&](int t, int at_s, uint32_t tile_number, int half, bool add) {
        const uint32_t va = base + L::kOffV + tile_number % kPreStages * L::kOperand + half * 8192;
        const uint32_t nth = p_phase[t][half]++;
        const bool turns = kOne && half == 1;
        const int bar_at = turns ? 1 + 2 * (nth & 1) : 2 * t + half;
        ok = ok && mbar_wait(p_full + bar_at, (turns ? nth >> 1 : nth) & 1, &s_abort, 51);
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k)
          pre_mma_ts(tmem + 256 + t * HD, tmem + at_s * 128 + half * 64 + k * 8, pre_desc_rows(va + k * 2048, L::kHalf), kIdescO,
                     add || k > 0);
        umma_commit(o_done + bar_at);
      };
      // Of two row tiles, a tile's next scores follow its weights' second half: products run in order, so those weights have been
      // read.  A row tile by itself has the other's scores' columns for every second token tile; its next scores follow its
      // weights' first half, whose arrival says that every row is through with the tile before, whose columns they take.
      for (;;) {
        const int rows = at.seq.n * a.g.G - at.rt * ROWS, groups = pre_groups(a.c, at), tiles = (groups + 1) / 2;
        const bool two = !kOne && rows > 128;
        ok = ok && mbar_wait(k_full + n % kPreStages, (n / kPreStages) & 1, &s_abort, 49);
        ok = ok && mbar_wait(q_full, q_phase[0]++ & 1, &s_abort, 47);
        if (!ok) break;
        tc_fence_after();
        scores(0, 0, n, tiles == 1);
        if (two) {
          ok = mbar_wait(q_full + 1, q_phase[1]++ & 1, &s_abort, 48);
          if (!ok) break;
          tc_fence_after();
          scores(1, 1, n, tiles == 1);
        }
        umma_commit(k_empty + n % kPreStages);
#pragma unroll 1
        for (int j = 0; j < tiles && ok; ++j, ++n) {
          const bool more = j + 1 < tiles, both = 2 * j + 1 < groups;
          ok = mbar_wait(v_full + n % kPreStages, (n / kPreStages) & 1, &s_abort, 50);
          if constexpr (!kOne) {
            values(0, 0, n, 0, j > 0);
            if (both) values(0, 0, n, 1, true);
            if (more) {
              ok = ok && mbar_wait(k_full + (n + 1) % kPreStages, ((n + 1) / kPreStages) & 1, &s_abort, 52);
              if (!ok) break;
              tc_fence_after();
              scores(0, 0, n + 1, j + 2 == tiles);
            }
            if (two) {
              values(1, 1, n, 0, j > 0);
              if (both) values(1, 1, n, 1, true);
              if (!ok) break;
              if (more) scores(1, 1, n + 1, j + 2 == tiles);
            }
          } else {
            values(0, j & 1, n, 0, j > 0);
            if (more) {
              ok = ok && mbar_wait(k_full + (n + 1) % kPreStages, ((n + 1) / kPreStages) & 1, &s_abort, 53);
              if (!ok) break;
              tc_fence_after();
              scores(0, (j & 1) ^ 1, n + 1, j + 2 == tiles);
            }
            if (both) values(0, j & 1, n, 1, true);
          }
          if (!ok) break;
          umma_commit(v_empty + n % kPreStages);
          if (more) umma_commit(k_empty + (n + 1) % kPreStages);
        }
        if (!ok || !kv4_next_segment<kPreTile>(a.c, a.m, a.g, ROWS, at)) break;
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------------------------------------ queries
    // All rows of a tile at once; the softmax warps make operands of them.
    constexpr int kRowLanes = HD / 16, kRowsAtOnce = 32 / kRowLanes, kStep = kPreLoaders * kRowsAtOnce;
    const int w = warp - 13, l = lane % kRowLanes, row0 = w * kRowsAtOnce + lane / kRowLanes;
    uint32_t uses[2] = {0, 0};
    for (;;) {
      const int rows = at.seq.n * a.g.G - at.rt * ROWS;
#pragma unroll 1
      for (int tile = 0; tile < (!kOne && rows > 128 ? 2 : 1); ++tile) {
        const uint32_t use = uses[tile]++;
        ok = ok && mbar_wait(q_empty + tile, (use & 1) ^ 1, &s_abort, 55);
        // 16-byte columns 2l and 2l + 1 of a row
        uint8_t* const dst = smem + L::kOffQ + tile * L::kOperand + (l >> 2) * L::kHalf;
        auto place = [&](int row, int c) { return dst + row * 128 + (((((2 * l) & 7) + c) ^ (row & 7)) << 4); };
#pragma unroll 1
        for (int row = row0; row < 128; row += kStep) {
          const bool there = tile * 128 + row < rows;
          const int r = at.rt * ROWS + tile * 128 + row, i_tok = there ? a.g.by(r) : 0;
          const int head = at.h * a.g.G + (there ? r - i_tok * a.g.G : 0);
          const unsigned short* src =
              a.q + static_cast<int64_t>(at.seq.row0 + i_tok) * a.q_row + static_cast<int64_t>(head) * a.q_head + 16 * l;
          pre_cp_async_16(smem_u32(place(row, 0)), src, there ? 16 : 0);
          pre_cp_async_16(smem_u32(place(row, 1)), src + 8, there ? 16 : 0);
        }
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
        mbar_arrive(q_raw + tile);
      }
      if (!ok || !kv4_next_segment<kPreTile>(a.c, a.m, a.g, ROWS, at)) break;
    }
  }
  // every product has been waited for by the softmax of its row tile (or a wait ran out)
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && s_abort != 0) atomicExch(status, s_abort);
}

template <int HD, int ROWS>
static int init_prefill() {
  DQ_CHECK_CUDA(cudaFuncSetAttribute(kv4_prefill_kernel<HD, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, PreSmem<HD>::kBytes));
  return DQ_OK;
}
int init_kv4_prefill_kernels() {
  int rc = init_prefill<64, 128>();
  if (rc == DQ_OK) rc = init_prefill<64, 256>();
  if (rc == DQ_OK) rc = init_prefill<128, 128>();
  if (rc == DQ_OK) rc = init_prefill<128, 256>();
  return rc;
}
template <int HD, int ROWS>
static int launch_prefill(const Kv4AttnArgs& a, int grid, cudaStream_t s, DeviceState* st) {
  DQ_CHECK_CUDA(launch_pdl(kv4_prefill_kernel<HD, ROWS>, dim3(grid), dim3(kPreThreads), PreSmem<HD>::kBytes, s, a, st->status_dev));
  return DQ_OK;
}
int launch_kv4_prefill(const Kv4AttnArgs& a, int hd, int R, int grid, cudaStream_t s, DeviceState* st) {
  if (hd == 128) return R == 128 ? launch_prefill<128, 128>(a, grid, s, st) : launch_prefill<128, 256>(a, grid, s, st);
  return R == 128 ? launch_prefill<64, 128>(a, grid, s, st) : launch_prefill<64, 256>(a, grid, s, st);
}

}  // namespace dq
