// Attention of a few query rows per sequence over the paged 4-bit cache (decode steps, drafted tokens), and the kernel that
// joins the sums of segments which several CTAs share.
//
//   o = sum_j p_j (s_j c_j + z_j) / sum_j p_j,   p_j = 2^(x_j - m),   x_j = scale log2(e) q . (s'_j c'_j + z'_j)
// with the scales outside of the matrix products:
//   q . (s c + z) = s (q . c) + z (q . 1),   sum_j p_j (s_j c_j + z_j) = sum_j (p_j s_j) c_j + sum_j p_j z_j
// so that the products run on the bare codes.  A 4-bit code in the low bits of an fp16 word IS an fp16 number, the subnormal
// c * 2^-24 (in bits 4 to 7: c * 2^-20): an AND makes two operands of mma.sync.m16n8k16, with no conversion, and the powers
// of two go into the scores' scale, into every other query element, and into the last factor of the output.  A code costs
// 0.6 (keys) and 0.75 (values) instructions.
//
// Both products are taken transposed, keys or head elements along the 16 rows and up to eight query rows along the columns
// (S' = K Q', O' = V' P'), which wastes nothing on groups of up to eight query rows.  movmatrix turns the weights of S' into
// the operand of O'.  Query elements are permuted to the order in which nibbles come out of a 16-byte load.
//
// Each warp has a ring of its own of tiles of 32 tokens in shared memory, filled by bulk copies from the pages (four per
// page), and takes every fourth tile of its CTA's share; the warps meet once per segment.  Weights and sums:
//   * p_j s_j is fp16 (an mma operand, 2^-11 relative, in the row's own scale): the reference point m is taken of
//     x_j + exponent(s_j), so that p_j s_j stays below 2^9 and what counts stays normal whatever the scales are;
//   * m moves only where a row would pass 2^8 above it; l, sum p z and O are fp32.
// Query rows are fp16 times a power of two of the tile: exact where a row is within 2^13 of the tile's largest value.
#include "kv4.cuh"

namespace dq {

constexpr int kDecTile = 32;     // tokens per tile
constexpr int kDecWarps = 4;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kDecStages = 3;    // tiles in flight per warp
constexpr int kDecLeast = 4;     // tiles that a CTA takes at least
constexpr float kNoMax = -1e30f;

template <int HD, int NT>
struct DecSmem {
  static constexpr int R = 8 * NT;
  static constexpr int kStage = kDecTile * (HD + 8);
  static constexpr int kPitch = HD + 8;  // floats per row of a warp's output in the meeting place
  static constexpr int kOffMeet = kDecWarps * kDecStages * kStage;
  static constexpr int kOffMl = kOffMeet + kDecWarps * R * kPitch * 4;
  static constexpr int kOffScan = kOffMl + kDecWarps * R * 2 * 4;
  static constexpr int kOffBar = kOffScan + (kDecThreads + 1) * 8;
  static constexpr int kOffValid = kOffBar + kDecWarps * kDecStages * 8;
  static constexpr int kBytes = kOffValid + kDecWarps * kDecStages * 4;
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
__device__ __forceinline__ float bf16_float(uint32_t bits) { return __uint_as_float(bits << 16); }

// The query rows of a segment as the second operand of S' = K Q'.
template <int HD, int NT>
struct DecQuery {
  static constexpr int KS = HD / 16;  // steps of 16 head elements
  uint32_t f[NT][KS][2];
  float zq[NT][2];   // sum of the row's elements, times scale log2(e); NaN for a row that is not finite
  int pos[NT][2];    // the row's position; -1: no such row
  float mul;         // what S' has to be multiplied with to be scores in base 2

  __device__ __forceinline__ void load(const Kv4AttnArgs& a, const Kv4Cursor& k, int lane) {
    constexpr int R = 8 * NT, W = HD / 32;  // W: 32-bit words of codes per lane
    const int g = lane >> 2, t = lane & 3, rows = k.seq.n * a.G;
    float q[NT][W * 8];
    float top = 0.0f, sum[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = k.rt * R + nt * 8 + g;
      const bool there = r < rows;
      const int i = there ? r / a.G : 0, head = k.h * a.G + (there ? r - i * a.G : 0);
      const unsigned short* src =
          a.q + static_cast<int64_t>(k.seq.row0 + i) * a.q_row + static_cast<int64_t>(head) * a.q_head + t * (W * 8);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (there) v = *reinterpret_cast<const uint4*>(src + 8 * w);
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          q[nt][8 * w + 2 * j] = __uint_as_float(u[j] << 16);
          q[nt][8 * w + 2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
        }
      }
      float s = 0.0f, big = 0.0f;
#pragma unroll
      for (int j = 0; j < W * 8; ++j) {
        s += q[nt][j];
        big = fmaxf(big, fabsf(q[nt][j]));
      }
      s += __shfl_xor_sync(0xFFFFFFFFu, s, 1);
      s += __shfl_xor_sync(0xFFFFFFFFu, s, 2);
      big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
      const bool fine = isfinite(s) && isfinite(big);
      sum[nt] = fine ? s * a.scale2 : __int_as_float(0x7FC00000);
      if (fine) {
        top = fmaxf(top, big);
      } else {
#pragma unroll
        for (int j = 0; j < W * 8; ++j) q[nt][j] = 0.0f;
      }
    }
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    const int e = top > 0.0f ? static_cast<int>((__float_as_uint(top) >> 23) & 255u) - 127 : 0;
    const int up = max(min(14 - e, 100), -103);  // largest element into [2^14, 2^15)
    const float by = __int_as_float((up + 127) << 23);
    mul = a.scale2 * __int_as_float((127 + 24 - up) << 23);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float* x = &q[nt][8 * w + 2 * u];
          f[nt][2 * w + u][0] = half2_bits(x[0] * by, x[4] * by);
          f[nt][2 * w + u][1] = half2_bits(x[1] * by * 0.0625f, x[5] * by * 0.0625f);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        zq[nt][i] = __shfl_sync(0xFFFFFFFFu, sum[nt], (2 * t + i) * 4);
        const int r = k.rt * R + nt * 8 + 2 * t + i;
        pos[nt][i] = r < rows ? k.seq.kv - k.seq.n + r / a.G : -1;
      }
    }
  }
};

template <int HD, int NT>
__global__ void __launch_bounds__(kDecThreads)
kv4_decode_kernel(const Kv4AttnArgs a, int* status) {
  grid_dep_launch_dependents();
  extern __shared__ __align__(128) uint8_t smem[];
  using L = DecSmem<HD, NT>;
  constexpr int R = L::R, MT = HD / 16, W = HD / 32;
  __shared__ volatile int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * kDecStages * L::kStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar) + warp * kDecStages;
  uint32_t* valid = reinterpret_cast<uint32_t*>(smem + L::kOffValid) + warp * kDecStages;
  long long* scan = reinterpret_cast<long long*>(smem + L::kOffScan);
  if (threadIdx.x == 0) s_abort = 0;
  if (lane == 0) {
    for (int i = 0; i < kDecStages; ++i) mbar_init(bars + i, 1);
    fence_mbar_init();
  }
  grid_dep_wait();
  const Kv4Share sh = kv4_share<kDecTile, kDecThreads>(a.c, a.m, a.G, R, kDecLeast, scan);
  const long long begin = blockIdx.x * sh.share;
  if (begin >= sh.total) return;
  Kv4Cursor at;
  kv4_locate<kDecTile, kDecThreads>(a.c, a.m, a.G, R, begin, min(sh.share, sh.total - begin), scan, at);
  Kv4Cursor ahead = at;  // where the copies are
  const int P = 1 << a.c.page_shift;
  const int step = min(P, kDecTile), pieces = kDecTile / step;
  const uint64_t policy = l2_policy_evict_first();

  // Lane l copies part l % 4 (key codes, value codes, key pairs, value pairs) of page piece l / 4 of a tile.
  const int piece = lane >> 2, part = lane & 3;
  const int part_src = part == 0 ? 0 : part == 1 ? P * (HD / 2) : part == 2 ? P * HD : P * HD + 4 * P;
  const int part_dst = part == 0 ? 0 : part == 1 ? kDecTile * (HD / 2) : part == 2 ? kDecTile * HD : kDecTile * (HD + 4);
  const int per_token = part < 2 ? HD / 2 : 4;
  bool more = true;
  int next_u = ahead.u0 + warp, next_page = -1, next_slot = 0;
  // the warp's next tile, and its page
  auto seek = [&]() {
    while (more && next_u >= ahead.u1) {
      more = kv4_next_segment<kDecTile>(a.c, a.m, a.G, R, ahead);
      next_u = ahead.u0 + warp;
    }
    next_page = -1;
    if (more && piece < pieces) {
      const int tok = ahead.span.tile(next_u) * kDecTile + piece * step;
      next_slot = tok & (P - 1);
      if (tok < min(ahead.seq.kv, a.c.capacity)) next_page = a.c.table[ahead.b * a.c.table_stride + (tok >> a.c.page_shift)];
    }
  };
  auto fetch = [&](int stage) {
    if (!more) return;
    const bool ok = next_page >= 0 && next_page < a.c.num_pages;
    const uint32_t got = __ballot_sync(0xFFFFFFFFu, ok) & 0x11111111u;  // one bit per piece
    if (lane == 0) {
      valid[stage] = got;
      mbar_expect_tx(bars + stage, __popc(got) * step * (HD + 8));
    }
    __syncwarp();
    if (ok) {
      const uint8_t* src = a.c.pages + next_page * a.c.page_stride + static_cast<int64_t>(ahead.h) * P * (HD + 8) + part_src +
                           next_slot * per_token;
      bulk_load_1d(ring + stage * L::kStage + part_dst + piece * step * per_token, src, step * per_token, bars + stage, policy);
    }
    next_u += kDecWarps;
    seek();
  };
  seek();
  for (int i = 0; i < kDecStages; ++i) fetch(i);

  int stage = 0;
  uint32_t parity = 0;
  const uint32_t all_pieces = pieces == 1 ? 0x1u : 0x11u;
  const int first_b = at.b, first_h = at.h, first_rt = at.rt;
  for (;;) {
    DecQuery<HD, NT> q;
    q.load(a, at, lane);
    float o[NT][MT][4], m[NT][2], l[NT][2], z[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < MT; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[nt][i] = kNoMax;
        l[nt][i] = z[nt][i] = 0.0f;
      }
    }
    const int kv = min(at.seq.kv, a.c.capacity);
    for (int u = at.u0 + warp; u < at.u1; u += kDecWarps) {
      const uint8_t* buf = ring + stage * L::kStage;
      const int base = at.span.tile(u) * kDecTile;
      mbar_wait(bars + stage, parity, &s_abort, 41);
      const uint32_t got = valid[stage];
      // every row sees every token of the tile?
      const bool whole = got == all_pieces && base + kDecTile <= kv && base + kDecTile <= at.span.p_lo + 1 &&
                         (a.m.window == 0 || base > at.span.p_hi - a.m.window || base + kDecTile <= a.m.sinks);
      const __half2* kpar = reinterpret_cast<const __half2*>(buf + kDecTile * HD);
      const __half2* vpar = kpar + kDecTile;
#pragma unroll
      for (int half = 0; half < kDecTile / 16; ++half) {
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
        // S' = K Q': rows g and g + 8 are tokens
        {
          uint32_t ka[W], kb[W];
          const uint8_t* row = buf + (half * 16 + g) * (HD / 2) + t * (HD / 8);
          if constexpr (W == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(row), y = *reinterpret_cast<const uint4*>(row + 8 * (HD / 2));
            ka[0] = x.x, ka[1] = x.y, ka[2] = x.z, ka[3] = x.w;
            kb[0] = y.x, kb[1] = y.y, kb[2] = y.z, kb[3] = y.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(row), y = *reinterpret_cast<const uint2*>(row + 8 * (HD / 2));
            ka[0] = x.x, ka[1] = x.y;
            kb[0] = y.x, kb[1] = y.y;
          }
#pragma unroll
          for (int w = 0; w < W; ++w)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              const uint32_t xa = ka[w] >> (8 * v), xb = kb[w] >> (8 * v);
              const uint32_t a0 = xa & 0x000F000Fu, a1 = xb & 0x000F000Fu, a2 = xa & 0x00F000F0u, a3 = xb & 0x00F000F0u;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt], a0, a1, a2, a3, q.f[nt][2 * w + v][0], q.f[nt][2 * w + v][1]);
            }
        }
        // scores, weights
        const int key = half * 16 + g;
        const float2 k0 = __half22float2(kpar[key]), k1 = __half22float2(kpar[key + 8]);
        __half2 v0h = vpar[key], v1h = vpar[key + 8];
        if (!whole) {  // slots that hold no token may hold anything
          if (base + key >= kv) v0h = __half2half2(__ushort_as_half(0));
          if (base + key + 8 >= kv) v1h = __half2half2(__ushort_as_half(0));
        }
        const float2 v0 = __half22float2(v0h), v1 = __half22float2(v1h);
        const float e0 = static_cast<float>(static_cast<int>((__half_as_ushort(__low2half(v0h)) >> 10) & 31u) - 15);
        const float e1 = static_cast<float>(static_cast<int>((__half_as_ushort(__low2half(v1h)) >> 10) & 31u) - 15);
        const float s0 = k0.x * q.mul, s1 = k1.x * q.mul;
        bool lift = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            s[nt][i] = fmaf(s0, s[nt][i], k0.y * q.zq[nt][i]);
            s[nt][2 + i] = fmaf(s1, s[nt][2 + i], k1.y * q.zq[nt][i]);
          }
        }
        if (!whole) {
          const bool here0 = (got >> (4 * (key / step))) & 1u, here1 = (got >> (4 * ((key + 8) / step))) & 1u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int p = q.pos[nt][i], j0 = base + key, j1 = j0 + 8;
              const bool see0 = here0 && j0 < kv && j0 <= p && (a.m.window == 0 || j0 > p - a.m.window || j0 < a.m.sinks);
              const bool see1 = here1 && j1 < kv && j1 <= p && (a.m.window == 0 || j1 > p - a.m.window || j1 < a.m.sinks);
              if (!see0) s[nt][i] = -INFINITY;
              if (!see1) s[nt][2 + i] = -INFINITY;
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            lift |= fmaxf(s[nt][i] + e0, s[nt][2 + i] + e1) > m[nt][i] + 8.0f;
        if (__any_sync(0xFFFFFFFFu, lift)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float top = fmaxf(s[nt][i] + e0, s[nt][2 + i] + e1);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
              top = fmaxf(top, m[nt][i]);
              const float by = exp2_approx(m[nt][i] - top);
              m[nt][i] = top;
              l[nt][i] *= by;
              z[nt][i] *= by;
#pragma unroll
              for (int j = 0; j < MT; ++j) {
                o[nt][j][i] *= by;
                o[nt][j][2 + i] *= by;
              }
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w0[2], w1[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = exp2_approx(s[nt][i] - m[nt][i]), p1 = exp2_approx(s[nt][2 + i] - m[nt][i]);
            l[nt][i] += p0 + p1;
            z[nt][i] = fmaf(p0, v0.y, fmaf(p1, v1.y, z[nt][i]));
            w0[i] = p0 * v0.x;
            w1[i] = p1 * v1.x;
          }
          pb[nt][0] = transpose_8x8(half2_bits(w0[0], w0[1]));
          pb[nt][1] = transpose_8x8(half2_bits(w1[0], w1[1]));
        }
        // O' += V' P': rows g and g + 8 are head elements, columns of V' the tokens 2t, 2t + 1, 2t + 8, 2t + 9
        {
          constexpr int VW = HD / 64;  // words of a token's value codes per lane
          const uint8_t* row = buf + kDecTile * (HD / 2) + (half * 16 + 2 * t) * (HD / 2) + g * (HD / 16);
          uint32_t v[4][VW];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint8_t* p = row + ((i & 1) + 8 * (i >> 1)) * (HD / 2);
            if constexpr (VW == 2) {
              const uint2 x = *reinterpret_cast<const uint2*>(p);
              v[i][0] = x.x, v[i][1] = x.y;
            } else {
              v[i][0] = *reinterpret_cast<const uint32_t*>(p);
            }
          }
#pragma unroll
          for (int w = 0; w < VW; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t x = __byte_perm(v[0][w], v[1][w], h ? 0x7632 : 0x5410);
              const uint32_t y = __byte_perm(v[2][w], v[3][w], h ? 0x7632 : 0x5410);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const uint32_t xs = x >> (8 * c), ys = y >> (8 * c);
                const uint32_t a0 = xs & 0x000F000Fu, a1 = xs & 0x00F000F0u, a2 = ys & 0x000F000Fu, a3 = ys & 0x00F000F0u;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][(w * 2 + h) * 2 + c], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
              }
            }
        }
      }
      __syncwarp();  // every lane has read the tile
      fetch(stage);
      if (++stage == kDecStages) {
        stage = 0;
        parity ^= 1;
      }
    }
    // the warps' sums meet
    float* meet = reinterpret_cast<float*>(smem + L::kOffMeet);
    float* ml = reinterpret_cast<float*>(smem + L::kOffMl);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l[nt][i] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][i], d);
          z[nt][i] += __shfl_xor_sync(0xFFFFFFFFu, z[nt][i], d);
        }
        const int r = nt * 8 + 2 * t + i;
        float* dst = meet + (warp * R + r) * L::kPitch + g * (2 * MT);
#pragma unroll
        for (int j = 0; j < MT / 2; ++j)
          reinterpret_cast<float4*>(dst)[j] =
              make_float4(fmaf(o[nt][2 * j][i], 16777216.0f, z[nt][i]), fmaf(o[nt][2 * j][2 + i], 1048576.0f, z[nt][i]),
                          fmaf(o[nt][2 * j + 1][i], 16777216.0f, z[nt][i]), fmaf(o[nt][2 * j + 1][2 + i], 1048576.0f, z[nt][i]));
        if (g == 0) {
          ml[(warp * R + r) * 2] = m[nt][i];
          ml[(warp * R + r) * 2 + 1] = l[nt][i];
        }
      }
    __syncthreads();
    const int rows = min(R, at.seq.n * a.G - at.rt * R);
    const bool whole_segment = at.u0 == 0 && at.u1 == at.span.count;
    const bool is_first = at.b == first_b && at.h == first_h && at.rt == first_rt;
    float* part_out = a.partial + (static_cast<size_t>(blockIdx.x) * 2 + (is_first ? 0 : 1)) * kv4_partial_floats(R, HD);
    for (int r = threadIdx.x / HD; r < rows; r += kDecThreads / HD) {
      const int d = threadIdx.x % HD;
      float top = kNoMax, sum = 0.0f, acc = 0.0f;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) top = fmaxf(top, ml[(w * R + r) * 2]);
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) {
        const float by = exp2_approx(ml[(w * R + r) * 2] - top);
        sum = fmaf(by, ml[(w * R + r) * 2 + 1], sum);
        acc = fmaf(by, meet[(w * R + r) * L::kPitch + d], acc);
      }
      if (whole_segment) {
        const int at_row = at.rt * R + r, i = at_row / a.G, head = at.h * a.G + (at_row - i * a.G);
        // no token seen: zero (and not 0 / 0); a row that is not finite stays NaN
        const float val = sum == 0.0f ? 0.0f : __fdividef(acc, sum);
        unsigned short bits;
        asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(bits) : "f"(val));
        a.out[(static_cast<int64_t>(at.seq.row0 + i) * a.c.hkv * a.G + head) * HD + d] = bits;
      } else {
        part_out[2 * R + r * HD + d] = acc;
        if (d == 0) {
          part_out[2 * r] = top;
          part_out[2 * r + 1] = sum;
        }
      }
    }
    if (!kv4_next_segment<kDecTile>(a.c, a.m, a.G, R, at)) break;
    __syncthreads();
  }
  __syncthreads();
  if (threadIdx.x == 0 && s_abort != 0) atomicExch(status, s_abort);
}

// Joins what several CTAs hold of a segment: block c the segment that begins in CTA c of the kernel before it and goes on
// behind it.  Always the same sums in the same order.
template <int HD, int R, int TK, int LEAST>
__global__ void __launch_bounds__(256)
kv4_combine_kernel(const Kv4AttnArgs a) {
  grid_dep_launch_dependents();
  __shared__ long long scan[257];
  grid_dep_wait();
  const Kv4Share sh = kv4_share<TK, 256>(a.c, a.m, a.G, R, LEAST, scan);
  const long long begin = blockIdx.x * sh.share, end = begin + sh.share;
  if (end >= sh.total) return;  // the last CTA's segments end with it
  Kv4Cursor k;
  const long long first = kv4_locate<TK, 256>(a.c, a.m, a.G, R, end - 1, 1, scan, k);
  const long long last = first + k.span.count - 1;
  if (first < begin || last < end) return;
  const int parts = static_cast<int>(last / sh.share - blockIdx.x) + 1;
  const int rows = min(R, k.seq.n * a.G - k.rt * R);
  const int d = threadIdx.x % HD;
  for (int r = threadIdx.x / HD + (256 / HD) * blockIdx.y; r < rows; r += (256 / HD) * gridDim.y) {
    float top = kNoMax, sum = 0.0f, acc = 0.0f;
    auto at = [&](int p) {
      const size_t slot = static_cast<size_t>(blockIdx.x + p) * 2 + (p == 0 && first > begin ? 1 : 0);
      return a.partial + slot * kv4_partial_floats(R, HD);
    };
    for (int p = 0; p < parts; ++p) top = fmaxf(top, at(p)[2 * r]);
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      const float* s = at(p);
      const float by = exp2_approx(s[2 * r] - top);
      sum = fmaf(by, s[2 * r + 1], sum);
      acc = fmaf(by, s[2 * R + r * HD + d], acc);
    }
    const int at_row = k.rt * R + r, i = at_row / a.G, head = k.h * a.G + (at_row - i * a.G);
    const float val = sum == 0.0f ? 0.0f : __fdividef(acc, sum);
    unsigned short bits;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(bits) : "f"(val));
    a.out[(static_cast<int64_t>(k.seq.row0 + i) * a.c.hkv * a.G + head) * HD + d] = bits;
  }
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

template <int HD, int NT>
static int launch_decode(const Kv4AttnArgs& a, int grid, cudaStream_t s, DeviceState* st) {
  constexpr int R = 8 * NT;
  DQ_CHECK_CUDA(launch_pdl(kv4_decode_kernel<HD, NT>, dim3(grid), dim3(kDecThreads), DecSmem<HD, NT>::kBytes, s, a,
                           st->status_dev));
  if (grid > 1)
    DQ_CHECK_CUDA(launch_pdl(kv4_combine_kernel<HD, R, kDecTile, kDecLeast>, dim3(grid, R * HD / 256 > 4 ? 4 : R * HD / 256), dim3(256), 0, s, a));
  return DQ_OK;
}

// Grid of a call: enough CTAs to fill the GPU, and no more than there can be shares.
static int decode_grid(const Kv4Batch& c, int G, int hd, int R, DeviceState* st) {
  const int64_t row_tiles = (static_cast<int64_t>(c.T) * G + R - 1) / R + c.B;
  const int64_t tiles = (c.capacity + kDecTile - 1) / kDecTile + 1;
  const int64_t most = (row_tiles * c.hkv * tiles + kDecLeast - 1) / kDecLeast;
  const int64_t fill = static_cast<int64_t>(st->sm_count) * g_resident[hd == 128][R / 8 - 1];
  return static_cast<int>(most < fill ? most : fill);
}

}  // namespace dq

using namespace dq;

static int kv4_rows(int G, int max_new) { return static_cast<int64_t>(G) * max_new <= 8 ? 8 : 16; }

extern "C" size_t dq_kv4_attention_workspace_bytes(const dq_kv4_batch* batch, int hq, int max_new) {
  DeviceState* st = current_state();
  Kv4Batch c;
  if (st == nullptr || kv4_batch_of(batch, &c) != DQ_OK || hq < 1 || max_new < 1) return 0;
  if (c.B == 0 || c.T == 0) return 0;
  const int G = hq / c.hkv > 0 ? hq / c.hkv : 1, R = kv4_rows(G, max_new);
  return static_cast<size_t>(decode_grid(c, G, batch->head_dim, R, st)) * 2 * kv4_partial_floats(R, batch->head_dim) * 4;
}

extern "C" int dq_kv4_attention(const dq_kv4_batch* batch, const void* q_bf16, int64_t q_row_stride, int64_t q_head_stride,
                                int hq, int max_new, int window, int sinks, float scale, void* out_bf16, void* workspace,
                                size_t workspace_bytes, void* stream) {
  DeviceState* st = current_state();
  if (st == nullptr) return DQ_ERR_NOT_INIT;
  Kv4AttnArgs a;
  int rc = kv4_batch_of(batch, &a.c);
  if (rc != DQ_OK) return rc;
  if (a.c.B == 0 || a.c.T == 0) return DQ_OK;
  DQ_REQUIRE(hq >= 1 && hq <= 4096 && hq % a.c.hkv == 0, DQ_ERR_SHAPE, "%d query heads over %d key/value heads", hq, a.c.hkv);
  DQ_REQUIRE(max_new >= 1 && window >= 0 && sinks >= 0, DQ_ERR_SHAPE, "max_new=%d window=%d sinks=%d", max_new, window, sinks);
  DQ_REQUIRE(q_bf16 != nullptr && out_bf16 != nullptr, DQ_ERR_NULL, "null pointer");
  DQ_REQUIRE(static_cast<int64_t>(a.c.T) * hq < (1ll << 30), DQ_ERR_SHAPE, "%d rows of %d heads", a.c.T, hq);
  DQ_REQUIRE(q_row_stride % 8 == 0 && q_head_stride % 8 == 0 && aligned(q_bf16, 16) && aligned(out_bf16, 16), DQ_ERR_ALIGN,
             "query heads and outputs must be 16-byte aligned");
  DQ_REQUIRE(isfinite(scale), DQ_ERR_SHAPE, "scale is not finite");
  const size_t need = dq_kv4_attention_workspace_bytes(batch, hq, max_new);
  DQ_REQUIRE(workspace_bytes >= need && (need == 0 || workspace != nullptr) && aligned(workspace, 16), DQ_ERR_WORKSPACE,
             "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  a.m.window = window < kKv4Far ? window : kKv4Far;
  a.m.sinks = sinks < kKv4Far ? sinks : kKv4Far;
  a.q = static_cast<const unsigned short*>(q_bf16);
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.out = static_cast<unsigned short*>(out_bf16);
  a.partial = static_cast<float*>(workspace);
  a.G = hq / a.c.hkv;
  a.scale2 = scale * 1.4426950408889634f;
  const int R = kv4_rows(a.G, max_new), hd = batch->head_dim;
  const int grid = decode_grid(a.c, a.G, hd, R, st);
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (hd == 128) return R == 8 ? launch_decode<128, 1>(a, grid, cs, st) : launch_decode<128, 2>(a, grid, cs, st);
  return R == 8 ? launch_decode<64, 1>(a, grid, cs, st) : launch_decode<64, 2>(a, grid, cs, st);
}
