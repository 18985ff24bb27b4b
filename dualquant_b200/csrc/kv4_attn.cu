// Attention over the paged 4-bit cache: choice of kernel, the kernel that joins what several CTAs hold of a segment, C entry.
#include <math.h>

#include "kv4.cuh"

namespace dq {

__device__ __forceinline__ float join_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Block (c, y) joins rows of the segment that begins in CTA c of the kernel before it and goes on behind it.  WARPS warps share a
// row and take every WARPS-th part of it (eight for the few rows of a decode step, whose long segments have dozens of parts; one
// for row tiles of a prompt, which have two or three), a lane holds HD / 32 elements: always the same sums in the same order.
// The first four parts of a warp are on the way before the largest maximum is known.
template <int HD, int R, int WARPS>
__global__ void __launch_bounds__(256)
kv4_combine_kernel(const __grid_constant__ Kv4AttnArgs a) {
  grid_dep_launch_dependents();
  constexpr int E = HD / 32, AHEAD = 4;
  __shared__ float s_acc[WARPS > 1 ? 8 : 1][HD], s_l[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % WARPS;
  grid_dep_wait();
  const Kv4Join j = a.join[blockIdx.x];
  if (j.parts == 0) return;
  auto part = [&](int p) {
    return a.partial + (static_cast<size_t>(blockIdx.x + p) * 2 + (p == 0 ? j.slot : 0)) * kv4_partial_floats(R, HD);
  };
  for (int r = blockIdx.y * (8 / WARPS) + warp / WARPS; r < j.rows; r += gridDim.y * (8 / WARPS)) {
    float ml[AHEAD][2], v[AHEAD][E];
    auto fetch = [&](int first) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int p = first + i * WARPS;
        ml[i][0] = kKv4NoMax;
        ml[i][1] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) v[i][e] = 0.0f;
        if (p < j.parts) {
          const float* s = part(p);
          const float2 x = *reinterpret_cast<const float2*>(s + 2 * r);
          ml[i][0] = x.x, ml[i][1] = x.y;
          const float* o = s + 2 * R + r * HD + lane * E;
          if constexpr (E == 4) {
            const float4 y = *reinterpret_cast<const float4*>(o);
            v[i][0] = y.x, v[i][1] = y.y, v[i][2] = y.z, v[i][3] = y.w;
          } else {
            const float2 y = *reinterpret_cast<const float2*>(o);
            v[i][0] = y.x, v[i][1] = y.y;
          }
        }
      }
    };
    fetch(sub);
    float top = kKv4NoMax;
    for (int p = lane; p < j.parts; p += 32) top = fmaxf(top, part(p)[2 * r]);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    float sum = 0.0f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    for (int first = sub;;) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const float by = join_exp2(ml[i][0] - top);
        sum = fmaf(by, ml[i][1], sum);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(by, v[i][e], acc[e]);
      }
      first += AHEAD * WARPS;
      if (first >= j.parts) break;
      fetch(first);
    }
    const int at_row = j.first_row + r, i = a.g.by(at_row), head = j.h * a.g.G + (at_row - i * a.g.G);
    unsigned short* out = a.out + (static_cast<int64_t>(j.row0 + i) * a.c.hkv * a.g.G + head) * HD;
    if constexpr (WARPS > 1) {
#pragma unroll
      for (int e = 0; e < E; ++e) s_acc[warp][lane * E + e] = acc[e];
      if (lane == 0) s_l[warp] = sum;
      __syncthreads();
      if (threadIdx.x < HD) {
        float l = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          l += s_l[w];
          o += s_acc[w][threadIdx.x];
        }
        const float val = l == 0.0f ? 0.0f : __fdividef(o, l);
        unsigned short bits;
        asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(bits) : "f"(val));
        out[threadIdx.x] = bits;
      }
      __syncthreads();
    } else {
      // no token seen: zero (and not 0 / 0); a row that is not finite stays NaN
      const float by = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
      uint32_t w[E / 2];
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        const float x = sum == 0.0f ? 0.0f : acc[2 * e] * by, y = sum == 0.0f ? 0.0f : acc[2 * e + 1] * by;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[e]) : "f"(y), "f"(x));
      }
      if constexpr (E == 4) *reinterpret_cast<uint2*>(out + lane * 4) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(out + lane * 2) = w[0];
    }
  }
}

// How a call runs: R query rows a segment (8, 16: kv4_decode_kernel, 128, 256: kv4_prefill_kernel) on `grid` CTAs.
struct Kv4Plan {
  int R, grid;
  size_t join_bytes, bytes;  // workspace
};

// grid: enough CTAs to fill the GPU, and no more than there can be shares.  0: too many tiles to number.
static Kv4Plan kv4_plan(const Kv4Batch& c, int G, int hd, int max_new, DeviceState* st) {
  Kv4Plan p;
  const int64_t rows = static_cast<int64_t>(G) * max_new;
  // The few-rows kernel reads the cache once for every 8 or 16 rows, the other one once for up to 128 or 256.  32 heads over 8, us:
  //                 tokens         8 rows by 8, 16   16 by 8, 16    32 by 16, 128   48 by 16, 128   64 by 16, 128
  //   heads of 128  16 x 4000         27   33          42   37         58   61         82   62         99   63
  //                  8 x 30000        61   79         110   83        148  184        215  186        279  187
  //                  1 x 4000         11              13   14         20              22   17         24   17
  //   heads of 64   16 x 4000         20   24          32   27         44   53         60   54         72   55
  //                  8 x 30000        44   57          77   60        107  163        155  163        201  164
  //                  1 x 4000          9              11   11         16              17   14         19   14
  // A row tile of 128 by itself in the two-tile kernel: 72, 218 and 17 (heads of 128).
  p.R = rows <= 8 ? 8 : rows <= 32 ? 16 : rows <= 128 ? 128 : 256;
  const bool many = p.R >= 128;
  const int tile = many ? kPreTile : kDecTile, least = many ? kPreLeast : kDecLeast;
  const int64_t row_tiles = (static_cast<int64_t>(c.T) * G + p.R - 1) / p.R + c.B;
  const int64_t units = row_tiles * c.hkv * ((c.capacity + tile - 1) / tile + 1);
  const int64_t most = (units + least - 1) / least;
  const int64_t fill = st->sm_count * (many ? 1 : kv4_decode_resident(hd, p.R));
  p.grid = units >= (1ll << 31) ? 0 : static_cast<int>(most < fill ? most : fill);
  p.join_bytes = (static_cast<size_t>(p.grid) * sizeof(Kv4Join) + 255) / 256 * 256;
  p.bytes = p.join_bytes + static_cast<size_t>(p.grid) * 2 * kv4_partial_floats(p.R, hd) * 4;
  return p;
}

template <int HD, int R, int WARPS>
static int launch_combine(const Kv4AttnArgs& a, int grid, cudaStream_t s) {
  constexpr int y = WARPS > 1 ? 4 : 8;
  DQ_CHECK_CUDA(launch_pdl(kv4_combine_kernel<HD, R, WARPS>, dim3(grid, y), dim3(256), 0, s, a));
  return DQ_OK;
}

template <int HD>
static int launch_combine_of(const Kv4AttnArgs& a, const Kv4Plan& p, cudaStream_t s) {
  switch (p.R) {
    case 8: return launch_combine<HD, 8, 8>(a, p.grid, s);
    case 16: return launch_combine<HD, 16, 8>(a, p.grid, s);
    case 128: return launch_combine<HD, 128, 1>(a, p.grid, s);
    default: return launch_combine<HD, 256, 1>(a, p.grid, s);
  }
}

}  // namespace dq

using namespace dq;

extern "C" size_t dq_kv4_attention_workspace_bytes(const dq_kv4_batch* batch, int hq, int max_new) {
  DeviceState* st = current_state();
  Kv4Batch c;
  if (st == nullptr || kv4_batch_of(batch, &c) != DQ_OK || hq < 1 || max_new < 1 || c.B == 0 || c.T == 0) return 0;
  return kv4_plan(c, hq / c.hkv > 0 ? hq / c.hkv : 1, batch->head_dim, max_new, st).bytes;
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
  const float scale2 = scale * 1.4426950408889634f;
  DQ_REQUIRE(isfinite(scale2), DQ_ERR_SHAPE, "scale log2(e) is not finite");
  a.g.G = hq / a.c.hkv;
  const int hd = batch->head_dim;
  const Kv4Plan p = kv4_plan(a.c, a.g.G, hd, max_new, st);
  DQ_REQUIRE(p.grid > 0, DQ_ERR_SHAPE, "%d rows over %d sequences of up to %d tokens are too many for one call", a.c.T, a.c.B,
             a.c.capacity);
  DQ_REQUIRE(workspace_bytes >= p.bytes && workspace != nullptr && aligned(workspace, 16), DQ_ERR_WORKSPACE,
             "workspace of %zu bytes, %zu needed", workspace_bytes, p.bytes);
  a.m.window = window < kKv4Far ? window : kKv4Far;
  a.m.sinks = sinks < kKv4Far ? sinks : kKv4Far;
  a.q = static_cast<const unsigned short*>(q_bf16);
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.out = static_cast<unsigned short*>(out_bf16);
  a.g.by = kv4_div(a.g.G);
  a.grid = kv4_div(p.grid);
  a.join = static_cast<Kv4Join*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.join_bytes);
  a.scale2 = scale2;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  rc = p.R >= 128 ? launch_kv4_prefill(a, hd, p.R, p.grid, cs, st) : launch_kv4_decode(a, hd, p.R, p.grid, cs);
  if (rc != DQ_OK || p.grid == 1) return rc;
  return hd == 128 ? launch_combine_of<128>(a, p, cs) : launch_combine_of<64>(a, p, cs);
}
