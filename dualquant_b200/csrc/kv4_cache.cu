// Writing to and reading from the paged 4-bit key/value cache (layout: kv4.cuh).
//
// kv4_append_kernel: position rotation of query and key heads, an optional Walsh-Hadamard rotation over the head (the
// online rotation that keeps outlier channels of keys from setting the grid of a whole head; applied to q and k alike it
// leaves their products as they are), 4-bit quantisation of keys and values, write into the pages.  All in fp32:
//   lo = x1 c - x2 s, hi = x2 c + x1 s        x1, x2: the halves of the head; each product and sum rounded on its own
//   butterflies h = 1, 2, 4 ... d / 2, then times fp32(d^-1/2)
//   scale = fp16((max - min) * fp32(1 / 15)), zero = fp16(min), code = clamp(rint((x - zero) * (1 / scale)), 0, 15)
//   (one step of fp16 less scale where 15 scale + zero would round to infinity there: only heads that reach past 65400)
// The two roundings to fp16 are the storage of the grid: codes are taken on the stored grid, and 4 bytes a head against
// d / 2 of codes are 6 to 12 % of the cache.  NaN is stored as 0 and what fp16 cannot hold as +-65504, so that a page that
// was written stands for finite numbers only, in fp16 too (the keys and values of kv4_prefill_kernel).
#include "kv4.cuh"

namespace dq {

__device__ __forceinline__ void bf16x8_to_float(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = __uint_as_float(w[j] << 16);
    f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint32_t bf16x2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// d / 16 lanes hold a head: lane l the elements 8l ... 8l + 7 of both halves, so that the rotation of positions, three
// butterfly stages and the last one stay in registers.  A warp's heads belong to one token; its row and the look-up of its sequence
// are on their way at once.  grid: (T, pieces of 4 warps).
//
// Bound by instruction issue for prompts (two thirds of the slots, most of them butterflies and their shuffles): arithmetic on
// pairs where that keeps every rounding, a - b as fma(b, -1, a).  9937 tokens of 32 + 2 * 8 heads of 128, 214 MB: 53 us; 86 with
// scalars and a chain of four loads.  Twelve blocks an SM at 40 registers: two or four tokens a block took 3 and 12 us longer.
template <int HD>
__global__ void __launch_bounds__(128, 12)
kv4_append_kernel(const __grid_constant__ Kv4Batch c, const unsigned short* qkv, int64_t ld, const float* cos_tab,
                  const float* sin_tab, int tab_rows, int hq, int rotate, unsigned short* __restrict__ q_out) {
  grid_dep_launch_dependents();
  grid_dep_wait();
  constexpr int LANES = HD / 16, HALF = HD / 2;
  const int lane = threadIdx.x & 31, l = threadIdx.x % LANES;
  const int head = blockIdx.y * (128 / LANES) + threadIdx.x / LANES, heads = hq + 2 * c.hkv;
  const bool live = head < heads;  // whole groups of lanes; the shuffles below want every lane
  const bool is_q = head < hq, is_v = head >= hq + c.hkv;
  const int row = blockIdx.x;
  uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (live) {
    const unsigned short* src = qkv + row * ld + static_cast<int64_t>(head) * HD + 8 * l;
    raw[0] = *reinterpret_cast<const uint4*>(src);
    raw[1] = *reinterpret_cast<const uint4*>(src + HALF);
  }
  const float2 minus = make_float2(-1.0f, -1.0f);
  int pos;
  const int b = kv4_find(c, row, lane, &pos);
  if (b >= c.B) return;
  const bool there = pos >= 0 && pos < c.capacity && pos < tab_rows;
  int page = -1;
  if (there && !is_q) page = c.table[b * c.table_stride + (pos >> c.page_shift)];
  float2 x[8];  // elements 8l + 2j, + 1 for j < 4, the same of the second half for j >= 4
  {
    const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
  }
  if (__any_sync(0xFFFFFFFFu, !is_v)) {
    if (!is_v && there) {
      const float4* cp = reinterpret_cast<const float4*>(cos_tab + static_cast<int64_t>(pos) * HALF + 8 * l);
      const float4* sp = reinterpret_cast<const float4*>(sin_tab + static_cast<int64_t>(pos) * HALF + 8 * l);
      const float4 c0 = cp[0], c1 = cp[1], s0 = sp[0], s1 = sp[1];
      const float2 cs[4] = {make_float2(c0.x, c0.y), make_float2(c0.z, c0.w), make_float2(c1.x, c1.y), make_float2(c1.z, c1.w)};
      const float2 sn[4] = {make_float2(s0.x, s0.y), make_float2(s0.z, s0.w), make_float2(s1.x, s1.y), make_float2(s1.z, s1.w)};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = x[j], d = x[j + 4];
        // (scalars: packed products and sums were joined into packed FMAs, without the product's own rounding)
        x[j] = make_float2(__fsub_rn(__fmul_rn(a.x, cs[j].x), __fmul_rn(d.x, sn[j].x)),
                           __fsub_rn(__fmul_rn(a.y, cs[j].y), __fmul_rn(d.y, sn[j].y)));
        x[j + 4] = make_float2(__fadd_rn(__fmul_rn(d.x, cs[j].x), __fmul_rn(a.x, sn[j].x)),
                               __fadd_rn(__fmul_rn(d.y, cs[j].y), __fmul_rn(a.y, sn[j].y)));
      }
    }
    if (rotate) {
      // (value heads of a mixed warp take part in the shuffles and keep their own numbers)
      float2 y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = make_float2(__fadd_rn(x[j].x, x[j].y), __fsub_rn(x[j].x, x[j].y));
#pragma unroll
      for (int h = 1; h < 4; h <<= 1)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if ((j & h) == 0) {
            const float2 u = y[j], w = y[j + h];
            y[j] = __fadd2_rn(u, w);
            y[j + h] = __ffma2_rn(w, minus, u);
          }
#pragma unroll
      for (int h = 1; h < LANES; h <<= 1) {
        const float sign = (l & h) ? -1.0f : 1.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 o = make_float2(__shfl_xor_sync(0xFFFFFFFFu, y[j].x, h), __shfl_xor_sync(0xFFFFFFFFu, y[j].y, h));
          y[j] = __ffma2_rn(y[j], make_float2(sign, sign), o);
        }
      }
      const float norm = HD == 128 ? 0.08838834764831845f : 0.125f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 u = y[j], w = y[j + 4];
        y[j] = __fmul2_rn(__fadd2_rn(u, w), make_float2(norm, norm));
        y[j + 4] = __fmul2_rn(__ffma2_rn(w, minus, u), make_float2(norm, norm));
      }
      if (!is_v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = y[j];
      }
    }
  }
  if (is_q && live) {
    // a token without a place in the cache has no position: its query row is zero
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = there ? bf16x2_of(x[j].x, x[j].y) : 0u;
    unsigned short* dst = q_out + (static_cast<int64_t>(row) * hq + head) * HD + 8 * l;
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(dst + HALF) = make_uint4(w[4], w[5], w[6], w[7]);
  }
  if (!__any_sync(0xFFFFFFFFu, live && !is_q)) return;
  // numbers that the grid cannot hold are rare: looked for in all of a warp's heads at once (0 * x is NaN for them, and fp16
  // ends at 65504)
  float2 odd = make_float2(0.0f, 0.0f);
  float lo = x[0].x, hi = x[0].x;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    odd = __ffma2_rn(x[j], make_float2(0.0f, 0.0f), odd);
    lo = fminf(lo, fminf(x[j].x, x[j].y));
    hi = fmaxf(hi, fmaxf(x[j].x, x[j].y));
  }
  if (__any_sync(0xFFFFFFFFu, !(odd.x + odd.y == 0.0f) || lo < -65504.0f || hi > 65504.0f)) {
    lo = 65504.0f, hi = -65504.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j].x = isnan(x[j].x) ? 0.0f : fminf(fmaxf(x[j].x, -65504.0f), 65504.0f);
      x[j].y = isnan(x[j].y) ? 0.0f : fminf(fmaxf(x[j].y, -65504.0f), 65504.0f);
      lo = fminf(lo, fminf(x[j].x, x[j].y));
      hi = fmaxf(hi, fmaxf(x[j].x, x[j].y));
    }
  }
#pragma unroll
  for (int h = 1; h < LANES; h <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, h));
    hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, h));
  }
  if (is_q || !live || static_cast<uint32_t>(page) >= static_cast<uint32_t>(c.num_pages)) return;
  __half hs = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  const __half hz = __float2half_rn(lo);
  // 15 scale + zero is at most 65504 + 16 (zero) + 7.5 ulp (scale), and 65520 is the first that rounds to infinity
  if (fmaf(15.0f, __half2float(hs), __half2float(hz)) >= 65520.0f) hs = __ushort_as_half(__half_as_ushort(hs) - 1);
  const float sf = __half2float(hs), zf = __half2float(hz);
  const float inv = sf > 0.0f ? __frcp_rn(sf) : 0.0f;
  // rint and clamp as clamp and an addition whose sum has no room for a fraction; its bits are a constant plus the code, and
  // the constants' sum is taken off the word at the end
  uint32_t code[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float2 r = __fmul2_rn(__fadd2_rn(x[j], make_float2(-zf, -zf)), make_float2(inv, inv));
    r = make_float2(fminf(fmaxf(r.x, 0.0f), 15.0f), fminf(fmaxf(r.y, 0.0f), 15.0f));
    r = __fadd2_rn(r, make_float2(12582912.0f, 12582912.0f));
    code[j >> 2] += __float_as_uint(r.x) << (8 * (j & 3));
    code[j >> 2] += __float_as_uint(r.y) << (8 * (j & 3) + 4);
  }
  uint32_t constants = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) constants += 0x4B400000u << (4 * j);
  const int P = 1 << c.page_shift, slot = pos & (P - 1), kvh = head - hq - (is_v ? c.hkv : 0);
  uint8_t* block = c.pages + page * c.page_stride + static_cast<int64_t>(kvh) * P * (HD + 8);
  uint32_t* dst = reinterpret_cast<uint32_t*>(block + (is_v ? P * HALF : 0) + slot * HALF) + l;
  dst[0] = code[0] - constants;
  dst[HALF / 8] = code[1] - constants;
  if (l == 0) {
    __half2* par = reinterpret_cast<__half2*>(block + P * HD + (is_v ? 4 * P : 0)) + slot;
    *par = __halves2half2(hs, hz);
  }
}

// Eight codes of a word as 2^23 + c 16^k with k such that the code stays where it is in the mantissa: one logic operation each
// (and a shift for the last three), then exact arithmetic on pairs.  -> bf16 of c * scale + zero, one rounding each
struct Kv4Grid {
  float2 by[3];  // scale / 16^k of codes 2j and 2j + 1: (k = 0, 1), (2, 3), (4, 2)
  float2 zero;
};
__device__ __forceinline__ Kv4Grid kv4_grid(__half2 pair) {
  const float2 f = __half22float2(pair);
  Kv4Grid r;
  r.by[0] = make_float2(f.x, f.x * 0.0625f);
  r.by[1] = make_float2(f.x * 0.00390625f, f.x * 0.000244140625f);
  r.by[2] = make_float2(f.x * 0.0000152587890625f, r.by[1].x);
  r.zero = make_float2(f.y, f.y);
  return r;
}
__device__ __forceinline__ uint4 kv4_values(uint32_t w, const Kv4Grid& g) {
  constexpr uint32_t k23 = 0x4B000000u;
  const float2 off = make_float2(-8388608.0f, -8388608.0f);
  const uint32_t v = w >> 12;  // codes 5, 6, 7 at k = 2, 3, 4
  auto at = [](uint32_t x, int k) { return __uint_as_float((x & (15u << (4 * k))) | k23); };
  auto pair = [&](float lo, float hi, float2 by) {
    const float2 x = __ffma2_rn(__fadd2_rn(make_float2(lo, hi), off), by, g.zero);
    return bf16x2_of(x.x, x.y);
  };
  return make_uint4(pair(at(w, 0), at(w, 1), g.by[0]), pair(at(w, 2), at(w, 3), g.by[1]), pair(at(w, 4), at(v, 2), g.by[2]),
                    pair(at(v, 3), at(v, 4), make_float2(g.by[1].y, g.by[2].x)));
}

// The values of the last n tokens of each sequence as bf16 rows.  A warp makes the keys and values of one head of 512 / d
// consecutive tokens, a lane 16 elements of both: the codes of a warp lie together, and so do the pairs.  Rows of tokens that the
// cache does not hold are zero.  Sixteen sequences of up to 4096 tokens, 8 heads of 128, 190 MB: 39 us (40 with a token a block, 44 to
// 46 with several tokens a lane).  grid: hkv blocks of kReadThreads threads for every kReadThreads * 16 / d tokens, heads fastest.
constexpr int kReadThreads = 128;
template <int HD>
__global__ void __launch_bounds__(kReadThreads)
kv4_read_kernel(const __grid_constant__ Kv4Batch c, Kv4Div by_hkv, unsigned short* __restrict__ k_out,
                unsigned short* __restrict__ v_out) {
  grid_dep_launch_dependents();
  grid_dep_wait();
  constexpr int LANES = HD / 16, ROWS = 32 / LANES;
  const int lane = threadIdx.x & 31, l = lane % LANES;
  const int group = by_hkv(blockIdx.x), head = blockIdx.x - group * c.hkv;
  const int row0 = (group * (kReadThreads / 32) + (threadIdx.x >> 5)) * ROWS, row = row0 + lane / LANES;
  int b = c.B, pos = -1;
  kv4_find_rows<ROWS>(c, row0, lane, lane / LANES, &b, &pos);
  if (b >= c.B) return;
  const int P = 1 << c.page_shift, slot = pos & (P - 1);
  uint4 k[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)}, v[2] = {k[0], k[0]};
  int page = -1;
  if (pos >= 0 && pos < c.capacity) page = c.table[b * c.table_stride + (pos >> c.page_shift)];
  if (static_cast<uint32_t>(page) < static_cast<uint32_t>(c.num_pages)) {
    const uint8_t* block = c.pages + page * c.page_stride + static_cast<int64_t>(head) * P * (HD + 8);
    const uint8_t *codes = block + slot * (HD / 2) + 8 * l, *pairs = block + P * HD + 4 * slot;
    const uint2 kw = *reinterpret_cast<const uint2*>(codes), vw = *reinterpret_cast<const uint2*>(codes + P * (HD / 2));
    const Kv4Grid kg = kv4_grid(*reinterpret_cast<const __half2*>(pairs)), vg = kv4_grid(*reinterpret_cast<const __half2*>(pairs + 4 * P));
    k[0] = kv4_values(kw.x, kg);
    k[1] = kv4_values(kw.y, kg);
    v[0] = kv4_values(vw.x, vg);
    v[1] = kv4_values(vw.y, vg);
  }
  const int64_t to = (static_cast<int64_t>(row) * c.hkv + head) * HD + 16 * l;
  reinterpret_cast<uint4*>(k_out + to)[0] = k[0];
  reinterpret_cast<uint4*>(k_out + to)[1] = k[1];
  reinterpret_cast<uint4*>(v_out + to)[0] = v[0];
  reinterpret_cast<uint4*>(v_out + to)[1] = v[1];
}

int kv4_batch_of(const dq_kv4_batch* in, Kv4Batch* out) {
  DQ_REQUIRE(in != nullptr, DQ_ERR_NULL, "null dq_kv4_batch");
  DQ_REQUIRE(in->batch >= 0 && in->tokens >= 0, DQ_ERR_SHAPE, "batch=%d tokens=%d", in->batch, in->tokens);
  DQ_REQUIRE(in->head_dim == 64 || in->head_dim == 128, DQ_ERR_UNSUPPORTED, "head_dim %d: 64 or 128", in->head_dim);
  DQ_REQUIRE(in->hkv >= 1 && in->hkv <= 1024, DQ_ERR_SHAPE, "hkv=%d", in->hkv);
  int shift = 4;
  while (shift < 8 && (1 << shift) != in->page_size) ++shift;
  DQ_REQUIRE((1 << shift) == in->page_size, DQ_ERR_UNSUPPORTED, "page_size %d: a power of two from 16 to 256", in->page_size);
  const int64_t block = static_cast<int64_t>(in->page_size) * (in->head_dim + 8);
  DQ_REQUIRE(in->num_pages >= 0 && in->num_pages < (1ll << 31), DQ_ERR_SHAPE, "num_pages=%lld", (long long)in->num_pages);
  DQ_REQUIRE(in->page_stride >= block * in->hkv && in->page_stride % 16 == 0 && in->page_stride < (1ll << 32), DQ_ERR_ALIGN,
             "page_stride %lld: a multiple of 16 below 4 GiB and at least hkv blocks of %lld", (long long)in->page_stride, (long long)block);
  DQ_REQUIRE(in->pages_per_seq >= 0 && static_cast<int64_t>(in->pages_per_seq) * in->page_size < (1ll << 30) &&
                 in->table_stride >= in->pages_per_seq,
             DQ_ERR_SHAPE, "pages_per_seq=%d table_stride=%lld", in->pages_per_seq, (long long)in->table_stride);
  if (in->batch > 0 && in->tokens > 0) {
    DQ_REQUIRE(in->kv_len != nullptr && (in->block_table != nullptr || in->pages_per_seq == 0) &&
                   (in->pages != nullptr || in->num_pages == 0),
               DQ_ERR_NULL, "null pointer");
    DQ_REQUIRE(aligned(in->pages, 16), DQ_ERR_ALIGN, "pages must be 16-byte aligned");
    DQ_REQUIRE(in->cu_new != nullptr || in->tokens % in->batch == 0, DQ_ERR_SHAPE,
               "%d rows do not divide by %d sequences", in->tokens, in->batch);
  }
  out->pages = static_cast<uint8_t*>(in->pages);
  out->page_stride = in->page_stride;
  out->num_pages = in->num_pages;
  out->table = in->block_table;
  out->table_stride = in->table_stride;
  out->kv_len = in->kv_len;
  out->cu_new = in->cu_new;
  out->B = in->batch;
  out->T = in->tokens;
  out->hkv = in->hkv;
  out->page_shift = shift;
  out->capacity = in->pages_per_seq << shift;
  return DQ_OK;
}

}  // namespace dq

using namespace dq;

extern "C" size_t dq_kv4_page_bytes(int hkv, int head_dim, int page_size) {
  if (hkv < 1 || head_dim < 1 || page_size < 1) return 0;
  return static_cast<size_t>(hkv) * page_size * (head_dim + 8);
}

extern "C" int dq_kv4_append(const dq_kv4_batch* batch, const void* qkv_bf16, int64_t ld_qkv, const float* cos_tab,
                             const float* sin_tab, int table_rows, int hq, int rotate, void* q_out_bf16, void* stream) {
  if (current_state() == nullptr) return DQ_ERR_NOT_INIT;
  Kv4Batch c;
  const int rc = kv4_batch_of(batch, &c);
  if (rc != DQ_OK) return rc;
  if (c.B == 0 || c.T == 0) return DQ_OK;
  const int heads = hq + 2 * c.hkv;
  DQ_REQUIRE(hq >= 1 && hq <= 4096 && table_rows >= 0, DQ_ERR_SHAPE, "hq=%d table_rows=%d", hq, table_rows);
  DQ_REQUIRE(qkv_bf16 != nullptr && q_out_bf16 != nullptr && (table_rows == 0 || (cos_tab != nullptr && sin_tab != nullptr)),
             DQ_ERR_NULL, "null pointer");
  DQ_REQUIRE(ld_qkv >= static_cast<int64_t>(heads) * batch->head_dim, DQ_ERR_SHAPE, "ld_qkv too small");
  DQ_REQUIRE(ld_qkv % 8 == 0 && aligned(qkv_bf16, 16) && aligned(cos_tab, 16) && aligned(sin_tab, 16) && aligned(q_out_bf16, 16),
             DQ_ERR_ALIGN, "rows must be 16-byte aligned (ld_qkv a multiple of 8)");
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const auto* x = static_cast<const unsigned short*>(qkv_bf16);
  auto* q = static_cast<unsigned short*>(q_out_bf16);
  if (batch->head_dim == 128)
    DQ_CHECK_CUDA(launch_pdl(kv4_append_kernel<128>, dim3(c.T, (heads + 15) / 16), dim3(128), 0, cs, c, x, ld_qkv, cos_tab,
                             sin_tab, table_rows, hq, rotate, q));
  else
    DQ_CHECK_CUDA(launch_pdl(kv4_append_kernel<64>, dim3(c.T, (heads + 31) / 32), dim3(128), 0, cs, c, x, ld_qkv, cos_tab,
                             sin_tab, table_rows, hq, rotate, q));
  return DQ_OK;
}

extern "C" int dq_kv4_read(const dq_kv4_batch* batch, void* k_out_bf16, void* v_out_bf16, void* stream) {
  if (current_state() == nullptr) return DQ_ERR_NOT_INIT;
  Kv4Batch c;
  const int rc = kv4_batch_of(batch, &c);
  if (rc != DQ_OK) return rc;
  if (c.B == 0 || c.T == 0) return DQ_OK;
  DQ_REQUIRE(k_out_bf16 != nullptr && v_out_bf16 != nullptr, DQ_ERR_NULL, "null pointer");
  DQ_REQUIRE(aligned(k_out_bf16, 16) && aligned(v_out_bf16, 16), DQ_ERR_ALIGN, "outputs must be 16-byte aligned");
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  auto* k = static_cast<unsigned short*>(k_out_bf16);
  auto* v = static_cast<unsigned short*>(v_out_bf16);
  // (T rows of hkv heads each are below 2^31 threads' worth: grid.x goes to 2^31 - 1)
  const int64_t rows = kReadThreads * 16 / batch->head_dim, blocks = (c.T + rows - 1) / rows * c.hkv;
  DQ_REQUIRE(blocks < (1ll << 31), DQ_ERR_SHAPE, "%d rows of %d heads", c.T, c.hkv);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (batch->head_dim == 128)
    DQ_CHECK_CUDA(launch_pdl(kv4_read_kernel<128>, grid, dim3(kReadThreads), 0, cs, c, kv4_div(c.hkv), k, v));
  else
    DQ_CHECK_CUDA(launch_pdl(kv4_read_kernel<64>, grid, dim3(kReadThreads), 0, cs, c, kv4_div(c.hkv), k, v));
  return DQ_OK;
}
