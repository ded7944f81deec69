// The 8-bit paged KV cache: what its kernels share (kv8_cache.cu, kv8_attn.cu).
//
// Codes are e4m3 [layers, pages, kv_heads, page, head_dim], for keys and for values. The 16-token
// block is the unit everywhere: page is a multiple of 16, a block of one head is 16 * head_dim
// contiguous bytes and has one f32 scale, a power of two, in [layers, pages, kv_heads, page / 16].
// A value is code * scale. So a block's number, (page * kv_heads + head) * (page / 16) + block in
// page, indexes the scales directly and the codes times 16 * head_dim.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "j4b_internal.h"
#include "j4b_wait.cuh"

namespace j4b {

constexpr int kKvBlock = 16;       // tokens that share a scale
constexpr float kE4m3Max = 448.f;  // 1.75 * 2^8

// One layer's cache as the kernels take it.
struct Kv8View {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int pages, kv_heads, bpp;  // bpp: blocks of a page
};

// The sequences' pages: row b of the table names them in token order (-1 or any number outside
// [0, pages): unmapped).
struct Kv8Table {
  const int* pages;
  int64_t stride;
  int width;
};

__device__ __forceinline__ int kv8_block_id(const Kv8View& c, const Kv8Table& t, int b, int head, int blk) {
  const int pg = blk / c.bpp;
  if (pg >= t.width) return -1;
  const int id = __ldg(t.pages + b * t.stride + pg);
  if ((unsigned)id >= (unsigned)c.pages) return -1;
  return (id * c.kv_heads + head) * c.bpp + (blk - pg * c.bpp);
}

// The smallest power of two s >= 2^-120 with amax <= 448 s, from amax's exponent and mantissa
// (amax = m 2^E, 1 <= m < 2: s = 2^(E - 8) if m <= 1.75, else 2^(E - 7)). A power of two costs no
// accuracy (the codes are floating point) and a block's scale can grow without rounding its codes
// again. amax is finite and not negative.
__device__ __forceinline__ float kv8_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
  e = e < 7 ? 7 : e;  // biased: 2^-120 and above
  return __uint_as_float((uint32_t)e << 23);
}
// 1 / s of a power of two in [2^-120, 2^120]
__device__ __forceinline__ float kv8_inverse(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// two f32 -> two e4m3 (round to nearest even, saturating; lo in the low byte)
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) { return e4m3x2(a, b) | (e4m3x2(c, d) << 16); }
// two e4m3 -> f16x2, exact
__device__ __forceinline__ uint32_t e4m3_f16x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
__device__ __forceinline__ void e4m3x4_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  uint16_t a, b;
  asm("mov.b32 {%0, %1}, %2;" : "=h"(a), "=h"(b) : "r"(w));
  lo = e4m3_f16x2(a);
  hi = e4m3_f16x2(b);
}

// Activation element types of the entry points (J4B_F32, J4B_BF16).
__device__ __forceinline__ float4 load4(const void* p, int type, int64_t i) {
  if (type == J4B_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
  const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + i);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ void store4(void* p, int type, int64_t i, float4 v) {
  if (type == J4B_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = v;
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    uint2 u;
    u.x = *reinterpret_cast<const uint32_t*>(&a);
    u.y = *reinterpret_cast<const uint32_t*>(&b);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p) + i) = u;
  }
}

// two f32 -> f16x2, a in the low half
__device__ __forceinline__ uint32_t h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Lengths, starts and offsets come from device memory, where nobody has looked at them: the kernels
// take them as they are within these bounds, so that no value leads out of a buffer or keeps a
// kernel walking over blocks that no table can name.
constexpr int kMaxLength = 0x7fffffc0;
constexpr int kNowhere = 0x7fffffe0;  // the position of what is not there: past every query
__device__ __forceinline__ int kv8_length(const int* lengths, int b) { return min(max(__ldg(lengths + b), 0), kMaxLength); }
// Rows of sequence b among the call's: what its offsets name past the `tokens` there are is not there.
__device__ __forceinline__ int kv8_rows(const int* offsets, int b, int64_t tokens) {
  const int from = __ldg(offsets + b), to = min(max(0, __ldg(offsets + b + 1)), (int)tokens);
  return from < 0 ? 0 : max(0, to - from);
}

// The blocks that queries at positions first .. last of a sequence of `len` tokens see: the first
// `sink_blocks` ones, then those from `from` on to `end` (exclusive). count() of them in order.
struct Span {
  int sink_blocks, from, end;
  __device__ __forceinline__ int count() const { return sink_blocks + end - from; }
  __device__ __forceinline__ int block(int i) const { return i < sink_blocks ? i : from + i - sink_blocks; }
};
__device__ __forceinline__ Span span_of(int first, int last, int window, int sinks, int cap) {
  const int lo = window > 0 ? max(0, first - window + 1) : 0;  // first position in the window of `first`
  Span s;
  s.from = min(lo / kKvBlock, cap);
  s.end = last < 0 ? s.from : max(s.from, min(last / kKvBlock + 1, cap));
  s.sink_blocks = min((sinks + kKvBlock - 1) / kKvBlock, s.from);
  return s;
}

struct AttnArgs {
  Kv8View c;
  Kv8Table t;
  const void* q;
  int64_t q_stride;
  int q_type;
  const int* lengths;
  const int* offsets;  // prefill
  int64_t tokens;      // rows of q
  int batch, heads, group;
  int window, sinks;
  int cap;  // blocks of a table row
  float scale_log2;
  void* out;
  int out_type;
  int* timeout;  // host memory; set when a wait gave up
};

// Of numbers that are not negative, and seldom past 31 bits: a 64-bit division takes as long as a load.
__device__ __forceinline__ int64_t kv8_quotient(int64_t a, int64_t b) {
  return ((a | b) >> 31) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

__device__ __forceinline__ uint8_t* aligned_smem(uint8_t* raw) {  // the swizzle goes by address bits
  return raw + ((1024u - ((uint32_t)__cvta_generic_to_shared(raw) & 1023u)) & 1023u);
}

// Waits for an mbarrier's phase, bounded as mbar_wait_timed's waits are, but the clock is read once
// in 64 polls: the read takes long enough to make a waiter late where tiles are handed on every
// microsecond. `more`: nanoseconds above the common bound.
__device__ __forceinline__ bool kv8_wait(uint64_t* bar, uint32_t parity, uint64_t more = 0) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(bar);
  if (mbar_try_wait_parity(at, parity)) return true;
  uint64_t t0 = 0;
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait_parity(at, parity)) return true;
    const uint64_t now = global_ns();
    if (t0 == 0)
      t0 = now;
    else if (now - t0 > kWaitNs + more)
      return false;
  }
}

// Where a unit of work lies when sequence b has count(b) consecutive units.
struct Kv8Place {
  int seq;        // -1: past the last unit
  int64_t at;     // its number among the sequence's
  int64_t total;  // units of all sequences
};

// Finds unit unit(total) for a CTA of THREADS threads (all of them call it): every thread sums a
// contiguous share of the sequences, the shares are scanned, and the thread whose share holds the
// unit walks it. each(b0, b1, before) sees every thread's share and the units before it.
template <int THREADS, class Count, class Unit, class Each>
__device__ __forceinline__ Kv8Place kv8_find(int batch, Count count, Unit unit, Each each) {
  __shared__ int64_t warp_sum[THREADS / 32];
  __shared__ int64_t found_at;
  __shared__ int found_seq;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (batch + THREADS - 1) / THREADS;
  const int b0 = min(batch, tid * per), b1 = min(batch, b0 + per);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += count(b);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int64_t before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  each(b0, b1, before);
  int64_t left = unit(total) - before;
  if (left >= 0 && left < mine) {
    int b = b0;
    for (int64_t n; left >= (n = count(b)); ++b) left -= n;
    found_seq = b;
    found_at = left;
  } else if (tid == 0 && unit(total) >= total) {
    found_seq = -1;
    found_at = 0;
  }
  __syncthreads();
  return {found_seq, found_at, total};
}
template <int THREADS, class Count, class Unit>
__device__ __forceinline__ Kv8Place kv8_find(int batch, Count count, Unit unit) {
  return kv8_find<THREADS>(batch, count, unit, [](int, int, int64_t) {});
}

// Checks an entry point's arguments (kv8_cache.cu, kv8_attn.cu).
int kv8_check(const j4b_kv8_cache* c, int64_t layer, Kv8View* view, int* dev);
int kv8_check_attention(const j4b_kv8_cache* cache, int64_t layer, j4b_buf q, int q_type, int64_t q_stride, int64_t tokens, int64_t heads,
                        j4b_buf table, int64_t table_stride, int64_t table_width, j4b_buf lengths, int64_t batch, int64_t window,
                        int64_t sinks, double scale, j4b_buf out, int out_type, AttnArgs* a, int* dev);

}  // namespace j4b
