// The 8-bit paged KV cache: writing tokens into it (RoPE, block quantisation) and copying pages.
// Format and scale rule: kv8_common.cuh. Attention over it: kv8_attn.cu.
#include <algorithm>
#include <new>
#include <vector>

#include "kv8_common.cuh"

namespace j4b {
namespace {

// ---------------------------------------------------------------------------------------------
// Append. Token i of sequence b goes to position pos = starts[b] + i: its q and k heads are rotated
// by the angles of row pos of the rope table ((x0, x1) -> (x0 c - x1 s, x0 s + x1 c), products and
// sums rounded one by one), q is written out, k and v are quantised into the block of pos.
//
// Work: an item is one (sequence, 16-token block) pair that gets tokens; a CTA of 128 threads takes
// an item and every gridDim.y-th of its heads + 2 kv_heads tiles of up to 16 tokens x D. A tile is
// held in registers (16 values a thread at D = 128): loaded once, its largest magnitude reduced
// across the CTA, quantised and stored, so each input byte is read once. When the item starts
// inside a block, the codes of the block's earlier tokens are rescaled by the (power of two) ratio
// of the scales if the block's scale grows, and left alone otherwise. Bound by
// HBM: 16 chunks of up to 2047 tokens of 32 + 16 heads of 128 take 101 us, 5.74 TB/s read and written.
struct AppendArgs {
  Kv8View c;
  Kv8Table t;
  const float* qkv;
  int64_t row_stride;
  int64_t tokens;
  const float2* rope;  // [positions, D / 2] (cos, sin)
  int64_t positions;
  const int* starts;
  const int* offsets;  // [batch + 1]; null in the one-token kernel
  int batch, heads;
  void* q;
  int q_type;
};

constexpr int kAppendThreads = 128;

__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) <= 3.402823466e38f ? fabsf(x) : 0.f; }

template <int D>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const AppendArgs a) {
  constexpr int kLanes = kAppendThreads / kKvBlock;  // threads of a token: D / 8 values each
  constexpr int kVec = D / (4 * kLanes);             // as float4
  auto rows_of = [&](int b) -> int {  // new tokens of sequence b
    const int n = kv8_rows(a.offsets, b, a.tokens), s = __ldg(a.starts + b);  // loads side by side
    return s < 0 ? 0 : min(n, kMaxLength - min(s, kMaxLength));
  };
  const Kv8Place at = kv8_find<kAppendThreads>(
      a.batch,
      [&](int b) -> int64_t {
        const int n = rows_of(b), s = a.starts[b];
        return n > 0 ? (s + n + kKvBlock - 1) / kKvBlock - s / kKvBlock : 0;
      },
      [&](int64_t) -> int64_t { return blockIdx.x; });
  if (at.seq < 0) return;
  const int b = at.seq, start = a.starts[b];
  const int row0 = a.offsets[b], n = rows_of(b);
  const int blk = start / kKvBlock + (int)at.at;     // block of the sequence
  const int p0 = max(start, blk * kKvBlock);         // first position written
  const int cnt = min(start + n, (blk + 1) * kKvBlock) - p0;
  const int slot0 = p0 - blk * kKvBlock;             // tokens that the block holds already
  const int tid = threadIdx.x, tok = tid / kLanes, sub = tid % kLanes;
  const int64_t row = (int64_t)row0 + (p0 - start) + tok;
  // a token past the rope table or the input is not written; its q is zero
  const bool mine = tok < cnt && row >= 0 && row < a.tokens;
  const bool known = mine && p0 + tok < a.positions;
  // this thread's dims are 4 (sub + kLanes i) .. + 3, i < kVec: neighbours read neighbouring float4
  float4 cs[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    cs[i] = known ? *reinterpret_cast<const float4*>(a.rope + (int64_t)(p0 + tok) * (D / 2) + 2 * (sub + kLanes * i))
                  : make_float4(0.f, 0.f, 0.f, 0.f);
  const int kv = a.c.kv_heads, tiles = a.heads + 2 * kv;
  __shared__ float part[2][kAppendThreads / 32];
  int flip = 0;
  for (int tile = blockIdx.y; tile < tiles; tile += gridDim.y) {
    float4 x[kVec];
    const float* src = a.qkv + row * a.row_stride + (int64_t)tile * D;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      x[i] = known ? __ldcs(reinterpret_cast<const float4*>(src + 4 * (sub + kLanes * i))) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (tile < a.heads + kv) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float4 v = x[i], r = cs[i];
        x[i] = make_float4(__fsub_rn(__fmul_rn(v.x, r.x), __fmul_rn(v.y, r.y)), __fadd_rn(__fmul_rn(v.x, r.y), __fmul_rn(v.y, r.x)),
                           __fsub_rn(__fmul_rn(v.z, r.z), __fmul_rn(v.w, r.w)), __fadd_rn(__fmul_rn(v.z, r.w), __fmul_rn(v.w, r.z)));
      }
    }
    if (tile < a.heads) {
      if (mine)
#pragma unroll
        for (int i = 0; i < kVec; ++i) store4(a.q, a.q_type, (row * a.heads + tile) * D + 4 * (sub + kLanes * i), x[i]);
      continue;
    }
    const bool is_k = tile < a.heads + kv;
    const int head = tile - a.heads - (is_k ? 0 : kv);
    const int id = kv8_block_id(a.c, a.t, b, head, blk);
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      m = fmaxf(m, fmaxf(fmaxf(finite_abs(x[i].x), finite_abs(x[i].y)), fmaxf(finite_abs(x[i].z), finite_abs(x[i].w))));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 31) == 0) part[flip][tid >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) m = fmaxf(m, part[flip][w]);
    flip ^= 1;  // the next tile's maxima go to the other half: one barrier a tile
    if (id < 0 || p0 >= a.positions) continue;
    float* scale = (is_k ? a.c.ks : a.c.vs) + id;
    uint8_t* codes = (is_k ? a.c.k : a.c.v) + (int64_t)id * (kKvBlock * D);
    float s = kv8_scale(m);
    if (slot0 > 0) {
      const float before = *scale;
      __syncthreads();  // everybody has read the scale that thread 0 replaces
      if (before > s) s = before;
      if (s != before && tok < slot0) {  // thread (tok, sub) rescales the same dims of an earlier token
        const float ratio = before * kv8_inverse(s);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          uint32_t* w = reinterpret_cast<uint32_t*>(codes + tok * D + 4 * (sub + kLanes * i));
          uint32_t lo, hi;
          e4m3x4_f16(*w, lo, hi);
          const float2 f = __half22float2(*reinterpret_cast<__half2*>(&lo)), g = __half22float2(*reinterpret_cast<__half2*>(&hi));
          *w = e4m3x4(f.x * ratio, f.y * ratio, g.x * ratio, g.y * ratio);
        }
      }
    }
    if (tid == 0) *scale = s;
    if (known) {
      const float inv = kv8_inverse(s);
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        *reinterpret_cast<uint32_t*>(codes + (slot0 + tok) * D + 4 * (sub + kLanes * i)) =
            e4m3x4(x[i].x * inv, x[i].y * inv, x[i].z * inv, x[i].w * inv);
    }
  }
}

// One token for each sequence: a warp takes one of its heads + 2 kv_heads tiles of D values, so a
// step's work is one load, one shuffle reduction and one store deep, without a search or a barrier.
// The block's earlier tokens are only read if its scale grows (then by the whole warp, a token at a
// time). What bounds it is the chain of dependent loads (start, rope row and page, scale). For 64
// sequences of 32 + 64 heads of 128 it takes 3.0 us, where the kernel above, its CTAs of 16 tokens
// mostly idle, took 9.6.
template <int D>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_one_kernel(const AppendArgs a) {
  constexpr int kVec = D / 64;  // 2 or 1 pairs of values of a lane: dims 2 lane + 64 i
  const int lane = threadIdx.x & 31, kv = a.c.kv_heads, tiles = a.heads + 2 * kv;
  const int64_t i = (int64_t)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  if (i >= (int64_t)a.batch * tiles) return;
  const int b = (int)(i / tiles), tile = (int)(i % tiles);
  const float* src = a.qkv + b * a.row_stride + (int64_t)tile * D + 2 * lane;
  float2 x[kVec];
#pragma unroll
  for (int c = 0; c < kVec; ++c) x[c] = __ldcs(reinterpret_cast<const float2*>(src + 64 * c));
  const int pos = __ldg(a.starts + b);
  const bool known = pos >= 0 && pos < a.positions;
  const bool is_q = tile < a.heads, is_k = !is_q && tile < a.heads + kv;
  const int head = tile - a.heads - (is_k ? 0 : kv), blk = pos / kKvBlock, slot = pos % kKvBlock;
  const int id = is_q || pos < 0 ? -1 : kv8_block_id(a.c, a.t, b, head, blk);
#pragma unroll
  for (int c = 0; c < kVec; ++c) {
    const float2 v = x[c];
    if (!known) x[c] = make_float2(0.f, 0.f);
    if (known && (is_q || is_k)) {
      const float2 r = __ldg(a.rope + (int64_t)pos * (D / 2) + lane + 32 * c);
      x[c] = make_float2(__fsub_rn(__fmul_rn(v.x, r.x), __fmul_rn(v.y, r.y)), __fadd_rn(__fmul_rn(v.x, r.y), __fmul_rn(v.y, r.x)));
    }
  }
  if (is_q) {
#pragma unroll
    for (int c = 0; c < kVec; ++c) {
      const int64_t at = ((int64_t)b * a.heads + tile) * D + 2 * lane + 64 * c;
      if (a.q_type == J4B_F32)
        *reinterpret_cast<float2*>(static_cast<float*>(a.q) + at) = x[c];
      else
        *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(a.q) + at) = __floats2bfloat162_rn(x[c].x, x[c].y);
    }
    return;
  }
  if (id < 0 || !known) return;
  float* scale = (is_k ? a.c.ks : a.c.vs) + id;
  uint8_t* codes = (is_k ? a.c.k : a.c.v) + (int64_t)id * (kKvBlock * D);
  const float before = slot > 0 ? *scale : 0.f;
  float m = 0.f;
#pragma unroll
  for (int c = 0; c < kVec; ++c) m = fmaxf(m, fmaxf(finite_abs(x[c].x), finite_abs(x[c].y)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float s = kv8_scale(m);
  if (slot > 0 && before >= s) s = before;
  if (slot > 0 && s != before) {
    const float ratio = before * kv8_inverse(s);
    for (int w = lane; w < slot * (D / 4); w += 32) {
      uint32_t* word = reinterpret_cast<uint32_t*>(codes) + w;
      uint32_t lo, hi;
      e4m3x4_f16(*word, lo, hi);
      const float2 f = __half22float2(*reinterpret_cast<__half2*>(&lo)), g = __half22float2(*reinterpret_cast<__half2*>(&hi));
      *word = e4m3x4(f.x * ratio, f.y * ratio, g.x * ratio, g.y * ratio);
    }
  }
  __syncwarp();  // every lane has read the scale
  if (lane == 0) *scale = s;
  if (known) {
    const float inv = kv8_inverse(s);
#pragma unroll
    for (int c = 0; c < kVec; ++c)
      *reinterpret_cast<uint16_t*>(codes + slot * D + 2 * lane + 64 * c) = (uint16_t)e4m3x2(x[c].x * inv, x[c].y * inv);
  }
}

// ---------------------------------------------------------------------------------------------
// Page copies: move m takes the first blocks[m] blocks of every head of page src[m] to page dst[m],
// codes and scales, in every layer. The moves come by value (no copy of them to the device); a CTA
// takes one (move, layer, k or v, group of heads), a head's blocks being contiguous. Bound by HBM: 147
// pages of 64 tokens x 8 heads of 128 in 16 layers take 96.9 us, 6.37 TB/s.
constexpr int kMaxMoves = 256;
struct CopyArgs {
  uint8_t* codes[2];
  float* scales[2];
  int64_t pages;
  int kv_heads, bpp, block_bytes, heads_per;
  int src[kMaxMoves], dst[kMaxMoves], blocks[kMaxMoves];
};

__global__ void __launch_bounds__(256) kv8_copy_kernel(const __grid_constant__ CopyArgs a) {
  const int m = blockIdx.x, kv = blockIdx.y & 1;
  const int64_t layer = blockIdx.y >> 1;
  const int h0 = blockIdx.z * a.heads_per, h1 = min(a.kv_heads, h0 + a.heads_per);
  const int nb = a.blocks[m];
  const int64_t from = ((layer * a.pages + a.src[m]) * a.kv_heads + h0) * a.bpp;
  const int64_t to = ((layer * a.pages + a.dst[m]) * a.kv_heads + h0) * a.bpp;
  const uint4* s = reinterpret_cast<const uint4*>(a.codes[kv] + from * a.block_bytes);
  uint4* d = reinterpret_cast<uint4*>(a.codes[kv] + to * a.block_bytes);
  const int per_head = nb * (a.block_bytes / 16), stride = a.bpp * (a.block_bytes / 16);
  const int total = per_head * (h1 - h0);
  for (int base = threadIdx.x; base < total; base += 256 * 4) {
    uint4 v[4];
    int at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + u * 256;
      at[u] = i < total ? i / per_head * stride + i % per_head : -1;
      if (at[u] >= 0) v[u] = __ldcs(s + at[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (at[u] >= 0) __stcs(d + at[u], v[u]);
  }
  for (int i = threadIdx.x; i < nb * (h1 - h0); i += 256) {
    const int at = i / nb * a.bpp + i % nb;
    a.scales[kv][to + at] = a.scales[kv][from + at];
  }
}

}  // namespace

int kv8_check(const j4b_kv8_cache* c, int64_t layer, Kv8View* view, int* dev) {
  J4B_REQUIRE(c, "kv8: null cache description");
  J4B_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "kv8: head_dim must be 64 or 128, got %d", c->head_dim);
  J4B_REQUIRE(c->page > 0 && c->page % kKvBlock == 0 && c->page <= 4096, "kv8: page must be a multiple of 16 up to 4096, got %d", c->page);
  J4B_REQUIRE(c->kv_heads > 0 && c->kv_heads <= 4096, "kv8: kv_heads must lie in [1, 4096], got %d", c->kv_heads);
  J4B_REQUIRE(c->layers > 0 && c->pages > 0, "kv8: layers and pages must be positive");
  const int bpp = c->page / kKvBlock;
  // rows of head_dim codes are numbered in 32 bits (coordinates of the copies)
  const int64_t blocks = c->pages <= 0x7ffffffLL / ((int64_t)c->kv_heads * bpp) ? c->pages * c->kv_heads * bpp : -1;
  J4B_REQUIRE(blocks > 0, "kv8: a layer must hold fewer than 2^31 rows (token and head)");
  J4B_REQUIRE(layer >= 0 && layer < c->layers, "kv8: layer %lld outside [0, %lld)", (long long)layer, (long long)c->layers);
  J4B_REQUIRE(c->k && c->v && c->k_scale && c->v_scale && ((c->k | c->v) & 15) == 0 && ((c->k_scale | c->v_scale) & 3) == 0,
              "kv8: codes must be 16-byte aligned, scales 4-byte");
  const int st = device_of((const void*)(uintptr_t)c->k, dev);
  if (st) return st;
  const int64_t code_at = layer * blocks * kKvBlock * c->head_dim, scale_at = layer * blocks;
  *view = {(uint8_t*)(uintptr_t)c->k + code_at, (uint8_t*)(uintptr_t)c->v + code_at, (float*)(uintptr_t)c->k_scale + scale_at,
           (float*)(uintptr_t)c->v_scale + scale_at, (int)c->pages, c->kv_heads, bpp};
  return J4B_OK;
}

}  // namespace j4b

using namespace j4b;

extern "C" int j4b_kv8_append(const j4b_kv8_cache* cache, int64_t layer, j4b_buf qkv, int64_t qkv_stride, int64_t tokens,
                              int64_t heads, j4b_buf rope, int64_t rope_positions, j4b_buf table, int64_t table_stride,
                              int64_t table_width, j4b_buf starts, j4b_buf offsets, int64_t batch, j4b_buf q_out, int q_type,
                              j4b_stream s) {
  Kv8View view;
  int dev = 0;
  if (const int st = kv8_check(cache, layer, &view, &dev)) return st;
  const int dim = cache->head_dim;
  J4B_REQUIRE(heads > 0 && heads <= 65536 && heads % cache->kv_heads == 0, "kv8 append: heads (%lld) must be a multiple of kv_heads (%d)",
              (long long)heads, cache->kv_heads);
  J4B_REQUIRE(batch >= 0 && batch <= 0xffffff && tokens >= 0 && tokens <= 0x7fffffff, "kv8 append: bad batch or token count");
  J4B_REQUIRE(offsets || tokens == batch, "kv8 append: without offsets there is one token for each sequence (%lld tokens, %lld sequences)",
              (long long)tokens, (long long)batch);
  J4B_REQUIRE(qkv_stride >= (heads + 2 * cache->kv_heads) * dim && qkv_stride % 4 == 0,
              "kv8 append: qkv rows must hold (heads + 2 kv_heads) * head_dim floats, a multiple of 4 apart");
  J4B_REQUIRE(q_type == J4B_F32 || q_type == J4B_BF16, "kv8 append: q type must be f32 or bf16, got %d", q_type);
  J4B_REQUIRE(table_width > 0 && table_width <= 0x7ffffff && table_stride >= table_width, "kv8 append: bad page table shape");
  J4B_REQUIRE(rope_positions > 0, "kv8 append: empty rope table");
  if (tokens == 0 || batch == 0) return J4B_OK;
  J4B_REQUIRE(qkv && rope && table && starts && q_out && ((qkv | rope | q_out) & 15) == 0 && ((table | starts | offsets) & 3) == 0,
              "kv8 append: misaligned or null buffers");
  DeviceGuard guard(dev);
  cudaStream_t stream = resolve_stream(dev, s);
  const AppendArgs a = {view,
                        {(const int*)(uintptr_t)table, table_stride, (int)table_width},
                        (const float*)(uintptr_t)qkv,
                        qkv_stride,
                        tokens,
                        (const float2*)(uintptr_t)rope,
                        rope_positions,
                        (const int*)(uintptr_t)starts,
                        (const int*)(uintptr_t)offsets,
                        (int)batch,
                        (int)heads,
                        (void*)(uintptr_t)q_out,
                        q_type};
  if (!offsets) {
    const int64_t ctas = (batch * (heads + 2 * cache->kv_heads) + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
    J4B_REQUIRE(ctas <= 0x7fffffffLL, "kv8 append: too many rows");
    if (dim == 128)
      kv8_append_one_kernel<128><<<(unsigned)ctas, kAppendThreads, 0, stream>>>(a);
    else
      kv8_append_one_kernel<64><<<(unsigned)ctas, kAppendThreads, 0, stream>>>(a);
    J4B_CHECK_LAUNCH("kv8_append_one_kernel");
    return J4B_OK;
  }
  // blocks that n tokens touch: at most (n + 14) / 16 + 1
  const int64_t items = std::min(tokens, (tokens + 14 * batch) / 16 + batch);
  const unsigned gy = (unsigned)std::min<int64_t>(heads + 2 * cache->kv_heads, 16);
  if (dim == 128)
    kv8_append_kernel<128><<<dim3((unsigned)items, gy), kAppendThreads, 0, stream>>>(a);
  else
    kv8_append_kernel<64><<<dim3((unsigned)items, gy), kAppendThreads, 0, stream>>>(a);
  J4B_CHECK_LAUNCH("kv8_append_kernel");
  return J4B_OK;
}

extern "C" int j4b_kv8_copy_pages(const j4b_kv8_cache* cache, int64_t moves, const int32_t* src, const int32_t* dst, const int32_t* tokens,
                                  j4b_stream s) {
  Kv8View view;
  int dev = 0;
  if (const int st = kv8_check(cache, 0, &view, &dev)) return st;
  J4B_REQUIRE(moves >= 0 && (moves == 0 || (src && dst)), "kv8 copy: null move list");
  J4B_REQUIRE(cache->layers <= 32767, "kv8 copy: at most 32767 layers");
  for (int64_t i = 0; i < moves; ++i) {
    J4B_REQUIRE(src[i] >= 0 && src[i] < cache->pages && dst[i] >= 0 && dst[i] < cache->pages && src[i] != dst[i],
                "kv8 copy: move %lld (page %d to %d) outside [0, %lld) or onto itself", (long long)i, src[i], dst[i], (long long)cache->pages);
    J4B_REQUIRE(!tokens || (tokens[i] >= 0 && tokens[i] <= cache->page), "kv8 copy: move %lld copies %d tokens of a page of %d",
                (long long)i, tokens ? tokens[i] : 0, cache->page);
  }
  // moves run at the same time: no page may be written twice, or written and read
  try {
    std::vector<int32_t> to(dst, dst + moves);
    std::sort(to.begin(), to.end());
    for (int64_t i = 0; i < moves; ++i) {
      J4B_REQUIRE(i == 0 || to[i] != to[i - 1], "kv8 copy: page %d is written twice", to[i]);
      J4B_REQUIRE(!std::binary_search(to.begin(), to.end(), src[i]), "kv8 copy: page %d is both read and written", src[i]);
    }
  } catch (const std::bad_alloc&) {
    return set_error(J4B_ENOMEM, "kv8 copy: out of host memory");
  }
  DeviceGuard guard(dev);
  cudaStream_t stream = resolve_stream(dev, s);
  CopyArgs a;
  a.codes[0] = view.k;
  a.codes[1] = view.v;
  a.scales[0] = view.ks;
  a.scales[1] = view.vs;
  a.pages = cache->pages;
  a.kv_heads = cache->kv_heads;
  a.bpp = view.bpp;
  a.block_bytes = kKvBlock * cache->head_dim;
  a.heads_per = std::max(1, 32768 / (cache->page * cache->head_dim));
  for (int64_t at = 0; at < moves; at += kMaxMoves) {
    const int n = (int)std::min<int64_t>(kMaxMoves, moves - at);
    for (int i = 0; i < n; ++i) {
      a.src[i] = src[at + i];
      a.dst[i] = dst[at + i];
      a.blocks[i] = tokens ? (tokens[at + i] + kKvBlock - 1) / kKvBlock : view.bpp;
    }
    const unsigned gz = (unsigned)((a.kv_heads + a.heads_per - 1) / a.heads_per);
    kv8_copy_kernel<<<dim3((unsigned)n, (unsigned)(2 * cache->layers), gz), 256, 0, stream>>>(a);
    J4B_CHECK_LAUNCH("kv8_copy_kernel");
  }
  return J4B_OK;
}
