// Causal attention of ragged query chunks over the 8-bit paged KV cache (format: kv8_common.cuh) on
// the tcgen05 tensor cores.
//
// The rows of one (sequence, kv head) are its queries times the heads of the group (row r: query
// r / group, head r % group), so one key tile serves every head that shares it. A CTA takes 256
// consecutive rows as two tiles of 128, each the M of its MMAs, and walks the blocks that any of
// its rows sees, 8 blocks (128 keys) at a time:
//   S_i = Q_i K^T   (Q, K f16 in shared memory; e4m3 codes are exact in f16)        -> TMEM
//   P_i = 2^(S_i - m + w)  by the tile's 128 softmax threads, one a row             -> TMEM, over S_i
//   O_i += P_i V    (P from TMEM, V f16 codes in shared memory, dims contiguous)    -> TMEM
// Scales never touch the operands: a block's key scale multiplies its scores, and its value scale,
// over the largest seen, is the w of its probabilities (both powers of two). The running maximum m
// moves only when a row outgrows it by 2^kLazy, so O is seldom rescaled.
//
// Warps: 0-3 and 4-7 softmax of tile 0 and 1; 8-11 bring pages: each thread loads 16-code pieces of
// the next tile while it turns this one's into the swizzled f16 operands; 12 issues the MMAs. S of
// one tile is computed while the other's softmax runs.
#include <algorithm>
#include <cmath>

#include "kv8_common.cuh"
#include "tc_common.cuh"

namespace j4b {
namespace {

constexpr int kRows = 128;           // of a tile
constexpr int kKeys = 128;           // of a key tile
constexpr int kTileBlocks = kKeys / kKvBlock;
constexpr int kThreads = 13 * 32;
constexpr int kStages = 2;           // of K and of V
constexpr int kInfos = 4;            // of what is known of a key tile: the softmax may be two behind
constexpr float kLazy = 5.f;         // log2: P <= 2^(kShift + kLazy) = 2^15, inside f16
constexpr int kShift = 10;           // log2: keeps f16's bits for blocks of small value scale

// What the softmax needs of a key tile.
struct TileInfo {
  int pos[kTileBlocks];    // first position of each block; far past every row where none is there
  float ks[kTileBlocks];
  int ev[kTileBlocks];     // exponent of the value scale
  unsigned nan[kKeys / 32];  // tokens whose values hold a NaN
};

template <int D>
struct Smem {
  static constexpr int kQ = kRows * D * 2;       // bytes of a query tile
  static constexpr int kOperand = kKeys * D * 2; // of K or V
  static constexpr int kBytes = 2 * kQ + 2 * kStages * kOperand + kInfos * (int)sizeof(TileInfo) + 1024;
};

// kind::f16 with f16 operands; b_rows: B's shared-memory rows run along N (its 16-bit "MN-major" form)
constexpr uint32_t idesc_f16(int m, int n, bool b_rows) {
  return (1u << 4) | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// B with rows along N, 128-byte swizzle: rows of 64 n (128 bytes), 8 rows (k) 1024 bytes, next 8 k
// `SBO` = 1024 bytes on, next 64 n `LBO` = `n_stride` bytes on
__device__ __forceinline__ uint64_t rows_sw128(uint32_t at, uint32_t n_stride) {
  return (uint64_t)((at >> 4) & 0x3FFFu) | ((uint64_t)(n_stride >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
// A from TMEM
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  const uint32_t z = 0;
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(z));
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
      "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};\n" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};\n" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void to_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Which key tiles a row tile takes: [begin, end) of the CTA's list.
struct Range {
  int begin, end;
  __device__ __forceinline__ bool has(int j) const { return j >= begin && j < end; }
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1) kv8_prefill_kernel(const AttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_smem(smem_raw);
  uint8_t* sq = smem;                                       // [2 tiles]
  uint8_t* sk = smem + 2 * Smem<D>::kQ;                     // [stage][K | V]
  TileInfo* infos = reinterpret_cast<TileInfo*>(sk + 2 * kStages * Smem<D>::kOperand);
  __shared__ uint64_t q_ready[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2], p_ready[2], o_full[2], info_full[kInfos];
  __shared__ uint32_t tmem_slot;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y;
  // the last rows of a sequence see the most keys: they go first
  const Kv8Place at = kv8_find<kThreads>(
      a.batch, [&](int b) -> int64_t { return ((int64_t)max(0, a.offsets[b + 1] - a.offsets[b]) * a.group + 2 * kRows - 1) / (2 * kRows); },
      [&](int64_t total) -> int64_t { return total > (int64_t)blockIdx.x ? total - 1 - (int64_t)blockIdx.x : total; });
  if (at.seq < 0) return;
  const int b = at.seq, row0 = a.offsets[b], n = a.offsets[b + 1] - row0, len = __ldg(a.lengths + b);
  const int64_t total_rows = (int64_t)n * a.group, r0 = at.at * (2 * kRows);
  const int pos0 = len - n;  // position of query 0 (queries before the cache see nothing)
  // positions of a tile's first and last row
  auto first_of = [&](int i) { return pos0 + (int)((r0 + i * kRows) / a.group); };
  auto last_of = [&](int i) { return min(len - 1, pos0 + (int)((min(total_rows, r0 + (i + 1) * kRows) - 1) / a.group)); };
  const int tiles = total_rows > r0 + kRows ? 2 : 1;
  const Span span = span_of(max(0, first_of(0)), last_of(tiles - 1), a.window, a.sinks);
  const int nb = max(0, span.count()), nt = (nb + kTileBlocks - 1) / kTileBlocks;
  // a tile leaves out key tiles past its last row, and those before its first row's window
  auto range_of = [&](int i) -> Range {
    if (i >= tiles) return {0, 0};
    const Span s = span_of(max(0, first_of(i)), last_of(i), a.window, a.sinks);
    if (s.count() <= 0) return {0, 0};
    const int end = span.sink_blocks + max(0, s.end - span.from);  // blocks of the list up to the tile's last
    // with sinks the tile also takes the list's first blocks, so it starts at 0
    const int begin = a.sinks > 0 ? 0 : span.sink_blocks + max(0, s.from - span.from);
    return {begin / kTileBlocks, (max(end, span.sink_blocks) + kTileBlocks - 1) / kTileBlocks};
  };
  const Range range[2] = {range_of(0), range_of(1)};

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(&q_ready[i], kRows);
      bar_init(&s_full[i], 1);
      bar_init(&p_ready[i], kRows);
      bar_init(&o_full[i], 1);
    }
    for (int s = 0; s < kStages; ++s) {
      bar_init(&k_full[s], 128);
      bar_init(&v_full[s], 128);
      bar_init(&k_empty[s], 1);
      bar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < kInfos; ++s) bar_init(&info_full[s], 128);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;  // S0, S1 at columns 0, 128 (P over them); O0, O1 at 256, 384
  bool ok = true;

  if (warp < 8) {
    // ---- softmax of tile i, one row a thread ----
    const int i = warp >> 2, r = tid & 127;
    const Range rg = range[i];
    const int64_t gr = r0 + i * kRows + r;
    const int tok = (int)(gr / a.group), gh = head * a.group + (int)(gr % a.group);
    const bool valid = gr < total_rows && row0 + tok >= 0 && row0 + tok < a.tokens;
    const int qp = valid ? pos0 + tok : -1;
    const int lo = a.window > 0 ? max(0, qp - a.window + 1) : 0;
    // every valid row of the tile sees the positions [most_lo, least]
    const int least = first_of(i), most_lo = a.window > 0 ? max(0, last_of(i) - a.window + 1) : 0;
    // Q: each row by a power of two to a largest element in [2^11, 2^12), then f16 (bf16 is exact there)
    float factor = a.scale_log2;
    if (i < tiles) {
      const int64_t src = valid ? (int64_t)(row0 + tok) * a.q_stride + (int64_t)gh * D : 0;
      float most = 0.f;
      if (valid)
#pragma unroll 4
        for (int c = 0; c < D; c += 4) {
          const float4 x = load4(a.q, a.q_type, src + c);
          most = fmaxf(most, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
        }
      const int e = (int)(__float_as_uint(most) >> 23);
      const bool plain = e < 24 || e > 240;
      float up = plain ? 1.f : __uint_as_float((uint32_t)(254 - (e - 11)) << 23);
      factor *= plain ? 1.f : __uint_as_float((uint32_t)(e - 11) << 23);
      if (factor < 0.f) {  // the maxima below are taken before the factor
        factor = -factor;
        up = -up;
      }
      uint8_t* tile = sq + i * Smem<D>::kQ;
#pragma unroll 4
      for (int c = 0; c < D; c += 8) {
        uint4 h = make_uint4(0, 0, 0, 0);
        if (valid) {
          const float4 x = load4(a.q, a.q_type, src + c), y = load4(a.q, a.q_type, src + c + 4);
          h = make_uint4(h2(x.x * up, x.y * up), h2(x.z * up, x.w * up), h2(y.x * up, y.y * up), h2(y.z * up, y.w * up));
        }
        *reinterpret_cast<uint4*>(tile + (c >> 6) * (kRows * 128) + sw128_offset(r, c & 63)) = h;
      }
      to_async_proxy();
      bar_arrive(&q_ready[i]);
    }
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_at = lanes + (uint32_t)(i * 128), o_at = lanes + 256u + (uint32_t)(i * 128);
    float m = -INFINITY, l = 0.f;
    int eref = 0;  // exponent of the value scale that O is in units of
    uint32_t use = 0;
    for (int j = rg.begin; j < rg.end; ++j, ++use) {
      ok = ok && bar_wait(&info_full[j % kInfos], (uint32_t)(j / kInfos & 1));
      ok = ok && bar_wait(&s_full[i], use & 1);
      tc_fence_after();
      const TileInfo& info = infos[j % kInfos];
      int near = kNowhere, far = 0;
#pragma unroll
      for (int k = 0; k < kTileBlocks; ++k) {
        near = min(near, info.pos[k]);
        far = max(far, info.pos[k] + kKvBlock);
      }
      const bool all = far - 1 <= least && (near >= most_lo || far <= a.sinks);
      uint32_t v[32];
      // the row's maximum, and whether it sees a token with a NaN value (the operand holds 0 there)
      float mx = -INFINITY;
      bool bad = false;
#pragma unroll 1
      for (int c = 0; c < kKeys; c += 32) {
        tmem_ld32(s_at + (uint32_t)c, v);
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int blk = c / kKvBlock + h;
          float t = -INFINITY;
          if (all) {
#pragma unroll
            for (int e = 0; e < 16; ++e) t = fmaxf(t, __uint_as_float(v[16 * h + e]));
          } else {
            const int p = info.pos[blk];
            const unsigned nan = info.nan[c / 32] >> (16 * h);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const bool see = (p + e >= lo || p + e < a.sinks) && p + e <= qp;
              if (see) t = fmaxf(t, __uint_as_float(v[16 * h + e]));
              bad |= see && (nan >> e & 1);
            }
          }
          mx = fmaxf(mx, t * (factor * info.ks[blk]));
        }
      }
      if (all) bad = (info.nan[0] | info.nan[1] | info.nan[2] | info.nan[3]) != 0;
      if (bad) l = NAN;
      int ev = info.ev[0];
#pragma unroll
      for (int k = 1; k < kTileBlocks; ++k) ev = max(ev, info.ev[k]);
      const bool begin = j == rg.begin;
      const int enew = begin ? ev : max(eref, ev);
      float mnew = m;
      if (mx > m + kLazy || (m == -INFINITY && mx > m)) mnew = mx;
      if (begin) {
        m = mnew;
      } else if (__any_sync(0xffffffffu, mnew != m || enew != eref)) {
        const float cm = m == -INFINITY ? 0.f : exp2_ftz(m - mnew), co = cm * exp2_ftz((float)(eref - enew));
        l *= m == mnew ? 1.f : cm;
        m = mnew;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          tmem_ld32(o_at + (uint32_t)c, v);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * co);
          tmem_st32(o_at + (uint32_t)c, v);
        }
      }
      eref = enew;
      const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 1
      for (int c = 0; c < kKeys; c += 32) {
        tmem_ld32(s_at + (uint32_t)c, v);
        tmem_ld_wait();
        uint32_t p[16];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int blk = c / kKvBlock + h;
          const float f = factor * info.ks[blk];
          const int w = max(-60, info.ev[blk] - eref) + kShift;
          const float add = (float)w - base;
          const int p0 = info.pos[blk];
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float x = exp2_ftz(fmaf(__uint_as_float(v[16 * h + e]), f, add)), y = exp2_ftz(fmaf(__uint_as_float(v[16 * h + e + 1]), f, add));
            if (!all) {
              if (!((p0 + e >= lo || p0 + e < a.sinks) && p0 + e <= qp)) x = 0.f;
              if (!((p0 + e + 1 >= lo || p0 + e + 1 < a.sinks) && p0 + e + 1 <= qp)) y = 0.f;
            }
            sum += x + y;
            p[8 * h + e / 2] = h2(x, y);
          }
          l = fmaf(sum, __uint_as_float((uint32_t)(127 - w) << 23), l);
        }
        tmem_st16(s_at + (uint32_t)(c / 2), p);
      }
      tmem_st_wait();
      tc_fence_before();
      bar_arrive(&p_ready[i]);
    }
    // the output row
    if (rg.end > rg.begin) {
      ok = ok && bar_wait(&o_full[i], 0);
      tc_fence_after();
    }
    const float inv = m == -INFINITY ? 0.f : exp2_ftz((float)(eref - kShift)) / l;
    const int64_t dst = ((int64_t)(row0 + tok) * a.heads + gh) * D;
#pragma unroll 1
    for (int c = 0; c < D && i < tiles; c += 32) {
      uint32_t v[32];
      if (rg.end > rg.begin) {
        tmem_ld32(o_at + (uint32_t)c, v);
        tmem_ld_wait();
      }
      if (valid) {
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 x = m == -INFINITY ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(__uint_as_float(v[e]) * inv, __uint_as_float(v[e + 1]) * inv,
                                                                                                  __uint_as_float(v[e + 2]) * inv, __uint_as_float(v[e + 3]) * inv);
          store4(a.out, a.out_type, dst + c + e, x);
        }
      }
    }
  } else if (warp < 12) {
    // ---- pages to operands: this warp the rows 32 w .. + 31 (2 blocks) of each key tile ----
    const int w = warp - 8;
    constexpr int kHalves = D / 64, kPieces = 4 * kHalves;  // 16-code pieces of a thread, K or V
    // piece x: row 32 w + 8 (x / kHalves) + lane / 4, codes 64 (x % kHalves) + 16 (lane % 4): 8 lanes of
    // a store phase are 2 rows x 4 pieces, whose swizzled places cover all banks
    const int pr = lane >> 2, pc = lane & 3;
    auto block_at = [&](int j, int k) {  // block 2 w + k of tile j
      const int x = j * kTileBlocks + 2 * w + k;
      return x < nb ? span.block(x) : -1;
    };
    auto id_at = [&](int blk) { return blk < 0 ? -1 : kv8_block_id(a.c, a.t, b, head, blk); };
    auto load = [&](const uint8_t* codes, const int (&id)[2], uint4 (&dst)[kPieces]) {
#pragma unroll
      for (int x = 0; x < kPieces; ++x) {
        const int row = 8 * (x / kHalves) + pr, k = row >> 4;  // of the warp's 32
        dst[x] = id[k] < 0 ? make_uint4(0, 0, 0, 0)
                           : __ldg(reinterpret_cast<const uint4*>(codes + (int64_t)id[k] * (kKvBlock * D) + (row & 15) * D + 64 * (x % kHalves) + 16 * pc));
      }
    };
    auto store = [&](uint8_t* tile, const uint4 (&src)[kPieces]) {
#pragma unroll
      for (int x = 0; x < kPieces; ++x) {
        const int row = 32 * w + 8 * (x / kHalves) + pr;
        uint4 lo, hi;
        e4m3x4_f16(src[x].x, lo.x, lo.y);
        e4m3x4_f16(src[x].y, lo.z, lo.w);
        e4m3x4_f16(src[x].z, hi.x, hi.y);
        e4m3x4_f16(src[x].w, hi.z, hi.w);
        uint8_t* half = tile + (x % kHalves) * (kKeys * 128);
        *reinterpret_cast<uint4*>(half + sw128_offset(row, 16 * pc)) = lo;
        *reinterpret_cast<uint4*>(half + sw128_offset(row, 16 * pc + 8)) = hi;
      }
    };
    int blk[2] = {block_at(0, 0), block_at(0, 1)};
    int id[2] = {id_at(blk[0]), id_at(blk[1])};
    uint4 kr[kPieces], vr[kPieces];
    float ks = 1.f, vs = 0.f;
    auto scales = [&] {
      if (lane < 2 && id[lane & 1] >= 0) {
        ks = __ldg(a.c.ks + id[lane & 1]);
        vs = __ldg(a.c.vs + id[lane & 1]);
      } else {
        ks = 1.f;
        vs = 0.f;
      }
    };
    load(a.c.k, id, kr);
    load(a.c.v, id, vr);
    scales();
    int nblk[2] = {block_at(1, 0), block_at(1, 1)};
    int nid[2] = {id_at(nblk[0]), id_at(nblk[1])};
    for (int j = 0; j < nt; ++j) {
      const int s = j % kStages;
      const uint32_t parity = (uint32_t)(j / kStages - 1) & 1;
      uint8_t* kt = sk + s * 2 * Smem<D>::kOperand;
      TileInfo& info = infos[j % kInfos];
      if (j >= kStages) ok = ok && bar_wait(&k_empty[s], parity);
      store(kt, kr);
      if (lane < 2) {
        const int k = 2 * w + lane;
        info.pos[k] = id[lane] < 0 ? kNowhere : blk[lane] * kKvBlock;
        info.ks[k] = ks;
        info.ev[k] = (int)(__float_as_uint(vs) >> 23) - 127;
      }
      // the values' tokens past the length hold anything; NaNs go to the info, as zeros to the operand
      {
        unsigned nan = 0;
#pragma unroll
        for (int x = 0; x < kPieces; ++x) {
          const int row = 8 * (x / kHalves) + pr, k = row >> 4;
          if (blk[k] * kKvBlock + (row & 15) >= len) vr[x] = make_uint4(0, 0, 0, 0);
          uint32_t* q = reinterpret_cast<uint32_t*>(&vr[x]);
          uint32_t any = 0;
#pragma unroll
          for (int y = 0; y < 4; ++y) any |= ((q[y] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          if (any) {
            nan |= 1u << row;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t bytes = (((q[y] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
              q[y] &= ~(bytes * 0xffu);
            }
          }
        }
        nan = __reduce_or_sync(0xffffffffu, nan);
        if (lane == 0) info.nan[w] = nan;
      }
      to_async_proxy();
      bar_arrive(&k_full[s]);
      bar_arrive(&info_full[j % kInfos]);
      if (j >= kStages) ok = ok && bar_wait(&v_empty[s], parity);
      store(kt + Smem<D>::kOperand, vr);
      to_async_proxy();
      bar_arrive(&v_full[s]);
      blk[0] = nblk[0], blk[1] = nblk[1], id[0] = nid[0], id[1] = nid[1];
      if (j + 1 < nt) {
        load(a.c.k, id, kr);
        load(a.c.v, id, vr);
        scales();
        nblk[0] = block_at(j + 2, 0), nblk[1] = block_at(j + 2, 1);
        nid[0] = id_at(nblk[0]), nid[1] = id_at(nblk[1]);
      }
    }
  } else if (lane == 0) {
    // ---- the MMAs ----
    constexpr uint32_t is = idesc_f16(kRows, kKeys, false), io = idesc_f16(kRows, D, true);
    for (int i = 0; i < tiles; ++i) ok = ok && bar_wait(&q_ready[i], 0);
    tc_fence_after();
    uint32_t uses[2] = {0, 0};
    for (int j = -1; j < nt && ok; ++j) {
      if (j + 1 < nt) ok = ok && bar_wait(&k_full[(j + 1) % kStages], (uint32_t)((j + 1) / kStages & 1));
      if (j >= 0) ok = ok && bar_wait(&v_full[j % kStages], (uint32_t)(j / kStages & 1));
      tc_fence_after();
      for (int i = 0; i < tiles; ++i) {
        const uint32_t s_at = tmem + (uint32_t)(i * 128), o_at = tmem + 256u + (uint32_t)(i * 128);
        if (range[i].has(j)) {
          ok = ok && bar_wait(&p_ready[i], uses[i]++ & 1);
          tc_fence_after();
          const uint32_t vt = saddr(sk + (j % kStages) * 2 * Smem<D>::kOperand + Smem<D>::kOperand);
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)  // 16 keys: 8 columns of P, 2 groups of 8 rows of V
            umma_ts(o_at, s_at + 8u * k, rows_sw128(vt + k * 2048, kKeys * 128), io, (j > range[i].begin || k > 0) ? 1u : 0u);
          if (j + 1 == range[i].end) umma_commit(&o_full[i]);
        }
        if (range[i].has(j + 1)) {
          const uint32_t kt = saddr(sk + ((j + 1) % kStages) * 2 * Smem<D>::kOperand), qt = saddr(sq + i * Smem<D>::kQ);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k >> 2) * (kRows * 128) + (k & 3) * 32;  // kRows == kKeys
            umma_bf16(s_at, kmajor_sw128(qt + off), kmajor_sw128(kt + off), is, k > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[i]);
        }
      }
      if (j + 1 < nt) umma_commit(&k_empty[(j + 1) % kStages]);
      if (j >= 0) umma_commit(&v_empty[j % kStages]);
    }
  }
  if (!ok) *a.timeout = 1;
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

template <int D>
int launch_prefill(const AttnArgs& a, int dev, cudaStream_t stream) {
  static bool done[kMaxDevices] = {};
  if (!done[dev]) {
    J4B_CUDA(cudaFuncSetAttribute(kv8_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::kBytes), "cudaFuncSetAttribute");
    done[dev] = true;
  }
  const int64_t rows = a.tokens * a.group, tiles = std::min(rows, rows / (2 * kRows) + a.batch);
  J4B_REQUIRE(tiles <= 0x7fffffffLL, "kv8 prefill: too many rows");
  kv8_prefill_kernel<D><<<dim3((unsigned)tiles, (unsigned)a.c.kv_heads), kThreads, Smem<D>::kBytes, stream>>>(a);
  J4B_CHECK_LAUNCH("kv8_prefill_kernel");
  return J4B_OK;
}

}  // namespace
}  // namespace j4b

using namespace j4b;

extern "C" int j4b_kv8_attention_prefill(const j4b_kv8_cache* cache, int64_t layer, j4b_buf q, int q_type, int64_t q_stride, int64_t tokens,
                                         int64_t heads, j4b_buf offsets, j4b_buf table, int64_t table_stride, int64_t table_width,
                                         j4b_buf lengths, int64_t batch, int64_t window, int64_t sinks, double scale, j4b_buf out,
                                         int out_type, j4b_stream s) {
  AttnArgs a;
  int dev = 0;
  if (const int st = kv8_check_attention(cache, layer, q, q_type, q_stride, tokens, heads, table, table_stride, table_width, lengths, batch,
                                         window, sinks, scale, out, out_type, &a, &dev))
    return st;
  if (batch == 0 || tokens == 0) return J4B_OK;
  J4B_REQUIRE(offsets && (offsets & 3) == 0, "kv8 prefill: misaligned or null offsets");
  a.offsets = (const int*)(uintptr_t)offsets;
  DeviceGuard guard(dev);
  cudaStream_t stream = resolve_stream(dev, s);
  return cache->head_dim == 128 ? launch_prefill<128>(a, dev, stream) : launch_prefill<64>(a, dev, stream);
}
