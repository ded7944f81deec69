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
// the next tile while it turns this one's into the swizzled f16 operands; 12 issues the MMAs (13-15
// only fill up their warpgroup, so that its registers can go to the softmax, which holds a row of
// 128 scores). S of one tile is computed while the other's softmax runs.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv8_common.cuh"
#include "tc_common.cuh"

namespace j4b {
namespace {

constexpr int kRows = 128;           // of a tile
constexpr int kKeys = 128;           // of a key tile
constexpr int kTileBlocks = kKeys / kKvBlock;
constexpr int kThreads = 16 * 32;
constexpr int kStages = 2;           // of K and of V (their parity is counted with & 1)
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

// pairs of f32 in one instruction
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The positions that a row sees: [lo, qp] and [0, sinks) up to qp.
struct View {
  int lo, qp, sinks;
  static __device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 16 ? 0xffffu : (1u << n) - 1u; }
  // bit e: it sees position p + e, e < 16
  __device__ __forceinline__ uint32_t mask(int p) const { return below(qp + 1 - p) & (~below(lo - p) | below(sinks - p)); }
};

// A row's scores of a key tile, held in registers from TMEM until its probabilities go back there.
struct Row {
  uint32_t v[4][32];

  __device__ __forceinline__ void load(uint32_t s_at) {
#pragma unroll
    for (int c = 0; c < 4; ++c) tmem_ld32(s_at + 32u * c, v[c]);
    tmem_ld_wait();
  }
  // The largest score (times its factor). ALL: the row sees the whole tile; otherwise the scores of
  // what it does not see become -inf, and `bad` says whether it sees a token with a NaN value (the
  // operand holds 0 there).
  template <bool ALL>
  __device__ __forceinline__ float most(const TileInfo& info, const View& view, float factor, bool& bad) {
    float mx = -INFINITY;
    uint32_t found = 0;
#pragma unroll
    for (int k = 0; k < kTileBlocks; ++k) {
      uint32_t* x = v[k >> 1] + 16 * (k & 1);
      if (!ALL) {
        const uint32_t see = view.mask(info.pos[k]);
        found |= see & (info.nan[k >> 1] >> (16 * (k & 1)));
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!(see >> e & 1)) x[e] = 0xff800000u;
      }
      float t = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
#pragma unroll
      for (int e = 2; e < 16; e += 2) t = fmaxf(t, fmaxf(__uint_as_float(x[e]), __uint_as_float(x[e + 1])));
      const float f = factor * info.ks[k];
      mx = fmaxf(mx, t == -INFINITY ? t : t * f);
    }
    bad = ALL ? (info.nan[0] | info.nan[1] | info.nan[2] | info.nan[3]) != 0 : found != 0;
    return mx;
  }
  // The probabilities, in f16, each block's weighed by its value scale, go over the scores in TMEM;
  // returns their sum without the weights.
  template <bool ALL>
  __device__ __forceinline__ float store(uint32_t s_at, const TileInfo& info, float factor, float base, int eref) {
    float l = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t p[16];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = 2 * c + h;
        const uint32_t* x = v[c] + 16 * h;
        // -inf * 0 would be NaN: with a key scale of 0 the visible scores are 0 whatever the factor
        const float f = ALL ? factor * info.ks[k] : fmaxf(factor * info.ks[k], 1e-37f);
        const int w = max(-60, info.ev[k] - eref) + kShift;
        const uint64_t ff = pair(f, f), add = pair((float)w - base, (float)w - base);
        uint64_t sum = 0;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float2 y = unpair(fma2(pair(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), ff, add));
          y.x = exp2_ftz(y.x);
          y.y = exp2_ftz(y.y);
          sum = add2(sum, pair(y.x, y.y));
          p[8 * h + e / 2] = h2(y.x, y.y);
        }
        const float2 t = unpair(sum);
        l = fmaf(t.x + t.y, __uint_as_float((uint32_t)(127 - w) << 23), l);
      }
      tmem_st16(s_at + 16u * c, p);
    }
    return l;
  }
};

// Which key tiles a row tile takes: [begin, end) of the CTA's list.
struct Range {
  int begin, end;
  __device__ __forceinline__ bool has(int j) const { return j >= begin && j < end; }
};

// Registers of a thread by warpgroup: the launch's 4 x 128 shared out as 2 x 176 + 104 + 56.
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) kv8_prefill_kernel(const AttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_smem(smem_raw);
  uint8_t* sq = smem;                                       // [2 tiles]
  uint8_t* sk = smem + 2 * Smem<D>::kQ;                     // [stage][K | V]
  TileInfo* infos = reinterpret_cast<TileInfo*>(sk + 2 * kStages * Smem<D>::kOperand);
  __shared__ uint64_t q_ready[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2], p_ready[2], o_full[2], info_full[kInfos];
  __shared__ uint32_t tmem_slot;
  __shared__ float factors[2][kRows];
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
  const Range range0 = range_of(0), range1 = range_of(1);

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
    more_registers<176>();
    // ---- softmax of tile i, one row a thread ----
    const int i = warp >> 2, r = tid & 127;
    const Range rg = i ? range1 : range0;
    const int64_t gr = r0 + i * kRows + r;
    const int tok = (int)(gr / a.group), gh = head * a.group + (int)(gr % a.group);
    const bool valid = gr < total_rows && row0 + tok >= 0 && row0 + tok < a.tokens;
    const int qp = valid ? pos0 + tok : -1;
    const View view = {a.window > 0 ? max(0, qp - a.window + 1) : 0, qp, a.sinks};
    // every valid row of the tile sees the positions [most_lo, least]
    const int least = first_of(i), most_lo = a.window > 0 ? max(0, last_of(i) - a.window + 1) : 0;
    // Q: each row by a power of two to a largest element in [2^11, 2^12), then f16 (bf16 is exact
    // there); 8 lanes a row, 4 rows at a time
    float factor = 0.f;
    if (i < tiles) {
      uint8_t* tile = sq + i * Smem<D>::kQ;
      const int sub = lane & 7;
      auto rows = [&](auto type) {
        constexpr bool kF32 = decltype(type)::value == J4B_F32;
        constexpr int kWords = kF32 ? D / 32 : D / 64, kStep = kF32 ? 4 : 8;  // 16-byte pieces of a row and lane, rows in flight
#pragma unroll 1
        for (int k0 = 0; k0 < 8; k0 += kStep) {
          uint4 raw[kStep][kWords];
#pragma unroll
          for (int k = 0; k < kStep; ++k) {
            const int64_t g = r0 + i * kRows + (warp & 3) * 32 + 4 * (k0 + k) + (lane >> 3), row = row0 + g / a.group;
            const bool there = g < total_rows && row >= 0 && row < a.tokens;
            const int64_t src = row * a.q_stride + (int64_t)(head * a.group + (int)(g % a.group)) * D + 8 * sub;
#pragma unroll
            for (int c = 0; c < kWords; ++c)
              raw[k][c] = !there ? make_uint4(0, 0, 0, 0)
                          : kF32 ? __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(a.q) + src + 64 * (c >> 1) + 4 * (c & 1)))
                                 : __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + src + 64 * c));
          }
#pragma unroll
          for (int k = 0; k < kStep; ++k) {
            const int qr = (warp & 3) * 32 + 4 * (k0 + k) + (lane >> 3);
            float x[D / 8];
            float most = 0.f;
#pragma unroll
            for (int c = 0; c < kWords; ++c) {
              const uint32_t w[4] = {raw[k][c].x, raw[k][c].y, raw[k][c].z, raw[k][c].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (kF32) {
                  x[4 * c + e] = __uint_as_float(w[e]);
                } else {
                  x[8 * c + 2 * e] = __uint_as_float(w[e] << 16);
                  x[8 * c + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                }
              }
            }
#pragma unroll
            for (int e = 0; e < D / 8; ++e) most = fmaxf(most, fabsf(x[e]));
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const int e = (int)(__float_as_uint(most) >> 23);
            const bool plain = e < 24 || e > 240;
            float up = plain ? 1.f : __uint_as_float((uint32_t)(254 - (e - 11)) << 23);
            float f = plain ? a.scale_log2 : a.scale_log2 * __uint_as_float((uint32_t)(e - 11) << 23);
            if (f < 0.f) {  // maxima are taken before the factor
              f = -f;
              up = -up;
            }
            if (sub == 0) factors[i][qr] = f;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              const float* y = x + 8 * c;
              *reinterpret_cast<uint4*>(tile + c * (kRows * 128) + sw128_offset(qr, 8 * sub)) =
                  make_uint4(h2(y[0] * up, y[1] * up), h2(y[2] * up, y[3] * up), h2(y[4] * up, y[5] * up), h2(y[6] * up, y[7] * up));
            }
          }
        }
      };
      if (a.q_type == J4B_F32)
        rows(std::integral_constant<int, J4B_F32>{});
      else
        rows(std::integral_constant<int, J4B_BF16>{});
      to_async_proxy();
      bar_arrive(&q_ready[i]);
      __syncwarp();  // a warp wrote the factors of its own rows
      factor = factors[i][r];
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
      bool bad = false;
      Row row;
      row.load(s_at);
      const float mx = all ? row.most<true>(info, view, factor, bad) : row.most<false>(info, view, factor, bad);
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
        uint32_t v[32];
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
      l += all ? row.store<true>(s_at, info, factor, base, eref) : row.store<false>(s_at, info, factor, base, eref);
      tmem_st_wait();
      tc_fence_before();
      bar_arrive(&p_ready[i]);
    }
    // the output row
    if (rg.end > rg.begin) {
      ok = ok && bar_wait(&o_full[i], 0);
      tc_fence_after();
    }
    const int64_t out_row = valid ? ((int64_t)(row0 + tok) * a.heads + gh) * D : -1;
    const float inv = m == -INFINITY ? 0.f : exp2_ftz((float)(eref - kShift)) / l;
    // through the warp's rows of the query tile (its MMAs are done), so that the stores are whole
    // rows: 256 bytes of a row at a time, 16-byte pieces swizzled by the row
    uint8_t* stage = sq + i * Smem<D>::kQ + (warp & 3) * (32 * 2 * D);
    const bool f32 = a.out_type == J4B_F32;
    const int bytes = min(f32 ? 4 * D : 2 * D, 2 * D), passes = f32 ? 2 : 1;  // of a row and pass
#pragma unroll 1
    for (int pass = 0; pass < passes && i < tiles; ++pass) {
      __syncwarp();
#pragma unroll 1
      for (int c = pass * (D / 2); c < (f32 ? (pass + 1) * (D / 2) : D); c += 32) {
        uint32_t v[32];
        if (rg.end > rg.begin) {
          tmem_ld32(o_at + (uint32_t)c, v);
          tmem_ld_wait();
        }
        float x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = m == -INFINITY ? 0.f : __uint_as_float(v[e]) * inv;
        const int first = (f32 ? 4 * (c - pass * (D / 2)) : 2 * c) / 16;  // 16-byte piece of the row
        if (f32) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<float4*>(stage + lane * bytes + (((first + e) ^ (lane & 7)) << 4)) = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const __nv_bfloat162 t = __floats2bfloat162_rn(x[8 * e + 2 * y], x[8 * e + 2 * y + 1]);
              w[y] = *reinterpret_cast<const uint32_t*>(&t);
            }
            *reinterpret_cast<uint4*>(stage + lane * bytes + (((first + e) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      __syncwarp();
      constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;  // lanes of a row, rows of a store
      uint8_t* out = static_cast<uint8_t*>(a.out) + pass * bytes;
#pragma unroll 8
      for (int k = 0; k < 32 / kAtOnce; ++k) {
        const int qr = kAtOnce * k + lane / kLanes, piece = lane % kLanes;
        const int64_t dst = __shfl_sync(0xffffffffu, out_row, qr);
        if (dst >= 0)
          *reinterpret_cast<uint4*>(out + dst * (f32 ? 4 : 2) + 16 * piece) =
              *reinterpret_cast<const uint4*>(stage + qr * bytes + ((piece ^ (qr & 7)) << 4));
      }
    }
  } else if (warp < 12) {
    fewer_registers<104>();
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
  } else {
    fewer_registers<56>();
    if (warp == 12 && lane == 0) {
    // ---- the MMAs ----
    constexpr uint32_t is = idesc_f16(kRows, kKeys, false), io = idesc_f16(kRows, D, true);
    // descriptors count in 16-byte units: stepping one is an addition
    uint64_t qd = kmajor_sw128(saddr(sq)), kd = kmajor_sw128(saddr(sk)), vd = rows_sw128(saddr(sk) + Smem<D>::kOperand, kKeys * 128);
    constexpr uint32_t kStage = 2 * Smem<D>::kOperand / 16;
    for (int i = 0; i < tiles; ++i) ok = ok && bar_wait(&q_ready[i], 0);
    tc_fence_after();
    uint32_t uses0 = 0, uses1 = 0;
    for (int j = -1; j < nt && ok; ++j) {
      if (j + 1 < nt) ok = ok && bar_wait(&k_full[(j + 1) % kStages], (uint32_t)((j + 1) / kStages & 1));
      if (j >= 0) ok = ok && bar_wait(&v_full[j % kStages], (uint32_t)(j / kStages & 1));
      tc_fence_after();
      // opaque, or every step's descriptor is kept across the loop and spilled: the issue then waits for
      // local memory (8 x 2048: PV's 8 MMAs took 2 us to issue instead of 0.3)
      asm volatile("" : "+l"(qd), "+l"(kd), "+l"(vd));
      const uint64_t vt = vd + (uint32_t)(j & 1) * kStage, kt = kd + (uint32_t)((j + 1) & 1) * kStage;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Range rg = i ? range1 : range0;
        uint32_t& uses = i ? uses1 : uses0;
        const uint32_t s_at = tmem + (uint32_t)(i * 128), o_at = tmem + 256u + (uint32_t)(i * 128);
        if (rg.has(j)) {
          ok = ok && bar_wait(&p_ready[i], uses & 1);
          ++uses;
          tc_fence_after();
          const uint32_t later = j > rg.begin;
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)  // 16 keys: 8 columns of P, 2 groups of 8 rows of V
            umma_ts(o_at, s_at + 8u * k, vt + k * (2048 / 16), io, k > 0 ? 1u : later);
          if (j + 1 == rg.end) umma_commit(&o_full[i]);
        }
        if (rg.has(j + 1)) {
          const uint64_t qt = qd + (uint32_t)(i * Smem<D>::kQ / 16);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = ((k >> 2) * (kRows * 128) + (k & 3) * 32) / 16;  // kRows == kKeys
            umma_bf16(s_at, qt + off, kt + off, is, k > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[i]);
        }
      }
      if (j + 1 < nt) umma_commit(&k_empty[(j + 1) % kStages]);
      if (j >= 0) umma_commit(&v_empty[j % kStages]);
    }
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
