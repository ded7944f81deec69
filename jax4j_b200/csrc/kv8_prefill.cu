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
// over the largest that the row sees, is the w of its probabilities (both powers of two). The running maximum m
// moves only when f16 would not hold a row's probabilities, so O is seldom rescaled.
//
// Warps: 0-3 and 4-7 queries, softmax and output of tile 0 and 1; 8-11 bring pages: each thread loads
// 16-code pieces of the next tile while it turns this one's into the swizzled f16 operands; 12 issues
// the MMAs; 13 finds the next item, and writes the output of those that see nothing. S of one tile is
// computed while the other's softmax runs.
//
// Measured: 8 x 2048 causal, 32 heads of 128: 392 us, 701 TFLOP/s (a bf16 product of matrices reaches
// 1672); 8001 tokens under a window of 1024, 32/8 heads: 200 us. A step of 128 keys takes 2.3 us, of
// which the tensor cores work 0.6: it is a chain of softmax (1.6, its warps waiting on one another's
// issue slots, MUFU a third busy) and MMAs (0.7 from the last probability to the next scores). What
// shortened it most was fewer instructions in the softmax and page warps, which share 4 schedulers.
//
// One CTA an SM stays for the whole call and takes items (256 rows of a sequence and kv head): the
// pages and queries of the next item come while this one's last tiles are worked on. Items are
// numbered by how far from their sequence's end they lie, so the longest come first, and dealt out
// to the CTAs forth and back.
#include <algorithm>
#include <cmath>

#include "kv8_common.cuh"
#include "tc_common.cuh"

namespace j4b {
namespace {

constexpr int kRows = 128;           // of a tile
constexpr int kKeys = 128;           // of a key tile
constexpr int kTileBlocks = kKeys / kKvBlock;
constexpr int kThreads = 14 * 32;
constexpr int kStages = 2;           // of K and of V (their parity is counted with & 1)
constexpr int kInfos = 8;            // of what is known of a key tile: the softmax may be some behind
constexpr float kMost = 65504.f;     // f16's largest
// log2 of the probability that stands for 1. Above it is room for a maximum outgrown 2^12 times; below
// it f16 has all its bits down to 2^-18 and some to 2^-28, for far keys and blocks of small value scale.
constexpr int kShift = 4;
// A block that a row sees a part of may outweigh the row's reference by this many binades: its scale
// may come from tokens that the row does not see. Such a probability of 1 is 2^15.
constexpr int kPartRoom = 11;
constexpr int kNoScale = -127;       // below every exponent of a scale

// What the softmax needs of a key tile.
struct __align__(16) TileInfo {
  int pos[kTileBlocks];    // first position of each block; far past every row where none is there
  float ks[kTileBlocks];
  int ev[kTileBlocks];     // exponent of the value scale
  __align__(16) unsigned nan[kKeys / 32];  // tokens whose values hold a NaN; there with the values, not the keys
};

template <int D>
struct Smem {
  static constexpr int kQ = kRows * D * 2;       // bytes of a query tile
  static constexpr int kOperand = kKeys * D * 2; // of K or V
  static constexpr int kRaw = kKeys * D;         // codes of the next tile's keys, and of its values
  static constexpr int kBytes = 2 * kQ + 2 * kStages * kOperand + 2 * kRaw + kInfos * (int)sizeof(TileInfo) + 1024;
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
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}

__device__ __forceinline__ uint32_t mul2h(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
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
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};\n" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void store_shared(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// acc + 0 * v in f16x2
__device__ __forceinline__ uint32_t zeros_of(const uint4& v, uint32_t acc) {
  const uint32_t z = 0;
  asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v.x), "r"(z));
  asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v.y), "r"(z));
  asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v.z), "r"(z));
  asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v.w), "r"(z));
  return acc;
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void to_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 16 bytes that are read once: past L1, which shared memory leaves little of
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

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

// Whether a row sees a token with a NaN value: the operand holds 0 in its place, since NaN times the
// probability 0 of a row that does not see it would be NaN too.
__device__ __forceinline__ bool sees_nan(const TileInfo& info, const View& view) {
  const uint4 nan = *reinterpret_cast<const uint4*>(info.nan);
  if ((nan.x | nan.y | nan.z | nan.w) == 0) return false;
  uint32_t found = 0;
  for (int k = 0; k < kTileBlocks; ++k) found |= view.mask(info.pos[k]) & (info.nan[k >> 1] >> (16 * (k & 1)));
  return found != 0;
}

// 256 rows (or 128, LOG2 7) of one (sequence, kv head).
struct Item {
  int seq, head;               // seq -1: no more
  int row0, len, pos0;         // the sequence's first row of q, its length, the position of its query 0
  int first_row, rows;         // this item's first row, and its number of rows
  Span span;                   // blocks that any of them sees
  int begin[2], end[2];        // key tiles of each tile of 128 rows: [begin, end) of the span's list
  __device__ __forceinline__ bool active(int i) const { return end[i] > begin[i]; }
  __device__ __forceinline__ int blocks() const { return max(0, span.count()); }
  __device__ __forceinline__ int tiles() const { return (blocks() + kTileBlocks - 1) / kTileBlocks; }
};

// Whether a value of the block's tokens in `see` has a code that is not zero.
__device__ __forceinline__ bool holds_values(const AttnArgs& a, int seq, int head, int pos, uint32_t see, int dim) {
  const int id = kv8_block_id(a.c, a.t, seq, head, pos / kKvBlock);
  uint32_t any = 0;
  if (id < 0) return false;
#pragma unroll 1
  for (; see != 0 && any == 0; see &= see - 1) {
    const uint4* v = reinterpret_cast<const uint4*>(a.c.v + ((int64_t)id * kKvBlock + (__ffs(see) - 1)) * dim);
#pragma unroll 1
    for (int i = 0; i < dim / 16; ++i) any |= (v[i].x | v[i].y | v[i].z | v[i].w) & 0x7f7f7f7fu;
  }
  return any != 0;
}

// The exponent of the value scale that a row's probabilities are weighed by: the largest of the blocks
// it sees, `before` or here. What it does not see must not count, or a loud value among it would
// shift the row's probabilities out of f16. A block seen in part has kPartRoom, and beyond that
// counts only if one of its seen values is not zero (next to a token that much louder, few are
// anything else). Runs where a tile's largest, `top`, exceeds a row's reference, so seldom; where its
// scales are alike, and they mostly are, one block seen whole stands for all, or a small rise does no
// harm (window 8001: 0.7 % more by blocks).
// `near`: the tile's first position.
constexpr int kAlike = 6;
__device__ __forceinline__ int seen_exponent(const AttnArgs& a, const Item& it, const TileInfo& info, const View& view, int before, int top,
                                             int near, int dim) {
  int low = top, far = 0, there = 0;
#pragma unroll 2
  for (int k = 0; k < kTileBlocks; ++k) {
    if (info.pos[k] == kNowhere) continue;
    low = min(low, info.ev[k]);
    far = max(far, info.pos[k] + kKvBlock);
    there += kKvBlock;
  }
  if ((view.lo >= far || view.qp < near) && view.sinks <= near) return before;  // it sees none
  // 31 positions in a row, or those of a block of sinks, hold a whole block
  const bool whole = (far - near == there && min(view.qp + 1, far) - max(view.lo, near) >= 2 * kKvBlock - 1) ||
                     (min(view.qp + 1, view.sinks) - near >= kKvBlock);
  if (top - low <= kAlike && (whole || top - before <= kAlike)) return max(before, top);
  int most = before, part = before;
#pragma unroll 1
  for (int k = 0; k < kTileBlocks; ++k) {
    const int ev = info.ev[k];
    if (ev <= most) continue;
    const uint32_t see = view.mask(info.pos[k]);
    if (see == 0xffffu)
      most = ev;
    else if (see != 0)
      part = max(part, ev - kPartRoom);
  }
  if (part <= most) return most;
#pragma unroll 1
  for (int k = 0; k < kTileBlocks; ++k) {
    const int ev = info.ev[k] - kPartRoom;
    if (ev <= most) continue;
    const uint32_t see = view.mask(info.pos[k]);
    if (see != 0 && see != 0xffffu && holds_values(a, it.seq, it.head, info.pos[k], see, dim)) most = ev;
  }
  return most;
}

// Columns of TMEM of a warp's rows times a factor of each: f32, or pairs of f16.
template <bool HALF>
__device__ __forceinline__ void rescale(uint32_t at, int columns, float by) {
  const uint32_t by2 = h2(by, by);
#pragma unroll 1
  for (int c = 0; c < columns; c += 16) {
    uint32_t v[16];
    tmem_ld16(at + (uint32_t)c, v);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = HALF ? mul2h(v[e], by2) : __float_as_uint(__uint_as_float(v[e]) * by);
    tmem_st16(at + (uint32_t)c, v);
  }
  tmem_st_wait();
}


// A row of scores becomes a row of probabilities, in f16 and over them, in one pass: 32 keys at a time,
// each block's weighed by its value scale, their sum without the weights added to l. ALL: the row sees
// the whole tile.
//
// No maximum is taken on the way: the last one stands until a chunk's sum shows that f16 would not
// hold its probabilities (or the row has none yet). The chunk's maximum is then found, what was made
// with the old one is brought to it, and the chunk done again. A maximum of every chunk beforehand
// cost a third of the pass (16 lanes' maxima a clock and a second read of the scores: 8 x 2048 causal
// 440 us against 414). With kShift 10 a chunk in nine was done again (539 us), with 4 hardly any.
//
// The loop stays rolled and short: its misses in the instruction cache cost more than a longer
// loop's parallelism gains (64 keys at a time: 491 us).
template <int D, bool ALL, class Settle>
__device__ __forceinline__ void row_pass(uint32_t s_at, uint32_t o_at, const TileInfo& info, const View& view, float factor, bool begin, int eref, float& m, float& l, Settle settle) {
  bool again = false;
#pragma unroll 1
  for (int c = 0; c < kKeys / 32;) {
    uint32_t v[32], p[16], seen = 0;
    tmem_ld32(s_at + 32u * c, v);
    const float2 ks = *reinterpret_cast<const float2*>(info.ks + 2 * c);
    const int2 ev = *reinterpret_cast<const int2*>(info.ev + 2 * c);
    const float base = m == -INFINITY ? 0.f : m;
    float total = 0.f, part = 0.f;
    tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t* x = v + 16 * h;
      const float f = factor * (h ? ks.y : ks.x);
      int w = max(-60, (h ? ev.y : ev.x) - eref) + kShift;
      if (!ALL) w = min(w, kShift + kPartRoom);  // more: nothing of the block is seen, or only zeros
      const uint32_t see = ALL ? 0xffffu : view.mask(info.pos[2 * c + h]);
      seen |= see;
      const uint64_t ff = pair(f, f), add = pair((float)w - base, (float)w - base);
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        float2 y = unpair(fma2(pair(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), ff, add));
        y.x = exp2_ftz(y.x);
        y.y = exp2_ftz(y.y);
        if (!ALL) {
          y.x = see >> e & 1 ? y.x : 0.f;
          y.y = see >> (e + 1) & 1 ? y.y : 0.f;
        }
        sum = add2(sum, pair(y.x, y.y));
        p[8 * h + e / 2] = h2(y.x, y.y);
      }
      const float2 s = unpair(sum);
      total += s.x + s.y;
      part = fmaf(s.x + s.y, __uint_as_float((uint32_t)(127 - w) << 23), part);
    }
    const bool outgrown = !(total <= kMost) || (m == -INFINITY && seen != 0);  // NaN, too: once
    if (__any_sync(0xffffffffu, outgrown) && !again) {
      float mx = m;
#pragma unroll 1
      for (int k = 2 * c; k < 2 * c + 2; ++k) {
        uint32_t x[16];
        tmem_ld16(s_at + 16u * k, x);
        tmem_ld_wait();
        const uint32_t see = ALL ? 0xffffu : view.mask(info.pos[k]);
        float t = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) t = fmaxf(t, see >> e & 1 ? __uint_as_float(x[e]) : -INFINITY);
        mx = fmaxf(mx, t == -INFINITY ? t : t * (factor * info.ks[k]));
      }
      const float mnew = outgrown ? mx : m, by = m == mnew ? 1.f : m == -INFINITY ? 0.f : exp2_ftz(m - mnew);
      l *= by;
      m = mnew;
      tmem_st_wait();
      rescale<true>(s_at, 16 * c, by);
      if (!begin) {
        settle();
        rescale<false>(o_at, D, by);
      }
      again = true;
      continue;
    }
    tmem_st16(s_at + 16u * c, p);
    l += part;
    ++c;
    again = false;
  }
}

// One arrival for a warp: 32 threads' arrivals on one word are 32 operations one after the other,
// and the waiter's time.
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) bar_arrive(bar);
}

// Items of a sequence, before its kv heads.
template <int LOG2>
__device__ __forceinline__ int items_of(const AttnArgs& a, int b) {
  const int64_t rows = (int64_t)kv8_rows(a.offsets, b, a.tokens) * a.group;
  return (int)((rows + (1 << LOG2) - 1) >> LOG2);
}
// Item number f of the call, for a warp: all last items of the sequences, then all last but one, ...
// `limit`: items that sequences of separate rows have at most; there are no more than 2^25, kv heads
// apart, so a lane's sum that reaches kSumMost is past every f.
constexpr unsigned kSumMost = 1u << 26;
template <int LOG2>
__device__ __forceinline__ void find_item(const AttnArgs& a, int64_t f, int64_t limit, int lane, Item& it) {
  it.seq = -1;
  if (f >= limit) return;
  const int64_t m = kv8_quotient(f, a.c.kv_heads);
  // of the first 32 sequences, which are mostly all
  const int own = lane < a.batch ? items_of<LOG2>(a, lane) : 0, own_len = lane < a.batch ? kv8_length(a.lengths, lane) : 0;
  auto items_up_to = [&](int most) -> int64_t {            // sum over the sequences of min(items, most)
    unsigned n = (unsigned)min(most, own);
    for (int b = lane + 32; b < a.batch; b += 32) n = min(n + (unsigned)min(most, items_of<LOG2>(a, b)), kSumMost);
    return __reduce_add_sync(0xffffffffu, n);
  };
  if (m >= items_up_to(0x7fffffff)) return;
  int lo = 0, hi = 1;  // items_up_to(lo) <= m < items_up_to(hi)
  while (items_up_to(hi) <= m) {
    lo = hi;
    hi *= 2;
  }
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (items_up_to(mid) <= m)
      lo = mid;
    else
      hi = mid;
  }
  int64_t left = m - items_up_to(lo);  // this many sequences of more than lo items come before
  int b = -1;
  for (int base = 0; base < a.batch; base += 32) {
    const uint32_t has = __ballot_sync(0xffffffffu, (base == 0 ? own : base + lane < a.batch ? items_of<LOG2>(a, base + lane) : 0) > lo);
    if (left >= __popc(has)) {
      left -= __popc(has);
      continue;
    }
    b = base + __fns(has, 0, (int)left + 1);
    break;
  }
  if (b < 0) return;
  it.seq = b;
  it.head = (int)(f - m * a.c.kv_heads);
  it.row0 = __ldg(a.offsets + b);
  const int n = kv8_rows(a.offsets, b, a.tokens);
  it.len = b < 32 ? __shfl_sync(0xffffffffu, own_len, b) : kv8_length(a.lengths, b);
  it.pos0 = it.len - n;  // negative: the first queries are before the cache and see nothing
  it.first_row = (items_of<LOG2>(a, b) - 1 - lo) << LOG2;
  it.rows = (int)min((int64_t)1 << LOG2, (int64_t)n * a.group - it.first_row);
  auto span_of_tile = [&](int i, int tiles) {  // of tiles i .. i + tiles - 1
    const int from = it.first_row + i * kRows, to = it.first_row + min(it.rows, (i + tiles) * kRows) - 1;
    return span_of(max(0, it.pos0 + from / a.group), min(it.len - 1, it.pos0 + to / a.group), a.window, a.sinks, a.cap);
  };
  it.span = span_of_tile(0, 2);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    it.begin[i] = it.end[i] = 0;
    if (i * kRows >= it.rows) continue;
    // a tile leaves out the key tiles past its last row, and without sinks those before its window
    const Span s = span_of_tile(i, 1);
    if (s.count() <= 0) continue;
    const int end = it.span.sink_blocks + max(0, s.end - it.span.from);
    const int begin = a.sinks > 0 ? 0 : max(0, s.from - it.span.from);
    it.begin[i] = begin / kTileBlocks;
    it.end[i] = (max(end, it.span.sink_blocks) + kTileBlocks - 1) / kTileBlocks;
  }
}

// A lane's output row from TMEM times `inv` (zeros where `none`): 64 or 128 bytes at a time, which
// fill whole sectors.
template <int D, int TYPE>
__device__ __forceinline__ void put_row(void* out, uint32_t o_at, bool none, float inv, int64_t out_row) {
#pragma unroll 1
  for (int c = 0; c < D; c += 32) {
    uint32_t v[32];
    tmem_ld32(o_at + (uint32_t)c, v);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] = none ? 0u : __float_as_uint(__uint_as_float(v[e]) * inv);
    if (out_row >= 0) {
      if (TYPE == J4B_F32) {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<float*>(out) + out_row + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[e] = make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
      } else {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + out_row + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t w[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(__uint_as_float(v[8 * e + 2 * y]), __uint_as_float(v[8 * e + 2 * y + 1]));
            w[y] = *reinterpret_cast<const uint32_t*>(&t);
          }
          dst[e] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    __syncwarp();  // the loads from TMEM are the whole warp's
  }
}

// A warp's 32 query rows of a tile, 8 lanes a row, into the tile's swizzled operand: each by a power
// of two to a largest element in [2^11, 2^12), then to f16 (bf16 is exact there). `factors` takes the
// (biased) exponent of the power of two by which a row's scores are to be multiplied. Rolled: the
// code runs once an item and would come from beyond the instruction cache every time.
template <int D, int TYPE>
__device__ __forceinline__ void bring_queries(const AttnArgs& a, const Item& it, int i, int warp, uint8_t* tile, uint8_t* factors, int lane) {
  constexpr int kWords = TYPE == J4B_F32 ? D / 32 : D / 64;  // 16-byte pieces of a row and lane
  constexpr int kHeld = 8 / kWords;                          // rows of a lane in flight
  // rows 4 apart, without a division each
  const int g0 = it.first_row + i * kRows + 32 * warp + (lane >> 3), on = 4 / a.group, over = 4 - on * a.group;
  int row = it.row0 + g0 / a.group, sub = g0 % a.group;
#pragma unroll 1
  for (int k0 = 0; k0 < 8; k0 += kHeld) {
    uint4 raw[kHeld][kWords];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int qr = 32 * warp + 4 * (k0 + k) + (lane >> 3);
      const bool there = i * kRows + qr < it.rows && row >= 0 && row < a.tokens;
      const int64_t src = (int64_t)row * a.q_stride + (int64_t)(it.head * a.group + sub) * D + 8 * (lane & 7);
#pragma unroll
      for (int c = 0; c < kWords; ++c)
        raw[k][c] = !there ? make_uint4(0, 0, 0, 0)
                    : TYPE == J4B_F32 ? load_once(static_cast<const float*>(a.q) + src + 64 * (c >> 1) + 4 * (c & 1))
                                      : load_once(static_cast<const __nv_bfloat16*>(a.q) + src + 64 * c);
      row += on;
      sub += over;
      if (sub >= a.group) {
        sub -= a.group;
        ++row;
      }
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int qr = 32 * warp + 4 * (k0 + k) + (lane >> 3);
      float x[D / 8];
      float most = 0.f;
#pragma unroll
      for (int c = 0; c < kWords; ++c) {
        const uint32_t w[4] = {raw[k][c].x, raw[k][c].y, raw[k][c].z, raw[k][c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (TYPE == J4B_F32) {
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
      const bool plain = e < 24 || e > 254;
      float up = plain ? 1.f : __uint_as_float((uint32_t)(254 - (e - 11)) << 23);
      if (a.scale_log2 < 0.f) up = -up;  // maxima are taken before the factor
      if ((lane & 7) == 0) factors[qr] = (uint8_t)(plain ? 127 : e - 11);
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const float* y = x + 8 * c;
        *reinterpret_cast<uint4*>(tile + c * (kRows * 128) + sw128_offset(qr, 8 * (lane & 7))) =
            make_uint4(h2(y[0] * up, y[1] * up), h2(y[2] * up, y[3] * up), h2(y[4] * up, y[5] * up), h2(y[6] * up, y[7] * up));
      }
    }
  }
}

// An item's queries on their way to L2 (8 x 2048 401 -> 397 us).
template <int D, int TYPE>
__device__ __forceinline__ void prefetch_queries(const AttnArgs& a, const Item& it, int lane) {
  constexpr int kSize = TYPE == J4B_F32 ? 4 : 2;
  if (it.seq < 0) return;
#pragma unroll 1
  for (int r = lane; r < it.rows; r += 32) {
    const int g = it.first_row + r, row = it.row0 + g / a.group;
    if (row < 0 || row >= a.tokens) continue;
    const char* src = static_cast<const char*>(a.q) + ((int64_t)row * a.q_stride + (int64_t)(it.head * a.group + g % a.group) * D) * kSize;
#pragma unroll
    for (int c = 0; c < D * kSize; c += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + c));
  }
}

// The output of an item whose rows see nothing.
template <int D>
__device__ __forceinline__ void put_zeros(const AttnArgs& a, const Item& it, int lane) {
  const int size = a.out_type == J4B_F32 ? 4 : 2;
#pragma unroll 1
  for (int r = 0; r < it.rows; ++r) {
    const int g = it.first_row + r, row = it.row0 + g / a.group;
    if (row < 0 || row >= a.tokens || lane * 16 >= D * size) continue;
    char* out = static_cast<char*>(a.out) + ((int64_t)row * a.heads + it.head * a.group + g % a.group) * (D * size);
    *reinterpret_cast<uint4*>(out + lane * 16) = make_uint4(0, 0, 0, 0);
  }
}

constexpr int kItems = 4;         // found ahead
constexpr int kItemReaders = 13;  // warps

// SINGLE: items of one tile of rows.
template <int D, int TYPE, bool SINGLE>
__global__ void __launch_bounds__(kThreads, 1) kv8_prefill_kernel(const AttnArgs a, int64_t limit) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_smem(smem_raw);
  uint8_t* sq = smem;                    // [2 tiles]
  uint8_t* sk = smem + 2 * Smem<D>::kQ;  // [stage][K | V]
  uint8_t* sraw = sk + 2 * kStages * Smem<D>::kOperand;
  TileInfo* infos = reinterpret_cast<TileInfo*>(sraw + 2 * Smem<D>::kRaw);
  __shared__ uint64_t item_full[kItems], item_empty[kItems], q_ready[2], q_empty[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages],
      s_full[2], p_ready[2], o_step, o_full[2], o_seen[2];
  __shared__ uint32_t tmem_slot;
  __shared__ Item items[kItems];
  __shared__ uint8_t factors[2][kRows];  // a warp's are its own rows'
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    bar_init(&o_step, 1);
    for (int i = 0; i < kItems; ++i) {
      bar_init(&item_full[i], 1);
      bar_init(&item_empty[i], kItemReaders);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(&q_ready[i], 4);  // warps
      bar_init(&q_empty[i], 1);
      bar_init(&s_full[i], 2);  // the MMAs, and the thread that saw keys, info and queries ready
      bar_init(&p_ready[i], 4);
      bar_init(&o_full[i], 2);
      bar_init(&o_seen[i], 4);
    }
    for (int s = 0; s < kStages; ++s) {
      bar_init(&k_full[s], 4);
      bar_init(&v_full[s], 4);
      bar_init(&k_empty[s], 1);
      bar_init(&v_empty[s], 1);
    }
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
  // The finder of items, and warps that have no part in one, wait while another walks over all its key
  // tiles: 2.3 us each, so 0.3 s for 2^24 tokens. Their bound is 8 times that above the common one.
  const uint64_t walk = (uint64_t)a.cap * (8 * 2300 / kTileBlocks);
  // An item of one tile has the other's columns, too: its scores, and the barriers s_full and p_ready,
  // alternate between the two, and a key tile's are there before the last one's softmax ends (5 turns
  // of up to 77 tokens on up to 1000: 27.0 -> 24.5 us).
  // The next item, for every warp but the one that finds them (null after the last); the one before
  // is given back. Read where it is: a copy would cost registers.
  uint32_t nth = 0;
  auto next_item = [&]() -> const Item* {
    __syncwarp();
    if (nth > 0 && lane == 0) bar_arrive(&item_empty[(nth - 1) % kItems]);
    ok = __all_sync(0xffffffffu, ok && kv8_wait(&item_full[nth % kItems], nth / kItems & 1, walk));  // the warp stays together
    const Item* it = &items[nth % kItems];
    ++nth;
    return ok && it->seq >= 0 ? it : nullptr;
  };

  if (warp < 8) {
    // ---- softmax of tile i, one row a thread ----
    const int i = warp >> 2, r = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_at = lanes + (uint32_t)(i * 128), o_at = lanes + 256u + (uint32_t)(i * 128);
    uint32_t use = 0, outs = 0, before = 0;  // tiles done, items done, key tiles of the earlier items
    const Item* item = next_item();
    // an item's queries, into the tile's operand once the last item's scores are done with it; returns
    // what the lane's row's scores are to be multiplied by
    auto bring = [&](const Item& it) -> float {
      if (outs > 0) ok = ok && kv8_wait(&q_empty[i], (outs - 1) & 1);
      bring_queries<D, TYPE>(a, it, i, warp & 3, sq + i * Smem<D>::kQ, factors[i], lane);
      to_async_proxy();
      warp_arrive(&q_ready[i], lane);
      return fabsf(a.scale_log2) * __uint_as_float((uint32_t)factors[i][r] << 23);
    };
    float factor = item && item->active(i) ? bring(*item) : 0.f;
    while (item) {
      const Item& it = *item;
      const bool active = it.active(i);
      const int gr = it.first_row + i * kRows + r, tok = gr / a.group, gh = it.head * a.group + gr % a.group;
      const bool valid = i * kRows + r < it.rows && it.row0 + tok >= 0 && it.row0 + tok < a.tokens;
      const int64_t out_row = valid ? ((int64_t)(it.row0 + tok) * a.heads + gh) * D : -1;
      const int qp = valid ? max(-1, it.pos0 + tok) : -1;
      const View view = {a.window > 0 ? max(0, qp - a.window + 1) : 0, qp, a.sinks};
      // every valid row of the tile sees the positions [most_lo, least]
      const int least = it.pos0 + (it.first_row + i * kRows) / a.group;
      const int most_lo = a.window > 0 ? max(0, it.pos0 + (it.first_row + min(it.rows, (i + 1) * kRows) - 1) / a.group - a.window + 1) : 0;
      float m = -INFINITY, l = 0.f;
      int eref = valid ? kNoScale : -kNoScale;  // exponent of the value scale that O is in units of
      const int j0 = it.begin[i], j1 = it.end[i];
      for (int j = j0; j < j1; ++j, ++use) {
        const uint32_t k = before + (uint32_t)j;
        const uint32_t buffer = SINGLE ? use & 1 : (uint32_t)i, parity = SINGLE ? use >> 1 & 1 : use & 1;
        const uint32_t s_now = SINGLE ? s_at + buffer * 128u : s_at;
        ok = ok && kv8_wait(&s_full[buffer], parity);  // with it comes the tile's info
        tc_fence_after();
        const TileInfo& info = infos[k % kInfos];
        int near = kNowhere, far = 0, ev = -127;
#pragma unroll
        for (int x = 0; x < kTileBlocks; ++x) {
          near = min(near, info.pos[x]);
          far = max(far, info.pos[x] + kKvBlock);
          ev = max(ev, info.ev[x]);
        }
        const bool all = far - 1 <= least && (near >= most_lo || far <= a.sinks);
        // the last tile's values (with a tile alone the last but one's) were ready before these scores were
        const int late = SINGLE ? 2 : 1;
        if (j - late >= j0 && sees_nan(infos[(k - late) % kInfos], view)) l = NAN;
        auto settle = [&] {  // the MMAs on O are done; of two tiles, before these scores
          if (SINGLE) {
            ok = ok && kv8_wait(&o_step, (use - 1) & 1);
            tc_fence_after();
          }
        };
        const bool begin = j == j0;
        if (__any_sync(0xffffffffu, ev > eref)) {
          const int now = all ? max(ev, eref) : seen_exponent(a, it, info, view, eref, ev, near, D);
          if (!begin && __any_sync(0xffffffffu, now > eref)) {
            settle();
            rescale<false>(o_at, D, exp2_ftz((float)(eref - now)));
          }
          eref = now;
        }
        if (all)
          row_pass<D, true>(s_now, o_at, info, view, factor, begin, eref, m, l, settle);
        else
          row_pass<D, false>(s_now, o_at, info, view, factor, begin, eref, m, l, settle);
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(&p_ready[buffer], lane);
      }
      const uint32_t last_tile = before + (uint32_t)j1 - 1;
      before += (uint32_t)it.tiles();
      const int rows = it.rows;
      if (active) ++outs;
      item = next_item();
      // the next item's queries first: its scores are computed while this one's output is written
      factor = item && item->active(i) ? bring(*item) : 0.f;
      if (active) {
        ok = ok && kv8_wait(&o_full[i], (outs - 1) & 1);
        tc_fence_after();
        if (sees_nan(infos[last_tile % kInfos], view) || (SINGLE && j1 - 1 > j0 && sees_nan(infos[(last_tile - 1) % kInfos], view))) l = NAN;
        warp_arrive(&o_seen[i], lane);
      }
      if (i * kRows < rows) {
        const bool none = m == -INFINITY;
        const float inv = none ? 0.f : exp2_ftz((float)(eref - kShift)) / l;
        if (a.out_type == J4B_F32)
          put_row<D, J4B_F32>(a.out, o_at, none, inv, out_row);
        else
          put_row<D, J4B_BF16>(a.out, o_at, none, inv, out_row);
      }
      tc_fence_before();
    }
  } else if (warp < 12) {
    // ---- pages to operands: this warp the rows 32 w .. + 31 (2 blocks) of each key tile ----
    const int w = warp - 8;
    constexpr int kHalves = D / 64, kPieces = 4 * kHalves;  // 16-code pieces of a thread, K or V
    // piece x: row 32 w + 8 (x / kHalves) + lane / 4, codes 64 (x % kHalves) + 16 (lane % 4): 8 lanes of
    // a store phase are 2 rows x 4 pieces, whose swizzled places cover all banks
    const int pr = lane >> 2, pc = lane & 3;
    // Codes wait in shared memory, each thread's pieces its own (so its own wait is all they need).
    const uint32_t mine_at = saddr(sraw) + (uint32_t)(tid & 127) * 16u;
    auto load = [&](const uint8_t* codes, int which, const int (&id)[2]) {
      const uint8_t* from = codes + pr * D + 16 * pc;
      const uint8_t* const src[2] = {from + (int64_t)max(id[0], 0) * (kKvBlock * D), from + (int64_t)max(id[1], 0) * (kKvBlock * D)};
      const uint32_t to = mine_at + (uint32_t)(which * Smem<D>::kRaw);
#pragma unroll
      for (int x = 0; x < kPieces; ++x) {
        const int k = x >= kPieces / 2;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + x * 2048u), "l"(src[k] + (x / kHalves & 1) * (8 * D) + 64 * (x % kHalves)), "r"(id[k] < 0 ? 0 : 16) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // Where the first half of piece 0 goes in an operand (the second is 16 bytes across); piece x's are 1024 (x / kHalves) + kKeys * 128 (x % kHalves) further.
    const uint32_t lo_at = (uint32_t)(w * 4096 + pr * 128 + (((2 * pc) ^ pr) << 4));
    auto turn = [&](uint32_t operand, int x, const uint4& src) -> uint32_t {
      uint4 lo, hi;
      e4m3x4_f16(src.x, lo.x, lo.y);
      e4m3x4_f16(src.y, lo.z, lo.w);
      e4m3x4_f16(src.z, hi.x, hi.y);
      e4m3x4_f16(src.w, hi.z, hi.w);
      const uint32_t at = operand + lo_at + (uint32_t)(1024 * (x / kHalves) + kKeys * 128 * (x % kHalves));
      store_shared(at, lo);
      store_shared(at ^ 16u, hi);
      // 0, or NaN where a code is one (the FMA units have room, the integer ones less)
      return zeros_of(lo, zeros_of(hi, 0));
    };
    // four pieces at a time, for the instruction cache (all eight: 8 x 2048 405 -> 414 us)
    auto turn_all = [&](uint32_t operand, int which) -> uint32_t {
      const uint8_t* from = sraw + which * Smem<D>::kRaw + (tid & 127) * 16;
      uint32_t any = 0;
#pragma unroll 4
      for (int x = 0; x < kPieces; ++x) {
        const uint32_t z = turn(operand, x, *reinterpret_cast<const uint4*>(from + x * 2048));
        if (which) any |= z;
      }
      return any;
    };
    // (it, j) runs two tiles ahead of the operands, into the next items: its page numbers are on their
    // way while a tile is turned, the codes and scales of the tile between from when this one's are out
    // of the way.
    const Item* it = next_item();
    int j = 0;
    // of its tile, for an even lane block 2 w, for an odd one 2 w + 1 (-1: past the end): its page as
    // loaded, its number in the page; the kv head, the length
    int blk = -1, page = -1, in_page = 0, head = 0, len = 0;
    int id[2] = {-1, -1};  // the blocks' numbers, once the pages are there
    auto find = [&]() -> bool {                        // tile j, and on to the next; false after the last
      while (it && j >= it->tiles()) {
        it = next_item();
        j = 0;
      }
      if (!it) return false;
      const int x = j * kTileBlocks + 2 * w + (lane & 1);
      blk = x < it->blocks() ? it->span.block(x) : -1;
      const int at = blk / a.c.bpp;
      in_page = blk - at * a.c.bpp;
      page = blk >= 0 && at < a.t.width ? __ldg(a.t.pages + it->seq * a.t.stride + at) : -1;
      head = it->head;
      len = it->len;
      ++j;
      return true;
    };
    auto number = [&] {
      const int mine = (unsigned)page < (unsigned)a.c.pages ? (page * a.c.kv_heads + head) * a.c.bpp + in_page : -1;
#pragma unroll
      for (int k = 0; k < 2; ++k) id[k] = __shfl_sync(0xffffffffu, mine, k);
    };
    float ks = 1.f, vs = 0.f;
    int now[2] = {-1, -1}, now_len = 0;  // first positions of the tile's blocks (-1: not there)
    auto scales = [&] {
      const int mine = lane == 0 ? id[0] : id[1];
      ks = 1.f, vs = 0.f;
      if (lane < 2 && mine >= 0) {
        ks = __ldg(a.c.ks + mine);
        vs = __ldg(a.c.vs + mine);
      }
    };
    auto take = [&] {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int b = __shfl_sync(0xffffffffu, blk, k);
        now[k] = id[k] < 0 ? -1 : b * kKvBlock;
      }
      now_len = len;
    };
    bool here = find();
    if (here) {
      number();
      load(a.c.k, 0, id);
      load(a.c.v, 1, id);
      scales();
      take();
    }
    bool next = here && find();
    for (uint32_t k = 0; here; ++k) {
      const int s = k % kStages;
      const uint32_t parity = (k / kStages - 1) & 1;
      const uint32_t kt = saddr(sk) + (uint32_t)(s * 2 * Smem<D>::kOperand);
      TileInfo& info = infos[k % kInfos];
      asm volatile("cp.async.wait_group 1;" ::: "memory");  // the keys; the values may be on their way
      if (k >= kStages) ok = ok && kv8_wait(&k_empty[s], parity);
      turn_all(kt, 0);
      if (lane < 2) {
        const int x = 2 * w + lane, pos = lane == 0 ? now[0] : now[1];
        info.pos[x] = pos < 0 ? kNowhere : pos;
        info.ks[x] = ks;
        info.ev[x] = (int)(__float_as_uint(vs) >> 23) + kNoScale;
      }
      to_async_proxy();
      warp_arrive(&k_full[s], lane);
      if (next) {
        number();
        load(a.c.k, 0, id);
      }
      // the values: one group after theirs is this tile's next keys'
      if (next)
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      else
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      if (k >= kStages) ok = ok && kv8_wait(&v_empty[s], parity);
      // tokens past the length hold anything; NaNs go to the info, as zeros to the operand
      unsigned nan = 0;
      const uint32_t any = turn_all(kt + Smem<D>::kOperand, 1);
      if (__any_sync(0xffffffffu, any != 0) || max(now[0], now[1]) + kKvBlock > now_len) {
#pragma unroll 1
        for (int x = 0; x < kPieces; ++x) {
          const int row = 8 * (x / kHalves) + pr;
          uint4 v = *reinterpret_cast<const uint4*>(sraw + Smem<D>::kRaw + x * 2048 + (tid & 127) * 16);
          if ((x >= kPieces / 2 ? now[1] : now[0]) + (row & 15) >= now_len) v = make_uint4(0, 0, 0, 0);
          uint32_t* q = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t bytes = (((q[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
            q[e] &= ~(bytes * 0xffu);
            if (bytes) nan |= 1u << row;
          }
          turn(kt + Smem<D>::kOperand, x, v);
        }
        nan = __reduce_or_sync(0xffffffffu, nan);
      }
      if (lane == 0) info.nan[w] = nan;
      to_async_proxy();
      warp_arrive(&v_full[s], lane);
      here = next;
      if (next) {
        load(a.c.v, 1, id);
        scales();
        take();
        next = find();
      }
    }
  } else {
    if (warp == 12) {
      // ---- the MMAs: the warp waits as one, an elected thread issues ----
      // One thread's branch would keep the descriptors out of uniform registers (8 x 2048 456 against 441 us).
      auto uni = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
      auto wait = [&](uint64_t* bar, uint32_t parity) { ok = __all_sync(0xffffffffu, ok && kv8_wait(bar, parity)); };
      constexpr uint32_t is = idesc_f16(kRows, kKeys, false), io = idesc_f16(kRows, D, true);
      // descriptors count in 16-byte units: stepping one is an addition
      uint64_t qd = kmajor_sw128(saddr(sq)), kd = kmajor_sw128(saddr(sk)), vd = rows_sw128(saddr(sk) + Smem<D>::kOperand, kKeys * 128);
      constexpr uint32_t kStage = 2 * Smem<D>::kOperand / 16;
      uint32_t p_use0 = 0, p_use1 = 0, q_use0 = 0, q_use1 = 0, before = 0;
      bool left0 = false, left1 = false;  // the last item's softmax may still need its last info
      uint32_t s_use0 = 0, s_use1 = 0, scores = 0;
      while (const Item* const item = next_item()) {
        const int nt = uni(item->tiles()), b0 = uni(item->begin[0]), b1 = uni(item->begin[1]), e0 = uni(item->end[0]), e1 = uni(item->end[1]);
        if constexpr (SINGLE) {
          for (int j = -1; j < nt && ok; ++j) {
            const uint32_t now = before + (uint32_t)j, next = now + 1;
            if (j + 1 < nt) wait(&k_full[next & 1], next >> 1 & 1);
            if (j == 0) {  // as below
              if (left0) wait(&o_seen[0], s_use0++ & 1);
              left0 = e0 > b0;
            }
            if (j + 1 >= b0 && j + 1 < e0) {
              if (j + 1 == b0) wait(&q_ready[0], q_use0++ & 1);
              tc_fence_after();
              if (elect_one()) {
                const uint64_t kt = kd + (next & 1) * kStage;
                const uint32_t s_at = tmem + (scores & 1) * 128u;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                  const uint32_t off = ((k >> 2) * (kRows * 128) + (k & 3) * 32) / 16;
                  umma_ss(s_at, qd + off, kt + off, is, k > 0 ? 1u : 0u);
                }
                umma_commit(&s_full[scores & 1]);
                bar_arrive(&s_full[scores & 1]);
                if (j + 2 == e0) umma_commit(&q_empty[0]);
              }
              ++scores;
            }
            if (j + 1 < nt && elect_one()) umma_commit(&k_empty[next & 1]);
            __syncwarp();
            if (j < 0) continue;
            wait(&v_full[now & 1], now >> 1 & 1);
            if (j >= b0 && j < e0) {
              wait(&p_ready[p_use0 & 1], p_use0 >> 1 & 1);
              tc_fence_after();
              if (elect_one()) {
                const uint64_t vt = vd + (now & 1) * kStage;
                const uint32_t later = j > b0;
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k) umma_ts(tmem + 256u, tmem + (p_use0 & 1) * 128u + 8u * k, vt + k * (2048 / 16), io, k > 0 ? 1u : later);
                umma_commit(&o_step);
                if (j + 1 == e0) {
                  umma_commit(&o_full[0]);
                  bar_arrive(&o_full[0]);
                }
              }
              ++p_use0;
            }
            if (elect_one()) umma_commit(&v_empty[now & 1]);
            __syncwarp();
          }
        } else {
          for (int j = -1; j < nt && ok; ++j) {
            const uint32_t now = before + (uint32_t)j, next = now + 1;
            if (j + 1 < nt) wait(&k_full[next & 1], next >> 1 & 1);
            if (j >= 0) wait(&v_full[now & 1], now >> 1 & 1);
            // No further until the last item's infos are read: a softmax that has no part in this item could
            // fall behind by more than kInfos tiles (three of this and the next item may have infos by now).
            if (j == 0) {
              if (left0) wait(&o_seen[0], s_use0++ & 1);
              if (left1) wait(&o_seen[1], s_use1++ & 1);
              left0 = e0 > b0;
              left1 = e1 > b1;
            }
            const uint64_t vt = vd + (now & 1) * kStage, kt = kd + (next & 1) * kStage;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int begin = i ? b1 : b0, end = i ? e1 : e0;
              uint32_t &p_use = i ? p_use1 : p_use0, &q_use = i ? q_use1 : q_use0;
              const uint32_t s_at = tmem + (uint32_t)(i * 128), o_at = tmem + 256u + (uint32_t)(i * 128);
              if (j >= begin && j < end) {
                wait(&p_ready[i], p_use & 1);
                ++p_use;
                tc_fence_after();
                if (elect_one()) {
                  const uint32_t later = j > begin;
#pragma unroll
                  for (int k = 0; k < kKeys / 16; ++k)  // 16 keys: 8 columns of P, 2 groups of 8 rows of V
                    umma_ts(o_at, s_at + 8u * k, vt + k * (2048 / 16), io, k > 0 ? 1u : later);
                  if (j + 1 == end) {
                    umma_commit(&o_full[i]);
                    bar_arrive(&o_full[i]);
                  }
                }
              }
              if (j + 1 >= begin && j + 1 < end) {
                if (j + 1 == begin) {
                  wait(&q_ready[i], q_use & 1);
                  ++q_use;
                }
                tc_fence_after();
                if (elect_one()) {
                  const uint64_t qt = qd + (uint32_t)(i * Smem<D>::kQ / 16);
#pragma unroll
                  for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = ((k >> 2) * (kRows * 128) + (k & 3) * 32) / 16;  // kRows == kKeys
                    umma_ss(s_at, qt + off, kt + off, is, k > 0 ? 1u : 0u);
                  }
                  umma_commit(&s_full[i]);
                  bar_arrive(&s_full[i]);
                  if (j + 2 == end) umma_commit(&q_empty[i]);
                }
              }
            }
            if (elect_one()) {
              if (j + 1 < nt) umma_commit(&k_empty[next & 1]);
              if (j >= 0) umma_commit(&v_empty[now & 1]);
            }
            __syncwarp();
          }
        }
        before += (uint32_t)nt;
      }
    } else if (warp == 13) {
      // ---- items ----
      // Ones whose rows see nothing go no further. Every other item has a key tile, so the page warps,
      // which look one tile ahead before they turn the last one, never wait for more than the next
      // item (past a run of empty ones they would wait for the very item that waits for them).
      uint32_t found = 0;
      bool more = true;
      for (uint32_t r = 0; more && ok; ++r) {
        Item it;
        find_item<SINGLE ? 7 : 8>(a, (int64_t)r * gridDim.x + (r & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x), limit, lane, it);
        more = it.seq >= 0;
        if (more && it.tiles() == 0) {
          put_zeros<D>(a, it, lane);
          continue;
        }
        const uint32_t slot = found % kItems;
        if (found >= kItems) ok = __all_sync(0xffffffffu, ok && kv8_wait(&item_empty[slot], (found / kItems - 1) & 1, walk));
        if (lane == 0) {
          items[slot] = it;
          bar_arrive(&item_full[slot]);
        }
        ++found;
        __syncwarp();
        prefetch_queries<D, TYPE>(a, it, lane);  // a CTA's numbers rise
      }
    }
  }
  if (!ok) *a.timeout = 1;
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

template <int D, int TYPE, bool SINGLE>
int launch_prefill_kernel(const AttnArgs& a, int64_t items, int dev, cudaStream_t stream) {
  static bool done[kMaxDevices] = {};
  if (!done[dev]) {
    J4B_CUDA(cudaFuncSetAttribute(kv8_prefill_kernel<D, TYPE, SINGLE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::kBytes), "cudaFuncSetAttribute");
    done[dev] = true;
  }
  kv8_prefill_kernel<D, TYPE, SINGLE><<<(unsigned)std::min<int64_t>(items, device_ctx(dev)->sm_count), kThreads, Smem<D>::kBytes, stream>>>(a, items);
  J4B_CHECK_LAUNCH("kv8_prefill_kernel");
  return J4B_OK;
}

template <int D, int TYPE>
int launch_prefill(const AttnArgs& a, int dev, cudaStream_t stream) {
  const int64_t rows = a.tokens * a.group;
  J4B_REQUIRE(rows <= 0x3fffffffLL, "kv8 prefill: too many rows");
  auto items = [&](int log2) { return std::min(rows, (rows >> log2) + a.batch) * a.c.kv_heads; };  // at most
  // A tile of 128 rows alone walks its keys faster than one of two, so where every such tile has an SM
  // to itself, items are one tile (5 turns of up to 77 tokens on up to 1000: 31.6 -> 24.5 us). Two
  // share the work on the pages elsewhere (8 x 2048: 390 us, by tiles alone 642).
  if (items(7) <= device_ctx(dev)->sm_count) return launch_prefill_kernel<D, TYPE, true>(a, items(7), dev, stream);
  return launch_prefill_kernel<D, TYPE, false>(a, items(8), dev, stream);
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
  if (q_type == J4B_F32)
    return cache->head_dim == 128 ? launch_prefill<128, J4B_F32>(a, dev, stream) : launch_prefill<64, J4B_F32>(a, dev, stream);
  return cache->head_dim == 128 ? launch_prefill<128, J4B_BF16>(a, dev, stream) : launch_prefill<64, J4B_BF16>(a, dev, stream);
}
