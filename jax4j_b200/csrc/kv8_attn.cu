// Decode attention over the 8-bit paged KV cache (format: kv8_common.cuh): one query per sequence,
// grouped heads, sliding window with sinks. Prefill: kv8_prefill.cu.
//
// A warp takes a 16-token block of one kv head at a time straight from the pages into mma.sync
// m16n8k16 operands: 8 tokens are the n columns of S = Q K^T, and since a contraction may run over
// its index in any order, a thread takes 16 consecutive dims of its token (one 16-byte load) as
// the k indices of four MMAs. For O = P V the 16 tokens are the k index and 8 dims the columns; a
// thread loads the 4 tokens whose probabilities it holds, whole 16-byte pieces, and pairs their
// bytes by byte permutes. e4m3 to f16 is exact, so the only roundings are those of Q and P.
// Scales are powers of two: a block's key scale multiplies its scores, and its value scale, over
// the largest seen so far, its probabilities.
#include <algorithm>
#include <cmath>

#include "kv8_common.cuh"
#include "tc_common.cuh"

namespace j4b {

namespace {

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// what h2 rounded away, as f16x2
__device__ __forceinline__ uint32_t h2_rest(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return h2(a - f.x, b - f.y);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// A block in shared memory: 16 rows of D bytes as TMA writes them with its 128-byte (D = 128) or
// 64-byte (D = 64) swizzle, so that the reads below touch every bank once (16-byte pieces whose
// rows are 128 bytes apart would meet in the same banks). A lane's pieces, g = lane / 4, t = lane % 4:
// keys of tokens g and 8 + g, dims kK 16 t .. + kK 16 - 1; values of tokens 2t, 2t + 1, 2t + 8,
// 2t + 9, dims (D / 8) g .. + D / 8 - 1.
template <int D>
struct Piece {
  static constexpr int kK = D / 64;            // 16-byte key pieces of a token
  static constexpr int kW = D / 32;            // 4-byte words of a value piece
  static constexpr int kBytes = kKvBlock * D;  // of a block's keys, and of its values
  static constexpr int kBuffer = 4 * kBytes;   // a warp's: keys of two blocks, then values of two blocks
  // 16-byte chunk `c` of row r
  static __device__ __forceinline__ int at(int r, int c) { return r * D + ((c ^ (D == 128 ? r & 7 : r >> 1 & 3)) << 4); }
  static __device__ __forceinline__ int key(int lane, int i) { return at(lane >> 2, kK * (lane & 3) + i); }
  static __device__ __forceinline__ int value(int lane, int j) {
    const int g = lane >> 2, r = 2 * (lane & 3) + j;
    return D == 128 ? at(r, g) : at(r, g >> 1) + (g & 1) * 8;
  }
};

// A warp's online softmax over the blocks it visits. The 16 rows of the MMAs are 8 queries: rows 0-7
// the f16 values of Q (and P), rows 8-15 what the rounding left, so that every product is
// f32-accurate at no extra MMA (a group of up to 8 heads leaves those rows idle otherwise). A thread's
// query is row g = lane / 4.
template <int D>
struct Warp {
  const uint4* q;  // the A operands of the D / 16 k steps, [step][lane], in shared memory
  float o[D / 8][4];
  float factor;  // scores in log2 units per unit of the MMA's result and of key scale
  float m, l;
  float ref;  // value scale that the accumulators are in units of (times 2^-kPShift)

  // probabilities enter the second product as p 2^kPShift <= 4096: f16 keeps p's bits down to
  // 2^-24 / 4096, below f32's for a row of a million tokens
  static constexpr int kPShift = 12;
  // A block that is seen in part may outweigh `ref` by this factor (f16 holds 2^12 times it): its
  // scale may come from tokens that are not seen.
  static constexpr float kPartRoom = 8.f;

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    m = -INFINITY, l = 0.f;
    ref = 0.f;
  }

  // A query row's elements of a lane (row < 0: zeros), on their way.
  struct Query {
    float4 x[D / 16];
  };
  __device__ __forceinline__ static void fetch_q(Query& f, const void* base, int type, int64_t row, int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      f.x[i] = row >= 0 ? load4(base, type, row + 16 * (Piece<D>::kK * t + (i >> 2)) + 4 * (i & 3)) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // Writes the operands of the query rows to `dst`, and keeps it. Each row is first brought to a
  // largest element in [2^11, 2^12) by a power of two, so f16's range does not limit queries. `warps`
  // warps with the same rows share the operands, each writes every warps-th step.
  __device__ __forceinline__ void load_q(uint4* dst, const Query& f, float scale_log2, int lane, int warp, int warps) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      most = fmaxf(most, fmaxf(fmaxf(fabsf(f.x[i].x), fabsf(f.x[i].y)), fmaxf(fabsf(f.x[i].z), fabsf(f.x[i].w))));
    most = quad_max(most);
    // the power of two below `most`, biased, whose e - 11 and 254 - (e - 11) are exponents of normal
    // numbers; queries of tiny, infinite or no magnitude stay as they are
    const int e = (int)(__float_as_uint(most) >> 23);
    const float down = e < 24 || e > 254 ? 1.f : __uint_as_float((uint32_t)(e - 11) << 23);
    const float up = e < 24 || e > 254 ? 1.f : __uint_as_float((uint32_t)(254 - (e - 11)) << 23);
    factor = scale_log2 * down;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const float4 y = make_float4(f.x[i].x * up, f.x[i].y * up, f.x[i].z * up, f.x[i].w * up);
      const uint32_t lo = h2(y.x, y.y), hi = h2(y.z, y.w);
      if (i % warps == warp) dst[i * 32 + lane] = make_uint4(lo, h2_rest(y.x, y.y, lo), hi, h2_rest(y.z, y.w, hi));
    }
    q = dst + lane;
  }

  // Two blocks, first half: their key codes in the lane's buffer, their scales, and which of their
  // tokens the lane's row sees: tokens j with (first <= j or j < sinks) and j <= last (a block that is
  // not there has p0 far past every row). `all`: every row sees every token of both. Two at a time:
  // their MMA chains are independent, and one maximum, one vote on rescaling serve both.
  // Leaves the probabilities in p, and in `seen` (bit 4 u + j) which of the lane's tokens any row
  // sees: a masked token's value codes are replaced by zeros in the second half, since they may
  // hold anything, NaN too, in a page that is not full. What is not seen does not count for `ref`
  // either: a block seen in part has kPartRoom, and beyond that counts only if one of its seen
  // values is not zero (`holds`, which waits for the values' codes).
  template <class Holds>
  __device__ __forceinline__ void scores(const uint8_t* stage, const float (&ks)[2], float (&vs)[2], bool all, int first, int last,
                                         int sinks, const int (&p0)[2], int lane, uint32_t (&p)[2][4], uint32_t& seen, Holds holds) {
    const int t = lane & 3;
    float s[2][2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int n = 0; n < 2; ++n) s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = 0.f;
#pragma unroll
    for (int i = 0; i < Piece<D>::kK; ++i) {
      uint32_t w[2][2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int n = 0; n < 2; ++n)
          *reinterpret_cast<uint4*>(w[u][n]) =
              *reinterpret_cast<const uint4*>(stage + u * Piece<D>::kBytes + n * (8 * D) + Piece<D>::key(lane, i));
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // the four chains in turn: an MMA never waits for the one before it
        const uint4 qf = q[(4 * i + j) * 32];
        const uint32_t a[4] = {qf.x, qf.y, qf.z, qf.w};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            uint32_t b0, b1;
            e4m3x4_f16(w[u][n][j], b0, b1);
            mma16816(s[u][n], a, b0, b1);
          }
      }
    }
    float x[2][4];  // scores of tokens 2t, 2t + 1, 2t + 8, 2t + 9 of each block
    seen = all ? 0xffu : 0u;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float f = factor * ks[u];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[u][j] = (s[u][j >> 1][j & 1] + s[u][j >> 1][2 + (j & 1)]) * f;
    }
    if (!all) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = p0[u] + 2 * t + (j & 1) + 8 * (j >> 1);
          const bool see = (tok >= first || tok < sinks) && tok <= last;
          if (!see) x[u][j] = -INFINITY;
          seen |= (uint32_t)see << (4 * u + j);
        }
      // the lanes of the same t hold the other rows
      seen |= __shfl_xor_sync(0xffffffffu, seen, 4);
      seen |= __shfl_xor_sync(0xffffffffu, seen, 8);
      seen |= __shfl_xor_sync(0xffffffffu, seen, 16);
    }
    float vmax = fmaxf(vs[0], vs[1]);
    if (!all) {
      const uint32_t some = __reduce_or_sync(0xffffffffu, seen), full = __reduce_and_sync(0xffffffffu, seen);
      float most = ref;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if ((some >> (4 * u) & 15u) == 0) vs[u] = 0.f;
        if ((full >> (4 * u) & 15u) == 15u) most = fmaxf(most, vs[u]);
      }
      vmax = most;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (vs[u] > kPartRoom * most) {
          if (holds(u, seen))
            vmax = fmaxf(vmax, vs[u] * (1.f / kPartRoom));
          else
            vs[u] = 0.f;
        }
    }
    const float mn = fmaxf(m, quad_max(fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])))));
    if (__any_sync(0xffffffffu, vmax > ref || mn > m)) {
      const float now = fmaxf(ref, vmax);
      const float down = ref * kv8_inverse(now);  // 0 at the first block
      ref = now;
      const float c = mn == -INFINITY ? 1.f : exp2f(m - mn);
      l *= c;
      m = mn;
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] *= c * down;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float weight = (float)(1 << kPShift) * (vs[u] * kv8_inverse(ref));
      float e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e[j] = exp2_ftz(x[u][j] - base);
        l += e[j];
        e[j] *= weight;
      }
      p[u][0] = h2(e[0], e[1]);
      p[u][2] = h2(e[2], e[3]);
      p[u][1] = h2_rest(e[0], e[1], p[u][0]);
      p[u][3] = h2_rest(e[2], e[3], p[u][2]);
    }
  }

  // Whether any value code of block u's tokens in `seen` is not zero.
  __device__ __forceinline__ static bool holds_values(const uint8_t* stage, int u, uint32_t seen, int lane) {
    const uint8_t* vb = stage + u * Piece<D>::kBytes;
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint8_t* at = vb + (j >> 1) * (8 * D) + Piece<D>::value(lane, j & 1);
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < Piece<D>::kW; ++i) w |= reinterpret_cast<const uint32_t*>(at)[i];
      if (seen >> (4 * u + j) & 1) any |= w & 0x7f7f7f7fu;
    }
    return __any_sync(0xffffffffu, any != 0);
  }

  // Second half: the accumulators take the two blocks' values, their codes in the lane's buffer.
  __device__ __forceinline__ void values(const uint8_t* stage, const uint32_t (&p)[2][4], uint32_t seen, int lane) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint8_t* vb = stage + u * Piece<D>::kBytes;
      uint32_t v[4][Piece<D>::kW];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (D == 128)
          *reinterpret_cast<uint4*>(v[j]) = *reinterpret_cast<const uint4*>(vb + (j >> 1) * (8 * D) + Piece<D>::value(lane, j & 1));
        else
          *reinterpret_cast<uint2*>(v[j]) = *reinterpret_cast<const uint2*>(vb + (j >> 1) * (8 * D) + Piece<D>::value(lane, j & 1));
        if (!(seen >> (4 * u + j) & 1))
#pragma unroll
          for (int w = 0; w < Piece<D>::kW; ++w) v[j][w] = 0;
      }
#pragma unroll
      for (int w = 0; w < Piece<D>::kW; ++w) {
        const uint32_t a0 = __byte_perm(v[0][w], v[1][w], 0x5140), a1 = __byte_perm(v[0][w], v[1][w], 0x7362);
        const uint32_t c0 = __byte_perm(v[2][w], v[3][w], 0x5140), c1 = __byte_perm(v[2][w], v[3][w], 0x7362);
        uint32_t b00, b01, b10, b11;
        e4m3x4_f16(a0, b00, b10);
        e4m3x4_f16(c0, b01, b11);
        mma16816(o[4 * w], p[u], b00, b01);
        mma16816(o[4 * w + 1], p[u], b10, b11);
        e4m3x4_f16(a1, b00, b10);
        e4m3x4_f16(c1, b01, b11);
        mma16816(o[4 * w + 2], p[u], b00, b01);
        mma16816(o[4 * w + 3], p[u], b10, b11);
      }
    }
  }
  // the accumulators' unit
  __device__ __forceinline__ float unit() const { return ref * (1.f / (1 << kPShift)); }
};

// What a warp knows of a block: its number in the cache (-1: unmapped, or past the end), the position
// of its first token (then far past every row) and its scales.
struct __align__(16) Block {
  int id, pos;
  float ks, vs;
};
constexpr int kBatch = 32;  // blocks that a warp looks up at once, one a lane

// A warp's copies. Lane 0 has TMA bring a pair of blocks' keys and values to the warp's buffer, each
// on an mbarrier of its own; a pair's keys are replaced by the next pair's once its scores are done,
// its values once they are accumulated, so either copy has the other half's work (and the SM's other
// warps) to arrive in. TMA for the copies because they are 2 KB rows of memory in one instruction:
// the same loop with 16-byte cp.async straight from the lanes' own places (64-byte pieces of rows)
// reached 4.7 TB/s with the arithmetic taken out, with TMA 6.4.
template <int D>
struct Copies {
  const CUtensorMap *mk, *mv;
  uint8_t* buffer;
  uint64_t* bars;  // keys, values
  uint32_t phase;  // of both: they are used in turn
  bool ok;

  __device__ __forceinline__ void init(const CUtensorMap* k, const CUtensorMap* v, uint8_t* buf, uint64_t* b, int lane) {
    mk = k;
    mv = v;
    buffer = buf;
    bars = b;
    phase = 0;
    ok = true;
    if (lane == 0) {
      bar_init(&bars[0], 1);
      bar_init(&bars[1], 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
  }
  // keys (which = 0) or values (1) of the pair's blocks that are there
  __device__ __forceinline__ void fetch(int which, const Block* pair, int lane) {
    if (lane == 0 && ok) {
      const int id0 = pair[0].id, id1 = pair[1].id;
      uint8_t* dst = buffer + which * 2 * Piece<D>::kBytes;
      bar_expect_tx(&bars[which], ((id0 >= 0) + (id1 >= 0)) * Piece<D>::kBytes);
      if (id0 >= 0) tma_tile(dst, which ? mv : mk, 0, id0 * kKvBlock, &bars[which]);
      if (id1 >= 0) tma_tile(dst + Piece<D>::kBytes, which ? mv : mk, 0, id1 * kKvBlock, &bars[which]);
    }
  }
  __device__ __forceinline__ void wait(int which) { ok = ok && kv8_wait(&bars[which], phase); }
  // At the kernel's end. After a wait that gave up nothing more is copied or waited for, but for
  // one last bounded wait for what was in flight then.
  __device__ __forceinline__ void finish(int* timeout) {
    if (ok) return;
    kv8_wait(&bars[0], phase);
    kv8_wait(&bars[1], phase);
    *timeout = 1;
  }
};

// ---------------------------------------------------------------------------------------------
// Decode. Rows are (sequence, kv head, run of up to 8 of its query heads); a row's units are its
// visible blocks, and kRowUnits more in front of them for what a row costs by itself. All units of
// the call, in order, are cut into equal shares, one a CTA (a CTA's warps take every fourth block of
// its segment of a row), so a batch of any mix of lengths fills the GPU evenly. A row whose blocks lie
// in one share is finished there; one cut by a share's end leaves an unnormalised part (running
// maximum, sum, 8 x D) in the workspace for kv8_join_kernel.
//
// Bound by HBM once the rows are long and D = 128: 64 x 2049 tokens of 32 heads in 185 us, 5.83 TB/s of
// the 6.55 that a copy reaches; 2 x 131071 of 8 heads 93 us. With D = 64 a pair of blocks has half the
// bytes and nearly all the ~560 warp instructions (its scores cost as many at any D), each step a
// chain that four warps of a scheduler do not hide (issue 0.53 a cycle, fixed waits the largest stall):
// window 4096 of 32 sequences, 40 us against 21 of traffic. What the short ones cost is latency, so a warp never lets its copies run dry: it looks
// up the next 32 blocks, of its next segment too, while it works on these, and fetches the first
// pair's keys of the next segment before it merges. At the start the pages and the queries are asked
// for together, and codes before scales (1 x 517 tokens 11.0 -> 10.4 us, ragged batch 61.8 -> 60.0).
constexpr int kDecWarps = 4;
// CTAs of an SM: D = 128 fills the registers at 3; with D = 64 (bound by its instructions' chain) 4 fit, too:
// 32 x window 4096, 40/8 heads of 64: 3 43.2 us, 4 41.0, 5 (spilling) 44.6.
constexpr int dec_ctas(int dim) { return dim == 64 ? 4 : 3; }
constexpr int kDecHeads = 8;
constexpr int kWholeTokens = 576;
constexpr int kRowUnits = 20;  // 12: ragged batch (48 x up to 8191 tokens) 64.2 us, 20: 60.0, 28: 61.1

struct DecArgs {
  AttnArgs a;
  int chunks;    // runs of 8 heads of a kv head
  float* part;   // [2 * CTAs][kDecHeads][D + 2]
  int64_t* cum;  // [batch + 1] units of the sequences before b
};

__device__ __forceinline__ int64_t row_units(const AttnArgs& a, int b) {
  const int len = kv8_length(a.lengths, b), n = span_of(len - 1, len - 1, a.window, a.sinks, a.cap).count();
  return n > 0 ? n + kRowUnits : 0;
}
// Units of a CTA: a whole number for each of its warps, the same for all CTAs (the last ones may get none).
__device__ __forceinline__ int64_t share_of(int64_t units, int ctas) {
  const int64_t each = (int64_t)ctas * kDecWarps;
  return kv8_quotient(units + each - 1, each) * kDecWarps;
}

// A CTA's part of a row: its blocks begin .. end - 1 of the row's nb.
struct Segment {
  int b, row, begin, end, nb, len;
  Span span;
  __device__ __forceinline__ int mine(int warp) const { return max(0, (end - begin - warp + kDecWarps - 1) / kDecWarps); }
};

// The share's segments one by one; false after the last.
struct Share {
  int b;
  int64_t at, left;  // the next unit among sequence b's, units left
  __device__ __forceinline__ bool next(const AttnArgs& a, int rows, Segment& s) {
    while (left > 0) {
      s.len = kv8_length(a.lengths, b);
      s.span = span_of(s.len - 1, s.len - 1, a.window, a.sinks, a.cap);
      s.nb = s.span.count();
      const int units = s.nb > 0 ? s.nb + kRowUnits : 0;
      if (at >= (int64_t)units * rows) {
        ++b;
        at = 0;
        continue;
      }
      s.b = b;
      s.row = (int)kv8_quotient(at, units);
      const int from = (int)(at - (int64_t)s.row * units), to = (int)min((int64_t)units, from + left);
      left -= to - from;
      at += to - from;
      s.begin = max(0, from - kRowUnits);
      s.end = to - kRowUnits;
      if (s.end > s.begin) return true;
    }
    return false;
  }
};

// where the merge keeps 4 floats c of head h's D: spread over the banks
__device__ __forceinline__ int merge_at(int h, int c, int d) { return h * d + 4 * (c ^ (((c >> 3) * 2 + (h & 1)) & 7)); }

// Where a CTA's share begins and the units of all. WHOLE: of its one row, whose units `total` are
// (rows that see nothing: zeros, and no share).
template <int D, bool WHOLE>
__device__ __forceinline__ Kv8Place find_share(const DecArgs& d, int rows, bool record) {
  const AttnArgs& a = d.a;
  if constexpr (WHOLE) {
    const int b = blockIdx.x / rows, row = blockIdx.x % rows;
    const int64_t units = row_units(a, b);
    if (units == 0) {
      const int head = row / d.chunks, h0 = head * a.group + row % d.chunks * kDecHeads, nh = min(kDecHeads, (head + 1) * a.group - h0);
      for (int e = threadIdx.x; e < nh * (D / 4); e += kDecWarps * 32)
        store4(a.out, a.out_type, ((int64_t)b * a.heads + h0) * D + 4 * e, make_float4(0.f, 0.f, 0.f, 0.f));
    }
    return {units == 0 ? -1 : b, row * units, units};
  } else {
    return kv8_find<kDecWarps * 32>(
        a.batch, [&](int b) -> int64_t { return row_units(a, b) * rows; },
        [&](int64_t units) -> int64_t { return share_of(units, gridDim.x) * blockIdx.x; },
        [&](int b0, int b1, int64_t before) {
          if (!record) return;
          for (int b = b0; b < b1; ++b) {
            d.cum[b] = before;
            before += row_units(a, b) * rows;
          }
          if (b1 == a.batch) d.cum[a.batch] = before;  // the threads past the last sequence write the same total
        });
  }
}

// WHOLE: a CTA per row, no shares and no join.
template <int D, bool WHOLE>
__global__ void __launch_bounds__(kDecWarps * 32, dec_ctas(D)) kv8_decode_kernel(const DecArgs d, const __grid_constant__ CUtensorMap mk,
                                                                              const __grid_constant__ CUtensorMap mv) {
  const AttnArgs& a = d.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_smem(smem_raw);
  __shared__ uint64_t bars[kDecWarps][2];
  __shared__ float2 states[kDecWarps][kDecHeads];  // (m, l)
  asm volatile("griddepcontrol.launch_dependents;");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int rows = a.c.kv_heads * d.chunks;
  const bool record = !WHOLE && blockIdx.x == 0;  // the sequences' first units, for the join
  const Kv8Place at = find_share<D, WHOLE>(d, rows, record);
  if (at.seq < 0) return;
  const int64_t share = WHOLE ? at.total : share_of(at.total, gridDim.x);
  Share work = {at.seq, at.at, WHOLE ? share : min(share, at.total - share * blockIdx.x)};
  // per warp: its copies (keys, values of a pair; the values' half holds its state in the merge) and
  // the blocks of this batch and of the next; per CTA: the row's queries
  uint8_t* buffer = smem + warp * Piece<D>::kBuffer;
  Block* blocks = reinterpret_cast<Block*>(smem + kDecWarps * Piece<D>::kBuffer) + warp * (2 * kBatch);
  uint4* queries = reinterpret_cast<uint4*>(smem + kDecWarps * (Piece<D>::kBuffer + 2 * kBatch * (int)sizeof(Block)));
  float* merge = reinterpret_cast<float*>(buffer + 2 * Piece<D>::kBytes);
  static_assert(2 * Piece<D>::kBytes >= kDecHeads * D * 4, "a warp's state must fit its values' buffer");
  Copies<D> copies;
  copies.init(&mk, &mv, buffer, bars[warp], lane);

  // Block i of this warp in a segment: first its page, then (once that is there) number and scales.
  auto page_of = [&](const Segment& s, int i, int count) -> int {
    if (i >= count) return -1;
    const int pg = s.span.block(s.begin + warp + kDecWarps * i) / a.c.bpp;
    return pg < a.t.width ? __ldg(a.t.pages + s.b * a.t.stride + pg) : -1;
  };
  auto look_up = [&](const Segment& s, int i, int page, Block* dst, auto numbered) {
    Block k = {-1, kNowhere, 0.f, 0.f};
    if ((unsigned)page < (unsigned)a.c.pages) {
      const int blk = s.span.block(s.begin + warp + kDecWarps * i);
      k.id = (page * a.c.kv_heads + s.row / d.chunks) * a.c.bpp + blk % a.c.bpp;
      k.pos = blk * kKvBlock;
      k.ks = __ldg(a.c.ks + k.id);
      k.vs = __ldg(a.c.vs + k.id);
    }
    // the numbers are there before the scales arrive, so that the first copies need not wait for those
    *reinterpret_cast<int2*>(&dst[lane]) = make_int2(k.id, k.pos);
    numbered();
    *reinterpret_cast<float2*>(&dst[lane].ks) = make_float2(k.ks, k.vs);
  };

  auto q_row = [&](const Segment& s) -> int64_t {  // of the lane's row, -1: none
    const int head = s.row / d.chunks, h = head * a.group + s.row % d.chunks * kDecHeads + g;
    return h < (head + 1) * a.group ? (int64_t)s.b * a.q_stride + (int64_t)h * D : -1;
  };

  Segment cur, nxt;
  Warp<D> w;
  bool more = work.next(a, rows, cur);
  int which = 0;  // half of `blocks` in use
  if (more) {
    const int page = page_of(cur, lane, cur.mine(warp));
    typename Warp<D>::Query query;
    Warp<D>::fetch_q(query, a.q, a.q_type, q_row(cur), lane);  // on their way with the pages, then the codes and scales
    look_up(cur, lane, page, blocks, [&] {
      __syncwarp();
      if (cur.mine(warp) > 0) {
        copies.fetch(0, blocks, lane);
        copies.fetch(1, blocks, lane);
      }
    });
    w.load_q(queries, query, a.scale_log2, lane, warp, kDecWarps);
    __syncwarp();
  }
  for (int done = 0; more; ++done, cur = nxt) {
    more = !WHOLE && work.next(a, rows, nxt);
    const int head = cur.row / d.chunks, h0 = head * a.group + cur.row % d.chunks * kDecHeads;
    const int nh = min(kDecHeads, (head + 1) * a.group - h0);
    const int first = a.window > 0 ? max(0, cur.len - a.window) : 0, last = cur.len - 1;
    w.reset();
    __syncthreads();
    const int mine = cur.mine(warp), next_mine = more ? nxt.mine(warp) : 0;
    for (int base = 0; base < mine; base += kBatch) {
      const int n = min(kBatch, mine - base);
      const bool same = base + kBatch < mine;  // the next batch is of this segment
      const int next_base = same ? base + kBatch : 0, next_n = same ? mine : next_mine;
      const int page = same ? page_of(cur, next_base + lane, next_n) : page_of(nxt, lane, next_n);
      const Block* now = blocks + which * kBatch;
      Block* then = blocks + (which ^ 1) * kBatch;
      const int look_at = min(4, (n - 1) & ~1);
      for (int i = 0; i < n; i += 2) {
        const Block b0 = now[i], b1 = now[i + 1];  // past n: not there
        const int p0[2] = {b0.pos, b1.pos};
        const float kk[2] = {b0.ks, b1.ks};
        float vv[2] = {b0.vs, b1.vs};
        const bool any = b0.id >= 0 || b1.id >= 0;
        const int far = max(p0[0], p0[1]) + kKvBlock, near = min(p0[0], p0[1]);
        const bool all = far <= cur.len && (near >= first || far <= a.sinks);
        if (i == look_at) look_up(same ? cur : nxt, next_base + lane, page, then, [] {});
        uint32_t p[2][4], seen;
        copies.wait(0);
        if (any)
          w.scores(buffer, kk, vv, all, first, last, a.sinks, p0, lane, p, seen, [&](int u, uint32_t see) {
            copies.wait(1);
            return Warp<D>::holds_values(buffer + 2 * Piece<D>::kBytes, u, see, lane);
          });
        __syncwarp();
        const bool end = i + 2 >= n;
        if (!end)
          copies.fetch(0, now + i + 2, lane);
        else if (next_n > next_base)
          copies.fetch(0, then, lane);
        copies.wait(1);
        if (any) w.values(buffer + 2 * Piece<D>::kBytes, p, seen, lane);
        __syncwarp();
        if (!end)
          copies.fetch(1, now + i + 2, lane);
        else if (same)
          copies.fetch(1, then, lane);
        copies.phase ^= 1;
      }
      which ^= 1;
    }
    if (mine == 0 && next_mine > 0) {  // a segment of fewer blocks than warps
      Block* then = blocks + (which ^ 1) * kBatch;
      look_up(nxt, lane, page_of(nxt, lane, next_mine), then, [] {});
      __syncwarp();
      copies.fetch(0, then, lane);
      which ^= 1;
    }
    // merge the warps
    const float l = quad_sum(w.l), unit = w.unit();
    if (g < nh) {
      if (t == 0) states[warp][g] = make_float2(w.m, l);
      // columns of tile j are dims (D / 8) n + j: this thread's n are 2t and 2t + 1
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < D / 8; j += 4)
          *reinterpret_cast<float4*>(merge + merge_at(g, ((D / 8) * (2 * t + n) + j) / 4, D)) =
              make_float4((w.o[j][n] + w.o[j][2 + n]) * unit, (w.o[j + 1][n] + w.o[j + 1][2 + n]) * unit,
                          (w.o[j + 2][n] + w.o[j + 2][2 + n]) * unit, (w.o[j + 3][n] + w.o[j + 3][2 + n]) * unit);
    }
    __syncthreads();
    const bool whole = WHOLE || (cur.begin == 0 && cur.end == cur.nb);
    for (int e = tid; e < nh * (D / 4); e += kDecWarps * 32) {
      const int h = e / (D / 4), c = e % (D / 4);
      float mt = -INFINITY;
#pragma unroll
      for (int i = 0; i < kDecWarps; ++i) mt = fmaxf(mt, states[i][h].x);
      float lt = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (mt != -INFINITY) {
#pragma unroll
        for (int i = 0; i < kDecWarps; ++i) {
          const float2 st = states[i][h];
          const float4 x = *reinterpret_cast<const float4*>(smem + i * Piece<D>::kBuffer + 2 * Piece<D>::kBytes + 4 * merge_at(h, c, D));
          const float f = exp2f(st.x - mt);
          lt = fmaf(st.y, f, lt);
          v.x = fmaf(x.x, f, v.x);
          v.y = fmaf(x.y, f, v.y);
          v.z = fmaf(x.z, f, v.z);
          v.w = fmaf(x.w, f, v.w);
        }
      }
      if (whole) {
        const float inv = mt == -INFINITY ? 0.f : 1.f / lt;
        store4(a.out, a.out_type, ((int64_t)cur.b * a.heads + h0 + h) * D + 4 * c, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
      } else {
        float* dst = d.part + (((int64_t)blockIdx.x * 2 + (done > 0)) * kDecHeads + h) * (D + 2);
        if (c == 0) *reinterpret_cast<float2*>(dst) = make_float2(mt, lt);
        *reinterpret_cast<float2*>(dst + 2 + 4 * c) = make_float2(v.x, v.y);
        *reinterpret_cast<float2*>(dst + 4 + 4 * c) = make_float2(v.z, v.w);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the values' half goes back to TMA
    __syncthreads();
    if (next_mine > 0) copies.fetch(1, blocks + which * kBatch, lane);
    if (more) {
      typename Warp<D>::Query query;
      Warp<D>::fetch_q(query, a.q, a.q_type, q_row(nxt), lane);
      w.load_q(queries, query, a.scale_log2, lane, warp, kDecWarps);
    }
  }
  copies.finish(a.timeout);
}

// Rows without a block give zeros; rows cut into parts are joined, in an order that only their
// lengths set. One CTA per (sequence, query head), its warps share the parts.
template <int D>
__global__ void __launch_bounds__(128) kv8_join_kernel(const DecArgs d, int ctas) {
  const AttnArgs& a = d.a;
  const int64_t i = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = (int)(i / a.heads), qh = (int)(i % a.heads);
  const int head = qh / a.group, chunk = qh % a.group / kDecHeads, h = qh % a.group % kDecHeads;
  __shared__ float sums[4][D];
  __shared__ float2 states[4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t before = d.cum[b], units = d.cum[a.batch];
  const int64_t row = kv8_quotient(d.cum[b + 1] - before, a.c.kv_heads * d.chunks);
  constexpr int kPer = D / 32;
  float acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
  float lt = 0.f, mt = -INFINITY;
  if (row > 0) {
    const int64_t share = share_of(units, ctas), u0 = before + (head * d.chunks + chunk) * row;
    const int c0 = (int)kv8_quotient(u0 + kRowUnits, share), c1 = (int)kv8_quotient(u0 + row - 1, share);
    if (c0 == c1) return;  // finished by its CTA
    // part i of the row is the first segment of CTA c0 + i, but for part 0 when c0 starts before the row
    const float* first = d.part + ((int64_t)(2 * c0 + (share * c0 < u0)) * kDecHeads + h) * (D + 2);
    const float* rest = d.part + ((int64_t)2 * (c0 + 1) * kDecHeads + h) * (D + 2);
    constexpr int64_t kNext = (int64_t)2 * kDecHeads * (D + 2);
    const int parts = c1 - c0 + 1;
    float head_start[kPer];  // of the warp's first part, while its state is on its way
#pragma unroll
    for (int e = 0; e < kPer; ++e) head_start[e] = warp < parts ? (warp == 0 ? first : rest + (warp - 1) * kNext)[2 + lane + 32 * e] : 0.f;
    // warp w takes parts w, w + 4, ..: lane j looks at the j-th of 32
    for (int base = 0; base * 4 < parts; base += 32) {
      const int mine = warp + 4 * (base + lane), n = min(32, (parts - warp + 3) / 4 - base);
      float2 ml = make_float2(-INFINITY, 0.f);
      if (mine < parts) ml = *reinterpret_cast<const float2*>(mine == 0 ? first : rest + (mine - 1) * kNext);
      float mn = ml.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mn = fmaxf(mn, mt);
      if (mn == -INFINITY) continue;
      const float old = exp2f(mt - mn), f = exp2f(ml.x - mn);  // 0 for parts that saw nothing
      mt = mn;
      float sum = f * ml.y;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      lt = lt * old + sum;
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] *= old;
#pragma unroll 8
      for (int p = 0; p < n; ++p) {
        const int at = warp + 4 * (base + p);
        const float fp = __shfl_sync(0xffffffffu, f, p);
        const float* src = (at == 0 ? first : rest + (at - 1) * kNext) + 2 + lane;
#pragma unroll
        for (int e = 0; e < kPer; ++e) acc[e] = fmaf(fp, at == warp ? head_start[e] : src[32 * e], acc[e]);
      }
    }
  }
  if (lane == 0) states[warp] = make_float2(mt, lt);
#pragma unroll
  for (int e = 0; e < kPer; ++e) sums[warp][lane + 32 * e] = acc[e];
  __syncthreads();
  if (tid >= D) return;
  float m = -INFINITY, l = 0.f, v = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) m = fmaxf(m, states[w].x);
  if (m != -INFINITY) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2f(states[w].x - m);
      l = fmaf(states[w].y, f, l);
      v = fmaf(sums[w][tid], f, v);
    }
    v /= l;
  }
  const int64_t o = i * D + tid;
  if (a.out_type == J4B_F32)
    static_cast<float*>(a.out)[o] = v;
  else
    static_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(v);
}

// Rows of one block of 16 tokens of D codes, swizzled as Piece<D>::at.
bool code_map(CUtensorMap* map, const uint8_t* codes, const Kv8View& v, int dim) {
  const auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)v.pages * v.kv_heads * v.bpp * kKvBlock};
  const cuuint64_t strides[1] = {(cuuint64_t)dim};
  const cuuint32_t box[2] = {(cuuint32_t)dim, kKvBlock}, ones[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// One word of page-locked host memory, which kernels of any device can write and the host reads
// without waiting: set when a bounded wait gave up, reported (and cleared) by the next call.
int* timeout_word() {
  static int* word = [] {
    void* p = nullptr;
    if (cudaHostAlloc(&p, sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped) != cudaSuccess) return (int*)nullptr;
    *(int*)p = 0;
    return (int*)p;
  }();
  return word;
}

int decode_ctas(int dev, int dim) {
  const DeviceCtx* ctx = device_ctx(dev);
  return dec_ctas(dim) * (ctx && ctx->sm_count > 0 ? ctx->sm_count : 148);
}

int64_t decode_bytes(int dim, int64_t batch, int ctas) {
  const int64_t part = (int64_t)2 * ctas * kDecHeads * (dim + 2) * 4;
  return (part + 15) / 16 * 16 + (batch + 1) * 8;
}

template <class Kernel>
int allow_smem(Kernel kernel, int bytes, int dev, bool (&done)[kMaxDevices]) {
  if (!done[dev]) {
    J4B_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "cudaFuncSetAttribute");
    done[dev] = true;
  }
  return J4B_OK;
}

template <int D, bool WHOLE>
int launch_decode_kernel(const DecArgs& d, int dev, int ctas, cudaStream_t stream) {
  static bool done[kMaxDevices] = {};
  const int smem = kDecWarps * (Piece<D>::kBuffer + 2 * kBatch * (int)sizeof(Block)) + 32 * D + 1024;
  CUtensorMap mk, mv;
  if (!code_map(&mk, d.a.c.k, d.a.c, D) || !code_map(&mv, d.a.c.v, d.a.c, D)) return set_error(J4B_ECUDA, "cuTensorMapEncodeTiled failed for the cache");
  if (const int st = allow_smem(kv8_decode_kernel<D, WHOLE>, smem, dev, done)) return st;
  kv8_decode_kernel<D, WHOLE><<<ctas, kDecWarps * 32, smem, stream>>>(d, mk, mv);
  J4B_CHECK_LAUNCH("kv8_decode_kernel");
  return J4B_OK;
}

template <int D>
int launch_decode(const DecArgs& d, int dev, int ctas, bool whole, cudaStream_t stream) {
  if (whole) return launch_decode_kernel<D, true>(d, dev, d.a.batch * d.a.c.kv_heads * d.chunks, stream);
  if (const int st = launch_decode_kernel<D, false>(d, dev, ctas, stream)) return st;
  // launched while the decode kernel runs: its CTAs wait for it on the device
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)((int64_t)d.a.batch * d.a.heads));
  config.blockDim = dim3(128);
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  J4B_CUDA(cudaLaunchKernelEx(&config, kv8_join_kernel<D>, d, ctas), "kv8_join_kernel");
  J4B_CHECK_LAUNCH("kv8_join_kernel");
  return J4B_OK;
}

}  // namespace

int kv8_check_attention(const j4b_kv8_cache* cache, int64_t layer, j4b_buf q, int q_type, int64_t q_stride, int64_t tokens, int64_t heads,
                    j4b_buf table, int64_t table_stride, int64_t table_width, j4b_buf lengths, int64_t batch, int64_t window, int64_t sinks,
                    double scale, j4b_buf out, int out_type, AttnArgs* a, int* dev) {
  Kv8View view;
  if (const int st = kv8_check(cache, layer, &view, dev)) return st;
  J4B_REQUIRE(heads > 0 && heads <= 65536 && heads % cache->kv_heads == 0, "kv8 attention: heads (%lld) must be a multiple of kv_heads (%d)",
              (long long)heads, cache->kv_heads);
  J4B_REQUIRE(batch >= 0 && batch <= 0xffffff && tokens >= 0 && tokens <= 0x7fffffff, "kv8 attention: bad batch or token count");
  J4B_REQUIRE((q_type == J4B_F32 || q_type == J4B_BF16) && (out_type == J4B_F32 || out_type == J4B_BF16),
              "kv8 attention: q and out types must be f32 or bf16, got %d and %d", q_type, out_type);
  J4B_REQUIRE(q_stride >= heads * cache->head_dim && q_stride % 8 == 0, "kv8 attention: rows of q must be at least heads * head_dim elements and a multiple of 8 apart");
  J4B_REQUIRE(table_width > 0 && table_width <= 0x7ffffff && table_stride >= table_width, "kv8 attention: bad page table shape");
  J4B_REQUIRE(window >= 0 && sinks >= 0, "kv8 attention: window and sinks must not be negative");
  J4B_REQUIRE(std::isfinite(scale), "kv8 attention: scale must be finite");
  if (batch > 0 && tokens > 0)
    J4B_REQUIRE(q && table && lengths && out && ((q | out) & 15) == 0 && ((table | lengths) & 3) == 0, "kv8 attention: misaligned or null buffers");
  const int64_t far = 0x3fffffff;
  *a = {view,
        {(const int*)(uintptr_t)table, table_stride, (int)table_width},
        (const void*)(uintptr_t)q,
        q_stride,
        q_type,
        (const int*)(uintptr_t)lengths,
        nullptr,
        tokens,
        (int)batch,
        (int)heads,
        (int)(heads / cache->kv_heads),
        (int)std::min(window, far),
        window > 0 ? (int)std::min(sinks, far) : 0,
        (int)std::min<int64_t>(table_width * view.bpp, 0x7fffffff / kKvBlock),
        (float)(scale * 1.4426950408889634),
        (void*)(uintptr_t)out,
        out_type,
        timeout_word()};
  if (!a->timeout) return set_error(J4B_ENOMEM, "kv8 attention: no host memory for the status word");
  if (*(volatile int*)a->timeout) {
    *(volatile int*)a->timeout = 0;
    return set_error(J4B_ETIMEOUT, "kv8 attention: a wait of an earlier call gave up; its output is not valid");
  }
  return J4B_OK;
}

}  // namespace j4b

using namespace j4b;

extern "C" int j4b_kv8_decode_workspace(const j4b_kv8_cache* cache, int64_t heads, int64_t batch, int64_t* bytes) {
  J4B_REQUIRE(bytes, "kv8 decode: bytes is null");
  Kv8View view;
  int dev = 0;
  if (const int st = kv8_check(cache, 0, &view, &dev)) return st;
  J4B_REQUIRE(heads > 0 && heads <= 65536 && heads % cache->kv_heads == 0, "kv8 decode: heads (%lld) must be a multiple of kv_heads (%d)",
              (long long)heads, cache->kv_heads);
  J4B_REQUIRE(batch >= 0 && batch <= 0xffffff, "kv8 decode: bad batch");
  *bytes = decode_bytes(cache->head_dim, batch, decode_ctas(dev, cache->head_dim));
  return J4B_OK;
}

extern "C" int j4b_kv8_attention_decode(const j4b_kv8_cache* cache, int64_t layer, j4b_buf q, int q_type, int64_t q_stride, int64_t heads,
                                        j4b_buf table, int64_t table_stride, int64_t table_width, j4b_buf lengths, int64_t batch,
                                        int64_t window, int64_t sinks, double scale, j4b_buf out, int out_type, j4b_buf workspace,
                                        int64_t workspace_bytes, j4b_stream s) {
  DecArgs d;
  int dev = 0;
  if (const int st = kv8_check_attention(cache, layer, q, q_type, q_stride, batch, heads, table, table_stride, table_width, lengths, batch,
                                     window, sinks, scale, out, out_type, &d.a, &dev))
    return st;
  J4B_REQUIRE(batch * heads <= 0x7fffffffLL, "kv8 decode: too many rows");
  if (batch == 0) return J4B_OK;
  const int ctas = decode_ctas(dev, cache->head_dim);
  J4B_REQUIRE(workspace && (workspace & 15) == 0 && workspace_bytes >= decode_bytes(cache->head_dim, batch, ctas),
              "kv8 decode: workspace must be 16-byte aligned and hold %lld bytes", (long long)decode_bytes(cache->head_dim, batch, ctas));
  DeviceGuard guard(dev);
  cudaStream_t stream = resolve_stream(dev, s);
  d.chunks = (d.a.group + kDecHeads - 1) / kDecHeads;
  // Few and short rows are done by a CTA each: no search for its share, no second launch. Measured on
  // 1 x 32/8 heads, whole against shared out: 1 token 5.1 against 7.9 us, 256 6.6 against 9.9, 517 10.4
  // against 10.3 (but 3 us less on the host), 768 11.8 against 10.4.
  const bool whole = batch * cache->kv_heads * d.chunks <= ctas && table_width * cache->page <= kWholeTokens;
  d.part = (float*)(uintptr_t)workspace;
  d.cum = (int64_t*)((uintptr_t)workspace + ((int64_t)2 * ctas * kDecHeads * (cache->head_dim + 2) * 4 + 15) / 16 * 16);
  return cache->head_dim == 128 ? launch_decode<128>(d, dev, ctas, whole, stream) : launch_decode<64>(d, dev, ctas, whole, stream);
}
