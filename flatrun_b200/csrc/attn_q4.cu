// Decode attention over the 4-bit paged cache: one query token for each of
// `batch` sequences of different lengths,
//
//   s_t = scale * q . k_t,   o = sum_t softmax(s)_t v_t,   t < length
//
// query head h reading KV head h / (nh / nkv).  A page number outside the
// cache hides the page's tokens, and a sequence of no (visible) tokens gives
// zeros, so no table can lead a read out of the cache.  Scores that all overflow
// to -inf leave 0 / 0: NaN, as prompt attention gives.
//
// Bound: a token and KV head is 5/4 HD bytes, read once for all its query
// heads, so HBM, if a value costs few instructions.  The products are
// therefore formed on the stored nibbles, and the scales are applied to sums:
//
//   s_t = sum_j d_tj (sum_{c in j} q_c n_tc) + sum_j m_tj (sum_{c in j} q_c)
//   o_c = sum_t (p_t d_tj) n_tc + sum_t p_t m_tj           (j the group of c)
//
// Two nibbles become two fp16 operands with two instructions: bits 0..3 under
// the exponent of 1024 are 1024 + n, bits 4..7 are 1024 + 16 n, and one add or
// fused multiply-add leaves n (or n - 8), exact.  (Without the exponent the
// bits are subnormals, exact too and an instruction less, but the tensor
// cores align the sum to the operands' exponents, not to their leading bits,
// which costs its last ten bits: fp32 results were off by 4e-5.)
//
//  * q . n: m16n8k16 with the query heads as rows (up to eight; the other eight
//    rows hold the low parts of fp32 queries), eight tokens as columns, channels as
//    the contraction, one accumulator a group; times d in fp32.  The queries
//    are scaled by a power of two to 2^14, so that fp16 holds them exactly for
//    16-bit types, and as a sum of two for fp32 (22 bits).
//  * m q: one more product, offsets (fp16 as stored) by the groups' query sums
//    as two fp16 each.
//  * p n: 16 channels of one group as rows, the heads as columns, 16 tokens as
//    the contraction; p d 2^-E is the fp16 operand, in two parts for fp32, rounded
//    once for fp16 (by 2^-11) and twice for bf16 (p and p d, an eighth of the
//    type's own rounding each).  The fragment of p is the one that the first
//    product leaves in the same lanes.
//  * p m: one more product, offsets as rows.
//    Here n - 8 and m + 8 d take the places of n and m: the sums then are as
//    large as the result, where sum p d n grows with the tokens and cancels
//    with sum p m (fp32: 2e-6 off at 4097 tokens), and roundings of p d count
//    relative to a value's distance from its group's middle.  m + 8 d is in two
//    parts for fp32, rounded to fp16 for 16-bit types as the stored m is.
//
// Range: the softmax's reference, the largest s, has p = 2^11 to 2^15, so p is a
// normal fp16 number down to 2^-25 of it, and smaller ones are off by 2^-36 of it.  The
// steps of a place have to lie within a window, 0 or 2^(E-12) to 2^E, and its |m + 8 d|
// below 2^(E+11) and fp16's largest.  Then what p d 2^-E loses below fp16's normal
// numbers is 2^-25 at most, against 2^11 2^-12 of the reference's smallest step: 2^-24.
// E is 2, for values between some hundredths and some tens; where a warp's first block
// of a unit does not fit that, four to eight times its largest step.  Blocks outside the
// window (tokens or groups of far larger or smaller values than the rest, groups that
// are not finite, values above 65504) are added in fp32 on the CUDA cores, whatever they
// hold: a call of nothing else takes 213 us where ordinary values take 56 (4 sequences of
// 32768 tokens, 32 / 8 heads of 128, bf16).  Taken from scores and steps together, as it
// was, the reference let a token of small weight and a large step take the bits of the
// others' weights; the check of the window costs 2 to 3 % (batch of 128 66.7 -> 68.1 us,
// 131071 tokens 57.6 -> 59.5 us).
//
// Split: all sequences' tokens, 32 (two blocks) a place, for each KV head (and
// part of eight query heads: a unit), form one line, with one empty place before
// each unit for the work of opening and closing it.  The line is cut into equal
// ranges, one a warp, 16 warps an SM: lengths need not be known to the host and
// may differ at will.  A warp streams its blocks through its own ring of shared
// memory (one bulk copy a block: it is contiguous; the page numbers of 16
// places are looked up at once, a block a lane, a batch ahead) and writes the
// units that lie wholly in its range.  (Whole CTAs on one unit with their warps
// taking blocks in turn spent 3 us on each short sequence's head: 404 us for a
// batch of 128 that takes 68 now.)  A unit that a boundary cuts is joined from its
// pieces, by the CTA where the CTA has all of them, otherwise from pieces that
// the CTAs leave in the workspace, by a second kernel.
//
// Measured: 128 sequences of 1 to 8192 tokens, 64 / 8 heads of 128, bf16: 68 us
// (190 MB of cache: 2.8 TB/s, 0.43 of a plain copy); 131071 tokens, 32 / 8 heads,
// fp16: 59 us.  36 million warp instructions (490 a block of 16 tokens and KV head,
// with all around the loop) would take 32 us at full issue; the slots are 60 % busy.  What
// binds is latency at 16 warps an SM (128 registers a thread; for head_dim 128 some spill:
// 64 bytes stored and 136 loaded for 16-bit types, 104 and 188 for fp32) and the work
// outside the loop: opening 7 us, joining 3, the second kernel 5, waiting for the last CTAs.
#include <cuda_runtime.h>

#include <atomic>
#include <cstdio>

#include "../../include/frcuda.h"
#include "gemv.cuh"
#include "kv_q4.cuh"

namespace frc {

struct AttnQ4Params {
  const void* q;
  int64_t q_seq, q_head;
  const uint8_t* cache;
  int64_t pages;
  int blocks_per_page;
  const int* table;
  int64_t table_stride;
  int max_pages;  // entries of a table row
  const int* lengths;
  int batch, nh, nkv;
  int parts;  // parts of up to eight query heads of a KV head
  float scale;
  void* out;
  int64_t o_seq, o_head;
  int q_vec, o_vec;  // rows allow vector loads / stores
  float* part;       // workspace: [2 grid][8][HD + 4] pieces that CTAs leave (max, sum, -, -, o)
  float* first;      // workspace: [8 grid][8][HD + 4] warps' first pieces
  int4* desc;        // workspace: [grid] (sequence, unit, CTAs that follow, -), a head cut at the CTA's end
  uint32_t* status;
  uint32_t bias;  // 0x64006400, the halves 1024: a parameter, so that it stays in a register
};

constexpr int kAqWarps = 8;
constexpr int kAqThreads = kAqWarps * 32;
constexpr int kAqHeads = 8;                       // query heads a unit
constexpr int kAqGrid = 2 * 148;
constexpr int kAqMinPlaces = kAqWarps;            // places a CTA, at least: one for each warp

// The window of a warp's steps (comment on top), in shared memory: halves in pairs.
struct alignas(16) AqWindow {
  float down;  // 2^-E
  uint32_t hi, lo, mid;
};

constexpr AqWindow kWindow{0.25f, 0x44004400u, 0x14001400u, 0x70007000u};  // E = 2: 2^-2, 4, 2^-10, 2^13

template <int HD>
struct AqSmem {
  static constexpr int kStages = HD == 128 ? 2 : 4;  // places in flight for each warp
  static constexpr int kBlock = 20 * HD;
  static constexpr int kRow = HD + 4;  // floats of a head in a piece
  static constexpr int kPieces = 2 * kAqWarps;  // of each warp: the unit that ends in its range, the one that goes on
  alignas(128) uint8_t ring[kAqWarps][kStages][2][kBlock];
  alignas(16) float m[kAqHeads][kPieces], l[kAqHeads][kPieces];
  int4 piece[kPieces];  // (sequence or -1, unit, start, end) in places of the CTA's range
  AqWindow window[kAqWarps];
  uint64_t full[kAqWarps][kStages];
  int64_t scan[kAqWarps];
  int64_t first_start;  // place of sequence first_seq in the line
  int first_seq;
  int abort;
  static_assert(kAqHeads * kRow * 4 <= 2 * kStages * kBlock, "a piece fits the ring");
};

// The sum of no weights: -0, which stays -0 until a token's weight is added, if only
// +0 (of a score of -inf), and through products with factors that are not negative.
constexpr float kNoTokens = -0.f;

FRC_DEVICE_INLINE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

FRC_DEVICE_INLINE void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same into a fresh accumulator.
FRC_DEVICE_INLINE void mma16816_new(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

FRC_DEVICE_INLINE uint32_t h2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
FRC_DEVICE_INLINE __half2 bits_h2(uint32_t b) { return *reinterpret_cast<const __half2*>(&b); }
FRC_DEVICE_INLINE uint32_t pack_half2(float lo, float hi) { return h2_bits(__floats2half2_rn(lo, hi)); }

// (w & MASK) | bias in one instruction: the mask is its one constant, the
// exponents of 1024 a register.
template <uint32_t MASK>
FRC_DEVICE_INLINE uint32_t and_or(uint32_t w, uint32_t bias) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "n"(MASK), "r"(bias));
  return v;
}

// Nibbles 0 and 4 (LOW) or 1 and 5 of a word as the halves n - B.
template <bool LOW, int B>
FRC_DEVICE_INLINE uint32_t nibbles(uint32_t w, uint32_t bias) {
  if constexpr (LOW)
    return h2_bits(__hadd2(bits_h2(and_or<0x000f000fu>(w, bias)), __float2half2_rn(-1024.f - B)));
  else
    return h2_bits(__hfma2(bits_h2(and_or<0x00f000f0u>(w, bias)), __float2half2_rn(0.0625f),
                           __float2half2_rn(-64.f - B)));
}

// Tokens of a sequence that the table covers.
FRC_DEVICE_INLINE int aq_length(const AttnQ4Params& p, int b) {
  const int64_t room = static_cast<int64_t>(p.max_pages) * p.blocks_per_page * kQ4Tokens;
  const int n = p.lengths[b];
  return n < 0 ? 0 : (n < room ? n : static_cast<int>(room));
}
// 32-token places of a sequence.
FRC_DEVICE_INLINE int aq_places(int length) { return static_cast<int>((static_cast<int64_t>(length) + 31) >> 5); }

// Walks the line: the unit that holds a place.  Places count from the start
// of the CTA's range (a unit may start before it).
struct AqWalk {
  int seq, unit, len, np;  // tokens and places of the sequence
  int u0;                  // place of the unit, which has np + 1
  FRC_DEVICE_INLINE void sequence(const AttnQ4Params& p, int s) {
    seq = s;
    len = aq_length(p, s);
    np = aq_places(len);
  }
  FRC_DEVICE_INLINE int end() const { return u0 + np + 1; }
  FRC_DEVICE_INLINE void to(const AttnQ4Params& p, int place, int units) {
    while (place >= end()) {
      u0 = end();
      if (++unit == units) {
        unit = 0;
        sequence(p, seq + 1);
      }
    }
  }
};

// One warp's running state for a unit: O^T fragments, offsets' sums, and the
// softmax reference and sum of head lane / 4.
template <int HD, typename T>
struct AqWarp {
  static constexpr int NG = HD / kQ4Group;
  static constexpr bool SPLIT = sizeof(T) == 4;  // operands in two parts
  static constexpr bool TWICE = std::is_same<T, __nv_bfloat16>::value;  // p rounded to 11 bits before p d is
  // p at the reference is 2^kLift, and may be 2^kSlack times that: below fp16's 65504
  static constexpr float kLift = 11.f, kSlack = 4.f;
  static constexpr float kLow = 2048.f;  // of the low parts of fp32 weights and offsets
  uint32_t a[NG][2][4];  // query fragments: (group, k step): rows 0-7 of both k halves, rows 8-15 (low parts) of both
  uint32_t am;                       // groups' query sums
  AqWindow* win;
  float f_n, f_m;                    // scale of the two score products, with log2 e
  float o[NG][2][4], om[4];
  float m_run, base, l_run;  // the reference, what is taken off the scores, the sum of p

  // q of head lane / 4: this lane holds channels 32 j + 8 (lane & 3) .. + 7.
  FRC_DEVICE_INLINE void load_q(const float (&x)[NG][8], float scale, int lane) {
    float mx = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[j][i]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // 2^(14 - exponent): the largest becomes 2^14 .. 2^15
    const int e = max(static_cast<int>(__float_as_uint(mx) >> 23) - 127, -100);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
    const float down = __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
    f_n = scale * 1.44269504088896341f * down;
    f_m = scale * 1.44269504088896341f * down * 64.f;
    if (mx == INFINITY) f_n = f_m = NAN;  // every score is infinite or NaN: so is the softmax
    float sum[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      float y[8], lo[8];
      sum[j] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = x[j][i] * up;
        sum[j] += y[i];
        if constexpr (SPLIT) {
          const float h = __half2float(__float2half_rn(y[i]));
          lo[i] = (y[i] - h) * 2048.f;
          y[i] = h;
        }
      }
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
      sum[j] *= 1.f / 64.f;
      // nibble i of a word: k step i / 2 % 2, k half i % 2, low or high half i / 4
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        a[j][s][0] = pack_half2(y[2 * s], y[2 * s + 4]);
        a[j][s][1] = pack_half2(y[2 * s + 1], y[2 * s + 5]);
        if constexpr (SPLIT) {
          a[j][s][2] = pack_half2(lo[2 * s], lo[2 * s + 4]);
          a[j][s][3] = pack_half2(lo[2 * s + 1], lo[2 * s + 5]);
        } else {  // zeros that the compiler keeps in place: the fragment is four neighbouring registers
          asm volatile("mov.b32 %0, 0;" : "=r"(a[j][s][2]));
          asm volatile("mov.b32 %0, 0;" : "=r"(a[j][s][3]));
        }
      }
    }
    // contraction index 2 q, 2 q + 1: the sums of two groups, high parts first, then low parts
    const int q = lane & 3, pair = q % (NG / 2), part = q / (NG / 2);
    float s0 = sum[0], s1 = sum[1];
    if constexpr (NG == 4)
      if (pair) {
        s0 = sum[2];
        s1 = sum[3];
      }
    const float h0 = __half2float(__float2half_rn(s0)), h1 = __half2float(__float2half_rn(s1));
    am = part == 0 ? pack_half2(h0, h1) : (part == 1 ? pack_half2(s0 - h0, s1 - h1) : 0u);
  }

  FRC_DEVICE_INLINE void reset(int lane) {
    __syncwarp();
    if (lane == 0) *win = kWindow;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][s][i] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) om[i] = 0.f;
    m_run = -INFINITY;
    base = 0.f;
    l_run = kNoTokens;
  }

  // Lane (r, q) = (lane / 4, lane % 4) has tokens 4 q .. 4 q + 3 of a block.

  // Scores of a block in shared memory, of which (TAIL) `left` tokens belong to
  // the sequence.
  template <bool TAIL>
  FRC_DEVICE_INLINE void scores(const uint8_t* blk, int left, int lane, uint32_t bias, float (&s)[4]) {
    constexpr Q4Layout lay(HD);
    const int r = lane >> 2, q = lane & 3;
    uint2 kd[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) kd[j] = *reinterpret_cast<const uint2*>(blk + lay.k_step(j, 4 * q));
#pragma unroll
    for (int t = 0; t < 2; ++t) {  // two tiles of eight tokens: column n is token 4 (n / 2) + 2 t + n % 2
      const int tok = 4 * (r >> 1) + 2 * t + (r & 1);
      uint32_t w[NG];
      if constexpr (NG == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(blk + lay.k_word(tok, q, 0));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(blk + lay.k_word(tok, q, 0));
        w[0] = v.x; w[1] = v.y;
      }
      float cm[4];
      uint64_t x = 0;  // the scores of tokens 4 q + 2 t and the next, of head r
      mma16816_new(cm, am, 0u, 0u, 0u, *reinterpret_cast<const uint32_t*>(blk + lay.k_offset(tok, 2 * (q % (NG / 2)))),
                   0u);
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        float c[4];
        const uint32_t hi = w[j] >> 8;
        mma16816_new(c, a[j][0][0], a[j][0][2], a[j][0][1], a[j][0][3], nibbles<true, 0>(w[j], bias),
                     nibbles<false, 0>(w[j], bias));
        mma16816(c, a[j][1][0], a[j][1][2], a[j][1][1], a[j][1][3], nibbles<true, 0>(hi, bias),
                 nibbles<false, 0>(hi, bias));
        if constexpr (SPLIT) {
          c[0] = fmaf(c[2], 1.f / 2048.f, c[0]);
          c[1] = fmaf(c[3], 1.f / 2048.f, c[1]);
        }
        const float2 d = __half22float2(bits_h2(t ? kd[j].y : kd[j].x));
        const uint64_t d2 = f32x2_two(d.x, d.y), c2 = f32x2_two(c[0], c[1]);
        x = j ? f32x2_fma(d2, c2, x) : f32x2_mul(d2, c2);
      }
      float x0, x1;
      f32x2_split(x, x0, x1);
      s[2 * t] = fmaf(x0, f_n, cm[0] * f_m);
      s[2 * t + 1] = fmaf(x1, f_n, cm[1] * f_m);
    }
    if constexpr (TAIL) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i >= left - 4 * q) s[i] = -INFINITY;
    }
  }

  // Masks of the lane's first and second pair of tokens, of which `mine` count:
  // what lies behind the last token may be anything, NaN among it.
  static FRC_DEVICE_INLINE void own_tokens(int mine, uint32_t& k0, uint32_t& k1) {
    k0 = mine >= 2 ? 0xffffffffu : (mine == 1 ? 0xffffu : 0u);
    k1 = mine >= 4 ? 0xffffffffu : (mine == 3 ? 0xffffu : 0u);
  }

  // The place's steps and middles m + 8 d as one lane sees them: lane (r, q) has group
  // r % NG and tokens 4 q .. 4 q + 3 of block r / NG, where bit r / NG of `present` is set.
  struct Extent {
    __half2 top, mid;  // largest step, largest |m + 8 d|: NaN if one is
    __half2 d0, d1;
  };
  static FRC_DEVICE_INLINE Extent extent(const uint8_t (*blk)[20 * HD], uint32_t present, int left, int lane) {
    constexpr Q4Layout lay(HD);
    const int r = lane >> 2, q = lane & 3, e = r / NG, j = r % NG;
    uint2 m = make_uint2(0u, 0u), d = m;
    if (present >> e & 1u) {
      m = *reinterpret_cast<const uint2*>(blk[e] + lay.v_offset(j, 4 * q));
      d = *reinterpret_cast<const uint2*>(blk[e] + lay.v_step(j, 4 * q));
      if (left < 2 * kQ4Tokens) {
        uint32_t k0, k1;
        own_tokens(left - e * kQ4Tokens - 4 * q, k0, k1);
        m.x &= k0;
        d.x &= k0;
        m.y &= k1;
        d.y &= k1;
      }
    }
    const __half2 eight = __float2half2_rn(8.f), d0 = bits_h2(d.x), d1 = bits_h2(d.y);
    return {__hmax2_nan(d0, d1),
            __hmax2_nan(__habs2(__hfma2(d0, eight, bits_h2(m.x))), __habs2(__hfma2(d1, eight, bits_h2(m.y)))), d0, d1};
  }
  static FRC_DEVICE_INLINE bool fits(const Extent& x, const AqWindow& w) {
    const __half2 lo = bits_h2(w.lo);
    // steps below the window, but for zeros
    const __half2 small = __hfma2(__hlt2(x.d0, lo), x.d0, __hmul2(__hlt2(x.d1, lo), x.d1));
    return __hble2(x.top, bits_h2(w.hi)) && __hble2(x.mid, bits_h2(w.mid)) && __hbeq2(small, bits_h2(0u));
  }
  // The window chosen for a block's steps: true if they fit then (if not, it stays as it was).
  FRC_DEVICE_INLINE bool adopt(const Extent& x, int lane) {
    const float mine = fmaxf(__low2float(x.top), __high2float(x.top));  // (NaN, or below 0: does not fit)
    const uint32_t top = __reduce_max_sync(0xffffffffu, mine > 0.f ? __float_as_uint(mine) : 0u);
    const int e = min(max(static_cast<int>(top >> 23) - 127 + 3, -12), 16);
    auto power = [](int n) { return __uint_as_float(static_cast<uint32_t>(127 + n) << 23); };
    auto both = [](float v) { return h2_bits(__float2half2_rn(fminf(v, 65504.f))); };
    const AqWindow w{power(-e), both(power(e)), both(power(e - 12)), both(power(e + 11))};
    const bool fit = __all_sync(0xffffffffu, fits(x, w));
    if (fit && lane == 0) *win = w;
    __syncwarp();
    return fit;
  }

  // The reference raised, where it has to be, to m (the largest score of the lane's
  // tokens) and the other lanes' of the head.  It may stay up to kSlack below: the
  // operands have that room, and most raises of a running maximum are small.  True: the
  // place does not fit the window.
  FRC_DEVICE_INLINE bool refer(float m, bool fit, int lane) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const bool up = m > m_run + kSlack;
    if (!__any_sync(0xffffffffu, up || !fit)) return false;
    if (__any_sync(0xffffffffu, up)) {
      const int q = lane & 3;
      const float m_new = fmaxf(m, m_run);
      const float keep = m_new == -INFINITY ? 1.f : ex2(m_run - m_new);
      const float f0 = __shfl_sync(0xffffffffu, keep, 8 * q), f1 = __shfl_sync(0xffffffffu, keep, 8 * q + 4);
#pragma unroll
      for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          o[j][t][0] *= f0;
          o[j][t][1] *= f1;
          o[j][t][2] *= f0;
          o[j][t][3] *= f1;
        }
      om[0] *= f0;
      om[1] *= f1;
      l_run *= keep;
      m_run = m_new;
      base = m_new == -INFINITY ? 0.f : m_new - kLift;
    }
    return !__all_sync(0xffffffffu, fit);
  }

  // The block's values, weighted by its scores: a block that fits the window.
  template <bool TAIL>
  FRC_DEVICE_INLINE void values(const uint8_t* blk, int left, int lane, uint32_t bias, const float (&s)[4]) {
    constexpr Q4Layout lay(HD);
    const int r = lane >> 2, q = lane & 3;
    uint2 vd[NG], vm = make_uint2(0u, 0u), vml = make_uint2(0u, 0u);
#pragma unroll
    for (int j = 0; j < NG; ++j) vd[j] = *reinterpret_cast<const uint2*>(blk + lay.v_step(j, 4 * q));
    if (r < NG) {  // offsets m + 8 d of n - 8, in two parts for fp32
      vm = *reinterpret_cast<const uint2*>(blk + lay.v_offset(r, 4 * q));
      const uint2 d = *reinterpret_cast<const uint2*>(blk + lay.v_step(r, 4 * q));
      if constexpr (SPLIT) {
        offset_parts(d.x, vm.x, vml.x);
        offset_parts(d.y, vm.y, vml.y);
      } else {
        vm.x = h2_bits(__hfma2(bits_h2(d.x), __float2half2_rn(8.f), bits_h2(vm.x)));
        vm.y = h2_bits(__hfma2(bits_h2(d.y), __float2half2_rn(8.f), bits_h2(vm.y)));
      }
    }
    if constexpr (TAIL) {
      uint32_t k0, k1;
      own_tokens(left - 4 * q, k0, k1);
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        vd[j].x &= k0;
        vd[j].y &= k1;
      }
      vm.x &= k0;
      vm.y &= k1;
      vml.x &= k0;
      vml.y &= k1;
    }
    const float p0 = ex2(s[0] - base), p1 = ex2(s[1] - base), p2 = ex2(s[2] - base), p3 = ex2(s[3] - base);
    l_run += (p0 + p1) + (p2 + p3);
    const uint32_t h01 = pack_half2(p0, p1), h23 = pack_half2(p2, p3);
    uint32_t l01 = 0u, l23 = 0u;  // fp32: 2^11 times the rest of p, so that it stays above fp16's subnormals
    if constexpr (SPLIT) {
      const float2 g01 = __half22float2(bits_h2(h01)), g23 = __half22float2(bits_h2(h23));
      l01 = pack_half2((p0 - g01.x) * kLow, (p1 - g01.y) * kLow);
      l23 = pack_half2((p2 - g23.x) * kLow, (p3 - g23.y) * kLow);
    }
    if constexpr (SPLIT) {
      float c[4], low[4];
      mma16816_new(low, vm.x, 0u, vm.y, 0u, l01, l23);
      mma16816(low, vml.x, 0u, vml.y, 0u, h01, h23);
      mma16816_new(c, vm.x, 0u, vm.y, 0u, h01, h23);
      om[0] += fmaf(low[0], 1.f / kLow, c[0]);
      om[1] += fmaf(low[1], 1.f / kLow, c[1]);
    } else {
      mma16816(om, vm.x, 0u, vm.y, 0u, h01, h23);
    }
    // rows of a tile: 16 channels of group j: word 4 j + r % 4, of it the nibbles
    // of its low half (r < 4) or high half: 2 t in row r, 2 t + 1 in row r + 8
    const uint32_t sel = r < 4 ? 0x5410u : 0x7632u;
    const float down = win->down;
    const uint64_t r01 = f32x2_two(p0 * down, p1 * down), r23 = f32x2_two(p2 * down, p3 * down);
    const __half2 down2 = __float2half2_rn(down);  // (a step in the window times it is exact)
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const uint4 v = *reinterpret_cast<const uint4*>(blk + lay.v_word(4 * j + (r & 3), 4 * q));
      const uint32_t w0 = __byte_perm(v.x, v.y, sel), w1 = __byte_perm(v.z, v.w, sel);
      uint32_t b0, b1, c0 = 0u, c1 = 0u;
      if constexpr (TWICE) {
        b0 = h2_bits(__hmul2(bits_h2(h01), __hmul2(bits_h2(vd[j].x), down2)));
        b1 = h2_bits(__hmul2(bits_h2(h23), __hmul2(bits_h2(vd[j].y), down2)));
      } else {
        const float2 e0 = __half22float2(bits_h2(vd[j].x)), e1 = __half22float2(bits_h2(vd[j].y));
        float y0, y1, y2, y3;
        f32x2_split(f32x2_mul(r01, f32x2_two(e0.x, e0.y)), y0, y1);
        f32x2_split(f32x2_mul(r23, f32x2_two(e1.x, e1.y)), y2, y3);
        b0 = pack_half2(y0, y1);
        b1 = pack_half2(y2, y3);
        if constexpr (SPLIT) {
          const float2 g0 = __half22float2(bits_h2(b0)), g1 = __half22float2(bits_h2(b1));
          c0 = pack_half2(y0 - g0.x, y1 - g0.y);
          c1 = pack_half2(y2 - g1.x, y3 - g1.y);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t u0 = t ? w0 >> 8 : w0, u1 = t ? w1 >> 8 : w1;
        const uint32_t n0 = nibbles<true, 8>(u0, bias), n1 = nibbles<false, 8>(u0, bias);
        const uint32_t n2 = nibbles<true, 8>(u1, bias), n3 = nibbles<false, 8>(u1, bias);
        if constexpr (SPLIT) {
          // into a fresh accumulator: the tensor cores cut their sums (towards zero),
          // which over thousands of tokens takes 2e-6 off a running one
          float c[4];
          mma16816_new(c, n0, n1, n2, n3, c0, c1);
          mma16816(c, n0, n1, n2, n3, b0, b1);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][t][i] += c[i];
        } else {
          mma16816(o[j][t], n0, n1, n2, n3, b0, b1);
        }
      }
    }
  }

  // The same for any block, in fp32: `left` tokens of it, each lane its channels of its
  // two heads.
  FRC_DEVICE_INLINE void values_apart(const uint8_t* blk, int left, int lane, const float (&s)[4]) {
    constexpr Q4Layout lay(HD);
    const int r = lane >> 2, q = lane & 3;
    const float p0 = ex2(s[0] - base), p1 = ex2(s[1] - base), p2 = ex2(s[2] - base), p3 = ex2(s[3] - base);
    l_run += (p0 + p1) + (p2 + p3);
    const float down = win->down;
#pragma unroll 1
    for (int tok = 0; tok < min(left, kQ4Tokens); ++tok) {
      const int i = tok & 3;
      const float mine = (i & 2 ? (i & 1 ? p3 : p2) : (i & 1 ? p1 : p0)) * down;
      const float f0 = __shfl_sync(0xffffffffu, mine, 8 * q + (tok >> 2));
      const float f1 = __shfl_sync(0xffffffffu, mine, 8 * q + 4 + (tok >> 2));
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const uint32_t w = *reinterpret_cast<const uint16_t*>(blk + lay.v_word(4 * j + (r & 3), tok) + 2 * (r >> 2));
        const float d = __half2float(*reinterpret_cast<const __half*>(blk + lay.v_step(j, tok)));
        const float m = __half2float(*reinterpret_cast<const __half*>(blk + lay.v_offset(j, tok)));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float v = fmaf(static_cast<float>(w >> (4 * k) & 15u), d, m);
          float* at = &o[j][k >> 1][2 * (k & 1)];
          at[0] = fmaf(f0, v, at[0]);
          at[1] = fmaf(f1, v, at[1]);
        }
      }
    }
  }

  static FRC_DEVICE_INLINE float largest(const float (&s)[4], float m) {
    return fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), m);
  }

  // The blocks of a place (bit e of `seen`: block e is there), of which `left`
  // tokens belong to the sequence.
  FRC_DEVICE_INLINE void place(const uint8_t (*blk)[20 * HD], uint32_t seen, int left, int lane, uint32_t bias) {
    if (left >= 2 * kQ4Tokens && seen == 3u) {
      float s0[4], s1[4];
      scores<false>(blk[0], 0, lane, bias, s0);
      scores<false>(blk[1], 0, lane, bias, s1);
      const bool fit = fits(extent(blk, 3u, 2 * kQ4Tokens, lane), *win);
      if (!refer(largest(s0, largest(s1, -INFINITY)), fit, lane) ) {
        values<false>(blk[0], 0, lane, bias, s0);
        values<false>(blk[1], 0, lane, bias, s1);
        return;
      }
    }
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      if (!(seen >> e & 1u)) continue;
      float s[4];
      scores<true>(blk[e], left - e * kQ4Tokens, lane, bias, s);
      const Extent x = extent(blk, 1u << e, left, lane);
      bool fit = __all_sync(0xffffffffu, fits(x, *win));
      if (!fit && __float_as_uint(l_run) == 0x80000000u) fit = adopt(x, lane);  // (no token yet)
      if (!refer(largest(s, -INFINITY), fit, lane) )
        values<true>(blk[e], left - e * kQ4Tokens, lane, bias, s);
      else
        values_apart(blk[e], left - e * kQ4Tokens, lane, s);
    }
  }

  // Two tokens' m + 8 d as the sum of two halves each, the second times kLow: m
  // becomes the high part.
  static FRC_DEVICE_INLINE void offset_parts(uint32_t d, uint32_t& m, uint32_t& low) {
    const float2 df = __half22float2(bits_h2(d)), mf = __half22float2(bits_h2(m));
    const float x = fmaf(df.x, 8.f, mf.x), y = fmaf(df.y, 8.f, mf.y);
    m = pack_half2(x, y);
    const float2 h = __half22float2(bits_h2(m));
    low = pack_half2((x - h.x) * kLow, (y - h.y) * kLow);
  }

  // The warp's sums: f(head, channel, o[4]) for this lane's channels of its two
  // heads, after l of head lane / 4 has been summed over its tokens.
  template <typename F>
  FRC_DEVICE_INLINE void sums(int lane, F&& f) {
    const int r = lane >> 2, q = lane & 3;
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
    const float up = __uint_as_float((254u << 23) - __float_as_uint(win->down));  // 1 / 2^-E
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float l = __shfl_sync(0xffffffffu, l_run, 4 * (2 * q + e));
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const float m = __shfl_sync(0xffffffffu, om[e], 4 * j + q);
        const float v[4] = {fmaf(o[j][0][e], up, m), fmaf(o[j][0][2 + e], up, m), fmaf(o[j][1][e], up, m),
                            fmaf(o[j][1][2 + e], up, m)};
        f(2 * q + e, kQ4Group * j + 8 * (r & 3) + 4 * (r >> 2), v, l);
      }
    }
  }
};

// The eight query heads of a unit.
struct AqHeads {
  int first, count;
  FRC_DEVICE_INLINE AqHeads(const AttnQ4Params& p, int unit) {
    const int group = p.nh / p.nkv, kvh = unit / p.parts;
    first = kvh * group + (unit - kvh * p.parts) * kAqHeads;
    count = min(kAqHeads, (kvh + 1) * group - first);
  }
};

template <int N, typename T>
FRC_DEVICE_INLINE void aq_store(const AttnQ4Params& p, int seq, int head, int c, float (&v)[N], float l) {
  const float inv = __float_as_uint(l) == 0x80000000u ? 0.f : 1.f / l;  // kNoTokens; 0: 0 / 0
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] *= inv;
  T* op = static_cast<T*>(p.out) + seq * p.o_seq + head * p.o_head + c;
  if (p.o_vec) store_run<N, true>(op, v);
  else store_run<N, false>(op, v);
}

template <typename T, int HD>
__global__ void __launch_bounds__(kAqThreads, 2) attn_q4_kernel(const AttnQ4Params p) {
  griddep_wait();
  griddep_launch_dependents();
  using SM = AqSmem<HD>;
  constexpr int NS = SM::kStages, NG = HD / kQ4Group;
  extern __shared__ __align__(128) uint8_t aq_smem[];
  SM* sh = reinterpret_cast<SM*>(aq_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int units = p.nkv * p.parts;

  // ---- the line and this CTA's range of it ----------------------------------------
  const int per_thread = (p.batch + kAqThreads - 1) / kAqThreads;
  const int s0 = min(tid * per_thread, p.batch), s1 = min(s0 + per_thread, p.batch);
  int64_t mine = 0;
  for (int b = s0; b < s1; ++b) mine += aq_places(aq_length(p, b)) + 1;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh->scan[warp] = incl;
  if (lane == 0) {
    for (int s = 0; s < NS; ++s) mbar_init(&sh->full[warp][s], 1);
    if (warp == 0) sh->abort = 0;
    fence_barrier_init();
  }
  if (tid < SM::kPieces) sh->piece[tid] = make_int4(-1, 0, 0, 0);
  __syncthreads();
  int64_t total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < kAqWarps; ++w) {
    if (w < warp) before += sh->scan[w];
    total += sh->scan[w];
  }
  total *= units;
  before *= units;
  int64_t per = (total + gridDim.x - 1) / gridDim.x;
  per = per > kAqMinPlaces ? per : kAqMinPlaces;
  const int64_t c0 = min(static_cast<int64_t>(blockIdx.x) * per, total), c1 = min(c0 + per, total);
  if (c0 >= before && c0 < before + mine * units) {  // one thread, unless the range is empty
    int s = s0;
    for (int64_t next; (next = before + static_cast<int64_t>(aq_places(aq_length(p, s)) + 1) * units) <= c0; ++s)
      before = next;
    sh->first_seq = s;
    sh->first_start = before;
  }
  if (tid == 0) p.desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
  __syncthreads();
  if (c0 >= c1) return;
  const int count = static_cast<int>(c1 - c0);  // below 2^30: checked by the host
  volatile int* abort = &sh->abort;

  auto piece_rows = [&](int k) {  // a warp's last piece lies in its ring, which is free by then
    return k & 1 ? reinterpret_cast<float*>(sh->ring[k >> 1])
                 : p.first + (static_cast<int64_t>(blockIdx.x) * kAqWarps + (k >> 1)) * kAqHeads * SM::kRow;
  };
  // ---- this warp's range [w0, w1) of it ------------------------------------------------
  const int w0 = static_cast<int>(static_cast<int64_t>(count) * warp / kAqWarps);
  const int w1 = static_cast<int>(static_cast<int64_t>(count) * (warp + 1) / kAqWarps);
  if (w0 < w1) {
    AqWalk walk;
    {
      int64_t start = sh->first_start;
      walk.sequence(p, sh->first_seq);
      while (c0 + w0 >= start + static_cast<int64_t>(walk.np + 1) * units) {
        start += static_cast<int64_t>(walk.np + 1) * units;
        walk.sequence(p, walk.seq + 1);
      }
      walk.unit = static_cast<int>((c0 + w0 - start) / (walk.np + 1));
      walk.u0 = static_cast<int>(start + static_cast<int64_t>(walk.unit) * (walk.np + 1) - c0);
    }
    int blk = -1, blk_next = -1;  // cache block (or none) lane % 2 of place lane / 2 of this batch of 16, and of the next
    auto look_up = [&](int batch) {
      const int place = w0 + batch + (lane >> 1);
      blk_next = -1;
      if (place < w1) {
        AqWalk w = walk;
        w.to(p, place, units);
        const int b = 2 * (place - w.u0 - 1) + (lane & 1);  // below 0: the unit's empty place
        if (b >= 0 && b * kQ4Tokens < w.len) {
          const int entry = b / p.blocks_per_page;
          const int page = p.table[w.seq * p.table_stride + entry];
          if (page >= 0 && page < p.pages)
            blk_next = (page * p.nkv + w.unit / p.parts) * p.blocks_per_page + (b - entry * p.blocks_per_page);
        }
      }
    };
    uint32_t seen = 0;  // two bits a stage: its blocks
    int issued = 0;
    auto issue = [&](int s) {  // copies the next place's blocks, if there is one, into the stage that is free
      if (w0 + issued >= w1) return;
      const int at = issued & 15;
      if (at == 0) {
        blk = blk_next;
      } else if (at == 8) {
        look_up(issued + 8);
      }
      const uint32_t bits = __ballot_sync(0xffffffffu, blk >= 0) >> (2 * at) & 3u;
      seen = (seen & ~(3u << (2 * s))) | bits << (2 * s);
      uint64_t* bar = &sh->full[warp][s];
      if (lane == 2 * at) {
        if (bits) mbar_arrive_expect_tx(bar, bits == 3u ? 2 * SM::kBlock : SM::kBlock);
        else mbar_arrive(bar);
      }
      __syncwarp();
      if ((lane >> 1) == at && blk >= 0)
        bulk_g2s(sh->ring[warp][s][lane & 1], p.cache + static_cast<int64_t>(blk) * SM::kBlock, SM::kBlock, bar);
      ++issued;
    };
    look_up(0);
    for (int s = 0; s < NS; ++s) issue(s);
    int s = 0;  // the stage of `place`, and the parity of its use
    uint32_t parity = 0;

    AqWarp<HD, T> st;
    st.win = &sh->window[warp];
    for (int place = w0; place < w1;) {
      walk.to(p, place, units);
      const AqHeads heads(p, walk.unit);
      const int end = min(walk.end(), w1);
      {
        float x[NG][8];
        const T* qp = static_cast<const T*>(p.q) + walk.seq * p.q_seq + (heads.first + (lane >> 2)) * p.q_head +
                      8 * (lane & 3);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[j][e] = 0.f;
          if ((lane >> 2) < heads.count) {
            if (p.q_vec) load_run<8, true>(qp + kQ4Group * j, x[j]);
            else load_run<8, false>(qp + kQ4Group * j, x[j]);
          }
        }
        st.load_q(x, p.scale, lane);
      }
      st.reset(lane);
      for (; place < end; ++place) {
        bool there = __all_sync(0xffffffffu, mbar_try_wait(&sh->full[warp][s], parity));
        if (!there) there = __all_sync(0xffffffffu, wait_phase(&sh->full[warp][s], parity, abort));
        if (!there && lane == 0) atomicOr(p.status, kStatusFullWaitTimeout);
        if (there && (seen >> (2 * s) & 3u))
          st.place(sh->ring[warp][s], seen >> (2 * s) & 3u, walk.len - (place - walk.u0 - 1) * 2 * kQ4Tokens, lane,
                   p.bias);
        __syncwarp();
        if (there) issue(s);
        if (++s == NS) {
          s = 0;
          parity ^= 1u;
        }
      }
      if (walk.u0 >= w0 && walk.end() <= w1) {
        st.sums(lane, [&](int h, int c, const float (&v)[4], float l) {
          float o[4] = {v[0], v[1], v[2], v[3]};
          if (h < heads.count) aq_store<4, T>(p, walk.seq, heads.first + h, c, o, l);
        });
      } else {
        const int k = 2 * warp + (end == w1 ? 1 : 0);
        if (end == w1 && *abort)  // after a wait that ran out: no copy may still be landing in the ring
          for (int j = issued > NS ? issued - NS : 0; j < issued; ++j) {
            int zero = 0;
            if (!wait_phase(&sh->full[warp][j % NS], (j / NS) & 1, &zero)) atomicOr(p.status, kStatusDrainTimeout);
          }
        float* rows = piece_rows(k);
        st.sums(lane, [&](int h, int c, const float (&v)[4], float) {
          *reinterpret_cast<float4*>(rows + h * SM::kRow + c) = make_float4(v[0], v[1], v[2], v[3]);
        });
        if ((lane & 3) == 0) {
          sh->m[lane >> 2][k] = st.m_run;
          sh->l[lane >> 2][k] = st.l_run;
        }
        if (lane == 0) sh->piece[k] = make_int4(walk.seq, walk.unit, walk.u0, walk.end());
      }
    }
    if (*abort)
      for (int j = issued > NS ? issued - NS : 0; j < issued; ++j) {
        int zero = 0;
        if (!wait_phase(&sh->full[warp][j % NS], (j / NS) & 1, &zero)) atomicOr(p.status, kStatusDrainTimeout);
      }
  }
  __syncthreads();
  // ---- the pieces, in order: warp h joins head h of each cut unit; lane k has piece k ----
  static_assert(SM::kPieces <= 32, "a piece a lane");
  const int4 pc = sh->piece[lane & (SM::kPieces - 1)];
  const bool own = lane < SM::kPieces && pc.x >= 0;
  const uint32_t present = __ballot_sync(0xffffffffu, own);
  constexpr int C = HD / 32, N = SM::kPieces;
  float v[N][C];  // the head's part of all pieces, loaded together
#pragma unroll
  for (int j = 0; j < N; ++j) {
#pragma unroll
    for (int e = 0; e < C; ++e) v[j][e] = 0.f;
    if (present >> j & 1u) load_run<C, true>(piece_rows(j) + warp * SM::kRow + C * lane, v[j]);
  }
  for (uint32_t left = present; left;) {
    const int k = __ffs(left) - 1;
    const int seq = __shfl_sync(0xffffffffu, pc.x, k), unit = __shfl_sync(0xffffffffu, pc.y, k);
    const int u0 = __shfl_sync(0xffffffffu, pc.z, k), u1 = __shfl_sync(0xffffffffu, pc.w, k);
    const uint32_t same = __ballot_sync(0xffffffffu, own && pc.z == u0);
    left &= ~same;
    const AqHeads heads(p, unit);
    if (warp < heads.count) {
      float m[N], l[N];
      load_run<N, true>(sh->m[warp], m);
      load_run<N, true>(sh->l[warp], l);
      float M = -INFINITY, L = kNoTokens, acc[C];
#pragma unroll
      for (int j = 0; j < N; ++j) M = fmaxf(M, same >> j & 1u ? m[j] : -INFINITY);
      const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int e = 0; e < C; ++e) acc[e] = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (!(same >> j & 1u)) continue;
        const float f = ex2(m[j] - base);
        L = fmaf(l[j], f, L);
#pragma unroll
        for (int e = 0; e < C; ++e) acc[e] = fmaf(v[j][e], f, acc[e]);
      }
      if (u0 >= 0 && u1 <= count) {
        aq_store<C, T>(p, seq, heads.first + warp, C * lane, acc, L);
      } else {
        float* row = p.part + ((2 * static_cast<int64_t>(blockIdx.x) + (u0 >= 0 ? 1 : 0)) * kAqHeads + warp) * SM::kRow;
        if (lane == 0) {
          row[0] = M;
          row[1] = L;
        }
        store_run<C, true>(row + 4 + C * lane, acc);
      }
    }
    if (u0 >= 0 && u1 > count && tid == 0)  // goes on in the next CTAs
      p.desc[blockIdx.x] = make_int4(seq, unit, static_cast<int>((c0 + u1 - 1) / per - blockIdx.x), 0);
  }
}

// Joins the pieces of a unit that the CTAs' ranges cut: block (i, h) head h of the
// unit that is cut at the end of CTA i's range, each warp every fourth piece.
constexpr int kAqJoinWarps = 4;

template <typename T, int HD>
__global__ void __launch_bounds__(kAqJoinWarps * 32) attn_q4_join_kernel(const AttnQ4Params p) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int ROW = AqSmem<HD>::kRow, C = HD / 32;
  const int4 d = p.desc[blockIdx.x];
  if (d.x < 0) return;
  const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AqHeads heads(p, d.y);
  if (h >= heads.count) return;
  const int np = d.z + 1;
  auto row = [&](int k) {  // the cut unit starts in CTA i (its second piece) and goes on as the others' first
    return p.part + (static_cast<int64_t>(k == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + k)) * kAqHeads + h) * ROW;
  };
  float M = -INFINITY, L = kNoTokens, acc[C];  // of the warp's pieces
#pragma unroll
  for (int e = 0; e < C; ++e) acc[e] = 0.f;
  for (int k = warp; k < np; k += 8 * kAqJoinWarps) {  // eight pieces' loads at a time
    float v[8][C], m[8], l[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int kj = k + j * kAqJoinWarps;
      m[j] = -INFINITY;
      l[j] = kNoTokens;
#pragma unroll
      for (int e = 0; e < C; ++e) v[j][e] = 0.f;
      if (kj < np) {
        const float* r = row(kj);
        m[j] = r[0];
        l[j] = r[1];
        load_run<C, true>(r + 4 + C * lane, v[j]);
      }
    }
    float top = M;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, m[j]);
    const float base = top == -INFINITY ? 0.f : top, keep = ex2(M - base);
    M = top;
    L *= keep;
#pragma unroll
    for (int e = 0; e < C; ++e) acc[e] *= keep;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = ex2(m[j] - base);
      L = fmaf(l[j], f, L);
#pragma unroll
      for (int e = 0; e < C; ++e) acc[e] = fmaf(v[j][e], f, acc[e]);
    }
  }
  __shared__ __align__(16) float sums[kAqJoinWarps][HD];
  __shared__ float ms[kAqJoinWarps], ls[kAqJoinWarps];
  store_run<C, true>(&sums[warp][C * lane], acc);
  if (lane == 0) {
    ms[warp] = M;
    ls[warp] = L;
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int w = 1; w < kAqJoinWarps; ++w) M = fmaxf(M, ms[w]);
    const float base = M == -INFINITY ? 0.f : M;
    L = kNoTokens;
#pragma unroll
    for (int e = 0; e < C; ++e) acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kAqJoinWarps; ++w) {
      float v[C];
      load_run<C, true>(&sums[w][C * lane], v);
      const float f = ex2(ms[w] - base);
      L = fmaf(ls[w], f, L);
#pragma unroll
      for (int e = 0; e < C; ++e) acc[e] = fmaf(v[e], f, acc[e]);
    }
    aq_store<C, T>(p, d.x, heads.first + h, C * lane, acc, L);
  }
}

static __device__ uint32_t g_serving_status;

cudaError_t serving_status(uint32_t** word) {
  static std::atomic<uint32_t*> known[64];  // by device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  *word = dev < 64 ? known[dev].load() : nullptr;
  if (*word) return cudaSuccess;
  e = cudaGetSymbolAddress(reinterpret_cast<void**>(word), g_serving_status);
  if (e == cudaSuccess && dev < 64) known[dev].store(*word);
  return e;
}

template <typename T, int HD>
cudaError_t launch_attn_q4(AttnQ4Params p, int grid, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may use its shared memory
  cudaError_t e = allow_smem(attn_q4_kernel<T, HD>, sizeof(AqSmem<HD>), ready);
  if (e != cudaSuccess) return e;
  e = launch_pdl(attn_q4_kernel<T, HD>, dim3(grid), dim3(kAqThreads), sizeof(AqSmem<HD>), st, p);
  if (e != cudaSuccess || grid == 1) return e;
  return launch_pdl(attn_q4_join_kernel<T, HD>, dim3(grid, min(kAqHeads, p.nh / p.nkv)), dim3(kAqJoinWarps * 32), 0,
                    st, p);
}

}  // namespace frc

extern "C" {

int frc_attention_decode_q4_workspace(int batch, int nh, int nkv, int hd, size_t* bytes) {
  FRC_REQUIRE(bytes && batch >= 0 && nh > 0 && nkv > 0 && nh % nkv == 0 && (hd == 64 || hd == 128),
              "frc_attention_decode_q4_workspace: bad arguments");
  // pieces of units, two a CTA and one a warp; and a descriptor a CTA
  *bytes = static_cast<size_t>(frc::kAqGrid) *
           ((2 + frc::kAqWarps) * frc::kAqHeads * (hd + 4) * sizeof(float) + sizeof(int4));
  return FRC_OK;
}

int frc_attention_decode_q4(int type, const void* q, int64_t q_seq_stride, int64_t q_head_stride, const void* cache,
                            int64_t pages, int page_size, const int* block_table, int64_t table_stride, int max_pages,
                            const int* lengths, int batch, int nh, int nkv, int hd, float scale, void* workspace,
                            size_t workspace_bytes, void* out, int64_t out_seq_stride, int64_t out_head_stride,
                            void* stream) {
  FRC_REQUIRE(frc_is_float_type(type), "frc_attention_decode_q4: type must be FRC_F32, FRC_F16 or FRC_BF16");
  FRC_REQUIRE(hd == 64 || hd == 128, "frc_attention_decode_q4: head_dim must be 64 or 128");
  FRC_REQUIRE(nh > 0 && nkv > 0 && nh <= 65535 && nh % nkv == 0,
              "frc_attention_decode_q4: needs nh a multiple of nkv");
  FRC_REQUIRE(page_size > 0 && page_size % frc::kQ4Tokens == 0,
              "frc_attention_decode_q4: page_size must be a multiple of 16");
  FRC_REQUIRE(pages > 0 && pages <= 0x7fffffff / (page_size / frc::kQ4Tokens) / nkv,
              "frc_attention_decode_q4: bad number of pages");
  FRC_REQUIRE(batch >= 0 && batch <= 65535 && max_pages >= 0 && table_stride >= 0,
              "frc_attention_decode_q4: bad batch or block table");
  FRC_REQUIRE(q_seq_stride >= 0 && q_head_stride >= 0 && out_seq_stride >= 0 && out_head_stride >= 0,
              "frc_attention_decode_q4: negative stride");
  FRC_REQUIRE(scale - scale == 0.f, "frc_attention_decode_q4: scale must be finite");
  if (batch == 0) return FRC_OK;
  FRC_REQUIRE(q && cache && (block_table || max_pages == 0) && lengths && out && workspace,
              "frc_attention_decode_q4: null pointer");
  FRC_REQUIRE(frc::aligned_to(cache, 16) && frc::aligned_to(workspace, 16),
              "frc_attention_decode_q4: cache and workspace must be 16-byte aligned");
  size_t need = 0;
  const int rc = frc_attention_decode_q4_workspace(batch, nh, nkv, hd, &need);
  if (rc) return rc;
  FRC_REQUIRE(workspace_bytes >= need, "frc_attention_decode_q4: workspace is too small");
  const int parts = (nh / nkv + frc::kAqHeads - 1) / frc::kAqHeads;
  // no more CTAs than the tables could give places for
  const int64_t blocks = static_cast<int64_t>(max_pages) * (page_size / frc::kQ4Tokens);
  FRC_REQUIRE(blocks < (int64_t(1) << 48) && static_cast<int64_t>(nkv) * parts <= 65535,
              "frc_attention_decode_q4: block table or heads too large");
  const int64_t most = static_cast<int64_t>(batch) * nkv * parts * ((blocks < (1 << 27) ? (blocks + 1) / 2 : (1 << 26)) + 1);
  const int64_t want = (most + frc::kAqMinPlaces - 1) / frc::kAqMinPlaces;
  const int grid = static_cast<int>(want < frc::kAqGrid ? want : frc::kAqGrid);
  FRC_REQUIRE(most / grid < (int64_t(1) << 30), "frc_attention_decode_q4: block table too large");
  const size_t es = type == FRC_F32 ? 4 : 2;
  const frc::View results(out, es, batch, out_seq_stride, nh, out_head_stride, hd), from(q, es, batch, q_seq_stride, nh, q_head_stride, hd);
  const frc::View blocks_of(cache, 1, 1, 0, 1, 0, pages * (page_size / frc::kQ4Tokens) * nkv * frc::Q4Layout(hd).block_bytes());
  FRC_REQUIRE(results.distinct(), "frc_attention_decode_q4: the rows or heads of out overlap");
  // (a row is written after all that read it have)
  const bool in_place = out == q && (batch == 1 || out_seq_stride == q_seq_stride) && (nh == 1 || out_head_stride == q_head_stride);
  FRC_REQUIRE((in_place || !frc::views_share(results, from)) && !frc::views_share(results, blocks_of),
              "frc_attention_decode_q4: out shares memory with the cache, or with q without being q");
  const int run = type == FRC_F32 ? 4 : 8;  // elements of a 16-byte load
  frc::AttnQ4Params p{};
  FRC_LAUNCHED(frc::serving_status(&p.status), "status word");
  p.q = q;
  p.q_seq = q_seq_stride;
  p.q_head = q_head_stride;
  p.cache = static_cast<const uint8_t*>(cache);
  p.pages = pages;
  p.blocks_per_page = page_size / frc::kQ4Tokens;
  p.table = block_table;
  p.table_stride = table_stride;
  p.max_pages = max_pages;
  p.lengths = lengths;
  p.batch = batch;
  p.nh = nh;
  p.nkv = nkv;
  p.parts = parts;
  p.scale = scale;
  p.out = out;
  p.o_seq = out_seq_stride;
  p.o_head = out_head_stride;
  p.q_vec = frc::aligned_to(q, 16) && q_seq_stride % run == 0 && q_head_stride % run == 0;
  p.o_vec = frc::aligned_to(out, 4 * es) && out_seq_stride % 4 == 0 && out_head_stride % 4 == 0;
  p.part = static_cast<float*>(workspace);
  p.first = p.part + static_cast<size_t>(frc::kAqGrid) * 2 * frc::kAqHeads * (hd + 4);
  p.desc = reinterpret_cast<int4*>(p.first + static_cast<size_t>(frc::kAqGrid) * frc::kAqWarps * frc::kAqHeads * (hd + 4));
  p.bias = 0x64006400u;
  return frc_with_type(type, [&](auto* z) -> int {
    using T = std::remove_pointer_t<decltype(z)>;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    FRC_LAUNCHED((hd == 128 ? frc::launch_attn_q4<T, 128>(p, grid, st) : frc::launch_attn_q4<T, 64>(p, grid, st)),
                 "attention_decode_q4 launch");
    return FRC_OK;
  });
}

}  // extern "C"
