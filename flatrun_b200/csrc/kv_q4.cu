// Writing keys and values into the 4-bit paged cache, and reading them back.
//
// Of the 32 values x of a group, in exact arithmetic:
//   m = fp16(min x), held within +-65504
//   d = fp16((max x - m) / 15), held within 0 .. 65504
//   n = round((x - m) / d) to the nearest integer, ties to even, held within
//       0 .. 15 (0 where d = 0)
// and a group with a value that is not finite gets m = NaN, so that it reads
// back as NaN.  The quotients are formed in fp32; where one lies so near a
// border between two results that fp32 could fall on the wrong side, the side is
// found exactly, so the cache's bits follow from the definition alone.
//
// Bound by HBM: 2 or 4 bytes a value in, 5/8 of a byte out (append), and the
// reverse (read), if a value takes few instructions.  A warp takes
// eight tokens of one head, four lanes a token and eight channels a lane, one
// group at a time: a group's minimum and maximum are two shuffles, a lane's eight
// nibbles are one word, a token's K words one 4 NG byte store, and the V words of
// eight consecutive tokens a full 32-byte sector.  65536 tokens of 8 heads of 128 in
// bf16: 117 us appended (750 warp instructions for eight tokens of a head, 23 a
// value and lane: the issue slots bind at 3.0 TB/s), 64 us read (5.5 TB/s).  Two lanes a token
// with twice the channels took 163 us where this took 121: fewer instructions, but
// more code than the instruction cache holds.
#include <cuda_runtime.h>

#include <cstdio>

#include "../../include/frcuda.h"
#include "kv_q4.cuh"

namespace frc {

struct KvQ4Params {
  uint8_t* cache;
  int64_t pages;
  int nkv, blocks_per_page;
  const int64_t* slots;
  int64_t tokens;
  const void *k, *v;     // append: inputs; read: outputs
  int64_t k_tok, k_head, v_tok, v_head;  // strides in elements
};

constexpr int kQ4Threads = 128;

// The least and the largest of three, NaN if one is.
FRC_DEVICE_INLINE float min_nan(float a, float b, float c) {
  float y;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
FRC_DEVICE_INLINE float max_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// fp16 of (hi - m) / 15, held within 0 .. 65504, rounded once.  The fp32 quotient
// is within 3 ulp (three roundings); 13 of its bits are dropped, so only within
// 4 ulp of their middle can the rounding fall on the wrong side (below fp16's
// normal range more bits are dropped: there, and there alone, the quotient is
// formed in fp64 too).
FRC_DEVICE_INLINE __half step_of(float hi, float m) {
  const float f = fminf(fmaxf((hi - m) * (1.0f / 15.0f), 0.f), 65504.f);
  const uint32_t low = __float_as_uint(f) & 0x1fffu;
  if (f > 6.2e-5f && (low < 0x1000u - 4u || low > 0x1000u + 4u)) return __float2half_rn(f);
  return __double2half(fmin(fmax((static_cast<double>(hi) - static_cast<double>(m)) / 15.0, 0.0), 65504.0));
}

// The nibbles of eight values by the side of the border that each lies on: where
// a lane has one that is too near for fp32's quotient, as 16-bit values often
// are (they meet borders exactly).  Out of line, so that the callers' code stays
// in the instruction cache.
__device__ __noinline__ uint32_t border8(float x0, float x1, float x2, float x3, float x4, float x5, float x6, float x7,
                                         float m, float d, float inv) {
  const float x[8] = {x0, x1, x2, x3, x4, x5, x6, x7};
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // h: the border nearest to t; e: on which side of it x - m lies.  s + err is
    // x - m exactly (two-sum), and s - h d is exact near the border
    const float t = fminf(fmaxf((x[i] - m) * inv, 0.f), 15.f);
    const float h = fminf(fmaxf(rintf(t - 0.5f), 0.f), 14.f) + 0.5f;
    const float s = __fsub_rn(x[i], m), v = __fsub_rn(s, x[i]);
    const float err = __fsub_rn(__fsub_rn(x[i], __fsub_rn(s, v)), __fadd_rn(m, v));
    const float e = __fadd_rn(__fmaf_rn(-h, d, s), err);
    const float n = e > 0.f ? h + 0.5f : (e < 0.f ? h - 0.5f : 2.f * rintf(0.5f * h));  // on it: the even one
    w |= static_cast<uint32_t>(n) << (4 * i);
  }
  return w;
}

// The lane's eight values of a group shared by the four lanes of its quad:
// its nibbles as one word, and the group's step and offset.
FRC_DEVICE_INLINE uint32_t quantise8(const float (&x)[8], __half& step, __half& offset) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    lo = min_nan(lo, x[i], x[i + 1]);
    hi = max_nan(hi, x[i], x[i + 1]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const float l = __shfl_xor_sync(0xffffffffu, lo, o), h = __shfl_xor_sync(0xffffffffu, hi, o);
    lo = min_nan(lo, l, l);
    hi = max_nan(hi, h, h);
  }
  if (!(lo >= -3.402823466e38f && hi <= 3.402823466e38f)) {  // a NaN or an infinity
    offset = __ushort_as_half(0x7fff);
    step = __ushort_as_half(0);
    return 0u;
  }
  offset = __float2half_rn(fminf(fmaxf(lo, -65504.f), 65504.f));
  const float m = __half2float(offset);
  step = step_of(hi, m);
  const float d = __half2float(step);
  float inv;  // of d, within an ulp
  asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(d));
  if (d == 0.f) inv = 0.f;
  // n = round((x - m) / d) in the low bits of the sum with 1.5 * 2^23.  The quotient is
  // off by 2^-24 (difference) and 2^-23 (reciprocal) of itself, less than 4e-6.
  constexpr float kMagic = 12582912.f;
  const uint64_t inv2 = f32x2_two(inv, inv), m2 = f32x2_two(-m, -m), magic2 = f32x2_two(kMagic, kMagic);
  uint32_t w = 0;
  // the largest distance from a whole number, or (where m or d was rounded by as much) of
  // the quotients beyond 0 and 15
  float far = max_nan((m - lo) * inv, fmaf(hi - m, inv, -15.f), 0.f);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t t = f32x2_add(f32x2_two(x[i], x[i + 1]), m2), u = f32x2_fma(t, inv2, magic2);
    float u0, u1, off0, off1;
    f32x2_split(u, u0, u1);
    // t inv - (u - magic)
    f32x2_split(f32x2_fma(t, inv2, f32x2_fma(u, f32x2_two(-1.f, -1.f), magic2)), off0, off1);
    far = max_nan(far, fabsf(off0), fabsf(off1));
    w += __float_as_uint(u0) << (4 * i);
    w += __float_as_uint(u1) << (4 * i + 4);
  }
  // the sums' other bits, 0x4B400000 each, add up to this
  constexpr uint32_t kSum = 0x4B400000u * 0x11111111u;
  w -= kSum;
  if (far > 0.5f - 6e-6f) w = border8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], m, d, inv);
  return w;
}

template <int NG>
FRC_DEVICE_INLINE void store_words(uint8_t* p, const uint32_t (&w)[NG]) {
  if constexpr (NG == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (NG == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else
#pragma unroll
    for (int j = 0; j < NG; ++j) reinterpret_cast<uint32_t*>(p)[j] = w[j];
}

// warp -> (eight tokens, K or V, head); lane -> (token, q)
FRC_DEVICE_INLINE bool q4_warp_item(const KvQ4Params& p, int64_t& tok, int& is_v, int& h, int& q, int64_t& block,
                                    int& t) {
  const uint32_t warp = blockIdx.x * (kQ4Threads / 32) + (threadIdx.x >> 5);  // below 2^31: checked by the host
  const int lane = threadIdx.x & 31;
  const uint32_t tg = warp / static_cast<uint32_t>(2 * p.nkv);
  const int rest = static_cast<int>(warp - tg * static_cast<uint32_t>(2 * p.nkv));
  is_v = rest >= p.nkv;
  h = is_v ? rest - p.nkv : rest;
  tok = static_cast<int64_t>(tg) * 8 + (lane >> 2);
  q = lane & 3;
  block = -1;
  t = 0;
  if (tok < p.tokens) {
    const int64_t slot = p.slots[tok];
    block = q4_block_of_slot(slot, h, p.pages, p.nkv, p.blocks_per_page);
    t = static_cast<int>(slot) & (kQ4Tokens - 1);
  }
  return static_cast<int64_t>(tg) * 8 < p.tokens;  // the same in all lanes
}

template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(kQ4Threads, 8) kv_append_q4_kernel(KvQ4Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" :::);
  constexpr Q4Layout lay(HD);
  constexpr int NG = HD / kQ4Group;
  int64_t tok, block;
  int is_v, h, q, t;
  if (!q4_warp_item(p, tok, is_v, h, q, block, t)) return;
  const bool live = block >= 0;
  const T* src = static_cast<const T*>(is_v ? p.v : p.k) + (live ? tok : 0) * (is_v ? p.v_tok : p.k_tok) +
                 h * (is_v ? p.v_head : p.k_head);
  uint8_t* blk = p.cache + (live ? block : 0) * lay.block_bytes();
  float x[NG][8];
#pragma unroll
  for (int j = 0; j < NG; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
    if (live) load_run<8, VEC>(src + kQ4Group * j + 8 * q, x[j]);
  }
  uint32_t w[NG];
  __half step = __ushort_as_half(0), offset = step;  // of group q: the lanes of a quad share them
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    __half d, m;
    w[j] = quantise8(x[j], d, m);
    if (q == j) {
      step = d;
      offset = m;
    }
    if (live && is_v) *reinterpret_cast<uint32_t*>(blk + lay.v_word(4 * j + q, t)) = w[j];
  }
  if (!live) return;
  if (!is_v) store_words(blk + lay.k_word(t, q, 0), w);
  if (q < NG) {
    *reinterpret_cast<__half*>(blk + (is_v ? lay.v_step(q, t) : lay.k_step(q, t))) = step;
    *reinterpret_cast<__half*>(blk + (is_v ? lay.v_offset(q, t) : lay.k_offset(t, q))) = offset;
  }
}

template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(kQ4Threads) kv_read_q4_kernel(KvQ4Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" :::);
  constexpr Q4Layout lay(HD);
  constexpr int NG = HD / kQ4Group;
  int64_t tok, block;
  int is_v, h, q, t;
  if (!q4_warp_item(p, tok, is_v, h, q, block, t) || block < 0) return;  // a row outside the cache stays as it is
  const uint8_t* blk = p.cache + block * lay.block_bytes();
  T* dst = static_cast<T*>(const_cast<void*>(is_v ? p.v : p.k)) + tok * (is_v ? p.v_tok : p.k_tok) +
           h * (is_v ? p.v_head : p.k_head);
  uint32_t w[NG];
  float d[NG], m[NG];
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    w[j] = *reinterpret_cast<const uint32_t*>(blk + (is_v ? lay.v_word(4 * j + q, t) : lay.k_word(t, q, j)));
    d[j] = __half2float(*reinterpret_cast<const __half*>(blk + (is_v ? lay.v_step(j, t) : lay.k_step(j, t))));
    m[j] = __half2float(*reinterpret_cast<const __half*>(blk + (is_v ? lay.v_offset(j, t) : lay.k_offset(t, j))));
  }
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // nibbles i and i + 4 as halves: 1024 + n, less 1024
      const uint32_t b = ((w[j] >> (4 * i)) & 0x000f000fu) | 0x64006400u;
      const float2 n = __half22float2(__hadd2(*reinterpret_cast<const __half2*>(&b), __float2half2_rn(-1024.f)));
      x[i] = fmaf(n.x, d[j], m[j]);
      x[i + 4] = fmaf(n.y, d[j], m[j]);
    }
    store_run<8, VEC>(dst + kQ4Group * j + 8 * q, x);
  }
}

template <bool READ>
int kv_q4_call(const char* what, int type, KvQ4Params p, int hd, int page_size, void* stream) {
  if (!frc_is_float_type(type)) return frc__fail(FRC_ERR_INVALID, "kv_q4: type must be FRC_F32, FRC_F16 or FRC_BF16");
  FRC_REQUIRE(hd == 64 || hd == 128, "kv_q4: head_dim must be 64 or 128");
  FRC_REQUIRE(p.nkv > 0 && p.nkv <= 65535 && p.pages > 0, "kv_q4: bad pages or heads");
  FRC_REQUIRE(page_size > 0 && page_size % kQ4Tokens == 0, "kv_q4: page_size must be a multiple of 16");
  p.blocks_per_page = page_size / kQ4Tokens;
  FRC_REQUIRE(p.pages <= 0x7fffffff / p.blocks_per_page, "kv_q4: too many blocks in the cache");
  FRC_REQUIRE(p.tokens >= 0 && p.tokens <= 0x7fffffff / (2 * p.nkv), "kv_q4: bad number of tokens");
  FRC_REQUIRE(p.k_tok >= 0 && p.k_head >= 0 && p.v_tok >= 0 && p.v_head >= 0, "kv_q4: negative stride");
  if (p.tokens == 0) return FRC_OK;
  FRC_REQUIRE(p.cache && p.slots && p.k && p.v, "kv_q4: null pointer");
  FRC_REQUIRE(aligned_to(p.cache, 16), "kv_q4: the cache must be 16-byte aligned");
  const size_t es = type == FRC_F32 ? 4 : 2;
  if (READ) {
    const View k(p.k, es, p.tokens, p.k_tok, p.nkv, p.k_head, hd), v(p.v, es, p.tokens, p.v_tok, p.nkv, p.v_head, hd);
    const View cache(p.cache, 1, 1, 0, 1, 0, p.pages * p.blocks_per_page * p.nkv * Q4Layout(hd).block_bytes());
    FRC_REQUIRE(k.distinct() && v.distinct(), "kv_q4: the rows or heads of an output overlap");
    FRC_REQUIRE(!views_share(k, v) && !views_share(k, cache) && !views_share(v, cache),
                "kv_q4: the outputs share memory with each other or with the cache");
  }
  const int run = type == FRC_F32 ? 4 : 8;  // elements of a 16-byte load
  const bool vec = aligned_to(p.k, 16) && aligned_to(p.v, 16) && p.k_tok % run == 0 && p.k_head % run == 0 &&
                   p.v_tok % run == 0 && p.v_head % run == 0;
  const int64_t warps = (p.tokens + 7) / 8 * 2 * p.nkv;
  const dim3 grid(static_cast<unsigned>((warps * 32 + kQ4Threads - 1) / kQ4Threads));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return frc_with_type(type, [&](auto* z) -> int {
    using T = std::remove_pointer_t<decltype(z)>;
    void (*fn)(KvQ4Params);
    if constexpr (READ)
      fn = hd == 128 ? (vec ? kv_read_q4_kernel<T, 128, true> : kv_read_q4_kernel<T, 128, false>)
                     : (vec ? kv_read_q4_kernel<T, 64, true> : kv_read_q4_kernel<T, 64, false>);
    else
      fn = hd == 128 ? (vec ? kv_append_q4_kernel<T, 128, true> : kv_append_q4_kernel<T, 128, false>)
                     : (vec ? kv_append_q4_kernel<T, 64, true> : kv_append_q4_kernel<T, 64, false>);
    FRC_LAUNCHED(launch_pdl(fn, grid, dim3(kQ4Threads), 0, st, p), what);
    return FRC_OK;
  });
}

}  // namespace frc

extern "C" {

int frc_kv_q4_bytes(int64_t pages, int page_size, int nkv, int hd, size_t* bytes) {
  FRC_REQUIRE(bytes && pages > 0 && nkv > 0 && page_size > 0 && page_size % frc::kQ4Tokens == 0 &&
                  (hd == 64 || hd == 128) && pages <= 0x7fffffff / (page_size / frc::kQ4Tokens),
              "frc_kv_q4_bytes: needs pages, heads, a page_size that is a multiple of 16 and head_dim 64 or 128");
  *bytes = static_cast<size_t>(pages) * nkv * (page_size / frc::kQ4Tokens) * frc::Q4Layout(hd).block_bytes();
  return FRC_OK;
}

int frc_kv_append_q4(int type, const void* k, int64_t k_tok_stride, int64_t k_head_stride, const void* v,
                     int64_t v_tok_stride, int64_t v_head_stride, int64_t tokens, const int64_t* slots_dev, int nkv,
                     int hd, int64_t pages, int page_size, void* cache, void* stream) {
  const frc::KvQ4Params p{static_cast<uint8_t*>(cache), pages, nkv, 0, slots_dev, tokens, k, v,
                          k_tok_stride, k_head_stride, v_tok_stride, v_head_stride};
  return frc::kv_q4_call<false>("kv_append_q4 launch", type, p, hd, page_size, stream);
}

int frc_kv_read_q4(int type, const void* cache, const int64_t* slots_dev, int64_t tokens, int nkv, int hd,
                   int64_t pages, int page_size, void* k, int64_t k_tok_stride, int64_t k_head_stride, void* v,
                   int64_t v_tok_stride, int64_t v_head_stride, void* stream) {
  const frc::KvQ4Params p{static_cast<uint8_t*>(const_cast<void*>(cache)), pages, nkv, 0, slots_dev, tokens, k, v,
                          k_tok_stride, k_head_stride, v_tok_stride, v_head_stride};
  return frc::kv_q4_call<true>("kv_read_q4 launch", type, p, hd, page_size, stream);
}

}  // extern "C"
