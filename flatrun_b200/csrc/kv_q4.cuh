// The 4-bit paged key/value cache: its layout, and the element types of the
// serving operators that surround it.
//
// A cache is (pages, kv_heads, page_size / 16) blocks.  A block holds 16
// tokens of one KV head; a token's D channels are quantised in groups of 32,
// value = d * n + m with an fp16 step d, an fp16 offset m and n in 0..15: 5
// bits a value with its share of the scales.  Inside a block (NG = D / 32
// groups; nibble i of a 32-bit word is bits 4i..4i+3, words little-endian):
//
//   bytes          what                              read by attention as
//   [0, 8D)        K nibbles: words (16 tokens, 4, NG); word (q, j) of a
//                  token has channels 32 j + 8 q .. + 7
//                                     one 4 NG byte load a lane: the lanes of
//                                     a quad hold the 32 channels of each group
//   [8D, 16D)      V nibbles: words (D / 8, 16 tokens); word w has channels
//                  8 w .. 8 w + 7     one 16-byte load a lane: four tokens
//   then halves    K steps (NG, 16 tokens), K offsets (16 tokens, NG),
//                  V steps (NG, 16), V offsets (NG, 16)
//
// The order makes every operand of the tensor-core products one aligned
// vector load away from its fragment, and one block one contiguous copy of
// 20 D bytes.  No byte is shared by two tokens, so tokens are written without
// reading the cache.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstdint>

#include "frc_common.cuh"

namespace frc {

constexpr int kQ4Tokens = 16;   // tokens of a block
constexpr int kQ4Group = 32;    // channels of a quantisation group

struct Q4Layout {
  int hd, ng;
  __host__ __device__ constexpr explicit Q4Layout(int hd_) : hd(hd_), ng(hd_ / kQ4Group) {}
  __host__ __device__ constexpr int block_bytes() const { return 20 * hd; }
  // byte offsets inside a block
  __host__ __device__ constexpr int k_word(int t, int q, int j) const { return 4 * ((t * 4 + q) * ng + j); }
  __host__ __device__ constexpr int v_word(int w, int t) const { return 8 * hd + 4 * (w * kQ4Tokens + t); }
  __host__ __device__ constexpr int k_step(int j, int t) const { return 16 * hd + 2 * (j * kQ4Tokens + t); }
  __host__ __device__ constexpr int k_offset(int t, int j) const { return 17 * hd + 2 * (t * ng + j); }
  __host__ __device__ constexpr int v_step(int j, int t) const { return 18 * hd + 2 * (j * kQ4Tokens + t); }
  __host__ __device__ constexpr int v_offset(int j, int t) const { return 19 * hd + 2 * (j * kQ4Tokens + t); }
};

// Index of the block that holds slot `slot` of head `h`, or -1 where the slot
// is outside the cache (a padding row, or a bad index: never touched).
__host__ __device__ inline int64_t q4_block_of_slot(int64_t slot, int h, int64_t pages, int nkv, int blocks_per_page) {
  if (slot < 0 || slot >= pages * blocks_per_page * kQ4Tokens) return -1;
  const uint32_t block = static_cast<uint32_t>(slot >> 4);  // pages * blocks_per_page < 2^31 (checked by the host)
  const uint32_t page = block / static_cast<uint32_t>(blocks_per_page);
  return (static_cast<int64_t>(page) * nkv + h) * blocks_per_page + (block - page * blocks_per_page);
}

// Element types: values are computed in fp32 and rounded once when stored.
FRC_DEVICE_INLINE float to_f32(float v) { return v; }
FRC_DEVICE_INLINE float to_f32(__half v) { return __half2float(v); }
FRC_DEVICE_INLINE float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
FRC_DEVICE_INLINE void from_f32(float v, float& o) { o = v; }
FRC_DEVICE_INLINE void from_f32(float v, __half& o) { o = __float2half_rn(v); }
FRC_DEVICE_INLINE void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

// Pairs of fp32 values: two operations in one instruction.
FRC_DEVICE_INLINE uint64_t f32x2_two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
FRC_DEVICE_INLINE void f32x2_split(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
FRC_DEVICE_INLINE uint64_t f32x2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
FRC_DEVICE_INLINE uint64_t f32x2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

FRC_DEVICE_INLINE uint64_t f32x2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// N consecutive elements at p as fp32, and back.  VEC: p is aligned to the
// run (at most 16 bytes); otherwise one element at a time.
template <int N, bool VEC, typename T>
FRC_DEVICE_INLINE void load_run(const T* p, float (&v)[N]) {
  if constexpr (VEC) {
    constexpr int B = N * sizeof(T) < 16 ? N * sizeof(T) : 16, E = B / sizeof(T);
    struct alignas(B) Run { T e[E]; };
#pragma unroll
    for (int i = 0; i < N / E; ++i) {
      const Run r = reinterpret_cast<const Run*>(p)[i];
#pragma unroll
      for (int j = 0; j < E; ++j) v[i * E + j] = to_f32(r.e[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32(p[i]);
  }
}

template <int N, bool VEC, typename T>
FRC_DEVICE_INLINE void store_run(T* p, const float (&v)[N]) {
  if constexpr (VEC) {
    constexpr int B = N * sizeof(T) < 16 ? N * sizeof(T) : 16, E = B / sizeof(T);
    struct alignas(B) Run { T e[E]; };
#pragma unroll
    for (int i = 0; i < N / E; ++i) {
      Run r;
#pragma unroll
      for (int j = 0; j < E; ++j) from_f32(v[i * E + j], r.e[j]);
      reinterpret_cast<Run*>(p)[i] = r;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) from_f32(v[i], p[i]);
  }
}

}  // namespace frc

// ---- host side: shared by the entry points ---------------------------------------

// Defined in frcuda_api.cu: records a message for frc_last_error.
extern "C" int frc__fail(int code, const char* msg);

namespace frc {

// Launch with the programmatic-stream-serialization attribute: every kernel
// launched so waits for its predecessor (griddepcontrol.wait) before it
// touches memory.
template <typename... P, typename... A>
inline cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Lets `kernel` use `bytes` of dynamic shared memory on the current device,
// once a device.
template <typename K>
inline cudaError_t allow_smem(K kernel, size_t bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (ready.load() >> dev & 1)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess && dev < 64) ready.fetch_or(uint64_t(1) << dev);
  return e;
}

// Address of the serving kernels' status word on the current device
// (attn_q4.cu): bits of bounded waits that ran out, read by frc_device_status.
cudaError_t serving_status(uint32_t** word);

// A (rows, heads, channels) operand as a call gives it, in bytes.
struct View {
  uintptr_t at;
  int64_t rows, row, heads, head, channels;
  View(const void* p, size_t size, int64_t rows_, int64_t row_, int64_t heads_, int64_t head_, int64_t channels_)
      : at(reinterpret_cast<uintptr_t>(p)), rows(rows_), row(row_ * static_cast<int64_t>(size)), heads(heads_),
        head(head_ * static_cast<int64_t>(size)), channels(channels_ * static_cast<int64_t>(size)) {}
  using Wide = __int128;  // strides times counts
  Wide row_span() const { return Wide(rows - 1) * row; }
  Wide head_span() const { return Wide(heads - 1) * head; }
  Wide end() const { return Wide(at) + row_span() + head_span() + channels; }
  bool empty() const { return rows < 1 || heads < 1 || channels < 1; }
  // No two rows or heads lie over each other.
  bool distinct() const {
    if (empty()) return true;
    const bool rows_inside = heads < 2 || (rows > 1 && row < head);
    const int64_t inner = rows_inside ? row : head, outer = rows_inside ? head : row;
    const int64_t n = rows_inside ? rows : heads, m = rows_inside ? heads : rows;
    return (n < 2 || inner >= channels) && (m < 2 || outer >= Wide(n - 1) * inner + channels);
  }
};

// Whether two operands share memory, for all that can be told from where they start
// and end, and from what each holds of a period: of rows or of heads that are equally far
// apart in both, or of the largest step that all of them are multiples of.
inline bool views_share(const View& a, const View& b) {
  if (a.empty() || b.empty() || a.end() <= View::Wide(b.at) || b.end() <= View::Wide(a.at)) return false;
  int64_t common = 0;
  auto with = [&](int64_t n, int64_t s) {
    if (n < 2) return;
    while (s) {
      const int64_t r = common % s;
      common = s;
      s = r;
    }
  };
  with(a.rows, a.row);
  with(a.heads, a.head);
  with(b.rows, b.row);
  with(b.heads, b.head);
  auto separate = [&](int64_t step, View::Wide a_holds, View::Wide b_holds) {  // in each period b is `off` behind a
    if (step <= 0) return false;
    const int64_t off = ((static_cast<int64_t>(b.at - a.at) % step) + step) % step;
    return a_holds <= off && off + b_holds <= step;
  };
  return !(a.row == b.row && separate(a.row, a.head_span() + a.channels, b.head_span() + b.channels)) &&
         !(a.head == b.head && separate(a.head, a.row_span() + a.channels, b.row_span() + b.channels)) &&
         !separate(common, a.channels, b.channels);
}

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace frc

#define FRC_REQUIRE(cond, msg)                          \
  do {                                                  \
    if (!(cond)) return frc__fail(FRC_ERR_INVALID, msg); \
  } while (0)

#define FRC_LAUNCHED(expr, what)                                                               \
  do {                                                                                         \
    const cudaError_t _e = (expr);                                                             \
    if (_e != cudaSuccess) {                                                                   \
      char _msg[192];                                                                          \
      snprintf(_msg, sizeof _msg, "%s: %s", what, cudaGetErrorString(_e));                     \
      (void)cudaGetLastError();                                                                \
      return frc__fail(FRC_ERR_CUDA, _msg);                                                    \
    }                                                                                          \
  } while (0)

// Calls f with a null pointer of the element type `type` (FRC_F32, FRC_F16
// or FRC_BF16, checked before).
template <typename F>
inline int frc_with_type(int type, F&& f) {
  if (type == FRC_F32) return f(static_cast<float*>(nullptr));
  if (type == FRC_F16) return f(static_cast<__half*>(nullptr));
  return f(static_cast<__nv_bfloat16*>(nullptr));
}
inline bool frc_is_float_type(int type) { return type == FRC_F32 || type == FRC_F16 || type == FRC_BF16; }
