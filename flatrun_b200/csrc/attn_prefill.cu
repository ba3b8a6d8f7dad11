// Attention of whole prompts: packed sequences of different lengths, grouped
// heads, causal or not,
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j
//
// over the keys j of the sequence of query i; causal: the last query sees
// every key, each earlier one a key less (so a prompt may follow tokens that
// are there already).  A query that sees no key gives zeros, and rows behind
// the last sequence stay as they are.
//
// Bound by the tensor cores and, as much, by the exponentials: a tile of 128
// rows by 128 keys is 2 * 128^3 multiply-adds (1024 cycles at 4096 a cycle) and
// 128^2 exponentials (1024 cycles at 16 a cycle).  Two tiles of rows therefore take
// turns: while one's scores pass through the softmax, the other's products run.
// A tile's rows are queries of all heads that share a KV head (as far as their
// number divides 128 well), so that short prompts fill tiles too; two such
// tiles, one behind the other, are a work item.  A CTA has an SM to itself and
// goes from item to item (it takes over blocks of the grid that have not
// started, clusterlaunchcontrol), so that an item's first loads and products run
// while the last one's results are written:
//
//   warp 9        loads: the two row tiles once an item, then K and V tiles of 128
//                 keys through a ring (TMA, 128-byte swizzle); finds the next item
//   warp 8        issues tcgen05.mma: S = Q K^T (128 x 128 fp32 in tensor
//                 memory), and O += P V with P read from tensor memory, where
//                 it takes the place of S; V is the transposed operand as it lies
//   warp 10       makes V tiles ready: rows behind the last key zeroed, and in tiles
//                 that some row does not see whole all elements that are not finite
//   warps 0-3,    softmax of tile 0 and 1, a row a thread: maximum, exponentials,
//   warps 4-7     P rounded to the type of the inputs, handed over in two parts;
//                 at the end O / sum.  (Two threads a row took 1134 us where one
//                 took 1057, for the measurement below.)
//
// The running maximum is a reference that may stay 2^8 behind: O in tensor
// memory is rescaled only when a row passes that, which few tiles do.  Scores,
// maxima, sums and O are fp32; P is rounded to the inputs' type, as its operand
// must be, and the sum is of the unrounded values.
//
// What is masked has no part in the result whatever it holds: scores are
// replaced, V rows behind the last key are zeroed in shared memory, and so are NaNs
// and infinities of V in tiles that some row does not see whole (0 * NaN would reach
// the rows that do not see them).  Rows that do see one get it added at the end
// (pf_add_seen), so that an element that is not finite costs the rows beside it
// nothing and no row is computed twice.
//
// Measured: 8192 tokens, causal, 64 / 8 heads of 128, bf16: 0.96 ms, 1145 TFLOP/s (0.69
// of cuBLAS's burst rate, 0.82 of its sustained one; the card is at its power
// limit).  A key tile's chain of scores, softmax and products takes a query tile
// 3000 cycles (1800 in the softmax); the two tiles in turn keep the tensor pipe two
// thirds busy.  Scores of the next 64 keys formed early, in the half of S's columns
// that P leaves free, took 9 % longer (two products of 64 columns in place of one of
// 128).  17 packed prompts of 1 to 1000 queries, 32 / 8 heads of 64, fp16: 48 us.  Code
// size counts: a second copy of the softmax step for tiles with masks took
// 52 us, and skipping hidden quarters' exponentials costs the long prompt 3 %.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdio>
#include <cstring>

#include "../../include/frcuda.h"
#include "gemv.cuh"
#include "kv_q4.cuh"
#include "launch.cuh"

namespace frc {

struct PrefillParams {
  const void *q, *k, *v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  const int *cu_q, *cu_k;
  int batch;
  int tokens_q, tokens_k;
  int nh, nkv;
  int heads, queries;       // query heads of a tile (of one KV head), and queries of each: heads * queries <= 128
  int k_mul, v_mul;         // 0: the heads are one (stride 0), 1: the map's second coordinate is the head
  float scale;              // not negative; times log2 e
  float signed_scale;       // as given
  int negate;               // scale was negative: Q is negated in the product
  int causal;
  int q_blocks;
  void* out;
  int64_t o_tok, o_head;
  uint32_t* status;
};

constexpr int kPfRows = 128;     // rows (queries of some heads) of a tile, keys of a tile
constexpr int kPfTiles = 2;      // row tiles of a work item
constexpr int kPfThreads = 384;
// Registers: the CTA is launched with 168 a thread; the softmax warps, which
// hold a row of scores, take over what the other four warps leave (two of
// them are there for that alone): 2 * 224 + 56 = 3 * 168.
constexpr int kPfRegsSoftmax = 224, kPfRegsOther = 56;
constexpr int kPfFirst = 64;     // keys whose P is handed over before the rest
static_assert(kPfFirst % 32 == 0 && kPfFirst >= 64 && kPfFirst < kPfRows, "a multiple of 32 behind the first 32");
constexpr float kPfSlack = 8.f;  // powers of two that the reference may stay behind

// A work item.
struct PfWork {
  int head, kvh;                       // first query head, KV head
  int q_start, q_len, k_start, k_len;  // the sequence
  int q0;                              // first query of the item in it
  // Item `block`: of its heads, block `block / units` of the queries, from a
  // sequence's last one on, and up to 32 sequences in the order of their keys (so
  // the longest items start first: 17 packed prompts 50.9 us in place of 54.7).  All
  // lanes of a warp call it.  False: there is none, nor any behind it.
  FRC_DEVICE_INLINE bool find(const PrefillParams& p, int block, int lane) {
    const int units = p.nh / p.heads;
    int rank = block / units;
    head = (block - rank * units) * p.heads;
    kvh = head / (p.nh / p.nkv);
    const int span = kPfTiles * p.queries;
    for (int top = p.batch; top > 0; top -= 32) {
      const int b = top - 1 - lane;
      int a0 = 0, a1 = 0, k0 = 0, k1 = 0;
      if (b >= 0) {
        a0 = min(max(p.cu_q[b], 0), p.tokens_q);
        a1 = min(max(p.cu_q[b + 1], a0), p.tokens_q);
        k0 = min(max(p.cu_k[b], 0), p.tokens_k);
        k1 = min(max(p.cu_k[b + 1], k0), p.tokens_k);
      }
      const int n = (a1 - a0 + span - 1) / span;
      int incl = n;
      if (p.batch > 1 && p.batch <= 32) {  // sequences with the most keys first: their items take longest
        const int keys = k1 - k0;
#pragma unroll 4
        for (int o = 0; o < 32; ++o) {
          const int other = __shfl_sync(0xffffffffu, keys, o), blocks = __shfl_sync(0xffffffffu, n, o);
          if (other > keys || (other == keys && o < lane)) incl += blocks;
        }
      } else {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, rank >= incl - n && rank < incl);
      if (!hit) {
        rank -= __shfl_sync(0xffffffffu, incl, 31);  // (of no account where there is no other 32)
        continue;
      }
      const int l = __ffs(hit) - 1;
      q_start = __shfl_sync(0xffffffffu, a0, l);
      q_len = __shfl_sync(0xffffffffu, a1, l) - q_start;
      const int blocks = __shfl_sync(0xffffffffu, n, l);
      const int in_seq = rank - (__shfl_sync(0xffffffffu, incl, l) - blocks);
      q0 = (blocks - 1 - in_seq) * span;
      k_start = __shfl_sync(0xffffffffu, k0, l);
      k_len = __shfl_sync(0xffffffffu, k1, l) - k_start;
      return true;
    }
    return false;
  }
  // Queries of a tile.
  FRC_DEVICE_INLINE int queries(const PrefillParams& p, int tile) const {
    return min(max(q_len - q0 - tile * p.queries, 0), p.queries);
  }
  // Keys that query `i` of the sequence sees.
  FRC_DEVICE_INLINE int seen(const PrefillParams& p, int i) const {
    return p.causal ? min(max(i + 1 + k_len - q_len, 0), k_len) : k_len;
  }
  // Key tiles of a query tile.
  FRC_DEVICE_INLINE int tiles(const PrefillParams& p, int tile) const {
    const int n = queries(p, tile);
    return n == 0 ? 0 : (seen(p, q0 + tile * p.queries + n - 1) + kPfRows - 1) / kPfRows;
  }
};

template <int HD>
struct PfSmem {
  static constexpr int kHalf = kPfRows * 128;           // 64 channels of 128 rows, swizzled: 16 KB
  static constexpr int kTile = HD / 64 * kHalf;
  static constexpr int kStages = HD == 128 ? 5 : 8;
  static constexpr int kVTiles = (kStages + 1) / 2;  // V tiles that the ring can hold: every second tile is one
  alignas(1024) uint8_t q[kPfTiles][kTile];
  alignas(1024) uint8_t ring[kStages][kTile];
  uint64_t q_full, q_empty, full[kStages], empty[kStages];
  uint64_t clean[kVTiles];  // V tile v of the CTA is ready: entry v % kVTiles
  uint64_t s_full[kPfTiles], p_ready[kPfTiles][2], o_done[kPfTiles], o_free[kPfTiles], drain;
  alignas(16) uint4 answer;  // to the request for the next block
  uint64_t answered;
  PfWork work[2];            // items 1, 2, ... by turns
  int any[2];                // whether there is one
  int taken_out[4];          // of items by turns: elements of V were zeroed
  uint64_t work_full[2], work_empty[2];
  uint32_t tmem;
  int abort;
};

// ---- tcgen05 ---------------------------------------------------------------------
// Descriptor of a tile of rows of 128 bytes, 128-byte swizzle (8-row atoms of
// 1024 bytes).  K-major (rows are M or N): the stride is between atoms and the
// leading offset unused.  MN-major (rows are K): the stride is between groups
// of eight rows of K, the leading offset between blocks of 64 columns.
FRC_DEVICE_INLINE uint64_t pf_desc(uint32_t addr, uint32_t leading) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | static_cast<uint64_t>((leading >> 4) & 0x3FFFu) << 16 |
         static_cast<uint64_t>(1024u >> 4) << 32 | static_cast<uint64_t>(1u) << 46 | static_cast<uint64_t>(2u) << 61;
}

template <typename T>
__host__ __device__ constexpr uint32_t pf_idesc(int n, bool b_mn_major) {
  constexpr uint32_t fmt = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;  // bf16 : fp16
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kPfRows >> 4) << 24);
}
constexpr uint32_t kPfNegateA = 1u << 13;

// One lane of the warp, the same each time.
FRC_DEVICE_INLINE uint32_t pf_elect() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one;
}

// The whole warp calls these, with the same operands in all lanes (so that they
// stay in uniform registers, which the instructions read); the elected lane issues.
// D (tensor memory) (+)= A (shared) B (shared)
FRC_DEVICE_INLINE void pf_mma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
// D (tensor memory) (+)= A (tensor memory) B (shared)
FRC_DEVICE_INLINE void pf_mma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
FRC_DEVICE_INLINE void pf_commit(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(one)
      : "memory");
}
FRC_DEVICE_INLINE void pf_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
FRC_DEVICE_INLINE void pf_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define FRC_R8(r, i) "=r"((r)[i]), "=r"((r)[i + 1]), "=r"((r)[i + 2]), "=r"((r)[i + 3]), "=r"((r)[i + 4]), "=r"((r)[i + 5]), "=r"((r)[i + 6]), "=r"((r)[i + 7])
#define FRC_I8(r, i) "r"((r)[i]), "r"((r)[i + 1]), "r"((r)[i + 2]), "r"((r)[i + 3]), "r"((r)[i + 4]), "r"((r)[i + 5]), "r"((r)[i + 6]), "r"((r)[i + 7])

// 32 columns of the lane's row; valid after tmem_wait_ld.
FRC_DEVICE_INLINE void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : FRC_R8(r, 0), FRC_R8(r, 8), FRC_R8(r, 16), FRC_R8(r, 24)
      : "r"(addr));
}
FRC_DEVICE_INLINE void tmem_ld16u(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : FRC_R8(r, 0), FRC_R8(r, 8)
      : "r"(addr));
}
FRC_DEVICE_INLINE void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::FRC_I8(r, 0),
      FRC_I8(r, 8), "r"(addr)
      : "memory");
}
FRC_DEVICE_INLINE void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
FRC_DEVICE_INLINE void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

FRC_DEVICE_INLINE void pf_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

FRC_DEVICE_INLINE float pf_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
FRC_DEVICE_INLINE uint32_t pf_pack(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

FRC_DEVICE_INLINE float pf_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// P of 32 scores: 2^(x scale + base), their sums, and the values rounded and
// packed.  (A quarter of the exponentials as polynomials on the multiply-add
// units took a third more instructions and gained nothing: 1042 against 1016 us
// for 64 heads of 8192 tokens.)
template <typename T>
FRC_DEVICE_INLINE void pf_exps(const uint32_t* x, uint64_t scale2, float base, uint64_t (&part)[4], uint32_t (&y)[16]) {
  const uint64_t base2 = f32x2_two(base, base);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint64_t v = f32x2_fma(f32x2_two(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), scale2, base2);
    float a, b;
    f32x2_split(v, a, b);
    a = pf_ex2(a);
    b = pf_ex2(b);
    part[e & 3] = f32x2_add(part[e & 3], f32x2_two(a, b));
    y[e] = pf_pack<T>(a, b);
  }
}

// Lane l of a quad has w of its row, four units of four words: afterwards unit k
// of lane l is unit l of lane k's row.
FRC_DEVICE_INLINE void pf_quad_transpose(uint32_t (&w)[16], int lane) {
#pragma unroll
  for (int o = 1; o < 4; o <<= 1)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (u & o) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t &a = w[4 * u + e], &b = w[4 * (u + o) + e];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, lane & o ? a : b, o);
        if (lane & o) a = got;
        else b = got;
      }
    }
}

// Asks for a block of the grid that has not started; the answer (16 bytes)
// arrives on `bar`.
FRC_DEVICE_INLINE void pf_ask(uint4* answer, uint64_t* bar) {
  mbar_arrive_expect_tx(bar, 16);
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
          smem_u32(answer)),
      "r"(smem_u32(bar))
      : "memory");
}
// Its index, or -1 where none is left.
FRC_DEVICE_INLINE int pf_answer(const uint4* answer) {
  int block;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "mov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n\t}"
      : "=r"(block)
      : "r"(smem_u32(answer))
      : "memory");
  fence_proxy_async_smem();  // before the next answer is written over it
  return block;
}

template <typename T>
constexpr uint32_t kPfInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;  // bits of infinity

// Zeroes the elements of a V tile's first `rows` rows that are not finite.  True:
// there are some.  A warp.
template <typename T, int HD>
FRC_DEVICE_INLINE bool pf_clean(uint8_t* tile, int rows, int lane) {
  constexpr uint32_t inf = kPfInf<T>;
  uint32_t top = 0;
  for (int h = 0; h < HD / 64; ++h) {
    const uint4* at = reinterpret_cast<const uint4*>(tile + h * PfSmem<HD>::kHalf);
#pragma unroll 4
    for (int e = lane; e < rows * 8; e += 32) {
      const uint4 v = at[e];
      top = __vmaxu2(top, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                   __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
    }
  }
  if (!__any_sync(0xffffffffu, (top & 0xffffu) >= inf || top >> 16 >= inf)) return false;
  for (int h = 0; h < HD / 64; ++h) {
    uint32_t* at = reinterpret_cast<uint32_t*>(tile + h * PfSmem<HD>::kHalf);
    for (int e = lane; e < rows * 32; e += 32) {
      const uint32_t v = at[e];
      const uint32_t keep = ((v & 0x7fffu) < inf ? 0xffffu : 0u) | ((v >> 16 & 0x7fffu) < inf ? 0xffff0000u : 0u);
      if (keep != 0xffffffffu) at[e] = v & keep;
    }
  }
  return true;
}

// Adds to the warp's rows what pf_clean took out of the tiles from key `first` on
// and they see: a value that is not finite makes the sum so whatever its weight.
// `at`: the lane's row of the output, `seen`: its keys (0: none, or no row).  At
// most 128 keys more than the item has queries, so the other warps do not wait long.
template <typename T, int HD>
__device__ __noinline__ void pf_add_seen(const PrefillParams& p, const PfWork& w, int first, int seen, int64_t at, int lane) {
  constexpr int C = HD / 32;
  const int end = __reduce_max_sync(0xffffffffu, seen);
  for (int j = first; j < end; ++j) {
    const T* vp = static_cast<const T*>(p.v) + (w.k_start + static_cast<int64_t>(j)) * p.v_tok + w.kvh * p.v_head + C * lane;
    float v[C];
    bool some = false;
#pragma unroll
    for (int e = 0; e < C; ++e) {
      v[e] = to_f32(vp[e]);
      if (fabsf(v[e]) <= 3.402823466e38f) v[e] = 0.f;  // finite: the products had it
      else some = true;
    }
    if (!__any_sync(0xffffffffu, some)) continue;
    for (uint32_t rows = __ballot_sync(0xffffffffu, seen > j); rows; rows &= rows - 1) {
      T* op = static_cast<T*>(p.out) + __shfl_sync(0xffffffffu, at, __ffs(rows) - 1) + C * lane;
#pragma unroll
      for (int e = 0; e < C; ++e)
        if (!(v[e] == 0.f)) from_f32(to_f32(op[e]) + v[e], op[e]);
    }
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kPfThreads, 1)
    attn_prefill_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap, const PrefillParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using SM = PfSmem<HD>;
  constexpr int NS = SM::kStages, H = HD / 64;
  extern __shared__ __align__(1024) uint8_t pf_smem[];
  SM* sh = reinterpret_cast<SM*>(pf_smem);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (smem_u32(pf_smem) & 1023u) {  // swizzled tiles need 1024-byte alignment
    if (threadIdx.x == 0) atomicOr(p.status, kStatusSmemMisaligned);
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(&sh->q_full, 1);
    mbar_init(&sh->q_empty, 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->empty[s], 1);
    }
    for (int t = 0; t < kPfTiles; ++t) {
      mbar_init(&sh->s_full[t], 1);
      mbar_init(&sh->p_ready[t][0], 4);
      mbar_init(&sh->p_ready[t][1], 4);
      mbar_init(&sh->o_done[t], 1);
      mbar_init(&sh->o_free[t], 4);
      mbar_init(&sh->work_full[t], 1);
      mbar_init(&sh->work_empty[t], 10);  // the softmax warps, the product warp and warp 10
    }
    for (int v = 0; v < SM::kVTiles; ++v) mbar_init(&sh->clean[v], 1);
    mbar_init(&sh->answered, 1);
    mbar_init(&sh->drain, 1);
    sh->abort = 0;
    fence_barrier_init();
  }
  // rows that no query is loaded to: zeros, so that they raise no reference
  for (int t = 0; t < kPfTiles; ++t)
    for (int h = 0; h < H; ++h)
      for (int i = p.heads * p.queries * 8 + threadIdx.x; i < kPfRows * 8; i += kPfThreads)
        reinterpret_cast<uint4*>(sh->q[t] + h * SM::kHalf)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh->tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (warp == 9 && lane == 0)
    for (const CUtensorMap* map : {&qmap, &kmap, &vmap}) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  // Item 0 of this CTA is the block it was launched as; the others are blocks it
  // took over, found by the loading warp an item ahead.
  PfWork w;
  bool any = w.find(p, blockIdx.x, lane);  // false: there is none, nor any behind it
  pf_fence_before();
  __syncthreads();
  pf_fence_after();
  const uint32_t tmem = sh->tmem;  // S of tile t at column 128 t, O at 256 + HD t
  volatile int* abort = &sh->abort;
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // a warp's bounded wait
    return __all_sync(0xffffffffu, wait_phase(bar, parity & 1, abort));
  };

  auto follow = [&](int i) {  // item i + 1 into w and any
    const int slot = (i + 1) & 1;
    if (!wait(&sh->work_full[slot], i >> 1)) return false;
    w = sh->work[slot];
    any = sh->any[slot] != 0;
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh->work_empty[slot]);
    return true;
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPfRegsOther));
    if (warp == 9) {
      // ---- loads -----------------------------------------------------------------------
      int issued = 0, items = 0;  // K and V tiles, items that had queries
      bool ok = true;
      for (int i = 0; any; ++i) {
        if (lane == 0) pf_ask(&sh->answer, &sh->answered);
        const int n = max(w.tiles(p, 0), w.tiles(p, 1));
        if (n > 0) {
          if (items > 0) ok = wait(&sh->q_empty, items - 1);
          if (ok && lane == 0) {
            const int q_tiles = w.queries(p, 1) > 0 ? 2 : 1;
            mbar_arrive_expect_tx(&sh->q_full, q_tiles * H * 128 * p.heads * p.queries);
            for (int t = 0; t < q_tiles; ++t)
              for (int h = 0; h < H; ++h)
                pf_load_3d(sh->q[t] + h * SM::kHalf, &qmap, 64 * h, w.head, w.q_start + w.q0 + t * p.queries,
                           &sh->q_full);
          }
          if (ok) ++items;
          for (int l = 0; ok && l < 2 * n; ++l) {  // K 0, V 0, K 1, V 1, ...
            const int s = issued % NS;
            if (issued >= NS) ok = wait(&sh->empty[s], issued / NS - 1);
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&sh->full[s], SM::kTile);
              const int key = w.k_start + (l >> 1) * kPfRows;
              for (int h = 0; h < H; ++h)
                pf_load_3d(sh->ring[s] + h * SM::kHalf, l & 1 ? &vmap : &kmap, 64 * h,
                           w.kvh * (l & 1 ? p.v_mul : p.k_mul), key, &sh->full[s]);
            }
            ++issued;
          }
        }
        // the answer is waited for in any case: it must not land after the CTA
        int zero = 0;
        ok = __all_sync(0xffffffffu, wait_phase(&sh->answered, i & 1, &zero)) && ok;
        const int block = pf_answer(&sh->answer), slot = (i + 1) & 1;
        any = ok && block >= 0 && w.find(p, block, lane);
        if (i >= 2) ok = ok && wait(&sh->work_empty[slot], (i >> 1) - 1);
        if (!ok) break;
        if (lane == 0) {
          sh->work[slot] = w;
          sh->any[slot] = any;
          mbar_arrive(&sh->work_full[slot]);
        }
        __syncwarp();
      }
      if (!ok) {
        *abort = 1;
        if (lane == 0) atomicOr(p.status, kStatusEmptyWaitTimeout);
      }
      // no copy may still be landing when the CTA exits
      int zero = 0;
      bool landed = items == 0 || wait_phase(&sh->q_full, (items - 1) & 1, &zero);
      for (int l = issued > NS ? issued - NS : 0; l < issued; ++l)
        landed = wait_phase(&sh->full[l % NS], (l / NS) & 1, &zero) && landed;
      if (!landed && lane == 0) atomicOr(p.status, kStatusDrainTimeout);
    } else if (warp == 8) {
      // ---- products: the elected lane issues -----------------------------------------------
      constexpr uint32_t id_pv = pf_idesc<T>(HD, true);
      const uint32_t id_qk = pf_idesc<T>(kPfRows, false) | (p.negate ? kPfNegateA : 0u);
      const uint32_t one = pf_elect();
      const uint64_t q_desc = pf_desc(smem_u32(sh->q[0]), 16);
      const uint64_t k_desc = pf_desc(smem_u32(sh->ring[0]), 16), v_desc = pf_desc(smem_u32(sh->ring[0]), SM::kHalf);
      auto qk = [&](int t, int stage) {
        const uint64_t a = q_desc + t * (SM::kTile >> 4), b = k_desc + stage * (SM::kTile >> 4);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const int off = k / 4 * (SM::kHalf >> 4) + k % 4 * (32 >> 4);
          pf_mma_ss(one, tmem + 128 * t, a + off, b + off, id_qk, k > 0);
        }
        pf_commit(one, &sh->s_full[t]);
      };
      auto pv = [&](int t, int stage, auto k0, auto k1, bool first) {
        const uint64_t b = v_desc + stage * (SM::kTile >> 4);
#pragma unroll
        for (int k = k0(); k < k1(); ++k)
          pf_mma_ts(one, tmem + 256 + HD * t, tmem + 128 * t + 8 * k, b + k * (2048 >> 4), id_pv, !first || k > 0);
      };
      auto release = [&](int stage) { pf_commit(one, &sh->empty[stage]); };
      bool ok = true;
      int used = 0, items = 0;                           // K and V tiles, items that had queries
      int v_used = 0;                                    // V tiles
      int done[kPfTiles] = {0, 0}, outs[kPfTiles] = {0, 0};  // key tiles and items of each query tile
      for (int i = 0; ok && any; ++i) {
        const int nt[kPfTiles] = {w.tiles(p, 0), w.tiles(p, 1)};
        const int n = max(nt[0], nt[1]);
        if (n > 0) {
          ok = wait(&sh->q_full, items) && wait(&sh->full[used % NS], used / NS);
          if (!ok) break;
          ++items;
          pf_fence_after();
          for (int t = 0; t < kPfTiles; ++t)
            if (nt[t] > 0) qk(t, used % NS);
          release(used % NS);
          if (n == 1) pf_commit(one, &sh->q_empty);
          ++used;
          for (int j = 0; ok && j < n; ++j) {
            const int sv = used % NS, sk = (used + 1) % NS;
            ok = wait(&sh->full[sv], used / NS) && wait(&sh->clean[v_used % SM::kVTiles], v_used / SM::kVTiles);
            if (!ok) break;
            ++v_used;
            bool k_there = false;
#pragma unroll
            for (int t = 0; t < kPfTiles; ++t) {
              if (j >= nt[t]) continue;
              // the last item's O has been read before it is overwritten
              if (j == 0 && outs[t] > 0) ok = ok && wait(&sh->o_free[t], outs[t] - 1);
              ok = ok && wait(&sh->p_ready[t][0], done[t]);
              if (!ok) break;
              pf_fence_after();
              pv(t, sv, [] { return 0; }, [] { return kPfFirst / 16; }, j == 0);
              ok = wait(&sh->p_ready[t][1], done[t]);
              if (!ok) break;
              pf_fence_after();
              pv(t, sv, [] { return kPfFirst / 16; }, [] { return kPfRows / 16; }, false);
              pf_commit(one, &sh->o_done[t]);
              ++done[t];
              if (j + 1 < nt[t]) {
                if (!k_there) ok = wait(&sh->full[sk], (used + 1) / NS);
                if (!ok) break;
                k_there = true;
                pf_fence_after();
                qk(t, sk);
              }
            }
            if (!ok) break;
            release(sv);
            ++used;
            if (j + 1 < n) {
              release(sk);
              ++used;
              if (j + 2 == n) pf_commit(one, &sh->q_empty);  // the queries' last use
            }
          }
          for (int t = 0; t < kPfTiles; ++t) outs[t] += nt[t] > 0;
        }
        ok = ok && follow(i);
      }
      if (!ok) {
        *abort = 1;
        if (lane == 0) atomicOr(p.status, kStatusFullWaitTimeout);
      }
      // no product may be in flight at the teardown
      pf_commit(one, &sh->drain);
      int zero = 0;
      if (!wait_phase(&sh->drain, 0, &zero) && lane == 0) atomicOr(p.status, kStatusDrainTimeout);
    } else if (warp == 10) {
      // ---- V tiles made ready ------------------------------------------------------------------
      // A V tile's stage is not filled again before the product warp has waited for
      // its entry of `clean`, so this warp misses no phase of `full`; and the ring holds
      // no more V tiles than `clean` has entries, so the product warp misses none.
      bool ok = true;
      int used = 0, v_used = 0;
      for (int i = 0; ok && any; ++i) {
        const int n = max(w.tiles(p, 0), w.tiles(p, 1));
        const int whole = p.causal ? w.seen(p, w.q0) / kPfRows : n;  // tiles that all rows see whole
        // read by the softmax warps at the end of the item; two items ahead at most, this
        // warp writes no other's entry
        volatile int* taken_out = &sh->taken_out[i & 3];
        if (lane == 0) *taken_out = 0;
        __syncwarp();
        for (int j = 0; j < n; ++j, used += 2, ++v_used) {
          const int s = (used + 1) % NS, left = w.k_len - j * kPfRows;
          ok = wait(&sh->full[s], (used + 1) / NS);
          if (!ok) break;
          if (j >= whole && pf_clean<T, HD>(sh->ring[s], min(left, kPfRows), lane)) *taken_out = 1;
          if (left < kPfRows) {  // rows behind the last key: zeros, whatever lies there
            uint4* row = reinterpret_cast<uint4*>(sh->ring[s]);
            for (int h = 0; h < H; ++h)
              for (int e = left * 8 + lane; e < kPfRows * 8; e += 32)
                row[h * (SM::kHalf / 16) + e] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->clean[v_used % SM::kVTiles]);
        }
        ok = ok && follow(i);
      }
      if (!ok) {
        *abort = 1;
        if (lane == 0) atomicOr(p.status, kStatusFullWaitTimeout);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPfRegsSoftmax));
    // ---- softmax: warps 4 t .. 4 t + 3 have tile t, a row a thread ------------------------
    const int t = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_at = tmem + lanes + 128 * t, o_at = tmem + lanes + 256 + HD * t;
    const int r = 32 * (warp & 3) + lane, my_query = r / p.heads, my_head = r - my_query * p.heads;
    const float scale = p.scale;
    const uint64_t scale2 = f32x2_two(scale, scale);
    bool ok = true;
    int done = 0;  // key tiles
    for (int i = 0; ok && any; ++i) {
      const int nt = w.tiles(p, t), row = w.q0 + p.queries * t + my_query;
      const bool live = my_query < w.queries(p, t);
      // rows without a query mask as the tile's last one
      const int seen = w.seen(p, min(row, w.q0 + p.queries * t + w.queries(p, t) - 1));
      float m_ref = -INFINITY, base = 0.f, sum = 0.f;  // reference in units of the unscaled score, and scaled
      for (int j = 0; j < nt; ++j, ++done) {
        ok = wait(&sh->s_full[t], done);
        if (!ok) break;
        pf_fence_after();
        uint32_t x[kPfRows];
#pragma unroll
        for (int c = 0; c < kPfRows; c += 32) tmem_ld32(s_at + c, x + c);
        tmem_wait_ld();
        const int mine = seen - j * kPfRows;  // columns that the row sees
        if (!__all_sync(0xffffffffu, mine >= kPfRows)) {
          const int least = __reduce_min_sync(0xffffffffu, mine);
#pragma unroll
          for (int c = 0; c < kPfRows; c += 32)
            if (c + 32 > least) {
#pragma unroll
              for (int e = c; e < c + 32; ++e) x[e] = e < mine ? x[e] : 0xff800000u;
            }
        }
        // the first quarter's exponentials run with the old reference while the
        // maximum is formed, and again in the few tiles that raise it
        uint64_t part[4] = {0, 0, 0, 0};
        uint32_t y[16];
        pf_exps<T>(x, scale2, base, part, y);
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kPfRows; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            mx[e] = pf_max3(mx[e], __uint_as_float(x[c + 2 * e]), __uint_as_float(x[c + 2 * e + 1]));
        const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (__any_sync(0xffffffffu, (m - m_ref) * scale > kPfSlack)) {
          const float m_new = fmaxf(m, m_ref);
          const float keep = m_new == -INFINITY ? 1.f : pf_ex2((m_ref - m_new) * scale);
          m_ref = m_new;
          base = m_new == -INFINITY ? 0.f : -m_new * scale;
          sum *= keep;
          if (j > 0) {
            ok = wait(&sh->o_done[t], done - 1);
            if (!ok) break;
            pf_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
              uint32_t o[16];
              tmem_ld16u(o_at + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
              tmem_st16(o_at + c, o);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) part[e] = 0;
          pf_exps<T>(x, scale2, base, part, y);
        }
        tmem_st16(s_at, y);
#pragma unroll
        for (int c = 32; c < kPfRows; c += 32) {
          pf_exps<T>(x + c, scale2, base, part, y);
          tmem_st16(s_at + c / 2, y);
          if (c == kPfFirst - 32) {  // P's first part can be multiplied
            tmem_wait_st();
            pf_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->p_ready[t][0]);
          }
        }
        tmem_wait_st();
        pf_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_ready[t][1]);
        float a0, a1;
        f32x2_split(f32x2_add(f32x2_add(part[0], part[1]), f32x2_add(part[2], part[3])), a0, a1);
        sum += a0 + a1;
      }
      // ---- O / sum ---------------------------------------------------------------------
      if (ok && nt > 0) ok = wait(&sh->o_done[t], done - 1);
      if (!ok) break;
      pf_fence_after();
      const float inv = 1.f / sum;  // all scores -inf: 0 / 0
      const int64_t at = static_cast<int64_t>(w.q_start + row) * p.o_tok + (w.head + my_head) * p.o_head;
      T* quad[4];  // the rows of the quad's lanes, from this lane's unit on
#pragma unroll
      for (int k = 0; k < 4; ++k)
        quad[k] = static_cast<T*>(p.out) + __shfl_sync(0xffffffffu, at, (lane & ~3) + k) + 8 * (lane & 3);
      const uint32_t rows = __ballot_sync(0xffffffffu, live) >> (lane & ~3);
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        uint32_t y[16];
        if (nt > 0) {
          uint32_t o[32];
          tmem_ld32(o_at + c, o);
          tmem_wait_ld();
          if (c == HD - 32) {
            pf_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->o_free[t]);
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float v0 = __uint_as_float(o[e]) * inv, v1 = __uint_as_float(o[e + 1]) * inv;
            y[e / 2] = seen == 0 ? 0u : pf_pack<T>(v0, v1);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = 0u;
        }
        // 64 bytes of a row in one store, not of 32 rows 16 each
        pf_quad_transpose(y, lane);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (rows >> k & 1u)
            *reinterpret_cast<uint4*>(quad[k] + c) = make_uint4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
      }
      if (nt > 0 && *static_cast<volatile int*>(&sh->taken_out[i & 3])) {
        __syncwarp();  // the rows were written by the lanes of their quads
        pf_add_seen<T, HD>(p, w, w.seen(p, w.q0) / kPfRows * kPfRows, live ? seen : 0, at, lane);
      }
      ok = follow(i);
    }
    if (!ok && lane == 0) atomicOr(p.status, kStatusFullWaitTimeout);
  }
  // ---- teardown: every warp here, no product or tensor-memory access in flight -----------
  pf_fence_before();
  __syncthreads();
  if (warp == 8) {
    pf_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Map of (tokens, heads, hd) in boxes of 64 channels of `box_heads` heads of
// `box_tokens` tokens; a head stride of 0 (a broadcast head) is a map of one head.
inline bool pf_map(CUtensorMap* map, int type, const void* base, int64_t tokens, int heads, int hd, int64_t tok_stride,
                   int64_t head_stride, int box_heads, int box_tokens) {
  auto encode = tensor_map_encoder();
  if (!encode) return false;
  const bool one = heads == 1 || head_stride == 0;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(hd), static_cast<cuuint64_t>(one ? 1 : heads),
                              static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(one ? hd : head_stride) * 2,
                                 static_cast<cuuint64_t>(tokens == 1 ? hd : tok_stride) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
  const cuuint32_t step[3] = {1, 1, 1};
  std::memset(map, 0, sizeof *map);
  return encode(map, type == FRC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Query heads of a tile: the most of a KV head's (a divisor of their number)
// that leave at most 4 of a tile's 128 rows unused.
inline int pf_heads(int group) {
  for (int d = group < kPfRows ? group : kPfRows; d > 1; --d)
    if (group % d == 0 && kPfRows / d * d >= kPfRows - 4) return d;
  return 1;
}

template <typename T, int HD>
cudaError_t launch_prefill(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const PrefillParams& p,
                           cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may use its shared memory
  const cudaError_t e = allow_smem(attn_prefill_kernel<T, HD>, sizeof(PfSmem<HD>), ready);
  if (e != cudaSuccess) return e;
  return launch_pdl(attn_prefill_kernel<T, HD>, dim3(static_cast<unsigned>(p.q_blocks) * (p.nh / p.heads)), dim3(kPfThreads),
                    sizeof(PfSmem<HD>), st, q, k, v, p);
}

}  // namespace frc

extern "C" int frc_attention_prefill(int type, const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                                     const void* k, int64_t k_tok_stride, int64_t k_head_stride, const void* v,
                                     int64_t v_tok_stride, int64_t v_head_stride, const int* cu_q, const int* cu_k,
                                     int batch, int64_t tokens_q, int64_t tokens_k, int nh, int nkv, int hd,
                                     float scale, int causal, void* out, int64_t out_tok_stride,
                                     int64_t out_head_stride, void* stream) {
  FRC_REQUIRE(type == FRC_F16 || type == FRC_BF16, "frc_attention_prefill: type must be FRC_F16 or FRC_BF16");
  FRC_REQUIRE(hd == 64 || hd == 128, "frc_attention_prefill: head_dim must be 64 or 128");
  FRC_REQUIRE(nh > 0 && nkv > 0 && nh <= 65535 && nh % nkv == 0, "frc_attention_prefill: needs nh a multiple of nkv");
  FRC_REQUIRE(batch >= 0 && tokens_q >= 0 && tokens_k >= 0 && tokens_q <= (1 << 30) && tokens_k <= (1 << 30),
              "frc_attention_prefill: bad batch or tokens");
  // (an item's sequence is found 32 at a time, while the other warps' waits run: some 15 ms for as many)
  FRC_REQUIRE(batch <= (1 << 20), "frc_attention_prefill: more than 2^20 sequences");
  const int64_t strides[] = {q_tok_stride, q_head_stride, k_tok_stride, k_head_stride,
                             v_tok_stride, v_head_stride, out_tok_stride, out_head_stride};
  for (const int64_t s : strides)
    FRC_REQUIRE(s >= 0 && s % 8 == 0 && s < (int64_t(1) << 38),
                "frc_attention_prefill: strides must be multiples of 8 elements, below 2^38");
  FRC_REQUIRE((q_tok_stride > 0 || tokens_q <= 1) && ((k_tok_stride > 0 && v_tok_stride > 0) || tokens_k <= 1),
              "frc_attention_prefill: token strides must not be zero");
  FRC_REQUIRE((q_head_stride > 0 && out_head_stride > 0) || nh == 1,
              "frc_attention_prefill: the heads of q and out must not be one");
  FRC_REQUIRE(scale == scale && scale - scale == 0.f, "frc_attention_prefill: scale must be finite");
  if (batch == 0 || tokens_q == 0) return FRC_OK;
  FRC_REQUIRE(q && ((k && v) || tokens_k == 0) && cu_q && cu_k && out, "frc_attention_prefill: null pointer");
  FRC_REQUIRE(frc::aligned_to(q, 16) && frc::aligned_to(k, 16) && frc::aligned_to(v, 16) && frc::aligned_to(out, 16),
              "frc_attention_prefill: q, k, v and out must be 16-byte aligned");
  const frc::View results(out, 2, tokens_q, out_tok_stride, nh, out_head_stride, hd);
  FRC_REQUIRE(results.distinct(), "frc_attention_prefill: the rows or heads of out overlap");
  FRC_REQUIRE(!frc::views_share(results, frc::View(q, 2, tokens_q, q_tok_stride, nh, q_head_stride, hd)) &&
                  !frc::views_share(results, frc::View(k, 2, tokens_k, k_tok_stride, nkv, k_head_stride, hd)) &&
                  !frc::views_share(results, frc::View(v, 2, tokens_k, v_tok_stride, nkv, v_head_stride, hd)),
              "frc_attention_prefill: out shares memory with q, k or v");
  frc::PrefillParams p{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_tok = q_tok_stride;
  p.q_head = q_head_stride;
  p.k_tok = k_tok_stride;
  p.k_head = k_head_stride;
  p.v_tok = v_tok_stride;
  p.v_head = v_head_stride;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.batch = batch;
  p.tokens_q = static_cast<int>(tokens_q);
  p.tokens_k = static_cast<int>(tokens_k);
  p.nh = nh;
  p.nkv = nkv;
  p.signed_scale = scale;
  p.negate = scale < 0.f;
  // a scale of 0 weighs all keys alike: so does one that takes any finite score to next to nothing
  const float size = scale < 0.f ? -scale : scale;
  p.scale = size < 1e-30f ? 1e-30f : size * 1.44269504088896341f;
  p.causal = causal != 0;
  p.heads = frc::pf_heads(nh / nkv);
  p.queries = frc::kPfRows / p.heads;
  p.k_mul = k_head_stride != 0;
  p.v_mul = v_head_stride != 0;
  // at most: a partly filled block for each sequence that has a query
  const int64_t per = frc::kPfTiles * p.queries;
  const int64_t blocks = tokens_q / per + (batch < tokens_q ? batch : tokens_q);
  FRC_REQUIRE(blocks * (nh / p.heads) <= 0x7fffffff, "frc_attention_prefill: too many queries");
  p.q_blocks = static_cast<int>(blocks);
  p.out = out;
  p.o_tok = out_tok_stride;
  p.o_head = out_head_stride;
  FRC_LAUNCHED(frc::serving_status(&p.status), "status word");
  CUtensorMap qm, km, vm;
  const bool none = tokens_k == 0;  // no key is read: any valid map will do
  const int rows = frc::kPfRows;
  if (!frc::pf_map(&qm, type, q, tokens_q, nh, hd, q_tok_stride, q_head_stride, p.heads, p.queries) ||
      !frc::pf_map(&km, type, none ? q : k, none ? tokens_q : tokens_k, none ? nh : nkv, hd,
                   none ? q_tok_stride : k_tok_stride, none ? q_head_stride : k_head_stride, 1, rows) ||
      !frc::pf_map(&vm, type, none ? q : v, none ? tokens_q : tokens_k, none ? nh : nkv, hd,
                   none ? q_tok_stride : v_tok_stride, none ? q_head_stride : v_head_stride, 1, rows))
    return frc__fail(FRC_ERR_CUDA, "frc_attention_prefill: cuTensorMapEncodeTiled failed");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = type == FRC_BF16;
  FRC_LAUNCHED((hd == 128 ? (bf ? frc::launch_prefill<__nv_bfloat16, 128>(qm, km, vm, p, st)
                                : frc::launch_prefill<__half, 128>(qm, km, vm, p, st))
                          : (bf ? frc::launch_prefill<__nv_bfloat16, 64>(qm, km, vm, p, st)
                                : frc::launch_prefill<__half, 64>(qm, km, vm, p, st))),
               "attention_prefill launch");
  return FRC_OK;
}
