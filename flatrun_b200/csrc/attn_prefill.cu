// Attention of whole prompts: packed sequences of different lengths, grouped
// heads, causal or not,
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j
//
// over the keys j of the sequence of query i; causal: the last query sees
// every key, each earlier one a key less (so a prompt may follow tokens that
// are there already).  A query that sees no key gives zeros, and rows behind
// the last sequence stay as they are.
#include <cuda_runtime.h>

#include <cstdio>

#include "../../include/frcuda.h"
#include "kv_q4.cuh"

namespace frc {

struct PrefillParams {
  const void *q, *k, *v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  const int *cu_q, *cu_k;
  int batch;
  int64_t tokens_q, tokens_k;
  int nh, nkv;
  float scale;
  int causal;
  void* out;
  int64_t o_tok, o_head;
};

// One warp for each (query, head).
template <typename T, int HD>
__global__ void __launch_bounds__(32) attn_prefill_kernel(PrefillParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" :::);
  constexpr int C = HD / 32;
  const int64_t i = blockIdx.x;
  const int h = blockIdx.y, g = h / (p.nh / p.nkv), lane = threadIdx.x;
  int b = 0;
  while (b < p.batch && p.cu_q[b + 1] <= i) ++b;
  if (b == p.batch || p.cu_q[b] > i) return;
  const int64_t k0 = max(p.cu_k[b], 0);
  int64_t k1 = min(static_cast<int64_t>(p.cu_k[b + 1]), p.tokens_k);
  if (p.causal) k1 -= p.cu_q[b + 1] - 1 - i;
  const T* qp = static_cast<const T*>(p.q) + i * p.q_tok + h * p.q_head;
  float qv[C], acc[C];
#pragma unroll
  for (int e = 0; e < C; ++e) {
    qv[e] = to_f32(qp[C * lane + e]) * p.scale;
    acc[e] = 0.f;
  }
  float mx = -INFINITY, sum = 0.f;
  for (int64_t j = k0; j < k1; ++j) {
    const T* kp = static_cast<const T*>(p.k) + j * p.k_tok + g * p.k_head + C * lane;
    const T* vp = static_cast<const T*>(p.v) + j * p.v_tok + g * p.v_head + C * lane;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < C; ++e) s = fmaf(qv[e], to_f32(kp[e]), s);
    s = warp_sum(s);
    const float m_new = fmaxf(mx, s), keep = mx == m_new ? 1.f : expf(mx - m_new), w = expf(s - m_new);
    mx = m_new;
    sum = fmaf(sum, keep, w);
#pragma unroll
    for (int e = 0; e < C; ++e) acc[e] = fmaf(acc[e], keep, w * to_f32(vp[e]));
  }
  T* op = static_cast<T*>(p.out) + i * p.o_tok + h * p.o_head;
  const float inv = mx == -INFINITY ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < C; ++e) from_f32(acc[e] * inv, op[C * lane + e]);
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
  FRC_REQUIRE(batch >= 0 && tokens_q >= 0 && tokens_k >= 0 && tokens_q <= 0x7fffffff && tokens_k <= 0x7fffffff,
              "frc_attention_prefill: bad batch or tokens");
  const int64_t strides[] = {q_tok_stride, q_head_stride, k_tok_stride, k_head_stride,
                             v_tok_stride, v_head_stride, out_tok_stride, out_head_stride};
  for (const int64_t s : strides)
    FRC_REQUIRE(s >= 0 && s % 8 == 0, "frc_attention_prefill: strides must be multiples of 8 elements");
  if (batch == 0 || tokens_q == 0) return FRC_OK;
  FRC_REQUIRE(q && ((k && v) || tokens_k == 0) && cu_q && cu_k && out, "frc_attention_prefill: null pointer");
  FRC_REQUIRE(frc::aligned_to(q, 16) && frc::aligned_to(k, 16) && frc::aligned_to(v, 16) && frc::aligned_to(out, 16),
              "frc_attention_prefill: q, k, v and out must be 16-byte aligned");
  const frc::PrefillParams p{q, k, v, q_tok_stride, q_head_stride, k_tok_stride, k_head_stride, v_tok_stride,
                             v_head_stride, cu_q, cu_k, batch, tokens_q, tokens_k, nh, nkv, scale, causal, out,
                             out_tok_stride, out_head_stride};
  return frc_with_type(type, [&](auto* z) -> int {
    using T = std::remove_pointer_t<decltype(z)>;
    void (*fn)(frc::PrefillParams) = hd == 128 ? frc::attn_prefill_kernel<T, 128> : frc::attn_prefill_kernel<T, 64>;
    FRC_LAUNCHED(frc::launch_pdl(fn, dim3(static_cast<unsigned>(tokens_q), nh), dim3(32), 0,
                                 static_cast<cudaStream_t>(stream), p),
                 "attention_prefill launch");
    return FRC_OK;
  });
}
