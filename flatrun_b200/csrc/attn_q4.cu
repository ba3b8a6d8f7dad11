// Decode attention over the 4-bit paged cache: one query token for each of
// `batch` sequences of different lengths,
//
//   s_t = scale * q . k_t,   o = sum_t softmax(s)_t v_t,   t < length
//
// query head h reading KV head h / (nh / nkv).  A page number outside the
// cache hides the page's tokens, and a sequence of no (visible) tokens gives
// zeros, so no table can lead a read out of the cache.
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdio>

#include "../../include/frcuda.h"
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
  float scale;
  void* out;
  int64_t o_seq, o_head;
};

// One warp for each (sequence, query head): a lane holds HD / 32 channels,
// and the tokens follow one another with a running maximum and sum.
template <typename T, int HD>
__global__ void __launch_bounds__(32) attn_q4_kernel(AttnQ4Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" :::);
  constexpr Q4Layout lay(HD);
  constexpr int C = HD / 32;
  const int b = blockIdx.y, h = blockIdx.x, g = h / (p.nh / p.nkv), lane = threadIdx.x;
  const T* qp = static_cast<const T*>(p.q) + b * p.q_seq + h * p.q_head;
  float qv[C], acc[C];
#pragma unroll
  for (int e = 0; e < C; ++e) {
    qv[e] = to_f32(qp[C * lane + e]) * p.scale;
    acc[e] = 0.f;
  }
  const int per_page = p.blocks_per_page * kQ4Tokens;
  const int64_t room = static_cast<int64_t>(p.max_pages) * per_page;
  const int len = static_cast<int>(p.lengths[b] < room ? p.lengths[b] : room);
  float mx = -INFINITY, sum = 0.f;
  for (int t = 0; t < len; ++t) {
    const int page = p.table[b * p.table_stride + t / per_page];
    if (page < 0 || page >= p.pages) continue;
    const uint8_t* blk = p.cache + ((static_cast<int64_t>(page) * p.nkv + g) * p.blocks_per_page +
                                    t % per_page / kQ4Tokens) * lay.block_bytes();
    const int u = t % kQ4Tokens;
    float s = 0.f, v[C];
#pragma unroll
    for (int e = 0; e < C; ++e) {
      const int c = C * lane + e, j = c / 32, w = c / 8;
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(blk + lay.k_word(u, w & 3, j));
      const uint32_t vw = *reinterpret_cast<const uint32_t*>(blk + lay.v_word(w, u));
      const float k = fmaf(static_cast<float>((kw >> (4 * (c & 7))) & 15u),
                           __half2float(*reinterpret_cast<const __half*>(blk + lay.k_step(j, u))),
                           __half2float(*reinterpret_cast<const __half*>(blk + lay.k_offset(u, j))));
      v[e] = fmaf(static_cast<float>((vw >> (4 * (c & 7))) & 15u),
                  __half2float(*reinterpret_cast<const __half*>(blk + lay.v_step(j, u))),
                  __half2float(*reinterpret_cast<const __half*>(blk + lay.v_offset(j, u))));
      s = fmaf(qv[e], k, s);
    }
    s = warp_sum(s);
    const float m_new = fmaxf(mx, s), keep = mx == m_new ? 1.f : expf(mx - m_new), w = expf(s - m_new);
    mx = m_new;
    sum = fmaf(sum, keep, w);
#pragma unroll
    for (int e = 0; e < C; ++e) acc[e] = fmaf(acc[e], keep, w * v[e]);
  }
  T* op = static_cast<T*>(p.out) + b * p.o_seq + h * p.o_head;
  const float inv = mx == -INFINITY ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < C; ++e) from_f32(acc[e] * inv, op[C * lane + e]);
}

}  // namespace frc

extern "C" {

int frc_attention_decode_q4_workspace(int batch, int nh, int nkv, int hd, size_t* bytes) {
  FRC_REQUIRE(bytes && batch >= 0 && nh > 0 && nkv > 0 && nh % nkv == 0 && (hd == 64 || hd == 128),
              "frc_attention_decode_q4_workspace: bad arguments");
  *bytes = 16;
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
  FRC_REQUIRE(pages > 0 && pages <= 0x7fffffff / (page_size / frc::kQ4Tokens),
              "frc_attention_decode_q4: bad number of pages");
  FRC_REQUIRE(batch >= 0 && batch <= 65535 && max_pages >= 0 && table_stride >= 0,
              "frc_attention_decode_q4: bad batch or block table");
  FRC_REQUIRE(q_seq_stride >= 0 && q_head_stride >= 0 && out_seq_stride >= 0 && out_head_stride >= 0,
              "frc_attention_decode_q4: negative stride");
  if (batch == 0) return FRC_OK;
  FRC_REQUIRE(q && cache && (block_table || max_pages == 0) && lengths && out && workspace,
              "frc_attention_decode_q4: null pointer");
  FRC_REQUIRE(frc::aligned_to(cache, 16) && frc::aligned_to(workspace, 16),
              "frc_attention_decode_q4: cache and workspace must be 16-byte aligned");
  size_t need = 0;
  const int rc = frc_attention_decode_q4_workspace(batch, nh, nkv, hd, &need);
  if (rc) return rc;
  FRC_REQUIRE(workspace_bytes >= need, "frc_attention_decode_q4: workspace is too small");
  const frc::AttnQ4Params p{q,       q_seq_stride, q_head_stride, static_cast<const uint8_t*>(cache), pages,
                            page_size / frc::kQ4Tokens, block_table, table_stride, max_pages, lengths, batch, nh, nkv,
                            scale,   out,          out_seq_stride, out_head_stride};
  return frc_with_type(type, [&](auto* z) -> int {
    using T = std::remove_pointer_t<decltype(z)>;
    void (*fn)(frc::AttnQ4Params) = hd == 128 ? frc::attn_q4_kernel<T, 128> : frc::attn_q4_kernel<T, 64>;
    FRC_LAUNCHED(frc::launch_pdl(fn, dim3(nh, batch), dim3(32), 0, static_cast<cudaStream_t>(stream), p),
                 "attention_decode_q4 launch");
    return FRC_OK;
  });
}

}  // extern "C"
