// Queries, keys and values of a batch of tokens made ready for attention in
// one pass: bias, RMS norm of each query and key head, position rotation,
// conversion to the type that attention reads.
//
//   h = x + bias;  h = h * (1 / sqrt(mean(h^2) + eps)) * w     (q and k heads)
//   (a, b) -> (a cos - b sin, b cos + a sin)                   (first rot channels)
//
// with the pairs (i, i + rot / 2) ("half") or (2 i, 2 i + 1) ("interleaved"),
// and cos / sin of the token's position from tables [max_pos][rot / 2].
//
// Bound by HBM: every element is read and written once (the tables are small
// beside them).  A head is handled by a group of L lanes of one warp, each
// lane holding two runs of VEC channels, so that both channels of a pair are
// in one lane for either layout, the norm is a sum over L lanes, and a head
// that is written in place has been read before.  A group walks over heads of
// ONE token and keeps the token's cos and sin in registers.  8192 tokens of 64 + 2 * 8
// heads of 128, fp32 to bf16: 87 us, 5.8 TB/s (0.89 of a plain copy).  16-bit rows
// have half the bytes in flight (two 8-byte loads a lane): 4096 tokens bf16 to bf16
// 41 us, 4.1 TB/s.
#include <cuda_runtime.h>

#include <cstdio>

#include "../../include/frcuda.h"
#include "kv_q4.cuh"

namespace frc {

struct RopeParams {
  const void* qkv;
  int64_t row_stride;  // elements between tokens
  int nh, nkv, hd, rot;
  const float *bias, *q_norm, *k_norm;
  float eps;
  const float *cos_t, *sin_t;
  int64_t max_pos;
  const int* pos;
  void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  int lanes;  // lanes of a group (a power of two)
};

constexpr int kRopeThreads = 256;

// Channels of run r (0 or 1) of item i, and whether the item is rotated: the
// rotated channels come first, then the rest in two halves.
template <int VEC, bool INTER>
FRC_DEVICE_INLINE bool rope_item(int i, int hd, int rot, int& a, int& b) {
  const int n_rot = rot / (2 * VEC);
  if (i < n_rot) {
    a = INTER ? 2 * VEC * i : VEC * i;
    b = INTER ? a + VEC : a + rot / 2;
    return true;
  }
  a = rot + VEC * (i - n_rot);
  b = a + (hd - rot) / 2;
  return false;
}

// VEC channels a run (4: vector loads; 1: any alignment and any even sizes,
// where interleaved pairs need both channels of a pair in the two runs), NI
// items a lane.
template <typename TI, typename TO, int VEC, int NI, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(RopeParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" :::);
  constexpr bool V = VEC > 1;
  const int64_t tok = blockIdx.x;
  const int pos = p.pos[tok];
  if (pos < 0 || pos >= p.max_pos) return;  // a padding row: its outputs stay as they are
  const int L = p.lanes, li = threadIdx.x & (L - 1);
  const int groups = kRopeThreads / L;
  const int n_items = p.hd / (2 * VEC);

  int a[NI], b[NI];
  bool rotated[NI], on[NI];
  float c[NI][VEC], s[NI][VEC];  // half: of the VEC pairs; interleaved: of the VEC / 2 + VEC / 2 pairs of both runs
#pragma unroll
  for (int u = 0; u < NI; ++u) {
    const int i = li + u * L;
    on[u] = i < n_items;
    rotated[u] = rope_item<VEC, INTER>(i, p.hd, p.rot, a[u], b[u]) && on[u];
    if (rotated[u]) {
      const int64_t row = static_cast<int64_t>(pos) * (p.rot / 2) + static_cast<int64_t>(VEC) * i;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        c[u][e] = p.cos_t[row + e];
        s[u][e] = p.sin_t[row + e];
      }
    }
  }
  const TI* row = static_cast<const TI*>(p.qkv) + tok * p.row_stride;
  const int heads = p.nh + 2 * p.nkv;
  for (int h = blockIdx.y * groups + threadIdx.x / L; h < heads; h += gridDim.y * groups) {
    const bool is_q = h < p.nh, is_k = !is_q && h < p.nh + p.nkv;
    TO* out = is_q   ? static_cast<TO*>(p.q) + tok * p.q_stride + h * p.hd
              : is_k ? static_cast<TO*>(p.k) + tok * p.k_stride + (h - p.nh) * p.hd
                     : static_cast<TO*>(p.v) + tok * p.v_stride + (h - p.nh - p.nkv) * p.hd;
    float x[NI][VEC], y[NI][VEC];
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      if (!on[u]) continue;
      load_run<VEC, V>(row + h * p.hd + a[u], x[u]);
      load_run<VEC, V>(row + h * p.hd + b[u], y[u]);
      if (p.bias) {
        float t[VEC];
        load_run<VEC, V>(p.bias + h * p.hd + a[u], t);
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[u][e] += t[e];
        load_run<VEC, V>(p.bias + h * p.hd + b[u], t);
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[u][e] += t[e];
      }
    }
    const float* w = is_q ? p.q_norm : (is_k ? p.k_norm : nullptr);
    if (w) {
      float ss = 0.f;
#pragma unroll
      for (int u = 0; u < NI; ++u)
        if (on[u]) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) ss = fmaf(x[u][e], x[u][e], fmaf(y[u][e], y[u][e], ss));
        }
      // the group's lanes only: groups of one warp may walk a different number of heads
      const uint32_t mask = (L == 32 ? 0xffffffffu : ((1u << L) - 1u)) << (threadIdx.x & 31 & ~(L - 1));
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      const float inv = 1.0f / sqrtf(ss / static_cast<float>(p.hd) + p.eps);
#pragma unroll
      for (int u = 0; u < NI; ++u) {
        if (!on[u]) continue;
        float t[VEC];
        load_run<VEC, V>(w + a[u], t);
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[u][e] = (x[u][e] * inv) * t[e];
        load_run<VEC, V>(w + b[u], t);
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[u][e] = (y[u][e] * inv) * t[e];
      }
    }
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      if (!on[u]) continue;
      if (rotated[u] && (is_q || is_k)) {
        if constexpr (INTER && VEC > 1) {
#pragma unroll
          for (int e = 0; e < VEC; e += 2) {
            const float x0 = x[u][e], x1 = x[u][e + 1], y0 = y[u][e], y1 = y[u][e + 1];
            const float cx = c[u][e / 2], sx = s[u][e / 2], cy = c[u][VEC / 2 + e / 2], sy = s[u][VEC / 2 + e / 2];
            x[u][e] = x0 * cx - x1 * sx;
            x[u][e + 1] = x1 * cx + x0 * sx;
            y[u][e] = y0 * cy - y1 * sy;
            y[u][e + 1] = y1 * cy + y0 * sy;
          }
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float xe = x[u][e], ye = y[u][e];
            x[u][e] = xe * c[u][e] - ye * s[u][e];
            y[u][e] = ye * c[u][e] + xe * s[u][e];
          }
        }
      }
      store_run<VEC, V>(out + a[u], x[u]);
      store_run<VEC, V>(out + b[u], y[u]);
    }
  }
}

template <typename TI, typename TO>
cudaError_t launch_rope(const RopeParams& p, int64_t tokens, bool inter, bool vec, cudaStream_t st) {
  const int items = p.hd / (vec ? 8 : 2);
  RopeParams q = p;
  q.lanes = 1;
  while (q.lanes < items && q.lanes < 32) q.lanes *= 2;
  const int groups = kRopeThreads / q.lanes, heads = p.nh + 2 * p.nkv;
  // few tokens: a head for each group; many: a block walks over a token's
  // heads and the tables are read once.  Walking against not, 64 + 2 * 8 heads of 128,
  // fp32 to bf16: 5.7 / 4.8 us for 256 tokens, 7.1 / 8.0 for 512, 11.1 / 11.1 for 768,
  // 12.3 / 14.5 for 1024, 25.0 / 29.2 for 2048; 28 + 2 * 4 heads 3.9 / 3.6, 4.7 / 5.3,
  // 6.9 / 6.9, 7.6 / 8.5, 11.9 / 15.4; bf16 rows the same way
  int gy = (heads + groups - 1) / groups;
  if (tokens >= 1024) gy = 1;
  const dim3 grid(static_cast<unsigned>(tokens), static_cast<unsigned>(gy));
  if (vec)
    return inter ? launch_pdl(qk_norm_rope_kernel<TI, TO, 4, 1, true>, grid, dim3(kRopeThreads), 0, st, q)
                 : launch_pdl(qk_norm_rope_kernel<TI, TO, 4, 1, false>, grid, dim3(kRopeThreads), 0, st, q);
  return inter ? launch_pdl(qk_norm_rope_kernel<TI, TO, 1, 4, true>, grid, dim3(kRopeThreads), 0, st, q)
               : launch_pdl(qk_norm_rope_kernel<TI, TO, 1, 4, false>, grid, dim3(kRopeThreads), 0, st, q);
}

}  // namespace frc

extern "C" int frc_qk_norm_rope(int in_type, int out_type, const void* qkv, int64_t row_stride, int64_t tokens, int nh,
                                int nkv, int hd, const float* bias, const float* q_norm, const float* k_norm,
                                float eps, const float* cos_table, const float* sin_table, int64_t max_pos, int rot,
                                int interleaved, const int* pos_dev, void* q_out, int64_t q_stride, void* k_out,
                                int64_t k_stride, void* v_out, int64_t v_stride, void* stream) {
  FRC_REQUIRE(frc_is_float_type(in_type) && frc_is_float_type(out_type),
              "frc_qk_norm_rope: types must be FRC_F32, FRC_F16 or FRC_BF16");
  FRC_REQUIRE(tokens >= 0 && tokens <= 0x7fffffff && nh > 0 && nkv > 0 && nh <= 65535 && nkv <= 65535,
              "frc_qk_norm_rope: bad tokens or heads");
  FRC_REQUIRE(hd > 0 && hd <= 256 && hd % 2 == 0, "frc_qk_norm_rope: head_dim must be even and at most 256");
  FRC_REQUIRE(rot >= 0 && rot <= hd && rot % 2 == 0, "frc_qk_norm_rope: rot must be even and at most head_dim");
  const int64_t nq = static_cast<int64_t>(nh) * hd, nk = static_cast<int64_t>(nkv) * hd;
  FRC_REQUIRE(row_stride >= nq + 2 * nk && q_stride >= nq && k_stride >= nk && v_stride >= nk,
              "frc_qk_norm_rope: a row stride is shorter than its row");
  FRC_REQUIRE(max_pos > 0 && max_pos <= 0x7fffffff, "frc_qk_norm_rope: bad max_pos");
  if (tokens == 0) return FRC_OK;
  FRC_REQUIRE(qkv && pos_dev && q_out && k_out && v_out && (rot == 0 || (cos_table && sin_table)),
              "frc_qk_norm_rope: null pointer");
  const size_t is = in_type == FRC_F32 ? 4 : 2, os = out_type == FRC_F32 ? 4 : 2;
  // outputs apart from everything, or all in the places of their inputs
  const frc::View q_rows(q_out, os, tokens, q_stride, 1, 0, nq), k_rows(k_out, os, tokens, k_stride, 1, 0, nk),
      v_rows(v_out, os, tokens, v_stride, 1, 0, nk), rows(qkv, is, tokens, row_stride, 1, 0, nq + 2 * nk);
  FRC_REQUIRE(!frc::views_share(q_rows, k_rows) && !frc::views_share(q_rows, v_rows) && !frc::views_share(k_rows, v_rows),
              "frc_qk_norm_rope: the outputs share memory");
  const char* in = static_cast<const char*>(qkv);
  const bool in_place = in_type == out_type && q_out == in && k_out == in + nq * is && v_out == in + (nq + nk) * is &&
                        (tokens == 1 || (q_stride == row_stride && k_stride == row_stride && v_stride == row_stride));
  FRC_REQUIRE(in_place || !(frc::views_share(q_rows, rows) || frc::views_share(k_rows, rows) || frc::views_share(v_rows, rows)),
              "frc_qk_norm_rope: an output shares memory with qkv, but not all three in the places of their inputs");
  // four channels a load: every run starts at a multiple of four channels
  const bool vec = hd % 8 == 0 && rot % 8 == 0 && row_stride % 4 == 0 && q_stride % 4 == 0 && k_stride % 4 == 0 &&
                   v_stride % 4 == 0 && frc::aligned_to(qkv, 4 * is) && frc::aligned_to(q_out, 4 * os) &&
                   frc::aligned_to(k_out, 4 * os) && frc::aligned_to(v_out, 4 * os) && frc::aligned_to(bias, 16) &&
                   frc::aligned_to(q_norm, 16) && frc::aligned_to(k_norm, 16);
  const frc::RopeParams p{qkv,  row_stride, nh,        nkv,       hd,      rot,     bias,  q_norm, k_norm,   eps,
                          cos_table, sin_table, max_pos, pos_dev, q_out, k_out, v_out, q_stride, k_stride, v_stride, 0};
  return frc_with_type(in_type, [&](auto* ti) {
    return frc_with_type(out_type, [&](auto* to) -> int {
      using TI = std::remove_pointer_t<decltype(ti)>;
      using TO = std::remove_pointer_t<decltype(to)>;
      FRC_LAUNCHED((frc::launch_rope<TI, TO>(p, tokens, interleaved != 0, vec, static_cast<cudaStream_t>(stream))),
                   "qk_norm_rope launch");
      return FRC_OK;
    });
  });
}
