// RMS norm of every query and key head with the position rotation in the same pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w          (one head vector of D elements)
//   (a, b) -> (a cos - b sin, b cos + a sin)     for the first 2 * half elements of y, angle = position * inv_freq[j]
//
// with (a, b) = (y_j, y_{j+half}) or, interleaved, (y_{2j}, y_{2j+1}).  Everything in fp32, one rounding at the store.
// The angle is a 64-bit product reduced to a fraction of a turn before the fp32 sine: at position 10^6 the fp32 product
// alone would be off by 0.06 rad.
//
// Bound by memory (each element read and written once).  A row of D elements is covered by LPR lanes of 16 bytes; a
// thread keeps its lane of the row for every head that it visits, so the cosines, sines and weights of its eight (four)
// elements are loaded once and stay in registers, and the angles of a token are computed once per block.
#include "ekv_common.cuh"

namespace ekv {

struct RopeArgs {
  const void* x[2];            // q, k
  void* y[2];
  const void* weight[2];       // [D] or null
  int64_t xs[2][3], ys[2][3];  // element strides: batch, head, token
  int heads[2];
  const void* positions;       // int32 or int64
  int64_t ps_b, ps_t;
  const float* inv_freq;
  int batch, tokens, half;
  int pos64, weight_f32, interleaved, norm;
  float eps;
  int tokens_per_block, slots_per_token, rows_per_block;   // see rope_launch
};

constexpr int kRopeThreads = 256;
constexpr int kRopeFlight = 4;      // rows of one thread whose loads are in flight together

template <typename T, int D>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int EPL = ElemTraits<T>::EPL;
  constexpr int LPR = D / EPL;
  extern __shared__ float2 s_turn[];                 // [tokens_per_block][half]: cosine, sine
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  const int tok = slot / a.slots_per_token;          // token of this block
  const int64_t n_tok = (int64_t)a.batch * a.tokens;
  const int64_t bt = (int64_t)blockIdx.x * a.tokens_per_block + tok;
  const bool live = tok < a.tokens_per_block && bt < n_tok;
  const int b = live ? (int)(bt / a.tokens) : 0, t = live ? (int)(bt % a.tokens) : 0;
  const int all = a.heads[0] + a.heads[1];
  const int first = blockIdx.y * a.rows_per_block, last = min(first + a.rows_per_block, all);
  const int e0 = lane * EPL;

  auto row_in = [&](int r) -> const uint4* {
    const int w = r >= a.heads[0];
    const int h = r - (w ? a.heads[0] : 0);
    return reinterpret_cast<const uint4*>(static_cast<const T*>(a.x[w]) + b * a.xs[w][0] + h * a.xs[w][1] +
                                          t * a.xs[w][2] + e0);
  };
  // the first rows are on their way while the angles are computed
  uint4 raw[kRopeFlight];
  const int r0 = first + slot % a.slots_per_token;
#pragma unroll
  for (int i = 0; i < kRopeFlight; ++i) {
    const int r = r0 + i * a.slots_per_token;
    raw[i] = live && r < last ? __ldcs(row_in(r)) : make_uint4(0, 0, 0, 0);
  }

  for (int i = threadIdx.x; i < a.tokens_per_block * a.half; i += kRopeThreads) {
    const int64_t at = (int64_t)blockIdx.x * a.tokens_per_block + i / a.half;
    if (at < n_tok) {
      const int64_t off = at / a.tokens * a.ps_b + at % a.tokens * a.ps_t;
      const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.positions)[off]
                                 : (double)static_cast<const int32_t*>(a.positions)[off];
      const double turns = pos * (double)a.inv_freq[i % a.half] * 0.15915494309189533577;   // 1 / (2 pi)
      float2 cs;
      sincospif(2.f * (float)(turns - rint(turns)), &cs.y, &cs.x);
      s_turn[i] = cs;
    }
  }
  __syncthreads();

  const bool turned = e0 < 2 * a.half;                       // a lane is rotated as a whole or not at all
  const bool upper = !a.interleaved && e0 >= a.half;
  float co[EPL], si[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    co[j] = 1.f;
    si[j] = 0.f;
    if (turned && live) {
      const int p = a.interleaved ? (e0 + j) / 2 : (upper ? e0 + j - a.half : e0 + j);
      const float2 cs = s_turn[tok * a.half + p];
      co[j] = cs.x;
      // y_a' = y_a cos - y_b sin;  y_b' = y_b cos + y_a sin
      si[j] = a.interleaved ? (j & 1 ? cs.y : -cs.y) : (upper ? cs.y : -cs.y);
    }
  }
  float w[2][EPL];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      w[which][j] = !a.weight[which] ? 1.f
                    : a.weight_f32   ? static_cast<const float*>(a.weight[which])[e0 + j]
                                     : to_float<T>(static_cast<const T*>(a.weight[which])[e0 + j]);
    }
  }
  const int warp_lane = threadIdx.x & 31;
  const int partner = a.interleaved || !turned ? warp_lane
                      : upper                  ? warp_lane - a.half / EPL
                                               : warp_lane + a.half / EPL;

  for (int base = first; base < last; base += kRopeFlight * a.slots_per_token) {
#pragma unroll
    for (int i = 0; i < kRopeFlight; ++i) {
      if (base + i * a.slots_per_token >= last) break;       // uniform over the block
      const int r = base + slot % a.slots_per_token + i * a.slots_per_token;
      const int which = r >= a.heads[0];
      float x[EPL];
      unpack<T>(raw[i], x);
      float scale = 1.f;
      if (a.norm) {
        float sq = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) sq = fmaf(x[j], x[j], sq);
        sq = row_sum<LPR>(sq);
        scale = 1.f / sqrtf(sq * (1.f / D) + a.eps);
      }
      float other[EPL];
#pragma unroll
      for (int j = 0; j < EPL; ++j) x[j] = x[j] * scale * (which ? w[1][j] : w[0][j]);
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) other[j] = x[j ^ 1];
      } else {
#pragma unroll
        for (int j = 0; j < EPL; ++j) other[j] = __shfl_sync(0xffffffffu, x[j], partner);
      }
      if (!turned) {                                         // an infinity outside the rotated part stays what it is
#pragma unroll
        for (int j = 0; j < EPL; ++j) other[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) x[j] = fmaf(x[j], co[j], other[j] * si[j]);
      if (live && r < last) {
        const int h = r - (which ? a.heads[0] : 0);
        *reinterpret_cast<uint4*>(static_cast<T*>(a.y[which]) + b * a.ys[which][0] + h * a.ys[which][1] +
                                  t * a.ys[which][2] + e0) = pack<T>(x);
      }
      const int next = r + kRopeFlight * a.slots_per_token;
      if (live && next < last) raw[i] = __ldcs(row_in(next));
    }
  }
}

}  // namespace ekv

extern "C" int ekv_qk_norm_rope(int32_t dtype, int32_t batch, int32_t tokens, int32_t q_heads, int32_t kv_heads,
                                int32_t head_dim, const void* q, const int64_t* q_strides, const void* k,
                                const int64_t* k_strides, void* q_out, const int64_t* q_out_strides, void* k_out,
                                const int64_t* k_out_strides, const void* positions, int32_t positions_64,
                                int64_t pos_stride_b, int64_t pos_stride_t, const float* inv_freq, int32_t half,
                                int32_t interleaved, const void* q_weight, const void* k_weight, int32_t weight_f32,
                                int32_t norm, float eps, void* stream) {
  using namespace ekv;
  if (dtype < EKV_F16 || dtype > EKV_F32 || (head_dim != 64 && head_dim != 128)) return EKV_ERR_DTYPE;
  if (batch < 0 || tokens < 0 || q_heads <= 0 || kv_heads < 0 || half < 0 || half % 8 || 2 * half > head_dim)
    return EKV_ERR_ARG;
  if (batch == 0 || tokens == 0) return EKV_OK;
  if (!positions || (half && !inv_freq) || (norm && !(eps >= 0.f))) return EKV_ERR_ARG;
  const int64_t esz = dtype == EKV_F32 ? 4 : 2;
  RopeArgs a{};
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const int64_t* is[2] = {q_strides, k_strides};
  const int64_t* os[2] = {q_out_strides, k_out_strides};
  for (int w = 0; w < 2; ++w) {
    a.heads[w] = w ? kv_heads : q_heads;
    if (!a.heads[w]) continue;
    if (!in[w] || !out[w] || !is[w] || !os[w]) return EKV_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(in[w]) | reinterpret_cast<uintptr_t>(out[w])) & 15) return EKV_ERR_ARG;
    a.x[w] = in[w];
    a.y[w] = out[w];
    for (int i = 0; i < 3; ++i) {
      if ((is[w][i] * esz) % 16 || (os[w][i] * esz) % 16) return EKV_ERR_ARG;
      a.xs[w][i] = is[w][i];
      a.ys[w][i] = os[w][i];
    }
  }
  a.weight[0] = norm ? q_weight : nullptr;
  a.weight[1] = norm ? k_weight : nullptr;
  a.positions = positions;
  a.ps_b = pos_stride_b;
  a.ps_t = pos_stride_t;
  a.inv_freq = inv_freq;
  a.batch = batch;
  a.tokens = tokens;
  a.half = half;
  a.pos64 = positions_64;
  a.weight_f32 = weight_f32;
  a.interleaved = interleaved;
  a.norm = norm;
  a.eps = eps;
  const int slots = kRopeThreads / (int)(head_dim * esz / 16);       // rows that a block handles side by side
  const int all = q_heads + kv_heads;
  const int64_t n_tok = (int64_t)batch * tokens;
  // few heads: several tokens share a block.  Many: one token's rows take several turns.
  a.tokens_per_block = all >= slots ? 1 : slots / all;
  a.slots_per_token = slots / a.tokens_per_block;
  // few tokens: the rows of a token are spread over blocks, one turn each (a decode step is latency)
  const int64_t blocks = (n_tok + a.tokens_per_block - 1) / a.tokens_per_block;
  a.rows_per_block = blocks >= 2 * sm_count() ? all : a.slots_per_token;
  const int parts = (all + a.rows_per_block - 1) / a.rows_per_block;
  if (blocks > 0x7fffffff || parts > 65535) return EKV_ERR_ARG;
  const size_t smem = sizeof(float2) * (size_t)a.tokens_per_block * half;
  EKV_DISPATCH(dtype, head_dim, {
    qk_norm_rope_kernel<T, D><<<dim3((unsigned)blocks, (unsigned)parts), kRopeThreads, smem, as_stream(stream)>>>(a);
  });
  return launch_status();
}
