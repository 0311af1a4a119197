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
// thread keeps its lane of the row for every head and token that it visits, so the weights of its eight (four) elements
// stay in registers, the cosines and sines are read once per token, and four rows are on their way while one is worked
// on.  A block takes several tokens, whose angles it computes first.
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
  int side, turns_in_row;      // tokens side by side in a block, and one after another
  int slots_per_token;         // rows of a token side by side
  int rows_per_block;
};

constexpr int kRopeThreads = 256;
constexpr int kRopeFlight = 4;      // rows of one thread whose loads are in flight together

template <typename T, int D>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int EPL = ElemTraits<T>::EPL;
  constexpr int LPR = D / EPL;
  extern __shared__ float2 s_turn[];                 // [side * turns_in_row][half]: cosine, sine
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  const int tok = slot / a.slots_per_token, place = slot % a.slots_per_token;
  const int per_block = a.side * a.turns_in_row;     // tokens of this block
  const int64_t n_tok = (int64_t)a.batch * a.tokens, bt0 = (int64_t)blockIdx.x * per_block;
  const int all = a.heads[0] + a.heads[1];
  const int first = blockIdx.y * a.rows_per_block, last = min(first + a.rows_per_block, all);
  const int per_token = (last - first + a.slots_per_token - 1) / a.slots_per_token;     // rows of a thread in a token
  const int e0 = lane * EPL;

  // this thread's rows, token after token: a place in that sequence
  struct At {
    int turn, i;
  };
  const auto step = [&](At& at) {
    if (++at.i == per_token) {
      at.i = 0;
      ++at.turn;
    }
  };
  const auto row_of = [&](const At& at) { return first + place + at.i * a.slots_per_token; };
  const auto token_of = [&](const At& at) { return bt0 + at.turn * a.side + tok; };
  const auto live = [&](const At& at) {
    return at.turn < a.turns_in_row && tok < a.side && row_of(at) < last && token_of(at) < n_tok;
  };
  const auto load = [&](const At& at) -> uint4 {
    if (!live(at)) return make_uint4(0, 0, 0, 0);
    const unsigned bt = (unsigned)token_of(at), b = bt / (unsigned)a.tokens, t = bt - b * a.tokens;
    const int r = row_of(at), w = r >= a.heads[0], h = r - (w ? a.heads[0] : 0);
    return __ldcs(reinterpret_cast<const uint4*>(static_cast<const T*>(a.x[w]) + b * a.xs[w][0] + h * a.xs[w][1] +
                                                 t * a.xs[w][2] + e0));
  };
  // the first rows are on their way while the angles are computed
  uint4 raw[kRopeFlight];
  At ahead{0, 0};
#pragma unroll
  for (int i = 0; i < kRopeFlight; ++i) {
    raw[i] = load(ahead);
    step(ahead);
  }
  for (int i = threadIdx.x; i < per_block * a.half; i += kRopeThreads) {
    const int64_t at = bt0 + i / a.half;
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
  const bool turned = e0 < 2 * a.half;                       // a lane is rotated as a whole or not at all
  const bool upper = !a.interleaved && e0 >= a.half;
  const int pair0 = a.interleaved ? e0 / 2 : (upper ? e0 - a.half : e0);
  const int warp_lane = threadIdx.x & 31;
  const int partner = a.interleaved || !turned ? warp_lane
                      : upper                  ? warp_lane - a.half / EPL
                                               : warp_lane + a.half / EPL;
  __syncthreads();

  float co[EPL], si[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    co[j] = 1.f;
    si[j] = 0.f;
  }
  At at{0, 0};
  for (int done = 0; done < a.turns_in_row * per_token; done += kRopeFlight) {
#pragma unroll
    for (int i = 0; i < kRopeFlight; ++i) {
      if (done + i >= a.turns_in_row * per_token) break;     // uniform over the block
      if (at.i == 0 && turned && tok < a.side) {             // a new token: y_a' = y_a cos - y_b sin; y_b' = y_b cos + y_a sin
        const float2* const cs = s_turn + (at.turn * a.side + tok) * a.half + pair0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          const float2 c = cs[a.interleaved ? j / 2 : j];
          co[j] = c.x;
          si[j] = a.interleaved ? (j & 1 ? c.y : -c.y) : (upper ? c.y : -c.y);
        }
      }
      const bool ok = live(at);
      const int r = row_of(at), which = r >= a.heads[0];
      float x[EPL], other[EPL];
      unpack<T>(raw[i], x);
      float scale = 1.f;
      if (a.norm) {
        float sq = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) sq = fmaf(x[j], x[j], sq);
        scale = rsqrtf(row_sum<LPR>(sq) * (1.f / D) + a.eps);
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) x[j] = x[j] * scale * (which ? w[1][j] : w[0][j]);
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) other[j] = x[j ^ 1];
      } else {
#pragma unroll
        for (int j = 0; j < EPL; ++j) other[j] = __shfl_sync(0xffffffffu, x[j], partner);
      }
      if (turned) {                                          // an infinity outside the rotated part stays what it is
#pragma unroll
        for (int j = 0; j < EPL; ++j) x[j] = fmaf(x[j], co[j], other[j] * si[j]);
      }
      if (ok) {
        const unsigned bt = (unsigned)token_of(at), b = bt / (unsigned)a.tokens, t = bt - b * a.tokens;
        const int h = r - (which ? a.heads[0] : 0);
        *reinterpret_cast<uint4*>(static_cast<T*>(a.y[which]) + b * a.ys[which][0] + h * a.ys[which][1] +
                                  t * a.ys[which][2] + e0) = pack<T>(x);
      }
      raw[i] = load(ahead);
      step(ahead);
      step(at);
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
  if (n_tok > 0x7fffffff) return EKV_ERR_ARG;
  // few heads: several tokens side by side.  Many: one token's rows take several turns.
  a.side = all >= slots ? 1 : slots / all;
  a.slots_per_token = slots / a.side;
  const int64_t want = 8 * sm_count();               // blocks that fill the GPU
  const int64_t sides = (n_tok + a.side - 1) / a.side;
  // few tokens: the rows of a token are spread over blocks (a decode step is latency); many: a block takes several
  // tokens, whose angles it then computes side by side
  const int64_t turns = (all + a.slots_per_token - 1) / a.slots_per_token;
  int64_t parts = want / sides > 1 ? want / sides : 1;
  if (parts > turns) parts = turns;
  a.rows_per_block = (int)((turns + parts - 1) / parts) * a.slots_per_token;
  parts = (all + a.rows_per_block - 1) / a.rows_per_block;
  int64_t in_row = sides / (2 * want);
  in_row = in_row < 1 ? 1 : (in_row > 8 ? 8 : in_row);
  a.turns_in_row = (int)in_row;
  const int64_t blocks = (sides + in_row - 1) / in_row;
  if (blocks > 0x7fffffff || parts > 65535) return EKV_ERR_ARG;
  const size_t smem = sizeof(float2) * (size_t)(a.side * in_row) * half;
  EKV_DISPATCH(dtype, head_dim, {
    qk_norm_rope_kernel<T, D><<<dim3((unsigned)blocks, (unsigned)parts), kRopeThreads, smem, as_stream(stream)>>>(a);
  });
  return launch_status();
}
