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
//
// Measured on a B200: 20,495 tokens of 64 heads of 64, bf16, half rotated: 80 us, 4.2 TB/s, 0.64 of a plain copy (about 85
// instructions per 16 bytes, with the products in packed pairs, take 69 % of the issue slots; 64 registers, of which the
// 16-bit forms spill 8 to 64 bytes, hold eight blocks to an SM); 512 tokens of 72 heads of 128: 10 us; one token: 6 us.
// 128-thread blocks took 0.95 of the time of 256-thread blocks, and 0.61 of that with cosines and weights held in
// registers for all heads (98 registers, two blocks to an SM).
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
  int pos64, weight_f32, norm;
  float eps;
  int side, turns_in_row;      // tokens side by side in a block, and one after another
  int slots_per_token;         // rows of a token side by side
  int rows_per_block;
};

constexpr int kRopeThreads = 128;
constexpr int kRopeFlight = 4;      // rows of one thread whose loads are in flight together

// two fp32 operations in one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// A thread's place in its sequence of rows: token after token, `per_token` rows of each.
struct RopePlace {
  int i;                       // row of the token, in turns
  int turn;                    // token of the block, in turns
  int b, t;
  int64_t q, k;                // offsets of token (b, t)
};

template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads, 8) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int EPL = ElemTraits<T>::EPL, P = EPL / 2;
  constexpr int LPR = D / EPL;
  extern __shared__ float s_rope[];                  // [2][D] weights, [side * turns_in_row][half] cosine, sine
  float2* const s_turn = reinterpret_cast<float2*>(s_rope + 2 * D);
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  const int tok = slot / a.slots_per_token, place = slot % a.slots_per_token;
  const int per_block = a.side * a.turns_in_row;     // tokens of this block
  const int64_t n_tok = (int64_t)a.batch * a.tokens, bt0 = (int64_t)blockIdx.x * per_block;
  const int first = blockIdx.y * a.rows_per_block, last = min(first + a.rows_per_block, a.heads[0] + a.heads[1]);
  const int per_token = (last - first + a.slots_per_token - 1) / a.slots_per_token;     // rows of a thread in a token
  const int e0 = lane * EPL;
  // turns of this thread's that are tokens
  const int turns = tok < a.side && bt0 + tok < n_tok
                        ? (int)min((int64_t)a.turns_in_row, (n_tok - bt0 - tok + a.side - 1) / a.side) : 0;

  const auto offsets = [&](RopePlace& at, const int64_t (&strides)[2][3]) {
    at.q = at.b * strides[0][0] + at.t * strides[0][2] + e0;
    at.k = at.b * strides[1][0] + at.t * strides[1][2] + e0;
  };
  const auto begin = [&](const int64_t (&strides)[2][3]) {
    RopePlace at;
    at.i = at.turn = 0;
    at.b = (int)((unsigned)(bt0 + tok) / (unsigned)a.tokens);
    at.t = (int)(bt0 + tok - (int64_t)at.b * a.tokens);
    offsets(at, strides);
    return at;
  };
  const auto step = [&](RopePlace& at, const int64_t (&strides)[2][3]) {
    if (++at.i == per_token) {
      at.i = 0;
      ++at.turn;
      for (at.t += a.side; at.t >= a.tokens; at.t -= a.tokens) ++at.b;
      offsets(at, strides);
    }
  };
  const auto load = [&](const RopePlace& at) -> uint4 {
    const int r = first + place + at.i * a.slots_per_token, w = r >= a.heads[0];
    if (at.turn >= turns || r >= last) return make_uint4(0, 0, 0, 0);
    const T* const x = w ? static_cast<const T*>(a.x[1]) + at.k + (r - a.heads[0]) * a.xs[1][1]
                         : static_cast<const T*>(a.x[0]) + at.q + r * a.xs[0][1];
    return __ldcs(reinterpret_cast<const uint4*>(x));
  };
  // the first rows are on their way while the angles are computed
  uint4 raw[kRopeFlight];
  RopePlace ahead = begin(a.xs);
#pragma unroll
  for (int i = 0; i < kRopeFlight; ++i) {
    raw[i] = load(ahead);
    step(ahead, a.xs);
  }
  for (int i = threadIdx.x; i < per_block * a.half; i += kRopeThreads) {
    const unsigned in_block = (unsigned)i / (unsigned)a.half;
    const int64_t at = bt0 + in_block;
    if (at < n_tok) {
      const unsigned b = (unsigned)at / (unsigned)a.tokens, t = (unsigned)at - b * a.tokens;
      const int64_t off = b * a.ps_b + t * a.ps_t;
      const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.positions)[off]
                                 : (double)static_cast<const int32_t*>(a.positions)[off];
      const double circles = pos * (double)a.inv_freq[i - in_block * a.half] * 0.15915494309189533577;   // 1 / (2 pi)
      float2 cs;
      sincospif(2.f * (float)(circles - rint(circles)), &cs.y, &cs.x);
      s_turn[i] = cs;
    }
  }
  for (int i = threadIdx.x; i < 2 * D; i += kRopeThreads) {
    const void* const w = a.weight[i / D];
    s_rope[i] = !w ? 1.f : a.weight_f32 ? static_cast<const float*>(w)[i % D] : to_float<T>(static_cast<const T*>(w)[i % D]);
  }
  const bool turned = e0 < 2 * a.half;                       // a lane is rotated as a whole or not at all
  const bool upper = !INTERLEAVED && e0 >= a.half;
  const int pair0 = INTERLEAVED ? e0 / 2 : (upper ? e0 - a.half : e0);
  const int warp_lane = threadIdx.x & 31;
  const int partner = !turned ? warp_lane : upper ? warp_lane - a.half / EPL : warp_lane + a.half / EPL;
  __syncthreads();

  float2 co[P], si[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    co[j] = make_float2(1.f, 1.f);
    si[j] = make_float2(0.f, 0.f);
  }
  RopePlace at = begin(a.ys);
  for (int done = 0; done < a.turns_in_row * per_token; done += kRopeFlight) {
#pragma unroll
    for (int i = 0; i < kRopeFlight; ++i) {
      if (done + i >= a.turns_in_row * per_token) break;     // uniform over the block
      if (at.i == 0 && turned && at.turn < turns) {          // a new token: y_a' = y_a cos - y_b sin; y_b' = y_b cos + y_a sin
        const float2* const cs = s_turn + (at.turn * a.side + tok) * a.half + pair0;
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const float2 c = cs[INTERLEAVED ? j : 2 * j], d = INTERLEAVED ? c : cs[2 * j + 1];
          co[j] = make_float2(c.x, d.x);
          si[j] = INTERLEAVED ? make_float2(-c.y, c.y) : upper ? make_float2(c.y, d.y) : make_float2(-c.y, -d.y);
        }
      }
      const int r = first + place + at.i * a.slots_per_token, w = r >= a.heads[0];
      float f[EPL];
      unpack<T>(raw[i], f);
      float2 x[P];
      float2 sq = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        x[j] = make_float2(f[2 * j], f[2 * j + 1]);
        sq = fma2(x[j], x[j], sq);
      }
      if (a.norm) {
        const float scale = rsqrtf(row_sum<LPR>(sq.x + sq.y) * (1.f / D) + a.eps);
        const float2* const weight = reinterpret_cast<const float2*>(s_rope + w * D + e0);
#pragma unroll
        for (int j = 0; j < P; ++j) x[j] = mul2(mul2(x[j], make_float2(scale, scale)), weight[j]);
      }
      float2 other[P];
#pragma unroll
      for (int j = 0; j < P; ++j)
        other[j] = INTERLEAVED ? make_float2(x[j].y, x[j].x)
                               : make_float2(__shfl_sync(0xffffffffu, x[j].x, partner), __shfl_sync(0xffffffffu, x[j].y, partner));
      if (turned) {                                          // an infinity outside the rotated part stays what it is
#pragma unroll
        for (int j = 0; j < P; ++j) x[j] = fma2(x[j], co[j], mul2(other[j], si[j]));
      }
      if (at.turn < turns && r < last) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
          f[2 * j] = x[j].x;
          f[2 * j + 1] = x[j].y;
        }
        T* const y = w ? static_cast<T*>(a.y[1]) + at.k + (r - a.heads[0]) * a.ys[1][1]
                       : static_cast<T*>(a.y[0]) + at.q + r * a.ys[0][1];
        *reinterpret_cast<uint4*>(y) = pack<T>(f);
      }
      raw[i] = load(ahead);
      step(ahead, a.xs);
      step(at, a.ys);
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
  a.norm = norm;
  a.eps = eps;
  const int slots = kRopeThreads / (int)(head_dim * esz / 16);       // rows that a block handles side by side
  const int all = q_heads + kv_heads;
  const int64_t n_tok = (int64_t)batch * tokens;
  if (n_tok > 0x7fffffff) return EKV_ERR_ARG;
  // few heads: several tokens side by side.  Many: one token's rows take several turns.
  a.side = all >= slots ? 1 : slots / all;
  a.slots_per_token = slots / a.side;
  const int64_t want = 8 * sm_count();               // blocks that the GPU holds at a time
  const int64_t sides = (n_tok + a.side - 1) / a.side;
  // few tokens: the rows of a token are spread over blocks (a decode step is latency); many: a block takes several
  // tokens, whose angles it then computes side by side
  const int64_t turns = (all + a.slots_per_token - 1) / a.slots_per_token;
  int64_t parts = want / sides > 1 ? want / sides : 1;
  if (parts > turns) parts = turns;
  a.rows_per_block = (int)((turns + parts - 1) / parts) * a.slots_per_token;
  parts = (all + a.rows_per_block - 1) / a.rows_per_block;
  int64_t in_row = sides / (4 * want);
  in_row = in_row < 1 ? 1 : (in_row > 8 ? 8 : in_row);
  a.turns_in_row = (int)in_row;
  const int64_t blocks = (sides + in_row - 1) / in_row;
  if (blocks > 0x7fffffff || parts > 65535) return EKV_ERR_ARG;
  const size_t smem = sizeof(float2) * ((size_t)(a.side * in_row) * half + head_dim);
  EKV_DISPATCH(dtype, head_dim, {
    const dim3 grid((unsigned)blocks, (unsigned)parts);
    if (interleaved) qk_norm_rope_kernel<T, D, true><<<grid, kRopeThreads, smem, as_stream(stream)>>>(a);
    else qk_norm_rope_kernel<T, D, false><<<grid, kRopeThreads, smem, as_stream(stream)>>>(a);
  });
  return launch_status();
}
