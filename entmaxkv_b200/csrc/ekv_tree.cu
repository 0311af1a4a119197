// Entmax attention of a tree of drafted tokens over the cache (see ekv_tree.cuh for the method).
#include <cudaTypedefs.h>

#include "ekv_tree_mma.cuh"

namespace ekv {

// ---- scores on the CUDA cores -------------------------------------------------------------------------------------
//
// For fp32 caches, which have no tensor-core product of their precision.  A block scores 32 rows against 64 keys at a
// time: lane = row, warp = eight of the keys, so a key's elements are one broadcast read per warp and each thread owns
// (row, eight keys of every half tile) with a list of its own.
constexpr int kSimtRows = 32, kSimtKeys = 64, kSimtWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kSimtWarps * 32) tree_scores_simt_kernel(const __grid_constant__ TreeArgs a) {
  constexpr int EPL = ElemTraits<T>::EPL, LPR = D / EPL, PITCH = D + 4;
  constexpr int KPW = kSimtKeys / kSimtWarps;
  extern __shared__ float smem[];
  float* const s_q = smem;                              // [32][PITCH]
  float* const s_k = smem + kSimtRows * PITCH;          // [64][PITCH]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int range = blockIdx.x / a.row_blocks, rb = blockIdx.x % a.row_blocks;
  const int H = a.c.kv_heads;
  const TreeSplit split = tree_split(tree_tiles_before(a, a.g1, lane), a.ranges);
  if (split.W == 0 || range >= split.N) return;
  const int64_t t_begin = split.begin(range), t_end = split.begin(range + 1);
  const TreeAt at = tree_find(a, t_begin, lane);
  int64_t g_first = at.first;                           // first tile of the group
  for (int g = at.g; g < a.g1 && g_first < t_end; ++g) {
    const int b = g / H, hkv = g % H;
    const int n = tree_tiles(a, b);
    if (n == 0) continue;
    const int64_t g_end = g_first + n;
    const int tile0 = (int)(max(t_begin, g_first) - g_first), tile1 = (int)(min(t_end, g_end) - g_first);
    const int part = range - split.piece_of(g_first);
    const int len = tree_len(a, b);
    const int live = min(tree_drafts(a, b) * a.group - a.row0, a.rows) - rb * kSimtRows;   // rows of this block
    g_first = g_end;
    if (live <= 0) continue;                            // uniform over the block
    __syncthreads();
    for (int i = tid; i < kSimtRows * LPR; i += kSimtWarps * 32) {
      const int row = i / LPR, e = i % LPR * EPL;
      const int r = a.row0 + rb * kSimtRows + row;
      float x[EPL];
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (row < live)
        raw = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.qs[0] +
                                              (int64_t)(hkv * a.group + r % a.group) * a.qs[1] +
                                              (int64_t)(r / a.group) * a.qs[2] + e);
      unpack<T>(raw, x);
#pragma unroll
      for (int j = 0; j < EPL; ++j) s_q[row * PITCH + e + j] = x[j];
    }
    const int64_t row_id = (int64_t)(g - a.g0) * a.rows + rb * kSimtRows + lane;
    uint2* const list = a.entries + row_id * a.region + (int64_t)tile0 * kTreeTile +
                        (int64_t)warp * (tile1 - tile0) * (kTreeTile / kSimtWarps);
    int count = 0;
    float top = -INFINITY;
    for (int key0 = tile0 * kTreeTile; key0 < min(tile1 * kTreeTile, len); key0 += kSimtKeys) {
      __syncthreads();
      for (int i = tid; i < kSimtKeys * LPR; i += kSimtWarps * 32) {
        const int key = key0 + i / LPR, e = i % LPR * EPL;
        float x[EPL];
        uint4 raw = make_uint4(0, 0, 0, 0);
        size_t off;
        if (key < len) {
          int page, in_page;
          a.by_page.divmod(key, page, in_page);
          if (kv_page_offset(a.c, b, hkv, page, off))
            raw = ld_stream(static_cast<const T*>(a.c.k) + off + (size_t)in_page * D + e);
        }
        unpack<T>(raw, x);
#pragma unroll
        for (int j = 0; j < EPL; ++j) s_k[(i / LPR) * PITCH + e + j] = x[j];
      }
      __syncthreads();
      float acc[KPW] = {};
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        const float4 qv = *reinterpret_cast<const float4*>(s_q + lane * PITCH + d);
#pragma unroll
        for (int j = 0; j < KPW; ++j) {
          const float4 kv = *reinterpret_cast<const float4*>(s_k + (warp * KPW + j) * PITCH + d);
          acc[j] = fmaf(qv.x, kv.x, acc[j]);
          acc[j] = fmaf(qv.y, kv.y, acc[j]);
          acc[j] = fmaf(qv.z, kv.z, acc[j]);
          acc[j] = fmaf(qv.w, kv.w, acc[j]);
        }
      }
      const int valid = len - (key0 + warp * KPW);      // keys of this warp that exist
#pragma unroll
      for (int j = 0; j < KPW; ++j) {
        acc[j] *= a.zscale;
        if (j < valid) top = max_nan(top, acc[j]);
      }
      if (lane < live) {
#pragma unroll
        for (int j = 0; j < KPW; ++j)
          if (j < valid && !(acc[j] <= top - 1.f)) list[count++] = make_uint2(__float_as_uint(acc[j]), key0 + warp * KPW + j);
      }
    }
    if (lane < live) {
      const int64_t at = row_id * a.max_parts * a.sub + part * a.sub + warp;
      a.counts[at] = count;
      a.bounds[at] = top - 1.f;
    }
  }
}

// ---- tau and output ------------------------------------------------------------------------------------------------

constexpr int kFinThreads = 256;
constexpr int kFinSlots = 2048;        // survivors in shared memory; more stay in the row's region
constexpr int kFinPer = 4;             // list entries per thread and round

struct FinRow {
  float* z;                            // [kFinSlots]
  int* key;
  uint2* region;
  __device__ __forceinline__ uint2 get(int i) const {
    return i < kFinSlots ? make_uint2(__float_as_uint(z[i]), (uint32_t)key[i]) : region[i];
  }
  __device__ __forceinline__ void put(int i, uint2 e) const {
    if (i < kFinSlots) {
      z[i] = __uint_as_float(e.x);
      key[i] = (int)e.y;
    } else {
      region[i] = e;
    }
  }
};

__device__ __forceinline__ float3 block_sum3(float3 v, float* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  v.z = warp_sum(v.z);
  __syncthreads();
  if (lane == 0) {
    scratch[warp * 3] = v.x;
    scratch[warp * 3 + 1] = v.y;
    scratch[warp * 3 + 2] = v.z;
  }
  __syncthreads();
  float3 t = make_float3(0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < kFinThreads / 32; ++w) {
    t.x += scratch[w * 3];
    t.y += scratch[w * 3 + 1];
    t.z += scratch[w * 3 + 2];
  }
  return t;
}

// exclusive scan of small counts over the block; also the total
__device__ __forceinline__ int block_excl(int v, int* scratch, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kFinThreads / 32; ++w) {
    if (w < warp) base += scratch[w];
    all += scratch[w];
  }
  *total = all;
  return base + inc - v;
}

template <typename T, int D>
__global__ void __launch_bounds__(kFinThreads) tree_finish_kernel(const __grid_constant__ TreeArgs a) {
  constexpr int EPL = ElemTraits<T>::EPL, LPR = D / EPL, GROUPS = kFinThreads / LPR;
  __shared__ float s_z[kFinSlots];
  __shared__ int s_key[kFinSlots];
  __shared__ float scratch[32];
  __shared__ float s_acc[GROUPS * D];
  extern __shared__ int s_dyn[];                 // [parts * sub + 1] list ends, [tokens] drafted scores
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int H = a.c.kv_heads;
  const int gl = blockIdx.x / a.rows, rl = blockIdx.x % a.rows;
  const int g = a.g0 + gl, r = a.row0 + rl;
  const int b = g / H, hkv = g % H, hq = hkv * a.group + r % a.group, t = r / a.group;
  const int drafts = tree_drafts(a, b);
  if (t >= drafts) return;                       // behind a short tree: left as it was
  const int64_t row_id = (int64_t)gl * a.rows + rl;
  int* const s_end = s_dyn;
  float* const s_zd = reinterpret_cast<float*>(s_dyn + a.max_parts * a.sub + 1);
  const FinRow row{s_z, s_key, a.entries + row_id * a.region};

  // drafted keys: a warp per key
  {
    const T* const qrow = static_cast<const T*>(a.q) + b * a.qs[0] + hq * a.qs[1] + t * a.qs[2];
    const unsigned char* const seen = a.mask + b * a.ms_b + t * a.ms_t;
    for (int j = warp; j < a.tokens; j += kFinThreads / 32) {
      float s = -INFINITY;
      if (j < drafts && seen[j]) {
        const T* const krow = static_cast<const T*>(a.k_draft) + b * a.ks[0] + hkv * a.ks[1] + j * a.ks[2];
        s = 0.f;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) s = fmaf(to_float<T>(qrow[lane + 32 * e]), to_float<T>(krow[lane + 32 * e]), s);
        s = warp_sum(s) * a.zscale;
      }
      if (lane == 0) s_zd[j] = s;
    }
  }
  // the pieces that hold this group's lists
  const int64_t W = tree_tiles_before(a, a.g1, lane), g_first = tree_tiles_before(a, g, lane);
  const int n_tiles = tree_tiles(a, b);
  const TreeSplit split = tree_split(W, a.ranges);
  const int piece0 = n_tiles ? split.piece_of(g_first) : 0;
  const int parts = n_tiles ? split.piece_of(g_first + n_tiles - 1) - piece0 + 1 : 0;
  const int lists = parts * a.sub;
  const int* const counts = a.counts + row_id * a.max_parts * a.sub;
  const float* const bounds = a.bounds + row_id * a.max_parts * a.sub;
  float floor_z = -INFINITY;                     // no weight at or below; fmaxf passes over a NaN
  __syncthreads();                               // s_zd
  for (int i = tid; i < lists; i += kFinThreads) floor_z = fmaxf(floor_z, bounds[i]);
  floor_z = warp_max(floor_z);
  if (lane == 0) scratch[warp] = floor_z;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kFinThreads / 32; ++w) floor_z = fmaxf(floor_z, scratch[w]);

  // ends of the lists in their concatenation
  int raw = 0;
  for (int i0 = 0; i0 < lists; i0 += kFinThreads) {
    int all;
    const int n = i0 + tid < lists ? counts[i0 + tid] : 0;
    const int ex = block_excl(n, reinterpret_cast<int*>(scratch), &all);
    if (i0 + tid < lists) s_end[i0 + tid] = raw + ex + n;
    raw += all;
  }
  __syncthreads();

  // what the largest bound leaves, in order; a NaN stays
  int n = 0;
  float top = -INFINITY;
  for (int i0 = 0; i0 < raw; i0 += kFinThreads * kFinPer) {
    uint2 e[kFinPer];
    int keep = 0, mine = 0;
    int i = i0 + tid * kFinPer;
    if (i < raw) {
      int lo = 0, hi = lists - 1;                // the list that holds entry i
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_end[mid] > i) hi = mid; else lo = mid + 1;
      }
      int l = lo;
#pragma unroll
      for (int j = 0; j < kFinPer; ++j) {
        if (i + j < raw) {
          while (s_end[l] <= i + j) ++l;
          const int p = l / a.sub, s = l % a.sub;
          const int64_t lo_t = max(split.begin(piece0 + p), g_first) - g_first;
          const int64_t hi_t = min(split.begin(piece0 + p + 1), g_first + n_tiles) - g_first;
          const int64_t base = lo_t * kTreeTile + s * (hi_t - lo_t) * (kTreeTile / a.sub);
          e[j] = row.region[base + (i + j - (l ? s_end[l - 1] : 0))];
          if (!(__uint_as_float(e[j].x) <= floor_z)) {
            keep |= 1 << j;
            ++mine;
            top = max_nan(top, __uint_as_float(e[j].x));
          }
        }
      }
    }
    int all;
    int at = n + block_excl(mine, reinterpret_cast<int*>(scratch), &all);
#pragma unroll
    for (int j = 0; j < kFinPer; ++j)
      if (keep >> j & 1) row.put(at++, e[j]);
    n += all;
    __syncthreads();
  }
  for (int j0 = 0; j0 < a.tokens; j0 += kFinThreads) {
    const int j = j0 + tid;
    const bool keep = j < a.tokens && !(s_zd[j] <= floor_z);             // -inf: not seen
    if (keep) top = max_nan(top, s_zd[j]);
    int all;
    const int at = n + block_excl(keep, reinterpret_cast<int*>(scratch), &all);
    if (keep) row.put(at, make_uint2(__float_as_uint(s_zd[j]), ~j));     // a negative key: drafted
    n += all;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  __syncthreads();
  if (lane == 0) scratch[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kFinThreads / 32; ++w) top = max_nan(top, scratch[w]);
  T* const out = static_cast<T*>(a.out) + b * a.os[0] + hq * a.os[1] + t * a.os[2];
  float* const tau_out = a.tau ? a.tau + ((int64_t)b * a.q_heads + hq) * a.tokens + t : nullptr;
  if (!(fabsf(top) < INFINITY)) {                // nothing visible: zeros.  NaN or +inf among the scores: NaN
    const float fill = top == -INFINITY ? 0.f : NAN;
    if (tid < D) out[tid] = from_float<T>(fill);
    if (tid == 0 && tau_out) *tau_out = top == -INFINITY ? INFINITY : NAN;
    return;
  }
  floor_z = fmaxf(floor_z, top - 1.f);

  // tau: the norm N(tau) = (sum (z - tau)_+^beta)^(1/beta) falls to 1 at the root and is convex for beta >= 1 (nearly
  // linear when the support is settled), so Newton's steps on it from max - 1 climb towards the root from the left;
  // the bracket keeps them safe for beta < 1.
  const float beta = 1.f / (a.alpha - 1.f);
  const int kind = alpha_kind_of(a.alpha);
  float lo = floor_z, hi = top, tau = floor_z;
  for (int it = 0; it < 40; ++it) {
    float3 s = make_float3(0.f, 0.f, 0.f);
    for (int i = tid; i < n; i += kFinThreads)
      halley_accumulate(__uint_as_float(row.get(i).x), tau, kind, beta, s.x, s.y, s.z);
    s = block_sum3(s, scratch);
    if (s.x >= 1.f) lo = tau; else hi = tau;
    // N - 1 over -N' = (s0^(1/beta) - 1) s0^(1 - 1/beta) / s1
    const float root = kind == 0 ? s.x : (kind == 1 ? sqrtf(s.x) : pow_pos(s.x, a.alpha - 1.f));
    const float step = s.x > 0.f ? (root - 1.f) * (s.x / root) / s.y : -INFINITY;
    // half a unit in the last place of the scores that tau is compared with
    const bool done = fabsf(step) <= 6e-8f * fmaxf(fabsf(tau), fabsf(top));
    const float next = tau + step;
    tau = next > lo && next < hi ? next : (done ? tau : 0.5f * (lo + hi));
    if (done) break;
  }

  // the support, in order: weight and key
  int m = 0;
  for (int i0 = 0; i0 < n; i0 += kFinThreads) {
    const int i = i0 + tid;
    uint2 e = make_uint2(0, 0);
    float w = 0.f;
    if (i < n) {
      e = row.get(i);
      w = entmax_weight(__uint_as_float(e.x), tau, kind, beta);
    }
    int all;
    const int at = m + block_excl(w > 0.f, reinterpret_cast<int*>(scratch), &all);
    if (w > 0.f) row.put(at, make_uint2(__float_as_uint(w), e.y));
    m += all;
  }
  __syncthreads();

  float acc[EPL] = {};
  const int sub = tid / LPR, col = tid % LPR * EPL;
#pragma unroll 4
  for (int i = sub; i < m; i += GROUPS) {
    const uint2 e = row.get(i);
    const float w = __uint_as_float(e.x);
    const int key = (int)e.y;
    const T* v;
    bool ok = true;
    if (key < 0) {
      v = static_cast<const T*>(a.v_draft) + b * a.vs[0] + hkv * a.vs[1] + (int64_t)~key * a.vs[2];
    } else {
      int page, in_page;
      size_t off;
      a.by_page.divmod(key, page, in_page);
      ok = kv_page_offset(a.c, b, hkv, page, off);
      v = static_cast<const T*>(a.c.v) + off + (size_t)in_page * D;
    }
    float x[EPL];
    unpack<T>(ok ? *reinterpret_cast<const uint4*>(v + col) : make_uint4(0, 0, 0, 0), x);
#pragma unroll
    for (int j = 0; j < EPL; ++j) acc[j] = fmaf(w, x[j], acc[j]);
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) s_acc[sub * D + col + j] = acc[j];
  __syncthreads();
  if (tid < D) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) s += s_acc[i * D + tid];
    out[tid] = from_float<T>(s);
  }
  if (tid == 0 && tau_out) *tau_out = tau;
}

// ---- host ----------------------------------------------------------------------------------------------------------

struct TreePlan {
  int64_t region;        // entries per row
  int tiles, rows, sub, row_blocks, ranges, tile_keys;
  int64_t row_bytes;     // workspace per row
  int max_parts;
  bool mma, sample;      // tensor cores; a sample before the pass
  int sample_tiles;
  TmShape shape;
};

constexpr int kSampleFrom = 8;         // tiles per block from which on there is a sample

static TreePlan tree_plan(const ekv_cache_desc* c, int q_heads, int tokens, int max_seq) {
  TreePlan p{};
  p.rows = tokens * (q_heads / c->kv_heads);
  p.mma = c->dtype != EKV_F32;
  p.tile_keys = kTreeTile;
  if (p.mma) {
    TmShape& sh = p.shape;
    const int blocks = (p.rows + kTmMaxRows - 1) / kTmMaxRows;
    sh.n_rows = ((p.rows + blocks - 1) / blocks + 15) / 16 * 16;
    p.row_blocks = (p.rows + sh.n_rows - 1) / sh.n_rows;
    p.sub = kTmSub;
    p.ranges = sm_count() / p.row_blocks;                 // one block per SM: its tiles fill the shared memory
    for (sh.acc_cols = 16; sh.acc_cols < sh.n_rows;) sh.acc_cols *= 2;
    for (sh.stages = kTmMaxStages; tm_smem_bytes(sh.n_rows, c->head_dim, sh.stages) > 227 * 1024;) --sh.stages;
    // a copy must not cross a page: the largest divisor of the page size that fits a tile
    sh.box_rows = kTreeTile;
    if (c->block_table)
      while (c->page_size % sh.box_rows) --sh.box_rows;
    p.tile_keys = kTreeTile / sh.box_rows * sh.box_rows;
  } else {
    p.row_blocks = (p.rows + kSimtRows - 1) / kSimtRows;
    p.sub = kSimtWarps;
    p.ranges = 2 * sm_count() / p.row_blocks;
  }
  if (p.ranges < 1) p.ranges = 1;
  p.tiles = (int)(((int64_t)max_seq + p.tile_keys - 1) / p.tile_keys);
  // drafted survivors are kept behind the cache's
  p.region = (int64_t)p.tiles * kTreeTile + (tokens + 1) / 2 * 2;
  p.max_parts = p.ranges < p.tiles ? p.ranges : (p.tiles > 0 ? p.tiles : 1);
  p.row_bytes = p.region * (int64_t)sizeof(uint2) + 8ll * p.max_parts * p.sub;
  if (p.mma && (int64_t)p.tiles * c->batch * c->kv_heads >= (int64_t)kSampleFrom * p.ranges) {
    p.sample = true;
    p.sample_tiles = (p.tiles + kSampleStride - 1) / kSampleStride;
    if (p.sample_tiles > kSampleTiles) p.sample_tiles = kSampleTiles;
    p.row_bytes += 16ll * p.sample_tiles;
  }
  return p;
}

// K as the copies see it: [blocks or sequences][KV heads][rows][D]
static int tree_k_map(CUtensorMap* map, const ekv_cache_desc* c, int box_rows) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess) return (int)e;
    if (found != cudaDriverEntryPointSuccess) return (int)cudaErrorNotSupported;
    encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }
  const bool paged = c->block_table != nullptr;
  const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)(paged ? c->page_size : c->capacity),
                              (cuuint64_t)c->kv_heads, (cuuint64_t)(paged ? c->num_blocks : c->batch)};
  // the stride of an axis of one entry may be anything
  const cuuint64_t row = (cuuint64_t)c->head_dim * 2;
  const cuuint64_t head = c->kv_heads > 1 ? (cuuint64_t)c->kv_stride_h * 2 : row * dims[1];
  const cuuint64_t block = dims[3] > 1 ? (cuuint64_t)(paged ? c->kv_stride_block : c->kv_stride_b) * 2 : head * dims[2];
  const cuuint64_t strides[3] = {row, head, block};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, unit[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, c->dtype == EKV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            4, c->k, dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? EKV_OK : EKV_ERR_ARG;
}

// what a launch may use of the GPU's memory before the groups are taken in several turns
constexpr int64_t kTreeWorkspace = (int64_t)2 << 30;

static int64_t tree_groups_per_turn(const TreePlan& p, int groups) {
  int64_t n = kTreeWorkspace / (p.row_bytes * p.rows);
  return n < 1 ? 1 : (n > groups ? groups : n);
}

template <typename T, int D>
static int launch_scores(const TreeArgs& a, const TreePlan& p, const CUtensorMap& k_map, cudaStream_t st) {
  const unsigned grid = (unsigned)(a.ranges * a.row_blocks);
  if constexpr (sizeof(T) == 2) {
    const int smem = (int)tm_smem_bytes(p.shape.n_rows, D, p.shape.stages);
    const auto pass = tree_scores_mma_kernel<T, D, false>, sample = tree_scores_mma_kernel<T, D, true>;
    cudaError_t e = cudaFuncSetAttribute(pass, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(sample, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    if (p.sample) sample<<<grid, kTmThreads, smem, st>>>(a, k_map, p.shape);
    pass<<<grid, kTmThreads, smem, st>>>(a, k_map, p.shape);
  } else {
    const size_t smem = sizeof(float) * (kSimtRows + kSimtKeys) * (D + 4);
    cudaError_t e = cudaFuncSetAttribute(tree_scores_simt_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return (int)e;
    tree_scores_simt_kernel<T, D><<<grid, kSimtWarps * 32, smem, st>>>(a);
  }
  return EKV_OK;
}

static bool tree_sizes_ok(const ekv_cache_desc* c, int q_heads, int tokens, int max_seq) {
  return q_heads > 0 && q_heads % c->kv_heads == 0 && tokens > 0 && tokens <= EKV_TREE_MAX_TOKENS && max_seq >= 0 &&
         max_seq <= c->capacity && max_seq <= c->page_capacity * (int64_t)c->page_size &&
         (int64_t)tokens * (q_heads / c->kv_heads) <= (1 << 20) && (int64_t)c->batch * q_heads * tokens <= 0x7fffffff;
}

unsigned int copy_timeouts_tree() { return copy_timeouts_here(); }

}  // namespace ekv

extern "C" size_t ekv_tree_workspace_bytes(const ekv_cache_desc* c, int32_t q_heads, int32_t tokens,
                                           int32_t max_seq_len) {
  using namespace ekv;
  if (check_desc(c) || !tree_sizes_ok(c, q_heads, tokens, max_seq_len)) return 0;
  const TreePlan p = tree_plan(c, q_heads, tokens, max_seq_len);
  return (size_t)(tree_groups_per_turn(p, c->batch * c->kv_heads) * p.rows * p.row_bytes + 256);
}

extern "C" int ekv_tree_decode(const ekv_cache_desc* c, const void* q, const int64_t* q_strides, int32_t q_heads,
                               int32_t tokens, const void* k_draft, const int64_t* k_strides, const void* v_draft,
                               const int64_t* v_strides, const uint8_t* mask, int64_t mask_stride_b,
                               int64_t mask_stride_t, const int32_t* draft_lens, int32_t max_seq_len, float alpha,
                               void* out, const int64_t* out_strides, float* tau, void* workspace,
                               size_t workspace_bytes, int32_t* status, void* stream) {
  using namespace ekv;
  if (int e = check_desc(c)) return e;
  if (!q || !q_strides || !k_draft || !k_strides || !v_draft || !v_strides || !mask || !out || !out_strides || !workspace)
    return EKV_ERR_ARG;
  if (!tree_sizes_ok(c, q_heads, tokens, max_seq_len)) return EKV_ERR_ARG;
  if (!(alpha > 1.f)) return EKV_ERR_ALPHA;
  const int64_t esz = c->dtype == EKV_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_draft) | reinterpret_cast<uintptr_t>(v_draft) |
       reinterpret_cast<uintptr_t>(workspace)) & 15)
    return EKV_ERR_ARG;
  TreeArgs a{};
  for (int i = 0; i < 3; ++i) {
    if ((q_strides[i] * esz) % 16 || (k_strides[i] * esz) % 16 || (v_strides[i] * esz) % 16) return EKV_ERR_ARG;
    a.qs[i] = q_strides[i];
    a.ks[i] = k_strides[i];
    a.vs[i] = v_strides[i];
    a.os[i] = out_strides[i];
  }
  const TreePlan p = tree_plan(c, q_heads, tokens, max_seq_len);
  const int groups = c->batch * c->kv_heads;
  const int64_t turn = tree_groups_per_turn(p, groups);
  if (workspace_bytes < (size_t)(turn * p.rows * p.row_bytes)) return EKV_ERR_WORKSPACE;
  a.c = *c;
  a.q = q;
  a.k_draft = k_draft;
  a.v_draft = v_draft;
  a.mask = mask;
  a.ms_b = mask_stride_b;
  a.ms_t = mask_stride_t;
  a.draft_lens = draft_lens;
  a.out = out;
  a.tau = tau;
  a.q_heads = q_heads;
  a.tokens = tokens;
  a.group = q_heads / c->kv_heads;
  a.by_page = make_fast_div(c->page_size);
  a.alpha = alpha;
  a.zscale = (float)(((double)alpha - 1.0) / sqrt((double)c->head_dim));
  a.max_seq = max_seq_len;
  a.row0 = 0;
  a.rows = p.rows;
  a.ranges = p.ranges;
  a.row_blocks = p.row_blocks;
  a.sub = p.sub;
  a.max_parts = p.max_parts;
  a.region = p.region;
  a.status = status;
  a.entries = static_cast<uint2*>(workspace);
  a.counts = reinterpret_cast<int*>(a.entries + turn * p.rows * p.region);
  a.bounds = reinterpret_cast<float*>(a.counts + turn * p.rows * p.max_parts * p.sub);
  a.classes = a.bounds + turn * p.rows * p.max_parts * p.sub;
  a.sample = p.sample;
  a.sample_tiles = p.sample_tiles;
  a.tile_keys = p.tile_keys;
  const size_t fin_smem = sizeof(int) * ((size_t)p.max_parts * p.sub + 1 + tokens);
  cudaStream_t st = as_stream(stream);
  CUtensorMap k_map{};
  if (p.mma && max_seq_len > 0)
    if (int e = tree_k_map(&k_map, c, p.shape.box_rows)) return e;
  for (int g0 = 0; g0 < groups; g0 += (int)turn) {
    a.g0 = g0;
    a.g1 = (int)(g0 + turn < groups ? g0 + turn : groups);
    const int64_t rows = (int64_t)(a.g1 - g0) * p.rows;
    if (rows > 0x7fffffff) return EKV_ERR_ARG;
    int err = EKV_OK;
    EKV_DISPATCH(c->dtype, c->head_dim, {
      if (max_seq_len > 0) err = launch_scores<T, D>(a, p, k_map, st);
      if (err) return err;
      tree_finish_kernel<T, D><<<(unsigned)rows, kFinThreads, fin_smem, st>>>(a);
    });
  }
  return launch_status();
}
