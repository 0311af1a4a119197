// Entmax attention of a tree of drafted tokens over the cache (see ekv_tree.cuh for the method).
#include <cudaTypedefs.h>

#include "ekv_tree_mma.cuh"

namespace ekv {

// ---- scores on the CUDA cores -------------------------------------------------------------------------------------
//
// For fp32 caches, which have no tensor-core product of their precision (8 sequences of 4096 tokens, 32 rows per KV head, 8
// heads of 128: 230 us the whole call, 8 % of them K's bytes).  A block scores 32 rows against 64 keys at a
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
  const TreeRange at = tree_range<false>(a, range, lane);
  if (at.t_begin == at.t_end) return;
  const int t_begin = at.t_begin, t_end = at.t_end;
  int g_first = at.first;                           // first tile of the group
  for (int g = at.g; g < a.g1 && g_first < t_end; ++g) {
    const int b = g / H, hkv = g % H;
    const int n = tree_tiles(a, b);
    if (n == 0) continue;
    const int g_end = g_first + n;
    const int tile0 = max(t_begin, g_first) - g_first, tile1 = min(t_end, g_end) - g_first;
    const int part = range - at.split.piece_of(g_first);
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
    uint2* const list = a.entries + row_id * a.region + tree_list_place(a, tile0, part, tile1 - tile0, warp);
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
          else if (a.status)
            atomicOr(a.status, EKV_STATUS_PAGE_RANGE);
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
          // (+inf - +inf is a NaN: an infinite score is listed, though nothing lies above its row's bound)
          if (j < valid && !(top - acc[j] >= 1.f)) list[count++] = make_uint2(__float_as_uint(acc[j]), key0 + warp * KPW + j);
      }
    }
    if (lane < live) {
      const int64_t at = row_id * a.max_parts * a.sub + part * a.sub + warp;
      a.counts[at] = count;
      a.bounds[at] = __fadd_rd(top, -1.f);
    }
  }
}

// ---- tau and output ------------------------------------------------------------------------------------------------
//
// A warp per row while at most 768 candidates lie above the row's best bound (the usual case: no barrier, sums by
// shuffle), the whole block per row where more do (flat scores), one such row after another.  Few rows (fewer warps than
// the GPU holds blocks) get a block each from the start.
//
// Bound by latency: the chain lists -> entries -> tau (five or six sums) -> value rows of some 40 keys.  4096 rows of 17k to
// 32k tokens: 31 us alone, of which most lies behind the last tiles of the score pass; 256 rows with all 4096 scores: 16 us
// with a block each (a warp each took about twice that).  The threshold relative to the maximum
// cost 1 to 2 us of a call.

constexpr int kFinWarps = 4;                    // warps of a block that takes a row per warp
constexpr int kFinOneWarps = 8;                 // and of one that takes a single row
constexpr int kFinLight = 768;                  // survivors of a row that one warp finishes
constexpr int kFinLists = 256;                  // and its lists
constexpr int kFinSlots = kFinWarps * kFinLight;   // of a heavy row on chip; more stay in the row's region

// What both ways need to know about a row.
struct FinRow {
  int b, hkv, hq, t, drafts;
  int64_t id;
  int first;                                    // the group's first tile
  int tiles, piece0, lists, len;
  TreeSplit split;
  uint2* region;
};
__device__ __forceinline__ FinRow fin_row(const TreeArgs& a, int64_t id, int lane) {
  FinRow r;
  r.id = id;
  const int gl = (int)((unsigned)id / (unsigned)a.rows), row = a.row0 + (int)id - gl * a.rows, g = a.g0 + gl;
  r.b = g / a.c.kv_heads;
  r.hkv = g % a.c.kv_heads;
  r.hq = r.hkv * a.group + row % a.group;
  r.t = row / a.group;
  r.drafts = tree_drafts(a, r.b);
  r.len = tree_len(a, r.b);
  r.lists = 0;
  r.region = a.entries + id * a.region;
  if (a.dense) return r;
  const TreeGroup at = tree_group(a, g, lane);
  r.split = at.split;
  r.first = at.first;
  r.tiles = tree_tiles(a, r.b);
  r.piece0 = r.tiles ? r.split.piece_of(r.first) : 0;
  r.lists = r.tiles ? (r.split.piece_of(r.first + r.tiles - 1) - r.piece0 + 1) * a.sub : 0;
  return r;
}
// A list of a row: its end in their concatenation, and what leads from a place in that to one in the row's region.
__device__ __forceinline__ int2 fin_list(const TreeArgs& a, const FinRow& r, int l, int before, int count) {
  const int p = l / a.sub, s = l % a.sub;
  const int t0 = max(r.split.begin(r.piece0 + p), r.first) - r.first;
  const int t1 = min(r.split.begin(r.piece0 + p + 1), r.first + r.tiles) - r.first;
  return make_int2(before + count, tree_list_place(a, t0, p, t1 - t0, s) - before);
}
// where entry i of the concatenation of the row's lists lies in its region
__device__ __forceinline__ int fin_place(const FinRow& r, const int2* lists, int i) {
  int lo = 0, hi = r.lists - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (lists[mid].x > i) hi = mid; else lo = mid + 1;
  }
  return lists[lo].y + i;
}
// N entries of the row, i0 + k * step (those from `raw` on: -inf).  The loads come one after another, without a branch
// between them: taken one by one their latencies would add up.
template <int N>
__device__ __forceinline__ void fin_entries(const TreeArgs& a, const FinRow& r, const int2* lists, int raw, int i0, int step,
                                            uint2 (&e)[N]) {
  if (a.dense) {
    const float* const z = reinterpret_cast<const float*>(r.region) + a.region;
#pragma unroll
    for (int k = 0; k < N; ++k) e[k] = make_uint2(__float_as_uint(z[min(i0 + k * step, raw - 1)]), (uint32_t)(i0 + k * step));
  } else {
    int at[N];
#pragma unroll
    for (int k = 0; k < N; ++k) at[k] = fin_place(r, lists, min(i0 + k * step, raw - 1));
#pragma unroll
    for (int k = 0; k < N; ++k) e[k] = r.region[at[k]];
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (i0 + k * step >= raw) e[k].x = __float_as_uint(-INFINITY);
}
// A key's number in the pool (block * page size + place in the page), or itself in a dense cache; -1: no block.  A
// drafted one (~j) becomes INT_MIN + j.
__device__ __forceinline__ int fin_pool_key(const TreeArgs& a, const FinRow& r, int key) {
  if (key < 0) return (int)0x80000000 + ~key;
  if (!a.c.block_table) return key;
  int page, in_page;
  a.by_page.divmod(key, page, in_page);
  const int block = a.c.block_table[(int64_t)r.b * a.c.bt_stride + page];
  return (unsigned)block < (unsigned)a.c.num_blocks ? block * a.c.page_size + in_page : -1;
}
// 16 bytes of the value rows of N such keys, without a branch between the loads
template <typename T, int D, int N>
__device__ __forceinline__ void fin_values(const TreeArgs& a, const FinRow& r, const int (&key)[N], int col, uint4 (&v)[N]) {
  const T* row[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int at = max(key[k], 0);
    int64_t off = r.hkv * a.c.kv_stride_h;
    if (a.c.block_table) {
      int block, in_page;
      a.by_page.divmod(at, block, in_page);
      off += block * a.c.kv_stride_block + (int64_t)in_page * D;
    } else {
      off += r.b * a.c.kv_stride_b + (int64_t)at * D;
    }
    row[k] = static_cast<const T*>(a.c.v) + off;
    if (key[k] < -1)
      row[k] = static_cast<const T*>(a.v_draft) + r.b * a.vs[0] + r.hkv * a.vs[1] + (int64_t)(key[k] & 0x7fffffff) * a.vs[2];
  }
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = *reinterpret_cast<const uint4*>(row[k] + col);
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (key[k] == -1) v[k] = make_uint4(0, 0, 0, 0);
}
// Scores of the drafted keys that the row sees, the others' are -inf; a warp's share: sets of 32 from `first`, every `step`.
template <typename T, int D>
__device__ __forceinline__ void fin_drafts(const TreeArgs& a, const FinRow& r, float* zd, int lane, int first, int step) {
  constexpr int EPL = ElemTraits<T>::EPL, LPR = D / EPL, SIDE = 32 / LPR, N = 4;
  const int col = lane % LPR * EPL, side = lane / LPR;
  float q[EPL];
  unpack<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + r.b * a.qs[0] + r.hq * a.qs[1] + r.t * a.qs[2] + col), q);
  const unsigned char* const mask = a.mask + r.b * a.ms_b + r.t * a.ms_t;
  const T* const k0 = static_cast<const T*>(a.k_draft) + r.b * a.ks[0] + r.hkv * a.ks[1] + col;
  for (int j0 = first * 32; j0 < a.tokens; j0 += step * 32) {
    const bool sees = j0 + lane < r.drafts && mask[j0 + lane];
    if (j0 + lane < a.tokens) zd[j0 + lane] = -INFINITY;
    unsigned left = __ballot_sync(0xffffffffu, sees);
    __syncwarp();
    while (left) {                               // SIDE * N of them at a time
      int j[N];
      uint4 k[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        j[n] = -1;
#pragma unroll
        for (int s = 0; s < SIDE; ++s) {
          const int next = __ffs(left) - 1;      // -1: none left
          if (s == side) j[n] = next;
          left &= left - 1;
        }
      }
#pragma unroll
      for (int n = 0; n < N; ++n) k[n] = *reinterpret_cast<const uint4*>(k0 + (j0 + max(j[n], 0)) * a.ks[2]);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        float x[EPL], s = 0.f;
        unpack<T>(k[n], x);
#pragma unroll
        for (int e = 0; e < EPL; ++e) s = fmaf(q[e], x[e], s);
        s = row_sum<LPR>(s);
        if (lane % LPR == 0 && j[n] >= 0) zd[j0 + j[n]] = s * a.zscale;
      }
    }
  }
}

// Root of sum (x - tau)_+^beta = 1 from below, x = z - (the row's largest score) and tau = c + t in [-1, 0].  In absolute
// scores tau would be rounded to a step of the scores' size, and every key of the support takes that error: with alpha 2
// and 100,000 equal scores of 10 the weights then sum to 0.954.  Relative to the maximum, and in two parts, of which the
// second holds what the first's step leaves, they sum to one within 1e-6.
//
// The norm N(tau) = (sum (x - tau)_+^beta)^(1/beta) falls to 1 at the root and is convex for beta >= 1 (nearly linear when
// the support is settled), so Newton's steps on it climb towards the root from the left; the bracket keeps them safe.  For
// beta < 1 (alpha > 2) the sum rises vertically where a key enters, so only the sum itself says when it is enough, and the
// bracket is halved in its logarithm: n equal scores lie n^-(alpha-1) above the root.  A bracket of two neighbouring numbers
// moves the origin c there.  Two to eight evaluations as a rule, some 30 for thousands of equal scores near the root, up to
// 65 for those with alpha above 4.  The sums are taken with d = (x - c) - t.
struct FinTau {
  float c, t;            // tau = c + t
  float lo, hi;          // bracket of t
};
constexpr int kFinSteps = 96;
__device__ __forceinline__ FinTau fin_tau_begin(float floor_x) { return {0.f, floor_x, floor_x, 0.f}; }
// One step, `s` = sum d^beta, sum d^(beta-1) at f; true: f is the root.
__device__ __forceinline__ bool fin_tau_step(FinTau& f, float2 s, int it, float alpha, int kind, float beta) {
  const bool smooth = beta >= 1.f;
  if (s.x >= 1.f) f.lo = f.t;
  else f.hi = f.t;
  if (it == 0 && s.x < 1.f) f.lo = -1.f;
  // (N - 1) / -N' = (s0^(1/beta) - 1) s0^(1 - 1/beta) / s1
  // (the step need not be exact: the sums at the new tau decide)
  const float root = kind == 0 ? s.x : (kind == 1 ? s.x * rsqrtf(s.x) : pow_pos(s.x, alpha - 1.f));
  const float step = s.x > 0.f ? __fdividef((root - 1.f) * __fdividef(s.x, root), s.y) : -INFINITY;
  // enough: the sum within the rounding of its terms, or a step of half a unit in the last place
  bool done = fabsf(s.x - 1.f) <= 5e-7f || (smooth && fabsf(step) <= 6e-8f * fabsf(f.t));
  if (done && smooth) {
    const bool first = f.c == 0.f;
    f.c = first ? f.t : f.c;
    f.t = first ? step : f.t + step;
  }
  if (!done) {
    float next = f.t + step;
    if (!(next > f.lo && next < f.hi)) {
      if (smooth || f.hi - f.lo < -0.5f * f.lo) next = 0.5f * (f.lo + f.hi);
      else next = f.hi < 0.f ? -sqrtf(-f.lo) * sqrtf(-f.hi) : f.lo * 0.015625f;
    }
    if (!(next > f.lo && next < f.hi)) {         // two neighbours
      done = f.c != 0.f || f.hi == 0.f;
      if (!done) {                               // exact differences from here on: the keys in question lie at c
        f.c = f.hi;
        f.lo -= f.hi;
        f.hi = 0.f;
        next = f.lo * 0.015625f;
      }
    }
    done |= it == kFinSteps - 1;
    f.t = done ? f.lo : next;
  }
  return done;
}

// exclusive scan of small counts over the block; also the total
template <int WARPS>
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
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) base += scratch[w];
    all += scratch[w];
  }
  *total = all;
  return base + inc - v;
}

// Survivors of a heavy row: the first kFinSlots on chip, the others over the row's lists (in place: what is written at i
// was entry i or a later one).
struct FinHeavy {
  uint2* slots;
  uint2* region;
  __device__ __forceinline__ uint2 get(int i) const { return i < kFinSlots ? slots[i] : region[i]; }
  __device__ __forceinline__ void put(int i, uint2 e) const { (i < kFinSlots ? slots[i] : region[i]) = e; }
};

// lists in shared memory: kFinLists per warp, or all of one row
static inline int fin_lists(int max_lists) {
  const int each = max_lists < kFinLists ? max_lists : kFinLists;
  return each * kFinWarps > max_lists ? each * kFinWarps : max_lists;
}

// One row by the whole block.  `lists`: room for all of its lists; `zd`: its drafts' scores, which the caller made.
template <typename T, int D, int WARPS>
__device__ void fin_block_row(const TreeArgs& a, const FinRow& r, uint2* s_slots, int2* lists, const float* zd,
                              float* scratch) {
  constexpr int EPL = ElemTraits<T>::EPL, LPR = D / EPL, THREADS = WARPS * 32, GROUPS = THREADS / LPR, N = 4;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kind = alpha_kind_of(a.alpha);
  const float beta = 1.f / (a.alpha - 1.f);
  int* const iscratch = reinterpret_cast<int*>(scratch);
  const FinHeavy rows{s_slots, r.region};
  const auto block_top = [&](float v) {
    v = warp_max_nan(v);
    __syncthreads();
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v = max_nan(v, scratch[w]);
    return v;
  };
  int raw = 0, n = 0;
  float floor_z = -INFINITY, top = -INFINITY;    // no weight at or below the floor; fmaxf passes over a NaN
  if (a.dense) {                                 // nothing bounds tau yet: the maximum first
    raw = r.len;
    const float* const z = reinterpret_cast<const float*>(r.region) + a.region;
#pragma unroll 8
    for (int i = tid; i < raw; i += THREADS) top = max_nan(top, z[i]);
    for (int j = tid; j < a.tokens; j += THREADS) top = max_nan(top, zd[j]);
    floor_z = __fadd_rd(block_top(top), -1.f);   // (rounded down: a large maximum must stay above it)
    top = -INFINITY;
  } else {
    const int* const counts = a.counts + r.id * a.max_parts * a.sub;
    const float* const bounds = a.bounds + r.id * a.max_parts * a.sub;
    for (int i0 = 0; i0 < r.lists; i0 += THREADS) {
      const bool in = i0 + tid < r.lists;
      const int c = in ? counts[i0 + tid] : 0;
      if (in) floor_z = fmaxf(floor_z, bounds[i0 + tid]);
      int total;
      const int before = block_excl<WARPS>(c, iscratch, &total);
      if (in) lists[i0 + tid] = fin_list(a, r, i0 + tid, raw + before, c);
      raw += total;
    }
    floor_z = block_max(floor_z, scratch);
  }
  __syncthreads();
  // what lies above the floor, in order; a NaN stays
  for (int i0 = 0; i0 < raw + a.tokens; i0 += THREADS * N) {
    uint2 e[N];
    const int i = i0 + tid * N;
    if (i0 < raw) {
      fin_entries(a, r, lists, raw, i, 1, e);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) e[k] = make_uint2(__float_as_uint(-INFINITY), 0);
    }
    int mine = 0;
    bool keep[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = i + k - raw;
      if (j >= 0 && j < a.tokens) e[k] = make_uint2(__float_as_uint(zd[j]), (uint32_t)~j);     // ~j: drafted
      const float z = __uint_as_float(e[k].x);
      keep[k] = !(z <= floor_z);
      top = max_nan(top, z);                     // of all that is read: the floor of an infinite row drops even its maximum
      mine += keep[k];
    }
    int total;
    int at = n + block_excl<WARPS>(mine, iscratch, &total);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (keep[k]) rows.put(at++, e[k]);
    n += total;
    __syncthreads();                             // before the next entries are read where these may have been written
  }
  top = block_top(top);
  T* const out = static_cast<T*>(a.out) + r.b * a.os[0] + r.hq * a.os[1] + r.t * a.os[2];
  float* const tau_out = a.tau ? a.tau + ((int64_t)r.b * a.q_heads + r.hq) * a.tokens + r.t : nullptr;
  if (!(fabsf(top) < INFINITY)) {                // nothing visible: zeros.  NaN or +inf among the scores: NaN
    if (tid < D) out[tid] = from_float<T>(top == -INFINITY ? 0.f : NAN);
    if (tid == 0 && tau_out) *tau_out = top == -INFINITY ? INFINITY : NAN;
    return;
  }
  // thread 0 makes the steps: all leave the loop by the flag that it writes
  FinTau tau = fin_tau_begin(fmaxf(floor_z - top, -1.f));
  __syncthreads();
  for (int it = 0; it < kFinSteps; ++it) {
    float s0 = 0.f, s1 = 0.f, s2 = 0.f;
    for (int i = tid; i < n; i += THREADS)
      halley_accumulate(__uint_as_float(rows.get(i).x) - top - tau.c, tau.t, kind, beta, s0, s1, s2);
    s0 = warp_sum(s0);
    s1 = warp_sum(s1);
    if (lane == 0) {
      scratch[warp * 2] = s0;
      scratch[warp * 2 + 1] = s1;
    }
    __syncthreads();
    if (tid == 0) {
      float2 s = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        s.x += scratch[w * 2];
        s.y += scratch[w * 2 + 1];
      }
      scratch[31] = fin_tau_step(tau, s, it, a.alpha, kind, beta) ? 1.f : 0.f;
      scratch[30] = tau.t;
      scratch[29] = tau.c;
    }
    __syncthreads();
    tau.c = scratch[29];
    tau.t = scratch[30];
    if (scratch[31] != 0.f) break;
  }
  int m = 0;
  float sum_w = 0.f;
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    uint2 e = make_uint2(0, 0);
    float w = 0.f;
    if (i0 + tid < n) {
      e = rows.get(i0 + tid);
      w = entmax_weight(__uint_as_float(e.x) - top - tau.c, tau.t, kind, beta);
      sum_w += w;
    }
    int total;
    const int at = m + block_excl<WARPS>(w > 0.f, iscratch, &total);
    if (w > 0.f) rows.put(at, make_uint2(__float_as_uint(w), (uint32_t)fin_pool_key(a, r, (int)e.y)));
    m += total;
  }
  // far from alpha 1.5 and 2 a power makes much of a rounding: above 2 keys next to the root weigh (rounding)^beta, near 1
  // every weight is off by beta roundings, and no tau that fp32 holds makes them sum to one
  sum_w = block_sum(sum_w, scratch);
  const float scale = kind == 2 ? 1.f / sum_w : 1.f;
  float acc[EPL] = {};
  const int sub = tid / LPR, col = tid % LPR * EPL;
  for (int i0 = sub; i0 < m; i0 += GROUPS * N) {
    uint4 v[N];
    float w[N];
    int key[N];
#pragma unroll
    for (int f = 0; f < N; ++f) {
      const uint2 e = rows.get(min(i0 + f * GROUPS, m - 1));
      w[f] = __uint_as_float(e.x);
      key[f] = (int)e.y;
    }
    fin_values<T, D>(a, r, key, col, v);
#pragma unroll
    for (int f = 0; f < N; ++f)
      if (i0 + f * GROUPS < m) {
        float x[EPL];
        unpack<T>(v[f], x);
#pragma unroll
        for (int j = 0; j < EPL; ++j) acc[j] = fmaf(w[f], x[j], acc[j]);
      }
  }
  __syncthreads();                               // the slots become partial sums
  float* const s_acc = reinterpret_cast<float*>(s_slots);
#pragma unroll
  for (int j = 0; j < EPL; ++j) s_acc[sub * D + col + j] = acc[j];
  __syncthreads();
  if (tid < D) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) s += s_acc[i * D + tid];
    out[tid] = from_float<T>(s * scale);
  }
  if (tid == 0 && tau_out) *tau_out = top + (tau.c + tau.t);
}

// A block per row.  Dynamic shared memory: [kFinSlots] slots, [n_lists] lists, [tokens] drafted scores.
template <typename T, int D>
__global__ void __launch_bounds__(kFinOneWarps * 32) tree_finish_one_kernel(const __grid_constant__ TreeArgs a,
                                                                            const int n_lists) {
  extern __shared__ uint2 s_slots[];
  __shared__ float scratch[32];
  int2* const lists = reinterpret_cast<int2*>(s_slots + kFinSlots);
  float* const zd = reinterpret_cast<float*>(lists + n_lists);
  const int lane = threadIdx.x & 31;
  const FinRow r = fin_row(a, blockIdx.x, lane);
  if (r.t < r.drafts) fin_drafts<T, D>(a, r, zd, lane, threadIdx.x >> 5, kFinOneWarps);
  tree_wait_for_previous();
  if (r.t >= r.drafts) return;                   // behind a short tree: left as it was
  __syncthreads();
  fin_block_row<T, D, kFinOneWarps>(a, r, s_slots, lists, zd, scratch);
}

// A warp per row.  Dynamic shared memory: [kFinSlots] slots, [n_lists] lists, [warps][tokens] drafted scores.
template <typename T, int D>
__global__ void __launch_bounds__(kFinWarps * 32, 7) tree_finish_kernel(const __grid_constant__ TreeArgs a,
                                                                        const int64_t n_rows, const int n_lists) {
  constexpr int EPL = ElemTraits<T>::EPL, LPR = D / EPL, SIDE = 32 / LPR;
  extern __shared__ uint2 s_slots[];
  __shared__ float scratch[32];
  __shared__ int s_heavy[kFinWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int2* const s_lists = reinterpret_cast<int2*>(s_slots + kFinSlots);
  int2* const lists = s_lists + warp * min(a.max_parts * a.sub, kFinLists);
  float* const zd = reinterpret_cast<float*>(s_lists + n_lists) + warp * a.tokens;
  uint2* const slots = s_slots + warp * kFinLight;
  const int64_t id0 = (int64_t)blockIdx.x * kFinWarps;
  const int kind = alpha_kind_of(a.alpha);
  const float beta = 1.f / (a.alpha - 1.f);

  // what needs nothing of the score pass
  FinRow r{};
  bool mine = id0 + warp < n_rows, heavy = false;
  if (mine) {
    r = fin_row(a, id0 + warp, lane);
    mine = r.t < r.drafts;                       // else behind a short tree: left as it was
  }
  if (mine) fin_drafts<T, D>(a, r, zd, lane, 0, 1);
  tree_wait_for_previous();
  __syncwarp();

  float floor_z = -INFINITY, top = -INFINITY;    // no weight at or below the floor; fmaxf passes over a NaN
  int raw = r.len, n = 0;
  if (mine) {
    if (!a.dense && r.lists > kFinLists) {
      n = kFinLight + 1;                         // the block's
    } else if (!a.dense) {
      raw = 0;
      const int* const counts = a.counts + r.id * a.max_parts * a.sub;
      const float* const bounds = a.bounds + r.id * a.max_parts * a.sub;
      for (int i0 = 0; i0 < r.lists; i0 += 32) {
        const bool in = i0 + lane < r.lists;
        const int c = in ? counts[i0 + lane] : 0;
        int end = c;
        if (in) floor_z = fmaxf(floor_z, bounds[i0 + lane]);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int m = __shfl_up_sync(0xffffffffu, end, o);
          if (lane >= o) end += m;
        }
        if (in) lists[i0 + lane] = fin_list(a, r, i0 + lane, raw + end - c, c);
        raw += __shfl_sync(0xffffffffu, end, 31);
      }
      floor_z = warp_max(floor_z);
    }
    __syncwarp();
    // what lies above the floor, in order; a NaN stays.  The floor follows the maximum, and where too much was kept under
    // an early one, the slots are gone through again
    constexpr int AT_ONCE = 8;
    for (int i0 = 0; i0 < raw + a.tokens && n <= kFinLight; i0 += 32 * AT_ONCE) {
      uint2 e[AT_ONCE];
      float most = -INFINITY;
      if (i0 < raw) {
        fin_entries(a, r, lists, raw, i0 + lane, 32, e);
      } else {
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) e[k] = make_uint2(__float_as_uint(-INFINITY), 0);
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int j = i0 + 32 * k + lane - raw;
        if (j >= 0 && j < a.tokens) e[k] = make_uint2(__float_as_uint(zd[j]), (uint32_t)~j);     // ~j: drafted
        most = max_nan(most, __uint_as_float(e[k].x));
      }
      top = max_nan(top, warp_max_nan(most));
      floor_z = fmaxf(floor_z, __fadd_rd(top, -1.f));      // (rounded down: a large maximum must stay above it)
      if (n > kFinLight - 32 * AT_ONCE) {
        int kept = 0;
        for (int j0 = 0; j0 < n; j0 += 32) {
          const uint2 x = j0 + lane < n ? slots[j0 + lane] : make_uint2(__float_as_uint(-INFINITY), 0);
          const bool keep = !(__uint_as_float(x.x) <= floor_z);
          const unsigned has = __ballot_sync(0xffffffffu, keep);
          if (keep) slots[kept + __popc(has & ((1u << lane) - 1))] = x;
          kept += __popc(has);
          __syncwarp();
        }
        n = kept;
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const bool keep = !(__uint_as_float(e[k].x) <= floor_z);
        const unsigned has = __ballot_sync(0xffffffffu, keep);
        const int to = n + __popc(has & ((1u << lane) - 1));
        if (keep && to < kFinLight) slots[to] = e[k];
        n += __popc(has);
      }
    }
    heavy = n > kFinLight;
    __syncwarp();
  }
  if (lane == 0) s_heavy[warp] = heavy;

  if (mine && !heavy) {
    T* const out = static_cast<T*>(a.out) + r.b * a.os[0] + r.hq * a.os[1] + r.t * a.os[2];
    float* const tau_out = a.tau ? a.tau + ((int64_t)r.b * a.q_heads + r.hq) * a.tokens + r.t : nullptr;
    if (!(fabsf(top) < INFINITY)) {              // nothing visible: zeros.  NaN or +inf among the scores: NaN
      for (int e = lane; e < D; e += 32) out[e] = from_float<T>(top == -INFINITY ? 0.f : NAN);
      if (lane == 0 && tau_out) *tau_out = top == -INFINITY ? INFINITY : NAN;
    } else {
      FinTau tau = fin_tau_begin(fmaxf(floor_z - top, -1.f));
      for (int it = 0; it < kFinSteps; ++it) {
        float2 s = make_float2(0.f, 0.f);
        float s2 = 0.f;
        if (kind == 1) {                         // alpha 1.5, the usual one, without a branch per score
#pragma unroll 4
          for (int i = lane; i < n; i += 32) {
            const float d = fmaxf(__uint_as_float(slots[i].x) - top - tau.c - tau.t, 0.f);
            s.x = fmaf(d, d, s.x);
            s.y += d;
          }
        } else {
          for (int i = lane; i < n; i += 32)
            halley_accumulate(__uint_as_float(slots[i].x) - top - tau.c, tau.t, kind, beta, s.x, s.y, s2);
        }
        s.x = warp_sum(s.x);
        s.y = warp_sum(s.y);
        if (fin_tau_step(tau, s, it, a.alpha, kind, beta)) break;      // the same in every lane
      }
      // the support, in order and in place
      int m = 0;
      float sum_w = 0.f;
      for (int i0 = 0; i0 < n; i0 += 32) {
        uint2 e = make_uint2(0, 0);
        float w = 0.f;
        if (i0 + lane < n) {
          e = slots[i0 + lane];
          w = entmax_weight(__uint_as_float(e.x) - top - tau.c, tau.t, kind, beta);
          sum_w += w;
        }
        const unsigned has = __ballot_sync(0xffffffffu, w > 0.f);
        if (w > 0.f) slots[m + __popc(has & ((1u << lane) - 1))] = make_uint2(__float_as_uint(w), e.y);
        m += __popc(has);
        __syncwarp();
      }
      if (a.c.block_table)                       // 32 table entries at a time instead of one before each value row
        for (int i = lane; i < m; i += 32) slots[i].y = (uint32_t)fin_pool_key(a, r, (int)slots[i].y);
      else
        for (int i = lane; i < m; i += 32)
          if ((int)slots[i].y < 0) slots[i].y = (uint32_t)fin_pool_key(a, r, (int)slots[i].y);
      __syncwarp();
      float acc[EPL] = {};
      const int col = lane % LPR * EPL;
      constexpr int FLIGHT = 4;
      for (int i0 = lane / LPR; i0 < m; i0 += SIDE * FLIGHT) {
        uint4 v[FLIGHT];
        float w[FLIGHT];
        int key[FLIGHT];
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) {
          const uint2 e = slots[min(i0 + f * SIDE, m - 1)];
          w[f] = __uint_as_float(e.x);
          key[f] = (int)e.y;
        }
        fin_values<T, D>(a, r, key, col, v);
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f)
          if (i0 + f * SIDE < m) {
            float x[EPL];
            unpack<T>(v[f], x);
#pragma unroll
            for (int j = 0; j < EPL; ++j) acc[j] = fmaf(w[f], x[j], acc[j]);
          }
      }
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
        for (int j = 0; j < EPL; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
      sum_w = warp_sum(sum_w);
      const float scale = kind == 2 ? 1.f / sum_w : 1.f;         // see fin_block_row
      if (lane < LPR)
#pragma unroll
        for (int j = 0; j < EPL; ++j) out[col + j] = from_float<T>(acc[j] * scale);
      if (lane == 0 && tau_out) *tau_out = top + (tau.c + tau.t);
    }
  }

  // ---- heavy rows: the whole block, one row after another
  __syncthreads();
  for (int w = 0; w < kFinWarps; ++w) {
    if (!s_heavy[w]) continue;                   // uniform over the block
    __syncthreads();                             // the slots are free
    fin_block_row<T, D, kFinWarps>(a, fin_row(a, id0 + w, lane), s_slots, s_lists,
                                   reinterpret_cast<const float*>(s_lists + n_lists) + w * a.tokens, scratch);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------

struct TreePlan {
  int64_t region;        // entries per row
  int tiles, rows, sub, list_turn, list_cols, row_blocks, ranges, tile_keys;
  int64_t row_bytes;     // workspace per row
  int max_parts;
  bool mma, dense;       // tensor cores; all scores written out, no sample
  int sample_tiles;
  TmShape shape;
};

// Tiles per block from which on there is a sample, and tiles per sequence up to which there need not be one: below both,
// all scores are written out.  One sequence of 4096 tokens, 32 rows: 35 us without a sample (score pass 15, finish 20); a
// sample and its bounds alone take 16.  The row of scores that the finish kernel then reads grows with the sequence.
constexpr int kSampleFrom = 8;

constexpr int kDenseTiles = 64;

// what a launch may use of the GPU's memory before the groups, and where one of them is too large the rows, take turns
constexpr int64_t kTreeWorkspace = (int64_t)6 << 30;

static TreePlan tree_plan_rows(const ekv_cache_desc* c, int rows, int tokens, int max_seq) {
  TreePlan p{};
  p.rows = rows;
  p.mma = c->dtype != EKV_F32;
  p.tile_keys = kTreeTile;
  p.list_turn = 1;
  if (p.mma) {
    TmShape& sh = p.shape;
    p.row_blocks = (p.rows + kTmMaxRows - 1) / kTmMaxRows;
    sh.n_rows = (p.rows + p.row_blocks - 1) / p.row_blocks;
    sh.row_tiles = sh.n_rows > kTreeTile ? 2 : 1;
    sh.copies = sh.n_rows <= 32 ? 4 : (sh.n_rows <= 64 ? 2 : 1);
    p.list_turn = sh.row_tiles == 2 ? 1 : 4;
    p.list_cols = sh.row_tiles == 2 ? kTreeTile / 2 : kTreeTile / sh.copies;
    p.sub = sh.row_tiles == 2 ? 2 : 4 * sh.copies;
    p.ranges = sm_count() / p.row_blocks;                 // one block per SM: its tiles fill the shared memory
    for (sh.stages = kTmMaxStages; tm_smem_bytes(sh.row_tiles, c->head_dim, sh.stages) > 227 * 1024;) --sh.stages;
    // a copy must not cross a page: the largest divisor of the page size that fits a tile
    sh.box_rows = kTreeTile;
    if (c->block_table)
      while (c->page_size % sh.box_rows) --sh.box_rows;
    p.tile_keys = kTreeTile / sh.box_rows * sh.box_rows;
  } else {
    p.row_blocks = (p.rows + kSimtRows - 1) / kSimtRows;
    p.sub = kSimtWarps;
    p.list_cols = kTreeTile / kSimtWarps;
    p.ranges = 2 * sm_count() / p.row_blocks;
  }
  if (p.ranges < 1) p.ranges = 1;
  p.tiles = (int)(((int64_t)max_seq + p.tile_keys - 1) / p.tile_keys);
  p.max_parts = p.ranges < p.tiles ? p.ranges : (p.tiles > 0 ? p.tiles : 1);
  p.dense = p.mma && p.tiles <= kDenseTiles && (int64_t)p.tiles * c->batch * c->kv_heads < (int64_t)kSampleFrom * p.ranges;
  // drafted survivors are kept behind the cache's
  p.region = ((int64_t)p.tiles + (p.dense ? 0 : (int64_t)p.max_parts * (p.list_turn - 1))) * kTreeTile + (tokens + 1) / 2 * 2;
  p.row_bytes = p.region * (int64_t)sizeof(uint2) + 8ll * p.max_parts * p.sub;
  if (p.mma && !p.dense) {
    p.sample_tiles = (p.tiles + kSampleStride - 1) / kSampleStride;
    if (p.sample_tiles > kSampleTiles) p.sample_tiles = kSampleTiles;
    p.row_bytes += 16ll * p.sample_tiles + 4;
  }
  return p;
}

// The plan of a turn: all rows of a group, or as many as the workspace holds (whole blocks of rows where it can be).
static TreePlan tree_plan(const ekv_cache_desc* c, int q_heads, int tokens, int max_seq) {
  int64_t rows = (int64_t)tokens * (q_heads / c->kv_heads);
  for (;;) {
    const TreePlan p = tree_plan_rows(c, (int)rows, tokens, max_seq);
    if (p.row_bytes * rows <= kTreeWorkspace || rows == 1) return p;
    rows = kTreeWorkspace / p.row_bytes;           // fewer; with fewer rows a row may have more pieces, hence more bytes
    if (rows >= kTmMaxRows) rows = rows / kTmMaxRows * kTmMaxRows;
    if (rows < 1) rows = 1;
  }
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

static int64_t tree_groups_per_turn(const TreePlan& p, int groups) {
  int64_t n = kTreeWorkspace / (p.row_bytes * p.rows);
  if (p.tiles > 0 && n > kTreeMaxTiles / p.tiles) n = kTreeMaxTiles / p.tiles;
  return n < 1 ? 1 : (n > groups ? groups : n);
}

// `after`: the kernel may start while the one before it in the stream still runs (it waits itself before it uses results)
template <typename... P, typename... V>
static cudaError_t launch_after(void (*kernel)(P...), unsigned grid, int threads, size_t smem, cudaStream_t st, bool after,
                                const V&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = after ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, int D>
static int launch_scores(const TreeArgs& a, const TreePlan& p, const CUtensorMap& k_map, cudaStream_t st) {
  const unsigned grid = (unsigned)(a.ranges * a.row_blocks);
  if constexpr (sizeof(T) == 2) {
    const int smem = (int)tm_smem_bytes(p.shape.row_tiles, D, p.shape.stages);
    const auto run = [&](auto kernel, bool after) -> int {
      cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e == cudaSuccess) e = launch_after(kernel, grid, kTmThreads, smem, st, after, a, k_map, p.shape);
      return (int)e;
    };
    if (p.dense) return run(tree_scores_mma_kernel<T, D, TM_DENSE>, false);
    if (int e = run(tree_scores_mma_kernel<T, D, TM_SAMPLE>, false)) return e;
    const int64_t rows = (int64_t)(a.g1 - a.g0) * a.rows;
    const cudaError_t e = launch_after(tree_bounds_kernel, (unsigned)((rows + 7) / 8), 256, 0, st, true, a, rows);
    if (e != cudaSuccess) return (int)e;
    return run(tree_scores_mma_kernel<T, D, TM_LISTS>, true);
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
         (int64_t)tokens * (q_heads / c->kv_heads) <= (1 << 20) && (int64_t)c->batch * q_heads * tokens <= 0x7fffffff &&
         (!c->block_table || (int64_t)c->num_blocks * c->page_size <= 0x7fffffff);
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
  if (!(alpha > 1.f) || !(alpha < INFINITY)) return EKV_ERR_ALPHA;
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
  a.row_bounds = a.classes + turn * p.rows * p.sample_tiles * 4;
  a.dense = p.dense;
  a.list_turn = p.list_turn;
  a.list_cols = p.list_cols;
  a.sample_tiles = p.sample_tiles;
  a.tile_keys = p.tile_keys;
  // few rows: a block each, while those fit the GPU in about two waves (three of these blocks to an SM)
  const bool one = (int64_t)groups * p.rows <= 6 * sm_count();
  const int n_lists = one ? p.max_parts * p.sub : fin_lists(p.max_parts * p.sub);
  const size_t fin_smem = sizeof(uint2) * ((size_t)kFinSlots + n_lists) + sizeof(float) * (size_t)(one ? 1 : kFinWarps) * tokens;
  cudaStream_t st = as_stream(stream);
  CUtensorMap k_map{};
  if (p.mma && max_seq_len > 0)
    if (int e = tree_k_map(&k_map, c, p.shape.box_rows)) return e;
  const int all_rows = tokens * a.group;
  for (int g0 = 0; g0 < groups; g0 += (int)turn)
    for (int row0 = 0; row0 < all_rows; row0 += p.rows) {
      a.g0 = g0;
      a.g1 = (int)(g0 + turn < groups ? g0 + turn : groups);
      a.row0 = row0;
      a.rows = p.rows < all_rows - row0 ? p.rows : all_rows - row0;
      const int64_t rows = (int64_t)(a.g1 - g0) * a.rows;
      if (rows > 0x7fffffff) return EKV_ERR_ARG;
      int err = EKV_OK;
      EKV_DISPATCH(c->dtype, c->head_dim, {
        if (max_seq_len > 0) err = launch_scores<T, D>(a, p, k_map, st);
        if (err) return err;
        const auto finish = [&](auto kernel, unsigned grid, int threads, auto... args) {
          const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)fin_smem);
          return e != cudaSuccess ? e : launch_after(kernel, grid, threads, fin_smem, st, max_seq_len > 0, a, args...);
        };
        const cudaError_t e = one ? finish(tree_finish_one_kernel<T, D>, (unsigned)rows, kFinOneWarps * 32, n_lists)
                                  : finish(tree_finish_kernel<T, D>, (unsigned)((rows + kFinWarps - 1) / kFinWarps),
                                           kFinWarps * 32, rows, n_lists);
        if (e != cudaSuccess) return (int)e;
      });
    }
  return launch_status();
}
