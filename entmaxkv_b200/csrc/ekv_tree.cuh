// Entmax attention of a tree of drafted tokens over the cache: what its kernels share.
//
// Row (b, h, t) - a query head of one drafted token - sees every key of sequence b and the drafted keys that its mask
// names.  z = (alpha-1)/sqrt(D) q.k, tau solves sum (z - tau)_+^beta = 1 with beta = 1/(alpha-1), and the output is
// sum (z - tau)_+^beta v.  The tau of some of the keys is a lower bound of the tau of all of them, and a key below a
// lower bound has no weight.  Three kernels:
//
//   sample   (not for few keys) scores a few tiles of every sequence and keeps each row's largest scores of disjoint
//            classes of keys; a small kernel makes their tau the row's bound.
//   scores   one pass over K.  The rows that share a KV head are scored together, and each row keeps a list of the
//            (z, key) above its bound.
//   finish   a warp per row, or a block where rows are few or a row's list is long: adds the drafted keys, solves tau on the
//            lists and sums the value rows of the support.
//            V is read only where a weight is non-zero.
//
// Work split of a pass over K: its 128-key tiles of all (sequence, KV head) groups in a row, cut into `ranges` equal
// pieces, one per resident block, whatever the lengths of the sequences are.  The part of a group that lies in one
// piece has lists of its own, and the later kernels find the pieces from the lengths alone.
#pragma once

#include "ekv_common.cuh"

namespace ekv {

constexpr int kTreeTile = 128;         // places for keys in a tile
// Tiles in a sequence's sample, at most, and at most every eighth one.  Half as many tiles: 258 instead of 242 us for one
// sequence of 131k tokens and 512 rows per KV head (twice the candidates); every fourth or sixteenth tile: 146 and 156
// instead of 143 us for eight sequences of 17k to 32k tokens.
constexpr int kSampleTiles = 128;
constexpr int kSampleStride = 8;
constexpr int kTreeMaxTiles = 1 << 23; // tiles of a launch, with at most 512 pieces

struct TreeArgs {
  ekv_cache_desc c;
  const void* q;                       // [B, H_q, T, D]
  int64_t qs[3];                       // element strides: batch, head, token
  const void* k_draft;                 // [B, H_kv, T, D]
  const void* v_draft;
  int64_t ks[3], vs[3];
  const unsigned char* mask;           // [B or 1, T, T]
  int64_t ms_b, ms_t;
  const int* draft_lens;               // [B] or null
  void* out;                           // [B, H_q, T, D]
  int64_t os[3];
  float* tau;                          // [B, H_q, T] or null
  int q_heads, tokens, group;          // group: query heads per KV head
  FastDiv by_page;
  float alpha, zscale;
  int max_seq;                         // lengths are clipped to this (the row regions' size)
  // one launch covers the (sequence, KV head) groups [g0, g1) and the rows [row0, row0 + rows) of each; row = t * group + g
  int g0, g1, row0, rows;
  int ranges, row_blocks;              // pieces of the tile sequence; row blocks
  int sub, list_turn, list_cols;       // lists per row and piece, each of list_cols columns of every list_turn-th tile
  int dense;                           // no lists: all scores of a row, floats from the middle of its region
  int max_parts;                       // pieces of one group, at most
  uint2* entries;                      // [groups][rows][region]: z bits, key
  int64_t region;
  int* counts;                         // [groups][rows][max_parts * sub]
  float* bounds;                       // same shape: tau lies above, and the list misses no key of its share that does
  int tile_keys;                       // keys of a tile (kTreeTile, or less: whole boxes of the copies)
  int sample_tiles;                    // tiles of one group in the sample, at most
  float* classes;                      // [groups][rows][sample_tiles][4]: largest raw score of 32 keys
  float* row_bounds;                   // [groups][rows]: the sample's bound of tau, in raw score units
  int* status;
};

__device__ __forceinline__ int tree_len(const TreeArgs& a, int b) { return min(max(a.c.seq_lens[b], 0), a.max_seq); }
// tiles of sequence b: all, or those of its sample
__device__ __forceinline__ int tree_all_tiles(const TreeArgs& a, int b) {
  return (tree_len(a, b) + a.tile_keys - 1) / a.tile_keys;
}
__host__ __device__ __forceinline__ int tree_sample_stride(int n_all) {
  const int s = (n_all + kSampleTiles - 1) / kSampleTiles;
  return s > kSampleStride ? s : kSampleStride;
}
template <bool SAMPLE = false>
__device__ __forceinline__ int tree_tiles(const TreeArgs& a, int b) {
  const int n = tree_all_tiles(a, b);
  if (!SAMPLE) return n;
  const int s = tree_sample_stride(n);
  return (n + s - 1) / s;
}
// place of the sample's j-th tile: the last one is the sequence's last (the newest keys), the others start with its first
__device__ __forceinline__ int tree_sample_tile(int j, int n_sample, int n_all) {
  return j + 1 == n_sample ? n_all - 1 : j * tree_sample_stride(n_all);
}
__device__ __forceinline__ int tree_drafts(const TreeArgs& a, int b) {
  return a.draft_lens ? min(max(a.draft_lens[b], 0), a.tokens) : a.tokens;
}

// The tile sequence of W tiles in N pieces (N <= W): piece i is [i W / N, (i + 1) W / N).  W N < 2^32 (see kTreeMaxTiles).
struct TreeSplit {
  unsigned W, N;
  __device__ __forceinline__ int begin(int i) const { return (int)((unsigned)i * W / N); }
  __device__ __forceinline__ int piece_of(int tile) const { return (int)((((unsigned)tile + 1) * N - 1) / W); }
};

// The lengths of 32 sequences at a time, one per lane: tiles of this lane's sequence that belong to the launch, and the
// launch's groups among its KV heads.
struct TreeLane {
  int first, tiles;      // first group, tiles per group
  int all, end;          // tiles of this sequence; running sum with it
};
template <bool SAMPLE>
__device__ __forceinline__ TreeLane tree_lane(const TreeArgs& a, int b0, int lane, int before) {
  const int H = a.c.kv_heads, b = b0 + lane;
  TreeLane t;
  t.first = max(a.g0, b * H);
  const int groups = max(min(a.g1, (b + 1) * H) - t.first, 0);
  t.tiles = b < a.c.batch && groups > 0 ? tree_tiles<SAMPLE>(a, b) : 0;
  t.all = t.end = groups * t.tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, t.end, o);
    if (lane >= o) t.end += n;
  }
  t.end += before;
  return t;
}

// Warp-cooperative: what piece `range` of the launch's tile sequence covers, and the group that it begins in.  An empty
// piece has t_begin == t_end.
struct TreeRange {
  TreeSplit split;
  int t_begin, t_end;
  int g;
  int first;             // the group's first tile
};
template <bool SAMPLE>
__device__ __forceinline__ TreeRange tree_range(const TreeArgs& a, int range, int lane) {
  const int b_first = a.g0 / a.c.kv_heads, b_last = (a.g1 - 1) / a.c.kv_heads;
  TreeRange r;
  int W = 0;
  TreeLane t;
  for (int b0 = b_first; b0 <= b_last; b0 += 32) {
    t = tree_lane<SAMPLE>(a, b0, lane, W);
    W = __shfl_sync(0xffffffffu, t.end, 31);
  }
  r.split.W = W;
  r.split.N = min(a.ranges, W);
  r.t_begin = r.t_end = 0;
  r.g = a.g1;
  r.first = 0;
  if (W == 0 || range >= (int)r.split.N) return r;
  r.t_begin = r.split.begin(range);
  r.t_end = r.split.begin(range + 1);
  int before = 0;
  for (int b0 = b_first; b0 <= b_last; b0 += 32) {
    if (b_last - b_first >= 32) t = tree_lane<SAMPLE>(a, b0, lane, before);     // else it is still in the registers
    const unsigned hit = __ballot_sync(0xffffffffu, t.end > r.t_begin);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int start = __shfl_sync(0xffffffffu, t.end - t.all, src);
      const int skip = (r.t_begin - start) / __shfl_sync(0xffffffffu, t.tiles, src);
      r.g = __shfl_sync(0xffffffffu, t.first, src) + skip;
      r.first = start + skip * __shfl_sync(0xffffffffu, t.tiles, src);
      break;
    }
    before = __shfl_sync(0xffffffffu, t.end, 31);
  }
  return r;
}

// Warp-cooperative: the launch's split, and the first tile of group g.
struct TreeGroup {
  TreeSplit split;
  int first;
};
__device__ __forceinline__ TreeGroup tree_group(const TreeArgs& a, int g, int lane) {
  const int H = a.c.kv_heads, b_first = a.g0 / H, b_last = (a.g1 - 1) / H, b = g / H;
  TreeGroup r;
  int W = 0;
  r.first = 0;
  for (int b0 = b_first; b0 <= b_last; b0 += 32) {
    const TreeLane t = tree_lane<false>(a, b0, lane, W);
    if (b >= b0 && b < b0 + 32)
      r.first = __shfl_sync(0xffffffffu, t.end - t.all, b - b0) +
                (g - __shfl_sync(0xffffffffu, t.first, b - b0)) * __shfl_sync(0xffffffffu, t.tiles, b - b0);
    W = __shfl_sync(0xffffffffu, t.end, 31);
  }
  r.split.W = W;
  r.split.N = min(a.ranges, W);
  return r;
}

// Where list s of a row's part begins in the row's region: the part-th piece of the group, `tiles` tiles from `tile0`.
__device__ __forceinline__ int tree_list_place(const TreeArgs& a, int tile0, int part, int tiles, int s) {
  return (tile0 + part * (a.list_turn - 1)) * kTreeTile + s * ((tiles + a.list_turn - 1) / a.list_turn) * a.list_cols;
}

// Programmatic launches: a kernel may start while the one before it still runs, up to the point where it needs its results.
__device__ __forceinline__ void tree_wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void tree_let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {      // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

}  // namespace ekv
