// Entmax attention of a tree of drafted tokens over the cache: what its kernels share.
//
// Row (b, h, t) - a query head of one drafted token - sees every key of sequence b and the drafted keys that its mask
// names.  z = (alpha-1)/sqrt(D) q.k, tau solves sum (z - tau)_+^beta = 1 with beta = 1/(alpha-1), and the output is
// sum (z - tau)_+^beta v.  The tau of some of the keys is a lower bound of the tau of all of them, and a key below a
// lower bound has no weight.  Three kernels:
//
//   sample   (long sequences) scores a few tiles of every sequence and keeps each row's largest scores of disjoint
//            classes of keys; their tau is the row's bound.
//   scores   one pass over K.  The rows that share a KV head are scored together, and each row keeps a list of the
//            (z, key) above its bound.
//   finish   one block per row: adds the drafted keys, solves tau on the lists and sums the value rows of the support.
//            V is read only where a weight is non-zero.
//
// Work split of a pass over K: its 128-key tiles of all (sequence, KV head) groups in a row, cut into `ranges` equal
// pieces, one per resident block, whatever the lengths of the sequences are.  The part of a group that lies in one
// piece has lists of its own, and the later kernels find the pieces from the lengths alone.
#pragma once

#include "ekv_common.cuh"

namespace ekv {

constexpr int kTreeTile = 128;         // places for keys in a tile
constexpr int kSampleTiles = 64;       // tiles of a sequence in its sample, at most
constexpr int kSampleStride = 8;       // and at most every eighth one

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
  int ranges, row_blocks, sub;         // pieces of the tile sequence; row blocks; lists per row and piece
  int max_parts;                       // pieces of one group, at most
  uint2* entries;                      // [groups][rows][region]: z bits, key
  int64_t region;
  int* counts;                         // [groups][rows][max_parts * sub]
  float* bounds;                       // same shape: tau lies above, and the list misses no key of its share that does
  int tile_keys;                       // keys of a tile (kTreeTile, or less: whole boxes of the copies)
  int sample;                          // there is a sample
  int sample_tiles;                    // tiles of one group in it, at most
  float* classes;                      // [groups][rows][sample_tiles][4]: largest raw score of a lane quadrant
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

// Tiles of the launch's groups before group g (warp-cooperative; every lane gets the sum).
template <bool SAMPLE = false>
__device__ __forceinline__ int64_t tree_tiles_before(const TreeArgs& a, int g, int lane) {
  const int H = a.c.kv_heads;
  const int b0 = a.g0 / H, b1 = g / H;
  int64_t n = 0;
  for (int b = b0 + lane; b <= b1 && b < a.c.batch; b += 32) {
    const int lo = max(a.g0, b * H), hi = min(g, (b + 1) * H);
    n += (int64_t)(hi - lo) * tree_tiles<SAMPLE>(a, b);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

// The group that tile `t` of the launch's tile sequence lies in, and that group's first tile (warp-cooperative; t must
// lie in the sequence).
struct TreeAt {
  int g;
  int64_t first;
};
template <bool SAMPLE = false>
__device__ __forceinline__ TreeAt tree_find(const TreeArgs& a, int64_t t, int lane) {
  const int H = a.c.kv_heads;
  int64_t before = 0;
  for (int b0 = a.g0 / H; b0 < a.c.batch; b0 += 32) {
    const int b = b0 + lane;
    const int lo = max(a.g0, b * H), hi = min(a.g1, (b + 1) * H);
    const int per = b < a.c.batch && hi > lo ? tree_tiles<SAMPLE>(a, b) : 0;
    int64_t end = (int64_t)max(hi - lo, 0) * per;
    const int64_t mine = end;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t n = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += n;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + end > t);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int64_t start = before + __shfl_sync(0xffffffffu, end - mine, src);
      const int tiles = __shfl_sync(0xffffffffu, per, src), first = __shfl_sync(0xffffffffu, lo, src);
      const int64_t skip = (t - start) / tiles;
      return TreeAt{first + (int)skip, start + skip * tiles};
    }
    before += __shfl_sync(0xffffffffu, end, 31);
  }
  return TreeAt{a.g1, before};
}

// The tile sequence of W tiles in N pieces (N <= W): piece i is [i W / N, (i + 1) W / N).
struct TreeSplit {
  int64_t W;
  int N;
  __device__ __forceinline__ int64_t begin(int i) const { return i * W / N; }
  __device__ __forceinline__ int piece_of(int64_t tile) const { return (int)(((tile + 1) * N - 1) / W); }
};
__device__ __forceinline__ TreeSplit tree_split(int64_t W, int ranges) {
  TreeSplit s;
  s.W = W;
  s.N = (int)min((int64_t)ranges, W);
  return s;
}

__device__ __forceinline__ float max_nan(float a, float b) {      // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

}  // namespace ekv
