// Tree attention, passes over K on the tensor cores (16-bit caches): S = Q K^T in tiles of 128 keys.
//
// Rows lie along M, one per TMEM lane, so a thread of the epilogue owns a row: its bound, its candidates' count and its
// place in the list are registers, and a score costs half a packed subtraction and a funnel shift (the sign says whether
// it lies under the bound).  Up to 64 (32) rows are laid out two (four) times over the 128 lanes, and each copy reads
// its own half (quarter) of a tile's columns; from 129 rows on there are two row tiles.
//
// Roles of the 20 warps: 0-15 epilogue (four warpgroups: every fourth tile each, or, with two row tiles, half of one of
// them each; they also lay the rows out for the products), 16-18 copy K tiles (cp.async.bulk.tensor, 128-byte swizzle:
// one box per tile of a dense cache, one per page of a block table, times two for 128 elements; a warp issues one in
// about 110 cycles, hence three of them), 19 issues the products.  Two or four accumulators in TMEM.
//
// Bounds.  The sample keeps the largest score of every 32 keys that it looks at; the tau of those maxima bounds the row's
// tau from below, far closer than the maximum - 1 does.  The bounds do not change during the pass, so the lists do not
// depend on timing.  Short sequences have no sample: there all scores are written out, which is less than a second launch
// costs.
//
// Measured on a B200 (a launch alone): 8 sequences of 17k to 32k tokens, 64 rows per KV head, 8 heads of 128: sample 20 us,
// pass 80 us, 387 MB at 4.8 TB/s, 1.2k cycles a tile where it streams; one sequence of 131k tokens, 512 rows per KV head
// (two blocks of rows share each K tile through L2): pass 172 us.  At half that length 101 us, 137 MB from memory, the tensor
// pipe 33 % and the issue slots 56 % busy: about 1.7k slots a tile of 128 keys by 256 rows beside 1.0k cycles of products,
// most of them the epilogue's comparisons and appends.  With keys along the lanes instead of rows the passes took 1.2 and 1.8
// times as long.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "ekv_tree.cuh"

namespace ekv {

constexpr int kTmEpiWarps = 16;
constexpr int kTmEpiThreads = kTmEpiWarps * 32;
constexpr int kTmCopyWarps = 3;
constexpr int kTmMmaWarp = kTmEpiWarps + kTmCopyWarps;
constexpr int kTmThreads = (kTmMmaWarp + 1) * 32;
constexpr int kTmMaxRows = 256;        // rows per block
constexpr int kTmMaxStages = 6;
constexpr int kTmMaxAcc = 4;           // accumulators

enum TmMode { TM_SAMPLE, TM_LISTS, TM_DENSE };

struct TmSmem {                        // behind the operand tiles
  uint64_t full[kTmMaxStages], empty[kTmMaxStages], acc_full[kTmMaxAcc], acc_empty[kTmMaxAcc], q_full;
  uint32_t tmem;
  int abort;
};

struct TmShape {
  int n_rows;                          // rows of a block
  int row_tiles;                       // 1 or 2
  int copies;                          // 1, 2 or 4 (one row tile)
  int stages;
  int box_rows;                        // keys per copy
};

__device__ __forceinline__ bool tm_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(20000u)
      : "memory");
  return ok;
}
// false: a wait of the block ran out.  From then on nothing more is copied, the other waits end at once, and the launch's
// results are undefined (the status says so).
__device__ __forceinline__ bool tm_wait(uint64_t* bar, uint32_t parity, TmSmem* s, int* status) {
  const uint32_t b = smem_addr(bar);
  if (tm_try(b, parity)) return true;
  const long long start = clock64();
  while (!tm_try(b, parity)) {
    if (*(volatile int*)&s->abort) return false;
    if (clock64() - start > (1ll << 32)) {       // some two seconds
      *(volatile int*)&s->abort = 1;
      note_copy_timeout(status);
    }
  }
  return true;
}
// a place in a ring of `size` barriers and the parity of its current turn
struct TmRing {
  int at = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next(int size) {
    if (++at == size) {
      at = 0;
      parity ^= 1;
    }
  }
};
__device__ __forceinline__ void tm_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void tm_copy_box(uint32_t dst, const CUtensorMap* map, int x, int row, int head, int block,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(dst),
      "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(row), "r"(head), "r"(block)
      : "memory");
}
__device__ __forceinline__ void tm_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}
__device__ __forceinline__ void tm_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// operand tile: rows of 128 bytes in the 128-byte swizzle, K-major; 8 rows = 1024 bytes
__device__ __forceinline__ uint64_t tm_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// byte offset of 16-byte chunk `c` (of the row's 64 elements) of row `r` in such a tile
__device__ __forceinline__ uint32_t tm_swizzle(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

__device__ __forceinline__ void tm_load16(float (&v)[16], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void tm_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// (a0, a1) - (b0, b1)
__device__ __forceinline__ void tm_sub2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\t"
      "mov.b64 y, {%4, %5};\n\t"
      "sub.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
// v[j] for a j that differs from lane to lane
__device__ __forceinline__ float tm_pick(const float (&v)[16], int j) {
  float a[8], b[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = j & 1 ? v[2 * i + 1] : v[2 * i];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = j & 2 ? a[2 * i + 1] : a[2 * i];
  const float c0 = j & 4 ? b[1] : b[0], c1 = j & 4 ? b[3] : b[2];
  return j & 8 ? c1 : c0;
}
__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kTmEpiThreads) : "memory"); }

__host__ __device__ inline size_t tm_smem_bytes(int row_tiles, int head_dim, int stages) {
  return 1024 + (size_t)(row_tiles + stages) * kTreeTile * head_dim * 2 + sizeof(TmSmem);
}

// The rows' bounds from the sample: a warp per row; each lane folds its share of the class maxima into 16, and bisection
// that keeps its lower end gives a bound of the tau of all of them.
__global__ void __launch_bounds__(256) tree_bounds_kernel(const __grid_constant__ TreeArgs a, const int64_t n_rows) {
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  tree_let_next_start();
  if (id >= n_rows) return;
  const int gl = (int)((unsigned)id / (unsigned)a.rows), b = (a.g0 + gl) / a.c.kv_heads;
  const int n = tree_tiles<true>(a, b) * 4;
  const bool live = (a.row0 + (int)id - gl * a.rows) / a.group < tree_drafts(a, b);
  static_assert(kSampleTiles * 4 == 16 * 32, "a lane holds 16 class maxima");
  tree_wait_for_previous();
  if (!live || n == 0) return;
  const float* const cls = a.classes + id * a.sample_tiles * 4;
  float t[16];                                   // at most kSampleTiles * 4 = 16 * 32 maxima
#pragma unroll
  for (int i = 0; i < 16; ++i) t[i] = cls[min(i * 32 + lane, n - 1)];
#pragma unroll
  for (int i = 0; i < 16; ++i) t[i] = i * 32 + lane < n ? t[i] * a.zscale : -INFINITY;
  float top = t[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) top = max_nan(top, t[i]);
  top = warp_max_nan(top);
  const int kind = alpha_kind_of(a.alpha);
  const float beta = 1.f / (a.alpha - 1.f);
  float lo = top - 1.f, hi = top;
#pragma unroll 1
  for (int it = 0; it < 8; ++it) {
    const float mid = 0.5f * (lo + hi);
    float sum = 0.f;
    if (kind == 1) {                             // alpha 1.5, the usual one, without a branch per score
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float d = fmaxf(t[i] - mid, 0.f);
        sum = fmaf(d, d, sum);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < n; i += 32)
        if (i + lane < n) sum += entmax_weight(cls[i + lane] * a.zscale, mid, kind, beta);
    }
    if (warp_sum(sum) >= 1.f) lo = mid; else hi = mid;
  }
  // the roundings of the scaling (2^-24 each) and of the sum: its relative error of 512 2^-24 moves tau by at most
  // (alpha - 1) 512 2^-24, as sum d^(beta-1) >= 1 where sum d^beta = 1.  A NaN: everything is a candidate
  float bound = (lo - 4e-5f * a.alpha * (fabsf(top) + 1.f)) / a.zscale;
  if (!(fabsf(top) < INFINITY)) bound = top == INFINITY ? INFINITY : -INFINITY;
  if (lane == 0) a.row_bounds[id] = bound;
}

// grid: ranges * row_blocks
template <typename T, int D, int MODE>
__global__ void __launch_bounds__(kTmThreads, 1)
    tree_scores_mma_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap k_map,
                           const TmShape sh) {
  constexpr bool SAMPLE = MODE == TM_SAMPLE;
  constexpr int KB = D / 64;                               // 64-element blocks of a row
  constexpr int CPR = D / 8;                               // 16-byte chunks of a row
  constexpr uint32_t kTileBytes = kTreeTile * D * 2;
  constexpr uint32_t kFormat = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  extern __shared__ unsigned char tm_raw[];
  unsigned char* const base = tm_raw + ((1024 - (smem_addr(tm_raw) & 1023)) & 1023);
  unsigned char* const s_q = base;                         // [row_tiles][KB][128][128 bytes]
  unsigned char* const s_k = base + (size_t)sh.row_tiles * kTileBytes;
  TmSmem* const s = reinterpret_cast<TmSmem*>(s_k + (size_t)sh.stages * kTileBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int range = blockIdx.x / a.row_blocks, rb = blockIdx.x % a.row_blocks;
  const int H = a.c.kv_heads;
  tree_let_next_start();
  const TreeRange at = tree_range<SAMPLE>(a, range, lane);
  if (at.t_begin == at.t_end) {
    if (MODE == TM_LISTS) tree_wait_for_previous();        // nothing ends before what it was launched behind
    return;
  }
  const int t_begin = at.t_begin, t_end = at.t_end;
  const int row_first = a.row0 + rb * sh.n_rows;
  const int n_acc = sh.row_tiles == 2 ? 2 : 4, acc_cols = sh.row_tiles * kTreeTile;      // 512 columns: all of TMEM

  if (warp == kTmMmaWarp) {
    if (lane == 0) {
      for (int i = 0; i < sh.stages; ++i) {
        mbar_init(&s->full[i], 1);
        mbar_init(&s->empty[i], 1);
      }
      for (int i = 0; i < n_acc; ++i) {
        mbar_init(&s->acc_full[i], 1);
        mbar_init(&s->acc_empty[i], sh.row_tiles == 2 ? kTmEpiWarps : 4);
      }
      mbar_init(&s->q_full, 1);
      s->abort = 0;
      mbar_fence_init();
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s->tmem)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tm_fence_before();
  __syncthreads();
  tm_fence_after();
  const uint32_t tmem = s->tmem;

  // the pieces of groups that this block scores: every role walks them alike
  int g_first = at.first;
  TmRing stage, acc_ring;
  int n = 0;                                               // tiles so far
  int segment = 0;
  bool go = true;                                          // (copies only) no wait ran out
  for (int g = at.g; g < a.g1 && g_first < t_end && go; ++g) {
    const int b = g / H, hkv = g % H;
    const int g_tiles = tree_tiles<SAMPLE>(a, b);
    if (g_tiles == 0) continue;
    const int tile0 = max(t_begin, g_first) - g_first, tile1 = min(t_end, g_first + g_tiles) - g_first;
    const int part = range - at.split.piece_of(g_first);
    const int len = tree_len(a, b), all_tiles = tree_all_tiles(a, b);
    const int live = min(tree_drafts(a, b) * a.group - row_first, min(a.rows - rb * sh.n_rows, sh.n_rows));
    g_first += g_tiles;
    if (live <= 0) continue;

    if (warp < kTmEpiWarps) {
      // ---- epilogue
      const int quad = warp & 3, wg = warp >> 2;
      const int64_t row_id = (int64_t)(g - a.g0) * a.rows + rb * sh.n_rows;
      const int per_copy = kTreeTile / sh.copies;          // lanes of a copy
      epi_sync();
      // the previous segment's products have all run (their accumulators were read): its rows may go
      for (int i = tid; i < sh.row_tiles * kTreeTile * CPR; i += kTmEpiThreads) {
        const int slot = i / CPR, c = i % CPR, in_tile = slot % kTreeTile;
        const int row = slot / kTreeTile * kTreeTile + in_tile % per_copy, r = row_first + row;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (row < live)
          x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.qs[0] +
                                              (int64_t)(hkv * a.group + r % a.group) * a.qs[1] +
                                              (int64_t)(r / a.group) * a.qs[2] + c * 8);
        *reinterpret_cast<uint4*>(s_q + slot / kTreeTile * kTileBytes + (c / 8) * (kTreeTile * 128) +
                                  tm_swizzle(in_tile, c % 8)) = x;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // plain stores, read by the tensor core
      epi_sync();
      if (tid == 0) tm_arrive(&s->q_full);
      if (MODE == TM_LISTS && segment == 0) tree_wait_for_previous();    // the bounds; K and the rows need no waiting
      // this thread's row, its columns, and which tiles are its warpgroup's
      const int row_tile = sh.row_tiles == 2 ? wg & 1 : 0;
      const int in_tile = quad * 32 + lane, row = row_tile * kTreeTile + in_tile % per_copy;
      const int cols = sh.row_tiles == 2 ? kTreeTile / 2 : per_copy;
      const int col0 = sh.row_tiles == 2 ? (wg >> 1) * cols : in_tile / per_copy * cols;
      const int turn = sh.row_tiles == 2 ? 1 : 4;          // a warpgroup takes every turn-th tile
      const bool ok = row < live;
      const float thr = MODE == TM_LISTS && ok ? a.row_bounds[row_id + row] : INFINITY;
      const int list = sh.row_tiles == 2 ? wg >> 1 : in_tile / per_copy * 4 + wg;
      uint2* const out = a.entries + (row_id + (ok ? row : 0)) * a.region;
      uint2* const first = MODE == TM_LISTS ? out + tree_list_place(a, tile0, part, tile1 - tile0, list) : nullptr;
      uint2* next = first;
      if (turn == 4) {                                     // this warpgroup's first tile
        for (int i = 0; i < ((wg - n % 4) & 3) && i < tile1 - tile0; ++i) acc_ring.next(n_acc);
      }
      for (int tile = tile0 + (turn == 4 ? (wg - n % 4) & 3 : 0); tile < tile1; tile += turn) {
        const int place = SAMPLE ? tree_sample_tile(tile, g_tiles, all_tiles) : tile;
        const int key0 = place * a.tile_keys;
        const int valid = min(a.tile_keys, len - key0);    // columns that are keys
        tm_wait(&s->acc_full[acc_ring.at], acc_ring.parity, s, a.status);
        tm_fence_after();
        const uint32_t acc = tmem + ((uint32_t)quad << 21) + acc_ring.at * acc_cols + row_tile * kTreeTile;
        float v[16], best = -INFINITY;
        for (int c0 = col0; c0 < col0 + cols; c0 += 16) {
          tm_load16(v, acc + c0);
          tm_load_wait();
          if (SAMPLE) {
#pragma unroll
            for (int j = 0; j < 16; ++j) best = max_nan(best, c0 + j < valid ? v[j] : -INFINITY);
            if (c0 & 16) {
              if (ok) a.classes[((row_id + row) * a.sample_tiles + tile) * 4 + c0 / 32] = best;
              best = -INFINITY;
            }
          } else if (MODE == TM_DENSE) {
            float* const to = reinterpret_cast<float*>(out) + a.region + key0 + c0;
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (ok && c0 + j < valid) to[j] = v[j] * a.zscale;
          } else {
            // v - thr: a candidate has no sign bit (a NaN has none either).  The signs are shifted into four words of four
            uint32_t sign[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float d[4];
              tm_sub2(d[0], d[1], v[4 * j], v[4 * j + 1], thr, thr);
              tm_sub2(d[2], d[3], v[4 * j + 2], v[4 * j + 3], thr, thr);
              sign[j] = __float_as_uint(d[0]) >> 31;
#pragma unroll
              for (int i = 1; i < 4; ++i) sign[j] = __funnelshift_l(__float_as_uint(d[i]), sign[j], 1);
            }
            // bit 15 - j: column c0 + j is a candidate
            uint32_t mine = ~((sign[0] << 12) | (sign[1] << 8) | (sign[2] << 4) | sign[3]) & 0xffffu;
            if (c0 + 16 > valid) mine &= 0xffff0000u >> max(valid - c0, 0);
            if (!ok) mine = 0;
            while (__any_sync(0xffffffffu, mine != 0)) {
              if (mine) {
                const int bit = 31 - __clz(mine), j = 15 - bit;
                mine &= ~(1u << bit);
                *next++ = make_uint2(__float_as_uint(tm_pick(v, j) * a.zscale), (uint32_t)(key0 + c0 + j));
              }
            }
          }
        }
        tm_fence_before();
        __syncwarp();
        if (lane == 0) tm_arrive(&s->acc_empty[acc_ring.at]);
        for (int i = 0; i < turn && tile + i < tile1; ++i) acc_ring.next(n_acc);
      }
      n += tile1 - tile0;
      if (MODE == TM_LISTS && ok) {
        const int64_t o = ((row_id + row) * a.max_parts + part) * a.sub + list;
        a.counts[o] = (int)(next - first);
        a.bounds[o] = thr * a.zscale;
      }
    } else if (warp < kTmMmaWarp) {
      // ---- copies of K: the warps take turns at the boxes of a tile (a page, or part of one; 64 elements wide)
      const int first_box = warp - kTmEpiWarps + lane * kTmCopyWarps;
      const int boxes = a.tile_keys / sh.box_rows * KB;
      for (int tile = tile0; tile < tile1; ++tile, ++n) {
        const int place = SAMPLE ? tree_sample_tile(tile, g_tiles, all_tiles) : tile;
        if (n >= sh.stages) go = tm_wait(&s->empty[stage.at], stage.parity ^ 1, s, a.status);
        if (first_box == 0 && go) mbar_expect_tx(&s->full[stage.at], (uint32_t)a.tile_keys * D * 2);
        go = __all_sync(0xffffffffu, go);
        if (!go) break;
        for (int i = first_box; i < boxes; i += 32 * kTmCopyWarps) {
          const int in_tile = i / KB * sh.box_rows, x = i % KB;
          const int key = place * a.tile_keys + in_tile;
          int row = key, block = b;
          if (a.c.block_table) {
            int page;
            a.by_page.divmod(key, page, row);
            // behind the sequence, or (reported) outside the pool: zeros
            block = key < len ? a.c.block_table[(int64_t)b * a.c.bt_stride + page] : -1;
            if ((unsigned)block >= (unsigned)a.c.num_blocks) {
              block = a.c.num_blocks;
              if (key < len && a.status) atomicOr(a.status, EKV_STATUS_PAGE_RANGE);
            }
          }
          tm_copy_box(smem_addr(s_k) + stage.at * kTileBytes + x * (kTreeTile * 128) + in_tile * 128, &k_map, x * 64,
                      row, hkv, block, &s->full[stage.at]);
        }
        stage.next(sh.stages);
      }
    } else if (lane == 0) {
      // ---- products
      constexpr uint32_t idesc = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((uint32_t)(kTreeTile >> 3) << 17) |
                                 ((uint32_t)(kTreeTile >> 4) << 24);
      const uint64_t k_desc = tm_desc(smem_addr(s_k)), q_desc = tm_desc(smem_addr(s_q));
      tm_wait(&s->q_full, segment & 1, s, a.status);
      for (int tile = tile0; tile < tile1; ++tile, ++n) {
        tm_wait(&s->full[stage.at], stage.parity, s, a.status);
        if (n >= n_acc) tm_wait(&s->acc_empty[acc_ring.at], acc_ring.parity ^ 1, s, a.status);
        tm_fence_after();
        const uint64_t k0 = k_desc + (uint64_t)(stage.at * kTileBytes >> 4);
        for (int m = 0; m < sh.row_tiles; ++m) {
          const uint64_t q0 = q_desc + (uint64_t)(m * kTileBytes >> 4);
          const uint32_t d = tmem + acc_ring.at * acc_cols + m * kTreeTile;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {   // 32 bytes further in the 128-byte rows, then the next 64 elements
            const uint64_t in = (k / 4) * (kTreeTile * 128 >> 4) + k % 4 * 2;
            tm_mma(d, q0 + in, k0 + in, idesc, k > 0);
          }
        }
        tm_commit(&s->empty[stage.at]);
        tm_commit(&s->acc_full[acc_ring.at]);
        stage.next(sh.stages);
        acc_ring.next(n_acc);
      }
    }
    ++segment;
  }
  if (warp == kTmMmaWarp) {
    if (lane == 0)                     // no arrival may come after the block's end: the last product of every stage
      for (int i = min(n, sh.stages); i > 0; --i) {
        TmRing last = stage;
        last.at -= i;
        if (last.at < 0) {
          last.at += sh.stages;
          last.parity ^= 1;
        }
        tm_wait(&s->empty[last.at], last.parity, s, a.status);
      }
    __syncwarp();
  }
  // after a wait that ran out: copies and products on their way still use this block's memory, so it stays some 8 ms longer
  if (warp >= kTmEpiWarps && *(volatile int*)&s->abort)
    for (const long long start = clock64(); clock64() - start < (1ll << 24);) __nanosleep(1000);
  if (MODE == TM_LISTS) tree_wait_for_previous();
  tm_fence_before();
  __syncthreads();
  tm_fence_after();
  if (warp == kTmMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

}  // namespace ekv
