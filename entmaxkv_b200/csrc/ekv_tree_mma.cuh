// Tree attention, passes over K on the tensor cores (16-bit caches): S^T = K Q^T in tiles of 128 keys by N rows.
//
// Keys lie along M and rows along N, so N is the number of rows that share the KV head (16..256, padded to 16), nothing
// is padded to 128, and a warp of the epilogue holds 32 keys of one row per register.
//
// Roles of the 18 warps: 0-15 epilogue (four warpgroups that share the columns; they also lay the rows out for the
// products), 16 copies K tiles (cp.async.bulk.tensor, 128-byte swizzle: one box per tile of a dense cache, one per page
// of a block table), 17 issues the products.  Two to eight accumulators in TMEM.
//
// Bounds.  The sample keeps the largest score of every 32 keys that it looks at; the tau of those maxima (at most 256, in
// 64 classes or more) bounds the row's tau from below, far closer than the maximum - 1 does.  Without a sample the
// maxima of a piece's first tile take its place.  The bounds do not change during the pass, so the lists do not depend on
// timing.
//
// Candidates are rare, so a warp collects them in a queue (one append per lane and turn) and sorts 32 at a time into the
// lists of their rows.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "ekv_tree.cuh"

namespace ekv {

constexpr int kTmEpiWarps = 16;
constexpr int kTmEpiThreads = kTmEpiWarps * 32;
constexpr int kTmThreads = kTmEpiThreads + 64;
constexpr int kTmMaxRows = 256;        // rows per block
constexpr int kTmSub = 4;              // lists per row and piece: one per lane quadrant
constexpr int kTmMaxStages = 6;
constexpr int kTmMaxAcc = 8;           // accumulators: as many as fit the 512 columns of TMEM
constexpr int kTmQueue = 64;           // candidates that a warp collects
constexpr int kTmClasses = 32;         // class maxima per thread

struct TmSmem {                        // behind the operand tiles
  float thr[kTmMaxRows];               // raw score units (before zscale)
  int count[kTmMaxRows][kTmSub];
  float first[kTmSub][kTmMaxRows];     // no sample: maxima of the first tile
  uint2 queue[kTmEpiWarps][kTmQueue];
  unsigned char queue_row[kTmEpiWarps][kTmQueue];
  uint64_t full[kTmMaxStages], empty[kTmMaxStages], acc_full[kTmMaxAcc], acc_empty[kTmMaxAcc], q_full;
  uint32_t tmem;
  int abort;
};

struct TmShape {
  int n_rows;                          // rows of a block, a multiple of 16
  int acc_cols;                        // TMEM columns per accumulator
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
__device__ __forceinline__ void tm_wait(uint64_t* bar, uint32_t parity, TmSmem* s, int* status) {
  const uint32_t b = smem_addr(bar);
  if (tm_try(b, parity)) return;
  const long long start = clock64();
  while (!tm_try(b, parity)) {
    if (*(volatile int*)&s->abort) return;
    if (clock64() - start > (1ll << 32)) {       // some two seconds: a wait that ran out ends all others of the block
      *(volatile int*)&s->abort = 1;
      note_copy_timeout(status);
    }
  }
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
__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kTmEpiThreads) : "memory"); }

// A lower bound of the tau of scores (raw units; -inf: none) that `width` neighbouring lanes hold N each, by bisection
// that keeps its lower end.  Every lane of the warp takes part.
template <int N>
__device__ __forceinline__ float tm_bound(const float (&t)[N], int width, float zscale, float alpha) {
  float top = t[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = max_nan(top, t[i]);
  for (int o = width / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  const int kind = alpha_kind_of(alpha);
  const float beta = 1.f / (alpha - 1.f), unit = 1.f / zscale;
  float lo = top - unit, hi = top;
#pragma unroll 1
  for (int it = 0; it < 6; ++it) {
    const float mid = 0.5f * (lo + hi);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += entmax_weight(t[i] * zscale, mid * zscale, kind, beta);
    for (int o = width / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (sum >= 1.f) lo = mid; else hi = mid;
  }
  if (!(fabsf(top) < INFINITY)) return top == INFINITY ? INFINITY : -INFINITY;   // a NaN: everything is a candidate
  // the roundings of the scaling (2^-24 each) and of the sum: its relative error of 256 2^-24 moves tau by at most
  // (alpha - 1) 256 2^-24, as sum d^(beta-1) >= 1 where sum d^beta = 1
  return lo - 2e-5f * alpha * (fabsf(top) + unit);
}

__host__ __device__ inline size_t tm_smem_bytes(int rows, int head_dim, int stages) {
  return 1024 + (size_t)(rows + stages * kTreeTile) * head_dim * 2 + sizeof(TmSmem);
}

// Sorts the `n` <= 32 oldest candidates of the warp's queue, from place `at`, into their rows' lists.
__device__ __forceinline__ void tm_flush(TmSmem* s, int warp, int lane, int at, int n, uint2* lists, int64_t region) {
  const unsigned who = n >= 32 ? 0xffffffffu : (1u << n) - 1;
  if (lane < n) {
    const int place = (at + lane) & (kTmQueue - 1);
    const uint2 e = s->queue[warp][place];
    const int row = s->queue_row[warp][place];
    const unsigned same = __match_any_sync(who, row);
    const int rank = __popc(same & ((1u << lane) - 1));
    int* const count = &s->count[row][warp & 3];
    const int at0 = *count;
    __syncwarp(who);
    if (rank == 0) *count = at0 + __popc(same);
    lists[row * region + at0 + rank] = e;
  }
  __syncwarp();
}

// grid: ranges * row_blocks
template <typename T, int D, bool SAMPLE>
__global__ void __launch_bounds__(kTmThreads, 1)
    tree_scores_mma_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap k_map,
                           const TmShape sh) {
  constexpr int KB = D / 64;                               // 64-element blocks of a row
  constexpr int CPR = D / 8;                               // 16-byte chunks of a row
  constexpr uint32_t kStageBytes = kTreeTile * D * 2;
  constexpr uint32_t kFormat = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  extern __shared__ unsigned char tm_raw[];
  unsigned char* const base = tm_raw + ((1024 - (smem_addr(tm_raw) & 1023)) & 1023);
  unsigned char* const s_q = base;                         // [KB][n_rows][128 bytes]
  unsigned char* const s_k = base + (size_t)sh.n_rows * D * 2;
  TmSmem* const s = reinterpret_cast<TmSmem*>(s_k + (size_t)sh.stages * kStageBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n_rows = sh.n_rows;
  const int range = blockIdx.x / a.row_blocks, rb = blockIdx.x % a.row_blocks;
  const int H = a.c.kv_heads;
  const TreeSplit split = tree_split(tree_tiles_before<SAMPLE>(a, a.g1, lane), a.ranges);
  if (split.W == 0 || range >= split.N) return;
  const int64_t t_begin = split.begin(range), t_end = split.begin(range + 1);
  const TreeAt at = tree_find<SAMPLE>(a, t_begin, lane);
  const int row_first = a.row0 + rb * n_rows;
  const int n_acc = min(512 / sh.acc_cols, kTmMaxAcc);

  if (warp == kTmEpiWarps + 1) {
    if (lane == 0) {
      for (int i = 0; i < sh.stages; ++i) {
        mbar_init(&s->full[i], 1);
        mbar_init(&s->empty[i], 1);
      }
      for (int i = 0; i < n_acc; ++i) {
        mbar_init(&s->acc_full[i], 1);
        mbar_init(&s->acc_empty[i], kTmEpiWarps);
      }
      mbar_init(&s->q_full, 1);
      s->abort = 0;
      mbar_fence_init();
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s->tmem)),
                 "r"(n_acc * sh.acc_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tm_fence_before();
  __syncthreads();
  tm_fence_after();
  const uint32_t tmem = s->tmem;

  // the pieces of groups that this block scores: every role walks them alike
  int64_t g_first = at.first;
  TmRing stage, acc_ring;
  int n = 0;                                               // tiles so far
  int segment = 0;
  for (int g = at.g; g < a.g1 && g_first < t_end; ++g) {
    const int b = g / H, hkv = g % H;
    const int g_tiles = tree_tiles<SAMPLE>(a, b);
    if (g_tiles == 0) continue;
    const int tile0 = (int)(max(t_begin, g_first) - g_first), tile1 = (int)(min(t_end, g_first + g_tiles) - g_first);
    const int part = range - split.piece_of(g_first);
    const int len = tree_len(a, b), all_tiles = tree_all_tiles(a, b);
    const int live = min(tree_drafts(a, b) * a.group - row_first, min(a.rows - rb * n_rows, n_rows));
    g_first += g_tiles;
    if (live <= 0) continue;

    if (warp < kTmEpiWarps) {
      // ---- epilogue
      const int quad = warp & 3, wg = warp >> 2;
      const int64_t row_id = (int64_t)(g - a.g0) * a.rows + rb * n_rows;
      const uint32_t lane_base = tmem + ((uint32_t)quad << 21);          // lane 32 * quad in the upper half
      epi_sync();                                          // the previous segment's results are written out
      // the previous segment's products have all run (their accumulators were read): its rows may go
      for (int i = tid; i < n_rows * CPR; i += kTmEpiThreads) {
        const int row = i / CPR, c = i % CPR, r = row_first + row;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (row < live)
          x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.qs[0] +
                                              (int64_t)(hkv * a.group + r % a.group) * a.qs[1] +
                                              (int64_t)(r / a.group) * a.qs[2] + c * 8);
        *reinterpret_cast<uint4*>(s_q + (c / 8) * (n_rows * 128) + tm_swizzle(row, c % 8)) = x;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // plain stores, read by the tensor core
      epi_sync();
      if (tid == 0) tm_arrive(&s->q_full);
      if (!SAMPLE) {
        for (int i = tid; i < n_rows * kTmSub; i += kTmEpiThreads) (&s->count[0][0])[i] = 0;
        for (int i = tid; i < n_rows; i += kTmEpiThreads)
          if (i >= live || !a.sample) s->thr[i] = i < live ? -INFINITY : INFINITY;      // no candidates of padding rows
        if (a.sample) {
          // 2..32 lanes share a row's class maxima, 32 each; more than that many are folded by maximum
          int width = 2;
          while (width < 32 && width * 2 * n_rows <= kTmEpiThreads) width *= 2;
          const int n_classes = tree_tiles<true>(a, b) * 4, part_of = tid % width;
          for (int r0 = 0; r0 < live; r0 += kTmEpiThreads / width) {
            const int row = r0 + tid / width;
            const float4* const cls = reinterpret_cast<const float4*>(
                a.classes + (row_id + min(row, live - 1)) * a.sample_tiles * 4);
            float t[kTmClasses];
#pragma unroll
            for (int i = 0; i < kTmClasses; ++i) t[i] = -INFINITY;
            for (int f = 0; f < n_classes; f += kTmClasses * width)
#pragma unroll
              for (int i = 0; i < kTmClasses; i += 4) {
                const int q4 = (f + i * width) / 4 + part_of;
                if (q4 * 4 < n_classes) {
                  const float4 v = cls[q4];
                  t[i] = max_nan(t[i], v.x);
                  t[i + 1] = max_nan(t[i + 1], v.y);
                  t[i + 2] = max_nan(t[i + 2], v.z);
                  t[i + 3] = max_nan(t[i + 3], v.w);
                }
              }
            const float bound = tm_bound(t, width, a.zscale, a.alpha);
            if (part_of == 0 && row < live) s->thr[row] = bound;
          }
        }
        epi_sync();
      }
      uint2* const lists = a.entries + row_id * a.region + (int64_t)tile0 * kTreeTile +
                           (int64_t)quad * (tile1 - tile0) * (kTreeTile / kTmSub);
      int queue_at = 0, queued = 0;                        // this warp's candidates
      constexpr int kStep = kTmEpiWarps * 4;               // columns that the warpgroups take side by side
      for (int tile = tile0; tile < tile1; ++tile) {
        const int place = SAMPLE ? tree_sample_tile(tile, g_tiles, all_tiles) : tile;
        const int in_tile = quad * 32 + lane, key = place * a.tile_keys + in_tile;
        const bool exists = in_tile < a.tile_keys && key < len;
        tm_wait(&s->acc_full[acc_ring.at], acc_ring.parity, s, a.status);
        tm_fence_after();
        const uint32_t acc = lane_base + acc_ring.at * sh.acc_cols;
        float v[16], ahead[16];
        if (SAMPLE || (tile == tile0 && !a.sample)) {
          if (wg * 16 < n_rows) tm_load16(v, acc + wg * 16);
          for (int c0 = wg * 16; c0 < n_rows; c0 += kStep) {
            tm_load_wait();
            if (c0 + kStep < n_rows) tm_load16(ahead, acc + c0 + kStep);
            float mine = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float m = warp_max_nan(exists ? v[j] : -INFINITY);
              if (lane == j) mine = m;
            }
            if (SAMPLE) {
              if (lane < 16 && c0 + lane < live)
                a.classes[((row_id + c0 + lane) * a.sample_tiles + tile) * 4 + quad] = mine;
            } else if (lane < 16) {
              s->first[quad][c0 + lane] = mine;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = ahead[j];
          }
          if (!SAMPLE) {
            // no sample: the first tile's maxima give the piece's bounds, before it is read for candidates
            epi_sync();
            for (int row = tid; row < (live + 31) / 32 * 32; row += kTmEpiThreads) {
              float t[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) t[i] = s->first[i][min(row, live - 1)];
              const float bound = tm_bound(t, 1, a.zscale, a.alpha);
              if (row < live) s->thr[row] = bound;
            }
            epi_sync();
          }
        }
        if (!SAMPLE) {
          if (wg * 16 < n_rows) tm_load16(v, acc + wg * 16);
          for (int c0 = wg * 16; c0 < n_rows; c0 += kStep) {
            tm_load_wait();
            // bit j of a lane: its key is a candidate of row c0 + j (a NaN is one)
            uint32_t bits[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 t = *reinterpret_cast<const float4*>(&s->thr[c0 + 4 * j]);
              bits[j] = (v[4 * j] <= t.x ? 0u : 1u << 4 * j) | (v[4 * j + 1] <= t.y ? 0u : 2u << 4 * j) |
                        (v[4 * j + 2] <= t.z ? 0u : 4u << 4 * j) | (v[4 * j + 3] <= t.w ? 0u : 8u << 4 * j);
            }
            uint32_t mine = (bits[0] | bits[1]) | (bits[2] | bits[3]);
            if (!exists) mine = 0;
            if (c0 + 16 > live) mine &= (1u << max(live - c0, 0)) - 1;     // a NaN key under the padding rows
            unsigned who;
            while ((who = __ballot_sync(0xffffffffu, mine != 0)) != 0) {
              // every lane that has one appends a candidate to the queue
              if (mine) {
                const int j = __ffs(mine) - 1;
                mine &= mine - 1;
                const int to = (queue_at + queued + __popc(who & ((1u << lane) - 1))) & (kTmQueue - 1);
                s->queue[warp][to] = make_uint2(__float_as_uint(tm_pick(v, j) * a.zscale), (uint32_t)key);
                s->queue_row[warp][to] = (unsigned char)(c0 + j);
              }
              queued += __popc(who);
              __syncwarp();
              if (queued >= 32) {
                tm_flush(s, warp, lane, queue_at, 32, lists, a.region);
                queue_at += 32;
                queued -= 32;
              }
            }
            if (c0 + kStep < n_rows) tm_load16(v, acc + c0 + kStep);
          }
        }
        tm_fence_before();
        __syncwarp();
        if (lane == 0) tm_arrive(&s->acc_empty[acc_ring.at]);
        acc_ring.next(n_acc);
      }
      if (!SAMPLE) {
        tm_flush(s, warp, lane, queue_at, queued, lists, a.region);
        epi_sync();
        for (int i = tid; i < live * kTmSub; i += kTmEpiThreads) {
          const int row = i / kTmSub, sub = i % kTmSub;
          const int64_t o = (row_id + row) * a.max_parts * kTmSub + part * kTmSub + sub;
          a.counts[o] = s->count[row][sub];
          a.bounds[o] = s->thr[row] * a.zscale;
        }
      }
    } else if (warp == kTmEpiWarps) {
      // ---- copies of K: lane i takes box i of the tile (a page, or part of one; 64 elements wide)
      const int boxes = a.tile_keys / sh.box_rows * KB;
      for (int tile = tile0; tile < tile1; ++tile, ++n) {
        const int place = SAMPLE ? tree_sample_tile(tile, g_tiles, all_tiles) : tile;
        if (n >= sh.stages) tm_wait(&s->empty[stage.at], stage.parity ^ 1, s, a.status);
        if (lane == 0) mbar_expect_tx(&s->full[stage.at], (uint32_t)a.tile_keys * D * 2);
        __syncwarp();
        for (int i = lane; i < boxes; i += 32) {
          const int in_tile = i / KB * sh.box_rows, x = i % KB;
          const int key = place * a.tile_keys + in_tile;
          int row = key, block = b;
          if (a.c.block_table) {
            int page;
            a.by_page.divmod(key, page, row);
            // outside the pool, or behind the sequence: zeros
            block = key < len ? a.c.block_table[(int64_t)b * a.c.bt_stride + page] : -1;
            if ((unsigned)block >= (unsigned)a.c.num_blocks) block = a.c.num_blocks;
          }
          tm_copy_box(smem_addr(s_k) + stage.at * kStageBytes + x * (kTreeTile * 128) + in_tile * 128, &k_map, x * 64,
                      row, hkv, block, &s->full[stage.at]);
        }
        stage.next(sh.stages);
      }
    } else if (lane == 0) {
      // ---- products
      const uint32_t idesc = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((uint32_t)(n_rows >> 3) << 17) |
                             ((uint32_t)(kTreeTile >> 4) << 24);
      const uint64_t k_desc = tm_desc(smem_addr(s_k)), q_desc = tm_desc(smem_addr(s_q));
      tm_wait(&s->q_full, segment & 1, s, a.status);
      for (int tile = tile0; tile < tile1; ++tile, ++n) {
        tm_wait(&s->full[stage.at], stage.parity, s, a.status);
        if (n >= n_acc) tm_wait(&s->acc_empty[acc_ring.at], acc_ring.parity ^ 1, s, a.status);
        tm_fence_after();
        const uint64_t k0 = k_desc + (uint64_t)(stage.at * kStageBytes >> 4);
        const uint32_t d = tmem + acc_ring.at * sh.acc_cols;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)       // 32 bytes further in the 128-byte rows, then the next 64 elements
          tm_mma(d, k0 + (k / 4) * (kTreeTile * 128 >> 4) + k % 4 * 2, q_desc + (k / 4) * (n_rows * 128 >> 4) + k % 4 * 2,
                 idesc, k > 0);
        tm_commit(&s->empty[stage.at]);
        tm_commit(&s->acc_full[acc_ring.at]);
        stage.next(sh.stages);
        acc_ring.next(n_acc);
      }
    }
    ++segment;
  }
  if (warp == kTmEpiWarps + 1) {
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
  tm_fence_before();
  __syncthreads();
  tm_fence_after();
  if (warp == kTmEpiWarps + 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(n_acc * sh.acc_cols));
}

}  // namespace ekv
