// Tree attention, score pass on the tensor cores (16-bit caches): S^T = K Q^T in tiles of 128 keys by N rows.
//
// Keys lie along M and rows along N, so N is the number of rows that share the KV head (16..256, padded to 16), nothing
// is padded to 128, and a warp of the epilogue holds 32 keys of one row per register: one threshold per register, and a
// row whose 32 scores all lie under it costs one comparison.
//
// Roles of the 13 warps: 0-7 epilogue (two warpgroups that share the columns), 8-11 copy K tiles and the rows into
// shared memory (cp.async, 16 bytes a thread, any strides and page size, into the 128-byte swizzle that tcgen05.mma
// reads), 12 issues the products.  Accumulators are double-buffered in TMEM.
//
// Thresholds.  For any k keys whose scores are at least t, tau >= t - k^-(alpha-1): k equal scores t already use up
// the sum.  Each row keeps the largest candidate of 16 disjoint classes of keys (lane quadrant x tile mod 4); sorted as
// t_1 >= t_2 >= ..., max_k (t_k - k^-(alpha-1)) bounds tau from below for every alpha, much closer than t_1 - 1 alone:
// for normal scores a tenth of the candidates is left.  The thresholds change between tiles only, at points that the
// tile number fixes, so the lists do not depend on timing.
#pragma once

#include <type_traits>

#include "ekv_tree.cuh"

namespace ekv {

constexpr int kTmEpiWarps = 8, kTmCopyWarps = 4;
constexpr int kTmThreads = (kTmEpiWarps + kTmCopyWarps + 1) * 32;
constexpr int kTmMaxRows = 256;        // rows per block
constexpr int kTmSlots = 16;
constexpr int kTmSub = 4;              // lists per row and piece: one per lane quadrant
constexpr int kTmMaxStages = 6;

struct TmSmem {                        // behind the operand tiles
  float thr[kTmMaxRows];               // raw score units (before zscale)
  int count[kTmMaxRows][kTmSub];
  float kpow[kTmSlots];                // k^-(alpha-1) / zscale
  uint64_t full[kTmMaxStages], empty[kTmMaxStages], acc_full[2], acc_empty[2], q_free;
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ void tm_wait(uint64_t* bar, uint32_t parity, TmSmem* s, int* status) {
  if (*(volatile int*)&s->abort) return;
  if (!mbar_wait(bar, parity)) {       // a wait that ran out ends all others of the block
    *(volatile int*)&s->abort = 1;
    note_copy_timeout(status);
  }
}
__device__ __forceinline__ void tm_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void tm_copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void tm_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void tm_copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// the copies were made by ordinary stores as far as the tensor core is concerned
__device__ __forceinline__ void tm_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
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
__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// The row's threshold from its 16 class maxima.  Batcher's odd-even merge sort on registers.
__device__ __forceinline__ float tm_threshold(const float* slots, const float* kpow) {
  float t[kTmSlots];
#pragma unroll
  for (int i = 0; i < kTmSlots; ++i) t[i] = slots[i * kTmMaxRows];
#pragma unroll
  for (int lp = 0; lp < 4; ++lp)
#pragma unroll
    for (int lk = lp; lk >= 0; --lk)
#pragma unroll
      for (int i = 0; i < kTmSlots; ++i) {
        const int p = 1 << lp, k = 1 << lk, x = i - k % p;
        if (x >= 0 && x / k % 2 == 0 && i + k < kTmSlots && i / (2 * p) == (i + k) / (2 * p)) {
          const float hi = max_nan(t[i], t[i + k]);
          t[i + k] = fminf(t[i], t[i + k]);
          t[i] = hi;
        }
      }
  float thr = -INFINITY;
#pragma unroll
  for (int i = 0; i < kTmSlots; ++i) thr = max_nan(thr, t[i] - kpow[i]);
  // the roundings of k^-(alpha-1), of the difference and of the scaling
  return thr - 1e-6f * (fabsf(t[0]) + kpow[0]);
}

__host__ __device__ inline size_t tm_smem_bytes(int rows, int head_dim, int stages) {
  return 1024 + (size_t)(rows + stages * kTreeTile) * head_dim * 2 + sizeof(float) * kTmSlots * kTmMaxRows +
         sizeof(TmSmem);
}

// grid: ranges * row_blocks.  `n_rows`: rows of a block, a multiple of 16; `acc_cols`: TMEM columns per accumulator.
template <typename T, int D>
__global__ void __launch_bounds__(kTmThreads, 1)
    tree_scores_mma_kernel(const __grid_constant__ TreeArgs a, const int n_rows, const int acc_cols,
                           const int stages) {
  constexpr int CPR = D / 8;                               // 16-byte chunks of a row
  constexpr uint32_t kStageBytes = kTreeTile * D * 2;
  constexpr uint32_t kFormat = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  extern __shared__ unsigned char tm_raw[];
  unsigned char* const base = tm_raw + ((1024 - (smem_addr(tm_raw) & 1023)) & 1023);
  unsigned char* const s_q = base;                         // [D / 64][n_rows][128 bytes]
  unsigned char* const s_k = base + (size_t)n_rows * D * 2;
  float* const s_slots = reinterpret_cast<float*>(s_k + (size_t)stages * kStageBytes);   // [16][256]
  TmSmem* const s = reinterpret_cast<TmSmem*>(s_slots + kTmSlots * kTmMaxRows);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int range = blockIdx.x / a.row_blocks, rb = blockIdx.x % a.row_blocks;
  const int H = a.c.kv_heads;
  const TreeSplit split = tree_split(tree_tiles_before(a, a.g1, lane), a.ranges);
  if (split.W == 0 || range >= split.N) return;
  const int64_t t_begin = split.begin(range), t_end = split.begin(range + 1);
  const TreeAt at = tree_find(a, t_begin, lane);
  const int row_first = a.row0 + rb * n_rows;

  if (warp == kTmEpiWarps + kTmCopyWarps) {
    if (lane == 0) {
      for (int i = 0; i < stages; ++i) {
        mbar_init(&s->full[i], kTmCopyWarps * 32);
        mbar_init(&s->empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s->acc_full[i], 1);
        mbar_init(&s->acc_empty[i], kTmEpiWarps);
      }
      mbar_init(&s->q_free, 1);
      s->abort = 0;
      mbar_fence_init();
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s->tmem)),
                 "r"(2 * acc_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid < kTmSlots) s->kpow[tid] = powf((float)(tid + 1), 1.f - a.alpha) / a.zscale;
  tm_fence_before();
  __syncthreads();
  tm_fence_after();
  const uint32_t tmem = s->tmem;

  // the pieces of groups that this block scores: every role walks them alike
  int64_t g_first = at.first;
  int n = 0;                                               // tiles so far
  int segment = 0;
  int signalled = 0;                                       // copy warps: tiles reported as landed
  for (int g = at.g; g < a.g1 && g_first < t_end; ++g) {
    const int b = g / H, hkv = g % H;
    const int g_tiles = tree_tiles(a, b);
    if (g_tiles == 0) continue;
    const int tile0 = (int)(max(t_begin, g_first) - g_first), tile1 = (int)(min(t_end, g_first + g_tiles) - g_first);
    const int part = range - split.piece_of(g_first);
    const int len = tree_len(a, b);
    const int live = min(tree_drafts(a, b) * a.group - row_first, min(a.rows - rb * n_rows, n_rows));
    g_first += g_tiles;
    if (live <= 0) continue;

    if (warp < kTmEpiWarps) {
      // ---- epilogue
      const int quad = warp & 3, wg = warp >> 2;
      const int64_t row_id = (int64_t)(g - a.g0) * a.rows + rb * n_rows;
      uint2* const lists = a.entries + row_id * a.region + (int64_t)tile0 * kTreeTile +
                           (int64_t)quad * (tile1 - tile0) * (kTreeTile / kTmSub);
      epi_sync();                                          // the previous segment's counts are written out
      if (tid < n_rows) {
        s->thr[tid] = tid < live ? -INFINITY : INFINITY;
#pragma unroll
        for (int i = 0; i < kTmSub; ++i) s->count[tid][i] = 0;
      }
      for (int i = tid; i < kTmSlots * kTmMaxRows; i += kTmEpiWarps * 32) s_slots[i] = -INFINITY;
      epi_sync();
      const uint32_t lane_base = tmem + ((uint32_t)quad << 21);          // lane 32 * quad in the upper half
      for (int tile = tile0; tile < tile1; ++tile, ++n) {
        const int buf = n & 1;
        tm_wait(&s->acc_full[buf], (n >> 1) & 1, s, a.status);
        tm_fence_after();
        const int key = tile * kTreeTile + quad * 32 + lane;
        const bool exists = key < len;
        const bool partial = (tile + 1) * kTreeTile > len;
        const uint32_t acc = lane_base + buf * acc_cols;
        if (tile == tile0) {
          // the first tile's maxima give the first thresholds, before it is read for candidates
          for (int c0 = wg * 16; c0 < n_rows; c0 += 32) {
            float v[16];
            tm_load16(v, acc + c0);
            tm_load_wait();
            float mine = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float m = warp_max_nan(exists ? v[j] : -INFINITY);
              if (lane == j) mine = m;
            }
            if (lane < 16) s_slots[(quad * 4 + (tile & 3)) * kTmMaxRows + c0 + lane] = mine;
          }
          epi_sync();
          if (tid < live) s->thr[tid] = tm_threshold(s_slots + tid, s->kpow);
          epi_sync();
        }
        const int slot = (quad * 4 + (tile & 3)) * kTmMaxRows;
        for (int c0 = wg * 16; c0 < n_rows; c0 += 32) {
          float v[16];
          tm_load16(v, acc + c0);
          tm_load_wait();
          if (partial) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (!exists) v[j] = -INFINITY;
          }
#pragma unroll
          for (int j4 = 0; j4 < 16; j4 += 4) {
            const float4 t4 = *reinterpret_cast<const float4*>(&s->thr[c0 + j4]);
            const float t[4] = {t4.x, t4.y, t4.z, t4.w};
            bool any = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) any |= !(v[j4 + j] <= t[j]);     // a NaN is a candidate
            if (__any_sync(0xffffffffu, any)) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const unsigned hit = __ballot_sync(0xffffffffu, !(v[j4 + j] <= t[j]));
                const int row = c0 + j4 + j;
                if (hit && row < live) {                   // a NaN key is a candidate of the padding rows, too
                  const int at0 = s->count[row][quad];
                  if (hit >> lane & 1)
                    lists[row * a.region + at0 + __popc(hit & ((1u << lane) - 1))] =
                        make_uint2(__float_as_uint(v[j4 + j] * a.zscale), (uint32_t)key);
                  const float m = warp_max_nan(v[j4 + j]);
                  __syncwarp();
                  if (lane == 0) {
                    s->count[row][quad] = at0 + __popc(hit);
                    s_slots[slot + row] = max_nan(s_slots[slot + row], m);
                  }
                  __syncwarp();
                }
              }
            }
          }
        }
        tm_fence_before();
        __syncwarp();
        if (lane == 0) tm_arrive(&s->acc_empty[buf]);
        // new thresholds: often while they still rise, then every fourth tile
        const int done = tile - tile0 + 1;
        if (done < 4 || (done & 3) == 0) {
          epi_sync();
          if (tid < live) s->thr[tid] = tm_threshold(s_slots + tid, s->kpow);
          epi_sync();
        }
      }
      epi_sync();
      if (tid < live) {
        const int64_t o = (row_id + tid) * a.max_parts * kTmSub + part * kTmSub;
        const float bound = s->thr[tid] * a.zscale;
#pragma unroll
        for (int i = 0; i < kTmSub; ++i) {
          a.counts[o + i] = s->count[tid][i];
          float m = -INFINITY;
#pragma unroll
          for (int j = 0; j < 4; ++j) m = max_nan(m, s_slots[(i * 4 + j) * kTmMaxRows + tid]);
          a.maxima[o + i] = m * a.zscale;
          a.bounds[o + i] = bound;
        }
      }
    } else if (warp < kTmEpiWarps + kTmCopyWarps) {
      // ---- copies
      const int ct = tid - kTmEpiWarps * 32;
      if (segment) {
        // the rows' buffer is free once the last product of the previous segment has run, which needs every tile
        tm_copy_wait<0>();
        tm_proxy_fence();
        for (; signalled < n; ++signalled) tm_arrive(&s->full[signalled % stages]);
        tm_wait(&s->q_free, (segment - 1) & 1, s, a.status);
      }
      const uint32_t q_dst = smem_addr(s_q);
      for (int i = ct; i < n_rows * CPR; i += kTmCopyWarps * 32) {
        const int row = i / CPR, c = i % CPR, r = row_first + row;
        const bool ok = row < live;
        const T* src = static_cast<const T*>(a.q);
        if (ok)
          src += b * a.qs[0] + (int64_t)(hkv * a.group + r % a.group) * a.qs[1] + (int64_t)(r / a.group) * a.qs[2] + c * 8;
        tm_copy16(q_dst + (c / 8) * (n_rows * 128) + tm_swizzle(row, c % 8), src, ok);
      }
      const int c = ct % CPR;
      for (int tile = tile0; tile < tile1; ++tile, ++n) {
        const int st = n % stages;
        if (n >= stages) tm_wait(&s->empty[st], (n / stages - 1) & 1, s, a.status);
        const uint32_t dst = smem_addr(s_k) + st * kStageBytes + (c / 8) * (kTreeTile * 128);
        constexpr int RPI = kTmCopyWarps * 32 / CPR;       // keys per turn of the copy warps
#pragma unroll 8
        for (int i = 0; i < kTreeTile / RPI; ++i) {
          const int row = i * RPI + ct / CPR, key = tile * kTreeTile + row;
          size_t off = 0;
          bool ok = key < len;
          if (ok) {
            int page, in_page;
            a.by_page.divmod(key, page, in_page);
            ok = kv_page_offset(a.c, b, hkv, page, off);
            off += (size_t)in_page * D + c * 8;
          }
          tm_copy16(dst + tm_swizzle(row, c % 8), static_cast<const T*>(a.c.k) + (ok ? off : 0), ok);
        }
        tm_copy_commit();
        // all but the newest stages - 1 tiles have landed
        if (n - signalled >= stages - 1) {
          switch (stages) {
            case 2: tm_copy_wait<1>(); break;
            case 3: tm_copy_wait<2>(); break;
            case 4: tm_copy_wait<3>(); break;
            case 5: tm_copy_wait<4>(); break;
            default: tm_copy_wait<5>(); break;
          }
          tm_proxy_fence();
          tm_arrive(&s->full[signalled % stages]);
          ++signalled;
        }
      }
    } else if (lane == 0) {
      // ---- products
      const uint32_t idesc = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((uint32_t)(n_rows >> 3) << 17) |
                             ((uint32_t)(kTreeTile >> 4) << 24);
      for (int tile = tile0; tile < tile1; ++tile, ++n) {
        const int st = n % stages, buf = n & 1;
        tm_wait(&s->full[st], (n / stages) & 1, s, a.status);
        if (n >= 2) tm_wait(&s->acc_empty[buf], ((n >> 1) - 1) & 1, s, a.status);
        tm_fence_after();
        const uint32_t k0 = smem_addr(s_k) + st * kStageBytes, q0 = smem_addr(s_q);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t in = (k % 4) * 32;
          tm_mma(tmem + buf * acc_cols, tm_desc(k0 + (k / 4) * (kTreeTile * 128) + in),
                 tm_desc(q0 + (k / 4) * (n_rows * 128) + in), idesc, k > 0);
        }
        tm_commit(&s->empty[st]);
        tm_commit(&s->acc_full[buf]);
        if (tile + 1 == tile1) tm_commit(&s->q_free);
      }
    }
    ++segment;
  }
  if (warp >= kTmEpiWarps && warp < kTmEpiWarps + kTmCopyWarps) {
    tm_copy_wait<0>();
    tm_proxy_fence();
    for (; signalled < n; ++signalled) tm_arrive(&s->full[signalled % stages]);
  } else if (warp == kTmEpiWarps + kTmCopyWarps) {
    if (lane == 0 && segment) {        // no arrival may come after the block's end
      for (int i = max(0, n - stages); i < n; ++i) tm_wait(&s->empty[i % stages], (i / stages) & 1, s, a.status);
      tm_wait(&s->q_free, (segment - 1) & 1, s, a.status);
    }
    __syncwarp();
  }
  tm_fence_before();
  __syncthreads();
  tm_fence_after();
  if (warp == kTmEpiWarps + kTmCopyWarps)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * acc_cols));
}

}  // namespace ekv
