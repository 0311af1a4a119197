// Several tokens per sequence written into the cache, with the statistics of every page that they touch.
//
// Row i < counts[b] of sequence b is row index[b, i] (or i) of k_new / v_new and lands at position start[b] + i.  A page
// is handled by LPR lanes, one 16-byte column each: the lane gathers the page's rows - those already in the cache and
// the new ones - into registers, stores the new ones, and forms the column's statistics from the same registers, so each
// new row is read once and written once and an old row is read only where it shares the first page.  Bound by memory.
#include "ekv_page_stats.cuh"

namespace ekv {

struct ExtendArgs {
  const void* k_new;
  const void* v_new;
  int64_t sb, sh, st;            // element strides of k_new and v_new: batch, head, token
  int tokens;
  const int* counts;             // [B] or null: all `tokens`
  const int* index;              // [B, tokens] or null
  int64_t index_sb;
  const int* start;              // [B] or null: the current lengths
  int* counters;
  int* status;
};

constexpr int kExtendThreads = 256;
constexpr int kExtendRows = 16;  // rows of a page held in registers at once

// grid: (B * H_kv, page groups)
template <typename T, int D>
__global__ void __launch_bounds__(kExtendThreads) extend_kernel(const __grid_constant__ ekv_cache_desc c,
                                                                const __grid_constant__ ExtendArgs a) {
  constexpr int EPL = ElemTraits<T>::EPL;
  constexpr int LPR = D / EPL;
  const int b = blockIdx.x / c.kv_heads, h = blockIdx.x % c.kv_heads;
  const int P = c.page_size;
  const int room = (int)min((int64_t)c.capacity, (int64_t)c.page_capacity * P);
  const int now = min(max(c.seq_lens[b], 0), room);   // every block of the sequence reads it before the last replaces it
  int flag = 0;
  int start = now, n = a.tokens;
  if (a.start) {
    start = min(max(a.start[b], 0), now);
    if (start != a.start[b]) flag = EKV_STATUS_TOKENS;
  }
  if (a.counts) {
    n = min(max(a.counts[b], 0), a.tokens);
    if (n != a.counts[b]) flag = EKV_STATUS_TOKENS;
  }
  if (n > room - start) {
    n = room - start;
    flag |= EKV_STATUS_CAPACITY;
  }
  const int end = start + n;
  const int page0 = start / P;
  const int64_t page64 = page0 + ((int64_t)blockIdx.y * kExtendThreads + threadIdx.x) / LPR;
  const int col = threadIdx.x % LPR * EPL;
  // a rewind without new rows still leaves its page with fewer rows
  if (page64 * P < end && (n > 0 || start < now)) {
    const int page = (int)page64;
    size_t off;
    if (kv_page_offset(c, b, h, page, off)) {
      T* const kb = static_cast<T*>(c.k) + off + col;
      T* const vb = static_cast<T*>(c.v) + off + col;
      const T* const kn = static_cast<const T*>(a.k_new) + b * a.sb + h * a.sh + col;
      const T* const vn = static_cast<const T*>(a.v_new) + b * a.sb + h * a.sh + col;
      const int64_t r0 = (int64_t)page * P;
      const int rows = (int)min((int64_t)P, end - r0);
      auto source = [&](int64_t pos) -> int64_t {      // element offset of the new row at position pos
        int i = (int)(pos - start);
        if (a.index) {
          const int j = a.index[b * a.index_sb + i];
          i = min(max(j, 0), a.tokens - 1);
          if (i != j) flag |= EKV_STATUS_TOKENS;
        }
        return i * a.st;
      };
      ColumnStats<T> st;
      st.begin();
      if (rows <= kExtendRows) {
        uint4 k[kExtendRows], v[kExtendRows];
#pragma unroll
        for (int i = 0; i < kExtendRows; ++i)
          if (i < rows) {
            if (r0 + i < start) {
              k[i] = *reinterpret_cast<const uint4*>(kb + (size_t)i * D);
            } else {
              const int64_t s = source(r0 + i);
              k[i] = ld_stream(kn + s);
              v[i] = ld_stream(vn + s);
            }
          }
#pragma unroll
        for (int i = 0; i < kExtendRows; ++i)
          if (i < rows) {
            if (r0 + i >= start) {
              *reinterpret_cast<uint4*>(kb + (size_t)i * D) = k[i];
              *reinterpret_cast<uint4*>(vb + (size_t)i * D) = v[i];
            }
            st.first_pass(k[i]);
          }
        st.middle((float)rows);
#pragma unroll
        for (int i = 0; i < kExtendRows; ++i)
          if (i < rows) st.second_pass(k[i]);
      } else {
        for (int i = 0; i < rows; ++i) {
          uint4 k;
          if (r0 + i < start) {
            k = *reinterpret_cast<const uint4*>(kb + (size_t)i * D);
          } else {
            const int64_t s = source(r0 + i);
            k = ld_stream(kn + s);
            *reinterpret_cast<uint4*>(kb + (size_t)i * D) = k;
            *reinterpret_cast<uint4*>(vb + (size_t)i * D) = ld_stream(vn + s);
          }
          st.first_pass(k);
        }
        st.middle((float)rows);
        // this lane re-reads only the column that it wrote itself
        for (int i = 0; i < rows; ++i) st.second_pass(*reinterpret_cast<const uint4*>(kb + (size_t)i * D));
      }
      const size_t mo = b * c.meta_stride_b + h * c.meta_stride_h + (size_t)page * D + col;
      st.finish((float)rows, static_cast<T*>(c.k_min) + mo, static_cast<T*>(c.k_max) + mo,
                static_cast<T*>(c.k_mean) + mo, static_cast<T*>(c.k_std) + mo);
    }
  }
  if (flag) atomicOr(a.status, flag);

  // the last block of the sequence publishes its length: up to the first page that has no block
  __shared__ int s_last, s_end;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(&a.counters[b], 1) == c.kv_heads * (int)gridDim.y - 1;
    s_end = end;
  }
  __syncthreads();
  if (!s_last) return;
  if (c.block_table) {
    for (int64_t p = page0 + threadIdx.x; p * P < end; p += kExtendThreads) {
      size_t off;
      if (!kv_page_offset(c, b, 0, (int)p, off)) atomicMin(&s_end, (int)max(p * P, (int64_t)start));
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    a.counters[b] = 0;
    c.seq_lens[b] = s_end;
    if (s_end < end) atomicOr(a.status, EKV_STATUS_PAGE_RANGE);
  }
}

}  // namespace ekv

extern "C" int ekv_extend(const ekv_cache_desc* c, const void* k_new, const void* v_new, int64_t new_stride_b,
                          int64_t new_stride_h, int64_t new_stride_t, int32_t tokens, const int32_t* counts,
                          const int32_t* index, int64_t index_stride_b, const int32_t* start, int32_t* counters,
                          int32_t* status, void* stream) {
  using namespace ekv;
  if (int e = check_desc(c)) return e;
  if (!k_new || !v_new || !counters || !status || tokens <= 0) return EKV_ERR_ARG;
  if (!c->k_min || !c->k_max || !c->k_mean || !c->k_std) return EKV_ERR_ARG;
  const int64_t esz = c->dtype == EKV_F32 ? 4 : 2;
  if ((new_stride_b * esz) % 16 || (new_stride_h * esz) % 16 || (new_stride_t * esz) % 16) return EKV_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new)) & 15) return EKV_ERR_ARG;
  const ExtendArgs a{k_new, v_new, new_stride_b, new_stride_h, new_stride_t, tokens, counts, index, index_stride_b,
                     start, counters, status};
  const int64_t pages = (int64_t)(tokens - 1) / c->page_size + 2;    // that `tokens` rows can touch
  const int64_t lanes = c->head_dim * esz / 16;
  const int64_t groups = (pages * lanes + kExtendThreads - 1) / kExtendThreads;
  if (groups > 65535 || groups * c->kv_heads > 0x7fffffff || (int64_t)c->batch * c->kv_heads > 0x7fffffff)
    return EKV_ERR_ARG;
  EKV_DISPATCH(c->dtype, c->head_dim, {
    extend_kernel<T, D><<<dim3((unsigned)(c->batch * c->kv_heads), (unsigned)groups), kExtendThreads, 0,
                          as_stream(stream)>>>(*c, a);
  });
  return launch_status();
}
