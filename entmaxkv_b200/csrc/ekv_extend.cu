// Several tokens per sequence written into the cache, with the statistics of every page that they touch.
//
// Row i < counts[b] of sequence b is row index[b, i] (or i) of k_new / v_new and lands at position start[b] + i.  A page
// of keys is handled by LPR lanes, one 16-byte column each: a lane gathers the page's rows - those already in the cache
// and the new ones, 16 on their way at a time - stores the new ones and forms the column's statistics from the same
// registers, so a new row is read once and written once and an old row is read only where it shares the first page.
// Values are copied by blocks of their own: with both in one thread the registers leave too few loads in flight.
// Bound by memory: 8 sequences, 3000 to 4096 rows each, 8 heads of 128, bf16: 56 us, 5.0 TB/s, 0.76 of a plain copy (a launch
// alone 54 us; 128-thread blocks took 0.97 of the time of 256-thread blocks, keys and values in one thread 1.22).  A tree's
// accepted path, 32 sequences: 10 us, latency.
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

constexpr int kExtendMaxThreads = 128;
constexpr int kExtendRows = 16;  // rows of a page held in registers at once

// grid: (B * H_kv, page groups, 2: keys, values)
template <typename T, int D>
__global__ void __launch_bounds__(kExtendMaxThreads) extend_kernel(const __grid_constant__ ekv_cache_desc c,
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
  const int64_t page64 = page0 + ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) / LPR;
  const int col = threadIdx.x % LPR * EPL;
  // a rewind without new rows still leaves its page with fewer rows
  if (page64 * P < end && (n > 0 || start < now)) {
    const int page = (int)page64;
    size_t off;
    if (kv_page_offset(c, b, h, page, off)) {
      const bool keys = blockIdx.z == 0;
      T* const to = static_cast<T*>(keys ? c.k : c.v) + off + col;
      const T* const from = static_cast<const T*>(keys ? a.k_new : a.v_new) + b * a.sb + h * a.sh + col;
      const int64_t r0 = (int64_t)page * P;
      const int rows = (int)min((int64_t)P, end - r0);
      const int old = (int)min(max(start - r0, (int64_t)0), (int64_t)rows);      // rows that are in the cache
      const auto source = [&](int i) -> const T* {     // the new row that becomes row i of the page
        int j = (int)(r0 + i - start);
        if (a.index) {
          const int given = a.index[b * a.index_sb + j];
          j = min(max(given, 0), a.tokens - 1);
          if (j != given) flag |= EKV_STATUS_TOKENS;
        }
        return from + j * a.st;
      };
      uint4 x[kExtendRows];
      ColumnStats<T> st;
      st.begin();
      for (int i0 = keys ? 0 : old; i0 < rows; i0 += kExtendRows) {
        const int n = min(rows - i0, kExtendRows);
#pragma unroll
        for (int i = 0; i < kExtendRows; ++i)
          if (i < n) x[i] = i0 + i < old ? *reinterpret_cast<const uint4*>(to + (size_t)(i0 + i) * D) : ld_stream(source(i0 + i));
#pragma unroll
        for (int i = 0; i < kExtendRows; ++i)
          if (i < n) {
            if (i0 + i >= old) *reinterpret_cast<uint4*>(to + (size_t)(i0 + i) * D) = x[i];
            if (keys) st.first_pass(x[i]);
          }
      }
      if (keys) {
        st.middle((float)rows);
        for (int i0 = 0; i0 < rows; i0 += kExtendRows) {
          const int n = min(rows - i0, kExtendRows);
          if (rows > kExtendRows) {                    // longer pages: this lane re-reads the column that it wrote itself
#pragma unroll
            for (int i = 0; i < kExtendRows; ++i)
              if (i < n) x[i] = *reinterpret_cast<const uint4*>(to + (size_t)(i0 + i) * D);
          }
#pragma unroll
          for (int i = 0; i < kExtendRows; ++i)
            if (i < n) st.second_pass(x[i]);
        }
        const size_t mo = b * c.meta_stride_b + h * c.meta_stride_h + (size_t)page * D + col;
        st.finish((float)rows, static_cast<T*>(c.k_min) + mo, static_cast<T*>(c.k_max) + mo,
                  static_cast<T*>(c.k_mean) + mo, static_cast<T*>(c.k_std) + mo);
      }
    }
  }
  if (flag) atomicOr(a.status, flag);

  // the last block of the sequence publishes its length: up to the first page that has no block
  __shared__ int s_last, s_end;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(&a.counters[b], 1) == c.kv_heads * (int)(gridDim.y * gridDim.z) - 1;
    s_end = end;
  }
  __syncthreads();
  if (!s_last) return;
  if (c.block_table) {
    for (int64_t p = page0 + threadIdx.x; p * P < end; p += blockDim.x) {
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
  const int threads = pages * lanes >= kExtendMaxThreads ? kExtendMaxThreads : (int)((pages * lanes + 31) / 32 * 32);
  const int64_t groups = (pages * lanes + threads - 1) / threads;
  if (groups > 65535 || 2 * groups * c->kv_heads > 0x7fffffff || (int64_t)c->batch * c->kv_heads > 0x7fffffff)
    return EKV_ERR_ARG;
  EKV_DISPATCH(c->dtype, c->head_dim, {
    extend_kernel<T, D><<<dim3((unsigned)(c->batch * c->kv_heads), (unsigned)groups, 2), threads, 0,
                          as_stream(stream)>>>(*c, a);
  });
  return launch_status();
}
