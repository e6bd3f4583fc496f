// hstu_paged: the key / value gather that turns a paged KV cache plus the new target rows into the packed
// [tokens, heads, dim] layout the attention kernels read.
//
// The reference operator (ascendc/attention/hstu_v1/torch_extension/hstu_paged_plugin.cpp:21-72; kernel
// .../hstu_forward_v1/op_kernel/atlas950/hstu_paged_forward_kernel.h, FetchKvMayFromCache) attends, per sequence,
// over   K/V = [ page 0 | page 1 | ... | last page cut to last_page_len ]  ++  [ the target rows of the input k / v ]
// where the pages are kv_cache[page_ids[page_offsets[b] .. page_offsets[b + 1])] and the target rows are the last
// num_target[b] rows of the sequence's segment of the input k / v (the history rows of the input are not used).
// Here one HBM-bound pass writes exactly that into two staging tensors inside the caller's workspace, after which the
// call is an ordinary jagged forward in its `.delta` form (len_q = new history + targets <= len_k = cache + targets)
// on the same tcgen05 / generic kernels, scheduler and mask algebra.  A page of the cache is contiguous
// [page_size, heads, dim], so every page is one straight copy of page_size * heads * dim elements.
//
// Inconsistent page tables are flagged by the scheduling pre-pass (HSTU_ST_BAD_PAGES); this pass only makes them
// harmless: a row whose source does not exist (a page slot outside the sequence's range, a page id outside the cache)
// becomes zeros, and nothing outside the tensors is ever addressed.
//
// hstu_paged_8bit calls that no kernel reads in place (fp32 queries, wide or odd heads) come through here too: the same pass,
// with the cached rows turned into the call's type, number * scale rounded once, on the way.
#include <type_traits>

#include "hstu_mma8.cuh"
#include "hstu_simt.cuh"

namespace hstu {

namespace {

constexpr int kGatherThreads = 256;
constexpr int kGatherRows = 64;   // consecutive staging rows per CTA

struct GatherParams {
  const unsigned char* cache;   // [pages, 2, page_size, heads_k, dim]
  const unsigned char* k_in;    // [total_q, heads_k, dim]
  const unsigned char* v_in;
  unsigned char* k_out;         // [capacity, heads_k, dim]
  unsigned char* v_out;
  const void* offq;
  const void* offk;
  const void* tgt;
  const void* page_offsets;
  const void* page_ids;
  long long total_q, capacity, num_pages, num_page_ids;
  int index_bytes, batch, page_size;
  int row_bytes;                // heads_k * dim * element size
  int skip_full_pages;          // the attention kernel reads whole pages from the cache: stage only the rest
  // a cache of 8-bit rows
  const float* scale;           // [pages, 2, page_size / block, heads_k]
  int block, heads, dim;
};

// What a row of the cache is made of, and the type it is staged in: bytes that are copied, or 8-bit numbers.
struct AsIs {};

// One CTA per kGatherRows consecutive rows of a staging tensor (grid.y = 0: keys, 1: values).
//   phase 1  one thread per row finds the row's source: its sequence by bisection over seq_offset_k, then either a row
//            of a cache page or a target row of the input; rows behind the last sequence become zeros for one K/V
//            tile's worth (a tile that runs past the end of the data multiplies those rows by P = 0, which must not
//            meet the NaN bit patterns uninitialised memory may hold), the rest of the capacity is never read
//   phase 2  all threads copy: a warp takes four rows at a time and issues their loads before the first store
// V: the piece that is copied at once; with 8-bit rows kN elements of type T at a time.
template <typename V, typename H, typename T, int kN>
__global__ void __launch_bounds__(kGatherThreads) hstu_paged_gather_kernel(const GatherParams p) {
  constexpr bool kHeld = !std::is_same<H, AsIs>::value;
  __shared__ const float* s_scale[kHeld ? kGatherRows : 1];   // of the row's block, null for a row of k / v
  __shared__ const unsigned char* s_src[kGatherRows];
  __shared__ unsigned char s_mode[kGatherRows];   // 0: skip the row, 1: copy from s_src, 2: zeros
  __shared__ long long s_off[kGatherRows + 1];    // seq_offset_k[b0 .. b0 + 64], b0 = the sequence of the CTA's first row
  __shared__ int s_b0;
  __shared__ int s_skip_all;
  const bool is_v = blockIdx.y != 0;
  unsigned char* out = is_v ? p.v_out : p.k_out;
  const long long first = static_cast<long long>(blockIdx.x) * kGatherRows;
  // The rows of a CTA are consecutive, so their sequences are b0, b0 + 1, ...: warp 0 finds b0 with a 32-way search
  // (three rounds of loads for 32 768 sequences instead of fifteen dependent ones per row), the offsets from b0 on go
  // to shared memory, and every row finds its sequence there.  Offsets that are not monotone (flagged by the
  // pre-pass) may send a row to the wrong sequence; the range check below then gives it no source.
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int lo = 0, hi = p.batch - 1;   // the last sequence whose first row is <= first lies in [lo, hi]
    while (hi > lo) {
      const int stride = (hi - lo + 31) >> 5;
      auto probe = [&](int l) { const int at = lo + (l + 1) * stride; return at < hi ? at : hi; };
      const bool le = load_index(p.offk, p.index_bytes, probe(lane)) <= first;
      const int c = __popc(__ballot_sync(0xffffffffu, le));
      if (c == 0) {
        hi = probe(0) - 1;
      } else {
        const int nlo = probe(c - 1);
        if (c < 32) hi = probe(c) - 1 > nlo ? probe(c) - 1 : nlo;
        lo = nlo;
      }
    }
    if (lane == 0) s_b0 = lo;
  }
  __syncthreads();
  const int b0 = s_b0;
  if (threadIdx.x <= kGatherRows) {
    const int at = b0 + static_cast<int>(threadIdx.x) < p.batch ? b0 + static_cast<int>(threadIdx.x) : p.batch;
    s_off[threadIdx.x] = load_index(p.offk, p.index_bytes, at);
  }
  __syncthreads();
  // Direct page reads: most CTAs lie wholly inside the whole pages of one sequence and have nothing to stage.
  if (p.skip_full_pages) {
    if (threadIdx.x == 0) {
      int all = 0;
      if (first >= s_off[0] && first + kGatherRows <= s_off[1]) {
        long long slot;
        const int n = paged_full_tiles(p.offq, p.offk, p.tgt, p.page_offsets, p.index_bytes, p.total_q, p.num_page_ids,
                                       b0, &slot);
        all = first + kGatherRows - s_off[0] <= static_cast<long long>(kTileN) * n ? 1 : 0;
      }
      s_skip_all = all;
    }
    __syncthreads();
    if (s_skip_all) return;
  }
  if (threadIdx.x < kGatherRows) {
    const long long row = first + threadIdx.x;
    const unsigned char* src = nullptr;
    const float* scale = nullptr;
    unsigned char mode = 0;
    long long k_end = load_index(p.offk, p.index_bytes, p.batch);
    if (k_end < 0) k_end = 0;
    if (k_end > p.capacity) k_end = p.capacity;
    if (row < p.capacity && row >= k_end) {
      mode = row < k_end + kTileN ? 2 : 0;
    } else if (row < p.capacity) {
      // the last sequence whose first row is <= row (sequences of length 0 share their offset with the next one)
      int b;
      long long k0, k1;
      if (row < s_off[kGatherRows] || b0 + kGatherRows >= p.batch) {
        int lo = 0, hi = kGatherRows - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (s_off[mid] <= row) lo = mid; else hi = mid - 1;
        }
        b = b0 + lo < p.batch - 1 ? b0 + lo : p.batch - 1;
        k0 = s_off[b - b0];
        k1 = s_off[b - b0 + 1];
      } else {   // more than 64 sequences begin inside this CTA's rows (runs of empty ones): the long way
        int lo = b0, hi = p.batch - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (load_index(p.offk, p.index_bytes, mid) <= row) lo = mid; else hi = mid - 1;
        }
        b = lo;
        k0 = load_index(p.offk, p.index_bytes, b);
        k1 = load_index(p.offk, p.index_bytes, b + 1);
      }
      if (row >= k0 && row < k1) {   // (offsets that are not monotone, flagged by the pre-pass, leave rows uncovered)
        mode = 2;                    // zeros unless a source exists (an inconsistent table has none for this row)
        const long long q0 = load_index(p.offq, p.index_bytes, b);
        long long q1 = load_index(p.offq, p.index_bytes, b + 1);
        if (q1 > p.total_q) q1 = p.total_q;
        long long t = p.tgt ? load_index(p.tgt, p.index_bytes, b) : 0;
        if (t < 0) t = 0;
        if (t > q1 - q0) t = q1 - q0 > 0 ? q1 - q0 : 0;
        const long long r = row - k0, cache_len = (k1 - k0) - t;
        long long unused_slot;
        if (p.skip_full_pages &&
            r < static_cast<long long>(kTileN) * paged_full_tiles(p.offq, p.offk, p.tgt, p.page_offsets, p.index_bytes,
                                                                  p.total_q, p.num_page_ids, b, &unused_slot)) {
          mode = 0;   // a row of a whole page: never read from the staging tensor
        } else if (r < cache_len) {
          long long pg0 = load_index(p.page_offsets, p.index_bytes, b), pg1 = load_index(p.page_offsets, p.index_bytes, b + 1);
          if (pg0 < 0) pg0 = 0;
          if (pg1 > p.num_page_ids) pg1 = p.num_page_ids;
          const long long slot = pg0 + r / p.page_size;
          if (slot < pg1) {
            const long long pid = load_index(p.page_ids, p.index_bytes, slot);
            if (pid >= 0 && pid < p.num_pages) {
              src = p.cache + ((pid * 2 + (is_v ? 1 : 0)) * p.page_size + r % p.page_size) *
                                  (kHeld ? p.heads * p.dim : p.row_bytes);
              if (kHeld)
                scale = p.scale + ((pid * 2 + (is_v ? 1 : 0)) * (p.page_size / p.block) + r % p.page_size / p.block) * p.heads;
              mode = 1;
            }
          }
        } else {
          const long long at = q1 - t + (r - cache_len);
          if (at >= 0 && at < p.total_q) {
            src = (is_v ? p.v_in : p.k_in) + at * p.row_bytes;
            mode = 1;
          }
        }
      }
    }
    s_src[threadIdx.x] = src;
    s_mode[threadIdx.x] = mode;
    if (kHeld) s_scale[threadIdx.x] = scale;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kWarps = kGatherThreads / 32;
  if constexpr (kHeld) {
    const int n = p.heads * p.dim;
    for (int r = warp; r < kGatherRows; r += kWarps) {
      if (!s_mode[r]) continue;
      T* to = reinterpret_cast<T*>(out) + (first + r) * n;
      const float* scale = s_scale[r];
      for (int i = lane * kN; i < n; i += 32 * kN) {
        alignas(16) T x[kN];
        if (s_mode[r] == 2) {
#pragma unroll
          for (int e = 0; e < kN; ++e) x[e] = simt::from_float<T>(0.f);
        } else if (scale) {
          uint8_t v[kN];
          if constexpr (kN == 8) {
            const uint2 u = *reinterpret_cast<const uint2*>(s_src[r] + i);
#pragma unroll
            for (int e = 0; e < kN; ++e) v[e] = reinterpret_cast<const uint8_t*>(&u)[e];
          } else {
            v[0] = s_src[r][i];
          }
          const float f = __ldg(scale + i / p.dim);
#pragma unroll
          for (int e = 0; e < kN; ++e) x[e] = simt::from_float<T>(H::to_float(v[e]) * f);
        } else {
#pragma unroll
          for (int e = 0; e < kN; ++e) x[e] = reinterpret_cast<const T*>(s_src[r])[i + e];
        }
#pragma unroll
        for (int e = 0; e < kN; ++e) to[i + e] = x[e];
      }
    }
    return;
  }
  constexpr int kBatch = 4;   // rows in flight per warp
  for (int r0 = warp * kBatch; r0 < kGatherRows; r0 += kWarps * kBatch) {
    for (int i = lane * static_cast<int>(sizeof(V)); i < p.row_bytes; i += 32 * static_cast<int>(sizeof(V))) {
      V v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) v[j] = s_mode[r0 + j] == 1 ? *reinterpret_cast<const V*>(s_src[r0 + j] + i) : V{};
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (s_mode[r0 + j]) *reinterpret_cast<V*>(out + (first + r0 + j) * p.row_bytes + i) = v[j];
    }
  }
}

// hstu_paged_8bit, calls that the kernel for short sequences then reads in place: the pages of the table, slot by slot, in the
// call's type - a cache of its own whose page i is slot i, with the table of its pages.  Rows nobody reads (behind a sequence's
// last one, and a whole tile of 64 keys away from what a window or its sinks show) stay unwritten.  HBM-bound: one byte in, two
// out (9760 pages of 128 rows, 4 heads of 64, 78 % full: 1.5 GB, 244 us, 6.2 TB/s; in pieces of 16 numbers, whose stores do not
// fill lines, 263); the pre-pass runs beside it (15 us of 600 of such a call).
constexpr int kUnpackThreads = 256;

struct UnpackParams {
  const unsigned char* cache;   // [pages, 2, page_size, heads, dim]
  const float* scale;
  void* out;                    // [num_page_ids, 2, page_size, heads, dim]
  void* table;                  // [num_page_ids]: 0, 1, 2, .. (-1: not a page of the cache)
  const void* offq;
  const void* offk;
  const void* tgt;
  const void* page_offsets;
  const void* page_ids;
  long long num_pages, num_page_ids;
  int index_bytes, batch, page_size, block, heads, dim, window, sink;
  uint32_t by_row, by_head, by_block;   // over(): pieces of a row, pieces of a head, rows of a block
};

template <typename T, typename H>
__global__ void __launch_bounds__(kUnpackThreads) hstu_unpack_kernel(const UnpackParams p) {
  __shared__ int s_b;
  const long long slot = blockIdx.x;
  if (threadIdx.x < 32) {   // the last sequence whose first slot is <= slot, by a 32-way search
    const int lane = threadIdx.x;
    int lo = 0, hi = p.batch - 1;
    while (hi > lo) {
      const int stride = (hi - lo + 31) >> 5;
      auto probe = [&](int l) { const int at = lo + (l + 1) * stride; return at < hi ? at : hi; };
      const bool le = load_index(p.page_offsets, p.index_bytes, probe(lane)) <= slot;
      const int c = __popc(__ballot_sync(0xffffffffu, le));
      if (c == 0) {
        hi = probe(0) - 1;
      } else {
        const int nlo = probe(c - 1);
        if (c < 32) hi = probe(c) - 1 > nlo ? probe(c) - 1 : nlo;
        lo = nlo;
      }
    }
    if (lane == 0) s_b = lo;
  }
  __syncthreads();
  const int b = s_b;
  const long long pid = load_index(p.page_ids, p.index_bytes, slot);
  const bool ok = pid >= 0 && pid < p.num_pages;
  if (threadIdx.x == 0) {   // (a page outside of the cache stays one)
    if (p.index_bytes == 8) static_cast<long long*>(p.table)[slot] = ok ? slot : -1;
    else static_cast<int*>(p.table)[slot] = ok ? static_cast<int>(slot) : -1;
  }
  const long long first = (slot - load_index(p.page_offsets, p.index_bytes, b)) * p.page_size;   // the page's first key
  const long long lk = load_index(p.offk, p.index_bytes, b + 1) - load_index(p.offk, p.index_bytes, b);
  const long long lq = load_index(p.offq, p.index_bytes, b + 1) - load_index(p.offq, p.index_bytes, b);
  long long t = p.tgt ? load_index(p.tgt, p.index_bytes, b) : 0;
  if (t < 0) t = 0;
  const long long cached = lk - t;
  // rows [0, n) of the page are read; with a window, those below `skip_from` and from `skip_to` on
  long long n = cached - first;
  n = n < 0 ? 0 : n > p.page_size ? p.page_size : n;
  long long skip_from = n, skip_to = n;
  if (p.window) {
    long long lo = lk - lq - p.window + 1;
    lo = lo < 0 ? 0 : lo / 64 * 64;
    const long long sinks = (p.sink + 63ll) / 64 * 64;
    skip_from = sinks - first < 0 ? 0 : sinks - first;
    skip_to = lo - first < skip_from ? skip_from : lo - first;
  }
  const int row_len = p.heads * p.dim, per_page = p.page_size / p.block;
  const long long page_len = static_cast<long long>(p.page_size) * row_len;
  const uint2* from = reinterpret_cast<const uint2*>(p.cache + (ok ? pid : 0) * 2 * page_len);
  const float* scale = p.scale + (ok ? pid : 0) * 2 * per_page * static_cast<long long>(p.heads);
  uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + slot * 2 * page_len);
  const int per_row = row_len / 8, pieces = static_cast<int>(n) * per_row;   // of 8 numbers (a warp's stores are 512 bytes in a row)
  constexpr int kFly = 8;
  for (int i0 = threadIdx.x; i0 < 2 * pieces; i0 += kFly * kUnpackThreads) {
    uint2 w[kFly];
    float f[kFly];
    int at[kFly];   // of the piece in the page, -1: nothing to do
#pragma unroll
    for (int u = 0; u < kFly; ++u) {
      const int both = i0 + u * kUnpackThreads, kv = both >= pieces ? 1 : 0, i = both - kv * pieces;
      const int row = over(i, p.by_row), head = over(i - row * per_row, p.by_head);
      at[u] = i < pieces && (row < skip_from || row >= skip_to) ? kv * (p.page_size * per_row) + i : -1;
      w[u] = make_uint2(0, 0);
      f[u] = 0.f;
      if (at[u] >= 0 && ok) {
        w[u] = __ldcs(from + at[u]);
        f[u] = __ldg(scale + (kv * per_page + over(row, p.by_block)) * p.heads + head);
      }
    }
#pragma unroll
    for (int u = 0; u < kFly; ++u) {
      if (at[u] < 0) continue;
      uint32_t h[4], x[4];
      to_halves<H>(w[u].x, h[0], h[1]);
      to_halves<H>(w[u].y, h[2], h[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 v = unpack2<__half>(h[e]);
        x[e] = pack2<T>(v.x * f[u], v.y * f[u]);
      }
      to[at[u]] = make_uint4(x[0], x[1], x[2], x[3]);
    }
  }
  // Launched beside the pre-pass, which writes nothing this one reads; the kernel behind it finds both complete.
  if (slot == p.num_page_ids - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace

// Whether a cache of 8-bit rows can be unpacked page by page: pieces of 8 numbers of one head.
bool unpack_supported(const KParams& p, int dtype) {
  return dtype != HSTU_DTYPE_FP32 && p.dqk % 8 == 0 && (reinterpret_cast<uintptr_t>(p.kv_cache) & 7u) == 0 &&
         p.page_size <= 65536 && static_cast<long long>(p.page_size) * p.hk * p.dqk / 8 < (1ll << 21) &&
         p.num_page_ids <= 0x7fffffffll;
}
cudaError_t launch_unpack(const KParams& p, void* out, void* table, int dtype, cudaStream_t stream) {
  UnpackParams u;
  u.cache = static_cast<const unsigned char*>(p.kv_cache);
  u.scale = p.kv_scale;
  u.out = out;
  u.table = table;
  u.offq = p.offq;
  u.offk = p.offk;
  u.tgt = p.tgt;
  u.page_offsets = p.page_offsets;
  u.page_ids = p.page_ids;
  u.num_pages = p.num_pages;
  u.num_page_ids = p.num_page_ids;
  u.index_bytes = p.index_bytes;
  u.batch = p.batch;
  u.page_size = p.page_size;
  u.block = p.scale_block;
  u.heads = p.hk;
  u.dim = p.dqk;
  u.window = p.window;
  u.sink = p.sink;
  // (at most 2^21 pieces - and as many again - by 1024 of a row, 1024 by 64 of a head, 2^16 rows by as many of a block)
  u.by_row = inverse_of(p.hk * p.dqk / 8);
  u.by_head = inverse_of(p.dqk / 8);
  u.by_block = inverse_of(p.scale_block);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.num_page_ids));
  cfg.blockDim = dim3(kUnpackThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool held = p.held == HSTU_HELD_E4M3;
  if (dtype == HSTU_DTYPE_BF16)
    return cudaLaunchKernelEx(&cfg, held ? hstu_unpack_kernel<__nv_bfloat16, E4m3> : hstu_unpack_kernel<__nv_bfloat16, Int8>, u);
  return cudaLaunchKernelEx(&cfg, held ? hstu_unpack_kernel<__half, E4m3> : hstu_unpack_kernel<__half, Int8>, u);
}

template <typename T, int kN>
static void launch_held(const GatherParams& g, int held, dim3 grid, cudaStream_t stream) {
  if (held == HSTU_HELD_E4M3) hstu_paged_gather_kernel<uint4, E4m3, T, kN><<<grid, kGatherThreads, 0, stream>>>(g);
  else hstu_paged_gather_kernel<uint4, Int8, T, kN><<<grid, kGatherThreads, 0, stream>>>(g);
}

// Enqueues the gather.  All pointers are device pointers; capacity = rows of each staging tensor.
cudaError_t launch_paged_gather(const KParams& p, const void* kv_cache, const void* k_in, const void* v_in,
                                void* k_out, void* v_out, long long capacity, long long num_pages,
                                long long num_page_ids, int dtype, cudaStream_t stream) {
  const int esize = dtype == HSTU_DTYPE_FP32 ? 4 : 2;
  GatherParams g;
  g.cache = static_cast<const unsigned char*>(kv_cache);
  g.k_in = static_cast<const unsigned char*>(k_in);
  g.v_in = static_cast<const unsigned char*>(v_in);
  g.k_out = static_cast<unsigned char*>(k_out);
  g.v_out = static_cast<unsigned char*>(v_out);
  g.offq = p.offq;
  g.offk = p.offk;
  g.tgt = p.tgt;
  g.page_offsets = p.page_offsets;
  g.page_ids = p.page_ids;
  g.total_q = p.total_q;
  g.capacity = capacity;
  g.num_pages = num_pages;
  g.num_page_ids = num_page_ids;
  g.index_bytes = p.index_bytes;
  g.batch = p.batch;
  g.page_size = p.page_size;
  g.row_bytes = p.hk * p.dqk * esize;
  g.skip_full_pages = p.paged_direct;
  g.scale = p.kv_scale;
  g.block = p.scale_block;
  g.heads = p.hk;
  g.dim = p.dqk;
  const dim3 grid(static_cast<unsigned>((capacity + kGatherRows - 1) / kGatherRows), 2, 1);
  const uintptr_t align = reinterpret_cast<uintptr_t>(kv_cache) | reinterpret_cast<uintptr_t>(k_in) |
                          reinterpret_cast<uintptr_t>(v_in) | reinterpret_cast<uintptr_t>(k_out) |
                          reinterpret_cast<uintptr_t>(v_out) | static_cast<uintptr_t>(g.row_bytes);
  if (p.kv_scale) {
    const bool vec = p.dqk % 8 == 0 && (reinterpret_cast<uintptr_t>(kv_cache) & 7u) == 0;
    if (dtype == HSTU_DTYPE_BF16)
      vec ? launch_held<__nv_bfloat16, 8>(g, p.held, grid, stream) : launch_held<__nv_bfloat16, 1>(g, p.held, grid, stream);
    else if (dtype == HSTU_DTYPE_FP16)
      vec ? launch_held<__half, 8>(g, p.held, grid, stream) : launch_held<__half, 1>(g, p.held, grid, stream);
    else
      vec ? launch_held<float, 8>(g, p.held, grid, stream) : launch_held<float, 1>(g, p.held, grid, stream);
  } else if ((align & 15u) == 0)
    hstu_paged_gather_kernel<uint4, AsIs, float, 1><<<grid, kGatherThreads, 0, stream>>>(g);
  else if ((align & 3u) == 0)
    hstu_paged_gather_kernel<uint32_t, AsIs, float, 1><<<grid, kGatherThreads, 0, stream>>>(g);
  else
    hstu_paged_gather_kernel<uint16_t, AsIs, float, 1><<<grid, kGatherThreads, 0, stream>>>(g);
  return cudaGetLastError();
}

}  // namespace hstu
