// hstu_cache_append: new keys and values into a paged cache of 8-bit rows with a scale per block of tokens and head.
//
//   scale = the smallest power of two with amax <= 448 scale (e4m3; int8: 127 scale), amax over the finite new values of a
//           block and head; where the block holds rows already, no smaller than the scale they have
//   row   = round(x / scale); the rows a block holds already are rounded anew to round(number * old / scale) when it grew
//
// A warp does one block of tokens, of the keys or of the values: two passes over at most `block` rows.  Where a head is 8, 16, ..
// 256 wide it takes 256 columns, whichever heads they belong to - a piece of 8 columns per lane, whole lines per row, and the
// look-ups in front shared by all of the heads - elsewhere one head.  Of 16-bit histories the rows arrive in shared memory, all
// requested at once (cp.async), and stay there between the passes; read twice from memory instead, eight rows at a time, they come
// out of the L2 the second time (80 us below), and kept in registers they leave an SM too few warps (140).
// Which blocks there are is known to the device only; sequence b owns the slots [seq_offset[b] / block + 2 b, ..) of the grid,
// which are never fewer than the blocks its rows touch (n rows touch at most n / block + 2), and finds them by a 32-way search.
// HBM-bound for histories (3 bytes per 16-bit element: 256 of 680 rows on average, 4 heads of 64, 43 us of bytes, take 53: 5 TB/s), a chain
// of six dependent reads for single rows (6 us of one row each of 128 users).
#include "hstu_held.cuh"
#include "hstu_simt.cuh"

namespace hstu {

namespace {

struct AppendParams {
  const void* k;                // [total, heads, dim]
  const void* v;
  uint8_t* cache;               // [num_pages, 2, page_size, heads, dim]
  float* scale;                 // [num_pages, 2, page_size / block, heads]
  const void* offset;           // [batch + 1] of the rows of k / v
  const void* tgt;              // [batch] or null: trailing rows that are not kept
  const void* page_offsets;
  const void* page_ids;
  const void* last_page_len;
  uint32_t* status;
  long long total, num_pages, num_page_ids;
  int index_bytes, batch, page_size, block, heads, dim;
};

constexpr int kAppendThreads = 256;
constexpr int kStagedThreads = 32;
constexpr int kStagedRows = 32;   // of a block, at most: 16 KB a warp, 13 warps on an SM

// Eight elements (or one) of a row, as floats.
template <typename T, int kN> struct Piece;
template <typename T> struct Piece<T, 1> {
  static __device__ __forceinline__ void load(const T* from, float (&x)[1]) { x[0] = simt::to_float<T>(*from); }
  static __device__ __forceinline__ void load_held(const uint8_t* from, uint8_t (&x)[1]) { x[0] = *from; }
  static __device__ __forceinline__ void store(uint8_t* to, const uint8_t (&x)[1]) { *to = x[0]; }
};
template <typename T> struct Piece<T, 8> {
  static __device__ __forceinline__ void load(const T* from, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4*>(from)[0], b = reinterpret_cast<const float4*>(from)[1];
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(from);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = simt::to_float<T>(e[i]);
    }
  }
  static __device__ __forceinline__ void load_held(const uint8_t* from, uint8_t (&x)[8]) {
    const uint2 u = *reinterpret_cast<const uint2*>(from);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = reinterpret_cast<const uint8_t*>(&u)[i];
  }
  static __device__ __forceinline__ void store(uint8_t* to, const uint8_t (&x)[8]) {
    uint2 u;
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<uint8_t*>(&u)[i] = x[i];
    *reinterpret_cast<uint2*>(to) = u;
  }
};

// (a 64-bit division is some hundred instructions)
__device__ __forceinline__ long long quotient(long long a, int b) {
  return (a >> 32) == 0 ? static_cast<long long>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}

// The largest magnitude of eight (the call's type): NaN take no part, infinities do.
template <typename T> struct Largest;
template <> struct Largest<float> {
  float m = 0.f;
  __device__ __forceinline__ void take(const float* from) {
    float x[8];
    Piece<float, 8>::load(from, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[e]));
  }
  __device__ __forceinline__ float get() const { return m; }
};
template <> struct Largest<__nv_bfloat16> {
  __nv_bfloat162 m = __floats2bfloat162_rn(0.f, 0.f);
  __device__ __forceinline__ void take(const __nv_bfloat16* from) {
    const uint4 u = *reinterpret_cast<const uint4*>(from);
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __hmax2(m, __habs2(reinterpret_cast<const __nv_bfloat162*>(&u)[e]));
  }
  __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <> struct Largest<__half> {
  __half2 m = __floats2half2_rn(0.f, 0.f);
  __device__ __forceinline__ void take(const __half* from) {
    const uint4 u = *reinterpret_cast<const uint4*>(from);
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __hmax2(m, __habs2(reinterpret_cast<const __half2*>(&u)[e]));
  }
  __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};

// What a warp's slot stands for: rows [r0, r1) of sequence b, in block `base / block` of its cache.
struct AppendWork {
  long long first;    // of the rows, in k and v
  long long place;    // of the block's first row in the cache, counted in rows of the keys' half of its page
  long long scale;    // of its scales: of the keys of head 0
  int held, count;    // rows the block holds already, new rows; 0 new rows: nothing to do
};
__device__ __forceinline__ AppendWork find_work(const AppendParams& p, long long slot) {
  const int lane = threadIdx.x & 31;
  AppendWork w = {0, 0, 0, 0, 0};
  // the last sequence whose first slot is <= slot
  auto first_slot = [&](int b) {
    long long o = load_index(p.offset, p.index_bytes, b);
    if (o < 0) o = 0;
    if (o > p.total) o = p.total;
    return quotient(o, p.block) + 2ll * b;
  };
  int lo = 0, hi = p.batch - 1;
  while (hi > lo) {
    const int stride = (hi - lo + 31) >> 5;
    auto probe = [&](int l) { const int at = lo + (l + 1) * stride; return at < hi ? at : hi; };
    const bool le = first_slot(probe(lane)) <= slot;
    const int c = __popc(__ballot_sync(0xffffffffu, le));
    if (c == 0) {
      hi = probe(0) - 1;
    } else {
      const int nlo = probe(c - 1);
      if (c < 32) hi = probe(c) - 1 > nlo ? probe(c) - 1 : nlo;
      lo = nlo;
    }
  }
  const int b = lo;
  // The sequence: its new rows, and the cached rows its pages describe (the new ones are the last of them).  What does not
  // fit together writes nothing.
  const long long q0 = load_index(p.offset, p.index_bytes, b), q1 = load_index(p.offset, p.index_bytes, b + 1);
  const long long t = p.tgt ? load_index(p.tgt, p.index_bytes, b) : 0;
  const long long pg0 = load_index(p.page_offsets, p.index_bytes, b), pg1 = load_index(p.page_offsets, p.index_bytes, b + 1);
  const long long last = load_index(p.last_page_len, p.index_bytes, b);
  unsigned bad = 0;
  if (q0 < 0 || q1 < q0 || q1 > p.total) bad |= HSTU_ST_BAD_OFFSETS;
  if (t < 0 || t > q1 - q0) bad |= HSTU_ST_BAD_CTX_TARGET;
  const long long fresh = q1 - q0 - t, pages = pg1 - pg0;
  if (pg0 < 0 || pages < 0 || pg1 > p.num_page_ids || last < 0 || last > p.page_size || (pages > 0 && last == 0))
    bad |= HSTU_ST_BAD_PAGES;
  const long long cached = pages > 0 ? (pages - 1) * p.page_size + last : 0, start = cached - fresh;
  if (!bad && start < 0) bad |= HSTU_ST_BAD_PAGES;
  if (bad) {
    if (lane == 0 && p.status) atomicOr(p.status, bad);
    return w;
  }
  const long long blk = quotient(start, p.block) + (slot - first_slot(b));
  const long long base = blk * p.block;
  const long long r0 = base > start ? base : start, r1 = base + p.block < cached ? base + p.block : cached;
  if (fresh == 0 || r0 >= r1) return w;
  const long long pid = load_index(p.page_ids, p.index_bytes, pg0 + quotient(base, p.page_size));
  if (pid < 0 || pid >= p.num_pages) {
    if (lane == 0 && p.status) atomicOr(p.status, static_cast<unsigned>(HSTU_ST_BAD_PAGES));
    return w;
  }
  const int in_page = static_cast<int>(base - quotient(base, p.page_size) * p.page_size);
  w.first = q0 + (r0 - start);
  w.place = pid * 2 * p.page_size + in_page;
  w.scale = (pid * 2 * (p.page_size / p.block) + in_page / p.block) * p.heads;
  w.held = static_cast<int>(r0 - base);
  w.count = static_cast<int>(r1 - r0);
  return w;
}

// 256 columns a warp: see the top.  kStaged: the block's rows lie in shared memory between the passes, 512 bytes each.
template <typename T, typename H, bool kStaged>
__global__ void __launch_bounds__(kStaged ? kStagedThreads : kAppendThreads) hstu_append_columns_kernel(const AppendParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kWarps = (kStaged ? kStagedThreads : kAppendThreads) / 32;
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int row_len = p.heads * p.dim, spans = (row_len + 255) / 256;
  const long long slot = unit / (2 * spans);
  if (slot >= p.total / p.block + 2ll * p.batch) return;
  const int rest = static_cast<int>(unit - slot * (2 * spans)), kv = rest / spans, col = (rest - kv * spans) * 256 + lane * 8;
  const AppendWork w = find_work(p, slot);
  if (w.count == 0) return;
  const bool on = col < row_len;
  const int head = on ? col / p.dim : 0;
  const T* src = static_cast<const T*>(kv ? p.v : p.k) + w.first * row_len + (on ? col : 0);
  long long src_len = row_len;
  if (kStaged) {   // (a lane reads back what it fetched itself)
    uint8_t* const mine = smem + (threadIdx.x >> 5) * p.block * 512 + lane * 16;
    for (int r = 0; r < w.count; ++r)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine + r * 512))),
                   "l"(src + static_cast<long long>(r) * row_len) : "memory");
    src = reinterpret_cast<const T*>(mine);
    src_len = 512 / sizeof(T);
  }
  uint8_t* dst = p.cache + (w.place + kv * static_cast<long long>(p.page_size)) * row_len + (on ? col : 0);
  float* scale_at = p.scale + w.scale + kv * static_cast<long long>(p.page_size / p.block) * p.heads + head;
  const float old = on && w.held > 0 ? *scale_at : 0.f;
  if (kStaged) asm volatile("cp.async.wait_all;" ::: "memory");
  Largest<T> most;
#pragma unroll 8
  for (int r = 0; r < w.count; ++r) most.take(src + r * src_len);
  float amax = most.get();
  if (__any_sync(0xffffffffu, amax > 3.402823466e38f)) {   // infinities among them: over the finite values alone
    amax = 0.f;
    for (int r = 0; r < w.count; ++r) {
      float x[8];
      Piece<T, 8>::load(src + r * src_len, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(x[e]);
        amax = a <= 3.402823466e38f && a > amax ? a : amax;
      }
    }
  }
  // over the lanes of the head (dim / 8 of them, a power of two; all of a warp hold parts of whole heads or of one)
  for (int o = p.dim / 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  float scale = block_scale<H>(amax);
  if (w.held > 0) {
    if (scale > old) {
      if (on)
        for (int r = 0; r < w.held; ++r) {
          uint8_t* at = dst + static_cast<long long>(r) * row_len;
          uint8_t v[8];
          Piece<T, 8>::load_held(at, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = H::from_float(H::to_float(v[e]) * (old / scale));
          Piece<T, 8>::store(at, v);
        }
    } else {
      scale = old;
    }
    __syncwarp();   // (every lane has read the scale before one writes it)
  }
  if (!on) return;
  if (col % p.dim == 0) *scale_at = scale;
  dst += static_cast<long long>(w.held) * row_len;
  auto write = [&](auto divide) {
#pragma unroll 8
    for (int r = 0; r < w.count; ++r) {
      float x[8];
      Piece<T, 8>::load(src + r * src_len, x);
      const uint32_t lo = H::from_floats(divide(x[0]), divide(x[1])) | (H::from_floats(divide(x[2]), divide(x[3])) << 16);
      const uint32_t hi = H::from_floats(divide(x[4]), divide(x[5])) | (H::from_floats(divide(x[6]), divide(x[7])) << 16);
      *reinterpret_cast<uint2*>(dst + static_cast<long long>(r) * row_len) = make_uint2(lo, hi);
    }
  };
  // the product with the reciprocal is the quotient wherever the scale is a power of two; another one was not written here
  const float inverse = 1.f / scale;
  if ((__float_as_uint(scale) & 0x7fffffu) == 0) write([&](float x) { return x * inverse; });
  else write([&](float x) { return x / scale; });
}

template <typename T, typename H, int kN>
__global__ void __launch_bounds__(kAppendThreads) hstu_append_kernel(const AppendParams p) {
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const int per_slot = 2 * p.heads;
  const long long slot = unit / per_slot;
  if (slot >= p.total / p.block + 2ll * p.batch) return;
  const int kv = static_cast<int>(unit - slot * per_slot) / p.heads, head = static_cast<int>(unit - slot * per_slot) % p.heads;
  const AppendWork w = find_work(p, slot);
  if (w.count == 0) return;
  const long long row_len = static_cast<long long>(p.heads) * p.dim;
  const T* src = static_cast<const T*>(kv ? p.v : p.k) + w.first * row_len + static_cast<long long>(head) * p.dim;
  uint8_t* dst = p.cache + (w.place + kv * static_cast<long long>(p.page_size)) * row_len + static_cast<long long>(head) * p.dim;
  float* scale_at = p.scale + w.scale + kv * static_cast<long long>(p.page_size / p.block) * p.heads + head;
  const int held = w.held, count = w.count;
  const int per_row = p.dim / kN;
  const int step_row = 32 / per_row, step_piece = 32 % per_row;

  float amax = 0.f;
#pragma unroll 4
  for (int i = lane, r = lane / per_row, c = lane % per_row; i < count * per_row; i += 32) {
    float x[kN];
    Piece<T, kN>::load(src + r * row_len + c * kN, x);
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const float a = fabsf(x[e]);
      amax = a <= 3.402823466e38f && a > amax ? a : amax;   // (infinities and NaN take no part in the scale)
    }
    r += step_row;
    c += step_piece;
    if (c >= per_row) c -= per_row, ++r;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  float scale = block_scale<H>(amax);
  if (held > 0) {
    const float old = *scale_at;
    __syncwarp();   // (every lane has read the scale before one writes it)
    if (scale > old) {
      for (int i = lane, r = lane / per_row, c = lane % per_row; i < held * per_row; i += 32) {
        uint8_t* at = dst + r * row_len + c * kN;
        uint8_t v[kN];
        Piece<T, kN>::load_held(at, v);
#pragma unroll
        for (int e = 0; e < kN; ++e) v[e] = H::from_float(H::to_float(v[e]) * (old / scale));
        Piece<T, kN>::store(at, v);
        r += step_row;
        c += step_piece;
        if (c >= per_row) c -= per_row, ++r;
      }
    } else {
      scale = old;
    }
  }
  if (lane == 0) *scale_at = scale;
  // the product with the reciprocal is the quotient wherever the scale is a power of two; another one was not written here
  const bool exact = (__float_as_uint(scale) & 0x7fffffu) == 0;
  const float inverse = 1.f / scale;
  dst += held * row_len;
#pragma unroll 4
  for (int i = lane, r = lane / per_row, c = lane % per_row; i < count * per_row; i += 32) {
    float x[kN];
    uint8_t v[kN];
    Piece<T, kN>::load(src + r * row_len + c * kN, x);
#pragma unroll
    for (int e = 0; e < kN; ++e) v[e] = H::from_float(exact ? x[e] * inverse : x[e] / scale);
    Piece<T, kN>::store(dst + r * row_len + c * kN, v);
    r += step_row;
    c += step_piece;
    if (c >= per_row) c -= per_row, ++r;
  }
}

template <typename T, typename H>
cudaError_t launch_append_t(const AppendParams& p, cudaStream_t stream) {
  const long long units = (p.total / p.block + 2ll * p.batch) * 2 * p.heads;
  const unsigned grid = static_cast<unsigned>((units + kAppendThreads / 32 - 1) / (kAppendThreads / 32));
  const bool vec = p.dim % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & 15u) == 0 &&
                   (reinterpret_cast<uintptr_t>(p.cache) & 7u) == 0;
  if (vec && p.dim <= 256 && (p.dim & (p.dim - 1)) == 0) {
    const long long columns = (p.total / p.block + 2ll * p.batch) * 2 * ((p.heads * p.dim + 255) / 256);
    // Staged where blocks are at least half full on average and rows fill a warp's columns.  us staged / not, 4 heads of 64, blocks
    // of 32: 2000 users of 1 / 8 / 16 rows 16.6 / 14.5, 18.8 / 18.6, 22.7 / 24.7, 1000 of 64 27 / 41; blocks of 8, 2000 of 4 rows 14.5 /
    // 16.6; 300 of 300 rows, 1 head of 32 37 / 29, 8 of 128 97 / 147.
    if constexpr (sizeof(T) == 2) {
      if (p.block <= kStagedRows && 2 * (p.total / p.batch) >= p.block && p.heads * p.dim >= 256) {
        constexpr int kWarps = kStagedThreads / 32;
        hstu_append_columns_kernel<T, H, true><<<static_cast<unsigned>((columns + kWarps - 1) / kWarps), kStagedThreads, kWarps * p.block * 512, stream>>>(p);
        return cudaGetLastError();
      }
    }
    constexpr int kWarps = kAppendThreads / 32;
    hstu_append_columns_kernel<T, H, false><<<static_cast<unsigned>((columns + kWarps - 1) / kWarps), kAppendThreads, 0, stream>>>(p);
  } else if (vec) hstu_append_kernel<T, H, 8><<<grid, kAppendThreads, 0, stream>>>(p);
  else hstu_append_kernel<T, H, 1><<<grid, kAppendThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_append(const HstuCacheAppendArgs& a, cudaStream_t stream) {
  AppendParams p;
  p.k = a.k;
  p.v = a.v;
  p.cache = static_cast<uint8_t*>(a.kv_cache);
  p.scale = static_cast<float*>(a.kv_scale);
  p.offset = a.seq_offset;
  p.tgt = a.num_target;
  p.page_offsets = a.page_offsets;
  p.page_ids = a.page_ids;
  p.last_page_len = a.last_page_len;
  p.status = static_cast<uint32_t*>(a.status);
  p.total = a.total;
  p.num_pages = a.num_pages;
  p.num_page_ids = a.num_page_ids;
  p.index_bytes = a.index_bytes;
  p.batch = a.batch;
  p.page_size = a.page_size;
  p.block = a.block;
  p.heads = a.heads_k;
  p.dim = a.dim;
  if (a.held == HSTU_HELD_E4M3) {
    return a.dtype == HSTU_DTYPE_BF16   ? launch_append_t<__nv_bfloat16, E4m3>(p, stream)
           : a.dtype == HSTU_DTYPE_FP16 ? launch_append_t<__half, E4m3>(p, stream)
                                        : launch_append_t<float, E4m3>(p, stream);
  }
  return a.dtype == HSTU_DTYPE_BF16   ? launch_append_t<__nv_bfloat16, Int8>(p, stream)
         : a.dtype == HSTU_DTYPE_FP16 ? launch_append_t<__half, Int8>(p, stream)
                                      : launch_append_t<float, Int8>(p, stream);
}

}  // namespace hstu
