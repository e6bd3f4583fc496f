// hstu_paged_8bit for few query rows: one new event per user, or a handful, against a long cached history (bf16 / fp16 queries,
// head dims that are multiples of 16 up to 128, no targets, pages of whole 16-row tiles).
//
// HBM-bound: a decode step reads every visible cached row once, at one byte per element (128 users of 200 - 2048 rows, 8 heads
// of 128: 294 MB, 46 us), and there is next to nothing to compute per byte.  So nothing is staged: a warp streams tiles of 16 keys
// through a ring of its own in shared memory (cp.async, four stages in flight, no barrier of the CTA in the loop), turns the 8-bit
// numbers into 16-bit ones in registers where the matrix instructions want them, and keeps its 16 rows of the output in registers.
// There is no softmax: partial outputs of any split of the keys add up, first over the four warps of a CTA, then - where a
// sequence has more keys than a CTA takes - over CTAs: each leaves its partial sums in the workspace, and the last one to arrive
// adds them in the order of the keys (the same bits every time).
//
// The rows of a call are (query, head of the group) pairs of one key head, 16 at a time: grouped heads share the cache's reads.
//   S = Q.K^T      mma.sync m16n8k16 in fp16: e4m3 and int8 numbers are exact there, one conversion per pair; bf16 queries are
//                  scaled by a power of two per row (their largest element to [1, 2)), which keeps all 8 bits of every element
//                  that counts.  A thread's 16 bytes of a key are contiguous; the same permutation of the contraction is applied
//                  to Q.  The key's scale, alpha and the row's power of two multiply the 32-bit score.
//   P              silu(x) * (scale of the value's block), rounded to 16 bits once: in bf16 as it is; in fp16 divided by a power
//                  of two per row that follows the largest P so far (raised, and the output rescaled, when P outgrows 2^14),
//                  since neither scores nor scales keep P inside fp16's narrow range
//   O += P.V       V is read with ldmatrix.trans as pairs of bytes, which puts the even and the odd columns of the head into
//                  two B operands.  bf16: the bits of an e4m3 number, shifted into place, are the number times 2^-120 (and
//                  exact, the small ones as subnormals); P carries 2^60 of what is missing, the output the rest.
// tcgen05 would need M = 128 rows and its operands in shared memory in 16 bits: the conversion would go through shared memory
// twice for a tile of which one row counts.
#include <type_traits>

#include "hstu_held.cuh"

namespace hstu {

namespace {

constexpr int kDecWarps = 4, kDecThreads = 32 * kDecWarps;
constexpr int kDecKeys = 16;      // keys of a tile
constexpr int kDecRows = 16;      // rows of a CTA
constexpr int kDecMostTiles = 128;   // of a CTA

template <int D> struct DecCfg {
  static constexpr int kStages = 4;
  static constexpr int kTile = kDecKeys * D;                    // bytes of K (V) of a tile
  static constexpr int kStage = 2 * kTile + 2 * kDecKeys * 4;   // K, V and their scales
  static constexpr int kRing = kStages * kStage;
  static constexpr int kSmem = kDecWarps * kRing;
  static_assert(kSmem >= kDecWarps * kDecRows * D * 4, "the rings hold the warps' partial outputs at the end");
};

struct DecParams {
  KParams f;
  uint32_t* counters;   // [batch * hk * row blocks], of CTAs that have left their sums
  float* partial;       // [batch * hk * row blocks][splits][rows][D]
  int splits, tiles, rows;   // CTAs along the keys, tiles of a CTA, rows of a partial block
  int block_shift;      // log2 of a scale's block, 4 at most (a tile has one scale from there on)
};

__device__ __forceinline__ uint32_t smem_of(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The bytes 0, 1 (2, 3) of w as two halves.
template <typename H, bool kHigh> __device__ __forceinline__ uint32_t halves_of(uint32_t w) {
  if constexpr (std::is_same<H, E4m3>::value) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(kHigh ? w >> 16 : w & 0xffffu), __NV_E4M3);
    return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
  } else {
    // 0x6400 + (v + 128) is 1024 + 128 + v
    const uint32_t u = __byte_perm(w ^ 0x80808080u, 0x64646464u, kHigh ? 0x4342 : 0x4140);
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(1152.f, 1152.f));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
}
// The bytes 0, 2 (kOdd: 1, 3) of w as a pair of the call's type, times 2^-120 where it is bf16 and the cache e4m3.
template <typename H, typename T, bool kOdd> __device__ __forceinline__ uint32_t pair_of(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) {
    return halves_of<H, false>(__byte_perm(w, 0u, kOdd ? 0x4431 : 0x4420));
  } else if constexpr (std::is_same<H, E4m3>::value) {
    return kOdd ? ((w >> 4) & 0x07f007f0u) | (w & 0x80008000u) : ((w << 4) & 0x07f007f0u) | ((w << 8) & 0x80008000u);
  } else {
    // 0x4b000000 + (v + 128) is 2^23 + 128 + v
    const uint32_t u = w ^ 0x80808080u;
    const float lo = __uint_as_float(__byte_perm(u, 0x4b000000u, kOdd ? 0x7441 : 0x7440)) - 8388736.f;
    const float hi = __uint_as_float(__byte_perm(u, 0x4b000000u, kOdd ? 0x7443 : 0x7442)) - 8388736.f;
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
// Whether a byte of w is an e4m3 NaN, which shifted into a bf16's place would be the number 480.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// pair_of() of bytes that may be NaN.
template <bool kOdd> __device__ __forceinline__ uint32_t pair_with_nan(uint32_t w) {
  const uint32_t v = pair_of<E4m3, __nv_bfloat16, kOdd>(w), nan = kOdd ? nan_bytes(w) : nan_bytes(w) << 8;
  return v | ((nan & 0x8000u) ? 0x7fffu : 0u) | ((nan & 0x80000000u) ? 0x7fff0000u : 0u);
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Clears the status word and the counters; the attention kernel, launched with programmatic stream serialization, streams
// keys meanwhile and waits before it touches either.
__global__ void hstu_decode8_init_kernel(uint32_t* header, uint32_t* counters, long long n) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i == 0) header[0] = 0;
  if (i < n) counters[i] = 0;
}

template <int D, typename T, typename H, bool kWin>
__global__ void __launch_bounds__(kDecThreads) hstu_decode8_kernel(const DecParams d) {
  using C = DecCfg<D>;
  using Mask = MaskOf<kWin>;
  const KParams& p = d.f;
  extern __shared__ __align__(128) uint8_t ring_of_all[];
  __shared__ long long s_row[kDecMostTiles];     // first row of the tile's keys in the cache, -1: no such page
  __shared__ long long s_scale[kDecMostTiles];   // its place in the scales
  __shared__ int s_last;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int b = blockIdx.x / p.hk, hk = blockIdx.x - b * p.hk, split = blockIdx.y, r_first = blockIdx.z * kDecRows;

  const SeqInfo s = load_seq(p, b);
  const int ratio = p.gqa_ratio, rows = s.lq * ratio - r_first;   // rows of this block, the group's heads inside a query
  long long pg0 = load_index(p.page_offsets, p.index_bytes, b), pg1 = load_index(p.page_offsets, p.index_bytes, b + 1);
  if (pg0 < 0) pg0 = 0;
  if (pg1 > p.num_page_ids) pg1 = p.num_page_ids;
  // What a call's index tensors say wrongly goes into the status word, once per sequence.
  if (hk == 0 && split == 0 && blockIdx.z == 0) {
    unsigned st = 0;
    if (tid == 0) st = check_seq(p, read_seq(p, b)) | check_page_count(p, b);
    for (long long i = pg0 + tid; i < pg1; i += kDecThreads) {
      const long long pid = load_index(p.page_ids, p.index_bytes, i);
      if (pid < 0 || pid >= p.num_pages) st |= HSTU_ST_BAD_PAGES;
    }
    if (st) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      atomicOr(p.ws_header, st);
    }
  }
  const int q_lo = r_first / ratio, q_n = (min(rows, kDecRows) + r_first + ratio - 1) / ratio - q_lo;   // the block's queries
  const KeyTiles tiles = rows > 0 ? Mask::tiles(p, s, q_lo, q_n, kDecKeys) : KeyTiles{0, 0, 0};
  const int active = max(1, (tiles.n + d.tiles - 1) / d.tiles);   // CTAs that share this block's keys
  const int t0 = split * d.tiles, t1 = min(tiles.n, t0 + d.tiles);
  if (rows <= 0 || split >= active) {   // uniform over the CTA
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  // The places of this CTA's tiles: a tile lies in one page.
  const int per_page = p.page_size / p.scale_block;
  for (int i = tid; i < t1 - t0; i += kDecThreads) {
    const int key = key_of_tile(tiles, t0 + i, kDecKeys), slot = key / p.page_size, in_page = key - slot * p.page_size;
    const long long pid = pg0 + slot < pg1 ? load_index(p.page_ids, p.index_bytes, pg0 + slot) : -1;
    const bool ok = pid >= 0 && pid < p.num_pages;
    s_row[i] = ok ? pid * 2 * p.page_size + in_page : -1;
    s_scale[i] = ok ? (pid * 2 * per_page + in_page / p.scale_block) * p.hk + hk : -1;
  }
  __syncthreads();

  uint8_t* ring = ring_of_all + warp * C::kRing;
  const uint32_t ring_at = smem_of(ring);
  const uint8_t* cache = static_cast<const uint8_t*>(p.kv_cache);
  const long long row_bytes = static_cast<long long>(p.hk) * p.dqk;
  constexpr int kChunks = D / 16;   // 16-byte chunks of a row
  // Requests tile t0 + i into stage i's slot: rows behind the last cached one and chunks behind the head read as zeros.
  auto request = [&](int i, int stage) {
    const long long row0 = s_row[i];
    const int left = s.lk - key_of_tile(tiles, t0 + i, kDecKeys);
    const uint32_t to = ring_at + stage * C::kStage;
#pragma unroll
    for (int u = 0; u < kDecKeys * kChunks / 32; ++u) {
      const int at = u * 32 + lane, r = at / kChunks, ch = at % kChunks;
      const bool on = row0 >= 0 && r < left && ch * 16 < p.dqk;
      const uint8_t* k_from = on ? cache + (row0 + r) * row_bytes + hk * p.dqk + ch * 16 : cache;
      const uint8_t* v_from = on ? k_from + p.page_size * row_bytes : cache;
      // (the chunks are permuted so that eight lanes' 16 bytes of a load fall on different banks)
      const int k_ch = D == 128 ? ch ^ ((r & 1) << 2) : ch, v_ch = D == 128 ? ch ^ (r & 7) : ch ^ ((r >> 1) & 3);
      cp16(to + r * D + k_ch * 16, k_from, on);
      cp16(to + C::kTile + r * D + v_ch * 16, v_from, on);
    }
    const int r = lane & 15;
    const bool on = row0 >= 0 && r < left;
    cp4(to + 2 * C::kTile + lane * 4,
        on ? p.kv_scale + s_scale[i] + ((lane < 16 ? 0 : per_page) + (r >> d.block_shift)) * static_cast<long long>(p.hk) : p.kv_scale, on);
  };
  const int mine = (t1 - t0 - warp + kDecWarps - 1) / kDecWarps;   // tiles of this warp: warp, warp + 4, ..
#pragma unroll
  for (int u = 0; u < C::kStages - 1; ++u) {
    if (u < mine) request(warp + u * kDecWarps, u);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // Q: rows g and g + 8 of the block; of each 64 columns the 16 from 16 c on.
  uint32_t qa[D / 16][4];
  float factor[2];   // alpha and the power of two a row was divided by
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h;
    const bool on = r < rows;
    const T* from = static_cast<const T*>(p.q) + ((s.q0 + (on ? (r_first + r) / ratio : 0)) * p.hq + hk * ratio + (on ? (r_first + r) % ratio : 0)) * p.dqk;
    uint32_t w[D / 8];   // the thread's pairs, in memory's order
#pragma unroll
    for (int blk = 0; blk < D / 64; ++blk) {
      const bool in = on && blk * 64 + 16 * c < p.dqk;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 v = in ? *reinterpret_cast<const uint4*>(from + blk * 64 + 16 * c + 8 * u) : make_uint4(0, 0, 0, 0);
        w[blk * 8 + 4 * u] = v.x, w[blk * 8 + 4 * u + 1] = v.y, w[blk * 8 + 4 * u + 2] = v.z, w[blk * 8 + 4 * u + 3] = v.w;
      }
    }
    factor[h] = p.alpha;
    if (!kHalf) {
      uint32_t top = 0;   // the largest exponent of the row (its bits: of finite values; an infinity keeps the row as it is)
#pragma unroll
      for (int u = 0; u < D / 8; ++u) top = max(top, max(w[u] & 0x7f80u, (w[u] >> 16) & 0x7f80u));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = top == 0x7f80u || top == 0 ? 0 : static_cast<int>(top >> 7) - 127;
      // (in two steps: 2^-e alone may lie outside of the normal range)
      const float down1 = __uint_as_float(static_cast<uint32_t>(127 - e / 2) << 23), down2 = __uint_as_float(static_cast<uint32_t>(127 - (e - e / 2)) << 23);
      const float up1 = __uint_as_float(static_cast<uint32_t>(127 + e / 2) << 23), up2 = __uint_as_float(static_cast<uint32_t>(127 + (e - e / 2)) << 23);
      factor[h] = p.alpha * up1 * up2;
#pragma unroll
      for (int u = 0; u < D / 8; ++u) {
        const float lo = __uint_as_float(w[u] << 16) * down1 * down2, hi = __uint_as_float(w[u] & 0xffff0000u) * down1 * down2;
        w[u] = pack2<__half>(lo, hi);
      }
    }
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qa[k][h] = w[(k >> 2) * 8 + (k & 3) * 2];
      qa[k][2 + h] = w[(k >> 2) * 8 + (k & 3) * 2 + 1];
    }
  }
  typename Mask::Bounds bounds[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) bounds[h] = Mask::bounds(p, s, min((r_first + min(g + 8 * h, rows - 1)) / ratio, s.lq - 1));

  float o[D / 16][2][4];   // even and odd columns of 16
#pragma unroll
  for (int j = 0; j < D / 16; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) o[j][e >> 2][e & 3] = 0.f;
  constexpr bool kShifted = std::is_same<H, E4m3>::value && !kHalf;   // V's numbers come times 2^-120
  constexpr float kUp = kShifted ? 0x1p60f : 1.f;
  const float p_scale = kHalf ? 1.f : p.scale * kUp;
  float down[2] = {0x1p126f, 0x1p126f};   // (fp16) what P of a row is multiplied by, a power of two

  for (int n = 0; n < mine; ++n) {
    if (n + C::kStages - 1 < mine) request(warp + (n + C::kStages - 1) * kDecWarps, (n + C::kStages - 1) % C::kStages);
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
    __syncwarp();
    const uint8_t* at = ring + (n % C::kStages) * C::kStage;
    const float* scales = reinterpret_cast<const float*>(at + 2 * C::kTile);
    // scores of the keys 0 .. 7 and 8 .. 15
    float sc[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
      const int r = 8 * t + g;
#pragma unroll
      for (int blk = 0; blk < D / 64; ++blk) {
        const int ch = D == 128 ? (4 * blk + c) ^ ((r & 1) << 2) : c;
        const uint4 w = *reinterpret_cast<const uint4*>(at + r * D + ch * 16);
        mma16816<__half>(sc[t], qa[4 * blk], halves_of<H, false>(w.x), halves_of<H, true>(w.x));
        mma16816<__half>(sc[t], qa[4 * blk + 1], halves_of<H, false>(w.y), halves_of<H, true>(w.y));
        mma16816<__half>(sc[t], qa[4 * blk + 2], halves_of<H, false>(w.z), halves_of<H, true>(w.z));
        mma16816<__half>(sc[t], qa[4 * blk + 3], halves_of<H, false>(w.w), halves_of<H, true>(w.w));
      }
    }
    // P
    const int key = key_of_tile(tiles, t0 + warp + n * kDecWarps, kDecKeys);
    const bool full = Mask::full(p, s, q_lo, q_n, key, kDecKeys);
    float pv[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float2 ks = *reinterpret_cast<const float2*>(scales + 8 * t + 2 * c);
      const float2 vs = *reinterpret_cast<const float2*>(scales + kDecKeys + 8 * t + 2 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = sc[t][e] * ((e & 1 ? ks.y : ks.x) * factor[e >> 1]);
        const float sg = rcp(1.f + ex2(x * -1.4426950408889634f));
        pv[t][e] = x * sg * ((e & 1 ? vs.y : vs.x) * p_scale);
        // (a select, not a multiply: a masked score may be anything)
        if (!full && !allowed(bounds[e >> 1], key + 8 * t + 2 * c + (e & 1))) pv[t][e] = 0.f;
      }
    }
    if (kHalf) {
      float top[2];
      bool grow = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(fmaxf(fabsf(pv[0][2 * h]), fabsf(pv[0][2 * h + 1])), fmaxf(fabsf(pv[1][2 * h]), fabsf(pv[1][2 * h + 1])));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        grow |= top[h] * down[h] > 16384.f;
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!(top[h] * down[h] > 16384.f) || top[h] > 3.402823466e38f) continue;
          // the largest P to [1, 2)
          const float next = __uint_as_float((254u - min(__float_as_uint(top[h]) >> 23, 253u)) << 23), ratio = next / down[h];
          down[h] = next;
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) o[j][u][2 * h] *= ratio, o[j][u][2 * h + 1] *= ratio;
        }
      }
    }
    uint32_t pa[4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        pa[2 * t + h] = pack2<T>(pv[t][2 * h] * (kHalf ? down[h] : 1.f), pv[t][2 * h + 1] * (kHalf ? down[h] : 1.f));
    // O += P.V
    const uint32_t v_at = ring_at + (n % C::kStages) * C::kStage + C::kTile;
    const int v_row = (lane & 7) + ((lane >> 3) & 1) * 8;   // ldmatrix: lanes 0-7 and 16-23 name keys 0-7, the others 8-15
    uint32_t w[D / 32][4];
    uint32_t nan = 0;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const int chunk = 2 * j + (lane >> 4);
      ldsm_x4_trans(v_at + v_row * D + (D == 128 ? chunk ^ (v_row & 7) : chunk ^ ((v_row >> 1) & 3)) * 16, w[j]);
      if (kShifted) {
#pragma unroll
        for (int u = 0; u < 4; ++u) nan |= nan_bytes(w[j][u]);
      }
    }
    if (kShifted && __any_sync(0xffffffffu, nan != 0)) {
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          mma16816<T>(o[2 * j + u][0], pa, pair_with_nan<false>(w[j][2 * u]), pair_with_nan<false>(w[j][2 * u + 1]));
          mma16816<T>(o[2 * j + u][1], pa, pair_with_nan<true>(w[j][2 * u]), pair_with_nan<true>(w[j][2 * u + 1]));
        }
    } else {
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          mma16816<T>(o[2 * j + u][0], pa, pair_of<H, T, false>(w[j][2 * u]), pair_of<H, T, false>(w[j][2 * u + 1]));
          mma16816<T>(o[2 * j + u][1], pa, pair_of<H, T, true>(w[j][2 * u]), pair_of<H, T, true>(w[j][2 * u + 1]));
        }
    }
    __syncwarp();   // the stage is free
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();   // every warp is through with its ring
  // The warps' outputs, added in order.
  float* all = reinterpret_cast<float*>(ring_of_all);   // [warps][16][D]
#pragma unroll
  for (int j = 0; j < D / 16; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float4 v = make_float4(o[j][0][2 * h], o[j][1][2 * h], o[j][0][2 * h + 1], o[j][1][2 * h + 1]);
      const float f = kHalf ? 1.f / down[h] : kUp;
      v.x *= f, v.y *= f, v.z *= f, v.w *= f;
      *reinterpret_cast<float4*>(all + (warp * kDecRows + g + 8 * h) * D + 16 * j + 4 * c) = v;
    }
  __syncthreads();
  const int valid = min(rows, kDecRows);
  const float o_scale = kHalf ? p.scale : 1.f;
  const long long group = static_cast<long long>(blockIdx.x) * gridDim.z + blockIdx.z;
  auto store = [&](int r, int col, float4 v) {
    if (col >= p.dqk) return;
    const int row = r_first + r;
    T* to = static_cast<T*>(p.out) + ((s.q0 + row / ratio) * p.hq + hk * ratio + row % ratio) * p.dqk + col;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
  };
  for (int i = tid; i < valid * (D / 4); i += kDecThreads) {
    const int r = i / (D / 4), col = i % (D / 4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(all + (w * kDecRows + r) * D + col);
      v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
    v.x *= o_scale, v.y *= o_scale, v.z *= o_scale, v.w *= o_scale;
    if (active == 1) store(r, col, v);
    else *reinterpret_cast<float4*>(d.partial + ((group * d.splits + split) * d.rows + r) * D + col) = v;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the counters are cleared (and this grid ends after that one)
  if (active == 1) return;
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(d.counters + group, 1u) == static_cast<unsigned>(active - 1) ? 1 : 0;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  for (int i = tid; i < valid * (D / 4); i += kDecThreads) {
    const int r = i / (D / 4), col = i % (D / 4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int n = 0; n < active; ++n) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(d.partial + ((group * d.splits + n) * d.rows + r) * D + col));
      v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
    store(r, col, v);
  }
}

// How a call is split: tiles of a CTA, CTAs along the keys, blocks of rows.
struct DecPlan {
  int tiles, splits, row_blocks, rows;
};
DecPlan plan(const KParams& p) {
  DecPlan d;
  const long long rows = static_cast<long long>(p.maxq) * p.gqa_ratio;
  d.row_blocks = static_cast<int>((rows + kDecRows - 1) / kDecRows);
  d.rows = rows < kDecRows ? static_cast<int>(rows) : kDecRows;
  long long most = (p.maxk + kDecKeys - 1) / kDecKeys;   // tiles of the longest sequence
  long long all = p.num_page_ids * p.page_size / kDecKeys;   // and of all of them together, at most
  if (p.window) {
    const long long seen = (static_cast<long long>(p.window) + p.maxq) / kDecKeys + 2 + (p.sink + kDecKeys - 1) / kDecKeys;
    if (seen < most) most = seen;
    if (seen * p.batch < all) all = seen * p.batch;
  }
  // Some twelve CTAs per SM, so that sequences of different lengths even out; a CTA of fewer than 8 tiles (two per warp) is
  // mostly set-up.
  long long tiles = all * p.hk * d.row_blocks / (12ll * 148);
  tiles = tiles < 8 ? 8 : tiles > kDecMostTiles ? kDecMostTiles : tiles;
  d.tiles = static_cast<int>((tiles + kDecWarps - 1) / kDecWarps * kDecWarps);
  d.splits = static_cast<int>((most + d.tiles - 1) / d.tiles);
  if (d.splits < 1) d.splits = 1;
  return d;
}
uint64_t counters_bytes(const KParams& p, const DecPlan& d) {
  return (static_cast<uint64_t>(p.batch) * p.hk * d.row_blocks * 4 + 255) & ~static_cast<uint64_t>(255);
}
int tile_width(const KParams& p) { return p.dqk <= 64 ? 64 : 128; }

template <int D, typename T, typename H>
cudaError_t launch_dec(const DecParams& d, const DecPlan& pl, cudaStream_t stream) {
  using C = DecCfg<D>;
  auto kern = d.f.window ? hstu_decode8_kernel<D, T, H, true> : hstu_decode8_kernel<D, T, H, false>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(d.f.batch) * d.f.hk, pl.splits, pl.row_blocks);
  cfg.blockDim = dim3(kDecThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, d);
}

}  // namespace

// Whether a call runs here.  The pointers count: rows are read in pieces of 16 bytes.
bool decode8_supported(const KParams& p, int dtype) {
  const uintptr_t align = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.kv_cache);
  const bool blocks = p.scale_block % kDecKeys == 0 || kDecKeys % p.scale_block == 0;
  return (dtype == HSTU_DTYPE_BF16 || dtype == HSTU_DTYPE_FP16) && p.dqk % 16 == 0 && p.dqk <= 128 && !p.tgt && blocks &&
         p.page_size % kDecKeys == 0 && (align & 15u) == 0 && !(p.flags & HSTU_FLAG_FORCE_GENERIC) &&
         static_cast<long long>(p.maxq) * p.gqa_ratio <= 64;
}

uint64_t decode8_workspace(const KParams& p) {
  const DecPlan d = plan(p);
  const uint64_t partial = d.splits > 1 ? static_cast<uint64_t>(p.batch) * p.hk * d.row_blocks * d.splits * d.rows * tile_width(p) * 4 : 0;
  return kWsHeaderBytes + counters_bytes(p, d) + partial;
}

cudaError_t launch_decode8(const KParams& p, int dtype, void* workspace, cudaStream_t stream) {
  const DecPlan pl = plan(p);
  DecParams d;
  d.f = p;
  d.f.ws_header = static_cast<uint32_t*>(workspace);
  char* base = static_cast<char*>(workspace) + kWsHeaderBytes;
  d.counters = reinterpret_cast<uint32_t*>(base);
  d.partial = reinterpret_cast<float*>(base + counters_bytes(p, pl));
  d.splits = pl.splits;
  d.tiles = pl.tiles;
  d.rows = pl.rows;
  d.block_shift = 4;
  while (d.block_shift > 0 && (1 << d.block_shift) > p.scale_block) --d.block_shift;
  const long long n = pl.splits > 1 ? static_cast<long long>(p.batch) * p.hk * pl.row_blocks : 0;
  hstu_decode8_init_kernel<<<static_cast<unsigned>(n / 256 + 1), 256, 0, stream>>>(d.f.ws_header, d.counters, n);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.total_q == 0) return e;
  const bool wide = tile_width(p) == 128, held = p.held == HSTU_HELD_E4M3;
  if (dtype == HSTU_DTYPE_BF16) {
    if (wide) return held ? launch_dec<128, __nv_bfloat16, E4m3>(d, pl, stream) : launch_dec<128, __nv_bfloat16, Int8>(d, pl, stream);
    return held ? launch_dec<64, __nv_bfloat16, E4m3>(d, pl, stream) : launch_dec<64, __nv_bfloat16, Int8>(d, pl, stream);
  }
  if (wide) return held ? launch_dec<128, __half, E4m3>(d, pl, stream) : launch_dec<128, __half, Int8>(d, pl, stream);
  return held ? launch_dec<64, __half, E4m3>(d, pl, stream) : launch_dec<64, __half, Int8>(d, pl, stream);
}

}  // namespace hstu
