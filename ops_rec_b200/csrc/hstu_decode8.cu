// hstu_paged_8bit for few query rows: one new event per user, or a handful, against a long cached history (bf16 / fp16 queries,
// head dims that are multiples of 16 up to 128, no targets, pages of whole 16-row tiles).
//
// HBM-bound: a decode step reads every visible cached row once, at one byte per element (128 users of 200 - 2048 rows, 8 heads
// of 128: 294 MB, 46 us; it takes 65, 4.5 TB/s), and there is little to compute per byte.  So nothing is staged: a warp streams
// pairs of tiles of 16 keys through a ring of its own in shared memory (cp.async, two stages of a pair, no barrier of the CTA in
// the loop; TMA boxes of 16 rows of 128 bytes, one for keys and one for values, came in at 3.4 TB/s at most, whatever the number
// of CTAs), turns the 8-bit numbers into 16-bit ones in registers where the matrix instructions want them, and keeps its rows of
// the output in registers.  What is left above the bytes is the set-up of a CTA, a thousand instructions a warp (4 users of 14000
// - 20000 rows: 40 us of 22; 512 users with a window of 1024, 541 MB: 103 of 84).
// There is no softmax: partial outputs of any split of the keys add up, first over the four warps of a CTA, then - where a
// sequence has more keys than a CTA takes - over CTAs: each leaves its partial sums in the workspace, and the last one to arrive
// adds them in the order of the keys (the same bits every time).
//
// The rows of a call are (query, head of the group) pairs of one key head: grouped heads share the cache's reads.  Both products
// have the cache as their A operand (16 keys, 16 columns of the head) and the rows as the eight columns of B, so that one row
// does not cost what sixteen do.
//   S^T = K.Q^T    bf16 queries are divided by a power of two per row, which keeps all 8 bits of every element that counts.  A
//                  thread's 16 bytes of a key are contiguous; the same permutation of the contraction is applied to Q.  The
//                  key's scale, alpha and the row's power of two multiply the 32-bit score.
//   P              silu(x) * (scale of the value's block), rounded once (two halves in fp16 calls), divided by a power of two per row that follows the
//                  largest P so far (raised, and the output rescaled, when P outgrows 2^14), since neither scores nor scales
//                  keep P inside fp16's narrow range
//   O^T += V^T.P^T V is read with ldmatrix.trans as pairs of bytes; the even columns of the head are the rows 0-7 of A, the odd
//                  ones the rows 8-15.  P changes from accumulator to operand with movmatrix.
// tcgen05 would need M = 128 rows and its operands in shared memory in 16 bits: the conversion would go through shared memory
// twice for a tile of which one row counts.
#include "hstu_mma8.cuh"

namespace hstu {

namespace {

constexpr int kDecWarps = 4, kDecThreads = 32 * kDecWarps;
constexpr int kDecKeys = 16;      // keys of a tile
constexpr int kPair = 2;          // tiles a warp works on at a time: their chains of dependent steps overlap

template <int D> struct DecCfg {
  static constexpr int kRows = 8;                               // rows of a CTA
  static constexpr int kStages = 2;                             // of kPair tiles each
  static constexpr int kTile = kDecKeys * D;                    // bytes of K (V) of a tile
  static constexpr int kStage = kPair * 2 * kTile;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kScales = kDecWarps * kStages * kPair * 2 * kDecKeys * 4;
  static constexpr int kSmem = kDecWarps * kRing + kScales;   // and 16 bytes per tile
  static_assert(kDecWarps * kRing >= kDecWarps * kRows * D * 4, "the rings hold the warps' partial outputs at the end");
};

struct DecParams {
  KParams f;
  uint32_t* counters;   // [batch * hk], of CTAs that have left their sums
  float* partial;       // [slots][hk][rows][D]
  int splits, tiles, by_pages, rows;   // see Split; rows of a partial sum
  int block_shift;      // log2 of a scale's block, 4 at most (a tile has one scale from there on)
  // ceil(2^32 / n): x / n is the upper half of the product, exactly, while x n < 2^32 (a warp with 20 tiles to do feels a
  // handful of divisions)
  uint32_t by_hk, by_ratio, by_page, by_block;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {   // (the rest of the 16 becomes zeros)
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
// (CTAs an SM: what 96 and 168 registers allow; without the bound some instantiations take 118 and 134, four of the one kind)
template <int D, typename T, typename H, bool kWin, bool kTanh>
__global__ void __launch_bounds__(kDecThreads, D == 64 ? 5 : 3) hstu_decode8_kernel(const DecParams d) {
  using C = DecCfg<D>;
  using Mask = MaskOf<kWin>;
  constexpr bool kFine = std::is_same<T, __half>::value;
  const KParams& p = d.f;
  extern __shared__ __align__(128) uint8_t ring_of_all[];
  long long* const s_row = reinterpret_cast<long long*>(ring_of_all + C::kSmem);   // where a tile's keys start in the cache, -1: no such page
  long long* const s_scale = s_row + d.tiles;                                      // where its scales start
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int b = over(blockIdx.x, d.by_hk), hk = blockIdx.x - b * p.hk, split = blockIdx.y;

  const SeqInfo s = load_seq(p, b);
  const int ratio = p.gqa_ratio, rows = min(s.lq * ratio, C::kRows);   // the group's heads inside a query
  long long pg0 = load_index(p.page_offsets, p.index_bytes, b), pg1 = load_index(p.page_offsets, p.index_bytes, b + 1);
  if (pg0 < 0) pg0 = 0;
  if (pg1 > p.num_page_ids) pg1 = p.num_page_ids;
  if (hk == 0 && split == 0) report_sequence<kDecThreads>(p, b, pg0, pg1);
  KeyTiles tiles = rows > 0 ? Mask::tiles(p, s, 0, s.lq, kDecKeys) : KeyTiles{0, 0, 0};
  tiles.n = min(tiles.n, d.splits * d.tiles);   // (lengths beyond the table's pages: flagged)
  // CTAs that share the keys, evenly, in whole rounds of the four warps' pairs
  int active = 1;
  while (active * d.tiles < tiles.n) ++active;
  if (active > 1) {
    active = min(active, most_partials(p, d.by_pages, b, d.splits, d.tiles));
    tiles.n = min(tiles.n, active * d.tiles);   // (more keys than pages: flagged)
  }
  constexpr int kRound = kDecWarps * kPair;
  const int each = active == 1 ? d.tiles : (tiles.n + active * kRound - 1) / (active * kRound) * kRound;
  const int t0 = split * each, t1 = min(tiles.n, t0 + each);
  if (rows <= 0 || split >= active) {   // uniform over the CTA
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  // The places of this CTA's tiles: a tile lies in one page.
  const int per_page = p.page_size / p.scale_block, row_bytes = p.hk * p.dqk;
  for (int i = tid; i < t1 - t0; i += kDecThreads) {
    const int key = key_of_tile(tiles, t0 + i, kDecKeys), slot = over(key, d.by_page), in_page = key - slot * p.page_size;
    const long long pid = pg0 + slot < pg1 ? load_index(p.page_ids, p.index_bytes, pg0 + slot) : -1;
    const bool ok = pid >= 0 && pid < p.num_pages;
    s_row[i] = ok ? (pid * 2 * p.page_size + in_page) * row_bytes : -1;
    s_scale[i] = ok ? (pid * 2 * per_page + over(in_page, d.by_block)) * p.hk : 0;
  }
  __syncthreads();

  float* const scales_of_mine = reinterpret_cast<float*>(ring_of_all + kDecWarps * C::kRing) + warp * C::kStages * kPair * 2 * kDecKeys;
  const uint32_t ring_at = ptx::smem_u32(ring_of_all) + warp * C::kRing;
  constexpr int kChunks = D / 16, kAtOnce = 32 / kChunks;   // 16-byte chunks of a row, rows that 32 lanes copy at once
  const int my_row = lane / kChunks, my_chunk = lane % kChunks;
  const int bytes = my_chunk * 16 < p.dqk ? 16 : 0;         // (chunks behind the head read as zeros)
  const uint8_t* const from_lane = static_cast<const uint8_t*>(p.kv_cache) + my_row * row_bytes + hk * p.dqk + (bytes ? my_chunk * 16 : 0);
  const long long to_v = static_cast<long long>(p.page_size) * row_bytes;
  const int to_rows = kAtOnce * row_bytes;
  const float* scale_from = p.kv_scale + hk + ((lane < 16 ? 0 : per_page) + ((lane & 15) >> d.block_shift)) * static_cast<long long>(p.hk);
  // Requests tile t0 + i into a slot; rows behind the last cached one, and tiles behind the last, read as zeros.  (Chunks are permuted so that the
  // pieces of 16 bytes eight lanes read at once fall on different banks.)
  auto request_tile = [&](int i, int slot) {
    const long long at = i < t1 - t0 ? s_row[i] : -1;
    const int left = at < 0 ? 0 : s.lk - key_of_tile(tiles, t0 + i, kDecKeys);
    const uint32_t to = ring_at + slot * 2 * C::kTile;
    const uint8_t* k_at = from_lane + (at < 0 ? 0 : at);
    const uint8_t* v_at = k_at + to_v;
    auto copy = [&](auto whole) {
#pragma unroll
      for (int u = 0; u < kDecKeys / kAtOnce; ++u) {
        const int r = u * kAtOnce + my_row;
        const int k_ch = D == 128 ? my_chunk ^ ((r & 1) << 2) : my_chunk, v_ch = D == 128 ? my_chunk ^ (r & 7) : my_chunk ^ ((r >> 1) & 3);
        const bool on = decltype(whole)::value || r < left;
        cp16(to + r * D + k_ch * 16, on ? k_at : from_lane, on ? bytes : 0);
        cp16(to + C::kTile + r * D + v_ch * 16, on ? v_at : from_lane, on ? bytes : 0);
        k_at += to_rows;
        v_at += to_rows;
      }
    };
    if (left >= kDecKeys) copy(std::true_type{});
    else copy(std::false_type{});
    const bool on = (lane & 15) < left;
    cp4(ptx::smem_u32(scales_of_mine + slot * 2 * kDecKeys + lane), on ? scale_from + s_scale[i] : p.kv_scale, on);
  };
  // the pair of tiles `i` of this warp: warp + 8 i and warp + 8 i + 4
  auto request = [&](int i) {
#pragma unroll
    for (int u = 0; u < kPair; ++u) request_tile(warp + (i * kPair + u) * kDecWarps, (i % C::kStages) * kPair + u);
  };
  const int mine = (t1 - t0 - warp + kDecWarps * kPair - 1) / (kDecWarps * kPair);   // pairs of this warp
#pragma unroll
  for (int u = 0; u < C::kStages - 1; ++u) {
    if (u < mine) request(u);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // Q: row g, of each 64 columns the 16 from 16 c on.
  uint32_t qb[D / 16][2];
  float factor[2];   // of the rows 2 c and 2 c + 1: alpha and the power of two a row was divided by
  int query[2];      // and their queries
  {
    const int row = g < rows ? g : 0, i_row = over(row, d.by_ratio);
    const T* from = static_cast<const T*>(p.q) + ((s.q0 + i_row) * p.hq + hk * ratio + row - i_row * ratio) * p.dqk;
    uint32_t w[D / 8];   // pairs in memory's order
#pragma unroll
    for (int blk = 0; blk < D / 64; ++blk) {
      const bool in = g < rows && blk * 64 + 16 * c < p.dqk;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 v = in ? *reinterpret_cast<const uint4*>(from + blk * 64 + 16 * c + 8 * u) : make_uint4(0, 0, 0, 0);
        w[blk * 8 + 4 * u] = v.x, w[blk * 8 + 4 * u + 1] = v.y, w[blk * 8 + 4 * u + 2] = v.z, w[blk * 8 + 4 * u + 3] = v.w;
      }
    }
    const float f = to_fp16_row<T>(w, p.alpha);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      factor[e] = __shfl_sync(0xffffffffu, f, 4 * (2 * c + e));
      query[e] = over(min(2 * c + e, rows - 1), d.by_ratio);
    }
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qb[k][0] = w[(k >> 2) * 8 + (k & 3) * 2];
      qb[k][1] = w[(k >> 2) * 8 + (k & 3) * 2 + 1];
    }
  }
  // Tiles that every row sees whole (tile_is_full's rule).
  const int full_end = min(s.lk, s.lk - s.lq + 1), full_from = kWin ? win_anchor(s, s.lq - 1, 0) - p.window : 0;

  float o[D / 16][4];   // column 2 g of 16 in rows 2 c, 2 c + 1; column 2 g + 1
  float down[2] = {0x1p126f, 0x1p126f};   // what P of a row is multiplied by, a power of two
#pragma unroll
  for (int j = 0; j < D / 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  // this thread's places in a stage: K row g and g + 8, V for ldmatrix (lanes 0-7 and 16-23 name keys 0-7, the others 8-15)
  const int v_row = (lane & 7) + ((lane >> 3) & 1) * 8;

  for (int i = 0; i < mine; ++i) {
    if (i + C::kStages - 1 < mine) request(i + C::kStages - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
    __syncwarp();
    const uint32_t at = (i % C::kStages) * C::kStage;
    const uint8_t* const stage = ring_of_all + warp * C::kRing + at;
    const float* const scales = scales_of_mine + (i % C::kStages) * kPair * 2 * kDecKeys;
    float sc[kPair][4];   // keys g and g + 8, rows 2 c and 2 c + 1
#pragma unroll
    for (int t = 0; t < kPair; ++t) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
    for (int blk = 0; blk < D / 64; ++blk) {
      const int ch = D == 128 ? (4 * blk + c) ^ ((g & 1) << 2) : c;
      uint4 w[kPair][2];
#pragma unroll
      for (int t = 0; t < kPair; ++t) {
        w[t][0] = *reinterpret_cast<const uint4*>(stage + t * 2 * C::kTile + g * D + ch * 16);
        w[t][1] = *reinterpret_cast<const uint4*>(stage + t * 2 * C::kTile + (g + 8) * D + ch * 16);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int t = 0; t < kPair; ++t) {
          uint32_t a[4];
          to_halves<H>(reinterpret_cast<const uint32_t*>(&w[t][0])[k], a[0], a[2]);
          to_halves<H>(reinterpret_cast<const uint32_t*>(&w[t][1])[k], a[1], a[3]);
          mma16816(sc[t], a, qb[4 * blk + k]);
        }
    }
    // P
    float pv[kPair][4], m[2] = {0.f, 0.f};
    int key[kPair];
    bool full = true;
#pragma unroll
    for (int t = 0; t < kPair; ++t) {
      const float* at_scales = scales + t * 2 * kDecKeys;
      const float ks[2] = {at_scales[g], at_scales[g + 8]}, vs[2] = {at_scales[kDecKeys + g], at_scales[kDecKeys + g + 8]};
      key[t] = key_of_tile(tiles, t0 + warp + (i * kPair + t) * kDecWarps, kDecKeys);
      full &= key[t] + kDecKeys <= full_end && (!kWin || key[t] > full_from || key[t] + kDecKeys <= p.sink);
#pragma unroll
      for (int e = 0; e < 4; ++e) pv[t][e] = silu_of<kTanh>(sc[t][e] * (ks[e >> 1] * factor[e & 1])) * vs[e >> 1];
    }
    if (!full) {   // (a select, not a multiply: a masked score may be anything; a tile behind the last one has scales of zero)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const typename Mask::Bounds rb = Mask::bounds(p, s, query[e]);
#pragma unroll
        for (int t = 0; t < kPair; ++t) {
          if (!allowed(rb, key[t] + g)) pv[t][e] = 0.f;
          if (!allowed(rb, key[t] + g + 8)) pv[t][2 + e] = 0.f;
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kPair; ++t) {
      m[0] = fmaxf(m[0], fmaxf(fabsf(pv[t][0]), fabsf(pv[t][2])));
      m[1] = fmaxf(m[1], fmaxf(fabsf(pv[t][1]), fabsf(pv[t][3])));
    }
    bool finite = true;
    if (__any_sync(0xffffffffu, m[0] * down[0] > 16384.f || m[1] * down[1] > 16384.f)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], x));
        finite &= !(m[e] > 3.402823466e38f);
        if (!(m[e] * down[e] > 16384.f) || m[e] > 3.402823466e38f) continue;
        const float next = down_to_one(m[e]), ratio2 = next / down[e];
        down[e] = next;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) o[j][e] *= ratio2, o[j][2 + e] *= ratio2;
      }
    }
    // In fp16 calls P is two halves, the rounded one and what it leaves: rounded once it costs as much again as the output's own
    // rounding (1.4 times the error; 3 bits less than fp16's, bf16's output does not notice).
    uint32_t pb[kPair][2], pl[kPair][2];
#pragma unroll
    for (int t = 0; t < kPair; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = pv[t][2 * h] * down[0], y = pv[t][2 * h + 1] * down[1];
        const uint32_t rounded = pack2<__half>(x, y);
        pb[t][h] = transposed(rounded);
        if (kFine) {   // (of an infinite P there is nothing left)
          const float2 r = unpack2<__half>(rounded);
          pl[t][h] = transposed(finite ? pack2<__half>(x - r.x, y - r.y) : 0u);
        }
      }
    // O^T += V^T.P^T
    const uint32_t v_at = ring_at + at + C::kTile + v_row * D;
#pragma unroll
    for (int t = 0; t < kPair; ++t)
#pragma unroll
      for (int j = 0; j < D / 16; j += 2) {
        const int chunk = j + (lane >> 4);
        uint32_t w[4];
        ldsm_x4_trans(v_at + t * 2 * C::kTile + (D == 128 ? chunk ^ (v_row & 7) : chunk ^ ((v_row >> 1) & 3)) * 16, w);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t a[4];   // columns 2 g (a pair of keys) and 2 g + 1, keys 0-7; the same, keys 8-15
          to_halves<H>(__byte_perm(w[2 * u], 0u, 0x3120), a[0], a[1]);
          to_halves<H>(__byte_perm(w[2 * u + 1], 0u, 0x3120), a[2], a[3]);
          mma16816(o[j + u], a, pb[t]);
          if (kFine) mma16816(o[j + u], a, pl[t]);
        }
      }
    __syncwarp();   // the stage is free
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();   // every warp is through with its ring
  // The warps' outputs, added in order.
  float* all = reinterpret_cast<float*>(ring_of_all);   // [warps][rows][D]
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float f = 1.f / down[e];
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
      *reinterpret_cast<float2*>(all + (warp * C::kRows + 2 * c + e) * D + 16 * j + 2 * g) = make_float2(o[j][e] * f, o[j][2 + e] * f);
  }
  __syncthreads();
  const long long group = blockIdx.x;
  const long long first = active > 1 ? first_partial(p, d.by_pages, b, d.splits, d.tiles) : 0;
  auto partial_of = [&](int n) { return d.partial + ((first + n) * p.hk + hk) * d.rows * D; };
  auto store = [&](int r, int col, float4 v) {
    if (col >= p.dqk) return;
    const int i_row = over(r, d.by_ratio);
    T* to = static_cast<T*>(p.out) + ((s.q0 + i_row) * p.hq + hk * ratio + r - i_row * ratio) * p.dqk + col;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(v.x * p.scale, v.y * p.scale), pack2<T>(v.z * p.scale, v.w * p.scale));
  };
  for (int i = tid; i < rows * (D / 4); i += kDecThreads) {
    const int r = i / (D / 4), col = i % (D / 4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(all + (w * C::kRows + r) * D + col);
      v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
    if (active == 1) store(r, col, v);
    else *reinterpret_cast<float4*>(partial_of(split) + r * D + col) = v;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the counters are cleared (and this grid ends after that one)
  if (active == 1) return;
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(d.counters + group, 1u) == static_cast<unsigned>(active - 1) ? 1 : 0;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  for (int i = tid; i < rows * (D / 4); i += kDecThreads) {
    const int r = i / (D / 4), col = i % (D / 4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int n = 0; n < active; ++n) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(partial_of(n) + r * D + col));
      v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
    store(r, col, v);
  }
}

int tile_width(const KParams& p) { return p.dqk <= 64 ? 64 : 128; }

// Some six CTAs per SM (three fit): fewer, and sequences of different lengths do not even out; more, and set-up and partial
// sums - a thousand instructions a warp, where a tile takes 300 - are what the SMs do.  Attention alone, us, at 4 / 6 / 8 / 12: 128
// users of 200 - 2048 rows and 8 heads 64 / 66 / 70 / 75, 4 users of 14000 - 20000 44 / 39 / 45 / 50.  With a loose bound of the
// lengths (1000 users of 60 - 128 rows, max_seq_len_k 128 / 20480): one head 14.6 / 18.7 us, 8 heads 70 / 86.
Split plan(const KParams& p) { return split_keys(p, 8, kDecWarps * kPair, 6 * 148, 1); }
uint64_t counters_bytes(const KParams& p) {
  return (static_cast<uint64_t>(p.batch) * p.hk * 4 + 255) & ~static_cast<uint64_t>(255);
}

template <int D, typename T, typename H>
cudaError_t launch_dec(const DecParams& d, const Split& pl, cudaStream_t stream) {
  using C = DecCfg<D>;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  auto kern = kBf16 && tanh_silu(d.f) ? (d.f.window ? hstu_decode8_kernel<D, T, H, true, kBf16> : hstu_decode8_kernel<D, T, H, false, kBf16>)
                                      : (d.f.window ? hstu_decode8_kernel<D, T, H, true, false> : hstu_decode8_kernel<D, T, H, false, false>);
  const int smem = C::kSmem + 16 * pl.tiles;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(d.f.batch) * d.f.hk, pl.splits, 1);
  cfg.blockDim = dim3(kDecThreads);
  cfg.dynamicSmemBytes = smem;
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
         static_cast<long long>(p.maxq) * p.gqa_ratio <= DecCfg<64>::kRows;
}

uint64_t decode8_workspace(const KParams& p) {
  return kWsHeaderBytes + counters_bytes(p) + static_cast<uint64_t>(plan(p).slots) * p.hk * p.maxq * p.gqa_ratio * tile_width(p) * 4;
}

cudaError_t launch_decode8(const KParams& p, int dtype, void* workspace, cudaStream_t stream) {
  const Split pl = plan(p);
  DecParams d;
  d.f = p;
  d.f.ws_header = static_cast<uint32_t*>(workspace);
  char* base = static_cast<char*>(workspace) + kWsHeaderBytes;
  d.counters = reinterpret_cast<uint32_t*>(base);
  d.partial = reinterpret_cast<float*>(base + counters_bytes(p));
  d.splits = pl.splits;
  d.tiles = pl.tiles;
  d.by_pages = pl.by_pages;
  d.rows = p.maxq * p.gqa_ratio;
  // (at most 2^20 heads of sequences by 16, 8 rows by 8, 20480 keys by a page of any size)
  d.by_hk = inverse_of(p.hk);
  d.by_ratio = inverse_of(p.gqa_ratio);
  d.by_page = inverse_of(p.page_size);
  d.by_block = inverse_of(p.scale_block);
  d.block_shift = 4;
  while (d.block_shift > 0 && (1 << d.block_shift) > p.scale_block) --d.block_shift;
  const long long n = pl.splits > 1 ? static_cast<long long>(p.batch) * p.hk : 0;
  clear_kernel<<<static_cast<unsigned>(n / 256 + 1), 256, 0, stream>>>(d.f.ws_header, d.counters, n);
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
