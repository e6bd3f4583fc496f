// hstu_paged_8bit for more rows than hstu_decode8.cu takes - several new events, and candidates to rank - in place: bf16 / fp16
// queries, head dims that are multiples of 16 up to 128, pages of whole 16-row tiles.
//
// What bounds such a call is arithmetic per score (4096 users of 271 cached rows and 48 queries on average, 4 heads of 64:
// 128 us of bytes, 28 us of products on the tcgen05 pipe, but 260 million scores, 59 us of SFU) and the latency of a problem this
// small: a (user, head) has 17 tiles of 16 keys.  So as in the decode kernel nothing is staged in memory, and the matrix
// instructions have the cache as their A operand; but here a warp owns rows - two groups of eight - and all four warps of a CTA
// share the tiles: 32 keys at a time arrive in a ring of raw numbers (cp.async, three stages ahead; each thread reads back only
// what it fetched itself), are turned into fp16 once, and put into one of two buffers, one barrier per 32 keys.  (64 users of 200 -
// 2048 rows, 4 heads of 64, 80 rows: 43 us, where pages unpacked for the tcgen05 kernel take 74; 128 users, 8 heads of 128, 9
// rows: 245 of 46 of bytes.  With many more problems than the SMs hold the set-up of each counts, and unpacking wins.)
//   S^T = K.Q^T, O^T += V^T.P^T   ldmatrix, for V with .trans; P changes from accumulator to operand with movmatrix
//   P    SiLU(x) times the value's scale and the row's power of two (see hstu_decode8.cu: rounded once, in fp16 calls two halves); the products around SiLU
//        on pairs of scores (tanh on two halves at once is no faster, and 1 + tanh from halves is 2^-12 off where it is small)
// Targets see the cached keys as a row right behind the history would; what they see of each other - their own group, up to
// themselves - is added at the end in 32 bits (groups of up to four; with one target per group a row's own key and value).
#include <algorithm>

#include "hstu_mma8.cuh"

namespace hstu {

namespace {

constexpr int kRwKeys = 16;        // keys of a tile
constexpr int kRwStage = 32;       // keys of a stage: two tiles
constexpr int kRwRows = 64;        // of a CTA
constexpr int kRwMostGroup = 4;    // targets of a group
constexpr int kRwMostRows = 256;   // of a sequence and key head

template <int D> struct RwCfg {
  static constexpr int kGroups = 2, kWarps = kRwRows / 8 / kGroups, kThreads = 32 * kWarps;   // groups of eight rows of a warp
  static constexpr int kTile = kRwStage * D * 2;       // bytes of a stage's K (V) in fp16
  static constexpr int kPitch = D + 4;                 // of the output's rows in floats: eight columns of four rows, 32 banks
  static constexpr int kOut = kRwRows * kPitch * 4;
  static constexpr int kDepth = 4;                     // stages of the ring of raw numbers
  static constexpr int kRaw = kRwStage * D * 2;        // bytes of a stage: K and V
  static constexpr int kBuffers = 4 * kTile > kOut ? 4 * kTile : kOut;
  static constexpr int kSmem = kBuffers + kDepth * (kRaw + 2 * kRwStage * 4);   // and 16 bytes per tile
};

struct RwParams {
  KParams f;
  uint32_t* counters;   // [batch * hk * row blocks], of CTAs that have left their sums
  float* partial;       // [slots][hk][row blocks][rows][D]
  int splits, tiles, by_pages, rows;   // see Split; rows of a partial sum
  int block_shift;      // log2 of a scale's block, 4 at most
  uint32_t by_hk, by_ratio, by_page, by_block, by_group;   // over()
};

__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {   // (off: zeros)
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
template <bool kTanh> __device__ __forceinline__ float2 silu_pair(float2 x) {
  if (kTanh) {
    const float2 h = __fmul2_rn(x, make_float2(0.5f, 0.5f));
    return __ffma2_rn(h, make_float2(ptx::tanh_approx(h.x), ptx::tanh_approx(h.y)), h);
  }
  return make_float2(silu_of<false>(x.x), silu_of<false>(x.y));
}

template <int D, typename T, typename H, bool kWin, bool kTanh>
__global__ void __launch_bounds__(RwCfg<D>::kThreads) hstu_rows8_kernel(const RwParams d) {
  using C = RwCfg<D>;
  constexpr int kRwGroups = C::kGroups, kRwWarps = C::kWarps, kRwThreads = C::kThreads;
  using Mask = MaskOf<kWin>;
  constexpr bool kFine = std::is_same<T, __half>::value;
  const KParams& p = d.f;
  extern __shared__ __align__(256) uint8_t smem[];   // [2][K, V][32][D] halves; at the end the output
  long long* const s_row = reinterpret_cast<long long*>(smem + C::kSmem);   // where the tile's keys start in the cache, -1: no such page
  long long* const s_scale = s_row + d.tiles;                               // and its scales
  __shared__ float s_factor[2][2][kRwStage];         // scales of a stage's keys and values
  __shared__ float s_own[kRwRows][kRwMostGroup];     // SiLU of a target's scores with its group
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int b = over(blockIdx.x, d.by_hk), hk = blockIdx.x - b * p.hk, split = blockIdx.y, r_first = blockIdx.z * kRwRows;

  // The cached keys alone, [0, cached).  A target counts as row `hist_rows` (with s.lq, s.lk one more than the history's rows and
  // keys, the mask's len_k - len_q is the call's).
  SeqInfo s = load_seq(p, b);
  const int total_rows = s.lq, targets = s.tgt, hist_rows = s.lq - s.tgt, cached = s.lk - s.tgt;
  s.tgt = 0;
  s.lq = hist_rows + (targets > 0 ? 1 : 0);
  s.lk = cached + (targets > 0 ? 1 : 0);
  const int ratio = p.gqa_ratio, rows = min(total_rows * ratio - r_first, kRwRows);   // rows of this block
  long long pg0 = load_index(p.page_offsets, p.index_bytes, b), pg1 = load_index(p.page_offsets, p.index_bytes, b + 1);
  if (pg0 < 0) pg0 = 0;
  if (pg1 > p.num_page_ids) pg1 = p.num_page_ids;
  if (hk == 0 && split == 0 && blockIdx.z == 0) report_sequence<kRwThreads>(p, b, pg0, pg1);
  const int q_lo = over(r_first, d.by_ratio), q_n = over(rows + r_first + ratio - 1, d.by_ratio) - q_lo;   // the block's queries
  const int v_lo = min(q_lo, hist_rows), v_n = min(q_lo + q_n - 1, hist_rows) - v_lo + 1;
  KeyTiles tiles = rows > 0 ? Mask::tiles(p, s, v_lo, v_n, kRwKeys) : KeyTiles{0, 0, 0};
  if (tiles.n > 0 && key_of_tile(tiles, tiles.n - 1, kRwKeys) >= cached) tiles.n -= 1;   // (the targets' own place)
  tiles.n = min(tiles.n, d.splits * d.tiles);   // (lengths beyond the table's pages: flagged)
  // CTAs that share this block's keys, evenly, in whole stages
  int active = 1;
  while (active * d.tiles < tiles.n) ++active;
  if (active > 1) {
    active = min(active, most_partials(p, d.by_pages, b, d.splits, d.tiles));
    tiles.n = min(tiles.n, active * d.tiles);   // (more keys than pages: flagged)
  }
  const int each = active == 1 ? d.tiles : (tiles.n + 2 * active - 1) / (2 * active) * 2;
  const int t0 = split * each, nt = min(tiles.n - t0, each);   // first tile, number of tiles
  if (rows <= 0 || split >= active) {   // uniform over the CTA
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int per_page = p.page_size / p.scale_block, row_bytes = p.hk * p.dqk;
  for (int i = tid; i < nt; i += kRwThreads) {
    const int key = key_of_tile(tiles, t0 + i, kRwKeys), slot = over(key, d.by_page), in_page = key - slot * p.page_size;
    const long long pid = pg0 + slot < pg1 ? load_index(p.page_ids, p.index_bytes, pg0 + slot) : -1;
    const bool ok = pid >= 0 && pid < p.num_pages;
    s_row[i] = ok ? (pid * 2 * p.page_size + in_page) * row_bytes : -1;
    s_scale[i] = ok ? (pid * 2 * per_page + over(in_page, d.by_block)) * p.hk + hk : 0;
  }
  __syncthreads();

  // This thread's numbers of a stage: chunk my_chunk of the rows my_row, my_row + 16; and, of 64 threads, a scale.
  constexpr int kChunks = D / 16, kStep = kRwThreads / kChunks, kPer = kRwStage / kStep;
  const int my_row = tid / kChunks, my_chunk = tid % kChunks;
  const bool in_row = my_chunk * 16 < p.dqk;
  const long long to_v = static_cast<long long>(p.page_size) * row_bytes;
  const uint8_t* const from = static_cast<const uint8_t*>(p.kv_cache) + hk * p.dqk + my_chunk * 16;
  uint8_t* const raw = smem + C::kBuffers + tid * 16;                                               // [kDepth][kPer][K, V][threads]
  float* const raw_scale = reinterpret_cast<float*>(smem + C::kBuffers + C::kDepth * C::kRaw) + tid;   // [kDepth][2 * 32]
  // Rows behind the last cached one, chunks behind the head and tiles behind the last read as zeros.
  auto fetch = [&](int stage) {
    const int slot = stage % C::kDepth;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int r = my_row + u * kStep, tile = 2 * stage + (r >> 4);
      const bool on = tile < nt && in_row && s_row[tile] >= 0 && key_of_tile(tiles, t0 + tile, kRwKeys) + (r & 15) < cached;
      const uint8_t* at = on ? from + s_row[tile] + (r & 15) * row_bytes : static_cast<const uint8_t*>(p.kv_cache);
      const uint32_t to = ptx::smem_u32(raw + slot * C::kRaw + u * 2 * kRwThreads * 16);
      cp16(to, at, on);
      cp16(to + kRwThreads * 16, on ? at + to_v : at, on);
    }
    if (tid < 2 * kRwStage) {
      const int r = tid & (kRwStage - 1), tile = 2 * stage + (r >> 4);
      const bool on = tile < nt && s_row[tile] >= 0 && key_of_tile(tiles, t0 + tile, kRwKeys) + (r & 15) < cached;
      const float* at = on ? p.kv_scale + s_scale[tile] + ((tid < kRwStage ? 0 : per_page) + ((r & 15) >> d.block_shift)) * static_cast<long long>(p.hk)
                           : p.kv_scale;
      cp4(ptx::smem_u32(raw_scale + slot * 2 * kRwStage), at, on);
    }
  };
  // a 16-byte chunk (eight halves) of row r: eight rows' chunks of one column lie in different banks
  auto place = [](int r, int chunk) { return r * D * 2 + (((chunk ^ r) & 7) | (chunk & 8)) * 16; };
  auto convert = [&](int stage) {
    const int buf = stage & 1, slot = stage % C::kDepth;
    uint8_t* to = smem + buf * 2 * C::kTile;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int r = my_row + u * kStep;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint4 w = *reinterpret_cast<const uint4*>(raw + slot * C::kRaw + (u * 2 + kv) * kRwThreads * 16);
        uint4 lo, hi;
        to_halves<H>(w.x, lo.x, lo.y);
        to_halves<H>(w.y, lo.z, lo.w);
        to_halves<H>(w.z, hi.x, hi.y);
        to_halves<H>(w.w, hi.z, hi.w);
        *reinterpret_cast<uint4*>(to + kv * C::kTile + place(r, 2 * my_chunk)) = lo;
        *reinterpret_cast<uint4*>(to + kv * C::kTile + place(r, 2 * my_chunk + 1)) = hi;
      }
    }
    if (tid < 2 * kRwStage) s_factor[buf][tid / kRwStage][tid % kRwStage] = raw_scale[slot * 2 * kRwStage];
  };
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  // (the stages up to the one that is converted next are complete)
  auto arrived = [] { asm volatile("cp.async.wait_group %0;" ::"n"(C::kDepth - 2) : "memory"); };
  const int stages = (nt + 1) / 2;
#pragma unroll
  for (int i = 0; i < C::kDepth - 1; ++i) {
    if (i < stages) fetch(i);
    commit();
  }

  // Q: the warp's groups warp and warp + 4, row g of each.
  uint32_t qb[kRwGroups][D / 16][2];
  float2 factor[kRwGroups];      // of the rows 2 c and 2 c + 1: alpha and the power of two a row was divided by
  int query[kRwGroups][2];       // and their queries, targets as row hist_rows
  int groups = 0;                // of this warp, that hold any rows
#pragma unroll
  for (int u = 0; u < kRwGroups; ++u) {
    const int base = 8 * (warp + kRwWarps * u);
    if (base < rows) groups = u + 1;
    const bool on = base + g < rows;
    const int row = on ? r_first + base + g : 0, i_row = over(row, d.by_ratio);
    const T* q_at = static_cast<const T*>(p.q) + ((s.q0 + i_row) * p.hq + hk * ratio + row - i_row * ratio) * p.dqk + 2 * c;
    uint32_t w[D / 8];
#pragma unroll
    for (int k = 0; k < D / 8; ++k) w[k] = on && 8 * k < p.dqk ? __ldg(reinterpret_cast<const uint32_t*>(q_at + 8 * k)) : 0u;
    const float f = to_fp16_row<T>(w, p.alpha);
    factor[u] = make_float2(__shfl_sync(0xffffffffu, f, 8 * c), __shfl_sync(0xffffffffu, f, 8 * c + 4));
#pragma unroll
    for (int e = 0; e < 2; ++e) query[u][e] = min(over(r_first + min(base + 2 * c + e, rows - 1), d.by_ratio), hist_rows);
#pragma unroll
    for (int k = 0; k < D / 16; ++k) qb[u][k][0] = w[2 * k], qb[u][k][1] = w[2 * k + 1];
  }
  // SiLU of what targets see of each other: a row by D / 8 lanes, eight columns each.
  const bool owns = targets > 0 && split == 0 && q_lo + q_n > hist_rows;
  const T* const k_new = static_cast<const T*>(p.k_new) + (s.q0 + hist_rows) * row_bytes + hk * p.dqk;
  const T* const v_new = static_cast<const T*>(p.v_new) + (s.q0 + hist_rows) * row_bytes + hk * p.dqk;
  if (owns) {
    constexpr int kLanes = D / 8;
    const int part = tid % kLanes;
    const bool in = part * 8 < p.dqk;
    constexpr int kAtOnce = kRwThreads / kLanes, kPasses = kRwRows / kAtOnce, kFly = 4;
    for (int pass = 0; pass < kPasses && pass * kAtOnce < rows; pass += kFly) {
      for (int j = 0; j < p.group; ++j) {
        uint4 q4[kFly], k4[kFly];
        bool on[kFly];
#pragma unroll
        for (int f = 0; f < kFly; ++f) {
          const int r = (pass + f) * kAtOnce + tid / kLanes, row = r_first + min(r, rows - 1), i_row = over(row, d.by_ratio);
          const int nth = i_row - hist_rows, first = nth < 0 ? 0 : over(nth, d.by_group) * p.group;
          on[f] = r < rows && nth >= 0 && first + j <= nth;
          q4[f] = k4[f] = make_uint4(0, 0, 0, 0);
          if (on[f] && in) {
            q4[f] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + ((s.q0 + i_row) * p.hq + hk * ratio + row - i_row * ratio) * p.dqk + part * 8));
            k4[f] = __ldg(reinterpret_cast<const uint4*>(k_new + static_cast<long long>(first + j) * row_bytes + part * 8));
          }
        }
#pragma unroll
        for (int f = 0; f < kFly; ++f) {
          float x = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 qf = unpack2<T>(reinterpret_cast<const uint32_t*>(&q4[f])[e]), kf = unpack2<T>(reinterpret_cast<const uint32_t*>(&k4[f])[e]);
            x = fmaf(qf.x, kf.x, fmaf(qf.y, kf.y, x));
          }
#pragma unroll
          for (int o2 = kLanes / 2; o2 > 0; o2 >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o2);
          if (part == 0 && on[f]) s_own[(pass + f) * kAtOnce + tid / kLanes][j] = silu_of<kTanh>(x * p.alpha);
        }
      }
    }
  }
  // Tiles that every row of the block sees whole (tile_is_full's rule).
  const int full_end = min(cached, v_lo + (s.lk - s.lq) + 1), full_from = kWin ? win_anchor(s, v_lo + v_n - 1, 0) - p.window : 0;

  float o[kRwGroups][D / 16][4];   // columns g and g + 8 of 16: rows 2 c, 2 c + 1 of the first, of the second
  float2 down[kRwGroups];          // what P of a row is multiplied by, a power of two
#pragma unroll
  for (int u = 0; u < kRwGroups; ++u) {
    down[u] = make_float2(0x1p126f, 0x1p126f);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[u][j][0] = o[u][j][1] = o[u][j][2] = o[u][j][3] = 0.f;
  }
  // ldmatrix: the keys and the column half of 16 this lane names, for K as it lies and for V transposed
  // (place() of chunk 2 k + half is this lane's address for k = 0 with the bits of 32 k flipped: rows are multiples of 128 bytes)
  const uint32_t k_lane = ptx::smem_u32(smem) + place((lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
  const uint32_t v_lane = ptx::smem_u32(smem) + C::kTile + place((lane & 7) + (lane >> 4) * 8, (lane >> 3) & 1);

  arrived();
  convert(0);
  __syncthreads();
  for (int i = 0; i < stages; ++i) {
    const int buf = i & 1;
    if (i + C::kDepth - 1 < stages) fetch(i + C::kDepth - 1);   // (into the slot of the stage before, converted two stages ago)
    commit();
    arrived();
    if (i + 1 < stages) convert(i + 1);   // (the buffer's readers are behind the barrier of the stage before)
#pragma unroll 1
    for (int t = 0; t < 2; ++t) {
      if (groups == 0 || 2 * i + t >= nt) break;
      const int key = key_of_tile(tiles, t0 + 2 * i + t, kRwKeys);
      const uint32_t tile_at = buf * 2 * C::kTile + t * 16 * D * 2;
      float sc[kRwGroups][4];   // keys g and g + 8: rows 2 c, 2 c + 1 of the first, of the second
#pragma unroll
      for (int u = 0; u < kRwGroups; ++u) sc[u][0] = sc[u][1] = sc[u][2] = sc[u][3] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t a[4];
        ldsm_x4((k_lane + tile_at) ^ (32 * k), a);
#pragma unroll
        for (int u = 0; u < kRwGroups; ++u)
          if (u < groups) mma16816(sc[u], a, qb[u][k]);
      }
      const bool full = key + kRwKeys <= full_end && (!kWin || key > full_from || key + kRwKeys <= p.sink);
      const float ks[2] = {s_factor[buf][0][t * 16 + g], s_factor[buf][0][t * 16 + g + 8]};
      const float vs[2] = {s_factor[buf][1][t * 16 + g], s_factor[buf][1][t * 16 + g + 8]};
      uint32_t pb[kRwGroups][2], pl[kRwGroups][2];   // pl: what the rounding of P leaves, in fp16 calls (see hstu_decode8.cu)
#pragma unroll
      for (int u = 0; u < kRwGroups; ++u) {
        if (u >= groups) continue;
        uint32_t see[2] = {0xffffffffu, 0xffffffffu};   // per key, the halves of the two rows
        if (!full) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const typename Mask::Bounds rb = Mask::bounds(p, s, query[u][e]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (key + g + 8 * h >= cached || !allowed(rb, key + g + 8 * h)) see[h] &= e ? 0x0000ffffu : 0xffff0000u;
          }
        }
        float2 y[2];   // per key, SiLU times the value's scale for the two rows
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 x = __fmul2_rn(make_float2(sc[u][2 * h], sc[u][2 * h + 1]), __fmul2_rn(factor[u], make_float2(ks[h], ks[h])));
          y[h] = __fmul2_rn(silu_pair<kTanh>(x), make_float2(vs[h], vs[h]));
        }
        // P times the row's power of two (a select of the bits: a masked score may be anything), and whether fp16 holds it with
        // room to spare
        auto form = [&]() {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 w = __fmul2_rn(y[h], down[u]);
            pb[u][h] = pack2<__half>(w.x, w.y);
            if (kFine) {
              const float2 r = unpack2<__half>(pb[u][h]);
              pl[u][h] = pack2<__half>(w.x - r.x, w.y - r.y) & see[h];
            }
            pb[u][h] &= see[h];
          }
          return __hble2(__hmax2_nan(__habs2(as_half2(pb[u][0])), __habs2(as_half2(pb[u][1]))), __floats2half2_rn(16384.f, 16384.f));
        };
        if (!__all_sync(0xffffffffu, form())) {   // (NaN too, to no avail)
          float top[2] = {0.f, 0.f};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (see[h] & 0xffffu) top[0] = fmaxf(top[0], fabsf(y[h].x));
            if (see[h] >> 16) top[1] = fmaxf(top[1], fabsf(y[h].y));
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int m = 4; m < 32; m <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], m));
            float& dn = e ? down[u].y : down[u].x;
            if (!(top[e] * dn > 16384.f) || top[e] > 3.402823466e38f) continue;
            const float next = down_to_one(top[e]), change = next / dn;
            dn = next;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) o[u][j][e] *= change, o[u][j][2 + e] *= change;
          }
          if (!form() && kFine) pl[u][0] = pl[u][1] = 0u;   // (nothing is left of an infinite P)
        }
        pb[u][0] = transposed(pb[u][0]);
        pb[u][1] = transposed(pb[u][1]);
        if (kFine) pl[u][0] = transposed(pl[u][0]), pl[u][1] = transposed(pl[u][1]);
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t a[4];
        ldsm_x4_trans((v_lane + tile_at) ^ (32 * j), a);
#pragma unroll
        for (int u = 0; u < kRwGroups; ++u)
          if (u < groups) {
            mma16816(o[u][j], a, pb[u]);
            if (kFine) mma16816(o[u][j], a, pl[u]);
          }
      }
    }
    __syncthreads();
  }
  float* out = reinterpret_cast<float*>(smem);   // [rows][kPitch]; every warp is through with the tiles
#pragma unroll
  for (int u = 0; u < kRwGroups; ++u) {
    if (u >= groups) continue;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float f = 1.f / (e ? down[u].y : down[u].x);
      float* to = out + (8 * (warp + kRwWarps * u) + 2 * c + e) * C::kPitch + g;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) to[16 * j] = o[u][j][e] * f, to[16 * j + 8] = o[u][j][2 + e] * f;
    }
  }
  __syncthreads();
  const long long group = static_cast<long long>(blockIdx.x) * gridDim.z + blockIdx.z;
  const long long first = active > 1 ? first_partial(p, d.by_pages, b, d.splits, d.tiles) : 0;
  auto partial_of = [&](int n) { return d.partial + (((first + n) * p.hk + hk) * gridDim.z + blockIdx.z) * d.rows * D; };
  auto store = [&](int r, int col, float4 v) {
    if (col >= p.dqk) return;
    const int row = r_first + r, i_row = over(row, d.by_ratio);
    T* to = static_cast<T*>(p.out) + ((s.q0 + i_row) * p.hq + hk * ratio + row - i_row * ratio) * p.dqk + col;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(v.x * p.scale, v.y * p.scale), pack2<T>(v.z * p.scale, v.w * p.scale));
  };
  constexpr int kFly = 4;
  for (int i0 = tid; i0 < rows * (D / 4); i0 += kFly * kRwThreads) {
    float4 v[kFly];
#pragma unroll
    for (int f = 0; f < kFly; ++f) {
      const int i = min(i0 + f * kRwThreads, rows * (D / 4) - 1), r = i / (D / 4), col = i % (D / 4) * 4;
      v[f] = *reinterpret_cast<const float4*>(out + r * C::kPitch + col);
    }
    if (owns) {
      for (int j = 0; j < p.group; ++j) {
        uint2 w[kFly];
        float pj[kFly];
#pragma unroll
        for (int f = 0; f < kFly; ++f) {
          const int i = min(i0 + f * kRwThreads, rows * (D / 4) - 1), r = i / (D / 4), col = i % (D / 4) * 4;
          const int nth = over(r_first + r, d.by_ratio) - hist_rows, first = nth < 0 ? 0 : over(nth, d.by_group) * p.group;
          w[f] = make_uint2(0, 0);
          pj[f] = 0.f;
          if (nth >= 0 && first + j <= nth && col < p.dqk) {
            w[f] = __ldg(reinterpret_cast<const uint2*>(v_new + static_cast<long long>(first + j) * row_bytes + col));
            pj[f] = s_own[r][j];
          }
        }
#pragma unroll
        for (int f = 0; f < kFly; ++f) {
          const float2 lo = unpack2<T>(w[f].x), hi = unpack2<T>(w[f].y);
          v[f].x = fmaf(pj[f], lo.x, v[f].x), v[f].y = fmaf(pj[f], lo.y, v[f].y);
          v[f].z = fmaf(pj[f], hi.x, v[f].z), v[f].w = fmaf(pj[f], hi.y, v[f].w);
        }
      }
    }
#pragma unroll
    for (int f = 0; f < kFly; ++f) {
      const int i = i0 + f * kRwThreads, r = i / (D / 4), col = i % (D / 4) * 4;
      if (i >= rows * (D / 4)) continue;
      if (active == 1) store(r, col, v[f]);
      else *reinterpret_cast<float4*>(partial_of(split) + r * D + col) = v[f];
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the counters are cleared (and this grid ends after that one)
  if (active == 1) return;
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(d.counters + group, 1u) == static_cast<unsigned>(active - 1) ? 1 : 0;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  for (int i = tid; i < rows * (D / 4); i += kRwThreads) {
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

int rows_of(const KParams& p) { return p.maxq * p.gqa_ratio; }
int row_blocks(const KParams& p) { return (rows_of(p) + kRwRows - 1) / kRwRows; }
// Some eight CTAs per SM, of at least 16 tiles: less is mostly set-up.  (A loose bound of the lengths - 1000 users of 60 - 128 rows, one
// head, 9 rows and 20 targets, max_seq_len_k 148 / 20480: 35 / 39 us.)
Split plan(const KParams& p) { return split_keys(p, 16, 2, 8 * 148, row_blocks(p)); }
uint64_t counters_bytes(const KParams& p) {
  return (static_cast<uint64_t>(p.batch) * p.hk * row_blocks(p) * 4 + 255) & ~static_cast<uint64_t>(255);
}

template <int D, typename T, typename H>
cudaError_t launch_rows(const RwParams& d, const Split& pl, cudaStream_t stream) {
  using C = RwCfg<D>;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  auto kern = kBf16 && tanh_silu(d.f) ? (d.f.window ? hstu_rows8_kernel<D, T, H, true, kBf16> : hstu_rows8_kernel<D, T, H, false, kBf16>)
                                      : (d.f.window ? hstu_rows8_kernel<D, T, H, true, false> : hstu_rows8_kernel<D, T, H, false, false>);
  const int smem = C::kSmem + 16 * pl.tiles;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(d.f.batch) * d.f.hk, pl.splits, row_blocks(d.f));
  cfg.blockDim = dim3(C::kThreads);
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

// Whether a call can run here.  The pointers count: rows are read in pieces of 16 bytes.
bool rows8_supported(const KParams& p, int dtype) {
  const uintptr_t align = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.kv_cache) |
                          (p.tgt ? reinterpret_cast<uintptr_t>(p.k_new) | reinterpret_cast<uintptr_t>(p.v_new) : 0);
  const bool blocks = p.scale_block % kRwKeys == 0 || kRwKeys % p.scale_block == 0;
  return (dtype == HSTU_DTYPE_BF16 || dtype == HSTU_DTYPE_FP16) && p.dqk % 16 == 0 && p.dqk <= 128 && (!p.tgt || p.group <= kRwMostGroup) &&
         blocks && p.page_size % kRwKeys == 0 && (align & 15u) == 0 && !(p.flags & HSTU_FLAG_FORCE_GENERIC) &&
         static_cast<long long>(p.maxq) * p.gqa_ratio <= kRwMostRows;
}

uint64_t rows8_workspace(const KParams& p) {
  const uint64_t slot = static_cast<uint64_t>(p.hk) * row_blocks(p) * std::min(rows_of(p), kRwRows) * tile_width(p) * 4;
  return kWsHeaderBytes + counters_bytes(p) + plan(p).slots * slot;
}

cudaError_t launch_rows8(const KParams& p, int dtype, void* workspace, cudaStream_t stream) {
  const Split pl = plan(p);
  RwParams d;
  d.f = p;
  d.f.ws_header = static_cast<uint32_t*>(workspace);
  char* base = static_cast<char*>(workspace) + kWsHeaderBytes;
  d.counters = reinterpret_cast<uint32_t*>(base);
  d.partial = reinterpret_cast<float*>(base + counters_bytes(p));
  d.splits = pl.splits;
  d.tiles = pl.tiles;
  d.by_pages = pl.by_pages;
  d.rows = std::min(rows_of(p), kRwRows);
  // (at most 2^20 heads of sequences by 16, 256 rows by 16, 20480 keys by a page of any size, 256 targets by 4)
  d.by_hk = inverse_of(p.hk);
  d.by_ratio = inverse_of(p.gqa_ratio);
  d.by_page = inverse_of(p.page_size);
  d.by_block = inverse_of(p.scale_block);
  d.by_group = inverse_of(p.group > 0 ? p.group : 1);
  d.block_shift = 4;
  while (d.block_shift > 0 && (1 << d.block_shift) > p.scale_block) --d.block_shift;
  const long long n = pl.splits > 1 ? static_cast<long long>(p.batch) * p.hk * row_blocks(p) : 0;
  clear_kernel<<<static_cast<unsigned>(n / 256 + 1), 256, 0, stream>>>(d.f.ws_header, d.counters, n);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.total_q == 0) return e;
  const bool wide = tile_width(p) == 128, held = p.held == HSTU_HELD_E4M3;
  if (dtype == HSTU_DTYPE_BF16) {
    if (wide) return held ? launch_rows<128, __nv_bfloat16, E4m3>(d, pl, stream) : launch_rows<128, __nv_bfloat16, Int8>(d, pl, stream);
    return held ? launch_rows<64, __nv_bfloat16, E4m3>(d, pl, stream) : launch_rows<64, __nv_bfloat16, Int8>(d, pl, stream);
  }
  if (wide) return held ? launch_rows<128, __half, E4m3>(d, pl, stream) : launch_rows<128, __half, Int8>(d, pl, stream);
  return held ? launch_rows<64, __half, E4m3>(d, pl, stream) : launch_rows<64, __half, Int8>(d, pl, stream);
}

}  // namespace hstu
