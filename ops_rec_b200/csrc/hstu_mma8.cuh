// What the two kernels that read an 8-bit cache in place share (hstu_decode8.cu: up to eight rows, hstu_rows8.cu: more): matrix
// instructions with the cache as their A operand, the conversions in front of them, and SiLU.  All operands are fp16, whatever
// the call's type: e4m3 and int8 numbers are exact there and take one conversion per pair (bf16 has no such instruction, and
// five integer operations per pair made the decode kernel issue-bound), and P has three bits more than in bf16.
#pragma once

#include <type_traits>

#include "hstu_held.cuh"
#include "ptx_sm100.cuh"

namespace hstu {
namespace {

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// An 8 x 8 matrix of halves, a row's pair per thread -> its transpose.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// The four numbers of w as two pairs of halves.
template <typename H> __device__ __forceinline__ void to_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (std::is_same<H, E4m3>::value) {
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // 0x6400 + (v + 128) is 1024 + 128 + v
    const uint32_t u = w ^ 0x80808080u, ul = __byte_perm(u, 0x64646464u, 0x4140), uh = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = __floats2half2_rn(1152.f, 1152.f);
    const __half2 l = __hsub2(*reinterpret_cast<const __half2*>(&ul), off), h = __hsub2(*reinterpret_cast<const __half2*>(&uh), off);
    lo = *reinterpret_cast<const uint32_t*>(&l);
    hi = *reinterpret_cast<const uint32_t*>(&h);
  }
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
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
// The power of two that brings m (finite, normal) to [1, 2); 2^-126 at least.
__device__ __forceinline__ float down_to_one(float m) {
  return __uint_as_float((254u - min(__float_as_uint(m) >> 23, 253u)) << 23);
}

// x / (1 + exp(-x)).  kTanh: x (1 + tanh(x / 2)) / 2, one SFU operation instead of two, where the framework's other kernels take
// that form too (tanh_silu()).
template <bool kTanh> __device__ __forceinline__ float silu_of(float x) {
  if (kTanh) {
    const float h = 0.5f * x;
    return fmaf(h, ptx::tanh_approx(h), h);
  }
  return x * ptx::rcp_approx(1.f + ptx::ex2_approx(x * -1.4426950408889634f));
}

// x / n by the upper half of a product with ceil(2^32 / n), exact while x n < 2^32; the inverse of 1 is 0.
__device__ __forceinline__ int over(int x, uint32_t inverse) {
  return static_cast<int>(inverse ? __umulhi(static_cast<uint32_t>(x), inverse) : static_cast<uint32_t>(x));
}
inline uint32_t inverse_of(int n) { return n == 1 ? 0u : static_cast<uint32_t>(((1ull << 32) + n - 1) / n); }

// Clears the status word and the counters; the attention kernel, launched with programmatic stream serialization, streams
// keys meanwhile and waits before it touches either.
__global__ void clear_kernel(uint32_t* header, uint32_t* counters, long long n) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i == 0) header[0] = 0;
  if (i < n) counters[i] = 0;
}

// What a call's index tensors say wrongly about sequence b goes into the status word (by one CTA per sequence).
template <int kThreads> __device__ __forceinline__ void report_sequence(const KParams& p, int b, long long pg0, long long pg1) {
  unsigned st = 0;
  if (threadIdx.x == 0) st = check_seq(p, read_seq(p, b)) | check_page_count(p, b);
  for (long long i = pg0 + threadIdx.x; i < pg1; i += kThreads) {
    const long long pid = load_index(p.page_ids, p.index_bytes, i);
    if (pid < 0 || pid >= p.num_pages) st |= HSTU_ST_BAD_PAGES;
  }
  if (st) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    atomicOr(p.ws_header, st);
  }
}

// Where the CTAs that share a sequence's keys leave their partial sums, and how many of them may: in slots of one CTA per key head
// and block of rows.  Either every sequence has `splits` slots, or - many sequences, few of them long - sequence b has the slots
// [2 f(b), 2 f(b + 1)) with f(b) = the tiles in front of its pages / tiles of a CTA, rounded down: whoever needs n > 1 CTAs has
// pages of more than n - 1 times a CTA's tiles, so f grows by n - 1 at least.
__device__ __forceinline__ long long tiles_before(const KParams& p, int b, int tiles) {
  const long long pg = load_index(p.page_offsets, p.index_bytes, b);
  return min(max(pg, 0ll), p.num_page_ids) * (p.page_size / 16) / tiles;
}
__device__ __forceinline__ long long first_partial(const KParams& p, bool by_pages, int b, int splits, int tiles) {
  return by_pages ? 2 * tiles_before(p, b, tiles) : static_cast<long long>(b) * splits;
}
__device__ __forceinline__ int most_partials(const KParams& p, bool by_pages, int b, int splits, int tiles) {
  return by_pages ? static_cast<int>(min(max(2 * (tiles_before(p, b + 1, tiles) - tiles_before(p, b, tiles)), 1ll), static_cast<long long>(splits))) : splits;
}

// How a call is split: tiles of 16 keys of a CTA, CTAs along the keys of a sequence, slots of partial sums.
struct Split {
  int tiles, splits, by_pages;
  long long slots;
};
// least: of a CTA's tiles; ctas: of the whole GPU, that fill it evenly; blocks: of rows.
inline Split split_keys(const KParams& p, int least, int step, long long ctas, int blocks) {
  long long most = (p.maxk + 15) / 16;                              // tiles of the longest sequence
  const long long pages = p.num_page_ids * (p.page_size / 16);      // and of all of them together, at most
  long long all = pages;
  if (all < most) most = all;
  if (p.window) {
    const long long seen = (static_cast<long long>(p.window) + p.maxq) / 16 + 2 + (p.sink + 15) / 16;
    if (seen < most) most = seen;
    if (seen * p.batch < all) all = seen * p.batch;
  }
  const long long heads = static_cast<long long>(p.hk) * blocks;
  long long tiles = all * heads / ctas;
  // Where the bound of the lengths is far above most of them, most CTAs find nothing to do, which costs as much as two tiles: at
  // most some 32 per SM and one for 8 tiles that there are, beside the one that each problem has.
  const long long busy = most * p.batch * heads / (32ll * 148 + all * heads / 8);
  if (tiles < busy) tiles = busy;
  if (tiles < least) tiles = least;
  if (tiles > most) tiles = most > least ? most : least;
  Split s;
  s.tiles = static_cast<int>((tiles + step - 1) / step * step);
  s.splits = static_cast<int>((most + s.tiles - 1) / s.tiles);
  if (s.splits < 1) s.splits = 1;
  const long long by_pages = 2 * (pages / s.tiles) + 2, each = static_cast<long long>(p.batch) * s.splits;
  s.by_pages = by_pages < each ? 1 : 0;
  s.slots = s.splits > 1 ? (s.by_pages ? by_pages : each) : 0;
  return s;
}

// Eight query rows as the B operands of S^T = K.Q^T: a bf16 row is divided by a power of two (its largest element to [1, 2)).
// Returns alpha times that power.  w: this thread's pairs of one row; the four threads of a lane group hold the rest of it.
template <typename T, int kPairs> __device__ __forceinline__ float to_fp16_row(uint32_t (&w)[kPairs], float alpha) {
  if constexpr (std::is_same<T, __half>::value) {
    return alpha;
  } else {
    uint32_t top = 0;   // the largest exponent of the row; an infinity or NaN leaves the row as it is
#pragma unroll
    for (int u = 0; u < kPairs; ++u) top = max(top, max(w[u] & 0x7f80u, (w[u] >> 16) & 0x7f80u));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = top == 0x7f80u || top == 0 ? 0 : static_cast<int>(top >> 7) - 127;
    const float d1 = power_of_two(-(e / 2)), d2 = power_of_two(-(e - e / 2));   // (2^-e itself may lie outside of fp32's normal range)
#pragma unroll
    for (int u = 0; u < kPairs; ++u)
      w[u] = pack2<__half>(__uint_as_float(w[u] << 16) * d1 * d2, __uint_as_float(w[u] & 0xffff0000u) * d1 * d2);
    return alpha * power_of_two(e / 2) * power_of_two(e - e / 2);
  }
}

}  // namespace
}  // namespace hstu
