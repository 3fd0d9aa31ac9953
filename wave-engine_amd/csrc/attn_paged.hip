// A paged key-value cache (gfx950): rows written into pages and read back, as they
// are or in 8 bits, and the attention of one new token per sequence over it.
//
// Cache rows in 8 bits: scale = max(max |x| / 127, 2^-126) of a row in fp32, and
// x / scale to the nearest step, ties to even: |error| <= scale / 2.  A row that
// holds an infinity or NaN has the scale NaN, so it reads back as NaN.
//
// All of it is a stream over the cache, so the aim is bytes in flight; the decode's
// products run on MFMAs only because the G query heads of a group share every row
// they read (16 heads in one MFMA), not because they would bound it.
#include <hip/hip_runtime.h>

#include "wha_elem.hpp"
#include "wha_packed.hpp"

namespace wha {

namespace {

// Eight consecutive elements of a row as they lie in memory.
template <class C>
struct Raw;
template <>
struct Raw<float> {
  floatx4 a, b;
};
template <>
struct Raw<__bf16> {
  uintx4 a;
};
template <>
struct Raw<_Float16> {
  uintx4 a;
};
template <>
struct Raw<int8_t> {
  uintx2 a;
};

// Elements d .. d + 7 of a row (zeros past the head dim, all zeros if !on: then
// nothing is read).  VEC: D a multiple of 8, rows 16-byte aligned (int8: 8).
template <class C, bool VEC>
__device__ __forceinline__ Raw<C> load8(const C* row, int d, int D, bool on) {
  Raw<C> r;
  if constexpr (VEC) {
    const bool in = on && d < D;
    if constexpr (sizeof(C) == 4) {
      r.a = r.b = floatx4{0.f, 0.f, 0.f, 0.f};
      if (in) {
        r.a = *reinterpret_cast<const floatx4*>(row + d);
        r.b = *reinterpret_cast<const floatx4*>(row + d + 4);
      }
    } else if constexpr (sizeof(C) == 2) {
      r.a = uintx4{0u, 0u, 0u, 0u};
      if (in) r.a = *reinterpret_cast<const uintx4*>(row + d);
    } else {
      r.a = uintx2{0u, 0u};
      if (in) r.a = *reinterpret_cast<const uintx2*>(row + d);
    }
  } else {
    C x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = on && d + e < D ? row[d + e] : (C)0;
    __builtin_memcpy(&r, x, sizeof(x));
  }
  return r;
}
// 16 bytes through a buffer descriptor, past whose end is zero; not to be kept in
// the caches (every row of a cache is read once by a decode: 110 -> 96 us at one
// sequence of 131072 keys, 8 heads of 128 in bf16).
constexpr int kPastEnd = (int)0x80000000, kOnce = 2;
__device__ __forceinline__ uintx4 buffer_load16(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(uintx4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, kOnce));
}
// As numbers.
template <class C>
__device__ __forceinline__ void widen(const Raw<C>& r, float (&x)[8]) {
  if constexpr (sizeof(C) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = r.a[e], x[4 + e] = r.b[e];
  } else if constexpr (sizeof(C) == 2) {
    const typename Elem<C>::Frag f = __builtin_bit_cast(typename Elem<C>::Frag, r.a);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)f[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)(((r.a[e >> 2] ^ 0x80808080u) >> (8 * (e & 3))) & 255u) - 128.f;
  }
}
// Four 8-bit steps as two pairs of fp16: 0x6400 + u is 1024 + u, exactly.
__device__ __forceinline__ uintx2 steps_f16(unsigned w) {
  const unsigned u = w ^ 0x80808080u;
  const f16x2 bias = {(_Float16)1152.f, (_Float16)1152.f};
  const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
  const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
  return uintx2{__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi)};
}
// As a fragment of the type that the products are formed in (8-bit steps are
// exact in all of them).
template <class X, class C>
__device__ __forceinline__ typename Elem<X>::Frag as_frag(const Raw<C>& r) {
  if constexpr (std::is_same<X, C>::value && sizeof(X) == 2) {
    return __builtin_bit_cast(typename Elem<X>::Frag, r.a);
  } else if constexpr (std::is_same<X, _Float16>::value && std::is_same<C, int8_t>::value) {
    const uintx2 a = steps_f16(r.a[0]), b = steps_f16(r.a[1]);
    return __builtin_bit_cast(typename Elem<X>::Frag, (uintx4{a[0], a[1], b[0], b[1]}));
  } else {
    float x[8];
    widen(r, x);
    return Elem<X>::pack(x);
  }
}
template <class T, bool VEC>
__device__ __forceinline__ void store8(T* row, int d, int D, const float (&x)[8]) {
  if constexpr (VEC) {
    if (d >= D) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row + d) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(row + d + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      *reinterpret_cast<typename Elem<T>::Frag*>(row + d) = Elem<T>::pack(x);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (d + e < D) row[d + e] = (T)x[e];
  }
}

// Maximum over the 16 lanes of a row's group.
__device__ __forceinline__ float max16(float x) {
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) x = fmaxf(x, xor_shfl(x, m));
  return x;
}

constexpr int kRowsPerBlock = 16;  // 16 lanes to a row of up to 128 elements

// One row of k or v into the cache.
template <class T, class C, bool VEC>
__device__ __forceinline__ void write_row(const T* src, C* dst, float* scale_at, int D, int d) {
  const Raw<T> r = load8<T, VEC>(src, d, D, true);
  if constexpr (!std::is_same<C, int8_t>::value) {
    if constexpr (VEC) {
      if (d < D) *reinterpret_cast<Raw<T>*>(dst + d) = r;
    } else {
      T x[8];
      __builtin_memcpy(x, &r, sizeof(x));
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d + e < D) dst[d + e] = x[e];
    }
  } else {
    float x[8], top = 0.f;
    widen(r, x);
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top = fmaxf(top, fabsf(x[e]));
      bad |= (__float_as_uint(x[e]) & 0x7f800000u) == 0x7f800000u;
    }
    top = max16(bad ? INFINITY : top);
    bad = top == INFINITY;
    const float scale = fmaxf(top / 127.f, 1.17549435e-38f);
    const float inv = 1.f / scale, half = 0.5f * scale;
    unsigned q[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // the nearest step by the reciprocal, then by what is left (exact: a step
      // times the scale cancels against x), ties to the even one
      float n = rintf(x[e] * inv);
      const float rest = fmaf(-n, scale, x[e]);
      const bool odd = ((int)n & 1) != 0;
      n += rest > half || (rest == half && odd) ? 1.f : rest < -half || (rest == -half && odd) ? -1.f : 0.f;
      const int c = bad ? 0 : (int)fminf(fmaxf(n, -127.f), 127.f);
      q[e >> 2] |= ((unsigned)c & 255u) << (8 * (e & 3));
    }
    if constexpr (VEC) {
      if (d < D) *reinterpret_cast<uintx2*>(dst + d) = uintx2{q[0], q[1]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d + e < D) dst[d + e] = (int8_t)(q[e >> 2] >> (8 * (e & 3)));
    }
    if (d == 0) *scale_at = bad ? __uint_as_float(0x7fc00000u) : scale;
  }
}
template <class T, class C, bool VEC>
__device__ __forceinline__ void read_row(const C* src, T* dst, const float* scale_at, int D, int d, bool on) {
  float x[8];
  widen(load8<C, VEC>(src, d, D, on), x);
  if constexpr (std::is_same<C, int8_t>::value) {
    const float scale = on ? *scale_at : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= scale;
  }
  store8<T, VEC>(dst, d, D, x);
}

}  // namespace

// 16 lanes to a (row, head), 8 elements a lane; k and v in one pass.
template <class T, class C, bool VEC>
__global__ __launch_bounds__(256) void paged_kv_write_kernel(const T* __restrict__ K, const T* __restrict__ V,
                                                             PagedRows r, PagedCache c) {
  const int64_t item = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 4);
  const int64_t n = item / c.HK;
  const int h = (int)(item - n * c.HK), d = 8 * (threadIdx.x & 15);
  if (n >= r.N) return;
  const int64_t slot = r.slots[n], page = slot >> c.shift;
  if (slot < 0 || page >= c.n_pages) return;
  const int64_t row = ((page * c.HK + h) << c.shift) + (slot & ((1 << c.shift) - 1));
  write_row<T, C, VEC>(K + n * r.k_st + h * r.k_sh, static_cast<C*>(c.k) + row * c.D, c.ks + row, c.D, d);
  write_row<T, C, VEC>(V + n * r.v_st + h * r.v_sh, static_cast<C*>(c.v) + row * c.D, c.vs + row, c.D, d);
}
template <class T, class C, bool VEC>
__global__ __launch_bounds__(256) void paged_kv_read_kernel(T* __restrict__ K, T* __restrict__ V, PagedRows r,
                                                            PagedCache c) {
  const int64_t item = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 4);
  const int64_t n = item / c.HK;
  const int h = (int)(item - n * c.HK), d = 8 * (threadIdx.x & 15);
  if (n >= r.N) return;
  const int64_t slot = r.slots[n], page = slot >> c.shift;
  const bool on = slot >= 0 && page < c.n_pages;
  const int64_t row = on ? ((page * c.HK + h) << c.shift) + (slot & ((1 << c.shift) - 1)) : 0;
  read_row<T, C, VEC>(static_cast<const C*>(c.k) + row * c.D, K + n * r.k_st + h * r.k_sh, c.ks + row, c.D, d, on);
  read_row<T, C, VEC>(static_cast<const C*>(c.v) + row * c.D, V + n * r.v_st + h * r.v_sh, c.vs + row, c.D, d, on);
}

// ---------------------------------------------------------------- decode
namespace {
constexpr int kTile = 32;       // keys a wave takes at a time
constexpr int kWaves = 4;
constexpr int kHeads = 16;      // query heads of a group in one MFMA

// Tiles that one split of `splits` takes of a sequence of n keys.
__device__ __forceinline__ int split_tiles(int n, int splits) {
  const int tiles = (n + kTile - 1) / kTile;
  return ((tiles + splits - 1) / splits + kWaves - 1) / kWaves * kWaves;
}
}  // namespace

// Splits of a sequence: blocks for every CU, of 256 keys or more.  Two to a CU are
// enough for one sequence, whose splits are alike (131072 keys, 8 heads of 128 in bf16:
// 81 us + 6 of the join; four to a CU 82 + 9, eight 84 + 15); sequences of different
// lengths fill the card evenly with four (32 of up to 8192 in 8 bits: 73 us, with two
// 75, with eight 76).
int paged_splits(int64_t n_seq, int n_head, int HK, int64_t capacity) {
  const int64_t blocks = n_seq * HK * ((n_head / HK + kHeads - 1) / kHeads);
  const int64_t want = ((n_seq == 1 ? 512 : 1024) + blocks - 1) / blocks, most = (capacity + 255) / 256;
  const int64_t n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n > 256 ? 256 : n);
}
// Per split and query head: maximum (log2 units), sum, then D outputs.
size_t paged_decode_floats(int64_t n_seq, int n_head, int HK, int D, int64_t capacity) {
  const int n = paged_splits(n_seq, n_head, HK, capacity);
  return n == 1 ? 0 : (size_t)n_seq * n_head * n * (D + 2);
}

// The type that a decode's products are formed in: the element type, but fp16 for
// 8-bit caches of the 16-bit types.  The steps turn into fp16 two at a time (bf16
// has no packed arithmetic), and weights keep 11 bits.
template <class T, class C>
using Product = typename std::conditional<std::is_same<C, int8_t>::value && sizeof(T) == 2, _Float16, T>::type;

// How a tile's rows are reached.  kElements: element by element, any head dim and
// alignment.  kPages: 16-byte loads, the page looked up row by row.  kOnePage: pages
// of at least a tile, which so lies in one, a run of memory: buffer loads whose
// offsets never change and whose descriptor (in scalar registers) ends at the last
// key, so that what lies behind it reads as zeros: 81 us against 98 of kPages for one
// sequence of 131072 keys, 8 heads of 128 in bf16; 73 against 109 for 32 of up to 8192
// in 8 bits.  (8-bit rows: 16 of them to a load, so head dims that are multiples of 16;
// with 8, lines are fetched twice.)
enum Reach { kElements, kPages, kOnePage };

// One block: a split of one sequence's keys for up to 16 query heads of one
// key-value head; its waves take 32-key tiles in turn, each with a softmax of its
// own, joined at the end.  S^T = K Q^T on 16 x 16 results (keys on rows, heads on
// columns), and P^T is the other operand of O^T += V^T P^T as it stands; V goes
// through LDS, which gives it transposed.  A wave loads the next tile's V as soon as
// this one's is in LDS and its K as soon as the scores are formed.
template <class T, class C, int NKS, Reach REACH>
__global__ __launch_bounds__(256, REACH == kOnePage && sizeof(Product<T, C>) == 2 ? 3 : 1) void paged_decode_kernel(const T* __restrict__ Q, T* __restrict__ O,
                                                           float* __restrict__ LSE, float* __restrict__ WS,
                                                           const int* __restrict__ TABLE, PagedDecode a, PagedCache c,
                                                           int splits, float sl2) {
  using X = Product<T, C>;
  constexpr bool VEC = REACH != kElements, Q8 = std::is_same<C, int8_t>::value;
  // fp16 weights of 8-bit values are kept relative to a power of two not below any
  // scale so far, and queries of another type to one not below any of their
  // elements, so that they stay in the range that fp16 holds to full precision
  constexpr bool SCALED_V = Q8 && std::is_same<X, _Float16>::value, SCALED_Q = !std::is_same<T, X>::value;
  constexpr int DP = 32 * NKS, NDT = 2 * NKS;
  // a load takes U elements of a row: UPR to a row, PER to a lane and tile of V
  constexpr int U = REACH == kOnePage && Q8 ? 16 : 8, UPR = DP / U, PER = kTile * UPR / 64;
  constexpr int QUADS = U * (int)sizeof(C) / 16;  // kOnePage: 16-byte loads of a unit
  // lane group g's 8 elements of k-step ks
  auto dim = [&](int ks, int g) { return U == 16 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g; };
  using L = LdsTile<X, DP>;
  constexpr int VB = kTile * L::kRow, JB = kHeads * DP * 4;
  __shared__ __align__(16) char lds[kWaves * (VB > JB ? VB : JB)];
  __shared__ __align__(16) float stat[kWaves][2 * kTile];

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n16 = lane & 15, D = c.D;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.n_head / c.HK, groups = (G + kHeads - 1) / kHeads;
  const int hk = blockIdx.x % c.HK, rest = blockIdx.x / c.HK, split = rest % splits, by = rest / splits;
  const int h0 = hk * G + (by % groups) * kHeads, nh = min(kHeads, G - (by % groups) * kHeads), b = by / groups;
  const int P = 1 << c.shift;
  const int64_t cap = (int64_t)a.max_pages << c.shift;
  const int len0 = a.lens[b], len = (int)min((int64_t)max(len0, 0), cap);
  const int* table = TABLE + (int64_t)b * a.table_stride;
  const int per = split_tiles(len, splits), t_end = min((split + 1) * per, (len + kTile - 1) / kTile);
  if (splits > 1 && split * per >= t_end) return;  // the join knows which splits there are

  const C* Kc = static_cast<const C*>(c.k);
  const C* Vc = static_cast<const C*>(c.v);
  // The table's entry for key k0 + lane % 32 (kOnePage: for the tile, a scalar load),
  // looked at one tile later only (page_of): loads come back in order, and a wait
  // for this one would be a wait for the tile loaded before it.
  auto entry_of = [&](int tile) {
    const int key = min(min(tile, t_end) * kTile + (REACH == kOnePage ? 0 : lane & 31), max(len - 1, 0));
    return len > 0 ? table[key >> c.shift] : 0;
  };
  // its page: -1 past the end, -2 outside the cache
  auto page_of = [&](int tile, int entry) {
    if (tile >= t_end || tile * kTile + (REACH == kOnePage ? 0 : lane & 31) >= len) return -1;
    return entry < 0 || entry >= c.n_pages ? -2 : entry;
  };
  auto row_of = [&](int pg, int key) { return (((int64_t)max(pg, 0) * c.HK + hk) << c.shift) + (key & (P - 1)); };
  typename std::conditional<REACH == kOnePage, uintx4, Raw<C>>::type kr[REACH == kOnePage ? 2 * NKS * 8 / U * QUADS : 2 * NKS],
      vr[REACH == kOnePage ? PER * QUADS : PER];
  float ksc = 0.f, vsc = 0.f;
  int k_off[2], v_off[PER];  // kOnePage: byte offsets in a tile
  if constexpr (REACH == kOnePage) {
#pragma unroll
    for (int x = 0; x < 2; ++x) k_off[x] = ((16 * x + n16) * D + U * g) * (int)sizeof(C);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int r = (u * 64 + lane) / UPR, d = U * (lane % UPR);
      v_off[u] = d < D ? (r * D + d) * (int)sizeof(C) : kPastEnd;
    }
  }
  // keys of the tile, none where there is no page
  auto keys = [&](int tile, int pg) { return pg >= 0 ? (uint32_t)min(kTile, len - tile * kTile) : 0u; };
  auto load_k = [&](int tile, int pg) {
    if constexpr (REACH == kOnePage) {
      const int64_t row = row_of(pg, tile * kTile);
      const uint32_t n = keys(tile, pg);
      const __amdgpu_buffer_rsrc_t r = buffer_rsrc(Kc + row * D, n * (uint32_t)(D * sizeof(C)));
      constexpr int PR = NKS * 8 / U;  // units of a row to a lane, 4 U elements apart
#pragma unroll
      for (int i = 0; i < 2 * PR; ++i)
#pragma unroll
        for (int e = 0; e < QUADS; ++e)
          kr[i * QUADS + e] = buffer_load16(
              r, 4 * U * (i % PR) + U * g < D ? k_off[i / PR] + 4 * U * (i % PR) * (int)sizeof(C) + 16 * e : kPastEnd);
      if constexpr (Q8) ksc = buffer_load_float(buffer_rsrc(c.ks + row, n * 4u), lane * 4, 0);
    } else {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int p = __shfl(pg, 16 * x + n16, 64);
        const C* row = Kc + row_of(p, tile * kTile + 16 * x + n16) * D;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) kr[x * NKS + ks] = load8<C, VEC>(row, dim(ks, g), D, p >= 0);
      }
      if constexpr (Q8) ksc = pg >= 0 ? c.ks[row_of(pg, tile * kTile + (lane & 31))] : 0.f;
    }
  };
  auto load_v = [&](int tile, int pg) {
    if constexpr (REACH == kOnePage) {
      const int64_t row = row_of(pg, tile * kTile);
      const uint32_t n = keys(tile, pg);
      const __amdgpu_buffer_rsrc_t r = buffer_rsrc(Vc + row * D, n * (uint32_t)(D * sizeof(C)));
#pragma unroll
      for (int u = 0; u < PER; ++u)
#pragma unroll
        for (int e = 0; e < QUADS; ++e) vr[u * QUADS + e] = buffer_load16(r, v_off[u] + 16 * e);
      if constexpr (Q8) vsc = buffer_load_float(buffer_rsrc(c.vs + row, n * 4u), lane * 4, 0);
    } else {
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int r = (u * 64 + lane) / UPR, p = __shfl(pg, r, 64);
        vr[u] = load8<C, VEC>(Vc + row_of(p, tile * kTile + r) * D, 8 * (lane % UPR), D, p >= 0);
      }
      if constexpr (Q8) vsc = pg >= 0 ? c.vs[row_of(pg, tile * kTile + (lane & 31))] : 0.f;
    }
  };
  // the i-th 8 elements of a lane's loads
  auto eight = [&](const auto& x, int i) {
    Raw<C> r;
    if constexpr (REACH != kOnePage) {
      r = x[i];
    } else if constexpr (sizeof(C) == 4) {
      r.a = __builtin_bit_cast(floatx4, x[2 * i]);
      r.b = __builtin_bit_cast(floatx4, x[2 * i + 1]);
    } else if constexpr (sizeof(C) == 2) {
      r.a = x[i];
    } else {
      r.a = (i & 1) ? uintx2{x[i / 2][2], x[i / 2][3]} : uintx2{x[i / 2][0], x[i / 2][1]};
    }
    return r;
  };

  int tile = split * per + wave, entry = entry_of(tile + kWaves), pg = page_of(tile, entry_of(tile));
  load_v(tile, pg);
  load_k(tile, pg);

  typename Elem<X>::Frag qf[NKS];
  {
    const T* row = Q + (int64_t)b * a.q_sb + (int64_t)(h0 + min(n16, nh - 1)) * a.q_sh;
    float x[NKS][8], top = 0.f;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const Raw<T> r = load8<T, VEC>(row, dim(ks, g), D, n16 < nh);
      if constexpr (SCALED_Q) {
        widen(r, x[ks]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[ks][e]));
      } else {
        qf[ks] = as_frag<X, T>(r);
      }
    }
    if constexpr (SCALED_Q) {
      top = pair_max32(pair_max16(top));
      const int e = top > 0.f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
      sl2 = __builtin_amdgcn_ldexpf(sl2, e);
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[ks][i] = __builtin_amdgcn_ldexpf(x[ks][i], -e);
        qf[ks] = Elem<X>::pack(x[ks]);
      }
    }
  }

  float m = -INFINITY, l = 0.f, vref = 0.f;
  floatx4 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = floatx4{0.f, 0.f, 0.f, 0.f};
  char* Vt = lds + wave * VB;
  for (; tile < t_end; tile += kWaves) {
    int ln = lane;
    pin(ln);
#pragma unroll
    for (int i = 0; i < PER * U / 8; ++i) {
      const int u = i / (U / 8), half = i % (U / 8);
      L::put(Vt, (u * 64 + ln) / UPR, (ln % UPR) * (U / 8) + half, as_frag<X, C>(eight(vr, i)));
    }
    if constexpr (Q8) {
      float w = vsc;
      if constexpr (SCALED_V) {
        float top = max16(lane < kTile ? vsc : 0.f);
        top = pair_max32(pair_max16(top));
        if (top > vref) {  // wave-uniform
          const float now = __builtin_amdgcn_ldexpf(1.f, __builtin_amdgcn_frexp_expf(top));
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[dt] *= vref / now;
          vref = now;
        }
        w = vref > 0.f ? vsc / vref : vsc;
      }
      if (lane < 32) {
        stat[wave][lane] = ksc;
        stat[wave][32 + lane] = w;
      }
    }
    // pages outside the cache: a score of NaN, which the sequence's outputs become
    const uint64_t out = __builtin_amdgcn_ballot_w64(pg == -2);
    const int k0 = tile * kTile;
    __builtin_amdgcn_wave_barrier();
    pg = page_of(tile + kWaves, entry);
    load_v(tile + kWaves, pg);
    floatx4 s[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      s[x] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) s[x] = Elem<X>::mma16(as_frag<X, C>(eight(kr, x * NKS + ks)), qf[ks], s[x]);
    }
    entry = entry_of(tile + 2 * kWaves);
    load_k(tile + kWaves, pg);
    if constexpr (Q8) {
#pragma unroll
      for (int x = 0; x < 2; ++x) s[x] *= *reinterpret_cast<const floatx4*>(&stat[wave][16 * x + 4 * g]);
    }
    if (k0 + kTile > len) {  // wave-uniform
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[x][i] = k0 + 16 * x + 4 * g + i < len ? s[x][i] : -INFINITY;
    }
    if (out != 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (REACH == kOnePage || ((out >> (16 * x + 4 * g + i)) & 1)) s[x][i] = __uint_as_float(0x7fc00000u);
    }
    float mx = vmax3(vmax3(s[0][0], s[0][1], s[0][2]), s[0][3], s[1][0]);
    mx = vmax3(vmax3(mx, s[1][1], s[1][2]), s[1][3], s[1][3]);
    mx = pair_max32(pair_max16(mx)) * sl2;
    if (__builtin_amdgcn_ballot_w64(mx > m + 8.f) != 0) {  // (as in the packed forward)
      const float mn = vmax2(m, mx);
      float alpha = mn == m ? 1.f : fast_exp2(m - mn);
      pin(alpha);  // (else the products are formed before the branch, every time)
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
    }
    const float sub = m == -INFINITY ? 0.f : m;
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = fast_exp2(fmaf(s[j >> 2][j & 3], sl2, -sub));
      l += p[j];
    }
    if constexpr (Q8) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const floatx4 y = *reinterpret_cast<const floatx4*>(&stat[wave][32 + 16 * x + 4 * g]);
#pragma unroll
        for (int i = 0; i < 4; ++i) p[4 * x + i] *= y[i];
      }
    }
    const typename Elem<X>::Frag pf = Elem<X>::pack(p);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      o[dt] = Elem<X>::mma16(L::cols16(Vt, dt, ln), pf, o[dt]);
      if (dt % 4 == 3) WHA_FENCE();
    }
    __builtin_amdgcn_wave_barrier();
  }
  l = pair_sum32(pair_sum16(l));
  if (len0 > cap) l = __uint_as_float(0x7fc00000u);  // more keys than the table has places

  // the four waves' parts: O[head][d] in LDS, maximum and sum beside it
  __syncthreads();
  float* part = reinterpret_cast<float*>(lds) + wave * kHeads * DP;
  const float mul = SCALED_V ? vref : 1.f;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[n16 * DP + 16 * dt + 4 * g + i] = o[dt][i] * mul;
  if (g == 0) {
    stat[wave][n16] = m;
    stat[wave][16 + n16] = l;
  }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(lds);
  for (int i = tid; i < nh * DP; i += 256) {
    const int n = i / DP, d = i % DP;
    if (d >= D) continue;
    float top = stat[0][n];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = vmax2(top, stat[w][n]);
    const float sub = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float e = fast_exp2(stat[w][n] - sub);
      sum = fmaf(stat[w][16 + n], e, sum);
      x = fmaf(all[(w * kHeads + n) * DP + d], e, x);
    }
    const int64_t row = (int64_t)b * a.n_head + h0 + n;
    if (splits == 1) {
      O[(int64_t)b * a.o_sb + (int64_t)(h0 + n) * a.o_sh + d] = (T)(len > 0 ? x / sum : 0.f);
      if (LSE != nullptr && d == 0) LSE[row] = len > 0 ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
    } else {
      float* dst = WS + (row * splits + split) * (D + 2);
      dst[2 + d] = x;
      if (d == 0) dst[0] = top, dst[1] = sum;
    }
  }
}

// Joins the splits of one (sequence, query head): the statistics by a wave, a
// split a lane; the outputs with kJoin splits in flight.
constexpr int kJoin = 8;
template <class T>
__global__ __launch_bounds__(256) void paged_join_kernel(const float* __restrict__ WS, T* __restrict__ O,
                                                         float* __restrict__ LSE, PagedDecode a, int D, int shift,
                                                         int splits) {
  __shared__ float weight[256], part[2 * 128];
  const int b = blockIdx.x / a.n_head, h = blockIdx.x % a.n_head, tid = threadIdx.x, lane = tid & 63;
  const int len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages << shift);
  const int per = split_tiles(len, splits), n = len > 0 ? ((len + kTile - 1) / kTile + per - 1) / per : 0;
  const float* src = WS + (int64_t)blockIdx.x * splits * (D + 2);
  if (tid < 64) {
    float m[4], l[4], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = lane + 64 * i;
      m[i] = s < n ? src[s * (D + 2)] : -INFINITY;
      l[i] = s < n ? src[s * (D + 2) + 1] : 0.f;
      top = vmax2(top, m[i]);
    }
    top = max16(top);
    top = pair_max32(pair_max16(top));
    const float sub = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = fast_exp2(m[i] - sub);
      sum = fmaf(l[i], m[i], sum);
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) sum += xor_shfl(sum, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) weight[lane + 64 * i] = m[i] / sum;
    if (lane == 0 && LSE != nullptr) LSE[blockIdx.x] = len > 0 ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
  }
  __syncthreads();
  const int d = tid & 127, half = tid >> 7;
  float x = 0.f;
  if (d < D) {
    for (int s = half; s < n; s += 2 * kJoin) {
      float y[kJoin];
#pragma unroll
      for (int i = 0; i < kJoin; ++i) y[i] = s + 2 * i < n ? src[(s + 2 * i) * (D + 2) + 2 + d] : 0.f;
#pragma unroll
      for (int i = 0; i < kJoin; ++i)
        if (s + 2 * i < n) x = fmaf(weight[s + 2 * i], y[i], x);
    }
  }
  part[tid] = x;
  __syncthreads();
  if (half == 0 && d < D)
    O[(int64_t)b * a.o_sb + (int64_t)h * a.o_sh + d] = (T)(len > 0 ? part[d] + part[128 + d] : 0.f);
}

// ---------------------------------------------------------------- launches
namespace {

template <class T, class C, bool VEC>
hipError_t write_t(const void* k, const void* v, const PagedRows& r, const PagedCache& c, hipStream_t stream) {
  TimingScope ts("paged_kv_write", stream);
  hipLaunchKernelGGL((paged_kv_write_kernel<T, C, VEC>),
                     dim3((unsigned)((r.N * c.HK + kRowsPerBlock - 1) / kRowsPerBlock)), dim3(256), 0, stream,
                     static_cast<const T*>(k), static_cast<const T*>(v), r, c);
  return hipGetLastError();
}
template <class T, class C, bool VEC>
hipError_t read_t(void* k, void* v, const PagedRows& r, const PagedCache& c, hipStream_t stream) {
  TimingScope ts("paged_kv_read", stream);
  hipLaunchKernelGGL((paged_kv_read_kernel<T, C, VEC>),
                     dim3((unsigned)((r.N * c.HK + kRowsPerBlock - 1) / kRowsPerBlock)), dim3(256), 0, stream,
                     static_cast<T*>(k), static_cast<T*>(v), r, c);
  return hipGetLastError();
}
template <class T, class C, int NKS, Reach REACH>
hipError_t decode_t(const void* q, void* o, float* lse, float* ws, const PagedDecode& d, const PagedCache& c,
                    float scale, hipStream_t stream) {
  const int splits = paged_splits(d.n_seq, d.n_head, c.HK, (int64_t)d.max_pages << c.shift);
  const int groups = (d.n_head / c.HK + kHeads - 1) / kHeads;
  {
    TimingScope ts("paged_decode", stream);
    hipLaunchKernelGGL((paged_decode_kernel<T, C, NKS, REACH>), dim3((unsigned)d.n_seq * groups * splits * c.HK),
                       dim3(256), 0, stream, static_cast<const T*>(q), static_cast<T*>(o), lse, ws, d.table, d, c, splits,
                       (float)((double)scale * 1.4426950408889634));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || splits == 1) return e;
  }
  TimingScope ts("paged_join", stream);
  hipLaunchKernelGGL((paged_join_kernel<T>), dim3((unsigned)d.n_seq * d.n_head), dim3(256), 0, stream, ws,
                     static_cast<T*>(o), lse, d, c.D, c.shift, splits);
  return hipGetLastError();
}
template <class T, class C>
hipError_t decode_c(const void* q, void* o, float* lse, float* ws, const PagedDecode& d, const PagedCache& c, bool vec,
                    float scale, hipStream_t stream) {
  auto dims = [&](auto reach) {
    constexpr Reach R = decltype(reach)::value;
    return c.D <= 64 ? decode_t<T, C, 2, R>(q, o, lse, ws, d, c, scale, stream)
                     : decode_t<T, C, 4, R>(q, o, lse, ws, d, c, scale, stream);
  };
  if (!vec) return dims(std::integral_constant<Reach, kElements>{});
  return (1 << c.shift) >= kTile && c.D * sizeof(C) % 16 == 0 ? dims(std::integral_constant<Reach, kOnePage>{})
                                 : dims(std::integral_constant<Reach, kPages>{});
}

}  // namespace

// F<element type, cache type, VEC>(args)
#define WHA_BY_TYPES(F, ...)                                                                                    \
  const bool q8 = cache_dtype == kI8;                                                                           \
  if (dtype == kF32)                                                                                            \
    return q8 ? (vec ? F<float, int8_t, true>(__VA_ARGS__) : F<float, int8_t, false>(__VA_ARGS__))              \
              : (vec ? F<float, float, true>(__VA_ARGS__) : F<float, float, false>(__VA_ARGS__));               \
  if (dtype == kBf16)                                                                                           \
    return q8 ? (vec ? F<__bf16, int8_t, true>(__VA_ARGS__) : F<__bf16, int8_t, false>(__VA_ARGS__))            \
              : (vec ? F<__bf16, __bf16, true>(__VA_ARGS__) : F<__bf16, __bf16, false>(__VA_ARGS__));           \
  return q8 ? (vec ? F<_Float16, int8_t, true>(__VA_ARGS__) : F<_Float16, int8_t, false>(__VA_ARGS__))          \
            : (vec ? F<_Float16, _Float16, true>(__VA_ARGS__) : F<_Float16, _Float16, false>(__VA_ARGS__))

hipError_t launch_paged_kv_write(int dtype, int cache_dtype, const void* k, const void* v, const PagedRows& r,
                                 const PagedCache& c, bool vec, hipStream_t stream) {
  WHA_BY_TYPES(write_t, k, v, r, c, stream);
}
hipError_t launch_paged_kv_read(int dtype, int cache_dtype, void* k, void* v, const PagedRows& r, const PagedCache& c,
                                bool vec, hipStream_t stream) {
  WHA_BY_TYPES(read_t, k, v, r, c, stream);
}
hipError_t launch_paged_decode(int dtype, int cache_dtype, const void* q, void* o, float* lse, float* ws,
                               const PagedDecode& d, const PagedCache& c, bool vec, float scale, hipStream_t stream) {
  const bool q8 = cache_dtype == kI8;
  if (dtype == kF32)
    return q8 ? decode_c<float, int8_t>(q, o, lse, ws, d, c, vec, scale, stream)
              : decode_c<float, float>(q, o, lse, ws, d, c, vec, scale, stream);
  if (dtype == kBf16)
    return q8 ? decode_c<__bf16, int8_t>(q, o, lse, ws, d, c, vec, scale, stream)
              : decode_c<__bf16, __bf16>(q, o, lse, ws, d, c, vec, scale, stream);
  return q8 ? decode_c<_Float16, int8_t>(q, o, lse, ws, d, c, vec, scale, stream)
            : decode_c<_Float16, _Float16>(q, o, lse, ws, d, c, vec, scale, stream);
}

}  // namespace wha
