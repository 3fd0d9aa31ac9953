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
    for (int e = 0; e < 8; ++e) x[e] = (float)((int)(r.a[e >> 2] << (24 - 8 * (e & 3))) >> 24);
  }
}
// As a fragment of the type that the products are formed in (8-bit steps are
// exact in all of them).
template <class T, class C>
__device__ __forceinline__ typename Elem<T>::Frag as_frag(const Raw<C>& r) {
  if constexpr (std::is_same<T, C>::value && sizeof(T) == 2) {
    return __builtin_bit_cast(typename Elem<T>::Frag, r.a);
  } else {
    float x[8];
    widen(r, x);
    return Elem<T>::pack(x);
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

int paged_splits(int64_t n_seq, int n_head, int HK, int64_t capacity) {
  const int64_t blocks = n_seq * HK * ((n_head / HK + kHeads - 1) / kHeads);
  const int64_t want = (1024 + blocks - 1) / blocks, most = (capacity + 255) / 256;
  const int64_t n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n > 256 ? 256 : n);
}
// Per split and query head: maximum (log2 units), sum, then D outputs.
size_t paged_decode_floats(int64_t n_seq, int n_head, int HK, int D, int64_t capacity) {
  const int n = paged_splits(n_seq, n_head, HK, capacity);
  return n == 1 ? 0 : (size_t)n_seq * n_head * n * (D + 2);
}

// One block: a split of one sequence's keys for up to 16 query heads of one
// key-value head; its waves take 32-key tiles in turn, each with a softmax of its
// own, joined at the end.  S^T = K Q^T on 16 x 16 results (keys on rows, heads on
// columns), and P^T is the other operand of O^T += V^T P^T as it stands; V goes
// through LDS, which gives it transposed.  A wave loads the next tile's rows into
// registers before it works on the present one.
template <class T, class C, int NKS, bool VEC>
__global__ __launch_bounds__(256) void paged_decode_kernel(const T* __restrict__ Q, T* __restrict__ O,
                                                           float* __restrict__ LSE, float* __restrict__ WS,
                                                           PagedDecode a, PagedCache c, int splits, float sl2) {
  constexpr int DP = 32 * NKS, NDT = 2 * NKS, UPR = DP / 8, PER = kTile * UPR / 64;  // units of 8 elements
  constexpr bool Q8 = std::is_same<C, int8_t>::value, SCALED_V = Q8 && std::is_same<T, _Float16>::value;
  using L = LdsTile<T, DP>;
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
  const int* table = a.table + (int64_t)b * a.table_stride;
  const int per = split_tiles(len, splits), t_end = min((split + 1) * per, (len + kTile - 1) / kTile);
  if (splits > 1 && split * per >= t_end) return;  // the join knows which splits there are

  const C* Kc = static_cast<const C*>(c.k);
  const C* Vc = static_cast<const C*>(c.v);
  typename Elem<T>::Frag qf[NKS];
  {
    const T* row = Q + (int64_t)b * a.q_sb + (int64_t)(h0 + min(n16, nh - 1)) * a.q_sh;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qf[ks] = as_frag<T, T>(load8<T, VEC>(row, 32 * ks + 8 * g, D, n16 < nh));
  }
  // the page of key k0 + lane % 32 of a tile: -1 past the end, -2 outside the cache
  auto page_of = [&](int tile) {
    const int key = tile * kTile + (lane & 31);
    if (tile >= t_end || key >= len) return -1;
    const int pg = table[key >> c.shift];
    return pg < 0 || pg >= c.n_pages ? -2 : pg;
  };
  auto row_of = [&](int pg, int key) { return (((int64_t)pg * c.HK + hk) << c.shift) + (key & (P - 1)); };
  Raw<C> kr[2 * NKS], vr[PER];
  float ksc = 0.f, vsc = 0.f;
  auto load = [&](int tile, int pg) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int p = __shfl(pg, 16 * x + n16, 64);
      const C* row = Kc + row_of(max(p, 0), tile * kTile + 16 * x + n16) * D;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) kr[x * NKS + ks] = load8<C, VEC>(row, 32 * ks + 8 * g, D, p >= 0);
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int r = (u * 64 + lane) / UPR, p = __shfl(pg, r, 64);
      vr[u] = load8<C, VEC>(Vc + row_of(max(p, 0), tile * kTile + r) * D, 8 * (lane % UPR), D, p >= 0);
    }
    if constexpr (Q8) {
      const int64_t row = row_of(max(pg, 0), tile * kTile + (lane & 31));
      ksc = pg >= 0 ? c.ks[row] : 0.f;
      vsc = pg >= 0 ? c.vs[row] : 0.f;
    }
  };

  float m = -INFINITY, l = 0.f, vref = 0.f;
  floatx4 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = floatx4{0.f, 0.f, 0.f, 0.f};
  char* Vt = lds + wave * VB;
  int tile = split * per + wave, pg = page_of(tile), pg_next = page_of(tile + kWaves);
  load(tile, pg);
  for (; tile < t_end; tile += kWaves) {
    typename Elem<T>::Frag kf[2 * NKS];
#pragma unroll
    for (int i = 0; i < 2 * NKS; ++i) kf[i] = as_frag<T, C>(kr[i]);
#pragma unroll
    for (int u = 0; u < PER; ++u) L::put(Vt, (u * 64 + lane) / UPR, lane % UPR, as_frag<T, C>(vr[u]));
    float w = 1.f;
    if constexpr (Q8) {
      // fp16 weights: relative to a power of two not below any scale so far, so that
      // they stay in the range that fp16 holds to full precision
      w = vsc;
      if constexpr (SCALED_V) {
        float top = max16(vsc);
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
    load(tile + kWaves, pg_next);
    pg = pg_next;
    pg_next = page_of(tile + 2 * kWaves);
    floatx4 s[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      s[x] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) s[x] = Elem<T>::mma16(kf[x * NKS + ks], qf[ks], s[x]);
      if constexpr (Q8) s[x] *= *reinterpret_cast<const floatx4*>(&stat[wave][16 * x + 4 * g]);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][i] = k0 + 16 * x + 4 * g + i < len ? s[x][i] : -INFINITY;
    }
    if (out != 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((out >> (16 * x + 4 * g + i)) & 1) s[x][i] = __uint_as_float(0x7fc00000u);
    }
    float mx = vmax3(vmax3(s[0][0], s[0][1], s[0][2]), s[0][3], s[1][0]);
    mx = vmax3(vmax3(mx, s[1][1], s[1][2]), s[1][3], s[1][3]);
    mx = vmax2(m, pair_max32(pair_max16(mx)) * sl2);
    const float sub = mx == -INFINITY ? 0.f : mx, alpha = fast_exp2(m - sub);
    m = mx;
    l *= alpha;
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
    const typename Elem<T>::Frag pf = Elem<T>::pack(p);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      o[dt] *= alpha;
      o[dt] = Elem<T>::mma16(L::cols16(Vt, dt, lane), pf, o[dt]);
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
template <class T, class C, int NKS, bool VEC>
hipError_t decode_t(const void* q, void* o, float* lse, float* ws, const PagedDecode& d, const PagedCache& c,
                    float scale, hipStream_t stream) {
  const int splits = paged_splits(d.n_seq, d.n_head, c.HK, (int64_t)d.max_pages << c.shift);
  const int groups = (d.n_head / c.HK + kHeads - 1) / kHeads;
  {
    TimingScope ts("paged_decode", stream);
    hipLaunchKernelGGL((paged_decode_kernel<T, C, NKS, VEC>), dim3((unsigned)d.n_seq * groups * splits * c.HK),
                       dim3(256), 0, stream, static_cast<const T*>(q), static_cast<T*>(o), lse, ws, d, c, splits,
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
  if (c.D <= 64)
    return vec ? decode_t<T, C, 2, true>(q, o, lse, ws, d, c, scale, stream)
               : decode_t<T, C, 2, false>(q, o, lse, ws, d, c, scale, stream);
  return vec ? decode_t<T, C, 4, true>(q, o, lse, ws, d, c, scale, stream)
             : decode_t<T, C, 4, false>(q, o, lse, ws, d, c, scale, stream);
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
