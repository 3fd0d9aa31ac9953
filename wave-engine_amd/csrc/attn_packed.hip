// Causal attention of packed sequences with grouped heads, forward and backward
// (gfx950): sequences of any lengths one after the other in [total][heads][D]
// rows, cu[i] .. cu[i + 1] - 1 the rows of sequence i (on the device), G query
// heads to a key-value head.
//
//   s_ij = scale q_i . k_j (j <= i, same sequence), lse_i = log sum_j exp s_ij,
//   o_i = sum_j exp(s_ij - lse_i) v_j
//   Delta_i = do_i . o_i, p = exp(s - lse), dp_ij = do_i . v_j, ds = p (dp - Delta)
//   dq_i = scale sum_j ds_ij k_j, dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij do_i
//   (i over the rows of all G heads of the group)
//
// The G query heads of a group are rows of one matrix: row r = t G + g is
// position t of head g, key j is before it iff j G <= r.  A block then holds
// 128 / G positions of all of them, so its tiles past the diagonal are few also
// for short sequences, and the key-stationary kernel sums the group as it goes.
//
// Scores are formed transposed where queries are kept (S^T = K Q^T: keys on MFMA
// rows, a wave's 32 queries on columns), so that P^T is the other operand of O^T
// += V^T P^T as it stands; with keys kept (dK, dV) as S = Q K^T, for the same
// reason.
#include <hip/hip_runtime.h>
#include <utility>

#include "wha_elem.hpp"
#include "wha_packed.hpp"

namespace wha {

namespace {

// Which tile of which sequence block number `order` takes (of one key-value head's).
// A tile's level is the number of tiles that it sweeps less one: those before it in
// its sequence, or with KEYS (tiles of keys, swept by the rows after them) those
// after it.  Up to 64 sequences: the highest level first, whatever the sequence, so
// that the longest sweeps start first and the short ones fill in behind them (16
// ragged sequences of up to 1024, 12 heads of 64 in 4 groups: 28 us, one sequence
// after the other 35; dQ of 12 of them 33 and 41).  More
// sequences: sequence i has the slots from floor(rows before it / BM) + i on, which
// is at least as many as it has tiles; that needs no sum over the sequences, and so
// many balance by themselves.  Either way the grid needs only the total.
struct Place {
  int tile, start, len;  // tile < 0: none left
};
__device__ __forceinline__ int seq_start(const int* cu, int i, int total) { return min(max(cu[i], 0), total); }
template <bool KEYS>
__device__ __forceinline__ Place find_place(const int* cu, int n_seq, int total, int G, int BM, int slots, int order,
                                            int lane) {
  Place p;
  if (n_seq <= 64) {
    int start = 0, len = 0;
    if (lane < n_seq) {
      start = seq_start(cu, lane, total);
      len = max(0, seq_start(cu, lane + 1, total) - start);
    }
    const int n = (int)(((int64_t)len * G + BM - 1) / BM);
    int most = 0, step = 1;
    for (int i = 0; i < n_seq; ++i) most = max(most, __builtin_amdgcn_readlane(n, i));
    while (step * 63 < most) step *= 64;
    // the level that `order` falls into: 64 levels at a time, narrowing down
    int level = 0, above = 0;  // above: tiles of higher levels than it
    for (; step > 0; step >>= 6) {
      const int x = level + lane * step;
      int count = 0;  // tiles of level x and higher
      for (int i = 0; i < n_seq; ++i) count += max(0, __builtin_amdgcn_readlane(n, i) - x);
      const int c = (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(count > order)) - 1;
      if (c < 0) return Place{-1, 0, 0};  // fewer tiles than this in all
      level += c * step;
      if (c < 63) above = __builtin_amdgcn_readlane(count, c + 1);
    }
    uint64_t has = __builtin_amdgcn_ballot_w64(n > level);
    for (int i = above; i < order; ++i) has &= has - 1;
    const int seq = has != 0 ? __builtin_ctzll(has) : 0;
    p.start = __builtin_amdgcn_readlane(start, seq);
    p.len = __builtin_amdgcn_readlane(len, seq);
    p.tile = KEYS ? __builtin_amdgcn_readlane(n, seq) - 1 - level : level;
    return p;
  }
  const int slot = KEYS ? order : slots - 1 - order;
  int lo = 0, n = n_seq;
  while (n > 1) {  // at most 6 rounds: n shrinks 64-fold
    const int step = (n + 63) / 64, i = lo + lane * step;
    bool before = false;
    if (lane * step < n) before = (int)((int64_t)seq_start(cu, i, total) * G / BM) + i <= slot;
    const int c = max(1, (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(before))) - 1;
    lo += c * step;
    n = min(step, n - c * step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  p.start = __builtin_amdgcn_readfirstlane(seq_start(cu, lo, total));
  p.len = __builtin_amdgcn_readfirstlane(max(0, seq_start(cu, lo + 1, total) - p.start));
  p.tile = slot - (int)((int64_t)p.start * G / BM) - lo;
  if ((int64_t)p.tile * BM >= (int64_t)p.len * G) p.tile = -1;
  return p;
}

// Kernels whose registers are full: addresses are formed again for every tile.
template <class T, int DP>
constexpr bool kTight = DP > 64 || sizeof(T) == 4;
// The LDS tiles that the products read.
template <class T, int DP, int ROWS>
using Tile = typename std::conditional<sizeof(T) == 4, SplitTile<DP, ROWS>, LdsTile<T, DP>>::type;

// A tile of rows from memory into LDS, ROWS x DP by NT threads, in two halves: begin
// (the loads) and end (what is left to do when they are there).  off(rr): byte
// offset of tile row rr in the range of the descriptor, past which is zero: rows
// behind the last one, and what lies past the head dim.  What moves from tile to
// tile is the descriptor, in scalar registers.
// A: alignment of rows in bytes.  16-bit types: 16 or 4 bytes at a time straight to
// LDS (complete after wait_vmem), or one element at a time (2).  float: 16 or 4
// bytes at a time to registers, split on the way to LDS.
constexpr int kPast = (int)0x80000000;
template <class T, int DP, int ROWS, int NT, int A>
struct Stage {
  using L = Tile<T, DP, ROWS>;
  static constexpr bool PIN = kTight<T, DP>;
  static constexpr int kRow = DP * (int)sizeof(T);  // bytes of a row in memory, padded
  static constexpr int UNIT = sizeof(T) == 2 && A == 4 ? 4 : 16, UPR = kRow / UNIT, PER = ROWS * UPR / NT;
  static_assert(ROWS * UPR % NT == 0, "whole rounds");
  floatx4 x[sizeof(T) == 4 ? PER : 1];

  template <class Off>
  __device__ __forceinline__ void begin(__amdgpu_buffer_rsrc_t r, char* lds, int D, int tid, Off&& off) {
    if constexpr (PIN) pin(tid);
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int i = p * NT + tid, rr = i / UPR, u = i % UPR;
      if constexpr (sizeof(T) == 4) {
        const int o = off(rr) + 16 * u;
        if constexpr (A == 16) {
          x[p] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(r, 4 * u < D ? o : kPast, 0, 0));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[p][e] = buffer_load_float(r, 4 * u + e < D ? o + 4 * e : kPast, 0);
        }
      } else {
        // unit u of the row in LDS holds elements d .. of the row in memory
        const int d = UNIT == 16 ? 8 * (u ^ L::swz(rr)) : 8 * ((u >> 2) ^ L::swz(rr)) + 2 * (u & 3);
        const int o = off(rr) + 2 * d;
        if constexpr (A == 2) {
          unsigned short y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_raw_buffer_load_b16(r, d + e < D ? o + 2 * e : kPast, 0, 0);
          uintx4 q;
          __builtin_memcpy(&q, y, 16);
          *reinterpret_cast<uintx4*>(lds + i * 16) = q;
        } else {
          auto* to = (void __attribute__((address_space(3)))*)(lds + (p * NT + (tid & ~63)) * UNIT);
          if constexpr (UNIT == 16)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to, 16, d < D ? o : kPast, 0, 0, 0);
          else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to, 4, d < D ? o : kPast, 0, 0, 0);
        }
      }
    }
  }
  __device__ __forceinline__ void end(char* lds, int tid) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const int i = p * NT + tid;
        L::put4(lds, i / UPR, i % UPR, x[p]);
      }
    }
  }
  // Rows row0 .. of one head, st elements apart, n of them in all.  Where the rounds of
  // the block's threads lie whole groups of 16 rows apart a lane has one offset, the
  // same in every round and tile, and each round a descriptor of its own.
  static constexpr int ROUND = NT / UPR;  // rows of a round
  __device__ __forceinline__ void begin_head(const T* base, int row0, int n, int64_t st, char* lds, int D, int tid) {
    if constexpr (UNIT == 16 && A == 16 && (sizeof(T) == 4 || ROUND % 16 == 0)) {
      const int rr = tid / UPR, u = tid % UPR;
      int d = 4 * u;
      if constexpr (sizeof(T) == 2) d = 8 * (u ^ L::swz(rr));
      const int off = d < D ? (rr * (int)st + d) * (int)sizeof(T) : kPast;
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const int first = row0 + p * ROUND, rows = min(n - first, ROUND);
        const uint32_t left = rows > 0 ? (uint32_t)(((int64_t)(rows - 1) * st + D) * (int64_t)sizeof(T)) : 0u;
        const __amdgpu_buffer_rsrc_t r = buffer_rsrc(base + (int64_t)first * st, left);
        if constexpr (sizeof(T) == 4)
          x[p] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
        else
          __builtin_amdgcn_raw_ptr_buffer_load_lds(
              r, (void __attribute__((address_space(3)))*)(lds + (p * NT + (tid & ~63)) * 16), 16, off, 0, 0, 0);
      }
    } else {
      const int64_t left = ((int64_t)(min(n - row0, ROWS) - 1) * st + D) * (int64_t)sizeof(T);
      begin(buffer_rsrc(base + (int64_t)row0 * st, (uint32_t)left), lds, D, tid,
            [&](int rr) { return rr * (int)st * (int)sizeof(T); });
    }
  }
};

// Elements c .. c + 7 of one row (zero past the head dim).
template <class T, int A>
__device__ __forceinline__ typename Elem<T>::Frag row8(const T* row, int c, int D) {
  if constexpr (A == 16 && sizeof(T) == 2) {
    uintx4 q = {0u, 0u, 0u, 0u};
    if (c < D) q = *reinterpret_cast<const uintx4*>(row + c);
    return __builtin_bit_cast(typename Elem<T>::Frag, q);
  } else if constexpr (A == 4 && sizeof(T) == 2) {
    uintx4 q = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + 2 * i < D) q[i] = *reinterpret_cast<const unsigned*>(row + c + 2 * i);
    return __builtin_bit_cast(typename Elem<T>::Frag, q);
  } else {
    float x[8];
    if constexpr (A == 16) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        floatx4 q = {0.f, 0.f, 0.f, 0.f};
        if (c + 4 * h < D) q = *reinterpret_cast<const floatx4*>(row + c + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * h + e] = q[e];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = c + j < D ? (float)row[c + j] : 0.f;
    }
    return Elem<T>::pack(x);
  }
}
template <class T>
__device__ __forceinline__ typename Fast<T>::Frag fast_of(const typename Elem<T>::Frag& f) {
  if constexpr (sizeof(T) == 4) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = f[j];
    return Fast<T>::pack(x);
  } else {
    return f;
  }
}

// Writes a lane's part of X^T[d][row] (d = 32 dt + row32(i, g)) to its row.
template <class T, int NDT, int A>
__device__ __forceinline__ void store_row(T* dst, int D, int g, const floatx16 (&x)[NDT], float mul) {
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = 32 * dt + 8 * u + 4 * g;
      if constexpr (A == 16) {
        if (c < D)
          Elem<T>::store4(dst + c, x[dt][4 * u] * mul, x[dt][4 * u + 1] * mul, x[dt][4 * u + 2] * mul,
                          x[dt][4 * u + 3] * mul);
      } else if constexpr (A == 4 && sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < 4; e += 2)
          if (c + e < D)
            *reinterpret_cast<unsigned*>(dst + c + e) = Elem<T>::pair(x[dt][4 * u + e] * mul, x[dt][4 * u + e + 1] * mul);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < D) dst[c + e] = (T)(x[dt][4 * u + e] * mul);
      }
    }
}

// N steps whose operands come from LDS: the reads of step i + AHEAD go out before
// the MFMAs of step i, no more of them, so that they cost few registers.  Two steps
// where the MFMAs of one take less than an LDS read (a fence behind the reads, or the
// scheduler puts them after the MFMAs and the next ones wait out their latency:
// forward of 64 x 4096 x 128 423 us without, 374 with), one for the six products of
// fp32 (no fence: 48 us against 58 with, for want of registers).
template <class T>
inline constexpr int kAhead = sizeof(T) == 4 ? 1 : 2;
template <class F, int... I>
__device__ __forceinline__ void each(std::integer_sequence<int, I...>, F&& f) {
  (f(std::integral_constant<int, I>()), ...);
}
template <class T, int FROM, int TO, int AHEAD = kAhead<T>, class Load, class Use>
__device__ __forceinline__ void ahead(Load&& load, Use&& use) {
  constexpr int N = TO - FROM;
  decltype(load(std::integral_constant<int, FROM>())) f[AHEAD + 1];
  each(std::make_integer_sequence<int, AHEAD>(), [&](auto i) { f[i] = load(std::integral_constant<int, FROM + i>()); });
  each(std::make_integer_sequence<int, N>(), [&](auto i) {
    if constexpr (i + AHEAD < N)
      f[(i + AHEAD) % (AHEAD + 1)] = load(std::integral_constant<int, FROM + i + AHEAD>());
    if constexpr (sizeof(T) == 2) WHA_FENCE();
    use(std::integral_constant<int, FROM + i>(), f[i % (AHEAD + 1)]);
    WHA_FENCE();
  });
}

// What a step reads: one or two fragments and its elements' statistics.
template <class F, int E>
struct Step {
  F a, b;
  float stat[E];
};

// p's two fragments of 16 rows, the weights of an MFMA with the tile's columns
template <class T>
__device__ __forceinline__ void pack_rows(const floatx16& p, typename Fast<T>::Frag (&f)[2]) {
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = p[8 * b + j];
    f[b] = Fast<T>::pack(y);
  }
}
// Step j of acc[d][column] += sum over 16 N rows of p[row][column] x[row][d]: N steps
// to each 32 columns of x, x the rows 16 (j % N) .. of them, f their p.
template <class T, int N = 2, int NDT>
__device__ __forceinline__ void add_cols(int j, const typename Fast<T>::Frag& x, const typename Fast<T>::Frag (&f)[2],
                                         floatx16 (&acc)[NDT], typename Fast<T>::Sum& sum) {
  if constexpr (sizeof(T) == 4) {
    if (j % N == 0) sum = typename Fast<T>::Sum();
    sum.add(x, f[j % 2]);
    if (j % N == N - 1) {
      const floatx16 y = sum.value();
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j / N][e] += y[e];
    }
  } else {
    acc[j / N] = Elem<T>::mma32(x, f[j % 2], acc[j / N]);
  }
}

// Results that are not finite are formed once more, from memory, by the wave alone:
// a weight of zero does not undo an infinity or NaN in the tiles that the mask cuts
// through (0 x inf), and the split of fp32 knows no infinity.  Here scores and
// products are Elem's, and the rows of a cut tile are added one by one, those only
// that the mask leaves.  32 rows at a time, x y^T by lane % 32:
template <class T, int NKS, int A>
__device__ __forceinline__ floatx16 scores_of(const T* x, const T* y, int g, int D) {
  floatx16 s = zeros16();
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    s = Elem<T>::mma32(row8<T, A>(x, 16 * ks + 8 * g, D), row8<T, A>(y, 16 * ks + 8 * g, D), s);
    WHA_FENCE();
  }
  return s;
}
// acc[d][column] += p[row][column] row(x)[d] over 32 rows.
template <class T, int NDT, class Row>
__device__ __forceinline__ void add_all(const floatx16& p, floatx16 (&acc)[NDT], int lane, int D, Row&& row) {
  const int g = lane >> 5, c = lane & 31;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = p[8 * s + j];
    const typename Elem<T>::Frag f = Elem<T>::pack(y);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 32 * dt + c < D ? (float)row(16 * s + row32(j, g))[32 * dt + c] : 0.f;
      acc[dt] = Elem<T>::mma32(Elem<T>::pack(x), f, acc[dt]);
      WHA_FENCE();
    }
  }
}
// The same over the rows with mine(x) only, the weights by way of `w` (32 x 32 of the
// wave's own LDS).
template <class T, int NDT, class Row, class Mine>
__device__ __forceinline__ void add_mine(const floatx16& p, floatx16 (&acc)[NDT], T* w, int lane, int D, Row&& row,
                                         Mine&& mine) {
  const int g = lane >> 5, c = lane & 31;
#pragma unroll
  for (int i = 0; i < 16; ++i) w[row32(i, g) * 32 + c] = (T)p[i];
  __builtin_amdgcn_wave_barrier();
#pragma unroll 1
  for (int x = 0; x < 32; ++x) {
    if (!mine(x)) continue;
    const float px = (float)w[x * 32 + c];
    const T* src = row(x);
    int dim = D;
    pin(dim);  // or 64 lane masks are held in registers
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int y = 0; y < 16; ++y) {
        const int d = 32 * dt + row32(y, g);
        if (d < dim) acc[dt][y] = fmaf(px, (float)src[d], acc[dt][y]);
      }
  }
  __builtin_amdgcn_wave_barrier();
}
// Whether any lane's `on` results are not all finite.
template <int NDT>
__device__ __forceinline__ bool any_not_finite(const floatx16 (&x)[NDT], bool on) {
  float chk = 0.f;  // NaN if any is not finite
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) chk = fmaf(x[dt][i], 0.f, chk);
  return __builtin_amdgcn_ballot_w64(on && chk != 0.f) != 0;
}

// The tiles that the mask leaves whole first, then the cut ones, in loops of their own:
// both forms of the sums in one loop would hold them twice.
//
// 32 rows of the forward: the maximum of each first (a running one would meet -inf -
// -inf), then weights and O.
template <class T, int NKS, int NDT, int A>
__device__ __forceinline__ void fwd_again(const T* Qr, const T* Kb, const T* Vb, T* Or, float* lse_at, T* w,
                                                    int64_t k_st, int64_t v_st, int len, int D, bool on, int t,
                                                    int t_first, int t_last, float sl2, int lane) {
  const int g = lane >> 5;
  auto scores = [&](int k0) {
    floatx16 s = scores_of<T, NKS, A>(Kb + (int64_t)min(k0 + (lane & 31), len - 1) * k_st, Qr, g, D);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = k0 + row32(i, g) > t ? -INFINITY : s[i];
    return s;
  };
  float m = -INFINITY, l = 0.f;
  floatx16 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = zeros16();
#pragma unroll 1
  for (int k0 = 0; k0 <= t_last; k0 += 32) {
    const floatx16 s = scores(k0);
#pragma unroll
    for (int i = 0; i < 16; ++i) m = vmax2(m, s[i]);
  }
  m = pair_max32(m) * sl2;
  const float sub = m == -INFINITY ? 0.f : m;
  auto weights = [&](int k0) {
    floatx16 s = scores(k0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = fast_exp2(fmaf(s[i], sl2, -sub));
      l += s[i];
    }
    return s;
  };
  int k0 = 0;
  auto row = [&](int x) { return Vb + (int64_t)min(k0 + x, len - 1) * v_st; };
#pragma unroll 1
  for (; k0 + 31 <= t_first; k0 += 32) add_all<T>(weights(k0), o, lane, D, row);
#pragma unroll 1
  for (; k0 <= t_last; k0 += 32) add_mine<T>(weights(k0), o, w, lane, D, row, [&](int x) { return k0 + x <= t; });
  l = pair_sum32(l);
  if (on) {
    store_row<T, NDT, A>(Or, D, g, o, 1.f / l);
    if (lse_at != nullptr && g == 0) *lse_at = fmaf(m, kLn2, logf(l));
  }
}
template <class T, int NKS, int NDT, int A>
__device__ __forceinline__ void dq_again(const T* Qr, const T* Kb, const T* Vb, const T* DOr, T* dq_at, T* w,
                                                   int64_t k_st, int64_t v_st, int len, int D, bool on, int t,
                                                   int t_first, int t_last, float sl2, float lse2, float delta,
                                                   float scale, int lane) {
  const int g = lane >> 5;
  floatx16 dq[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) dq[dt] = zeros16();
  int k0 = 0;
  auto row = [&](int x) { return Kb + (int64_t)min(k0 + x, len - 1) * k_st; };
  auto weights = [&]() {
    floatx16 s = scores_of<T, NKS, A>(row(lane & 31), Qr, g, D);
    const floatx16 dp = scores_of<T, NKS, A>(Vb + (int64_t)min(k0 + (lane & 31), len - 1) * v_st, DOr, g, D);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = fast_exp2(fmaf(s[i], sl2, -lse2)) * (dp[i] - delta);
    return s;
  };
#pragma unroll 1
  for (; k0 + 31 <= t_first; k0 += 32) add_all<T>(weights(), dq, lane, D, row);
#pragma unroll 1
  for (; k0 <= t_last; k0 += 32) add_mine<T>(weights(), dq, w, lane, D, row, [&](int x) { return k0 + x <= t; });
  if (on) store_row<T, NDT, A>(dq_at, D, g, dq, scale);
}
// dK (KEYS) or dV of 32 keys; lse2, delta: the statistics of the group's rows.
template <class T, int NKS, int NDT, int A, bool KEYS>
__device__ __forceinline__ void dkv_again(const T* Qb, const T* Kr, const T* Vr, const T* Db, const float* lse2,
                                          const float* delta, T* to, T* w, int64_t q_st, int64_t q_sh, int64_t o_st,
                                          int64_t o_sh, int total, int G, int D, int rows, int key0, bool on,
                                          float sl2, float scale, int lane) {
  const int g = lane >> 5, first = (key0 + (lane & 31)) * G;
  floatx16 acc[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) acc[dt] = zeros16();
  int r0 = 0;
  auto q_row = [&](int y) {
    const int r = min(r0 + y, rows - 1);
    return Qb + (int64_t)(r / G) * q_st + (int64_t)(r % G) * q_sh;
  };
  auto do_row = [&](int y) {
    const int r = min(r0 + y, rows - 1);
    return Db + (int64_t)(r / G) * o_st + (int64_t)(r % G) * o_sh;
  };
  auto row = [&](int y) { return KEYS ? q_row(y) : do_row(y); };
  auto mine = [&](int y) { return r0 + y >= first && r0 + y < rows; };
  auto weights = [&]() {
    floatx16 p = scores_of<T, NKS, A>(q_row(lane & 31), Kr, g, D), dp = zeros16();
    if constexpr (KEYS) dp = scores_of<T, NKS, A>(do_row(lane & 31), Vr, g, D);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = min(r0 + row32(i, g), rows - 1);
      const int64_t at = (int64_t)(r % G) * total + r / G;
      p[i] = fast_exp2(fmaf(p[i], sl2, -lse2[at]));
      if constexpr (KEYS) p[i] *= dp[i] - delta[at];
      if (i % 4 == 3) WHA_FENCE();
    }
    return p;
  };
  const int begin = key0 * G & ~31, whole = ((key0 + 31) * G + 31) & ~31;  // sub-tiles from `whole` on are not cut
#pragma unroll 1
  for (r0 = whole; r0 + 32 <= rows; r0 += 32) add_all<T>(weights(), acc, lane, D, row);
  const int last = max(r0, whole);  // the one that the sequence's end cuts
#pragma unroll 1
  for (r0 = begin; r0 < rows; r0 = r0 + 32 < whole ? r0 + 32 : r0 < whole ? last : rows)
    add_mine<T>(weights(), acc, w, lane, D, row, mine);
  if (on) store_row<T, NDT, A>(to, D, g, acc, scale);
}

}  // namespace

// ---------------------------------------------------------------- forward
// A tile of K and one of V at a time, two of each in LDS; a wave keeps 32 queries' Q,
// maximum, sum and O^T in registers.  16 bits, 32 query heads of 128 in 8 groups, 4
// sequences of 4096: 373 us, 0.86 PFLOP/s of the products that the mask leaves; the
// matrix cores are busy 45% of it, the VALU (exponentials, maxima) as long, and the
// two overlap only where a wave's own instructions alternate.  Waves to a SIMD: as
// many as the loop's registers leave room for.
template <class T, int NKS, int NDT, int A>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? (NDT <= 2 ? 3 : 2) : (NDT <= 2 ? 2 : 1)) void packed_fwd_kernel(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, T* __restrict__ O,
    float* __restrict__ LSE, PackedArgs a, float sl2) {
  constexpr int DP = 32 * NDT, NT = 256, BM = 128, KT = sizeof(T) == 4 ? 32 : 64, NSUB = KT / 32;
  using L = Tile<T, DP, KT>;
  using E = Elem<T>;
  using F = Fast<T>;
  constexpr int BYTES = KT * L::kRow;
  __shared__ __align__(16) char K0[BYTES], K1[BYTES], V0[BYTES], V1[BYTES];

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, G = a.G, D = a.D;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // a key-value head's blocks share an XCD's L2 where there are 8 of them
  const int hk = blockIdx.x % a.HK;
  const Place pl = find_place<false>(a.cu, a.n_seq, a.total, G, BM, a.slots, (int)(blockIdx.x / a.HK), lane);
  if (pl.tile < 0) return;
  const int rows = pl.len * G, r0 = pl.tile * BM + wave * 32;
  const int r = r0 + (lane & 31), rc = min(r, rows - 1), t = rc / G, h = hk * G + rc % G;
  const T* Kb = K + (int64_t)pl.start * a.k_st + (int64_t)hk * a.k_sh;
  const T* Vb = V + (int64_t)pl.start * a.v_st + (int64_t)hk * a.v_sh;
  Stage<T, DP, KT, NT, A> ks_, vs_;
  auto begin = [&](int kt, char* Kd, char* Vd) {
    ks_.begin_head(Kb, kt * KT, pl.len, a.k_st, Kd, D, tid);
    vs_.begin_head(Vb, kt * KT, pl.len, a.v_st, Vd, D, tid);
  };
  auto end = [&](char* Kd, char* Vd) {
    ks_.end(Kd, tid);
    vs_.end(Vd, tid);
  };
  const int n_kt = min(pl.tile * BM + BM - 1, rows - 1) / G / KT + 1;  // tiles that the block sweeps
  const int t_first = __builtin_amdgcn_readfirstlane(t), t_last = __builtin_amdgcn_readlane(t, 31);
  const int n_w = r0 < rows ? t_last / KT + 1 : 0;  // tiles with a key before some query of the wave
  begin(0, K0, V0);

  typename F::Frag qf[NKS];
  const T* Qr = Q + (int64_t)(pl.start + t) * a.q_st + (int64_t)h * a.q_sh;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) qf[ks] = fast_of<T>(row8<T, A>(Qr, 16 * ks + 8 * g, D));
  end(K0, V0);

  float m = -INFINITY, l = 0.f;  // running maximum (log2 units), this lane's part of the row sum
  floatx16 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = zeros16();
  auto tile = [&](int kt, const char* Kt, const char* Vt) {
    const int k0 = kt * KT;
    int ln = lane;
    if constexpr (kTight<T, DP>) pin(ln);
    floatx16 s[NSUB];
    typename F::Sum sum;
    typename F::Frag f[2];
    const bool cut = k0 + KT - 1 > t_first;  // the mask cuts through the tile
    float mx = -INFINITY, sub = 0.f;
    auto weigh = [&](int x, int i) {
      s[x][i] = fast_exp2(fmaf(s[x][i], sl2, -sub));
      l += s[x][i];
    };
    // the scores of the tile's rows, 32 by 32, beside them the maximum of the last 32;
    // then O += P V, beside it the weights of the next 32
    constexpr int S = NSUB * NKS, C = 2 * NDT, E = 16 / NKS;
    static_assert(NKS == C, "as many steps to a product as to the other");
    ahead<T, 0, S + NSUB * C>(
        [&](auto i) {
          return i < S ? L::rows32(Kt, 32 * (i / NKS), i % NKS, ln)
                       : L::cols32(Vt, 2 * ((i - S) / C) + i % 2, (i - S) % C / 2, ln);
        },
        [&](auto i, const typename F::Frag& y) {
          if (i < S) {
            const int x = i / NKS, ks = i % NKS;
            if (ks == 0) sum = typename F::Sum();
            sum.add(y, qf[ks]);
            if (x > 0)
#pragma unroll
              for (int e = 0; e < E; ++e) mx = vmax2(mx, s[x - 1][E * ks + e]);
            if (ks == NKS - 1) {
              s[x] = sum.value();
              if (cut) {  // wave-uniform
                int mine = t - k0;
                pin(mine);  // (else the masks are formed before the branch, every time)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[x][e] = 32 * x + row32(e, g) > mine ? -INFINITY : s[x][e];
              }
            }
            if (i == S - 1) {
#pragma unroll
              for (int e = 0; e < 16; ++e) mx = vmax2(mx, s[x][e]);
              mx = pair_max32(mx) * sl2;
              // O and l keep the maximum they have until one passes it by 2^8: the sums
              // stay far from fp32's and P from its type's limits, and most tiles need no
              // rescaling
              if (__builtin_amdgcn_ballot_w64(mx > m + 8.f) != 0) {
                const float mn = vmax2(m, mx);
                float alpha = mn == m ? 1.f : fast_exp2(m - mn);
                pin(alpha);  // (else the products are formed before the branch, every time)
                m = mn;
                l *= alpha;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
              }
              sub = m == -INFINITY ? 0.f : m;  // only scores of -inf so far: weights of 0
#pragma unroll
              for (int e = 0; e < 16; ++e) weigh(0, e);
              pack_rows<T>(s[0], f);
            }
          } else {
            const int x = (i - S) / C, j = (i - S) % C;
            add_cols<T>(j, y, f, o, sum);
            if (x + 1 < NSUB) {
#pragma unroll
              for (int e = 0; e < E; ++e) weigh(x + 1, E * j + e);
              if (j == C - 1) pack_rows<T>(s[x + 1], f);
            }
          }
        });
  };
  auto step = [&](int kt, char* Kt, char* Vt, char* Kn, char* Vn) {
    if constexpr (sizeof(T) == 2) wait_vmem();
    __syncthreads();  // tile kt is in LDS; every wave is done with the other buffers
    if (kt + 1 < n_kt) begin(kt + 1, Kn, Vn);
    if (kt < n_w) tile(kt, Kt, Vt);
    if (kt + 1 < n_kt) end(Kn, Vn);
  };
  for (int kt = 0; kt < n_kt; kt += 2) {
    step(kt, K0, V0, K1, V1);
    if (kt + 1 < n_kt) step(kt + 1, K1, V1, K0, V0);
  }
  l = pair_sum32(l);
  __syncthreads();  // the tiles' LDS is free
  T* Or = O + (int64_t)(pl.start + t) * a.o_st + (int64_t)h * a.o_sh;
  float* lse_at = LSE == nullptr ? nullptr : LSE + (int64_t)h * a.total + pl.start + t;
  if (any_not_finite(o, r < rows)) {
    fwd_again<T, NKS, NDT, A>(Qr, Kb, Vb, Or, lse_at, reinterpret_cast<T*>(wave & 2 ? K1 : K0) + (wave & 1) * 1024,
                              a.k_st, a.v_st, pl.len, D, r < rows, t, t_first, t_last, sl2, lane);
  } else if (r < rows) {
    store_row<T, NDT, A>(Or, D, g, o, 1.f / l);
    if (lse_at != nullptr && g == 0) *lse_at = fmaf(m, kLn2, logf(l));
  }
}

// ---------------------------------------------------------------- backward
// Query-stationary: dQ, and the row statistics lse log2(e) and Delta that the
// key-stationary kernel reads.
//
// Delta = do . o takes o as the forward rounded it; in 16 bits the error is as large
// as that of the rounded score gradients where a row has few keys.  Blocks whose
// rows all lie below kShort sum Delta over p dp in a sweep of its own instead: dQ of
// 12 ragged sequences of up to 1024 is off by 1.7e-3 of its norm that way, by 2.5e-3
// with Delta from o everywhere; a sequence of 1024 is swept a sixteenth longer.
//
// 16 bits, 32 query heads of 128 in 8 groups, 4 sequences of 4096: 480 us, 1.0
// PFLOP/s of its three products; bound as the forward is.  fp32 takes one wave to a
// SIMD: 45 us for 16 sequences of up to 512, 8 heads of 48, with two (and spills) 48.
constexpr int kShort = 256;
template <class T, int NKS, int NDT, int A>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) void packed_dq_kernel(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, const T* __restrict__ O,
    const T* __restrict__ DO, const float* __restrict__ LSE, T* __restrict__ DQ, float* __restrict__ LSE2,
    float* __restrict__ DELTA, PackedArgs a, float sl2, float scale) {
  constexpr int DP = 32 * NDT, NT = 256, BM = 128, KT = sizeof(T) == 4 ? 32 : 64, NSUB = KT / 32;
  using L = Tile<T, DP, KT>;
  using F = Fast<T>;
  constexpr int BYTES = KT * L::kRow;
  __shared__ __align__(16) char K0[BYTES], K1[BYTES], V0[BYTES], V1[BYTES];

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, G = a.G, D = a.D;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x % a.HK;
  const Place pl = find_place<false>(a.cu, a.n_seq, a.total, G, BM, a.slots, (int)(blockIdx.x / a.HK), lane);
  if (pl.tile < 0) return;
  const int rows = pl.len * G, r0 = pl.tile * BM + wave * 32;
  const int r = r0 + (lane & 31), rc = min(r, rows - 1), t = rc / G, h = hk * G + rc % G;
  const T* Kb = K + (int64_t)pl.start * a.k_st + (int64_t)hk * a.k_sh;
  const T* Vb = V + (int64_t)pl.start * a.v_st + (int64_t)hk * a.v_sh;
  Stage<T, DP, KT, NT, A> ks_, vs_;
  auto begin = [&](int kt, char* Kd, char* Vd) {
    ks_.begin_head(Kb, kt * KT, pl.len, a.k_st, Kd, D, tid);
    vs_.begin_head(Vb, kt * KT, pl.len, a.v_st, Vd, D, tid);
  };
  auto end = [&](char* Kd, char* Vd) {
    ks_.end(Kd, tid);
    vs_.end(Vd, tid);
  };
  const int t_end = min(pl.tile * BM + BM - 1, rows - 1) / G;
  const int n_kt = t_end / KT + 1;
  const int t_first = __builtin_amdgcn_readfirstlane(t), t_last = __builtin_amdgcn_readlane(t, 31);
  const int n_w = r0 < rows ? t_last / KT + 1 : 0;
  begin(0, K0, V0);

  typename F::Frag qf[NKS], dof[NKS];
  const T* Qr = Q + (int64_t)(pl.start + t) * a.q_st + (int64_t)h * a.q_sh;
  const int64_t o_at = (int64_t)(pl.start + t) * a.o_st + (int64_t)h * a.o_sh;
  const int64_t stat_at = (int64_t)h * a.total + pl.start + t;
  float delta = 0.f;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    qf[ks] = fast_of<T>(row8<T, A>(Qr, 16 * ks + 8 * g, D));
    const typename Elem<T>::Frag d = row8<T, A>(DO + o_at, 16 * ks + 8 * g, D);
    const typename Elem<T>::Frag of = row8<T, A>(O + o_at, 16 * ks + 8 * g, D);
#pragma unroll
    for (int j = 0; j < 8; ++j) delta = fmaf((float)of[j], (float)d[j], delta);
    dof[ks] = fast_of<T>(d);
  }
  delta = pair_sum32(delta);
  const float lse2 = LSE[stat_at] * kLog2e;
  end(K0, V0);
  floatx16 dq[NDT];
  float sum_delta = 0.f;
  auto tile = [&](auto sums, int kt, const char* Kt, const char* Vt) {
    constexpr bool SUMS = decltype(sums)::value;  // the sweep that sums Delta
    const int k0 = kt * KT;
    int ln = lane;
    if constexpr (kTight<T, DP>) pin(ln);
    const bool cut = k0 + KT - 1 > t_first;
    // the scores and dO V^T of 32 keys after 32, two chains of MFMAs side by side, and
    // dS = p (dO V^T - Delta); then dQ += dS K
    typename F::Frag f[NSUB][2];
    floatx16 all[NSUB];
    typedef Step<typename F::Frag, 1> Reads;
    each(std::make_integer_sequence<int, NSUB>(), [&](auto x) {
      typename F::Sum sum, dsum;
      ahead<T, 0, NKS>(
          [&](auto ks) {
            Reads y;
            y.a = L::rows32(Kt, 32 * x, ks, ln);
            y.b = L::rows32(Vt, 32 * x, ks, ln);
            return y;
          },
          [&](auto ks, const Reads& y) {
            sum.add(y.a, qf[ks]);
            dsum.add(y.b, dof[ks]);
          });
      const floatx16 s = sum.value(), dp = dsum.value();
      floatx16 ds;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = fast_exp2(fmaf(s[i], sl2, -lse2));
        ds[i] = SUMS ? p * dp[i] : p * (dp[i] - delta);
      }
      if (cut) {
        int mine = t;
        pin(mine);  // (else the masks are formed before the branch, every time)
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[i] = k0 + 32 * x + row32(i, g) > mine ? 0.f : ds[i];
      }
      if constexpr (SUMS) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sum_delta += ds[i];
      } else {
        all[x] = ds;
      }
    });
    if constexpr (!SUMS)
#pragma unroll
      for (int x = 0; x < NSUB; ++x) pack_rows<T>(all[x], f[x]);
    if constexpr (!SUMS) {
      constexpr int N = 2 * NSUB;
      typename F::Sum sum;
      ahead<T, 0, N * NDT>([&](auto i) { return L::cols32(Kt, i % N, i / N, ln); },
                           [&](auto i, const typename F::Frag& y) {
                             add_cols<T, N>(i, y, f[i % N / 2], dq, sum);
                           });
    }
  };
  auto sweep = [&](auto sums) {
    auto step = [&](int kt, char* Kt, char* Vt, char* Kn, char* Vn) {
      if constexpr (sizeof(T) == 2) wait_vmem();
      __syncthreads();
        if (kt + 1 < n_kt) begin(kt + 1, Kn, Vn);
      if (kt < n_w) tile(sums, kt, Kt, Vt);
      if (kt + 1 < n_kt) end(Kn, Vn);
    };
    for (int kt = 0; kt < n_kt; kt += 2) {
      step(kt, K0, V0, K1, V1);
      if (kt + 1 < n_kt) step(kt + 1, K1, V1, K0, V0);
    }
    __syncthreads();
  };
  if constexpr (sizeof(T) == 2) {
    if (t_end < kShort) {
      sweep(std::true_type{});
      delta = pair_sum32(sum_delta);
      begin(0, K0, V0);
    }
  }
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) dq[dt] = zeros16();
  sweep(std::false_type{});
  if (r < rows && g == 0) {
    LSE2[stat_at] = lse2;
    DELTA[stat_at] = delta;
  }
  T* dq_at = DQ + (int64_t)(pl.start + t) * a.q_st + (int64_t)h * a.q_sh;
  if (any_not_finite(dq, r < rows))
    dq_again<T, NKS, NDT, A>(Qr, Kb, Vb, DO + o_at, dq_at, reinterpret_cast<T*>(wave & 2 ? K1 : K0) + (wave & 1) * 1024,
                             a.k_st, a.v_st, pl.len, D, r < rows, t, t_first, t_last, sl2, lse2, delta, scale, lane);
  else if (r < rows)
    store_row<T, NDT, A>(dq_at, D, g, dq, scale);
}

// Key-stationary: dK and dV of 32 KG keys, over the rows of the group that come
// after them: KG waves of 32 keys each, times 4 / KG that take every other 32 rows
// and are added up at the end (KG = 2: where blocks of 128 keys are too few for the
// CUs).
//
// 16 bits, 32 query heads of 128 in 8 groups, 4 sequences of 4096: 1000 us, 0.64
// PFLOP/s of its four products: dK, dV and K fill the registers (V is read from LDS
// again for every tile), which leaves none to read ahead from one product to the next
// or to form p and dS beside the MFMAs (1470 us: a spill among the loads in flight
// waits for all of them).  64 columns leave them: 50 us for 12 sequences of up to
// 1024, 12 heads of 64 in 4 groups, one product after the other 56.
template <class T, int NKS, int NDT, int KG, int A>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) void packed_dkv_kernel(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, const T* __restrict__ DO,
    const float* __restrict__ LSE2, const float* __restrict__ DELTA, T* __restrict__ DK, T* __restrict__ DV,
    PackedArgs a, float sl2, float scale) {
  static_assert(KG == 4 || KG == 2, "one or two row groups");
  constexpr int DP = 32 * NDT, NT = 256, BN = 32 * KG, RG = 4 / KG, QT = 32 * RG;
  using L = Tile<T, DP, QT>;
  using F = Fast<T>;
  constexpr int BYTES = QT * L::kRow;
  // 16-bit: V of the block's keys in LDS, in registers it would not fit beside K, dK
  // and dV of 128; fp32: in registers, LDS would hold fewer blocks
  constexpr bool V_LDS = sizeof(T) == 2;
  using LV = LdsTile<typename std::conditional<V_LDS, T, __bf16>::type, DP>;
  __shared__ __align__(16) char Q0[BYTES], Q1[BYTES], D0[BYTES], D1[BYTES];
  __shared__ __align__(16) float S0[2 * QT], S1[2 * QT];  // a tile's lse log2(e), then its Delta
  __shared__ __align__(16) char VS[V_LDS ? BN * LV::kRow : 16];

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, G = a.G, D = a.D;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave % KG, rg = wave / KG;
  const int hk = blockIdx.x % a.HK;
  const Place pl = find_place<true>(a.cu, a.n_seq, a.total, 1, BN, a.slots, (int)(blockIdx.x / a.HK), lane);
  if (pl.tile < 0) return;
  const int rows = pl.len * G, key0 = pl.tile * BN + kg * 32;
  const int key = key0 + (lane & 31);
  const int first = key * G;  // the first row that comes at or after the key
  const T* Qb = Q + (int64_t)pl.start * a.q_st + (int64_t)hk * G * a.q_sh;
  const T* Db = DO + (int64_t)pl.start * a.o_st + (int64_t)hk * G * a.o_sh;
  const T* Vb = V + (int64_t)pl.start * a.v_st + (int64_t)hk * a.v_sh;
  const int64_t stat0 = (int64_t)hk * G * a.total + pl.start;
  // position and head of row rr of a tile (G <= 128: a 16-bit reciprocal is exact
  // below 512); rows behind the last one repeat it
  const int magic = 65535 / G + 1;
  Stage<T, DP, QT, NT, A> qs_, ds_;
  auto begin = [&](int rt, char* Qd, char* Dd, float* Sd) {
    const int t0 = rt * QT / G, g0 = rt * QT % G, last = rows - 1 - rt * QT;
    auto place = [&](int rr, int& t, int& gq) {
      const int x = min(rr, last) + g0;
      t = (x * magic) >> 16;
      gq = x - t * G;
    };
    auto at = [&](int rr, int64_t st, int64_t sh) {
      int t, gq;
      place(rr, t, gq);
      return ((int)__umul24(t, (int)st) + gq * (int)sh) * (int)sizeof(T);  // (64 st is below 2^31 / size)
    };
    const __amdgpu_buffer_rsrc_t rq = buffer_rsrc(Qb + (int64_t)t0 * a.q_st, 0x7fffffffu);
    const __amdgpu_buffer_rsrc_t rd = buffer_rsrc(Db + (int64_t)t0 * a.o_st, 0x7fffffffu);
    qs_.begin(rq, Qd, D, tid, [&](int rr) { return at(rr, a.q_st, a.q_sh); });
    ds_.begin(rd, Dd, D, tid, [&](int rr) { return at(rr, a.o_st, a.o_sh); });
    if (wave < RG) {  // 64 of the 2 QT statistics to a wave
      int t, gq;
      place((wave * 64 + lane) % QT, t, gq);
      const int64_t i = stat0 + (int64_t)gq * a.total + t0 + t;
      dma_dword((wave * 64 + lane < QT ? LSE2 : DELTA) + i, Sd + wave * 64);
    }
  };
  auto end = [&](char* Qd, char* Dd) {
    qs_.end(Qd, tid);
    ds_.end(Dd, tid);
  };
  const int rt0 = pl.tile * BN * G / QT, n_rt = (rows + QT - 1) / QT;
  // sub-tiles of 32 rows: the first with a row after some key of the wave
  const int sub0 = key0 < pl.len ? key0 * G / 32 : 0x7fffffff;
  if constexpr (V_LDS) Stage<T, DP, BN, NT, A>().begin_head(Vb, pl.tile * BN, pl.len, a.v_st, VS, D, tid);
  begin(rt0, Q0, D0, S0);
  const char* Vw = VS + kg * 32 * LV::kRow;

  typename F::Frag kf[NKS], vf[V_LDS ? 1 : NKS];
  {
    const int kc = min(key, pl.len - 1);
    const T* Kr = K + (int64_t)(pl.start + kc) * a.k_st + (int64_t)hk * a.k_sh;
    const T* Vr = Vb + (int64_t)kc * a.v_st;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      kf[ks] = fast_of<T>(row8<T, A>(Kr, 16 * ks + 8 * g, D));
      if constexpr (!V_LDS) vf[ks] = fast_of<T>(row8<T, A>(Vr, 16 * ks + 8 * g, D));
    }
  }
  end(Q0, D0);
  floatx16 dk[NDT], dv[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) dk[dt] = zeros16(), dv[dt] = zeros16();
  // the mask (or the sequence's end) cuts through sub-tile x
  auto is_cut = [&](int x) { return x * 32 < (key0 + 31) * G || x * 32 + 32 > rows; };
  auto tile = [&](int x, const char* Qt, const char* Dt, const float* St) {
    const int r0 = x * 32;
    int ln = lane;
    if constexpr (kTight<T, DP>) pin(ln);
    // the scores; V dO^T, beside it the weights p; dV += p dO, beside it
    // dS = p (V dO^T - Delta), in dp's place; dK += dS Q
    floatx16 p, dp;
    typename F::Sum sum;
    typename F::Frag f[2];
    constexpr int C = 2 * NDT, E = 16 / NKS;
    static_assert(NKS == C, "as many steps to a product as to the others");
    constexpr bool BESIDE = NDT <= 2;  // where there are registers for it
    typedef Step<typename F::Frag, E> Reads;
    auto load = [&](auto i) {
          Reads y;
          const int k = i % NKS, el = E * k;
          const float* st = St + 8 * (el / 4) + 4 * g + el % 4;
          if (i < NKS) {
            y.a = L::rows32(Qt, 0, k, ln);
          } else if (i < 2 * NKS) {
            y.a = L::rows32(Dt, 0, k, ln);
            if constexpr (V_LDS) y.b = LV::rows32(Vw, 0, k, ln);
            if constexpr (BESIDE)
#pragma unroll
              for (int e = 0; e < E; ++e) y.stat[e] = st[e];
          } else if (i < 2 * NKS + C) {
            y.a = L::cols32(Dt, k % 2, k / 2, ln);
            if constexpr (BESIDE)
#pragma unroll
              for (int e = 0; e < E; ++e) y.stat[e] = st[QT + e];
          } else {
            y.a = L::cols32(Qt, k % 2, k / 2, ln);
          }
          return y;
        };
    auto use = [&](auto i, const Reads& y) {
          const int k = i % NKS;
          if (i < 2 * NKS && k == 0) sum = typename F::Sum();
          if (i < NKS) {
            sum.add(y.a, kf[k]);
            if (k == NKS - 1) p = sum.value();
          } else if (i < 2 * NKS) {
            if constexpr (V_LDS)
              sum.add(y.a, y.b);
            else
              sum.add(y.a, vf[k]);
            if constexpr (BESIDE)
#pragma unroll
              for (int e = 0; e < E; ++e) p[E * k + e] = fast_exp2(fmaf(p[E * k + e], sl2, -y.stat[e]));
            if (k == NKS - 1) {
              dp = sum.value();
              if constexpr (!BESIDE) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                  const floatx4 lse2 = *reinterpret_cast<const floatx4*>(St + 8 * u + 4 * g);
                  const floatx4 delta = *reinterpret_cast<const floatx4*>(St + QT + 8 * u + 4 * g);
#pragma unroll
                  for (int e = 4 * u; e < 4 * u + 4; ++e) {
                    p[e] = fast_exp2(fmaf(p[e], sl2, -lse2[e % 4]));
                    dp[e] = p[e] * (dp[e] - delta[e % 4]);
                  }
                  // (no more of the statistics in registers: one spill in this loop is a wait
                  // for all loads in flight, the next tile's)
                  WHA_FENCE();
                }
              }
              if (is_cut(x)) {
                int from = first;
                pin(from);  // (else the masks are formed before the branch, every time)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  const int row = r0 + row32(e, g);
                  const bool in = row >= from && row < rows;
                  p[e] = in ? p[e] : 0.f;
                  if constexpr (!BESIDE) dp[e] = in ? dp[e] : 0.f;
                }
              }
              pack_rows<T>(p, f);
            }
          } else if (i < 2 * NKS + C) {
            add_cols<T>(k, y.a, f, dv, sum);
            if constexpr (BESIDE)
#pragma unroll
              for (int e = 0; e < E; ++e) dp[E * k + e] = p[E * k + e] * (dp[E * k + e] - y.stat[e]);
            if (k == C - 1) pack_rows<T>(dp, f);
          } else {
            add_cols<T>(k, y.a, f, dk, sum);
          }
        };
    if constexpr (BESIDE) {
      ahead<T, 0, 2 * NKS + 2 * C>(load, use);
    } else {  // (and no reads on the way from one product to the next)
      ahead<T, 0, NKS, 1>(load, use);
      ahead<T, NKS, 2 * NKS, 1>(load, use);
      ahead<T, 2 * NKS, 2 * NKS + C, 1>(load, use);
      ahead<T, 2 * NKS + C, 2 * NKS + 2 * C, 1>(load, use);
    }
  };
  // rows 32 rg .. of a tile (fp32: of each of its parts)
  const int own = rg * 32 * (V_LDS ? L::kRow : LV::kRow);
  auto step = [&](int rt, char* Qt, char* Dt, float* St, char* Qn, char* Dn, float* Sn) {
    wait_vmem();
    __syncthreads();
    if (rt + 1 < n_rt) begin(rt + 1, Qn, Dn, Sn);
    const int x = rt * RG + rg;
    if (x >= sub0 && x * 32 < rows) tile(x, Qt + own, Dt + own, St + rg * 32);
    if (rt + 1 < n_rt) end(Qn, Dn);
  };
  for (int rt = rt0; rt < n_rt; rt += 2) {
    step(rt, Q0, D0, S0, Q1, D1, S1);
    if (rt + 1 < n_rt) step(rt + 1, Q1, D1, S1, Q0, D0, S0);
  }
  __syncthreads();  // the tiles' LDS is free
  if constexpr (RG == 2) {  // the second row group's sums by way of LDS: dK in Q0 or Q1, dV in D0 or D1
    __syncthreads();
    float* k_sum = reinterpret_cast<float*>(kg ? Q1 : Q0) + lane;
    float* v_sum = reinterpret_cast<float*>(kg ? D1 : D0) + lane;
    static_assert(BYTES >= NDT * 16 * 64 * 4, "a wave's sums in one buffer");
    if (rg == 1) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          k_sum[(16 * dt + i) * 64] = dk[dt][i];
          v_sum[(16 * dt + i) * 64] = dv[dt][i];
        }
    }
    __syncthreads();
    if (rg == 1) return;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        dk[dt][i] += k_sum[(16 * dt + i) * 64];
        dv[dt][i] += v_sum[(16 * dt + i) * 64];
      }
  }
  // (the lane's addresses once more: kept over the loop they would be spilled, or K)
  int ln = lane;
  pin(ln);
  const int my_key = key0 + (ln & 31), row = pl.start + min(my_key, pl.len - 1);
  const bool on = my_key < pl.len;
  T* dk_at = DK + (int64_t)row * a.k_st + (int64_t)hk * a.k_sh;
  T* dv_at = DV + (int64_t)row * a.v_st + (int64_t)hk * a.v_sh;
  const bool bad_k = any_not_finite(dk, on), bad_v = any_not_finite(dv, on);
  if (bad_k || bad_v) {
    const T* Kr = K + (int64_t)row * a.k_st + (int64_t)hk * a.k_sh;
    const T* Vr = V + (int64_t)row * a.v_st + (int64_t)hk * a.v_sh;
    // (two row groups: a wave's own buffer, the other wave may still read its sums)
    T* w = RG == 2 ? reinterpret_cast<T*>(kg ? Q1 : Q0) : reinterpret_cast<T*>(wave & 2 ? Q1 : Q0) + (wave & 1) * 1024;
    dkv_again<T, NKS, NDT, A, true>(Qb, Kr, Vr, Db, LSE2 + stat0, DELTA + stat0, dk_at, w, a.q_st, a.q_sh, a.o_st,
                                    a.o_sh, a.total, G, D, rows, key0, on, sl2, scale, ln);
    dkv_again<T, NKS, NDT, A, false>(Qb, Kr, Vr, Db, LSE2 + stat0, DELTA + stat0, dv_at, w, a.q_st, a.q_sh, a.o_st,
                                     a.o_sh, a.total, G, D, rows, key0, on, sl2, 1.f, ln);
  } else if (on) {
    store_row<T, NDT, A>(dk_at, D, ln >> 5, dk, scale);
    store_row<T, NDT, A>(dv_at, D, ln >> 5, dv, 1.f);
  }
}

// ---------------------------------------------------------------- launches
namespace {

template <class T, int NKS, int NDT, int A>
hipError_t fwd_t(const void* q, const void* k, const void* v, void* o, float* lse, PackedArgs a, float scale,
                 hipStream_t stream) {
  a.slots = packed_slots(a, 128, a.G);
  TimingScope ts("packed_fwd", stream);
  hipLaunchKernelGGL((packed_fwd_kernel<T, NKS, NDT, A>), dim3((unsigned)a.slots * a.HK), dim3(256), 0, stream,
                     static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                     static_cast<T*>(o), lse, a, (float)((double)scale * 1.4426950408889634));
  return hipGetLastError();
}

template <class T, int NKS, int NDT, int A>
hipError_t bwd_t(const void* q, const void* k, const void* v, const void* o, const void* d_o, const float* lse,
                 void* dq, void* dk, void* dv, float* ws, PackedArgs a, float scale, hipStream_t stream) {
  const float sl2 = (float)((double)scale * 1.4426950408889634);
  float *lse2 = ws, *delta = ws + (int64_t)a.total * a.HK * a.G;
  {
    TimingScope ts("packed_bwd_dq", stream);
    a.slots = packed_slots(a, 128, a.G);
    hipLaunchKernelGGL((packed_dq_kernel<T, NKS, NDT, A>), dim3((unsigned)a.slots * a.HK), dim3(256), 0, stream,
                       static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                       static_cast<const T*>(o), static_cast<const T*>(d_o), lse, static_cast<T*>(dq), lse2, delta, a,
                       sl2, scale);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  TimingScope ts("packed_bwd_dkv", stream);
  auto launch = [&](auto kernel, int keys) {
    a.slots = packed_slots(a, keys, 1);
    hipLaunchKernelGGL(kernel, dim3((unsigned)a.slots * a.HK), dim3(256), 0, stream, static_cast<const T*>(q),
                       static_cast<const T*>(k), static_cast<const T*>(v), static_cast<const T*>(d_o), lse2, delta,
                       static_cast<T*>(dk), static_cast<T*>(dv), a, sl2, scale);
  };
  // Blocks of 64 keys where those of 128 come to fewer than two to a CU: 12 sequences
  // of up to 1024, 12 heads of 64 in 4 groups 63 us against 111, fp32 of 16 sequences
  // of up to 512, 8 heads of 48 60 against 64.  Heads of more than 64 take 128 always:
  // 4 sequences of 4096, 8 heads of 128 1090 us against 1556.
  if constexpr (NDT <= 2) {
    if ((int64_t)a.total * a.HK < 512 * 128) {
      launch(packed_dkv_kernel<T, NKS, NDT, 2, A>, 64);
      return hipGetLastError();
    }
  }
  launch(packed_dkv_kernel<T, NKS, NDT, 4, A>, 128);
  return hipGetLastError();
}

// F<T, steps of 16 over the head dim, 32-wide tiles of it, alignment of rows>
#define WHA_BY_DIM(F, T, ...)                                                                     \
  (a.D <= 64 ? (align == 16  ? F<T, 4, 2, 16>(__VA_ARGS__)                                        \
                : align == 4 ? F<T, 4, 2, 4>(__VA_ARGS__)                                         \
                             : F<T, 4, 2, sizeof(T) == 4 ? 4 : 2>(__VA_ARGS__))                   \
             : (align == 16  ? F<T, 8, 4, 16>(__VA_ARGS__)                                        \
                : align == 4 ? F<T, 8, 4, 4>(__VA_ARGS__)                                         \
                             : F<T, 8, 4, sizeof(T) == 4 ? 4 : 2>(__VA_ARGS__)))

}  // namespace

hipError_t launch_packed_fwd(int dtype, const void* q, const void* k, const void* v, void* o, float* lse,
                             const PackedArgs& a, int align, float scale, hipStream_t stream) {
  if (dtype == kF32) return WHA_BY_DIM(fwd_t, float, q, k, v, o, lse, a, scale, stream);
  if (dtype == kBf16) return WHA_BY_DIM(fwd_t, __bf16, q, k, v, o, lse, a, scale, stream);
  return WHA_BY_DIM(fwd_t, _Float16, q, k, v, o, lse, a, scale, stream);
}

hipError_t launch_packed_bwd(int dtype, const void* q, const void* k, const void* v, const void* o, const void* d_o,
                             const float* lse, void* dq, void* dk, void* dv, float* ws, const PackedArgs& a, int align,
                             float scale, hipStream_t stream) {
  if (dtype == kF32) return WHA_BY_DIM(bwd_t, float, q, k, v, o, d_o, lse, dq, dk, dv, ws, a, scale, stream);
  return WHA_BY_DIM(bwd_t, __bf16, q, k, v, o, d_o, lse, dq, dk, dv, ws, a, scale, stream);
}

}  // namespace wha
