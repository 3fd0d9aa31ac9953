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

#include "wha_elem.hpp"
#include "wha_packed.hpp"

namespace wha {

namespace {

// Which tile of which sequence block number `order` takes (of one key-value head's).
// A tile's level is the number of tiles that it sweeps less one: those before it in
// its sequence, or with KEYS (tiles of keys, swept by the rows after them) those
// after it.  Up to 64 sequences: the highest level first, whatever the sequence, so
// that the longest sweeps start first and the short ones fill in behind them.  More
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

// A tile of rows into LDS, ROWS x DP by NT threads.  VEC: direct-to-LDS buffer loads
// from `base`, the address of the tile's first row, complete after wait_vmem: a
// lane's offsets stay the same from tile to tile, and what moves is the descriptor,
// in scalar registers.  Offsets past its range read as zeros: rows behind the last
// one, and quads past the head dim.
constexpr int kPast = (int)0x80000000;
template <class T, int DP, int ROWS, int NT>
struct Stage {
  using L = LdsTile<T, DP>;
  static constexpr int PER = ROWS * L::kQuads / NT, Q = Elem<T>::kQuad;
  static_assert(ROWS * L::kQuads % NT == 0, "whole rounds");
  __device__ __forceinline__ static int row(int p, int tid) { return (p * NT + tid) / L::kQuads; }
  __device__ __forceinline__ static int quad(int p, int tid) {
    return ((p * NT + tid) % L::kQuads) ^ L::swz(row(p, tid));
  }
  // byte offset of quad c of a row `off` elements from the base
  __device__ __forceinline__ static int at(int64_t off, int c, int D) {
    return c * Q < D ? (int)((off + c * Q) * (int)sizeof(T)) : kPast;
  }
  __device__ __forceinline__ static void dma(__amdgpu_buffer_rsrc_t r, int off, char* lds, int p, int tid) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        r, (void __attribute__((address_space(3)))*)(lds + (p * NT + (tid & ~63)) * 16), 16, off, 0, 0, 0);
  }
  // one element at a time, from the row at `src`
  __device__ __forceinline__ static void copy(const T* src, char* lds, int p, int tid, int D) {
    const int c = quad(p, tid);
    T x[Q];
#pragma unroll
    for (int e = 0; e < Q; ++e) x[e] = c * Q + e < D ? src[c * Q + e] : (T)0.f;
    uintx4 y;
    __builtin_memcpy(&y, x, 16);
    *reinterpret_cast<uintx4*>(lds + (p * NT + tid) * 16) = y;
  }
  // rows row0 .. of one head, st elements apart, n of them in all
  struct Lanes {
    int off[PER];
  };
  template <bool VEC>
  __device__ __forceinline__ static void lanes(Lanes& l, int64_t st, int D, int tid) {
    if constexpr (VEC) {
#pragma unroll
      for (int p = 0; p < PER; ++p) l.off[p] = at(row(p, tid) * st, quad(p, tid), D);
    }
  }
  template <bool VEC>
  __device__ __forceinline__ static void head(const Lanes& l, const T* base, int row0, int n, int64_t st, int D,
                                              char* lds, int tid) {
    if constexpr (VEC) {
      const int64_t left = ((int64_t)(min(n - row0, ROWS) - 1) * st + D) * (int64_t)sizeof(T);
      const __amdgpu_buffer_rsrc_t r = buffer_rsrc(base + (int64_t)row0 * st, (uint32_t)left);
#pragma unroll
      for (int p = 0; p < PER; ++p) dma(r, l.off[p], lds, p, tid);
    } else {
#pragma unroll
      for (int p = 0; p < PER; ++p) copy(base + (int64_t)min(row0 + row(p, tid), n - 1) * st, lds, p, tid, D);
    }
  }
};

// d = 16 ks + 8 g .. + 7 of one row as a fragment (zero past the head dim).
template <class T, bool VEC>
__device__ __forceinline__ typename Elem<T>::Frag row_frag(const T* row, int ks, int g, int D) {
  const int c = 16 * ks + 8 * g;
  float x[8];
  if constexpr (VEC && sizeof(T) == 2) {
    uintx4 q = {0u, 0u, 0u, 0u};
    if (c < D) q = *reinterpret_cast<const uintx4*>(row + c);
    return __builtin_bit_cast(typename Elem<T>::Frag, q);
  } else if constexpr (VEC) {
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

// Writes a lane's part of X^T[d][row] (d = 32 dt + row32(i, g)) to its row.
template <class T, int NDT, bool VEC>
__device__ __forceinline__ void store_row(T* dst, int D, int g, const floatx16 (&x)[NDT], float mul) {
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = 32 * dt + 8 * u + 4 * g;
      if constexpr (VEC) {
        if (c < D)
          Elem<T>::store4(dst + c, x[dt][4 * u] * mul, x[dt][4 * u + 1] * mul, x[dt][4 * u + 2] * mul,
                          x[dt][4 * u + 3] * mul);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < D) dst[c + e] = (T)(x[dt][4 * u + e] * mul);
      }
    }
}

// N steps whose operands come from LDS: the reads of step i + 1 go out before the
// MFMAs of step i, no more of them, so that they cost few registers.
template <int N, class Load, class Use>
__device__ __forceinline__ void one_ahead(Load&& load, Use&& use) {
  auto f = load(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    auto next = f;
    if (i + 1 < N) next = load(i + 1);
    use(i, f);
    WHA_FENCE();
    f = next;
  }
}
template <class F, int N>
struct Frags {
  F f[N];
};

// Whether a tile holds an infinity or NaN (one wave looks at all of it).
template <class T, int DP, int ROWS>
__device__ __forceinline__ bool tile_not_finite(const char* t, int lane) {
  unsigned bad = 0;
#pragma unroll 1
  for (int i = lane; i < ROWS * LdsTile<T, DP>::kQuads; i += 64) {
    const uintx4 q = *reinterpret_cast<const uintx4*>(t + 16 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) bad |= not_finite_bits<T>(q[e]);
  }
  return __builtin_amdgcn_ballot_w64(bad != 0) != 0;
}

// acc[d][column] += sum over the tile's rows of p[row][column] x[row][d]; weights of
// rows that do not belong to a column are zero.
template <class T, int DP, int NDT, int NSUB>
__device__ __forceinline__ void add_cols(const char* t, const floatx16 (&p)[NSUB], floatx16 (&acc)[NDT], int lane) {
  typename Elem<T>::Frag f[2 * NSUB];
#pragma unroll
  for (int s = 0; s < 2 * NSUB; ++s) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = p[s / 2][8 * (s & 1) + j];
    f[s] = Elem<T>::pack(x);
  }
  one_ahead<2 * NSUB * NDT>([&](int i) { return LdsTile<T, DP>::cols32(t, i / NDT, i % NDT, lane); },
                            [&](int i, const typename Elem<T>::Frag& x) {
                              acc[i % NDT] = Elem<T>::mma32(x, f[i / NDT], acc[i % NDT]);
                            });
}

// A weight of zero does not undo an infinity or NaN (0 x inf).  So where the mask
// cuts through a tile that holds one, a wave leaves that tile's products and those
// of the cut tiles after it out of its loop, and forms them here at the end: the
// scores once more from memory, then row by row over the rows the mask leaves.  At
// the end, because a second form of the products inside the loop costs the whole
// kernel 60 registers and more.
//
// x y^T of 32 rows of memory each, by lane % 32.
template <class T, int NKS, bool VEC>
__device__ __forceinline__ floatx16 scores_of(const T* x, const T* y, int g, int D) {
  floatx16 s = zeros16();
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    s = Elem<T>::mma32(row_frag<T, VEC>(x, ks, g, D), row_frag<T, VEC>(y, ks, g, D), s);
    WHA_FENCE();
  }
  return s;
}
// acc[d][column] += p[row][column] row(x)[d] over the rows x with mine(x), of 32, the
// weights by way of `w` (32 x 32 of the wave's own LDS).
template <class T, int NDT, class Row, class Mine>
__device__ __forceinline__ void add_rows(const floatx16& p, floatx16 (&acc)[NDT], T* w, int lane, int D, Row&& row,
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

}  // namespace

// Whether a result of any wave of the block is not finite (bad: of this lane).
__device__ __forceinline__ bool any_bad(bool bad, int* flags, int wave, int lane) {
  const uint64_t some = __builtin_amdgcn_ballot_w64(bad);
  if (lane == 0) flags[wave] = some != 0;
  __syncthreads();
  return (flags[0] | flags[1] | flags[2] | flags[3]) != 0;
}
template <int NDT>
__device__ __forceinline__ bool not_finite(const floatx16 (&x)[NDT]) {
  float chk = 0.f;  // NaN if any is not finite
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) chk = fmaf(x[dt][i], 0.f, chk);
  return chk != 0.f;
}

// ---------------------------------------------------------------- forward
template <class T, int NKS, int NDT, bool VEC>
__global__ __launch_bounds__(256, 2) void packed_fwd_kernel(const T* __restrict__ Q, const T* __restrict__ K,
                                                            const T* __restrict__ V, T* __restrict__ O,
                                                            float* __restrict__ LSE, PackedArgs a, float sl2) {
  constexpr int DP = 32 * NDT, NT = 256, BM = 128, KT = sizeof(T) == 4 ? 32 : 64, NSUB = KT / 32;
  using L = LdsTile<T, DP>;
  using St = Stage<T, DP, KT, NT>;
  constexpr int BYTES = KT * L::kRow;
  __shared__ __align__(16) char K0[BYTES], K1[BYTES], V0[BYTES], V1[BYTES];
  __shared__ int flags[4];

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
  typename St::Lanes kl, vl;
  St::template lanes<VEC>(kl, a.k_st, D, tid);
  St::template lanes<VEC>(vl, a.v_st, D, tid);
  auto stage_kv = [&](int kt, char* Kd, char* Vd) {
    St::template head<VEC>(kl, Kb, kt * KT, pl.len, a.k_st, D, Kd, tid);
    St::template head<VEC>(vl, Vb, kt * KT, pl.len, a.v_st, D, Vd, tid);
  };
  const int n_kt = min(pl.tile * BM + BM - 1, rows - 1) / G / KT + 1;  // tiles that the block sweeps
  const int t_first = __builtin_amdgcn_readfirstlane(t), t_last = __builtin_amdgcn_readlane(t, 31);
  const int n_w = r0 < rows ? t_last / KT + 1 : 0;  // tiles with a key before some query of the wave
  stage_kv(0, K0, V0);

  typename Elem<T>::Frag qf[NKS];
  const T* Qr = Q + (int64_t)(pl.start + t) * a.q_st + (int64_t)h * a.q_sh;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) qf[ks] = row_frag<T, VEC>(Qr, ks, g, D);

  float m, l;  // running maximum (log2 units), this lane's part of the row sum
  floatx16 o[NDT];
  bool check = false;
  int left;  // the first cut tile left to the end
  auto tile = [&](int kt, const char* Kt, const char* Vt) {
    const int k0 = kt * KT;
    int ln = lane;
    pin(ln);
    floatx16 s[NSUB];
#pragma unroll
    for (int x = 0; x < NSUB; ++x) s[x] = zeros16();
    one_ahead<NSUB * NKS>([&](int i) { return L::rows32(Kt, 32 * (i / NKS), i % NKS, ln); },
                          [&](int i, const typename Elem<T>::Frag& f) {
                            s[i / NKS] = Elem<T>::mma32(f, qf[i % NKS], s[i / NKS]);
                          });
    const bool cut = k0 + KT - 1 > t_first;  // wave-uniform: the mask cuts through the tile
    if (cut) {
#pragma unroll
      for (int x = 0; x < NSUB; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[x][i] = k0 + 32 * x + row32(i, g) > t ? -INFINITY : s[x][i];
    }
    float mx = s[0][0];
#pragma unroll
    for (int x = 0; x < NSUB; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = vmax2(mx, s[x][i]);
    mx = pair_max32(mx) * sl2;
    // O and l keep the maximum they have until one passes it by 2^8: the sums
    // stay far from fp32's and P from its type's limits, and most tiles need no
    // rescaling
    if (__builtin_amdgcn_ballot_w64(mx > m + 8.f) != 0) {
      const float mn = vmax2(m, mx), alpha = mn == m ? 1.f : fast_exp2(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
    }
    const float sub = m == -INFINITY ? 0.f : m;  // only scores of -inf so far: weights of 0
#pragma unroll
    for (int x = 0; x < NSUB; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[x][i] = fast_exp2(fmaf(s[x][i], sl2, -sub));
        l += s[x][i];
      }
    if (check && cut && kt < left && tile_not_finite<T, DP, KT>(Vt, lane)) left = kt;
    if (kt < left) add_cols<T, DP>(Vt, s, o, ln);
  };
  auto step = [&](int kt, char* Kt, char* Vt, char* Kn, char* Vn) {
    if constexpr (VEC) wait_vmem();
    __syncthreads();  // tile kt is in LDS; every wave is done with the other buffers
    if (kt + 1 < n_kt) stage_kv(kt + 1, Kn, Vn);
    if (kt < n_w) tile(kt, Kt, Vt);
  };
  for (;;) {
    m = -INFINITY, l = 0.f, left = n_w;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = zeros16();
    for (int kt = 0; kt < n_kt; kt += 2) {
      step(kt, K0, V0, K1, V1);
      if (kt + 1 < n_kt) step(kt + 1, K1, V1, K0, V0);
    }
    // an infinity or NaN: once more, with an eye on the tiles that the mask cuts
    if (check || !any_bad(r < rows && not_finite(o), flags, wave, lane)) break;
    check = true;
    stage_kv(0, K0, V0);
  }
  if (check) {
    __syncthreads();  // the tiles' LDS is free
    T* w = reinterpret_cast<T*>(wave & 2 ? K1 : K0) + (wave & 1) * 1024;
    for (int k0 = left * KT; k0 < n_w * KT; k0 += 32) {
      floatx16 s = scores_of<T, NKS, VEC>(Kb + (int64_t)min(k0 + (lane & 31), pl.len - 1) * a.k_st, Qr, g, D);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = fast_exp2(fmaf(s[i], sl2, -(m == -INFINITY ? 0.f : m)));
      add_rows<T>(
          s, o, w, lane, D, [&](int x) { return Vb + (int64_t)min(k0 + x, pl.len - 1) * a.v_st; },
          [&](int x) { return k0 + x <= t; });
    }
  }
  l = pair_sum32(l);
  if (r < rows) {
    store_row<T, NDT, VEC>(O + (int64_t)(pl.start + t) * a.o_st + (int64_t)h * a.o_sh, D, g, o, 1.f / l);
    if (LSE != nullptr && g == 0) LSE[(int64_t)h * a.total + pl.start + t] = fmaf(m, kLn2, logf(l));
  }
}

// ---------------------------------------------------------------- backward
// (fp32 rows of 128 fill a wave's registers with two operands and a result: one
// wave to a SIMD, without spills)
constexpr int waves_per_simd(int size, int ndt) { return size == 4 && ndt > 2 ? 1 : 2; }

// Query-stationary: dQ, and the row statistics lse log2(e) and Delta that the
// key-stationary kernel reads.
template <class T, int NKS, int NDT, bool VEC>
__global__ __launch_bounds__(256, waves_per_simd(sizeof(T), NDT)) void packed_dq_kernel(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, const T* __restrict__ O,
    const T* __restrict__ DO, const float* __restrict__ LSE, T* __restrict__ DQ, float* __restrict__ LSE2,
    float* __restrict__ DELTA, PackedArgs a, float sl2, float scale) {
  constexpr int DP = 32 * NDT, NT = 256, BM = 128, KT = sizeof(T) == 4 ? 32 : 64, NSUB = KT / 32;
  using L = LdsTile<T, DP>;
  using St = Stage<T, DP, KT, NT>;
  constexpr int BYTES = KT * L::kRow;
  __shared__ __align__(16) char K0[BYTES], K1[BYTES], V0[BYTES], V1[BYTES];
  __shared__ int flags[4];

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, G = a.G, D = a.D;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x % a.HK;
  const Place pl = find_place<false>(a.cu, a.n_seq, a.total, G, BM, a.slots, (int)(blockIdx.x / a.HK), lane);
  if (pl.tile < 0) return;
  const int rows = pl.len * G, r0 = pl.tile * BM + wave * 32;
  const int r = r0 + (lane & 31), rc = min(r, rows - 1), t = rc / G, h = hk * G + rc % G;
  const T* Kb = K + (int64_t)pl.start * a.k_st + (int64_t)hk * a.k_sh;
  const T* Vb = V + (int64_t)pl.start * a.v_st + (int64_t)hk * a.v_sh;
  typename St::Lanes kl, vl;
  St::template lanes<VEC>(kl, a.k_st, D, tid);
  St::template lanes<VEC>(vl, a.v_st, D, tid);
  auto stage_kv = [&](int kt, char* Kd, char* Vd) {
    St::template head<VEC>(kl, Kb, kt * KT, pl.len, a.k_st, D, Kd, tid);
    St::template head<VEC>(vl, Vb, kt * KT, pl.len, a.v_st, D, Vd, tid);
  };
  const int n_kt = min(pl.tile * BM + BM - 1, rows - 1) / G / KT + 1;
  const int t_first = __builtin_amdgcn_readfirstlane(t), t_last = __builtin_amdgcn_readlane(t, 31);
  const int n_w = r0 < rows ? t_last / KT + 1 : 0;
  stage_kv(0, K0, V0);

  typename Elem<T>::Frag qf[NKS], dof[NKS];
  const T* Qr = Q + (int64_t)(pl.start + t) * a.q_st + (int64_t)h * a.q_sh;
  const int64_t o_at = (int64_t)(pl.start + t) * a.o_st + (int64_t)h * a.o_sh;
  const int64_t stat_at = (int64_t)h * a.total + pl.start + t;
  float delta = 0.f;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    qf[ks] = row_frag<T, VEC>(Qr, ks, g, D);
    dof[ks] = row_frag<T, VEC>(DO + o_at, ks, g, D);
    const typename Elem<T>::Frag of = row_frag<T, VEC>(O + o_at, ks, g, D);
#pragma unroll
    for (int j = 0; j < 8; ++j) delta = fmaf((float)of[j], (float)dof[ks][j], delta);
  }
  delta = pair_sum32(delta);
  const float lse2 = LSE[stat_at] * kLog2e;
  if (r < rows && g == 0) {
    LSE2[stat_at] = lse2;
    DELTA[stat_at] = delta;
  }
  floatx16 dq[NDT];
  bool check = false;
  int left;
  auto tile = [&](int kt, const char* Kt, const char* Vt) {
    const int k0 = kt * KT;
    int ln = lane;
    pin(ln);
    floatx16 ds[NSUB];
    const bool cut = k0 + KT - 1 > t_first;
#pragma unroll
    for (int x = 0; x < NSUB; ++x) {
      floatx16 s = zeros16(), dp = zeros16();
      typedef Frags<typename Elem<T>::Frag, 2> F2;
      one_ahead<NKS>([&](int ks) { return F2{{L::rows32(Kt, 32 * x, ks, ln), L::rows32(Vt, 32 * x, ks, ln)}}; },
                     [&](int ks, const F2& f) {
                       s = Elem<T>::mma32(f.f[0], qf[ks], s);
                       dp = Elem<T>::mma32(f.f[1], dof[ks], dp);
                     });
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[x][i] = fast_exp2(fmaf(s[i], sl2, -lse2)) * (dp[i] - delta);
      if (cut) {
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[x][i] = k0 + 32 * x + row32(i, g) > t ? 0.f : ds[x][i];
      }
    }
    if (check && cut && kt < left && tile_not_finite<T, DP, KT>(Kt, lane)) left = kt;
    if (kt < left) add_cols<T, DP>(Kt, ds, dq, ln);
  };
  auto step = [&](int kt, char* Kt, char* Vt, char* Kn, char* Vn) {
    if constexpr (VEC) wait_vmem();
    __syncthreads();
    if (kt + 1 < n_kt) stage_kv(kt + 1, Kn, Vn);
    if (kt < n_w) tile(kt, Kt, Vt);
  };
  for (;;) {
    left = n_w;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) dq[dt] = zeros16();
    for (int kt = 0; kt < n_kt; kt += 2) {
      step(kt, K0, V0, K1, V1);
      if (kt + 1 < n_kt) step(kt + 1, K1, V1, K0, V0);
    }
    if (check || !any_bad(r < rows && not_finite(dq), flags, wave, lane)) break;
    check = true;
    stage_kv(0, K0, V0);
  }
  if (check) {
    __syncthreads();
    T* w = reinterpret_cast<T*>(wave & 2 ? K1 : K0) + (wave & 1) * 1024;
    for (int k0 = left * KT; k0 < n_w * KT; k0 += 32) {
      const int64_t key = min(k0 + (lane & 31), pl.len - 1);
      floatx16 s = scores_of<T, NKS, VEC>(Kb + key * a.k_st, Qr, g, D);
      const floatx16 dp = scores_of<T, NKS, VEC>(Vb + key * a.v_st, DO + o_at, g, D);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = fast_exp2(fmaf(s[i], sl2, -lse2)) * (dp[i] - delta);
      add_rows<T>(
          s, dq, w, lane, D, [&](int x) { return Kb + (int64_t)min(k0 + x, pl.len - 1) * a.k_st; },
          [&](int x) { return k0 + x <= t; });
    }
  }
  if (r < rows)
    store_row<T, NDT, VEC>(DQ + (int64_t)(pl.start + t) * a.q_st + (int64_t)h * a.q_sh, D, g, dq, scale);
}

// Key-stationary: dK and dV of 32 KG keys, over the rows of the group that come
// after them: KG waves of 32 keys each, times 4 / KG that take every other 32 rows
// and are added up at the end (KG = 2: where blocks of 128 keys are too few for the
// CUs).
template <class T, int NKS, int NDT, int KG, bool VEC>
__global__ __launch_bounds__(256, waves_per_simd(sizeof(T), NDT)) void packed_dkv_kernel(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, const T* __restrict__ DO,
    const float* __restrict__ LSE2, const float* __restrict__ DELTA, T* __restrict__ DK, T* __restrict__ DV,
    PackedArgs a, float sl2, float scale) {
  static_assert(KG == 4 || KG == 2, "one or two row groups");
  constexpr int DP = 32 * NDT, NT = 256, BN = 32 * KG, RG = 4 / KG, QT = 32 * RG;
  using L = LdsTile<T, DP>;
  using St = Stage<T, DP, QT, NT>;
  using StV = Stage<T, DP, BN, NT>;
  constexpr int BYTES = QT * L::kRow;
  __shared__ __align__(16) char Q0[BYTES], Q1[BYTES], D0[BYTES], D1[BYTES];
  __shared__ __align__(16) float S0[2 * QT], S1[2 * QT];  // a tile's lse log2(e), then its Delta
  __shared__ __align__(16) char VS[BN * L::kRow];  // V of the block's keys: in registers it would not fit beside K, dK, dV
  __shared__ int flags[4];

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, G = a.G, D = a.D;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave % KG, rg = wave / KG;
  const int hk = blockIdx.x % a.HK;
  const Place pl = find_place<true>(a.cu, a.n_seq, a.total, 1, BN, a.slots, (int)(blockIdx.x / a.HK), lane);
  if (pl.tile < 0) return;
  const int rows = pl.len * G, key0 = pl.tile * BN + kg * 32;
  const int key = key0 + (lane & 31), kc = min(key, pl.len - 1);
  const int first = key * G;  // the first row that comes at or after the key
  const T* Qb = Q + (int64_t)pl.start * a.q_st + (int64_t)hk * G * a.q_sh;
  const T* Db = DO + (int64_t)pl.start * a.o_st + (int64_t)hk * G * a.o_sh;
  const T* Vb = V + (int64_t)pl.start * a.v_st + (int64_t)hk * a.v_sh;
  const int64_t stat0 = (int64_t)hk * G * a.total + pl.start;
  // position and head of row rr of a tile (G <= 128: a 16-bit reciprocal is exact
  // below 512); rows behind the last one repeat it
  const int magic = 65535 / G + 1;
  auto stage_q = [&](int rt, char* Qd, char* Dd, float* Sd) {
    const int t0 = rt * QT / G, g0 = rt * QT % G, end = rows - 1 - rt * QT;
    auto place = [&](int rr, int& t, int& gq) {
      const int x = min(rr, end) + g0;
      t = (x * magic) >> 16;
      gq = x - t * G;
    };
    const T *q = Qb + (int64_t)t0 * a.q_st, *d = Db + (int64_t)t0 * a.o_st;
#pragma unroll
    for (int p = 0; p < St::PER; ++p) {
      int t, gq;
      place(St::row(p, tid), t, gq);
      if constexpr (VEC) {
        const int c = St::quad(p, tid);
        St::dma(buffer_rsrc(q, 0x7fffffffu), St::at((int)(t * a.q_st + gq * a.q_sh), c, D), Qd, p, tid);
        St::dma(buffer_rsrc(d, 0x7fffffffu), St::at((int)(t * a.o_st + gq * a.o_sh), c, D), Dd, p, tid);
      } else {
        St::copy(q + t * a.q_st + gq * a.q_sh, Qd, p, tid, D);
        St::copy(d + t * a.o_st + gq * a.o_sh, Dd, p, tid, D);
      }
    }
    if (wave < RG) {  // 64 of the 2 QT statistics to a wave
      int t, gq;
      place((wave * 64 + lane) % QT, t, gq);
      const int64_t at = stat0 + (int64_t)gq * a.total + t0 + t;
      dma_dword((wave * 64 + lane < QT ? LSE2 : DELTA) + at, Sd + wave * 64);
    }
  };
  const int rt0 = pl.tile * BN * G / QT, n_rt = (rows + QT - 1) / QT;
  // sub-tiles of 32 rows: the first with a row after some key of the wave
  const int sub0 = key0 < pl.len ? key0 * G / 32 : 0x7fffffff;
  {
    typename StV::Lanes vl;
    StV::template lanes<VEC>(vl, a.v_st, D, tid);
    StV::template head<VEC>(vl, Vb, pl.tile * BN, pl.len, a.v_st, D, VS, tid);
  }
  stage_q(rt0, Q0, D0, S0);
  const char* Vw = VS + kg * 32 * L::kRow;

  typename Elem<T>::Frag kf[NKS];
  const T* Kr = K + (int64_t)(pl.start + kc) * a.k_st + (int64_t)hk * a.k_sh;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) kf[ks] = row_frag<T, VEC>(Kr, ks, g, D);
  floatx16 dk[NDT], dv[NDT];
  bool check = false;
  int left;  // the first cut sub-tile left to the end
  // the mask (or the sequence's end) cuts through sub-tile x
  auto is_cut = [&](int x) { return x * 32 < (key0 + 31) * G || x * 32 + 32 > rows; };
  auto tile = [&](int rt, const char* Qt, const char* Dt, const float* St_) {
    const int x = rt * RG + rg, r0 = x * 32;
    int ln = lane;
    pin(ln);
    floatx16 p[1], ds[1];
    floatx16 s = zeros16(), dp = zeros16();
    one_ahead<NKS>([&](int ks) { return L::rows32(Qt, 0, ks, ln); },
                   [&](int ks, const typename Elem<T>::Frag& f) { s = Elem<T>::mma32(f, kf[ks], s); });
    typedef Frags<typename Elem<T>::Frag, 2> F2;
    one_ahead<NKS>([&](int ks) { return F2{{L::rows32(Dt, 0, ks, ln), L::rows32(Vw, 0, ks, ln)}}; },
                   [&](int ks, const F2& f) { dp = Elem<T>::mma32(f.f[0], f.f[1], dp); });
    const bool cut = is_cut(x);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const floatx4 lse2 = *reinterpret_cast<const floatx4*>(St_ + 8 * u + 4 * g);
      const floatx4 delta = *reinterpret_cast<const floatx4*>(St_ + QT + 8 * u + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * u + e;
        p[0][i] = fast_exp2(fmaf(s[i], sl2, -lse2[e]));
        ds[0][i] = p[0][i] * (dp[i] - delta[e]);
      }
    }
    if (cut) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int row = r0 + row32(i, g);
        const bool in = row >= first && row < rows;
        p[0][i] = in ? p[0][i] : 0.f;
        ds[0][i] = in ? ds[0][i] : 0.f;
      }
    }
    if (check && cut && x < left && (tile_not_finite<T, DP, 32>(Qt, lane) || tile_not_finite<T, DP, 32>(Dt, lane)))
      left = x;
    if (!cut || x < left) {
      add_cols<T, DP>(Dt, p, dv, ln);
      add_cols<T, DP>(Qt, ds, dk, ln);
    }
  };
  auto step = [&](int rt, char* Qt, char* Dt, float* St_, char* Qn, char* Dn, float* Sn) {
    wait_vmem();
    __syncthreads();
    if (rt + 1 < n_rt) stage_q(rt + 1, Qn, Dn, Sn);
    const int x = rt * RG + rg;
    if (x >= sub0 && x * 32 < rows)
      tile(rt, Qt + rg * 32 * L::kRow, Dt + rg * 32 * L::kRow, St_ + rg * 32);
  };
  for (;;) {
    left = 0x7fffffff;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) dk[dt] = zeros16(), dv[dt] = zeros16();
    for (int rt = rt0; rt < n_rt; rt += 2) {
      step(rt, Q0, D0, S0, Q1, D1, S1);
      if (rt + 1 < n_rt) step(rt + 1, Q1, D1, S1, Q0, D0, S0);
    }
    if (check || !any_bad(key < pl.len && (not_finite(dk) || not_finite(dv)), flags, wave, lane)) break;
    check = true;
    stage_q(rt0, Q0, D0, S0);
  }
  __syncthreads();  // the tiles' LDS is free
  if (check && left != 0x7fffffff) {
    T* w = reinterpret_cast<T*>(wave & 2 ? Q1 : Q0) + (wave & 1) * 1024;
    const T* Vr = Vb + (int64_t)kc * a.v_st;
    for (int x = left; x * 32 < rows; x += RG) {
      if (!is_cut(x)) continue;
      const int r0 = x * 32;
      auto q_row = [&](int y) {
        const int r = min(r0 + y, rows - 1);
        return Qb + (int64_t)(r / G) * a.q_st + (int64_t)(r % G) * a.q_sh;
      };
      auto do_row = [&](int y) {
        const int r = min(r0 + y, rows - 1);
        return Db + (int64_t)(r / G) * a.o_st + (int64_t)(r % G) * a.o_sh;
      };
      auto mine = [&](int y) { return r0 + y >= first && r0 + y < rows; };
      floatx16 p = scores_of<T, NKS, VEC>(q_row(lane & 31), Kr, g, D);
      floatx16 ds = scores_of<T, NKS, VEC>(do_row(lane & 31), Vr, g, D);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = min(r0 + row32(i, g), rows - 1);
        const int64_t at = stat0 + (int64_t)(r % G) * a.total + r / G;
        p[i] = fast_exp2(fmaf(p[i], sl2, -LSE2[at]));
        ds[i] = p[i] * (ds[i] - DELTA[at]);
      }
      add_rows<T>(p, dv, w, lane, D, do_row, mine);
      add_rows<T>(ds, dk, w, lane, D, q_row, mine);
    }
  }
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
  if (key < pl.len) {
    store_row<T, NDT, VEC>(DK + (int64_t)(pl.start + key) * a.k_st + (int64_t)hk * a.k_sh, D, g, dk, scale);
    store_row<T, NDT, VEC>(DV + (int64_t)(pl.start + key) * a.v_st + (int64_t)hk * a.v_sh, D, g, dv, 1.f);
  }
}

// ---------------------------------------------------------------- launches
namespace {

template <class T, int NKS, int NDT, bool VEC>
hipError_t fwd_t(const void* q, const void* k, const void* v, void* o, float* lse, PackedArgs a, float scale,
                 hipStream_t stream) {
  a.slots = packed_slots(a, 128, a.G);
  TimingScope ts("packed_fwd", stream);
  hipLaunchKernelGGL((packed_fwd_kernel<T, NKS, NDT, VEC>), dim3((unsigned)a.slots * a.HK), dim3(256), 0, stream,
                     static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                     static_cast<T*>(o), lse, a, (float)((double)scale * 1.4426950408889634));
  return hipGetLastError();
}

template <class T, int NKS, int NDT, bool VEC>
hipError_t bwd_t(const void* q, const void* k, const void* v, const void* o, const void* d_o, const float* lse,
                 void* dq, void* dk, void* dv, float* ws, PackedArgs a, float scale, hipStream_t stream) {
  const float sl2 = (float)((double)scale * 1.4426950408889634);
  float *lse2 = ws, *delta = ws + (int64_t)a.total * a.HK * a.G;
  {
    TimingScope ts("packed_bwd_dq", stream);
    a.slots = packed_slots(a, 128, a.G);
    hipLaunchKernelGGL((packed_dq_kernel<T, NKS, NDT, VEC>), dim3((unsigned)a.slots * a.HK), dim3(256), 0, stream,
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
  // blocks of 64 keys where 128 would leave CUs without a second block (16-bit rows
  // of up to 64), or without one (they fill a CU alone)
  if constexpr (sizeof(T) * NDT <= 8) {
    if ((int64_t)a.total * a.HK < (sizeof(T) * NDT <= 4 ? 512 : 128) * 128) {
      launch(packed_dkv_kernel<T, NKS, NDT, 2, VEC>, 64);
      return hipGetLastError();
    }
  }
  launch(packed_dkv_kernel<T, NKS, NDT, 4, VEC>, 128);
  return hipGetLastError();
}

// NKS: steps of 16 over the head dim, NDT: 32-wide tiles of it
#define WHA_BY_DIM(F, T, D, vec, ...)                       \
  (D) <= 64 ? ((vec) ? F<T, 4, 2, true>(__VA_ARGS__) : F<T, 4, 2, false>(__VA_ARGS__)) \
            : ((vec) ? F<T, 8, 4, true>(__VA_ARGS__) : F<T, 8, 4, false>(__VA_ARGS__))

}  // namespace

hipError_t launch_packed_fwd(int dtype, const void* q, const void* k, const void* v, void* o, float* lse,
                             const PackedArgs& a, bool vec, float scale, hipStream_t stream) {
  if (dtype == kF32) return WHA_BY_DIM(fwd_t, float, a.D, vec, q, k, v, o, lse, a, scale, stream);
  if (dtype == kBf16) return WHA_BY_DIM(fwd_t, __bf16, a.D, vec, q, k, v, o, lse, a, scale, stream);
  return WHA_BY_DIM(fwd_t, _Float16, a.D, vec, q, k, v, o, lse, a, scale, stream);
}

hipError_t launch_packed_bwd(int dtype, const void* q, const void* k, const void* v, const void* o, const void* d_o,
                             const float* lse, void* dq, void* dk, void* dv, float* ws, const PackedArgs& a, bool vec,
                             float scale, hipStream_t stream) {
  if (dtype == kF32)
    return WHA_BY_DIM(bwd_t, float, a.D, vec, q, k, v, o, d_o, lse, dq, dk, dv, ws, a, scale, stream);
  return WHA_BY_DIM(bwd_t, __bf16, a.D, vec, q, k, v, o, d_o, lse, dq, dk, dv, ws, a, scale, stream);
}

}  // namespace wha
