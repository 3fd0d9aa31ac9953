// Element types of the packed and paged operators -- float, bf16 and fp16 --
// behind one set of MFMA fragments and LDS tiles (gfx950 only).
//
// A fragment holds 8 consecutive k of one row or column; lane group g takes k =
// 8g .. 8g + 7 of every step.  16-bit types: one MFMA a step, all products exact
// in its fp32 accumulator.  float: the same 8 numbers go through 8 fp32 MFMAs,
// number j of every lane group in MFMA j (k can be mapped to any index as long
// as both operands agree), so one kernel serves all three types.
//
//   32 x 32 results, k steps of 16, g = lane / 32 (v_mfma_f32_32x32x16_bf16/_f16,
//   v_mfma_f32_32x32x2_f32): lane l supplies row (or column) l % 32 and holds
//   D[acc_row(i, g)][l % 32], acc_row(i, g) = 8 (i / 4) + 4 g + i % 4, i = 0..15
//   16 x 16 results, k steps of 32, g = lane / 16 (v_mfma_f32_16x16x32_bf16/_f16,
//   v_mfma_f32_16x16x4_f32): row (or column) l % 16, D[4 g + i][l % 16], i = 0..3
#pragma once
#include <type_traits>

#include "wha_device.hpp"

namespace wha {

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

template <class T>
struct Elem;

template <>
struct Elem<float> {
  typedef floatx8 Frag;
  static constexpr int kQuad = 4;  // elements in 16 bytes
  __device__ __forceinline__ static floatx16 mma32(Frag a, Frag b, floatx16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static floatx4 mma16(Frag a, Frag b, floatx4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static Frag pack(const float (&x)[8]) {
    Frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = x[j];
    return f;
  }
  __device__ __forceinline__ static void store4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
  }
};

template <>
struct Elem<__bf16> {
  typedef bf16x8 Frag;
  static constexpr int kQuad = 8;
  __device__ __forceinline__ static floatx16 mma32(Frag a, Frag b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static floatx4 mma16(Frag a, Frag b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static unsigned pair(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2{a, b}), bf16x2));
  }
  __device__ __forceinline__ static Frag pack(const float (&x)[8]) {
    return __builtin_bit_cast(Frag, (uintx4{pair(x[0], x[1]), pair(x[2], x[3]), pair(x[4], x[5]), pair(x[6], x[7])}));
  }
  __device__ __forceinline__ static void store4(__bf16* p, float a, float b, float c, float d) {
    *reinterpret_cast<uintx2*>(p) = uintx2{pair(a, b), pair(c, d)};
  }
};

template <>
struct Elem<_Float16> {
  typedef f16x8 Frag;
  static constexpr int kQuad = 8;
  __device__ __forceinline__ static floatx16 mma32(Frag a, Frag b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static floatx4 mma16(Frag a, Frag b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static unsigned pair(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2{a, b}), f16x2));
  }
  __device__ __forceinline__ static Frag pack(const float (&x)[8]) {
    return __builtin_bit_cast(Frag, (uintx4{pair(x[0], x[1]), pair(x[2], x[3]), pair(x[4], x[5]), pair(x[6], x[7])}));
  }
  __device__ __forceinline__ static void store4(_Float16* p, float a, float b, float c, float d) {
    *reinterpret_cast<uintx2*>(p) = uintx2{pair(a, b), pair(c, d)};
  }
};

// The products of the packed operators.  16-bit types: as they are.  float: on the
// bf16 matrix cores at fp32 precision, each number as three bf16 parts, x = h + m +
// l, of whose nine products the six that reach fp32 precision are summed (Henry,
// Tang and Heinecke, "Leveraging the bfloat16 artificial intelligence datatype for
// higher-precision computations", 2019): 192 cycles for what takes the fp32 MFMA
// 512.  The small products go to an accumulator of their own, added once at the
// end: a small product added to a large sum would lose its low bits each time.  The
// parts of an infinity hold NaN, so results that are not finite are formed again
// in Elem's arithmetic.
template <class T>
struct Fast {
  typedef typename Elem<T>::Frag Frag;
  struct Sum {
    floatx16 big;
    __device__ __forceinline__ Sum() { zero(); }
    __device__ __forceinline__ void zero() {
#pragma unroll
      for (int i = 0; i < 16; ++i) big[i] = 0.f;
    }
    __device__ __forceinline__ void add(const Frag& a, const Frag& b) { big = Elem<T>::mma32(a, b, big); }
    __device__ __forceinline__ floatx16 value() const { return big; }
  };
  __device__ __forceinline__ static Frag pack(const float (&x)[8]) { return Elem<T>::pack(x); }
};
struct Frag3 {
  bf16x8 h, m, l;
};
template <>
struct Fast<float> {
  typedef Frag3 Frag;
  typedef Elem<__bf16> B;
  struct Sum {
    floatx16 big, small;
    __device__ __forceinline__ Sum() {
#pragma unroll
      for (int i = 0; i < 16; ++i) big[i] = small[i] = 0.f;
    }
    __device__ __forceinline__ void add(const Frag& a, const Frag& b) {
      small = B::mma32(a.l, b.h, small);
      small = B::mma32(a.h, b.l, small);
      small = B::mma32(a.m, b.m, small);
      small = B::mma32(a.m, b.h, small);
      small = B::mma32(a.h, b.m, small);
      big = B::mma32(a.h, b.h, big);
    }
    __device__ __forceinline__ floatx16 value() const {
      floatx16 x;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = big[i] + small[i];
      return x;
    }
  };
  // a pair rounded to bf16 (first in the low half), leaving what remains of it
  __device__ __forceinline__ static unsigned take(float& a, float& b) {
    const unsigned h = B::pair(a, b);
    a -= __uint_as_float(h << 16);
    b -= __uint_as_float(h & 0xffff0000u);
    return h;
  }
  __device__ __forceinline__ static Frag pack(const float (&x)[8]) {
    uintx4 h, m, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a = x[2 * i], b = x[2 * i + 1];
      h[i] = take(a, b);
      m[i] = take(a, b);
      l[i] = B::pair(a, b);
    }
    return Frag{__builtin_bit_cast(bf16x8, h), __builtin_bit_cast(bf16x8, m), __builtin_bit_cast(bf16x8, l)};
  }
};

// Keeps what is formed from x where it stands in program order (an empty
// statement that x passes through).  The addresses that a tile's reads are made
// from are formed again for every tile, from a pinned lane: held in registers
// over the loop they cost the 128-wide kernels more than a wave has.
template <class T>
__device__ __forceinline__ void pin(T& x) {
  asm volatile("" : "+v"(x));
}
__device__ __forceinline__ floatx16 zeros16() {
  floatx16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}
// Row within a 32 x 32 result of element i of lane group g.
__device__ __forceinline__ int row32(int i, int g) { return 8 * (i >> 2) + 4 * g + (i & 3); }

// A tile of rows of DP elements in LDS, read both as the rows operand of
// contractions over d (8 consecutive d of one row per lane) and as the columns
// operand of contractions over the tile's rows (8 rows of one d per lane).  16-bit
// types read the columns with ds_read_b64_tr_b16: the 16 lanes of a group name
// four rows of 16 d in 8-byte pieces (lane i: row i / 4, d = 4 (i % 4) ..), and
// lane n gets the four rows of column n; float reads them one by one.
//
// Quads (16 bytes) of a row are permuted by XOR with swz(row): rows of 16 lanes
// distinct mod 16 (the rows operand) then meet 16 different quads of the 256
// bytes that the LDS serves together, and so do the four rows x 64 bytes of
// which a transposing read's half wave asks, and the two rows x 128 bytes of 32
// single ones.
template <class T, int DP>
struct LdsTile {
  static constexpr int kRow = DP * (int)sizeof(T);  // bytes
  static constexpr int kQuads = kRow / 16;
  static_assert(kQuads == 8 || kQuads == 16 || kQuads == 32, "rows of 128, 256 or 512 bytes");

  __device__ __forceinline__ static int swz(int r) {
    if constexpr (sizeof(T) == 4) return (((r >> 2) & 1) << 3) | (((r >> 3) & 1) << 2) | (r & 3);
    else if constexpr (kQuads == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
  }
  // byte offset of quad c of row r (rows 16 apart are 16 kRow apart)
  __device__ __forceinline__ static int at(int r, int c) { return (r * kRow + (swz(r) << 4)) ^ (c << 4); }

  // d = 16 ks + 8 (lane / 32) .. + 7 of row r0 + lane % 32, r0 a multiple of 16
  __device__ __forceinline__ static typename Elem<T>::Frag rows32(const char* t, int r0, int ks, int lane) {
    return rows(t + r0 * kRow, lane & 31, 2 * ks + (lane >> 5));
  }
  // elements 8 c .. 8 c + 7 of row r
  __device__ __forceinline__ static typename Elem<T>::Frag rows(const char* t, int r, int c) {
    if constexpr (sizeof(T) == 4) {
      const floatx4 a = *reinterpret_cast<const floatx4*>(t + at(r, 2 * c));
      const floatx4 b = *reinterpret_cast<const floatx4*>(t + at(r, 2 * c + 1));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return *reinterpret_cast<const typename Elem<T>::Frag*>(t + at(r, c));
    }
  }
  // four rows r .. r + 3 of column d0 + (lane & 15), 16-bit types; all 16 lanes
  // of a group pass the same r and d0 (multiples of 4 and 16)
  __device__ __forceinline__ static shortx4 tr4(const char* t, int r, int d0, int lane) {
    const int i = lane & 15, row = r + (i >> 2), d = d0 + 4 * (i & 3);
    const char* p = t + at(row, d >> 3) + 2 * (d & 7);
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (shortx4 __attribute__((address_space(3)))*)(p));
  }
  // rows 16 ks + row32(j, g), j = 0..7, of column 32 dt + lane % 32
  __device__ __forceinline__ static typename Elem<T>::Frag cols32(const char* t, int ks, int dt, int lane) {
    const int g = lane >> 5;
    if constexpr (sizeof(T) == 4) {
      typename Elem<T>::Frag f;
      const int d = 32 * dt + (lane & 31);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = *reinterpret_cast<const float*>(t + 16 * ks * kRow + at(row32(j, g), d >> 2) + 4 * (d & 3));
      }
      return f;
    } else {
      const int d0 = 32 * dt + 16 * ((lane >> 4) & 1);
      const char* t0 = t + 16 * ks * kRow;
      const shortx4 a = tr4(t0, 4 * g, d0, lane), b = tr4(t0, 8 + 4 * g, d0, lane);
      return __builtin_bit_cast(typename Elem<T>::Frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
  // rows 4 g + j (j < 4) and 16 + 4 g + j - 4 of column 16 dt + lane % 16, g = lane
  // / 16: the order in which a lane holds two 16 x 16 results, one above the other
  __device__ __forceinline__ static typename Elem<T>::Frag cols16(const char* t, int dt, int lane) {
    const int g = lane >> 4;
    if constexpr (sizeof(T) == 4) {
      typename Elem<T>::Frag f;
      const int d = 16 * dt + (lane & 15);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = 16 * (j >> 2) + 4 * g + (j & 3);
        f[j] = *reinterpret_cast<const float*>(t + at(r, d >> 2) + 4 * (d & 3));
      }
      return f;
    } else {
      const shortx4 a = tr4(t, 4 * g, 16 * dt, lane), b = tr4(t + 16 * kRow, 4 * g, 16 * dt, lane);
      return __builtin_bit_cast(typename Elem<T>::Frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
  // elements 8 c .. 8 c + 7 of row r
  __device__ __forceinline__ static void put(char* t, int r, int c, typename Elem<T>::Frag x) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<floatx4*>(t + at(r, 2 * c)) = __builtin_shufflevector(x, x, 0, 1, 2, 3);
      *reinterpret_cast<floatx4*>(t + at(r, 2 * c + 1)) = __builtin_shufflevector(x, x, 4, 5, 6, 7);
    } else {
      *reinterpret_cast<typename Elem<T>::Frag*>(t + at(r, c)) = x;
    }
  }
};

// A tile of ROWS fp32 rows in its three bf16 parts, each a tile of its own.
template <int DP, int ROWS>
struct SplitTile {
  typedef LdsTile<__bf16, DP> Part;
  static constexpr int kPart = ROWS * Part::kRow, kRow = 3 * Part::kRow;
  __device__ __forceinline__ static Frag3 rows32(const char* t, int r0, int ks, int lane) {
    return Frag3{Part::rows32(t, r0, ks, lane), Part::rows32(t + kPart, r0, ks, lane),
                 Part::rows32(t + 2 * kPart, r0, ks, lane)};
  }
  __device__ __forceinline__ static Frag3 cols32(const char* t, int ks, int dt, int lane) {
    return Frag3{Part::cols32(t, ks, dt, lane), Part::cols32(t + kPart, ks, dt, lane),
                 Part::cols32(t + 2 * kPart, ks, dt, lane)};
  }
  // elements 4 q .. 4 q + 3 of row r
  __device__ __forceinline__ static void put4(char* t, int r, int q, floatx4 x) {
    uintx2 h, m, l;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float a = x[2 * i], b = x[2 * i + 1];
      h[i] = Fast<float>::take(a, b);
      m[i] = Fast<float>::take(a, b);
      l[i] = Elem<__bf16>::pair(a, b);
    }
    char* p = t + Part::at(r, q >> 1) + 8 * (q & 1);
    *reinterpret_cast<uintx2*>(p) = h;
    *reinterpret_cast<uintx2*>(p + kPart) = m;
    *reinterpret_cast<uintx2*>(p + 2 * kPart) = l;
  }
};

}  // namespace wha
