// Host-side launch interface of the packed and paged operators
// (attn_packed.hip, attn_paged.hip).  Launchers validate nothing (wha_api.hip does).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "wha_launch.hpp"

namespace wha {

// Element types (WHA_F32 ..).
enum : int { kF32 = 0, kBf16 = 1, kF16 = 2, kI8 = 3 };
inline size_t elem_size(int dtype) { return dtype == kF32 ? 4 : dtype == kI8 ? 1 : 2; }

// Packed sequences: rows [total][heads][D], strides in elements.
struct PackedArgs {
  const int* cu;  // [n_seq + 1], device
  int n_seq, total, HK, G, D;
  int slots;  // set by the launchers
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;
};
// Slots of tiles of BM rows, G rows to a position: an upper bound of the tiles.
inline int64_t packed_slots64(int64_t total, int n_seq, int BM, int G) { return total * G / BM + n_seq; }
inline int packed_slots(const PackedArgs& a, int BM, int G) { return (int)packed_slots64(a.total, a.n_seq, BM, G); }

// align: 16 or 4 where every row of every tensor is (and D elements are) a multiple
// of so many bytes, else 2.
hipError_t launch_packed_fwd(int dtype, const void* q, const void* k, const void* v, void* o, float* lse,
                             const PackedArgs& a, int align, float scale, hipStream_t stream);
// ws: 2 * total * n_head floats.
hipError_t launch_packed_bwd(int dtype, const void* q, const void* k, const void* v, const void* o, const void* d_o,
                             const float* lse, void* dq, void* dk, void* dv, float* ws, const PackedArgs& a, int align,
                             float scale, hipStream_t stream);

// Paged cache: [n_pages][HK][P][D] elements of `cache_dtype` in k and v, P = 1 <<
// shift; int8 rows with a scale each in [n_pages][HK][P] floats.
struct PagedCache {
  void *k, *v;
  float *ks, *vs;  // int8 only
  int64_t n_pages;
  int HK, D, shift;
};
// Rows of k and v of `dtype`, [N][HK][D] with these strides, to or from `slots`.
struct PagedRows {
  int64_t N, k_st, k_sh, v_st, v_sh;
  const int64_t* slots;
};
hipError_t launch_paged_kv_write(int dtype, int cache_dtype, const void* k, const void* v, const PagedRows& r,
                                 const PagedCache& c, bool vec, hipStream_t stream);
hipError_t launch_paged_kv_read(int dtype, int cache_dtype, void* k, void* v, const PagedRows& r, const PagedCache& c,
                                bool vec, hipStream_t stream);

struct PagedDecode {
  const int* table;  // [n_seq][table_stride], device; pages of a sequence
  const int* lens;   // [n_seq], device
  int64_t table_stride;
  int n_seq, n_head, max_pages;
  int64_t q_sb, q_sh, o_sb, o_sh;
};
// Splits of a sequence's keys: by the number of (sequence, key-value head) pairs
// and the table's capacity alone, so that a captured call serves any lengths.
int paged_splits(int64_t n_seq, int n_head, int HK, int64_t capacity);
size_t paged_decode_floats(int64_t n_seq, int n_head, int HK, int D, int64_t capacity);
hipError_t launch_paged_decode(int dtype, int cache_dtype, const void* q, void* o, float* lse, float* ws,
                               const PagedDecode& d, const PagedCache& c, bool vec, float scale, hipStream_t stream);

}  // namespace wha
