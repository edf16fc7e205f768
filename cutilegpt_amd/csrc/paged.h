// Addressing shared by the kernels of the paged key-value cache.
#pragma once

#include "common.h"

namespace cgpt {

// Exact n / d for 0 <= n < 2^31 by one multiply and a shift: with s = ceil(log2 d)
// and m = ceil(2^(31+s) / d) < 2^32, m d - 2^(31+s) < d <= 2^s, so the error
// n (m d - 2^(31+s)) / (d 2^(31+s)) stays below 1/d and never reaches the next
// quotient.
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(int64_t v = 1) {
    d = static_cast<uint32_t>(v);
    s = 0;
    while ((uint64_t{1} << s) < d) ++s;
    m = static_cast<uint32_t>(((uint64_t{1} << (31 + s)) + d - 1) / d);
    s += 31;
  }
  __device__ __forceinline__ int div(int n) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * m) >> s);
  }
};

// One pool of pages: element (page, head, slot, d) at base + page * sp + head * sh
// + slot * ss + d.
struct PagePool {
  void* base;
  int64_t sp, sh, ss;
};

// The sequences of a step.  Sequence b holds lens[b] keys, its last tokens being
// the step's: tokens cu[b] .. cu[b+1]-1 of the packed rows (cu NULL: token b).
// Key t lives in slot t % page of page table[b * stride + t / page].
struct PagedBatch {
  const int* table;
  const int* lens;
  const int* cu;
  int64_t stride;
  int n_tokens, B, n_pages, cols;
  int cap;  // keys a table row can name
  FastDiv page;
};

struct PagedAttnArgs {
  const void* q;
  void* o;
  PagePool kc, vc;
  PagedBatch seq;
  const int* prefix;  // pages of the shared prefix
  int prefix_len, prefix_cols;
  int64_t q_st, q_sh, o_st, o_sh;
  int Hq, Hkv;
  FastDiv group;  // query heads a key head
  float scale_log2;
  int* err;
};

// Attention of the query tiles of long steps (paged_tile.hip), 16-bit types of head_dim
// 64 and 128.  flat: rows are all packed tokens, keys the shared prefix; else rows are a
// sequence's and keys all of its own, those below prefix_len read from the prefix's
// pages.  qt: 16-row sub-tiles of a wave (1 or 2; 4 waves).  n_split > 1 or flat: every
// split leaves (m, l, O) of each (token, head) row in part_ml / part_o, else o is written.
bool paged_tile_ok(int dtype, int head_dim);
int launch_paged_tile(int dtype, int head_dim, const PagedAttnArgs& a, bool flat, int qt, int n_split,
                      float* part_ml, float* part_o, hipStream_t s);

// The checks that the entry points share.
inline int check_paged(int64_t n_tokens, int64_t B, int64_t Hq, int64_t Hkv, int64_t head_dim,
                       int64_t page_size, int64_t n_pages, int64_t cols, int64_t stride,
                       const PagePool& k, const PagePool& v, int dtype) {
  if (n_tokens < 0 || B < 0 || Hq <= 0 || Hkv <= 0 || page_size <= 0 || n_pages <= 0 || cols < 0)
    return CGPT_EINVAL;
  if (Hq % Hkv != 0 || (cols > 0 && B > 1 && stride < 0)) return CGPT_EINVAL;
  if (dtype != CGPT_F32 && dtype != CGPT_BF16 && dtype != CGPT_F16) return CGPT_EDTYPE;
  if (head_dim != 16 && head_dim != 32 && head_dim != 64 && head_dim != 128) return CGPT_ESHAPE;
  if (n_tokens > 0x3fffffff || B > 0x3fffffff || Hq > 0x7fff || page_size > 0x3fffffff ||
      n_pages > 0x7fffffff || cols > 0x3fffffff || n_tokens * Hq > 0x7fffffff)
    return CGPT_ESHAPE;
  if (page_size * cols > 0x3fffffff) return CGPT_ESHAPE;
  const int64_t epv = dtype == CGPT_F32 ? 4 : 8;
  for (const PagePool* p : {&k, &v}) {
    if (p->base == nullptr || (reinterpret_cast<uintptr_t>(p->base) & 15)) return CGPT_EINVAL;
    // Rows are read and written as 16-byte vectors; no two may overlap.
    if (p->sp % epv != 0 || p->sh % epv != 0 || p->ss % epv != 0) return CGPT_EINVAL;
    if ((n_pages > 1 && p->sp < head_dim) || (Hkv > 1 && p->sh < head_dim) ||
        (page_size > 1 && p->ss < head_dim))
      return CGPT_EINVAL;
  }
  return CGPT_OK;
}

#if defined(__HIP_DEVICE_COMPILE__) || defined(__HIPCC__)

// Tokens of sequence b: [first, first + count) within the packed rows, whatever
// the device memory holds.
__device__ __forceinline__ void seq_tokens(const PagedBatch& s, int b, int* first, int* count) {
  if (s.cu == nullptr) {
    *first = b;
    *count = b < s.n_tokens ? 1 : 0;
    return;
  }
  const int f = max(s.cu[b], 0), e = min(s.cu[b + 1], s.n_tokens);
  *first = f;
  *count = max(e - f, 0);
}

// The sequence that packed token t belongs to, B when it lies behind the last.
__device__ __forceinline__ int seq_of(const PagedBatch& s, int t) {
  if (s.cu == nullptr) return min(t, s.B);
  int lo = 0, hi = s.B;  // the first b with cu[b + 1] > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (s.cu[mid + 1] > t)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// Page of key t of the table row, clamped into the pool; *bad when it was not.
__device__ __forceinline__ int page_of(const int* row, int col, int n_pages, bool* bad) {
  const int p = row[col];
  if (static_cast<uint32_t>(p) >= static_cast<uint32_t>(n_pages)) {
    *bad = true;
    return 0;
  }
  return p;
}

// Bit 31 (or, of a 16-bit type, 15) set where a value of the word is not finite: its
// exponent field, all ones, carries into the sign.
template <typename T> __device__ __forceinline__ uint32_t special_bits(uint32_t w) {
  if constexpr (sizeof(T) == 4) return ((w & 0x7f800000u) + 0x00800000u) & 0x80000000u;
  if constexpr (std::is_same<T, bf16_t>::value) return (w & 0x7f807f80u) + 0x00800080u;
  return (w & 0x7c007c00u) + 0x04000400u;
}
// The word with 0 in the place of values that are not finite.
template <typename T> __device__ __forceinline__ uint32_t finite_part(uint32_t w) {
  if constexpr (sizeof(T) == 4) return special_bits<T>(w) ? 0u : w;
  const uint32_t bits = special_bits<T>(w);
  return w & ~(((bits & 0x80000000u) ? 0xffff0000u : 0u) | ((bits & 0x8000u) ? 0xffffu : 0u));
}

// Half of a V^T operand: the 16-lane group's lane k points at 4 consecutive d of its
// row and receives the 4 keys of column 16 dt + k.
template <int KROW, int SWZ>
__device__ __forceinline__ u32x2_t vt_read(const uint8_t* sv, int row, int dt, int frow) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  const int byte = dt * 32 + 8 * (frow & 3);
  const uint8_t* p = sv + row * KROW + (((byte >> 4) ^ (row & SWZ)) << 4) + (byte & 15);
  const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4*)((__attribute__((address_space(3))) uint8_t*)(p)));
  return __builtin_bit_cast(u32x2_t, r);
}

#endif

}  // namespace cgpt
