// Addressing shared by the kernels of the paged key-value cache.
#pragma once

#include <algorithm>
#include <array>
#include <initializer_list>
#include <utility>

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
  int n_tokens, B, n_pages;
  int cap;  // keys a table row can name
  FastDiv page;
};

struct PagedAttnArgs {
  const void* q;
  void* o;
  PagePool kc, vc;
  PagedBatch seq;
  const int* prefix;  // pages of the shared prefix
  int prefix_len;
  int64_t q_st, q_sh, o_st, o_sh;
  int Hq, Hkv;
  FastDiv group;  // query heads a key head
  float scale_log2;
  int* err;
};

// What the tile kernel (paged_tile.hip; every type and head_dim) is to do: all packed rows
// against the shared prefix in flat_split parts of its keys (0: not at all), and every
// sequence's rows against its keys from `from` on, those below prefix_len read from the
// prefix's pages, in `split` parts (0: not at all).  With ml each part leaves (m, l, O) of its
// (token, head) rows there, the prefix's parts first; else the rows' results are written.  The
// other fields are launch_paged_tile's.
struct TileJob {
  float* ml;
  float* o;
  int flat_split, split, from;
  int flat_tiles, tiles, flat_blocks;
};
// qt: 16-row sub-tiles of each of a block's four waves, 1 or 2.
int launch_paged_tile(int64_t dtype, int head_dim, const PagedAttnArgs& a, const TileJob& job, int qt, hipStream_t s);

// Blocks of 256 threads that one launch holds, fewer than 2^32 threads.
constexpr int64_t kMaxBlocks = 0xffffff;

// Offsets within 16 consecutive slots of a page fit 32 bits.
inline bool short_rows(const PagedAttnArgs& a) { return a.kc.ss <= (1 << 25) && a.vc.ss <= (1 << 25); }

// Whether the rows of n values that these extents and strides place are apart: each stride
// reaches past all that the smaller ones place.
inline bool rows_apart(std::initializer_list<std::pair<int64_t, int64_t>> dims, int64_t n) {
  std::array<std::pair<int64_t, int64_t>, 3> by_stride;
  auto end = by_stride.begin();
  for (auto [extent, stride] : dims)
    if (extent > 1) *end++ = {stride, extent};
  std::sort(by_stride.begin(), end);
  __int128 span = n;
  for (auto d = by_stride.begin(); d != end; ++d) {
    if (d->first < span) return false;
    span += static_cast<__int128>(d->first) * (d->second - 1);
  }
  return true;
}

// The sizes that a plan goes by, small enough for its products to stay within 64 bits.
inline int check_sizes(const cgpt_paged_args& a) {
  if (a.n_tokens < 0 || a.B < 0 || a.Hq <= 0 || a.Hkv <= 0 || a.page_size <= 0 || a.max_pages < 0 || a.Hq % a.Hkv != 0)
    return CGPT_EINVAL;
  if (a.dtype != CGPT_F32 && a.dtype != CGPT_BF16 && a.dtype != CGPT_F16) return CGPT_EDTYPE;
  if (a.head_dim != 16 && a.head_dim != 32 && a.head_dim != 64 && a.head_dim != 128) return CGPT_ESHAPE;
  if (a.n_tokens > 0x3fffffff || a.B > 0x3fffffff || a.Hq > 0x7fff || a.page_size > 0x3fffffff ||
      a.max_pages > 0x3fffffff || a.n_tokens * a.Hq > 0x7fffffff || a.page_size * a.max_pages > 0x3fffffff)
    return CGPT_ESHAPE;
  return CGPT_OK;
}

// The checks that the entry points share: the sizes, then (with tokens to work on) the
// pointers.  CGPT_OK with *empty when there is nothing to launch.  `writes`: the pools are
// written too.
inline int check_paged(const cgpt_paged_args* p, bool writes, bool* empty) {
  if (p == nullptr) return CGPT_EINVAL;
  const cgpt_paged_args& a = *p;
  if (a.n_pages <= 0 || a.bt_stride < 0) return CGPT_EINVAL;
  const int rc = check_sizes(a);
  if (rc != CGPT_OK) return rc;
  if (a.n_pages > 0x7fffffff) return CGPT_ESHAPE;
  // Rows are read and written as 16-byte vectors; no two that are written may overlap.
  const int64_t epv = a.dtype == CGPT_F32 ? 4 : 8;
  const int64_t pools[2][3] = {{a.kc_sp, a.kc_sh, a.kc_ss}, {a.vc_sp, a.vc_sh, a.vc_ss}};
  const void* bases[2] = {a.k_cache, a.v_cache};
  for (int i = 0; i < 2; ++i) {
    const int64_t *s = pools[i], hd = a.head_dim;
    if (bases[i] == nullptr || (reinterpret_cast<uintptr_t>(bases[i]) & 15)) return CGPT_EINVAL;
    if (s[0] % epv != 0 || s[1] % epv != 0 || s[2] % epv != 0) return CGPT_EINVAL;
    if ((a.n_pages > 1 && s[0] < hd) || (a.Hkv > 1 && s[1] < hd) || (a.page_size > 1 && s[2] < hd)) return CGPT_EINVAL;
    if (writes && !rows_apart({{a.n_pages, s[0]}, {a.Hkv, s[1]}, {a.page_size, s[2]}}, hd)) return CGPT_EINVAL;
  }
  *empty = a.n_tokens == 0 || a.B == 0;
  if (*empty) return CGPT_OK;
  if (a.seq_lens == nullptr || (a.max_pages > 0 && a.block_table == nullptr)) return CGPT_EINVAL;
  if (a.cu_q == nullptr && a.n_tokens != a.B) return CGPT_EINVAL;
  for (int64_t st : {a.q_st, a.q_sh, a.k_st, a.k_sh, a.v_st, a.v_sh, a.out_st, a.out_sh})
    if (st < 0 || st % epv != 0) return CGPT_EINVAL;
  for (const void* r : {a.q, a.k, a.v, static_cast<const void*>(a.out)})
    if (reinterpret_cast<uintptr_t>(r) & 15) return CGPT_EINVAL;
  if (a.out != nullptr && !rows_apart({{a.n_tokens, a.out_st}, {a.Hq, a.out_sh}}, a.head_dim)) return CGPT_EINVAL;
  return CGPT_OK;
}

inline PagedBatch paged_batch(const cgpt_paged_args& a) {
  return PagedBatch{a.block_table, a.seq_lens, a.cu_q, a.bt_stride, static_cast<int>(a.n_tokens), static_cast<int>(a.B),
                    static_cast<int>(a.n_pages), static_cast<int>(a.page_size * a.max_pages), FastDiv(a.page_size)};
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

// The sequence that packed token t belongs to, B when it lies behind the last (a token in
// front of the first gets sequence 0, whose first token is behind it).
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

// How many of pred(0) .. pred(n - 1), true up to some index and false from there on, are
// true: 64 probes at a time, all lanes with the same answer.
template <typename F> __device__ __forceinline__ int wave_count(int n, int lane, F&& pred) {
  int lo = 0, hi = n;
  for (;;) {
    const int step = (hi - lo + 63) >> 6, i = lo + (lane + 1) * max(step, 1) - 1;
    const int k = __popcll(__builtin_amdgcn_ballot_w64(i < hi && pred(i)));
    lo += k * step;
    if (step <= 1) return lo;
    hi = min(hi, lo + step - 1);
  }
}

// seq_of for a token that the whole wave asks for.
__device__ __forceinline__ int wave_seq_of(const PagedBatch& s, int t, int lane) {
  if (s.cu == nullptr) return min(t, s.B);
  return wave_count(s.B, lane, [&](int b) { return s.cu[b + 1] <= t; });
}

// Row tiles of R rows over sequences of any numbers of tokens: sequence b has the slots
// from start(b) = cu[b] G / R + b on, at least as many as its rows fill.  The sequence
// of slot *slot, which becomes its tile within the sequence (possibly behind its rows);
// B when there is none.
template <int R>
__device__ __forceinline__ int slot_seq(const PagedBatch& s, int G, int lane, int* slot) {
  if (s.cu == nullptr && G <= R) {  // one tile each
    const int b = *slot;
    *slot = 0;
    return b;
  }
  auto start = [&](int b) { return (s.cu == nullptr ? b : min(max(s.cu[b], 0), s.n_tokens)) * G / R + b; };
  const int b = wave_count(s.B, lane, [&](int i) { return start(i + 1) <= *slot; });
  if (b < s.B) *slot -= start(b);
  return b;
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

// The largest weight of a row is made 2^kDrop at least and 2^(kDrop + 8) at most (the shift
// moves up only where it would pass that).  fp16 ends at 2^-24 below and 2^16 above: with
// weights of 1 and more, keys of 2^-25 and less are lost however many they are (2^17 beside
// one key in a block: 0.3 % of the result, five of its half steps).  2^7 further up, a key's
// weight is off by 2^-32 of the largest at most, below the result's half step up to 2^20 keys.
// The other types reach as far down as fp32 itself.
template <typename T> constexpr float kDrop = std::is_same<T, f16_t>::value ? 7.f : 0.f;

// Half of a V^T operand: the 16-lane group's lane k points at 4 consecutive d of its
// row and receives the 4 keys of column 16 dt + k.
template <int KROW>
__device__ __forceinline__ u32x2_t vt_read(const uint8_t* sv, int row, int swz, int dt, int frow) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  const int byte = dt * 32 + 8 * (frow & 3);
  const uint8_t* p = sv + row * KROW + (((byte >> 4) ^ swz) << 4) + (byte & 15);
  const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4*)((__attribute__((address_space(3))) uint8_t*)(p)));
  return __builtin_bit_cast(u32x2_t, r);
}

// Adds the values of one key that are not finite to the rows that see it (key <=
// lim): lane (g, frow) holds row frow's query chunks 4 ks + g and O[row][16 dt + 4 g + e];
// nm is minus the shift of the row's weights.
template <typename T, int HD, int QT, int NKS>
__device__ __forceinline__ void add_odd_key(const T* k, const T* v, int key, int g, float scale_log2,
                                            const int (&lim)[QT], const u32x4_t (&qf)[QT][NKS], const float (&nm)[QT],
                                            f32x4_t (&o)[QT][HD / 16]) {
  constexpr int EPC = 16 / sizeof(T), CPR = HD / EPC;
  bool odd = false;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt)
    for (int e = 0; e < 4; ++e) odd |= !(fabsf(Elem<T>::load(v + 16 * dt + 4 * g + e)) < INFINITY);
  if (__builtin_amdgcn_ballot_w64(odd) == 0) return;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    float s = 0.f;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const int c = 4 * ks + g;
      if (c < CPR) {
        float x[EPC], y[EPC];
        load_vec(k + c * EPC, x);
        unpack_vec<T>(qf[qt][ks], y);
#pragma unroll
        for (int e = 0; e < EPC; ++e) s = fmaf(x[e], y[e], s);
      }
    }
    s = column_sum(s);
    if (key > lim[qt]) continue;
    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s, scale_log2, nm[qt]));
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = Elem<T>::load(v + 16 * dt + 4 * g + e);
        if (!(fabsf(x) < INFINITY)) o[qt][dt][e] = fmaf(p, x, o[qt][dt][e]);
      }
  }
}

#endif

}  // namespace cgpt
