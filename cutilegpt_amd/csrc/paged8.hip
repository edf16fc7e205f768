// Writing the 8-bit paged cache, and reading it back as values.
//
// append8_kernel and, for single tokens, append8_step_kernel: the step's keys and values into
// codes, a power of two for each block of tokens and head (see paged8.h), keys and queries turned
// by their positions on the way.  read8_kernel: code * 2^e as rows of a wider type.
//
// 20 thousand tokens, 12 heads of 64 with turned queries, bf16 into int8: 71 us where the 153 MB
// alone would take 30 at a copy's 5.18 TB/s.  No unit is busy throughout: the VALU 53 % (some 35
// instructions a value: turning in 64 bits 9, rounding to odd 5, maximum 2, code 2, addresses and
// unpacking), the memory 2.2 TB/s, and 2.3 waves a SIMD (153 registers, which every way of turning
// shares; 128 spill, 77 us) wait at three barriers a head, with none of the next head's rows on
// their way meanwhile.  With a wave for an item and eight values a lane it took 204.  Eight
// tokens: 3.9 us (launch and dependent loads).  Reading the 20 thousand tokens back: 23 us, 4.0
// TB/s.
#include <algorithm>

#include "internal.h"
#include "paged8.h"

namespace cgpt {

typedef unsigned long long u64_t;

struct Append8Args {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  PagePool kc, vc;
  PagedBatch seq;
  Paged8 quant;
  const float* rot;  // row pos: rot_dim / 2 cosines, then rot_dim / 2 sines
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, rot_stride;
  int Hq, Hkv, rot_dim, n_pos, turn;
  int per_item, per_slot;  // blocks of tokens an item; blocks of threads a slot
  FastDiv width;         // positions an item, per_item * block
  int* err;
};

// A double as a float whose last bit is set when something was cut off: rounding that
// to a type of 22 bits or fewer gives what rounding the double would, and so do comparisons
// with its numbers.  (Numbers past the floats become infinite.)
__device__ __forceinline__ float to_odd(double r) {
  const u64_t b = __double_as_longlong(r);
  const uint32_t lo = static_cast<uint32_t>(b);
  // The 29 bits that a float has not, as one.
  const uint32_t cut = (lo | ((lo & 0x1fffffffu) + 0x1fffffffu)) & 0xe0000000u;
  return static_cast<float>(__longlong_as_double((b & ~u64_t{0xffffffffu}) | cut));
}

// How keys and queries are turned.
enum Turn {
  kNone,
  kNeighbours,  // pairs side by side
  kApart,       // pairs half of rot_dim apart, in whole chunks of eight values
  kApartOne     // the same, value by value
};

// A lane has two chunks of eight values of a row, the first from x0, the second from x1: those
// that are turned together (kApart), or neighbours.
struct Chunks {
  int x0, x1;
  __device__ __forceinline__ Chunks(int lane, int turn, int rot_dim) {
    const bool apart = turn == kApart && lane < rot_dim / 16;
    x0 = apart ? 8 * lane : 16 * lane;
    x1 = apart ? x0 + rot_dim / 2 : x0 + 8;
  }
};

// Their values, turned by the angles `cs`.  Products of two floats are exact in 64 bits, so a
// turned value is rounded once, to 53 bits, and then to the type: a code is what rounding the
// exact value would give, but for one in some 2^40.  ODD: floats by to_odd, else to nearest.
template <typename T, bool ODD>
__device__ __forceinline__ void turned16(const T* row, const Chunks& c, int turn, int rot_dim, const float* cs, float (&y)[16]) {
#pragma unroll
  for (int i = 0; i < 8; i += Elem<T>::kVec) {
    load_vec(row + c.x0 + i, y + i);
    load_vec(row + c.x1 + i, y + 8 + i);
  }
  if (turn == kNone || c.x0 >= rot_dim) return;
  auto narrow = [](double r) __attribute__((always_inline)) { return ODD ? to_odd(r) : static_cast<float>(r); };
  typedef float f32x4u_t __attribute__((ext_vector_type(4), aligned(4)));
  const int half = rot_dim / 2;
  if (turn == kNeighbours) {
#pragma unroll
    for (int i = 0; i < 16; i += 2)
      if (c.x0 + i < rot_dim) {
        const double co = cs[(c.x0 + i) / 2], si = cs[half + (c.x0 + i) / 2], u = y[i], v = y[i + 1];
        y[i] = narrow(__builtin_fma(-v, si, u * co));
        y[i + 1] = narrow(__builtin_fma(u, si, v * co));
      }
  } else if (turn == kApart) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const f32x4u_t c4 = *reinterpret_cast<const f32x4u_t*>(cs + c.x0 + i), s4 = *reinterpret_cast<const f32x4u_t*>(cs + half + c.x0 + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double co = c4[e], si = s4[e], u = y[i + e], v = y[8 + i + e];
        y[i + e] = narrow(__builtin_fma(-v, si, u * co));
        y[8 + i + e] = narrow(__builtin_fma(u, si, v * co));
      }
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < 16; ++i) {
      const int d = c.x0 + i;
      if (d >= rot_dim) break;
      const int at = d < half ? d : d - half;
      const double co = cs[at], si = d < half ? -cs[half + at] : cs[half + at];
      const double z = Elem<T>::load(row + (d < half ? d + half : at)), own = Elem<T>::load(row + d);
      const float r = narrow(__builtin_fma(z, si, own * co));
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = e == i ? r : y[e];
    }
  }
}

// The bits of the largest finite |y| of the lanes of a row (LPR neighbours).  *odd: one of the
// lane's is not finite.
template <int LPR> __device__ __forceinline__ uint32_t row_top(const float (&y)[16], bool* odd) {
  float t = 0.f, none = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    t = fmaxf(fmaxf(t, fabsf(y[i])), fabsf(y[i + 1]));
    none = __builtin_fmaf(y[i], 0.f, __builtin_fmaf(y[i + 1], 0.f, none));
  }
  *odd = none != 0.f;  // (inf and NaN times 0 are NaN)
  if (*odd) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t = fabsf(y[i]) < INFINITY ? fmaxf(t, fabsf(y[i])) : t;
  }
  if (LPR >= 2) t = fmaxf(t, dpp<kDppXor1>(t));
  if (LPR >= 4) t = fmaxf(t, dpp<kDppXor2>(t));
  if (LPR >= 8) t = fmaxf(t, dpp<kDppMirror8>(t));
  return __float_as_uint(t);
}

// Four values of at most the largest code (and no NaN) as codes.
template <int CODE> __device__ __forceinline__ uint32_t encode4_within(const float* y) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (CODE == CGPT_E4M3) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true));
  } else {
    // The sum with 1.5 * 2^23 rounds to a whole number, whose last byte it holds.
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(y[i] + 12582912.f);
    return __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | (__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u) << 16);
  }
#else
  return 0;
#endif
}

// An exponent with the word whether values may be past the codes or no numbers.
constexpr int kPast = 0x100;
template <int CODE> __device__ __forceinline__ bool is_last(int e) { return e == clamp_exp<CODE>(255); }

// The lane's values over 2^e as codes, in a row from `row` on.
template <int CODE> __device__ __forceinline__ void put16(uint8_t* row, const Chunks& c, const float (&y)[16], int e) {
  const float f = __uint_as_float(static_cast<uint32_t>(254 - (e & 0xff)) << 23);
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = y[i] * f;
  uint32_t w[4];
  if (e & kPast)
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = Codec<CODE>::encode4(x + 4 * i);
  else
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = encode4_within<CODE>(x + 4 * i);
  *reinterpret_cast<u32x2_t*>(row + c.x0) = u32x2_t{w[0], w[1]};
  *reinterpret_cast<u32x2_t*>(row + c.x1) = u32x2_t{w[2], w[3]};
}
// Sixteen codes shifted to an exponent that is `grown` larger.
template <int CODE> __device__ __forceinline__ void shift16(uint8_t* at, int grown) {
  const float f = __uint_as_float(static_cast<uint32_t>(max(127 - grown, 0)) << 23);
  u32x4_t w = *reinterpret_cast<const u32x4_t*>(at);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[4];
    Codec<CODE>::decode4(w[i], x);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] *= f;
    w[i] = Codec<CODE>::encode4(x);
  }
  *reinterpret_cast<u32x4_t*>(at) = w;
}

// Both are read first: a choice of which argument to read would put them all into memory.
template <typename P> __device__ __forceinline__ P choose(bool first, P a, P b) { return first ? a : b; }
__device__ __forceinline__ PagePool choose(bool first, const PagePool& a, const PagePool& b) {
  return PagePool{choose<void*>(first, a.base, b.base), choose(first, a.sp, b.sp), choose(first, a.sh, b.sh), choose(first, a.ss, b.ss)};
}
__device__ __forceinline__ ScalePool choose(bool first, const ScalePool& a, const ScalePool& b) {
  return ScalePool{choose<uint8_t*>(first, a.base, b.base), choose(first, a.sp, b.sp), choose(first, a.sh, b.sh), choose(first, a.sb, b.sb)};
}

// One head of the keys, the values or the queries, and the lane's chunks of its rows.
template <typename T> struct Unit8 {
  const T* src;
  int64_t st;
  int h, turn;
  bool is_q, is_v;
  Chunks c;
  __device__ __forceinline__ Unit8(const Append8Args& a, int unit, int lane)
      : is_q(unit >= 2 * a.Hkv), is_v(!is_q && unit >= a.Hkv), c(lane, !is_q && unit >= a.Hkv ? +kNone : a.turn, a.rot_dim) {
    h = is_q ? unit - 2 * a.Hkv : is_v ? unit - a.Hkv : unit;
    src = static_cast<const T*>(choose<const void*>(is_q, a.q, choose<const void*>(is_v, a.v, a.k))) +
          h * choose(is_q, a.q_sh, choose(is_v, a.v_sh, a.k_sh));
    st = choose(is_q, a.q_st, choose(is_v, a.v_st, a.k_st));
    turn = choose<int>(is_v, kNone, a.turn);
  }
  template <bool ODD>
  __device__ __forceinline__ void load(const Append8Args& a, int64_t token, int pos, bool* flag, float (&y)[16]) const {
    const bool off = turn != kNone && pos >= a.n_pos;
    *flag |= off;
    const float* cs = a.rot + (turn != kNone ? (off ? a.n_pos - 1 : pos) * a.rot_stride : 0);
    turned16<T, ODD>(src + token * st, c, turn, a.rot_dim, cs, y);
  }
  // A query's row.
  __device__ __forceinline__ void turn_query(const Append8Args& a, int64_t token, int pos, bool* flag) const {
    float y[16];
    load<sizeof(T) != 4>(a, token, pos, flag, y);
    T* const dst = static_cast<T*>(a.q_out) + token * a.qo_st + h * a.qo_sh;
#pragma unroll
    for (int i = 0; i < 8; i += Elem<T>::kVec) {
      store_vec(dst + c.x0 + i, y + i);
      store_vec(dst + c.x1 + i, y + 8 + i);
    }
  }
  // A row for the cache, and the bits of its largest finite value.
  template <int LPR>
  __device__ __forceinline__ uint32_t row(const Append8Args& a, int64_t token, int pos, bool* flag, bool* odd, float (&y)[16]) const {
    load<true>(a, token, pos, flag, y);
    return row_top<LPR>(y, odd);
  }
};

// One token a sequence: a row's lanes take one head.  Bound by the launch and dependent loads
// (length, page, exponent): 64 sequences, 25 heads of 64, 2 to 3 us within a graph, whatever the
// block.  But where a head's exponent grows, its row's lanes shift the block's earlier rows one
// after another, a load and a store each: a last token in blocks of 16 / 64 / 256 slots, two heads
// growing, e4m3 9 / 34 / 127 us, int8 17 / 63 / 248.
template <typename T, int CODE, int HD>
__global__ __launch_bounds__(256) void append8_step_kernel(Append8Args a) {
  constexpr int LPR = HD / 16;
  const int tid = threadIdx.x;
  const int b = static_cast<int>(blockIdx.x) / a.per_slot;
  const int unit = (static_cast<int>(blockIdx.x) - b * a.per_slot) * (256 / LPR) + tid / LPR;
  if (unit >= 2 * a.Hkv + (a.q != nullptr ? a.Hq : 0)) return;
  const Unit8<T> u(a, unit, tid % LPR);
  // (A length past 2^30, which no table has, is cut there.)
  const int len = min(a.seq.lens[b], 1 << 30), pos = len - 1;
  if (pos < 0) return;
  bool flag = false;
  if (u.is_q) {
    u.turn_query(a, b, pos, &flag);
  } else if (pos >= a.seq.cap) {
    flag = true;
  } else {
    const int col = a.seq.page.div(pos), slot = pos - col * static_cast<int>(a.seq.page.d);
    const int page = a.seq.table[b * a.seq.stride + col];
    float y[16];
    bool odd;
    const uint32_t t = u.template row<LPR>(a, b, pos, &flag, &odd, y);
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.seq.n_pages)) {
      flag = true;
    } else {
      const ScalePool sp = choose(u.is_v, a.quant.vs, a.quant.ks);
      const PagePool pool = choose(u.is_v, a.vc, a.kc);
      const int block = a.quant.block.div(slot), front = slot - block * static_cast<int>(a.quant.block.d);
      uint8_t* const at = sp.base + page * sp.sp + u.h * sp.sh + block * sp.sb;
      uint8_t* const rows = static_cast<uint8_t*>(pool.base) + page * pool.sp + u.h * pool.sh;
      const int old = front > 0 ? clamp_exp<CODE>(*at) : 0;
      const int e = max(Codec<CODE>::exponent(t), old);
      if (front > 0 && e > old)
        for (int i = slot - front; i < slot; ++i) shift16<CODE>(rows + i * pool.ss + 16 * (tid % LPR), e - old);
      if (tid % LPR == 0) *at = static_cast<uint8_t>(e);
      flag |= odd;
      put16<CODE>(rows + slot * pool.ss, u.c, y, e | (odd || is_last<CODE>(e) ? kPast : 0));
    }
  }
  if (flag && a.err != nullptr) *a.err = 1;
}

// Any numbers of tokens.  A block takes an item, per_item neighbouring blocks of one sequence, for
// `units` of the heads, one after the other; the sequence's items are those that its step
// touches.  Its waves take rows in turn, lanes 16 values each of a row.  First the largest value of
// every block (in LDS), then its exponent, then the codes.  One step of rows stays in registers for
// that; longer items are read twice, the second time from the cache.
constexpr int kItemBlocks = 64;
template <typename T, int CODE, int HD>
__global__ __launch_bounds__(256) void append8_kernel(Append8Args a, int units) {
  constexpr int LPR = HD / 16, RPI = 256 / LPR;
  __shared__ uint32_t top[2][kItemBlocks], past[2][kItemBlocks];
  __shared__ int exps[2][kItemBlocks], page_of_block[kItemBlocks], grown_by[2];
  const int tid = threadIdx.x, lane = tid & 63;
  int slot = static_cast<int>(blockIdx.x) / a.per_slot;
  const int unit0 = (static_cast<int>(blockIdx.x) - slot * a.per_slot) * units;
  const int unit1 = min(unit0 + units, 2 * a.Hkv + (a.q != nullptr ? a.Hq : 0));
  // Sequence b has the slots from start(b) on, as many as its items and more.
  auto start = [&](int i) { return a.width.div(min(max(a.seq.cu[i], 0), a.seq.n_tokens)) + 2 * i; };
  const int b = wave_count(a.seq.B, lane, [&](int i) { return start(i + 1) <= slot; });
  if (b >= a.seq.B) return;
  slot -= start(b);
  if (slot < 0) return;
  int first, count;
  seq_tokens(a.seq, b, &first, &count);
  // (A length past 2^30, which no table has, is cut there: positions stay far from 2^31.)
  const int len = min(max(a.seq.lens[b], 0), 1 << 30), pos0 = len - count;  // the first token's position
  const int W = static_cast<int>(a.width.d), blk = static_cast<int>(a.quant.block.d);
  const int page_size = static_cast<int>(a.seq.page.d);
  const int lo = max(pos0, 0), hi = min(len, a.seq.cap);
  bool flag = len > a.seq.cap && count > 0;
  const int64_t base64 = (static_cast<int64_t>(a.width.div(lo)) + slot) * W;
  if (base64 >= len) {
    if (flag && a.err != nullptr && tid == 0) *a.err = 1;
    return;
  }
  const int base = static_cast<int>(base64), p0 = max(lo, base);
  // (Queries past the table are still turned.)
  const int q1 = static_cast<int>(min(static_cast<int64_t>(len), base64 + W)), p1 = min(q1, hi);
  const int r = tid / LPR;
  // Thread i: block i's place, of those that rows are written to (a sequence without tokens has none).
  const int first_p = base + tid * blk, col = a.seq.page.div(max(min(first_p, hi - 1), 0));
  const bool mine = p0 < p1 && tid < a.per_item && first_p < p1 && first_p + blk > p0;
  const int page = mine ? a.seq.table[b * a.seq.stride + col] : -1;
  const bool there = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.seq.n_pages);
  flag |= mine && !there;
  if (mine) page_of_block[tid] = page;
  if (tid < kItemBlocks) top[0][tid] = past[0][tid] = 0;
  for (int unit = unit0; unit < unit1; ++unit) {
    const Unit8<T> u(a, unit, tid % LPR);
    if (u.is_q) {
      for (int p = p0 + r; p < q1; p += RPI) u.turn_query(a, first + (p - pos0), p, &flag);
      continue;
    }
    if (p0 >= p1) continue;
    // ---- the blocks' largest values (of two units in turn: no wait before the next begins)
    const int turn = (unit - unit0) & 1;
    float y[16];
    uint32_t row_max = 0;
    bool odd = false;
    auto load_rows = [&](int from) __attribute__((always_inline)) {
      const int p = from + r;
      if (p < p1) row_max = u.template row<LPR>(a, first + (p - pos0), p, &flag, &odd, y);
    };
    load_rows(p0);
    __syncthreads();
    if (tid < kItemBlocks) top[turn ^ 1][tid] = past[turn ^ 1][tid] = 0;
    if (tid == 0) grown_by[turn] = 0;
    for (int from = p0; from < p1; from += RPI) {
      if (from != p0) load_rows(from);
      const int p = from + r;
      if (p < p1) {
        const int i = a.quant.block.div(p - base);
        if (tid % LPR == 0) atomicMax(&top[turn][i], row_max);
        if (odd) {
          flag = true;
          past[turn][i] = 1;
        }
      }
    }
    __syncthreads();
    // ---- the exponents
    const ScalePool sp = choose(u.is_v, a.quant.vs, a.quant.ks);
    const PagePool pool = choose(u.is_v, a.vc, a.kc);
    if (mine) {
      uint8_t* const at = sp.base + (there ? page : 0) * sp.sp + u.h * sp.sh + a.quant.block.div(first_p - col * page_size) * sp.sb;
      int e = Codec<CODE>::exponent(top[turn][tid]);
      if (first_p < p0 && there) {
        // The block that the step goes on in.
        const int old = clamp_exp<CODE>(*at);
        e = max(e, old);
        grown_by[turn] = e - old;
      }
      if (there) *at = static_cast<uint8_t>(e);
      exps[turn][tid] = there ? e | (past[turn][tid] || is_last<CODE>(e) ? kPast : 0) : -1;
    }
    __syncthreads();
    // The row of position p in block i; a block lies in one page.
    uint8_t* const dst = static_cast<uint8_t*>(pool.base) + u.h * pool.sh;
    auto row_of = [&](int p, int i) __attribute__((always_inline)) {
      return dst + page_of_block[i] * pool.sp + (p - a.seq.page.div(p) * page_size) * pool.ss;
    };
    if (grown_by[turn] > 0) {
      const int i = a.quant.block.div(p0 - base);
      for (int p = base + i * blk + r; p < p0; p += RPI) shift16<CODE>(row_of(p, i) + 16 * (tid % LPR), grown_by[turn]);
    }
    // ---- the codes
    const bool again = p1 - p0 > RPI;
    for (int from = p0; from < p1; from += RPI) {
      if (again) load_rows(from);
      const int p = from + r;
      if (p >= p1) continue;
      const int i = a.quant.block.div(p - base), e = exps[turn][i];
      if (e >= 0) put16<CODE>(row_of(p, i), u.c, y, e);
    }
  }
  if (flag && a.err != nullptr) *a.err = 1;
}

struct Read8Args {
  PagePool kc, vc;
  PagedBatch seq;
  Paged8 quant;
  void* k_out;
  void* v_out;
  int64_t ko_st, ko_sh, vo_st, vo_sh;
  int Hkv;
  int* err;
};

// A thread takes 8 codes at a time of one row's heads; `heads_log2` heads of a row side by
// side, 2^tokens_log2 rows a block.
template <typename T, int CODE, int HD>
__global__ __launch_bounds__(256) void read8_kernel(Read8Args a, int tokens_log2) {
  constexpr int LPR = HD / 8;
  const int tid = threadIdx.x, x0 = tid % LPR * 8;
  const int side = (256 / LPR) >> tokens_log2;  // heads side by side
  const int h0 = tid / LPR % side;
  const int t = (blockIdx.x << tokens_log2) + tid / LPR / side;
  if (t >= a.seq.n_tokens) return;
  const int b = seq_of(a.seq, t);
  if (b >= a.seq.B) return;
  int first, count;
  seq_tokens(a.seq, b, &first, &count);
  if (t < first) return;
  const int pos = max(a.seq.lens[b], 0) - count + (t - first);
  bool bad = pos >= a.seq.cap;
  const bool none = pos < 0 || bad;  // rows that are not in the cache: zeros
  int page = 0, slot = 0;
  if (!none) {
    const int col = a.seq.page.div(pos);
    slot = pos - col * static_cast<int>(a.seq.page.d);
    page = page_of(a.seq.table + b * a.seq.stride, col, a.seq.n_pages, &bad);
  }
  const int block = a.quant.block.div(slot);
  for (int h = h0; h < 2 * a.Hkv; h += side) {
    const bool is_v = h >= a.Hkv;
    const int hk = is_v ? h - a.Hkv : h;
    const PagePool pool = choose(is_v, a.vc, a.kc);
    const ScalePool sp = choose(is_v, a.quant.vs, a.quant.ks);
    float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (!none) {
      const float f = scale_of<CODE>(sp.base[page * sp.sp + hk * sp.sh + block * sp.sb]);
      const u32x2_t w = *reinterpret_cast<const u32x2_t*>(static_cast<const uint8_t*>(pool.base) + page * pool.sp +
                                                          hk * pool.sh + slot * pool.ss + x0);
      Codec<CODE>::decode4(w[0], y);
      Codec<CODE>::decode4(w[1], y + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= f;
    }
    T* const dst = (is_v ? static_cast<T*>(a.v_out) + t * a.vo_st + hk * a.vo_sh
                         : static_cast<T*>(a.k_out) + t * a.ko_st + hk * a.ko_sh) + x0;
#pragma unroll
    for (int i = 0; i < 8; i += Elem<T>::kVec) store_vec(dst + i, y + i);
  }
  if (bad && a.err != nullptr) *a.err = 1;
}

}  // namespace cgpt

extern "C" int cgpt_paged_kv_append_8bit(const cgpt_paged8_args* args, void* stream) {
  using namespace cgpt;
  bool empty;
  const int rc = check_paged8(args, true, &empty);
  if (rc != CGPT_OK) return rc;
  const cgpt_paged_args& p = args->p;
  if (p.k_cache == p.v_cache || args->k_scale == args->v_scale || (p.q == nullptr) != (p.out == nullptr)) return CGPT_EINVAL;
  if (p.rot_dim < 0 || p.rot_dim > p.head_dim || p.rot_dim % 2 != 0) return CGPT_ESHAPE;
  if (p.rot_dim > 0 && (p.rotary == nullptr || (reinterpret_cast<uintptr_t>(p.rotary) & 3) || p.n_pos <= 0 ||
                        p.n_pos > 0x7fffffff || p.rot_stride < p.rot_dim))
    return CGPT_EINVAL;
  if (empty) return CGPT_OK;
  if (p.k == nullptr || p.v == nullptr) return CGPT_EINVAL;
  if (p.out != nullptr && !rows_apart({{p.n_tokens, p.out_st}, {p.Hq, p.out_sh}}, p.head_dim)) return CGPT_EINVAL;
  Append8Args a{p.q, p.k, p.v, p.out, PagePool{p.k_cache, p.kc_sp, p.kc_sh, p.kc_ss},
                PagePool{p.v_cache, p.vc_sp, p.vc_sh, p.vc_ss}, paged_batch(p), paged8(*args), p.rotary, p.q_st, p.q_sh,
                p.k_st, p.k_sh, p.v_st, p.v_sh, p.out_st, p.out_sh, p.rot_stride, static_cast<int>(p.Hq),
                static_cast<int>(p.Hkv), static_cast<int>(p.rot_dim), static_cast<int>(p.n_pos),
                p.rot_dim == 0 ? kNone : p.interleaved ? kNeighbours : p.rot_dim % 16 == 0 ? kApart : kApartOne, 0, 0, FastDiv(),
                p.err_flag};
  // (rows: of a block's threads, 16 values each.)
  const int64_t units = 2 * p.Hkv + (p.q != nullptr ? p.Hq : 0), rows = 256 * 16 / p.head_dim;
  a.per_item = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kItemBlocks, rows / args->block)));
  a.width = FastDiv(a.per_item * args->block);
  const bool step = p.cu_q == nullptr;
  const int64_t slots = step ? p.B : p.n_tokens / a.width.d + 2 * p.B;
  // Heads that a block takes: as many as leave 24 blocks a CU.
  const int64_t each = step ? rows : std::max<int64_t>(1, std::min(units, slots * units / (24 * num_cus())));
  a.per_slot = static_cast<int>((units + each - 1) / each);
  if (slots * a.per_slot > kMaxBlocks) return CGPT_ESHAPE;
  const dim3 grid(static_cast<unsigned>(slots * a.per_slot));
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_types8(*args, [&](auto t, auto code, auto hd) {
    if (step)
      hipLaunchKernelGGL((append8_step_kernel<decltype(t), decltype(code)::value, decltype(hd)::value>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((append8_kernel<decltype(t), decltype(code)::value, decltype(hd)::value>), grid, dim3(256), 0, s, a,
                         static_cast<int>(each));
    return hip_status(hipGetLastError());
  });
}

extern "C" int cgpt_paged_kv_read_8bit(const cgpt_paged8_args* args, void* stream) {
  using namespace cgpt;
  bool empty;
  const int rc = check_paged8(args, false, &empty);
  if (rc != CGPT_OK) return rc;
  if (empty) return CGPT_OK;
  const cgpt_paged_args& p = args->p;
  if (p.out == nullptr || args->v_out == nullptr) return CGPT_EINVAL;
  if (!rows_apart({{p.n_tokens, p.out_st}, {p.Hkv, p.out_sh}}, p.head_dim) ||
      !rows_apart({{p.n_tokens, args->vo_st}, {p.Hkv, args->vo_sh}}, p.head_dim))
    return CGPT_EINVAL;
  const Read8Args a{PagePool{p.k_cache, p.kc_sp, p.kc_sh, p.kc_ss}, PagePool{p.v_cache, p.vc_sp, p.vc_sh, p.vc_ss},
                    paged_batch(p), paged8(*args), p.out, args->v_out, p.out_st, p.out_sh, args->vo_st, args->vo_sh,
                    static_cast<int>(p.Hkv), p.err_flag};
  // As many rows a block as leave eight blocks a CU.
  int tokens_log2 = 0;
  while ((p.head_dim / 8 << (tokens_log2 + 1)) <= 256 && (p.n_tokens >> (tokens_log2 + 1)) >= 8 * num_cus()) ++tokens_log2;
  const int64_t blocks = (p.n_tokens + (int64_t{1} << tokens_log2) - 1) >> tokens_log2;
  if (blocks > kMaxBlocks) return CGPT_ESHAPE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_types8(*args, [&](auto t, auto code, auto hd) {
    hipLaunchKernelGGL((read8_kernel<decltype(t), decltype(code)::value, decltype(hd)::value>),
                       dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a, tokens_log2);
    return hip_status(hipGetLastError());
  });
}
