// Attention over the paged key-value cache.
//
// o[i, h] = softmax(scale q[i, h] K^T) V over the keys 0 .. pos(i) of token i's
// sequence, read from its pages; with a shared prefix the first prefix_len keys of
// every sequence are read from one list of pages.
//
// Softmax runs in base 2 in one pass over the keys with a running shift m: p = 2^(s
// scale log2(e) - m), l = sum p, O = sum p v; parts of a row's keys join by m = max m_i,
// l = sum l_i 2^(m_i - m), O likewise.  m, l, O and the scores are 32-bit; p is rounded to
// the 16-bit type for the second product (the other operand has no more bits; kDrop keeps
// fp16's range from losing small ones), while l adds the unrounded ones.
//
// Three kernels: the stream kernel here for few rows (a decode step reads every key once:
// the bound is HBM), the tile kernel (paged_tile.hip) for many, the join of their
// partials.  make_plan below chooses.  Measured: 64 sequences of 1 to 8192 keys, 25 heads
// of head_dim 64, bf16 295 us, 5.7 TB/s, fp32 577 us, 5.8 TB/s; four of 90 to 130 thousand, 8
// heads of 128, fp16 308 us, 5.8 TB/s (a kernel that only reads reaches 6.3 on the same card
// with this cache policy, 7.2 with nontemporal loads); one of 500 keys 8 us.
#include <algorithm>

#include "internal.h"
#include "paged.h"

namespace cgpt {

// Chunk swizzle of V row `key` in LDS.  16-bit rows are read by transposing loads, eight
// rows apart in the low bits; fp32 columns by four lane groups, four rows apart.
template <typename T, int CPR> __device__ __forceinline__ int vswz(int key) {
  if (sizeof(T) == 2) return key & ((CPR < 8 ? CPR : 8) - 1);
  return ((key >> 2) << 2) & (CPR - 1);
}

// ------------------------------------------------------------------ work units
//
// The work is a list of items, each one tile of R query rows of one key head against
// a run of keys:
//   * (prefix only) rows are the packed tokens of all sequences, token-major, G
//     heads each; keys are [0, prefix_len);
//   * rows are one sequence's; keys are [prefix_len, length).
// An item's keys are cut into units of UK << unit_shift keys (a shift of 0, unless the units of
// the longest sequences that the table allows would pass 32 bits).  The units of all items, in order (prefix:
// head, row tile, unit; then sequence, head, row tile, unit), are dealt to the blocks in
// equal contiguous runs, so a batch of any lengths keeps every CU busy to the end: the
// lengths live on the device, and the host launches one grid for all of them.  A run
// ends inside an item at most twice; those pieces leave (m, l, O) partials, which the
// join kernel adds in key order.  Nothing depends on which block runs first.

struct SeqUnits {
  int first, count;  // tokens
  int len, n;        // keys; keys the table can name (0 without a token)
  int kb, base0;     // first own key, and the 16-key boundary at or below it
  int rt, kt;        // row tiles, key units
};

// ceil(n / (UK << shift)).
template <int UK> __device__ __forceinline__ int key_units(int n, int shift) {
  static_assert((UK & (UK - 1)) == 0, "divided by a shift");
  return (n + (UK << shift) - 1) >> (__builtin_ctz(UK) + shift);
}

template <int R, int UK>
__device__ __forceinline__ SeqUnits seq_units(const PagedAttnArgs& a, int b, int shift) {
  SeqUnits u;
  seq_tokens(a.seq, b, &u.first, &u.count);
  u.len = max(a.seq.lens[b], 0);
  u.n = u.count > 0 ? min(u.len, a.seq.cap) : 0;
  u.kb = a.prefix_len;
  u.base0 = u.kb & ~15;
  u.rt = (u.count * static_cast<int>(a.group.d) + R - 1) / R;
  u.kt = u.n > u.kb ? key_units<UK>(u.n - u.base0, shift) : 0;
  return u;
}

// U units dealt to at most `grid` blocks: the first r blocks have q + 1, the rest q.
struct Deal {
  int g, q, r;
  __device__ Deal(int grid, int U) {
    g = min(grid, max(U, 1));
    q = U / g;
    r = U - q * g;
  }
  __device__ int start(int block) const { return block * q + min(block, r); }
  __device__ int owner(int u) const {
    const int t = r * (q + 1);
    return u < t ? u / (q + 1) : r + (u - t) / q;
  }
};

// The workspace: unit starts of the sequences; the two edge partials of every block
// (2 x R rows each); with a prefix also one partial a row for the items that one block
// holds whole.
struct PagedWs {
  int* starts;       // B + 1
  float* edge_ml;    // grid x 2 x R x {m, l}
  float* edge_o;     // grid x 2 x R x HD
  float* whole_ml;   // {prefix, own} x n_tokens x Hq x {m, l}
  float* whole_o;    // {prefix, own} x n_tokens x Hq x HD
  float* tile_ml;    // the tile kernel's splits x n_tokens x Hq x {m, l}
  float* tile_o;     // splits x n_tokens x Hq x HD
  int unit_shift;    // units of UK << unit_shift keys
};

template <typename T, int HD, int QTW, int NW>
struct StreamShape {
  static constexpr int ES = sizeof(T);
  static constexpr int EPC = 16 / ES;              // elements of a 16-byte chunk
  static constexpr int CPR = HD / EPC;             // chunks of a row
  static constexpr int SWZ = (CPR < 8 ? CPR : 8) - 1;  // see vswz
  static constexpr int KSTEP = 4 * EPC;            // head_dim of one k-slab
  static constexpr int NKS = (HD + KSTEP - 1) / KSTEP;
  static constexpr int ND = HD / 16;
  // 16-key tiles a wave takes at once: 8 KiB of K and V, 16 KiB for the lone wave, which
  // has the registers for it (and at head_dim 128).
  static constexpr int NT = (ES == 2 ? 2 : 1) * (HD >= 64 ? 1 : 2) * (NW == 1 ? 2 : 1);
  static constexpr int KT = 16 * NT;
  static constexpr int UK = NW * KT;               // keys of a unit, KT a wave
  static constexpr int QT = QTW, R = 16 * QTW;
  static constexpr int KROW = HD * ES;
  static constexpr int VBYTES = KT * KROW;         // a wave's V tile in LDS; holds 16 fp32 rows of O too
  // Chunk of a row that lane group g takes in slab ks; rows of 16 16-bit values have but two.
  __device__ static constexpr bool has(int ks, int g) { return CPR >= 4 * NKS || 4 * ks + g < CPR; }
  __device__ static constexpr int chunk(int ks, int g) { return has(ks, g) ? 4 * ks + g : CPR - 1; }
  static_assert(VBYTES >= 16 * HD * 4, "the join of the waves reuses the V tiles");
};

// Waves of a block with one row tile: lone waves need no join of the four and take
// twice the keys at once (64 sequences x 25 heads of head_dim 64: 256 keys 39 -> 33 us,
// 1024 keys 97 -> 88, 8192 keys 578 -> 569); at head_dim 128 four of them read a page's
// rows together (128 x 8 heads, 2048 keys: 201 us alone, 192 together).
constexpr int stream_waves(int hd) { return hd == 128 ? 4 : 1; }

// Each wave streams keys by itself: K and V rows go from their pages into registers,
// one subtile of KT keys ahead of the one in use, in the layout of the matrix cores' A
// operand (lane l: row l % 16, 16-byte chunk l / 16), so S^T = K Q^T needs no LDS at
// all; V passes through the wave's own LDS tile for its transpose (O^T = V^T P^T).
// The NW waves of a block take a unit's KT-key parts and meet only at an item's end.
// P comes straight from the S^T accumulators, the key order inside a slab permuted alike
// on both operands.
//
// A subtile costs some 450 instructions whatever rows it serves, an item 1200 (scan of the
// lengths, addresses, join): 60 % of the issue slots at the rate HBM delivers, so short
// items are bound by them (64 x 25 items of 256 keys: 33 us, 3.2 TB/s).
//
// WHOLE: a block is one item with all its keys, the prefix's among them, and writes its
// rows' results; no workspace, no join.
// A16: 16 keys from a multiple of 16 on lie in one page (and on one side of the prefix's
// end), whose id comes by a scalar load; else every lane looks its own key up.
template <typename T, int HD, int QTW, bool A16, int NW, bool WHOLE>
__global__ __launch_bounds__(64 * NW, NW == 16 ? 4 : HD == 128 && QTW > 1 ? 1 : 2) void
paged_stream_kernel(PagedAttnArgs a, PagedWs ws, int prefix_units) {
  using C = StreamShape<T, HD, QTW, NW>;
  constexpr int QT = C::QT, NT = C::NT, NKS = C::NKS, ND = C::ND, KT = C::KT, UK = C::UK, R = C::R;
  __shared__ __attribute__((aligned(16))) uint8_t smem[NW * C::VBYTES];
  __shared__ float wave_m[NW][R], wave_l[NW][R];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int g = lane >> 4, frow = lane & 15;
  const int G = static_cast<int>(a.group.d), page_size = static_cast<int>(a.seq.page.d);
  uint8_t* const sv = smem + wave * C::VBYTES;
  bool bad = false;

  // Units of up to 64 sequences from c0 on: lane l holds sequence c0 + l.  `before` counts
  // the units in front of them.
  int c0 = 0, n_units = 0, incl = 0, before = prefix_units, total = 0;
  SeqUnits mine{};
  auto scan = [&](int v) __attribute__((always_inline)) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int w = __shfl_up(v, off, 64);
      if (lane >= off) v += w;
    }
    return v;
  };
  auto load_chunk = [&](int c, int end) __attribute__((always_inline)) {
    c0 = c;
    n_units = 0;
    if (c + lane < end) {
      mine = seq_units<R, UK>(a, c + lane, ws.unit_shift);
      n_units = mine.rt * mine.kt * a.Hkv;
    }
    incl = scan(n_units);
    total = __builtin_amdgcn_readlane(incl, 63);
  };
  // More than 64 sequences: lane l adds up `per` of them, from l per on.
  const int per = (a.seq.B + 63) >> 6;
  int group_units = 0, group_incl = 0;
  // The item at hand: rows of tile rt of key head hk, keys [kb, n), cut into kt_item units
  // from base0 on; t0 is its first unit here.
  int u = 0, u_end = 1, hk = 0, rt = 0, rts = 1, t0 = 0, kt_item = 0, kb = 0, base0 = 0, n_all = 0, rows = 0, first = 0,
      pos0 = 0;
  bool prefix = false;
  const int* trow = nullptr;
  // The sequence whose units u lies in; false when there is none (the lengths changed
  // under the call).
  auto enter_sequence = [&]() __attribute__((always_inline)) {
    if (per > 1) {
      const int gi = __popcll(__builtin_amdgcn_ballot_w64(prefix_units + group_incl <= u));
      if (gi >= 64) return false;
      const int end = min((gi + 1) * per, a.seq.B);
      before = prefix_units + __builtin_amdgcn_readlane(group_incl - group_units, gi);
      for (load_chunk(gi * per, end); u >= before + total; load_chunk(c0 + 64, end)) {
        if (c0 + 64 >= end) return false;
        before += total;
      }
    }
    if (u >= before + total) return false;
    const int at = __popcll(__builtin_amdgcn_ballot_w64(before + incl <= u));
    auto of = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, at); };
    prefix = false;
    rts = of(mine.rt);
    kt_item = of(mine.kt);
    t0 = u - before - of(incl - n_units);  // units into the sequence
    n_all = of(mine.n);
    first = of(mine.first);
    const int count = of(mine.count), len = of(mine.len);
    rows = count * G;
    pos0 = len - count;
    kb = a.prefix_len;
    base0 = kb & ~15;
    trow = a.seq.table + (c0 + at) * a.seq.stride;
    bad |= len > a.seq.cap;
    return true;
  };
  if constexpr (WHOLE) {
    rt = static_cast<int>(blockIdx.x) / a.Hkv;
    hk = static_cast<int>(blockIdx.x) - rt * a.Hkv;
    const int b = slot_seq<R>(a.seq, G, lane, &rt);
    if (b >= a.seq.B) return;
    int count;
    seq_tokens(a.seq, b, &first, &count);
    rows = count * G;
    if (rt < 0 || rt * R >= rows) return;
    const int len = max(a.seq.lens[b], 0);
    n_all = min(len, a.seq.cap);
    pos0 = len - count;
    trow = a.seq.table + b * a.seq.stride;
    bad = len > a.seq.cap;
  } else {
    const bool writes = blockIdx.x == 0 && wave == 0;
    if (per == 1) {
      load_chunk(0, a.seq.B);
      group_incl = incl;
      if (writes && lane < a.seq.B) ws.starts[lane] = prefix_units + incl - n_units;
    } else {
      const int first_b = lane * per, end_b = min(first_b + per, a.seq.B);
#pragma unroll 4
      for (int b = first_b; b < end_b; ++b) {
        const SeqUnits su = seq_units<R, UK>(a, b, ws.unit_shift);
        group_units += su.rt * su.kt * a.Hkv;
      }
      group_incl = scan(group_units);
      if (writes) {
        int at = prefix_units + group_incl - group_units;
        for (int b = first_b; b < end_b; ++b) {
          const SeqUnits su = seq_units<R, UK>(a, b, ws.unit_shift);
          ws.starts[b] = at;
          at += su.rt * su.kt * a.Hkv;
        }
      }
    }
    const int U = prefix_units + __builtin_amdgcn_readlane(group_incl, 63);
    if (blockIdx.x == 0 && tid == 0) ws.starts[a.seq.B] = U;
    const Deal deal(gridDim.x, U);
    if (static_cast<int>(blockIdx.x) >= deal.g || U == 0) return;
    u = deal.start(blockIdx.x);
    u_end = deal.start(blockIdx.x + 1);
    if (u < prefix_units) {
      prefix = true;
      kt_item = key_units<UK>(a.prefix_len, ws.unit_shift);
      rows = a.seq.n_tokens * G;
      rts = (rows + R - 1) / R;
      n_all = a.prefix_len;
      trow = a.prefix;
      t0 = u;
    } else if (!enter_sequence()) {
      return;
    }
    const int item = t0 / kt_item;
    t0 -= item * kt_item;
    hk = item / rts;
    rt = item - hk * rts;
  }

  for (;;) {
    // Addresses are made anew for every item: kept over the loop they cost registers that
    // the loads in flight need.
    asm volatile("" : "+v"(g), "+v"(frow));
    // Keys that the tile's last row sees.
    const int n = prefix ? n_all : min(n_all, max(pos0 + a.group.div(min(rt * R + R, rows) - 1) + 1, 0));
    if constexpr (WHOLE) kt_item = (n + UK - 1) / UK;
    const int t1 = WHOLE ? kt_item : min(kt_item, t0 + (u_end - u));

    // ---- its rows: lane (g, frow) works for rows rt R + 16 qt + frow
    const int r0 = rt * R, nqt = min(QT, (rows - r0 + 15) >> 4);
    int lim[QT];  // last key the row sees; rows that do not exist are never masked
    u32x4_t qf[QT][NKS];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int r = r0 + 16 * qt + frow;
      const bool live = r < rows;
      const int i = a.group.div(live ? r : 0), h = hk * G + (live ? r : 0) - i * G;
      const int t = first + i;
      if (prefix) {
        const int bb = seq_of(a.seq, t);
        int f, c;
        lim[qt] = -1;
        if (bb < a.seq.B) {
          seq_tokens(a.seq, bb, &f, &c);
          lim[qt] = min(a.seq.lens[bb] - c + (t - f), a.prefix_len - 1);
        }
      } else {
        lim[qt] = min(pos0 + i, n - 1);
      }
      if (!live) lim[qt] = 0x7fffffff;
      const T* qp = static_cast<const T*>(a.q) + t * a.q_st + h * a.q_sh;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const u32x4_t v = *reinterpret_cast<const u32x4_t*>(qp + C::chunk(ks, g) * C::EPC);
        qf[qt][ks] = live && C::has(ks, g) ? v : u32x4_t{0, 0, 0, 0};
      }
    }
    f32x4_t o[QT][ND];
    float m_run[QT], l_run[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      m_run[qt] = -INFINITY;
      l_run[qt] = 0.f;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) o[qt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    // ---- its keys
    const T* const kh = static_cast<const T*>(a.kc.base) + hk * a.kc.sh;
    const T* const vh = static_cast<const T*>(a.vc.base) + hk * a.vc.sh;
    const int shift = WHOLE ? 0 : ws.unit_shift;
    const int sub0 = base0 + ((t0 * UK) << shift) + wave * KT;  // first subtile; the next is UK further
    const int cnt = sub0 < n ? min((t1 - t0) << shift, (n - sub0 + UK - 1) / UK) : 0;
    int odd_from = 0x7fffffff;  // first masked key tile of the wave with a value that is not finite
    u32x4_t kf[NT][NKS], vf[NT][NKS];
    // Pages of subtile i: one a 16-key tile, or one a lane's key.
    auto fetch = [&](int i, int (&pg)[NT]) __attribute__((always_inline)) {
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        const int tile = sub0 + i * UK + 16 * kt;
        if (A16) {
          const int key = min(tile, (n - 1) & ~15), col = a.seq.page.div(key);
          const int* const row = WHOLE && key < a.prefix_len ? a.prefix : trow;
          pg[kt] = ((const __attribute__((address_space(4))) int*)row)[__builtin_amdgcn_readfirstlane(col)];
        } else {
          const int key = max(min(tile + frow, n - 1), kb);
          pg[kt] = (WHOLE && key < a.prefix_len ? a.prefix : trow)[a.seq.page.div(key)];
        }
      }
    };
    // A lane's bytes into a key tile, and into its chunk of the row (A16).
    const uint32_t k_row = static_cast<uint32_t>(sizeof(T) * a.kc.ss), v_row = static_cast<uint32_t>(sizeof(T) * a.vc.ss);
    auto load = [&](int i, const int (&pg)[NT], u32x4_t (&kd)[NT][NKS], u32x4_t (&vd)[NT][NKS]) __attribute__((always_inline)) {
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        const int tile = sub0 + i * UK + 16 * kt;
        const int key = A16 ? min(tile, (n - 1) & ~15) : max(min(tile + frow, n - 1), kb);
        const int slot = key - a.seq.page.div(key) * page_size;
        int p = A16 ? __builtin_amdgcn_readfirstlane(pg[kt]) : pg[kt];
        if (static_cast<uint32_t>(p) >= static_cast<uint32_t>(a.seq.n_pages)) {
          p = 0;
          bad = true;
        }
        const uint8_t* const kp = reinterpret_cast<const uint8_t*>(kh + p * a.kc.sp + slot * a.kc.ss);
        const uint8_t* const vp = reinterpret_cast<const uint8_t*>(vh + p * a.vc.sp + slot * a.vc.ss);
        uint32_t row = 0;
        if (A16) row = tile >= kb && tile + 16 <= n ? frow : max(min(tile + frow, n - 1), kb) - key;
        const uint32_t ko = row * k_row, vo = row * v_row;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          const int c = 16 * C::chunk(ks, g);
          kd[kt][ks] = *reinterpret_cast<const u32x4_t*>(kp + (ko + c));
          vd[kt][ks] = *reinterpret_cast<const u32x4_t*>(vp + (vo + c));
          // Lanes past a short row's chunks: 0 x inf would be NaN.
          if (!C::has(ks, g)) kd[kt][ks] = u32x4_t{0, 0, 0, 0};
        }
      }
    };
    auto v_slot = [&](int kt, int ks) __attribute__((always_inline)) {
      const int key = 16 * kt + frow;
      return sv + key * C::KROW + (((4 * ks + g) ^ vswz<T, C::CPR>(key)) << 4);
    };
    auto compute = [&](int base, const u32x4_t (&kd)[NT][NKS], const u32x4_t (&vd)[NT][NKS]) __attribute__((always_inline)) {
      bool masked = base < kb;
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
        if (qt < nqt) masked |= __builtin_amdgcn_ballot_w64(lim[qt] < base + KT - 1) != 0;
      asm volatile("" ::: "memory");
      if (!masked) {
#pragma unroll
        for (int kt = 0; kt < NT; ++kt)
#pragma unroll
          for (int ks = 0; ks < NKS; ++ks)
            if (C::has(ks, g)) *reinterpret_cast<u32x4_t*>(v_slot(kt, ks)) = vd[kt][ks];
      } else {
        // A masked key's weight is 0, but 0 x NaN is NaN: where a row is masked the matrix
        // cores get the finite values alone, and the others are added at the item's end to
        // the rows that see them.
        uint32_t bits = 0;
#pragma unroll
        for (int kt = 0; kt < NT; ++kt)
#pragma unroll
          for (int ks = 0; ks < NKS; ++ks) {
            u32x4_t v = vd[kt][ks];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              bits |= special_bits<T>(v[e]);
              v[e] = finite_part<T>(v[e]);
            }
            if (C::has(ks, g)) *reinterpret_cast<u32x4_t*>(v_slot(kt, ks)) = v;
          }
        if (__builtin_amdgcn_ballot_w64((bits & 0x80008000u) != 0) != 0) odd_from = min(odd_from, base);
      }
      asm volatile("" ::: "memory");
      f32x4_t s[QT][NT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) s[qt][kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
        if (qt < nqt)
#pragma unroll
          for (int kt = 0; kt < NT; ++kt)
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) Mfma<T>::run(kd[kt][ks], qf[qt][ks], s[qt][kt]);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
        if (qt < nqt) {
          if (masked) {
            const int hi = lim[qt] - base - 4 * g, lo = kb - base - 4 * g;
#pragma unroll
            for (int kt = 0; kt < NT; ++kt)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                s[qt][kt][r] = (16 * kt + r > hi || 16 * kt + r < lo) ? -INFINITY : s[qt][kt][r];
          }
          float mx = -INFINITY;
#pragma unroll
          for (int kt = 0; kt < NT; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[qt][kt][r]);
          mx = column_max(mx) * a.scale_log2;
          // The shift moves only when the maximum outgrows it by more than 8 (see kDrop), so
          // P <= 2^8 and the accumulators are rescaled on few subtiles.
          const bool grow = mx > m_run[qt] + (8.0f + kDrop<T>);
          if (__builtin_amdgcn_ballot_w64(grow) != 0) {
            const float m_new = grow ? mx - kDrop<T> : m_run[qt];
            const float alpha = grow ? __builtin_amdgcn_exp2f(m_run[qt] - m_new) : 1.0f;
            m_run[qt] = m_new;
            l_run[qt] *= alpha;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
              for (int r = 0; r < 4; ++r) o[qt][dt][r] *= alpha;
          }
          const float shift = m_run[qt] == -INFINITY ? 0.f : -m_run[qt];
          float sum = 0.f;
#pragma unroll
          for (int kt = 0; kt < NT; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qt][kt][r], a.scale_log2, shift));
              s[qt][kt][r] = p;
              sum += p;
            }
          l_run[qt] += sum;
        }
      if constexpr (sizeof(T) == 2) {
        const int vrow = 4 * g + (frow >> 2);
#pragma unroll
        for (int c = 0; c < NT / 2; ++c) {
          u32x4_t pf[QT];
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
            pf[qt] = u32x4_t{pack2<T>(s[qt][2 * c][0], s[qt][2 * c][1]), pack2<T>(s[qt][2 * c][2], s[qt][2 * c][3]),
                             pack2<T>(s[qt][2 * c + 1][0], s[qt][2 * c + 1][1]),
                             pack2<T>(s[qt][2 * c + 1][2], s[qt][2 * c + 1][3])};
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) {
            const u32x2_t lo = vt_read<C::KROW>(sv, 32 * c + vrow, vrow & C::SWZ, dt, frow);
            const u32x2_t hi = vt_read<C::KROW>(sv, 32 * c + 16 + vrow, vrow & C::SWZ, dt, frow);
            const u32x4_t w = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
              if (qt < nqt) Mfma<T>::run(w, pf[qt], o[qt][dt]);
          }
        }
      } else {
#pragma unroll
        for (int kt = 0; kt < NT; ++kt)
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) {
            u32x4_t w;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int key = 16 * kt + 4 * g + j, d = 16 * dt + frow;
              w[j] = *reinterpret_cast<const uint32_t*>(sv + key * C::KROW + (((d >> 2) ^ vswz<T, C::CPR>(key)) << 4) +
                                                        4 * (d & 3));
            }
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
              if (qt < nqt) {
                const u32x4_t pf = {__float_as_uint(s[qt][kt][0]), __float_as_uint(s[qt][kt][1]),
                                    __float_as_uint(s[qt][kt][2]), __float_as_uint(s[qt][kt][3])};
                Mfma<T>::run(w, pf, o[qt][dt]);
              }
          }
      }
      asm volatile("" ::: "memory");
    };
    if (cnt > 0) {
      int pg[NT];
      fetch(0, pg);
      load(0, pg, kf, vf);
      fetch(1, pg);
#pragma unroll 1
      for (int i = 0; i < cnt; ++i) {
        u32x4_t kn[NT][NKS], vn[NT][NKS];
        if (i + 1 < cnt) {
          int pn[NT];
          fetch(i + 2, pn);
          load(i + 1, pg, kn, vn);
#pragma unroll
          for (int kt = 0; kt < NT; ++kt) pg[kt] = pn[kt];
        }
        compute(sub0 + i * UK, kf, vf);
#pragma unroll
        for (int kt = 0; kt < NT; ++kt)
#pragma unroll
          for (int ks = 0; ks < NKS; ++ks) {
            kf[kt][ks] = kn[kt][ks];
            vf[kt][ks] = vn[kt][ks];
          }
      }
    }

    // ---- values that are not finite in masked subtiles: key by key, rarely
    if (__builtin_expect(odd_from < n, 0)) {
      float nm[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) nm[qt] = m_run[qt] == -INFINITY ? 0.f : -m_run[qt];
      for (int i = 0; i < cnt; ++i) {
        const int base = sub0 + i * UK;
        // Subtiles that no row was masked in have their values in O already.
        bool masked = base < kb;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
          if (qt < nqt) masked |= __builtin_amdgcn_ballot_w64(lim[qt] < base + KT - 1) != 0;
        if (!masked) continue;
        for (int key = max(base, kb); key < min(base + KT, n); ++key) {
          const int slot = key - a.seq.page.div(key) * page_size;
          int p = (WHOLE && key < a.prefix_len ? a.prefix : trow)[a.seq.page.div(key)];
          if (static_cast<uint32_t>(p) >= static_cast<uint32_t>(a.seq.n_pages)) p = 0;
          add_odd_key<T, HD, QT>(kh + p * a.kc.sp + slot * a.kc.ss, vh + p * a.vc.sp + slot * a.vc.ss, key, g,
                                 a.scale_log2, lim, qf, nm, o);
        }
      }
    }

    // ---- the waves' parts joined
    const bool whole = t0 == 0 && t1 == kt_item;
    const int slot = 2 * blockIdx.x + (t0 == 0 ? 1 : 0);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      if (qt >= nqt) break;
      const float l = column_sum(l_run[qt]);
      if (g == 0) {
        wave_m[wave][16 * qt + frow] = m_run[qt];
        wave_l[wave][16 * qt + frow] = l;
      }
    }
    for (int qt = 0; qt < nqt; ++qt) {
      __syncthreads();  // the maxima are there, the V tiles (or the rows before) are done with
      const int row = 16 * qt + frow;
      float m = wave_m[0][row];
#pragma unroll
      for (int w = 1; w < NW; ++w) m = fmaxf(m, wave_m[w][row]);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(wave_m[wave][row] - m);
      float* os = reinterpret_cast<float*>(sv);
#pragma unroll
      for (int q2 = 0; q2 < QT; ++q2)
        if (q2 == qt)
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) {
            const f32x4_t v = {o[q2][dt][0] * f, o[q2][dt][1] * f, o[q2][dt][2] * f, o[q2][dt][3] * f};
            *reinterpret_cast<f32x4_t*>(os + frow * HD + ((((4 * dt + g) ^ frow) & (HD / 4 - 1)) << 2)) = v;
          }
      __syncthreads();
      for (int i = tid; i < min(16, rows - r0 - 16 * qt) * (HD / 4); i += 64 * NW) {
        const int rr = i / (HD / 4), c = i % (HD / 4), r = r0 + 16 * qt + rr;
        const int wr = 16 * qt + rr;
        float mm = wave_m[0][wr];
#pragma unroll
        for (int w = 1; w < NW; ++w) mm = fmaxf(mm, wave_m[w][wr]);
        float l = 0.f;
        f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float* ow = reinterpret_cast<const float*>(smem + w * C::VBYTES);
          const f32x4_t x = *reinterpret_cast<const f32x4_t*>(ow + rr * HD + (((c ^ rr) & (HD / 4 - 1)) << 2));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += x[e];
          l += wave_l[w][wr] * (mm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(wave_m[w][wr] - mm));
        }
        const int tok = a.group.div(r), h = hk * G + r - tok * G, t = first + tok;
        if (WHOLE || (whole && a.prefix_len == 0)) {
          const float inv = l == 0.f ? 0.f : 1.0f / l;  // no key, or a NaN that stays one
          const float out[4] = {v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
          store4_out(static_cast<T*>(a.o) + t * a.o_st + h * a.o_sh + 4 * c, out);
        } else {
          float *ml, *ov;
          if (whole) {
            const int64_t at = (prefix ? 0 : static_cast<int64_t>(a.seq.n_tokens) * a.Hq) + static_cast<int64_t>(t) * a.Hq + h;
            ml = ws.whole_ml + 2 * at;
            ov = ws.whole_o + HD * at;
          } else {
            const int64_t at = static_cast<int64_t>(slot) * R + wr;
            ml = ws.edge_ml + 2 * at;
            ov = ws.edge_o + HD * at;
          }
          *reinterpret_cast<f32x4_t*>(ov + 4 * c) = v;
          if (c == 0) {
            ml[0] = mm;
            ml[1] = l;
          }
        }
      }
    }
    if constexpr (WHOLE) break;
    // ---- the next item
    u += t1 - t0;
    if (u >= u_end) break;
    t0 = 0;
    if (++rt == rts) {
      rt = 0;
      if (++hk == a.Hkv) {
        hk = 0;
        if (!enter_sequence()) break;
      }
    }
    __syncthreads();  // wave_m, wave_l and the tiles are free again
  }
  if (bad && a.err != nullptr) *a.err = 1;
}

// One wave, or with WAVES = 4 one block, a (token, head) row: its partials, each read by
// HD / 4 lanes, added group of lanes by group and then across the groups, always in the
// same order.  Rows that one block has written whole are left; rows without a key become
// zeros.
template <typename T, int HD, int R, int UK, int WAVES>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a, PagedWs ws, int prefix_units, int grid,
                                                         int n_tile) {
  constexpr int LP = HD / 4, GW = 64 / LP, NG = GW * WAVES;
  __shared__ float gm[WAVES], gl[WAVES];
  __shared__ __attribute__((aligned(16))) float go[WAVES][HD];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = WAVES == 1 ? static_cast<int>(blockIdx.x) * 4 + wave : static_cast<int>(blockIdx.x);
  if (row >= a.seq.n_tokens * a.Hq) return;
  const int t = row / a.Hq, h = row - t * a.Hq;
  const int G = static_cast<int>(a.group.d), hk = a.group.div(h);
  // Runs of partials: the splits of the tile kernel, or blocks [i0, i1] of an item, or one
  // whole row.
  int i0[2] = {0, 0}, n_part[2] = {n_tile, 0}, wr[2] = {0, 0};
  if (grid == 0) {
    if (a.seq.cu != nullptr && (t < a.seq.cu[0] || t >= a.seq.cu[a.seq.B])) return;
  } else {
    const int b = wave_seq_of(a.seq, t, lane);
    if (b >= a.seq.B) return;
    const SeqUnits su = seq_units<R, UK>(a, b, ws.unit_shift);
    if (t < su.first || t >= su.first + su.count) return;  // in front of the first sequence
    // A length past a table that names no key past the prefix: no block has units of it.
    if (su.kt == 0 && su.len > a.seq.cap && a.err != nullptr) *a.err = 1;
    const int U = ws.starts[a.seq.B], start = ws.starts[b];
    const Deal deal(grid, U);
    auto run = [&](int k, int from, int units, int r) {
      if (U <= 0) return;
      // (The bounds hold by themselves unless the lengths change under the call.)
      i0[k] = deal.owner(max(min(from, U - 1), 0));
      n_part[k] = deal.owner(max(min(from + units, U) - 1, 0)) - i0[k] + 1;
      wr[k] = r;
    };
    if (prefix_units > 0) {
      const int rows = a.seq.n_tokens * G, rts = (rows + R - 1) / R, kt = key_units<UK>(a.prefix_len, ws.unit_shift);
      const int r = t * G + h - hk * G;
      run(0, (hk * rts + r / R) * kt, kt, r % R);
    }
    if (su.kt > 0) {
      const int r = (t - su.first) * G + h - hk * G;
      run(1, start + (hk * su.rt + r / R) * su.kt, su.kt, r % R);
    }
    if (a.prefix_len == 0 && n_part[1] == 1) return;
  }
  const int lg = wave % WAVES * GW + lane / LP, c = lane % LP;
  float m = -INFINITY, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](float mi, float li, const f32x4_t& x) __attribute__((always_inline)) {
    const float mn = fmaxf(m, mi);
    const float fo = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    const float fi = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi - mn);
    m = mn;
    l = l * fo + li * fi;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * fo + x[e] * fi;
  };
  const int np = n_part[0] + n_part[1];
#pragma unroll 4
  for (int j = lg; j < np; j += NG) {
    const int k = j < n_part[0] ? 0 : 1, i = j - (k ? n_part[0] : 0);
    const float *ml, *ov;
    if (k == 0 && n_tile > 0) {
      const int64_t at = static_cast<int64_t>(i) * a.seq.n_tokens * a.Hq + row;
      ml = ws.tile_ml + 2 * at;
      ov = ws.tile_o + HD * at;
    } else if (n_part[k] == 1) {
      const int64_t at = (k ? static_cast<int64_t>(a.seq.n_tokens) * a.Hq : 0) + row;
      ml = ws.whole_ml + 2 * at;
      ov = ws.whole_o + HD * at;
    } else {
      const int64_t at = static_cast<int64_t>(2 * (i0[k] + i) + (i == 0 ? 1 : 0)) * R + wr[k];
      ml = ws.edge_ml + 2 * at;
      ov = ws.edge_o + HD * at;
    }
    add(ml[0], ml[1], *reinterpret_cast<const f32x4_t*>(ov + 4 * c));
  }
#pragma unroll
  for (int off = LP; off < 64; off <<= 1) {
    const float mi = __shfl_xor(m, off, 64), li = __shfl_xor(l, off, 64);
    const f32x4_t x = {__shfl_xor(o[0], off, 64), __shfl_xor(o[1], off, 64), __shfl_xor(o[2], off, 64),
                       __shfl_xor(o[3], off, 64)};
    add(mi, li, x);
  }
  if constexpr (WAVES > 1) {
    if (lane == 0) {
      gm[wave] = m;
      gl[wave] = l;
    }
    if (lane < LP) *reinterpret_cast<f32x4_t*>(&go[wave][4 * c]) = o;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) add(gm[w], gl[w], *reinterpret_cast<const f32x4_t*>(&go[w][4 * c]));
  }
  if (lane >= LP) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // no key, or a NaN that stays one
  const float out[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  store4_out(static_cast<T*>(a.o) + t * a.o_st + h * a.o_sh + 4 * c, out);
}

// ------------------------------------------------------------------------- host

// What a call runs: the tile kernel on the sequences' rows or on all rows against the
// prefix, the stream kernel, and the join.  Workspace offsets in bytes.
struct PagedPlan {
  bool whole = false;               // stream kernel, a block an item
  int tile_qt = 1, flat_split = 0, split = 0, n_tile = 0;  // tile kernel, and its partials a row
  int stream_qt = 0, grid = 0, prefix_units = 0, unit_shift = 0;  // stream kernel (stream_qt 0: none)
  int64_t o_starts = 0, o_eml = 0, o_eo = 0, o_wml = 0, o_wo = 0, o_tml = 0, o_to = 0, bytes = 0;
};

// A block that takes a whole item has as many waves as the registers allow.  It saves the
// second launch (B x heads sequences of 256 keys, head_dim 64: 1 x 12 13 -> 9.6 us,
// 16 x 12 15 -> 10.3, 16 x 25 17.7 -> 16.4, but 32 x 25 23 -> 28; head_dim 128: 8 x 8 15 ->
// 11, 128 x 8 43 -> 39) while an item takes its waves few rounds: with few items and more
// than two rounds the split over blocks is faster (1 x 12 of 2048 keys: 23 us whole, 15
// split; 16 x 12: 26 and 32).  A prefix is then read again by every sequence, up to
// kWholeAgain bytes.
constexpr int whole_waves(int hd) { return hd == 128 ? 8 : 16; }
constexpr int64_t kWholeKeys = 2048, kWholeAgain = int64_t{16} << 20;
// Rows of a sequence up to which it shares the reading of a prefix: tiles filled by all
// sequences and keys that stay in the L2s, against partials written and joined (32
// sequences, 12 heads of head_dim 64: 63 rows each behind 1024 keys 60 us alone, 52 shared;
// 104 rows 58 and 63; behind 16384 keys 255 rows 794 and 707, 455 rows 681 and 694; 8 heads
// of 128, 255 rows behind 512 keys 97 and 113, 2048 keys 216 and 176, 16384 keys 1349 and 740).
constexpr int64_t shared_rows(int64_t prefix_len, int hd) {
  const int64_t r = prefix_len * hd / 1024;
  return r < 96 ? 96 : r > 4 * hd ? 4 * hd : r;
}
constexpr int64_t kOwnKeys = 4096;
// Where the fp32 products are the bound and a tile's empty rows cost: from head_dim 64 on.
template <typename T, int HD> constexpr bool kDear = sizeof(T) == 4 && HD >= 64;

template <typename T, int HD>
static int make_plan(const cgpt_paged_args& call, PagedPlan* p) {
  const int64_t n_tokens = call.n_tokens, B = call.B, Hq = call.Hq, Hkv = call.Hkv, prefix_len = call.prefix_len;
  const int64_t cap = call.page_size * call.max_pages, rows = n_tokens * (Hq / Hkv), cus = num_cus();
  auto take = [&](int64_t bytes) {
    const int64_t o = p->bytes;
    p->bytes += (bytes + 63) / 64 * 64;
    return o;
  };
  // Short sequences: one launch, as long as the items do not crowd the card.  The plan goes by
  // what the workspace's question holds, the sizes: as many tokens as sequences count as one
  // each, with offsets too; only the grid has slots for any spread of them (see slot_seq).
  const int64_t spread = Hkv * (rows / 16 + B);
  const int64_t items = n_tokens == B && Hq / Hkv <= 16 ? Hkv * B : spread;
  const int64_t again = prefix_len * Hkv * HD * static_cast<int64_t>(sizeof(T)) * 2 * (B - 1);
  const int64_t most = 2 * items >= cus ? kWholeKeys : 5 * StreamShape<T, HD, 1, whole_waves(HD)>::UK / 2;
  if (rows <= 16 * B && cap <= most && (HD == 128 || 2 * items <= 3 * cus) && again <= kWholeAgain &&
      spread * whole_waves(HD) <= 4 * kMaxBlocks) {
    p->whole = true;
    p->grid = static_cast<int>(call.cu_q == nullptr ? items : spread);
    return CGPT_OK;
  }
  // Rows that the tile kernel takes: more than 16 a sequence, or a batch's against a prefix.
  // Where empty rows cost, more than 32 a sequence (100 sequences of up to 2000 keys, 1 to 2
  // tokens, 16 heads to a key head of 64: 120 us by the stream kernel, 173 in tiles; 24 of up
  // to 64 tokens behind 2048, 12 heads: 144 and 89), or a full tile of rows against 1024 keys
  // (20 rows, 12 heads, 16000 keys: 46 and 58; 100 rows, 500 keys: 36 and 45; 64 rows, 25
  // heads, 4096 keys: 116 and 89).
  constexpr bool dear = kDear<T, HD>;
  const bool tall = rows > (dear ? 32 : 16) * B;
  if (tall || (prefix_len > 0 && (dear ? rows >= 64 && prefix_len >= 1024 : rows > 16))) {
    const bool flat = prefix_len > 0 && rows <= shared_rows(prefix_len, HD) * B;
    auto blocks = [&](int64_t bq) { return Hkv * (flat ? (rows + bq - 1) / bq : rows / bq + B); };
    // 128-row tiles where there are four of them a CU, or at head_dim 128 against a prefix
    // (32768 keys, 512 rows a head: 188 us, 218 in tiles of 64; at head_dim 64 tiles of 64
    // rows win up to 2048 rows, 61 us against 65; fp32 tiles that sequences leave half empty
    // too: 24 of up to 64 tokens behind 2048 keys, 12 heads 190 us, 174 in tiles of 64), else
    // 64.  The keys are split, 256 a part at least (fp32 from head_dim 64 on 128: 64 tokens
    // behind 1000 keys, 12 heads of 128 34 -> 23 us), while a CU has fewer than six blocks of
    // own rows (16 prompts of up to 128 tokens, 12 heads of head_dim 64: 55 us whole, 43 in 3
    // parts; of up to 512: 67 whole, 86 in 2) or the resident number of prefix rows, whose
    // partials are many.  Keys are those that the table's width allows: a wide table of short
    // sequences has parts without a key (24 of up to 64 tokens behind 2048 keys, 12 heads: 30
    // us, 32 with a table eight times as wide as needed).
    p->tile_qt = blocks(128) >= 4 * cus || (flat && HD == 128 && rows > 128 && (!dear || !tall || rows >= 128 * B)) ? 2 : 1;
    const int64_t BQ = 64 * p->tile_qt;
    auto parts = [&](int64_t n, int64_t room, int64_t of) {
      return static_cast<int>(std::max<int64_t>(1, std::min(room * cus / n, of / (dear ? 128 : 256))));
    };
    // A sequence's own keys behind a prefix go by the same launch, even for a single row
    // (64 sequences, 25 heads, 4096 keys shared: 64 keys of their own 42 -> 36 us, 512 69 ->
    // 60, 2048 159 -> 153), unless its tiles have 128 rows (128 sequences, 8 heads of
    // head_dim 128, 2048 keys: 226 us, 211 by the stream kernel) or one sequence may, by the
    // table's width, have so many that its few blocks end last (the launch more where it has
    // not: 64 sequences behind 4096 keys 40 us, 50 with a table twice as wide as needed).
    const bool own = tall || (flat && !dear && p->tile_qt == 1 && cap - prefix_len <= kOwnKeys);
    const int64_t n_own = Hkv * (rows / BQ + B);
    if (flat) p->flat_split = parts(blocks(BQ), HD <= 64 ? 4 : 2, prefix_len);
    if (own) p->split = parts(n_own, 6, cap - (flat ? prefix_len : 0));
    // (head_blocks rounds the heads' blocks up by fewer than 8 a kind.)
    if ((flat ? blocks(BQ) : 0) * p->flat_split + n_own * p->split > kMaxBlocks - 16) return CGPT_ESHAPE;
    p->n_tile = flat || p->split > 1 ? p->flat_split + p->split : 0;
    p->o_tml = take(p->n_tile * n_tokens * Hq * 8);
    p->o_to = take(p->n_tile * n_tokens * Hq * HD * 4);
  }
  if (p->split == 0) {
    // 64-row tiles (32 at head_dim 128, whose accumulators are twice as wide) where a
    // sequence, or the batch against its prefix, has more than 16 rows a key head.
    const bool flat = p->flat_split > 0, wide = kDear<T, HD> && !flat && (prefix_len > 0 ? rows > 16 : rows > 16 * B);
    p->stream_qt = wide ? (HD == 128 ? 2 : 4) : 1;
    const int64_t R = 16 * p->stream_qt;
    const int64_t UK = wide ? StreamShape<T, HD, 1, 4>::UK : StreamShape<T, HD, 1, stream_waves(HD)>::UK;
    // Units as large as keep their number, had every sequence the length that the table
    // allows, within 32 bits.
    if (Hkv * (rows / R + B) > 0x7fffffff) return CGPT_ESHAPE;
    int64_t pu = 0, own = 0;
    for (;; ++p->unit_shift) {
      const int64_t unit = UK << p->unit_shift;
      if (unit > int64_t{1} << 30) return CGPT_ESHAPE;
      pu = prefix_len > 0 && !flat ? Hkv * ((rows + R - 1) / R) * ((prefix_len + unit - 1) / unit) : 0;
      own = Hkv * (rows / R + B) * ((cap - (prefix_len & ~int64_t{15}) + unit - 1) / unit);
      if (pu + own <= 0x7fffffff) break;
    }
    // Eight waves a CU; four of the widest, which need more registers than two a SIMD
    // leave (fp32, 8 x 512 tokens: 712 us with spills, 321 without).
    const int64_t per_cu = HD == 128 ? (wide ? 1 : 2) : wide ? 2 : 8;
    p->grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(pu + own, per_cu * cus)));
    p->prefix_units = static_cast<int>(pu);
    p->o_starts = take((B + 1) * 4);
    p->o_eml = take(int64_t{p->grid} * 2 * R * 8);
    p->o_eo = take(int64_t{p->grid} * 2 * R * HD * 4);
    p->o_wml = take(prefix_len > 0 ? 2 * n_tokens * Hq * 8 : 0);
    p->o_wo = take(prefix_len > 0 ? 2 * n_tokens * Hq * HD * 4 : 0);
  }
  // The join: four rows a block.
  if ((p->split == 0 || p->n_tile > 0) && n_tokens * Hq > 4 * kMaxBlocks) return CGPT_ESHAPE;
  return CGPT_OK;
}

template <typename T, int HD, int QTW, int NW, bool WHOLE>
static void launch_stream(const PagedAttnArgs& a, const PagedWs& ws, const PagedPlan& p, hipStream_t s) {
  const bool a16 = a.seq.page.d % 16 == 0 && (!WHOLE || a.prefix_len % 16 == 0) && short_rows(a);
  if (a16)
    hipLaunchKernelGGL((paged_stream_kernel<T, HD, QTW, true, NW, WHOLE>), dim3(p.grid), dim3(64 * NW), 0, s, a, ws,
                       p.prefix_units);
  else
    hipLaunchKernelGGL((paged_stream_kernel<T, HD, QTW, false, NW, WHOLE>), dim3(p.grid), dim3(64 * NW), 0, s, a, ws,
                       p.prefix_units);
}

template <typename T, int HD, int QTW, int NW>
static void launch_join(const PagedAttnArgs& a, const PagedWs& ws, const PagedPlan& p, hipStream_t s) {
  using C = StreamShape<T, HD, QTW, NW>;
  const int rows = a.seq.n_tokens * a.Hq;
  // Few rows have many partials each; many rows want many of them on a CU, since each
  // is a chain of dependent loads (10 thousand rows of two partials: 16 us a block
  // each, 5 us a wave each).
  if (rows < 4 * num_cus())
    hipLaunchKernelGGL((paged_join_kernel<T, HD, C::R, C::UK, 4>), dim3(rows), dim3(256), 0, s, a, ws, p.prefix_units,
                       p.grid, p.n_tile);
  else
    hipLaunchKernelGGL((paged_join_kernel<T, HD, C::R, C::UK, 1>), dim3((rows + 3) / 4), dim3(256), 0, s, a, ws,
                       p.prefix_units, p.grid, p.n_tile);
}

template <typename T, int HD>
static int run_plan(const PagedAttnArgs& a, const cgpt_paged_args& call, hipStream_t s) {
  PagedPlan p;
  int rc = make_plan<T, HD>(call, &p);
  if (rc != CGPT_OK) return rc;
  char* w = static_cast<char*>(call.workspace);
  if (p.bytes > 0 && (call.workspace_bytes < p.bytes || w == nullptr)) return CGPT_ESCRATCH;
  if (reinterpret_cast<uintptr_t>(w) & 15) return CGPT_EINVAL;
  auto f32 = [&](int64_t o) { return reinterpret_cast<float*>(w + o); };
  const PagedWs ws{reinterpret_cast<int*>(w + p.o_starts), f32(p.o_eml), f32(p.o_eo), f32(p.o_wml), f32(p.o_wo),
                   f32(p.o_tml), f32(p.o_to), p.unit_shift};
  if (p.flat_split + p.split > 0) {
    TileJob job{};
    if (p.n_tile > 0) {
      job.ml = ws.tile_ml;
      job.o = ws.tile_o;
    }
    job.flat_split = p.flat_split;
    job.split = p.split;
    job.from = p.flat_split > 0 ? a.prefix_len : 0;
    rc = launch_paged_tile(call.dtype, HD, a, job, p.tile_qt, s);
    if (rc != CGPT_OK) return rc;
  }
  if (p.whole) {
    launch_stream<T, HD, 1, whole_waves(HD), true>(a, ws, p, s);
    return hip_status(hipGetLastError());
  }
  if constexpr (kDear<T, HD>) {
    if (p.stream_qt > 1) {
      constexpr int QT = HD == 128 ? 2 : 4;
      launch_stream<T, HD, QT, 4, false>(a, ws, p, s);
      launch_join<T, HD, QT, 4>(a, ws, p, s);
    }
  }
  if (p.stream_qt == 1) launch_stream<T, HD, 1, stream_waves(HD), false>(a, ws, p, s);
  if (p.stream_qt == 1 || (p.stream_qt == 0 && p.n_tile > 0)) launch_join<T, HD, 1, stream_waves(HD)>(a, ws, p, s);
  return hip_status(hipGetLastError());
}

template <typename F>
static int with_type(const cgpt_paged_args& p, F&& f) {
#define CGPT_PAGED_HD(T)                                                \
  switch (p.head_dim) {                                                 \
    case 16: return f(T{}, std::integral_constant<int, 16>{});          \
    case 32: return f(T{}, std::integral_constant<int, 32>{});          \
    case 64: return f(T{}, std::integral_constant<int, 64>{});          \
    case 128: return f(T{}, std::integral_constant<int, 128>{});        \
    default: return CGPT_ESHAPE;                                        \
  }
  if (p.dtype == CGPT_BF16) CGPT_PAGED_HD(bf16_t)
  if (p.dtype == CGPT_F16) CGPT_PAGED_HD(f16_t)
  CGPT_PAGED_HD(float)
#undef CGPT_PAGED_HD
}

}  // namespace cgpt

extern "C" int cgpt_paged_attention(const cgpt_paged_args* args, void* stream) {
  using namespace cgpt;
  bool empty;
  const int rc = check_paged(args, false, &empty);
  if (rc != CGPT_OK) return rc;
  const cgpt_paged_args& p = *args;
  const float scale = static_cast<float>(p.scale), scale_log2 = scale * 1.4426950408889634f;
  if (p.prefix_len < 0 || p.prefix_len > p.page_size * p.max_pages || !(scale > 0.f) || !(scale_log2 < INFINITY))
    return CGPT_EINVAL;
  if (empty) return CGPT_OK;
  if (p.q == nullptr || p.out == nullptr || (p.prefix_len > 0 && p.prefix_pages == nullptr)) return CGPT_EINVAL;
  const PagedAttnArgs a{p.q, p.out, PagePool{p.k_cache, p.kc_sp, p.kc_sh, p.kc_ss},
                        PagePool{p.v_cache, p.vc_sp, p.vc_sh, p.vc_ss}, paged_batch(p), p.prefix_pages,
                        static_cast<int>(p.prefix_len), p.q_st, p.q_sh, p.out_st, p.out_sh, static_cast<int>(p.Hq),
                        static_cast<int>(p.Hkv), FastDiv(p.Hq / p.Hkv), scale_log2, p.err_flag};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(p, [&](auto t, auto hd) {
    return run_plan<decltype(t), decltype(hd)::value>(a, p, s);
  });
}

extern "C" int cgpt_paged_attention_workspace(const cgpt_paged_args* args, int64_t* workspace_bytes) {
  using namespace cgpt;
  if (args == nullptr || workspace_bytes == nullptr) return CGPT_EINVAL;
  *workspace_bytes = 0;
  const cgpt_paged_args& p = *args;
  const int rc = check_sizes(p);
  if (rc != CGPT_OK) return rc;
  if (p.prefix_len < 0 || p.prefix_len > p.page_size * p.max_pages) return CGPT_EINVAL;
  if (p.n_tokens == 0 || p.B == 0) return CGPT_OK;
  return with_type(p, [&](auto t, auto hd) {
    PagedPlan plan;
    const int rc = make_plan<decltype(t), decltype(hd)::value>(p, &plan);
    if (rc == CGPT_OK) *workspace_bytes = plan.bytes;
    return rc;
  });
}
