// Attention over the 8-bit paged cache.
//
// o[i, h] = softmax(scale q[i, h] K^T) V over the keys 0 .. pos(i) of token i's sequence,
// K and V being code * 2^e, in base 2 and one pass over the keys with a running shift, as in
// paged_attention.hip.
//
// A cached value is exact in bf16 (see paged8.h), so the products run on the bf16 matrix cores
// whatever the queries' type, and a query or a weight of more bits goes in as the sum of its
// bf16 parts: one for bf16, two for fp16 (8 + 8 bits hold its 11), three for fp32 (24).  All
// types so have bf16's range on the way, and fp32 costs three products, not the sixteen times
// that the fp32 matrix instruction takes.  A weight is rounded to its parts (2^-8, 2^-17 or
// 2^-26 relative) for the second product, where the result is rounded to the queries' type
// as coarsely (bf16: results are 0.0019 off in all, 0.0017 with exact weights; a second part
// would be a second product and five instructions a pair of weights more); sums, maxima and the
// shift are fp32.
//
// Two kernels, the stream kernel here for few rows (a decode step reads every key once: the
// bound is HBM) and the tile kernel (paged8_tile.hip) for more than 16 a sequence and head; make_plan8
// chooses, by the whole call's rows a sequence: where one long chunk comes with many single tokens
// its keys are read once for every 16 of its rows (63 single tokens behind 500 to 4000 keys 65 to
// 70 us, 500 tokens behind 3000 keys 35, both in one call 113).
//
// 64 sequences of 1 to 8192 keys, 25 heads of 64: int8 158 to 163 us, 5.1 to 5.3 TB/s, e4m3
// 153 to 155, where the 16-bit cache takes 295 (queries in fp32: 192 and 176); four of 90 to 130
// thousand, 8 heads of 128, e4m3, fp16 173 us, 5.2 TB/s (308 in 16 bits).  With heads of 32, half
// the bytes, int8 142 us and e4m3 134 (3.0 and 3.1 TB/s), of 16 147 and 133: the instructions a key
// costs hardly shrink with it (vector ones 5.4 of a wave, 6.5 at 64; scalar 6.2 and 6.2), and no
// unit is busy throughout (VALU 42 %, 1.5 waves a SIMD).  One sequence of 500 keys: 7.4 us.
#include <algorithm>

#include "internal.h"
#include "paged8.h"
#include "paged_units.h"

namespace cgpt {

template <int HD, int NW>
struct Shape8 {
  static constexpr int LB = HD >= 64 ? 16 : 8;                 // bytes of a lane's load
  static constexpr int NL = HD == 128 ? 2 : 1;                 // loads of a row and lane
  static constexpr int NS = HD >= 32 ? HD / 32 : 1;            // 32-wide slabs of a product
  static constexpr int ND = HD / 16;
  static constexpr int NT = HD == 128 ? 4 : NW == 1 ? 8 : 4;   // 16-key tiles a wave takes at once
  static constexpr int KT = 16 * NT;
  static constexpr int UK = NW * KT;                           // keys of a unit, KT a wave
  static constexpr int R = 16;
  static constexpr int KROW = 2 * HD;                          // a V row in LDS, as bf16
  static constexpr int SWZ = (HD / 8 < 8 ? HD / 8 : 8) - 1;    // its chunks are swizzled by the key
  static constexpr int VBYTES = KT * KROW;
  // First value that lane group g has in slab s: a lane's 16 codes are halves of two slabs.
  __device__ static constexpr int dim(int s, int g) { return HD >= 64 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 8 * g; }
  static_assert(VBYTES >= 16 * HD * 4, "the join of the waves reuses the V tiles");
};

constexpr int stream_waves8(int hd) { return hd == 128 ? 4 : 1; }

// As the stream kernel of paged_attention.hip: each wave streams keys by itself, K and V rows
// from their pages into registers one subtile of KT keys ahead of the one in use, S^T = K Q^T
// from registers, V through the wave's own LDS tile (as bf16) for its transpose.  WHOLE: a
// block is one item with all its keys.  A16: 16 keys from a multiple of 16 on lie in one page and
// block of the exponents: page ids come by scalar loads; else every lane looks its own key up.
// (Exponents by scalar loads would make every LDS read wait for them: 64 sequences of up to 8192
// keys, 25 heads of 64, e4m3 188 us so, 172 now.)
// The exponents: e4m3's go into the conversion to bf16; int8's would cost a product a value
// there, so with one exponent a tile (A16) they go to the scores' scale and the weights instead.
template <typename T, int CODE, int HD, bool A16, int NW, bool WHOLE>
__global__ __launch_bounds__(64 * NW, NW == 16 ? 4 : 2) void
paged8_stream_kernel(PagedAttnArgs a, Paged8 quant, PagedWs ws) {
  using C = Shape8<HD, NW>;
  constexpr int NT = C::NT, NL = C::NL, NS = C::NS, ND = C::ND, KT = C::KT, UK = C::UK, R = C::R, NP = kParts<T>;
  constexpr bool FOLD = A16 && CODE == CGPT_INT8;
  typedef std::conditional_t<C::LB == 16, u32x4_t, u32x2_t> chunk_t;
  __shared__ __attribute__((aligned(16))) uint8_t smem[NW * C::VBYTES];
  __shared__ float wave_m[NW][R], wave_l[NW][R];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int g = lane >> 4, frow = lane & 15;
  const int G = static_cast<int>(a.group.d), page_size = static_cast<int>(a.seq.page.d);
  uint8_t* const sv = smem + wave * C::VBYTES;
  bool bad = false;

  // Units of up to 64 sequences from c0 on: lane l holds sequence c0 + l.  `before` counts
  // the units in front of them.
  int c0 = 0, n_units = 0, incl = 0, before = 0, total = 0;
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
  // The item at hand: rows of tile rt of key head hk, keys [0, n), cut into kt_item units; t0 is
  // its first unit here.
  int u = 0, u_end = 1, hk = 0, rt = 0, rts = 1, t0 = 0, kt_item = 0, n_all = 0, rows = 0, first = 0, pos0 = 0;
  const int* trow = nullptr;
  // The sequence whose units u lies in; false when there is none (the lengths changed
  // under the call).
  auto enter_sequence = [&]() __attribute__((always_inline)) {
    if (per > 1) {
      const int gi = __popcll(__builtin_amdgcn_ballot_w64(group_incl <= u));
      if (gi >= 64) return false;
      const int end = min((gi + 1) * per, a.seq.B);
      before = __builtin_amdgcn_readlane(group_incl - group_units, gi);
      for (load_chunk(gi * per, end); u >= before + total; load_chunk(c0 + 64, end)) {
        if (c0 + 64 >= end) return false;
        before += total;
      }
    }
    if (u >= before + total) return false;
    const int at = __popcll(__builtin_amdgcn_ballot_w64(before + incl <= u));
    auto of = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, at); };
    rts = of(mine.rt);
    kt_item = of(mine.kt);
    t0 = u - before - of(incl - n_units);  // units into the sequence
    n_all = of(mine.n);
    first = of(mine.first);
    const int count = of(mine.count), len = of(mine.len);
    rows = count * G;
    pos0 = len - count;
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
      if (writes && lane < a.seq.B) ws.starts[lane] = incl - n_units;
    } else {
      const int first_b = lane * per, end_b = min(first_b + per, a.seq.B);
#pragma unroll 4
      for (int b = first_b; b < end_b; ++b) {
        const SeqUnits su = seq_units<R, UK>(a, b, ws.unit_shift);
        group_units += su.rt * su.kt * a.Hkv;
      }
      group_incl = scan(group_units);
      if (writes) {
        int at = group_incl - group_units;
        for (int b = first_b; b < end_b; ++b) {
          const SeqUnits su = seq_units<R, UK>(a, b, ws.unit_shift);
          ws.starts[b] = at;
          at += su.rt * su.kt * a.Hkv;
        }
      }
    }
    const int U = __builtin_amdgcn_readlane(group_incl, 63);
    if (blockIdx.x == 0 && tid == 0) ws.starts[a.seq.B] = U;
    const Deal deal(gridDim.x, U);
    if (static_cast<int>(blockIdx.x) >= deal.g || U == 0) return;
    u = deal.start(blockIdx.x);
    u_end = deal.start(blockIdx.x + 1);
    if (!enter_sequence()) return;
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
    const int n = min(n_all, max(pos0 + a.group.div(min(rt * R + R, rows) - 1) + 1, 0));
    if constexpr (WHOLE) kt_item = (n + UK - 1) / UK;
    const int t1 = WHOLE ? kt_item : min(kt_item, t0 + (u_end - u));

    // ---- its rows: lane (g, frow) works for row rt R + frow
    const int r0 = rt * R;
    int lim;  // last key the row sees; rows that do not exist are never masked
    u32x4_t qf[NS][NP];
    {
      const int r = r0 + frow;
      const bool live = r < rows;
      const int i = a.group.div(live ? r : 0), h = hk * G + (live ? r : 0) - i * G;
      lim = live ? min(pos0 + i, n - 1) : 0x7fffffff;
      const T* qp = static_cast<const T*>(a.q) + (first + i) * a.q_st + h * a.q_sh;
      const bool has = live && (HD > 16 || g < 2);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e += Elem<T>::kVec) load_vec(qp + C::dim(s, HD > 16 ? g : g & 1) + e, x + e);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = has ? x[e] : 0.f;
        split_parts<NP>(x, qf[s]);
      }
    }
    f32x4_t o[ND];
    float m_run = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) o[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    // ---- its keys
    const uint8_t* const kh = static_cast<const uint8_t*>(a.kc.base) + hk * a.kc.sh;
    const uint8_t* const vh = static_cast<const uint8_t*>(a.vc.base) + hk * a.vc.sh;
    const uint8_t* const ksh = quant.ks.base + hk * quant.ks.sh;
    const uint8_t* const vsh = quant.vs.base + hk * quant.vs.sh;
    const int shift = WHOLE ? 0 : ws.unit_shift;
    const int sub0 = ((t0 * UK) << shift) + wave * KT;  // first subtile; the next is UK further
    const int cnt = sub0 < n ? min((t1 - t0) << shift, (n - sub0 + UK - 1) / UK) : 0;
    int odd_from = 0x7fffffff;  // first masked subtile of the wave with a value that is no number
    chunk_t kf[NT][NL], vf[NT][NL];
    int kx[NT], vx[NT];  // exponent bytes
    // Pages of subtile i: one a 16-key tile, or one a lane's key.
    auto fetch = [&](int i, int (&pg)[NT]) __attribute__((always_inline)) {
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        const int tile = sub0 + i * UK + 16 * kt;
        if (A16) {
          const int col = a.seq.page.div(min(tile, (n - 1) & ~15));
          pg[kt] = ((const __attribute__((address_space(4))) int*)trow)[__builtin_amdgcn_readfirstlane(col)];
        } else {
          pg[kt] = trow[a.seq.page.div(min(tile + frow, n - 1))];
        }
      }
    };
    // Past the caches, which have no use for a key that is read once (as all are but those of
    // sequences of more than 16 rows beside many short ones): 64 sequences of up to 8192 keys,
    // 25 heads of 64, int8 182 -> 169 us; but not rows of two loads, which share their lines (four of
    // 90 to 130 thousand keys, 8 heads of 128, 164 us, 174 so).
    auto read_once = [&](const chunk_t* p) __attribute__((always_inline)) {
      return HD == 128 ? *p : __builtin_nontemporal_load(p);
    };
    const uint32_t k_row = static_cast<uint32_t>(a.kc.ss), v_row = static_cast<uint32_t>(a.vc.ss);
    auto load = [&](int i, const int (&pg)[NT], chunk_t (&kd)[NT][NL], chunk_t (&vd)[NT][NL], int (&kxd)[NT], int (&vxd)[NT])
        __attribute__((always_inline)) {
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        const int tile = sub0 + i * UK + 16 * kt;
        const int key = A16 ? min(tile, (n - 1) & ~15) : min(tile + frow, n - 1);
        const int slot = key - a.seq.page.div(key) * page_size;
        int p = A16 ? __builtin_amdgcn_readfirstlane(pg[kt]) : pg[kt];
        if (static_cast<uint32_t>(p) >= static_cast<uint32_t>(a.seq.n_pages)) {
          p = 0;
          bad = true;
        }
        const uint8_t* const kp = kh + p * a.kc.sp + slot * a.kc.ss;
        const uint8_t* const vp = vh + p * a.vc.sp + slot * a.vc.ss;
        const int block = quant.block.div(A16 ? __builtin_amdgcn_readfirstlane(slot) : slot);
        const uint8_t* const ke = ksh + p * quant.ks.sp + block * quant.ks.sb;
        const uint8_t* const ve = vsh + p * quant.vs.sp + block * quant.vs.sb;
        kxd[kt] = *ke;
        vxd[kt] = *ve;
        uint32_t row = 0;
        if (A16) row = tile + 16 <= n ? frow : min(tile + frow, n - 1) - key;
        const uint32_t ko = row * k_row, vo = row * v_row;
        const int c = C::LB * (HD > 16 ? g : g & 1);
#pragma unroll
        for (int l = 0; l < NL; ++l) {
          kd[kt][l] = read_once(reinterpret_cast<const chunk_t*>(kp + (ko + c + 64 * l)));
          vd[kt][l] = read_once(reinterpret_cast<const chunk_t*>(vp + (vo + c + 64 * l)));
        }
        // Lanes past a short row's chunks: 0 x NaN would be NaN.
        if (HD == 16 && g >= 2) kd[kt][0] = chunk_t{};
      }
    };
    auto compute = [&](int base, const chunk_t (&kd)[NT][NL], const chunk_t (&vd)[NT][NL], const int (&kxd)[NT],
                       const int (&vxd)[NT]) __attribute__((always_inline)) {
      const bool masked = __builtin_amdgcn_ballot_w64(lim < base + KT - 1) != 0;
      // A masked key's weight is 0, but 0 x NaN is NaN: where a row is masked the matrix cores
      // get 0 for it, and it is added at the item's end to the rows that see it.
      uint32_t bits = 0;
      asm volatile("" ::: "memory");
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        const int key = 16 * kt + frow;
        const float f = FOLD ? 1.f : value_scale_of<CODE>(vxd[kt]);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          uint32_t w0 = vd[kt][s >> 1][2 * (s & 1)], w1 = vd[kt][s >> 1][2 * (s & 1) + 1];
          if (CODE == CGPT_E4M3 && masked) {
            const uint32_t n0 = nan_codes(w0), n1 = nan_codes(w1);
            bits |= n0 | n1;
            w0 &= ~((n0 >> 7) * 0xffu);
            w1 &= ~((n1 >> 7) * 0xffu);
          }
          const u32x2_t lo = bf16x4_of<CODE>(w0, f), hi = bf16x4_of<CODE>(w1, f);
          if (HD > 16 || g < 2)
            *reinterpret_cast<u32x4_t*>(sv + key * C::KROW + (((C::dim(s, g) >> 3) ^ (key & C::SWZ)) << 4)) =
                u32x4_t{lo[0], lo[1], hi[0], hi[1]};
        }
      }
      if (CODE == CGPT_E4M3 && masked && __builtin_amdgcn_ballot_w64(bits != 0) != 0) odd_from = min(odd_from, base);
      asm volatile("" ::: "memory");
      f32x4_t s[NT];
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        s[kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        const float f = FOLD ? 1.f : scale_of<CODE>(kxd[kt]);
#pragma unroll
        for (int sl = 0; sl < NS; ++sl) {
          const u32x2_t lo = bf16x4_of<CODE>(kd[kt][sl >> 1][2 * (sl & 1)], f);
          const u32x2_t hi = bf16x4_of<CODE>(kd[kt][sl >> 1][2 * (sl & 1) + 1], f);
          const u32x4_t w = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
          for (int p = 0; p < NP; ++p) Mfma<bf16_t>::run(w, qf[sl][p], s[kt]);
        }
      }
      if (masked) {
        const int hi = lim - base - 4 * g;
#pragma unroll
        for (int kt = 0; kt < NT; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[kt][r] = 16 * kt + r > hi ? -INFINITY : s[kt][r];
      }
      float fk[NT];  // what makes a tile's sums scores in base 2
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        fk[kt] = FOLD ? scale_of<CODE>(kxd[kt]) * a.scale_log2 : a.scale_log2;
        const float m = fmaxf(fmaxf(s[kt][0], s[kt][1]), fmaxf(s[kt][2], s[kt][3]));
        mx = fmaxf(mx, FOLD ? m * fk[kt] : m);
      }
      mx = column_max(mx) * (FOLD ? 1.f : a.scale_log2);
      // The shift moves only when the maximum outgrows it by more than 8, so P <= 2^8 and
      // the accumulators are rescaled on few subtiles.
      const bool grow = mx > m_run + 8.0f;
      if (__builtin_amdgcn_ballot_w64(grow) != 0) {
        const float m_new = grow ? mx : m_run;
        const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[dt][r] *= alpha;
      }
      const float shift = m_run == -INFINITY ? 0.f : -m_run;
      float sum = 0.f;
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        const float fv = FOLD ? value_scale_of<CODE>(vxd[kt]) : 1.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r], fk[kt], shift));
          sum += p;
          s[kt][r] = FOLD ? p * fv : p;
        }
      }
      l_run += sum;
      const int vrow = 4 * g + (frow >> 2);
#pragma unroll
      for (int c = 0; c < NT / 2; ++c) {
        const float p[8] = {s[2 * c][0], s[2 * c][1], s[2 * c][2], s[2 * c][3],
                            s[2 * c + 1][0], s[2 * c + 1][1], s[2 * c + 1][2], s[2 * c + 1][3]};
        u32x4_t pf[NP];
        split_parts<NP>(p, pf);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          const u32x2_t lo = vt_read<C::KROW>(sv, 32 * c + vrow, vrow & C::SWZ, dt, frow);
          const u32x2_t hi = vt_read<C::KROW>(sv, 32 * c + 16 + vrow, vrow & C::SWZ, dt, frow);
          const u32x4_t w = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
          for (int q = 0; q < NP; ++q) Mfma<bf16_t>::run(w, pf[q], o[dt]);
        }
      }
      asm volatile("" ::: "memory");
    };
    if (cnt > 0) {
      int pg[NT];
      fetch(0, pg);
      load(0, pg, kf, vf, kx, vx);
      fetch(1, pg);
#pragma unroll 1
      for (int i = 0; i < cnt; ++i) {
        chunk_t kn[NT][NL], vn[NT][NL];
        int kxn[NT], vxn[NT];
        if (i + 1 < cnt) {
          int pn[NT];
          fetch(i + 2, pn);
          load(i + 1, pg, kn, vn, kxn, vxn);
#pragma unroll
          for (int kt = 0; kt < NT; ++kt) pg[kt] = pn[kt];
        }
        compute(sub0 + i * UK, kf, vf, kx, vx);
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) {
          kx[kt] = kxn[kt];
          vx[kt] = vxn[kt];
#pragma unroll
          for (int l = 0; l < NL; ++l) {
            kf[kt][l] = kn[kt][l];
            vf[kt][l] = vn[kt][l];
          }
        }
      }
    }

    // ---- values that are no numbers in masked subtiles: key by key, rarely
    if (CODE == CGPT_E4M3 && __builtin_expect(odd_from < n, 0)) {
      for (int i = 0; i < cnt; ++i) {
        const int base = sub0 + i * UK;
        // Subtiles that no row was masked in have their values in O already.
        if (__builtin_amdgcn_ballot_w64(lim < base + KT - 1) == 0) continue;
        for (int key = base; key < min(base + KT, n); ++key) {
          const int col = a.seq.page.div(key), slot = key - col * page_size;
          int p = trow[col];
          if (static_cast<uint32_t>(p) >= static_cast<uint32_t>(a.seq.n_pages)) p = 0;
          const uint8_t* const v = vh + p * a.vc.sp + slot * a.vc.ss + 4 * g;
#pragma unroll
          for (int dt = 0; dt < ND; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if ((v[16 * dt + e] & 0x7f) == 0x7f && key <= lim) o[dt][e] = NAN;
        }
      }
    }

    // ---- the waves' parts joined
    const bool whole = t0 == 0 && t1 == kt_item;
    const int slot = 2 * blockIdx.x + (t0 == 0 ? 1 : 0);
    {
      const float l = column_sum(l_run) * kSumDrop;
      if (g == 0) {
        wave_m[wave][frow] = m_run;
        wave_l[wave][frow] = l;
      }
    }
    __syncthreads();  // the maxima are there, the V tiles are done with
    {
      float m = wave_m[0][frow];
#pragma unroll
      for (int w = 1; w < NW; ++w) m = fmaxf(m, wave_m[w][frow]);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(wave_m[wave][frow] - m);
      float* os = reinterpret_cast<float*>(sv);
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) {
        const f32x4_t v = {o[dt][0] * f, o[dt][1] * f, o[dt][2] * f, o[dt][3] * f};
        *reinterpret_cast<f32x4_t*>(os + frow * HD + ((((4 * dt + g) ^ frow) & (HD / 4 - 1)) << 2)) = v;
      }
    }
    __syncthreads();
    for (int i = tid; i < min(16, rows - r0) * (HD / 4); i += 64 * NW) {
      const int rr = i / (HD / 4), c = i % (HD / 4), r = r0 + rr;
      float mm = wave_m[0][rr];
#pragma unroll
      for (int w = 1; w < NW; ++w) mm = fmaxf(mm, wave_m[w][rr]);
      float l = 0.f;
      f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float* ow = reinterpret_cast<const float*>(smem + w * C::VBYTES);
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(ow + rr * HD + (((c ^ rr) & (HD / 4 - 1)) << 2));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += x[e];
        l += wave_l[w][rr] * (mm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(wave_m[w][rr] - mm));
      }
      const int tok = a.group.div(r), h = hk * G + r - tok * G, t = first + tok;
      if (WHOLE || whole) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;  // no key, or a NaN that stays one
        const float out[4] = {v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
        store4_out(static_cast<T*>(a.o) + t * a.o_st + h * a.o_sh + 4 * c, out);
      } else {
        const int64_t at = static_cast<int64_t>(slot) * R + rr;
        *reinterpret_cast<f32x4_t*>(ws.edge_o + HD * at + 4 * c) = v;
        if (c == 0) {
          ws.edge_ml[2 * at] = mm;
          ws.edge_ml[2 * at + 1] = l;
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

// ------------------------------------------------------------------------- host

// What a call runs: the tile kernel, or the stream kernel, and the join.  Workspace offsets in
// bytes.
struct Plan8 {
  bool whole = false;             // stream kernel, a block an item, no workspace
  int tile_qt = 0, split = 0;     // tile kernel (0: not at all), parts of the keys
  int grid = 0, unit_shift = 0;   // stream kernel
  int64_t o_starts = 0, o_ml = 0, o_o = 0, bytes = 0;
};

constexpr int whole_waves8(int hd) { return hd == 128 ? 8 : 16; }
constexpr int64_t kWholeKeys8 = 2048;

template <int HD> static int make_plan8(const cgpt_paged_args& call, Plan8* p) {
  const int64_t n_tokens = call.n_tokens, B = call.B, Hq = call.Hq, Hkv = call.Hkv;
  const int64_t cap = call.page_size * call.max_pages, rows = n_tokens * (Hq / Hkv), cus = num_cus();
  auto take = [&](int64_t bytes) {
    const int64_t o = p->bytes;
    p->bytes += (bytes + 63) / 64 * 64;
    return o;
  };
  // Short sequences: one launch, as long as the items do not crowd the card.
  const int64_t spread = Hkv * (rows / 16 + B);
  const int64_t items = n_tokens == B && Hq / Hkv <= 16 ? Hkv * B : spread;
  const int64_t most = 2 * items >= cus ? kWholeKeys8 : 5 * Shape8<HD, whole_waves8(HD)>::UK / 2;
  if (rows <= 16 * B && cap <= most && (HD == 128 || 2 * items <= 3 * cus) && spread * whole_waves8(HD) <= 4 * kMaxBlocks) {
    p->whole = true;
    p->grid = static_cast<int>(call.cu_q == nullptr ? items : spread);
    return CGPT_OK;
  }
  // The join: four rows a block.
  if (n_tokens * Hq > 4 * kMaxBlocks) return CGPT_ESHAPE;
  if (rows > 16 * B) {
    p->tile_qt = Hkv * (rows / 128 + B) >= 4 * cus ? 2 : 1;
    const int64_t tiles = Hkv * (rows / (64 * p->tile_qt) + B);
    p->split = static_cast<int>(std::max<int64_t>(1, std::min(6 * cus / tiles, cap / 256)));
    if (tiles * p->split > kMaxBlocks - 16) return CGPT_ESHAPE;
    if (p->split > 1) {
      p->o_ml = take(p->split * n_tokens * Hq * 8);
      p->o_o = take(p->split * n_tokens * Hq * HD * 4);
    }
    return CGPT_OK;
  }
  constexpr int64_t R = 16, UK = Shape8<HD, stream_waves8(HD)>::UK;
  // Units as large as keep their number, had every sequence the length that the table
  // allows, within 32 bits.
  if (spread > 0x7fffffff) return CGPT_ESHAPE;
  int64_t units = 0;
  for (;; ++p->unit_shift) {
    const int64_t unit = UK << p->unit_shift;
    if (unit > int64_t{1} << 30) return CGPT_ESHAPE;
    units = spread * ((cap + unit - 1) / unit);
    if (units <= 0x7fffffff) break;
  }
  const int64_t per_cu = HD == 128 ? 2 : 8;
  p->grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(units, per_cu * cus)));
  p->o_starts = take((B + 1) * 4);
  p->o_ml = take(int64_t{p->grid} * 2 * R * 8);
  p->o_o = take(int64_t{p->grid} * 2 * R * HD * 4);
  return CGPT_OK;
}

template <typename T, int CODE, int HD, int NW, bool WHOLE>
static void launch_stream8(const PagedAttnArgs& a, const Paged8& quant, const PagedWs& ws, const Plan8& p, hipStream_t s) {
  // Offsets of 16 slots fit 32 bits; and where a tile's exponent and the scale become one factor
  // (int8), it is a normal float whatever the exponent, -100 to 121: else a masked key's
  // -inf x 0 or a zero key's 0 x inf would be a NaN.
  const bool one_factor = CODE != CGPT_INT8 || (a.scale_log2 >= 0x1p-26f && a.scale_log2 <= 0x1p6f);
  if (quant.block.d % 16 == 0 && short_rows(a) && one_factor)
    hipLaunchKernelGGL((paged8_stream_kernel<T, CODE, HD, true, NW, WHOLE>), dim3(p.grid), dim3(64 * NW), 0, s, a, quant, ws);
  else
    hipLaunchKernelGGL((paged8_stream_kernel<T, CODE, HD, false, NW, WHOLE>), dim3(p.grid), dim3(64 * NW), 0, s, a, quant, ws);
}

template <typename T, int CODE, int HD>
static int run_plan8(const PagedAttnArgs& a, const Paged8& quant, const cgpt_paged8_args& args, hipStream_t s) {
  const cgpt_paged_args& call = args.p;
  Plan8 p;
  int rc = make_plan8<HD>(call, &p);
  if (rc != CGPT_OK) return rc;
  char* w = static_cast<char*>(call.workspace);
  if (p.bytes > 0 && (call.workspace_bytes < p.bytes || w == nullptr)) return CGPT_ESCRATCH;
  if (reinterpret_cast<uintptr_t>(w) & 15) return CGPT_EINVAL;
  PagedWs ws{};
  ws.starts = reinterpret_cast<int*>(w + p.o_starts);
  ws.edge_ml = ws.tile_ml = reinterpret_cast<float*>(w + p.o_ml);
  ws.edge_o = ws.tile_o = reinterpret_cast<float*>(w + p.o_o);
  ws.unit_shift = p.unit_shift;
  if (p.whole) {
    launch_stream8<T, CODE, HD, whole_waves8(HD), true>(a, quant, ws, p, s);
    return hip_status(hipGetLastError());
  }
  constexpr int NW = stream_waves8(HD), UK = Shape8<HD, NW>::UK;
  if (p.split > 0) {
    TileJob job{};
    if (p.split > 1) {
      job.ml = ws.tile_ml;
      job.o = ws.tile_o;
    }
    job.split = p.split;
    rc = launch_paged8_tile(args, a, quant, job, p.tile_qt, s);
    if (rc != CGPT_OK || p.split == 1) return rc;
  } else {
    launch_stream8<T, CODE, HD, NW, false>(a, quant, ws, p, s);
  }
  const int n_tile = p.split;
  const int rows = a.seq.n_tokens * a.Hq;
  // Few rows have many partials each; many rows want many of them on a CU.
  if (rows < 4 * num_cus())
    hipLaunchKernelGGL((paged_join_kernel<T, HD, 16, UK, 4>), dim3(rows), dim3(256), 0, s, a, ws, 0, p.grid, n_tile);
  else
    hipLaunchKernelGGL((paged_join_kernel<T, HD, 16, UK, 1>), dim3((rows + 3) / 4), dim3(256), 0, s, a, ws, 0, p.grid, n_tile);
  return hip_status(hipGetLastError());
}

}  // namespace cgpt

extern "C" int cgpt_paged_attention_8bit(const cgpt_paged8_args* args, void* stream) {
  using namespace cgpt;
  bool empty;
  const int rc = check_paged8(args, false, &empty);
  if (rc != CGPT_OK) return rc;
  const cgpt_paged_args& p = args->p;
  const float scale = static_cast<float>(p.scale), scale_log2 = scale * 1.4426950408889634f;
  if (!(scale > 0.f) || !(scale_log2 < INFINITY)) return CGPT_EINVAL;
  if (empty) return CGPT_OK;
  if (p.q == nullptr || p.out == nullptr) return CGPT_EINVAL;
  if (!rows_apart({{p.n_tokens, p.out_st}, {p.Hq, p.out_sh}}, p.head_dim)) return CGPT_EINVAL;
  const PagedAttnArgs a{p.q, p.out, PagePool{p.k_cache, p.kc_sp, p.kc_sh, p.kc_ss},
                        PagePool{p.v_cache, p.vc_sp, p.vc_sh, p.vc_ss}, paged_batch(p), nullptr, 0, p.q_st, p.q_sh,
                        p.out_st, p.out_sh, static_cast<int>(p.Hq), static_cast<int>(p.Hkv), FastDiv(p.Hq / p.Hkv),
                        scale_log2, p.err_flag};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_types8(*args, [&](auto t, auto code, auto hd) {
    return run_plan8<decltype(t), decltype(code)::value, decltype(hd)::value>(a, paged8(*args), *args, s);
  });
}

extern "C" int cgpt_paged_attention_8bit_workspace(const cgpt_paged8_args* args, int64_t* workspace_bytes) {
  using namespace cgpt;
  if (args == nullptr || workspace_bytes == nullptr) return CGPT_EINVAL;
  *workspace_bytes = 0;
  const cgpt_paged_args& p = args->p;
  const int rc = check_sizes(p);
  if (rc != CGPT_OK) return rc;
  if (args->code != CGPT_E4M3 && args->code != CGPT_INT8) return CGPT_EDTYPE;
  if (p.n_tokens == 0 || p.B == 0) return CGPT_OK;
  return with_types8(*args, [&](auto, auto, auto hd) {
    Plan8 plan;
    const int rc = make_plan8<decltype(hd)::value>(p, &plan);
    if (rc == CGPT_OK) *workspace_bytes = plan.bytes;
    return rc;
  });
}
