// Attention over the 8-bit paged cache for tiles of many query rows: prompts taken in chunks.
//
// A block is 4 waves of QT x 16 query rows of one key head, as in paged_tile.hip (grouped heads'
// rows side by side).  Keys come 64 at a time: each thread brings a quarter of one key's and one
// value's codes into registers, a step ahead, turns them into bf16 there, once for all rows of
// the block, and writes them into the buffer that the block does not read.  (Codes loaded
// straight to LDS would have to be turned by every wave for itself.)  S^T = K Q^T and
// O^T = V^T P^T as there; queries and weights of more bits than bf16 go in as parts (see
// paged8_attention.hip).
//
// 16 chunks of up to 2048 tokens behind up to 4096 keys, 16 heads of 64, e4m3: bf16 334 us, 562
// TFLOP/s of what the mask leaves (16-bit cache: 303; the stream kernel: 1387), fp16 485, fp32 628
// (16-bit cache: 1911 in fp32).  No unit alone bounds it, as there: the VALU is busy 60 % of the time
// (8.5 instructions for 64 weights, 6.4 there: the keys' way into bf16), the matrix cores 23 %,
// LDS 18 % without conflicts, and 19 % of the CUs have no wave (the mean over the call).  In fp16,
// with two parts of each, VALU 57 % and matrix cores 33 %.
#include "internal.h"
#include "paged8.h"
#include "paged_units.h"

namespace cgpt {

constexpr int kTile8Threads = 256, kTile8Keys = 64;

template <typename T, int CODE, int HD, int QT>
__global__ __launch_bounds__(kTile8Threads) void paged8_tile_kernel(PagedAttnArgs a, Paged8 quant, TileJob job) {
  constexpr int BQ = 64 * QT, BKV = kTile8Keys, NP = kParts<T>;
  constexpr int KROW = 2 * HD, XB = BKV * KROW, STAGE = 2 * XB;
  constexpr int NW = HD / 16;                    // words of codes a thread has of a row
  constexpr int NS = HD >= 32 ? HD / 32 : 1, ND = HD / 16;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * STAGE];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, frow = lane & 15;
  const int G = static_cast<int>(a.group.d), page_size = static_cast<int>(a.seq.page.d);

  // The last row tiles, which see most keys, come first.
  int hk, unit;
  if (!head_unit(blockIdx.x, a.Hkv, job.tiles * job.split, &hk, &unit)) return;
  const int rev = unit / job.split, split = unit - rev * job.split;
  int rt = job.tiles - 1 - rev, first, count;
  const int b = slot_seq<BQ>(a.seq, G, lane, &rt);
  if (b >= a.seq.B) return;
  seq_tokens(a.seq, b, &first, &count);
  const int rows = count * G, r0 = rt * BQ;
  if (r0 < 0 || r0 >= rows) return;
  const int len = max(a.seq.lens[b], 0), pos0 = len - count;
  bool bad = len > a.seq.cap;
  const int n = min(min(len, a.seq.cap), max(pos0 + a.group.div(min(r0 + BQ, rows) - 1) + 1, 0));
  const int* const trow = a.seq.table + b * a.seq.stride;
  const int wr0 = r0 + wave * 16 * QT;
  const bool wave_live = wr0 < rows;
  // Keys of this split, in blocks of 64.
  const int n_kv = (n + BKV - 1) / BKV, per = (n_kv + job.split - 1) / job.split;
  const int j0 = split * per, j1 = min(j0 + per, n_kv);

  // ---- a thread's part of the keys: row tid / 4 of a block, a quarter of its values
  const int krow = tid >> 2, part = tid & 3;
  const uint8_t* const kh = static_cast<const uint8_t*>(a.kc.base) + hk * a.kc.sh + part * (HD / 4);
  const uint8_t* const vh = static_cast<const uint8_t*>(a.vc.base) + hk * a.vc.sh + part * (HD / 4);
  const uint8_t* const ksh = quant.ks.base + hk * quant.ks.sh;
  const uint8_t* const vsh = quant.vs.base + hk * quant.vs.sh;
  uint32_t kr[NW], vr[NW];
  int kx = 0, vx = 0, pg = 0;
  bool odd = false;
  auto key_of = [&](int j) __attribute__((always_inline)) { return min(j * BKV + krow, n - 1); };
  auto fetch = [&](int j) __attribute__((always_inline)) { pg = trow[a.seq.page.div(key_of(j))]; };
  auto load = [&](int j) __attribute__((always_inline)) {
    const int key = key_of(j), slot = key - a.seq.page.div(key) * page_size;
    int p = pg;
    if (static_cast<uint32_t>(p) >= static_cast<uint32_t>(a.seq.n_pages)) {
      p = 0;
      bad = true;
    }
    const int block = quant.block.div(slot);
    const uint8_t* const kp = kh + p * a.kc.sp + slot * a.kc.ss;
    const uint8_t* const vp = vh + p * a.vc.sp + slot * a.vc.ss;
    kx = ksh[p * quant.ks.sp + block * quant.ks.sb];
    vx = vsh[p * quant.vs.sp + block * quant.vs.sb];
    typedef uint32_t words_t __attribute__((ext_vector_type(NW < 4 ? NW : 4)));
    if constexpr (NW == 1) {
      kr[0] = *reinterpret_cast<const uint32_t*>(kp);
      vr[0] = *reinterpret_cast<const uint32_t*>(vp);
    } else {
#pragma unroll
      for (int i = 0; i < NW; i += 4) {
        const words_t kw = *reinterpret_cast<const words_t*>(kp + 4 * i), vw = *reinterpret_cast<const words_t*>(vp + 4 * i);
#pragma unroll
        for (int e = 0; e < (NW < 4 ? NW : 4); ++e) {
          kr[i + e] = kw[e];
          vr[i + e] = vw[e];
        }
      }
    }
  };
  // The loaded codes as bf16 into a buffer.  Values that are no numbers become 0 there (0 x NaN
  // would spoil rows that do not see them) and are added at the end.
  auto stage = [&](uint8_t* buf) __attribute__((always_inline)) {
    const float fk = scale_of<CODE>(kx), fv = value_scale_of<CODE>(vx);
    uint8_t* const kd = buf + krow * KROW;
    uint8_t* const vd = kd + XB;
    const int swz = tile_swz<KROW>(krow);
#pragma unroll
    for (int i = 0; i < NW; ++i)
      if (CODE == CGPT_E4M3) {
        const uint32_t bits = nan_codes(vr[i]);
        odd |= bits != 0;
        vr[i] &= ~((bits >> 7) * 0xffu);
      }
    if constexpr (NW == 1) {
      const int at = (((part >> 1) ^ swz) << 4) + 8 * (part & 1);
      *reinterpret_cast<u32x2_t*>(kd + at) = bf16x4_of<CODE>(kr[0], fk);
      *reinterpret_cast<u32x2_t*>(vd + at) = bf16x4_of<CODE>(vr[0], fv);
    } else {
#pragma unroll
      for (int i = 0; i < NW; i += 2) {
        const int at = ((part * (NW / 2) + i / 2) ^ swz) << 4;
        const u32x2_t k0 = bf16x4_of<CODE>(kr[i], fk), k1 = bf16x4_of<CODE>(kr[i + 1], fk);
        *reinterpret_cast<u32x4_t*>(kd + at) = u32x4_t{k0[0], k0[1], k1[0], k1[1]};
        const u32x2_t v0 = bf16x4_of<CODE>(vr[i], fv), v1 = bf16x4_of<CODE>(vr[i + 1], fv);
        *reinterpret_cast<u32x4_t*>(vd + at) = u32x4_t{v0[0], v0[1], v1[0], v1[1]};
      }
    }
  };
  if (j0 < j1) {
    fetch(j0);
    load(j0);
    fetch(min(j0 + 1, j1 - 1));
  }

  u32x4_t qf[QT][NS][NP];
  int lim[QT];  // last key the row sees; rows that do not exist are never masked
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = wr0 + 16 * qt + frow;
    const bool live = r < rows;
    const int i = a.group.div(live ? r : 0), h = hk * G + (live ? r : 0) - i * G;
    lim[qt] = live ? min(pos0 + i, n - 1) : 0x7fffffff;
    const T* qp = static_cast<const T*>(a.q) + (first + i) * a.q_st + h * a.q_sh;
    const bool has = live && (HD > 16 || g < 2);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; e += Elem<T>::kVec) load_vec(qp + 32 * s + 8 * (HD > 16 ? g : g & 1) + e, x + e);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = has ? x[e] : 0.f;
      split_parts<NP>(x, qf[qt][s]);
    }
  }
  // nm = minus the shift of a row's scaled scores (their running maximum), +inf while it has none.
  f32x4_t o[QT][ND];
  float nm[QT], l_run[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    nm[qt] = INFINITY;
    l_run[qt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) o[qt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // The last key that any row of the wave sees.
  const int wave_last = pos0 + a.group.div(min(wr0 + 16 * QT, rows) - 1);

  const int tr_row = 4 * g + (frow >> 2);
  if (j0 < j1) {
    stage(smem);
    if (j0 + 1 < j1) {
      load(j0 + 1);
      fetch(min(j0 + 2, j1 - 1));
    }
  }
  for (int j = j0; j < j1; ++j) {
    __syncthreads();
    const uint8_t* sk = smem + ((j - j0) & 1) * STAGE;
    const uint8_t* sv = sk + XB;
    if (j + 1 < j1) {
      stage(smem + ((j + 1 - j0) & 1) * STAGE);
      if (j + 2 < j1) {
        load(j + 2);
        fetch(min(j + 3, j1 - 1));
      }
    }
    const int base = j * BKV;
    if (!wave_live || base > wave_last) continue;
    f32x4_t s[QT][4];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) s[qt][kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int sl = 0; sl < NS; ++sl)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        const int key = kt * 16 + frow, c = HD > 16 ? 4 * sl + g : g & 1;
        u32x4_t kf = *reinterpret_cast<const u32x4_t*>(sk + key * KROW + ((c ^ tile_swz<KROW>(key)) << 4));
        if (HD == 16 && g >= 2) kf = u32x4_t{0, 0, 0, 0};  // 0 x NaN would be NaN
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
          for (int p = 0; p < NP; ++p) Mfma<bf16_t>::run(kf, qf[qt][sl][p], s[qt][kt]);
      }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
      if (__builtin_amdgcn_ballot_w64(lim[qt] < base + BKV - 1) != 0) {
        const int hi = lim[qt] - base - 4 * g;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[qt][kt][r] = 16 * kt + r > hi ? -INFINITY : s[qt][kt][r];
      }
    // P against the running shift as it stands.  A lane whose 16 values sum to at most 2^7 has
    // none above it, so its shift need not move; only when some lane fails that (a NaN sum
    // fails it, and a row without a maximum) is the block's maximum taken and, where it
    // outgrows the one behind the shift by more than 8, the row rescaled and its P made again.
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float p[4][4], sum = 0.f;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qt][kt][r], a.scale_log2, nm[qt]));
          sum += p[kt][r];
        }
      if (__builtin_amdgcn_ballot_w64(sum <= 128.0f) != __builtin_amdgcn_read_exec()) {
        const float m_old = -nm[qt];
        float mx = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[qt][kt][r]);
        mx = column_max(mx) * a.scale_log2;
        const bool grow = mx > m_old + 8.0f;
        const float m_new = grow ? mx : m_old;
        const float alpha = grow ? __builtin_amdgcn_exp2f(m_old - m_new) : 1.0f;
        nm[qt] = m_new == -INFINITY ? INFINITY : -m_new;
        l_run[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[qt][dt][r] *= alpha;
        // A row that has seen no key yet: its scores are all -inf and its P 0.
        const float shift = m_new == -INFINITY ? 0.f : -m_new;
        sum = 0.f;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qt][kt][r], a.scale_log2, shift));
            sum += p[kt][r];
          }
      }
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[qt][kt][r] = p[kt][r];
      l_run[qt] += sum;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      u32x4_t pf[QT][NP];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const float p[8] = {s[qt][2 * c][0], s[qt][2 * c][1], s[qt][2 * c][2], s[qt][2 * c][3],
                            s[qt][2 * c + 1][0], s[qt][2 * c + 1][1], s[qt][2 * c + 1][2], s[qt][2 * c + 1][3]};
        split_parts<NP>(p, pf[qt]);
      }
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) {
        const u32x2_t lo = vt_read<KROW>(sv, 32 * c + tr_row, tile_swz<KROW>(tr_row), dt, frow);
        const u32x2_t hi = vt_read<KROW>(sv, 32 * c + 16 + tr_row, tile_swz<KROW>(tr_row), dt, frow);
        const u32x4_t w = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
          for (int p = 0; p < NP; ++p) Mfma<bf16_t>::run(w, pf[qt][p], o[qt][dt]);
      }
    }
  }

  // ---- values that are no numbers: key by key, rarely
  if (CODE == CGPT_E4M3 && __builtin_expect(__syncthreads_or(odd), 0)) {
    for (int key = j0 * BKV; key < min(n, j1 * BKV); ++key) {
      const int col = a.seq.page.div(key), slot = key - col * page_size;
      int p = trow[col];
      if (static_cast<uint32_t>(p) >= static_cast<uint32_t>(a.seq.n_pages)) p = 0;
      const uint8_t* const v = static_cast<const uint8_t*>(a.vc.base) + hk * a.vc.sh + p * a.vc.sp + slot * a.vc.ss + 4 * g;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) {
        const uint32_t bits = nan_codes(*reinterpret_cast<const uint32_t*>(v + 16 * dt));
        if (bits != 0)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if ((bits >> (8 * e + 7)) & 1 && key <= lim[qt]) o[qt][dt][e] = NAN;
      }
    }
  }

  // ---- out: lane holds O[row][16 dt + 4 g .. +3]
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float l = column_sum(l_run[qt]) * kSumDrop;
    const int r = wr0 + 16 * qt + frow;
    if (r >= rows) continue;
    const int i = a.group.div(r), h = hk * G + r - i * G, t = first + i;
    if (job.ml == nullptr) {
      const float inv = l == 0.f ? 0.f : 1.0f / l;  // no key, or a NaN that stays one
      T* orow = static_cast<T*>(a.o) + t * a.o_st + h * a.o_sh;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) {
        const float v[4] = {o[qt][dt][0] * inv, o[qt][dt][1] * inv, o[qt][dt][2] * inv, o[qt][dt][3] * inv};
        store4_out(orow + 16 * dt + 4 * g, v);
      }
    } else {
      const int64_t at = (static_cast<int64_t>(split) * a.seq.n_tokens + t) * a.Hq + h;
      if (g == 0) {
        job.ml[2 * at] = -nm[qt];
        job.ml[2 * at + 1] = l;
      }
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) *reinterpret_cast<f32x4_t*>(job.o + at * HD + 16 * dt + 4 * g) = o[qt][dt];
    }
  }
  if (bad && a.err != nullptr) *a.err = 1;
}

template <typename T, int CODE, int HD, int QT>
static int launch_tile8(const PagedAttnArgs& a, const Paged8& quant, TileJob job, hipStream_t s) {
  constexpr int BQ = 64 * QT;
  const int64_t rows = static_cast<int64_t>(a.seq.n_tokens) * (a.Hq / a.Hkv);
  const int64_t tiles = a.seq.cu == nullptr && a.Hq / a.Hkv <= BQ ? a.seq.B : rows / BQ + a.seq.B;
  if (tiles * job.split * a.Hkv > kMaxBlocks - 16) return CGPT_ESHAPE;
  job.tiles = static_cast<int>(tiles);
  const int blocks = head_blocks(a.Hkv, job.tiles * job.split);
  hipLaunchKernelGGL((paged8_tile_kernel<T, CODE, HD, QT>), dim3(blocks), dim3(kTile8Threads), 0, s, a, quant, job);
  return hip_status(hipGetLastError());
}

int launch_paged8_tile(const cgpt_paged8_args& call, const PagedAttnArgs& a, const Paged8& quant, const TileJob& job, int qt,
                       hipStream_t s) {
  return with_types8(call, [&](auto t, auto code, auto hd) {
    typedef decltype(t) T;
    constexpr int CODE = decltype(code)::value, HD = decltype(hd)::value;
    return qt == 2 ? launch_tile8<T, CODE, HD, 2>(a, quant, job, s) : launch_tile8<T, CODE, HD, 1>(a, quant, job, s);
  });
}

}  // namespace cgpt
