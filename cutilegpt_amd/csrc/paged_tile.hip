// Attention over the paged cache for tiles of many query rows: prompts taken in
// chunks, and all sequences of a batch against their shared prefix.
//
// A block is 4 waves of QT x 16 query rows of one key head (with grouped heads the
// rows are token-major, the group's heads side by side, so a key row is read once for
// all of them); keys come 64 at a time, K and V straight from their pages into LDS by
// direct-to-LDS loads with an address a lane, the next 64 in flight while these are
// used.  The page ids are read one block of keys ahead of the loads that need them: where
// a page is a multiple of 16 keys (A16) by scalar loads, which do not queue with the
// key loads, so more than one block may be on its way.
// S^T = K Q^T and O^T = V^T P^T on 16x16x32 MFMAs (fp32: 16x16x4) as in cgpt_attention_fwd's
// kernel: a lane owns one query row, P goes from the accumulators straight into the second
// product, V is transposed by the LDS read (fp32: read word by word).
//
// What bounds it: no unit alone.  16 chunks of up to 2048 tokens behind up to 4096 keys, 16
// heads of head_dim 64, take 303 us: 619 TFLOP/s of what the mask leaves.  By the counters the
// VALU is busy 53 % of that, the matrix cores 25 %, a CU has no wave for 19 % (the last
// tiles), and a SIMD holds two waves where three fit.  64 weights take 6.4 vector
// instructions, 3.5 of them their own arithmetic (an FMA, an exponential, an add, half a
// conversion); masks, addresses, moves and the maximum's check are the rest.  128 rows a block
// (two sub-tiles a wave) use a loaded key for twice the rows of 64; blocks of eight waves with
// 128 or 256 rows were slower (350 and 412 us), and 128 registers, for four waves a SIMD,
// spill (524 us).  At head_dim 32 the same chunks take 236 us, 561 by the stream kernel, at 16
// 215 and 548.  fp32 is bound by its products: 1911 us at head_dim 64 (2227 by the stream
// kernel), 98 TFLOP/s where a large product reaches 153; the matrix cores are busy 65 %, a CU
// has no wave for 13 %, and two waves a SIMD, all that the registers leave, do not fill the
// rest; 3940 us at 128 (6570).
#include "internal.h"
#include "paged.h"

namespace cgpt {

constexpr int kTileThreads = 256, kTileKeys = 64;

#if defined(__HIP_DEVICE_COMPILE__)
// 16 bytes a lane from its own address to LDS: lane l's land at M0 + 16 l.  Not counted
// by the compiler (see dma_lds16).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma_lds16_at(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
#pragma clang diagnostic pop
#endif

// Block i -> (key head, unit of that head), units 0 .. T - 1.  Blocks go to the eight XCDs
// in turn, each with an L2 of its own: eight heads at a time take one XCD each, the
// last Hkv % 8 (1, 2 or 4) share the XCDs evenly, so an L2 holds the keys of few heads.
// Against heads in turn: 2048 tokens behind 20000 keys, 25 heads 274 -> 198 us, 12 heads
// 116 -> 112; 16 prompts, 4 heads 322 -> 302, 25 heads 521 -> 499, 16 heads 392 -> 396.
__host__ __device__ inline int head_blocks(int Hkv, int T) {
  const int r = Hkv & 7;
  return (Hkv - r) * T + (r == 0 ? 0 : 8 % r == 0 ? (T + 8 / r - 1) / (8 / r) * 8 : r * T);
}
__device__ __forceinline__ bool head_unit(int i, int Hkv, int T, int* hk, int* unit) {
  const int r = Hkv & 7, whole = Hkv - r;
  if (i < whole * T) {
    const int group = i / (8 * T), rem = i - group * 8 * T;
    *hk = 8 * group + (rem & 7);
    *unit = rem >> 3;
    return true;
  }
  i -= whole * T;
  if (8 % r == 0) {
    const int per = 8 / r, x = i & 7;
    *hk = whole + x / per;
    *unit = (i >> 3) * per + x % per;
  } else {
    *hk = whole + i % r;
    *unit = i / r;
  }
  return *unit < T;
}

// Chunk swizzle of a key's row in LDS.  Rows of 64 bytes lie four to the banks' 256: a
// K read's 16 rows then take each chunk four times, and neighbouring groups of four
// rows, which a transposing V read takes two chunks of, the other two.  Of 32-byte rows the
// first eight and the next take the other chunk.
template <int KROW> __device__ __forceinline__ int tile_swz(int row) {
  if (KROW == 32) return (row >> 3) & 1;
  return KROW == 64 ? ((row >> 1) & 2) | ((row >> 3) & 1) : row & (KROW >= 256 ? 15 : 7);
}
// And of V's: fp32 columns are read by four lane groups, four rows apart and 64 bytes wide each.
template <typename T, int KROW> __device__ __forceinline__ int tile_vswz(int row) {
  return sizeof(T) == 2 ? tile_swz<KROW>(row) : row & 12 & (KROW / 16 - 1);
}

// What a launch holds (compiled apart: the choices cost 8 % inside the key loop).
enum TileMode { kOwnRows, kFlatRows, kBoth };

template <typename T, int HD, int QTW, TileMode MODE, bool A16, int STAGES>
__global__ __launch_bounds__(kTileThreads) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 ? (HD <= 32 ? 3 : HD == 64 ? 2 : 1) : HD <= 64 && STAGES == 2 ? 3 : HD <= 64 || STAGES == 2 ? 2 : 1, 4))) void
paged_tile_kernel(PagedAttnArgs a, TileJob job) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int QT = QTW, BQ = 64 * QTW, BKV = kTileKeys, NWAVE = 4;
  constexpr int ES = sizeof(T), EPC = 16 / ES;
  constexpr int KROW = HD * ES, CPR = KROW / 16, RPI = 64 / CPR;  // bytes, chunks of a row; rows of a 1 KiB load
  constexpr int XB = BKV * KROW, STAGE = 2 * XB;
  constexpr bool HALF = KROW == 32;                              // two waves load K, two V; else each both
  constexpr int INS = HALF ? 1 : XB / 1024 / NWAVE;              // loads a wave makes of K (and of V) a block
  constexpr int NKS = (HD + 4 * EPC - 1) / (4 * EPC), ND = HD / 16;
  constexpr int LPS = HALF ? 1 : 2 * INS;                        // and of both
  static_assert(CPR % 4 == 0 || HALF, "a lane group has a chunk in every slab, or two of the four do");
  static_assert(A16 || STAGES == 2, "page ids by vector loads drain the queue at every block");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[STAGES * STAGE];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, frow = lane & 15;
  const int G = static_cast<int>(a.group.d), page_size = static_cast<int>(a.seq.page.d);

  // Blocks of the whole batch against the prefix come first; then, like them, the last row
  // tiles, which see most keys.
  const bool flat = MODE == kFlatRows || (MODE == kBoth && static_cast<int>(blockIdx.x) < job.flat_blocks);
  const int n_split = flat ? job.flat_split : job.split, n_tiles = flat ? job.flat_tiles : job.tiles;
  int hk, unit;
  if (!head_unit(blockIdx.x - (flat ? 0 : job.flat_blocks), a.Hkv, n_tiles * n_split, &hk, &unit)) return;
  const int rev = unit / n_split, split = unit - rev * n_split, tile = n_tiles - 1 - rev;
  const int kb = MODE == kBoth && !flat ? job.from : 0;  // first key

  // ---- rows
  int r0, rows, first = 0, pos0 = 0, n;
  const int* trow = nullptr;
  bool bad = false;
  if (flat) {
    r0 = tile * BQ;
    rows = a.seq.n_tokens * G;
    n = a.prefix_len;
  } else {
    int rt = tile, count;
    const int b = slot_seq<BQ>(a.seq, G, lane, &rt);
    if (b >= a.seq.B) return;
    seq_tokens(a.seq, b, &first, &count);
    rows = count * G;
    r0 = rt * BQ;
    if (r0 < 0 || r0 >= rows) return;
    const int len = max(a.seq.lens[b], 0);
    bad = len > a.seq.cap;
    pos0 = len - count;
    n = min(min(len, a.seq.cap), max(pos0 + a.group.div(min(r0 + BQ, rows) - 1) + 1, 0));
    trow = a.seq.table + b * a.seq.stride;
  }
  const int wr0 = r0 + wave * 16 * QT;
  const bool wave_live = wr0 < rows;

  // ---- keys of this split, in blocks of 64
  // (None for rows that see nothing past the prefix, whose table may end with it.)
  const int jb = MODE == kBoth ? kb / BKV : 0, n_kv = n > kb ? (n + BKV - 1) / BKV - jb : 0,
            per = (n_kv + n_split - 1) / n_split;
  const int j0 = jb + split * per, j1 = min(j0 + per, jb + n_kv);

  const int lrow = lane / CPR, slot16 = lane % CPR, part = HALF ? wave & 1 : wave;
  const uint8_t* const kh = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.kc.base) + hk * a.kc.sh);
  const uint8_t* const vh = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.vc.base) + hk * a.vc.sh);
  int pg[INS];
  // First key of load ii of block j (one page's, A16), or the lane's own.
  auto key_of = [&](int j, int ii) __attribute__((always_inline)) {
    const int key = j * BKV + (ii * NWAVE + part) * RPI;
    const int k = A16 ? min(key, (n - 1) & ~(RPI - 1)) : min(key + lrow, n - 1);
    return MODE == kBoth ? max(k, kb) : k;
  };
  auto fetch = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int ii = 0; ii < INS; ++ii) {
      const int key = key_of(j, ii), col = a.seq.page.div(key);
      const int* const row = flat || key < a.prefix_len ? a.prefix : trow;
      pg[ii] = A16 ? ((const __attribute__((address_space(4))) int*)row)[__builtin_amdgcn_readfirstlane(col)] : row[col];
    }
  };
  auto issue = [&](int j, uint8_t* buf) __attribute__((always_inline)) {
#pragma unroll
    for (int ii = 0; ii < INS; ++ii) {
      const int row = (ii * NWAVE + part) * RPI + lrow, key = key_of(j, ii);
      const int slot = (A16 ? min(key + lrow, n - 1) : key) - a.seq.page.div(key) * page_size;
      int p = pg[ii];
      if (static_cast<uint32_t>(p) >= static_cast<uint32_t>(a.seq.n_pages)) {
        p = 0;
        bad = true;
      }
      const int k_chunk = (slot16 ^ tile_swz<KROW>(row)) << 4, v_chunk = (slot16 ^ tile_vswz<T, KROW>(row)) << 4;
      const uint32_t lds = (ii * NWAVE + part) * 1024;
      if (!HALF || wave < 2)
        dma_lds16_at(kh + ES * (p * a.kc.sp) + ES * (slot * a.kc.ss) + k_chunk, lds_addr(buf + lds));
      if (!HALF || wave >= 2)
        dma_lds16_at(vh + ES * (p * a.vc.sp) + ES * (slot * a.vc.ss) + v_chunk, lds_addr(buf + XB + lds));
    }
  };

  // Blocks j0 .. j0 + STAGES - 2 are on their way before the loop; pg is one further.
  if (j0 < j1) {
    fetch(j0);
#pragma unroll
    for (int st = 0; st < STAGES - 1; ++st)
      if (j0 + st < j1) {
        issue(j0 + st, smem + st * STAGE);
        fetch(min(j0 + st + 1, j1 - 1));
      }
  }

  u32x4_t qf[QT][NKS];
  int lim[QT];  // last key the row sees; rows that do not exist are never masked
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = wr0 + 16 * qt + frow;
    const bool live = r < rows;
    const int i = a.group.div(live ? r : 0), h = hk * G + (live ? r : 0) - i * G, t = first + i;
    if (flat) {
      const int b = seq_of(a.seq, t);
      lim[qt] = -1;
      if (b < a.seq.B) {
        int f, c;
        seq_tokens(a.seq, b, &f, &c);
        lim[qt] = min(a.seq.lens[b] - c + (t - f), n - 1);
      }
    } else {
      lim[qt] = min(pos0 + i, n - 1);
    }
    if (!live) lim[qt] = 0x7fffffff;
    const T* qp = static_cast<const T*>(a.q) + t * a.q_st + h * a.q_sh;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(qp + (HALF ? g & 1 : 4 * ks + g) * EPC);
      qf[qt][ks] = live && (!HALF || g < 2) ? v : u32x4_t{0, 0, 0, 0};
    }
  }
  // nm = minus the shift of a row's scaled scores (their running maximum, less kDrop), +inf
  // while it has none.
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
  const int wave_last = flat ? n - 1 : pos0 + a.group.div(min(wr0 + 16 * QT, rows) - 1);
  wait_vmcnt<0>();

  const int tr_row = 4 * g + (frow >> 2);
  int odd_from = 0x7fffffff;  // first masked block of keys with a value that is not finite
  for (int j = j0; j < j1; ++j) {
    raw_barrier();
    const uint8_t* sk = smem + ((j - j0) & (STAGES - 1)) * STAGE;
    const uint8_t* sv = sk + XB;
    if (j + STAGES - 1 < j1) {
      issue(j + STAGES - 1, smem + ((j - j0 + STAGES - 1) & (STAGES - 1)) * STAGE);
      fetch(min(j + STAGES, j1 - 1));
    }
    const int base = j * BKV;
    if (wave_live && base <= wave_last) {
      f32x4_t s[QT][4];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) s[qt][kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
          const int key = kt * 16 + frow, c = HALF ? g & 1 : 4 * ks + g;
          u32x4_t kf = *reinterpret_cast<const u32x4_t*>(sk + key * KROW + ((c ^ tile_swz<KROW>(key)) << 4));
          if (HALF && g >= 2) kf = u32x4_t{0, 0, 0, 0};  // 0 x inf would be NaN
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) Mfma<T>::run(kf, qf[qt][ks], s[qt][kt]);
        }
      bool masked = false;
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
        if ((MODE == kBoth && base < kb) || __builtin_amdgcn_ballot_w64(lim[qt] < base + BKV - 1) != 0) {
          masked = true;
          const int hi = lim[qt] - base - 4 * g, lo = MODE == kBoth ? kb - base - 4 * g : -0x7fffffff;
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              s[qt][kt][r] = 16 * kt + r > hi || (MODE == kBoth && 16 * kt + r < lo) ? -INFINITY : s[qt][kt][r];
        }
      // P against the running shift as it stands.  A lane whose 16 values sum to at most 2^7
      // (2^14 in fp16, see kDrop) has none above it, so its shift need not move; only when some
      // lane fails that (a NaN sum fails it, and a row without a maximum) is the block's maximum
      // taken and, where it outgrows the one behind the shift by more than 8, the row rescaled
      // and its P made again.
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
        if (__builtin_amdgcn_ballot_w64(sum <= (kDrop<T> > 0 ? 16384.0f : 128.0f)) != __builtin_amdgcn_read_exec()) {
          const float m_old = -nm[qt];
          float mx = -INFINITY;
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[qt][kt][r]);
          mx = column_max(mx) * a.scale_log2;
          const bool grow = mx > m_old + (8.0f + kDrop<T>);
          const float m_new = grow ? mx - kDrop<T> : m_old;
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
      // A masked key's weight is 0, but 0 x NaN is NaN: where a row is masked the matrix
      // cores get the finite values alone, and the others are added after the loop to
      // the rows that see them.
      uint32_t bits = 0;
      auto pv = [&](auto clean) __attribute__((always_inline)) {
        if constexpr (ES == 2) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            u32x4_t pf[QT];
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
              pf[qt] = u32x4_t{pack2<T>(s[qt][2 * c][0], s[qt][2 * c][1]), pack2<T>(s[qt][2 * c][2], s[qt][2 * c][3]),
                               pack2<T>(s[qt][2 * c + 1][0], s[qt][2 * c + 1][1]),
                               pack2<T>(s[qt][2 * c + 1][2], s[qt][2 * c + 1][3])};
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
              const u32x2_t lo = vt_read<KROW>(sv, 32 * c + tr_row, tile_vswz<T, KROW>(tr_row), dt, frow);
              const u32x2_t hi = vt_read<KROW>(sv, 32 * c + 16 + tr_row, tile_vswz<T, KROW>(tr_row), dt, frow);
              u32x4_t w = {lo[0], lo[1], hi[0], hi[1]};
              if constexpr (decltype(clean)::value)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  bits |= special_bits<T>(w[e]);
                  w[e] = finite_part<T>(w[e]);
                }
#pragma unroll
              for (int qt = 0; qt < QT; ++qt) Mfma<T>::run(w, pf[qt], o[qt][dt]);
            }
          }
        } else {
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
              u32x4_t w;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int key = 16 * kt + 4 * g + e, d = 16 * dt + frow;
                w[e] = *reinterpret_cast<const uint32_t*>(sv + key * KROW + (((d >> 2) ^ tile_vswz<T, KROW>(key)) << 4) +
                                                          4 * (d & 3));
                if constexpr (decltype(clean)::value) {
                  bits |= special_bits<T>(w[e]);
                  w[e] = finite_part<T>(w[e]);
                }
              }
#pragma unroll
              for (int qt = 0; qt < QT; ++qt) {
                const u32x4_t pf = {__float_as_uint(s[qt][kt][0]), __float_as_uint(s[qt][kt][1]),
                                    __float_as_uint(s[qt][kt][2]), __float_as_uint(s[qt][kt][3])};
                Mfma<T>::run(w, pf, o[qt][dt]);
              }
            }
        }
      };
      if (masked) {
        pv(std::true_type{});
        if (__builtin_amdgcn_ballot_w64((bits & 0x80008000u) != 0) != 0) odd_from = min(odd_from, j);
      } else {
        pv(std::false_type{});
      }
    }
    // This wave's part of block j + 1 has landed (loads return in order), and its LDS reads
    // are done; the blocks behind it may be on their way.
    const int later = min(j1 - 1, j + STAGES - 1) - (j + 1);
    if (STAGES > 2 && later >= 2)
      wait_vmcnt<STAGES == 4 ? 2 * LPS : 0>();
    else if (STAGES > 2 && later == 1)
      wait_vmcnt<STAGES == 4 ? LPS : 0>();
    else
      wait_vmcnt<0>();
  }

  // ---- values that are not finite in masked blocks: key by key, rarely
  if (__builtin_expect(odd_from < j1, 0)) {
    // Blocks that no row of the wave was masked in have theirs in O already; once a row is
    // masked at its end it stays so, but the block across kb stands alone.
    for (int key = max(odd_from * BKV, kb); key < min(n, j1 * BKV); ++key) {
      const int base = key & ~(BKV - 1);
      bool masked = MODE == kBoth && base < kb;
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) masked |= __builtin_amdgcn_ballot_w64(lim[qt] < base + BKV - 1) != 0;
      if (!masked) continue;
      const int slot = key - a.seq.page.div(key) * page_size;
      int p = (flat || key < a.prefix_len ? a.prefix : trow)[a.seq.page.div(key)];
      if (static_cast<uint32_t>(p) >= static_cast<uint32_t>(a.seq.n_pages)) p = 0;
      const T* kr = reinterpret_cast<const T*>(kh) + p * a.kc.sp + slot * a.kc.ss;
      const T* vr = reinterpret_cast<const T*>(vh) + p * a.vc.sp + slot * a.vc.ss;
      add_odd_key<T, HD, QT>(kr, vr, key, g, a.scale_log2, lim, qf, nm, o);
    }
  }

  // ---- out: lane holds O[row][16 dt + 4 g .. +3]
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float l = column_sum(l_run[qt]);
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
      const int64_t part = flat ? split : job.flat_split + split;
      const int64_t at = (part * a.seq.n_tokens + t) * a.Hq + h;
      if (g == 0) {
        job.ml[2 * at] = -nm[qt];
        job.ml[2 * at + 1] = l;
      }
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) *reinterpret_cast<f32x4_t*>(job.o + at * HD + 16 * dt + 4 * g) = o[qt][dt];
    }
  }
  if (bad && a.err != nullptr) *a.err = 1;
#endif  // __HIP_DEVICE_COMPILE__
}

template <typename T, int HD, int QTW>
static int launch_tile(const PagedAttnArgs& a, TileJob job, hipStream_t s) {
  constexpr int BQ = 64 * QTW;
  const int64_t rows = static_cast<int64_t>(a.seq.n_tokens) * (a.Hq / a.Hkv);
  const int64_t flat = job.flat_split > 0 ? (rows + BQ - 1) / BQ : 0;
  const int64_t own = job.split == 0 ? 0 : a.seq.cu == nullptr && a.Hq / a.Hkv <= BQ ? a.seq.B : rows / BQ + a.seq.B;
  if ((flat * job.flat_split + own * job.split) * a.Hkv > kMaxBlocks - 16) return CGPT_ESHAPE;
  job.flat_tiles = static_cast<int>(flat);
  job.tiles = static_cast<int>(own);
  job.flat_blocks = head_blocks(a.Hkv, job.flat_tiles * job.flat_split);
  const int blocks = job.flat_blocks + head_blocks(a.Hkv, job.tiles * job.split);
  // The keys of a load (at most 16, 32 of 32-byte rows) lie in one page, and on one side of
  // the prefix's end.
  constexpr int RUN = HD * sizeof(T) == 32 ? 32 : 16;
  const bool a16 = a.seq.page.d % RUN == 0 && a.prefix_len % RUN == 0;
#define CGPT_TILE(A16, ST)                                                                                           \
  do {                                                                                                               \
    if (own == 0)                                                                                                    \
      hipLaunchKernelGGL((paged_tile_kernel<T, HD, QTW, kFlatRows, A16, ST>), dim3(blocks), dim3(kTileThreads), 0, s, \
                         a, job);                                                                                    \
    else if (flat == 0)                                                                                              \
      hipLaunchKernelGGL((paged_tile_kernel<T, HD, QTW, kOwnRows, A16, ST>), dim3(blocks), dim3(kTileThreads), 0, s, \
                         a, job);                                                                                    \
    else                                                                                                             \
      hipLaunchKernelGGL((paged_tile_kernel<T, HD, QTW, kBoth, A16, ST>), dim3(blocks), dim3(kTileThreads), 0, s, a, \
                         job);                                                                                       \
  } while (0)
  if (!a16)
    CGPT_TILE(false, 2);
  else if (sizeof(T) == 2 && QTW == 1 && blocks <= (HD <= 64 ? 2 : 1) * num_cus())
    // Few blocks: little else on the CU hides the loads, so three blocks of keys are kept
    // on their way.
    CGPT_TILE(true, (sizeof(T) == 2 && QTW == 1 ? 4 : 2));
  else
    CGPT_TILE(true, 2);
#undef CGPT_TILE
  return hip_status(hipGetLastError());
}

template <typename T, int HD>
static int launch_tile_qt(const PagedAttnArgs& a, const TileJob& job, int qt, hipStream_t s) {
  return qt == 2 ? launch_tile<T, HD, 2>(a, job, s) : launch_tile<T, HD, 1>(a, job, s);
}

int launch_paged_tile(int64_t dtype, int head_dim, const PagedAttnArgs& a, const TileJob& job, int qt, hipStream_t s) {
  if (dtype == CGPT_BF16 && head_dim == 64) return launch_tile_qt<bf16_t, 64>(a, job, qt, s);
  if (dtype == CGPT_BF16 && head_dim == 128) return launch_tile_qt<bf16_t, 128>(a, job, qt, s);
  if (dtype == CGPT_F16 && head_dim == 64) return launch_tile_qt<f16_t, 64>(a, job, qt, s);
  if (dtype == CGPT_F16 && head_dim == 128) return launch_tile_qt<f16_t, 128>(a, job, qt, s);
  if (dtype == CGPT_BF16 && head_dim == 32) return launch_tile_qt<bf16_t, 32>(a, job, qt, s);
  if (dtype == CGPT_F16 && head_dim == 32) return launch_tile_qt<f16_t, 32>(a, job, qt, s);
  if (dtype == CGPT_BF16 && head_dim == 16) return launch_tile_qt<bf16_t, 16>(a, job, qt, s);
  if (dtype == CGPT_F16 && head_dim == 16) return launch_tile_qt<f16_t, 16>(a, job, qt, s);
  if (dtype == CGPT_F32 && head_dim == 16) return launch_tile_qt<float, 16>(a, job, qt, s);
  if (dtype == CGPT_F32 && head_dim == 32) return launch_tile_qt<float, 32>(a, job, qt, s);
  if (dtype == CGPT_F32 && head_dim == 64) return launch_tile_qt<float, 64>(a, job, qt, s);
  if (dtype == CGPT_F32 && head_dim == 128) return launch_tile_qt<float, 128>(a, job, qt, s);
  return CGPT_EDTYPE;
}

}  // namespace cgpt
