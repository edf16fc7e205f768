// How the kernels of the paged caches share out their work, and the kernel that joins their
// partials.
#pragma once

#include "paged.h"

namespace cgpt {

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

// ------------------------------------------------------------------ row tiles

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

// ------------------------------------------------------------------ the join

// One wave, or with WAVES = 4 one block, a (token, head) row: its partials, each read by
// HD / 4 lanes, added group of lanes by group and then across the groups, always in the
// same order.  Rows that one block has written whole are left; rows without a key become
// zeros.
template <typename T, int HD, int R, int UK, int WAVES>
static __global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a, PagedWs ws, int prefix_units, int grid,
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

}  // namespace cgpt
