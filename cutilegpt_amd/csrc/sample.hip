// The next token of a row of logits: temperature, top-k, top-p, min-p, and a draw with a given
// random number.
//
// With l the row, m its maximum: w_i = 2^((l_i - m) log2(e) / T).  In the order of the logits
// (largest first, equal ones by index) the cuts keep a first run: top_k entries, then of these
// the shortest run with at least top_p of their weight; of the run min_p drops weights below
// min_p.  The token is the first index, in the order of the vocabulary, at which the running
// sum of the kept weights passes u times their sum.
//
// Weights are held as whole multiples of 2^-43 of the largest, computed in 64 bits: their sums
// are exact, whatever the order, so that neither the number of threads nor the order of their
// additions decides where a border lies, and a border is off by 2^-44 of the largest weight an
// entry.  (In fp32 a sum of 50 thousand flat weights is off by some 1e-7 of it, and one draw in
// a hundred would take a neighbour.)
//
// A block takes a row and passes over it: for the maximum; then, where top_k, min_p or the row
// itself leave few entries that can be kept, for those alone, which are put in order; else for a
// histogram of the weights by their logits (for a long top_k first one of the counts), and for
// the sums of the weights in front of the bin that the cut falls into, whose own entries are put
// in order.  Bins of too many entries are cut again by their keys.  The draw finds the wave's
// run, the step and the entry.
//
// One row of 50257 fp32 logits, top_k 40: 19 us, mostly latencies (of a block's some forty barriers,
// the passes 4 and 2 us; temperature 0, two passes alone, 10).  64 rows in bf16, top_p among them: 68
// us, on 64 of 256 CUs (a wave on 9 % of them, the mean over the call).  256 rows of 128000 in fp32,
// top_p 0.95: 164 us, a row a CU; 126 vector instructions an entry (two weights of some 24, 14 of
// those in 64 bits, beside bins, cuts and atomics) keep the VALU busy 60 %.  33 rows of 32001, 97 % masked: 22 us.  (Rows shared out over blocks,
// a launch for each pass, were slower where rows are few: 37 us for the one, 33 for the 33, 58
// for the 64.)
#include "internal.h"
#include "common.h"

namespace cgpt {

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr int kBins = 2048;       // of a histogram
constexpr int kList = 1024;       // entries that are put in order
constexpr int kWaveList = 128;    // of a wave's finding
constexpr int kPairs = 192;       // in order each against all others
constexpr int kShort = 512;       // top_k up to which a bound is taken from the threads' largest entries
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxIts = kMaxVocab / (4 * kSampleThreads);
constexpr uint64_t kOne = uint64_t{1} << 43;
constexpr float kReach = 44.5f;  // weights below 2^-44 are 0

typedef unsigned long long u64_t;

struct SampleArgs {
  const void* x;
  const float* u;
  const float* t;   // a row's settings, or NULL for the one that follows
  const int* k;
  const float* p;
  const float* m;
  double t1, p1, m1;
  int64_t k1;
  int64_t ld;
  int V;
  int64_t* ids;
};

struct SampleShared {
  double roots[256];  // 2^(43 + i / 256)
  u64_t mass[kBins];
  u64_t list[kList];  // places in the order: a larger number comes first
  u64_t list_w[kPairs];
  u64_t found[kSampleWaves][kWaveList];
  u64_t its[kMaxIts];
  u64_t wave_a[kSampleWaves], sums[kSampleWaves];
  int n_found[kSampleWaves];
  u64_t sel_a;
  uint32_t sel_lo, sel_hi;
  int sel_bin, sel_idx;
};

// Order of the numbers as order of unsigned integers; both zeros are one.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// An entry's place in the order.
__device__ __forceinline__ u64_t place(float v, int i) {
  return (static_cast<u64_t>(order_key(v)) << 32) | ~static_cast<uint32_t>(i);
}

__device__ __forceinline__ u64_t shfl64(u64_t v, int l) {
  return (static_cast<u64_t>(__shfl(static_cast<uint32_t>(v >> 32), l, 64)) << 32) |
         __shfl(static_cast<uint32_t>(v), l, 64);
}
template <int CTRL, int ROWS> __device__ __forceinline__ u64_t dpp_or_0(u64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false);
  return (static_cast<u64_t>(hi) << 32) | lo;
}
// The inclusive sum over the wave's lanes up to this one: within rows of 16 by shifts, then
// each row's last lane to the rows behind it.
__device__ __forceinline__ u64_t wave_scan64(u64_t v) {
  v += dpp_or_0<0x111, 0xf>(v);
  v += dpp_or_0<0x112, 0xf>(v);
  v += dpp_or_0<0x114, 0xf>(v);
  v += dpp_or_0<0x118, 0xf>(v);
  v += dpp_or_0<0x142, 0xa>(v);
  v += dpp_or_0<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ u64_t lane64(u64_t v, int l) {
  return (static_cast<u64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), l))) << 32) |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), l));
}

// 2^(43 + i / 256), by the exponential's series.
struct Roots {
  double r[256];
  constexpr Roots() : r{} {
    for (int i = 0; i < 256; ++i) {
      double sum = 1.0, term = 1.0;
      for (int n = 1; n < 24; ++n) {
        term *= i * (0.6931471805599453 / 256.0) / n;
        sum += term;
      }
      r[i] = sum * static_cast<double>(kOne);
    }
  }
};
__device__ constexpr Roots kRoots{};

// The row as its weights' function needs it.
struct RowScale {
  float fmax;        // the largest entry
  float bins;        // bins a unit of the logits
  double max, rate;  // 256 log2(e) / T
  bool odd;          // infinite logits, or a temperature next to 0: the largest weigh 1, others 0
};

// An entry's weight: 2^(z / 256) by a table of 256 roots and a polynomial in the rest of z, whose
// relative error is 2^-54 in exact arithmetic.  2^-46 and less round to 0 all alike: z ends there,
// as what follows adds z >> 8 to an exponent, which must not wrap (-inf, and the NaN of -inf
// times a rate of 0, end there too).  So every entry can be weighed, kept or not.
__device__ __forceinline__ u64_t weight(const SampleShared& sh, const RowScale& r, float v) {
  double z = (static_cast<double>(v) - r.max) * r.rate;
  if (r.odd) z = v == r.fmax ? 0.0 : -INFINITY;  // (inf - inf, or 0 / 0)
  z = __builtin_fmax(z, -46.0 * 256.0);
  // The nearest whole number, and as an integer, from the sum's last bits.
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52
  const double big = z + kMagic;
  const uint32_t i = static_cast<uint32_t>(__double_as_longlong(big));
  const double f = z - (big - kMagic);
  constexpr double c = 0.6931471805599453 / 256.0;
  double e = c * c * c * c / 24.0;
  e = __builtin_fma(e, f, c * c * c / 6.0);
  e = __builtin_fma(e, f, c * c / 2.0);
  e = __builtin_fma(e, f, c);
  e = __builtin_fma(e, f, 1.0);
  e *= sh.roots[i & 255];
  // (The table holds 2^43 as well.)  Times 2^(i >> 8) in its exponent, then rounded to a whole
  // number by the sum with 2^52.
  const u64_t scaled = __double_as_longlong(e) + (static_cast<u64_t>((i & ~255u) << 12) << 32);
  return __double_as_longlong(__longlong_as_double(scaled) + 4503599627370496.0) & 0xfffffffffffffull;
}

__device__ __forceinline__ int bin_of(const RowScale& r, float v) {
  return static_cast<int>(fminf((r.fmax - v) * r.bins, static_cast<float>(kBins - 1)));
}

// A row's entries: a wave has a run of 256 n_it of them, 256 a step, four a lane.  Loads go without
// regard to alignment (ld and the row's place may be odd); the row's last four entries are loaded
// whole by every lane that reaches past them, and what is not its own becomes -inf, as a NaN does.
// Every pass reads the row anew, out of the caches: kept in registers (49 for 50 thousand
// entries) the passes have to be unrolled over them, and wait for their own instructions.
// TINY: rows of fewer than four entries.
template <typename T, bool TINY> struct RowValues {
  typedef T vec_t __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  const T* row;
  int V, n_it;

  __device__ __forceinline__ RowValues(const T* r, int n)
      : row(r), V(n), n_it((n + 4 * kSampleThreads - 1) / (4 * kSampleThreads)) {}
  __device__ __forceinline__ int index(int wave, int it) const {
    return 4 * ((wave * n_it + it) * 64 + static_cast<int>(threadIdx.x & 63));
  }
  __device__ __forceinline__ vec_t load(int i) const {
    if (TINY) return vec_t{};
    return *reinterpret_cast<const vec_t*>(row + min(i, V - 4));
  }
  // The four values from index i on (`raw` as loaded), -inf in the place of the row's earlier ones
  // where they begin in front of i; the first one's index.
  __device__ __forceinline__ int values(int i, const vec_t& raw, float (&v)[4]) const {
    if (TINY) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = i + e < V ? fmaxf(Elem<T>::load(row + i + e), -INFINITY) : -INFINITY;
      return i;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const T x = raw[e];
      v[e] = fmaxf(Elem<T>::load(&x), -INFINITY);
    }
    if (i > V - 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = V - 4 + e < i ? -INFINITY : v[e];
      return V - 4;
    }
    return i;
  }
  // f(index of the first of four entries, their values), in order; NI loads a run, the next run's
  // on their way meanwhile.
  template <int NI, typename F> __device__ __forceinline__ void each(int wave, F&& f) const {
    vec_t now[NI], next[NI];
#pragma unroll
    for (int it = 0; it < NI; ++it) now[it] = load(index(wave, it));
#pragma unroll 1
    for (int it0 = 0; it0 < n_it; it0 += NI) {
#pragma unroll
      for (int it = 0; it < NI; ++it) next[it] = load(index(wave, it0 + NI + it));
#pragma unroll
      for (int it = 0; it < NI; ++it)
        if (it0 + it < n_it) {
          float v[4];
          const int i = values(index(wave, it0 + it), now[it], v);
          f(i, v);
        }
#pragma unroll
      for (int it = 0; it < NI; ++it) now[it] = next[it];
    }
  }
};

// The inclusive sum over the block's threads up to this one, and the sum of all.
__device__ __forceinline__ u64_t block_scan(SampleShared& sh, u64_t a, u64_t* all) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  a = wave_scan64(a);
  __syncthreads();
  if (lane == 63) sh.wave_a[wave] = a;
  __syncthreads();
  // (Lane l < 16 holds the sum of waves 0 .. l.)
  const u64_t w = wave_scan64(sh.wave_a[lane & 15]);
  *all = lane64(w, 15);
  return wave == 0 ? a : a + lane64(w, wave - 1);
}

// The end of a run of the order: entries above this value, and of this value up to this index.
struct Cut {
  float v;
  int idx;
  __device__ bool keeps(float x, int i) const { return x > v || (x == v && i <= idx); }
};

// The block's values, one a thread of the first n2 (a power of two from 64 on; 0 in the others),
// in falling order: exchanges between lanes by shuffles, between waves through `lds`.
__device__ __forceinline__ u64_t sort_down(u64_t mine, int n2, u64_t* lds) {
  const int tid = threadIdx.x;
  for (int k = 2; k <= n2; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      u64_t other;
      if (j >= 64) {
        __syncthreads();
        lds[tid] = mine;
        __syncthreads();
        other = lds[tid ^ j];
      } else {
        other = shfl64(mine, (tid & 63) ^ j);
      }
      // The lower place of a pair keeps the larger value in falling runs.
      const bool larger = ((tid & j) == 0) == ((tid & k) == 0);
      mine = (mine > other) == larger ? mine : other;
    }
  return mine;
}

// What a pass over the row does.
enum SamplePass {
  kGather,  // entries of the range into the list
  kCount,   // a histogram of the range
  kEnds,    // the range's smallest and largest value
  kSum      // kept weights, the cut bin's entries into the list
};
// What it is for.
enum SamplePhase {
  kBound,  // all entries from a value on, which hold all that top_k or min_p keep
  kTopK,   // the end of the first top_k entries
  kTopP,   // the end of the run that has top_p of their weight
  kDraw    // the draw
};

template <typename T, bool TINY>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs a) {
  __shared__ SampleShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x;
  const RowValues<T, TINY> row(static_cast<const T*>(a.x) + b * a.ld, a.V);

  if (tid < 256) sh.roots[tid] = kRoots.r[tid];
  for (int i = tid; i < kBins; i += kSampleThreads) sh.mass[i] = 0;
  // ---- the maximum
  float best = -INFINITY;
  row.template each<4>(wave, [&](int, const float (&v)[4]) { best = fmaxf(fmaxf(fmaxf(best, v[0]), fmaxf(v[1], v[2])), v[3]); });
  float fmax_row = wave_max(best);
  if (lane == 0) sh.wave_a[wave] = __float_as_uint(fmax_row);
  __syncthreads();
  fmax_row = wave_max(__uint_as_float(static_cast<uint32_t>(sh.wave_a[lane & 15])));
  const double T0 = a.t != nullptr ? static_cast<double>(a.t[b]) : a.t1;
  if (!(fmax_row > -INFINITY) || !(T0 > 0.0)) {
    // Nothing to choose from, or the most likely token, the first of equals.
    if (tid == 0) sh.sel_lo = 0xffffffffu;
    __syncthreads();
    uint32_t at = 0xffffffffu;
    row.template each<2>(wave, [&](int i, const float (&v)[4]) {
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (v[e] == fmax_row && v[e] > -INFINITY) at = min(at, static_cast<uint32_t>(i + e));
    });
    if (at != 0xffffffffu) atomicMin(&sh.sel_lo, at);
    __syncthreads();
    if (tid == 0) a.ids[b] = static_cast<int>(sh.sel_lo);
    return;
  }
  RowScale r;
  r.fmax = fmax_row;
  r.max = r.fmax;
  const double per_t = 1.4426950408889634 / T0;
  r.rate = 256.0 * per_t;
  r.odd = !(r.max < INFINITY) || !(r.rate < INFINITY);
  r.bins = static_cast<float>(per_t * (kBins / static_cast<double>(kReach)));

  const int64_t k = a.k != nullptr ? a.k[b] : a.k1;
  const double p = a.p != nullptr ? static_cast<double>(a.p[b]) : a.p1;
  const double m = a.m != nullptr ? static_cast<double>(a.m[b]) : a.m1;
  const bool by_k = k > 0 && k < a.V, by_p = p < 1.0;
  const double part = by_p ? fmax(p, 0.0) : 1.0;
  const u64_t least = m > 0.0 ? static_cast<u64_t>(__builtin_ceil(fmin(m, 1.0) * static_cast<double>(kOne))) : 1;
  const double u = fmin(fmax(static_cast<double>(a.u[b]), 0.0), 1.0);
  auto part_of = [&](u64_t all) {
    const u64_t t = static_cast<u64_t>(__builtin_ceil(part * static_cast<double>(all)));
    return t < 1 ? u64_t{1} : t > all ? all : t;
  };

  Cut in{-INFINITY, -1}, cut = in;      // what earlier cuts leave; the cut that is looked for
  float lo = -INFINITY, hi = INFINITY;  // the range that holds the cut: values from lo to hi, of one bin
  int bin0 = -1;
  uint32_t hi_key = 0;
  int bits = 0;                         // keys a bin, below the first level
  bool first_level = true;
  u64_t target = 0, before = 0;         // entries (weight) that the run needs; those in front of the range
  int pass, phase;

  // The bin of the histogram in which the running sum reaches target; `before` moves up to it.
  auto find_bin = [&](auto&& target_of) {
    const u64_t f0 = sh.mass[2 * tid], f1 = sh.mass[2 * tid + 1];
    sh.mass[2 * tid] = sh.mass[2 * tid + 1] = 0;  // for the next
    u64_t all;
    const u64_t s2 = block_scan(sh, f0 + f1, &all) + before, s1 = s2 - f1, s0 = s1 - f0;
    target = target_of(all);
    if (s0 < target && target <= s2) {
      sh.sel_bin = 2 * tid + (target <= s1 ? 0 : 1);
      sh.sel_a = target <= s1 ? s0 : s1;
    }
    __syncthreads();
    const bool found = target <= before + all;
    const int bin = sh.sel_bin;
    if (found) before = sh.sel_a;
    return found ? bin : kBins - 1;
  };
  // Lanes that take their entry put it into the wave's list, n_mine long.
  int n_mine = 0;
  auto enlist = [&](bool take, float v, int i) {
    const uint64_t who = __builtin_amdgcn_ballot_w64(take);
    if (who == 0) return;
    const int at = n_mine + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32),
                                                      __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), 0));
    if (take && at < kWaveList) sh.found[wave][at] = place(v, i);
    n_mine += __popcll(who);
  };
  // The waves' lists as one, and its length; kList + 1 where one of them was too short.
  auto join_lists = [&]() -> int {
    if (lane == 0) sh.n_found[wave] = n_mine;
    __syncthreads();
    const int n = sh.n_found[lane & 15];
    if (__builtin_amdgcn_ballot_w64(n > kWaveList) != 0) return kList + 1;
    int before_me = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) {
      const int nw = __builtin_amdgcn_readlane(n, w);
      before_me += w < wave ? nw : 0;
      all += nw;
    }
    if (all <= kList)
      for (int j = lane; j < n_mine; j += 64) sh.list[before_me + j] = sh.found[wave][j];
    __syncthreads();
    return all;
  };

  // The lower end of a bin, and a little more for the roundings (of the last, which is open: none).
  auto bin_end = [&](int bin) {
    const float end = r.fmax - (static_cast<float>(bin) + 1.5f) / r.bins;
    return bin < kBins - 1 && end > -INFINITY ? end : -INFINITY;
  };
  // Entries below `lightest` weigh nothing (a little less, for the roundings).
  const float slack = fabsf(r.fmax) * 0x1p-20f;
  const float lightest = fmaxf(r.fmax - static_cast<float>(kReach * 0.6931471805599453 * (1.0 + 0x1p-20) * T0) - slack, -INFINITY);
  bool enough = true;  // the range holds all that is kept, however few
  if (__syncthreads_count(best >= lightest) <= kList / 2) lo = lightest;  // (of the threads have more)
  if (!by_k && !by_p && m > 0.0)
    lo = fmaxf(lo, r.fmax + 0.6931472f * static_cast<float>(T0) * (__builtin_amdgcn_logf(static_cast<float>(fmin(m, 1.0))) * (1.f + 0x1p-18f) - 0x1p-18f) - slack);
  if (by_k && k <= kShort) {
    // The k-th largest of the threads' largest entries is at most the k-th largest entry; the lower
    // end of its bin, and a little more for the roundings, do as well.
    if (best > -INFINITY) atomicAdd(&sh.mass[bin_of(r, best)], u64_t{1});
    __syncthreads();
    const int bin = find_bin([&](u64_t) { return static_cast<u64_t>(k); });
    before = 0;
    const float low = bin_end(bin);
    if (low > lo) {
      lo = low;
      enough = false;
    }
  }
  phase = lo > -INFINITY ? kBound : by_k ? kTopK : by_p ? kTopP : kDraw;
  pass = phase == kBound ? kGather : phase == kDraw ? kSum : kCount;

  // ---- passes over the row, each followed by what its phase makes of it
  for (;;) {
    __syncthreads();
    if (tid == 0) {
      sh.sel_lo = 0xffffffffu;
      sh.sel_hi = 0;
    }
    const bool by_mass = phase == kTopP;
    // Where the cut falls among equal entries their number is added up.
    const bool ties = pass == kSum && (phase == kTopK || (phase == kTopP && !first_level));
    const bool in_bins = pass == kSum && phase == kTopP && !ties, weigh = (by_mass && !ties) || phase == kDraw;
    // Nothing below this counts in the pass (nor does -inf: the smallest number is above it).
    const float floor_v = fmaxf(fmaxf(weigh ? fmaxf(lo, lightest) : lo, in_bins ? bin_end(bin0) : cut.v), -3.4028235e38f);
    float v0 = INFINITY, v1 = -INFINITY;
    u64_t sum = 0;
    n_mine = 0;
    if (phase == kBound) {
      row.template each<4>(wave, [&](int i, const float (&v)[4]) {
        if (__builtin_amdgcn_ballot_w64(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= floor_v) != 0)
#pragma unroll
          for (int e = 0; e < 4; ++e) enlist(v[e] >= floor_v, v[e], i + e);
      });
    } else {
      row.template each<2>(wave, [&](int i, const float (&v)[4]) {
        if (__builtin_amdgcn_ballot_w64(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= floor_v) == 0) return;
        bool takes[4];
        int bin[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          takes[e] = v[e] >= floor_v && v[e] <= hi && in.keeps(v[e], i + e);
          bin[e] = bin0 < 0 && pass != kCount ? -1 : first_level ? bin_of(r, v[e]) : static_cast<int>((hi_key - order_key(v[e])) >> bits);
        }
        if (pass == kGather || in_bins) {
#pragma unroll
          for (int e = 0; e < 4; ++e) enlist(takes[e] && bin[e] == bin0, v[e], i + e);
          // (in is the cut so far: bins above the cut's are kept whole.)
#pragma unroll
          for (int e = 0; e < 4; ++e) takes[e] = takes[e] && bin[e] < bin0;
        }
        if (pass == kCount || pass == kSum) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const u64_t w = weigh ? weight(sh, r, v[e]) : 1;
            if (pass == kCount) {
              if (takes[e]) atomicAdd(&sh.mass[bin[e]], w);
            } else {
              sum += takes[e] && (ties || w >= least) ? w : 0;
            }
          }
        } else if (pass == kEnds) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (takes[e] && bin[e] == bin0) {
              v0 = fminf(v0, v[e]);
              v1 = fmaxf(v1, v[e]);
            }
        }
      });
    }
    __syncthreads();

    if (pass == kCount) {
      const int bin = find_bin([&](u64_t all) {
        return !first_level ? target : phase == kTopK ? (static_cast<u64_t>(k) > all ? u64_t{0} : static_cast<u64_t>(k)) : part_of(all);
      });
      if (target == 0) {  // fewer than top_k to choose from
        phase = by_p ? kTopP : kDraw;
        pass = by_p ? kCount : kSum;
        before = 0;
        continue;
      }
      if (first_level) {
        bin0 = bin;
      } else {
        bin0 = -1;
        hi_key -= static_cast<uint32_t>(bin) << bits;
        lo = fmaxf(lo, key_value(hi_key - ((1u << bits) - 1u)));
        hi = key_value(hi_key);
      }
      pass = first_level && phase == kTopP ? kSum : kGather;
      continue;
    }
    if (pass == kEnds) {
      v1 = wave_max(v1);
      v0 = -wave_max(-v0);
      if (lane == 0) {
        atomicMin(&sh.sel_lo, order_key(v0));
        atomicMax(&sh.sel_hi, order_key(v1));
      }
      __syncthreads();
      const uint32_t lo_key = sh.sel_lo;
      hi_key = sh.sel_hi;
      lo = key_value(lo_key);
      hi = key_value(hi_key);
      first_level = false;
      bin0 = -1;
      bits = lo_key == hi_key ? 0 : max(0, 32 - __builtin_clz(hi_key - lo_key) - 11);
      pass = lo_key == hi_key ? kSum : kCount;  // all the same: the first of them by index
      continue;
    }
    if (pass == kSum) {
      sum = wave_scan64(sum);
      if (lane == 63) sh.sums[wave] = sum;
      __syncthreads();
    }
    if (pass == kGather || in_bins) {
      const int c = join_lists();
      if (!(c <= kList && (phase != kBound || enough || c >= k))) {
        // ---- a longer list than it can be: narrow the range, or leave the bound
        if (phase == kBound) {
          phase = by_k ? kTopK : by_p ? kTopP : kDraw;
          pass = phase == kDraw ? kSum : kCount;
          lo = -INFINITY;
        } else {
          pass = kEnds;
        }
        continue;
      }
      // ---- the list in order; the last entry that stays is the cut
      u64_t mine = tid < c ? sh.list[tid] : 0, front = 0, w;
      int ahead = 0;
      auto value = [&]() -> u64_t {
        return mine == 0 ? 0 : phase != kTopK ? weight(sh, r, key_value(static_cast<uint32_t>(mine >> 32))) : 1;
      };
      if (c <= kPairs) {
        w = value();
        if (tid < c) sh.list_w[tid] = w;
        __syncthreads();
        if (tid < c)
#pragma unroll 8
          for (int j = 0; j < c; ++j) {
            const bool first = sh.list[j] > mine;
            ahead += first ? 1 : 0;
            front += first ? sh.list_w[j] : 0;
          }
      } else {
        mine = sort_down(mine, 1 << (32 - __builtin_clz(c - 1)), sh.list);
        w = value();
        u64_t all;
        front = block_scan(sh, w, &all) - w;
        ahead = tid;
      }
      bool stays = mine != 0;
      if (phase == kBound) {
        stays = stays && (!by_k || ahead < k);
        if (by_p) {
          u64_t all;
          block_scan(sh, stays ? w : 0, &all);
          stays = stays && front < part_of(all);
        }
      } else {
        stays = stays && before + front < target;
      }
      if (tid == 0) sh.sel_a = ~u64_t{0};
      if (phase == kBound && tid < kSampleWaves) sh.sums[tid] = 0;
      __syncthreads();
      if (stays) atomicMin(&sh.sel_a, mine);
      if (stays && phase != kTopK && w >= least)
        // What stays is the draw's, or belongs to it beside the bins above.
        atomicAdd(&sh.sums[(~static_cast<uint32_t>(mine) >> 8) / static_cast<uint32_t>(row.n_it)], w);
      __syncthreads();
      cut = Cut{key_value(static_cast<uint32_t>(sh.sel_a >> 32)), static_cast<int>(~static_cast<uint32_t>(sh.sel_a))};
      if (phase == kBound || in_bins) phase = kDraw;
    }
    if (pass == kSum || phase == kDraw) {
      // ---- the draw: the wave's run, then its step, then the entry
      auto drawn = [&](float v, int i) -> u64_t {
        if (ties) return v == lo && in.keeps(v, i) ? 1 : 0;
        if (!cut.keeps(v, i)) return 0;
        const u64_t w = weight(sh, r, v);
        return w >= least ? w : 0;
      };
      const u64_t runs = wave_scan64(lane < kSampleWaves ? sh.sums[lane & 15] : 0), total = lane64(runs, 15);
      u64_t goal = static_cast<u64_t>(u * static_cast<double>(total));
      if (goal >= total) goal = total - 1;
      if (ties) {
        const u64_t w = by_mass ? weight(sh, r, lo) : 1;
        goal = (target - before + w - 1) / w - 1;
      }
      const int run = __builtin_ctzll(__builtin_amdgcn_ballot_w64(runs > goal));
      const u64_t front = run == 0 ? 0 : lane64(runs, run - 1);
      for (int it = wave; it < row.n_it; it += kSampleWaves) {
        const int i0 = row.index(run, it);
        float v[4];
        const int i = row.values(i0, row.load(i0), v);
        u64_t s = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) s += drawn(v[e], i + e);
        s = wave_scan64(s);
        if (lane == 63) sh.its[it] = s;
      }
      __syncthreads();
      if (wave == 0) {
        u64_t at = front;
        int step = 0;
        for (int it0 = 0; it0 < row.n_it; it0 += 64) {
          const u64_t s = at + wave_scan64(it0 + lane < row.n_it ? sh.its[it0 + lane] : 0);
          const uint64_t past = __builtin_amdgcn_ballot_w64(s > goal);
          if (past != 0) {
            const int l = __builtin_ctzll(past);
            step = it0 + l;
            if (l > 0) at = lane64(s, l - 1);
            break;
          }
          at = lane64(s, 63);
        }
        const int i0 = row.index(run, step);
        float v[4];
        const int i = row.values(i0, row.load(i0), v);
        u64_t w4[4], s = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w4[e] = drawn(v[e], i + e);
          s += w4[e];
        }
        at += wave_scan64(s) - s;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (at <= goal && goal < at + w4[e]) {
            if (ties)
              sh.sel_idx = i + e;
            else
              a.ids[b] = i + e;
          }
          at += w4[e];
        }
      }
      if (!ties) return;
      __syncthreads();
      cut = Cut{lo, sh.sel_idx};
    }
    // ---- a cut is made: the next
    in = cut;
    const bool more = phase == kTopK && by_p;
    phase = more ? kTopP : kDraw;
    pass = more ? kCount : kSum;
    first_level = true;
    lo = -INFINITY;
    hi = INFINITY;
    bin0 = -1;
    before = 0;
  }
}

template <typename T> static int launch_sample(const SampleArgs& a, int rows, hipStream_t s) {
  if (a.V < 4)
    hipLaunchKernelGGL((sample_kernel<T, true>), dim3(rows), dim3(kSampleThreads), 0, s, a);
  else
    hipLaunchKernelGGL((sample_kernel<T, false>), dim3(rows), dim3(kSampleThreads), 0, s, a);
  return hip_status(hipGetLastError());
}

}  // namespace cgpt

extern "C" int cgpt_sample(const void* x, int64_t rows, int64_t cols, int64_t ld, int dtype, const float* u,
                           const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                           double temperature_all, int64_t top_k_all, double top_p_all, double min_p_all, int64_t* ids,
                           void* stream) {
  using namespace cgpt;
  if (rows < 0 || cols <= 0 || ld < cols) return CGPT_EINVAL;
  if (dtype != CGPT_F32 && dtype != CGPT_BF16 && dtype != CGPT_F16) return CGPT_EDTYPE;
  if (cols > kMaxVocab || rows > (0xffffffffll / kSampleThreads)) return CGPT_ESHAPE;
  if ((temperature == nullptr && !(temperature_all >= 0.0)) || (top_k == nullptr && top_k_all < 0) ||
      (top_p == nullptr && !(top_p_all >= 0.0)) || (min_p == nullptr && !(min_p_all >= 0.0 && min_p_all <= 1.0)))
    return CGPT_EINVAL;
  if (rows == 0) return CGPT_OK;
  if (x == nullptr || u == nullptr || ids == nullptr) return CGPT_EINVAL;
  const uintptr_t low = dtype == CGPT_F32 ? 3 : 1;
  if ((reinterpret_cast<uintptr_t>(x) & low) || (reinterpret_cast<uintptr_t>(ids) & 7)) return CGPT_EINVAL;
  for (const void* q : {static_cast<const void*>(u), static_cast<const void*>(temperature), static_cast<const void*>(top_k),
                        static_cast<const void*>(top_p), static_cast<const void*>(min_p)})
    if (reinterpret_cast<uintptr_t>(q) & 3) return CGPT_EINVAL;
  const SampleArgs a{x, u, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all, ld,
                     static_cast<int>(cols), ids};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == CGPT_BF16) return launch_sample<bf16_t>(a, static_cast<int>(rows), s);
  if (dtype == CGPT_F16) return launch_sample<f16_t>(a, static_cast<int>(rows), s);
  return launch_sample<float>(a, static_cast<int>(rows), s);
}
