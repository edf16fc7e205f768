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
// A block takes a row.  It needs the maximum, then a histogram of the logits below it (counts
// and weights), the cut bins' entries, and the sums of the kept weights by segments of the
// vocabulary.
#include "internal.h"
#include "common.h"

namespace cgpt {

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr int kBins = 2048;     // of a histogram
constexpr int kList = 1024;     // entries that are put in order one by one
constexpr int kMaxVocab = 1 << 20;
constexpr int kSegs = kMaxVocab / 256 + kSampleWaves;  // a segment: 4 entries a lane of a wave
constexpr uint64_t kOne = uint64_t{1} << 43;
constexpr float kReach = 44.5f;  // weights below 2^-44 are 0

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
  double exp2_tab[64];
  unsigned long long mass[2][kBins];
  uint32_t count[2][kBins];
  unsigned long long seg[kSegs];
  uint32_t list_key[kList];
  int list_idx[kList];
  unsigned long long list_w[kList];
  unsigned long long wave_a[kSampleWaves], wave_b[kSampleWaves];
  unsigned long long sel_a, sel_b;
  uint32_t sel_key;
  int sel_bin, sel_idx, n_list;
};

// Order of the numbers as order of unsigned integers, 0 for what is never chosen (-inf, NaN);
// both zeros are one.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x > -INFINITY ? b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u) : 0u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ unsigned long long shfl_up64(unsigned long long v, int off) {
  return (static_cast<unsigned long long>(__shfl_up(static_cast<uint32_t>(v >> 32), off, 64)) << 32) |
         __shfl_up(static_cast<uint32_t>(v), off, 64);
}
__device__ __forceinline__ unsigned long long wave_scan64(unsigned long long v, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const unsigned long long w = shfl_up64(v, off);
    if (lane >= off) v += w;
  }
  return v;
}
__device__ __forceinline__ unsigned long long shfl64(unsigned long long v, int l) {
  return (static_cast<unsigned long long>(__shfl(static_cast<uint32_t>(v >> 32), l, 64)) << 32) |
         __shfl(static_cast<uint32_t>(v), l, 64);
}

// The row as its weights' function needs it.
struct RowScale {
  uint32_t top;      // key of the maximum
  double max, rate;  // log2(e) / T
  float fmax, bins;  // level-0 bins a unit of the logits
};

// The weight of an entry: 2^z by a table of 64 roots and a polynomial, |rest| <= 1/128, of
// relative error 2^-54 in exact arithmetic.
__device__ __forceinline__ unsigned long long weight(const SampleShared& sh, const RowScale& r, uint32_t key) {
  if (key == r.top) return kOne;
  if (key == 0) return 0;
  const double z = (static_cast<double>(key_value(key)) - r.max) * r.rate;
  if (!(z > -kReach)) return 0;
  const double n = __builtin_rint(z * 64.0);
  const double f = (z - n * (1.0 / 64.0)) * 0.6931471805599453;
  const int i = static_cast<int>(n);
  double e = 1.0 / 120.0;
  e = __builtin_fma(e, f, 1.0 / 24.0);
  e = __builtin_fma(e, f, 1.0 / 6.0);
  e = __builtin_fma(e, f, 0.5);
  e = __builtin_fma(e, f, 1.0);
  e = __builtin_fma(e, f, 1.0);
  e *= sh.exp2_tab[i & 63];
  // Times 2^(i >> 6) and 2^43, then rounded to a whole number by the sum with 2^52.
  const unsigned long long scaled = __double_as_longlong(e) + (static_cast<unsigned long long>(static_cast<long long>((i >> 6) + 43)) << 52);
  return __double_as_longlong(__longlong_as_double(scaled) + 4503599627370496.0) & 0xfffffffffffffull;
}

__device__ __forceinline__ int level0_bin(const RowScale& r, uint32_t key) {
  return static_cast<int>(fminf((r.fmax - key_value(key)) * r.bins, static_cast<float>(kBins - 1)));
}

// f(first index, keys of four entries) for the thread's entries of the row in order, `it` from 0
// on: entries 4 (1024 it + tid) - shift .. + 3, the shift making loads aligned.  Entries outside
// the row have key 0.
template <typename T, typename F>
__device__ __forceinline__ void for_row(const T* row, int V, int shift, F&& f) {
  typedef T vec_t __attribute__((ext_vector_type(4), aligned(4 * sizeof(T))));
  const int n_it = (V + shift + 4 * kSampleThreads - 1) / (4 * kSampleThreads);
  for (int it = 0; it < n_it; ++it) {
    const int i = 4 * (it * kSampleThreads + static_cast<int>(threadIdx.x)) - shift;
    uint32_t key[4] = {0, 0, 0, 0};
    if (i >= 0 && i + 4 <= V) {
      const vec_t v = *reinterpret_cast<const vec_t*>(row + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const T x = v[e];
        key[e] = order_key(Elem<T>::load(&x));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e >= 0 && i + e < V) key[e] = order_key(Elem<T>::load(row + i + e));
    }
    f(it, i, key);
  }
}

// Inclusive sums of a and b over the block's threads; every thread gets its own.
__device__ __forceinline__ void block_scan2(SampleShared& sh, unsigned long long* a, unsigned long long* b) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  *a = wave_scan64(*a, lane);
  *b = wave_scan64(*b, lane);
  __syncthreads();
  if (lane == 63) {
    sh.wave_a[wave] = *a;
    sh.wave_b[wave] = *b;
  }
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    *a += sh.wave_a[w];
    *b += sh.wave_b[w];
  }
}

// The run's end: entries up to this key, and of this key up to this index.
struct Cut {
  uint32_t key;
  int idx;
  __device__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= idx); }
};

// The shortest run of the order whose count (or weight, by_mass) reaches target >= 1, which the
// whole row does; *through becomes the run's weight.  Level 0 of the histograms is there.
template <typename T>
__device__ Cut find_cut(SampleShared& sh, const RowScale& r, const T* row, int V, int shift, bool by_mass,
                        unsigned long long target, unsigned long long* through) {
  const int tid = threadIdx.x;
  unsigned long long before = 0, mass_before = 0;  // of the entries in front of the range
  int level = 0, bin0 = 0;
  uint32_t lo = 1, hi = 0xffffffffu;  // the range's keys, once level > 0
  auto in_range = [&](uint32_t k) { return k != 0 && (level == 0 ? level0_bin(r, k) == bin0 : k >= lo && k <= hi); };
  uint32_t kmax = 0;
  int sh_bits = 0;
  for (int pass = 0;; ++pass) {
    // ---- the bin that the target lies in
    const int h = pass == 0 ? 0 : 1;
    const uint32_t c0 = sh.count[h][2 * tid], c1 = sh.count[h][2 * tid + 1];
    const unsigned long long m0 = sh.mass[h][2 * tid], m1 = sh.mass[h][2 * tid + 1];
    const unsigned long long f0 = by_mass ? m0 : c0, f1 = by_mass ? m1 : c1;
    unsigned long long a = f0 + f1, b = m0 + m1;
    block_scan2(sh, &a, &b);
    const unsigned long long s0 = before + a - f0 - f1, s1 = s0 + f0;
    if (s0 < target && target <= s1) {
      sh.sel_bin = 2 * tid;
      sh.sel_a = s0;
      sh.sel_b = mass_before + b - m0 - m1;
      sh.n_list = static_cast<int>(c0);
    } else if (s1 < target && target <= s1 + f1) {
      sh.sel_bin = 2 * tid + 1;
      sh.sel_a = s1;
      sh.sel_b = mass_before + b - m1;
      sh.n_list = static_cast<int>(c1);
    }
    __syncthreads();
    const int bin = sh.sel_bin, n = sh.n_list;
    before = sh.sel_a;
    mass_before = sh.sel_b;
    if (pass == 0) {
      bin0 = bin;
    } else {
      level = 1;
      hi = kmax - (static_cast<uint32_t>(bin) << sh_bits);
      lo = sh_bits == 0 ? hi : hi - ((1u << sh_bits) - 1u);
    }
    __syncthreads();
    if (n <= kList) {
      // ---- few: each against all
      if (tid == 0) sh.n_list = 0;
      __syncthreads();
      for_row<T>(row, V, shift, [&](int, int i, const uint32_t (&key)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (in_range(key[e])) {
            const int at = atomicAdd(&sh.n_list, 1);
            if (at < kList) {
              sh.list_key[at] = key[e];
              sh.list_idx[at] = i + e;
              sh.list_w[at] = weight(sh, r, key[e]);
            }
          }
      });
      __syncthreads();
      const int m = min(sh.n_list, kList);
      if (tid < m) {
        const uint32_t k = sh.list_key[tid];
        const int idx = sh.list_idx[tid];
        unsigned long long front = before, mass = mass_before;
        for (int j = 0; j < m; ++j) {
          const uint32_t kj = sh.list_key[j];
          if (kj > k || (kj == k && sh.list_idx[j] < idx)) {
            front += by_mass ? sh.list_w[j] : 1ull;
            mass += sh.list_w[j];
          }
        }
        const unsigned long long own = sh.list_w[tid];
        if (front < target && target <= front + (by_mass ? own : 1ull)) {
          sh.sel_key = k;
          sh.sel_idx = idx;
          sh.sel_a = mass + own;
        }
      }
      __syncthreads();
      const Cut cut{sh.sel_key, sh.sel_idx};
      *through = sh.sel_a;
      __syncthreads();
      return cut;
    }
    // ---- many: the range's ends, then a histogram of its keys
    if (tid == 0) {
      sh.sel_key = 0xffffffffu;  // the smallest
      sh.sel_idx = 0;            // the largest, as an integer
    }
    for (int i = tid; i < kBins; i += kSampleThreads) {
      sh.count[1][i] = 0;
      sh.mass[1][i] = 0;
    }
    __syncthreads();
    uint32_t k0 = 0xffffffffu, k1 = 0;
    for_row<T>(row, V, shift, [&](int, int, const uint32_t (&key)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (in_range(key[e])) {
          k0 = min(k0, key[e]);
          k1 = max(k1, key[e]);
        }
    });
    atomicMin(&sh.sel_key, k0);
    atomicMax(reinterpret_cast<uint32_t*>(&sh.sel_idx), k1);
    __syncthreads();
    const uint32_t kmin = sh.sel_key;
    kmax = static_cast<uint32_t>(sh.sel_idx);
    __syncthreads();
    if (kmin == kmax) {
      // All the same: the first of them by index.
      const unsigned long long w = weight(sh, r, kmin);
      const unsigned long long need = by_mass ? (target - before + w - 1) / w : target - before;
      const int lane = tid & 63, wave = tid >> 6;
      unsigned long long seen = 0;
      for_row<T>(row, V, shift, [&](int, int i, const uint32_t (&key)[4]) {
        int c = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) c += key[e] == kmin ? 1 : 0;
        unsigned long long a = c, b = 0;
        block_scan2(sh, &a, &b);
        unsigned long long at = seen + a - c;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key[e] == kmin && ++at == need) sh.sel_idx = i + e;
        if (tid == kSampleThreads - 1) sh.sel_a = seen + a;
        __syncthreads();
        seen = sh.sel_a;
        __syncthreads();
      });
      const Cut cut{kmin, sh.sel_idx};
      *through = mass_before + need * w;
      __syncthreads();
      return cut;
    }
    level = 1;
    lo = kmin;
    hi = kmax;
    sh_bits = max(0, 32 - __builtin_clz(kmax - kmin) - 11);
    for_row<T>(row, V, shift, [&](int, int, const uint32_t (&key)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (key[e] >= lo && key[e] <= hi && key[e] != 0) {
          const uint32_t at = (kmax - key[e]) >> sh_bits;
          atomicAdd(&sh.count[1][at], 1u);
          atomicAdd(&sh.mass[1][at], weight(sh, r, key[e]));
        }
    });
    __syncthreads();
  }
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs a) {
  __shared__ SampleShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x, V = a.V;
  const T* const row = static_cast<const T*>(a.x) + b * a.ld;
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(row) / sizeof(T) % 4);

  if (tid < 64) sh.exp2_tab[tid] = exp2(tid * (1.0 / 64.0));
  for (int i = tid; i < kBins; i += kSampleThreads) {
    sh.count[0][i] = 0;
    sh.mass[0][i] = 0;
  }
  // ---- the maximum, the first of its equals
  uint32_t best = 0;
  int best_i = 0x7fffffff;
  for_row<T>(row, V, shift, [&](int, int i, const uint32_t (&key)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (key[e] > best) {
        best = key[e];
        best_i = i + e;
      }
  });
  // Larger keys first, then smaller indexes.
  unsigned long long top = (static_cast<unsigned long long>(best) << 32) | static_cast<uint32_t>(~best_i);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const unsigned long long o = shfl64(top, lane ^ off);
    top = o > top ? o : top;
  }
  if (lane == 0) sh.wave_a[wave] = top;
  __syncthreads();
  for (int w = 0; w < kSampleWaves; ++w) top = sh.wave_a[w] > top ? sh.wave_a[w] : top;
  __syncthreads();
  const double T0 = a.t != nullptr ? static_cast<double>(a.t[b]) : a.t1;
  if ((top >> 32) == 0 || !(T0 > 0.0)) {  // nothing to choose from, or the most likely token
    if (tid == 0) a.ids[b] = (top >> 32) == 0 ? -1 : static_cast<int>(~static_cast<uint32_t>(top));
    return;
  }
  RowScale r;
  r.top = static_cast<uint32_t>(top >> 32);
  r.fmax = key_value(r.top);
  r.max = r.fmax;
  r.rate = 1.4426950408889634 / T0;
  r.bins = static_cast<float>(r.rate * (kBins / static_cast<double>(kReach)));

  const int64_t k = a.k != nullptr ? a.k[b] : a.k1;
  const double p = a.p != nullptr ? static_cast<double>(a.p[b]) : a.p1;
  const double m = a.m != nullptr ? static_cast<double>(a.m[b]) : a.m1;
  const bool by_k = k > 0 && k < V, by_p = p < 1.0;
  Cut cut{1, 0x7fffffff};  // everything
  if (by_k || by_p) {
    unsigned long long n = 0, mass = 0;
    for_row<T>(row, V, shift, [&](int, int, const uint32_t (&key)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (key[e] != 0) {
          const int at = level0_bin(r, key[e]);
          const unsigned long long w = weight(sh, r, key[e]);
          ++n;
          mass += w;
          atomicAdd(&sh.count[0][at], 1u);
          if (w != 0) atomicAdd(&sh.mass[0][at], w);
        }
    });
    block_scan2(sh, &n, &mass);
    if (tid == kSampleThreads - 1) {
      sh.sel_a = n;
      sh.sel_b = mass;
    }
    __syncthreads();
    const unsigned long long n_all = sh.sel_a;
    mass = sh.sel_b;
    __syncthreads();
    if (by_k && static_cast<unsigned long long>(k) < n_all)
      cut = find_cut<T>(sh, r, row, V, shift, false, static_cast<unsigned long long>(k), &mass);
    if (by_p) {
      const double part = __builtin_ceil(fmax(p, 0.0) * static_cast<double>(mass));
      unsigned long long target = static_cast<unsigned long long>(part);
      target = target < 1 ? 1 : target > mass ? mass : target;
      cut = find_cut<T>(sh, r, row, V, shift, true, target, &mass);
    }
  }
  const unsigned long long least = m > 0.0 ? static_cast<unsigned long long>(__builtin_ceil(fmin(m, 1.0) * static_cast<double>(kOne))) : 1;

  // ---- kept weights by segments of the vocabulary
  auto kept = [&](uint32_t key, int i) -> unsigned long long {
    if (key == 0 || !cut.keeps(key, i)) return 0;
    const unsigned long long w = weight(sh, r, key);
    return w >= least ? w : 0;
  };
  int n_seg = 0;
  for_row<T>(row, V, shift, [&](int it, int i, const uint32_t (&key)[4]) {
    unsigned long long s = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) s += kept(key[e], i + e);
    s = wave_scan64(s, lane);
    if (lane == 63) sh.seg[it * kSampleWaves + wave] = s;
    n_seg = (it + 1) * kSampleWaves;
  });
  __syncthreads();
  // Threads take runs of segments.
  const int per = (n_seg + kSampleThreads - 1) / kSampleThreads;
  unsigned long long mine = 0, none = 0;
  for (int i = tid * per; i < min(tid * per + per, n_seg); ++i) mine += sh.seg[i];
  unsigned long long incl = mine;
  block_scan2(sh, &incl, &none);
  if (tid == kSampleThreads - 1) sh.sel_a = incl;
  __syncthreads();
  const unsigned long long total = sh.sel_a;
  const double u = fmin(fmax(static_cast<double>(a.u[b]), 0.0), 1.0);
  unsigned long long goal = static_cast<unsigned long long>(u * static_cast<double>(total));
  goal = goal >= total ? total - 1 : goal;
  __syncthreads();
  unsigned long long at = incl - mine;
  if (at <= goal && goal < incl)
    for (int i = tid * per; i < min(tid * per + per, n_seg); ++i) {
      if (goal < at + sh.seg[i]) {
        sh.sel_bin = i;
        sh.sel_a = at;
        break;
      }
      at += sh.seg[i];
    }
  __syncthreads();
  // ---- the segment's entry: one wave
  if (wave != 0) return;
  const int i0 = 4 * (sh.sel_bin * 64 + lane) - shift;
  unsigned long long w4[4], s = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int i = i0 + e;
    w4[e] = i >= 0 && i < V ? kept(order_key(Elem<T>::load(row + i)), i) : 0;
    s += w4[e];
  }
  unsigned long long run = sh.sel_a + wave_scan64(s, lane) - s;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (run <= goal && goal < run + w4[e]) a.ids[b] = i0 + e;
    run += w4[e];
  }
}

template <typename T> static int launch_sample(const SampleArgs& a, int rows, hipStream_t s) {
  hipLaunchKernelGGL((sample_kernel<T>), dim3(rows), dim3(kSampleThreads), 0, s, a);
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
