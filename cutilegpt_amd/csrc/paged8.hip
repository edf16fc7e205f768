// Writing the 8-bit paged cache, and reading it back as values.
//
// append8_kernel: the step's keys and values into codes, a power of two for each block of
// tokens and head (see paged8.h), keys and queries turned by their positions on the way.
// read8_kernel: code * 2^e as rows of a wider type.
#include "internal.h"
#include "paged8.h"

namespace cgpt {

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
  int Hq, Hkv, rot_dim, n_pos, interleaved;
  int per_item, units4;  // blocks of tokens an item; ceil(heads / 4)
  FastDiv width;         // positions an item, per_item * block
  int* err;
};

// A double as a float whose last bit is set when something was cut off: rounding that
// to a type of 22 bits or fewer gives what rounding the double would, and so do comparisons
// with its numbers.
__device__ __forceinline__ float to_odd(double r) {
  const float f = __double2float_rz(r);
  return static_cast<double>(f) == r ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// Eight values of a row from x0 on, turned by the angles `cs`.  Products of two floats are
// exact in 64 bits, so a turned value is rounded once, to 53 bits: a code is what rounding
// the exact value would give, but for one in some 2^40.
template <typename T>
__device__ __forceinline__ void turned8(const T* row, int x0, int rot_dim, int interleaved, const float* cs, double* y) {
  const int half = rot_dim / 2;
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; i += Elem<T>::kVec) load_vec(row + x0 + i, x + i);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x[i];
  if (x0 >= rot_dim) return;
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      if (x0 + i < rot_dim) {
        const double c = cs[(x0 + i) / 2], s = cs[half + (x0 + i) / 2];
        y[i] = x[i] * c - x[i + 1] * s;
        y[i + 1] = x[i + 1] * c + x[i] * s;
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = x0 + i;
    if (d >= rot_dim) break;
    const int at = d < half ? d : d - half;
    const double c = cs[at], s = cs[half + at], z = Elem<T>::load(row + (d < half ? d + half : at));
    y[i] = d < half ? x[i] * c - z * s : x[i] * c + z * s;
  }
}

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A wave takes an item: per_item neighbouring blocks of one sequence, of one head of the
// keys, the values or the queries; the sequence's items are those that its step touches.
// Lanes take 8 values each of a row.  First the largest value of every block (in LDS), then its
// exponent, then the codes.  The rows are read twice, the second time from the cache.
template <typename T, int CODE, int HD>
__global__ __launch_bounds__(256) void append8_kernel(Append8Args a) {
  constexpr int LPR = HD / 8, RPI = 64 / LPR, kMost = 32;
  __shared__ uint32_t top[4][kMost];
  __shared__ int exps[4][kMost];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int slot = static_cast<int>(blockIdx.x) / a.units4;
  const int unit = (static_cast<int>(blockIdx.x) - slot * a.units4) * 4 + wave;
  if (unit >= 2 * a.Hkv + (a.q != nullptr ? a.Hq : 0)) return;
  // Sequence b has the slots from start(b) on, as many as its items and more.
  int b = slot;
  if (a.seq.cu == nullptr) {
    slot = 0;
  } else {
    auto start = [&](int i) { return a.width.div(min(max(a.seq.cu[i], 0), a.seq.n_tokens)) + 2 * i; };
    b = wave_count(a.seq.B, lane, [&](int i) { return start(i + 1) <= slot; });
    if (b < a.seq.B) slot -= start(b);
  }
  if (b >= a.seq.B || slot < 0) return;
  int first, count;
  seq_tokens(a.seq, b, &first, &count);
  // (A length past 2^30, which no table has, is cut there: positions stay far from 2^31.)
  const int len = min(max(a.seq.lens[b], 0), 1 << 30), pos0 = len - count;  // the first token's position
  const int W = static_cast<int>(a.width.d), blk = static_cast<int>(a.quant.block.d);
  const int page_size = static_cast<int>(a.seq.page.d);
  const int lo = max(pos0, 0), hi = min(len, a.seq.cap);
  bool flag = len > a.seq.cap && count > 0;
  const int64_t base64 = (static_cast<int64_t>(a.width.div(lo)) + slot) * W;
  const bool is_q = unit >= 2 * a.Hkv, is_v = !is_q && unit >= a.Hkv;
  const int h = is_q ? unit - 2 * a.Hkv : is_v ? unit - a.Hkv : unit;
  // (Queries past the table are still turned.)
  const int end_all = is_q ? len : hi;
  if (base64 >= end_all) {
    if (flag && a.err != nullptr && lane == 0) *a.err = 1;
    return;
  }
  const int base = static_cast<int>(base64);
  const int p0 = max(lo, base), p1 = static_cast<int>(min(static_cast<int64_t>(end_all), base64 + W));
  const T* const src = static_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k) + h * (is_q ? a.q_sh : is_v ? a.v_sh : a.k_sh);
  const int64_t st = is_q ? a.q_st : is_v ? a.v_st : a.k_st;
  const int x0 = lane % LPR * 8, r = lane / LPR;
  const int rot = is_v ? 0 : a.rot_dim;
  auto load = [&](int pos, double* y) __attribute__((always_inline)) {
    const bool off = rot > 0 && pos >= a.n_pos;
    flag |= off;
    const float* cs = a.rot + (rot > 0 ? (off ? a.n_pos - 1 : pos) * a.rot_stride : 0);
    turned8<T>(src + (first + (pos - pos0)) * st, x0, rot, a.interleaved, cs, y);
  };
  if (is_q) {
    for (int p = p0 + r; p < p1; p += RPI) {
      double y[8];
      float f[8];
      load(p, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = sizeof(T) == 4 ? static_cast<float>(y[i]) : to_odd(y[i]);
      T* const dst = static_cast<T*>(a.q_out) + (first + (p - pos0)) * a.qo_st + h * a.qo_sh + x0;
#pragma unroll
      for (int i = 0; i < 8; i += Elem<T>::kVec) store_vec(dst + i, f + i);
    }
    if (flag && a.err != nullptr) *a.err = 1;
    return;
  }
  if (lane < kMost) top[wave][lane] = 0;
  wave_sync();
  for (int p = p0 + r; p < p1; p += RPI) {
    double y[8];
    load(p, y);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = __float_as_uint(to_odd(y[i])) & 0x7fffffffu;
      if (bits < 0x7f800000u)
        m = max(m, bits);
      else
        flag = true;  // not finite: the block's exponent goes by the others
    }
    atomicMax(&top[wave][a.quant.block.div(p - base)], m);
  }
  wave_sync();
  // Lane i: the exponent of block i.
  const ScalePool& sp = is_v ? a.quant.vs : a.quant.ks;
  const PagePool& pool = is_v ? a.vc : a.kc;
  const int* const trow = a.seq.table + b * a.seq.stride;
  int grown = 0;  // lane 0: bytes that the exponent of the block at p0 grew by
  const int i0 = a.quant.block.div(p0 - base);
  if (lane < a.per_item) {
    const int first_p = base + lane * blk;
    if (first_p < p1 && first_p + blk > p0) {
      const int col = a.seq.page.div(first_p);
      const int page = page_of(trow, col, a.seq.n_pages, &flag);
      const bool there = static_cast<uint32_t>(trow[col]) < static_cast<uint32_t>(a.seq.n_pages);
      uint8_t* const at = sp.base + page * sp.sp + h * sp.sh + a.quant.block.div(first_p - col * page_size) * sp.sb;
      int e = Codec<CODE>::exponent(top[wave][lane]);
      if (first_p < p0 && there) {
        const int old = clamp_exp<CODE>(*at);
        e = max(e, old);
        grown = e - old;
      }
      if (there) *at = static_cast<uint8_t>(e);
      exps[wave][lane] = there ? e : -1;
    }
  }
  wave_sync();
  grown = __builtin_amdgcn_readlane(grown, i0);
  uint8_t* const dst = static_cast<uint8_t*>(pool.base) + h * pool.sh + x0;
  auto slot_of = [&](int p) __attribute__((always_inline)) {
    const int col = a.seq.page.div(p);
    return dst + trow[col] * pool.sp + (p - col * page_size) * pool.ss;
  };
  if (grown > 0) {
    // Rows that were there: shifted to the new exponent.
    const float f = __uint_as_float(static_cast<uint32_t>(max(127 - grown, 0)) << 23);
    for (int p = base + i0 * blk + r; p < p0; p += RPI) {
      uint8_t* const at = slot_of(p);
      u32x2_t w = *reinterpret_cast<const u32x2_t*>(at);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float y[4];
        Codec<CODE>::decode4(w[i], y);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] *= f;
        w[i] = Codec<CODE>::encode4(y);
      }
      *reinterpret_cast<u32x2_t*>(at) = w;
    }
  }
  for (int p = p0 + r; p < p1; p += RPI) {
    const int e = exps[wave][a.quant.block.div(p - base)];
    if (e < 0) continue;
    double y[8];
    load(p, y);
    const float f = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_odd(y[i]) * f;
    *reinterpret_cast<u32x2_t*>(slot_of(p)) = u32x2_t{Codec<CODE>::encode4(x), Codec<CODE>::encode4(x + 4)};
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
    const PagePool& pool = is_v ? a.vc : a.kc;
    const ScalePool& sp = is_v ? a.quant.vs : a.quant.ks;
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
                static_cast<int>(p.interleaved), 0, 0, FastDiv(), p.err_flag};
  a.per_item = static_cast<int>(std::max<int64_t>(1, 32 / args->block));
  a.width = FastDiv(a.per_item * args->block);
  a.units4 = static_cast<int>((2 * p.Hkv + (p.q != nullptr ? p.Hq : 0) + 3) / 4);
  const int64_t slots = p.cu_q == nullptr ? p.B : p.n_tokens / a.width.d + 2 * p.B;
  if (slots * a.units4 > kMaxBlocks) return CGPT_ESHAPE;
  const dim3 grid(static_cast<unsigned>(slots * a.units4));
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_types8(*args, [&](auto t, auto code, auto hd) {
    hipLaunchKernelGGL((append8_kernel<decltype(t), decltype(code)::value, decltype(hd)::value>), grid, dim3(256), 0, s, a);
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
