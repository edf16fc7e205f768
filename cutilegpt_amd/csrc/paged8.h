// What the kernels of the 8-bit paged cache share: the codes, the exponents of their
// blocks, the checks of the entry points.
//
// A cached value is code * 2^e.  The code is an OCP e4m3 number or an int8; e belongs to
// `block` consecutive slots of a page and key head and is held as the byte e + 127.  A power
// of two: a code times 2^e is exact in bf16 (4 or 7 significant bits against 8), so the
// matrix cores take cached values as they are; and where a block's exponent grows as tokens
// are added, its codes are shifted, not rounded to another grid (e4m3: exact above its
// subnormals; int8: the half steps of all shifts add up to less than one step).
// Exponents lie between kMinExp and 119 (e4m3) or 121 (int8): from there up every code's value is
// a normal bf16 number, 2^-kValueDrop of it too; up to there the largest code's value is finite.
#pragma once

#include "paged.h"

namespace cgpt {

constexpr int kMinExp = -100;

// Exponent bytes of a pool: that of (page, head, block) at base + page * sp + head * sh +
// block * sb.
struct ScalePool {
  uint8_t* base;
  int64_t sp, sh, sb;
};

struct Paged8 {
  ScalePool ks, vs;
  FastDiv block;
};

// The checks that the entry points share, as check_paged's.  Pools are bytes here, rows of
// the step (k, v, q, out) of dtype.
inline int check_paged8(const cgpt_paged8_args* args, bool writes, bool* empty) {
  if (args == nullptr) return CGPT_EINVAL;
  const cgpt_paged_args& a = args->p;
  if (a.n_pages <= 0 || a.bt_stride < 0) return CGPT_EINVAL;
  const int rc = check_sizes(a);
  if (rc != CGPT_OK) return rc;
  if (a.n_pages > 0x7fffffff) return CGPT_ESHAPE;
  if (args->code != CGPT_E4M3 && args->code != CGPT_INT8) return CGPT_EDTYPE;
  if (args->block <= 0 || a.page_size % args->block != 0) return CGPT_EINVAL;
  const int64_t blocks = a.page_size / args->block;
  const int64_t pools[2][3] = {{a.kc_sp, a.kc_sh, a.kc_ss}, {a.vc_sp, a.vc_sh, a.vc_ss}};
  const int64_t scales[2][3] = {{args->ks_sp, args->ks_sh, args->ks_sb}, {args->vs_sp, args->vs_sh, args->vs_sb}};
  const void* bases[2] = {a.k_cache, a.v_cache};
  const uint8_t* sbases[2] = {args->k_scale, args->v_scale};
  for (int i = 0; i < 2; ++i) {
    const int64_t *s = pools[i], *e = scales[i], hd = a.head_dim;
    if (bases[i] == nullptr || (reinterpret_cast<uintptr_t>(bases[i]) & 15) || sbases[i] == nullptr) return CGPT_EINVAL;
    if (s[0] % 16 != 0 || s[1] % 16 != 0 || s[2] % 16 != 0) return CGPT_EINVAL;
    if ((a.n_pages > 1 && s[0] < hd) || (a.Hkv > 1 && s[1] < hd) || (a.page_size > 1 && s[2] < hd)) return CGPT_EINVAL;
    if ((a.n_pages > 1 && e[0] < 1) || (a.Hkv > 1 && e[1] < 1) || (blocks > 1 && e[2] < 1)) return CGPT_EINVAL;
    if (writes && (!rows_apart({{a.n_pages, s[0]}, {a.Hkv, s[1]}, {a.page_size, s[2]}}, hd) ||
                   !rows_apart({{a.n_pages, e[0]}, {a.Hkv, e[1]}, {blocks, e[2]}}, 1)))
      return CGPT_EINVAL;
  }
  *empty = a.n_tokens == 0 || a.B == 0;
  if (*empty) return CGPT_OK;
  if (a.seq_lens == nullptr || (a.max_pages > 0 && a.block_table == nullptr)) return CGPT_EINVAL;
  if (a.cu_q == nullptr && a.n_tokens != a.B) return CGPT_EINVAL;
  const int64_t epv = a.dtype == CGPT_F32 ? 4 : 8;
  for (int64_t st : {a.q_st, a.q_sh, a.k_st, a.k_sh, a.v_st, a.v_sh, a.out_st, a.out_sh, args->vo_st, args->vo_sh})
    if (st < 0 || st % epv != 0) return CGPT_EINVAL;
  for (const void* r : {a.q, a.k, a.v, static_cast<const void*>(a.out), static_cast<const void*>(args->v_out)})
    if (reinterpret_cast<uintptr_t>(r) & 15) return CGPT_EINVAL;
  return CGPT_OK;
}

inline Paged8 paged8(const cgpt_paged8_args& a) {
  return Paged8{ScalePool{a.k_scale, a.ks_sp, a.ks_sh, a.ks_sb}, ScalePool{a.v_scale, a.vs_sp, a.vs_sh, a.vs_sb},
                FastDiv(a.block)};
}

// The tile kernel (paged8_tile.hip): every sequence's rows against its keys in job.split parts;
// with job.ml each part leaves (m, l, O) of its rows there, else the results are written.  qt:
// 16-row sub-tiles of each of a block's four waves, 1 or 2.
int launch_paged8_tile(const cgpt_paged8_args& call, const PagedAttnArgs& a, const Paged8& quant, const TileJob& job, int qt,
                       hipStream_t s);

// f(T{}, code, head_dim) with the call's types as compile-time values.
template <typename F> inline int with_types8(const cgpt_paged8_args& a, F&& f) {
  auto by_dim = [&](auto t, auto code) {
    switch (a.p.head_dim) {
      case 16: return f(t, code, std::integral_constant<int, 16>{});
      case 32: return f(t, code, std::integral_constant<int, 32>{});
      case 64: return f(t, code, std::integral_constant<int, 64>{});
      default: return f(t, code, std::integral_constant<int, 128>{});
    }
  };
  auto by_code = [&](auto t) {
    return a.code == CGPT_E4M3 ? by_dim(t, std::integral_constant<int, CGPT_E4M3>{})
                               : by_dim(t, std::integral_constant<int, CGPT_INT8>{});
  };
  if (a.p.dtype == CGPT_BF16) return by_code(bf16_t{});
  if (a.p.dtype == CGPT_F16) return by_code(f16_t{});
  return by_code(float{});
}

#if defined(__HIP_DEVICE_COMPILE__) || defined(__HIPCC__)

// 2^e of an exponent byte; bytes that no append writes count as the nearest that one does.
template <int CODE> __device__ __forceinline__ int clamp_exp(int byte) {
  constexpr int hi = CODE == CGPT_E4M3 ? 119 : 121;
  return min(max(byte, kMinExp + 127), hi + 127);
}
template <int CODE> __device__ __forceinline__ float scale_of(int byte) {
  return __uint_as_float(static_cast<uint32_t>(clamp_exp<CODE>(byte)) << 23);
}

// Values enter the attention's second product 2^kValueDrop smaller, and the weights' sum is made as
// much smaller before it divides.  A weight reaches 2^8 where its score comes up to 8 above the
// running shift, so without that the largest exponents' products would be infinite where the
// result is not (and with the exponent in the weight, int8, inf x 0 a NaN for codes of 0).
// So much holds for one key; a sum of weights times values may still pass fp32 where values
// above 2^120 meet hundreds of keys as heavy as the heaviest.
constexpr int kValueDrop = 8;
constexpr float kSumDrop = 1.f / (1 << kValueDrop);
template <int CODE> __device__ __forceinline__ float value_scale_of(int byte) {
  return __uint_as_float(static_cast<uint32_t>(clamp_exp<CODE>(byte) - kValueDrop) << 23);
}

// The codes.  kTop: the largest code's value.
template <int CODE> struct Codec;

template <> struct Codec<CGPT_E4M3> {
  static constexpr float kTop = 448.f;
  // The smallest exponent byte that leaves values of |x| = the bits `b` within the codes:
  // 448 is 1.75 * 2^8.
  __device__ static int exponent(uint32_t b) {
    return clamp_exp<CGPT_E4M3>(static_cast<int>(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0));
  }
  // Four values in units of the block to codes: to nearest even, a NaN stays one.
  __device__ static uint32_t encode4(const float* y) {
    float c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = y[i] != y[i] ? y[i] : fminf(fmaxf(y[i], -kTop), kTop);
#if defined(__HIP_DEVICE_COMPILE__)
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], w, true));
#else
    return 0;
#endif
  }
  __device__ static void decode4(uint32_t w, float* y) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    y[0] = lo[0];
    y[1] = lo[1];
    y[2] = hi[0];
    y[3] = hi[1];
#endif
  }
};

template <> struct Codec<CGPT_INT8> {
  static constexpr float kTop = 127.f;
  // 127 is 1.984375 * 2^6.
  __device__ static int exponent(uint32_t b) {
    return clamp_exp<CGPT_INT8>(static_cast<int>(b >> 23) - 6 + ((b & 0x7fffffu) > 0x7e0000u ? 1 : 0));
  }
  // A NaN becomes 0: the codes have none.
  __device__ static uint32_t encode4(const float* y) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = y[i] != y[i] ? 0.f : fminf(fmaxf(y[i], -kTop), kTop);
      w |= (static_cast<uint32_t>(static_cast<int>(__builtin_rintf(c))) & 0xffu) << (8 * i);
    }
    return w;
  }
  __device__ static void decode4(uint32_t w, float* y) {
#if defined(__HIP_DEVICE_COMPILE__)
    // Kept a word up to here: else the compiler carries its four bytes in as many registers.
    asm("" : "+v"(w));
#endif
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
  }
};

// Four codes times 2^e (exact in bf16), as two packed pairs.
template <int CODE> __device__ __forceinline__ u32x2_t bf16x4_of(uint32_t w, float scale) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (CODE == CGPT_E4M3) {
    return u32x2_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))};
  } else {
    float y[4];
    Codec<CODE>::decode4(w, y);
    return u32x2_t{pack_bf16x2(y[0] * scale, y[1] * scale), pack_bf16x2(y[2] * scale, y[3] * scale)};
  }
#else
  return u32x2_t{0, 0};
#endif
}

// The queries' values as sums of bf16 parts.
template <typename T> constexpr int kParts = std::is_same<T, bf16_t>::value ? 1 : std::is_same<T, f16_t>::value ? 2 : 3;

// Eight values as NP bf16 fragments.
template <int NP> __device__ __forceinline__ void split_parts(const float* x, u32x4_t (&f)[NP]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = pack_bf16x2(r[2 * i], r[2 * i + 1]);
      f[p][i] = w;
      if (p + 1 < NP) {
        r[2 * i] -= __uint_as_float(w << 16);
        r[2 * i + 1] -= __uint_as_float(w & 0xffff0000u);
      }
    }
}

// e4m3 has one code of either sign that is no number, all ones: the sign bits of such bytes.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

#endif

}  // namespace cgpt
