// Writing the paged key-value cache.
//
// append_kernel copies the step's keys and values into their pages and turns keys
// and queries by their positions on the way: (x, y) -> (x c - y s, y c + x s) in 32 bits.
// The bound is the bytes (k, v and q of a token read once and written once): 18 thousand
// tokens, 12 heads of head_dim 64 with queries, bf16, 44 us, 4.3 TB/s where a large copy
// reaches 4.9 (33 us when its 190 MB lie in the 256 MB cache from the call before); or,
// for a decode step, the launch and three dependent loads (length, page id, row): 32 tokens
// x 25 heads 3.7 us.
#include "internal.h"
#include "paged.h"

namespace cgpt {

constexpr int kAppendThreads = 256;

struct AppendArgs {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  PagePool kc, vc;
  PagedBatch seq;
  const float* rot;  // row pos: rot_dim / 2 cosines, then rot_dim / 2 sines
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, rot_stride;
  int Hq, Hkv, head_dim, rot_dim, n_pos, interleaved;
  int* err;
};

// Four floats on a 4-byte boundary (rows of the rotation table may start anywhere).
typedef float f32x4u_t __attribute__((ext_vector_type(4), aligned(4)));

// A block holds `tokens` tokens.  A thread keeps one of a head's pairs of 16-byte chunks
// of one token and goes through the token's heads (keys, values, queries): consecutive
// lanes take the pairs of a head, then the next head, so a wave reads runs of a
// projection's row, and the angles of its values stay in registers.  A pair is what a
// rotation needs: chunks c and c + rot_dim / 2 (pairs of values a half apart), else two
// neighbours.  PAIRS: the halves are whole chunks, or the pairs lie side by side; else
// (rot_dim / 2 no multiple of a chunk) values are turned one by one.
template <typename T, bool PAIRS>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(AppendArgs a, int unit_log2, int tokens_log2) {
  constexpr int EPV = Elem<T>::kVec;
  const int tid = threadIdx.x;
  const int u = tid & ((1 << unit_log2) - 1);
  const int head_log2 = 8 - unit_log2 - tokens_log2;
  const int h0 = (tid >> unit_log2) & ((1 << head_log2) - 1);
  const int t = (blockIdx.x << tokens_log2) + (tid >> (unit_log2 + head_log2));
  if (t >= a.seq.n_tokens) return;
  const int b = seq_of(a.seq, t);
  if (b >= a.seq.B) return;
  int first, count;
  seq_tokens(a.seq, b, &first, &count);
  const int pos = a.seq.lens[b] - count + (t - first);
  if (t < first || pos < 0) return;  // a padding row
  bool bad = pos >= a.seq.cap;
  int slot = 0, page = 0;
  if (!bad) {
    const int col = a.seq.page.div(pos);
    slot = pos - col * static_cast<int>(a.seq.page.d);
    page = page_of(a.seq.table + b * a.seq.stride, col, a.seq.n_pages, &bad);
  }
  const int half = a.rot_dim / 2;
  const bool off = half > 0 && pos >= a.n_pos;
  if ((bad || off) && a.err != nullptr) *a.err = 1;
  const float* cs = a.rot + (off ? a.n_pos - 1 : pos) * a.rot_stride;

  // The thread's two chunks (first value of each), and how its values are turned.
  const int rh = half / EPV;
  const bool apart = PAIRS && !a.interleaved && u < rh;
  const int x0 = (apart ? u : 2 * u) * EPV;
  const int x1 = apart ? x0 + half : x0 + EPV;
  float c[EPV], sn[EPV];
  if (PAIRS) {
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      c[e] = 1.f;
      sn[e] = 0.f;
    }
    if (apart) {
#pragma unroll
      for (int e = 0; e < EPV; e += 4) {
        const f32x4u_t cv = *reinterpret_cast<const f32x4u_t*>(cs + x0 + e);
        const f32x4u_t sv = *reinterpret_cast<const f32x4u_t*>(cs + half + x0 + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          c[e + i] = cv[i];
          sn[e + i] = sv[i];
        }
      }
    } else if (a.interleaved) {
      // Angle e belongs to values x0 + 2 e, x0 + 2 e + 1 of the two neighbours.
#pragma unroll
      for (int e = 0; e < EPV; ++e)
        if (x0 / 2 + e < half) {
          c[e] = cs[x0 / 2 + e];
          sn[e] = cs[half + x0 / 2 + e];
        }
    }
  }
  const int heads = 2 * a.Hkv + (a.q != nullptr ? a.Hq : 0);
  for (int h = h0; h < heads; h += 1 << head_log2) {
    const T* src;
    T* dst;
    bool turned = true;
    if (h < 2 * a.Hkv) {
      if (bad) continue;
      const bool is_v = h >= a.Hkv;
      const int hk = is_v ? h - a.Hkv : h;
      turned = !is_v;
      src = is_v ? static_cast<const T*>(a.v) + t * a.v_st + hk * a.v_sh : static_cast<const T*>(a.k) + t * a.k_st + hk * a.k_sh;
      dst = is_v ? static_cast<T*>(a.vc.base) + page * a.vc.sp + hk * a.vc.sh + slot * a.vc.ss
                 : static_cast<T*>(a.kc.base) + page * a.kc.sp + hk * a.kc.sh + slot * a.kc.ss;
    } else {
      src = static_cast<const T*>(a.q) + t * a.q_st + (h - 2 * a.Hkv) * a.q_sh;
      dst = static_cast<T*>(a.q_out) + t * a.qo_st + (h - 2 * a.Hkv) * a.qo_sh;
    }
    if (PAIRS) {
      u32x4_t r0 = *reinterpret_cast<const u32x4_t*>(src + x0), r1 = *reinterpret_cast<const u32x4_t*>(src + x1);
      if (turned && (apart || a.interleaved) && half > 0) {
        float x[2 * EPV], y[2 * EPV];
        unpack_vec<T>(r0, x);
        unpack_vec<T>(r1, x + EPV);
        if (apart) {
#pragma unroll
          for (int e = 0; e < EPV; ++e) {
            y[e] = x[e] * c[e] - x[EPV + e] * sn[e];
            y[EPV + e] = x[EPV + e] * c[e] + x[e] * sn[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < EPV; ++e) {
            const bool in = x0 / 2 + e < half;  // values past rot_dim go over as they are
            y[2 * e] = in ? x[2 * e] * c[e] - x[2 * e + 1] * sn[e] : x[2 * e];
            y[2 * e + 1] = in ? x[2 * e + 1] * c[e] + x[2 * e] * sn[e] : x[2 * e + 1];
          }
        }
        store_vec(dst + x0, y);
        store_vec(dst + x1, y + EPV);
      } else {
        *reinterpret_cast<u32x4_t*>(dst + x0) = r0;
        *reinterpret_cast<u32x4_t*>(dst + x1) = r1;
      }
    } else {
      // Values 2 u EPV .. + 2 EPV of the pairs' order: the turned pairs, then the rest.
      for (int e = 0; e < EPV; ++e) {
        const int i = u * EPV + e;  // pair i < half is (i, i + half), pair i >= half (2 i, 2 i + 1)
        const int p0 = i < half ? i : 2 * i, p1 = i < half ? i + half : 2 * i + 1;
        if (turned && i < half) {
          const float x = Elem<T>::load(src + p0), y = Elem<T>::load(src + p1);
          Elem<T>::store(dst + p0, x * cs[i] - y * cs[half + i]);
          Elem<T>::store(dst + p1, y * cs[i] + x * cs[half + i]);
        } else {
          const T v0 = src[p0], v1 = src[p1];
          dst[p0] = v0;
          dst[p1] = v1;
        }
      }
    }
  }
}

template <typename T>
static int launch_append(const AppendArgs& a, hipStream_t s) {
  constexpr int EPV = Elem<T>::kVec;
  int unit_log2 = 0;
  while ((2 * EPV << unit_log2) < a.head_dim) ++unit_log2;
  // As many tokens a block as leave eight blocks a CU, so that a wave's writes into a
  // page run over neighbouring slots; a decode step gives each token a block.
  int tokens_log2 = 0;
  while (tokens_log2 < 8 - unit_log2 && (a.seq.n_tokens >> (tokens_log2 + 1)) >= 8 * num_cus()) ++tokens_log2;
  const unsigned blocks = static_cast<unsigned>((a.seq.n_tokens + (1 << tokens_log2) - 1) >> tokens_log2);
  if (blocks > kMaxBlocks) return CGPT_ESHAPE;
  if (a.interleaved || (a.rot_dim / 2) % EPV == 0)
    hipLaunchKernelGGL((append_kernel<T, true>), dim3(blocks), dim3(kAppendThreads), 0, s, a, unit_log2, tokens_log2);
  else
    hipLaunchKernelGGL((append_kernel<T, false>), dim3(blocks), dim3(kAppendThreads), 0, s, a, unit_log2, tokens_log2);
  return hip_status(hipGetLastError());
}

}  // namespace cgpt

extern "C" int cgpt_paged_kv_append(const cgpt_paged_args* args, void* stream) {
  using namespace cgpt;
  bool empty;
  const int rc = check_paged(args, true, &empty);
  if (rc != CGPT_OK) return rc;
  const cgpt_paged_args& p = *args;
  if (p.k_cache == p.v_cache || (p.q == nullptr) != (p.out == nullptr)) return CGPT_EINVAL;
  if (p.rot_dim < 0 || p.rot_dim > p.head_dim || p.rot_dim % 2 != 0) return CGPT_ESHAPE;
  if (p.rot_dim > 0 && (p.rotary == nullptr || (reinterpret_cast<uintptr_t>(p.rotary) & 3) || p.n_pos <= 0 ||
                        p.n_pos > 0x7fffffff || p.rot_stride < p.rot_dim))
    return CGPT_EINVAL;
  if (empty) return CGPT_OK;
  if (p.k == nullptr || p.v == nullptr) return CGPT_EINVAL;
  const AppendArgs a{p.q, p.k, p.v, p.out, PagePool{p.k_cache, p.kc_sp, p.kc_sh, p.kc_ss},
                     PagePool{p.v_cache, p.vc_sp, p.vc_sh, p.vc_ss}, paged_batch(p), p.rotary, p.q_st, p.q_sh, p.k_st,
                     p.k_sh, p.v_st, p.v_sh, p.out_st, p.out_sh, p.rot_stride, static_cast<int>(p.Hq),
                     static_cast<int>(p.Hkv), static_cast<int>(p.head_dim), static_cast<int>(p.rot_dim),
                     static_cast<int>(p.n_pos), static_cast<int>(p.interleaved), p.err_flag};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.dtype == CGPT_BF16) return launch_append<bf16_t>(a, s);
  if (p.dtype == CGPT_F16) return launch_append<f16_t>(a, s);
  return launch_append<float>(a, s);
}
