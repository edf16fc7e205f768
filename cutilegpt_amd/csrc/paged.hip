// Writing the paged key-value cache.
//
// append_kernel copies the step's keys and values into their pages and turns keys
// and queries by their positions on the way.  Nothing is computed that matters: the
// bound is the bytes (each token's k, v and q read once and written once) or, for a
// decode step, the launch.
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

// One block per token; a thread owns element pairs of its heads.
template <typename T>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(AppendArgs a) {
  const int t = blockIdx.x;
  const int b = seq_of(a.seq, t);
  if (b >= a.seq.B) return;
  int first, count;
  seq_tokens(a.seq, b, &first, &count);
  const int pos = a.seq.lens[b] - count + (t - first);
  if (pos < 0) return;  // a padding row
  bool bad = pos >= a.seq.cap;
  int col = 0, slot = 0, page = 0;
  if (!bad) {
    col = a.seq.page.div(pos);
    slot = pos - col * static_cast<int>(a.seq.page.d);
    page = page_of(a.seq.table + b * a.seq.stride, col, a.seq.n_pages, &bad);
  }
  int at = pos;
  bool off = false;
  if (a.rot_dim > 0 && pos >= a.n_pos) {
    off = true;
    at = a.n_pos - 1;
  }
  if ((bad || off) && a.err != nullptr && threadIdx.x == 0) *a.err = 1;
  const float* cs = a.rot + at * a.rot_stride;
  const int half = a.rot_dim / 2, pairs = a.head_dim / 2;
  auto turn = [&](const T* src, T* dst, int i) {
    int x = 2 * i, y = 2 * i + 1;
    if (i < half && !a.interleaved) x = i, y = i + half;
    const float u = Elem<T>::load(src + x), w = Elem<T>::load(src + y);
    if (i < half) {
      const float c = cs[i], s = cs[half + i];
      Elem<T>::store(dst + x, u * c - w * s);
      Elem<T>::store(dst + y, w * c + u * s);
    } else {
      dst[x] = src[x];
      dst[y] = src[y];
    }
  };
  if (!bad)
    for (int i = threadIdx.x; i < a.Hkv * pairs; i += kAppendThreads) {
      const int h = i / pairs, p = i % pairs;
      const T* ks = static_cast<const T*>(a.k) + t * a.k_st + h * a.k_sh;
      const T* vs = static_cast<const T*>(a.v) + t * a.v_st + h * a.v_sh;
      T* kd = static_cast<T*>(a.kc.base) + page * a.kc.sp + h * a.kc.sh + slot * a.kc.ss;
      T* vd = static_cast<T*>(a.vc.base) + page * a.vc.sp + h * a.vc.sh + slot * a.vc.ss;
      turn(ks, kd, p);
      vd[2 * p] = vs[2 * p];
      vd[2 * p + 1] = vs[2 * p + 1];
    }
  if (a.q != nullptr)
    for (int i = threadIdx.x; i < a.Hq * pairs; i += kAppendThreads) {
      const int h = i / pairs, p = i % pairs;
      turn(static_cast<const T*>(a.q) + t * a.q_st + h * a.q_sh,
           static_cast<T*>(a.q_out) + t * a.qo_st + h * a.qo_sh, p);
    }
}

template <typename T>
static int launch_append(const AppendArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(append_kernel<T>, dim3(static_cast<unsigned>(a.seq.n_tokens)), dim3(kAppendThreads), 0, s, a);
  return hip_status(hipGetLastError());
}

}  // namespace cgpt

extern "C" int cgpt_paged_kv_append(const cgpt_paged_args* args, void* stream) {
  using namespace cgpt;
  bool empty;
  const int rc = check_paged(args, &empty);
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
