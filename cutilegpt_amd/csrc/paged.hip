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

extern "C" int cgpt_paged_kv_append(const void* q, const void* k, const void* v, void* q_out, void* k_cache,
                                    void* v_cache, const int* block_table, const int* seq_lens,
                                    const int* cu_q, const float* rotary, int64_t n_tokens, int64_t B,
                                    int64_t Hq, int64_t Hkv, int64_t head_dim, int64_t page_size,
                                    int64_t n_pages, int64_t max_pages, int64_t bt_stride, int64_t q_st,
                                    int64_t q_sh, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh,
                                    int64_t qo_st, int64_t qo_sh, int64_t kc_sp, int64_t kc_sh, int64_t kc_ss,
                                    int64_t vc_sp, int64_t vc_sh, int64_t vc_ss, int64_t rot_dim,
                                    int64_t n_pos, int64_t rot_stride, int interleaved, int dtype,
                                    int* err_flag, void* stream) {
  using namespace cgpt;
  const PagePool kc{k_cache, kc_sp, kc_sh, kc_ss}, vc{v_cache, vc_sp, vc_sh, vc_ss};
  const int rc = check_paged(n_tokens, B, Hq, Hkv, head_dim, page_size, n_pages, max_pages, bt_stride, kc, vc, dtype);
  if (rc != CGPT_OK) return rc;
  if (k_cache == v_cache) return CGPT_EINVAL;
  if ((q == nullptr) != (q_out == nullptr)) return CGPT_EINVAL;
  if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 2 != 0) return CGPT_ESHAPE;
  if (rot_dim > 0 && (rotary == nullptr || n_pos <= 0 || rot_stride < rot_dim || n_pos > 0x7fffffff)) return CGPT_EINVAL;
  if (n_tokens == 0 || B == 0) return CGPT_OK;
  if (k == nullptr || v == nullptr || seq_lens == nullptr || (max_pages > 0 && block_table == nullptr)) return CGPT_EINVAL;
  if (cu_q == nullptr && n_tokens != B) return CGPT_EINVAL;
  const int64_t epv = dtype == CGPT_F32 ? 4 : 8;
  for (int64_t st : {q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh})
    if (st < 0 || st % epv != 0) return CGPT_EINVAL;
  for (const void* p : {q, k, v, static_cast<const void*>(q_out)})
    if (reinterpret_cast<uintptr_t>(p) & 15) return CGPT_EINVAL;
  if (reinterpret_cast<uintptr_t>(rotary) & 3) return CGPT_EINVAL;
  AppendArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_out = q_out;
  a.kc = kc;
  a.vc = vc;
  a.seq = PagedBatch{block_table, seq_lens, cu_q, bt_stride, static_cast<int>(n_tokens), static_cast<int>(B),
                     static_cast<int>(n_pages), static_cast<int>(max_pages),
                     static_cast<int>(page_size * max_pages), FastDiv(page_size)};
  a.rot = rotary;
  a.q_st = q_st;
  a.q_sh = q_sh;
  a.k_st = k_st;
  a.k_sh = k_sh;
  a.v_st = v_st;
  a.v_sh = v_sh;
  a.qo_st = qo_st;
  a.qo_sh = qo_sh;
  a.rot_stride = rot_stride;
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.head_dim = static_cast<int>(head_dim);
  a.rot_dim = static_cast<int>(rot_dim);
  a.n_pos = static_cast<int>(n_pos);
  a.interleaved = interleaved;
  a.err = err_flag;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == CGPT_BF16) return launch_append<bf16_t>(a, s);
  if (dtype == CGPT_F16) return launch_append<f16_t>(a, s);
  return launch_append<float>(a, s);
}
