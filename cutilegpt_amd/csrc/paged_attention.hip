// Attention over the paged key-value cache.
//
// o[i, h] = softmax(scale q[i, h] K^T) V over the keys 0 .. pos(i) of token i's
// sequence, read from its pages; with a shared prefix the first prefix_len keys of
// every sequence are read from one list of pages.
#include "paged.h"

namespace cgpt {

struct PagedAttnArgs {
  const void* q;
  void* o;
  PagePool kc, vc;
  PagedBatch seq;
  const int* prefix;  // pages of the shared prefix
  int prefix_len, prefix_cols;
  int64_t q_st, q_sh, o_st, o_sh;
  int Hq, Hkv;
  float scale_log2;
  int* err;
};

constexpr int kRowThreads = 256;

// One wave per (token, head): 64 keys at a time, a lane's key against the whole
// query, then a running softmax and the values with a lane per column.
template <typename T, int HD>
__global__ __launch_bounds__(kRowThreads) void paged_rows_kernel(PagedAttnArgs a) {
  constexpr int EPV = Elem<T>::kVec, DPL = (HD + 63) / 64;
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * (kRowThreads / 64) + (threadIdx.x >> 6);
  if (row >= a.seq.n_tokens * a.Hq) return;
  const int t = row / a.Hq, h = row % a.Hq, hk = h / (a.Hq / a.Hkv);
  const int b = seq_of(a.seq, t);
  if (b >= a.seq.B) return;
  int first, count;
  seq_tokens(a.seq, b, &first, &count);
  const int len = a.seq.lens[b];
  bool bad = len > a.seq.cap;
  const int n = min(len - count + (t - first) + 1, a.seq.cap);  // keys this row sees
  const T* q = static_cast<const T*>(a.q) + t * a.q_st + h * a.q_sh;
  const int* trow = a.seq.table + b * a.seq.stride;
  float m = -INFINITY, l = 0.f, acc[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) acc[i] = 0.f;
  for (int k0 = 0; k0 < n; k0 += 64) {
    const int key = min(k0 + lane, n - 1);
    const int col = a.seq.page.div(key), slot = key - col * static_cast<int>(a.seq.page.d);
    const int page = page_of(key < a.prefix_len ? a.prefix : trow, col, a.seq.n_pages, &bad);
    const int64_t kr = page * a.kc.sp + hk * a.kc.sh + slot * a.kc.ss;
    const int64_t vr = page * a.vc.sp + hk * a.vc.sh + slot * a.vc.ss;
    const T* kp = static_cast<const T*>(a.kc.base) + kr;
    float s = 0.f;
    for (int c = 0; c < HD; c += EPV) {
      float kv[EPV], qv[EPV];
      load_vec(kp + c, kv);
      load_vec(q + c, qv);
#pragma unroll
      for (int e = 0; e < EPV; ++e) s = fmaf(kv[e], qv[e], s);
    }
    s = k0 + lane < n ? s * a.scale_log2 : -INFINITY;
    const float mn = fmaxf(m, wave_max(s));
    const float shift = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - shift), p = __builtin_amdgcn_exp2f(s - shift);
    m = mn;
    l = l * alpha + wave_sum(p);
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[i] *= alpha;
    const int live = min(64, n - k0);
    for (int j = 0; j < live; ++j) {
      const int64_t r = __shfl(vr, j, 64);
      const float pj = __shfl(p, j, 64);
      const T* vp = static_cast<const T*>(a.vc.base) + r;
#pragma unroll
      for (int i = 0; i < DPL; ++i)
        if (lane + 64 * i < HD) acc[i] = fmaf(pj, Elem<T>::load(vp + lane + 64 * i), acc[i]);
    }
  }
  if (bad && a.err != nullptr) *a.err = 1;
  T* o = static_cast<T*>(a.o) + t * a.o_st + h * a.o_sh;
#pragma unroll
  for (int i = 0; i < DPL; ++i)
    if (lane + 64 * i < HD) Elem<T>::store(o + lane + 64 * i, l > 0.f ? acc[i] / l : 0.f);
}

template <typename T, int HD>
static int launch_rows(const PagedAttnArgs& a, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.seq.n_tokens) * a.Hq;
  hipLaunchKernelGGL((paged_rows_kernel<T, HD>), dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(kRowThreads), 0, s, a);
  return hip_status(hipGetLastError());
}

template <typename T>
static int launch_paged(int hd, const PagedAttnArgs& a, hipStream_t s) {
  switch (hd) {
    case 16: return launch_rows<T, 16>(a, s);
    case 32: return launch_rows<T, 32>(a, s);
    case 64: return launch_rows<T, 64>(a, s);
    case 128: return launch_rows<T, 128>(a, s);
    default: return CGPT_ESHAPE;
  }
}

}  // namespace cgpt

extern "C" int cgpt_shared_prefix_attention(const void* q, const void* k_cache, const void* v_cache, void* o,
                                            const int* block_table, const int* seq_lens, const int* cu_q,
                                            const int* prefix_pages, int64_t prefix_len, int64_t n_tokens,
                                            int64_t B, int64_t Hq, int64_t Hkv, int64_t head_dim,
                                            int64_t page_size, int64_t n_pages, int64_t max_pages,
                                            int64_t bt_stride, int64_t q_st, int64_t q_sh, int64_t o_st,
                                            int64_t o_sh, int64_t kc_sp, int64_t kc_sh, int64_t kc_ss,
                                            int64_t vc_sp, int64_t vc_sh, int64_t vc_ss, float scale,
                                            void* workspace, int64_t workspace_bytes, int dtype,
                                            int* err_flag, void* stream) {
  using namespace cgpt;
  const PagePool kc{const_cast<void*>(k_cache), kc_sp, kc_sh, kc_ss}, vc{const_cast<void*>(v_cache), vc_sp, vc_sh, vc_ss};
  const int rc = check_paged(n_tokens, B, Hq, Hkv, head_dim, page_size, n_pages, max_pages, bt_stride, kc, vc, dtype);
  if (rc != CGPT_OK) return rc;
  if (prefix_len < 0 || prefix_len > page_size * max_pages) return CGPT_EINVAL;
  if (!(scale > 0.f)) return CGPT_EINVAL;
  if (n_tokens == 0 || B == 0) return CGPT_OK;
  if (q == nullptr || o == nullptr || seq_lens == nullptr || (max_pages > 0 && block_table == nullptr) ||
      (prefix_len > 0 && prefix_pages == nullptr))
    return CGPT_EINVAL;
  if (cu_q == nullptr && n_tokens != B) return CGPT_EINVAL;
  const int64_t epv = dtype == CGPT_F32 ? 4 : 8;
  for (int64_t st : {q_st, q_sh, o_st, o_sh})
    if (st < 0 || st % epv != 0) return CGPT_EINVAL;
  for (const void* p : {q, static_cast<const void*>(o)})
    if (reinterpret_cast<uintptr_t>(p) & 15) return CGPT_EINVAL;
  PagedAttnArgs a;
  a.q = q;
  a.o = o;
  a.kc = kc;
  a.vc = vc;
  a.seq = PagedBatch{block_table, seq_lens, cu_q, bt_stride, static_cast<int>(n_tokens), static_cast<int>(B),
                     static_cast<int>(n_pages), static_cast<int>(max_pages),
                     static_cast<int>(page_size * max_pages), FastDiv(page_size)};
  a.prefix = prefix_pages;
  a.prefix_len = static_cast<int>(prefix_len);
  a.prefix_cols = static_cast<int>((prefix_len + page_size - 1) / page_size);
  a.q_st = q_st;
  a.q_sh = q_sh;
  a.o_st = o_st;
  a.o_sh = o_sh;
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.err = err_flag;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int hd = static_cast<int>(head_dim);
  if (dtype == CGPT_BF16) return launch_paged<bf16_t>(hd, a, s);
  if (dtype == CGPT_F16) return launch_paged<f16_t>(hd, a, s);
  return launch_paged<float>(hd, a, s);
}

extern "C" int cgpt_paged_attention(const void* q, const void* k_cache, const void* v_cache, void* o,
                                    const int* block_table, const int* seq_lens, const int* cu_q,
                                    int64_t n_tokens, int64_t B, int64_t Hq, int64_t Hkv, int64_t head_dim,
                                    int64_t page_size, int64_t n_pages, int64_t max_pages, int64_t bt_stride,
                                    int64_t q_st, int64_t q_sh, int64_t o_st, int64_t o_sh, int64_t kc_sp,
                                    int64_t kc_sh, int64_t kc_ss, int64_t vc_sp, int64_t vc_sh, int64_t vc_ss,
                                    float scale, void* workspace, int64_t workspace_bytes, int dtype,
                                    int* err_flag, void* stream) {
  return cgpt_shared_prefix_attention(q, k_cache, v_cache, o, block_table, seq_lens, cu_q, nullptr, 0, n_tokens, B,
                                      Hq, Hkv, head_dim, page_size, n_pages, max_pages, bt_stride, q_st, q_sh, o_st,
                                      o_sh, kc_sp, kc_sh, kc_ss, vc_sp, vc_sh, vc_ss, scale, workspace,
                                      workspace_bytes, dtype, err_flag, stream);
}

extern "C" int cgpt_paged_attention_workspace(int64_t n_tokens, int64_t B, int64_t Hq, int64_t Hkv,
                                              int64_t head_dim, int64_t page_size, int64_t max_pages,
                                              int64_t prefix_len, int dtype, int64_t* workspace_bytes) {
  if (workspace_bytes == nullptr) return CGPT_EINVAL;
  *workspace_bytes = 0;
  return CGPT_OK;
}
