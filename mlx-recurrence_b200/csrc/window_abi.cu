// Entry points of sliding-window attention (include/mlrec.h): validation and
// dispatch. Nothing here allocates or synchronises.
#include "window_attn.cuh"

namespace mr {

int attn_fwd_f32_launch(const AttnArgs&, cudaStream_t);
int attn_bwd_f32_launch(const AttnArgs&, void* ws, cudaStream_t);
size_t attn_bwd_f32_ws_bytes(int64_t T, int64_t Hq, int64_t Dh, int64_t sinks);
template <typename T> int attn_fwd_launch(const AttnArgs&, cudaStream_t);
template <typename T> int attn_bwd_launch(const AttnArgs&, void*, cudaStream_t);
size_t attn_bwd_ws_bytes(bool half, int64_t T, int64_t Hq, int64_t Hkv, int64_t Dh, int64_t sinks);

static int attn_check(const char* what, const AttnArgs& A, int64_t S, int64_t L, int dtype, int64_t T, int64_t Hq,
                      int64_t Hkv, int64_t Dh, int64_t window, int64_t sinks) {
  if (dtype != MR_F32 && dtype != MR_BF16 && dtype != MR_F16)
    return set_error(MR_E_DTYPE, "%s: unsupported dtype code %d (0=f32, 1=bf16, 2=f16)", what, dtype);
  if (T < 0 || T > INT32_MAX / 2 || S < 0 || S > INT32_MAX / 2)
    return set_error(MR_E_SHAPE, "%s: T=%lld or S=%lld out of range", what, (long long)T, (long long)S);
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || Hq > 65535)
    return set_error(MR_E_SHAPE, "%s: Hq=%lld must be a multiple of Hkv=%lld (at most 65535)", what, (long long)Hq,
                     (long long)Hkv);
  if (Dh != 32 && Dh != 64 && Dh != 96 && Dh != 128)
    return set_error(MR_E_SHAPE, "%s: Dh=%lld must be 32, 64, 96 or 128", what, (long long)Dh);
  if (window <= 0 || sinks < 0 || sinks > 64)
    return set_error(MR_E_SHAPE, "%s: window=%lld must be positive and sinks=%lld in 0..64", what, (long long)window,
                     (long long)sinks);
  if (!(A.scale > 0.f) || A.scale > 2e38f)
    return set_error(MR_E_SHAPE, "%s: scale must be positive and at most 2e38", what);
  if (A.cu == nullptr && T > 0 && (L <= 0 || L > T || S * L != T))
    return set_error(MR_E_SHAPE, "%s: without cu_seqlens T must be S * L", what);
  const int64_t n = dtype == MR_F32 ? 4 : 8;
  for (int64_t s : {A.q_ts, A.q_hs, A.k_ts, A.k_hs, A.v_ts, A.v_hs})
    if (s % n != 0 || s < 0) return set_error(MR_E_ALIGN, "%s: strides must be multiples of 16 bytes", what);
  return MR_OK;
}

static int ptrs(const char* what, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (p == nullptr || ((uintptr_t)p & 15u))
      return set_error(MR_E_ALIGN, "%s: a pointer is NULL or not 16-byte aligned", what);
  return MR_OK;
}

static AttnArgs attn_args(const void* q, const void* k, const void* v, int64_t q_ts, int64_t q_hs, int64_t k_ts,
                          int64_t k_hs, int64_t v_ts, int64_t v_hs, const int32_t* cu, int64_t S, int64_t L,
                          int64_t T, int64_t Hq, int64_t Hkv, int64_t Dh, int64_t window, int64_t sinks, float scale) {
  AttnArgs A{};
  A.q = q, A.k = k, A.v = v;
  A.q_ts = q_ts, A.q_hs = q_hs, A.k_ts = k_ts, A.k_hs = k_hs, A.v_ts = v_ts, A.v_hs = v_hs;
  A.cu = cu;
  A.S = (int)S, A.L = (int)L, A.T = (int)T, A.Hq = (int)Hq, A.Hkv = (int)Hkv, A.Dh = (int)Dh;
  A.window = (int)(window < T ? window : T), A.sinks = (int)sinks;
  A.scale = scale;
  return A;
}

}  // namespace mr

using namespace mr;

extern "C" {

int mr_window_attn_fwd(const void* q, const void* k, const void* v, int64_t q_ts, int64_t q_hs, int64_t k_ts,
                       int64_t k_hs, int64_t v_ts, int64_t v_hs, const int32_t* cu_seqlens, int64_t S, int64_t L,
                       int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t Dh, int64_t window, int64_t sinks,
                       float scale, void* y, void* y_low, float* lse, void* stream) {
  const char* what = "mr_window_attn_fwd";
  AttnArgs A = attn_args(q, k, v, q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, cu_seqlens, S, L, T, Hq, Hkv, Dh, window, sinks,
                         scale);
  if (int rc = attn_check(what, A, S, L, dtype, T, Hq, Hkv, Dh, window, sinks)) return rc;
  if (T == 0) return MR_OK;
  if (int rc = ptrs(what, {q, k, v, y})) return rc;
  if (dtype != MR_F32 && lse != nullptr)
    if (int rc = ptrs(what, {y_low})) return rc;
  A.y = y, A.y_low = dtype == MR_F32 ? nullptr : y_low, A.lse = lse;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case MR_F32: return attn_fwd_f32_launch(A, st);
    case MR_BF16: return attn_fwd_launch<__nv_bfloat16>(A, st);
    default: return attn_fwd_launch<__half>(A, st);
  }
}

size_t mr_window_attn_bwd_workspace_bytes(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t Dh, int64_t sinks) {
  if (T <= 0 || Hq <= 0 || Hkv <= 0 || Dh <= 0 || sinks < 0) return 0;
  return dtype == MR_F32 ? attn_bwd_f32_ws_bytes(T, Hq, Dh, sinks) : attn_bwd_ws_bytes(dtype == MR_F16, T, Hq, Hkv, Dh, sinks);
}

int mr_window_attn_bwd(const void* grad_y, const void* y, const void* y_low, const float* lse, const void* q,
                       const void* k, const void* v, int64_t q_ts, int64_t q_hs, int64_t k_ts, int64_t k_hs, int64_t v_ts,
                       int64_t v_hs, const int32_t* cu_seqlens, int64_t S, int64_t L, int dtype, int64_t T,
                       int64_t Hq, int64_t Hkv, int64_t Dh, int64_t window, int64_t sinks, float scale, void* grad_q,
                       void* grad_k, void* grad_v, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "mr_window_attn_bwd";
  AttnArgs A = attn_args(q, k, v, q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, cu_seqlens, S, L, T, Hq, Hkv, Dh, window, sinks,
                         scale);
  if (int rc = attn_check(what, A, S, L, dtype, T, Hq, Hkv, Dh, window, sinks)) return rc;
  if (T == 0) return MR_OK;
  if (int rc = ptrs(what, {grad_y, y, q, k, v, grad_q, grad_k, grad_v})) return rc;
  if (dtype != MR_F32)
    if (int rc = ptrs(what, {y_low})) return rc;
  const size_t need = mr_window_attn_bwd_workspace_bytes(dtype, T, Hq, Hkv, Dh, sinks);
  if (lse == nullptr || workspace == nullptr || workspace_bytes < need || ((uintptr_t)workspace & 15u))
    return set_error(MR_E_WORKSPACE, "%s: needs lse and %zu bytes of workspace, got %zu", what, need, workspace_bytes);
  A.y = const_cast<void*>(y), A.y_low = const_cast<void*>(y_low), A.lse = const_cast<float*>(lse), A.gy = grad_y;
  A.gq = grad_q, A.gk = grad_k, A.gv = grad_v;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case MR_F32: return attn_bwd_f32_launch(A, workspace, st);
    case MR_BF16: return attn_bwd_launch<__nv_bfloat16>(A, workspace, st);
    default: return attn_bwd_launch<__half>(A, workspace, st);
  }
}

}  // extern "C"
