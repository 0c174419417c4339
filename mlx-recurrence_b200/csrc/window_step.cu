// One-token decode step of sliding-window attention on a cache of the last
// `window` keys and values plus the first `sinks` ones, and the kernel that
// leaves such a cache behind a prefill.
//
// Slot of token t: t (t < sinks), else sinks + (t - sinks) % window. The
// visible tokens at position p are then exactly the slots below
// min(p + 1, sinks + window), the newest one among them.
#include "common.cuh"

namespace mr {

struct StepArgs {
  const void *q, *k, *v;  // [B, Hq, Dh], [B, Hkv, Dh] dense
  void *ck, *cv;          // [B, slots, Hkv, Dh] dense
  const void* pos;        // [B] int32 or int64
  int pos64;
  int B, Hq, Hkv, Dh, slots, sinks;
  float scale;
  void* y;                // [B, Hq, Dh]
};

__device__ __forceinline__ int64_t step_pos(const StepArgs& A, int b) {
  return A.pos64 ? ((const int64_t*)A.pos)[b] : (int64_t)((const int*)A.pos)[b];
}
__device__ __forceinline__ int slot_of(int64_t p, int slots, int sinks) {
  return p < sinks ? (int)p : sinks + (int)((p - sinks) % (slots - sinks));
}

constexpr int kStepWarps2 = 8;

template <typename T, int NV>  // NV = Dh / 32
__global__ void __launch_bounds__(32 * kStepWarps2) window_step_kernel(const __grid_constant__ StepArgs A) {
  __shared__ float sm[kStepWarps2], sl[kStepWarps2], so[kStepWarps2][NV * 32];
  const int b = blockIdx.y, h = blockIdx.x, G = A.Hq / A.Hkv, hk = h / G;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  T* y = (T*)A.y + ((int64_t)b * A.Hq + h) * A.Dh;
  const int64_t p = step_pos(A, b);
  if (p < 0) {
    for (int d = threadIdx.x; d < A.Dh; d += blockDim.x) y[d] = from_f<T>(0.f);
    return;
  }
  const int n = (int)(p < A.slots - 1 ? p + 1 : A.slots), cur = slot_of(p, A.slots, A.sinks);
  const int64_t in = ((int64_t)b * A.Hkv + hk) * A.Dh, at = ((int64_t)b * A.slots * A.Hkv + hk) * A.Dh;
  const int64_t step = (int64_t)A.Hkv * A.Dh;
  float q[NV], o[NV], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    q[i] = to_f(((const T*)A.q)[((int64_t)b * A.Hq + h) * A.Dh + lane + 32 * i]) * (A.scale * 1.4426950408889634f);
    o[i] = 0.f;
  }
  for (int s = w; s < n; s += kStepWarps2) {
    const T* kp = s == cur ? (const T*)A.k + in : (const T*)A.ck + at + s * step;
    const T* vp = s == cur ? (const T*)A.v + in : (const T*)A.cv + at + s * step;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) dot = fmaf(q[i], to_f(kp[lane + 32 * i]), dot);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, x);
    const float mx = fmaxf(m, dot), base = mx == -INFINITY ? 0.f : mx, keep = exp2f(m - base), e = exp2f(dot - base);
    m = mx;
    l = l * keep + e;
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i] = o[i] * keep + e * to_f(vp[lane + 32 * i]);
  }
  if (lane == 0) sm[w] = m, sl[w] = l;
#pragma unroll
  for (int i = 0; i < NV; ++i) so[w][lane + 32 * i] = o[i];
  __syncthreads();
  if (h % G == 0)
    for (int d = threadIdx.x; d < A.Dh; d += blockDim.x) {
      ((T*)A.ck)[at + cur * step + d] = ((const T*)A.k)[in + d];
      ((T*)A.cv)[at + cur * step + d] = ((const T*)A.v)[in + d];
    }
  for (int d = threadIdx.x; d < A.Dh; d += blockDim.x) {
    float mx = -INFINITY, ls = 0.f, os = 0.f;
    for (int i = 0; i < kStepWarps2; ++i) mx = fmaxf(mx, sm[i]);
    if (mx == -INFINITY) mx = 0.f;
    for (int i = 0; i < kStepWarps2; ++i) {
      const float e = exp2f(sm[i] - mx);
      ls += sl[i] * e;
      os += so[i][d] * e;
    }
    y[d] = from_f<T>(os / ls);
  }
}

// cache[s][slot] <- the token that the slot holds after sequence s, or zeros
template <typename V>
__global__ void __launch_bounds__(256) window_cache_kernel(const V* __restrict__ k, const V* __restrict__ v,
                                                           int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs,
                                                           const int* __restrict__ cu, int S, int L, int T, int Hkv,
                                                           int DhV, int slots, int sinks, V* __restrict__ ck,
                                                           V* __restrict__ cv) {
  const int64_t per = (int64_t)Hkv * DhV, total = (int64_t)S * slots * per;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = e / per;
    const int s = (int)(row / slots), slot = (int)(row % slots), h = (int)(e % per) / DhV, d = (int)(e % DhV);
    const int lo = cu ? min(max(cu[s], 0), T) : s * L, hi = cu ? min(cu[s + 1], T) : min(lo + L, T);
    const int n = hi - lo, W = slots - sinks;
    int t = slot;  // a sink, or a ring slot that has been written once at most
    if (slot >= sinks && n > slots) t = slot + (n - 1 - slot) / W * W;
    V a = {}, b = {};
    if (t < n) {
      a = k[(lo + t) * k_ts + h * k_hs + d];
      b = v[(lo + t) * v_ts + h * v_hs + d];
    }
    ck[e] = a;
    cv[e] = b;
  }
}

template <typename T> int window_step_launch(const StepArgs& A, cudaStream_t st) {
  const dim3 g(A.Hq, A.B);
  switch (A.Dh) {
    case 32: window_step_kernel<T, 1><<<g, 32 * kStepWarps2, 0, st>>>(A); break;
    case 64: window_step_kernel<T, 2><<<g, 32 * kStepWarps2, 0, st>>>(A); break;
    case 96: window_step_kernel<T, 3><<<g, 32 * kStepWarps2, 0, st>>>(A); break;
    default: window_step_kernel<T, 4><<<g, 32 * kStepWarps2, 0, st>>>(A); break;
  }
  return check_launch("window_step_kernel");
}

}  // namespace mr

using namespace mr;

extern "C" {

int mr_window_step(const void* q, const void* k, const void* v, void* cache_k, void* cache_v, const void* pos,
                   int pos_is_int64, int dtype, int64_t batch, int64_t Hq, int64_t Hkv, int64_t Dh, int64_t slots,
                   int64_t sinks, float scale, void* y, void* stream) {
  const char* what = "mr_window_step";
  if (dtype != MR_F32 && dtype != MR_BF16 && dtype != MR_F16)
    return set_error(MR_E_DTYPE, "%s: unsupported dtype code %d (0=f32, 1=bf16, 2=f16)", what, dtype);
  if (batch < 0 || batch > 65535 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || Hq > 65535)
    return set_error(MR_E_SHAPE, "%s: batch=%lld must be 0..65535, Hq=%lld a multiple of Hkv=%lld", what,
                     (long long)batch, (long long)Hq, (long long)Hkv);
  if (Dh != 32 && Dh != 64 && Dh != 96 && Dh != 128)
    return set_error(MR_E_SHAPE, "%s: Dh=%lld must be 32, 64, 96 or 128", what, (long long)Dh);
  if (sinks < 0 || slots <= sinks || slots > (1 << 30))
    return set_error(MR_E_SHAPE, "%s: slots=%lld must exceed sinks=%lld >= 0", what, (long long)slots,
                     (long long)sinks);
  if (!(scale > 0.f) || scale > 3e38f) return set_error(MR_E_SHAPE, "%s: scale must be positive and finite", what);
  if (batch == 0) return MR_OK;
  for (const void* p : {q, k, v, (const void*)cache_k, (const void*)cache_v, (const void*)y})
    if (p == nullptr || ((uintptr_t)p & 15u))
      return set_error(MR_E_ALIGN, "%s: a pointer is NULL or not 16-byte aligned", what);
  if (pos == nullptr) return set_error(MR_E_ALIGN, "%s: pos is NULL", what);
  const StepArgs A{q, k, v, cache_k, cache_v, pos, pos_is_int64, (int)batch, (int)Hq, (int)Hkv, (int)Dh, (int)slots,
                   (int)sinks, scale, y};
  switch (dtype) {
    case MR_F32: return window_step_launch<float>(A, (cudaStream_t)stream);
    case MR_BF16: return window_step_launch<__nv_bfloat16>(A, (cudaStream_t)stream);
    default: return window_step_launch<__half>(A, (cudaStream_t)stream);
  }
}

int mr_window_cache(const void* k, const void* v, int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs,
                    const int32_t* cu_seqlens, int64_t S, int64_t L, int dtype, int64_t T, int64_t Hkv, int64_t Dh,
                    int64_t slots, int64_t sinks, void* cache_k, void* cache_v, void* stream) {
  const char* what = "mr_window_cache";
  if (dtype != MR_F32 && dtype != MR_BF16 && dtype != MR_F16)
    return set_error(MR_E_DTYPE, "%s: unsupported dtype code %d (0=f32, 1=bf16, 2=f16)", what, dtype);
  const int eb = dtype == MR_F32 ? 4 : 2;
  if (S < 0 || T < 0 || T > INT32_MAX / 2 || S > INT32_MAX / 2 || Hkv <= 0 || Dh <= 0 || Dh % 32 != 0 ||
      sinks < 0 || slots <= sinks || slots > (1 << 30))
    return set_error(MR_E_SHAPE, "%s: bad shape (Dh a multiple of 32, slots > sinks >= 0)", what);
  if (cu_seqlens == nullptr && (L <= 0 || S * L != T))
    return set_error(MR_E_SHAPE, "%s: without cu_seqlens T must be S * L", what);
  if (S == 0) return MR_OK;
  for (const void* p : {k, v, (const void*)cache_k, (const void*)cache_v})
    if ((p == nullptr && T > 0) || ((uintptr_t)p & 15u))
      return set_error(MR_E_ALIGN, "%s: a pointer is NULL or not 16-byte aligned", what);
  const int n = 16 / eb;
  for (int64_t s : {k_ts, k_hs, v_ts, v_hs})
    if (s % n != 0) return set_error(MR_E_ALIGN, "%s: strides must be multiples of 16 bytes", what);
  const int64_t total = S * slots * Hkv * (Dh / n);
  const unsigned grid = (unsigned)(total / 256 + 1 < 148 * 16 ? total / 256 + 1 : 148 * 16);
  window_cache_kernel<int4><<<grid, 256, 0, (cudaStream_t)stream>>>(
      (const int4*)k, (const int4*)v, k_ts / n, k_hs / n, v_ts / n, v_hs / n, cu_seqlens, (int)S, (int)L, (int)T,
      (int)Hkv, (int)(Dh / n), (int)slots, (int)sinks, (int4*)cache_k, (int4*)cache_v);
  return check_launch("window_cache_kernel");
}

}  // extern "C"
