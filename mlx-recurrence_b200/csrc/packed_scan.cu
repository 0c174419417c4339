// RG-LRU recurrence h_t = a_t h_{t-1} + x_t over a packed batch: sequences of
// any lengths (zero included) lie back to back in [T, D]; sequence s holds the
// tokens cu[s] .. cu[s+1]-1 and starts from h0[s] (zero without h0). Rows
// outside every sequence get zeros (outputs and gradients).
//
// Adjoint: adj_t = gy_t + [t last of s] gf_s + a_{t+1} adj_{t+1} (within the
// sequence), grad_x = adj, grad_a[t] = adj_t h_{t-1}, grad_h0[s] = a adj at
// its first token (gf_s for an empty sequence).
#include "common.cuh"

namespace mr {

constexpr int kPackedChunk = 128;  // steps between the states kept for the backward

// Walks cu with t: `s` is the sequence holding t, or the next one.
struct SeqWalk {
  const int* cu;
  int S;
  __device__ bool holds(int s, int64_t t) const { return s >= 0 && s < S && t >= cu[s] && t < cu[s + 1]; }
};

template <typename T>
__global__ void packed_fwd_walk(const T* __restrict__ a, const T* __restrict__ x, const int* __restrict__ cu, int S,
                                int64_t L, int64_t D, const float* __restrict__ h0, float* __restrict__ y,
                                float* __restrict__ ckpt, float* __restrict__ fin) {
  const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (d >= D) return;
  const SeqWalk w{cu, S};
  int s = 0;
  float h = 0.f;
  for (int64_t t = 0; t < L; ++t) {
    if (ckpt != nullptr && t % kPackedChunk == 0) ckpt[t / kPackedChunk * D + d] = h;
    while (s < S && cu[s + 1] <= t) {
      if (fin != nullptr && cu[s + 1] <= cu[s]) fin[s * D + d] = h0 ? h0[s * D + d] : 0.f;
      ++s;
    }
    if (!w.holds(s, t)) {
      y[t * D + d] = 0.f;
      continue;
    }
    if (t == cu[s]) h = h0 ? h0[s * D + d] : 0.f;
    h = fmaf(to_f(a[t * D + d]), h, to_f(x[t * D + d]));
    y[t * D + d] = h;
    if (fin != nullptr && t + 1 == cu[s + 1]) fin[s * D + d] = h;
  }
  for (; s < S; ++s)
    if (fin != nullptr && cu[s + 1] <= cu[s]) fin[s * D + d] = h0 ? h0[s * D + d] : 0.f;
}

template <typename T>
__global__ void packed_bwd_walk(const float* __restrict__ gy, const float* __restrict__ gf,
                                const float* __restrict__ ckpt, const T* __restrict__ a, const T* __restrict__ x,
                                const int* __restrict__ cu, int S, int64_t L, int64_t D,
                                const float* __restrict__ h0, T* __restrict__ ga, T* __restrict__ gx,
                                float* __restrict__ gh0) {
  const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (d >= D) return;
  const SeqWalk w{cu, S};
  for (int s = 0; gh0 != nullptr && s < S; ++s)
    if (cu[s + 1] <= cu[s]) gh0[s * D + d] = gf ? gf[s * D + d] : 0.f;
  int s = S - 1;
  float carry = 0.f;  // a_{t+1} adj_{t+1}
  float hp[kPackedChunk];
  for (int64_t c = (L + kPackedChunk - 1) / kPackedChunk - 1; c >= 0; --c) {
    const int64_t t0 = c * kPackedChunk, t1 = min(t0 + kPackedChunk, L);
    int sf = 0;
    float h = ckpt[c * D + d];
    for (int64_t t = t0; t < t1; ++t) {
      while (sf < S && cu[sf + 1] <= t) ++sf;
      if (!w.holds(sf, t)) continue;
      if (t == cu[sf]) h = h0 ? h0[sf * D + d] : 0.f;
      hp[t - t0] = h;
      h = fmaf(to_f(a[t * D + d]), h, to_f(x[t * D + d]));
    }
    for (int64_t t = t1 - 1; t >= t0; --t) {
      while (s >= 0 && (cu[s] > t || cu[s + 1] <= cu[s])) --s;
      if (!w.holds(s, t)) {
        ga[t * D + d] = from_f<T>(0.f);
        gx[t * D + d] = from_f<T>(0.f);
        continue;
      }
      if (t + 1 == cu[s + 1]) carry = gf ? gf[s * D + d] : 0.f;
      const float adj = gy[t * D + d] + carry;
      ga[t * D + d] = from_f<T>(adj * hp[t - t0]);
      gx[t * D + d] = from_f<T>(adj);
      carry = to_f(a[t * D + d]) * adj;
      if (gh0 != nullptr && t == cu[s]) gh0[s * D + d] = carry;
    }
  }
}

static int packed_check(const char* what, int dtype, int64_t T, int64_t D, int64_t S) {
  if (dtype != MR_F32 && dtype != MR_BF16 && dtype != MR_F16)
    return set_error(MR_E_DTYPE, "%s: unsupported dtype code %d (0=f32, 1=bf16, 2=f16)", what, dtype);
  if (T < 0 || D <= 0 || S < 0) return set_error(MR_E_SHAPE, "%s: T and S must not be negative, D positive", what);
  if (T > (int64_t)INT32_MAX / 2 || S > (int64_t)INT32_MAX / 2)
    return set_error(MR_E_SHAPE, "%s: T=%lld or S=%lld too large", what, (long long)T, (long long)S);
  return MR_OK;
}

template <typename T>
static int fwd_launch(const void* a, const void* x, const int* cu, int64_t S, int64_t L, int64_t D, const float* h0,
                      float* y, float* ckpt, float* fin, cudaStream_t st) {
  packed_fwd_walk<T><<<(unsigned)((D + 63) / 64), 64, 0, st>>>((const T*)a, (const T*)x, cu, (int)S, L, D, h0, y,
                                                               ckpt, fin);
  return check_launch("packed_fwd");
}
template <typename T>
static int bwd_launch(const float* gy, const float* gf, const float* ckpt, const void* a, const void* x,
                      const int* cu, int64_t S, int64_t L, int64_t D, const float* h0, void* ga, void* gx, float* gh0,
                      cudaStream_t st) {
  packed_bwd_walk<T><<<(unsigned)((D + 63) / 64), 64, 0, st>>>(gy, gf, ckpt, (const T*)a, (const T*)x, cu, (int)S, L,
                                                               D, h0, (T*)ga, (T*)gx, gh0);
  return check_launch("packed_bwd");
}

}  // namespace mr

using namespace mr;

extern "C" {

int64_t mr_rglru_packed_chunk(void) { return kPackedChunk; }

size_t mr_rglru_packed_workspace_bytes(int64_t T, int64_t D) {
  (void)T, (void)D;
  return 0;
}

int mr_rglru_packed_fwd(const void* a, const void* x, const int32_t* cu_seqlens, int64_t S, int dtype, int64_t T,
                        int64_t D, const float* h0, float* y, float* ckpt, float* final_state, void* ws,
                        size_t ws_bytes, void* stream) {
  if (int rc = packed_check("mr_rglru_packed_fwd", dtype, T, D, S)) return rc;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case MR_F32: return fwd_launch<float>(a, x, cu_seqlens, S, T, D, h0, y, ckpt, final_state, st);
    case MR_BF16: return fwd_launch<__nv_bfloat16>(a, x, cu_seqlens, S, T, D, h0, y, ckpt, final_state, st);
    default: return fwd_launch<__half>(a, x, cu_seqlens, S, T, D, h0, y, ckpt, final_state, st);
  }
}

int mr_rglru_packed_bwd(const float* grad_y, const float* grad_final, const float* ckpt, const void* a, const void* x,
                        const int32_t* cu_seqlens, int64_t S, int dtype, int64_t T, int64_t D, const float* h0,
                        void* grad_a, void* grad_x, float* grad_h0, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = packed_check("mr_rglru_packed_bwd", dtype, T, D, S)) return rc;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case MR_F32:
      return bwd_launch<float>(grad_y, grad_final, ckpt, a, x, cu_seqlens, S, T, D, h0, grad_a, grad_x, grad_h0, st);
    case MR_BF16:
      return bwd_launch<__nv_bfloat16>(grad_y, grad_final, ckpt, a, x, cu_seqlens, S, T, D, h0, grad_a, grad_x,
                                       grad_h0, st);
    default:
      return bwd_launch<__half>(grad_y, grad_final, ckpt, a, x, cu_seqlens, S, T, D, h0, grad_a, grad_x, grad_h0, st);
  }
}

}  // extern "C"
