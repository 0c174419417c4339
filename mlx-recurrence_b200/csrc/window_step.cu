// One-token decode step of sliding-window attention on a cache of the last
// `window` keys and values plus the first `sinks` ones, and the kernel that
// leaves such a cache behind a prefill.
//
// Slot of token t: t (t < sinks), else sinks + (t - sinks) % window. The
// visible tokens at position p are then exactly the slots below
// min(p + 1, sinks + window), the newest one among them.
#include <cooperative_groups.h>

#include "common.cuh"
#include "launch.cuh"

namespace mr {

namespace cg = cooperative_groups;

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

// ---- float32 -------------------------------------------------------------------
// One CTA per (batch row, query head): a warp takes kAhead slots at a time (their
// loads and dot products are independent), lanes over Dh, one online softmax per
// warp, joined in the warps' order. Key heads that several query heads share are
// read once each from L2.
constexpr int kF32Warps = 16, kAhead = 8;

template <int NV>  // NV = Dh / 32
__global__ void __launch_bounds__(32 * kF32Warps) window_step_f32(const __grid_constant__ StepArgs A) {
  __shared__ float sm[kF32Warps], sl[kF32Warps], so[kF32Warps][NV * 32];
  const int b = blockIdx.y, h = blockIdx.x, G = A.Hq / A.Hkv, hk = h / G;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  float* y = (float*)A.y + ((int64_t)b * A.Hq + h) * A.Dh;
  const int64_t p = step_pos(A, b);
  if (p < 0) {
    for (int d = threadIdx.x; d < A.Dh; d += blockDim.x) y[d] = 0.f;
    return;
  }
  const int n = (int)(p < A.slots - 1 ? p + 1 : A.slots), cur = slot_of(p, A.slots, A.sinks);
  const int64_t in = ((int64_t)b * A.Hkv + hk) * A.Dh, at = ((int64_t)b * A.slots * A.Hkv + hk) * A.Dh;
  const int64_t step = (int64_t)A.Hkv * A.Dh;
  float q[NV], o[NV], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    q[i] = ((const float*)A.q)[((int64_t)b * A.Hq + h) * A.Dh + lane + 32 * i] * (A.scale * 1.4426950408889634f);
    o[i] = 0.f;
  }
  for (int s = w * kAhead; s < n; s += kF32Warps * kAhead) {
    float dot[kAhead], v[kAhead][NV], mx = m;
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {  // (slots behind the last: that one again, with weight zero)
      const int slot = min(s + x, n - 1);
      const float* kp = slot == cur ? (const float*)A.k + in : (const float*)A.ck + at + slot * step;
      const float* vp = slot == cur ? (const float*)A.v + in : (const float*)A.cv + at + slot * step;
      dot[x] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        dot[x] = fmaf(q[i], kp[lane + 32 * i], dot[x]);
        v[x][i] = vp[lane + 32 * i];
      }
    }
#pragma unroll
    for (int e = 16; e > 0; e >>= 1)
#pragma unroll
      for (int x = 0; x < kAhead; ++x) dot[x] += __shfl_xor_sync(0xffffffffu, dot[x], e);
#pragma unroll
    for (int x = 0; x < kAhead; ++x) mx = fmaxf(mx, dot[x]);
    const float base = mx == -INFINITY ? 0.f : mx, keep = exp2f(m - base);
    m = mx;
    l *= keep;
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i] *= keep;
#pragma unroll
    for (int x = 0; x < kAhead; ++x)
      if (s + x < n) {
        const float e = exp2f(dot[x] - base);
        l += e;
#pragma unroll
        for (int i = 0; i < NV; ++i) o[i] = fmaf(e, v[x][i], o[i]);
      }
  }
  if (lane == 0) sm[w] = m, sl[w] = l;
#pragma unroll
  for (int i = 0; i < NV; ++i) so[w][lane + 32 * i] = o[i];
  __syncthreads();
  if (h % G == 0)  // after every warp has read the caches (no CTA reads the slot itself)
    for (int d = threadIdx.x; d < A.Dh; d += blockDim.x) {
      ((float*)A.ck)[at + cur * step + d] = ((const float*)A.k)[in + d];
      ((float*)A.cv)[at + cur * step + d] = ((const float*)A.v)[in + d];
    }
  for (int d = threadIdx.x; d < A.Dh; d += blockDim.x) {
    float mx = -INFINITY, ls = 0.f, os = 0.f;
    for (int i = 0; i < kF32Warps; ++i) mx = fmaxf(mx, sm[i]);
    if (mx == -INFINITY) mx = 0.f;
    for (int i = 0; i < kF32Warps; ++i) {
      const float e = exp2f(sm[i] - mx);
      ls += sl[i] * e;
      os += so[i][d] * e;
    }
    y[d] = os / ls;
  }
}

// ---- bf16 and fp16 ------------------------------------------------------------
// HBM-bound: each visible slot of both caches is read once, for all query heads
// of the group (up to 16 at a time as the rows of m16n8k16 products, so the
// arithmetic stays far below the loads whatever the group). A cluster of up to 8
// CTAs splits a (batch row, key head)'s slots in tiles of 64, brought into shared
// memory by asynchronous copies kRing tiles ahead; a warp takes 16 slots of a tile
// with its own online softmax. Warps, then CTAs (over distributed shared memory)
// join their maxima, sums and outputs in a fixed order; one launch, no workspace.
// P goes into its product in two parts, rounded to the inputs' type and what that
// drops, so its rounding is squared (y's error was 1.2 times that of rounding y alone):
// as rows of their own where the group leaves half of the sixteen, or in a second product.
// B=96, 16 heads of 128 on 4, 2052 slots: 66 us, 6.1 TB/s of the caches' bytes (67 by
// second products, 66 without the second part); B=33, 10 heads of 64 on 1, 1024 slots: 7.5
// us (7.1 without); B=1, 8 heads of 64 on 2, 516 slots: 6.3 us, a launch and a few
// dependent loads.

constexpr int kTile = 64, kRing = 2;

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  static __device__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ uint32_t pack(float a, float b) {
    __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static __device__ float2 unpack(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
};
template <> struct Mma<__half> {
  static __device__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ uint32_t pack(float a, float b) {
    __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static __device__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
};

template <bool TRANS> __device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes, or zeros where `bytes` is 0
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// 16-byte chunk c of slot row r of a tile: rotated so that the 8 rows of a matrix lie in different banks
template <int DH> __device__ __forceinline__ int chunk_at(int r, int c) {
  return r * (DH / 8) + (DH % 64 == 0 ? c ^ (r & 7) : c ^ (r >> 1 & 3));
}

template <typename T, int DH> constexpr int kStepSmem = kRing * 2 * kTile * DH * 2;

template <typename T, int DH>
__global__ void __launch_bounds__(128) window_step_mma(const __grid_constant__ StepArgs A, int splits, int head_tiles) {
  constexpr int NC = DH / 8, KS = DH / 16, kTileB = kTile * DH * 2;
  extern __shared__ __align__(128) unsigned char sm[];
  __shared__ float wm[4][16], wl[4][16], cm[16], cl[16];
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % splits, unit = blockIdx.x / splits;
  const int b = blockIdx.y, hk = unit / head_tiles, h0 = unit % head_tiles * 16, G = A.Hq / A.Hkv;
  const int rows = min(16, G - h0);
  const bool paired = rows <= 8;  // P's second part takes the place of rows 8 .. 15
  const int64_t qat = ((int64_t)b * A.Hq + hk * G + h0) * DH;
  T* y = (T*)A.y + qat;
  const int64_t p = step_pos(A, b);
  if (p < 0) {  // the whole cluster
    if (rank == 0)
      for (int e = tid; e < rows * DH; e += 128) y[e] = from_f<T>(0.f);
    return;
  }
  const int n = (int)(p < A.slots - 1 ? p + 1 : A.slots), cur = slot_of(p, A.slots, A.sinks);
  const int tiles = (n + kTile - 1) / kTile, t0 = tiles * rank / splits, t1 = tiles * (rank + 1) / splits;
  const int64_t in = ((int64_t)b * A.Hkv + hk) * DH, at = ((int64_t)b * A.slots * A.Hkv + hk) * DH;
  const int64_t step = (int64_t)A.Hkv * DH;
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(sm));

  auto load = [&](int t) {
    if (t < t1) {
      const uint32_t dst = base + (t % kRing) * 2 * kTileB;
      for (int e = tid; e < kTile * NC; e += 128) {
        const int r = e / NC, c = e % NC, slot = t * kTile + r;
        const bool now = slot == cur;  // the new token comes from the call, not from the cache
        const int bytes = slot < n ? 16 : 0;
        const int64_t off = now ? in + c * 8 : at + min(slot, n - 1) * step + c * 8;
        copy16(dst + chunk_at<DH>(r, c) * 16, (now ? (const T*)A.k : (const T*)A.ck) + off, bytes);
        copy16(dst + kTileB + chunk_at<DH>(r, c) * 16, (now ? (const T*)A.v : (const T*)A.cv) + off, bytes);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int i = 0; i < kRing - 1; ++i) load(t0 + i);
  if (cur / kTile >= t0 && cur / kTile < t1 && h0 == 0 && tid < 2 * NC) {
    const int c = tid % NC;
    const T* src = (tid < NC ? (const T*)A.k : (const T*)A.v) + in + c * 8;
    T* dst = (tid < NC ? (T*)A.ck : (T*)A.cv) + at + cur * step + c * 8;
    *reinterpret_cast<int4*>(dst) = *reinterpret_cast<const int4*>(src);
  }
  // Q as the A operand: rows lane / 4 and + 8
  uint32_t q[KS][4];
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (lane >> 2) + (i & 1) * 8, d = k * 16 + (lane & 3) * 2 + (i >> 1) * 8;
      q[k][i] = r < rows ? *reinterpret_cast<const uint32_t*>((const T*)A.q + qat + r * DH + d) : 0u;
    }
  const float c = A.scale * 1.4426950408889634f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[NC][4];
#pragma unroll
  for (int i = 0; i < NC; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  for (int t = t0; t < t1; ++t) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
    __syncthreads();
    load(t + kRing - 1);
    const uint32_t sk = base + (t % kRing) * 2 * kTileB, sv = sk + kTileB;
    const int s0 = w * 16;  // this warp's slots of the tile
    if (t * kTile + s0 >= n) continue;
    float s[2][4] = {};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      uint32_t f[4];
      ldmatrix4<false>(f, sk + chunk_at<DH>(s0 + (lane >> 4) * 8 + (lane & 7), k * 2 + (lane >> 3 & 1)) * 16);
      Mma<T>::run(s[0], q[k], f[0], f[1]);
      Mma<T>::run(s[1], q[k], f[2], f[3]);
    }
    uint32_t pa[4], pb[4];  // P in the inputs' type, and what that rounding drops
    float keep[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {  // rows lane / 4 and + 8
      if (r == 1 && paired) {
        pa[1] = pb[0], pa[3] = pb[2], keep[1] = keep[0];
        break;
      }
      float mx = m[r];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int slot = t * kTile + s0 + (i >> 1) * 8 + (lane & 3) * 2 + (i & 1);
        float& v = s[i >> 1][r * 2 + (i & 1)];
        v = slot < n ? v * c : -INFINITY;
        mx = fmaxf(mx, v);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float to = mx == -INFINITY ? 0.f : mx;
      keep[r] = exp2f(m[r] - to);
      m[r] = mx;
      l[r] *= keep[r];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float& v = s[i >> 1][r * 2 + (i & 1)];
        v = exp2f(v - to);
        l[r] += v;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float p0 = s[i][r * 2], p1 = s[i][r * 2 + 1];
        pa[r + 2 * i] = Mma<T>::pack(p0, p1);
        const float2 back = Mma<T>::unpack(pa[r + 2 * i]);
        pb[r + 2 * i] = Mma<T>::pack(p0 - back.x, p1 - back.y);
      }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i][0] *= keep[0], o[i][1] *= keep[0], o[i][2] *= keep[1], o[i][3] *= keep[1];
#pragma unroll
    for (int i = 0; i < NC; i += 4) {
      uint32_t f[2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x)
        ldmatrix4<true>(f[x], sv + chunk_at<DH>(s0 + (lane >> 3 & 1) * 8 + (lane & 7), i + 2 * x + (lane >> 4)) * 16);
#pragma unroll
      for (int x = 0; x < 4; ++x) Mma<T>::run(o[i + x], pa, f[x >> 1][(x & 1) * 2], f[x >> 1][(x & 1) * 2 + 1]);
      if (!paired)
#pragma unroll
        for (int x = 0; x < 4; ++x) Mma<T>::run(o[i + x], pb, f[x >> 1][(x & 1) * 2], f[x >> 1][(x & 1) * 2 + 1]);
    }
  }
  if (paired)
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i][0] += o[i][2], o[i][1] += o[i][3];
  // join the warps: the ring's memory is free
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if ((lane & 3) == 0) wm[w][(lane >> 2) + r * 8] = m[r], wl[w][(lane >> 2) + r * 8] = l[r];
  }
  __syncthreads();
  float* so = reinterpret_cast<float*>(sm);  // [warp][16][DH], then the sum in warp 0's place
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      *reinterpret_cast<float2*>(so + (w * 16 + (lane >> 2) + r * 8) * DH + i * 8 + (lane & 3) * 2) =
          make_float2(o[i][r * 2], o[i][r * 2 + 1]);
  __syncthreads();
  for (int e = tid; e < rows * DH; e += 128) {
    const int r = e / DH;
    float mx = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
    const float to = mx == -INFINITY ? 0.f : mx;
    float os = 0.f, ls = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = exp2f(wm[i][r] - to);
      os = fmaf(so[i * 16 * DH + e], f, os);
      ls = fmaf(wl[i][r], f, ls);
    }
    if (splits == 1) {
      y[e] = from_f<T>(os / ls);
    } else {
      so[e] = os;  // this element's own slot of warp 0
      if (e % DH == 0) cm[r] = mx, cl[r] = ls;
    }
  }
  if (splits == 1) return;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int all = rows * DH;
  for (int e = all * rank / splits + tid; e < all * (rank + 1) / splits; e += 128) {
    const int r = e / DH;
    float mx = -INFINITY;
    for (int i = 0; i < splits; ++i) mx = fmaxf(mx, *cluster.map_shared_rank(&cm[r], i));
    const float to = mx == -INFINITY ? 0.f : mx;
    float os = 0.f, ls = 0.f;
    for (int i = 0; i < splits; ++i) {
      const float f = exp2f(*cluster.map_shared_rank(&cm[r], i) - to);
      os = fmaf(*cluster.map_shared_rank(&so[e], i), f, os);
      ls = fmaf(*cluster.map_shared_rank(&cl[r], i), f, ls);
    }
    y[e] = from_f<T>(os / ls);
  }
  cluster.sync();  // nobody leaves while its memory is read
}

template <typename T, int DH> static int step_mma_dh(const StepArgs& A, cudaStream_t st) {
  const int G = A.Hq / A.Hkv, head_tiles = (G + 15) / 16, tiles = (A.slots + kTile - 1) / kTile;
  const int64_t units = (int64_t)A.B * A.Hkv * head_tiles;
  // CTAs for two on every SM (three fit: one wave), each with two tiles at least. At B=96, Hkv=4, Dh=128, 2052 slots:
  // 66 us unsplit, 76 in two, 85 in four (later waves leave SMs idle); at B=8: 12.5 us in eight
  int splits = 1;
  while (splits < 8 && units * splits < 148 * 2 && splits * 4 <= tiles) splits *= 2;
  auto kernel = window_step_mma<T, DH>;
  constexpr int smem = kStepSmem<T, DH>;
  if (int rc = allow_smem<window_step_mma<T, DH>>(smem, "window_step_mma")) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(A.Hkv * head_tiles * splits), (unsigned)A.B);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, A, splits, head_tiles);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(MR_E_LAUNCH, "window_step_mma: %s", cudaGetErrorString(e));
  }
  return check_launch("window_step_mma");
}
template <typename T> static int step_mma(const StepArgs& A, cudaStream_t st) {
  switch (A.Dh) {
    case 32: return step_mma_dh<T, 32>(A, st);
    case 64: return step_mma_dh<T, 64>(A, st);
    case 96: return step_mma_dh<T, 96>(A, st);
    default: return step_mma_dh<T, 128>(A, st);
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

static int step_f32(const StepArgs& A, cudaStream_t st) {
  const dim3 g(A.Hq, A.B);
  switch (A.Dh) {
    case 32: window_step_f32<1><<<g, 32 * kF32Warps, 0, st>>>(A); break;
    case 64: window_step_f32<2><<<g, 32 * kF32Warps, 0, st>>>(A); break;
    case 96: window_step_f32<3><<<g, 32 * kF32Warps, 0, st>>>(A); break;
    default: window_step_f32<4><<<g, 32 * kF32Warps, 0, st>>>(A); break;
  }
  return check_launch("window_step_f32");
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
  if (!(scale > 0.f) || scale > 2e38f) return set_error(MR_E_SHAPE, "%s: scale must be positive and at most 2e38", what);
  if (batch == 0) return MR_OK;
  for (const void* p : {q, k, v, (const void*)cache_k, (const void*)cache_v, (const void*)y})
    if (p == nullptr || ((uintptr_t)p & 15u))
      return set_error(MR_E_ALIGN, "%s: a pointer is NULL or not 16-byte aligned", what);
  if (pos == nullptr) return set_error(MR_E_ALIGN, "%s: pos is NULL", what);
  const StepArgs A{q, k, v, cache_k, cache_v, pos, pos_is_int64, (int)batch, (int)Hq, (int)Hkv, (int)Dh, (int)slots,
                   (int)sinks, scale, y};
  switch (dtype) {
    case MR_F32: return step_f32(A, (cudaStream_t)stream);
    case MR_BF16: return step_mma<__nv_bfloat16>(A, (cudaStream_t)stream);
    default: return step_mma<__half>(A, (cudaStream_t)stream);
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
  if (cu_seqlens == nullptr && (L < 0 || S * L != T))
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
