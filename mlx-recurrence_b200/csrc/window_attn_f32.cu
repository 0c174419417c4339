// Sliding-window attention with sinks on the CUDA cores, in float32: forward,
// and the backward as one pass over key tiles per query tile (grad_q) and one
// pass over query tiles per key tile (grad_k, grad_v; a shared key/value head
// sums its query heads in a fixed order, so results do not vary).
//
//   s_ij = scale q_i.k_j,  p = softmax over the visible j,  y_i = sum_j p_ij v_j
//   ds_ij = p_ij (gy_i.v_j - delta_i),  delta_i = gy_i.y_i
//   grad_q_i = scale sum_j ds_ij k_j,  grad_k_j = scale sum_i ds_ij q_i,  grad_v_j = sum_i p_ij gy_i
//
// Tiles are 64 x 64; 256 threads own 4 x 4 results of a tile and 4 rows x Dh/16
// columns of the products that follow. Operands lie transposed ([d][64 + 4]) in
// shared memory, so a thread's rows and columns come as 16-byte reads. Bound by
// the latency between a tile's barriers (few warps per SM): T=3001, 8 heads of 32,
// window 300: forward 75 us, backward 269 us; T=4000, 8 heads of 128 on 4, window
// 1000: 547 us (19 TFLOP/s) and 1.92 ms. (128 threads with 8 x 4 results: 831 us, 3.14
// ms.)
#include "window_attn.cuh"

namespace mr {

constexpr int kBT = 64;        // tile edge
constexpr int kPitch = kBT + 4;
constexpr int kThreads = 256;
constexpr int kR = 4;  // rows of a thread

// rows r0 .. r0+63 of one head, on their way to [d][kPitch] in shared memory; zeros outside [lo, hi). In two steps, so
// that the next tile's loads run under this tile's arithmetic. Lanes take consecutive rows: conflict-free stores.
template <int DH> struct Tile {
  static constexpr int N = kBT * DH / 4 / kThreads;
  float4 v[N];
  __device__ __forceinline__ void fetch(const float* src, int64_t ts, int r0, int lo, int hi) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = threadIdx.x + i * kThreads, t = r0 + (e & 63);
      v[i] = t >= lo && t < hi ? *reinterpret_cast<const float4*>(src + t * ts + (e >> 6) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  __device__ __forceinline__ void stash(float* dst) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = threadIdx.x + i * kThreads;
      float* p = dst + (e >> 6) * 4 * kPitch + (e & 63);
      p[0] = v[i].x, p[kPitch] = v[i].y, p[2 * kPitch] = v[i].z, p[3 * kPitch] = v[i].w;
    }
  }
};

// acc = sum_d R[d][kR rows of ty] C[d][4 columns of tx], two rows to an instruction
template <int DH>
__device__ __forceinline__ void tile_dot(float (&acc)[kR][4], const float* R, const float* C, int ty, int tx) {
  uint64_t a[kR / 2][4];
#pragma unroll
  for (int i = 0; i < kR / 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) a[i][j] = 0;
#pragma unroll 4
  for (int d = 0; d < DH; ++d) {
    const ulonglong2 rr = *reinterpret_cast<const ulonglong2*>(R + d * kPitch + ty * kR);
    const float4 c = *reinterpret_cast<const float4*>(C + d * kPitch + tx * 4);
    const uint64_t cc[4] = {pair(c.x, c.x), pair(c.y, c.y), pair(c.z, c.z), pair(c.w, c.w)};
    const uint64_t r[kR / 2] = {rr.x, rr.y};
#pragma unroll
    for (int i = 0; i < kR / 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) a[i][j] = fma2(r[i], cc[j], a[i][j]);
  }
#pragma unroll
  for (int i = 0; i < kR / 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) unpair(a[i][j], acc[2 * i][j], acc[2 * i + 1][j]);
}

// out[row pairs][DH/16] += sum_n P[n][kR rows of ty] C[tx + 16 m][n], four n at a time: their columns come as one
// 16-byte read
template <int DH>
__device__ __forceinline__ void tile_acc(uint64_t (&out)[kR / 2][DH / 16], const float* P, const float* C, int ty, int tx) {
#pragma unroll 1
  for (int n = 0; n < kBT; n += 4) {
    float c[DH / 16][4];
#pragma unroll
    for (int m = 0; m < DH / 16; ++m)
      *reinterpret_cast<float4*>(c[m]) = *reinterpret_cast<const float4*>(C + (tx + 16 * m) * kPitch + n);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const ulonglong2 r = *reinterpret_cast<const ulonglong2*>(P + (n + x) * kPitch + ty * kR);
#pragma unroll
      for (int m = 0; m < DH / 16; ++m) {
        const uint64_t cc = pair(c[m][x], c[m][x]);
        out[0][m] = fma2(r.x, cc, out[0][m]);
        out[1][m] = fma2(r.y, cc, out[1][m]);
      }
    }
  }
}
template <int N> __device__ __forceinline__ void rows_of(float (&v)[kR][N], const uint64_t (&a)[kR / 2][N]) {
#pragma unroll
  for (int i = 0; i < kR / 2; ++i)
#pragma unroll
    for (int n = 0; n < N; ++n) unpair(a[i][n], v[2 * i][n], v[2 * i + 1][n]);
}

// P[column][row] <- a thread's kR x 4 block
__device__ __forceinline__ void put_block(float* P, const float (&v)[kR][4], int ty, int tx) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float* p = P + (tx * 4 + j) * kPitch + ty * kR;
    *reinterpret_cast<float4*>(p) = make_float4(v[0][j], v[1][j], v[2][j], v[3][j]);
  }
}

template <int DH>
__global__ void __launch_bounds__(kThreads, DH <= 64 ? 2 : 1) attn_fwd_f32(const __grid_constant__ AttnArgs A) {
  extern __shared__ float sm[];
  float *sQ = sm, *sK = sQ + DH * kPitch, *sV = sK + DH * kPitch, *sP = sV + DH * kPitch;
  __shared__ RowMask rows[kBT];
  __shared__ int again[kBT];
  const int q0 = blockIdx.x * kBT, h = blockIdx.y, hk = h / (A.Hq / A.Hkv);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const float* q = (const float*)A.q + h * A.q_hs;
  const float* k = (const float*)A.k + hk * A.k_hs;
  const float* v = (const float*)A.v + hk * A.v_hs;
  const KeyRange R = keys_of(A, q0, q0 + kBT);
  const int first = first_token(A), last = end_token(A);
  if (threadIdx.x < kBT) rows[threadIdx.x] = row_mask(A, q0 + threadIdx.x), again[threadIdx.x] = 0;
  Tile<DH> tq;
  tq.fetch(q, A.q_ts, q0, first, last);
  tq.stash(sQ);
  const float c = A.scale * kAttnLog2e;
  float m[kR], l[kR], keep[kR], o[kR][DH / 16];
  uint64_t o2[kR / 2][DH / 16];
#pragma unroll
  for (int i = 0; i < kR; ++i) {
    m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int n = 0; n < DH / 16; ++n) o2[i / 2][n] = 0;
  }
  const int nsink = R.send > R.s0 ? (R.send - R.s0 + kBT - 1) / kBT : 0;
  const int nband = R.kend > R.kmin ? (R.kend - R.kmin + kBT - 1) / kBT : 0;
  auto beg = [&](int it) { return it < nsink ? R.s0 + it * kBT : R.kmin + (it - nsink) * kBT; };
  auto lim = [&](int it) { return min(beg(it) + kBT, it < nsink ? R.send : R.kend); };
  Tile<DH> tk, tv;
  auto fetch = [&](int it) {
    tk.fetch(k, A.k_ts, beg(it), first, lim(it));
    tv.fetch(v, A.v_ts, beg(it), first, lim(it));
  };
  if (nsink + nband > 0) fetch(0);
  for (int it = 0; it < nsink + nband; ++it) {
    const int k0 = beg(it), k1 = lim(it);
    __syncthreads();
    tk.stash(sK);
    tv.stash(sV);
    __syncthreads();
    if (it + 1 < nsink + nband) fetch(it + 1);
    float s[kR][4];
    tile_dot<DH>(s, sQ, sK, ty, tx);
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const RowMask w = rows[ty * kR + i];
      float mx = m[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + tx * 4 + j;
        s[i][j] = key < k1 && w.sees(key) ? s[i][j] * c : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x, 16));
      const float base = mx == -INFINITY ? 0.f : mx;  // nothing visible so far: every term is exp2(-inf)
      keep[i] = exp2f(m[i] - base);
      m[i] = mx;
      l[i] *= keep[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2f(s[i][j] - base);
        l[i] += s[i][j];
      }
    }
#pragma unroll
    for (int i = 0; i < kR / 2; ++i)
#pragma unroll
      for (int n = 0; n < DH / 16; ++n) o2[i][n] = mul2(o2[i][n], pair(keep[2 * i], keep[2 * i + 1]));
    put_block(sP, s, ty, tx);
    __syncthreads();
    tile_acc<DH>(o2, sP, sV, ty, tx);
  }
  rows_of(o, o2);
#pragma unroll
  for (int i = 0; i < kR; ++i) {
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x, 16);
    const int t = q0 + ty * kR + i;
    if (t >= A.T) continue;
    const bool live = rows[ty * kR + i].i >= 0;  // a row of no sequence is zero whatever its tiles hold
    const float inv = l[i] > 0.f ? 1.f / l[i] : (l[i] == 0.f ? 0.f : l[i]);
    float* y = (float*)A.y + ((int64_t)t * A.Hq + h) * A.Dh;
    float odd = 0.f;  // NaN as soon as one element is not finite
#pragma unroll
    for (int n = 0; n < DH / 16; ++n) {
      y[tx + 16 * n] = live ? o[i][n] * inv : 0.f;
      odd = fmaf(o[i][n], 0.f, odd);
    }
    if (A.lse != nullptr && tx == 0) A.lse[(int64_t)h * A.T + t] = l[i] == 0.f ? INFINITY : m[i] + log2f(l[i]);
    if (live && (odd != 0.f || l[i] == 0.f)) again[ty * kR + i] = 1;  // (l = 0: scores of -infinity alone)
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < kBT; r += kThreads / 32)
    if (again[r]) exact_fwd_row<float>(A, h, q0 + r);
}

// delta[h][t] = sum_d gy y: one warp per row
__global__ void __launch_bounds__(256) attn_delta_f32(const __grid_constant__ AttnArgs A) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= (int64_t)A.T * A.Hq) return;
  const float* g = (const float*)A.gy + row * A.Dh;
  const float* y = (const float*)A.y + row * A.Dh;
  float s = 0.f;
  for (int d = lane; d < A.Dh; d += 32) s = fmaf((g[d]), (y[d]), s);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
  if (lane == 0) A.delta[(row % A.Hq) * A.T + row / A.Hq] = s;
}

// KV = false: rows are queries, columns keys, out1 = grad_q.
// KV = true: rows are keys, columns queries, out1 = grad_k, out2 = grad_v.
template <int DH, bool KV>
__global__ void __launch_bounds__(kThreads, DH <= 64 ? 2 : 1) attn_bwd_f32(const __grid_constant__ AttnArgs A) {
  extern __shared__ float sm[];
  float *sR1 = sm, *sR2 = sR1 + DH * kPitch, *sC1 = sR2 + DH * kPitch, *sC2 = sC1 + DH * kPitch, *sP = sC2 + DH * kPitch;
  __shared__ RowMask rows[kBT];
  __shared__ int limit[kBT], again[kBT];
  __shared__ float lse[kBT], delta[kBT];
  const int r0 = blockIdx.x * kBT, G = A.Hq / A.Hkv;
  const int hk = KV ? blockIdx.y : blockIdx.y / G;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int first = first_token(A), last = end_token(A);
  const float* k = (const float*)A.k + hk * A.k_hs;
  const float* v = (const float*)A.v + hk * A.v_hs;
  const int64_t gts = (int64_t)A.Hq * A.Dh;
  const float c = A.scale * kAttnLog2e;
  uint64_t a1[kR / 2][DH / 16], a2[kR / 2][DH / 16];  // (a2: KV only)
#pragma unroll
  for (int i = 0; i < kR / 2; ++i)
#pragma unroll
    for (int n = 0; n < DH / 16; ++n) a1[i][n] = a2[i][n] = 0;

  const KeyRange R = keys_of(A, r0, r0 + kBT);
  const QueryRange Q = near_queries<6>(A, r0, r0 + kBT);
  const int nsink = !KV && R.send > R.s0 ? (R.send - R.s0 + kBT - 1) / kBT : 0;
  const int nband = KV ? (Q.qend > Q.qbeg ? (Q.qend - Q.qbeg + kBT - 1) / kBT : 0)
                       : (R.kend > R.kmin ? (R.kend - R.kmin + kBT - 1) / kBT : 0);
  if (threadIdx.x < kBT) {
    const int t = r0 + threadIdx.x;
    again[threadIdx.x] = 0;
    if (KV) {
      limit[threadIdx.x] = near_limit<6>(A, t);
    } else {
      rows[threadIdx.x] = row_mask(A, t);
      lse[threadIdx.x] = t < A.T ? A.lse[(int64_t)blockIdx.y * A.T + t] : INFINITY;
      delta[threadIdx.x] = t < A.T ? A.delta[(int64_t)blockIdx.y * A.T + t] : 0.f;
    }
  }
  Tile<DH> t1, t2;
  if (KV) {
    t1.fetch(k, A.k_ts, r0, first, last);
    t2.fetch(v, A.v_ts, r0, first, last);
  } else {
    t1.fetch((const float*)A.q + blockIdx.y * A.q_hs, A.q_ts, r0, first, last);
    t2.fetch((const float*)A.gy + (int64_t)blockIdx.y * A.Dh, gts, r0, first, last);
  }
  t1.stash(sR1);
  t2.stash(sR2);
  const int n_it = (KV ? G : 1) * (nsink + nband);
  auto head = [&](int it) { return KV ? hk * G + it / nband : (int)blockIdx.y; };
  auto beg = [&](int it) {
    const int n = KV ? it % nband : it;
    return KV ? Q.qbeg + n * kBT : n < nsink ? R.s0 + n * kBT : R.kmin + (n - nsink) * kBT;
  };
  auto lim = [&](int it) { return min(beg(it) + kBT, KV ? Q.qend : it < nsink ? R.send : R.kend); };
  float lse_n = INFINITY, delta_n = 0.f;
  auto fetch = [&](int it) {
    const int h = head(it), c0 = beg(it), c1 = lim(it);
    if (KV) {
      t1.fetch((const float*)A.q + h * A.q_hs, A.q_ts, c0, first, c1);
      t2.fetch((const float*)A.gy + (int64_t)h * A.Dh, gts, c0, first, c1);
      const int t = c0 + (threadIdx.x & 63);
      lse_n = t < c1 ? A.lse[(int64_t)h * A.T + t] : INFINITY;
      delta_n = t < c1 ? A.delta[(int64_t)h * A.T + t] : 0.f;
    } else {
      t1.fetch(k, A.k_ts, c0, first, c1);
      t2.fetch(v, A.v_ts, c0, first, c1);
    }
  };
  if (n_it > 0) fetch(0);
  for (int it = 0; it < n_it; ++it) {
    const int c0 = beg(it), c1 = lim(it);
    __syncthreads();
    t1.stash(sC1);
    t2.stash(sC2);
    if (KV && threadIdx.x < kBT) lse[threadIdx.x] = lse_n, delta[threadIdx.x] = delta_n;
    __syncthreads();
    if (it + 1 < n_it) fetch(it + 1);
    float s[kR][4], dp[kR][4];
    tile_dot<DH>(s, sR1, sC1, ty, tx);
    tile_dot<DH>(dp, sR2, sC2, ty, tx);
#pragma unroll
    for (int i = 0; i < kR; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = ty * kR + i, col = tx * 4 + j;
        const bool see = c0 + col < c1 && (KV ? (c0 + col >= r0 + r && c0 + col < limit[r]) : rows[r].sees(c0 + col));
        const int qi = KV ? col : r;
        const float p = see ? exp2f(s[i][j] * c - lse[qi]) : 0.f;
        dp[i][j] = see ? p * (dp[i][j] - delta[qi]) : 0.f;
        s[i][j] = p;
      }
    if (KV) {
      put_block(sP, s, ty, tx);
      __syncthreads();
      tile_acc<DH>(a2, sP, sC2, ty, tx);
      __syncthreads();
    }
    put_block(sP, dp, ty, tx);
    __syncthreads();
    tile_acc<DH>(a1, sP, sC1, ty, tx);
    if (!KV && it < nsink) {  // the sinks' gradients from these queries: P and dS once more, as [query][key]
      float og[kR][DH / 16];
      uint64_t ag[kR / 2][DH / 16];
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kR; ++i) {
          const float(&b)[4] = kv ? s[i] : dp[i];
          *reinterpret_cast<float4*>(sP + (ty * kR + i) * kPitch + tx * 4) = make_float4(b[0], b[1], b[2], b[3]);
#pragma unroll
          for (int n = 0; n < DH / 16; ++n) ag[i / 2][n] = 0;
        }
        __syncthreads();
        tile_acc<DH>(ag, sP, kv ? sR2 : sR1, ty, tx);
        rows_of(og, ag);
#pragma unroll
        for (int i = 0; i < kR; ++i)
          if (ty * kR + i < c1 - c0)
#pragma unroll
            for (int n = 0; n < DH / 16; ++n)
              A.part[part_at(A, blockIdx.x, blockIdx.y, kv, ty * kR + i) + tx + 16 * n] = og[i][n];
      }
    }
  }
  float o1[kR][DH / 16], o2[kR][DH / 16];
  rows_of(o1, a1);
  rows_of(o2, a2);
#pragma unroll
  for (int i = 0; i < kR; ++i) {
    const int t = r0 + ty * kR + i;
    if (t >= A.T) continue;
    const bool live = KV ? limit[ty * kR + i] > 0 : rows[ty * kR + i].i >= 0;
    const int H = KV ? A.Hkv : A.Hq;
    const int64_t at = ((int64_t)t * H + blockIdx.y) * A.Dh;
    float* g1 = (float*)(KV ? A.gk : A.gq) + at;
    float odd = 0.f;  // NaN as soon as one element is not finite
    if (KV)
      if (const float* far = far_sum<6>(A, t, hk))
#pragma unroll
        for (int n = 0; n < DH / 16; ++n) {
          o1[i][n] += far[tx + 16 * n];
          o2[i][n] += far[A.sinks * A.Dh + tx + 16 * n];
        }
#pragma unroll
    for (int n = 0; n < DH / 16; ++n) {
      g1[tx + 16 * n] = live ? o1[i][n] * A.scale : 0.f;
      if (KV) ((float*)A.gv + at)[tx + 16 * n] = live ? o2[i][n] : 0.f;
      odd = fmaf(o1[i][n], 0.f, fmaf(o2[i][n], 0.f, odd));
    }
    if (live && odd != 0.f) again[ty * kR + i] = 1;
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < kBT; r += kThreads / 32)
    if (again[r]) {
      if (KV) exact_gkv_row<float>(A, blockIdx.y, r0 + r);
      else exact_gq_row<float>(A, blockIdx.y, r0 + r);
    }
}

template <typename K>
static int launch(K kernel, dim3 grid, size_t smem, const AttnArgs& A, cudaStream_t st, const char* what) {
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return set_error(MR_E_LAUNCH, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
  }
  kernel<<<grid, kThreads, smem, st>>>(A);
  return check_launch(what);
}

template <int DH> static int fwd_dh(const AttnArgs& A, cudaStream_t st) {
  return launch(attn_fwd_f32<DH>, dim3((A.T + kBT - 1) / kBT, A.Hq), (3 * DH + kBT) * kPitch * 4, A, st, "attn_fwd_f32");
}
template <int DH> static int bwd_dh(const AttnArgs& A, cudaStream_t st) {
  const size_t sm = (4 * DH + kBT) * kPitch * 4;
  const unsigned n = (A.T + kBT - 1) / kBT;
  if (int rc = launch(attn_bwd_f32<DH, false>, dim3(n, A.Hq), sm, A, st, "attn_bwd_f32 (grad_q)")) return rc;
  if (A.part != nullptr)
    if (int rc = attn_sink_sum_launch<6>(A, st)) return rc;
  return launch(attn_bwd_f32<DH, true>, dim3(n, A.Hkv), sm, A, st, "attn_bwd_f32 (grad_k, grad_v)");
}

int attn_fwd_f32_launch(const AttnArgs& A, cudaStream_t st) {
  switch (A.Dh) {
    case 32: return fwd_dh<32>(A, st);
    case 64: return fwd_dh<64>(A, st);
    case 96: return fwd_dh<96>(A, st);
    default: return fwd_dh<128>(A, st);
  }
}

size_t attn_bwd_f32_ws_bytes(int64_t T, int64_t Hq, int64_t Dh, int64_t sinks) {
  return (size_t)((T * Hq + 3) / 4 * 16) + part_bytes<6>(T, Hq, Dh, sinks);
}

// ws: attn_bwd_f32_ws_bytes, 16-byte aligned
int attn_bwd_f32_launch(const AttnArgs& A0, void* ws, cudaStream_t st) {
  AttnArgs A = A0;
  A.delta = (float*)ws;
  if (has_far(A)) A.part = A.delta + ((int64_t)A.T * A.Hq + 3) / 4 * 4;
  attn_delta_f32<<<(unsigned)(((int64_t)A.T * A.Hq + 7) / 8), 256, 0, st>>>(A);
  if (int rc = check_launch("attn_delta_f32")) return rc;
  switch (A.Dh) {
    case 32: return bwd_dh<32>(A, st);
    case 64: return bwd_dh<64>(A, st);
    case 96: return bwd_dh<96>(A, st);
    default: return bwd_dh<128>(A, st);
  }
}

}  // namespace mr
