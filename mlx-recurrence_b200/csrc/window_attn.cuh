// Sliding-window attention with sinks: arguments, masks and the exact
// row-by-row forms shared by the attention kernels.
//
// A batch is T tokens in a row, [T, H, Dh]; sequences are the ranges
// cu[s] .. cu[s+1]-1, or (cu == NULL) consecutive runs of L tokens. Query i
// sees key j of its own sequence when
//   j <= i  and  (i - j < window  or  j - start < sinks).
// Tokens outside every sequence are nobody's key; their rows are zero.
#pragma once

#include "common.cuh"

namespace mr {

// two float32 operations in one instruction
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) { return pair(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
  lo = __uint_as_float(a), hi = __uint_as_float(b);
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

struct AttnArgs {
  const void *q, *k, *v;            // [T, H, Dh], rows dense, strides in elements
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  const int* cu;                    // [S + 1] or NULL
  int S, L;                         // L: sequence length when cu is NULL
  int T, Hq, Hkv, Dh;
  int window, sinks;                // window <= T
  float scale;                      // > 0
  void* y;                          // [T, Hq, Dh] dense
  void* y_low;                      // [T, Hq, Dh]: what rounding y to its type drops, rounded too; NULL when not wanted
  float* lse;                       // [Hq, T]: log2 of the row's sum of exponentials; NULL when not wanted
  // backward
  const void* gy;                   // [T, Hq, Dh] dense
  float* delta;                     // [Hq, T]: sum_d gy y
  void *gq, *gk, *gv;               // [T, Hq, Dh], [T, Hkv, Dh] dense
  float* part;                      // sink partials (below), or NULL
};

struct SeqRange {
  int start, end;  // end <= start: no sequence
};

// The sequence that holds token t. Entries of cu are only compared and clamped
// to [0, T], so a malformed cu cannot lead an access out of range.
__device__ __forceinline__ SeqRange seq_of(const AttnArgs& A, int t) {
  if (t < 0 || t >= A.T) return {0, 0};
  if (A.cu == nullptr) {
    const int s = t / A.L * A.L;
    return {s, min(s + A.L, A.T)};
  }
  int lo = 0, hi = A.S;  // the last s with cu[s] <= t
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if (A.cu[m] <= t) lo = m; else hi = m - 1;
  }
  const int s = A.cu[lo];
  if (lo >= A.S || s > t) return {0, 0};
  return {max(s, 0), min(A.cu[lo + 1], A.T)};
}

__device__ __forceinline__ int first_token(const AttnArgs& A) { return A.cu ? min(max(A.cu[0], 0), A.T) : 0; }
__device__ __forceinline__ int end_token(const AttnArgs& A) { return A.cu ? min(max(A.cu[A.S], 0), A.T) : A.T; }

// What a query sees: keys [lo, i] and sinks [start, sink_end).
struct RowMask {
  int i, lo, start, sink_end;
  __device__ bool sees(int j) const { return (j >= lo && j <= i) || (j >= start && j < sink_end && j <= i); }
};
__device__ __forceinline__ RowMask row_mask(const AttnArgs& A, int i) {
  const SeqRange s = seq_of(A, i);
  if (s.end <= i) return {-1, INT32_MAX, INT32_MAX, -1};
  return {i, max(s.start, i - A.window + 1), s.start, s.start + min(A.sinks, A.T)};
}

// Keys that the queries [q0, q1) may see: the band [kmin, kend) and the sinks
// before it, [s0, send), which belong to the first query's sequence (any later
// sequence starts inside the band). Nothing when kend <= kmin.
struct KeyRange {
  int kmin, kend, s0, send;
};
__device__ __forceinline__ KeyRange keys_of(const AttnArgs& A, int q0, int q1) {
  const int f = max(q0, first_token(A)), e = min(q1, end_token(A));
  if (f >= e) return {0, 0, 0, 0};
  const SeqRange s = seq_of(A, f);
  const int kmin = max(min(s.start, f), f - A.window + 1);
  return {kmin, e, s.start, min(s.start + min(A.sinks, A.T), kmin)};
}

// The first query that no longer sees key j (0: j is nobody's key); queries
// j .. hi-1 see it.
__device__ __forceinline__ int key_limit(const AttnArgs& A, int j) {
  const SeqRange s = seq_of(A, j);
  if (s.end <= j) return 0;
  return j - s.start < A.sinks ? s.end : min(s.end, j + A.window);
}

// ---- the sinks' far queries ----------------------------------------------------
// A key that stays visible to the end of a long sequence would make the pass over
// its row tile walk every later query. Instead a query tile (2^SH queries) whose
// window has left the sinks (its band of keys starts behind them) adds their
// gradients on the way, as float32 partials [query tile][head][k, v][sink][Dh];
// attn_sink_sum adds them up in their order, and the sink's row tile takes the sum.

// Query tiles from this one on are far from key j of their own sequence: 2^SH n >= j + window.
template <int SH> __device__ __forceinline__ int first_far(const AttnArgs& A, int j) {
  return (int)(((int64_t)j + A.window + (1 << SH) - 1) >> SH);
}
__device__ __forceinline__ int64_t part_at(const AttnArgs& A, int n, int h, int kv, int r) {
  return ((((int64_t)n * A.Hq + h) * 2 + kv) * A.sinks + r) * A.Dh;
}
// The first query that the pass over key tiles leaves to the partials, for a sink j of a sequence that ends at `end`.
template <int SH> __device__ __forceinline__ int near_end(const AttnArgs& A, int j, int end) {
  return (int)min((int64_t)end, (int64_t)first_far<SH>(A, j) << SH);
}
// key_limit without the far queries.
template <int SH> __device__ __forceinline__ int near_limit(const AttnArgs& A, int j) {
  const SeqRange s = seq_of(A, j);
  if (s.end <= j) return 0;
  const int hi = min(s.end, j + A.window);
  return j - s.start < A.sinks ? max(hi, near_end<SH>(A, j, s.end)) : hi;
}
// Queries [qbeg, qend) that may see the keys [k0, k1), without the far ones.
struct QueryRange {
  int qbeg, qend;
};
template <int SH> __device__ __forceinline__ QueryRange near_queries(const AttnArgs& A, int k0, int k1) {
  const int f = max(k0, first_token(A)), e = min(k1, end_token(A));
  if (f >= e) return {0, 0};
  const SeqRange s = seq_of(A, e - 1);
  int end = max(e, min(s.end, e - 1 + A.window));
  const int last_sink = min(e - 1, s.start + A.sinks - 1);
  if (last_sink >= max(f, s.start)) end = max(end, near_end<SH>(A, last_sink, s.end));
  return {f, end};
}
// The summed partials (k, then v `A.sinks * A.Dh` further on) of key j for key head hk, or NULL.
template <int SH> __device__ __forceinline__ const float* far_sum(const AttnArgs& A, int j, int hk) {
  if (A.part == nullptr) return nullptr;
  const SeqRange s = seq_of(A, j);
  if (s.end <= j || j - s.start >= A.sinks || (int64_t)first_far<SH>(A, j) << SH >= s.end) return nullptr;
  return A.part + part_at(A, first_far<SH>(A, s.start), hk * (A.Hq / A.Hkv), 0, j - s.start);
}
template <int SH> size_t part_bytes(int64_t T, int64_t Hq, int64_t Dh, int64_t sinks) {
  return (size_t)((T + (1 << SH) - 1) / (1 << SH) * Hq * 2 * sinks * Dh * 4);
}
static inline bool has_far(const AttnArgs& A) { return A.sinks > 0 && A.window < A.T; }

// part[first far tile of a sequence][first head of a group] <- the sum over the
// sequence's far tiles and the group's heads, in their order: 4 threads per
// element take a quarter of the terms each. Grid: query tiles, key heads, sinks.
template <int SH> __global__ void __launch_bounds__(1024) attn_sink_sum(const __grid_constant__ AttnArgs A) {
  __shared__ float sums[4][256];
  const int n = blockIdx.x, hk = blockIdx.y, r = blockIdx.z, G = A.Hq / A.Hkv;
  const KeyRange R = keys_of(A, n << SH, (n + 1) << SH);
  if (R.send <= R.s0 || first_far<SH>(A, R.s0) != n) return;
  const SeqRange s = seq_of(A, R.s0);
  const int beg = max(n, first_far<SH>(A, s.start + r)), tiles = ((s.end + (1 << SH) - 1) >> SH) - beg;
  if (tiles <= 0 || s.start + r >= s.end) return;
  const int v = threadIdx.x & 255, quarter = threadIdx.x >> 8, terms = tiles * G;
  const int kv = v / A.Dh, d = v % A.Dh;
  float sum = 0.f;
  if (kv < 2)
#pragma unroll 8
    for (int x = terms * quarter / 4; x < terms * (quarter + 1) / 4; ++x)
      sum += A.part[part_at(A, beg + x / G, hk * G + x % G, kv, r) + d];
  sums[quarter][v] = sum;
  __syncthreads();
  if (quarter == 0 && kv < 2)
    A.part[part_at(A, n, hk * G, kv, r) + d] = (sums[0][v] + sums[1][v]) + (sums[2][v] + sums[3][v]);
}
template <int SH> int attn_sink_sum_launch(const AttnArgs& A, cudaStream_t st) {
  attn_sink_sum<SH><<<dim3((A.T + (1 << SH) - 1) >> SH, A.Hkv, A.sinks), 1024, 0, st>>>(A);
  return check_launch("attn_sink_sum");
}

// ---- exact rows --------------------------------------------------------------
// The tiled kernels multiply masked terms by zero, which an infinity or a NaN
// that a row must not see (another sequence's, a later token's) turns into a
// NaN. A row whose results are not finite, or whose scores are all -infinity, is
// therefore computed again here, one warp per row, from its visible keys (queries)
// alone: whatever non-finite value then remains is the row's own. Only ever reached by
// inputs that hold infinities or NaN, which pay for it (fp16 loss scaling's probes
// among them). T=16384, fp16, 32 heads of 64, window 1024: one infinity in grad_y 5.5
// ms of backward in place of 1.0 (18 with a shuffle reduction per term), one token of v
// that is NaN 4.2 ms of forward in place of 0.27 (16), everything infinite or NaN 149
// and 46 ms (543, 200); bf16, 16 heads of 128 on 4, window 2048, 4 sinks: 40 and 10 ms
// (92, 32), everything 230 and 62 (656, 205).

constexpr float kAttnLog2e = 1.4426950408889634f;

__device__ __forceinline__ float attn_warp_sum(float v) {
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
  return v;
}

__device__ __forceinline__ float attn_warp_max(float v) {
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
  return v;
}

struct RowVec {
  float v[4];  // elements lane + 32 n of one head's row, Dh <= 128
};
template <typename T> __device__ __forceinline__ RowVec row_load(const T* p, int Dh, int lane) {
  RowVec r;
#pragma unroll
  for (int n = 0; n < 4; ++n) r.v[n] = 32 * n < Dh ? to_f(p[lane + 32 * n]) : 0.f;
  return r;
}
template <typename T> __device__ __forceinline__ void row_store(T* p, const RowVec& r, float f, int Dh, int lane) {
#pragma unroll
  for (int n = 0; n < 4; ++n)
    if (32 * n < Dh) p[lane + 32 * n] = from_f<T>(r.v[n] * f);
}
__device__ __forceinline__ void row_axpy(RowVec& a, float f, const RowVec& b) {
#pragma unroll
  for (int n = 0; n < 4; ++n) a.v[n] = fmaf(f, b.v[n], a.v[n]);
}
// A lane's own product of two rows (16-byte aligned).
template <typename T> __device__ __forceinline__ float lane_dot(const T* a, const T* b, int Dh) {
  constexpr int N = 16 / sizeof(T);
  float s = 0.f;
#pragma unroll 4
  for (int d = 0; d < Dh; d += N) {
    const Vec<T, N> x = ld_vec<T, N>(a + d), y = ld_vec<T, N>(b + d);
#pragma unroll
    for (int j = 0; j < N; ++j) s = fmaf(to_f(x.v[j]), to_f(y.v[j]), s);
  }
  return s;
}
// a += sum over the warp's first `n` lanes of f x row(j), the rows' loads eight ahead
template <typename T>
__device__ __forceinline__ void rows_axpy(RowVec& a, float f, int j, int n, const T* p, int64_t ts, int Dh, int lane) {
  for (int x = 0; x < n; x += 8) {
    RowVec r[8];
#pragma unroll
    for (int y = 0; y < 8; ++y) r[y] = row_load(p + __shfl_sync(0xffffffffu, j, min(x + y, n - 1)) * ts, Dh, lane);
#pragma unroll
    for (int y = 0; y < 8; ++y) {
      const float fy = __shfl_sync(0xffffffffu, f, min(x + y, n - 1));
      if (x + y < n) row_axpy(a, fy, r[y]);
    }
  }
}

// A row's visible terms, 32 at a time: each lane the scores of one, then all lanes the sums over them, term by term.
template <typename T> __device__ __noinline__ void exact_fwd_row(const AttnArgs& A, int h, int i) {
  const int lane = threadIdx.x & 31, hk = h / (A.Hq / A.Hkv);
  const RowMask w = row_mask(A, i);
  if (w.i < 0) return;
  const T* k = (const T*)A.k + hk * A.k_hs;
  const T* v = (const T*)A.v + hk * A.v_hs;
  const T* q = (const T*)A.q + i * A.q_ts + h * A.q_hs;
  RowVec o = {};
  float m = -INFINITY, l = 0.f;
  const int sinks = max(0, min(w.sink_end, w.lo) - w.start), n = sinks + i - w.lo + 1;
  for (int b = 0; b < n; b += 32) {
    const int x = min(b + lane, n - 1), j = x < sinks ? w.start + x : w.lo + x - sinks;
    const float d = lane_dot(q, k + j * A.k_ts, A.Dh) * (A.scale * kAttnLog2e), s = b + lane < n ? d : -INFINITY;
    const float mx = fmaxf(m, attn_warp_max(s)), base = mx == -INFINITY ? 0.f : mx, keep = exp2f(m - base);
    const float e = b + lane < n ? exp2f(s - base) : 0.f;
    m = mx;
    l = l * keep + attn_warp_sum(e);
#pragma unroll
    for (int c = 0; c < 4; ++c) o.v[c] *= keep;
    rows_axpy(o, e, j, min(32, n - b), v, A.v_ts, A.Dh, lane);
  }
  const int64_t at = ((int64_t)i * A.Hq + h) * A.Dh;
  const float inv = 1.f / l;
#pragma unroll
  for (int c = 0; c < 4; ++c) o.v[c] *= inv;
  row_store((T*)A.y + at, o, 1.f, A.Dh, lane);
  if (A.y_low != nullptr) {
#pragma unroll
    for (int c = 0; c < 4; ++c) o.v[c] -= to_f(from_f<T>(o.v[c]));
    row_store((T*)A.y_low + at, o, 1.f, A.Dh, lane);
  }
  if (A.lse != nullptr && lane == 0) A.lse[(int64_t)h * A.T + i] = m + log2f(l);
}

template <typename T> __device__ __noinline__ void exact_gq_row(const AttnArgs& A, int h, int i) {
  const int lane = threadIdx.x & 31, hk = h / (A.Hq / A.Hkv);
  const RowMask w = row_mask(A, i);
  if (w.i < 0) return;
  const T* k = (const T*)A.k + hk * A.k_hs;
  const T* v = (const T*)A.v + hk * A.v_hs;
  const int64_t at = ((int64_t)i * A.Hq + h) * A.Dh;
  const T *q = (const T*)A.q + i * A.q_ts + h * A.q_hs, *g = (const T*)A.gy + at;
  const float lse = A.lse[(int64_t)h * A.T + i], delta = A.delta[(int64_t)h * A.T + i];
  RowVec o = {};
  const int sinks = max(0, min(w.sink_end, w.lo) - w.start), n = sinks + i - w.lo + 1;
  for (int b = 0; b < n; b += 32) {
    const int x = min(b + lane, n - 1), j = x < sinks ? w.start + x : w.lo + x - sinks;
    const float p = exp2f(lane_dot(q, k + j * A.k_ts, A.Dh) * (A.scale * kAttnLog2e) - lse);
    const float f = p * (lane_dot(g, v + j * A.v_ts, A.Dh) - delta);
    rows_axpy(o, f, j, min(32, n - b), k, A.k_ts, A.Dh, lane);
  }
  row_store((T*)A.gq + at, o, A.scale, A.Dh, lane);
}

template <typename T> __device__ __noinline__ void exact_gkv_row(const AttnArgs& A, int hk, int j) {
  const int lane = threadIdx.x & 31, G = A.Hq / A.Hkv, end = key_limit(A, j);
  if (end == 0) return;
  const T* k = (const T*)A.k + j * A.k_ts + hk * A.k_hs;
  const T* v = (const T*)A.v + j * A.v_ts + hk * A.v_hs;
  const int64_t gts = (int64_t)A.Hq * A.Dh;
  RowVec gk = {}, gv = {};
  for (int h = hk * G; h < (hk + 1) * G; ++h) {
    const T *q = (const T*)A.q + h * A.q_hs, *g = (const T*)A.gy + (int64_t)h * A.Dh;
    const float *lse = A.lse + (int64_t)h * A.T, *delta = A.delta + (int64_t)h * A.T;
    for (int b = j; b < end; b += 32) {
      const int i = min(b + lane, end - 1), n = min(32, end - b);
      const float p = exp2f(lane_dot(k, q + i * A.q_ts, A.Dh) * (A.scale * kAttnLog2e) - lse[i]);
      const float f = p * (lane_dot(v, g + i * gts, A.Dh) - delta[i]);
      rows_axpy(gv, p, i, n, g, gts, A.Dh, lane);
      rows_axpy(gk, f, i, n, q, A.q_ts, A.Dh, lane);
    }
  }
  const int64_t at = ((int64_t)j * A.Hkv + hk) * A.Dh;
  row_store((T*)A.gk + at, gk, A.scale, A.Dh, lane);
  row_store((T*)A.gv + at, gv, 1.f, A.Dh, lane);
}

}  // namespace mr
