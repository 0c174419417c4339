// RG-LRU recurrence h_t = a_t h_{t-1} + x_t over a packed batch: sequences of
// any lengths (zero included) lie back to back in [T, D]; sequence s holds the
// tokens cu[s] .. cu[s+1]-1 and starts from h0[s] (zero without h0). Rows
// outside every sequence get zeros (outputs and gradients).
//
// Adjoint: adj_t = gy_t + r_t, r_{t-1} = a_t adj_t, where r starts from gf_s at
// the sequence's last token; grad_x = adj, grad_a[t] = adj_t h_{t-1},
// grad_h0[s] = r left of its first token (gf_s for an empty sequence).
//
// One pass over the data, HBM-bound: a CTA takes kChunk steps of 32 V channels,
// 8 warps x kSteps steps each, and holds them in registers. A step is the affine
// map h -> a h + x, so runs of steps compose to one map (A, B): per thread, per
// CTA (shared memory) and per chunk. A chunk publishes its map, looks back over
// the chunks before it (8 at a time, one per warp) until it meets one whose state
// is known, and publishes its own state. A sequence border cuts the chain: what
// follows it does not depend on the past. Borders are the same for all channels,
// so every branch on them is uniform. The backward runs the same scheme from the
// right and rebuilds h from the states that the forward kept per chunk.
#include "common.cuh"
#include "tma.cuh"

namespace mr {

constexpr int kWarps = 8;
constexpr int kSteps = 16;               // steps of a thread
constexpr int kChunk = kWarps * kSteps;  // steps of a CTA

// A chunk's map or state for one channel, written and read as one 16-byte access
// (single-copy atomic), so no flag or fence stands beside it.
struct alignas(16) Rec {
  float A, B;    // kMap: state out = A state in + B; kState: state out = B
  uint32_t tag;  // 0: not there yet
  uint32_t pad;
};
enum : uint32_t { kMap = 1, kState = 2 };

__device__ __forceinline__ void rec_store(Rec* p, float A, float B, uint32_t tag) {
  const uint64_t lo = (uint64_t)__float_as_uint(B) << 32 | __float_as_uint(A), hi = tag;
  asm volatile("{\n\t.reg .b128 r;\n\tmov.b128 r, {%1, %2};\n\tst.relaxed.gpu.global.b128 [%0], r;\n\t}" ::"l"(p), "l"(lo),
               "l"(hi)
               : "memory");
}
__device__ __forceinline__ Rec rec_load(const Rec* p) {
  uint64_t lo, hi;
  asm volatile("{\n\t.reg .b128 r;\n\tld.relaxed.gpu.global.b128 r, [%2];\n\tmov.b128 {%0, %1}, r;\n\t}"
               : "=l"(lo), "=l"(hi)
               : "l"(p)
               : "memory");
  return {__uint_as_float((uint32_t)lo), __uint_as_float((uint32_t)(lo >> 32)), (uint32_t)hi, 0};
}

// Polls until the record is there; after 2 s (its writer is always a CTA that
// started earlier, so only a device failure gets here) sets the device error word.
__device__ __forceinline__ Rec rec_wait(const Rec* p) {
  Rec r = rec_load(p);
  if (r.tag != 0) return r;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    r = rec_load(p);
    if (r.tag != 0) return r;
    if ((i & 255u) == 255u &&
        (*reinterpret_cast<volatile int*>(&g_device_error) != 0 || globaltimer_ns() - t0 > 2000000000ull))
      break;
  }
  atomicCAS(&g_device_error, 0, 1);
  return {0.f, 0.f, kState, 0};
}

// The borders inside a chunk, per token: the sequence that starts there (else -1)
// and the sequence that ends there; tokens [lo, hi) of the chunk lie in sequences.
struct Borders {
  int start[kChunk], end[kChunk];
  int lo, hi;
  uint32_t starts, ends;  // bit w: a sequence starts (ends) in warp w's steps
  // no border in warp w's steps, and all of them in a sequence: the short loops serve
  __device__ bool plain(int w) const {
    return !((starts | ends) >> w & 1) && w * kSteps >= lo && (w + 1) * kSteps <= hi;
  }
};

// All threads call it; the result is there after the next barrier.
__device__ __forceinline__ void find_borders(Borders& b, const int* __restrict__ cu, int S, int64_t t0, int n) {
  for (int i = threadIdx.x; i < kChunk; i += kWarps * 32) b.start[i] = b.end[i] = -1;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  int l = 0, r = S;  // the first s with cu[s] >= t0
  while (l < r) {
    const int m = (l + r) >> 1;
    if (cu[m] < t0) l = m + 1; else r = m;
  }
  uint32_t starts = 0, ends = 0;
  for (int s = l + threadIdx.x; s <= S; s += 32) {
    const int64_t at = cu[s] - t0;
    if (at > n) break;
    if (at >= 0 && at < n && s < S && cu[s + 1] > cu[s]) b.start[at] = s, starts |= 1u << (at / kSteps);
    if (at >= 1 && s > 0 && cu[s] > cu[s - 1]) b.end[at - 1] = s - 1, ends |= 1u << ((at - 1) / kSteps);
  }
  starts = __reduce_or_sync(0xffffffffu, starts);
  ends = __reduce_or_sync(0xffffffffu, ends);
  if (threadIdx.x == 0) {
    b.lo = (int)min(max((int64_t)cu[0] - t0, (int64_t)0), (int64_t)n);
    b.hi = (int)min(max((int64_t)cu[S] - t0, (int64_t)0), (int64_t)n);
    b.starts = starts, b.ends = ends;
  }
}

// V channels of one step; those at or behind D read as zero
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> ld_step(const T* p, bool ok) {
  Vec<T, V> r;
  if (ok) {
    r = ld_vec<T, V>(p);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) r.v[v] = from_f<T>(0.f);
  }
  return r;
}

struct Chain {
  float A[kWarps][64], B[kWarps][64];  // the warps' maps
  Rec back[kWarps][64];                // what the look-back read
  float carry[64];                     // the state entering the chunk
};

// State entering chunk `rank` of the chain (0: the first to start). `cut`: the
// chunk holds a border, so its outgoing state is B whatever enters; `need`:
// whether anything in the chunk depends on what enters. Publishes this chunk's
// own record. All threads call it, after the warps' maps are in sh.
template <int V, typename F>
__device__ __forceinline__ void look_back(Chain& sh, Rec* recs, int64_t stride, int64_t ch, bool live, int rank, int last,
                                          bool cut, bool need, F total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  float A[V], B[V];
  if (w == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      total(lane * V + v, A[v], B[v]);
      if (live && rank < last) rec_store(recs + rank * stride + ch + v, A[v], B[v], cut || rank == 0 ? kState : kMap);
    }
  }
  float a[V], b[V];  // the composed map of the chunks looked at so far
  bool known[V];     // a record may turn from map to state between two reads, so each channel stops by itself
#pragma unroll
  for (int v = 0; v < V; ++v) a[v] = 1.f, b[v] = 0.f, known[v] = false;
  if (need && rank > 0) {
    for (int at = rank - 1;; at -= kWarps) {
      const int mine = at - w;
#pragma unroll
      for (int v = 0; v < V; ++v)
        sh.back[w][lane * V + v] = mine >= 0 && live ? rec_wait(recs + mine * stride + ch + v) : Rec{0.f, 0.f, kState, 0};
      __syncthreads();
      bool open = false;
#pragma unroll
      for (int v = 0; w == 0 && v < V; ++v) {
        for (int i = 0; i < kWarps && !known[v]; ++i) {
          const Rec r = sh.back[i][lane * V + v];
          b[v] = fmaf(a[v], r.B, b[v]);
          a[v] *= r.A;
          known[v] = r.tag == kState;
        }
        open |= !known[v];
      }
      if (!__syncthreads_or(open)) break;
    }
  }
  if (w == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sh.carry[lane * V + v] = b[v];
      if (live && rank < last && need && !cut && rank > 0)
        rec_store(recs + rank * stride + ch + v, 0.f, fmaf(A[v], b[v], B[v]), kState);
    }
  }
  __syncthreads();
}

// (chunk rank, channel tile) of this CTA: tickets follow the order in which CTAs
// start, so whatever a chunk waits for is already running.
__device__ __forceinline__ int64_t take_ticket(uint32_t* counter) {
  __shared__ uint32_t t;
  if (counter == nullptr) return blockIdx.x;
  if (threadIdx.x == 0) t = atomicAdd(counter, 1u);
  __syncthreads();
  return t;
}

template <typename T, int V>
__global__ void __launch_bounds__(kWarps * 32, V == 1 ? 4 : 3)
packed_fwd_kernel(const T* __restrict__ a, const T* __restrict__ x, const int* __restrict__ cu, int S, int64_t L,
                  int64_t D, const float* __restrict__ h0, float* __restrict__ y, float* __restrict__ ckpt,
                  float* __restrict__ fin, uint32_t* counter, Rec* recs, int nchunk, int ntile) {
  __shared__ Chain sh;
  __shared__ Borders bd;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t ticket = take_ticket(counter);
  const int chunk = (int)(ticket / ntile);
  const int64_t ch = (ticket % ntile) * (32 * V) + lane * V, t0 = (int64_t)chunk * kChunk;
  const int n = (int)min((int64_t)kChunk, L - t0), k0 = w * kSteps;
  const bool live = ch < D;
  Vec<T, V> av[kSteps], xv[kSteps];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int64_t at = (t0 + k0 + k) * D + ch;
    av[k] = ld_step<T, V>(a + at, live && k0 + k < n);
    xv[k] = ld_step<T, V>(x + at, live && k0 + k < n);
  }
  find_borders(bd, cu, S, t0, n);
  __syncthreads();
  const bool plain = bd.plain(w);
  {
    float A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
    if (plain) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          B[v] = fmaf(to_f(av[k].v[v]), B[v], to_f(xv[k].v[v]));
          A[v] *= to_f(av[k].v[v]);
        }
    } else {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int i = k0 + k, s = bd.start[i];
      if (i < bd.lo || i >= bd.hi) continue;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (s >= 0) B[v] = h0 && live ? h0[s * D + ch + v] : 0.f;
        B[v] = fmaf(to_f(av[k].v[v]), B[v], to_f(xv[k].v[v]));
        A[v] *= to_f(av[k].v[v]);
      }
    }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) sh.A[w][lane * V + v] = A[v], sh.B[w][lane * V + v] = B[v];
  }
  __syncthreads();
  const uint32_t cut = bd.starts;
  // the state after warps 0 .. e-1, given the one before them
  auto through = [&](int c, int e, float& A, float& B) {
    for (int i = 0; i < e; ++i) {
      if (cut >> i & 1) {
        A = 0.f;
        B = sh.B[i][c];
      } else {
        B = fmaf(sh.A[i][c], B, sh.B[i][c]);
        A *= sh.A[i][c];
      }
    }
  };
  const bool need = bd.lo == 0 && bd.hi > 0 && bd.start[0] < 0;
  look_back<V>(sh, recs, D, ch, live, chunk, nchunk - 1, cut != 0, need, [&](int c, float& A, float& B) {
    A = 1.f, B = 0.f;
    through(c, kWarps, A, B);
  });
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float A = 1.f;
    h[v] = sh.carry[lane * V + v];
    if (ckpt != nullptr && w == 0 && live && n > 0) ckpt[chunk * D + ch + v] = h[v];
    through(lane * V + v, w, A, h[v]);
  }
  if (plain) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = fmaf(to_f(av[k].v[v]), h[v], to_f(xv[k].v[v]));
      if (live) st_stream_f32<V>(y + (t0 + k0 + k) * D + ch, h);
    }
  } else {
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int i = k0 + k;
    if (i >= n) break;
    const bool in = i >= bd.lo && i < bd.hi;
    const int s = bd.start[i], e = bd.end[i];
    float out[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (in && s >= 0) h[v] = h0 && live ? h0[s * D + ch + v] : 0.f;
      if (in) h[v] = fmaf(to_f(av[k].v[v]), h[v], to_f(xv[k].v[v]));
      out[v] = in ? h[v] : 0.f;
      if (fin != nullptr && in && e >= 0 && live) fin[e * D + ch + v] = h[v];
    }
    if (live) st_stream_f32<V>(y + (t0 + i) * D + ch, out);
  }
  }
  if (fin != nullptr && live)  // empty sequences, spread over the chunks
    for (int s = (int)((int64_t)chunk * S / nchunk) + w; s < (int)((int64_t)(chunk + 1) * S / nchunk); s += kWarps)
      if (cu[s + 1] <= cu[s])
#pragma unroll
        for (int v = 0; v < V; ++v) fin[s * D + ch + v] = h0 ? h0[s * D + ch + v] : 0.f;
}

template <typename T, int V>
__global__ void __launch_bounds__(kWarps * 32, 2)
packed_bwd_kernel(const float* __restrict__ gy, const float* __restrict__ gf, const float* __restrict__ ckpt,
                  const T* __restrict__ a, const T* __restrict__ x, const int* __restrict__ cu, int S, int64_t L,
                  int64_t D, const float* __restrict__ h0, T* __restrict__ ga, T* __restrict__ gx,
                  float* __restrict__ gh0, uint32_t* counter, Rec* recs, int nchunk, int ntile) {
  __shared__ Chain sh;
  __shared__ float fA[kWarps][64], fB[kWarps][64];  // the warps' maps of the forward recurrence
  __shared__ Borders bd;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t ticket = take_ticket(counter);
  const int rank = (int)(ticket / ntile), chunk = nchunk - 1 - rank;
  const int64_t ch = (ticket % ntile) * (32 * V) + lane * V, t0 = (int64_t)chunk * kChunk;
  const int n = (int)min((int64_t)kChunk, L - t0), k0 = w * kSteps;
  const bool live = ch < D;
  Vec<T, V> av[kSteps], xv[kSteps];
  Vec<float, V> gv[kSteps];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int64_t at = (t0 + k0 + k) * D + ch;
    av[k] = ld_step<T, V>(a + at, live && k0 + k < n);
    gv[k] = ld_step<float, V>(gy + at, live && k0 + k < n);
    xv[k] = ld_step<T, V>(x + at, live && k0 + k < n);
  }
  find_borders(bd, cu, S, t0, n);
  __syncthreads();
  const bool plain = bd.plain(w);
  {
    float A[V], B[V], P[V], Q[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = P[v] = 1.f, B[v] = Q[v] = 0.f;
    if (plain) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          B[v] = fmaf(to_f(av[k].v[v]), B[v], to_f(xv[k].v[v]));
          A[v] *= to_f(av[k].v[v]);
        }
#pragma unroll
      for (int k = kSteps - 1; k >= 0; --k)
#pragma unroll
        for (int v = 0; v < V; ++v) Q[v] = to_f(av[k].v[v]) * (gv[k].v[v] + Q[v]);
#pragma unroll
      for (int v = 0; v < V; ++v) P[v] = A[v];
    } else {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int i = k0 + k, s = bd.start[i];
      if (i < bd.lo || i >= bd.hi) continue;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (s >= 0) B[v] = h0 && live ? h0[s * D + ch + v] : 0.f;
        B[v] = fmaf(to_f(av[k].v[v]), B[v], to_f(xv[k].v[v]));
        A[v] *= to_f(av[k].v[v]);
      }
    }
#pragma unroll
    for (int k = kSteps - 1; k >= 0; --k) {
      const int i = k0 + k, e = bd.end[i];
      if (i < bd.lo || i >= bd.hi) continue;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (e >= 0) Q[v] = gf && live ? gf[e * D + ch + v] : 0.f;
        Q[v] = to_f(av[k].v[v]) * (gv[k].v[v] + Q[v]);
        P[v] *= to_f(av[k].v[v]);
      }
    }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      fA[w][lane * V + v] = A[v], fB[w][lane * V + v] = B[v];
      sh.A[w][lane * V + v] = P[v], sh.B[w][lane * V + v] = Q[v];
    }
  }
  __syncthreads();
  const uint32_t cut = bd.starts, end = bd.ends;
  // r left of warps 7 .. e, given the one right of them
  auto through = [&](int c, int e, float& P, float& Q) {
    for (int i = kWarps - 1; i >= e; --i) {
      if (end >> i & 1) {
        P = 0.f;
        Q = sh.B[i][c];
      } else {
        Q = fmaf(sh.A[i][c], Q, sh.B[i][c]);
        P *= sh.A[i][c];
      }
    }
  };
  const bool need = bd.hi == n && bd.hi > bd.lo && bd.end[n - 1] < 0;
  look_back<V>(sh, recs, D, ch, live, rank, nchunk - 1, end != 0, need, [&](int c, float& P, float& Q) {
    P = 1.f, Q = 0.f;
    through(c, 0, P, Q);
  });
  float r[V], h[V], before[kSteps][V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float P = 1.f;
    r[v] = sh.carry[lane * V + v];
    through(lane * V + v, w + 1, P, r[v]);
    h[v] = live && n > 0 ? ckpt[chunk * D + ch + v] : 0.f;
    for (int i = 0; i < w; ++i)
      h[v] = cut >> i & 1 ? fB[i][lane * V + v] : fmaf(fA[i][lane * V + v], h[v], fB[i][lane * V + v]);
  }
  if (plain) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        before[k][v] = h[v];
        h[v] = fmaf(to_f(av[k].v[v]), h[v], to_f(xv[k].v[v]));
      }
#pragma unroll
    for (int k = kSteps - 1; k >= 0; --k) {
      float oa[V], ox[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        ox[v] = gv[k].v[v] + r[v];
        oa[v] = ox[v] * before[k][v];
        r[v] = to_f(av[k].v[v]) * ox[v];
      }
      if (live) {
        st_vec<T, V>(ga + (t0 + k0 + k) * D + ch, oa);
        st_vec<T, V>(gx + (t0 + k0 + k) * D + ch, ox);
      }
    }
  } else {
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int i = k0 + k, s = bd.start[i];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (s >= 0) h[v] = h0 && live ? h0[s * D + ch + v] : 0.f;
      before[k][v] = h[v];
      h[v] = fmaf(to_f(av[k].v[v]), h[v], to_f(xv[k].v[v]));
    }
  }
#pragma unroll
  for (int k = kSteps - 1; k >= 0; --k) {
    const int i = k0 + k;
    if (i >= n) continue;
    const bool in = i >= bd.lo && i < bd.hi;
    const int s = bd.start[i], e = bd.end[i];
    float oa[V], ox[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (in && e >= 0) r[v] = gf && live ? gf[e * D + ch + v] : 0.f;
      const float adj = gv[k].v[v] + r[v];
      oa[v] = in ? adj * before[k][v] : 0.f;
      ox[v] = in ? adj : 0.f;
      if (in) r[v] = to_f(av[k].v[v]) * adj;
      if (gh0 != nullptr && in && s >= 0 && live) gh0[s * D + ch + v] = r[v];
    }
    if (live) {
      st_vec<T, V>(ga + (t0 + i) * D + ch, oa);
      st_vec<T, V>(gx + (t0 + i) * D + ch, ox);
    }
  }
  }
  if (gh0 != nullptr && live)
    for (int s = (int)((int64_t)chunk * S / nchunk) + w; s < (int)((int64_t)(chunk + 1) * S / nchunk); s += kWarps)
      if (cu[s + 1] <= cu[s])
#pragma unroll
        for (int v = 0; v < V; ++v) gh0[s * D + ch + v] = gf ? gf[s * D + ch + v] : 0.f;
}

static int64_t chunks(int64_t T) { return (T + kChunk - 1) / kChunk; }
static size_t ws_bytes_of(int64_t T, int64_t D) {
  // a ticket counter, and a record per chunk and channel; one chunk needs neither
  return chunks(T) > 1 ? 16 + (size_t)chunks(T) * D * sizeof(Rec) : 0;
}

static int prepare_ws(const char* what, int64_t T, int64_t D, int ntile, void* ws, size_t bytes, cudaStream_t st) {
  const size_t need = ws_bytes_of(T, D);
  if (need > 0 && (ws == nullptr || bytes < need || ((uintptr_t)ws & 15u)))
    return set_error(MR_E_WORKSPACE, "%s: needs %zu bytes of 16-byte aligned workspace, got %zu", what, need, bytes);
  if (chunks(T) * (int64_t)ntile > INT32_MAX) return set_error(MR_E_SHAPE, "%s: T * D too large", what);
  if (need > 0) {
    const cudaError_t e = cudaMemsetAsync(ws, 0, need, st);
    if (e != cudaSuccess) return set_error(MR_E_LAUNCH, "%s: cudaMemsetAsync: %s", what, cudaGetErrorString(e));
  }
  return MR_OK;
}

// Two 2-byte channels per thread (128-byte rows per warp) where D and every
// pointer allow it; float32 fills 128-byte rows with one.
static bool pairs(int64_t D, std::initializer_list<const void*> half, std::initializer_list<const void*> full) {
  bool ok = D % 2 == 0;
  for (const void* p : half) ok = ok && ((uintptr_t)p & 3u) == 0;
  for (const void* p : full) ok = ok && ((uintptr_t)p & 7u) == 0;
  return ok;
}

static int packed_check(const char* what, int dtype, int64_t T, int64_t D, int64_t S) {
  if (dtype != MR_F32 && dtype != MR_BF16 && dtype != MR_F16)
    return set_error(MR_E_DTYPE, "%s: unsupported dtype code %d (0=f32, 1=bf16, 2=f16)", what, dtype);
  if (T < 0 || D <= 0 || S < 0) return set_error(MR_E_SHAPE, "%s: T and S must not be negative, D positive", what);
  if (T > (int64_t)INT32_MAX / 2 || S > (int64_t)INT32_MAX / 2)
    return set_error(MR_E_SHAPE, "%s: T=%lld or S=%lld too large", what, (long long)T, (long long)S);
  return MR_OK;
}

template <typename T, int V>
static int fwd_launch(const void* a, const void* x, const int* cu, int64_t S, int64_t L, int64_t D, const float* h0,
                      float* y, float* ckpt, float* fin, void* ws, size_t wsb, cudaStream_t st) {
  const int ntile = (int)((D + 32 * V - 1) / (32 * V)), nchunk = (int)(L > 0 ? chunks(L) : 1);
  if (int rc = prepare_ws("mr_rglru_packed_fwd", L, D, ntile, ws, wsb, st)) return rc;
  packed_fwd_kernel<T, V><<<(unsigned)(nchunk * ntile), kWarps * 32, 0, st>>>(
      (const T*)a, (const T*)x, cu, (int)S, L, D, h0, y, ckpt, fin, nchunk > 1 ? (uint32_t*)ws : nullptr,
      (Rec*)((char*)ws + 16), nchunk, ntile);
  return check_launch("packed_fwd_kernel");
}
template <typename T, int V>
static int bwd_launch(const float* gy, const float* gf, const float* ckpt, const void* a, const void* x,
                      const int* cu, int64_t S, int64_t L, int64_t D, const float* h0, void* ga, void* gx, float* gh0,
                      void* ws, size_t wsb, cudaStream_t st) {
  const int ntile = (int)((D + 32 * V - 1) / (32 * V)), nchunk = (int)(L > 0 ? chunks(L) : 1);
  if (int rc = prepare_ws("mr_rglru_packed_bwd", L, D, ntile, ws, wsb, st)) return rc;
  packed_bwd_kernel<T, V><<<(unsigned)(nchunk * ntile), kWarps * 32, 0, st>>>(
      gy, gf, ckpt, (const T*)a, (const T*)x, cu, (int)S, L, D, h0, (T*)ga, (T*)gx, gh0,
      nchunk > 1 ? (uint32_t*)ws : nullptr, (Rec*)((char*)ws + 16), nchunk, ntile);
  return check_launch("packed_bwd_kernel");
}

int packed_device_error(bool clear) { return read_device_error(clear); }

}  // namespace mr

using namespace mr;

extern "C" {

int64_t mr_rglru_packed_chunk(void) { return kChunk; }

size_t mr_rglru_packed_workspace_bytes(int64_t T, int64_t D) { return T > 0 && D > 0 ? ws_bytes_of(T, D) : 0; }

int mr_rglru_packed_fwd(const void* a, const void* x, const int32_t* cu_seqlens, int64_t S, int dtype, int64_t T,
                        int64_t D, const float* h0, float* y, float* ckpt, float* final_state, void* ws,
                        size_t ws_bytes, void* stream) {
  const char* what = "mr_rglru_packed_fwd";
  if (int rc = packed_check(what, dtype, T, D, S)) return rc;
  if (T == 0 && S == 0) return MR_OK;
  if (cu_seqlens == nullptr || (T > 0 && (a == nullptr || x == nullptr || y == nullptr)))
    return set_error(MR_E_ALIGN, "%s: a pointer is NULL", what);
  const cudaStream_t st = (cudaStream_t)stream;
  const bool two = pairs(D, {a, x}, {y});
#define MR_CALL(T_, V_) fwd_launch<T_, V_>(a, x, cu_seqlens, S, T, D, h0, y, ckpt, final_state, ws, ws_bytes, st)
  switch (dtype) {
    case MR_F32: return MR_CALL(float, 1);
    case MR_BF16: return two ? MR_CALL(__nv_bfloat16, 2) : MR_CALL(__nv_bfloat16, 1);
    default: return two ? MR_CALL(__half, 2) : MR_CALL(__half, 1);
  }
#undef MR_CALL
}

int mr_rglru_packed_bwd(const float* grad_y, const float* grad_final, const float* ckpt, const void* a, const void* x,
                        const int32_t* cu_seqlens, int64_t S, int dtype, int64_t T, int64_t D, const float* h0,
                        void* grad_a, void* grad_x, float* grad_h0, void* ws, size_t ws_bytes, void* stream) {
  const char* what = "mr_rglru_packed_bwd";
  if (int rc = packed_check(what, dtype, T, D, S)) return rc;
  if (T == 0 && S == 0) return MR_OK;
  if (cu_seqlens == nullptr || (T > 0 && (a == nullptr || x == nullptr || grad_y == nullptr || ckpt == nullptr ||
                                          grad_a == nullptr || grad_x == nullptr)))
    return set_error(MR_E_ALIGN, "%s: a pointer is NULL", what);
  const cudaStream_t st = (cudaStream_t)stream;
  const bool two = pairs(D, {a, x, grad_a, grad_x}, {grad_y});
#define MR_CALL(T_, V_)                                                                                         \
  bwd_launch<T_, V_>(grad_y, grad_final, ckpt, a, x, cu_seqlens, S, T, D, h0, grad_a, grad_x, grad_h0, ws, ws_bytes, \
                     st)
  switch (dtype) {
    case MR_F32: return MR_CALL(float, 1);
    case MR_BF16: return two ? MR_CALL(__nv_bfloat16, 2) : MR_CALL(__nv_bfloat16, 1);
    default: return two ? MR_CALL(__half, 2) : MR_CALL(__half, 1);
  }
#undef MR_CALL
}

}  // extern "C"
