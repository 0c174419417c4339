// RG-LRU recurrence h_t = a_t h_{t-1} + x_t over a packed batch: sequences of
// any lengths (zero included) lie back to back in [T, D]; sequence s holds the
// tokens cu[s] .. cu[s+1]-1 and starts from h0[s] (zero without h0). Rows
// outside every sequence get zeros (outputs and gradients).
//
// Adjoint: adj_t = gy_t + r_t, r_{t-1} = a_t adj_t, where r starts from gf_s at
// the sequence's last token; grad_x = adj, grad_a[t] = adj_t h_{t-1},
// grad_h0[s] = r left of its first token (gf_s for an empty sequence).
//
// One pass over the data, HBM-bound. An item is kChunk steps of 32 V channels
// (rows of 128 bytes of the inputs); 8 warps x kSteps steps each work on it out
// of shared memory, where TMA copies bring it; the other CTAs of the SM (five
// forward, three backward) cover the copies and the waits. A step is the affine
// map h -> a h + x, so runs of steps compose to one map (A, B): per thread, per
// warp prefix and per item. An item publishes its map, looks back over the items
// before it in time until it meets one whose state is known, and publishes its
// own state. A sequence border cuts the chain: what follows it does not depend on
// the past. Borders are the same for all channels, so every branch on them is
// uniform. The backward runs the same scheme from the right, and rebuilds h from
// the states that the forward kept per chunk.
//
// A product of gates above one may leave float32's range where the recurrence does not
// (a state of zero under a = 2). A channel whose composed map is not finite publishes no
// map, and its state only from the item's last step; a warp whose entering state comes out
// as not finite computes it again step by step (walk_h, walk_both). Inputs that hold
// infinities or NaN pay for it too, in their channels: with NaN everywhere the two sizes
// below take 1.4 and 3.8 ms, 9.3 and 18.5 ms, since their chunks then run one after the
// other. (Products that fall below float32's smallest number count as zero: what a state
// contributes 1e38 times smaller than itself is dropped.)
//
// bf16, T=32768, D=2560, 24 sequences: forward 144 us (4.7 TB/s of the 8 bytes an
// element needs), backward 233 us (4.3 TB/s of 12 bytes); fp16, T=131072, D=512, one
// sequence: 144 and 202 us. What is left is the wait for the items before, so nothing
// delays an item that others wait for: a branch around the stores of the records instead
// of a tag that says "not there yet" takes 147 and 235 us (148 and 207). The look-back
// keeps the maps it meets and applies them in the items' order; composing them newest
// first took 138 and 224 us (128 and 186), but its bits varied with the timing, and reading
// them a second time instead of keeping them took 148 and 232 us (365 and 390). Eight maps
// kept in the forward instead of sixteen: 140 us (171), where sixteen took 140 (142).
// Measured before, beside 138 and 224 us at the first size: tickets taken a stage ahead of
// the data 182 and 304 us; a plain loop for the steps at borders 227 us; rounds of 4 (8)
// records of the look-back in place of 1: 160 and 268 us (199 and 343), since they read
// maps that are not there yet where a state is about to come.
#include "common.cuh"
#include "launch.cuh"
#include "tma.cuh"
#include "tmap.cuh"

namespace mr {

constexpr int kWarps = 8;
constexpr int kSteps = 16;               // steps of a thread
constexpr int kChunk = kWarps * kSteps;  // steps of an item

// A chunk's map or state for one channel, written and read as one 16-byte access, so no flag or fence stands beside
// it. The last word is a function of the others: a read whose words are not of one write (an assembler may narrow a
// load to the words that are used, which is then no longer one access) counts as not there yet.
struct alignas(16) Rec {
  float A, B;    // kMap: state out = A state in + B; kState: state out = B
  uint32_t tag;  // kNone: not there yet
  uint32_t sum;
};
enum : uint32_t { kNone = 0, kMap = 1, kState = 2 };

__device__ __forceinline__ void rec_store(Rec* p, float A, float B, uint32_t tag) {
  const uint32_t a = __float_as_uint(A), b = __float_as_uint(B);
  const uint64_t lo = (uint64_t)b << 32 | a, hi = (uint64_t)(a ^ b ^ tag) << 32 | tag;
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
  const uint32_t a = (uint32_t)lo, b = (uint32_t)(lo >> 32), tag = (uint32_t)hi, sum = (uint32_t)(hi >> 32);
  return {__uint_as_float(a), __uint_as_float(b), sum == (a ^ b ^ tag) ? tag : 0, sum};
}

// Polls until the record's tag is `least` at least; after 2 s (its writer is always a CTA that
// started earlier, so only a device failure gets here) sets the device error word.
__device__ __forceinline__ Rec rec_wait(const Rec* p, uint32_t least) {
  Rec r = rec_load(p);
  if (r.tag >= least) return r;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    r = rec_load(p);
    if (r.tag >= least) return r;
    if ((i & 255u) == 255u &&
        (*reinterpret_cast<volatile int*>(&g_device_error) != 0 || globaltimer_ns() - t0 > 2000000000ull))
      break;
  }
  atomicCAS(&g_device_error, 0, 1);
  return {0.f, 0.f, kState, 0};
}

// The borders of a chunk, found ahead by packed_prep_kernel (a search in cu is a
// chain of dependent loads): the first s with cu[s] >= t0, the tokens [lo, hi) of
// the chunk that lie in sequences, and a bit per warp for the steps that hold a
// sequence's start (its end).
struct alignas(16) ChunkInfo {
  int first, lo, hi;
  uint32_t starts, ends;
  int pad[3];
  // no border in warp w's steps, and all of them in a sequence: the short loops serve
  __device__ bool plain(int w) const {
    return !((starts | ends) >> w & 1) && w * kSteps >= lo && (w + 1) * kSteps <= hi;
  }
};

__device__ __forceinline__ ChunkInfo chunk_info(const int* __restrict__ cu, int S, int64_t t0, int n) {
  int l = 0, r = S;
  while (l < r) {
    const int m = (l + r) >> 1;
    if (cu[m] < t0) l = m + 1; else r = m;
  }
  ChunkInfo c = {};
  c.first = l;
  for (int s = l, next; s <= S; s = next) {  // from the first border of a run of equal ones to the next run's
    const int64_t at = cu[s] - t0;
    if (at > n) break;
    next = s + 1;
    if (next <= S && cu[next] <= cu[s])  // empty sequences, however many
      for (int r = S + 1; next < r;) {
        const int m = next + ((r - next) >> 1);
        if (cu[m] <= cu[s]) next = m + 1; else r = m;
      }
    if (at >= 0 && at < n && next <= S) c.starts |= 1u << (at / kSteps);
    if (at >= 1 && s > 0) c.ends |= 1u << ((at - 1) / kSteps);
  }
  c.lo = (int)min(max((int64_t)cu[0] - t0, (int64_t)0), (int64_t)n);
  c.hi = (int)min(max((int64_t)cu[S] - t0, (int64_t)0), (int64_t)n);
  return c;
}

// Clears the ticket counter and the records, and describes the chunks.
__global__ void __launch_bounds__(256) packed_prep_kernel(const int* __restrict__ cu, int S, int64_t L, int nchunk,
                                                          uint4* ws, ChunkInfo* info, uint4* recs, int64_t nrec) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)gridDim.x * 256;
  for (int64_t c = id; c < nchunk; c += all)
    info[c] = chunk_info(cu, S, c * kChunk, (int)min((int64_t)kChunk, L - c * kChunk));
  if (id == 0) *ws = make_uint4(0, 0, 0, 0);
  for (int64_t i = id; i < nrec; i += all) recs[i] = make_uint4(0, 0, 0, 0);
}

struct PackedArgs {
  const int* cu;
  int S, nchunk, ntile;
  int64_t L, D;
  const float *h0, *gf, *gy;
  float *y, *ckpt, *fin, *gh0;
  const void *a, *x;
  void *ga, *gx;
  uint32_t* counter;  // NULL when there is one chunk: item = blockIdx.x, no records
  const ChunkInfo* info;
  Rec* recs;
  bool vec;  // rows of V elements may be accessed whole
};

// CTAs per SM, by shared memory
template <bool BWD> constexpr int kCtas = BWD ? 3 : 5;

template <typename T> constexpr int kV = 4 / sizeof(T);  // channels of a thread: 4 bytes of an input row
template <typename T, bool BWD> constexpr int kStage = kChunk * 32 * kV<T> * (2 * (int)sizeof(T) + (BWD ? 4 : 0));

template <typename T, int V, typename P>
__device__ __forceinline__ Vec<T, V> get(const P* p, bool vec, int live) {
  Vec<T, V> r;
  if (vec && live == V) return ld_vec<T, V>(p);
#pragma unroll
  for (int v = 0; v < V; ++v) r.v[v] = v < live ? p[v] : from_f<T>(0.f);
  return r;
}
template <typename T, int V> __device__ __forceinline__ void put(T* p, const float (&f)[V], bool vec, int live) {
  if (vec && live == V) {
    if constexpr (sizeof(T) == 4) st_stream_f32<V>(p, f);
    else st_vec<T, V>(p, f);
    return;
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (v < live) p[v] = from_f<T>(f[v]);
}

// What a CTA keeps in shared memory beside the stages.
template <int V, bool BWD> struct Work {
  static constexpr int kKept = BWD ? kWarps : 2 * kWarps;
  float map[kKept][2][32 * V];              // the warps' maps A, B along the chain; then the look-back's, newest first
  float fmap[BWD ? kWarps : 1][2][32 * V];  // backward: the warps' maps of the forward recurrence
  float carry[32 * V];                           // the state entering the item
  int mark[kChunk];                              // per token at a border: its sequence, and which end of it
  uint64_t full;
  ChunkInfo info;
  int item;
};
constexpr int kStart = 1 << 30, kEnd = INT32_MIN, kSeq = kStart - 1;  // of Work::mark; 0 in both bits: no border

// The items of a CTA, in the order of the tickets. Tickets follow the order in
// which CTAs ask, so whatever an item waits for has been taken by a running CTA,
// which works through its items in order: the smallest one never waits.
//
// TMA form: thread 0 takes a ticket and issues the copies once the last item has
// been read (not before: an item taken early and left waiting holds up those
// behind it). Plain form (rows that are no multiple of 16 bytes): every thread brings its own
// elements.
template <typename T, bool BWD, bool TMA> struct Feed {
  static constexpr int V = kV<T>, CH = 32 * V;
  unsigned char* stage;
  Work<V, BWD>& sh;
  const PackedArgs& P;
  const CUtensorMap *ta, *tx, *tg;
  int n = 0;  // items so far

  __device__ T* a() const { return reinterpret_cast<T*>(stage); }
  __device__ T* x() const { return a() + kChunk * CH; }
  __device__ float* g() const { return reinterpret_cast<float*>(x() + kChunk * CH); }
  __device__ int64_t chunk_of(int item) const { return BWD ? P.nchunk - 1 - item / P.ntile : item / P.ntile; }

  // The next item, once its data is there, or -1.
  __device__ int next() {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if constexpr (TMA) {
      if (threadIdx.x == 0) {
        const int next = P.counter ? (int)min(atomicAdd(P.counter, 1u), (uint32_t)INT32_MAX)
                                   : (n == 0 ? (int)blockIdx.x : INT32_MAX);
        const bool more = next < P.nchunk * P.ntile;
        sh.item = more ? next : -1;
        if (more) {
          const int64_t chunk = chunk_of(next), t0 = chunk * kChunk;
          const int c0 = next % P.ntile * CH;
          sh.info = P.info ? P.info[chunk] : chunk_info(P.cu, P.S, t0, (int)min((int64_t)kChunk, P.L - t0));
          mbar_arrive_expect_tx(&sh.full, kStage<T, BWD>);
          tma_load_2d(a(), ta, c0, (int)t0, &sh.full);
          tma_load_2d(x(), tx, c0, (int)t0, &sh.full);
          if (BWD) tma_load_2d(g(), tg, c0, (int)t0, &sh.full);
        } else {
          mbar_arrive(&sh.full);
        }
      }
      mbar_wait(&sh.full, n++ & 1);
      return sh.item;
    } else {
      if (P.counter == nullptr) {
        if (n++ > 0) return -1;
        sh.item = blockIdx.x;
      } else {
        __syncthreads();  // everybody has read the last item's number
        if (threadIdx.x == 0) sh.item = (int)min(atomicAdd(P.counter, 1u), (uint32_t)INT32_MAX);
      }
      __syncthreads();
      const int item = sh.item;
      if (item >= P.nchunk * P.ntile) return -1;
      const int64_t t0 = chunk_of(item) * kChunk, ch = (int64_t)(item % P.ntile) * CH + lane * V;
      const int live = (int)min((int64_t)V, max((int64_t)0, P.D - ch)), rows = (int)min((int64_t)kChunk, P.L - t0);
      Vec<T, V> va[kSteps], vx[kSteps];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int i = w * kSteps + k;
        const int64_t at = (t0 + i) * P.D + ch;
        va[k] = get<T, V>((const T*)P.a + at, P.vec, i < rows ? live : 0);
        vx[k] = get<T, V>((const T*)P.x + at, P.vec, i < rows ? live : 0);
      }
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int i = (w * kSteps + k) * CH + lane * V;
        *reinterpret_cast<Vec<T, V>*>(a() + i) = va[k];
        *reinterpret_cast<Vec<T, V>*>(x() + i) = vx[k];
      }
      if constexpr (BWD) {
        Vec<float, V> vg[kSteps];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const int i = w * kSteps + k;
          vg[k] = get<float, V>(P.gy + (t0 + i) * P.D + ch, P.vec, i < rows ? live : 0);
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
          *reinterpret_cast<Vec<float, V>*>(g() + (w * kSteps + k) * CH + lane * V) = vg[k];
      }
      return item;
    }
  }
};

// Marks of a chunk that holds borders; all threads call it. A token belongs to
// one sequence, so one entry serves its start and its end.
template <int V, bool BWD>
__device__ __forceinline__ void mark_borders(Work<V, BWD>& sh, const ChunkInfo& c, const PackedArgs& P, int64_t t0, int n) {
  if (threadIdx.x < kChunk) sh.mark[threadIdx.x] = 0;
  __syncthreads();
  for (int s = c.first + threadIdx.x; s <= P.S; s += kWarps * 32) {
    const int64_t at = P.cu[s] - t0;
    if (at > n) break;
    if (at >= 0 && at < n && s < P.S && P.cu[s + 1] > P.cu[s]) atomicOr(&sh.mark[at], s | kStart);
    if (at >= 1 && s > 0 && P.cu[s] > P.cu[s - 1]) atomicOr(&sh.mark[at - 1], (s - 1) | kEnd);
  }
  __syncthreads();
}

// A warp's steps as bit masks: in a sequence, at a start, at an end; the same in every lane, so the unrolled loops branch
// on them without divergence.
struct StepMasks {
  uint32_t in, start, end;
};
__device__ __forceinline__ StepMasks step_masks(const int* mark, const ChunkInfo& c, int w) {
  const int lane = threadIdx.x & 31, k0 = w * kSteps;
  const int m = lane < kSteps && (c.starts | c.ends) ? mark[k0 + lane] : 0;
  const int lo = max(c.lo - k0, 0), hi = min(c.hi - k0, kSteps);
  const uint32_t in = hi > lo ? ((1u << hi) - 1) & ~((1u << lo) - 1) : 0;
  return {in, __ballot_sync(0xffffffffu, m & kStart) & in, __ballot_sync(0xffffffffu, m & kEnd) & in};
}

// The sequence of a marked token (clamped, so that a malformed cu stays in range).
__device__ __forceinline__ int seq_at(const int* mark, int i, int S) { return min(mark[i] & kSeq, S - 1); }
// v <- the V channels of row s of a [S, D] state, or zeros without one
template <int V> __device__ __forceinline__ void begin(const float* state, int s, int64_t D, int64_t ch, int live, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = state && i < live ? state[s * D + ch + i] : 0.f;
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

// What enters this warp's steps, where the composed maps gave something that is not finite: through the steps of the
// warps before it, one by one. From the left out of shared memory; from the right with gy from global memory (in
// shared memory adj takes its place), eight steps ahead. All channels of the lane in one call that finds its data in
// sh, P and the stages, so that the call costs those that do not make it little.
template <int V> struct Lane {
  float v[V];
};
template <typename T, int V, bool BWD>
__device__ __noinline__ Lane<V> walk_h(const Work<V, BWD>& sh, const PackedArgs& P, const unsigned char* stage, Lane<V> from, Lane<V> got) {
  constexpr int CH = 32 * V;
  const int c = (threadIdx.x & 31) * V, end = min(sh.info.hi, (int)(threadIdx.x >> 5) * kSteps);
  const T *a = reinterpret_cast<const T*>(stage) + c, *x = a + kChunk * CH;
  const int64_t ch = (int64_t)(sh.item % P.ntile) * CH + c;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (finite(got.v[v]) || ch + v >= P.D) continue;
    float h = from.v[v];
    for (int k = sh.info.lo; k < end; ++k) {
      if (sh.info.starts != 0 && (sh.mark[k] & kStart)) h = P.h0 ? P.h0[seq_at(sh.mark, k, P.S) * P.D + ch + v] : 0.f;
      h = fmaf(to_f(a[k * CH + v]), h, to_f(x[k * CH + v]));
    }
    got.v[v] = h;
  }
  return got;
}
template <int V> struct Both {
  Lane<V> h, r;
};
template <typename T, int V>
__device__ __noinline__ Both<V> walk_both(const Work<V, true>& sh, const PackedArgs& P, const unsigned char* stage, Lane<V> carry, Lane<V> h, Lane<V> r) {
  constexpr int CH = 32 * V;
  const int c = (threadIdx.x & 31) * V, beg = max(sh.info.lo, (int)(threadIdx.x >> 5) * kSteps + kSteps);
  const T* a = reinterpret_cast<const T*>(stage) + c;
  const int64_t ch = (int64_t)(sh.item % P.ntile) * CH + c, chunk = P.nchunk - 1 - sh.item / P.ntile;
  Lane<V> ckpt = {};
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (ch + v >= P.D) continue;
    ckpt.v[v] = P.ckpt[chunk * P.D + ch + v];
    if (finite(r.v[v])) continue;
    const float* gy = P.gy + chunk * kChunk * P.D + ch + v;
    float s = carry.v[v];
    for (int k0 = sh.info.hi; k0 > beg; k0 -= 8) {
      float g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = gy[max(k0 - 1 - i, beg) * P.D];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = k0 - 1 - i;
        if (k < beg) break;
        if (sh.info.ends != 0 && (sh.mark[k] & kEnd)) s = P.gf ? P.gf[seq_at(sh.mark, k, P.S) * P.D + ch + v] : 0.f;
        s = to_f(a[k * CH + v]) * (g[i] + s);
      }
    }
    r.v[v] = s;
  }
  return {walk_h<T, V, true>(sh, P, stage, ckpt, h), r};
}

// The chain. Along it (left to right in the forward, right to left in the
// backward) item `rank` of a channel tile follows rank - 1. Composes the warps'
// maps in sh.map (bit w of `cut`: warp w's steps hold a border, so its
// outgoing state is B whatever enters), publishes this item's record, and returns
// in p, q the map from the state entering the item to the one entering this warp
// and in carry the former. `need`: whether anything in the item depends on it.
//
// The look-back goes to the nearest item whose state is there and applies the maps
// on the way in the items' order, with the fmaf that the items themselves apply:
// the bits do not depend on how far the others have come. Maps wait in the place of
// sh.map, which every warp has read by then; behind kKept of them a state is waited for.
//
// The chain's last warp does it, which composes the whole item on its way and ends in
// the state that the item hands on. A map or state that is not finite is published as not
// there yet (a store without a branch: the others wait for it): for these channels (bits of
// `late`, in that warp) publish_late does it.
template <int V, bool BWD>
__device__ __forceinline__ void chain(Work<V, BWD>& sh, const PackedArgs& P, int64_t ch, int live, int rank, uint32_t cut,
                                      bool need, float (&carry)[V], float (&p)[V], float (&q)[V], uint32_t& late) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = lane * V;
  constexpr int kLast = BWD ? 0 : kWarps - 1;
  const bool wait = need && rank > 0, tell = P.counter != nullptr && rank < P.nchunk - 1;
  Rec* recs = P.recs + ch;
  float tp[V], tq[V];  // the last warp: the item's own map
  auto through = [&](int i, const float(&p)[V], const float(&q)[V], float(&op)[V], float(&oq)[V]) {  // and warp i's map
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float A = sh.map[i][0][c + v], B = sh.map[i][1][c + v];
      oq[v] = cut >> i & 1 ? B : fmaf(A, q[v], B);
      op[v] = cut >> i & 1 ? 0.f : p[v] * A;
    }
  };
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] = 1.f, q[v] = 0.f;
  late = 0;
  if (w == kLast) {
#pragma unroll
    for (int i = 0; i < kWarps - 1; ++i) through(BWD ? kWarps - 1 - i : i, p, q, p, q);
    through(kLast, p, q, tp, tq);
    if (tell) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const bool state = cut || !wait, good = finite(tq[v]) && (state || finite(tp[v]));
        if (v < live) rec_store(recs + rank * P.D + v, tp[v], tq[v], !good ? kNone : state ? kState : kMap);
        late |= (good ? 0u : 1u) << v;
      }
    }
  } else {
    if (BWD)
      for (int i = kWarps - 1; i > w; --i) through(i, p, q, p, q);
    else
      for (int i = 0; i < w; ++i) through(i, p, q, p, q);
  }
  if (wait) {
    __syncthreads();
    if (w == kLast) {
      float b[V];
      for (int keep = Work<V, BWD>::kKept;; keep = 0) {
        int kept[V];  // maps between this item and the one whose state is b
        bool known[V];
#pragma unroll
        for (int v = 0; v < V; ++v) b[v] = 0.f, kept[v] = 0, known[v] = v >= live;
        int n = 0;
        for (bool open = live > 0; open; ++n) {
          const int at = rank - 1 - n;  // (item 0 always has a state)
          const uint32_t least = n == keep || at == 0 ? kState : kMap;
          Rec r[V];
#pragma unroll
          for (int v = 0; v < V; ++v) r[v] = known[v] ? Rec{0.f, 0.f, kState, 0} : rec_load(recs + at * P.D + v);
          open = false;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            if (known[v]) continue;
            if (r[v].tag < least) r[v] = rec_wait(recs + at * P.D + v, least);
            if (r[v].tag == kState) {
              b[v] = r[v].B, kept[v] = n, known[v] = true;
            } else {
              sh.map[n][0][c + v] = r[v].A, sh.map[n][1][c + v] = r[v].B;
              open = true;
            }
          }
        }
#pragma unroll 4
        for (--n; n >= 0; --n)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float A = sh.map[n][0][c + v], B = sh.map[n][1][c + v];
            if (n < kept[v]) b[v] = fmaf(A, b[v], B);
          }
        bool good = true;
#pragma unroll
        for (int v = 0; v < V; ++v) good &= finite(b[v]);
        if (good || keep == 0) break;  // once not finite, always: then what the item before ended in decides
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        sh.carry[c + v] = b[v];
        const float out = fmaf(tp[v], b[v], tq[v]);
        if (tell && !cut) {
          if (v < live) rec_store(recs + rank * P.D + v, 0.f, out, finite(out) ? kState : kNone);
          late = (late & ~(1u << v)) | (finite(out) ? 0u : 1u) << v;
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int v = 0; v < V; ++v) carry[v] = wait ? sh.carry[c + v] : 0.f;
}

template <int V>
__device__ __forceinline__ void publish_late(const PackedArgs& P, int64_t ch, int live, int rank, uint32_t late, const float (&out)[V]) {
  if (late == 0) return;
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (v < live && (late >> v & 1)) rec_store(P.recs + ch + rank * P.D + v, 0.f, out[v], kState);
}

// state entering the warp, from the one entering the item; a cut leaves p = 0 and q alone (0 x infinity would not)
__device__ __forceinline__ float enter(float p, float q, float carry, bool cut) { return cut ? q : fmaf(p, carry, q); }

template <typename T, bool TMA>
__global__ void __launch_bounds__(kWarps * 32, kCtas<false>)
packed_fwd_kernel(const __grid_constant__ PackedArgs P, const __grid_constant__ CUtensorMap ta,
                  const __grid_constant__ CUtensorMap tx) {
  constexpr int V = kV<T>, CH = 32 * V;
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ Work<V, false> sh;
  Feed<T, false, TMA> feed{dyn, sh, P, &ta, &tx, nullptr};
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, k0 = w * kSteps;
  if constexpr (TMA) {
    if (threadIdx.x == 0) {
      mbar_init(&sh.full, 1);
      fence_mbar_init();
    }
    __syncthreads();
  }
  for (int item; (item = feed.next()) >= 0;) {
    const int chunk = item / P.ntile;
    const int64_t ch = (int64_t)(item % P.ntile) * CH + lane * V, t0 = (int64_t)chunk * kChunk;
    const int n = (int)min((int64_t)kChunk, P.L - t0), live = (int)min((int64_t)V, max((int64_t)0, P.D - ch));
    const ChunkInfo info = TMA ? sh.info : P.info ? P.info[chunk] : chunk_info(P.cu, P.S, t0, n);
    if (!TMA && threadIdx.x == 0) sh.info = info;
    if (info.starts | info.ends) mark_borders(sh, info, P, t0, n);
    const bool plain = info.plain(w);
    const StepMasks mask = step_masks(sh.mark, info, w);
    const T *sa = feed.a() + k0 * CH + lane * V, *sx = feed.x() + k0 * CH + lane * V;
    float A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
    if (plain) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const Vec<T, V> av = ld_vec<T, V>(sa + k * CH), xv = ld_vec<T, V>(sx + k * CH);
#pragma unroll
        for (int v = 0; v < V; ++v) B[v] = fmaf(to_f(av.v[v]), B[v], to_f(xv.v[v])), A[v] *= to_f(av.v[v]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        if (!(mask.in >> k & 1)) continue;
        if (mask.start >> k & 1) begin(P.h0, seq_at(sh.mark, k0 + k, P.S), P.D, ch, live, B);
#pragma unroll
        for (int v = 0; v < V; ++v)
          B[v] = fmaf(to_f(sa[k * CH + v]), B[v], to_f(sx[k * CH + v])), A[v] *= to_f(sa[k * CH + v]);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) sh.map[w][0][lane * V + v] = A[v], sh.map[w][1][lane * V + v] = B[v];
    __syncthreads();
    const bool need = info.lo == 0 && info.hi > 0 && !(info.starts && (sh.mark[0] & kStart));
    float carry[V], p[V], q[V], h[V];
    uint32_t late;
    chain<V, false>(sh, P, ch, live, chunk, info.starts, need, carry, p, q, late);
    const bool cut = info.starts & ((1u << w) - 1);
    bool good = true;
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = enter(p[v], q[v], carry[v], cut), good &= finite(h[v]);
    if (!good) {
      Lane<V> from, got;
#pragma unroll
      for (int v = 0; v < V; ++v) from.v[v] = carry[v], got.v[v] = h[v];
      got = walk_h<T>(sh, P, dyn, from, got);
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = got.v[v];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (P.ckpt != nullptr && w == 0 && v < live && n > 0) P.ckpt[chunk * P.D + ch + v] = h[v];
    }
    float* y = P.y + (t0 + k0) * P.D + ch;
    if (plain) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k, y += P.D) {
        const Vec<T, V> av = ld_vec<T, V>(sa + k * CH), xv = ld_vec<T, V>(sx + k * CH);
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = fmaf(to_f(av.v[v]), h[v], to_f(xv.v[v]));
        put<float, V>(y, h, P.vec, live);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kSteps; ++k, y += P.D) {
        if (k0 + k >= n) continue;
        const bool in = mask.in >> k & 1;
        float out[V];
        if (mask.start >> k & 1) begin(P.h0, seq_at(sh.mark, k0 + k, P.S), P.D, ch, live, h);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (in) h[v] = fmaf(to_f(sa[k * CH + v]), h[v], to_f(sx[k * CH + v]));
          out[v] = in ? h[v] : 0.f;
        }
        if (P.fin != nullptr && (mask.end >> k & 1)) {
          const int64_t at = (int64_t)seq_at(sh.mark, k0 + k, P.S) * P.D + ch;
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (v < live) P.fin[at + v] = h[v];
        }
        put<float, V>(y, out, P.vec, live);
      }
    }
    publish_late(P, ch, live, chunk, late, h);
    if (P.fin != nullptr)  // empty sequences, spread over the chunks
      for (int s = (int)((int64_t)chunk * P.S / P.nchunk) + w; s < (int)((int64_t)(chunk + 1) * P.S / P.nchunk); s += kWarps)
        if (P.cu[s + 1] <= P.cu[s])
          for (int v = 0; v < live; ++v) P.fin[s * P.D + ch + v] = P.h0 ? P.h0[s * P.D + ch + v] : 0.f;
    __syncthreads();  // sh is free for the next item
  }
}

template <typename T, bool TMA>
__global__ void __launch_bounds__(kWarps * 32, kCtas<true>)
packed_bwd_kernel(const __grid_constant__ PackedArgs P, const __grid_constant__ CUtensorMap ta,
                  const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tg) {
  constexpr int V = kV<T>, CH = 32 * V;
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ Work<V, true> sh;
  Feed<T, true, TMA> feed{dyn, sh, P, &ta, &tx, &tg};
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, k0 = w * kSteps;
  if constexpr (TMA) {
    if (threadIdx.x == 0) {
      mbar_init(&sh.full, 1);
      fence_mbar_init();
    }
    __syncthreads();
  }
  for (int item; (item = feed.next()) >= 0;) {
    const int rank = item / P.ntile, chunk = P.nchunk - 1 - rank;
    const int64_t ch = (int64_t)(item % P.ntile) * CH + lane * V, t0 = (int64_t)chunk * kChunk;
    const int n = (int)min((int64_t)kChunk, P.L - t0), live = (int)min((int64_t)V, max((int64_t)0, P.D - ch));
    const ChunkInfo info = TMA ? sh.info : P.info ? P.info[chunk] : chunk_info(P.cu, P.S, t0, n);
    if (!TMA && threadIdx.x == 0) sh.info = info;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = v < live && n > 0 ? P.ckpt[chunk * P.D + ch + v] : 0.f;
    if (info.starts | info.ends) mark_borders(sh, info, P, t0, n);
    const bool plain = info.plain(w);
    const StepMasks mask = step_masks(sh.mark, info, w);
    const T *sa = feed.a() + k0 * CH + lane * V, *sx = feed.x() + k0 * CH + lane * V;
    float* sg = feed.g() + k0 * CH + lane * V;
    {
      float A[V], B[V], C[V], Q[V];
#pragma unroll
      for (int v = 0; v < V; ++v) A[v] = C[v] = 1.f, B[v] = Q[v] = 0.f;
      if (plain) {
        // h forward, and r backward as sum of (product of the gates so far) x gy: Q = sum_k (a_0 .. a_k) gy_k
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const Vec<T, V> av = ld_vec<T, V>(sa + k * CH), xv = ld_vec<T, V>(sx + k * CH);
          const Vec<float, V> gv = ld_vec<float, V>(sg + k * CH);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            B[v] = fmaf(to_f(av.v[v]), B[v], to_f(xv.v[v]));
            A[v] *= to_f(av.v[v]);
            Q[v] = fmaf(A[v], gv.v[v], Q[v]);
          }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) C[v] = A[v];
      } else {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          if (!(mask.in >> k & 1)) continue;
          if (mask.start >> k & 1) begin(P.h0, seq_at(sh.mark, k0 + k, P.S), P.D, ch, live, B);
#pragma unroll
          for (int v = 0; v < V; ++v)
            B[v] = fmaf(to_f(sa[k * CH + v]), B[v], to_f(sx[k * CH + v])), A[v] *= to_f(sa[k * CH + v]);
        }
#pragma unroll
        for (int k = kSteps - 1; k >= 0; --k) {
          if (!(mask.in >> k & 1)) continue;
          if (mask.end >> k & 1) begin(P.gf, seq_at(sh.mark, k0 + k, P.S), P.D, ch, live, Q);
#pragma unroll
          for (int v = 0; v < V; ++v)
            Q[v] = to_f(sa[k * CH + v]) * (sg[k * CH + v] + Q[v]), C[v] *= to_f(sa[k * CH + v]);
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        sh.fmap[w][0][lane * V + v] = A[v], sh.fmap[w][1][lane * V + v] = B[v];
        sh.map[w][0][lane * V + v] = C[v], sh.map[w][1][lane * V + v] = Q[v];
      }
    }
    __syncthreads();
    const bool need = info.hi == n && info.hi > info.lo && !(info.ends && (sh.mark[n - 1] & kEnd));
    float carry[V], p[V], q[V], r[V];
    uint32_t late;
    chain<V, true>(sh, P, ch, live, rank, info.ends, need, carry, p, q, late);
    const bool cut = info.ends >> (w + 1);
    bool good = true;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      r[v] = enter(p[v], q[v], carry[v], cut);
      for (int i = 0; i < w; ++i) {
        const float A = sh.fmap[i][0][lane * V + v], B = sh.fmap[i][1][lane * V + v];
        h[v] = info.starts >> i & 1 ? B : fmaf(A, h[v], B);
      }
      good &= finite(r[v]) && finite(h[v]);
    }
    if (!good) {
      Lane<V> from;
      Both<V> got;
#pragma unroll
      for (int v = 0; v < V; ++v) from.v[v] = carry[v], got.h.v[v] = h[v], got.r.v[v] = r[v];
      got = walk_both<T>(sh, P, dyn, from, got.h, got.r);
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = got.h.v[v], r[v] = got.r.v[v];
    }
    T *ga = (T*)P.ga + (t0 + k0) * P.D + ch, *gx = (T*)P.gx + (t0 + k0) * P.D + ch;
    if (plain) {
      // right to left, adj over gy in shared memory; then left to right with h
#pragma unroll
      for (int k = kSteps - 1; k >= 0; --k) {
        const Vec<T, V> av = ld_vec<T, V>(sa + k * CH);
        Vec<float, V> gv = ld_vec<float, V>(sg + k * CH);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          gv.v[v] += r[v];
          r[v] = to_f(av.v[v]) * gv.v[v];
        }
        *reinterpret_cast<Vec<float, V>*>(sg + k * CH) = gv;
      }
      publish_late(P, ch, live, rank, late, r);
#pragma unroll
      for (int k = 0; k < kSteps; ++k, ga += P.D, gx += P.D) {
        const Vec<T, V> av = ld_vec<T, V>(sa + k * CH), xv = ld_vec<T, V>(sx + k * CH);
        const Vec<float, V> gv = ld_vec<float, V>(sg + k * CH);
        float oa[V], ox[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          ox[v] = gv.v[v];
          oa[v] = gv.v[v] * h[v];
          h[v] = fmaf(to_f(av.v[v]), h[v], to_f(xv.v[v]));
        }
        put<T, V>(ga, oa, P.vec, live);
        put<T, V>(gx, ox, P.vec, live);
      }
    } else {
#pragma unroll
      for (int k = kSteps - 1; k >= 0; --k) {
        if (!(mask.in >> k & 1)) continue;
        if (mask.end >> k & 1) begin(P.gf, seq_at(sh.mark, k0 + k, P.S), P.D, ch, live, r);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float adj = sg[k * CH + v] + r[v];
          sg[k * CH + v] = adj;
          r[v] = to_f(sa[k * CH + v]) * adj;
        }
        if (P.gh0 != nullptr && (mask.start >> k & 1)) {
          const int64_t at = (int64_t)seq_at(sh.mark, k0 + k, P.S) * P.D + ch;
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (v < live) P.gh0[at + v] = r[v];
        }
      }
      publish_late(P, ch, live, rank, late, r);
#pragma unroll
      for (int k = 0; k < kSteps; ++k, ga += P.D, gx += P.D) {
        if (k0 + k >= n) continue;
        const bool in = mask.in >> k & 1;
        float oa[V], ox[V];
        if (mask.start >> k & 1) begin(P.h0, seq_at(sh.mark, k0 + k, P.S), P.D, ch, live, h);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          ox[v] = in ? sg[k * CH + v] : 0.f;
          oa[v] = in ? sg[k * CH + v] * h[v] : 0.f;
          if (in) h[v] = fmaf(to_f(sa[k * CH + v]), h[v], to_f(sx[k * CH + v]));
        }
        put<T, V>(ga, oa, P.vec, live);
        put<T, V>(gx, ox, P.vec, live);
      }
    }
    if constexpr (TMA) fence_proxy_async_smem();  // this thread's writes over gy before the next copy into it
    if (P.gh0 != nullptr)
      for (int s = (int)((int64_t)chunk * P.S / P.nchunk) + w; s < (int)((int64_t)(chunk + 1) * P.S / P.nchunk); s += kWarps)
        if (P.cu[s + 1] <= P.cu[s])
          for (int v = 0; v < live; ++v) P.gh0[s * P.D + ch + v] = P.gf ? P.gf[s * P.D + ch + v] : 0.f;
    __syncthreads();
  }
}

static int64_t chunks(int64_t T) { return (T + kChunk - 1) / kChunk; }
static size_t ws_bytes_of(int64_t T, int64_t D) {
  // a ticket counter, the chunks' borders, and a record per chunk and channel; one chunk needs none
  return chunks(T) > 1 ? 32 + (size_t)chunks(T) * (sizeof(ChunkInfo) + D * sizeof(Rec)) : 0;
}

static int packed_check(const char* what, int dtype, int64_t T, int64_t D, int64_t S) {
  if (dtype != MR_F32 && dtype != MR_BF16 && dtype != MR_F16)
    return set_error(MR_E_DTYPE, "%s: unsupported dtype code %d (0=f32, 1=bf16, 2=f16)", what, dtype);
  if (T < 0 || D <= 0 || S < 0) return set_error(MR_E_SHAPE, "%s: T and S must not be negative, D positive", what);
  if (T > (int64_t)INT32_MAX / 2 || S > (int64_t)INT32_MAX / 2 || D > (int64_t)INT32_MAX / 2)
    return set_error(MR_E_SHAPE, "%s: T=%lld, S=%lld or D=%lld too large", what, (long long)T, (long long)S, (long long)D);
  return MR_OK;
}

static int prepare_ws(const char* what, PackedArgs& P, void* ws, size_t bytes, cudaStream_t st) {
  const size_t need = ws_bytes_of(P.L, P.D);
  if (need > 0 && (ws == nullptr || bytes < need || ((uintptr_t)ws & 15u)))
    return set_error(MR_E_WORKSPACE, "%s: needs %zu bytes of 16-byte aligned workspace, got %zu", what, need, bytes);
  if (chunks(P.L) * (int64_t)P.ntile > INT32_MAX / 2) return set_error(MR_E_SHAPE, "%s: T * D too large", what);
  if (need == 0) return MR_OK;
  P.counter = (uint32_t*)ws;
  ChunkInfo* info = (ChunkInfo*)((char*)ws + 32);
  P.info = info;
  P.recs = (Rec*)(info + P.nchunk);
  const int64_t nrec = P.nchunk * P.D, blocks = (nrec + 1023) / 1024;
  packed_prep_kernel<<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, st>>>(
      P.cu, P.S, P.L, P.nchunk, (uint4*)ws, info, (uint4*)P.recs, nrec);
  return check_launch("packed_prep_kernel");
}

template <typename T, bool BWD> static int launch(const char* what, PackedArgs P, void* ws, size_t wsb, cudaStream_t st) {
  constexpr int V = kV<T>, e = sizeof(T);
  P.ntile = (int)((P.D + 32 * V - 1) / (32 * V));
  P.nchunk = (int)(P.L > 0 ? chunks(P.L) : 1);
  if (int rc = prepare_ws(what, P, ws, wsb, st)) return rc;
  auto at = [](const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; };
  P.vec = P.D % V == 0 && (BWD ? at(P.ga, 4) && at(P.gx, 4) && at(P.gy, 4 * V) : at(P.y, 4 * V)) && at(P.a, 4) && at(P.x, 4);
  // the copies take rows that are multiples of 16 bytes, 16-byte aligned
  const bool tma = P.L > 0 && P.D * e % 16 == 0 && at(P.a, 16) && at(P.x, 16) && (!BWD || at(P.gy, 16));
  const int64_t items = (int64_t)P.nchunk * P.ntile;
  const unsigned grid = (unsigned)(P.counter && items > 148 * kCtas<BWD> ? 148 * kCtas<BWD> : items);
  constexpr int smem = kStage<T, BWD>;
  CUtensorMap ta, tx, tg;
  if (tma) {
    if (int rc = make_tmap_2d(&ta, P.a, TmapType<T>::v, e, P.D, P.L, P.D * e, 32 * V, kChunk)) return rc;
    if (int rc = make_tmap_2d(&tx, P.x, TmapType<T>::v, e, P.D, P.L, P.D * e, 32 * V, kChunk)) return rc;
    if (BWD)
      if (int rc = make_tmap_2d(&tg, P.gy, TmapType<float>::v, 4, P.D, P.L, P.D * 4, 32 * V, kChunk)) return rc;
  }
  // (one instantiation each: the shared memory is the same for every call of it)
#define MR_GO(KERNEL, THREADS, ...)                                \
  do {                                                             \
    if (int rc = allow_smem<KERNEL>(smem, what)) return rc;        \
    KERNEL<<<grid, THREADS, smem, st>>>(P, __VA_ARGS__);           \
    return check_launch(what);                                     \
  } while (0)
  if constexpr (BWD) {
    if (tma) MR_GO((packed_bwd_kernel<T, true>), kWarps * 32, ta, tx, tg);
    MR_GO((packed_bwd_kernel<T, false>), kWarps * 32, ta, tx, tg);
  } else {
    if (tma) MR_GO((packed_fwd_kernel<T, true>), kWarps * 32, ta, tx);
    MR_GO((packed_fwd_kernel<T, false>), kWarps * 32, ta, tx);
  }
#undef MR_GO
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
  PackedArgs P{};
  P.cu = cu_seqlens, P.S = (int)S, P.L = T, P.D = D, P.h0 = h0, P.y = y, P.ckpt = ckpt, P.fin = final_state;
  P.a = a, P.x = x;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case MR_F32: return launch<float, false>(what, P, ws, ws_bytes, st);
    case MR_BF16: return launch<__nv_bfloat16, false>(what, P, ws, ws_bytes, st);
    default: return launch<__half, false>(what, P, ws, ws_bytes, st);
  }
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
  PackedArgs P{};
  P.cu = cu_seqlens, P.S = (int)S, P.L = T, P.D = D, P.h0 = h0, P.gy = grad_y, P.gf = grad_final;
  P.ckpt = const_cast<float*>(ckpt), P.gh0 = grad_h0, P.a = a, P.x = x, P.ga = grad_a, P.gx = grad_x;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case MR_F32: return launch<float, true>(what, P, ws, ws_bytes, st);
    case MR_BF16: return launch<__nv_bfloat16, true>(what, P, ws, ws_bytes, st);
    default: return launch<__half, true>(what, P, ws, ws_bytes, st);
  }
}

}  // extern "C"
