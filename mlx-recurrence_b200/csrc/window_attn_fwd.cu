// Sliding-window attention with sinks, forward, on the tensor cores (tcgen05):
// bf16 and fp16, Dh <= 128.
//
// A CTA takes 128 queries of one head and walks the keys they may see in tiles
// of 128: S = Q K^T into TMEM, the online softmax by four warps (one thread per
// query, so no reduction across threads), P back into TMEM as the A operand of
// O += P V. The row's maximum is only moved when it grows by more than 2^8 (the
// factor cancels in O / l), so O is rarely rescaled. P is rounded to the inputs'
// type, which the product takes; l sums it unrounded. Where TMEM has room for P
// beside S (Dh <= 64) the next S runs under this tile's exponentials. Two CTAs per
// SM (256 TMEM columns and at most 96 KB of shared memory each) fill each other's
// gaps; the issuing warpgroup gives its registers to the softmax's, which holds a
// row of S.
//
// For a backward pass it also writes what the rounding of y drops (y_low), so that
// delta = gy.y is of float32 quality.
//
// bf16, 16384 tokens, 32 heads of 64, window 1024: 259 us (497 TFLOP/s), 273 with
// y_low; 16 heads of 128 on 4, window 2048, 4 sinks: 248 us (597), 272 with y_low.
// Bound by the chain of a tile (load S, maximum, exponentials, on two warps per
// scheduler), not by one pipe: a tile's exponentials alone would take 1,024 cycles,
// its products 500 or 1,000, a tile takes about 1,800. Measured and not kept (at 297
// us, before whole tiles had loops without bounds): two threads per query 304 us, a
// quarter of the exponentials by a polynomial on the FMA pipe 299 us, the issuing
// done by a softmax warp 352 us.
#include "window_tc.cuh"

namespace mr {

constexpr int kFwdThreads = 256;  // a warpgroup for the softmax, one (a single busy warp) that issues
constexpr float kRescale = 8.f;
// Registers a thread: at launch, and after the issuing warpgroup has passed its own on (128 threads each).
constexpr int kFwdRegs = 128, kIssueRegs = 40, kSoftmaxRegs = 2 * kFwdRegs - kIssueRegs;

struct FwdShared {
  uint64_t k_full, v_full, s_done, s_read, p_ready, o_done;
  uint32_t tmem;
  int lo_max;  // the largest first key of the tile's queries
};

template <typename T, int NB>  // NB = 64-wide blocks of a row
__global__ void __launch_bounds__(kFwdThreads, 2)
attn_fwd_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ CUtensorMap tq,
                const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv) {
  // TMEM columns: S at 0; P over its first half or, where O leaves room, in columns of its own
  constexpr bool kOwnP = NB == 1;
  constexpr uint32_t kP = kOwnP ? 128 : 0, kO = kOwnP ? 192 : 128;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  unsigned char *sQ = sm, *sK = sQ + NB * kTileBytes, *sV = sK + NB * kTileBytes;
  __shared__ FwdShared sh;
  const int tid = threadIdx.x, w = tid >> 5;
  const int h = blockIdx.y, hk = h / (A.Hq / A.Hkv), q0 = blockIdx.x * 128, i = q0 + tid;
  const KeyRange R = keys_of(A, q0, q0 + 128);
  const int nsink = R.send > R.s0 ? 1 : 0;  // at most 64 sinks: one tile
  const int ntile = R.kend > R.kmin ? nsink + (R.kend - R.kmin + 127) / 128 : 0;
  T* y = (T*)A.y + ((int64_t)i * A.Hq + h) * A.Dh;
  T* low = A.y_low ? (T*)A.y_low + ((int64_t)i * A.Hq + h) * A.Dh : nullptr;
  if (ntile == 0) {  // no sequence reaches this tile
    if (tid < 128 && i < A.T) {
      for (int d = 0; d < A.Dh; d += 8) {
        *reinterpret_cast<int4*>(y + d) = make_int4(0, 0, 0, 0);
        if (low != nullptr) *reinterpret_cast<int4*>(low + d) = make_int4(0, 0, 0, 0);
      }
      if (A.lse != nullptr) A.lse[(int64_t)h * A.T + i] = INFINITY;
    }
    return;
  }
  if (tid == 0) {
    mbar_init(&sh.k_full, 1), mbar_init(&sh.v_full, 1), mbar_init(&sh.s_done, 1), mbar_init(&sh.o_done, 1);
    mbar_init(&sh.s_read, 128), mbar_init(&sh.p_ready, 128);
    fence_mbar_init();
    sh.lo_max = 0;
  }
  if (w == 4) {
    umma::tmem_alloc(&sh.tmem, 256);
    umma::tmem_relinquish();
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tm = sh.tmem;
  // the sink tile has few keys: products and softmax take whole 16 (32) column groups of it
  const int sink_n = nsink ? (R.send - R.s0 + 15) & ~15 : 0;

  if (w >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (w == 4) {
      // Descriptors are made once and stepped by additions.
      const bool lead = umma::elect_one();
      const uint64_t dq = umma::sdesc_k(smem_u32(sQ)), dk = umma::sdesc_k(smem_u32(sK)), dv = umma::sdesc_mn(smem_u32(sV), kTileBytes);
      const int ks = A.Dh / 16;
      const uint32_t ido = umma::idesc_f16(128, A.Dh, Fmt<T>::id, 0, 1);
      auto load = [&](const CUtensorMap* m, unsigned char* dst, int head, int r, uint64_t* bar) {
#pragma unroll
        for (int b = 0; b < NB; ++b) tma_load_3d(dst + b * kTileBytes, m, b * 64, head, r, bar);
      };
      auto key0 = [&](int t) { return t < nsink ? R.s0 : R.kmin + (t - nsink) * 128; };
      auto cols = [&](int t) { return t < nsink ? sink_n : 128; };
      auto load_k = [&](int t) {
        if (lead) {
          mbar_arrive_expect_tx(&sh.k_full, NB * kTileBytes);
          load(&tk, sK, hk, key0(t), &sh.k_full);
        }
      };
      auto load_v = [&](int t) {
        if (lead) {
          mbar_arrive_expect_tx(&sh.v_full, NB * kTileBytes);
          load(&tv, sV, hk, key0(t), &sh.v_full);
        }
      };
      auto issue_s = [&](int t) {
        mbar_wait(&sh.k_full, t & 1);
        umma::fence_after_sync();
        const uint32_t ids = umma::idesc_f16(128, cols(t), Fmt<T>::id, 0, 0);
#pragma unroll
        for (int k = 0; k < NB * 4; ++k) {
          const int o = (k >> 2) * (kTileBytes / 16) + (k & 3) * 2;
          if (k < ks && lead) umma::mma_f16(tm, dq + o, dk + o, ids, k > 0);
        }
        if (lead) umma::commit(&sh.s_done);
      };
      auto issue_o = [&](int t) {
        mbar_wait(&sh.v_full, t & 1);
        umma::fence_after_sync();
        const int kp = cols(t) / 16;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < kp && lead) umma::mma_f16_ta(tm + kO, tm + kP + k * 8, dv + k * 128, ido, t > 0 || k > 0);
        if (lead) umma::commit(&sh.o_done);
      };
      if (lead) {
        mbar_arrive_expect_tx(&sh.k_full, 2 * NB * kTileBytes);
        load(&tq, sQ, h, q0, &sh.k_full);
        load(&tk, sK, hk, key0(0), &sh.k_full);
      }
      load_v(0);
      issue_s(0);
      for (int t = 0; t < ntile; ++t) {
        mbar_wait(&sh.s_done, t & 1);
        if (t + 1 < ntile) load_k(t + 1);
        if (kOwnP) {
          if (t + 1 < ntile) {
            mbar_wait(&sh.s_read, t & 1);
            issue_s(t + 1);
          }
          if (t > 0) {
            mbar_wait(&sh.o_done, (t - 1) & 1);
            load_v(t);
          }
        }
        mbar_wait(&sh.p_ready, t & 1);
        issue_o(t);
        if (!kOwnP && t + 1 < ntile) {
          mbar_wait(&sh.o_done, t & 1);  // P is read: the next S overwrites it
          load_v(t + 1);
          issue_s(t + 1);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const RowMask rm = row_mask(A, i);
    const int lo = rm.i < 0 ? 0 : rm.lo;
    atomicMax(&sh.lo_max, __reduce_max_sync(0xffffffffu, lo));
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const int lo_max = sh.lo_max, end = end_token(A);
    const uint32_t trow = tm + ((uint32_t)(w * 32) << 16);
    const float c = A.scale * kAttnLog2e;
    float m = -INFINITY, l = 0.f;
    for (int t = 0; t < ntile; ++t) {
      const bool sink = t < nsink;
      const int k0 = sink ? R.s0 : R.kmin + (t - nsink) * 128;
      const int nch = sink ? (sink_n + 31) / 32 : 4;
      // every query of the tile sees every key of a tile between the last window's start and the first query
      const bool full = !sink && k0 >= lo_max && k0 + 127 <= q0;
      mbar_wait(&sh.s_done, t & 1);
      umma::fence_after_sync();
      // what the query sees of the tile, a word per 32 keys
      uint32_t see[4] = {};
      if (!full) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int at = k0 + b * 32;
          see[b] = bits(rm.start - at, min(min(rm.sink_end, rm.i + 1), sink ? R.send : INT32_MAX) - at);
          if (!sink) see[b] |= bits(rm.lo - at, rm.i + 1 - at);
        }
      }
      uint32_t s[4][32];
      // the blocks' bounds and the masks' selects are kept out of the tiles that every query sees in full
      auto maximum = [&](auto whole) {
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        umma::tmem_ld32(trow, s[0]);
#pragma unroll
        for (int b = 0; b < 4; ++b) {  // a block's maximum while the next block comes
          if (!whole && b >= nch) continue;
          umma::tmem_wait_ld(s[b]);
          if (b + 1 < 4 && (whole || b + 1 < nch)) umma::tmem_ld32(trow + (b + 1) * 32, s[b + 1 < 4 ? b + 1 : 3]);
          if (!whole)
#pragma unroll
            for (int j = 0; j < 32; ++j) s[b][j] = see[b] >> j & 1 ? s[b][j] : 0xff800000u;
#pragma unroll
          for (int j = 0; j < 32; j += 2)
            mx4[j >> 1 & 3] = max3(mx4[j >> 1 & 3], __uint_as_float(s[b][j]), __uint_as_float(s[b][j + 1]));
        }
        return fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      };
      const float mx = full ? maximum(std::true_type{}) : maximum(std::false_type{});
      if (kOwnP) {  // the next S may start under this tile's exponentials
        umma::fence_before_sync();
        mbar_arrive(&sh.s_read);
      }
      if (t > 0) {  // P and O are free
        mbar_wait(&sh.o_done, (t - 1) & 1);
        umma::fence_after_sync();
      }
      if (__any_sync(0xffffffffu, (mx - m) * c > kRescale || m == -INFINITY)) {
        const float to = fmaxf(mx, m);
        const float f = to == -INFINITY ? 1.f : ex2((m - to) * c);
        m = to, l *= f;
        if (t > 0)
          for (int d = 0; d < A.Dh; d += 32) {
            uint32_t o[32];
            umma::tmem_ld32(trow + kO + d, o);
            umma::tmem_wait_ld(o);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
            umma::tmem_st32(trow + kO + d, o);
          }
      }
      const float mc = m == -INFINITY ? 0.f : m * c;
      const uint64_t c2 = pair(c, c), mc2 = pair(-mc, -mc);
      uint64_t sum[2] = {0, 0};
      auto exponentials = [&](auto whole) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (!whole && b >= nch) continue;
          uint32_t p[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float x0, x1;
            unpair(fma2(pair(s[b][2 * j], s[b][2 * j + 1]), c2, mc2), x0, x1);
            x0 = ex2(x0), x1 = ex2(x1);
            sum[j & 1] = add2(sum[j & 1], pair(x0, x1));
            p[j] = Fmt<T>::pack(x0, x1);
          }
          umma::tmem_st16(trow + kP + b * 16, p);
        }
      };
      if (full) exponentials(std::true_type{});
      else exponentials(std::false_type{});
      float l0, l1;
      unpair(add2(sum[0], sum[1]), l0, l1);
      l += l0 + l1;
      if (k0 + 128 > end) {  // rows behind the last sequence may hold anything: 0 x NaN would reach O
        mbar_wait(&sh.v_full, t & 1);
        if (k0 + tid >= end)
#pragma unroll
          for (int b = 0; b < NB * 8; ++b)
            *reinterpret_cast<int4*>(sV + (b >> 3) * kTileBytes + tid * 128 + (b & 7) * 16) = make_int4(0, 0, 0, 0);
        fence_proxy_async_smem();
      }
      umma::tmem_wait_st();
      umma::fence_before_sync();
      mbar_arrive(&sh.p_ready);
    }
    mbar_wait(&sh.o_done, (ntile - 1) & 1);
    umma::fence_after_sync();
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    float odd = 0.f;  // NaN as soon as one element is not finite
    for (int d = 0; d < A.Dh; d += 32) {
      uint32_t o[32];
      umma::tmem_ld32(trow + kO + d, o);
      umma::tmem_wait_ld(o);
#pragma unroll
      for (int j = 0; j < 32; ++j) odd = fmaf(__uint_as_float(o[j]), 0.f, odd);
      if (i < A.T)
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          uint32_t p[4], r[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v0 = __uint_as_float(o[j + 2 * e]) * inv, v1 = __uint_as_float(o[j + 2 * e + 1]) * inv;
            p[e] = rm.i < 0 ? 0u : Fmt<T>::pack(v0, v1);
            const float2 back = Fmt<T>::unpack(p[e]);
            r[e] = rm.i < 0 ? 0u : Fmt<T>::pack(v0 - back.x, v1 - back.y);
          }
          *reinterpret_cast<uint4*>(y + d + j) = make_uint4(p[0], p[1], p[2], p[3]);
          if (low != nullptr) *reinterpret_cast<uint4*>(low + d + j) = make_uint4(r[0], r[1], r[2], r[3]);
        }
    }
    if (i < A.T && A.lse != nullptr) A.lse[(int64_t)h * A.T + i] = rm.i < 0 || l == 0.f ? INFINITY : m * c + log2f(l);
    // l = 0: nothing but scores of -infinity, whose softmax is the row's own NaN
    const uint32_t again = __ballot_sync(0xffffffffu, rm.i >= 0 && (odd != 0.f || l == 0.f));
    __syncwarp();
    for (int r = 0; r < 32 && again; ++r)
      if (again >> r & 1) exact_fwd_row<T>(A, h, q0 + w * 32 + r);
    umma::fence_before_sync();
  }
  __syncthreads();
  if (w == 4) umma::tmem_dealloc(tm, 256);
}

template <typename T, int NB> static int fwd_nb(const AttnArgs& A, cudaStream_t st) {
  CUtensorMap tq, tk, tv;
  constexpr auto dt = TmapType<T>::v;
  if (int rc = head_map(&tq, A.q, dt, A, A.Hq, A.q_ts, A.q_hs, 128)) return rc;
  if (int rc = head_map(&tk, A.k, dt, A, A.Hkv, A.k_ts, A.k_hs, 128)) return rc;
  if (int rc = head_map(&tv, A.v, dt, A, A.Hkv, A.v_ts, A.v_hs, 128)) return rc;
  constexpr int smem = 3 * NB * kTileBytes + 1024;
  if (int rc = allow_smem<attn_fwd_kernel<T, NB>>(smem, "attn_fwd_kernel")) return rc;
  if (int rc = expect_regs<attn_fwd_kernel<T, NB>>(kFwdRegs, "attn_fwd_kernel")) return rc;
  attn_fwd_kernel<T, NB><<<dim3((A.T + 127) / 128, A.Hq), kFwdThreads, smem, st>>>(A, tq, tk, tv);
  return check_launch("attn_fwd_kernel");
}

template <typename T> int attn_fwd_launch(const AttnArgs& A, cudaStream_t st) {
  return A.Dh <= 64 ? fwd_nb<T, 1>(A, st) : fwd_nb<T, 2>(A, st);
}
template int attn_fwd_launch<__nv_bfloat16>(const AttnArgs&, cudaStream_t);
template int attn_fwd_launch<__half>(const AttnArgs&, cudaStream_t);

int attn_fwd_device_error(bool clear) { return read_device_error(clear); }

}  // namespace mr
