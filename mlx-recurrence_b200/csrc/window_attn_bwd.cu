// Sliding-window attention with sinks, backward, on the tensor cores (tcgen05):
// bf16 and fp16, Dh <= 128. No atomics: every sum has one order.
//
//   p_ij = exp(scale q_i.k_j - lse_i),  ds_ij = p_ij (gy_i.v_j - delta_i)
//   grad_q = scale ds K,  grad_k = scale ds^T Q,  grad_v = p^T gy
//
// One kernel, twice: rows of a tile (128, resident in shared memory) against a
// stream of 64-wide column tiles.
//   KV = false: rows are queries, columns the keys they see; grad_q.
//   KV = true:  rows are keys, columns the queries that see them, over every
//               query head that shares the key head; grad_k, grad_v.
// Per column tile S = R1 C1^T and dP = R2 C2^T land in TMEM, a warpgroup (a
// thread per row) turns them into P and dS, written back over them as the A
// operands of the sums P C2 and dS C1, which stay in TMEM. That is 7 products
// where one pass with atomic sums would need 5.
//
// Two column tiles are in flight per SM, a warpgroup each: in two CTAs of 256 TMEM
// columns (Dh <= 64), or in one, whose sums take 256 of its 512 columns. What
// bounds it: a tile is a chain (S, exponentials, dS, sums), so the issuing warp
// starts the next S of a stage before the last sum of the old tile: P C2 runs
// under the dS arithmetic, the next S follows as soon as P (KV = false: S) has
// been read, the next dP after dS C1.
//
// P and dS are rounded to the inputs' type, which the products take; lse, delta and the
// sums are float32. In fp16 dS goes in at a power of two of each row's own (a query's, or
// a key's), taken from a bound of what the row can meet, |dS_ij| <= |gy_i| |v_j| + |delta_i|
// over the j it sees (the i that see it): nothing leaves fp16's range whatever the loss
// scale, and no other sequence, head or token out of reach costs it precision.
//
// bf16, 16384 tokens, 32 heads of 64, window 1024: 824 us (391 TFLOP/s of the 5
// products); 16 heads of 128 on 4, window 2048, 4 sinks: 772 us (480). Measured and
// not kept (where this form took 851 and 762 us): both products of S and dP before
// any sum of the old tile (918 and 826 us), three warpgroups in one CTA for Dh <= 64
// (1,034 us), two threads per row (827 and 790 us).
//
// The sinks' far queries (window_attn.cuh): a query tile that meets a sink tile adds
// the sinks' gradients by products over its 128 queries, with P and dS handed
// through shared memory.
#include "window_tc.cuh"

namespace mr {

constexpr int kNC = 64;                  // columns of a tile
constexpr int kColBytes = kNC * 128;     // one 64-wide block of a column tile
template <int NB> constexpr int kNS = NB;      // column tiles in flight: TMEM stages and warpgroups
constexpr int kStages = 4;                     // column tiles in shared memory
template <int NB> constexpr int kBwdThreads = kNS<NB> * 128 + 32;

struct BwdArgs {
  AttnArgs a;
  const float *fq, *fk;  // fp16: [Hq, T], [Hkv, T], dS's scale per query and per key
};

struct BwdShared {
  uint64_t r_full, c_full[kStages], s_done[2], dp_done[2], p_ready[2], ds_ready[2], acc2_done, acc1_done, all_done, sink_done, sink_read;
  uint32_t tmem;
  int lo_max, lim_min, f_min;
  int again[128];
  alignas(16) float lse[2][kNC], delta[2][kNC];  // negated, of the column tile's queries
};

template <typename T, int NB, bool KV>
__global__ void __launch_bounds__(kBwdThreads<NB>, NB == 1 ? 2 : 1)
attn_bwd_kernel(const __grid_constant__ BwdArgs P, const __grid_constant__ CUtensorMap tr1,
                const __grid_constant__ CUtensorMap tr2, const __grid_constant__ CUtensorMap tc1,
                const __grid_constant__ CUtensorMap tc2) {
  constexpr int NS = kNS<NB>, NC = kStages;
  constexpr int kStageBytes = 2 * NB * kColBytes;
  constexpr uint32_t kAcc1 = NS * 128, kAcc2 = kAcc1 + NB * 64, kCols = NB == 1 ? 256 : 512, kSinkK = NB == 1 ? 0 : 128;
  extern __shared__ unsigned char raw[];
  unsigned char* sC = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  unsigned char *sR1 = sC + NC * kStageBytes, *sR2 = sR1 + NB * kTileBytes;
  __shared__ BwdShared sh;
  const AttnArgs& A = P.a;
  const int tid = threadIdx.x, w = tid >> 5, G = A.Hq / A.Hkv;
  const int hr = blockIdx.y, hk = KV ? hr : hr / G, r0 = blockIdx.x * 128;
  const int end = end_token(A);

  // the columns: keys (a sink tile, then the band) or queries, per query head
  int c_beg = 0, c_end = 0, s0 = 0, send = 0;
  if (KV) {
    const QueryRange Q = near_queries<7>(A, r0, r0 + 128);
    c_beg = Q.qbeg, c_end = Q.qend;
  } else {
    const KeyRange R = keys_of(A, r0, r0 + 128);
    c_beg = R.kmin, c_end = R.kend, s0 = R.s0, send = R.send;
  }
  const int nsink = send > s0 ? 1 : 0, per = (c_end - c_beg + kNC - 1) / kNC;
  const int n = c_end > c_beg ? (KV ? G * per : nsink + per) : 0;
  const int H = KV ? A.Hkv : A.Hq;
  if (n == 0) {
    if (tid < 128 && r0 + tid < A.T) {
      const int64_t at = ((int64_t)(r0 + tid) * H + hr) * A.Dh;
      for (int d = 0; d < A.Dh; d += 8) {
        *reinterpret_cast<int4*>((T*)(KV ? A.gk : A.gq) + at + d) = make_int4(0, 0, 0, 0);
        if (KV) *reinterpret_cast<int4*>((T*)A.gv + at + d) = make_int4(0, 0, 0, 0);
      }
    }
    return;
  }
  auto col0 = [&](int t) { return KV ? c_beg + t % per * kNC : t < nsink ? s0 : c_beg + (t - nsink) * kNC; };

  if (tid == 0) {
    mbar_init(&sh.r_full, 1);
    for (int i = 0; i < NC; ++i) mbar_init(&sh.c_full[i], 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sh.s_done[i], 1), mbar_init(&sh.dp_done[i], 1);
      mbar_init(&sh.p_ready[i], 128), mbar_init(&sh.ds_ready[i], 128);
    }
    mbar_init(&sh.acc1_done, 1), mbar_init(&sh.acc2_done, 1), mbar_init(&sh.all_done, 1);
    mbar_init(&sh.sink_done, 1), mbar_init(&sh.sink_read, 128);
    fence_mbar_init();
    sh.lo_max = 0, sh.lim_min = INT32_MAX, sh.f_min = 0x7f000000;
  }
  if (tid < 128) sh.again[tid] = 0;
  if (w == 4 * NS) {
    umma::tmem_alloc(&sh.tmem, kCols);
    umma::tmem_relinquish();
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tm = sh.tmem;

  if (w == 4 * NS) {
    {
      const bool lead = umma::elect_one();
      const uint32_t ar1 = smem_u32(sR1), ar2 = smem_u32(sR2), ac = smem_u32(sC);
      // descriptors are made once and stepped by additions
      const uint64_t dr1 = umma::sdesc_k(ar1), dr2 = umma::sdesc_k(ar2), dck = umma::sdesc_k(ac), dcm = umma::sdesc_mn(ac, kColBytes);
      const int ks = A.Dh / 16;
      auto row_step = [](int k) { return (k >> 2) * (kTileBytes / 16) + (k & 3) * 2; };
      auto col_step = [](int k) { return (k >> 2) * (kColBytes / 16) + (k & 3) * 2; };
      auto load_c = [&](int t) {
        const int st = t % NC, hc = KV ? hr * G + t / per : hk;
        unsigned char* dst = sC + st * kStageBytes;
        if (lead) {
          mbar_arrive_expect_tx(&sh.c_full[st], kStageBytes);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            tma_load_3d(dst + b * kColBytes, &tc1, b * 64, hc, col0(t), &sh.c_full[st]);
            tma_load_3d(dst + (NB + b) * kColBytes, &tc2, b * 64, hc, col0(t), &sh.c_full[st]);
          }
        }
      };
      const uint32_t id_s = umma::idesc_f16(128, kNC, Fmt<T>::id, 0, 0);
      const uint32_t id_a = umma::idesc_f16(128, A.Dh, Fmt<T>::id, 0, 1);
      auto issue_s = [&](int t) {
        const uint32_t d = tm + t % NS * 128;
        const uint64_t c1 = dck + t % NC * (kStageBytes / 16);
        mbar_wait(&sh.c_full[t % NC], (t / NC) & 1);
        umma::fence_after_sync();
#pragma unroll
        for (int k = 0; k < NB * 4; ++k)
          if (k < ks && lead) umma::mma_f16(d, dr1 + row_step(k), c1 + col_step(k), id_s, k > 0);
        if (lead) umma::commit(&sh.s_done[t % NS]);
      };
      auto issue_dp = [&](int t) {
        const uint32_t d = tm + t % NS * 128 + 64;
        const uint64_t c2 = dck + t % NC * (kStageBytes / 16) + NB * kColBytes / 16;
#pragma unroll
        for (int k = 0; k < NB * 4; ++k)
          if (k < ks && lead) umma::mma_f16(d, dr2 + row_step(k), c2 + col_step(k), id_s, k > 0);
        if (lead) umma::commit(&sh.dp_done[t % NS]);
      };
      auto issue_acc = [&](int t, uint32_t acc, int which, uint64_t* bar) {  // which = 0: dS C1, 1: P C2
        const uint32_t d = tm + t % NS * 128 + (which ? 0 : 64);
        const uint64_t cm = dcm + t % NC * (kStageBytes / 16) + which * (NB * kColBytes / 16);
        umma::fence_after_sync();
#pragma unroll
        for (int k = 0; k < kNC / 16; ++k)
          if (lead) umma::mma_f16_ta(tm + acc, d + k * 8, cm + k * 128, id_a, t > 0 || k > 0);
        if (lead) umma::commit(bar);
      };
      if (lead) {
        mbar_arrive_expect_tx(&sh.r_full, 2 * NB * kTileBytes);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          tma_load_3d(sR1 + b * kTileBytes, &tr1, b * 64, hr, r0, &sh.r_full);
          tma_load_3d(sR2 + b * kTileBytes, &tr2, b * 64, hr, r0, &sh.r_full);
        }
      }
      load_c(0);
      if (nsink == 0)
        for (int t = 1; t < min(n, NC); ++t) load_c(t);
      mbar_wait(&sh.r_full, 0);
      if (nsink) {
        // the sink tile by itself: its sums over the queries use the other stages' memory and columns
        issue_s(0);
        issue_dp(0);
        mbar_wait(&sh.p_ready[0], 0);
        mbar_wait(&sh.ds_ready[0], 0);
        issue_acc(0, kAcc1, 0, &sh.acc1_done);
        const uint32_t id_t = umma::idesc_f16(128, A.Dh, Fmt<T>::id, 1, 1);  // rows at and behind 64 are not used
        const uint64_t pt = umma::sdesc_mn(ac + kStageBytes, kTileBytes), dst = pt + kTileBytes / 16;
        const uint64_t r1m = umma::sdesc_mn(ar1, kTileBytes), r2m = umma::sdesc_mn(ar2, kTileBytes);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (lead) umma::mma_f16(tm + kAcc2, pt + k * 128, r2m + k * 128, id_t, k > 0);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (lead) umma::mma_f16(tm + kSinkK, dst + k * 128, r1m + k * 128, id_t, k > 0);
        if (lead) umma::commit(&sh.sink_done);
        mbar_wait(&sh.acc1_done, 0);
        mbar_wait(&sh.sink_read, 0);
        umma::fence_after_sync();
        for (int t = 1; t < min(n, NC + 1); ++t) load_c(t);
      }
      for (int t = nsink; t < min(n, nsink + NS); ++t) {
        issue_s(t);
        issue_dp(t);
      }
      auto next_dp = [&](int t) {  // the dP that takes the place of tile t's dS
        mbar_wait(&sh.acc1_done, t & 1);
        umma::fence_after_sync();
        if (t + NC < n) load_c(t + NC);
        if (t + NS < n) issue_dp(t + NS);
      };
      for (int t = nsink; t < n; ++t) {
        if (NS == 1 && t > nsink) next_dp(t - 1);
        mbar_wait(&sh.p_ready[t % NS], (t / NS) & 1);
        if (KV) issue_acc(t, kAcc2, 1, &sh.acc2_done);
        else if (t + NS < n) issue_s(t + NS);
        if (NS > 1 && t > nsink) next_dp(t - 1);
        mbar_wait(&sh.ds_ready[t % NS], (t / NS) & 1);
        if (KV && t + NS < n) {
          mbar_wait(&sh.acc2_done, t & 1);
          issue_s(t + NS);
        }
        issue_acc(t, kAcc1, 0, &sh.acc1_done);
      }
      if (lead) umma::commit(&sh.all_done);
    }
    __syncwarp();
  } else {
    const int wg = w >> 2, row = tid & 127, r = r0 + row;
    const uint32_t trow = tm + ((uint32_t)((w & 3) * 32) << 16);
    const float c = A.scale * kAttnLog2e;
    float f = 1.f;  // dS's scale
    // what the row sees: columns [lo, hi) and (queries) sinks [s_lo, s_hi)
    int lo = INT32_MAX, hi = 0, s_lo = INT32_MAX, s_hi = 0;
    float lse_r = INFINITY, delta_r = 0.f;
    bool alive = false;
    if (KV) {
      hi = near_limit<7>(A, r);
      alive = hi > 0;
      if (alive) {
        lo = r;
        atomicMin(&sh.lim_min, hi);
        if (Fmt<T>::id == 0) f = P.fk[(int64_t)hr * A.T + r];
      }
    } else {
      const RowMask m = row_mask(A, r);
      alive = m.i >= 0;
      if (alive) {
        lo = m.lo, hi = r + 1, s_lo = m.start, s_hi = min(m.sink_end, r + 1);
        lse_r = A.lse[(int64_t)hr * A.T + r], delta_r = A.delta[(int64_t)hr * A.T + r];
        atomicMax(&sh.lo_max, lo);
        if (Fmt<T>::id == 0) {
          f = P.fq[(int64_t)hr * A.T + r];
          if (nsink && m.start == s0) atomicMin(&sh.f_min, __float_as_int(f));
        }
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(NS * 128) : "memory");
    const int lo_max = sh.lo_max, lim_min = sh.lim_min;
    // the sinks' sums need one scale for all queries that see them
    auto f_sink = [&] { return Fmt<T>::id == 0 ? __int_as_float(*reinterpret_cast<volatile int*>(&sh.f_min)) : 1.f; };
    if (!KV && nsink && r0 + 128 > end) {
      // queries behind the last sequence may hold anything: they must not reach the sinks' sums as 0 x NaN
      mbar_wait(&sh.r_full, 0);
      if (r >= end && wg == 0)
#pragma unroll
        for (int b = 0; b < NB * 8; ++b) {
          const int o = (b >> 3) * kTileBytes + row * 128 + (b & 7) * 16;
          *reinterpret_cast<int4*>(sR1 + o) = make_int4(0, 0, 0, 0);
          *reinterpret_cast<int4*>(sR2 + o) = make_int4(0, 0, 0, 0);
        }
      fence_proxy_async_smem();
    }
    // KV: lse (rows below 64) or delta of a column tile's query, a tile ahead of its use
    auto stat = [&](int head, int c) {
      const int q = c_beg + c * kNC + (row & 63);
      const float* v = (row < 64 ? A.lse : A.delta) + (int64_t)(hr * G + head) * A.T;
      return q < c_end ? -v[q] : row < 64 ? -INFINITY : 0.f;
    };
    int head = 0, c_at = wg;  // KV: query head of the group, and tile of its columns
    while (KV && c_at >= per) c_at -= per, ++head;
    float next_stat = KV && wg < n ? stat(head, c_at) : 0.f;
    for (int t = wg; t < n; t += NS) {
      const bool sink = !KV && t < nsink;
      const int k0 = KV ? c_beg + c_at * kNC : col0(t), b = t % NS, ph = (t / NS) & 1;
      const bool full = KV ? k0 >= r0 + 127 && k0 + kNC <= lim_min : !sink && k0 >= lo_max && k0 + kNC - 1 <= r0;
      if (KV) {
        asm volatile("bar.sync %0, 128;" ::"r"(2 + wg) : "memory");  // the last tile's values have been read
        (row < 64 ? sh.lse[wg] : sh.delta[wg])[row & 63] = next_stat;
        asm volatile("bar.sync %0, 128;" ::"r"(2 + wg) : "memory");
        c_at += NS;
        while (c_at >= per) c_at -= per, ++head;
        if (t + NS < n) next_stat = stat(head, c_at);
      }
      uint32_t s[2][32], p[32], ds[32], see[2] = {0, 0};
      const uint64_t c2 = pair(c, c), l2 = pair(-lse_r, -lse_r), d2 = pair(-delta_r, -delta_r), f2 = pair(f, f);
      if (!full)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int at = k0 + x * 32;
          see[x] = sink ? bits(s_lo - at, min(s_hi, send) - at) : bits(lo - at, hi - at) | bits(s_lo - at, s_hi - at);
        }
      // the masks' selects are kept out of the tiles that every row sees in full
      auto to_p = [&](auto masked) {
        ulonglong2 l4 = {};
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (KV && j % 2 == 0) l4 = *reinterpret_cast<const ulonglong2*>(&sh.lse[wg][x * 32 + 2 * j]);
            const uint64_t l = KV ? (j % 2 ? l4.y : l4.x) : l2;
            float e0, e1;
            unpair(fma2(pair(s[x][2 * j], s[x][2 * j + 1]), c2, l), e0, e1);
            e0 = ex2(e0), e1 = ex2(e1);
            if (masked) {
              e0 = see[x] >> (2 * j) & 1 ? e0 : 0.f;
              e1 = see[x] >> (2 * j + 1) & 1 ? e1 : 0.f;
            }
            s[x][2 * j] = __float_as_uint(e0), s[x][2 * j + 1] = __float_as_uint(e1);
            if (KV || (masked && sink)) p[x * 16 + j] = Fmt<T>::pack(e0, e1);
          }
      };
      auto to_ds = [&](auto masked) {
        ulonglong2 d4 = {};
        [[maybe_unused]] uint32_t to_sink[4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          uint32_t dp[32];
          umma::tmem_ld32(trow + b * 128 + 64 + x * 32, dp);
          umma::tmem_wait_ld(dp);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (KV && j % 2 == 0) d4 = *reinterpret_cast<const ulonglong2*>(&sh.delta[wg][x * 32 + 2 * j]);
            const uint64_t d = KV ? (j % 2 ? d4.y : d4.x) : d2;
            uint64_t g = mul2(pair(s[x][2 * j], s[x][2 * j + 1]), add2(pair(dp[2 * j], dp[2 * j + 1]), d));
            float g0, g1;
            if constexpr (Fmt<T>::id == 0) {
              if (!KV && masked && sink) {  // at the sinks' scale, to shared memory
                const float fs = f_sink();
                unpair(mul2(g, pair(fs, fs)), g0, g1);
                to_sink[j & 3] = Fmt<T>::pack(see[x] >> (2 * j) & 1 ? g0 : 0.f, see[x] >> (2 * j + 1) & 1 ? g1 : 0.f);
                if ((j & 3) == 3)
                  *reinterpret_cast<uint4*>(sC + kStageBytes + kTileBytes + umma::sw128_off(row, x * 32 + (j & ~3) * 2)) =
                      make_uint4(to_sink[0], to_sink[1], to_sink[2], to_sink[3]);
              }
              g = mul2(g, f2);
            }
            unpair(g, g0, g1);
            if (masked) {  // not 0 x NaN of what the row does not see
              g0 = see[x] >> (2 * j) & 1 ? g0 : 0.f;
              g1 = see[x] >> (2 * j + 1) & 1 ? g1 : 0.f;
            }
            ds[x * 16 + j] = Fmt<T>::pack(g0, g1);
          }
        }
      };
      mbar_wait(&sh.s_done[b], ph);
      umma::fence_after_sync();
#pragma unroll
      for (int x = 0; x < 2; ++x) umma::tmem_ld32(trow + b * 128 + x * 32, s[x]);
#pragma unroll
      for (int x = 0; x < 2; ++x) umma::tmem_wait_ld(s[x]);
      if (!KV) {  // S has been read
        umma::fence_before_sync();
        mbar_arrive(&sh.p_ready[b]);
      }
      if (full) to_p(std::false_type{});
      else to_p(std::true_type{});
      if (k0 + kNC > end) {  // columns behind the last sequence: as above
        mbar_wait(&sh.c_full[t % NC], (t / NC) & 1);
        for (int x = row; x < kNC * NB * 2; x += 128) {
          const int cr = x % kNC;
          if (k0 + cr >= end)
#pragma unroll
            for (int y = 0; y < 8; ++y)
              *reinterpret_cast<int4*>(sC + t % NC * kStageBytes + x / kNC * kColBytes + cr * 128 + y * 16) = make_int4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      if (KV) {
        umma::tmem_st32(trow + b * 128, p);
        umma::tmem_wait_st();
        umma::fence_before_sync();
        mbar_arrive(&sh.p_ready[b]);
      }
      mbar_wait(&sh.dp_done[b], ph);
      umma::fence_after_sync();
      if (full) to_ds(std::false_type{});
      else to_ds(std::true_type{});
      umma::tmem_st32(trow + b * 128 + 64, ds);
      if (sink) {
        unsigned char *sp = sC + kStageBytes, *sd = sp + kTileBytes;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          *reinterpret_cast<uint4*>(sp + umma::sw128_off(row, x * 8)) = make_uint4(p[x * 4], p[x * 4 + 1], p[x * 4 + 2], p[x * 4 + 3]);
          if (Fmt<T>::id != 0)
            *reinterpret_cast<uint4*>(sd + umma::sw128_off(row, x * 8)) = make_uint4(ds[x * 4], ds[x * 4 + 1], ds[x * 4 + 2], ds[x * 4 + 3]);
        }
        fence_proxy_async_smem();
      }
      umma::tmem_wait_st();
      umma::fence_before_sync();
      mbar_arrive(&sh.ds_ready[b]);
      if (sink) {
        mbar_wait(&sh.sink_done, 0);
        umma::fence_after_sync();
        if (row < 64) {  // lanes 0 .. 63 hold the sinks
          float* pk = A.part + part_at(A, blockIdx.x, hr, 0, row);
          float* pv = A.part + part_at(A, blockIdx.x, hr, 1, row);
          for (int d = 0; d < A.Dh; d += 32) {
            uint32_t gk[32], gv[32];
            umma::tmem_ld32(trow + kSinkK + d, gk);
            umma::tmem_ld32(trow + kAcc2 + d, gv);
            umma::tmem_wait_ld(gk);
            umma::tmem_wait_ld(gv);
            if (row < send - s0) {
              const float back = 1.f / f_sink();
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                *reinterpret_cast<float4*>(pk + d + j) = make_float4(__uint_as_float(gk[j]) * back, __uint_as_float(gk[j + 1]) * back,
                                                                     __uint_as_float(gk[j + 2]) * back, __uint_as_float(gk[j + 3]) * back);
                *reinterpret_cast<uint4*>(pv + d + j) = make_uint4(gv[j], gv[j + 1], gv[j + 2], gv[j + 3]);
              }
            }
          }
        }
        umma::fence_before_sync();
        mbar_arrive(&sh.sink_read);
      }
    }
    mbar_wait(&sh.all_done, 0);
    umma::fence_after_sync();
    const int64_t at = ((int64_t)r * H + hr) * A.Dh;
    float odd = 0.f;  // NaN as soon as one element is not finite
    // a sink's far queries
    const float* far = KV ? far_sum<7>(A, r, hk) : nullptr;
    // the warpgroups share the blocks of 32 columns
    for (int a = 0; a < (KV ? 2 : 1); ++a) {
      const float scale = a == 0 ? A.scale : 1.f, fa = a == 0 ? 1.f / f : 1.f;
      T* g = (T*)(a == 1 ? A.gv : KV ? A.gk : A.gq) + at;
      for (int d = 0; d < A.Dh; d += 32) {
        if ((a * A.Dh + d) / 32 % NS != wg) continue;
        uint32_t o[32];
        umma::tmem_ld32(trow + (a == 0 ? kAcc1 : kAcc2) + d, o);
        umma::tmem_wait_ld(o);
        if (far != nullptr)
#pragma unroll
          for (int j = 0; j < 32; ++j)
            o[j] = __float_as_uint(fmaf(__uint_as_float(o[j]), fa, far[(int64_t)a * A.sinks * A.Dh + d + j]));
        else if (Fmt<T>::id == 0)
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * fa);
#pragma unroll
        for (int j = 0; j < 32; ++j) odd = fmaf(__uint_as_float(o[j]), 0.f, odd);
        if (r < A.T)
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = alive ? Fmt<T>::pack(__uint_as_float(o[j + 2 * e]) * scale, __uint_as_float(o[j + 2 * e + 1]) * scale) : 0u;
            *reinterpret_cast<uint4*>(g + d + j) = make_uint4(v[0], v[1], v[2], v[3]);
          }
      }
    }
    if (alive && odd != 0.f) sh.again[row] = 1;
    asm volatile("bar.sync 1, %0;" ::"n"(NS * 128) : "memory");
    for (int x = w; x < 128; x += 4 * NS)
      if (sh.again[x]) {
        if (KV) exact_gkv_row<T>(A, hr, r0 + x);
        else exact_gq_row<T>(A, hr, r0 + x);
      }
    umma::fence_before_sync();
  }
  __syncthreads();
  if (w == 4 * NS) umma::tmem_dealloc(tm, kCols);
}

// delta[h][t] = sum_d gy y with y and what its rounding dropped (from the rounded y alone the gradients' error is 1.55
// times the output rounding's, so 1.4), zero for rows outside every sequence; fp16: norm[h][t] = |gy| over its finite
// elements. 8 lanes per row, 16 bytes each at a time.
template <typename T> __global__ void __launch_bounds__(256) attn_delta_kernel(const __grid_constant__ AttnArgs A, float* norm) {
  const int64_t row = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  const int sub = threadIdx.x & 7;
  float s = 0.f, sq = 0.f;
  if (row < (int64_t)A.T * A.Hq) {
    const int64_t t = row / A.Hq, h = row % A.Hq;
    const bool in = A.lse[h * A.T + t] != INFINITY;
    if (in)
      for (int d = sub * 8; d < A.Dh; d += 64) {
        const Vec<T, 8> g = ld_vec<T, 8>((const T*)A.gy + row * A.Dh + d), y = ld_vec<T, 8>((const T*)A.y + row * A.Dh + d);
        const Vec<T, 8> r = ld_vec<T, 8>((const T*)A.y_low + row * A.Dh + d);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = to_f(g.v[j]);
          s = fmaf(x, to_f(y.v[j]) + to_f(r.v[j]), s);
          if (fabsf(x) < INFINITY) sq = fmaf(x, x, sq);
        }
      }
  }
#pragma unroll
  for (int x = 4; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x, 8), sq += __shfl_xor_sync(0xffffffffu, sq, x, 8);
  if (sub == 0 && row < (int64_t)A.T * A.Hq) {
    const int64_t at = row % A.Hq * A.T + row / A.Hq;
    A.delta[at] = s;
    if (norm != nullptr) norm[at] = sqrtf(sq);
  }
}

// ---- fp16: dS's scales ------------------------------------------------------------
// A row's bound is a maximum over the window of tokens around it, so norms are kept per token and, for whole runs of
// kRun tokens, as the run's maximum.
constexpr int kRun = 64;
struct ScaleArgs {
  float* fq;            // [Hq, T]: |gy|, then the queries' scales
  float *g, *d, *v;     // [Hkv, T]: |gy| and |delta|, the largest of the key head's query heads, and |v|
  float *rg, *rd, *rv;  // [Hkv, runs]: their maxima
  float* fk;            // [Hkv, T]: the keys' scales
};

// g, d, v and the runs' maxima: a CTA per run and key head, 4 lanes per token. Values that are not finite are left out
// (what they reach is not finite whatever the scale), tokens of no sequence count as zero.
template <typename T>
__global__ void __launch_bounds__(4 * kRun) attn_norm_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ ScaleArgs W) {
  __shared__ uint32_t top[3][4 * kRun / 32];
  const int hk = blockIdx.y, G = A.Hq / A.Hkv, t = blockIdx.x * kRun + (threadIdx.x >> 2), sub = threadIdx.x & 3;
  float sq = 0.f, g = 0.f, d = 0.f;
  if (t < A.T && A.lse[(int64_t)hk * G * A.T + t] != INFINITY) {
    const T* v = (const T*)A.v + t * A.v_ts + hk * A.v_hs;
    for (int e = sub * 8; e < A.Dh; e += 32) {
      const Vec<T, 8> x = ld_vec<T, 8>(v + e);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (fabsf(to_f(x.v[j])) < INFINITY) sq = fmaf(to_f(x.v[j]), to_f(x.v[j]), sq);
    }
    for (int h = hk * G + sub; h < (hk + 1) * G; h += 4) {
      const float dl = fabsf(A.delta[(int64_t)h * A.T + t]);
      g = fmaxf(g, W.fq[(int64_t)h * A.T + t]);
      if (dl < INFINITY) d = fmaxf(d, dl);
    }
  }
#pragma unroll
  for (int x = 1; x < 4; x *= 2) {
    sq += __shfl_xor_sync(0xffffffffu, sq, x);
    g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, x));
    d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, x));
  }
  const float n = sqrtf(sq);
  if (sub == 0 && t < A.T) {
    const int64_t at = (int64_t)hk * A.T + t;
    W.g[at] = g, W.d[at] = d, W.v[at] = n;
  }
  // (the bits of floats that are not negative have the floats' order)
  const uint32_t m[3] = {__reduce_max_sync(0xffffffffu, __float_as_uint(g)), __reduce_max_sync(0xffffffffu, __float_as_uint(d)),
                         __reduce_max_sync(0xffffffffu, __float_as_uint(n))};
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < 3; ++i) top[i][threadIdx.x >> 5] = m[i];
  __syncthreads();
  if (threadIdx.x < 3) {
    uint32_t x = 0;
    for (int i = 0; i < 4 * kRun / 32; ++i) x = max(x, top[threadIdx.x][i]);
    float* r = threadIdx.x == 0 ? W.rg : threadIdx.x == 1 ? W.rd : W.rv;
    r[(int64_t)hk * gridDim.x + blockIdx.x] = __uint_as_float(x);
  }
}

// the largest of x[a .. b-1], whole runs by their maxima
__device__ __forceinline__ float range_max(const float* x, const float* runs, int a, int b) {
  float m = 0.f;
  const int a1 = min((a + kRun - 1) / kRun * kRun, b), b0 = max(b / kRun * kRun, a1);
  for (int i = a; i < a1; ++i) m = fmaxf(m, x[i]);
  for (int i = a1 / kRun; i < b0 / kRun; ++i) m = fmaxf(m, runs[i]);
  for (int i = b0; i < b; ++i) m = fmaxf(m, x[i]);
  return m;
}
// a power of two that takes the bound to 2^14 .. 2^15, below fp16's largest number (1 for zero)
__device__ __forceinline__ float ds_scale(float bound) {
  if (bound == 0.f) return 1.f;
  const int e = max((int)(__float_as_uint(bound) >> 23) - 127, -86);
  return __int_as_float((127 + 14 - e) << 23);
}
// Grid: tokens, key heads. T=16384, 32 heads of 64, window 1024: 34 us, and 24 for the norms, of a backward of 953 us
// (bf16, which needs neither: 820); 16 heads of 128 on 4, window 2048: 838 us (775).
__global__ void __launch_bounds__(128) attn_scale_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ ScaleArgs W, int runs) {
  const int t = blockIdx.x * 128 + threadIdx.x, hk = blockIdx.y, G = A.Hq / A.Hkv;
  if (t >= A.T) return;
  const int64_t at = (int64_t)hk * A.T, rat = (int64_t)hk * runs;
  const RowMask m = row_mask(A, t);
  float v = 0.f;
  if (m.i >= 0) {
    v = range_max(W.v + at, W.rv + rat, m.lo, t + 1);
    if (m.start < min(m.sink_end, m.lo)) v = fmaxf(v, range_max(W.v + at, W.rv + rat, m.start, min(m.sink_end, m.lo)));
  }
  for (int h = hk * G; h < (hk + 1) * G; ++h) {  // |delta| <= |gy| max |v|
    float* f = W.fq + (int64_t)h * A.T + t;
    *f = ds_scale(2.f * *f * v);
  }
  const int end = key_limit(A, t);
  float g = 0.f, d = 0.f;
  if (end > 0) g = range_max(W.g + at, W.rg + rat, t, end), d = range_max(W.d + at, W.rd + rat, t, end);
  W.fk[at + t] = ds_scale(fmaf(g, W.v[at + t], d));
}

static int64_t delta_floats(int64_t T, int64_t Hq) { return (T * Hq + 3) / 4 * 4; }
size_t attn_bwd_ws_bytes(bool half, int64_t T, int64_t Hq, int64_t Hkv, int64_t Dh, int64_t sinks) {
  const int64_t scales = half ? T * Hq + 4 * T * Hkv + 3 * Hkv * ((T + kRun - 1) / kRun) : 0;
  return (size_t)((delta_floats(T, Hq) + scales) * 4) + part_bytes<7>(T, Hq, Dh, sinks);
}

template <typename T, int NB, bool KV>
static int bwd_one(const BwdArgs& P, cudaStream_t st) {
  const AttnArgs& A = P.a;
  CUtensorMap r1, r2, c1, c2;
  constexpr auto dt = TmapType<T>::v;
  const int64_t gts = (int64_t)A.Hq * A.Dh;
  if (int rc = head_map(KV ? &c1 : &r1, A.q, dt, A, A.Hq, A.q_ts, A.q_hs, KV ? kNC : 128)) return rc;
  if (int rc = head_map(KV ? &c2 : &r2, A.gy, dt, A, A.Hq, gts, A.Dh, KV ? kNC : 128)) return rc;
  if (int rc = head_map(KV ? &r1 : &c1, A.k, dt, A, A.Hkv, A.k_ts, A.k_hs, KV ? 128 : kNC)) return rc;
  if (int rc = head_map(KV ? &r2 : &c2, A.v, dt, A, A.Hkv, A.v_ts, A.v_hs, KV ? 128 : kNC)) return rc;
  constexpr int smem = kStages * 2 * NB * kColBytes + 2 * NB * kTileBytes + 1024;
  if (int rc = allow_smem<attn_bwd_kernel<T, NB, KV>>(smem, "attn_bwd_kernel")) return rc;
  attn_bwd_kernel<T, NB, KV><<<dim3((A.T + 127) / 128, KV ? A.Hkv : A.Hq), kBwdThreads<NB>, smem, st>>>(P, r1, r2, c1, c2);
  return check_launch(KV ? "attn_bwd_kernel (grad_k, grad_v)" : "attn_bwd_kernel (grad_q)");
}

template <typename T, int NB> static int bwd_nb(const BwdArgs& P, cudaStream_t st) {
  if (int rc = bwd_one<T, NB, false>(P, st)) return rc;
  if (P.a.part != nullptr)
    if (int rc = attn_sink_sum_launch<7>(P.a, st)) return rc;
  return bwd_one<T, NB, true>(P, st);
}

// ws: attn_bwd_ws_bytes, 16-byte aligned: delta, the sinks' partials, the scales
template <typename T> int attn_bwd_launch(const AttnArgs& A0, void* ws, cudaStream_t st) {
  BwdArgs P{A0, nullptr, nullptr};
  AttnArgs& A = P.a;
  A.delta = (float*)ws;
  float* rest = A.delta + delta_floats(A.T, A.Hq);
  if (has_far(A)) A.part = rest;
  rest += part_bytes<7>(A.T, A.Hq, A.Dh, A.sinks) / 4;
  constexpr bool half = Fmt<T>::id == 0;
  attn_delta_kernel<T><<<(unsigned)(((int64_t)A.T * A.Hq + 31) / 32), 256, 0, st>>>(A, half ? rest : nullptr);
  if (int rc = check_launch("attn_delta_kernel")) return rc;
  if constexpr (half) {
    const int runs = (A.T + kRun - 1) / kRun;
    const int64_t n = (int64_t)A.Hkv * A.T, r = (int64_t)A.Hkv * runs;
    ScaleArgs W;
    W.fq = rest;
    W.g = W.fq + (int64_t)A.Hq * A.T, W.d = W.g + n, W.v = W.d + n, W.fk = W.v + n;
    W.rg = W.fk + n, W.rd = W.rg + r, W.rv = W.rd + r;
    P.fq = W.fq, P.fk = W.fk;
    attn_norm_kernel<T><<<dim3(runs, A.Hkv), 4 * kRun, 0, st>>>(A, W);
    if (int rc = check_launch("attn_norm_kernel")) return rc;
    attn_scale_kernel<<<dim3((A.T + 127) / 128, A.Hkv), 128, 0, st>>>(A, W, runs);
    if (int rc = check_launch("attn_scale_kernel")) return rc;
  }
  return A.Dh <= 64 ? bwd_nb<T, 1>(P, st) : bwd_nb<T, 2>(P, st);
}
template int attn_bwd_launch<__nv_bfloat16>(const AttnArgs&, void*, cudaStream_t);
template int attn_bwd_launch<__half>(const AttnArgs&, void*, cudaStream_t);

int attn_bwd_device_error(bool clear) { return read_device_error(clear); }

}  // namespace mr
