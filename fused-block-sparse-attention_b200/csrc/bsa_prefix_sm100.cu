// Shared-prefix decode on tcgen05: the query rows of the whole batch that read one
// K/V head (B * grp * T of them) as M = 128 tiles over one split of the prefix.
//
//   S = Q K^T, P = 2^(S * scale * log2e - m), O += P V   per 128 prefix keys,
// with K, V through shared memory by TMA, S, P and O in TMEM, and (m, l, O) of the
// split left in fp32 for split_join_kernel.  P goes in as two 16-bit terms (split2), as in
// the split kernels, so that its rounding does not add to the output's and a sequence's
// precision does not hang on how many others are served beside it: in one term the error
// against 64 bits was 1.4 times that of the output's rounding alone (bf16, 65536 keys
// 2.33e-3 -> 1.65e-3; f16, 32768 keys 2.92e-4 -> 2.08e-4).  The second product with V and
// its terms took these from 46 to 51.5 us and from 108 to 123.  Unlike the sequence forward, a row tile
// gathers its rows from different sequences, every key is visible to every row, and the
// keys are split so that all SMs work on few rows.
//
// NT = 2 (D 64, 128; more than 128 rows): one CTA owns two row tiles that share every
// K/V tile: half the shared-memory fill per product.  NT = 1: up to 128 rows.  PAIR (D 256,
// more than 128 rows; O fills TMEM, so a CTA holds one row tile): two CTAs' row tiles in
// one product (M = 256), each with half of every K and V tile in its shared memory; alone,
// each read all of K and V, and their way from L2 bounded both (39 bytes per cycle and SM;
// 65536 keys, 256 rows of 2 heads, P in one term: 58.9 us alone, 44.5 in pairs).  The first
// CTA issues for both and its barriers take both CTAs' loads and softmax warps; commits go
// to both.  A tile's step is a chain S -> softmax -> PV, so what counts is
// that the next S is there when a softmax ends:
//   NT = 1: steps of 128 keys; P has columns of its own, so S of the next step runs
//     under the exponentials of this one.  Eight softmax warps, half a row per thread;
//     the halves exchange their maxima through shared memory.
//   NT = 2 ("half steps"): TMEM holds O and 128 columns per tile besides; steps of 64
//     keys use them as two S buffers, each overlaid by both terms of its own P, so S runs
//     one step ahead.  (One buffer of 128 keys left S waiting for PV: 6600 cycles per 128
//     keys and pair of tiles, tensor pipe 33% busy.)  Four warps per tile, a row per thread.
//
// K and V move as units of min(D, 128) columns x one step's keys in one ring, so that PV is
// issued with N = 128: a 128x64x16 product costs as much tensor time as three quarters
// of a 128x128x16 one.  S of each tile has an issuing warp, PV another: with one
// warp for all of it the tensor pipe ran dry between the batches.
// Softmax warps first, then the TMA producer, then the issuers, the first of which
// owns TMEM.  Every wait is bounded; a timeout sets BSA_DEVERR_TIMEOUT and the CTA runs
// on to its end.
#include <algorithm>
#include <type_traits>

#include "bsa_host.h"
#include "bsa_split.cuh"
#include "bsa_tc05.cuh"

namespace bsa {

namespace {
constexpr int PX_KEYS = 128;
constexpr int PX_CHUNK = PX_KEYS * 64 * 2;  // 16 KB: 128 rows x 64 columns
// O and l are rescaled only when a row's maximum grows by more than px_rescale (log2 units),
// so P may be as much larger than 1.  f16 ends at 2^16 and has nothing below 2^-24: there P is
// 2^13 larger (at most 2^15; m is stored lower by as much), so that keys 18 nats below the
// largest, many of them behind an attention sink, still count to half a step of f16.  With
// 2^7 and 8 their sum was off by 0.5% (one split of 2900 keys); 2^13 and 2 cost 5% of the
// time (32768 keys, 512 rows of 8 heads, D 128, at the power limit: 138.2 us with 8, 138.5
// with 4, 142 with 3, 146 with 2, 150 with 1).
template <typename T>
constexpr float px_shift() {
  return std::is_same<T, __half>::value ? 13.f : 0.f;
}
template <typename T>
constexpr float px_rescale() {
  return std::is_same<T, __half>::value ? 15.f - px_shift<T>() : 8.f;
}

template <int DP, int NT, bool PAIR>
struct PX {
  static constexpr int NCH = DP / 64;
  static constexpr bool HALF = NT == 2;
  static constexpr int KB = HALF ? 64 : 128;       // keys per step
  static constexpr int UC = DP >= 128 ? 2 : 1;     // 64-column chunks per unit
  static constexpr int NU = NCH / UC;              // units per K or V step
  static constexpr int UROWS = PAIR ? 64 : KB;     // keys per unit
  static constexpr int CHUNK = UROWS * 64 * 2;     // a unit's rows x 64 columns
  static constexpr int UNIT = UC * CHUNK;
  static constexpr int U = HALF ? (DP == 64 ? 16 : 10) : PAIR ? 10 : DP == 256 ? 5 : 6;  // ring units
  static constexpr int WPT = HALF ? 4 : 8;         // softmax warps per tile
  static constexpr int WARPS = WPT * NT, THREADS = 32 * (WARPS + 2 + NT);
  static constexpr int XCH = HALF ? 0 : NT * 2 * 4 * 2 * 32 * 4;
  static constexpr int SMEM = NT * NCH * PX_CHUNK + U * UNIT + XCH + 512;
  // TMEM columns of tile t (step parity b)
  static constexpr int S(int t, int b) { return 128 * t + (HALF ? 64 * b : 0); }
  static constexpr int P(int t, int b) { return HALF ? S(t, b) : 128 * NT + 64 * t; }
  static constexpr int PLO = HALF ? 32 : 64;       // from P's first term to its second
  static constexpr int O(int t) { return 256 + DP * t; }
  static constexpr uint32_t COLS = O(NT - 1) + DP <= 256 ? 256 : 512;
  static_assert(O(NT - 1) + DP <= 512 && SMEM <= 232448 && (2 * U + 7 * NT + 2) * 8 + 4 <= 512, "fits the SM");
};
}  // namespace

template <typename T, int DP, int NT, bool PAIR>
__global__ void __launch_bounds__(PX<DP, NT, PAIR>::THREADS, 1)
    prefix_sm100_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                        const int perm_k, const int perm_v, const SplitParams p, const int D,
                        const int rtiles, const int cps, const int qvec) {
  using X = PX<DP, NT, PAIR>;
  static_assert(!PAIR || (DP == 256 && NT == 1), "a pair shares the columns of D 256");
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value, HALF = X::HALF;
  constexpr uint32_t IDESC_S = tc05::idesc_f16(kBF16, PAIR ? 256 : 128, X::KB, false);
  constexpr uint32_t IDESC_PV = tc05::idesc_f16(kBF16, PAIR ? 256 : 128, PAIR ? DP : 64 * X::UC, true);
  constexpr int NCH = X::NCH, U = X::U, NU = X::NU, UC = X::UC, KB = X::KB, ROWS = 128 * NT;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *sQ = smem;                            // tile t, chunk c at (t * NCH + c) * CHUNK
  uint8_t *sR = sQ + NT * NCH * PX_CHUNK;        // ring
  float *s_xch = reinterpret_cast<float *>(sR + U * X::UNIT);  // [parity][tile][quad][half][32]
  uint64_t *bars = reinterpret_cast<uint64_t *>(reinterpret_cast<uint8_t *>(s_xch) + X::XCH);
  // s_full, p_full, o_done: two per tile, by step parity, so that none can complete a
  // second time before the first was seen
  uint64_t *r_full = bars, *r_empty = bars + U, *s_full = bars + 2 * U, *p_full = s_full + 2 * NT,
           *o_done = p_full + 2 * NT, *s_empty = o_done + 2 * NT;
  uint64_t *go = s_empty + NT;                   // half steps: tile 1 may start
  uint64_t *q_full = go + 1;
  uint32_t *tmem_sh = reinterpret_cast<uint32_t *>(q_full + 1);

  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int item = PAIR ? blockIdx.x >> 1 : blockIdx.x, rank = PAIR ? blockIdx.x & 1 : 0;
  const int rt = item % rtiles, hk = item / rtiles;
  const int r0 = PAIR ? (2 * rt + rank) * ROWS : rt * ROWS;
  const int nkt = (p.nkeys + PX_KEYS - 1) / PX_KEYS;
  const int j0 = blockIdx.y * cps;
  // this CTA's keys, at least one by the launcher's choice of splits, in steps of KB
  const int nsteps = (min(p.nkeys, min(nkt, j0 + cps) * PX_KEYS) - j0 * PX_KEYS + KB - 1) / KB;
  const int split = p.split0 + blockIdx.y;
  // The swizzled layouts count on this alignment of the dynamic shared memory.
  if (smem_u32(smem) & 1023) {
    if (tid == 0) report(p.status, BSA_DEVERR_TIMEOUT);
    return;
  }

  if (warp == X::WARPS && tc05::elect_one()) {
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
    for (int s = 0; s < U; ++s) {
      mbar_init(&r_full[s], 1);
      mbar_init(&r_empty[s], NT);
    }
    for (int t = 0; t < NT; ++t) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&s_full[2 * t + b], 1);
        mbar_init(&p_full[2 * t + b], PAIR ? 2 * X::WPT : X::WPT);
        mbar_init(&o_done[2 * t + b], 1);
      }
      mbar_init(&s_empty[t], PAIR ? 2 * X::WPT : X::WPT);
    }
    mbar_init(go, 1);
    mbar_init(q_full, PAIR ? 2 * X::WARPS : X::WARPS);
    fence_mbar_init();
  }
  if (warp == X::WARPS + 1) {
    if constexpr (PAIR) {
      tc05::pair_alloc(tmem_sh, X::COLS);
    } else {
      tc05::alloc(tmem_sh, X::COLS);
      tc05::relinquish();
    }
  }
  // Ring sequence, in steps of NU units: K_0, K_1, V_0, K_2, V_1, ...: S of the next
  // step goes before PV of this one.  k_at, v_at: position of step j's K and V.
  auto k_at = [&](int j) { return (j == 0 ? 0 : 2 * j - 1) * NU; };
  auto v_at = [&](int j) { return (j + 1 < nsteps ? 2 * j + 2 : 2 * j + 1) * NU; };
  bool bad = false;  // a wait gave up
  auto load = [&](int x) {  // unit x of the sequence, by the producer warp
    const int s = x / NU, u = x % NU, sl = x % U;
    const bool isv = s > 0 && (s % 2 == 0 || s == 2 * nsteps - 1);
    const int j = s == 2 * nsteps - 1 ? nsteps - 1 : isv ? s / 2 - 1 : (s + 1) / 2;
    if (x >= U) bad |= !mbar_wait_warp(&r_empty[sl], ((x / U) - 1) & 1);
    if (tc05::elect_one()) {
      uint8_t *dst = sR + sl * X::UNIT;
      const int perm = isv ? perm_v : perm_k;
      if constexpr (PAIR) {  // this CTA's half of B, counted in the first CTA
        if (rank == 0) mbar_expect_tx(&r_full[sl], 2 * X::UNIT);
        const uint32_t bar = tc05::pair_first(&r_full[sl]);
        const int pr = perm & 3, ph = (perm >> 2) & 3;
        const int row = j0 * PX_KEYS + j * KB + 64 * (isv ? u : rank), col = 128 * (isv ? rank : u);
        for (int c = 0; c < UC; ++c)
          tc05::pair_tma_load_4d(dst + c * X::CHUNK, isv ? &tv : &tk, bar, col + 64 * c,
                                 pr == 1 ? row : ph == 1 ? hk : 0, pr == 2 ? row : ph == 2 ? hk : 0,
                                 pr == 3 ? row : ph == 3 ? hk : 0);
      } else {
        mbar_expect_tx(&r_full[sl], X::UNIT);
        for (int c = 0; c < UC; ++c)
          tma_load_rhb(dst + c * X::CHUNK, isv ? &tv : &tk, &r_full[sl], perm, 64 * (u * UC + c),
                       j0 * PX_KEYS + j * KB, hk, 0);
      }
    }
    __syncwarp();
  };
  const int units = 2 * nsteps * NU;
  // The ring's first fill goes out before anything else (in a pair, once the first CTA's
  // barriers stand), the query rows behind it: zeros past the rows and, for D 32, past the
  // columns; each lane finds one row's place (the divisions), then 16-byte loads, a row's
  // pieces side by side, all in flight.  (One load at a time, its place found before it, and
  // the fill behind them: 10 us of a CTA's 40.)
  if constexpr (PAIR) {
    tc05::fence_before();
    tc05::pair_sync();
  }
  if (warp == X::WARPS)
    for (int x = 0; x < min(U, units); ++x) load(x);
  constexpr int PCS = DP / 8, RPI = 32 / PCS, RW = ROWS / X::WARPS, IT = RW / RPI;
  static_assert(RW <= 32 && IT <= 16, "a row per lane, 64 registers");
  uint4 qu[IT];
  if (warp < X::WARPS) {
    const int mine = warp * RW + lane % RW, ch = lane % PCS;
    long long off = -1;
    if (r0 + mine < p.R) {
      int rb, rh, rtt;
      split_row(p, 0, hk, r0 + mine, rb, rh, rtt);
      off = rb * p.q_sb + rh * p.q_sh + rtt * p.q_sl;
    }
    const T *q = reinterpret_cast<const T *>(p.q) + ch * 8;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const long long at = __shfl_sync(0xffffffffu, off, i * RPI + lane / PCS);
      qu[i] = make_uint4(0, 0, 0, 0);
      if (at >= 0 && ch * 8 < D) {
        if (qvec) {
          qu[i] = *reinterpret_cast<const uint4 *>(q + at);
        } else {
          T *e = reinterpret_cast<T *>(&qu[i]);
#pragma unroll
          for (int x = 0; x < 8; ++x) e[x] = q[at + x];
        }
      }
    }
  }
  if constexpr (!PAIR) {
    tc05::fence_before();
    __syncthreads();
  }
  tc05::fence_after();
  const uint32_t tmem = *tmem_sh;
  if (warp == X::WARPS) {
    // ================= TMA producer
    for (int x = U; x < units; ++x) load(x);
    if constexpr (PAIR)  // the other CTA's commits arrive here: none may come after this CTA's end
      for (int x = max(0, units - U); x < units; ++x) bad |= !mbar_wait_warp(&r_empty[x % U], (x / U) & 1);
  } else if (warp > X::WARPS) {
    // ================= issuers: one warp per tile for S, one for every tile's PV.  The
    // whole warp runs the sequence, one elected lane (always the same) issues the products
    // and commits.
    const int t_s = warp - X::WARPS - 1;
    const bool is_s = t_s < NT;
    const uint32_t on = tc05::elect_one();
    const uint64_t dq = tc05::sdesc(smem_u32(sQ), 16, 1024);
    const uint32_t sR0 = smem_u32(sR);
    auto wait = [&](uint64_t *bar, uint32_t parity) {
      bad |= !mbar_wait_warp(bar, parity);
      tc05::fence_after();
    };
    auto mma = [&](uint32_t dst, uint64_t a, uint64_t b, uint32_t acc) {
      if constexpr (PAIR)
        tc05::pair_mma_if(on, dst, a, b, IDESC_S, acc);
      else
        tc05::mma_f16_if(on, dst, a, b, IDESC_S, acc);
    };
    auto commit = [&](uint64_t *bar) {
      if constexpr (PAIR)
        tc05::pair_commit_if(on, bar);
      else
        tc05::commit_if(on, bar);
    };
    // a unit is free once every tile's products on it are done (r_empty counts the tiles)
    auto issue_s = [&](int t, int j) {
      const int b = j & 1, n0 = k_at(j);
      const uint32_t ds = tc05::taddr(tmem, 0, b ? X::S(t, 1) : X::S(t, 0));
      for (int u = 0; u < NU; ++u) {
        const int sl = (n0 + u) % U;
        wait(&r_full[sl], ((n0 + u) / U) & 1);
        const uint64_t dk = tc05::sdesc(sR0 + sl * X::UNIT, 16, 1024);
        const uint64_t dqu = dq + (t * NCH + u * UC) * (PX_CHUNK >> 4);
#pragma unroll
        for (int c = 0; c < UC; ++c)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            mma(ds, dqu + c * (PX_CHUNK >> 4) + 2 * ks, dk + c * (X::CHUNK >> 4) + 2 * ks,
                (u > 0 || c > 0 || ks > 0) ? 1u : 0u);
        commit(&r_empty[sl]);
      }
      commit(&s_full[2 * t + b]);
    };
    auto issue_pv = [&](int t, int j) {
      const int b = j & 1, n0 = v_at(j);
      const uint32_t ap = tc05::taddr(tmem, 0, b ? X::P(t, 1) : X::P(t, 0));
      for (int u = 0; u < NU; ++u) {
        const int sl = (n0 + u) % U;
        wait(&r_full[sl], ((n0 + u) / U) & 1);
        const uint64_t dv = tc05::sdesc(sR0 + sl * X::UNIT, X::CHUNK, 1024);
#pragma unroll
        for (int term = 0; term < 2; ++term)
#pragma unroll
          for (int ks = 0; ks < X::UROWS / 16; ++ks)
            if constexpr (PAIR)  // units are halves of the keys, N all columns
              tc05::pair_mma_ts_if(on, tc05::taddr(tmem, 0, X::O(t)), ap + X::PLO * term + 32 * u + 8 * ks,
                                   dv + 128 * ks, IDESC_PV, (j > 0 || u > 0 || term > 0 || ks > 0) ? 1u : 0u);
            else
              tc05::mma_f16_ts_if(on, tc05::taddr(tmem, 0, X::O(t) + 64 * UC * u), ap + X::PLO * term + 8 * ks,
                                  dv + 128 * ks, IDESC_PV, (j > 0 || term > 0 || ks > 0) ? 1u : 0u);
        commit(&r_empty[sl]);
      }
      commit(&o_done[2 * t + b]);
    };
    if (is_s && rank == 0) wait(q_full, 0);
    if (rank != 0) {  // the first CTA of a pair issues for both
    } else if (is_s) {
      const int t = t_s;
      // Half steps: the tiles run half a step apart, so that the exponentials of one fall
      // between those of the other (the MUFU is half of a step when both wait for it).
      if (HALF && t == 1) wait(go, 0);
      for (int j = 0; j < nsteps; ++j) {
        // the columns of S_j: free once S_{j-1} has been read; with half steps, once
        // PV_{j-2}, whose P lies in them, is complete
        if (!HALF && j >= 1) wait(&s_empty[t], (j - 1) & 1);
        if (HALF && j >= 2) wait(&o_done[2 * t + (j & 1)], ((j - 2) >> 1) & 1);
        issue_s(t, j);
      }
    } else {
      for (int j = 0; j < nsteps; ++j)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          wait(&p_full[2 * t + (j & 1)], (j >> 1) & 1);
          issue_pv(t, j);
        }
    }
  } else {
    // ================= softmax
    // The query rows into the swizzled layout.
    {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int r = warp * RW + i * RPI + lane / PCS;
        *reinterpret_cast<uint4 *>(sQ + (r >> 7) * NCH * PX_CHUNK + swz(0, 128, r & 127, (lane % PCS) * 8)) = qu[i];
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          tc05::pair_arrive(tc05::pair_first(q_full));
        else
          tc05::mbar_arrive(q_full);
      }
    }
    const int t = warp / X::WPT, quad = warp & 3, hf = HALF ? 0 : (warp >> 2) & 1;
    const int r = t * 128 + quad * 32 + lane;    // row within the CTA
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    constexpr int OC = HALF ? DP : DP / 2;       // O columns of this thread
    const uint32_t to = tmem + lane_base + X::O(t) + hf * OC;
    const bool rows_here = r0 + t * 128 + quad * 32 < p.R;  // the warp has a row (warp-uniform)
    const int bar = 1 + t * 4 + quad;
    auto xch = [&](int par, int half) -> float & {
      return s_xch[(((par * NT + t) * 4 + quad) * 2 + half) * 32 + lane];
    };
    auto wait_pv = [&](int j) {
      bad |= !mbar_wait(&o_done[2 * t + (j & 1)], (j >> 1) & 1);
      tc05::fence_after();
    };
    uint64_t *const se = &s_empty[t], *const pf = &p_full[2 * t];
    const uint32_t se0 = PAIR ? tc05::pair_first(se) : 0, pf0 = PAIR ? tc05::pair_first(pf) : 0;
    auto arrive_s = [&] { PAIR ? tc05::pair_arrive(se0) : tc05::mbar_arrive(se); };
    auto arrive_p = [&](int b) { PAIR ? tc05::pair_arrive(pf0 + 8 * b) : tc05::mbar_arrive(pf + b); };
    float m_used = -INFINITY, l = 0.f;
    for (int j = 0; j < nsteps; ++j) {
      const uint32_t ts = tmem + lane_base + (j & 1 ? X::S(t, 1) : X::S(t, 0)) + 64 * hf;
      const uint32_t tp = tmem + lane_base + (j & 1 ? X::P(t, 1) : X::P(t, 0)) + 32 * hf;
      bad |= !mbar_wait(&s_full[2 * t + (j & 1)], (j >> 1) & 1);
      tc05::fence_after();
      if (!rows_here) {  // nothing to do but keep step; its P stays what it is
        __syncwarp();
        if (!HALF && j >= 1) wait_pv(j - 1);
        tc05::fence_before();
        __syncwarp();
        if (lane == 0) {
          if (!HALF) arrive_s();
          arrive_p(j & 1);
        }
        continue;
      }
      float s[64];
      tc05::ld32(ts, s);
      tc05::ld32(ts + 32, s + 32);
      tc05::wait_ld();
      if (!HALF) {
        tc05::fence_before();
        __syncwarp();
        if (lane == 0) arrive_s();
      }
      const int left = p.nkeys - j0 * PX_KEYS - j * KB - 64 * hf;  // keys of this thread's columns
      if (left < 64) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c >= left) s[c] = -INFINITY;
      }
      float mh = max64(s);
      if constexpr (!HALF) {
        xch(j & 1, hf) = mh;
        named_bar_sync(bar, 64);
        mh = fmaxf(mh, xch(j & 1, hf ^ 1));
      }
      const float mx = mh * p.scale2;
      bool need = false;
      float alpha = 1.f;
      if (mx > -INFINITY && (m_used == -INFINITY || mx > m_used + px_rescale<T>())) {
        alpha = m_used == -INFINITY ? 0.f : ex2(m_used - mx);
        m_used = mx;
        l *= alpha;
        need = true;
      }
      const float off = m_used == -INFINITY ? 0.f : px_shift<T>() - m_used;
      const float2 sc2 = make_float2(p.scale2, p.scale2), of2 = make_float2(off, off);
      uint32_t w[32], w2[32];  // the two terms of P
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < 64; c += 2) {
        const float2 x = fma2(make_float2(s[c], s[c + 1]), sc2, of2);
        const float2 e = make_float2(ex2(x.x), ex2(x.y));
        sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], e);
        split2<T>(e.x, e.y, w[c >> 1], w2[c >> 1]);
      }
      const float2 st = add2(sum[0], sum[1]);
      l += st.x + st.y;
      if (HALF && j == 0 && warp == 0 && lane == 0) tc05::mbar_arrive(go);
      const bool rescale = __any_sync(0xffffffffu, need) && j >= 1;
      // PV of the step before: has read its P (one P buffer), and O may be rescaled
      if (j >= 1 && (!HALF || rescale)) wait_pv(j - 1);
      if (rescale) {
#pragma unroll 1
        for (int c = 0; c < OC; c += 32) {
          float o[32];
          tc05::ld32(to + c, o);
          tc05::wait_ld();
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] *= alpha;
          tc05::st32(to + c, o);
        }
        tc05::wait_st();
      }
      tc05::st32(tp, reinterpret_cast<const float *>(w));
      tc05::st32(tp + X::PLO, reinterpret_cast<const float *>(w2));
      tc05::wait_st();
      tc05::fence_before();
      __syncwarp();
      if (lane == 0) arrive_p(j & 1);
    }
    // ---- (m, l) and the unnormalised O of this split
    wait_pv(nsteps - 1);
    if (rows_here) {
      if constexpr (!HALF) {  // past the last PV both halves have read the last maxima
        xch(nsteps & 1, hf) = l;
        named_bar_sync(bar, 64);
        l += xch(nsteps & 1, hf ^ 1);
      }
      const bool live = r0 + r < p.R;
      long long at = 0;
      if (live) {
        int rb, rh, rtt;
        at = (long long)split * p.rows + split_row(p, 0, hk, r0 + r, rb, rh, rtt);
        // a NaN sum with no maximum (every logit NaN) must not read as an empty row
        if (hf == 0) p.pml[at] = make_float2(m_used == -INFINITY && isnan(l) ? l : m_used - px_shift<T>(), l);
      }
      // O through shared memory, whose tiles have been read (this tile's queries; with one
      // tile, the ring too): 32 columns of 32 rows, so that a store covers 128 bytes of a
      // row (16 bytes of 32 rows each: 6 us for 128 KB)
      uint8_t *stage = HALF ? sQ + t * NCH * PX_CHUNK + quad * 4096 : sQ + warp * 4096;
      if (!live) at = -1;
#pragma unroll 1
      for (int c = 0; c < OC; c += 32) {
        float o[32];
        tc05::ld32(to + c, o);
        tc05::wait_ld();
        if (hf * OC + c >= D) break;
#pragma unroll
        for (int x = 0; x < 8; ++x)
          *reinterpret_cast<float4 *>(stage + lane * 128 + ((x ^ (lane & 7)) << 4)) =
              make_float4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = i * 4 + (lane >> 3), x = lane & 7;
          const long long a = __shfl_sync(0xffffffffu, at, row);
          if (a >= 0)
            *reinterpret_cast<float4 *>(p.po + a * D + hf * OC + c + 4 * x) =
                *reinterpret_cast<const float4 *>(stage + row * 128 + ((x ^ (row & 7)) << 4));
        }
        __syncwarp();
      }
    }
  }
  if (bad) report(p.status, BSA_DEVERR_TIMEOUT);
  tc05::fence_before();
  if constexpr (PAIR)
    tc05::pair_sync();  // neither leaves while the products read its tiles
  else
    __syncthreads();
  if (warp == X::WARPS + 1) {
    tc05::fence_after();
    if constexpr (PAIR)
      tc05::pair_dealloc(tmem, X::COLS);
    else
      tc05::dealloc(tmem, X::COLS);
  }
}

namespace {
// Row tiles of 128 or 256, and the splits of the prefix (an SM each, or two for a pair).
// The kernel that reads the sequences' own slots starts on the SMs that this one leaves
// free, so fewer splits than fill the SMs can be the faster whole.  The split is the one of
// the least estimate, from measured times: a CTA's key tile (all 148 SMs busy, us, bf16 and
// f16: one row tile D 32 1.2, D 64 1.3, D 128 1.3, D 256 2.6; two row tiles D 32 2.0, D 64
// 2.1, D 128 2.4; a pair 2.1) and its start and end; own slots at 19.5 GB/s per CTA beside
// this kernel, two per SM up to D 128; what does not fit beside it comes after, never in less
// than most of a CTA's time; the join reads and writes 8 bytes per row, column and split.
// Lengths are not known here: half of the capacity is assumed.  Only speed hangs on any of
// it.  Measured at two shapes, us: 32768 keys, 512 rows of 8 heads, D 128, 128 sequences of
// up to 1024 slots: 4, 5, 6, 7, 8 splits 163, 140, 126, 129, 133; 65536 keys, 256 rows of 2
// heads, D 256, 32 of up to 512: 26, 28, 31, 32, 37 splits 57, 56, 53, 54, 62.
void prefix_shape(const bsa_decode_prefix_args *a, int &nt, bool &pair, int &rtiles, int &cps, int &nsplit) {
  const int R = a->B * (a->Hq / a->Hkv) * a->T;
  nt = a->D <= 128 && R > 128 ? 2 : 1;
  pair = a->D == 256 && R > 128;
  const int sms = pair ? 2 : 1;  // of one CTA or pair
  rtiles = (R + 128 * nt * sms - 1) / (128 * nt * sms);
  const long long items = (long long)a->Hkv * rtiles, nkt = (a->P + PX_KEYS - 1) / PX_KEYS;
  const double tile = pair ? 2.1 : nt == 2 ? (a->D == 128 ? 2.4 : 2.1) : a->D == 256 ? 2.6 : 1.3;  // us
  const double ends = pair ? 9 : 5;
  const double cta = (double)a->S * a->D * 2 / 19.5e3;                          // of one sequence and head
  const double own = (double)a->B * a->Hkv * cta / (a->D == 256 ? 1 : 2);       // SM time
  const double join = (double)a->Hkv * R * a->D * 8 / 5e6;                      // per split
  double best = -1;
  cps = (int)nkt;
  for (long long s = 1; s <= nkt && s <= 148; ++s) {
    const long long c = (nkt + s - 1) / s, ns = (nkt + c - 1) / c, busy = items * ns * sms;
    const double one = (double)((busy + 147) / 148) * (c * tile + ends);
    const double beside = busy < 148 ? (148 - busy) * one : 0;
    const double after = own <= beside ? 0 : std::max((own - beside) / 148, 0.75 * cta);
    const double cost = one + after + ns * join;
    if (best < 0 || cost < best) {
      best = cost;
      cps = (int)c;
    }
  }
  nsplit = (int)((nkt + cps - 1) / cps);
}
}  // namespace

// Whether the tcgen05 kernel takes this prefix: 16-bit types, rows for more than one
// mma.sync row tile, and K/V strides that a TMA map can hold.
bool prefix_sm100_applicable(const bsa_decode_prefix_args *a) {
  if (a->dtype == BSA_F32 || a->P < PX_KEYS) return false;
  const long long R = (long long)a->B * (a->Hq / a->Hkv) * a->T;
  if (R <= 16) return false;
  for (const bsa_view *v : {&a->pk, &a->pv})
    if ((a->P > 1 && v->sl <= 0) || (a->Hkv > 1 && v->sh <= 0)) return false;
  return true;
}

int prefix_sm100_splits(const bsa_decode_prefix_args *a, int &left) {
  int nt, rtiles, cps, ns;
  bool pair;
  prefix_shape(a, nt, pair, rtiles, cps, ns);
  const long long busy = (long long)a->Hkv * rtiles * ns * (pair ? 2 : 1);
  left = busy < 148 ? 148 - (int)busy : 148;
  return ns;
}

bsa_status launch_prefix_sm100(const bsa_decode_prefix_args *a, const SplitParams &p, cudaStream_t st) {
  int nt, rtiles, cps, ns;
  bool pair;
  prefix_shape(a, nt, pair, rtiles, cps, ns);
  const int rows = nt == 2 || pair ? 64 : 128;  // keys per unit
  TensorMap4 mk, mv;
  bsa_status s;
  if ((s = make_tmap(&mk, a->pk.ptr, a->dtype, 1, a->Hkv, a->P, a->D, 0, a->pk.sh, a->pk.sl, rows, "pk"))) return s;
  if ((s = make_tmap(&mv, a->pv.ptr, a->dtype, 1, a->Hkv, a->P, a->D, 0, a->pv.sh, a->pv.sl, rows, "pv"))) return s;
  auto pk = [](const TensorMap4 &m) { return m.perm[0] | (m.perm[1] << 2) | (m.perm[2] << 4); };
  const int qvec = reinterpret_cast<uintptr_t>(a->q.ptr) % 16 == 0 && a->q.sb % 8 == 0 && a->q.sh % 8 == 0 &&
                   a->q.sl % 8 == 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a->Hkv * rtiles * (pair ? 2 : 1)), ns);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 2, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = pair ? 1 : 0;
#define BSA_PX(T_, D_, N_, P_)                                                                        \
  {                                                                                                   \
    auto kern = prefix_sm100_kernel<T_, D_, N_, P_>;                                                  \
    static std::atomic<uint64_t> done{0};                                                             \
    allow_smem(reinterpret_cast<const void *>(kern), PX<D_, N_, P_>::SMEM, done);                     \
    cfg.blockDim = dim3(PX<D_, N_, P_>::THREADS);                                                     \
    cfg.dynamicSmemBytes = PX<D_, N_, P_>::SMEM;                                                      \
    cudaLaunchKernelEx(&cfg, kern, mk.map, mv.map, pk(mk), pk(mv), p, (int)a->D, rtiles, cps, qvec);  \
  }
#define BSA_PX_D(T_)                                                        \
  if (a->D <= 64) {                                                         \
    if (nt == 2) BSA_PX(T_, 64, 2, false) else BSA_PX(T_, 64, 1, false)     \
  } else if (a->D == 128) {                                                 \
    if (nt == 2) BSA_PX(T_, 128, 2, false) else BSA_PX(T_, 128, 1, false)   \
  } else if (pair)                                                          \
    BSA_PX(T_, 256, 1, true)                                                \
  else                                                                      \
    BSA_PX(T_, 256, 1, false)
  if (a->dtype == BSA_BF16) {
    BSA_PX_D(__nv_bfloat16)
  } else {
    BSA_PX_D(__half)
  }
#undef BSA_PX_D
#undef BSA_PX
  return check_launch("prefix_sm100");
}

}  // namespace bsa
