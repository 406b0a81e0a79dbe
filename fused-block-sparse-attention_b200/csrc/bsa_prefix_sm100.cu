// Shared-prefix decode on tcgen05: the query rows of the whole batch that read one
// K/V head (B * grp * T of them) as M = 128 tiles over one split of the prefix.
//
//   S = Q K^T, P = 2^(S * scale * log2e - m), O += P V   per 128 prefix keys,
// with K, V through shared memory by TMA, S, P and O in TMEM, and (m, l, O) of the
// split left in fp32 for split_join_kernel.  Unlike the sequence forward, a row tile
// gathers its rows from different sequences, every key is visible to every row, and
// the keys are split so that all SMs work on few rows.
//
// NT = 2 (D 64, 128; more than 128 rows): one CTA owns two row tiles that share every
// K/V tile: half the shared-memory fill per product, which at one tile per CTA is the
// bound (64 KB of K/V per 128 x 128 step at D 128: the SMs drain L2).  Four softmax
// warps per tile, one row per thread; P overlays its tile's S, so S of the next step
// is issued once PV of this one is complete, while the other tile's softmax runs.
// NT = 1 (up to 128 rows, or D 256, whose O fills TMEM): eight softmax warps, half a
// row per thread; S, P and O in separate columns, S of the next step under the
// exponentials of this one.
//
// Warps 0-7 softmax, 8 TMA producer, 9 TMEM owner and MMA issuer.  K/V tiles move as
// 64-column chunks (16 KB) through one ring in the order the products use them.
// Every wait is bounded; a timeout sets BSA_DEVERR_TIMEOUT and the CTA runs on.
#include <type_traits>

#include "bsa_host.h"
#include "bsa_split.cuh"
#include "bsa_tc05.cuh"

namespace bsa {

namespace {
constexpr int PX_KEYS = 128;
constexpr int PX_TILE = PX_KEYS * 64 * 2;  // 16 KB chunk: 128 rows x 64 columns
constexpr int PX_WPROD = 8, PX_WMMA = 9, PX_THREADS = 320;
constexpr float PX_RESCALE = 8.f;          // log2 units

template <int DP, int NT>
struct PX {
  static constexpr int NCH = DP / 64;
  static constexpr int NSL = DP == 256 ? 9 : DP == 128 ? (NT == 2 ? 9 : 11) : (NT == 2 ? 11 : 12);
  static constexpr int SMEM = 1024 + NT * NCH * PX_TILE + NSL * PX_TILE;
  // TMEM columns
  static constexpr int S(int t) { return NT == 2 ? 128 * t : 0; }
  static constexpr int P(int t) { return NT == 2 ? 128 * t : 128; }
  static constexpr int O(int t) { return NT == 2 ? 256 + DP * t : 192; }
  static constexpr uint32_t COLS = DP == 64 && NT == 1 ? 256 : 512;
};
}  // namespace

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(PX_THREADS, 1)
    prefix_sm100_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                        const int perm_k, const int perm_v, const SplitParams p, const int D,
                        const int rtiles, const int cps, const int qvec) {
  using X = PX<DP, NT>;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_S = tc05::idesc_f16(kBF16, 128, 128, false);
  constexpr uint32_t IDESC_PV = tc05::idesc_f16(kBF16, 128, 64, true);
  constexpr int NCH = X::NCH, NSL = X::NSL, ROWS = 128 * NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem;                            // tile t, chunk c at (t * NCH + c) * TILE
  uint8_t *sR = sQ + NT * NCH * PX_TILE;
  __shared__ __align__(8) uint64_t r_full[NSL], r_empty[NSL], s_full[NT], s_empty, p_full[NT], o_done[NT];
  __shared__ uint32_t tmem_base_sh;
  __shared__ float s_xch[3][4][2][32];           // NT = 1: half-row maxima (by step parity), row sums

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rt = blockIdx.x % rtiles, hk = blockIdx.x / rtiles;
  const int r0 = rt * ROWS;
  const int nkt = (p.nkeys + PX_KEYS - 1) / PX_KEYS;
  const int j0 = blockIdx.y * cps;
  const int nsteps = min(nkt, j0 + cps) - j0;    // >= 1 by the launcher's choice of splits
  const int split = p.split0 + blockIdx.y;

  if (tid == 0) {
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
    for (int s = 0; s < NSL; ++s) {
      mbar_init(&r_full[s], 1);
      mbar_init(&r_empty[s], 1);
    }
    for (int t = 0; t < NT; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 8 / NT);
      mbar_init(&o_done[t], 1);
    }
    mbar_init(&s_empty, 8);
    fence_mbar_init();
  }
  if (warp == PX_WMMA) {
    tc05::alloc(&tmem_base_sh, X::COLS);
    tc05::relinquish();
  }
  // query rows of this tile, 16 bytes at a time into the swizzled layout; zeros past
  // the rows and, for D 32, past the columns
  for (int i = tid; i < ROWS * (DP / 8); i += PX_THREADS) {
    const int r = i / (DP / 8), ch = i % (DP / 8);
    uint4 u = make_uint4(0, 0, 0, 0);
    if (r0 + r < p.R && ch * 8 < D) {
      int rb, rh, rtt;
      split_row(p, 0, hk, r0 + r, rb, rh, rtt);
      const T *qp = reinterpret_cast<const T *>(p.q) + rb * p.q_sb + rh * p.q_sh + rtt * p.q_sl + ch * 8;
      if (qvec) {
        u = *reinterpret_cast<const uint4 *>(qp);
      } else {
        T *e = reinterpret_cast<T *>(&u);
#pragma unroll
        for (int x = 0; x < 8; ++x) e[x] = qp[x];
      }
    }
    *reinterpret_cast<uint4 *>(sQ + (r >> 7) * NCH * PX_TILE + swz(0, 128, r & 127, ch * 8)) = u;
  }
  fence_proxy_async_smem();
  tc05::fence_before();
  __syncthreads();
  tc05::fence_after();
  const uint32_t tmem = tmem_base_sh;

  // Ring sequence.  NT = 2: K_0, V_0, K_1, V_1, ...; NT = 1: K_0, K_1, V_0, K_2, V_1, ...
  // (S of the next step goes before PV of this one).
  if (warp == PX_WPROD) {
    int n = 0;
    auto load = [&](bool isv, int j) {
      for (int c = 0; c < NCH; ++c, ++n) {
        const int sl = n % NSL;
        if (n >= NSL && !mbar_wait_warp(&r_empty[sl], ((n / NSL) - 1) & 1)) report(p.status, BSA_DEVERR_TIMEOUT);
        if (tc05::elect_one()) {
          mbar_expect_tx(&r_full[sl], PX_TILE);
          tma_load_rhb(sR + sl * PX_TILE, isv ? &tv : &tk, &r_full[sl], isv ? perm_v : perm_k, 64 * c,
                       (j0 + j) * PX_KEYS, hk, 0);
        }
        __syncwarp();
      }
    };
    load(false, 0);
    for (int j = 0; j < nsteps; ++j) {
      if (NT == 1 && j + 1 < nsteps) load(false, j + 1);
      load(true, j);
      if (NT == 2 && j + 1 < nsteps) load(false, j + 1);
    }
  } else if (warp == PX_WMMA) {
    const uint64_t dq = tc05::sdesc(smem_u32(sQ), 16, 1024);
    // S of tile t from the K tile at ring position n0; frees the chunks when `last`
    auto issue_s = [&](int t, int n0, bool last) {
      for (int c = 0; c < NCH; ++c) {
        const int n = n0 + c, sl = n % NSL;
        if (!mbar_wait_warp(&r_full[sl], (n / NSL) & 1)) report(p.status, BSA_DEVERR_TIMEOUT);
        tc05::fence_after();
        const uint64_t dk = tc05::sdesc(smem_u32(sR + sl * PX_TILE), 16, 1024);
        const uint64_t dqc = dq + (t * NCH + c) * (PX_TILE >> 4);
        if (tc05::elect_one()) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            tc05::mma_f16(tc05::taddr(tmem, 0, X::S(t)), dqc + 2 * ks, dk + 2 * ks, IDESC_S,
                          (c > 0 || ks > 0) ? 1u : 0u);
          if (last) tc05::commit(&r_empty[sl]);
        }
        __syncwarp();
      }
      if (tc05::elect_one()) tc05::commit(&s_full[t]);
      __syncwarp();
    };
    auto issue_pv = [&](int t, int n0, int j, bool last) {
      for (int c = 0; c < NCH; ++c) {
        const int n = n0 + c, sl = n % NSL;
        if (!mbar_wait_warp(&r_full[sl], (n / NSL) & 1)) report(p.status, BSA_DEVERR_TIMEOUT);
        tc05::fence_after();
        const uint64_t dv = tc05::sdesc(smem_u32(sR + sl * PX_TILE), PX_TILE, 1024);
        if (tc05::elect_one()) {
#pragma unroll
          for (int ks = 0; ks < PX_KEYS / 16; ++ks)
            tc05::mma_f16_ts(tc05::taddr(tmem, 0, X::O(t) + 64 * c), tc05::taddr(tmem, 0, X::P(t) + 8 * ks),
                             dv + 128 * ks, IDESC_PV, (j > 0 || ks > 0) ? 1u : 0u);
          if (last) tc05::commit(&r_empty[sl]);
        }
        __syncwarp();
      }
      if (tc05::elect_one()) tc05::commit(&o_done[t]);
      __syncwarp();
    };
    if constexpr (NT == 2) {
      issue_s(0, 0, false);
      issue_s(1, 0, true);
      for (int j = 0; j < nsteps; ++j) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!mbar_wait_warp(&p_full[t], j & 1)) report(p.status, BSA_DEVERR_TIMEOUT);
          tc05::fence_after();
          issue_pv(t, (2 * j + 1) * NCH, j, t == 1);
          if (j + 1 < nsteps) {
            // P shares its columns with S: its readers must be done
            if (!mbar_wait_warp(&o_done[t], j & 1)) report(p.status, BSA_DEVERR_TIMEOUT);
            tc05::fence_after();
            issue_s(t, (2 * j + 2) * NCH, t == 1);
          }
        }
      }
    } else {
      // ring position of K_j: 0 for j = 0, else (2j - 1) * NCH; V_j: (2j + 2) * NCH, and
      // one tile earlier for the last step (no K follows)
      issue_s(0, 0, true);
      for (int j = 0; j < nsteps; ++j) {
        if (j + 1 < nsteps) {
          if (!mbar_wait_warp(&s_empty, j & 1)) report(p.status, BSA_DEVERR_TIMEOUT);
          tc05::fence_after();
          issue_s(0, (2 * j + 1) * NCH, true);
        }
        if (!mbar_wait_warp(&p_full[0], j & 1)) report(p.status, BSA_DEVERR_TIMEOUT);
        tc05::fence_after();
        issue_pv(0, (j + 1 < nsteps ? 2 * j + 2 : 2 * j + 1) * NCH, j, true);
      }
    }
  } else {
    // ================= softmax
    constexpr int W = 128 * NT / 2;              // columns per thread: 128 or 64
    const int quad = warp & 3, up = warp >> 2;   // up: the tile (NT = 2) or the half row
    const int t = NT == 2 ? up : 0, hf = NT == 2 ? 0 : up;
    const int r = t * 128 + quad * 32 + lane;    // row within the CTA
    const int cb = W * hf;
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const uint32_t ts = tmem + lane_base + X::S(t) + cb, tp = tmem + lane_base + X::P(t) + cb / 2;
    const uint32_t to = tmem + lane_base + X::O(t);
    constexpr int OC = NT == 2 ? DP : DP / 2;    // O columns of this thread
    const bool rows_here = r0 + t * 128 + quad * 32 < p.R;  // the warp has a row (warp-uniform)
    float m_used = -INFINITY, l = 0.f;
    for (int j = 0; j < nsteps; ++j) {
      if (!mbar_wait(&s_full[t], j & 1)) report(p.status, BSA_DEVERR_TIMEOUT);
      tc05::fence_after();
      if (!rows_here) {  // nothing to do but keep step; its P stays what it is
        __syncwarp();
        if (NT == 1 && j >= 1 && !mbar_wait(&o_done[0], (j - 1) & 1)) report(p.status, BSA_DEVERR_TIMEOUT);
        tc05::fence_before();
        __syncwarp();
        if (lane == 0) {
          if (NT == 1) tc05::mbar_arrive(&s_empty);
          tc05::mbar_arrive(&p_full[t]);
        }
        continue;
      }
      float s[W];
#pragma unroll
      for (int c = 0; c < W; c += 32) tc05::ld32(ts + c, s + c);
      tc05::wait_ld();
      if (NT == 1) {
        tc05::fence_before();
        __syncwarp();
        if (lane == 0) tc05::mbar_arrive(&s_empty);
      }
      const int left = p.nkeys - (j0 + j) * PX_KEYS - cb;  // keys of this thread's columns
      if (left < W) {
#pragma unroll
        for (int c = 0; c < W; ++c)
          if (c >= left) s[c] = -INFINITY;
      }
      float mr = max64(s);
      if constexpr (NT == 2) {
        mr = fmaxf(mr, max64(s + W / 2));
      } else {
        s_xch[j & 1][quad][hf][lane] = mr;
        named_bar_sync(1 + quad, 64);
        mr = fmaxf(mr, s_xch[j & 1][quad][hf ^ 1][lane]);
      }
      const float mx = mr * p.scale2;
      bool need = false;
      float alpha = 1.f;
      if (mx > -INFINITY && (m_used == -INFINITY || mx > m_used + PX_RESCALE)) {
        alpha = m_used == -INFINITY ? 0.f : ex2(m_used - mx);
        m_used = mx;
        l *= alpha;
        need = true;
      }
      const float off = m_used == -INFINITY ? 0.f : -m_used;
      const float2 sc2 = make_float2(p.scale2, p.scale2), of2 = make_float2(off, off);
      uint32_t w[W / 2];
      float2 sum[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < W; c += 2) {
        const float2 x = fma2(make_float2(s[c], s[c + 1]), sc2, of2);
        const float2 e = make_float2(ex2(x.x), ex2(x.y));
        sum[(c >> 1) & 3] = add2(sum[(c >> 1) & 3], e);
        w[c >> 1] = Mma<T>::pack(e.x, e.y);
      }
      const float2 st = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
      l += st.x + st.y;
      if (NT == 1 && j >= 1) {  // PV of the step before has read its P (and O may be rescaled)
        if (!mbar_wait(&o_done[0], (j - 1) & 1)) report(p.status, BSA_DEVERR_TIMEOUT);
        tc05::fence_after();
      }
      if (__any_sync(0xffffffffu, need) && j >= 1) {
#pragma unroll 1
        for (int c = 0; c < OC; c += 32) {
          float o[32];
          tc05::ld32(to + hf * OC + c, o);
          tc05::wait_ld();
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] *= alpha;
          tc05::st32(to + hf * OC + c, o);
        }
        tc05::wait_st();
      }
#pragma unroll
      for (int c = 0; c < W / 2; c += 32) tc05::st32(tp + c, reinterpret_cast<const float *>(w) + c);
      tc05::wait_st();
      tc05::fence_before();
      __syncwarp();
      if (lane == 0) tc05::mbar_arrive(&p_full[t]);
    }
    // ---- (m, l) and the unnormalised O of this split
    if (NT == 1 && rows_here) {
      s_xch[2][quad][hf][lane] = l;
      named_bar_sync(1 + quad, 64);
      l += s_xch[2][quad][hf ^ 1][lane];
    }
    if (!mbar_wait(&o_done[t], (nsteps - 1) & 1)) report(p.status, BSA_DEVERR_TIMEOUT);
    tc05::fence_after();
    const bool live = r0 + r < p.R;
    long long at = 0;
    if (live) {
      int rb, rh, rtt;
      at = (long long)split * p.rows + split_row(p, 0, hk, r0 + r, rb, rh, rtt);
      // a NaN sum with no maximum (every logit NaN) must not read as an empty row
      if (hf == 0) p.pml[at] = make_float2(m_used == -INFINITY && isnan(l) ? l : m_used, l);
    }
    if (rows_here) {
#pragma unroll 1
      for (int c = 0; c < OC; c += 32) {
        float o[32];
        tc05::ld32(to + hf * OC + c, o);
        tc05::wait_ld();
        if (live && hf * OC + c < D) {
          float *op = p.po + at * D + hf * OC + c;
#pragma unroll
          for (int x = 0; x < 32; x += 4)
            *reinterpret_cast<float4 *>(op + x) = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
        }
      }
    }
  }
  tc05::fence_before();
  __syncthreads();
  if (warp == PX_WMMA) {
    tc05::fence_after();
    tc05::dealloc(tmem, X::COLS);
  }
}

namespace {
// Row tiles of 128 or 256, and the splits of the prefix that fill the SMs (one CTA each).
void prefix_shape(int D, int Hkv, int R, int P, int &nt, int &rtiles, int &cps, int &nsplit) {
  nt = D <= 128 && R > 128 ? 2 : 1;
  rtiles = (R + 128 * nt - 1) / (128 * nt);
  const long long items = (long long)Hkv * rtiles, nkt = (P + PX_KEYS - 1) / PX_KEYS;
  const int fixed = 3;  // prologue, first fill and epilogue of a CTA, in key tiles
  long long best = -1;
  cps = (int)nkt;
  for (long long s = 1; s <= nkt && s <= 148; ++s) {
    const long long c = (nkt + s - 1) / s, ns = (nkt + c - 1) / c;
    const long long cost = ((items * ns + 147) / 148) * (c + fixed);
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

int prefix_sm100_splits(const bsa_decode_prefix_args *a) {
  int nt, rtiles, cps, ns;
  prefix_shape(a->D, a->Hkv, a->B * (a->Hq / a->Hkv) * a->T, a->P, nt, rtiles, cps, ns);
  return ns;
}

bsa_status launch_prefix_sm100(const bsa_decode_prefix_args *a, const SplitParams &p, cudaStream_t st) {
  TensorMap4 mk, mv;
  bsa_status s;
  if ((s = make_tmap(&mk, a->pk.ptr, a->dtype, 1, a->Hkv, a->P, a->D, 0, a->pk.sh, a->pk.sl, 128, "pk"))) return s;
  if ((s = make_tmap(&mv, a->pv.ptr, a->dtype, 1, a->Hkv, a->P, a->D, 0, a->pv.sh, a->pv.sl, 128, "pv"))) return s;
  auto pk = [](const TensorMap4 &m) { return m.perm[0] | (m.perm[1] << 2) | (m.perm[2] << 4); };
  int nt, rtiles, cps, ns;
  prefix_shape(a->D, a->Hkv, p.R, a->P, nt, rtiles, cps, ns);
  const int qvec = reinterpret_cast<uintptr_t>(a->q.ptr) % 16 == 0 && a->q.sb % 8 == 0 && a->q.sh % 8 == 0 &&
                   a->q.sl % 8 == 0;
  const dim3 grid((unsigned)(a->Hkv * rtiles), ns);
#define BSA_PX(T_, D_, N_)                                                                              \
  {                                                                                                     \
    auto kern = prefix_sm100_kernel<T_, D_, N_>;                                                        \
    static_assert(PX<D_, N_>::SMEM <= 231000, "shared memory of one CTA");                              \
    static std::atomic<uint64_t> done{0};                                                               \
    allow_smem(reinterpret_cast<const void *>(kern), PX<D_, N_>::SMEM, done);                           \
    kern<<<grid, PX_THREADS, PX<D_, N_>::SMEM, st>>>(mk.map, mv.map, pk(mk), pk(mv), p, a->D, rtiles,   \
                                                     cps, qvec);                                        \
  }
#define BSA_PX_D(T_)                             \
  if (a->D <= 64) {                              \
    if (nt == 2) BSA_PX(T_, 64, 2) else BSA_PX(T_, 64, 1)     \
  } else if (a->D == 128) {                      \
    if (nt == 2) BSA_PX(T_, 128, 2) else BSA_PX(T_, 128, 1)   \
  } else                                         \
    BSA_PX(T_, 256, 1)
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
