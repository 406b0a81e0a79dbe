// Reduction of a K/V cache to a budget of slots by accumulated attention weight.
//
// Of the L slots of each (batch, K/V head) the `budget` best survive: protected
// slots first (the first `sink` and the last `recent` token positions), then by
// weight, ties to the lower slot.  Survivors below the budget keep their slot; the
// others fill the freed slots, both in ascending order.  That moves the fewest
// rows, and since every source is >= budget and every destination below it, the
// moves run in place in any order.
//
//   evict_pick_kernel  a cluster of CTAs per (b, head), each with its share of the
//                      slots: the key of the budget-th best slot by a radix search
//                      (11 + 11 + 10 bits, histograms summed over the cluster), then
//                      the lists of freed slots and of sources by prefix counts
//   evict_move_kernel  CTA per (b, head, block of slots): moves rows, weights and
//                      positions, and pools the min / max of a changed block while
//                      its rows pass through registers
// Bound by HBM for a large cut (rows moved) and by latency for a single slot.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "bsa_common.cuh"
#include "bsa_host.h"

namespace cg = cooperative_groups;

namespace bsa {

namespace {
constexpr int kPickThreads = 1024;
constexpr int kBins = 2048;

struct EvictWork {
  int *hole, *tail;  // [B*Hkv][m_cap]
  int *off;          // [B*Hkv][nblk + 1]: freed slots before each block
  int m_cap, nblk;
};

// Monotone 32-bit key: protected slots above everything, NaN with -infinity below.
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int sink, int first_recent) {
  if (pos < sink || pos >= first_recent) return 0xffffffffu;
  if (isnan(w)) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 becomes +0
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix over the 32 warps of one count per warp (the same in all its
// lanes) and the total over the CTA; s: 32 ints of its own, one barrier.
__device__ __forceinline__ int warp_prefix(int v, int *s, int *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) s[warp] = v;
  __syncthreads();
  const int mine = s[lane];
  int x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  *total = __shfl_sync(0xffffffffu, x, 31);
  return __shfl_sync(0xffffffffu, x - mine, warp);
}
}  // namespace

// Exclusive prefix over the lanes of a warp, and its total.
__device__ __forceinline__ int lane_prefix(int v, int *total) {
  const int lane = threadIdx.x & 31;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  *total = __shfl_sync(0xffffffffu, x, 31);
  return x - v;
}

// Lane l of warp w owns IPT consecutive slots of each of `groups` runs of 32 * IPT, so a
// rank is a bit count in the lane, one prefix over the lanes and one over the warps, not
// a ballot per row of 32 slots.  groups == 1: the keys stay in registers (up to 8 * 1024
// * 16 slots per head); more: they are read again in every pass, for any length.
template <int IPT>
__global__ void __launch_bounds__(kPickThreads)
    evict_pick_kernel(const bsa_evict_args a, const EvictWork w, const int groups, const int vec) {
  cg::cluster_group cl = cg::this_cluster();
  const int nc = cl.num_blocks(), rank = cl.block_rank();
  const int bh = blockIdx.x / nc, b = bh / a.Hkv, h = bh % a.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_trigger();
  __shared__ int hist[3][kBins];
  __shared__ int s_scan[6][32];
  __shared__ int s_bin[3], s_need[3], s_cnt[3];
  const float *wt = a.weight + b * a.w_sb + h * a.w_sh;
  const int32_t *ps = a.pos + b * a.p_sb + h * a.p_sh;
  const int first_recent = a.seen - a.recent;
  const bool guards = a.sink > 0 || a.recent > 0;
  const long long first = (long long)(rank * 32 + warp) * groups * (32 * IPT);  // this warp's first slot
  uint32_t kr[IPT];
  int base = 0;  // this lane's first slot of the group; slots past L get key 0, below every real one
  auto load = [&](int g) {
    base = (int)min(first + (long long)g * (32 * IPT) + lane * IPT, (long long)a.L);
    if (vec && base + IPT <= a.L) {
      float4 x[IPT / 4];
      int4 y[IPT / 4];
#pragma unroll
      for (int i = 0; i < IPT / 4; ++i) {
        x[i] = __ldg(reinterpret_cast<const float4 *>(wt + base) + i);
        y[i] = guards ? __ldg(reinterpret_cast<const int4 *>(ps + base) + i) : make_int4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < IPT; ++i)
        kr[i] = evict_key(reinterpret_cast<const float *>(x)[i], reinterpret_cast<const int *>(y)[i], a.sink,
                          guards ? first_recent : 1);
    } else {
#pragma unroll
      for (int i = 0; i < IPT; ++i) {
        const int s = base + i;
        kr[i] = s < a.L ? evict_key(__ldg(wt + s), guards ? __ldg(ps + s) : 0, a.sink, guards ? first_recent : 1)
                        : 0u;
      }
    }
  };
  // the lane's slots below `end`, as a bit mask
  auto below = [&](int end) { return (1u << min(max(end - base, 0), IPT)) - 1u; };
  auto sync_all = [&] {
    if (nc > 1)
      cl.sync();
    else
      __syncthreads();
  };
  for (int i = tid; i < 3 * kBins; i += kPickThreads) (&hist[0][0])[i] = 0;
  load(0);
  __syncthreads();

  // ---- key of the budget-th best slot, 11 + 11 + 10 bits from the top
  uint32_t prefix = 0;
  int need = a.budget;  // slots still wanted among those that share the prefix
#pragma unroll
  for (int r3 = 0; r3 < 3; ++r3) {
    const int sh = r3 == 0 ? 21 : r3 == 1 ? 10 : 0, nb = r3 == 2 ? 1024 : 2048;
    int *hs = hist[r3];
    for (int g = 0; g < groups; ++g) {
      if (groups > 1) load(g);
#pragma unroll
      for (int i = 0; i < IPT; ++i) {
        const uint32_t k = kr[i];
        if (k != 0u && (r3 == 0 || (k >> (sh + (r3 == 2 ? 10 : 11))) == prefix))
          atomicAdd(&hs[(k >> sh) & (nb - 1)], 1);
      }
    }
    sync_all();
    // bins from the top, two per thread; sums over the cluster
    int c0 = 0, c1 = 0;
    const int b0 = nb - 1 - 2 * tid, b1 = b0 - 1;
    if (b1 >= 0) {
      if (nc > 1) {
        for (int r = 0; r < nc; ++r) {
          const int *hr = cl.map_shared_rank(hs, r);
          c0 += hr[b0];
          c1 += hr[b1];
        }
      } else {
        c0 = hs[b0];
        c1 = hs[b1];
      }
    }
    int wsum, total;
    const int lp = lane_prefix(c0 + c1, &wsum);
    const int before = warp_prefix(wsum, s_scan[r3], &total) + lp;
    if (before < need && before + c0 >= need) {
      s_bin[r3] = b0;
      s_need[r3] = need - before;
    } else if (before + c0 < need && before + c0 + c1 >= need) {
      s_bin[r3] = b1;
      s_need[r3] = need - before - c0;
    }
    __syncthreads();
    prefix = (prefix << (r3 == 2 ? 10 : 11)) | (uint32_t)s_bin[r3];
    need = s_need[r3];
  }
  const uint32_t kth = prefix;  // better keys survive, and the first `need` equal ones

  // ---- equal keys before this warp's slots
  int eq = 0;
  for (int g = 0; g < groups; ++g) {
    if (groups > 1) load(g);
#pragma unroll
    for (int i = 0; i < IPT; ++i) eq += kr[i] == kth;
  }
  eq = __reduce_add_sync(0xffffffffu, eq);
  int eq_total;
  int eq0 = warp_prefix(eq, s_scan[3], &eq_total);
  if (nc > 1) {
    if (tid == 0) s_cnt[0] = eq_total;
    cl.sync();
    for (int r = 0; r < rank; ++r) eq0 += cl.map_shared_rank(s_cnt, r)[0];
  }
  // the lane's slots of the group that survive, as a bit mask; e: equal keys before the group
  auto kept = [&](int &e) {
    uint32_t keep = 0, same = 0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      keep |= (uint32_t)(kr[i] > kth) << i;
      same |= (uint32_t)(kr[i] == kth) << i;
    }
    if (__any_sync(0xffffffffu, same != 0u)) {
      int sum;
      int before = e + lane_prefix(__popc(same), &sum);
      for (uint32_t s = same; s != 0u && before < need; s &= s - 1u, ++before) keep |= s & (0u - s);
      e += sum;
    }
    return keep;
  };
  // ---- freed slots below the budget and survivors beyond it, in this warp
  int holes = 0, tails = 0, e = eq0;
  for (int g = 0; g < groups; ++g) {
    if (groups > 1) load(g);
    const uint32_t keep = kept(e), low = below(a.budget);
    holes += __popc(low & ~keep);
    tails += __popc(keep & ~low);
  }
  holes = __reduce_add_sync(0xffffffffu, holes);
  tails = __reduce_add_sync(0xffffffffu, tails);
  int hall, tall;
  int hb = warp_prefix(holes, s_scan[4], &hall), tb = warp_prefix(tails, s_scan[5], &tall);
  if (nc > 1) {
    if (tid == 0) s_cnt[1] = hall, s_cnt[2] = tall;
    cl.sync();
    hall = 0;
    for (int r = 0; r < nc; ++r) {
      const int *c = cl.map_shared_rank(s_cnt, r);
      hall += c[1];
      if (r < rank) {
        hb += c[1];
        tb += c[2];
      }
    }
    cl.sync();  // nobody leaves while its counts may be read
  }
  // ---- the lists
  int *hole = w.hole + (long long)bh * w.m_cap, *tail = w.tail + (long long)bh * w.m_cap;
  int *off = w.off + (long long)bh * (w.nblk + 1);
  if (rank == 0 && tid == 0) off[w.nblk] = hall;
  e = eq0;
  for (int g = 0; g < groups; ++g) {
    if (groups > 1) load(g);
    const uint32_t keep = kept(e), low = below(a.budget);
    const uint32_t fr = low & ~keep, sv = keep & ~low;
    int nh, nt;
    int hr = hb + lane_prefix(__popc(fr), &nh), tr = tb + lane_prefix(__popc(sv), &nt);
    // blocks that start in this lane's slots
    for (int blk = (base + a.bs - 1) / a.bs; blk < w.nblk && blk * a.bs < base + IPT; ++blk)
      off[blk] = hr + __popc(fr & ((1u << (blk * a.bs - base)) - 1u));
    for (uint32_t m = fr; m != 0u; m &= m - 1u) hole[hr++] = base + __ffs(m) - 1;
    for (uint32_t m = sv; m != 0u; m &= m - 1u) tail[tr++] = base + __ffs(m) - 1;
    hb += nh;
    tb += nt;
  }
}

// Min / max of 16 bytes of a row, element by element, in the row's own type (exact).
template <typename T>
__device__ __forceinline__ uint4 min16(uint4 a, uint4 b, bool top) {
  uint32_t *x = reinterpret_cast<uint32_t *>(&a);
  const uint32_t *y = reinterpret_cast<const uint32_t *>(&b);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(T) == 4) {
      const float u = __uint_as_float(x[e]), v = __uint_as_float(y[e]);
      x[e] = __float_as_uint(top ? fmaxf(u, v) : fminf(u, v));
    } else {
      using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const P u = *reinterpret_cast<const P *>(&x[e]), v = *reinterpret_cast<const P *>(&y[e]);
      const P r = top ? __hmax2(u, v) : __hmin2(u, v);
      x[e] = *reinterpret_cast<const uint32_t *>(&r);
    }
  }
  return a;
}
template <typename T>
__device__ __forceinline__ uint4 splat16(float x) {
  uint4 u;
  if constexpr (sizeof(T) == 4)
    u.x = __float_as_uint(x);
  else
    u.x = Mma<T>::pack(x, x);
  u.y = u.z = u.w = u.x;
  return u;
}
__device__ __forceinline__ uint4 shfl_xor16(uint4 a, int o) {
  return make_uint4(__shfl_xor_sync(0xffffffffu, a.x, o), __shfl_xor_sync(0xffffffffu, a.y, o),
                    __shfl_xor_sync(0xffffffffu, a.z, o), __shfl_xor_sync(0xffffffffu, a.w, o));
}

// One CTA of 256 threads per block of slots.  A row is PC 16-byte pieces; a thread
// owns one piece column (PC <= 32: its warp holds 32 / PC rows side by side) and every
// RG-th row.  A block is a few rows per thread behind a chain of dependent loads
// (offsets, lists, rows), so CTAs side by side hide it: min and max stay in the row's
// type and are joined by shuffles, which leaves room for six CTAs per SM and takes
// most of the instructions out (an fp32 min / max through shared memory: 42% of the
// issue slots at half the HBM rate).  Rows pass through once: streaming loads and
// stores (a prompt to a quarter: 112 -> 102 us).
template <typename T, int D>
__global__ void __launch_bounds__(256, 6) evict_move_kernel(const bsa_evict_args a, const EvictWork w) {
  constexpr int E = 16 / sizeof(T), PC = D / E, RG = 256 / PC;
  extern __shared__ int s_src[];  // [bs] source slot, then per warp the min and the max
  const int blk = blockIdx.x % w.nblk, bh = blockIdx.x / w.nblk;
  const int b = bh / a.Hkv, h = bh % a.Hkv, tid = threadIdx.x, warp = tid >> 5;
  const int s0 = blk * a.bs, rows = min(a.bs, a.budget - s0);
  for (int i = tid; i < rows; i += 256) s_src[i] = s0 + i;
  pdl_wait();
  const int *off = w.off + (long long)bh * (w.nblk + 1);
  const int m0 = off[blk], m1 = off[blk + 1];
  const bool moves = m1 > m0;
  const bool same = a.weight_out == a.weight && a.pos_out == a.pos;
  const bool pool = a.kmin && (moves || rows < a.bs);
  if (!moves && !pool && same) return;
  __syncthreads();
  const long long list = (long long)bh * w.m_cap;
  for (int m = m0 + tid; m < m1; m += 256) s_src[w.hole[list + m] - s0] = w.tail[list + m];
  __syncthreads();
  const int c = tid % PC, r0 = tid / PC;
  uint4 mn = splat16<T>(rows < a.bs ? 0.f : INFINITY);  // rows past the budget count as zeros
  uint4 mx = splat16<T>(rows < a.bs ? 0.f : -INFINITY);
  if (moves || pool) {
    T *kp = reinterpret_cast<T *>(a.k.ptr) + b * a.k.sb + h * a.k.sh + c * E;
    T *vp = reinterpret_cast<T *>(a.v.ptr) + b * a.v.sb + h * a.v.sh + c * E;
    constexpr int U = 2;  // rows in flight per thread
    for (int rb = r0; rb < rows; rb += U * RG) {
      uint4 kv[U], vv[U];
      int src[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = rb + u * RG;
        src[u] = r < rows ? s_src[r] : -1;
        if (src[u] >= 0 && (pool || src[u] != s0 + r))
          kv[u] = __ldcs(reinterpret_cast<const uint4 *>(kp + (long long)src[u] * a.k.sl));
        if (src[u] >= 0 && src[u] != s0 + r)
          vv[u] = __ldcs(reinterpret_cast<const uint4 *>(vp + (long long)src[u] * a.v.sl));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = rb + u * RG;
        if (src[u] >= 0 && src[u] != s0 + r) {
          __stcs(reinterpret_cast<uint4 *>(kp + (long long)(s0 + r) * a.k.sl), kv[u]);
          __stcs(reinterpret_cast<uint4 *>(vp + (long long)(s0 + r) * a.v.sl), vv[u]);
        }
        if (src[u] >= 0 && pool) {
          mn = min16<T>(mn, kv[u], false);
          mx = min16<T>(mx, kv[u], true);
        }
      }
    }
  }
  const float *wt = a.weight + b * a.w_sb + h * a.w_sh;
  const int32_t *ps = a.pos + b * a.p_sb + h * a.p_sh;
  float *wo = a.weight_out + b * a.wo_sb + h * a.wo_sh;
  int32_t *po = a.pos_out + b * a.po_sb + h * a.po_sh;
  for (int i = tid; i < rows; i += 256) {
    const int s = s_src[i];
    if (s != s0 + i || !same) {
      wo[s0 + i] = wt[s];
      po[s0 + i] = ps[s];
    }
  }
  if (!pool) return;
#pragma unroll
  for (int o = PC; o < 32; o <<= 1) {
    mn = min16<T>(mn, shfl_xor16(mn, o), false);
    mx = min16<T>(mx, shfl_xor16(mx, o), true);
  }
  // [min, max][warp row][PC]: at PC 64 (fp32, D 256) two warps hold a row
  constexpr int WR = PC <= 32 ? 8 : 256 / PC;
  uint4 *sp = reinterpret_cast<uint4 *>(s_src + (a.bs + 3) / 4 * 4);
  const int wrow = PC <= 32 ? warp : r0;
  if (PC > 32 || (tid & 31) < PC) {
    sp[wrow * PC + c] = mn;
    sp[(WR + wrow) * PC + c] = mx;
  }
  __syncthreads();
  for (int i = tid; i < 2 * D; i += 256) {
    const bool top = i >= D;
    const int d = top ? i - D : i;
    const T *s = reinterpret_cast<const T *>(sp + (top ? WR * PC : 0)) + d;
    float x;
#pragma unroll
    for (int r = 0; r < WR; ++r) {
      float y;
      if constexpr (sizeof(T) == 4)
        y = s[r * D];
      else
        y = Mma<T>::to_f(s[r * D]);
      x = r == 0 ? y : top ? fmaxf(x, y) : fminf(x, y);
    }
    (top ? a.kmax : a.kmin)[b * a.km_sb + h * a.km_sh + (long long)blk * a.km_sn + d] = x;
  }
}

// ------------------------------------------------------------------ host
// Whether rows of an output (budget words each, x) meet rows of its source (L words, y)
// without being the same view.  Exact for equal strides, else by the spans.
static bool rows_meet(const void *x, int64_t xb, int64_t xh, const void *y, int64_t yb, int64_t yh,
                      const bsa_evict_args *a) {
  const int64_t B = a->B, H = a->Hkv, d = ((const char *)x - (const char *)y) / 4;
  const bool like = (xb == yb || B == 1) && (xh == yh || H == 1);
  if (like && d == 0) return false;
  if (d >= yb * (B - 1) + yh * (H - 1) + a->L || -d >= xb * (B - 1) + xh * (H - 1) + a->budget) return false;
  if (!like) return true;
  for (int64_t j = 1 - B; j < B; ++j) {  // row offsets d + j sb + i sh in (-budget, L), |i| < H
    const int64_t e = d + (B > 1 ? j * yb : 0);
    if (H == 1 || yh == 0) {
      if (e > -(int64_t)a->budget && e < a->L) return true;
      continue;
    }
    int64_t i = -e / yh;  // the three around the nearest row
    for (int64_t k = i - 1; k <= i + 1; ++k)
      if (k > -H && k < H && e + k * yh > -(int64_t)a->budget && e + k * yh < a->L) return true;
  }
  return false;
}

static bsa_status evict_check(const bsa_evict_args *a) {
  if (a->dtype != BSA_BF16 && a->dtype != BSA_F16 && a->dtype != BSA_F32)
    return fail(BSA_ERR_DTYPE, "evict: dtype must be bf16, f16 or f32");
  if (a->B <= 0 || a->Hkv <= 0 || a->L <= 0 || a->bs <= 0)
    return fail(BSA_ERR_SHAPE, "evict: sizes must be positive");
  if (a->D != 32 && a->D != 64 && a->D != 128 && a->D != 256)
    return fail(BSA_ERR_UNSUPPORTED, "evict: D must be 32, 64, 128 or 256");
  if (a->bs > 1024) return fail(BSA_ERR_UNSUPPORTED, "evict: bs must be <= 1024");
  if (a->budget <= 0 || a->budget > a->L) return fail(BSA_ERR_SHAPE, "evict: needs 1 <= budget <= L");
  if (a->recent < 0 || a->sink < 0 || (long long)a->recent + a->sink > a->budget)
    return fail(BSA_ERR_SHAPE, "evict: recent + sink must lie in [0, budget]");
  if (a->seen < a->L) return fail(BSA_ERR_SHAPE, "evict: seen must be at least L");
  if (a->L > (1 << 29) || (long long)a->B * a->Hkv >= (1 << 24))
    return fail(BSA_ERR_SHAPE, "evict: L or B*Hkv too large");
  if (!a->k.ptr || !a->v.ptr || !a->weight || !a->pos || !a->weight_out || !a->pos_out)
    return fail(BSA_ERR_ARG, "evict: NULL tensor");
  if (!a->kmin != !a->kmax) return fail(BSA_ERR_ARG, "evict: kmin and kmax go together");
  const int64_t es = (int64_t)elem_size(a->dtype);
  for (const bsa_view *v : {&a->k, &a->v})
    if (reinterpret_cast<uintptr_t>(v->ptr) % 16 || (v->sb * es) % 16 || (v->sh * es) % 16 || (v->sl * es) % 16)
      return fail(BSA_ERR_STRIDE, "evict: k and v need 16-byte aligned bases and strides");
  for (const bsa_view *v : {&a->k, &a->v})
    if (!lies_apart(a->B, v->sb, a->Hkv, v->sh, a->L, v->sl, a->D))
      return fail(BSA_ERR_STRIDE, "evict: rows of k or v share memory");
  const long long nblk = (a->budget + a->bs - 1) / a->bs;
  if (!lies_apart(a->B, a->wo_sb, a->Hkv, a->wo_sh, 1, 0, a->budget) ||
      !lies_apart(a->B, a->po_sb, a->Hkv, a->po_sh, 1, 0, a->budget) ||
      (a->kmin && !lies_apart(a->B, a->km_sb, a->Hkv, a->km_sh, nblk, a->km_sn, a->D)))
    return fail(BSA_ERR_STRIDE, "evict: rows of an output share memory");
  if (rows_meet(a->weight_out, a->wo_sb, a->wo_sh, a->weight, a->w_sb, a->w_sh, a) ||
      rows_meet(a->pos_out, a->po_sb, a->po_sh, a->pos, a->p_sb, a->p_sh, a))
    return fail(BSA_ERR_STRIDE, "evict: weight_out / pos_out must be weight / pos or lie apart from them");
  if (nblk * a->B * a->Hkv >= (1LL << 31)) return fail(BSA_ERR_SHAPE, "evict: too many blocks");
  return BSA_OK;
}

static size_t evict_plan(const bsa_evict_args *a, EvictWork *w, uint8_t *base) {
  w->m_cap = std::max(1, std::min(a->budget, a->L - a->budget));
  w->nblk = (a->budget + a->bs - 1) / a->bs;
  const size_t bh = (size_t)a->B * a->Hkv, list = align_up(bh * w->m_cap * 4, 256);
  w->hole = reinterpret_cast<int *>(base);
  w->tail = reinterpret_cast<int *>(base + list);
  w->off = reinterpret_cast<int *>(base + 2 * list);
  return 2 * list + align_up(bh * (w->nblk + 1) * 4, 256);
}

size_t evict_workspace(const bsa_evict_args *a) {
  EvictWork w;
  return evict_check(a) == BSA_OK ? evict_plan(a, &w, nullptr) : 0;
}

bsa_status run_evict(const bsa_evict_args *a, void *ws, size_t ws_bytes, cudaStream_t st) {
  if (bsa_status s = evict_check(a)) return s;
  EvictWork w;
  const size_t need = evict_plan(a, &w, static_cast<uint8_t *>(ws));
  if (!ws || ws_bytes < need) return fail(BSA_ERR_WORKSPACE, "evict: workspace too small");
  const int bh = a->B * a->Hkv;
  // CTAs per (b, head): as few as hold its slots in registers (16 per thread), at most 8,
  // the portable cluster size: a pass over a cluster costs twice the barrier of one CTA
  int nc = 1;
  while (nc < 8 && (long long)nc * 16 * kPickThreads < a->L) nc *= 2;
  const int ipt = (int)((a->L + (long long)nc * kPickThreads - 1) / ((long long)nc * kPickThreads));
  const int groups = std::max(1, (ipt + 15) / 16);
  // 16-byte loads of the sums and positions
  const int vec = !(reinterpret_cast<uintptr_t>(a->weight) % 16 || reinterpret_cast<uintptr_t>(a->pos) % 16 ||
                    a->w_sb % 4 || a->w_sh % 4 || a->p_sb % 4 || a->p_sh % 4);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)bh * nc);
  cfg.blockDim = dim3(kPickThreads);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = nc, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  if (ipt <= 4)
    cudaLaunchKernelEx(&cfg, evict_pick_kernel<4>, *a, w, 1, vec);
  else if (ipt <= 8)
    cudaLaunchKernelEx(&cfg, evict_pick_kernel<8>, *a, w, 1, vec);
  else
    cudaLaunchKernelEx(&cfg, evict_pick_kernel<16>, *a, w, groups, vec);
  if (bsa_status s = check_launch("evict_pick")) return s;
  const unsigned grid = (unsigned)bh * w.nblk;
  const size_t smem = (size_t)align_up(a->bs * 4, 16) + 2ull * 8 * a->D * elem_size(a->dtype);
#define BSA_MOVE(T_)                                                                          \
  switch (a->D) {                                                                             \
    case 32: launch_after(evict_move_kernel<T_, 32>, grid, 256, smem, st, *a, w); break;      \
    case 64: launch_after(evict_move_kernel<T_, 64>, grid, 256, smem, st, *a, w); break;      \
    case 128: launch_after(evict_move_kernel<T_, 128>, grid, 256, smem, st, *a, w); break;    \
    default: launch_after(evict_move_kernel<T_, 256>, grid, 256, smem, st, *a, w);            \
  }
  if (a->dtype == BSA_BF16) {
    BSA_MOVE(__nv_bfloat16)
  } else if (a->dtype == BSA_F16) {
    BSA_MOVE(__half)
  } else {
    BSA_MOVE(float)
  }
#undef BSA_MOVE
  return check_launch("evict_move");
}

}  // namespace bsa
