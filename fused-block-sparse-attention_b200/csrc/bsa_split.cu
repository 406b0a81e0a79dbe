// Split-key attention of few query rows (decode steps) in bf16 / f16 / fp32, the
// join of the splits, and the running sum of every slot's attention weight.
//
//   split_mma_kernel, split_f32_kernel, split_f32_rows_kernel   partial softmax and O of
//                       one split
//   split_join_kernel   joins the splits of every row; with weights, also adds the sum
//                       over the rows of p = 2^(x - lse) to each slot's sum
// The kernels are bound by reading K and V once (HBM).
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

#include "bsa_host.h"
#include "bsa_split.cuh"

namespace cg = cooperative_groups;

namespace bsa {

namespace {
constexpr int NW = 4;          // warps per CTA of the partial kernel
constexpr int kMaxLive = 512;  // block ids of one selection row

// K and V are read once: they leave L2 first, so that the logits stay there for the join
// (3 x 32777 slots, 32 heads, 4 rows each, D 128: 88 us, 97 without).  A shared prefix that
// several clusters or row tiles read comes with the same policy: without it those times are
// the same within 1%.
__device__ __forceinline__ uint64_t evict_first_policy() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool live, uint64_t policy) {
  const int n = live ? 16 : 0;  // the rest of the 16 bytes is filled with zeros
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(n),
               "l"(policy)
               : "memory");
}

// Without the policy: rows that other CTAs read too.
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

// fp32 products on the tensor cores: x = x1 + x2 + x3, each what is left cut off to bf16 (8
// bits each, so all 24), and x y = x1 y1 + x1 y2 + x2 y1 + x2 y2 + x1 y3 + x3 y1 up to
// 2^-21 |x y| (the other three).  Six bf16 products take the time of one and a half tf32
// ones (mma.sync, measured 300 against 80 TFLOP/s), of which two-term tf32 splits need
// three.  The terms of two neighbours, packed.  Each is cut off below what is left, so that
// all have the sign of x and none is zero: an infinity (its own first term, the others zero)
// times them stays what it is, where terms of unlike sign make infinity - infinity of it,
// and cutting off does not take the largest floats to infinity.
__device__ __forceinline__ void split3(float x, float y, uint32_t *u) {
  constexpr float kBelow = 1.f - 0x1p-24f;  // the next float below
  uint32_t a = __float_as_uint(x * kBelow), b = __float_as_uint(y * kBelow);
  u[0] = __byte_perm(a, b, 0x7632);
  float x1 = __uint_as_float(a & 0xffff0000u), y1 = __uint_as_float(b & 0xffff0000u);
  const float rx = x == x1 ? 0.f : x - x1, ry = y == y1 ? 0.f : y - y1;
  a = __float_as_uint(rx * kBelow), b = __float_as_uint(ry * kBelow);
  u[1] = __byte_perm(a, b, 0x7632);
  x1 = __uint_as_float(a & 0xffff0000u), y1 = __uint_as_float(b & 0xffff0000u);
  u[2] = __byte_perm(__float_as_uint(rx - x1), __float_as_uint(ry - y1), 0x7632);
}
// The same for K and V, whose terms may have any sign, as long as those of q and P have not:
// the first is x without its low bits (no border to infinity), the others are rounded, so
// that what the products drop is half as large.
__device__ __forceinline__ void split3_kv(float x, float y, uint32_t *u) {
  u[0] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
  float x1 = __uint_as_float(__float_as_uint(x) & 0xffff0000u), y1 = __uint_as_float(__float_as_uint(y) & 0xffff0000u);
  const float rx = x == x1 ? 0.f : x - x1, ry = y == y1 ? 0.f : y - y1;
  u[1] = Mma<__nv_bfloat16>::pack(rx, ry);
  x1 = __uint_as_float(u[1] << 16), y1 = __uint_as_float(u[1] & 0xffff0000u);
  u[2] = Mma<__nv_bfloat16>::pack(rx - x1, ry - y1);
}
// Maximum that keeps a NaN: a row with a NaN logit ends as NaN, not as an empty row.
__device__ __forceinline__ float fmax_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Live block ids (and gates) of one selection row: the first occurrence of each id
// that holds slots before L, unless its gate is -inf; in the selection's order; by one
// warp, which compares each id with all before it (kk^2 / 64 steps).  Returns their count.
__device__ int build_live(const SplitParams &p, int b, int hk, int len, int *s_blk, float *s_gate,
                          int *s_raw) {
  const int lane = threadIdx.x & 31;
  const int32_t *row = p.sel + b * p.sel_sb + hk * p.sel_sh;
  const float *gr = p.gate ? p.gate + b * p.gate_sb + hk * p.gate_sh : nullptr;
  const int nblk = (len + p.bs - 1) / p.bs;
  for (int j = lane; j < p.kk; j += 32) s_raw[j] = __ldg(row + j);
  __syncwarp();
  int n = 0;
  for (int j0 = 0; j0 < p.kk; j0 += 32) {
    const int j = j0 + lane;
    bool ok = false;
    int kb = 0;
    float gv = 0.f;
    if (j < p.kk) {
      kb = s_raw[j];
      if (kb < 0 || kb >= nblk) {
        report(p.status, BSA_DEVERR_INDEX);
      } else {
        ok = true;
        for (int i = 0; i < j && ok; ++i) ok = s_raw[i] != kb;
        if (gr) gv = __ldg(gr + j) * kLog2e;
        if (gv == -INFINITY) ok = false;  // masked as a whole: its rows are not read
      }
    }
    const unsigned live = __ballot_sync(0xffffffffu, ok);
    const int at = n + __popc(live & ((1u << lane) - 1u));
    if (ok) {
      s_blk[at] = kb;
      s_gate[at] = gv;
    }
    n += __popc(live);
  }
  return n;
}
}  // namespace

// ------------------------------------------------------------------ partial kernels
// CTA = (K/V head group, a tile of query rows, split); each of its NW = 4 warps takes
// every fourth chunk of KC keys and keeps its own m, l and O, so the warps meet only at
// the end.  A chunk's K and V rows arrive by 16-byte cp.async in a ring of NST stages
// per warp, rows past the end zero-filled (never read).  Keys that some rows of the tile
// must not see (the newest T - 1) are multiplied one by one in fp32 and skipped where
// p = 0: an infinity or NaN in a masked V row never reaches a row that does not see it.
//
// 16-bit types, split_mma_kernel: the keys are M of the m16n8k16 products and the query
// rows N, eight at a time: S^T = K Q^T, O^T += V^T P^T.  A decode step has few rows (a
// head group, times the new tokens), and with the rows as M half of every product and of
// O's registers was padding; 480 instructions per 16 keys at D 128 kept the warps from
// drawing their share of HBM.  P^T reaches its operand layout by movmatrix, in two 16-bit
// terms (split2), so its rounding does not add to the output's; the extra products are
// free under HBM's time.  f16 has nothing below 2^-24, so there P, l and O are 2^15 larger
// and m is kept 15 lower: with p = 1 for the largest, many keys 2^-20 and less below it
// (behind an attention sink) lost bits or came to nothing in O while l counted them.
//
// fp32, split_f32_kernel: the same on three bf16 terms of every operand (above).  A
// contraction may take its index in any order and O's rows any place, so a thread's
// 16-byte piece of a K row is its two pairs of a k-step (dims 4t .. 4t+3), and 16-byte
// pieces of V rows feed four tiles of O (tile e holds columns 4j + e of a group).  The
// products truncate their sums, always towards zero, so a chunk's part of O starts at zero
// and is added by a rounding addition (20000 keys, D 256: 5.2e-7 of the output's norm, plain fp32
// arithmetic 8.2e-7; summed on in the products it was 25 times as much).
template <typename T, int D>
struct SplitCfg {
  static constexpr int ES = sizeof(T), E16 = 16 / ES;
  static constexpr int KC = ES == 2 && D <= 64 ? 32 : 16;
  static constexpr int STAGE = KC * D * ES * 2;       // K and V of a chunk, bytes
  static constexpr int NST = STAGE <= 4096 ? 5 : STAGE == 32768 ? 1 : 3;
  static constexpr int MINB = STAGE >= 16384 ? 1 : 2; // CTAs per SM
  static constexpr int RING = NW * NST * STAGE;
  // most rows per CTA: O fits the registers, P a chunk of K
  static constexpr int MAXROWS = D == 256 || (ES == 2 && D == 32) ? 16 : 32;
};

// Rows per CTA for R query rows.
template <typename T, int D>
constexpr int split_rows(int R) {
  using C = SplitCfg<T, D>;
  return R <= 8 ? 8 : R <= 16 || C::MAXROWS == 16 ? 16 : 32;
}

// Byte offset of 16-byte chunk `chunk` of a D-wide row: chunks are permuted within
// 128 bytes so that the eight rows (16-bit: ldmatrix) or two / four rows (fp32: the
// pieces of K / V above) read together fall into different banks.
template <int ES, int D>
__device__ __forceinline__ uint32_t sw_off(int row, int chunk) {
  if constexpr (ES == 2 && D == 32)
    return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
  else if constexpr (ES == 2)
    return row * (D * 2) + (((chunk & ~7) | ((chunk ^ row) & 7)) << 4);
  else
    return row * (D * 4) + ((chunk ^ ((row & 6) ^ ((row & 1) << 2))) << 4);
}

// What a CTA works on; chunks [0, nch2) are those of the shared keys (one launch only).
struct Span {
  int b, hk, grpid, r0, len, nch2, c_lo, c_hi, split;
};

// Row tile, length, live blocks and chunk range of this CTA.  False: nothing to see
// (the rows' m is written as -inf and the join skips the split).
template <int KC, int ROWS, bool CL>
__device__ __forceinline__ bool split_span(const SplitParams &p, int rtiles, int min_chunks, Span &s, int *s_blk,
                                           float *s_gate, int *s_raw, int *s_n) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rt = blockIdx.x % rtiles;
  s.grpid = blockIdx.x / rtiles;
  s.b = p.fold ? 0 : s.grpid / p.Hkv;
  s.hk = s.grpid % p.Hkv;
  s.r0 = rt * ROWS;
  s.len = p.nkeys;
  if (p.lens) {
    s.len = __ldg(p.lens + s.b);
    if (s.len < 0 || s.len > p.nkeys) {
      if (tid == 0) report(p.status, BSA_DEVERR_INDEX);
      s.len = s.len < 0 ? 0 : p.nkeys;
    }
  }
  int nv = s.len;  // virtual keys: the slots, or those of the live blocks one after another
  if (p.sel) {
    if (warp == 0) {
      const int n = build_live(p, s.b, s.hk, s.len, s_blk, s_gate, s_raw);
      if (lane == 0) *s_n = n;
      if (p.live && blockIdx.y == 0 && rt == 0) {
        __syncwarp();
        int *lv = p.live + (long long)s.grpid * (1 + p.kk);
        for (int i = lane; i < n; i += 32) lv[1 + i] = s_blk[i];
        if (lane == 0) lv[0] = n;
      }
    }
    __syncthreads();
    nv = *s_n * p.bs;
  }
  s.nch2 = CL ? (p.n2 + KC - 1) / KC : 0;
  const int nch = s.nch2 + (nv + KC - 1) / KC;
  const int cps = max(min_chunks, (nch + p.nsplit - 1) / p.nsplit);
  s.c_lo = min(nch, (int)blockIdx.y * cps);
  s.c_hi = min(nch, s.c_lo + cps);
  s.split = p.split0 + blockIdx.y;
  if constexpr (!CL) {
    if (s.c_lo >= s.c_hi) {
      for (int r = tid; r < ROWS && s.r0 + r < p.R; r += blockDim.x) {
        int rb, rh, rtt;
        const long long gr = split_row(p, s.b, s.hk, s.r0 + r, rb, rh, rtt);
        p.pml[(long long)s.split * p.rows + gr] = make_float2(-INFINITY, 0.f);
      }
      return false;
    }
  }
  return true;
}

// First key of chunk c, and its gate.
template <int KC>
__device__ __forceinline__ int split_key(const SplitParams &p, const int *s_blk, const float *s_gate, int c,
                                         float &gate) {
  const int j = c * KC;
  if (!p.sel) {
    gate = 0.f;
    return j;
  }
  const int i = j / p.bs;
  gate = s_gate[i];
  return s_blk[i] * p.bs + (j - i * p.bs);
}

// K and V rows [key0, key0 + KC) of one chunk into a stage, by one warp.
template <typename T, int D>
__device__ __forceinline__ void split_load(const T *kb, const T *vb, int64_t ksl, int64_t vsl, int key0, int len,
                                           uint32_t stage, uint64_t policy) {
  using C = SplitCfg<T, D>;
  constexpr int CPR = D / C::E16;                    // 16-byte pieces per row
  constexpr int IT = C::KC * CPR / 32;
  const int lane = threadIdx.x & 31;
  const uint32_t dv = stage + C::KC * D * C::ES;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int i = it * 32 + lane, row = i / CPR, ch = i % CPR;
    const bool ok = key0 + row < len;
    const int64_t key = ok ? key0 + row : 0;
    const uint32_t off = sw_off<C::ES, D>(row, ch);
    cp16(stage + off, kb + key * ksl + ch * C::E16, ok, policy);
    cp16(dv + off, vb + key * vsl + ch * C::E16, ok, policy);
  }
}

// The query rows of the tile into shared memory (swizzled), zeros past R.
template <typename T, int D, int ROWS>
__device__ __forceinline__ void split_queries(const SplitParams &p, const Span &s, uint8_t *sQ) {
  constexpr int E16 = SplitCfg<T, D>::E16, CPR = D / E16;
  for (int i = threadIdx.x; i < ROWS * CPR; i += blockDim.x) {
    const int r = i / CPR, ch = i % CPR;
    alignas(16) T e[E16];
    *reinterpret_cast<uint4 *>(e) = make_uint4(0, 0, 0, 0);
    if (s.r0 + r < p.R) {
      int rb, rh, rtt;
      split_row(p, s.b, s.hk, s.r0 + r, rb, rh, rtt);
      const T *qp = reinterpret_cast<const T *>(p.q) + rb * p.q_sb + rh * p.q_sh + rtt * p.q_sl + ch * E16;
#pragma unroll
      for (int x = 0; x < E16; ++x) e[x] = qp[x];
    }
    *reinterpret_cast<uint4 *>(sQ + sw_off<sizeof(T), D>(r, ch)) = *reinterpret_cast<uint4 *>(e);
  }
}

// Sum of the warps' O (so: [warp][ROWS][STRIDE], scaled to the common maximum) and their
// (m, l), to the split's place.
template <int D, int ROWS, int STRIDE>
__device__ __forceinline__ void split_write(const SplitParams &p, const Span &s, const float *so,
                                            const float (*s_m)[ROWS], const float (*s_l)[ROWS]) {
  const int nr = min(ROWS, p.R - s.r0);
  for (int i = threadIdx.x; i < nr * (D / 4); i += blockDim.x) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
    float4 o = *reinterpret_cast<const float4 *>(so + r * STRIDE + d);
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      const float4 x = *reinterpret_cast<const float4 *>(so + (w * ROWS + r) * STRIDE + d);
      o.x += x.x;
      o.y += x.y;
      o.z += x.z;
      o.w += x.w;
    }
    int rb, rh, rtt;
    const long long at = (long long)s.split * p.rows + split_row(p, s.b, s.hk, s.r0 + r, rb, rh, rtt);
    *reinterpret_cast<float4 *>(p.po + at * D + d) = o;
    if (d == 0) {
      float M = s_m[0][r], L = 0.f;
#pragma unroll
      for (int w = 1; w < NW; ++w) M = fmax_nan(M, s_m[w][r]);
#pragma unroll
      for (int w = 0; w < NW; ++w) L += s_m[w][r] == -INFINITY ? 0.f : s_l[w][r] * ex2(s_m[w][r] - M);
      p.pml[at] = make_float2(M, L);
    }
  }
}

// m16n8k16 product that the compiler may move: with one or two warps per SM quarter the
// order of independent products is what hides their latency.
template <typename T>
__device__ __forceinline__ void mma16(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2^(x - m) f, and 0 where f is: a row that saw nothing or padding, whatever its x holds.
__device__ __forceinline__ float join_p(float x, float m, float f) { return f == 0.f ? 0.f : ex2(x - m) * f; }

// The join within a cluster, instead of partial sums in memory and a second launch: the
// CTAs of one (b, hk) hold its splits.  so: this CTA's [warp][ROWS][SO] (scaled to the
// warps' common maximum).  Each CTA writes its share of o and adds the weights of its own
// slots, whose logits it wrote itself.
template <typename T, int KC, int D, int ROWS, int SO>
__device__ __forceinline__ void cluster_join(const SplitParams &p, const Span &s, float *so, float (*s_m)[ROWS],
                                             float (*s_l)[ROWS], const int *s_blk) {
  cg::cluster_group cl = cg::this_cluster();
  const int cs = cl.num_blocks(), rank = cl.block_rank(), tid = threadIdx.x;
  __shared__ float s_f[8][ROWS], s_M[ROWS], s_inv[ROWS];
  // the CTA's own (m, l) and O: warp 0's place takes the sums
  const int nr = min(ROWS, p.R);
  float cm = 0.f, cl_ = 0.f;
  if (tid < ROWS) {
    cm = s_m[0][tid];
#pragma unroll
    for (int w = 1; w < NW; ++w) cm = fmax_nan(cm, s_m[w][tid]);
#pragma unroll
    for (int w = 0; w < NW; ++w) cl_ += s_m[w][tid] == -INFINITY ? 0.f : s_l[w][tid] * ex2(s_m[w][tid] - cm);
  }
  for (int i = tid; i < nr * (D / 4); i += blockDim.x) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
    float4 o = *reinterpret_cast<const float4 *>(so + r * SO + d);
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      const float4 x = *reinterpret_cast<const float4 *>(so + (w * ROWS + r) * SO + d);
      o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
    }
    *reinterpret_cast<float4 *>(so + r * SO + d) = o;
  }
  __syncthreads();
  if (tid < ROWS) {
    s_m[0][tid] = cm;
    s_l[0][tid] = cl_;
  }
  if (cs > 1)
    cl.sync();
  else
    __syncthreads();
  if (tid < ROWS) {
    float m[8], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < cs) {
        m[c] = cl.map_shared_rank(&s_m[0][0], c)[tid];
        M = fmax_nan(M, m[c]);
      }
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < cs) {
        const float f = m[c] == -INFINITY ? 0.f : ex2(m[c] - M);
        s_f[c][tid] = f;
        if (f != 0.f) L = fmaf(cl.map_shared_rank(&s_l[0][0], c)[tid], f, L);
      }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    s_M[tid] = M;
    s_inv[tid] = tid < nr ? inv : 0.f;
  }
  __syncthreads();
  for (int i = rank * blockDim.x + tid; i < nr * (D / 4); i += cs * blockDim.x) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < cs; ++c) {
      const float f = s_f[c][r];
      if (f == 0.f) continue;  // nothing seen there
      const float4 x = *reinterpret_cast<const float4 *>(cl.map_shared_rank(so, c) + r * SO + d);
      o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
    }
    const float inv = s_inv[r];
    int rb, rh, rt;
    split_row(p, s.b, s.hk, r, rb, rh, rt);
    T *op = reinterpret_cast<T *>(p.o) + rb * p.o_sb + rh * p.o_sh + rt * p.o_sl + d;
    const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 2)
        op[e] = Mma<T>::from_f(y[e]);
      else
        op[e] = y[e];
    }
  }
  if (p.weight) {
    float *wp = p.weight + s.b * p.w_sb + s.hk * p.w_sh;
    const float *lg = p.logits + (long long)s.grpid * p.ncap * p.rpad;
    const int rpad = p.rpad;  // 8, 16, 24 or 32 here
    for (int j = s.c_lo * KC + tid; j < s.c_hi * KC; j += blockDim.x) {
      int key = j;
      if (p.sel) {
        const int blk = j / p.bs;
        key = s_blk[blk] * p.bs + (j - blk * p.bs);
      }
      if (key >= s.len) continue;
      const float4 *x = reinterpret_cast<const float4 *>(lg + (long long)j * rpad);
      const float w0 = wp[key];
      float w = 0.f;
      for (int r = 0; r < rpad; r += 8) {
        const float4 a = x[r / 4], b = x[r / 4 + 1];
        w += (join_p(a.x, s_M[r], s_inv[r]) + join_p(a.y, s_M[r + 1], s_inv[r + 1])) +
             (join_p(a.z, s_M[r + 2], s_inv[r + 2]) + join_p(a.w, s_M[r + 3], s_inv[r + 3]));
        w += (join_p(b.x, s_M[r + 4], s_inv[r + 4]) + join_p(b.y, s_M[r + 5], s_inv[r + 5])) +
             (join_p(b.z, s_M[r + 6], s_inv[r + 6]) + join_p(b.w, s_M[r + 7], s_inv[r + 7]));
      }
      wp[key] = w0 + w;
    }
  }
  if (cs > 1) cl.sync();  // nobody leaves while its O may be read
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {  // 8x8 of 16 bits, transposed over the warp
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// ------------------------------------------------------------------ bf16 / f16
template <typename T, int D, int NR, bool CL>
__global__ void __launch_bounds__(NW * 32, SplitCfg<T, D>::MINB)
    split_mma_kernel(const SplitParams p, int rtiles, int min_chunks) {
  using C = SplitCfg<T, D>;
  constexpr int KC = C::KC, NST = C::NST, KS = D / 16, KT = KC / 16, ROWS = 8 * NR, SO = D + 4;
  constexpr float SHIFT = std::is_same<T, __half>::value ? 15.f : 0.f;  // of m below the maximum
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ int s_n;
  __shared__ float s_m[NW][ROWS], s_l[NW][ROWS];
  uint8_t *sQ = sm;                                   // [ROWS][D] swizzled
  uint8_t *ring = sm + ROWS * D * 2;
  int *s_blk = reinterpret_cast<int *>(ring + p.ring);  // with a selection: 3 * kMaxLive words
  float *s_gate = reinterpret_cast<float *>(s_blk + kMaxLive);
  // Launched to start beside the prefix kernel: its last CTA ends no earlier than that
  // kernel, so that waiting for this grid is waiting for both.
  const bool last = p.after && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, tq = lane & 3;
  pdl_trigger();  // the join may take its place on the SMs; it waits for this grid
  Span sp;
  if (!split_span<KC, ROWS, CL>(p, rtiles, min_chunks, sp, s_blk, s_gate, s_blk + 2 * kMaxLive, &s_n)) {
    if (last) pdl_wait();
    return;
  }
  const int len = sp.len, r0 = sp.r0;
  const T *kb_ = reinterpret_cast<const T *>(p.k) + (p.fold ? 0 : sp.b * p.k_sb) + sp.hk * p.k_sh;
  const T *vb_ = reinterpret_cast<const T *>(p.v) + (p.fold ? 0 : sp.b * p.v_sb) + sp.hk * p.v_sh;
  uint8_t *wring = ring + warp * p.stages * C::STAGE;
  const uint32_t wr0 = smem_u32(wring);
  const uint64_t policy = evict_first_policy();
  const T *k2_ = nullptr, *v2_ = nullptr;  // the shared keys
  if constexpr (CL) {
    k2_ = reinterpret_cast<const T *>(p.k2) + sp.hk * p.k2_sh;
    v2_ = reinterpret_cast<const T *>(p.v2) + sp.hk * p.v2_sh;
  }
  auto load = [&](int c, int st) {
    if (c < sp.c_hi) {
      if (CL && c < sp.nch2) {
        split_load<T, D>(k2_, v2_, p.k2_sl, p.v2_sl, c * KC, p.n2, wr0 + st * C::STAGE, policy);
      } else {
        float gt;
        const int key0 = split_key<KC>(p, s_blk, s_gate, c - sp.nch2, gt);
        split_load<T, D>(kb_, vb_, p.k_sl, p.v_sl, key0, len, wr0 + st * C::STAGE, policy);
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) load(sp.c_lo + warp + s * NW, s);
  split_queries<T, D, ROWS>(p, sp, sQ);
  __syncthreads();

  // Q^T as the second operand: (dims 2t, 2t+1 and 8 further; row g)
  uint32_t qf[NR][KS][2];
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        qf[n][ks][h] = *reinterpret_cast<const uint32_t *>(sQ + sw_off<2, D>(n * 8 + g, ks * 2 + h) + tq * 4);

  float acc[NR][KS][4], m[NR][2], l[NR][2];  // O^T: dims g, g + 8 of tile ks; rows 2t, 2t + 1 of group n
  int qlast[NR][2];                          // newest key that the row sees
#pragma unroll
  for (int n = 0; n < NR; ++n) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][ks][e] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[n][h] = -INFINITY;
      l[n][h] = 0.f;
      const int r = r0 + n * 8 + 2 * tq + h;
      qlast[n][h] = p.causal ? len - p.T + r % p.T : len - 1;
    }
  }
  const int all_see = p.causal ? len - p.T : len - 1;  // newest key that every row sees
  float *lg = p.logits ? p.logits + ((long long)sp.grpid * p.ncap + g) * p.rpad + r0 + 2 * tq : nullptr;
  // lane parts of the ldmatrix addresses
  const int krow = (lane & 7) + ((lane >> 3) & 1) * 8, kch = lane >> 4;
  const int vrow = (lane & 7) + (lane >> 4) * 8, vch = (lane >> 3) & 1;

  int st = 0;
  for (int c = sp.c_lo + warp; c < sp.c_hi; c += NW) {
    cp_wait<NST - 2>();
    __syncwarp();
    {
      int nst = st + NST - 1;
      if (nst >= NST) nst -= NST;
      load(c + (NST - 1) * NW, nst);
    }
    const uint32_t ka = wr0 + st * C::STAGE, va = ka + KC * D * 2;
    const bool pre = CL && c < sp.nch2;  // shared keys: every row sees them
    float gate = 0.f;
    const int key0 = pre ? c * KC : split_key<KC>(p, s_blk, s_gate, c - sp.nch2, gate);
    // ---- S^T = K Q^T
    float s[KT][NR][4];  // keys g, g + 8 of tile kt; rows 2t, 2t + 1
    constexpr int PS = KT * NR >= 4 ? 1 : 2;  // partial sums over the dims: independent chains
    float s2[PS][KT][NR][4];
#pragma unroll
    for (int q = 0; q < PS; ++q)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s2[q][kt][n][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        uint32_t a[4];
        ldsm_x4(ka + sw_off<2, D>(kt * 16 + krow, ks * 2 + kch), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int n = 0; n < NR; ++n) mma16<T>(s2[ks % PS][kt][n], a, qf[n][ks][0], qf[n][ks][1]);
      }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[kt][n][e] = PS == 2 ? s2[0][kt][n][e] + s2[PS - 1][kt][n][e] : s2[0][kt][n][e];
    // ---- online softmax (log2 domain); masked and missing keys are -inf
    const bool masked = key0 + KC - 1 > (pre ? p.n2 - 1 : all_see);
    const bool mixed = !pre && masked && all_see < len - 1;  // some row misses a key that another sees
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = fmaf(s[kt][n][e], p.scale2, gate);
          if (masked && key0 + kt * 16 + g + 8 * (e >> 1) > (pre ? p.n2 - 1 : qlast[n][e & 1])) x = -INFINITY;
          s[kt][n][e] = x;
          mx[e & 1] = fmax_nan(mx[e & 1], x);
        }
      if (lg && r0 + n * 8 < p.R) {  // rows are padded to rpad: whole groups of eight
        float *lp = lg + (long long)c * KC * p.rpad + n * 8;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2 *>(lp + (long long)(kt * 16 + 8 * h) * p.rpad) =
                make_float2(s[kt][n][2 * h], s[kt][n][2 * h + 1]);
      }
      float al[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx[h] = fmax_nan(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], o));
        const float mn = fmax_nan(m[n][h], mx[h] - SHIFT);
        al[h] = mn == -INFINITY ? 1.f : ex2(m[n][h] - mn);
        m[n][h] = mn;
      }
      if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {
        l[n][0] *= al[0];
        l[n][1] *= al[1];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][ks][e] *= al[e & 1];
      }
      const float off[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[kt][n][e] = ex2(s[kt][n][e] - off[e & 1]);
          l[n][e & 1] += s[kt][n][e];
        }
    }
    // ---- O^T += V^T P^T
    if (!mixed) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        uint32_t hi[NR][2], lo[NR][2];
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            split2<T>(s[kt][n][2 * h], s[kt][n][2 * h + 1], hi[n][h], lo[n][h]);
            hi[n][h] = movmatrix(hi[n][h]);
            lo[n][h] = movmatrix(lo[n][h]);
          }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t a[4];
          ldsm_x4_t(va + sw_off<2, D>(kt * 16 + vrow, ks * 2 + vch), a[0], a[1], a[2], a[3]);
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            mma16<T>(acc[n][ks], a, hi[n][0], hi[n][1]);
            mma16<T>(acc[n][ks], a, lo[n][0], lo[n][1]);
          }
        }
      }
    } else {
      // P through the chunk's K buffer (its reads are done), then key by key
      __syncwarp();
      float *sp_ = reinterpret_cast<float *>(wring + st * C::STAGE);  // [KC][ROWS]
      const uint8_t *sv = wring + st * C::STAGE + KC * D * 2;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sp_[(kt * 16 + g + 8 * (e >> 1)) * ROWS + n * 8 + 2 * tq + (e & 1)] = s[kt][n][e];
      __syncwarp();
#pragma unroll 1
      for (int k = 0; k < KC && key0 + k < len; ++k) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const float2 pk = *reinterpret_cast<const float2 *>(sp_ + k * ROWS + n * 8 + 2 * tq);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const float v0 = Mma<T>::to_f(*reinterpret_cast<const T *>(sv + sw_off<2, D>(k, ks * 2) + g * 2));
            const float v1 = Mma<T>::to_f(*reinterpret_cast<const T *>(sv + sw_off<2, D>(k, ks * 2 + 1) + g * 2));
            if (pk.x != 0.f) {
              acc[n][ks][0] = fmaf(pk.x, v0, acc[n][ks][0]);
              acc[n][ks][2] = fmaf(pk.x, v1, acc[n][ks][2]);
            }
            if (pk.y != 0.f) {
              acc[n][ks][1] = fmaf(pk.y, v0, acc[n][ks][1]);
              acc[n][ks][3] = fmaf(pk.y, v1, acc[n][ks][3]);
            }
          }
        }
      }
      __syncwarp();
    }
    if (++st == NST) st = 0;
  }

  // ---- join the four warps
  cp_wait<0>();
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], o);
      if (g == 0) {
        s_m[warp][n * 8 + 2 * tq + h] = m[n][h];
        s_l[warp][n * 8 + 2 * tq + h] = l[n][h];
      }
    }
  __syncthreads();
  float *so = reinterpret_cast<float *>(ring);  // [warp][ROWS][SO]; SO: rows 2t apart in banks
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = n * 8 + 2 * tq + h;
      float M = s_m[0][r];
#pragma unroll
      for (int w = 1; w < NW; ++w) M = fmax_nan(M, s_m[w][r]);
      const float f = m[n][h] == -INFINITY ? 0.f : ex2(m[n][h] - M);
      float *op = so + (warp * ROWS + r) * SO + g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        op[ks * 16] = acc[n][ks][h] * f;
        op[ks * 16 + 8] = acc[n][ks][2 + h] * f;
      }
    }
  __syncthreads();
  if constexpr (CL) {
    cluster_join<T, KC, D, ROWS, SO>(p, sp, so, s_m, s_l, s_blk);
  } else {
    split_write<D, ROWS, SO>(p, sp, so, s_m, s_l);
    if (last) pdl_wait();
  }
}

// ------------------------------------------------------------------ fp32
template <int D, int NR, bool CL>
__global__ void __launch_bounds__(NW * 32, SplitCfg<float, D>::MINB)
    split_f32_kernel(const SplitParams p, int rtiles, int min_chunks) {
  using C = SplitCfg<float, D>;
  constexpr int KC = C::KC, NST = C::NST, KS = D / 16, ROWS = 8 * NR, SO = D + 4;
  constexpr int VW = D >= 64 ? 4 : 2, VG = D / (16 * VW);  // columns per piece of V, column groups
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ int s_n;
  __shared__ float s_m[NW][ROWS], s_l[NW][ROWS];
  uint8_t *sQ = sm;                                   // fp32 rows first, then three bf16 terms [ROWS][D]
  uint8_t *ring = sm + 3 * ROWS * D * 2;
  int *s_blk = reinterpret_cast<int *>(ring + p.ring);  // with a selection: 3 * kMaxLive words
  float *s_gate = reinterpret_cast<float *>(s_blk + kMaxLive);
  const bool last = p.after && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, tq = lane & 3;
  pdl_trigger();
  Span sp;
  if (!split_span<KC, ROWS, CL>(p, rtiles, min_chunks, sp, s_blk, s_gate, s_blk + 2 * kMaxLive, &s_n)) {
    if (last) pdl_wait();
    return;
  }
  const int len = sp.len, r0 = sp.r0;
  const float *kb_ = reinterpret_cast<const float *>(p.k) + (p.fold ? 0 : sp.b * p.k_sb) + sp.hk * p.k_sh;
  const float *vb_ = reinterpret_cast<const float *>(p.v) + (p.fold ? 0 : sp.b * p.v_sb) + sp.hk * p.v_sh;
  uint8_t *wring = ring + warp * p.stages * C::STAGE;
  const uint32_t wr0 = smem_u32(wring);
  const uint64_t policy = evict_first_policy();
  const float *k2_ = nullptr, *v2_ = nullptr;  // the shared keys
  if constexpr (CL) {
    k2_ = reinterpret_cast<const float *>(p.k2) + sp.hk * p.k2_sh;
    v2_ = reinterpret_cast<const float *>(p.v2) + sp.hk * p.v2_sh;
  }
  auto load = [&](int c, int st) {
    if (c < sp.c_hi) {
      if (CL && c < sp.nch2) {
        split_load<float, D>(k2_, v2_, p.k2_sl, p.v2_sl, c * KC, p.n2, wr0 + st * C::STAGE, policy);
      } else {
        float gt;
        const int key0 = split_key<KC>(p, s_blk, s_gate, c - sp.nch2, gt);
        split_load<float, D>(kb_, vb_, p.k_sl, p.v_sl, key0, len, wr0 + st * C::STAGE, policy);
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) load(sp.c_lo + warp + s * NW, s);
  // the three terms of Q, in a thread's order: row g, dims 4t .. 4t+3 of a k-step
  for (int i = tid; i < ROWS * (D / 4); i += blockDim.x) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (r0 + r < p.R) {
      int rb, rh, rtt;
      split_row(p, sp.b, sp.hk, r0 + r, rb, rh, rtt);
      const float *qp = reinterpret_cast<const float *>(p.q) + rb * p.q_sb + rh * p.q_sh + rtt * p.q_sl + d;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = qp[e];
    }
    uint32_t u[3], w[3];
    split3(x[0], x[1], u);
    split3(x[2], x[3], w);
#pragma unroll
    for (int k = 0; k < 3; ++k)
      *reinterpret_cast<uint2 *>(sQ + k * ROWS * D * 2 + sw_off<2, D>(r, d / 8) + (d & 4) * 2) = make_uint2(u[k], w[k]);
  }
  __syncthreads();
  auto ldq = [&](int k, int n, int ks) {
    return *reinterpret_cast<const uint2 *>(sQ + k * ROWS * D * 2 + sw_off<2, D>(n * 8 + g, ks * 2 + (tq >> 1)) +
                                            (tq & 1) * 8);
  };
  constexpr bool QREG = NR == 1 && D <= 128;
  uint2 qf[QREG ? KS : 1][3];
  if constexpr (QREG)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int k = 0; k < 3; ++k) qf[ks][k] = ldq(k, 0, ks);

  // O^T: tile (v, e) holds columns v * 16 VW + VW g + e (and 8 VW further) x rows 2t, 2t + 1
  float acc[NR][KS][4], m[NR][2], l[NR][2];
  int qlast[NR][2];  // newest key that the row sees
#pragma unroll
  for (int n = 0; n < NR; ++n) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][ks][e] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[n][h] = -INFINITY;
      l[n][h] = 0.f;
      const int r = r0 + n * 8 + 2 * tq + h;
      qlast[n][h] = p.causal ? len - p.T + r % p.T : len - 1;
    }
  }
  const int all_see = p.causal ? len - p.T : len - 1;  // newest key that every row sees
  float *lg = p.logits ? p.logits + ((long long)sp.grpid * p.ncap + g) * p.rpad + r0 + 2 * tq : nullptr;

  int st = 0;
  for (int c = sp.c_lo + warp; c < sp.c_hi; c += NW) {
    if constexpr (NST == 1) {
      load(c, 0);  // D 256: a chunk is 32 KB, the other warps cover its way
      cp_wait<0>();
      __syncwarp();
    } else {
      cp_wait<NST - 2>();
      __syncwarp();
      int nst = st + NST - 1;
      if (nst >= NST) nst -= NST;
      load(c + (NST - 1) * NW, nst);
    }
    const uint8_t *sk = wring + st * C::STAGE, *sv = sk + KC * D * 4;
    const bool pre = CL && c < sp.nch2;  // shared keys: every row sees them
    float gate = 0.f;
    const int key0 = pre ? c * KC : split_key<KC>(p, s_blk, s_gate, c - sp.nch2, gate);
    // ---- S^T = K Q^T
    float s[NR][4], sr[NR][4];  // keys g, g + 8; rows 2t, 2t + 1: the leading products, the others
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = sr[n][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t a[3][4], u[3];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 x = *reinterpret_cast<const float4 *>(sk + sw_off<4, D>(g + 8 * h, ks * 4 + tq));
        split3_kv(x.x, x.y, u);
        a[0][h] = u[0], a[1][h] = u[1], a[2][h] = u[2];
        split3_kv(x.z, x.w, u);
        a[0][2 + h] = u[0], a[1][2 + h] = u[1], a[2][2 + h] = u[2];
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        uint2 q[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          if constexpr (QREG)
            q[k] = qf[ks][k];
          else
            q[k] = ldq(k, n, ks);
        }
        mma16<__nv_bfloat16>(s[n], a[0], q[0].x, q[0].y);
        mma16<__nv_bfloat16>(sr[n], a[2], q[0].x, q[0].y);
        mma16<__nv_bfloat16>(sr[n], a[0], q[2].x, q[2].y);
        mma16<__nv_bfloat16>(sr[n], a[1], q[1].x, q[1].y);
        mma16<__nv_bfloat16>(sr[n], a[1], q[0].x, q[0].y);
        mma16<__nv_bfloat16>(sr[n], a[0], q[1].x, q[1].y);
      }
    }
    // ---- online softmax (log2 domain); masked and missing keys are -inf
    const bool masked = key0 + KC - 1 > (pre ? p.n2 - 1 : all_see);
    const bool mixed = !pre && masked && all_see < len - 1;  // some row misses a key that another sees
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = fmaf(s[n][e] + sr[n][e], p.scale2, gate);
          if (masked && key0 + g + 8 * (e >> 1) > (pre ? p.n2 - 1 : qlast[n][e & 1])) x = -INFINITY;
          s[n][e] = x;
          mx[e & 1] = fmax_nan(mx[e & 1], x);
        }
      if (lg && r0 + n * 8 < p.R) {  // rows are padded to rpad: whole groups of eight
        float *lp = lg + (long long)c * KC * p.rpad + n * 8;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2 *>(lp + (long long)(8 * h) * p.rpad) =
                make_float2(s[n][2 * h], s[n][2 * h + 1]);
      }
      float al[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx[h] = fmax_nan(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], o));
        const float mn = fmax_nan(m[n][h], mx[h]);
        al[h] = mn == -INFINITY ? 1.f : ex2(m[n][h] - mn);
        m[n][h] = mn;
      }
      if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {
        l[n][0] *= al[0];
        l[n][1] *= al[1];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][ks][e] *= al[e & 1];
      }
      const float off[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] = ex2(s[n][e] - off[e & 1]);
          l[n][e & 1] += s[n][e];
        }
    }
    // ---- O^T += V^T P^T
    if (!mixed) {
      uint32_t pb[NR][2][3];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          split3(s[n][2 * h], s[n][2 * h + 1], pb[n][h]);
#pragma unroll
          for (int k = 0; k < 3; ++k) pb[n][h][k] = movmatrix(pb[n][h][k]);
        }
#pragma unroll
      for (int v = 0; v < VG; ++v) {
        float x[4][2][VW];  // keys 2t, 2t+1, 2t+8, 2t+9; columns and those 8 VW further
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int key = 2 * tq + (q & 1) + (q >> 1) * 8, col = (v * 2 + h) * 8 * VW + VW * g;
            const uint8_t *at = sv + sw_off<4, D>(key, col >> 2) + (col & 3) * 4;
            if constexpr (VW == 4)
              *reinterpret_cast<float4 *>(x[q][h]) = *reinterpret_cast<const float4 *>(at);
            else
              *reinterpret_cast<float2 *>(x[q][h]) = *reinterpret_cast<const float2 *>(at);
          }
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          uint32_t a[3][4], u[3];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            split3_kv(x[0][h][e], x[1][h][e], u);
            a[0][h] = u[0], a[1][h] = u[1], a[2][h] = u[2];
            split3_kv(x[2][h][e], x[3][h][e], u);
            a[0][2 + h] = u[0], a[1][2 + h] = u[1], a[2][2 + h] = u[2];
          }
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            float o[4] = {0.f, 0.f, 0.f, 0.f};  // this chunk's part (above)
            mma16<__nv_bfloat16>(o, a[2], pb[n][0][0], pb[n][1][0]);
            mma16<__nv_bfloat16>(o, a[0], pb[n][0][2], pb[n][1][2]);
            mma16<__nv_bfloat16>(o, a[1], pb[n][0][1], pb[n][1][1]);
            mma16<__nv_bfloat16>(o, a[1], pb[n][0][0], pb[n][1][0]);
            mma16<__nv_bfloat16>(o, a[0], pb[n][0][1], pb[n][1][1]);
            mma16<__nv_bfloat16>(o, a[0], pb[n][0][0], pb[n][1][0]);
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[n][v * VW + e][x] += o[x];
          }
        }
      }
    } else {
      // P through the chunk's K buffer (its reads are done), then key by key
      __syncwarp();
      float *sp_ = reinterpret_cast<float *>(wring + st * C::STAGE);  // [KC][ROWS]
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sp_[(g + 8 * (e >> 1)) * ROWS + n * 8 + 2 * tq + (e & 1)] = s[n][e];
      __syncwarp();
#pragma unroll 1
      for (int k = 0; k < KC && key0 + k < len; ++k) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const float2 pk = *reinterpret_cast<const float2 *>(sp_ + k * ROWS + n * 8 + 2 * tq);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const int c0 = (ks / VW) * 16 * VW + VW * g + ks % VW, c1 = c0 + 8 * VW;
            const float v0 = *reinterpret_cast<const float *>(sv + sw_off<4, D>(k, c0 >> 2) + (c0 & 3) * 4);
            const float v1 = *reinterpret_cast<const float *>(sv + sw_off<4, D>(k, c1 >> 2) + (c1 & 3) * 4);
            if (pk.x != 0.f) {
              acc[n][ks][0] = fmaf(pk.x, v0, acc[n][ks][0]);
              acc[n][ks][2] = fmaf(pk.x, v1, acc[n][ks][2]);
            }
            if (pk.y != 0.f) {
              acc[n][ks][1] = fmaf(pk.y, v0, acc[n][ks][1]);
              acc[n][ks][3] = fmaf(pk.y, v1, acc[n][ks][3]);
            }
          }
        }
      }
    }
    __syncwarp();
    if (++st == NST) st = 0;
  }

  // ---- join the four warps
  cp_wait<0>();
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], o);
      if (g == 0) {
        s_m[warp][n * 8 + 2 * tq + h] = m[n][h];
        s_l[warp][n * 8 + 2 * tq + h] = l[n][h];
      }
    }
  __syncthreads();
  float *so = reinterpret_cast<float *>(ring);  // [warp][ROWS][SO]; SO: rows 2t apart in banks
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = n * 8 + 2 * tq + h;
      float M = s_m[0][r];
#pragma unroll
      for (int w = 1; w < NW; ++w) M = fmax_nan(M, s_m[w][r]);
      const float f = m[n][h] == -INFINITY ? 0.f : ex2(m[n][h] - M);
      float *op = so + (warp * ROWS + r) * SO + VW * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        op[(ks / VW) * 16 * VW + ks % VW] = acc[n][ks][h] * f;
        op[(ks / VW) * 16 * VW + 8 * VW + ks % VW] = acc[n][ks][2 + h] * f;
      }
    }
  __syncthreads();
  if constexpr (CL) {
    cluster_join<float, KC, D, ROWS, SO>(p, sp, so, s_m, s_l, s_blk);
  } else {
    split_write<D, ROWS, SO>(p, sp, so, s_m, s_l);
    if (last) pdl_wait();
  }
}

// fp32, a shared prefix for many rows: the warps take different rows (16 each) and the
// same keys.  The chunk's K and V are turned into operands (three bf16 terms, in the order
// of the products' registers) once for the CTA, where the kernel above does it for every
// 16 or 32 rows: with many rows that was two thirds of its instructions.  Bound by the
// products (mma.sync): 1200 rows x 20000 keys, D 256, 8 heads, in 5.48 ms, 215 TFLOP/s of
// bf16 products (of 300 measured); 8.22 ms by the kernel above.  Which rows take it:
// rows_over_warps.
template <int D>
struct RowsCfg {
  static constexpr int W = D == 256 ? 4 : 8, NR = 2, ROWS = 8 * NR * W, KC = 16;
  static constexpr int STAGE = KC * D * 8, FRAGS = KC * D * 6;
  static constexpr int SMEM = 3 * ROWS * D * 2 + 2 * STAGE + 2 * FRAGS;
};

template <int D>
__global__ void __launch_bounds__(RowsCfg<D>::W * 32, 1)
    split_f32_rows_kernel(const SplitParams p, int rtiles) {
  using C = RowsCfg<D>;
  constexpr int KC = C::KC, NR = C::NR, KS = D / 16, ROWS = C::ROWS;
  constexpr int VW = D >= 64 ? 4 : 2, VG = D / (16 * VW);
  extern __shared__ __align__(128) uint8_t sm[];
  uint8_t *sQ = sm;                              // three bf16 terms [ROWS][D]
  uint8_t *raw = sm + 3 * ROWS * D * 2;          // [stage]: K and V as they are
  uint4 *fk = reinterpret_cast<uint4 *>(raw + 2 * C::STAGE);  // [k-step][term][lane]
  uint4 *fv = fk + KS * 3 * 32;                  // [tile of O^T][term][lane]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, tq = lane & 3;
  pdl_trigger();
  const int hk = blockIdx.x / rtiles, row0 = (blockIdx.x % rtiles) * ROWS, r0 = row0 + warp * 8 * NR;
  const int len = p.nkeys, nch = (len + KC - 1) / KC, cps = (nch + p.nsplit - 1) / p.nsplit;
  const int c_lo = min(nch, (int)blockIdx.y * cps), c_hi = min(nch, c_lo + cps), split = p.split0 + blockIdx.y;
  int rb, rh, rtt;
  if (c_lo >= c_hi) {
    for (int r = row0 + tid; r < min(p.R, row0 + ROWS); r += C::W * 32)
      p.pml[(long long)split * p.rows + split_row(p, 0, hk, r, rb, rh, rtt)] = make_float2(-INFINITY, 0.f);
    return;
  }
  const float *kb_ = reinterpret_cast<const float *>(p.k) + hk * p.k_sh;
  const float *vb_ = reinterpret_cast<const float *>(p.v) + hk * p.v_sh;
  const uint32_t raw0 = smem_u32(raw);
  auto load = [&](int c) {
    if (c < c_hi) {
      const uint32_t dk = raw0 + (c & 1) * C::STAGE, dv = dk + KC * D * 4;
#pragma unroll
      for (int it = 0; it < KC * D / 4 / (C::W * 32); ++it) {
        const int i = it * C::W * 32 + tid, row = i / (D / 4), ch = i % (D / 4);
        const bool ok = c * KC + row < len;
        const int64_t key = ok ? c * KC + row : 0;
        const uint32_t off = sw_off<4, D>(row, ch);
        cp16(dk + off, kb_ + key * p.k_sl + ch * 4, ok);
        cp16(dv + off, vb_ + key * p.v_sl + ch * 4, ok);
      }
    }
    cp_commit();
  };
  load(c_lo);
  for (int i = tid; i < ROWS * (D / 4); i += blockDim.x) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (row0 + r < p.R) {
      split_row(p, 0, hk, row0 + r, rb, rh, rtt);
      const float *qp = reinterpret_cast<const float *>(p.q) + rb * p.q_sb + rh * p.q_sh + rtt * p.q_sl + d;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = qp[e];
    }
    uint32_t u[3], w[3];
    split3(x[0], x[1], u);
    split3(x[2], x[3], w);
#pragma unroll
    for (int k = 0; k < 3; ++k)
      *reinterpret_cast<uint2 *>(sQ + k * ROWS * D * 2 + sw_off<2, D>(r, d / 8) + (d & 4) * 2) = make_uint2(u[k], w[k]);
  }

  float acc[NR][KS][4], m[NR][2], l[NR][2];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][ks][e] = 0.f;
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
  }
  for (int c = c_lo; c < c_hi; ++c) {
    cp_wait<0>();
    __syncthreads();  // the chunk is here, and nobody reads the last one's operands
    load(c + 1);
    const uint8_t *sk = raw + (c & 1) * C::STAGE, *sv = sk + KC * D * 4;
    for (int i = tid; i < KS * 32; i += C::W * 32) {  // K: (k-step, lane)
      const int ks = i >> 5, gg = (i & 31) >> 2, tt = i & 3;
      uint4 f[3];
      uint32_t u[3];
      const float4 x = *reinterpret_cast<const float4 *>(sk + sw_off<4, D>(gg, ks * 4 + tt));
      const float4 y = *reinterpret_cast<const float4 *>(sk + sw_off<4, D>(gg + 8, ks * 4 + tt));
      split3_kv(x.x, x.y, u);
      f[0].x = u[0], f[1].x = u[1], f[2].x = u[2];
      split3_kv(y.x, y.y, u);
      f[0].y = u[0], f[1].y = u[1], f[2].y = u[2];
      split3_kv(x.z, x.w, u);
      f[0].z = u[0], f[1].z = u[1], f[2].z = u[2];
      split3_kv(y.z, y.w, u);
      f[0].w = u[0], f[1].w = u[1], f[2].w = u[2];
#pragma unroll
      for (int k = 0; k < 3; ++k) fk[(ks * 3 + k) * 32 + (i & 31)] = f[k];
    }
    for (int i = tid; i < VG * 32; i += C::W * 32) {  // V: (column group, lane), VW tiles each
      const int v = i >> 5, gg = (i & 31) >> 2, tt = i & 3;
      float x[4][2][VW];
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = 2 * tt + (q & 1) + (q >> 1) * 8, col = (v * 2 + h) * 8 * VW + VW * gg;
          const uint8_t *at = sv + sw_off<4, D>(key, col >> 2) + (col & 3) * 4;
          if constexpr (VW == 4)
            *reinterpret_cast<float4 *>(x[q][h]) = *reinterpret_cast<const float4 *>(at);
          else
            *reinterpret_cast<float2 *>(x[q][h]) = *reinterpret_cast<const float2 *>(at);
        }
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        uint4 f[3];
        uint32_t u[3];
        split3_kv(x[0][0][e], x[1][0][e], u);
        f[0].x = u[0], f[1].x = u[1], f[2].x = u[2];
        split3_kv(x[0][1][e], x[1][1][e], u);
        f[0].y = u[0], f[1].y = u[1], f[2].y = u[2];
        split3_kv(x[2][0][e], x[3][0][e], u);
        f[0].z = u[0], f[1].z = u[1], f[2].z = u[2];
        split3_kv(x[2][1][e], x[3][1][e], u);
        f[0].w = u[0], f[1].w = u[1], f[2].w = u[2];
#pragma unroll
        for (int k = 0; k < 3; ++k) fv[((v * VW + e) * 3 + k) * 32 + (i & 31)] = f[k];
      }
    }
    __syncthreads();
    // ---- S^T = K Q^T
    float s[NR][4], sr[NR][4];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = sr[n][e] = 0.f;
#pragma unroll 4
    for (int ks = 0; ks < KS; ++ks) {
      uint4 a[3];
#pragma unroll
      for (int k = 0; k < 3; ++k) a[k] = fk[(ks * 3 + k) * 32 + lane];
      const uint32_t a0[4] = {a[0].x, a[0].y, a[0].z, a[0].w}, a1[4] = {a[1].x, a[1].y, a[1].z, a[1].w};
      const uint32_t a2[4] = {a[2].x, a[2].y, a[2].z, a[2].w};
      uint2 q[NR][3];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int k = 0; k < 3; ++k)
          q[n][k] = *reinterpret_cast<const uint2 *>(
              sQ + k * ROWS * D * 2 + sw_off<2, D>(warp * 8 * NR + n * 8 + g, ks * 2 + (tq >> 1)) + (tq & 1) * 8);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(s[n], a0, q[n][0].x, q[n][0].y);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(sr[n], a2, q[n][0].x, q[n][0].y);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(sr[n], a0, q[n][2].x, q[n][2].y);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(sr[n], a1, q[n][1].x, q[n][1].y);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(sr[n], a1, q[n][0].x, q[n][0].y);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(sr[n], a0, q[n][1].x, q[n][1].y);
    }
    // ---- online softmax (log2 domain); missing keys are -inf
    uint32_t pb[NR][2][3];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = (s[n][e] + sr[n][e]) * p.scale2;
        if (c * KC + g + 8 * (e >> 1) >= len) x = -INFINITY;
        s[n][e] = x;
        mx[e & 1] = fmax_nan(mx[e & 1], x);
      }
      float al[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx[h] = fmax_nan(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], o));
        const float mn = fmax_nan(m[n][h], mx[h]);
        al[h] = mn == -INFINITY ? 1.f : ex2(m[n][h] - mn);
        m[n][h] = mn;
      }
      if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {
        l[n][0] *= al[0];
        l[n][1] *= al[1];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][ks][e] *= al[e & 1];
      }
      const float off[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = ex2(s[n][e] - off[e & 1]);
        l[n][e & 1] += s[n][e];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        split3(s[n][2 * h], s[n][2 * h + 1], pb[n][h]);
#pragma unroll
        for (int k = 0; k < 3; ++k) pb[n][h][k] = movmatrix(pb[n][h][k]);
      }
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint4 a[3];
#pragma unroll
      for (int k = 0; k < 3; ++k) a[k] = fv[(ks * 3 + k) * 32 + lane];
      const uint32_t a0[4] = {a[0].x, a[0].y, a[0].z, a[0].w}, a1[4] = {a[1].x, a[1].y, a[1].z, a[1].w};
      const uint32_t a2[4] = {a[2].x, a[2].y, a[2].z, a[2].w};
      float o[NR][4];
#pragma unroll
      for (int n = 0; n < NR; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(o[n], a2, pb[n][0][0], pb[n][1][0]);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(o[n], a0, pb[n][0][2], pb[n][1][2]);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(o[n], a1, pb[n][0][1], pb[n][1][1]);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(o[n], a1, pb[n][0][0], pb[n][1][0]);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(o[n], a0, pb[n][0][1], pb[n][1][1]);
#pragma unroll
      for (int n = 0; n < NR; ++n) mma16<__nv_bfloat16>(o[n], a0, pb[n][0][0], pb[n][1][0]);
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][ks][e] += o[n][e];
    }
  }
  // ---- this warp's rows
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], o);
      const int r = r0 + n * 8 + 2 * tq + h;
      if (r >= p.R) continue;
      const long long at = (long long)split * p.rows + split_row(p, 0, hk, r, rb, rh, rtt);
      if (g == 0) p.pml[at] = make_float2(m[n][h], l[n][h]);
      float *op = p.po + at * D + VW * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        op[(ks / VW) * 16 * VW + ks % VW] = acc[n][ks][h];
        op[(ks / VW) * 16 * VW + 8 * VW + ks % VW] = acc[n][ks][2 + h];
      }
    }
}

// ------------------------------------------------------------------ join
struct JoinParams {
  void *o;
  int64_t o_sb, o_sh, o_sl;
  int B, Hq, Hkv, grp, T, D, nsplit, R;
  long long rows;
  const float *po;
  const float2 *pml;
  const float *logits;  // with weights: [b*Hkv + hk][ncap][rpad]
  long long ncap;
  int rpad;
  const int *live;
  int kk, bs, L;
  float *weight;
  int64_t w_sb, w_sh;
  int wtiles, kpb;      // weight blocks per (b, hk) and slots of each; they follow the row blocks
};

constexpr int kJoinThreads = 256;

// Row blocks: 8 / wpr query rows each.  A row's columns take D/4 lanes; the remaining
// lanes of its warps, and its wpr warps, take splits side by side.  Weight blocks:
// kpb slots of one (b, hk): lse of its R rows from the splits' (m, l), then the sum over
// the rows of 2^(x - m) / l, eight rows to a lane and LPK lanes to a slot, so that a
// warp reads whole lines of the logits.
template <int LPK, bool SEL>
__device__ __forceinline__ void join_weights(const JoinParams &p, int bh, int b, int hk, int tile, const float *sj) {
  constexpr int KPW = 32 / LPK, STEP = KPW * (kJoinThreads / 32);  // slots of a warp, of the CTA per step
  constexpr int U = 4;                                             // steps in flight
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LPK;
  const int *lv = SEL ? p.live + (long long)bh * (1 + p.kk) : nullptr;
  const int nv = SEL ? lv[0] * p.bs : p.L;       // (virtual) slots
  const int jw0 = tile * p.kpb + warp * KPW;     // the warp's first slot
  const int end = min(nv, tile * p.kpb + p.kpb);
  float *wp = p.weight + b * p.w_sb + hk * p.w_sh;
  const float *lg = p.logits + ((long long)bh * p.ncap + jw0 + lane / LPK) * p.rpad + sub * 8;
  const int step = STEP * p.rpad;
  // this lane's first eight rows (none when there are fewer)
  float m8[8], f8[8];
  const bool rows = sub * 8 < p.rpad;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    m8[e] = rows ? sj[sub * 8 + e] : 0.f;
    f8[e] = rows ? sj[p.rpad + sub * 8 + e] : 0.f;
  }
  for (int jw = jw0; jw < end; jw += U * STEP, lg += U * step) {
    float4 x4[U][2];
    float w0[U];
    int key[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = jw + u * STEP + lane / LPK;
      const bool in = j < end;
      key[u] = j;
      if (SEL && in) {  // the warp's slots lie in one block (bs is a multiple of 32)
        const int blk = (jw + u * STEP) / p.bs;
        key[u] = lv[1 + blk] * p.bs + (j - blk * p.bs);
      }
      const bool live = in && (!SEL || key[u] < p.L);
      x4[u][0] = x4[u][1] = make_float4(0, 0, 0, 0);
      w0[u] = 0.f;
      if (live && rows) {
        x4[u][0] = __ldcs(reinterpret_cast<const float4 *>(lg + u * step));
        x4[u][1] = __ldcs(reinterpret_cast<const float4 *>(lg + u * step + 4));
      }
      if (live && sub == 0) w0[u] = wp[key[u]];
      if (!live) key[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float w = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w += (join_p(x4[u][h].x, m8[4 * h], f8[4 * h]) + join_p(x4[u][h].y, m8[4 * h + 1], f8[4 * h + 1])) +
             (join_p(x4[u][h].z, m8[4 * h + 2], f8[4 * h + 2]) + join_p(x4[u][h].w, m8[4 * h + 3], f8[4 * h + 3]));
      if (LPK == 4 && key[u] >= 0)  // more than 32 rows
        for (int r = LPK * 8; r + sub * 8 < p.rpad; r += LPK * 8) {
          const float *x = lg + u * step + r, *sm = sj + r + sub * 8, *sf = sm + p.rpad;
#pragma unroll
          for (int e = 0; e < 8; ++e) w += join_p(x[e], sm[e], sf[e]);
        }
#pragma unroll
      for (int o = 1; o < LPK; o <<= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
      if (key[u] >= 0 && sub == 0) wp[key[u]] = w0[u] + w;
    }
  }
}

template <int LPK>
__device__ __forceinline__ void join_weights(const JoinParams &p, int bh, int b, int hk, int tile, const float *sj) {
  if (p.live)
    join_weights<LPK, true>(p, bh, b, hk, tile, sj);
  else
    join_weights<LPK, false>(p, bh, b, hk, tile, sj);
}

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) split_join_kernel(const JoinParams p, const int wpr) {
  extern __shared__ __align__(16) float sj[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rpb = 8 / wpr;
  const long long rblocks = (p.rows + rpb - 1) / rpb;
  pdl_wait();
  if (blockIdx.x < rblocks) {
    constexpr int LPR = D / 4 < 32 ? D / 4 : 32, G = 32 / LPR, V = D / 4 / LPR;
    const int sub = warp % wpr, col = (lane % LPR) * 4;
    const long long gr = blockIdx.x * (long long)rpb + warp / wpr;
    const bool live = gr < p.rows;
    float m = -INFINITY;
    if (live)
      for (int s = lane; s < p.nsplit; s += 32) m = fmax_nan(m, p.pml[s * p.rows + gr].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    float4 acc[V];
#pragma unroll
    for (int c = 0; c < V; ++c) acc[c] = make_float4(0, 0, 0, 0);
    float l = 0.f;
    if (live && m != -INFINITY) {
#pragma unroll 4
      for (int s = sub * G + lane / LPR; s < p.nsplit; s += wpr * G) {
        const float2 ml = p.pml[s * p.rows + gr];
        if (ml.x == -INFINITY) continue;  // its O was not written
        const float f = ex2(ml.x - m);
        l = fmaf(ml.y, f, l);
        const float *op = p.po + (s * p.rows + gr) * D + col;
#pragma unroll
        for (int c = 0; c < V; ++c) {
          const float4 x = *reinterpret_cast<const float4 *>(op + 128 * c);
          acc[c].x = fmaf(x.x, f, acc[c].x);
          acc[c].y = fmaf(x.y, f, acc[c].y);
          acc[c].z = fmaf(x.z, f, acc[c].z);
          acc[c].w = fmaf(x.w, f, acc[c].w);
        }
      }
    }
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
      l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
      for (int c = 0; c < V; ++c) {
        acc[c].x += __shfl_xor_sync(0xffffffffu, acc[c].x, o);
        acc[c].y += __shfl_xor_sync(0xffffffffu, acc[c].y, o);
        acc[c].z += __shfl_xor_sync(0xffffffffu, acc[c].z, o);
        acc[c].w += __shfl_xor_sync(0xffffffffu, acc[c].w, o);
      }
    }
    if (wpr > 1) {  // the row's other warps, through shared memory: [warp][D] and [warp]
      float *sl = sj + 8 * D;
      if (lane < LPR)
#pragma unroll
        for (int c = 0; c < V; ++c) *reinterpret_cast<float4 *>(sj + warp * D + col + 128 * c) = acc[c];
      if (lane == 0) sl[warp] = l;
      __syncthreads();
      if (sub != 0) return;
      for (int w = 1; w < wpr; ++w) {
        l += sl[warp + w];
#pragma unroll
        for (int c = 0; c < V; ++c) {
          const float4 x = *reinterpret_cast<const float4 *>(sj + (warp + w) * D + col + 128 * c);
          acc[c].x += x.x;
          acc[c].y += x.y;
          acc[c].z += x.z;
          acc[c].w += x.w;
        }
      }
    }
    if (!live || lane >= LPR) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int t = (int)(gr % p.T);
    const long long bh = gr / p.T;
    T *op = reinterpret_cast<T *>(p.o) + (bh / p.Hq) * p.o_sb + (bh % p.Hq) * p.o_sh + t * p.o_sl + col;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const float y[4] = {acc[c].x * inv, acc[c].y * inv, acc[c].z * inv, acc[c].w * inv};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 2)
          op[128 * c + e] = Mma<T>::from_f(y[e]);
        else
          op[128 * c + e] = y[e];
      }
    }
    return;
  }
  const long long wb = blockIdx.x - rblocks;
  const int bh = (int)(wb / p.wtiles), tile = (int)(wb % p.wtiles);
  const int b = bh / p.Hkv, hk = bh % p.Hkv;
  for (int r = warp; r < p.R; r += 8) {
    const long long gr = ((long long)b * p.Hq + hk * p.grp) * p.T + r;
    float m = -INFINITY;
    for (int s = lane; s < p.nsplit; s += 32) m = fmax_nan(m, p.pml[s * p.rows + gr].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    float l = 0.f;
    for (int s = lane; s < p.nsplit; s += 32) {
      const float2 ml = p.pml[s * p.rows + gr];
      if (ml.x != -INFINITY) l = fmaf(ml.y, ex2(ml.x - m), l);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) {  // offset and factor of the row
      sj[r] = m;
      sj[p.rpad + r] = l == 0.f ? 0.f : 1.f / l;
    }
  }
  for (int r = p.R + tid; r < p.rpad; r += kJoinThreads) sj[r] = sj[p.rpad + r] = 0.f;
  __syncthreads();
  if (p.rpad == 8)
    join_weights<1>(p, bh, b, hk, tile, sj);
  else if (p.rpad == 16)
    join_weights<2>(p, bh, b, hk, tile, sj);
  else
    join_weights<4>(p, bh, b, hk, tile, sj);
}

// ------------------------------------------------------------------ launchers
// Number of key splits: the one with the least (waves of CTAs) x (key steps of a
// CTA + its fixed cost in steps), for `groups` CTAs per split and `slots` resident.
static int choose_split(long long groups, long long steps, int slots, int fixed, int cap) {
  long long best = -1;
  int ns = 1;
  for (int s = 1; s <= cap && s <= std::max<long long>(1, steps); ++s) {
    const long long cost = ((groups * s + slots - 1) / slots) * ((steps + s - 1) / s + fixed);
    if (best < 0 || cost < best) {
      best = cost;
      ns = s;
    }
  }
  return ns;
}

constexpr int kMaxSplit = 296;

template <typename T, int D>
static int split_count_t(long long groups, int R, long long n, int sms) {
  using C = SplitCfg<T, D>;
  const int rows = split_rows<T, D>(R);
  const long long step = C::KC * NW;
  return choose_split(groups * ((R + rows - 1) / rows), (n + step - 1) / step, sms * C::MINB, 4, kMaxSplit);
}

// Whether the rows of a shared prefix go over the warps (split_f32_rows_kernel).  Times of
// it against split_f32_kernel, 20000 keys, 8 heads, us: D 256, 36 rows 294 : 378, 1200 rows
// 5484 : 8224; D 128, 64 rows 246 : 212, 96 rows 248 : 310, 1200 rows 2325 : 3424; D 64,
// 96 rows 154 : 112, 1200 rows 1410 : 1249 (its barriers and the one CTA per SM show where
// a chunk has few products).
static bool rows_over_warps(int dtype, int D, bool fold, int R) {
  return dtype == BSA_F32 && fold && (D == 256 ? R > 32 : D == 128 && R > 64);
}

// Splits of the partial kernel for n keys, `groups` K/V head groups and R rows each, on
// `sms` SMs.
int split_count(int dtype, int D, long long groups, int R, long long n, bool fold = false, int sms = 148) {
  const bool f = dtype == BSA_F32;
  if (rows_over_warps(dtype, D, fold, R)) {
    const int rows = D == 256 ? RowsCfg<256>::ROWS : RowsCfg<128>::ROWS;
    return choose_split(groups * ((R + rows - 1) / rows), (n + 15) / 16, 148, 6, kMaxSplit);
  }
  switch (D) {
    case 32: return f ? split_count_t<float, 32>(groups, R, n, sms) : split_count_t<__half, 32>(groups, R, n, sms);
    case 64: return f ? split_count_t<float, 64>(groups, R, n, sms) : split_count_t<__half, 64>(groups, R, n, sms);
    case 128: return f ? split_count_t<float, 128>(groups, R, n, sms) : split_count_t<__half, 128>(groups, R, n, sms);
    default: return f ? split_count_t<float, 256>(groups, R, n, sms) : split_count_t<__half, 256>(groups, R, n, sms);
  }
}

template <typename T, int D, int ROWS, bool CL>
static bsa_status launch_rows(SplitParams p, long long groups, cudaStream_t st) {
  using C = SplitCfg<T, D>;
  const int rtiles = (p.R + ROWS - 1) / ROWS;
  constexpr int rows = ROWS * D * (C::ES == 4 ? 6 : 2), join = NW * ROWS * (D + 4) * 4;
  constexpr int most = rows + C::RING + 3 * kMaxLive * 4;
  static_assert(C::RING >= join, "the ring holds the warps' O for the join");
  static_assert(C::KC * D * C::ES >= ROWS * C::KC * 4, "a chunk's K buffer holds its P");
  void (*kern)(const SplitParams, int, int);
  if constexpr (C::ES == 2)
    kern = split_mma_kernel<T, D, ROWS / 8, CL>;
  else
    kern = split_f32_kernel<D, ROWS / 8, CL>;
  static std::atomic<uint64_t> done{0};
  allow_smem(reinterpret_cast<const void *>(kern), most, done);
  // The ring: no more warps and stages than a CTA has chunks, so that short caches get more
  // CTAs per SM (D 256, 1256 heads of 21 slots, us: fp32 79 -> 47, bf16 45 -> 27).
  const long long n = p.sel ? (long long)p.kk * p.bs : p.nkeys;
  const long long nch = (CL ? (p.n2 + C::KC - 1) / C::KC : 0) + (n + C::KC - 1) / C::KC;
  const long long cps = std::max<long long>(NW, (nch + p.nsplit - 1) / p.nsplit);
  p.stages = (int)std::min<long long>(C::NST, (cps + NW - 1) / NW);
  p.ring = std::max(join, (int)std::min<long long>(NW, nch) * p.stages * C::STAGE);
  const dim3 grid((unsigned)(groups * rtiles), p.nsplit);
  const int smem = rows + p.ring + (p.sel ? 3 * kMaxLive * 4 : 0);
  if constexpr (CL) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(NW * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 1, at.val.clusterDim.y = p.nsplit, at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kern, p, rtiles, NW);
  } else if (p.after) {
    launch_after(kern, grid, NW * 32, smem, st, p, rtiles, NW);
  } else {
    kern<<<grid, NW * 32, smem, st>>>(p, rtiles, NW);
  }
  return check_launch("split");
}

template <typename T, int D, bool CL>
static bsa_status launch_mma_d(const SplitParams &p, long long groups, cudaStream_t st) {
  const int rows = split_rows<T, D>(p.R);
  if (rows == 8) return launch_rows<T, D, 8, CL>(p, groups, st);
  if constexpr (SplitCfg<T, D>::MAXROWS == 32)
    if (rows == 32) return launch_rows<T, D, 32, CL>(p, groups, st);
  return launch_rows<T, D, 16, CL>(p, groups, st);
}

template <int D>
static bsa_status launch_f32_rows(const SplitParams &p, long long groups, cudaStream_t st) {
  using C = RowsCfg<D>;
  static_assert(C::SMEM <= 232448, "shared memory of one CTA");
  const int rtiles = (p.R + C::ROWS - 1) / C::ROWS;
  static std::atomic<uint64_t> done{0};
  allow_smem(reinterpret_cast<const void *>(split_f32_rows_kernel<D>), C::SMEM, done);
  split_f32_rows_kernel<D>
      <<<dim3((unsigned)(groups * rtiles), p.nsplit), C::W * 32, C::SMEM, st>>>(p, rtiles);
  return check_launch("split_f32_rows");
}

template <int D, bool CL>
static bsa_status launch_split_d(int dtype, const SplitParams &p, long long groups, cudaStream_t st) {
  if constexpr (!CL && D >= 128)
    if (rows_over_warps(dtype, D, p.fold, p.R)) return launch_f32_rows<D>(p, groups, st);
  if (dtype == BSA_BF16) return launch_mma_d<__nv_bfloat16, D, CL>(p, groups, st);
  if (dtype == BSA_F16) return launch_mma_d<__half, D, CL>(p, groups, st);
  return launch_mma_d<float, D, CL>(p, groups, st);
}

template <bool CL>
static bsa_status launch_split(int dtype, int D, const SplitParams &p, cudaStream_t st) {
  const long long groups = p.fold ? p.Hkv : (long long)p.B * p.Hkv;
  switch (D) {
    case 32: return launch_split_d<32, CL>(dtype, p, groups, st);
    case 64: return launch_split_d<64, CL>(dtype, p, groups, st);
    case 128: return launch_split_d<128, CL>(dtype, p, groups, st);
    default: return launch_split_d<256, CL>(dtype, p, groups, st);
  }
}

// CTAs of the cluster that does a (b, hk) of R rows and n keys in one launch, or 0 where
// splits and a join are the better way: more rows than a tile, or more than 16 rounds of a
// CTA's warps in all (fp32: 4, its rounds are three times as long), unless one CTA per head
// is what the splits come to.  One launch saves 3 us of the host's time and the partial
// sums' way through memory; with few heads and many keys eight CTAs per head draw too little
// of HBM.  Device time, clusters : splits, us: bf16, D 256, one sequence, 1000 slots, 2 heads
// 10.4 : 8.9, 2000 slots, 8 heads 12.2 : 9.6; fp32, D 128, 500 slots, 32 heads 11.2 : 12.1,
// 1000 slots, 16 heads 22.3 : 12.6.  All CTAs of a launch have to run at once (bf16, D 256,
// 148 heads of 300 slots: 20.4 in pairs, one CTA per SM, 12.3 alone).
static int cluster_size(int dtype, int D, long long groups, int R, long long n) {
  const int es = (int)elem_size(dtype), kc = es == 2 && D <= 64 ? 32 : 16;
  const int most = D == 256 || (es == 2 && D == 32) ? 16 : 32;
  const long long steps = (n + kc * NW - 1) / (kc * NW);
  if (R > most) return 0;
  if (steps > (es == 4 ? 4 : 16)) return split_count(dtype, D, groups, R, n) == 1 ? 1 : 0;
  const int slots = kc * D * es * 2 >= 16384 ? 148 : 2 * 148;  // SplitCfg's CTAs per SM
  int cs = 1;
  while (cs < 8 && cs * 2 <= steps && groups * cs * 2 <= slots) cs *= 2;
  return cs;
}

template <typename T>
static void launch_join_t(const JoinParams &p, cudaStream_t st) {
  // warps per row: enough that a warp walks a few splits at most (8 loads in flight)
  const int wpr = p.nsplit <= 8 ? 1 : p.nsplit <= 16 ? 2 : p.nsplit <= 32 ? 4 : 8;
  const long long rblocks = (p.rows * wpr + 7) / 8;
  const dim3 grid((unsigned)(rblocks + (p.weight ? (long long)p.B * p.Hkv * p.wtiles : 0)));
  const size_t smem = std::max<size_t>((8 * p.D + 8) * 4, p.weight ? (size_t)p.rpad * 8 : 0);
  switch (p.D) {
    case 32: return launch_after(split_join_kernel<T, 32>, grid, kJoinThreads, smem, st, p, wpr);
    case 64: return launch_after(split_join_kernel<T, 64>, grid, kJoinThreads, smem, st, p, wpr);
    case 128: return launch_after(split_join_kernel<T, 128>, grid, kJoinThreads, smem, st, p, wpr);
    default: return launch_after(split_join_kernel<T, 256>, grid, kJoinThreads, smem, st, p, wpr);
  }
}

static bsa_status launch_join(int dtype, const JoinParams &p, cudaStream_t st) {
  if (dtype == BSA_BF16)
    launch_join_t<__nv_bfloat16>(p, st);
  else if (dtype == BSA_F16)
    launch_join_t<__half>(p, st);
  else
    launch_join_t<float>(p, st);
  return check_launch("split_join");
}

static bsa_status check_rows(const char *who, int dtype, int B, int Hq, int Hkv, int D, int T, float scale) {
  const std::string w(who);
  if (dtype != BSA_BF16 && dtype != BSA_F16 && dtype != BSA_F32)
    return fail(BSA_ERR_DTYPE, w + ": dtype must be bf16, f16 or f32");
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || Hq % Hkv)
    return fail(BSA_ERR_SHAPE, w + ": sizes must be positive and Hq a multiple of Hkv");
  if (D != 32 && D != 64 && D != 128 && D != 256)
    return fail(BSA_ERR_UNSUPPORTED, w + ": D must be 32, 64, 128 or 256");
  if ((long long)B * Hq * T >= (1LL << 30)) return fail(BSA_ERR_SHAPE, w + ": B*Hq*T too large");
  if (!(scale > 0.f) || !std::isfinite(scale)) return fail(BSA_ERR_ARG, w + ": bad scale");
  return BSA_OK;
}

// A K/V operand: 16-byte aligned base and strides.
static bsa_status check_kv(const bsa_view &v, int dtype, const char *who, const char *name, bool batch) {
  const int64_t es = (int64_t)elem_size(dtype);
  if (!v.ptr) return fail(BSA_ERR_ARG, std::string(who) + ": " + name + " is NULL");
  if (reinterpret_cast<uintptr_t>(v.ptr) % 16 || (v.sl * es) % 16 || (v.sh * es) % 16 ||
      (batch && (v.sb * es) % 16))
    return fail(BSA_ERR_STRIDE, std::string(who) + ": " + name + " needs a 16-byte aligned base and strides");
  return BSA_OK;
}

// ------------------------------------------------------------------ decode_weighted
bool lies_apart(int64_t B, int64_t sb, int64_t H, int64_t sh, int64_t L, int64_t sl, int64_t D) {
  std::pair<int64_t, int64_t> ax[3] = {{sb, B}, {sh, H}, {sl, L}};
  std::sort(ax, ax + 3);
  int64_t span = D;
  for (const auto &[stride, n] : ax) {
    if (n <= 1) continue;
    if (stride < span) return false;
    span += stride * (n - 1);
  }
  return true;
}

// The output of a decode step.
static bsa_status check_out(const char *who, const bsa_view &o, int B, int Hq, int T, int D) {
  if (!o.ptr) return fail(BSA_ERR_ARG, std::string(who) + ": o is NULL");
  if (!lies_apart(B, o.sb, Hq, o.sh, T, o.sl, D))
    return fail(BSA_ERR_STRIDE, std::string(who) + ": rows of o share memory");
  return BSA_OK;
}

namespace {
constexpr int kMaxWeightRows = 4096;
struct WeightedPlan {
  int cl, nsplit;  // cl: CTAs of a cluster per head (one launch), or 0
  int rpad;
  long long ncap, rows;
  size_t o_po, o_ml, o_lg, o_lv, bytes;
};
WeightedPlan weighted_plan(const bsa_decode_weighted_args *a) {
  WeightedPlan w;
  const int R = (a->Hq / a->Hkv) * a->T;
  const long long n = a->sel ? (long long)a->kk * a->bs : a->L;
  w.cl = cluster_size(a->dtype, a->D, (long long)a->B * a->Hkv, R, n);
  w.nsplit = w.cl ? w.cl : split_count(a->dtype, a->D, (long long)a->B * a->Hkv, R, n);
  w.ncap = (n + 31) / 32 * 32;
  w.rpad = (R + 7) / 8 * 8;
  w.rows = (long long)a->B * a->Hq * a->T;
  const size_t parts = w.cl ? 0 : (size_t)w.nsplit * w.rows;
  w.o_po = 0;
  w.o_ml = align_up(parts * a->D * 4, 256);
  w.o_lg = align_up(w.o_ml + parts * 8, 256);
  w.o_lv = align_up(w.o_lg + (size_t)a->B * a->Hkv * w.rpad * w.ncap * 4, 256);
  w.bytes = align_up(w.o_lv + (a->sel ? (size_t)a->B * a->Hkv * (1 + a->kk) * 4 : 0), 256);
  return w;
}
}  // namespace

static bsa_status weighted_check(const bsa_decode_weighted_args *a) {
  if (bsa_status s = check_rows("decode_weighted", a->dtype, a->B, a->Hq, a->Hkv, a->D, a->T, a->scale)) return s;
  if (a->L <= 0 || a->T > a->L) return fail(BSA_ERR_SHAPE, "decode_weighted: needs 1 <= T <= L");
  if ((a->Hq / a->Hkv) * (long long)a->T > kMaxWeightRows)
    return fail(BSA_ERR_UNSUPPORTED, "decode_weighted: (Hq/Hkv) * T must be <= 4096");
  if (a->sel) {
    if (a->kk <= 0) return fail(BSA_ERR_SHAPE, "decode_weighted: kk must be positive");
    if (a->kk > kMaxLive) return fail(BSA_ERR_UNSUPPORTED, "decode_weighted: kk must be <= 512");
    if (a->bs <= 0 || a->bs % 32) return fail(BSA_ERR_UNSUPPORTED, "decode_weighted: bs must be a multiple of 32");
    if ((long long)a->kk * a->bs >= (1LL << 30)) return fail(BSA_ERR_SHAPE, "decode_weighted: kk*bs too large");
  } else if (a->gate) {
    return fail(BSA_ERR_ARG, "decode_weighted: a gate needs a selection");
  }
  if (a->L >= (1 << 30)) return fail(BSA_ERR_SHAPE, "decode_weighted: L too large");
  if (!a->q.ptr || !a->weight) return fail(BSA_ERR_ARG, "decode_weighted: NULL tensor");
  if (bsa_status s = check_out("decode_weighted", a->o, a->B, a->Hq, a->T, a->D)) return s;
  if (!lies_apart(a->B, a->weight_sb, a->Hkv, a->weight_sh, 1, 0, a->L))
    return fail(BSA_ERR_STRIDE, "decode_weighted: rows of weight share memory");
  if (bsa_status s = check_kv(a->k, a->dtype, "decode_weighted", "k", true)) return s;
  return check_kv(a->v, a->dtype, "decode_weighted", "v", true);
}

size_t weighted_workspace(const bsa_decode_weighted_args *a) {
  return weighted_check(a) == BSA_OK ? weighted_plan(a).bytes : 0;
}

bsa_status run_weighted(const bsa_decode_weighted_args *a, void *ws, size_t ws_bytes, cudaStream_t st) {
  if (bsa_status s = weighted_check(a)) return s;
  const WeightedPlan w = weighted_plan(a);
  if (!ws || ws_bytes < w.bytes) return fail(BSA_ERR_WORKSPACE, "decode_weighted: workspace too small");
  uint8_t *base = static_cast<uint8_t *>(ws);
  SplitParams p{};
  p.q = a->q.ptr, p.q_sb = a->q.sb, p.q_sh = a->q.sh, p.q_sl = a->q.sl;
  p.k = a->k.ptr, p.k_sb = a->k.sb, p.k_sh = a->k.sh, p.k_sl = a->k.sl;
  p.v = a->v.ptr, p.v_sb = a->v.sb, p.v_sh = a->v.sh, p.v_sl = a->v.sl;
  p.B = a->B, p.Hq = a->Hq, p.Hkv = a->Hkv, p.grp = a->Hq / a->Hkv, p.T = a->T;
  p.R = p.grp * a->T;
  p.nkeys = a->L;
  p.causal = 1;
  p.scale2 = a->scale * kLog2e;
  p.sel = a->sel, p.sel_sb = a->sel_sb, p.sel_sh = a->sel_sh;
  p.kk = a->sel ? a->kk : 0, p.bs = a->bs;
  p.gate = a->gate, p.gate_sb = a->gate_sb, p.gate_sh = a->gate_sh;
  p.nsplit = w.nsplit;
  p.rows = w.rows;
  p.po = reinterpret_cast<float *>(base + w.o_po);
  p.pml = reinterpret_cast<float2 *>(base + w.o_ml);
  p.logits = reinterpret_cast<float *>(base + w.o_lg);
  p.ncap = w.ncap;
  p.rpad = w.rpad;
  p.live = a->sel ? reinterpret_cast<int *>(base + w.o_lv) : nullptr;
  p.status = a->status;
  if (w.cl) {
    p.live = nullptr;
    p.o = a->o.ptr, p.o_sb = a->o.sb, p.o_sh = a->o.sh, p.o_sl = a->o.sl;
    p.weight = a->weight, p.w_sb = a->weight_sb, p.w_sh = a->weight_sh;
    return launch_split<true>(a->dtype, a->D, p, st);
  }
  if (bsa_status s = launch_split<false>(a->dtype, a->D, p, st)) return s;
  JoinParams j{};
  j.o = a->o.ptr, j.o_sb = a->o.sb, j.o_sh = a->o.sh, j.o_sl = a->o.sl;
  j.B = a->B, j.Hq = a->Hq, j.Hkv = a->Hkv, j.grp = p.grp, j.T = a->T, j.D = a->D;
  j.nsplit = w.nsplit, j.R = p.R, j.rows = w.rows, j.po = p.po, j.pml = p.pml;
  j.logits = p.logits, j.ncap = w.ncap, j.rpad = w.rpad, j.live = p.live, j.kk = p.kk, j.bs = a->bs, j.L = a->L;
  j.weight = a->weight, j.w_sb = a->weight_sb, j.w_sh = a->weight_sh;
  // slots per weight block: enough work to hide the lse of its rows, unless few blocks
  // come of it
  const long long heads = (long long)a->B * a->Hkv;
  j.kpb = heads * (w.ncap / 1024) >= 148 ? 1024 : heads * (w.ncap / 512) >= 148 ? 512 : 256;
  j.wtiles = (int)((w.ncap + j.kpb - 1) / j.kpb);
  return launch_join(a->dtype, j, st);
}

// ------------------------------------------------------------------ decode_prefix
bool prefix_sm100_applicable(const bsa_decode_prefix_args *a);
int prefix_sm100_splits(const bsa_decode_prefix_args *a, int &left);
bsa_status launch_prefix_sm100(const bsa_decode_prefix_args *a, const SplitParams &p, cudaStream_t st);

namespace {
// Bytes of the prefix read by all sequences together, up to which each reads it for
// itself: 5 us of L2 (18 groups that share 2311 keys, 43 MB, fp32: 19 us by splits, 33 by
// clusters).
constexpr long long kAgainBytes = 32 << 20;
struct PrefixPlan {
  int cl;      // CTAs of a cluster per (b, hk) (one launch), or 0
  bool tc;     // the prefix on the tensor-memory kernel
  int np, ns;  // splits of the prefix and of the own slots
  long long rows;
  size_t o_ml, bytes;
};
PrefixPlan prefix_plan(const bsa_decode_prefix_args *a) {
  PrefixPlan w;
  const int R = (a->Hq / a->Hkv) * a->T;
  // a small step: every sequence reads the prefix for itself (from L2 but once), in one launch
  const long long groups = (long long)a->B * a->Hkv, again = groups * a->P * a->D * 2 * (long long)elem_size(a->dtype);
  w.cl = again <= kAgainBytes ? cluster_size(a->dtype, a->D, groups, R, (long long)a->P + a->S) : 0;
  w.tc = !w.cl && prefix_sm100_applicable(a);
  int left = 148;  // SMs that the prefix leaves to the own slots
  w.np = w.tc ? prefix_sm100_splits(a, left) : a->P > 0 ? split_count(a->dtype, a->D, a->Hkv, a->B * R, a->P, true) : 0;
  w.ns = split_count(a->dtype, a->D, (long long)a->B * a->Hkv, R, a->S, false, left);
  w.rows = (long long)a->B * a->Hq * a->T;
  const size_t parts = w.cl ? 0 : (size_t)(w.np + w.ns) * w.rows;
  w.o_ml = align_up(parts * a->D * 4, 256);
  w.bytes = align_up(w.o_ml + parts * 8 + 256, 256);
  return w;
}
}  // namespace

static bsa_status prefix_check(const bsa_decode_prefix_args *a) {
  if (bsa_status s = check_rows("decode_prefix", a->dtype, a->B, a->Hq, a->Hkv, a->D, a->T, a->scale)) return s;
  if (a->P < 0 || a->S <= 0) return fail(BSA_ERR_SHAPE, "decode_prefix: needs P >= 0 and S >= 1");
  if (a->P >= (1 << 30) || a->S >= (1 << 30)) return fail(BSA_ERR_SHAPE, "decode_prefix: P or S too large");
  if (!a->q.ptr || !a->lens) return fail(BSA_ERR_ARG, "decode_prefix: NULL tensor");
  if (bsa_status s = check_out("decode_prefix", a->o, a->B, a->Hq, a->T, a->D)) return s;
  if (a->P > 0) {
    if (bsa_status s = check_kv(a->pk, a->dtype, "decode_prefix", "pk", false)) return s;
    if (bsa_status s = check_kv(a->pv, a->dtype, "decode_prefix", "pv", false)) return s;
  }
  if (bsa_status s = check_kv(a->k, a->dtype, "decode_prefix", "k", true)) return s;
  return check_kv(a->v, a->dtype, "decode_prefix", "v", true);
}

size_t prefix_workspace(const bsa_decode_prefix_args *a) {
  return prefix_check(a) == BSA_OK ? prefix_plan(a).bytes : 0;
}

bsa_status run_prefix(const bsa_decode_prefix_args *a, void *ws, size_t ws_bytes, cudaStream_t st) {
  if (bsa_status s = prefix_check(a)) return s;
  const PrefixPlan w = prefix_plan(a);
  if (!ws || ws_bytes < w.bytes) return fail(BSA_ERR_WORKSPACE, "decode_prefix: workspace too small");
  uint8_t *base = static_cast<uint8_t *>(ws);
  SplitParams p{};
  p.q = a->q.ptr, p.q_sb = a->q.sb, p.q_sh = a->q.sh, p.q_sl = a->q.sl;
  p.B = a->B, p.Hq = a->Hq, p.Hkv = a->Hkv, p.grp = a->Hq / a->Hkv, p.T = a->T;
  p.scale2 = a->scale * kLog2e;
  p.rows = w.rows;
  p.po = reinterpret_cast<float *>(base);
  p.pml = reinterpret_cast<float2 *>(base + w.o_ml);
  p.status = a->status;
  if (w.cl) {
    p.k2 = a->pk.ptr, p.k2_sh = a->pk.sh, p.k2_sl = a->pk.sl;
    p.v2 = a->pv.ptr, p.v2_sh = a->pv.sh, p.v2_sl = a->pv.sl;
    p.n2 = a->P;
    p.o = a->o.ptr, p.o_sb = a->o.sb, p.o_sh = a->o.sh, p.o_sl = a->o.sl;
  } else if (a->P > 0) {
    p.k = a->pk.ptr, p.k_sb = 0, p.k_sh = a->pk.sh, p.k_sl = a->pk.sl;
    p.v = a->pv.ptr, p.v_sb = 0, p.v_sh = a->pv.sh, p.v_sl = a->pv.sl;
    p.fold = 1;
    p.R = a->B * p.grp * a->T;
    p.nkeys = a->P;
    p.split0 = 0, p.nsplit = w.np;
    if (bsa_status s = w.tc ? launch_prefix_sm100(a, p, st) : launch_split<false>(a->dtype, a->D, p, st))
      return s;
  }
  p.k = a->k.ptr, p.k_sb = a->k.sb, p.k_sh = a->k.sh, p.k_sl = a->k.sl;
  p.v = a->v.ptr, p.v_sb = a->v.sb, p.v_sh = a->v.sh, p.v_sl = a->v.sl;
  p.fold = 0;
  p.R = p.grp * a->T;
  p.nkeys = a->S;
  p.lens = a->lens;
  p.causal = 1;
  if (w.cl) {
    p.nsplit = w.cl;
    return launch_split<true>(a->dtype, a->D, p, st);
  }
  p.split0 = w.np, p.nsplit = w.ns;
  p.after = a->P > 0;
  if (bsa_status s = launch_split<false>(a->dtype, a->D, p, st)) return s;
  JoinParams j{};
  j.o = a->o.ptr, j.o_sb = a->o.sb, j.o_sh = a->o.sh, j.o_sl = a->o.sl;
  j.B = a->B, j.Hq = a->Hq, j.Hkv = a->Hkv, j.grp = p.grp, j.T = a->T, j.D = a->D;
  j.nsplit = w.np + w.ns, j.R = p.R, j.rows = w.rows, j.po = p.po, j.pml = p.pml;
  return launch_join(a->dtype, j, st);
}

}  // namespace bsa
