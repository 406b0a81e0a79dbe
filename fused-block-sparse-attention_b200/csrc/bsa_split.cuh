// Split attention of a few query rows over a long K/V: parameters shared by the
// partial kernels (mma.sync, fp32 and tcgen05) and by the kernel that joins them.
//
// Every partial kernel leaves, for each query row and each split of the keys,
//   m = max_j x_j,   l = sum_j 2^(x_j - m),   O = sum_j 2^(x_j - m) v_j
// in fp32, with x_j = (scale * q.k_j + gate) * log2(e).  The join is
//   M = max_s m_s,   o = (sum_s 2^(m_s - M) O_s) / (sum_s 2^(m_s - M) l_s),
// so splits of one cache and splits of two different K/V (a shared prefix and a
// sequence's own slots) are joined alike.
#pragma once
#include <type_traits>

#include "bsa_common.cuh"

namespace bsa {

struct SplitParams {
  const void *q;
  int64_t q_sb, q_sh, q_sl;
  const void *k, *v;
  int64_t k_sb, k_sh, k_sl, v_sb, v_sh, v_sl;
  int B, Hq, Hkv, grp, T;
  int fold;             // 1: the rows of all sequences read one K/V (a shared prefix)
  int R;                // query rows per K/V head: grp*T, or B*grp*T when folded
  int nkeys;            // rows of k, v in use (the capacity when lens is given)
  const int32_t *lens;  // optional (B): each sequence's own count, clamped to [0, nkeys]
  int causal;           // row t sees key j <= len - T + t (else every key)
  float scale2;         // scale * log2(e)
  const int32_t *sel;   // optional block ids per (b, hk)
  int64_t sel_sb, sel_sh;
  int kk, bs;
  const float *gate;
  int64_t gate_sb, gate_sh;
  int split0, nsplit;   // this kernel's splits are split0 .. split0 + nsplit - 1
  long long rows;       // B*Hq*T
  float *po;            // [split][rows][D]
  float2 *pml;          // [split][rows] (m, l); m = -inf: nothing visible, O not written
  float *logits;        // optional [b*Hkv + hk][ncap][rpad]: x_j of each row
  long long ncap;
  int rpad;             // rows padded to a multiple of 8
  int *live;            // with sel and logits: [b*Hkv + hk][1 + kk] count and live block ids
  // One launch (a cluster per (b, hk) joins its own splits): keys before the own ones,
  // shared by the batch and seen by every row, the output, and the running sums.
  const void *k2, *v2;
  int64_t k2_sh, k2_sl, v2_sh, v2_sl;
  int n2;
  void *o;
  int64_t o_sb, o_sh, o_sl;
  float *weight;        // optional, with logits
  int64_t w_sb, w_sh;
  int after;            // launched beside the kernel before it, whose end it waits for at its own
  int stages, ring;     // ring stages per warp and bytes of the ring (split_mma, split_f32)
  int32_t *status;
};

// p, q >= 0 as two 16-bit terms each, p = hi + lo up to 2^-16 p (bf16) or 2^-22 p + 2^-25
// (f16), packed.  hi is cut off below p, never rounded to it, so that both terms of a
// positive p are positive and an infinity times them stays what it is (a term that is zero
// or negative makes infinity - infinity of it); p = 0 gives 0 and 0.  f16 has no terms below
// 2^-24: there hi is left 2^-24 further below p, and p < 2^-23 may lose a term.
template <typename T>
__device__ __forceinline__ void split2(float p, float q, uint32_t &hi, uint32_t &lo) {
  constexpr float kBelow = 1.f - 0x1p-24f;  // the next float below
  if constexpr (std::is_same<T, __half>::value) {
    asm("cvt.rz.relu.f16x2.f32 %0, %1, %2;"
        : "=r"(hi)
        : "f"(fmaf(q, kBelow, -0x1p-24f)), "f"(fmaf(p, kBelow, -0x1p-24f)));
    const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    lo = Mma<T>::pack(p - h.x, q - h.y);
  } else {
    const uint32_t a = __float_as_uint(p * kBelow), b = __float_as_uint(q * kBelow);
    hi = __byte_perm(a, b, 0x7632);
    lo = Mma<T>::pack(p - __uint_as_float(a & 0xffff0000u), q - __uint_as_float(b & 0xffff0000u));
  }
}

// Global row (b*Hq + h)*T + t of local row r of K/V head hk.
__device__ __forceinline__ long long split_row(const SplitParams &p, int b, int hk, int r, int &rb,
                                               int &rh, int &rt) {
  const int per = p.grp * p.T;
  if (p.fold) {
    rb = r / per;
    r -= rb * per;
  } else {
    rb = b;
  }
  rh = hk * p.grp + r / p.T;
  rt = r % p.T;
  return ((long long)rb * p.Hq + rh) * p.T + rt;
}

}  // namespace bsa
