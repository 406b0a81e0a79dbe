"""Block-sparse decode over a K/V cache (no counterpart in the reference, which
has no decode path; this is the next consumer of its selection).

    cache = DecodeCache(B, Hkv, max_len, D, bs=128, dtype=torch.bfloat16, device="cuda")
    cache.append(k_new, v_new)                      # (B, Hkv, T, D) each
    sel = cache.select_quest(q_new, topk=32)        # Quest bound, _finish layout
    o = decode_attention(q_new, cache, sel)         # (B, Hq, T, D)

The new tokens (positions L-T .. L-1) must lie in the cache's last block.
Selection is the reference's SelectMax rule (src/qwen_blocksparse.py:108-121)
applied to the current block: the query summary is the mean of the new tokens'
queries over the GQA group (for T = bs at a block boundary exactly the prefill
summary of that block), the key summaries are per-block min/max of the
cache (kept incrementally: an append re-pools only the blocks it touches),
then causal top-k + own block (+ sink) sorted ascending (:87-99).  Attention
masks are the TOKEN rules (key position <= query position, repeated ids
once), as in blocksparse_forward.

A cache within a budget.  With track=True the cache also keeps, per slot, the sum of
the attention weight it has received and its token position; a decode step through
decode_attention_weighted adds to the sums, and evict keeps the slots of most weight
beside the first `sink` and the last `recent` tokens:

    cache = DecodeCache(B, Hkv, 4096 + 64, D, bs=128, track=True)
    o = decode_attention_weighted(q_new, cache)     # every slot; or sel, as above
    cache.evict(4096, recent=256, sink=4)

A survivor may move to a freed slot (cache.pos tells its token position), so keys are
cached with their rotary embedding already applied, as the attention expects them.  Masks
go by slot: with several new tokens (T > 1) attend before evicting, as above.

A batch behind one prefix.  PrefixCache holds the prefix's K/V once and every
sequence's own continuation, of any length; prefix_attention reads the prefix once
for the whole batch:

    cache = PrefixCache(prefix_k, prefix_v, B, max_len)   # (Hkv, P, D) each
    cache.append(k_new, v_new)                      # (B, Hkv, T, D) each
    o = prefix_attention(q_new, cache)              # (B, Hq, T, D)
"""
import torch

import _bsa

__all__ = ["DecodeCache", "decode_attention", "decode_attention_weighted", "PrefixCache",
           "prefix_attention"]


class DecodeCache:
    """K/V cache (B, Hkv, max_len, D) with per-block min / max key summaries; with
    track=True also each slot's accumulated attention weight (fp32) and token position
    (int32), both (B, Hkv, max_len)."""

    def __init__(self, B, Hkv, max_len, D, *, bs, dtype=torch.bfloat16, device="cuda", track=False):
        self.bs = bs
        self.k = torch.zeros(B, Hkv, max_len, D, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        nblk = (max_len + bs - 1) // bs
        self.kmin = torch.zeros(B, Hkv, nblk, D, dtype=torch.float32, device=device)
        self.kmax = torch.zeros_like(self.kmin)
        self.L = 0          # slots in use
        self.seen = 0       # tokens appended so far
        self.ordered = 0    # newest tokens that lie in the last slots, in order
        self.weight = self.pos = None
        if track:
            self.weight = torch.zeros(B, Hkv, max_len, dtype=torch.float32, device=device)
            self.pos = torch.zeros(B, Hkv, max_len, dtype=torch.int32, device=device)

    def append(self, k_new, v_new):
        T = k_new.shape[2]
        L0, L1 = self.L, self.L + T
        if L1 > self.k.shape[2]:
            raise ValueError("cache full")
        self.k[:, :, L0:L1] = k_new
        self.v[:, :, L0:L1] = v_new
        self.L = L1
        b0, b1 = L0 // self.bs, (L1 - 1) // self.bs + 1
        # re-pool the touched blocks; rows past L count as zeros, as in the prefill pooling
        mn, mx = _bsa.pool(self.k[:, :, b0 * self.bs:min(b1 * self.bs, L1)], self.bs, mean=False,
                           vmin=True, vmax=True)
        self.kmin[:, :, b0:b1] = mn
        self.kmax[:, :, b0:b1] = mx
        if self.weight is not None:
            self.weight[:, :, L0:L1] = 0
            self.pos[:, :, L0:L1] = torch.arange(self.seen, self.seen + T, dtype=torch.int32,
                                                 device=self.pos.device)
        self.seen += T
        self.ordered += T

    def evict(self, budget, *, recent=0, sink=0):
        """Keeps `budget` slots per (b, hk): the first `sink` and last `recent` tokens,
        then the slots of most accumulated weight.  Returns how many slots went."""
        if self.weight is None:
            raise ValueError("evict needs a cache with track=True")
        gone = self.L - budget
        if gone <= 0:
            return 0
        _bsa.evict(self.k, self.v, self.weight, self.pos, budget=budget, L=self.L, seen=self.seen,
                   recent=recent, sink=sink, kmin=self.kmin, kmax=self.kmax, bs=self.bs)
        self.L = budget
        self.ordered = 0
        return gone

    def select_quest(self, q_new, *, topk, sink=True):
        """(B, Hkv, W) block ids for the current block: Quest bound of the new tokens'
        group-mean query against every block up to the current one."""
        Hq, Hkv = q_new.shape[1], self.k.shape[1]
        qb = (self.L - 1) // self.bs
        # group-and-row mean (rows past T count as zeros: a positive scale of the
        # summary, which leaves the Quest ranking unchanged)
        (qp,) = _bsa.pool(q_new, self.bs, grp=Hq // Hkv)
        # at least topk key blocks, so the row is topk + 1 (+ sink) wide from the start
        # (blocks after the current one are causally masked; missing picks -> own)
        nb = min(self.kmin.shape[2], max(qb + 1, topk))
        sel, _, _ = _bsa.select(qp.contiguous(), self.kmax[:, :, :nb].contiguous(),
                                self.kmin[:, :, :nb].contiguous(), kind=_bsa.SCORE_QUEST,
                                layout=_bsa.SEL_FINISH, topk=topk, sink=sink, q_blk0=qb)
        return sel[:, :, 0]


def decode_attention(q_new, cache, sel, gate=None, *, scale=None, mask_mode=_bsa.MASK_TOKEN):
    """o (B, Hq, T, D) of the T newest tokens attending to their selected cache blocks; rows
    before the last count on the new tokens lying in the last slots, in order."""
    return _bsa.decode(q_new, cache.k, cache.v, sel, gate, bs=cache.bs, L=cache.L,
                       mask_mode=mask_mode, scale=scale)


def decode_attention_weighted(q_new, cache, sel=None, gate=None, *, scale=None):
    """decode_attention under TOKEN masks that also adds every slot's attention weight to
    cache.weight (a cache with track=True).  sel=None attends to every slot."""
    if cache.weight is None:
        raise ValueError("decode_attention_weighted needs a cache with track=True")
    T = q_new.shape[2]
    if T > max(1, cache.ordered) and cache.ordered < cache.seen:
        # masks go by slot, and the eviction may have moved a row's own and later tokens; one
        # row sees every slot, in any order
        raise ValueError("%d rows after an eviction, but only %d tokens appended since: attend "
                         "before evicting" % (T, cache.ordered))
    return _bsa.decode_weighted(q_new, cache.k, cache.v, cache.weight, sel, gate, bs=cache.bs,
                                L=cache.L, scale=scale)


class PrefixCache:
    """The K/V of one prefix, (Hkv, P, D) each and not copied, and the continuations of B
    sequences behind it: k, v (B, Hkv, max_len, D), lens int32 (B,) on the device."""

    def __init__(self, prefix_k, prefix_v, B, max_len):
        if prefix_k.dim() != 3 or prefix_v.shape != prefix_k.shape:
            raise ValueError("prefix_k and prefix_v must be (Hkv, P, D)")
        Hkv, _, D = prefix_k.shape
        self.prefix_k, self.prefix_v = prefix_k, prefix_v
        self.k = torch.zeros(B, Hkv, max_len, D, dtype=prefix_k.dtype, device=prefix_k.device)
        self.v = torch.zeros_like(self.k)
        self.lens = torch.zeros(B, dtype=torch.int32, device=prefix_k.device)
        self.used = [0] * B     # the same lengths on the host

    def append(self, k_new, v_new, active=None):
        """Appends T tokens (B, Hkv, T, D) to every sequence, or to those whose entry of
        `active` (B truth values) is true."""
        B, Hkv, _, D = self.k.shape
        if k_new.dim() != 4 or v_new.shape != k_new.shape or \
                (k_new.shape[0], k_new.shape[1], k_new.shape[3]) != (B, Hkv, D):
            raise ValueError("k_new and v_new must be (%d, %d, T, %d)" % (B, Hkv, D))
        if active is not None and len(active) != B:
            raise ValueError("active must hold %d truth values" % B)
        T = k_new.shape[2]
        who = [b for b in range(len(self.used)) if active is None or active[b]]
        if any(self.used[b] + T > self.k.shape[2] for b in who):
            raise ValueError("cache full")
        dev = self.k.device
        b = torch.tensor(who, device=dev, dtype=torch.long)
        at = torch.tensor([self.used[i] for i in who], device=dev, dtype=torch.long).view(-1, 1) + \
            torch.arange(T, device=dev)
        self.k[b.view(-1, 1), :, at] = k_new[b].transpose(1, 2).to(self.k.dtype)
        self.v[b.view(-1, 1), :, at] = v_new[b].transpose(1, 2).to(self.v.dtype)
        self.lens[b] += T
        for i in who:
            self.used[i] += T

    def reset(self, b):
        """Empties the continuation of sequence b (a new question about the same prefix)."""
        self.used[b] = 0
        self.lens[b] = 0


def prefix_attention(q_new, cache, *, scale=None):
    """o (B, Hq, T, D) of every sequence's T newest tokens attending to the shared prefix
    and to their own continuation (a PrefixCache)."""
    return _bsa.decode_prefix(q_new, cache.prefix_k, cache.prefix_v, cache.k, cache.v, cache.lens,
                              scale=scale)
