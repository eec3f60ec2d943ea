"""Batches of drafted tokens for the tests: page tables with the new tokens cached, trees, tolerances.

The tolerance of an output element against 64 bits, from what the kernels round (u16 = 2^-11, u = 2^-24, half a
step of fp16 and fp32 relative to the value):
    u16 |o|                    the result's rounding to fp16 (2^-25 below fp16's normal range)
    u16 sum p |v|              the weights' rounding to fp16 in the PV product
    2 u (sum p e |v| + |o| sum p e)   the scores' errors e (oracle.tree_attention's slack), which move a weight p by p e u and
                               through the sum every other; twice for the maximum's part of the exponent
    (keys / 16 + 64) u sum p |v|, and the same of |o|   sums over the keys: a lane holds a sixteenth of them where
                               waves split the keys; where they do not it holds a quarter, held to the same bound (the
                               roundings of a sum go either way)
and of lse: 2 u sum p e + (keys / 16 + 64) u + 4 u |lse|. Both twice, for products of these and second orders.
"""
from dataclasses import dataclass

import numpy as np

from pdattn import inputs

U16, U = 2.0 ** -11, 2.0 ** -24


@dataclass
class Draft:
    bt: inputs.Batch
    q: np.ndarray            # [n_tokens, Hq, 128] fp16
    q_indptr: np.ndarray
    mask: np.ndarray | None  # [n_tokens, words] int32
    depth: np.ndarray | None
    parent: list             # per sequence

    @property
    def n_tokens(self):
        return self.q.shape[0]

    @property
    def max_tokens(self):
        return max(1, int(np.diff(self.q_indptr).max(initial=1)))


def random_tree(n, rng, bushy=0.5):
    """Parents (-1: the context) of n nodes, each before its children."""
    parent = np.full(n, -1)
    for i in range(1, n):
        parent[i] = i - 1 if rng.random() > bushy else rng.integers(-1, i)
    return parent


def tree_rows(parent, words):
    """Mask rows (ancestors and the node itself, 32 bits a word) and depths."""
    n = len(parent)
    seen = np.zeros((n, 32 * words), bool)
    depth = np.zeros(n, np.int64)
    for i, p in enumerate(parent):
        if p >= 0:
            seen[i] = seen[p]
            depth[i] = depth[p] + 1
        if i < seen.shape[1]:
            seen[i, i] = True
    return pack(seen), depth


def pack(seen):
    """[n, 32 w] truth values -> [n, w] int32."""
    bits = seen.reshape(len(seen), -1, 32).astype(np.uint64) << np.arange(32, dtype=np.uint64)
    return bits.sum(2).astype(np.uint32).view(np.int32)


def make_draft(ctx, new, Hq, Hkv, seed, tree=True, extra_rows=0, words=None, dist="normal"):
    """Sequences with ctx[b] cached tokens before new[b] drafted ones (cached as well); extra_rows: rows of q behind
    the last sequence."""
    rng = np.random.default_rng(seed)
    bt = inputs.make_batch([c + n for c, n in zip(ctx, new)], Hq, Hkv, seed, dist=dist)
    q_indptr = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    total = int(q_indptr[-1]) + extra_rows
    q = rng.standard_normal((total, Hq, 128)).astype(np.float16)
    parent = [random_tree(n, rng) for n in new]
    mask = depth = None
    if tree:
        words = max(1, -(-max(new) // 32)) if words is None else words
        mask, depth = np.zeros((total, words), np.int32), np.zeros(total, np.int32)
        for b, p in enumerate(parent):
            if len(p):
                rows = slice(int(q_indptr[b]), int(q_indptr[b + 1]))
                mask[rows], depth[rows] = tree_rows(p, words)
    return Draft(bt, q, q_indptr, mask, depth, parent)


def check_attention(out, lse, ref, tag="", rows=None):
    """out and lse (numpy) against oracle.tree_attention's result, with the tolerances above."""
    ro, rl, slack = ref
    rows = slice(None) if rows is None else rows
    out, lse, ro, rl = np.asarray(out, np.float64)[rows], np.asarray(lse, np.float64)[rows], ro[rows], rl[rows]
    weight, score, score_v, keys = (slack[k][rows] for k in ("weight", "score", "score_v", "keys"))
    none = np.isneginf(rl)
    assert np.array_equal(np.isneginf(lse), none), f"{tag}: rows without a key differ"
    assert np.all(out[none] == 0), f"{tag}: a row without a key is not 0"
    assert np.array_equal(np.isnan(rl), np.isnan(lse)) and np.array_equal(np.isnan(ro), np.isnan(out)), f"{tag}: NaN"
    fin = np.isfinite(rl)
    sums = (keys / 16 + 64) * U
    tol = 2 * (U16 * (np.abs(ro) + weight) + 2 ** -25 + 2 * U * (score_v + np.abs(ro) * score[..., None]) +
               sums[..., None] * (weight + np.abs(ro)))
    off = np.abs(out[fin] - ro[fin]) / tol[fin]
    assert off.size == 0 or off.max() <= 1, f"{tag}: out {off.max():.2f} of its tolerance"
    tol_l = 2 * (2 * U * score + sums + 4 * U * np.abs(rl, where=fin, out=np.zeros_like(rl)))
    off_l = np.abs(lse[fin] - rl[fin]) / tol_l[fin]
    assert off_l.size == 0 or off_l.max() <= 1, f"{tag}: lse {off_l.max():.2f} of its tolerance"
    return (float(off.max()) if off.size else 0.0, float(off_l.max()) if off_l.size else 0.0)


class DeviceDraft:
    """Device copies of a Draft."""

    def __init__(self, dr):
        import torch
        from _gpu import DeviceBatch, device
        dev = device()
        self.dr, self.db = dr, DeviceBatch(dr.bt)
        put = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
        self.q, self.q_indptr, self.mask, self.depth = put(dr.q), put(dr.q_indptr), put(dr.mask), put(dr.depth)
        self.out = torch.full(dr.q.shape, float("nan"), dtype=torch.float16, device=dev)
        self.lse = torch.full(dr.q.shape[:2], float("nan"), dtype=torch.float32, device=dev)

    def params(self, single=False, max_tokens=None, **score):
        import pdattn
        import torch
        db, bt = self.db, self.dr.bt
        if score.get("slopes") is not None:
            self.slopes = torch.tensor(score["slopes"], dtype=torch.float32, device=self.q.device)
            score = dict(score, slopes=self.slopes)
        return pdattn.make_tree_params(self.q, db.k, db.v, db.indptr, db.indices, db.last, bt.B, bt.Hq, bt.Hkv,
                                       q_indptr=None if single else self.q_indptr,
                                       max_tokens=self.dr.max_tokens if max_tokens is None else max_tokens,
                                       mask=self.mask, depth=self.depth, **score)

    def run(self, stream=None, **kw):
        import pdattn
        import torch
        p = self.params(**kw)
        ws = pdattn.Workspace()
        try:
            pdattn.tree_attention(p, self.out, self.lse, ws, stream)
            torch.cuda.synchronize()
        finally:
            pdattn.workspace_release(ws)
        return self.out.float().cpu().numpy(), self.lse.cpu().numpy()


def oracle_attention(dr, **kw):
    import oracle
    bt = dr.bt
    return oracle.tree_attention(dr.q, bt.k, bt.v, bt.indptr, bt.indices, bt.last, bt.Hq, bt.Hkv, dr.q_indptr,
                                 dr.mask, dr.depth, **kw)
