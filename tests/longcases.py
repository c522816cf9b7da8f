"""Inputs and 64-bit oracles of the long-cache operators: plain loops over rows
and heads on the CPU oracle's int_gemm, di_softmax and matmul_i64."""

import numpy as np

from oracle import gemm as ogemm
from oracle import ops as oops
from oracle.intmath import I64


def make(B, n_q, n_kv, S, seed, T=None, p_valid=1.0, gaps=(), dead_rows=(), tpos=(29, 34),
         flat_heads=(), extreme=()):
    """Random queries (one per row, or T per row), K [B, n_kv, S, 128], V^T
    [B, n_kv, 128, S], validity [B, S] and score scales. gaps: (row, lo, hi)
    slots that are not valid; dead_rows: nothing valid; tpos: the range of the
    scales' exponents (small: constants near 1, large: wide ones); flat_heads:
    q = 0; extreme: heads whose q and a seventh of K are -128."""
    rng = np.random.default_rng(seed)
    lead = (B, n_q) if T is None else (B, n_q, T)
    q8 = rng.integers(-128, 128, lead + (128,), dtype=np.int8)
    kc = rng.integers(-128, 128, (B, n_kv, S, 128), dtype=np.int8)
    vc = rng.integers(-128, 128, (B, n_kv, 128, S), dtype=np.int8)
    for h in flat_heads:
        q8[:, h] = 0
    for h in extreme:
        q8[:, h] = -128
        kc[:, h // (n_q // n_kv), ::7] = -128
    sm = rng.integers(1 << 15, 1 << 16, lead + (1,), dtype=np.int64)
    sk = rng.integers(tpos[0], tpos[1] + 1, lead + (1,), dtype=np.int64)
    valid = rng.random((B, S)) < p_valid
    for row, lo, hi in gaps:
        valid[row, lo:hi] = False
    for row in dead_rows:
        valid[row] = False
    return dict(q8=q8, kc=kc, vc=vc, sm=sm, sk=sk, valid=valid, n_kv=n_kv,
                tpos=oops.di_exp_tpos(sm, sk)[..., 0])


def visible(valid, t, window=None, sinks=0):
    """The slots [0, t] that the query at slot t sees, one by one."""
    live = np.flatnonzero(valid[:t + 1])
    if window is not None:
        live = np.union1d(live[:sinks], live[max(0, len(live) - window):])
    see = np.zeros(t + 1, dtype=bool)
    see[live] = True
    return see


def attend(c, T=None, past=0, window=None, sinks=0, S=None):
    """(context, weights): decode over S slots (T None), or T queries behind
    ``past`` slots. weights [B, n_kv, slots]: p summed over the kv head's query
    heads and the queries at valid slots."""
    B, n_q = c["q8"].shape[:2]
    n_kv, cap = c["n_kv"], c["kc"].shape[2]
    slots = [S - 1] if T is None else list(range(past, past + T))
    out = np.zeros((B, len(slots), n_q * 128), dtype=I64)
    acc = np.zeros((B, n_kv, cap), dtype=I64)
    for b in range(B):
        for i, t in enumerate(slots):
            if t < 0:
                continue
            see = visible(c["valid"][b], t, window, sinks)
            for h in range(n_q):
                kv = h // (n_q // n_kv)
                at = (b, h) if T is None else (b, h, i)
                s = ogemm.int_gemm(c["q8"][at][None],
                                   np.ascontiguousarray(c["kc"][b, kv, :t + 1].T))
                p = oops.di_softmax(s, c["sm"][at][None], c["sk"][at][None], see[None])
                out[b, i, h * 128:(h + 1) * 128] = ogemm.matmul_i64(
                    p, np.ascontiguousarray(c["vc"][b, kv, :, :t + 1].T))[0]
                if c["valid"][b, t]:
                    acc[b, kv, :t + 1] += p[0]
    return (out[:, 0] if T is None else out), acc


def select(acc, valid, budget, recent, sinks):
    """keep [B, budget] and the kept accumulators, by sorting."""
    B, n_kv, _ = acc.shape
    keep = np.full((B, budget), -1, dtype=np.int32)
    kept = np.zeros((B, n_kv, budget), dtype=I64)
    for b in range(B):
        live = [int(s) for s in np.flatnonzero(valid[b])]
        if len(live) > budget:
            with np.errstate(over="ignore"):
                w = acc[b].sum(axis=0)
            hi = len(live) - recent
            mid = sorted(live[sinks:hi], key=lambda s: (-int(w[s]), s))
            live = sorted(live[:sinks] + mid[:budget - sinks - recent] + live[hi:])
        keep[b, :len(live)] = live
        kept[b, :, :len(live)] = acc[b][:, live]
    return keep, kept
