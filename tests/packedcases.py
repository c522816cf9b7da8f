"""Inputs and 64-bit oracles of the packed-step operators: plain loops over rows
on the CPU oracle's int_gemm, di_softmax and matmul_i64, and Python integers."""

import numpy as np

from oracle import gemm as ogemm
from oracle import intmath as im
from oracle import ops as oops
from oracle.intmath import I64

PAGE = 128


def make(past, new, n_q, n_kv, seed, tpos=(29, 34), extra=3, tail=0, holes=(), width=None,
         extreme=False, flat=False):
    """Rows of past[b] slots and new[b] tokens over a paged cache whose page ids are
    a permutation (extra pages belong to nobody). tpos: the range of the score
    scales' exponents (12: constants 1, 32: about 2^16, 60: about 2^44); tail: token
    rows behind the last row's; holes: (row, page, id) of the table; extreme: head
    0's queries and a seventh of K are -128; flat: head 1's queries are 0."""
    rng = np.random.default_rng(seed)
    past, new = np.asarray(past, np.int32), np.asarray(new, np.int32)
    pages = -(-(past + new) // PAGE)
    width = max(int(pages.max()), 1) if width is None else width
    total = int(pages.sum()) + extra
    ids = rng.permutation(total).astype(np.int32)
    table = np.full((len(past), width), -1, np.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = ids[at:at + n]
        at += n
    for b, j, page in holes:
        table[b, j] = page
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    N = int(cu[-1]) + tail
    q8 = rng.integers(-128, 128, (N, n_q, 128), dtype=np.int8)
    kpool = rng.integers(-128, 128, (total, n_kv, PAGE, 128), dtype=np.int8)
    vpool = rng.integers(-128, 128, (total, n_kv, 128, PAGE), dtype=np.int8)
    if extreme:
        q8[:, 0] = -128
        kpool[:, 0, ::7] = -128
        vpool[:, 0, :5] = -128
    if flat:
        q8[:, 1] = 0
    sm = rng.integers(1 << 15, 1 << 16, (N, n_q, 1), dtype=np.int64)
    sk = rng.integers(tpos[0], tpos[1] + 1, (N, n_q, 1), dtype=np.int64)
    return dict(q8=q8, kpool=kpool, vpool=vpool, table=table, cu=cu, past=past, new=new, sm=sm,
                sk=sk, tpos=oops.di_exp_tpos(sm, sk)[..., 0], S=int(max((past + new).max(), 1)),
                max_new=int(new.max()))


def attend(c, S=None):
    """Contexts [N, n_q * 128] of make()'s rows (S: slots from there on unseen)."""
    N, n_q = c["q8"].shape[:2]
    n_pages, n_kv = c["kpool"].shape[:2]
    out = np.zeros((N, n_q, 128), dtype=I64)
    for b in range(len(c["past"])):
        T, past, i0 = int(c["new"][b]), int(c["past"][b]), int(c["cu"][b])
        if T == 0:
            continue
        n = past + T if S is None else min(past + T, S)
        w = -(-n // PAGE)
        ids = c["table"][b, :w]
        there = (ids >= 0) & (ids < n_pages)
        safe = np.where(there, ids, 0)
        k = c["kpool"][safe].transpose(1, 0, 2, 3).reshape(n_kv, w * PAGE, 128)[:, :n]
        v = c["vpool"][safe].transpose(1, 0, 3, 2).reshape(n_kv, w * PAGE, 128)[:, :n]
        see = np.repeat(there, PAGE)[:n] & (np.arange(n) <= past + np.arange(T)[:, None])
        for h in range(n_q):
            kv = h // (n_q // n_kv)
            s = ogemm.int_gemm(c["q8"][i0:i0 + T, h], np.ascontiguousarray(k[kv].T))
            p = oops.di_softmax(s, c["sm"][i0:i0 + T, h], c["sk"][i0:i0 + T, h], see)
            out[i0:i0 + T, h] = ogemm.matmul_i64(p, np.ascontiguousarray(v[kv]))
    return out.reshape(N, n_q * 128)


def plan(table, free, n_free, past, new, N):
    """A step's bookkeeping, row by row (the arguments are not changed): (table,
    free, n_free, cu, row, pos, slot, err)."""
    table, free = table.copy(), free.copy()
    B, width = table.shape
    err, count, need, cu = 0, [], [], [0]
    for b in range(B):
        have = 0
        while have < width and table[b, have] >= 0:
            have += 1
        end = int(past[b]) + int(new[b])
        ok = past[b] >= 0 and new[b] >= 0 and end <= min(width * PAGE, 131071)
        err |= 0 if ok else 4
        need.append(-(-end // PAGE) if ok else have)
        count.append(int(new[b]) if ok else 0)
        cu.append(cu[-1] + count[b])
        for j in range(need[b], have):
            free[n_free] = table[b, j]
            table[b, j] = -1
            n_free += 1
    missing = [(b, j) for b in range(B) for j in range(need[b]) if table[b, j] < 0]
    if len(missing) > n_free:
        err |= 8
    else:
        for b, j in missing:
            n_free -= 1
            table[b, j] = free[n_free]
    row, pos, slot = np.full(N, -1, np.int32), np.zeros(N, I64), np.full(N, -1, I64)
    err |= 4 if cu[-1] > N else 0
    for b in range(B):
        for t in range(count[b]):
            if cu[b] + t < N:
                s = int(past[b]) + t
                page = int(table[b, s // PAGE])
                row[cu[b] + t], pos[cu[b] + t] = b, s
                slot[cu[b] + t] = page * PAGE + s % PAGE if page >= 0 else -1
    return table, free, n_free, np.array(cu, np.int32), row, pos, slot, err


def lora(P, x8, a8, b8, bm, bk, adapter):
    """P plus each token row's adapter, in Python's own integers where it matters."""
    P = P.astype(np.int64).copy()
    for i, ad in enumerate(adapter):
        if not 0 <= ad < len(a8):
            continue
        u = a8[ad].astype(I64) @ x8[i].astype(I64)
        h = max(max(int(np.abs(u).max()), 1).bit_length() - 1 - 12, 0)
        w = im.rshift_round(u, h) if h else u
        assert np.abs(w).max() <= 1 << 13
        v = b8[ad].astype(I64) @ w
        s = int(bk[ad]) - h
        with np.errstate(over="ignore"):
            t = v * bm[ad]
            d = im.rshift_round(t, s) if s > 0 else im.shl(t, -s)
            P[i] += d
    return im.to_i32(P)
