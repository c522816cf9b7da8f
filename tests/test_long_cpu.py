"""The long-cache operators without a GPU: what they refuse (the native
kernels' checks on host tensors, before any launch), the entry points' error
codes, the fakes, and the KV cache's page bookkeeping."""

import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from idempotent_llm_amd import _lib, torch_ops
from idempotent_llm_amd.kvcache import PAGE, KVCache

KEY = torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA)
I8, I32, I64 = torch.int8, torch.int32, torch.int64


def _ops():
    return torch.ops.detllm_rocm


def _call(name, *args):
    """The operator's native kernel on host tensors (checks run first)."""
    return getattr(_ops(), name).default.redispatch(KEY, *args)


def _cache(B=2, n_q=4, n_kv=2, w=3, T=None):
    lead = (B, n_q) if T is None else (B, n_q, T)
    return dict(q8=torch.zeros(lead + (128,), dtype=I8), tpos=torch.ones(lead, dtype=I64),
                kpool=torch.zeros(B * w, n_kv, 128, 128, dtype=I8),
                vpool=torch.zeros(B * w, n_kv, 128, 128, dtype=I8),
                table=torch.zeros(B, w, dtype=I32), valid=torch.ones(B, w * 128, dtype=torch.bool))


# (operator, chunk length or None, trailing arguments that it takes)
ATTENTION = [("attn_window_prefill", 8, (100, 16, 4)), ("attn_window_decode", None, (200, 16, 4)),
             ("attn_prefill_acc", 8, (100, "acc")), ("attn_decode_acc", None, (200, "acc")),
             ("attn_decode_shared", None, (200, 128))]


def _tail(tail, B=2, n_kv=2, slots=384):
    return [torch.zeros(B, n_kv, slots, dtype=I64) if t == "acc" else t for t in tail]


BAD_CACHE = {
    "query rank": lambda c: c.update(q8=c["q8"][0]),
    "query type": lambda c: c.update(q8=c["q8"].to(I32)),
    "query channels": lambda c: c.update(q8=c["q8"][..., :64].contiguous()),
    "constants": lambda c: c.update(tpos=c["tpos"][:, :1].contiguous()),
    "constant type": lambda c: c.update(tpos=c["tpos"].to(I32)),
    "pool type": lambda c: c.update(kpool=c["kpool"].to(I32)),
    "pool channels": lambda c: c.update(kpool=c["kpool"][..., :64].contiguous()),
    "pools differ": lambda c: c.update(vpool=c["vpool"][:1].contiguous()),
    "no pages": lambda c: c.update(kpool=c["kpool"][:0], vpool=c["vpool"][:0]),
    "strided pool": lambda c: c.update(kpool=c["kpool"].transpose(2, 3)),
    "kv heads": lambda c: c.update(kpool=torch.zeros(6, 3, 128, 128, dtype=I8),
                                   vpool=torch.zeros(6, 3, 128, 128, dtype=I8)),
    "table rows": lambda c: c.update(table=c["table"][:1].contiguous()),
    "table type": lambda c: c.update(table=c["table"].long()),
    "strided table": lambda c: c.update(table=c["table"].t().contiguous().t()),
    "table short": lambda c: c.update(table=c["table"][:, :0].contiguous()),
    "mask rows": lambda c: c.update(valid=c["valid"][:1]),
    "mask type": lambda c: c.update(valid=c["valid"].long()),
    "mask short": lambda c: c.update(valid=c["valid"][:, :100]),
    "strided mask": lambda c: c.update(valid=c["valid"].t().contiguous().t()),
}


@pytest.mark.parametrize("op,T,tail", ATTENTION, ids=lambda v: v if isinstance(v, str) else "")
@pytest.mark.parametrize("bad", list(BAD_CACHE))
def test_attention_refuses(op, T, tail, bad):
    c = _cache(T=T)
    BAD_CACHE[bad](c)
    with pytest.raises(ValueError, match=op):
        _call(op, *c.values(), *_tail(tail))


BAD_TAILS = [
    ("attn_window_prefill", 8, (-1, 16, 4)), ("attn_window_prefill", 8, (100, 0, 4)),
    ("attn_window_prefill", 8, (100, 16, -1)), ("attn_window_prefill", 8, (377, 16, 4)),
    ("attn_window_decode", None, (385, 16, 4)), ("attn_window_decode", None, (-1, 16, 4)),
    ("attn_window_decode", None, (200, 0, 4)), ("attn_window_decode", None, (200, 16, -1)),
    ("attn_window_prefill", 8, (2**63 - 1, 16, 4)), ("attn_prefill_acc", 8, (2**63 - 1, "acc")),
    ("attn_prefill_acc", 8, (-1, "acc")), ("attn_prefill_acc", 8, (377, "acc")),
    ("attn_decode_acc", None, (385, "acc")),
    ("attn_decode_shared", None, (200, 100)), ("attn_decode_shared", None, (200, 256)),
    ("attn_decode_shared", None, (200, -128)), ("attn_decode_shared", None, (385, 128)),
]


@pytest.mark.parametrize("op,T,tail", BAD_TAILS)
def test_attention_refuses_sizes(op, T, tail):
    with pytest.raises(ValueError, match=op):
        _call(op, *_cache(T=T).values(), *_tail(tail))


@pytest.mark.parametrize("op,T,first", [("attn_prefill_acc", 8, 100), ("attn_decode_acc", None, 200)])
@pytest.mark.parametrize("acc", [torch.zeros(2, 2, 384), torch.zeros(2, 2, 384, dtype=I32),
                                 torch.zeros(2, 4, 384, dtype=I64), torch.zeros(1, 2, 384, dtype=I64),
                                 torch.zeros(2, 2, 100, dtype=I64), torch.zeros(4, 384, dtype=I64),
                                 torch.zeros(2, 384, 2, dtype=I64).transpose(1, 2)],
                         ids=["float", "int32", "heads", "rows", "short", "rank", "strided"])
def test_accumulators_refused(op, T, first, acc):
    with pytest.raises(ValueError, match=op):
        _call(op, *_cache(T=T).values(), first, acc)


def test_decode_refuses_other_groups():
    """Three or sixteen query heads per kv head: no decode kernel."""
    for n_q, n_kv in ((6, 2), (32, 2)):
        for op, T, tail in ATTENTION:
            if T is None:
                with pytest.raises(RuntimeError, match="code -38"):
                    _call(op, *_cache(n_q=n_q, n_kv=n_kv).values(), *_tail(tail))


def test_select_refuses():
    acc, valid = torch.zeros(2, 2, 300, dtype=I64), torch.ones(2, 300, dtype=torch.bool)
    good = (acc, valid, 300, 100, 20, 4)
    bad = [(acc.to(I32),) + good[1:], (acc[0],) + good[1:], (acc.transpose(1, 2),) + good[1:],
           (acc, valid.long()) + good[2:], (acc, valid[:1]) + good[2:],
           (acc, valid[:, :200]) + good[2:], good[:2] + (301,) + good[3:],
           good[:2] + (-1,) + good[3:], good[:3] + (0, 0, 0), good[:3] + (100, 97, 4),
           good[:3] + (100, -1, 4), good[:3] + (100, 4, -1),
           good[:3] + (100, 2**62, 2**62), (acc[:, :0],) + good[1:]]
    for args in bad:
        with pytest.raises(ValueError, match="kv_select|dimensions"):
            _call("kv_select", *args)


def test_compact_refuses():
    pool = lambda *s: torch.zeros(*(s or (6, 2, 128, 128)), dtype=I8)
    table, dst = torch.zeros(2, 3, dtype=I32), torch.zeros(2, 2, dtype=I32)
    keep = torch.zeros(2, 200, dtype=I32)
    same, wide = pool(), pool(9, 2, 128, 128)
    bad = [([], [], table, dst, keep), ([pool()], [pool(), pool()], table, dst, keep),
           ([pool()], [pool(5, 2, 128, 128)], table, dst, keep),
           ([pool(), pool(5, 2, 128, 128)], [pool(), pool()], table, dst, keep),
           ([pool().to(I32)], [pool()], table, dst, keep),
           ([pool(6, 2, 64, 128)], [pool(6, 2, 64, 128)], table, dst, keep),
           ([pool()], [pool().transpose(2, 3)], table, dst, keep),
           ([pool()], [pool()], table.long(), dst, keep),
           ([pool()], [pool()], table, dst[:1], keep), ([pool()], [pool()], table, dst, keep[:1]),
           ([pool()], [pool()], table, dst[:, :1].contiguous(), keep),
           ([pool()], [pool()], table, dst, keep.long()),
           ([pool()], [pool()], table[:, :0].contiguous(), dst, keep),
           ([same, pool()], [pool(), same], table, dst, keep), ([same], [same], table, dst, keep),
           ([same, same], [pool(), pool()], table, dst, keep),
           ([wide[:6]], [wide[3:]], table, dst, keep),
           ([pool()], [pool()], torch.zeros(2, 1025, dtype=I32), dst, keep),
           ([pool()], [pool()], table, torch.zeros(2, 1025, dtype=I32),
            torch.zeros(2, 131073, dtype=I32))]
    for args in bad:
        with pytest.raises(ValueError, match="kv_compact|dimensions"):
            _call("kv_compact", *args)


def test_entry_error_codes():
    """Bad sizes and missing scratch return their code before any launch;
    empty problems return at once."""
    e = _lib.native().entries()
    t = torch.zeros(16, dtype=I8)
    cache = (t, t, t, t, t, 3, t, 384)
    win = lambda S=200, nq=4, window=16, sinks=4, work=t, n=1 << 40, B=2: (
        *cache, B, S, nq, 2, None, window, sinks, work, n, t, None)
    assert e["detllm_attn_window_decode"](0, *win(B=0)) is None
    for kw, code in ((dict(window=0), -22), (dict(sinks=-1), -22), (dict(S=385), -22),
                     (dict(nq=6), -38), (dict(nq=5), -22), (dict(S=131072), -34)):
        with pytest.raises(RuntimeError, match=f"code {code}"):
            e["detllm_attn_window_decode"](0, *win(**kw))
    big = (*cache[:5], 200, t, 25600)                     # scores past LDS: scratch is needed
    for work, n in ((None, 1 << 40), (t, 16)):
        with pytest.raises(RuntimeError, match="code -34"):
            e["detllm_attn_window_decode"](0, *big, 2, 25000, 4, 2, None, 9000, 4, work, n, t, None)
        with pytest.raises(RuntimeError, match="code -34"):
            e["detllm_attn_decode_acc"](0, *big, 2, 25000, 4, 2, None, t, 25000, work, n, t, None)
        with pytest.raises(RuntimeError, match="code -34"):
            e["detllm_attn_decode_shared"](0, *big, 2, 25000, 4, 2, None, 24960, work, n, t, None)
    with pytest.raises(RuntimeError, match="code -22"):    # accumulators shorter than the slots
        e["detllm_attn_decode_acc"](0, *cache, 2, 200, 4, 2, None, t, 199, None, 0, t, None)
    with pytest.raises(RuntimeError, match="code -22"):
        e["detllm_attn_prefill_acc"](0, *cache, 2, 8, 100, 4, 2, t, 107, t)
    with pytest.raises(RuntimeError, match="code -22"):    # not a whole number of pages
        e["detllm_attn_decode_shared"](0, *cache, 2, 200, 4, 2, None, 64, t, 1 << 40, t, None)
    with pytest.raises(RuntimeError, match="code -22"):
        e["detllm_kv_select"](0, t, 300, t, 300, 2, 300, 2, 100, 97, 4, t, t, t, 1 << 40)
    with pytest.raises(RuntimeError, match="code -34"):
        e["detllm_kv_select"](0, t, 20000, t, 20000, 2, 20000, 2, 100, 9, 4, t, t, None, 0)
    assert e["detllm_kv_compact"](0, None, None, 0, 6, t, 3, t, 2, t, 2, 100, 2) is None
    pools = (ctypes.c_void_p * 1)(0)
    with pytest.raises(RuntimeError, match="code -22"):
        e["detllm_kv_compact"](0, ctypes.addressof(pools), ctypes.addressof(pools), 1, 6, t, 3, t,
                               2, t, 2, 100, 2)
    for width, budget in ((1025, 100), (3, 131073)):
        with pytest.raises(RuntimeError, match="code -34"):
            e["detllm_kv_compact"](0, ctypes.addressof(pools), ctypes.addressof(pools), 1, 6, t,
                                   width, t, 2, t, 2, budget, 2)


def test_scratch_sizes_cover_every_shape():
    """The planners answer for every size, and few slots need none."""
    for n_q, n_kv in ((8, 8), (16, 8), (32, 8), (64, 8), (8, 1)):
        for B in (1, 3, 16, 64, 300):
            for S in (0, 1, 127, 768, 5000, 131071):
                n = _lib.attn_acc_work(B, S, n_q, n_kv)
                assert 0 <= n <= B * n_q * (S + 4096) * 8
                for shared in (0, S // 2 // PAGE * PAGE, S // PAGE * PAGE):
                    n, joint = _lib.attn_shared_work(B, S, n_q, n_kv, shared)
                    assert n >= 0 and not (joint and (shared == 0 or B == 1))
    assert _lib.attn_acc_work(1, 300, 16, 8) == 0


def test_operators_mutate_what_they_declare():
    want = {"attn_prefill_acc": {"acc"}, "attn_decode_acc": {"acc"},
            "kv_compact": {"kpools", "vpools"}}
    for name in torch_ops.LONG_OPS:
        op = getattr(_ops(), name).default
        got = {a.name for a in op._schema.arguments if a.alias_info and a.alias_info.is_write}
        assert got == want.get(name, set()), name
        assert torch.Tag.pt2_compliant_tag in op.tags
        assert torch._C._dispatch_has_kernel_for_dispatch_key(f"detllm_rocm::{name}", "CUDA")


def test_fakes_have_the_outputs_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        dev = lambda c: [x.to("cuda") for x in c.values()]
        acc = torch.empty(2, 2, 384, dtype=I64, device="cuda")
        chunk, one = dev(_cache(T=8)), dev(_cache())
        for out in (_ops().attn_window_prefill(*chunk, 100, 16, 4),
                    _ops().attn_prefill_acc(*chunk, 100, acc)):
            assert out.shape == (2, 8, 512) and out.dtype == I64
        for out in (_ops().attn_window_decode(*one, 200, 16, 4),
                    _ops().attn_decode_acc(*one, 200, acc),
                    _ops().attn_decode_shared(*one, 200, 128)):
            assert out.shape == (2, 512) and out.dtype == I64
        keep, kept = _ops().kv_select(acc, one[5], 300, 100, 10, 4)
        assert keep.shape == (2, 100) and keep.dtype == I32
        assert kept.shape == (2, 2, 100) and kept.dtype == I64
        dst = torch.empty(2, 1, dtype=I32, device="cuda")
        assert _ops().kv_compact([one[2]], [one[3]], one[4], dst, keep) is None


# ------------------------------------------------------------------ KVCache

def _model():
    return SimpleNamespace(n_layers=2, n_kv=1, hd=128, device=torch.device("cpu"))


def _one_row(length):
    c = KVCache()
    c.reserve(_model(), 1, length)
    for li, (kp, vp) in enumerate(zip(c.k_pools, c.v_pools)):
        for p in range(kp.shape[0]):
            kp[p], vp[p] = 10 * li + p, 50 + 10 * li + p
    c.valid_buf[:, :length] = True
    c.length = length
    return c


@pytest.mark.parametrize("length", [1, 128, 200, 384, 500])
def test_fork_shares_full_pages(length):
    c = _one_row(length)
    k = [x.clone() for x in c.k8]
    v = [x.clone() for x in c.v8]
    full = length // PAGE
    c.fork(3)
    assert c.shared == full * PAGE and c.table.shape[0] == 3 and c.valid.shape == (3, length)
    assert torch.equal(c.table, torch.from_numpy(c._table_host))
    for li in range(2):
        assert torch.equal(c.k8[li], k[li].expand(3, -1, -1, -1))
        assert torch.equal(c.v8[li], v[li].expand(3, -1, -1, -1))
    assert (c._table_host[:, :full] == c._table_host[0, :full]).all()
    c.check_rows(3)
    c.reserve(_model(), 3, length + 300)      # the rows' own pages from here on
    own = c._table_host[:, full:-(-(length + 300) // PAGE)]
    assert (own >= 0).all() and len(np.unique(own)) == own.size
    assert not np.isin(own, c._table_host[0, :full]).any()


def test_fork_refuses_other_caches():
    with pytest.raises(ValueError, match="one row"):
        KVCache().fork(2)
    c = KVCache()
    c.reserve(_model(), 2, 100)
    with pytest.raises(ValueError, match="one row"):
        c.fork(2)
    c = _one_row(100)
    with pytest.raises(ValueError, match="one row"):
        c.fork(0)
    c.static_cap = 256
    for f in (lambda: c.fork(2), lambda: c.evict(10), c.track_weights):
        with pytest.raises(ValueError, match="graphed"):
            f()


def test_evict_refuses_without_weights_and_budget():
    c = _one_row(300)
    with pytest.raises(ValueError, match="track_weights"):
        c.evict(100)
    c.track_weights()
    for args in ((0,), (10, 8, 3), (10, -1, 0), (10, 0, -1)):
        with pytest.raises(ValueError, match="evict"):
            c.evict(*args)
    assert c.evict(300) is c and c.length == 300      # nothing to do


def test_tracked_weights_grow_with_the_cache():
    c = KVCache().track_weights()
    assert c.acc is None
    c.reserve(_model(), 2, 100)
    assert c.acc.shape == (2, 1, c.cap) and not c.acc.any()
    c.acc[:, :, :100] = 7
    c.reserve(_model(), 2, 500)
    assert c.acc.shape == (2, 1, c.cap) and (c.acc[:, :, :100] == 7).all()
    assert not c.acc[:, :, 100:].any()


def test_pages_handed_back_are_used_again():
    c = _one_row(300)
    c._free = [7, 9]
    n = c.n_pages
    assert c._take_pages(3).tolist() == [9, 7, n] and c.n_pages == n + 1 and not c._free
