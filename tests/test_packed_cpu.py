"""The packed-step operators without a GPU: what they refuse (the native kernels'
checks on host tensors, before any launch), the entry points' error codes, the
planners, the fakes, the cache's and the adapters' host side."""

import ctypes
import json
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import packedcases as pc
from idempotent_llm_amd import _lib, lora, packed, torch_ops
from idempotent_llm_amd.kvcache import PAGE

KEY = torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA)
I8, I32, I64 = torch.int8, torch.int32, torch.int64


def _ops():
    return torch.ops.detllm_rocm


def _call(name, *args):
    """The operator's native kernel on host tensors (checks run first)."""
    return getattr(_ops(), name).default.redispatch(KEY, *args)


def _refused(name, good, bad, error=ValueError):
    for what, change in bad.items():
        c = dict(good)
        c.update(change(c))
        with pytest.raises(error, match=name):
            _call(name, *c.values())
            pytest.fail(what)


def _odd(*shape):
    """int8 zeros that start one byte past a 16-byte address."""
    return torch.zeros(int(np.prod(shape)) + 1, dtype=I8)[1:].view(shape)


def _attention(N=3, B=2, n_q=4, n_kv=2, w=3):
    return dict(q8=torch.zeros(N, n_q, 128, dtype=I8), tpos=torch.ones(N, n_q, dtype=I64),
                kpool=torch.zeros(6, n_kv, 128, 128, dtype=I8),
                vpool=torch.zeros(6, n_kv, 128, 128, dtype=I8),
                table=torch.zeros(B, w, dtype=I32), cu=torch.zeros(B + 1, dtype=I32),
                past=torch.zeros(B, dtype=I32), S=300, max_new=2, err=torch.zeros(1, dtype=I32))


def test_attention_refuses():
    _refused("attn_packed", _attention(), {
        "query rank": lambda c: dict(q8=c["q8"][0]),
        "query type": lambda c: dict(q8=c["q8"].to(I32)),
        "channels": lambda c: dict(q8=c["q8"][..., :64].contiguous()),
        "three heads a kv head": lambda c: dict(q8=torch.zeros(3, 6, 128, dtype=I8)),
        "heads": lambda c: dict(q8=torch.zeros(3, 5, 128, dtype=I8)),
        "sixteen a kv head": lambda c: dict(q8=torch.zeros(3, 32, 128, dtype=I8)),
        "constants": lambda c: dict(tpos=c["tpos"][:, :2]),
        "constant type": lambda c: dict(tpos=c["tpos"].to(I32)),
        "pool type": lambda c: dict(kpool=c["kpool"].to(I32)),
        "pool rank": lambda c: dict(kpool=c["kpool"][0]),
        "pools differ": lambda c: dict(vpool=c["vpool"][:5]),
        "pool channels": lambda c: dict(kpool=c["kpool"][..., :64].contiguous()),
        "no pages": lambda c: dict(kpool=c["kpool"][:0], vpool=c["vpool"][:0]),
        "strided pool": lambda c: dict(kpool=c["kpool"].transpose(2, 3)),
        "unaligned pool": lambda c: dict(vpool=_odd(6, 2, 128, 128)),
        "table rows": lambda c: dict(table=c["table"][:1]),
        "table type": lambda c: dict(table=c["table"].long()),
        "table rank": lambda c: dict(table=c["table"][0]),
        "strided table": lambda c: dict(table=c["table"].t().contiguous().t()),
        "no rows": lambda c: dict(table=c["table"][:0], cu=c["cu"][:1], past=c["past"][:0]),
        "offsets": lambda c: dict(cu=c["cu"][:2]),
        "offset type": lambda c: dict(cu=c["cu"].long()),
        "lengths": lambda c: dict(past=c["past"][:1]),
        "length type": lambda c: dict(past=c["past"].long()),
        "strided lengths": lambda c: dict(past=torch.zeros(4, dtype=I32)[::2]),
        "slots": lambda c: dict(S=385), "no slots": lambda c: dict(S=0),
        "too many slots": lambda c: dict(S=131072, table=torch.zeros(2, 1024, dtype=I32)),
        "negative bound": lambda c: dict(max_new=-1),
        "error word": lambda c: dict(err=torch.zeros(1, dtype=I64)),
        "two error words": lambda c: dict(err=torch.zeros(2, dtype=I32)),
    })


def _plan_args(B=3, w=4, cap=12):
    return dict(table=torch.zeros(B, w, dtype=I32), free=torch.zeros(cap, dtype=I32),
                n_free=torch.zeros(1, dtype=I32), past=torch.zeros(B, dtype=I32),
                new=torch.zeros(B, dtype=I32), N=5, err=torch.zeros(1, dtype=I32))


def test_plan_refuses():
    _refused("packed_plan", _plan_args(), {
        "table rank": lambda c: dict(table=c["table"][0]),
        "table type": lambda c: dict(table=c["table"].long()),
        "strided table": lambda c: dict(table=c["table"].t().contiguous().t()),
        "no rows": lambda c: dict(table=c["table"][:0], past=c["past"][:0], new=c["new"][:0]),
        "no pages a row": lambda c: dict(table=c["table"][:, :0].contiguous()),
        "rows": lambda c: _plan_args(B=2049), "width": lambda c: _plan_args(w=1025),
        "free type": lambda c: dict(free=c["free"].long()),
        "free rank": lambda c: dict(free=c["free"][None]),
        "free length": lambda c: dict(n_free=torch.zeros(2, dtype=I32)),
        "free length type": lambda c: dict(n_free=torch.zeros(1, dtype=I64)),
        "past": lambda c: dict(past=c["past"][:2]),
        "past type": lambda c: dict(past=c["past"].long()),
        "new": lambda c: dict(new=torch.zeros(4, dtype=I32)),
        "strided new": lambda c: dict(new=torch.zeros(6, dtype=I32)[::2]),
        "negative": lambda c: dict(N=-1), "too many": lambda c: dict(N=2**31),
        "error word": lambda c: dict(err=torch.zeros(0, dtype=I32)),
    })


def _epilogue(N=3, n_q=4, n_kv=2, pages=2):
    v = lambda n: torch.ones(n, dtype=I64)
    k = n_kv * 128
    return dict(P=torch.zeros(2, N, (n_q + 2 * n_kv) * 128, dtype=I32), n_q=n_q, n_kv=n_kv,
                xm=v(N), xk=v(N), positions=v(N), slots=v(N), q_m=v(n_q * 128), q_k=1, k_m=v(k),
                k_k=1, v_m=v(k), v_k=1, q_norm_m=v(128), q_norm_k=1, k_norm_m=v(128), k_norm_k=1,
                qs_m=v(k), qs_k=1, kq_m=v(k), kq_k=v(k), ks_m=v(n_kv), ks_k=v(n_kv), vq_m=v(n_kv),
                vq_k=v(n_kv), cos=torch.zeros(9, 128, dtype=torch.int16),
                sin=torch.zeros(9, 128, dtype=torch.int16),
                kpool=torch.zeros(pages, n_kv, 128, 128, dtype=I8),
                vpool=torch.zeros(pages, n_kv, 128, 128, dtype=I8), err=torch.zeros(1, dtype=I32))


def test_epilogue_refuses():
    bad = {
        "rank": lambda c: dict(P=c["P"][0]), "type": lambda c: dict(P=c["P"].long()),
        "heads": lambda c: dict(n_q=3), "no heads": lambda c: dict(n_kv=0),
        "columns": lambda c: dict(n_q=6), "negative heads": lambda c: dict(n_q=-4, n_kv=-2),
        "no partials": lambda c: dict(P=c["P"][:0]),
        "tables": lambda c: dict(sin=c["sin"][:8]),
        "table rank": lambda c: dict(cos=c["cos"][0]),
        "table type": lambda c: dict(cos=c["cos"].int()),
        "no table rows": lambda c: dict(cos=c["cos"][:0], sin=c["sin"][:0]),
        "pool": lambda c: dict(kpool=c["kpool"][:, :1]),
        "pools differ": lambda c: dict(vpool=c["vpool"][:1]),
        "unaligned pool": lambda c: dict(kpool=_odd(2, 2, 128, 128)),
        "error word": lambda c: dict(err=torch.zeros(1, dtype=I8)),
    }
    for k, v in _epilogue().items():
        if torch.is_tensor(v) and v.dim() == 1 and k != "err":
            bad[f"{k} short"] = lambda c, k=k: {k: c[k][:-1]}
            bad[f"{k} type"] = lambda c, k=k: {k: c[k].to(I32)}
            bad[f"{k} strided"] = lambda c, k=k: {k: torch.ones(2 * c[k].numel(), dtype=I64)[::2]}
    _refused("qkv_epilogue_packed", _epilogue(), bad)


def _lora(N=3, K=64, C=10, r=16, n=2):
    return dict(x8=torch.zeros(N, K, dtype=I8), w=torch.zeros(C, K, dtype=I8),
                a8=torch.zeros(n, r, K, dtype=I8), b8=torch.zeros(n, C, r, dtype=I8),
                bm=torch.zeros(n, C, dtype=I64), bk=torch.zeros(n, dtype=I64),
                adapter=torch.zeros(N, dtype=I32))


def test_lora_refuses():
    _refused("lora_gemm", _lora(), {
        "rank of x8": lambda c: dict(x8=c["x8"][None]), "w": lambda c: dict(w=c["w"][:, :48]),
        "type": lambda c: dict(x8=c["x8"].to(I32)), "w type": lambda c: dict(w=c["w"].to(I32)),
        "K": lambda c: _lora(K=40), "deep": lambda c: _lora(K=65552), "K 0": lambda c: _lora(K=0),
        "rank": lambda c: _lora(r=24), "large rank": lambda c: _lora(r=144),
        "rank 0": lambda c: _lora(r=0), "no adapters": lambda c: _lora(n=0),
        "no columns": lambda c: _lora(C=0),
        "a8": lambda c: dict(a8=c["a8"][:1]), "a8 rank": lambda c: dict(a8=c["a8"][0]),
        "a8 K": lambda c: dict(a8=torch.zeros(2, 16, 32, dtype=I8)),
        "b8": lambda c: dict(b8=c["b8"][:, :9]), "b8 type": lambda c: dict(b8=c["b8"].to(I32)),
        "b8 order": lambda c: dict(b8=torch.zeros(2, 16, 10, dtype=I8)),
        "bm": lambda c: dict(bm=c["bm"][:, :9]), "bm type": lambda c: dict(bm=c["bm"].to(I32)),
        "strided bm": lambda c: dict(bm=torch.zeros(10, 2, dtype=I64).t()),
        "bk": lambda c: dict(bk=c["bk"][:1]), "adapter": lambda c: dict(adapter=c["adapter"][:2]),
        "adapter type": lambda c: dict(adapter=c["adapter"].long()),
    })


def test_entry_error_codes():
    """Bad sizes, missing scratch and unaligned operands return their code before
    any launch; empty problems return at once."""
    e = _lib.native().entries()
    t = torch.zeros(64, dtype=I64)
    odd = t.data_ptr() + 8

    def code(name, want, *args):
        with pytest.raises(RuntimeError, match=rf"{name} failed \(code {want}\)"):
            e[name](0, *args)

    plan = lambda table=t, width=4, cap=9, B=2, N=3, work=t, n=1 << 20: (
        table, width, t, cap, t, t, t, B, N, t, t, t, t, work, n, None)
    for kw, want in ((dict(B=0), -22), (dict(B=2049), -34), (dict(width=0), -22), (dict(N=-1), -22),
                     (dict(width=1025), -34), (dict(cap=-1), -22), (dict(table=None), -22),
                     (dict(N=5000, work=None), -22), (dict(N=5000, work=odd), -22),
                     (dict(N=5000, n=16), -34)):
        code("detllm_packed_plan", want, *plan(**kw))

    attn = lambda q8=t, kp=t, vp=t, n_pages=2, width=30, N=3, B=2, S=100, new=2, nq=4, nkv=2, \
        work=t, n=1 << 40: (q8, t, kp, vp, n_pages, t, width, t, t, N, B, S, new, nq, nkv, work, n,
                            t, None)
    name = "detllm_attn_packed"
    assert e[name](0, *attn(N=0)) is None
    for kw, want in ((dict(N=-1), -22), (dict(B=0), -22), (dict(S=0), -22), (dict(new=-1), -22),
                     (dict(nq=5), -22), (dict(nkv=0), -22), (dict(nq=6), -38), (dict(nq=32), -38),
                     (dict(S=131072), -34), (dict(B=65537), -34), (dict(N=1 << 23), -34),
                     (dict(S=3841), -22), (dict(width=0), -22), (dict(n_pages=0), -22),
                     (dict(q8=None), -22), (dict(q8=odd), -22), (dict(kp=odd), -22),
                     (dict(vp=odd), -22), (dict(S=3000, work=None), -22),
                     (dict(S=3000, work=odd), -22), (dict(S=3000, n=64), -34),
                     (dict(S=3000, new=900, N=900, n=64), -34)):
        code(name, want, *attn(**kw))

    lr = lambda P=t, x=t, a=t, b=t, N=3, K=64, C=10, r=16, n=2: (P, x, a, b, t, t, t, N, K, C, r, n)
    name = "detllm_lora_add"
    assert e[name](0, *lr(N=0)) is None
    for kw, want in ((dict(N=-1), -22), (dict(K=0), -22), (dict(K=24), -22), (dict(C=0), -22),
                     (dict(r=0), -22), (dict(r=24), -22), (dict(n=0), -22), (dict(K=65552), -34),
                     (dict(r=144), -34), (dict(C=(1 << 24) + 1), -34), (dict(N=(1 << 20) + 1), -34),
                     (dict(P=None), -22), (dict(x=odd), -22), (dict(a=odd), -22),
                     (dict(b=odd), -22)):
        code(name, want, *lr(**kw))

    epi = lambda P=t, ns=1, N=3, nq=4, nkv=2, slots=t, kp=t, pages=2, maxp=9: (
        P, ns, 0, N, nq, nkv, t, t, t, slots, t, 1, t, 1, t, 1, t, 1, t, 1, t, 1, t, t, t, t, t, t,
        t, t, maxp, t, t, kp, t, pages, None, None)
    name = "detllm_qkv_epilogue_packed"
    assert e[name](0, *epi(N=0)) is None
    for kw, want in ((dict(nq=3), -22), (dict(nkv=0), -22), (dict(ns=0), -22), (dict(maxp=0), -22),
                     (dict(P=None), -22), (dict(slots=None), -22), (dict(kp=None), -22),
                     (dict(pages=0), -22), (dict(N=2**31 - 1), -34)):
        code(name, want, *epi(**kw))


def test_scratch_sizes():
    """The planners answer for every size and refuse the ones that the entries
    refuse; short rows need no scratch, and what is needed grows with the bounds
    at most as their product does."""
    work = ctypes.c_int64(0)
    lib = _lib.load()
    for B, N, want in ((1, 0, 0), (2048, 2048, 0), (2048, 2049, 2049 * 16), (3, 1 << 30, 64)):
        assert lib.detllm_packed_plan_work(B, N, ctypes.byref(work)) == 0 and work.value == want
    for B, N, rc in ((0, 1, -22), (2049, 1, -34), (1, -1, -22)):
        assert lib.detllm_packed_plan_work(B, N, ctypes.byref(work)) == rc
    assert lib.detllm_packed_plan_work(1, 1, None) == -22
    for n_q, n_kv in ((1, 1), (8, 8), (16, 8), (32, 8), (64, 8), (8, 1)):
        for B in (1, 3, 64, 300, 2048):
            for new in (0, 1, 2, 16, 17, 500, 2**31 - 1):
                for N in (1, 5, 64, 4096):
                    for S in (1, 512, 513, 2048, 2049, 8000, 131071):
                        n = _lib.packed_work(N, B, S, new, n_q, n_kv)
                        top = (S + 1024) * 4 * (B * n_kv * 16 + N * n_q) + (N + B + 64) * n_kv * 64 * 12 * 300
                        assert 0 <= n <= top and (S > 512 or n == 0)
    for args in ((1, 1, 0, 1, 2, 1), (1, 0, 5, 1, 2, 1), (-1, 1, 5, 1, 2, 1), (1, 1, 131072, 1, 2, 1),
                 (1, 65537, 5, 1, 2, 1), (1 << 24, 1, 5, 1, 2, 1), (1, 1, 5, -1, 2, 1),
                 (1, 1, 5, 1, 3, 1), (1, 1, 5, 1, 3, 2)):
        with pytest.raises(RuntimeError, match="detllm_attn_packed_work"):
            _lib.packed_work(*args)


def test_operators_mutate_what_they_declare():
    want = {"packed_plan": {"table", "free", "n_free", "err"},
            "qkv_epilogue_packed": {"kpool", "vpool", "err"}, "attn_packed": {"err"}}
    for name in torch_ops.PACKED_OPS:
        op = getattr(_ops(), name).default
        got = {a.name for a in op._schema.arguments if a.alias_info and a.alias_info.is_write}
        assert got == want.get(name, set()), name
        assert torch.Tag.pt2_compliant_tag in op.tags
        assert torch._C._dispatch_has_kernel_for_dispatch_key(f"detllm_rocm::{name}", "CUDA")


def test_fakes_have_the_outputs_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        dev = lambda c: [x.to("cuda") if torch.is_tensor(x) else x for x in c.values()]
        cu, row, pos, slot = _ops().packed_plan(*dev(_plan_args()))
        assert cu.shape == (4,) and row.shape == pos.shape == slot.shape == (5,)
        assert (cu.dtype, row.dtype, pos.dtype, slot.dtype) == (I32, I32, I64, I64)
        q8, tpos = _ops().qkv_epilogue_packed(*dev(_epilogue()))
        assert q8.shape == (3, 4, 128) and q8.dtype == I8
        assert tpos.shape == (3, 4) and tpos.dtype == I64
        out = _ops().attn_packed(*dev(_attention()))
        assert out.shape == (3, 512) and out.dtype == I64
        out = _ops().lora_gemm(*dev(_lora()))
        assert out.shape == (3, 10) and out.dtype == I32


# ------------------------------------------------------------------ the cache

def _model():
    return SimpleNamespace(n_layers=2, n_kv=1, hd=128, device=torch.device("cpu"))


def test_cache_sizes():
    c = packed.PackedCache(_model(), 3, 300)
    assert c.pages == 9 and c.table.shape == (3, 3) and (c.table == -1).all()
    assert sorted(c.free.tolist()) == list(range(9)) and int(c.n_free) == 9
    assert len(c.k_pools) == 2 and c.k_pools[0].shape == (9, 1, PAGE, 128)
    for args in ((0, 300), (2049, 10), (1, 0), (1, 131072), (1, 10, 0)):
        with pytest.raises(ValueError, match="PackedCache"):
            packed.PackedCache(_model(), *args)


def test_cache_checks_a_step():
    c = packed.PackedCache(_model(), 3, 300, pages=5)
    for new in ((1, 1), (1, 1, -1), (301, 0, 0)):
        with pytest.raises(ValueError, match="packed step"):
            c.check(new)
    c.check((300, 129, 0))
    with pytest.raises(packed.OutOfPages):
        c.check((300, 257, 1))
    c.lens = [300, 129, 0]
    assert c.pages_left() == 0
    with pytest.raises(packed.OutOfPages):
        c.check((0, 0, 1))
    with pytest.raises(ValueError, match="packed step"):
        c.check((1, 0, 0))
    for args in ((3,), (-1,), (0, 301), (0, -1)):
        with pytest.raises(ValueError, match="release"):
            c.release(*args)
    c.release(0, 128)
    assert c.lens == [128, 129, 0] and c.past.tolist() == [128, 0, 0] and c.pages_left() == 2
    c.check((0, 0, 200))
    c.release(1)
    assert c.lens == [128, 0, 0]


class _Echo:
    """A model whose reply to a request is its tokens' running sum (and
    whose step notes what it was given)."""
    n_layers, n_kv, hd, max_pos, device = 1, 1, 128, 500, torch.device("cpu")
    cfg = {"eos_token_id": 40}

    def __init__(self):
        self.steps, self.sums = [], {}

    def forward_packed(self, ids, new, cache, adapters=None, adapter_of=None):
        cache.check(new)
        self.steps.append(list(new))
        at, out = 0, []
        for b, n in enumerate(new):
            if cache.lens[b] == 0:
                self.sums[b] = 0 if adapter_of is None else 100 * (adapter_of[b] + 1)
            self.sums[b] += int(ids[at:at + n].sum())
            at += n
            cache.lens[b] += n
            if n:
                out.append(self.sums[b])
        assert at == len(ids)
        return torch.tensor(out)

    def greedy_pick(self, logits):
        return logits

    def raise_if_device_error(self):
        pass


def _echo(prompt, n, first=0, eos=None):
    total, out = first + sum(prompt), []
    for _ in range(n):
        out.append(total)
        if total == eos:
            break
        total += out[-1]
    return out


@pytest.mark.parametrize("rows,step_tokens,pages", [(1, 1, None), (2, 3, None), (3, 64, 3),
                                                    (32, 512, None), (5, 7, 1)])
def test_generate_packed_schedules_every_request(rows, step_tokens, pages):
    m = _Echo()
    prompts = [[1, 2, 3], [5], [2] * 20, [7, 7], [9] * 6, [4]]
    most = [3, 0, 2, 5, 1, 4]
    which = [None, 0, 1, None, -1, 0]
    got = packed.generate_packed(m, [torch.tensor(p) for p in prompts], most, rows=rows,
                                 step_tokens=step_tokens, pages=pages, adapter_of=which)
    for p, n, w, g in zip(prompts, most, which, got):
        assert g.dtype == I64
        assert g.tolist() == _echo(p, n, 100 * ((-1 if w is None else w) + 1))
    assert all(0 < sum(s) <= max(step_tokens, 1) for s in m.steps)
    assert all(len(s) <= rows for s in m.steps)


def test_generate_packed_stops_and_refuses():
    m = _Echo()
    p = [torch.tensor([10]), torch.tensor([3])]
    got = packed.generate_packed(m, p, 6, stop_at_eos=True)
    assert got[0].tolist() == [10, 20, 40] == _echo([10], 6, eos=40)
    assert got[1].tolist() == _echo([3], 6)
    assert [g.tolist() for g in packed.generate_packed(m, p, 0)] == [[], []]
    assert packed.generate_packed(m, [], 3) == []
    for args in ((p, [1]), (p, -1), ([torch.tensor([], dtype=I64)], 1)):
        with pytest.raises(ValueError, match="generate_packed"):
            packed.generate_packed(m, *args)
    for kw in (dict(rows=0), dict(step_tokens=0)):
        with pytest.raises(ValueError, match="generate_packed"):
            packed.generate_packed(m, p, 3, **kw)
    with pytest.raises(packed.OutOfPages):
        packed.generate_packed(m, [torch.ones(200, dtype=I64)], 3, pages=1)
    with pytest.raises(IndexError):
        packed.generate_packed(m, [torch.ones(498, dtype=I64)], 4)
    m.steps.clear()
    packed.generate_packed(m, [torch.ones(498, dtype=I64)], 3)
    assert sum(map(sum, m.steps)) == 500


# ---------------------------------------------------------------- adapters

@pytest.mark.parametrize("K,C,r,scale,seed", [(64, 40, 4, 1.0, 1), (256, 300, 16, 0.5, 2),
                                              (512, 33, 30, 2.0, 3)])
def test_quantized_adapter_is_near_the_float_one(K, C, r, scale, seed):
    """The integers that are added, against scale B A x in the product's units. a8
    is off by half a step of its row's maximum / 127 in each of K places, w by half
    a unit of its shift, b8 by half a step in each of r places, bm by half of one and
    the result's shift by less than one: the bound adds these up."""
    g = torch.Generator().manual_seed(seed)
    A = torch.randn(r, K, generator=g, dtype=torch.float64) / K ** 0.5
    B = torch.randn(C, r, generator=g, dtype=torch.float64)
    col_m = torch.randint(1 << 15, 1 << 16, (C,), generator=g)
    col_k = 26
    in_scale = 2.0 ** torch.randn(K, generator=g, dtype=torch.float64)
    a8, b8, bm, bk = lora.quantize(A, B, col_m, col_k, in_scale, scale)
    assert a8.dtype == b8.dtype == I8 and bm.dtype == I64
    assert (1 << 15) <= int(bm.max()) <= 1 << 16
    x = torch.randint(-127, 128, (1, K), generator=g, dtype=I8)
    pad = -r % 16
    z = lambda t, dim: torch.cat([t, torch.zeros([pad if i == dim else n for i, n in
                                                  enumerate(t.shape)], dtype=I8)], dim)
    got = pc.lora(np.zeros((1, C), np.int32), x.numpy(), z(a8, 0).numpy()[None],
                  z(b8, 1).numpy()[None], bm.numpy()[None], np.array([bk]), [0])[0]
    unit = col_m.double() / 2.0 ** col_k                  # what one of the product's units is
    As = A * in_scale
    u = As @ x[0].double()                                # exact
    want = scale * (B @ u) / unit
    sa = As.abs().amax(1) / 127
    Bs = scale * B * sa                                   # B in steps of A's rows
    sb = Bs.abs().amax(1) / 127
    uq = (u / sa).abs()                                   # in a8's units
    du = x[0].double().abs().sum() / 2                    # a8 off by half a step each
    h = max(int((uq.max() + du).log2()) - 12, 0) + 1
    dw = du + 2.0 ** (h - 1)                              # and u shifted by up to h, rounded
    top = uq.max() + dw
    err = (Bs.abs().sum(1) * dw + r * (sb / 2) * top) / unit
    # bm rounded to 1 of its ratio 2^bk, the last shift to 1
    err = err + 0.5 * 2.0 ** -bk * r * 127 * top + 1
    assert ((torch.from_numpy(got).double() - want).abs() <= err).all()


def test_quantize_zeros_and_refusals():
    a8, b8, bm, bk = lora.quantize(torch.zeros(3, 32), torch.randn(5, 3), torch.ones(5), 3)
    assert not a8.any() and not bm.any() and bk == 0
    a8, b8, bm, bk = lora.quantize(torch.randn(3, 32), torch.zeros(5, 3), torch.ones(5), 3)
    assert not b8.any() and not bm.any() and bk == 0
    for A, B, n in ((torch.zeros(3, 32), torch.zeros(5, 4), 5), (torch.zeros(3, 32), torch.zeros(5, 3), 4),
                    (torch.zeros(32), torch.zeros(5, 3), 5)):
        with pytest.raises(ValueError, match="quantize"):
            lora.quantize(A, B, torch.ones(n), 3)


def _bank_model():
    v = lambda n, s: torch.randint(1 << 15, 1 << 16, (n,), generator=torch.Generator().manual_seed(s))
    cols = dict(q=256, k=128, v=128, o=64, gate=96, up=96, down=64)
    layer = lambda s: SimpleNamespace(**{f"{m}_m": v(c, s) for m, c in cols.items()},
                                      **{f"{m}_k": 24 + i for i, m in enumerate(cols)})
    return SimpleNamespace(n_layers=2, n_q=2, n_kv=1, hd=128, hidden=64, inter=96,
                           device=torch.device("cpu"), layers=[layer(0), layer(1)])


def test_bank_stacks_the_modules_of_a_product():
    """Each module's change of the stacked site is its own quantised one, to a
    rounding of its column scale where the site's exponent is smaller."""
    m = _bank_model()
    bank = lora.AdapterBank(m, 3, 5)
    g = torch.Generator().manual_seed(0)
    w = {(1, n): (torch.randn(5 - (n == "v"), 64, generator=g) * s,
                  torch.randn(bank.cols[n], 5 - (n == "v"), generator=g))
         for n, s in (("q", 1.0), ("v", 30.0), ("gate", 0.01))}
    bank.set(2, w, scale=0.5)
    x = np.random.default_rng(1).integers(-127, 128, (4, 64), dtype=np.int8)
    for s, ms in lora.SITES.items():
        for li in range(2):
            a8, b8, bm, bk = (t.numpy() for t in bank.sites[li][s])
            assert not a8[:2].any() and not b8[:2].any() and not bm[:2].any()
            if s in ("o", "d") or li == 0:
                assert not bm.any()
                continue
            at = 0
            for j, n in enumerate(ms):
                c = slice(at, at + bank.cols[n])
                at += bank.cols[n]
                if (li, n) not in w:
                    assert not b8[2, c].any()
                    continue
                cm, ck = getattr(m.layers[li], f"{n}_m"), getattr(m.layers[li], f"{n}_k")
                qa, qb, qm, qk = lora.quantize(*w[li, n], cm, ck, None, 0.5)
                r = qa.shape[0]
                assert np.array_equal(a8[2, 16 * j:16 * j + r], qa.numpy())
                assert np.array_equal(b8[2, c, 16 * j:16 * j + r], qb.numpy())
                assert (np.abs(b8[2, c]).sum(1) == np.abs(qb.numpy().astype(int)).sum(1)).all()
                assert qk >= bk[2]
                assert (np.abs(bm[2, c] - qm.numpy() / 2.0 ** (qk - bk[2])) <= 0.5).all()
            # the site's part of a product, from the stacked and the single forms
            P = np.zeros((4, b8.shape[1]), np.int32)
            pc.lora(P, x, a8, b8, bm, bk, [2, -1, 2, 0])
    bank.set(2, {})
    assert all(not t.any() for site in bank.sites for v in site.values() for t in v)


def test_in_scales_are_what_the_weights_have_folded_in(tmp_path):
    """Every int8 weight of a quantised model, times its column's scale, is the float
    weight times in_scales within half a step (and the scales' 16 bits)."""
    from floatmodel import small_float_model
    from safetensors.torch import load_file

    from idempotent_llm_amd import prepare as P
    fm = small_float_model(seed=0)
    ids = torch.randint(0, 1000, (2, 16), generator=torch.Generator().manual_seed(0))
    P.prepare(str(tmp_path), fm, ids, device="cpu", model_id="test")
    t = load_file(tmp_path / "model.safetensors")
    cfg = json.loads((tmp_path / "config.json").read_text())
    layers = []
    for i, Lc in enumerate(cfg["layers"]):
        layers.append(SimpleNamespace(**{f"{n}_m": t[f"layers.{i}.{n}_m"] for n in ("as", "os", "ms", "ds")},
                                      **{f"{n}_k": Lc[f"{n}_k"] for n in ("as", "os", "ms", "ds")}))
    got = lora.in_scales(SimpleNamespace(layers=layers),
                         [x.input_layernorm.weight for x in fm.model.layers],
                         [x.post_attention_layernorm.weight for x in fm.model.layers])
    for i, x in enumerate(fm.model.layers):
        mods = dict(q=x.self_attn.q_proj, k=x.self_attn.k_proj, v=x.self_attn.v_proj,
                    o=x.self_attn.o_proj, gate=x.mlp.gate_proj, up=x.mlp.up_proj,
                    down=x.mlp.down_proj)
        for site, ms in lora.SITES.items():
            for m in ms:
                step = (t[f"layers.{i}.{m}.m"].double() / 2.0 ** cfg["layers"][i][m]["k"])[:, None]
                w8 = t[f"layers.{i}.{m}.w8t"].double().t()
                want = mods[m].weight.detach().double() * got[i, site]
                # half a step, and 127 steps of a 16-bit mantissa's half unit (2^-16)
                assert ((w8 * step - want).abs() <= step * (0.5 + 127 * 2.0 ** -15)).all()


def test_bank_refusals():
    m = _bank_model()
    for n, r in ((0, 4), (2, 0), (2, 33)):
        with pytest.raises(ValueError, match="AdapterBank"):
            lora.AdapterBank(m, n, r)
    bank = lora.AdapterBank(m, 2, 32)
    ok = (torch.zeros(4, 64), torch.zeros(256, 4))
    for i, w in ((2, {}), (-1, {}), (0, {(2, "q"): ok}), (0, {(0, "x"): ok}),
                 (0, {(0, "q"): (torch.zeros(33, 64), torch.zeros(256, 33))}),
                 (0, {(0, "q"): (torch.zeros(4, 65), torch.zeros(256, 4))}),
                 (0, {(0, "q"): (torch.zeros(4, 64), torch.zeros(255, 4))})):
        with pytest.raises(ValueError):
            bank.set(i, w)


# ---------------------------------------------------------------- the model's step

def _step_model():
    """An IntQwen3 of sizes alone: what forward_packed checks before it launches."""
    from idempotent_llm_amd.model import IntQwen3
    m = object.__new__(IntQwen3)
    vars(m).update(vars(_bank_model()), max_pos=4000, vocab=50, _err=torch.zeros(1, dtype=I32))
    return m


class _Launched(Exception):
    pass


@pytest.fixture
def step_bounds(monkeypatch):
    """The bounds that forward_packed sizes its launches by; it goes no further."""
    from idempotent_llm_amd import model
    seen = []

    def work(N, B, S, max_new, n_q, n_kv):
        seen.append(dict(N=N, B=B, S=S, max_new=max_new))
        raise _Launched

    monkeypatch.setattr(model, "packed_work", work)
    return seen


def test_step_refuses_adapters_without_a_bank(step_bounds):
    """Adapters that a call names are in a bank, or the call is refused: it does not
    answer with the plain model."""
    m = _step_model()
    cache, ids = packed.PackedCache(m, 2, 100), torch.zeros(3, dtype=I64)
    for of in ((0, -1), (-1, 5), (-2, -1), (-1,), (-1, -1, -1)):
        with pytest.raises(ValueError, match="packed step"):
            m.forward_packed(ids, (1, 2), cache, None, of)
    bank = lora.AdapterBank(m, 2, 4)
    for of in (None, (0,), (0, 2), (-2, 0)):
        with pytest.raises(ValueError, match="packed step"):
            m.forward_packed(ids, (1, 2), cache, bank, of)
    assert not step_bounds
    for bk, of in ((None, None), (None, (-1, -1)), (bank, (-1, -1)), (bank, (1, -1))):
        with pytest.raises(_Launched):
            m.forward_packed(ids, (1, 2), cache, bk, of)


def test_generate_packed_checks_every_request_first(monkeypatch):
    """A request that the model refuses is refused before the first step, however late
    it would be admitted: the others' replies are not lost with it."""
    m = _step_model()
    steps = []

    def forward_packed(ids, new, cache, adapters=None, adapter_of=None):
        steps.append(list(new))
        raise _Launched

    monkeypatch.setattr(m, "forward_packed", forward_packed, raising=False)
    good, bank = [torch.tensor([1, 2])] * 3, lora.AdapterBank(m, 2, 4)
    for bad in (torch.tensor([50]), torch.tensor([3, -51, 3])):
        with pytest.raises(IndexError, match="token id"):
            packed.generate_packed(m, good + [bad], 2, rows=1)
    for bk, of in ((None, (-1, -1, 0)), (None, (0, None, None)), (bank, (0, 1, 2)),
                   (bank, (0, 1, -2)), (bank, (0, 1)), (None, (-1,) * 4), (bank, ())):
        with pytest.raises(ValueError, match="packed"):
            packed.generate_packed(m, good, 2, rows=1, adapters=bk, adapter_of=of)
    bank.cols = dict(bank.cols, q=384)
    with pytest.raises(ValueError, match="adapters of a model"):
        packed.generate_packed(m, good, 2, rows=1, adapters=bank, adapter_of=(0, None, 1))
    assert not steps
    with pytest.raises(_Launched):
        packed.generate_packed(m, good, 2, rows=1, adapters=lora.AdapterBank(m, 2, 4),
                               adapter_of=(0, None, 1))
    assert steps == [[2]]


def test_bank_keeps_an_adapter_that_cannot_be_replaced():
    """A set that is refused, in whichever layer, leaves every adapter as it was."""
    bank = lora.AdapterBank(_bank_model(), 2, 4)
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g)
    bank.set(1, {(0, "q"): (r(4, 64), r(256, 4)), (1, "down"): (r(4, 96), r(64, 4))})
    before = [{s: [t.clone() for t in v] for s, v in site.items()} for site in bank.sites]
    first = {(0, "q"): (r(4, 64), r(256, 4)), (0, "o"): (r(4, 256), r(64, 4))}
    nan = r(64, 4)
    nan[3, 1] = float("nan")
    for bad in ((r(5, 96), r(64, 5)), (r(4, 95), r(64, 4)), (r(4, 96), r(63, 4)),
                (r(4, 96), r(64, 3)), (r(4, 96), nan)):
        with pytest.raises(ValueError):
            bank.set(1, {**first, (1, "down"): bad})
        for site, was in zip(bank.sites, before):
            for s, v in site.items():
                assert all(torch.equal(a, b) for a, b in zip(v, was[s]))


@pytest.mark.parametrize("small", [1e-14, 1e-19, 1e-22, 1e-38])
def test_bank_takes_modules_of_far_scales(small):
    """Modules of one product whose scales are any factor apart: the larger one's
    integers are those of the module alone, the smaller one's are what is left of
    it at the larger one's exponent."""
    m = _bank_model()
    bank = lora.AdapterBank(m, 1, 4)
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g)
    q, k = (r(4, 64), r(256, 4)), (r(4, 64), r(128, 4) * small)
    bank.set(0, {(0, "q"): q, (0, "k"): k})
    _, _, bm, bk = bank.sites[0]["qkv"]
    _, _, qm, qk = lora.quantize(*q, m.layers[0].q_m, m.layers[0].q_k)
    _, _, km, kk = lora.quantize(*k, m.layers[0].k_m, m.layers[0].k_k)
    assert int(bk[0]) == qk and torch.equal(bm[0, :256], qm)
    exact = km.double() * 2.0 ** (qk - kk)
    assert ((bm[0, 256:384] - exact).abs() <= 0.5).all()


def test_step_is_sized_by_the_rows_in_it(step_bounds):
    """Rows without new tokens, however long, do not size a step's launches and
    scratch."""
    m = _step_model()
    cache = packed.PackedCache(m, 3, 3000)
    for lens, new, S in (([2900, 5, 0], (0, 1, 0), 6), ([2900, 5, 0], (1, 1, 0), 2901),
                         ([0, 0, 2999], (7, 0, 0), 7), ([130, 0, 2999], (2, 64, 0), 132)):
        cache.lens = lens
        with pytest.raises(_Launched):
            m.forward_packed(torch.zeros(sum(new), dtype=I64), new, cache)
        assert step_bounds[-1] == dict(N=sum(new), B=3, S=S, max_new=max(new))


def test_lora_refuses_more_rows_than_a_launch_takes():
    """Before the product is launched, by name."""
    _refused("lora_gemm", _lora(), {"rows": lambda c: _lora(N=1 << 20, K=16)})
    t = torch.zeros(64, dtype=I64)
    with pytest.raises(RuntimeError, match=r"detllm_lora_add failed \(code -34\)"):
        _lib.native().entries()["detllm_lora_add"](0, t, t, t, t, t, t, t, 1 << 20, 64, 10, 16, 2)
