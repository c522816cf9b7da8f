"""Performance cases of the long-context operators over the paged int8 KV
cache: the calls, their plain forms in elementary torch operations, and the
work of each.

Everything is integer arithmetic that the definition fixes to the last bit.
With int8 queries and keys, scores are s_j = q . k_j; over the visible slots
the row maximum m (0 if nothing is visible), n_j = m - s_j, u = n_j div tpos,
r = n_j mod tpos, e_j = (tpos - ceil(r / 2)) >> min(u, 62), den = max(sum e, 1),
p_j = floor((e_j 2^14 + floor(den / 2)) / den), context = sum p_j v_j.

Kinds (``case["kind"]``):

* ``window_decode`` / ``window_prefill``: attention in which a query sees the
  last ``window`` valid slots up to its own and the first ``sinks`` valid slots.
* ``acc_decode`` / ``acc_prefill``: attention that adds each slot's weight p,
  summed over the query heads of a kv head (and over a chunk's valid queries),
  to accumulators [B, n_kv, slots].
* ``evict``: from those accumulators the slots of each row that stay (the
  first ``sinks``, the last ``recent`` and the heaviest others, ties to the
  lower slot), and the K and V of all layers moved together.
* ``shared_decode``: one query per row where the rows' first ``shared`` slots
  are the same pages.

Products of int8 by int8 over 128 channels (below 2^24) and of p by v (the p of
a row sum to at most 2^15, so below 2^22) are exact in float32 in any order.
"""

import functools
import math

import torch

own = False

I32, I64, F32 = torch.int32, torch.int64, torch.float32
PAGE = HD = 128


def listed():
    return [
        # the smallest call: one user's step shortly after a short prompt
        dict(name="window_decode_1x320", kind="window_decode", B=1, S=320, n_q=16, n_kv=8,
             window=128, sinks=4),
        # a serving batch far into long replies, window of 2048
        dict(name="window_decode_32x8000", kind="window_decode", B=32, S=8000, n_q=16, n_kv=8,
             window=2048, sinks=4),
        # short ragged prompts, odd sizes
        dict(name="window_prefill_3x333", kind="window_prefill", B=3, T=333, past=0, n_q=16,
             n_kv=8, window=100, sinks=1),
        # a chunk of a long document after 6144 slots, four query heads per kv head
        dict(name="window_prefill_1x2048_past", kind="window_prefill", B=1, T=2048, past=6144,
             n_q=32, n_kv=8, window=1024, sinks=4),
        # one step of a small batch that tracks its weights, no grouped heads
        dict(name="acc_decode_8x320", kind="acc_decode", B=8, S=320, n_q=8, n_kv=8),
        # the same for a full serving batch at a long context
        dict(name="acc_decode_32x4000", kind="acc_decode", B=32, S=4000, n_q=16, n_kv=8),
        # ordinary short prompts whose weights are tracked from the start
        dict(name="acc_prefill_2x200", kind="acc_prefill", B=2, T=200, past=0, n_q=16, n_kv=8),
        # a long prompt
        dict(name="acc_prefill_1x2048", kind="acc_prefill", B=1, T=2048, past=0, n_q=16, n_kv=8),
        # one user's short cache cut to a small budget
        dict(name="evict_1x400", kind="evict", B=1, S=400, n_kv=8, budget=150, recent=32,
             sinks=4, layers=2),
        # a batch of long caches cut to a quarter
        dict(name="evict_8x4000", kind="evict", B=8, S=4000, n_kv=8, budget=1024, recent=256,
             sinks=4, layers=8),
        # four samples of one prompt
        dict(name="shared_decode_4x552", kind="shared_decode", B=4, S=552, shared=512, n_q=32,
             n_kv=8),
        # a full batch behind one long system prompt
        dict(name="shared_decode_64x8392", kind="shared_decode", B=64, S=8392, shared=8192,
             n_q=16, n_kv=8),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["window_decode", "window_prefill", "acc_decode", "acc_prefill", "evict",
                       "shared_decode"])
    n_q, n_kv = rng.choice([(16, 8), (16, 8), (8, 8), (32, 8), (8, 1), (4, 2)])
    heads = dict(n_q=n_q, n_kv=n_kv)
    rows = 16 / max(16, n_q)     # more heads, fewer rows
    if kind == "window_decode":
        return dict(kind=kind, B=_log(rng, 1, int(32 * rows)), S=_log(rng, 2, 8000),
                    window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 64]), **heads)
    if kind == "window_prefill":
        B = _log(rng, 1, 8)
        T = _log(rng, 2, 2048 // B)
        return dict(kind=kind, B=B, T=T, past=rng.choice([0, _log(rng, 1, 6144 // B)]),
                    window=_log(rng, 1, 2048), sinks=rng.choice([0, 1, 4, 64]), **heads)
    if kind == "acc_decode":
        return dict(kind=kind, B=_log(rng, 1, int(32 * rows)), S=_log(rng, 1, 4000),
                    **heads)
    if kind == "acc_prefill":
        B = _log(rng, 1, 8)
        T = _log(rng, 2, 1024 // B)
        return dict(kind=kind, B=B, T=T, past=rng.choice([0, _log(rng, 1, 1024 // B)]), **heads)
    if kind == "evict":
        S = _log(rng, 16, 4000)
        budget = _log(rng, 4, S)
        recent = rng.randint(0, budget // 2)
        return dict(kind=kind, B=_log(rng, 1, 8), S=S, n_kv=n_kv, budget=budget, recent=recent,
                    sinks=rng.randint(0, min(4, budget - recent)), layers=_log(rng, 1, 8))
    shared = PAGE * _log(rng, 1, 64)
    return dict(kind=kind, B=_log(rng, 2, int(64 * rows)), S=shared + _log(rng, 1, 200),
                shared=shared, **heads)


# ------------------------------------------------------------------ preparation

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)


def _gauss_i8(g, std, *shape):
    x = torch.randn(shape, dtype=F32, device="cuda", generator=g)
    return (x * std).round_().clamp_(-127, 127).to(torch.int8)


def _pools(g, pages, n_kv, *lead):
    """K and V pages as the cache's static scales leave them: a bell of int8."""
    return (_gauss_i8(g, 30, *lead, pages, n_kv, PAGE, HD),
            _gauss_i8(g, 30, *lead, pages, n_kv, HD, PAGE))


def _queries(g, *shape):
    """Queries quantised per head row, and the exponential's constant of each:
    the score step in which a weight halves, for logits of a few units."""
    return (_gauss_i8(g, 42, *shape, HD),
            torch.randint(1500, 24000, shape, dtype=I64, device="cuda", generator=g))


def _ragged(g, B, T):
    """[B, T] of right-padded rows: lengths in (T/2, T], the first row full."""
    lens = torch.randint(T // 2 + 1, T + 1, (B,), device="cuda", generator=g)
    lens[0] = T
    return torch.arange(T, device="cuda")[None] < lens[:, None]


def _table(g, B, w):
    return torch.randperm(B * w, device="cuda", generator=g).view(B, w).to(I32)


def prepare(case, seed):
    g = _gen(seed)
    kind, B, n_kv = case["kind"], case["B"], case["n_kv"]
    T = case.get("T", 1)
    S = case["past"] + T if "past" in case else case["S"]
    w = -(-S // PAGE)
    valid = torch.zeros(B, w * PAGE, dtype=torch.bool, device="cuda")
    if "past" in case:      # what is there, then a chunk of prompts, both right-padded
        past = case["past"]
        if past:
            valid[:, :past] = _ragged(g, B, past)
        valid[:, past:S] = _ragged(g, B, T)
    else:                   # right-padded prompts, then the replies' slots
        P = 3 * S // 4
        valid[:, P:S] = True
        if P:
            valid[:, :P] = _ragged(g, B, P)
    if kind == "evict":
        L, wb = case["layers"], -(-case["budget"] // PAGE)
        kp, vp = _pools(g, B * (w + wb), n_kv, L)
        pages = torch.randperm(B * (w + wb), device="cuda", generator=g).to(I32)
        # weights fall off with rank, as attention's do: a few slots carry most
        x = torch.rand(B, n_kv, w * PAGE, dtype=F32, device="cuda", generator=g)
        acc = (2.0 ** (22 * x)).to(I64) * valid[:, None]
        return dict(case, kp=kp, vp=vp, table=pages[:B * w].view(B, w).contiguous(),
                    dst=pages[B * w:].view(B, wb).contiguous(), valid=valid, acc=acc)
    if kind == "shared_decode":
        ws = case["shared"] // PAGE
        kp, vp = _pools(g, ws + B * (w - ws), n_kv)
        pages = torch.randperm(kp.shape[0], device="cuda", generator=g).to(I32)
        table = torch.cat([pages[:ws].expand(B, ws), pages[ws:].view(B, w - ws)], dim=1)
        valid[:, :case["shared"]] = True
        table = table.contiguous()
    else:
        kp, vp = _pools(g, B * w, n_kv)
        table = _table(g, B, w)
    lead = (B, case["n_q"], T) if "past" in case else (B, case["n_q"])
    q8, tpos = _queries(g, *lead)
    state = dict(case, q8=q8, tpos=tpos, kp=kp, vp=vp, table=table, valid=valid)
    if kind.startswith("acc"):
        state["acc"] = torch.randint(0, 1 << 30, (B, n_kv, w * PAGE), dtype=I64, device="cuda",
                                     generator=g)
    return state


# ------------------------------------------------------------------ plain forms

def _keys(pool, table, S):
    """[B, n_kv, S, 128] float32 of the rows' slots from a K pool."""
    x = pool[table.long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, HD)[:, :, :S].to(F32)


def _values(pool, table, S):
    """The same of a V pool, whose pages hold V transposed."""
    return _keys(pool.transpose(-1, -2), table, S)


def _weights(x, tpos, vis):
    """p [.., S] int32 of integer scores x, the rows' constants tpos [.., 1]
    and visibility vis: differences and exponentials in 32 bits, the
    denominator and the last quotient in 64."""
    x = x.to(I32)
    lowest = torch.full((), -(1 << 30), dtype=I32, device=x.device)
    m = torch.where(vis, x, lowest).amax(-1, keepdim=True)
    n = torch.where(vis, m - x, 0)
    t = tpos.to(I32)
    u = n // t
    r = n - u * t
    e = torch.where(vis, (t - ((r + 1) >> 1)) >> u.clamp(max=31), 0)
    den = e.sum(-1, keepdim=True, dtype=I64).clamp(min=1)
    return (((e.to(I64) << 14) + den // 2) // den).to(I32)


def _visible(valid, T, past, window=None, sinks=0):
    """[B, 1, T, S]: what the query at slot past + t sees."""
    S = past + T
    v = valid[:, :S]
    s, t = torch.arange(S, device=v.device), torch.arange(past, S, device=v.device)
    vis = v[:, None, :] & (s[None] <= t[:, None])
    if window is not None:
        c = v.cumsum(1)      # valid slots up to and with this one
        ahead = c[:, past:, None] - c[:, None, :]
        vis = vis & ((ahead < window) | (c[:, None, :] <= sinks))
    return vis[:, None]


def _attend(state, vis):
    """(weights [B, n_kv, G * T, S] int32, context int64) of the queries."""
    q, tpos, n_kv = state["q8"], state["tpos"], state["n_kv"]
    if q.dim() == 3:
        q, tpos = q[:, :, None], tpos[:, :, None]
    B, n_q, T, _ = q.shape
    G, S = n_q // n_kv, vis.shape[-1]
    k, v = (f(state[n], state["table"], S) for f, n in ((_keys, "kp"), (_values, "vp")))
    x = q.reshape(B, n_kv, G * T, HD).to(F32) @ k.transpose(-1, -2).contiguous()
    see = vis.expand(B, G, T, S).reshape(B, 1, G * T, S)
    p = _weights(x, tpos.reshape(B, n_kv, G * T, 1), see)
    ctx = (p.to(F32) @ v).to(I64).view(B, n_q, T, HD).transpose(1, 2).reshape(B, T, n_q * HD)
    return p, ctx


def _plain_decode(state, window=None, sinks=0):
    S = state["S"]
    p, ctx = _attend(state, _visible(state["valid"], 1, S - 1, window, sinks))
    return p, ctx[:, 0]


def _plain_acc(state, p, past, T):
    """The accumulators with the weights of the queries at valid slots added."""
    B, n_kv, R, S = p.shape
    counts = state["valid"][:, None, past:past + T].expand(B, R // T, T).reshape(B, 1, R, 1)
    acc = state["acc"].clone()
    acc[:, :, :S] += torch.where(counts, p, 0).sum(2, dtype=I64)
    return acc


def _plain_select(state):
    """Slots that stay [B, budget] in ascending order (-1 behind them), and
    their accumulators."""
    S, budget, recent, sinks = (state[k] for k in ("S", "budget", "recent", "sinks"))
    v = state["valid"][:, :S]
    c = v.cumsum(1)
    n = c[:, -1:]
    always = (c <= sinks) | (n - c < recent) | (n <= budget)
    w = state["acc"][:, :, :S].sum(1)
    first = torch.iinfo(I64).max
    key = torch.where(v, torch.where(always, first, w), -1)
    best = key.sort(dim=1, descending=True, stable=True)
    keep = torch.where(best.values[:, :budget] >= 0, best.indices[:, :budget], S).sort(dim=1).values
    there = keep < S
    at = torch.where(there, keep, 0)
    acc = state["acc"].gather(2, at[:, None].expand(-1, state["n_kv"], -1))
    return torch.where(there, keep, -1).to(I32), torch.where(there[:, None], acc, 0)


def _plain_compact(state, keep):
    """The kept slots of every layer written to the pages of dst, zeros
    behind them."""
    B, wb = state["dst"].shape
    slots = torch.full((B, wb * PAGE), -1, dtype=I64, device=keep.device)
    slots[:, :keep.shape[1]] = keep.long()
    at = slots.clamp(min=0)
    pg, off = state["table"].long().gather(1, at // PAGE), at % PAGE
    there = (slots >= 0)[:, :, None, None]
    k = torch.where(there, state["kp"][:, pg, :, off].permute(2, 0, 1, 3, 4), 0)
    v = torch.where(there, state["vp"][:, pg, :, :, off].permute(2, 0, 1, 3, 4), 0)
    L, n_kv = k.shape[0], k.shape[3]
    dst = state["dst"].reshape(-1).long()
    k = k.reshape(L, B * wb, PAGE, n_kv, HD).transpose(2, 3)
    v = v.reshape(L, B * wb, PAGE, n_kv, HD).permute(0, 1, 3, 4, 2)
    state["kp"][:, dst] = k
    state["vp"][:, dst] = v


def _plain_shared(state):
    """The prefix's products once for the whole batch, the suffixes' per row."""
    B, S, P, n_q, n_kv = (state[k] for k in ("B", "S", "shared", "n_q", "n_kv"))
    G, tb = n_q // n_kv, state["table"]
    q = state["q8"].view(B, n_kv, G, HD).to(F32)
    qa = q.transpose(0, 1).reshape(n_kv, B * G, HD)
    pre, own_pages = tb[:1, :P // PAGE], tb[:, P // PAGE:]
    kf, vf = _keys(state["kp"], pre, P)[0], _values(state["vp"], pre, P)[0]
    ks, vs = _keys(state["kp"], own_pages, S - P), _values(state["vp"], own_pages, S - P)
    xf = (qa @ kf.transpose(-1, -2).contiguous()).view(n_kv, B, G, P).transpose(0, 1)
    x = torch.cat([xf, q @ ks.transpose(-1, -2).contiguous()], dim=-1)
    p = _weights(x, state["tpos"].view(B, n_kv, G, 1), state["valid"][:, None, None, :S]).to(F32)
    pf = p[..., :P].transpose(0, 1).reshape(n_kv, B * G, P)
    ctx = (pf @ vf).view(n_kv, B, G, HD).transpose(0, 1) + p[..., P:].contiguous() @ vs
    return ctx.to(I64).reshape(B, n_q * HD)


# ------------------------------------------------------------------ one pass

@functools.lru_cache(maxsize=None)
def _ops():
    from idempotent_llm_amd import torch_ops  # noqa: F401  (registers the operators)
    return torch.ops.detllm_rocm


def run(state):
    kind = state["kind"]
    if own:
        return _run_own(kind, state)
    if kind == "window_decode":
        return _plain_decode(state, state["window"], state["sinks"])[1]
    if kind == "window_prefill":
        return _attend(state, _visible(state["valid"], state["T"], state["past"],
                                       state["window"], state["sinks"]))[1]
    if kind == "acc_decode":
        p, ctx = _plain_decode(state)
        return dict(out=ctx, acc=_plain_acc(state, p, state["S"] - 1, 1))
    if kind == "acc_prefill":
        T, past = state["T"], state["past"]
        p, ctx = _attend(state, _visible(state["valid"], T, past))
        return dict(out=ctx, acc=_plain_acc(state, p, past, T))
    if kind == "evict":
        keep, acc = _plain_select(state)
        _plain_compact(state, keep)
        return dict(keep=keep, acc=acc, k=state["kp"], v=state["vp"])
    return _plain_shared(state)


def _run_own(kind, state):
    ops = _ops()
    if kind == "evict":
        keep, acc = ops.kv_select(state["acc"], state["valid"], state["S"], state["budget"],
                                  state["recent"], state["sinks"])
        ops.kv_compact(state["kp"].unbind(0), state["vp"].unbind(0), state["table"], state["dst"],
                       keep)
        return dict(keep=keep, acc=acc, k=state["kp"], v=state["vp"])
    args = [state[k] for k in ("q8", "tpos", "kp", "vp", "table", "valid")]
    if kind == "window_decode":
        return ops.attn_window_decode(*args, state["S"], state["window"], state["sinks"])
    if kind == "window_prefill":
        return ops.attn_window_prefill(*args, state["past"], state["window"], state["sinks"])
    if kind == "shared_decode":
        return ops.attn_decode_shared(*args, state["S"], state["shared"])
    acc = state["acc"].clone()      # added to in place: this pass's own copy
    if kind == "acc_decode":
        out = ops.attn_decode_acc(*args, state["S"], acc)
    else:
        out = ops.attn_prefill_acc(*args, state["past"], acc)
    return dict(out=out, acc=acc)


# ------------------------------------------------------------------ the work of a pass

def work(case):
    kind, B, n_kv = case["kind"], case["B"], case["n_kv"]
    if kind == "evict":
        S, kept, L = case["S"], min(case["S"], case["budget"]), case["layers"]
        return dict(bytes=B * (S * (8 * n_kv + 1) + kept * (16 * n_kv + 4)
                               + 2 * L * n_kv * 2 * HD * kept), flops=0)
    n_q = case["n_q"]
    T = case.get("T", 1)
    past = case["past"] if "past" in case else case["S"] - 1
    S = past + T
    rows = B * T * n_q * (HD + 8 + 8 * HD)      # queries, constants, contexts
    slot = 2 * n_kv * HD + 1                    # K, V and the flag of a slot
    if kind == "shared_decode":
        P = case["shared"]
        return dict(bytes=(P + B * (S - P)) * slot + B * P + rows, flops=4 * B * S * n_q * HD)
    if "window" in case:
        see = case["window"] + case["sinks"]
        pairs = sum(min(past + t + 1, see) for t in range(T))
        slots = min(S, see + T - 1)
    else:
        pairs, slots = T * past + T * (T + 1) // 2, S
    extra = 16 * n_kv * S if kind.startswith("acc") else 0
    return dict(bytes=B * (slots * slot + extra) + rows, flops=4 * B * pairs * n_q * HD)


# ------------------------------------------------------------------ in 64 bits

def _exact_row(q, tpos, k, v, see):
    """Weights and context of one query over one head's slots, on the CPU in
    float64 products (exact below 2^53) and int64 arithmetic."""
    j = see.nonzero()[:, 0]
    p = torch.zeros(see.shape[0], dtype=I64)
    if j.numel():
        s = (k[j].double() @ q.double()).to(I64)
        n = s.max() - s
        u = torch.div(n, tpos, rounding_mode="floor")
        half = torch.div(n - u * tpos + 1, 2, rounding_mode="floor")
        e = (tpos - half) >> u.clamp(max=62)
        den = max(int(e.sum()), 1)
        p[j] = torch.div(e * 16384 + den // 2, den, rounding_mode="floor")
    return p, (p.double() @ v.double()).to(I64)


def exact(case, seed):
    kind, B, n_kv = case["kind"], case["B"], case["n_kv"]
    if kind == "evict":
        if B * case["S"] * case["layers"] > 40000:
            return None
        return _exact_evict(case, prepare(case, seed))
    n_q, T = case["n_q"], case.get("T", 1)
    past = case["past"] if "past" in case else case["S"] - 1
    if B * n_q * T * (300 + past + T) > 12_000_000:
        return None
    s = prepare(case, seed)
    q8, tpos, kp, vp, tb, valid = (s[n].cpu() for n in ("q8", "tpos", "kp", "vp", "table", "valid"))
    out = torch.zeros(B, T, n_q * HD, dtype=I64)
    acc = s["acc"].cpu() if "acc" in s else None
    for b in range(B):
        ids = tb[b].long()
        for h in range(n_q):
            kv = h // (n_q // n_kv)
            k = kp[ids, kv].reshape(-1, HD)
            v = vp[ids, kv].transpose(1, 2).reshape(-1, HD)
            for t in range(T):
                at = past + t
                live = valid[b, :at + 1].nonzero()[:, 0]
                if "window" in case:
                    live = torch.cat([live[:case["sinks"]], live[-case["window"]:]])
                see = torch.zeros(at + 1, dtype=torch.bool)
                see[live] = True
                row = (b, h, t) if q8.dim() == 4 else (b, h)
                p, ctx = _exact_row(q8[row], int(tpos[row]), k[:at + 1], v[:at + 1], see)
                out[b, t, h * HD:(h + 1) * HD] = ctx
                if acc is not None and bool(valid[b, at]):
                    acc[b, kv, :at + 1] += p
    out = out if "past" in case else out[:, 0]
    return dict(out=out, acc=acc) if acc is not None else out


def _exact_evict(case, s):
    S, budget = case["S"], case["budget"]
    acc, valid, tb, dst = (s[n].cpu() for n in ("acc", "valid", "table", "dst"))
    kp, vp = s["kp"].cpu(), s["vp"].cpu()
    keep = torch.full((case["B"], budget), -1, dtype=I32)
    kept = torch.zeros(case["B"], case["n_kv"], budget, dtype=I64)
    old_k, old_v = kp.clone(), vp.clone()
    for b in range(case["B"]):
        live = valid[b, :S].nonzero()[:, 0].tolist()
        if len(live) > budget:
            lo, hi = case["sinks"], len(live) - case["recent"]
            weight = acc[b].sum(0).tolist()
            mid = sorted(live[lo:hi], key=lambda j: (-weight[j], j))[:budget - lo - case["recent"]]
            live = sorted(live[:lo] + mid + live[hi:])
        n = len(live)
        keep[b, :n] = torch.tensor(live, dtype=I32)
        kept[b, :, :n] = acc[b][:, live]
        for page in dst[b].tolist():
            kp[:, page], vp[:, page] = 0, 0
        for i, j in enumerate(live):
            a, c = int(dst[b, i // PAGE]), int(tb[b, j // PAGE])
            kp[:, a, :, i % PAGE] = old_k[:, c, :, j % PAGE]
            vp[:, a, :, :, i % PAGE] = old_v[:, c, :, :, j % PAGE]
    return dict(keep=keep, acc=kept, k=kp, v=vp)
