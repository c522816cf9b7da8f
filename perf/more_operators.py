"""Performance cases of the packed serving step: requests of any lengths in one
batch without padding, prompts fed in chunks beside running replies, pages
mapped on the GPU, a low-rank adapter per request.

Everything is integer arithmetic that the definition fixes to the last bit.
Kinds (``case["kind"]``); a batch has rows b with past_b slots filled and new_b
tokens, whose token rows follow each other (row b's at cu_b .. cu_{b+1} - 1):

* ``plan``: the step's bookkeeping. Row b needs ceil((past_b + new_b) / 128)
  pages and has the leading mapped ones of its table row. Surplus pages are
  appended to the free list, missing ones popped from its end, both in
  row-major order. Out: cu, and per token its row, position and slot
  (page * 128 + position % 128).
* ``epilogue``: the product of the Q, K and V projections to int8 queries,
  their DI-Exp constants, and K and V at the tokens' slots: per head a common
  shift to 16 bits, RMS norm (20 fraction bits), gamma, rotation (14 bits);
  queries smoothed and quantised by their maximum, keys and values
  requantised to static scales.
* ``attn``: token t of row b sees the slots up to past_b + t. With s_j = q . k_j,
  m their maximum, n_j = m - s_j, u = n_j div tpos, r = n_j mod tpos,
  e_j = (tpos - ceil(r / 2)) >> min(u, 62), den = max(sum e, 1),
  p_j = floor((e_j 2^14 + floor(den / 2)) / den), context = sum p_j v_j.
* ``lora``: y = x W^T and the adapter of each token: u = A x, h = max(ilog2(max
  |u|) - 12, 0), w = round(u / 2^h), v = B w, y += round(v bm / 2^(bk - h))
  (rounding half up).

Products of int8 by int8 over at most 1024 channels and sums of p v (a row's p
sum to at most 2^14 + S / 2) stay below 2^24, so they are exact in float32 in
any order; the adapters' products are made in float64.
"""

import functools
import math
import random

import torch

own = False

I8, I32, I64, F32, F64 = torch.int8, torch.int32, torch.int64, torch.float32, torch.float64
PAGE = HD = 128


def listed():
    return [
        # the bookkeeping of a small batch's decode step
        dict(name="plan_8", kind="plan", mix="decode", B=8, lo=40, hi=900, N=8, width=64, rows=1),
        # a large batch: prompts admitted beside replies, and rows that ended
        dict(name="plan_384", kind="plan", mix="admit", B=384, lo=100, hi=8000, N=16384, width=128,
             rows=2),
        # eight decode rows
        dict(name="epilogue_8", kind="epilogue", N=8, parts=1, n_q=16, n_kv=8, rows=3),
        # a full step of prompt chunks
        dict(name="epilogue_2048", kind="epilogue", N=2048, parts=1, n_q=16, n_kv=8, rows=4),
        # one user's step shortly after a short prompt
        dict(name="attn_1x300", kind="attn", mix="decode", B=1, lo=300, hi=300, n_q=16, n_kv=8,
             rows=5),
        # a serving batch of replies, from short to long
        dict(name="attn_decode_48", kind="attn", mix="decode", B=48, lo=100, hi=8000, n_q=16,
             n_kv=8, rows=6),
        # short drafts verified in one step, four query heads per kv head
        dict(name="attn_verify_16x4", kind="attn", mix="verify", B=16, lo=200, hi=3000, new=4,
             n_q=32, n_kv=8, rows=7),
        # a few ordinary prompts admitted together
        dict(name="attn_prompts_6", kind="attn", mix="prompts", B=6, lo=60, hi=700, n_q=16, n_kv=8,
             rows=8),
        # a chunk of a long document beside a batch of replies
        dict(name="attn_mixed_25", kind="attn", mix="mixed", B=25, lo=200, hi=6000, new=512,
             n_q=16, n_kv=8, rows=9),
        # a whole long prompt in one step
        dict(name="attn_prompt_2500", kind="attn", mix="prompts", B=1, lo=2500, hi=2500, n_q=16,
             n_kv=8, rows=10),
        # eight users with an adapter each, one token
        dict(name="lora_8", kind="lora", N=8, runs=8, n_ad=8, rank=16, K=1024, C=4096, rows=11),
        # a step of prompt chunks of six users, some without an adapter
        dict(name="lora_2000", kind="lora", N=2000, runs=6, n_ad=4, rank=32, K=1024, C=4096,
             rows=12),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "epilogue", "attn", "attn", "attn", "lora"])
    rows = rng.randrange(1 << 30)
    if kind == "plan":
        B = _log(rng, 1, 384)
        hi = _log(rng, 40, 8000)
        return dict(kind=kind, mix=rng.choice(["decode", "admit"]), B=B, lo=_log(rng, 1, hi), hi=hi,
                    N=max(B, _log(rng, 1, 16384)), width=rng.choice([64, 100, 128]), rows=rows)
    n_q, n_kv = rng.choice([(16, 8), (16, 8), (8, 8), (32, 8), (8, 1), (4, 2)])
    if kind == "epilogue":
        return dict(kind=kind, N=_log(rng, 1, 2048 * 16 // max(16, n_q)), parts=rng.choice([1, 1, 4]),
                    n_q=n_q, n_kv=n_kv, rows=rows)
    if kind == "lora":
        N = _log(rng, 1, 2000)
        return dict(kind=kind, N=N, runs=_log(rng, 1, min(N, 32)), n_ad=rng.choice([1, 3, 4, 8]),
                    rank=rng.choice([16, 32, 48]), K=16 * _log(rng, 16, 64),
                    C=16 * _log(rng, 16, 256), rows=rows)
    mix = rng.choice(["decode", "verify", "prompts", "mixed"])
    case = dict(kind=kind, mix=mix, n_q=n_q, n_kv=n_kv, rows=rows)
    less = max(16, n_q) // 16    # more heads, fewer rows
    if mix == "decode":
        case.update(B=_log(rng, 1, 48 // less), hi=_log(rng, 1, 8000))
    elif mix == "verify":
        case.update(B=_log(rng, 1, 16), hi=_log(rng, 8, 3000), new=rng.choice([2, 3, 4, 5, 8]))
    elif mix == "prompts":
        B = _log(rng, 1, 8)
        case.update(B=B, hi=_log(rng, 2, 2500 // (B * less)))
    else:
        case.update(B=_log(rng, 2, 25 // less), hi=_log(rng, 64, 6000), new=_log(rng, 2, 512 // less))
    return dict(case, lo=_log(rng, 1, case["hi"]))


@functools.lru_cache(maxsize=256)
def _rows_of(mix, B, lo, hi, new, seed):
    """[(past, new)] of a batch's rows: lengths even over their logarithm, the
    first row the longest."""
    rng = random.Random(seed)
    out = []
    for b in range(B):
        n = hi if b == 0 else _log(rng, lo, hi)
        if mix == "decode":
            out.append((n - 1, 1))
        elif mix == "verify":
            out.append((max(0, n - new), new))
        elif mix == "prompts":
            out.append((0, n))
        elif mix == "mixed":      # the first row's chunk, the others' single tokens
            out.append((max(0, n - new), min(n, new)) if b == 0 else (n - 1, 1))
        else:                     # admit: a third each ended, running and new
            out.append([(0, 0), (n - 1, 1), (0, n)][rng.randrange(3)])
    return out


def _rows(case):
    rows = _rows_of(case["mix"], case["B"], case["lo"], case["hi"], case.get("new", 0), case["rows"])
    if case["kind"] != "plan":
        return rows
    left, out = case["N"] - case["B"], []    # new prompts while the step has room for them
    for past, new in rows:
        out.append((past, new) if new <= 1 or new - 1 <= left else (0, 1))
        left -= max(0, out[-1][1] - 1)
    return out


# ------------------------------------------------------------------ preparation

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)


def _gauss_i8(g, std, *shape):
    x = torch.randn(shape, dtype=F32, device="cuda", generator=g)
    return (x * std).round_().clamp_(-127, 127).to(I8)


def _ints(g, lo, hi, *shape, dtype=I64):
    return torch.randint(lo, hi, shape, dtype=dtype, device="cuda", generator=g)


def _i32(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "plan":
        return _prepare_plan(case, g)
    if case["kind"] == "epilogue":
        return _prepare_epilogue(case, g)
    if case["kind"] == "lora":
        return _prepare_lora(case, g)
    rows, n_q, n_kv = _rows(case), case["n_q"], case["n_kv"]
    lens = [p + n for p, n in rows]
    w = [-(-n // PAGE) for n in lens]
    N, pages = sum(n for _, n in rows), sum(w)
    order = torch.randperm(pages, device="cuda", generator=g).to(I32)
    table = torch.full((len(rows), max(w)), -1, dtype=I32, device="cuda")
    at = 0
    for b, n in enumerate(w):
        table[b, :n] = order[at:at + n]
        at += n
    cu = [0]
    for _, n in rows:
        cu.append(cu[-1] + n)
    # K and V as the cache's static scales leave them, queries quantised per head
    # row, the exponential's constant the score step in which a weight halves
    return dict(case, q8=_gauss_i8(g, 42, N, n_q, HD), tpos=_ints(g, 1500, 24000, N, n_q),
                kp=_gauss_i8(g, 30, pages, n_kv, PAGE, HD),
                vp=_gauss_i8(g, 30, pages, n_kv, HD, PAGE), table=table, cu=_i32(cu),
                past=_i32([p for p, _ in rows]), lens=rows, S=max(lens),
                max_new=max(n for _, n in rows),
                err=torch.zeros(1, dtype=I32, device="cuda"))


def _prepare_plan(case, g):
    """Rows as the step before left them: a running row's pages, an ended
    row's (some of which it still has), none for a new one."""
    rows, width = _rows(case), case["width"]
    rng = random.Random(case["rows"] + 1)
    have = [-(-p // PAGE) if p else (rng.randrange(1, 9) if not n else 0) for p, n in rows]
    pages = sum(have) + sum(-(-(p + n) // PAGE) for p, n in rows)
    order = torch.randperm(pages, device="cuda", generator=g).to(I32)
    # the table, the free list and its length, one buffer
    book = torch.full((len(rows) * width + pages + 1,), -1, dtype=I32, device="cuda")
    table, at = book[:len(rows) * width].view(len(rows), width), 0
    for b, n in enumerate(have):
        table[b, :n] = order[at:at + n]
        at += n
    book[len(rows) * width:-1][:pages - at] = order[at:]
    book[-1] = pages - at
    return dict(case, book=book, past=_i32([p for p, _ in rows]), new=_i32([n for _, n in rows]),
                err=torch.zeros(1, dtype=I32, device="cuda"))


def _prepare_epilogue(case, g):
    N, n_q, n_kv = case["N"], case["n_q"], case["n_kv"]
    C = (n_q + 2 * n_kv) * HD
    pages = -(-N // PAGE) + 3
    ang = torch.arange(4096, dtype=F64)[:, None] * 1e6 ** (-torch.arange(0, HD, 2, dtype=F64) / HD)
    ang = torch.cat([ang, ang], dim=1)
    P = (torch.randn(case["parts"], N, C, dtype=F32, device="cuda", generator=g)
         * (60000 / case["parts"] ** 0.5)).to(I32)
    return dict(case, P=P, xm=_ints(g, 1 << 15, 1 << 16, N), xk=_ints(g, 18, 22, N),
                pos=_ints(g, 0, 4096, N),
                slot=torch.randperm(pages * PAGE, device="cuda", generator=g)[:N].contiguous(),
                q_m=_ints(g, 1 << 14, 1 << 16, n_q * HD), q_k=24,
                k_m=_ints(g, 1 << 14, 1 << 16, n_kv * HD), k_k=24,
                v_m=_ints(g, 1 << 14, 1 << 16, n_kv * HD), v_k=24,
                q_norm_m=_ints(g, 1 << 10, 1 << 12, HD), q_norm_k=11,
                k_norm_m=_ints(g, 1 << 10, 1 << 12, HD), k_norm_k=11,
                qs_m=_ints(g, 1 << 8, 1 << 10, n_kv * HD), qs_k=9,
                kq_m=_ints(g, 1 << 15, 1 << 16, n_kv * HD), kq_k=_ints(g, 18, 21, n_kv * HD),
                ks_m=_ints(g, 1 << 15, 1 << 16, n_kv), ks_k=_ints(g, 24, 27, n_kv),
                vq_m=_ints(g, 1 << 15, 1 << 16, n_kv), vq_k=_ints(g, 16, 20, n_kv),
                cos=torch.round(torch.cos(ang) * 16384).to(torch.int16).cuda(),
                sin=torch.round(torch.sin(ang) * 16384).to(torch.int16).cuda(),
                kp=_gauss_i8(g, 30, pages, n_kv, PAGE, HD),
                vp=_gauss_i8(g, 30, pages, n_kv, HD, PAGE),
                err=torch.zeros(1, dtype=I32, device="cuda"))


def _prepare_lora(case, g):
    N, K, C, r, n_ad = (case[k] for k in ("N", "K", "C", "rank", "n_ad"))
    rng = random.Random(case["rows"])
    cuts = sorted(rng.sample(range(1, N), min(case["runs"], N) - 1)) + [N]
    ids, at = [], 0
    for i, c in enumerate(cuts):      # a request's tokens follow each other
        ids += [-1 if i % 5 == 4 else rng.randrange(n_ad)] * (c - at)
        at = c
    # an adapter's change of a column is a small part of the column's own value
    return dict(case, x8=_gauss_i8(g, 40, N, K), w=_gauss_i8(g, 50, C, K),
                a8=_gauss_i8(g, 40, n_ad, r, K), b8=_gauss_i8(g, 40, n_ad, C, r),
                bm=_ints(g, 1 << 12, 1 << 15, n_ad, C), bk=_ints(g, 19, 23, n_ad),
                adapter=_i32(ids))


# ------------------------------------------------------------------ plain forms

def _plain_plan(state, table, free, n_free):
    B, width, N, dev = state["B"], state["width"], state["N"], table.device
    past, new = state["past"].long(), state["new"].long()
    need = (past + new + PAGE - 1) // PAGE
    have = (table >= 0).long().cumprod(1).sum(1)
    col = torch.arange(width, device=dev)[None]
    surplus = (col >= need[:, None]) & (col < have[:, None])
    missing = (col >= have[:, None]) & (col < need[:, None])
    n0, cap = n_free.long(), free.shape[0]
    at = torch.where(surplus.view(-1), n0 + surplus.view(-1).cumsum(0) - 1, cap)
    more = torch.cat([free, free[:1]]).index_put((at,), table.view(-1))[:cap]
    n1 = n0 + surplus.sum()
    n_mis = missing.sum()
    fits = n_mis <= n1
    take = (n1 - missing.view(-1).cumsum(0)).clamp(min=0)
    got = torch.where(missing & fits, more[take].view(B, width), torch.where(surplus, -1, table))
    table.copy_(got)
    free.copy_(more)
    n_free.copy_(n1 - torch.where(fits, n_mis, 0))
    cu = torch.zeros(B + 1, dtype=I64, device=dev)
    cu[1:] = new.cumsum(0)
    i = torch.arange(N, device=dev)
    row = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    live = row < B
    rc = row.clamp(max=B - 1)
    pos = torch.where(live, past[rc] + i - cu[rc], 0)
    page = table[rc, (pos // PAGE).clamp(max=width - 1)].long()
    slot = torch.where(live & (page >= 0), page * PAGE + pos % PAGE, -1)
    return cu.to(I32), torch.where(live, row, -1).to(I32), pos, slot


def _ilog2(x):
    """floor(log2 x) of x >= 1 below 2^53."""
    return torch.frexp(x.to(F64)).exponent.to(I64) - 1


def _rshift_round(x, s):
    return torch.where(s > 0, (x + (1 << (s.clamp(min=1) - 1))) >> s.clamp(min=1), x)


def _div_away(a, b):
    """Half away from zero, b > 0."""
    return torch.where(a < 0, -1, 1) * torch.div(a.abs() + torch.div(b, 2, rounding_mode="floor"), b,
                                                 rounding_mode="floor")


def _fit(num, den):
    """A 16-bit mantissa m and exponent e with m / 2^e nearest num / den."""
    def at(e):
        return _div_away(num << e.clamp(min=0), den << (-e).clamp(min=0))
    e = 15 - (_ilog2(num) - _ilog2(den))
    m = at(e)
    adj = torch.where(m >= 1 << 16, -1, torch.where(m < 1 << 15, 1, 0))
    e = e + adj
    m = torch.where(adj != 0, at(e), m)
    over = m >= 1 << 16
    return torch.where(over, (m + 1) >> 1, m), e - over.long()


def _norm_scale(m, k):
    """m as 16 bits, its exponent."""
    s = 15 - _ilog2(m.clamp(min=1))
    m = _rshift_round(m << s.clamp(min=0), (-s).clamp(min=0))
    over = m >= 1 << 16
    return torch.where(over, (m + 1) >> 1, m), k + s - over.long()


def _heads_normed(x, m, gamma, c, s):
    """[N, heads, 128]: the common shift, the norm with gamma, the rotation."""
    x = x * m.view(1, -1, HD)
    x = _rshift_round(x, (_ilog2(x.abs().amax(-1, keepdim=True).clamp(min=1)) - 15).clamp(min=0))
    up = 25 - _ilog2(x.abs().amax(-1, keepdim=True).clamp(min=1))
    x = x << up
    mean = _div_away((x * x).sum(-1, keepdim=True), torch.full((), HD, device=x.device))
    r = mean.to(F64).sqrt().to(I64)
    r = r - (r * r > mean).long()
    r = (r + ((r + 1) * (r + 1) <= mean).long()).clamp(min=1)
    x = _div_away(x << 20, r) * gamma
    half = torch.cat([-x[..., HD // 2:], x[..., :HD // 2]], dim=-1)
    return (x * c + half * s + (1 << 13)) >> 14


def _static(num, shift, s_m):
    """Requantised to the scale s_m: num / (s_m 2^shift), clamped."""
    return _div_away(num << (-shift).clamp(min=0), s_m << shift.clamp(min=0)).clamp(-128, 127).to(I8)


def _plain_epilogue(st):
    N, n_q, n_kv = st["N"], st["n_q"], st["n_kv"]
    G = n_q // n_kv
    P = st["P"].sum(0, dtype=I64).view(N, n_q + 2 * n_kv, HD)
    c, s = (st[n].long()[st["pos"]][:, None] for n in ("cos", "sin"))
    q = _heads_normed(P[:, :n_q], st["q_m"], st["q_norm_m"], c, s)
    k = _heads_normed(P[:, n_q:n_q + n_kv], st["k_m"], st["k_norm_m"], c, s)
    q = q * st["qs_m"].view(n_kv, HD).repeat_interleave(G, 0)
    am = q.abs().amax(-1).clamp(min=1)
    q8 = _div_away(q * 127, am[..., None]).clamp(-128, 127).to(I8)
    one, kk = _norm_scale(torch.ones_like(am), torch.full_like(am, 20 + st["q_norm_k"] + st["qs_k"]))
    qm, e = _fit(am * one, torch.full_like(am, 127))
    sm, sk = _norm_scale(qm * st["ks_m"].repeat_interleave(G), kk + e + st["ks_k"].repeat_interleave(G))
    tpos = _div_away(torch.ones_like(sk) << sk, sm + (sm >> 1) - (sm >> 4)).clamp(min=1)
    k8 = _static(k, (20 + st["k_norm_k"] - st["kq_k"]).view(n_kv, HD), st["kq_m"].view(n_kv, HD))
    v = P[:, n_q + n_kv:] * st["v_m"].view(n_kv, HD) * st["xm"].view(N, 1, 1)
    v8 = _static(v, (st["xk"].view(N, 1) + st["v_k"] - st["vq_k"])[..., None],
                 st["vq_m"].view(n_kv, 1))
    pg, off = st["slot"] // PAGE, st["slot"] % PAGE
    st["kp"][pg, :, off] = k8
    st["vp"][pg, :, :, off] = v8
    return dict(q8=q8, tpos=tpos, k=st["kp"], v=st["vp"])


def _weights(x, tpos, vis):
    """p [.., S] int32 of integer scores x, the rows' constants tpos [.., 1] and
    visibility vis: differences and exponentials in 32 bits, the denominator and
    the last quotient in 64."""
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


def _slots(st, b, S):
    """K and V of rows b (a slice), [rows, n_kv, S, 128] float32."""
    ids = st["table"][b, :-(-S // PAGE)].clamp(min=0).long()
    k = st["kp"][ids].transpose(1, 2).reshape(ids.shape[0], st["n_kv"], -1, HD)[:, :, :S]
    v = st["vp"][ids].transpose(1, 2).transpose(-1, -2).reshape(ids.shape[0], st["n_kv"], -1, HD)
    return k.to(F32), v[:, :, :S].to(F32)


def _plain_attn(st):
    """Neighbours of one number of tokens, at most 8, together, padded to the
    longest; the others one by one."""
    rows, n_q, n_kv = st["lens"], st["n_q"], st["n_kv"]
    G, dev = n_q // n_kv, st["q8"].device
    out = torch.empty(st["q8"].shape[0], n_q * HD, dtype=I64, device=dev)
    groups, b = [], 0
    while b < len(rows):
        e = b + 1
        while rows[b][1] <= 8 and e < len(rows) and rows[e][1] == rows[b][1]:
            e += 1
        groups.append((b, e))
        b = e
    at = 0
    for b, e in groups:
        R, T = e - b, rows[b][1]
        S = max(p + n for p, n in rows[b:e])
        k, v = _slots(st, slice(b, e), S)
        q = st["q8"][at:at + R * T].view(R, T, n_kv, G, HD).permute(0, 2, 3, 1, 4)
        tp = st["tpos"][at:at + R * T].view(R, T, n_kv, G).permute(0, 2, 3, 1)
        x = q.reshape(R, n_kv, G * T, HD).to(F32) @ k.transpose(-1, -2).contiguous()
        last = st["past"][b:e, None] + torch.arange(T, device=dev)
        vis = torch.arange(S, device=dev) <= last[..., None]
        p = _weights(x, tp.reshape(R, n_kv, G * T, 1),
                     vis[:, None].repeat(1, 1, G, 1))
        ctx = (p.to(F32) @ v).view(R, n_kv, G, T, HD).permute(0, 3, 1, 2, 4)
        out[at:at + R * T] = ctx.reshape(R * T, n_q * HD).to(I64)
        at += R * T
    return out


def _plain_lora(st):
    n_ad, r = st["n_ad"], st["rank"]
    y = (st["x8"].to(F32) @ st["w"].to(F32).t().contiguous()).to(I64)
    mine = st["adapter"][:, None] == torch.arange(n_ad, device=y.device)
    u = st["x8"].to(F64) @ st["a8"].view(n_ad * r, -1).to(F64).t().contiguous()
    u = (u.view(-1, n_ad, r) * mine[..., None]).to(I64)
    h = (_ilog2(u.abs().amax((1, 2)).clamp(min=1)) - 12).clamp(min=0)
    w = _rshift_round(u, h[:, None, None]).view(-1, n_ad * r).to(F64)
    v = (w @ st["b8"].transpose(1, 2).reshape(n_ad * r, -1).to(F64)).to(I64)
    a = st["adapter"].clamp(min=0).long()
    v = v * st["bm"][a]
    s = (st["bk"][a] - h)[:, None]
    return (y + _rshift_round(v << (-s).clamp(min=0), s.clamp(min=0))).to(I32)


# ------------------------------------------------------------------ one pass

@functools.lru_cache(maxsize=None)
def _ops():
    from idempotent_llm_amd import torch_ops  # noqa: F401  (registers the operators)
    return torch.ops.detllm_rocm


def run(state):
    kind = state["kind"]
    if kind == "plan":
        # the table and the free list are changed in place: this pass's own copy
        book, n = state["book"].clone(), state["B"] * state["width"]
        table, free, n_free = book[:n].view(-1, state["width"]), book[n:-1], book[-1:]
        if own:
            got = _ops().packed_plan(table, free, n_free, state["past"], state["new"], state["N"],
                                     state["err"])
        else:
            got = _plain_plan(state, table, free, n_free)
        return dict(zip(("cu", "row", "pos", "slot"), got), table=table, free=free, n_free=n_free)
    if not own:
        return {"epilogue": _plain_epilogue, "attn": _plain_attn, "lora": _plain_lora}[kind](state)
    if kind == "epilogue":
        names = ("q_m", "q_k", "k_m", "k_k", "v_m", "v_k", "q_norm_m", "q_norm_k", "k_norm_m",
                 "k_norm_k", "qs_m", "qs_k", "kq_m", "kq_k", "ks_m", "ks_k", "vq_m", "vq_k", "cos",
                 "sin", "kp", "vp", "err")
        q8, tpos = _ops().qkv_epilogue_packed(state["P"], state["n_q"], state["n_kv"], state["xm"],
                                              state["xk"], state["pos"], state["slot"],
                                              *(state[n] for n in names))
        return dict(q8=q8, tpos=tpos, k=state["kp"], v=state["vp"])
    if kind == "attn":
        return _ops().attn_packed(state["q8"], state["tpos"], state["kp"], state["vp"],
                                  state["table"], state["cu"], state["past"], state["S"],
                                  state["max_new"], state["err"])
    return _ops().lora_gemm(state["x8"], state["w"], state["a8"], state["b8"], state["bm"],
                            state["bk"], state["adapter"])


# ------------------------------------------------------------------ the work of a pass

def work(case):
    kind = case["kind"]
    if kind == "plan":
        rows = _rows(case)
        pages = sum(-(-(p + n) // PAGE) for p, n in rows)
        return dict(bytes=12 * len(rows) + 20 * case["N"] + 4 * pages, flops=0)
    if kind == "lora":
        N, K, C, r = case["N"], case["K"], case["C"], case["rank"]
        ads = min(case["n_ad"], case["runs"])
        return dict(bytes=N * K + C * K + ads * (r * (K + C) + 8 * C) + 4 * N * C,
                    flops=2 * N * (K * C + r * (K + C)))
    n_q, n_kv = case["n_q"], case["n_kv"]
    if kind == "epilogue":
        N = case["N"]
        return dict(bytes=N * (4 * case["parts"] * (n_q + 2 * n_kv) * HD + 32 + n_q * (HD + 8)
                               + 2 * n_kv * HD + 4 * HD)
                    + 8 * HD * (n_q + 5 * n_kv + 2), flops=0)
    rows = _rows(case)
    N, slots = sum(n for _, n in rows), sum(p + n for p, n in rows)
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in rows)
    return dict(bytes=slots * n_kv * 2 * HD + N * n_q * (HD + 8 + 8 * HD), flops=4 * HD * n_q * pairs)


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return _exact_plan(case, prepare(case, seed))
    if kind == "epilogue":
        if case["N"] * (case["n_q"] + 2 * case["n_kv"]) > 70_000:
            return None
        return _exact_epilogue(case, prepare(case, seed))
    if kind == "lora":
        return _exact_lora(prepare(case, seed))
    if case["n_q"] * sum(n * (p + n) for p, n in _rows(case)) > 120_000_000:
        return None
    return _exact_attn(prepare(case, seed))


def _exact_plan(case, st):
    rows, width, N = _rows(case), case["width"], case["N"]
    book = st["book"].tolist()
    table = [book[b * width:(b + 1) * width] for b in range(len(rows))]
    free, n = book[len(rows) * width:-1], book[-1]
    have = [(t + [-1]).index(-1) for t in table]
    need = [-(-(p + k) // PAGE) for p, k in rows]
    for t, h, q in zip(table, have, need):
        for j in range(q, h):
            free[n], t[j] = t[j], -1
            n += 1
    lack = [(b, j) for b in range(len(rows)) for j in range(have[b], need[b])]
    if len(lack) <= n:
        for b, j in lack:
            n -= 1
            table[b][j] = free[n]
    cu, row, pos, slot = [0], [-1] * N, [0] * N, [-1] * N
    for b, (p, k) in enumerate(rows):
        for t in range(k):
            i, s = cu[-1] + t, p + t
            row[i], pos[i] = b, s
            if table[b][s // PAGE] >= 0:
                slot[i] = table[b][s // PAGE] * PAGE + s % PAGE
        cu.append(cu[-1] + k)
    t32, t64 = (lambda x: torch.tensor(x, dtype=I32)), (lambda x: torch.tensor(x, dtype=I64))
    return dict(cu=t32(cu), row=t32(row), pos=t64(pos), slot=t64(slot), table=t32(table),
                free=t32(free), n_free=t32([n]))


def _bits(x):
    """The bit length of non-negative int64, by halving."""
    x, n = x.clone(), torch.zeros_like(x)
    for s in (32, 16, 8, 4, 2, 1):
        big = x >= (1 << s)
        n += torch.where(big, s, 0)
        x = torch.where(big, x >> s, x)
    return n + (x > 0).long()


def _near(a, b):
    """Quotients rounded to the nearest integer, halves away from zero."""
    q = torch.div(2 * a.abs() + b, 2 * b, rounding_mode="floor")
    return torch.where(a < 0, -q, q)


def _half_up(x, s):
    two = torch.bitwise_left_shift(torch.ones_like(s), s)
    return torch.div(x + torch.div(two, 2, rounding_mode="floor"), two, rounding_mode="floor")


def _exact_qk(x, m, gamma, cos, sin):
    x = x * m.view(-1, HD)
    x = _half_up(x, (_bits(x.abs().amax(-1, keepdim=True)) - 16).clamp(min=0))
    x = x * (1 << (26 - _bits(x.abs().amax(-1, keepdim=True)).clamp(min=1)))
    mean = _near((x * x).sum(-1, keepdim=True), torch.tensor(HD))
    root = torch.zeros_like(mean)
    for bit in range(31, -1, -1):
        try_ = root + (1 << bit)
        root = torch.where(try_ * try_ <= mean, try_, root)
    # (the runtime adds floor(b / 2) to the magnitude: for odd b that is the nearest as well)
    x = _near(x * (1 << 20), root.clamp(min=1)) * gamma
    lo, hi = x[..., :HD // 2], x[..., HD // 2:]
    a = lo * cos[..., :HD // 2] - hi * sin[..., :HD // 2]
    b = hi * cos[..., HD // 2:] + lo * sin[..., HD // 2:]
    return torch.div(torch.cat([a, b], dim=-1) + 8192, 16384, rounding_mode="floor")


def _exact_16(m, k):
    """A positive m as a 16-bit mantissa (halves up), value m / 2^k kept."""
    d = _bits(m) - 16
    m = torch.where(d > 0, _half_up(m, d.clamp(min=0)), m * (1 << (-d).clamp(min=0)))
    carry = m == 1 << 16
    return torch.where(carry, 1 << 15, m), k - d - carry.long()


def _exact_epilogue(case, s):
    s = {k: v.cpu() if torch.is_tensor(v) else v for k, v in s.items()}
    N, n_q, n_kv = case["N"], case["n_q"], case["n_kv"]
    G = n_q // n_kv
    P = s["P"].long().sum(0).view(N, -1, HD)
    cos, sin = s["cos"].long()[s["pos"]][:, None], s["sin"].long()[s["pos"]][:, None]
    q = _exact_qk(P[:, :n_q], s["q_m"], s["q_norm_m"], cos, sin)
    q = (q.view(N, n_kv, G, HD) * s["qs_m"].view(n_kv, 1, HD)).view(N, n_q, HD)
    top = q.abs().amax(-1).clamp(min=1)
    q8 = _near(q * 127, top[..., None])
    # the row's scale top / 127 at 20 + norm + smoothing bits as 16 bits by 2^-e
    num, k0 = top * (1 << 15), 15 + 20 + s["q_norm_k"] + s["qs_k"]
    e = 15 - (_bits(num) - 7)
    m = _near(num * (1 << e.clamp(min=0)), 127 * (1 << (-e).clamp(min=0)))
    short = m < 1 << 15
    e = e + short.long()
    m = torch.where(short, _near(num * (1 << e.clamp(min=0)), 127 * (1 << (-e).clamp(min=0))), m)
    m, e = _exact_16(m, e)
    m, k = _exact_16(m.view(N, n_kv, G) * s["ks_m"].view(n_kv, 1),
                     (k0 + e).view(N, n_kv, G) + s["ks_k"].view(n_kv, 1))
    f = m + torch.div(m, 2, rounding_mode="floor") - torch.div(m, 16, rounding_mode="floor")
    tpos = _near(1 << k, f).clamp(min=1).view(N, n_q)
    kk = _exact_qk(P[:, n_q:n_q + n_kv], s["k_m"], s["k_norm_m"], cos, sin)
    sh = (20 + s["k_norm_k"] - s["kq_k"]).view(n_kv, HD)
    k8 = _near(kk * (1 << (-sh).clamp(min=0)), s["kq_m"].view(n_kv, HD) * (1 << sh.clamp(min=0)))
    v = P[:, n_q + n_kv:] * s["v_m"].view(n_kv, HD) * s["xm"].view(N, 1, 1)
    sh = s["xk"].view(N, 1, 1) + s["v_k"] - s["vq_k"].view(n_kv, 1)
    v8 = _near(v * (1 << (-sh).clamp(min=0)), s["vq_m"].view(n_kv, 1) * (1 << sh.clamp(min=0)))
    for i, at in enumerate(s["slot"].tolist()):
        s["kp"][at // PAGE, :, at % PAGE] = k8[i].clamp(-128, 127).to(I8)
        s["vp"][at // PAGE, :, :, at % PAGE] = v8[i].clamp(-128, 127).to(I8)
    return dict(q8=q8.clamp(-128, 127).to(I8), tpos=tpos, k=s["kp"], v=s["vp"])


def _exact_attn(s):
    q8, tpos, kp, vp, tb = (s[n].cpu() for n in ("q8", "tpos", "kp", "vp", "table"))
    n_q, G, at = s["n_q"], s["n_q"] // s["n_kv"], 0
    out = torch.zeros(q8.shape[0], n_q * HD, dtype=I64)
    for b, (past, new) in enumerate(s["lens"]):
        S = past + new
        ids = tb[b, :-(-S // PAGE)].long()
        hidden = torch.arange(S)[None] > past + torch.arange(new)[:, None]
        for h in range(n_q):
            k = kp[ids, h // G].reshape(-1, HD)[:S].double()
            v = vp[ids, h // G].transpose(1, 2).reshape(-1, HD)[:S].double()
            sc = (q8[at:at + new, h].double() @ k.t()).long()
            n = sc.masked_fill(hidden, -(1 << 40)).amax(1, keepdim=True) - sc
            t = tpos[at:at + new, h, None]
            u = torch.div(n, t, rounding_mode="floor")
            e = (t - torch.div(n - u * t + 1, 2, rounding_mode="floor")) >> u.clamp(0, 62)
            e = e.masked_fill(hidden, 0)
            den = e.sum(1, keepdim=True).clamp(min=1)
            p = torch.div(e * 16384 + torch.div(den, 2, rounding_mode="floor"), den,
                          rounding_mode="floor")
            out[at:at + new, h * HD:(h + 1) * HD] = (p.double() @ v).long()
        at += new
    return out


def _exact_lora(s):
    s = {k: v.cpu() if torch.is_tensor(v) else v for k, v in s.items()}
    y = (s["x8"].double() @ s["w"].double().t()).long()
    for a in range(s["n_ad"]):
        i = (s["adapter"] == a).nonzero()[:, 0]
        if not len(i):
            continue
        u = (s["x8"][i].double() @ s["a8"][a].double().t()).long()
        h = (_bits(u.abs().amax(1)) - 13).clamp(min=0)
        w = _half_up(u, h[:, None].expand_as(u))
        v = (w.double() @ s["b8"][a].double().t()).long() * s["bm"][a]
        sh = (int(s["bk"][a]) - h)[:, None].expand_as(v)
        y[i] += torch.where(sh >= 0, _half_up(v, sh.clamp(min=0)), v * (1 << (-sh).clamp(min=0)))
    return y.to(I32)
