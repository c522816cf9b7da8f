"""Low-rank adapters for packed steps: many requests, each with its own, beside
one set of weights (no counterpart in the reference).

An ``AdapterBank`` holds up to ``n`` adapters for a model. Per layer there are
four sites, one for each product of the layer (q|k|v, o, gate|up, down); an
adapter's modules that share a product are stacked: their A matrices along the
rank, their B matrices as blocks (w's 13 bits then go by the largest of them). ``quantize`` turns float A and B into int8 with
dyadic scales in the product's own units (offline and float, as prepare.py is);
``detllm_lora_add`` adds them in integers.
"""

from __future__ import annotations

import torch

from ._lib import call

I64 = torch.int64
F64 = torch.float64
STEP = 16           # ranks are filled up to multiples of it
MAX_RANK = 128      # of a site
SITES = {"qkv": ("q", "k", "v"), "o": ("o",), "gu": ("gate", "up"), "d": ("down",)}


def quantize(A, B, col_m, col_k: int, in_scale=None, scale: float = 1.0):
    """Float A [r, K], B [C, r] of y += scale B A x as (a8 [r, K], b8 [C, r]
    int8, bm [C] int64, bk): each row of A and of B by its own maximum, A's
    scales folded into B, B's as 16-bit mantissas bm / 2^bk of the product's
    column scales col_m / 2^col_k. in_scale [K]: what one unit of the product's
    int8 input (before its row scale) stands for in x, where the artifact folds
    norm weights and smoothing factors into its own weights."""
    A, B = A.detach().to("cpu", F64), B.detach().to("cpu", F64) * scale
    if A.dim() != 2 or B.dim() != 2 or A.shape[0] != B.shape[1] or B.shape[0] != col_m.numel():
        raise ValueError(f"quantize: A {tuple(A.shape)} and B {tuple(B.shape)} for "
                         f"{col_m.numel()} columns")
    if in_scale is not None:
        A = A * in_scale.detach().to("cpu", F64)[None, :]
    sa = A.abs().amax(dim=1) / 127
    a8 = torch.round(A / torch.where(sa > 0, sa, 1)[:, None]).clamp(-127, 127).to(torch.int8)
    B = B * sa[None, :]
    sb = B.abs().amax(dim=1) / 127
    b8 = torch.round(B / torch.where(sb > 0, sb, 1)[:, None]).clamp(-127, 127).to(torch.int8)
    ratio = sb * 2.0 ** col_k / col_m.detach().to("cpu", F64)
    top = float(ratio.max()) if ratio.numel() else 0.0
    if top <= 0:
        return a8, b8, torch.zeros(col_m.numel(), dtype=I64), 0
    bk = 15 - int(torch.floor(torch.log2(ratio.max())))
    return a8, b8, torch.round(ratio * 2.0 ** bk).to(I64), bk


def in_scales(model, attn_gains, mlp_gains) -> dict:
    """What one unit of each product's int8 input stands for, per channel and
    (layer, site), for adapters trained beside the float model: the artifact's
    inputs are normalised rows without the norms' gains (attn_gains and mlp_gains,
    float, one vector per layer) times the smoothing factors 1 / s; its weights have
    both folded in (prepare.py)."""
    out = {}
    for li, L in enumerate(model.layers):
        s = lambda m, k: 2.0 ** k / m.detach().to("cpu", F64)
        out[li, "qkv"] = s(L.as_m, L.as_k) * attn_gains[li].detach().to("cpu", F64)
        out[li, "o"] = s(L.os_m, L.os_k)
        out[li, "gu"] = s(L.ms_m, L.ms_k) * mlp_gains[li].detach().to("cpu", F64)
        out[li, "d"] = s(L.ds_m, L.ds_k)
    return out


class AdapterBank:
    """``n`` adapters of rank up to ``rank`` per module for ``model``."""

    def __init__(self, model, n: int, rank: int):
        pad = -(-int(rank) // STEP) * STEP
        if n < 1 or rank < 1 or 3 * pad > MAX_RANK:
            raise ValueError(f"AdapterBank: {n} adapters of rank {rank} (at most "
                             f"{MAX_RANK // 3 // STEP * STEP})")
        self.n, self.rank, self.pad, self.device = n, int(rank), pad, model.device
        self.n_layers = model.n_layers
        self.cols, self.depth = self._sizes(model)
        self.scales = [{m: (getattr(L, f"{m}_m"), getattr(L, f"{m}_k")) for m in self.cols}
                       for L in model.layers]
        dev = self.device
        self.sites = []      # per layer: site -> (a8, b8, bm, bk)
        for _ in range(model.n_layers):
            self.sites.append({
                s: (torch.zeros(n, pad * len(ms), self.depth[s], dtype=torch.int8, device=dev),
                    torch.zeros(n, sum(self.cols[m] for m in ms), pad * len(ms), dtype=torch.int8,
                                device=dev),
                    torch.zeros(n, sum(self.cols[m] for m in ms), dtype=I64, device=dev),
                    torch.zeros(n, dtype=I64, device=dev))
                for s, ms in SITES.items()})

    @staticmethod
    def _sizes(model):
        nq, nkv, hd, H, I = model.n_q, model.n_kv, model.hd, model.hidden, model.inter
        return ({"q": nq * hd, "k": nkv * hd, "v": nkv * hd, "o": H, "gate": I, "up": I, "down": H},
                {"qkv": H, "o": nq * hd, "gu": H, "d": I})

    def check_model(self, model) -> None:
        """ValueError for a model of other layers or sizes."""
        if (model.n_layers, *self._sizes(model)) != (self.n_layers, self.cols, self.depth) \
                or model.device != self.device:
            raise ValueError("adapters of a model of other sizes, or on another device")

    def set(self, i: int, weights: dict, scale: float = 1.0, in_scales: dict | None = None) -> None:
        """Adapter i from float weights {(layer, module): (A, B)}, module one of q,
        k, v, o, gate, up, down; modules that are not there add nothing.
        in_scales {(layer, site): in_scale} as quantize takes it (in_scales())."""
        if not 0 <= i < self.n:
            raise ValueError(f"adapter {i} of a bank of {self.n}")
        known = {(li, m) for li in range(self.n_layers) for m in self.cols}
        if set(weights) - known:
            raise ValueError(f"no such module: {sorted(set(weights) - known)[0]}")
        # (all modules before anything is written: one that is refused leaves the
        # adapter as it was)
        made = {}       # (layer, site): its exponent, [(place, first column, module, ...)]
        for li in range(self.n_layers):
            for s, ms in SITES.items():
                parts, at = [], 0
                for j, m in enumerate(ms):
                    if (li, m) in weights:
                        A, B = weights[li, m]
                        if A.shape[0] > self.rank or A.shape[1] != self.depth[s]:
                            raise ValueError(f"{m} of layer {li}: A {tuple(A.shape)} for rank "
                                             f"{self.rank} and {self.depth[s]} inputs")
                        cm, ck = self.scales[li][m]
                        sc = None if in_scales is None else in_scales.get((li, s))
                        parts.append((j, at, m, *quantize(A, B, cm, ck, sc, scale)))
                    at += self.cols[m]
                # one exponent per site: the smallest, so that no mantissa passes 16 bits
                made[li, s] = min((p[-1] for p in parts if int(p[-2].max()) > 0), default=0), parts
        for (li, s), (k, parts) in made.items():
            a8, b8, bm, bk = self.sites[li][s]
            for t in (a8, b8, bm):
                t[i].zero_()
            bk[i] = k
            for j, c, m, qa, qb, qm, qk in parts:
                r = qa.shape[0]
                a8[i, j * self.pad:j * self.pad + r] = qa.to(self.device)
                b8[i, c:c + self.cols[m], j * self.pad:j * self.pad + r] = qb.to(self.device)
                down = min(max(0, qk - k), 62)      # (62: nothing of 17 bits is left)
                qm = (qm + (1 << (down - 1)) >> down) if down else qm
                bm[i, c:c + self.cols[m]] = qm.to(self.device)

    def add(self, li: int, site: str, P, x8, adapter) -> None:
        """The adapters' part of layer li's product P ([.., N, C], its first
        partial) of x8 [N, K], in place; adapter [N] int32."""
        a8, b8, bm, bk = self.sites[li][site]
        N, K = x8.shape
        call("detllm_lora_add", P, x8, a8, b8, bm, bk, adapter, N, K, b8.shape[1], a8.shape[1],
             self.n)
