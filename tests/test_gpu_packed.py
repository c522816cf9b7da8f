"""GPU checks of the packed-step operators (page bookkeeping, slot-mapped Q/K/V
epilogue, attention of ragged rows, low-rank adapters per token row) against
64-bit loops over the CPU oracle (packedcases.py). Everything is integer
arithmetic: exact equality."""

import numpy as np
import pytest
import torch

import packedcases as pc
from packedcases import PAGE

pytestmark = pytest.mark.gpu
I8, I32, I64 = torch.int8, torch.int32, torch.int64


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from idempotent_llm_amd import _lib, torch_ops  # noqa: F401
    _lib.load()


def _ops():
    return torch.ops.detllm_rocm


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _err():
    return torch.zeros(1, dtype=I32, device="cuda")


def _eq(got, want):
    got = got.cpu().numpy()
    assert got.dtype == want.dtype and got.shape == want.shape
    assert np.array_equal(got, want), np.argwhere(got != want)[:4].tolist()


# --------------------------------------------------------------- attention

ORDER = ("q8", "tpos", "kpool", "vpool", "table", "cu", "past")


def _attend(c, S=None, max_new=None):
    err = _err()
    out = _ops().attn_packed(*(_cuda(c[k]) for k in ORDER), c["S"] if S is None else S,
                             c["max_new"] if max_new is None else max_new, err)
    return out, int(err)


def _spread(n, hi, seed, lo=0):
    return np.random.default_rng(seed).integers(lo, hi, n).tolist()


# past, new, n_q, n_kv, extras of packedcases.make
ATTENTION = {
    "first_token": ([0], [1], 2, 1, {}),
    "second_token": ([1], [1], 2, 2, {}),
    "lengths": ([0, 1, 62, 63, 64, 126, 127, 128, 129, 255, 256], [1] * 11, 4, 2, {}),
    "idle_rows": ([5, 200, 0, 300, 77], [0, 1, 0, 0, 1], 4, 2, {}),
    "all_idle": ([5, 200], [0, 0], 4, 2, dict(tail=3)),
    "tail": ([5, 200, 17], [1, 2, 0], 4, 2, dict(tail=150)),
    "group_1": ([3, 500, 130], [16, 1, 7], 3, 3, {}),
    "group_2": ([3, 500, 130], [8, 1, 7], 4, 2, {}),
    "group_4": ([3, 500, 130], [4, 1, 2], 8, 2, {}),
    "group_8": ([3, 500, 130], [2, 1, 2], 16, 2, {}),
    "group_8_one": ([3, 500, 130, 513], [1, 1, 1, 1], 8, 1, {}),
    "few_1024": ([700, 1000, 40], [3, 4, 1], 4, 2, {}),
    "few_2048": ([2000, 1023, 0], [3, 4, 8], 4, 2, {}),
    "few_2048_edge": ([2044], [4], 2, 1, {}),
    "few_2049": ([2048, 0, 511, 512], [1, 1, 1, 1], 2, 1, {}),
    "few_chunks": ([6000, 10, 2300, 0, 512], [1, 1, 0, 1, 1], 4, 2, dict(tail=2)),
    "few_chunks_16": ([5000, 10, 2300], [8, 3, 8], 4, 2, {}),
    "seventeen_rows": ([40, 100], [17, 1], 2, 2, {}),
    "prompt_3": ([0], [3], 8, 1, {}),
    "prompt_63": ([0], [63], 2, 2, {}),
    "prompt_64": ([0, 0], [64, 65], 2, 2, {}),
    "prompt_page": ([0, 64], [128, 128], 2, 1, {}),
    "prompt_300": ([0], [300], 4, 2, {}),
    "chunk_behind": ([211, 0, 77], [120, 9, 33], 8, 1, {}),
    "mixed": ([130, 900, 0, 333, 512], [1, 30, 200, 0, 2], 4, 2, dict(tail=9)),
    "mixed_few_long": ([1500, 0], [2, 40], 2, 1, {}),
    "mixed_chunks": ([3000, 0, 4001, 700], [70, 130, 1, 0], 4, 2, dict(tail=5)),
    "mixed_chunks_group_8": ([1300, 2000], [20, 2], 8, 1, {}),
    "few_one_launch_2048": ([2047, 1500, 3, 900], [1, 1, 1, 1], 32, 32, {}),
    "prompt_behind_one_launch": ([400, 3], [300, 1], 8, 8, {}),
    "prompts_one_launch": ([700, 0, 1300, 90], [300, 260, 200, 1], 8, 8, {}),
    "mixed_one_launch": (_spread(60, 900, 1), [1] * 55 + [40, 30, 20, 90, 0], 8, 8, {}),
    "many_rows": (_spread(300, 400, 2), _spread(300, 3, 3), 2, 1, {}),
    "many_rows_idle": (_spread(200, 300, 4), [0] * 130 + [1] + [0] * 60 + [25] + [0] * 8, 2, 1, {}),
    "many_rows_chunks": (_spread(150, 3000, 5), _spread(150, 2, 6), 1, 1, {}),
    "constants_1": ([300, 5, 40], [1, 40, 3], 4, 2, dict(tpos=(8, 17))),
    "constants_border": ([300, 5, 40], [1, 40, 3], 4, 2, dict(tpos=(32, 34))),
    "constants_wide": ([300, 5, 40], [1, 40, 3], 4, 2, dict(tpos=(33, 62))),
    "constants_wide_few": ([1200, 5, 40], [2, 1, 3], 4, 2, dict(tpos=(30, 62))),
    "constants_wide_chunks": ([3000, 5], [1, 1], 2, 1, dict(tpos=(30, 62))),
    "constants_wide_mixed_chunks": ([1900, 5], [70, 1], 2, 1, dict(tpos=(30, 62))),
    "extreme": ([300, 0, 2500], [3, 70, 1], 4, 2, dict(extreme=True, flat=True)),
    "extreme_few": ([2500, 100], [3, 1], 4, 2, dict(extreme=True, flat=True, tpos=(8, 62))),
    "wide_table": ([100, 300], [1, 50], 2, 1, dict(width=700)),
    "holes_few": ([700, 20, 300], [1, 1, 2], 4, 2,
                  dict(holes=((0, 2, -1), (1, 0, -1), (2, 0, 99), (2, 1, -7)))),
    "holes_all": ([127], [1], 2, 1, dict(holes=((0, 0, 2**31 - 1),))),
    "holes_chunks": ([3000, 2600], [1, 1], 2, 1,
                     dict(holes=tuple((1, j, -1) for j in range(21)) + ((0, 4, -1), (0, 7, 60)))),
    "holes_tiles": ([0, 100], [300, 90], 2, 1, dict(holes=((0, 0, -1), (1, 1, -2**31)))),
    "holes_tiles_chunks": ([900, 2000], [80, 50], 2, 1,
                           dict(holes=tuple((1, j, -1) for j in range(17)) + ((0, 0, 50),))),
}


@pytest.mark.parametrize("name", list(ATTENTION))
def test_attention(name):
    print(f"[attention {name}]", flush=True)
    past, new, n_q, n_kv, extra = ATTENTION[name]
    c = pc.make(past, new, n_q, n_kv, seed=len(name), **extra)
    out, err = _attend(c)
    assert err == 0
    _eq(out, pc.attend(c))


def test_attention_of_the_longest_rows():
    """131071 slots: one token at the last of them, and a prompt's last chunk."""
    print("[attention 131071]", flush=True)
    for past, new in ((131070, 1), (131071 - 40, 40)):
        c = pc.make([past, 3], [new, 1], 2, 1, seed=new, extreme=True)
        out, err = _attend(c)
        assert err == 0
        _eq(out, pc.attend(c))


def test_attention_wider_bounds():
    """S and max_new are bounds: wider ones give the same (other chunks, other
    launches)."""
    print("[attention bounds]", flush=True)
    for past, new in (([100, 300, 40], [1, 2, 1]), ([100, 300, 40], [30, 2, 70])):
        c = pc.make(past, new, 4, 2, seed=5, width=80)
        want = pc.attend(c)
        for S in (c["S"], 513, 1025, 2049, 10240):
            for max_new in (c["max_new"], 9, 200, 2**31 - 1):
                if max_new >= c["max_new"]:
                    out, err = _attend(c, S, max_new)
                    assert err == 0
                    _eq(out, want)


def test_attention_past_its_bounds():
    """Rows of more slots than S, or more tokens than max_new, set bit 4; the
    slots that a row has within S are seen, other rows are computed."""
    print("[attention past its bounds]", flush=True)
    for past, new in (([100, 300, 40], [1, 2, 1]), ([100, 300, 40], [30, 2, 70]),
                      ([2900, 2300], [1, 2]), ([900, 700], [40, 1])):
        c = pc.make(past, new, 4, 2, seed=6)
        for S in (1, 130, int(c["S"]) - 1):
            out, err = _attend(c, S)
            assert err == 4
            _eq(out, pc.attend(c, S))
    c = pc.make([100, 300, 40], [30, 2, 1], 4, 2, seed=7)
    out, err = _attend(c, max_new=10)
    assert err == 4
    want = pc.attend(c)
    _eq(out[:10], want[:10])
    _eq(out[30:], want[30:])
    out, err = _attend(c, max_new=0)
    assert err == 4


@pytest.mark.parametrize("cu", [[0, 10, 0, 10, 0, 10], [40, 40, 40, 40, 40, 40],
                                [-5, 3, 2, 1, 0, 60], [0, 90, 90, 90, -1, 2**31 - 1],
                                [0, 40, 0, 40, 0, 40], [9, 8, 7, 6, 5, 4]])
@pytest.mark.parametrize("S,n_kv", [(300, 2), (700, 2), (700, 8), (3000, 1)])
def test_attention_offsets_that_do_not_ascend(cu, S, n_kv):
    """Token offsets that overlap, decrease or leave the rows: nothing is read or
    written out of range (what out holds is not specified), and a good call
    behind it is right."""
    print(f"[attention offsets {cu} {S} {n_kv}]", flush=True)
    c = pc.make([5, 70, 290, 0, 130], [8] * 5, 8, n_kv, seed=8, width=24)
    want = pc.attend(c)
    for max_new in (1, 8, 40):
        _attend(dict(c, cu=np.array(cu, np.int32)), S, max_new)
    out, err = _attend(c, S)
    assert err == 0
    _eq(out, want)


def test_attention_far_pages():
    """Pages past 4 GiB of a pool."""
    print("[attention far pages]", flush=True)
    c = pc.make([300, 200, 3000], [1, 20, 1], 8, 8, seed=9)
    n = len(c["kpool"])
    far = 40000                                    # 5.2 GB a pool
    kp = torch.empty(far, 8, 128, 128, dtype=I8, device="cuda")
    vp = torch.empty_like(kp)
    kp[far - n:], vp[far - n:] = _cuda(c["kpool"]), _cuda(c["vpool"])
    table = _cuda(np.where(c["table"] >= 0, c["table"] + far - n, -1).astype(np.int32))
    want = pc.attend(c)
    for S, max_new in ((c["S"], 20), (c["S"], 400)):
        err = _err()
        out = _ops().attn_packed(_cuda(c["q8"]), _cuda(c["tpos"]), kp, vp, table, _cuda(c["cu"]),
                                 _cuda(c["past"]), S, max_new, err)
        assert int(err) == 0
        _eq(out, want)


def test_attention_strided_operands():
    print("[attention strided]", flush=True)
    c = pc.make([300, 20], [1, 30], 4, 2, seed=10)
    want = pc.attend(c)
    args = [_cuda(c[k]) for k in ORDER]
    N = args[0].shape[0]
    wide = torch.zeros(N, 4, 256, dtype=I8, device="cuda")
    wide[..., 100:228] = args[0]
    odd = torch.zeros(args[0].numel() + 1, dtype=I8, device="cuda")[1:].view(args[0].shape)
    odd.copy_(args[0])
    for q8 in (wide[..., 100:228], odd):
        for tpos in (args[1], args[1].t().contiguous().t()):
            _eq(_ops().attn_packed(q8, tpos, *args[2:], c["S"], 30, _err()), want)


def test_attention_no_token_rows():
    c = pc.make([3], [0], 2, 1, seed=1)
    out, err = _attend(c)
    assert out.shape == (0, 256) and err == 0


# ------------------------------------------------------------- bookkeeping

def _plan(state, past, new, N):
    """One call on the device state, checked against the loops."""
    table, free, n_free, err = state
    before = [t.cpu().numpy() for t in (table, free)] + [int(n_free)]
    err.zero_()
    got = _ops().packed_plan(table, free, n_free, _cuda(np.asarray(past, np.int32)),
                             _cuda(np.asarray(new, np.int32)), N, err)
    want = pc.plan(*before, past, new, N)
    n = want[2]
    _eq(table, want[0])
    assert int(n_free) == n
    _eq(free[:n], want[1][:n])
    for g, w in zip(got, want[3:7]):
        _eq(g, w)
    assert int(err) == want[7]
    return want[7]


def _state(B, width, pages, seed):
    free = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    return (torch.full((B, width), -1, dtype=I32, device="cuda"), _cuda(free),
            torch.tensor([pages], dtype=I32, device="cuda"), _err())


@pytest.mark.parametrize("B,width,cap,top", [(1, 1, 1, 128), (1, 20, 20, 600), (3, 4, 12, 200),
                                             (7, 16, 60, 900), (64, 9, 400, 200), (65, 5, 300, 60),
                                             (1025, 3, 2500, 9), (2048, 2, 4096, 4)])
def test_plan_steps(B, width, cap, top):
    """Steps of rows that start, grow, idle, shrink and leave; some steps ask for
    more pages than there are, which changes nothing but what is given back."""
    print(f"[plan {B} {width} {cap}]", flush=True)
    rng = np.random.default_rng(B)
    st = _state(B, width, cap, B)
    past = np.zeros(B, np.int32)
    seen = 0
    for step in range(12):
        new = rng.integers(0, top + 1, B).astype(np.int32) * (rng.random(B) < 0.6)
        new = np.minimum(new, width * PAGE - past).astype(np.int32)
        N = int(new.sum()) + int(rng.integers(0, 5))
        err = _plan(st, past, new, N)
        seen |= err
        if err == 0:
            past = (past + new).astype(np.int32)
        past = np.where(rng.random(B) < 0.25, rng.integers(0, past + 1), past).astype(np.int32)
        past = np.where(rng.random(B) < 0.1, 0, past).astype(np.int32)
    _plan(st, np.zeros(B, np.int32), np.zeros(B, np.int32), 0)    # everything comes back
    assert int(st[2]) == cap and sorted(st[1].tolist()) == list(range(cap))
    assert seen in (0, 8)


@pytest.mark.parametrize("N", [2047, 2048, 2049, 20000])
def test_plan_many_tokens(N):
    """Token rows of one launch and of two, some behind the last row's."""
    print(f"[plan N={N}]", flush=True)
    st = _state(6, 100, 400, N)
    new = [N // 2, 0, 1, N // 3, 7, 0]
    assert _plan(st, [0] * 6, new, N) == 0
    assert _plan(st, new, [1, 128, 0, 1, 5, 300], N) == 0


def test_plan_widest_table():
    print("[plan width 1024]", flush=True)
    st = _state(2, 1024, 2048, 1)
    assert _plan(st, [0, 0], [131071, 5], 131076) == 0
    assert _plan(st, [131071, 5], [0, 131000], 131000) == 0
    assert _plan(st, [131071, 131005], [1, 0], 1) == 4      # 131072 slots: refused
    assert _plan(st, [4000, 64], [3, 64], 67) == 0


def test_plan_refused_rows():
    """Negative counts and rows past the table keep their pages and have no
    tokens; too few token rows are reported, the others are written."""
    print("[plan refused rows]", flush=True)
    st = _state(4, 5, 20, 2)
    assert _plan(st, [0] * 4, [200, 1, 300, 128], 629) == 0
    for past, new in (([200, 1, -1, 128], [1, 1, 1, 1]), ([200, 1, 300, 128], [1, -1, 1, 1]),
                      ([200, 640, 300, 128], [1, 1, 1, 1]),
                      ([200, 2**31 - 1, 300, 128], [1, 2**31 - 1, 1, 1]),
                      ([-2**31, 1, 300, 128], [-2**31, 1, 1, 1])):
        assert _plan(st, past, new, 4) == 4
    assert _plan(st, [201, 2, 301, 129], [5, 5, 5, 5], 12) == 4
    assert _plan(st, [201, 2, 301, 129], [0] * 4, 0) == 0


def test_plan_out_of_pages():
    """None of the missing pages is taken; rows whose pages are there have slots,
    and surplus pages come back all the same."""
    print("[plan out of pages]", flush=True)
    st = _state(3, 8, 6, 3)
    assert _plan(st, [0] * 3, [300, 200, 100], 600) == 0
    assert _plan(st, [300, 200, 100], [1, 0, 100], 101) == 8
    assert _plan(st, [100, 200, 100], [1, 0, 100], 101) == 0
    assert _plan(st, [101, 200, 200], [700, 0, 1], 701) == 8


# ---------------------------------------------------------------- epilogue

EPI = ("q_m", "q_k", "k_m", "k_k", "v_m", "v_k", "q_norm_m", "q_norm_k", "k_norm_m", "k_norm_k",
       "qs_m", "qs_k", "kq_m", "kq_k", "ks_m", "ks_k", "vq_m", "vq_k", "cos", "sin")


def _slots(kind, N, pages, rng):
    if kind == "random":
        return rng.permutation(pages * PAGE)[:N]
    if kind == "runs":        # runs of consecutive slots that start anywhere
        s, at = [], 0
        while len(s) < N:
            at += int(rng.integers(0, 7))
            n = int(rng.integers(1, 12))
            s += list(range(at, at + n))
            at += n
        return np.array(s[:N])
    s = np.arange(N)          # one run, some token rows without a slot
    s[::5] = -1
    if N > 3:
        s[1], s[2], s[3] = pages * PAGE, 2**62, -2**62
    return s


@pytest.mark.parametrize("variant", ["none", "ranges", "gamma"])
@pytest.mark.parametrize("N,kind,nsplit", [(1, "random", 1), (5, "random", 3), (8, "gaps", 2),
                                           (64, "runs", 2), (65, "random", 1), (130, "gaps", 1),
                                           (300, "runs", 2), (301, "one", 1)])
def test_epilogue(variant, N, kind, nsplit):
    from idempotent_llm_amd import artifact as art
    from test_gpu_attention import _layer_params, _plant, _qkv_oracle
    print(f"[epilogue {variant} N={N} {kind}]", flush=True)
    dims = art.MID
    nq, nkv = dims["n_q_heads"], dims["n_kv_heads"]
    prm = _plant(_layer_params(dims, 6), variant, nq, nkv)
    rng = np.random.default_rng(N)
    P = rng.integers(-(1 << 19), 1 << 19, (1, N, (nq + 2 * nkv) * 128), dtype=np.int32)
    P[0, 0, :128] = 0                          # a zero head
    P[0, N - 1, nq * 128:(nq + 1) * 128] = 0
    P = _cuda(P)
    xm = rng.integers(1 << 15, 1 << 16, N, dtype=np.int64)
    xm[N // 2] = (1 << 40) + 7                 # V numerators of this row wrap
    xm, xk = _cuda(xm), _cuda(rng.integers(22, 30, N, dtype=np.int64))
    pos = _cuda(rng.integers(0, dims["max_pos"], N, dtype=np.int64))
    want_q8, want_tpos, want_k, want_v, _ = _qkv_oracle(P, xm, xk, pos, prm, N, 1, nq, nkv)
    pages = 9
    slots = _slots(kind, N, pages, rng).astype(np.int64)
    if kind == "one":
        slots = np.arange(77, 77 + N)
    k0 = rng.integers(-128, 128, (pages, nkv, PAGE, 128), dtype=np.int8)
    v0 = rng.integers(-128, 128, (pages, nkv, 128, PAGE), dtype=np.int8)
    kp, vp, err = _cuda(k0), _cuda(v0), _err()
    parts = torch.cat([P - 1000 * (nsplit - 1)] + [torch.full_like(P, 1000)] * (nsplit - 1))
    q8, tpos = _ops().qkv_epilogue_packed(parts, nq, nkv, xm, xk, pos, _cuda(slots),
                                          *(prm[k] for k in EPI), kp, vp, err)
    assert int(err) == 0
    _eq(q8, want_q8[:, :, 0])
    _eq(tpos, want_tpos[:, :, 0])
    for i, s in enumerate(slots):
        if 0 <= s < pages * PAGE:
            k0[s // PAGE, :, s % PAGE] = want_k[i, :, 0]
            v0[s // PAGE, :, :, s % PAGE] = want_v[i, :, 0]
    _eq(kp, k0)
    _eq(vp, v0)


def test_epilogue_reports_positions():
    from idempotent_llm_amd import artifact as art
    from test_gpu_attention import _layer_params
    print("[epilogue positions]", flush=True)
    dims = art.MID
    nq, nkv = dims["n_q_heads"], dims["n_kv_heads"]
    prm = _layer_params(dims, 6)
    for N in (3, 100):
        one = torch.ones(N, dtype=I64, device="cuda")
        P = torch.ones(1, N, (nq + 2 * nkv) * 128, dtype=I32, device="cuda")
        kp = torch.zeros(2, nkv, 128, 128, dtype=I8, device="cuda")
        for at, want in ((dims["max_pos"] - 1, 0), (dims["max_pos"], 2), (2**40, 2)):
            pos, err = one.clone(), _err()
            pos[N // 2] = at
            _ops().qkv_epilogue_packed(P, nq, nkv, one, 25 * one, pos,
                                       torch.arange(N, device="cuda"), *(prm[k] for k in EPI), kp,
                                       kp.clone(), err)
            assert int(err) == want


# ---------------------------------------------------------------- adapters

def _lora_case(N, K, C, rank, n_ad, seed, kind="mixed", wide=False):
    rng = np.random.default_rng(seed)
    i8 = lambda *s: rng.integers(-128, 128, s, dtype=np.int8)
    x8, w, a8, b8 = i8(N, K), i8(C, K), i8(n_ad, rank, K), i8(n_ad, C, rank)
    hi = 62 if wide else 16
    bm = rng.integers(-(1 << hi), 1 << hi, (n_ad, C), dtype=np.int64)
    bk = rng.integers(-40 if wide else 14, 70 if wide else 30, n_ad, dtype=np.int64)
    if kind == "mixed":
        ad = rng.integers(-1, n_ad, N)
    elif kind == "one":
        ad = np.full(N, n_ad - 1)
    elif kind == "none":
        ad = np.full(N, -1)
    else:                      # ids that name no adapter
        ad = rng.choice([-1, -2**31, 2**31 - 1, n_ad, 0], N)
    x8[0] = 0                  # u = 0
    if N > 2:
        x8[1], a8[0, 0] = -128, -128
    return x8, w, a8, b8, bm, bk, ad.astype(np.int32)


@pytest.mark.parametrize("N,K,C,rank,n_ad,kind", [
    (1, 16, 1, 16, 1, "one"), (1, 1024, 300, 16, 4, "one"), (2, 64, 17, 32, 2, "mixed"),
    (7, 1040, 255, 48, 5, "mixed"), (8, 2048, 1000, 64, 8, "mixed"), (16, 512, 256, 80, 3, "one"),
    (17, 512, 257, 96, 3, "mixed"), (33, 1024, 4096, 112, 40, "mixed"),
    (64, 208, 700, 128, 64, "mixed"), (65, 1024, 513, 16, 2, "ids"), (130, 768, 2049, 16, 3, "one"),
    (300, 1024, 4100, 32, 6, "mixed"), (700, 256, 9000, 16, 4, "one"), (5, 128, 40, 16, 2, "none"),
    (100, 128, 40, 16, 2, "none")])
@pytest.mark.parametrize("wide", [False, True])
def test_lora(N, K, C, rank, n_ad, kind, wide):
    print(f"[lora {N} {K} {C} {rank} {n_ad} {kind}]", flush=True)
    c = _lora_case(N, K, C, rank, n_ad, N + K, kind, wide)
    P = (c[0].astype(np.int64) @ c[1].astype(np.int64).T).astype(np.int32)
    _eq(_ops().lora_gemm(*(_cuda(t) for t in c)), pc.lora(P, c[0], *c[2:]))


def test_lora_deepest():
    """K 65536 of the largest bytes: u reaches 2^30."""
    print("[lora K 65536]", flush=True)
    c = list(_lora_case(3, 65536, 40, 16, 2, 1, "one"))
    c[0][1:], c[2][:] = -128, -128
    P = (c[0].astype(np.int64) @ c[1].astype(np.int64).T).astype(np.int32)
    _eq(_ops().lora_gemm(*(_cuda(t) for t in c)), pc.lora(P, c[0], *c[2:]))


def test_lora_strided_and_empty():
    print("[lora strided]", flush=True)
    c = _lora_case(20, 256, 100, 16, 3, 4)
    P = (c[0].astype(np.int64) @ c[1].astype(np.int64).T).astype(np.int32)
    want = pc.lora(P, c[0], *c[2:])
    d = [_cuda(t) for t in c]
    odd = torch.zeros(20, 300, dtype=I8, device="cuda")[:, 3:259]
    odd.copy_(d[0])
    cols = d[3].transpose(1, 2).contiguous().transpose(1, 2)
    _eq(_ops().lora_gemm(odd, d[1].t().contiguous().t(), d[2], cols, *d[4:]), want)
    assert _ops().lora_gemm(d[0][:0], *d[1:6], d[6][:0]).shape == (0, 100)


# ---------------------------------------------------------------- together

def _step_inputs(m, N, seed):
    """A layer's product and scales for N token rows."""
    rng = np.random.default_rng(seed)
    P = rng.integers(-(1 << 19), 1 << 19, (1, N, (m["n_q"] + 2 * m["n_kv"]) * 128), dtype=np.int32)
    return (_cuda(P), _cuda(rng.integers(1 << 15, 1 << 16, N, dtype=np.int64)),
            _cuda(rng.integers(22, 30, N, dtype=np.int64)))


def _run(m, st, cu_args, P, xm, xk, pools, new, past, S, most, err):
    ops, N = _ops(), P.shape[1]
    cu, row, pos, slot = ops.packed_plan(*st[:3], past, new, N, err)
    q8, tpos = ops.qkv_epilogue_packed(P, m["n_q"], m["n_kv"], xm, xk, pos, slot, *cu_args, *pools,
                                       err)
    out = ops.attn_packed(q8, tpos, *pools, st[0], cu, past, S, most, err)
    return out, q8, tpos, cu, row


def _together(seed=0):
    from idempotent_llm_amd import artifact as art
    from test_gpu_attention import _layer_params
    dims = art.MID
    m = dict(n_q=dims["n_q_heads"], n_kv=dims["n_kv_heads"])
    prm = _layer_params(dims, seed)
    for k in ("cos", "sin"):      # positions to 4096
        prm[k] = torch.cat([prm[k], prm[k]])
    return m, [prm[k] for k in EPI]


def _whole(m, epi, P, xm, xk, slots):
    """The prefill operators on one row of a cache of its own: contexts."""
    T, w = P.shape[1], -(-slots // PAGE)
    kp = torch.zeros(w, m["n_kv"], 128, 128, dtype=I8, device="cuda")
    vp, err = torch.zeros_like(kp), _err()
    table = torch.arange(w, dtype=I32, device="cuda")[None]
    q8, tpos = _ops().qkv_epilogue(P, 1, T, m["n_q"], m["n_kv"], xm, xk,
                                   torch.arange(T, device="cuda"), *epi, kp, vp, table, 0, err)
    valid = torch.ones(1, w * PAGE, dtype=torch.bool, device="cuda")
    out = _ops().attn_prefill(q8, tpos, kp, vp, table, valid, 0)
    return out.reshape(T, -1)


def test_steps_together():
    """Three requests, their prompts fed in chunks of other sizes beside each other
    and then token by token: each token's context is the one of the request
    alone, its prompt in one piece."""
    print("[steps together]", flush=True)
    m, epi = _together()
    lens = (150, 40, 300)
    data = [_step_inputs(m, n, 20 + n) for n in lens]
    want = [_whole(m, epi, *d, n) for d, n in zip(data, lens)]
    steps = ([100, 0, 7], [40, 0, 1], [1, 33, 250], [1, 1, 1], [8, 6, 41])
    st = _state(3, 4, 8, 5)
    pools = [torch.randint(-128, 128, (8, m["n_kv"], 128, 128), dtype=I8, device="cuda")
             for _ in range(2)]
    past, err = np.zeros(3, np.int32), _err()
    for new in steps:
        cut = lambda k: torch.cat([d[k][..., p:p + n, :] if k == 0 else d[k][p:p + n]
                                   for d, p, n in zip(data, past, new)], dim=1 if k == 0 else 0)
        S = int(max(past + new))
        out, *_ = _run(m, st, epi, cut(0), cut(1), cut(2), pools, _cuda(np.array(new, np.int32)),
                       _cuda(past), S, max(new), err)
        want_step = torch.cat([w[p:p + n] for w, p, n in zip(want, past, new)])
        assert torch.equal(out, want_step) and int(err) == 0
        past = (past + np.array(new)).astype(np.int32)
    assert past.tolist() == list(lens)


@pytest.mark.parametrize("lens,news", [((130, 40, 300), (1, 1, 1)), ((2900, 40, 2500), (1, 2, 1)),
                                       ((900, 70, 0), (40, 1, 100))])
def test_captured_step(lens, news):
    """plan, epilogue, attention and an adapter captured into a graph, two graphs
    alive at once, replayed in turn with eager work and synchronizations between:
    each replay is the eager call's result. The lengths are read at the replay."""
    print(f"[captured step {lens} {news}]", flush=True)
    m, epi = _together()
    N, width, S = sum(news), 26, 26 * PAGE
    P, xm, xk = _step_inputs(m, N, 3)
    lo = [_cuda(t) for t in _lora_case(N, 256, 500, 16, 3, 6)]
    gen = torch.Generator(device="cuda").manual_seed(1)
    pools0 = [torch.randint(-128, 128, (90, m["n_kv"], 128, 128), dtype=I8, device="cuda",
                            generator=gen) for _ in range(2)]
    new = _cuda(np.array(news, np.int32))

    def fresh():
        st = _state(3, width, 90, 7)
        _ops().packed_plan(*st[:3], torch.zeros_like(new), _cuda(np.array(lens, np.int32)), 0,
                           _err())
        return st, [p.clone() for p in pools0], _cuda(np.array(lens, np.int32))

    def go(st, pools, past, err):
        out = _run(m, st, epi, P, xm, xk, pools, new, past, S, max(news), err)[0]
        past += new
        return out, _ops().lora_gemm(*lo)

    def eager(n):
        st, pools, past = fresh()
        res = []
        err = _err()
        for _ in range(n):
            out, y = go(st, pools, past, err)
            res.append((out.clone(), y.clone()))
        assert int(err) == 0
        return res, st, pools

    want, st_w, pools_w = eager(4)
    graphs = []
    for _ in range(2):
        st, pools, past = fresh()
        err = _err()
        keep = [t.clone() for t in (*st[:3], past)], [p.clone() for p in pools]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            go(st, pools, past, err)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        for t, k in zip((*st[:3], past), keep[0]):
            t.copy_(k)
        for t, k in zip(pools, keep[1]):
            t.copy_(k)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = go(st, pools, past, err)
        graphs.append((g, out, st, pools, past, err))
    for i in range(4):
        for g, out, st, pools, past, err in graphs:
            g.replay()
            torch.cuda.synchronize()
            eager(1)
            assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])
    for g, out, st, pools, past, err in graphs:
        assert int(err) == 0
        assert all(torch.equal(a, b) for a, b in zip(pools, pools_w))
        assert torch.equal(st[0], st_w[0]) and int(st[2]) == int(st_w[2])


def test_opcheck():
    """The fakes agree with the kernels, and only what is declared changes."""
    print("[opcheck]", flush=True)
    tests = ("test_schema", "test_faketensor")
    check = lambda op, *args: torch.library.opcheck(op.default, args, test_utils=tests)
    m, epi = _together()
    P, xm, xk = _step_inputs(m, 6, 1)
    pools = [torch.zeros(4, m["n_kv"], 128, 128, dtype=I8, device="cuda") for _ in range(2)]
    arange = torch.arange(6, device="cuda")
    check(_ops().qkv_epilogue_packed, P, m["n_q"], m["n_kv"], xm, xk, arange, arange, *epi, *pools,
          _err())
    c = pc.make([300, 20], [1, 30], 4, 2, seed=10)
    check(_ops().attn_packed, *(_cuda(c[k]) for k in ORDER), c["S"], 30, _err())
    st = _state(2, 3, 6, 1)
    check(_ops().packed_plan, *st[:3], _cuda(np.array([0, 0], np.int32)),
          _cuda(np.array([200, 3], np.int32)), 205, _err())
    check(_ops().lora_gemm, *(_cuda(t) for t in _lora_case(5, 64, 30, 16, 2, 1)))


def test_side_stream():
    """Two calls at once on streams of their own."""
    print("[side streams]", flush=True)
    cases = [pc.make([3000, 5], [1, 1], 4, 2, seed=1), pc.make([900, 5], [60, 1], 4, 2, seed=2)]
    args = [[_cuda(c[k]) for k in ORDER] for c in cases]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in cases], []
    for _ in range(3):
        for c, a, s in zip(cases, args, streams):
            with torch.cuda.stream(s):
                outs.append((_ops().attn_packed(*a, c["S"], c["max_new"], _err()),
                             c))
    torch.cuda.synchronize()
    wants = [pc.attend(c) for c in cases]
    for i, (out, _) in enumerate(outs):
        _eq(out, wants[i % 2])


@pytest.mark.parametrize("new", [[0, 1, 0, 1], [0, 20, 0, 1], [0, 1, 70, 0]])
def test_attention_idle_rows_past_the_bound(new):
    """S bounds the rows that have new tokens: idle rows of more slots are neither
    reported nor read, and the others are exact."""
    print(f"[attention idle rows past the bound {new}]", flush=True)
    c = pc.make([4000, 300, 1500 if new[2] == 0 else 30, 5], new, 4, 2, seed=11)
    busy = [p + n for p, n in zip(c["past"], new) if n]
    out, err = _attend(c, int(max(busy)))
    assert err == 0
    _eq(out, pc.attend(c))


# past, new, n_q, n_kv, whether the call is one launch (no scratch), extras
PATHS = {
    "few_one": ([2047, 1500, 3], [1, 1, 1], 64, 64, True, {}),
    "few_chunks": ([2048, 3], [1, 1], 64, 64, False, {}),
    "short_row_past_512": ([650, 10], [1, 40], 8, 8, True, dict(holes=((0, 3, -1),))),
    "short_rows_past_512": ([700, 513, 690, 511, 0, 30], [1, 2, 1, 1, 0, 40], 8, 8, True, {}),
    "prompts": ([560, 0, 400, 300], [300, 260, 100, 1], 8, 8, True, {}),
    "prompts_group_4": ([300, 0, 37], [90, 120, 1], 16, 4, True, {}),
    "tile_chunks": ([700, 3], [300, 1], 8, 8, False, {}),
    # from 420 tiles on one launch takes any length: rows of more than 64 pages, whose
    # ids a wave holds in two lots, with holes on both sides of the 64th
    "long_rows_beside_many_tiles": (
        [9000, 8300, 0, 100, 0, 0, 5, 0, 2047], [1, 70, 128, 128, 128, 128, 128, 128, 1], 32, 32,
        True, dict(holes=((0, 3, -1), (0, 64, -1), (0, 66, 2**31 - 1), (1, 1, -1), (1, 63, -1),
                          (1, 64, -5)))),
    "long_few_rows_beside_many_tiles": (
        [8191, 8192, 8320, 0, 3], [1, 4, 1, 700, 200], 32, 32, True,
        dict(holes=((1, 64, -1), (2, 0, -1)), tpos=(30, 40))),
}


@pytest.mark.parametrize("name", list(PATHS))
def test_attention_paths(name):
    """Cases of each launch, which the scratch tells apart (a rule that moves them
    elsewhere fails here)."""
    from idempotent_llm_amd import _lib
    print(f"[attention path {name}]", flush=True)
    past, new, n_q, n_kv, one, extra = PATHS[name]
    c = pc.make(past, new, n_q, n_kv, seed=len(name), **extra)
    work = _lib.packed_work(int(sum(new)), len(past), c["S"], c["max_new"], n_q, n_kv)
    assert (work == 0) == one
    out, err = _attend(c)
    assert err == 0
    _eq(out, pc.attend(c))


class _Guarded:
    """Buffers of exact sizes between marks that no launch may change."""
    MARK = 0x5A

    def __init__(self):
        self.made = []

    def __call__(self, shape, dtype):
        n = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
        whole = torch.full((n + 8192 - n % 4096,), self.MARK, dtype=torch.uint8, device="cuda")
        self.made.append((whole, n))
        return whole[2048:2048 + n].view(dtype).view(shape)

    def check(self):
        for whole, n in self.made:
            assert bool((whole[:2048] == self.MARK).all()), "written before a buffer"
            assert bool((whole[2048 + n:] == self.MARK).all()), "written behind a buffer"


def _args(c, work, out, err, S, max_new):
    dev = [_cuda(c[k]) for k in ORDER]
    q8, tpos, kp, vp, table, cu, past = dev
    N, n_q = q8.shape[:2]
    return dev, ["detllm_attn_packed", q8, tpos, kp, vp, kp.shape[0], table, table.shape[1], cu,
                 past, N, past.shape[0], S, max_new, n_q, kp.shape[1], work,
                 work.numel() if work is not None else 0, out, err]


# a call's scratch is used up to its last byte in some of these, the outputs in all
GUARDED = {
    "few": ([300, 20, 5], [1, 2, 0], 4, 2, 321, 2, 0),
    "few_chunks": ([6000, 10, 2300, 0], [1, 1, 1, 1], 4, 2, None, 1, 3),
    "few_chunks_16": ([5000, 10, 2300], [8, 3, 8], 4, 2, None, 8, 0),
    "few_by_token": ([3000, 40, 2999, 0, 7, 1], [8, 1, 1, 0, 1, 1], 4, 2, None, 8, 0),
    "tiles": ([560, 0, 40], [300, 26, 1], 4, 2, None, 300, 2),
    "tile_chunks": ([3000, 0, 4001, 700], [70, 130, 1, 0], 4, 2, None, 130, 5),
    "tile_chunks_8": ([2900, 17], [33, 2], 8, 1, None, 33, 0),
    "tile_chunks_wider": ([900, 40, 5], [40, 1, 1], 4, 2, 10240, 500, 0),
}


def _attend_guarded(c, S, max_new, cus):
    """Calls with each of the offsets; the last is the case's own. -> its contexts."""
    from idempotent_llm_amd import _lib
    buf = _Guarded()
    N, n_q = c["q8"].shape[:2]
    B, n_kv = len(c["past"]), c["kpool"].shape[1]
    work = buf((_lib.packed_work(N, B, S, max_new, n_q, n_kv),), torch.uint8)
    out, err = buf((N, n_q * 128), I64), buf((1,), I32)
    for cu in [*cus, c["cu"]]:
        err.zero_()
        dev, args = _args(dict(c, cu=np.asarray(cu, np.int32)), work, out, err, S, max_new)
        before = [t.clone() for t in dev]
        _lib.call(*args)
        torch.cuda.synchronize()
        buf.check()
        assert all(torch.equal(a, b) for a, b in zip(dev, before)), "an operand changed"
    assert int(err) == 0
    return out


@pytest.mark.parametrize("name", list(GUARDED))
def test_attention_stays_in_its_buffers(name):
    """Scratch of exactly the stated size, outputs and the error word: nothing
    beside them is written, no operand changes, and the size suffices."""
    print(f"[attention buffers {name}]", flush=True)
    past, new, n_q, n_kv, S, max_new, tail = GUARDED[name]
    c = pc.make(past, new, n_q, n_kv, seed=len(name), tail=tail,
                width=80 if S == 10240 else None)
    _eq(_attend_guarded(c, S or c["S"], max_new, ()), pc.attend(c))


@pytest.mark.parametrize("S,n_kv", [(300, 2), (700, 2), (700, 8), (3000, 1)])
@pytest.mark.parametrize("max_new", [1, 8, 40])
def test_attention_of_odd_offsets_stays_in_its_buffers(S, n_kv, max_new):
    """Token offsets that overlap, decrease or leave the rows: the same."""
    print(f"[attention odd offsets {S} {n_kv} {max_new}]", flush=True)
    c = pc.make([5, 70, 290, 0, 130], [8] * 5, 8, n_kv, seed=8, width=24)
    odd = ([0, 10, 0, 10, 0, 10], [40] * 6, [-5, 3, 2, 1, 0, 60], [0, 90, 90, 90, -1, 2**31 - 1],
           [0, 40, 0, 40, 0, 40], [9, 8, 7, 6, 5, 4], [0, 0, 0, 0, 0, 2**31 - 1],
           [-2**31, 2**31 - 1, -2**31, 2**31 - 1, -2**31, 2**31 - 1])
    if max_new < 8:                       # the good call behind them needs its bound
        c = pc.make([5, 70, 290, 0, 130], [1] * 5, 8, n_kv, seed=8, width=24, tail=35)
    _eq(_attend_guarded(c, S, max_new, odd), pc.attend(c))


@pytest.mark.parametrize("N", [5, 700, 2049, 5000])
def test_plan_stays_in_its_buffers(N):
    """A plan's table, free list, outputs and scratch of exact sizes, and fewer token
    rows than tokens."""
    from idempotent_llm_amd import _lib
    print(f"[plan buffers {N}]", flush=True)
    B, width, cap = 5, 30, 120
    buf = _Guarded()
    table, free, n_free = buf((B, width), I32), buf((cap,), I32), buf((1,), I32)
    past, new = _cuda(np.zeros(B, np.int32)), _cuda(np.array([N, 0, 129, 7, 2000], np.int32))
    cu, row, pos, slot = buf((B + 1,), I32), buf((N,), I32), buf((N,), I64), buf((N,), I64)
    work, err = buf(((B + 1) * 16 if N > 2048 else 0,), torch.uint8), buf((1,), I32)
    if N > 3840:
        new[0] = 3840                     # the row's own slots
    table.fill_(-1)
    free.copy_(torch.arange(cap, dtype=I32))
    n_free.fill_(cap)
    err.zero_()
    before = [table.cpu().numpy(), free.cpu().numpy(), cap]
    _lib.call("detllm_packed_plan", table, width, free, cap, n_free, past, new, B, N, cu, row, pos,
              slot, work, work.numel(), err)
    torch.cuda.synchronize()
    buf.check()
    want = pc.plan(*before, past.cpu().numpy(), new.cpu().numpy(), N)
    assert int(n_free) == want[2] and int(err) == want[7]
    for g, w in zip((table, free[:want[2]], cu, row, pos, slot),
                    (want[0], want[1][:want[2]], *want[3:7])):
        _eq(g, w)


@pytest.mark.parametrize("bk", [-70, -64, -63, 0, 61, 62, 63, 64, 65, 70, 77, 116, 2**40])
def test_lora_shifts_of_any_size(bk):
    """Adapters whose scale is far from the product's: a shift that nothing survives
    adds nothing (quantize gives exponents past 64 for very small adapters)."""
    print(f"[lora shift {bk}]", flush=True)
    rng = np.random.default_rng(3)
    N, K, C, rank = 20, 64, 300, 16
    x8, w, a8, b8 = (rng.integers(-128, 128, s, dtype=np.int8)
                     for s in ((N, K), (C, K), (2, rank, K), (2, C, rank)))
    x8[0], b8[:, 5] = 0, 0                     # u = 0, and a column of zeros
    bm = rng.integers(1, 1 << 16, (2, C), dtype=np.int64)
    ad = rng.integers(-1, 2, N).astype(np.int32)
    ad[0] = 0
    P = (x8.astype(np.int64) @ w.astype(np.int64).T).astype(np.int32)
    want = P.astype(np.int64)
    for i in range(N):
        if ad[i] < 0:
            continue
        u = a8[ad[i]].astype(np.int64) @ x8[i].astype(np.int64)
        h = max(max(int(np.abs(u).max()), 1).bit_length() - 13, 0)
        v = b8[ad[i]].astype(np.int64) @ ((u + (1 << h >> 1)) >> h)
        s = bk - h
        for c in range(C):
            t = int(v[c]) * int(bm[ad[i], c])          # below 2^43
            if s >= 64:
                d = 0
            else:
                d = (t + (1 << s >> 1)) >> s if s > 0 else (t << -s if -s < 64 else 0)
            want[i, c] += (d + 2**31) % 2**32 - 2**31
    want = ((want + 2**31) % 2**32 - 2**31).astype(np.int32)
    got = _ops().lora_gemm(*(_cuda(t) for t in (x8, w, a8, b8, bm, np.full(2, bk, np.int64), ad)))
    _eq(got, want)
