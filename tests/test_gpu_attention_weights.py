"""The attention weights of the last tokens of every row, against float64."""

import numpy as np
import pytest
import torch

import cases
import oracle as O
import scored_util as su
from test_gpu_scored_prefill import RULES, make, masked, rule_of

pytestmark = pytest.mark.gpu


def call(ff, c, d, r, **kw):
    up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(d[8].device)  # noqa: E731
    return ff.attention_weights(d[8], d[0], d[4], d[5], score_cap=r["cap"], slopes=up(r["slopes"]), window=r["window"],
                                key_begin=up(r["begin"]), key_end=up(r["end"]), k_scale=d[2], **kw)


def expected(c, r, most=None):
    kf, q = su.values(c, "k"), cases.decode(c.q, c.act).astype(np.float64)
    got = []
    for b in range(c.B):
        pos = int(c.ctx[b])
        n = min(max(pos + c.S, 0), c.max_blocks * 16, most or 1 << 30)
        k, _, absent = su.row(c, b, n, kf, None)
        rg = [None if r[x] is None else r[x][b].astype(np.int64) for x in ("begin", "end")]
        got.append(su.attention(q[b], k, None, pos, r["cap"], r["slopes"], r["window"], *rg, absent=absent, act=c.act,
                                kv=c.kv)[2:])
    return got


def check(c, w, want, prior=None, decay=0.0, left=None):
    w = su.host(w)
    for b, (x, e) in enumerate(want):
        n = x.shape[1]
        if prior is not None:
            m = max(0, min(int(c.ctx[b]), n))
            x = x.copy()
            x[:, :m] += decay * su.host(prior)[b, :, :m]
        su.check(w[b, :, :n], x, e + 2.0 ** -23 * np.abs(x), f"row {b}")
        if left is not None:
            assert (w[b, :, n:] == left).all()


CONFIGS = [  # act, kv, heads, kv heads, head_dim
    ("bf16", "bf16", 8, 2, 128), ("f16", "f16", 6, 6, 64), ("bf16", "i8", 7, 1, 128), ("bf16", "fp8", 8, 1, 128),
    ("f32", "bf16", 4, 2, 128), ("bf16", "bf16", 4, 2, 256), ("f16", "i8", 4, 1, 64), ("bf16", "fp8", 3, 1, 96),
    ("f16", "f16", 5, 1, 80), ("bf16", "i8", 4, 2, 112), ("f32", "fp8", 20, 1, 256), ("bf16", "bf16", 34, 2, 112),
    ("f32", "f32", 4, 2, 128), ("f32", "f32", 3, 1, 256), ("bf16", "bf16", 5, 1, 72), ("f16", "i8", 2, 2, 40),
    ("bf16", "fp8", 6, 2, 8), ("f16", "f32", 4, 2, 64), ("f32", "i8", 2, 1, 96), ("f16", "f16", 4, 4, 24),
]


@pytest.mark.parametrize("rule", list(RULES))
@pytest.mark.parametrize("act,kv,Hq,Hkv,D", CONFIGS)
def test_rules(ff, gpu, act, kv, Hq, Hkv, D, rule):
    c = make(3, [0, 5, 64, 700], 19, Hq, Hkv, D, act, kv)
    r = rule_of(c, **RULES[rule])
    check(c, call(ff, c, su.device(c, gpu), r), expected(c, r), left=0)


@pytest.mark.parametrize("kind", ["documents", "both ways", "prefix", "some see nothing"])
@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [CONFIGS[i] for i in (0, 1, 2, 3, 5, 12, 14)])
@pytest.mark.parametrize("S", [1, 100])
def test_ranges(ff, gpu, act, kv, Hq, Hkv, D, kind, S):
    c = make(5, [0, 90, 333], S, Hq, Hkv, D, act, kv)
    r = masked(c, rule_of(c, **RULES["all"]), kind)
    check(c, call(ff, c, su.device(c, gpu), r), expected(c, r), left=0)


@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [CONFIGS[i] for i in (0, 2, 4, 5, 11, 12, 15)])
@pytest.mark.parametrize("S,ctx", [(1, [3000, 9]), (64, [2100, 500, 0]), (300, [513])])
def test_prior(ff, gpu, act, kv, Hq, Hkv, D, S, ctx):
    """More query rows than a workgroup stages, several chunks of keys; prior apart, in place, none; what lies past the
    rows is left alone."""
    c = make(7, ctx, S, Hq, Hkv, D, act, kv)
    r = rule_of(c, **RULES["window"])
    d, want = su.device(c, gpu), expected(c, r)
    T = max(ctx) + S + 5
    prior = torch.rand(c.B, Hkv, T, device=gpu) * 0.01
    ws = ff.attention_weights_workspace(c.B, S, Hq, Hkv, D, c.max_blocks, max(ctx) + S, device=gpu)
    for how in ("apart", "in place", "none"):
        w = torch.full_like(prior, 3.0) if how != "in place" else prior.clone()
        got = call(ff, c, d, r, weights=w, prior={"apart": prior, "in place": w, "none": None}[how], decay=0.5,
                   max_context_len=max(ctx) + S, workspace=ws if how == "apart" else None)
        assert got is w
        check(c, w, want, None if how == "none" else prior, 0.5)
        for b in range(c.B):
            n = ctx[b] + S
            assert torch.equal(w[b, :, n:], prior[b, :, n:] if how == "in place" else torch.full_like(w[b, :, n:], 3.0))


@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [CONFIGS[i] for i in (0, 1, 2, 3, 5, 8, 9, 12, 14, 15)])
def test_hidden_places(ff, gpu, act, kv, Hq, Hkv, D):
    """NaN in keys that no query sees, and NaN queries that see nothing (a padded batch): no weight is touched by them.  A NaN
    query that sees keys makes their weights NaN and no others."""
    S, real = 40, [40, 17, 3]
    c = make(9, [300, 700, 100], S, Hq, Hkv, D, act, kv)
    r = rule_of(c, window=120)
    r["end"] = np.array([[n + t + 1 if t < m else 0 for t in range(S)] for n, m in zip(c.ctx, real)], np.int32)
    want = expected(c, r)
    for b, n in enumerate(c.ctx):
        for t in list(range(int(n) + 1 - 120)) + list(range(int(n) + real[b], c.max_blocks * 16)):
            su.poison(c, b, t)
        c.q[b, real[b]:] = su.NAN[c.act]
    check(c, call(ff, c, su.device(c, gpu), r), want, left=0)
    c.q[0, 5, 0] = su.NAN[c.act]
    got = su.host(call(ff, c, su.device(c, gpu), r))
    seen = np.zeros(340, bool)
    seen[300 + 5 + 1 - 120:300 + 6] = True
    assert np.isnan(got[0, 0, :340][seen]).all() and np.isfinite(got[0, 0, :340][~seen]).all()
    assert np.isfinite(got[1:]).all() and (Hkv == 1 or np.isfinite(got[0, 1:]).all())


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_cut_and_absent(ff, gpu, kv):
    c = make(11, [300, 0, 0, 90], 40, 4, 2, 128, kv, kv)
    c.ctx[1:3] = [-20, -60]
    c.block_table[3, 1:3] = [-1, c.num_blocks]
    r = rule_of(c, slopes=True, window=90)
    w = torch.full((4, 2, 310), 5.0, device=gpu)
    check(c, call(ff, c, su.device(c, gpu), r, weights=w, max_context_len=310), expected(c, r, 310), left=5)


@pytest.mark.parametrize("kv,D", [("bf16", 128), ("i8", 112), ("fp8", 64), ("f32", 40)])
def test_no_queries(ff, gpu, kv, D):
    """No tokens: what the rows have decays, whether or not anything earlier is given."""
    c = make(19, [300, 0, 17, -4], 1, 4, 2, D, "f32" if kv == "f32" else "bf16", kv)
    d = list(su.device(c, gpu))
    d[8] = d[8][:, :0]
    r = rule_of(c, **RULES["plain"])
    prior = torch.rand(4, 2, 310, device=gpu)
    for given in (prior, None):
        w = call(ff, c, d, r, weights=torch.full_like(prior, 3.0), prior=given, decay=0.25, max_context_len=310)
        for b, n in enumerate(c.ctx):
            n = max(int(n), 0)
            assert torch.equal(w[b, :, :n], prior[b, :, :n] * 0.25 if given is not None else torch.zeros_like(w[b, :, :n]))
            assert (w[b, :, n:] == 3.0).all()


@pytest.mark.parametrize("D", [64, 112, 128, 256])
def test_large_queries_int8(ff, gpu, D):
    """bf16 queries over int8 keys, far beyond fp16's range, infinite and ordinary ones side by side in two tiles of 16 rows:
    each one's weights are its own.  (Every query has ten keys of its own; beyond the cap any score weighs as the cap, and
    the rows that are too large for a bound on their scores still give every head's weights a sum of 1.)"""
    c = make(21, [200], 16, 2, 1, D, "bf16", "i8")
    q = cases.decode(c.q, c.act)
    q[0, 3] *= np.float32(2.0 ** 20)
    q[0, 4] *= np.float32(2.0 ** -10)
    q[0, 5] *= np.float32(2.0 ** 60)
    c.q = cases.encode(q, c.act)
    r = dict(rule_of(c, cap=6.0), begin=10 * np.arange(16, dtype=np.int32)[None], end=10 * np.arange(1, 17, dtype=np.int32)[None])
    small = r["end"].copy()
    small[0, [3, 5]] = 0
    (want, bound), = expected(c, dict(r, end=small))
    for infinite in (False, True):
        if infinite:
            c.q[0, 6, :, 2] = su.INF[c.act]
        got = su.host(call(ff, c, su.device(c, gpu), r))[0, 0]
        for t in range(16):
            at = slice(10 * t, 10 * t + 10)
            if t in (3, 5):
                assert abs(got[at].sum() - 2) <= 2.0 ** -14
            elif not (infinite and t == 6):
                su.check(got[at], want[0, at], bound[0, at], f"query {t}")
        assert (got[160:] == 0).all()


def test_as_the_decode(ff, gpu):
    """One query per row: the weights of the scored decode."""
    c = make(13, [2000, 3, 450], 1, 8, 2, 128)
    r = rule_of(c, **RULES["all"])
    d = su.device(c, gpu)
    T = 2001
    prior = torch.rand(3, 2, T, device=gpu) * 1e-3
    a, b = torch.zeros_like(prior), torch.zeros_like(prior)
    call(ff, c, d, r, weights=a, prior=prior, max_context_len=T)
    ff.paged_attention_scored(d[8], d[0], d[1], d[4], d[5], score_cap=r["cap"], slopes=torch.from_numpy(r["slopes"]).to(gpu),
                              window=r["window"], weights=b, prior=prior, max_context_len=T)
    want = expected(c, r)
    check(c, a, want, prior, 1.0)
    check(c, b, want, prior, 1.0)


def test_long_row(ff, gpu):
    c = make(15, [70000], 9, 8, 1, 64, "f16", "i8")
    for kw in ({"slopes": True}, {"window": 20000, "cap": 4.0}):
        r = rule_of(c, **kw)
        check(c, call(ff, c, su.device(c, gpu), r), expected(c, r), left=0)


def test_streams_and_graph(ff, gpu):
    c = make(17, [900, 40], 30)
    r = masked(c, rule_of(c, **RULES["all"]), "documents")
    d = su.device(c, gpu)
    want = call(ff, c, d, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    w = torch.zeros_like(want)
    call(ff, c, d, r, weights=w, stream=side)
    side.synchronize()
    assert torch.equal(w, want)
    ws = ff.attention_weights_workspace(2, 30, 8, 2, 128, c.max_blocks, device=gpu)
    begin, sl = torch.from_numpy(r["begin"]).to(gpu), torch.from_numpy(r["slopes"]).to(gpu)
    total, eager = torch.zeros_like(want), torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ff.attention_weights(d[8], d[0], d[4], d[5], total, total, 0.5, r["cap"], sl, r["window"], begin, workspace=ws)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        ff.attention_weights(d[8], d[0], d[4], d[5], eager, eager, 0.5, r["cap"], sl, r["window"], begin, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(total, eager)


@pytest.mark.parametrize("B,Hkv", [(5, 2), (70, 1), (130, 2), (256, 1), (255, 2)])
def test_uneven_rows(ff, gpu, B, Hkv):
    """Rows of very different lengths, empty ones among them, in calls whose rows are cut into pieces and in ones of too many
    rows for that."""
    g = np.random.default_rng(23)
    ctx = [int(x) for x in g.integers(0, 60, B)]
    ctx[B // 2], ctx[-1], ctx[0] = 9000, 2500, -9
    c = make(23, ctx, 3, 2 * Hkv, Hkv, 64, "bf16", "bf16")
    r = rule_of(c, cap=9.0, slopes=True)
    check(c, call(ff, c, su.device(c, gpu), r, max_context_len=9003), expected(c, r, 9003), left=0)


@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [CONFIGS[i] for i in (0, 2, 12)])
def test_few_keys_seen(ff, gpu, act, kv, Hq, Hkv, D):
    """Windows and ranges that leave most of a row out, at its front, its end and whole; earlier weights decay everywhere."""
    c = make(25, [3000, 900, 2600, 5], 70, Hq, Hkv, D, act, kv)
    d = su.device(c, gpu)
    prior = torch.rand(4, Hkv, 3070, device=gpu)
    for kind in ("window", "front", "middle", "none"):
        r = rule_of(c, cap=7.0, window=100 if kind == "window" else 0)
        if kind != "window":
            lo, hi = {"front": (-4, 30), "middle": (700, 1300), "none": (50, 50)}[kind]
            r["begin"], r["end"] = np.full((4, 70), lo, np.int32), np.full((4, 70), hi, np.int32)
            r["end"][2, 3] = lo
        w = call(ff, c, d, r, weights=torch.zeros_like(prior), prior=prior, decay=0.5, max_context_len=3070)
        check(c, w, expected(c, r), prior, 0.5, left=0)


def test_new_weights_on_another_stream(ff, gpu):
    """Without `weights` the new tensor's zeros are written on the call's stream, however busy the current one is."""
    c = make(29, [900, 40], 30)
    r = rule_of(c, cap=5.0)
    d = su.device(c, gpu)
    want = call(ff, c, d, r)
    side = torch.cuda.Stream()
    x = torch.randn(4096, 4096, device=gpu)
    for stream in (side, side.cuda_stream):
        torch.cuda.synchronize()
        for _ in range(40):  # some tens of milliseconds
            x = (x @ x).mul_(1.0 / 64.0)
        w = call(ff, c, d, r, stream=stream)
        side.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(w, want)
