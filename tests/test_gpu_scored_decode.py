"""The decode under a score rule (cap, distance bias, window, first key) and the weights it gives, against float64."""

import numpy as np
import pytest
import torch

import cases
import scored_util as su

pytestmark = pytest.mark.gpu

RULES = {
    "plain": {},
    "cap": {"cap": 5.0},
    "slopes": {"slopes": True},
    "window": {"window": 37},
    "begin": {"begin": True},
    "all": {"cap": 8.0, "slopes": True, "window": 300, "begin": True},
}


def make(seed, ctx, Hq=8, Hkv=2, D=128, act="bf16", kv=None, spread=2.0, **kw):
    c = cases.make_case(seed, len(ctx), Hq, Hkv, D, ctx, act=act, kv=kv, **kw)
    c.q = cases.encode(cases.decode(c.q, c.act) * np.float32(spread), c.act)
    c.rng = np.random.default_rng(seed + 1)
    return c


def rule_of(c, cap=0.0, slopes=False, window=0, begin=False):
    """The rule's arguments for the library and for the reference."""
    sl = (2.0 ** (-8.0 * (np.arange(c.Hq) + 1) / c.Hq)).astype(np.float32) if slopes else None
    bg = np.array([c.rng.integers(-3, max(1, int(n) + 3)) for n in c.ctx], np.int32) if begin else None
    return {"cap": cap, "slopes": sl, "window": window, "begin": bg}


def call(ff, c, d, r, **kw):
    kp, vp, ks, vs, bt, cx, kn, vn, q = d
    up = lambda a: None if a is None else torch.from_numpy(a).to(q.device)  # noqa: E731
    return ff.paged_attention_scored(q, kp, vp, bt, cx, score_cap=r["cap"], slopes=up(r["slopes"]), window=r["window"],
                                     key_begin=up(r["begin"]), k_scale=ks, v_scale=vs, **kw)


def expected(c, r, bound=None, kf=None, vf=None):
    """Per row: out, its bound, weights, their bound."""
    kf = su.values(c, "k") if kf is None else kf
    vf = su.values(c, "v") if vf is None else vf
    q = cases.decode(c.q, c.act).astype(np.float64)
    got = []
    for b in range(c.B):
        pos = int(c.ctx[b])
        n = min(max(pos + 1, 0), c.max_blocks * 16, bound or 1 << 30)
        k, v, absent = su.row(c, b, n, kf, vf)
        bg = None if r["begin"] is None else r["begin"][b:b + 1]
        got.append(su.attention(q[b], k, v, pos, r["cap"], r["slopes"], r["window"], bg, absent=absent, act=c.act, kv=c.kv))
    return got


def check_out(c, out, want):
    out = su.host(out).reshape(c.B, c.Hq, c.D)
    for b, (o, e, _, _) in enumerate(want):
        su.check(out[b], o[0], e[0], f"row {b}")


CONFIGS = [  # act, kv, heads, kv heads, head_dim
    ("bf16", "bf16", 8, 2, 128), ("f16", "f16", 6, 6, 64), ("bf16", "i8", 7, 1, 128), ("bf16", "fp8", 8, 1, 128),
    ("f32", "f32", 8, 4, 128), ("bf16", "bf16", 34, 2, 128), ("bf16", "bf16", 4, 2, 80), ("f16", "f16", 4, 1, 96),
    ("bf16", "i8", 4, 2, 96), ("bf16", "bf16", 5, 1, 112), ("bf16", "bf16", 4, 2, 256), ("f16", "i8", 4, 1, 256),
    ("f32", "f32", 3, 1, 72), ("bf16", "bf16", 8, 1, 40), ("f16", "fp8", 16, 1, 8), ("f32", "f32", 4, 4, 256),
    ("f32", "bf16", 4, 2, 64), ("f32", "f32", 2, 2, 64), ("f16", "i8", 4, 4, 64), ("bf16", "fp8", 6, 3, 112),
]
CTX = [0, 1, 15, 16, 17, 63, 200, 513, 900]


@pytest.mark.parametrize("rule", list(RULES))
@pytest.mark.parametrize("act,kv,Hq,Hkv,D", CONFIGS)
def test_rules(ff, gpu, act, kv, Hq, Hkv, D, rule):
    c = make(3, CTX, Hq, Hkv, D, act, kv)
    r = rule_of(c, **RULES[rule])
    check_out(c, call(ff, c, su.device(c, gpu), r), expected(c, r))


@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [CONFIGS[i] for i in (0, 1, 2, 3, 4, 5, 10, 12, 15)])
@pytest.mark.parametrize("rule", ["plain", "window", "all"])
@pytest.mark.parametrize("ctx", [CTX, [5], [4000, 2, 6001], [30] * 70])
def test_weights(ff, gpu, act, kv, Hq, Hkv, D, rule, ctx):
    """One launch, the split with and without a merge, many rows; prior of its own, in place, none."""
    c = make(5, ctx, Hq, Hkv, D, act, kv)
    r = rule_of(c, **RULES[rule])
    d, want = su.device(c, gpu), expected(c, r)
    T = max(c.ctx) + 1
    prior = torch.rand(c.B, Hkv, T, device=gpu)
    for how in ("own", "none", "in place"):
        w = torch.full_like(prior, 7.0) if how != "in place" else prior.clone()
        out = call(ff, c, d, r, weights=w, prior={"own": prior, "none": None, "in place": w}[how], decay=0.75,
                   max_context_len=int(T))
        check_out(c, out, want)
        got = su.host(w)
        for b, (_, _, x, e) in enumerate(want):
            n = int(c.ctx[b]) + 1
            before = su.host(prior)[b, :, :n - 1] * (0.0 if how == "none" else 0.75)
            x = x + np.pad(before, ((0, 0), (0, 1)))
            su.check(got[b, :, :n], x, e + 2.0 ** -23 * x, f"weights, row {b}, {how}")
            left = prior if how == "in place" else torch.full_like(prior, 7.0)
            assert np.array_equal(got[b, :, n:], su.host(left)[b, :, n:]), "tokens past the row's end are left alone"


@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [CONFIGS[i] for i in (0, 1, 2, 3, 4, 6, 7, 8, 10, 13)])
@pytest.mark.parametrize("rule", ["window", "all"])
def test_hidden_places(ff, gpu, act, kv, Hq, Hkv, D, rule):
    """NaN and infinities in keys and values that no query sees: before the window, past the row's end."""
    ctx = [3, 40, 77, 500, 1200]
    c = make(7, ctx, Hq, Hkv, D, act, kv)
    r = rule_of(c, **RULES[rule])
    want = expected(c, r)
    for b, n in enumerate(ctx):
        lo = max(0 if r["begin"] is None else int(r["begin"][b]), n + 1 - r["window"], 0)
        for t in list(range(min(lo, n + 1))) + list(range(n + 1, c.max_blocks * 16)):
            su.poison(c, b, t)
    w = torch.zeros(c.B, Hkv, max(ctx) + 1, device=gpu)
    out = call(ff, c, su.device(c, gpu), r, weights=w, max_context_len=max(ctx) + 1)
    check_out(c, out, want)
    for b, (_, _, x, e) in enumerate(want):
        su.check(su.host(w)[b, :, :ctx[b] + 1], x, e, f"weights, row {b}")


@pytest.mark.parametrize("kv,D", [("bf16", 128), ("f32", 128), ("i8", 64), ("bf16", 72)])
def test_rows_without_keys(ff, gpu, kv, D):
    """A row of no tokens, one whose first key lies past its end, one whose pages are absent: zeros; their tokens get no
    weight, and earlier weights still decay."""
    c = make(9, [-1, 50, 33, 20, 40], 4, 2, D, "f32" if kv == "f32" else "bf16", kv)
    r = rule_of(c)
    r["begin"] = np.array([0, 51, 0, 1000, 33], np.int32)
    c.block_table[2, :3] = [-1, c.num_blocks, -5]
    c.block_table[4, 1] = -1
    d = su.device(c, gpu)
    prior = torch.rand(5, 2, 64, device=gpu)
    w = torch.full_like(prior, 9.0)
    out = call(ff, c, d, r, weights=w, prior=prior, decay=0.5, max_context_len=64)
    check_out(c, out, expected(c, r))
    got, before = su.host(w), su.host(prior)
    assert np.array_equal(su.host(out)[:4], np.zeros((4, 1, 4 * D)))
    assert (got[0] == 9.0).all()
    for b, n in ((1, 50), (2, 33), (3, 20)):
        assert np.array_equal(got[b, :, :n], before[b, :, :n] * 0.5)
        assert (got[b, :, n] == 0).all() and (got[b, :, n + 1:] == 9.0).all()


@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [CONFIGS[i] for i in (0, 1, 2, 3, 4, 13)])
@pytest.mark.parametrize("ctx", [[0, 31, 16, 700], [2000, 9, 3000]])
def test_append(ff, gpu, act, kv, Hq, Hkv, D, ctx):
    """k_new / v_new: the pages are append_kv_cache's bit for bit (also of a row that does not attend its own token), and
    the output is that of the call on them."""
    c = make(11, ctx, Hq, Hkv, D, act, kv)
    r = rule_of(c, **RULES["all"])
    r["begin"][1] = ctx[1] + 5
    a, b = su.device(c, gpu), su.device(c, gpu)
    ff.append_kv_cache(a[6], a[7], a[0], a[1], a[4], a[5], a[2], a[3])
    want = call(ff, c, a, r)
    got = call(ff, c, b, r, k_new=b[6], v_new=b[7])
    for x, y in zip(a[:4], b[:4]):
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert torch.equal(want, got)


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("most", [1, 100, 131])
def test_max_context_len(ff, gpu, kv, most):
    """Rows are cut at max_context_len; their queries stay where they are."""
    c = make(13, [300, 130, 131, 50], 4, 2, 128, "f32" if kv == "f32" else "bf16", kv)
    r = rule_of(c, cap=6.0, slopes=True, window=250)
    w = torch.full((4, 2, most), 5.0, device=gpu)
    out = call(ff, c, su.device(c, gpu), r, max_context_len=most, weights=w)
    want = expected(c, r, most)
    check_out(c, out, want)
    for b, (_, _, x, e) in enumerate(want):
        su.check(su.host(w)[b, :, :x.shape[1]], x, e, f"weights, row {b}")


def test_scores_past_the_cap(ff, gpu):
    """Scores far past the cap, infinite ones among them, weigh as the cap does."""
    c = make(15, [100, 700], 4, 2, 128)
    c.q = cases.encode(cases.decode(c.q, c.act) * np.float32(1e3), c.act)
    r = rule_of(c, cap=3.0)
    check_out(c, call(ff, c, su.device(c, gpu), r), expected(c, r))
    c.q = cases.encode(np.full(c.q.shape, 1e30, np.float32), c.act)
    c.k_pool = cases.encode(np.sign(cases.decode(c.k_pool, c.kv)) * np.float32(1e30), c.kv)
    c.k_pool[...] = c.k_pool[..., :1]  # every product has the key's sign
    out = su.host(call(ff, c, su.device(c, gpu), r)).reshape(2, 4, 128)
    kf, vf = cases.decode(c.k_pool, c.kv), su.values(c, "v")
    for b in range(2):
        k, v, _ = su.row(c, b, int(c.ctx[b]) + 1, kf, vf)
        for h in range(4):
            p = np.exp(3.0 * np.sign(k[:, h // 2, 0]))
            o = p @ v[:, h // 2] / p.sum()
            assert np.abs(out[b, h] - o).max() <= 2.0 ** -8 * np.abs(o).max() + 1e-4


@pytest.mark.parametrize("kv", ["bf16", "i8", "f32"])
def test_smallest_cap(ff, gpu, kv):
    """A cap of next to nothing leaves all keys the same weight."""
    c = make(21, [100, 700], 4, 2, 128, "f32" if kv == "f32" else "bf16", kv)
    for cap in (1e-44, 1e-38, 1e-20):
        r = rule_of(c, cap=cap)
        check_out(c, call(ff, c, su.device(c, gpu), r), expected(c, dict(r, cap=1e-20)))


def test_streams_graph_and_workspace(ff, gpu):
    """A captured step replays to the same as an eager one, with eager calls in between; a workspace and a stream of the
    caller's give the same bits."""
    c = make(17, [1500, 40, 260], 8, 2, 128)
    r = rule_of(c, **RULES["all"])
    d = su.device(c, gpu)
    T = 1600
    w = torch.zeros(3, 2, T, device=gpu)
    want = call(ff, c, d, r, weights=w, max_context_len=T)
    ws = ff.decode_scored_workspace(3, 8, 128, c.max_blocks, T, weights=True, device=gpu)
    w2, out = torch.zeros_like(w), torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(ff, c, d, r, weights=w2, max_context_len=T, workspace=ws, out=out)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(w, w2)
    rule = {"score_cap": r["cap"], "slopes": torch.from_numpy(r["slopes"]).to(gpu), "window": r["window"],
            "key_begin": torch.from_numpy(r["begin"]).to(gpu)}
    kp, vp, _, _, bt, cx, _, _, q = d
    g = torch.cuda.CUDAGraph()
    w3, out3 = torch.zeros_like(w), torch.empty_like(want)
    with torch.cuda.graph(g):
        ff.paged_attention_scored(q, kp, vp, bt, cx, weights=w3, prior=w3, out=out3, workspace=ws, max_context_len=T, **rule)
    total = torch.zeros_like(w)
    for _ in range(3):
        out3.zero_()
        g.replay()
        torch.cuda.synchronize()
        ff.paged_attention_scored(q, kp, vp, bt, cx, weights=total, prior=total, out=out, workspace=ws, max_context_len=T, **rule)
        torch.cuda.synchronize()
        assert torch.equal(out3, want) and torch.equal(out, want) and torch.equal(w3, total)


def test_long_row(ff, gpu):
    """A row past 2^16 tokens, few and many visible, and its weights."""
    c = make(19, [70000], 8, 1, 64, "f16", "i8")
    for kw in ({"slopes": True}, {"window": 20000, "cap": 4.0}):
        r = rule_of(c, **kw)
        w = torch.zeros(1, 1, 70001, device=gpu)
        out = call(ff, c, su.device(c, gpu), r, weights=w, max_context_len=70001)
        want = expected(c, r)
        check_out(c, out, want)
        su.check(su.host(w)[0], want[0][2], want[0][3], "weights")


@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [("f32", "f32", 16, 2, 128), ("bf16", "bf16", 8, 2, 72), ("f16", "i8", 16, 1, 40),
                                             ("f32", "f32", 4, 2, 64), ("bf16", "bf16", 8, 2, 128)])
@pytest.mark.parametrize("window", [0, 50])
def test_no_pages(ff, gpu, act, kv, Hq, Hkv, D, window):
    """num_blocks 0: no key is on a page, so the rows' outputs are zeros and their weights the earlier ones decayed, whatever
    the workspace held."""
    c = make(31, [300, 5000, 0], Hq, Hkv, D, act, kv)
    T = 16 * c.max_blocks
    prior, w = torch.rand(3, Hkv, T, device=gpu), torch.full((3, Hkv, T), -7.0, device=gpu)
    ws = ff.decode_scored_workspace(3, Hq, D, c.max_blocks, weights=True, device=gpu).fill_(0x7f)
    out = call(ff, c, su.device(c, gpu), rule_of(c, window=window), weights=w, prior=prior, decay=0.5, workspace=ws, num_blocks=0)
    assert not out.float().any()
    for b, n in enumerate([300, 5000, 0]):
        assert torch.equal(w[b, :, :n], 0.5 * prior[b, :, :n])
        assert not w[b, :, n].any() and (w[b, :, n + 1:] == -7.0).all()
