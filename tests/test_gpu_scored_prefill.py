"""Prefill attention under a score rule (cap, distance bias, window, ranges of visible keys), against float64."""

import numpy as np
import pytest
import torch

import cases
import oracle as O
import scored_util as su

pytestmark = pytest.mark.gpu

RULES = {
    "plain": {},
    "cap": {"cap": 5.0},
    "slopes": {"slopes": True},
    "window": {"window": 50},
    "cap_window": {"cap": 8.0, "window": 1},
    "all": {"cap": 8.0, "slopes": True, "window": 300},
}


def make(seed, ctx, S, Hq=8, Hkv=2, D=128, act="bf16", kv=None, spread=2.0, **kw):
    c = cases.make_case(seed, len(ctx), Hq, Hkv, D, ctx, act=act, kv=kv, S=S, **kw)
    c.rng = np.random.default_rng(seed + 1)
    c.q = cases.encode(c.rng.standard_normal((c.B, S, Hq, D), dtype=np.float32) * np.float32(spread), c.act)
    return c


def rule_of(c, cap=0.0, slopes=False, window=0):
    sl = (2.0 ** (-8.0 * (np.arange(c.Hq) + 1) / c.Hq)).astype(np.float32) if slopes else None
    return {"cap": cap, "slopes": sl, "window": window, "begin": None, "end": None}


def masked(c, r, kind):
    """r with ranges of visible keys."""
    B, S = c.B, c.S
    begin, end = np.zeros((B, S), np.int32), np.zeros((B, S), np.int32)
    for b in range(B):
        n = int(c.ctx[b])
        cuts = sorted({0, n} | {int(x) for x in c.rng.integers(0, n + S, 4)})
        prefix = int(c.rng.integers(0, n + S + 1))
        for t in range(S):
            i = n + t
            doc = max(x for x in cuts if x <= i)
            nxt = min([x for x in cuts if x > i] + [n + S])
            if kind == "documents":
                begin[b, t], end[b, t] = doc, i + 1
            elif kind == "both ways":
                begin[b, t], end[b, t] = doc, nxt
            elif kind == "prefix":
                begin[b, t], end[b, t] = -5, max(prefix, i + 1)
            elif kind == "some see nothing":
                begin[b, t], end[b, t] = (i + 1, 7) if t % 3 == 0 else (0, 1 << 30) if t % 3 == 1 else (0, i + 1)
    return dict(r, begin=begin if kind != "prefix" else None, end=end if kind != "documents" else None)


def call(ff, c, d, r, **kw):
    kp, vp, ks, vs, bt, cx, _, _, q = d
    up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(q.device)  # noqa: E731
    return ff.paged_prefill_scored(q, kp, vp, bt, cx, score_cap=r["cap"], slopes=up(r["slopes"]), window=r["window"],
                                   key_begin=up(r["begin"]), key_end=up(r["end"]), k_scale=ks, v_scale=vs, **kw)


def expected(c, r, most=None, kf=None, vf=None):
    kf = su.values(c, "k") if kf is None else kf
    vf = su.values(c, "v") if vf is None else vf
    q = cases.decode(c.q, c.act).astype(np.float64)
    got = []
    for b in range(c.B):
        pos = int(c.ctx[b])
        n = min(max(pos + c.S, 0), c.max_blocks * 16, most or 1 << 30)
        k, v, absent = su.row(c, b, n, kf, vf)
        rg = [None if r[x] is None else r[x][b].astype(np.int64) for x in ("begin", "end")]
        got.append(su.attention(q[b], k, v, pos, r["cap"], r["slopes"], r["window"], *rg, absent=absent, act=c.act,
                                kv=c.kv, p_step=2.0 ** -10))
    return got


def check(c, out, want):
    out = su.host(out).reshape(c.B, c.S, c.Hq, c.D)
    for b, (o, e, _, _) in enumerate(want):
        su.check(out[b], o, e, f"row {b}")


CONFIGS = [  # act, kv, heads, kv heads, head_dim
    ("bf16", "bf16", 8, 2, 128), ("f16", "f16", 6, 6, 64), ("bf16", "i8", 7, 1, 128), ("bf16", "fp8", 8, 1, 128),
    ("f32", "bf16", 4, 2, 128), ("bf16", "bf16", 4, 2, 256), ("f16", "i8", 4, 1, 64), ("bf16", "fp8", 3, 1, 64),
    ("f16", "f16", 5, 1, 256), ("f32", "i8", 4, 2, 256), ("f16", "fp8", 20, 1, 256), ("bf16", "bf16", 2, 2, 64),
]
CTX = [0, 5, 64, 700]


@pytest.mark.parametrize("rule", list(RULES))
@pytest.mark.parametrize("act,kv,Hq,Hkv,D", CONFIGS)
def test_rules(ff, gpu, act, kv, Hq, Hkv, D, rule):
    c = make(3, CTX, 45, Hq, Hkv, D, act, kv)
    r = rule_of(c, **RULES[rule])
    check(c, call(ff, c, su.device(c, gpu), r), expected(c, r))


@pytest.mark.parametrize("kind", ["documents", "both ways", "prefix", "some see nothing"])
@pytest.mark.parametrize("rule", ["plain", "all"])
@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [CONFIGS[i] for i in (0, 1, 2, 3, 5, 10)])
def test_ranges(ff, gpu, act, kv, Hq, Hkv, D, rule, kind):
    c = make(5, [0, 90, 333], 150, Hq, Hkv, D, act, kv)
    r = masked(c, rule_of(c, **RULES[rule]), kind)
    check(c, call(ff, c, su.device(c, gpu), r), expected(c, r))


@pytest.mark.parametrize("S", [1, 2, 17, 300])
@pytest.mark.parametrize("kv,kind", [("bf16", "documents"), ("f16", "both ways"), ("bf16", "prefix"), ("f16", "")])
def test_contiguous(ff, gpu, S, kv, kind):
    c = make(7, [0, 0], S, 6, 2, 128, kv, kv)
    r = rule_of(c, cap=7.0, window=120)
    r = masked(c, r, kind) if kind else r
    k, v = (np.stack([su.row(c, b, S, cases.decode(p, c.kv), None)[0] for b in range(2)]) for p in (c.k_pool, c.v_pool))
    d = su.device(c, gpu)
    up = lambda a: torch.from_numpy(a.astype(np.float32)).to(gpu).to(d[0].dtype)  # noqa: E731
    rg = {n: None if r[m] is None else torch.from_numpy(r[m]).to(gpu) for n, m in (("key_begin", "begin"), ("key_end", "end"))}
    out = ff.paged_prefill_scored(d[8], up(k), up(v), None, None, score_cap=7.0, window=120, **rg)
    check(c, out, expected(c, r))


@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [CONFIGS[i] for i in (0, 1, 2, 3, 5, 6, 7, 8, 9)])
@pytest.mark.parametrize("rule", ["window", "all", "padded"])
def test_hidden_places(ff, gpu, act, kv, Hq, Hkv, D, rule):
    """NaN and infinities where no query looks: before every window, past the row's tokens, and in a padded batch at the
    padding's own keys, whose queries see nothing."""
    S, real = 70, [70, 70, 33, 1]
    c = make(9, [3, 400, 128, 60], S, Hq, Hkv, D, act, kv)
    r = rule_of(c, **RULES["window" if rule == "padded" else rule])
    if rule == "padded":
        r["end"] = np.array([[n + t + 1 if t < m else 0 for t in range(S)] for n, m in zip(c.ctx, real)], np.int32)
    want = expected(c, r)
    for b, n in enumerate(c.ctx):
        lo = max(0, int(n) + 1 - r["window"])
        hi = int(n) + (real[b] if rule == "padded" else S)
        for t in list(range(lo)) + list(range(hi, c.max_blocks * 16)):
            su.poison(c, b, t)
    check(c, call(ff, c, su.device(c, gpu), r), want)


@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [CONFIGS[i] for i in (0, 1, 2, 3, 5, 7, 8, 11)])
@pytest.mark.parametrize("value", ["inf", "nan"])
def test_seen_by_some(ff, gpu, act, kv, Hq, Hkv, D, value):
    """A key whose V is infinite or NaN reaches the queries that see it, in its dims, and no other."""
    S = 100
    c = make(11, [0, 250], S, Hq, Hkv, D, act, kv)
    r = dict(masked(c, rule_of(c, cap=6.0), "both ways"), window=40)
    want = expected(c, r)
    key, dims = {0: 55, 1: 290}, [0, 5, D - 1]
    for b, t in key.items():
        page, slot = int(c.block_table[b, t // 16]), t % 16
        if c.kv == O.DTYPE_I8:
            c.v_scale[page, slot] = np.inf if value == "inf" else np.nan
        else:
            c.v_pool[page, slot, :, dims] = su.INF[c.kv] if value == "inf" and c.kv in su.INF else su.NAN[c.kv]
    out = su.host(call(ff, c, su.device(c, gpu), r)).reshape(2, S, Hq, D)
    some = 0
    for b, t in key.items():
        n = int(c.ctx[b])
        for s in range(S):
            lo = max(int(r["begin"][b, s]), n + s + 1 - 40)
            seen = lo <= t < min(int(r["end"][b, s]), n + S)
            some += seen
            o, e = want[b][0][s], want[b][1][s]
            for h in range(Hq):
                if not seen:
                    su.check(out[b, s, h], o[h], e[h], (b, s, h))
                elif c.kv != O.DTYPE_I8:
                    rest = np.delete(np.arange(D), dims)
                    su.check(out[b, s, h, rest], o[h, rest], e[h, rest], (b, s, h))
                    hit = out[b, s, h, dims]
                    assert np.isnan(hit).all() or (value == "inf" and np.isposinf(hit).all()), (b, s, h, hit)
                else:
                    assert not np.isfinite(out[b, s, h]).any()
    assert 0 < some < 2 * S


@pytest.mark.parametrize("act,kv,Hq,Hkv,D", [CONFIGS[i] for i in (0, 1, 2, 3, 5, 9)])
@pytest.mark.parametrize("ctx,S", [([5000], 30), ([3000, 100], 64), ([2500], 1)])
@pytest.mark.parametrize("rule,kind", [("slopes", ""), ("cap", "prefix"), ("all", ""), ("plain", "documents")])
def test_split(ff, gpu, act, kv, Hq, Hkv, D, ctx, S, rule, kind):
    """Few query rows over long contexts, whose keys are split: whole and split calls agree with float64."""
    c = make(13, ctx, S, Hq, Hkv, D, act, kv)
    r = rule_of(c, **dict(RULES[rule], **({"window": 2000} if rule == "all" else {})))
    r = masked(c, r, kind) if kind else r
    d = su.device(c, gpu)
    q, kp = d[8], d[0]
    need = ff.lib.ffkv_prefill_scored_workspace_bytes(ff.torch_dtype_code(q), ff.torch_dtype_code(kp), c.B, S, Hq, Hkv, D, 1,
                                                      c.max_blocks, 0, r["window"], r["end"] is not None)
    assert need > 0
    check(c, call(ff, c, d, r), expected(c, r))


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_cut_and_absent(ff, gpu, kv):
    """max_context_len cuts rows, absent pages hide their keys, rows before their first token see nothing."""
    c = make(15, [300, 0, 0, 90], 40, 4, 2, 128, "bf16", kv)
    c.ctx[1:3] = [-20, -60]
    c.block_table[3, 1:3] = [-1, c.num_blocks]
    r = rule_of(c, slopes=True, window=90)
    check(c, call(ff, c, su.device(c, gpu), r, max_context_len=310), expected(c, r, 310))


def test_large_v(ff, gpu):
    """bf16 values past fp16's range rerun on bf16 products, int8 scales past it on shifted ones."""
    for kv, big in (("bf16", 3e5), ("i8", 1e6)):
        c = make(17, [200], 60, 4, 2, 128, "bf16", kv)
        if kv == "i8":
            c.v_scale *= np.float32(big)
        else:
            c.v_pool = cases.encode(cases.decode(c.v_pool, c.kv) * np.float32(big), c.kv)
        r = rule_of(c, **RULES["all"])
        want = expected(c, r)
        if kv == "i8":  # on the rerun p enters 2^-12 smaller: its fp16 step is 2^-13 of the V scale per key
            step = 2.0 ** -13 * 127 * float(np.abs(c.v_scale).max()) / 64
            want = [(o, e + step, w, x) for o, e, w, x in want]
        check(c, call(ff, c, su.device(c, gpu), r), want)


def test_plain_rule_is_prefill(ff, gpu):
    """Without a rule the call is paged_prefill's, up to the order of its sums."""
    c = make(19, [100, 900], 130)
    d = su.device(c, gpu)
    a = call(ff, c, d, rule_of(c))
    b = ff.paged_prefill(d[8], d[0], d[1], d[4], d[5])
    want = expected(c, rule_of(c))
    check(c, a, want)
    check(c, b, want)


def test_streams_and_graph(ff, gpu):
    """Eager, on another stream, captured and replayed between eager calls."""
    c = make(21, [700, 40], 200)
    r = masked(c, rule_of(c, **RULES["cap"]), "documents")
    d = su.device(c, gpu)
    want = call(ff, c, d, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = call(ff, c, d, r, stream=side)
    side.synchronize()
    assert torch.equal(want, other)
    out = torch.zeros_like(want)
    begin = torch.from_numpy(r["begin"]).to(gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ff.paged_prefill_scored(d[8], d[0], d[1], d[4], d[5], score_cap=5.0, key_begin=begin, out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(call(ff, c, d, r), want)
        assert torch.allclose(out.float(), want.float(), rtol=2.0 ** -7, atol=1e-3)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("ctx", [[6000], [200, 30]])
def test_fp8_head_scale_not_finite(ff, gpu, bad, ctx):
    """A head whose V scale is infinite or NaN: queries that see nothing still give zeros, whole and split over the keys, the
    others nothing finite; the other head is untouched."""
    c = make(33, ctx, 40, 8, 2, 128, "bf16", "fp8")
    kp, vp, ks, vs, bt, cx, _, _, q = su.device(c, gpu)
    end = cx[:, None].repeat(1, 40)
    end[:, 1::2] = 0
    call = lambda: ff.paged_prefill_scored(q, kp, vp, bt, cx, key_end=end, k_scale=ks, v_scale=vs).view(len(ctx), 40, 2, -1)  # noqa: E731
    want = call()
    vs[0] = bad
    got = call()
    assert not got[:, 1::2].float().any()
    assert not got[:, ::2, 0].isfinite().any()
    assert torch.equal(got[:, :, 1], want[:, :, 1])
