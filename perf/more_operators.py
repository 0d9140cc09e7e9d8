"""Rotary positions on several axes, and attention over selected pages of the cache: what an engine has them do, layer by layer.

Image and video tokens have positions on several axes (time, height, width), and their prompts are long; a query then
attends a few pages of its row, chosen by a score that reads far less than the keys.  ``op`` says which call of a layer a
case makes:

  rope    the step's or chunk's q, k and v out of the packed projection: q and k turned by their positions, k and v
          written to their pages (``rope_append_axes``)
  bounds  the smallest and largest key of every page that new tokens went to, per KV head and dim (``update_key_bounds``)
  select  for every block of ``query_block`` queries and KV head, the ``count`` pages to attend (``select_blocks``): the first
          ``sinks``, the last ``recent``, and those with the largest sum over the block's queries and heads of
          sum_d max(q_d lo_d, q_d hi_d), which no q.k of the page's tokens exceeds
  attend  attention over the listed pages (``paged_attention_blocks``)

Context lengths (tokens cached before the call's ``seq`` ones) are spread evenly over [ctx_lo, ctx_hi] and dealt to the
rows in an order drawn from the seed; pages are scattered over a pool 10 % larger than needed.  Keys, values and queries
are N(0, 1), queries times ``spread``; 8-bit caches hold 1 % of the elements 8 times larger.
"""

from __future__ import annotations

import math
import random

import torch

own = False
BLOCK = 16
THETA = 1e6
_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "fp8": torch.uint8}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "fp8": 1}


def _case(op, batch, heads, kv_heads, head_dim, ctx_lo, ctx_hi, q="bf16", kv="bf16", seq=1, sections=(), interleaved=False,
          far=0, count=0, sinks=0, recent=0, query_block=1, wide=False, spread=2.0, **name):
    return {**name, "op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "ctx_lo": ctx_lo,
            "ctx_hi": ctx_hi, "q": q, "kv": kv, "seq": seq, "sections": ",".join(map(str, sections)), "interleaved": interleaved,
            "far": far, "count": count, "sinks": sinks, "recent": recent, "query_block": query_block, "wide": wide,
            "spread": spread}


def listed():
    return [
        # A few short chats on a small model, time, height and width in sections: the smallest step, all launch and latency.
        _case("rope", 4, 16, 8, 128, 17, 255, sections=(16, 24, 24), name="rope_step_small"),
        # Eight prompts' chunks with images in them, the axes interleaved.
        _case("rope", 8, 32, 8, 128, 0, 2000, q="f16", kv="f16", seq=1500, sections=(24, 20, 20), interleaved=True,
              name="rope_images_b8"),
        # One long video, far along in a conversation.
        _case("rope", 1, 28, 4, 128, 0, 0, seq=32000, sections=(16, 24, 24), far=100000, name="rope_video"),
        # A busy server's step: the pages that its 64 new tokens went to.
        _case("bounds", 64, 32, 8, 128, 512, 4096, name="bounds_step_b64"),
        # Eight prompts on an int8 cache.
        _case("bounds", 8, 32, 8, 128, 0, 300, kv="i8", seq=4001, name="bounds_prompts_int8"),
        # A busy server's step over long rows: 64 pages of each.
        _case("select", 64, 32, 8, 128, 2000, 16000, count=64, sinks=1, recent=4, wide=True, name="select_step_b64"),
        # Few very long rows, 7 heads per KV head.
        _case("select", 4, 28, 4, 128, 131000, 131000, q="f16", kv="f16", count=256, sinks=4, recent=16, name="select_long"),
        # A prompt's chunk deep in a long row: every 64 queries share their pages.
        _case("select", 2, 32, 8, 128, 30000, 32000, seq=512, count=128, sinks=4, recent=12, query_block=64,
              name="select_chunk"),
        # A few chats on a small model: the smallest attention.
        _case("attend", 4, 16, 8, 128, 100, 1000, count=16, sinks=1, recent=2, name="attend_step_small"),
        # A busy server's step, 1024 tokens of each long row.
        _case("attend", 64, 32, 8, 128, 2000, 16000, count=64, sinks=1, recent=4, wide=True, name="attend_step_b64"),
        # Few very long rows, 4096 tokens of each.
        _case("attend", 4, 28, 4, 128, 131000, 131000, q="f16", kv="f16", count=256, sinks=4, recent=16, name="attend_long"),
        # Two prompts' chunks deep in long rows on an fp8 cache.
        _case("attend", 2, 32, 8, 128, 30000, 32000, kv="fp8", seq=512, count=128, sinks=4, recent=12, query_block=64,
              name="attend_chunk_fp8"),
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# Bytes and operations of the largest listed case of each kind, which no drawn one goes beyond; the bytes of a drawn
# case's pools (what is attended may be a small part), and of the keys gathered for its queries.
_MOST = {"rope": (5.8e8, 1e12), "bounds": (4.2e7, 1e12), "select": (1.4e8, 1e12), "attend": (2.6e8, 1.8e10)}
_POOLS = 2e9
_GATHERED = 1.5e9


def _cut(case):
    """The case with its rows, queries and contexts cut until it costs no more than the largest listed one."""
    while True:
        w, most = work(case), _MOST[case["op"]]
        blocks = -(-case["seq"] // case["query_block"])
        pools = 2 * case["batch"] * (case["ctx_hi"] + case["seq"]) * case["kv_heads"] * case["head_dim"] * _BYTES[case["kv"]]
        gathered = case["batch"] * blocks * case["kv_heads"] * case["count"] * BLOCK * case["head_dim"] * 4
        pairs = case["batch"] * case["seq"] * case["kv_heads"] * (case["ctx_hi"] / BLOCK) if case["op"] == "select" else 0
        if (w["bytes"] <= most[0] and w["flops"] <= most[1] and pools <= _POOLS and gathered <= _GATHERED
                and pairs <= 2e8):
            return case
        case["batch"] = max(1, case["batch"] * 2 // 3)
        case["ctx_hi"] = case["ctx_hi"] * 4 // 5
        case["ctx_lo"] = min(case["ctx_lo"], case["ctx_hi"])
        case["seq"] = max(1, case["seq"] * 4 // 5)


def draw(rng):
    op = rng.choices(["rope", "bounds", "select", "attend"], [3, 2, 3, 4])[0]
    kv_heads = rng.choice([1, 2, 4, 8, 8, 8])
    group = rng.choice([1, 2, 4, 4, 5, 7, 8])
    kv = rng.choices(["bf16", "f16", "i8", "fp8", "f32"], [5, 2, 2, 2, 1])[0]
    head_dim = rng.choice([64, 80, 96, 112, 128, 128, 128, 128, 256])
    wide, spread = rng.random() < 0.5, rng.uniform(1.0, 3.0)
    hi = _log(rng, 32, 32768)
    lo = max(1, int(hi * rng.uniform(0.1, 1.0)))
    if op == "rope":
        head_dim = rng.choice([64, 128, 128, 256])
        kv = rng.choice(["bf16", "bf16", "f16", "f32"])
        axes, half = rng.choice([2, 3, 3, 4]), head_dim // 2
        interleaved = rng.random() < 0.5
        if interleaved:
            rest = [rng.randint(1, half // axes) for _ in range(axes - 1)]
        else:
            rest = [rng.randint(1, half // axes + half // (2 * axes)) for _ in range(axes - 1)]
        sections = (half - sum(rest), *rest)
        chunk = rng.random() < 0.6
        return _cut(_case(op, _log(rng, 1, 8 if chunk else 128), kv_heads * group, kv_heads, head_dim, lo, hi, q=kv, kv=kv,
                          seq=_log(rng, 2, 8000) if chunk else 1, sections=sections, interleaved=interleaved, wide=wide,
                          far=rng.choice([0, 0, 5000, 200000])))
    if op == "bounds":
        chunk = rng.random() < 0.5
        return _cut(_case(op, _log(rng, 1, 16 if chunk else 128), kv_heads * group, kv_heads, head_dim, lo, hi, kv=kv,
                          seq=_log(rng, 2, 8000) if chunk else 1, wide=wide))
    chunk = rng.random() < 0.4
    seq, query_block = (_log(rng, 2, 1000), rng.choice([1, 4, 16, 32, 64, 100, 128])) if chunk else (1, 1)
    if op == "attend" and kv == "f32" and chunk:
        seq, query_block = min(seq, 64), 1
    if op == "attend" and head_dim in (80, 96, 112) and chunk:
        seq, query_block = min(seq, 64), 1
    if op == "attend" and query_block == 1:
        seq = min(seq, 200)
    count = _log(rng, 4, 256)
    sinks = rng.randint(0, min(4, count // 4))
    recent = rng.randint(min(count - sinks, 1 + query_block // BLOCK), max(1 + query_block // BLOCK, count // 3))
    recent = min(recent, count - sinks)
    batch = _log(rng, 1, 4 if chunk else 96)
    q = "f16" if kv == "f16" else "f32" if kv == "f32" else "bf16"
    if op == "select":  # the longest row has twice the pages that it keeps, and some that are chosen
        hi = max(hi, 200)
        lo = max(lo, hi // 20)
    case = _cut(_case(op, batch, kv_heads * group, kv_heads, head_dim, lo, hi, q=q, kv=kv, seq=seq, count=count, sinks=sinks,
                      recent=recent, query_block=query_block, wide=wide, spread=spread))
    if op == "select":
        case["count"] = max(2, min(count, (max(_lens(case)) + case["seq"]) // BLOCK // 2))
        case["sinks"] = min(sinks, case["count"] - 2)
        case["recent"] = min(recent, case["count"] - 1 - case["sinks"])
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------


def _sections(case):
    """How many pairs of dims turn by each axis."""
    return [int(n) for n in case["sections"].split(",") if n]


def _lens(case):
    """Cached tokens of the rows before the call, evenly spread over [ctx_lo, ctx_hi]."""
    n, lo, hi = case["batch"], case["ctx_lo"], case["ctx_hi"]
    if n == 1:
        return [hi if lo == hi else (lo + hi) // 2]
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _randn(shape, dtype, gen, times=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * times).to(dtype)


def _pool(pages, case, gen):
    """One pool of K or V pages and its scales, as a cache in use holds them."""
    hkv, d, kv = case["kv_heads"], case["head_dim"], case["kv"]
    pool = torch.empty((pages, BLOCK, hkv, d), dtype=_TORCH[kv], device="cuda")
    scale = None
    if kv == "i8":
        scale = torch.empty((pages, BLOCK, hkv), dtype=torch.float32, device="cuda")
    elif kv == "fp8":
        scale = torch.empty(hkv, device="cuda").uniform_(0.08, 0.1, generator=gen)
    slab = max(1, (1 << 26) // (BLOCK * hkv * d))
    for p in range(0, pages, slab):
        shape = (min(slab, pages - p), BLOCK, hkv, d)
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
        if kv in ("i8", "fp8"):
            x.mul_(torch.rand(shape, generator=gen, device="cuda").lt_(0.01).mul_(7.0).add_(1.0))
        if kv == "i8":
            s = x.abs().amax(dim=-1) / 127.0
            scale[p:p + slab] = s
            pool[p:p + slab] = torch.round(x / s[..., None]).to(torch.int8)
        elif kv == "fp8":
            y = (x / scale[None, None, :, None]).clamp_(-448.0, 448.0)
            pool[p:p + slab] = y.to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            pool[p:p + slab] = x
    return pool, scale


def _positions(case, lens, order):
    """Positions [axes, B, S] of the call's tokens: runs of text, where all axes advance together, and images or video
    frames, a grid of height x width per point of time; the next run starts past the largest position so far."""
    axes, s = len(_sections(case)), case["seq"]
    rows = []
    for n in lens:
        at = case["far"] + (n * order.randint(50, 100)) // 100  # earlier images took fewer positions than tokens
        got = []
        while len(got) < s:
            if s == 1 or order.random() < 0.3:
                run = order.randint(1, 200)
                got += [(at + i,) * axes for i in range(run)]
                at += run
                continue
            size = [order.randint(1, 8)] + [order.randint(4, 30) for _ in range(axes - 1)]
            grid = [()]
            for k in size:
                grid = [g + (at + i,) for g in grid for i in range(k)]
            got += grid
            at += max(size)
        rows.append(got[:s])
    return torch.tensor(rows, dtype=torch.int32, device="cuda").permute(2, 0, 1).contiguous()


def _bound_type(case):
    """What an engine keeps the bounds in: the cache's own type, bf16 beside an 8-bit cache."""
    return _TORCH["bf16" if case["kv"] in ("i8", "fp8") else case["kv"]]


def _lists(case, lens, gen):
    """Lists of pages as a selection gives them: ascending, the row's first and last pages among them, -1 behind."""
    b, s, t, hkv, count = case["batch"], case["seq"], case["query_block"], case["kv_heads"], case["count"]
    blocks = -(-s // t)
    last = torch.tensor([min((r + 1) * t, s) - 1 for r in range(blocks)], device="cuda")
    pages = (torch.tensor(lens, device="cuda")[:, None] + last) // BLOCK + 1
    width = max(count, int(pages.max()))
    out = torch.empty((b, blocks, hkv, count), dtype=torch.int32, device="cuda")
    p = torch.arange(width, device="cuda")
    for i in range(b):
        x = torch.rand((blocks, hkv, width), generator=gen, device="cuda")
        n = pages[i][:, None, None]
        x = torch.where((p < case["sinks"]) | (p >= n - case["recent"]), 2.0, x).masked_fill(p >= n, -1.0)
        got = torch.topk(x, count, dim=-1)
        got = torch.where(got.values >= 0, got.indices, 1 << 30).sort(dim=-1).values
        out[i] = torch.where(got == 1 << 30, -1, got)
    return out


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 29)
    order = random.Random(seed * 31 + 11)
    b, s, hq, hkv, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    act, op = _TORCH[case["q"]], case["op"]
    st = {"case": case, "k_scale": None, "v_scale": None}
    lens = _lens(case)
    order.shuffle(lens)
    need = [(n + s + BLOCK - 1) // BLOCK for n in lens]
    pages = math.ceil(sum(need) * 1.1) + 1
    perm = list(range(pages))
    order.shuffle(perm)
    width = max(256, 2 * max(need)) if case["wide"] else max(need)
    rows, at = [], 0
    for n in need:
        rows.append(perm[at:at + n] + [-1] * (width - n))
        at += n
    st["table"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["most"] = max(lens) + s  # tokens of the longest row, as the program that packs the batch knows it
    if op == "rope":
        packed = _randn((b, s, hq + 2 * hkv, d), act, gen)
        st["q"], st["k"], st["v"] = packed[:, :, :hq], packed[:, :, hq:hq + hkv], packed[:, :, hq + hkv:]
        st["positions"] = _positions(case, lens, order)
        st["q_out"] = torch.empty((b, s, hq, d), dtype=act, device="cuda")
        shape = (pages, BLOCK, hkv, d)
        st["k_cache"] = torch.zeros(shape, dtype=_TORCH[case["kv"]], device="cuda")
        st["v_cache"] = torch.zeros(shape, dtype=_TORCH[case["kv"]], device="cuda")
        return st
    if op == "select":
        st["q"] = _randn((b, s, hq, d), act, gen, case["spread"])
        # of 16 keys the smallest and the largest lie near -1.8 and 1.8 around what the page is about
        bounds = torch.empty((pages, hkv, 2, d), dtype=_bound_type(case), device="cuda")
        slab = max(1, (1 << 25) // (hkv * d))
        for p in range(0, pages, slab):
            shape = (min(slab, pages - p), hkv, d)
            mean, half = _randn(shape, torch.float32, gen, 0.4), _randn(shape, torch.float32, gen, 0.3).add_(1.77).abs_()
            bounds[p:p + slab, :, 0], bounds[p:p + slab, :, 1] = mean - half, mean + half
        st["bounds"] = bounds
        blocks = -(-s // case["query_block"])
        st["blocks"] = torch.full((b, blocks, hkv, case["count"]), -1, dtype=torch.int32, device="cuda")
        return st
    st["k_cache"], st["k_scale"] = _pool(pages, case, gen)
    if op == "bounds":
        st["bounds"] = torch.zeros((pages, hkv, 2, d), dtype=_bound_type(case), device="cuda")
        return st
    st["v_cache"], st["v_scale"] = _pool(pages, case, gen)
    st["q"] = _randn((b, s, hq, d), act, gen, case["spread"])
    st["blocks"] = _lists(case, lens, gen)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "attend":
        st["out"] = torch.empty((case["batch"], case["seq"], case["heads"] * case["head_dim"]), dtype=_TORCH[case["q"]],
                                device="cuda")
    return st


# ---- one pass ----------------------------------------------------------------------------------------------------


def run(st):
    return _run_own(st) if own else _PLAIN[st["case"]["op"]](st)


def _run_own(st):
    import firefly_amd as ff

    case = st["case"]
    op = case["op"]
    if op == "rope":
        ff.rope_append_axes(st["q"], st["k"], st["v"], st["positions"], _sections(case), st["k_cache"], st["v_cache"],
                            st["table"], st["lens"], interleaved=case["interleaved"], theta=THETA, q_out=st["q_out"])
        return {"q": st["q_out"], "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if op == "bounds":
        ff.update_key_bounds(st["k_cache"], st["bounds"], st["table"], st["lens"], case["seq"], k_scale=st["k_scale"])
        return {"bounds": st["bounds"]}
    if op == "select":
        ff.select_blocks(st["q"], st["bounds"], st["table"], st["lens"], case["count"], sinks=case["sinks"],
                         recent=case["recent"], query_block=case["query_block"], blocks=st["blocks"],
                         max_context_len=st["most"])
        return {"blocks": st["blocks"]}
    out = ff.paged_attention_blocks(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"], st["blocks"],
                                    query_block=case["query_block"], out=st["out"], k_scale=st["k_scale"],
                                    v_scale=st["v_scale"])
    return {"out": out}


# ---- the same in elementary operations ---------------------------------------------------------------------------


def _pair_axes(case):
    """The axis of each pair of dims."""
    half, axes = case["head_dim"] // 2, len(_sections(case))
    if not case["interleaved"]:
        return [a for a, n in enumerate(_sections(case)) for _ in range(n)]
    got = [0] * half
    for a in range(1, axes):
        for j in range(_sections(case)[a]):
            got[a + axes * j] = a
    return got


def _angles(st):
    """[B, S, D / 2] in 64 bits: far positions turn by many thousand radians."""
    case = st["case"]
    half = case["head_dim"] // 2
    rate = THETA ** (-2.0 * torch.arange(half, dtype=torch.float64, device="cuda") / case["head_dim"])
    axes = torch.tensor(_pair_axes(case), device="cuda")
    return st["positions"].permute(1, 2, 0)[:, :, axes].to(torch.float64) * rate


def _turn(x, cos, sin):
    half = x.shape[-1] // 2
    x = x.to(cos.dtype)
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1)


def _slots(st):
    """Page and slot of the call's tokens, [B, S] each."""
    s = st["case"]["seq"]
    at = st["lens"].long()[:, None] + torch.arange(s, device="cuda")
    return torch.gather(st["table"].long(), 1, at // BLOCK), at % BLOCK


def _plain_rope(st):
    angle = _angles(st)[:, :, None]
    cos, sin = torch.cos(angle).to(torch.float32), torch.sin(angle).to(torch.float32)
    st["q_out"].copy_(_turn(st["q"], cos, sin))
    page, slot = _slots(st)
    k = _turn(st["k"], cos, sin).to(st["q"].dtype)
    st["k_cache"][page, slot] = k.to(st["k_cache"].dtype)
    st["v_cache"][page, slot] = st["v"].to(st["v_cache"].dtype)
    return {"q": st["q_out"], "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _value(pool, scale, kv):
    """Cached rows [..., Hkv, D] in 32 bits."""
    if kv == "fp8":
        return pool.view(torch.float8_e4m3fn).to(torch.float32) * scale[:, None]
    return pool.to(torch.float32) * (scale[..., None] if kv == "i8" else 1.0)


def _outward(lo, hi):
    """fp32 bounds as bf16 ones that still hold what lies between: the lower ones rounded down, the upper ones up."""
    def away(x, sign):  # larger in magnitude where x has the sign, else cut
        u = x.view(torch.int32)
        u = torch.where((u >> 31 != 0) == sign, u + 0xFFFF, u)
        return (u >> 16).to(torch.int16).view(torch.bfloat16)

    return away(lo, True), away(hi, False)


def _touched(st):
    """Rows, pages and live slots [.., 16] of the pages that the call's tokens went to."""
    case = st["case"]
    lens, s = st["lens"].long(), case["seq"]
    first, last = lens // BLOCK, (lens + s - 1) // BLOCK
    most = (case["seq"] + BLOCK - 2) // BLOCK + 1
    at = first[:, None] + torch.arange(most, device="cuda")
    row, j = torch.nonzero(at <= last[:, None], as_tuple=True)
    at = at[row, j]
    live = at[:, None] * BLOCK + torch.arange(BLOCK, device="cuda") < (lens + s)[row][:, None]
    return st["table"].long()[row, at], live


def _plain_bounds(st):
    case = st["case"]
    page, live = _touched(st)
    scale = st["k_scale"][page] if case["kv"] == "i8" else st["k_scale"]
    x = _value(st["k_cache"][page], scale, case["kv"])
    live = live[:, :, None, None]
    lo = x.masked_fill(~live, math.inf).amin(dim=1)
    hi = x.masked_fill(~live, -math.inf).amax(dim=1)
    if case["kv"] in ("i8", "fp8"):
        lo, hi = _outward(lo, hi)
    st["bounds"][page] = torch.stack((lo, hi), dim=2).to(st["bounds"].dtype)
    return {"bounds": st["bounds"]}


def _plain_select(st):
    case = st["case"]
    b, s, hq, hkv, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    t, count = case["query_block"], case["count"]
    blocks = -(-s // t)
    # in 64 bits, rounded once: scores next to the last page that stays are told apart by their last bits
    q = torch.nn.functional.pad(st["q"].to(torch.float64), (0, 0, 0, 0, 0, blocks * t - s))
    q = q.view(b, blocks, t, hkv, hq // hkv, d)
    up, down = q.clamp_min(0.0).sum(dim=(2, 4)), q.clamp_max(0.0).sum(dim=(2, 4))
    both = torch.cat((down, up), dim=-1).transpose(1, 2)  # [B, Hkv, blocks, 2 D], as the bounds lie
    live = (st["most"] + BLOCK - 1) // BLOCK
    table = st["table"][:, :live].long().clamp_min(0)
    box = st["bounds"][table].to(torch.float64).flatten(3).permute(0, 2, 3, 1).contiguous()
    score = torch.matmul(both, box).to(torch.float32)
    last = torch.arange(1, blocks + 1, device="cuda").mul_(t).clamp_max_(s) - 1
    n = ((st["lens"].long()[:, None] + last) // BLOCK + 1)[:, None, :, None]
    p = torch.arange(live, device="cuda")
    score = torch.where((p < case["sinks"]) | (p >= n - case["recent"]), math.inf, score).masked_fill(p >= n, -math.inf)
    at = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :count]
    at = at.masked_fill(at >= n, 1 << 30).sort(dim=-1).values
    at = at.masked_fill(at == 1 << 30, -1).transpose(1, 2).to(torch.int32)
    st["blocks"].copy_(torch.nn.functional.pad(at, (0, count - at.shape[-1]), value=-1))
    return {"blocks": st["blocks"]}


def _plain_attend(st):
    case = st["case"]
    b, s, hq, hkv, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    t, g = case["query_block"], hq // hkv
    blocks = -(-s // t)
    q = torch.nn.functional.pad(st["q"].to(torch.float32), (0, 0, 0, 0, 0, blocks * t - s))
    q = q.view(b, blocks, t, hkv, g, d).permute(0, 1, 3, 2, 4, 5).reshape(b, blocks, hkv, t * g, d)
    lists, slot = st["blocks"].long(), torch.arange(BLOCK, device="cuda")
    pages = torch.gather(st["table"].long()[:, None, None].expand(b, blocks, hkv, -1), 3, lists.clamp_min(0))
    at = (pages[..., None], slot, torch.arange(hkv, device="cuda")[:, None, None])

    def gathered(name):
        x, scale = st[name + "_cache"][at], st[name + "_scale"]
        if case["kv"] == "fp8":
            x = x.view(torch.float8_e4m3fn).to(torch.float32) * scale[:, None, None, None]
        else:
            x = x.to(torch.float32) * (scale[at][..., None] if case["kv"] == "i8" else 1.0)
        return x.flatten(3, 4)

    x = torch.matmul(q, gathered("k").transpose(-1, -2).contiguous()).div_(math.sqrt(d))
    key = (lists[..., None] * BLOCK + slot).masked_fill(lists[..., None] < 0, 1 << 40).flatten(3)
    pos = st["lens"].long()[:, None, None] + torch.arange(blocks * t, device="cuda").view(blocks, t)
    x = x.view(b, blocks, hkv, t, g, -1).masked_fill_(key[:, :, :, None, None] > pos[:, :, None, :, None, None], -math.inf)
    x.sub_(x.amax(dim=-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)).exp_()
    total = x.sum(dim=-1, keepdim=True)
    x.div_(total.masked_fill(total == 0, 1.0))
    o = torch.matmul(x.view(b, blocks, hkv, t * g, -1), gathered("v"))
    out = o.view(b, blocks, hkv, t, g, d).permute(0, 1, 3, 2, 4, 5).reshape(b, blocks * t, hq * d)[:, :s]
    return {"out": out.to(_TORCH[case["q"]])}


_PLAIN = {"rope": _plain_rope, "bounds": _plain_bounds, "select": _plain_select, "attend": _plain_attend}


# ---- what a pass cannot do without -------------------------------------------------------------------------------


def work(case):
    b, s, hq, hkv, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    es, qs, op = _BYTES[case["kv"]], _BYTES[case["q"]], case["op"]
    row = hkv * d * es + (4 * hkv if case["kv"] == "i8" else 0)  # a cached token's K (or V), with scales
    lens = _lens(case)
    bound = hkv * d * 2 * (2 if case["kv"] in ("i8", "fp8") else es)  # a page's bounds
    if op == "rope":
        tokens = b * s
        return {"bytes": tokens * (2.0 * hq * d * qs + 2 * hkv * d * qs + 2 * row + 4 * len(_sections(case))) + 8.0 * b,
                "flops": 3.0 * tokens * (hq + hkv) * d}
    if op == "bounds":
        pages = keys = 0
        for n in lens:
            first = n // BLOCK
            pages += (n + s - 1) // BLOCK - first + 1
            keys += n + s - first * BLOCK
        return {"bytes": float(keys * row + pages * (bound + 4)), "flops": 2.0 * keys * hkv * d}
    t = case["query_block"]
    blocks = -(-s // t)
    q = b * s * hq * d * qs
    if op == "select":
        pages = sum((n + s - 1) // BLOCK + 1 for n in lens)
        scored = sum((n + min((r + 1) * t, s) - 1) // BLOCK + 1 for n in lens for r in range(blocks))
        return {"bytes": float(q + pages * (bound + 4) + 4 * b * blocks * hkv * case["count"]),
                "flops": 4.0 * scored * hkv * d + q / qs}
    keys = pairs = 0
    for n in lens:
        have = [(n + min((r + 1) * t, s) - 1) // BLOCK + 1 for r in range(blocks)]
        took = [min(case["count"], h) for h in have]
        keys += min(have[-1], sum(took)) * BLOCK  # a page that several blocks of queries list is read once
        pairs += sum(k * BLOCK * min(t, s - r * t) for r, k in enumerate(took))
    return {"bytes": float(2 * q + 2 * keys * row + 4 * b * blocks * hkv * case["count"]), "flops": 4.0 * pairs * hq * d}


# ---- the same in 64 bits -------------------------------------------------------------------------------------------


def _exact_rope(case, st):
    wide, half = torch.float64, case["head_dim"] // 2
    pos = st["positions"].to(wide)
    angle = torch.empty((case["batch"], case["seq"], half), dtype=wide, device="cuda")
    for i, a in enumerate(_pair_axes(case)):
        angle[:, :, i] = pos[a] * math.exp(-2.0 * i / case["head_dim"] * math.log(THETA))
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]

    def turned(x):
        y = torch.complex(x[..., :half].to(wide), x[..., half:].to(wide)) * turn
        return torch.cat((y.real, y.imag), dim=-1)

    got = {}
    for name, x in (("k_cache", turned(st["k"])), ("v_cache", st["v"].to(wide))):
        pool = st[name].to(wide)
        for i, n in enumerate(st["lens"].tolist()):
            at = torch.arange(n, n + case["seq"], device="cuda")
            pool[st["table"][i, at // BLOCK].long(), at % BLOCK] = x[i]
        got[name] = pool
    return {"q": turned(st["q"]), **got}


def _cached(st, name, i, n):
    """Row i's first n keys or values [n, Hkv, D] in 64 bits."""
    pool, scale, kv, wide = st[name + "_cache"], st[name + "_scale"], st["case"]["kv"], torch.float64
    pages = st["table"][i, :(n + BLOCK - 1) // BLOCK].long()
    x = pool[pages]
    if kv == "fp8":
        x = x.view(torch.float8_e4m3fn).float().to(wide) * scale.to(wide)[:, None]
    elif kv == "i8":
        x = x.to(wide) * scale[pages].to(wide)[..., None]
    return x.to(wide).flatten(0, 1)[:n]


def _exact_bounds(case, st):
    got = st["bounds"].to(torch.float64)
    for i, n in enumerate(st["lens"].tolist()):
        total, first = n + case["seq"], n // BLOCK
        x = _cached(st, "k", i, total)[first * BLOCK:]
        ends = list(range(BLOCK, x.shape[0], BLOCK)) + [x.shape[0]]
        whole = x.shape[0] // BLOCK
        page = st["table"][i, first:first + len(ends)].long()
        if whole:
            y = x[:whole * BLOCK].unflatten(0, (whole, BLOCK))
            got[page[:whole], :, 0], got[page[:whole], :, 1] = y.amin(dim=1), y.amax(dim=1)
        if x.shape[0] % BLOCK:
            y = x[whole * BLOCK:]
            got[page[-1], :, 0], got[page[-1], :, 1] = y.amin(dim=0), y.amax(dim=0)
    return {"bounds": got}


def _exact_attend(case, st):
    b, s, hq, hkv, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    t, wide = case["query_block"], torch.float64
    if b * s * hq * case["count"] * BLOCK * d > 3e11:
        return None
    out = torch.zeros((b, s, hq, d), dtype=wide, device="cuda")
    for i, n in enumerate(st["lens"].tolist()):
        k, v = _cached(st, "k", i, n + s), _cached(st, "v", i, n + s)
        for first in range(0, s, t):
            some = slice(first, min(first + t, s))
            pos = n + torch.arange(s, device="cuda")[some]
            for h in range(hkv):
                at = st["blocks"][i, first // t, h].long()
                at = (at[at >= 0][:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).flatten()
                at = at[at < n + s]
                heads = slice(h * hq // hkv, (h + 1) * hq // hkv)
                x = torch.einsum("tgd,nd->tgn", st["q"][i, some, heads].to(wide), k[at, h]) / math.sqrt(d)
                x = x.masked_fill(at > pos[:, None, None], -math.inf)
                p = torch.nan_to_num(torch.softmax(x, dim=-1), nan=0.0)  # no key at all
                out[i, some, heads] = torch.einsum("tgn,nd->tgd", p, v[at, h])
    return {"out": out.flatten(2)}


def exact(case, seed):
    if case["op"] == "select":  # indices alone
        return None
    st = _inputs(case, seed)
    return {"rope": _exact_rope, "bounds": _exact_bounds, "attend": _exact_attend}[case["op"]](case, st)
