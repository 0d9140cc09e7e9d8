"""Scored attention and cache eviction on the paged KV cache: what an engine has them do, layer by layer.

Models that cap their scores by a tanh, bias them by distance, attend a window, or mask by documents or a prefix need
that inside the attention; long conversations need tokens evicted from the cache by the attention they get.  ``op``
says which call of a layer a case makes:

  decode   a decode step (``paged_attention_scored``): append one token per row, attend its visible context under the
           score rule, and with ``weights`` add each key's attention weight to what it had
  prefill  a prompt chunk under a score rule over its cached prefix (``paged_prefill_scored``; the chunk is already
           appended), or, with ``contiguous``, a packed prompt over its own K/V
  weights  the attention weights that the last ``seq`` tokens of every row give to its keys (``attention_weights``)
  evict    keep the ``keep`` tokens of every row and KV head with the largest weights, its first ``sinks`` and last
           ``recent`` tokens always among them, and pack them into new pages (``evict_tokens``)

Score rule, for the query at position i and key j: s = scale q.k, capped to cap * tanh(s / cap) where ``cap`` is set,
less slope[head] * |i - j| where ``slopes`` is; ``window`` hides keys j <= i - window.  ``mask`` "documents" gives every
query the keys of its own document (causal, or all of them in the prompt's first document), "prefix" makes the first
keys of a row visible to all its queries.

Context lengths are spread evenly over [ctx_lo, ctx_hi] and dealt to the rows in an order drawn from the seed.  Pages
are scattered over a pool 10 % larger than needed; ``wide`` block tables have the row stride of an engine whose context
limit is well above the contexts at hand.  Keys, values and queries are N(0, 1), the queries times ``spread``, so that
scores reach the cap; quantized caches hold 1 % of the elements 8 times larger.
"""

from __future__ import annotations

import math
import random

import torch

own = False
BLOCK = 16
_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "fp8": torch.uint8}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "fp8": 1}


def _case(op, batch, heads, kv_heads, head_dim, ctx_lo, ctx_hi, q="bf16", kv="bf16", seq=1, cap=0.0, slopes=False,
          window=0, mask="", weights=False, keep=0, sinks=0, recent=0, contiguous=False, wide=False, spread=3.0, **name):
    return {**name, "op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "q": q, "kv": kv, "seq": seq, "cap": cap, "slopes": slopes,
            "window": window, "mask": mask, "weights": weights, "keep": keep, "sinks": sinks, "recent": recent,
            "contiguous": contiguous, "wide": wide, "spread": spread}


def listed():
    return [
        # A few short chats on a small model with capped scores: the smallest step, all launch and latency.
        _case("decode", 4, 16, 8, 128, 17, 255, cap=30.0, name="decode_small"),
        # A busy server's step in one of the windowed layers of a model that caps its scores.
        _case("decode", 64, 32, 8, 128, 512, 4096, cap=50.0, window=1024, wide=True, name="decode_window_b64"),
        # Long documents on a model that knows positions by distance alone: few rows of 32k tokens, 7 heads per KV head.
        _case("decode", 8, 28, 4, 128, 32768, 32768, q="f16", kv="f16", slopes=True, name="decode_distance_long"),
        # The step of a server that evicts: attention, and the weights that it gives, accumulated.
        _case("decode", 64, 32, 8, 128, 512, 4096, weights=True, name="decode_weights_b64"),
        # Eight prompts' chunks in a windowed, capped layer.
        _case("prefill", 8, 32, 8, 128, 2000, 2900, seq=512, cap=50.0, window=1024, name="prefill_window_b8"),
        # Documents packed into one prompt, the first attended both ways as a prefix is.
        _case("prefill", 1, 32, 8, 128, 0, 0, q="f16", kv="f16", seq=2000, mask="documents", contiguous=True,
              name="prefill_documents"),
        # One request's 256-token chunk deep in a long prompt on an fp8 cache, biased by distance.
        _case("prefill", 1, 32, 8, 128, 7919, 7919, kv="fp8", seq=256, slopes=True, wide=True, name="prefill_distance_one"),
        # What the last 32 tokens of one long prompt look at, before it is cut to size.
        _case("weights", 1, 32, 8, 128, 32700, 32700, seq=32, name="weights_one_long"),
        # The same for a batch of ordinary prompts on an int8 cache, capped scores.
        _case("weights", 16, 32, 8, 128, 400, 4000, kv="i8", seq=64, cap=50.0, name="weights_int8_b16"),
        # A few short chats cut to 256 tokens on an fp32 cache.
        _case("evict", 4, 16, 8, 128, 200, 1000, q="f32", kv="f32", keep=256, sinks=4, recent=64, name="evict_small"),
        # A full server's rows cut to 1000 tokens on an int8 cache.
        _case("evict", 64, 32, 8, 128, 900, 8000, kv="i8", keep=1000, sinks=4, recent=250, name="evict_int8_b64"),
        # One very long conversation cut to an eighth.
        _case("evict", 1, 32, 8, 128, 131000, 131000, keep=16384, sinks=16, recent=1024, name="evict_one_long"),
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rule(rng, hi, masks):
    """A score rule: what caps, biases and masks, alone and together."""
    kind = rng.choice(["cap", "window", "slopes", "cap_window", "cap_slopes", "slopes_window", "all", "plain"])
    cap = rng.choice([15.0, 30.0, 50.0]) if kind in ("cap", "cap_window", "cap_slopes", "all") else 0.0
    window = _log(rng, 16, max(17, hi)) if kind in ("window", "cap_window", "slopes_window", "all") else 0
    return {"cap": cap, "window": window, "slopes": kind in ("slopes", "cap_slopes", "slopes_window", "all"),
            "mask": rng.choice(masks)}


# Bytes and operations of the largest listed case of each kind, which no drawn one goes beyond, and the bytes of a
# drawn case's pools (a window's case may hold far more than it reads).
_MOST = {"decode": (6.1e8, 1e12), "prefill": (6e8, 6.8e10), "weights": (6.9e7, 1.8e10), "evict": (2.8e8, 0.0)}
_POOLS = 2e9


def _cut(case):
    """The case with its rows, queries and contexts cut until it costs no more than the largest listed one."""
    while True:
        w, most = work(case), _MOST[case["op"]]
        pools = 2 * case["batch"] * case["ctx_hi"] * case["kv_heads"] * case["head_dim"] * _BYTES[case["kv"]]
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and pools <= _POOLS:
            break
        case["batch"] = max(1, case["batch"] * 2 // 3)
        case["ctx_hi"] = case["ctx_hi"] * 4 // 5
        case["ctx_lo"] = min(case["ctx_lo"], case["ctx_hi"])
        if case["op"] in ("prefill", "weights"):
            case["seq"] = max(1, case["seq"] * 4 // 5)
    return case


def draw(rng):
    op = rng.choices(["decode", "prefill", "weights", "evict"], [4, 3, 2, 2])[0]
    kv_heads = rng.choice([2, 4, 8, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 7, 8])
    kv = rng.choices(["bf16", "f16", "i8", "fp8", "f32"], [5, 2, 2, 2, 0 if op == "prefill" else 1])[0]
    head_dim = rng.choice([64, 128, 128, 128, 256] if op == "prefill" else [64, 80, 96, 112, 128, 128, 128, 128, 256])
    common = {"wide": rng.random() < 0.5, "spread": rng.uniform(1.0, 4.0)}
    if op == "prefill" and rng.random() < 0.3:
        kv = rng.choice(["bf16", "f16"])
        common.update(contiguous=True, wide=False)
    common.update(kv=kv, q=kv if kv in ("f16", "f32") else "bf16")
    if op == "decode":
        hi = _log(rng, 32, 32768)
        return _cut(_case(op, _log(rng, 1, 96), heads, kv_heads, head_dim, max(1, int(hi * rng.uniform(0.1, 1.0))), hi,
                          weights=rng.random() < 0.4, **common, **_rule(rng, hi, ["", "", "", "documents"])))
    if op == "prefill":
        seq, hi = _log(rng, 16, 2000), 0 if common.get("contiguous") else _log(rng, 64, 16000)
        return _cut(_case(op, _log(rng, 1, 4 if hi == 0 else 12), heads, kv_heads, head_dim,
                          int(hi * rng.uniform(0.1, 1.0)), hi, seq=seq, **common,
                          **_rule(rng, hi + seq, ["", "", "documents", "prefix"])))
    if op == "weights":
        seq, hi = _log(rng, 1, 128), _log(rng, 64, 32000)
        return _cut(_case(op, _log(rng, 1, 24), heads, kv_heads, head_dim, max(1, int(hi * rng.uniform(0.1, 1.0))), hi,
                          seq=seq, **common, **_rule(rng, hi, ["", "", "documents", "prefix"])))
    hi = _log(rng, 64, 120000)
    keep = _log(rng, 16, hi)
    sinks = min(keep // 2, rng.choice([0, 1, 4, 64]))
    return _cut(_case(op, _log(rng, 1, 64), heads, kv_heads, head_dim, max(1, int(hi * rng.uniform(0.05, 1.0))), hi,
                      keep=keep, sinks=sinks, recent=int((keep - sinks) * rng.uniform(0.0, 1.0)), **common))


# ---- inputs ------------------------------------------------------------------------------------------------------


def _lens(case):
    """Cached tokens of the rows before the call, evenly spread over [ctx_lo, ctx_hi]."""
    n, lo, hi = case["batch"], case["ctx_lo"], case["ctx_hi"]
    if n == 1:
        return [hi if lo == hi else (lo + hi) // 2]
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _randn(shape, dtype, gen, times=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * times).to(dtype)


def _outliers(shape, gen):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return x.mul_(torch.rand(shape, generator=gen, device="cuda").lt_(0.01).mul_(7.0).add_(1.0))


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
        if kv in ("i8", "fp8"):
            x = _outliers(shape, gen)
            if kv == "i8":
                s = x.abs().amax(dim=-1) / 127.0
                scale[p:p + slab] = s
                pool[p:p + slab] = torch.round(x / s[..., None]).to(torch.int8)
            else:
                y = (x / scale[None, None, :, None]).clamp_(-448.0, 448.0)
                pool[p:p + slab] = y.to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            pool[p:p + slab] = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return pool, scale


def _ranges(case, lens, order):
    """Visible keys [begin, end) of every query, as the engine's packing gives them: None where the rule is causal."""
    b, s = case["batch"], case["seq"]
    begin, end = [], []
    for n in lens:
        if case["mask"] == "prefix":
            p = order.randrange(0, n + s + 1)
            begin += [0] * s
            end += [max(p, n + t + 1) for t in range(s)]
            continue
        cuts = sorted({n} | {n + order.randrange(1, s) for _ in range(min(7, s - 1))} if s > 1 else {n})
        if n > 0:  # the row's cached tokens are documents too; the chunk's first goes on with the last of them
            cuts[0] = order.randrange(0, n)
        for t in range(s):
            k = sum(c <= n + t for c in cuts) - 1
            begin.append(cuts[k])
            both = k == 0 and n == 0
            end.append((cuts[1] if len(cuts) > 1 else n + s) if both else n + t + 1)
    shape = (b, s)
    return (torch.tensor(begin, dtype=torch.int32, device="cuda").view(shape),
            torch.tensor(end, dtype=torch.int32, device="cuda").view(shape))


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 17)
    order = random.Random(seed * 31 + 5)
    b, s, hq, hkv, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    act, op = _TORCH[case["q"]], case["op"]
    st = {"begin": None, "end": None, "slopes": None, "k_scale": None, "v_scale": None}
    if case["slopes"]:
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device="cuda")
    if op != "evict":
        st["q"] = _randn((b, s, hq, d), act, gen, case["spread"])
    lens = _lens(case)
    order.shuffle(lens)
    if case["contiguous"]:
        lens = [0] * b
        st["k_cache"], st["v_cache"] = _randn((b, s, hkv, d), act, gen), _randn((b, s, hkv, d), act, gen)
    if case["mask"]:
        st["begin"], st["end"] = _ranges(case, lens, order)
    if case["contiguous"]:
        return st
    if op == "decode":
        make = _outliers if case["kv"] in ("i8", "fp8") else lambda shape, gen: _randn(shape, torch.float32, gen)
        st["k"], st["v"] = make((b, 1, hkv, d), gen).to(act), make((b, 1, hkv, d), gen).to(act)
    new = 0 if op == "evict" else s
    need = [(n + new + BLOCK - 1) // BLOCK for n in lens]
    room = (case["keep"] + BLOCK - 1) // BLOCK if op == "evict" else 0
    pages = math.ceil((sum(need) + b * room) * 1.1) + 1
    perm = list(range(pages - 1))  # the pool's last page belongs to no row
    order.shuffle(perm)
    width = max(need)
    if case["wide"]:
        width = max(256, 2 * width)
    rows, at = [], 0
    for n in need:
        rows.append(perm[at:at + n] + [-1] * (width - n))
        at += n
    st["table"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["most"] = max(lens) + new  # tokens of the longest row, as the program that packs the batch knows it
    st["k_cache"], st["k_scale"] = _pool(pages, case, gen)
    if op != "weights":
        st["v_cache"], st["v_scale"] = _pool(pages, case, gen)
    if op == "evict" or op == "weights" or case["weights"]:
        # accumulated weights: few tokens have most of them, some have had none at all (of an accumulating call: of the
        # size of what it adds)
        w = torch.randn((b, hkv, st["most"]), generator=gen, device="cuda").mul_(2.0).exp_()
        w.mul_(1.0 if op == "evict" else 1e-3)
        st["prior"] = w * torch.rand(w.shape, generator=gen, device="cuda").ge_(0.1)
        st["weights"] = torch.zeros_like(w)
    if op == "evict":
        dst = [perm[at + i * room:at + (i + 1) * room] for i in range(b)]
        st["dst"] = torch.tensor(dst, dtype=torch.int32, device="cuda")
        st["kept"] = torch.full((b, hkv, case["keep"]), -1, dtype=torch.int32, device="cuda")
    return st


DECAY = 0.875  # of earlier weights, per step


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    b, s, hq, d = case["batch"], case["seq"], case["heads"], case["head_dim"]
    if case["op"] in ("decode", "prefill"):
        st["out"] = torch.empty((b, s, hq * d), dtype=_TORCH[case["q"]], device="cuda")
    return st


# ---- one pass ----------------------------------------------------------------------------------------------------


def _caches(st):
    got = {"k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if st["case"]["kv"] == "i8":
        got.update(k_scale=st["k_scale"], v_scale=st["v_scale"])
    return got


def run(st):
    return _run_own(st) if own else _PLAIN[st["case"]["op"]](st)


def _run_own(st):
    import firefly_amd as ff

    case = st["case"]
    op = case["op"]
    rule = {"score_cap": case["cap"], "slopes": st["slopes"], "window": case["window"]}
    scales = {"k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    if op == "decode":
        more = {"weights": st["weights"], "prior": st["prior"], "decay": DECAY} if case["weights"] else {}
        begin = None if st["begin"] is None else st["begin"][:, 0]
        out = ff.paged_attention_scored(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"], k_new=st["k"],
                                        v_new=st["v"], key_begin=begin, out=st["out"], max_context_len=st["most"], **rule,
                                        **scales, **more)
        return {"out": out, **_caches(st), **({"weights": st["weights"]} if case["weights"] else {})}
    if op == "prefill":
        if case["contiguous"]:
            return {"out": ff.paged_prefill_scored(st["q"], st["k_cache"], st["v_cache"], None, None, key_begin=st["begin"],
                                                   key_end=st["end"], out=st["out"], **rule)}
        return {"out": ff.paged_prefill_scored(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"],
                                               key_begin=st["begin"], key_end=st["end"], out=st["out"],
                                               max_context_len=st["most"], **rule, **scales)}
    if op == "weights":
        return {"weights": ff.attention_weights(st["q"], st["k_cache"], st["table"], st["lens"], weights=st["weights"],
                                                prior=st["prior"], decay=DECAY, key_begin=st["begin"], key_end=st["end"],
                                                k_scale=st["k_scale"], max_context_len=st["most"], **rule)}
    kept, lens = ff.evict_tokens(st["prior"], st["k_cache"], st["v_cache"], st["table"], st["lens"], case["keep"],
                                 sinks=case["sinks"], recent=case["recent"], dst_table=st["dst"], kept=st["kept"],
                                 weights_out=st["weights"], **scales)
    return {"kept": kept, "lens": lens, "weights": st["weights"], **_caches(st)}


# ---- the same in elementary operations ---------------------------------------------------------------------------


def _value(pool, scale, kv):
    """Cached rows [..., Hkv, D] in 32 bits."""
    if kv == "fp8":
        return pool.view(torch.float8_e4m3fn).to(torch.float32) * scale[:, None]
    return pool.to(torch.float32) * (scale[..., None] if kv == "i8" else 1.0)


def _rows(st, name):
    """[B, Hkv, T, D] in 32 bits: the rows' keys or values up to the longest row's last token."""
    case, pool, scale = st["case"], st[name + "_cache"], st[name + "_scale"]
    if case["contiguous"]:
        return pool.to(torch.float32).transpose(1, 2).contiguous()
    live = (st["most"] + BLOCK - 1) // BLOCK
    pages = st["table"][:, :live].long().clamp_min(0)
    x = _value(pool[pages], scale[pages] if case["kv"] == "i8" else scale, case["kv"])
    return x.flatten(1, 2)[:, :st["most"]].transpose(1, 2).contiguous()


def _probabilities(st, k):
    """softmax of the scores [B, Hkv, G, S, T] in 32 bits; rows without a visible key are zero."""
    case = st["case"]
    b, s, hq, hkv, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    g, n = hq // hkv, k.shape[2]
    q = st["q"].to(torch.float32).view(b, s, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * s, d)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).div_(math.sqrt(d)).view(b, hkv, g, s, n)
    if case["cap"]:
        x.div_(case["cap"]).tanh_().mul_(case["cap"])
    first = 0 if case["contiguous"] else st["lens"][:, None]
    i = (first + torch.arange(s, device="cuda")).expand(b, s)[:, :, None]
    j = torch.arange(n, device="cuda")
    if st["slopes"] is not None:
        x.sub_(st["slopes"].view(1, hkv, g, 1, 1) * (i - j).abs().to(torch.float32)[:, None, None])
    total = s if case["contiguous"] else st["lens"][:, None, None] + s
    seen = j <= i if st["end"] is None else j < st["end"][:, :, None]
    seen = seen & (j < total)
    if st["begin"] is not None:
        seen = seen & (j >= st["begin"][:, :, None])
    if case["window"]:
        seen = seen & (j > i - case["window"])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    most = x.amax(dim=-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    x = x.sub_(most).exp_()
    total = x.sum(dim=-1, keepdim=True)
    return x.div_(total.masked_fill_(total == 0, 1.0))


def _attend(st):
    case = st["case"]
    b, s, hq, hkv, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    p = _probabilities(st, _rows(st, "k"))
    o = torch.matmul(p.view(b, hkv, -1, p.shape[-1]), _rows(st, "v"))
    out = o.view(b, hkv, hq // hkv, s, d).permute(0, 3, 1, 2, 4).reshape(b, s, hq * d)
    return out.to(_TORCH[case["q"]]), p


def _add_weights(st, p):
    """decay * prior + the weights of this call's queries, those of its own tokens alone for its own tokens."""
    w = p.sum(dim=(2, 3))
    j = torch.arange(w.shape[2], device="cuda")
    lens = st["lens"][:, None, None]
    got = torch.where(j < lens, st["prior"] * DECAY + w, w)
    return torch.where(j < lens + st["case"]["seq"], got, st["weights"])


def _append(st, name):
    """The step's new token of every row to its slot."""
    case, x, pool, scale = st["case"], st[name], st[name + "_cache"], st[name + "_scale"]
    lens = st["lens"].long()
    page, slot = torch.gather(st["table"].long(), 1, lens[:, None] // BLOCK)[:, 0], lens % BLOCK
    x = x[:, 0]
    if case["kv"] == "i8":
        sc = x.to(torch.float32).abs().amax(dim=-1) / 127.0
        scale[page, slot] = sc
        x = torch.round(x.to(torch.float32) / sc[..., None]).to(torch.int8)
    elif case["kv"] == "fp8":
        x = (x.to(torch.float32) / scale[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    pool[page, slot] = x.to(pool.dtype)


def _plain_decode(st):
    _append(st, "k")
    _append(st, "v")
    out, p = _attend(st)
    return {"out": out, **_caches(st), **({"weights": _add_weights(st, p)} if st["case"]["weights"] else {})}


def _plain_prefill(st):
    return {"out": _attend(st)[0]}


def _plain_weights(st):
    return {"weights": _add_weights(st, _probabilities(st, _rows(st, "k")))}


def _plain_evict(st):
    case, w = st["case"], st["prior"]
    keep, kv = case["keep"], case["kv"]
    j = torch.arange(w.shape[2], device="cuda")
    lens = st["lens"].long()[:, None, None]
    always = (j < case["sinks"]) | (j >= lens - case["recent"])
    key = torch.where(always, math.inf, w).masked_fill(j >= lens, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    order = torch.nn.functional.pad(order, (0, max(0, keep - order.shape[2])))[..., :keep]
    count = st["lens"].clamp_max(keep)
    rank = torch.arange(keep, device="cuda")
    live = rank < count[:, None, None]
    src = torch.where(live, order, 1 << 40).sort(dim=-1).values.masked_fill(~live, 0)
    weights = st["weights"].clone()
    got = torch.gather(w, 2, src)[..., :w.shape[2]]
    weights[..., :got.shape[2]] = torch.where(live[..., :w.shape[2]], got, weights[..., :got.shape[2]])
    # a row's slots past its kept tokens go from and to the pool's last page, which belongs to no row
    spare = st["k_cache"].shape[0] - 1
    b, h = torch.arange(w.shape[0], device="cuda")[:, None, None], torch.arange(w.shape[1], device="cuda")[:, None]
    at = torch.where(live, st["table"].long()[b, src // BLOCK], spare), src % BLOCK, h
    to = torch.where(live, st["dst"].long()[b, rank // BLOCK], spare), torch.where(live, rank % BLOCK, 0), h
    st["k_cache"][to] = st["k_cache"][at]
    st["v_cache"][to] = st["v_cache"][at]
    if kv == "i8":
        st["k_scale"][to] = st["k_scale"][at]
        st["v_scale"][to] = st["v_scale"][at]
    return {"kept": src.masked_fill(~live, -1).int(), "lens": count, "weights": weights, **_caches(st)}


_PLAIN = {"decode": _plain_decode, "prefill": _plain_prefill, "weights": _plain_weights, "evict": _plain_evict}


# ---- what a pass cannot do without -------------------------------------------------------------------------------


def _pairs(case, lens):
    """(query, key) pairs that are visible, and the keys that some query sees: without a drawn mask."""
    s, w = case["seq"], case["window"]
    pairs = keys = 0
    for n in lens:
        if w == 0:
            pairs += s * n + s * (s + 1) // 2
            keys += n + s
        else:
            full = max(0, min(s, w - 1 - n))  # queries that the window cuts nothing from
            pairs += full * n + full * (full + 1) // 2 + (s - full) * w
            keys += min(n + s, w + s - 1)
    return pairs, keys


def work(case):
    b, s, hq, hkv, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    es, qs, op = _BYTES[case["kv"]], _BYTES[case["q"]], case["op"]
    row = hkv * d * es + (4 * hkv if case["kv"] == "i8" else 0)  # a cached token's K (or V), with scales
    lens = [0] * b if case["contiguous"] else _lens(case)
    if op == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        # weights read; kept tokens read and written, their weights and indices written
        return {"bytes": 4.0 * hkv * sum(lens) + kept * (4.0 * row + 8.0 * hkv) + 8 * b, "flops": 0.0}
    pairs, keys = _pairs(case, lens)
    masks = 2 * 4 * b * s if case["mask"] else 0
    tables = 0 if case["contiguous"] else 4 * ((keys + BLOCK - 1) // BLOCK + b)
    slopes = 4 * hq if case["slopes"] else 0
    nbytes = b * s * hq * d * qs + tables + masks + slopes
    if op == "weights":
        return {"bytes": nbytes + keys * row + 2 * 4.0 * hkv * (sum(lens) + b * s), "flops": 2.0 * pairs * hq * d}
    nbytes += b * s * hq * d * qs
    if op == "decode":  # the new tokens come from their source and are written
        nbytes += 2 * (keys - b) * row + 2 * b * hkv * d * qs + 2 * b * row
        nbytes += 2 * 4.0 * hkv * (sum(lens) + b) if case["weights"] else 0
    else:
        nbytes += 2 * keys * row
    return {"bytes": float(nbytes), "flops": 4.0 * pairs * hq * d}


# ---- the same in 64 bits -------------------------------------------------------------------------------------------


def _exact_row(case, q, k, first, slopes, begin, end, total):
    """Probabilities [Hq, S, T] of queries q [S, Hq, D] at positions first + t over keys k [T, Hkv, D], 64 bits."""
    s, hq, d = q.shape
    hkv, n = k.shape[1], k.shape[0]
    x = torch.empty((hq, s, n), dtype=torch.float64, device="cuda")
    for h in range(hq):
        x[h] = q[:, h].double() @ k[:, h * hkv // hq].T.contiguous()
    x *= 1.0 / math.sqrt(d)
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    pos = first + torch.arange(s, device="cuda")
    key = torch.arange(n, device="cuda")
    if slopes is not None:
        x -= slopes.double()[:, None, None] * (pos[:, None] - key[None, :]).abs().double()
    lo = torch.zeros(s, dtype=torch.int64, device="cuda") if begin is None else begin.long()
    hi = pos + 1 if end is None else end.long()
    if case["window"]:
        lo = torch.maximum(lo, pos + 1 - case["window"])
    hidden = (key[None, :] < lo[:, None]) | (key[None, :] >= hi[:, None]) | (key[None, :] >= total)
    x[:, hidden] = -math.inf
    p = torch.softmax(x, dim=-1)
    return torch.nan_to_num(p, nan=0.0)  # no key at all


def _exact_attention(case, st):
    b, s, hkv, d, kv = case["batch"], case["seq"], case["kv_heads"], case["head_dim"], case["kv"]
    got = {}
    lens = [0] * b if case["contiguous"] else st["lens"].tolist()
    if case["op"] == "decode":
        quant = kv in ("i8", "fp8")
        for i, n in enumerate(lens):
            page, slot = int(st["table"][i, n // BLOCK]), n % BLOCK
            for name in ("k", "v"):
                x, pool, scale = st[name][i, 0].float(), st[name + "_cache"], st[name + "_scale"]
                if kv == "i8":
                    scale[page, slot] = x.abs().amax(dim=-1) / 127.0
                    x = torch.round(x / scale[page, slot][:, None])
                elif kv == "fp8":
                    x = (x / scale[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
                pool[page, slot] = x.to(pool.dtype)
        got.update(k_cache=None if quant else st["k_cache"], v_cache=None if quant else st["v_cache"])
        if kv == "i8":
            got.update(k_scale=st["k_scale"], v_scale=st["v_scale"])
    wide = torch.float64

    def cached(name, i, live):
        pool, scale = st[name + "_cache"], st[name + "_scale"]
        if case["contiguous"]:
            return pool[i].to(wide)
        pages = st["table"][i, :(live + BLOCK - 1) // BLOCK].long()
        x = pool[pages]
        if kv == "fp8":
            x = x.view(torch.float8_e4m3fn).float().to(wide) * scale.to(wide)[:, None]
        elif kv == "i8":
            x = x.to(wide) * scale[pages].to(wide)[..., None]
        return x.to(wide).reshape(-1, hkv, d)[:live]

    out, weights = [], []
    for i, n in enumerate(lens):
        live = n + s
        p = _exact_row(case, st["q"][i], cached("k", i, live), n, st["slopes"],
                       None if st["begin"] is None else st["begin"][i], None if st["end"] is None else st["end"][i], live)
        if case["op"] != "weights":
            v = cached("v", i, live)
            out.append(torch.stack([p[h] @ v[:, h * hkv // p.shape[0]].contiguous() for h in range(p.shape[0])], dim=1)
                       .reshape(s, -1))
        if case["op"] == "weights" or case["weights"]:
            w = p.view(hkv, -1, s, live).sum(dim=(1, 2))
            w[:, :n] += DECAY * st["prior"][i, :, :n].to(wide)
            weights.append(torch.nn.functional.pad(w, (0, st["most"] - live)))
    if out:
        got["out"] = torch.stack(out)
    if weights:
        got["weights"] = torch.stack(weights)
    return got


def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] != "evict":
        return _exact_attention(case, st)
    quant = case["kv"] in ("i8", "fp8")
    for i, n in enumerate(st["lens"].tolist()):
        m = min(n, case["keep"])
        first, last = min(case["sinks"], m), min(case["recent"], m)
        for h in range(case["kv_heads"]):
            if n <= case["keep"]:
                idx = torch.arange(n, device="cuda")
            else:
                w = st["prior"][i, h, first:n - last].double()
                by = torch.sort(-w, stable=True).indices[:m - first - last] + first
                idx = torch.cat((torch.arange(first, device="cuda"), by.sort().values, torch.arange(n - last, n, device="cuda")))
            st["weights"][i, h, :m] = st["prior"][i, h, idx]
            at, to = st["table"][i, idx // BLOCK].long(), torch.arange(m, device="cuda")
            page = st["dst"][i, to // BLOCK].long()
            for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
                if st[name] is not None and st[name].dim() > 1:
                    st[name][page, to % BLOCK, h] = st[name][at, idx % BLOCK, h]
    got = {"kept": None, "lens": None, "weights": st["weights"], "k_cache": None, "v_cache": None}
    if not quant:
        got.update(k_cache=st["k_cache"], v_cache=st["v_cache"])
    elif case["kv"] == "i8":
        got.update(k_scale=st["k_scale"], v_scale=st["v_scale"])
    return got
