"""The cache operators' workloads: what they are measured on, and their plain forms.

Four operators that a batch of sequences on one key/value cache needs, each in two forms: elementary
torch operations (``own = False``) and the calls a user makes of this package (``own = True``).

* ``head_norm_rope``: the fused QKV projection's rows -> queries, and keys and values at their cache
  slots; RMS norm of every query and key head, rotation by one or several position axes.
* ``prefix_attention``: attention of a batch over a prefix that all its sequences share and over each
  sequence's own keys.
* ``cache_weights``: the softmax weight that every cached key received, accumulated.
* ``cache_evict``: the cache without the keys of least accumulated weight.

Head counts and widths are those of the four models of this repository's benchmark.
"""
import importlib
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
# (query heads, key/value heads, head width): Llama-3-8B, TinyLlama, SmolLM-135M, SmolLM-360M
HEADS = [(32, 8, 128), (32, 4, 64), (9, 3, 64), (15, 5, 64)]
# the most that a drawn case may need: that of the largest listed one
MOST_PAIRS = 64 * 32 * 65536      # (query row, head, key) triples of an attention
MOST_CACHE = 16 * 16384 * 8       # (token, key/value head) pairs of a cache


def listed():
    a = dict(op="head_norm_rope", norm=True, far=131072)
    p = dict(op="prefix_attention")
    w = dict(op="cache_weights", decay=0.9)
    e = dict(op="cache_evict")
    return [
        # one decode step of 32 sequences: latency
        dict(a, name="rope decode 32 rows", rows=32, heads=32, kv_heads=8, width=128, src="f32", dst="bf16", axes=1,
             cyclic=False),
        # one prefill pass of 2048 tokens, the length of the benchmark's prompt
        dict(a, name="rope prefill 2048 rows", rows=2048, heads=32, kv_heads=8, width=128, src="f32", dst="bf16",
             axes=1, cyclic=False),
        # a clip's patches: time, height and width positions, a ragged number of rows
        dict(a, name="rope 3 axes 10007 rows", rows=10007, heads=32, kv_heads=4, width=64, src="f16", dst="f16",
             axes=3, cyclic=True),
        # four short answers to one short prompt on the smallest model: latency
        dict(p, name="attention small", batch=4, rows=1, heads=9, kv_heads=3, width=64, prefix=333, own_max=41,
             type="bf16"),
        # 32 users behind one system prompt
        dict(p, name="attention 32 x 8192", batch=32, rows=1, heads=32, kv_heads=8, width=128, prefix=8192,
             own_max=512, type="bf16"),
        # 64 users of one long document: the largest
        dict(p, name="attention 64 x 65536", batch=64, rows=1, heads=32, kv_heads=8, width=128, prefix=65536,
             own_max=1024, type="bf16"),
        # lookahead: a token and four drafts of each sequence scored at once, odd lengths
        dict(p, name="attention drafts", batch=24, rows=5, heads=32, kv_heads=4, width=64, prefix=20011, own_max=701,
             type="f16"),
        # the weights of one decode step of 16 sequences, added to what their keys had
        dict(w, name="weights decode", batch=16, rows=1, heads=32, kv_heads=8, width=128, cache=8192, type="bf16"),
        # the weights of a prompt's last 1024 queries over its whole cache
        dict(w, name="weights window", batch=1, rows=1024, heads=32, kv_heads=8, width=128, cache=16384,
             type="bf16"),
        # two short caches of the smallest model: latency
        dict(e, name="evict small", batch=2, kv_heads=3, width=64, cache=1000, budget=601, recent=64, type="f16"),
        # one long document cut to an eighth
        dict(e, name="evict 131072", batch=1, kv_heads=8, width=128, cache=131072, budget=16384, recent=512,
             type="bf16"),
        # a full batch cut to half
        dict(e, name="evict 16 x 16384", batch=16, kv_heads=8, width=128, cache=16384, budget=8192, recent=256,
             type="bf16"),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], its logarithm uniform."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["head_norm_rope", "prefix_attention", "cache_weights", "cache_evict"])
    heads, kv_heads, width = rng.choice(HEADS)
    half = rng.choice(["bf16", "f16"])
    if op == "head_norm_rope":
        axes = rng.choice([1, 1, 3])
        return dict(op=op, norm=rng.random() < 0.8, far=_spread(rng, 64, 1 << 20), rows=_spread(rng, 1, 16384),
                    heads=heads, kv_heads=kv_heads, width=width, src=rng.choice(["f32", "f32", "bf16", "f16"]),
                    dst=rng.choice(["f32", half, half]), axes=axes, cyclic=axes > 1 and rng.random() < 0.5)
    if op == "prefix_attention":
        batch, rows = _spread(rng, 1, 64), rng.choice([1, 1, 1, 2, 3, 5, 8])
        prefix = 0 if rng.random() < 0.08 else min(_spread(rng, 1, 65536), MOST_PAIRS // (batch * rows * heads))
        own_max = min(_spread(rng, 1, 2048), 64 * 1024 // batch)
        return dict(op=op, batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, width=width, prefix=prefix,
                    own_max=own_max, type=half)
    if op == "cache_weights":
        rows = rng.choice([1, 1, 2, 4]) if rng.random() < 0.5 else _spread(rng, 16, 1024)
        batch = _spread(rng, 1, 16)
        cache = _spread(rng, 64, 131072)
        cache = max(1, min(cache, MOST_CACHE // (2 * batch * kv_heads), 1024 * 32 * 16384 // (batch * rows * heads)))
        return dict(op=op, decay=rng.choice([0.9, 0.99]), batch=batch, rows=rows, heads=heads, kv_heads=kv_heads,
                    width=width, cache=cache, type=half)
    batch = _spread(rng, 1, 16)
    cache = min(_spread(rng, 64, 131072), MOST_CACHE // (batch * kv_heads))
    budget = _spread(rng, 16, cache)
    return dict(op=op, batch=batch, kv_heads=kv_heads, width=width, cache=cache, budget=budget,
                recent=rng.randrange(0, budget + 1), type=half)


def _sections(case):
    """Rotated pairs of each position axis: a quarter for time, the rest for height and width."""
    pairs = case["width"] // 2
    if case["axes"] == 1:
        return [pairs]
    side = 3 * pairs // 10 if case["cyclic"] else 3 * pairs // 8
    return [pairs - 2 * side, side, side]


def _lens(batch, least, most):
    """Lengths of a batch's sequences, spread over [least, most] in no order of their own."""
    if batch == 1:
        return [most]
    return [least + (most - least) * ((5 * i + batch - 1) % batch) // (batch - 1) for i in range(batch)]


def _own_lens(case):
    return _lens(case["batch"], 0, case["own_max"])


def _cache_lens(case):
    return _lens(case["batch"], (case["cache"] + 1) // 2, case["cache"])


def _seen(n, rows):
    """Own keys that the rows of a sequence of n own keys see, in all (a row sees none of the later rows' keys)."""
    return sum(max(0, n - r) for r in range(rows))


def work(case):
    op = case["op"]
    if op == "head_norm_rope":
        heads = case["heads"] + 2 * case["kv_heads"]
        n = case["rows"] * heads * case["width"]
        return {"bytes": n * (SIZE[case["src"]] + SIZE[case["dst"]]) + case["rows"] * (4 * case["axes"] + 8)
                + 8 * case["width"], "flops": 8 * n}
    size, D, kv = SIZE[case["type"]], case["width"], case["kv_heads"]
    if op == "prefix_attention":
        q = case["batch"] * case["rows"] * case["heads"]
        lens = _own_lens(case)
        seen = case["batch"] * case["rows"] * case["prefix"] + sum(_seen(n, case["rows"]) for n in lens)
        return {"bytes": 2 * (case["prefix"] + sum(lens)) * kv * D * size + q * (2 * D * size + 4)
                + 4 * case["batch"], "flops": 4 * seen * case["heads"] * D}
    lens = _cache_lens(case)
    if op == "cache_weights":
        seen = sum(_seen(n, case["rows"]) for n in lens)
        return {"bytes": sum(lens) * kv * (D * size + 8) + case["batch"] * case["rows"] * case["heads"] * (D * size + 4),
                "flops": 2 * seen * case["heads"] * D}
    kept = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": kv * (4 * sum(lens) + kept * (4 * D * size + 8)), "flops": 0}


# ---- inputs -------------------------------------------------------------------------------------------------------


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _queries_keys(g, case, keys):
    """Queries (batch, rows, heads, width) and keys (keys..., kv_heads, width) as attention meets them: logits of a
    spread that differs from head to head, and a part that all queries of a group share."""
    kv, D = case["kv_heads"], case["width"]
    group = case["heads"] // kv
    shared = _normal(g, kv, 1, D)
    gain = 0.5 + 1.5 * torch.rand(kv, group, 1, generator=g, device=DEV)
    q = _normal(g, case["batch"], case["rows"], kv, group, D) * gain + 0.7 * shared
    return q.reshape(case["batch"], case["rows"], case["heads"], D), _normal(g, *keys, kv, D), shared[:, 0]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op, kv, D = case["op"], case["kv_heads"], case["width"]
    s = {"case": dict(case)}
    if op == "head_norm_rope":
        rows, heads, dst = case["rows"], case["heads"], TYPES[case["dst"]]
        # hidden activations have channels far above the others
        loud = torch.exp(0.5 * _normal(g, (heads + 2 * kv) * D))
        s["qkv"] = (_normal(g, rows, (heads + 2 * kv) * D) * loud).to(TYPES[case["src"]])
        s["wq"] = 1 + 0.2 * _normal(g, D) if case["norm"] else None
        s["wk"] = 1 + 0.2 * _normal(g, D) if case["norm"] else None
        pos = torch.randint(0, case["far"], (case["axes"], rows), generator=g, device=DEV, dtype=torch.int32)
        s["pos"] = pos[0] if case["axes"] == 1 else pos
        s["sections"] = _sections(case)
        # a cache of some more slots than rows, in no order; one row in 16 is padding (slot -1); slot 0 is spare
        spare = rows + rows // 8 + 2
        slots = 1 + torch.randperm(spare - 1, generator=g, device=DEV)[:rows]
        s["slots"] = torch.where(torch.arange(rows, device=DEV) % 16 == 15, -1, slots)
        s["k"] = torch.zeros(spare, kv, D, dtype=dst, device=DEV)
        s["v"] = torch.zeros(spare, kv, D, dtype=dst, device=DEV)
        return s
    t = TYPES[case["type"]]
    if op == "prefix_attention":
        B, n = case["batch"], case["own_max"]
        q, k, shared = _queries_keys(g, case, (case["prefix"],))
        if case["prefix"]:
            k[0] += shared  # the first token takes a large part of many heads' weight
        s["q"], s["k_pre"] = q.to(t), k.to(t)
        s["v_pre"] = (_normal(g, case["prefix"], kv, D) + 0.3 * _normal(g, kv, D)).to(t)
        s["k_own"] = _normal(g, B, n, kv, D).to(t)
        s["v_own"] = _normal(g, B, n, kv, D).to(t)
        s["lens"] = torch.tensor(_own_lens(case), dtype=torch.int32, device=DEV)
        return s
    B, L = case["batch"], case["cache"]
    s["lens"] = torch.tensor(_cache_lens(case), dtype=torch.int32, device=DEV)
    if op == "cache_weights":
        q, k, _ = _queries_keys(g, case, (B, L))
        s["q"], s["k"] = q.to(t), k.to(t)
        s["acc"] = torch.rand(B, kv, L, generator=g, device=DEV)
        x = _masked_logits(s["q"], s["k"], s["lens"])
        s["lse"] = torch.logsumexp(x, -1).permute(0, 2, 1, 3).reshape(B, case["rows"], case["heads"])
        return s
    s["k"] = _normal(g, B, L, kv, D).to(t)
    s["v"] = _normal(g, B, L, kv, D).to(t)
    # accumulated weights: a few keys hold most of it, one in ten none at all
    acc = torch.exp(2.0 * _normal(g, B, kv, L))
    s["acc"] = torch.where(torch.rand(B, kv, L, generator=g, device=DEV) < 0.1, 0.0, acc)
    n = case["budget"]
    s["k_out"], s["v_out"] = (torch.zeros(B, n, kv, D, dtype=t, device=DEV) for _ in range(2))
    s["acc_out"] = torch.zeros(B, kv, n, device=DEV)
    s["index"] = torch.zeros(B, kv, n, dtype=torch.int32, device=DEV)
    s["lens_out"] = torch.zeros(B, dtype=torch.int32, device=DEV)
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------


def _masked_logits(q, k, lens):
    """(batch, kv_heads, rows, group, keys) scaled products in 32 bits, -inf where a row does not see the key: a row
    sees the first lens - (rows - 1 - row) keys."""
    B, R, heads, D = q.shape
    L, kv = k.shape[1], k.shape[2]
    qg = q.float().reshape(B, R, kv, heads // kv, D).permute(0, 2, 1, 3, 4).reshape(B, kv, -1, D)
    x = (qg @ k.float().permute(0, 2, 3, 1)).mul_(1 / math.sqrt(D)).reshape(B, kv, R, heads // kv, L)
    limit = lens.view(B, 1) - (R - 1 - torch.arange(R, device=q.device))
    seen = torch.arange(L, device=q.device) < limit.unsqueeze(-1)
    return x.masked_fill_(~seen.view(B, 1, R, 1, L), -math.inf)


def _plain_head_norm_rope(s):
    case = s["case"]
    rows, heads, kv, D = case["rows"], case["heads"], case["kv_heads"], case["width"]
    x = s["qkv"].float().view(rows, heads + 2 * kv, D)
    pairs = torch.arange(D // 2, device=DEV)
    axis = torch.zeros_like(pairs)
    sec = s["sections"]
    if case["axes"] > 1 and case["cyclic"]:
        a = pairs % len(sec)
        axis = torch.where(pairs < len(sec) * torch.tensor(sec, device=DEV)[a], a, 0)
    elif case["axes"] > 1:
        axis = torch.bucketize(pairs, torch.tensor(sec, device=DEV).cumsum(0), right=True)
    pos = s["pos"].view(case["axes"], rows)[axis].t().double()
    angle = pos * torch.pow(10000.0, -2.0 * pairs.double() / D)
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)

    def turned(h, w):
        if w is not None:
            h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5) * w
        lo, hi = h[..., : D // 2], h[..., D // 2:]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(TYPES[case["dst"]])

    q = turned(x[:, :heads], s["wq"])
    keep = (s["slots"] >= 0).view(rows, 1, 1)
    at = s["slots"].clamp(min=0)
    for buf, new in ((s["k"], turned(x[:, heads:heads + kv], s["wk"])), (s["v"], x[:, heads + kv:].to(s["v"].dtype))):
        buf.index_copy_(0, at, torch.where(keep, new, 0))  # slot 0 is spare and stays zero
    return {"q": q, "k": s["k"], "v": s["v"]}


def _plain_prefix_attention(s):
    q, kp, vp, ko, vo = s["q"], s["k_pre"], s["v_pre"], s["k_own"], s["v_own"]
    B, R, heads, D = q.shape
    kv, G, P = ko.shape[2], heads // ko.shape[2], kp.shape[0]
    # every sequence's rows of one key/value head against the prefix: one product
    qp = q.float().view(B * R, kv, G, D).permute(1, 0, 2, 3).reshape(kv, B * R * G, D)
    xp = (qp @ kp.float().permute(1, 2, 0)).mul_(1 / math.sqrt(D))
    xo = _masked_logits(q, ko, s["lens"])
    top_p = xp.amax(-1) if P else xp.new_full((kv, B * R * G), -math.inf)
    top = torch.maximum(top_p.view(kv, B, R, G).permute(1, 0, 2, 3), xo.amax(-1))
    top = torch.where(torch.isfinite(top), top, 0.0)
    ep = xp.sub_(top.permute(1, 0, 2, 3).reshape(kv, -1, 1)).exp_()
    eo = xo.sub_(top.unsqueeze(-1)).exp_()
    z = ep.sum(-1).view(kv, B, R, G).permute(1, 0, 2, 3) + eo.sum(-1)
    op = (ep @ vp.float().permute(1, 0, 2)).view(kv, B, R, G, D).permute(1, 0, 2, 3, 4)
    oo = (eo.view(B, kv, R * G, -1) @ vo.float().permute(0, 2, 1, 3)).view(B, kv, R, G, D)
    out = (op + oo) / torch.where(z > 0, z, 1.0).unsqueeze(-1)
    lse = top + z.log()
    return {"out": out.permute(0, 2, 1, 3, 4).reshape(B, R, heads, D).to(q.dtype),
            "lse": lse.permute(0, 2, 1, 3).reshape(B, R, heads)}


def _plain_cache_weights(s):
    B, R, heads, _ = s["q"].shape
    kv, L = s["k"].shape[2], s["k"].shape[1]
    lse = s["lse"].view(B, R, kv, heads // kv).permute(0, 2, 1, 3).unsqueeze(-1)
    w = _masked_logits(s["q"], s["k"], s["lens"]).sub_(lse).exp_().sum((2, 3))
    held = torch.arange(L, device=DEV) < s["lens"].view(B, 1, 1)
    s["acc"].copy_(torch.where(held, s["case"]["decay"] * s["acc"] + w, s["acc"]))
    return {"acc": s["acc"]}


def _plain_cache_evict(s):
    case, acc, lens = s["case"], s["acc"], s["lens"]
    B, kv, L = acc.shape
    n, D = case["budget"], case["width"]
    at = torch.arange(L, device=DEV)
    length = lens.view(B, 1, 1)
    # whole numbers in the order of the weights; the newest tokens above all, what is no token below all
    key = (acc + 0.0).view(torch.int32).long()
    key = torch.where(at >= length - case["recent"], 1 << 40, key)
    key = torch.where(at >= length, -1, key)
    index = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :n]
    index = torch.where(index < length, index, L).sort(-1).values
    keep = index < length
    src = index.clamp(max=L - 1)
    lens_out = lens.clamp(max=n)
    for name, out in (("k", s["k_out"]), ("v", s["v_out"])):
        new = s[name].permute(0, 2, 1, 3).gather(2, src.unsqueeze(-1).expand(B, kv, n, D)).permute(0, 2, 1, 3)
        out.copy_(torch.where(keep.permute(0, 2, 1).unsqueeze(-1), new, out))
    s["acc_out"].copy_(torch.where(keep, acc.gather(2, src), s["acc_out"]))
    s["index"].copy_(torch.where(keep, index.int(), s["index"]))
    s["lens_out"].copy_(lens_out)
    return {k: s[k] for k in ("k_out", "v_out", "acc_out", "index", "lens_out")}


# ---- the framework's calls ----------------------------------------------------------------------------------------

_core = None


def _compute():
    global _core
    if _core is None:
        package = importlib.import_module("daisychain-infer_b200")
        _core = package.init_compute(torch.cuda.current_device(), stream=torch.cuda.current_stream())
    return _core


def _own_run(s):
    comp, case = _compute(), s["case"]
    op = case["op"]
    if op == "head_norm_rope":
        q = torch.empty(case["rows"], case["heads"], case["width"], dtype=TYPES[case["dst"]], device=DEV)
        comp.head_norm_rope_dev(s["qkv"], s["pos"], q, s["k"], s["v"], slots=s["slots"], wq=s["wq"], wk=s["wk"],
                                eps=1e-5, theta=10000.0, sections=s["sections"], cyclic=case["cyclic"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if op == "prefix_attention":
        out = torch.empty_like(s["q"])
        lse = torch.empty(s["q"].shape[:3], dtype=torch.float32, device=DEV)
        comp.prefix_attention_dev(s["q"], out, k_pre=s["k_pre"], v_pre=s["v_pre"], k_own=s["k_own"], v_own=s["v_own"],
                                  lens=s["lens"], lse=lse)
        return {"out": out, "lse": lse}
    if op == "cache_weights":
        comp.cache_weights_dev(s["q"], s["k"], s["lens"], s["lse"], s["acc"], decay=case["decay"])
        return {"acc": s["acc"]}
    comp.cache_evict_dev(s["k"], s["v"], s["acc"], s["lens"], s["k_out"], s["v_out"], s["acc_out"], s["index"],
                         s["lens_out"], budget=case["budget"], recent=case["recent"])
    return {k: s[k] for k in ("k_out", "v_out", "acc_out", "index", "lens_out")}


def run(state):
    if own:
        return _own_run(state)
    return {"head_norm_rope": _plain_head_norm_rope, "prefix_attention": _plain_prefix_attention,
            "cache_weights": _plain_cache_weights, "cache_evict": _plain_cache_evict}[state["case"]["op"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------


def _exact_head_norm_rope(s, case):
    heads, kv, D, rows = case["heads"], case["kv_heads"], case["width"], case["rows"]
    x = s["qkv"].double().view(rows, heads + 2 * kv, D)
    pos = s["pos"].view(case["axes"], rows).double()
    sec = _sections(case)
    turn = torch.empty(rows, D // 2, dtype=torch.complex128, device=DEV)
    first = 0
    owner = [0] * (D // 2)
    for a, n in enumerate(sec):
        for j in range(n):
            if case["cyclic"] and a:
                owner[a + len(sec) * j] = a
            elif not case["cyclic"]:
                owner[first + j] = a
        first += n
    for i in range(D // 2):
        angle = pos[owner[i]] * 10000.0 ** (-2.0 * i / D)
        turn[:, i] = torch.polar(torch.ones_like(angle), angle)
    out = {}
    for name, lo, n, w in (("q", 0, heads, s["wq"]), ("k", heads, kv, s["wk"])):
        h = x[:, lo:lo + n]
        if w is not None:
            h = h / torch.sqrt((h * h).sum(-1, keepdim=True) / D + 1e-5) * w.double()
        z = torch.complex(h[..., :D // 2].contiguous(), h[..., D // 2:].contiguous()) * turn.unsqueeze(1)
        out[name] = torch.cat([z.real, z.imag], -1)
    kept = s["slots"] >= 0
    for name, new in (("k", out["k"]), ("v", x[:, heads + kv:])):
        buf = s[name].double()
        buf[s["slots"][kept]] = new[kept]
        out[name] = buf
    return out


def _exact_prefix_attention(s, case):
    B, R, heads, D, kv = case["batch"], case["rows"], case["heads"], case["width"], case["kv_heads"]
    G = heads // kv
    out = torch.zeros(B, R, heads, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, R, heads), -math.inf, dtype=torch.float64, device=DEV)
    lens = _own_lens(case)
    for h in range(kv):
        q = s["q"][:, :, h * G:(h + 1) * G].double() / math.sqrt(D)
        K, V = s["k_pre"][:, h].double(), s["v_pre"][:, h].double()
        shared = torch.einsum("brgd,kd->brgk", q, K)
        for b in range(B):
            k, v = s["k_own"][b, :, h].double(), s["v_own"][b, :, h].double()
            for r in range(R):
                n = max(0, lens[b] - (R - 1 - r))
                x = torch.cat([shared[b, r], q[b, r] @ k[:n].t()], -1)
                if x.shape[-1]:
                    at = slice(h * G, (h + 1) * G)
                    out[b, r, at] = torch.softmax(x, -1) @ torch.cat([V, v[:n]])
                    lse[b, r, at] = torch.logsumexp(x, -1)
    return {"out": out, "lse": lse}


def _exact_cache_weights(s, case):
    R, heads, D, kv = case["rows"], case["heads"], case["width"], case["kv_heads"]
    G = heads // kv
    acc = s["acc"].double()
    for b, n in enumerate(_cache_lens(case)):
        late = torch.arange(n, device=DEV).view(1, n) >= n - (R - 1 - torch.arange(R, device=DEV).view(R, 1))
        for h in range(kv):
            got = torch.zeros(n, dtype=torch.float64, device=DEV)
            for head in range(h * G, (h + 1) * G):
                x = s["q"][b, :, head].double() @ s["k"][b, :n, h].double().t() / math.sqrt(D)
                p = torch.exp(x - s["lse"][b, :, head].double().unsqueeze(1))
                got += torch.where(late, 0.0, p).sum(0)
            acc[b, h, :n] = case["decay"] * acc[b, h, :n] + got
    return {"acc": acc}


def _exact_cache_evict(s, case):
    kv, budget = case["kv_heads"], case["budget"]
    out = {k: s[k].double() for k in ("k_out", "v_out", "acc_out")}
    index, lens_out = s["index"].clone(), s["lens_out"].clone()
    for b, n in enumerate(_cache_lens(case)):
        kept = min(n, budget)
        lens_out[b] = kept
        for h in range(kv):
            old = max(0, n - case["recent"])
            if n <= budget:
                chosen = torch.arange(n)
            else:
                w = s["acc"][b, h, :old].cpu().double().numpy()
                best = (-w).argsort(kind="stable")[:budget - (n - old)]
                chosen = torch.cat([torch.from_numpy(best).sort().values, torch.arange(old, n)])
            chosen = chosen.to(DEV)
            index[b, h, :kept] = chosen.int()
            out["acc_out"][b, h, :kept] = s["acc"][b, h, chosen].double()
            out["k_out"][b, :kept, h] = s["k"][b, chosen, h].double()
            out["v_out"][b, :kept, h] = s["v"][b, chosen, h].double()
    return {**out, "index": index, "lens_out": lens_out}


def exact(case, seed):
    s = prepare(case, seed)
    return {"head_norm_rope": _exact_head_norm_rope, "prefix_attention": _exact_prefix_attention,
            "cache_weights": _exact_cache_weights, "cache_evict": _exact_cache_evict}[case["op"]](s, case)
