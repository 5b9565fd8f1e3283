"""The operators of a batch's cache on the B200, against their definitions in 64 bits.

Tolerances are bounds, from u = half a unit in the last place (relative): 2^-24
for f32, 2^-11 for f16, 2^-8 for bf16.

* rotation: a norm is off by D u/2 (its sum) + 8 u (quotient, root, two products),
  an angle's fraction by 2^-25 of half a turn and sincospi by 2 ulp (together 8 u),
  the rotation's products and sums by 3 u: (D/2 + 24) u (|lo| + |hi|), and the
  output's rounding u_T |y|.
* scores: a D-term f32 sum is off by at most D 2^-23 scale sum |q| |k| (truncation
  included), which moves an exponential by that factor, and the exponent's own
  product, sum and 2^x by 4 u of it and 2^-21; call it E.
* attention: probabilities rounded to the type, so out is off by (u_T + E) sum p |v| /
  sum p plus the output's rounding; for f16 a probability below 2^-14 is off by up to
  2^-25 absolutely.  lse is off by E + n u (its sum) + 4 u |lse|.
* accumulated weights: (E + rows u) of each sum, the rounding of the result and that
  of the decay.
* eviction: the same bits.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


# ---- head norm and rotation ---------------------------------------------------------


def rope_ref(x, pos, heads, kv, D, rot, sections, cyclic, wq, wk, eps, theta, inv_freq=None):
    """(q, k, v, bound of |lo| + |hi|) in 64 bits from the definition."""
    rows, pairs = x.shape[0], rot // 2
    x = x.double().view(rows, heads + 2 * kv, D)
    pos = pos.view(-1, rows).double()
    axis = []
    for a, n in enumerate(sections):
        axis += [a] * n
    if cyclic:
        A = len(sections)
        axis = [i % A if i // A < sections[i % A] else 0 for i in range(pairs)]
    freq = inv_freq if inv_freq is not None else [theta ** (-2.0 * i / rot) for i in range(pairs)]
    ang = torch.stack([pos[axis[i]] * freq[i] for i in range(pairs)], 1) if pairs else x.new_zeros(rows, 0)
    c, s = ang.cos().unsqueeze(1), ang.sin().unsqueeze(1)
    out, size = [], []
    for lo_, n, w in ((0, heads, wq), (heads, kv, wk)):
        h = x[:, lo_:lo_ + n]
        if w is not None:
            h = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()
        a, b, rest = h[..., :pairs], h[..., pairs:rot], h[..., rot:]
        out.append(torch.cat([a * c - b * s, b * c + a * s, rest], -1))
        both = a.abs() + b.abs()
        size.append(torch.cat([both, both, rest.abs()], -1))
    return out[0], out[1], x[:, heads + kv:], size


def check_rope(got, want, size, D, t):
    err = (got.double() - want).abs()
    tol = (D / 2 + 24) * U[F32] * size + (U[t] * want.abs() if t != F32 else 0) + 2.0 ** -25 * (t == F16)
    assert torch.isfinite(got).all() and (err <= tol).all(), float((err - tol).max())


ROPE = [  # rows, heads, kv, D, rot, sections, cyclic, x type, out type, norm
    (1, 1, 1, 8, 8, [4], False, F32, F32, True),
    (3, 4, 2, 16, 16, [8], False, F32, BF16, True),
    (5, 9, 3, 64, 64, [32], False, F32, F16, True),
    (33, 32, 8, 128, 128, [64], False, F32, BF16, True),
    (7, 3, 1, 40, 40, [20], False, F16, F32, True),         # groups of four channels
    (7, 3, 1, 72, 24, [12], False, BF16, BF16, True),       # partial rotation, groups of four
    (6, 5, 5, 96, 48, [8, 8, 8], False, F32, F32, True),    # partial rotation, three axes
    (9, 15, 5, 64, 64, [14, 9, 9], True, F16, F16, True),   # axes by turns
    (9, 4, 2, 128, 128, [16, 24, 24], False, BF16, F32, False),
    (4, 2, 1, 256, 256, [128], False, F32, F32, True),
    (4, 2, 2, 200, 200, [100], False, F32, BF16, True),
    (4, 3, 2, 80, 0, [0], False, F32, F32, True),           # no rotation
    (2, 0, 2, 64, 64, [32], False, F32, F32, True),         # keys and values alone
    (2, 6, 0, 64, 64, [32], False, F32, F32, True),         # queries alone
    (1500, 9, 3, 64, 64, [20, 4, 4, 4], False, F32, BF16, True),
]


@pytest.mark.parametrize("case", ROPE, ids=lambda c: "x".join(str(v).replace("torch.", "") for v in c))
def test_head_norm_rope(comp, case):
    rows, heads, kv, D, rot, sections, cyclic, ti, to, norm = case
    g = gen(rows + D)
    x = (normal(g, rows, (heads + 2 * kv) * D) * 3).to(ti)
    wq, wk = (1 + 0.3 * normal(g, D) if norm else None for _ in range(2))
    pos = torch.randint(-50, 1 << 20, (len(sections), rows), generator=g, device="cuda", dtype=torch.int32)
    q = torch.full((rows, heads, D), math.nan, dtype=to, device="cuda")
    slots = torch.randperm(rows + 3, generator=g, device="cuda")[:rows]
    if rows > 2:
        slots[1] = -1
    k, v = (torch.full((rows + 3, kv, D), 7.0, dtype=to, device="cuda") for _ in range(2))
    comp.head_norm_rope_dev(x, pos if len(sections) > 1 else pos[0], q, k, v, slots=slots, wq=wq, wk=wk, eps=1e-6,
                            theta=5e5, rot=rot, sections=sections, cyclic=cyclic)
    comp.sync()
    rq, rk, rv, size = rope_ref(x, pos, heads, kv, D, rot, sections, cyclic, wq, wk, 1e-6, 5e5)
    check_rope(q, rq, size[0], D, to)
    on = slots >= 0
    check_rope(k[slots[on]], rk[on], size[1][on], D, to)
    assert torch.equal(v[slots[on]], rv[on].to(to))
    rest = torch.ones(rows + 3, dtype=torch.bool, device="cuda")
    rest[slots[on]] = False
    assert (k[rest] == 7).all() and (v[rest] == 7).all()  # (unwritten slots stay)


def test_rope_strides_and_sequences(comp):
    """A cache of sequences with keys and values side by side, head-major queries, a wider projection
    row at an address that is no multiple of 16 bytes, inverse frequencies of the caller's own."""
    g = gen(5)
    rows, heads, kv, D = 11, 4, 2, 64
    wide = normal(g, rows, (heads + 2 * kv) * D + 5)
    x = wide[:, 3:3 + (heads + 2 * kv) * D]
    pos = torch.arange(rows, dtype=torch.int32, device="cuda") * 1000
    q = torch.empty(heads, rows, D, dtype=BF16, device="cuda").transpose(0, 1)
    both = torch.zeros(3, 8, kv, 2, D, dtype=BF16, device="cuda")
    slots = torch.tensor([0, 5, 7, 8, 9, 15, 16, 18, 20, 23, 22], device="cuda")
    inv = [1.0 / (i + 1) for i in range(D // 2)]
    comp.head_norm_rope_dev(x, pos, q, both[:, :, :, 0], both[:, :, :, 1], slots=slots, inv_freq=inv)
    comp.sync()
    rq, rk, rv, size = rope_ref(x.contiguous(), pos, heads, kv, D, D, [D // 2], False, None, None, 0, 1, inv)
    check_rope(q, rq, size[0], D, BF16)
    flat = both.view(24, kv, 2, D)
    check_rope(flat[slots, :, 0], rk, size[1], D, BF16)
    assert torch.equal(flat[slots, :, 1], rv.to(BF16))


def test_rope_rows_without_slots_and_one_row(comp):
    x = normal(gen(1), 1, 6 * 32)
    q, k, v = (torch.empty(1, n, 32, device="cuda") for n in (4, 1, 1))
    pos = torch.tensor([3], dtype=torch.int32, device="cuda")
    comp.head_norm_rope_dev(x, pos, q, k, v)
    rq, rk, rv, size = rope_ref(x, pos, 4, 1, 32, 32, [16], False, None, None, 0, 1e4)
    check_rope(q, rq, size[0], 32, F32)
    check_rope(k, rk, size[1], 32, F32)
    assert torch.equal(v.double(), rv)


def test_rope_nan_rows_stay_their_own(comp):
    x = normal(gen(2), 4, 6 * 64)
    x[1, 70] = math.nan  # head 1 of row 1
    q, k, v = (torch.empty(4, n, 64, device="cuda") for n in (4, 1, 1))
    comp.head_norm_rope_dev(x, torch.arange(4, dtype=torch.int32, device="cuda"), q, k, v, wq=torch.ones(64, device="cuda"),
                            wk=torch.ones(64, device="cuda"))
    comp.sync()
    bad = torch.isnan(q)
    assert bad[1, 1].all() and int(bad.sum()) == 64 and not torch.isnan(k).any()


def test_rope_slot_behind_the_cache_is_reported(P, comp):
    x = normal(gen(3), 3, 6 * 64)
    q = torch.empty(3, 4, 64, device="cuda")
    kv = torch.zeros(2, 5, 1, 64, device="cuda")
    k, v = kv[0], kv[1]
    comp.head_norm_rope_dev(x, torch.zeros(3, dtype=torch.int32, device="cuda"), q, k, v,
                            slots=torch.tensor([4, 5, 1 << 40], device="cuda"))
    with pytest.raises(P.DeviceError, match="bounds"):
        comp.sync()
    comp.sync()  # (reported once)
    assert int((k.abs().sum((1, 2)) > 0).sum()) == 1 and int((v.abs().sum((1, 2)) > 0).sum()) == 1


# ---- attention over a shared prefix and own keys ---------------------------------------


def attention_ref(q, kp, vp, ko, vo, lens, scale):
    """out, lse, sum p |v| / sum p, E, keys of a row: 64 bits, row by row."""
    B, R, H, D = q.shape
    kv = kp.shape[1] if kp is not None else ko.shape[2]
    G = H // kv
    q = q.double()
    out, mag = (torch.zeros(B, R, H, D, dtype=torch.float64, device="cuda") for _ in range(2))
    lse = torch.full((B, R, H), -math.inf, dtype=torch.float64, device="cuda")
    E = torch.zeros(B, R, H, dtype=torch.float64, device="cuda")
    n = torch.zeros(B, R, 1, dtype=torch.float64, device="cuda")
    for b in range(B):
        own = 0 if ko is None else max(0, min(int(lens[b]), ko.shape[1]))
        for r in range(R):
            m = max(0, own - (R - 1 - r))
            K = torch.cat(([kp.double()] if kp is not None else []) + ([ko[b, :m].double()] if ko is not None else []))
            V = torch.cat(([vp.double()] if vp is not None else []) + ([vo[b, :m].double()] if vo is not None else []))
            if not K.shape[0]:
                continue
            x = torch.einsum("hd,khd->hk", q[b, r], K.repeat_interleave(G, 1)) * scale
            size = torch.einsum("hd,khd->hk", q[b, r].abs(), K.abs().repeat_interleave(G, 1)) * scale
            n[b, r] = K.shape[0]
            E[b, r] = D * 2.0 ** -23 * size.amax(-1) + 4 * U[F32] * x.abs().amax(-1) + 2.0 ** -21
            top = x.amax(-1, keepdim=True)
            p = torch.exp(x - torch.where(torch.isfinite(top), top, 0.0))
            z = p.sum(-1, keepdim=True)
            some = z > 0
            w = torch.where(some, p / z, 0.0)
            Vr = V.repeat_interleave(G, 1)
            out[b, r] = torch.einsum("hk,khd->hd", w, Vr)
            mag[b, r] = torch.einsum("hk,khd->hd", w, Vr.abs())
            lse[b, r] = torch.where(some[:, 0], top[:, 0] + z[:, 0].log(), -math.inf)
    return out, lse, mag, E, n


def check_attention(out, lse, ref, t, vmax):
    want, wlse, mag, E, n = ref
    E = E.unsqueeze(-1)
    tol = (U[t] + E) * mag + (n.unsqueeze(-1) * 2.0 ** -25 * vmax if t == F16 else 0)
    tol = tol + (U[out.dtype] * (want.abs() + tol) if out.dtype != F32 else 4 * U[F32] * mag) + 2.0 ** -25
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all() and (err <= tol).all(), float((err - tol).max())
    if lse is not None:
        empty = torch.isinf(wlse)
        assert torch.equal(torch.isneginf(lse), empty)
        err = (lse.double() - wlse)[~empty].abs()
        tol = (E[..., 0] + n * U[F32] + 4 * U[F32] * wlse.abs())[~empty]
        assert (err <= tol).all(), float((err - tol).max())


ATTN = [  # batch, rows, heads, kv, D, prefix, own_max, lens, type, out type
    (1, 1, 1, 1, 8, 1, 0, None, BF16, BF16),
    (1, 1, 1, 1, 8, 0, 1, [1], F16, F16),
    (2, 1, 4, 2, 64, 0, 5, [0, 5], BF16, BF16),              # a row that sees nothing
    (2, 3, 4, 2, 64, 0, 5, [2, 9], F16, F32),                # rows before the first key; a length above the cache
    (3, 1, 9, 3, 64, 65, 17, [0, 16, 17], BF16, BF16),
    (3, 2, 15, 5, 64, 127, 33, [1, 2, 33], F16, F16),
    (2, 1, 32, 8, 128, 128, 64, [64, 63], BF16, F32),
    (2, 5, 8, 2, 128, 129, 81, [80, -3], F16, F16),          # a negative length
    (4, 1, 7, 1, 40, 257, 100, [3, 99, 100, 50], BF16, BF16),
    (1, 16, 8, 8, 72, 64, 200, [200], BF16, BF16),
    (2, 4, 32, 1, 128, 300, 40, [37, 4], BF16, BF16),        # 128 rows of one sequence and head
    (33, 1, 32, 8, 64, 400, 20, list(range(-5, 28)), F16, F16),   # two tiles of rows, the second short
    (19, 4, 32, 8, 128, 1000, 9, [5] * 19, BF16, BF16),      # three: a pair and one by itself
    (70, 1, 8, 1, 64, 2000, 1, [1] * 70, F16, F16),          # five tiles of rows
    (1, 1, 8, 1, 128, 5003, 1301, [1300], F16, F16),         # split keys, few rows
    (2, 1, 16, 2, 112, 1025, 515, [500, 515], BF16, BF16),
]


@pytest.mark.parametrize("case", ATTN, ids=lambda c: "x".join(str(v).replace("torch.", "") for v in c[:7]) + str(c[8])[6:])
def test_prefix_attention(comp, case):
    B, R, H, kv, D, P, L, lens, t, to = case
    g = gen(B + D + P)
    q = (normal(g, B, R, H, D) * 1.5).to(t)
    # what lies behind the prefix and behind a sequence's tokens is NaN
    kp, vp = (torch.cat([normal(g, P, kv, D), torch.full((3, kv, D), math.nan, device="cuda")]).to(t)[:P] if P else None
              for _ in range(2))
    ko = vo = ln = None
    if lens is not None:
        ko, vo = (normal(g, B, L, kv, D).to(t) for _ in range(2))
        for b, n in enumerate(lens):
            ko[b, max(0, n):] = math.nan
            vo[b, max(0, n):] = math.nan
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full((B, R, H, D), math.nan, dtype=to, device="cuda")
    lse = torch.full((B, R, H), math.nan, device="cuda")
    comp.prefix_attention_dev(q, out, k_pre=kp, v_pre=vp, k_own=ko, v_own=vo, lens=ln, lse=lse)
    comp.sync()
    ref = attention_ref(q, kp, vp, ko, vo, lens, D ** -0.5)
    vmax = max(float(v.nan_to_num().abs().max()) for v in (vp, vo) if v is not None)
    check_attention(out, lse, ref, t, vmax)


def test_attention_layouts_scale_and_workspace(comp):
    """Head-major caches, keys and values in one buffer, strided queries and outputs, a scale, no lse, a
    workspace of the caller's own that holds anything."""
    g = gen(8)
    B, R, H, kv, D, P, L, t = 3, 2, 12, 4, 64, 333, 50, BF16
    q = normal(g, H, B, R, D).to(t).permute(1, 2, 0, 3)
    pre = normal(g, kv, P, 2, D).to(t)
    own = normal(g, kv, B, L, 2, D).to(t)
    kp, vp = (pre[:, :, i].transpose(0, 1) for i in range(2))
    ko, vo = (own[:, :, :, i].permute(1, 2, 0, 3) for i in range(2))
    lens = [50, 1, 23]
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.empty(B, H, R, D, device="cuda").transpose(1, 2)
    args = (q, out, kp, vp, ko, vo, ln)
    ws = torch.full((comp.prefix_attention_ws(*args, scale=0.3),), 255, dtype=torch.uint8, device="cuda")
    comp.prefix_attention_dev(*args, scale=0.3, ws=ws)
    comp.sync()
    check_attention(out, None, attention_ref(q, kp, vp, ko, vo, lens, 0.3), t, 6.0)


@pytest.mark.parametrize("t", [F16, BF16])
def test_attention_with_growing_scores(comp, t):
    """Every tile's scores are above the tile before's, so the running maximum is raised all the time."""
    g = gen(9)
    B, R, H, kv, D, P, L = 2, 1, 8, 2, 128, 700, 300
    q = torch.ones(B, R, H, D, device="cuda").to(t) * 0.5
    ramp = lambda n, lo: (torch.linspace(lo, lo + 40, n, device="cuda").view(n, 1, 1) / D * 2).expand(n, kv, D)  # noqa: E731
    kp, ko = ramp(P, -30).to(t), ramp(L, -10).expand(B, L, kv, D).to(t).contiguous()
    vp, vo = normal(g, P, kv, D).to(t), normal(g, B, L, kv, D).to(t)
    lens = [300, 150]
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(B, R, H, device="cuda")
    comp.prefix_attention_dev(q, out, kp, vp, ko, vo, ln, lse, scale=1.0)
    comp.sync()
    check_attention(out, lse, attention_ref(q, kp, vp, ko, vo, lens, 1.0), t, 6.0)


def test_attention_non_finite_scores(comp):
    """Keys at -inf take no part, a row of nothing else is empty, a NaN spoils its own head's rows only,
    and a later draft's value does not reach an earlier row."""
    g = gen(10)
    B, R, H, kv, D, P, L, t = 2, 2, 4, 2, 64, 200, 20, BF16
    q = normal(g, B, R, H, D).abs().to(t)
    kp, vp = normal(g, P, kv, D).to(t), normal(g, P, kv, D).to(t)
    ko, vo = normal(g, B, L, kv, D).to(t), normal(g, B, L, kv, D).to(t)
    kp[:, 0] = -math.inf      # head 0's prefix scores are all -inf
    ko[0, :, 0] = -math.inf   # and all of sequence 0
    vo[1, 9] = math.inf       # the value of sequence 1's last token, which row 0 does not see
    ln = torch.tensor([10, 10], dtype=torch.int32, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(B, R, H, device="cuda")
    comp.prefix_attention_dev(q, out, kp, vp, ko, vo, ln, lse)
    comp.sync()
    assert (out[0, :, :2] == 0).all() and torch.isneginf(lse[0, :, :2]).all()
    assert torch.isfinite(out[1, 0]).all() and not torch.isfinite(out[1, 1]).any()
    fine = attention_ref(q[:1], kp, vp, ko[:1], vo[:1], [10], D ** -0.5)
    check_attention(out[:1, :, 2:], lse[:1, :, 2:], tuple(x[:, :, 2:] if x.shape[-1] != 1 else x for x in fine), t, 6.0)
    kp[3, 1, 5] = math.nan
    comp.prefix_attention_dev(q, out, kp, vp, ko, vo, ln, lse)
    comp.sync()
    assert torch.isnan(out[:, :, 2:]).all() and torch.isnan(lse[:, :, 2:]).all() and (out[0, :, :2] == 0).all()


# Row counts around what one tile of rows, two, and the small batches' kernel take; key counts around its
# tiles of 16 and 64 and the others' of 128: batch, rows, heads, kv, D, prefix, own_max, lens, type, out type
ATTN_EDGES = [
    (31, 1, 1, 1, 64, 15, 0, None, BF16, BF16),
    (32, 1, 2, 2, 64, 16, 3, [3] * 32, F16, F16),
    (33, 1, 2, 2, 64, 17, 3, [2] * 33, F16, F16),
    (4, 4, 8, 4, 128, 63, 0, None, F16, F32),
    (4, 4, 8, 4, 128, 1025, 30, [4, 30, 0, 17], BF16, BF16),
    (11, 3, 4, 4, 128, 127, 0, None, BF16, BF16),
    (11, 3, 4, 4, 128, 256, 0, None, BF16, F32),
    (128, 1, 2, 2, 8, 128, 0, None, F16, F16),
    (129, 1, 2, 2, 64, 129, 0, None, BF16, BF16),
    (16, 16, 2, 2, 128, 385, 20, [20] * 16, F16, F16),
    (257, 1, 1, 1, 120, 130, 0, None, BF16, BF16),
    (64, 1, 4, 1, 64, 1, 0, None, BF16, BF16),
]


@pytest.mark.parametrize("case", ATTN_EDGES,
                         ids=lambda c: "x".join(str(v).replace("torch.", "") for v in c[:7]) + str(c[8])[6:])
def test_prefix_attention_edges(comp, case):
    test_prefix_attention(comp, case)


@pytest.mark.parametrize("B, D, t", [(12, 128, BF16), (12, 64, F16), (40, 128, F16), (40, 64, BF16), (100, 128, BF16)])
def test_shared_prefix_with_growing_scores(comp, B, D, t):
    """As above for more rows: one tile of rows whose groups join, pairs of tiles, a pair and one by itself."""
    g = gen(B + D)
    H, kv, P = 8, 2, 1500
    q = torch.ones(B, 1, H, D, device="cuda").to(t) * 0.5
    kp = (torch.linspace(-30, 60, P, device="cuda").view(P, 1, 1) / D * 2).expand(P, kv, D).to(t)
    vp = normal(g, P, kv, D).to(t)
    out, lse = torch.empty_like(q), torch.empty(B, 1, H, device="cuda")
    comp.prefix_attention_dev(q, out, kp, vp, lse=lse, scale=1.0)
    comp.sync()
    check_attention(out, lse, attention_ref(q, kp, vp, None, None, None, 1.0), t, 6.0)


@pytest.mark.parametrize("B, D", [(12, 128), (12, 64), (40, 128), (40, 64)])
def test_shared_prefix_non_finite_scores(comp, B, D):
    """The same at -inf and NaN: an empty head, one whose later keys take no part, one that is spoiled."""
    g = gen(B + D + 1)
    H, kv, P, t = 12, 3, 600, BF16
    q = normal(g, B, 1, H, D).abs().to(t)
    kp, vp = normal(g, P, kv, D).to(t), normal(g, P, kv, D).to(t)
    kp[:, 0] = -math.inf
    kp[:200, 1] = -math.inf
    kp[301:, 1] = -math.inf
    out, lse = torch.empty_like(q), torch.empty(B, 1, H, device="cuda")
    comp.prefix_attention_dev(q, out, kp, vp, lse=lse)
    comp.sync()
    assert (out[:, :, :4] == 0).all() and torch.isneginf(lse[:, :, :4]).all()
    fine = attention_ref(q[:, :, 4:8], kp[200:301, 1:2], vp[200:301, 1:2], None, None, None, D ** -0.5)
    check_attention(out[:, :, 4:8], lse[:, :, 4:8], fine, t, 6.0)
    fine = attention_ref(q[:, :, 8:], kp[:, 2:], vp[:, 2:], None, None, None, D ** -0.5)
    check_attention(out[:, :, 8:], lse[:, :, 8:], fine, t, 6.0)
    kp[599, 2, 5] = math.nan
    comp.prefix_attention_dev(q, out, kp, vp, lse=lse)
    comp.sync()
    assert torch.isnan(out[:, :, 8:]).all() and torch.isnan(lse[:, :, 8:]).all() and (out[:, :, :4] == 0).all()


def test_attention_equal_inputs_equal_bits(comp):
    g = gen(11)
    q = normal(g, 40, 1, 8, 128).to(BF16)
    kp, vp = normal(g, 3001, 2, 128).to(BF16), normal(g, 3001, 2, 128).to(BF16)
    outs = []
    for _ in range(3):
        out, lse = torch.empty_like(q), torch.empty(40, 1, 8, device="cuda")
        comp.prefix_attention_dev(q, out, kp, vp, lse=lse)
        outs.append((out, lse))
    comp.sync()
    assert all(torch.equal(outs[0][i], o[i]) for o in outs for i in range(2))


# ---- accumulated weights -----------------------------------------------------------------


def weights_ref(q, k, lens, lse, acc, scale, decay, causal):
    B, R, H, D = q.shape
    L, kv = k.shape[1:3]
    G = H // kv
    out, tol = acc.double().clone(), torch.zeros(acc.shape, dtype=torch.float64, device="cuda")
    for b in range(B):
        n = max(0, min(int(lens[b]), L))
        if not n:
            continue
        K = k[b, :n].double().repeat_interleave(G, 1)
        x = torch.einsum("rhd,khd->rhk", q[b].double(), K) * scale
        size = torch.einsum("rhd,khd->rhk", q[b].double().abs(), K.abs()) * scale
        seen = torch.arange(n, device="cuda").view(1, 1, n) < (
            n - (R - 1 - torch.arange(R, device="cuda").view(R, 1, 1)) if causal else n)
        z = lse[b].double().unsqueeze(-1)
        w = torch.where(seen & ~torch.isneginf(z), torch.exp(x - torch.where(torch.isneginf(z), 0.0, z)), 0.0)
        E = D * 2.0 ** -23 * size + 4 * U[F32] * (x.abs() + z.abs().nan_to_num(posinf=0.0)) + 2.0 ** -21 + R * G * U[F32]
        got = w.sum(0).view(kv, G, n).sum(1)
        old = out[b, :, :n] * decay if decay else 0.0
        out[b, :, :n] = old + got
        # the result's rounding, and that of the decay itself, which is f32: with d' = d (1 + e), |e| <= u,
        # fl(d' acc + sum) is off by u |d acc| + u (|d acc| + sum) to first order
        tol[b, :, :n] = (w * E).sum(0).view(kv, G, n).sum(1) + U[F32] * (2 * got + (2 * old.abs() if decay else 0))
    return out, tol


WEIGHTS = [  # batch, rows, heads, kv, D, cache, lens, type, decay, causal
    (1, 1, 1, 1, 8, 1, [1], BF16, 0.5, True),
    (2, 1, 4, 2, 64, 127, [127, 0], F16, 1.0, True),
    (3, 5, 9, 3, 64, 129, [129, 3, -1], BF16, 0.9, True),      # more rows than tokens; a negative length
    (2, 16, 8, 1, 128, 300, [300, 150], BF16, 0.9, True),      # one full column tile
    (2, 17, 8, 1, 128, 300, [999, 150], F16, 0.0, True),       # one row more; a length above the cache
    (1, 50, 15, 5, 64, 513, [513], BF16, 0.9, True),           # three heads a key head: 126 columns of 128
    (1, 200, 7, 1, 72, 700, [650], F16, 0.9, True),
    (1, 33, 4, 4, 40, 200, [199], BF16, 0.9, False),
    (1, 300, 32, 8, 128, 1000, [1000], BF16, 0.9, True),
    (2, 3, 256, 2, 16, 140, [140, 139], F16, 0.9, True),       # 128 heads a key head
    (2, 1, 16, 2, 128, 20000, [20000, 10001], BF16, 0.9, True),
]


@pytest.mark.parametrize("case", WEIGHTS, ids=lambda c: "x".join(str(v) for v in c[:6]) + str(c[7])[6:])
def test_cache_weights(comp, case):
    B, R, H, kv, D, L, lens, t, decay, causal = case
    g = gen(R + L)
    q, k = (normal(g, B, R, H, D) * 1.5).to(t), normal(g, B, L, kv, D).to(t)
    for b, n in enumerate(lens):
        k[b, max(0, n):] = math.nan
    lse = 1.0 + 3 * torch.rand(B, R, H, generator=g, device="cuda") + math.log(L)
    lse[0, 0, 0] = -math.inf  # a row that saw nothing
    acc = torch.rand(B, kv, L, generator=g, device="cuda")
    if decay == 0:
        acc[:] = math.nan
    before = acc.clone()
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    comp.cache_weights_dev(q, k, ln, lse, acc, decay=decay, causal=causal)
    comp.sync()
    want, tol = weights_ref(q, k, lens, lse, before, D ** -0.5, decay, causal)
    for b, n in enumerate(lens):
        n = max(0, min(n, L))
        err = (acc[b, :, :n].double() - want[b, :, :n]).abs()
        assert (err <= tol[b, :, :n]).all(), float((err - tol[b, :, :n]).max())
        assert torch.equal(acc[b, :, n:].nan_to_num(), before[b, :, n:].nan_to_num())  # (the rest stays)


def test_cache_weights_layouts_and_repeat(comp):
    g = gen(21)
    B, R, H, kv, D, L, t = 2, 40, 6, 2, 64, 260, F16
    q = normal(g, H, B, R, D).to(t).permute(1, 2, 0, 3)
    k = normal(g, kv, B, L, D).to(t).permute(1, 2, 0, 3)
    lens = [260, 200]
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    lse = torch.full((B, R, H), 6.0, device="cuda")
    got = []
    for _ in range(2):
        acc = torch.zeros(kv, B, L + 4, device="cuda").transpose(0, 1)[..., :L]
        comp.cache_weights_dev(q, k, ln, lse, acc, scale=0.2)
        got.append(acc)
    comp.sync()
    assert torch.equal(got[0], got[1])
    want, tol = weights_ref(q, k, lens, lse, torch.zeros(B, kv, L, device="cuda"), 0.2, 1.0, True)
    assert ((got[0].double() - want).abs() <= tol).all()


def test_weights_of_attention_sum_to_one(comp):
    """With lse from the attention, what prefix and own keys receive from a row and head is 1."""
    g = gen(22)
    B, R, H, kv, D, P, L, t = 3, 2, 8, 2, 64, 150, 40, BF16
    q = normal(g, B, R, H, D).to(t)
    kp, vp = normal(g, P, kv, D).to(t), normal(g, P, kv, D).to(t)
    ko, vo = normal(g, B, L, kv, D).to(t), normal(g, B, L, kv, D).to(t)
    ln = torch.tensor([40, 7, 2], dtype=torch.int32, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(B, R, H, device="cuda")
    comp.prefix_attention_dev(q, out, kp, vp, ko, vo, ln, lse)
    own, pre = torch.zeros(B, kv, L, device="cuda"), torch.zeros(1, kv, P, device="cuda")
    comp.cache_weights_dev(q, ko, ln, lse, own)
    comp.cache_weights_dev(q.view(1, B * R, H, D), kp.unsqueeze(0), torch.tensor([P], dtype=torch.int32, device="cuda"),
                           lse.view(1, B * R, H), pre, causal=False)
    comp.sync()
    total = float(own.double().sum() + pre.double().sum())
    # E of these logits is below 2e-5 (|q||k| sums of some 60, times D 2^-23, and lse's own)
    assert abs(total - B * R * H) < 1e-4 * B * R * H


# ---- eviction -----------------------------------------------------------------------------


def evict_ref(acc, n, budget, recent):
    if n <= budget:
        return np.arange(n)
    old = n - recent
    a = acc[:old].astype(np.float64)
    a = np.where(np.isnan(a), -np.inf, a)
    # (a NaN is below -inf: order by that first)
    order = np.lexsort((np.arange(old), -a, np.isnan(acc[:old])))
    return np.concatenate([np.sort(order[:budget - recent]), np.arange(old, n)])


def run_evict(comp, k, v, acc, lens, budget, recent, room=None):
    B, L, kv, D = k.shape
    n = room or max(1, min(budget, L))
    ko, vo = (torch.full((B, n, kv, D), 9.0, dtype=k.dtype, device="cuda") for _ in range(2))
    ao = torch.full((B, kv, n), -5.0, device="cuda")
    ix = torch.full((B, kv, n), -7, dtype=torch.int32, device="cuda")
    lo = torch.full((B,), -1, dtype=torch.int32, device="cuda")
    comp.cache_evict_dev(k, v, acc, torch.tensor(lens, dtype=torch.int32, device="cuda"), ko, vo, ao, ix, lo,
                         budget=budget, recent=recent)
    comp.sync()
    return ko, vo, ao, ix, lo


def check_evict(got, k, v, acc, lens, budget, recent):
    ko, vo, ao, ix, lo = got
    B, L, kv, _ = k.shape
    for b in range(B):
        n = max(0, min(lens[b], L))
        kept = min(n, budget)
        assert int(lo[b]) == kept
        for h in range(kv):
            want = torch.from_numpy(evict_ref(acc[b, h].cpu().numpy(), n, budget, recent)).cuda()
            assert torch.equal(ix[b, h, :kept].long(), want), (b, h)
            assert torch.equal(ko[b, :kept, h], k[b, want, h]) and torch.equal(vo[b, :kept, h], v[b, want, h])
            assert torch.equal(ao[b, h, :kept].view(torch.int32), acc[b, h, want].view(torch.int32))
            assert (ix[b, h, kept:] == -7).all() and (ao[b, h, kept:] == -5).all()
            assert (ko[b, kept:, h] == 9).all() and (vo[b, kept:, h] == 9).all()


EVICT = [  # batch, kv, D, cache, lens, budget, recent, type
    (1, 1, 8, 1, [1], 1, 0, F16),
    (1, 1, 8, 1, [0], 1, 1, F16),
    (2, 3, 64, 100, [100, 40], 60, 7, F16),
    (2, 2, 64, 100, [100, 61], 60, 60, BF16),        # nothing but the newest
    (2, 2, 64, 100, [100, -4], 60, 0, F32),
    (1, 2, 64, 100, [1000], 99, 1, BF16),
    (1, 2, 64, 100, [100], 0, 0, BF16),              # nothing kept
    (1, 2, 40, 100, [100], 200, 3, F16),             # room for more than there is
    (3, 5, 72, 4097, [4097, 4096, 1], 1000, 33, BF16),
    (1, 2, 128, 16385, [16385], 5000, 100, BF16),
    (40, 4, 64, 600, list(range(-10, 590, 15)), 250, 16, F16),
    (1, 1, 16, 140000, [139999], 70001, 64, F16),
    (1, 1, 8, 270000, [270000], 1234, 5, F16),       # a slice longer than a block keeps on chip
]


@pytest.mark.parametrize("case", EVICT, ids=lambda c: "x".join(str(v) for v in (*c[:4], *c[5:7])) + str(c[7])[6:])
def test_cache_evict(comp, case):
    B, kv, D, L, lens, budget, recent, t = case
    g = gen(L + budget)
    k, v = (normal(g, B, L, kv, D).to(t) for _ in range(2))
    acc = torch.exp(2 * normal(g, B, kv, L))
    acc[torch.rand(B, kv, L, generator=g, device="cuda") < 0.2] = 0.25  # equal ones among them
    check_evict(run_evict(comp, k, v, acc, lens, budget, recent), k, v, acc, lens, budget, recent)


@pytest.mark.parametrize("L", [300, 9000])
@pytest.mark.parametrize("kind", ["equal", "zeros", "special", "negative", "close"])
def test_cache_evict_orders(comp, kind, L):
    """Equal weights go by place; -0 is 0, a NaN is below -inf; neighbouring floats are told apart."""
    g = gen(L)
    k, v = (normal(g, 2, L, 2, 16).to(F16) for _ in range(2))
    acc = torch.full((2, 2, L), 0.5, device="cuda")
    if kind == "zeros":
        acc = torch.where(torch.rand(2, 2, L, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    elif kind == "special":
        pick = torch.randint(0, 6, (2, 2, L), generator=g, device="cuda")
        acc = torch.tensor([math.nan, math.inf, -math.inf, 1e-45, -1e-45, 0.0], device="cuda")[pick]
    elif kind == "negative":
        acc = normal(g, 2, 2, L)
    elif kind == "close":
        acc = (torch.randint(0, 40, (2, 2, L), generator=g, device="cuda", dtype=torch.int32) + 0x3F800000).view(F32)
    lens = [L, L - 13]
    check_evict(run_evict(comp, k, v, acc, lens, L // 3, 11), k, v, acc, lens, L // 3, 11)


def test_cache_evict_layouts(comp):
    """Head-major caches, keys and values of one buffer, outputs with more room than the budget."""
    g = gen(31)
    B, kv, D, L = 2, 3, 64, 200
    kvs = normal(g, kv, B, L, 2, D).to(BF16)
    k, v = (kvs[:, :, :, i].permute(1, 2, 0, 3) for i in range(2))
    acc = torch.rand(kv, B, L + 3, generator=g, device="cuda").transpose(0, 1)[..., :L]
    lens = [200, 150]
    check_evict(run_evict(comp, k, v, acc, lens, 90, 10, room=130), k, v, acc, lens, 90, 10)


# ---- refusals of the library ----------------------------------------------------------------


def z(*shape, t=F16):
    return torch.zeros(*shape, dtype=t, device="cuda")


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_library_refuses(P, comp):
    """Arguments that only the library looks at: refused before anything is launched."""
    before = comp.L.dc_launch_count()

    def refused(call, match):
        with pytest.raises(P.DeviceError, match=match):
            call()

    r = dict(x=z(2, 64 * 4, t=F32), pos=i32(0, 1), q=z(2, 2, 64), k=z(2, 1, 64), v=z(2, 1, 64))
    refused(lambda: comp.head_norm_rope_dev(**{**r, "rot": 12}), "multiples of 8")
    refused(lambda: comp.head_norm_rope_dev(**{**r, "rot": 72}), "multiples of 8")
    refused(lambda: comp.head_norm_rope_dev(**{**r, "sections": [31]}), "sections")
    refused(lambda: comp.head_norm_rope_dev(**{**r, "pos": z(2, 2, t=torch.int32), "sections": [33, -1]}), "section")
    refused(lambda: comp.head_norm_rope_dev(**{**r, "pos": z(3, 2, t=torch.int32), "sections": [8, 12, 12], "cyclic": True}),
            "cyclic")
    refused(lambda: comp.head_norm_rope_dev(**{**r, "eps": -1.0}), "eps")
    refused(lambda: comp.head_norm_rope_dev(**{**r, "theta": 0.0}), "theta")
    refused(lambda: comp.head_norm_rope_dev(**{**r, "k": z(1, 1, 64), "v": z(1, 1, 64)}), "rows for a cache")
    refused(lambda: comp.head_norm_rope_dev(**{**r, "v": r["k"]}), "overlaps")
    x = z(2, 64 * 4)
    refused(lambda: comp.head_norm_rope_dev(x, r["pos"], x.view(4, 2, 64)[:2], r["k"], r["v"]), "overlaps")
    refused(lambda: comp.head_norm_rope_dev(z(1, 12 * 3, t=F32), i32(0), z(1, 1, 12), z(1, 1, 12), z(1, 1, 12), rot=8),
            "multiples of 8")

    a = dict(q=z(2, 1, 4, 64), out=z(2, 1, 4, 64), k_pre=z(5, 2, 64), v_pre=z(5, 2, 64))
    refused(lambda: comp.prefix_attention_dev(**{**a, "scale": 0.0}), "scale")
    refused(lambda: comp.prefix_attention_dev(**{**a, "scale": math.nan}), "scale")
    refused(lambda: comp.prefix_attention_dev(z(1, 17, 4, 64), z(1, 17, 4, 64), a["k_pre"], a["v_pre"]), "rows 17")
    refused(lambda: comp.prefix_attention_dev(z(1, 1, 3, 64), z(1, 1, 3, 64), a["k_pre"], a["v_pre"]), "heads")
    refused(lambda: comp.prefix_attention_dev(z(1, 1, 2, 136), z(1, 1, 2, 136), z(5, 2, 136), z(5, 2, 136)), "head_dim")
    refused(lambda: comp.prefix_attention_dev(z(1, 1, 2, 12), z(1, 1, 2, 12), z(5, 2, 12), z(5, 2, 12)), "head_dim")
    refused(lambda: comp.prefix_attention_dev(z(1, 1, 2, 64, t=F32), z(1, 1, 2, 64, t=F32), z(5, 2, 64, t=F32),
                                              z(5, 2, 64, t=F32)), "type")
    refused(lambda: comp.prefix_attention_dev(a["q"], z(2, 1, 4, 64, t=BF16), a["k_pre"], a["v_pre"]), "type")
    refused(lambda: comp.prefix_attention_dev(a["q"], a["out"], z(5 * 128 + 1)[1:].view(5, 2, 64), a["v_pre"]), "16-byte")
    refused(lambda: comp.prefix_attention_dev(a["q"], a["q"], a["k_pre"], a["v_pre"]), "overlaps")
    refused(lambda: comp.prefix_attention_dev(**{**a, "ws": z(64, t=torch.uint8)}), "workspace")
    need = comp.prefix_attention_ws(**a)
    refused(lambda: comp.prefix_attention_dev(**{**a, "ws": z(need + 1, t=torch.uint8)[1:]}), "workspace")

    w = dict(q=z(2, 1, 4, 64), k=z(2, 5, 2, 64), lens=i32(5, 5), lse=z(2, 1, 4, t=F32), acc=z(2, 2, 5, t=F32))
    refused(lambda: comp.cache_weights_dev(**w, scale=-1.0), "scale")
    refused(lambda: comp.cache_weights_dev(**w, decay=math.inf), "decay")
    refused(lambda: comp.cache_weights_dev(**{**w, "q": z(2, 0, 4, 64), "lse": z(2, 0, 4, t=F32)}), "rows 0")
    refused(lambda: comp.cache_weights_dev(**{**w, "q": z(2, 1, 258, 64), "lse": z(2, 1, 258, t=F32)}), "heads")
    refused(lambda: comp.cache_weights_dev(**{**w, "lse": w["acc"].view(-1)[:8].view(2, 1, 4)}), "overlaps")

    e = dict(k=z(2, 9, 2, 64), v=z(2, 9, 2, 64), acc=z(2, 2, 9, t=F32), lens=i32(9, 9), k_out=z(2, 4, 2, 64),
             v_out=z(2, 4, 2, 64), acc_out=z(2, 2, 4, t=F32), index=z(2, 2, 4, t=torch.int32), lens_out=i32(0, 0))
    refused(lambda: comp.cache_evict_dev(**e, budget=4, recent=5), "recent")
    refused(lambda: comp.cache_evict_dev(**e, budget=4, recent=-1), "recent")
    refused(lambda: comp.cache_evict_dev(**e, budget=-1), "budget")
    refused(lambda: comp.cache_evict_dev(**{**e, "k_out": e["k"][:, :4]}, budget=4), "overlaps")
    refused(lambda: comp.cache_evict_dev(**{**e, "v_out": e["k_out"]}, budget=4), "overlap")
    refused(lambda: comp.cache_evict_dev(**{**e, "lens_out": e["lens"]}, budget=4), "overlaps")
    refused(lambda: comp.cache_evict_dev(**{**e, **{n: z(2, 9, 2, 12) for n in ("k", "v")},
                                            **{n: z(2, 4, 2, 12) for n in ("k_out", "v_out")}}, budget=4), "rows of 12")
    assert comp.L.dc_launch_count() == before


def test_empty_calls_do_nothing(comp):
    before = comp.L.dc_launch_count()
    comp.head_norm_rope_dev(z(0, 256, t=F32), z(0, t=torch.int32), z(0, 2, 64), z(3, 1, 64), z(3, 1, 64))
    comp.prefix_attention_dev(z(0, 1, 4, 64), z(0, 1, 4, 64), z(5, 2, 64), z(5, 2, 64))
    comp.cache_weights_dev(z(0, 1, 4, 64), z(0, 5, 2, 64), z(0, t=torch.int32), z(0, 1, 4, t=F32), z(0, 2, 5, t=F32))
    comp.cache_evict_dev(z(0, 9, 2, 64), z(0, 9, 2, 64), z(0, 2, 9, t=F32), z(0, t=torch.int32), z(0, 4, 2, 64),
                         z(0, 4, 2, 64), z(0, 2, 4, t=F32), z(0, 2, 4, t=torch.int32), z(0, t=torch.int32), budget=4)
    comp.sync()
    assert comp.L.dc_launch_count() == before


# ---- streams, graphs, and the operators in a row ----------------------------------------------


class Layer:
    """One attention layer of a batch on resident int8 weights: projection, rotation and append,
    attention, projection, weights, and eviction of the own caches above a length."""

    def __init__(self, comp, g, B, H, kv, D, hidden, P, L, t):
        self.comp, self.t, self.H, self.kv, self.D, self.hidden = comp, t, H, kv, D, hidden
        w = lambda k, n: comp.register_weight((normal(g, k, n) / math.sqrt(k)).cpu().numpy(), k, n)  # noqa: E731
        self.qkv, self.o = w(hidden, (H + 2 * kv) * D), w(H * D, hidden)
        self.wq, self.wk = 1 + 0.1 * normal(g, D), 1 + 0.1 * normal(g, D)
        self.kp, self.vp = z(P, kv, D, t=t), z(P, kv, D, t=t)
        self.k, self.v, self.acc = z(B, L, kv, D, t=t), z(B, L, kv, D, t=t), z(B, kv, L, t=F32)
        self.lens = z(B, t=torch.int32)
        self.B, self.L = B, L

    def project(self, x):
        rows = x.shape[0]
        out = torch.empty(rows, (self.H + 2 * self.kv) * self.D, device="cuda")
        self.comp.vgemm_dev(x, rows, self.qkv, 0, out)
        return out

    def prefill(self, x):
        rows = self.project(x)
        q = z(x.shape[0], self.H, self.D, t=self.t)
        self.comp.head_norm_rope_dev(rows, torch.arange(x.shape[0], dtype=torch.int32, device="cuda"), q, self.kp, self.vp,
                                     wq=self.wq, wk=self.wk)

    def step(self, x, pos, slots, hidden):
        """x (batch, hidden): one token of each sequence; lens already counts it."""
        rows = self.project(x)
        q = torch.empty(self.B, 1, self.H, self.D, dtype=self.t, device="cuda")
        self.comp.head_norm_rope_dev(rows, pos, q.view(self.B, self.H, self.D), self.k, self.v, slots=slots, wq=self.wq,
                                     wk=self.wk)
        att = torch.empty(self.B, 1, self.H, self.D, device="cuda")
        lse = torch.empty(self.B, 1, self.H, device="cuda")
        self.comp.prefix_attention_dev(q, att, self.kp, self.vp, self.k, self.v, self.lens, lse)
        self.comp.vgemm_dev(att, self.B, self.o, 0, hidden)
        self.comp.cache_weights_dev(q, self.k, self.lens, lse, self.acc, decay=0.9)
        return rows, q, att, lse


def test_operators_in_a_row(comp):
    """A batch behind one prompt: prefill, steps, an eviction, more steps; each part against 64 bits on
    what the part before gave."""
    g = gen(41)
    B, H, kv, D, hidden, P, L, t = 3, 8, 2, 64, 256, 70, 12, BF16
    lay = Layer(comp, g, B, H, kv, D, hidden, P, L, t)
    lay.prefill(normal(g, P, hidden))
    base = torch.arange(B, device="cuda") * L
    lens, place = [0] * B, [0] * B
    for step in range(9):
        lens = [n + 1 for n in lens]
        place = [n + 1 for n in place]
        lay.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        pos = torch.tensor([P + n - 1 for n in place], dtype=torch.int32, device="cuda")
        slots = base + torch.tensor([n - 1 for n in lens], device="cuda")
        hidden_out = torch.empty(B, hidden, device="cuda")
        before = lay.acc.clone()
        rows, q, att, lse = lay.step(normal(g, B, hidden), pos, slots, hidden_out)
        comp.sync()
        rq, rk, rv, size = rope_ref(rows, pos, H, kv, D, D, [D // 2], False, lay.wq, lay.wk, 1e-5, 1e4)
        check_rope(q.view(B, H, D), rq, size[0], D, t)
        check_rope(lay.k.view(B * L, kv, D)[slots], rk, size[1], D, t)
        check_attention(att, lse, attention_ref(q, lay.kp, lay.vp, lay.k, lay.v, lens, D ** -0.5), t, 20.0)
        want, tol = weights_ref(q, lay.k, lens, lse, before, D ** -0.5, 0.9, True)
        assert ((lay.acc.double() - want).abs() <= tol).all()
        assert torch.isfinite(hidden_out).all()
        if lens[0] == 6:
            old = (lay.k, lay.v, lay.acc)
            new = (z(B, L, kv, D, t=t), z(B, L, kv, D, t=t), z(B, kv, L, t=F32))
            index, out = z(B, kv, L, t=torch.int32), z(B, t=torch.int32)
            comp.cache_evict_dev(*old, lay.lens, *new, index, out, budget=4, recent=2)
            comp.sync()
            for b in range(B):
                for h in range(kv):
                    want = torch.from_numpy(evict_ref(old[2][b, h].cpu().numpy(), 6, 4, 2)).cuda()
                    assert torch.equal(index[b, h, :4].long(), want)
                    assert torch.equal(new[0][b, :4, h], old[0][b, want, h])
            lay.k, lay.v, lay.acc = new
            lens = out.tolist()


def test_capture_replay_and_two_graphs(comp, P):
    """The four calls in two captured graphs, replayed at once on two streams: the results of eager calls."""
    sides = []
    for i in range(2):
        core = P.init_compute(0)
        g = gen(50 + i)
        B, H, kv, D, Pn, L, t = 5, 8, 2, 128, 1500, 300, BF16
        s = dict(core=core, x=normal(g, B, (H + 2 * kv) * D), pos=torch.randint(0, 4000, (B,), generator=g, device="cuda",
                                                                              dtype=torch.int32),
                 q=z(B, H, D, t=t), k=normal(g, B, L, kv, D).to(t), v=normal(g, B, L, kv, D).to(t),
                 kp=normal(g, Pn, kv, D).to(t), vp=normal(g, Pn, kv, D).to(t), lens=i32(300, 1, 50, 299, 0),
                 slots=torch.arange(B, device="cuda") * L + 7, out=z(B, 1, H, D, t=t), lse=z(B, 1, H, t=F32),
                 acc=torch.rand(B, kv, L, generator=g, device="cuda"), ko=z(B, 64, kv, D, t=t), vo=z(B, 64, kv, D, t=t),
                 ao=z(B, kv, 64, t=F32), ix=z(B, kv, 64, t=torch.int32), lo=z(B, t=torch.int32))
        sides.append(s)

    def calls(s):
        c = s["core"]
        c.head_norm_rope_dev(s["x"], s["pos"], s["q"], s["k"], s["v"], slots=s["slots"])
        c.prefix_attention_dev(s["q"].unsqueeze(1), s["out"], s["kp"], s["vp"], s["k"], s["v"], s["lens"], s["lse"])
        c.cache_weights_dev(s["q"].unsqueeze(1), s["k"], s["lens"], s["lse"], s["acc"], decay=0.0)
        c.cache_evict_dev(s["k"], s["v"], s["acc"], s["lens"], s["ko"], s["vo"], s["ao"], s["ix"], s["lo"], budget=64,
                          recent=8)

    names = ("q", "k", "v", "out", "lse", "acc", "ko", "vo", "ao", "ix", "lo")
    torch.cuda.synchronize()
    graphs = []
    for s in sides:
        calls(s)  # (on the context's own stream)
        s["core"].sync()
        s["want"] = {n: s[n].clone() for n in names}
        for n in ("out", "lse"):
            s[n].fill_(3.0)
        for n in ("ko", "vo", "ao", "ix", "lo"):
            s[n].zero_()  # (as they began: what lies behind a sequence's kept tokens stays)
        held = torch.arange(L, device="cuda") < s["lens"].view(B, 1, 1)
        s["acc"].copy_(torch.where(held, 3.0, s["acc"]))
        torch.cuda.synchronize()
        s["stream"] = torch.cuda.Stream()
        s["core"].set_stream(s["stream"])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s["stream"]):
            calls(s)
        graphs.append(graph)
    for _ in range(3):
        for s, graph in zip(sides, graphs):
            with torch.cuda.stream(s["stream"]):
                graph.replay()
    torch.cuda.synchronize()
    for s in sides:
        for n in names:
            assert torch.equal(s[n], s["want"][n]), n
        s["core"].sync()
    del graphs
    for s in sides:
        s["core"].close()


def test_calls_follow_the_stream_they_are_on(comp, P):
    """A context on a stream of its own: its calls come behind that stream's earlier work."""
    core = P.init_compute(0)
    stream = torch.cuda.Stream()
    core.set_stream(stream)
    g = gen(60)
    kp, vp = normal(g, 4000, 2, 64).to(BF16), normal(g, 4000, 2, 64).to(BF16)
    q0 = normal(g, 20, 1, 8, 64).to(BF16)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        a = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            a = a @ a * 1e-4
        q = torch.where(torch.isnan(a[0, 0]), q0, q0)  # (there only once the products are done)
        out = torch.empty_like(q)
    core.prefix_attention_dev(q, out, kp, vp)
    core.sync()
    check_attention(out, None, attention_ref(q0, kp, vp, None, None, None, 0.125), BF16, 6.0)
    core.close()
