"""The cache operators at the ends of what their arguments may hold, against 64 bits."""
import math

import pytest
import torch

from test_cache_gpu import BF16, F16, F32, U, attention_ref, check_attention, gen, i32, normal, weights_ref, z

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B, kv", [(4, 2), (60, 2)], ids=["few rows", "shared"])
@pytest.mark.parametrize("D", [64, 128])
def test_f16_keeps_what_lies_far_below_the_maximum(comp, B, kv, D):
    """One key in 16 takes nearly all weight and has the value 0; the others weigh 2^-26 of it and have large values.

    With the exponent shifted so that a row's maximum is 2^7, a probability below f16's normal range is off
    by half of its smallest step, 2^-25, so by 2^-32 of the maximum: out is off by 2^-32 sum |v| / sum p beside
    its relative bounds.  (Unshifted, 2^-26 rounds to 0 and the output with it.)"""
    g = gen(B + D)
    P, H = 1024, 2 * kv
    x = torch.zeros(P, device="cuda")
    x[::16] = 18.015625
    kp = z(P, kv, D)
    kp[..., 0] = x.to(F16).view(P, 1)
    vp = (20000 + 20000 * torch.rand(P, kv, D, generator=g, device="cuda")).to(F16)
    vp[::16] = 0
    q = z(B, 1, H, D)
    q[..., 0] = 1
    out, lse = torch.empty(B, 1, H, D, device="cuda"), torch.empty(B, 1, H, device="cuda")
    comp.prefix_attention_dev(q, out, kp, vp, lse=lse, scale=1.0)
    comp.sync()
    want, wlse, mag, E, n = attention_ref(q[:1], kp, vp, None, None, None, 1.0)
    p = torch.exp(x.double() - x.double().max())
    tol = (U[F16] + E.unsqueeze(-1)) * mag + 2.0 ** -32 * vp.double().sum(0).amax() / p.sum() + 4 * U[F32] * mag
    assert (tol < 0.1 * want).all()  # (the bound says something)
    err = (out.double() - want).abs()
    assert (err <= tol).all(), (float(err.max()), float(want.max()))
    assert ((lse.double() - wlse).abs() <= E + n * U[F32] + 4 * U[F32] * wlse.abs()).all()


@pytest.mark.parametrize("prefix", [0, 70])
@pytest.mark.parametrize("R", [1, 4, 16])
def test_attention_of_the_lowest_lengths(comp, prefix, R):
    """A length is taken as at least 0, however far below it lies."""
    g = gen(prefix + R)
    lens = [-2 ** 31, -2 ** 31 + 1, -2 ** 31 + R - 1, -1, 100]
    B, H, kv, D, L, t = len(lens), 4, 2, 64, 100, BF16
    q = normal(g, B, R, H, D).to(t)
    kp, vp = (normal(g, prefix, kv, D).to(t) if prefix else None for _ in range(2))
    ko, vo = normal(g, B, L, kv, D).to(t), normal(g, B, L, kv, D).to(t)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(B, R, H, device="cuda")
    comp.prefix_attention_dev(q, out, kp, vp, ko, vo, ln, lse)
    comp.sync()
    check_attention(out, lse, attention_ref(q, kp, vp, ko, vo, lens, D ** -0.5), t, 6.0)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("R, H, kv, D, L, causal", [
    (4, 8, 2, 64, 300, False), (4, 8, 2, 128, 300, True), (128, 2, 2, 128, 200, False),   # few rows
    (300, 8, 2, 64, 300, False), (200, 15, 5, 128, 260, True)])                            # many
def test_weights_of_rows_that_are_left_out(comp, R, H, kv, D, L, causal, bad):
    """A row of lse -inf adds nothing, whatever its queries hold: a batch's padding is left out that way."""
    g = gen(R + D)
    B, t = 2, BF16
    q, k = normal(g, B, R, H, D).to(t), normal(g, B, L, kv, D).to(t)
    lse = 1.0 + 3 * torch.rand(B, R, H, generator=g, device="cuda") + math.log(L)
    out = torch.rand(B, R, H, generator=g, device="cuda") < 0.2
    out[0, 0, 0] = out[1, R - 1, H - 1] = True
    lse[out] = -math.inf
    q[out] = bad
    acc = torch.rand(B, kv, L, generator=g, device="cuda")
    before, lens = acc.clone(), [L, L - 70]
    comp.cache_weights_dev(q, k, torch.tensor(lens, dtype=torch.int32, device="cuda"), lse, acc, decay=0.9, causal=causal)
    comp.sync()
    want, tol = weights_ref(torch.where(out.unsqueeze(-1), 0.0, q), k, lens, lse, before, D ** -0.5, 0.9, causal)
    assert ((acc.double() - want).abs() <= tol).all()


def test_outputs_that_overlap_themselves_are_refused(P, comp):
    """Expanded outputs, and values a token behind their keys: refused before anything is launched.  Interleaved
    and permuted ones are taken."""
    before = comp.L.dc_launch_count()

    def refused(call, match):
        with pytest.raises(P.DeviceError, match=match):
            call()

    r = dict(x=z(2, 64 * 4, t=F32), pos=i32(0, 1), q=z(2, 2, 64), k=z(2, 1, 64), v=z(2, 1, 64))
    for name in ("q", "k", "v"):
        refused(lambda: comp.head_norm_rope_dev(**{**r, name: r[name][:1].expand_as(r[name])}), "share an address")
    line = z(3, 1, 64)
    refused(lambda: comp.head_norm_rope_dev(**{**r, "k": line[:2], "v": line[1:]}), "overlaps")

    a = dict(q=z(2, 1, 4, 64), k_pre=z(5, 2, 64), v_pre=z(5, 2, 64))
    refused(lambda: comp.prefix_attention_dev(out=z(1, 1, 4, 64).expand(2, 1, 4, 64), **a), "share an address")
    refused(lambda: comp.prefix_attention_dev(out=z(2, 1, 1, 64).expand(2, 1, 4, 64), **a), "share an address")

    w = dict(q=z(2, 1, 4, 64), k=z(2, 5, 2, 64), lens=i32(5, 5), lse=z(2, 1, 4, t=F32))
    refused(lambda: comp.cache_weights_dev(acc=z(2, 1, 5, t=F32).expand(2, 2, 5), **w), "share an address")
    refused(lambda: comp.cache_weights_dev(acc=z(1, 2, 5, t=F32).expand(2, 2, 5), **w), "share an address")
    refused(lambda: comp.cache_weights_dev(acc=z(24, t=F32).as_strided((2, 2, 5), (10, 4, 1)), **w), "share an address")

    e = dict(k=z(2, 9, 2, 64), v=z(2, 9, 2, 64), acc=z(2, 2, 9, t=F32), lens=i32(9, 9), k_out=z(2, 4, 2, 64),
             v_out=z(2, 4, 2, 64), acc_out=z(2, 2, 4, t=F32), index=z(2, 2, 4, t=torch.int32), lens_out=i32(0, 0))
    for name in ("k_out", "v_out", "acc_out", "index"):
        refused(lambda: comp.cache_evict_dev(**{**e, name: e[name][:1].expand_as(e[name])}, budget=4), "share an address")
    line = z(2, 5, 2, 64)
    refused(lambda: comp.cache_evict_dev(**{**e, "k_out": line[:, :4], "v_out": line[:, 1:]}, budget=4), "overlap")
    assert comp.L.dc_launch_count() == before
    comp.cache_evict_dev(**{**e, "k_out": (both := z(2, 4, 2, 2, 64))[:, :, 0], "v_out": both[:, :, 1]}, budget=4)
    comp.cache_evict_dev(**{**e, "k_out": (both := z(2, 4, 2, 2, 64))[..., 0, :], "v_out": both[..., 1, :]}, budget=4)
    comp.sync()


def test_workspace_size_is_refused_as_the_call_is(P, comp):
    """prefix_attention_ws raises what the call would raise, and is 0 only where nothing is needed."""
    kv = dict(k_pre=z(5, 2, 64), v_pre=z(5, 2, 64))
    with pytest.raises(P.DeviceError, match="rows 17"):
        comp.prefix_attention_ws(z(1, 17, 4, 64), z(1, 17, 4, 64), **kv)
    with pytest.raises(P.DeviceError, match="scale"):
        comp.prefix_attention_ws(z(1, 1, 4, 64), z(1, 1, 4, 64), scale=0.0, **kv)
    assert comp.prefix_attention_ws(z(0, 1, 4, 64), z(0, 1, 4, 64), **kv) == 0
    assert comp.prefix_attention_ws(z(2, 1, 4, 64), z(2, 1, 4, 64)) == 0
    with pytest.raises(P.DeviceError, match="rows 17"):
        comp.prefix_attention_ws(z(0, 17, 4, 64), z(0, 17, 4, 64), **kv)
    assert comp.prefix_attention_ws(z(2, 1, 4, 64), z(2, 1, 4, 64), **kv) > 0


def test_rope_outputs_over_what_it_reads_are_refused(P, comp):
    """Positions, slots and weights that lie in an output: refused before anything is launched."""
    before = comp.L.dc_launch_count()
    t = z(2, 2, 64, t=F32)
    r = dict(x=z(2, 64 * 4, t=F32), pos=z(2, t=torch.int32), q=t, k=z(2, 1, 64, t=F32), v=z(2, 1, 64, t=F32),
             slots=z(2, t=torch.int64), wq=z(64, t=F32), wk=z(64, t=F32))
    for name in ("q", "k", "v"):
        out = r[name].view(-1)
        for change in (dict(pos=out[8:10].view(torch.int32)), dict(slots=out[4:8].view(torch.int64)), dict(wq=out[:64]),
                       dict(wk=out[-64:])):
            with pytest.raises(P.DeviceError, match="overlaps"):
                comp.head_norm_rope_dev(**{**r, **change})
    assert comp.L.dc_launch_count() == before


def test_rope_with_the_same_positions_on_all_axes(comp):
    """Text between images has one position on every axis, as an expanded tensor."""
    g = gen(70)
    x, pos = normal(g, 5, 6 * 64), torch.arange(5, dtype=torch.int32, device="cuda") * 100
    got = []
    for p in (pos.expand(3, 5), pos.expand(3, 5).contiguous()):
        q, k, v = (z(5, n, 64, t=F32) for n in (4, 1, 1))
        comp.head_norm_rope_dev(x, p, q, k, v, sections=[16, 8, 8])
        got.append((q, k, v))
    comp.sync()
    assert all(torch.equal(a, b) for a, b in zip(*got)) and (got[0][0] != 0).any()


@pytest.mark.parametrize("B", [3, 40], ids=["few rows", "shared"])
def test_expanded_inputs(comp, B):
    """Keys and values that all heads or all sequences share, and one query for a batch, as expanded tensors: the
    bits of their copies."""
    g = gen(B + 80)
    H, kv, D, P, L, t = 8, 4, 64, 700, 90, BF16
    kp, vp = (normal(g, P, 1, D).to(t).expand(P, kv, D) for _ in range(2))
    ko, vo = (normal(g, 1, L, kv, D).to(t).expand(B, L, kv, D) for _ in range(2))
    q = normal(g, 1, 2, H, D).to(t).expand(B, 2, H, D)
    ln = torch.arange(B, dtype=torch.int32, device="cuda") * 5 % 91
    got = []
    for same in (lambda x: x, lambda x: x.contiguous()):
        out, lse = torch.empty(B, 2, H, D, device="cuda"), torch.empty(B, 2, H, device="cuda")
        comp.prefix_attention_dev(same(q), out, same(kp), same(vp), same(ko), same(vo), ln, lse)
        acc = torch.zeros(B, kv, L, device="cuda")
        comp.cache_weights_dev(same(q), same(ko), ln, lse, acc)
        rows = torch.zeros(1, kv, P, device="cuda")  # (the prefix, against 2 B rows)
        comp.cache_weights_dev(same(q[:, :1].transpose(0, 1)), same(kp.unsqueeze(0)), i32(P), lse[:, 0].contiguous().unsqueeze(0),
                               rows, causal=False)
        got.append((out, lse, acc, rows))
    comp.sync()
    assert all(torch.equal(a, b) for a, b in zip(*got)) and all((a != 0).any() for a in got[0])


@pytest.mark.parametrize("case", [(5, 8, 2, 64, 2000), (50, 32, 8, 128, 300), (3, 15, 5, 64, 40)],
                         ids=["few rows", "shared", "short"])
def test_calls_on_two_streams_at_once(P, comp, case):
    """Two contexts on two streams, calls of all four operators in flight together: the bits of calls one by one."""
    B, H, kv, D, n = case
    sides = []
    for i in range(2):
        g = gen(90 + i + B)
        t = BF16
        s = dict(x=normal(g, B, (H + 2 * kv) * D), pos=torch.arange(B, dtype=torch.int32, device="cuda"),
                 k=normal(g, B, 200, kv, D).to(t), v=normal(g, B, 200, kv, D).to(t), kp=normal(g, n, kv, D).to(t),
                 vp=normal(g, n, kv, D).to(t), lens=(torch.arange(B, device="cuda") * 37 % 201).int(),
                 slots=torch.arange(B, device="cuda") * 200 + 3, acc0=torch.rand(B, kv, 200, generator=g, device="cuda"))
        s["core"], s["stream"] = P.init_compute(0), torch.cuda.Stream()
        sides.append(s)

    def calls(s, core):
        t = BF16
        q, out, lse = z(B, 1, H, D, t=t), z(B, 1, H, D, t=F32), z(B, 1, H, t=F32)
        acc = s["acc0"].clone()
        ko, vo, ao, ix, lo = z(B, 50, kv, D, t=t), z(B, 50, kv, D, t=t), z(B, kv, 50, t=F32), z(B, kv, 50, t=torch.int32), z(
            B, t=torch.int32)
        core.head_norm_rope_dev(s["x"], s["pos"], q.view(B, H, D), s["k"], s["v"], slots=s["slots"])
        core.prefix_attention_dev(q, out, s["kp"], s["vp"], s["k"], s["v"], s["lens"], lse)
        core.cache_weights_dev(q, s["k"], s["lens"], lse, acc, decay=0.5)
        core.cache_evict_dev(s["k"], s["v"], acc, s["lens"], ko, vo, ao, ix, lo, budget=50, recent=9)
        return q, out, lse, acc, ko, vo, ao, ix, lo

    want = [calls(s, comp) for s in sides]
    torch.cuda.synchronize()
    for s in sides:
        s["core"].set_stream(s["stream"])
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(sides):
            with torch.cuda.stream(s["stream"]):
                got[i].append(calls(s, s["core"]))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[i]))
        sides[i]["core"].sync()
        sides[i]["core"].close()


def test_offsets_beyond_32_bits(comp):
    """Tokens 2^24 elements apart in a buffer beyond 2^32: the results of a compact cache, to the bit."""
    g = gen(99)
    B, H, kv, D, L, t, far = 2, 8, 2, 64, 150, BF16, 1 << 24
    whole = torch.empty(B * L * far + far, dtype=t, device="cuda")
    assert whole.numel() > 1 << 32
    k, v = (whole.as_strided((B, L, kv, D), (L * far, far, 2 * D, 1), at) for at in (0, D))
    near = [normal(g, B, L, kv, D).to(t) for _ in range(2)]
    x, pos = normal(g, 4, (H + 2 * kv) * D), torch.arange(4, dtype=torch.int32, device="cuda")
    slots = torch.tensor([0, L - 1, L + 7, 2 * L - 1], device="cuda")
    lens, got = i32(L, L - 3), []
    for kk, vv in ((k, v), near):
        kk.copy_(near[0]), vv.copy_(near[1])
        q = z(4, H, D, t=t)
        comp.head_norm_rope_dev(x, pos, q, kk, vv, slots=slots)
        q = q.view(2, 2, H, D)
        out, lse = torch.empty(B, 2, H, D, device="cuda"), torch.empty(B, 2, H, device="cuda")
        comp.prefix_attention_dev(q, out, kk[1], vv[1], kk, vv, lens, lse)
        acc = torch.zeros(B, kv, L, device="cuda")
        comp.cache_weights_dev(q, kk, lens, lse, acc)
        many = torch.zeros(1, kv, L, device="cuda")
        comp.cache_weights_dev(q.view(1, 4, H, D).repeat(1, 20, 1, 1), kk[1:], i32(L),
                               lse.view(1, 4, H).repeat(1, 20, 1), many, causal=False)
        ko, vo = z(B, 40, kv, D, t=t), z(B, 40, kv, D, t=t)
        outs = (z(B, kv, 40, t=F32), z(B, kv, 40, t=torch.int32), i32(0, 0))
        comp.cache_evict_dev(kk, vv, acc, lens, ko, vo, *outs, budget=40, recent=5)
        got.append((q, out, lse, acc, many, ko, vo, *outs, kk.clone(), vv.clone()))
    comp.sync()
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_eviction_to_offsets_beyond_32_bits(comp):
    """Kept tokens and their weights and places, as far apart."""
    g = gen(100)
    B, kv, D, L, t, far = 1, 2, 64, 300, BF16, 1 << 24
    k, v = (normal(g, B, L, kv, D).to(t) for _ in range(2))
    acc = torch.rand(B, kv, L, generator=g, device="cuda")
    whole = torch.empty(140 * far, dtype=t, device="cuda")
    words = torch.empty((1 << 32) + 512, dtype=torch.int32, device="cuda")
    got = []
    for wide in (True, False):
        if wide:
            ko, vo = (whole.as_strided((B, 130, kv, D), (130 * far, far, 2 * D, 1), at) for at in (0, D))
            ix, ao = words[:(1 << 31) + 256], words[(1 << 31) + 256:].view(F32)
            ix, ao = (b.as_strided((B, kv, 130), (1 << 31, 1 << 31, 1)) for b in (ix, ao))
        else:
            ko, vo, ix, ao = z(B, 130, kv, D, t=t), z(B, 130, kv, D, t=t), z(B, kv, 130, t=torch.int32), z(B, kv, 130, t=F32)
        lo = i32(0)
        comp.cache_evict_dev(k, v, acc, i32(L), ko, vo, ao, ix, lo, budget=130, recent=20)
        got.append((ko.clone(), vo.clone(), ao.clone(), ix.clone(), lo))
    comp.sync()
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("B, heads", [(3, 4), (40, 2), (40, 150), (200, 130)],
                         ids=["few rows", "shared", "many tiles", "two tiles of rows"])
@pytest.mark.parametrize("t, q0, k0", [(F16, 2.0 ** 4, 2.0 ** 15), (F16, 2.0 ** 10, 2.0 ** 15), (F16, 2.0 ** 15, 2.0 ** 15),
                                       (F16, -2.0 ** 15, 2.0 ** 15), (BF16, 2.0 ** 20, 2.0 ** 14), (BF16, 2.0 ** 50, 2.0 ** 50),
                                       (BF16, -2.0 ** 50, 2.0 ** 50)], ids=str)
@pytest.mark.parametrize("D", [64, 128])
def test_attention_of_far_scores(comp, D, t, q0, k0, B, heads):
    """Scores far from 0, as exact products of one channel: those of the largest are equal, the next lies 2^-4 of it
    below, so each row is the mean of the values that have the largest, off by the roundings of
    the probabilities (equal ones: none), the output (f32) and a sum of up to 1024 terms, and lse is the largest to f32."""
    g = gen(B + heads)
    P, L, R = 700, 90, 2
    pick = torch.randint(0, 6, (P + L,), generator=g, device="cuda")
    pick[3], pick[P + 5] = 5, 5  # (each cache has the largest, the first two drafts' common tokens too)
    value = torch.tensor([1.0, 1.125, 1.25, 1.5, 1.75, 1.875], device="cuda")[pick] * k0
    if q0 < 0:  # (the largest score is then the one nearest to 0, below it)
        value = torch.where(pick == 5, 1.0 * k0, value * 1.0625)
    k, v = z(P + L, heads, D, t=t), normal(g, P + L, heads, D).to(t)
    k[..., 0] = value.to(t).view(-1, 1)
    q = z(B, R, heads, D, t=t)
    q[..., 0] = q0
    ko, vo = (x[P:].unsqueeze(0).expand(B, L, heads, D).contiguous() for x in (k, v))
    out, lse = torch.empty(B, R, heads, D, device="cuda"), torch.empty(B, R, heads, device="cuda")
    comp.prefix_attention_dev(q, out, k[:P], v[:P], ko, vo, torch.full((B,), L, dtype=torch.int32, device="cuda"), lse,
                              scale=1.0)
    comp.sync()
    for r in range(R):
        seen = P + L - (R - 1 - r)
        x = k[:seen, 0, 0].double() * q0
        best = x == x.max()
        want = v[:seen][best].double().mean(0)
        size = v[:seen][best].double().abs().mean(0)
        assert ((out[:, r].double() - want).abs() <= (2 * 1024 * U[F32] + 4 * U[F32]) * size).all()
        top = float(x.max()) + math.log(int(best.sum()))
        assert ((lse[:, r].double() - top).abs() <= 8 * U[F32] * abs(top)).all()


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B, kv", [(4, 296), (40, 128), (200, 128)], ids=["few rows", "one tile of rows", "two"])
def test_attention_of_near_and_far_rows(comp, B, kv, D, t):
    """Rows whose scores end anywhere from 6 to 12000, side by side, and grow from tile to tile: a row's
    maximum passes where the exponents are formed in another way while its neighbours' do not."""
    g = gen(B + D)
    P = 1100
    kp, vp = z(P, kv, D, t=t), normal(g, P, kv, D).to(t)
    kp[..., 0] = (torch.linspace(-300, 375, P, device="cuda") + torch.randn(P, generator=g, device="cuda")).to(t).view(P, 1)
    q = z(B, 1, kv, D, t=t)
    q[..., 0] = (32 * 0.5 ** (torch.arange(B, device="cuda") % 12)).to(t).view(B, 1, 1)
    out, lse = torch.empty(B, 1, kv, D, device="cuda"), torch.empty(B, 1, kv, device="cuda")
    comp.prefix_attention_dev(q, out, kp, vp, lse=lse, scale=1.0)
    comp.sync()
    n = min(B, 12)
    ref = attention_ref(q[:n], kp, vp, None, None, None, 1.0)
    for b in range(0, B, n):
        m = min(n, B - b)
        check_attention(out[b:b + m], lse[b:b + m], tuple(x[:m] for x in ref), t, float(vp.abs().max()))
