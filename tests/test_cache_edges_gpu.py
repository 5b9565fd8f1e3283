"""The cache operators at the ends of what their arguments may hold, against 64 bits."""
import math

import pytest
import torch

from test_cache_gpu import BF16, F16, F32, U, attention_ref, check_attention, gen, normal, weights_ref, z

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
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731

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
