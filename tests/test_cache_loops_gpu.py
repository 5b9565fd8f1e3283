"""The cache operators where one block walks many tiles: rings that turn, maxima that are raised, buffers that alternate.

The kernels cut small problems so that a block has one tile of keys; these have so many heads or sequences
that it has many.  How many is taken from the call itself (an attention's workspace holds one part a split,
so its size tells the splits) and asserted, so that another rule of splitting cannot empty the tests.
Tolerances are those of test_cache_gpu.
"""
import math

import pytest
import torch

from test_cache_gpu import BF16, F16, F32, attention_ref, check_attention, gen, normal, weights_ref

pytestmark = pytest.mark.gpu


def splits_of(comp, q, out, k_pre=None, v_pre=None, k_own=None, v_own=None, lens=None, lse=None):
    """Splits of the prefix, or of the own keys where there is no prefix, from the workspace's size."""
    B, R, H, D = q.shape
    kv = (k_pre if k_pre is not None else k_own).shape[-2]
    part = (64 if D <= 64 else 128) * 4 + 8
    n = comp.prefix_attention_ws(q, out, k_pre, v_pre, k_own, v_own, lens, lse)
    rows = B * R * (H // kv) * kv  # (parts of one split)
    assert n % (part * rows) == 0
    return n // (part * rows)


def scores(kind, P, tile, g):
    """A score for each of P keys (scale 1): what the running maximum meets from tile to tile."""
    at = torch.arange(P, device="cuda") // tile
    if kind == "growing":       # 12 bits a tile: raised by every one
        return at * 8.5 - 40
    if kind == "at the limit":  # 8 bits a tile at most: raised by every other one or two
        return at * 5.5 - 30
    if kind == "falling":
        return 40 - at * 8.5
    if kind == "empty then finite":  # tiles of -inf, one key, tiles of -inf, the rest
        x = torch.where((at % 7 < 3), -math.inf, at * 3.0 - 10)
        x[:4 * tile] = -math.inf
        x[2 * tile + 5] = -20.0
        return x
    return torch.randn(P, generator=g, device="cuda") * 6  # "random"


KINDS = ["growing", "at the limit", "falling", "empty then finite", "random"]


def keys_of(x, kv, D, t):
    """Keys whose product with queries of 1/2 in each channel is x: x spread over the channels (kept exact by
    taking what the type makes of it; the reference sees the same keys)."""
    return (x / D * 2).view(-1, 1, 1).expand(-1, kv, D).to(t).contiguous()


def check_alike(out, lse, q, kp, vp, t):
    """Against 64 bits where all queries are alike: one sequence's reference is everyone's.  Keys at -inf
    (the same for all heads) take no part: the reference leaves them out, and its bounds stay finite."""
    keep = torch.isfinite(kp[:, 0, 0])
    ref = attention_ref(q[:1], kp[keep], vp[keep], None, None, None, 1.0)
    check_attention(out, lse, tuple(x.expand(q.shape[0], *x.shape[1:]) for x in ref), t, float(vp.abs().max()))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, t", [(64, BF16), (64, F16), (128, BF16), (128, F16)])
@pytest.mark.parametrize("B", [40, 200], ids=["one tile of rows", "two"])
def test_shared_prefix_over_many_tiles(comp, B, D, t, kind):
    """128 key heads fill the SMs: every block walks the whole prefix, its ring several times round."""
    g = gen(B + D)
    kv, P = 128, 1500
    kp, vp = keys_of(scores(kind, P, 128, g), kv, D, t), normal(g, P, kv, D).to(t)
    q = (0.5 * torch.ones(B, 1, kv, D, device="cuda")).to(t)
    out, lse = torch.empty(B, 1, kv, D, device="cuda"), torch.empty(B, 1, kv, device="cuda")
    assert -(-P // 128) / splits_of(comp, q, out, kp, vp) >= 8
    comp.prefix_attention_dev(q, out, kp, vp, lse=lse, scale=1.0)
    comp.sync()
    check_alike(out, lse, q, kp, vp, t)


@pytest.mark.parametrize("D, t", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("B", [33, 129, 300], ids=["one tile of rows", "a pair, the second short", "a pair and one"])
def test_shared_prefix_of_many_tiles_and_different_rows(comp, B, D, t):
    g = gen(B + D + 1)
    kv, P = 160 if B < 129 else 80 if B > 256 else 150, 1413
    q = (normal(g, B, 1, kv, D) * torch.linspace(0.2, 6, B, device="cuda").view(B, 1, 1, 1)).to(t)
    kp, vp = normal(g, P, kv, D).to(t), normal(g, P, kv, D).to(t)
    out, lse = torch.empty_like(q), torch.empty(B, 1, kv, device="cuda")
    assert -(-P // 128) / splits_of(comp, q, out, kp, vp) >= 6
    comp.prefix_attention_dev(q, out, kp, vp, lse=lse)
    comp.sync()
    rows = list(range(0, B, max(1, B // 12))) + [B - 1]
    ref = attention_ref(q[rows], kp, vp, None, None, None, D ** -0.5)
    check_attention(out[rows], lse[rows], ref, t, float(vp.abs().max()))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B", [40, 200], ids=["one tile of rows", "two"])
def test_shared_prefix_nan_in_a_later_tile(comp, B, D):
    """A NaN in the seventh tile of one head spoils that head and no other."""
    g = gen(B + D + 2)
    kv, P, t = 128, 1500, BF16
    q = normal(g, B, 1, kv, D).to(t)
    kp, vp = normal(g, P, kv, D).to(t), normal(g, P, kv, D).to(t)
    kp[6 * 128 + 3, 5, 1] = math.nan
    out, lse = torch.empty_like(q), torch.empty(B, 1, kv, device="cuda")
    assert -(-P // 128) / splits_of(comp, q, out, kp, vp) >= 8
    comp.prefix_attention_dev(q, out, kp, vp, lse=lse)
    comp.sync()
    assert torch.isnan(out[:, :, 5]).all() and torch.isnan(lse[:, :, 5]).all()
    rest = [h for h in range(kv) if h != 5]
    assert torch.isfinite(out[:, :, rest]).all() and torch.isfinite(lse[:, :, rest]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, t", [(64, F16), (128, BF16)])
def test_few_rows_over_many_tiles(comp, D, t, kind):
    """A batch of four before 296 key heads: each warp of a block takes ten tiles of 16 keys or more."""
    g = gen(D)
    B, kv, P = 4, 296, 801
    kp, vp = keys_of(scores(kind, P, 64, g), kv, D, t), normal(g, P, kv, D).to(t)
    q = (0.5 * torch.ones(B, 1, kv, D, device="cuda")).to(t)
    out, lse = torch.empty(B, 1, kv, D, device="cuda"), torch.empty(B, 1, kv, device="cuda")
    assert -(-P // 64) / splits_of(comp, q, out, kp, vp) >= 7
    comp.prefix_attention_dev(q, out, kp, vp, lse=lse, scale=1.0)
    comp.sync()
    check_alike(out, lse, q, kp, vp, t)


@pytest.mark.parametrize("kind", ["growing", "empty then finite", "random"])
@pytest.mark.parametrize("R, G, D, t", [(1, 4, 128, BF16), (3, 4, 64, F16), (5, 8, 64, BF16)])
def test_own_keys_over_many_tiles(comp, R, G, D, t, kind):
    """37 sequences of 8 key heads, up to 700 own keys of which each warp takes seven tiles or more; ragged lengths;
    NaN behind them; with five rows of eight heads three tiles of rows."""
    g = gen(R + D)
    B, kv, L = 37, 8, 700
    H = kv * G
    x = scores(kind, L, 64, g)
    ko = keys_of(x, kv, D, t).expand(B, L, kv, D).contiguous()
    vo = normal(g, B, L, kv, D).to(t)
    lens = [700 - 19 * b if b % 3 else 640 + b for b in range(B)]
    for b, n in enumerate(lens):
        ko[b, n:] = math.nan
        vo[b, n:] = math.nan
    q = (0.5 * torch.ones(B, R, H, D, device="cuda")).to(t)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = torch.empty(B, R, H, D, device="cuda"), torch.empty(B, R, H, device="cuda")
    assert -(-L // 64) / splits_of(comp, q, out, k_own=ko, v_own=vo, lens=ln) >= 7
    comp.prefix_attention_dev(q, out, k_own=ko, v_own=vo, lens=ln, lse=lse, scale=1.0)
    comp.sync()
    vmax = float(vo.nan_to_num().abs().max())
    for b in (0, 1, 2, 9, 17, 36):
        for r in range(R):
            seen = lens[b] - (R - 1 - r)
            keep = torch.isfinite(x[:seen]).nonzero().view(-1)  # (as in check_alike)
            ref = attention_ref(q[b:b + 1, r:r + 1], None, None, ko[b:b + 1, keep], vo[b:b + 1, keep], [len(keep)], 1.0)
            check_attention(out[b:b + 1, r:r + 1], lse[b:b + 1, r:r + 1], ref, t, vmax)
    assert torch.isfinite(out).all()


def test_prefix_and_own_keys_over_many_tiles(comp):
    """Both kernels and the join, each over many tiles; the same bits on every call."""
    g = gen(7)
    B, R, kv, D, P, L, t = 9, 4, 150, 128, 1300, 400, BF16
    q = (2 * normal(g, B, R, kv, D)).to(t)
    kp, vp = normal(g, P, kv, D).to(t), normal(g, P, kv, D).to(t)
    ko, vo = normal(g, B, L, kv, D).to(t), normal(g, B, L, kv, D).to(t)
    lens = [400, 0, 3, 399, 64, 65, 200, 333, 1]
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = []
    for _ in range(3):
        out, lse = torch.empty_like(q), torch.empty(B, R, kv, device="cuda")
        comp.prefix_attention_dev(q, out, kp, vp, ko, vo, ln, lse)
        got.append((out, lse))
    comp.sync()
    assert all(torch.equal(got[0][i], o[i]) for o in got for i in range(2))
    check_attention(*got[0], attention_ref(q, kp, vp, ko, vo, lens, D ** -0.5), t, 6.0)


WEIGHTS = [  # batch, rows, heads, kv, D, cache, lens, type, causal
    (37, 1, 32, 8, 64, 1500, None, BF16, True),       # a block walks its head's twelve key tiles
    (37, 3, 24, 8, 40, 1427, None, F16, True),
    (37, 2, 32, 8, 128, 1500, None, BF16, True),
    (30, 5, 50, 10, 64, 1300, None, F16, False),
    (1, 300, 32, 8, 64, 500, [500], BF16, True),      # ten tiles of queries, ring of six
    (1, 700, 15, 5, 64, 300, [290], F16, False),      # 17 tiles of 42 rows
    (2, 1500, 3, 3, 64, 200, [200, 131], BF16, True),  # 12 tiles of 128 rows; more rows than tokens
    (1, 260, 64, 2, 128, 300, [300], F16, True),      # 65 tiles of four rows
    (1, 900, 8, 8, 128, 400, [399], BF16, False),
]


@pytest.mark.parametrize("case", WEIGHTS, ids=lambda c: "x".join(str(v) for v in c[:6]) + str(c[7])[6:])
def test_cache_weights_over_many_tiles(comp, case):
    B, R, H, kv, D, L, lens, t, causal = case
    lens = lens or [L - 31 * b if b % 4 else L for b in range(B)]
    G = H // kv
    tile_rows = 128 // G
    if R <= tile_rows:  # (key tiles of a block: a head's, shared by the blocks that two an SM give it)
        tiles, shares = -(-L // 128), max(1, 2 * torch.cuda.get_device_properties(0).multi_processor_count // (B * kv))
        assert tiles / min(tiles, shares) >= 8
    else:
        assert -(-R // tile_rows) > 6
    g = gen(R + L)
    q, k = (normal(g, B, R, H, D) * 1.5).to(t), normal(g, B, L, kv, D).to(t)
    for b, n in enumerate(lens):
        k[b, n:] = math.nan
    lse = 1.0 + 3 * torch.rand(B, R, H, generator=g, device="cuda") + math.log(L)
    acc = torch.rand(B, kv, L, generator=g, device="cuda")
    before = acc.clone()
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    comp.cache_weights_dev(q, k, ln, lse, acc, decay=0.9, causal=causal)
    again = before.clone()
    comp.cache_weights_dev(q, k, ln, lse, again, decay=0.9, causal=causal)
    comp.sync()
    assert torch.equal(acc, again)
    for b in sorted({0, B // 2, B - 1}):
        n = lens[b]
        want, tol = weights_ref(q[b:b + 1], k[b:b + 1], [n], lse[b:b + 1], before[b:b + 1], D ** -0.5, 0.9, causal)
        err = (acc[b, :, :n].double() - want[0, :, :n]).abs()
        assert (err <= tol[0, :, :n]).all(), float((err - tol[0, :, :n]).max())
        assert torch.equal(acc[b, :, n:], before[b, :, n:])
    assert acc.dtype is F32 and torch.isfinite(acc).all()
