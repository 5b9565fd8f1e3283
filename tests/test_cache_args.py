"""What the cache operators' Python entry points check and pass on, without a GPU.

A compute object whose library only records its calls stands in for the real
one (device -1 is what torch calls the CPU): every refusal is raised before the
library is called, and a good call hands over the addresses, strides and sizes
of its tensors in the field order of include/dcinfer.h.
"""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def core(P):
    c = object.__new__(P.compute.Compute)
    c.L, c.h, c.device = Recorder(), None, -1
    return c


def sent(core, P, name, layout):
    calls = [a for n, a in core.L.calls if n == name]
    assert len(calls) == 1, core.L.calls
    return getattr(P._lib, layout).unpack(calls[0][1])


@pytest.mark.parametrize("struct,layout", [("dc_head_rope", "HEAD_ROPE"), ("dc_prefix_attn", "PREFIX_ATTN"),
                                           ("dc_cache_weight", "CACHE_WEIGHT"), ("dc_cache_evict", "CACHE_EVICT")])
def test_layouts_follow_the_header(P, struct, layout):
    """The packed layout has the header's fields: pointers, 64-bit, doubles, ints, in that order."""
    src = open(os.path.join(ROOT, "include", "dcinfer.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S).replace("DC_MAX_AXES", "4")
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), src, re.S).group(1)
    fields = []
    for decl in body.split(";"):
        decl = decl.strip()
        if not decl:
            continue
        for part in re.sub(r"^(const\s+)?\w+", "", decl).split(","):
            base = re.match(r"(const\s+)?(\w+)", decl).group(2)
            n = re.search(r"\[(\d+)\]", part)
            kind = ctypes.c_void_p if "*" in part or "*" in decl.split(",")[0] and base != "int" else {
                "int64_t": ctypes.c_int64, "double": ctypes.c_double, "int": ctypes.c_int}[base]
            fields.append(("f%d" % len(fields), kind * int(n.group(1)) if n else kind))
    c = type("S", (ctypes.Structure,), {"_fields_": fields})
    fmt = getattr(P._lib, layout)
    assert ctypes.sizeof(c) == fmt.size
    codes = "".join({ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_double: "d", ctypes.c_int: "i"}.get(k, "i" * 4)
                    for _, k in fields)
    spelled = re.sub(r"(\d+)(\w)", lambda m: m.group(2) * int(m.group(1)), fmt.format.lstrip("@")).rstrip("P")
    assert codes == spelled


def rope_args(rows=5, heads=4, kv=2, D=16, axes=1, dst=torch.bfloat16):
    return dict(x=torch.zeros(rows, (heads + 2 * kv) * D), pos=torch.zeros((rows,) if axes == 1 else (axes, rows), dtype=torch.int32),
                q=torch.zeros(rows, heads, D, dtype=dst), k=torch.zeros(7, kv, D, dtype=dst), v=torch.zeros(7, kv, D, dtype=dst))


def test_head_norm_rope_passes_its_arguments(core, P):
    a = rope_args()
    big = torch.zeros(3, 9, 2, 16, dtype=torch.bfloat16)
    core.head_norm_rope_dev(a["x"], a["pos"], a["q"], big, big.clone(), slots=torch.zeros(5, dtype=torch.int64),
                            wq=torch.ones(16), eps=1e-6, theta=5e5)
    f = sent(core, P, "dc_head_norm_rope_dev", "HEAD_ROPE")
    assert f[0] == a["x"].data_ptr() and f[3] != 0 and f[4] == 0 and f[5] == 0
    #        ldx ld_pos q_row q_head  k_seq k_tok k_head  v_seq v_tok v_head seqs len
    assert f[9:21] == (128, 5, 64, 16, 288, 32, 16, 288, 32, 16, 3, 9)
    assert f[21:23] == (1e-6, 5e5)
    #         rows heads kv D  rot axes cyclic x_type out_type, sections
    assert f[23:] == (5, 4, 2, 16, 16, 1, 0, 0, 2, 8, 0, 0, 0)


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(5, 127)), dict(x=torch.zeros(5, 128, dtype=torch.float64)), dict(x=torch.zeros(128)),
    dict(pos=torch.zeros(4, dtype=torch.int32)), dict(pos=torch.zeros(5, dtype=torch.int64)),
    dict(pos=torch.zeros(5, 5, dtype=torch.int32)), dict(q=torch.zeros(4, 4, 16, dtype=torch.bfloat16)),
    dict(q=torch.zeros(5, 4, 16)), dict(k=torch.zeros(7, 2, 8, dtype=torch.bfloat16)),
    dict(v=torch.zeros(6, 2, 16, dtype=torch.bfloat16)), dict(slots=torch.zeros(5, dtype=torch.int32)),
    dict(slots=torch.zeros(4, dtype=torch.int64)), dict(wq=torch.zeros(15)), dict(wk=torch.zeros(16, dtype=torch.bfloat16)),
    dict(sections=[4, 4]), dict(inv_freq=[1.0]), dict(x=torch.zeros(128, 5).t()),
    dict(q=torch.zeros(5, 16, 4, dtype=torch.bfloat16).transpose(1, 2))], ids=lambda c: "-".join(c))
def test_head_norm_rope_refuses(core, change):
    a = {**rope_args(), **change}
    with pytest.raises(ValueError):
        core.head_norm_rope_dev(a.pop("x"), a.pop("pos"), a.pop("q"), a.pop("k"), a.pop("v"), **a)
    assert not core.L.calls


def attn_args(B=3, R=2, H=4, KV=2, D=16, P=10, L=6, t=torch.float16):
    return dict(q=torch.zeros(B, R, H, D, dtype=t), out=torch.zeros(B, R, H, D, dtype=t),
                k_pre=torch.zeros(P, KV, D, dtype=t), v_pre=torch.zeros(P, KV, D, dtype=t),
                k_own=torch.zeros(B, L, KV, D, dtype=t), v_own=torch.zeros(B, L, KV, D, dtype=t),
                lens=torch.zeros(B, dtype=torch.int32), lse=torch.zeros(B, R, H))


def test_prefix_attention_passes_its_arguments(core, P):
    a = attn_args()
    a["k_pre"] = torch.zeros(2, 10, 16, dtype=torch.float16).transpose(0, 1)  # head-major
    core.prefix_attention_dev(**a)
    f = sent(core, P, "dc_prefix_attention_dev", "PREFIX_ATTN")
    assert f[:8] == tuple(a[n].data_ptr() for n in ("q", "k_pre", "v_pre", "k_own", "v_own", "lens", "out", "lse"))
    assert f[8:24] == (128, 64, 16, 128, 64, 16, 16, 160, 32, 16, 192, 32, 16, 192, 32, 16)
    assert f[24:] == (0.25, 3, 2, 4, 2, 16, 10, 6, 1, 1)


def test_prefix_attention_takes_either_cache_alone(core, P):
    a = attn_args()
    core.prefix_attention_dev(a["q"], a["out"].float(), k_pre=a["k_pre"], v_pre=a["v_pre"], scale=2.0)
    f = sent(core, P, "dc_prefix_attention_dev", "PREFIX_ATTN")
    assert f[3:6] == (0, 0, 0) and f[24] == 2.0 and f[30:32] == (10, 0) and f[-1] == 0


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(3, 2, 4, 16, dtype=torch.float64)), dict(out=torch.zeros(3, 2, 4, 8, dtype=torch.float16)),
    dict(v_pre=None), dict(k_own=None), dict(lens=None), dict(k_pre=torch.zeros(10, 2, 16)),
    dict(v_pre=torch.zeros(9, 2, 16, dtype=torch.float16)), dict(k_own=torch.zeros(2, 6, 2, 16, dtype=torch.float16)),
    dict(v_own=torch.zeros(3, 6, 2, 16)), dict(lens=torch.zeros(3, dtype=torch.int64)),
    dict(lens=torch.zeros(4, dtype=torch.int32)), dict(lse=torch.zeros(3, 2, 4, dtype=torch.float16)),
    dict(k_pre=torch.zeros(10, 16, 2, dtype=torch.float16).transpose(1, 2)),
    dict(q=torch.zeros(3, 2, 4, 16, dtype=torch.float16)[..., ::2].repeat(1, 1, 1, 2)[..., ::1].transpose(2, 3))],
    ids=lambda c: "-".join(c))
def test_prefix_attention_refuses(core, change):
    with pytest.raises(ValueError):
        core.prefix_attention_dev(**{**attn_args(), **change})
    assert not core.L.calls


def weight_args(B=2, R=3, H=4, KV=2, D=16, L=9, t=torch.bfloat16):
    return dict(q=torch.zeros(B, R, H, D, dtype=t), k=torch.zeros(B, L, KV, D, dtype=t),
                lens=torch.zeros(B, dtype=torch.int32), lse=torch.zeros(B, R, H), acc=torch.zeros(B, KV, L))


def test_cache_weights_passes_its_arguments(core, P):
    a = weight_args()
    core.cache_weights_dev(**a, decay=0.5, causal=False)
    f = sent(core, P, "dc_cache_weights_dev", "CACHE_WEIGHT")
    assert f[:5] == tuple(a[n].data_ptr() for n in ("q", "k", "lens", "lse", "acc"))
    assert f[5:13] == (192, 64, 16, 288, 32, 16, 18, 9)
    assert f[13:] == (0.25, 0.5, 2, 3, 4, 2, 16, 9, 0, 2)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 3, 4, 16)), dict(k=torch.zeros(3, 9, 2, 16, dtype=torch.bfloat16)),
    dict(k=torch.zeros(2, 9, 2, 8, dtype=torch.bfloat16)), dict(acc=torch.zeros(2, 2, 8)),
    dict(acc=torch.zeros(2, 2, 9, dtype=torch.float64)), dict(lens=torch.zeros(2)), dict(lse=torch.zeros(2, 4, 3)),
    dict(acc=torch.zeros(2, 9, 2).transpose(1, 2))], ids=lambda c: "-".join(c))
def test_cache_weights_refuses(core, change):
    with pytest.raises(ValueError):
        core.cache_weights_dev(**{**weight_args(), **change})
    assert not core.L.calls


def evict_args(B=2, KV=2, D=16, L=9, n=4, t=torch.float16):
    return dict(k=torch.zeros(B, L, KV, D, dtype=t), v=torch.zeros(B, L, KV, D, dtype=t), acc=torch.zeros(B, KV, L),
                lens=torch.zeros(B, dtype=torch.int32), k_out=torch.zeros(B, n, KV, D, dtype=t),
                v_out=torch.zeros(B, n, KV, D, dtype=t), acc_out=torch.zeros(B, KV, n),
                index=torch.zeros(B, KV, n, dtype=torch.int32), lens_out=torch.zeros(B, dtype=torch.int32))


def test_cache_evict_passes_its_arguments(core, P):
    a = evict_args()
    core.cache_evict_dev(**a, budget=4, recent=1)
    f = sent(core, P, "dc_cache_evict_dev", "CACHE_EVICT")
    assert f[:9] == tuple(a[n].data_ptr() for n in a)
    assert f[9:27] == (288, 32, 16, 288, 32, 16, 18, 9, 128, 32, 16, 128, 32, 16, 8, 4, 8, 4)
    assert f[27:] == (2, 2, 16, 9, 4, 1, 2)


@pytest.mark.parametrize("change", [
    dict(v=torch.zeros(2, 9, 2, 16)), dict(k=torch.zeros(2, 9, 2, 16, dtype=torch.int16)), dict(acc=torch.zeros(2, 2, 8)),
    dict(k_out=torch.zeros(2, 3, 2, 16, dtype=torch.float16)), dict(v_out=torch.zeros(2, 4, 2, 16)),
    dict(acc_out=torch.zeros(2, 2, 3)), dict(index=torch.zeros(2, 2, 4, dtype=torch.int64)),
    dict(index=torch.zeros(2, 4, dtype=torch.int32)), dict(lens_out=torch.zeros(1, dtype=torch.int32)),
    dict(lens=torch.zeros(2, dtype=torch.int64))], ids=lambda c: "-".join(c))
def test_cache_evict_refuses(core, change):
    with pytest.raises(ValueError):
        core.cache_evict_dev(**{**evict_args(), **change}, budget=4)
    assert not core.L.calls


def test_tensors_of_another_device_are_refused(core):
    core.device = 0  # (these are CPU tensors)
    with pytest.raises(ValueError, match="cuda:0"):
        core.cache_weights_dev(**weight_args())
    with pytest.raises(ValueError, match="cuda:0"):
        core.cache_evict_dev(**evict_args(), budget=4)
    with pytest.raises(ValueError, match="cuda:0"):
        core.prefix_attention_dev(**attn_args())
    a = rope_args()
    with pytest.raises(ValueError, match="cuda:0"):
        core.head_norm_rope_dev(a["x"], a["pos"], a["q"], a["k"], a["v"])
    assert not core.L.calls
