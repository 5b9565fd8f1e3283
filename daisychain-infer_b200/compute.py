"""The compute core: the object ``Compute.initCompute`` returns in the reference.

Mirrors public/webgpu.js: ``init_compute`` (initCompute :284-648),
``load_luts`` (loadLUTs :247-257), ``kernel_probe`` (:1047-1060) and the
compute object's ``bgemm`` (gpuBgemmDP4 / gpuBgemmLUT :819-857), so that the
reference's vgemmBlock contract (public/verified_core.js:425-449) is met:

    out = compute.bgemm(Xq, Wq, rs, cs, dict(m=.., k=.., n=.., batch=1, relu=False, acc=False))

with host int8/f32 arrays in the reference's layouts; ``out`` is a fresh
int32 array (acc) or f32 array owned by the caller.  Errors carry the
reference's names: ``AccumulatorBoundError`` before any launch for
k > 131071, ``NonFiniteError`` for a non-finite quantiser input.

Device-resident entry points take torch CUDA tensors (torch is used only as
the device-memory allocator and for its current stream).
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import DC_ACC, DC_RELU, DC_REQUANT, AccumulatorBoundError, NonFiniteError, raise_for  # noqa: F401


def _ptr(a):
    if a is None:
        return None
    if isinstance(a, np.ndarray):
        return a.ctypes.data_as(C.c_void_p)
    return C.c_void_p(a.data_ptr())  # torch tensor


def flags_of(d: dict) -> int:
    f = 0
    if d.get("relu"):
        f |= DC_RELU
    if d.get("acc"):
        f |= DC_ACC
    if d.get("requant"):
        f |= DC_REQUANT
    return f


class Compute:
    """One B200 bound to one stream: ``backend``, ``label``, ``bgemm``."""

    backend = "cuda-sm100a"

    def __init__(self, device: int = 0, stream=None):
        self.L = _lib.load()
        self.device = device
        h = C.c_void_p()
        rc = self.L.dc_init(device, C.byref(h))
        if rc:
            raise_for(rc, "dc_init: " + (self.L.dc_init_error() or b"").decode())
        self.h = h
        if stream is not None:
            self.set_stream(stream)
        self.label = self.L.dc_backend_label(self.h).decode()

    # ---- plumbing -------------------------------------------------------------
    def _check(self, rc: int, where: str) -> None:
        if rc:
            raise_for(rc, f"{where}: " + (self.L.dc_last_error(self.h) or b"").decode())

    def set_stream(self, stream) -> None:
        """Launch on an existing stream (a torch.cuda.Stream or a raw handle)."""
        handle = getattr(stream, "cuda_stream", stream)
        # torch reports the legacy default stream as handle 0; CUDA names it cudaStreamLegacy (0x1)
        self._check(self.L.dc_set_stream(self.h, C.c_void_p(handle if handle else 1)), "dc_set_stream")

    def sync(self) -> None:
        self._check(self.L.dc_sync(self.h), "dc_sync")

    @property
    def tc_enabled(self) -> bool:
        return bool(self.L.dc_tc_enabled(self.h))

    def close(self) -> None:
        if getattr(self, "h", None):
            self.L.dc_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- the LUT units ----------------------------------------------------------
    def luts(self) -> dict:
        """loadLUTs: {mul int16[65536], requant int8[65536], relu int8[256], shift 8},
        rebuilt by the library and checked against the reference's sha256 ids."""
        mul = np.empty(65536, np.int16)
        req = np.empty(65536, np.int8)
        relu = np.empty(256, np.int8)
        self._check(self.L.dc_luts(self.h, _ptr(mul), _ptr(req), _ptr(relu)), "dc_luts")
        return dict(mul=mul, requant=req, relu=relu, shift=8)

    # ---- compute.bgemm (host buffers) -------------------------------------------
    def bgemm(self, Xq, Wq, rs, cs, d: dict) -> np.ndarray:
        m, k, n = int(d["m"]), int(d["k"]), int(d["n"])
        batch = int(d.get("batch") or 1)
        flags = flags_of(d)
        if k > _lib.MAX_INT32_K:
            raise AccumulatorBoundError(f"bgemm: contraction length {k} exceeds the int32 accumulator headroom "
                                        f"{_lib.MAX_INT32_K} (the sum would wrap)")
        Xq = np.ascontiguousarray(Xq, np.int8).reshape(-1)
        Wq = np.ascontiguousarray(Wq, np.int8).reshape(-1)
        rs = np.ascontiguousarray(rs, np.float32).reshape(-1)
        cs = np.ascontiguousarray(cs, np.float32).reshape(-1)
        if Xq.size != batch * m * k or Wq.size != batch * k * n or rs.size != batch * m or cs.size != batch * n:
            raise ValueError("bgemm: buffer sizes do not match d")
        dt = np.int32 if flags & DC_ACC else (np.int8 if flags & DC_REQUANT else np.float32)
        out = np.empty(batch * m * n, dt)
        self._check(self.L.dc_bgemm(self.h, _ptr(Xq), _ptr(Wq), _ptr(rs), _ptr(cs), m, k, n, batch, flags,
                                    _ptr(out)), "bgemm")
        return out

    # ---- device-resident entry points (torch CUDA tensors) ---------------------
    def bgemm_dev(self, xq, ldx, wt, ldw, rs, cs, m, k, n, batch, flags, out, kind: int = 0) -> None:
        if kind:
            rc = self.L.dc_bgemm_dev_kind(self.h, _ptr(xq), ldx, _ptr(wt), ldw, _ptr(rs), _ptr(cs), m, k, n, batch,
                                          flags, _ptr(out), kind)
        else:
            rc = self.L.dc_bgemm_dev(self.h, _ptr(xq), ldx, _ptr(wt), ldw, _ptr(rs), _ptr(cs), m, k, n, batch, flags,
                                     _ptr(out))
        self._check(rc, "bgemm_dev")

    def bgemm_lut_dev(self, xq, wq, rs, cs, m, k, n, batch, flags, out) -> None:
        self._check(self.L.dc_bgemm_lut_dev(self.h, _ptr(xq), _ptr(wq), _ptr(rs), _ptr(cs), m, k, n, batch, flags,
                                            _ptr(out)), "bgemm_lut_dev")

    def quantize_rows_dev(self, X, rows, cols, q, ldq, s) -> None:
        self._check(self.L.dc_quantize_rows(self.h, _ptr(X), rows, cols, _ptr(q), ldq, _ptr(s)), "quantize_rows")

    def quantize_cols_t_dev(self, W, rows, cols, qt, ldq, s) -> None:
        self._check(self.L.dc_quantize_cols_t(self.h, _ptr(W), rows, cols, _ptr(qt), ldq, _ptr(s)),
                    "quantize_cols_t")

    def register_weight(self, W: np.ndarray, k: int, n: int) -> "Weight":
        return Weight(self, W, k, n)

    def vgemm_dev(self, X, m, w: "Weight", flags, out) -> None:
        self._check(self.L.dc_vgemm(self.h, _ptr(X), m, w.h, flags, _ptr(out)), "vgemm")

    def ordered_sum_dev(self, terms, rows, n, out) -> None:
        """out[r] = serial double sum of terms[r] in index order (infer.js:73-76, :100-104)."""
        self._check(self.L.dc_ordered_sum_dev(self.h, _ptr(terms), rows, n, _ptr(out)), "ordered_sum")

    def exp_dev(self, x, n, y, sel=False) -> None:
        """y = Math.exp(x) by the fdlibm method (sel True or 1: the branch-free form the kernels
        use; 2: the table-driven exp of the chunk softmax; 3: f32(Math.exp(x)) as that softmax
        settles it; 4, 5: the SwiGLU value of g = f32(x), u = f32(x/2 + 1/4), settled and exact)."""
        self._check(self.L.dc_exp_dev(self.h, _ptr(x), n, _ptr(y), int(sel)), "exp")

    def rmsnorm_dev(self, x, rows, cols, w, eps, y, exact_sum: bool = False) -> None:
        """infer.js rmsnorm (:70-80) of rows x cols f32 (exact_sum: always the serial-order sum)."""
        self._check(self.L.dc_rmsnorm_dev(self.h, _ptr(x), rows, cols, _ptr(w), float(eps), _ptr(y),
                                          1 if exact_sum else 0), "rmsnorm")

    # ---- a batch's key/value cache (torch CUDA tensors) ---------------------------
    def _types(self) -> dict:
        """torch's element types by the C ABI's names (DC_F32, DC_F16, DC_BF16)."""
        t = Compute._type_of
        if not t:
            import torch
            t.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, "i32": torch.int32, "i64": torch.int64,
                      "u8": torch.uint8, "torch": torch})
        return t

    _type_of: dict = {}

    def _ptrs(self, what: str, *tensors) -> list:
        """The tensors' addresses (0 for None), all on this object's device."""
        dev, at = self.device, []
        for t in tensors:
            if t is None:
                at.append(0)
            elif t.get_device() == dev:
                at.append(t.data_ptr())
            else:
                raise ValueError(f"{what}: a tensor is not on cuda:{dev}")
        return at

    @staticmethod
    def _flat(t, shape, dtype) -> bool:
        return t.shape == shape and t.dtype is dtype and t.is_contiguous()

    def _scratch(self, n: int):
        """n bytes of torch's memory, in the order of the stream that this object launches on."""
        T = self._types()
        torch, stream = T["torch"], self.L.dc_stream(self.h)
        dev = T.get(self.device)
        if dev is None:
            dev = T[self.device] = torch.device("cuda", self.device)
        # (the legacy default stream is 0 to torch and 1 to the library)
        if (torch._C._cuda_getCurrentRawStream(self.device) or 1) == (stream or 1):
            return torch.empty(n, dtype=T["u8"], device=dev)
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=dev)):
            return torch.empty(n, dtype=T["u8"], device=dev)

    def head_norm_rope_dev(self, x, pos, q, k, v, slots=None, *, wq=None, wk=None, eps=1e-5, theta=10000.0,
                           inv_freq=None, rot=None, sections=None, cyclic: bool = False) -> None:
        """RMS norm of every query and key head, rotary positions, and the cache
        append, in one pass over the rows of a fused QKV projection.

        x (rows, (heads + 2 kv_heads) * head_dim) holds [queries | keys | values]
        of each row (vgemm_dev's output; f32, f16 or bf16).  q (rows, heads,
        head_dim) receives the queries; k and v, both (slots, kv_heads, head_dim) or
        (sequences, length, kv_heads, head_dim), the keys and values at slots[row]
        (int64; a negative one is padding and writes neither; None: row i at slot
        i).  Slots count through the sequences, and no two rows of a call share one.
        wq, wk (head_dim, f32): the norm's weights, None for no norm.  pos int32,
        (rows,) or (axes, rows), an expanded row too; sections: pairs of channels that
        each axis turns, in runs, or with cyclic by turns (pair i on axis i % axes).
        rot: channels that are rotated (all); inv_freq (host f64, rot/2) in place of theta.
        A slot behind the cache is not written and makes the next sync() raise."""
        T = self._types()
        if x.ndim != 2 or q.ndim != 3 or k.ndim not in (3, 4) or v.shape != k.shape:
            raise ValueError("head_norm_rope: x (rows, width), q (rows, heads, head_dim), k and v (slots.., kv_heads, "
                             "head_dim)")
        rows, width = x.shape
        rows_q, heads, D = q.shape
        seqs, (length, kv, Dk) = (1, k.shape) if k.ndim == 3 else (k.shape[0], k.shape[1:])
        if rows_q != rows or Dk != D or width != (heads + 2 * kv) * D:
            raise ValueError(f"head_norm_rope: x {tuple(x.shape)}, q {tuple(q.shape)}, k {tuple(k.shape)} do not match")
        dt = q.dtype
        if k.dtype is not dt or v.dtype is not dt or dt not in T or x.dtype not in T:
            raise ValueError("head_norm_rope: x, and q, k and v of one type: float32, float16 or bfloat16")
        axes, npos = (1, pos.shape[0]) if pos.ndim == 1 else pos.shape if pos.ndim == 2 else (0, 0)
        if npos != rows or pos.dtype is not T["i32"] or not 1 <= axes <= 4:
            raise ValueError("head_norm_rope: pos is int32 of (rows,) or (1 to 4 axes, rows)")
        if slots is not None and not self._flat(slots, (rows,), T["i64"]):
            raise ValueError("head_norm_rope: slots is int64 of (rows,)")
        for w in (wq, wk):
            if w is not None and not (T.get(w.dtype) == 0 and w.shape == (D,) and w.is_contiguous()):
                raise ValueError("head_norm_rope: wq and wk are f32 of (head_dim,)")
        rot = D if rot is None else int(rot)
        sec = [rot // 2] if sections is None else [int(n) for n in sections]
        if len(sec) != axes:
            raise ValueError(f"head_norm_rope: {len(sec)} sections for {axes} position axes")
        freq = 0
        if inv_freq is not None:
            inv_freq = np.ascontiguousarray(inv_freq, np.float64)
            if inv_freq.shape != (rot // 2,):
                raise ValueError("head_norm_rope: inv_freq has rot/2 values")
            freq = inv_freq.ctypes.data
        sx, sp, sq, sk, sv = x.stride(), pos.stride(), q.stride(), k.stride(), v.stride()
        if (sx[-1], sp[-1] if rows > 1 else 1, sq[-1], sk[-1], sv[-1]) != (1, 1, 1, 1, 1):
            raise ValueError("head_norm_rope: the last dimension of x, pos, q, k and v must be contiguous")
        px, pp, ps, pwq, pwk, pq, pk, pv = self._ptrs("head_norm_rope", x, pos, slots, wq, wk, q, k, v)
        a = _lib.HEAD_ROPE.pack(
            px, pp, ps, pwq, pwk, freq, pq, pk, pv, sx[0], sp[0] if axes > 1 else rows, sq[0], sq[1],
            *((0, *sk[:2], 0, *sv[:2]) if k.ndim == 3 else (*sk[:3], *sv[:3])), seqs, length, eps, theta, rows, heads,
            kv, D, rot, axes, 1 if cyclic else 0, T[x.dtype], T[dt], *sec, *(0,) * (4 - axes))
        rc = self.L.dc_head_norm_rope_dev(self.h, a)
        if rc:
            self._check(rc, "head_norm_rope")

    def prefix_attention_dev(self, q, out, k_pre=None, v_pre=None, k_own=None, v_own=None, lens=None, lse=None, *,
                             scale=None, ws=None) -> None:
        """Attention of a batch over a prefix that its sequences share, computed for
        all of them in one pass over the prefix, and over each one's own cache.

        q (batch, rows, heads, head_dim), f16 or bf16, up to 16 rows a sequence (a
        decode step's token, or a token and its drafts); k_pre, v_pre (tokens,
        kv_heads, head_dim): seen by every row; k_own, v_own (batch, length,
        kv_heads, head_dim) with lens (batch, int32, on the device): row r of
        sequence b sees the first lens[b] - (rows - 1 - r) tokens, so a row sees
        itself and what came before.  Either pair may be left out.  out (as q, or
        f32) and lse (batch, rows, heads, f32; optional): softmax(scale q k) v and
        log(sum(exp(scale q k))), 0 and -inf for a row that sees nothing.  scale:
        1/sqrt(head_dim) unless given.  ws: workspace (prefix_attention_ws bytes)
        for callers that hold their own; otherwise torch's allocator gives it."""
        a = self._prefix_attn(q, out, k_pre, v_pre, k_own, v_own, lens, lse, scale)
        if ws is None:
            n = self.L.dc_prefix_attention_ws(self.h, a)
            if n:
                ws = self._scratch(n)
        elif ws.is_contiguous():
            self._ptrs("prefix_attention", ws)
            n = ws.numel() * ws.element_size()
        else:
            raise ValueError("prefix_attention: ws is contiguous")
        rc = self.L.dc_prefix_attention_dev(self.h, a, ws.data_ptr() if n else None, n)
        if rc:
            self._check(rc, "prefix_attention")

    def prefix_attention_ws(self, q, out, k_pre=None, v_pre=None, k_own=None, v_own=None, lens=None, lse=None, *,
                            scale=None) -> int:
        """Bytes of workspace that prefix_attention_dev takes for these arguments (their sizes alone count).
        Raises where it would refuse them."""
        n = self.L.dc_prefix_attention_ws(
            self.h, self._prefix_attn(q, out, k_pre, v_pre, k_own, v_own, lens, lse, scale))
        if not n and self.L.dc_last_error(self.h):
            self._check(_lib.DC_E_INVAL, "prefix_attention_ws")
        return n

    def _prefix_attn(self, q, out, k_pre, v_pre, k_own, v_own, lens, lse, scale) -> bytes:
        T = self._types()
        dt = q.dtype
        if q.ndim != 4 or out.shape != q.shape or dt not in T or out.dtype not in T:
            raise ValueError("prefix_attention: q and out are (batch, rows, heads, head_dim), f16 or bf16 (out also f32)")
        B, R, heads, D = q.shape
        if (k_pre is None) != (v_pre is None) or not (k_own is None) == (v_own is None) == (lens is None):
            raise ValueError("prefix_attention: k_pre comes with v_pre, k_own with v_own and lens")
        sq, so = q.stride(), out.stride()
        last = sq[3] == 1 and so[3] == 1
        kv = k_pre.shape[-2] if k_pre is not None else k_own.shape[-2] if k_own is not None else heads
        pre, own, prefix, own_max = (0,) * 4, (0,) * 6, 0, 0
        if k_pre is not None:
            prefix = k_pre.shape[0]
            if k_pre.shape != (prefix, kv, D) or v_pre.shape != k_pre.shape or k_pre.dtype is not dt or (
                    v_pre.dtype is not dt):
                raise ValueError("prefix_attention: k_pre and v_pre are (tokens, kv_heads, head_dim) of q's type")
            a, b, c = k_pre.stride()
            d, e, f = v_pre.stride()
            pre, last = (a, b, d, e), last and c == 1 and f == 1
        if k_own is not None:
            own_max = k_own.shape[1] if k_own.ndim == 4 else 0
            if k_own.shape != (B, own_max, kv, D) or v_own.shape != k_own.shape or k_own.dtype is not dt or (
                    v_own.dtype is not dt):
                raise ValueError("prefix_attention: k_own and v_own are (batch, length, kv_heads, head_dim) of q's type")
            if not self._flat(lens, (B,), T["i32"]):
                raise ValueError("prefix_attention: lens is int32 of (batch,)")
            a, b, c = k_own.stride(), v_own.stride(), last
            own, last = (*a[:3], *b[:3]), last and a[3] == 1 and b[3] == 1
        if not last:
            raise ValueError("prefix_attention: the last dimension of q, k, v and out must be contiguous")
        if lse is not None and not (T.get(lse.dtype) == 0 and lse.shape == (B, R, heads) and lse.is_contiguous()):
            raise ValueError("prefix_attention: lse is f32 of (batch, rows, heads)")
        return _lib.PREFIX_ATTN.pack(
            *self._ptrs("prefix_attention", q, k_pre, v_pre, k_own, v_own, lens, out, lse), *sq[:3], *so[:3], *pre,
            *own, D ** -0.5 if scale is None else scale, B, R, heads, kv, D, prefix, own_max, T[dt], T[out.dtype])

    def cache_weights_dev(self, q, k, lens, lse, acc, *, scale=None, decay: float = 1.0, causal: bool = True) -> None:
        """Adds to acc (batch, kv_heads, length, f32) the softmax weight that every
        cached key receives from these queries: acc = decay * acc + the sum over
        rows and heads of a group of exp(scale q k - lse), for the first lens[b]
        tokens of sequence b; the rest of acc stays.

        q (batch, rows, heads, head_dim), k (batch, length, kv_heads, head_dim), f16
        or bf16; lens (batch, int32) and lse (batch, rows, heads, f32) as
        prefix_attention_dev takes and gives them (with a prefix, lse spans both).
        causal: row r sees lens[b] - (rows - 1 - r) tokens; False: all rows see all
        (the shared prefix: its k as one sequence, all rows of the batch as rows).
        decay 0 overwrites; a row of lse -inf (padding) adds nothing, whatever q holds there."""
        T = self._types()
        dt = q.dtype
        if q.ndim != 4 or k.ndim != 4 or k.dtype is not dt or dt not in T:
            raise ValueError("cache_weights: q (batch, rows, heads, head_dim), k (batch, length, kv_heads, head_dim) of "
                             "one type, f16 or bf16")
        B, R, heads, D = q.shape
        Bk, L, kv, Dk = k.shape
        if Bk != B or Dk != D or acc.shape != (B, kv, L) or T.get(acc.dtype) != 0:
            raise ValueError("cache_weights: acc is f32 of (batch, kv_heads, length), q and k of one batch and head_dim")
        if not self._flat(lens, (B,), T["i32"]):
            raise ValueError("cache_weights: lens is int32 of (batch,)")
        if lse.shape != (B, R, heads) or T.get(lse.dtype) != 0 or not lse.is_contiguous():
            raise ValueError("cache_weights: lse is f32 of (batch, rows, heads)")
        sq, sk, sa = q.stride(), k.stride(), acc.stride()
        if sq[3] != 1 or sk[3] != 1 or (sa[2] != 1 and L > 1):
            raise ValueError("cache_weights: the last dimension of q, k and acc must be contiguous")
        a = _lib.CACHE_WEIGHT.pack(*self._ptrs("cache_weights", q, k, lens, lse, acc), *sq[:3], *sk[:3], *sa[:2],
                                   D ** -0.5 if scale is None else scale, decay, B, R, heads, kv, D, L,
                                   1 if causal else 0, T[dt])
        rc = self.L.dc_cache_weights_dev(self.h, a)
        if rc:
            self._check(rc, "cache_weights")

    def cache_evict_dev(self, k, v, acc, lens, k_out, v_out, acc_out, index, lens_out, *, budget: int,
                        recent: int = 0) -> None:
        """Writes the kept tokens of a batch's cache to another one, for each
        sequence and key/value head: all where lens[b] <= budget, else the last
        `recent` and, of those before, the budget - recent of largest acc (equal
        ones: the lower index; a NaN is the lowest), in their order.

        k, v (batch, length, kv_heads, head_dim) and acc (batch, kv_heads, length,
        f32); k_out, v_out, acc_out and index (batch, kv_heads, .., int32: each kept
        token's old place) alike, with room for `budget` tokens; lens, lens_out
        (batch, int32).  What lies behind a sequence's last kept token is left as
        it is.  Heads keep different tokens but equally many.  The outputs must not
        overlap the inputs."""
        T = self._types()
        budget, recent, dt = int(budget), int(recent), k.dtype
        if k.ndim != 4 or v.shape != k.shape or v.dtype is not dt or dt not in T:
            raise ValueError("cache_evict: k and v are (batch, length, kv_heads, head_dim) of one type")
        B, L, kv, D = k.shape
        room = min(budget, L)
        if k_out.ndim != 4 or v_out.shape != k_out.shape or k_out.dtype is not dt or v_out.dtype is not dt or (
                k_out.shape[1] < room or k_out.shape != (B, k_out.shape[1], kv, D)):
            raise ValueError("cache_evict: k_out and v_out are as k, with room for the budget")
        if acc.shape != (B, kv, L) or T.get(acc.dtype) != 0:
            raise ValueError("cache_evict: acc is f32 of (batch, kv_heads, length)")
        for t, ok in ((acc_out, T.get(acc_out.dtype) == 0), (index, index.dtype is T["i32"])):
            if not ok or t.ndim != 3 or t.shape[2] < room or t.shape != (B, kv, t.shape[2]):
                raise ValueError("cache_evict: acc_out is f32 and index int32 of (batch, kv_heads, room for the budget)")
        if not (self._flat(lens, (B,), T["i32"]) and self._flat(lens_out, (B,), T["i32"])):
            raise ValueError("cache_evict: lens and lens_out are int32 of (batch,)")
        strides = []
        for t in (k, v, acc, k_out, v_out, acc_out, index):
            s = t.stride()
            if s[-1] != 1 and t.shape[-1] > 1:
                raise ValueError("cache_evict: the last dimension of every buffer must be contiguous")
            strides += s[:-1]
        # (a budget beyond the cache keeps all, however large: the library's integers have 32 bits)
        a = _lib.CACHE_EVICT.pack(
            *self._ptrs("cache_evict", k, v, acc, lens, k_out, v_out, acc_out, index, lens_out), *strides,
            B, kv, D, L, *(max(-1, min(n, 2 ** 31 - 1)) for n in (budget, recent)), k.element_size())
        rc = self.L.dc_cache_evict_dev(self.h, a)
        if rc:
            self._check(rc, "cache_evict")

    def measure_capacity(self, spec=None, T: int = 16, seconds: float = 0.3) -> float:
        """The capacity the ring's planner apportions layers by, in the
        reference's unit: verified 32x64x64 GEMMs per second (app.js
        measureCapacity, :508-519).  Without ``spec`` it is that probe itself
        (vgemmBlock of the same X = sin(i)/2, W = cos(i)/2, each call waited
        for).  With a model ``spec`` it is measured at the real shapes: the
        four projection GEMMs of a T-row chunk (QKV, O, gate/up, down) on
        device-resident int8 weights, back to back, as MACs per second over the
        probe's 32*64*64 MACs -- the unit shard.estimate_lap_ms divides by."""
        import time

        import torch
        from .shard import UNIT_MACS
        dev = torch.device("cuda", self.device)
        if spec is None:
            m, k, n = 32, 64, 64
            X = torch.from_numpy((np.sin(np.arange(m * k)) * 0.5).astype(np.float32)).to(dev)
            w = self.register_weight((np.cos(np.arange(k * n)) * 0.5).astype(np.float32), k, n)
            out = torch.empty(m * n, dtype=torch.float32, device=dev)
            self.vgemm_dev(X, m, w, 0, out)
            self.sync()
            t0, it = time.perf_counter(), 0
            while time.perf_counter() - t0 < seconds:
                self.vgemm_dev(X, m, w, 0, out)
                self.sync()
                it += 1
            return it / (time.perf_counter() - t0)
        C_, hd = spec.hidden, spec.headDim or spec.hidden // spec.heads
        q, kv, I_ = spec.heads * hd, spec.kvHeads * hd, spec.inter
        g = torch.Generator(device=dev)
        g.manual_seed(0x5EED)
        ops = []
        for k, n in ((C_, q + 2 * kv), (q, C_), (C_, 2 * I_), (I_, C_)):
            ld = (k + 15) // 16 * 16
            wt = torch.randint(-127, 128, (n, ld), dtype=torch.int8, device=dev, generator=g)
            xq = torch.randint(-127, 128, (T, ld), dtype=torch.int8, device=dev, generator=g)
            cs = torch.rand(n, device=dev, generator=g) * 1e-3
            rs = torch.rand(T, device=dev, generator=g)
            out = torch.empty(T * n, dtype=torch.float32, device=dev)
            ops.append((xq, ld, wt, rs, cs, k, n, out))

        def one_pass():
            for xq, ld, wt, rs, cs, k, n, out in ops:
                self.bgemm_dev(xq, ld, wt, ld, rs, cs, T, k, n, 1, 0, out)

        one_pass()
        self.sync()
        t0, passes = time.perf_counter(), 0
        while True:
            for _ in range(8):
                one_pass()
            passes += 8
            self.sync()
            el = time.perf_counter() - t0
            if el >= seconds:
                break
        macs = T * sum(k * n for _, _, _, _, _, k, n, _ in ops)
        return macs * passes / UNIT_MACS / el

    def kernel_probe(self) -> int:
        """kernelProbe's int32 hash (webgpu.js:1047-1055, before the math fold)."""
        h = C.c_uint32()
        self._check(self.L.dc_kernel_probe(self.h, C.byref(h)), "kernel_probe")
        return h.value


class Weight:
    """A weight quantised once and resident in HBM (dc_weight_register)."""

    def __init__(self, comp: Compute, W: np.ndarray, k: int, n: int):
        self.comp = comp
        W = np.ascontiguousarray(W, np.float32).reshape(-1)
        if W.size != k * n:
            raise ValueError("weight: size does not match k x n")
        h = C.c_void_p()
        comp._check(comp.L.dc_weight_register(comp.h, _ptr(W), k, n, C.byref(h)), "weight_register")
        self.h = h
        self.k, self.n = k, n
        qt, ld, cs = C.c_void_p(), C.c_int(), C.c_void_p()
        comp.L.dc_weight_info(self.h, C.byref(qt), C.byref(ld), C.byref(cs), None, None)
        self.qt_ptr, self.ldw, self.cs_ptr = qt.value, ld.value, cs.value

    def __del__(self):
        try:
            if self.h:
                self.comp.L.dc_weight_free(self.h)
                self.h = None
        except Exception:
            pass


def init_compute(device: int = 0, stream=None) -> Compute:
    """initCompute (webgpu.js:284): a gated compute object, or an exception."""
    return Compute(device, stream)
