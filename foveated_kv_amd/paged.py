"""A paged KV cache beside the foveated one: many sequences of different
lengths that grow token by token, held exactly (fp16 / bf16) or quantised as
they are written (E4M3 keys and values, or E4M3 keys and INT4 values), and
attended to in place.

  Rope            rotary positions: half or interleaved pairs, part of the
                  head, scaled for long contexts
  PagedLayer      one layer's pages: write (rotate, encode, store), read
                  (decode, gather) and attend (one new token a sequence)
  PagedKVCache    layers that share one page table and one set of lengths,
                  pages handed out as sequences grow

The reference has no such cache: it keeps a prompt's K and V whole until
they are compressed into tiers.  ``PagedKVCache.to_foveated`` does the latter
from pages, ``generate.generate_paged`` serves a batch of prompts.

Like the rest of the package this is for inference: nothing is recorded by
autograd.  Calls run on torch's current stream of the tensors' device, and
every call's workspace comes from torch's caching allocator for that call
alone, so calls on several streams and several captured graphs do not share
any.  A page, once written by one stream and read by another, is ordered by
the caller, as any tensor is.
"""

import ctypes
import math

import torch

from . import _lib
from ._lib import check, dtype_code, ptr
from .ext import _require_device

FORMATS = {"fp16": 0, "bf16": 1, "fp8": 2, "fp8_int4": 3}
_NEW = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------

def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}")


def _no_grad_needed(**tensors):
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} requires grad: this package is for inference and records nothing for "
                                   "autograd (call it under torch.no_grad())")


def _rows(t):
    """(B, H, L, D) tensor as C rows, copied only if its last dimension is
    strided or a row not 16-byte aligned -> (rows, tensor)."""
    if t.stride(3) != 1 or t.data_ptr() % 16 or any(t.shape[i] > 1 and t.stride(i) % 8 for i in range(3)):
        t = t.clone(memory_format=torch.contiguous_format)
    s = [t.stride(i) if t.shape[i] > 1 else 0 for i in range(3)]
    return _lib.RowsC(t.data_ptr(), *s), t


def _int_tensor(name, t):
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")


def _positions(p, B, L, device, per_token_allowed=True):
    """int | one-element tensor | (B,) tensor: the first token's position of
    each sequence; (B, L) or (1, L): every token's."""
    if not torch.is_tensor(p):
        return _lib.PositionsC(None, 0, 0, int(p), 0, 0), None
    _int_tensor("positions", p)
    _same_device(device, positions=p)
    is64 = int(p.dtype == torch.int64)
    if p.dim() == 2 and per_token_allowed:
        if p.shape[0] not in (1, B) or p.shape[1] != L:
            raise ValueError(f"positions must be (B, L) = {(B, L)}, (B,) or one number, got {tuple(p.shape)}")
        return _lib.PositionsC(p.data_ptr(), p.stride(0) if p.shape[0] > 1 else 0, p.stride(1), 0, is64, 1), p
    if p.dim() == 0 or (p.dim() == 1 and p.shape[0] == 1):
        return _lib.PositionsC(p.data_ptr(), 0, 0, 0, is64, 0), p
    if p.dim() != 1 or p.shape[0] != B:
        raise ValueError(f"positions must hold one number per sequence ({B}), got {tuple(p.shape)}")
    return _lib.PositionsC(p.data_ptr(), p.stride(0), 0, 0, is64, 0), p


def _lens(name, t, B, device):
    if not torch.is_tensor(t) or t.dtype != torch.int32 or tuple(t.shape) != (B,):
        raise TypeError(f"{name} must be an int32 tensor of shape ({B},)")
    _same_device(device, **{name: t})
    return t.contiguous()


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

def _frequencies(rot_dim, base, scaling):
    """Angle per position of each pair in 64 bits, and the factor that cos and
    sin carry."""
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    inv = base ** (-2.0 * i / rot_dim)
    if scaling is None:
        return inv, 1.0
    s = dict(scaling)
    kind, factor = s.pop("kind", None), float(s.pop("factor", 0.0))
    if not (math.isfinite(factor) and factor >= 1.0):
        raise ValueError(f"scaling factor must be at least 1, got {factor}")

    def need(**defaults):
        out = [float(s.pop(n)) if n in s else d for n, d in defaults.items()]
        if s or any(v is None or not v > 0 for v in out):
            raise ValueError(f"scaling {kind!r} takes {sorted(defaults)} (each positive), got {scaling}")
        return out

    if kind == "linear":
        need()
        return inv / factor, 1.0
    if kind == "ntk":
        need()
        return (base * factor ** (rot_dim / (rot_dim - 2))) ** (-2.0 * i / rot_dim), 1.0
    if kind == "bands":
        orig, low, high = need(original_positions=None, low_freq_factor=1.0, high_freq_factor=4.0)
        if high <= low:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        keep = ((orig * inv / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return inv * keep + inv / factor * (1 - keep), 1.0
    if kind == "yarn":
        orig, fast, slow = need(original_positions=None, beta_fast=32.0, beta_slow=1.0)

        def pair(turns):
            return rot_dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot_dim // 2 - 1)
        stretch = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return inv / factor * stretch + inv * (1 - stretch), 0.1 * math.log(factor) + 1.0
    raise ValueError(f"unknown scaling kind {kind!r} (linear, ntk, yarn, bands)")


class Rope:
    """Rotary positions.  Pair i of a row at position p turns by the angle
    p * f_i, f_i = base^(-2 i / rot_dim) in 64 bits, the pairs being elements
    (i, i + rot_dim / 2), or (2 i, 2 i + 1) with ``interleaved``, of the row's
    first ``rot_dim`` elements (a multiple of 16; default: all).

    ``scaling`` (None or a dict with ``kind`` and ``factor`` >= 1) stretches
    the positions for contexts longer than a model was trained on:

      linear  f / factor
      ntk     base * factor^(rot_dim / (rot_dim - 2)) in the base's place
      bands   f for pairs that turn more than ``high_freq_factor`` times over
              ``original_positions``, f / factor below ``low_freq_factor``,
              between them by their turns
      yarn    f to f / factor along a ramp over the pairs between those that
              turn ``beta_fast`` and ``beta_slow`` times over
              ``original_positions``; cos and sin times 0.1 ln(factor) + 1

    cos and sin of positions 0 .. max_positions - 1 are kept as a table of
    fp32 numbers on the device (8 bytes a position and pair); a row at any
    other position comes out NaN in its rotated elements."""

    def __init__(self, head_dim, rot_dim=None, base=10000.0, interleaved=False, scaling=None, max_positions=32768,
                 device="cuda"):
        rot_dim = head_dim if rot_dim is None else rot_dim
        if rot_dim % 16 or not 16 <= rot_dim <= head_dim:
            raise ValueError(f"rot_dim must be a multiple of 16 from 16 to the head dim, got {rot_dim}")
        if not (math.isfinite(base) and base > 1.0):
            raise ValueError(f"base must be above 1, got {base}")
        if not 1 <= max_positions < 2 ** 31:
            raise ValueError(f"max_positions must be positive and below 2^31, got {max_positions}")
        self.head_dim, self.rot_dim, self.interleaved = int(head_dim), int(rot_dim), bool(interleaved)
        self.base, self.scaling, self.max_positions = float(base), scaling, int(max_positions)
        inv, factor = _frequencies(self.rot_dim, self.base, scaling)
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        inv = inv.to(device)
        self.table = torch.empty((self.max_positions, 2, self.rot_dim // 2), dtype=torch.float32, device=device)
        for p in range(0, self.max_positions, 65536):  # (64-bit angles of 64K positions at a time)
            a = torch.arange(p, min(p + 65536, self.max_positions), dtype=torch.float64, device=device)[:, None] * inv
            self.table[p:p + 65536, 0] = a.cos() * factor
            self.table[p:p + 65536, 1] = a.sin() * factor
        self._c = _lib.RopeC(self.table.data_ptr(), self.max_positions, self.rot_dim, int(self.interleaved))

    def __call__(self, x, positions=0, out=None):
        """x (B, H, L, head_dim) fp16 / bf16 / fp32, any strides -> the rotated
        rows, in ``out`` (may be x itself; else a new tensor like x).
        ``positions``: a number or one-element tensor (the first token's
        position), a (B,) tensor (each sequence's first token's) or (B, L) /
        (1, L) (every token's); int32 or int64 tensors on the device, read
        there, so a captured call follows them."""
        _require_device(x, out)
        if x.dim() != 4 or x.shape[3] != self.head_dim:
            raise ValueError(f"x must be (B, H, L, {self.head_dim}), got {tuple(x.shape)}")
        if self.head_dim % 8 or self.head_dim > 512:
            raise ValueError("the head dim must be a multiple of 8, at most 512")
        _no_grad_needed(x=x, out=out)
        _same_device(self.table.device, x=x, out=out)
        B, H, L, D = x.shape
        code = dtype_code(x.dtype)
        if out is None:
            out = torch.empty_like(x)
        elif out.shape != x.shape or out.dtype != x.dtype:
            raise ValueError("out must have x's shape and dtype")
        pos, keep = _positions(positions, B, L, x.device)
        src, x_held = _rows(x)
        dst, result = _rows(out)
        with torch.cuda.device(x.device):
            check(_lib.load().fkv_rope_apply(ctypes.byref(self._c), ctypes.byref(src), ctypes.byref(dst), code, B, H,
                                             L, D, ctypes.byref(pos), _lib.stream_ptr(x.device)), "fkv_rope_apply")
            if result is not out:
                out.copy_(result)
        return out


# ---------------------------------------------------------------------------
# one layer
# ---------------------------------------------------------------------------

class PagedLayer:
    """One layer's pages: ``n_pages`` pages of ``page_size`` tokens (a power
    of two from 16 to 1024) for ``n_kv_heads`` heads of 64 or 128 dims.

    ``fmt``: ``fp16`` or ``bf16`` (the rows, rounded to nearest even),
    ``fp8`` (E4M3 keys and values, each row of a token and head times a power
    of two that brings its largest magnitude into (224, 448]) or ``fp8_int4``
    (keys as ``fp8``; values in 16 levels from the row's minimum to its
    maximum).  The tensors k, v, k_exp and v_scale are laid out as
    include/fkv.h says (fkv_pages).

    Which page holds which tokens is the caller's: ``table`` (B, P) int32
    holds the pages of each sequence in order, the page of tokens
    [i * page_size, (i + 1) * page_size) at (b, i).  A page id outside
    [0, n_pages) holds no tokens: nothing is stored there, it reads as zeros
    and takes no part in attention.  Entries past a sequence's last page are
    not read."""

    def __init__(self, n_pages, n_kv_heads, head_dim, page_size=64, fmt="fp16", device="cuda"):
        if fmt not in FORMATS:
            raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
        shape = (int(n_pages), int(n_kv_heads), int(page_size))
        if min(shape) < 1:
            raise ValueError(f"pages, heads and page size must be positive, got {shape}")
        D = int(head_dim)
        dt = _NEW.get(fmt, torch.uint8)
        new = dict(device=device)
        k = torch.zeros((*shape, D), dtype=dt, **new)
        v = torch.zeros((*shape, D // 2 if fmt == "fp8_int4" else D), dtype=dt, **new)
        k_exp = v_scale = None
        if dt == torch.uint8:
            k_exp = torch.full(shape, 127, dtype=torch.uint8, **new)
            v_scale = torch.full(shape, 127, dtype=torch.uint8, **new) if fmt == "fp8" else \
                torch.zeros((*shape, 2), dtype=torch.float32, **new)
        self._take(fmt, k, v, k_exp, v_scale)

    @classmethod
    def wrap(cls, fmt, k, v, k_exp=None, v_scale=None):
        """A layer over existing page tensors (kept, not copied)."""
        self = cls.__new__(cls)
        self._take(fmt, k, v, k_exp, v_scale)
        return self

    def _take(self, fmt, k, v, k_exp, v_scale):
        if fmt not in FORMATS:
            raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
        _require_device(k, v, k_exp, v_scale)
        if k.dim() != 4:
            raise ValueError(f"k must be (n_pages, H, page_size, D), got {tuple(k.shape)}")
        n, H, page, D = k.shape
        dt = _NEW.get(fmt, torch.uint8)
        want = {"k": (k, (n, H, page, D), dt), "v": (v, (n, H, page, D // 2 if fmt == "fp8_int4" else D), dt)}
        if dt == torch.uint8:
            want["k_exp"] = (k_exp, (n, H, page), torch.uint8)
            want["v_scale"] = (v_scale, (n, H, page), torch.uint8) if fmt == "fp8" else \
                (v_scale, (n, H, page, 2), torch.float32)
        elif k_exp is not None or v_scale is not None:
            raise ValueError(f"{fmt} pages have no scales")
        for name, (t, shape, dtype) in want.items():
            if t is None or tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {shape} {dtype} tensor")
            _same_device(k.device, **{name: t})
        self.fmt, self.k, self.v, self.k_exp, self.v_scale = fmt, k, v, k_exp, v_scale
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = n, H, page, D
        self.device = k.device
        self._c = _lib.PagesC(k.data_ptr(), v.data_ptr(), ptr(k_exp), ptr(v_scale), n, page, H, D, FORMATS[fmt])
        check(min(int(_lib.load().fkv_paged_attn_workspace(ctypes.byref(self._c), H, 1, 0)), 0), "PagedLayer")

    def _table(self, table):
        if not torch.is_tensor(table) or table.dtype != torch.int32 or table.dim() != 2:
            raise TypeError("table must be a (B, pages per sequence) int32 tensor")
        _same_device(self.device, table=table)
        return table if table.shape[1] <= 1 or table.stride(1) == 1 else table.contiguous()

    def memory_bytes(self):
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_exp, self.v_scale) if t is not None)

    def write(self, k, v, table, start, n_new=None, q=None, rope=None, q_out=None):
        """Stores L new tokens of B sequences: k, v (B, H, L, D) fp16 / bf16 /
        fp32, any strides, token (b, l) at position start(b) + l of its
        sequence (``start``: a number, a one-element tensor or (B,), int32 or
        int64 on the device).  Keys, and the queries q (B, Hq, L, D) of the
        same dtype where given, are rotated by ``rope`` first; returns the
        rotated queries (``q_out``, which may be q, else a new tensor), or
        None without q.

        ``n_new`` (B,) int32 on the device: only the first n_new[b] tokens of
        sequence b are real; the rest of a padded batch is not stored, and
        its queries come back as ``q_out`` held them (zero in a new tensor).
        Positions outside the table are not stored either.  No two tokens of
        a call may name the same slot."""
        _require_device(k, v, table, q, q_out, n_new)
        B, H, L, D = k.shape if k.dim() == 4 else (-1, -1, -1, -1)
        if (H, D) != (self.n_kv_heads, self.head_dim) or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError(f"k and v must be (B, {self.n_kv_heads}, L, {self.head_dim}) of one dtype, got "
                             f"{tuple(k.shape)} {k.dtype} / {tuple(v.shape)} {v.dtype}")
        code = dtype_code(k.dtype)
        table = self._table(table)
        if table.shape[0] != B:
            raise ValueError(f"table must have {B} rows, got {tuple(table.shape)}")
        _no_grad_needed(k=k, v=v, q=q, q_out=q_out)
        _same_device(self.device, k=k, v=v, q=q, q_out=q_out)
        if rope is not None:
            if rope.head_dim != D:
                raise ValueError(f"rope is for head dim {rope.head_dim}, not {D}")
            _same_device(self.device, rope=rope.table)
        pos, keep = _positions(start, B, L, self.device, per_token_allowed=False)
        if n_new is not None:
            n_new = _lens("n_new", n_new, B, self.device)
        rk, k_held = _rows(k)
        rv, v_held = _rows(v)
        rq = ro = None
        Hq = 0
        if q is None:
            if q_out is not None:
                raise ValueError("q_out without q")
        else:
            if q.dim() != 4 or (q.shape[0], q.shape[2], q.shape[3]) != (B, L, D) or q.dtype != k.dtype:
                raise ValueError(f"q must be ({B}, Hq, {L}, {D}) {k.dtype}, got {tuple(q.shape)} {q.dtype}")
            if q_out is None:
                q_out = torch.empty_like(q) if n_new is None else torch.zeros_like(q)
            elif q_out.shape != q.shape or q_out.dtype != q.dtype:
                raise ValueError("q_out must have q's shape and dtype")
            Hq = q.shape[1]
            rq, q_held = _rows(q)
            ro, result = _rows(q_out)
        with torch.cuda.device(self.device):
            ref = lambda c: None if c is None else ctypes.byref(c)  # noqa: E731
            check(_lib.load().fkv_paged_write(
                ctypes.byref(self._c), ref(rk), ref(rv), code, B, L, ptr(table), table.shape[1],
                table.stride(0) if B > 1 else table.shape[1], ctypes.byref(pos), ptr(n_new),
                None if rope is None else ctypes.byref(rope._c), ref(rq), ref(ro), Hq,
                _lib.stream_ptr(self.device)), "fkv_paged_write")
            if q is not None and result is not q_out:
                q_out.copy_(result)
        return q_out

    def read(self, table, lens, max_len=None, dtype=None):
        """K and V (B, H, max_len, D) of B sequences out of their pages, in
        ``dtype`` (default: the pages' own, fp16 for quantised ones); rows
        past lens[b] ((B,) int32 on the device) are zero.  ``max_len``
        defaults to the table's width in tokens."""
        _require_device(table, lens)
        table = self._table(table)
        B, P = table.shape
        lens = _lens("lens", lens, B, self.device)
        S = P * self.page_size if max_len is None else int(max_len)
        if S < 0:
            raise ValueError("max_len must not be negative")
        dtype = _NEW.get(self.fmt, torch.float16) if dtype is None else dtype
        out = [torch.empty((B, self.n_kv_heads, S, self.head_dim), dtype=dtype, device=self.device) for _ in range(2)]
        with torch.cuda.device(self.device):
            check(_lib.load().fkv_paged_read(
                ctypes.byref(self._c), ptr(table), P, table.stride(0) if B > 1 else P, ptr(lens), B, S,
                ptr(out[0]), ptr(out[1]), dtype_code(dtype), _lib.stream_ptr(self.device)), "fkv_paged_read")
        return tuple(out)

    def attend(self, query, table, lens, max_len=None, lens_add=0, scale=None, out=None, return_lse=False):
        """Attention of one new token per sequence, query (B, Hq, 1, D) fp16
        or bf16 (the pages' own type where they hold 16 bits), over the first
        lens[b] + lens_add tokens of its pages -> out (B, Hq, 1, D) of the
        query's type, and with ``return_lse`` the natural logarithm (B, Hq)
        fp32 of each head's sum of exponentials (by which several such results
        are joined).  A sequence without tokens gives zeros and -inf.

        ``max_len`` is an upper bound of the lengths if the host knows one
        (default: the table's width); it decides how the work is split, not
        what is attended to.  ``scale`` defaults to D^-1/2."""
        _require_device(query, table, lens, out)
        D = self.head_dim
        if query.dim() != 4 or query.shape[2] != 1 or query.shape[3] != D or query.shape[1] % self.n_kv_heads or \
                query.shape[1] == 0:
            raise ValueError(f"query must be (B, a multiple of {self.n_kv_heads}, 1, {D}), got {tuple(query.shape)}")
        if query.dtype not in (torch.float16, torch.bfloat16) or query.dtype != _NEW.get(self.fmt, query.dtype):
            raise TypeError(f"{self.fmt} pages take {'fp16 or bf16' if self.fmt not in _NEW else self.fmt} queries, "
                            f"got {query.dtype}")
        _no_grad_needed(query=query, out=out)
        table = self._table(table)
        B, Hq = query.shape[:2]
        if table.shape[0] != B:
            raise ValueError(f"table must have {B} rows, got {tuple(table.shape)}")
        lens = _lens("lens", lens, B, self.device)
        _same_device(self.device, query=query, out=out)
        P = table.shape[1]
        cap = P * self.page_size
        most = cap if max_len is None else min(int(max_len), cap)
        rows, held = _rows(query)
        if out is None:
            out = torch.empty((B, Hq, 1, D), dtype=query.dtype, device=self.device)
        elif tuple(out.shape) != (B, Hq, 1, D) or out.dtype != query.dtype or not out.is_contiguous() or \
                out.data_ptr() % 16:
            raise ValueError(f"out must be a contiguous, 16-byte aligned {(B, Hq, 1, D)} {query.dtype} tensor")
        lse = torch.empty((B, Hq), dtype=torch.float32, device=self.device) if return_lse else None
        lib = _lib.load()
        with torch.cuda.device(self.device):
            n = int(lib.fkv_paged_attn_workspace(ctypes.byref(self._c), Hq, B, most))
            check(min(n, 0), "fkv_paged_attn_workspace")
            ws = torch.empty(n, dtype=torch.uint8, device=self.device)
            check(lib.fkv_paged_attn(
                ctypes.byref(self._c), ctypes.byref(rows), dtype_code(query.dtype), Hq, B, ptr(table), P,
                table.stride(0) if B > 1 else P, ptr(lens), int(lens_add), most,
                D ** -0.5 if scale is None else float(scale), ptr(out), ptr(lse), ptr(ws), n,
                _lib.stream_ptr(self.device)), "fkv_paged_attn")
        return (out, lse) if return_lse else out
