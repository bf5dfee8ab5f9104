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
import operator
import struct

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, dtype_code, ptr
from .ext import _require_device

FORMATS = {"fp16": 0, "bf16": 1, "fp8": 2, "fp8_int4": 3}
_NEW = {"fp16": torch.float16, "bf16": torch.bfloat16}
# A plain call goes through the compiled module of csrc/fkv_calls.cpp, which
# does what stands here behind it; NotImplemented: it has done nothing, and the
# call is checked, and its arguments copied where they must be, here.
#
# fkv_rows and fkv_positions (include/fkv.h) as bytes
_pack_rows = struct.Struct("Pqqq").pack
_pack_positions = struct.Struct("Pqqqii").pack


# ---------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------

def _on(index, name, t):
    """Refuses what is not a tensor on GPU ``index``, wants a gradient or
    carries a forward-mode tangent."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.get_device() != index:
        _require_device(t)
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires grad: this package is for inference and records nothing for autograd "
                           "(call it under torch.no_grad())")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{name} has a forward-mode tangent: this package is for inference and would drop it")


_raw_stream, _current_gpu = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _call(index, what, *args):
    """The entry point ``what`` on GPU ``index``'s current stream, that GPU
    being current (switched to only where it is not)."""
    fn = getattr(_lib.load(), what)
    if _current_gpu() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        check(rc, what)


def _rows(t, shape):
    """(B, H, L, D) tensor of that shape as C rows, copied only where its last
    dimension is strided or a row not 16-byte aligned -> (rows, tensor)."""
    at, (sb, sh, sl, sd) = t.data_ptr(), t.stride()
    if sd != 1 or at & 15 or (sb | sh | sl) & 7:
        # (strides of dimensions of one element mean nothing)
        B, H, L, _ = shape
        sb, sh, sl = sb if B > 1 else 0, sh if H > 1 else 0, sl if L > 1 else 0
        if sd != 1 or at & 15 or (sb | sh | sl) & 7:
            t = t.clone(memory_format=torch.contiguous_format)
            at, (sb, sh, sl, _) = t.data_ptr(), t.stride()
    return _pack_rows(at, sb, sh, sl), t


def _result(index, name, t, shape, dtype):
    """Refuses a result tensor that does not fit, or whose rows share memory."""
    _on(index, name, t)
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{name} must have shape {tuple(shape)} and dtype {dtype}, got {tuple(t.shape)} {t.dtype}")
    if 0 in t.stride() and any(s == 0 and n > 1 for s, n in zip(t.stride(), shape)):
        raise ValueError(f"{name} is an expanded tensor: its rows share memory")


def _positions(p, B, L, index, per_token_allowed=True):
    """int | one-element tensor | (B,) tensor: the first token's position of
    each sequence; (B, L) or (1, L): every token's."""
    if not isinstance(p, torch.Tensor):
        return _pack_positions(0, 0, 0, int(p), 0, 0)
    dtype = p.dtype
    is64 = dtype == torch.int64
    if not is64 and dtype != torch.int32:
        raise TypeError(f"positions must be int32 or int64, got {dtype}")
    _on(index, "positions", p)
    shape, at = p.shape, p.data_ptr()
    if shape == (B,):
        return _pack_positions(at, p.stride(0), 0, 0, is64, 0)
    if shape == () or shape == (1,):
        return _pack_positions(at, 0, 0, 0, is64, 0)
    if per_token_allowed and shape in ((B, L), (1, L)):
        return _pack_positions(at, p.stride(0) if shape[0] > 1 else 0, p.stride(1), 0, is64, 1)
    raise ValueError(f"positions must be one number, one per sequence ({B},)"
                     f"{f' or one per token {(B, L)}' if per_token_allowed else ''}, got {tuple(shape)}")


def _lens(name, t, B, index):
    _on(index, name, t)
    if t.dtype != torch.int32 or t.shape != (B,):
        raise TypeError(f"{name} must be an int32 tensor of shape ({B},)")
    return t if B <= 1 or t.stride(0) == 1 else t.contiguous()


def _index_of(device):
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        return torch.device("cuda", torch.cuda.current_device())
    return device


class _Fixed:
    """An object whose attributes say what its calls, which know addresses
    and sizes, work on: another value would change nothing there."""

    def __setattr__(self, name, value):
        if "_key" in self.__dict__ and name in self.__dict__:
            raise AttributeError(f"{name} cannot be set: a {type(self).__name__} is made for what it holds (make another one)")
        super().__setattr__(name, value)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

def _frequencies(rot_dim, base, scaling):
    """Angle per position of each pair in 64 bits, and the factor that cos and
    sin carry."""
    i = torch.arange(rot_dim // 2, dtype=torch.float64, device="cpu")  # (whose numbers the library reads on the host)
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


class Rope(_Fixed):
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
        if head_dim % 8 or head_dim > 512:
            raise ValueError(f"the head dim must be a multiple of 8, at most 512, got {head_dim}")
        self.head_dim, self.rot_dim, self.interleaved = int(head_dim), int(rot_dim), bool(interleaved)
        self.base, self.scaling, self.max_positions = float(base), scaling, int(max_positions)
        inv, factor = _frequencies(self.rot_dim, self.base, scaling)
        device = _index_of(device)
        self.table = torch.empty((self.max_positions, 2, self.rot_dim // 2), dtype=torch.float32, device=device)
        if device.type == "cuda":
            _call(device.index, "fkv_rope_table", inv.data_ptr(), self.rot_dim, factor, self.max_positions,
                  self.table.data_ptr())
        else:  # (to look at: calls take tables on a GPU)
            a = torch.arange(self.max_positions, dtype=torch.float64, device="cpu")[:, None] * inv
            self.table[:, 0], self.table[:, 1] = a.cos() * factor, a.sin() * factor
        c = _lib.RopeC(self.table.data_ptr(), self.max_positions, self.rot_dim, int(self.interleaved))
        self._c, self._index = ctypes.byref(c), self.table.get_device()
        self._key = ctypes.addressof(c), self._index, self.head_dim

    def __call__(self, x, positions=0, out=None):
        """x (B, H, L, head_dim) fp16 / bf16 / fp32, any strides -> the rotated
        rows, in ``out`` (may be x itself, and shares no memory with it
        otherwise; default a new tensor like x).
        ``positions``: a number or one-element tensor (the first token's
        position), a (B,) tensor (each sequence's first token's) or (B, L) /
        (1, L) (every token's); int32 or int64 tensors on the device, read
        there, so a captured call follows them."""
        done = _lib.calls().rope(self._key, x, positions, out)
        if done is not NotImplemented:
            return done
        index = self._index
        if index < 0:
            _require_device(self.table)
        _on(index, "x", x)
        shape, dtype = x.shape, x.dtype
        if len(shape) != 4 or shape[3] != self.head_dim:
            raise ValueError(f"x must be (B, H, L, {self.head_dim}), got {tuple(shape)}")
        code = dtype_code(dtype)
        if out is None:
            out = torch.empty_like(x)
        else:
            _result(index, "out", out, shape, dtype)
        B, H, L, D = shape
        pos = _positions(positions, B, L, index)
        src, held = _rows(x, shape)
        dst, result = _rows(out, shape)
        _call(index, "fkv_rope_apply", self._c, src, dst, code, B, H, L, D, pos)
        if result is not out:
            out.copy_(result)
        return out


# ---------------------------------------------------------------------------
# one layer
# ---------------------------------------------------------------------------

class PagedLayer(_Fixed):
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
            _on(k.get_device(), name, t)
        self.fmt, self.k, self.v, self.k_exp, self.v_scale = fmt, k, v, k_exp, v_scale
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = n, H, page, D
        self.device, self._index = k.device, k.get_device()
        c = _lib.PagesC(k.data_ptr(), v.data_ptr(), ptr(k_exp), ptr(v_scale), n, page, H, D, FORMATS[fmt])
        self._c = ctypes.byref(c)
        check(min(int(_lib.load().fkv_paged_attn_workspace(self._c, H, 1, 0)), 0), "PagedLayer")
        self._key = ctypes.addressof(c), self._index

    def _table(self, table, B=None):
        """-> table, its rows, pages per sequence and row stride."""
        _on(self._index, "table", table)
        if table.dtype != torch.int32 or table.dim() != 2:
            raise TypeError("table must be a (B, pages per sequence) int32 tensor")
        rows, P = table.shape
        if B is not None and rows != B:
            raise ValueError(f"table must have {B} rows, got {(rows, P)}")
        stride, step = table.stride()
        if (P > 1 and step != 1) or (rows > 1 and stride < P):
            table = table.contiguous()
            stride = P
        return table, rows, P, stride if rows > 1 else P

    def memory_bytes(self):
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_exp, self.v_scale) if t is not None)

    def write(self, k, v, table, start, n_new=None, q=None, rope=None, q_out=None):
        """Stores L new tokens of B sequences: k, v (B, H, L, D) fp16 / bf16 /
        fp32, any strides, token (b, l) at position start(b) + l of its
        sequence (``start``: a number, a one-element tensor or (B,), int32 or
        int64 on the device).  Keys, and the queries q (B, Hq, L, D) of the
        same dtype where given, are rotated by ``rope`` first; returns the
        rotated queries (``q_out``, which may be q, and shares no memory with
        q, k or v otherwise; default a new tensor), or None without q.

        ``n_new`` (B,) int32 on the device: only the first n_new[b] tokens of
        sequence b are real; the rest of a padded batch is not stored, and
        its queries come back as ``q_out`` held them (zero in a new tensor).
        Positions outside the table are not stored either.  No two tokens of
        a call may name the same slot."""
        done = _lib.calls().write(self._key, k, v, table, start, n_new, q, None if rope is None else rope._key, q_out)
        if done is not NotImplemented:
            return done
        index = self._index
        _on(index, "k", k)
        _on(index, "v", v)
        shape, dtype = k.shape, k.dtype
        if len(shape) != 4 or shape[1] != self.n_kv_heads or shape[3] != self.head_dim or v.shape != shape or \
                v.dtype != dtype:
            raise ValueError(f"k and v must be (B, {self.n_kv_heads}, L, {self.head_dim}) of one dtype, got "
                             f"{tuple(shape)} {dtype} / {tuple(v.shape)} {v.dtype}")
        B, H, L, D = shape
        code = dtype_code(dtype)
        table, _, P, stride = self._table(table, B)
        rope_c = None
        if rope is not None:
            if rope.head_dim != D:
                raise ValueError(f"rope is for head dim {rope.head_dim}, not {D}")
            _on(index, "rope", rope.table)
            rope_c = rope._c
        pos = _positions(start, B, L, index, per_token_allowed=False)
        if n_new is not None:
            n_new = _lens("n_new", n_new, B, index)
        rk, k_held = _rows(k, shape)
        rv, v_held = _rows(v, shape)
        rq = ro = result = None
        Hq = 0
        if q is not None:
            _on(index, "q", q)
            qs = q.shape
            if len(qs) != 4 or qs[0] != B or qs[2] != L or qs[3] != D or q.dtype != dtype:
                raise ValueError(f"q must be ({B}, Hq, {L}, {D}) {dtype}, got {tuple(qs)} {q.dtype}")
            if q_out is None:
                q_out = torch.empty_like(q) if n_new is None else torch.zeros_like(q)
            else:
                _result(index, "q_out", q_out, qs, dtype)
            Hq = qs[1]
            rq, q_held = _rows(q, qs)
            ro, result = _rows(q_out, qs)
        elif q_out is not None:
            raise ValueError("q_out without q")
        _call(index, "fkv_paged_write", self._c, rk, rv, code, B, L, table.data_ptr(), P, stride, pos,
              None if n_new is None else n_new.data_ptr(), rope_c, rq, ro, Hq)
        if result is not q_out:
            q_out.copy_(result)
        return q_out

    def read(self, table, lens, max_len=None, dtype=None):
        """K and V (B, H, max_len, D) of B sequences out of their pages, in
        ``dtype`` (default: the pages' own, fp16 for quantised ones); rows
        past lens[b] ((B,) int32 on the device) are zero.  ``max_len``
        defaults to the table's width in tokens."""
        done = _lib.calls().read(self._key, table, lens, max_len, dtype)
        if done is not NotImplemented:
            return done
        table, B, P, stride = self._table(table)
        lens = _lens("lens", lens, B, self._index)
        S = P * self.page_size if max_len is None else int(max_len)
        if not 0 <= S < 2 ** 31:
            raise ValueError(f"max_len must be in [0, 2^31), got {S}")
        dtype = _NEW.get(self.fmt, torch.float16) if dtype is None else dtype
        code = dtype_code(dtype)
        k = torch.empty((B, self.n_kv_heads, S, self.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        _call(self._index, "fkv_paged_read", self._c, table.data_ptr(), P, stride, lens.data_ptr(), B, S, k.data_ptr(),
              v.data_ptr(), code)
        return k, v

    def attend(self, query, table, lens, max_len=None, lens_add=0, scale=None, out=None, return_lse=False):
        """Attention of one new token per sequence, query (B, Hq, 1, D) fp16
        or bf16 (the pages' own type where they hold 16 bits), over the first
        lens[b] + lens_add tokens of its pages -> out (B, Hq, 1, D) of the
        query's type, and with ``return_lse`` the natural logarithm (B, Hq)
        fp32 of each head's sum of exponentials (by which several such results
        are joined).  A sequence without tokens gives zeros and -inf; one that
        has an infinite value among its tokens NaN or infinity in that dim.

        ``out`` may be the query where that is contiguous.  ``max_len`` is an
        upper bound of the lengths if the host knows one
        (default: the table's width); it decides how the work is split, not
        what is attended to.  ``scale`` defaults to D^-1/2."""
        done = _lib.calls().attend(self._key, query, table, lens, max_len, lens_add, scale, out, return_lse)
        if done is not NotImplemented:
            return done
        index, D = self._index, self.head_dim
        _on(index, "query", query)
        shape, dtype = query.shape, query.dtype
        if len(shape) != 4 or shape[2] != 1 or shape[3] != D or shape[1] % self.n_kv_heads or shape[1] == 0:
            raise ValueError(f"query must be (B, a multiple of {self.n_kv_heads}, 1, {D}), got {tuple(shape)}")
        if dtype not in (torch.float16, torch.bfloat16) or dtype != _NEW.get(self.fmt, dtype):
            raise TypeError(f"{self.fmt} pages take {'fp16 or bf16' if self.fmt not in _NEW else self.fmt} queries, "
                            f"got {dtype}")
        B, Hq = shape[:2]
        table, _, P, stride = self._table(table, B)
        lens = _lens("lens", lens, B, index)
        most = P * self.page_size
        if max_len is not None and max_len < most:
            most = int(max_len)
        if not -2 ** 31 <= lens_add < 2 ** 31:
            raise ValueError(f"lens_add must fit 32 bits, got {lens_add}")
        rows, held = _rows(query, shape)
        if out is None:
            out = torch.empty_like(query, memory_format=torch.contiguous_format)
        else:
            _on(index, "out", out)
            if out.shape != shape or out.dtype != dtype or not out.is_contiguous() or out.data_ptr() % 16:
                raise ValueError(f"out must be a contiguous, 16-byte aligned {tuple(shape)} {dtype} tensor")
        lse = torch.empty((B, Hq), dtype=torch.float32, device=self.device) if return_lse else None
        n = _lib.load().fkv_paged_attn_workspace(self._c, Hq, B, most)
        if n < 0:
            check(n, "fkv_paged_attn_workspace")
        ws = torch.empty(n, dtype=torch.uint8, device=self.device) if n else None
        _call(index, "fkv_paged_attn", self._c, rows, dtype_code(dtype), Hq, B, table.data_ptr(), P, stride,
              lens.data_ptr(), lens_add, most, D ** -0.5 if scale is None else scale, out.data_ptr(), ptr(lse),
              None if ws is None else ws.data_ptr(), n)
        return (out, lse) if return_lse else out


# ---------------------------------------------------------------------------
# layers that grow together
# ---------------------------------------------------------------------------

class PageTable:
    """Which pages hold which sequence's tokens, for ``max_seqs`` sequences of
    up to ``max_tokens`` tokens over a pool of ``n_pages`` pages.

    On the device: ``table`` (max_seqs, pages per sequence) int32, -1 where
    nothing is held, ``lens``, ``start`` and ``new`` (max_seqs,) int32: the
    tokens of each sequence now, before its last ``extend``, and their
    difference.  The host keeps its own copy and hands out pages; device
    updates are work on the current stream."""

    def __init__(self, n_pages, page_size, max_seqs, max_tokens, device="cuda"):
        n_pages, page_size, max_seqs, max_tokens = (int(x) for x in (n_pages, page_size, max_seqs, max_tokens))
        if min(n_pages, page_size, max_seqs, max_tokens) < 1:
            raise ValueError("pages, page size, sequences and tokens must be positive")
        self.n_pages, self.page_size, self.max_seqs, self.max_tokens = n_pages, page_size, max_seqs, max_tokens
        width = -(-max_tokens // page_size)
        self.table = torch.full((max_seqs, width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.start = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.new = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages = [[] for _ in range(max_seqs)]
        self._lens = [0] * max_seqs
        self._new = [0] * max_seqs

    @property
    def free_pages(self):
        return len(self._free)

    def lengths(self, seqs=None):
        """Tokens of the sequences, from the host's copy."""
        return self._lens[self._range(seqs)]

    def starts(self, seqs=None):
        """Tokens of the sequences before their last ``extend``, from the
        host's copy."""
        sl = self._range(seqs)
        return [n - t for n, t in zip(self._lens[sl], self._new[sl])]

    def pages(self, seq):
        """Page ids of one sequence, in order."""
        return list(self._pages[seq])

    def _range(self, seqs):
        if seqs is None:
            return slice(0, self.max_seqs)
        first, stop, step = seqs.indices(self.max_seqs)
        if step != 1 or stop < first:
            raise ValueError(f"seqs must be a slice of neighbouring sequences, got {seqs}")
        return slice(first, stop)

    @staticmethod
    def _each(n, count):
        """A number for all of them, or one for each."""
        if hasattr(n, "__index__") and not getattr(n, "ndim", 0):
            return [operator.index(n)] * count
        each = [int(t) for t in n]
        if len(each) != count:
            raise ValueError(f"{len(each)} numbers of tokens for {count} sequences")
        return each

    def _not_captured(self):
        if self.table.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("pages are handed out on the host: extend, reserve and free outside of a capture, or "
                               "capture the layer's calls with lengths of your own")

    def _view(self, t, sl):
        # (a slice of a tensor takes longer than a decode step's kernel launch)
        return t if sl.stop - sl.start == self.max_seqs else t[sl]

    def reserve(self, tokens, seqs=None):
        """Gives each sequence the pages for ``tokens`` tokens (a number, or one
        per sequence) in all; those it holds stay.  Raises MemoryError, and
        changes nothing, where the pool or a sequence's row is too small."""
        self._not_captured()
        sl = self._range(seqs)
        each = range(sl.start, sl.stop)
        want = self._each(tokens, len(each))
        if want and max(want) > self.max_tokens:
            raise MemoryError(f"a sequence of {max(want)} tokens: the table holds {self.max_tokens}")
        more = [max(0, -(-t // self.page_size) - len(self._pages[b])) for b, t in zip(each, want)]
        if sum(more) > len(self._free):
            raise MemoryError(f"{sum(more)} pages needed, {len(self._free)} free")
        rows, cols, ids = [], [], []
        for b, n in zip(each, more):
            for _ in range(n):
                rows.append(b)
                cols.append(len(self._pages[b]))
                ids.append(self._free.pop())
                self._pages[b].append(ids[-1])
        if ids:
            d = self.table.device
            self.table[torch.tensor(rows, device=d), torch.tensor(cols, device=d)] = \
                torch.tensor(ids, dtype=torch.int32, device=d)

    def extend(self, n=1, seqs=None):
        """``n`` more tokens (a number, or one per sequence): reserves their
        pages and advances start, new and lens."""
        self._not_captured()
        sl = self._range(seqs)
        each = self._each(n, sl.stop - sl.start)
        if each and min(each) < 0:
            raise ValueError("sequences do not shrink (free them)")
        self.reserve([a + t for a, t in zip(self._lens[sl], each)], seqs=sl)
        start, new, lens = (self._view(t, sl) for t in (self.start, self.new, self.lens))
        start.copy_(lens)
        if self._new[sl] != each:
            new.copy_(torch.tensor(each, dtype=torch.int32))
            self._new[sl] = each
        lens.add_(new)
        self._lens[sl] = [a + t for a, t in zip(self._lens[sl], each)]

    def free(self, seq):
        """Sequence ``seq`` is over: its pages go back to the pool."""
        if not 0 <= seq < self.max_seqs:
            raise ValueError(f"no sequence {seq}")
        self._not_captured()
        self._free.extend(reversed(self._pages[seq]))
        self._pages[seq] = []
        self._lens[seq] = self._new[seq] = 0
        self.table[seq].fill_(-1)
        for t in (self.lens, self.start, self.new):
            t[seq].fill_(0)


class PagedKVCache:
    """``n_layers`` layers of pages over one ``PageTable``:

        cache = PagedKVCache(n_layers, n_kv_heads, head_dim, n_pages, max_seqs, max_tokens, fmt="fp8", rope=rope)
        cache.extend(n)                          # n tokens more per sequence
        q = cache.write(layer, k, v, q)          # rotated, encoded, stored
        out = cache.attend(layer, q)             # one-token queries
        k, v = cache.read(layer)                 # what is stored

    ``seqs`` (a slice, default all sequences) picks the neighbouring
    sequences that a call's batch stands for.  With ``rope`` the cache rotates
    what it is handed; without it keys and queries come rotated."""

    def __init__(self, n_layers, n_kv_heads, head_dim, n_pages, max_seqs=1, max_tokens=32768, page_size=64,
                 fmt="fp16", rope=None, device="cuda"):
        if rope is not None and rope.head_dim != head_dim:
            raise ValueError(f"rope is for head dim {rope.head_dim}, not {head_dim}")
        self.layers = [PagedLayer(n_pages, n_kv_heads, head_dim, page_size, fmt, device) for _ in range(n_layers)]
        self.pages = PageTable(n_pages, page_size, max_seqs, max_tokens, device)
        self.rope, self.fmt = rope, fmt

    def extend(self, n=1, seqs=None):
        """As ``PageTable.extend``; with one number per sequence, a write's
        batch is padded to the largest of them.  Raises ValueError, and changes
        nothing, where a token would stand past the rotary table, whose keys
        would be NaN."""
        if self.rope is not None:
            sl = self.pages._range(seqs)
            n = self.pages._each(n, sl.stop - sl.start)
            most = max((a + t for a, t in zip(self.pages._lens[sl], n) if t > 0), default=0)
            if most > self.rope.max_positions:
                raise ValueError(f"a sequence of {most} tokens: the rotary table holds {self.rope.max_positions} positions")
        self.pages.extend(n, seqs)

    def free(self, seq):
        self.pages.free(seq)

    def _batch(self, seqs):
        sl = self.pages._range(seqs)
        return sl, self.pages._view(self.pages.table, sl)

    def write(self, layer, k, v, q=None, seqs=None, q_out=None):
        """The new tokens of the last ``extend`` of the same sequences; see
        ``PagedLayer.write``."""
        sl, table = self._batch(seqs)
        new = self.pages._new[sl]
        if new and max(new) != k.shape[2]:
            raise ValueError(f"k holds {k.shape[2]} tokens, the last extend made room for {max(new)}")
        n_new = None if len(set(new)) <= 1 else self.pages._view(self.pages.new, sl)
        return self.layers[layer].write(k, v, table, self.pages._view(self.pages.start, sl), n_new=n_new, q=q, rope=self.rope,
                                        q_out=q_out)

    def attend(self, layer, query, seqs=None, scale=None, out=None):
        sl, table = self._batch(seqs)
        return self.layers[layer].attend(query, table, self.pages._view(self.pages.lens, sl), max(self.pages._lens[sl], default=0),
                                         scale=scale, out=out)

    def read(self, layer, seqs=None, dtype=None):
        """K, V (B, H, longest length, D); rows past a sequence's length are
        zero."""
        sl, table = self._batch(seqs)
        return self.layers[layer].read(table, self.pages._view(self.pages.lens, sl), max(self.pages._lens[sl], default=0), dtype)

    def to_foveated(self, cfg=None, seqs=None, importance=None):
        """A ``FoveatedKVCache`` of the sequences' contexts, compressed into
        tiers: a prompt prefilled into pages decodes on with the fused
        two-tier attention.  The sequences must have one length."""
        from .tier_cache import FoveatedKVCache

        lens = self.pages.lengths(seqs)
        if not lens or len(set(lens)) != 1 or lens[0] == 0:
            raise ValueError(f"tiers need sequences of one length, got {lens}")
        cache = FoveatedKVCache(cfg)
        for i in range(len(self.layers)):
            cache.update(*self.read(i, seqs), i)
        cache.compress(importance=importance)
        return cache

    def memory_bytes(self):
        return sum(layer.memory_bytes() for layer in self.layers)
