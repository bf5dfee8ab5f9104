"""Performance cases of the paged cache's operators: what a program that
serves many sequences from a paged KV cache has the library do.

Kinds of call:

  rotary  ``Rope.__call__``: rotary positions of a projection's heads.
  write   ``PagedLayer.write``: a step's or a prompt chunk's queries and keys
          rotated, keys and values stored into their pages, 16 bits an
          element.
  store   the same into quantised pages, then ``PagedLayer.read`` of the
          whole context: the keys and values that the codes stand for (a
          chunk of a prompt that attends to what was stored before it).
  read    ``PagedLayer.read`` alone: a long context out of its pages, to be
          compressed into tiers.
  attend  ``PagedLayer.attend``: one new token of each sequence over its
          pages.

Pages are (n_pages, Hkv, page, D): 16-bit elements (``fp16``, ``bf16``);
E4M3 codes with one power of two per token and head (``fp8``); or E4M3 keys
and INT4 values (``fp8_int4``, even dims in the low nibble) with a 32-bit
scale and zero per token and head.  Inputs are made on the GPU from the seed:
K, V ~ N(0, 1) with a few outlier key channels; pages lie in random order.
"""

import math

import torch

own = False

_DEFAULTS = {"dtype": "float16", "fmt": "fp16", "page": 64, "rot": 0, "interleaved": False, "scaling": "none",
             "start": 0, "ragged": False, "layout": "blhd"}


def _case(name, kind, B, Hkv, G, D, L, **options):
    c = {"kind": kind, "B": B, "Hkv": Hkv, "G": G, "D": D, "L": L, **_DEFAULTS, **options}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one token of 64 running sequences at their own positions: the
        # smallest call, host time and latency
        _case("rotary_step_b64", "rotary", 64, 8, 4, 128, 1, dtype="bfloat16", rot=128, interleaved=True, start=30000),
        # a 16K prompt's queries, stretched positions, heads interleaved with
        # tokens as a projection leaves them
        _case("rotary_prompt_16k", "rotary", 1, 8, 4, 128, 16384, dtype="bfloat16", rot=128, scaling="yarn"),
        # one decode step of 64 sequences: q and k rotated, k and v stored
        _case("write_step_b64", "write", 64, 8, 4, 128, 1, dtype="bfloat16", fmt="bf16", rot=128, start=900),
        # a prompt of odd length on a small model, float32 activations, half
        # of each head rotated
        _case("write_prompt_odd", "write", 2, 4, 7, 64, 5003, dtype="float32", page=32, rot=32, scaling="linear",
              layout="bhld"),
        # a chunk of four prompts onto a stored beginning, 8-bit pages
        _case("store_chunk_fp8", "store", 4, 8, 4, 128, 512, dtype="bfloat16", fmt="fp8", page=32, rot=128,
              start=1536),
        # a whole prompt into 8-bit keys and 4-bit values, positions by bands
        _case("store_prompt_fp8_int4", "store", 1, 8, 4, 128, 16384, fmt="fp8_int4", rot=128, scaling="bands",
              interleaved=True),
        # a 64K context out of 8-bit pages
        _case("read_64k_fp8", "read", 1, 8, 8, 128, 65536, dtype="bfloat16", fmt="fp8"),
        # a short chat on a half-billion-parameter model: latency
        _case("attend_small_512", "attend", 1, 2, 7, 64, 512, page=16),
        # batched serving at 16K, 16-bit pages: the largest
        _case("attend_7b_16k_b8", "attend", 8, 8, 4, 128, 16384, dtype="bfloat16", fmt="bf16"),
        # 64 sequences from nothing to 8K tokens in small 8-bit pages
        _case("attend_ragged_b64_fp8", "attend", 64, 8, 4, 128, 8192, dtype="bfloat16", fmt="fp8", page=16,
              ragged=True),
        # a long document on a 70B model, 8-bit keys and 4-bit values
        _case("attend_70b_64k_fp8_int4", "attend", 1, 8, 8, 128, 65536, fmt="fp8_int4"),
        # an odd group and an odd length
        _case("attend_odd_11003", "attend", 3, 4, 5, 128, 11003, page=32),
    ]


def draw(rng):
    kind = rng.choice(["rotary", "write", "store", "read", "attend", "attend", "attend"])
    D, Hkv, G = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8]), rng.choice([1, 4, 5, 7, 8, 16])
    o = {"page": rng.choice([16, 32, 64, 128])}
    if kind in ("rotary", "write"):
        o["dtype"] = rng.choice(["float16", "bfloat16", "float32"])
        o["fmt"] = {"float16": "fp16", "bfloat16": "bf16", "float32": rng.choice(["fp16", "bf16"])}[o["dtype"]]
    else:
        o["dtype"] = rng.choice(["float16", "bfloat16"])
        plain = {"float16": "fp16", "bfloat16": "bf16"}[o["dtype"]]
        o["fmt"] = rng.choice(["fp8", "fp8_int4"] + ([] if kind == "store" else [plain, plain]))
    if kind in ("rotary", "write", "store"):
        o["rot"] = rng.choice([0 if kind != "rotary" else D, 16, D // 2, D, D])
        o["interleaved"] = rng.random() < 0.4
        o["scaling"] = rng.choice(["none", "linear", "ntk", "yarn", "bands"])
        o["layout"] = rng.choice(["blhd", "bhld"])
        o["start"] = rng.choice([0, rng.randint(1, 4000)])
    if kind == "attend":
        o["ragged"] = rng.random() < 0.5
    B = int(math.exp(rng.uniform(0, math.log(65)))) if kind in ("rotary", "write", "attend") else rng.choice([1, 2, 4])
    # most tokens times heads of a kind (the largest listed case's)
    most = {"rotary": 16384 * 32, "write": 2 * 5003 * 36, "store": 16384 * 48, "read": 65536 * 8,
            "attend": 8 * 16384 * 8}[kind]
    heads = Hkv if kind in ("read", "attend") else Hkv * G + (0 if kind == "rotary" else 2 * Hkv)
    if kind == "attend":
        most = min(most, 8 * 16384 * 32 // G)
    top = max(1, min(65536 if kind in ("read", "attend") else 16384, most // (B * heads)))
    L = 1 if kind in ("rotary", "write") and rng.random() < 0.3 else int(math.exp(rng.uniform(0, math.log(top + 1))))
    return _case(None, kind, B, Hkv, G, D, max(1, min(L, top)), **o)


# ---------------------------------------------------------------------------
# the formats and positions in plain form
# ---------------------------------------------------------------------------

_BASE = 10000.0
_SCALING = {"none": None, "linear": {"kind": "linear", "factor": 4.0}, "ntk": {"kind": "ntk", "factor": 4.0},
            "yarn": {"kind": "yarn", "factor": 4.0, "original_positions": 8192, "beta_fast": 32.0, "beta_slow": 1.0},
            "bands": {"kind": "bands", "factor": 8.0, "original_positions": 8192, "low_freq_factor": 1.0,
                      "high_freq_factor": 4.0}}


def _frequencies(case):
    """Angle per position of each pair (64 bits) and the factor of cos and sin."""
    rot, s = case["rot"], _SCALING[case["scaling"]]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    if s is None:
        return _BASE ** (-2 * i / rot), 1.0
    f = s["factor"]
    if s["kind"] == "ntk":
        return (_BASE * f ** (rot / (rot - 2))) ** (-2 * i / rot), 1.0
    inv = _BASE ** (-2 * i / rot)
    if s["kind"] == "linear":
        return inv / f, 1.0
    turns = s["original_positions"] * inv / (2 * math.pi)  # over the original context
    if s["kind"] == "bands":
        w = ((turns - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])).clamp(0, 1)
        return inv * w + inv / f * (1 - w), 1.0

    def dim(beta):  # the pair that turns beta times over the original context
        return rot * math.log(s["original_positions"] / (beta * 2 * math.pi)) / (2 * math.log(_BASE))

    lo, hi = max(math.floor(dim(s["beta_fast"])), 0), min(math.ceil(dim(s["beta_slow"])), rot // 2 - 1)
    stretched = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return inv / f * stretched + inv * (1 - stretched), 0.1 * math.log(f) + 1.0


def _cos_sin(case, positions):
    """cos and sin (B, 1, L, rot / 2) of 64-bit angles, rounded to 32 bits."""
    inv, factor = _frequencies(case)
    a = positions.double()[:, None, :, None] * inv
    return (a.cos() * factor).float(), (a.sin() * factor).float()


def _rotate(case, x, cos, sin):
    """Rows x (B, H, L, D) turned, in the precision that x has."""
    rot = case["rot"]
    if not rot:
        return x
    cos, sin = cos.to(x.dtype), sin.to(x.dtype)
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _encode8(x):
    """float32 rows -> E4M3 codes of x 2^-e and e + 127, 2^e the least power
    of two that brings the row's largest magnitude to 448 or less."""
    m, ex = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = torch.where(m > 0, torch.where(m <= 0.875, ex - 9, ex - 8).clamp_min(-126), 0)
    codes = torch.ldexp(x, -e).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, (e.squeeze(-1) + 127).to(torch.uint8)


def _decode8(codes, exps):
    return codes.view(torch.float8_e4m3fn).float() * torch.ldexp(torch.ones_like(exps, dtype=torch.float32),
                                                                 exps.int() - 127).unsqueeze(-1)


def _encode4(x):
    """float32 rows -> INT4 codes (even dims low) and (scale, zero)."""
    x = x.double()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((hi - lo) / torch.full_like(lo, 15.0)).float()
    c = torch.where(s > 0, (x - lo) / s.double(), 0.0).round().clamp(0, 15).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.cat([s, lo.float()], -1)


def _decode4(codes, sz):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    return c * sz[..., :1] + sz[..., 1:]


def _encode(fmt, k, v):
    """float32 K and V rows as the tensors of a layer's pages."""
    if fmt in ("fp16", "bf16"):
        dt = torch.float16 if fmt == "fp16" else torch.bfloat16
        return {"k": k.to(dt), "v": v.to(dt)}
    out = dict(zip(("k", "k_exp"), _encode8(k)))
    out.update(zip(("v", "v_scale"), _encode8(v) if fmt == "fp8" else _encode4(v)))
    return out


def _decode(fmt, p):
    """Rows of pages as float32 K and V."""
    if fmt in ("fp16", "bf16"):
        return p["k"].float(), p["v"].float()
    k = _decode8(p["k"], p["k_exp"])
    return k, (_decode8 if fmt == "fp8" else _decode4)(p["v"], p["v_scale"])


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _dtype(case):
    return getattr(torch, case["dtype"])


def _lengths(case, seed):
    """Tokens of each sequence's context."""
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [L] * B
    g = torch.Generator().manual_seed(7919 * seed + 13)
    u = torch.rand(B, generator=g).tolist()
    return [0 if B > 8 and i == 5 else max(1, int(round((L + 1) ** x)) - 1) for i, x in enumerate(u[:-1])] + [L]


def _inputs(case, seed):
    B, Hkv, G, D, L, page = (case[n] for n in ("B", "Hkv", "G", "D", "L", "page"))
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    def rows(heads, outliers=False):
        x = normal(B, L, heads, D) if case["layout"] == "blhd" else normal(B, heads, L, D)
        if outliers:
            x[..., torch.randperm(D, generator=g, device="cuda")[:4]] *= 8.0
        x = x.to(_dtype(case))
        return x.transpose(1, 2) if case["layout"] == "blhd" else x

    if case["kind"] == "rotary":
        x = {"x": rows(Hkv * G)}
        x["start"] = torch.randint(0, case["start"] + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        return x
    x = {}
    if case["kind"] in ("write", "store"):
        x["q"], x["k"], x["v"] = rows(Hkv * G), rows(Hkv, True), rows(Hkv)
        # each sequence's own beginning; a chunk's (store) is stored whole
        n = case["start"] + 1
        start = torch.randint(0, n, (B,), generator=g, device="cuda") if case["kind"] == "write" else \
            torch.full((B,), n - 1, device="cuda")
        x["start"] = start.to(torch.int32)
        lens = [case["start"] + L] * B
        x["lens"] = (start + L).to(torch.int32)
    else:
        lens = _lengths(case, seed)
        x["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    x["max_len"] = max(lens)
    P = -(-x["max_len"] // page)
    counts = [-(-n // page) for n in lens]
    n_pages = sum(counts) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    ends = torch.tensor(counts).cumsum(0).tolist()
    x["table"] = torch.zeros((B, P), dtype=torch.int32, device="cuda")
    for b in range(B):
        x["table"][b, :counts[b]] = order[ends[b] - counts[b]:ends[b]]
    if case["kind"] == "attend":
        q = normal(B, Hkv * G, 1, D)
        x["q"] = q.to(_dtype(case))
    channels = torch.randperm(D, generator=g, device="cuda")[:4]
    parts = []
    step = max(1, 2 ** 26 // (Hkv * page * D))  # pages that are made at a time
    for p in range(0, n_pages, step):
        k, v = normal(min(step, n_pages - p), Hkv, page, D), normal(min(step, n_pages - p), Hkv, page, D)
        k[..., channels] *= 8.0
        parts.append(_encode(case["fmt"], k.to(_dtype(case)).float(), v.to(_dtype(case)).float()))
    x["pages"] = {n: torch.cat([part[n] for part in parts]) for n in parts[0]}
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    x["case"] = case
    if own:
        from foveated_kv_amd.paged import PagedLayer, Rope

        if case["rot"]:
            last = case["start"] + case["L"]
            x["rope"] = Rope(case["D"], rot_dim=case["rot"], base=_BASE, interleaved=case["interleaved"],
                             scaling=_SCALING[case["scaling"]], max_positions=last + 1, device="cuda")
        if "pages" in x:
            x["layer"] = PagedLayer.wrap(case["fmt"], **x["pages"])
    return x


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _gather(case, x):
    """Every sequence's rows out of its pages, float32 (B, Hkv, P * page, D)."""
    flat = {n: p[x["table"].long()].transpose(1, 2).flatten(2, 3) for n, p in x["pages"].items()}
    return _decode(case["fmt"], flat)


def _read(case, x):
    k, v = _gather(case, x)
    held = torch.arange(k.shape[2], device="cuda") < x["lens"][:, None]
    return [torch.where(held[:, None, :, None], t, 0.0)[:, :, :x["max_len"]].to(_dtype(case)) for t in (k, v)]


def _plain_write(case, x):
    L, page = case["L"], case["page"]
    pos = x["start"].long()[:, None] + torch.arange(L, device="cuda")
    wide = torch.float64 if case["kind"] == "store" else torch.float32
    q, k = x["q"], x["k"].to(wide)
    if case["rot"]:
        cos, sin = _cos_sin(case, pos)
        q, k = _rotate(case, q.float(), cos, sin).to(q.dtype), _rotate(case, k, cos, sin)
    rows = _encode(case["fmt"], k.float(), x["v"].float())
    page_of = x["table"].long().gather(1, pos // page)
    for n, p in x["pages"].items():
        p[page_of, :, pos % page] = rows[n].transpose(1, 2)
    return q


def _plain_attend(case, x):
    B, Hkv, G, D = case["B"], case["Hkv"], case["G"], case["D"]
    out = []
    for b in range(0, B, 8):  # eight sequences at a time
        part = {**x, "table": x["table"][b:b + 8]}
        k, v = _gather(case, part)
        q = x["q"][b:b + 8].float().view(-1, Hkv, G, D)
        held = (torch.arange(k.shape[2], device="cuda") < x["lens"][b:b + 8, None])[:, None, None]
        s = torch.where(held, torch.matmul(q, k.transpose(-1, -2)) * D ** -0.5, -math.inf)
        w = torch.where(held, torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30)), 0.0)
        o = torch.matmul(w, v) / w.sum(-1, keepdim=True).clamp_min(1e-30)
        out.append(o.view(-1, Hkv * G, 1, D).to(_dtype(case)))
    return torch.cat(out)


def run(state):
    case, x = state["case"], state
    kind = case["kind"]
    if kind == "rotary":
        if own:
            return x["rope"](x["x"], x["start"])
        cos, sin = _cos_sin(case, x["start"][:, None] + torch.arange(case["L"], device="cuda"))
        return _rotate(case, x["x"].float(), cos, sin).to(_dtype(case))
    if kind == "read":
        return list(x["layer"].read(x["table"], x["lens"], x["max_len"], dtype=_dtype(case))) if own else \
            _read(case, x)
    if kind == "attend":
        return x["layer"].attend(x["q"], x["table"], x["lens"], x["max_len"]) if own else _plain_attend(case, x)
    if own:
        q = x["layer"].write(x["k"], x["v"], x["table"], x["start"], q=x["q"], rope=x.get("rope"))
    else:
        q = _plain_write(case, x)
    if kind == "write":
        return [q, x["pages"]["k"], x["pages"]["v"]]
    if own:
        return [q, *x["layer"].read(x["table"], x["lens"], x["max_len"], dtype=_dtype(case))]
    return [q, *_read(case, x)]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    B, Hkv, G, D, L, page = (case[n] for n in ("B", "Hkv", "G", "D", "L", "page"))
    item = torch.finfo(_dtype(case)).bits // 8
    row = {"fp16": 4 * D, "bf16": 4 * D, "fp8": 2 * D + 2, "fp8_int4": D + 1 + D // 2 + 8}[case["fmt"]]
    if case["kind"] == "rotary":
        angles = 4 * case["rot"] * B * L
        return {"bytes": 2 * B * Hkv * G * L * D * item + angles, "flops": 3 * B * Hkv * G * L * case["rot"]}
    if case["kind"] == "attend":
        # (the lengths of a ragged batch are the seed's: their mean)
        tokens = B * L if not case["ragged"] else L + int((B - 1) * L / math.log(L + 1))
        return {"bytes": tokens * Hkv * row + 4 * (tokens // page + 2 * B) + 2 * B * Hkv * G * D * item,
                "flops": 4 * tokens * Hkv * G * D}
    if case["kind"] == "read":
        return {"bytes": B * Hkv * L * (row + 2 * D * item), "flops": 2 * B * Hkv * L * D}
    nbytes = B * L * ((2 * Hkv + (2 * Hkv * G if case["rot"] else 0)) * D * item + Hkv * row + 4 * case["rot"])
    flops = 3 * B * L * (Hkv + Hkv * G) * case["rot"]
    if case["kind"] == "store":
        nbytes += B * Hkv * (case["start"] + L) * (row + 2 * D * item)
        flops += B * Hkv * L * D * 6 + 2 * B * Hkv * (case["start"] + L) * D
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_turn(case, x, first):
    """Each pair as a complex number times factor e^(i angle), whose parts the
    definition rounds to 32 bits."""
    rot = case["rot"]
    if not rot:
        return x.double()
    f = torch.ones(rot // 2, dtype=torch.float64)
    s = _SCALING[case["scaling"]] or {"kind": "none", "factor": 1.0}
    factor = 0.1 * math.log(s["factor"]) + 1.0 if s["kind"] == "yarn" else 1.0
    base = _BASE * s["factor"] ** (rot / (rot - 2)) if s["kind"] == "ntk" else _BASE
    for i in range(rot // 2):
        f[i] = base ** (-2.0 * i / rot) / (s["factor"] if s["kind"] == "linear" else 1.0)
        if s["kind"] == "yarn":
            ends = [rot * math.log(s["original_positions"] / (b * 2 * math.pi)) / (2 * math.log(base))
                    for b in (s["beta_fast"], s["beta_slow"])]
            lo, hi = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), rot // 2 - 1)
            t = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f[i] = f[i] / s["factor"] * t + f[i] * (1 - t)
        if s["kind"] == "bands":
            turns = s["original_positions"] * f[i].item() / (2 * math.pi)
            t = (turns - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])
            t = min(max(t, 0.0), 1.0)
            f[i] = f[i] * t + f[i] / s["factor"] * (1 - t)
    pos = first.double()[:, None] + torch.arange(x.shape[2], device="cuda", dtype=torch.float64)
    z = torch.polar(torch.full((), factor, dtype=torch.float64, device="cuda"), pos[..., None] * f.cuda())
    z = torch.complex(z.real.float().double(), z.imag.float().double())[:, None]
    head = x[..., :rot].double()
    pairs = head.unflatten(-1, (-1, 2)) if case["interleaved"] else \
        torch.stack([head[..., :rot // 2], head[..., rot // 2:]], -1)
    w = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
    w = w.flatten(-2) if case["interleaved"] else torch.cat([w[..., 0], w[..., 1]], -1)
    return torch.cat([w, x[..., rot:].double()], -1)


def _exact_e4m3(x):
    """Rows (64 bits) -> the values that their codes stand for: 448 2^e, e an
    integer, is the least bound on the row; steps of 2^-3 of the binade, of
    2^-9 below 2^-6."""
    x = x.float().double()
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 448.0))
    e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, torch.where(top > 448.0 * torch.exp2(e), e + 1, e))
    one = torch.exp2(torch.where(top > 0, e.clamp_min(-126), torch.zeros_like(e)))
    u = x / one
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(u / step) * step * one


def _exact_int4(x):
    x = x.double()
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    s = ((hi - lo) / 15.0 + torch.zeros_like(lo)).float().double()
    return lo + s * torch.clamp(torch.round((x - lo) / s), 0, 15)


def _exact_rows(case, x, b, n):
    """The first n rows of sequence b's pages in 64 bits (Hkv, n, D)."""
    page = case["page"]
    ids = x["table"][b, :-(-n // page)].long()
    out = []
    for name, scale in (("k", "k_exp"), ("v", "v_scale")):
        t = x["pages"][name].index_select(0, ids).movedim(1, 0).flatten(1, 2)[:, :n]
        if case["fmt"] in ("fp16", "bf16"):
            out.append(t.double())
            continue
        z = x["pages"][scale].index_select(0, ids).movedim(1, 0).flatten(1, 2)[:, :n]
        if name == "v" and case["fmt"] == "fp8_int4":
            c = torch.stack([t % 16, t // 16], -1).flatten(-2).double()
            out.append(c * z[..., 0:1].double() + z[..., 1:2].double())
        else:
            m, ex = (t & 7).double(), ((t >> 3) & 15).double()
            value = torch.where(ex > 0, (m + 8) * torch.exp2(ex - 10), m * 2.0 ** -9)
            out.append(torch.where(t > 127, -value, value) * torch.exp2(z.double() - 127).unsqueeze(-1))
    return out


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "rotary":
        return _exact_turn(case, x["x"], x["start"])
    B, Hkv, D, page = case["B"], case["Hkv"], case["D"], case["page"]
    lens = x["lens"].tolist()
    if case["kind"] == "attend":
        out = torch.zeros((B, Hkv, case["G"], D), dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            if n:
                k, v = _exact_rows(case, x, b, n)
                for h in range(Hkv):
                    s = x["q"][b].double().view(Hkv, case["G"], D)[h] @ k[h].T.contiguous() / math.sqrt(D)
                    out[b, h] = torch.softmax(s, -1) @ v[h]
        return out.view(B, -1, 1, D)
    shape = (B, Hkv, x["max_len"], D)
    k, v = (torch.zeros(shape, dtype=torch.float64, device="cuda") for _ in range(2))
    if case["kind"] in ("read", "store"):
        for b, n in enumerate(lens):
            k[b, :, :n], v[b, :, :n] = _exact_rows(case, x, b, n)
        if case["kind"] == "read":
            return [k, v]
    q = _exact_turn(case, x["q"], x["start"])
    nk, nv = _exact_turn(case, x["k"], x["start"]), x["v"].double()
    if case["kind"] == "store":
        n = case["start"]
        k[:, :, n:], v[:, :, n:] = _exact_e4m3(nk), (_exact_e4m3 if case["fmt"] == "fp8" else _exact_int4)(nv)
        return [q, k, v]
    pk, pv = x["pages"]["k"].double(), x["pages"]["v"].double()
    for b, first in enumerate(x["start"].tolist()):
        pos = torch.arange(first, first + case["L"], device="cuda")
        at = x["table"][b].long()[pos // page]
        pk[at, :, pos % page], pv[at, :, pos % page] = nk[b].transpose(0, 1), nv[b].transpose(0, 1)
    return [q, pk, pv]
