"""Performance cases of the paged cache's operators for prompts that begin
alike, drafted tokens and long contexts.

Kinds of call:

  rows    ``PagedLayer.attend_tokens`` of several new tokens a sequence, each over
          the tokens up to itself: drafted tokens to be verified, a prompt's
          chunk.
  shared  the same where all sequences begin with the same pages
          (``shared`` tokens), which are attended to once for all of them.
  bound   ``PagedLayer.bound``: each page's least and largest key per dim.
  sparse  ``PagedLayer.attend_sparse``: one new token a sequence over the
          pages whose bounds promise the largest scores.
  verify  ``verify_drafts``: how many drafted tokens stand against the
          target's probabilities, and the token that follows them.

Pages are (n_pages, Hkv, page, D): 16-bit elements (``fp16``, ``bf16``);
E4M3 codes with one power of two per token and head (``fp8``); or E4M3 keys
and INT4 values (``fp8_int4``, even dims in the low nibble) with a 32-bit
scale and zero per token and head.  Inputs are made on the GPU from the seed;
pages lie in random order.
"""

import math

import torch

own = False

_DEFAULTS = {"B": 1, "Hkv": 8, "G": 4, "D": 128, "L": 1, "ctx": 0, "shared": 0, "select": 0, "page": 64,
             "dtype": "bfloat16", "fmt": "bf16", "ragged": False, "padded": False, "V": 0, "draft": True}


def _case(name, kind, **options):
    c = {"kind": kind, **_DEFAULTS, **options}
    return {"name": name, **c} if name else c


def listed():
    return [
        # four drafted tokens of a short chat on a half-billion-parameter
        # model: latency
        _case("rows_draft_small_512", "rows", Hkv=2, G=7, D=64, L=4, ctx=512, page=16, dtype="float16", fmt="fp16"),
        # up to five drafted tokens of 32 running sequences at their own
        # lengths, some with fewer drafts than others
        _case("rows_draft_ragged_b32", "rows", B=32, L=5, ctx=8192, ragged=True, padded=True),
        # a prompt's chunk of 2K tokens after 14K stored ones: the largest
        _case("rows_chunk_2k_of_16k", "rows", L=2048, ctx=16384),
        # an odd chunk of three prompts, 8-bit pages
        _case("rows_chunk_odd_fp8", "rows", B=3, Hkv=4, G=5, L=333, ctx=5003, page=32, dtype="float16", fmt="fp8"),
        # 64 chats behind one instruction of 16K tokens, to 1K tokens each
        _case("shared_16k_b64", "shared", B=64, ctx=1024, shared=16384, ragged=True),
        # questions about one long document, 8-bit keys and 4-bit values
        _case("shared_64k_b12_fp8_int4", "shared", B=12, G=8, ctx=300, shared=65536, fmt="fp8_int4"),
        # a short instruction, odd sizes, three drafted tokens each
        _case("shared_odd_drafts", "shared", B=7, Hkv=2, G=7, D=64, L=3, ctx=401, shared=1008, page=16, ragged=True,
              dtype="float16", fmt="fp16"),
        # the bounds of a 64K prompt's pages
        _case("bound_prompt_64k", "bound", ctx=65536),
        # one page in 32 of a 128K context
        _case("sparse_128k", "sparse", ctx=131072, select=64),
        # 16 sequences to 32K tokens, 8-bit pages of 32 tokens
        _case("sparse_ragged_b16_fp8", "sparse", B=16, ctx=32768, page=32, select=48, ragged=True, dtype="float16",
              fmt="fp8"),
        # five drafted tokens of one sequence, a small vocabulary: latency
        _case("verify_one_32k", "verify", L=5, V=32000, dtype="float32"),
        # up to six drafted tokens of 64 sequences, a large vocabulary
        _case("verify_b64_128k", "verify", B=64, L=6, V=128000, padded=True, dtype="float32"),
    ]


def draw(rng):
    kind = rng.choice(["rows", "rows", "shared", "shared", "sparse", "sparse", "verify", "bound"])

    def spread(lo, hi):
        return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    if kind == "verify":
        V, L = spread(1000, 150000), rng.randint(1, 8)
        return _case(None, kind, B=spread(1, max(1, 64 * 128000 * 6 // (V * L))) if V * L > 12000 else spread(1, 256), L=L,
                     V=V, padded=rng.random() < 0.5, draft=rng.random() < 0.8,
                     dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]))
    o = {"Hkv": rng.choice([1, 2, 4, 8]), "G": rng.choice([1, 2, 4, 5, 7, 8]), "D": rng.choice([64, 128, 128]),
         "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["float16", "bfloat16"])}
    plain = {"float16": "fp16", "bfloat16": "bf16"}[o["dtype"]]
    o["fmt"] = rng.choice([plain, plain, "fp8", "fp8_int4"])
    o["ragged"] = rng.random() < 0.5
    heads = o["Hkv"] * o["G"]
    if kind == "bound":
        o["B"] = spread(1, 8)
        return _case(None, kind, ctx=spread(16, 65536 * 8 // (o["B"] * o["Hkv"]) if o["B"] * o["Hkv"] > 8 else 65536), **o)
    if kind == "sparse":
        o["B"] = spread(1, 32)
        ctx = spread(64, min(131072, 16 * 32768 * 8 // (o["B"] * o["Hkv"])))
        return _case(None, kind, ctx=ctx, select=rng.choice([4, 16, 31, 64, 96]), **o)
    o["L"] = 1 if kind == "shared" and rng.random() < 0.5 else rng.choice([2, 3, 4, 5, 8]) if rng.random() < 0.6 else \
        spread(2, 2048)
    o["B"] = spread(1 if kind == "rows" else 2, 4 if o["L"] > 16 else 64)
    o["padded"] = rng.random() < 0.4
    # new tokens times heads times tokens attended to: no more than the
    # largest listed case has, and a cache of 512 MB at most in 16 bits
    most = min(2048 * 32 * 16384 // (o["B"] * o["L"] * heads), 65536)
    if kind == "shared":
        o["shared"] = max(o["page"], spread(o["page"], max(o["page"], most)) // o["page"] * o["page"])
        most = max(1, min(most, 2048))
    ctx = spread(1, max(1, min(most, 2 ** 20 // (o["B"] * o["Hkv"]))))
    return _case(None, kind, ctx=max(ctx, o["L"]), **o)


# ---------------------------------------------------------------------------
# the formats in plain form
# ---------------------------------------------------------------------------

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
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = (hi - lo) / 15.0
    c = torch.where(s > 0, (x - lo) / s, 0.0).round().clamp(0, 15).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.cat([s, lo], -1)


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


def _keys(fmt, p):
    """Key rows of pages as float32."""
    return p["k"].float() if fmt in ("fp16", "bf16") else _decode8(p["k"], p["k_exp"])


def _values(fmt, p):
    if fmt in ("fp16", "bf16"):
        return p["v"].float()
    return (_decode8 if fmt == "fp8" else _decode4)(p["v"], p["v_scale"])


def _outward(x, up):
    """float32 -> the nearest bfloat16 that is not below (up) or above x."""
    bits = x.view(torch.int32)
    cut = bits & -65536  # towards zero
    grow = (cut != bits) & ((bits >= 0) if up else (bits < 0))
    return torch.where(grow, cut + 65536, cut).view(torch.float32).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _dtype(case):
    return getattr(torch, case["dtype"])


def _verify_inputs(case, seed):
    B, K, V = case["B"], case["L"], case["V"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    target = torch.randn((B, K + 1, V), generator=g, device="cuda") * 3.0
    x = {}
    if case["draft"]:
        logits = target[:, :K] + torch.randn((B, K, V), generator=g, device="cuda")
        x["draft"] = torch.softmax(logits, -1).to(_dtype(case))
        noise = torch.rand((B, K, V), generator=g, device="cuda").clamp_min(1e-30)
        x["tokens"] = (logits - torch.log(-torch.log(noise))).argmax(-1)  # drawn by the draft's probabilities
    else:
        x["tokens"] = (target[:, :K] + torch.randn((B, K, V), generator=g, device="cuda")).argmax(-1)
    x["target"] = torch.softmax(target, -1).to(_dtype(case))
    x["uniforms"] = torch.rand((B, K + 1), generator=g, device="cuda")
    x["n_draft"] = torch.randint(0, K + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if case["padded"] else None
    return x


def _inputs(case, seed):
    if case["kind"] == "verify":
        return _verify_inputs(case, seed)
    B, Hkv, G, D, L, page, shared = (case[n] for n in ("B", "Hkv", "G", "D", "L", "page", "shared"))
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.Generator().manual_seed(7919 * seed + 13)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    x = {}
    new = torch.randint(0, L + 1, (B,), generator=h).tolist() if case["padded"] else [L] * B
    u = torch.rand(B, generator=h).tolist()
    tokens = [max(n, 1 + int(case["ctx"] * t) if case["ragged"] else case["ctx"]) for n, t in zip(new, u)]
    tokens[-1] = max(tokens[-1], case["ctx"])
    lens = [shared + n for n in tokens]
    x["n_new"] = torch.tensor(new, dtype=torch.int32, device="cuda") if case["padded"] else None
    x["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    x["max_len"] = max(lens)
    # the shared pages, then each sequence's own
    n_shared = shared // page
    counts = [-(-n // page) for n in tokens]
    n_pages = n_shared + sum(counts) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    ends = (torch.tensor(counts).cumsum(0) + n_shared).tolist()
    x["table"] = torch.zeros((B, n_shared + max(counts)), dtype=torch.int32, device="cuda")
    x["table"][:, :n_shared] = order[:n_shared]
    for b in range(B):
        x["table"][b, n_shared:n_shared + counts[b]] = order[ends[b] - counts[b]:ends[b]]
    q = normal(B, L, Hkv * G, D)
    x["q"] = q.to(_dtype(case)).transpose(1, 2)  # (tokens before heads, as a projection leaves them)
    channels = torch.randperm(D, generator=g, device="cuda")[:4]
    parts = []
    step = max(1, 2 ** 26 // (Hkv * page * D))  # pages that are made at a time
    for p in range(0, n_pages, step):
        n = min(step, n_pages - p)
        k, v = normal(n, Hkv, page, D), normal(n, Hkv, page, D)
        if case["kind"] in ("bound", "sparse"):
            k = 0.7 * k + 0.7 * normal(n, Hkv, 1, D)  # neighbours are alike
        k[..., channels] *= 4.0
        parts.append(_encode(case["fmt"], k.to(_dtype(case)).float(), v.to(_dtype(case)).float()))
    x["pages"] = {n: torch.cat([part[n] for part in parts]) for n in parts[0]}
    if case["kind"] in ("bound", "sparse"):
        x["bounds"] = torch.zeros((n_pages, Hkv, 2, D), dtype=torch.bfloat16, device="cuda")
        if case["kind"] == "sparse":
            _plain_bound(case, x)
        else:
            x["start"] = torch.zeros(B, dtype=torch.int32, device="cuda")
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    x["case"] = case
    if own and case["kind"] != "verify":
        from foveated_kv_amd.paged import PagedLayer

        x["layer"] = PagedLayer.wrap(case["fmt"], **x["pages"], bounds=x.get("bounds"))
    return x


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _gather(case, x, table, parts="kv"):
    """Rows of the table's pages, float32 (rows of the table, Hkv, P * page, D)."""
    names = [n for n in x["pages"] if n[0] in parts]
    flat = {n: x["pages"][n][table.long()].transpose(1, 2).flatten(2, 3) for n in names}
    return [f(case["fmt"], flat) for f, c in ((_keys, "k"), (_values, "v")) if c in parts]


def _limits(case, x):
    """How many tokens query l of sequence b attends to (B, L), 0 for padding."""
    L = case["L"]
    new = x["n_new"] if x["n_new"] is not None else torch.full_like(x["lens"], L)
    l = torch.arange(L, device="cuda")
    return torch.where(l < new[:, None], x["lens"][:, None] - new[:, None] + l + 1, 0)


def _plain_rows(case, x):
    """Scores of the shared tokens from one product, of each sequence's own
    from another; a few sequences and heads at a time."""
    B, Hkv, G, D, L, page = (case[n] for n in ("B", "Hkv", "G", "D", "L", "page"))
    n_shared = case["shared"] // page
    P = -(-x["max_len"] // page)
    q = x["q"].float().reshape(B, Hkv, G * L, D)
    limits = _limits(case, x)[:, None, None].expand(B, 1, G, L).reshape(B, 1, G * L, 1)
    at = torch.arange(P * page, device="cuda")
    out = torch.empty((B, Hkv, G * L, D), dtype=torch.float32, device="cuda")
    if n_shared:
        pk, pv = _gather(case, x, x["table"][:1, :n_shared])
    step = max(1, 2 ** 28 // (Hkv * max(G * L, D) * P * page))  # sequences at a time
    heads = Hkv if step > 1 else max(1, 2 ** 28 // (G * L * P * page))
    for b in range(0, B, step):
        k, v = _gather(case, x, x["table"][b:b + step, n_shared:P])
        n = k.shape[0]
        for h in range(0, Hkv, heads):
            sl = slice(h, h + heads)
            s = torch.matmul(q[b:b + n, sl], k[:, sl].transpose(-1, -2).contiguous())
            m = s.shape[1]
            if n_shared:
                ps = torch.matmul(q[b:b + n, sl].transpose(0, 1).reshape(m, -1, D), pk[0, sl].transpose(-1, -2).contiguous())
                s = torch.cat([ps.view(m, n, G * L, -1).transpose(0, 1), s], -1)
            held = at < limits[b:b + n]
            s = torch.where(held, s * D ** -0.5, -math.inf)
            w = torch.where(held, torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30)), 0.0)
            o = torch.matmul(w[..., n_shared * page:], v[:, sl])
            if n_shared:
                pw = w[..., :n_shared * page].transpose(0, 1).reshape(m, n * G * L, -1)
                o += torch.matmul(pw, pv[0, sl]).view(m, n, G * L, D).transpose(0, 1)
            out[b:b + n, sl] = o / w.sum(-1, keepdim=True).clamp_min(1e-30)
    return out.view(B, Hkv * G, L, D).to(_dtype(case))


def _plain_bound(case, x):
    """Bounds of the pages that hold tokens, in x["bounds"]."""
    page = case["page"]
    i = torch.arange(x["table"].shape[1], device="cuda") * page
    for b in range(case["B"]):
        ids = x["table"][b].long()[i < x["lens"][b]]
        k = _keys(case["fmt"], {n: t[ids] for n, t in x["pages"].items() if n[0] == "k"})
        held = (torch.arange(page, device="cuda") + i[:ids.shape[0], None] < x["lens"][b])[:, None, :, None]
        lo = torch.where(held, k, math.inf).amin(2)
        hi = torch.where(held, k, -math.inf).amax(2)
        x["bounds"][ids] = torch.stack([_outward(lo, False), _outward(hi, True)], 2)
    return x["bounds"]


def _plain_sparse(case, x):
    """Bounds of the scores in 64 bits, which decide; the rest in 32."""
    B, Hkv, G, D, page, n = (case[k] for k in ("B", "Hkv", "G", "D", "page", "select"))
    P = -(-x["max_len"] // page)
    count = (x["lens"] + page - 1) // page  # pages of each sequence
    q = x["q"].view(B, Hkv, G, D).double()
    table = x["table"][:, :P].long()
    score = torch.full((B, Hkv, P), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(B):
        lo, hi = x["bounds"][table[b]].double().permute(2, 1, 0, 3)  # (Hkv, P, D)
        s = torch.matmul(q[b].clamp_min(0.0), hi.transpose(-1, -2).contiguous()) + \
            torch.matmul(q[b].clamp_max(0.0), lo.transpose(-1, -2).contiguous())
        score[b] = s.amax(1)
    i = torch.arange(P, device="cuda")
    score = torch.where(i < count[:, None, None] - 1, score, -math.inf)
    score = torch.where(i == count[:, None, None] - 1, math.inf, score)  # (the newest page is always one)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :n]
    taken = torch.arange(order.shape[-1], device="cuda") < count[:, None, None]
    first = torch.where(taken, order, P).sort(-1).values
    pages = torch.full((B, Hkv, n), -1, dtype=torch.int32, device="cuda")
    pages[..., :first.shape[-1]] = torch.where(first < P, first, -1).int()
    out = torch.empty((B, Hkv, G, D), dtype=torch.float32, device="cuda")
    for b in range(B):
        ids = torch.where(first[b] < P, table[b][first[b].clamp_max(P - 1)], table[b, 0])
        rows = {name: t[ids, torch.arange(Hkv, device="cuda")[:, None]].flatten(1, 2) for name, t in x["pages"].items()}
        at = (first[b, :, :, None] * page + torch.arange(page, device="cuda")).flatten(1, 2)
        held = (at < x["lens"][b])[:, None]
        s = torch.matmul(q[b].float(), _keys(case["fmt"], rows).transpose(-1, -2).contiguous()) * D ** -0.5
        s = torch.where(held, s, -math.inf)
        w = torch.where(held, torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30)), 0.0)
        out[b] = torch.matmul(w, torch.where(held.transpose(-1, -2), _values(case["fmt"], rows), 0.0)) / \
            w.sum(-1, keepdim=True).clamp_min(1e-30)
    return out.view(B, Hkv * G, 1, D).to(_dtype(case)), pages


def _plain_verify(case, x):
    """Products and sums in 64 bits: what decides lies next to a border."""
    B, K, V = case["B"], case["L"], case["V"]
    n = x["n_draft"].long() if x["n_draft"] is not None else torch.full((B,), K, device="cuda")
    rows = torch.arange(B, device="cuda")
    p = x["target"][:, :K].gather(-1, x["tokens"][..., None])[..., 0].double()
    d = x["draft"].gather(-1, x["tokens"][..., None])[..., 0].double() if case["draft"] else torch.ones_like(p)
    stands = (x["uniforms"][:, :K].double() * d < p) & (torch.arange(K, device="cuda") < n[:, None])
    accepted = stands.long().cumprod(-1).sum(-1)
    w = x["target"][rows, accepted].double()
    at = accepted.clamp_max(K - 1)
    if case["draft"]:
        q = x["draft"][rows, at].double()
    else:
        q = torch.zeros((B, V), dtype=torch.float64, device="cuda").scatter(1, x["tokens"].gather(1, at[:, None]), 1.0)
    w = torch.where((accepted < n)[:, None], (w - q).clamp_min(0.0), w)
    c = w.cumsum(-1)
    follows = torch.searchsorted(c, x["uniforms"][:, K:].double() * c[:, -1:], right=True)[:, 0]
    i = torch.arange(K + 1, device="cuda")
    drafts = torch.cat([x["tokens"], follows[:, None]], 1)
    tokens = torch.where(i < accepted[:, None], drafts, torch.where(i == accepted[:, None], follows[:, None], -1))
    return tokens, accepted.int()


def run(state):
    case, x = state["case"], state
    kind = case["kind"]
    if kind == "verify":
        if own:
            from foveated_kv_amd import verify_drafts

            return list(verify_drafts(x["target"], x.get("draft"), x["tokens"], x["uniforms"], n_draft=x["n_draft"]))
        return list(_plain_verify(case, x))
    if kind == "bound":
        if not own:
            return _plain_bound(case, x)
        x["layer"].bound(x["table"], x["start"], x["max_len"], n_new=x["lens"])
        return x["bounds"]
    if kind == "sparse":
        if not own:
            return list(_plain_sparse(case, x))
        return list(x["layer"].attend_sparse(x["q"], x["table"], x["lens"], case["select"], max_len=x["max_len"],
                                             return_pages=True))
    if not own:
        return _plain_rows(case, x)
    return x["layer"].attend_tokens(x["q"], x["table"], x["lens"], x["max_len"], n_new=x["n_new"], shared=case["shared"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    B, Hkv, G, D, L, page, ctx = (case[n] for n in ("B", "Hkv", "G", "D", "L", "page", "ctx"))
    item = torch.finfo(_dtype(case)).bits // 8
    if case["kind"] == "verify":
        # the row that follows the last accepted token, of both; the tests
        return {"bytes": B * case["V"] * item * (2 if case["draft"] else 1) + 32 * B * L, "flops": 3 * B * case["V"]}
    own_key = {"fp16": 2 * D, "bf16": 2 * D}.get(case["fmt"], D + 1)
    row = own_key + {"fp16": 2 * D, "bf16": 2 * D, "fp8": D + 1, "fp8_int4": D // 2 + 8}[case["fmt"]]
    # (a ragged batch's lengths are the seed's: their mean)
    tokens = B * ctx if not case["ragged"] else max(1, (B - 1) * ctx // 2) + ctx
    new = L if not case["padded"] else L / 2
    heads = Hkv * G
    if case["kind"] == "bound":
        return {"bytes": Hkv * (tokens * own_key + tokens // page * 4 * D), "flops": 2 * tokens * Hkv * D}
    if case["kind"] == "sparse":
        taken = min(tokens, B * case["select"] * page)
        return {"bytes": Hkv * (tokens // page * 4 * D + taken * row) + 4 * B * heads * D,
                "flops": 4 * heads * D * (tokens // page + taken)}
    pairs = new * (tokens + B * case["shared"] - B * (L - 1) / 2)  # query times token
    return {"bytes": int(Hkv * (tokens + case["shared"]) * row + 4 * B * new * heads * D),
            "flops": int(4 * D * heads * max(pairs, new * B))}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_rows(case, x, b, h, n):
    """The first n keys and values of sequence b and KV head h in 64 bits."""
    page = case["page"]
    ids = x["table"][b, :-(-n // page)].long()
    out = []
    for name, scale in (("k", "k_exp"), ("v", "v_scale")):
        t = x["pages"][name][ids, h].flatten(0, 1)[:n]
        if case["fmt"] in ("fp16", "bf16"):
            out.append(t.double())
            continue
        z = x["pages"][scale][ids, h].flatten(0, 1)[:n]
        if name == "v" and case["fmt"] == "fp8_int4":
            c = torch.stack([t % 16, t // 16], -1).flatten(-2).double()
            out.append(c * z[..., 0:1].double() + z[..., 1:2].double())
        else:
            m, ex = (t & 7).double(), ((t >> 3) & 15).double()
            value = torch.where(ex > 0, (m + 8) * torch.exp2(ex - 10), m * 2.0 ** -9)
            out.append(torch.where(t > 127, -value, value) * torch.exp2(z.double() - 127).unsqueeze(-1))
    return out


def _exact_attention(case, x):
    B, Hkv, G, D, L = (case[n] for n in ("B", "Hkv", "G", "D", "L"))
    out = torch.zeros((B, Hkv * G, L, D), dtype=torch.float64, device="cuda")
    new = [L] * B if x["n_new"] is None else x["n_new"].tolist()
    for b, n in enumerate(x["lens"].tolist()):
        m = new[b]
        if m == 0:
            continue
        future = torch.arange(n, device="cuda") > torch.arange(n - m, n, device="cuda")[:, None]
        for h in range(Hkv):
            k, v = _exact_rows(case, x, b, h, n)
            for i in range(h * G, (h + 1) * G):
                s = (x["q"][b, i, :m].double() @ k.T.contiguous() / math.sqrt(D)).masked_fill(future, -math.inf)
                out[b, i, :m] = torch.softmax(s, -1) @ v
    return out


def _exact_bounds(case, x):
    """The least and largest key of each page, a step of bfloat16 outwards."""
    bounds = x["bounds"].double()
    page = case["page"]
    for b, n in enumerate(x["lens"].tolist()):
        for h in range(case["Hkv"]):
            k = _exact_rows(case, x, b, h, n)[0]
            pad = -n % page
            blocks = torch.cat([k, k[-1:].expand(pad, -1)]).view(-1, page, k.shape[-1])
            ends = torch.stack([blocks.amin(1), blocks.amax(1)], 1)
            step = torch.exp2(torch.floor(torch.log2(ends.abs().clamp_min(2.0 ** -126))) - 7)
            ids = x["table"][b, :-(-n // page)].long()
            bounds[ids, h] = torch.stack([torch.floor(ends[:, 0] / step[:, 0]) * step[:, 0],
                                          torch.ceil(ends[:, 1] / step[:, 1]) * step[:, 1]], 1)
    return bounds


def _exact_sparse(case, x):
    B, Hkv, G, D, page, n = (case[k] for k in ("B", "Hkv", "G", "D", "page", "select"))
    out = torch.zeros((B, Hkv * G, 1, D), dtype=torch.float64, device="cuda")
    pages = torch.full((B, Hkv, n), -1, dtype=torch.int64, device="cuda")
    for b, length in enumerate(x["lens"].tolist()):
        count = -(-length // page)
        for h in range(Hkv):
            q = x["q"][b, h * G:(h + 1) * G, 0].double()
            box = x["bounds"][x["table"][b, :count].long(), h].double()  # (count, 2, D)
            bound = torch.maximum(q[:, None] * box[:, 0], q[:, None] * box[:, 1]).sum(-1).amax(0)
            best = sorted(range(count - 1), key=lambda i, s=bound.tolist(): (-s[i], i))[:n - 1]
            picked = torch.tensor(sorted(best + [count - 1]), device="cuda")
            pages[b, h, :len(picked)] = picked
            k, v = _exact_rows(case, x, b, h, length)
            at = (picked[:, None] * page + torch.arange(page, device="cuda")).flatten()
            at = at[at < length]
            out[b, h * G:(h + 1) * G, 0] = torch.softmax(q @ k[at].T.contiguous() / math.sqrt(D), -1) @ v[at]
    return [out, pages]


def _exact_verify(case, x):
    B, K = case["B"], case["L"]
    tokens = torch.full((B, K + 1), -1, dtype=torch.int64, device="cuda")
    accepted = torch.zeros(B, dtype=torch.int64, device="cuda")
    drafted, u = x["tokens"].tolist(), x["uniforms"].double().tolist()
    n_draft = [K] * B if x["n_draft"] is None else x["n_draft"].tolist()
    for b in range(B):
        p = x["target"][b].double()
        a = 0
        while a < n_draft[b]:
            t = drafted[b][a]
            q = x["draft"][b, a, t].double().item() if case["draft"] else 1.0
            if not u[b][a] * q < p[a, t].item():
                break
            tokens[b, a] = t
            a += 1
        w = p[a].clone()
        if a < n_draft[b]:
            if case["draft"]:
                w = torch.clamp(w - x["draft"][b, a].double(), min=0.0)
            else:
                w[drafted[b][a]] = 0.0
        c = torch.cumsum(w, 0)
        tokens[b, a] = int((c <= u[b][K] * c[-1]).sum())
        accepted[b] = a
    return [tokens, accepted]


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(case, x)
    if case["kind"] == "bound":
        return _exact_bounds(case, x)
    if case["kind"] == "sparse":
        return _exact_sparse(case, x)
    return _exact_attention(case, x)
