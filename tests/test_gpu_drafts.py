"""Verification of drafted tokens against a restatement in 64 bits: accepted
counts and tokens exactly, the distribution of what comes out, rows without
weight, numbers that are not finite, strides, captured graphs."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def verify():
    import foveated_kv_amd

    assert foveated_kv_amd.is_available(), "libfkv.so loaded but no gfx950 device"
    return foveated_kv_amd.verify_drafts


def _rand(seed, *shape):
    return torch.rand(shape, generator=torch.Generator().manual_seed(seed))


def _want(target, draft, tokens, uniforms, n_draft=None):
    """The definition, a token at a time, sums exact (math.fsum) over each
    running prefix's floats."""
    B, K1, V = target.shape
    K = K1 - 1
    p, q = target.double().numpy(), None if draft is None else draft.double().numpy()
    out, accepted = np.full((B, K1), -1, dtype=np.int64), np.zeros(B, dtype=np.int32)
    for b in range(B):
        n = K if n_draft is None else min(max(int(n_draft[b]), 0), K)
        a = 0
        while a < n:
            t = int(tokens[b, a])
            inside = 0 <= t < V
            if not (inside and float(uniforms[b, a]) * (1.0 if q is None else q[b, a, t]) < p[b, a, t]):
                break
            out[b, a] = t
            a += 1
        accepted[b] = a
        own = np.where(p[b, a] > 0, p[b, a], 0.0)
        w = own
        if a < n:
            d = p[b, a] - (q[b, a] if q is not None else 0.0)
            if q is None and 0 <= int(tokens[b, a]) < V:
                d[int(tokens[b, a])] = 0.0
            w = np.where(d > 0, d, 0.0)
            if not w.sum() > 0:
                w = own
        c = np.cumsum(w)
        if 0 < c[-1] < math.inf:
            past = np.nonzero(c > float(uniforms[b, K]) * c[-1])[0]
            out[b, a] = past[0]
    return out, accepted


def _check(verify, target, draft, tokens, uniforms, n_draft=None):
    got, acc = verify(target.cuda(), None if draft is None else draft.cuda(), tokens.cuda(), uniforms.cuda(),
                      None if n_draft is None else n_draft.cuda())
    want, wacc = _want(target, draft, tokens, uniforms, n_draft)
    assert got.dtype == tokens.dtype and acc.dtype == torch.int32 and got.shape == want.shape
    assert np.array_equal(acc.cpu().numpy(), wacc)
    assert np.array_equal(got.cpu().numpy(), want)
    return wacc


def _probs(seed, dtype, *shape):
    return torch.softmax(3 * torch.randn(shape, generator=torch.Generator().manual_seed(seed)), -1).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (3, 5, 97), (40, 4, 1000), (5, 63, 333), (2, 3, 4096), (3, 2, 4099), (4, 6, 50021),
                                   (2, 1, 131072), (6, 0, 700)])
@pytest.mark.parametrize("drawn", [True, False])
def test_verify(verify, dtype, B, K, V, drawn):
    print("verify", dtype, B, K, V, drawn, flush=True)
    target = _probs(V + B, dtype, B, K + 1, V)
    noisy = target[:, :K].float() * torch.exp(0.3 * torch.randn((B, K, V), generator=torch.Generator().manual_seed(B)))
    draft = (noisy / noisy.sum(-1, keepdim=True)).to(dtype)
    tokens = (noisy / -torch.log(_rand(1, B, K, V).clamp(1e-7, 1 - 1e-7))).argmax(-1) if K else torch.zeros(B, 0, dtype=torch.int64)
    if drawn is False:
        draft = None
    for i, (kind, n) in enumerate([(torch.int64, None), (torch.int32, None),
                                   (torch.int64, torch.tensor([(2 * b) % (K + 2) - 1 for b in range(B)], dtype=torch.int32))]):
        _check(verify, target, draft, tokens.to(kind), _rand(2 + i, B, K + 1), n)


def test_tokens_are_distributed_as_the_target(verify):
    """A grid of uniform numbers and all first tokens in the draft's shares: the
    shares of the first token that comes out are the target's.  On an N-point grid
    a share is off by a point at each end of an interval, of which there are two
    for each pair of tokens."""
    p = torch.tensor([0.05, 0.3, 0.0, 0.4, 0.25])
    q = torch.tensor([0.3, 0.25, 0.25, 0.2, 0.0])
    N, V = 100, 5
    grid = (torch.arange(N) + 0.5) / N
    share = torch.zeros(V, dtype=torch.float64)
    for x in range(V):
        u = torch.cartesian_prod(grid, grid)
        B = u.shape[0]
        out, _ = verify(p.expand(B, 2, V).cuda(), q.expand(B, 1, V).cuda(), torch.full((B, 1), x).cuda(), u.cuda())
        share += q[x].double() * torch.bincount(out[:, 0].cpu(), minlength=V) / B
    assert float((share - p.double()).abs().max()) <= 2 * V / N
    assert share[2] == 0


def test_borders(verify):
    """A product equal to the probability refuses; a running sum equal to the
    goal is not past it; tokens of weight zero are never chosen."""
    V = 8
    p = torch.tensor([[[0.25, 0, 0.25, 0, 0, 0.5, 0, 0], [0.0, 0, 0.5, 0, 0.5, 0, 0, 0]]])
    q = torch.tensor([[[0.5, 0, 0.25, 0, 0, 0.25, 0, 0]]])
    for x, u0 in ((0, 0.5), (0, 0.49), (2, 0.9999), (5, 0.9999), (1, 0.0), (7, 0.0), (-1, 0.0), (V, 0.0), (2 ** 31 + 5, 0.0)):
        for u1 in (0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24):
            _check(verify, p, q, torch.tensor([[x]]), torch.tensor([[u0, u1]]))
            _check(verify, p, None, torch.tensor([[x]]), torch.tensor([[u0, u1]]))


def test_rows_that_leave_nothing(verify):
    """No difference is positive: the target's own; no probability at all, or an
    infinite one: no token.  NaN has no weight."""
    B, V = 6, 5000
    p = _probs(9, torch.float32, 1, 2, V).repeat(B, 1, 1)
    q = p[:, :1] * 1.5
    p[1, 0], p[2, 0, 4999], p[3, 0, 7] = 0.0, math.inf, math.nan
    p[4, 0] = 0.0
    p[4, 0, 4321] = 1e-40  # (a subnormal)
    p[5, 0] = math.nan
    q[3, 0, 100] = math.nan
    tokens = torch.full((B, 1), 3)
    u = torch.tensor([[1.0 - 2.0 ** -24, 0.3]] * B)
    got, acc = verify(p.cuda(), q.cuda(), tokens.cuda(), u.cuda())
    want, wacc = _want(torch.nan_to_num(p, nan=0.0, posinf=math.inf), torch.nan_to_num(q, nan=9.0), tokens, u)
    assert np.array_equal(got.cpu().numpy(), want) and np.array_equal(acc.cpu().numpy(), wacc)
    assert got[1, 0] == -1 and got[2, 0] == -1 and got[4, 0] == 4321 and got[5, 0] == -1


def test_strides_and_alignment(verify):
    B, K, V = 3, 2, 1001
    target, draft = _probs(20, torch.float32, B, K + 1, V), _probs(21, torch.float32, B, K, V)
    tokens, u = torch.randint(0, V, (B, K), generator=torch.Generator().manual_seed(3)), _rand(22, B, K + 1)
    want = _want(target, draft, tokens, u)
    wide = torch.zeros(B, K + 1, 2 * V, device="cuda")[..., ::2]
    wide.copy_(target)
    odd = torch.zeros(B * (K + 1) * 1024 + 1, device="cuda")[1:].view(B, K + 1, 1024)[..., :V]
    odd.copy_(target)
    turned = torch.zeros(K, B, V, device="cuda").transpose(0, 1)
    turned.copy_(draft)
    one = target[:, :1].expand(-1, K + 1, -1)
    for t in (wide, odd):
        got, acc = verify(t, turned, tokens.cuda().t().contiguous().t(), u.cuda())
        assert np.array_equal(got.cpu().numpy(), want[0]) and np.array_equal(acc.cpu().numpy(), want[1])
    _check(verify, one, draft, tokens, u)


def test_refusals(verify):
    t, d = torch.ones(2, 4, 9, device="cuda"), torch.ones(2, 3, 9, device="cuda")
    x, u = torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.zeros(2, 4, device="cuda")
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    from foveated_kv_amd._lib import FkvLibraryError

    bad = [
        (TypeError, lambda: verify(None, d, x, u)), (TypeError, lambda: verify(t.cpu(), d, x, u)),
        (TypeError, lambda: verify(t, d.cpu(), x, u)), (TypeError, lambda: verify(t.double(), d.double(), x, u)),
        (ValueError, lambda: verify(t, d.half(), x, u)), (ValueError, lambda: verify(t, d[:, :2], x, u)),
        (ValueError, lambda: verify(t[0], d, x, u)), (ValueError, lambda: verify(t[:, :, :0], d[:, :, :0], x, u)),
        (TypeError, lambda: verify(t, d, x.float(), u)), (TypeError, lambda: verify(t, d, x[:1], u)),
        (TypeError, lambda: verify(t, d, x, u.double())), (TypeError, lambda: verify(t, d, x, u[:, :3])),
        (TypeError, lambda: verify(t, d, x, u, n.long())), (TypeError, lambda: verify(t, d, x, u, n[:1])),
        (RuntimeError, lambda: verify(t.clone().requires_grad_(), d, x, u)),
        (FkvLibraryError, lambda: verify(t.repeat(1, 17, 1)[:, :65], None, x.repeat(1, 22)[:, :64], u.repeat(1, 17)[:, :65])),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            print("accepted", i)
    out, acc = verify(t[:0], d[:0], x[:0], u[:0])
    assert out.shape == (0, 4) and acc.shape == (0,)


def test_captured(verify):
    """Captured once on each of two streams and replayed with other inputs,
    eager work between the replays."""
    B, K, V = 5, 4, 9000
    runs, data = [], [[(_probs(100 * j + i, torch.float32, B, K + 1, V), _probs(100 * j + i + 50, torch.float32, B, K, V),
                        torch.randint(0, V, (B, K), generator=torch.Generator().manual_seed(i + j)), _rand(i + j, B, K + 1))
                       for i in range(8)] for j in range(2)]
    for j in range(2):
        bufs = [t.cuda() for t in data[j][0]]
        verify(*bufs)
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            out = verify(*bufs)
        runs.append((g, s, bufs, out))
    for i in range(8):
        for (g, s, bufs, _), d in zip(runs, data):
            with torch.cuda.stream(s):
                for dst, src in zip(bufs, d[i]):
                    dst.copy_(src)
                g.replay()
        torch.randn(1000, device="cuda").sum().item()
        torch.cuda.synchronize()
        for (g, s, bufs, out), d in zip(runs, data):
            want = _want(*d[i])
            assert np.array_equal(out[0].cpu().numpy(), want[0]) and np.array_equal(out[1].cpu().numpy(), want[1])


@pytest.mark.parametrize("V", [300, 12000, 40000, 300000])
def test_small_weights_before_large_ones(verify, V):
    """A number of zero takes the first token with a weight, however small beside
    those behind it: none is lost in a difference of sums."""
    target = torch.zeros((6, 1, V))
    first = [0, 1, V // 7, V // 2, V - 2, V - 1]
    for b, t in enumerate(first):
        target[b, 0, t] = 1e-30
        for later in (t + 1, t + 70, t + 300, t + 5000, V - 1):
            if later < V and later != t:
                target[b, 0, later] = 1.0
    none = torch.zeros((6, 0), dtype=torch.long)
    _check(verify, target, None, none, torch.zeros((6, 1)))
    got, _ = verify(target.cuda(), None, none.cuda(), torch.zeros((6, 1)).cuda())
    assert got[:, 0].tolist() == first
