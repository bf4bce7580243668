"""token_logprobs on the GPU (msq_token_logprobs, _bwd) against oracle/logprobs.py (64 bits).

Tolerances. Forward, fp32 (the logits are read as they are): x - M is rounded
once, an exponential is off by 2^-22 relative and its argument's scaling by
2^-23 |x - M| (terms with |x - M| > 20 do not count), a sum of V terms of one sign in
any order by at most V 2^-24 (kept generous; pairwise trees do far better), so
log s by that much absolute: A = (V + 64) 2^-24. logprob: A + 3 * 2^-24 (|x - M| +
log s). Entropy: log s - t / s: A + (V + 64) 2^-24 (t / s), all <= A (2 + H) + 2^-22 H.
Backward: p is off relative by A + 2^-22 (1 + |lp|), an element by that times |p|
times the row's gradients (|g|, times 1 + |lp| + H for the entropy's); a bf16
element by another 2^-8 of its value. p under 2^-126 may come out as 0."""
import numpy as np
import pytest
import torch

from midiseq.loss import token_logprobs
from oracle import logprobs as olp

pytestmark = pytest.mark.gpu
dev = "cuda"


def forward_tol(x, V, lp, ent):
    A = (V + 64) * 2.0 ** -24
    ls = np.log(V)
    return (A + 3 * 2.0 ** -24 * (np.abs(lp) + ls),
            A * (2 + np.nan_to_num(ent)) + 2.0 ** -22 * (1 + np.nan_to_num(ent)))


def close(got, want, tol):
    got = got.detach().double().cpu().numpy()
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        ok = same | (np.isfinite(want) & (np.abs(got - want) <= tol))
    assert ok.all(), (got[~ok][:4], want[~ok][:4])


def check_forward(x64, tokens, r, top):
    lp, ent, ids, tlp = olp.forward(x64, tokens, top)
    V = x64.shape[1]
    t_lp, t_ent = forward_tol(x64, V, lp, ent)
    close(r.logprob.reshape(-1), lp, t_lp)
    close(r.entropy.reshape(-1), ent, t_ent)
    if top:
        np.testing.assert_array_equal(r.top_ids.reshape(-1, top).cpu().numpy(), ids)
        close(r.top_logprobs.reshape(-1, top), tlp, (V + 64) * 2.0 ** -24 + 3 * 2.0 ** -24 * (np.abs(tlp) + np.log(V)))
    else:
        assert r.top_ids is None and r.top_logprobs is None


def check_backward(x64, tokens, ids, g, dx, dtype):
    want = olp.backward(x64, tokens, ids, *g)
    V = x64.shape[1]
    lp = np.stack([olp.row_logp(r) for r in x64])
    with np.errstate(invalid="ignore", over="ignore"):
        p = np.nan_to_num(np.exp(lp))
        alp = np.where(p > 0, np.abs(np.nan_to_num(lp, neginf=0)), 0)
        H = (p * alp).sum(-1, keepdims=True)
        rel = (V + 64) * 2.0 ** -24 + 2.0 ** -22 * (1 + alp)
        g1 = sum(np.abs(t).reshape(len(x64), -1).sum(-1, keepdims=True) for t in (g[0], g[2]) if t is not None)
        g2 = np.abs(g[1])[:, None] if g[1] is not None else 0
        tol = p * (rel + 4 * 2.0 ** -24) * (g1 + g2 * (1 + alp + H)) + p * g2 * ((V + 64) * 2.0 ** -24 * (2 + H) + 2.0 ** -22 * (1 + H + alp))
        # an exponential under the smallest normal fp32, 2^-126, may come out as 0: off by less than
        # 2^-126 in p, so by that times the row's gradients
        tol += 4 * 2.0 ** -24 * np.abs(want) + 2.0 ** -126 * (1 + g1 + g2 * (1 + alp + H))
        if dtype == torch.bfloat16:
            tol += 2.0 ** -8 * np.abs(want) * (1 + 2.0 ** -7)
    close(dx, want, tol)


def reference(x, tok, gl, gh):
    """the same answers in 64 bits by torch, for many rows: logprob, entropy, sorted log probabilities, gradient"""
    lp = torch.log_softmax(x.double(), -1)
    p = lp.exp()
    ent = -torch.special.xlogy(p, p).sum(-1)
    at = torch.arange(len(x), device=dev)
    d = p * (-gl - gh * ent)[:, None] - gh[:, None] * torch.special.xlogy(p, p)
    d[at, tok] += gl
    return lp[at, tok], ent, lp, d


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", [(1025, 60), (1026, 700), (1027, 1501), (1025, 4099), (1030, 9001), (1025, 17914),
                                    (1024, 20011), (1025, 40009), (1024, 80003), (1023, 3001)])
def test_many_rows(rows, V, dtype):
    """Each of the kernel's forms (by the row's length, and whether the rows are many), both passes.
    Tolerances as above, of the tensors' largest."""
    g = torch.Generator(dev).manual_seed(V)
    x = (torch.randn(rows, V, device=dev, generator=g) * 3).to(dtype)
    tok = torch.randint(0, V, (rows,), device=dev, generator=g)
    gl, gh = torch.randn(rows, device=dev, generator=g), torch.randn(rows, device=dev, generator=g)
    lp, ent, all_lp, d = reference(x, tok, gl.double(), gh.double())
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, tok, 6)
    r0 = token_logprobs(x, tok, 6)  # the form without a gradient
    for a, b in zip(r, r0):
        assert torch.equal(a, b)
    A = (V + 64) * 2.0 ** -24
    big = lp.abs().max().item() + np.log(V)
    assert ((r.logprob - lp).abs().max() <= A + 3 * 2.0 ** -24 * big).item()
    assert ((r.entropy - ent).abs().max() <= A * (2 + np.log(V)) + 2.0 ** -22 * (1 + np.log(V))).item()
    # stable: equal values by index
    want = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :6]
    assert torch.equal(r.top_ids, want)
    assert ((r.top_logprobs - all_lp.gather(1, want)).abs().max() <= A + 3 * 2.0 ** -24 * big).item()
    (dx,) = torch.autograd.grad((r.logprob, r.entropy), leaf, (gl, gh))
    g1, g2 = gl.abs()[:, None], gh.abs()[:, None]
    alp = all_lp.abs()
    tol = all_lp.exp() * ((A + 2.0 ** -22 * (1 + alp)) * (g1 + g2 * (1 + alp + np.log(V))) * 2)
    tol += 2.0 ** -22 * d.abs() + 2.0 ** -126 * (1 + g1 + g2 * (1 + alp + np.log(V)))
    if dtype == torch.bfloat16:
        tol += 2.0 ** -8 * d.abs() * (1 + 2.0 ** -7)
    off = (dx.double() - d).abs() - tol
    assert (off.max() <= 0).item(), off.max().item()


SIZES = [(1, 1), (3, 2), (5, 7), (4, 33), (2, 255), (6, 1025), (3, 4099), (2, 17914), (2, 70001), (300, 40)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", SIZES)
def test_forward_and_gradient(rows, V, dtype):
    g = np.random.default_rng(rows + V)
    x = torch.from_numpy(g.standard_normal((rows, V)) * 3).to(dtype)
    tok = torch.from_numpy(g.integers(0, V, rows))
    if rows > 2:
        tok[0], tok[1] = -100, V  # padded places
    x64, t = x.double().numpy(), tok.numpy()
    for top in sorted({0, 1, min(5, V), min(32, V)}):
        check_forward(x64, t, token_logprobs(x.to(dev), tok.to(dev), top), top)
    for top, use in ((0, (1, 1, 0)), (0, (1, 0, 0)), (0, (0, 1, 0)), (min(4, V), (1, 1, 1)), (min(4, V), (0, 0, 1))):
        leaf = x.to(dev).requires_grad_(True)
        r = token_logprobs(leaf, tok.to(dev), top)
        gs = [g.standard_normal(s) * u if u else None for s, u in zip(((rows,), (rows,), (rows, top)), use)]
        outs = [o for o, u in zip((r.logprob, r.entropy, r.top_logprobs), use) if u]
        (dx,) = torch.autograd.grad(outs, leaf, [torch.from_numpy(v).float().to(dev) for v in gs if v is not None])
        gs = [None if v is None else torch.from_numpy(v).float().double().numpy() for v in gs]
        assert dx.dtype == dtype and dx.shape == leaf.shape
        check_backward(x64, t, None if r.top_ids is None else r.top_ids.cpu().numpy(), gs, dx, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    """Padded rows, rows at odd offsets, a model's [B, T, V] view, a transposed last axis, every
    second row: the same answers as from a contiguous copy, and gradients of the view's base."""
    g = torch.Generator().manual_seed(2)
    B, T, V = 3, 5, 1003
    big = torch.randn(B * T * 2, 1040, generator=g).to(dtype).to(dev)
    wide = torch.randn(V, B * T, generator=g).to(dtype).to(dev)
    tok = torch.randint(0, V, (B, T), generator=g).to(dev)
    views = [big[:B * T, :V], big[:B * T, 1:V + 1], big[::2, 5:V + 5], big.view(-1)[3:3 + B * T * V].view(-1, V),
             big.view(-1)[:B * T * V].view(-1, V), wide.t()]
    for v in views:
        want = token_logprobs(v.contiguous().clone(), tok.view(-1), 7)
        got = token_logprobs(v, tok.view(-1), 7)
        for a, b in zip(got, want):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-5) if a.is_floating_point() else torch.equal(a, b)
        if v.stride(0) % 1 == 0 and v.numel() == B * T * V:
            v3 = v.unflatten(0, (B, T))
            got3 = token_logprobs(v3, tok, 7)
            assert got3.logprob.shape == (B, T) and got3.top_ids.shape == (B, T, 7)
            assert torch.equal(got3.logprob.view(-1), got.logprob)
        leaf, ref = v.detach().requires_grad_(True), v.detach().contiguous().clone().requires_grad_(True)
        grads = [torch.autograd.grad(token_logprobs(t, tok.view(-1)).logprob.sum() +
                                     token_logprobs(t, tok.view(-1)).entropy.sum(), t)[0] for t in (leaf, ref)]
        assert torch.allclose(grads[0].float(), grads[1].float(), rtol=2 ** -7 if dtype == torch.bfloat16 else 1e-4, atol=1e-6)


def test_broadcast_rows():
    """One row of logits for many tokens (stride 0): its gradient is the rows' sum."""
    g = torch.Generator().manual_seed(3)
    base = torch.randn(1, 57, generator=g).to(dev).requires_grad_(True)
    tok = torch.randint(0, 57, (64,), generator=g).to(dev)
    (got,) = torch.autograd.grad(token_logprobs(base.expand(64, 57), tok).logprob.sum(), base)
    p = torch.softmax(base.detach().double(), -1)
    want = torch.zeros_like(p).index_add_(1, tok, torch.ones(1, 64, device=dev, dtype=torch.float64)) - 64 * p
    assert torch.allclose(got.double(), want, atol=1e-4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [9, 700, 5003, 80003])
def test_masks(V, dtype):
    """-inf, the type's lowest value, empty rows, one live logit, +inf and NaN, and ties of all of them."""
    g = np.random.default_rng(V)
    low = torch.finfo(dtype).min
    x = torch.from_numpy(g.standard_normal((12, V))).to(dtype)
    x[0, V // 3:] = float("-inf")
    x[1, : V - 2] = low
    x[2] = float("-inf")
    x[3] = low
    x[4] = float("-inf")
    x[4, V // 2] = -5.0
    x[5] = 1.5                      # all equal
    x[6, V // 2] = float("nan")
    x[7, 1] = float("inf")
    x[8] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0).to(dtype)   # equal, both zeros
    x[9, : V // 2], x[9, V // 2:] = 2.0, 2.0 - 2.0 ** -6
    x[10] = float("nan")
    x[11] = torch.arange(V).flip(0).to(dtype)
    tok = torch.tensor([1, V - 1, 0, 3, V // 2, 4, 0, 1, 2, V - 1, 0, V - 1])
    x64 = x.double().numpy()
    top = min(9, V)
    leaf = x.to(dev).requires_grad_(True)
    r = token_logprobs(leaf, tok.to(dev), top)
    check_forward(x64, tok.numpy(), r, top)
    gl, gh = torch.from_numpy(g.standard_normal(12)).float(), torch.from_numpy(g.standard_normal(12)).float()
    (dx,) = torch.autograd.grad((r.logprob, r.entropy), leaf, (gl.to(dev), gh.to(dev)))
    check_backward(x64, tok.numpy(), None, (gl.double().numpy(), gh.double().numpy(), None), dx, dtype)
    assert (dx[2] == 0).all()


def test_large_logits():
    """Logits of tens of thousands: differences are taken before anything is scaled."""
    g = np.random.default_rng(0)
    x = torch.from_numpy(30000 + g.standard_normal((4, 600)) * 3).float()
    tok = torch.tensor([0, 1, 2, 3])
    leaf = x.to(dev).requires_grad_(True)
    r = token_logprobs(leaf, tok.to(dev), 3)
    check_forward(x.double().numpy(), tok.numpy(), r, 3)
    (dx,) = torch.autograd.grad((r.logprob.sum() + r.entropy.sum()), leaf)
    check_backward(x.double().numpy(), tok.numpy(), None, (np.ones(4), np.ones(4), None), dx, torch.float32)


def test_gradient_against_differences():
    """Directional differences of the kernel's own forward: (f(x + h d) - f(x - h d)) / 2h. f is off by at
    most 32 * 2^-24 (|f| < 16), so the quotient by 32 * 2^-24 * 16 / h, and by h^2 / 6 times a third
    derivative <= 8 |d|^3; h = 2^-6, |d| = 1."""
    g = torch.Generator().manual_seed(7)
    x = torch.randn(6, 11, generator=g).to(dev)
    tok = torch.tensor([0, 10, 3, 3, 7, -1], device=dev)
    w = torch.randn(3, 6, generator=g).to(dev)

    def f(x):
        r = token_logprobs(x, tok, 2)
        return (w[0] * r.logprob + w[1] * r.entropy + w[2] * r.top_logprobs.sum(-1)).sum()

    leaf = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(f(leaf), leaf)
    h = 2.0 ** -6
    for _ in range(8):
        d = torch.randn(6, 11, generator=g).to(dev)
        d /= d.norm()
        num = (f(x + h * d).double() - f(x - h * d).double()) / (2 * h)
        tol = w.abs().sum() * (32 * 2.0 ** -24 * 16 / h + h * h / 6 * 8)
        assert abs(num - (dx.double() * d).sum()) <= tol


def test_no_rows_and_one_token():
    x = torch.randn(2, 0, 5, device=dev, requires_grad=True)
    r = token_logprobs(x, torch.zeros(2, 0, dtype=torch.int64, device=dev), 3)
    assert r.logprob.shape == (2, 0) and r.top_ids.shape == (2, 0, 3) and r.top_logprobs.shape == (2, 0, 3)
    (dx,) = torch.autograd.grad(r.logprob.sum() + r.entropy.sum() + r.top_logprobs.sum(), x)
    assert dx.shape == x.shape
    r = token_logprobs(torch.randn(9, device=dev), torch.tensor(4, device=dev), 2)  # a row alone
    assert r.logprob.shape == () and r.top_ids.shape == (2,)


def test_second_derivatives_are_refused():
    x = torch.randn(3, 8, device=dev, requires_grad=True)
    (g,) = torch.autograd.grad(token_logprobs(x, torch.zeros(3, dtype=torch.int64, device=dev)).logprob.sum(), x,
                               create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_changed_logits_are_refused():
    x = torch.randn(3, 8, device=dev, requires_grad=True)
    y = x * 1.0
    r = token_logprobs(y, torch.zeros(3, dtype=torch.int64, device=dev))
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        r.logprob.sum().backward()


def test_graph_and_stream():
    """Captured and replayed over changing logits (eager work between); forward and backward on
    another stream give the same bits."""
    g = torch.Generator(dev).manual_seed(1)
    x, tok = torch.randn(33, 2050, device=dev, generator=g), torch.randint(0, 2050, (33,), device=dev, generator=g)
    token_logprobs(x, tok, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(x, tok, 4)
    side = torch.cuda.Stream()
    for _ in range(4):
        x.normal_(generator=g)
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            leaf = x.clone().requires_grad_(True)
            want = token_logprobs(leaf, tok, 4)
            (dx,) = torch.autograd.grad(want.logprob.sum(), leaf)
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        leaf = x.clone().requires_grad_(True)
        (dx2,) = torch.autograd.grad(token_logprobs(leaf, tok).logprob.sum(), leaf)
        assert torch.equal(dx, dx2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_in_a_graph(dtype):
    """Both passes captured, replayed over other logits, tokens and incoming gradients with eager work
    between; the leaf has no eager graph while its backward pass is captured."""
    g = torch.Generator(dev).manual_seed(2)
    x = torch.randn(70, 4001, device=dev, generator=g).to(dtype).requires_grad_(True)
    tok = torch.randint(-3, 4001, (70,), device=dev, generator=g)
    gl, gh, gt = (torch.randn(70, *s, device=dev, generator=g) for s in ((), (), (3,)))

    def both(x):
        r = token_logprobs(x, tok, 3)
        return [*(t.detach() for t in r), *torch.autograd.grad((r.logprob, r.entropy, r.top_logprobs), x, (gl, gh, gt))]

    both(x.detach().clone().requires_grad_(True))  # everything loaded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(x)
    for _ in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device=dev, generator=g))
        tok.copy_(torch.randint(-3, 4001, (70,), device=dev, generator=g))
        for t in (gl, gh, gt):
            t.normal_(generator=g)
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        for a, b in zip(got, both(x.detach().clone().requires_grad_(True))):
            assert torch.equal(a, b)


def test_rows_past_32_bits():
    """130 000 rows of 17 920 elements: 2.3 G elements; the last rows and their gradient."""
    rows, V, ld = 130_000, 17914, 17920
    x = torch.zeros(rows, ld, device=dev, dtype=torch.bfloat16)
    x[-3:].normal_(generator=torch.Generator(dev).manual_seed(0))
    tok = torch.zeros(rows, dtype=torch.int64, device=dev)
    tok[-3:] = torch.tensor([5, 17913, 9000], device=dev)
    leaf = x[:, :V].requires_grad_(True)
    r = token_logprobs(leaf, tok, 2)
    x64, t = x[-3:, :V].double().cpu().numpy(), tok[-3:].cpu().numpy()
    from midiseq.loss import TokenLogprobs
    check_forward(x64, t, TokenLogprobs(*[v[-3:] for v in r]), 2)
    (dx,) = torch.autograd.grad((r.logprob, r.entropy), leaf, (torch.ones(rows, device=dev), torch.ones(rows, device=dev)))
    check_backward(x64, t, None, (np.ones(3), np.ones(3), None), dx[-3:], torch.bfloat16)
    assert abs(r.logprob[0].item() + np.log(V)) < 1e-3
