"""token_logprobs on the GPU at the edges of its range, against the formulas in 64 bits.

Error of the kernel's sums: a lane adds at most n = max(72, V / 1024 + 32) terms in order, lanes and
waves another 24, so s is off by S = (n + 24) 2^-24 relative; its terms by X = 2^-22 + 2^-22 |x - M|
each (the exponential, its argument's product with log2 e), here averaged over the terms' weights.
A row that is streamed rescales its sums once per pass of 4 vectors of 16 bytes a lane, by factors
that are off by 2^-22 + 2^-22 |M - m| each. log s is off by all of that (E) and 2^-23 log V;
t, whose terms have one sign, relatively by E and one more rounding a term."""
import math

import numpy as np
import pytest
import torch

from midiseq.loss import token_logprobs

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0 ** -24


def exact(x, tok, gl, gh, ids=None, gt=None):
    """logprob, entropy, all log probabilities, gradient; 64 bits, a row without a finite logit is empty"""
    x = x.double()
    empty = torch.isneginf(x).all(-1)
    lp = torch.log_softmax(x, -1)
    lp[empty] = -math.inf
    p = lp.exp()
    plp = torch.where(p > 0, p * lp.clamp(min=-1e6), torch.zeros_like(p))
    ent = -plp.sum(-1)
    at = torch.arange(len(x), device=x.device)
    d = -p * gl[:, None] - gh[:, None] * (plp + p * ent[:, None])
    d[at, tok] += gl
    if ids is not None:
        d -= p * gt.sum(-1, keepdim=True)
        d.scatter_add_(1, ids, gt)
    d[empty] = 0
    return lp[at, tok], ent, lp, d


def bounds(x, lp, ent, dtype):
    """(error of log s, of logprob for every id, of the entropy); [rows, 1], [rows, V], [rows]"""
    V = x.shape[1]
    x = x.double()
    M = x.max(-1, keepdim=True).values
    dist = (x - M).clamp(min=-200).abs()
    p = lp.exp()
    # 1024 lanes, 4 vectors each; rows that fit the registers are summed against their maximum at once
    N = 16 // x.new_empty(0, dtype=dtype).element_size()
    rescales = math.ceil(V / (4096 * N)) + 1 if V > 9 * 1024 * N - 16 else 0
    E = (max(72, V / 1024 + 32) + 24) * U + (p * (4 * U + 4 * U * dist)).sum(-1, keepdim=True)
    E += rescales * 4 * U * (1 + dist.amax(-1, keepdim=True).clamp(max=40))
    ls = math.log(V)
    t = (ent - ls).abs()[:, None] + ls  # |t / s| = |log s - H| and less
    return E + 2 * U * ls, E + 4 * U * (lp.clamp(min=-1e4).abs() + ls), (E + 2 * U * ls + t * (2 * E + 4 * U))[:, 0]


def gradient_bound(x, lp, ent, d, g1, gh, dtype):
    V = x.shape[1]
    E, _, eH = bounds(x, lp, ent, dtype)
    p, alp, ls, H = lp.exp(), lp.clamp(min=-200).abs(), math.log(V), ent[:, None]
    g2 = gh.abs()[:, None]
    tol = p * ((E + 4 * U * (2 + alp + ls)) * (g1 + g2 * (alp + H)) + g2 * (eH[:, None] + 4 * U * (alp + H)))
    tol += 8 * U * (d.abs() + g1 * (d.abs() > 0.5 * g1)) + 2.0 ** -126 * (1 + g1 + g2 * (1 + alp + H))
    if dtype == torch.bfloat16:
        tol += 2.0 ** -8 * d.abs() * (1 + 2.0 ** -7)
    return tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, 1e9, 1e30, 1e37])
@pytest.mark.parametrize("V", [9, 700, 2600, 17914, 40009])
def test_large_gradients_of_masked_rows(V, scale, dtype):
    """Incoming gradients up to near the type's largest (a loss scale): a masked logit has p = 0 and takes nothing,
    whatever its log probability; the others take finite values."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(8, V, generator=g) * 3).to(dtype)
    x[0, V // 3:] = float("-inf")
    x[1, : V - 3] = torch.finfo(dtype).min
    x[2] = float("-inf")
    x[2, V // 2:V // 2 + max(1, V // 8)] = -1.5          # one class of events
    x[4] = float("-inf")                                # empty
    x[5] = float("-inf")
    x[5, V // 2] = -5.0
    x[6, ::2] = float("-inf")
    x[7, : V // 2] -= 150.0                             # p below the smallest number, but not masked
    tok = torch.tensor([0, V - 1, V // 2, 3, 2, V // 2, 1, V - 1])
    x, tok = x.to(dev), tok.to(dev)
    sign = torch.randint(0, 2, (8, 4), generator=g) * 2 - 1
    gl, gh, gt = ((torch.rand(8, n, generator=g) + 0.5) * sign[:, :n] * scale for n in (1, 1, 2))
    gl, gh, gt = gl[:, 0].to(dev), gh[:, 0].to(dev), (gt / 2).to(dev)
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, tok, 2)
    for use in ((1, 1, 1), (0, 1, 0), (1, 1, 0)):
        outs = [o for o, u in zip((r.logprob, r.entropy, r.top_logprobs), use) if u]
        (dx,) = torch.autograd.grad(outs, leaf, [v for v, u in zip((gl, gh, gt), use) if u], retain_graph=True)
        l64, t64 = gl.double() * use[0], gt.double() * use[2]
        _, ent, lp, d = exact(x, tok, l64, gh.double(), r.top_ids, t64)
        lp = torch.where(torch.isneginf(x).all(-1, keepdim=True), torch.full_like(lp, -1e4), lp)
        g1 = l64.abs()[:, None] + t64.abs().sum(-1, keepdim=True)
        tol = gradient_bound(x.clamp(min=-1e4), lp, ent, d, g1, gh.double(), dtype)
        assert torch.isfinite(dx).all(), (use, torch.nonzero(~torch.isfinite(dx))[:4])
        off = ((dx.double() - d).abs() - tol).max().item()
        assert off <= 0, (use, off)
        assert (dx[4] == 0).all()
        if not use[2]:  # (an alternative may be a masked one)
            masked = torch.isneginf(x)
            masked[torch.arange(8, device=dev), tok] = False
            assert (dx[masked] == 0).all()


def test_nan_still_spreads_over_its_row():
    x = torch.randn(3, 700, device=dev)
    x[1, 5], x[0, 100:] = float("nan"), float("-inf")
    leaf = x.requires_grad_(True)
    r = token_logprobs(leaf, torch.tensor([1, 2, 3], device=dev))
    (dx,) = torch.autograd.grad((r.logprob, r.entropy), leaf, (torch.full((3,), 1e9, device=dev),) * 2)
    assert torch.isnan(dx[1]).all() and torch.isfinite(dx[[0, 2]]).all()


def test_forward_over_reverse_is_refused():
    import torch.autograd.forward_ad as fwad
    x = torch.randn(3, 8, device=dev, requires_grad=True)
    tok = torch.zeros(3, dtype=torch.int64, device=dev)
    with fwad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            token_logprobs(fwad.make_dual(x.detach(), torch.ones_like(x)), tok)
        lp = token_logprobs(x, tok).logprob
        g = fwad.make_dual(torch.ones(3, device=dev), torch.ones(3, device=dev))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(lp, x, g)


def check(x, tok, dtype, seed=0):
    """both passes within the bounds above"""
    g = torch.Generator(dev).manual_seed(seed)
    gl, gh = torch.randn(len(x), device=dev, generator=g), torch.randn(len(x), device=dev, generator=g)
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, tok)
    (dx,) = torch.autograd.grad((r.logprob, r.entropy), leaf, (gl, gh))
    want, ent, lp, d = exact(x, tok, gl.double(), gh.double())
    _, tol, tol_ent = bounds(x, lp, ent, dtype)
    tol = tol[torch.arange(len(x), device=dev), tok]
    assert ((r.logprob.double() - want).abs() <= tol).all(), ((r.logprob.double() - want).abs() / tol).max().item()
    off = ((r.entropy.double() - ent).abs() / tol_ent).max().item()
    assert off <= 1, off
    off = ((dx.double() - d).abs() / gradient_bound(x, lp, ent, d, gl.double().abs()[:, None], gh.double(), dtype)).max().item()
    assert off <= 1, off
    assert tol.max().item() < 2e-4  # (the bounds are as tight as meant)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [7, 1029])
@pytest.mark.parametrize("V", [60, 700, 1501, 4099, 9001, 17914, 20011, 36001, 80003])
def test_every_form_is_tight(rows, V, dtype):
    g = torch.Generator(dev).manual_seed(V)
    x = (torch.randn(rows, V, device=dev, generator=g) * 3).to(dtype)
    check(x, torch.randint(0, V, (rows,), device=dev, generator=g), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5000, 36001, 80003, 400_009])
def test_running_maximum(V, dtype):
    """Rows whose maximum rises (or falls) all along, whose largest value is the last or the first of a pass, and rows
    of a low plateau with a high end: a wrong rescale or a vector left out shows in the sum."""
    ramp = torch.linspace(0, 12, V, device=dev)
    x = torch.stack([ramp, ramp.flip(0), torch.where(ramp < 6, -4.0, ramp), (ramp * 2 - 12).abs(), ramp * 0 - 7.5,
                     torch.where(torch.arange(V, device=dev) == V - 1, 8.0, 0.0),
                     torch.where(torch.arange(V, device=dev) == 0, 8.0, 0.0)]).to(dtype)
    check(x, torch.tensor([V - 1, 0, 5, V // 2, V // 3, V - 1, 1], device=dev), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 8, 9, 63, 511, 4096, 17914, 40009, 80003])
def test_equal_values_give_log_V(V, dtype):
    """Every term is 1 and their sum exact, so only the logarithm is rounded: two units of it."""
    x = torch.full((3, V), -2.75, device=dev, dtype=dtype)
    r = token_logprobs(x, torch.tensor([0, V - 1, V // 2], device=dev))
    tol = 2 * 2.0 ** (math.floor(math.log2(max(math.log(V), 2.0 ** -20))) - 23)
    for got, want in ((r.logprob, -math.log(V)), (r.entropy, math.log(V))):
        assert ((got.double() - want).abs() <= tol).all(), (got, want)
