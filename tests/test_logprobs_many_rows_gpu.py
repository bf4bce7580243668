"""token_logprobs over more rows than one launch can take (2^32 lanes): one row of logits that is
broadcast, so that every row has the answers of a call of a few thousand."""
import pytest
import torch

from midiseq.loss import token_logprobs

pytestmark = pytest.mark.gpu
dev = "cuda"


def logits(V, seed=0):
    g = torch.Generator(dev).manual_seed(seed)
    return (torch.randn(1, V, device=dev, generator=g) * 3).to(torch.bfloat16)


@pytest.mark.parametrize("rows,V,top", [
    ((1 << 26) + 5, 60, 0),      # four rows to a workgroup of 256
    ((1 << 24) + 3, 5000, 0),    # 256 lanes a row
    ((1 << 23) + 3, 20011, 0),   # 512
    ((1 << 22) + 3, 40009, 0),   # 1024
    (2 * ((1 << 22) - 1), 100, 2), (2 * ((1 << 22) - 1) + 1, 100, 2)])
def test_forward(rows, V, top):
    base = logits(V)
    tok = torch.arange(rows, device=dev) % (V + 3) - 1  # some outside
    few = token_logprobs(base.expand(2 * (V + 3), V) if V > 1000 else base.expand(2048, V),
                         torch.arange(max(2048, 2 * (V + 3)) if V <= 1000 else 2 * (V + 3), device=dev) % (V + 3) - 1, top)
    r = token_logprobs(base.expand(rows, V), tok, top)
    assert torch.equal(r.logprob, few.logprob[tok + 1])
    assert (r.entropy == few.entropy[0]).all()
    if top:
        assert (r.top_ids == few.top_ids[0]).all() and (r.top_logprobs == few.top_logprobs[0]).all()


@pytest.mark.parametrize("rows,V", [((1 << 26) + 5, 3), ((1 << 22) + 3, 2064), (2 * ((1 << 22) - 1), 9)])
def test_gradient(rows, V):
    base, many = logits(V), 4 * (V + 3)
    dx = []
    for n in (max(2048, many), rows):
        leaf = base.expand(n, V).detach().requires_grad_(True)
        tok = torch.arange(n, device=dev) % (V + 3) - 1
        gl, gh = ((torch.arange(n, device=dev) % m).float() - 1 for m in (2, 4))
        r = token_logprobs(leaf, tok, 2)
        gt = torch.stack([gh, gl], -1)
        dx.append(torch.autograd.grad((r.logprob, r.entropy, r.top_logprobs), leaf, (gl, gh, gt))[0])
    # tokens repeat after V + 3 rows, gradients after 4: rows of one place in that period agree
    period = many
    few = dx[0][:period]
    for a in range(0, rows, period << 12):
        part = dx[1][a:a + (period << 12)]
        whole = len(part) // period * period
        assert (part[:whole].view(-1, period, V) == few).all()
        assert torch.equal(part[whole:], few[:len(part) - whole])
