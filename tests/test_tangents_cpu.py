"""Forward-mode tangents (torch.autograd.forward_ad): a dual tensor has no requires_grad and an
ordinary address, so an entry point that does not look for one would drop it in silence. Refused
before any launch (no GPU), also under no_grad, where tangents still pass through torch's operations."""
import contextlib
from types import SimpleNamespace

import pytest
import torch
import torch.autograd.forward_ad as fwad

from midiseq import attention as A
from midiseq.loss import _TokenLogprobs, token_logprobs

ZERO = torch.zeros(2, dtype=torch.int64)


def dual(*shape):
    return fwad.make_dual(torch.zeros(shape), torch.ones(shape))


def score(x):
    return token_logprobs(x, ZERO, 1)


def write(k, v):
    A.kv8_write(*A.kv8_cache(2, 3, 22, 16, device="cpu", block=16), k, v, ZERO, block=16)


def attend(q, R, out=None):
    A.relattn_decode_kv8(q, *A.kv8_cache(2, 3, 22, 16, device="cpu", block=16), R, ZERO, 1.0, out=out, block=16)


K, Q, R = (2, 1, 3, 16), (2, 3, 16), (3, 22, 16)


@pytest.mark.parametrize("mode", [contextlib.nullcontext, torch.no_grad])
@pytest.mark.parametrize("call,error", [
    (lambda: score(dual(2, 7)), NotImplementedError),
    (lambda: score(dual(7, 2).t()), NotImplementedError),
    (lambda: score(dual(2, 7).requires_grad_()), NotImplementedError),
    (lambda: write(dual(*K), torch.zeros(K)), ValueError),
    (lambda: write(torch.zeros(K), dual(*K)), ValueError),
    (lambda: attend(dual(*Q), torch.zeros(R)), ValueError),
    (lambda: attend(torch.zeros(Q), dual(*R)), ValueError),
    (lambda: attend(torch.zeros(Q), torch.zeros(R), dual(*Q)), ValueError)])
def test_tangents_are_refused(call, error, mode):
    with fwad.dual_level(), mode():
        with pytest.raises(error, match="forward-mode|no gradient"):
            call()


@pytest.mark.parametrize("call", [lambda: score(torch.zeros(2, 7)), lambda: write(torch.zeros(K), torch.zeros(K)),
                                  lambda: attend(torch.zeros(Q), torch.zeros(R))])
def test_others_pass_the_check(call):
    """inside a dual level, and in inference mode, tensors without a tangent get as far as the GPU's own check"""
    with fwad.dual_level(), pytest.raises(RuntimeError, match="GPU only"):
        call()
    with torch.inference_mode(), pytest.raises(RuntimeError, match="GPU only"):
        call()


def test_the_primal_is_taken():
    with fwad.dual_level(), pytest.raises(RuntimeError, match="GPU only"):
        score(fwad.unpack_dual(dual(2, 7)).primal)


@pytest.mark.parametrize("at", [0, 1, 3])
def test_tangents_of_incoming_gradients_are_refused(at):
    """forward over reverse: the incoming gradients carry them"""
    x = torch.zeros(2, 7)
    ctx = SimpleNamespace(saved_tensors=(x, ZERO, torch.zeros(2, 2), torch.zeros(2), ZERO[:, None]), top=1)
    with fwad.dual_level():
        g = [None] * 4
        g[at] = dual(2, 1) if at == 3 else dual(2)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _TokenLogprobs.backward(ctx, *g)
