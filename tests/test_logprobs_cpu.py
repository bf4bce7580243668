"""Refusals of token_logprobs (no GPU: argument checks run on the host)."""
import pytest
import torch

from midiseq import _lib as L
from midiseq.loss import token_logprobs

X, T = torch.zeros(4, 7), torch.zeros(4, dtype=torch.int64)


@pytest.mark.parametrize("x,t,top", [
    (X.half(), T, 0), (X.double(), T, 0), (X, T.int(), 0), (X, T[:3], 0), (X, T[None], 0), (X, T, 8), (X, T, -1),
    (torch.zeros(4, 40), T, 33), (torch.zeros(4, 0), T, 0), (torch.tensor(1.0), torch.tensor(0), 0)])
def test_refusals(x, t, top):
    with pytest.raises(ValueError):
        token_logprobs(x, t, top)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU only"):
        token_logprobs(X, T)


def test_c_refusals():
    lib, a = L.lib(), 1 << 40
    good = dict(lp=a, ent=a, ids=a, tlp=a, x=a, dt=0, ld=7, tok=a, rows=4, V=7, top=2)
    for bad in (dict(lp=None), dict(x=None), dict(tok=None), dict(dt=2), dict(ld=-1), dict(rows=0), dict(rows=1 << 31),
                dict(V=0), dict(V=1 << 31), dict(top=33, V=50), dict(top=8), dict(top=-1), dict(ids=None), dict(tlp=None)):
        g = {**good, **bad}
        assert lib.msq_token_logprobs(g["lp"], g["ent"], None, g["ids"], g["tlp"], g["x"], g["dt"], g["ld"], g["tok"],
                                      g["rows"], g["V"], g["top"], None) == -1, bad
    good = dict(dx=a, ldd=7, gt=None, stats=a, ids=None, top=0, x=a, dt=1, ld=7, rows=4, V=7)
    for bad in (dict(dx=None), dict(ldd=6), dict(stats=None), dict(gt=a), dict(gt=a, ids=a), dict(top=33), dict(dt=5),
                dict(rows=0), dict(V=0)):
        g = {**good, **bad}
        assert lib.msq_token_logprobs_bwd(g["dx"], g["ldd"], None, None, g["gt"], g["stats"], a, g["ids"], g["top"],
                                          g["x"], g["dt"], g["ld"], a, g["rows"], g["V"], None) == -1, bad
