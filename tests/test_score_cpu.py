"""generate.score refuses rows whose ids the embedding could not look up (it would read outside its
table), before it runs the model; no GPU."""
from types import SimpleNamespace

import pytest
import torch

from midiseq.generate import score

ROWS, META = torch.arange(10).view(2, 5), torch.zeros(2, 6, dtype=torch.int64)


class Reached(Exception):
    pass


def model():
    def forward(*a, **kw):
        raise Reached
    return SimpleNamespace(engine=SimpleNamespace(cfg=SimpleNamespace(vocab_size=10, metadata_vocab_size=3),
                                                  forward=forward))


def at(t, i, v):
    t = t.clone()
    t.view(-1)[i] = v
    return t


@pytest.mark.parametrize("rows,meta", [
    (ROWS.int(), META), (ROWS.float(), META), (ROWS, META.int()), (ROWS[:, :1], META), (ROWS[0], META), (ROWS, META[:1]),
    (ROWS, META[:, :5]), (ROWS, META[0]), (at(ROWS, 3, -100), META), (at(ROWS, 9, -1), META), (at(ROWS, 0, 10), META),
    (ROWS, at(META, 0, 3)), (ROWS, at(META, 11, -1))])
def test_refusals(rows, meta):
    with pytest.raises(ValueError):
        score(model(), rows, meta, device="cpu")


@pytest.mark.parametrize("rows,meta", [(ROWS, META), (ROWS[:, 3:], META), (ROWS.t().contiguous().t(), at(META, 5, 2))])
def test_others_reach_the_model(rows, meta):
    with pytest.raises(Reached):
        score(model(), rows, meta, device="cpu")
