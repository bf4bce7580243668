"""Refusals of the 8-bit decode cache (no GPU: argument checks run on the host)
and the oracle's own rounding against torch's e4m3 cast."""
import numpy as np
import pytest
import torch

from midiseq import _lib as L
from midiseq import attention as A
from oracle import kv8 as okv

F8 = torch.float8_e4m3fn


def cache(B=2, H=3, S=22, hs=16, block=16):
    return list(A.kv8_cache(B, H, S, hs, device="cpu", block=block))


def test_oracle_rounding_is_torchs():
    y = np.concatenate([np.linspace(-448, 448, 20011), okv._GRID, (okv._GRID[1:] + okv._GRID[:-1]) / 2,
                        2.0 ** -np.arange(1, 20)])
    t = torch.from_numpy(y).to(torch.float32)  # torch's cast from fp32: the same inputs for both
    np.testing.assert_array_equal(okv.e4m3_round(t.double().numpy()), t.to(F8).double().numpy())


def test_oracle_scale():
    for amax, want in [(0.0, 2.0 ** -126), (448.0, 1.0), (448.0001, 2.0), (224.0, 0.5), (225.0, 1.0), (1.0, 2.0 ** -8)]:
        assert okv.scale_of(amax) == want


def test_oracle_largest_values():
    """Finite fp32 values stay finite and within 2^-4, also once they are coded again."""
    r = okv.Ring(1, 16, 8, 0, 16)
    x = np.array([3.4028234663852886e38, -1.9375 * 2.0 ** 127, 1.875 * 2.0 ** 127, 1.75 * 2.0 ** 127, 0, 0, 0, 0])
    r.write(x[None, None], 0)
    for p in (1, 2):
        r.write(np.full((1, 1, 8), 0.5), p)
        got = r.rows()[0, 0].astype(np.float32).astype(np.float64)
        assert (np.abs(got - x) <= 2.0 ** -4 * np.abs(x)).all()


@pytest.mark.parametrize("kw", [dict(hs=12), dict(hs=0), dict(hs=136), dict(block=48), dict(block=8)])
def test_cache_refusals(kw):
    with pytest.raises(ValueError):
        cache(**kw)


def _write(c, k=None, v=None, pos=None, **kw):
    k = torch.zeros(2, 1, 3, 16) if k is None else k
    A.kv8_write(*c, k, k.clone() if v is None else v, torch.zeros(2, dtype=torch.int64) if pos is None else pos,
                **{"block": 16, **kw})


def _attend(c, q=None, R=None, pos=None, **kw):
    return A.relattn_decode_kv8(torch.zeros(2, 3, 16) if q is None else q, *c,
                                torch.zeros(3, 22, 16) if R is None else R,
                                torch.zeros(2, dtype=torch.int64) if pos is None else pos, 1.0, **{"block": 16, **kw})


@pytest.mark.parametrize("kw", [
    dict(k=torch.zeros(2, 1, 3, 8)), dict(k=torch.zeros(2, 1, 2, 16)), dict(k=torch.zeros(3, 1, 3, 16)),
    dict(k=torch.zeros(2, 3, 16)), dict(k=torch.zeros(2, 1, 3, 16, dtype=torch.float16)),
    dict(v=torch.zeros(2, 1, 3, 16, dtype=torch.bfloat16)), dict(v=torch.zeros(2, 2, 3, 16)),
    dict(k=torch.zeros(2, 1, 16, 3).transpose(2, 3)), dict(k=torch.zeros(2, 1, 3, 32)[..., :16]),
    dict(pos=torch.zeros(3, dtype=torch.int64)), dict(pos=torch.zeros(2)), dict(pos=torch.zeros(2, 1, dtype=torch.int64)),
    dict(pos=torch.zeros(4, dtype=torch.int64)[::2]), dict(block=32), dict(block=17), dict(n_meta=22), dict(n_meta=-1)])
def test_write_refusals(kw):
    with pytest.raises(ValueError):
        _write(cache(), **kw)


def test_scale_and_code_refusals():
    for i, t in [(0, torch.zeros(2, 3, 22, 16)), (2, torch.zeros(2, 3, 21, 16).to(F8)), (1, torch.zeros(2, 3, 3)),
                 (1, torch.zeros(2, 3, 2, dtype=torch.float64)),
                 (0, torch.zeros(2, 3, 16, 22, dtype=torch.uint8).view(F8).transpose(2, 3))]:
        c = cache()
        c[i] = t
        with pytest.raises(ValueError):
            _write(c)
        with pytest.raises(ValueError):
            _attend(c)


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(2, 3, 8)), dict(q=torch.zeros(1, 3, 16)), dict(q=torch.zeros(2, 3, 16, dtype=torch.bfloat16)),
    dict(q=torch.zeros(2, 3, 32)[..., :16]), dict(q=torch.zeros(2, 48)), dict(R=torch.zeros(3, 21, 16)),
    dict(R=torch.zeros(2, 22, 16)), dict(R=torch.zeros(3, 44, 16)[:, ::2]), dict(out=torch.zeros(2, 3, 8)),
    dict(out=torch.zeros(2, 3, 16, dtype=torch.bfloat16)), dict(pos=torch.zeros(5, dtype=torch.int64)),
    dict(block=64)])
def test_attend_refusals(kw):
    with pytest.raises(ValueError):
        _attend(cache(), **kw)


def test_no_gradient_is_refused():
    q = torch.zeros(2, 3, 16, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        _attend(cache(), q=q)
    with pytest.raises(ValueError, match="no gradient"):
        _write(cache(), k=torch.zeros(2, 1, 3, 16, requires_grad=True))


@pytest.mark.parametrize("kw", [dict(first=-1), dict(rows=23), dict(first=20, rows=3), dict(dtype=torch.float16),
                                dict(rows=-1)])
def test_read_refusals(kw):
    with pytest.raises(ValueError):
        A.kv8_read(*cache(), torch.zeros(2, dtype=torch.int64), block=16, **kw)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU only"):
        _write(cache())
    with pytest.raises(RuntimeError, match="GPU only"):
        _attend(cache())
    with pytest.raises(RuntimeError, match="GPU only"):
        A.kv8_read(*cache(), torch.zeros(2, dtype=torch.int64), block=16)


def test_c_refusals():
    """the C entry points check before they launch: bad arguments with made-up (never read) addresses"""
    lib, a = L.lib(), 1 << 40
    good = dict(dtype=1, kc=a, ks=a, vc=a, vs=a, k=a, v=a, ld_b=1, ld_t=1, B=1, T=1, H=1, hs=16, S=22, n_meta=6,
                block=16, pos=a, ps=0)
    for bad in (dict(dtype=2), dict(kc=None), dict(k=None), dict(pos=None), dict(kc=a + 4), dict(B=0), dict(B=65536),
                dict(T=0), dict(H=0), dict(hs=20), dict(hs=136), dict(S=6), dict(n_meta=-1), dict(block=24),
                dict(ps=2), dict(ld_t=-1), dict(S=(1 << 30) + 1), dict(H=32767, T=1 << 30, S=1 << 30)):
        g = {**good, **bad}
        rc = lib.msq_kv8_write(g["dtype"], g["kc"], g["ks"], g["vc"], g["vs"], g["k"], g["v"], g["ld_b"], g["ld_t"],
                               g["B"], g["T"], g["H"], g["hs"], g["S"], g["n_meta"], g["block"], g["pos"], g["ps"], None)
        assert rc == -1, bad
        assert b"msq_kv8_write" in lib.msq_last_error()
    good = dict(dtype=1, out=a, ldo=48, q=a, ldq=48, kc=a, R=a, S_max=22, B=1, H=3, hs=16, S=22, n_meta=6, block=16,
                pos=a, ps=1, ws=a, n=1 << 30)
    for bad in (dict(dtype=0 + 2), dict(out=None), dict(R=None), dict(ldq=40), dict(ldq=52), dict(ldo=47),
                dict(q=a + 2), dict(R=a + 8), dict(S_max=21), dict(hs=132), dict(block=0), dict(ps=-1),
                dict(B=64, S=2054, S_max=2054, n=16), dict(B=1, S=2054, S_max=2054, ws=None),
                dict(B=1, S=2054, S_max=2054, ws=a + 4)):
        g = {**good, **bad}
        rc = lib.msq_relattn_decode_kv8(g["dtype"], g["out"], g["ldo"], g["q"], g["ldq"], g["kc"], a, a, a, g["R"],
                                        g["S_max"], g["B"], g["H"], g["hs"], g["S"], g["n_meta"], g["block"], g["pos"],
                                        g["ps"], 1.0, g["ws"], g["n"], None)
        assert rc == -1, bad
    assert lib.msq_kv8_blocks(100, 33) == -1 and lib.msq_kv8_blocks(100, 32) == 4
    for first, rows in ((-1, 2), (0, 0), (20, 3)):
        assert lib.msq_kv8_read(1, a, a, a, a, a, a, 1, 1, 16, 22, 6, 16, a, 0, first, rows, None) == -1
