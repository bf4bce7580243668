"""The bf16 SSD passes give the same bits every time, and their two forms (the fused scans, and the
kernels per chunk with passes of their own) the same bits as each other: what they hand on in bf16
is rounded from sums in one order, so that no rounding near a tie falls differently from run to run."""
import pytest
import torch

from midiseq import _lib as L
from midiseq import ops
from midiseq._lib import call, ptr, stream

pytestmark = pytest.mark.gpu


def data(B, T, H, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    di = 64 * H
    conv, ldz = di + 128, (2 * di + 128 + H + 3) // 4 * 4
    return dict(B=B, T=T, H=H, di=di, conv=conv, ldz=ldz, xc=rnd(B * T, conv).bfloat16(), zx=rnd(B * T, ldz).bfloat16(),
                dt_bias=rnd(H) - 2, A_log=torch.log(torch.linspace(1, 16, H, device="cuda")), D=rnd(H),
                dy=rnd(B * T, di).bfloat16())


def passes(d):
    """y, dxc and the dt columns of dzx"""
    B, T, H, di = d["B"], d["T"], d["H"], d["di"]
    f = torch.empty(L.lib().msq_mamba_states_size(B, T, H) // 4, device="cuda")
    y = torch.empty(B * T, di, device="cuda", dtype=torch.bfloat16)
    call("msq_mamba_ssd_fwd", ptr(y), di, ptr(f), ptr(d["xc"]), d["conv"], ptr(d["zx"]), d["ldz"], L.BF16,
         ptr(d["dt_bias"]), ptr(d["A_log"]), ptr(d["D"]), B, T, di, H, stream())
    dxc = torch.zeros(B * T, d["conv"], device="cuda")
    dzx = torch.zeros_like(d["zx"])
    gA, gD, gdt = (torch.zeros(H, device="cuda") for _ in range(3))
    ws = ops.workspace(L.lib().msq_mamba_ssd_bwd_workspace(B, T, H), torch.device("cuda", 0), "ssd_bwd")
    call("msq_mamba_ssd_bwd", ptr(dxc), d["conv"], ptr(dzx), ptr(d["dy"]), di, ptr(f), ptr(d["xc"]), d["conv"],
         ptr(d["zx"]), d["ldz"], L.BF16, ptr(d["dt_bias"]), ptr(d["A_log"]), ptr(d["D"]), ptr(gA), ptr(gD), ptr(gdt), B, T,
         di, H, ptr(ws), stream())
    at = di + d["conv"]
    assert (dzx[:, :at] == 0).all()
    return y, dxc, dzx[:, at:at + H].clone()


SHAPES = [(2, 200, 4), (2, 700, 8), (1, 1, 2), (3, 64, 1), (4, 1030, 16)]


@pytest.mark.parametrize("B,T,H", SHAPES)
def test_runs_repeat_bitwise(B, T, H):
    d = data(B, T, H)
    first = passes(d)
    for t in first:
        assert torch.isfinite(t).all()
    for _ in range(15):
        for a, b in zip(first, passes(d)):
            assert torch.equal(a, b), int((a != b).sum())


@pytest.mark.parametrize("B,T,H", SHAPES)
def test_scan_forms_agree_bitwise(B, T, H, monkeypatch):
    d = data(B, T, H, 1)
    monkeypatch.delenv("MSQ_MAMBA_SSD_3K", raising=False)
    fused = passes(d)
    monkeypatch.setenv("MSQ_MAMBA_SSD_3K", "1")
    for a, b in zip(fused, passes(d)):
        assert torch.equal(a, b), int((a != b).sum())
