"""A launch takes fewer than 2^32 lanes: the 8-bit cache's entry points name that limit before they
launch (made-up, never read addresses; no GPU)."""
import pytest

from midiseq import _lib as L

A = 1 << 40


def write(B, T, H, hs, S, block=64):
    return L.lib().msq_kv8_write(1, A, A, A, A, A, A, H * hs * T, H * hs, B, T, H, hs, S, 6, block, A, 0, None)


def read(rows, hs, dtype, S=1 << 30):
    return L.lib().msq_kv8_read(dtype, A, A, A, A, A, A, 1, 1, hs, S, 6, 64, A, 0, 0, rows, None)


def attend(B, H, hs, S):
    lib = L.lib()
    n = lib.msq_relattn_decode_kv8_workspace(B, H, hs, S)
    return lib.msq_relattn_decode_kv8(1, A, H * hs, A, H * hs, A, A, A, A, A, S, B, H, hs, S, 6, 64, A, 0, 1.0, A, n, None)


@pytest.mark.parametrize("call", [
    lambda: write(65535, 1, 128, 8, 70),            # 2^24 - 2^8 workgroups: within; 129 heads below are past it
    lambda: read((1 << 29) - 16 * 32, 128, 1), lambda: read((1 << 28) - 32, 128, 0),
    lambda: attend(65535, 255, 8, 22)])
def test_within(call):
    """gets as far as the launch (there is no GPU here to take it)"""
    import torch
    if torch.cuda.is_available():
        pytest.skip("would launch with made-up addresses")
    assert call() != -1


@pytest.mark.parametrize("call", [
    lambda: write(65535, 1, 129, 8, 70), lambda: write(8192, 1 << 20, 8, 128, 1 << 25),
    lambda: read(1 << 29, 128, 1), lambda: read(1 << 28, 128, 0), lambda: read((1 << 30), 64, 1),
    lambda: attend(65535, 257, 8, 22), lambda: attend(16384, 1024, 64, 64)])
def test_past_it(call):
    assert call() == -1
    assert b"launch takes under" in L.lib().msq_last_error()
