"""What a Transformer decode cache allocates (no GPU)."""
import pytest
import torch

from midiseq.transformer import TransformerConfig, TransformerDecodeCache


@pytest.mark.parametrize("kv", [None, "fp8"])
def test_buffers(kv):
    cfg = TransformerConfig(n_embd=64, n_heads=2, n_layer=3, block_len=200, dropout=0.0)
    c = TransformerDecodeCache(cfg, 2, 200, torch.device("cpu"), torch.bfloat16, kv)
    assert c.k.shape == c.v.shape == (3, 2, 2, 206, 32)
    if kv:
        assert c.k.dtype == torch.float8_e4m3fn and c.k_scale.shape == (3, 2, 2, 4)
        assert c.attn_ws is None  # the bf16 attention's
    else:
        assert c.k.dtype == torch.bfloat16 and c.attn_ws.numel() > 0
