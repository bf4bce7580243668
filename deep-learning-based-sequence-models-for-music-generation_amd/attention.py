"""Relative-position attention launchers (HeadRelPos x n_heads,
models/transformer/model_transformer.py:41-90) over the libmidiseq C ABI."""
import functools

import torch

from . import _lib as L
from ._lib import ptr, call, stream, dt, stream_of, has_tangent
from .ops import workspace

N_META = 6  # metadata prefix (generate_matrix, model_transformer.py:14)


def relattn_fwd(qkv, R, B, S, H, hs, scale, out=None, lse=None, n_meta=N_META, drop=None):
    """qkv [B*S, >=3*H*hs] (bf16 -> flash MFMA path, fp32 -> exact path),
    R [H, S_max, hs]. Returns (out [B*S, H*hs], lse fp32 [B, H, S]).
    drop=(masks [2, n] from ops.dropout_attn_mask, p): attention-probability dropout."""
    if out is None:
        out = torch.empty(B * S, H * hs, device=qkv.device, dtype=qkv.dtype)
    if lse is None:
        lse = torch.empty(B, H, S, device=qkv.device, dtype=torch.float32)
    masks, p = drop if drop is not None else (None, 0.0)
    call("msq_relattn_fwd_dropout", dt(qkv), ptr(out), out.stride(0), ptr(lse), ptr(qkv), qkv.stride(0), ptr(R), B,
         S, H, hs, R.shape[1], float(scale), n_meta, ptr(masks[0]) if masks is not None else None,
         ptr(masks[1]) if masks is not None else None, float(p), stream())
    return out, lse


# workspace slot ("attn", device, stream) -> (buffer address, (dtype, B, S, H,
# n_meta)) of the backward it last served: its zero bands stay valid for the
# next backward of the same shape in the SAME buffer (msq_relattn_bwd_ws). A
# slot whose buffer was replaced (grown) has a new address and starts cold.
_ws_served = {}


def relattn_bwd(dout, out, lse, qkv, R, B, S, H, hs, scale, dqkv=None, dR=None, n_meta=N_META, drop=None):
    """Returns (dqkv [B*S, 3*H*hs] (overwritten), dR fp32 [H, S_max, hs] (accumulated))."""
    if dqkv is None:
        dqkv = torch.empty(B * S, 3 * H * hs, device=qkv.device, dtype=qkv.dtype)
    if dR is None:
        dR = torch.zeros(R.shape, device=qkv.device, dtype=torch.float32)
    nbytes = L.lib().msq_relattn_bwd_workspace(dt(qkv), B, S, H)
    ws = workspace(nbytes, qkv.device, "attn")
    masks, p = drop if drop is not None else (None, 0.0)
    key = (dt(qkv), B, S, H, n_meta)
    slot = ("attn", qkv.device, torch.cuda.current_stream(qkv.device).cuda_stream)
    ready = int(_ws_served.get(slot) == (ws.data_ptr(), key))  # the "attn" workspace serves only this op
    call("msq_relattn_bwd_ws", dt(qkv), ptr(dqkv), dqkv.stride(0), ptr(dR), ptr(dout), dout.stride(0), ptr(out),
         ptr(lse), ptr(qkv), qkv.stride(0), ptr(R), B, S, H, hs, R.shape[1], float(scale), n_meta,
         ptr(masks[0]) if masks is not None else None, ptr(masks[1]) if masks is not None else None, float(p),
         ptr(ws), ready, stream())
    _ws_served[slot] = (ws.data_ptr(), key)
    return dqkv, dR


# ---- the decode cache in 8 bits (msq_kv8_*, msq_relattn_decode_kv8)

KV8_BLOCK = 64  # slots that share a scale
_F8, _F32, _BF16, _I64 = torch.float8_e4m3fn, torch.float32, torch.bfloat16, torch.int64


def kv8_cache(B, H, S_ring, hs, device="cuda", block=KV8_BLOCK, layers=()):
    """An empty 8-bit ring (kc, ks, vc, vs): e4m3 codes [*layers, B, H, S_ring,
    hs] and fp32 scales [*layers, B, H, ceil(S_ring / block)] of the keys and of
    the values."""
    nblk = L.lib().msq_kv8_blocks(S_ring, block)
    if nblk < 0:
        raise ValueError(f"a ring of {S_ring} slots in blocks of {block} (16, 32, 64 or 128)")
    if hs <= 0 or hs > 128 or hs % 8:
        raise ValueError(f"head size {hs}: the 8-bit cache needs 8 | hs <= 128")
    codes = [torch.zeros(*layers, B, H, S_ring, hs, device=device, dtype=torch.uint8).view(torch.float8_e4m3fn)
             for _ in range(2)]
    scales = [torch.ones(*layers, B, H, nblk, device=device, dtype=torch.float32) for _ in range(2)]
    return codes[0], scales[0], codes[1], scales[1]


def _kv8_args(kc, ks, vc, vs, pos, n_meta, block):
    """the checked cache: (pointers, (B, H, hs, S_ring, n_meta, block, pos, pos_stride))"""
    shape = kc.shape
    if kc.dtype is not _F8 or vc.dtype is not _F8 or len(shape) != 4 or vc.shape != shape:
        raise ValueError(f"the cache is two float8_e4m3fn [B, H, S_ring, hs] tensors, got {kc.dtype} "
                         f"{tuple(kc.shape)} and {vc.dtype} {tuple(vc.shape)}")
    B, H, S_ring, hs = shape
    if not 0 <= n_meta < S_ring or block not in (16, 32, 64, 128):
        raise ValueError(f"a ring of {S_ring} slots, {n_meta} of them metadata, in blocks of {block}")
    want = (B, H, -(-S_ring // block))
    if ks.dtype is not _F32 or vs.dtype is not _F32 or ks.shape != want or vs.shape != want:
        raise ValueError(f"the scales are two float32 {list(want)} tensors, got {ks.dtype} {tuple(ks.shape)} and "
                         f"{vs.dtype} {tuple(vs.shape)}")
    if not (kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("the cache and its scales have to be contiguous")
    n = pos.numel()
    if pos.dtype is not _I64 or pos.dim() > 1 or (n != 1 and n != B) or not pos.is_contiguous():
        raise ValueError(f"pos is an int64 tensor of 1 or {B} positions, got {pos.dtype} {tuple(pos.shape)}")
    dev = kc.get_device()
    if not dev == vc.get_device() == ks.get_device() == vs.get_device() == pos.get_device():
        raise ValueError("the cache, its scales and pos have to be on one device")
    return ((kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr()),
            (B, H, hs, S_ring, n_meta, block, pos.data_ptr(), 0 if n == 1 else 1))


def _kv8_beside(kc, *others):
    """operands that go with the cache: on its device, without a gradient"""
    grad = torch.is_grad_enabled()
    for t in others:
        if t.get_device() != kc.get_device():
            raise ValueError(f"the cache is on {kc.device}, an operand on {t.device}")
        if grad and t.requires_grad:
            raise ValueError("the 8-bit cache has no gradient: call it under torch.no_grad()")
    if has_tangent(*others):
        raise ValueError("the 8-bit cache has no gradient: forward-mode tangents would be lost")


def kv8_write(kc, ks, vc, vs, k, v, pos, *, n_meta=N_META, block=KV8_BLOCK):
    """Writes new keys and values k, v [B, T, H, hs] (fp32 / bf16; heads hs
    apart, any other strides, the same for both: e.g. views of a packed
    projection) at positions pos .. pos + T - 1 of the ring, in place
    (msq_kv8_write). pos: int64 [B], or [1] for all rows; -n_meta for a prompt
    whose first n_meta rows are metadata; below that a row is left alone.
    Positions are written in order; a row may be taken back to an earlier one
    (a prompt's padding, rejected tokens) while the ring has not come round. An
    element is off by at most 2^-4 of its value plus 2^-9 of the largest scale
    that its block has had since it was written, taken-back rows' among them:
    padding that is far larger than the prompt's last rows costs them (zeros cost
    nothing)."""
    shape, strides = k.shape, k.stride()
    if len(shape) != 4 or v.shape != shape or v.dtype != k.dtype or v.stride() != strides:
        raise ValueError(f"k and v are [B, T, H, hs] alike, got {k.dtype} {tuple(k.shape)} {k.stride()} and "
                         f"{v.dtype} {tuple(v.shape)} {v.stride()}")
    cache, (B, H, hs, *rest) = _kv8_args(kc, ks, vc, vs, pos, n_meta, block)
    _kv8_beside(kc, k, v)
    T = shape[1]
    if shape != (B, T, H, hs) or not (k.dtype is _F32 or k.dtype is _BF16):
        raise ValueError(f"{k.dtype} {tuple(shape)} rows for a cache of {B} x {H} heads of {hs}")
    if strides[3] != 1 or (H > 1 and strides[2] != hs):
        raise ValueError(f"a token's heads have to lie {hs} apart, got strides {strides}")
    s = stream_of(kc)
    if T and B and H:
        call("msq_kv8_write", dt(k), *cache, k.data_ptr(), v.data_ptr(), strides[0], strides[1], B, T, H, hs, *rest, s)


def kv8_read(kc, ks, vc, vs, pos, *, first=0, rows=None, dtype=torch.bfloat16, n_meta=N_META, block=KV8_BLOCK):
    """Keys and values of the windows whose newest position is pos, oldest row
    first: rows first .. first + rows - 1 (default: all that a window can hold)
    as [B, H, rows, hs] in dtype, zeros past a row's window (msq_kv8_read)."""
    cache, (B, H, hs, S_ring, *rest) = _kv8_args(kc, ks, vc, vs, pos, n_meta, block)
    rows = S_ring - first if rows is None else rows
    if first < 0 or rows < 0 or first + rows > S_ring or dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"rows {first} .. {first + rows} of a ring of {S_ring} in {dtype}")
    s = stream_of(kc)
    k = ks.new_empty((B, H, rows, hs), dtype=dtype)
    v = torch.empty_like(k)
    if rows and B and H:
        call("msq_kv8_read", dt(k), k.data_ptr(), v.data_ptr(), *cache, B, H, hs, S_ring, *rest, first, rows, s)
    return k, v


@functools.lru_cache(maxsize=None)
def _kv8_scratch(B, H, hs, S_ring):
    """floats of the attention's workspace"""
    return L.lib().msq_relattn_decode_kv8_workspace(B, H, hs, S_ring) // 4


def relattn_decode_kv8(q, kc, ks, vc, vs, R, pos, scale, *, out=None, n_meta=N_META, block=KV8_BLOCK):
    """One decode position of the relative attention over the 8-bit cache, whose
    newest position is pos (msq_relattn_decode_kv8): q [B, H, hs] (heads hs
    apart, rows a multiple of 8 elements), R [H, S_max, hs] contiguous, both fp32
    or bf16 and 16-byte aligned. Returns out [B, H, hs] in that type, or fills out
    (any alignment); rows that are not in use (pos < -n_meta) get zeros."""
    if len(q.shape) != 3 or not (q.dtype is _BF16 or q.dtype is _F32) or R.dtype is not q.dtype:
        raise ValueError(f"q [B, H, hs] and R in fp32 or bf16, got {q.dtype} {tuple(q.shape)} and {R.dtype}")
    cache, (B, H, hs, S_ring, *rest) = _kv8_args(kc, ks, vc, vs, pos, n_meta, block)
    _kv8_beside(kc, q, R)
    S_max = R.shape[1] if len(R.shape) == 3 else 0
    if q.shape != (B, H, hs) or S_max < S_ring or R.shape != (H, S_max, hs) or not R.is_contiguous():
        raise ValueError(f"q {tuple(q.shape)} and R {tuple(R.shape)} (contiguous: {R.is_contiguous()}) for a cache of "
                         f"{B} x {H} x {S_ring} x {hs}")
    sq = q.stride()
    if out is None:
        so = (H * hs, hs, 1)
    else:
        _kv8_beside(kc, out)
        so = out.stride()
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError(f"out {out.dtype} {tuple(out.shape)} for q {q.dtype} {tuple(q.shape)}")
    if sq[2] != 1 or so[2] != 1 or (H > 1 and (sq[1] != hs or so[1] != hs)):
        raise ValueError(f"a row's heads have to lie {hs} apart, got strides {sq} and {so}")
    s = stream_of(kc)
    if out is None:
        out = q.new_empty((B, H, hs))
    if B == 0 or H == 0:
        return out
    n = _kv8_scratch(B, H, hs, S_ring)
    # a scratch of its own for every call: captured graphs and streams never share one
    ws = ks.new_empty(n) if n else None
    call("msq_relattn_decode_kv8", dt(q), out.data_ptr(), so[0] if B > 1 else H * hs, q.data_ptr(),
         sq[0] if B > 1 else H * hs, *cache, R.data_ptr(), S_max, B, H, hs, S_ring, *rest, float(scale),
         ws.data_ptr() if n else None, 4 * n, s)
    return out
