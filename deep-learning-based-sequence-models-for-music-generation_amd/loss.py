"""Drop-in for train.py's loss surface (train.py:79-138 / train_parallel.py:
83-141 + torch.nn.CrossEntropyLoss) on the HIP kernels of csrc/loss.hip.

* ``filtered_logit(input, output)`` returns Z = -log_softmax(output, dim=1) *
  W[bucket(input)] exactly like the reference (autograd supported);
* ``filtered_cross_entropy(src, logits, trg)`` fuses filtered_logit and the
  cross-entropy (mean over B*T, no ignore_index) into one pass and produces
  d(loss)/d(logits) in the same pass when gradients are needed.
No [B,T,V] weight tensor is ever materialised.

* ``token_logprobs(logits, tokens, top)``: log probability of given tokens,
  entropy and the top alternatives of rows of logits (csrc/logprobs.hip,
  autograd supported)."""
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from ._lib import ptr, call, stream, dt, stream_of, has_tangent
from .config import Grammar
from .ops import workspace

_tables = {}


def grammar_table(device, grammar: Grammar = None):
    grammar = grammar or Grammar()
    key = (str(device), grammar.disc.vocab_size, grammar.bounds)
    t = _tables.get(key)
    if t is None:
        t = grammar.table(device).contiguous()
        _tables[key] = t
    return t


def _ws(B, T, V, device):
    return workspace(L.lib().msq_filtered_workspace(B, T, V), device, "loss")


def ce_forward_backward(src, logits, trg, V, grammar=None, dlogits=None, grad_scale=None, col_lse=None, dbias=None,
                        colpart=None):
    """logits [B,T,ld] (fp32/bf16, ld >= V). Returns (loss scalar tensor,
    dlogits or None). grad_scale defaults to 1/(B*T) (gradient of the mean).
    dbias (fp32 [V], with dlogits): += column sums of dlogits (the output
    layer's bias gradient) in the same pass. colpart ([B*T/128, 2, ld] fp32,
    with dlogits): the time-axis column (max, sum exp) partials the lm_head
    GEMM epilogue produced (ops.gemm_bias_colstats); the loss then skips its
    own pass over the logits for them."""
    grammar = grammar or Grammar()
    B, T = src.shape
    ld = logits.stride(1)
    assert logits.stride(2) == 1 and logits.stride(0) == T * ld, "logits must be [B,T,ld] row-major"
    wtab = grammar_table(logits.device, grammar)
    loss = torch.empty((), device=logits.device, dtype=torch.float32)
    if col_lse is None:
        col_lse = torch.empty(B, V, device=logits.device, dtype=torch.float32)
    gs = (1.0 / (B * T)) if grad_scale is None else float(grad_scale)
    b = grammar.bounds
    if colpart is not None:
        assert dlogits is not None and colpart.shape[0] == B * T // 128
        call("msq_filtered_ce_bias_part", ptr(loss), ptr(dlogits), dlogits.stride(1), ptr(dbias), ptr(logits),
             dt(logits), ld, ptr(src), ptr(trg), ptr(wtab), b[0], b[1], b[2], b[3], B, T, V, gs, ptr(col_lse),
             ptr(colpart), T // 128, colpart.stride(1), ptr(_ws(B, T, V, logits.device)), stream())
        return loss, dlogits
    call("msq_filtered_ce_bias", ptr(loss), ptr(dlogits), dlogits.stride(1) if dlogits is not None else 0,
         ptr(dbias), ptr(logits), dt(logits), ld, ptr(src), ptr(trg), ptr(wtab), b[0], b[1], b[2], b[3], B, T, V, gs,
         ptr(col_lse), ptr(_ws(B, T, V, logits.device)), stream())
    return loss, dlogits


class _FilteredCE(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, src, trg, grammar):
        B, T, V = logits.shape
        x = logits if logits.stride(2) == 1 and logits.stride(1) % 4 == 0 and logits.stride(0) == T * logits.stride(1) \
            else _padded(logits)
        need = logits.requires_grad
        dl = torch.empty(B, T, x.stride(1), device=x.device, dtype=x.dtype)[:, :, :V] if need else None
        loss, dl = ce_forward_backward(src.contiguous(), x, trg.contiguous(), V, grammar, dl)
        ctx.save_for_backward(dl if need else None)
        return loss

    @staticmethod
    def backward(ctx, gout):
        (dl,) = ctx.saved_tensors
        return (dl * gout.to(dl.dtype)) if dl is not None else None, None, None, None


def filtered_cross_entropy(src, logits, trg, grammar: Grammar = None):
    """== CrossEntropyLoss()(filtered_logit(src, logits).reshape(-1,V), trg.view(-1))."""
    return _FilteredCE.apply(logits, src, trg, grammar)


class _FilteredLogit(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, src, grammar):
        grammar = grammar or Grammar()
        B, T, V = logits.shape
        x = logits if logits.stride(2) == 1 and logits.stride(1) % 4 == 0 and logits.stride(0) == T * logits.stride(1) \
            else _padded(logits)
        wtab = grammar_table(x.device, grammar)
        col_lse = torch.empty(B, V, device=x.device, dtype=torch.float32)
        ldz = (V + 3) // 4 * 4
        z = torch.empty(B, T, ldz, device=x.device, dtype=torch.float32)
        b = grammar.bounds
        src = src.contiguous()
        call("msq_filtered_logit", ptr(z), ldz, ptr(x), dt(x), x.stride(1), ptr(src), ptr(wtab), b[0], b[1], b[2],
             b[3], B, T, V, 0, ptr(col_lse), ptr(_ws(B, T, V, x.device)), stream())
        ctx.save_for_backward(x, src, col_lse)
        ctx.grammar = grammar
        ctx.V = V
        return z[:, :, :V]

    @staticmethod
    def backward(ctx, dz):
        x, src, col_lse = ctx.saved_tensors
        g, V = ctx.grammar, ctx.V
        B, T = src.shape
        ldz = (V + 3) // 4 * 4
        dzp = torch.zeros(B, T, ldz, device=x.device, dtype=torch.float32)
        dzp[:, :, :V] = dz
        dl = torch.empty(B, T, x.stride(1), device=x.device, dtype=x.dtype)
        b = g.bounds
        call("msq_filtered_logit_bwd", ptr(dl), dl.stride(1), ptr(dzp), ldz, ptr(x), dt(x), x.stride(1), ptr(src),
             ptr(grammar_table(x.device, g)), b[0], b[1], b[2], b[3], B, T, V, ptr(col_lse),
             ptr(_ws(B, T, V, x.device)), stream())
        return dl[:, :, :V], None, None


def _padded(t):
    B, T, V = t.shape
    ld = (V + 3) // 4 * 4
    p = torch.empty(B, T, ld, device=t.device, dtype=t.dtype)
    p[:, :, :V] = t
    return p[:, :, :V]


def filtered_logit(input, output, grammar: Grammar = None):
    """train.py:133-138 drop-in: -log_softmax(output, dim=1) * weights[bucket(input)]."""
    return _FilteredLogit.apply(output, input, grammar)


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                  # fp32 [...]
    entropy: torch.Tensor                  # fp32 [...]
    top_ids: Optional[torch.Tensor]        # int64 [..., top] (None: top = 0)
    top_logprobs: Optional[torch.Tensor]   # fp32 [..., top]


def _token_logprobs(x, tokens, top, stats):
    """the launch on rows x [rows, V]; results in the tokens' shape"""
    lp = torch.empty_like(tokens, dtype=torch.float32)
    ent = torch.empty_like(lp)
    ids = top_lp = None
    if top:
        ids = tokens.new_empty(tokens.shape + (top,))
        top_lp = torch.empty_like(ids, dtype=torch.float32)
    rows, V = x.shape
    call("msq_token_logprobs", lp.data_ptr(), ent.data_ptr(), stats.data_ptr() if stats is not None else None,
         ids.data_ptr() if top else None, top_lp.data_ptr() if top else None, x.data_ptr(), dt(x), x.stride(0),
         tokens.data_ptr(), rows, V, top, stream_of(x))
    return lp, ent, ids, top_lp


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tokens, top):
        stats = torch.empty(x.shape[0], 2, device=x.device, dtype=torch.float32)
        lp, ent, ids, top_lp = _token_logprobs(x, tokens, top, stats)
        ctx.save_for_backward(x, tokens, stats, ent, ids)
        ctx.top = top
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(ids)
        return lp, ent, ids, top_lp

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, _, g_top):
        x, tokens, stats, ent, ids = ctx.saved_tensors
        if g_lp is None and g_ent is None and g_top is None:
            return None, None, None
        if has_tangent(*(t for t in (g_lp, g_ent, g_top) if t is not None)):
            raise NotImplementedError("the gradient of token_logprobs has no forward-mode derivative")
        rows, V = x.shape
        # rows of the gradient as far apart as those of x where that only pads
        # them: both then meet the same 16-byte boundaries
        ld = x.stride(0) if V <= x.stride(0) < V + 64 else V
        dx = torch.empty(rows, ld, device=x.device, dtype=x.dtype)[:, :V]
        g = [None if t is None else t.to(torch.float32).contiguous() for t in (g_lp, g_ent, g_top)]
        call("msq_token_logprobs_bwd", ptr(dx), ld, ptr(g[0]), ptr(g[1]), ptr(g[2]), ptr(stats), ptr(ent), ptr(ids),
             ctx.top, ptr(x), dt(x), x.stride(0), ptr(tokens), rows, V, stream_of(x))
        return dx, None, None


def token_logprobs(logits, tokens, top=0):
    """Of every row of logits [..., V] (fp32 / bf16; e.g. the model's logits or
    filtered_logit's Z): the log probability of its token (int64 [...]; outside
    [0, V), e.g. -100: 0 and no gradient), the entropy, and the ids and log
    probabilities of the ``top`` <= 32 largest logits (equal ones by index).
    logprob, entropy and top_logprobs are differentiable in logits (backward once;
    forward-mode tangents are refused). A row of nothing but -inf gives log
    probability -inf, entropy 0 and no gradient; NaN or +inf makes its row NaN.
    Both passes can be captured into a graph; as with every torch operator, only
    while no eager graph of the same leaves is alive."""
    V = logits.shape[-1] if logits.dim() else 0
    if logits.dtype not in (torch.float32, torch.bfloat16) or V == 0:
        raise ValueError(f"logits [..., V] in fp32 or bf16, got {logits.dtype} {tuple(logits.shape)}")
    if tokens.dtype != torch.int64 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"int64 tokens {list(logits.shape[:-1])}, got {tokens.dtype} {tuple(tokens.shape)}")
    if not 0 <= top <= min(32, V):
        raise ValueError(f"{top} alternatives of {V} (at most 32)")
    if tokens.get_device() != logits.get_device():
        raise ValueError(f"logits on {logits.device}, tokens on {tokens.device}")
    if has_tangent(logits):  # refused here: without requires_grad no autograd function would see it
        raise NotImplementedError("token_logprobs has no forward-mode derivative")
    stream_of(logits)  # refuses the CPU and another device than the current one
    if tokens.numel() == 0:  # no rows: empty results, on the graph of logits
        z = logits.sum(-1).float()
        t = logits[..., :top].float()
        return TokenLogprobs(z, z.clone(), torch.empty(t.shape, device=t.device, dtype=torch.int64) if top else None,
                             t if top else None)
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if x.stride(1) != 1:
        x = x.contiguous()
    tokens = tokens.contiguous()
    if x.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(x, tokens, top))
    return TokenLogprobs(*_token_logprobs(x, tokens, top, None))
