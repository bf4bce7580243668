"""The 8-bit decode cache on the GPU (msq_kv8_write / _read, msq_relattn_decode_kv8)
against oracle/kv8.py (64 bits, position by position).

Codes and scales are compared exactly: the kernel's fp32 steps before a code is
rounded are products with powers of two. (fp32 inputs below 2^-126 * 448 / 2
times a scale of 2^126 stay exact too.)

Attention, fp32 accumulation of n keys and head size hs: a score is off by at
most (hs + 8) 2^-24 of scale * sum_d |q_d| (|k_d| + |R_d|) (hs products and
additions, the scales, the change to base 2), the weights then by that and a few
2^-23 for the exponential, and the output by twice the weights' relative error
times max |v| (numerator and denominator), plus (n + 8) 2^-24 max |v| of
summation; a bf16 output by another 2^-8 of its value."""
import numpy as np
import pytest
import torch

from midiseq import attention as A
from oracle import kv8 as okv

pytestmark = pytest.mark.gpu
dev = "cuda"


def rng(seed):
    return np.random.default_rng(seed)


def rows(g, shape, dtype, spread=1.0):
    """random rows of uneven size, rounded to dtype; (tensor on the GPU, 64-bit values)"""
    x = g.standard_normal(shape) * np.exp(spread * g.standard_normal(shape[:-1] + (1,)))
    t = torch.from_numpy(x).to(dtype)
    return t.to(dev), t.double().numpy()


class Pair:
    """A cache on the GPU and its oracle, filled with garbage where nothing was written."""

    def __init__(self, B, H, hs, ctx, n_meta, block, seed=0):
        self.B, self.H, self.hs, self.S, self.n_meta, self.block = B, H, hs, ctx + n_meta, n_meta, block
        self.c = A.kv8_cache(B, H, self.S, hs, dev, block)
        g = torch.Generator().manual_seed(seed)
        for t in (self.c[0], self.c[2]):  # any code, NaN among them
            t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
        for t in (self.c[1], self.c[3]):
            t.fill_(float("nan"))
        self.garbage = [t.view(torch.uint8).cpu().numpy().copy() for t in (self.c[0], self.c[2])]
        self.o = [[okv.Ring(H, self.S, hs, n_meta, block) for _ in range(2)] for _ in range(B)]

    def write(self, k, v, pos):
        p = torch.tensor(pos if isinstance(pos, list) else [pos], device=dev)
        A.kv8_write(*self.c, k[0], v[0], p, n_meta=self.n_meta, block=self.block)
        for b in range(self.B):
            q = pos[b] if isinstance(pos, list) else pos
            self.o[b][0].write(k[1][b], q)
            self.o[b][1].write(v[1][b], q)

    def check(self):
        for i in range(2):
            code, scale = self.c[2 * i].view(torch.uint8).cpu().numpy(), self.c[2 * i + 1].cpu().numpy()
            for b in range(self.B):
                r = self.o[b][i]
                w = sorted(r.window())
                np.testing.assert_array_equal(okv.e4m3_value(code[b][:, w]), r.val[:, w])
                rest = [s for s in range(self.S) if s not in w]
                np.testing.assert_array_equal(code[b][:, rest], self.garbage[i][b][:, rest])  # left as they were
                blocks = sorted({s // self.block for s in w})
                np.testing.assert_array_equal(scale[b][:, blocks], r.scale[:, blocks])
                assert np.isnan(scale[b][:, [g for g in range(scale.shape[2]) if g not in blocks]]).all()


SHAPES = [  # B, H, hs, ctx, n_meta, block
    (2, 3, 16, 24, 6, 16), (1, 1, 8, 1, 0, 16), (2, 2, 128, 130, 6, 64), (1, 2, 24, 50, 20, 16), (3, 1, 120, 33, 6, 32),
    (1, 2, 64, 300, 0, 128), (2, 1, 96, 16, 16, 16), (1, 1, 128, 259, 6, 128)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_write_runs(shape, dtype):
    """A prompt, single tokens and chunks, round the ring more than once; T > ctx at the end."""
    B, H, hs, ctx, n_meta, block = shape
    g = rng(sum(shape))
    p = Pair(*shape)
    at = -n_meta
    for T in [n_meta + min(ctx, 9), 1, 1, 5, 1] + [max(1, ctx // 3)] * 4 + [1, ctx, 1, 2 * ctx + 3, 1]:
        p.write(rows(g, (B, T, H, hs), dtype), rows(g, (B, T, H, hs), dtype), at)
        at += T
        p.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_write_ragged(dtype):
    """Rows at positions of their own, some not in use, some still inside the metadata."""
    g, shape = rng(5), (6, 2, 32, 40, 6, 16)
    p = Pair(*shape)
    at = [-6, -7, -6, -1000, -6, -6]
    p.write(rows(g, (6, 10, 2, 32), dtype), rows(g, (6, 10, 2, 32), dtype), at)
    p.check()
    at = [4, -7, -9, -6, 4, 4]
    for T in (3, 1, 47, 1):
        p.write(rows(g, (6, T, 2, 32), dtype), rows(g, (6, T, 2, 32), dtype), at)
        p.check()
        at = [q + T if q >= -6 else q for q in at]


def test_write_values():
    """Zeros, subnormals, the type's extremes, infinities (they saturate) and NaN; one block a head."""
    p = Pair(1, 1, 8, 16, 0, 16)
    big, tiny = 3.4028234663852886e38, 1e-45
    table = [[0.0] * 8, [tiny, -tiny, 1e-40, 0, 0, 0, 0, -0.0], [1.0, 448, -448, 449, 1e-3, 0, 0, 0],
             [np.inf, -np.inf, np.nan, 1.0, 0, 0, 0, 0], [np.inf] * 8, [np.nan] * 8, [big, -big, 1.0, 0, 0, 0, 0, 0]]
    for i, row in enumerate(table):
        t = torch.tensor(row, dtype=torch.float32).view(1, 1, 1, 8)
        p.write((t.to(dev), t.double().numpy()), (-t.to(dev), -t.double().numpy()), i)
        p.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_largest_values(dtype):
    """Finite values next to 2^128 come back finite, within 2^-4, and stay so when their block is written again
    (256 at the scale 2^120 would be an infinity, and then saturate at whatever scale the others ask for)."""
    p = Pair(1, 1, 8, 16, 0, 16)
    big = torch.finfo(dtype).max
    row = torch.tensor([big, -big, 1.9375 * 2.0 ** 127, -1.875 * 2.0 ** 127, 1.75 * 2.0 ** 127, -2.0 ** 127, 1.0, 0.0])
    quiet = torch.tensor([1.0, -2.0, 3e-3, 0, 0, 0, 0, 0])
    wild = torch.tensor([float("inf"), float("-inf"), float("nan"), big, 1.0, 0, 0, 0])
    for i, r in enumerate([row, quiet, quiet, wild, quiet]):
        t = r.to(dtype).view(1, 1, 1, 8)
        p.write((t.to(dev), t.double().numpy()), (-t.to(dev), -t.double().numpy()), i)
        p.check()
        for out in (torch.float32, torch.bfloat16):
            k, v = A.kv8_read(*p.c, torch.tensor([i], device=dev), n_meta=0, block=16, dtype=out, rows=1)
            want = row.to(dtype).double()
            for got in (k.cpu().double().view(8), -v.cpu().double().view(8)):
                assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** 110).all(), got


def test_scale_falls_again():
    """A scale follows the block's contents, down as well as up, and the old codes with it."""
    g, p = rng(3), Pair(1, 2, 16, 16, 0, 16)
    for i in range(16):
        p.write(rows(g, (1, 1, 2, 16), torch.float32), rows(g, (1, 1, 2, 16), torch.float32), i)
    quiet = p.c[1].clone()
    loud = torch.full((1, 1, 2, 16), 3e6)
    p.write((loud.to(dev), loud.double().numpy()), (loud.to(dev), loud.double().numpy()), 16)
    p.check()
    assert (p.c[1] > 1000 * quiet).all()
    p.write(rows(g, (1, 1, 2, 16), torch.float32), rows(g, (1, 1, 2, 16), torch.float32), 17)
    assert (p.c[1] > 1000 * quiet).all()
    p.write(rows(g, (1, 1, 2, 16), torch.float32), rows(g, (1, 1, 2, 16), torch.float32), 32)  # over the loud row
    p.check()
    assert (p.c[1] < 100 * quiet).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_write_strides(dtype):
    """Views of a packed projection, of a transposed batch, and rows that are not 16-byte aligned."""
    g, (B, T, H, hs) = rng(9), (3, 7, 2, 24)
    for make in (lambda t: t, lambda t: torch.stack([t, t, t], 2)[:, :, 1],
                 lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: torch.nn.functional.pad(t.reshape(B, T, H * hs), (3, 2))[..., 3:3 + H * hs].view(B, T, H, hs)):
        p = Pair(B, H, hs, 40, 6, 16)
        k, v = rows(g, (B, T, H, hs), dtype), rows(g, (B, T, H, hs), dtype)
        p.write((make(k[0]), k[1]), (make(v[0]), v[1]), -6)
        p.check()
    k = torch.zeros(B, 0, H, hs, device=dev, dtype=dtype)
    before = [t.clone() for t in p.c]
    A.kv8_write(*p.c, k, k, torch.tensor([1], device=dev), block=16)  # no rows: nothing happens
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, p.c))


def test_write_padded_prompts():
    """A batch of prompts padded to one length: the padding's rows lie behind each row's newest
    position once the first token is written at the prompt's own end (positions taken back), and a
    scale that they had raised falls again."""
    g, p = rng(12), Pair(4, 2, 32, 64, 6, 16)
    k, v = rows(g, (4, 46, 2, 32), torch.bfloat16), rows(g, (4, 46, 2, 32), torch.bfloat16)
    for x in (k, v):
        x[0][:, 30:] *= 1024
        x[1][:, 30:] *= 1024
    p.write(k, v, -6)
    p.check()
    at = [40, 33, 24, 9]  # prompts of 46, 39, 30 and 15 rows
    for i in range(20):
        p.garbage = [t.view(torch.uint8).cpu().numpy().copy() for t in (p.c[0], p.c[2])]
        scales = [t.clone() for t in (p.c[1], p.c[3])]
        p.write(rows(g, (4, 1, 2, 32), torch.bfloat16), rows(g, (4, 1, 2, 32), torch.bfloat16), at)
        for j in range(2):
            code = p.c[2 * j].view(torch.uint8).cpu().numpy()
            for b in range(4):
                r, w = p.o[b][j], sorted(p.o[b][j].window())
                np.testing.assert_array_equal(okv.e4m3_value(code[b][:, w]), r.val[:, w])
                rest = [s for s in range(p.S) if s not in w]
                np.testing.assert_array_equal(code[b][:, rest], p.garbage[j][b][:, rest])
                np.testing.assert_array_equal(p.c[2 * j + 1][b].cpu().numpy(), np.where(
                    np.arange(5) == r.slot(at[b]) // 16, r.scale, scales[j][b].cpu().numpy()))
        at = [q + 1 for q in at]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_read(shape, dtype):
    B, H, hs, ctx, n_meta, block = shape
    g, p = rng(sum(shape)), Pair(*shape)
    T = n_meta + ctx // 2 + 1
    k, v = rows(g, (B, T, H, hs), torch.float32), rows(g, (B, T, H, hs), torch.float32)
    at = [-n_meta if b != 1 else -n_meta - 1 for b in range(B)]
    p.write(k, v, at)
    for last in (T - n_meta - 1, None):
        if last is None:  # round the ring
            T2 = ctx
            p.write(rows(g, (B, T2, H, hs), torch.float32), rows(g, (B, T2, H, hs), torch.float32),
                    [T - n_meta if b != 1 else -n_meta - 1 for b in range(B)])
            last = T - n_meta + T2 - 1
        pos = [last if b != 1 else -n_meta - 1 for b in range(B)]
        S = p.S
        for first, n in {(0, S), (0, 1), (S // 2, S - S // 2), (S - 1, 1)}:
            got = A.kv8_read(*p.c, torch.tensor(pos, device=dev), first=first, rows=n, dtype=dtype, n_meta=n_meta,
                             block=block)
            for i in range(2):
                want = np.zeros((B, H, S, hs))
                for b in range(B):
                    r = p.o[b][i].rows(pos[b])
                    want[b, :, :r.shape[1]] = r
                want = torch.from_numpy(want[:, :, first:first + n]).to(dtype)
                assert torch.equal(got[i].cpu(), want)
    assert A.kv8_read(*p.c, torch.tensor(pos, device=dev), rows=0, n_meta=n_meta, block=block)[0].shape == (B, H, 0, hs)


def filled(shape, pos, dtype, seed=1, spread=0.5):
    """A cache whose rows end at positions pos (written at once, the ring's last rows), q and R"""
    B, H, hs, ctx, n_meta, block = shape
    g, p = rng(seed), Pair(*shape)
    for b in range(B):  # one row of the batch at a time: the others are not in use meanwhile
        T = pos[b] + n_meta + 1
        if T <= 0:
            continue
        k, v = rows(g, (1, T, H, hs), dtype, spread), rows(g, (1, T, H, hs), dtype, spread)
        one = [t[b:b + 1] for t in p.c]
        A.kv8_write(*one, k[0], v[0], torch.tensor([-n_meta], device=dev), n_meta=n_meta, block=block)
        p.o[b][0].write(k[1][0], -n_meta)
        p.o[b][1].write(v[1][0], -n_meta)
    q, R = rows(g, (B, H, hs), dtype, 0.2), rows(g, (H, ctx + n_meta + 3, hs), dtype, 0.2)
    return p, q, R


def check_attend(p, q, R, pos, got, scale, dtype):
    want, tol = expect(p, q, R, pos, scale, dtype)
    err = np.abs(got.double().cpu().numpy() - want)
    off = float((err - tol).max())
    assert off <= 0, (off, float(err.max()))


def expect(p, q, R, pos, scale, dtype):
    want, tol = np.zeros((p.B, p.H, p.hs)), np.zeros((p.B, p.H, p.hs))
    for b in range(p.B):
        k, v = p.o[b][0].rows(pos[b]), p.o[b][1].rows(pos[b])
        n = k.shape[1]
        want[b] = okv.attend(q[1][b], k, v, R[1], scale)
        if n:
            big = np.abs(v).max((1, 2))[:, None]
            mag = (np.abs(q[1][b])[:, None] * (np.abs(k) + np.abs(R[1][:, :n]))).sum(-1).max(-1)[:, None] * scale
            w = (p.hs + 8) * 2.0 ** -24 * mag + 4 * 2.0 ** -23
            tol[b] = 2 * w * big + (n + 8) * 2.0 ** -24 * big
            if dtype == torch.bfloat16:
                tol[b] += 2.0 ** -8 * np.abs(want[b])
    return want, tol


ATTEND = [  # shape, positions
    ((2, 3, 16, 24, 6, 16), [40, 3]), ((1, 1, 8, 1, 0, 16), [0]), ((3, 2, 128, 130, 6, 64), [129, 130, 131]),
    ((4, 2, 24, 50, 20, 16), [-1, -20, -21, 77]), ((3, 1, 120, 33, 0, 32), [-1, 0, 32]),
    ((1, 2, 64, 1000, 6, 128), [2500]), ((2, 4, 80, 517, 6, 32), [400, 516]), ((7, 1, 32, 70, 6, 16), [69, 70, 139, 0, 1, 5, 68]),
    ((1, 1, 128, 5000, 6, 64), [9999]), ((2, 1, 8, 3000, 2, 16), [10, 2999]), ((40, 8, 128, 64, 6, 64), [63 + b for b in range(40)])]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,pos", ATTEND)
def test_attend(shape, pos, dtype):
    """Windows of no, one and many keys, growing, full and wrapped; slots behind the window hold
    garbage (NaN codes and scales among it)."""
    p, q, R = filled(shape, pos, dtype)
    scale = (shape[1] * shape[2]) ** -0.5
    got = A.relattn_decode_kv8(q[0], *p.c, R[0], torch.tensor(pos, device=dev), scale, n_meta=shape[4], block=shape[5])
    check_attend(p, q, R, pos, got, scale, dtype)
    for b, x in enumerate(pos):
        if x < -shape[4]:
            assert (got[b] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,pos", [((5, 3, 64, 90, 6, 16), 50), ((5, 3, 64, 90, 6, 16), 1000), ((9, 2, 128, 300, 6, 64), 450),
                                       ((3, 2, 40, 33, 0, 32), 32), ((17, 8, 128, 2048, 6, 64), 3001), ((2, 2, 16, 8, 6, 16), -7)])
def test_attend_one_position(shape, pos, dtype):
    """All rows at one position (pos of one element), strided q and out."""
    B, H, hs = shape[:3]
    p, q, R = filled(shape, [pos] * B, dtype, seed=2)
    wide = torch.full((B, 3 * H * hs + 8), 7.0, device=dev, dtype=dtype)
    wide[:, H * hs:2 * H * hs] = q[0].view(B, -1)
    out = torch.full((B, H * hs + 24), 5.0, device=dev, dtype=dtype)
    got = A.relattn_decode_kv8(wide[:, H * hs:2 * H * hs].view(B, H, hs), *p.c, R[0], torch.tensor([pos], device=dev),
                               0.25, out=out[:, 8:8 + H * hs].view(B, H, hs), n_meta=shape[4], block=shape[5])
    check_attend(p, q, R, [pos] * B, got, 0.25, dtype)
    assert (out[:, :8] == 5).all() and (out[:, 8 + H * hs:] == 5).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hs", [16, 32, 64, 128])
def test_cache_on_8_bytes(hs, dtype):
    """A cache that is 8- but not 16-byte aligned takes half the codes a lane."""
    shape, pos = (2, 3, hs, 200, 6, 64), [150, 333]
    p, q, R = filled(shape, pos, dtype)
    c = [t.clone() for t in p.c]
    for i in (0, 2):
        raw = torch.zeros(c[i].numel() + 8, device=dev, dtype=torch.uint8)
        raw[8:] = c[i].view(torch.uint8).flatten()
        c[i] = raw[8:].view(torch.float8_e4m3fn).view(c[i].shape)
        assert c[i].data_ptr() % 16 == 8
    check_attend(p, q, R, pos, A.relattn_decode_kv8(q[0], *c, R[0], torch.tensor(pos, device=dev), 0.1), 0.1, dtype)
    k, v = rows(rng(3), (2, 2, 3, hs), dtype), rows(rng(4), (2, 2, 3, hs), dtype)
    at = torch.tensor([q + 1 for q in pos], device=dev)
    A.kv8_write(*c, k[0], v[0], at)
    A.kv8_write(*p.c, k[0], v[0], at)
    for a, b in zip(c, p.c):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for a, b in zip(A.kv8_read(*c, at + 1), A.kv8_read(*p.c, at + 1)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attend_large_scores(dtype):
    """Scores of hundreds: the running maximum carries them; one key takes all."""
    shape, pos = (2, 2, 128, 700, 6, 64), [699, 1300]
    p, q, R = filled(shape, pos, dtype, spread=2.0)
    got = A.relattn_decode_kv8(q[0], *p.c, R[0], torch.tensor(pos, device=dev), 8.0)
    assert torch.isfinite(got).all()
    # beyond what the tolerance of one score leaves of the weights, rows are dominated by one key
    want, tol = expect(p, q, R, pos, 8.0, dtype)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all()


def test_attend_nan_stays_in_its_row():
    shape, pos = (3, 2, 32, 40, 6, 16), [39, 39, 39]
    p, q, R = filled(shape, pos, torch.float32)
    p.c[0].view(torch.uint8)[1, 0, 7, 3] = 0x7f
    got = A.relattn_decode_kv8(q[0], *p.c, R[0], torch.tensor(pos, device=dev), 0.2, block=16)
    assert torch.isnan(got[1, 0]).all() and torch.isfinite(got[[0, 2]]).all() and torch.isfinite(got[1, 1]).all()


def test_steps_in_a_graph_and_on_a_stream():
    """write + attend captured once with the position on the device, replayed over a wrapping ring
    with eager work between the replays; every step equals the eager calls on another cache. Two
    graphs of different sizes replayed in turn keep apart. The eager side runs on another stream."""
    scale, side = 0.2, torch.cuda.Stream()
    runs = []
    for shape in ((2, 4, 64, 40, 6, 16), (3, 2, 128, 600, 6, 64)):
        B, H, hs, ctx, n_meta, block = shape
        g = rng(ctx)
        p, q, R = filled(shape, [ctx - 3] * B, torch.bfloat16)
        twin = [t.clone() for t in p.c]
        kv = torch.zeros(B, 1, 2, H, hs, device=dev, dtype=torch.bfloat16)
        qb, pos = q[0].clone(), torch.tensor([ctx - 2], device=dev)

        def step(c, kv=kv, qb=qb, pos=pos, R=R, block=block):
            A.kv8_write(*c, kv[:, :, 0], kv[:, :, 1], pos, block=block)
            return A.relattn_decode_kv8(qb, *c, R[0], pos, scale, block=block)

        torch.cuda.synchronize()
        keep = [t.clone() for t in p.c]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(p.c)
        for t, x in zip(p.c, keep):
            assert torch.equal(t.view(torch.uint8), x.view(torch.uint8))  # capturing ran nothing
        runs.append((graph, out, p.c, twin, kv, qb, pos, step, g))
    for i in range(8):
        for graph, out, c, twin, kv, qb, pos, step, g in runs:
            kv.copy_(torch.from_numpy(g.standard_normal(kv.shape)))
            qb.copy_(torch.from_numpy(g.standard_normal(qb.shape)))
            graph.replay()
            got = out.clone()
            torch.cuda.synchronize()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                want = step(twin)
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(got, want), i
            for a, b in zip(c, twin):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            pos += 1


def test_same_inputs_same_bits():
    shape, pos = (4, 4, 128, 2000, 6, 64), [1999, 900, 4000, 5]
    p, q, R = filled(shape, pos, torch.bfloat16)
    a, b = (A.relattn_decode_kv8(q[0], *p.c, R[0], torch.tensor(pos, device=dev), 0.1) for _ in range(2))
    assert torch.equal(a, b)


def test_long_ring():
    """Slots and rows of the batch whose offsets pass 32 bits (17.5 M slots x 128 = 2.2 G codes a
    head): the last token's write and read, and attention with q = 0 (the mean of the values)."""
    ctx, hs = 17_500_000, 128
    c = A.kv8_cache(2, 1, ctx + 6, hs, dev)
    g = torch.Generator(dev).manual_seed(4)
    c[2].view(torch.uint8).random_(0, 100, generator=g)  # e4m3 codes of 0 .. 14
    k = torch.randn(2, 1, 1, hs, device=dev, generator=g)
    pos = torch.tensor([3, 2 * ctx - 1], device=dev)  # row 1: the ring's last slot
    A.kv8_write(*c, k, k, pos)
    for b, last in enumerate((3, 2 * ctx - 1)):
        at = 6 + last % ctx
        rk, rv = A.kv8_read(*[t[b:b + 1] for t in c], pos[b:b + 1], first=9 if b == 0 else ctx + 5, rows=1,
                            dtype=torch.float32)
        blk = at // 64
        for t, s, r in ((c[0], c[1], rk), (c[2], c[3], rv)):
            assert torch.equal(r[0, 0, 0], t[b, 0, at].float() * s[b, 0, blk])
        assert (rk[0, 0, 0] - k[b, 0, 0]).abs().max() <= 2 ** -4 * k[b].abs().max()
    q, R = torch.zeros(2, 1, hs, device=dev), torch.zeros(1, ctx + 6, hs, device=dev)
    got = A.relattn_decode_kv8(q, *c, R, pos, 1.0)
    total = torch.zeros(hs, device=dev, dtype=torch.float64)
    for a in range(0, ctx + 6, 1 << 20):
        e = min(ctx + 6, a + (1 << 20))
        s = c[3][1, 0].repeat_interleave(64)[a:e, None].double()
        total += (c[2][1, 0, a:e].double() * s).sum(0)
    # fp32 sums of ctx values >= 0 in runs of at most 64 Ki: 2^16 roundings of 2^-24
    assert torch.allclose(got[1, 0].double(), total / (ctx + 6), rtol=2 ** -8, atol=0)
    rv = A.kv8_read(*[t[:1] for t in c], pos[:1], rows=10, dtype=torch.float32)[1]
    assert torch.allclose(got[0, 0], rv[0, 0].mean(0), rtol=1e-5, atol=1e-6)
