"""The decode-step operators against plain forms in 64 bits: RMSNorm with the
residual's addition (plain and Q8_0 outputs), 4-bit weights and products of a
few rows with them, the verification of drafted tokens, and a run of all of
them on a quantized model.

Tolerances count roundings: u(t) = eps(t) / 2 is the most that one rounding to t
moves a value, relative to it.
"""
import ctypes
import threading

import numpy as np
import pytest
import torch

import qllama_b200 as qb
from qllama_b200 import model as qm
from tests import llama_host as lh
from tests import model_util as mu

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U32 = 2.0 ** -24


def u(t) -> float:
    return torch.finfo(DT[t] if isinstance(t, str) else t).eps / 2


def least(t) -> float:
    """What one rounding to t moves a value at most that is below t's normal range
    (there values are smallest_normal * eps apart: 2^-24 in f16, so 2^-25)."""
    f = torch.finfo(DT[t])
    return f.smallest_normal * f.eps / 2


@pytest.fixture(scope="module")
def stream():
    return torch.cuda.Stream()


@pytest.fixture(scope="module")
def ctx(stream):
    c = qb.Context(0)
    c.set_stream(stream.cuda_stream)
    return c


@pytest.fixture(autouse=True)
def on_stream(stream):
    """Tensors are made, and the operators run, on one stream."""
    stream.wait_stream(torch.cuda.default_stream())
    with torch.cuda.stream(stream):
        yield
    stream.synchronize()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


# ------------------------------------------------------------------ RMSNorm --

def norm_f64(x, r, w, eps):
    s = x.double() + (0 if r is None else r.double())
    return s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * w.double(), s


def norm_tol(hidden):
    """Relative error of y before its last rounding: s, inverse root, two
    products (each 1 rounding, the root's division and square root 1 each, half
    the mean's), and the f32 sum of squares, whose partial sums are at most
    hidden / 64 long before they are joined in a tree of at most 16 levels."""
    return (8 + hidden / 64 + 16) * U32


@pytest.mark.parametrize("rows, hidden", [(1, 1), (1, 64), (3, 7), (2, 288), (5, 2048), (33, 4096),
                                          (2, 5473), (7, 8192), (1, 16384), (2, 40000),
                                          (700, 640)])
@pytest.mark.parametrize("dt, out, residual", [("f32", "f32", True), ("bf16", "bf16", True),
                                               ("f16", "f32", False), ("f32", "bf16", False),
                                               ("bf16", "f16", True)])
def test_norm(ctx, rows, hidden, dt, out, residual):
    g = gen(rows * 100003 + hidden)
    x = randn(g, rows, hidden).to(DT[dt])
    r = (randn(g, rows, hidden) * 3).to(DT[dt]) if residual else None
    w = (1 + 0.2 * randn(g, hidden)).to(DT[dt])
    total = torch.empty_like(x) if residual else None
    y = qm.rms_norm(ctx, x, w, 1e-5, residual=r, sum_out=total, out_dtype=out)
    ctx.synchronize()
    ref, s = norm_f64(x, r, w, 1e-5)
    assert y.dtype == DT[out] and y.shape == x.shape
    most = ref.abs() * (norm_tol(hidden) + u(out)) + least(out)
    assert ((y.double() - ref).abs() <= most).all()
    if residual:  # one rounding of the f32 sum, itself one rounding
        assert ((total.double() - s).abs() <= s.abs() * (u(dt) + 2 * U32) + least(dt)).all()


def dequantize(q, d):
    return (q.view(*q.shape[:-1], -1, 32).double() * d.double().unsqueeze(-1)).view(q.shape)


def check_q8(q, d, ref, tol):
    """Half a step, the f16 scale's rounding over up to 127 steps, y's own error."""
    step = ref.view(*ref.shape[:-1], -1, 32).abs().amax(-1, keepdim=True) / 127
    most = step * (0.5 + 0.01 + 127 * (2 ** -11 + tol)) + 127 * 2 ** -25
    err = (dequantize(q, d) - ref).view(*ref.shape[:-1], -1, 32).abs()
    assert (err <= most).all()
    scale = d.double().unsqueeze(-1)
    assert ((scale - step).abs() <= step * (2 ** -11 + tol) + 2 ** -25).all()
    assert (q.abs().int() <= 127).all()


@pytest.mark.parametrize("rows, hidden", [(1, 32), (1, 288), (24, 8192), (3, 2048), (2, 40000),
                                          (513, 96)])
@pytest.mark.parametrize("dt, residual", [("f32", True), ("bf16", True), ("f16", False)])
def test_norm_q8(ctx, rows, hidden, dt, residual):
    g = gen(rows + hidden)
    x = randn(g, rows, hidden).to(DT[dt])
    r = randn(g, rows, hidden).to(DT[dt]) if residual else None
    w = (1 + 0.2 * randn(g, hidden)).to(DT[dt])
    q, d = qm.rms_norm(ctx, x, w, 1e-6, residual=r, out_dtype="q8_0")
    ctx.synchronize()
    check_q8(q, d, norm_f64(x, r, w, 1e-6)[0], norm_tol(hidden))


@pytest.mark.parametrize("hidden", [1, 7, 64, 96, 300, 512])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_norm_many_short_rows(ctx, hidden, dt):
    """Rows that share a CTA, the last CTA not full."""
    g = gen(hidden)
    x, r = randn(g, 1201, hidden).to(DT[dt]), randn(g, 1201, hidden).to(DT[dt])
    x[5] *= 1e-3 if dt == "f16" else 1e-30
    w = 1 + 0.2 * randn(g, hidden)
    total = torch.empty_like(x)
    y = qm.rms_norm(ctx, x, w, 1e-5, residual=r, sum_out=total)
    ctx.synchronize()
    ref, s = norm_f64(x, r, w, 1e-5)
    assert ((y.double() - ref).abs() <= ref.abs() * (norm_tol(hidden) + u(dt)) + least(dt)).all()
    assert ((total.double() - s).abs() <= s.abs() * (u(dt) + 2 * U32) + least(dt)).all()
    if hidden % 32 == 0:
        q, d = qm.rms_norm(ctx, x, w, 1e-5, out_dtype="q8_0")
        ctx.synchronize()
        check_q8(q, d, norm_f64(x, None, w, 1e-5)[0], norm_tol(hidden))


@pytest.mark.parametrize("hidden", [64, 4096, 4100])
def test_norm_strides_and_in_place(ctx, hidden):
    g = gen(hidden)
    wide = randn(g, 6, hidden + 5).bfloat16()
    x = wide[:, 3:3 + hidden]  # odd offset and stride
    r = randn(g, 6, hidden).bfloat16()
    w = (1 + 0.1 * randn(g, hidden))
    ref, s = norm_f64(x, r, w, 1e-5)
    before = wide.clone()
    y = qm.rms_norm(ctx, x, w, 1e-5, residual=r, sum_out=r, out_dtype="f32")  # r += x
    ctx.synchronize()
    assert torch.equal(wide, before)
    assert ((y.double() - ref).abs() <= ref.abs() * (norm_tol(hidden) + U32) + 1e-30).all()
    assert ((r.double() - s).abs() <= s.abs() * (u("bf16") + 2 * U32)).all()
    x2 = randn(g, 6, hidden)
    ref2, _ = norm_f64(x2, None, w, 1e-5)
    qm.rms_norm(ctx, x2, w, 1e-5, out=x2)  # in place
    ctx.synchronize()
    assert ((x2.double() - ref2).abs() <= ref2.abs() * (norm_tol(hidden) + U32) + 1e-30).all()


def test_norm_extremes(ctx):
    """Squares beyond f32 in both directions, zeros, NaN and infinities."""
    g = gen(1)
    x = randn(g, 6, 256)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0
    x[3, 5] = float("nan")
    x[4, 40] = float("inf")
    w = torch.ones(256, device="cuda")
    y = qm.rms_norm(ctx, x, w, 0.0)
    q, d = qm.rms_norm(ctx, x, w, 1e-5, out_dtype="q8_0")
    ctx.synchronize()
    ref, _ = norm_f64(x, None, w, 0.0)
    for row in (0, 1, 5):
        assert ((y[row].double() - ref[row]).abs() <= ref[row].abs() * (norm_tol(256) + U32)).all()
    assert y[2].isnan().all()  # 0 / 0, as the formula has it at eps = 0
    assert y[3].isnan().all() and y[4, 40].isnan() and (y[4, :40] == 0).all()
    v = dequantize(q, d)
    assert (v[2] == 0).all() and v[3].isnan().all() and (d[2] == 0).all()
    # infinity: inf / inf in its own block, zeros elsewhere
    assert v[4, 32:64].isnan().all() and (v[4, :32] == 0).all()


def test_norm_scale_saturates(ctx):
    x = torch.ones(1, 64, device="cuda")
    w = torch.full((64,), 1e9, device="cuda")
    w[32:] = 1e-9
    q, d = qm.rms_norm(ctx, x, w, 0.0, out_dtype="q8_0")
    ctx.synchronize()
    assert d[0, 0].item() == 65504 and (q[0, :32] == 127).all()
    assert d[0, 1].item() == 0  # below f16's smallest: reads back as zeros


# ------------------------------------------------------------- 4-bit weights --

def random_weight(g, n, k, group):
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g).to(torch.uint8)
    scales = (randn(g, n, k // group) * 0.02).half()
    return codes, scales


def dense(codes, scales):
    n, k = codes.shape[0], 2 * codes.shape[1]
    q = torch.stack((codes & 15, codes >> 4), -1).view(n, scales.shape[1], -1)
    return ((q.double() - 8) * scales.double().unsqueeze(-1)).view(n, k)


@pytest.mark.parametrize("n, k, group", [(1, 32, 32), (17, 96, 32), (16, 64, 64), (50, 384, 128),
                                         (33, 2080, 32)])
def test_weight_round_trips(ctx, n, k, group):
    g = gen(n + k)
    codes, scales = random_weight(g, n, k, group)
    for c, s in ((codes, scales), (codes.cpu().numpy(), scales.cpu().numpy())):
        w = qm.Q4Weight(ctx, c, s)
        assert (w.out_features, w.in_features, w.group) == (n, k, group)
        c2, s2 = w.get()
        assert np.array_equal(c2, codes.cpu().numpy())
        assert np.array_equal(s2, scales.cpu().numpy())
        w.close()


def test_weight_from_gguf_blocks(ctx):
    """Q4_0 blocks: an f16 scale, then 16 bytes; low bits columns 0-15, high bits 16-31."""
    rng = np.random.default_rng(4)
    n, k = 21, 160
    codes = rng.integers(0, 16, (n, k), dtype=np.uint8)
    scales = rng.standard_normal((n, k // 32)).astype(np.float16)
    blocks = np.empty((n, k // 32, 18), np.uint8)
    blocks[:, :, :2] = scales.view(np.uint8).reshape(n, k // 32, 2)
    c = codes.reshape(n, k // 32, 32)
    blocks[:, :, 2:] = c[:, :, :16] | c[:, :, 16:] << 4
    for b in (blocks.tobytes(), blocks, torch.from_numpy(blocks).cuda()):
        w = qm.Q4Weight.from_gguf(ctx, b, n, k)
        c2, s2 = w.get()
        assert np.array_equal(c2, codes[:, 0::2] | codes[:, 1::2] << 4)
        assert np.array_equal(s2, scales)
        w.close()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_quantize(ctx, group, dt):
    g = gen(group)
    n, k = 37, 256
    a = (randn(g, n, k + 8) * 0.05).to(DT[dt])[:, :k]  # a row stride
    a[3, :group] = 0
    a[5, 1] = float("nan")
    a[6, 2] = float("-inf")
    w = qm.Q4Weight.from_dense(ctx, a, group)
    codes, scales = (torch.from_numpy(t).cuda() for t in w.get())
    v = a.double().view(n, -1, group)
    s = scales.double()
    assert s[5, 0].isnan() and s[6, 0].isnan() and s[3, 0] == 0
    assert (codes[3, :group // 2] == 0x88).all()
    ok = torch.ones_like(s, dtype=torch.bool)
    ok[5, 0] = ok[6, 0] = False
    big = v.gather(-1, v.abs().argmax(-1, keepdim=True)).squeeze(-1)
    assert ((s + big / 8).abs()[ok] <= (big / 8).abs()[ok] * (2 ** -11 + U32) + 2 ** -25).all()
    # codes -8 .. 7 steps: half a step, and one more where +8 would have been needed
    err = (dense(codes, scales).view(n, -1, group) - v).abs()
    top = v * torch.sign(s).unsqueeze(-1) > 7.5 * s.abs().unsqueeze(-1)
    most = s.abs().unsqueeze(-1) * torch.where(top, 1.0 + 8 * 2 ** -10, 0.5 + 8 * 2 ** -10)
    assert (err <= most + 1e-12)[ok].all()
    b = qm.Q4Weight.from_dense(ctx, a.float().cpu().numpy(), group)  # the host form
    assert np.array_equal(b.get()[0], w.get()[0])


def quantized_rows(x):
    b = x.view(x.shape[0], -1, 32)
    d = b.abs().amax(-1, keepdim=True) / 127
    return (b / d).round().to(torch.int8).view(x.shape), d.squeeze(-1).half()


def linear_tol(k):
    """Roundings on the way of a product into the f32 sum (relative to the sum
    of magnitudes): up to 32 additions inside a block on the tensor cores, which
    may cut instead of round (2 u each), two scale products, one addition for
    each block of 32, and the joins of at most 64 partial sums."""
    return (2 * 32 + 2 + k / 32 + 64) * U32


def check_linear(y, x, w, out):
    ref = x @ w.t()
    most = (x.abs() @ w.abs().t()) * linear_tol(w.shape[1]) + ref.abs() * u(out)
    assert ((y.double() - ref).abs() <= most + least(out)).all()


def rows_of(dt, x):
    """(x, x_scale, the f64 values they stand for)"""
    if dt == "q8_0":
        q, d = quantized_rows(x)
        return q, d, dequantize(q, d)
    x = x.to(DT[dt])
    return x, None, x.double()


@pytest.mark.parametrize("n, k, group", [(1, 32, 32), (15, 96, 32), (768, 288, 32), (16, 64, 64),
                                         (130, 1152, 128), (2560, 2048, 32), (257, 4160, 64),
                                         (64, 28672, 128)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16", "q8_0"])
def test_linear(ctx, n, k, group, dt):
    g = gen(n * 7 + k)
    codes, scales = random_weight(g, n, k, group)
    w, wd = qm.Q4Weight(ctx, codes, scales), dense(codes, scales)
    out = "f32" if dt == "q8_0" else dt
    x, d, xd = rows_of(dt, randn(g, 70, k))
    every = qm.linear_q4(w, x, d)
    ctx.synchronize()
    assert every.shape == (70, n) and every.dtype == DT[out]
    check_linear(every, xd, wd, out)
    for rows in (1, 2, 3, 5, 8, 9, 11, 17, 32, 33, 64):  # the same bits, however many rows
        y = qm.linear_q4(w, x[:rows], None if d is None else d[:rows])
        ctx.synchronize()
        assert torch.equal(y, every[:rows])
    w.close()


@pytest.mark.parametrize("dt, out", [("q8_0", "bf16"), ("q8_0", "f16"), ("f32", "f16"),
                                     ("bf16", "f32")])
def test_linear_strides_and_types(ctx, dt, out):
    g = gen(3)
    n, k, rows = 100, 320, 6
    codes, scales = random_weight(g, n, k, 32)
    w, wd = qm.Q4Weight(ctx, codes, scales), dense(codes, scales)
    x, d, xd = rows_of(dt, randn(g, rows, k))
    for shift in (0, 1, 3):  # misaligned rows, and an output inside a wider matrix
        wide = torch.zeros(rows, k + 5, dtype=x.dtype, device="cuda")
        wide[:, shift:shift + k] = x
        room = torch.full((rows, n + 7), 9.0, dtype=DT[out], device="cuda")
        y = qm.linear_q4(w, wide[:, shift:shift + k], d, out=room[:, shift:shift + n])
        ctx.synchronize()
        check_linear(y, xd, wd, out)
        assert (room[:, :shift] == 9).all() and (room[:, shift + n:] == 9).all()
    y3 = qm.linear_q4(w, x.view(2, 3, k), None if d is None else d.view(2, 3, -1), out_dtype=out)
    ctx.synchronize()
    assert y3.shape == (2, 3, n)
    check_linear(y3.view(rows, n), xd, wd, out)
    w.close()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_linear_keeps_rows_apart(ctx, dt):
    """NaN and infinities stay in their rows; a row's bits do not depend on its neighbours."""
    g = gen(5)
    codes, scales = random_weight(g, 96, 256, 64)
    w = qm.Q4Weight(ctx, codes, scales)
    x = randn(g, 12, 256).to(DT[dt])
    a = qm.linear_q4(w, x)
    x2 = x.clone()
    x2[3, 17] = float("nan")
    x2[7] = float("inf")
    b = qm.linear_q4(w, x2)
    ctx.synchronize()
    keep = [i for i in range(12) if i not in (3, 7)]
    assert torch.equal(a[keep], b[keep])
    assert b[3].isnan().all() and not b[7].isfinite().any()
    w.close()


def test_linear_large_and_tiny_values(ctx):
    """f32 rows over f32's range: three 16-bit parts of a value carry all of its bits."""
    g = gen(6)
    codes, scales = random_weight(g, 40, 128, 32)
    w, wd = qm.Q4Weight(ctx, codes, scales), dense(codes, scales)
    for size in (1e-20, 1.0, 1e30):
        x = randn(g, 4, 128) * size
        y = qm.linear_q4(w, x)
        ctx.synchronize()
        check_linear(y, x.double(), wd, "f32")
    w.close()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_linear_rows_near_the_types_largest(ctx, dt, group):
    """Sums of a block's products with its codes, before the scale makes them smaller, are
    beyond f32's range; the results are not."""
    g = gen(7)
    codes, scales = random_weight(g, 70, 256, group)
    scales = (scales.float() * 2.0 ** -10).half()
    w, wd = qm.Q4Weight(ctx, codes, scales), dense(codes, scales)
    for rows in (1, 9, 33):
        x = (torch.sign(randn(g, rows, 256)) * 3e38).to(DT[dt])
        y = qm.linear_q4(w, x)
        ctx.synchronize()
        assert y.isfinite().all()
        check_linear(y, x.double(), wd, dt)
    w.close()


@pytest.mark.parametrize("where", ["captured", "another context"])
def test_linear_after_new_weights_wherever_the_last_product_was(ctx, stream, where):
    """New weights, a product of them that has not run or ran on another stream, and at
    once a product on the stream that wrote them."""
    g = gen(31)
    n, k = 4096, 4096
    old, new = random_weight(g, n, k, 32), random_weight(g, n, k, 32)
    x = randn(g, 1, k).half()
    w = qm.Q4Weight(ctx, *new)
    want = qm.linear_q4(w, x)
    y, y2 = torch.empty_like(want), torch.empty_like(want)
    other, s2 = qb.Context(0), torch.cuda.Stream()
    other.set_stream(s2.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    # a context's handle of the same weight, for calls on the other stream
    view = object.__new__(qm.Q4Weight)
    view.__dict__.update(w.__dict__)
    view.ctx = other
    for _ in range(10):
        w.set(*old)
        qm.linear_q4(w, x, out=y)
        stream.synchronize()
        assert not torch.equal(y, want)
        w.set(*new)
        if where == "captured":
            stream.synchronize()
            graph.reset()
            with torch.cuda.graph(graph, stream=stream):
                qm.linear_q4(w, x, out=y2)
            w.set(*new)
        else:
            s2.wait_stream(stream)
            with torch.cuda.stream(s2):
                qm.linear_q4(view, x, out=y2)
        qm.linear_q4(w, x, out=y)
        stream.synchronize()
        s2.synchronize()
        assert torch.equal(y, want)
        if where == "captured":
            graph.replay()
            stream.synchronize()
        assert torch.equal(y2, want)
    graph.reset()
    view._h = None  # the handle is w's
    w.close()


def test_empty_calls(ctx):
    codes, scales = random_weight(gen(1), 8, 64, 32)
    w = qm.Q4Weight(ctx, codes, scales)
    assert qm.linear_q4(w, torch.empty(0, 64, device="cuda")).shape == (0, 8)
    assert qm.rms_norm(ctx, torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda"),
                       1e-5).shape == (0, 64)
    t, n = qm.verify_drafts(ctx, torch.empty(0, 3, 9, device="cuda"), None,
                            torch.empty(0, 2, dtype=torch.int32, device="cuda"),
                            torch.empty(0, 3, dtype=torch.float64, device="cuda"))
    assert t.shape == (0, 3) and n.shape == (0,)


def test_python_refusals(ctx):
    x = torch.zeros(2, 64, device="cuda")
    one = torch.ones(64, device="cuda")
    w = qm.Q4Weight(ctx, *random_weight(gen(1), 8, 64, 32))
    bad = [lambda: qm.rms_norm(ctx, x.cpu(), one, 1e-5),
           lambda: qm.rms_norm(ctx, x.double(), one, 1e-5),
           lambda: qm.rms_norm(ctx, x, one[:32], 1e-5),
           lambda: qm.rms_norm(ctx, x, one, 1e-5, residual=x.half()),
           lambda: qm.rms_norm(ctx, x, one, 1e-5, sum_out=x),
           lambda: qm.rms_norm(ctx, x.t(), one[:2], 1e-5),
           lambda: qm.rms_norm(ctx, x, one, 1e-5, out_dtype="f8"),
           lambda: qm.rms_norm(ctx, x[:, :40], one[:40], 1e-5, out_dtype="q8_0"),
           lambda: qm.linear_q4(w, x[:, :32]),
           lambda: qm.linear_q4(w, x.to(torch.int8)),
           lambda: qm.linear_q4(w, x, out=torch.empty(2, 9, device="cuda")),
           lambda: qm.linear_q4(w, x.t().contiguous().t()),
           lambda: qm.Q4Weight(ctx, torch.zeros(8, 32), torch.zeros(8, 2)),
           lambda: qm.Q4Weight(ctx, shape=(8, 48, 32)),
           lambda: qm.Q4Weight.from_gguf(ctx, b"12", 1, 32),
           lambda: w.set(torch.zeros(8, 16, dtype=torch.uint8), torch.zeros(8, 2).half()),
           lambda: qm.verify_drafts(ctx, x, None, None, None),
           lambda: qm.verify_drafts(ctx, x.view(1, 2, 64), None,
                                    torch.zeros(1, 1, dtype=torch.int32, device="cuda"), None),
           lambda: qm.verify_drafts(ctx, x.view(1, 2, 64), None,
                                    torch.zeros(1, 1, dtype=torch.int64, device="cuda"),
                                    torch.zeros(1, 2, dtype=torch.float64, device="cuda"))]
    for call in bad:
        with pytest.raises(qb.QllamaError):
            call()
    w.close()


# ---------------------------------------------------- verification of drafts --

def verify_f64(target, draft, ids, uniforms, T, n_draft, probs):
    """The definition, sequence by sequence, in 64 bits."""
    target = target.double().cpu().numpy()
    draft = None if draft is None else draft.double().cpu().numpy()
    ids = ids.cpu().numpy()
    uniforms = None if uniforms is None else uniforms.cpu().numpy()
    B, rows, V = target.shape
    tokens, accepted = np.full((B, rows), -1, np.int32), np.zeros(B, np.int32)

    def dist(row):
        if probs:
            return row
        with np.errstate(over="ignore", invalid="ignore"):
            e = np.exp((row - row.max()) / T)
        return e / e.sum()

    for b in range(B):
        n = rows - 1 if n_draft is None else int(min(max(int(n_draft[b]), 0), rows - 1))
        a, left, bad = 0, None, False
        while True:
            row = target[b, a]
            bad = bool(np.isnan(row).any() or (row == np.inf).any() or
                       (row.max() <= 0 if probs else row.max() == -np.inf))
            if bad:
                break
            if not probs and T <= 0:
                left = int(row.argmax())
                if a == n or left != ids[b, a]:
                    break
            else:
                p = dist(row)
                left = p
                if a == n:
                    break
                x = ids[b, a]
                q = np.zeros(V)
                if draft is None:
                    q[x] = 1
                else:
                    q = dist(draft[b, a])
                if not uniforms[b, a] * q[x] < p[x]:
                    left = np.maximum(p - q, 0)
                    if not left.sum() > 0:
                        left = p
                    break
            tokens[b, a] = ids[b, a]
            a += 1
        accepted[b] = a
        if bad:
            continue
        if not isinstance(left, int):
            cum = np.cumsum(left)
            left = int(np.flatnonzero((left > 0) & (cum >= uniforms[b, n] * cum[-1]))[0])
        tokens[b, a] = left
    return tokens, accepted


def check_verify(ctx, target, draft, ids, uniforms, T=1.0, n_draft=None, probs=False):
    tokens, accepted = qm.verify_drafts(ctx, target, draft, ids, uniforms, T, n_draft, probs)
    ctx.synchronize()
    t, a = verify_f64(target, draft, ids, uniforms, T, n_draft, probs)
    assert np.array_equal(accepted.cpu().numpy(), a)
    assert np.array_equal(tokens.cpu().numpy(), t)
    return t, a


def drafted(g, B, m, V, dt, near=0.7, spread=2.5):
    base = randn(g, B, m + 1, V) * spread
    draft = base[:, :m] + near * randn(g, B, m, V)
    target, draft = base.to(DT[dt]), draft.to(DT[dt])
    ids = torch.distributions.Categorical(logits=draft.float()).sample().int() if m else \
        torch.zeros(B, 0, dtype=torch.int32, device="cuda")
    un = torch.rand(B, m + 1, dtype=torch.float64, device="cuda", generator=g)
    return target, draft, ids, un


@pytest.mark.parametrize("B, m, V", [(1, 0, 1), (1, 1, 2), (3, 2, 31), (2, 4, 1000), (17, 5, 4099),
                                     (1, 4, 32000), (4, 7, 128000), (40, 3, 513), (2, 31, 777)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_verify_logits(ctx, B, m, V, dt):
    g = gen(B * 1009 + m * 31 + V)
    torch.manual_seed(V)
    target, draft, ids, un = drafted(g, B, m, V, dt)
    seen = set()
    for T in (1.0, 0.6, 0.0):
        seen |= set(check_verify(ctx, target, draft, ids, un, T)[1].tolist())
    n = torch.randint(-1, m + 2, (B,), device="cuda", generator=g).int()
    check_verify(ctx, target, draft, ids, un, 0.9, n_draft=n)
    check_verify(ctx, target, None, target[:, :m].argmax(-1).int(), un, 0.7)
    if B >= 17 and m > 2:
        assert len(seen) > 2  # several of the possible counts occur


@pytest.mark.parametrize("B, m, V", [(1, 1, 3), (5, 4, 50021), (3, 3, 700)])
def test_verify_probabilities(ctx, B, m, V):
    g = gen(V)
    torch.manual_seed(V + 1)
    target, draft, ids, un = drafted(g, B, m, V, "f32")
    keep = min(V, 50)  # a top-k filter: most entries are zero
    least = target.topk(keep, -1).values[..., -1:]
    p = torch.softmax(target.masked_fill(target < least, float("-inf")), -1)
    q = torch.softmax(draft, -1)
    t, _ = check_verify(ctx, p, q, ids, un, probs=True)
    for b in range(B):
        a = int((t[b] >= 0).sum()) - 1
        assert p[b, a, t[b, a]] > 0  # only tokens that the filter left
    check_verify(ctx, p, None, ids, un, probs=True)


def test_verify_accepts_equal_distributions(ctx):
    g = gen(8)
    torch.manual_seed(8)
    target, draft, ids, un = drafted(g, 9, 6, 5000, "f32", near=0.0)
    _, a = check_verify(ctx, target, draft, ids, un)
    assert (a == 6).all()


@pytest.mark.parametrize("V, near", [(5000, 1e-5), (128000, 1e-3), (32000, 3e-2)])
def test_verify_rejects_from_nearly_equal_distributions(ctx, V, near):
    """Little is left of a target that its draft nearly equals: the few ids that keep a
    difference, and how much, are those of the definition."""
    g = gen(V)
    torch.manual_seed(V)
    target, draft, ids, un = drafted(g, 6, 2, V, "f32", near=near)
    # a drafted id whose draft probability is the larger, and a uniform that rejects it
    p, q = torch.softmax(target.double(), -1)[:, :2], torch.softmax(draft.double(), -1)
    ids = ((q - p) / q).argmax(-1).int()
    un[:, :2] = 1 - 2.0 ** -53
    t, a = check_verify(ctx, target, draft, ids, un)
    assert (a == 0).all()


@pytest.mark.parametrize("base, T", [(30.0, 1.6e-9), (30.0, 2.65e-8), (300.0, 3.5e-8),
                                     (300.0, 4.24e-7), (30.0, 1e-6)])
def test_verify_temperatures_near_a_step_of_the_logits(ctx, base, T):
    """Logits some f32 steps below the largest, at temperatures that make their weights
    too small for 64 bits: they weigh nothing."""
    g = gen(11)
    V, B, m = 500, 24, 2
    step = 2.0 ** -19 if base < 32 else 2.0 ** -15

    def below(*shape):
        n = torch.randint(0, 14, shape, device="cuda", generator=g)
        return (base - n.double() * step).float()

    target, draft = below(B, m + 1, V), below(B, m, V)
    ids = draft.argmax(-1).int()  # (the first of the largest: mostly rejected)
    un = torch.rand(B, m + 1, dtype=torch.float64, device="cuda", generator=g)
    a = check_verify(ctx, target, draft, ids, un, T)[1]
    assert (a < m).any()


def test_verify_probabilities_below_f32(ctx):
    """A decision between probabilities that are no f32 numbers any more."""
    target = torch.zeros(2, 2, 50, device="cuda")
    draft = torch.zeros(2, 1, 50, device="cuda")
    target[:, 0, 7], draft[:, 0, 7] = -120.0, -118.0  # e^-120 and e^-118 of some 49
    ids = torch.full((2, 1), 7, dtype=torch.int32, device="cuda")
    un = torch.tensor([[0.13, 0.5], [0.14, 0.5]], dtype=torch.float64, device="cuda")
    tokens, accepted = qm.verify_drafts(ctx, target, draft, ids, un)
    ctx.synchronize()
    assert accepted.tolist() == [1, 0]  # e^-2 = 0.1353
    assert tokens[0].tolist() == [7, 24]
    # what is left of the other rows (the 49 ids' shares of e^-118 - e^-120) is below
    # f64's resolution, the definition's as well: any of the 49
    assert tokens[1, 0].item() != 7 and tokens[1, 0].item() >= 0


@pytest.mark.parametrize("depth, T", [(702.0, 1.0), (7.0, 0.01), (690.5, 1.0), (725.0, 1.0)])
def test_verify_probabilities_near_f64s_smallest(ctx, depth, T):
    """A decision between probabilities of 1e-300 to 1e-317, and a probability that is not
    0 against a uniform of 0 or a draft's probability of 0."""
    inf = float("inf")
    target = torch.zeros(5, 2, 50, device="cuda")
    draft = torch.zeros(5, 1, 50, device="cuda")
    target[:, 0, 7], draft[:, 0, 7] = -depth - 2 * T, -depth
    target[2, 0, 7] = -inf
    draft[3, 0, 7] = -inf
    ids = torch.full((5, 1), 7, dtype=torch.int32, device="cuda")
    un = torch.full((5, 2), 0.5, dtype=torch.float64, device="cuda")
    # e^-2 = 0.135; at e^-727 / 50 a step of f64's smallest numbers is 2e-6 of p
    un[:, 0] = torch.tensor([0.13, 0.14, 0.0, 0.5, 0.0])
    tokens, accepted = qm.verify_drafts(ctx, target, draft, ids, un, T)
    ctx.synchronize()
    assert accepted.tolist() == [1, 0, 0, 1, 1]
    assert tokens[:, 0].tolist()[3:] == [7, 7] and not {7, -1} & set(tokens[1:3, 0].tolist())
    assert accepted.tolist() == verify_f64(target, draft, ids, un, T, None, False)[1].tolist()
    certain, accepted = qm.verify_drafts(ctx, target, None, ids, un, T)
    ctx.synchronize()
    assert accepted.tolist() == [0, 0, 0, 0, 1]


def test_verify_masked_and_bad_rows(ctx):
    g = gen(9)
    torch.manual_seed(9)
    V, inf = 3000, float("inf")
    target, draft, ids, un = drafted(g, 6, 3, V, "f32", near=0.3)
    target[:, :, V // 2:] = -inf  # masked: probability 0
    target[0, :, :] = torch.finfo(torch.float32).min  # the type's lowest everywhere: uniform
    draft[1, 0] = -inf
    draft[1, 0, 7] = 0.0  # a certain draft
    ids[1, 0] = 7
    target[2, 3, :] = -inf  # the row behind the drafts has nothing left
    target[2, :3] = draft[2, :3]  # all accepted, so that it is reached
    ids[2] = draft[2, :3].argmax(-1).int()
    un[2, :3] = 0.0
    target[3, 0, 5] = float("nan")
    target[4, 1, 5] = inf
    un[5, 0] = 0.999999
    ids[5, 0] = V - 1  # masked in the target: rejected, and what follows is not looked at
    target[5, 1:] = float("nan")
    tokens, accepted = qm.verify_drafts(ctx, target, draft, ids, un)
    with pytest.raises(qb.QllamaError, match="non-finite"):
        ctx.synchronize()
    t, a = verify_f64(target, draft, ids, un, 1.0, None, False)
    assert np.array_equal(accepted.cpu().numpy(), a) and np.array_equal(tokens.cpu().numpy(), t)
    assert a[2] == 3 and (t[2, 3] == -1) and t[3, 0] == -1 and a[5] == 0 and t[5, 0] >= 0
    ctx.synchronize()  # the status was read and cleared


@pytest.mark.parametrize("T", [1.0, 0.0])
def test_verify_drafted_id_outside_the_vocabulary(ctx, T):
    g = gen(10)
    torch.manual_seed(10)
    target, draft, ids, un = drafted(g, 3, 2, 100, "f32")
    ids[1, 0], ids[2, 0] = 100, -5
    tokens, accepted = qm.verify_drafts(ctx, target, draft, ids, un, T)
    with pytest.raises(qb.QllamaError, match="vocabulary"):
        ctx.synchronize()
    t, a = verify_f64(target[:1], draft[:1], ids[:1], un[:1], T, None, False)
    assert np.array_equal(tokens[:1].cpu().numpy(), t)
    assert (accepted[1:] == 0).all() and (tokens[1:] == -1).all()


def test_verify_ties_go_to_the_lowest_id(ctx):
    V = 9000
    target = torch.zeros(2, 2, V, device="cuda")
    target[0, 0, [41, 40, 8999]] = 3.0
    target[1, 0, 8000] = 3.0
    target[:, 1, [5000, 77]] = 1.0
    ids = torch.tensor([[41], [8000]], dtype=torch.int32, device="cuda")
    tokens, accepted = qm.verify_drafts(ctx, target, None, ids, None, 0.0)
    ctx.synchronize()
    assert accepted.tolist() == [0, 1] and tokens.tolist() == [[40, -1], [8000, 77]]


def test_verify_strided_rows(ctx):
    g = gen(12)
    torch.manual_seed(12)
    target, draft, ids, un = drafted(g, 3, 4, 1001, "bf16")
    wide = torch.full((3, 5, 1024), float("nan"), device="cuda", dtype=torch.bfloat16)
    wide[:, :, :1001] = target
    check_verify(ctx, wide[:, :, :1001], draft, ids, un, 0.8)
    odd = torch.full((3 * 5 * 1001 + 1,), float("nan"), device="cuda", dtype=torch.bfloat16)
    odd[1:] = target.reshape(-1)
    check_verify(ctx, odd[1:].view(3, 5, 1001), draft, ids, un, 0.8)


def test_verify_edges_of_the_draw(ctx):
    """Uniforms at the ends of [0, 1): the first and the last token with any probability."""
    p = torch.tensor([0.0, 0.25, 0.0, 0.5, 0.25, 0.0], device="cuda").repeat(4, 1, 1)
    un = torch.tensor([[0.0], [0.25], [0.75], [1 - 2.0 ** -53]], dtype=torch.float64,
                      device="cuda")
    ids = torch.empty(4, 0, dtype=torch.int32, device="cuda")
    tokens, accepted = qm.verify_drafts(ctx, p, None, ids, un, probs=True)
    ctx.synchronize()
    assert tokens[:, 0].tolist() == [1, 1, 3, 4] and (accepted == 0).all()


def test_verify_without_drafts_is_the_sampler(ctx):
    g = gen(14)
    logits = randn(g, 1, 1, 32000) * 3
    ids = torch.empty(1, 0, dtype=torch.int32, device="cuda")
    for r in (0.0, 0.1, 0.5, 0.77, 0.999):
        un = torch.tensor([[r]], dtype=torch.float64, device="cuda")
        tokens, _ = qm.verify_drafts(ctx, logits, None, ids, un, 1.0)
        assert qm.sample(ctx, logits.view(-1), None, (1.0, 0, 1.0, 1.0), r) == tokens.item()


def test_verified_tokens_follow_the_target(ctx):
    """Accepted or redrawn, the first token's distribution is the target's."""
    g = gen(15)
    N, V = 40000, 6
    lt, ld = randn(g, V), randn(g, V)
    q = torch.softmax(ld.double(), 0)
    ids = torch.multinomial(q.float(), N, replacement=True, generator=g).int()[:, None]
    un = torch.rand(N, 2, dtype=torch.float64, device="cuda", generator=g)
    tokens, accepted = qm.verify_drafts(ctx, lt.repeat(N, 2, 1), ld.repeat(N, 1, 1), ids, un)
    ctx.synchronize()
    p = torch.softmax(lt.double(), 0).cpu().numpy()
    got = np.bincount(tokens[:, 0].cpu().numpy(), minlength=V) / N
    assert (np.abs(got - p) <= 6 * np.sqrt(p * (1 - p) / N)).all()
    rate = float(np.minimum(p, q.cpu().numpy()).sum())
    assert abs(accepted.double().mean().item() - rate) <= 6 * (rate * (1 - rate) / N) ** 0.5


# ------------------------------------------------------- streams and graphs --

def test_calls_in_a_graph(ctx, stream):
    """Norm, product and verification captured once and replayed on new inputs."""
    g = gen(20)
    torch.manual_seed(20)
    rows, k, V = 4, 256, 500
    w = qm.Q4Weight(ctx, *random_weight(g, V, k, 32))
    x, r = randn(g, rows, k), randn(g, rows, k)
    wt = 1 + 0.1 * randn(g, k)
    ids = torch.randint(0, V, (1, rows - 1), device="cuda", generator=g).int()
    un = torch.rand(1, rows, dtype=torch.float64, device="cuda", generator=g)
    q = torch.empty(rows, k, dtype=torch.int8, device="cuda")
    d = torch.empty(rows, k // 32, dtype=torch.float16, device="cuda")
    y = torch.empty(rows, V, device="cuda")
    total = torch.empty_like(x)
    tokens = torch.empty(1, rows, dtype=torch.int32, device="cuda")
    accepted = torch.empty(1, dtype=torch.int32, device="cuda")

    def step():
        qm.rms_norm(ctx, x, wt, 1e-5, residual=r, sum_out=total, out=q, scale=d)
        qm.linear_q4(w, q, d, out=y)
        qm.verify_drafts(ctx, y.view(1, rows, V), None, ids, un, 0.5, tokens=tokens,
                         accepted=accepted)

    graph = torch.cuda.CUDAGraph()
    stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for seed in (21, 22):
        x.copy_(randn(gen(seed), rows, k))
        for t in (y, total, tokens, accepted, q, d):
            t.zero_()
        graph.replay()
        got = [t.clone() for t in (q, d, y, total, tokens, accepted)]
        step()
        ctx.synchronize()
        for a, b in zip(got, (q, d, y, total, tokens, accepted)):
            assert torch.equal(a, b)
    w.close()


def test_two_contexts_on_two_streams(stream):
    """Two contexts' calls in flight at once do not touch each other's results."""
    g = gen(30)
    torch.manual_seed(30)
    k, V, B, m = 1024, 6000, 3, 3
    codes, scales = random_weight(g, V, k, 32)
    runs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        c = qb.Context(0)
        c.set_stream(s.cuda_stream)
        x = randn(g, B * (m + 1), k)
        target, draft, ids, un = drafted(g, B, m, V, "f32")
        stream.synchronize()
        w = qm.Q4Weight(c, codes, scales)
        c.synchronize()
        runs.append((s, c, w, x, target, draft, ids, un, torch.ones(k, device="cuda")))
    stream.synchronize()

    def go(run):
        s, c, w, x, target, draft, ids, un, one = run
        with torch.cuda.stream(s):
            q, d = qm.rms_norm(c, x, one, 1e-5, out_dtype="q8_0")
            y = qm.linear_q4(w, q, d)
            return (q, d, y) + qm.verify_drafts(c, target, draft, ids, un)

    alone = []
    for run in runs:
        alone.append(go(run))
        run[1].synchronize()
    for _ in range(20):
        both = [go(run) for run in runs]
        for run in runs:
            run[1].synchronize()
        for a, b in zip(alone, both):
            for t1, t2 in zip(a, b):
                assert torch.equal(t1, t2)
    for run in runs:
        run[2].close()


@pytest.fixture
def own():
    """A context on its own stream, as it comes."""
    c = qb.Context(0)
    yield c
    c.synchronize()
    c.close()


def busy():
    torch.cuda._sleep(2_000_000)  # about a millisecond of the current stream


def spoil(n):
    """Fills memory that was just dropped on the current stream."""
    for _ in range(4):
        torch.full((n,), 0x7f, dtype=torch.uint8, device="cuda")


def test_tensors_of_the_current_stream_on_a_context_of_its_own(ctx, own):
    """Inputs that the current stream is still writing, dropped and overwritten at once, and
    results used there, without a synchronisation."""
    g = gen(40)
    torch.manual_seed(40)
    rows, k, n = 6, 4096, 2048
    x, r, wt = randn(g, rows, k), randn(g, rows, k), 1 + 0.1 * randn(g, k)
    a = randn(g, n, k) * 0.02
    target, draft, ids, un = drafted(g, 3, 3, 5000, "f32")

    def run(c):
        out = []
        busy()
        w = qm.Q4Weight.from_dense(c, a.half() * 1, 64)
        spoil(2 * n * k)
        y = qm.linear_q4(w, x + r)
        spoil(4 * rows * k)
        out += [y * 1]
        busy()
        q, d = qm.rms_norm(c, x * 1, wt * 1, 1e-5, residual=r * 1, out_dtype="q8_0")
        spoil(4 * rows * k)
        out += [q * 1, d * 1, qm.linear_q4(w, q * 1, d * 1) * 1]
        del q, d, y
        busy()
        codes, scales = (torch.from_numpy(t).cuda() for t in w.get())
        busy()
        w.set(codes * 1, scales * 1)
        spoil(n * k // 2)
        out += [qm.linear_q4(w, x * 1) * 1]
        busy()
        out += [t * 1 for t in qm.verify_drafts(c, target * 1, draft * 1, ids * 1, un * 1)]
        spoil(4 * target.numel())
        return out

    want = run(ctx)
    torch.cuda.synchronize()
    for _ in range(3):
        got = run(own)
        assert all(torch.equal(s, t) for s, t in zip(want, got))


def test_a_context_of_its_own_in_a_captured_stream(ctx, own, stream):
    """Calls of a context on its own stream are part of a graph that torch's current
    stream captures."""
    g = gen(41)
    k, n = 512, 300
    w = qm.Q4Weight(own, *random_weight(g, n, k, 32))
    x, wt = randn(g, 3, k), 1 + 0.1 * randn(g, k)
    graph = torch.cuda.CUDAGraph()
    stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        y = qm.linear_q4(w, *qm.rms_norm(own, x, wt, 1e-5, out_dtype="q8_0"))
    for seed in (42, 43):
        x.copy_(randn(gen(seed), 3, k))
        graph.replay()
        got = y.clone()
        assert torch.equal(got, qm.linear_q4(w, *qm.rms_norm(own, x, wt, 1e-5, out_dtype="q8_0")))
    stream.synchronize()
    w.close()


def test_a_captured_context_called_from_another_stream(ctx, stream):
    """A context whose stream is being captured, while torch's current stream is not: the
    call is part of the graph, and nothing orders it with the current stream."""
    g = gen(44)
    k = 256
    x, wt, y = randn(g, 3, k), 1 + 0.1 * randn(g, k), torch.empty(3, k, device="cuda")
    want = qm.rms_norm(ctx, x, wt, 1e-5)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.synchronize()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        with torch.cuda.stream(other):
            qm.rms_norm(ctx, x, wt, 1e-5, out=y)
    y.zero_()
    graph.replay()
    stream.synchronize()
    assert torch.equal(y, want)


def test_two_threads_on_a_context_of_its_own(own):
    """Calls of one context from two threads with streams of their own: each is ordered
    with its own stream."""
    g = gen(45)
    k, n = 2048, 512
    w = qm.Q4Weight(own, *random_weight(g, n, k, 32))
    xs = [randn(g, 4, k) for _ in range(2)]
    want = [qm.linear_q4(w, x) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(100):
                torch.cuda._sleep(20_000)
                if not torch.equal(qm.linear_q4(w, xs[i] * 1), want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    w.close()


# --------------------------------------------------------- a quantized model --

def small_model(ctx, layers=2):
    cfg = dict(vocab=515, dim=128, ff=320, heads=4, kv_heads=2, layers=layers, max_pos=128,
               eps=1e-5, theta=10000.0)
    tensors = mu.c1_weights(seed=3, cfg=cfg)
    for name in tensors:  # weights of a scale at which layers matter
        if tensors[name].ndim == 2:
            tensors[name] = tensors[name] * 4
    m = qm.Llama(ctx, qm.LlamaConfig(cfg["vocab"], cfg["dim"], cfg["ff"], cfg["heads"],
                                     cfg["kv_heads"], cfg["layers"], cfg["max_pos"], cfg["eps"],
                                     cfg["theta"]))
    for name, a in tensors.items():
        m.set_tensor(name, a)
    return m, cfg, tensors


def silu(x):
    x = x.cpu().numpy()
    with np.errstate(over="ignore"):
        up = np.exp(-x.astype(np.float64)).astype(np.float32)
        down = np.exp(x.astype(np.float64)).astype(np.float32)
        y = np.where(x >= 0, x / (np.float32(1) + up), (x * down) / (np.float32(1) + down))
    return torch.from_numpy(y.astype(np.float32)).cuda()


@pytest.mark.parametrize("n", [1, 5])
def test_quantized_model_is_the_operators_in_turn(ctx, n):
    """ql_llama_forward of a quantized model, bit for bit the public calls in turn."""
    m, cfg, t = small_model(ctx)
    m.quantize(32)
    kv = m.kv_cache()
    ids = np.random.default_rng(n).integers(0, cfg["vocab"], n)
    got = m.forward_with_cache(ids, 0, kv)
    E, H, KV, hd = cfg["dim"], cfg["heads"], cfg["kv_heads"], cfg["dim"] // cfg["heads"]
    kv2 = m.kv_cache()

    def q4(*names):
        return qm.Q4Weight.from_dense(ctx, np.concatenate([t[x] for x in names]), 32)

    def norm(x, name, add):
        w = torch.from_numpy(t[name]).cuda()
        return qm.rms_norm(ctx, x, w, cfg["eps"], residual=add,
                           sum_out=x if add is not None else None, out_dtype="q8_0")

    x = torch.from_numpy(t["token_embd.weight"][ids]).cuda()
    add = None
    for layer in range(cfg["layers"]):
        p = f"blk.{layer}."
        qkv = qm.linear_q4(q4(p + "attn_q.weight", p + "attn_k.weight", p + "attn_v.weight"),
                           *norm(x, p + "attn_norm.weight", add))
        a, b, c = qkv.split([E, KV * hd, KV * hd], 1)
        att = qb.attention_forward(kv2, layer, a.reshape(1, n, H, hd).contiguous(),
                                   b.reshape(1, n, KV, hd).contiguous(),
                                   c.reshape(1, n, KV, hd).contiguous(), [0], H, KV, hd,
                                   cfg["theta"])
        add = qm.linear_q4(q4(p + "attn_output.weight"), att.view(n, E))
        gu = qm.linear_q4(q4(p + "ffn_gate.weight", p + "ffn_up.weight"),
                          *norm(x, p + "ffn_norm.weight", add))
        ctx.synchronize()
        h = silu(gu[:, :cfg["ff"]].contiguous()) * gu[:, cfg["ff"]:]
        add = qm.linear_q4(q4(p + "ffn_down.weight"), h.contiguous())
    logits = qm.linear_q4(q4("output.weight"), *norm(x, "output_norm.weight", add))
    ctx.synchronize()
    assert np.array_equal(got.view(np.uint32), logits.cpu().numpy().view(np.uint32))
    # and it is the model: the f32 weights' logits with 4-bit noise on them
    host = lh.TinyModel(t, "", E, H, KV, cfg["layers"], cfg["eps"], cfg["theta"])
    import oracle
    cache = oracle.KvCache(cfg["layers"], cfg["max_pos"], KV, hd)
    ref = host.forward(ids, 0, lh.oracle_cached_attend(host, cache))
    assert np.corrcoef(got.ravel(), np.asarray(ref).ravel())[0, 1] > 0.9
    for c in (kv, kv2, m):
        c.close()


def test_quantized_model_refusals(ctx):
    m, cfg, t = small_model(ctx, layers=1)
    with pytest.raises(qb.QllamaError, match="group"):
        m.quantize(48)
    with pytest.raises(qb.QllamaError, match="divisible"):
        m.quantize(128)  # intermediate_size 320
    kv = m.kv_cache()
    before = m.forward_with_cache([1, 2, 3], 0, kv)  # the f32 model still runs
    assert np.isfinite(before).all()
    m.quantize(64)
    with pytest.raises(qb.QllamaError, match="already"):
        m.quantize(64)
    with pytest.raises(qb.QllamaError, match="quantized"):
        m.set_tensor("output_norm.weight", t["output_norm.weight"])
    kv.clear()
    assert np.isfinite(m.forward_with_cache([1, 2, 3], 0, kv)).all()
    for c in (kv, m):
        c.close()


def test_quantized_model_takes_a_prompt_of_more_than_65535_tokens(ctx):
    """Without an attention output each row's logits are those of its token alone."""
    n, V = 65537, 32
    cfg = dict(vocab=V, dim=64, ff=96, heads=1, kv_heads=1, layers=1, max_pos=n, eps=1e-5,
               theta=10000.0)
    tensors = mu.c1_weights(seed=5, cfg=cfg)
    m = qm.Llama(ctx, qm.LlamaConfig(V, 64, 96, 1, 1, 1, n, 1e-5, 10000.0))
    for name, a in tensors.items():
        m.set_tensor(name, np.zeros_like(a) if name.endswith("attn_output.weight") else a)
    m.quantize(32)
    ids = np.arange(n) % V
    kv = m.kv_cache(dtype="f16")
    got = np.asarray(m.forward_with_cache(ids, 0, kv)).reshape(-1, V)
    for row in {0, len(got) // 2, len(got) - 1}:
        kv.clear()
        alone = np.asarray(m.forward_with_cache([ids[n - len(got) + row]], 0, kv)).reshape(V)
        assert np.array_equal(got[row].view(np.uint32), alone.view(np.uint32))
    for c in (kv, m):
        c.close()


def test_a_refused_allocation_is_not_the_next_calls_error(ctx):
    with pytest.raises(qb.QllamaError) as e:  # 2^53 bytes of codes
        qm.Q4Weight(ctx, shape=(1 << 30, 1 << 24, 32))
    assert e.value.code == qb.ERR_OOM
    codes, scales = random_weight(gen(2), 8, 64, 32)
    w = qm.Q4Weight(ctx, codes, scales)  # its launch check reads the last error
    got = w.get()
    ctx.synchronize()
    assert np.array_equal(got[0], codes.cpu().numpy())
    w.close()


def test_a_refused_workspace_or_cache_is_not_the_next_calls_error(ctx):
    """A forward whose workspace (210 GB of logits) is refused, and a cache that is, leave
    the next calls as they were."""
    n, V = 1 << 17, 400000
    m = qm.Llama(ctx, qm.LlamaConfig(V, 64, 96, 1, 1, 1, n, 1e-5, 10000.0))
    kv = m.kv_cache(dtype="f16")
    L, ids = qb.load(), (ctypes.c_int32 * n)()

    def forward(tokens):
        rc = L.ql_llama_forward(m._h, kv._h, 0, ids, tokens, kv.seq_len(), None, qb.MEM_HOST)
        return rc, L.ql_last_error().decode()

    rc, message = forward(n)
    assert rc == qb.ERR_OOM and "workspace" in message
    rc, message = forward(3)
    assert rc == qb.OK, message
    with pytest.raises(qb.QllamaError) as e:  # 2^45 bytes a layer
        qb.KvCache(ctx, 1, 1 << 30, 64, 128, "f32")
    assert e.value.code == qb.ERR_OOM
    rc, message = forward(3)
    assert rc == qb.OK, message
    for c in (kv, m):
        c.close()


@pytest.mark.parametrize("sampled", [False, True])
def test_drafted_generation_on_a_quantized_model(ctx, sampled):
    """Drafts, some right and some wrong, verified step by step with the rejected
    rows dropped from the cache: greedy tokens are those of plain generation, and
    sampled ones those of the definition on the same logits."""
    m, cfg, _ = small_model(ctx)
    m.quantize(32)
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, cfg["vocab"], 9)
    kv = m.kv_cache()
    plain = m.generate(kv, prompt, 24)
    kv.clear()
    out, drafts = [], 3
    logits = m.forward_with_cache(prompt, 0, kv)[-1]
    counts = set()
    last = int(logits.argmax())
    out.append(last)
    T = 0.9 if sampled else 0.0
    while len(out) < 20:
        # the continuation of plain generation, spoiled now and then
        ids = [(t if rng.random() < 0.7 else int(rng.integers(0, cfg["vocab"])))
               for t in plain[len(out):len(out) + drafts]]
        pos = kv.seq_len()
        assert pos == len(prompt) + len(out) - 1
        rows = m.forward_with_cache([last] + ids, pos, kv)
        target = torch.from_numpy(rows).cuda()[None]
        un = torch.from_numpy(rng.random((1, drafts + 1))).cuda()
        di = torch.tensor([ids], dtype=torch.int32, device="cuda")
        tokens, accepted = qm.verify_drafts(ctx, target, None, di, un, T)
        ctx.synchronize()
        t, a = verify_f64(target, None, di, un, T, None, False)
        assert np.array_equal(tokens.cpu().numpy(), t) and accepted.item() == a[0]
        counts.add(int(a[0]))
        new = t[0, :a[0] + 1].tolist()
        kv.truncate(0, pos + 1 + int(a[0]))
        out += new
        last = new[-1]
    if not sampled:
        assert len(counts) > 1
        # a row's sums do not depend on how many rows a call has
        assert out[:20] == plain[:20]
    for c in (kv, m):
        c.close()
