"""The operators around the paged cache against plain forms in 64 bits: the Q4_0 storage,
appending and reading the rows of several sequences, attention over a Q4_0 cache, attention
over selected blocks, and a run of them together.

Tolerances count roundings: u(t) = eps(t) / 2 is the most that one rounding to t moves a
value, relative to it.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import qllama_b200 as qb
from qllama_b200 import model as qm

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TILE = 64
THETA = 10000.0


def u(t) -> float:
    return torch.finfo(DT[t] if isinstance(t, str) else t).eps / 2


@pytest.fixture(scope="module")
def stream():
    return torch.cuda.Stream()


@pytest.fixture(scope="module")
def ctx(stream):
    c = qb.Context(0)
    c.set_stream(stream.cuda_stream)
    return c


@pytest.fixture(autouse=True)
def on_stream(stream, ctx):
    """Tensors are made, and the operators run, on one stream; no kernel raised its status."""
    stream.wait_stream(torch.cuda.default_stream())
    with torch.cuda.stream(stream):
        yield
    ctx.synchronize()


def normal(seed, *shape, scale=1.0, dtype="f32"):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(DT[dtype])


# ------------------------------------------------------------------ the definitions --

def q4_plain(x):
    """f32 rows [..., hd] -> the values (f64) that a Q4_0 cache holds for them."""
    b = x.detach().float().cpu().numpy().astype(np.float64)
    shape = b.shape
    b = b.reshape(-1, 32)
    at = np.abs(np.where(np.isfinite(b), b, np.inf)).argmax(1)  # the first of equals
    m = np.take_along_axis(b, at[:, None], 1)[:, 0]
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        d = (m / -8).astype(np.float32).astype(np.float16).astype(np.float64)
        bad = ~np.isfinite(b).all(1) | ~np.isfinite(d)
        code = np.where(d[:, None] != 0, np.rint(b / d[:, None]) + 8, 8)
        code = np.clip(np.nan_to_num(code, nan=8), 0, 15)
        y = (code - 8) * d[:, None]
    y[bad] = np.nan
    return torch.from_numpy(y.reshape(shape)).cuda()


def q8_plain(x):
    """The append's Q8_0 rule, in f32 as it is defined (d = amax * (1 / 127), round(x * (1 / d)))."""
    b = x.detach().float().cpu().numpy().reshape(-1, 32)
    d = (np.abs(b).max(1, keepdims=True) * (np.float32(1) / np.float32(127))).astype(np.float32)
    inv = np.where(d != 0, np.float32(1) / np.where(d != 0, d, 1), 0).astype(np.float32)
    r = (b * inv).astype(np.float32).astype(np.float64)
    code = np.trunc(r + np.copysign(0.5, r))
    y = code * d.astype(np.float16).astype(np.float64)
    return torch.from_numpy(y.reshape(x.shape)).cuda()


def stored(x, cache):
    """f32 rows as the values (f64) that a cache of that type holds."""
    if cache == "q4_0":
        return q4_plain(x)
    return q8_plain(x) if cache == "q8_0" else x.to(DT[cache]).double()


def rotated(x, places, theta=THETA):
    """Rows [tokens, heads, hd] turned in f64 by libm's angles, rounded once to f32."""
    hd = x.shape[-1]
    freq = [math.pow(theta, -2.0 * p / hd) for p in range(hd // 2)]
    cs = np.array([[(math.cos(float(t) * f), math.sin(float(t) * f)) for f in freq]
                   for t in places]).reshape(len(places), 1, hd // 2, 2)
    z = x.double().cpu().numpy().reshape(*x.shape[:-1], hd // 2, 2)
    a, b, c, s = z[..., 0], z[..., 1], cs[..., 0], cs[..., 1]
    y = np.stack((a * c - b * s, a * s + b * c), -1).reshape(x.shape)
    return torch.from_numpy(y.astype(np.float32)).cuda()


def attention(q, k, v, start, keep=None):
    """(softmax attention [n, hq, hd] in f64 of q [n, hq, hd] over k, v [L, hkv, hd] with row t
    at position start + t, the largest sum_d |q_d k_d| / sqrt(hd) that any score is made of).
    keep: [n, hkv, L] further mask."""
    n, hq, hd = q.shape
    hkv = k.shape[1]
    qq = q.double().view(n, hkv, hq // hkv, hd)
    x = torch.einsum("nhgd,lhd->nhgl", qq, k.double()) / math.sqrt(hd)
    seen = torch.arange(k.shape[0], device="cuda")[None] <= start + torch.arange(n, device="cuda")[:, None]
    mask = seen[:, None, None]
    if keep is not None:
        mask = mask & keep[:, :, None]
    x = x.masked_fill(~mask, -math.inf)
    big = torch.einsum("nhgd,lhd->nhgl", qq.abs(), k.double().abs()).amax() / math.sqrt(hd)
    y = torch.einsum("nhgl,lhd->nhgd", torch.softmax(x, -1), v.double())
    return y.reshape(n, hq, hd), float(big)


def near(got, want, big, vmax, kind="decode"):
    """What the tensor-core kernels may be off by, beyond the output's own rounding.

    A score is a sum of products whose magnitudes add up to `big` at most.  decode: q enters
    as two f16 parts (what is left is below 2^-22 of it) and the sums are f32 over at most 256
    terms in a tree of matrix instructions: 2^-18 * big covers both, and moves each
    probability by that share.  prompt: q and the keys are rounded to f16, 2^-11 each, and
    what is smaller than 2^-10 keeps 2^-25 absolute: 2^-9 * big.  A probability (decode: times
    its block's scale) is rounded to f16, which moves an output by 2^-11 of the largest
    value, times 15 / 8 where codes 0..15 stand for -8..7; values of a prompt are rounded
    to f16 as well: 2^-9 * vmax covers all of these.  Numerator and denominator both move.
    """
    score = 2.0 ** (-18 if kind == "decode" else -9) * big
    bound = vmax * (2 * math.expm1(score) + 2.0 ** -9)
    off = (got.double() - want).abs()
    allowed = bound + u(got.dtype) * want.abs() + 1e-30
    assert torch.equal(torch.isnan(got), torch.isnan(want))  # blocks with a NaN scale
    worst = float((off / allowed).nan_to_num(nan=0.0).max())
    assert worst <= 1, worst


def top(v) -> float:
    """The largest magnitude."""
    return float(v.abs().nan_to_num(nan=0.0).max())


# --------------------------------------------------------------------- Q4_0 storage --

def tie_rows(seed, n, hd):
    """Values next to and on the borders between two codes, blocks with equal extremes, zeros,
    tiny and huge blocks."""
    x = normal(seed, n, hd)
    b = x.view(-1, 32)
    half = torch.arange(-8, 8, device="cuda").repeat(2).float() + 0.5
    for i in range(0, b.shape[0], 4):
        d = float(torch.rand(()) * 0.1 + 0.01)
        d = float(torch.tensor(d).half())
        b[i] = half * d
        b[i, 7] = -8 * d               # the largest: the scale is d exactly
        ulp = torch.nextafter(b[i], b[i] * 2)
        if i % 8 == 0:
            b[i, 8:20] = ulp[8:20]
    if b.shape[0] > 24:
        b[1, 3], b[1, 17] = 5.0, -5.0  # equal magnitudes: the first one counts
        b[2, 3], b[2, 17] = -5.0, 5.0
        b[5] = 0
        b[6] *= 1e-6                   # the scale is subnormal in f16
        b[7] *= 1e-9                   # ... and zero
        b[9] *= 3e4
        b[10] = -b[9]
        b[11] *= 1e30
        b[13, 4] = math.nan
        b[14, 0] = math.inf
        b[15, 31] = -math.inf
        b[17] = 0
        b[17, 30] = 1.0
        b[18] = 1.0
    return x


@pytest.mark.parametrize("hd, hkv", [(32, 3), (64, 2), (96, 2), (128, 4), (256, 1)])
def test_q4_codes_are_the_rules(ctx, hd, hkv):
    n = 70
    k = tie_rows(1, n * hkv, hd).view(n, hkv, hd)
    v = tie_rows(2, n * hkv, hd).view(n, hkv, hd)
    kv = qb.KvCache(ctx, 1, 128, hkv, hd, "q4_0")
    kv.update(0, k, v, range(n))
    got = kv.read(0, [0], [n])
    for x, y in zip(got, (k, v)):
        torch.testing.assert_close(x.double(), q4_plain(y), rtol=0, atol=0, equal_nan=True)
    for x, y in zip(kv.get(0, range(n)), got):
        np.testing.assert_array_equal(x, y.cpu().numpy())


def test_q4_needs_whole_blocks(ctx):
    with pytest.raises(qb.QllamaError, match="Q4_0 storage needs head_dim divisible by 32"):
        qb.KvCache(ctx, 1, 64, 2, 48, "q4_0")


# ---------------------------------------------------------------- append and read --

@pytest.mark.parametrize("cache, dtype, hq, hkv, hd, start, lens", [
    ("q4_0", "bf16", 8, 2, 128, [0, 5, 63, 130], [3, 0, 2, 70]),
    ("q4_0", "f16", 4, 4, 64, [64, 0], [1, 1]),
    ("q4_0", "f32", 7, 1, 128, [200], [33]),
    ("q4_0", "f32", 3, 3, 96, [1, 2], [64, 65]),
    ("q8_0", "bf16", 6, 3, 128, [0, 61], [128, 5]),
    ("q8_0", "f32", 2, 2, 64, [9], [1]),
    ("f16", "bf16", 8, 8, 64, [100, 0, 1], [1, 40, 0]),
    ("bf16", "f32", 10, 5, 128, [0], [77]),
    ("f32", "f16", 4, 2, 48, [0, 7], [9, 10]),
    ("f32", "f32", 4, 1, 128, [3, 0], [1, 1]),
    ("bf16", "bf16", 5, 1, 30, [62], [5]),
])
@pytest.mark.parametrize("layout", ["packed", "strided", "odd"])
def test_append_rows_and_queries(ctx, cache, dtype, hq, hkv, hd, start, lens, layout):
    """Rows and rotated queries bit for bit, in slots of any order; what the call does not
    write stays as it was."""
    B, total = len(lens), sum(lens)
    seqs = list(range(B))[::-1]
    kv = qb.KvCache(ctx, 2, 300, hkv, hd, cache, 64, B + 1)
    before = {}
    for s in range(B + 1):
        n = start[seqs.index(s)] if s < B else 40
        k, v = normal(10 + s, n, hkv, hd), normal(20 + s, n, hkv, hd)
        for layer in (0, 1):
            kv.update(layer, k, v, range(n), seq=s)
        before[s] = kv.read(1, [0], [n], [s])
    width = (hq + 2 * hkv) * hd
    row = normal(5, max(1, total), width + (3 if layout == "odd" else 0), dtype=dtype)
    if layout == "odd":  # elements off every wider alignment
        row = row[:, 1:1 + width]
    q, k, v = (x.unflatten(1, (-1, hd))[:total] for x in
               row.split((hq * hd, hkv * hd, hkv * hd), 1))
    if layout == "packed":
        q, k, v = (x.contiguous() for x in (q, k, v))
    places = [a + i for a, n in zip(start, lens) for i in range(n)]
    out = kv.append(1, k, v, start, lens, THETA, seq_ids=seqs, q=q)
    assert out.dtype is DT[dtype]
    torch.testing.assert_close(out, rotated(q, places).to(DT[dtype]), rtol=0, atol=0)
    got = kv.read(1, start, lens, seqs)
    for x, y in zip(got, (rotated(k, places), v.float())):
        torch.testing.assert_close(x.double(), stored(y, cache), rtol=0, atol=0)
    for s in range(B + 1):
        n = before[s][0].shape[0]
        assert kv.layer_len(1, s) == n + (lens[seqs.index(s)] if s < B else 0)
        assert kv.layer_len(0, s) == n
        for layer in (0, 1):
            for x, y in zip(kv.read(layer, [0], [n], [s]), before[s]):
                assert torch.equal(x, y)


def test_append_equals_the_operators_own_append(ctx):
    """ql_kv_append leaves what ql_attn_forward leaves; of Q8_0, whose d is rounded apart by a
    unit in f32's last place, a value next to a tie may be the neighbour, one d off."""
    for cache in ("f16", "q8_0", "q4_0"):
        a, b = (qb.KvCache(ctx, 1, 256, 2, 128, cache, 64, 2) for _ in range(2))
        k, v, q = (normal(i, 2, 80, h, 128, dtype="bf16") for i, h in ((1, 2), (2, 2), (3, 4)))
        qb.attention_forward(a, 0, q, k, v, [0, 0], 4, 2, 128, THETA, out_dtype="bf16")
        b.append(0, k.flatten(0, 1), v.flatten(0, 1), [0, 0], [80, 80], THETA)
        for x, y in zip(a.read(0, [0, 0], [80, 80]), b.read(0, [0, 0], [80, 80])):
            if cache != "q8_0":
                assert torch.equal(x, y)
                continue
            d = x.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True) / 127
            off = (x - y).unflatten(-1, (-1, 32)).abs()
            # (d itself may round to f16's neighbour: 2^-10 of the largest value)
            assert bool((off <= 1.13 * d).all()) and float((off > 0).float().mean()) < 1e-3


def test_append_in_place_and_q_out_types(ctx):
    kv = qb.KvCache(ctx, 1, 64, 2, 64, "f16")
    q, k, v = (normal(i, 5, h, 64, dtype="f16") for i, h in ((1, 6), (2, 2), (3, 2)))
    want = rotated(q, range(5))
    out = torch.empty(5, 6, 64, device="cuda")
    kv.append(0, k, v, [0], [5], THETA, q=q, q_out=out)
    assert torch.equal(out, want)
    kv.truncate(0, 0)
    assert kv.append(0, k, v, [0], [5], THETA, q=q, q_out=q) is q
    assert torch.equal(q, want.half())


def test_read_types_and_repeats(ctx):
    kv = qb.KvCache(ctx, 1, 256, 2, 64, "q4_0", 64, 3)
    k, v = normal(1, 200, 2, 64), normal(2, 200, 2, 64)
    for s in range(3):
        kv.update(0, k[: 200 - 60 * s] + s, v[: 200 - 60 * s] - s, range(200 - 60 * s), seq=s)
    start, lens, seqs = [3, 0, 63, 100], [120, 1, 2, 0], [2 - 2, 2, 0, 1]
    for t in ("f32", "f16", "bf16"):
        got = kv.read(0, start, lens, seqs, out_dtype=t)
        at = 0
        for a, n, s in zip(start, lens, seqs):
            for x, y in zip(got, (k + s, v - s)):
                want = q4_plain(y[a:a + n]).float().to(DT[t])
                assert torch.equal(x[at:at + n], want)
            at += n
        assert at == got[0].shape[0]


def test_truncate_several(ctx):
    kv = qb.KvCache(ctx, 2, 128, 1, 32, "q4_0", 64, 4)
    x = normal(1, 100, 1, 32)
    for layer in (0, 1):
        for s in range(4):
            kv.update(layer, x, x, range(100), seq=s)
    with pytest.raises(qb.QllamaError, match="cannot truncate"):
        kv.truncate([0, 3], [5, 101])
    assert [kv.seq_len(s) for s in range(4)] == [100] * 4
    kv.truncate([2, 0, 2], [90, 0, 70])
    assert [kv.layer_len(1, s) for s in range(4)] == [0, 100, 70, 100]
    kv.truncate([], [])
    with pytest.raises(qb.QllamaError, match="length"):
        kv.truncate([0, 1], [0])


# ------------------------------------------------------- attention over a Q4_0 cache --

def filled(ctx, cache, lens, hkv, hd, seed=1, scale=1.0, page=64, layers=1, spare=0):
    """A cache whose sequences hold random rows, and those rows as it holds them (f64)."""
    kv = qb.KvCache(ctx, layers, max(lens) + spare + 1, hkv, hd, cache, page, len(lens))
    rows = []
    for b, n in enumerate(lens):
        k = normal(seed + 2 * b, n, hkv, hd, scale=scale)
        v = normal(seed + 2 * b + 1, n, hkv, hd, scale=scale)
        for layer in range(layers):
            kv.update(layer, k, v, range(n), seq=b)
        rows.append(tuple(x.double() for x in kv.read(0, [0], [n], [b], out_dtype="f32")))
    return kv, rows


@pytest.mark.parametrize("hq, hkv, hd, n, lens, dtype", [
    (8, 2, 128, 1, [1, 2, 63, 64, 65, 700], "bf16"),
    (32, 4, 64, 1, [701], "f16"),
    (4, 4, 128, 1, [1500, 31], "f32"),
    (5, 1, 64, 1, [4097], "bf16"),
    (16, 1, 128, 1, [333, 1000], "f16"),        # more than eight heads on one KV head
    (9, 1, 64, 1, [64], "f16"),
    (8, 8, 128, 3, [10, 129], "bf16"),          # drafted tokens
    (16, 2, 128, 5, [5, 70, 1025], "f16"),
    (21, 3, 64, 4, [4, 333], "bf16"),
    (2, 1, 128, 63, [63, 200], "f16"),
    (8, 2, 128, 64, [64, 300], "bf16"),         # prompts
    (6, 2, 64, 200, [200, 777], "f16"),
    (4, 4, 128, 129, [1300], "f32"),
    (3, 3, 96, 2, [2, 100], "f32"),             # other head sizes
    (2, 1, 32, 70, [70], "bf16"),
    (4, 2, 256, 1, [130], "f16"),
])
def test_attention_over_4_bits(ctx, hq, hkv, hd, n, lens, dtype):
    kv, rows = filled(ctx, "q4_0", lens, hkv, hd)
    q = normal(99, len(lens), n, hq, hd, dtype=dtype)
    start = [m - n for m in lens]
    out = qm.attention_forward_appended(kv, 0, q, start, hq, hkv, hd, THETA, out_dtype=dtype)
    for b, (k, v) in enumerate(rows):
        want, big = attention(q[b], k, v, start[b])
        near(out[b].view(n, hq, hd), want, big, top(v),
             "prompt" if n >= 64 else "decode")


@pytest.mark.parametrize("n", [1, 4, 90])
@pytest.mark.parametrize("hd", [64, 128])
def test_4_bit_forward_appends(ctx, n, hd):
    """ql_attn_forward: q and k arrive unrotated, the rows are appended, several steps on."""
    hq, hkv, lens = 8, 2, [0, 60, 191]
    kv = qb.KvCache(ctx, 1, 600, hkv, hd, "q4_0", 128, 3)
    for b, m in enumerate(lens):
        kv.update(0, normal(b, m, hkv, hd), normal(b + 9, m, hkv, hd), range(m), seq=b)
    for step in range(3):
        q, k, v = (normal(50 + 3 * step + i, 3, n, h, hd, dtype="bf16")
                   for i, h in enumerate((hq, hkv, hkv)))
        out = qb.attention_forward(kv, 0, q, k, v, lens, hq, hkv, hd, THETA, out_dtype="bf16")
        for b, m in enumerate(lens):
            kc, vc = (x.double() for x in kv.read(0, [0], [m + n], [b]))
            places = range(m, m + n)
            torch.testing.assert_close(kc[m:], q4_plain(rotated(k[b], places)), rtol=0, atol=0)
            torch.testing.assert_close(vc[m:], q4_plain(v[b].float()), rtol=0, atol=0)
            want, big = attention(rotated(q[b], places), kc, vc, m)
            near(out[b].view(n, hq, hd), want, big, top(vc),
                 "prompt" if n >= 64 else "decode")
        lens = [m + n for m in lens]


@pytest.mark.parametrize("scale", [1e-4, 3e-2, 200.0, 2e4])
def test_4_bit_values_of_any_size(ctx, scale):
    """Values far from 1, some beyond a scale's range (their blocks read back as NaN), and a
    head whose values are a thousand times another's."""
    hq, hkv, hd, n = 8, 2, 128, 333
    kv = qb.KvCache(ctx, 1, 400, hkv, hd, "q4_0")
    k = normal(1, n, hkv, hd)
    v = normal(2, n, hkv, hd, scale=scale)
    v[:, 1] *= 1e-3
    v[100:200] *= 8
    kv.update(0, k, v, range(n))
    kc, vc = (x.double() for x in kv.read(0, [0], [n]))
    for t in (1, 70):
        q = normal(3, 1, t, hq, hd)
        out = qm.attention_forward_appended(kv, 0, q, [n - t], hq, hkv, hd, THETA)
        want, big = attention(q[0], kc, vc, n - t)
        for h in range(hkv):
            part = slice(4 * h, 4 * h + 4)
            near(out[0].view(t, hq, hd)[:, part], want[:, part], big, top(vc[:, h]),
                 "prompt" if t >= 64 else "decode")


@pytest.mark.parametrize("hd", [64, 128])
def test_4_bit_scores_far_from_zero(ctx, hd):
    """All scores near -400 (or, of the other heads, +400), over pieces of which some rows see
    nothing."""
    hq, hkv, n = 8, 2, 64 * 40 + 2
    kv = qb.KvCache(ctx, 1, n, hkv, hd, "q4_0")
    k = normal(1, n, hkv, hd, scale=0.1) + 1
    v = normal(2, n, hkv, hd)
    kv.update(0, k, v, range(n))
    kc, vc = (x.double() for x in kv.read(0, [0], [n]))
    for t in (1, 5):
        q = normal(3, 1, t, hq, hd, scale=0.1) - 400 / math.sqrt(hd)
        q[:, :, 1::2] *= -1
        out = qm.attention_forward_appended(kv, 0, q, [n - t], hq, hkv, hd, THETA)
        want, big = attention(q[0], kc, vc, n - t)
        near(out[0].view(t, hq, hd), want, big, top(vc))


def test_rows_behind_the_end_are_never_read(ctx):
    """A rolled-back sequence leaves NaN rows behind its end; other sequences' stay apart."""
    hq, hkv, hd = 8, 2, 128
    kv = qb.KvCache(ctx, 1, 256, hkv, hd, "q4_0", 64, 2)
    bad = torch.full((200, hkv, hd), math.nan, device="cuda")
    for s in (0, 1):
        kv.update(0, bad, bad, range(200), seq=s)
    kv.truncate([0, 1], [0, 0])
    for n in (1, 17, 70, 130):
        k, v = normal(n, n, hkv, hd), normal(n + 1, n, hkv, hd)
        kv.update(0, k, v, range(n), seq=0)
        kc, vc = (x.double() for x in kv.read(0, [0], [n]))
        for t in (1, min(n, 3), 64 if n >= 64 else 1):
            q = normal(3, 1, t, hq, hd, dtype="bf16")
            out = qm.attention_forward_appended(kv, 0, q, [n - t], hq, hkv, hd, THETA)
            want, big = attention(q[0], kc, vc, n - t)
            near(out[0].view(t, hq, hd), want, big, top(vc),
                 "prompt" if t >= 64 else "decode")
        kv.truncate(0, 0)


def test_4_bit_nan_rows_reach_the_output(ctx):
    """A NaN value of a seen position makes its columns' outputs NaN, no others."""
    hq, hkv, hd, n = 8, 2, 128, 100
    kv = qb.KvCache(ctx, 1, 128, hkv, hd, "q4_0")
    k, v = normal(1, n, hkv, hd), normal(2, n, hkv, hd)
    v[50, 1, 40] = math.nan  # block 1 of head 1
    kv.update(0, k, v, range(n))
    q = normal(3, 1, 1, hq, hd)
    out = qm.attention_forward_appended(kv, 0, q, [n - 1], hq, hkv, hd, THETA).view(2, 4, hd)
    assert torch.isfinite(out[0]).all()
    assert torch.isnan(out[1, :, 32:64]).all()
    assert torch.isfinite(out[1, :, :32]).all() and torch.isfinite(out[1, :, 64:]).all()


# ---------------------------------------------------------- attention over some blocks --

def chosen(q, k, cache, start, blocks, first, last):
    """The blocks of each (token, KV head) by the definition, in f64, and each score's gap."""
    n, hq, hd = q.shape
    hkv = k.shape[1]
    kind = torch.float16 if cache == "f16" else torch.bfloat16
    out = torch.full((n, hkv, blocks), -1, dtype=torch.int32)
    for t in range(n):
        newest = (start + t) // TILE
        old = k[: newest * TILE].view(newest, TILE, hkv, hd) if newest else k.new_zeros(0, 1, hkv, hd)
        lo, hi = (f(1).float().to(kind).double() for f in (old.amin, old.amax))
        qq = q[t].double().view(hkv, -1, hd)
        s = torch.maximum(torch.einsum("hgd,jhd->jhgd", qq, lo), torch.einsum("hgd,jhd->jhgd", qq, hi))
        s = s.sum((2, 3)).nan_to_num(nan=math.inf, posinf=math.inf, neginf=-math.inf).cpu()
        for h in range(hkv):
            always = {j for j in range(newest + 1) if j < first or j > newest - last}
            rest = sorted((j for j in range(newest) if j not in always),
                          key=lambda j: (-float(s[j, h]), j))
            if newest + 1 > blocks:
                rest = rest[: blocks - len(always)]
            pick = sorted(always | set(rest))
            out[t, h, : len(pick)] = torch.tensor(pick)
    return out.cuda()


def keep_of(pick, length):
    """[n, hkv, L] mask of the positions in the chosen blocks."""
    places = torch.arange(length, device="cuda") // TILE
    return (pick[..., None] == places).any(-2)


@pytest.mark.parametrize("cache, hq, hkv, hd, n, lens, blocks, first, last, page, dtype", [
    ("f16", 8, 2, 128, 1, [1, 64, 65, 1000], 4, 1, 1, 64, "f16"),
    ("bf16", 32, 4, 64, 1, [5000, 130], 9, 0, 2, 128, "bf16"),
    ("q4_0", 8, 2, 128, 1, [2049, 500, 3], 6, 1, 2, 64, "bf16"),
    ("q4_0", 4, 4, 64, 3, [700, 66], 3, 0, 1, 192, "f16"),
    ("q4_0", 16, 1, 128, 1, [3000], 12, 1, 1, 64, "f16"),
    ("q8_0", 8, 2, 128, 2, [1400, 200], 5, 2, 1, 64, "f32"),
    ("q8_0", 4, 2, 64, 1, [600], 4, 1, 1, 64, "f32"),
    ("f16", 3, 3, 128, 4, [450], 7, 1, 3, 64, "f32"),
    ("bf16", 9, 1, 128, 1, [640], 1, 0, 1, 64, "bf16"),
    ("f32", 6, 2, 48, 2, [400, 90], 3, 1, 1, 64, "f32"),
    ("q4_0", 2, 2, 96, 1, [400], 3, 1, 1, 64, "f32"),
    ("f16", 8, 1, 128, 1, [40000], 40, 1, 4, 64, "f16"),
    ("q4_0", 8, 1, 128, 1, [40000], 300, 1, 4, 64, "f16"),
    ("bf16", 8, 8, 128, 1, [900] * 8, 1000000 // 1000, 1, 1, 64, "bf16"),  # all of them
])
def test_attention_over_blocks(ctx, cache, hq, hkv, hd, n, lens, blocks, first, last, page, dtype):
    kv, rows = filled(ctx, cache, lens, hkv, hd, page=page)
    q = normal(7, len(lens), n, hq, hd, dtype=dtype)
    start = [m - n for m in lens]
    sel = torch.empty(len(lens), n, hkv, blocks, dtype=torch.int32, device="cuda")
    out, _ = qm.attention_forward_sparse(kv, 0, q, start, hq, hkv, hd, blocks, first, last,
                                         out_dtype=dtype, selected=sel)
    again, _ = qm.attention_forward_sparse(kv, 0, q, start, hq, hkv, hd, blocks, first, last,
                                           out_dtype=dtype)
    assert torch.equal(out, again)  # with the lists in the workspace
    for b, (k, v) in enumerate(rows):
        pick = chosen(q[b], k, cache, start[b], blocks, first, last)
        assert torch.equal(sel[b], pick)
        want, big = attention(q[b], k, v, start[b], keep_of(pick, lens[b]))
        near(out[b].view(n, hq, hd), want, big, top(v))


@pytest.mark.parametrize("cache", ["f16", "q4_0"])
def test_equal_scores_take_the_lower_block(ctx, cache):
    """Blocks that repeat tie exactly."""
    hq, hkv, hd = 4, 2, 64
    kv = qb.KvCache(ctx, 1, 64 * 20, hkv, hd, cache)
    k = normal(1, 64, hkv, hd).repeat(16, 1, 1)
    kv.update(0, k, k, range(1024))
    q = normal(2, 1, 1, hq, hd, dtype="bf16")
    sel = torch.empty(1, 1, hkv, 6, dtype=torch.int32, device="cuda")
    qm.attention_forward_sparse(kv, 0, q, [1023], hq, hkv, hd, 6, 2, 1, selected=sel)
    assert (sel.view(hkv, 6).cpu() == torch.tensor([0, 1, 2, 3, 4, 15])).all()


def test_blocks_with_nan_keys_come_first(ctx):
    hq, hkv, hd = 4, 1, 128
    kv = qb.KvCache(ctx, 1, 64 * 20, hkv, hd, "bf16")
    k = normal(1, 1024, hkv, hd)
    k[64 * 9 + 3, 0, 5] = math.nan
    kv.update(0, k, k.nan_to_num(0.0), range(1024))
    sel = torch.empty(1, 1, hkv, 3, dtype=torch.int32, device="cuda")
    q = normal(2, 1, 1, hq, hd, dtype="bf16")
    qm.attention_forward_sparse(kv, 0, q, [1023], hq, hkv, hd, 3, 1, 1, selected=sel)
    assert sel.flatten().tolist() == [0, 9, 15]


@pytest.mark.parametrize("cache", ["bf16", "q4_0", "q8_0"])
def test_bounds_follow_rewritten_rows(ctx, cache):
    """A rolled-back and rewritten prefix is scored by its new keys, in each layer, and after
    a slot has changed hands."""
    hq, hkv, hd, n = 8, 2, 128, 1000
    kv = qb.KvCache(ctx, 2, 1024, hkv, hd, cache, 64, 2)
    q = normal(1, 1, 1, hq, hd, dtype="bf16")
    sel = torch.empty(1, 1, hkv, 5, dtype=torch.int32, device="cuda")

    def check(layer, seq, m):
        out, _ = qm.attention_forward_sparse(kv, layer, q, [m - 1], hq, hkv, hd, 5, 1, 1, [seq],
                                             selected=sel)
        k, v = (x.double() for x in kv.read(layer, [0], [m], [seq], out_dtype="f32"))
        pick = chosen(q[0], k, cache, m - 1, 5, 1, 1)
        assert torch.equal(sel[0], pick)
        want, big = attention(q[0], k, v, m - 1, keep_of(pick, m))
        near(out.view(1, hq, hd), want, big, top(v))

    def write(layer, seq, a, m, seed):
        kv.update(layer, normal(seed, m - a, hkv, hd), normal(seed + 1, m - a, hkv, hd),
                  range(a, m), seq=seq)

    for layer in (0, 1):
        write(layer, 0, 0, n, 10 + layer)
        check(layer, 0, n)
    kv.truncate(0, 300)
    for layer in (0, 1):
        write(layer, 0, 300, 900, 30 + layer)
        check(layer, 0, 900)
    kv.clear_seq(0)
    write(0, 1, 0, 700, 50)
    check(0, 1, 700)
    write(1, 1, 0, 700, 52)
    write(0, 0, 0, 640, 60)
    write(1, 0, 0, 640, 62)
    for layer in (0, 1):
        check(layer, 0, 640)
        check(layer, 1, 700)
    kv.clear()
    write(0, 0, 0, 500, 70)
    check(0, 0, 500)
    write(0, 0, 500, 580, 72)  # blocks that fill up between two calls
    check(0, 0, 580)


# ------------------------------------------------------------------------- together --

@pytest.mark.parametrize("cache", ["q4_0", "bf16"])
def test_prompts_then_steps(ctx, cache):
    """Packed prompts, then decode steps: append with rotated queries, dense attention in one
    layer, over chosen blocks in the other, drafts rolled back between them."""
    hq, hkv, hd, lens = 8, 2, 128, [300, 171, 515]
    kv = qb.KvCache(ctx, 2, 700, hkv, hd, cache, 64, 3)
    k, v = normal(1, sum(lens), hkv, hd, dtype="bf16"), normal(2, sum(lens), hkv, hd, dtype="bf16")
    for layer in (0, 1):
        kv.append(layer, k, v, [0, 0, 0], lens, THETA)
    for step in range(4):
        n = (1, 4, 3, 1)[step]
        for layer in (0, 1):
            q, k, v = (normal(100 * step + 10 * layer + i, 3 * n, h, hd, dtype="bf16")
                       for i, h in enumerate((hq, hkv, hkv)))
            qr = kv.append(layer, k, v, lens, [n] * 3, THETA, q=q).view(3, n, hq, hd)
            if layer == 0:
                out = qm.attention_forward_appended(kv, 0, qr, lens, hq, hkv, hd, THETA)
                picks = None
            else:
                picks = torch.empty(3, n, hkv, 4, dtype=torch.int32, device="cuda")
                out, _ = qm.attention_forward_sparse(kv, 1, qr, lens, hq, hkv, hd, 4, 1, 1,
                                                     selected=picks)
            for b, m in enumerate(lens):
                kc, vc = (x.double() for x in kv.read(layer, [0], [m + n], [b], out_dtype="f32"))
                keep = None
                if picks is not None:
                    want = chosen(qr[b], kc, cache, m, 4, 1, 1)
                    assert torch.equal(picks[b], want)
                    keep = keep_of(want, m + n)
                want, big = attention(qr[b], kc, vc, m, keep)
                near(out[b].view(n, hq, hd), want, big, top(vc))
        lens = [m + max(1, n - 1 - b) for b, m in enumerate(lens)]
        kv.truncate(range(3), lens)


# -------------------------------------------------------------------------- refusals --

def refuses(text, call):
    with pytest.raises(qb.QllamaError, match=text):
        call()


def test_append_and_read_refusals(ctx):
    kv = qb.KvCache(ctx, 1, 100, 2, 64, "q4_0", 64, 3, 3)
    k, v = normal(1, 10, 2, 64), normal(2, 10, 2, 64)
    q = normal(3, 10, 4, 64)
    refuses("must continue", lambda: kv.append(0, k, v, [1], [10], THETA))
    refuses("exceeds cache capacity", lambda: kv.append(0, normal(1, 101, 2, 64), normal(1, 101, 2, 64), [0], [101], THETA))
    refuses("appears twice", lambda: kv.append(0, k, v, [0, 0], [5, 5], THETA, seq_ids=[1, 1]))
    refuses("out of range", lambda: kv.append(0, k, v, [0], [10], THETA, seq_ids=[3]))
    refuses("out of range", lambda: kv.append(1, k, v, [0], [10], THETA))
    refuses("has shape", lambda: kv.append(0, k, v, [0], [9], THETA))
    refuses("has shape", lambda: kv.append(0, k, v[:, :1], [0], [10], THETA))
    refuses("k's type", lambda: kv.append(0, k, v.half(), [0], [10], THETA))
    refuses("contiguous", lambda: kv.append(0, k, v.transpose(1, 2).contiguous().transpose(1, 2), [0], [10], THETA))
    refuses("theta", lambda: kv.append(0, k, v, [0], [10], -1.0))
    refuses("rows", lambda: kv.append(0, k[:0], v[:0], [0, 0], [5, -5], THETA))
    refuses("overlaps", lambda: kv.append(0, k, v, [0], [10], THETA, q=q[:, :2], q_out=k))
    refuses("position", lambda: kv.append(0, k, v, [0, 0], [10], THETA))
    assert kv.seq_len() == 0
    # the pool is out of pages: nothing has moved
    refuses("exhausted", lambda: kv.append(0, normal(1, 240, 2, 64), normal(1, 240, 2, 64),
                                           [0, 0, 0], [80, 80, 80], THETA))
    assert [kv.seq_len(s) for s in range(3)] == [0, 0, 0]
    kv.append(0, k, v, [0], [10], THETA)
    refuses("beyond the written prefix", lambda: kv.read(0, [5], [6]))
    refuses("beyond the written prefix", lambda: kv.read(0, [11], [0]))
    refuses("negative", lambda: kv.read(0, [-1], [1]))
    refuses("overlap", lambda: kv.read(0, [0], [10], out=(k, k)))
    refuses("shape", lambda: kv.read(0, [0], [10], out=(k, v[:9])))
    assert kv.read(0, [10], [0])[0].shape == (0, 2, 64)
    assert kv.read(0, [], [])[0].shape == (0, 2, 64)


def test_sparse_refusals(ctx):
    kv, _ = filled(ctx, "q4_0", [100], 2, 64)
    q = normal(1, 1, 1, 4, 64)
    call = lambda *a, **k: qm.attention_forward_sparse(kv, 0, q, [99], 4, 2, 64, *a, **k)
    refuses("must hold", lambda: call(0))
    refuses("must hold", lambda: call(3, 2, 2))
    refuses("must hold", lambda: call(3, 0, 0))
    refuses("must hold", lambda: call(3, -1, 1))
    refuses("selected", lambda: call(3, selected=torch.zeros(1, 1, 2, 4, dtype=torch.int32, device="cuda")))
    refuses("not the last ones", lambda: qm.attention_forward_sparse(kv, 0, q, [98], 4, 2, 64, 3))
    refuses("q_rot", lambda: qm.attention_forward_sparse(kv, 0, q[..., :32], [99], 4, 2, 64, 3))


# ------------------------------------------------ streams, graphs, several callers --

def run_of(kv, seqs, lens, q, k, v, out, picked, sel, hq, hkv, hd):
    """One decode step of listed slots: append with rotated queries, both attentions."""
    n = len(seqs)
    qr = kv.append(0, k, v, lens, [1] * n, THETA, seq_ids=seqs, q=q).view(n, 1, hq, hd)
    qm.attention_forward_appended(kv, 0, qr, lens, hq, hkv, hd, THETA, seq_ids=seqs, out=out)
    qm.attention_forward_sparse(kv, 0, qr, lens, hq, hkv, hd, 4, 1, 1, seq_ids=seqs, out=picked,
                                selected=sel)
    return qr


def step_buffers(n, hq, hkv, hd, seed, dtype="bf16"):
    q, k, v = (normal(seed + i, n, h, hd, dtype=dtype) for i, h in enumerate((hq, hkv, hkv)))
    out, picked = (torch.zeros(n, 1, hq * hd, dtype=DT[dtype], device="cuda") for _ in range(2))
    return q, k, v, out, picked, torch.zeros(n, 1, hkv, 4, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("cache", ["q4_0", "f16"])
def test_captured_step_replays(ctx, stream, cache):
    """A captured step replays on new inputs, also after the workspace has been outgrown by
    other calls, and the eager call on the same inputs leaves the same bits."""
    hq, hkv, hd, lens = 8, 2, 128, [449, 63]
    kv, _ = filled(ctx, cache, [450, 64], hkv, hd, spare=2)
    kv.truncate(range(2), lens)
    buf = step_buffers(2, hq, hkv, hd, 1, "f16")
    rest = (hq, hkv, hd)
    run_of(kv, [0, 1], lens, *buf, *rest)  # pages, tables and bounds are there
    kv.truncate(range(2), lens)
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run_of(kv, [0, 1], lens, *buf, *rest)
    # a call that needs a larger workspace
    big, _ = filled(ctx, "f16", [200] * 8, 8, 128, seed=50)
    qm.attention_forward_appended(big, 0, normal(9, 8, 150, 64, 128), [50] * 8, 64, 8, 128, THETA)
    for seed in (7, 8):
        new = step_buffers(2, hq, hkv, hd, 10 * seed, "f16")
        for a, b in zip(buf[:3], new[:3]):
            a.copy_(b)
        graph.replay()
        kv.truncate(range(2), lens)
        run_of(kv, [0, 1], lens, *new, *rest)
        for a, b in zip(buf[3:], new[3:]):
            assert torch.equal(a, b)
    del graph


def test_first_sparse_call_is_not_captured(ctx, stream):
    """The allocation of the bounds is refused under capture, and the capture goes on."""
    kv, _ = filled(ctx, "q4_0", [200], 2, 64)
    q = normal(1, 1, 1, 4, 64, dtype="bf16")
    out = torch.zeros(1, 1, 256, dtype=torch.bfloat16, device="cuda")
    qm.attention_forward_appended(kv, 0, q, [199], 4, 2, 64, THETA, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(qb.QllamaError, match="before the capture"):
            qm.attention_forward_sparse(kv, 0, q, [199], 4, 2, 64, 2, out=out)
        qm.attention_forward_appended(kv, 0, q, [199], 4, 2, 64, THETA, out=out)
    want = out.clone()
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)


@pytest.mark.parametrize("cache", ["q4_0", "f16"])
def test_blocks_around_captures(ctx, stream, cache):
    """Blocks are chosen by the keys that the cache holds: after a call that has been captured
    and not yet replayed, and after each replay of a captured append."""
    hq, hkv, hd = 8, 2, 128
    kv, _ = filled(ctx, cache, [130], hkv, hd, spare=400)
    q = normal(1, 1, 1, hq, hd, dtype="f16")
    out = torch.zeros(1, 1, hq * hd, dtype=torch.float16, device="cuda")
    sel = torch.zeros(1, 1, hkv, 4, dtype=torch.int32, device="cuda")

    def choose(m, kv=kv):
        qm.attention_forward_sparse(kv, 0, q, [m - 1], hq, hkv, hd, 4, 1, 1, out=out, selected=sel)

    def check(m):
        k, v = (x.double() for x in kv.read(0, [0], [m], out_dtype="f32"))
        pick = chosen(q[0], k, cache, m - 1, 4, 1, 1)
        assert torch.equal(sel[0], pick)
        want, big = attention(q[0], k, v, m - 1, keep_of(pick, m))
        near(out.view(1, hq, hd), want, big, top(v))

    def rows(seed, n):
        return normal(seed, n, hkv, hd, dtype="f16"), normal(seed + 1, n, hkv, hd, dtype="f16")

    choose(520, filled(ctx, cache, [520], hkv, hd)[0])  # the workspace is there
    choose(130)
    kv.append(0, *rows(3, 320), [130], [320], THETA)
    choose_only, append_only = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    ctx.synchronize()
    with torch.cuda.graph(choose_only, stream=stream):
        choose(450)
    choose(450)  # the captured call has not run
    check(450)
    out.zero_(), sel.zero_()
    choose_only.replay()
    check(450)
    k, v = rows(5, 70)
    kv.append(0, k, v, [450], [70], THETA)  # pages and tables are there
    kv.truncate(0, 450)
    ctx.synchronize()
    with torch.cuda.graph(append_only, stream=stream):
        kv.append(0, k, v, [450], [70], THETA)
    for seed in (7, 9, 11):
        for a, b, gain in zip((k, v), rows(seed, 70), (seed, 1)):
            a.copy_(b * gain)
        append_only.replay()
        choose(520)
        check(520)
    del choose_only, append_only


def test_first_call_with_a_theta_is_not_captured(ctx, stream):
    """The upload of the rotations is refused under capture, and the capture goes on."""
    kv, _ = filled(ctx, "f16", [70], 2, 64, spare=2)
    row = normal(1, 1, 2, 64, dtype="f16")
    kv.append(0, row, row, [70], [1], THETA)
    kv.truncate(0, 70)
    graph = torch.cuda.CUDAGraph()
    ctx.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(qb.QllamaError, match="before the capture"):
            kv.append(0, row, row, [70], [1], 2 * THETA)
        kv.append(0, row, row, [70], [1], THETA)
    graph.replay()
    assert kv.read(0, [70], [1])[1].float().equal(row.float())
    del graph


def test_tensors_of_another_stream(ctx):
    """Tensors of torch's current stream, while the context has its own: made late on a busy
    stream, used and dropped at once."""
    hq, hkv, hd = 8, 2, 128
    kv, rows = filled(ctx, "q4_0", [500], hkv, hd)
    ctx.synchronize()
    side = torch.cuda.Stream()
    want = None
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            q = normal(3, 1, 1, hq, hd, dtype="bf16")
            out = qm.attention_forward_appended(kv, 0, q, [499], hq, hkv, hd, THETA)
            picked, _ = qm.attention_forward_sparse(kv, 0, q, [499], hq, hkv, hd, 3)
            del q
            junk = torch.full((1, 1, hq, hd), 1e9, dtype=torch.bfloat16, device="cuda")
            got = (out.clone(), picked.clone())
        side.synchronize()
        if want is None:
            want = got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del junk
    k, v = rows[0]
    y, big = attention(normal(3, 1, 1, hq, hd, dtype="bf16")[0], k, v, 499)
    near(want[0].view(1, hq, hd), y, big, top(v))


def test_two_threads_with_contexts_of_their_own():
    """Two host threads, each with its context, caches and stream, at once."""
    import threading

    hq, hkv, hd = 8, 2, 64
    fails = []

    def work(seed):
        try:
            s = torch.cuda.Stream()
            c = qb.Context(0)
            c.set_stream(s.cuda_stream)
            with torch.cuda.stream(s):
                kv, rows = filled(c, "q4_0", [300 + seed, 64], hkv, hd, seed=seed, spare=40)
                rows = [tuple(x.float() for x in r) for r in rows]
                lens = [300 + seed, 64]
                for step in range(20):
                    buf = step_buffers(2, hq, hkv, hd, 100 * seed + step)
                    qr = run_of(kv, [0, 1], lens, *buf, hq, hkv, hd)
                    for b, m in enumerate(lens):
                        kc, vc = (x.double() for x in kv.read(0, [0], [m + 1], [b]))
                        want, big = attention(qr[b], kc, vc, m)
                        near(buf[3][b].view(1, hq, hd), want, big, top(vc))
                        assert torch.equal(buf[5][b], chosen(qr[b], kc, "q4_0", m, 4, 1, 1))
                    lens = [m + 1 for m in lens]
                c.synchronize()
        except BaseException as e:  # noqa: BLE001 -- reported by the main thread
            fails.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not fails, fails


def test_results_do_not_depend_on_the_rest_of_the_batch(ctx):
    """Twice the same call, the same bits; a context's other work in between changes nothing."""
    hq, hkv, hd = 32, 8, 128
    kv, _ = filled(ctx, "q4_0", [3000, 100, 1700], hkv, hd)
    q = normal(5, 3, 2, hq, hd, dtype="bf16")
    start = [2998, 98, 1698]
    a = qm.attention_forward_appended(kv, 0, q, start, hq, hkv, hd, THETA)
    s, _ = qm.attention_forward_sparse(kv, 0, q, start, hq, hkv, hd, 9)
    for _ in range(3):
        assert torch.equal(a, qm.attention_forward_appended(kv, 0, q, start, hq, hkv, hd, THETA))
        t, _ = qm.attention_forward_sparse(kv, 0, q, start, hq, hkv, hd, 9)
        assert torch.equal(s, t)


def test_host_buffers_and_sharded_free_paths(ctx):
    """numpy in and out (ql_attn_forward with host memory) over a Q4_0 cache; the no-allocation
    entry point and the fused projection refuse it."""
    hq, hkv, hd = 4, 2, 64
    kv = qb.KvCache(ctx, 1, 200, hkv, hd, "q4_0")
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal((70, h, hd)).astype(np.float32) for h in (hq, hkv, hkv))
    out = qb.attention_forward(kv, 0, q, k, v, 0, hq, hkv, hd, THETA)
    kc, vc = (x.double() for x in kv.read(0, [0], [70]))
    want, big = attention(rotated(torch.from_numpy(q).cuda(), range(70)), kc, vc, 0)
    near(torch.from_numpy(out).cuda().view(70, hq, hd), want, big, top(vc), "prompt")
    t = [torch.from_numpy(x[:1]).cuda() for x in (q, k, v)]
    starts, seqs = (ctypes.c_int64 * 1)(70), (ctypes.c_int32 * 1)(0)
    o = torch.empty(1, hq * hd, device="cuda")
    args = qb.AttnArgs(0, 1, 1, seqs, starts, hq, hkv, hd, THETA, qb.F32, qb.F32, qb.MEM_DEVICE,
                       *(x.data_ptr() for x in t), o.data_ptr())
    L = qb.load()
    assert L.ql_attn_decode_noalloc(ctx._h, kv._h, ctypes.byref(args)) == qb.ERR_UNSUPPORTED
    assert L.ql_qkv_rope_append(ctx._h, kv._h, ctypes.byref(args), t[0].data_ptr(), 64,
                                t[0].data_ptr(), o.data_ptr()) == qb.ERR_UNSUPPORTED


def test_model_on_a_4_bit_cache(ctx):
    """The model host over a Q4_0 cache (head_dim 32: the reference-order kernel): a prompt in two
    calls leaves the bits of the prompt at once."""
    cfg = qm.LlamaConfig(97, 128, 256, 4, 2, 2, 128, 1e-5, 1e4)
    model = qm.Llama(ctx, cfg)
    rng = np.random.default_rng(3)
    E, F, kvd = 128, 256, 64
    shapes = {"token_embd.weight": (97, E), "output_norm.weight": (E,)}
    for i in range(2):
        b = f"blk.{i}."
        shapes.update({b + "attn_norm.weight": (E,), b + "ffn_norm.weight": (E,),
                       b + "attn_q.weight": (E, E), b + "attn_k.weight": (kvd, E),
                       b + "attn_v.weight": (kvd, E), b + "attn_output.weight": (E, E),
                       b + "ffn_gate.weight": (F, E), b + "ffn_up.weight": (F, E),
                       b + "ffn_down.weight": (E, F)})
    for name, shape in shapes.items():
        w = np.ones(shape) if "norm" in name else rng.standard_normal(shape) * 0.1
        model.set_tensor(name, w.astype(np.float32))
    ids = rng.integers(0, 97, 20).astype(np.int32)
    one = model.kv_cache(dtype="q4_0")
    whole = model.forward_with_cache(ids, 0, one)
    two = model.kv_cache(dtype="q4_0")
    a = model.forward_with_cache(ids[:13], 0, two)
    b = model.forward_with_cache(ids[13:], 13, two)
    assert np.isfinite(whole).all()
    np.testing.assert_array_equal(np.concatenate((a, b)), whole)
