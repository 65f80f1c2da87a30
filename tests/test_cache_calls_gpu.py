"""Calls on the paged cache that its documentation allows at the edges of what
tests/test_cache_ops_gpu.py covers: rows and blocks around captures, clears and other
rotations, keys and values far from 1, and what Python callers may pass.

Tolerances count roundings, as there: u(t) = eps(t) / 2 for one rounding to t.
"""
import math

import numpy as np
import pytest
import torch

import qllama_b200 as qb
from qllama_b200 import model as qm
from tests.test_cache_ops_gpu import (DT, THETA, attention, chosen, ctx, filled, keep_of, near, normal,  # noqa: F401
                                      on_stream, q4_plain, q8_plain, refuses, rotated, stored, stream,
                                      top, u)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache, hq, hkv, hd", [("f16", 8, 2, 128), ("q4_0", 8, 2, 64),
                                                ("f32", 4, 2, 48)])
def test_choice_over_blocks_without_pages(stream, cache, hq, hkv, hd):
    """A captured selection replayed after its sequence has been cleared: the table holds no
    pages.  The status says so, and nothing is written beside the lists, whatever the
    workspace held (here NaNs)."""
    c = qb.Context(0)
    c.set_stream(stream.cuda_stream)
    m, blocks = 1300, 4
    kv, _ = filled(c, cache, [m], hkv, hd)
    other = qb.KvCache(c, 1, 256, 2, 64, "f16")
    q = normal(1, 1, 1, hq, hd, dtype="f16")
    out = torch.zeros(1, 1, hq * hd, dtype=torch.float16, device="cuda")
    room = torch.full((3 * hkv, blocks), -7, dtype=torch.int32, device="cuda")
    sel = room[hkv:2 * hkv].view(1, 1, hkv, blocks)
    call = lambda: qm.attention_forward_sparse(kv, 0, q, [m - 1], hq, hkv, hd, blocks, 1, 1,
                                               out=out, selected=sel)
    nan = np.full((128, 64, 64), 0xffffffff, np.uint32).view(np.float32)

    def fill_workspace():  # host rows are staged at its beginning
        qb.attention_forward(other, 0, nan, nan[:, :2], nan[:, :2], 0, 64, 2, 64, THETA)
        other.clear()

    fill_workspace()
    call()
    c.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    kv.clear_seq(0)
    fill_workspace()
    graph.replay()
    with pytest.raises(qb.QllamaError, match="block-table"):
        c.synchronize()
    assert (room[:hkv] == -7).all() and (room[2 * hkv:] == -7).all()
    # the first and the newest block, and of equal scores the lower ones
    assert sel.view(hkv, blocks).tolist() == [[0, 1, 2, (m - 1) // 64]] * hkv
    c.synchronize()
    del graph


@pytest.mark.parametrize("cache, hq, hkv, hd", [("f16", 8, 2, 128), ("bf16", 6, 2, 64),
                                                ("f32", 4, 2, 48), ("f16", 9, 1, 128)])
@pytest.mark.parametrize("signs", ["positive", "negative", "mixed", "zeros"])
def test_blocks_with_infinite_keys(ctx, cache, hq, hkv, hd, signs):
    """A bound that is infinite counts by the score's definition: a key of -inf under
    positive queries only adds what the block's largest key gives.  (The keys' own weight is 0
    there, but 0 * inf in the sums over their products is not: outputs are not compared.)"""
    m, blocks = 64 * 14, 5
    kv = qb.KvCache(ctx, 1, m, hkv, hd, cache)
    k = normal(1, m, hkv, hd)
    k[64 * 3 + 5, 0, 7] = -math.inf
    k[64 * 5 + 1, :, 2] = math.inf
    k[64 * 7:64 * 8, 0, 9] = -math.inf    # both bounds
    k[64 * 8 + 2, :, 11] = -math.inf
    k[64 * 8 + 3, :, 12] = math.inf
    k[64 * 9:64 * 10, :, 13] = math.inf
    kv.update(0, k, normal(2, m, hkv, hd), range(m))
    q = normal(3, 1, 1, hq, hd, dtype="bf16")
    q = q.abs() if signs == "positive" else -q.abs() if signs == "negative" else q
    if signs == "zeros":
        q[..., [7, 13]] = 0
    sel = torch.empty(1, 1, hkv, blocks, dtype=torch.int32, device="cuda")
    qm.attention_forward_sparse(kv, 0, q, [m - 1], hq, hkv, hd, blocks, 1, 1, selected=sel)
    rows = kv.read(0, [0], [m], out_dtype="f32")[0].double()
    assert torch.equal(sel[0], chosen(q[0], rows, cache, m - 1, blocks, 1, 1))


def off_by(got, want):
    """The largest distance of a head's output, relative to its norm."""
    return float(((got.double() - want).norm(dim=-1) / want.norm(dim=-1)).max())


# Of outputs that are sums of many independent values of mean 0, each times a probability that
# has been rounded to f16 alone and once more with V's scale: 2 * 2^-11 of each at most, and the
# sums' norms are in the same proportion.  (Scores add 2^-18 of their sum of magnitudes.)
NORM = 1e-3


@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4, 300.0])
@pytest.mark.parametrize("gap", [0, 10, 14])
def test_small_values_beside_a_position_without_any(ctx, size, gap):
    """Values far from 1, and a first position that takes nearly all of the weight, `gap` above
    the others' scores, but has no value (an attention sink)."""
    B, hq, hkv, hd, m = 20, 8, 2, 128, 2050
    kv = qb.KvCache(ctx, 1, m, hkv, hd, "q4_0", 64, B)
    for b in range(B):
        k, v = normal(b, m, hkv, hd), normal(b + 100, m, hkv, hd, scale=size)
        k[0], v[0] = 0, 0
        k[:, :, 0] = 0
        k[0, :, 0] = 8
        kv.update(0, k, v, range(m), seq=b)
    q = normal(200, B, 1, hq, hd)
    q[..., 0] = gap * math.sqrt(hd) / 8
    out = qm.attention_forward_appended(kv, 0, q, [m - 1] * B, hq, hkv, hd, THETA)
    for b in range(B):
        kc, vc = (x.double() for x in kv.read(0, [0], [m], [b]))
        want, _ = attention(q[b], kc, vc, m - 1)
        assert off_by(out[b].view(1, hq, hd), want) <= NORM


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 4])
@pytest.mark.parametrize("order", ["rising", "falling", "behind the end"])
def test_values_of_changing_size(ctx, hd, n, order):
    """Values whose size doubles (or halves) from tile to tile, over f16's range and more; and
    large and NaN rows behind the end of a sequence of small ones."""
    hq, hkv, m = 8, 2, 64 * 24 + 37
    kv = qb.KvCache(ctx, 1, 64 * 27, hkv, hd, "q4_0", 128, 2)
    k, v = normal(1, m, hkv, hd), normal(2, m, hkv, hd)
    if order == "behind the end":
        bad = torch.full((64 * 27, hkv, hd), 3e4, device="cuda")
        bad[1::2] = math.nan
        kv.update(0, bad, bad, range(64 * 27), seq=0)
        kv.update(0, bad, bad, range(64 * 27), seq=1)
        kv.truncate([0, 1], [0, 0])
        v *= 1e-3
    else:
        tile = torch.arange(m, device="cuda") // 64
        v *= 2.0 ** (tile - 13 if order == "rising" else 11 - tile)[:, None, None]
    for s in (0, 1):
        kv.update(0, k[:m - 900 * s], v[:m - 900 * s], range(m - 900 * s), seq=s)
    q = normal(3, 2, n, hq, hd)
    start = [m - n, m - 900 - n]
    out = qm.attention_forward_appended(kv, 0, q, start, hq, hkv, hd, THETA)
    for s in (0, 1):
        kc, vc = (x.double() for x in kv.read(0, [0], [m - 900 * s], [s]))
        want, _ = attention(q[s], kc, vc, start[s])
        assert off_by(out[s].view(n, hq, hd), want) <= NORM


@pytest.mark.parametrize("call", ["append", "forward", "appended rows of a projection"])
def test_captured_rotations_stay_those_of_their_theta(ctx, stream, call):
    """A captured call replays with its own theta, whatever other calls on the cache rotate by
    in between; calls of several thetas alternate, also inside one graph."""
    hq, hkv, hd, n = 4, 2, 64, 3
    thetas = [1e4, 5e5, 1e6, 1e3, 2e4, 3e4]
    kv = qb.KvCache(ctx, 1, 128, hkv, hd, "f32")
    q, k, v = (normal(i, n, h, hd) for i, h in ((1, hq), (2, hkv), (3, hkv)))
    x, w = normal(4, 1, n, 32), normal(5, 32, (hq + 2 * hkv) * hd)

    def run(theta, start=40):
        """(the rotated keys' positions, the keys before the rotation)"""
        if call == "append":
            kv.append(0, k, v, [start], [n], theta)
            return k
        if call == "forward":
            qb.attention_forward(kv, 0, q, k, v, start, hq, hkv, hd, theta)
            return k
        qm.qkv_rope_append(kv, 0, x, w, start, hq, hkv, hd, theta)
        return (x[0].double() @ w.double())[:, hq * hd:(hq + hkv) * hd].float().view(n, hkv, hd)

    def check(theta, start=40):
        got, want = kv.read(0, [start], [n])[0], rotated(keys, range(start, start + n), theta)
        # (a projection's products are summed in f32: 32 terms of up to 4 * 4)
        off = 0 if call != "appended rows of a projection" else 32 * 32 * 16 * 2.0 ** -24
        torch.testing.assert_close(got, want, rtol=0, atol=off)

    zeros = torch.zeros(40, hkv, hd, device="cuda")
    kv.update(0, zeros, zeros, range(40))
    for t in thetas[:2]:
        keys = run(t)
        check(t)
        kv.truncate(0, 40)
    ctx.synchronize()
    graph, both = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run(thetas[0])
    kv.truncate(0, 40)
    with torch.cuda.graph(both, stream=stream):
        run(thetas[1])
        run(thetas[0], 40 + n)
    for t in thetas[1:]:
        kv.truncate(0, 40)
        run(t)
        check(t)
        graph.replay()
        check(thetas[0])
    kv.truncate(0, 40)
    run(thetas[2])
    run(thetas[2], 40 + n)
    both.replay()
    check(thetas[1])
    check(thetas[0], 40 + n)
    del graph, both


@pytest.mark.parametrize("cache", ["f16", "q4_0"])
@pytest.mark.parametrize("then", ["discarded", "refused", "replayed late"])
def test_pages_taken_under_capture(ctx, stream, cache, then):
    """Pages that a captured call takes are the sequence's for later calls too: where the
    capture is thrown away, where a part of it is refused, and before its first replay."""
    hq, hkv, hd, m, n = 4, 2, 64, 60, 70
    kv = qb.KvCache(ctx, 1, 256, hkv, hd, cache, 64, 2)
    old, k, v = (normal(i, r, hkv, hd, dtype="f16") for i, r in ((1, m), (2, n), (3, n)))
    q = normal(4, n, hq, hd, dtype="f16")
    kv.append(0, old, old, [m - 60], [60], THETA)
    first = normal(5, 200, hkv, hd, dtype="f16")
    kv.append(0, first, first, [0], [200], THETA, seq_ids=[1])
    kv.clear_seq(1)  # its pages are handed out anew
    q_out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        if then == "refused":
            with pytest.raises(qb.QllamaError, match="before the capture"):
                kv.append(0, k, v, [m], [n], 3 * THETA, q=q, q_out=q_out)
        kv.append(0, k, v, [m], [n], THETA, q=q, q_out=q_out)
    kv.truncate(0, m)
    if then == "discarded":
        graph.reset()
    places = range(m, m + n)

    def check(k, v):
        got = kv.read(0, [m], [n])
        for x, y in zip(got, (rotated(k, places), v.float())):
            torch.testing.assert_close(x.double(), stored(y, cache), rtol=0, atol=0)
        out = qm.attention_forward_appended(kv, 0, normal(6, 1, 1, hq, hd), [m + n - 1], hq, hkv,
                                            hd, THETA)
        kc, vc = (x.double() for x in kv.read(0, [0], [m + n], out_dtype="f32"))
        want, big = attention(normal(6, 1, hq, hd), kc, vc, m + n - 1)
        near(out.view(1, hq, hd), want, big, top(vc))
        ctx.synchronize()  # no kernel met an entry outside the pool

    other = normal(7, n, hkv, hd, dtype="f16")
    kv.append(0, other, k, [m], [n], THETA, q=q)
    check(other, k)
    if then != "discarded":
        graph.replay()
        check(k, v)
        assert torch.equal(q_out, rotated(q, places).half())
    del graph


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
def test_q8_appends_have_one_rule(ctx, hd):
    """ql_kv_append takes a Q8_0 block's d as max|x| times the f32 nearest to 1/127 whatever the
    head size: for these maxima half of them then lies on the other side of a tie."""
    hkv, n = 3, 66
    v = normal(1, n, hkv, hd, dtype="bf16") * 0.2
    b = v.view(-1, 32)
    for i, m in enumerate((1.1171875, 1.6171875, 1.8671875)):
        b[i::4, 5], b[i::4, 20], b[i::4, 31] = m, m / 2, -m / 2
    kv = qb.KvCache(ctx, 1, 128, hkv, hd, "q8_0")
    kv.append(0, v, v, [0], [n], THETA)
    k, got = kv.read(0, [0], [n])
    torch.testing.assert_close(got.double(), q8_plain(v.float()), rtol=0, atol=0)
    torch.testing.assert_close(k.double(), q8_plain(rotated(v, range(n))), rtol=0, atol=0)


@pytest.mark.parametrize("contiguous", [True, False])
def test_update_with_tensors_of_another_stream(contiguous):
    """KvCache.update of tensors that torch's current stream has yet to write, while the context
    has a stream of its own; they are dropped, and their memory written to, right after it."""
    hkv, hd, n = 2, 64, 100
    c = qb.Context(0)
    kv = qb.KvCache(c, 1, 128, hkv, hd, "f32")
    side = torch.cuda.Stream()
    rows = [normal(i, n, hkv, hd) for i in range(3)]
    torch.cuda.synchronize()
    for i in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            k, v = rows[i] + 1, rows[i] - 1
            if not contiguous:
                k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
            kv.update(0, k, v, range(n))
            del k, v
            junk = [torch.full((n, hkv, hd), 7.0, device="cuda") for _ in range(4)]
            got = kv.read(0, [0], [n])
        side.synchronize()
        assert torch.equal(got[0], rows[i] + 1) and torch.equal(got[1], rows[i] - 1)
        kv.truncate(0, 0)
        del junk


def test_a_context_may_go_first():
    """Caches and weights outlive their context's handle, also in a cycle that the collector
    takes apart in an order of its own; with the last of them the context's memory goes."""
    import gc

    def free():
        gc.collect()
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        return torch.cuda.mem_get_info()[0]

    def use(c, kv):
        q, k, v = (normal(i, 1, 300, h, 64) for i, h in ((1, 8), (2, 2), (3, 2)))
        kv.truncate(0, 0)
        return qb.attention_forward(kv, 0, q, k, v, 0, 8, 2, 64, THETA)

    c = qb.Context(0)
    use(c, qb.KvCache(c, 1, 1 << 14, 2, 64, "f32"))  # what is loaded once is loaded
    del c
    before = free()
    for way in ("closed", "cycle"):
        stream = torch.cuda.Stream()
        c = qb.Context(0)
        c.set_stream(stream.cuda_stream)
        kv = qb.KvCache(c, 1, 1 << 16, 2, 64, "f32")
        w = qm.Q4Weight(c, np.zeros((1 << 14, 1 << 11), np.uint8), np.zeros((1 << 14, 1 << 7), np.float16))
        with torch.cuda.stream(stream):
            use(c, kv)
        assert free() < before - (64 << 20)
        if way == "closed":
            c.close()
            c.close()
            del stream
            kv.close()
            w.close()
        else:
            c.others, kv.others = [kv, w, c], [c, w]
        del c, kv, w
        stream = None
        assert free() >= before - (8 << 20)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("places", ["even", "odd", "all"])
@pytest.mark.parametrize("hd", [64, 128])
def test_queries_far_below_their_largest(ctx, dtype, places, hd):
    """Rotated 16-bit queries with values 2^-22 of the row's largest and less, in either nibble
    of the codes' words, on keys that are as much larger there."""
    hq, hkv, m = 8, 2, 1000
    k = normal(1, m, hkv, hd)
    k[..., 32:] *= 2.0 ** 15
    q = normal(2, 1, 1, hq, hd)
    if dtype == "f16":  # 2^-24 is the least of its values
        q[..., :32] *= 2.0 ** 8
        k[..., :32] *= 2.0 ** -8
    q[..., 32:] *= 2.0 ** (-22 if dtype == "bf16" else -14)
    if places != "all":
        q[..., 32 + (places == "even")::2] = 0
    k[..., 32:] *= 2.0 ** (2 if dtype == "bf16" else -4)  # a 32nd of what the others give
    k.clamp_(-5e5, 5e5)  # what a block of the cache can hold
    q = q.to(torch.bfloat16 if dtype == "bf16" else torch.float16)
    kv = qb.KvCache(ctx, 1, m, hkv, hd, "q4_0")
    kv.update(0, k, normal(3, m, hkv, hd), range(m))
    kc, vc = (x.double() for x in kv.read(0, [0], [m]))
    assert torch.isfinite(kc).all()
    out = qm.attention_forward_appended(kv, 0, q, [m - 1], hq, hkv, hd, THETA)
    want, _ = attention(q[0], kc, vc, m - 1)
    assert off_by(out.view(1, hq, hd), want) <= NORM


@pytest.mark.parametrize("size", [1e25, 1e33, 1e36, 3e38])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("call", ["appended", "forward"])
def test_queries_up_to_the_types_largest(ctx, size, dtype, call):
    """The largest score takes all of the weight, and the output is its position's row."""
    hq, hkv, hd, m = 8, 2, 128, 300
    kv = qb.KvCache(ctx, 1, m + 1, hkv, hd, "q4_0")
    kv.update(0, normal(1, m, hkv, hd, scale=1e-3), normal(2, m, hkv, hd), range(m))
    q = (torch.rand(1, 1, hq, hd, device="cuda") * 2 - 1).mul_(0.7)
    q[..., 64:] = 0
    q = (q * size).to(DT[dtype])
    if call == "forward":
        row = normal(3, 1, 1, hkv, hd, scale=1e-3)
        out = qb.attention_forward(kv, 0, q, row.to(q.dtype), row.to(q.dtype), [m], hq, hkv, hd, THETA)
        q, n = rotated(q[0].float(), [m])[None], m + 1
    else:
        out, n = qm.attention_forward_appended(kv, 0, q, [m - 1], hq, hkv, hd, THETA), m
    kc, vc = (x.double() for x in kv.read(0, [0], [n]))
    x = torch.einsum("hgd,lhd->hgl", q[0, 0].double().view(hkv, -1, hd), kc)
    best = x.argmax(-1)
    want = torch.stack([vc[best[h], h] for h in range(hkv)])
    # a probability of 1, rounded to f16 with its scale
    torch.testing.assert_close(out.view(hkv, -1, hd).double(), want, rtol=2.0 ** -10, atol=1e-30)


@pytest.mark.parametrize("size", [1.0, 1e9, 1e30, 3e38])
@pytest.mark.parametrize("sign", [1, -1])
def test_equal_scores_share_the_weight(ctx, size, sign):
    """However large the scores: the output of equal keys is the mean of the values."""
    B, hq, hkv, hd, m = 3, 8, 2, 128, 2000
    kv = qb.KvCache(ctx, 1, m, hkv, hd, "q4_0", 64, B)
    for b in range(B):
        kv.update(0, normal(b, 1, hkv, hd, scale=1e-2).expand(m - b, -1, -1).contiguous(),
                  normal(b + 9, m - b, hkv, hd), range(m - b), seq=b)
    q = torch.full((B, 1, hq, hd), sign * size, device="cuda")
    out = qm.attention_forward_appended(kv, 0, q, [m - 1 - b for b in range(B)], hq, hkv, hd, THETA)
    for b in range(B):
        mean = kv.read(0, [0], [m - b], [b])[1].double().mean(0).repeat_interleave(hq // hkv, 0)
        assert off_by(out[b].view(hq, hd), mean) <= NORM


# What the kernels' outputs may be off by relative to their norm, by the cache's type.  f16 and
# bf16: queries and probabilities enter as two 16-bit parts (bf16: what is left is below 2^-17 of
# them; scores are sums of up to 16 in magnitude here); Q8_0: queries as two 8-bit parts, 2^-16 of
# the row's largest, which 128 channels add up to 2^-12.  A key left out of 20000 is 2^-7.1 off.
NORMS = {"f32": 2.0 ** -12, "f16": 2.0 ** -12, "bf16": 2.0 ** -12, "q8_0": NORM, "q4_0": NORM}


@pytest.mark.parametrize("cache", ["f16", "bf16", "q8_0", "q4_0"])
@pytest.mark.parametrize("n", [1, 3])
def test_no_key_of_a_long_cache_is_left_out(ctx, cache, n):
    """Distances by norm, dense and over chosen blocks: a mean over many keys is small beside
    its largest value, and so is what one of them adds."""
    hq, hkv, hd, lens = 8, 2, 128, [4097, 20000, 130]
    kv, rows = filled(ctx, cache, lens, hkv, hd)
    q = normal(50, 3, n, hq, hd)
    start = [m - n for m in lens]
    out = qm.attention_forward_appended(kv, 0, q, start, hq, hkv, hd, THETA)
    sel = torch.empty(3, n, hkv, 60, dtype=torch.int32, device="cuda")
    part, _ = qm.attention_forward_sparse(kv, 0, q, start, hq, hkv, hd, 60, 1, 2, selected=sel)
    for b, (k, v) in enumerate(rows):
        want, _ = attention(q[b], k, v, start[b])
        assert off_by(out[b].view(n, hq, hd), want) <= NORMS[cache]
        pick = chosen(q[b], k, cache, start[b], 60, 1, 2)
        assert torch.equal(sel[b], pick)
        want, _ = attention(q[b], k, v, start[b], keep_of(pick, lens[b]))
        assert off_by(part[b].view(n, hq, hd), want) <= NORMS[cache]


@pytest.mark.parametrize("cache, hq, hkv, hd, n", [("f16", 24, 2, 128, 1), ("bf16", 16, 1, 64, 3),
                                                   ("q8_0", 20, 2, 128, 1), ("f32", 12, 1, 128, 2),
                                                   ("q4_0", 24, 2, 128, 2), ("q8_0", 8, 2, 64, 1)])
def test_blocks_with_more_heads_on_a_kv_head(ctx, cache, hq, hkv, hd, n):
    lens = [1500, 64, 700]
    kv, rows = filled(ctx, cache, lens, hkv, hd)
    q = normal(60, 3, n, hq, hd, dtype="bf16")
    start = [m - n for m in lens]
    sel = torch.empty(3, n, hkv, 5, dtype=torch.int32, device="cuda")
    out, _ = qm.attention_forward_sparse(kv, 0, q, start, hq, hkv, hd, 5, 1, 1, selected=sel)
    for b, (k, v) in enumerate(rows):
        pick = chosen(q[b], k, cache, start[b], 5, 1, 1)
        assert torch.equal(sel[b], pick)
        want, _ = attention(q[b], k, v, start[b], keep_of(pick, lens[b]))
        assert off_by(out[b].view(n, hq, hd), want) <= NORMS[cache]


@pytest.mark.parametrize("cache", ["q4_0", "f16"])
def test_a_sequence_alone_and_in_a_batch(ctx, cache):
    """The split of the work goes by the whole batch, so a sequence's bits may differ with its
    company, by roundings only; the blocks chosen do not."""
    hq, hkv, hd, lens = 32, 8, 128, [3000, 100, 1700, 9000]
    kv, _ = filled(ctx, cache, lens, hkv, hd)
    q = normal(5, 4, 1, hq, hd, dtype="bf16")
    start = [m - 1 for m in lens]

    def run(seqs):
        sel = torch.empty(len(seqs), 1, hkv, 9, dtype=torch.int32, device="cuda")
        args = (q[seqs], [start[s] for s in seqs], hq, hkv, hd)
        a = qm.attention_forward_appended(kv, 0, *args, THETA, seq_ids=seqs)
        b, _ = qm.attention_forward_sparse(kv, 0, *args, 9, seq_ids=seqs, selected=sel)
        return a.view(-1, hq, hd), b.view(-1, hq, hd), sel

    a, b, sel = run([0, 1, 2, 3])
    for s in range(4):
        x, y, z = run([s])
        assert torch.equal(z[0], sel[s])
        assert off_by(x[0], a[s].double()) <= NORMS[cache] and off_by(y[0], b[s].double()) <= NORMS[cache]


@pytest.mark.parametrize("cache", ["f16", "bf16", "q8_0", "q4_0"])
@pytest.mark.parametrize("n, gap", [(1, 10), (1, 14), (1, 18), (64, 10), (64, 14)])
def test_every_kernel_beside_a_position_without_a_value(ctx, cache, n, gap):
    """As test_small_values_beside_a_position_without_any, for every storage type and for
    prompts, dense and over chosen blocks.

    Prompts round queries, keys and values to f16, 2^-11 of each at most: of independent errors
    less than NORM comes of it, but the first position's score is one product, whose error of
    2^-11 * gap is in every output's sum of weights.
    Beside a gap of 18, decode over f16 and Q8_0 has probabilities that are e^-18 of 2^7: they
    lose up to half of f16's smallest step, 2^-25, and their root mean square is
    2^(7 - 18 * 1.4427) * e = 2^-17.5 (scores are normal with a variance of 1): 2^-7.5."""
    B, hq, hkv, hd, m = 3, 8, 2, 128, 2050
    kv = qb.KvCache(ctx, 1, m, hkv, hd, cache, 64, B)
    for b in range(B):
        k, v = normal(b, m, hkv, hd), normal(b + 100, m, hkv, hd, scale=0.01)
        k[0], v[0] = 0, 0
        k[:, :, 0] = 0
        k[0, :, 0] = 8
        kv.update(0, k, v, range(m), seq=b)
    q = normal(200, B, n, hq, hd)
    q[..., 0] = gap * math.sqrt(hd) / 8
    start = [m - n] * B
    few = 2.0 ** -7.5 if gap == 18 else NORM
    out = qm.attention_forward_appended(kv, 0, q, start, hq, hkv, hd, THETA)
    sel = torch.empty(B, n, hkv, 20, dtype=torch.int32, device="cuda")
    part, _ = qm.attention_forward_sparse(kv, 0, q, start, hq, hkv, hd, 20, 1, 1, selected=sel)
    for b in range(B):
        kc, vc = (x.double() for x in kv.read(0, [0], [m], [b], out_dtype="f32"))
        want, _ = attention(q[b], kc, vc, start[b])
        assert off_by(out[b].view(n, hq, hd), want) <= (NORM + gap * 2.0 ** -11 if n >= 64 else few)
        want, _ = attention(q[b], kc, vc, start[b], keep_of(sel[b], m))
        assert off_by(part[b].view(n, hq, hd), want) <= few


@pytest.mark.parametrize("cache", ["bf16", "q8_0", "q4_0", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [1e-4, 2e-4, 2.4e-4, 3e-4, 1e-3, 0.06, 1e-6, 1.0, 6e3])
@pytest.mark.parametrize("tiles", ["alike", "apart"])
def test_prompts_over_values_of_any_size(ctx, cache, hd, size, tiles):
    """Values around the sizes at which tiles of an f16 copy begin to be scaled, and far from
    them; tiles of like values, and of values up to 2^10 apart.

    Queries, keys, values and probabilities are rounded to f16: independent errors of 2^-11 at
    most, of which scores collect theirs over hd products (variance 1): 4 * 2^-11."""
    B, hq, hkv, n, m = 2, 6, 3, 70, 1000
    kv = qb.KvCache(ctx, 1, m, hkv, hd, cache, 64, B)
    for b in range(B):
        v = normal(b + 100, m, hkv, hd, scale=size)
        if tiles == "apart":
            v *= 2.0 ** (((torch.arange(m, device="cuda") // 64) * 7 + b) % 11 - 10)[:, None, None]
        if cache == "f16" and size < 1e-2:
            v *= 1e2 if size > 1e-5 else 1e4  # such a cache's own steps
        kv.update(0, normal(b, m, hkv, hd), v, range(m), seq=b)
    q = normal(200, B, n, hq, hd)
    out = qm.attention_forward_appended(kv, 0, q, [m - n] * B, hq, hkv, hd, THETA)
    for b in range(B):
        kc, vc = (x.double() for x in kv.read(0, [0], [m], [b], out_dtype="f32"))
        want, _ = attention(q[b], kc, vc, m - n)
        off = (out[b].view(n, hq, hd).double() - want).norm(dim=-1)
        assert (off <= 4 * 2.0 ** -11 * want.norm(dim=-1)).all()  # (0: what a Q8_0 scale rounds off)


def test_small_rows_in_front_of_large_ones(ctx):
    """The first rows of a prompt see only values that are 2^-8 of those further on in their
    tile: as exact as the others."""
    B, hq, hkv, hd, n = 3, 4, 2, 128, 130
    kv = qb.KvCache(ctx, 1, n, hkv, hd, "bf16", 64, B)
    for b, size in enumerate((1e-4, 2.0, 1e-7)):
        v = normal(b + 10, n, hkv, hd, scale=size)
        v[:64] *= 2.0 ** -8
        kv.update(0, normal(b, n, hkv, hd), v, range(n), seq=b)
    q = normal(200, B, n, hq, hd)
    out = qm.attention_forward_appended(kv, 0, q, [0] * B, hq, hkv, hd, THETA)
    for b in range(B):
        kc, vc = (x.double() for x in kv.read(0, [0], [n], [b], out_dtype="f32"))
        want, _ = attention(q[b], kc, vc, 0)
        # (rounding of values and scores as above)
        assert off_by(out[b].view(n, hq, hd), want) <= 4 * 2.0 ** -11
