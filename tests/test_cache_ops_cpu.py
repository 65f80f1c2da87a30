"""Refusals of the operators around the paged cache (ql_kv_append, ql_kv_read,
ql_kv_truncate_batch, ql_attn_forward_appended, ql_attn_forward_sparse): every argument is
checked before any device work, so stand-ins for the context and the cache serve, without a
device."""
import ctypes

import pytest

import qllama_b200 as qb
from qllama_b200 import model as qm

BUF = ctypes.create_string_buffer(1 << 16)
P = (ctypes.addressof(BUF) + 255) // 256 * 256  # an aligned address that is never read
SLOTS, LAYERS, HKV, HD, CAP = 4, 2, 2, 64, 200


class Ctx(ctypes.Structure):  # the head of ql_ctx: a device number, then pointers
    _fields_ = [("device", ctypes.c_int), ("num_sms", ctypes.c_int),
                ("rest", ctypes.c_void_p * 24)]


class Vector(ctypes.Structure):  # std::vector
    _fields_ = [("begin", ctypes.c_void_p), ("end", ctypes.c_void_p), ("cap", ctypes.c_void_p)]


class Kv(ctypes.Structure):  # ql_kv
    _fields_ = [("ctx", ctypes.c_void_p), ("cfg", qb.KvConfig), ("pages_per_seq", ctypes.c_int),
                ("k", Vector), ("v", Vector), ("ks", Vector), ("vs", Vector), ("kmap", Vector),
                ("vmap", Vector), ("have_maps", ctypes.c_bool), ("d_table", ctypes.c_void_p),
                ("table", Vector), ("seq_pages", Vector), ("free_pages", Vector), ("len", Vector),
                ("d_rope", ctypes.c_void_p), ("d_rope_id", ctypes.c_void_p),
                ("rope_theta", ctypes.c_float), ("seen_mark", Vector),
                ("seen_epoch", ctypes.c_uint32), ("patch_idx", Vector), ("bounds", Vector),
                ("bounded", Vector)]


class Cache:
    """A cache of SLOTS sequences whose lengths can be set and read."""

    def __init__(self, lens=(0, 0, 0, 0), dtype=qb.Q4_0):
        self.lens = (ctypes.c_int64 * (LAYERS * SLOTS))(*(list(lens) * LAYERS))
        self.marks = (ctypes.c_uint32 * SLOTS)()
        self.bounded = (ctypes.c_int32 * (LAYERS * SLOTS))(*[n // 64 for n in list(lens) * LAYERS])
        self.ctx = Ctx()
        self.kv = Kv(ctypes.addressof(self.ctx),
                     qb.KvConfig(LAYERS, CAP, HKV, HD, dtype, 64, SLOTS, 16), 4)
        for name, data in (("len", self.lens), ("seen_mark", self.marks),
                           ("bounded", self.bounded)):
            a = ctypes.addressof(data)
            setattr(self.kv, name, Vector(a, a + ctypes.sizeof(data), a + ctypes.sizeof(data)))

    def args(self):
        return ctypes.byref(self.ctx), ctypes.byref(self.kv)


KEEP = []  # arrays whose addresses are in structures


def i32(*x):
    return (ctypes.c_int32 * len(x))(*x)


def i64(*x):
    return (ctypes.c_int64 * len(x))(*x)


def address(x):
    if not isinstance(x, ctypes.Array):
        return x
    KEEP.append(x)
    return ctypes.addressof(x)


def refused(rc, text, code=qb.ERR_INVALID):
    assert rc == code
    assert text in qb.load().ql_last_error().decode()


def append_args(**change):
    a = dict(layer_idx=0, batch=2, seq_ids=i32(0, 1), start_pos=i64(5, 0), new_len=i32(3, 4),
             num_heads=4, num_kv_heads=HKV, head_dim=HD, rope_theta=1e4, in_dtype=qb.F32,
             q_out_dtype=qb.F16, q=P, k=P + 8192, v=P + 16384, q_out=P + 32768)
    return qb.AppendArgs(**{k: address(x) for k, x in {**a, **change}.items()})


@pytest.mark.parametrize("change, text", [
    (dict(num_heads=-1), "positive"), (dict(num_kv_heads=0), "positive"),
    (dict(head_dim=63), "even head_dim"), (dict(rope_theta=0.0), "theta"),
    (dict(rope_theta=float("inf")), "theta"), (dict(in_dtype=qb.Q8_0), "dtype"),
    (dict(q_out_dtype=9), "dtype"), (dict(num_kv_heads=4), "does not match"),
    (dict(head_dim=128), "does not match"), (dict(k_stride=127), "stride"),
    (dict(v_stride=-128), "stride"), (dict(q_stride=8), "stride"),
    (dict(layer_idx=2), "out of range"), (dict(layer_idx=-1), "out of range"),
    (dict(batch=-1), "batch"), (dict(batch=257), "batch"), (dict(seq_ids=None), "NULL"),
    (dict(start_pos=None), "NULL"), (dict(new_len=None), "NULL"),
    (dict(seq_ids=i32(0, 4)), "out of range"), (dict(seq_ids=i32(-1, 0)), "out of range"),
    (dict(seq_ids=i32(1, 1), start_pos=i64(0, 0)), "appears twice"),
    (dict(start_pos=i64(4, 0)), "must continue"), (dict(start_pos=i64(5, -1)), "negative"),
    (dict(start_pos=i64(5, 1 << 40)), "must continue"),
    (dict(new_len=i32(3, -1)), "rows"), (dict(new_len=i32(196, 1)), "exceeds cache capacity"),
    (dict(new_len=i32(3, 2**31 - 1)), "exceeds cache capacity"),
    (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(q=None), "NULL"),
    (dict(q_out=None), "NULL"), (dict(k=P + 2), "aligned"), (dict(v=P + 1), "aligned"),
    (dict(q=P + 2), "aligned"), (dict(q_out=P + 1), "aligned"),
    (dict(q_out=P), "overlaps"), (dict(q_out=P + 8192), "overlaps"),
    (dict(q_out=P + 16384 + 7 * 512 - 4), "overlaps"),
    (dict(q_out=P, q_out_dtype=qb.F32, q_stride=512), "overlaps")])
def test_append_refusals(change, text):
    c = Cache(lens=(5, 0, 0, 0))
    a = append_args(**change)
    refused(qb.load().ql_kv_append(*c.args(), ctypes.byref(a)), text)
    assert list(c.lens[:SLOTS]) == [5, 0, 0, 0]


def test_a_cache_of_another_context_is_refused():
    c, other = Cache(lens=(100, 0, 0, 0)), Ctx()
    L, x, kv = qb.load(), ctypes.byref(other), ctypes.byref(c.kv)
    text = "belongs to another context"
    refused(L.ql_kv_append(x, kv, ctypes.byref(append_args())), text)
    refused(L.ql_kv_read(x, kv, 0, 1, i32(0), i64(0), i32(1), qb.F32, P, P + 8192), text)
    refused(L.ql_attn_forward_sparse(x, kv, ctypes.byref(attn_args()),
                                     ctypes.byref(qm.SparseArgs(4, 1, 1, None))), text)


def test_too_many_heads_are_refused():
    c = Cache()
    refused(qb.load().ql_kv_append(*c.args(), ctypes.byref(append_args(num_heads=1 << 17))),
            "heads", qb.ERR_UNSUPPORTED)


def test_append_of_nothing_is_a_no_op():
    c = Cache(lens=(5, 0, 0, 0))
    for change in (dict(batch=0, seq_ids=None, start_pos=None, new_len=None),
                   dict(new_len=i32(0, 0), k=None, v=None, q=None, q_out=None)):
        a = append_args(**change)
        assert qb.load().ql_kv_append(*c.args(), ctypes.byref(a)) == qb.OK
    for args in ((None, None, None), (*c.args(), None)):
        refused(qb.load().ql_kv_append(*args), "NULL")


@pytest.mark.parametrize("change, text", [
    (dict(layer=2), "out of range"), (dict(batch=257), "batch"), (dict(batch=-1), "batch"),
    (dict(seq=None), "NULL"), (dict(lens=None), "NULL"), (dict(seq=i32(0, 7)), "out of range"),
    (dict(start=i64(-1, 0)), "negative"), (dict(lens=i32(-1, 0)), "rows"),
    (dict(lens=i32(101, 0)), "beyond the written prefix"),
    (dict(start=i64(1 << 40, 0)), "beyond the written prefix"),
    (dict(dtype=qb.Q4_0), "dtype"), (dict(k=None), "NULL"), (dict(v=None), "NULL"),
    (dict(k=P + 2), "aligned"), (dict(v=P + 1), "aligned"), (dict(v=P), "overlap"),
    (dict(v=P + 55 * 512 - 4), "overlap")])
def test_read_refusals(change, text):
    c = Cache(lens=(100, 50, 0, 0))
    a = {**dict(layer=0, batch=2, seq=i32(0, 0), start=i64(0, 95), lens=i32(50, 5), dtype=qb.F32,
                k=P, v=P + 32768), **change}
    rc = qb.load().ql_kv_read(*c.args(), a["layer"], a["batch"], a["seq"], a["start"], a["lens"],
                              a["dtype"], a["k"], a["v"])
    refused(rc, text)


def test_read_of_nothing_is_a_no_op():
    c = Cache(lens=(100, 50, 0, 0))
    assert qb.load().ql_kv_read(*c.args(), 0, 1, i32(0), i64(100), i32(0), qb.F32, None,
                                None) == qb.OK


def test_truncate_several():
    c = Cache(lens=(100, 130, 7, 0))
    t = qb.load().ql_kv_truncate_batch
    kv = ctypes.byref(c.kv)
    refused(t(None, 0, None, None), "NULL")
    refused(t(kv, 1, None, i64(0)), "NULL")
    refused(t(kv, -1, None, None), "batch")
    refused(t(kv, 2, i32(0, 4), i64(0, 0)), "out of range")
    refused(t(kv, 2, i32(0, 2), i64(0, 8)), "cannot truncate")
    refused(t(kv, 2, i32(0, 2), i64(-1, 0)), "cannot truncate")
    assert list(c.lens) == [100, 130, 7, 0] * 2
    assert t(kv, 3, i32(1, 0, 1), i64(128, 63, 129)) == qb.OK
    assert list(c.lens) == [63, 128, 7, 0] * 2
    assert list(c.bounded) == [0, 2, 0, 0] * 2  # bounds of rewritten blocks are dropped
    assert t(kv, 0, None, None) == qb.OK


def attn_args(**change):
    a = dict(layer_idx=0, batch=1, new_len=1, seq_ids=i32(0), start_pos=i64(99), num_heads=4,
             num_kv_heads=HKV, head_dim=HD, rope_theta=1e4, in_dtype=qb.F32, out_dtype=qb.F32,
             mem=qb.MEM_DEVICE, q=P, out=P + 8192)
    return qb.AttnArgs(**{**a, **change})


@pytest.mark.parametrize("blocks, first, last", [(0, 0, 1), (3, 0, 0), (3, 2, 2), (3, -1, 1),
                                                 (2**31 - 1, 2**31 - 1, 1), (5, 1, 2**31 - 1)])
def test_sparse_refuses_block_counts(blocks, first, last):
    c = Cache(lens=(100, 0, 0, 0))
    s = qm.SparseArgs(blocks, first, last, None)
    refused(qb.load().ql_attn_forward_sparse(*c.args(), ctypes.byref(attn_args()),
                                             ctypes.byref(s)), "must hold")


@pytest.mark.parametrize("change, text", [
    (dict(mem=qb.MEM_HOST), "device buffers"), (dict(start_pos=i64(98)), "not the last ones"),
    (dict(layer_idx=5), "out of range"), (dict(q=None), "NULL"), (dict(out=None), "NULL"),
    (dict(num_heads=5), "divisible"), (dict(in_dtype=qb.Q4_0), "dtype"),
    (dict(out_dtype=qb.Q8_0), "dtype"), (dict(batch=5), "batch"), (dict(new_len=-1), "new_len")])
def test_sparse_refusals(change, text):
    c = Cache(lens=(100, 0, 0, 0))
    a = attn_args(**change)
    refused(qb.load().ql_attn_forward_sparse(*c.args(), ctypes.byref(a),
                                             ctypes.byref(qm.SparseArgs(4, 1, 1, None))), text)
    if "mem" not in change:
        refused(qb.load().ql_attn_forward_appended(*c.args(), ctypes.byref(a)), text)


def test_sparse_list_must_be_aligned():
    c = Cache(lens=(100, 0, 0, 0))
    refused(qb.load().ql_attn_forward_sparse(*c.args(), ctypes.byref(attn_args()),
                                             ctypes.byref(qm.SparseArgs(4, 1, 1, P + 2))),
            "aligned")


def test_unknown_cache_types_are_refused():
    h = ctypes.c_void_p()
    for dtype, text in ((5, "unknown KV cache dtype"), (-1, "unknown KV cache dtype")):
        cfg = qb.KvConfig(1, 64, 1, 64, dtype, 64, 1, 0)
        refused(qb.load().ql_kv_create(ctypes.byref(Ctx()), ctypes.byref(cfg), ctypes.byref(h)),
                text)
    for dtype, name in ((qb.Q8_0, "Q8_0"), (qb.Q4_0, "Q4_0")):
        cfg = qb.KvConfig(1, 64, 1, 48, dtype, 64, 1, 0)
        refused(qb.load().ql_kv_create(ctypes.byref(Ctx()), ctypes.byref(cfg), ctypes.byref(h)),
                f"{name} storage needs head_dim divisible by 32")


def test_python_calls_check_their_lists():
    kv = object.__new__(qb.KvCache)
    kv._h = None
    with pytest.raises(qb.QllamaError, match="length"):
        kv.truncate([0, 1], [3])
    with pytest.raises(qb.QllamaError, match="position"):
        qb._ragged(None, [0], [1, 2])
    with pytest.raises(qb.QllamaError, match="sequence"):
        qb._ragged([0], [0, 0], [1, 2])
    batch, total, rows, keep = qb._ragged([3, 1], [10, 0], [2, 5])
    assert (batch, total) == (2, 7)
    assert [list(x) for x in keep] == [[3, 1], [10, 0], [2, 5]]
    assert list(rows) == [x.buffer_info()[0] for x in keep]
    assert list(qb._ragged(None, [0] * 3, [1] * 3)[3][0]) == [0, 1, 2]


@pytest.mark.parametrize("positions", [range(3, 9), range(0), range(9, 3, -2), [4, 5, 7]])
def test_positions(positions):
    got = qb._positions(positions)
    assert got.dtype == "int32" and got.flags.c_contiguous and list(got) == list(positions)
