"""Refusals of the decode-step operators (ql_rms_norm, ql_q4_*, ql_linear_q4,
ql_verify_drafts, ql_llama_quantize): every argument is checked before any
device work, so a zeroed stand-in for the context serves, without a device."""
import ctypes

import pytest

import qllama_b200 as qb
from qllama_b200 import model as qm

BUF = ctypes.create_string_buffer(1 << 12)
P = (ctypes.addressof(BUF) + 255) // 256 * 256  # an aligned address that is never read


class Ctx(ctypes.Structure):  # the head of ql_ctx: a device number, then pointers
    _fields_ = [("device", ctypes.c_int), ("num_sms", ctypes.c_int),
                ("rest", ctypes.c_void_p * 16)]


class Q4(ctypes.Structure):  # the head of ql_q4
    _fields_ = [("ctx", ctypes.c_void_p), ("n", ctypes.c_int), ("k", ctypes.c_int),
                ("group", ctypes.c_int), ("tiles", ctypes.c_int), ("chunks", ctypes.c_int),
                ("rest", ctypes.c_void_p * 4)]


CTX = Ctx()


def q4(n=48, k=64, group=32):
    return Q4(ctypes.addressof(CTX), n, k, group, (n + 15) // 16, (k + 63) // 64)


def refused(rc, text, code=qb.ERR_INVALID):
    assert rc == code
    assert text in qb.load().ql_last_error().decode()


NORM = dict(rows=2, hidden=64, in_dtype=qb.F32, weight_dtype=qb.F32, out_dtype=qb.F32, eps=1e-5,
            x=P, weight=P + 512, out=P)


@pytest.mark.parametrize("change, text", [
    (dict(rows=-1), "negative"), (dict(hidden=0), "positive"), (dict(in_dtype=qb.Q8_0), "types"),
    (dict(weight_dtype=7), "types"), (dict(out_dtype=4), "types"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(out_dtype=qb.Q8_0, hidden=80, out_scale=P), "divisible"),
    (dict(sum_out=P), "residual"), (dict(x_stride=63), "stride"), (dict(x_stride=-64), "stride"),
    (dict(residual=P, residual_stride=8), "stride"), (dict(x=None), "NULL"),
    (dict(weight=None), "NULL"), (dict(out=None), "NULL"), (dict(out_dtype=qb.Q8_0), "NULL"),
    (dict(x=P + 2), "aligned"), (dict(residual=P + 1), "aligned"), (dict(out=P + 2), "aligned"),
    (dict(out_dtype=qb.Q8_0, out_scale=P + 1), "aligned"),
    (dict(out=P + 4), "overlaps"), (dict(residual=P, sum_out=P), "overlaps"),
    (dict(x_stride=128), "overlaps"), (dict(out=P + 1024, weight=P + 1200), "overlaps"),
    (dict(in_dtype=qb.F16), "overlaps"),
    (dict(out_dtype=qb.Q8_0, out=P + 1024, out_scale=P + 1024), "overlaps"),
    (dict(residual=P, sum_out=P + 1024, out=P + 1024), "overlaps")])
def test_norm_refusals(change, text):
    a = qm.NormArgs(**{**NORM, **change})
    refused(qb.load().ql_rms_norm(ctypes.byref(CTX), ctypes.byref(a)), text)


def test_norm_of_no_rows_is_a_no_op():
    a = qm.NormArgs(**{**NORM, "rows": 0, "x": None, "out": None})
    assert qb.load().ql_rms_norm(ctypes.byref(CTX), ctypes.byref(a)) == qb.OK


@pytest.mark.parametrize("n, k, group, text", [
    (0, 64, 32, "positive"), (8, -64, 32, "positive"), (8, 64, 16, "group"),
    (8, 96, 64, "divisible"), (8, 32, 128, "divisible")])
def test_weight_refusals(n, k, group, text):
    h = ctypes.c_void_p()
    refused(qb.load().ql_q4_create(ctypes.byref(CTX), n, k, group, ctypes.byref(h)), text)
    assert not h.value


def test_sizes_beyond_the_kernels_are_refused():
    L, h = qb.load(), ctypes.c_void_p()
    refused(L.ql_q4_create(ctypes.byref(CTX), 8, (1 << 24) + 32, 32, ctypes.byref(h)), "too large",
            qb.ERR_UNSUPPORTED)
    a = qm.NormArgs(**{**NORM, "hidden": (1 << 30) + 32})
    refused(L.ql_rms_norm(ctypes.byref(CTX), ctypes.byref(a)), "too large", qb.ERR_UNSUPPORTED)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32", "int16"])
def test_scales_of_another_type_are_refused(dtype):
    torch = pytest.importorskip("torch")
    q = object.__new__(qm.Q4Weight)
    with pytest.raises(qb.QllamaError, match="scales must be float16"):
        q._buffer(torch.zeros(4, 2, dtype=getattr(torch, dtype)), "float16", "scales")
    p, mem, keep = q._buffer(torch.zeros(4, 2, dtype=torch.float16), "float16", "scales")
    assert p == keep.data_ptr() and mem == qb.MEM_HOST


@pytest.mark.parametrize("kind", ["bytes", "numpy", "torch", "torch, every other byte"])
def test_gguf_blocks_in_host_memory(monkeypatch, kind):
    """Blocks as bytes, an array or a CPU tensor reach the library with their byte count."""
    torch = pytest.importorskip("torch")
    raw = torch.arange(2 * 3 * 2 * 18, dtype=torch.uint8).view(3, -1)
    blocks = raw[:, ::2] if "every" in kind else raw[:, :36].contiguous()
    plain = blocks.numpy().tobytes()
    blocks = {"bytes": plain, "numpy": blocks.numpy()}.get(kind, blocks)

    class Library:
        got = None

        def ql_q4_create(self, *args):
            return 0

        def ql_q4_set_blocks(self, handle, p, n, mem):
            Library.got = (ctypes.string_at(p, n), mem)
            return 0

    monkeypatch.setattr(qb, "load", Library)
    monkeypatch.setattr(CTX, "_h", None, raising=False)
    qm.Q4Weight.from_gguf(CTX, blocks, 3, 64)
    assert Library.got == (plain, qb.MEM_HOST)


def test_weight_value_refusals():
    L, w, w64 = qb.load(), q4(), q4(group=64)
    refused(L.ql_q4_set(ctypes.byref(w), None, P, 0), "NULL")
    refused(L.ql_q4_set(ctypes.byref(w), P, P, 2), "memory kind")
    refused(L.ql_q4_set(ctypes.byref(w), P, P + 1, 0), "aligned")
    refused(L.ql_q4_set_blocks(ctypes.byref(w64), P, 48 * 2 * 18, 0), "group of 32")
    refused(L.ql_q4_set_blocks(ctypes.byref(w), P, 48 * 2 * 18 - 1, 0), "bytes")
    refused(L.ql_q4_quantize(ctypes.byref(w), P, qb.Q8_0, 0, 0), "type")
    refused(L.ql_q4_quantize(ctypes.byref(w), P, qb.F32, 32, 0), "stride")
    refused(L.ql_q4_quantize(ctypes.byref(w), P + 2, qb.F32, 0, 0), "aligned")
    refused(L.ql_q4_get(None, P, P, 0), "NULL")
    refused(L.ql_q4_shape(None, None, None, None), "NULL")
    assert L.ql_q4_destroy(None) == qb.OK


LINEAR = dict(rows=2, in_dtype=qb.F32, out_dtype=qb.F32, x=P, y=P)


@pytest.mark.parametrize("change, text", [
    (dict(rows=-1), "negative"), (dict(in_dtype=5), "types"), (dict(out_dtype=qb.Q8_0), "types"),
    (dict(x_stride=63), "stride"), (dict(y_stride=47), "stride"), (dict(x=None), "NULL"),
    (dict(y=None), "NULL"), (dict(in_dtype=qb.Q8_0), "NULL"), (dict(x=P + 2), "aligned"),
    (dict(y=P + 1), "aligned"), (dict(in_dtype=qb.Q8_0, x_scale=P + 1), "aligned")])
def test_linear_refusals(change, text):
    a = qm.LinearArgs(**{**LINEAR, **change})
    w = q4()
    refused(qb.load().ql_linear_q4(ctypes.byref(CTX), ctypes.byref(w), ctypes.byref(a)), text)


def test_linear_refuses_another_device_and_takes_no_rows():
    other, w = Ctx(device=1), q4()
    a = qm.LinearArgs(**LINEAR)
    refused(qb.load().ql_linear_q4(ctypes.byref(other), ctypes.byref(w), ctypes.byref(a)),
            "device")
    a.rows = 0
    assert qb.load().ql_linear_q4(ctypes.byref(CTX), ctypes.byref(w), ctypes.byref(a)) == qb.OK


VERIFY = dict(batch=2, drafts=3, vocab=50, dtype=qb.F32, form=qm.VERIFY_LOGITS, temperature=1.0,
              target=P, draft=P, draft_ids=P, uniforms=P, tokens=P, accepted=P)


@pytest.mark.parametrize("change, text, code", [
    (dict(batch=-1), "negative", 1), (dict(drafts=-1), "drafts", 1),
    (dict(drafts=qm.VERIFY_MAX_DRAFTS + 1), "drafts", 1), (dict(vocab=0), "non-empty", 1),
    (dict(vocab=(1 << 22) + 1), "exceeds", qb.ERR_UNSUPPORTED), (dict(dtype=qb.Q8_0), "type", 1),
    (dict(form=2), "form", 1), (dict(temperature=float("inf")), "temperature", 1),
    (dict(target_stride=49), "stride", 1), (dict(draft_stride=-50), "stride", 1),
    (dict(target=None), "NULL", 1), (dict(draft_ids=None), "NULL", 1),
    (dict(uniforms=None), "NULL", 1), (dict(tokens=None), "NULL", 1),
    (dict(accepted=None), "NULL", 1), (dict(form=qm.VERIFY_PROBS, uniforms=None), "NULL", 1),
    (dict(target=P + 2), "aligned", 1), (dict(uniforms=P + 4), "aligned", 1),
    (dict(n_draft=P + 2), "aligned", 1), (dict(tokens=P + 1), "aligned", 1)])
def test_verify_refusals(change, text, code):
    a = qm.VerifyArgs(**{**VERIFY, **change})
    refused(qb.load().ql_verify_drafts(ctypes.byref(CTX), ctypes.byref(a)), text, code)


@pytest.mark.parametrize("T, refuse", [(1e-39, True), (1e-45, True), (1.2e-38, False),
                                       (0.0, False), (-1e-39, False)])
def test_verify_temperatures_below_the_normal_range(T, refuse):
    """(A batch of no sequences shows which ones pass the checks.)"""
    a = qm.VerifyArgs(**{**VERIFY, "batch": 0, "temperature": T})
    rc = qb.load().ql_verify_drafts(ctypes.byref(CTX), ctypes.byref(a))
    if refuse:
        refused(rc, "temperature", qb.ERR_UNSUPPORTED)
    else:
        assert rc == qb.OK


def test_verify_of_no_sequences_is_a_no_op():
    a = qm.VerifyArgs(**{**VERIFY, "batch": 0, "target": None})
    assert qb.load().ql_verify_drafts(ctypes.byref(CTX), ctypes.byref(a)) == qb.OK


@pytest.mark.parametrize("current, own, ordered", [(7, 7, False), (0, 0, False), (7, None, True),
                                                   (0, None, True), (7, 9, True)])
def test_calls_are_ordered_with_the_current_stream(monkeypatch, current, own, ordered):
    """Around a call whose context has another stream than torch's current one: the context
    waits for that stream before it, and that stream for the context after it."""
    class Context:
        device, _stream, _h = 0, own, 5

    class Library:
        log = []

        def __getattr__(self, name):
            def call(handle, *args):
                self.log.append(name if name == "ql_q4_set" else (name, handle, *args))
                return 0
            return call

    lib = Library()
    monkeypatch.setattr(qm, "_L", lib)
    monkeypatch.setattr(qm, "_current", lambda device: current)
    w = object.__new__(qm.Q4Weight)
    w.ctx, w._h = Context(), 6
    w._write(qb.MEM_DEVICE, lib.ql_q4_set, P, P, 0)
    w._h = None
    around = [("ql_ctx_wait_stream", 5, current), "ql_q4_set", ("ql_ctx_join_stream", 5, current)]
    assert lib.log == (around if ordered else ["ql_q4_set"])


def test_a_contexts_stream_as_torch_names_it(monkeypatch):
    class Library:
        def ql_ctx_set_stream(self, handle, stream):
            return 0

    monkeypatch.setattr(qb, "load", Library)
    c = object.__new__(qb.Context)
    c._h = None
    for handle, name in ((None, None), (0, None), (1, 0), (0x7f00, 0x7f00)):
        c.set_stream(handle)
        assert c._stream == name


def test_null_arguments():
    L = qb.load()
    for rc in (L.ql_rms_norm(None, None), L.ql_q4_create(None, 1, 32, 32, None),
               L.ql_linear_q4(None, None, None), L.ql_verify_drafts(None, None),
               L.ql_llama_quantize(None, 32)):
        refused(rc, "NULL")
