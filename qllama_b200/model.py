"""Python view of include/qllama_model.h: the device Llama model, GGUF loading
and the device sampler.

Mirrors the reference's interface for these pieces:

* ``Llama``            -- Transformer (src/transformer/transformer.rs):
  ``from_gguf`` / ``forward_with_cache`` / the weights by GGUF name;
* ``Llama.generate``   -- generate() of src/main.rs:387-429;
* ``SamplerConfig`` / ``sample`` -- src/sampler/sampler.rs (the uniform draw
  is passed in: the reference draws it from its seeded generator).

and, with no counterpart in the reference, attention over rows that are in the cache
already, whole (``attention_forward_appended``) or over the blocks that a bound on
their scores selects (``attention_forward_sparse``), and the pieces of a decode step
on 4-bit weights with drafted tokens:

* ``rms_norm``         -- RMSNorm with the residual's addition, plain or Q8_0 out;
* ``Q4Weight`` / ``linear_q4`` -- 4-bit weight matrices and products of a few
  rows with them (``Llama.quantize`` moves a model onto them);
* ``verify_drafts``    -- speculative sampling's acceptance and next token.

These take CUDA tensors and queue their work on the context's stream
(``Context.set_stream``).  Where torch's current stream is another one, they make
the context's stream wait for it first and it for the context's afterwards, so
that tensors of the current stream may be passed, used and dropped as with any
torch call; tensors of a third stream have to be ordered by the caller.
"""
from __future__ import annotations

import ctypes

import numpy as np


class LlamaConfig(ctypes.Structure):
    _fields_ = [("vocab_size", ctypes.c_int32), ("hidden_size", ctypes.c_int32),
                ("intermediate_size", ctypes.c_int32), ("num_heads", ctypes.c_int32),
                ("num_kv_heads", ctypes.c_int32), ("num_layers", ctypes.c_int32),
                ("max_position_embeddings", ctypes.c_int32), ("rms_norm_eps", ctypes.c_float),
                ("rope_theta", ctypes.c_float)]

    @property
    def head_dim(self) -> int:
        return self.hidden_size // self.num_heads


class SamplerConfig(ctypes.Structure):
    """SamplerConfig (sampler.rs:15-25); temperature <= 0 is greedy."""
    _fields_ = [("temperature", ctypes.c_float), ("top_k", ctypes.c_int32),
                ("top_p", ctypes.c_float), ("repeat_penalty", ctypes.c_float)]


class NormArgs(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int32), ("hidden", ctypes.c_int32),
                ("in_dtype", ctypes.c_int32), ("weight_dtype", ctypes.c_int32),
                ("out_dtype", ctypes.c_int32), ("eps", ctypes.c_float),
                ("x_stride", ctypes.c_int64), ("residual_stride", ctypes.c_int64),
                ("x", ctypes.c_void_p), ("residual", ctypes.c_void_p),
                ("weight", ctypes.c_void_p), ("sum_out", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("out_scale", ctypes.c_void_p)]


class SparseArgs(ctypes.Structure):
    _fields_ = [("blocks", ctypes.c_int32), ("first", ctypes.c_int32),
                ("last", ctypes.c_int32), ("selected", ctypes.c_void_p)]


class LinearArgs(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int32), ("in_dtype", ctypes.c_int32),
                ("out_dtype", ctypes.c_int32), ("x_stride", ctypes.c_int64),
                ("y_stride", ctypes.c_int64), ("x", ctypes.c_void_p),
                ("x_scale", ctypes.c_void_p), ("y", ctypes.c_void_p)]


class VerifyArgs(ctypes.Structure):
    _fields_ = [("batch", ctypes.c_int32), ("drafts", ctypes.c_int32),
                ("vocab", ctypes.c_int32), ("dtype", ctypes.c_int32), ("form", ctypes.c_int32),
                ("temperature", ctypes.c_float), ("target_stride", ctypes.c_int64),
                ("draft_stride", ctypes.c_int64), ("target", ctypes.c_void_p),
                ("draft", ctypes.c_void_p), ("draft_ids", ctypes.c_void_p),
                ("n_draft", ctypes.c_void_p), ("uniforms", ctypes.c_void_p),
                ("tokens", ctypes.c_void_p), ("accepted", ctypes.c_void_p)]


GREEDY = (0.0, 0, 1.0, 1.0)
VERIFY_LOGITS, VERIFY_PROBS, VERIFY_MAX_DRAFTS = 0, 1, 31
_Q8_0 = 3  # the package's Q8_0


def bind(L: ctypes.CDLL) -> None:
    vp, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
    i32p = ctypes.POINTER(i32)
    L.ql_llama_create.argtypes = [vp, ctypes.POINTER(LlamaConfig), ctypes.POINTER(vp)]
    L.ql_llama_destroy.argtypes = [vp]
    L.ql_llama_get_config.argtypes = [vp, ctypes.POINTER(LlamaConfig)]
    L.ql_llama_set_tensor.argtypes = [vp, ctypes.c_char_p, vp, i64]
    L.ql_llama_load_gguf.argtypes = [vp, ctypes.c_char_p, ctypes.POINTER(vp)]
    L.ql_llama_forward.argtypes = [vp, vp, i32, i32p, i32, i64, vp, i32]
    L.ql_sample.argtypes = [vp, vp, i32, vp, i32, ctypes.POINTER(SamplerConfig), ctypes.c_double,
                            vp]
    L.ql_qkv_rope_append.argtypes = [vp, vp, ctypes.c_void_p, vp, i32, vp, vp]
    L.ql_attn_forward_appended.argtypes = [vp, vp, ctypes.c_void_p]
    L.ql_attn_forward_sparse.argtypes = [vp, vp, ctypes.c_void_p, ctypes.POINTER(SparseArgs)]
    L.ql_llama_generate.argtypes = [vp, vp, i32, i32p, i32, i32, i32,
                                    ctypes.POINTER(SamplerConfig),
                                    ctypes.POINTER(ctypes.c_double), i32p, i32p]
    L.ql_rms_norm.argtypes = [vp, ctypes.POINTER(NormArgs)]
    L.ql_q4_create.argtypes = [vp, i32, i32, i32, ctypes.POINTER(vp)]
    L.ql_q4_destroy.argtypes = [vp]
    L.ql_q4_shape.argtypes = [vp, i32p, i32p, i32p]
    L.ql_q4_set.argtypes = [vp, vp, vp, i32]
    L.ql_q4_set_blocks.argtypes = [vp, vp, i64, i32]
    L.ql_q4_quantize.argtypes = [vp, vp, i32, i64, i32]
    L.ql_q4_get.argtypes = [vp, vp, vp, i32]
    L.ql_linear_q4.argtypes = [vp, vp, ctypes.POINTER(LinearArgs)]
    L.ql_llama_quantize.argtypes = [vp, i32]
    L.ql_verify_drafts.argtypes = [vp, ctypes.POINTER(VerifyArgs)]


def _qb():
    import qllama_b200 as qb

    return qb


class Llama:
    """A Llama model on one device (ql_llama)."""

    def __init__(self, ctx, config: LlamaConfig | None = None, handle=None):
        qb = _qb()
        self.ctx = ctx
        if handle is None:
            h = ctypes.c_void_p()
            qb._check(qb.load().ql_llama_create(ctx._h, ctypes.byref(config), ctypes.byref(h)))
            handle = h
        self._h = handle
        cfg = LlamaConfig()
        qb._check(qb.load().ql_llama_get_config(self._h, ctypes.byref(cfg)))
        self.config = cfg

    @classmethod
    def from_gguf(cls, ctx, path: str) -> "Llama":
        """GgufFile::from_path + Transformer::from_gguf."""
        qb = _qb()
        h = ctypes.c_void_p()
        qb._check(qb.load().ql_llama_load_gguf(ctx._h, path.encode(), ctypes.byref(h)))
        return cls(ctx, handle=h)

    def set_tensor(self, name: str, data) -> None:
        """One weight by GGUF name, in the reference's [out, in] layout (f32)."""
        a = np.ascontiguousarray(data, dtype=np.float32)
        qb = _qb()
        qb._check(qb.load().ql_llama_set_tensor(self._h, name.encode(), a.ctypes.data, a.size))

    def quantize(self, group: int = 32) -> None:
        """Projections and lm_head to 4-bit weights of `group` (ql_llama_quantize)."""
        qb = _qb()
        qb._check(qb.load().ql_llama_quantize(self._h, group))

    def kv_cache(self, max_batch: int = 1, dtype: str = "f32"):
        """KvCache::new(num_layers, max_position_embeddings, num_kv_heads, head_dim)."""
        c = self.config
        return _qb().KvCache(self.ctx, c.num_layers, c.max_position_embeddings, c.num_kv_heads,
                             c.head_dim, dtype, 64, max_batch)

    def forward_with_cache(self, ids, start_pos: int, kv, seq: int = 0) -> np.ndarray:
        """Transformer::forward_with_cache: logits [n, vocab] (host f32)."""
        qb = _qb()
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        out = np.empty((ids.size, self.config.vocab_size), np.float32)
        qb._check(qb.load().ql_llama_forward(self._h, kv._h, seq,
                                             ids.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)),
                                             ids.size, start_pos, out.ctypes.data, qb.MEM_HOST))
        return out

    def generate(self, kv, prompt, steps: int, sampler=GREEDY, uniforms=None, eos_id: int = -1,
                 seq: int = 0) -> list[int]:
        """generate() (main.rs:387-429) on the device; `uniforms`: one draw per step."""
        qb = _qb()
        prompt = np.ascontiguousarray(prompt, dtype=np.int32)
        cfg = SamplerConfig(*sampler)
        out = np.zeros(max(1, steps), np.int32)
        n = ctypes.c_int32()
        u = None
        if uniforms is not None:
            uu = np.ascontiguousarray(uniforms, dtype=np.float64)
            u = uu.ctypes.data_as(ctypes.POINTER(ctypes.c_double))
        qb._check(qb.load().ql_llama_generate(
            self._h, kv._h, seq, prompt.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)),
            prompt.size, steps, eos_id, ctypes.byref(cfg), u,
            out.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), ctypes.byref(n)))
        return out[:n.value].tolist()

    def close(self) -> None:
        if getattr(self, "_h", None):
            _qb().load().ql_llama_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # interpreter shutdown: the library may already be gone
            pass


def sample(ctx, logits, context, sampler, r: float) -> int:
    """Sampler::sample_slice on the device: logits and context are CUDA tensors
    (f32 / int32); returns the token id (synchronises the context)."""
    import torch

    qb = _qb()
    tok = torch.full((1,), -2, dtype=torch.int32, device=logits.device)
    torch.cuda.synchronize(logits.device)  # inputs and tok are written on torch's stream
    cfg = SamplerConfig(*sampler)
    ctxp = context.data_ptr() if context is not None and context.numel() else None
    n = int(context.numel()) if context is not None else 0
    qb._check(qb.load().ql_sample(ctx._h, logits.data_ptr(), int(logits.numel()), ctxp, n,
                                  ctypes.byref(cfg), float(r), tok.data_ptr()))
    ctx.synchronize()
    return int(tok.item())


def qkv_rope_append(kv, layer: int, x, wqkv_t, start_pos, num_heads: int, num_kv_heads: int,
                    head_dim: int, rope_theta: float, seq_ids=None):
    """ql_qkv_rope_append: x [batch, new_len, in_features] and the fused
    transposed weight [in_features, (Hq + 2 Hkv) * hd] as f32 CUDA tensors;
    returns the rotated queries [batch, new_len, Hq, hd] (K/V go to the cache)."""
    import torch

    qb = _qb()
    batch, new_len, K = (int(v) for v in x.shape)
    q_rot = torch.empty(batch, new_len, num_heads, head_dim, dtype=torch.float32, device=x.device)
    starts = np.atleast_1d(np.asarray(start_pos, dtype=np.int64))
    if starts.size == 1 and batch > 1:
        starts = np.repeat(starts, batch)
    seqs = np.arange(batch, dtype=np.int32) if seq_ids is None else np.asarray(seq_ids, np.int32)
    args = qb.AttnArgs(layer, batch, new_len, seqs.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)),
                       starts.ctypes.data_as(ctypes.POINTER(ctypes.c_int64)), num_heads,
                       num_kv_heads, head_dim, rope_theta, qb.F32, qb.F32, qb.MEM_DEVICE,
                       None, None, None, None)
    qb._check(qb.load().ql_qkv_rope_append(kv.ctx._h, kv._h, ctypes.byref(args),
                                           x.contiguous().data_ptr(), K,
                                           wqkv_t.contiguous().data_ptr(), q_rot.data_ptr()))
    return q_rot


_first = {}  # batch -> the sequences 0 .. batch - 1 (the library only reads them)


def _numbers(x, batch, kind):
    """A C array of `batch` numbers: that many, or one for all, in any form that numpy takes;
    None if there are others."""
    if type(x) is int:
        return (kind * batch)(*((x,) * batch))
    if type(x) in (list, tuple, range) and len(x) == batch:
        try:
            return (kind * batch)(*x)
        except TypeError:  # not whole numbers
            pass
    x = np.asarray(x, dtype=np.int64).ravel()
    if x.size not in (1, batch):
        return None
    return (kind * batch)(*np.broadcast_to(x, batch).tolist())


def _appended_args(kv, layer, q_rot, start_pos, num_heads, num_kv_heads, head_dim, rope_theta,
                   seq_ids, out, out_dtype):
    """(AttnArgs, out) of attention over rows that are in the cache."""
    qb = _qb()
    shape = q_rot.shape
    if len(shape) < 3 or not q_rot.is_contiguous() or \
            q_rot.numel() != shape[0] * shape[1] * num_heads * head_dim:
        raise _invalid(f"q_rot must be contiguous [batch, new_len, {num_heads}, {head_dim}], got "
                       f"{tuple(shape)}")
    batch, new_len = shape[0], shape[1]
    t = out.dtype if out is not None else _named_type(out_dtype or "f32")
    out = _output(kv.ctx, out, (batch, new_len, num_heads * head_dim), t, "out")
    starts = _numbers(start_pos, batch, ctypes.c_int64)
    if seq_ids is not None:
        seqs = _numbers(seq_ids, batch, ctypes.c_int32)
    elif (seqs := _first.get(batch)) is None:
        seqs = _first[batch] = (ctypes.c_int32 * batch)(*range(batch))
    if starts is None or seqs is None:
        raise _invalid(f"one position and one sequence for each of {batch} rows of q_rot")
    dev = kv.ctx.device
    args = qb.AttnArgs(layer, batch, new_len, seqs, starts, num_heads, num_kv_heads, head_dim,
                       rope_theta, _float_code(q_rot, "q_rot"), _float_code(out, "out"),
                       qb.MEM_DEVICE, _on(dev, q_rot, "q_rot"), None, None, _on(dev, out, "out"))
    return args, out


def attention_forward_appended(kv, layer: int, q_rot, start_pos, num_heads: int,
                               num_kv_heads: int, head_dim: int, rope_theta: float,
                               seq_ids=None, out_dtype: str | None = None, out=None):
    """ql_attn_forward_appended over the rows that qkv_rope_append or KvCache.append
    wrote: q_rot [batch, new_len, heads, head_dim] f32, f16 or bf16; returns
    [batch, new_len, heads * head_dim] (`out`, or a new tensor of out_dtype, default f32)."""
    L = _L or _start()
    args, out = _appended_args(kv, layer, q_rot, start_pos, num_heads, num_kv_heads, head_dim,
                               rope_theta, seq_ids, out, out_dtype)
    side = _fork(kv.ctx)
    rc = L.ql_attn_forward_appended(kv.ctx._h, kv._h, ctypes.byref(args))
    if rc:
        _raise(rc)
    if side is not None:
        _join(kv.ctx, side)
    return out


def attention_forward_sparse(kv, layer: int, q_rot, start_pos, num_heads: int,
                             num_kv_heads: int, head_dim: int, blocks: int, first: int = 1,
                             last: int = 1, seq_ids=None, out_dtype: str | None = None, out=None,
                             selected=None):
    """attention_forward_appended over `blocks` blocks of 64 positions for each token and
    KV head: the first `first`, the newest `last` and those whose keys can score highest
    (ql_attn_forward_sparse).  Returns (out, selected): selected, int32
    [batch, new_len, num_kv_heads, blocks] or None, receives the blocks' numbers in
    ascending order, -1 behind them.  A layer's first call allocates its blocks' bounds: make
    it before a capture; after rows that a captured call has scored were truncated and
    appended anew, make an uncaptured call before its replay."""
    import torch

    L = _L or _start()
    args, out = _appended_args(kv, layer, q_rot, start_pos, num_heads, num_kv_heads, head_dim,
                               1.0, seq_ids, out, out_dtype)
    sp = None
    if selected is not None:
        _output(kv.ctx, selected, (args.batch, args.new_len, num_kv_heads, blocks), torch.int32,
                "selected")
        sp = _on(kv.ctx.device, selected, "selected")
    sparse = SparseArgs(blocks, first, last, sp)
    side = _fork(kv.ctx)
    rc = L.ql_attn_forward_sparse(kv.ctx._h, kv._h, ctypes.byref(args), ctypes.byref(sparse))
    if rc:
        _raise(rc)
    if side is not None:
        _join(kv.ctx, side)
    return out, selected


# ------------------------------------ 4-bit decode step and drafted tokens --

# The calls below are a few microseconds of GPU work each, so their own path is
# kept short: these are filled at the first call.
_codes = {}  # torch dtype -> QL element type
_L = None    # the library
_current = None  # a device's current stream in torch, as a handle


def _start():
    global _L, _current
    import torch

    qb = _qb()
    # (torch.cuda.current_stream makes an object of it: a microsecond and more a call)
    _current = torch._C._cuda_getCurrentRawStream
    _codes.update({torch.float32: qb.F32, torch.float16: qb.F16, torch.bfloat16: qb.BF16})
    _L = qb.load()
    return _L


def _invalid(message: str):
    qb = _qb()
    return qb.QllamaError(qb.ERR_INVALID, message)


def _raise(rc: int):
    raise _qb().QllamaError(rc, _L.ql_last_error().decode())


def _fork(ctx):
    """Where torch's current stream is not the context's: the context waits for it.
    Returns its handle for _join, or None."""
    s = _current(ctx.device)
    if s == ctx._stream:
        return None
    if rc := _L.ql_ctx_wait_stream(ctx._h, s):
        _raise(rc)
    return s


def _join(ctx, s) -> None:
    """The current stream waits for the call: its tensors may be used, or dropped and
    their memory taken by the next ones."""
    if s is not None and (rc := _L.ql_ctx_join_stream(ctx._h, s)):
        _raise(rc)


def _float_code(t, name: str) -> int:
    code = _codes.get(t.dtype)
    if code is None:
        raise _invalid(f"{name}: unsupported element type {t.dtype}")
    return code


def _on(device: int, t, name: str) -> int:
    """The pointer of a tensor on the context's device."""
    if t.get_device() != device:
        raise _invalid(f"{name} is on {t.device}, the context on cuda:{device}")
    return t.data_ptr()


def _stride_of(t, width: int, name: str) -> int:
    """Elements from row to row (0: contiguous) of a tensor [..., width]: a matrix
    whose rows are contiguous, or a contiguous tensor of any rank."""
    if t.is_contiguous():
        return 0
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= width:
        return t.stride(0)
    raise _invalid(f"{name} must have contiguous rows")


def _output(ctx, t, shape, dtype, name: str):
    """A given output checked (contiguous, of that shape and type), or a new one."""
    if t is None:
        import torch

        return torch.empty(shape, dtype=dtype, device=f"cuda:{ctx.device}")
    if t.shape != shape or t.dtype is not dtype or not t.is_contiguous():
        raise _invalid(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")
    return t


def _named_type(name: str):
    import torch

    named = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
    if name not in named:
        raise _invalid(f"unknown element type {name}")
    return named[name]


def rms_norm(ctx, x, weight, eps: float, residual=None, sum_out=None, out=None, scale=None,
             out_dtype: str | None = None):
    """y = s / sqrt(mean(s^2) + eps) * weight over the last dimension, s = x + residual.

    x [..., hidden] (f32, f16 or bf16); residual like x; sum_out receives s (it
    may be x or residual).  out_dtype: None (x's, or out's), "f32", "f16",
    "bf16", or "q8_0", also chosen by giving an int8 `out`.  Returns y, or for
    Q8_0 (int8 values [..., hidden], f16 scales [..., hidden / 32]).
    """
    L = _L or _start()
    shape, dtype, dev = x.shape, x.dtype, ctx.device
    if not shape or not shape[-1]:
        raise _invalid("x needs a last dimension to normalise")
    hidden = shape[-1]
    in_dt = _float_code(x, "x")
    if weight.shape != (hidden,) or not weight.is_contiguous():
        raise _invalid(f"weight must be contiguous [{hidden}], got {tuple(weight.shape)}")
    rs, rp, sp = 0, None, None
    if residual is not None:
        if residual.shape != shape or residual.dtype is not dtype:
            raise _invalid("residual must have x's shape and type")
        rs = _stride_of(residual, hidden, "residual")
        rp = _on(dev, residual, "residual")
    if sum_out is not None:
        sp = _on(dev, _output(ctx, sum_out, shape, dtype, "sum_out"), "sum_out")
    if out_dtype == "q8_0" or scale is not None or (
            out is not None and out_dtype is None and out.dtype not in _codes):
        import torch

        if hidden % 32:
            raise _invalid(f"a Q8_0 output needs hidden divisible by 32, got {hidden}")
        out = _output(ctx, out, shape, torch.int8, "out")
        scale = _output(ctx, scale, shape[:-1] + (hidden // 32,), torch.float16, "scale")
        out_dt, scp = _Q8_0, _on(dev, scale, "scale")
    else:
        t = _named_type(out_dtype) if out_dtype else dtype if out is None else out.dtype
        out = _output(ctx, out, shape, t, "out")
        out_dt, scp = _codes[t], None
    args = NormArgs(
        x.numel() // hidden, hidden, in_dt, _float_code(weight, "weight"), out_dt, eps,
        _stride_of(x, hidden, "x"), rs, _on(dev, x, "x"), rp, _on(dev, weight, "weight"), sp,
        _on(dev, out, "out"), scp)
    side = _fork(ctx)
    rc = L.ql_rms_norm(ctx._h, ctypes.byref(args))
    if rc:
        _raise(rc)
    if side is not None:
        _join(ctx, side)
    return out if scp is None else (out, scale)


class Q4Weight:
    """A 4-bit weight matrix [out_features, in_features] on the device (ql_q4).

    Q4Weight(ctx, codes, scales): codes uint8 [out, in/2] (column 2j in the low
    four bits of byte j), scales f16 [out, in/group]; CUDA tensors or numpy
    arrays.  The group (32, 64 or 128) follows from the shapes.
    """

    def __init__(self, ctx, codes=None, scales=None, *, shape=None):
        qb = _qb()
        self.ctx, self._h = ctx, None
        if shape is None:
            if codes is None or scales is None or len(codes.shape) != 2 or \
                    len(scales.shape) != 2 or codes.shape[0] != scales.shape[0] or \
                    not scales.shape[1] or 2 * codes.shape[1] % scales.shape[1]:
                raise _invalid("codes [out, in/2] and scales [out, in/group] are needed")
            k = 2 * int(codes.shape[1])
            shape = (int(codes.shape[0]), k, k // int(scales.shape[1]))
        self.out_features, self.in_features, self.group = shape
        h = ctypes.c_void_p()
        qb._check(qb.load().ql_q4_create(ctx._h, *shape, ctypes.byref(h)))
        self._h = h
        if codes is not None:
            self.set(codes, scales)

    @classmethod
    def from_dense(cls, ctx, w, group: int = 32) -> "Q4Weight":
        """Quantises a dense [out, in] matrix (f32, f16 or bf16)."""
        qb = _qb()
        if len(w.shape) != 2:
            raise _invalid("a dense weight has two dimensions")
        q = cls(ctx, shape=(int(w.shape[0]), int(w.shape[1]), group))
        p, mem, keep = q._buffer(w, None, "w")
        stride = 0 if mem == qb.MEM_HOST else _stride_of(keep, int(w.shape[1]), "w")
        q._write(mem, qb.load().ql_q4_quantize, p, qb._dtype_code(keep), stride, mem)
        return q

    @classmethod
    def from_gguf(cls, ctx, blocks, out_features: int, in_features: int) -> "Q4Weight":
        """From GGUF Q4_0 blocks (bytes, a numpy uint8 array or a uint8 tensor)."""
        qb = _qb()
        q = cls(ctx, shape=(out_features, in_features, 32))
        if isinstance(blocks, (bytes, bytearray, memoryview)):
            blocks = np.frombuffer(blocks, np.uint8)
        p, mem, keep = q._buffer(blocks, "uint8", "blocks")
        q._write(mem, qb.load().ql_q4_set_blocks, p, int(keep.nbytes), mem)
        return q

    def _write(self, mem: int, call, *args) -> None:
        """One of the calls that write the weight, from tensors of the current stream."""
        qb = _qb()
        side = None
        if mem == qb.MEM_DEVICE:
            _L or _start()
            side = _fork(self.ctx)
        qb._check(call(self._h, *args))
        _join(self.ctx, side)

    def _buffer(self, x, dtype, name: str):
        """(pointer, memory kind, keep-alive) of an array or a CUDA tensor."""
        qb = _qb()
        if dtype and str(x.dtype).split(".")[-1] != dtype:  # bfloat16 ends in float16
            raise _invalid(f"{name} must be {dtype}, got {x.dtype}")
        if not isinstance(x, np.ndarray):
            if not x.is_cuda:
                x = x.contiguous()
                return x.data_ptr(), qb.MEM_HOST, x
            if dtype and not x.is_contiguous():
                raise _invalid(f"{name} must be contiguous")
            return _on(self.ctx.device, x, name), qb.MEM_DEVICE, x
        x = np.ascontiguousarray(x)
        return x.ctypes.data, qb.MEM_HOST, x

    def set(self, codes, scales) -> None:
        """New codes and scales of the same shape (ql_q4_set)."""
        qb = _qb()
        n, k = self.out_features, self.in_features
        if tuple(codes.shape) != (n, k // 2) or tuple(scales.shape) != (n, k // self.group):
            raise _invalid(f"codes and scales must be [{n}, {k // 2}] and "
                           f"[{n}, {k // self.group}]")
        cp, mem, c = self._buffer(codes, "uint8", "codes")
        sp, mem2, s = self._buffer(scales, "float16", "scales")
        if mem != mem2:
            raise _invalid("codes and scales must live in the same memory")
        self._write(mem, qb.load().ql_q4_set, cp, sp, mem)

    def get(self):
        """(codes, scales) as numpy arrays in the constructor's layout."""
        qb = _qb()
        codes = np.empty((self.out_features, self.in_features // 2), np.uint8)
        scales = np.empty((self.out_features, self.in_features // self.group), np.float16)
        qb._check(qb.load().ql_q4_get(self._h, codes.ctypes.data, scales.ctypes.data,
                                      qb.MEM_HOST))
        return codes, scales

    def close(self) -> None:
        if getattr(self, "_h", None):
            _qb().load().ql_q4_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # interpreter shutdown: the library may already be gone
            pass


def linear_q4(weight: Q4Weight, x, x_scale=None, out=None, out_dtype: str | None = None):
    """x W^T of a few rows x [..., in_features] with 4-bit weights (ql_linear_q4).

    x is f32, f16 or bf16, or int8 with x_scale f16 [..., in_features / 32] (the
    Q8_0 output of rms_norm).  The result is [..., out_features] of out_dtype
    (default: out's type, else x's, f32 for Q8_0); `out` may be a matrix with a
    row stride.
    """
    L = _L or _start()
    ctx, k, n, dtype, lead = (weight.ctx, weight.in_features, weight.out_features, x.dtype,
                              x.shape[:-1])
    dev = ctx.device
    if not x.dim() or x.shape[-1] != k:
        raise _invalid(f"x has shape {tuple(x.shape)}, its last dimension must be {k}")
    in_dt = _codes.get(dtype)
    if in_dt is None or x_scale is not None:
        import torch

        if dtype is not torch.int8:
            raise _invalid(f"x: unsupported element type {dtype}" if in_dt is None else
                           "x_scale belongs to int8 x")
        if x_scale is None:
            raise _invalid("int8 x needs x_scale")
        _output(ctx, x_scale, lead + (k // 32,), torch.float16, "x_scale")
        in_dt, scp, dtype = _Q8_0, _on(dev, x_scale, "x_scale"), torch.float32
    else:
        scp = None
    if out_dtype is not None:
        dtype = _named_type(out_dtype)
    elif out is not None:
        dtype = out.dtype
    shape = lead + (n,)
    if out is None:
        import torch

        out, ys = torch.empty(shape, dtype=dtype, device=x.device), 0
    else:
        if out.shape != shape or out.dtype is not dtype:
            raise _invalid(f"out must be {dtype} of shape {tuple(shape)}")
        ys = _stride_of(out, n, "out")
    args = LinearArgs(x.numel() // k, in_dt, _float_code(out, "out"), _stride_of(x, k, "x"), ys,
                      _on(dev, x, "x"), scp, _on(dev, out, "out"))
    side = _fork(ctx)
    rc = L.ql_linear_q4(ctx._h, weight._h, ctypes.byref(args))
    if rc:
        _raise(rc)
    if side is not None:
        _join(ctx, side)
    return out


def verify_drafts(ctx, target, draft, draft_ids, uniforms, temperature: float = 1.0,
                  n_draft=None, probs: bool = False, tokens=None, accepted=None):
    """Speculative sampling's acceptance and next token (ql_verify_drafts).

    target [batch, drafts + 1, vocab] and draft [batch, drafts, vocab] (or None:
    the drafts are certain) hold logits, or probabilities with probs=True;
    draft_ids int32 [batch, drafts]; uniforms f64 [batch, drafts + 1] (None when
    temperature <= 0); n_draft int32 [batch] or None.  Returns (tokens int32
    [batch, drafts + 1], accepted int32 [batch]): the accepted drafts, the new
    token, then -1.
    """
    import torch

    L = _L or _start()
    dev, dtype = ctx.device, target.dtype
    if target.dim() != 3 or target.shape[1] < 1:
        raise _invalid("target must be [batch, drafts + 1, vocab]")
    batch, m, vocab = target.shape
    m -= 1
    dt = _float_code(target, "target")

    def rows(t, count, name):
        if t.shape != (batch, count, vocab) or t.dtype is not dtype:
            raise _invalid(f"{name} must be {dtype} [{batch}, {count}, {vocab}]")
        if t.is_contiguous():
            return 0
        row = t.stride(1) if count > 1 else t.stride(0)
        if (t.stride(2) != 1 and vocab > 1) or row < vocab or (
                batch > 1 and t.stride(0) != count * row):
            raise _invalid(f"{name} must have its rows at one stride")
        return row

    def plain(t, shape, kind, name):
        if t.shape != shape or t.dtype is not kind or not t.is_contiguous():
            raise _invalid(f"{name} must be contiguous {kind} {list(shape)}")
        return _on(dev, t, name)

    ts, ds, dp, ip, up = rows(target, m + 1, "target"), 0, None, None, None
    if draft is not None:
        ds = rows(draft, m, "draft")
        dp = _on(dev, draft, "draft") if m else None
    if m:
        ip = plain(draft_ids, (batch, m), torch.int32, "draft_ids")
    np_ = plain(n_draft, (batch,), torch.int32, "n_draft") if n_draft is not None else None
    if probs or temperature > 0:
        if uniforms is None:
            raise _invalid("sampling needs uniforms")
        up = plain(uniforms, (batch, m + 1), torch.float64, "uniforms")
    tokens = _output(ctx, tokens, (batch, m + 1), torch.int32, "tokens")
    accepted = _output(ctx, accepted, (batch,), torch.int32, "accepted")
    args = VerifyArgs(
        batch, m, vocab, dt, VERIFY_PROBS if probs else VERIFY_LOGITS, temperature, ts, ds,
        _on(dev, target, "target"), dp, ip, np_, up, _on(dev, tokens, "tokens"),
        _on(dev, accepted, "accepted"))
    side = _fork(ctx)
    rc = L.ql_verify_drafts(ctx._h, ctypes.byref(args))
    if rc:
        _raise(rc)
    if side is not None:
        _join(ctx, side)
    return tokens, accepted
