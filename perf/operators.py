"""Cases of the operators around a decode step: RMSNorm with the residual's
addition (plain and Q8_0 outputs), products of a few rows with 4-bit weights,
and the verification of drafted tokens.

`run` computes each operator in its plain form out of elementary torch
operations, or, where `own` is true, through the framework's entry points
(qllama_b200.model: rms_norm, Q4Weight / linear_q4, verify_drafts).
"""
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
Q8_BLOCK = 32


def listed():
    return [
        # the norm before a layer of a 1.1B-shaped model, one token of one sequence
        {"name": "norm one token", "op": "norm", "rows": 1, "hidden": 2048, "dtype": "f32",
         "out": "f32", "residual": True},
        # eight sequences with three drafted tokens each, 70B-shaped, for 8-bit products
        {"name": "norm drafted rows to Q8_0", "op": "norm", "rows": 24, "hidden": 8192,
         "dtype": "bf16", "out": "q8_0", "residual": True},
        # a prompt's rows, a ragged count, 8B-shaped
        {"name": "norm prompt", "op": "norm", "rows": 4099, "hidden": 4096, "dtype": "bf16",
         "out": "bf16", "residual": True},
        # the same prompt's rows for 8-bit products
        {"name": "norm prompt to Q8_0", "op": "norm", "rows": 2048, "hidden": 4096,
         "dtype": "f16", "out": "q8_0", "residual": True},
        # the SwiGLU up projection of the smallest model (288 -> 768), one token
        {"name": "linear smallest", "op": "linear", "rows": 1, "k": 288, "n": 768, "group": 32,
         "dtype": "f32"},
        # gate and up of a 1.1B-shaped model side by side, one token from the Q8_0 norm
        {"name": "linear 1.1B gate+up", "op": "linear", "rows": 1, "k": 2048, "n": 11264,
         "group": 32, "dtype": "q8_0"},
        # gate and up of a 70B-shaped model, one token
        {"name": "linear 70B gate+up", "op": "linear", "rows": 1, "k": 8192, "n": 57344,
         "group": 128, "dtype": "f16"},
        # Q, K and V of a 70B-shaped model, a batch of drafted rows from the Q8_0 norm
        {"name": "linear 70B qkv, drafts", "op": "linear", "rows": 8, "k": 8192, "n": 10240,
         "group": 32, "dtype": "q8_0"},
        # the down projection of a 70B-shaped model, 32 sequences
        {"name": "linear 70B down, batch", "op": "linear", "rows": 32, "k": 28672, "n": 8192,
         "group": 64, "dtype": "bf16"},
        # one sequence with four drafted tokens of a small draft model
        {"name": "verify one sequence", "op": "verify", "batch": 1, "drafts": 4, "vocab": 32000,
         "dtype": "f32", "temperature": 0.8, "form": "logits", "ragged": False},
        # a served batch: sequences come with different numbers of drafted tokens
        {"name": "verify batch", "op": "verify", "batch": 32, "drafts": 7, "vocab": 128000,
         "dtype": "bf16", "temperature": 1.0, "form": "logits", "ragged": True},
        # probabilities that the caller's own filters left, an odd vocabulary
        {"name": "verify probabilities", "op": "verify", "batch": 8, "drafts": 5, "vocab": 50021,
         "dtype": "f32", "temperature": 1.0, "form": "probs", "ragged": False},
    ]


def _log(rng, lo, hi):
    return min(hi, int(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["norm", "linear", "verify"])
    if op == "norm":
        rows = _log(rng, 1, 8192)
        hidden = _log(rng, 64, min(16384, 16_000_000 // rows))
        dtype = rng.choice(["f32", "f16", "bf16"])
        out = rng.choice(["f32", "f16", "bf16", "q8_0"])
        if out == "q8_0":
            hidden -= hidden % Q8_BLOCK
        return {"op": op, "rows": rows, "hidden": hidden, "dtype": dtype, "out": out,
                "residual": rng.random() < 0.7}
    if op == "linear":
        group = rng.choice([32, 64, 128])
        k = _log(rng, 256, 28672) // group * group
        n = _log(rng, 16, min(57344, 460_000_000 // k))
        return {"op": op, "rows": _log(rng, 1, 32), "k": k, "n": n, "group": group,
                "dtype": rng.choice(["f32", "f16", "bf16", "q8_0"])}
    vocab = _log(rng, 1000, 128000)
    form = rng.choice(["logits", "logits", "probs", "lookup", "greedy"])
    return {"op": op, "batch": _log(rng, 1, 32), "drafts": rng.randint(0, 7), "vocab": vocab,
            "dtype": "f32" if form == "probs" else rng.choice(["f32", "f16", "bf16"]),
            "temperature": 0.0 if form == "greedy" else 1.0 if form == "probs" else
            rng.choice([0.6, 0.8, 1.0, 1.3]),
            "form": "logits" if form == "greedy" else form, "ragged": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs --

_ctx = None


def _context():
    """The program's context, on torch's stream (0x1: the legacy default stream)."""
    global _ctx
    if _ctx is None:
        import qllama_b200 as qb

        _ctx = qb.Context(torch.cuda.current_device())
        _ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    return _ctx


def _quantised_rows(x):
    """Q8_0 blocks of f32 rows: int8 [rows, k] and f16 scales [rows, k / 32]."""
    b = x.view(x.shape[0], -1, Q8_BLOCK)
    d = b.abs().amax(-1, keepdim=True) / 127
    q = (b / d).round().clamp(-127, 127).to(torch.int8)
    return q.view_as(x), d.squeeze(-1).half()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    c = dict(case)
    s = {"op": c["op"], "case": c}
    if c["op"] == "norm":
        rows, hidden, t = c["rows"], c["hidden"], TYPES[c["dtype"]]
        # a residual stream has a few channels far above the others
        gain = 1 + 20 * (torch.rand(hidden, device="cuda", generator=g) < 0.01).float()
        s["x"] = normal(rows, hidden).to(t)
        s["residual"] = (normal(rows, hidden) * gain).to(t) if c["residual"] else None
        s["weight"] = (1 + 0.1 * normal(hidden)).to(t)
        s["eps"] = 1e-5
        if own:
            s["ctx"] = _context()
            s["sum"] = torch.empty_like(s["x"]) if c["residual"] else None
            if c["out"] == "q8_0":
                s["out"] = torch.empty(rows, hidden, dtype=torch.int8, device="cuda")
                s["scale"] = torch.empty(rows, hidden // Q8_BLOCK, dtype=torch.float16,
                                         device="cuda")
            else:
                s["out"] = torch.empty(rows, hidden, dtype=TYPES[c["out"]], device="cuda")
                s["scale"] = None
    elif c["op"] == "linear":
        rows, k, n, group = c["rows"], c["k"], c["n"], c["group"]
        # codes of normally distributed weights: 8 stands for zero
        codes = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 26) // k)
        for i in range(0, n, step):
            q = (normal(min(step, n - i), k) * 2.7 + 8).round_().clamp_(0, 15).to(torch.uint8)
            codes[i:i + step] = q[:, 0::2] | (q[:, 1::2] << 4)
        scales = ((0.5 + torch.rand(n, k // group, device="cuda", generator=g)) *
                  (0.35 / k ** 0.5)).half()
        s["codes"], s["scales"], s["group"] = codes, scales, group
        x = normal(rows, k)
        if c["dtype"] == "q8_0":
            s["x"], s["x_scale"] = _quantised_rows(x)
            t = torch.float32
        else:
            t = TYPES[c["dtype"]]
            s["x"], s["x_scale"] = x.to(t), None
        s["out_dtype"] = t
        if own:
            from qllama_b200 import model as qm

            s["weight"] = qm.Q4Weight(_context(), codes, scales)
            s["out"] = torch.empty(rows, n, dtype=t, device="cuda")
    else:
        B, m, V, t = c["batch"], c["drafts"], c["vocab"], TYPES[c["dtype"]]
        # a model's logits are peaked; the draft model's are near the target's
        base = normal(B, m + 1, V)
        target = base * 2.5
        draft = (base[:, :m] * 2.5 + 0.7 * normal(B, m, V))
        if c["form"] == "probs":
            target = _filtered(target)
            draft = _filtered(draft)
        s["target"] = target.to(t)
        s["draft"] = None if c["form"] == "lookup" else draft.to(t)
        if m == 0:
            s["ids"] = torch.zeros(B, 0, dtype=torch.int32, device="cuda")
        elif c["form"] == "lookup":  # drafted from the text: often the likeliest token
            likely = target[:, :m].argmax(-1)
            other = torch.randint(0, V, (B, m), device="cuda", generator=g)
            pick = torch.rand(B, m, device="cuda", generator=g) < 0.7
            s["ids"] = torch.where(pick, likely, other).int()
        elif c["temperature"] == 0:
            s["ids"] = s["draft"].float().argmax(-1).int()
        else:  # drawn from the draft's distribution
            p = s["draft"].float()
            p = p if c["form"] == "probs" else torch.softmax(p / c["temperature"], -1)
            u = torch.rand(B, m, 1, device="cuda", generator=g) * 0.999999
            cum = torch.cumsum(p.double(), -1)
            s["ids"] = torch.searchsorted(cum, u.double() * cum[..., -1:]).squeeze(-1)
            s["ids"] = s["ids"].clamp_(max=V - 1).int()
        s["n_draft"] = (torch.randint(0, m + 1, (B,), device="cuda", generator=g).int()
                        if c["ragged"] else None)
        s["uniforms"] = torch.rand(B, m + 1, dtype=torch.float64, device="cuda", generator=g)
        if own:
            s["ctx"] = _context()
            s["tokens"] = torch.empty(B, m + 1, dtype=torch.int32, device="cuda")
            s["accepted"] = torch.empty(B, dtype=torch.int32, device="cuda")
    return s


def _filtered(logits):
    """Softmax over each row's 200 largest logits, zero elsewhere."""
    k = min(200, logits.shape[-1])
    if logits.shape[1] == 0:
        return logits
    least = logits.topk(k, -1).values[..., -1:]
    return torch.softmax(logits.masked_fill(logits < least, float("-inf")), -1)


# -------------------------------------------------------------- plain forms --

def _norm(s):
    c = s["case"]
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    inv = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + s["eps"])
    y = x * inv * s["weight"].float()
    if c["out"] == "q8_0":
        b = y.view(y.shape[0], -1, Q8_BLOCK)
        d = b.abs().amax(-1, keepdim=True) / 127
        q = torch.where(d > 0, b / d, torch.zeros_like(b))
        q = torch.sign(q) * torch.floor(q.abs() + 0.5)
        y = (q * d.half().float()).half().view_as(y)
    else:
        y = y.to(TYPES[c["out"]])
    return (y, x.to(s["x"].dtype)) if s["residual"] is not None else (y,)


def _linear(s):
    codes, scales, group = s["codes"], s["scales"], s["group"]
    n, k = codes.shape[0], 2 * codes.shape[1]
    w = torch.stack((codes & 15, codes >> 4), -1).view(n, k // group, group)
    w = (w.float() - 8) * scales.float().unsqueeze(-1)
    x = s["x"].float()
    if s["x_scale"] is not None:
        x = (x.view(x.shape[0], -1, Q8_BLOCK) * s["x_scale"].float().unsqueeze(-1)).view_as(x)
    return torch.matmul(x, w.view(n, k).t()).to(s["out_dtype"])


def _verify(s):
    c = s["case"]
    B, m, V = c["batch"], c["drafts"], c["vocab"]
    ids = s["ids"].long()
    # 64 bits: a token is decided by sums over the vocabulary next to a border
    target = s["target"].double()
    count = (s["n_draft"].long() if s["n_draft"] is not None
             else torch.full((B,), m, device="cuda"))
    place = torch.arange(m, device="cuda")
    if c["temperature"] == 0:
        best = target.argmax(-1)
        ok = (best[:, :m] == ids) & (place < count[:, None])
        accepted = ok.long().cumprod(-1).sum(-1)
        token = best.gather(1, accepted[:, None]).squeeze(1)
    else:
        p = target
        if c["form"] != "probs":
            p = torch.exp((p - p.amax(-1, keepdim=True)) / c["temperature"])
            p = p / p.sum(-1, keepdim=True)
        if s["draft"] is None:
            q = torch.zeros(B, m, V, dtype=torch.float64, device="cuda")
            q.scatter_(-1, ids.unsqueeze(-1), 1.0)
        else:
            q = s["draft"].double()
            if c["form"] != "probs" and m:
                q = torch.exp((q - q.amax(-1, keepdim=True)) / c["temperature"])
                q = q / q.sum(-1, keepdim=True)
        px = p[:, :m].gather(-1, ids.unsqueeze(-1)).squeeze(-1)
        qx = q.gather(-1, ids.unsqueeze(-1)).squeeze(-1)
        ok = (s["uniforms"][:, :m] * qx < px) & (place < count[:, None])
        accepted = ok.long().cumprod(-1).sum(-1)
        at = accepted[:, None, None].expand(B, 1, V)
        row = p.gather(1, at).squeeze(1)
        if m:
            less = q.gather(1, at.clamp(max=m - 1)).squeeze(1)
            rejected = (accepted < count)[:, None]
            row = torch.where(rejected, (row - less).clamp(min=0), row)
        u = s["uniforms"].gather(1, count[:, None])
        cum = torch.cumsum(row, -1)
        hit = (row > 0) & (cum >= u * cum[:, -1:])
        token = hit.int().argmax(-1)
    # the accepted drafts, then the new token, then -1
    full = torch.cat((ids, ids.new_zeros(B, 1)), 1)
    places = torch.arange(m + 1, device="cuda")
    tokens = torch.where(places < accepted[:, None], full,
                         torch.where(places == accepted[:, None], token[:, None], -1))
    return tokens.int(), accepted.int()


# --------------------------------------------------------------------- run --

def run(state):
    s, c = state, state["case"]
    if not own:
        return {"norm": _norm, "linear": _linear, "verify": _verify}[s["op"]](s)
    from qllama_b200 import model as qm

    if s["op"] == "norm":
        qm.rms_norm(s["ctx"], s["x"], s["weight"], s["eps"], residual=s["residual"],
                    sum_out=s["sum"], out=s["out"], scale=s["scale"])
        y = s["out"]
        if c["out"] == "q8_0":  # the values that the bytes and scales stand for
            b = y.view(y.shape[0], -1, Q8_BLOCK)
            y = torch.mul(b, s["scale"].unsqueeze(-1)).view_as(y)
        return (y, s["sum"]) if s["sum"] is not None else (y,)
    if s["op"] == "linear":
        return qm.linear_q4(s["weight"], s["x"], s["x_scale"], out=s["out"])
    return qm.verify_drafts(s["ctx"], s["target"], s["draft"], s["ids"], s["uniforms"],
                            temperature=c["temperature"], n_draft=s["n_draft"],
                            probs=c["form"] == "probs", tokens=s["tokens"],
                            accepted=s["accepted"])


def work(case):
    """Each input read once and each output written once."""
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2, "q8_0": 1 + 2 / Q8_BLOCK}
    if c["op"] == "norm":
        e = c["rows"] * c["hidden"]
        moved = e * (size[c["dtype"]] * (3 if c["residual"] else 1) + size[c["out"]])
        return {"bytes": moved + c["hidden"] * size[c["dtype"]], "flops": 5 * e}
    if c["op"] == "linear":
        n, k, rows = c["n"], c["k"], c["rows"]
        out = 4 if c["dtype"] in ("f32", "q8_0") else 2
        return {"bytes": n * k / 2 + n * (k // c["group"]) * 2 + rows * k * size[c["dtype"]] +
                rows * n * out, "flops": 2 * rows * k * n}
    B, m, V, e = c["batch"], c["drafts"], c["vocab"], size[c["dtype"]]
    if c["form"] == "probs":  # the drafted tokens' entries and one row (pair) of each sequence
        return {"bytes": B * V * e * 2, "flops": 3 * B * V}
    # the ragged cases' rows past a sequence's drafts need not be read: half on average
    drafts = m / 2 if c["ragged"] else m
    rows = B * (drafts + 1)
    if c["form"] != "lookup" and c["temperature"] > 0:
        rows += B * drafts
    return {"bytes": rows * V * e, "flops": 4 * rows * V}


# ------------------------------------------------- the definitions, 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "norm":
        v = s["x"].double()
        if s["residual"] is not None:
            v += s["residual"].double()
        norm = torch.linalg.vector_norm(v, dim=1).square_() / c["hidden"]
        y = torch.einsum("rh,r,h->rh", v, (norm + s["eps"]).rsqrt(), s["weight"].double())
        if c["out"] == "q8_0":
            blocks = y.reshape(-1, Q8_BLOCK)
            d = torch.linalg.vector_norm(blocks, ord=float("inf"), dim=1) / 127
            near = torch.trunc(blocks / d.clamp(min=1e-300)[:, None] + 0.5 * blocks.sign())
            y = (near * d.to(torch.float16).double()[:, None]).reshape(y.shape)
        return (y, v) if s["residual"] is not None else (y,)
    if c["op"] == "linear":
        x = s["x"].double()
        if s["x_scale"] is not None:
            x = x * s["x_scale"].double().repeat_interleave(Q8_BLOCK, 1)
        n, k, group = c["n"], c["k"], c["group"]
        y = torch.empty(c["rows"], n, dtype=torch.float64, device="cuda")
        step = max(1, (1 << 26) // k)
        for i in range(0, n, step):
            b = s["codes"][i:i + step].long()
            low, high = b % 16 - 8, b // 16 - 8
            d = s["scales"][i:i + step].double().repeat_interleave(group // 2, 1)
            y[:, i:i + step] = x[:, 0::2] @ (low * d).t() + x[:, 1::2] @ (high * d).t()
        return y
    # sequence by sequence, token by token
    B, m, T = c["batch"], c["drafts"], c["temperature"]
    tokens, accepted = [], []
    for b in range(B):
        count = int(s["n_draft"][b]) if s["n_draft"] is not None else m
        said, left = [], None
        for i in range(count + 1):
            row = s["target"][b, i].double()
            if T == 0:
                token = int((row == row.max()).nonzero()[0])
                said.append(token)
                if i == count or token != int(s["ids"][b, i]):
                    break
                continue
            p = row if c["form"] == "probs" else torch.softmax(row / T, 0)
            left = p
            if i == count:
                break
            x = int(s["ids"][b, i])
            if s["draft"] is None:
                q = torch.zeros_like(p)
                q[x] = 1
            else:
                q = s["draft"][b, i].double()
                q = q if c["form"] == "probs" else torch.softmax(q / T, 0)
            if float(s["uniforms"][b, i]) * float(q[x]) < float(p[x]):
                said.append(x)
                continue
            left = torch.relu(p - q)
            break
        if T != 0:
            at = float(s["uniforms"][b, count]) * float(left.sum())
            some = left.nonzero().squeeze(1)
            sums = left[some].cumsum(0)
            said.append(int(some[min(int((sums < at).sum()), some.numel() - 1)]))
        accepted.append(len(said) - 1)
        tokens.append(said + [-1] * (m + 1 - len(said)))
    return (torch.tensor(tokens, dtype=torch.int32), torch.tensor(accepted, dtype=torch.int32))
