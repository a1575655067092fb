"""Cases and plain forms of the training operators of cresso_b200.ops: the scaled
embedding lookup and its gradient, the norms around a block with its gate and
residual scale, and the distillation from a teacher's top logits.

`own` selects the framework's kernels; otherwise `run` evaluates the formulas with
elementary torch operations in float32.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
VOCAB = 32000  # rows of the embedding table of the 7B-shaped set, its width is 4096


def listed():
    return [
        # one token of a decoding or evaluation loop: latency
        dict(name="gather one token", op="gather", tokens=1, rows=VOCAB, row0=0, width=4096, table="bf16", act="bf16"),
        # a micro-batch of 8 sequences of 2048 tokens, float32 master table, 16-bit activations
        dict(name="gather 8x2048", op="gather", tokens=16384, rows=VOCAB, row0=0, width=4096, table="f32", act="bf16"),
        # one rank's quarter of a row-sharded table, a ragged number of tokens
        dict(name="embedding grad quarter table", op="gather_grad", tokens=2047, rows=8000, row0=8000, width=4096,
             table="bf16", act="bf16"),
        # the dense float32 gradient that the optimizer step reads, for the same micro-batch as above
        dict(name="embedding grad 8x2048", op="gather_grad", tokens=16384, rows=VOCAB, row0=0, width=4096, table="f32",
             act="bf16"),
        # one token between two blocks: latency
        dict(name="norm one token", op="norm", batch=1, length=1, width=4096, res="bf16", act="bf16", gate="channel"),
        # a micro-batch with a float32 residual stream and a learned gate for each channel
        dict(name="norm 8x2048", op="norm", batch=8, length=2048, width=4096, res="f32", act="bf16", gate="channel"),
        # the backward pass of a micro-batch with a 16-bit residual stream
        dict(name="norm grad 8x2048", op="norm_grad", batch=8, length=2048, width=4096, res="bf16", act="bf16",
             gate="channel"),
        # an odd width and a gate for each sample, as a conditioned block has it
        dict(name="norm grad 3x341 odd width", op="norm_grad", batch=3, length=341, width=2050, res="f16", act="f16",
             gate="sample"),
        # evaluation of a short answer against the teacher: few rows
        dict(name="distill loss 16 rows", op="distill_loss", tokens=16, vocab=VOCAB, k=32, act="f32", tau=1.0),
        # evaluation over a vocabulary of odd size, whose rows start at any alignment
        dict(name="distill loss odd vocabulary", op="distill_loss", tokens=1023, vocab=100003, k=17, act="f16", tau=2.0),
        # a training micro-batch: loss and gradient of the logits
        dict(name="distill grad 2x2048", op="distill_grad", tokens=4096, vocab=VOCAB, k=64, act="bf16", tau=2.0),
        # a large vocabulary with float32 logits
        dict(name="distill grad large vocabulary", op="distill_grad", tokens=301, vocab=128259, k=100, act="f32", tau=1.0),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["gather", "gather_grad", "norm", "norm_grad", "distill_loss", "distill_grad"])
    act = rng.choice(["bf16", "f16", "f32"])
    if op in ("gather", "gather_grad"):
        rows = _log_int(rng, 100, VOCAB)
        width = _log_int(rng, 64, 4096)
        if rng.random() < 0.6:
            width = max(64, width // 64 * 64)
        return dict(op=op, tokens=_log_int(rng, 1, 16384), rows=rows, row0=rng.choice([0, 0, rng.randint(0, VOCAB - rows)]),
                    width=width, table=rng.choice(["f32", act]), act=act)
    if op in ("norm", "norm_grad"):
        width = _log_int(rng, 64, 8192)
        if rng.random() < 0.6:
            width = max(64, width // 64 * 64)
        batch, res, gate = rng.choice([1, 2, 3, 8]), rng.choice(["f32", act]), rng.choice(["none", "channel", "sample", "full"])
        element = (3 if op == "norm_grad" else 2) * (BYTES[res] + BYTES[act]) + (2 * BYTES[act] if gate == "full" else 0)
        most = min(2048, 16384 * 4096 * 12 // (element * width * batch))
        return dict(op=op, batch=batch, length=_log_int(rng, 1, most), width=width, res=res, act=act, gate=gate)
    vocab = _log_int(rng, 1000, 131072)
    if rng.random() < 0.5:
        vocab = max(1000, vocab // 64 * 64)
    most = 2048 * VOCAB // vocab
    return dict(op=op, tokens=_log_int(rng, 1, min(4096, most)), vocab=vocab, k=_log_int(rng, 1, 128), act=act,
                tau=rng.choice([1.0, 2.0, 4.0]))


# Token ids follow a rank-frequency law over the whole vocabulary, as ids of a merged-pair tokenizer do.
def _frequencies(case):
    n = max(VOCAB, case["row0"] + case["rows"])
    p = 1.0 / (torch.arange(n, dtype=torch.float64) + 2.7)
    return p / p.sum()


def _window(case):
    """Expected numbers of tokens in the row window, and of different rows they hit."""
    p = _frequencies(case)[case["row0"]:case["row0"] + case["rows"]]
    return float(p.sum()) * case["tokens"], float((1 - (1 - p) ** case["tokens"]).sum())


def _gate_rows(case):
    return {"none": 0, "channel": 1, "sample": case["batch"], "full": case["batch"] * case["length"]}[case["gate"]]


MASKED = 0.125  # share of the rows of a distillation batch that carry no loss (prompts, padding)


def work(case):
    op = case["op"]
    if op in ("gather", "gather_grad"):
        t, d = case["tokens"], case["width"]
        hit, distinct = _window(case)
        if op == "gather":
            return dict(bytes=8 * t + distinct * d * BYTES[case["table"]] + t * d * BYTES[case["act"]], flops=hit * d)
        return dict(bytes=8 * t + hit * d * BYTES[case["act"]] + case["rows"] * d * BYTES[case["table"]], flops=hit * d)
    if op in ("norm", "norm_grad"):
        n, d, g = case["batch"] * case["length"], case["width"], _gate_rows(case)
        res, act = BYTES[case["res"]], BYTES[case["act"]]
        if op == "norm":
            return dict(bytes=n * d * 2 * (res + act) + 8 * d + g * d * act, flops=10 * n * d)
        return dict(bytes=n * d * 3 * (res + act) + 16 * d + 2 * g * d * act, flops=26 * n * d)
    t, v, k = case["tokens"], case["vocab"], case["k"]
    read = t * (1 - MASKED) * v * BYTES[case["act"]] + t * k * 12 + 8 * t
    if op == "distill_loss":
        return dict(bytes=read, flops=4 * t * v)
    return dict(bytes=read + t * v * BYTES[case["act"]], flops=7 * t * v)


def _randn(gen, *shape, scale=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda").mul_(scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = dict(case=case)
    if op in ("gather", "gather_grad"):
        t, d = case["tokens"], case["width"]
        cdf = _frequencies(case).cumsum(0).cuda()
        state["tokens"] = torch.searchsorted(cdf, torch.rand(t, generator=gen, device="cuda", dtype=torch.float64)).clamp_(
            max=cdf.numel() - 1)
        state["scale"] = math.sqrt(d)
        if op == "gather":
            state["weight"] = _randn(gen, case["rows"], d, scale=0.02, dtype=TYPES[case["table"]])
        else:
            state["grad"] = _randn(gen, t, d, scale=1e-3, dtype=TYPES[case["act"]])
        return state
    if op in ("norm", "norm_grad"):
        b, n, d = case["batch"], case["length"], case["width"]
        res, act = TYPES[case["res"]], TYPES[case["act"]]
        state["residual"] = _randn(gen, b, n, d, scale=2.0, dtype=res)  # before the block, or (backward) after it
        state["x"] = _randn(gen, b, n, d, scale=0.7, dtype=act)
        state["post_weight"] = 1 + _randn(gen, d, scale=0.1)
        state["pre_weight"] = 1 + _randn(gen, d, scale=0.1)
        shape = {"none": None, "channel": (d,), "sample": (b, 1, d), "full": (b, n, d)}[case["gate"]]
        state["gate"] = None if shape is None else _randn(gen, *shape, scale=0.5, dtype=act)
        state["scale"] = 0.35
        if op == "norm_grad":
            state["d_residual"] = _randn(gen, b, n, d, scale=0.02, dtype=res)
            state["d_y"] = _randn(gen, b, n, d, scale=0.02, dtype=act)
        return state
    t, v, k, act = case["tokens"], case["vocab"], case["k"], TYPES[case["act"]]
    teacher = 14.0 - torch.rand(t, k, generator=gen, device="cuda").mul_(1.2).cumsum(1)
    start = torch.randint(v, (t, 1), generator=gen, device="cuda")
    step = 1 + torch.randint(max(1, v // k - 1), (t, 1), generator=gen, device="cuda")
    ids = (start + step * torch.arange(k, device="cuda")) % v
    logits = torch.randn((t, v), generator=gen, device="cuda").mul_(2.0)
    logits.scatter_(1, ids, teacher + _randn(gen, t, k, scale=1.5))
    # one row in eight has fewer teacher entries than k: the rest of its list is padded with id -1
    short = torch.rand(t, 1, generator=gen, device="cuda") < 0.125
    count = 1 + torch.randint(k, (t, 1), generator=gen, device="cuda")
    ids = torch.where(short & (torch.arange(k, device="cuda") >= count), -1, ids)
    mask = torch.rand(t, generator=gen, device="cuda") >= MASKED
    mask[0] = True
    state["logits"], state["ids"], state["teacher"] = logits.to(act), ids, teacher
    # mean over the rows with a loss; float16 gradients carry a loss scale
    state["weight"] = mask.float() * (32768.0 if case["act"] == "f16" else 1.0) / mask.sum()
    return state


def _gather(state):
    case, w = state["case"], state["weight"]
    at = state["tokens"] - case["row0"]
    inside = (at >= 0) & (at < case["rows"])
    rows = w[at.clamp(0, case["rows"] - 1)].float() * state["scale"]
    return torch.where(inside[:, None], rows, 0.0).to(TYPES[case["act"]])


def _gather_grad(state):
    case = state["case"]
    at = state["tokens"] - case["row0"]
    inside = (at >= 0) & (at < case["rows"])
    total = torch.zeros(case["rows"], case["width"], device="cuda")
    total.index_add_(0, at[inside], state["grad"][inside].float())
    return (total * state["scale"]).to(TYPES[case["table"]])


EPS = 1e-6


def _norm(state):
    h, x = state["residual"].float(), state["x"].float()
    p = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * state["post_weight"]
    if state["gate"] is not None:
        p = p * state["gate"].float()
    h = h + state["scale"] * p
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * state["pre_weight"]
    return h.to(state["residual"].dtype), y.to(state["x"].dtype)


def _norm_grad(state):
    h, x, dh, dy = (state[k].float() for k in ("residual", "x", "d_residual", "d_y"))
    rh = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    rx = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    n, q = h * rh, x * rx
    dn = dy * state["pre_weight"]
    e = dh + rh * (dn - n * (dn * n).mean(-1, keepdim=True))
    d_pre = (dy * n).sum((0, 1))
    d_gate, ge = None, state["scale"] * e
    if state["gate"] is not None:
        gate = state["gate"]
        full = ge * (q * state["post_weight"])
        d_gate = full if gate.dim() == 3 and gate.shape[1] == h.shape[1] else full.sum(1, keepdim=True) if gate.dim() == 3 else full.sum((0, 1))
        d_gate, ge = d_gate.to(gate.dtype), ge * gate.float()
    d_post = (ge * q).sum((0, 1))
    dq = ge * state["post_weight"]
    dx = rx * (dq - q * (dq * q).mean(-1, keepdim=True))
    return e.to(state["d_residual"].dtype), dx.to(state["x"].dtype), d_post, d_pre, d_gate


def _distill(state, backward):
    z, ids, tau = state["logits"].float(), state["ids"], state["case"]["tau"]
    valid, at, weight = ids >= 0, ids.clamp(min=0), state["weight"]
    u = torch.where(valid, state["teacher"] / tau, -math.inf)
    u = u - u.amax(1, keepdim=True)
    p = torch.exp(u)
    total = p.sum(1, keepdim=True)
    p, log_p = p / total, torch.where(valid, u - total.log(), 0.0)
    z = z / tau
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    norm = e.sum(1, keepdim=True)
    log_q = z.gather(1, at) - norm.log()
    loss = weight * tau * tau * (p * (log_p - log_q)).sum(1)
    if not backward:
        return loss
    grad = (e / norm).scatter_add_(1, at, -p) * (weight * tau)[:, None]
    return loss, grad.to(state["logits"].dtype)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from cresso_b200 import ops

        if op == "gather":
            return ops.embedding_gather(state["weight"], state["tokens"], state["scale"], row0=case["row0"],
                                        dtype=TYPES[case["act"]])
        if op == "gather_grad":
            return ops.embedding_grad(state["grad"], state["tokens"], case["rows"], state["scale"], row0=case["row0"],
                                      dtype=TYPES[case["table"]])
        if op == "norm":
            return ops.block_norm(state["residual"], state["x"], state["post_weight"], state["pre_weight"],
                                  state["gate"], state["scale"], EPS)
        if op == "norm_grad":
            return ops.block_norm_grad(state["residual"], state["x"], state["d_residual"], state["d_y"],
                                       state["post_weight"], state["pre_weight"], state["gate"], state["scale"], EPS)
        f = ops.distill_loss if op == "distill_loss" else ops.distill_grad
        return f(state["logits"], state["ids"], state["teacher"], state["weight"], case["tau"])
    if op == "gather":
        return _gather(state)
    if op == "gather_grad":
        return _gather_grad(state)
    if op == "norm":
        return _norm(state)
    if op == "norm_grad":
        return _norm_grad(state)
    return _distill(state, op == "distill_grad")


def exact(case, seed):
    """The operators' definitions in float64, apart from the plain forms above."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "gather":
        padded = torch.cat([s["weight"].double(), torch.zeros(1, case["width"], device="cuda", dtype=torch.float64)])
        at = s["tokens"] - case["row0"]
        return padded[torch.where((at < 0) | (at >= case["rows"]), case["rows"], at)] * s["scale"]
    if op == "gather_grad":
        # one more row takes the tokens outside the window
        at = s["tokens"] - case["row0"]
        at = torch.where((at < 0) | (at >= case["rows"]), case["rows"], at)
        total = torch.zeros(case["rows"] + 1, case["width"], device="cuda", dtype=torch.float64)
        total.index_put_((at,), s["grad"].double() * s["scale"], accumulate=True)
        return total[:-1]
    if op in ("norm", "norm_grad"):
        v = {k: t.double().requires_grad_(op == "norm_grad") for k, t in s.items() if isinstance(t, torch.Tensor)}
        d = case["width"]
        p = v["x"] / ((v["x"] ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * v["post_weight"]
        block = s["scale"] * p if s["gate"] is None else s["scale"] * p * v["gate"]
        if op == "norm":
            h = v["residual"] + block
            return h, h / ((h ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * v["pre_weight"]
        before = (v["residual"] - block).detach().requires_grad_()
        h = before + block
        y = h / ((h ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * v["pre_weight"]
        leaves = [before, v["x"], v["post_weight"], v["pre_weight"]] + ([] if s["gate"] is None else [v["gate"]])
        got = list(torch.autograd.grad([h, y], leaves, [v["d_residual"].detach(), v["d_y"].detach()]))
        return tuple(got + [None] * (5 - len(got)))
    tau = case["tau"]
    z = s["logits"].double() / tau
    log_q = z - torch.logsumexp(z, 1, keepdim=True)
    # a further column takes the padded entries of the teacher's list
    t, vocab = z.shape
    target = torch.zeros(t, vocab + 1, device="cuda", dtype=torch.float64)
    held = s["ids"] >= 0
    u = (s["teacher"].double() / tau).masked_fill(~held, -math.inf)
    p = torch.softmax(u, 1)
    target.scatter_add_(1, torch.where(held, s["ids"], vocab), p)
    target = target[:, :vocab]
    weight = s["weight"].double()
    loss = weight * tau ** 2 * (torch.special.xlogy(p, p).sum(1) - (target * log_q).sum(1))
    if op == "distill_loss":
        return loss
    return loss, (weight * tau)[:, None] * (log_q.exp() - target)
