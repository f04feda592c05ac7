"""Workloads of the 8-bit operators and of the token log probabilities.

Each case is one pass through one operator on the GPU:

- norm:     residual addition, root-mean-square norm, output in 8 bits with a
            scale per token (B200.add_rmsnorm_q8);
- quantize: f32 rows in 8 bits with a scale per row (B200.quantize);
- matmul:   product of 8-bit activations and 8-bit weights with a scale per
            token and per channel (B200.matmul_q8);
- logprobs: log probabilities of given tokens, the entropy of each row and
            its most likely alternatives (LogProbs).

`run` computes them in plain torch operations, or, with `own` set, through the
framework. What an operator holds in 8 bits is returned as the values it
stands for (integer times scale), so a pass of norm and quantize ends with
that product on both sides.
"""

import math

import torch

own = False

EPS = 1e-6
VOCAB = 151936  # rows of the embedding and of lm_head in both checkpoints' configurations

_device = None


def _dev():
    """The framework's device, opened once. Its stream becomes torch's current one, so that what torch does with
    the operators' inputs and outputs, which share the framework's memory, stands in order with them."""
    global _device
    if _device is None:
        import titania_b200

        _device = titania_b200.B200(torch.cuda.current_device())
    if torch.cuda.current_stream().cuda_stream != _device.stream:
        torch.cuda.set_stream(torch.cuda.ExternalStream(_device.stream))
    return _device


# ---- cases ---------------------------------------------------------------------

def listed():
    return [
        # One decode step of the 0.6B model: one token, hidden size 1024. Latency counts.
        {"name": "norm-token", "op": "norm", "rows": 1, "cols": 1024, "residual": True},
        # The first norm of a pass (no residual yet) over a few tokens of a width that no vector load divides.
        {"name": "norm-ragged", "op": "norm", "rows": 61, "cols": 1001, "residual": False},
        # A long prompt through the 4B model's hidden size.
        {"name": "norm-prompt", "op": "norm", "rows": 5003, "cols": 2560, "residual": True},
        # One token's MLP activations in front of the 4B model's down_proj.
        {"name": "quantize-token", "op": "quantize", "rows": 1, "cols": 9728},
        # The same for a prompt.
        {"name": "quantize-prompt", "op": "quantize", "rows": 2048, "cols": 9728},
        # q|k|v of the 0.6B model for one token: the smallest product.
        {"name": "matmul-token", "op": "matmul", "rows": 1, "cols": 1024, "channels": 4096},
        # lm_head of the 0.6B model for one token: bound by the weights' bytes.
        {"name": "matmul-head", "op": "matmul", "rows": 1, "cols": 1024, "channels": VOCAB},
        # gate|up of the 4B model for 64 decoding sequences.
        {"name": "matmul-batch", "op": "matmul", "rows": 64, "cols": 2560, "channels": 19456},
        # One half of it for a prompt of a length that no tile divides.
        {"name": "matmul-prompt", "op": "matmul", "rows": 1999, "cols": 2560, "channels": 9728},
        # A generated token with the alternatives that a chat interface shows.
        {"name": "logprobs-token", "op": "logprobs", "rows": 1, "vocab": VOCAB, "top": 20},
        # One decode step of 64 sequences.
        {"name": "logprobs-batch", "op": "logprobs", "rows": 64, "vocab": VOCAB, "top": 5},
        # Scoring a prompt: every position's log probability.
        {"name": "logprobs-prompt", "op": "logprobs", "rows": 1111, "vocab": VOCAB, "top": 1},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "matmul", "matmul", "logprobs"])
    if op in ("norm", "quantize"):
        cols = _log_int(rng, 64, 10240)
        rows = _log_int(rng, 1, min(8192, 12_000_000 // cols))
        case = {"op": op, "rows": rows, "cols": cols}
        if op == "norm":
            case["residual"] = rng.random() < 0.75
        return case
    if op == "matmul":
        cols = _log_int(rng, 64, 10240)
        channels = _log_int(rng, 64, min(VOCAB, 160_000_000 // cols))
        rows = _log_int(rng, 1, max(1, min(2048, 45_000_000_000 // (cols * channels), 40_000_000 // channels)))
        return {"op": op, "rows": rows, "cols": cols, "channels": channels}
    vocab = _log_int(rng, 500, 200_000)
    return {"op": op, "rows": _log_int(rng, 1, max(1, min(2048, 160_000_000 // vocab))), "vocab": vocab,
            "top": rng.choice([0, 1, 3, 5, 10, 20, 40])}


# ---- inputs --------------------------------------------------------------------

def _inputs(case, seed):
    """The operator's inputs as torch tensors on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    rows, op = case["rows"], case["op"]
    if op == "norm":
        cols = case["cols"]
        # A residual stream: rows of different size, a few channels far larger than the rest.
        x = normal(rows, cols) * torch.exp(normal(rows, 1)) * torch.exp(0.5 * normal(1, cols))
        y = normal(rows, cols) * 0.3 if case["residual"] else None
        return {"x": x, "y": y, "w": (1 + 0.2 * normal(cols)).to(torch.bfloat16)}
    if op == "quantize":
        return {"x": normal(rows, case["cols"]) * torch.exp(normal(rows, 1))}
    if op == "matmul":
        cols, channels = case["cols"], case["channels"]

        def q8(n):
            values = torch.empty(n, cols, dtype=torch.int8, device="cuda")
            step = max(1, 64_000_000 // cols)
            for i in range(0, n, step):  # in parts, so that the f32 draws stay small
                part = values[i:i + step]
                part.copy_((normal(*part.shape) * 32).round_().clamp_(-127, 127))
            return values, torch.exp(0.5 * normal(n)) * 0.01

        xq, xs = q8(rows)
        wq, ws = q8(channels)
        return {"xq": xq, "xs": xs, "wq": wq, "ws": ws}
    vocab = case["vocab"]
    logits = normal(rows, vocab).mul_(1.5 + normal(rows, 1).abs_())
    # Half of the rows are scored at a likely token, the others at any; one row in eight excludes
    # a part of the vocabulary, as a grammar does.
    likely = logits.topk(min(4, vocab), dim=1).indices[:, -1]
    anyone = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    pick = torch.rand(rows, generator=g, device="cuda")
    tokens = torch.where(pick < 0.5, likely, anyone)
    cut = torch.where(pick * 4 % 1 < 0.125, vocab - vocab // 5, vocab)
    logits.masked_fill_(torch.arange(vocab, device="cuda")[None, :] >= cut[:, None], -math.inf)
    return {"logits": logits, "tokens": tokens.to(torch.int32)}


def _view(array):
    """A torch tensor over the framework's device memory."""
    return torch.as_tensor(array, device="cuda")


def prepare(case, seed):
    if own:
        _dev()
    state = _inputs(case, seed)
    state["op"] = case["op"]
    if case["op"] == "logprobs":
        state["top"] = case["top"]
    if own:
        return _framework_state(case, state)
    return state


def _framework_state(case, given):
    """The same inputs in the framework's buffers, with views of its outputs."""
    import titania_b200 as tb

    dev = _dev()
    rows, op = case["rows"], case["op"]
    state = {"op": op, "dev": dev}

    def buffer(tensor):
        b = dev.alloc(tensor.numel())
        dev.sync()
        _view(b).copy_(tensor.reshape(-1))
        return b

    if op in ("norm", "quantize"):
        cols = case["cols"]
        state["x"] = buffer(given["x"])
        state["q"] = dev.q8(rows, cols)
        state["values"] = dev.alloc(rows * cols)
        if op == "norm":
            state["y"] = buffer(given["y"]) if given["y"] is not None else None
            bits = given["w"].view(torch.int16).cpu().numpy().view("uint16")
            state["w"] = dev.upload(tb.Tensor([cols], bits))
        views = [_view(state["values"]).view(rows, cols), _view(state["q"].scales)]
        state["out"] = views if op == "quantize" else [_view(state["x"]).view(rows, cols)] + views
    elif op == "matmul":
        for name, n in (("x", rows), ("w", case["channels"])):
            q = dev.q8(n, case["cols"])
            dev.sync()
            _view(q.values).copy_(given[name + "q"])
            _view(q.scales).copy_(given[name + "s"])
            state[name] = q
        state["product"] = dev.alloc(rows * case["channels"])
        state["out"] = _view(state["product"]).view(rows, case["channels"])
    else:
        state["logits"] = buffer(given["logits"])
        state["tokens"] = given["tokens"]
        lp = state["scorer"] = tb.LogProbs(dev, rows, case["vocab"], case["top"])
        state["out"] = {"logprob": _view(lp.logprob), "entropy": _view(lp.entropy)}
        if case["top"]:
            state["out"]["top_ids"] = _view(lp.top_ids)
            state["out"]["top_logprobs"] = _view(lp.top_logprobs)
    torch.cuda.synchronize()
    return state


# ---- one pass ------------------------------------------------------------------

def run(state):
    if own:
        return _framework(state)
    return _PLAIN[state["op"]](state)


def _framework(state):
    dev, op = state["dev"], state["op"]
    if op == "norm":
        dev.add_rmsnorm_q8(state["q"], state["x"], state["y"], state["w"], EPS)
        dev.dequantize(state["values"], state["q"])
    elif op == "quantize":
        dev.quantize(state["q"], state["x"])
        dev.dequantize(state["values"], state["q"])
    elif op == "matmul":
        dev.matmul_q8(state["product"], state["w"], state["x"])
    else:
        state["scorer"].enqueue(state["logits"], state["tokens"])
    return state["out"]


def _rows_q8(n):
    """Rows of f64 values as (integers, f32 scales): the integers are computed in 64 bits, since a
    value next to the middle of two of them would go either way in 32."""
    scale = (n.abs().amax(1) / 127).float()
    step = scale.double()[:, None]
    q = torch.where(step > 0, n / step, 0).round().clamp(-127, 127)
    return q.to(torch.int8), scale


def _values(q, scale):
    return q.float() * scale[:, None]


def _plain_norm(state):
    x = state["x"]
    if state["y"] is not None:
        x += state["y"]
    h = x.double()
    r = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    q, scale = _rows_q8(h * state["w"].double() * r)
    return [x, _values(q, scale), scale]


def _plain_quantize(state):
    q, scale = _rows_q8(state["x"].double())
    return [_values(q, scale), scale]


def _plain_matmul(state):
    product = state["xq"].float() @ state["wq"].float().T
    return product * state["xs"][:, None] * state["ws"]


def _plain_logprobs(state):
    logits, tokens = state["logits"], state["tokens"].long()
    z = logits - logits.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1)
    log_total = torch.log(total)
    out = {
        "logprob": z.gather(1, tokens[:, None])[:, 0] - log_total,
        "entropy": log_total - torch.where(e > 0, e * z, 0).sum(1) / total,
    }
    if state["top"]:
        # Keys of 64 bits that no two tokens share: the logit's order, then the lowest id.
        bits = logits.view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
        ids = torch.arange(logits.shape[1], device=logits.device)
        top = ((order << 32) | (0xFFFFFFFF - ids)).topk(state["top"], dim=1).values
        at = 0xFFFFFFFF - (top & 0xFFFFFFFF)
        out["top_ids"] = at.to(torch.int32)
        out["top_logprobs"] = z.gather(1, at) - log_total[:, None]
    return out


_PLAIN = {"norm": _plain_norm, "quantize": _plain_quantize, "matmul": _plain_matmul, "logprobs": _plain_logprobs}


# ---- what a pass cannot do without ------------------------------------------------

def work(case):
    rows, op = case["rows"], case["op"]
    if op == "norm":
        n, cols = rows * case["cols"], case["cols"]
        # x (and the residual) in, the residual stream out where it changed, 8 bits and scales out.
        return {"bytes": (13 if case["residual"] else 5) * n + 2 * cols + 4 * rows,
                "flops": (6 if case["residual"] else 5) * n}
    if op == "quantize":
        n = rows * case["cols"]
        return {"bytes": 5 * n + 4 * rows, "flops": 2 * n}
    if op == "matmul":
        cols, channels = case["cols"], case["channels"]
        return {"bytes": (rows + channels) * (cols + 4) + 4 * rows * channels, "flops": 2 * rows * cols * channels}
    n = rows * case["vocab"]
    return {"bytes": 4 * n + 4 * rows * (3 + 2 * case["top"]), "flops": 5 * n}


# ---- the definition in 64 bits -------------------------------------------------------

def exact(case, seed):
    given = _inputs(case, seed)
    op = case["op"]
    if op in ("norm", "quantize"):
        import numpy as np

        x = given["x"].cpu().numpy()
        head = []
        if op == "norm":
            if given["y"] is not None:
                x = np.add(x, given["y"].cpu().numpy(), dtype=np.float32)
            head = [x.astype(np.float64)]
            h = x.astype(np.float64)
            n = h * given["w"].float().cpu().numpy().astype(np.float64)
            n /= np.sqrt(np.einsum("ij,ij->i", h, h) / h.shape[1] + EPS)[:, None]
        else:
            n = x.astype(np.float64)
        scale = (np.abs(n).max(axis=1) / 127.0).astype(np.float32).astype(np.float64)
        safe = np.where(scale > 0, scale, 1.0)[:, None]
        q = np.clip(np.rint(n / safe), -127, 127) * (scale > 0)[:, None]
        return head + [q * scale[:, None], scale]
    if op == "matmul":
        xq, xs = given["xq"].double(), given["xs"].double()
        out = torch.empty(case["rows"], case["channels"], dtype=torch.float64, device="cuda")
        step = max(1, 64_000_000 // case["cols"])
        for i in range(0, case["channels"], step):
            part = slice(i, i + step)
            scaled = given["wq"][part].double() * given["ws"][part].double()[:, None]
            out[:, part] = (xq * xs[:, None]) @ scaled.T
        return out
    logits, tokens = given["logits"], given["tokens"].long()
    out = {"logprob": [], "entropy": [], "top_logprobs": []}
    step = max(1, 40_000_000 // case["vocab"])
    for i in range(0, case["rows"], step):
        lp = torch.log_softmax(logits[i:i + step].double(), dim=1)
        out["logprob"].append(lp.gather(1, tokens[i:i + step, None])[:, 0])
        out["entropy"].append(torch.special.entr(lp.exp()).sum(1))
        if case["top"]:
            out["top_logprobs"].append(lp.topk(case["top"], dim=1).values)
    return {k: torch.cat(v) for k, v in out.items() if v} | ({"top_ids": None} if case["top"] else {})
