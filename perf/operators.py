"""Operators that turn a decoder's hidden rows into its next tokens, with their sizes and plain forms.

Three of them, in the order a decoding step runs them:

* ``linear``: a matrix product with 4-bit weights, one scale (and, where given, one zero point) per
  group of inputs of each output: ``c = scale * act(a . w^T + bias)``, ``w = (code - zero) * scale``;
* ``constrain``: logits with a repetition penalty, frequency and presence penalties over each
  row's tokens so far, a list of biases, and a bit mask of the tokens a grammar state allows;
* ``choose``: the best tokens of each row under the same rules and their log-probabilities.

``run`` computes the plain form in torch where ``own`` is false and calls the package where it is
true. ``exact`` states the same definitions in 64 bits.
"""

import math

import torch

own = False

_context = None


def _ctx():
    """The one context a program keeps for its GPU."""
    global _context
    if _context is None:
        import telmo_b200
        _context = telmo_b200.Context(torch.cuda.current_device())
    return _context


_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _linear(name, m, n, k, group, zeros, dtype, out, act, bias):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "group": group, "zeros": zeros,
            "dtype": dtype, "out": out, "act": act, "bias": bias}


def _rules(name, op, rows, vocab, dtype, history, biases, states, k=1):
    return {"name": name, "op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "history": history,
            "biases": biases, "states": states, "k": k}


def listed():
    return [
        # The joint network's output layer (8192 tokens, the blank and five durations over 640
        # inputs) for one utterance's step: a call of a few microseconds, where latency counts.
        _linear("joint_1", 1, 8198, 640, 32, False, "f32", "f32", "none", True),
        # The widest layer of a text decoder for a single token: the weights' bytes are the cost.
        _linear("token_1", 1, 32768, 4096, 128, False, "bf16", "f32", "none", False),
        # Eight streams' feed-forward up products in one step, with zero points.
        _linear("streams_8", 8, 4096, 1024, 32, True, "f32", "f32", "silu", True),
        # A batch of decoder steps, a down projection with an odd number of inputs.
        _linear("steps_24", 24, 4096, 11009, 64, True, "f16", "f16", "none", False),
        # One update of a stream: the rows of a span of audio through an encoder's up projection.
        _linear("span_200", 200, 4096, 1024, 32, False, "f32", "f32", "silu", True),
        # A 30 s utterance's feature rows through the same projection.
        _linear("utterance_1500", 1500, 4096, 1024, 64, False, "f32", "f32", "none", True),
        # A long prompt, or a batch of utterances, through a large layer.
        _linear("prompt_4096", 4096, 8192, 4096, 128, False, "bf16", "bf16", "none", False),
        # One row over the Granite head's 2049 tokens with a short history and a grammar.
        _rules("constrain_1", "constrain", 1, 2049, "f32", 64, 16, 4),
        # A full batch over a large vocabulary with long histories.
        _rules("constrain_256", "constrain", 256, 131072, "bf16", 2000, 100, 64),
        # One row of a large, odd vocabulary: the single-stream step.
        _rules("choose_1", "choose", 1, 49157, "f32", 500, 32, 8, 1),
        # A beam's hypotheses over the TDT vocabulary, four tokens each, half-precision logits.
        _rules("choose_64", "choose", 64, 8193, "f16", 100, 0, 16, 4),
        # A full batch over a large vocabulary, eight tokens each.
        _rules("choose_256", "choose", 256, 131072, "f32", 2000, 100, 64, 8),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over their logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "constrain", "choose"])
    if op == "linear":
        n, k = _spread(rng, 64, 16384), _spread(rng, 64, 8192)
        m = min(_spread(rng, 1, 4096), max(1, 4096 * 8192 * 4096 // (n * k)))
        dtype = rng.choice(["f32", "bf16", "f16"])
        c = _linear("", m, n, k, rng.choice([32, 64, 128]), rng.random() < 0.5, dtype,
                    rng.choice(["f32", dtype]), rng.choice(["none", "relu", "silu"]), rng.random() < 0.5)
    else:
        vocab = _spread(rng, 1000, 131072)
        rows = _spread(rng, 1, 256)
        c = _rules("", op, rows, vocab, rng.choice(["f32", "bf16", "f16"]),
                   rng.choice([0, _spread(rng, 1, 4000)]), rng.choice([0, _spread(rng, 1, 256)]),
                   rng.choice([0, _spread(rng, 1, 64)]), rng.choice([1, 2, 3, 4, 8]) if op == "choose" else 1)
    del c["name"]
    return c


# ---- inputs -----------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = _prepare_linear(case, g) if case["op"] == "linear" else _prepare_rules(case, g)
    s["case"] = case
    return s


def _prepare_linear(case, g):
    m, n, k, group = case["m"], case["n"], case["k"], case["group"]
    groups = -(-k // group)
    # A quantizer's output: codes 0..15, two to a byte (the even input in the low half), scales
    # that are f16 values, zero points near the middle of the range (8 where there are none).
    codes = torch.randint(0, 256, (n, -(-k // 2)), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.5 + torch.rand((n, groups), generator=g, device="cuda")) / (4.6 * math.sqrt(k))
    scales = scales.half().float()
    zeros = torch.randint(5, 12, (n, groups), generator=g, device="cuda", dtype=torch.uint8) \
        if case["zeros"] else None
    # Normalised activations, a few channels of which are much larger than the rest.
    a = torch.randn((m, k), generator=g, device="cuda")
    a = (a * (1 + 10 * (torch.rand((1, k), generator=g, device="cuda") < 0.005))).to(_TYPES[case["dtype"]])
    bias = torch.randn((n,), generator=g, device="cuda") * 0.02 if case["bias"] else None
    s = {"codes": codes, "scales": scales, "zeros": zeros, "a": a, "bias": bias}
    if own:
        # The handle a program keeps: the same codes, scales and zero points laid out on the device.
        from telmo_b200 import Kernels, PackedWeights, Precision
        packed = PackedWeights(n, k, Precision.Q4, codes.cpu().numpy(), scales.cpu().numpy(),
                               zeros=None if zeros is None else zeros.cpu().numpy(), group=group)
        s["weights"] = packed.upload(_ctx())
        s["kernels"] = Kernels(_ctx())
    return s


def _prepare_rules(case, g):
    rows, vocab, width = case["rows"], case["vocab"], case["history"]
    logits = torch.randn((rows, vocab), generator=g, device="cuda") * 2.5
    logits = (logits + 6 * (torch.rand((rows, vocab), generator=g, device="cuda") < 0.001)).to(_TYPES[case["dtype"]])
    s = {"logits": logits}
    if width:
        # Tokens so far: a few of them often, most of them rarely; each row with its own length,
        # and unused places filled with -1.
        u = torch.rand((rows, width), generator=g, device="cuda")
        history = (vocab * u * u * u).int().clamp_(0, vocab - 1)
        length = (width * (0.25 + 0.75 * torch.rand((rows,), generator=g, device="cuda"))).int().clamp_(0, width)
        past = torch.arange(width, device="cuda")[None, :] >= length[:, None]
        s["history"] = history.masked_fill_(past, -1)
        s["history_len"] = length
        s["repetition"] = 1 + 0.3 * torch.rand((rows,), generator=g, device="cuda")
        s["frequency"] = 0.5 * torch.rand((rows,), generator=g, device="cuda")
        s["presence"] = 0.5 * torch.rand((rows,), generator=g, device="cuda")
    if case["biases"]:
        s["bias_ids"] = torch.randint(0, vocab, (rows, case["biases"]), generator=g, device="cuda", dtype=torch.int32)
        s["bias"] = 4 * torch.randn((rows, case["biases"]), generator=g, device="cuda")
    if case["states"]:
        # A grammar's states: the first allows few tokens, the others about half; the last rows
        # (where there are several) are in a state that leaves nothing and without a mask.
        words = -(-vocab // 32)
        allowed = torch.randint(-(1 << 31), 1 << 31, (case["states"] + 1, words), generator=g, device="cuda",
                                dtype=torch.int64)
        few = torch.rand((words,), generator=g, device="cuda") < 0.02
        allowed[0] *= few
        allowed[-1] = 0
        s["allowed"] = allowed.int()
        state = torch.randint(0, case["states"], (rows,), generator=g, device="cuda", dtype=torch.int32)
        if rows > 2:
            state[-2] = case["states"]
            state[-1] = -1
        s["state"] = state
    if own:
        from telmo_b200 import Kernels, LogitRules
        s["kernels"] = Kernels(_ctx())
        s["rules"] = LogitRules(**{name: s[name] for name in ("history", "history_len", "repetition", "frequency",
                                                              "presence", "bias_ids", "bias", "allowed", "state")
                                   if name in s})
    return s


# ---- one pass -----------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "constrain": _own_constrain, "choose": _own_choose}[op](state)
    return {"linear": _plain_linear, "constrain": _plain_constrain, "choose": _plain_choose}[op](state)


def _own_linear(s):
    from telmo_b200 import Act, Epilogue
    case = s["case"]
    c = torch.empty((case["m"], case["n"]), dtype=_TYPES[case["out"]], device="cuda")
    s["kernels"].linear(s["a"], case["m"], s["weights"], c,
                        Epilogue(bias=s["bias"], act=Act[case["act"].upper()]))
    return c


def _own_constrain(s):
    case = s["case"]
    out = torch.empty_like(s["logits"])
    s["kernels"].constrain_logits(s["logits"], case["vocab"], case["rows"], case["vocab"], s["rules"], out,
                                  case["vocab"])
    return out


def _own_choose(s):
    case = s["case"]
    ids = torch.empty((case["rows"], case["k"]), dtype=torch.int32, device="cuda")
    logprobs = torch.empty((case["rows"], case["k"]), dtype=torch.float32, device="cuda")
    s["kernels"].choose_tokens(s["logits"], case["vocab"], case["rows"], case["vocab"], s["rules"], case["k"], ids,
                               logprobs)
    return {"ids": ids, "logprobs": logprobs}


def _plain_linear(s):
    case = s["case"]
    k, group = case["k"], case["group"]
    q = torch.stack((s["codes"] & 15, s["codes"] >> 4), dim=2).reshape(case["n"], -1)[:, :k].float()
    d = s["scales"].repeat_interleave(group, dim=1)[:, :k]
    z = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(group, dim=1)[:, :k]
    y = s["a"].float() @ ((q - z) * d).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["act"] == "relu":
        y = y.clamp(min=0)
    elif case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    return y.to(_TYPES[case["out"]])


def _plain_rules(s):
    """The logits under the rules, in 32 bits."""
    x = s["logits"].float()
    rows, vocab = x.shape
    if "history" in s:
        history = s["history"].long()
        live = torch.arange(history.shape[1], device=x.device)[None, :] < s["history_len"][:, None]
        live = live & (history >= 0) & (history < vocab)
        counts = torch.zeros_like(x).scatter_add_(1, history.clamp(0, vocab - 1), live.float())
        seen = counts > 0
        penalty = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / penalty, x * penalty), x)
        x = x - s["frequency"][:, None] * counts
        x = x - s["presence"][:, None] * seen
    if "bias" in s:
        ids = s["bias_ids"].long()
        live = (ids >= 0) & (ids < vocab)
        x = x + torch.zeros_like(x).scatter_add_(1, ids.clamp(0, vocab - 1), s["bias"] * live)
    if "allowed" in s:
        token = torch.arange(vocab, device=x.device)
        masks = s["allowed"][s["state"].clamp(min=0).long()]
        bits = (masks[:, token >> 5] >> (token & 31)) & 1
        x = torch.where((bits > 0) | (s["state"] < 0)[:, None], x, -math.inf)
    return x


def _plain_constrain(s):
    return _plain_rules(s).to(s["logits"].dtype)


def _plain_choose(s):
    x = _plain_rules(s)
    value, token = torch.sort(x, dim=1, descending=True, stable=True)  # ties: the lowest token first
    value, token = value[:, : s["case"]["k"]], token[:, : s["case"]["k"]].int()
    top = value[:, :1].clamp(min=-3e38)
    total = torch.log(torch.exp(x - top).sum(dim=1, keepdim=True))
    none = value == -math.inf
    return {"ids": token.masked_fill(none, -1),
            "logprobs": ((value - top) - total).masked_fill(none, -math.inf)}


# ---- what a pass cannot do without, and its definition in 64 bits ----------------------------------


def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        weights = n * -(-k // 2) + n * groups * (3 if case["zeros"] else 2)
        return {"bytes": weights + m * k * _SIZE[case["dtype"]] + m * n * _SIZE[case["out"]] + 4 * n * case["bias"],
                "flops": 2.0 * m * n * k}
    rows, vocab = case["rows"], case["vocab"]
    logits = rows * vocab * _SIZE[case["dtype"]]
    lists = rows * (4 * case["history"] + 8 * case["biases"]) + 16 * rows
    masks = min(rows, case["states"]) * -(-vocab // 32) * 4
    if case["op"] == "constrain":
        return {"bytes": 2 * logits + lists + masks, "flops": 4.0 * rows * vocab}
    return {"bytes": logits + lists + masks + 8 * rows * case["k"], "flops": 6.0 * rows * vocab}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(case, s)
    x = torch.stack([_exact_row(s, r) for r in range(case["rows"])])
    if case["op"] == "constrain":
        return x
    value = torch.topk(x, case["k"], dim=1).values
    logprobs = value - torch.logsumexp(x, dim=1, keepdim=True)
    return {"ids": None, "logprobs": torch.where(torch.isneginf(value), value, logprobs)}


def _exact_linear(case, s):
    n, k, group = case["n"], case["k"], case["group"]
    w = torch.empty((n, 2 * s["codes"].shape[1]), dtype=torch.float64, device="cuda")
    w[:, 0::2] = (s["codes"] % 16).double()
    w[:, 1::2] = torch.div(s["codes"], 16, rounding_mode="floor").double()
    for i in range(s["scales"].shape[1]):
        at = slice(i * group, min(k, (i + 1) * group))
        w[:, at] -= 8 if s["zeros"] is None else s["zeros"][:, i : i + 1].double()
        w[:, at] *= s["scales"][:, i : i + 1].double()
    y = torch.matmul(s["a"].double(), w[:, :k].T)
    if s["bias"] is not None:
        y += s["bias"].double()
    return {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v)}[case["act"]](y)


def _exact_row(s, r):
    x = s["logits"][r].double()
    vocab = x.numel()
    if "history" in s:
        said = s["history"][r, : int(s["history_len"][r])].long()
        count = torch.bincount(said[(said >= 0) & (said < vocab)], minlength=vocab).double()
        theta = s["repetition"][r].double()
        at = count > 0
        x[at] = torch.where(x[at] > 0, x[at] / theta, x[at] * theta)
        x[at] -= s["frequency"][r].double() * count[at] + s["presence"][r].double()
    if "bias" in s:
        x.index_add_(0, s["bias_ids"][r].long(), s["bias"][r].double())
    if "allowed" in s and int(s["state"][r]) >= 0:
        word = s["allowed"][int(s["state"][r])].long() & 0xFFFFFFFF
        bit = (word[:, None] >> torch.arange(32, device="cuda")[None, :]) & 1
        x[bit.reshape(-1)[:vocab] == 0] = -math.inf
    return x
