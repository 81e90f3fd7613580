"""The operators on compressed weights, as the cases their speed and exactness are measured on.

A weight stays compressed in GPU memory (the blob that compress_tensor makes of it) and the
operators compute with it: blob_linear (matrix product with bias, activation and residual in its
epilogue), blob_cross_entropy (softmax cross entropy over a large vocabulary, in pieces of the
vocabulary, without keeping the logits) and blob_distillation (from a teacher's top logits), each
forward and backward.  With `own` true, run() makes those calls; otherwise it computes the same
from the uncompressed weight with elementary torch operations in 32 bits.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
#: Compressed over original size of N(0, 0.02) weights: the order-0 entropy of their exponent bytes.
RATIO = {"bf16": 0.659, "fp16": 0.842}
ACTIVATIONS = (None, "relu", "gelu", "gelu_tanh", "silu")


def listed():
    return [
        # One token through the key projection of the 7B bf16 decoder: the smallest weight of a
        # layer, where latency counts.
        {"name": "linear_token_kv", "op": "linear", "dtype": "bf16", "tokens": 1, "out": 512, "inner": 3584,
         "bias": True, "act": None, "residual": False, "grad": False},
        # One token through the 7B feed-forward gate: a whole weight is decoded for one product.
        {"name": "linear_token_gate", "op": "linear", "dtype": "bf16", "tokens": 1, "out": 18944, "inner": 3584,
         "bias": False, "act": "silu", "residual": False, "grad": False},
        # Beams of a speech decoder through fc1 of the fp16 model (an odd number of tokens).
        {"name": "linear_beams_fc1", "op": "linear", "dtype": "fp16", "tokens": 7, "out": 5120, "inner": 1280,
         "bias": True, "act": "gelu", "residual": False, "grad": False},
        # A batch of decoding sequences through the 7B down projection, added to the residual stream.
        {"name": "linear_batch_down", "op": "linear", "dtype": "bf16", "tokens": 48, "out": 3584, "inner": 18944,
         "bias": False, "act": None, "residual": True, "grad": False},
        # Odd sizes everywhere: an adapter-like weight whose rows are not a multiple of 16 bytes.
        {"name": "linear_odd_train", "op": "linear", "dtype": "bf16", "tokens": 333, "out": 1001, "inner": 517,
         "bias": True, "act": "relu", "residual": True, "grad": True},
        # A ragged prompt through the 7B feed-forward gate.
        {"name": "linear_prompt_gate", "op": "linear", "dtype": "bf16", "tokens": 2047, "out": 18944, "inner": 3584,
         "bias": True, "act": "silu", "residual": False, "grad": False},
        # A training step of adapters beside a frozen compressed feed-forward layer: the gradient
        # goes through the weight to the input.
        {"name": "linear_train_up", "op": "linear", "dtype": "bf16", "tokens": 4096, "out": 18944, "inner": 3584,
         "bias": True, "act": "gelu_tanh", "residual": False, "grad": True},
        # Scoring one next token against the whole 7B vocabulary.
        {"name": "entropy_token", "op": "entropy", "dtype": "bf16", "tokens": 1, "vocab": 152064, "inner": 3584,
         "ignored": 0.0, "reduction": "none", "grad": False},
        # Per-token scores of one transcript (fp16, vocabulary of no round size).
        {"name": "entropy_scores_fp16", "op": "entropy", "dtype": "fp16", "tokens": 448, "vocab": 51866, "inner": 1280,
         "ignored": 0.0, "reduction": "none", "grad": False},
        # A training step of the 7B model with its head frozen and compressed, prompts masked out.
        {"name": "entropy_train", "op": "entropy", "dtype": "bf16", "tokens": 4096, "vocab": 152064, "inner": 3584,
         "ignored": 0.3, "reduction": "mean", "grad": True},
        # Distilling the fp16 speech model: the teacher's best few tokens, softened, some rows short.
        {"name": "distil_fp16", "op": "distil", "dtype": "fp16", "tokens": 301, "vocab": 51866, "inner": 1280,
         "top": 8, "short": 0.3, "temperature": 2.0, "reduction": "sum", "grad": True},
        # Distilling into the 4B model from stored top-32 logits.
        {"name": "distil_train", "op": "distil", "dtype": "bf16", "tokens": 2048, "vocab": 151936, "inner": 2560,
         "top": 32, "short": 0.0, "temperature": 1.0, "reduction": "mean", "grad": True},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "entropy", "distil"])
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "grad": rng.random() < 0.5}
    if op == "linear":
        case |= {"tokens": _log(rng, 1, 4096), "out": _log(rng, 64, 18944), "inner": _log(rng, 64, 18944),
                 "bias": rng.random() < 0.5, "act": rng.choice(ACTIVATIONS), "residual": rng.random() < 0.5}
        return case
    case |= {"tokens": _log(rng, 1, 4096), "vocab": _log(rng, 2000, 152064), "inner": _log(rng, 64, 3584),
             "reduction": rng.choice(["mean", "sum", "none"])}
    if op == "entropy":
        return case | {"ignored": rng.choice([0.0, 0.1, 0.5])}
    return case | {"top": _log(rng, 1, 64), "short": rng.choice([0.0, 0.3]), "temperature": rng.choice([0.7, 1.0, 2.0])}


def _chunk(numel):
    """Elements of a compressed chunk: small weights are cut finer, so that their decoding spreads
    over the GPU (a chunk is one block's work), between 16 Ki and the codec's default 128 Ki."""
    return min(131072, max(16384, 1 << round(math.log2(numel / 740))))


def _weight(rows, cols, dtype, gen):
    w = torch.empty((rows, cols), dtype=dtype, device=DEVICE)
    w.normal_(0.0, 0.02, generator=gen)
    if own:
        import cuzipnn_b200

        chunk = _chunk(w.numel())
        return cuzipnn_b200.compress_tensor(w, chunk_bytes=chunk, sub_chunk_bytes=chunk // 16, readback_to_cpu=False)
    return w


def _inputs(case, seed):
    """(generator, tensors) of a case: everything but the weight, which is drawn after them."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, tokens, inner = DTYPES[case["dtype"]], case["tokens"], case["inner"]

    def normal(*shape, scale=1.0, dt=dtype):
        return (torch.randn(shape, generator=gen, device=DEVICE) * scale).to(dt)

    s = {"x": normal(tokens, inner)}
    if case["op"] == "linear":
        out = case["out"]
        s["bias"] = normal(out, scale=0.1) if case["bias"] else None
        s["residual"] = normal(tokens, out) if case["residual"] else None
        s["g"] = normal(tokens, out) if case["grad"] else None
        return gen, s
    vocab = case["vocab"]
    if case["op"] == "entropy":
        s["targets"] = torch.randint(vocab, (tokens,), generator=gen, device=DEVICE)
        drop = torch.rand(tokens, generator=gen, device=DEVICE) < case["ignored"]
        s["targets"][drop] = -100
    else:
        top = case["top"]
        steps = torch.randint(1, vocab // top + 1, (tokens, top), generator=gen, device=DEVICE)
        first = torch.randint(vocab, (tokens, 1), generator=gen, device=DEVICE)
        s["ids"] = (first + steps.cumsum(1) - steps[:, :1]) % vocab
        s["logits"] = (torch.randn((tokens, top), generator=gen, device=DEVICE) * 2.0 + 8.0).sort(1, descending=True)[0]
        short = torch.rand(tokens, 1, generator=gen, device=DEVICE) < case["short"]
        keep = torch.randint(top + 1, (tokens, 1), generator=gen, device=DEVICE)
        place = torch.arange(top, device=DEVICE)
        s["ids"] = torch.where(short & (place >= keep), -1, s["ids"])
    # A loss scale as mixed precision training uses it (fp16 gradients would vanish without).
    scale = 1024.0 if case["dtype"] == "fp16" else 1.0
    if case["reduction"] == "mean":
        scale *= tokens
    s["g"] = torch.full((tokens,) if case["reduction"] == "none" else (), scale, device=DEVICE) if case["grad"] else None
    return gen, s


def _rows(case):
    return case["out"] if case["op"] == "linear" else case["vocab"]


def prepare(case, seed):
    gen, s = _inputs(case, seed)
    s["weight"] = _weight(_rows(case), case["inner"], DTYPES[case["dtype"]], gen)
    s["case"] = case
    for name in ("x", "bias", "residual"):
        if case["grad"] and s.get(name) is not None:
            s[name].requires_grad_()
    return s


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _PLAIN[s["case"]["op"]](s, s["case"])


def _run_own(s):
    import cuzipnn_b200 as z

    case = s["case"]
    with torch.set_grad_enabled(case["grad"]):
        if case["op"] == "linear":
            y = z.blob_linear(s["x"], s["weight"], bias=s["bias"], activation=case["act"], residual=s["residual"])
        elif case["op"] == "entropy":
            y = z.blob_cross_entropy(s["x"], s["weight"], s["targets"], reduction=case["reduction"])
        else:
            y = z.blob_distillation(s["x"], s["weight"], s["logits"], s["ids"], temperature=case["temperature"],
                                    reduction=case["reduction"])
    if not case["grad"]:
        return [y]
    leaves = [s[n] for n in ("x", "bias", "residual") if s.get(n) is not None]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["g"])]


def _plain_linear(s, case):
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    act = case["act"]
    if act == "relu":
        y, d = z.clamp(min=0.0), (z > 0).float()
    elif act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        y, d = z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    elif act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        y, d = 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)
    elif act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        y, d = z * sig, sig * (1.0 + z * (1.0 - sig))
    else:
        y, d = z, None
    if s["residual"] is not None:
        y = y + s["residual"].float()
    dtype = s["x"].dtype
    if not case["grad"]:
        return [y.to(dtype)]
    g = s["g"].float()
    dz = g if d is None else g * d
    out = [y.to(dtype), (dz @ w).to(dtype)]
    if s["bias"] is not None:
        out.append(dz.sum(0).to(dtype))
    if s["residual"] is not None:
        out.append(s["g"])
    return out


def _plain_sparse(s, case, ids, q, temperature):
    """Cross entropy of the distribution q over the tokens `ids` (rows of zeros where none counts)
    with the softmax of the logits over the whole vocabulary, less q's own entropy."""
    h, w = s["x"].float(), s["weight"].float()
    logits = (h @ w.t()) / temperature
    m = logits.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(logits - m).sum(1, keepdim=True))
    counts = q.sum(1) > 0
    at = ids.clamp(min=0)
    loss = (q * (torch.log(q.clamp(min=1e-45)) - (torch.gather(logits, 1, at) - lse))).sum(1) * temperature**2
    loss = torch.where(counts, loss, 0.0)
    n = counts.sum().clamp(min=1)
    reduction = case["reduction"]
    out = [loss.sum() / n if reduction == "mean" else loss.sum() if reduction == "sum" else loss]
    if case["grad"]:
        p = torch.exp(logits - lse)
        p.scatter_add_(1, at, -q)
        scale = s["g"] * temperature / (n if reduction == "mean" else 1)
        scale = torch.where(counts, scale, 0.0)
        out.append(((p @ w) * scale[:, None]).to(s["x"].dtype))
    return out


def _plain_entropy(s, case):
    t = s["targets"][:, None]
    return _plain_sparse(s, case, t, (t >= 0).float(), 1.0)


def _plain_distil(s, case):
    ids, temperature = s["ids"], case["temperature"]
    t = torch.where(ids >= 0, s["logits"].float(), -math.inf)
    e = torch.exp((t - t.amax(1, keepdim=True).clamp(min=-3e38)) / temperature)
    return _plain_sparse(s, case, ids, e / e.sum(1, keepdim=True).clamp(min=1e-30), temperature)


_PLAIN = {"linear": _plain_linear, "entropy": _plain_entropy, "distil": _plain_distil}


def work(case):
    rows, inner, tokens = _rows(case), case["inner"], case["tokens"]
    flops = 2.0 * tokens * rows * inner * (2 if case["grad"] else 1)
    read = rows * inner * 2 * RATIO[case["dtype"]] + tokens * inner * 2
    if case["op"] == "linear":
        wide = tokens * rows * 2
        read += rows * 2 * case["bias"] + wide * case["residual"] + wide * case["grad"]
        written = wide + case["grad"] * (tokens * inner * 2 + rows * 2 * case["bias"])
    else:
        read += tokens * (8 if case["op"] == "entropy" else case["top"] * 12)
        written = 4 * (tokens if case["reduction"] == "none" else 1) + case["grad"] * tokens * inner * 2
    return {"bytes": int(read + written), "flops": int(flops)}


def exact(case, seed):
    gen, s = _inputs(case, seed)
    w = torch.empty((_rows(case), case["inner"]), dtype=DTYPES[case["dtype"]], device=DEVICE)
    w.normal_(0.0, 0.02, generator=gen)
    w = w.double()
    F = torch.nn.functional
    x = s["x"].double().requires_grad_(case["grad"])
    if case["op"] == "linear":
        bias, res = (None if s[n] is None else s[n].double().requires_grad_(case["grad"]) for n in ("bias", "residual"))
        y = F.linear(x, w, bias)
        act = {None: lambda v: v, "relu": F.relu, "gelu": F.gelu, "silu": F.silu,
               "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}[case["act"]]
        y = act(y) if res is None else act(y) + res
        leaves = [v for v in (x, bias, res) if v is not None]
        g = None if s["g"] is None else s["g"].double()
    else:
        t = case.get("temperature", 1.0)
        logp = F.log_softmax(F.linear(x, w) / t, dim=1)
        if case["op"] == "entropy":
            valid = s["targets"] >= 0
            loss = F.nll_loss(logp, s["targets"], reduction="none", ignore_index=-100)
        else:
            held = s["ids"] >= 0
            valid = held.any(1)
            tl = s["logits"].double().masked_fill(~held, -math.inf)
            q = torch.where(valid[:, None], torch.softmax(tl / t, 1), 0.0)
            ent = torch.special.xlogy(q, q).sum(1)
            loss = (ent - (q * logp.gather(1, s["ids"].clamp(min=0))).sum(1)) * t * t
        count = valid.sum().clamp(min=1)
        y = {"none": loss, "sum": loss.sum(), "mean": loss.sum() / count}[case["reduction"]]
        leaves, g = [x], None if s["g"] is None else s["g"].double()
    if not case["grad"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, g)]
