"""What is measured of the operators between a model's logits and its update.

Four operators, each with a plain form in elementary torch operations and the
call of `kernix_b200` that computes it:

* ``log_probs``: of each row of logits, the log probability of its given token,
  the log-sum-exp, the entropy and the likeliest alternatives;
* ``log_probs_grad``: the gradient of the first three with respect to the logits;
* ``grad_norm``: the 2-norm over all elements of a list of gradients;
* ``clip_grads``: the gradients scaled down to a largest global norm.
"""
import torch

own = False

DTYPES = {"f32": torch.float32, "f64": torch.float64}


def listed():
    return [
        # One sequence decoding on its own: the log probability of the token just sampled and five alternatives.
        {"name": "score one token", "op": "log_probs", "rows": 1, "vocab": 32000, "dtype": "f32", "top": 5,
         "entropy": False, "temperature": 1.0, "wide": 0, "masked": 0.0, "padded": 0.0},
        # A serving batch, one token for each sequence, a large vocabulary and twenty alternatives.
        {"name": "score a serving batch", "op": "log_probs", "rows": 64, "vocab": 131072, "dtype": "f32", "top": 20,
         "entropy": False, "temperature": 0.7, "wide": 0, "masked": 0.0, "padded": 0.0},
        # A training batch: loss and entropy of 4096 positions, no alternatives.
        {"name": "loss of a training batch", "op": "log_probs", "rows": 4096, "vocab": 32000, "dtype": "f32", "top": 0,
         "entropy": True, "temperature": 1.0, "wide": 0, "masked": 0.0, "padded": 0.0},
        # Scoring prompts of unequal lengths: an odd vocabulary (rows at any 4-byte offset), half of it masked, padded
        # positions without a token, a last row whose mask leaves nothing.
        {"name": "score ragged masked prompts", "op": "log_probs", "rows": 1501, "vocab": 50021, "dtype": "f32",
         "top": 8, "entropy": True, "temperature": 1.3, "wide": 0, "masked": 0.5, "padded": 0.2},
        # A check in double precision, with logits in a wider buffer (a vocabulary padded for the product).
        {"name": "loss in double precision", "op": "log_probs", "rows": 509, "vocab": 32003, "dtype": "f64", "top": 4,
         "entropy": True, "temperature": 1.0, "wide": 61, "masked": 0.0, "padded": 0.1},
        # The same training batch's gradient, with an entropy bonus and a penalty on the log-sum-exp.
        {"name": "gradient of a training batch", "op": "log_probs_grad", "rows": 4096, "vocab": 32000, "dtype": "f32",
         "entropy": True, "temperature": 1.0, "wide": 0, "masked": 0.0, "padded": 0.05},
        # A small model's step: a small odd vocabulary and few rows, where the launch counts.
        {"name": "gradient of a small batch", "op": "log_probs_grad", "rows": 16, "vocab": 4099, "dtype": "f32",
         "entropy": False, "temperature": 1.0, "wide": 0, "masked": 0.0, "padded": 0.0},
        # Double precision, masked logits, and rows of a wider buffer that start elsewhere than the gradient's.
        {"name": "gradient in double precision", "op": "log_probs_grad", "rows": 509, "vocab": 20011, "dtype": "f64",
         "entropy": True, "temperature": 0.9, "wide": 13, "masked": 0.3, "padded": 0.1},
        # The gradients of a small model: two blocks, odd widths.
        {"name": "norm of a small model", "op": "grad_norm", "layers": 2, "width": 96, "hidden": 257, "vocab": 1000,
         "dtype": "f32", "transposed": False},
        # The gradients of a model of 24 blocks, 0.37 billion elements, half of the weights held transposed.
        {"name": "norm of 24 blocks", "op": "grad_norm", "layers": 24, "width": 1024, "hidden": 4096, "vocab": 65536,
         "dtype": "f32", "transposed": True},
        # Clipping a middling model's gradients, which the second-level cache holds.
        {"name": "clip 4 blocks", "op": "clip_grads", "layers": 4, "width": 512, "hidden": 2048, "vocab": 8192,
         "dtype": "f32", "transposed": False, "max_norm": 1.0},
        # Clipping a model of 6 wide blocks with a large embedding, 0.37 billion elements.
        {"name": "clip 6 wide blocks", "op": "clip_grads", "layers": 6, "width": 2048, "hidden": 8192, "vocab": 32000,
         "dtype": "f32", "transposed": False, "max_norm": 1.0},
    ]


def _log(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["log_probs", "log_probs_grad", "grad_norm", "clip_grads"])
    dtype = rng.choice(["f32", "f32", "f32", "f64"])
    if op in ("log_probs", "log_probs_grad"):
        vocab = _log(rng, 1000, 131072)
        rows = min(_log(rng, 1, 4096), (100_000_000 if dtype == "f32" else 16_000_000) // vocab)
        case = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "entropy": rng.random() < 0.6,
                "temperature": rng.choice([1.0, 1.0, 0.6, 1.7]), "wide": rng.choice([0, 0, 0, 1, 37, 64]),
                "masked": rng.choice([0.0, 0.0, 0.4, 0.95]), "padded": rng.choice([0.0, 0.0, 0.15])}
        if op == "log_probs":
            case["top"] = rng.choice([0, 1, 3, 8, 20, 32])
        return case
    width = _log(rng, 64, 1500)
    case = {"op": op, "layers": rng.randint(1, 6), "width": width,
            "hidden": min(4096, width * rng.randint(2, 4) + rng.randint(0, 9)), "vocab": _log(rng, 500, 40000),
            "dtype": dtype, "transposed": rng.random() < 0.3}
    if op == "clip_grads":
        # A step in four stays below the largest norm: its gradients are as they were.
        case["max_norm"] = rng.choice([1.0, 1.0, 1.0, 1e4])
    return case


def _shapes(case):
    """Nine gradients for each block (four square products, two of the feed-forward part, two norms, a bias) and two more."""
    w, h = case["width"], case["hidden"]
    block = [(w, w)] * 4 + [(w, h), (h, w), (w,), (w,), (h,)]
    return block * case["layers"] + [(case["vocab"], w), (w,)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dt)

    state = {"case": case}
    if case["op"] in ("log_probs", "log_probs_grad"):
        rows, vocab = case["rows"], case["vocab"]
        buffer = normal(rows, vocab + case["wide"])
        buffer.mul_(2.5)
        logits = buffer[:, case["wide"]:]
        tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        # A trained model gives its token a larger logit than the rest.
        at = tokens[:, None]
        logits.scatter_(1, at, logits.gather(1, at) + 6.0)
        if case["masked"]:
            gone = torch.rand(rows, vocab, generator=gen, device="cuda") < case["masked"]
            logits.masked_fill_(gone, -torch.inf)
            logits[-1] = -torch.inf
        if case["padded"]:
            pad = torch.rand(rows, generator=gen, device="cuda") < case["padded"]
            tokens.masked_fill_(pad, -1)
        state |= {"logits": logits, "tokens": tokens}
        if case["op"] == "log_probs_grad":
            # What the forward pass left, and the gradients that reach its outputs.
            state["forward"] = _log_probs(logits, tokens, case["temperature"], 0, case["entropy"])
            state["grad_log_probs"] = normal(rows) / rows
            if case["entropy"]:
                state["grad_entropy"] = normal(rows) * (0.01 / rows)
                state["grad_lse"] = normal(rows) * (0.001 / rows)
        return state
    grads = [normal(*s).mul_(0.02 / (1 + i % 3)) for i, s in enumerate(_shapes(case))]
    if case["transposed"]:
        grads = [g.t() if g.dim() == 2 and i % 2 else g for i, g in enumerate(grads)]
    state["grads"] = grads
    if case["op"] == "clip_grads":
        state["outs"] = [torch.empty_like(g) for g in grads]
    return state


def _log_probs(logits, tokens, temperature, top, entropy):
    """Plain form.  A logit of -inf is a token that the mask takes out; a row without any other has a
    log-sum-exp of -inf and no entropy; a token of -1 stands for a position that has none."""
    z = logits / temperature
    most = z.amax(-1, keepdim=True)
    most = torch.where(torch.isinf(most), 0.0, most)
    lse = most + torch.log(torch.exp(z - most).sum(-1, keepdim=True))
    given = z.gather(1, tokens.clamp_min(0)[:, None])
    lp = torch.where(torch.isinf(given), given, given - lse)[:, 0]
    out = {"log_probs": torch.where(tokens < 0, 0.0, lp), "lse": lse[:, 0], "entropy": None,
           "top_log_probs": None, "top_tokens": None}
    if entropy:
        lq = torch.where(torch.isinf(z), 0.0, z - lse)
        out["entropy"] = -torch.where(torch.isinf(z), 0.0, torch.exp(lq) * lq).sum(-1)
    if top:
        values, ids = _largest(logits, top)
        gone = torch.isinf(values)
        out["top_log_probs"] = torch.where(gone, -torch.inf, values / temperature - lse)
        out["top_tokens"] = torch.where(gone, -1, ids)
    return out


def _largest(x, count):
    """The largest values of each row and their places, the lowest place first among equal ones."""
    if x.dtype == torch.float64:
        values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
        return values[:, :count], ids[:, :count]
    # One 64-bit key for each element: the float's order above, the place, counted down, below.
    bits = (x + 0.0).view(torch.int32)
    bits = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    places = torch.arange(x.shape[-1], device=x.device)
    keys = torch.topk((bits.long() << 32) | (0xFFFFFFFF - places), count, dim=-1).values
    ids = 0xFFFFFFFF - (keys & 0xFFFFFFFF)
    return x.gather(1, ids), ids


def _log_probs_grad(s):
    """Plain form: p_j (g_lse - g_lp - g_H (log p_j + H)) + g_lp [j = token], over the temperature; none for a
    logit that the mask took out."""
    z = s["logits"] / s["case"]["temperature"]
    lse, tokens = s["forward"]["lse"][:, None], s["tokens"][:, None]
    inside = ~torch.isinf(z)
    lq = torch.where(inside, z - lse, 0.0)
    p = torch.where(inside, torch.exp(lq), 0.0)
    g = torch.where(tokens < 0, 0.0, s["grad_log_probs"][:, None])
    factor = -g
    if s["case"]["entropy"]:
        factor = s["grad_lse"][:, None] - g - s["grad_entropy"][:, None] * (lq + s["forward"]["entropy"][:, None])
    grad = p * factor
    grad = grad.scatter_add_(1, tokens.clamp_min(0), g) / s["case"]["temperature"]
    return torch.where(inside, grad, 0.0)


def _norm(grads):
    """Plain form: squares in the gradients' type, their sum in 64 bits, as it is long."""
    return torch.stack([torch.square(g).sum(dtype=torch.float64) for g in grads]).sum().sqrt()


def _call(s):
    """The framework's calls."""
    import kernix_b200 as kx

    case = s["case"]
    if case["op"] == "log_probs":
        return kx.token_log_probs(s["logits"], s["tokens"], temperature=case["temperature"], top=case["top"],
                                  entropy=case["entropy"])._asdict()
    if case["op"] == "log_probs_grad":
        forward = s["forward"]
        return kx.token_log_probs_backward(s["logits"], s["tokens"], lse=forward["lse"], entropy=forward["entropy"],
                                           grad_log_probs=s["grad_log_probs"], grad_entropy=s.get("grad_entropy"),
                                           grad_lse=s.get("grad_lse"), temperature=case["temperature"])
    if case["op"] == "grad_norm":
        return kx.grad_norm(s["grads"])
    norm = kx.clip_grad_norm_into(s["grads"], s["case"]["max_norm"], s["outs"])
    return {"norm": norm, "grads": s["outs"]}


def run(state):
    if own:
        return _call(state)
    case = state["case"]
    if case["op"] == "log_probs":
        return _log_probs(state["logits"], state["tokens"], case["temperature"], case["top"], case["entropy"])
    if case["op"] == "log_probs_grad":
        return _log_probs_grad(state)
    norm = _norm(state["grads"])
    rounded = norm.to(DTYPES[case["dtype"]])
    if case["op"] == "grad_norm":
        return rounded
    scale = torch.clamp(case["max_norm"] / norm, max=1.0).to(DTYPES[case["dtype"]])
    return {"norm": rounded, "grads": [g * scale for g in state["grads"]]}


def work(case):
    size = 4 if case["dtype"] == "f32" else 8
    if case["op"] in ("log_probs", "log_probs_grad"):
        rows, n = case["rows"], case["rows"] * case["vocab"]
        if case["op"] == "log_probs":
            # Logits and tokens once; for each row two or three numbers and the alternatives with their places.
            each = 8 + size * (2 + case["entropy"]) + case["top"] * (size + 8)
            return {"bytes": n * size + rows * each, "flops": n * (6 if case["entropy"] else 4)}
        each = 8 + size * (2 + 3 * case["entropy"])
        return {"bytes": 2 * n * size + rows * each, "flops": n * (7 if case["entropy"] else 4)}
    n = sum(s[0] * (s[1] if len(s) > 1 else 1) for s in _shapes(case))
    if case["op"] == "grad_norm":
        return {"bytes": n * size + size, "flops": 2 * n}
    return {"bytes": 2 * n * size + size, "flops": 3 * n}


def exact(case, seed):
    """The same outputs from the definitions, in 64 bits, a few rows at a time."""
    s = prepare(case, seed)
    if case["op"] in ("grad_norm", "clip_grads"):
        flat = torch.cat([torch.linalg.vector_norm(g.double()).reshape(1) for g in s["grads"]])
        norm = torch.linalg.vector_norm(flat)
        if case["op"] == "grad_norm":
            return norm
        by = 1.0 if norm <= s["case"]["max_norm"] else s["case"]["max_norm"] / norm
        return {"norm": norm, "grads": [g.double() * by for g in s["grads"]]}
    parts = []
    for at in range(0, case["rows"], 128):
        x = s["logits"][at:at + 128].double()
        t = s["tokens"][at:at + 128]
        has = t >= 0
        one = torch.nn.functional.one_hot(t.clamp_min(0), case["vocab"]).bool() & has[:, None]
        lse = torch.logsumexp(x / case["temperature"], -1)
        empty = lse == -torch.inf
        lq = (x / case["temperature"]).sub(torch.where(empty, 0.0, lse)[:, None])
        p = lq.exp()
        plogp = torch.special.entr(p).neg()
        h = -plogp.sum(-1)
        if case["op"] == "log_probs_grad":
            g = s["grad_log_probs"][at:at + 128].double()[:, None]
            d = one * g - p * (has[:, None] * g)
            if case["entropy"]:
                g_h, g_l = (s[k][at:at + 128].double()[:, None] for k in ("grad_entropy", "grad_lse"))
                d = d + p * g_l - g_h * (plogp + p * h[:, None])
            parts.append((d / case["temperature"]).masked_fill(x == -torch.inf, 0.0))
            continue
        lp = torch.where(one, lq, -torch.inf).amax(-1)
        part = [torch.where(has, lp, 0.0), lse, h if case["entropy"] else None, None, None]
        if case["top"]:
            order = torch.sort(x, dim=-1, descending=True, stable=True)
            left = order.values[:, :case["top"]] > -torch.inf
            ids = order.indices[:, :case["top"]]
            part[3:] = [torch.where(left, lq.gather(1, ids), -torch.inf), torch.where(left, ids, -1)]
        parts.append(part)
    if case["op"] == "log_probs_grad":
        return torch.cat(parts)
    whole = [None if p[0] is None else torch.cat(p) for p in zip(*parts)]
    return dict(zip(("log_probs", "lse", "entropy", "top_log_probs", "top_tokens"), whole))
