"""What the operators around the RACE layer are measured on: the residual RMS norm, its 8-bit form,
the 8-bit SwiGLU, the 8-bit matrix product and the token log probabilities, each in its plain form
(`own` false: elementary torch operations in fp32) or through the package (`own` true).

Sizes come from the hybrid decoder (hidden 2048, MLP 8192, vocabulary 128256, batch 64, 32 K
contexts prefilled in slices) and the GPT harness (width 768, vocabulary 50257, 8 x 16 K tokens),
or are generic odd ones.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # the norms of one GPT training step at width 768 over 8 x 16384 tokens, forward and backward
        {"name": "norm_train_gpt", "op": "norm", "rows": 131072, "width": 768, "dtype": "bf16", "residual": True},
        # a small fp32 model of odd width: rows that start at no 16-byte boundary
        {"name": "norm_train_odd", "op": "norm", "rows": 1000, "width": 2047, "dtype": "fp32", "residual": True},
        # one decode step of 64 sequences: the norm in front of the int8 qkv product (latency)
        {"name": "norm8_decode", "op": "norm8", "rows": 64, "width": 2048, "dtype": "bf16", "residual": True},
        # a prefill slice of one 32 K context
        {"name": "norm8_prefill", "op": "norm8", "rows": 32768, "width": 2048, "dtype": "bf16", "residual": True},
        # the MLP's activation in a decode step, in front of the int8 down product (latency)
        {"name": "swiglu8_decode", "op": "swiglu8", "rows": 64, "width": 8192, "dtype": "bf16"},
        # the MLP's activation in a prefill slice
        {"name": "swiglu8_prefill", "op": "swiglu8", "rows": 16384, "width": 8192, "dtype": "bf16"},
        # a single sequence's output projection: one token (latency)
        {"name": "int8_token", "op": "int8", "m": 1, "n": 2048, "k": 2048, "dtype": "bf16", "bias": False},
        # gate and up projections of a decode step of 64 sequences (a stream over the weights)
        {"name": "int8_decode", "op": "int8", "m": 64, "n": 16384, "k": 2048, "dtype": "bf16", "bias": False},
        # a ragged batch through a layer of odd sizes, fp32 out with a bias
        {"name": "int8_ragged", "op": "int8", "m": 777, "n": 1001, "k": 2050, "dtype": "fp32", "bias": True},
        # gate and up projections of a prefill slice (a product of matrices)
        {"name": "int8_prefill", "op": "int8", "m": 16384, "n": 16384, "k": 2048, "dtype": "bf16", "bias": False},
        # the answers of a decode step: the sampled tokens' log probabilities with 20 alternatives
        {"name": "logp_decode", "op": "logp", "rows": 64, "vocab": 128256, "dtype": "bf16", "top": 20, "grad": False,
         "masked": False, "temperature": 1.0},
        # the loss of a training micro-batch over the GPT vocabulary (rows at 2-byte boundaries), with its gradient
        {"name": "logp_train", "op": "logp", "rows": 8192, "vocab": 50257, "dtype": "bf16", "top": 0, "grad": True,
         "masked": False, "temperature": 1.0},
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]: as it falls, or a multiple of 16."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(hi, max(lo, v))
    return v if v < 32 or rng.random() < 0.5 else v // 16 * 16


def draw(rng):
    op = rng.choice(["norm", "norm8", "swiglu8", "int8", "int8", "logp", "logp"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op in ("norm", "norm8", "swiglu8"):
        width = _log_int(rng, 64, 8192)
        most = {"norm": 131072 * 768, "norm8": 32768 * 2048, "swiglu8": 16384 * 8192}[op]
        rows = _log_int(rng, 1, min(131072, most // width // (2 if dtype == "fp32" else 1)))
        case = {"op": op, "rows": rows, "width": width, "dtype": dtype}
        if op != "swiglu8":
            case["residual"] = rng.random() < 0.75
        return case
    if op == "int8":
        k = _log_int(rng, 32, 8192)
        n = _log_int(rng, 32, 16384)
        m = _log_int(rng, 1, min(16384, 16384 * 2048 * 16384 // (n * k)))
        return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.3}
    vocab = _log_int(rng, 64, 131072)
    rows = _log_int(rng, 1, min(8192, 8192 * 50257 // vocab // (2 if dtype == "fp32" else 1)))
    grad = rng.random() < 0.5
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "top": 0 if grad else rng.randint(0, 20), "grad": grad,
            "masked": rng.random() < 0.3, "temperature": rng.choice([1.0, 1.0, 0.7])}


def _rows8(g, rows, width):
    """8-bit rows as the quantisers lay them out (row stride a multiple of 16 bytes) and their scales."""
    q = torch.empty(rows, -(-width // 16) * 16, dtype=torch.int8, device="cuda")[:, :width]
    q.copy_((torch.randn(rows, width, generator=g, device="cuda") * 36).round_().clamp_(-127, 127))
    scale = (torch.rand(rows, generator=g, device="cuda") + 0.5) * 0.02
    return q, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt) * scale

    op = case["op"]
    s = dict(case)
    if op in ("norm", "norm8"):
        r, w = case["rows"], case["width"]
        # a few channels of the residual stream are much larger than the rest
        stream = 1 + 9 * (torch.rand(w, generator=g, device="cuda") < 0.01).to(dt)
        s["x"] = normal(r, w)
        s["residual_in"] = normal(r, w) * stream if case["residual"] else None
        s["weight"] = 1 + 0.2 * torch.randn(w, generator=g, device="cuda")
        if op == "norm":
            s["dy"], s["dh"] = normal(r, w), normal(r, w)  # dh: what reaches the residual stream from above
    elif op == "swiglu8":
        s["gate_up"] = normal(case["rows"], 2 * case["width"], scale=1.5)
    elif op == "int8":
        s["xq"], s["xs"] = _rows8(g, case["m"], case["k"])
        s["wq"], s["ws"] = _rows8(g, case["n"], case["k"])
        s["b"] = torch.randn(case["n"], generator=g, device="cuda") if case["bias"] else None
    else:
        r, v = case["rows"], case["vocab"]
        s["logits"] = normal(r, v, scale=2.5)
        if case["masked"]:  # constrained answers: half of the vocabulary is not allowed
            s["logits"].masked_fill_(torch.rand(v, generator=g, device="cuda") < 0.5, -math.inf)
            s["logits"][:, 0] = 0
        s["tokens"] = torch.randint(0, v, (r,), generator=g, device="cuda")
        if case["masked"]:
            s["tokens"] = torch.where(s["logits"].gather(1, s["tokens"][:, None])[:, 0] > -math.inf, s["tokens"], 0)
        if case["grad"]:
            # padded positions of a batch carry no loss
            s["tokens"] = torch.where(torch.rand(r, generator=g, device="cuda") < 0.05, -100, s["tokens"])
            s["g_logp"] = torch.randn(r, generator=g, device="cuda")
            s["g_ent"] = torch.randn(r, generator=g, device="cuda") * 0.1
    return s


# ---------------------------------------------------------------------------------------- plain forms
def _quant(y, dt):
    """The values that the 8-bit rows of y stand for (in the rows' consumer type), and their scales."""
    scale = y.abs().amax(-1) / 127
    q = (y / scale[:, None]).round().clamp(-127, 127)
    q = torch.where(scale[:, None] > 0, q, 0)
    return (q * scale[:, None]).to(dt), scale


def _norm(s):
    dt = s["x"].dtype
    h = s["x"].float()
    if s["residual_in"] is not None:
        h = (h + s["residual_in"].float()).to(dt).float()
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    return h, rstd


def _plain_norm(s):
    dt = s["x"].dtype
    h, rstd = _norm(s)
    xhat = h * rstd
    dy = s["dy"].float()
    g = dy * s["weight"]
    dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    grads = {"weight": (dy * xhat).sum(0)}
    if s["residual_in"] is not None:
        dx = (dx + s["dh"].float()).to(dt)  # one gradient for both of the sum's terms
        grads["residual"] = dx
    grads["x"] = dx.to(dt)
    return {"y": (xhat * s["weight"]).to(dt), "h": h.to(dt), "grads": grads}


def _plain_norm8(s):
    dt = s["x"].dtype
    h, rstd = _norm(s)
    y, scale = _quant(h * rstd * s["weight"], torch.bfloat16)
    return {"y": y, "scale": scale, "h": h.to(dt)}


def _plain_swiglu8(s):
    gate, up = s["gate_up"].float().chunk(2, -1)
    y, scale = _quant(gate / (1 + torch.exp(-gate)) * up, torch.bfloat16)
    return {"y": y, "scale": scale}


def _plain_int8(s):
    y = (s["xq"].float() @ s["wq"].float().t()) * s["xs"][:, None] * s["ws"]
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(DTYPES[s["dtype"]])


def _plain_logp(s):
    logits, tokens = s["logits"].float(), s["tokens"]
    z = logits / s["temperature"]
    kept = tokens != -100
    at = tokens.clamp(min=0)[:, None]
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(-1, keepdim=True)
    lse = m + total.log()
    p = e / total
    entropy = -(p * torch.where(p > 0, z - lse, 0)).sum(-1)
    logp = (z.gather(1, at) - lse)[:, 0]
    out = {"logp": torch.where(kept, logp, 0), "entropy": torch.where(kept, entropy, 0)}
    if s["top"]:
        # one whole number per entry, in the order of (value, lower index first)
        bits = (logits + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32
        key = key - torch.arange(logits.shape[1], device=logits.device)
        ids = key.topk(s["top"], -1).indices
        out["top_ids"] = ids
        out["top_logp"] = z.gather(1, ids) - lse
    if s["grad"]:
        g_logp, g_ent = torch.where(kept, s["g_logp"], 0)[:, None], torch.where(kept, s["g_ent"], 0)[:, None]
        dz = -p * (g_logp + g_ent * (torch.where(p > 0, z - lse, 0) + entropy[:, None]))
        dz.scatter_add_(1, at, g_logp)
        out["dlogits"] = (dz / s["temperature"]).to(s["logits"].dtype)
    return out


# ---------------------------------------------------------------------------------------- the package
def _own(s):
    import race_attention_b200 as rb

    op = s["op"]
    if op == "norm":
        x = s["x"].detach().requires_grad_(True)
        w = s["weight"].detach().requires_grad_(True)
        r = None if s["residual_in"] is None else s["residual_in"].detach().requires_grad_(True)
        y, h = rb.add_rms_norm(x, r, w, eps=EPS)
        wanted = {"x": x, "weight": w} if r is None else {"x": x, "weight": w, "residual": r}
        outs, gins = ((y,), (s["dy"],)) if r is None else ((y, h), (s["dy"], s["dh"]))
        grads = torch.autograd.grad(outs, tuple(wanted.values()), gins)
        return {"y": y.detach(), "h": h.detach(), "grads": dict(zip(wanted, grads))}
    if op == "norm8":
        rows, h = rb.add_rms_norm_int8(s["x"], s["residual_in"], s["weight"], eps=EPS)
        return {"y": rows.dequant(torch.bfloat16), "scale": rows.scale, "h": h}
    if op == "swiglu8":
        rows = rb.swiglu_int8(s["gate_up"])
        return {"y": rows.dequant(torch.bfloat16), "scale": rows.scale}
    if op == "int8":
        return rb.int8_linear(rb.Int8Rows(s["xq"], s["xs"]), rb.Int8Rows(s["wq"], s["ws"]), s["b"], DTYPES[s["dtype"]])
    logits = s["logits"].detach().requires_grad_(s["grad"])
    r = rb.token_logprobs(logits, s["tokens"], temperature=s["temperature"], n_top=s["top"])
    out = {"logp": r.logp.detach(), "entropy": r.entropy.detach()}
    if s["top"]:
        out["top_ids"], out["top_logp"] = r.top_ids, r.top_logp
    if s["grad"]:
        out["dlogits"], = torch.autograd.grad((r.logp, r.entropy), (logits,), (s["g_logp"], s["g_ent"]))
    return out


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "norm8": _plain_norm8, "swiglu8": _plain_swiglu8, "int8": _plain_int8,
            "logp": _plain_logp}[state["op"]](state)


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + (4 * n if case["bias"] else 0) + e * m * n, "flops": 2 * m * n * k}
    if op == "logp":
        rv = case["rows"] * case["vocab"]
        return {"bytes": e * rv * (3 if case["grad"] else 1) + case["rows"] * (16 + 12 * case["top"]),
                "flops": (10 if case["grad"] else 5) * rv}
    rw = case["rows"] * case["width"]
    if op == "norm":  # x, residual, dy, dh in; y, h, dx out, and h (x where there is no residual) again for the backward
        return {"bytes": e * rw * (8 if case["residual"] else 5) + 8 * case["width"], "flops": 14 * rw}
    if op == "norm8":  # x, residual in; h, 8-bit rows out
        return {"bytes": rw * (e * (3 if case["residual"] else 1) + 1) + 4 * case["rows"] + 4 * case["width"],
                "flops": 7 * rw}
    return {"bytes": rw * (2 * e + 1) + 4 * case["rows"], "flops": 8 * rw}


# ---------------------------------------------------------------------------------------- in 64 bits
def _exact_rows(y):
    """Nearest multiples of a 127th of each row's largest magnitude."""
    step = y.abs().max(1, keepdim=True).values.div(127.0)
    return torch.where(step > 0, torch.round(y / step) * step, torch.zeros_like(y)), step[:, 0]


def _exact_norm_block(s, lo, hi):
    h = s["x"][lo:hi]
    if s["residual_in"] is not None:
        # the residual stream is held in the inputs' type
        h = torch.add(h.double(), s["residual_in"][lo:hi].double()).float().to(h.dtype)
    h = h.double()
    n = (h * h).sum(1, keepdim=True) / h.shape[1]
    return h, (n + EPS).pow(-0.5)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "int8":
        a = s["xq"].double() * s["xs"].double().unsqueeze(1)
        b = s["wq"].double() * s["ws"].double().unsqueeze(1)
        y = torch.mm(a, b.T)
        return y if s["b"] is None else y + s["b"].double()
    rows = case["rows"]
    width = case["vocab"] if op == "logp" else case["width"]
    block = max(1, (1 << 27) // width)
    parts = []
    dw = torch.zeros(width, dtype=torch.float64, device="cuda")
    for lo in range(0, rows, block):
        hi = min(rows, lo + block)
        if op == "norm":
            h, rstd = _exact_norm_block(s, lo, hi)
            dy, w = s["dy"][lo:hi].double(), s["weight"].double()
            dw += torch.einsum("rk,rk,r->k", dy, h, rstd[:, 0])
            proj = torch.einsum("rk,rk,k->r", dy, h, w)[:, None] / width
            dx = dy * w * rstd - h * proj * rstd.pow(3)
            if s["residual_in"] is not None:
                dx = dx + s["dh"][lo:hi].double()
            parts.append((h * w * rstd, h, dx))
        elif op == "norm8":
            h, rstd = _exact_norm_block(s, lo, hi)
            y, step = _exact_rows(h * s["weight"].double() * rstd)
            parts.append((y, step, h))
        elif op == "swiglu8":
            a = s["gate_up"][lo:hi].double()
            parts.append(_exact_rows(a[:, :width] * torch.sigmoid(a[:, :width]) * a[:, width:]))
        else:
            z = s["logits"][lo:hi].double() / case["temperature"]
            t = s["tokens"][lo:hi]
            logq = z - torch.logsumexp(z, 1, keepdim=True)
            q = logq.exp()
            plogq = torch.where(q > 0, q * logq, torch.zeros_like(q))
            ent = -plogq.sum(1)
            used = t >= 0
            pick = torch.where(used, t, torch.zeros_like(t))
            got = [torch.where(used, logq[torch.arange(hi - lo, device="cuda"), pick], 0.0), torch.where(used, ent, 0.0)]
            if case["top"]:
                got.append(logq.sort(1, descending=True).values[:, :case["top"]])
            if case["grad"]:
                gl = torch.where(used, s["g_logp"][lo:hi].double(), 0.0)[:, None]
                ge = torch.where(used, s["g_ent"][lo:hi].double(), 0.0)[:, None]
                d = -gl * q - ge * (plogq + q * ent[:, None])
                d[torch.arange(hi - lo, device="cuda"), pick] += gl[:, 0]
                got.append(d / case["temperature"])
            parts.append(tuple(got))
    cols = [torch.cat(c) for c in zip(*parts)]
    if op == "norm":
        grads = {"x": cols[2], "weight": dw}
        if case["residual"]:
            grads["residual"] = cols[2]
        return {"y": cols[0], "h": cols[1], "grads": grads}
    if op == "norm8":
        return {"y": cols[0], "scale": cols[1], "h": cols[2]}
    if op == "swiglu8":
        return {"y": cols[0], "scale": cols[1]}
    out = {"logp": cols[0], "entropy": cols[1]}
    if case["top"]:
        out["top_ids"], out["top_logp"] = None, cols[2]
    if case["grad"]:
        out["dlogits"] = cols[-1]
    return out
