"""The operators of the networks' training, and what is measured of them.

Three operators that a training step of a token network chains: LayerNorm with the residual add before
it (forward and backward), log probabilities of given tokens with entropy and top alternatives (forward
and backward), and an AdamW step over many tensors at once.  `run` has each in its plain form,
elementary torch operations in 32 bits, and as the call of the framework's operator (`own`).

Definitions shared by both forms:

  layer norm   s = x + delta rounded to the tensors' type; y = (s - mean) / sqrt(var + eps) * w + b over
               the last dimension; gradients of y and of s flow into x (delta's gradient is x's).
  log probs    z = logits / temperature, masked entries -inf; logprobs = z[token] - logsumexp(z), a
               negative padding token gives 0; entropy = -sum p log p; the top tokens by descending
               logit, equal ones by ascending index, -1 (and -inf) behind the last allowed one.  A row
               with nothing allowed has entropy 0, log probabilities -inf and no gradient.
  AdamW        decoupled weight decay, bias-corrected moments.  Tensors lie in flat buffers, each at the
               next multiple of 256 elements.  8-bit states: e4m3 codes of m and of sqrt(v) with one f32
               scale (largest magnitude / 448) for each 256 elements; a positive sqrt(v) is not rounded
               to zero; the step itself uses the moments before they are rounded.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256


def listed():
    norm = {"op": "norm", "type": "f32", "rows": 62, "d": 160, "residual": False, "grad": False}
    logp = {"op": "logp", "type": "f32", "rows": 1, "vocab": 39, "n": 1, "top": 0, "mask": False, "grad": False, "temperature": 1.0}
    adam = {"op": "adamw", "type": "f32", "bits": 32, "master": False, "tensors": 1, "size": 0, "d": 0, "layers": 0, "classes": 0}
    return [
        # one information state through a norm of the AlphaZero network: 62 tokens, latency alone
        dict(norm, name="norm one state"),
        # a training batch of 512 positions of the IMPI network (d 256), as every half block has it
        dict(norm, name="norm network training", rows=512 * 62, d=256, residual=True, grad=True),
        # a wide model's training batch in bf16
        dict(norm, name="norm wide training", type="bf16", rows=16384, d=4096, residual=True, grad=True),
        # rows that start at no alignment: an odd width in fp16, norm alone
        dict(norm, name="norm odd width", type="f16", rows=5003, d=1111, grad=True),
        # the policy loss of an AlphaZero batch: all 39 actions under the mask of the legal ones
        dict(logp, name="logp policy loss", rows=8192, n=39, top=3, mask=True, grad=True),
        # one decoded token of a large vocabulary with its 20 best alternatives
        dict(logp, name="logp one token", type="bf16", vocab=131072, top=20),
        # the loss of a language model's training batch, an odd vocabulary
        dict(logp, name="logp vocabulary loss", type="bf16", rows=4096, vocab=65537, grad=True),
        # scoring a given prompt in f32 at a sampling temperature, with its five best alternatives
        dict(logp, name="logp prompt scores", rows=700, vocab=32003, top=5, temperature=0.7),
        # a step of the AlphaZero network: 6 blocks of d 160, heads of 4 + 39 classes, ~100 tensors
        dict(adam, name="adamw network", d=160, layers=6, classes=43),
        # a step of the IMPI network with states in 8 bits
        dict(adam, name="adamw network 8 bits", bits=8, d=256, layers=4, classes=33),
        # a large model's shard: bf16 weights with f32 masters
        dict(adam, name="adamw large masters", type="bf16", master=True, tensors=8, size=8 << 20),
        # a large model's shard with states in 8 bits, odd sizes
        dict(adam, name="adamw large 8 bits", bits=8, tensors=9, size=7000003),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "logp", "adamw"))
    kind = rng.choice(("f32", "bf16", "f16"))
    if op == "norm":
        d = _log(rng, 17, 8192)
        most = min(200000, (1 << 26) // d)
        return {"op": op, "type": kind, "rows": _log(rng, 1, most), "d": d, "residual": rng.random() < 0.5, "grad": rng.random() < 0.7}
    if op == "logp":
        vocab = _log(rng, 5, 131072)
        most = max(1, min(100000, (1 << 27) // vocab))
        grad = rng.random() < 0.5
        return {"op": op, "type": kind, "rows": _log(rng, 1, most), "vocab": vocab, "n": rng.choice((1, 1, 1, 2, 7, 33)),
                "top": min(vocab, rng.choice((0, 0, 1, 5, 20, 32))), "mask": rng.random() < 0.3, "grad": grad,
                "temperature": rng.choice((1.0, 1.0, 0.6, 1.5))}
    bits, tensors = rng.choice((32, 8)), _log(rng, 1, 150)
    return {"op": op, "type": kind, "bits": bits, "master": kind != "f32" and rng.random() < 0.7, "tensors": tensors,
            "size": _log(rng, 33, (1 << 25) // tensors), "d": 0, "layers": 0, "classes": 0}


def _sizes(case):
    """Elements of each tensor of an AdamW case: a token network's tensors, or `tensors` of about `size`."""
    d, c = case["d"], case["classes"]
    if not d:
        return [case["size"] + 7 * (i % 5) for i in range(case["tensors"])]
    block = [d, d, 3 * d * d, 3 * d, d * d, d, d * d, d, d, d, 4 * d * d, 4 * d, 4 * d * d, d]
    return [v * d for v in (43, 57, 5, 13, 3, 3)] + block * case["layers"] + [d, d, c * d, c * d, c * d, c * d * d, c * d, c * d, c]


def _places(case):
    """(offset, elements) of each tensor in the flat buffers, and the buffers' length."""
    got, at = [], 0
    for n in _sizes(case):
        got.append((at, n))
        at += -(-n // BLOCK) * BLOCK
    return got, at


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0, to=t):
        return torch.empty(shape, device=dev).normal_(shift, scale, generator=g).to(to)

    state = {"case": case}
    if case["op"] == "norm":
        rows, d = case["rows"], case["d"]
        # a residual stream: columns with an offset of their own
        state["x"] = (normal(rows, d, scale=2.0, to=torch.float32) + normal(d, to=torch.float32)).to(t)
        state["delta"] = normal(rows, d) if case["residual"] else None
        state["w"], state["b"] = normal(d, scale=0.1, shift=1.0), normal(d, scale=0.1)
        if case["grad"]:
            state["dy"] = normal(rows, d, scale=0.02)
            state["ds"] = normal(rows, d, scale=0.02) if case["residual"] else None
            for k in ("x", "delta", "w", "b"):
                if state[k] is not None:
                    state[k].requires_grad_()
        return state
    if case["op"] == "logp":
        rows, vocab, n = case["rows"], case["vocab"], case["n"]
        state["logits"] = normal(rows, vocab, scale=2.5, to=torch.float32).add_(normal(rows, 1, scale=3.0, to=torch.float32)).to(t)
        tokens = torch.randint(0, vocab, (rows, n), device=dev, generator=g)
        if n == vocab:
            tokens = torch.arange(vocab, device=dev).expand(rows, n).contiguous()
        else:  # some rows are padded
            tokens = torch.where(torch.rand(rows, 1, device=dev, generator=g) < 0.05, torch.full_like(tokens, -100), tokens)
        state["tokens"], state["mask"] = tokens, None
        if case["mask"]:  # about a third is allowed, in some rows nothing
            allowed = torch.rand(rows, vocab, device=dev, generator=g) < 0.35
            allowed &= torch.rand(rows, 1, device=dev, generator=g) > 0.01
            state["mask"] = allowed
        if case["grad"]:  # of a mean over the rows; fp16 training scales its loss
            scale = (1024.0 if t == torch.float16 else 1.0) / rows
            state["dlogp"] = normal(rows, n, scale=scale, to=torch.float32)
            state["dent"] = normal(rows, scale=0.01 * scale, to=torch.float32)
            state["logits"].requires_grad_()
        return state
    places, total = _places(case)
    live = torch.zeros(total, device=dev, dtype=torch.bool)
    for at, n in places:
        live[at:at + n] = True

    def flat(scale, to=torch.float32):
        return torch.where(live, normal(total, scale=scale, to=torch.float32), 0.0).to(to)

    state["hyper"] = {"lr": 1e-3, "betas": (0.9, 0.99), "eps": 1e-8, "weight_decay": 0.01}
    master = flat(0.05)
    state["p"] = master.to(t)
    state["master"] = master if case["master"] else None
    state["g"] = flat(1e-3, t)
    state["step"] = torch.full((), 7, device=dev, dtype=torch.int32)
    m, v = flat(3e-4), flat(1e-3).square_()
    if case["bits"] == 8:
        state["m"], state["m_scale"] = _quantised(m, False)
        state["v"], state["v_scale"] = _quantised(v.sqrt(), True)
    else:
        state["m"], state["v"] = m, v
    if own:
        from master_doko_reinforcement_learning_amd import AdamW
        params = []
        for at, n in places:
            p = state["p"][at:at + n].detach().requires_grad_()
            p.grad = state["g"][at:at + n]
            params.append(p)
        opt = AdamW(params, state_bits=case["bits"], master_weights=case["master"], **state["hyper"])
        b = opt.buffers[0]
        b["step"].fill_(7)
        b["exp_avg"].copy_(state["m"])
        b["exp_avg_sq"].copy_(state["v"])
        if case["bits"] == 8:
            b["exp_avg_scale"].copy_(state["m_scale"])
            b["exp_avg_sq_scale"].copy_(state["v_scale"])
        if case["master"]:
            b["master"].copy_(master)
        state["opt"] = opt
    return state


def run(state):
    return {"norm": _norm, "logp": _logp, "adamw": _adamw}[state["case"]["op"]](state)


def _norm(s):
    x, delta, w, b, grad = s["x"], s["delta"], s["w"], s["b"], s["case"]["grad"]
    if own:
        from master_doko_reinforcement_learning_amd import layer_norm
        new, y = layer_norm(x, w, b, EPS, delta=delta) if delta is not None else (None, layer_norm(x, w, b, EPS))
        out = {"y": y, "x": new}
        if grad:
            outs, douts = ([y], [s["dy"]]) if delta is None else ([y, new], [s["dy"], s["ds"]])
            out["dx"], out["dw"], out["db"] = torch.autograd.grad(outs, [x, w, b], douts)
        return out
    with torch.no_grad():
        t = x.dtype
        new = x if delta is None else (x.float() + delta.float()).to(t)
        f, w, b = new.float(), w.float(), b.float()
        f = f - f.mean(-1, keepdim=True)
        r = 1.0 / torch.sqrt((f * f).mean(-1, keepdim=True) + EPS)
        f = f * r
        out = {"y": (f * w + b).to(t), "x": None if delta is None else new}
        if grad:
            dy = s["dy"].float()
            h = dy * w
            dx = r * (h - h.mean(-1, keepdim=True) - f * (h * f).mean(-1, keepdim=True))
            out["dx"] = (dx if delta is None else dx + s["ds"].float()).to(t)
            out["dw"], out["db"] = (dy * f).sum(0).to(t), dy.sum(0).to(t)
        return out


def _logp(s):
    c, logits, tokens, mask = s["case"], s["logits"], s["tokens"], s["mask"]
    if own:
        from master_doko_reinforcement_learning_amd import token_logprobs
        got = token_logprobs(logits, tokens, mask=mask, temperature=c["temperature"], top=c["top"])
        out = {"logprobs": got.logprobs, "entropy": got.entropy}
        if c["top"]:
            out["top_logprobs"], out["top_tokens"] = got.top_logprobs, got.top_tokens
        if c["grad"]:
            out["dlogits"], = torch.autograd.grad([got.logprobs, got.entropy], [logits], [s["dlogp"], s["dent"]])
        return out
    with torch.no_grad():
        z = logits.float()
        if mask is not None:
            z = torch.where(mask, z, -math.inf)
        out = {}
        if c["top"]:
            best, at = torch.sort(z, dim=-1, descending=True, stable=True)
            best, at = best[:, :c["top"]], at[:, :c["top"]]
        z = z / c["temperature"]
        most = z.amax(-1, keepdim=True)
        empty = most == -math.inf
        most = torch.where(empty, 0.0, most)
        e = torch.exp(z - most)
        lse = most + torch.log(e.sum(-1, keepdim=True))
        logp = z - lse
        p = torch.where(empty, 0.0, torch.exp(logp))
        del e
        # p log p is 0 where p is; log p there may be -inf
        finite = torch.where(z == -math.inf, 0.0, logp)
        entropy = -(p * finite).sum(-1, keepdim=True)
        pad = tokens < 0
        given = torch.where(empty, -math.inf, logp).gather(-1, tokens.clamp(min=0))
        out["logprobs"], out["entropy"] = torch.where(pad, 0.0, given), entropy[:, 0]
        if c["top"]:
            gone = best == -math.inf
            out["top_tokens"] = torch.where(gone, -1, at)
            out["top_logprobs"] = torch.where(gone, -math.inf, best / c["temperature"] - lse)
        if c["grad"]:
            g = torch.where(pad | torch.isinf(given), 0.0, s["dlogp"])
            d = -p * (g.sum(-1, keepdim=True) + s["dent"][:, None] * (finite + entropy))
            d.scatter_add_(-1, tokens.clamp(min=0), g)
            out["dlogits"] = (d / c["temperature"]).to(logits.dtype)
        return out


def _quantised(x, positive):
    """(e4m3 codes, scales) of a flat f32 tensor by blocks."""
    blocks = x.view(-1, BLOCK)
    most = blocks.abs().amax(-1)
    most = torch.where(most < 1e-30, 0.0, most)
    q = blocks * torch.where(most > 0, 448.0 / most, 0.0)[:, None]
    code = q.to(torch.float8_e4m3fn)
    if positive:
        code = torch.where(q > 0, code.float().clamp(min=2.0 ** -9), 0.0).to(torch.float8_e4m3fn)
    return code.view(-1), most * (1.0 / 448.0)


def _value(code, scale):
    return (code.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _adamw(s):
    c, h = s["case"], s["hyper"]
    eight = c["bits"] == 8
    if own:
        s["opt"].step()
        b = s["opt"].buffers[0]
        out = {"p": s["p"], "m": b["exp_avg"], "v": b["exp_avg_sq"]}
        if eight:
            out["m_scale"], out["v_scale"] = b["exp_avg_scale"], b["exp_avg_sq_scale"]
        if c["master"]:
            out["master"] = b["master"]
        return out
    with torch.no_grad():
        b1, b2 = h["betas"]
        s["step"] += 1
        t = s["step"].double()
        size, root = (h["lr"] / (1 - b1 ** t)).float(), torch.sqrt(1 - b2 ** t).float()
        g = s["g"].float()
        m = _value(s["m"], s["m_scale"]) if eight else s["m"]
        v = _value(s["v"], s["v_scale"]).square() if eight else s["v"]
        m = m * b1 + g * (1 - b1)
        v = v * b2 + g * g * (1 - b2)
        p = s["master"] if c["master"] else s["p"].float()
        p = p * (1 - h["lr"] * h["weight_decay"]) - size * (m / (torch.sqrt(v) / root + h["eps"]))
        if c["master"]:
            s["master"].copy_(p)
        s["p"].copy_(p)
        if eight:
            s["m"], s["m_scale"] = _quantised(m, False)
            s["v"], s["v_scale"] = _quantised(torch.sqrt(v), True)
        else:
            s["m"], s["v"] = m, v
        out = {"p": s["p"], "m": s["m"], "v": s["v"]}
        if eight:  # an e4m3 code is a value; what it stands for is that times its block's scale
            out["m_scale"], out["v_scale"] = s["m_scale"], s["v_scale"]
        if c["master"]:
            out["master"] = s["master"]
        return out


def work(case):
    e = TYPES[case["type"]].itemsize
    if case["op"] == "norm":
        n = case["rows"] * case["d"]
        moved = (2 + 2 * case["residual"]) + case["grad"] * (2 + case["residual"])
        return {"bytes": e * (n * moved + case["d"] * (2 + 2 * case["grad"])), "flops": n * (8 + 14 * case["grad"])}
    if case["op"] == "logp":
        rows, n = case["rows"], case["rows"] * case["vocab"]
        small = rows * (case["n"] * (12 + 4 * case["grad"]) + 4 + 4 * case["grad"] + 12 * case["top"])
        return {"bytes": n * (e * (1 + case["grad"]) + case["mask"]) + small, "flops": n * (6 + 8 * case["grad"])}
    n = sum(_sizes(case))
    each = e + (8 + e if case["master"] else 2 * e) + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)
    return {"bytes": n * each, "flops": n * 16}


def exact(case, seed):
    global own
    mine, own = own, False
    s = prepare(case, seed)  # the inputs alone
    own = mine
    return {"norm": _exact_norm, "logp": _exact_logp, "adamw": _exact_adamw}[case["op"]](case, s)


@torch.no_grad()
def _exact_norm(case, s):
    t = s["x"].dtype
    x = s["x"].double()
    if case["residual"]:  # the sum is a value of the tensors' type, so the norm of it is defined by its rounding
        x = (x + s["delta"].double()).to(t).double()
    w, b = s["w"].double(), s["b"].double()
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    std = (var + EPS).sqrt()
    n = (x - mean) / std
    out = {"y": torch.addcmul(b, n, w), "x": x if case["residual"] else None}
    if case["grad"]:
        dy = s["dy"].double()
        # the Jacobian of a normalised row, applied: (I - 1 1'/d - n n'/d) (w dy) / std
        u = dy * w
        d = case["d"]
        u = u - u.sum(-1, keepdim=True) / d - n * ((u * n).sum(-1, keepdim=True) / d)
        u = u / std
        out["dx"] = u + s["ds"].double() if case["residual"] else u
        out["dw"], out["db"] = (dy * n).sum(0), dy.sum(0)
    return out


@torch.no_grad()
def _exact_logp(case, s):
    x = s["logits"].double() / case["temperature"]
    if s["mask"] is not None:
        x = x.masked_fill(~s["mask"], -math.inf)
    lp = torch.log_softmax(x, -1)
    none = torch.isneginf(x).all(-1, keepdim=True)
    lp = lp.masked_fill(none, -math.inf)
    p = lp.exp()
    weighted = torch.nan_to_num(lp, neginf=0.0)
    entropy = -(p * weighted).sum(-1)
    tokens = s["tokens"]
    valid = tokens >= 0
    picked = lp.gather(1, tokens.clamp(min=0))
    out = {"logprobs": picked.masked_fill(~valid, 0.0), "entropy": entropy}
    if case["top"]:
        out["top_logprobs"] = lp.sort(-1, descending=True).values[:, :case["top"]]
        out["top_tokens"] = None
    if case["grad"]:
        g = s["dlogp"].double().masked_fill(~valid | picked.isneginf(), 0.0)
        d = torch.zeros_like(p).scatter_add_(1, tokens.clamp(min=0), g)
        d -= p * g.sum(1, keepdim=True)
        d -= p * (weighted + entropy[:, None]) * s["dent"].double()[:, None]
        out["dlogits"] = d / case["temperature"]
    return out


@torch.no_grad()
def _exact_adamw(case, s):
    h = s["hyper"]
    b1, b2 = h["betas"]
    t = int(s["step"]) + 1
    g, m, v = s["g"].double(), s["m"].double(), s["v"].double()
    eight = case["bits"] == 8
    if eight:
        m = m * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (v * s["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g * g, v, b2)
    p = s["master"].double() if case["master"] else s["p"].double()
    hat = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + h["eps"])
    p = p - h["lr"] * (hat + h["weight_decay"] * p)
    out = {"p": p, "m": m, "v": v}
    if eight:
        out["m"], out["m_scale"] = _exact_codes(m)
        root, out["v_scale"] = _exact_codes(v.sqrt())
        out["v"] = torch.where(v > 0, root.clamp(min=2.0 ** -9), 0.0)
    if case["master"]:
        out["master"] = p
    return out


def _exact_codes(x):
    """Nearest e4m3 values (3 bits behind the leading one, least exponent -6) of x / scale, and the scales."""
    scale = x.view(-1, BLOCK).abs().amax(1) / 448
    q = x / scale.repeat_interleave(BLOCK).clamp(min=1e-300)
    step = torch.exp2(torch.frexp(q)[1].clamp(min=-5).double() - 4)
    return torch.round(q / step) * step, scale
