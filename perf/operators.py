"""The operators of a decoded block, as cases that can be timed and compared: drawing a token for every slot
(``sample_tokens``), committing the surest slots (``unmask``) and orthogonalising the gradient that the write takes
(``newton_schulz``).  ``run`` computes them in a plain form of elementary torch operations, or, where ``own`` is true,
through the package's operators."""
import math

import torch

own = False
DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NS = (3.4445, -4.7750, 2.0315)          # the quintic of the Newton-Schulz iteration (the inner step's own coefficients)


# ------------------------------------------------------------------------------------------------------------ cases
def _sample(name, seqs, slots, vocab, dtype, temperature, top_k=0, top_p=1.0, min_p=0.0, bias=False, lead=False, priority="logp"):
    return dict(name=name, op="sample", seqs=seqs, slots=slots, vocab=vocab, dtype=dtype, temperature=temperature, top_k=top_k,
                top_p=top_p, min_p=min_p, bias=bias, lead=lead, priority=priority)


def _unmask(name, seqs, slots, part, sure):
    return dict(name=name, op="unmask", seqs=seqs, slots=slots, part=part, sure=sure)


def _ns(name, batch, rows, cols, dtype, steps, grad):
    return dict(name=name, op="ns", batch=batch, rows=rows, cols=cols, dtype=dtype, steps=steps, grad=grad)


def listed():
    return [
        # one open slot of one sequence: the last token of a block, where only latency counts
        _sample("sample 1 row", 1, 1, 128256, "f32", 0.8, top_p=0.9),
        # a whole block of the 1B configurations in one denoising round, nucleus sampling
        _sample("sample block top-p", 1, 1024, 128256, "f32", 0.7, top_p=0.9),
        # the same block drawn from the full distribution, slots ranked by entropy
        _sample("sample block full", 1, 1024, 128256, "f32", 1.0, priority="entropy"),
        # four sequences with presence penalties, logits kept in 16 bits, the outer shift's view of the block
        _sample("sample 4 seqs bf16", 4, 63, 128256, "bf16", 0.9, top_k=50, min_p=0.02, bias=True, lead=True),
        # greedy rounds of a small odd vocabulary with the margin as the priority
        _sample("sample greedy small", 8, 64, 1023, "f16", 0.0, priority="margin"),
        # one sequence's block: quota commit of a denoising round
        _unmask("unmask 1 x 1024", 1, 1024, False, False),
        # many sequences at once, sub-block filling and the probability threshold
        _unmask("unmask 256 x 1024", 256, 1024, True, True),
        # the write's gradients of the gate matrices of four fast-weight layers (1B configurations)
        _ns("ns 4 x 2048 x 8192", 4, 2048, 8192, "f32", 5, False),
        # a down matrix, tall, in training: the direction and its derivative
        _ns("ns 8192 x 2048 grad", 1, 8192, 2048, "bf16", 5, True),
        # odd sizes
        _ns("ns 3 x 509 x 1283 grad", 3, 509, 1283, "bf16", 5, True),
        # the smoke configuration's fast weights, two iterations
        _ns("ns 2 x 128 x 256", 2, 128, 256, "f32", 2, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("sample", "sample", "unmask", "ns", "ns"))
    if op == "sample":
        vocab = _log_int(rng, 1000, 160000)
        most = 1024 * 128256 // vocab
        seqs = _log_int(rng, 1, 16)
        slots = _log_int(rng, 1, max(1, min(1024, most // seqs)))
        t = rng.choice((0.0, rng.uniform(0.4, 1.5), rng.uniform(0.4, 1.5), rng.uniform(0.4, 1.5)))
        c = _sample("", seqs, slots, vocab, rng.choice(("f32", "f32", "bf16", "f16")), t, rng.choice((0, 0, _log_int(rng, 1, 500))),
                    rng.choice((1.0, rng.uniform(0.3, 0.99))), rng.choice((0.0, 0.0, rng.uniform(0.005, 0.3))), rng.random() < 0.3,
                    rng.random() < 0.3, rng.choice(("logp", "margin", "entropy")))
    elif op == "unmask":
        c = _unmask("", _log_int(rng, 1, 256), _log_int(rng, 16, 2048), rng.random() < 0.5, rng.random() < 0.5)
    else:
        steps = rng.randint(1, 5)
        rows, cols = _log_int(rng, 48, 4096), _log_int(rng, 48, 4096)
        batch = max(1, min(_log_int(rng, 1, 24), int(4 * 2048 ** 2 * 8192 / (min(rows, cols) ** 2 * max(rows, cols)))))
        dtype = rng.choice(("f32", "bf16"))
        c = _ns("", batch, rows, cols, dtype, steps, dtype == "bf16" and rng.random() < 0.6)
    del c["name"]
    return c


# ----------------------------------------------------------------------------------------------------------- inputs
def _logits(c, gen):
    """Head-shaped logits: Zipf-like with noise, from rows that hardly know (flatter than word frequencies) to sure ones; the
    mask token ruled out."""
    n, slots, vocab = c["seqs"], c["slots"] + int(c["lead"]), c["vocab"]
    order = torch.randperm(vocab, generator=gen, device=DEV)
    start = torch.randint(0, vocab, (n, slots, 1), generator=gen, device=DEV)
    sharp = 0.9 + 1.6 * torch.rand(n, slots, 1, generator=gen, device=DEV)
    x = -sharp * torch.log1p(((order + start) % vocab).float())
    x += 0.7 * torch.randn(n, slots, vocab, generator=gen, device=DEV)
    x[..., vocab - 1] = float("-inf")
    return x.to(DT[c["dtype"]])


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": c}
    if c["op"] == "sample":
        x = _logits(c, gen)
        s["logits"] = x[:, :-1] if c["lead"] else x
        s["u"] = torch.rand(c["seqs"], c["slots"], generator=gen, device=DEV)
        s["bias"] = None
        if c["bias"]:                       # a presence penalty: -0.5 on the tokens the sequence holds already
            seen = torch.rand(c["seqs"], c["vocab"], generator=gen, device=DEV) < 0.01
            s["bias"] = torch.where(seen, -0.5, 0.0)
    elif c["op"] == "unmask":
        b, n = c["seqs"], c["slots"]
        s["priority"] = torch.log(torch.rand(b, n, generator=gen, device=DEV).clamp_(1e-7))
        s["priority"] = torch.round(s["priority"] * 512) / 512          # ties, as quantised confidences have them
        s["logp"] = torch.log(torch.rand(b, n, generator=gen, device=DEV).clamp_(1e-7))
        s["tokens"] = torch.randint(0, 128000, (b, n), generator=gen, device=DEV)
        s["known"] = torch.rand(b, n, generator=gen, device=DEV) < 0.4
        s["ids"] = torch.where(s["known"], torch.randint(0, 128000, (b, n), generator=gen, device=DEV), 128002)
        s["held"] = torch.where(s["known"], -0.1, 0.0)
        s["quota"] = torch.randint(0, max(2, n // 4), (b,), generator=gen, device=DEV)
        s["allowed"] = (torch.rand(b, n, generator=gen, device=DEV) < 0.7) if c["part"] else None
        s["sure"] = math.log(0.9) if c["sure"] else None
    else:
        # a weight gradient: tokens x hidden activations against tokens x output gradients, the tokens unequal in size
        t = 2 * min(c["rows"], c["cols"])
        h = torch.randn(c["batch"], t, c["rows"], generator=gen, device=DEV)
        d = torch.randn(c["batch"], t, c["cols"], generator=gen, device=DEV)
        d *= torch.rand(c["batch"], t, 1, generator=gen, device=DEV) * 1e-3
        s["g"] = (h.transpose(1, 2) @ d).to(DT[c["dtype"]])
        s["gy"] = torch.randn(s["g"].shape, generator=gen, device=DEV).to(torch.bfloat16) if c["grad"] else None
    return s


# ------------------------------------------------------------------------------------------------------ plain forms
def _plain_sample(c, logits, u, bias):
    x = logits.float()
    if bias is not None:
        x = x + bias[:, None]
    # untempered: the drawn token's log-probability and the priority
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    if c["priority"] == "margin":
        top = x.topk(2, -1).values
        rank = ((top[..., 0] - m[..., 0]).exp() - (top[..., 1] - m[..., 0]).exp()) / z[..., 0]
    elif c["priority"] == "entropy":
        rank = (e * torch.where(torch.isfinite(x), x - m, 0.0)).sum(-1) / z[..., 0] - torch.log(z[..., 0])
    # tempered: masses in 64 bits, because a draw may fall next to a border between two tokens
    if c["temperature"] == 0:
        top = x.amax(-1, keepdim=True)
        tokens = (x == top).to(torch.int8).argmax(-1)
    else:
        w = torch.exp((x.double() - m.double()) / c["temperature"])
        if c["top_k"] or c["top_p"] < 1 or c["min_p"] > 0:
            order = torch.sort(x, dim=-1, descending=True, stable=True).indices         # equal values: lowest index first
            ws = w.gather(-1, order)
            keep = ws >= c["min_p"]
            if c["top_k"]:
                keep[..., c["top_k"]:] = False
                ws[..., c["top_k"]:] = 0
            if c["top_p"] < 1:
                before = ws.cumsum(-1) - ws
                keep &= before < c["top_p"] * ws.sum(-1, keepdim=True)
            w = w * torch.zeros_like(keep).scatter(-1, order, keep)
        cum = w.cumsum(-1)
        tokens = torch.searchsorted(cum, u.double()[..., None] * cum[..., -1:], right=True)[..., 0]
    logp = x.gather(-1, tokens[..., None])[..., 0] - m[..., 0] - torch.log(z[..., 0])
    return tokens, logp, logp if c["priority"] == "logp" else rank


def _plain_unmask(s):
    shut = s["known"] if s["allowed"] is None else s["known"] | ~s["allowed"]
    p = torch.where(shut, float("-inf"), s["priority"])
    rank = torch.argsort(torch.argsort(-p, dim=-1, stable=True), dim=-1)
    where = (rank < s["quota"][:, None]) & ~shut
    if s["sure"] is not None:
        where |= (s["logp"] >= s["sure"]) & ~s["known"]
    return (torch.where(where, s["tokens"], s["ids"]), s["known"] | where, torch.where(where, s["logp"], s["held"]), where)


def _ns_form(g, gy, steps, dtype):
    """``y = P g / |g|`` and, for a cotangent ``gy``, ``P gy / |g|`` (``P`` and the norm held constant)."""
    a, b, c = NS
    g = g.to(dtype)
    norm = g.norm(dim=(-2, -1), keepdim=True)
    x = g / norm
    wide = x.shape[-2] <= x.shape[-1]
    polys = []
    for _ in range(steps):
        gram = x @ x.mT if wide else x.mT @ x
        polys.append(b * gram + c * (gram @ gram))
        x = a * x + (polys[-1] @ x if wide else x @ polys[-1])
    if gy is None:
        return x, None
    r = gy.to(dtype) / norm
    for p in reversed(polys):
        r = a * r + (p @ r if wide else r @ p)
    return x, r


def run(state):
    s, c = state, state["case"]
    if c["op"] == "sample":
        if own:
            from dttt_b200.ops.sampling import sample_tokens
            out = sample_tokens(s["logits"], s["u"], temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"],
                                bias=s["bias"], priority=c["priority"])
            return tuple(out)
        return _plain_sample(c, s["logits"], s["u"], s["bias"])
    if c["op"] == "unmask":
        if own:
            from dttt_b200.ops.sampling import unmask
            out = unmask(s["ids"], s["known"], s["held"], s["tokens"], s["logp"], s["priority"], s["quota"], allowed=s["allowed"],
                         sure=s["sure"])
            return tuple(out)
        return _plain_unmask(s)
    if own:
        from dttt_b200.ops.newton_schulz import newton_schulz
        if not c["grad"]:
            return newton_schulz(s["g"], steps=c["steps"])
        g = s["g"].detach().requires_grad_(True)
        y = newton_schulz(g, steps=c["steps"])
        return y.detach(), torch.autograd.grad(y, g, s["gy"])[0]
    x, r = _ns_form(s["g"], s["gy"], c["steps"], torch.float32)
    if r is None:
        return x.to(torch.bfloat16)
    return x.to(torch.bfloat16), r.to(s["g"].dtype)


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "sample":
        rows = c["seqs"] * c["slots"]
        return {"bytes": rows * (c["vocab"] * (4 if c["dtype"] == "f32" else 2) + 4 + 16) + (c["seqs"] * c["vocab"] * 4 if c["bias"] else 0),
                "flops": 4 * rows * c["vocab"]}
    if c["op"] == "unmask":
        # read: priority, logp, ids, tokens, known, committed logp, quota; write: ids, known, committed logp, the pick
        return {"bytes": c["seqs"] * (c["slots"] * (4 + 4 + 8 + 8 + 1 + 4 + int(c["part"]) + 8 + 1 + 4 + 1) + 8), "flops": c["seqs"] * c["slots"]}
    m, n = sorted((c["rows"], c["cols"]))
    # per step: one half of a symmetric m x n x m product, one half of a symmetric m x m x m one, a full m x m x n one
    flops = c["steps"] * (m * m * n + m ** 3 + 2 * m * m * n) + (c["steps"] * 2 * m * m * n if c["grad"] else 0)
    size = 4 if c["dtype"] == "f32" else 2
    return {"bytes": c["batch"] * m * n * ((size + 2) + ((2 + size) if c["grad"] else 0)), "flops": c["batch"] * flops}


# ------------------------------------------------------------------------------------------------------------ exact
def _exact_rows(c, x, u):
    """A handful of rows ``x [R, V]`` (64 bits): tokens, log-probabilities, priorities, by rank."""
    m = x.max(-1, keepdim=True).values
    logz = torch.logsumexp(x, -1, keepdim=True)
    logp = x - logz
    if c["temperature"] == 0:
        tokens = torch.where(x == m, torch.arange(x.shape[1], device=x.device), x.shape[1]).min(-1).values
    else:
        v, idx = torch.sort(x, dim=-1, descending=True, stable=True)
        w = torch.exp((v - m) / c["temperature"])
        count = torch.full((x.shape[0], 1), c["top_k"] or x.shape[1], device=x.device)
        rank = torch.arange(x.shape[1], device=x.device)[None]
        w = torch.where(rank < count, w, 0.0)
        if c["top_p"] < 1:
            whole = w.sum(-1, keepdim=True)
            w = torch.where(torch.cat([torch.zeros_like(whole), w.cumsum(-1)[:, :-1]], -1) < c["top_p"] * whole, w, 0.0)
        w = torch.where(w >= max(c["min_p"], 0.0), w, 0.0)
        back = torch.empty_like(w).scatter_(-1, idx, w)
        cum = back.cumsum(-1)
        tokens = (cum <= u[:, None] * cum[:, -1:]).sum(-1)
    chosen = logp.gather(-1, tokens[:, None])[:, 0]
    if c["priority"] == "logp":
        return tokens, chosen, chosen
    if c["priority"] == "margin":
        two = torch.sort(x, dim=-1, descending=True).values[:, :2]
        return tokens, chosen, torch.exp(two[:, 0] - logz[:, 0]) - torch.exp(two[:, 1] - logz[:, 0])
    return tokens, chosen, torch.special.xlogy(torch.exp(logp), torch.exp(logp)).sum(-1)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "sample":
        x, u = s["logits"], s["u"].double()
        if s["bias"] is not None:
            x = x.float() + s["bias"][:, None]          # the sum's rounding to 32 bits is part of the definition
        parts = [_exact_rows(c, x[i, j:j + 128].double(), u[i, j:j + 128]) for i in range(c["seqs"]) for j in range(0, c["slots"], 128)]
        return tuple(torch.cat(p).view(c["seqs"], c["slots"]) for p in zip(*parts))
    if c["op"] == "unmask":
        n = c["slots"]
        shut = s["known"] | (~s["allowed"] if s["allowed"] is not None else False)
        key = torch.where(shut, float("-inf"), s["priority"]).double()
        slot = torch.arange(n, device=DEV)
        where = torch.empty_like(s["known"])
        for i in range(c["seqs"]):
            ahead = (key[i][None] > key[i][:, None]) | ((key[i][None] == key[i][:, None]) & (slot[None] < slot[:, None]))
            where[i] = (ahead.sum(1) < s["quota"][i]) & ~shut[i]
        if s["sure"] is not None:
            where |= (s["logp"] >= s["sure"]) & ~s["known"]
        return (torch.where(where, s["tokens"], s["ids"]), s["known"] | where, torch.where(where, s["logp"].double(), s["held"].double()), where)
    # by the matrix's singular values: the iteration is an odd polynomial of each
    if min(c["rows"], c["cols"]) > 1024:
        x, r = _ns_form(s["g"], s["gy"], c["steps"], torch.float64)
        return x if r is None else (x, r)
    g = s["g"].double()
    w, v = torch.linalg.eigh(g @ g.mT if c["rows"] <= c["cols"] else g.mT @ g)
    norm = g.square().sum((-2, -1)).sqrt()
    sv = w.clamp_min(0).sqrt() / norm[:, None]
    gain = torch.ones_like(sv)
    for _ in range(c["steps"]):
        step = NS[0] + NS[1] * sv ** 2 + NS[2] * sv ** 4
        gain, sv = gain * step, sv * step
    gain = gain / norm[:, None]
    p = (v * gain[:, None, :]) @ v.mT
    apply = (lambda t: p @ t) if c["rows"] <= c["cols"] else (lambda t: t @ p)
    return apply(g) if s["gy"] is None else (apply(g), apply(s["gy"].double()))
