"""The two ends of the tied complex table, one pass each, for timing and for
comparing outputs: token ids in (the embedding lookup with scaling and its
gradient) and token log-probabilities out (from logits, and from hidden rows
and the table without logits), with entropy, top alternatives and gradients.

`listed()` names the cases, `draw(rng)` gives others of the same ranges.  With
`own` false a pass is computed in plain torch operations in 32 bits; with `own`
true it is the framework's call.  `exact` computes a case from the definitions
in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "bf16": 2}
IGNORE = -100
MOST_LOGITS = 16384 * 50261             # entries of the largest [rows, vocabulary] product
MOST_PRODUCT = MOST_LOGITS * 1024 * 3   # multiply-adds of the largest training case


def listed():
    return [
        # the tokens of one decode step of 192 live sequences: latency of one lookup
        dict(name="embed_step_fp32", kind="embed", n=192, V=50261, dim=768, dtype="fp32", grad=False),
        # the lookup of a training batch and the gradient of both tables, tokens as text has them
        dict(name="embed_train_bf16", kind="embed", n=16384, V=50261, dim=512, dtype="bf16", grad=True),
        # fine-tuning on a ragged batch with fp32 master tables
        dict(name="embed_train_fp32", kind="embed", n=3001, V=32003, dim=768, dtype="fp32", grad=True),
        # one sequence's decode step: the drawn token and five alternatives
        dict(name="logprobs_one_fp32", kind="logprobs", n=1, V=50261, dtype="fp32", k=5, temperature=1.0, masked=0.0,
             grad=False),
        # a decode step of 192 live sequences under a grammar that forbids half the vocabulary
        dict(name="logprobs_step_fp32", kind="logprobs", n=192, V=50261, dtype="fp32", k=20, temperature=0.7, masked=0.5,
             grad=False),
        # the rows of a long prompt, bf16 logits (many equal values), alternatives for each position
        dict(name="logprobs_prompt_bf16", kind="logprobs", n=4000, V=50261, dtype="bf16", k=5, temperature=1.0, masked=0.0,
             grad=False),
        # distillation and policy gradients on logits: values and the gradient of the logits
        dict(name="logprobs_train_fp32", kind="logprobs", n=2048, V=50261, dtype="fp32", k=0, temperature=1.0, masked=0.0,
             grad=True),
        # scoring the tokens of a decode step from the head's rows
        dict(name="linear_step_bf16", kind="linear", n=16, V=50261, D=1536, dtype="bf16", temperature=1.0, grad=False),
        # scoring a ragged prompt
        dict(name="linear_prompt_bf16", kind="linear", n=2047, V=50261, D=1536, dtype="bf16", temperature=1.0, grad=False),
        # a policy-gradient step with an entropy term over a full training batch
        dict(name="linear_train_bf16", kind="linear", n=16384, V=50261, D=1024, dtype="bf16", temperature=1.0, grad=True),
        # the same in fp32 at a small vocabulary and ragged sizes
        dict(name="linear_train_fp32", kind="linear", n=1000, V=8191, D=768, dtype="fp32", temperature=0.8, grad=True),
    ]


def _span(rng, lo, hi):
    """An integer of [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed", "logprobs", "linear"])
    dtype, grad = rng.choice(["fp32", "bf16"]), rng.random() < 0.5
    if kind == "embed":
        return dict(kind=kind, n=_span(rng, 1, 32768), V=_span(rng, 1000, 100000), dim=_span(rng, 32, 1024), dtype=dtype,
                    grad=grad)
    if kind == "logprobs":
        V = _span(rng, 1000, 160000)
        return dict(kind=kind, n=min(_span(rng, 1, 8192), MOST_LOGITS // V), V=V, dtype=dtype,
                    k=0 if grad else rng.choice([0, 1, 5, 20, 32]), temperature=round(rng.uniform(0.5, 1.5), 2),
                    masked=rng.choice([0.0, 0.0, 0.5, 0.9]), grad=grad)
    D, V = 32 * _span(rng, 2, 60), _span(rng, 1000, 60000)
    most = MOST_PRODUCT // (3 if grad else 1) // (8 if dtype == "fp32" else 1)
    return dict(kind=kind, n=min(_span(rng, 1, 16384), MOST_LOGITS // V, most // (V * D)), V=V, D=D, dtype=dtype,
                temperature=round(rng.uniform(0.7, 1.3), 2), grad=grad)


# ---------------------------------------------------------------- inputs

def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.empty(*shape, device=DEV, dtype=torch.float32).normal_(0.0, std, generator=g).to(dtype)


def _text_ids(g, n, V):
    """Token ids with the frequencies of text: rank r about 1 / (r + 2.7)."""
    p = 1.0 / (torch.arange(V, device=DEV, dtype=torch.float64) + 2.7)
    cdf = (p / p.sum()).cumsum(0)
    u = torch.rand(n, device=DEV, generator=g, dtype=torch.float64)
    rank = torch.searchsorted(cdf, u).clamp_(max=V - 1)
    return (rank * 7919 + 13) % V if V % 7919 else rank    # a frequent token is anywhere in the table


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[c["dtype"]]
    s = dict(case=c)
    if c["kind"] == "embed":
        s["ids"] = _text_ids(g, c["n"], c["V"])
        s["re"], s["im"] = (_randn(g, c["V"], c["dim"], std=0.02, dtype=dt).requires_grad_(c["grad"]) for _ in range(2))
        s["scale"] = math.sqrt(c["dim"])
        if c["grad"]:
            s["dz"] = _randn(g, c["n"], c["dim"], 2, std=1.0 / c["n"], dtype=dt)
        return s
    n, V = c["n"], c["V"]
    s["ids"] = torch.randint(0, V, (n,), device=DEV, generator=g)
    if n > 1:
        s["ids"][torch.rand(n, device=DEV, generator=g) < 0.1] = IGNORE    # prompt and padding rows
    if c["kind"] == "logprobs":
        x = _randn(g, n, V, std=2.5)
        x[torch.arange(n, device=DEV), torch.randint(0, V, (n,), device=DEV, generator=g)] += 10.0   # a likely token
        if c["masked"]:
            x.masked_fill_(torch.rand(V, device=DEV, generator=g) < c["masked"], float("-inf"))
        s["logits"] = x.to(dt).requires_grad_(c["grad"])
    else:
        s["h"] = _randn(g, n, c["D"], dtype=dt).requires_grad_(c["grad"])
        s["w"] = _randn(g, V, c["D"], std=2.5 / math.sqrt(c["D"]), dtype=dt).requires_grad_(c["grad"])
    if c["grad"]:
        s["g_lp"], s["g_ent"] = _randn(g, n, std=1.0 / n), _randn(g, n, std=0.1 / n)
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    return (_own if own else _plain)[state["case"]["kind"]](state)


def _own_embed(s):
    from qllm2_amd.embedding import complex_embedding
    z = complex_embedding(s["ids"], s["re"], s["im"], scale=s["scale"])
    out = {"z": z}
    if s["case"]["grad"]:
        out["d_re"], out["d_im"] = torch.autograd.grad(z, [s["re"], s["im"]], s["dz"])
    return out


def _own_logprobs(s):
    from qllm2_amd.token_logprobs import token_logprobs
    c = s["case"]
    r = token_logprobs(s["logits"], s["ids"], temperature=c["temperature"], top_k=c["k"], ignore_index=IGNORE)
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if c["k"]:
        out["top_logprobs"], out["top_ids"] = r.top_logprobs, r.top_ids
    if c["grad"]:
        out["d_logits"], = torch.autograd.grad([r.logprobs, r.entropy], [s["logits"]], [s["g_lp"], s["g_ent"]])
    return out


def _own_linear(s):
    from qllm2_amd.token_logprobs import linear_token_logprobs
    c = s["case"]
    r = linear_token_logprobs(s["h"], s["w"], s["ids"], temperature=c["temperature"], ignore_index=IGNORE)
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if c["grad"]:
        out["d_h"], out["d_w"] = torch.autograd.grad([r.logprobs, r.entropy], [s["h"], s["w"]], [s["g_lp"], s["g_ent"]])
    return out


def _plain_embed(s):
    re, im, ids, scale = s["re"].detach(), s["im"].detach(), s["ids"], s["scale"]
    out = {"z": (torch.stack((re[ids], im[ids]), -1).float() * scale).to(re.dtype)}
    if s["case"]["grad"]:
        g = torch.zeros(*re.shape, 2, device=re.device).index_add_(0, ids, s["dz"].float()) * scale
        out["d_re"], out["d_im"] = (g[..., i].to(re.dtype) for i in (0, 1))
    return out


def _statistics(x, ids):
    """Log probabilities of every entry, of the given tokens, probabilities, and the entropy, of fp32 rows x."""
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    valid = ids != IGNORE
    safe = torch.where(valid, ids, 0)
    lp = torch.where(valid, logp.gather(1, safe[:, None])[:, 0], 0.0)
    ent = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    return logp, p, valid, safe, lp, ent


def _grad_logits(s, logp, p, valid, safe, ent):
    """d logprobs / dx_v = [v = token] - p_v,  d entropy / dx_v = -p_v (log p_v + H)."""
    g_lp = torch.where(valid, s["g_lp"], 0.0)[:, None]
    gx = -p * (g_lp + s["g_ent"][:, None] * torch.where(p > 0, logp + ent[:, None], 0.0))
    return gx.scatter_add_(1, safe[:, None], g_lp) / s["case"]["temperature"]


def _plain_logprobs(s):
    c, logits = s["case"], s["logits"].detach()
    x = logits.float() / c["temperature"]
    logp, p, valid, safe, lp, ent = _statistics(x, s["ids"])
    out = {"logprobs": lp, "entropy": ent}
    if c["k"]:
        # keys that order by value and, among equal values, by the lower index
        b = (logits.float() + 0.0).view(torch.int32)
        b = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long()
        key = b * 2 ** 32 + (2 ** 31 - torch.arange(c["V"], device=b.device))
        out["top_ids"] = key.topk(c["k"], -1).indices
        out["top_logprobs"] = logp.gather(1, out["top_ids"])
    if c["grad"]:
        out["d_logits"] = _grad_logits(s, logp, p, valid, safe, ent).to(logits.dtype)
    return out


def _plain_linear(s):
    c = s["case"]
    h, w = s["h"].detach().float(), s["w"].detach().float()
    logp, p, valid, safe, lp, ent = _statistics(h @ w.T / c["temperature"], s["ids"])
    out = {"logprobs": lp, "entropy": ent}
    if c["grad"]:
        gx = _grad_logits(s, logp, p, valid, safe, ent)
        out["d_h"], out["d_w"] = (gx @ w).to(s["h"].dtype), (gx.T @ h).to(s["w"].dtype)
    return out


_own = {"embed": _own_embed, "logprobs": _own_logprobs, "linear": _own_linear}
_plain = {"embed": _plain_embed, "logprobs": _plain_logprobs, "linear": _plain_linear}


# ---------------------------------------------------------------- work and definition

def work(case):
    """Bytes: each input read once, each output written once (of the tables, the
    rows of the distinct tokens).  Flops: the products, a training pass three of them."""
    c, e, n, V = case, BYTES[case["dtype"]], case["n"], case["V"]
    if c["kind"] == "embed":
        norm = sum(1.0 / (r + 2.7) for r in range(V))
        rows = sum(-math.expm1(n * math.log1p(-1.0 / (r + 2.7) / norm)) for r in range(V))   # distinct tokens expected
        row = 2 * c["dim"] * e
        return {"bytes": 8 * n + (rows + n) * row + ((n + V) * row + 8 * n if c["grad"] else 0),
                "flops": 2 * n * c["dim"] * (2 if c["grad"] else 1)}
    small = 16 * n + (8 * n if c["grad"] else 0)
    if c["kind"] == "logprobs":
        return {"bytes": n * V * e * (3 if c["grad"] else 1) + small + 12 * n * c["k"], "flops": n * V * (12 if c["grad"] else 5)}
    operands = (n + V) * c["D"] * e
    return {"bytes": operands * (2 if c["grad"] else 1) + small, "flops": 2 * n * V * c["D"] * (3 if c["grad"] else 1)}


def _exact_rows(c, s, x):
    """Outputs and d x of fp64 rows x (logits over the temperature)."""
    m = x.max(-1, keepdim=True).values
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    lse = m + z.log()
    p = e / z
    valid = s["ids"] != IGNORE
    onehot = torch.zeros_like(x)
    onehot[valid.nonzero()[:, 0], s["ids"][valid]] = 1.0
    finite = torch.where(x > -math.inf, x, torch.zeros((), device=x.device, dtype=x.dtype))
    surprise = torch.where(x > -math.inf, lse - finite, torch.zeros((), device=x.device, dtype=x.dtype))   # -log p
    ent = (p * surprise).sum(-1)
    lp = torch.where(valid, x.gather(1, torch.where(valid, s["ids"], 0)[:, None])[:, 0] - lse[:, 0], 0.0)
    gx = None
    if c["grad"]:
        g_lp = torch.where(valid, s["g_lp"].double(), 0.0)[:, None]
        gx = (g_lp * (onehot - p) + s["g_ent"].double()[:, None] * p * (surprise - ent[:, None])) / c["temperature"]
    return lp, ent, lse, gx


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "embed":
        re, im = (s[k].detach().double().mul(s["scale"]).index_select(0, s["ids"]) for k in ("re", "im"))
        out = {"z": torch.stack((re, im), -1)}
        if c["grad"]:
            order = s["ids"].argsort(stable=True)
            tokens, counts = s["ids"][order].unique_consecutive(return_counts=True)
            total = s["dz"].double()[order].mul(s["scale"]).cumsum(0)
            ends = counts.cumsum(0) - 1
            sums = total[ends].diff(dim=0, prepend=torch.zeros_like(total[:1]))
            for i, k in ((0, "d_re"), (1, "d_im")):
                out[k] = torch.zeros(c["V"], c["dim"], device=DEV, dtype=torch.float64)
                out[k][tokens] = sums[..., i]
        return out
    if c["kind"] == "logprobs":
        x = s["logits"].detach().double() / c["temperature"]
        lp, ent, lse, gx = _exact_rows(c, s, x)
        out = {"logprobs": lp, "entropy": ent}
        if c["k"]:
            out["top_ids"] = None
            out["top_logprobs"] = x.topk(c["k"], -1).values - lse
        if c["grad"]:
            out["d_logits"] = gx
        return out
    h, w = s["h"].detach().double(), s["w"].detach().double()
    lp, ent, _, gx = _exact_rows(c, s, h @ w.T / c["temperature"])
    out = {"logprobs": lp, "entropy": ent}
    if c["grad"]:
        out["d_h"], out["d_w"] = gx @ w, gx.T @ h
    return out
