"""Serving a model with 4-bit weights and many sequences, one pass each, for timing
and for comparing outputs: the products of a few rows (or a prompt's) with weights of
4 bits and group scales, real ones (the logits of the tied table) and those of a
ComplexLinear, and the pages of the decode's state pool copied (one sequence forked
into many, beams that continue from each other's states, a pool compacted).

`listed()` names the cases, `draw(rng)` gives others of the same ranges.  With
`own` false a pass is computed in plain torch operations in 32 bits; with `own`
true it is the framework's call.  `exact` computes a case from the definitions
in 64 bits.

A 4-bit code is a sign and a magnitude of 0, 0.5, 1, 1.5, 2, 3, 4 or 6 (the E2M1
format); `group` neighbouring codes of an output's row share a bf16 scale.  A complex
weight is two neighbouring codes, its real and its imaginary part.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "bf16": 2}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MOST_PRODUCTS = 2 * 2000 * 4608 * 1536  # real multiply-adds of the largest product
MOST_POOL = 128 * 16 * 12 * 3 * 8192    # fp32 values of the largest state pool


def listed():
    return [
        # one sequence's token: the output projection of a PAM layer, where latency is all
        dict(name="one_out_bf16", kind="complex", n=1, K=768, N=768, group=32, dtype="bf16", bias=False, planes=False, tail=0),
        # one sequence's token: the gate and up projections of a block's channel mix
        dict(name="one_gate_up_fp32", kind="complex", n=1, K=768, N=4608, group=64, dtype="fp32", bias=False, planes=False,
             tail=0),
        # a decode step of 16 live sequences: the channel mix's down projection, a bias on it
        dict(name="step_down_fp32", kind="complex", n=16, K=2304, N=768, group=128, dtype="fp32", bias=True, planes=False,
             tail=0),
        # a decode step of 192: q, k, v of a PAM layer as planes, the decay logits from weights kept whole
        dict(name="step_in_bf16", kind="complex", n=192, K=768, N=2304, group=32, dtype="bf16", bias=False, planes=True,
             tail=12),
        # odd sizes in every place
        dict(name="ragged_fp32", kind="complex", n=37, K=515, N=771, group=32, dtype="fp32", bias=True, planes=False, tail=0),
        # a prompt's rows through the gate and up projections
        dict(name="prompt_gate_up_bf16", kind="complex", n=2000, K=768, N=4608, group=32, dtype="bf16", bias=False,
             planes=False, tail=0),
        # the logits of one token and of a step from a table in 4 bits
        dict(name="logits_one_bf16", kind="real", n=1, K=1536, N=50261, group=32, dtype="bf16", bias=False),
        dict(name="logits_step_bf16", kind="real", n=192, K=1536, N=50261, group=64, dtype="bf16", bias=False),
        # one sequence forked into four in a small model's pool: latency
        dict(name="fork_small", kind="pages", how="fork", slots=64, count=4, layers=2, heads=4, states=1, d=32, lists="host"),
        # 15 samples more of one prompt, 16 layers of three states
        dict(name="fork_samples", kind="pages", how="fork", slots=32, count=15, layers=16, heads=12, states=3, d=64,
             lists="host"),
        # 16 searches of 8 beams each, in place, the parents chosen on the device
        dict(name="beams", kind="pages", how="beams", slots=160, count=128, layers=16, heads=12, states=1, d=64,
             lists="device"),
        # a half empty pool's sequences moved to its front, the places they leave cleared
        dict(name="compact", kind="pages", how="compact", slots=128, count=64, layers=16, heads=12, states=3, d=64,
             lists="host"),
    ]


def _span(rng, lo, hi):
    """An integer of [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["complex", "complex", "real", "pages"])
    if kind == "pages":
        c = dict(kind=kind, how=rng.choice(["fork", "beams", "compact"]), slots=_span(rng, 8, 300), count=0,
                 layers=_span(rng, 1, 24), heads=_span(rng, 1, 12), states=rng.choice([1, 2, 3, 4]),
                 d=rng.choice([16, 32, 64, 128]), lists=rng.choice(["host", "device"]))
        c["slots"] = max(8, min(c["slots"], MOST_POOL // (c["layers"] * c["heads"] * c["states"] * 2 * c["d"] ** 2)))
        c["count"] = _span(rng, 1, c["slots"] // 2)
        return c
    c = dict(kind=kind, n=_span(rng, 1, 2000), K=_span(rng, 48, 2600), N=_span(rng, 48, 5000 if kind == "complex" else 60000),
             group=rng.choice([32, 64, 128]), dtype=rng.choice(["fp32", "bf16"]), bias=rng.random() < 0.3)
    if kind == "complex":
        c["planes"] = rng.random() < 0.4
        c["tail"] = rng.choice([0, _span(rng, 1, 24)]) if c["planes"] else 0
    each = c["K"] * c["N"] * (4 if kind == "complex" else 1)
    c["n"] = max(1, min(c["n"], MOST_PRODUCTS // (each * (6 if c["dtype"] == "fp32" else 1))))
    return c


# ---------------------------------------------------------------- inputs

def _randn(g, *shape, std=1.0):
    return torch.empty(*shape, device=DEV, dtype=torch.float32).normal_(0.0, std, generator=g)


def _quantized(w, group):
    """Codes [N, ceil(K / 2)] (the even column in the low half of a byte) and scales [N, ceil(K / group)] of w [N, K]."""
    N, K = w.shape
    groups = -(-K // group)
    w = torch.cat([w, w.new_zeros(N, groups * group - K)], 1).view(N, groups, group)
    scales = (w.abs().amax(-1) / 6).to(torch.bfloat16)
    r = w / scales.float().clamp_min(1e-30)[..., None]
    borders = torch.tensor([(a + b) / 2 for a, b in zip(MAGNITUDES, MAGNITUDES[1:])], device=DEV)
    codes = torch.bucketize(r.abs(), borders).to(torch.uint8) | (r < 0).to(torch.uint8) << 3
    codes = codes.view(N, -1)[:, :K + K % 2]
    if K % 2:
        codes[:, K] = 0
    return (codes[:, 0::2] | codes[:, 1::2] << 4).contiguous(), scales


def _moves(c, g):
    """Host lists (src, dst) of a page case: state[dst[i]] = state[src[i]], a src of -1 clears."""
    S, n = c["slots"], c["count"]
    order = torch.randperm(S, generator=g, device=DEV)
    if c["how"] == "fork":       # one sequence into n free slots
        return [int(order[0])] * n, order[1:n + 1].tolist()
    if c["how"] == "beams":      # groups of 8 slots, each continues from one of its group
        live = order[:n]
        at = torch.arange(n, device=DEV)
        first = at // 8 * 8
        size = (n - first).clamp_max(8)
        pick = first + (torch.rand(n, device=DEV, generator=g) ** 2 * size).long().clamp_max(size - 1)   # the better beams more often
        return live[pick].tolist(), live.tolist()
    live = order[:n].sort().values   # compact: live slots at n and above go to the free ones below, and are cleared
    out = live[live >= n]
    free = torch.ones(n, dtype=torch.bool, device=DEV)
    free[live[live < n]] = False
    into = free.nonzero()[:, 0]
    return out.tolist() + [-1] * out.numel(), into.tolist() + out.tolist()


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV).manual_seed(int(seed))
    s = dict(case=c)
    if c["kind"] == "pages":
        s["state"] = _randn(g, c["slots"], c["layers"], c["heads"], c["states"], c["d"], c["d"], 2, std=0.1)
        s["pos"] = torch.randint(1, 4000, (c["slots"],), device=DEV, generator=g, dtype=torch.int32)
        s["src"], s["dst"] = _moves(c, g)
        s["on_device"] = [torch.tensor(s[k], device=DEV, dtype=torch.int32) for k in ("src", "dst")]
        return s
    dt, z = DTYPES[c["dtype"]], 2 if c["kind"] == "complex" else 1
    K, N = c["K"] * z, c["N"]
    s["codes"], s["scales"] = _quantized(_randn(g, N, K, std=1.0 / math.sqrt(K)), c["group"])
    x = _randn(g, c["n"], K) * (1.0 + 9.0 * (torch.rand(K, device=DEV, generator=g) < 0.01))   # normed rows, a few loud channels
    s["x"] = (x.view(c["n"], c["K"], 2) if z == 2 else x).to(dt)
    s["bias"] = _randn(g, *((N, 2) if z == 2 else (N,)), std=0.1) if c["bias"] else None
    s["tail"] = _randn(g, c["tail"], K, std=1.0 / math.sqrt(K)).to(dt) if c.get("tail") else None
    if own:  # a program lays its weights out once, when it loads them
        from qllm2_amd.linear4 import Weight4
        s["weight"] = Weight4(s["codes"], s["scales"], c["K"], c["group"], complex=z == 2)
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    return (_own if own else _plain)[state["case"]["kind"]](state)


def _own_real(s):
    from qllm2_amd.linear4 import linear4
    return linear4(s["x"], s["weight"], s["bias"])


def _own_complex(s):
    from qllm2_amd.linear4 import complex_linear4
    return complex_linear4(s["x"], s["weight"], s["bias"], planes=s["case"]["planes"], tail=s["tail"])


def _own_pages(s):
    from qllm2_amd.decode import copy_slots
    src, dst = s["on_device"] if s["case"]["lists"] == "device" else (s["src"], s["dst"])
    copy_slots(s["state"], src, dst, pos=s["pos"])
    return {"state": s["state"], "pos": s["pos"]}


def _weight(s, K):
    """The fp32 weight [N, K] that the codes and scales stand for."""
    values = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=DEV)
    codes = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).flatten(1)[:, :K]
    return values[codes.int()] * s["scales"].float().repeat_interleave(s["case"]["group"], 1)[:, :K]


def _plain_real(s):
    y = s["x"].float() @ _weight(s, s["case"]["K"]).T
    return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)


def _plain_complex(s):
    c, x = s["case"], s["x"].float()
    w = _weight(s, 2 * c["K"])
    wr, wi, xr, xi = w[:, 0::2], w[:, 1::2], x[..., 0], x[..., 1]
    y = torch.stack((xr @ wr.T - xi @ wi.T, xr @ wi.T + xi @ wr.T), -1)
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["planes"]:
        parts = [y[..., 0], y[..., 1]]
        if s["tail"] is not None:
            parts.append(x.flatten(1) @ s["tail"].float().T)
        y = torch.cat(parts, 1)
    return y.to(s["x"].dtype)


def _plain_pages(s):
    src, dst = (t.long() for t in s["on_device"])
    clear = src < 0
    for t in (s["state"], s["pos"]):
        rows = t[src.clamp_min(0)]
        t[dst] = rows.masked_fill_(clear.view(-1, *[1] * (t.dim() - 1)), 0)
    return {"state": s["state"], "pos": s["pos"]}


_own = {"real": _own_real, "complex": _own_complex, "pages": _own_pages}
_plain = {"real": _plain_real, "complex": _plain_complex, "pages": _plain_pages}


# ---------------------------------------------------------------- work and definition

def work(case):
    """Bytes: each input read once, each output written once (of a pool, the distinct
    pages that are copied elsewhere, those they replace, and the lists).  Flops: the products."""
    c = case
    if c["kind"] == "pages":
        page, n = c["layers"] * c["heads"] * c["states"] * 2 * c["d"] ** 2 * 4 + 4, c["count"]
        if c["how"] == "fork":
            pages = 1 + n
        elif c["how"] == "beams":    # the k-th of g is picked with probability sqrt((k + 1) / g) - sqrt(k / g)
            pages = 0.0
            for size in [8] * (n // 8) + ([n % 8] if n % 8 else []):
                p = [math.sqrt((k + 1) / size) - math.sqrt(k / size) for k in range(size)]
                moved = size - sum(p)
                pages += moved + sum(1 - (1 - q) ** (size - 1) for q in p)
        else:                        # read, written and cleared: the live ones outside the front
            pages = 3 * n * (c["slots"] - n) / c["slots"]
        return {"bytes": max(1.0, pages * page + 8 * n), "flops": 0}
    z, e = 2 if c["kind"] == "complex" else 1, BYTES[c["dtype"]]
    K, N, n, tail = c["K"] * z, c["N"], c["n"], c.get("tail", 0)
    size = N * -(-K // 2) + 2 * N * -(-K // c["group"]) + n * (K + N * z + tail) * e + tail * K * e + (4 * N * z if c["bias"] else 0)
    return {"bytes": size, "flops": 2 * n * K * (N * z + tail)}


def _exact_weight(codes, scales, K, group):
    """In 64 bits from the format: sign, 2 bits of exponent, 1 of mantissa (subnormal at exponent 0)."""
    N = codes.shape[0]
    w = torch.empty(N, 2 * codes.shape[1], device=DEV, dtype=torch.float64)
    for half in (0, 1):
        q = (codes >> (4 * half)).to(torch.int64) & 15
        e, m = (q >> 1) & 3, (q & 1).double()
        size = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2((e - 1).double()))
        w[:, half::2] = torch.where(q >= 8, -size, size)
    at = torch.arange(K, device=DEV) // group
    return w[:, :K] * scales.double()[:, at]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "pages":
        out = {"state": s["state"].clone(), "pos": s["pos"].clone()}
        for src, dst in zip(s["src"], s["dst"]):
            for k in out:
                out[k][dst] = 0 if src < 0 else s[k][src]
        return out
    z = 2 if c["kind"] == "complex" else 1
    w = _exact_weight(s["codes"], s["scales"], z * c["K"], c["group"])
    x = s["x"].double().flatten(1)
    if z == 1:
        y = torch.mm(x, w.t().contiguous())
        return y if s["bias"] is None else y + s["bias"].double()
    # the real matrix of the complex one: rows (wr, -wi) give the real parts, (wi, wr) the imaginary
    pairs = w.view(c["N"], c["K"], 2)
    to_re = torch.stack((pairs[..., 0], -pairs[..., 1]), -1).flatten(1)
    to_im = pairs.flip(-1).flatten(1)
    re, im = torch.mm(x, to_re.t().contiguous()), torch.mm(x, to_im.t().contiguous())
    if s["bias"] is not None:
        re, im = re + s["bias"][:, 0].double(), im + s["bias"][:, 1].double()
    if not c["planes"]:
        return torch.stack((re, im), -1)
    parts = [re, im]
    if s["tail"] is not None:
        parts.append(torch.mm(x, s["tail"].double().t().contiguous()))
    return torch.cat(parts, 1)
