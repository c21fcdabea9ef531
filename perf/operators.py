"""The operators on a model's vocabulary, as cases that can be timed and compared: the embedding with its scale and its gradient
by sorted tokens, the distillation loss against a teacher's top logits with its gradient, and the sampling of tokens from given
random numbers.  Shapes are those of the repository's configurations (vocabularies of 32000 and 128256 tokens, widths of 2048 and
4096, sequences of 2048 and 8192 tokens) and generic ones with odd sizes; `draw` gives further cases of the same ranges.

Plain forms are elementary torch operations in 32 bits (sampling in 64: a token is right or wrong, and cumulated masses lie next to
their borders).  `exact` states every operator at 64 bits on its own.
"""
import math

import numpy as np
import torch

own = False                                                  # True: the framework's operators; False: the plain forms

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one short sequence through a small model: launches are all there is
        {"name": "embed-short", "kind": "embed", "tokens": 128, "vocab": 8192, "dim": 512, "type": "bf16", "scale": 1.0, "pad": False},
        # a sequence of the 1.1B configuration
        {"name": "embed-1.1b", "kind": "embed", "tokens": 2048, "vocab": 32000, "dim": 2048, "type": "bf16", "scale": 1.0, "pad": False},
        # a sequence of the headline shape; the scale that some families put on their embeddings, sqrt(width)
        {"name": "embed-8b", "kind": "embed", "tokens": 8192, "vocab": 128256, "dim": 4096, "type": "bf16", "scale": 64.0, "pad": False},
        # 32-bit training on a padded batch with odd sizes
        {"name": "embed-padded-fp32", "kind": "embed", "tokens": 40001, "vocab": 50257, "dim": 1027, "type": "fp32", "scale": 32.0, "pad": True},
        # a few positions with a small vocabulary: latency
        {"name": "distill-few", "kind": "distill", "rows": 32, "vocab": 32000, "top": 16, "type": "bf16", "temperature": 1.0, "ragged": False, "reduction": "mean"},
        # a micro-batch of the headline vocabulary, softened
        {"name": "distill-8b", "kind": "distill", "rows": 4096, "vocab": 128256, "top": 64, "type": "bf16", "temperature": 2.0, "ragged": False, "reduction": "mean"},
        # odd vocabulary, teacher entries of unequal number (some rows have none), a weight for every row
        {"name": "distill-ragged-fp32", "kind": "distill", "rows": 1000, "vocab": 50257, "top": 20, "type": "fp32", "temperature": 1.0, "ragged": True, "reduction": "none"},
        # many entries a row, 16-bit floats
        {"name": "distill-fp16", "kind": "distill", "rows": 2048, "vocab": 32000, "top": 128, "type": "fp16", "temperature": 1.5, "ragged": False, "reduction": "sum"},
        # interactive use: one sequence, nucleus
        {"name": "sample-one", "kind": "sample", "rows": 1, "vocab": 32000, "type": "bf16", "peaked": True, "filters": "p"},
        # a loaded server, every request with its own parameters
        {"name": "sample-server", "kind": "sample", "rows": 64, "vocab": 128256, "type": "fp32", "peaked": True, "filters": "mixed"},
        # answers for on-policy training from an odd vocabulary: top-k with min-p
        {"name": "sample-odd", "kind": "sample", "rows": 256, "vocab": 50257, "type": "bf16", "peaked": True, "filters": "k+min"},
        # the same from the whole distribution, which is flat
        {"name": "sample-whole", "kind": "sample", "rows": 512, "vocab": 128256, "type": "bf16", "peaked": False, "filters": "none"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _bytes(case):
    return work(case)["bytes"]


def draw(rng):
    kind = rng.choice(["embed", "distill", "sample"])
    limit = max(_bytes(c) for c in listed() if c["kind"] == kind)
    while True:
        if kind == "embed":
            case = {"kind": kind, "tokens": _log(rng, 1, 65536), "vocab": _log(rng, 500, 128256), "dim": _log(rng, 60, 4096), "type": rng.choice(list(TYPES)),
                    "scale": rng.choice([1.0, 22.627417, 0.125]), "pad": rng.random() < 0.4}
            if rng.random() < 0.5:
                case["dim"] = (case["dim"] + 63) // 64 * 64
        elif kind == "distill":
            case = {"kind": kind, "rows": _log(rng, 1, 8192), "vocab": _log(rng, 300, 128256), "top": _log(rng, 1, 256), "type": rng.choice(list(TYPES)),
                    "temperature": rng.choice([1.0, 0.8, 2.0, 3.5]), "ragged": rng.random() < 0.4, "reduction": rng.choice(["mean", "sum", "none"])}
            if rng.random() < 0.5:
                case["vocab"] = (case["vocab"] + 7) // 8 * 8
        else:
            case = {"kind": kind, "rows": _log(rng, 1, 512), "vocab": _log(rng, 300, 262144), "type": rng.choice(list(TYPES)), "peaked": rng.random() < 0.7,
                    "filters": rng.choice(["none", "p", "k", "min", "k+min", "k+p", "mixed"])}
            if rng.random() < 0.5:
                case["vocab"] = (case["vocab"] + 7) // 8 * 8
        if _bytes(case) <= limit and (kind != "distill" or case["top"] <= case["vocab"] // 4):
            return case


# ------------------------------------------------------------------------------------------------ inputs
def _frequencies(vocab):
    """How often the tokens of a text come: about inversely to their rank."""
    p = 1.0 / (np.arange(vocab, dtype=np.float64) + 10.0)
    return p / p.sum()


def _logits(rows, vocab, dtype, peaked, g):
    """(logits, contenders [rows, 24]): a bell of all tokens and, where peaked, some that stand out of it."""
    z = torch.randn(rows, vocab, device=DEV, generator=g, dtype=torch.float32).mul_(2.0)
    first = torch.randint(0, vocab, (rows, 1), device=DEV, generator=g)
    at = (first + torch.randint(1, vocab // 24, (rows, 1), device=DEV, generator=g) * torch.arange(24, device=DEV)) % vocab       # all different
    if peaked:
        z.scatter_(1, at, 12.0 + 3.0 * torch.randn(rows, 24, device=DEV, generator=g))
    return z.to(dtype), at


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = TYPES[case["type"]]
    if case["kind"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        cdf = torch.from_numpy(np.cumsum(_frequencies(v))).to(DEV)
        idx = torch.searchsorted(cdf, torch.rand(n, device=DEV, dtype=torch.float64, generator=g)).clamp_(max=v - 1)
        pad = None
        if case["pad"]:                                      # sequences that end early, filled up with the last token
            pad = v - 1
            idx[torch.rand(n, device=DEV, generator=g) < 0.3] = pad
        table = torch.randn(v, d, device=DEV, generator=g).to(dtype).requires_grad_()
        dout = torch.randn(n, d, device=DEV, generator=g).mul_(0.01).to(dtype)
        return {"case": case, "idx": idx, "table": table, "dout": dout, "pad": pad}
    if case["kind"] == "distill":
        n, v, k = case["rows"], case["vocab"], case["top"]
        z, at = _logits(n, v, dtype, True, g)
        first = torch.randint(0, v, (n, 1), device=DEV, generator=g)
        step = torch.randint(1, max(2, v // k), (n, 1), device=DEV, generator=g)
        idx = (first + step * torch.arange(k, device=DEV)) % v           # k different tokens,
        m = min(k, 12)
        idx[:, :m] = at[:, :m]                                           # the first of them where the student has its own
        t = (10.0 + 3.0 * torch.randn(n, k, device=DEV, generator=g)).sort(1, descending=True).values.to(dtype)
        if case["ragged"]:
            have = torch.randint(0, k + 1, (n, 1), device=DEV, generator=g)
            idx[torch.arange(k, device=DEV) >= have] = -1
        up = torch.rand(n, device=DEV, generator=g) if case["reduction"] == "none" else None
        return {"case": case, "z": z.requires_grad_(), "t": t, "idx": idx, "up": up}
    n, v, kind = case["rows"], case["vocab"], case["filters"]
    z, _ = _logits(n, v, dtype, case["peaked"], g)
    state = {"case": case, "z": z, "u": torch.rand(n, device=DEV, generator=g), "tau": 1.0, "k": 0, "p": 1.0, "min": 0.0}
    if kind == "mixed":                                                  # parameters of the requests, on the device
        state["tau"] = 0.5 + torch.rand(n, device=DEV, generator=g)
        state["k"] = torch.randint(0, 100, (n,), device=DEV, generator=g, dtype=torch.int32) * (torch.rand(n, device=DEV, generator=g) < 0.5)
        state["p"] = torch.where(torch.rand(n, device=DEV, generator=g) < 0.7, 0.7 + 0.3 * torch.rand(n, device=DEV, generator=g), torch.ones(n, device=DEV))
        state["min"] = torch.where(torch.rand(n, device=DEV, generator=g) < 0.3, torch.full((n,), 0.02, device=DEV), torch.zeros(n, device=DEV))
    else:
        state["tau"] = 0.75 if kind != "none" else 1.0
        if "k" in kind:
            state["k"] = 50
        if "p" in kind.split("+"):
            state["p"] = 0.9
        if "min" in kind:
            state["min"] = 0.05
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from litetorch_b200.ops import functional as Fn
    case = s["case"]
    if case["kind"] == "embed":
        out = Fn.token_embedding(s["idx"], s["table"], scale=case["scale"], padding_idx=s["pad"])
        grad, = torch.autograd.grad(out, s["table"], s["dout"])
        return {"rows": out.detach(), "grad": grad}
    if case["kind"] == "distill":
        loss = Fn.distillation_loss(s["z"], s["t"], s["idx"], temperature=case["temperature"], reduction=case["reduction"])
        grad, = torch.autograd.grad(loss, s["z"], s["up"])
        return {"loss": loss.detach(), "grad": grad}
    tokens, logprobs = Fn.sample_tokens(s["z"], s["u"], temperature=s["tau"], top_k=s["k"], top_p=s["p"], min_p=s["min"])
    return {"tokens": tokens, "logprobs": logprobs}


def _run_plain(s):
    return {"embed": _plain_embed, "distill": _plain_distill, "sample": _plain_sample}[s["case"]["kind"]](s)


@torch.no_grad()
def _plain_embed(s):
    case, idx, table, dout = s["case"], s["idx"], s["table"], s["dout"]
    out = (table[idx].float() * case["scale"]).to(table.dtype)
    rows = dout.float()
    if s["pad"] is not None:
        rows = rows * (idx != s["pad"])[:, None]
    grad = torch.zeros(table.shape, dtype=torch.float32, device=DEV).index_add_(0, idx, rows)
    return {"rows": out, "grad": grad.mul_(case["scale"]).to(table.dtype)}


@torch.no_grad()
def _plain_distill(s):
    case, z, t, idx = s["case"], s["z"], s["t"].float(), s["idx"]
    tau, inf = case["temperature"], float("-inf")
    here = idx >= 0
    safe = idx.clamp(min=0)
    rows = here.any(1)
    a = (t / tau).masked_fill(~here, inf)
    top = a.amax(1, keepdim=True).masked_fill(~rows[:, None], 0.0)
    ea = torch.exp(a - top)
    mass = ea.sum(1, keepdim=True).masked_fill(~rows[:, None], 1.0)
    p = ea / mass
    logp = (a - top - torch.log(mass)).masked_fill(~here, 0.0)
    y = z.float() / tau
    big = y.amax(1, keepdim=True)
    y -= big
    picked = y.gather(1, safe)
    e = y.exp_()
    total = e.sum(1, keepdim=True)
    loss = tau * tau * (p * (logp - (picked - torch.log(total)))).sum(1)
    weight = rows.float()
    if case["reduction"] == "mean":
        weight = weight / rows.sum().clamp(min=1)
    grad = e.div_(total).scatter_add_(1, safe, -p)
    if s["up"] is not None:
        weight = weight * s["up"]
    grad = grad.mul_((weight * tau)[:, None]).to(z.dtype)
    if case["reduction"] == "mean":
        loss = loss.sum() / rows.sum().clamp(min=1)
    elif case["reduction"] == "sum":
        loss = loss.sum()
    return {"loss": loss, "grad": grad}


def _column(v, n):
    return v.double()[:, None] if torch.is_tensor(v) else torch.full((n, 1), float(v), dtype=torch.float64, device=DEV)


@torch.no_grad()
def _plain_sample(s):
    z = s["z"]
    n, v = z.shape
    y = z.double() / _column(s["tau"], n)
    e = torch.exp(y - y.amax(1, keepdim=True))
    keep = torch.ones_like(e, dtype=torch.bool)
    if s["case"]["filters"] not in ("none", "min"):
        order = torch.sort(z, dim=1, descending=True, stable=True).indices
        k = _column(s["k"], n)
        place = torch.arange(v, device=DEV)
        first = (place < k) | (k <= 0)
        ranked = e.gather(1, order) * first
        before = ranked.cumsum(1) - ranked
        p = _column(s["p"], n)
        first &= (before < p * ranked.sum(1, keepdim=True)) | (p >= 1.0)
        keep.scatter_(1, order, first)
    keep &= e >= _column(s["min"], n)
    e = e * keep
    cum = e.cumsum(1)
    total = cum[:, -1:]
    tokens = (cum <= s["u"].double()[:, None] * total).sum(1)
    logprobs = torch.log(e.gather(1, tokens[:, None]) / total)[:, 0]
    return {"tokens": tokens, "logprobs": logprobs.float()}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b = SIZE[case["type"]]
    if case["kind"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        p = _frequencies(v) * (0.7 if case["pad"] else 1.0)
        rows = float(-np.expm1(n * np.log1p(-p)).sum()) + (1 if case["pad"] else 0)      # different tokens among n: table rows that are read
        live = n * (0.7 if case["pad"] else 1.0)                                         # rows that bear a gradient
        return {"bytes": int(8 * n + (rows + n + live + v) * d * b), "flops": int((n + live) * d)}
    if case["kind"] == "distill":
        n, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": 2 * n * v * b + n * k * (8 + b) + 4 * n, "flops": 6 * n * v}
    n, v = case["rows"], case["vocab"]
    return {"bytes": n * v * b + 16 * n, "flops": 3 * n * v}


# ------------------------------------------------------------------------------------------------ the definitions at 64 bits
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "embed":
        idx, w, dy = s["idx"], s["table"].double(), s["dout"].double()
        out = w.index_select(0, idx) * case["scale"]
        del w
        live = torch.ones_like(idx, dtype=torch.bool) if s["pad"] is None else idx != s["pad"]
        grad = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device=DEV)
        grad.index_put_((idx[live],), dy[live] * case["scale"], accumulate=True)
        return {"rows": out, "grad": grad}
    if case["kind"] == "distill":
        n, v, tau = case["rows"], case["vocab"], case["temperature"]
        loss = torch.zeros(n, dtype=torch.float64, device=DEV)
        grad = torch.zeros(n, v, dtype=torch.float64, device=DEV)
        there = s["idx"] >= 0
        has = there.any(1)
        share = 1.0 / max(int(has.sum()), 1) if case["reduction"] == "mean" else 1.0
        for r in range(0, n, 512):
            z, t, i, ok = (x[r:r + 512] for x in (s["z"], s["t"], s["idx"], there))
            log_q = torch.log_softmax(z.double() / tau, 1)
            log_p = torch.log_softmax(torch.where(ok, t.double() / tau, torch.tensor(-1e300, dtype=torch.float64, device=DEV)), 1)
            p = torch.where(ok, log_p.exp(), torch.zeros_like(log_p))
            j = torch.where(ok, i, torch.zeros_like(i))
            loss[r:r + 512] = tau ** 2 * (p * torch.where(ok, log_p - log_q.gather(1, j), torch.zeros_like(p))).sum(1)
            target = torch.zeros_like(log_q).scatter_add_(1, j, p)
            scale = has[r:r + 512].double() * tau * share
            if s["up"] is not None:
                scale = scale * s["up"][r:r + 512].double()
            grad[r:r + 512] = (log_q.exp() - target) * scale[:, None]
        if case["reduction"] != "none":
            loss = loss.sum() * share
        return {"loss": loss, "grad": grad}
    n, v = case["rows"], case["vocab"]
    z = s["z"].double().cpu().numpy()
    u = s["u"].double().cpu().numpy()

    def row(name, kind):
        x = s[name]
        return (x.double().cpu().numpy() if torch.is_tensor(x) else np.full(n, float(x))).astype(kind)
    tau, k, p, low = row("tau", np.float64), row("k", np.int64), row("p", np.float64), row("min", np.float64)
    tokens, logprobs = np.zeros(n, np.int64), np.zeros(n)
    for r in range(n):
        e = np.exp((z[r] - z[r].max()) / tau[r])
        chosen = np.arange(v)
        if k[r] > 0 or p[r] < 1.0:
            chosen = np.argsort(-z[r], kind="stable")
            if k[r] > 0:
                chosen = chosen[:k[r]]
            if p[r] < 1.0:
                c = np.concatenate([[0.0], np.cumsum(e[chosen])])
                chosen = chosen[c[:-1] < p[r] * c[-1]]
        chosen = np.sort(chosen[e[chosen] >= low[r]])
        c = np.cumsum(e[chosen])
        at = int(np.searchsorted(c, u[r] * c[-1], side="right"))
        tokens[r], logprobs[r] = chosen[at], math.log(e[chosen[at]] / c[-1])
    return {"tokens": torch.from_numpy(tokens).to(DEV), "logprobs": torch.from_numpy(logprobs).to(DEV)}
