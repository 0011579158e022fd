"""The scoring operators as measured cases: log probabilities of given tokens from logits, log probabilities
straight from a language-model head, and the projection with a fused epilogue.

``run`` computes the plain form (elementary torch operations in 32 bits, rounded once at the end) or, with ``own``
set, makes the calls a user of the framework makes.  Formulas, with z = x / T (T the temperature):

* logprob = z_t - lse, lse = log sum_i exp z_i; entropy H = -sum_i p_i log p_i, p = exp(z - lse); rank = how many ids
  come before t in descending order of value, equal values in ascending order of id; top: the first K ids of that
  order with their log probabilities.  A token below 0 is no token: logprob 0, rank -1, no gradient through logprob.
* gradient: dx_i = (g_logprob ([i = t] - p_i) - g_entropy p_i (log p_i + H)) / T.
* head: x = hidden head^T; d hidden = dx head, d head = dx^T hidden.
* linear: y = act(x w^T + b) + r; dz = dy act'(z), db = sum dz, dx = dz w, dw = dz^T x, dr = dy.
"""

from __future__ import annotations

import math

import torch

own = False

V_THINKER, H_THINKER = 151_936, 4096  # the Thinker's vocabulary and hidden size
V_TALKER, H_TALKER = 6562, 768        # the Talker's codec vocabulary and hidden size
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}


def listed():
    return [
        # one Talker row scored as it is sampled: the smallest call, latency counts
        dict(name="logits_row", op="logits", rows=1, vocab=V_TALKER, dtype="f32", top=0, pad=0, masked=0.0, grad=False,
             temperature=0.8),
        # a Thinker decode step that returns 20 alternatives beside the sampled tokens
        dict(name="logits_step_top20", op="logits", rows=64, vocab=V_THINKER, dtype="bf16", top=20, pad=0, masked=0.0,
             grad=False, temperature=0.7),
        # processed logits (most ids masked) of a padded codec batch, an odd vocabulary, rows inside a wider buffer
        dict(name="logits_masked_odd", op="logits", rows=384, vocab=V_TALKER - 1, dtype="f32", top=8, pad=5, masked=0.98,
             grad=False, temperature=1.0),
        # scoring a large batch of fp32 rows
        dict(name="logits_large", op="logits", rows=1024, vocab=V_THINKER, dtype="f32", top=0, pad=0, masked=0.0,
             grad=False, temperature=1.0),
        # a policy-gradient step on stored logits: logprob and entropy with their gradient
        dict(name="logits_train", op="logits", rows=2048, vocab=V_THINKER, dtype="bf16", top=0, pad=0, masked=0.0,
             grad=True, temperature=1.0),
        # a Thinker decode step scored from its hidden rows: one read of the head
        dict(name="head_step", op="head", rows=16, vocab=V_THINKER, hidden=H_THINKER, grad=False, temperature=1.0),
        # scoring a prompt's positions from their hidden rows
        dict(name="head_prompt", op="head", rows=2000, vocab=V_THINKER, hidden=H_THINKER, grad=False, temperature=1.0),
        # fine-tuning the Talker's codec head on a ragged batch
        dict(name="head_codec_train", op="head", rows=777, vocab=V_TALKER, hidden=H_TALKER, grad=True, temperature=1.0),
        # fine-tuning with the Thinker's head: gradients of the hidden rows and of the whole head
        dict(name="head_train", op="head", rows=1024, vocab=V_THINKER, hidden=H_THINKER, grad=True, temperature=1.0),
        # one Thinker row projected to the Talker's width
        dict(name="linear_row", op="linear", rows=1, inputs=H_THINKER, outputs=H_TALKER, activation="silu", bias=True,
             residual=False, grad=False),
        # a prompt's rows through a square projection with everything in the epilogue
        dict(name="linear_prompt", op="linear", rows=2000, inputs=H_THINKER, outputs=H_THINKER, activation="gelu",
             bias=True, residual=True, grad=False),
        # training a projection to an odd width on a ragged batch
        dict(name="linear_train", op="linear", rows=4099, inputs=H_TALKER, outputs=2 * H_TALKER + 1, activation="silu",
             bias=True, residual=True, grad=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logits", "logits", "head", "head", "linear"])
    if op == "logits":
        vocab = _log_uniform(rng, 500, V_THINKER + 300)
        rows = _log_uniform(rng, 1, 150_000_000 // vocab)
        rows = min(rows, 20_000)
        return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["f32", "bf16"]), top=rng.choice([0, 0, 1, 5, 20, 32]),
                    pad=rng.choice([0, 0, 3, 8]), masked=rng.choice([0.0, 0.0, 0.9]), grad=rng.random() < 0.35,
                    temperature=rng.choice([0.7, 1.0, 1.0, 1.3]))
    if op == "head":
        hidden = 8 * _log_uniform(rng, 16, H_THINKER // 8)
        vocab = _log_uniform(rng, 700, V_THINKER)
        grad = rng.random() < 0.4
        most = int(min(1.2e12 / (2 * hidden * vocab * (3 if grad else 1)), 4e8 / vocab))
        return dict(op=op, rows=_log_uniform(rng, 1, max(1, min(8192, most))), vocab=vocab, hidden=hidden, grad=grad,
                    temperature=rng.choice([0.7, 1.0, 1.0]))
    inputs = 8 * _log_uniform(rng, 8, 1024)
    outputs = _log_uniform(rng, 40, 8192)
    grad = rng.random() < 0.4
    most = int(1.2e12 / (2 * inputs * outputs * (3 if grad else 1)))
    return dict(op=op, rows=_log_uniform(rng, 1, max(1, min(8192, most))), inputs=inputs, outputs=outputs,
                activation=rng.choice(["none", "relu", "gelu", "silu"]), bias=rng.random() < 0.7,
                residual=rng.random() < 0.5, grad=grad)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    n = case["rows"]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    if case["op"] == "linear":
        k, m = case["inputs"], case["outputs"]
        s = dict(x=normal(n, k).bfloat16(), weight=(normal(m, k) / math.sqrt(k)).bfloat16(),
                 bias=(normal(m) * 0.5).bfloat16() if case["bias"] else None,
                 residual=normal(n, m).bfloat16() if case["residual"] else None)
        if case["grad"]:
            s["dy"] = normal(n, m).bfloat16()
        return {"case": dict(case), **s}
    vocab = case["vocab"]
    tokens = torch.randint(0, vocab, (n,), device=dev, generator=g)
    if case["op"] == "head":
        hidden = case["hidden"]
        head = torch.empty(vocab, hidden, device=dev, dtype=torch.bfloat16)
        head.normal_(0.0, 2.0 / math.sqrt(hidden), generator=g)
        s = dict(hidden=normal(n, hidden).bfloat16(), head=head)
    else:
        buf = normal(n, vocab + case["pad"]).mul_(2.0)
        logits = buf[:, :vocab]
        if case["masked"]:
            logits.masked_fill_(torch.rand(n, vocab, device=dev, generator=g) < case["masked"], float("-inf"))
            # the tokens of processed rows were drawn from what is left; every fifth row is padding (no token), and
            # of those one in five is masked throughout
            tokens = (logits + normal(n, vocab).mul_(3.0)).argmax(-1)
            tokens[4::5] = -1
            logits[4::25] = float("-inf")
        s = dict(logits=buf.to(DTYPES[case["dtype"]])[:, :vocab])
    s["tokens"] = tokens
    if case["grad"]:
        # advantages of either sign, and the small weight of an entropy bonus
        s["g_logprob"], s["g_entropy"] = normal(n), 0.01 * torch.rand(n, device=dev, generator=g)
    return {"case": dict(case), **s}


# ------------------------------------------------------------------------------------------ the plain forms

def _activation(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _activation_slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _statistics(x, temperature):
    """z, log p, p (0 throughout a row that is masked throughout), the entropy and which rows hold something."""
    z = x / temperature
    top = z.amax(-1, keepdim=True)
    some = top > float("-inf")
    e = torch.exp(z - torch.where(some, top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    logp = z - top - torch.log(total)
    p = torch.where(some, e / total, torch.zeros_like(e))
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    return logp, p, plogp, -plogp.sum(-1), some[:, 0]


def _token_logprob(logp, tokens, some):
    lp = logp.gather(1, tokens.clamp_min(0)[:, None])[:, 0]
    lp = torch.where(some, lp, torch.full_like(lp, float("-inf")))
    return torch.where(tokens >= 0, lp, torch.zeros_like(lp))


def _logits_gradient(s, p, plogp, entropy):
    live = (s["tokens"] >= 0).to(p.dtype) * s["g_logprob"]
    dx = -p * live[:, None] - (plogp + p * entropy[:, None]) * s["g_entropy"][:, None]
    some = (p.sum(-1) > 0).to(p.dtype)
    dx.scatter_add_(1, s["tokens"].clamp_min(0)[:, None], (live * some)[:, None])
    return dx / s["case"]["temperature"]


def _plain_logits(s):
    c, t = s["case"], s["tokens"]
    x = s["logits"].float()
    logp, p, plogp, entropy, some = _statistics(x, c["temperature"])
    out = dict(logprob=_token_logprob(logp, t, some), entropy=entropy)
    at = t.clamp_min(0)[:, None]
    mine = x.gather(1, at)
    ids = torch.arange(x.shape[1], device=x.device)[None, :]
    rank = ((x > mine) | ((x == mine) & (ids < at))).sum(-1)
    out["rank"] = torch.where(t >= 0, rank, torch.full_like(rank, -1))
    if c["top"]:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
        out["top_ids"] = order
        out["top_logprobs"] = torch.where(some[:, None], logp.gather(1, order), torch.full_like(mine, float("-inf")))
    if c["grad"]:
        out["d_logits"] = _logits_gradient(s, p, plogp, entropy).to(s["logits"].dtype)
    return out


def _plain_head(s):
    c = s["case"]
    h, w = s["hidden"].float(), s["head"].float()
    logp, p, plogp, entropy, some = _statistics(h @ w.t(), c["temperature"])
    out = dict(logprob=_token_logprob(logp, s["tokens"], some), entropy=entropy)
    if c["grad"]:
        del logp
        dz = _logits_gradient(s, p, plogp, entropy)
        out["d_hidden"], out["d_head"] = (dz @ w).bfloat16(), (dz.t() @ h).bfloat16()
    return out


def _plain_linear(s):
    c = s["case"]
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if c["bias"]:
        z = z + s["bias"].float()
    y = _activation(z, c["activation"])
    if c["residual"]:
        y = y + s["residual"].float()
    out = dict(y=y.bfloat16())
    if c["grad"]:
        dz = s["dy"].float() * _activation_slope(z, c["activation"])
        out["d_x"], out["d_weight"] = (dz @ w).bfloat16(), (dz.t() @ x).bfloat16()
        if c["bias"]:
            out["d_bias"] = dz.sum(0).bfloat16()
        if c["residual"]:
            out["d_residual"] = s["dy"]
    return out


# ------------------------------------------------------------------------------------------ the framework's calls

def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _own_logits(s):
    c, lp = s["case"], _package().logprobs
    if not c["grad"]:
        r = lp.token_logprobs(s["logits"], s["tokens"], top=c["top"], temperature=c["temperature"])
        out = dict(logprob=r.logprob, entropy=r.entropy, rank=r.rank)
    else:
        x = s["logits"].detach().requires_grad_(True)
        r = lp.token_logprobs(x, s["tokens"], top=c["top"], temperature=c["temperature"])
        d, = torch.autograd.grad((r.logprob, r.entropy), (x,), (s["g_logprob"], s["g_entropy"]))
        out = dict(logprob=r.logprob.detach(), entropy=r.entropy.detach(), rank=r.rank, d_logits=d)
    if c["top"]:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
    return out


def _own_head(s):
    c, lp = s["case"], _package().logprobs
    if not c["grad"]:
        r = lp.LMHeadLogprobs(s["head"])(s["hidden"], s["tokens"], temperature=c["temperature"])
        return dict(logprob=r.logprob, entropy=r.entropy)
    h, w = s["hidden"].detach().requires_grad_(True), s["head"].detach().requires_grad_(True)
    r = lp.LMHeadLogprobs(w)(h, s["tokens"], temperature=c["temperature"])
    dh, dw = torch.autograd.grad((r.logprob, r.entropy), (h, w), (s["g_logprob"], s["g_entropy"]))
    return dict(logprob=r.logprob.detach(), entropy=r.entropy.detach(), d_hidden=dh, d_head=dw)


def _own_linear(s):
    c, linear = s["case"], _package().projection.linear
    act = None if c["activation"] == "none" else c["activation"]
    if not c["grad"]:
        return dict(y=linear(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"]))
    leaf = {k: s[k].detach().requires_grad_(True) for k in ("x", "weight", "bias", "residual") if s[k] is not None}
    y = linear(leaf["x"], leaf["weight"], leaf.get("bias"), activation=act, residual=leaf.get("residual"))
    grads = torch.autograd.grad(y, tuple(leaf.values()), s["dy"])
    return dict(y=y.detach(), **{"d_" + k: d for k, d in zip(leaf, grads)})


def run(state):
    op = state["case"]["op"]
    if own:
        return {"logits": _own_logits, "head": _own_head, "linear": _own_linear}[op](state)
    return {"logits": _plain_logits, "head": _plain_head, "linear": _plain_linear}[op](state)


def work(case):
    n = case["rows"]
    if case["op"] == "linear":
        k, m = case["inputs"], case["outputs"]
        moved = 2 * (n * k + k * m + n * m + (m if case["bias"] else 0) + (n * m if case["residual"] else 0))
        flops = 2 * n * k * m
        if case["grad"]:  # dy read; dx, dw, db and dr written
            moved += 2 * (n * m + n * k + k * m + (m if case["bias"] else 0) + (n * m if case["residual"] else 0))
            flops *= 3
        return {"bytes": moved, "flops": flops}
    v = case["vocab"]
    if case["op"] == "head":
        h = case["hidden"]
        moved, flops = 2 * (v * h + n * h) + 16 * n, 2 * n * v * h
        if case["grad"]:
            moved, flops = moved + 2 * (v * h + n * h) + 8 * n, 3 * flops
        return {"bytes": moved, "flops": flops}
    moved = n * (v * BYTES[case["dtype"]] + 24 + 12 * case["top"])
    if case["grad"]:
        moved += n * (v * BYTES[case["dtype"]] + 8)
    return {"bytes": moved, "flops": n * v * (12 if case["grad"] else 6)}


# ------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x, w = s["x"].double(), s["weight"].double()
        z = torch.einsum("nk,mk->nm", x, w)
        if s["bias"] is not None:
            z += s["bias"].double()
        kind = case["activation"]
        cdf = torch.special.ndtr(z) if kind == "gelu" else torch.sigmoid(z) if kind == "silu" else (z > 0).double()
        act = z if kind == "none" else z * cdf
        out = dict(y=act if s["residual"] is None else act + s["residual"].double())
        if case["grad"]:
            slope = {"none": lambda: torch.ones_like(z), "relu": lambda: cdf, "silu": lambda: cdf + z * cdf * (1 - cdf),
                     "gelu": lambda: cdf + z * torch.exp(-z * z / 2) * (2 * math.pi) ** -0.5}[kind]()
            dz = s["dy"].double() * slope
            out.update(d_x=torch.einsum("nm,mk->nk", dz, w), d_weight=torch.einsum("nm,nk->mk", dz, x))
            if s["bias"] is not None:
                out["d_bias"] = dz.sum(0)
            if s["residual"] is not None:
                out["d_residual"] = None
        return out
    tokens, n, v = s["tokens"], case["rows"], case["vocab"]
    grad = case["grad"]
    if case["op"] == "head":
        h, w = s["hidden"].double(), s["head"].double()
        out = dict(logprob=[], entropy=[], d_hidden=[], d_head=torch.zeros_like(w) if grad else None)
    else:
        out = dict(logprob=[], entropy=[], d_logits=[], top_logprobs=[])
    step = max(1, 60_000_000 // v)
    for a in range(0, n, step):
        rows = slice(a, min(n, a + step))
        x = (h[rows] @ w.t() if case["op"] == "head" else s["logits"][rows].double()) / case["temperature"]
        t = tokens[rows]
        lse = torch.logsumexp(x, -1)
        empty = torch.isneginf(lse)
        lp = x - torch.where(empty, torch.zeros_like(lse), lse)[:, None]
        p = torch.exp(lp)
        info = torch.special.entr(p)  # -p log p, 0 at p = 0
        out["logprob"].append(torch.where(t >= 0, lp[torch.arange(len(t), device=t.device), t.clamp_min(0)], 0.0))
        out["entropy"].append(info.sum(-1))
        if case.get("top"):
            out["top_logprobs"].append(torch.topk(lp, case["top"], dim=-1).values)
        if grad:
            gl, ge = s["g_logprob"][rows].double(), s["g_entropy"][rows].double()
            gl = torch.where((t >= 0) & ~empty, gl, 0.0)
            d = ge[:, None] * (info - p * info.sum(-1, keepdim=True)) - gl[:, None] * p
            d[torch.arange(len(t), device=t.device), t.clamp_min(0)] += gl
            d /= case["temperature"]
            if case["op"] == "head":
                out["d_hidden"].append(d @ w)
                out["d_head"] += d.t() @ h[rows]
            else:
                out["d_logits"].append(d)
        del x, lp, p, info
    got = {k: torch.cat(x) if isinstance(x, list) else x for k, x in out.items() if x is not None and len(x)}
    if case["op"] == "logits":
        got["rank"] = None
        if case["top"]:
            got["top_ids"] = None
    return got
