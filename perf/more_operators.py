"""More operators as measured cases: the embedding lookup with its gradient, microscaled 4-bit quantisation, the product
of microscaled operands, and the projection whose saved activations take 8 bits.

``run`` computes the plain form (elementary torch operations in 32 bits, rounded once at the end) or, with ``own`` set,
makes the calls a user of the framework makes.  Formulas:

* lookup: y_i = s T[t_i], zeros for t_i < 0 (padding); dT_v = s sum of dy_i over the positions i with t_i = v.
* microscaled blocks (OCP MX): 32 consecutive elements of a row share a scale 2^e, e = max(floor(log2 max |x|) - E, -127),
  and each element is x 2^-e rounded to the nearest E2M1 value (4 bits, E = 2, at most 6) or E4M3 value (8 bits, E = 8, at
  most 448), ties to the even one.
* product: y = act(x^ w^^T + b) + r with both operands in microscaled 4 bits (x rounded within the call);
  dz = dy act'(z), dx = dz w^ (straight through the rounding of x), db = sum dz, dr = dy.
* checkpoint: y = act(x w^T + b) + r; backward from x^ and z^, x and z = x w^T + b in microscaled 8 bits:
  dz = dy act'(z^), db = sum dz, dx = dz w, dw = dz^T x^, dr = dy.
"""

from __future__ import annotations

import math

import torch

own = False

V_THINKER, H_THINKER = 151_936, 4096  # the Thinker's vocabulary and hidden size
V_TALKER, H_TALKER = 6562, 768        # the Talker's codec vocabulary and hidden size
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}
MX = 17 / 32  # bytes of a microscaled 4-bit element, its part of the scale included


def listed():
    return [
        # the next step's input rows of a Thinker decode batch, scaled: the smallest call, latency counts
        dict(name="lookup_step", op="lookup", tokens=64, vocab=V_THINKER, width=H_THINKER, table="bf16", pads=0.1,
             scale=12.0, grad=False),
        # fine-tuning the Talker's codec embedding, an fp32 table: many positions of few ids
        dict(name="lookup_codec_train", op="lookup", tokens=30_001, vocab=V_TALKER, width=H_TALKER, table="f32", pads=0.05,
             scale=1.0, grad=True),
        # training with the Thinker's whole table on a padded batch of text
        dict(name="lookup_train", op="lookup", tokens=16_000, vocab=V_THINKER, width=H_THINKER, table="bf16", pads=0.05,
             scale=12.0, grad=True),
        # a batch of activations of an odd width to 4 bits and back
        dict(name="quantize_rows", op="quantize", rows=2000, width=H_THINKER - 1, dtype="f32"),
        # the Thinker's head to 4 bits and back
        dict(name="quantize_head", op="quantize", rows=V_THINKER, width=H_THINKER, dtype="bf16"),
        # one Thinker row projected to the Talker's width from 4-bit weights
        dict(name="product_row", op="product", rows=1, inputs=H_THINKER, outputs=H_TALKER, activation="silu", bias=True,
             residual=False, grad=False),
        # a Thinker decode step's logits from a 4-bit head: one read of the head
        dict(name="product_head_step", op="product", rows=16, inputs=H_THINKER, outputs=V_THINKER, activation="none",
             bias=False, residual=False, grad=False),
        # a prompt's rows through a square projection with everything in the epilogue
        dict(name="product_prompt", op="product", rows=2000, inputs=H_THINKER, outputs=H_THINKER, activation="gelu",
             bias=True, residual=True, grad=False),
        # the logits of a prompt's positions from a 4-bit head
        dict(name="product_head_prompt", op="product", rows=1000, inputs=H_THINKER, outputs=V_THINKER, activation="none",
             bias=False, residual=False, grad=False),
        # training below a frozen 4-bit projection to an odd width on a ragged batch
        dict(name="product_train", op="product", rows=4099, inputs=H_TALKER, outputs=2 * H_TALKER + 1, activation="silu",
             bias=True, residual=True, grad=True),
        # training a projection to an odd width on a ragged batch, activations kept in 8 bits
        dict(name="checkpoint_train", op="checkpoint", rows=4099, inputs=H_TALKER, outputs=2 * H_TALKER + 1,
             activation="silu", bias=True, residual=True),
        # training a square projection on a long batch, activations kept in 8 bits
        dict(name="checkpoint_large", op="checkpoint", rows=8192, inputs=H_THINKER, outputs=H_THINKER, activation="gelu",
             bias=True, residual=False),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "lookup", "quantize", "product", "product", "checkpoint"])
    if op == "lookup":
        table = rng.choice(["bf16", "bf16", "f32", "mx"])
        width = _log_uniform(rng, 16, 8192)
        vocab = _log_uniform(rng, 500, min(V_THINKER, 620_000_000 // width // (2 if table == "f32" else 1)))
        return dict(op=op, tokens=_log_uniform(rng, 1, min(32_768, 65_000_000 // width)), vocab=vocab, width=width,
                    table=table, pads=rng.choice([0.0, 0.1, 0.6]), scale=rng.choice([1.0, 12.0, 0.25]),
                    grad=table != "mx" and rng.random() < 0.6)
    if op == "quantize":
        width = _log_uniform(rng, 1, 16_384)
        return dict(op=op, rows=_log_uniform(rng, 1, min(200_000, 300_000_000 // width)), width=width,
                    dtype=rng.choice(["f32", "bf16"]))
    activation, bias = rng.choice(["none", "relu", "gelu", "silu"]), rng.random() < 0.7
    residual = rng.random() < 0.5
    if op == "product":
        inputs = _log_uniform(rng, 30, 8192)
        outputs = _log_uniform(rng, 40, min(V_THINKER, 600_000_000 // inputs))
        grad = rng.random() < 0.3
        most = min(1.2e12 / (2 * inputs * outputs * (2 if grad else 1)), 150_000_000 / outputs / (2 if grad else 1))
        return dict(op=op, rows=_log_uniform(rng, 1, max(1, min(8192, int(most)))), inputs=inputs, outputs=outputs,
                    activation=activation, bias=bias, residual=residual, grad=grad)
    inputs, outputs = 8 * _log_uniform(rng, 8, 1024), _log_uniform(rng, 40, 8192)
    most = int(min(0.8e12 / (6 * inputs * outputs), 33_000_000 / max(inputs, outputs)))
    return dict(op=op, rows=_log_uniform(rng, 1, max(1, min(8192, most))), inputs=inputs, outputs=outputs,
                activation=activation, bias=bias, residual=residual)


# ------------------------------------------------------------------------------------------ microscaled blocks

def _pow2(e):
    """2^e in fp32 for whole e in [-149, 127], by its bits."""
    e = e.to(torch.int32)
    return torch.where(e >= -126, (e + 127) << 23, 1 << (e + 149).clamp(0, 22)).view(torch.float32)


def _blocks(x):
    """Rows of fp32 as [rows, blocks, 32], the last block filled up with zeros."""
    rows, k = x.shape
    full = -(-k // 32) * 32
    return torch.nn.functional.pad(x, (0, full - k)).view(rows, full // 32, 32)


def _mx(x, top, fraction, lowest, largest):
    """The blocks of x [rows, k] (fp32): each element's value in units of its scale, and the scales' exponents."""
    b = _blocks(x)
    e = (torch.frexp(b.abs().amax(-1, keepdim=True)).exponent - 1 - top).clamp(-127, 127)
    y = b * _pow2(-e)
    step = _pow2((torch.frexp(y).exponent - 1).clamp_min(lowest) - fraction)
    return (torch.round(y / step) * step).clamp(-largest, largest), e


def _mx_rounded(x, fmt):
    q, e = _mx(x.float(), 2, 1, 0, 6.0) if fmt == "e2m1" else _mx(x.float(), 8, 3, -6, 448.0)
    return (q * _pow2(e)).view(x.shape[0], -1)[:, :x.shape[1]]


def _mx_pack(w):
    """w [rows, k] as E2M1 codes ([rows, 16 bytes a block], the first of two elements in the low half of a byte) and E8M0
    scales in tiles of 128 rows x 8 blocks, 1024 bytes each: two halves of 4 blocks, in each row % 32 and row / 32."""
    rows, k = w.shape
    nb = -(-k // 32)
    codes, scales = [], torch.zeros(-(-rows // 128) * 128, -(-nb // 8) * 8, dtype=torch.uint8, device=w.device)
    for a in range(0, rows, 16_384):
        q, e = _mx(w[a:a + 16_384].float(), 2, 1, 0, 6.0)
        m = q.abs()
        c = torch.where(m < 2, m * 2, torch.where(m < 4, m + 2, m * 0.5 + 4)).to(torch.uint8) + (q < 0).to(torch.uint8) * 8
        c = c.view(len(q), -1, 2)
        codes.append(c[:, :, 0] | c[:, :, 1] << 4)
        scales[a:a + 16_384, :nb][:len(q)] = (e[:, :, 0] + 127).to(torch.uint8)
    tiles = scales.view(-1, 4, 32, scales.shape[1] // 8, 2, 4).permute(0, 3, 4, 2, 1, 5)
    return torch.cat(codes), tiles.reshape(tiles.shape[0], tiles.shape[1], 1024).contiguous()


def _mx_values(codes, scales, k):
    """The values [rows, k] (fp32) of packed codes and their scales' tiles."""
    rows = codes.shape[0]
    c = torch.stack((codes & 15, codes >> 4), -1).view(rows, -1, 32)
    at = scales.view(scales.shape[0], scales.shape[1], 2, 32, 4, 4).permute(0, 4, 3, 1, 2, 5)
    e = at.reshape(scales.shape[0] * 128, -1)[:rows, :c.shape[1]].to(torch.int32) - 127
    m = (c & 7).float()
    v = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2, m * 2 - 8))
    return (torch.where(c >= 8, -v, v) * _pow2(e)[:, :, None]).view(rows, -1)[:, :k]


# ------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def weight(n, k, dtype=torch.bfloat16):
        return torch.empty(n, k, device=dev, dtype=dtype).normal_(0.0, 1 / math.sqrt(k), generator=g)

    op = case["op"]
    if op == "lookup":
        n, v = case["tokens"], case["vocab"]
        # ids fall off like a vocabulary's, P(t) ~ 1 / (t + 1), and some positions are padding
        t = torch.exp(torch.rand(n, device=dev, generator=g, dtype=torch.float64) * math.log(v + 1)).long().sub_(1).clamp_(0, v - 1)
        t[torch.rand(n, device=dev, generator=g) < case["pads"]] = -1
        table = weight(v, case["width"], DTYPES.get(case["table"], torch.bfloat16))
        s = dict(tokens=t)
        if case["table"] == "mx":
            s["codes"], s["scales"] = _mx_pack(table)
        else:
            s["table"] = table
        if case["grad"]:
            s["dy"] = normal(n, case["width"]).to(table.dtype)
        return {"case": dict(case), **s}
    if op == "quantize":
        # rows of different magnitudes, a few outlying columns
        n, k = case["rows"], case["width"]
        x = torch.empty(n, k, device=dev, dtype=DTYPES[case["dtype"]]).normal_(generator=g)
        x *= torch.exp2(torch.randint(-6, 7, (n, 1), device=dev, generator=g)).to(x.dtype)
        x[:, ::97] *= 8
        return {"case": dict(case), "x": x}
    n, k, m = case["rows"], case["inputs"], case["outputs"]
    s = dict(x=normal(n, k).bfloat16(), bias=(normal(m) * 0.5).bfloat16() if case["bias"] else None,
             residual=normal(n, m).bfloat16() if case["residual"] else None)
    if op == "product":
        s["codes"], s["scales"] = _mx_pack(weight(m, k))
    else:
        s["weight"] = weight(m, k)
    if op == "checkpoint" or case["grad"]:
        s["dy"] = normal(n, m).bfloat16()
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


def _plain_lookup(s):
    c, t = s["case"], s["tokens"]
    at, real = t.clamp_min(0), (t >= 0)[:, None]
    if c["table"] == "mx":
        tiles = torch.arange(s["scales"].shape[1], device=t.device)[None, :]
        inside = s["scales"].view(*s["scales"].shape[:2], 2, 32, 4, 4)[
            (at // 128)[:, None], tiles, :, (at % 32)[:, None], (at % 128 // 32)[:, None]]
        e = inside.reshape(len(t), -1)[:, :s["codes"].shape[1] // 16].to(torch.int32) - 127
        b = s["codes"][at]
        q = torch.stack((b & 15, b >> 4), -1).view(len(t), -1, 32)
        m = (q & 7).float()
        v = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2, m * 2 - 8))
        rows = (torch.where(q >= 8, -v, v) * _pow2(e)[:, :, None]).view(len(t), -1)[:, :c["width"]]
        return dict(y=torch.where(real, rows * c["scale"], torch.zeros_like(rows)).bfloat16())
    rows = s["table"][at].float()
    out = dict(y=torch.where(real, rows * c["scale"], torch.zeros_like(rows)).to(s["table"].dtype))
    if c["grad"]:
        d = torch.zeros(c["vocab"], c["width"], device=t.device)
        d.index_add_(0, at, torch.where(real, s["dy"].float(), torch.zeros_like(rows)))
        out["d_table"] = (d * c["scale"]).to(s["table"].dtype)
    return out


def _plain_quantize(s):
    return dict(values=_mx_rounded(s["x"], "e2m1").to(s["x"].dtype))


def _plain_products(s):
    c = s["case"]
    x, kind = s["x"].float(), c["activation"]
    product = c["op"] == "product"
    w = _mx_values(s["codes"], s["scales"], c["inputs"]) if product else s["weight"].float()
    z = (_mx_rounded(x, "e2m1") if product else x) @ w.t()
    if c["bias"]:
        z = z + s["bias"].float()
    y = _activation(z, kind)
    if c["residual"]:
        y = y + s["residual"].float()
    out = dict(y=y.bfloat16())
    if not product or c["grad"]:
        dy = s["dy"].float()
        dz = dy if kind == "none" else dy * _activation_slope(z if product else _mx_rounded(z, "e4m3"), kind)
        out["d_x"] = (dz @ w).bfloat16()
        if not product:
            out["d_weight"] = (dz.t() @ _mx_rounded(x, "e4m3")).bfloat16()
        if c["bias"]:
            out["d_bias"] = dz.sum(0).bfloat16()
        if c["residual"]:
            out["d_residual"] = s["dy"]
    return out


# ------------------------------------------------------------------------------------------ the framework's calls

def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _own_lookup(s):
    c, p = s["case"], _package()
    if c["table"] == "mx":
        table = p.mx.MXTensor(s["codes"], s["scales"], (c["vocab"], c["width"]))
        return dict(y=p.embedding.lookup(s["tokens"], table, scale=c["scale"]))
    if not c["grad"]:
        return dict(y=p.embedding.lookup(s["tokens"], s["table"], scale=c["scale"]))
    table = s["table"].detach().requires_grad_(True)
    y = p.embedding.lookup(s["tokens"], table, scale=c["scale"])
    d, = torch.autograd.grad(y, (table,), s["dy"])
    return dict(y=y.detach(), d_table=d)


def _own_quantize(s):
    mx = _package().mx
    return dict(values=mx.dequantize(mx.quantize(s["x"]), dtype=s["x"].dtype))


def _own_products(s):
    c, p = s["case"], _package()
    act = None if c["activation"] == "none" else c["activation"]
    if c["op"] == "product":
        w = p.mx.MXTensor(s["codes"], s["scales"], (c["outputs"], c["inputs"]))
        if not c["grad"]:
            return dict(y=p.mx.linear(s["x"], w, s["bias"], activation=act, residual=s["residual"]))
        leaf = {k: s[k].detach().requires_grad_(True) for k in ("x", "bias", "residual") if s[k] is not None}
        y = p.mx.linear(leaf["x"], w, leaf.get("bias"), activation=act, residual=leaf.get("residual"))
    else:
        leaf = {k: s[k].detach().requires_grad_(True) for k in ("x", "weight", "bias", "residual") if s[k] is not None}
        y = p.projection.linear(leaf["x"], leaf["weight"], leaf.get("bias"), activation=act,
                                residual=leaf.get("residual"), checkpoint="e4m3")
    grads = torch.autograd.grad(y, tuple(leaf.values()), s["dy"])
    return dict(y=y.detach(), **{"d_" + k: d for k, d in zip(leaf, grads)})


def run(state):
    op = state["case"]["op"]
    if own:
        return {"lookup": _own_lookup, "quantize": _own_quantize}.get(op, _own_products)(state)
    return {"lookup": _plain_lookup, "quantize": _plain_quantize}.get(op, _plain_products)(state)


def work(case):
    if case["op"] == "lookup":
        n, v, w = case["tokens"], case["vocab"], case["width"]
        e = BYTES.get(case["table"], MX)
        moved = 8 * n + min(n, v) * w * e + n * w * max(e, 2)
        if case["grad"]:
            moved += n * w * e + v * w * e
        return {"bytes": moved, "flops": n * w * (2 if case["grad"] else 1)}
    if case["op"] == "quantize":  # there and back
        n = case["rows"] * case["width"]
        return {"bytes": 2 * n * (BYTES[case["dtype"]] + MX), "flops": 6 * n}
    n, k, m = case["rows"], case["inputs"], case["outputs"]
    extra = (m if case["bias"] else 0) + (n * m if case["residual"] else 0)
    if case["op"] == "product":
        moved, flops = 2 * (n * k + n * m + extra) + m * k * MX, 2 * n * k * m
        if case["grad"]:  # dy and the weight read; dx, db and dr written
            moved, flops = moved + 2 * (n * m + n * k + extra) + m * k * MX, 2 * flops
        return {"bytes": moved, "flops": flops}
    # dy read; x kept and read, z too, in 8 bits; dx, dw, db and dr written
    kept = 2 * 33 / 32 * (n * k + (n * m if case["activation"] != "none" else 0))
    return {"bytes": 2 * (n * k + k * m + n * m + extra) * 2 + kept, "flops": 6 * n * k * m}


# ------------------------------------------------------------------------------------------ in 64 bits

def _nearest(x, grid, top):
    """Each block of 32 of x (float64, [rows, k]) on the nearest of its scaled grid's values, ties to the even code."""
    rows, k = x.shape
    out = torch.zeros(rows, -(-k // 32) * 32, dtype=torch.float64, device=x.device)
    out[:, :k] = x
    out = out.view(rows, -1, 32)
    most = out.abs().amax(-1, keepdim=True)
    scale = torch.ldexp(torch.ones_like(most), (torch.frexp(most).exponent - 1 - top).clamp_min(-127))
    y = out.abs() / scale
    mid = (grid[1:] + grid[:-1]) / 2
    up, down = torch.bucketize(y, mid, right=True), torch.bucketize(y, mid)  # a tie lies between the two
    return (torch.copysign(grid[torch.where(up % 2 == 0, up, down)], out) * scale).view(rows, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    dev = torch.device("cuda")
    four = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=dev)
    eight = torch.tensor([i * 2.0 ** -9 for i in range(8)] + [(8 + i % 8) * 2.0 ** (i // 8 - 9) for i in range(119)],
                         dtype=torch.float64, device=dev)
    if case["op"] == "quantize":
        x = s["x"]
        step = max(1, 100_000_000 // x.shape[1])
        return dict(values=torch.cat([_nearest(x[a:a + step].double(), four, 2).to(x.dtype) for a in range(0, len(x), step)]))

    def unpacked(rows):  # of the packed matrix: signed codes, then the scale of each block found by its address
        c = s["codes"][rows].long()
        q = torch.stack((c % 16, c // 16), -1).flatten(1)
        v = four[q % 8] * (1 - 2 * (q // 8))
        b = torch.arange(q.shape[1], device=dev)[None, :] // 32
        r = rows[:, None]
        place = (r // 128 * s["scales"].shape[1] + b // 8) * 1024 + b % 8 // 4 * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4
        return torch.ldexp(v, s["scales"].flatten()[place].int() - 127)

    if case["op"] == "lookup":
        t, w = s["tokens"], case["width"]
        pad = (t < 0)[:, None]
        rows = unpacked(t.clamp_min(0))[:, :w] if case["table"] == "mx" else s["table"][t.clamp_min(0)].double()
        out = dict(y=rows.mul_(case["scale"]).masked_fill_(pad, 0.0))
        if case["grad"]:
            d = torch.zeros(case["vocab"] + 1, w, dtype=torch.float64, device=dev)  # padding goes to a row of its own
            d.index_add_(0, torch.where(t < 0, case["vocab"], t), s["dy"].double())
            out["d_table"] = d[:-1].mul_(case["scale"])
        return out
    n, k, m, kind = case["rows"], case["inputs"], case["outputs"], case["activation"]
    product = case["op"] == "product"
    x = s["x"].double()
    xq = _nearest(x, four, 2) if product else x
    z = torch.empty(n, m, dtype=torch.float64, device=dev)
    step = max(1, 100_000_000 // k)
    weight = lambda a: unpacked(torch.arange(a, min(a + step, m), device=dev))[:, :k] if product else s["weight"][a:a + step].double()  # noqa: E731
    for a in range(0, m, step):
        z[:, a:a + step] = torch.einsum("nk,mk->nm", xq, weight(a))
    if s["bias"] is not None:
        z += s["bias"].double()

    def gate(u):
        return torch.special.ndtr(u) if kind == "gelu" else torch.sigmoid(u) if kind == "silu" else (u > 0).double()

    y = z if kind == "none" else z * gate(z)
    out = dict(y=y if s["residual"] is None else y + s["residual"].double())
    if product and not case["grad"]:
        return out
    u = z if product or kind == "none" else _nearest(z, eight, 8)
    dz = s["dy"].double()
    if kind != "none":
        p = gate(u)
        dz = dz * {"relu": lambda: p, "silu": lambda: p + u * p * (1 - p),
                   "gelu": lambda: p + u * torch.exp(-u * u / 2) * (2 * math.pi) ** -0.5}[kind]()
    out["d_x"] = sum(torch.einsum("nm,mk->nk", dz[:, a:a + step], weight(a)) for a in range(0, m, step))
    if not product:
        out["d_weight"] = torch.einsum("nm,nk->mk", dz, _nearest(x, eight, 8))
    if s["bias"] is not None:
        out["d_bias"] = dz.sum(0)
    if s["residual"] is not None:
        out["d_residual"] = None
    return out
