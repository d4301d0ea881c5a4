"""The operators of a training step on weights in FP8 blocks as timed cases: layer
norm and its gradients, the product of FP8 operands with a scale for each block of
128 and its gradients, and the AdamW step of many tensors with its states in 32 or
8 bits, which writes the weights' blocks again.

A case is one call, or one forward and backward, as a program that trains or
serves a token model on such weights makes it.  ``run`` computes it in plain fp32
torch operations, or with ``own`` set through ``novann_amd``.  ``exact`` restates
every case in 64 bits from the same seeded inputs.

Blocks.  A scale is a power of two, kept as its exponent e in 8 bits: 2^(e - 127)
is the smallest with max |x| of the block within the type's largest value (1 for a
block of zeros).  An activation or a gradient has one for 128 columns of a row, a
weight one for 128 x 128; rows of codes are padded with zeros to whole blocks, rows
of exponents to whole fours.

States in 8 bits.  128 elements in a row share two such exponents.  m is E4M3, v
has no sign: code c > 0 is the float whose bits are (c << 20) + ((e - 31) << 23).
Both are rounded up with the probability of their place between two codes, by the
halves of a 32-bit random number made from the step's seed and the element's place
in the list; a v that is not zero never becomes zero.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FMT_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
TOP = {"e4m3": 8, "e5m2": 15}      # the exponent of the largest value
BLOCK = 128
EPS = 1e-5
ADAM = {"lr": 1e-4, "betas": (0.9, 0.999), "weight_decay": 0.1, "epsilon": 1e-8}


# --------------------------------------------------------------------------
# the cases

def listed():
    return [
        # one decoding step: the norm before a layer, stored in blocks, and the layer
        serve("serve 1x4096 to 4096", 1, 4096, 4096, "bf16"),
        # a small ragged batch of requests through a wide layer
        serve("serve 37x1024 to 4096", 37, 1024, 4096, "f16"),
        # a fine-tuning micro-batch, odd width: norm and its gradients
        norm("norm train 1000x784", 1000, 784, "f16"),
        # a training batch of a wide model: norm and its gradients
        norm("norm train 16384x4096", 16384, 4096, "bf16"),
        # a prompt through one layer, activations that are not in blocks yet
        linear("linear 2048x4096x4096", 2048, 4096, 4096, "bf16", "e4m3", False),
        # the ragged batch of the second norm, its layer in training, gradients of wide range
        linear("linear train 1000x784x1000", 1000, 784, 1000, "f16", "e5m2", True),
        # a training batch of a small model's feed-forward layer
        linear("linear train 8192x1024x4096", 8192, 1024, 4096, "bf16", "e4m3", True),
        # a wide model's feed-forward layer: the largest products
        linear("linear train 8192x4096x16384", 8192, 4096, 16384, "bf16", "e4m3", True),
        # a small model, where the calls' latency counts
        step("step small", 2, 128, 1000, "f32", 32),
        # a model of odd widths, float16 gradients, states in 8 bits
        step("step ragged 8-bit", 12, 500, 30001, "f16", 8),
        # a model of 24 blocks: bf16 gradients, states in 8 bits
        step("step 24 blocks 8-bit", 24, 1024, 50000, "bf16", 8),
        # the square weights of a model's layers and their FP8 blocks, fp32 states
        blocks("step 8 weights 4096x4096", 8, 4096, 4096, "bf16", 32),
    ]


def serve(name, rows, width, outs, x):
    return {"name": name, "op": "serve", "rows": rows, "width": width, "outs": outs, "xdtype": x}


def norm(name, rows, width, x):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "xdtype": x}


def linear(name, rows, width, outs, x, g, train):
    return {"name": name, "op": "linear", "rows": rows, "width": width, "outs": outs,
            "xdtype": x, "gdtype": g, "train": train}


def step(name, layers, width, vocab, g, bits):
    return {"name": name, "op": "step", "layers": layers, "width": width, "vocab": vocab,
            "gdtype": g, "bits": bits}


def blocks(name, count, rows, cols, g, bits):
    return {"name": name, "op": "blocks", "count": count, "rows": rows, "cols": cols,
            "gdtype": g, "bits": bits}


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def _width(rng, lo, hi):
    """A width: whole multiples of 16, 64 or 256, or (one in four) any number."""
    v = _log(rng, lo, hi)
    unit = rng.choice([1, 16, 64, 256])
    return v if v < 2 * unit else v // unit * unit


def draw(rng):
    kind = rng.choice(["serve", "norm", "norm", "linear", "linear train", "linear train",
                       "step", "step", "blocks"])
    x = rng.choice(["bf16", "f16"])
    if kind == "serve":
        c = serve("", _log(rng, 1, 256), _width(rng, 64, 4096), _width(rng, 64, 8192), x)
    elif kind == "norm":
        x = rng.choice(["f32", "bf16", "f16"])
        c = norm("", _log(rng, 1, 16384), _width(rng, 64, 4096), x)
    elif kind in ("linear", "linear train"):
        width, outs = _width(rng, 64, 4096), _width(rng, 64, 16384)
        c = linear("", _log(rng, 1, 8192), width, outs, x, rng.choice(["e4m3", "e5m2"]),
                   kind == "linear train")
    elif kind == "step":
        c = step("", _log(rng, 1, 24), _width(rng, 64, 1024), _width(rng, 1000, 50000),
                 rng.choice(["f32", "bf16", "f16"]), rng.choice([8, 32]))
    else:
        c = blocks("", rng.randint(1, 8), _width(rng, 64, 4096), _width(rng, 64, 4096),
                   rng.choice(["f32", "bf16", "f16"]), rng.choice([8, 32]))
    c.pop("name", None)
    return c


# --------------------------------------------------------------------------
# blocks in plain torch

def _pad(n, unit):
    return -(-n // unit) * unit


def _exponents(amax, top):
    """The exponents of blocks whose largest magnitudes are amax (fp32)."""
    bits = amax.view(torch.int32)
    e = (bits >> 23) - top + ((bits & 0x7FFFFF) > 0x600000).int()
    return torch.where(amax > 0, e.clamp(1, 254), 127).to(torch.uint8)


def _power(e):
    """2^(e - 127) in fp32, e from 1 to 254."""
    return (e.int() << 23).view(torch.float32)


def _padded(e):
    """Rows of exponents padded to whole fours with those of 1."""
    return torch.nn.functional.pad(e, (0, -e.shape[-1] % 4), value=127)


def _row_blocks(x, dtype):
    """(codes with whole blocks of columns, exponents) of x (..., R, C), a scale for 128
    columns of a row."""
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % BLOCK))
    b = x.unflatten(-1, (-1, BLOCK))
    e = _exponents(b.abs().amax(-1), TOP[dtype])
    q = b * _power(254 - e).unsqueeze(-1)
    q = q.clamp(-FMT_MAX[dtype], FMT_MAX[dtype]).to(FP8[dtype])
    return q.flatten(-2), e


def _tile_blocks(x, dtype):
    """The same with a scale for 128 x 128."""
    rows = x.shape[-2]
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % BLOCK, 0, -rows % BLOCK))
    b = x.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, BLOCK))   # (..., Rb, 128, Cb, 128)
    e = _exponents(b.abs().amax((-3, -1)), TOP[dtype])
    q = b * _power(254 - e).unsqueeze(-2).unsqueeze(-1)
    q = q.clamp(-FMT_MAX[dtype], FMT_MAX[dtype]).to(FP8[dtype])
    return q.flatten(-2).flatten(-3, -2)[..., :rows, :], e


def _values(q, e, cols):
    """What codes with a scale for 128 columns of a row stand for, in fp32."""
    v = q.float().unflatten(-1, (-1, BLOCK)) * _power(e).unsqueeze(-1)
    return v.flatten(-2)[..., :cols]


def _tile_values(q, e, cols):
    """What codes with a scale for 128 x 128 stand for, in fp32."""
    return _values(q, e.repeat_interleave(BLOCK, -2)[..., :q.shape[-2], :], cols)


# --------------------------------------------------------------------------
# states in 8 bits

_M32 = (1 << 32) - 1
_M64 = (1 << 64) - 1


def _key(seed):
    """A seed's 32 bits."""
    x = (seed * 0x9E3779B97F4A7C15 + 0x3C6EF372FE94F82B) & _M64
    x = ((x ^ (x >> 32)) * 0xBB67AE8584CAA73B) & _M64
    x = ((x ^ (x >> 29)) * 0x6A09E667F3BCC909) & _M64
    return x >> 32


def _random(n, seed, dev):
    """The random numbers of elements 0 .. n - 1: 20 bits for m and 20 for v (the lowest
    four the middle of what the upper sixteen leave open)."""
    h = ((torch.arange(n, device=dev) + _key(seed)) * 0x9E3779B9) & _M32
    h = ((h ^ (h >> 16)) * 0x6A09E667) & _M32
    h = h ^ (h >> 15)
    return ((h >> 16) << 4 | 8).int(), ((h & 0xFFFF) << 4 | 8).int()


def _pack(m, v, seed):
    """m, v (n,), n whole blocks, as {"m", "me", "v", "ve"}."""
    rm, rv = _random(m.numel(), seed, m.device)
    a = m.abs().view(-1, BLOCK)
    bits = a.amax(1).view(torch.int32)
    e = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(1, 254)
    a = (a * _power(254 - e).unsqueeze(1)).flatten()
    normal = ((a.view(torch.int32) + rm) & ~0xFFFFF).view(torch.float32)
    small = (a * 512.0 + rm.float() * 2.0 ** -20).floor() * 2.0 ** -9
    s = {"m": torch.where(a < 2.0 ** -6, small, normal).copysign_(m).to(FP8["e4m3"]),
         "me": e.to(torch.uint8)}
    bits = v.view(-1, BLOCK).amax(1).view(torch.int32)
    e = ((bits >> 23) + ((bits & 0x7FFFFF) > 0x700000).int()).clamp(40, 254)
    c = v.view(torch.int32).view(-1, BLOCK) - ((e - 31) << 23).unsqueeze(1)
    c = torch.where(c < 1 << 20, 1, (c + rv.view(-1, BLOCK)) >> 20).clamp(max=255)
    s["v"] = torch.where(v.view(-1, BLOCK) > 0, c, 0).to(torch.uint8).flatten()
    s["ve"] = e.to(torch.uint8)
    return s


def _unpack(s):
    """(m, v) in fp32."""
    m = (s["m"].float().view(-1, BLOCK) * _power(s["me"]).unsqueeze(1)).flatten()
    c = s["v"].int().view(-1, BLOCK)
    v = ((c << 20) + ((s["ve"].int() - 31) << 23).unsqueeze(1)).view(torch.float32)
    return m, torch.where(c > 0, v, 0.0).flatten()


# --------------------------------------------------------------------------
# inputs

class Inputs:
    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.gen = torch.Generator(device=self.dev)
        self.gen.manual_seed(int(seed))

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device=self.dev)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.gen, device=self.dev)

    def hidden(self, rows, width, dtype):
        """Hidden states: tokens of different size and a few columns that stand out."""
        x = self.normal(rows, width) * (0.25 + 2 * self.uniform(rows, 1))
        return (x * (1 + 15 * (self.uniform(width) < 0.01))).to(TORCH[dtype])

    def grad(self, rows, width, dtype):
        """Their gradients, of a mean over many tokens in a loss scaled for 16 bits."""
        g = self.normal(rows, width) * (0.02 + self.uniform(rows, 1) ** 4)
        return (g / 16).to(TORCH[dtype])

    def weight(self, outs, width):
        """A layer's weight in E4M3 blocks, as a product reads it and as its gradient
        does."""
        q, e = _tile_blocks(self.normal(outs, width) / math.sqrt(width), "e4m3")
        t = q[:, :width].view(torch.uint8).t()
        t = torch.nn.functional.pad(t, (0, -outs % BLOCK)).contiguous().view(FP8["e4m3"])
        return {"shape": (outs, width), "q": q, "e": _padded(e), "qt": t,
                "et": _padded(e.t().contiguous())}


def _shapes(case):
    """The parameters of a model of that many layers: per layer two scale vectors, an
    attention's four matrices and a feed-forward's two, then the table and a last scale
    vector; or the weights of a case of blocks."""
    if case["op"] == "blocks":
        return [(case["rows"], case["cols"])] * case["count"]
    d = case["width"]
    layer = [(d,), (d, d), (d, d), (d, d), (d, d), (d,), (4 * d, d), (d, 4 * d)]
    return layer * case["layers"] + [(case["vocab"], d), (d,)]


def _parts(flat, shapes, unit=1):
    """Views of the tensors in one buffer, each from whole blocks on, a value for `unit`
    elements."""
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at // unit:(at + _pad(n, BLOCK)) // unit] if unit > 1
                   else flat[at:at + n].view(s))
        at += _pad(n, BLOCK)
    return out


def prepare(case, seed):
    make = Inputs(seed)
    s = {"case": case}
    op = case["op"]
    if op in ("serve", "norm"):
        d = case["width"]
        s["x"] = make.hidden(case["rows"], d, case["xdtype"])
        s["gamma"] = 1 + 0.2 * make.normal(d)
        s["beta"] = 0.1 * make.normal(d)
    if op == "norm":
        s["g"] = make.grad(case["rows"], case["width"], case["xdtype"])
    if op == "linear":
        s["x"] = make.hidden(case["rows"], case["width"], case["xdtype"])
        if case["train"]:
            s["g"] = make.grad(case["rows"], case["outs"], case["xdtype"])
    if op in ("serve", "linear"):
        s["w"] = make.weight(case["outs"], case["width"])
        s["bias"] = 0.1 * make.normal(case["outs"])
    if op in ("step", "blocks"):
        s["t"] = 1 + seed % 1000
        shapes = _shapes(case)
        n = sum(_pad(math.prod(p), BLOCK) for p in shapes)
        w, g = torch.zeros(n, device=make.dev), torch.zeros(n, device=make.dev)
        m, v = torch.zeros_like(w), torch.zeros_like(w)
        sizes = 10 ** (-2 * make.uniform(len(shapes))) * 1e-3
        for i, (a, b, c, d) in enumerate(zip(*(_parts(f, shapes) for f in (w, g, m, v)))):
            a.copy_(make.normal(*a.shape) * (0.5 / math.sqrt(a.shape[-1])))
            std = sizes[i] * (0.3 + make.uniform(*a.shape[:-1], 1))
            b.copy_(make.normal(*a.shape) * std)
            c.copy_(make.normal(*a.shape) * std / 4)
            d.copy_((std * (0.5 + make.uniform(*a.shape))) ** 2)
        s["w"], s["g"] = w, g.to(TORCH[case["gdtype"]])
        if case["bits"] == 8:
            s["s"] = _pack(m, v, seed)
        else:
            s["m"], s["v"] = m, v
        if op == "blocks":
            s["codes"] = _codes(case, w)
    return s


def _matrices(case, w):
    """The weights of a case of blocks, as one array."""
    n = case["rows"] * case["cols"]
    return w.view(case["count"], -1)[:, :n].view(-1, case["rows"], case["cols"])


def _codes(case, w):
    """Their blocks: what a product reads, and the transposed codes of its gradient."""
    q, e = _tile_blocks(_matrices(case, w), "e4m3")
    t = q[..., :case["cols"]].view(torch.uint8).transpose(1, 2)
    t = torch.nn.functional.pad(t, (0, -case["rows"] % BLOCK)).contiguous().view(FP8["e4m3"])
    return {"q": q, "e": _padded(e), "qt": t, "et": _padded(e.transpose(1, 2).contiguous())}


# --------------------------------------------------------------------------
# one pass

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from novann_amd import functional as F
    from novann_amd import optim, quant
    case = s["case"]
    if case["op"] == "norm":
        y, mean, rstd = F.layer_norm(s["x"], s["gamma"], s["beta"], eps=EPS, extras=True)
        gx, gw, gb = F.layer_norm_backward(s["g"], s["x"], s["gamma"], mean, rstd)
        return {"out": y, "grad_input": gx, "grad_weight": gw, "grad_bias": gb}
    if case["op"] == "serve":
        x = F.layer_norm(s["x"], s["gamma"], s["beta"], eps=EPS, out_dtype="e4m3")
        return {"out": F.block_linear(x, _weight(s["w"]), s["bias"], out_dtype=case["xdtype"])}
    if case["op"] == "linear":
        w = _weight(s["w"])
        if not case["train"]:
            return {"out": F.block_linear(s["x"], w, s["bias"], out_dtype=case["xdtype"])}
        y, kept = F.block_linear(s["x"], w, s["bias"], out_dtype=case["xdtype"], extras=True)
        gx, gw, gb = F.block_linear_backward(s["g"], kept, w, grad_dtype=case["gdtype"])
        return {"out": y, "grad_input": gx, "grad_weight": gw, "grad_bias": gb.view(-1)}
    shapes = _shapes(case)
    if case["bits"] == 8:
        names = [("m", 1), ("me", BLOCK), ("v", 1), ("ve", BLOCK)]
        states = [optim.State8(*parts) for parts in zip(
            *(_parts(s["s"][k], shapes, unit) for k, unit in names))]
    else:
        states = list(zip(_parts(s["m"], shapes), _parts(s["v"], shapes)))
    weights = _parts(s["w"], shapes)
    if case["op"] == "blocks":
        weights = [_quantized(w, *c) for w, c in zip(weights, zip(*(
            s["codes"][k] for k in ("q", "e", "qt", "et"))))]
    optim.adamw_step(weights, _parts(s["g"], shapes), states, step=s["t"], seed=s["t"], **ADAM)
    out = {"w": s["w"]}
    if case["bits"] == 8:
        out["m"], out["v"] = optim.State8(*(s["s"][k] for k in ("m", "me", "v", "ve"))).decode(
            "bf16")
    else:
        out["m"], out["v"] = s["m"], s["v"]
    if case["op"] == "blocks":
        out["q"] = [quant.dequantize_blocks(w.blocks(), "bf16") for w in weights]
        out["qt"] = s["codes"]["qt"]
    return out


def _weight(w):
    from novann_amd.module import BlockQuantizedParameters
    return BlockQuantizedParameters(w["q"], w["e"], w["shape"], "e4m3", codes_t=w["qt"],
                                    exponents_t=w["et"])


def _quantized(master, q, e, qt, et):
    from novann_amd.module import BlockQuantizedParameters
    return BlockQuantizedParameters(q, e, master.shape, "e4m3", codes_t=qt, exponents_t=et,
                                    master=master)


def _normed(s):
    """(the norm's output, the normalised rows, their 1 / deviation) in fp32."""
    x = s["x"].float()
    c = x - x.mean(1, keepdim=True)
    rstd = 1 / (c.square().mean(1, keepdim=True) + EPS).sqrt()
    n = c * rstd
    return n * s["gamma"] + s["beta"], n, rstd


def _plain(s):
    case = s["case"]
    if case["op"] in ("step", "blocks"):
        return _plain_step(s)
    xdt = TORCH[case["xdtype"]]
    if case["op"] == "norm":
        y, n, rstd = _normed(s)
        g = s["g"].float()
        h = g * s["gamma"]
        gx = rstd * (h - h.mean(1, keepdim=True) - n * (h * n).mean(1, keepdim=True))
        return {"out": y.to(xdt), "grad_input": gx.to(xdt), "grad_weight": (g * n).sum(0),
                "grad_bias": g.sum(0)}
    w, d, outs = s["w"], case["width"], case["outs"]
    wf = _tile_values(w["q"], w["e"][:, :-(-d // BLOCK)], d)
    x = _normed(s)[0] if case["op"] == "serve" else s["x"].float()
    y = (_values(*_row_blocks(x, "e4m3"), d) @ wf.t() + s["bias"]).to(xdt)
    if case["op"] == "serve" or not case["train"]:
        return {"out": y}
    n, g = case["rows"], s["g"].float()
    gx = _values(*_row_blocks(g, case["gdtype"]), outs) @ wf
    gt = _values(*_row_blocks(g.t(), case["gdtype"]), n)
    xt = _values(*_row_blocks(x.t(), "e4m3"), n)
    return {"out": y, "grad_input": gx.to(xdt), "grad_weight": (gt @ xt.t()).to(xdt),
            "grad_bias": g.sum(0)}


def _plain_step(s):
    case, w, g = s["case"], s["w"], s["g"].float()
    (b1, b2), lr = ADAM["betas"], ADAM["lr"]
    m, v = _unpack(s["s"]) if case["bits"] == 8 else (s["m"], s["v"])
    m.mul_(b1).add_(g * (1 - b1))
    v.mul_(b2).add_((g * g) * (1 - b2))
    # (device scalars: torch divides by a Python number by multiplying)
    bc1 = torch.full((), 1 - b1 ** s["t"], device=w.device)
    bc2 = torch.full((), 1 - b2 ** s["t"], device=w.device)
    w.sub_(((m / bc1) * lr) / ((v / bc2).sqrt() + ADAM["epsilon"]))
    w.sub_(w * (lr * ADAM["weight_decay"]))
    out = {"w": w, "m": m, "v": v}
    if case["bits"] == 8:
        new = _pack(m, v, s["t"])
        for k in new:
            s["s"][k].copy_(new[k])
        m, v = _unpack(s["s"])
        out["m"], out["v"] = m.bfloat16(), v.bfloat16()
    if case["op"] == "blocks":
        new, c = _codes(case, w), s["codes"]
        for k in new:
            c[k].copy_(new[k])
        q = _tile_values(c["q"], c["e"][..., :-(-case["cols"] // BLOCK)], case["cols"])
        out["q"] = list(q.bfloat16().unbind(0))
        out["qt"] = c["qt"]
    return out


# --------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "norm":
        n, b = case["rows"] * case["width"], BYTES[case["xdtype"]]
        return {"bytes": 4 * n * b + 16 * case["width"] + 8 * case["rows"], "flops": 20 * n}
    if op in ("serve", "linear"):
        n, d, outs, b = case["rows"], case["width"], case["outs"], BYTES[case["xdtype"]]
        moved = (n * d + n * outs) * b + outs * d + 4 * outs
        if op == "serve":
            return {"bytes": moved + 8 * d, "flops": 2 * n * d * outs}
        if case["train"]:  # the output's gradient, and three gradients
            moved += (n * outs + n * d + outs * d) * b + 4 * outs
        return {"bytes": moved, "flops": (6 if case["train"] else 2) * n * d * outs}
    n = sum(math.prod(p) for p in _shapes(case))
    each = 8 + BYTES[case["gdtype"]] + (16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4)
    if op == "blocks":  # codes, transposed ones, and the values that are returned
        each += 4
    return {"bytes": n * each, "flops": 16 * n}


# --------------------------------------------------------------------------
# the same in 64 bits

def _exact_blocks(x, dtype, rows):
    """What x (R, C) stands for after rounding with a scale for 128 columns of `rows`
    rows."""
    R, C = x.shape
    p = torch.zeros(_pad(R, rows), _pad(C, BLOCK), dtype=torch.float64, device=x.device)
    p[:R, :C] = x
    t = p.view(p.shape[0] // rows, rows, -1, BLOCK)
    top = t.abs().amax((1, 3), keepdim=True)
    k = torch.ceil(torch.log2(top / FMT_MAX[dtype]))
    k = torch.where(top > 0, k, 0.0).clamp(-126, 127)
    # (log2 is off by an ulp at most: a power that is one off shows in the quotient)
    k = torch.where(top * torch.exp2(-k) > FMT_MAX[dtype], k + 1, k)
    k = torch.where((top > 0) & (top * torch.exp2(1 - k) <= FMT_MAX[dtype]), k - 1, k)
    k = k.clamp(-126, 127)
    a = t * torch.exp2(-k)
    bits, low = (3, -6) if dtype == "e4m3" else (2, -14)
    unit = torch.exp2((torch.frexp(a)[1] - 1).clamp(min=low).double() - bits)
    a = (torch.round(a / unit) * unit).clamp(-FMT_MAX[dtype], FMT_MAX[dtype])
    return (a * torch.exp2(k)).reshape(p.shape)[:R, :C]


def _exact_states(m, v, seed):
    """m and v (n,) after rounding to 8 bits, in 64 bits."""
    rm, rv = (r.double() * 2.0 ** -20 for r in _random(m.numel(), seed, m.device))
    a = m.abs().view(-1, BLOCK)
    top = a.amax(1, keepdim=True)
    f, x = torch.frexp(top)  # top = f 2^x, f in [1/2, 1): the largest code is 0.875 2^9
    k = (x - 9 + (f > 0.875).int()).clamp(-126, 127).double()
    a = (a * torch.exp2(-k)).flatten()
    unit = torch.exp2((torch.frexp(a)[1] - 1).clamp(min=-6).double() - 3)
    a = (torch.floor(a / unit + rm) * unit).view(-1, BLOCK) * torch.exp2(k)
    mq = a.flatten().copysign(m)
    top = v.view(-1, BLOCK).amax(1, keepdim=True)
    f, x = torch.frexp(top)  # the largest code is 0.9375 2^(e - 126)
    e = (x + 126 + (f > 0.9375).int()).clamp(40, 254).double()
    least = torch.exp2(e - 158) * 1.125
    unit = torch.exp2(torch.frexp(v)[1].double() - 4)
    q = (torch.floor(v / unit + rv) * unit).view(-1, BLOCK)
    q = torch.where(v.view(-1, BLOCK) < least, least, q)
    return mq, torch.where(v > 0, q.flatten(), 0.0)


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] in ("step", "blocks"):
        return _exact_step(case, s)
    x = s["x"].to(f64)
    if case["op"] in ("norm", "serve"):
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        dev = torch.sqrt(var + EPS)
        n = (x - mean) / dev
        y = torch.addcmul(s["beta"].to(f64), n, s["gamma"].to(f64))
    if case["op"] == "norm":
        g = s["g"].to(f64)
        h = g * s["gamma"].to(f64)
        d = case["width"]
        gx = (h - (h.sum(1, keepdim=True) + n * torch.linalg.vecdot(h, n).unsqueeze(1)) / d) / dev
        return {"out": y, "grad_input": gx, "grad_weight": torch.linalg.vecdot(g, n, dim=0),
                "grad_bias": g.sum(0)}
    w, d = s["w"], case["width"]
    scale = torch.exp2(w["e"][:, :-(-d // BLOCK)].to(f64) - 127)
    scale = torch.repeat_interleave(torch.repeat_interleave(scale, BLOCK, 0), BLOCK, 1)
    wd = w["q"].float().to(f64)[:, :d] * scale[:case["outs"], :d]
    xq = _exact_blocks(y if case["op"] == "serve" else x, "e4m3", 1)
    out = torch.addmm(s["bias"].to(f64), xq, wd.t().contiguous())
    if case["op"] == "serve" or not case["train"]:
        return {"out": out}
    g = s["g"].to(f64)
    gx = torch.mm(_exact_blocks(g, case["gdtype"], 1), wd)
    gt = _exact_blocks(g.t(), case["gdtype"], 1)
    xt = _exact_blocks(x.t(), "e4m3", 1)
    return {"out": out, "grad_input": gx, "grad_weight": torch.mm(gt, xt.t().contiguous()),
            "grad_bias": g.sum(0)}


def _exact_step(case, s):
    f64 = torch.float64
    (b1, b2), t = ADAM["betas"], s["t"]
    if case["bits"] == 8:
        c = s["s"]
        m = c["m"].float().to(f64) * torch.exp2(c["me"].to(f64) - 127).repeat_interleave(BLOCK)
        code = c["v"].to(f64)
        v = torch.exp2(torch.floor(code / 8) - 31) * (1 + torch.remainder(code, 8) / 8)
        v = v * torch.exp2(c["ve"].to(f64) - 127).repeat_interleave(BLOCK)
        v = torch.where(code > 0, v, 0.0)
    else:
        m, v = s["m"].to(f64), s["v"].to(f64)
    g = s["g"].to(f64)
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g.square(), v, b2)
    w = s["w"].to(f64)
    w = torch.addcdiv(w, m, (v / (1 - b2 ** t)).sqrt() + ADAM["epsilon"],
                      value=-ADAM["lr"] / (1 - b1 ** t))
    w = w * (1 - ADAM["lr"] * ADAM["weight_decay"])
    out = {"w": w}
    out["m"], out["v"] = _exact_states(m, v, t) if case["bits"] == 8 else (m, v)
    if case["op"] == "blocks":
        out["q"] = [_exact_blocks(x, "e4m3", BLOCK) for x in _matrices(case, w)]
        out["qt"] = None  # (codes without their scales)
    return out
