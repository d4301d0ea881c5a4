"""The token model's operators as timed cases: the embedding lookup and its
gradient, the vocabulary loss (linear_cross_entropy) and its gradients, and the
clipping of many gradients by their global norm.

A case is one call, or one forward and backward, as a program that trains or
serves a token model on quantized tables makes it.  ``run`` computes it in
plain fp32 torch operations, or with ``own`` set through ``novann_amd``.
``exact`` restates every case in 64 bits from the same seeded inputs.
"""
import itertools
import math

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BITS = {"f32": 32, "bf16": 16, "f16": 16, "e4m3": 8, "e5m2": 8, "e2m1": 4}
FMT_MAX = {"e4m3": 448.0, "e5m2": 57344.0, "e2m1": 6.0}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
IGNORE = -100      # the target of a position that has no loss
MAX_NORM = 1.0
CLIP_EPS = 1e-6


# --------------------------------------------------------------------------
# the cases

def listed():
    return [
        # one decoding step of one request: a single row of a wide FP8 table
        embed("embed 1 token", 1, 4096, 131072, "e4m3", "bf16", False),
        # a short ragged batch on a table of odd height, in float16 training
        embed("embed train 1000x784 of 30001", 1000, 784, 30001, "e5m2", "f16", True),
        # a training batch: 32768 tokens, the frequent ones many times over
        embed("embed train 32768x1024 of 50000", 32768, 1024, 50000, "e4m3", "bf16", True),
        # scoring one token against a large vocabulary
        loss("loss 1x4096x131072", 1, 4096, 131072, "e4m3", "bf16", False),
        # scoring a small ragged batch against an FP4 table
        loss("loss 37x1024x50000 fp4", 37, 1024, 50000, "e2m1", "f16", False),
        # a fine-tuning micro-batch of a small model
        loss("loss train 64x512x10000", 64, 512, 10000, "e4m3", "bf16", True),
        # the ragged batch of the second embedding case, its loss in training
        loss("loss train 1000x784x30001", 1000, 784, 30001, "e5m2", "f16", True),
        # a quarter of the third embedding case's batch, its loss in training
        loss("loss train 8192x1024x50000", 8192, 1024, 50000, "e4m3", "bf16", True),
        # a wide model with an unquantized table: the largest products
        loss("loss train 4096x4096x131072", 4096, 4096, 131072, "bf16", "bf16", True),
        # clipping a small model's gradients, where the calls' latency counts
        clip("clip small", 2, 128, 1000, "f32", "f32"),
        # a model of odd widths, float16 gradients clipped as they are stored
        clip("clip ragged", 12, 500, 30001, "f16", "f16"),
        # a model of 24 blocks: bf16 gradients, clipped ones in fp32 for the
        # optimizer
        clip("clip 24 blocks", 24, 1024, 50000, "bf16", "f32"),
    ]


def embed(name, tokens, width, vocab, w, x, train):
    return {"name": name, "op": "embed", "tokens": tokens, "width": width, "vocab": vocab,
            "wdtype": w, "xdtype": x, "train": train}


def loss(name, rows, width, vocab, w, x, train):
    return {"name": name, "op": "loss", "rows": rows, "width": width, "vocab": vocab,
            "wdtype": w, "xdtype": x, "train": train}


def clip(name, blocks, width, vocab, g, out):
    return {"name": name, "op": "clip", "blocks": blocks, "width": width, "vocab": vocab,
            "gdtype": g, "odtype": out}


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm (3 * 256 and
    3 * 1024 apart: no model here has them)."""
    v = min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))
    return v - 1 if v in (768, 3072) else v


def _width(rng, lo, hi):
    """A width or vocabulary: whole multiples of 16, 64 or 256, or (one in
    four) any number; the same two apart."""
    v = _log(rng, lo, hi)
    step = rng.choice([1, 16, 64, 256])
    v = v if v < 2 * step else v // step * step
    return v - 16 if v in (768, 3072) else v


def draw(rng):
    kind = rng.choice(["embed", "embed train", "loss", "loss train", "loss train", "clip"])
    width = _width(rng, 64, 4096)
    vocab = _width(rng, 1000, 131072)
    w = rng.choice(["e4m3", "e5m2", "e2m1", "bf16"])
    x = rng.choice(["bf16", "f16"])
    if w == "bf16":
        x = "bf16"
    if kind in ("embed", "embed train"):
        x = rng.choice(["f32", "bf16", "f16"])
        c = embed("", _log(rng, 1, 65536), width, vocab, w, x, kind == "embed train")
    elif kind == "loss":  # scoring: one row to a few hundred
        c = loss("", _log(rng, 1, 512), width, vocab, w, x, False)
    elif kind == "loss train":
        most = 4096 * 4096 * 131072 // (width * vocab)
        c = loss("", min(most, _log(rng, 16, 8192)), width, vocab, w, x, True)
    else:
        g, o = rng.choice([("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
        width = _width(rng, 64, 1024)
        c = clip("", _log(rng, 1, 24), width, _width(rng, 1000, 50000), g, o)
    c.pop("name", None)
    return c


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

    def tokens(self, n, vocab):
        """Token ids whose frequency falls with the id, as a vocabulary sorted
        by use has them: id + 1 is spread over its logarithm."""
        u = self.uniform(n).double()
        return ((u * math.log(vocab)).exp().long() - 1).clamp_(0, vocab - 1)

    def table(self, rows, cols, dtype, std):
        """{"codes", "scale", "dtype", "shape"}: a table of N(0, std) weights as
        stored, FP8 / FP4 with one scale for the tensor (E2M1: two a byte, the
        even column in the low nibble, odd widths with a zero column more)."""
        w = self.normal(rows, cols) * std
        t = {"dtype": dtype, "shape": (rows, cols), "scale": None}
        if dtype in TORCH:
            t["codes"] = w.to(TORCH[dtype])
            return t
        s = (w.abs().amax() / FMT_MAX[dtype]).reshape(1)
        w.div_(s)
        t["scale"] = s
        if dtype == "e2m1":
            w = torch.nn.functional.pad(w, (0, cols % 2))
            a = w.abs()
            mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
            code = sum((a > m).to(torch.uint8) for m in mids) + (w < 0).to(torch.uint8) * 8
            t["codes"] = (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous().reshape(-1)
        else:
            f8 = torch.float8_e4m3fn if dtype == "e4m3" else torch.float8_e5m2
            t["codes"] = w.clamp_(-FMT_MAX[dtype], FMT_MAX[dtype]).to(f8).reshape(-1)
        return t


def _decoded(t, dtype):
    """The table's values before the scale, in dtype."""
    rows, cols = t["shape"]
    if t["dtype"] == "e2m1":
        lut = torch.tensor(E2M1 + [-v for v in E2M1], dtype=dtype, device=t["codes"].device)
        c = t["codes"].view(rows, -1)
        return torch.stack((lut[(c & 15).int()], lut[(c >> 4).int()]), 2).view(rows, -1)[:, :cols]
    return t["codes"].view(rows, cols).to(torch.float32).to(dtype)


def _dense(t, dtype):
    v = _decoded(t, dtype)
    return v if t["scale"] is None else v * t["scale"].to(dtype)


def _clip_shapes(case):
    """The parameters of a model of that many blocks: per block two scale
    vectors, an attention's four matrices and a feed-forward's two, then the
    table and a last scale vector."""
    d = case["width"]
    block = [(d,), (d, d), (d, d), (d, d), (d, d), (d,), (4 * d, d), (d, 4 * d)]
    return block * case["blocks"] + [(case["vocab"], d), (d,)]


def _flat(shapes, dtype, dev):
    """One zeroed buffer for all tensors, each on a 16-byte boundary (as buckets
    of gradients are kept), and the tensors as its views."""
    sizes = [math.prod(s) for s in shapes]
    per = 16 // (BITS[dtype] // 8)
    starts = list(itertools.accumulate((-(-n // per) * per for n in sizes), initial=0))
    buf = torch.zeros(starts[-1], dtype=TORCH[dtype], device=dev)
    return buf, [buf[a:a + n].view(s) for a, n, s in zip(starts, sizes, shapes)]


def prepare(case, seed):
    make = Inputs(seed)
    s = {"case": case}
    if case["op"] == "embed":
        # rows of unit norm, brought to a deviation of one by the factor
        s["factor"] = math.sqrt(case["width"])
        s["table"] = make.table(case["vocab"], case["width"], case["wdtype"],
                                1 / math.sqrt(case["width"]))
        s["tokens"] = make.tokens(case["tokens"], case["vocab"])
        if case["train"]:
            s["grad"] = (make.normal(case["tokens"], case["width"]) / 64).to(TORCH[case["xdtype"]])
    elif case["op"] == "loss":
        n, d, v = case["rows"], case["width"], case["vocab"]
        s["table"] = make.table(v, d, case["wdtype"], 1.5 / math.sqrt(d))
        s["targets"] = make.tokens(n, v)
        # hidden states of a model under training: noise, and the target's
        # direction with a strength that differs by position
        rows = s["table"]["codes"].view(v, -1)[s["targets"]].reshape(-1)
        row = _dense({**s["table"], "codes": rows, "shape": (n, d)}, torch.float32)
        s["x"] = (make.normal(n, d) + 4 * make.uniform(n, 1) * row).to(TORCH[case["xdtype"]])
        s["targets"][make.uniform(n) < 0.06] = IGNORE
        if n == 1:
            s["targets"].clamp_(min=0)
    else:
        shapes = _clip_shapes(case)
        s["gflat"], s["grads"] = _flat(shapes, case["gdtype"], make.dev)
        for t in s["grads"]:
            t.copy_(make.normal(*t.shape) * (3e-2 / math.sqrt(t.shape[-1])))
        s["oflat"], s["outs"] = _flat(shapes, case["odtype"], make.dev)
    return s


# --------------------------------------------------------------------------
# one pass

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from novann_amd import functional as F
    from novann_amd import optim
    case = s["case"]
    if case["op"] == "clip":
        norm = optim.clip_grad_norm(s["grads"], MAX_NORM, eps=CLIP_EPS, out=s["outs"])
        return {"norm": norm, "grads": s["oflat"]}
    w = _weight(s["table"])
    if case["op"] == "embed":
        out = {"out": F.embedding(s["tokens"], w, factor=s["factor"], out_dtype=case["xdtype"])}
        if case["train"]:
            out["grad_weight"] = F.embedding_backward(s["grad"], s["tokens"], w,
                                                      factor=s["factor"])
        return out
    if not case["train"]:
        return {"loss": F.linear_cross_entropy(s["x"], w, s["targets"], reduction="none")}
    value, lse = F.linear_cross_entropy(s["x"], w, s["targets"], extras=True)
    gx, gw = F.linear_cross_entropy_backward(s["x"], w, s["targets"], lse)
    return {"loss": value, "grad_input": gx, "grad_weight": gw}


def _weight(t):
    from novann_amd.module import Parameters, QuantizedParameters
    if t["scale"] is None:
        return Parameters(t["codes"])
    return QuantizedParameters(t["codes"], t["shape"], t["dtype"], t["scale"])


def _plain(s):
    case = s["case"]
    if case["op"] == "clip":
        norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
        coef = (MAX_NORM / (norm + CLIP_EPS)).clamp(max=1.0)
        s["oflat"].copy_(s["gflat"].float() * coef)
        return {"norm": norm, "grads": s["oflat"]}
    xdt = TORCH[case["xdtype"]]
    if case["op"] == "embed":
        t, tokens = s["table"], s["tokens"]
        rows = t["codes"].view(case["vocab"], -1)[tokens].reshape(-1)
        picked = _dense({**t, "codes": rows, "shape": (case["tokens"], case["width"])},
                        torch.float32)
        out = {"out": (picked * s["factor"]).to(xdt)}
        if case["train"]:
            g = torch.zeros(case["vocab"], case["width"], device=tokens.device)
            out["grad_weight"] = g.index_add_(0, tokens, s["grad"].float() * s["factor"])
        return out
    w, x, targets = _dense(s["table"], torch.float32), s["x"].float(), s["targets"]
    logits = x @ w.t()
    kept = targets != IGNORE
    at = targets.clamp(min=0).unsqueeze(1)
    top = logits.amax(1, keepdim=True)
    e = (logits - top).exp()
    total = e.sum(1, keepdim=True)
    each = torch.where(kept, (total.log() + top - logits.gather(1, at)).squeeze(1), 0.0)
    if not case["train"]:
        return {"loss": each}
    count = kept.sum()
    p = e / total
    p.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    p = p * (kept / count).unsqueeze(1)
    return {"loss": each.sum() / count, "grad_input": (p @ w).to(xdt),
            "grad_weight": (p.t() @ x).to(xdt)}


# --------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _clip_shapes(case))
        return {"bytes": n * (BITS[case["gdtype"]] + BITS[case["odtype"]]) / 8, "flops": 3 * n}
    d, v, wbits, xbytes = (case["width"], case["vocab"], BITS[case["wdtype"]],
                           BITS[case["xdtype"]] / 8)
    if case["op"] == "embed":
        n = case["tokens"]
        moved = 8 * n + min(n, v) * d * wbits / 8 + n * d * xbytes
        if case["train"]:
            moved += n * d * xbytes + 4 * v * d
        return {"bytes": moved, "flops": n * d * (3 if case["train"] else 1)}
    n = case["rows"]
    moved = n * d * xbytes + v * d * wbits / 8 + 8 * n + 4 * (1 if case["train"] else n)
    if case["train"]:
        moved += (n + v) * d * xbytes
    return {"bytes": moved, "flops": (6 if case["train"] else 2) * n * v * d}


# --------------------------------------------------------------------------
# the same in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "clip":
        g = s["gflat"].to(f64)  # the padding between the tensors is zero
        norm = torch.linalg.vector_norm(g)
        return {"norm": norm, "grads": g.mul_(min(1.0, MAX_NORM / (norm.item() + CLIP_EPS)))}
    t = s["table"]
    if case["op"] == "embed":
        n, d, v = case["tokens"], case["width"], case["vocab"]
        rows = t["codes"].view(v, -1).index_select(0, s["tokens"]).reshape(-1)
        out = {"out": _dense({**t, "codes": rows, "shape": (n, d)}, f64) * s["factor"]}
        if case["train"]:
            order = torch.argsort(s["tokens"], stable=True)
            ids, counts = torch.unique_consecutive(s["tokens"][order], return_counts=True)
            sums = torch.cumsum(s["grad"].to(f64)[order], 0)
            ends = sums[counts.cumsum(0) - 1]
            g = torch.zeros(v, d, dtype=f64, device=ids.device)
            g[ids] = torch.diff(ends, dim=0, prepend=torch.zeros_like(ends[:1])) * s["factor"]
            out["grad_weight"] = g
        return out
    w, x = _dense(t, f64), s["x"].to(f64)
    valid = (s["targets"] >= 0).nonzero().squeeze(1)
    hit = s["targets"][valid]
    logits = torch.mm(x, w.t().contiguous())
    lse = torch.logsumexp(logits, 1)
    each = torch.zeros_like(lse)
    each[valid] = lse[valid] - logits[valid, hit]
    if not case["train"]:
        return {"loss": each}
    p = torch.zeros_like(logits)
    p[valid] = torch.exp(logits[valid] - lse[valid].unsqueeze(1))
    del logits
    p[valid, hit] -= 1.0
    p /= max(1, valid.numel())
    return {"loss": each.sum() / valid.numel(), "grad_input": torch.mm(p, w),
            "grad_weight": torch.mm(p.t().contiguous(), x)}
