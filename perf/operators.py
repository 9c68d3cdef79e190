"""The 8-bit layer operators and their plain forms, as cases that can be timed and compared.

Three operators and their run in a row: the root-mean-square norm with the residual's addition (floating output, or 8-bit
output with one scale per row), the quantisation of rows to 8 bits (time splicing included), and the 8-bit affine product with
a scale per row and per output channel.

`run` computes a case either in its plain form -- elementary torch operations in 32 bits -- or, with `own`, by the package's
calls (`kaldi_amd.int8`).  8-bit results come back as the values they stand for (code times scale, in bfloat16): that
conversion is part of the pass on both sides.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
#: the largest products and matrices that a drawn case may have: those of the largest listed ones
MOST_MACS = 16384 * 8192 * 8192
MOST_VALUES = 16384 * 8192


def listed():
    return [
        # one frame of a stream (or one token being answered) through a layer's norm: nothing but latency
        dict(name="norm one row bf16", op="norm", rows=1, dim=1536, type="bf16", residual=True),
        # a chunk of acoustic frames behind a ReLU, as NormalizeComponent sees them: 32-bit, no residual
        dict(name="norm frames f32", op="norm", rows=12000, dim=1536, type="f32", residual=False),
        # a long prompt or a large batch of a wide model, 16-bit residual stream
        dict(name="norm long bf16", op="norm", rows=16384, dim=8192, type="bf16", residual=True),
        # the same with the 8-bit output that the product reads, at a width no vector divides
        dict(name="norm to int8 odd f16", op="norm8", rows=2777, dim=2561, type="f16", residual=True),
        dict(name="norm to int8 bf16", op="norm8", rows=16384, dim=4096, type="bf16", residual=True),
        # the spliced input (-3, 0, 3) of a TDNN layer of width 768, one stream's chunk and a pass of many utterances
        dict(name="quantize chunk f32", op="quantize", rows=56, dim=768, type="f32", offsets="-3,0,3"),
        dict(name="quantize frames f32", op="quantize", rows=40000, dim=768, type="f32", offsets="-3,0,3"),
        # one token or frame against a square layer: the weights' bytes are what counts
        dict(name="affine one row bf16", op="affine", rows=1, in_dim=4096, out_dim=4096, type="bf16", relu=False),
        # a few streams' frames against the 6000-pdf output layer
        dict(name="affine 24 rows f32", op="affine", rows=24, in_dim=1536, out_dim=6000, type="f32", relu=False),
        # a minute of audio, odd sizes, the 2328-pdf output layer
        dict(name="affine odd f16", op="affine", rows=1999, in_dim=1537, out_dim=2328, type="f16", relu=True),
        # a large batch of a wide model: the matrix units are what counts
        dict(name="affine large bf16", op="affine", rows=16384, in_dim=8192, out_dim=8192, type="bf16", relu=False),
        # norm, 8-bit output and product as a model runs them, at an acoustic model's batch
        dict(name="layer frames bf16", op="layer", rows=12000, in_dim=1536, out_dim=1536, type="bf16", relu=True),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm8", "quantize", "affine", "affine", "affine", "layer"])
    if op in ("norm", "norm8"):
        dim = _spread(rng, 32, 16384)
        if rng.random() < 0.6:
            dim = max(32, dim // 32 * 32)
        return dict(op=op, rows=min(_spread(rng, 1, 32768), MOST_VALUES // dim), dim=dim, type=rng.choice(sorted(TYPES)), residual=rng.random() < 0.6)
    if op == "quantize":
        dim = _spread(rng, 32, 4096)
        if rng.random() < 0.6:
            dim = max(32, dim // 32 * 32)
        offsets = rng.choice(["0", "0", "-1,0,1", "-3,0", "-2,0,1", "0,3"])
        return dict(op=op, rows=min(_spread(rng, 8, 32768), MOST_VALUES // (dim * 3)), dim=dim, type=rng.choice(sorted(TYPES)), offsets=offsets)
    in_dim, out_dim = _spread(rng, 32, 8192), _spread(rng, 32, 8192)
    if rng.random() < 0.6:
        in_dim, out_dim = max(32, in_dim // 32 * 32), max(32, out_dim // 32 * 32)
    rows = min(_spread(rng, 1, 16384), MOST_MACS // (in_dim * out_dim))
    kinds = sorted(TYPES) if op == "affine" else ["bf16", "f16"]
    return dict(op=op, rows=rows, in_dim=in_dim, out_dim=out_dim, type=rng.choice(kinds), relu=rng.random() < 0.5)


def _offsets(case):
    return [int(o) for o in case["offsets"].split(",")]


def _activations(g, rows, dim, dtype):
    """Rows as a layer's output has them: each channel with a spread of its own, one in about 200 of them much wider."""
    x = torch.randn(rows, dim, generator=g, device="cuda")
    spread = torch.exp(0.5 * torch.randn(dim, generator=g, device="cuda"))
    wide = torch.rand(dim, generator=g, device="cuda") < 0.005
    return x.mul_(torch.where(wide, spread * 6.0, spread)).to(dtype)


def _codes(g, rows, cols, spread):
    return torch.randn(rows, cols, generator=g, device="cuda").mul_(spread).round_().clamp_(-127, 127).to(torch.int8)


def _pad16(q):
    """8-bit rows in memory as the product takes them: each begins on a multiple of 16 bytes."""
    buf = torch.zeros(q.shape[0], (q.shape[1] + 15) // 16 * 16, dtype=torch.int8, device=q.device)
    buf[:, :q.shape[1]] = q
    return buf[:, :q.shape[1]]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case=case, dtype=TYPES[case["type"]], hundred27=torch.full((1,), 127.0, device="cuda"))
    op = case["op"]
    if op in ("norm", "norm8"):
        s["x"] = _activations(g, case["rows"], case["dim"], s["dtype"])
        s["residual"] = (_activations(g, case["rows"], case["dim"], torch.float32) * 2.0).to(s["dtype"]) if case["residual"] else None
        s["gain"] = 1.0 + 0.2 * torch.randn(case["dim"], generator=g, device="cuda")
        return s
    if op == "quantize":
        s["x"] = _activations(g, case["rows"], case["dim"], s["dtype"]).clamp_min_(0)      # behind a ReLU
        return s
    rows, in_dim, out_dim = case["rows"], case["in_dim"], case["out_dim"]
    if op == "affine":
        s["q"] = _pad16(_codes(g, rows, in_dim, 30.0))
        s["scale"] = 0.02 + 0.02 * torch.rand(rows, generator=g, device="cuda")
    else:
        s["x"] = _activations(g, rows, in_dim, s["dtype"])
        s["residual"] = (_activations(g, rows, in_dim, torch.float32) * 2.0).to(s["dtype"])
        s["gain"] = 1.0 + 0.2 * torch.randn(in_dim, generator=g, device="cuda")
    s["w"] = _codes(g, out_dim, in_dim, 36.0)
    s["w_scale"] = (0.5 + torch.rand(out_dim, generator=g, device="cuda")) / (36.0 * math.sqrt(in_dim))
    s["bias"] = 0.1 * torch.randn(out_dim, generator=g, device="cuda")
    if own:
        from kaldi_amd import int8
        s["layer"] = int8.AffineInt8(s["w"], s["w_scale"], bias=s["bias"], relu=case["relu"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _sum_and_factor(s):
    """h = x + residual and 1 / sqrt(mean(h^2) + eps), in 32 bits"""
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    return h, torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)


def _to_int8(t, factor, hundred27):
    """codes and scales of rows t * factor: the positive factor cancels in the codes"""
    most = t.abs().amax(1, keepdim=True)
    codes = torch.round(t * torch.where(most > 0, hundred27 / most, most))
    return codes, (most * factor if factor is not None else most) / hundred27


def _affine(codes, scale, s):
    y = torch.matmul(codes, s["w"].float().t()) * scale * s["w_scale"] + s["bias"]
    return (y.clamp_min(0) if s["case"]["relu"] else y).to(s["dtype"])


def _splice(x, offsets):
    low, n = min(offsets), x.shape[0] - (max(offsets) - min(offsets))
    return torch.cat([x[o - low:o - low + n] for o in offsets], 1)


def _run_plain(s):
    op = s["case"]["op"]
    if op == "affine":
        return _affine(s["q"].float(), s["scale"][:, None], s)
    if op == "quantize":
        codes, scale = _to_int8(_splice(s["x"].float(), _offsets(s["case"])), None, s["hundred27"])
        return {"values": (codes * scale).bfloat16(), "scale": scale[:, 0]}
    h, factor = _sum_and_factor(s)
    out = {} if s["residual"] is None else {"sum": h.to(s["dtype"])}
    if op == "norm":
        return out | {"y": (h * factor * s["gain"]).to(s["dtype"])}
    codes, scale = _to_int8(h * s["gain"], factor, s["hundred27"])
    if op == "norm8":
        return out | {"values": (codes * scale).bfloat16(), "scale": scale[:, 0]}
    return out | {"y": _affine(codes, scale, s)}


# ---- the package's calls -----------------------------------------------------------------------------------------------

def _values(q, scale):
    return torch.mul(q, scale[:, None], out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device))


def _run_own(s):
    from kaldi_amd import int8
    op = s["case"]["op"]
    if op == "affine":
        return s["layer"].propagate(s["q"], s["scale"], dtype=s["dtype"])
    if op == "quantize":
        q, scale = int8.quantize_rows(s["x"], offsets=_offsets(s["case"]))
        return {"values": _values(q, scale), "scale": scale}
    if op == "norm":
        r = int8.rms_norm(s["x"], gain=s["gain"], eps=EPS, residual=s["residual"])
        return {"y": r} if s["residual"] is None else {"y": r[0], "sum": r[1]}
    r = int8.rms_norm_int8(s["x"], gain=s["gain"], eps=EPS, residual=s["residual"])
    out = {} if s["residual"] is None else {"sum": r[2]}
    if op == "norm8":
        return out | {"values": _values(r[0], r[1]), "scale": r[1]}
    return out | {"y": s["layer"].propagate(r[0], r[1], dtype=s["dtype"])}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without, and its definition in 64 bits ---------------------------------------------------------

def work(case):
    op, b = case["op"], BYTES[case["type"]]
    if op in ("norm", "norm8"):
        n = case["rows"] * case["dim"]
        out = n * b if op == "norm" else n + 4 * case["rows"]
        return {"bytes": n * b * (3 if case["residual"] else 1) + out + 4 * case["dim"], "flops": 5 * n}
    if op == "quantize":
        offsets = _offsets(case)
        rows = case["rows"] - (max(offsets) - min(offsets))
        n = rows * case["dim"] * len(offsets)
        return {"bytes": case["rows"] * case["dim"] * b + n + 4 * rows, "flops": 3 * n}
    rows, k, n = case["rows"], case["in_dim"], case["out_dim"]
    fixed = n * k + 8 * n + rows * n * b
    if op == "affine":
        return {"bytes": rows * k + 4 * rows + fixed, "flops": 2 * rows * n * k}
    return {"bytes": 3 * rows * k * b + 4 * k + fixed, "flops": 2 * rows * n * k + 5 * rows * k}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]

    def product(q, scale):
        y = (q @ s["w"].double().mT) * (scale * s["w_scale"].double()[None, :]) + s["bias"].double()[None, :]
        return torch.where(y > 0, y, torch.zeros_like(y)) if case["relu"] else y

    def codes(v):
        """nearest of the 255 codes of v / scale, scale = (largest magnitude of the row) / 127"""
        scale = torch.linalg.vector_norm(v, math.inf, dim=1, keepdim=True) / 127.0
        return torch.round(v / torch.where(scale > 0, scale, torch.ones_like(scale))), scale

    if op == "affine":
        return product(s["q"].double(), s["scale"].double()[:, None])
    if op == "quantize":
        offsets = _offsets(case)
        span = max(offsets) - min(offsets)
        at = torch.arange(case["rows"] - span, device="cuda")
        q, scale = codes(torch.stack([s["x"].double()[at + (o - min(offsets))] for o in offsets], 1).flatten(1))
        return {"values": q * scale, "scale": scale[:, 0]}
    h = s["x"].double()
    if s["residual"] is not None:
        h += s["residual"].double()
    y = h / torch.sqrt(torch.linalg.vecdot(h, h)[:, None] / h.shape[1] + EPS) * s["gain"].double()
    out = {} if s["residual"] is None else {"sum": h}
    if op == "norm":
        return out | {"y": y}
    q, scale = codes(y)
    return out | ({"values": q * scale, "scale": scale[:, 0]} if op == "norm8" else {"y": product(q, scale)})
