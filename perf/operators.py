"""Performance cases of the engine's 8-bit operators.

Each case is one call (or one short chain of calls) that a user of this
framework makes of them through `bbh.engine`: rows quantised with a scale each
and read back, norms with the residual's addition that write 8-bit rows, and
the Linear on 8-bit integers.  Where `own` is false, `run` computes the same
with elementary torch operations.

Kinds:
  quantize   launch_quantize_rows, then launch_dequantize_rows: what the codes
             and scales stand for
  rmsnorm    launch_rmsnorm_quantize (residual added, the sum and / or the fp16
             rows kept where asked), then the codes read back
  layernorm  launch_layernorm_quantize, the same
  linear     launch_matmul_i8: one Linear on 8-bit rows and weights
  ffn        a post-norm feed-forward block as it is served in 8 bits: residual
             LayerNorm, Linear + GELU, quantise, Linear
"""

import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bert-by-hand_amd")

RMS_EPS, LN_EPS = 1e-6, 1e-12


def _engine():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from bbh import engine

    return engine


def listed():
    return [
        # sentence embeddings of one corpus, stored in 8 bits
        {"name": "quantize_2000x384", "kind": "quantize", "rows": 2000, "dim": 384},
        # the GELU outputs of a large batch of long documents
        {"name": "quantize_65536x1536", "kind": "quantize", "rows": 65536, "dim": 1536},
        # one token of a pre-norm decoder
        {"name": "rmsnorm_1x4096", "kind": "rmsnorm", "rows": 1, "dim": 4096, "residual": True,
         "keep_sum": True, "keep_y": False},
        # a long prompt of the same
        {"name": "rmsnorm_16384x4096", "kind": "rmsnorm", "rows": 16384, "dim": 4096,
         "residual": True, "keep_sum": True, "keep_y": False},
        # the encoder's residual LayerNorm at a ragged number of rows; the next
        # residual needs the fp16 rows too
        {"name": "layernorm_2003x384", "kind": "layernorm", "rows": 2003, "dim": 384,
         "residual": True, "keep_sum": False, "keep_y": True},
        # the same over the largest batch, 256 x 512
        {"name": "layernorm_131072x384", "kind": "layernorm", "rows": 131072, "dim": 384,
         "residual": True, "keep_sum": False, "keep_y": True},
        # FFN1 + GELU of one short query
        {"name": "linear_16x1536x384", "kind": "linear", "rows": 16, "n": 1536, "k": 384,
         "bias": True, "gelu": True},
        # one token against a square weight: the weight's bytes count
        {"name": "linear_1x4096x4096", "kind": "linear", "rows": 1, "n": 4096, "k": 4096,
         "bias": False, "gelu": False},
        # 64 queries scored against an 8-bit index of sentence embeddings
        {"name": "linear_64x200003x384", "kind": "linear", "rows": 64, "n": 200003, "k": 384,
         "bias": False, "gelu": False},
        # odd sizes everywhere
        {"name": "linear_2003x1111x777", "kind": "linear", "rows": 2003, "n": 1111, "k": 777,
         "bias": True, "gelu": False},
        # a large Linear, bound by the matrix cores
        {"name": "linear_8192x8192x8192", "kind": "linear", "rows": 8192, "n": 8192, "k": 8192,
         "bias": True, "gelu": False},
        # the operators together: the encoder's feed-forward block at 64 x 128
        {"name": "ffn_8192x384x1536", "kind": "ffn", "rows": 8192, "dim": 384, "ffn": 1536},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _to16(rng, n, share):
    """n, or (for `share` of the calls) the multiple of 16 at or above it."""
    return (n + 15) // 16 * 16 if rng.random() < share else n


def draw(rng):
    kind = rng.choice(["quantize", "rmsnorm", "layernorm", "linear", "linear", "linear", "ffn"])
    if kind in ("quantize", "rmsnorm", "layernorm"):
        dim = _to16(rng, _log(rng, 32, 8192), 0.7)
        case = {"kind": kind, "rows": _log(rng, 1, min(131072, (1 << 26) // dim)), "dim": dim}
        if kind != "quantize":
            case["residual"] = rng.random() < 0.7
            case["keep_sum"] = case["residual"] and rng.random() < 0.5
            case["keep_y"] = rng.random() < 0.5
        return case
    if kind == "linear":
        k = _to16(rng, _log(rng, 32, 16384), 0.7)
        n = _to16(rng, _log(rng, 16, min(262144, (1 << 27) // k)), 0.5)
        rows = _log(rng, 1, max(1, min(65536, (1 << 26) // n, (1 << 37) // (n * k))))
        return {"kind": kind, "rows": rows, "n": n, "k": k, "bias": rng.random() < 0.6,
                "gelu": rng.random() < 0.3}
    dim = _to16(rng, _log(rng, 128, 2048), 0.8)
    ffn = _to16(rng, _log(rng, 2 * dim, 5 * dim), 0.8)
    return {"kind": kind, "rows": _log(rng, 1, min(65536, (1 << 36) // (dim * ffn))), "dim": dim,
            "ffn": ffn}


# ---- what a user's program holds ---------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, rows, dim):
    """fp16 activations: columns of different size, a few of them outliers."""
    x = torch.randn((rows, dim), device="cuda", generator=g)
    size = 0.5 + torch.rand((dim,), device="cuda", generator=g)
    size = torch.where(torch.rand((dim,), device="cuda", generator=g) < 0.01, 8 * size, size)
    return (x * size).half()


def _affine(g, dim):
    gamma = (0.6 + 0.8 * torch.rand((dim,), device="cuda", generator=g)).half()
    beta = (0.1 * torch.randn((dim,), device="cuda", generator=g)).half()
    return gamma, beta


def _codes(x):
    """8-bit codes and the scale of each row, as the operands arrive."""
    x = x.float()
    scale = x.abs().amax(1) / 127
    return (x / scale[:, None]).round().clamp(-127, 127).to(torch.int8), scale


def _weight(g, n, k):
    return _codes(torch.randn((n, k), device="cuda", generator=g) * 0.05)


def _bias(g, n):
    return (0.05 * torch.randn((n,), device="cuda", generator=g)).half()


def _inputs(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "quantize":
        return {"x": _rows(g, case["rows"], case["dim"])}
    if kind in ("rmsnorm", "layernorm"):
        d = {"x": _rows(g, case["rows"], case["dim"])}
        d["gamma"], d["beta"] = _affine(g, case["dim"])
        d["residual"] = _rows(g, case["rows"], case["dim"]) if case["residual"] else None
        return d
    if kind == "linear":
        d = {}
        d["a"], d["sa"] = _codes(_rows(g, case["rows"], case["k"]))
        d["b"], d["sb"] = _weight(g, case["n"], case["k"])
        d["bias"] = _bias(g, case["n"]) if case["bias"] else None
        return d
    rows, dim, ffn = case["rows"], case["dim"], case["ffn"]
    d = {"x": _rows(g, rows, dim), "residual": _rows(g, rows, dim)}
    d["gamma"], d["beta"] = _affine(g, dim)
    d["w1"], d["s1"] = _weight(g, ffn, dim)
    d["w2"], d["s2"] = _weight(g, dim, ffn)
    d["b1"], d["b2"] = _bias(g, ffn), _bias(g, dim)
    return d


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"], kind = case, case["kind"]
    half = lambda *s: torch.empty(s, dtype=torch.float16, device="cuda")  # noqa: E731
    code = lambda *s: torch.empty(s, dtype=torch.int8, device="cuda")  # noqa: E731
    scale = lambda n: torch.empty((n,), dtype=torch.float32, device="cuda")  # noqa: E731
    m = case["rows"]
    if kind == "linear":
        st["out"] = half(m, case["n"])
        return st
    d = case["dim"]
    st["q"], st["scale"] = code(m, d), scale(m)
    if kind == "ffn":
        st["y"], st["mid"], st["out"] = half(m, d), half(m, case["ffn"]), half(m, d)
        st["q2"], st["scale2"] = code(m, case["ffn"]), scale(m)
        return st
    st["values"] = half(m, d)
    st["sum"] = half(m, d) if case.get("keep_sum") else None
    st["y"] = half(m, d) if case.get("keep_y") else None
    return st


# ---- the plain form, in 32 bits ---------------------------------------------------

def _quantize32(v):
    """fp32 rows -> codes (held in fp32) and scales."""
    amax = v.abs().amax(1, keepdim=True)
    q = torch.where(amax > 0, (127 * v / amax).round(), 0.0)
    return q, amax / 127


def _norm32(x, residual, gamma, beta, eps):
    h = x.float() if residual is None else x.float() + residual.float()
    c = h if beta is None else h - h.mean(1, keepdim=True)
    v = c * torch.rsqrt((c * c).mean(1, keepdim=True) + eps) * gamma.float()
    return h, v if beta is None else v + beta.float()


def _linear32(a, sa, b, sb, bias, gelu):
    y = (a.float() @ b.float().t()) * (sa.reshape(-1, 1) * sb)
    if bias is not None:
        y = y + bias.float()
    return 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5)) if gelu else y


def _plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "linear":
        return {"out": _linear32(st["a"], st["sa"], st["b"], st["sb"], st["bias"],
                                 case["gelu"]).half()}
    if kind == "quantize":
        q, scale = _quantize32(st["x"].float())
        return {"values": (q * scale).half(), "scale": scale[:, 0]}
    if kind == "ffn":
        _, y = _norm32(st["x"], st["residual"], st["gamma"], st["beta"], LN_EPS)
        q, scale = _quantize32(y)
        mid = _linear32(q, scale, st["w1"], st["s1"], st["b1"], True).half().float()
        q, scale = _quantize32(mid)
        out = _linear32(q, scale, st["w2"], st["s2"], st["b2"], False)
        return {"y": y.half(), "out": out.half()}
    eps = RMS_EPS if kind == "rmsnorm" else LN_EPS
    h, y = _norm32(st["x"], st["residual"], st["gamma"],
                   st["beta"] if kind == "layernorm" else None, eps)
    q, scale = _quantize32(y)
    return {"values": (q * scale).half(), "scale": scale[:, 0],
            "sum": h.half() if case["keep_sum"] else None,
            "y": y.half() if case["keep_y"] else None}


# ---- the framework's calls -----------------------------------------------------------

def _own(st):
    e, case = _engine(), st["case"]
    kind, m = case["kind"], case["rows"]
    if kind == "linear":
        return {"out": e.launch_matmul_i8(st["a"], st["sa"], st["b"], st["sb"], st["out"], m,
                                          case["n"], case["k"], bias=st["bias"],
                                          gelu=case["gelu"])}
    d, q, scale = case["dim"], st["q"], st["scale"]
    if kind == "ffn":
        f = case["ffn"]
        e.launch_layernorm_quantize(st["x"], st["gamma"], st["beta"], q, scale, m, d, eps=LN_EPS,
                                    residual=st["residual"], y=st["y"])
        e.launch_matmul_i8(q, scale, st["w1"], st["s1"], st["mid"], m, f, d, bias=st["b1"],
                           gelu=True)
        e.launch_quantize_rows(st["mid"], st["q2"], st["scale2"], m, f)
        e.launch_matmul_i8(st["q2"], st["scale2"], st["w2"], st["s2"], st["out"], m, d, f,
                           bias=st["b2"])
        return {"y": st["y"], "out": st["out"]}
    if kind == "quantize":
        e.launch_quantize_rows(st["x"], q, scale, m, d)
        return {"values": e.launch_dequantize_rows(q, scale, st["values"], m, d), "scale": scale}
    if kind == "rmsnorm":
        e.launch_rmsnorm_quantize(st["x"], st["gamma"], q, scale, m, d, eps=RMS_EPS,
                                  residual=st["residual"], sum=st["sum"], y=st["y"])
    else:
        e.launch_layernorm_quantize(st["x"], st["gamma"], st["beta"], q, scale, m, d, eps=LN_EPS,
                                    residual=st["residual"], sum=st["sum"], y=st["y"])
    return {"values": e.launch_dequantize_rows(q, scale, st["values"], m, d), "scale": scale,
            "sum": st["sum"], "y": st["y"]}


def run(st):
    return _own(st) if own else _plain(st)


# ---- least work -----------------------------------------------------------------

def work(case):
    kind, m = case["kind"], case["rows"]
    if kind == "linear":
        n, k = case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + 2 * n * case["bias"] + 2 * m * n,
                "flops": 2 * m * n * k}
    d = case["dim"]
    if kind == "ffn":
        f = case["ffn"]
        # x, the residual, both weights, y and out
        return {"bytes": 8 * m * d + 2 * d * f + 6 * (d + f) + 4 * d, "flops": 4 * m * d * f}
    # read back: codes and scales read, values written
    b = 2 * m * d + m * d + 4 * m + (m * d + 4 * m + 2 * m * d)
    if kind != "quantize":
        b += 2 * m * d * (case["residual"] + case["keep_sum"] + case["keep_y"])
        b += 2 * d * (1 if kind == "rmsnorm" else 2)
    return {"bytes": b, "flops": (6 if kind == "quantize" else 14) * m * d}


# ---- the same in 64 bits ----------------------------------------------------------

def _quantize64(v):
    scale = v.abs().max(dim=-1).values / 127.0
    return torch.round(v / scale.unsqueeze(-1)), scale


def _linear64(q, sq, w, sw, bias, gelu):
    acc = torch.matmul(q.double(), w.double().t().contiguous())
    y = acc * sq.double().unsqueeze(-1) * sw.double().unsqueeze(0)
    if bias is not None:
        y = y + bias.double()
    return y * torch.special.ndtr(y) if gelu else y


def _norm64(d, kind, eps):
    h = d["x"].double()
    if d["residual"] is not None:
        h = h + d["residual"].double()
    g = d["gamma"].double()
    if kind == "rmsnorm":
        return h, h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * g
    var, mean = torch.var_mean(h, dim=-1, keepdim=True, correction=0)
    return h, (h - mean) / torch.sqrt(var + eps) * g + d["beta"].double()


def exact(case, seed):
    d, kind = _inputs(case, seed), case["kind"]
    if kind == "linear":
        return {"out": _linear64(d["a"], d["sa"], d["b"], d["sb"], d["bias"], case["gelu"])}
    if kind == "quantize":
        q, scale = _quantize64(d["x"].double())
        return {"values": q * scale.unsqueeze(-1), "scale": scale}
    if kind == "ffn":
        _, y = _norm64(d, "layernorm", LN_EPS)
        mid = _linear64(*_quantize64(y), d["w1"], d["s1"], d["b1"], True)
        return {"y": y, "out": _linear64(*_quantize64(mid), d["w2"], d["s2"], d["b2"], False)}
    h, y = _norm64(d, kind, RMS_EPS if kind == "rmsnorm" else LN_EPS)
    q, scale = _quantize64(y)
    return {"values": q * scale.unsqueeze(-1), "scale": scale,
            "sum": h if case["keep_sum"] else None, "y": y if case["keep_y"] else None}
