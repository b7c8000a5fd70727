"""Performance cases of the engine's rotary positions and of its attention for
models other than MiniLM.

Each case is one call (or one short chain of calls) that a user of this
framework makes of them through `bbh.engine`: heads rotated by their positions,
with or without an RMS norm of each head, keys and values put into a cache on the
way; and attention with shared key/value heads, capped scores, a bias by
distance, a window, a prefix, a key mask, documents packed end to end, and few
queries over a long cache.  Where `own` is false, `run` computes the same with
elementary torch operations.

Kinds:
  rope    launch_rope: queries and keys out of fused QKV rows
  attend  launch_attend
  block   launch_rope over fused QKV rows, then launch_attend
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bert-by-hand_amd")

EPS = 1e-6


def _engine():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from bbh import engine

    return engine


def _rope_case(rows, heads, kv_heads, dim, rot, interleaved=False, scaling="none", norm=False,
               cache=False, far=512):
    """`far`: positions run up to it; `cache`: keys and values go to rows of a cache."""
    return {"kind": "rope", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "interleaved": interleaved, "scaling": scaling, "norm": norm,
            "cache": cache, "far": far}


def _attend_case(layout, batch, q_len, k_len, heads, kv_heads, dim, left=-1, right=-1, cap=0.0,
                 bias="none", half=0, prefix=0, mask=False, lens=0):
    """`layout`: packed (documents end to end), padded (batch, length) or cache (a few
    queries of each sequence over its own keys); `lens`: seed of the lengths, 0: all
    as long as q_len / k_len; `prefix`: longest prefix that every query sees."""
    return {"kind": "attend", "layout": layout, "batch": batch, "q_len": q_len, "k_len": k_len,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "left": left, "right": right,
            "cap": cap, "bias": bias, "half": half, "prefix": prefix, "mask": mask, "lens": lens}


def listed():
    return [
        # one new token of each of 16 sequences, far into a long context: norms,
        # rotation, keys and values into the cache
        {"name": "rope_16_tokens_cached", **_rope_case(16, 32, 8, 128, 128, norm=True, cache=True,
                                                      scaling="bands", far=131072)},
        # the encoder's largest batch, 256 x 512 tokens of 12 heads, rotated only
        {"name": "rope_131072x24x32", **_rope_case(131072, 12, 12, 32, 32)},
        # a ragged number of tokens, half of each head in interleaved pairs
        {"name": "rope_20003x24x80", **_rope_case(20003, 16, 8, 80, 40, interleaved=True,
                                                  scaling="linear", far=4096)},
        # a long prompt with shared key/value heads, norms and rotation
        {"name": "rope_32768x40x128", **_rope_case(32768, 32, 8, 128, 128, norm=True,
                                                   scaling="ramp", far=32768)},
        # the smallest call: one token of one sequence over a short cache
        {"name": "attend_1_token_over_500", **_attend_case("cache", 1, 1, 500, 12, 12, 64,
                                                           right=0)},
        # one token of each of 64 sequences over caches of up to 8192 keys
        {"name": "attend_64_tokens_over_8192", **_attend_case("cache", 64, 1, 8192, 32, 8, 128,
                                                              right=0, lens=7)},
        # one sequence, a few drafted tokens over a very long cache, capped scores
        {"name": "attend_5_tokens_over_100003", **_attend_case("cache", 1, 5, 100003, 16, 4, 128,
                                                               right=0, cap=50.0)},
        # 2000 sentences packed end to end, bias by distance with a slope a head
        {"name": "attend_2000_documents_slopes", **_attend_case("packed", 2000, 160, 160, 12, 12,
                                                                64, bias="slopes", lens=3)},
        # odd lengths, padded: a learned bias by distance, a key mask with holes
        {"name": "attend_32x509_table_masked", **_attend_case("padded", 32, 509, 509, 12, 12, 64,
                                                              bias="table", half=128, mask=True)},
        # an instruction that every token sees, then a causal window, capped scores
        {"name": "attend_4x4096_prefix_window", **_attend_case("padded", 4, 4096, 4096, 16, 4, 256,
                                                               left=1023, right=0, cap=30.0,
                                                               prefix=200)},
        # a long prompt, causal
        {"name": "attend_8192_causal", **_attend_case("padded", 1, 8192, 8192, 32, 8, 128, right=0)},
        # the operators together: norms and rotation of fused QKV rows, then
        # bidirectional attention over a padded batch
        {"name": "block_64x512", "kind": "block", "batch": 64, "len": 512, "heads": 12,
         "kv_heads": 4, "dim": 64, "rot": 64, "interleaved": False, "scaling": "none",
         "left": 128, "right": 128, "far": 512},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _scaling(rng):
    return rng.choice(["none", "none", "linear", "base", "ramp", "bands"])


def _shape(rng):
    """(heads, kv_heads, dim)"""
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    kv = rng.choice([1, 2, 3, 4, 8, 12])
    group = rng.choice([g for g in (1, 1, 2, 3, 4, 7, 8) if kv * g <= 32])
    return kv * group, kv, dim


def draw(rng):
    heads, kv, dim = _shape(rng)
    kind = rng.choice(["rope", "rope", "attend", "attend", "attend", "attend", "block"])
    if kind == "rope":
        rows = _log(rng, 1, min(131072, 160000000 // (dim * (heads + 2 * kv))))
        rot = dim if rng.random() < 0.6 else max(2, dim // rng.choice([2, 4]) // 2 * 2)
        return _rope_case(rows, heads, kv, dim, rot, rng.random() < 0.4, _scaling(rng),
                          rng.random() < 0.5, rng.random() < 0.4, _log(rng, 64, 1000000))
    if kind == "block":
        n = _log(rng, 8, 2048)
        batch = _log(rng, 1, max(1, min(128, 60000 // n, (1 << 29) // (n * n * heads))))
        left = rng.choice([-1, 64, 300])
        return {"kind": "block", "batch": batch, "len": n, "heads": heads, "kv_heads": kv,
                "dim": dim, "rot": dim if rng.random() < 0.6 else dim // 2,
                "interleaved": rng.random() < 0.4, "scaling": _scaling(rng), "left": left,
                "right": left if rng.random() < 0.5 else 0, "far": _log(rng, 4096, 1000000)}
    layout = rng.choice(["packed", "padded", "cache"])
    cap = rng.choice([0.0, 0.0, 30.0, 50.0])
    bias = rng.choice(["none", "none", "slopes", "table"])
    half = _log(rng, 8, 512) if bias == "table" else 0
    left, right = rng.choice([(-1, -1), (-1, 0), (-1, 0), (64, 64), (500, 0)])
    lens = rng.randrange(1, 1000) if rng.random() < 0.7 else 0
    if layout == "cache":
        q_len = rng.choice([1, 1, 1, 2, 5, 16, 100])
        k_len = _log(rng, max(16, q_len), 131072)
        room = 500000000 // (k_len * kv * dim)
        batch = _log(rng, 1, max(1, min(128, room, (1 << 31) // (k_len * heads * q_len))))
        return _attend_case(layout, batch, q_len, k_len, heads, kv, dim, left, 0, cap, bias, half,
                            0, False, lens)
    n = _log(rng, 1, 6000)
    batch = _log(rng, 1, max(1, min(2000, 60000 // n, (1 << 30) // (n * n * heads))))
    mask = layout == "padded" and rng.random() < 0.5
    prefix = _log(rng, 1, n) if right == 0 and rng.random() < 0.4 else 0
    return _attend_case(layout, batch, n, n, heads, kv, dim, left, right, cap, bias, half, prefix,
                        mask, lens if layout == "packed" else 0)


# ---- what a user's program holds ---------------------------------------------

# long-context scalings of the frequencies: (factor, original context, low, high)
_SCALED = {"none": (1.0, 0.0, 0.0, 0.0), "linear": (4.0, 0.0, 0.0, 0.0),
           "base": (8.0, 0.0, 0.0, 0.0), "ramp": (8.0, 4096.0, 1.0, 32.0),
           "bands": (8.0, 8192.0, 1.0, 4.0)}
_BASE = 500000.0


def _magnitude(scaling):
    return 0.1 * math.log(_SCALED[scaling][0]) + 1.0 if scaling == "ramp" else 1.0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, device="cuda", generator=g).half()


def _lengths(case):
    """(queries, keys) of each sequence, from the case alone."""
    n, q, k = case["batch"], case["q_len"], case["k_len"]
    if not case["lens"]:
        return np.full(n, q), np.full(n, k)
    rng = np.random.default_rng(case["lens"])
    if case["layout"] == "cache":
        keys = np.exp(rng.uniform(np.log(max(q, k // 8, 1)), np.log(k + 0.999), n)).astype(np.int64)
        keys[0] = k
        return np.full(n, q), np.maximum(keys, q)
    keys = np.exp(rng.uniform(np.log(max(1, k // 20)), np.log(k + 0.999), n)).astype(np.int64)
    keys[0] = k
    return keys, keys


def _prefixes(case):
    return np.random.default_rng(11).integers(0, case["prefix"] + 1, case["batch"])


def _key_mask(case):
    """A padded batch's key mask: right padding and a few holes."""
    rng = np.random.default_rng(12)
    n, k = case["batch"], case["k_len"]
    valid = rng.integers((k + 3) // 4, k + 1, n)
    m = (np.arange(k) < valid[:, None]) & (rng.random((n, k)) > 0.05)
    return m.astype(np.int32)


def _starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def _rope_inputs(case, g, rows):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    st = {"qkv": _normal(g, rows, h + 2 * kv, d)}
    for name in ("q_gamma", "k_gamma"):
        st[name] = (0.5 + torch.rand((d,), device="cuda", generator=g)).half()
    st["positions"] = torch.randint(0, case["far"], (rows,), device="cuda", dtype=torch.int32,
                                    generator=g)
    return st


def _inputs(case, seed):
    g = _gen(seed)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rope":
        st = _rope_inputs(case, g, case["rows"])
        if case["cache"]:
            slots = 2 * case["rows"]
            st["k_cache"], st["v_cache"] = _normal(g, slots, kv, d), _normal(g, slots, kv, d)
            st["kv_rows"] = torch.randperm(slots, device="cuda", generator=g)[:case["rows"]]
        return st
    if case["kind"] == "block":
        return _rope_inputs(case, g, case["batch"] * case["len"])
    n, q, k = case["batch"], case["q_len"], case["k_len"]
    nq, nk = _lengths(case)
    st = {}
    if case["layout"] == "packed":
        total = int(nk.sum())
        # queries, keys and values of one fused projection
        qkv = _normal(g, total, h + 2 * kv, d)
        st["q"], st["k"], st["v"] = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
        st["offsets"] = torch.from_numpy(_starts(nk)).cuda()
    else:
        st["q"], st["k"], st["v"] = (_normal(g, n, m, heads, d)
                                     for m, heads in ((q, h), (k, kv), (k, kv)))
        if case["layout"] == "cache":
            st["k_lengths"] = torch.from_numpy(nk.astype(np.int32)).cuda()
    if case["mask"]:
        st["mask"] = torch.from_numpy(_key_mask(case)).cuda()
    if case["prefix"]:
        st["prefix"] = torch.from_numpy(_prefixes(case).astype(np.int32)).cuda()
    if case["bias"] == "slopes":
        st["slopes"] = torch.from_numpy((2.0 ** (-8.0 * np.arange(1, h + 1) / h)).astype(np.float32)).cuda()
    elif case["bias"] == "table":
        st["table"] = torch.randn((h, 2 * case["half"] + 1), device="cuda", generator=g)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"], kind = case, case["kind"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if kind == "attend":
        st["out"] = torch.empty(st["q"].shape, dtype=torch.float16, device="cuda")
        # scratch of the framework's call for few queries over many keys, kept between calls
        st["scratch"] = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
        return st
    rows = st["qkv"].shape[0]
    st["q_out"] = torch.empty((rows, h, d), dtype=torch.float16, device="cuda")
    st["k_out"] = torch.empty((rows, kv, d), dtype=torch.float16, device="cuda")
    if kind == "block":
        st["out"] = torch.empty((rows, h, d), dtype=torch.float16, device="cuda")
    st["rope"] = None
    if own:
        factor, original, low, high = _SCALED[case["scaling"]]
        st["rope"] = _engine().Rope(
            case["rot"], base=_BASE, interleaved=case["interleaved"], scaling=case["scaling"],
            factor=factor, original=original, low=low, high=high,
            magnitude=_magnitude(case["scaling"]))
    return st


# ---- the plain form, in 32 bits (angles in 64) -----------------------------------

def _frequencies(case):
    """Radians a position of each pair, float64."""
    rot = case["rot"]
    factor, original, low, high = _SCALED[case["scaling"]]
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    base = _BASE
    if case["scaling"] == "base" and rot > 2:
        base = _BASE * factor ** (rot / (rot - 2))
    f = base ** (-2 * i / rot)
    if case["scaling"] == "linear":
        return f / factor
    if case["scaling"] == "ramp":
        # between the pairs that turn `high` and `low` times over the original context
        at = [rot * math.log(original / (2 * math.pi * t)) / (2 * math.log(base)) for t in (high, low)]
        first = min(max(math.floor(at[0]), 0), rot - 1)
        last = min(max(math.ceil(at[1]), 0), rot - 1)
        share = ((i - first) / max(last - first, 1e-3)).clamp(0, 1)
        return f * (1 - share) + f / factor * share
    if case["scaling"] == "bands":
        keep = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep)
    return f


def _rotate32(x, positions, case, gamma):
    """(rows, heads, dim) -> the same, normed where gamma is given, rotated."""
    x = x.float()
    if gamma is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma.float()
    angle = positions.double()[:, None] * _frequencies(case)
    m = _magnitude(case["scaling"])
    cos, sin = (m * angle.cos()).float()[:, None], (m * angle.sin()).float()[:, None]
    rot = case["rot"]
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rot:]), -1).half()


def _attend32(q, k, v, case, nq, nk, left, right, cap=0.0, mask=None, prefix=None, slopes=None,
              table=None):
    """q (batch, queries, heads, dim), k and v (batch, keys, kv_heads, dim); nq, nk
    (batch): how many of them count."""
    b, lq, h, d = q.shape
    lk, kv = k.shape[1:3]
    qf = q.float().reshape(b, lq, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    s = torch.matmul(qf, k.float().permute(0, 2, 3, 1).contiguous()) * d ** -0.5
    s = s.view(b, h, lq, lk)
    if cap:
        s = torch.tanh(s / cap) * cap
    j = torch.arange(lk, device=q.device)
    distance = j - (torch.arange(lq, device=q.device)[:, None] + (nk - nq)[:, None, None])
    seen = distance > -1 - lk - lq
    if left >= 0:
        seen = seen & (distance >= -left)
    if right >= 0:
        seen = seen & (distance <= right)
    if prefix is not None:
        seen = seen | (j < prefix[:, None, None])
    seen = seen & (j < nk[:, None, None])
    if mask is not None:
        seen = seen & (mask[:, None] != 0)
    if slopes is not None:
        s = s - slopes[:, None, None] * distance.abs()[:, None].float()
    if table is not None:
        half = table.shape[1] // 2
        s = s + table[:, distance.clamp(-half, half) + half].transpose(0, 1)
    s = s.masked_fill(~seen[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p.view(b, kv, -1, lk), v.float().transpose(1, 2).contiguous())
    return o.view(b, h, lq, d).transpose(1, 2).half()


def _plain(st):
    case = st["case"]
    h, kv = case["heads"], case["kv_heads"]
    if case["kind"] == "attend":
        extra = {n: st.get(n) for n in ("mask", "prefix", "slopes", "table")}
        args = (case, case["left"], case["right"], case["cap"])
        if case["layout"] != "packed":
            q, k = st["q"], st["k"]
            full = torch.full((q.shape[0],), k.shape[1], device="cuda")
            nq = torch.full((q.shape[0],), q.shape[1], device="cuda")
            nk = st["k_lengths"].long() if "k_lengths" in st else full
            return {"out": _attend32(q, k, st["v"], args[0], nq, nk, *args[1:], **extra)}
        # documents end to end -> padded, and back
        offsets = st["offsets"].long()
        n = offsets[1:] - offsets[:-1]
        i = torch.arange(case["q_len"], device="cuda")
        total = st["q"].shape[0]
        row = torch.where(i < n[:, None], offsets[:-1, None] + i, total)
        at = row.clamp(max=total - 1)
        o = _attend32(st["q"][at], st["k"][at], st["v"][at], args[0], n, n, *args[1:], **extra)
        out = torch.empty((total + 1,) + o.shape[2:], dtype=o.dtype, device="cuda")
        out[row.flatten()] = o.flatten(0, 1)
        return {"out": out[:total]}
    q, k, v = st["qkv"][:, :h], st["qkv"][:, h:h + kv], st["qkv"][:, h + kv:]
    norm = case["kind"] == "block" or case["norm"]
    q = _rotate32(q, st["positions"], case, st["q_gamma"] if norm else None)
    k = _rotate32(k, st["positions"], case, st["k_gamma"] if norm else None)
    if case["kind"] == "rope":
        if not case["cache"]:
            return {"q": q, "k": k}
        k_cache, v_cache = st["k_cache"], st["v_cache"]
        k_cache[st["kv_rows"]] = k
        v_cache[st["kv_rows"]] = v
        return {"q": q, "k_cache": k_cache, "v_cache": v_cache}
    b, n = case["batch"], case["len"]
    full = torch.full((b,), n, device="cuda")
    q, k, v = (t.unflatten(0, (b, n)) for t in (q, k, v))
    return {"out": _attend32(q, k, v, case, full, full, case["left"], case["right"]).flatten(0, 1)}


# ---- the framework's calls -----------------------------------------------------------

def _own(st):
    e, case = _engine(), st["case"]
    h, kv = case["heads"], case["kv_heads"]
    if case["kind"] == "attend":
        packed = case["layout"] == "packed"
        return {"out": e.launch_attend(
            st["q"], st["k"], st["v"], st["out"], q_len=case["q_len"], k_len=case["k_len"],
            q_offsets=st["offsets"] if packed else None,
            k_offsets=st["offsets"] if packed else None, k_lengths=st.get("k_lengths"),
            left=case["left"], right=case["right"], cap=case["cap"], mask=st.get("mask"),
            prefix=st.get("prefix"), slopes=st.get("slopes"), table=st.get("table"),
            scratch=st["scratch"])}
    qkv = st["qkv"]
    q, k, v = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
    norm = case["kind"] == "block" or case["norm"]
    gammas = {"q_gamma": st["q_gamma"], "k_gamma": st["k_gamma"], "eps": EPS} if norm else {}
    if case["kind"] == "rope" and case["cache"]:
        e.launch_rope(st["rope"], q, st["q_out"], k=k, k_out=st["k_cache"], v=v,
                      v_out=st["v_cache"], kv_rows=st["kv_rows"], positions=st["positions"],
                      **gammas)
        return {"q": st["q_out"], "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    e.launch_rope(st["rope"], q, st["q_out"], k=k, k_out=st["k_out"], positions=st["positions"],
                  **gammas)
    if case["kind"] == "rope":
        return {"q": st["q_out"], "k": st["k_out"]}
    b, n = case["batch"], case["len"]
    e.launch_attend(st["q_out"].unflatten(0, (b, n)), st["k_out"].unflatten(0, (b, n)),
                    v.unflatten(0, (b, n)), st["out"].unflatten(0, (b, n)), left=case["left"],
                    right=case["right"])
    return {"out": st["out"]}


def run(st):
    return _own(st) if own else _plain(st)


# ---- least work -----------------------------------------------------------------

def _seen(nq, nk, left, right, prefix, mask):
    """(pairs of a query and a key that it sees, keys that any query sees) of one sequence."""
    pos = np.arange(nq) + nk - nq
    lo = np.maximum(pos - left, 0) if left >= 0 else np.zeros(nq, np.int64)
    hi = np.minimum(pos + right + 1, nk) if right >= 0 else np.full(nq, nk)  # past the last
    hi = np.maximum(hi, lo)
    ones = np.ones(nk, np.int64) if mask is None else mask[:nk]
    upto = np.concatenate([[0], np.cumsum(ones)])
    p = min(prefix, nk)
    pairs = upto[hi] - upto[lo] + upto[np.minimum(lo, p)] + upto[p] - upto[np.minimum(hi, p)]
    any_ = max(int(upto[hi.max()] - upto[lo.min()]), 0) + int(upto[min(int(lo.min()), p)])
    return int(pairs.sum()), min(any_, nk)


def work(case):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rope":
        moved = h + kv * (2 if case["cache"] else 1)
        rows = case["rows"]
        return {"bytes": 4 * rows * moved * d + 4 * rows + 8 * rows * case["cache"],
                "flops": rows * (h + kv) * (3 * case["rot"] + 4 * d * case["norm"])}
    if case["kind"] == "block":
        b, n = case["batch"], case["len"]
        pairs = b * _seen(n, n, case["left"], case["right"], 0, None)[0]
        # the fused rows once, the heads' outputs once
        return {"bytes": 2 * b * n * d * (2 * h + 2 * kv) + 4 * b * n, "flops": 4 * d * h * pairs}
    nq, nk = _lengths(case)
    mask = _key_mask(case).astype(np.int64) if case["mask"] else None
    prefix = _prefixes(case) if case["prefix"] else np.zeros(case["batch"], np.int64)
    seen = [_seen(int(nq[b]), int(nk[b]), case["left"], case["right"], int(prefix[b]),
                  None if mask is None else mask[b]) for b in range(case["batch"])]
    pairs, keys = sum(s[0] for s in seen), sum(s[1] for s in seen)
    read = 2 * d * (2 * h * int(nq.sum()) + 2 * kv * keys)
    extra = 4 * case["batch"] * case["k_len"] * case["mask"]
    return {"bytes": read + extra, "flops": 4 * d * h * pairs}


# ---- the same in 64 bits ----------------------------------------------------------

def _turns64(case):
    """The frequencies by another route: turns over 2 pi positions, in numpy."""
    rot = case["rot"]
    factor, original, low, high = _SCALED[case["scaling"]]
    k = np.arange(0, rot, 2) / rot
    log_base = np.log(_BASE)
    if case["scaling"] == "base" and rot > 2:
        log_base = log_base + np.log(factor) * rot / (rot - 2)
    f = np.exp(-k * log_base)
    if case["scaling"] == "linear":
        f = np.exp(-k * log_base - np.log(factor))
    elif case["scaling"] == "ramp":
        def pair(turns):
            return rot / 2 * (np.log(original) - np.log(2 * np.pi * turns)) / log_base

        i0, i1 = np.clip(np.floor(pair(high)), 0, rot - 1), np.clip(np.ceil(pair(low)), 0, rot - 1)
        f = f * (1 + (1 / factor - 1) * np.clip((np.arange(rot // 2) - i0) / max(i1 - i0, 1e-3), 0, 1))
    elif case["scaling"] == "bands":
        wave = 2 * np.pi / f
        w = np.clip((original / wave - low) / (high - low), 0, 1)
        f = (1 - w) * f / factor + w * f
    return torch.from_numpy(f).cuda()


def _rotate64(x, positions, case, gamma):
    x = x.double()
    if gamma is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * gamma.double()
    rot = case["rot"]
    t = torch.polar(torch.full((1,), _magnitude(case["scaling"]), device="cuda", dtype=torch.float64),
                    positions.double().unsqueeze(1) * _turns64(case)).unsqueeze(1)
    part = x[..., :rot]
    if case["interleaved"]:
        z = torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous()) * t
        part = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(*part.unflatten(-1, (2, -1)).unbind(-2)) * t
        part = torch.cat((z.real, z.imag), -1)
    return torch.cat((part, x[..., rot:]), -1)


def _attend64(q, k, v, left, right, cap=0.0, mask=None, prefix=0, slopes=None, table=None):
    """One sequence: q (queries, heads, dim), k and v (keys, kv_heads, dim), a key/value
    head at a time."""
    nq, h, d = q.shape
    nk, kv = k.shape[:2]
    g = h // kv
    i = torch.arange(nk - nq, nk, device=q.device).unsqueeze(1)
    j = torch.arange(nk, device=q.device).unsqueeze(0)
    hidden = torch.zeros((nq, nk), dtype=torch.bool, device=q.device)
    if left >= 0:
        hidden |= i - j > left
    if right >= 0:
        hidden |= j - i > right
    hidden &= j >= prefix
    if mask is not None:
        hidden |= (mask[:nk] == 0).unsqueeze(0)
    out = torch.empty((nq, h, d), dtype=torch.float64, device=q.device)
    for c in range(kv):
        heads = slice(c * g, (c + 1) * g)
        s = torch.matmul(q[:, heads].double().transpose(0, 1), k[:, c].double().t().contiguous())
        s = s / math.sqrt(d)
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            s = s - slopes[heads].double().view(-1, 1, 1) * (i - j).abs()
        if table is not None:
            half = table.shape[1] // 2
            s = s + table[heads].double()[:, torch.clamp(j - i, -half, half) + half]
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        p = p.nan_to_num(0.0)  # rows that see nothing
        out[:, heads] = torch.matmul(p, v[:, c].double()).transpose(0, 1)
    return out


def exact(case, seed):
    st = _inputs(case, seed)
    h, kv = case["heads"], case["kv_heads"]
    if case["kind"] == "attend":
        nq, nk = _lengths(case)
        if h * float((nq * nk).sum()) * case["dim"] > 2e12 or case["batch"] * kv > 40000:
            return None
        rest = {n: st.get(n) for n in ("slopes", "table")}
        starts = _starts(nk)
        out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
        prefix = _prefixes(case) if case["prefix"] else np.zeros(case["batch"], np.int64)
        for b in range(case["batch"]):
            if case["layout"] == "packed":
                part = slice(int(starts[b]), int(starts[b + 1]))
                q, k, v, o = st["q"][part], st["k"][part], st["v"][part], out[part]
            else:
                n = int(nk[b])
                q, k, v, o = st["q"][b], st["k"][b, :n], st["v"][b, :n], out[b]
            o.copy_(_attend64(q, k, v, case["left"], case["right"], case["cap"],
                              st["mask"][b] if case["mask"] else None, int(prefix[b]), **rest))
        return {"out": out}
    q, k, v = st["qkv"].split((h, kv, kv), dim=1)
    norm = case["kind"] == "block" or case["norm"]
    q = _rotate64(q, st["positions"], case, st["q_gamma"] if norm else None)
    k = _rotate64(k, st["positions"], case, st["k_gamma"] if norm else None)
    if case["kind"] == "rope":
        if not case["cache"]:
            return {"q": q, "k": k}
        k_cache, v_cache = st["k_cache"].double(), st["v_cache"].double()
        k_cache[st["kv_rows"]] = k
        v_cache[st["kv_rows"]] = v.double()
        return {"q": q, "k_cache": k_cache, "v_cache": v_cache}
    b, n = case["batch"], case["len"]
    out = torch.stack([_attend64(*(t.unflatten(0, (b, n))[i] for t in (q, k, v)), case["left"],
                                 case["right"]) for i in range(b)])
    return {"out": out.flatten(0, 1)}
