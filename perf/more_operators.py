"""Training operators in front of and inside an element network, as cases that can be timed and checked.

Three operators, each through the package's public entry points where ``own`` is true and as elementary torch
operations in FP32, rounded once at the end, where it is not:

  embed  rows of a table chosen by an id (the element of an atom, the pair of elements of an edge) and scaled: the rows
         alone, or with the table's gradient, the sum of the rows' gradients of each id.  An id outside the table
         (padding) gives a zero row and adds to no gradient.
  gnorm  group norm over samples [samples, positions, channels] (an atom's or an edge's channels: one position; the
         atoms of a cell: many), statistics over all positions and the channels of a group, then SiLU or nothing: the
         output alone, with its gradients, or with the gradients of its own input gradient (what a loss on forces asks)
  saved  activations that the backward pass takes from 8 bits: the codes and their values by themselves, group norm
         with its gradients, and per-expert linears with theirs

Row counts come from the repository's systems: 8,192 atoms (32 cells of 256), 131,072 atoms (the large MD system),
about 52 edges an atom at 5 A; widths from its channel counts and radial layers (64); 10 and 89 elements.

Activations in 8 bits.  A block is 128 consecutive elements of the last axis, the last block of a row what is left.
scale = max(max |x|, 2^-100) c with c = 1/127, code = x (1 / scale) rounded to the nearest whole number (ties to even)
and held to [-127, 127], value = code scale, rounded to the type of x; every step in FP32, so the codes are defined to
the last bit.  What the forward pass returns comes from x itself, what the backward pass takes of x from the values;
mean and deviation of the group norm are those of x.
"""
from __future__ import annotations

import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "ictc-o3-hp-k100_amd")

own = False

DEV = "cuda"
BLOCK = 128
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5


def _framework():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import ictc_o3
    return ictc_o3


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # a small molecule's atoms in training: launch latency and host time
        {"name": "embed_few", "kind": "embed", "rows": 5, "entries": 10, "width": 64, "dtype": "float32",
         "train": True},
        # the atoms of the large system, ten elements of 128 channels: a few entries that all rows share
        {"name": "embed_atoms", "kind": "embed", "rows": 131072, "entries": 10, "width": 128, "dtype": "float32",
         "train": True},
        # the edges of a training batch by their pair of elements (89 x 89), 64 channels
        {"name": "embed_pairs", "kind": "embed", "rows": 425991, "entries": 7921, "width": 64, "dtype": "bfloat16",
         "train": True},
        # a table with about as many entries as rows, wide, an odd width, common and rare entries
        {"name": "embed_vocabulary", "kind": "embed", "rows": 60013, "entries": 50021, "width": 1021,
         "dtype": "float16", "train": True},
        # three atoms through a hidden layer's norm: launch latency and host time
        {"name": "gnorm_few", "kind": "gnorm", "samples": 3, "positions": 1, "channels": 64, "groups": 8,
         "dtype": "float32", "activation": "silu", "mode": "train"},
        # the radial layers' hidden rows of a training batch: many short rows
        {"name": "gnorm_edges", "kind": "gnorm", "samples": 425991, "positions": 1, "channels": 64, "groups": 8,
         "dtype": "float32", "activation": "silu", "mode": "train"},
        # a batch of 32 cells of 256 atoms, normalised over each cell, under a loss on forces
        {"name": "gnorm_cells", "kind": "gnorm", "samples": 32, "positions": 256, "channels": 128, "groups": 16,
         "dtype": "float32", "activation": "silu", "mode": "second"},
        # sizes that no chunk and no tile divides
        {"name": "gnorm_odd", "kind": "gnorm", "samples": 7, "positions": 1999, "channels": 330, "groups": 11,
         "dtype": "float16", "activation": "none", "mode": "train"},
        # the large system as one sample
        {"name": "gnorm_large", "kind": "gnorm", "samples": 1, "positions": 131072, "channels": 256, "groups": 32,
         "dtype": "bfloat16", "activation": "silu", "mode": "train"},
        # wide rows of the large system to codes and back, as a caller's own function keeps them
        {"name": "saved_codes", "kind": "saved", "part": "codes", "rows": 131072, "width": 512, "dtype": "bfloat16"},
        # the radial layers' norm, its rows kept in 8 bits
        {"name": "saved_norm", "kind": "saved", "part": "norm", "rows": 425991, "width": 64, "groups": 8,
         "dtype": "float32"},
        # the large system's per-element layer, its rows kept in 8 bits
        {"name": "saved_linear", "kind": "saved", "part": "linear", "rows": 131072, "width": 512, "outputs": 512,
         "experts": 10, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case of the same ranges: sizes over their logarithm, odd ones among them."""
    kind = rng.choice(("embed", "gnorm", "saved"))
    dtype = rng.choice(("float32", "bfloat16", "float16"))
    if kind == "embed":
        width = rng.choice((_log(rng, 1, 2048), 64, 128))
        return {"kind": "embed", "rows": _log(rng, 1, min(425991, 61000000 // width)),
                "entries": _log(rng, 1, min(150000, 51000000 // width)), "width": width, "dtype": dtype,
                "train": rng.choice((True, True, False))}
    if kind == "gnorm":
        # (a group of one position has four channels at least: of two, the input gradient cancels to eps / var)
        one = rng.choice((True, False))
        per = rng.choice((4, 8, 16, 32, _log(rng, 4, 512)) if one else (1, 2, 4, 8, 16, _log(rng, 1, 512)))
        groups = _log(rng, 1, max(1, min(64, 4096 // per)))
        channels = per * groups
        most = 16777216 // channels
        positions = 1 if one else _log(rng, 4, most)
        samples = _log(rng, 1, min(425991, most // positions))
        return {"kind": "gnorm", "samples": samples, "positions": positions, "channels": channels, "groups": groups,
                "dtype": dtype, "activation": rng.choice(("silu", "silu", "none")),
                "mode": rng.choice(("infer", "train", "train", "second"))}
    part = rng.choice(("codes", "norm", "linear"))
    if part == "codes":
        width = rng.choice((_log(rng, 1, 8192), 64, 128, 512))
        return {"kind": "saved", "part": "codes", "rows": _log(rng, 1, min(425991, 67108864 // width)),
                "width": width, "dtype": dtype}
    if part == "norm":
        groups = _log(rng, 1, 32)
        width = groups * rng.choice((4, 8, 16, _log(rng, 4, 128)))
        return {"kind": "saved", "part": "norm", "rows": _log(rng, 1, min(425991, 27000000 // width)),
                "width": width, "groups": groups, "dtype": dtype}
    width = rng.choice((_log(rng, 16, 1024), 64, 128, 256))
    outputs = rng.choice((_log(rng, 16, 1024), 64, 128, 256))
    most = min(131072, 131072 * 256 * 256 // (width * outputs))
    return {"kind": "saved", "part": "linear", "rows": _log(rng, 1, most), "width": width, "outputs": outputs,
            "experts": _log(rng, 1, 96), "dtype": dtype}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    s["type"] = dtype = DTYPES[case["dtype"]]
    if case["kind"] == "embed":
        n, v, c = case["rows"], case["entries"], case["width"]
        # common and rare entries: shares fall as one over the rank, from the middle of the table
        place = torch.rand(n, device=DEV, generator=g, dtype=torch.float64)
        rank = (2.0 * (1.0 + v / 2.0) ** place - 2.0).long().clamp(max=v - 1)
        s["ids"] = (rank + v // 2) % v
        s["ids"][torch.rand(n, device=DEV, generator=g) < 0.01] = -1          # padding
        s["scale"] = math.sqrt(c)
        s["table"] = (_randn(g, v, c) / math.sqrt(c)).to(dtype).requires_grad_(case["train"])
        s["gy"] = _randn(g, n, c).to(dtype)
        return s
    if case["kind"] == "gnorm":
        n, p, c, groups = case["samples"], case["positions"], case["channels"], case["groups"]
    elif case["part"] == "norm":
        n, p, c, groups = case["rows"], 1, case["width"], case["groups"]
        s.update(samples=n, positions=1, channels=c, activation="silu", mode="train")
    else:
        n, p, c, groups = case["rows"], 1, case["width"], 1
    # samples of different size, channels of different mean
    x = (0.5 + _randn(g, n, 1, 1).exp()) * (_randn(g, n, p, c) + 0.3 * _randn(g, 1, 1, c))
    if case["kind"] == "saved" and case["part"] == "codes":
        s["x"] = x.view(n, c).to(dtype)
        return s
    if case["kind"] == "saved" and case["part"] == "linear":
        e, m = case["experts"], case["outputs"]
        share = 1.0 / (2.0 + torch.arange(e, device=DEV) / max(1.0, e / 4))
        s["ids"] = torch.multinomial(share, n, replacement=True, generator=g)
        s["counts"] = torch.bincount(s["ids"], minlength=e).tolist()
        s["x"] = _randn(g, n, c).to(dtype)
        s["w"] = (_randn(g, e, m, c) / math.sqrt(c)).to(dtype)
        s["b"] = (0.1 * _randn(g, e, m)).to(dtype)
        s["gy"] = _randn(g, n, m).to(dtype)
        for name in ("x", "w", "b"):
            s[name].requires_grad_()
        return s
    s["x"] = x.to(dtype) if case["kind"] == "gnorm" else x.view(n, c).to(dtype)
    s["w"] = (1.0 + 0.2 * _randn(g, c)).to(dtype)
    s["b"] = (0.2 * _randn(g, c)).to(dtype)
    s["gy"] = _randn(g, *s["x"].shape).to(dtype)
    second = s["mode"] == "second"
    s["v"] = _randn(g, *s["x"].shape).to(dtype) if second else None
    for name in ("x", "w", "b"):
        s[name].requires_grad_(s["mode"] != "infer")
    s["gy"].requires_grad_(second)
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------


def _plain_embed(s):
    table, ids, dtype = s["table"].detach(), s["ids"], s["type"]
    valid = (ids >= 0) & (ids < s["entries"])
    at = torch.where(valid, ids, torch.zeros_like(ids))
    keep = valid[:, None] * s["scale"]
    out = {"y": (table[at].float() * keep).to(dtype)}
    if s["train"]:
        grad = torch.zeros(table.shape, device=DEV)
        grad.index_add_(0, at, s["gy"].float() * keep)
        out["gtable"] = grad.to(dtype)
    return out


def _encode(x):
    """(codes as FP32 [rows, blocks, 128], scales [rows, blocks, 1]) of x [rows, width] in the definition's steps."""
    n, c = x.shape
    blocks = -(-c // BLOCK)
    f = x.detach().float()
    if blocks * BLOCK != c:
        f = torch.cat([f, f.new_zeros(n, blocks * BLOCK - c)], 1)
    f = f.view(n, blocks, BLOCK)
    scale = f.abs().amax(2, keepdim=True).clamp(min=2.0 ** -100) * (1.0 / 127.0)
    return torch.round(f * torch.reciprocal(scale)).clamp(-127, 127), scale


def _decode(codes, scale, like):
    return (codes * scale).view(codes.shape[0], -1)[:, :like.shape[1]].to(like.dtype)


def _grouped(t, s):
    return t.detach().float().view(s["samples"], s["positions"], s["groups"], -1)


def _mean(t):
    return t.mean((1, 3), keepdim=True)


def _plain_gnorm(s, saved=False):
    x, dtype = s["x"], s["type"]
    w, b = (s[name].detach().float().view(s["groups"], -1) for name in ("w", "b"))
    silu = s["activation"] == "silu"
    f = _grouped(x, s)
    mean = _mean(f)
    r = (_mean((f - mean).square()) + EPS).rsqrt()
    h = (f - mean) * r
    z = h * w + b
    out = {"y": (z / (1.0 + torch.exp(-z)) if silu else z).view(x.shape).to(dtype)}
    if s["mode"] == "infer":
        return out
    if saved:
        codes, scale = _encode(x)
        h = (_grouped(_decode(codes, scale, x), s) - mean) * r
        z = h * w + b
    g = _grouped(s["gy"], s)
    if silu:
        sg = 1.0 / (1.0 + torch.exp(-z))
        slope = sg * (1.0 + z * (1.0 - sg))
        ga = g * slope
    else:
        ga = g
    u = ga * w
    ua, uh = _mean(u), _mean(u * h)
    out["gx"] = (r * (u - ua - h * uh)).view(x.shape).to(dtype)
    if s["mode"] == "train":
        out["gw"], out["gb"] = (ga * h).sum((0, 1)).view(-1).to(dtype), ga.sum((0, 1)).view(-1).to(dtype)
        return out
    # gradients of <v, gx>
    v = _grouped(s["v"], s)
    va, vh = _mean(v), _mean(v * h)
    pv = r * (v - va - h * vh)
    q = _mean(u * v) - ua * va - uh * vh
    t = -r * (vh * u + uh * v)
    e = w * pv
    out["vw"] = (ga * pv).sum((0, 1))
    if silu:
        zz = e * g * (sg * (1.0 - sg) * (2.0 + z * (1.0 - 2.0 * sg)))
        t = t + zz * w
        out["vw"], out["vb"] = out["vw"] + (zz * h).sum((0, 1)), zz.sum((0, 1)).view(-1).to(dtype)
        e = e * slope
    out["vw"] = out["vw"].view(-1).to(dtype)
    out["vg"] = e.view(x.shape).to(dtype)
    out["vx"] = (r * (t - _mean(t) - h * _mean(t * h)) - r * r * q * h).view(x.shape).to(dtype)
    return out


def _plain_linear(s):
    dtype, counts = s["type"], s["counts"]
    ids, perm = torch.sort(s["ids"], stable=True)
    w, b = s["w"].detach().float(), s["b"].detach().float()
    codes, scale = _encode(s["x"])
    x = torch.split(s["x"].detach()[perm].float(), counts)
    value = torch.split(_decode(codes, scale, s["x"])[perm].float(), counts)
    g = torch.split(s["gy"][perm].float(), counts)

    def back(parts):
        rows = torch.cat(parts)
        out = torch.empty_like(rows)
        out[perm] = rows
        return out.to(dtype)

    return {"y": back([torch.mm(i, j.t()) + k for i, j, k in zip(x, w, b)]),
            "gx": back([torch.mm(i, j) for i, j in zip(g, w)]),
            "gw": torch.stack([torch.mm(i.t(), j) for i, j in zip(g, value)]).to(dtype),
            "gb": torch.stack([i.sum(0) for i in g]).to(dtype)}


def _plain_saved(s):
    if s["part"] == "norm":
        return _plain_gnorm(s, saved=True)
    if s["part"] == "linear":
        return _plain_linear(s)
    codes, scale = _encode(s["x"])
    return {"values": _decode(codes, scale, s["x"]), "scales": scale.view(s["rows"], -1)}


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------


def _own_embed(s):
    y = _framework().embedding(s["table"], s["ids"], s["scale"])
    if not s["train"]:
        return {"y": y}
    (grad,) = torch.autograd.grad(y, s["table"], s["gy"])
    return {"y": y, "gtable": grad}


def _own_gnorm(s, save_bits=None):
    activation = None if s["activation"] == "none" else s["activation"]
    y = _framework().group_norm(s["x"], s["groups"], s["w"], s["b"], eps=EPS, activation=activation,
                                save_bits=save_bits)
    if s["mode"] == "infer":
        return {"y": y}
    if s["mode"] == "train":
        gx, gw, gb = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["gy"])
        return {"y": y, "gx": gx, "gw": gw, "gb": gb}
    (gx,) = torch.autograd.grad(y, s["x"], s["gy"], create_graph=True)
    if activation is None:
        vx, vw, vg = torch.autograd.grad(gx, (s["x"], s["w"], s["gy"]), s["v"])
        return {"y": y, "gx": gx, "vw": vw, "vg": vg, "vx": vx}
    vx, vw, vb, vg = torch.autograd.grad(gx, (s["x"], s["w"], s["b"], s["gy"]), s["v"])
    return {"y": y, "gx": gx, "vw": vw, "vb": vb, "vg": vg, "vx": vx}


def _own_saved(s):
    o3 = _framework()
    if s["part"] == "norm":
        return _own_gnorm(s, save_bits=8)
    if s["part"] == "linear":
        y = o3.expert_linear(s["x"], s["w"], o3.expert_order(s["ids"], s["experts"]), s["b"], save_bits=8)
        gx, gw, gb = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["gy"])
        return {"y": y, "gx": gx, "gw": gw, "gb": gb}
    codes, scales = o3.encode_activations(s["x"])
    return {"values": o3.decode_activations(codes, scales, dtype=s["type"]), "scales": scales}


def run(state):
    return {("embed", False): _plain_embed, ("embed", True): _own_embed, ("gnorm", False): _plain_gnorm,
            ("gnorm", True): _own_gnorm, ("saved", False): _plain_saved, ("saved", True): _own_saved,
            }[state["kind"], own](state)


# ---------------------------------------------------------------------------
# Work and results in 64 bits
# ---------------------------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "embed":
        n, v, c = case["rows"], case["entries"], case["width"]
        moved, ops = n * c + min(n, v) * c, n * c
        if case["train"]:
            moved, ops = moved + n * c + v * c, 3 * ops
        return {"bytes": size * moved + 8 * n, "flops": ops}
    if case["kind"] == "gnorm":
        elements = case["samples"] * case["positions"] * case["channels"]
        # rows read and written: x, y; gy, gx; v, vx, vg
        rows, ops = {"infer": (2, 12), "train": (4, 35), "second": (7, 80)}[case["mode"]]
        return {"bytes": size * elements * rows, "flops": ops * elements}
    n, c = case["rows"], case["width"]
    codes = n * c + 4 * n * -(-c // BLOCK)                     # written once and read once
    if case["part"] == "codes":
        return {"bytes": 2 * size * n * c + 2 * codes, "flops": 5 * n * c}
    if case["part"] == "norm":
        return {"bytes": 4 * size * n * c + 2 * codes, "flops": 40 * n * c}
    m, e = case["outputs"], min(n, case["experts"])
    elements = 2 * n * c + 2 * n * m + e * m * (c + 1) + case["experts"] * m * (c + 1)
    return {"bytes": size * elements + 8 * n + 2 * codes, "flops": 6 * n * c * m}


def _values64(x):
    """What the 8-bit codes of x [rows, width] stand for, and the scales, each FP32 step as its 64-bit result rounded."""
    n, c = x.shape
    pad = -c % BLOCK
    f = torch.nn.functional.pad(x.detach().double(), (0, pad)).view(n, -1, BLOCK)
    third = torch.tensor(1.0 / 127.0, dtype=torch.float64).float().double().item()
    top = torch.maximum(f.max(2).values, -f.min(2).values)
    scale = (top.clamp_min(2.0 ** -100) * third).float()
    inverse = (1.0 / scale.double()).float().double()
    codes = (f * inverse[..., None]).float().round().clamp(-127, 127)
    value = (codes.double() * scale.double()[..., None]).float().view(n, -1)[:, :c]
    return value.to(x.dtype).double(), scale


def _exact_gnorm(s, saved=False):
    groups = s["groups"]

    def act(z):
        return z * torch.sigmoid(z) if s["activation"] == "silu" else z

    x, w, b, gy = (s[name].detach().double().requires_grad_() for name in ("x", "w", "b", "gy"))
    n, c = s["samples"], s["channels"]
    X = x.view(n, -1, groups, c // groups)
    var, mean = torch.var_mean(X, (1, 3), correction=0, keepdim=True)
    r = 1.0 / torch.sqrt(var + EPS)
    y = act(((X - mean) * r).reshape(n, -1, c) * w + b).reshape(x.shape)
    out = {"y": y.detach()}
    if saved:
        h = ((_values64(s["x"])[0].view(X.shape) - mean) * r).detach().requires_grad_()
        again = act(h.reshape(n, -1, c) * w + b).reshape(x.shape)
        gh, out["gw"], out["gb"] = torch.autograd.grad(again, (h, w, b), gy)
        flat, gflat = (t.detach().transpose(1, 2).reshape(n, groups, -1) for t in (h, gh))
        drop = gflat.mean(2)[:, None, :, None] + h.detach() * (flat * gflat).mean(2)[:, None, :, None]
        out["gx"] = ((gh - drop) * r.detach()).view(x.shape)
    elif s["mode"] == "train":
        out["gx"], out["gw"], out["gb"] = torch.autograd.grad(y, (x, w, b), gy)
    elif s["mode"] == "second":
        (gx,) = torch.autograd.grad(y, x, gy, create_graph=True)
        out["gx"] = gx.detach()
        names = ["vx", "vw", "vg"] + (["vb"] if s["activation"] == "silu" else [])
        wrt = [{"vx": x, "vw": w, "vg": gy, "vb": b}[i] for i in names]
        out.update(zip(names, torch.autograd.grad(gx, wrt, s["v"].double())))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "gnorm":
        return _exact_gnorm(s)
    if case["kind"] == "embed":
        ids, table = s["ids"], s["table"].detach().double()
        padded = torch.cat([table, table.new_zeros(1, table.shape[1])])      # (-1 is the zero row)
        out = {"y": padded[ids] * s["scale"]}
        if case["train"]:
            grad = torch.zeros_like(padded)
            grad.index_put_((ids,), s["gy"].double(), accumulate=True)
            out["gtable"] = grad[:-1] * s["scale"]
        return out
    if case["part"] == "norm":
        return _exact_gnorm(s, saved=True)
    values, scales = _values64(s["x"])
    if case["part"] == "codes":
        return {"values": values, "scales": scales.double()}
    x, w, b, gy = (s[name].detach().double() for name in ("x", "w", "b", "gy"))
    out = {"y": torch.empty_like(gy), "gx": torch.empty_like(x), "gw": torch.zeros_like(w), "gb": torch.zeros_like(b)}
    for i in range(case["experts"]):
        at = (s["ids"] == i).nonzero().view(-1)
        if at.numel():
            out["y"][at] = torch.addmm(b[i], x[at], w[i].t())
            out["gx"][at] = gy[at] @ w[i]
            out["gw"][i], out["gb"][i] = gy[at].t() @ values[at], gy[at].sum(0)
    return out
