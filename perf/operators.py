"""What a rotary, gated encoder layer adds to the encoder, timed and compared:
rotary positions, layer norm and its gradients, and the gated feed-forward block
and its gradients, through ``include/edgebert_hip_ops.h``.

``own`` False: the operators from elementary torch operations, in 32 bits (the
angles of rotary positions in 64), rounded once at the end.  ``own`` True: the
library's entry points on the same inputs.

Cases, by ``op``:

* ``rope``: ``T`` tokens of packed sequences of ``lo`` .. ``hi`` tokens, ``n`` heads
  (q and k, of rows that hold v as well) of ``d`` columns, ``rot`` of them rotated;
  ``layout``, ``scaling`` and ``transpose`` (the gradient) as the entry point's.
* ``norm`` / ``norm_bwd``: ``rows`` x ``H``; ``affine`` with gamma and beta; ``res``
  with a residual path's gradient added.
* ``ffn`` / ``ffn_bwd``: ``M`` tokens, hidden size ``H``, intermediate size ``I``;
  ``act``, ``bias``; ``train``: the forward keeps what the backward reads.
"""
import ctypes
import math

import numpy as np
import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-12
_LAYOUTS = ("half", "interleaved")
_SCALINGS = ("none", "linear", "ntk", "wavelength")
_ACTS = ("silu", "gelu_tanh", "gelu_erf")


def _rope(name, dtype, T, lo, hi, n, d, rot, layout="half", scaling="none", transpose=False):
    return {"name": name, "op": "rope", "dtype": dtype, "T": T, "lo": lo, "hi": hi, "n": n, "d": d, "rot": rot,
            "layout": layout, "scaling": scaling, "transpose": transpose}


def _norm(name, op, dtype, rows, H, affine=True, res=False):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "H": H, "affine": affine, "res": res}


def _ffn(name, op, dtype, M, H, I, act, bias, train=False):
    return {"name": name, "op": op, "dtype": dtype, "M": M, "H": H, "I": I, "act": act, "bias": bias, "train": train}


def listed():
    return [
        # One short query's q and k: nothing but latency.
        _rope("rope_query", "fp32", 16, 16, 16, 24, 32, 32),
        # A bulk batch of 256 x 128 tokens, heads of 64 as in the wider model.
        _rope("rope_bulk", "bf16", 32768, 128, 128, 24, 64, 64),
        # Long documents past the trained length, part of each head, adjacent pairs;
        # the gradient's direction.
        _rope("rope_long", "fp32", 17011, 700, 16000, 24, 64, 32, "interleaved", "wavelength", True),
        # A server's mixed batch of sentences in fp32 rows of the narrow model.
        _norm("norm_mixed", "norm", "fp32", 2161, 384),
        # The largest bulk batch's rows, 1024 x 128 tokens, without parameters' shift or scale.
        _norm("norm_bulk", "norm", "bf16", 131072, 768, affine=False),
        # A training step's rows in bf16, the residual path's gradient joining in.
        _norm("norm_bwd_bulk", "norm_bwd", "bf16", 32768, 768, res=True),
        # A small step in fp32 with an odd row length.
        _norm("norm_bwd_odd", "norm_bwd", "fp32", 1061, 769),
        # One token at a time: a weight-bound pass.
        _ffn("ffn_token", "ffn", "bf16", 1, 768, 2048, "silu", False),
        # A server's mixed batch, inference.
        _ffn("ffn_mixed", "ffn", "bf16", 4322, 768, 2048, "gelu_tanh", True),
        # A training step's forward on the bulk batch.
        _ffn("ffn_train", "ffn", "bf16", 32768, 768, 2048, "silu", False, True),
        # Its backward pass: the largest work here.
        _ffn("ffn_bwd_train", "ffn_bwd", "bf16", 32768, 768, 2048, "silu", False),
        # A small fp32 step of the narrow model, sizes that no tile divides.
        _ffn("ffn_bwd_odd", "ffn_bwd", "fp32", 1061, 384, 1000, "gelu_erf", True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(("fp32", "bf16"))
    op = rng.choice(("rope", "norm", "norm_bwd", "ffn", "ffn", "ffn_bwd", "ffn_bwd"))
    if op == "rope":
        d = rng.choice((32, 64, 64, 80, 96, 128))
        rot = rng.choice((d, d, d // 2, 2 * rng.randint(1, d // 2)))
        n = rng.randint(2, 40)
        T = _log(rng, 1, max(2, min(131072, 100_000_000 // (n * d))))
        hi = _log(rng, 1, T)
        c = _rope("", dtype, T, rng.randint(1, hi), hi, n, d, rot, rng.choice(_LAYOUTS), rng.choice(_SCALINGS), rng.random() < 0.4)
    elif op in ("norm", "norm_bwd"):
        H = rng.choice((rng.randint(16, 4096), 8 * rng.randint(4, 512), rng.choice((384, 768, 1024))))
        c = _norm("", op, dtype, _log(rng, 1, min(131072, 100_000_000 // H)), H, rng.random() < 0.7,
                  op == "norm_bwd" and rng.random() < 0.5)
    else:
        H = 8 * rng.randint(16, 128)
        I = 8 * rng.randint(16, 512)
        most = 50_000_000_000 if dtype == "bf16" else 4_000_000_000   # of M H I: at most the listed cases' time
        c = _ffn("", op, dtype, _log(rng, 1, max(2, min(32768, most // (H * I)))), H, I, rng.choice(_ACTS), rng.random() < 0.5,
                 op == "ffn" and rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _positions(c, rng):
    """Positions in packed sequences, as packing writes them, until T tokens are there."""
    parts, left = [], c["T"]
    while left > 0:
        n = min(left, rng.randint(c["lo"], c["hi"] + 1))
        parts.append(np.arange(n, dtype=np.int32))
        left -= n
    return np.concatenate(parts)


def _scaling_of(c):
    """base, factor, original length, turns, magnitude of a case."""
    factor = 1.0 if c["scaling"] == "none" else 8.0
    m = 0.1 * math.log(factor) + 1.0 if c["scaling"] == "wavelength" else 1.0
    return {"base": 10000.0, "factor": factor, "length": 512, "fast": 32.0, "slow": 1.0, "magnitude": m}


def _hidden(g, rows, H, dtype):
    """Rows as they stand in an encoder: unit variance and a few features that are far larger."""
    x = torch.randn(rows, H, generator=g, device="cuda")
    x[:, :: max(97, H // 4)] *= 6.0
    return x.to(dtype)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[c["dtype"]]
    s = {"case": c}
    if c["op"] == "rope":
        s["qkv"] = torch.randn(c["T"], (c["n"] + c["n"] // 2) * c["d"], generator=g, device="cuda").to(dt)
        s["pos"] = torch.from_numpy(_positions(c, np.random.RandomState(seed % 2**32))).cuda()
    elif c["op"] in ("norm", "norm_bwd"):
        rows, H = c["rows"], c["H"]
        s["x"] = _hidden(g, rows, H, dt) + 0.5
        s["gamma"] = 1.0 + 0.1 * torch.randn(H, generator=g, device="cuda") if c["affine"] else None
        s["beta"] = 0.1 * torch.randn(H, generator=g, device="cuda") if c["affine"] else None
        if c["op"] == "norm_bwd":
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = 1.0 / torch.sqrt((x - s["mean"][:, None]).square().mean(1) + _EPS)
            s["dy"] = (0.01 * torch.randn(rows, H, generator=g, device="cuda")).to(dt)
            s["dres"] = (0.01 * torch.randn(rows, H, generator=g, device="cuda")).to(dt) if c["res"] else None
    else:
        M, H, I = c["M"], c["H"], c["I"]
        s["x"] = _hidden(g, M, H, dt)
        s["wgu"] = (torch.randn(2 * I, H, generator=g, device="cuda") / math.sqrt(H)).to(dt)
        s["wd"] = (torch.randn(H, I, generator=g, device="cuda") / math.sqrt(I)).to(dt)
        s["bgu"] = 0.1 * torch.randn(2 * I, generator=g, device="cuda") if c["bias"] else None
        s["bd"] = 0.1 * torch.randn(H, generator=g, device="cuda") if c["bias"] else None
        if c["op"] == "ffn_bwd":
            gu = _linear(s["x"].float(), s["wgu"].float(), s["bgu"])
            s["gu"] = gu.to(dt)
            s["h"] = (_act(gu[:, :I], c["act"]) * gu[:, I:]).to(dt)
            s["dy"] = (0.01 * torch.randn(M, H, generator=g, device="cuda")).to(dt)
            del gu
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _linear(x, w, b):
    y = torch.mm(x, w.t())
    return y if b is None else y + b


def _act(g, act):
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    if act == "gelu_erf":
        return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return 0.5 * g * (1.0 + torch.tanh(0.7978845608 * (g + 0.044715 * g * g * g)))


def _act_slope(g, act):
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-g))
        return p * (1.0 + g * (1.0 - p))
    if act == "gelu_erf":
        return 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    t = torch.tanh(0.7978845608 * (g + 0.044715 * g * g * g))
    return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * 0.7978845608 * (1.0 + 3.0 * 0.044715 * g * g)


def _frequencies(c):
    p, half = _scaling_of(c), c["rot"] // 2
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    base = p["base"]
    if c["scaling"] == "ntk" and c["rot"] > 2:
        base = base * p["factor"] ** (c["rot"] / (c["rot"] - 2))
    f = torch.exp(i * (-2.0 * math.log(base) / c["rot"]))
    if c["scaling"] == "linear":
        f = f / p["factor"]
    elif c["scaling"] == "wavelength":
        turns = f * (p["length"] / (2.0 * math.pi))
        keep = torch.clamp((turns - p["slow"]) / (p["fast"] - p["slow"]), 0.0, 1.0)
        f = f * (keep + (1.0 - keep) / p["factor"])
    return f


def _plain_rope(s):
    c = s["case"]
    T, n, d, rot, half = c["T"], c["n"], c["d"], c["rot"], c["rot"] // 2
    m = _scaling_of(c)["magnitude"]
    angle = s["pos"].double()[:, None] * _frequencies(c)
    cos = (m * torch.cos(angle)).float()[:, None, :]
    sin = (m * torch.sin(angle)).float()[:, None, :]
    if c["transpose"]:
        sin = -sin
    x = s["qkv"][:, : n * d].float().reshape(T, n, d)
    if c["layout"] == "half":
        a, b = x[..., :half], x[..., half:rot]
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    ra, rb = a * cos - b * sin, a * sin + b * cos
    r = torch.cat([ra, rb], -1) if c["layout"] == "half" else torch.stack([ra, rb], -1).reshape(T, n, rot)
    return torch.cat([r, x[..., rot:]], -1).reshape(T, n * d).to(_DT[c["dtype"]])


def _plain_norm(s):
    c = s["case"]
    x = s["x"].float()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1.0 / torch.sqrt(d.square().mean(1) + _EPS)
    y = d * rstd[:, None]
    if c["affine"]:
        y = y * s["gamma"] + s["beta"]
    return {"y": y.to(_DT[c["dtype"]]), "mean": mean, "rstd": rstd}


def _plain_norm_bwd(s):
    c = s["case"]
    dy = s["dy"].float()
    xh = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["gamma"] if c["affine"] else dy
    dx = s["rstd"][:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    if c["res"]:
        dx = dx + s["dres"].float()
    out = {"dx": dx.to(_DT[c["dtype"]])}
    if c["affine"]:
        out["dgamma"] = (dy * xh).sum(0)
        out["dbeta"] = dy.sum(0)
    return out


def _plain_ffn(s):
    c = s["case"]
    I, dt = c["I"], _DT[c["dtype"]]
    gu = _linear(s["x"].float(), s["wgu"].float(), s["bgu"])
    h = _act(gu[:, :I], c["act"]) * gu[:, I:]
    out = {"y": _linear(h, s["wd"].float(), s["bd"]).to(dt)}
    if c["train"]:
        out["gu"], out["h"] = gu.to(dt), h.to(dt)
    return out


def _plain_ffn_bwd(s):
    c = s["case"]
    I, dt = c["I"], _DT[c["dtype"]]
    dy, x = s["dy"].float(), s["x"].float()
    g, u = s["gu"][:, :I].float(), s["gu"][:, I:].float()
    dh = torch.mm(dy, s["wd"].float())
    dgu = torch.cat([dh * u * _act_slope(g, c["act"]), dh * _act(g, c["act"])], 1)
    out = {"dx": torch.mm(dgu, s["wgu"].float()).to(dt), "dwgu": torch.mm(dgu.t(), x).to(dt),
           "dwd": torch.mm(dy.t(), s["h"].float()).to(dt)}
    if c["bias"]:
        out["dbgu"], out["dbd"] = dgu.sum(0), dy.sum(0)
    return out


# ---------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------
def _own(s):
    from edgebert_amd import _native as N
    c, L = s["case"], N.lib()
    dt = _DT[c["dtype"]]
    code = N.EBH_DTYPE_F32 if c["dtype"] == "fp32" else N.EBH_DTYPE_BF16
    stream = torch.cuda.current_stream().cuda_stream

    def ptr(t):
        return None if t is None else t.data_ptr()

    def new(*shape, dtype=dt):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if c["op"] == "rope":
        p, x = _scaling_of(c), s["qkv"]
        n, d, T = c["n"], c["d"], c["T"]
        y = new(T, n * d)
        cfg = N.EbhRope(rot_dim=c["rot"], layout=_LAYOUTS.index(c["layout"]), scaling=_SCALINGS.index(c["scaling"]),
                        original_len=p["length"], base=p["base"], factor=p["factor"], turns_fast=p["fast"],
                        turns_slow=p["slow"], magnitude=p["magnitude"])
        N.check(L.ebh_op_rope(ptr(x), x.stride(0), ptr(y), n * d, code, ptr(s["pos"]), None, T, n, d, ctypes.byref(cfg),
                              int(c["transpose"]), stream))
        return y
    if c["op"] in ("norm", "norm_bwd"):
        rows, H, x = c["rows"], c["H"], s["x"]
        f32 = torch.float32
        if c["op"] == "norm":
            y, mean, rstd = new(rows, H), new(rows, dtype=f32), new(rows, dtype=f32)
            N.check(L.ebh_op_layer_norm_fwd(ptr(x), H, code, ptr(s["gamma"]), ptr(s["beta"]), rows, H, _EPS, ptr(y), H,
                                            ptr(mean), ptr(rstd), stream))
            return {"y": y, "mean": mean, "rstd": rstd}
        dx = new(rows, H)
        dgamma, dbeta = (new(H, dtype=f32), new(H, dtype=f32)) if c["affine"] else (None, None)
        size = L.ebh_op_layer_norm_bwd_workspace(rows, H) if c["affine"] else 0
        ws = new(size, dtype=torch.uint8)
        N.check(L.ebh_op_layer_norm_bwd(ptr(s["dy"]), H, ptr(x), H, code, ptr(s["gamma"]), ptr(s["mean"]), ptr(s["rstd"]),
                                        ptr(s["dres"]), H, rows, H, ptr(dx), H, ptr(dgamma), ptr(dbeta), ptr(ws), size, stream))
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    M, H, I = c["M"], c["H"], c["I"]
    act, x = _ACTS.index(c["act"]), s["x"]
    if c["op"] == "ffn":
        y, h = new(M, H), new(M, I)
        gu = new(M, 2 * I) if c["train"] else None
        size = L.ebh_op_gated_ffn_workspace(M, H, I, code)
        ws = new(size, dtype=torch.uint8)
        N.check(L.ebh_op_gated_ffn(ptr(x), H, ptr(s["wgu"]), ptr(s["bgu"]), ptr(s["wd"]), ptr(s["bd"]), ptr(y), H, ptr(h),
                                   ptr(gu), M, H, I, act, code, ptr(ws), size, stream))
        return {"y": y, "gu": gu, "h": h} if c["train"] else {"y": y}
    dx, dwgu, dwd = new(M, H), new(2 * I, H), new(H, I)
    dbgu, dbd = (new(2 * I, dtype=torch.float32), new(H, dtype=torch.float32)) if c["bias"] else (None, None)
    size = L.ebh_op_gated_ffn_bwd_workspace(M, H, I, code)
    ws = new(size, dtype=torch.uint8)
    N.check(L.ebh_op_gated_ffn_bwd(ptr(s["dy"]), H, ptr(x), H, ptr(s["h"]), ptr(s["gu"]), ptr(s["wgu"]), ptr(s["wd"]), ptr(dx), H,
                                   ptr(dwgu), ptr(dbgu), ptr(dwd), ptr(dbd), M, H, I, act, code, ptr(ws), size, stream))
    return {"dx": dx, "dwgu": dwgu, "dwd": dwd, "dbgu": dbgu, "dbd": dbd}


_PLAIN = {"rope": _plain_rope, "norm": _plain_norm, "norm_bwd": _plain_norm_bwd, "ffn": _plain_ffn, "ffn_bwd": _plain_ffn_bwd}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


def work(case):
    c = case
    e = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "rope":
        v = c["T"] * c["n"] * c["d"]
        return {"bytes": 2 * v * e + 4 * c["T"], "flops": 3 * c["T"] * c["n"] * c["rot"]}
    if c["op"] in ("norm", "norm_bwd"):
        v = c["rows"] * c["H"]
        params = 4 * c["H"] * (0 if not c["affine"] else 2 if c["op"] == "norm" else 3)
        passes = 2 if c["op"] == "norm" else 3 + int(c["res"])
        return {"bytes": passes * v * e + 8 * c["rows"] + params, "flops": (8 if c["op"] == "norm" else 14) * v}
    M, H, I = c["M"], c["H"], c["I"]
    biases = 4 * (2 * I + H) if c["bias"] else 0
    if c["op"] == "ffn":
        kept = 3 * M * I if c["train"] else 0
        return {"bytes": e * (2 * M * H + 3 * H * I + kept) + biases, "flops": 6 * M * H * I}
    return {"bytes": e * (3 * M * H + 3 * M * I + 6 * H * I) + biases, "flops": 12 * M * H * I}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _phi64(g, act):
    """The activation and its derivative, from their definitions: g s(g) with s the logistic
    function, the tanh form's logistic function of 2u, or the normal distribution's."""
    if act == "gelu_erf":
        s = torch.special.ndtr(g)
        return g * s, s + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        arg, darg = g, torch.ones_like(g)
    else:
        arg = 2 * 0.7978845608 * (g + 0.044715 * g ** 3)
        darg = 2 * 0.7978845608 * (1 + 3 * 0.044715 * g ** 2)
    s = torch.sigmoid(arg)
    return g * s, s + g * s * torch.sigmoid(-arg) * darg


def _exact_rope(c, s):
    p, n, d, rot = _scaling_of(c), c["n"], c["d"], c["rot"]
    freq = np.empty(rot // 2)
    for i in range(rot // 2):
        base = p["base"] * (p["factor"] ** (rot / (rot - 2.0)) if c["scaling"] == "ntk" and rot > 2 else 1.0)
        f = base ** (-2.0 * i / rot)
        if c["scaling"] == "linear":
            f /= p["factor"]
        if c["scaling"] == "wavelength":
            turns = p["length"] * f / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (turns - p["slow"]) / (p["fast"] - p["slow"])))
            f = keep * f + (1.0 - keep) * f / p["factor"]
        freq[i] = f
    theta = s["pos"].to(torch.float64)[:, None] * torch.from_numpy(freq).cuda()
    turn = torch.polar(torch.full_like(theta, p["magnitude"]), -theta if c["transpose"] else theta)[:, None, :]
    x = s["qkv"][:, : n * d].double().reshape(c["T"], n, d)
    y = x.clone()
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if c["layout"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y.reshape(c["T"], n * d)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "rope":
        return _exact_rope(c, s)
    if c["op"] in ("norm", "norm_bwd"):
        x = s["x"].double()
        if c["op"] == "norm":
            var, mean = torch.var_mean(x, 1, correction=0)
            rstd = (var + _EPS) ** -0.5
            y = (x - mean[:, None]) * rstd[:, None]
            return {"y": torch.addcmul(s["beta"].double(), y, s["gamma"].double()) if c["affine"] else y, "mean": mean, "rstd": rstd}
        r, dy = s["rstd"].double()[:, None], s["dy"].double()
        xh = (x - s["mean"].double()[:, None]) * r
        g = dy * (s["gamma"].double() if c["affine"] else 1.0)
        H = c["H"]
        dx = (H * g - g.sum(1, True) - xh * (g * xh).sum(1, True)) * r / H
        out = {"dx": dx + s["dres"].double() if c["res"] else dx, "dgamma": None, "dbeta": None}
        if c["affine"]:
            out["dgamma"], out["dbeta"] = (dy * xh).sum(0), dy.sum(0)
        return out
    I = c["I"]
    x, wgu, wd = s["x"].double(), s["wgu"].double(), s["wd"].double()
    if c["op"] == "ffn":
        gu = x @ wgu.T
        if c["bias"]:
            gu += s["bgu"].double()
        h = _phi64(gu[:, :I], c["act"])[0] * gu[:, I:]
        y = h @ wd.T
        if c["bias"]:
            y += s["bd"].double()
        return {"y": y, "gu": gu, "h": h} if c["train"] else {"y": y}
    a, da = _phi64(s["gu"][:, :I].double(), c["act"])
    dy = s["dy"].double()
    dh = dy @ wd
    dg, du = dh * s["gu"][:, I:].double() * da, dh * a
    out = {"dx": dg @ wgu[:I] + du @ wgu[I:], "dwgu": torch.cat([dg.T @ x, du.T @ x]), "dwd": dy.T @ s["h"].double(),
           "dbgu": None, "dbd": None}
    if c["bias"]:
        out["dbgu"], out["dbd"] = torch.cat([dg.sum(0), du.sum(0)]), dy.sum(0)
    return out
