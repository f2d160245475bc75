"""Rotary positions, layer norm and the gated feed-forward block with their
gradients (include/edgebert_hip_ops.h), each against its definition in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of fp32, E half a step of
the operand type (bf16 2^-8, fp32 2^-24).  A sum of K products rounds its
partial sums, each at most |a| |b| (the operands' 2-norms), with signs as they
fall: 4 (sqrt(K) + 4) u |a| |b|.  Independent relative errors of at most E on
one operand add up to 4 E sqrt(sum a^2 b^2)."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def env():
    import torch
    import edgebert_amd as eb
    from edgebert_amd import _native as N
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    return torch, N, eb.lib()


def dtype_of(torch, bf16):
    return (torch.bfloat16, 1, 2.0 ** -8) if bf16 else (torch.float32, 0, U)


def stream(torch):
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def padded(torch, rows, cols, ld, dt, values=None, shift=0):
    """[rows, cols] with row stride ld inside a buffer of NaN: a view, and a check
    that everything around it still is NaN.  shift: elements its start is off a
    64-element border."""
    buf = torch.full((64 + shift + max(rows, 1) * ld + 256,), float("nan"), device="cuda", dtype=dt)
    view = buf[64 + shift:].as_strided((rows, cols), (ld, 1))
    if values is not None:
        view.copy_(values)

    def untouched():
        rest = buf.clone()
        rest[64 + shift:].as_strided((rows, cols), (ld, 1)).fill_(float("nan"))
        return bool(torch.isnan(rest).all())
    return view, untouched


def near(torch, got, want, tol, what):
    got, want = got.double(), want.double()
    over = (got - want).abs() - tol
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = int(over.argmax()) if over.numel() else 0
    assert over.numel() == 0 or float(over.max()) <= 0, (
        f"{what}: {got.flatten()[worst].item()} for {want.flatten()[worst].item()}, over by {float(over.max()):.3e} at {worst}, "
        f"{int((over > 0).sum())} of {over.numel()}")


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------
def frequencies64(rot, cfg):
    i = np.arange(rot // 2, dtype=np.float64)
    base = cfg.base * (cfg.factor ** (rot / (rot - 2.0)) if cfg.scaling == 2 and rot > 2 else 1.0)
    f = base ** (-2.0 * i / rot)
    if cfg.scaling == 1:
        f = f / cfg.factor
    if cfg.scaling == 3:
        g = np.clip((cfg.original_len * f / (2 * np.pi) - cfg.turns_slow) / (cfg.turns_fast - cfg.turns_slow), 0, 1)
        f = f * (g + (1 - g) / cfg.factor)
    return f


def rope64(torch, x, pos, n, d, cfg, transpose):
    rot, T = cfg.rot_dim, x.shape[0]
    ang = pos.double()[:, None] * torch.from_numpy(frequencies64(rot, cfg)).cuda()
    c, s = torch.cos(ang)[:, None] * cfg.magnitude, torch.sin(ang)[:, None] * cfg.magnitude * (-1 if transpose else 1)
    x = x.double().reshape(T, n, d)
    y, size = x.clone(), x.abs()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if cfg.layout == 0 else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = abs(cfg.magnitude) * (x[..., a].abs() + x[..., b].abs())
    return y.reshape(T, n * d), size.reshape(T, n * d)


def rope_cfg(N, rot, layout=0, scaling=0, magnitude=1.0, base=10000.0):
    return N.EbhRope(rot_dim=rot, layout=layout, scaling=scaling, original_len=512, base=base, factor=8.0,
                     turns_fast=32.0, turns_slow=1.0, magnitude=magnitude)


def check_rope(env, T, n, d, cfg, bf16, transpose=0, ldx=None, ldy=None, shift=0, inplace=False, n_tokens=None, far=0):
    torch, N, L = env
    dt, code, E = dtype_of(torch, bf16)
    g = torch.Generator(device="cuda").manual_seed(T * 31 + n * 7 + d)
    ldx, ldy = ldx or n * d, ldy or n * d
    x, x_same = padded(torch, T, n * d, ldx, dt, torch.randn(T, n * d, generator=g, device="cuda"), shift)
    y, y_rest = (x, x_same) if inplace else padded(torch, T, n * d, ldy, dt, shift=shift)
    x0, y0 = x.clone(), y.clone()
    pos = torch.randint(0, 512, (T,), generator=g, device="cuda", dtype=torch.int32) + far
    nt = None if n_tokens is None else torch.tensor([n_tokens], device="cuda", dtype=torch.int32)
    N.check(L.ebh_op_rope(ptr(x), ldx, ptr(y), ldx if inplace else ldy, code, ptr(pos), ptr(nt), T, n, d,
                          ctypes.byref(cfg), transpose, stream(torch)))
    torch.cuda.synchronize()
    live = T if n_tokens is None else min(T, n_tokens)
    want, size = rope64(torch, x0[:live], pos[:live], n, d, cfg, transpose)
    # cos and sin: 2 u of the function, u of its argument (at most pi / 4), u of
    # the magnitude; two products and a sum of them: 3 u
    e32 = 8 * U * size
    near(torch, y[:live], want, e32 + E * (want.abs() + e32), "rope")
    cols = torch.arange(n * d, device="cuda") % d >= cfg.rot_dim
    assert torch.equal(y[:live][:, cols], x0[:live][:, cols]), "columns that pass"
    assert y_rest() and x_same()
    same = (y[live:] == y0[live:]) | (torch.isnan(y[live:]) & torch.isnan(y0[live:]))
    assert bool(same.all()), "rows behind the last token"


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("T,n,d,rot", [(1, 1, 2, 2), (1, 24, 32, 32), (7, 3, 64, 64), (130, 24, 64, 32), (33, 5, 80, 80),
                                       (19, 2, 96, 10), (5, 3, 33, 32), (3, 1, 1024, 1024), (4099, 4, 64, 64),
                                       (70, 2, 128, 126), (1000, 12, 64, 48)])
def test_rope(env, T, n, d, rot, layout, bf16):
    check_rope(env, T, n, d, rope_cfg(env[1], rot, layout), bf16)


@pytest.mark.parametrize("scaling", [0, 1, 2, 3])
@pytest.mark.parametrize("rot", [2, 32, 64])
@pytest.mark.parametrize("transpose", [0, 1])
def test_rope_scalings_and_transpose(env, scaling, rot, transpose):
    check_rope(env, 65, 3, 64, rope_cfg(env[1], rot, rot // 32 % 2, scaling, 1.25), False, transpose)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kw", [dict(ldx=3 * 256), dict(ldx=257, ldy=263), dict(shift=1), dict(inplace=True),
                                dict(inplace=True, ldx=771, shift=3), dict(n_tokens=0), dict(n_tokens=11),
                                dict(n_tokens=500, inplace=True), dict(far=1_000_000), dict(far=-700), dict(far=2_147_480_000)],
                         ids=str)
def test_rope_strides_alignment_and_positions(env, kw, bf16):
    """Positions near 2^31: the angle in turns is good to 2^31 * 2^-49 (the
    exponential's 64-bit rounding), 2^-18 of a turn; tested with frequencies
    that keep it below: a base of 1 turns every pair by the position itself."""
    cfg = rope_cfg(env[1], 64, 0)
    if abs(kw.get("far", 0)) > 10_000_000:
        cfg = rope_cfg(env[1], 64, 0, base=1.0)
    for layout in (0, 1):
        cfg.layout = layout
        check_rope(env, 37, 4, 64, cfg, bf16, **kw)


def test_rope_transpose_takes_gradients_back(env):
    """<y', R x> = <R^T y', x> with a magnitude, and R^T R = magnitude^2."""
    torch, N, L = env
    T, n, d, cfg = 50, 4, 64, rope_cfg(N, 48, 1, 3, 1.5)
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dy = (torch.randn(T, n * d, generator=g, device="cuda") for _ in range(2))
    pos = torch.arange(T, device="cuda", dtype=torch.int32) * 97
    y, dx, back = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    for src, dst, tr in ((x, y, 0), (dy, dx, 1), (y, back, 1)):
        N.check(L.ebh_op_rope(ptr(src), n * d, ptr(dst), n * d, 0, ptr(pos), None, T, n, d, ctypes.byref(cfg), tr, stream(torch)))
    torch.cuda.synchronize()
    lhs, rhs = (dy.double() * y.double()).sum(), (dx.double() * x.double()).sum()
    assert abs(float(lhs - rhs)) <= 16 * U * 1.5 * float(dy.norm() * x.norm())
    turned = torch.arange(n * d, device="cuda") % d < 48
    near(torch, back[:, turned], 2.25 * x[:, turned].double(), 32 * U * 2.25 * 2 * x.abs().max().double(), "R^T R x")


# ---------------------------------------------------------------------------
# Layer norm
# ---------------------------------------------------------------------------
NORM_SHAPES = [(1, 1), (1, 8), (3, 5), (2, 64), (65, 384), (1061, 769), (257, 768), (33, 1024), (9, 1000), (50, 2048),
               (17, 2050), (5, 4096), (3, 8192), (2, 8191), (2, 7000), (5000, 24), (3000, 128), (4, 300), (31, 6000)]


def norm_case(torch, rows, H, bf16, seed, offset=0.5, affine=True):
    dt, code, E = dtype_of(torch, bf16)
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, H, generator=g, device="cuda") * (1 + torch.rand(rows, 1, generator=g, device="cuda")) + offset
    gamma = 1 + 0.3 * torch.randn(H, generator=g, device="cuda") if affine else None
    beta = 0.5 * torch.randn(H, generator=g, device="cuda") if affine else None
    return dt, code, E, g, x.to(dt), gamma, beta


def norm_stats64(torch, x, eps):
    x = x.double()
    mean = x.mean(1)
    var = (x - mean[:, None]).square().mean(1)
    return mean, 1 / torch.sqrt(var + eps)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("affine", [True, False])
@pytest.mark.parametrize("rows,H", NORM_SHAPES)
@pytest.mark.parametrize("offset", [0.5, 300.0])
def test_layer_norm_fwd(env, rows, H, affine, bf16, offset):
    torch, N, L = env
    dt, code, E, g, x, gamma, beta = norm_case(torch, rows, H, bf16, rows + H, offset, affine)
    eps = 1e-5
    for ld, shift in ((H, 0), (H + 8, 0), (H + 3, 1)):
        xv, _ = padded(torch, rows, H, ld, dt, x, shift)
        yv, y_rest = padded(torch, rows, H, ld, dt, shift=shift)
        mean, m_rest = padded(torch, 1, rows, rows, torch.float32)
        rstd, r_rest = padded(torch, 1, rows, rows, torch.float32)
        N.check(L.ebh_op_layer_norm_fwd(ptr(xv), ld, code, ptr(gamma), ptr(beta), rows, H, eps, ptr(yv), ld, ptr(mean),
                                        ptr(rstd), stream(torch)))
        torch.cuda.synchronize()
        m64, r64 = norm_stats64(torch, x, eps)
        # a lane adds at most 64 values, then at most 16 partial sums; the same
        # again for the variance, whose relative error halves in rstd
        m_tol = 80 * U * x.double().abs().mean(1)
        d = (x.double() - m64[:, None]).abs()
        # a mean that is off by m adds m^2 to the variance
        r_tol = r64 * (50 * U + 0.5 * (m_tol * r64) ** 2)
        near(torch, mean[0], m64, m_tol, "mean")
        near(torch, rstd[0], r64, r_tol, "rstd")
        want = (x.double() - m64[:, None]) * r64[:, None]
        scale = gamma.double().abs() if affine else 1.0
        tol = scale * ((m_tol * r64)[:, None] + d * r_tol[:, None] + 4 * U * (want.abs() + (m_tol * r64)[:, None]))
        if affine:
            want = want * gamma.double() + beta.double()
            tol = tol + 2 * U * want.abs()
        near(torch, yv, want, tol + E * (want.abs() + tol), "y")
        assert y_rest() and m_rest() and r_rest()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("affine,res", [(True, False), (True, True), (False, True)])
@pytest.mark.parametrize("rows,H", NORM_SHAPES + [(20000, 64), (9001, 384)])
def test_layer_norm_bwd(env, rows, H, affine, res, bf16):
    torch, N, L = env
    dt, code, E, g, x, gamma, _ = norm_case(torch, rows, H, bf16, rows + H + 1, 0.5, affine)
    dy = torch.randn(rows, H, generator=g, device="cuda").to(dt)
    dres = torch.randn(rows, H, generator=g, device="cuda").to(dt) if res else None
    m64, r64 = norm_stats64(torch, x, 1e-5)
    mean, rstd = m64.float(), r64.float()
    for ld, shift in ((H, 0), (H + 5, 1)):
        xv, _ = padded(torch, rows, H, ld, dt, x, shift)
        dyv, _ = padded(torch, rows, H, ld, dt, dy, shift)
        rv = padded(torch, rows, H, ld, dt, dres, shift)[0] if res else None
        dxv, dx_rest = padded(torch, rows, H, ld, dt, shift=shift)
        dgamma, dg_rest = padded(torch, 1, H, H, torch.float32)
        dbeta, db_rest = padded(torch, 1, H, H, torch.float32)
        size = L.ebh_op_layer_norm_bwd_workspace(rows, H)
        ws, ws_rest = padded(torch, 1, size // 4, size // 4, torch.float32)
        N.check(L.ebh_op_layer_norm_bwd(ptr(dyv), ld, ptr(xv), ld, code, ptr(gamma), ptr(mean), ptr(rstd), ptr(rv), ld,
                                        rows, H, ptr(dxv), ld, ptr(dgamma), ptr(dbeta), ptr(ws), size, stream(torch)))
        torch.cuda.synchronize()
        xh = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
        gr = dy.double() * (gamma.double() if affine else 1.0)
        s, q = gr.mean(1, keepdim=True), (gr * xh).mean(1, keepdim=True)
        want = rstd.double()[:, None] * (gr - s - xh * q)
        # sums as in the forward (80 roundings); xh is off by 2 u |xh| + u |mean| rstd
        sa, qa = gr.abs().mean(1, keepdim=True), (gr.abs() * (xh.abs() + 1)).mean(1, keepdim=True)
        tol = rstd.double()[:, None] * 90 * U * (gr.abs() + sa + (xh.abs() + 1) * qa)
        if res:
            want = want + dres.double()
            tol = tol + U * want.abs()
        near(torch, dxv, want, tol + E * (want.abs() + tol), "dx")
        # columns: at most min(rows, 1100) sums in a chain
        n = min(rows, 1100) + 8
        near(torch, dgamma[0], (dy.double() * xh).sum(0), n * U * (dy.double().abs() * (xh.abs() + 1)).sum(0), "dgamma")
        near(torch, dbeta[0], dy.double().sum(0), n * U * dy.double().abs().sum(0), "dbeta")
        assert dx_rest() and dg_rest() and db_rest() and ws_rest()


def test_layer_norm_bwd_parts_in_place_and_no_rows(env):
    torch, N, L = env
    rows, H = 300, 384
    dt, code, E, g, x, gamma, _ = norm_case(torch, rows, H, True, 5)
    dy, dres = (torch.randn(rows, H, generator=g, device="cuda").to(dt) for _ in range(2))
    m64, r64 = norm_stats64(torch, x, 1e-5)
    mean, rstd = m64.float(), r64.float()
    size = L.ebh_op_layer_norm_bwd_workspace(rows, H)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def run(dyv, xv, rv, dxv, dgamma, dbeta, n=rows):
        w, sz = (ws, size) if dgamma is not None or dbeta is not None else (None, 0)
        N.check(L.ebh_op_layer_norm_bwd(ptr(dyv), H, ptr(xv), H, code, ptr(gamma), ptr(mean), ptr(rstd), ptr(rv), H, n, H,
                                        ptr(dxv), H, ptr(dgamma), ptr(dbeta), ptr(w), sz, stream(torch)))
        torch.cuda.synchronize()

    new = lambda: torch.full((H,), float("nan"), device="cuda")
    dx, dgamma, dbeta = torch.empty_like(x), new(), new()
    run(dy, x, dres, dx, dgamma, dbeta)
    for k in range(3):                       # over dy, x and dres
        ops = [dy.clone(), x.clone(), dres.clone()]
        g2, b2 = new(), new()
        run(*ops, ops[k], g2, b2)
        assert torch.equal(ops[k], dx) and torch.equal(g2, dgamma) and torch.equal(b2, dbeta)
    for want in ((True, False), (False, True), (False, False)):
        out, g2, b2 = torch.empty_like(x), new() if want[0] else None, new() if want[1] else None
        run(dy, x, dres, out, g2, b2)
        assert torch.equal(out, dx)
        assert (g2 is None or torch.equal(g2, dgamma)) and (b2 is None or torch.equal(b2, dbeta))
    g2, b2 = new(), new()
    run(dy, x, dres, dx, g2, b2, 0)
    assert not g2.any() and not b2.any()
    y = x.clone()                            # the forward in place
    z = torch.empty_like(x)
    for src, dst in ((x, z), (y, y)):
        N.check(L.ebh_op_layer_norm_fwd(ptr(src), H, code, ptr(gamma), None, rows, H, 1e-5, ptr(dst), H, None, None, stream(torch)))
    torch.cuda.synchronize()
    assert torch.equal(y, z)


def test_layer_norm_rows_with_nan_and_infinity_stay_alone(env):
    torch, N, L = env
    rows, H = 40, 768
    dt, code, E, g, x, gamma, beta = norm_case(torch, rows, H, True, 6)
    clean = torch.empty_like(x)
    N.check(L.ebh_op_layer_norm_fwd(ptr(x), H, code, ptr(gamma), ptr(beta), rows, H, 1e-5, ptr(clean), H, None, None, stream(torch)))
    bad = x.clone()
    bad[7, 5], bad[20, 767], bad[39, 0] = float("nan"), float("inf"), float("-inf")
    y = torch.empty_like(x)
    N.check(L.ebh_op_layer_norm_fwd(ptr(bad), H, code, ptr(gamma), ptr(beta), rows, H, 1e-5, ptr(y), H, None, None, stream(torch)))
    torch.cuda.synchronize()
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[[7, 20, 39]] = False
    assert torch.equal(y[rest], clean[rest])
    assert torch.isnan(y[~rest]).all()


# ---------------------------------------------------------------------------
# Gated feed-forward block
# ---------------------------------------------------------------------------
def act64(torch, g, act):
    if act == 0:
        s, ds = torch.sigmoid(g), torch.sigmoid(g) * torch.sigmoid(-g)
    elif act == 1:
        z = 2 * 0.7978845608 * (g + 0.044715 * g ** 3)
        s = torch.sigmoid(z)
        ds = s * torch.sigmoid(-z) * 2 * 0.7978845608 * (1 + 3 * 0.044715 * g ** 2)
    else:
        s, ds = torch.special.ndtr(g), torch.exp(-g * g / 2) / (2 * np.pi) ** 0.5
    return g * s, s + g * ds


def act_tol(g):
    """act and its slope in fp32: the exponential's argument t of at most 2 |g|
    (1 + g^2 / 20) gives 2 |t| u; what is formed of it, a few more u, scaled by
    at most 1 + |g|."""
    t = 2 * g.abs() * (1 + g * g / 20)
    return 8 * U * (1 + g.abs()) * (2 + t.clamp(max=100))


def product_tol(torch, A, B, E=0.0):
    """A [m, K], B [K, n]: a sum's roundings, and independent errors E of one operand."""
    K = A.shape[1]
    t = 4 * (K ** 0.5 + 4) * U * A.norm(dim=1)[:, None] * B.norm(dim=0)[None]
    return t + 4 * E * torch.sqrt((A * A) @ (B * B)) if E else t


def ffn_case(torch, M, H, I, bf16, bias, seed, extra=0):
    dt, code, E = dtype_of(torch, bf16)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    c = {"dt": dt, "code": code, "E": E, "M": M, "H": H, "I": I, "ld": H + extra}
    c["x"] = padded(torch, M, H, H + extra, dt, rnd(M, H))[0]
    c["wgu"] = padded(torch, 2 * I, H, H, dt, rnd(2 * I, H) / H ** 0.5 * 1.5)[0]
    c["wd"] = padded(torch, H, I, I, dt, rnd(H, I) / I ** 0.5)[0]
    c["bgu"] = padded(torch, 1, 2 * I, 2 * I, torch.float32, rnd(1, 2 * I))[0] if bias else None
    c["bd"] = padded(torch, 1, H, H, torch.float32, rnd(1, H))[0] if bias else None
    c["dy"] = padded(torch, M, H, H + extra, dt, rnd(M, H))[0]
    return c


def workspace(torch, size):
    if size == 0:
        return None, lambda: True
    return padded(torch, 1, size // 4, size // 4, torch.float32)


def run_ffn(env, c, act, keep=True):
    torch, N, L = env
    M, H, I = c["M"], c["H"], c["I"]
    y, y_rest = padded(torch, M, H, c["ld"], c["dt"])
    h, h_rest = padded(torch, M, I, I, c["dt"])
    gu, gu_rest = padded(torch, M, 2 * I, 2 * I, c["dt"]) if keep else (None, lambda: True)
    size = L.ebh_op_gated_ffn_workspace(M, H, I, c["code"])
    ws, ws_rest = workspace(torch, size)
    N.check(L.ebh_op_gated_ffn(ptr(c["x"]), c["ld"], ptr(c["wgu"]), ptr(c["bgu"]), ptr(c["wd"]), ptr(c["bd"]), ptr(y), c["ld"],
                               ptr(h), ptr(gu), M, H, I, act, c["code"], ptr(ws), size, stream(torch)))
    torch.cuda.synchronize()
    assert y_rest() and h_rest() and gu_rest() and ws_rest(), "a write outside the outputs"
    return y, h, gu


def run_ffn_bwd(env, c, act, h, gu, skip=()):
    torch, N, L = env
    M, H, I = c["M"], c["H"], c["I"]
    out = {"dx": padded(torch, M, H, c["ld"], c["dt"]), "dwgu": padded(torch, 2 * I, H, H, c["dt"]),
           "dbgu": padded(torch, 1, 2 * I, 2 * I, torch.float32), "dwd": padded(torch, H, I, I, c["dt"]),
           "dbd": padded(torch, 1, H, H, torch.float32)}
    a = {k: None if k in skip else v[0] for k, v in out.items()}
    size = L.ebh_op_gated_ffn_bwd_workspace(M, H, I, c["code"])
    ws, ws_rest = workspace(torch, size)
    N.check(L.ebh_op_gated_ffn_bwd(ptr(c["dy"]), c["ld"], ptr(c["x"]), c["ld"], ptr(h), ptr(gu), ptr(c["wgu"]), ptr(c["wd"]),
                                   ptr(a["dx"]), c["ld"], ptr(a["dwgu"]), ptr(a["dbgu"]), ptr(a["dwd"]), ptr(a["dbd"]), M, H, I,
                                   act, c["code"], ptr(ws), size, stream(torch)))
    torch.cuda.synchronize()
    assert ws_rest() and all(rest() for _, rest in out.values()), "a write outside the outputs"
    assert all(bool(torch.isnan(out[k][0]).all()) for k in skip), "a gradient that was not asked for"
    return a


def check_ffn(env, M, H, I, act, bf16, bias, extra=0, keep=True):
    torch, N, L = env
    c = ffn_case(torch, M, H, I, bf16, bias, M + H + I + act, extra)
    y, h, gu = run_ffn(env, c, act, keep)
    E, x, wgu, wd = c["E"], c["x"].double(), c["wgu"].double(), c["wd"].double()
    gu64 = x @ wgu.T + (c["bgu"].double() if bias else 0.0)
    t = product_tol(torch, x, wgu.T) + 2 * U * gu64.abs()
    if keep:
        near(torch, gu, gu64, t + E * (gu64.abs() + t), "gu")
    g, u, tg, tu = gu64[:, :I], gu64[:, I:], t[:, :I], t[:, I:]
    a, da = act64(torch, g, act)
    # |act'| <= 1.13 and |act''| <= 1.2 of the three
    ta = 1.2 * tg + act_tol(g)
    h64 = a * u
    th = a.abs() * tu + ta * (u.abs() + tu) + 2 * U * h64.abs()
    near(torch, h, h64, th + E * (h64.abs() + th), "h")
    bd = c["bd"].double() if bias else 0.0
    if bf16 and M <= 64:
        # of h before its rounding, as two bf16 (2^-17 of each value)
        y64 = h64 @ wd.T + bd
        ty = product_tol(torch, h64, wd.T, 2.0 ** -17) + th @ wd.T.abs() + 2 * U * y64.abs()
    else:                                                            # of the h that was written
        y64 = h.double() @ wd.T + bd
        ty = product_tol(torch, h.double(), wd.T) + 2 * U * y64.abs()
    near(torch, y, y64, ty + E * (y64.abs() + ty), "y")
    return c


def check_ffn_bwd(env, M, H, I, act, bf16, bias, extra=0):
    torch, N, L = env
    c = ffn_case(torch, M, H, I, bf16, bias, M + H + I + act + 1, extra)
    E, x, wgu, wd, dy = c["E"], c["x"].double(), c["wgu"].double(), c["wd"].double(), c["dy"].double()
    gu0 = x @ wgu.T + (c["bgu"].double() if bias else 0.0)
    gu = padded(torch, M, 2 * I, 2 * I, c["dt"], gu0)[0]
    h = padded(torch, M, I, I, c["dt"], act64(torch, gu0[:, :I], act)[0] * gu0[:, I:])[0]
    got = run_ffn_bwd(env, c, act, h, gu)
    g, u = gu[:, :I].double(), gu[:, I:].double()
    a, da = act64(torch, g, act)
    dh = dy @ wd
    th = product_tol(torch, dy, wd)
    dgu = torch.cat([dh * u * da, dh * a], 1)
    t = torch.cat([th * (u * da).abs() + (dh * u).abs() * act_tol(g), th * a.abs() + dh.abs() * act_tol(g)], 1) + 3 * U * dgu.abs()
    rounds = E if bf16 else 0.0                                   # [dg du] rounded once for the products

    def through(A, B, tA=None, tB=None):
        extra = (tA @ B.abs() if tA is not None else 0) + (A.abs() @ tB if tB is not None else 0)
        return extra

    dx64 = dgu @ wgu
    tx = product_tol(torch, dgu, wgu, rounds) + through(dgu, wgu, tA=t)
    near(torch, got["dx"], dx64, tx + E * (dx64.abs() + tx), "dx")
    dw64 = dgu.T @ x
    tw = product_tol(torch, dgu.T, x, rounds) + through(dgu.T, x, tA=t.T)
    near(torch, got["dwgu"], dw64, tw + E * (dw64.abs() + tw), "dwgu")
    dd64 = dy.T @ h.double()
    td = product_tol(torch, dy.T, h.double())
    near(torch, got["dwd"], dd64, td + E * (dd64.abs() + td), "dwd")
    n = 4 * (M ** 0.5 + 4) * U
    near(torch, got["dbgu"][0], dgu.sum(0), t.sum(0) + n * M ** 0.5 * dgu.norm(dim=0), "dbgu")
    near(torch, got["dbd"][0], dy.sum(0), n * M ** 0.5 * dy.norm(dim=0), "dbd")
    return c, h, gu, got


FFN_SHAPES = [(1, 8, 8), (1, 64, 128), (2, 24, 40), (5, 384, 1000), (15, 128, 64), (16, 200, 264), (17, 64, 128), (33, 72, 504),
              (64, 384, 512), (65, 128, 136), (100, 1024, 72), (129, 256, 384), (257, 264, 520), (300, 64, 2048), (1061, 384, 1000)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,H,I", FFN_SHAPES)
def test_gated_ffn(env, M, H, I, bf16):
    for act, bias, extra, keep in ((0, False, 0, True), (1, True, 8, False), (2, True, 40, True)):
        check_ffn(env, M, H, I, act, bf16, bias, extra, keep)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,H,I", FFN_SHAPES)
def test_gated_ffn_bwd(env, M, H, I, bf16):
    for act, bias, extra in ((0, False, 0), (1, True, 8), (2, True, 40)):
        check_ffn_bwd(env, M, H, I, act, bf16, bias, extra)


@pytest.mark.parametrize("M,H,I", [(4322, 768, 2048), (9000, 384, 1536), (2500, 1024, 520)])
def test_gated_ffn_many_tokens(env, M, H, I):
    check_ffn(env, M, H, I, 1, True, True)
    check_ffn_bwd(env, M, H, I, 0, True, True)


def test_gated_ffn_many_tokens_fp32(env):
    check_ffn(env, 2161, 384, 1536, 0, False, False)
    check_ffn_bwd(env, 2161, 384, 1536, 2, False, True)


def test_gated_ffn_bwd_parts_agree_with_the_whole(env):
    """Each gradient alone, and all but one: the same bits as all together; and the
    same bits again on a second call."""
    torch, N, L = env
    for bf16, M in ((True, 700), (False, 130)):
        c, h, gu, whole = check_ffn_bwd(env, M, 128, 264, 0, bf16, True)
        names = list(whole)
        for skip in [[]] + [[n for n in names if n != k] for k in names] + [[k] for k in names]:
            got = run_ffn_bwd(env, c, 0, h, gu, skip)
            for k in names:
                assert k in skip or torch.equal(got[k], whole[k]), (k, skip)


def test_gated_ffn_no_rows(env):
    torch, N, L = env
    for bf16 in (False, True):
        c = ffn_case(torch, 0, 64, 72, bf16, True, 9)
        h = torch.empty(0, 72, device="cuda", dtype=c["dt"])
        got = run_ffn_bwd(env, c, 0, h, torch.empty(0, 144, device="cuda", dtype=c["dt"]))
        for k in ("dwgu", "dbgu", "dwd", "dbd"):
            assert not got[k].any(), k
        N.check(L.ebh_op_gated_ffn(None, 64, None, None, None, None, None, 64, None, None, 0, 64, 72, 0, c["code"], None, 0, stream(torch)))


@pytest.mark.parametrize("M", [1, 70, 600])
def test_gated_ffn_token_with_nan_stays_alone(env, M):
    """A token's NaN or infinity reaches its own row of Y and dX, and no other."""
    torch, N, L = env
    c = ffn_case(torch, M, 128, 264, True, False, 4)
    y, h, gu = run_ffn(env, c, 0)
    base = run_ffn_bwd(env, c, 0, h, gu)
    bad = M // 2
    c["x"][bad, 3] = float("nan")
    c["dy"][bad, 7] = float("inf")
    rest = torch.arange(M, device="cuda") != bad
    y2, h2, gu2 = run_ffn(env, c, 0)
    assert torch.equal(y2[rest], y[rest]) and torch.isnan(y2[bad]).all()
    got = run_ffn_bwd(env, c, 0, h, gu)
    assert torch.equal(got["dx"][rest], base["dx"][rest]) and not torch.isfinite(got["dx"][bad]).all()


@pytest.mark.parametrize("act", [0, 1, 2])
def test_gated_ffn_saturated_gates(env, act):
    """Gates far out on both sides: act(g) goes to g and 0, its slope to 1 and 0, with no NaN."""
    torch, N, L = env
    H = I = 64
    x = torch.eye(64, device="cuda")
    for scale in (30.0, 200.0, 3.0e4):
        g = torch.linspace(-scale, scale, 64, device="cuda").repeat(64, 1)
        wgu = torch.cat([g.T.contiguous().T, torch.ones(64, 64, device="cuda")]).contiguous()
        c = {"dt": torch.float32, "code": 0, "E": U, "M": 64, "H": H, "I": I, "ld": 64, "x": x, "wgu": wgu, "bgu": None,
             "wd": torch.eye(64, device="cuda"), "bd": None, "dy": torch.ones(64, 64, device="cuda")}
        y, h, gu = run_ffn(env, c, act)
        a, da = act64(torch, gu[:, :I].double(), act)
        assert torch.isfinite(h).all()
        near(torch, h, a, act_tol(gu[:, :I].double()) + 4 * U * a.abs(), "h")
        got = run_ffn_bwd(env, c, act, h, gu)
        assert all(torch.isfinite(v).all() for v in got.values())
        n = da.sum(0)
        near(torch, got["dbgu"][0, :I], n, (act_tol(gu[:, :I].double()) + 100 * U * (1 + da.abs())).sum(0), "dbgu")


def test_gradients_against_differences(env):
    """Directional differences of the forward in 64 bits against the fp32 gradients
    of norm -> gated block + residual, in every argument."""
    torch, N, L = env
    M, H, I, eps = 37, 64, 104, 1e-5
    for act in (0, 1, 2):
        c = ffn_case(torch, M, H, I, False, True, 20 + act)
        g = torch.Generator(device="cuda").manual_seed(99)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float64)
        p = {"x": rnd(M, H).float().double(), "gamma": (1 + 0.2 * rnd(H)).float().double(), "beta": rnd(H).float().double(),
             "wgu": c["wgu"].double(), "bgu": c["bgu"][0].double(), "wd": c["wd"].double(), "bd": c["bd"][0].double()}
        R = c["dy"].double()

        def loss(q):
            m, r = norm_stats64(torch, q["x"], eps)
            z = (q["x"] - m[:, None]) * r[:, None] * q["gamma"] + q["beta"]
            gu = z @ q["wgu"].T + q["bgu"]
            return ((act64(torch, gu[:, :I], act)[0] * gu[:, I:]) @ q["wd"].T + q["bd"] + q["x"]).mul(R).sum()

        f32 = {k: v.float().contiguous() for k, v in p.items()}
        z, mean, rstd = torch.empty(M, H, device="cuda"), torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
        N.check(L.ebh_op_layer_norm_fwd(ptr(f32["x"]), H, 0, ptr(f32["gamma"]), ptr(f32["beta"]), M, H, eps, ptr(z), H, ptr(mean),
                                        ptr(rstd), stream(torch)))
        c.update(x=z, ld=H, dy=c["dy"].contiguous())
        y, h, gu = run_ffn(env, c, act)
        got = run_ffn_bwd(env, c, act, h, gu)
        dx, dgamma, dbeta = torch.empty(M, H, device="cuda"), torch.empty(H, device="cuda"), torch.empty(H, device="cuda")
        size = L.ebh_op_layer_norm_bwd_workspace(M, H)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        N.check(L.ebh_op_layer_norm_bwd(ptr(got["dx"]), H, ptr(f32["x"]), H, 0, ptr(f32["gamma"]), ptr(mean), ptr(rstd),
                                        ptr(c["dy"]), H, M, H, ptr(dx), H, ptr(dgamma), ptr(dbeta), ptr(ws), size, stream(torch)))
        torch.cuda.synchronize()
        grads = {"x": dx, "gamma": dgamma, "beta": dbeta, "wgu": got["dwgu"], "bgu": got["dbgu"][0], "wd": got["dwd"],
                 "bd": got["dbd"][0]}
        for k, grad in grads.items():
            v = rnd(*p[k].shape)
            e = 1e-4
            diff = (loss({**p, k: p[k] + e * v}) - loss({**p, k: p[k] - e * v})) / (2 * e)
            # the difference's own error, e^2 of the third derivative, and the
            # gradient's roundings: both far below 1e-4 of |grad| |v|
            assert abs(float(diff - (grad.double() * v).sum())) <= 1e-4 * float(grad.double().norm() * v.norm()), (act, k)


# ---------------------------------------------------------------------------
# Offsets past 32 bits
# ---------------------------------------------------------------------------
def test_rows_past_32_bit_offsets(env):
    """Rotary positions and layer norm over three rows 4.4 GB apart."""
    torch, N, L = env
    H, ld = 256, 2_200_000_000
    assert ld * 2 > 2 ** 32
    big = torch.zeros(2 * ld + H, device="cuda", dtype=torch.bfloat16)
    rows = big.as_strided((3, H), (ld, 1))
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(3, H, generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.tensor([5, 77, 300], device="cuda", dtype=torch.int32)
    cfg = rope_cfg(N, 64)

    def both(src, sld, dst, dld, base):
        mean, rstd = base.float().mean(1), 1 / base.float().std(1)
        dg, db = torch.empty(H, device="cuda"), torch.empty(H, device="cuda")
        size = L.ebh_op_layer_norm_bwd_workspace(3, H)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        outs = []
        for call in (lambda: L.ebh_op_rope(ptr(src), sld, ptr(dst), dld, 1, ptr(pos), None, 3, 4, 64, ctypes.byref(cfg), 0, stream(torch)),
                     lambda: L.ebh_op_layer_norm_fwd(ptr(src), sld, 1, None, None, 3, H, 1e-5, ptr(dst), dld, None, None, stream(torch)),
                     lambda: L.ebh_op_layer_norm_bwd(ptr(src), sld, ptr(src), sld, 1, None, ptr(mean), ptr(rstd), ptr(src), sld, 3, H,
                                                     ptr(dst), dld, ptr(dg), ptr(db), ptr(ws), size, stream(torch))):
            src.copy_(base)
            N.check(call())
            outs.append(dst.clone())
        return outs + [dg.clone(), db.clone()]

    near_rows = torch.empty(3, H, device="cuda", dtype=torch.bfloat16)
    want = both(x.clone(), H, near_rows, H, x)
    got = both(rows, ld, rows, ld, x)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del big, rows
    torch.cuda.empty_cache()


def test_gated_ffn_activations_past_4_gb(env):
    """560,000 tokens, g | u and their gradients of 4.6 GB each: the last tokens have
    the bits of a call of their own, weight gradients are near a sum over parts in 64 bits."""
    torch, N, L = env
    M, H, I, tail = 560_000, 64, 2048, 1000
    assert M * 2 * I * 2 > 2 ** 32
    c = ffn_case(torch, M, H, I, True, True, 3)
    y, h, gu = run_ffn(env, c, 0)
    got = run_ffn_bwd(env, c, 0, h, gu)
    t = {**c, "M": tail, "x": c["x"][-tail:], "dy": c["dy"][-tail:]}
    ty, th, tgu = run_ffn(env, t, 0)
    for a, b in ((y, ty), (h, th), (gu, tgu)):
        near(torch, a[-tail:], b, 2 ** -7 * b.double().abs() + 1e-3, "the last tokens")
    g, u = tgu[:, :I].double(), tgu[:, I:].double()
    a64, d64 = act64(torch, g, 0)
    dh = t["dy"].double() @ c["wd"].double()
    dgu = torch.cat([dh * u * d64, dh * a64], 1)
    wgu = c["wgu"].double()
    want = dgu @ wgu
    near(torch, got["dx"][-tail:], want, product_tol(torch, dgu, wgu, 2 ** -7) + 2 ** -8 * want.abs() + 1e-4, "dx of the last tokens")
    dwd, dbd = torch.zeros(H, I, device="cuda", dtype=torch.float64), torch.zeros(H, device="cuda", dtype=torch.float64)
    for at in range(0, M, 70_000):
        dy = c["dy"][at:at + 70_000].double()
        dwd += dy.T @ h[at:at + 70_000].double()
        dbd += dy.sum(0)
    ny, nh = c["dy"].float().norm(dim=0).double(), h.float().norm(dim=0).double()
    near(torch, got["dwd"], dwd, 4 * (M ** 0.5 + 4) * U * ny[:, None] * nh[None] + 2 ** -8 * dwd.abs(), "dwd")
    near(torch, got["dbd"][0], dbd, 4 * (M ** 0.5 + 4) * U * M ** 0.5 * ny, "dbd")
    del c, y, h, gu, got
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------
# Together, as a layer and a training step run them
# ---------------------------------------------------------------------------
def test_rotary_attention_over_packed_sequences(env):
    """qkv product, rotary positions in place on q and k, attention: packed sequences
    of uneven length, bf16, against 64 bits step by step."""
    torch, N, L = env
    lens, H, nh = [1, 77, 16, 128, 33], 128, 2
    T, d = sum(lens), H // nh
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(3 * H, H, generator=g, device="cuda") / H ** 0.5).to(torch.bfloat16)
    b = torch.randn(3 * H, generator=g, device="cuda")
    qkv = torch.empty(T, 3 * H, device="cuda", dtype=torch.bfloat16)
    N.check(L.ebh_op_gemm_bf16(ptr(x), H, ptr(w), H, ptr(b), ptr(qkv), 3 * H, 1, T, 3 * H, H, 0, stream(torch)))
    before = qkv.clone()
    pos = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in lens])
    cu = torch.tensor([0] + list(np.cumsum(lens)), device="cuda", dtype=torch.int32)
    cfg = rope_cfg(N, d)
    N.check(L.ebh_op_rope(ptr(qkv), 3 * H, ptr(qkv), 3 * H, 1, ptr(pos), None, T, 2 * nh, d, ctypes.byref(cfg), 0, stream(torch)))
    ctx = torch.empty(T, H, device="cuda", dtype=torch.bfloat16)
    N.check(L.ebh_op_attention_bf16(ptr(qkv), ptr(cu), len(lens), max(lens), H, nh, ptr(ctx), stream(torch)))
    torch.cuda.synchronize()
    want, size = rope64(torch, before[:, :2 * H], pos, 2 * nh, d, cfg, 0)
    near(torch, qkv[:, :2 * H], want, 8 * U * size + 2 ** -8 * (want.abs() + 8 * U * size), "q, k")
    assert torch.equal(qkv[:, 2 * H:], before[:, 2 * H:])
    at = 0
    for n in lens:
        for hd in range(nh):
            q, k, v = (qkv[at:at + n, s * H + hd * d: s * H + (hd + 1) * d].double() for s in range(3))
            p = torch.softmax(q @ k.T / d ** 0.5, 1)
            o = p @ v
            # probabilities rounded to bf16 for the product, the context once more
            near(torch, ctx[at:at + n, hd * d:(hd + 1) * d], o, 2 ** -7 * (p @ v.abs()) + 1e-5, "context")
        at += n


def block_step(env, c, act, f, out):
    """norm -> gated block, and both backward: every launch on the current stream."""
    torch, N, L = env
    M, H, I, code = c["M"], c["H"], c["I"], c["code"]
    s = stream(torch)
    N.check(L.ebh_op_rope(ptr(f["x"]), H, ptr(out["r"]), H, code, ptr(f["pos"]), None, M, H // 32, 32, ctypes.byref(f["cfg"]), 0, s))
    N.check(L.ebh_op_layer_norm_fwd(ptr(out["r"]), H, code, ptr(f["gamma"]), ptr(f["beta"]), M, H, 1e-5, ptr(out["z"]), H,
                                    ptr(out["mean"]), ptr(out["rstd"]), s))
    N.check(L.ebh_op_gated_ffn(ptr(out["z"]), H, ptr(c["wgu"]), ptr(c["bgu"]), ptr(c["wd"]), ptr(c["bd"]), ptr(out["y"]), H,
                               ptr(out["h"]), ptr(out["gu"]), M, H, I, act, code, ptr(out["ws"]), out["ws"].numel(), s))
    N.check(L.ebh_op_gated_ffn_bwd(ptr(c["dy"]), H, ptr(out["z"]), H, ptr(out["h"]), ptr(out["gu"]), ptr(c["wgu"]), ptr(c["wd"]),
                                   ptr(out["dz"]), H, ptr(out["dwgu"]), ptr(out["dbgu"]), ptr(out["dwd"]), ptr(out["dbd"]), M, H, I,
                                   act, code, ptr(out["ws"]), out["ws"].numel(), s))
    N.check(L.ebh_op_layer_norm_bwd(ptr(out["dz"]), H, ptr(out["r"]), H, code, ptr(f["gamma"]), ptr(out["mean"]), ptr(out["rstd"]),
                                    ptr(c["dy"]), H, M, H, ptr(out["dr"]), H, ptr(out["dgamma"]), ptr(out["dbeta"]),
                                    ptr(out["ws2"]), out["ws2"].numel(), s))
    N.check(L.ebh_op_rope(ptr(out["dr"]), H, ptr(out["dx"]), H, code, ptr(f["pos"]), None, M, H // 32, 32, ctypes.byref(f["cfg"]), 1, s))


def block_buffers(torch, L, c):
    M, H, I, dt = c["M"], c["H"], c["I"], c["dt"]
    e = lambda *s, d=dt: torch.full(s, float("nan"), device="cuda", dtype=d)
    f32 = torch.float32
    size = max(L.ebh_op_gated_ffn_workspace(M, H, I, c["code"]), L.ebh_op_gated_ffn_bwd_workspace(M, H, I, c["code"]), 16)
    b = lambda n: torch.zeros(n, device="cuda", dtype=torch.uint8)
    return {"r": e(M, H), "z": e(M, H), "mean": e(M, d=f32), "rstd": e(M, d=f32), "y": e(M, H), "h": e(M, I), "gu": e(M, 2 * I),
            "dz": e(M, H), "dwgu": e(2 * I, H), "dbgu": e(2 * I, d=f32), "dwd": e(H, I), "dbd": e(H, d=f32), "dr": e(M, H),
            "dgamma": e(H, d=f32), "dbeta": e(H, d=f32), "dx": e(M, H), "ws": b(size),
            "ws2": b(L.ebh_op_layer_norm_bwd_workspace(M, H))}


def block_inputs(torch, N, M, H, bf16, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.bfloat16 if bf16 else torch.float32
    return {"x": torch.randn(M, H, generator=g, device="cuda").to(dt), "gamma": 1 + 0.1 * torch.randn(H, generator=g, device="cuda"),
            "beta": torch.randn(H, generator=g, device="cuda"), "pos": torch.arange(M, device="cuda", dtype=torch.int32),
            "cfg": rope_cfg(N, 32)}


RESULTS = ("z", "mean", "rstd", "y", "h", "gu", "dz", "dwgu", "dbgu", "dwd", "dbd", "dr", "dgamma", "dbeta", "dx")


@pytest.mark.parametrize("bf16,M", [(True, 1), (True, 50), (True, 700), (False, 130)])
def test_step_captured_and_replayed(env, bf16, M):
    """A whole step as one graph: every replay, on new inputs and with eager work
    between, has the eager step's bits."""
    torch, N, L = env
    c = ffn_case(torch, M, 128, 264, bf16, True, 7)
    c["ld"], c["dy"] = 128, c["dy"].contiguous()
    f = block_inputs(torch, N, M, 128, bf16, 0)
    eager, replayed = block_buffers(torch, L, c), block_buffers(torch, L, c)
    block_step(env, c, 0, f, eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block_step(env, c, 0, f, replayed)
    for seed in range(4):
        f["x"].copy_(block_inputs(torch, N, M, 128, bf16, seed)["x"])
        block_step(env, c, 0, f, eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in RESULTS:
            assert torch.equal(eager[k], replayed[k]), (seed, k)


def test_steps_on_two_streams_at_once(env):
    torch, N, L = env
    cases, alone, both = [], [], []
    for seed in (0, 1):
        c = ffn_case(torch, 500, 128, 264, True, True, 30 + seed)
        c["ld"], c["dy"] = 128, c["dy"].contiguous()
        f = block_inputs(torch, N, 500, 128, True, seed)
        cases.append((c, f))
        alone.append(block_buffers(torch, L, c))
        both.append(block_buffers(torch, L, c))
        block_step(env, c, 1, f, alone[-1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for s, (c, f), out in zip(streams, cases, both):
            with torch.cuda.stream(s):
                block_step(env, c, 1, f, out)
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        for k in RESULTS:
            assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("M", [1, 20, 64, 65, 300])
@pytest.mark.parametrize("bf16", [False, True])
def test_gated_ffn_infinite_products_stay_infinite(env, bf16, M):
    """g u past the type's largest value is infinite, and so is Y = h.Wd^T of
    weights above 0, at every size; the other tokens are as without it."""
    torch, N, L = env
    c = ffn_case(torch, M, 64, 96, bf16, False, 5)
    c["wgu"].abs_()
    c["wd"].abs_().add_(0.25)
    plain, _, _ = run_ffn(env, c, 0)
    c["x"][M - 1] = 1e30
    y, h, _ = run_ffn(env, c, 0)
    assert bool((h[M - 1] == float("inf")).all()) and bool((y[M - 1] == float("inf")).all())
    assert torch.equal(y[: M - 1], plain[: M - 1]) and bool(torch.isfinite(plain).all())

