"""Refusals and workspace sizes of the rotary, layer norm and gated feed-forward
entry points, on the host: every bad argument is an error code and a message
before any launch, and calls without rows launch nothing."""
import ctypes

import numpy as np
import pytest

from edgebert_amd import _native as N

BUF = np.zeros(4096, np.float32)
BASE = BUF.ctypes.data + (-BUF.ctypes.data) % 64
BAD = N.EBH_ERR_INVALID_ARG


@pytest.fixture(scope="module")
def L():
    return N.lib()


def refused(rc, words):
    assert rc == BAD and words in N.last_error(), (rc, N.last_error())


def rope_args(**kw):
    cfg = dict(rot_dim=32, layout=0, scaling=0, original_len=512, base=1e4, factor=8.0, turns_fast=32.0, turns_slow=1.0,
               magnitude=1.0)
    cfg.update({k: kw.pop(k) for k in list(kw) if k in cfg})
    a = dict(x=BASE, ldx=64, y=BASE + 4096, ldy=64, dtype=0, pos=BASE + 8192, n_tokens=None, T=4, n=2, d=32,
             cfg=ctypes.byref(N.EbhRope(**cfg)), transpose=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,words", [
    (dict(cfg=None), "null rope config"), (dict(dtype=2), "unknown dtype"), (dict(dtype=-1), "unknown dtype"),
    (dict(T=-1), "bad rope shape"), (dict(n=0), "bad rope shape"), (dict(n=65537), "bad rope shape"), (dict(d=0), "bad rope shape"), (dict(d=1025), "bad rope shape"),
    (dict(rot_dim=31), "rot_dim"), (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=-2), "rot_dim"), (dict(rot_dim=34), "rot_dim"),
    (dict(layout=2), "layout"), (dict(scaling=4), "scaling"), (dict(scaling=-1), "scaling"),
    (dict(base=0.0), "base"), (dict(base=float("nan")), "base"), (dict(base=float("inf")), "base"),
    (dict(magnitude=float("nan")), "magnitude"),
    (dict(scaling=1, factor=0.0), "factor"), (dict(scaling=2, factor=-1.0), "factor"), (dict(scaling=3, factor=float("inf")), "factor"),
    (dict(scaling=3, original_len=0), "wavelength"), (dict(scaling=3, turns_fast=1.0), "wavelength"),
    (dict(scaling=3, turns_slow=float("nan")), "wavelength"),
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(pos=None), "null"),
    (dict(ldx=63), "strides"), (dict(ldy=63), "strides"), (dict(ldx=-64), "strides"),
    (dict(x=BASE + 2), "aligned"), (dict(dtype=1, y=BASE + 4097), "aligned"), (dict(pos=BASE + 2), "aligned"),
    (dict(n_tokens=BASE + 1), "aligned"), (dict(y=BASE, ldx=64, ldy=72), "in place"),
])
def test_rope_refusals(L, kw, words):
    refused(L.ebh_op_rope(*rope_args(**kw)), words)


def norm_fwd(**kw):
    a = dict(x=BASE, ldx=64, dtype=0, gamma=BASE, beta=BASE, rows=2, H=64, eps=1e-12, y=BASE + 1024, ldy=64, mean=None, rstd=None,
             stream=None)
    a.update(kw)
    return list(a.values())


def norm_bwd(**kw):
    a = dict(dy=BASE, lddy=64, x=BASE + 1024, ldx=64, dtype=0, gamma=BASE, mean=BASE, rstd=BASE, dres=None, lddres=0, rows=2,
             H=64, dx=BASE + 2048, lddx=64, dgamma=BASE + 4096, dbeta=BASE + 5120, ws=BASE + 6144, size=1 << 30, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,words", [
    (dict(dtype=2), "unknown dtype"), (dict(rows=-1), "shape"), (dict(H=0), "shape"), (dict(H=8193), "shape"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(x=None), "null"), (dict(y=None), "null"),
    (dict(ldx=63), "strides"), (dict(ldy=63), "strides"), (dict(y=BASE, ldy=65), "strides"),
    (dict(x=BASE + 2), "aligned"), (dict(y=BASE + 1), "aligned"), (dict(gamma=BASE + 2), "aligned"), (dict(beta=BASE + 1), "aligned"),
    (dict(mean=BASE + 2), "aligned"), (dict(rstd=BASE + 2), "aligned"),
])
def test_layer_norm_fwd_refusals(L, kw, words):
    refused(L.ebh_op_layer_norm_fwd(*norm_fwd(**kw)), words)


@pytest.mark.parametrize("kw,words", [
    (dict(dtype=2), "unknown dtype"), (dict(rows=-1), "shape"), (dict(H=0), "shape"), (dict(H=8193), "shape"),
    (dict(dy=None), "null"), (dict(x=None), "null"), (dict(mean=None), "null"), (dict(rstd=None), "null"), (dict(dx=None), "null"),
    (dict(lddy=63), "strides"), (dict(ldx=63), "strides"), (dict(lddx=63), "strides"), (dict(dres=BASE, lddres=63), "strides"),
    (dict(dx=BASE, lddx=65), "strides"), (dict(dx=BASE + 1024, lddx=65), "strides"),
    (dict(dres=BASE + 2048, lddres=65), "strides"),
    (dict(dy=BASE + 2), "aligned"), (dict(dx=BASE + 2), "aligned"), (dict(dgamma=BASE + 2), "aligned"), (dict(dbeta=BASE + 2), "aligned"),
    (dict(ws=None), "workspace"), (dict(size=16), "workspace"), (dict(ws=BASE + 8), "workspace"),
    (dict(dgamma=None, ws=None, size=0), "workspace"),
])
def test_layer_norm_bwd_refusals(L, kw, words):
    refused(L.ebh_op_layer_norm_bwd(*norm_bwd(**kw)), words)


def ffn(**kw):
    a = dict(X=BASE, ldx=64, Wgu=BASE, bgu=None, Wd=BASE, bd=None, Y=BASE + 1024, ldy=64, h=BASE + 2048, gu=None, M=2, H=64, I=72,
             act=0, dtype=1, ws=BASE + 4096, size=1 << 30, stream=None)
    a.update(kw)
    return list(a.values())


def ffn_bwd(**kw):
    a = dict(dY=BASE, lddy=64, X=BASE, ldx=64, h=BASE, gu=BASE, Wgu=BASE, Wd=BASE, dX=BASE + 1024, lddx=64, dWgu=BASE + 2048,
             dbgu=None, dWd=BASE + 4096, dbd=None, M=2, H=64, I=72, act=0, dtype=1, ws=BASE + 8192, size=1 << 30, stream=None)
    a.update(kw)
    return list(a.values())


SHAPES = [(dict(dtype=2), "unknown dtype"), (dict(M=-1), "shape"), (dict(M=2 ** 30 + 1), "shape"), (dict(H=0), "shape"), (dict(I=0), "shape"), (dict(H=60), "shape"),
          (dict(I=68), "shape"), (dict(H=65544, ldx=65544), "shape"), (dict(I=65544), "shape"), (dict(H=32768, I=32768, ldx=32768), "too large"), (dict(act=3), "activation"),
          (dict(act=-1), "activation")]


@pytest.mark.parametrize("kw,words", SHAPES + [
    (dict(X=None), "null"), (dict(Wgu=None), "null"), (dict(Wd=None), "null"), (dict(Y=None), "null"), (dict(h=None), "null"),
    (dict(ldx=56), "ldx"), (dict(ldx=68), "ldx"), (dict(ldx=2_796_208), "ldx"), (dict(ldy=63), "ldy"), (dict(ldy=2_796_208), "ldy"),
    (dict(X=BASE + 8), "aligned"), (dict(Y=BASE + 8), "aligned"), (dict(h=BASE + 2), "aligned"), (dict(gu=BASE + 8), "aligned"),
    (dict(bgu=BASE + 4), "aligned"), (dict(bd=BASE + 4), "aligned"), (dict(Wgu=BASE + 8), "aligned"), (dict(Wd=BASE + 8), "aligned"),
])
def test_gated_ffn_refusals(L, kw, words):
    refused(L.ebh_op_gated_ffn(*ffn(**kw)), words)


@pytest.mark.parametrize("kw,words", SHAPES + [
    (dict(dY=None), "null"), (dict(X=None), "null"), (dict(h=None), "null"), (dict(gu=None), "null"), (dict(Wgu=None), "null"),
    (dict(Wd=None), "null"), (dict(lddy=56), "lddy"), (dict(ldx=60), "ldx"), (dict(lddx=66), "lddx"), (dict(lddx=2_796_208), "lddx"),
    (dict(dY=BASE + 8), "aligned"), (dict(dX=BASE + 8), "aligned"), (dict(dWgu=BASE + 8), "aligned"), (dict(dbgu=BASE + 8), "aligned"),
    (dict(dWd=BASE + 8), "aligned"), (dict(dbd=BASE + 8), "aligned"), (dict(gu=BASE + 8), "aligned"), (dict(h=BASE + 8), "aligned"),
    (dict(ws=None), "workspace"), (dict(size=16), "workspace"), (dict(ws=BASE + 8), "workspace"),
])
def test_gated_ffn_bwd_refusals(L, kw, words):
    refused(L.ebh_op_gated_ffn_bwd(*ffn_bwd(**kw)), words)


def test_calls_without_rows_are_fine(L):
    assert L.ebh_op_rope(*rope_args(T=0, x=None, y=None, pos=None)) == N.EBH_OK
    assert L.ebh_op_layer_norm_fwd(*norm_fwd(rows=0, x=None, y=None)) == N.EBH_OK
    none = dict(dgamma=None, dbeta=None, ws=None, size=0)
    assert L.ebh_op_layer_norm_bwd(*norm_bwd(rows=0, dy=None, x=None, dx=None, **none)) == N.EBH_OK
    assert L.ebh_op_gated_ffn(*ffn(M=0, X=None, Y=None, h=None)) == N.EBH_OK
    none = dict(dX=None, dWgu=None, dWd=None, ws=None, size=0)
    assert L.ebh_op_gated_ffn_bwd(*ffn_bwd(M=0, **none)) == N.EBH_OK


def test_workspace_sizes(L):
    for rows, H in ((-1, 8), (1, 0), (1, 8193)):
        refused(L.ebh_op_layer_norm_bwd_workspace(rows, H), "shape")
    for size in (L.ebh_op_gated_ffn_workspace, L.ebh_op_gated_ffn_bwd_workspace):
        for bad in ((-1, 64, 64, 0), (1, 60, 64, 0), (1, 64, 0, 0), (1, 64, 64, 2)):
            assert size(*bad) == BAD
        sizes = [size(M, 768, 2048, d) for M in (0, 1, 64, 65, 5000, 32768) for d in (0, 1)]
        assert all(s >= 0 and s % 16 == 0 for s in sizes)
    # [dg du] of every token is held
    assert L.ebh_op_gated_ffn_bwd_workspace(5000, 768, 2048, 1) >= 5000 * 4096 * 2
    # sizes past 32 bits
    assert L.ebh_op_gated_ffn_bwd_workspace(2 ** 30, 768, 2048, 0) >= 2 ** 30 * 4096 * 4
    # a bound on what a caller has to keep for norms, however many rows
    assert max(L.ebh_op_layer_norm_bwd_workspace(r, 768) for r in (1, 1000, 2 ** 31 - 1)) <= 64 << 20


def test_rope_tokens_are_bounded(L):
    """A grid has less than 2^32 lanes."""
    refused(L.ebh_op_rope(*rope_args(T=(1 << 26) + 1)), "bad rope shape")
