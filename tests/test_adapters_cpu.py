"""The adapter entry points without a GPU: what the C ABI and the Python calls refuse, and with which error."""
from __future__ import annotations

import types

import pytest
import torch

import engraft_ngram_b200 as eb
from engraft_ngram_b200 import _lib as L
from engraft_ngram_b200 import adapters as AD


@pytest.fixture(scope="module")
def lib():
    from engraft_ngram_b200 import build
    build.build()
    return L.load()


X, A, B, IX, BASE, OUT, WS = (0x100000 * k for k in range(1, 8))
BIG = 1 << 40


def forward(lib, **kw):
    v = dict(dtype=0, x=X, ldx=64, a=A, b=B, index=IX, scale=None, T=10, n=3, rank=4, K=64, N=32, base=BASE, ldb=32,
             out=OUT, ldo=32, ws=WS, ws_bytes=BIG)
    v.update(kw)
    return lib.engram_adapter_forward(*v.values(), None)


def backward(lib, **kw):
    v = dict(dtype=0, grad=BASE, ldg=32, x=X, ldx=64, a=A, b=B, index=IX, scale=None, T=10, n=3, rank=4, K=64, N=32,
             dx_base=None, lddb=0, dx=OUT, lddx=64, da=A + 64, db=B + 64, ws=WS, ws_bytes=BIG)
    v.update(kw)
    return lib.engram_adapter_backward(*v.values(), None)


@pytest.mark.parametrize("bad, code", [
    (dict(dtype=3), L.ERR_FORMAT), (dict(dtype=-1), L.ERR_FORMAT), (dict(T=-1), L.ERR_ARG), (dict(n=-1), L.ERR_ARG),
    (dict(rank=0), L.ERR_ARG), (dict(rank=129), L.ERR_RANGE), (dict(n=16385), L.ERR_RANGE), (dict(K=0), L.ERR_ARG),
    (dict(N=0), L.ERR_ARG), (dict(T=(1 << 30) + 1), L.ERR_RANGE), (dict(x=None), L.ERR_ARG),
    (dict(index=None), L.ERR_ARG), (dict(a=None), L.ERR_ARG), (dict(b=None), L.ERR_ARG), (dict(ws=None), L.ERR_ARG),
    (dict(ws=WS + 8), L.ERR_ARG), (dict(ldx=63), L.ERR_ARG), (dict(x=X + 2), L.ERR_ARG),
    (dict(dtype=1, x=X + 1), L.ERR_ARG), (dict(ws_bytes=64), L.ERR_WORKSPACE)])
def test_both_directions_refuse_with_the_documented_code(lib, bad, code):
    assert forward(lib, **bad) == code
    assert backward(lib, **bad) == code


@pytest.mark.parametrize("bad", [dict(out=None), dict(ldo=31), dict(ldb=31), dict(base=OUT, ldb=40),
                                 dict(base=BASE + 2)])
def test_forward_refuses(lib, bad):
    assert forward(lib, **bad) == L.ERR_ARG


@pytest.mark.parametrize("bad", [dict(grad=None), dict(ldg=31), dict(lddx=63), dict(dx_base=X, lddb=63),
                                 dict(dx_base=OUT, lddb=80), dict(dx=OUT + 2), dict(da=A + 1)])
def test_backward_refuses(lib, bad):
    assert backward(lib, **bad) == L.ERR_ARG


def test_no_positions_is_no_work_and_the_workspace_grows_with_them(lib):
    assert forward(lib, T=0, x=None, index=None, out=None, ws=None, ws_bytes=0) == 0
    size = [lib.engram_adapter_workspace_bytes(T, 8, 16, 64, 128, back) for T in (1, 500, 9000) for back in (0, 1)]
    assert size[0] < size[2] < size[4] and size[0] < size[1] and size[4] < size[5]
    assert lib.engram_adapter_workspace_bytes(5, 8, 0, 64, 128, 0) == L.ERR_ARG
    assert lib.engram_adapter_workspace_bytes(5, 8, 129, 64, 128, 1) == L.ERR_RANGE


def test_python_calls_refuse_what_they_cannot_read():
    x, a, b = torch.zeros(5, 8), torch.zeros(2, 3, 8), torch.zeros(2, 6, 3)
    index = torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        eb.adapter_add(torch.zeros(5, 6), x, a, b, index)
    with pytest.raises(ValueError, match="CUDA"):
        eb.adapter_gradients(torch.zeros(5, 6), x, a, b, index)
    with pytest.raises(ValueError, match="CUDA"):
        eb.adapter_add(None, x.double(), a, b, index)
    with pytest.raises(ValueError, match="out="):
        eb.adapter_add(None, x, a.requires_grad_(), b, index, out=torch.zeros(5, 6))


@pytest.mark.parametrize("stride, T, ok", [((8, 1), 5, True), ((16, 1), 5, True), ((0, 1), 5, False),
                                           ((1, 5), 5, False), ((0, 1), 1, True)])
def test_row_strides(stride, T, ok):
    like = torch.zeros(1)
    v = torch.zeros(200).as_strided((T, 8), stride)
    if ok:
        assert AD._rows(v, "v", T, 8, like) == (stride[0] if T > 1 else 8)
    else:
        with pytest.raises(ValueError, match="strides"):
            AD._rows(v, "v", T, 8, like)


# the workspace is too small: what is accepted ends with ERR_WORKSPACE, before any launch
@pytest.mark.parametrize("alias, refused", [
    (dict(dx=X), True), (dict(dx=BASE, lddx=64, ldg=64, N=64), True), (dict(da=X), True), (dict(db=X), True),
    (dict(da=BASE), True), (dict(db=BASE), True), (dict(dx=OUT, da=OUT), True), (dict(dx=OUT, db=OUT), True),
    (dict(da=B + 64, db=B + 64), True), (dict(dx=X, da=None), False), (dict(dx=BASE, ldg=64, N=64, db=None), False),
    (dict(dx_base=OUT, lddb=64), False), (dict(), False)])
def test_backward_refuses_outputs_that_destroy_what_it_still_reads(lib, alias, refused):
    assert backward(lib, ws_bytes=64, **alias) == (L.ERR_ARG if refused else L.ERR_WORKSPACE)


def test_a_scale_that_requires_grad_is_refused_where_its_gradient_would_be_lost():
    x, a, b = torch.zeros(5, 8), torch.zeros(2, 3, 8), torch.zeros(2, 6, 3)
    index, scale = torch.zeros(5, dtype=torch.int32), torch.ones(2, requires_grad=True)
    for leaf in (x, x.clone().requires_grad_()):
        with pytest.raises(ValueError, match="scale requires grad"):
            eb.adapter_add(None, leaf, a, b, index, scale)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # nothing is lost: on to the other checks
        eb.adapter_add(None, x, a, b, index, scale)
    with pytest.raises(ValueError, match="CUDA"):
        eb.adapter_add(None, x, a, b, index, scale.detach())


def test_ple_forward_refuses_a_scale_that_requires_grad():
    n, hc = 8, 2
    w = types.SimpleNamespace(w_key=torch.zeros(hc * n, n), w_value=torch.zeros(n, n), norm_key=torch.zeros(hc, n),
                              norm_query=torch.zeros(hc, n), norm_conv=torch.zeros(hc, n), conv1d=torch.zeros(hc * n, 4))
    hp = types.SimpleNamespace(hc_mult=hc, n_embd=n, f_norm_rms_eps=1e-6, ple_ngram_size=3)
    ad = eb.PleAdapters(torch.zeros(2, 3, n), torch.zeros(2, hc * n + n, 3), torch.zeros(4, dtype=torch.int32),
                        torch.ones(2, requires_grad=True))
    with pytest.raises(ValueError, match="scale requires grad"):
        eb.ple_forward(torch.zeros(4, n), torch.zeros(4, hc, n), w, torch.zeros(0, hc, n), hp, adapters=ad)
