"""The orthogonalisation entry points without a GPU: what the C ABI and the Python calls refuse."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import engraft_ngram_b200 as eb
from engraft_ngram_b200 import _lib as L
from engraft_ngram_b200 import muon as MU


@pytest.fixture(scope="module")
def lib():
    from engraft_ngram_b200 import build
    build.build()
    return L.load()


X, OUT, G, M, P2, M2, WS = (0x100000 * k for k in range(1, 8))
BIG = 1 << 44
DEFAULT = (C.c_double * 15)(*(MU.COEFFICIENTS * 5))


def coefficients(*triple, steps=5):
    return (C.c_double * (3 * steps))(*(triple * steps))


def ortho(lib, **kw):
    v = dict(dtype=0, x=X, stack=2, rows=8, cols=100, steps=5, c=DEFAULT, eps=1e-7, out=OUT, ws=WS, ws_bytes=BIG)
    v.update(kw)
    return lib.engram_orthogonalize(*v.values(), None)


def muon(lib, **kw):
    v = dict(dtype=0, p=X, g=G, m=M, p_out=P2, m_out=M2, stack=2, rows=8, cols=100, lr=1e-2, beta=0.9, nesterov=1,
             wd=0.0, steps=5, c=DEFAULT, eps=1e-7, ws=WS, ws_bytes=BIG)
    v.update(kw)
    return lib.engram_muon_step(*v.values(), None)


@pytest.mark.parametrize("bad, code", [
    (dict(dtype=3), L.ERR_FORMAT), (dict(stack=-1), L.ERR_ARG), (dict(rows=0), L.ERR_ARG), (dict(cols=-4), L.ERR_ARG),
    (dict(stack=65536), L.ERR_RANGE), (dict(rows=(1 << 24) + 1), L.ERR_RANGE),
    (dict(rows=(1 << 15) + 1, cols=1 << 16), L.ERR_RANGE), (dict(steps=0), L.ERR_ARG), (dict(steps=33), L.ERR_RANGE),
    (dict(c=None), L.ERR_ARG), (dict(eps=0.0), L.ERR_ARG), (dict(eps=float("nan")), L.ERR_ARG),
    (dict(ws=None), L.ERR_ARG), (dict(ws=WS + 8), L.ERR_ARG), (dict(ws_bytes=16), L.ERR_WORKSPACE),
    (dict(x=None), L.ERR_ARG), (dict(x=X + 2), L.ERR_ARG),
    # iterates that leave the range: a polynomial of 16, one that grows, and one that is no number
    (dict(c=coefficients(16.0, 0.0, 0.0)), L.ERR_RANGE), (dict(c=coefficients(1.5, 1.0, 0.0)), L.ERR_RANGE),
    (dict(c=coefficients(float("nan"), 0.0, 0.0)), L.ERR_RANGE)])
def test_both_entry_points_refuse_with_the_documented_code(lib, bad, code):
    assert ortho(lib, **bad) == code
    if "x" in bad:
        bad = dict(p=bad["x"])
    assert muon(lib, **bad) == code


@pytest.mark.parametrize("name", ["g", "m", "p_out", "m_out"])
def test_muon_refuses_missing_and_misaligned_arrays(lib, name):
    assert muon(lib, **{name: None}) == L.ERR_ARG
    assert muon(lib, **{name: X + 2}) == L.ERR_ARG


@pytest.mark.parametrize("alias", [dict(p=M), dict(p_out=M), dict(m_out=X), dict(p_out=M2), dict(g=P2), dict(g=M2)])
def test_muon_refuses_arrays_that_would_overwrite_one_another(lib, alias):
    assert muon(lib, **alias) == L.ERR_ARG


def test_nothing_to_do_and_the_workspace(lib):
    assert ortho(lib, stack=0, x=None, out=None, ws=None, ws_bytes=0) == 0
    size = lib.engram_orthogonalize_workspace_bytes
    assert size(0, 1, 100, 200) == size(0, 1, 100, 200) > size(1, 1, 100, 200) > 0  # bf16 keeps one plane of two
    assert size(0, 4, 16, 2560) < size(0, 40, 16, 2560)
    assert size(5, 1, 8, 8) == L.ERR_FORMAT and size(0, 1, 0, 8) == L.ERR_ARG and size(0, 1 << 20, 8, 8) == L.ERR_RANGE


def test_python_calls_refuse():
    x = torch.zeros(4, 6)
    with pytest.raises(ValueError, match="CUDA"):
        eb.orthogonalize(x)
    with pytest.raises(ValueError, match="CUDA"):
        eb.muon_step(x, x, x, 0.1)
    with pytest.raises(ValueError, match="steps"):
        MU._coefficients(MU.COEFFICIENTS, 0)
    with pytest.raises(ValueError, match="coefficients"):
        MU._coefficients((1.0, 2.0), 5)
    with pytest.raises(ValueError, match="coefficients"):
        MU._coefficients((), 5)
    with pytest.raises(ValueError, match="coefficients"):
        MU._coefficients(((1.0, 0.0, 0.0),) * 4, 5)
    assert list(MU._coefficients([[1, 2, 3], (4, 5, 6)], 2)) == [1, 2, 3, 4, 5, 6]
    with pytest.raises(ValueError, match="Muon"):
        eb.Muon([torch.nn.Parameter(torch.zeros(5))])
    with pytest.raises(ValueError, match="hyper-parameters"):
        eb.Muon([torch.nn.Parameter(torch.zeros(5, 5))], momentum=1.0)


# |c1 g + c2 g g| reaches 17 and 19.3 while the polynomial with c0 stays below 15: more than bf16's plane of longer sides
# holds, which has no c0
@pytest.mark.parametrize("triple", [(14.0, -40.0, 23.0), (14.9, -57.0, 42.0)])
def test_bf16_of_longer_sides_refuses_a_polynomial_that_leaves_the_range_without_c0(lib, triple):
    c = coefficients(*triple, steps=1)
    grid = torch.linspace(0, 1, 1001, dtype=torch.float64)
    rest = triple[1] * grid + triple[2] * grid ** 2
    assert rest.abs().max() > 65504 / 4096 and (triple[0] + rest).abs().max() < 15
    assert ortho(lib, dtype=1, rows=100, cols=100, steps=1, c=c) == L.ERR_RANGE
    assert ortho(lib, dtype=1, rows=300, cols=65, steps=1, c=c) == L.ERR_RANGE
    for dtype, rows in ((0, 100), (2, 100), (1, 64)):  # c0 on the diagonal, or sums in fp64: taken (and then no room)
        assert ortho(lib, dtype=dtype, rows=rows, cols=100, steps=1, c=c, ws_bytes=16) == L.ERR_WORKSPACE
    assert muon(lib, dtype=1, rows=100, cols=100, steps=1, c=c, ws_bytes=16) == L.ERR_WORKSPACE
