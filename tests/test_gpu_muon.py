"""orthogonalize, muon_step and Muon on the GPU against the formula in 64 bits.

The reference is the definition by singular values: U diag(f(s)) V^T with f the
steps applied to each normalised singular value, from an SVD in 64 bits.

Bounds.  Sides up to 64 are summed in fp64, so an element is off by half a step
of its type and by fp64's rounding, enlarged by the steps' growth of weak
directions squared (c0^10 = 2.4e5) and the sums' lengths: far below 2^-28 of the
matrix' root mean square.  Longer sides round every product as fp32 does, up to
a factor: a split product is off by at most 2^-21 of itself where fp32 rounds to
2^-24, and the tensor cores' sums round toward zero (twice the step).  Both are
enlarged by the steps in the same way, so the 2-norm of the error may be 16
times that of the plain fp32 form on the same input, plus the half step of the
type.  bf16 takes one product of operands rounded to 2^-12: a step is off by about
2^-11 of its sums, whose magnitudes are at most 3.5 times its result, and the steps
after it enlarge an error as they do the result: 2^-8 of the result's norm in all.
"""
from __future__ import annotations

import math

import pytest
import torch

import engraft_ngram_b200 as eb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
C = (3.4445, -4.7750, 2.0315)


def make(stack, rows, cols, kind, dtype=F32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    noise = torch.randn(stack, rows, cols, device=DEV, generator=g)
    if kind == "noise":
        x = noise
    else:
        k = min(6, rows, cols)
        u = torch.randn(stack, rows, k, device=DEV, generator=g) * 0.6 ** torch.arange(k, device=DEV)
        x = u @ torch.randn(stack, k, cols, device=DEV, generator=g)
        if kind == "strong":
            x = x + 0.1 * noise
        elif kind == "weak":
            x = x + 0.003 * noise
        elif kind == "tiny":
            x = 1e-18 * (x + 0.3 * noise)
        # "lowrank": nothing along the other directions
    return x.to(dtype)


def formula(x, steps=5, coefficients=C, eps=1e-7):
    x = x.double()
    u, s, v = torch.linalg.svd(x, full_matrices=False)
    s = s / s.square().sum(-1, keepdim=True).sqrt().clamp_min(eps)
    for i in range(steps):
        c = coefficients[i] if isinstance(coefficients[0], tuple) else coefficients
        s = s * (c[0] + c[1] * s ** 2 + c[2] * s ** 4)
    return u @ (s.unsqueeze(-1) * v)


def plain(x, steps=5, coefficients=C, eps=1e-7):
    x = x.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / x.double().square().sum((-2, -1), keepdim=True).sqrt().clamp_min(eps).float()
    for i in range(steps):
        c = coefficients[i] if isinstance(coefficients[0], tuple) else coefficients
        g = x @ x.mT
        x = c[0] * x + (c[1] * g + c[2] * (g @ g)) @ x
    return x.mT if tall else x


def check(got, x, **kw):
    want, dtype = formula(x, **kw), got.dtype
    half = torch.finfo(dtype).eps / 2
    assert torch.isfinite(got).all()
    for i in range(want.shape[0]):
        off, w = got[i].double() - want[i], want[i]
        if min(w.shape) <= 64:
            rms = float(w.square().mean().sqrt())
            tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
            bound = half * w.abs() * (1 + half) + 2.0 ** -28 * rms + tiny
            assert float((off.abs() / bound).max()) <= 1.0, i
        else:
            own = float((plain(x[i], **kw).double() - w).norm())
            bound = 2.0 ** -8 * float(w.norm()) if dtype == BF16 else 16.0 * own
            assert float(off.norm()) <= bound + half * float(w.norm()), (i, float(off.norm()), own)


SMALL = [(1, 1, 1), (3, 1, 70), (3, 70, 1), (2, 5, 7), (4, 8, 8), (5, 16, 2560), (5, 2560, 16), (3, 17, 300),
         (3, 301, 31), (2, 64, 64), (2, 64, 1000), (2, 999, 63), (70, 4, 130), (1, 40, 12800)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("shape", SMALL, ids=str)
def test_short_sides_match_the_singular_values(shape, dtype):
    for kind in ("noise", "strong"):
        x = make(*shape, kind, dtype, seed=sum(shape))
        check(eb.orthogonalize(x), x)


LONG = [(1, 65, 65), (1, 128, 128), (1, 130, 257), (2, 257, 130), (1, 256, 512), (1, 512, 384), (3, 100, 90),
        (1, 300, 1000), (1, 1001, 299), (1, 1024, 640), (2, 70, 4097),
        (1, 2200, 2100), (1, 2100, 2300), (40, 100, 130), (3, 1300, 700),  # pairs of blocks
        (1, 90, 9000), (1, 6000, 200), (2, 66, 3000)]  # sums over a long side shared by blocks


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("shape", LONG, ids=str)
def test_longer_sides_match_the_singular_values(shape, dtype):
    for kind in ("noise", "strong", "weak"):
        x = make(*shape, kind, dtype, seed=sum(shape))
        check(eb.orthogonalize(x), x)


@pytest.mark.parametrize("shape", [(2, 24, 200), (2, 200, 24), (1, 200, 150)], ids=str)
def test_rank_deficient_and_tiny_updates(shape):
    for kind in ("lowrank", "tiny"):
        x = make(*shape, kind, seed=3)
        check(eb.orthogonalize(x, eps=1e-30), x, eps=1e-30)


@pytest.mark.parametrize("shape", [(4, 12, 90), (3, 90, 120)], ids=str)
def test_zero_matrices_stay_zero_and_a_nan_stays_in_its_matrix(shape):
    x = make(*shape, "noise", seed=4)
    want = eb.orthogonalize(x)
    x[1] = 0.0
    got = eb.orthogonalize(x)
    assert (got[1] == 0).all() and torch.equal(got[0], want[0]) and torch.equal(got[2:], want[2:])
    x[1, 0, 0] = float("nan")
    got = eb.orthogonalize(x)
    assert torch.isnan(got[1]).all() and torch.equal(got[0], want[0]) and torch.equal(got[2:], want[2:])


@pytest.mark.parametrize("shape", [(2, 20, 100), (1, 150, 100)], ids=str)
def test_steps_and_coefficients(shape):
    x = make(*shape, "noise", seed=5)
    for steps, c in ((1, C), (2, (1.5, -0.5, 0.0)), (8, (1.875, -1.25, 0.375)), (3, ((3.0, -3.2, 1.2), C, (1.5, -0.5, 0.0)))):
        check(eb.orthogonalize(x, steps=steps, coefficients=c), x, steps=steps, coefficients=c)
    with pytest.raises(ValueError):
        eb.orthogonalize(x, coefficients=(9.0, 9.0, 9.0))


@pytest.mark.parametrize("shape", [(3, 10, 60), (1, 130, 70)], ids=str)
def test_in_place_again_and_a_single_matrix(shape):
    x = make(*shape, "strong", seed=6)
    want = eb.orthogonalize(x)
    assert torch.equal(eb.orthogonalize(x), want)
    assert torch.equal(eb.orthogonalize(x[0]), want[0]) or min(shape[1:]) <= 64  # other chunks: other sums
    version = x._version
    y = eb.orthogonalize(x, out=x)
    assert y is x and torch.equal(x, want) and x._version > version


def test_nothing_to_do():
    assert eb.orthogonalize(torch.zeros(0, 5, 7, device=DEV)).shape == (0, 5, 7)
    assert eb.orthogonalize(torch.zeros(3, 0, 7, device=DEV)).shape == (3, 0, 7)


def muon_formula(p, g, m, lr, beta, nesterov, wd):
    p, g, m = p.double(), g.double(), m.double()
    m = m + (1 - beta) * (g - m)
    u = g + beta * (m - g) if nesterov else m
    ratio = math.sqrt(max(1.0, p.shape[-2] / p.shape[-1]))
    return (1 - lr * wd) * p, lr * ratio, u, m


@pytest.mark.parametrize("grad_dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("shape", [(3, 16, 200), (2, 300, 24), (1, 200, 130), (1, 130, 300)], ids=str)
def test_muon_step(shape, grad_dtype):
    g = make(*shape, "strong", grad_dtype, seed=7)
    p, m = make(*shape, "noise", seed=8), make(*shape, "strong", seed=9)
    for nesterov, wd in ((True, 0.1), (False, 0.0)):
        keep, step, u, m_want = muon_formula(p, g, m, 0.05, 0.9, nesterov, wd)
        out = (torch.empty_like(p), torch.empty_like(p))
        got = eb.muon_step(p, g, m, 0.05, 0.9, nesterov, wd, out=out)
        assert got[0] is out[0] and got[1] is out[1]
        # m': a subtraction, a product and a sum, each rounded once
        assert float(((out[1].double() - m_want).abs() / (m_want.abs() + m.abs() + g.abs().float())).max()) <= 3 * 2.0 ** -24
        o_want = formula(u)
        # p': fp32's rounding of its two products and their sum, and step times the error of the orthogonalised
        # update, for which u is itself rounded (2^-22 of it, enlarged by at most c0^5 = 485 and beside the plain form's)
        own = float((plain(u.float()).double() - o_want).norm())
        rounding = 3 * 2.0 ** -24 * float((keep.abs() + step * o_want.abs()).norm())
        bound = rounding + step * (16 * own + 485 * 2.0 ** -22 * math.sqrt(shape[0]))
        assert float((out[0].double() - (keep - step * o_want)).norm()) <= bound
        p2, m2 = p.clone(), m.clone()
        assert eb.muon_step(p2, g, m2, 0.05, 0.9, nesterov, wd)[0] is p2
        assert torch.equal(p2, out[0]) and torch.equal(m2, out[1])


def test_the_optimizer_is_the_step_and_saves_its_state():
    p = [torch.nn.Parameter(make(*s, "noise", seed=i)) for i, s in enumerate(((4, 16, 100), (1, 100, 80), (2, 6, 9)))]
    q = [x.detach().clone() for x in p]
    m = [torch.zeros_like(x) for x in q]
    opt = eb.Muon(p, lr=0.02, weight_decay=0.05, momentum=0.9)
    for k in range(3):
        for i, x in enumerate(p):
            x.grad = make(*x.shape, "strong", seed=10 * k + i) if (i, k) != (2, 1) else None
        if k == 2:
            again = eb.Muon(p, lr=0.5)
            again.load_state_dict(opt.state_dict())
            opt = again
        opt.step()
        for i, x in enumerate(p):
            if x.grad is not None:
                eb.muon_step(q[i], x.grad, m[i], 0.02, 0.9, weight_decay=0.05)
    assert all(torch.equal(x.detach(), y) for x, y in zip(p, q))
    assert opt.step(lambda: torch.tensor(3.0)) == 3.0


def test_another_stream_and_a_captured_step_replayed_on_new_gradients():
    p, m = make(2, 150, 90, "noise", seed=1), make(2, 150, 90, "strong", seed=2)
    f = make(8, 12, 100, "strong", seed=3)
    grads = [make(2, 150, 90, "strong", seed=20 + k) for k in range(3)]
    q, n = p.clone(), m.clone()
    want = []
    for g in grads:
        eb.muon_step(q, g, n, 0.1)
        want.append((q.clone(), eb.orthogonalize(f * len(want))))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = eb.orthogonalize(f)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[1][1])
    g, x = grads[0].clone(), torch.zeros_like(f)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eb.muon_step(p, g, m, 0.1)
        o = eb.orthogonalize(x)
    for k in range(3):
        g.copy_(grads[k])
        x.copy_(f * k)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(p, want[k][0]) and torch.equal(o, want[k][1])


def test_two_streams_at_once():
    """Calls whose kernels overlap keep to their own workspaces: pairs of blocks, single blocks and short sides."""
    xs = [make(1, 2560, 2560, "noise", seed=40).to(BF16), make(1, 300, 1200, "noise", seed=41), make(9, 16, 400, "noise", seed=42)]
    want = [eb.orthogonalize(x) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [[] for _ in xs]
    for _ in range(6):
        for k, x in enumerate(xs):
            with torch.cuda.stream(streams[k]):
                got[k].append(eb.orthogonalize(x))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[k]) for k in range(len(xs)) for y in got[k])


def test_inference_mode_and_overlapping_arrays():
    p, g, m = (make(2, 20, 90, "noise", seed=50 + k) for k in range(3))
    want = eb.muon_step(p, g, m, 0.1, out=(torch.empty_like(p), torch.empty_like(m)))
    with torch.inference_mode():
        q, n = p.clone(), m.clone()
        eb.muon_step(q, g, n, 0.1)
        assert torch.equal(q, want[0]) and torch.equal(n, want[1])
        assert torch.equal(eb.orthogonalize(g), eb.orthogonalize(g, out=g.clone()))
    for arrays in ((p, g, p), (g, g, m), (p, m, m)):
        with pytest.raises(ValueError):
            eb.muon_step(*arrays, 0.1)


@pytest.mark.parametrize("bad", [
    lambda x: eb.orthogonalize(x.double()), lambda x: eb.orthogonalize(x.mT), lambda x: eb.orthogonalize(x[0, 0]),
    lambda x: eb.orthogonalize(x, out=x.to(BF16)), lambda x: eb.orthogonalize(x, out=x[:1]),
    lambda x: eb.orthogonalize(x, steps=0), lambda x: eb.orthogonalize(x, eps=0.0),
    lambda x: eb.muon_step(x.to(BF16), x, x, 0.1), lambda x: eb.muon_step(x, x, x.to(BF16), 0.1),
    lambda x: eb.muon_step(x, x[:1], x, 0.1), lambda x: eb.muon_step(x, x, x.cpu(), 0.1),
    lambda x: eb.muon_step(x, x, x, 0.1, out=(x, x[:1]))])
def test_refusals(bad):
    with pytest.raises(ValueError):
        bad(make(2, 6, 9, "noise"))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("c", [(12.0, -25.0, 13.5), (2.0, -14.0, 13.0)], ids=str)
def test_polynomials_near_the_limit_on_matrices_along_the_axes(c, dtype):
    """Entries of the polynomial reach its largest value, with c0 and without, where the singular vectors are axes.

    One entry a row and column, so no sums: each entry's result is s (c0 + c1 g + c2 g g), g = s s, off by the rounding
    of six operands at most (2^-22 each, in bf16 2^-12 beside an exact c0 s), of fp32's products and of its own type."""
    x = torch.zeros(3, 100, 130, device=DEV)
    x[0, 3, 5] = 2.0
    x[1].fill_diagonal_(0.25)
    x[2, 7, 0], x[2, 8, 1] = 1.0, -0.3
    x = x.to(dtype)
    s = x.double()
    s = s / s.square().sum((1, 2), keepdim=True).sqrt()
    g = s * s
    want = s * (c[0] + c[1] * g + c[2] * g * g)
    apart = s.abs() * (abs(c[1]) * g + abs(c[2]) * g * g)
    bound = 12 * 2.0 ** -22 * (c[0] * s.abs() + apart) + torch.finfo(dtype).eps / 2 * want.abs()
    if dtype == BF16:
        bound += 6 * 2.0 ** -12 * apart
    got = eb.orthogonalize(x, steps=1, coefficients=c)
    assert ((got.double() - want).abs() <= bound).all()
    with pytest.raises(ValueError):
        eb.orthogonalize(x.to(BF16), steps=1, coefficients=(14.0, -40.0, 23.0))


def iterated(x, steps=5, c=C):
    """The definition step by step in 64 bits."""
    tall = x.shape[-2] > x.shape[-1]
    x = x.double().mT if tall else x.double()
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt()
    for _ in range(steps):
        g = x @ x.mT
        x = c[0] * x + (c[1] * g + c[2] * (g @ g)) @ x
    return x.mT if tall else x


# 128 x 64 tiles whose blocks share sums, 128 x 256 tiles, a stack of them, pairs of blocks; each sum of 10^5 terms or
# more but the second
VERY_LONG = [(1, 66, 1 << 21), (150, 70, 20000), (1, 1536, 131072), (1, 140000, 1300), (1, 2600, 100001)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("shape", VERY_LONG, ids=str)
def test_the_gram_matrix_of_a_very_long_side(shape, dtype):
    """One step of X <- G X on matrices of nearly one direction, where G is a sum of squares and any loss is one-sided.

    Each MMA cuts its 16 products and the sum so far to one grid, 2^-25 of the sum: half of it for each of 16 products
    of heads (those with a remainder are 2^-11 of them) is 2^-22 of the sum so far, and 2^-23 of the whole sum, which
    grows from zero.  An accumulator takes 4096 / 16 = 256 of them in fp32: 3.1e-5, 1024 of one term in bf16: 1.2e-4.
    2^-14 for fp32 and fp16, 2^-13 for bf16 leave room for nothing but the update's own sums, of 2600 or fewer and of
    both signs.
    Without an end to a sum, 131072 terms lost 9e-4 in fp32.  The loss is looked for along the result itself,
    where errors of rounding average out.  Not all of bf16's: its values lie on the grid of the 11-bit operands, and all
    of a matrix are multiplied by the same 1 / |U|; where that is (1 + e) 2^k with |e| < 2^-12 they all round back to the
    grid, so all of X is off by e, G by 2 e and G X by 3 e, and rounding G adds 2^-12 at most: 2^-10 in all.  (The next
    test takes that away.)"""
    torch.manual_seed(160)
    x = make(*shape, "noise", seed=60) * 0.05
    x = (x + torch.randn(shape[0], shape[1], 1, device=DEV) * torch.randn(shape[0], 1, shape[2], device=DEV)).to(dtype)
    want = iterated(x, 1, (0.0, 1.0, 0.0))
    got = eb.orthogonalize(x, steps=1, coefficients=(0.0, 1.0, 0.0)).double()
    along = (got * want).sum((1, 2)) / want.square().sum((1, 2)) - 1
    assert float(along.abs().max()) <= (2.0 ** -13 + 2.0 ** -10 if dtype == BF16 else 2.0 ** -14), along
    off = (got - want).norm() / want.norm()
    assert float(off) <= (2.0 ** -8 if dtype == BF16 else 2.0 ** -13 + torch.finfo(dtype).eps / 2)
    del x, want, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(1, 1536, 131072), (1, 131072, 1536), (1, 2600, 131072)], ids=str)
def test_the_gram_matrix_of_a_very_long_side_in_bf16(shape):
    """As above, divided by a power of two (eps, above the norm), so that the operands hold bf16's values as they are.
    G's entries are rounded to 2^-12, each its own way, and average out over some 10^5 of them: 2^-13 for the sums."""
    torch.manual_seed(162)
    x = make(*shape, "noise", seed=62) * 0.05
    x = (x + torch.randn(shape[0], shape[1], 1, device=DEV) * torch.randn(shape[0], 1, shape[2], device=DEV)).to(BF16)
    eps = 2.0 ** math.ceil(math.log2(float(x.double().norm())))
    tall = shape[1] > shape[2]
    want = x.double().mT / eps if tall else x.double() / eps
    want = (want @ want.mT) @ want
    got = eb.orthogonalize(x, steps=1, coefficients=(0.0, 1.0, 0.0), eps=eps).double()
    got = got.mT if tall else got
    along = float((got * want).sum() / want.square().sum()) - 1
    assert abs(along) <= 2.0 ** -13
    del x, want, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(1, 66, 1 << 21), (1, 1536, 131072), (1, 4200, 4300), (1, 4300, 4200)], ids=str)
def test_all_steps_of_very_long_sides(shape):
    """fp32.  A sum of one sign loses 3.1e-5 (above), one of both signs less, and the five steps hand on what they lose:
    2^-13 of the result in all, and the plain fp32 form's own error."""
    x = make(*shape, "noise", seed=61)
    want, own = iterated(x), plain(x).double()
    own = float((own - want).norm())
    got = eb.orthogonalize(x).double()
    assert float((got - want).norm()) <= 2.0 ** -13 * float(want.norm()) + own
    y = x.to(BF16)
    want = iterated(y)
    assert float((eb.orthogonalize(y).double() - want).norm()) <= (2.0 ** -8 + 2.0 ** -9) * float(want.norm())
    torch.cuda.empty_cache()
