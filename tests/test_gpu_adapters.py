"""adapter_add and its gradients on the GPU against the formula in 64 bits.

Bounds.  A product of fp32 operands in three TF32 terms is off by at most
2^-21 of it (each operand's remainder is read to 2^-22, the dropped term is
2^-24); a sum of k products in fp32 adds at most k 2^-23 of the sum of their
magnitudes (tensor-core partial sums round toward zero: a whole step).  With
M = the sum of magnitudes of the inner sums carried through the outer one, an
element is off by at most (2^-20 + (k + r) 2^-23) M, plus the half step of its
own type.  k is the length of the inner sum, r of the outer one.
"""
from __future__ import annotations

import types

import pytest
import torch

import engraft_ngram_b200 as eb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(T, K, N, rank, n, dtype, index="random", seed=0, scale=True):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g).to(dtype)

    if index == "random":
        ix = torch.randint(-1, n, (T,), device=DEV, generator=g)
    elif index == "segments":
        ix = torch.sort(torch.randint(-1, n, (T,), device=DEV, generator=g)).values
    elif index == "none":
        ix = torch.full((T,), -1, device=DEV)
    elif index == "outside":  # everything past the stack is no adapter either
        ix = torch.randint(-5, n + 5, (T,), device=DEV, generator=g)
        ix[0], ix[-1] = 2 ** 31 - 1, -2 ** 31
    else:  # one adapter for all
        ix = torch.full((T,), int(index), device=DEV)
    s = 0.5 + torch.rand(n, device=DEV, generator=g) if scale else None
    return dict(base=normal(T, N), x=normal(T, K), a=normal(n, rank, K), b=normal(n, N, rank),
                index=ix.to(torch.int32), scale=s), normal(T, N)


def formula(c, grad, mag=False):
    """out, dx, da, db in 64 bits; mag: of the magnitudes (each sum without cancellation)."""
    f = (lambda v: v.double().abs()) if mag else (lambda v: v.double())
    base, x, a, b, grad = f(c["base"]), f(c["x"]), f(c["a"]), f(c["b"]), f(grad)
    n = a.shape[0]
    out, dx, da, db = base.clone(), torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for i in range(n):
        t = (c["index"] == i).nonzero().flatten()
        s = 1.0 if c["scale"] is None else float(c["scale"][i])
        h, dh = s * (x[t] @ a[i].T), s * (grad[t] @ b[i])
        out[t] += h @ b[i].T
        dx[t] = dh @ a[i]
        da[i] = dh.T @ x[t]
        db[i] = grad[t].T @ h
    return out, dx, da, db


def check(got, want, mag, k, dtype):
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bound = (2.0 ** -20 + k * 2.0 ** -23) * mag * (1 + half) + half * want.abs() + tiny
    off = (got.double() - want).abs() / bound
    assert got.dtype == dtype and torch.isfinite(got).all()
    assert float(off.max() if off.numel() else 0) <= 1.0, float(off.max())


CASES = [
    (1, 2560, 12800, 16, 4, BF16, "0"), (1, 64, 40, 1, 1, F32, "0"), (3, 1, 1, 1, 2, F32, "random"),
    (256, 512, 640, 16, 40, F32, "random"), (300, 256, 384, 32, 3, BF16, "segments"),
    (129, 130, 77, 11, 5, F16, "random"), (517, 97, 515, 7, 9, BF16, "random"), (200, 96, 72, 24, 2, F32, "segments"),
    (65, 264, 136, 64, 1, BF16, "0"), (260, 264, 136, 64, 2, F32, "segments"), (130, 64, 96, 128, 3, F32, "random"),
    (130, 64, 96, 100, 3, F16, "segments"), (90, 72, 1000, 33, 90, F32, "random"), (64, 64, 64, 8, 3, F32, "none"),
    (64, 64, 64, 8, 3, BF16, "outside"), (2049, 80, 48, 16, 5, F32, "random"), (33, 40, 24, 16, 300, F32, "random"),
    (5000, 16, 16, 4, 2000, F32, "random"),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_gradients_match_the_formula(case):
    T, K, N, rank, n, dtype, index = case
    c, grad = make(*case, scale=T % 2 == 0)
    want, mag = formula(c, grad), formula(c, grad, mag=True)
    out = eb.adapter_add(**c)
    check(out, want[0], mag[0], K + rank, dtype)
    dx, da, db = eb.adapter_gradients(grad, c["x"], c["a"], c["b"], c["index"], c["scale"])
    check(dx, want[1], mag[1], N + rank, dtype)
    check(da, want[2], mag[2], N + T, dtype)
    check(db, want[3], mag[3], K + T, dtype)
    again = eb.adapter_add(**c)
    assert torch.equal(out, again)
    assert all(torch.equal(u, v) for u, v in zip((dx, da, db), eb.adapter_gradients(
        grad, c["x"], c["a"], c["b"], c["index"], c["scale"])))


# many positions and rows on 16 bytes, ranks that end inside 16, widths that end inside a stage and inside 128 bytes
WIDE = [(1500, 96, 264, 16, 3, F32, "random"), (1300, 64, 520, 12, 2, F32, "segments"), (1200, 128, 100, 32, 4, F32, "random"),
        (1100, 64, 1300, 64, 3, F32, "random"), (1400, 72, 264, 128, 2, F32, "random"),
        (1500, 128, 264, 16, 3, BF16, "random"), (1300, 64, 520, 8, 2, BF16, "segments"), (1200, 136, 104, 32, 4, BF16, "random"),
        (1100, 64, 1304, 64, 3, BF16, "random"), (1400, 72, 264, 128, 2, BF16, "segments"), (1030, 64, 264, 24, 1, BF16, "0"),
        (1500, 128, 264, 16, 3, F16, "random"), (1200, 136, 104, 40, 4, F16, "segments"), (1100, 64, 776, 128, 3, F16, "random"),
        (20000, 64, 136, 16, 5, BF16, "segments"), (9000, 64, 72, 16, 2, F32, "random"), (1100, 64, 264, 16, 2, F32, "none")]


@pytest.mark.parametrize("case", WIDE, ids=str)
def test_many_positions(case):
    test_forward_and_gradients_match_the_formula(case)
    c, _ = make(*case)
    want = eb.adapter_add(**c)
    held = c["base"].clone()
    assert torch.equal(eb.adapter_add(held, *list(c.values())[1:], out=held), want)
    wide = torch.full((case[0], case[2] + 24), 7.0, dtype=case[5], device=DEV)
    eb.adapter_add(**c, out=wide[:, 8:8 + case[2]])
    assert torch.equal(wide[:, 8:8 + case[2]], want) and (wide[:, :8] == 7).all() and (wide[:, 8 + case[2]:] == 7).all()
    zeros = {**c, "base": torch.zeros_like(c["base"])}
    assert torch.equal(eb.adapter_add(None, *list(c.values())[1:]), eb.adapter_add(**zeros))


# as much work as the tensor-memory kernel takes, at each of its operand layouts (rows of 64, 128 and more bytes of the
# rank), ranks that end inside one and widths that end inside a stage
HUGE = [(96003, 40, 1072, 24, 3, F32, "random"), (50001, 40, 1040, 40, 2, F32, "segments"), (100001, 64, 1056, 32, 5, BF16, "random"),
        (50007, 64, 1056, 48, 3, F16, "segments"), (26001, 72, 1056, 128, 9, BF16, "random"), (26001, 72, 1056, 104, 2, F16, "segments"),
        (100001, 64, 1056, 24, 1, F16, "0"), (50001, 40, 1056, 64, 4, BF16, "outside")]


@pytest.mark.parametrize("case", HUGE, ids=str)
def test_much_work(case):
    test_many_positions(case)
    c, _ = make(*case)
    c["x"][::5] *= 100 if case[5] == F16 else 1e4
    c["x"][1::5] /= 100 if case[5] == F16 else 1e4
    if case[5] == F16:
        c["b"] /= 64  # keeps the results inside the type
    check(eb.adapter_add(**c), formula(c, _)[0], formula(c, _, mag=True)[0], case[1] + case[3], case[5])


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_large_and_small_positions_side_by_side(dtype):
    """One position's values 1e4 times another's: each keeps its own accuracy."""
    c, grad = make(1200, 64, 256, 16, 2, dtype, "random", seed=12)
    c["x"][::5] *= 100 if dtype == F16 else 1e4
    c["x"][1::5] /= 100 if dtype == F16 else 1e4
    c["base"].zero_()
    if dtype == F16:
        c["b"] /= 64  # keeps the results inside the type
    check(eb.adapter_add(**c), formula(c, grad)[0], formula(c, grad, mag=True)[0], 80, dtype)


def test_rows_without_an_adapter_keep_base_bit_for_bit_and_their_inputs_are_not_read():
    c, grad = make(100, 64, 48, 8, 4, F32, "random", seed=3)
    c["index"][::3] = -1
    free = c["index"] < 0
    c["x"][free] = float("nan")
    c["base"][free] = float("inf")
    grad[free] = float("nan")
    out = eb.adapter_add(**c)
    dx, da, db = eb.adapter_gradients(grad, c["x"], c["a"], c["b"], c["index"], c["scale"])
    assert torch.equal(out[free], c["base"][free]) and torch.isfinite(out[~free]).all()
    assert (dx[free] == 0).all()
    assert torch.isfinite(dx).all() and torch.isfinite(da).all() and torch.isfinite(db).all()


def test_in_place_without_base_and_into_a_view():
    c, _ = make(77, 96, 136, 16, 3, BF16, "random", seed=4)
    want = eb.adapter_add(**c)
    wide = torch.zeros(77, 200, dtype=BF16, device=DEV)
    wide[:, 8:144] = c["base"]
    got = eb.adapter_add(wide[:, 8:144], c["x"], c["a"], c["b"], c["index"], c["scale"], out=wide[:, 8:144])
    assert torch.equal(got, want) and (wide[:, :8] == 0).all() and (wide[:, 144:] == 0).all()
    c["base"] = torch.zeros_like(c["base"])
    assert torch.equal(eb.adapter_add(**c), eb.adapter_add(None, *list(c.values())[1:]))


@pytest.mark.parametrize("shift", [1, 3])
def test_unaligned_rows_match_aligned_ones(shift):
    c, grad = make(150, 64, 48, 8, 4, BF16, "random", seed=5)
    odd = {k: torch.empty(150, v.shape[1] + 5, dtype=BF16, device=DEV)[:, shift:shift + v.shape[1]].copy_(v)
           for k, v in (("x", c["x"]), ("base", c["base"]), ("grad", grad))}
    want, mag = formula(c, grad), formula(c, grad, mag=True)
    rest = (c["a"], c["b"], c["index"], c["scale"])
    check(eb.adapter_add(odd["base"], odd["x"], *rest), want[0], mag[0], 72, BF16)
    for got, w, m in zip(eb.adapter_gradients(odd["grad"], odd["x"], *rest), want[1:], mag[1:]):
        check(got, w, m, 250, BF16)


def test_autograd_matches_the_gradients_and_differences():
    c, grad = make(60, 40, 56, 12, 3, F32, "random", seed=6)
    leaves = {k: c[k].clone().requires_grad_() for k in ("base", "x", "a", "b")}
    out = eb.adapter_add(leaves["base"], leaves["x"], leaves["a"], leaves["b"], c["index"], c["scale"])
    out.backward(grad)
    dx, da, db = eb.adapter_gradients(grad, c["x"], c["a"], c["b"], c["index"], c["scale"])
    assert torch.equal(leaves["base"].grad, grad) and torch.equal(leaves["x"].grad, dx)
    assert torch.equal(leaves["a"].grad, da) and torch.equal(leaves["b"].grad, db)
    # the product is linear in each argument, so a central difference is its derivative: what is left
    # is rounding, of 2^-20 + (K + rank) 2^-23 of the magnitudes on either side
    mag = formula(c, grad, mag=True)[0]
    for k in ("x", "a", "b"):
        d = torch.randn_like(c[k])
        up, down = eb.adapter_add(**{**c, k: c[k] + d}), eb.adapter_add(**{**c, k: c[k] - d})
        slope = float(((up.double() - down.double()) / 2 * grad.double()).sum())
        want = float((leaves[k].grad.double() * d.double()).sum())
        wider = formula({**c, k: c[k].abs() + d.abs()}, grad, mag=True)[0]
        bound = (2.0 ** -20 + 120 * 2.0 ** -23) * float(((mag + 2 * wider) * grad.double().abs()).sum())
        assert abs(slope - want) <= bound, k


def test_only_the_gradients_asked_for():
    c, grad = make(60, 40, 56, 12, 3, F32, "random", seed=7)
    full = eb.adapter_gradients(grad, c["x"], c["a"], c["b"], c["index"], c["scale"])
    for k, i in (("x", 0), ("a", 1), ("b", 2)):
        leaf = c[k].clone().requires_grad_()
        eb.adapter_add(**{**c, k: leaf}).backward(grad)
        assert torch.equal(leaf.grad, full[i])
    leaf = c["x"].clone().requires_grad_()
    out = eb.adapter_add(None, leaf, c["a"], c["b"], c["index"])
    (g,) = torch.autograd.grad(out.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):  # once differentiable
        g.sum().backward()


def test_nothing_to_do():
    c, grad = make(0, 40, 56, 12, 3, F32, "random")
    assert eb.adapter_add(**c).shape == (0, 56)
    dx, da, db = eb.adapter_gradients(grad, c["x"], c["a"], c["b"], c["index"], c["scale"])
    assert dx.shape == (0, 40) and (da == 0).all() and (db == 0).all()
    c, grad = make(6, 40, 56, 12, 1, F32, "none")
    c["a"], c["b"], c["scale"] = c["a"][:0], c["b"][:0], None
    assert torch.equal(eb.adapter_add(**c), c["base"])
    dx, da, db = eb.adapter_gradients(grad, c["x"], c["a"], c["b"], c["index"])
    assert (dx == 0).all() and da.shape == (0, 12, 40) and db.shape == (0, 56, 12)


def test_another_stream_and_a_captured_call_replayed_on_new_inputs():
    c, grad = make(256, 128, 160, 16, 12, F32, "random", seed=8)
    d, _ = make(256, 128, 160, 16, 12, F32, "segments", seed=9)
    want_c, want_d = eb.adapter_add(**c), eb.adapter_add(**d)
    grads_d = eb.adapter_gradients(grad, d["x"], d["a"], d["b"], d["index"], d["scale"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = eb.adapter_add(**c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want_c)
    held = {k: v.clone() for k, v in c.items()}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = eb.adapter_add(**held)
        grads = eb.adapter_gradients(grad, held["x"], held["a"], held["b"], held["index"], held["scale"])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want_c)
    for k in held:
        held[k].copy_(d[k])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want_d) and all(torch.equal(u, v) for u, v in zip(grads, grads_d))


def test_two_streams_at_once():
    """Calls whose kernels overlap keep to their own workspaces: planned and small batches, both directions."""
    cases = [make(2000, 256, 1024, 16, 3, BF16, "segments", seed=30), make(300, 512, 640, 16, 20, BF16, "random", seed=31)]
    want = [(eb.adapter_add(**c), *eb.adapter_gradients(g, c["x"], c["a"], c["b"], c["index"], c["scale"]))
            for c, g in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for k, (c, g) in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                got[k].append((eb.adapter_add(**c),
                               *eb.adapter_gradients(g, c["x"], c["a"], c["b"], c["index"], c["scale"])))
    torch.cuda.synchronize()
    for k in range(2):
        for run in got[k]:
            assert all(torch.equal(u, v) for u, v in zip(run, want[k]))


def test_hundred_thousands_of_positions():
    test_forward_and_gradients_match_the_formula((200003, 24, 40, 8, 3, F32, "random"))
    test_forward_and_gradients_match_the_formula((131072, 32, 64, 16, 2, BF16, "segments"))


@pytest.mark.parametrize("T", [60, 1100])
def test_the_largest_stack_of_adapters(T):
    c, grad = make(T, 24, 40, 4, 3, F32, "random", seed=33)
    want, mag = formula(c, grad), formula(c, grad, mag=True)
    used = torch.tensor([0, 9000, 16383], device=DEV)
    d = dict(c)
    for k in ("a", "b", "scale"):
        d[k] = torch.full((16384, *c[k].shape[1:]), float("nan"), device=DEV)
        d[k][used] = c[k]
    d["index"] = torch.where(c["index"] < 0, -1, used[c["index"].clamp(min=0)]).to(torch.int32)
    check(eb.adapter_add(**d), want[0], mag[0], 24 + 4, F32)
    dx, da, db = eb.adapter_gradients(grad, d["x"], d["a"], d["b"], d["index"], d["scale"])
    check(dx, want[1], mag[1], 40 + 4, F32)
    check(da[used], want[2], mag[2], 40 + T, F32)
    check(db[used], want[3], mag[3], 24 + T, F32)
    others = torch.ones(16384, dtype=torch.bool, device=DEV)
    others[used] = False
    assert (da[others] == 0).all() and (db[others] == 0).all()


@pytest.mark.parametrize("T", [40, 1500])
def test_inference_mode_and_an_output_that_needs_gradients(T):
    c, _ = make(T, 64, 96, 8, 3, F32, "random", seed=32)
    want = eb.adapter_add(**c)
    with torch.inference_mode():
        assert torch.equal(eb.adapter_add(**c), want)
        held = c["base"].clone()
        assert torch.equal(eb.adapter_add(**{**c, "base": held}, out=held), want)
    with pytest.raises(ValueError, match="requires grad"):
        eb.adapter_add(**c, out=torch.nn.Parameter(c["base"].clone()))


@pytest.mark.parametrize("bad, text", [
    (lambda c: dict(x=c["x"].double()), "x:"), (lambda c: dict(a=c["a"][:, :, :-1]), "a "),
    (lambda c: dict(a=c["a"].transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
    (lambda c: dict(b=c["b"].to(BF16)), "b:"), (lambda c: dict(index=c["index"].long()), "index"),
    (lambda c: dict(index=c["index"][:-1]), "index"), (lambda c: dict(scale=c["scale"].double()), "scale"),
    (lambda c: dict(scale=c["scale"][:-1]), "scale"), (lambda c: dict(base=c["base"][:, :-1]), "base"),
    (lambda c: dict(base=c["base"].cpu()), "base"), (lambda c: dict(base=c["base"][:1].expand(20, -1)), "strides"),
    (lambda c: dict(x=c["x"].t().contiguous().t()), "strides"),
    (lambda c: dict(a=c["a"].repeat(1, 17, 1), b=c["b"].repeat(1, 1, 17)), "rank")])
def test_refusals(bad, text):
    c, _ = make(20, 16, 24, 8, 3, F32)
    with pytest.raises(ValueError, match=text):
        eb.adapter_add(**{**c, **bad(c)})


PLE_WEIGHTS = ("w_key", "w_value", "norm_key", "norm_query", "norm_conv", "conv1d")


def ple_case(T=37, n=32, hc=3, H=5, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(11)
    r = lambda *s, std=1.0: torch.randn(*s, device=DEV, generator=g) * std  # noqa: E731
    w = types.SimpleNamespace(w_key=r(hc * n, n, std=n ** -0.5), w_value=r(n, n, std=n ** -0.5), norm_key=r(hc, n),
                              norm_query=r(hc, n), norm_conv=r(hc, n), conv1d=r(hc * n, 4, std=0.5))
    hp = types.SimpleNamespace(hc_mult=hc, n_embd=n, f_norm_rms_eps=1e-6, ple_ngram_size=3)
    ad = eb.PleAdapters(r(4, 8, n, std=n ** -0.5), r(4, hc * n + n, 8, std=0.3),
                        torch.randint(-1, 4, (T,), device=DEV, generator=g).to(torch.int32),
                        0.5 + torch.rand(4, device=DEV, generator=g))
    return r(T, n), r(T, hc, n), w, r(H, hc, n), hp, ad


def ple_formula(emb, hidden, w, hist, hp, ad):
    """The block in plain torch, in the type of its inputs, with each position's own projection W + s b a."""
    T, n = emb.shape
    hc, K, dil = hp.hc_mult, w.conv1d.shape[1], hp.ple_ngram_size
    kv = emb @ torch.cat([w.w_key, w.w_value]).T
    live = ad.index >= 0
    i = ad.index.clamp_min(0).long()
    delta = torch.einsum("tfr,trk,tk->tf", ad.b[i], ad.a[i], emb) * ad.scale.to(emb.dtype)[i].unsqueeze(1)
    kv = kv + torch.where(live.unsqueeze(1), delta, 0.0)
    key, value = kv[:, :hc * n].reshape(T, hc, n), kv[:, hc * n:]

    def rms(x, g):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + hp.f_norm_rms_eps) * g.reshape(hc, n)

    s = (rms(key, w.norm_key) * rms(hidden, w.norm_query)).sum(-1) / n ** 0.5
    gated = value.unsqueeze(1) * torch.sigmoid(torch.sign(s) * s.abs().clamp_min(1e-6).sqrt()).unsqueeze(-1)
    full = torch.cat([hist, rms(gated, w.norm_conv)]).reshape(-1, hc * n)
    back = torch.nn.functional.pad(full, (0, 0, (K - 1) * dil, 0))
    H = hist.shape[0]
    conv = sum(back[H + k * dil:H + k * dil + T] * w.conv1d[:, k] for k in range(K))
    return hidden + gated + torch.nn.functional.silu(conv).reshape(T, hc, n)


# the block's own tests hold it to 2e-5 of the largest magnitude in fp32 (its norms and its gate enlarge the
# projections' rounding); the adapters' rounding stands beside the projections' and is no larger
PLE_TOL = 2e-5


@pytest.mark.parametrize("projection", ["3xtf32", "fp32", "tcgen05"])
def test_ple_block_with_adapters_trains_their_factors(monkeypatch, projection):
    from engraft_ngram_b200 import ple
    monkeypatch.setattr(ple, "PROJECTION", projection)
    emb, hidden, w, hist, hp, ad = ple_case()
    free, _ = eb.ple_forward(emb, hidden, w, hist, hp)
    out, tail = eb.ple_forward(emb, hidden, w, hist, hp, adapters=ad)
    none = ad.index < 0
    assert not torch.equal(out, free) and none.any()
    up = lambda v: v.double()  # noqa: E731
    w64 = types.SimpleNamespace(**{k: up(getattr(w, k)) for k in PLE_WEIGHTS})
    leaves = {k: up(v).requires_grad_() for k, v in (("emb", emb), ("hidden", hidden), ("hist", hist), ("a", ad.a),
                                                    ("b", ad.b))}
    ad64 = eb.PleAdapters(leaves["a"], leaves["b"], ad.index, ad.scale)
    want = ple_formula(leaves["emb"], leaves["hidden"], w64, leaves["hist"], hp, ad64)
    assert float((out.double() - want).abs().max()) <= PLE_TOL * float(want.abs().max())
    grad = torch.randn(out.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    want.backward(up(grad))
    mine = {k: v.clone().requires_grad_() for k, v in (("emb", emb), ("hidden", hidden), ("hist", hist), ("a", ad.a),
                                                      ("b", ad.b))}
    diag = {}
    got, _ = eb.ple_forward(mine["emb"], mine["hidden"], w, mine["hist"], hp, diag=diag,
                            adapters=eb.PleAdapters(mine["a"], mine["b"], ad.index, ad.scale))
    assert torch.equal(got.detach(), out)
    got.backward(grad)
    for k in mine:
        ref = leaves[k].grad
        assert float((mine[k].grad.double() - ref).abs().max()) <= 5 * PLE_TOL * float(ref.abs().max()), k
    # only the factors are trained, and stepped
    a, b = torch.nn.Parameter(ad.a.clone()), torch.nn.Parameter(ad.b.clone())
    opt = eb.Muon([a, b], lr=0.01, weight_decay=0.0)
    eb.ple_forward(emb, hidden, w, hist, hp, adapters=eb.PleAdapters(a, b, ad.index, ad.scale))[0].backward(grad)
    assert torch.equal(a.grad, mine["a"].grad) and torch.equal(b.grad, mine["b"].grad)
    opt.step()
    want_a, _ = eb.muon_step(ad.a.clone(), mine["a"].grad, torch.zeros_like(ad.a), 0.01)
    assert torch.equal(a.detach(), want_a) and not torch.equal(b.detach(), ad.b)


def test_ple_block_refuses_adapters_of_other_widths():
    emb, hidden, w, hist, hp, ad = ple_case()
    with pytest.raises(ValueError, match="adapters"):
        eb.ple_forward(emb, hidden, w, hist, hp, adapters=eb.PleAdapters(ad.a, ad.b[:, :-1], ad.index))
    with pytest.raises(ValueError, match="index"):
        eb.ple_forward(emb, hidden, w, hist, hp, adapters=eb.PleAdapters(ad.a, ad.b, ad.index[:-1]))


def test_second_derivatives_of_the_ple_block_are_an_error_and_not_left_out():
    emb, hidden, w, hist, hp, ad = ple_case()
    leaves = [v.clone().requires_grad_() for v in (emb, ad.a, ad.b)]
    for k in (slice(0, 1), slice(1, 3), slice(0, 3)):  # emb alone is the block without adapters' factors
        use = [v if i in range(3)[k] else v.detach() for i, v in enumerate(leaves)]
        adapters = None if k == slice(0, 1) else eb.PleAdapters(use[1], use[2], ad.index, ad.scale)
        out, _ = eb.ple_forward(use[0], hidden, w, hist, hp, adapters=adapters)
        grads = torch.autograd.grad(out.square().sum(), leaves[k], create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            sum(g.sum() for g in grads).backward()


def test_scale_of_the_weight_gradients_over_more_positions_than_32_bits_of_elements():
    """fp16 at rank 65: 2^26 positions of one adapter are 2^31 fours of h, whose largest magnitude sets their scale.

    h is 2^17, beyond fp16 unless scaled, and of few significant bits, so that every product is exact: db sums the 40
    positions whose gradient is not zero, and da (whose dh they alone have) 40 terms more."""
    T, rank = (1 << 26) + 7, 65
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GB of device memory")
    x = torch.full((T, 1), 512.0, dtype=F16, device=DEV)
    a = torch.full((1, rank, 1), 256.0, dtype=F16, device=DEV)
    a[0, ::2] = -128.0
    b = torch.full((1, 1, rank), 2.0 ** -4, dtype=F16, device=DEV)
    grad = torch.zeros(T, 1, dtype=F16, device=DEV)
    grad[T % (T // 39) - 1::T // 39] = 2.0 ** -8  # 40, the last position among them
    assert int(torch.count_nonzero(grad)) == 40
    dx, da, db = eb.adapter_gradients(grad, x, a, b, torch.zeros(T, dtype=torch.int32, device=DEV))
    assert (db[0, 0].float() == 40 * 2.0 ** -8 * 512 * a[0, :, 0].float()).all()
    assert (da.float() == 40 * 2.0 ** -12 * 512).all()
    dh = 2.0 ** -12 * float(a.double().sum())
    assert (dx.float() == (grad != 0) * dh).all()
    torch.cuda.empty_cache()


def formula_with_sums_in_fp32(c, grad):
    """The formula in 64 bits where its sums and products in fp32 are finite, and those where they are not: h, dh and
    every sum are fp32 by definition, so a product beyond fp32 is an infinity, and one of each sign make a NaN."""
    def evaluate(up):
        base, x, a, b, grad_ = (up(v) for v in (c["base"], c["x"], c["a"], c["b"], grad))
        out, dx, da, db = base.clone(), torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
        for i in range(a.shape[0]):
            t = (c["index"] == i).nonzero().flatten()
            h, dh = (c["scale"][i] * v for v in (x[t] @ a[i].T, grad_[t] @ b[i]))
            out[t] += h @ b[i].T
            dx[t] = dh @ a[i]
            da[i] = dh.T @ x[t]
            db[i] = grad_[t].T @ h
        return out, dx, da, db
    return [torch.where(torch.isfinite(v), w, v.double()) for v, w in zip(evaluate(torch.Tensor.float),
                                                                          evaluate(torch.Tensor.double))]


def same_as_formula(got, want, mag, k, dtype):
    """NaN and infinities where the formula has them (or leaves the type), and check()'s bound elsewhere."""
    half = torch.finfo(dtype).eps / 2
    rounded = want.to(dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(rounded))
    there = torch.isinf(rounded)
    assert torch.equal(torch.isinf(got), there) and torch.equal(got[there], rounded[there])
    ok = torch.isfinite(rounded)
    bound = (2.0 ** -20 + k * 2.0 ** -23) * mag[ok] * (1 + half) + half * want[ok].abs()
    bound += torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert ((got[ok].double() - want[ok]).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("shape", [(60, 40, 56, 12), (100, 41, 57, 11), (1100, 41, 57, 11), (1500, 96, 264, 16), (1500, 64, 136, 48),
                                   (1400, 72, 264, 100), (26001, 72, 1056, 128), (50001, 40, 1056, 40)], ids=str)
def test_values_that_are_not_finite_or_near_the_types_largest(shape, dtype):
    """Infinities and NaN in x, grad, base and the factors, and the type's largest values where products of them are
    finite: as the formula has them, in their own adapters only."""
    T, K, N, rank = shape
    n = 8 if T > 200 else 7
    c, grad = make(T, K, N, rank, n, dtype, "random", seed=70)
    inf, most, small = float("inf"), torch.finfo(dtype).max, 2.0 ** -14 if dtype == F16 else 2.0 ** -100
    c["scale"].copy_(2.0 ** torch.arange(n, device=DEV).remainder(3))
    c["index"][:n] = torch.arange(n, device=DEV)
    at = [(c["index"] == i).nonzero().flatten() for i in range(n)]
    c["x"][at[0][0], 3] = inf
    c["x"][at[0][-1], 5] = -inf
    c["x"][at[1][0], 0] = float("nan")
    c["x"][at[2][0], 7] = most  # an infinity in TF32's 11 bits
    c["a"][2, :, 7] = small
    grad[at[3][0], 2] = -inf
    grad[at[3][-1], 4] = most
    c["b"][3, 4] = small
    c["a"][4, 0, 6] = most
    c["x"][at[4], 6] = small
    c["b"][5, 9, 1] = inf
    c["b"][5, 8, 0] = -most
    c["base"][at[6], 1] = -inf
    c["base"][at[6][0], 2] = float("nan")
    want, mag = formula_with_sums_in_fp32(c, grad), formula(c, grad, mag=True)
    out = eb.adapter_add(**c)
    same_as_formula(out, want[0], mag[0], K + rank, dtype)
    if rank * K * N < 1 << 20:  # in place, where the base is overwritten
        held = c["base"].clone()
        assert torch.equal(eb.adapter_add(held, *list(c.values())[1:], out=held).nan_to_num(), out.nan_to_num())
    for k, (got, w, m, terms) in enumerate(zip(eb.adapter_gradients(grad, c["x"], c["a"], c["b"], c["index"], c["scale"]),
                                               want[1:], mag[1:], (N + rank, N + T, K + T))):
        same_as_formula(got, w, m, terms, dtype)
    assert torch.isfinite(out[at[2]]).all() and torch.isfinite(out[at[6][0], 3:]).all()


def test_one_adapter_of_rank_one_hands_on_infinities_and_large_values():
    for dtype in (F32, BF16, F16):
        x = torch.zeros(2, 8, device=DEV, dtype=dtype)
        x[0, 0], x[1, 0] = -float("inf"), torch.finfo(dtype).max
        a, b = torch.zeros(1, 1, 8, device=DEV, dtype=dtype), torch.full((1, 4, 1), 0.5, device=DEV, dtype=dtype)
        a[0, 0] = 0.25
        out = eb.adapter_add(None, x, a, b, torch.zeros(2, dtype=torch.int32, device=DEV))
        assert (out[0] == -float("inf")).all() and (out[1].double() == torch.finfo(dtype).max / 8).all()


def along(got, want):
    """How far got is along want: what is lost of sums of one sign, beside the rounding of the results."""
    return float((got.double() * want).sum() / want.square().sum()) - 1


# Truncating accumulators lose at most 2^-22 of the sum so far an MMA of 16 terms (16 products cut to a grid of 2^-25), half
# of that over a sum that grows from zero: 2^-23 a time.  h is split to 2^-17.  Sums of so many values are nearly equal,
# so the rounding of the results (half a step, 2^-8 or 2^-11) may be the same for all of them and does not average out.
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("rank", [16, 40, 100])
def test_weight_gradients_of_millions_of_positions_of_one_sign(dtype, rank):
    """16384 positions an accumulator, of which half a block's warps have each half: 512 MMAs, 2^-14, twice that for the
    two sums."""
    T, K, N, half = (1 << 22) + 5, 48, 64, torch.finfo(dtype).eps / 2
    g = torch.Generator(device=DEV).manual_seed(80)
    one = lambda *s: torch.rand(*s, device=DEV, generator=g) + 0.5  # noqa: E731
    x, a, b = one(T, K).to(dtype), (one(2, rank, K) / 64).to(dtype), (one(2, N, rank) / 64).to(dtype)
    grad = (one(T, N) * 2.0 ** -10).to(dtype)
    index = torch.ones(T, dtype=torch.int32, device=DEV)
    index[::4096] = 0
    dx, da, db = eb.adapter_gradients(grad, x, a, b, index)
    for i in range(2):
        t = (index == i).nonzero().flatten()
        xi, gi = x[t].double(), grad[t].double()
        assert abs(along(da[i], (gi @ b[i].double()).T @ xi)) <= 2.0 ** -13 + half
        assert abs(along(db[i], gi.T @ (xi @ a[i].double().T))) <= 2.0 ** -13 + half
        del xi, gi
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("T", [20, 200])
def test_widths_of_millions_of_one_sign(T, dtype):
    """2^17 columns a split, of which two groups of warps have half each: 4096 MMAs, 2^-11.  2^24 columns in 16 splits
    would be 32768 MMAs, 2^-8."""
    K, N = 1 << 24, 24
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    g = torch.Generator(device=DEV).manual_seed(81)
    x = torch.empty(T, K, dtype=dtype, device=DEV)
    for t in range(T):
        x[t] = torch.rand(K, device=DEV, generator=g) + 0.5
    a = ((torch.rand(1, 2, K, device=DEV, generator=g) + 0.5) * 2.0 ** -12).to(dtype)
    b = (torch.rand(1, N, 2, device=DEV, generator=g) * 2.0 ** -4 + 2.0 ** -4).to(dtype)
    out = eb.adapter_add(None, x, a, b, torch.zeros(T, dtype=torch.int32, device=DEV))
    h = torch.cat([x[t:t + 1].double() @ a[0].double().T for t in range(T)])
    assert abs(along(out, h @ b[0].double().T)) <= 2.0 ** -11 + torch.finfo(dtype).eps / 2
    del x
    torch.cuda.empty_cache()


def plain_gradients(c, grad):
    """dx, da and db by fp32 products, rounded once."""
    x, a, b, grad = (v.float() for v in (c["x"], c["a"], c["b"], grad))
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for i in range(a.shape[0]):
        t = (c["index"] == i).nonzero().flatten()
        s = 1.0 if c["scale"] is None else c["scale"][i]
        h, dh = s * (x[t] @ a[i].T), s * (grad[t] @ b[i])
        dx[t], da[i], db[i] = dh @ a[i], dh.T @ x[t], grad[t].T @ h
    return [v.to(c["x"].dtype) for v in (dx, da, db)]


@pytest.mark.parametrize("case", [(200003, 24, 40, 8, 3, F32, "random"), (131072, 32, 64, 16, 2, BF16, "segments"),
                                  (200003, 24, 40, 8, 3, F16, "random"), (96003, 40, 1072, 24, 3, F32, "random"),
                                  (50007, 64, 1056, 48, 3, F16, "segments"), (26001, 72, 1056, 128, 9, BF16, "random"),
                                  (150000, 32, 48, 40, 50, F32, "segments"), (150000, 33, 47, 11, 700, BF16, "random")],
                         ids=str)
def test_gradients_of_many_positions_to_the_accuracy_of_the_plain_form(case):
    """Each adapter's gradients by the 2-norm of their error, which grows as that of a sum of many roundings does: at
    most four times the plain fp32 form's (TF32 remainders are read to 2^-22 of their products, fp32 rounds to 2^-24),
    a half step of the type and, where h is split in 16 bits, 2^-17 of it.  The bound is under 2^-7 of the result (the
    half step of bf16 is 2^-8): none that misses positions would pass."""
    c, grad = make(*case, seed=90)
    dtype = case[5]
    want, plain = formula(c, grad)[1:], plain_gradients(c, grad)
    got = eb.adapter_gradients(grad, c["x"], c["a"], c["b"], c["index"], c["scale"])
    half = torch.finfo(dtype).eps / 2 + (2.0 ** -17 if dtype == BF16 else 0.0)
    for k in range(3):
        rows = [c["index"] == i for i in range(case[4])] if k == 0 else range(case[4])
        for i in rows:
            w = want[k][i]
            size = float(w.norm())
            own = float((plain[k][i].double() - w).norm()) if dtype == F32 else 2.0 ** -20 * size
            bound = 4 * own + half * size
            assert bound <= 2.0 ** -7 * size and float((got[k][i].double() - w).norm()) <= bound, (k, size, own)
    assert (got[0][c["index"] < 0] == 0).all()


@pytest.mark.parametrize("case", [(2048, 6400, 12800, 128, 3, BF16), (2048, 4096, 12800, 100, 3, F32)], ids=str)
def test_a_poisoned_adapter_leaves_the_others_their_bits(case):
    """Each result of an adapter that is all NaN is summed twice, from sums of several splits, while the other adapters'
    accumulators wait: no wait may give up, and no other row may change."""
    c, grad = make(*case, index="random", seed=95)
    before = eb.waits_given_up()
    want = eb.adapter_add(**c)
    grads = eb.adapter_gradients(grad, c["x"], c["a"], c["b"], c["index"], c["scale"])
    for k in ("a", "b"):
        c[k][1] = float("nan")
    got = eb.adapter_add(**c)
    sick = c["index"] == 1
    assert torch.isnan(got[sick]).all() and torch.equal(got[~sick], want[~sick])
    dx, da, db = eb.adapter_gradients(grad, c["x"], c["a"], c["b"], c["index"], c["scale"])
    well = [0, 2]
    assert torch.isnan(dx[sick]).all() and torch.equal(dx[~sick], grads[0][~sick])
    assert torch.equal(da[well], grads[1][well]) and torch.equal(db[well], grads[2][well])
    assert torch.isnan(da[1]).all() and torch.isnan(db[1]).all()
    assert eb.waits_given_up() == before
