"""Cases of the adapter and orthogonalisation operators: their inputs, their plain form, the framework's calls.

Four operators, two that apply low-rank adapters beside a shared projection and
two that train such factors (or the projections themselves):

  add    adapter_add: out[t] = base[t] + scale[i] * b[i] @ (a[i] @ x[t]) with i = index[t],
         the adapter of position t's request; a position without one (-1) keeps base[t]
  grad   adapter_gradients: from the gradient of out, those of x, a and b
  ortho  orthogonalize: each matrix of a stack divided by its Frobenius norm, then five
         steps X <- c0 X + (c1 G + c2 G G) X with G = X X^T
  muon   muon_step: momentum, Nesterov's update, its orthogonalisation, the parameter step

The widths are the PLE block's: 2560 embedding columns projected to 4 streams of
key and one value, 5 * 2560 = 12800 columns.  2048 is the packed batch, 256 the
number of sequences of a decode step.
"""
import math

import torch

own = False

DEVICE = "cuda"
N_EMBD, N_KV = 2560, 5 * 2560
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, BETA, WEIGHT_DECAY = 2e-2, 0.95, 0.1
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def adapters(op, name, T, K, N, rank, n, dtype, order):
    """order: "single" (one request), "segments" (packed requests one after the other), "random" (decode slots)."""
    return {"name": name, "op": op, "T": T, "K": K, "N": N, "rank": rank, "n": n, "dtype": dtype, "order": order}


def matrices(op, name, stack, rows, cols, dtype):
    return {"name": name, "op": op, "stack": stack, "rows": rows, "cols": cols, "dtype": dtype}


def listed():
    return [
        # one new token of one request: the smallest call of a serving loop
        adapters("add", "add_token", 1, N_EMBD, N_KV, 16, 16, "bf16", "single"),
        # one new token of each of 256 sequences, 40 adapters among them, in slot order
        adapters("add", "add_decode256", 256, N_EMBD, N_KV, 16, 40, "f32", "random"),
        # one packed batch of the PLE block, a few requests one after the other
        adapters("add", "add_packed2048", 2048, N_EMBD, N_KV, 16, 8, "f32", "segments"),
        # eight packed batches of prompts at rank 64
        adapters("add", "add_prompts16384", 16384, N_EMBD, N_KV, 64, 16, "bf16", "segments"),
        # widths, rank and length that no tile divides, rows that start off any alignment
        adapters("add", "add_odd", 777, 1283, 641, 11, 37, "f16", "random"),
        # the training step of four adapters over one packed batch
        adapters("grad", "grad_packed2048", 2048, N_EMBD, N_KV, 16, 4, "f32", "segments"),
        # four packed batches in 16 bits, 32 adapters
        adapters("grad", "grad_packed8192", 8192, N_EMBD, N_KV, 32, 32, "bf16", "segments"),
        adapters("grad", "grad_odd", 391, 515, 1285, 7, 19, "f32", "random"),
        # the down factors of 64 adapters, all in one call; some got no gradient
        matrices("ortho", "ortho_factors", 64, 16, N_EMBD, "f32"),
        # the update of the key projection, in 16 bits
        matrices("ortho", "ortho_key", 1, 4 * N_EMBD, N_EMBD, "bf16"),
        # the step of the value projection
        matrices("muon", "muon_value", 1, N_EMBD, N_EMBD, "f32"),
        # the step of the up factors of 40 adapters
        matrices("muon", "muon_factors", 40, N_KV, 16, "f32"),
    ]


def spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["add", "add", "grad", "ortho", "muon"])
    if op in ("add", "grad"):
        T = spread(rng, 1, 16384 if op == "add" else 8192)
        rank, n = rng.randint(1, 64), spread(rng, 1, 64)
        K, N = spread(rng, 64, N_EMBD), spread(rng, 64, N_KV)
        if rng.random() < 0.5:  # a width that vectors of 16 bytes divide
            K, N = 8 * (K // 8), 8 * (N // 8)
        n = max(1, min(n, (16384 * 16 * 32) // (T * rank)))
        return adapters(op, "drawn", T, K, N, rank, n, rng.choice(list(TYPES)), rng.choice(["segments", "random"]))
    dtype = "f32" if op == "muon" else rng.choice(list(TYPES))
    if rng.random() < 0.5:
        small, large, stack = rng.randint(1, 64), spread(rng, 64, N_KV), spread(rng, 1, 64)
    else:
        small = spread(rng, 65, N_EMBD)
        large = spread(rng, small, 4 * N_EMBD)
        stack = rng.randint(1, 3) if small * large < 1 << 20 else 1
    rows, cols = (small, large) if rng.random() < 0.5 else (large, small)
    return matrices(op, "drawn", stack, rows, cols, dtype)


def update_like(shape, gen):
    """Gradients as training gives them: a few strong directions over a floor of noise."""
    stack, rows, cols = shape
    k = min(16, rows, cols)
    u = torch.randn(stack, rows, k, device=DEVICE, generator=gen) * torch.pow(0.7, torch.arange(k, device=DEVICE))
    v = torch.randn(stack, k, cols, device=DEVICE, generator=gen)
    return 1e-3 * (torch.bmm(u, v) + 0.2 * torch.randn(shape, device=DEVICE, generator=gen))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device=DEVICE, generator=gen).mul_(std).to(dtype)

    if case["op"] in ("ortho", "muon"):
        shape = (case["stack"], case["rows"], case["cols"])
        g = update_like(shape, gen)
        if case["stack"] > 8:
            g[::7] = 0.0  # adapters that no request of the batch used
        if case["op"] == "ortho":
            return {"op": "ortho", "update": g.to(dtype)}
        param = torch.randn(shape, device=DEVICE, generator=gen) * case["cols"] ** -0.5
        momentum = 0.5 * g + update_like(shape, gen) * (g != 0)
        return {"op": "muon", "param": param, "grad": g, "momentum": momentum,
                "out": (torch.empty_like(param), torch.empty_like(param))}

    T, K, N, rank, n = (case[k] for k in ("T", "K", "N", "rank", "n"))
    if case["order"] == "segments":  # requests of unlike lengths one after the other, the last without an adapter
        request = torch.sort((torch.rand(T, device=DEVICE, generator=gen).square() * (n + 1)).long()).values
        adapter = torch.cat([torch.randperm(n, device=DEVICE, generator=gen), torch.tensor([-1], device=DEVICE)])
        index = adapter[request.clamp_max(n)]
    else:
        index = torch.randint(0, n, (T,), device=DEVICE, generator=gen)
        if case["order"] == "random":
            index[torch.rand(T, device=DEVICE, generator=gen) < 0.1] = -1
    state = {"op": case["op"], "x": normal(T, K), "a": normal(n, rank, K, std=K ** -0.5),
             "b": normal(n, N, rank, std=0.3), "index": index.to(torch.int32),
             "scale": 0.5 + 1.5 * torch.rand(n, device=DEVICE, generator=gen)}
    if case["op"] == "add":
        state["base"] = normal(T, N)
    else:
        state["grad"] = normal(T, N, std=1e-3)
    return state


def chosen(index, n):
    """[T, n]: whether position t uses adapter i."""
    return index.unsqueeze(1) == torch.arange(n, device=index.device)


def plain_add(base, x, a, b, index, scale):
    n, rank, K = a.shape
    N = b.shape[1]
    h = (x.float() @ a.float().reshape(n * rank, K).t()).view(-1, n, rank)
    h = torch.where(chosen(index, n).unsqueeze(2), h * scale.view(1, n, 1), 0.0)
    up = b.float().transpose(1, 2).reshape(n * rank, N)
    return (base.float() + h.view(-1, n * rank) @ up).to(base.dtype)


def plain_grad(grad, x, a, b, index, scale):
    n, rank, K = a.shape
    N = b.shape[1]
    xf, af, gf = x.float(), a.float().reshape(n * rank, K), grad.float()
    use = chosen(index, n).unsqueeze(2)
    h = torch.where(use, (xf @ af.t()).view(-1, n, rank) * scale.view(1, n, 1), 0.0).view(-1, n * rank)
    up = b.float().transpose(1, 2).reshape(n * rank, N)
    dh = torch.where(use, (gf @ up.t()).view(-1, n, rank) * scale.view(1, n, 1), 0.0).view(-1, n * rank)
    dx = dh @ af
    da = (dh.t() @ xf).view(n, rank, K)
    db = (h.t() @ gf).view(n, rank, N).transpose(1, 2).contiguous()
    return dx.to(x.dtype), da.to(a.dtype), db.to(b.dtype)


def plain_ortho(update):
    x = update.float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / x.square().sum((1, 2), keepdim=True).sqrt().clamp_min(EPS)
    c0, c1, c2 = COEFFICIENTS
    for _ in range(STEPS):
        g = torch.bmm(x, x.transpose(1, 2))
        x = c0 * x + torch.bmm(c1 * g + c2 * torch.bmm(g, g), x)
    return (x.transpose(1, 2) if tall else x).contiguous().to(update.dtype)


def plain_muon(param, grad, momentum):
    momentum = momentum + (1.0 - BETA) * (grad - momentum)
    update = grad + BETA * (momentum - grad)
    ratio = math.sqrt(max(1.0, param.shape[1] / param.shape[2]))
    return param * (1.0 - LR * WEIGHT_DECAY) - LR * ratio * plain_ortho(update), momentum


def run(state):
    op = state["op"]
    if own:
        import engraft_ngram_b200 as eb
        if op == "add":
            return eb.adapter_add(state["base"], state["x"], state["a"], state["b"], state["index"], state["scale"])
        if op == "grad":
            return eb.adapter_gradients(state["grad"], state["x"], state["a"], state["b"], state["index"],
                                        state["scale"])
        if op == "ortho":
            return eb.orthogonalize(state["update"])
        return eb.muon_step(state["param"], state["grad"], state["momentum"], LR, BETA, weight_decay=WEIGHT_DECAY,
                            out=state["out"])
    if op == "add":
        return plain_add(state["base"], state["x"], state["a"], state["b"], state["index"], state["scale"])
    if op == "grad":
        return plain_grad(state["grad"], state["x"], state["a"], state["b"], state["index"], state["scale"])
    if op == "ortho":
        return plain_ortho(state["update"])
    return plain_muon(state["param"], state["grad"], state["momentum"])


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["op"] in ("ortho", "muon"):
        s, m, n = case["stack"], *sorted((case["rows"], case["cols"]))
        # a step: G and G G are symmetric, so half their entries; the product with X is whole.  Where X is
        # long, the polynomial of the first G (four symmetric products a step) and one product with X.
        direct = STEPS * (m * m * n + m ** 3 + 2 * m * m * n)
        by_gram = m * m * n + STEPS * 4 * m ** 3 + 2 * m * m * n
        tensors = 2 if case["op"] == "ortho" else 5
        return {"bytes": tensors * s * m * n * size, "flops": s * min(direct, by_gram)}
    T, K, N, rank, n = (case[k] for k in ("T", "K", "N", "rank", "n"))
    # positions with an adapter, and the adapters that some position uses, as prepare() draws them
    if case["order"] == "segments":
        live = T * math.sqrt(n / (n + 1))
        used = sum(1.0 - (1.0 - math.sqrt((i + 1) / (n + 1)) + math.sqrt(i / (n + 1))) ** T for i in range(n))
    else:
        live = T if case["order"] == "single" else 0.9 * T
        used = 1 if case["order"] == "single" else n * (1.0 - (1.0 - 0.9 / n) ** T)
    factors = used * rank * (K + N) * size
    if case["op"] == "add":
        return {"bytes": live * K * size + factors + 2 * T * N * size + 4 * T, "flops": 2 * live * rank * (K + N)}
    return {"bytes": live * (K + N) * size + T * K * size + factors + n * rank * (K + N) * size + 4 * T,
            "flops": 6 * live * rank * (K + N) - 2 * live * rank * N}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("ortho", "muon"):
        if case["op"] == "ortho":
            u = s["update"].double()
        else:
            m = BETA * s["momentum"].double() + (1.0 - BETA) * s["grad"].double()
            u = BETA * m + (1.0 - BETA) * s["grad"].double()
        c0, c1, c2 = COEFFICIENTS
        each = []
        for x in u:
            x = x / max(float(torch.linalg.norm(x)), EPS)
            eye = torch.eye(min(x.shape), dtype=torch.float64, device=x.device)
            for _ in range(STEPS):
                if x.shape[0] <= x.shape[1]:
                    g = x @ x.t()
                    x = (c0 * eye + c1 * g + c2 * (g @ g)) @ x
                else:
                    g = x.t() @ x
                    x = x @ (c0 * eye + c1 * g + c2 * (g @ g))
            each.append(x)
        x = torch.stack(each)
        if case["op"] == "ortho":
            return x
        grow = LR * max(1.0, case["rows"] / case["cols"]) ** 0.5
        return (1.0 - LR * WEIGHT_DECAY) * s["param"].double() - grow * x, m
    index = s["index"].long()
    x, a, b, scale = s["x"].double(), s["a"].double(), s["b"].double(), s["scale"].double()
    if case["op"] == "add":
        out = s["base"].double().clone()
        for i in range(case["n"]):
            rows = (index == i).nonzero().flatten()
            out[rows] += scale[i] * ((x[rows] @ a[i].t()) @ b[i].t())
        return out
    grad = s["grad"].double()
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for i in range(case["n"]):
        rows = (index == i).nonzero().flatten()
        dh = scale[i] * (grad[rows] @ b[i])
        dx[rows] = dh @ a[i]
        da[i] = dh.t() @ x[rows]
        db[i] = scale[i] * (grad[rows].t() @ (x[rows] @ a[i].t()))
    return dx, da, db
