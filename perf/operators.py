"""Cases of the operators that pick a weight per row: grouped products and low-rank adapters.

Three kinds of pass, each in fp16 and bf16:

* ``grouped``  y = act(A · B[expert of the row] + bias): rows sorted by expert, ragged counts;
* ``grad``     one training step of the same product: y, dA and dB;
* ``lora``     y = act(x · W + scale · (x · down[a]) · up[a] + bias): a shared projection with the
               adapter of each row's request.

``own`` false: elementary torch operations in 32 bits, rounded once.  ``own`` true: the framework.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# Bounds of a drawn case: multiply-adds of one product, and elements of its weights.
MOST_MADS = 8192 * 4096 * 14336
MOST_WEIGHTS = 8 * 4096 * 14336


def _ext():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "infinite-dreams_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from infinite_dreams import grouped, infinite_dreams_ext
    return infinite_dreams_ext, grouped


def listed():
    return [
        # A decode step of a sparse layer: 16 requests, two experts each, most weights touched once.
        {"name": "grouped decode", "op": "grouped", "dtype": "bf16", "T": 32, "E": 64, "K": 2048, "N": 1024,
         "skew": 0.3, "mix": 1, "spare": 0, "stored": "nk", "bias": False, "act": "none"},
        # One token, two experts, small layer: the latency of the call.
        {"name": "grouped one token", "op": "grouped", "dtype": "fp16", "T": 2, "E": 8, "K": 512, "N": 1024,
         "skew": 0.3, "mix": 2, "spare": 0, "stored": "kn", "bias": False, "act": "none"},
        # A prompt batch through the first product of the experts, activation fused.
        {"name": "grouped prompt", "op": "grouped", "dtype": "bf16", "T": 8192, "E": 8, "K": 4096, "N": 14336,
         "skew": 0.4, "mix": 3, "spare": 0, "stored": "nk", "bias": False, "act": "gelu"},
        # Many experts with tens of rows each, weights stored K x N, a padded batch (rows behind the last group).
        {"name": "grouped many experts", "op": "grouped", "dtype": "fp16", "T": 4096, "E": 64, "K": 2048, "N": 1024,
         "skew": 1.0, "mix": 4, "spare": 100, "stored": "kn", "bias": True, "act": "none"},
        # Sizes no vector load likes: odd K and N, empty groups.
        {"name": "grouped odd", "op": "grouped", "dtype": "fp16", "T": 1000, "E": 5, "K": 777, "N": 1023,
         "skew": 1.5, "mix": 5, "spare": 0, "stored": "kn", "bias": True, "act": "relu"},
        # One training step of an expert layer.
        {"name": "grad large", "op": "grad", "dtype": "bf16", "T": 8192, "E": 8, "K": 4096, "N": 4096,
         "skew": 0.4, "mix": 6, "spare": 0, "stored": "kn"},
        # Fine-grained experts: short ragged reductions in dB.
        {"name": "grad many experts", "op": "grad", "dtype": "bf16", "T": 4096, "E": 64, "K": 2048, "N": 1024,
         "skew": 1.0, "mix": 7, "spare": 37, "stored": "nk"},
        {"name": "grad small", "op": "grad", "dtype": "fp16", "T": 333, "E": 7, "K": 1000, "N": 520,
         "skew": 1.2, "mix": 8, "spare": 0, "stored": "kn"},
        # Decode: 64 requests, 32 adapters in memory, one token each.
        {"name": "lora decode", "op": "lora", "dtype": "fp16", "T": 64, "L": 32, "K": 4096, "N": 4096, "R": 16,
         "run": 1, "without": 0.1, "mix": 9, "stored": "nk", "bias": False, "act": "none"},
        # One request: the latency of the call.
        {"name": "lora one token", "op": "lora", "dtype": "bf16", "T": 1, "L": 4, "K": 1024, "N": 1024, "R": 8,
         "run": 1, "without": 0.0, "mix": 10, "stored": "kn", "bias": True, "act": "none"},
        # Prompts of many requests, packed: runs of rows share an adapter.
        {"name": "lora prompt", "op": "lora", "dtype": "bf16", "T": 4096, "L": 8, "K": 4096, "N": 14336, "R": 64,
         "run": 300, "without": 0.1, "mix": 11, "stored": "nk", "bias": False, "act": "none"},
        # Prompts and single tokens in one batch, odd sizes.
        {"name": "lora mixed odd", "op": "lora", "dtype": "fp16", "T": 333, "L": 6, "K": 1000, "N": 520, "R": 24,
         "run": 20, "without": 0.2, "mix": 12, "stored": "kn", "bias": True, "act": "gelu"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """A size of a weight: mostly a multiple of 64, sometimes of 8, sometimes any."""
    n = _log(rng, low, high)
    step = rng.choice((64, 64, 64, 8, 1))
    return max(step, n // step * step)


def draw(rng):
    op = rng.choice(("grouped", "grad", "lora"))
    case = {"op": op, "dtype": rng.choice(("fp16", "bf16")), "T": _log(rng, 1, 8192)}
    if op == "lora":
        case.update(L=_log(rng, 1, 64), R=rng.choice((4, 8, 16, 24, 32, 64, 128)), run=_log(rng, 1, 1000),
                    without=rng.choice((0.0, 0.1, 0.5)))
    else:
        case.update(E=_log(rng, 1, 128), skew=rng.choice((0.0, 0.5, 1.0, 2.0)), spare=rng.choice((0, 0, 0, 50)))
    case.update(mix=rng.randrange(1 << 20), stored=rng.choice(("kn", "nk")))
    if op != "grad":
        case.update(bias=rng.random() < 0.3, act=rng.choice(("none", "none", "relu", "gelu")))
    while True:
        K, N = _size(rng, 64, 8192), _size(rng, 64, 14336)
        # a training step makes three products
        mads = case["T"] * K * N * (3 if op == "grad" else 1)
        # and the plain form pads every group to the longest
        weights = K * N * (4 if op == "grad" else 1) * case.get("E", 1)
        if mads <= MOST_MADS and weights <= MOST_WEIGHTS:
            break
    case.update(K=K, N=N)
    return case


def _counts(case):
    """Rows of each group: ragged, some empty; `spare` rows at the end belong to none."""
    rng = random.Random(case["mix"])
    share = [math.exp(case["skew"] * rng.gauss(0, 1)) for _ in range(case["E"])]
    counts = [0] * case["E"]
    for e in rng.choices(range(case["E"]), share, k=case["T"] - min(case["spare"], case["T"] // 2)):
        counts[e] += 1
    return counts


def _adapters(case):
    """The adapter of each row: runs of rows of one request, some requests without one (-1)."""
    rng = random.Random(case["mix"])
    ids = []
    while len(ids) < case["T"]:
        n = 1 if case["run"] == 1 else rng.randint(1, 2 * case["run"])
        ids += [-1 if rng.random() < case["without"] else rng.randrange(case["L"])] * n
    return ids[: case["T"]]


def _normal(g, dtype, scale, *shape):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _weight(g, dtype, stored, scale, lead, K, N):
    """A logical [lead..., K, N] weight, stored so or as the transposed view of [lead..., N, K]."""
    if stored == "kn":
        return _normal(g, dtype, scale, *lead, K, N)
    return _normal(g, dtype, scale, *lead, N, K).transpose(-1, -2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    T, K, N, op = case["T"], case["K"], case["N"], case["op"]
    state = {"op": op, "dtype": dtype, "act": case.get("act", "none"), "bias": None}
    state["x"] = _normal(g, dtype, 1.0, T, K)
    if op == "lora":
        L, R = case["L"], case["R"]
        state["W"] = _weight(g, dtype, case["stored"], K ** -0.5, (), K, N)
        state["down"] = _weight(g, dtype, case["stored"], K ** -0.5, (L,), K, R)
        state["up"] = _weight(g, dtype, case["stored"], 0.2 * R ** -0.5, (L,), R, N)
        state["scale"] = torch.rand(L, generator=g, device="cuda") + 0.5
        state["adapter"] = torch.tensor(_adapters(case), dtype=torch.int32, device="cuda")
        if case["bias"]:
            state["bias"] = _normal(g, dtype, 0.5, N)
        return state
    E, counts = case["E"], _counts(case)
    state["W"] = _weight(g, dtype, case["stored"], K ** -0.5, (E,), K, N)
    state["offsets"] = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    state["longest"] = max(counts)
    if op == "grad":
        state["dy"] = _normal(g, dtype, 1.0, T, N)
        state["x"].requires_grad_(True)
        state["W"].requires_grad_(True)
    elif case["bias"]:
        state["bias"] = _normal(g, dtype, 0.5, E, N)
    return state


def _act(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    return v


class _Groups:
    """Rows in groups padded to the longest one, and back."""

    def __init__(self, state):
        off = state["offsets"].long()
        self.T, self.E, self.longest = state["x"].shape[0], off.numel() - 1, max(state["longest"], 1)
        row = torch.arange(self.T, device=off.device)
        group = torch.searchsorted(off, row, right=True) - 1
        self.inside = (group >= 0) & (group < self.E)
        self.group = group.clamp(0, self.E - 1)
        # rows of no group go to a slot of their own behind the last
        self.slot = torch.where(self.inside, self.group * self.longest + row - off[self.group], self.E * self.longest)

    def pad(self, rows):
        flat = torch.zeros(self.E * self.longest + 1, rows.shape[1], dtype=torch.float32, device=rows.device)
        flat[self.slot] = rows * self.inside[:, None]
        return flat[:-1].view(self.E, self.longest, rows.shape[1])

    def rows(self, padded):
        flat = padded.reshape(self.E * self.longest, -1)
        return flat[self.slot.clamp_max(self.E * self.longest - 1)] * self.inside[:, None]


def _plain_grouped(state):
    at = _Groups(state)
    y = torch.bmm(at.pad(state["x"].float()), state["W"].float())
    if state["bias"] is not None:
        y = y + state["bias"].float()[:, None, :]
    return at.rows(_act(y, state["act"])).to(state["dtype"])


def _plain_grad(state):
    with torch.no_grad():
        at = _Groups(state)
        x, dy, W = at.pad(state["x"].float()), at.pad(state["dy"].float()), state["W"].float()
        y, dx, dW = torch.bmm(x, W), torch.bmm(dy, W.transpose(1, 2)), torch.bmm(x.transpose(1, 2), dy)
        return {"y": at.rows(y).to(state["dtype"]), "dx": at.rows(dx).to(state["dtype"]), "dW": dW.to(state["dtype"])}


def _plain_lora(state):
    x, down, up = state["x"].float(), state["down"].float(), state["up"].float()
    L, K, R = down.shape
    # every adapter's low-rank product, then a mask that leaves the row's own
    mine = (state["adapter"][:, None] == torch.arange(L, device=x.device)).float() * state["scale"]
    h = (x @ down.permute(1, 0, 2).reshape(K, L * R)).view(-1, L, R) * mine[:, :, None]
    y = x @ state["W"].float() + h.reshape(-1, L * R) @ up.reshape(L * R, -1)
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return _act(y, state["act"]).to(state["dtype"])


def run(state):
    if not own:
        return {"grouped": _plain_grouped, "grad": _plain_grad, "lora": _plain_lora}[state["op"]](state)
    ext, grouped = _ext()
    if state["op"] == "grouped":
        return ext.grouped_gemm(state["x"], state["W"], state["offsets"], bias=state["bias"], activation=state["act"])
    if state["op"] == "lora":
        return ext.lora_gemm(state["x"], state["W"], state["down"], state["up"], state["adapter"],
                             scale=state["scale"], bias=state["bias"], activation=state["act"])
    y = grouped.grouped_linear(state["x"], state["W"], state["offsets"])
    dx, dW = torch.autograd.grad(y, (state["x"], state["W"]), state["dy"])
    return {"y": y.detach(), "dx": dx, "dW": dW}


def work(case):
    T, K, N = case["T"], case["K"], case["N"]
    if case["op"] == "lora":
        ids = _adapters(case)
        rows, active, R = sum(i >= 0 for i in ids), len(set(i for i in ids if i >= 0)), case["R"]
        return {"bytes": 2 * (T * K + K * N + active * R * (K + N) + T * N) + 4 * T,
                "flops": 2 * T * K * N + 2 * rows * R * (K + N)}
    counts = _counts(case)
    rows, active = sum(counts), sum(c > 0 for c in counts)
    if case["op"] == "grouped":
        return {"bytes": 2 * (rows * K + active * K * N + T * N) + 4 * (case["E"] + 1), "flops": 2 * rows * K * N}
    # x, dy and the weights are read once; y, dx and every expert's dW are written
    return {"bytes": 2 * (rows * (K + N) + active * K * N + T * (K + N) + case["E"] * K * N) + 4 * (case["E"] + 1),
            "flops": 6 * rows * K * N}


def _exact_act(v, act):
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "gelu":
        return v * 0.5 * torch.erfc(-v / math.sqrt(2.0))
    return v


def exact(case, seed):
    """The definitions, group by group and adapter by adapter, in 64 bits."""
    s = prepare(case, seed)
    x = s["x"].detach().double()
    if case["op"] == "lora":
        y = x @ s["W"].double()
        ids = torch.tensor(_adapters(case), device=x.device)
        for a in range(case["L"]):
            at = (ids == a).nonzero().flatten()
            if at.numel():
                y[at] += s["scale"][a].double() * (x[at] @ s["down"][a].double() @ s["up"][a].double())
        if s["bias"] is not None:
            y += s["bias"].double()
        return _exact_act(y, s["act"])
    y = torch.zeros(case["T"], case["N"], dtype=torch.float64, device=x.device)
    W = s["W"].detach()
    if case["op"] == "grad":
        dx, dW = torch.zeros_like(x), torch.zeros(W.shape, dtype=torch.float64, device=x.device)
    first = 0
    for e, n in enumerate(_counts(case)):
        at = slice(first, first + n)
        first += n
        if not n:
            continue
        w = W[e].double()
        y[at] = x[at] @ w
        if case["op"] == "grad":
            d = s["dy"][at].double()
            dx[at] = d @ w.T
            dW[e] = x[at].T @ d
            continue
        if s["bias"] is not None:
            y[at] += s["bias"][e].double()
        y[at] = _exact_act(y[at], s["act"])
    return {"y": y, "dx": dx, "dW": dW} if case["op"] == "grad" else y
