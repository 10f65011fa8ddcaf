"""The operators of a classification head, as a user's program calls them, and their plain forms.

Three operators that follow each other in a head behind the pooled feature:

* ``linear``                y = act(x W^T + b) + r                       (forward; with its gradients)
* ``dropout``               y = r + keep(seed, i) x / (1 - p)            (with its gradient)
* ``linear_cross_entropy``  cross entropy of softmax(x W^T + b)          (forward; with its gradients)

``own`` selects between the plain torch form and ``pointnetgpd_amd.head``.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ESIZE = {"f32": 4, "bf16": 2, "f16": 2}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
IGNORE = -100


# ---- cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # The first layer of the grasp classifier's head (1024 -> 512, float32, ReLU) at the evaluation batch of 64.
        dict(name="linear_fc_f32_eval", op="linear", train=False, type="f32", M=64, K=1024, N=512, act="relu",
             bias=True, residual=False),
        # The same layer in training over a scoring batch: forward and all gradients in float32.
        dict(name="linear_fc_f32_train", op="linear", train=True, type="f32", M=4096, K=1024, N=512, act="relu",
             bias=True, residual=False),
        # One sample through a wide layer when a single request is answered: the weights are all the traffic.
        dict(name="linear_single_bf16", op="linear", train=False, type="bf16", M=1, K=4096, N=4096, act="silu",
             bias=True, residual=True),
        # A wide layer over a large batch, forward only.
        dict(name="linear_wide_bf16", op="linear", train=False, type="bf16", M=8192, K=4096, N=8192, act="gelu_tanh",
             bias=True, residual=True),
        # A training step of a wide layer.
        dict(name="linear_wide_bf16_train", op="linear", train=True, type="bf16", M=8192, K=2048, N=8192, act="gelu",
             bias=True, residual=False),
        # Sizes that fit no tile and rows that start at any even address: a feature with odd extras appended.
        dict(name="linear_ragged_f16_train", op="linear", train=True, type="f16", M=1531, K=1001, N=777, act="silu",
             bias=True, residual=True),
        # Dropout behind the classifier's first layer at the training batch of 256.
        dict(name="dropout_fc_f32_train", op="dropout", train=True, type="f32", rows=256, cols=512, p=0.3,
             residual=False),
        # Dropout joined with the residual of a wide block over a large batch.
        dict(name="dropout_wide_bf16_train", op="dropout", train=True, type="bf16", rows=16384, cols=4096, p=0.1,
             residual=True),
        # The classifier's own loss: three classes at the training batch of 256.
        dict(name="loss_classes_f32_train", op="loss", train=True, type="f32", T=256, D=256, V=3, bias=True,
             smoothing=0.0, reduction="mean"),
        # A training step over a large vocabulary of labels.
        dict(name="loss_wide_bf16_train", op="loss", train=True, type="bf16", T=4096, D=2048, V=32768, bias=False,
             smoothing=0.0, reduction="mean"),
        # Float32 training with label smoothing and sizes that fit no tile.
        dict(name="loss_ragged_f32_train", op="loss", train=True, type="f32", T=1023, D=1000, V=10007, bias=True,
             smoothing=0.1, reduction="mean"),
        # Scoring a few samples against a vocabulary: one loss a row, no gradient.
        dict(name="loss_score_bf16", op="loss", train=False, type="bf16", T=16, D=4096, V=131071, bias=False,
             smoothing=0.0, reduction="none"),
    ]


def _log_int(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; one in two is made a multiple of a power of two that it
    allows, as most layers' sizes are."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        step = 1
        while step < 256 and step * 8 <= v:
            step *= 2
        v = (v + step // 2) // step * step
    return max(lo, min(hi, v))


LARGEST_FLOPS = 6 * 4096 * 2048 * 32768      # the largest listed case
LARGEST_ELEMENTS = 16384 * 4096              # the largest listed dropout


def draw(rng):
    op = rng.choice(["linear", "linear", "dropout", "loss", "loss"])
    kind = rng.choice(["f32", "bf16", "bf16", "f16"])
    train = rng.random() < 0.6
    if op == "dropout":
        while True:
            rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 16, 8192)
            if rows * cols <= LARGEST_ELEMENTS:
                break
        return dict(op=op, train=train, type=kind, rows=rows, cols=cols, p=rng.choice([0.05, 0.1, 0.3, 0.5]),
                    residual=rng.random() < 0.5)
    # float32 products cost the plain form as much but the matrix unit several times more: a lower ceiling
    cap = LARGEST_FLOPS // (8 if kind == "f32" else 1)
    while True:
        if op == "linear":
            case = dict(op=op, train=train, type=kind, M=_log_int(rng, 1, 8192), K=_log_int(rng, 16, 8192),
                        N=_log_int(rng, 16, 8192), act=rng.choice(ACTS), bias=rng.random() < 0.8,
                        residual=rng.random() < 0.5)
        else:
            case = dict(op=op, train=train, type=kind, T=_log_int(rng, 1, 8192), D=_log_int(rng, 64, 4096),
                        V=_log_int(rng, 2, 131072), bias=rng.random() < 0.5,
                        smoothing=rng.choice([0.0, 0.0, 0.1]), reduction=rng.choice(["mean", "mean", "sum", "none"]))
            if case["T"] * case["V"] > 2 ** 28:
                continue
        if work(case)["flops"] <= cap:
            return case


def work(case):
    e = ESIZE[case["type"]]
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        streams = 2 + (1 if case["residual"] else 0) + (2 if case["train"] else 0)
        return {"bytes": e * n * streams, "flops": n * (4 if case["train"] else 2)}
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        b = M * K + N * K + M * N
        b += N if case["bias"] else 0
        b += M * N if case["residual"] else 0
        f = 2 * M * N * K
        if case["train"]:
            b += M * N + M * K + N * K + (N if case["bias"] else 0)      # dy in; dx, dW, db out
            f *= 3
        return {"bytes": e * b, "flops": f}
    T, D, V = case["T"], case["D"], case["V"]
    b = e * (T * D + V * D + (V if case["bias"] else 0)) + 8 * T + 4 * (T if case["reduction"] == "none" else 1)
    f = 2 * T * D * V
    if case["train"]:
        b += e * (T * D + V * D + (V if case["bias"] else 0))
        f *= 3
    return {"bytes": b, "flops": f}


# ---- what a user's program has in hand ----------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=torch.float32) * scale).to(dt)

    state = dict(case)
    if case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        state["x"] = normal(*shape)
        state["r"] = normal(*shape) if case["residual"] else None
        state["seed"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) % 2 ** 63
        state["offset"] = seed % 1000
        leaves = ["x", "r"]
        out_shape = shape
    elif case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        # features behind a ReLU and a pool are mostly positive: half of them are here
        x = torch.randn(M, K, generator=g, device=dev, dtype=torch.float32)
        x = torch.where(x < -0.5, torch.zeros_like(x), x)
        w = torch.randn(N, K, generator=g, device=dev, dtype=torch.float32) * (1.5 / math.sqrt(K))
        b = torch.randn(N, generator=g, device=dev, dtype=torch.float32) * 0.2
        if case["act"] == "relu":
            # a ReLU's slope jumps at zero: on this grid the sums are exact in 32 bits whatever their order, and no
            # sum that is zero comes out on one side of it
            x, w, b = (torch.round(t * s) / s for t, s in ((x, 2.0 ** 6), (w, 2.0 ** 12), (b, 2.0 ** 12)))
        state["x"], state["w"] = x.to(dt), w.to(dt)
        state["b"] = b.to(dt) if case["bias"] else None
        state["r"] = normal(M, N) if case["residual"] else None
        leaves = ["x", "w", "b", "r"]
        out_shape = (M, N)
    else:
        T, D, V = case["T"], case["D"], case["V"]
        state["x"] = normal(T, D)
        state["w"] = normal(V, D, scale=2.5 / math.sqrt(D))              # logits spread over about +-10
        state["b"] = normal(V, scale=0.5) if case["bias"] else None
        # labels are skewed, as those of real data are; one in twenty rows is padding
        u = torch.rand(T, generator=g, device=dev)
        target = torch.clamp((V * u ** 3).long(), max=V - 1)
        pad = torch.rand(T, generator=g, device=dev) < 0.05
        pad[0] = False
        state["target"] = torch.where(pad, torch.full_like(target, IGNORE), target)
        leaves = ["x", "w", "b"]
        out_shape = (T,) if case["reduction"] == "none" else ()
    if case["train"]:
        for name in leaves:
            if state[name] is not None:
                state[name].requires_grad_(True)
        if case["op"] == "loss":
            # the gradient a loss receives: 1 for the mean, 1 / T for the sum, the rows' weights for rows; half
            # precision trains with a scaled loss
            gy = torch.rand(out_shape, generator=g, device=dev) if out_shape else torch.ones((), device=dev)
            gy = gy * (1024.0 if case["type"] == "f16" else 1.0)
            state["gy"] = gy if case["reduction"] == "mean" else gy / case["T"]
        else:
            state["gy"] = normal(*out_shape, scale=0.05)
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the framework's operators ------------------------------------------------------------------------------------------

def _run_own(state):
    from pointnetgpd_amd import head

    op = state["op"]
    if op == "dropout":
        y = head.dropout(state["x"], state["p"], state["seed"], state["offset"], residual=state["r"])
        leaves = ["x", "r"]
    elif op == "linear":
        act = None if state["act"] == "none" else state["act"]
        y = head.linear(state["x"], state["w"], state["b"], activation=act, residual=state["r"])
        leaves = ["x", "w", "b", "r"]
    else:
        y = head.linear_cross_entropy(state["x"], state["w"], state["target"], state["b"], ignore_index=IGNORE,
                                      label_smoothing=state["smoothing"], reduction=state["reduction"])
        leaves = ["x", "w", "b"]
    if not state["train"]:
        return [y]
    grads = torch.autograd.grad(y, [state[n] for n in leaves if state[n] is not None], state["gy"])
    return [y.detach(), *grads]


# ---- plain forms: elementary torch operations in 32 bits, rounded once ------------------------------------------------------

def _act_plain(z, act):
    """(act(z), act'(z)) in z's type."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _shift_right(z, s):
    return (z >> s) & ((1 << (64 - s)) - 1)


def _signed(c):
    return c - 2 ** 64 if c >= 2 ** 63 else c


def _mix64_plain(z):
    """The framework's 64-bit counter hash on int64 tensors, whose products wrap as unsigned ones do."""
    z = z + _signed(0x9E3779B97F4A7C15)
    z = (z ^ _shift_right(z, 30)) * _signed(0xBF58476D1CE4E5B9)
    z = (z ^ _shift_right(z, 27)) * _signed(0x94D049BB133111EB)
    return z ^ _shift_right(z, 31)


def _keep_plain(n, p, seed, offset, device):
    inner = _mix64_plain(torch.full((1,), _signed(offset), dtype=torch.int64, device=device))
    key = _mix64_plain(inner ^ _signed(seed))
    words = _mix64_plain(torch.arange((n + 1) // 2, dtype=torch.int64, device=device) + key)
    draws = torch.stack([words & 0xFFFFFFFF, _shift_right(words, 32)], dim=1).reshape(-1)[:n]
    return draws >= int(round(p * 2 ** 32))


def _run_plain(state):
    with torch.no_grad():
        op = state["op"]
        x = state["x"].detach()
        dt = x.dtype
        gy = state["gy"].float() if state["train"] else None
        r = state.get("r")
        b = state.get("b")
        if op == "dropout":
            keep = _keep_plain(x.numel(), state["p"], state["seed"], state["offset"], x.device).view_as(x)
            scale = 1 / (1 - state["p"])
            y = torch.where(keep, x.float() * scale, torch.zeros((), device=x.device))
            if r is not None:
                y = y + r.detach().float()
            out = [y.to(dt)]
            if state["train"]:
                out.append(torch.where(keep, gy * scale, torch.zeros((), device=x.device)).to(dt))
                if r is not None:
                    out.append(state["gy"])
            return out
        x32, w32 = x.float(), state["w"].detach().float()
        z = x32 @ w32.t()
        if b is not None:
            z = z + b.detach().float()
        if op == "linear":
            y, slope = _act_plain(z, state["act"])
            if r is not None:
                y = y + r.detach().float()
            out = [y.to(dt)]
            if state["train"]:
                dz = gy * slope
                out += [(dz @ w32).to(dt), (dz.t() @ x32).to(dt)]
                if b is not None:
                    out.append(dz.sum(0).to(dt))
                if r is not None:
                    out.append(state["gy"])
            return out
        target, eps, V = state["target"], state["smoothing"], z.shape[1]
        used = target != IGNORE
        index = torch.where(used, target, torch.zeros_like(target))
        top = z.max(dim=1, keepdim=True).values
        lse = top + torch.log(torch.exp(z - top).sum(dim=1, keepdim=True))
        loss = lse[:, 0] - (1 - eps) * z.gather(1, index[:, None])[:, 0]
        if eps > 0:
            loss = loss - (eps / V) * z.sum(dim=1)
        loss = torch.where(used, loss, torch.zeros_like(loss))
        count = used.sum().float()
        out = [loss if state["reduction"] == "none" else loss.sum() if state["reduction"] == "sum" else
               loss.sum() / count]
        if state["train"]:
            rows = gy / count if state["reduction"] == "mean" else gy
            rows = torch.where(used, rows.expand(z.shape[0]), torch.zeros_like(loss))
            dz = torch.exp(z - lse) - eps / V
            dz.scatter_add_(1, index[:, None], torch.full_like(lse, eps - 1))
            dz = dz * rows[:, None]
            out += [(dz @ w32).to(dt), (dz.t() @ x32).to(dt)]
            if b is not None:
                out.append(dz.sum(0).to(dt))
        return out


# ---- 64 bits, from the definitions ------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "dropout":
        return _exact_dropout(state)
    with torch.no_grad():
        return _exact_linear(state) if case["op"] == "linear" else _exact_loss(state)


def _exact_dropout(state):
    n, p = state["x"].numel(), state["p"]
    mask64 = (1 << 64) - 1

    def mix(v):
        v = (v + 0x9E3779B97F4A7C15) & mask64
        v = ((v ^ (v >> 30)) * 0xBF58476D1CE4E5B9) & mask64
        v = ((v ^ (v >> 27)) * 0x94D049BB133111EB) & mask64
        return v ^ (v >> 31)

    key = mix(state["seed"] ^ mix(state["offset"]))
    border = int(round(p * 2 ** 32))
    keep = np.empty(2 * ((n + 1) // 2), dtype=bool)
    step = 1 << 20
    with np.errstate(over="ignore"):
        for lo in range(0, keep.size // 2, step):
            hi = min(keep.size // 2, lo + step)
            v = np.arange(lo, hi, dtype=np.uint64) + np.uint64(key) + np.uint64(0x9E3779B97F4A7C15)
            v = (v ^ (v >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
            v = (v ^ (v >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
            v ^= v >> np.uint64(31)
            keep[2 * lo:2 * hi:2] = (v & np.uint64(0xFFFFFFFF)) >= border
            keep[2 * lo + 1:2 * hi:2] = (v >> np.uint64(32)) >= border
    kept = torch.from_numpy(keep[:n]).to(state["x"].device).view(state["x"].shape).double()
    y = kept * state["x"].detach().double() / (1 - p)
    if state["r"] is not None:
        y += state["r"].detach().double()
    out = [y]
    if state["train"]:
        out.append(kept * state["gy"].double() / (1 - p))
        if state["r"] is not None:
            out.append(state["gy"].double())
    return out


def _exact_linear(state):
    x, w = state["x"].detach().double(), state["w"].detach().double()
    z = torch.matmul(x, w.transpose(0, 1))
    if state["b"] is not None:
        z += state["b"].detach().double()
    act = state["act"]
    if act == "none":
        y, d = z.clone(), torch.ones_like(z)
    elif act == "relu":
        d = torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
        y = z * d
    elif act == "silu":
        e = 1 / (1 + torch.exp(-z))
        y, d = z * e, e + z * e * (1 - e)
    elif act == "gelu":
        half = torch.special.erfc(-z / math.sqrt(2)) / 2
        y, d = z * half, half + z * torch.exp(-z ** 2 / 2) / math.sqrt(2 * math.pi)
    else:
        # 0.5 (1 + tanh(u)) = sigmoid(2u)
        u2 = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        e = torch.sigmoid(u2)
        y, d = z * e, e + z * e * (1 - e) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
    if state["r"] is not None:
        y = y + state["r"].detach().double()
    out = [y]
    if state["train"]:
        dz = state["gy"].double() * d
        out.append(torch.matmul(dz, w))
        out.append(torch.matmul(dz.transpose(0, 1), x))
        if state["b"] is not None:
            out.append(torch.matmul(torch.ones(1, dz.shape[0], dtype=dz.dtype, device=dz.device), dz)[0])
        if state["r"] is not None:
            out.append(state["gy"].double())
    return out


def _exact_loss(state):
    x, w, target = state["x"].detach().double(), state["w"].detach().double(), state["target"]
    T, V, eps = x.shape[0], w.shape[0], state["smoothing"]
    count = int((target != IGNORE).sum())
    loss = torch.zeros(T, dtype=torch.float64, device=x.device)
    dx = torch.zeros_like(x)
    dw = torch.zeros_like(w)
    db = torch.zeros(V, dtype=torch.float64, device=x.device)
    step = max(1, (1 << 26) // V)
    for lo in range(0, T, step):
        rows = slice(lo, min(T, lo + step))
        y = target[rows]
        live = y != IGNORE
        z = torch.matmul(x[rows], w.transpose(0, 1))
        if state["b"] is not None:
            z += state["b"].detach().double()
        logp = torch.log_softmax(z, dim=1)
        wanted = torch.full_like(z, eps / V)
        wanted[live.nonzero()[:, 0], y[live]] += 1 - eps
        wanted[~live] = 0
        loss[rows] = -(wanted * logp).sum(dim=1)
        if state["train"]:
            g = state["gy"].double()
            g = g[rows] if state["reduction"] == "none" else g / count if state["reduction"] == "mean" else g
            dz = (torch.exp(logp) * live[:, None] - wanted) * (g[:, None] if g.dim() else g)
            dx[rows] = torch.matmul(dz, w)
            dw += torch.matmul(dz.transpose(0, 1), x[rows])
            db += dz.sum(dim=0)
    out = [loss if state["reduction"] == "none" else loss.sum() / (count if state["reduction"] == "mean" else 1)]
    if state["train"]:
        out += [dx, dw]
        if state["b"] is not None:
            out.append(db)
    return out
