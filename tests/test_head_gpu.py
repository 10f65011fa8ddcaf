"""GPU parity of the classification-head operators (pointnetgpd_amd/head.py) against their 64-bit restatement, within the
bounds that oracle/head_oracle.py derives element by element."""
import math

import pytest
import torch

from oracle import head_oracle as ho
from pointnetgpd_amd import head

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(seed, *shapes, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g) * scale for s in shapes]


def grid(t, step):
    """On a grid whose sums are exact in 32 bits: a ReLU's border is then on the same side for every order of the sum."""
    return torch.round(t / step) * step


def check(outputs, want):
    bad = {k: r for k, r in ((k, ho.worst(outputs[k], *want[k])) for k in outputs) if not r <= 1.0}
    assert not bad, bad


def linear_case(seed, M, N, K, dt, act, bias, residual):
    x, w, b, r, dy = make(seed, (M, K), (N, K), (N,), (M, N), (M, N))
    w = w / math.sqrt(K)
    if act == "relu":
        x, w, b = grid(x, 2.0 ** -6), grid(w, 2.0 ** -10), grid(b, 2.0 ** -10)
    x, w, b, r, dy = (t.to(dt) for t in (x, w, b, r, dy))
    return x, w, b if bias else None, r if residual else None, dy


def run_linear(x, w, b, r, act, dy):
    leaves = [t.cuda().requires_grad_() if t is not None else None for t in (x, w, b, r)]
    y = head.linear(*leaves[:3], activation=act, residual=leaves[3])
    used = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(("dx", "dw", "db", "dr"), leaves) if t is not None],
                     torch.autograd.grad(y, used, dy.cuda())))
    return {"y": y, **grads}


SIZES = [(1, 1, 1), (1, 16, 8), (2, 3, 5), (1, 512, 4096), (3, 1030, 200), (16, 200, 1030), (64, 64, 64), (65, 130, 67),
         (128, 256, 64), (200, 7, 1024), (257, 513, 129), (300, 777, 1001), (1023, 40, 24), (512, 384, 640)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("kind", list(TYPES))
def test_linear_and_its_gradients(kind, M, N, K):
    i = SIZES.index((M, N, K))
    act = (None, "relu", "gelu", "gelu_tanh", "silu")[i % 5]
    x, w, b, r, dy = linear_case(M + N + K, M, N, K, TYPES[kind], act, bias=i % 3 != 2, residual=i % 2 == 0)
    got = run_linear(x, w, b, r, act, dy)
    want = ho.linear(x, w, b, act, r, dy)
    if "dr" in got:
        assert torch.equal(got.pop("dr").cpu(), dy)
    assert got["y"].dtype == x.dtype
    check(got, want)


@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("kind", list(TYPES))
def test_every_activation_with_bias_and_residual(kind, act):
    x, w, b, r, dy = linear_case(5, 70, 96, 80, TYPES[kind], act, True, True)
    got = run_linear(x, w, b, r, act, dy)
    got.pop("dr")
    check(got, ho.linear(x, w, b, act, r, dy))


@pytest.mark.parametrize("M,N,K", [(2048, 1024, 512), (1500, 1100, 1300), (4096, 256, 128)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_linear_over_many_tiles(kind, M, N, K):
    x, w, b, r, dy = linear_case(17, M, N, K, TYPES[kind], "gelu", True, True)
    got = run_linear(x, w, b, r, "gelu", dy)
    got.pop("dr")
    check(got, ho.linear(x, w, b, "gelu", r, dy))


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("N,K", [(1, 8), (70, 24), (2050, 1000), (4100, 513), (513, 8200)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_linear_of_a_few_rows(kind, N, K, M):
    act = (None, "relu", "gelu", "gelu_tanh", "silu")[M - 1]
    x, w, b, r, dy = linear_case(N + K + M, M, N, K, TYPES[kind], act, True, True)
    got = run_linear(x, w, b, r, act, dy)
    got.pop("dr")
    check(got, ho.linear(x, w, b, act, r, dy))


@pytest.mark.parametrize("kind", list(TYPES))
def test_linear_takes_any_strides_and_alignment(kind):
    dt = TYPES[kind]
    M, N, K = 130, 72, 88
    x, w, b, r, dy = linear_case(23, M, N, K, dt, "silu", True, True)
    want = ho.linear(x, w, b, "silu", r, dy)

    def odd_start(t):                       # a view that starts one element into its storage
        s = torch.full((t.numel() + 1,), float("nan"), dtype=dt, device="cuda")
        s[1:] = t.reshape(-1).cuda()
        return s[1:].view(t.shape)

    def wide(t):                            # rows further apart than they are long, NaN between them
        s = torch.full((t.shape[0], t.shape[1] + 9), float("nan"), dtype=dt, device="cuda")
        s[:, 3:3 + t.shape[1]] = t.cuda()
        return s[:, 3:3 + t.shape[1]]

    def lying(t):                           # columns dense instead of rows
        return t.t().contiguous().cuda().t()

    for lay in (odd_start, wide, lying):
        xs, ws, rs, ds = (lay(t).detach().requires_grad_() for t in (x, w, r, dy))
        bs = b.cuda().requires_grad_()
        y = head.linear(xs, ws, bs, activation="silu", residual=rs)
        dx, dw, db = torch.autograd.grad(y, (xs, ws, bs), ds.detach())
        check({"y": y, "dx": dx, "dw": dw, "db": db}, want)
    # one residual row for all, one gradient value for all, and more than two dimensions
    row = r[:1].expand(M, N)
    y = head.linear(x.cuda().view(2, 65, K), w.cuda(), b.cuda(), activation="silu",
                    residual=r[:1].cuda().expand(M, N).view(2, 65, N))
    assert y.shape == (2, 65, N)
    check({"y": y.reshape(M, N)}, ho.linear(x, w, b, "silu", row, None))
    xs = x.cuda().requires_grad_()
    dx, = torch.autograd.grad(head.linear(xs, w.cuda()).float().sum(), xs)
    check({"dx": dx}, {"dx": ho.linear(x, w, None, None, None, torch.ones(M, N, dtype=dt))["dx"]})


@pytest.mark.parametrize("kind", list(TYPES))
def test_no_rows(kind):
    dt = TYPES[kind]
    x = torch.empty(0, 24, dtype=dt, device="cuda", requires_grad=True)
    w = torch.randn(16, 24, device="cuda").to(dt).requires_grad_()
    b = torch.randn(16, device="cuda").to(dt).requires_grad_()
    y = head.linear(x, w, b, activation="relu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (0, 16) and dx.shape == (0, 24) and not dw.any() and not db.any()
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    loss = head.linear_cross_entropy(x, w, t, b, reduction="sum")
    dx, dw, db = torch.autograd.grad(loss, (x, w, b))
    assert loss.item() == 0 and not dw.any() and not db.any()
    assert math.isnan(head.linear_cross_entropy(x, w, t).item())
    assert head.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)
    assert head.dropout(x, 0.5, 3).shape == (0, 24)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh", "silu"])
def test_linear_carries_infinities_and_nan_in_their_rows_only(kind, act):
    dt = TYPES[kind]
    x, w, b, _, _ = linear_case(3, 70, 40, 48, dt, act, True, False)
    x, w = x.abs() + 0.125, w.abs() + 0.125                     # one sign: an infinity stays one in every sum
    x[3, 5], x[40, 7], x[66, 0] = math.inf, -math.inf, math.nan
    y = head.linear(x.cuda(), w.cuda(), b.cuda(), activation=act).cpu()
    assert torch.isnan(y[66]).all() and (y[3] == math.inf).all()
    assert (y[40] == (-math.inf if act is None else 0.0)).all()
    rest = [i for i in range(70) if i not in (3, 40, 66)]
    want = ho.linear(x[rest], w, b, act, None, None)["y"]
    assert ho.worst(y[rest], *want) <= 1.0


def test_float32_products_keep_the_types_range():
    """Operands near both ends of float32's range, whose products lie inside it."""
    x, w = make(2, (130, 64), (130, 64))
    big, small = (x * 2.0 ** 100), (w * 2.0 ** -100)
    for a, b in ((big, small), (small, big), (x * 2.0 ** -60, w * 2.0 ** -60), (x * 2.0 ** 126 / 8, w * 2.0 ** -20)):
        y = head.linear(a.cuda(), b.cuda())
        want, bound = ho.linear(a, b, None, None, None, None)["y"]
        assert ho.worst(y, want, bound + 2.0 ** -149 * 64) <= 1.0
    top = torch.full((1, 8), torch.finfo(torch.float32).max)
    one = torch.zeros(1, 8)
    one[0, 0] = 1.0
    assert head.linear(top.cuda(), one.cuda()).item() == top[0, 0].item()


# ---- dropout --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", [(1,), (1, 1), (3, 5), (7, 1), (256, 512), (33, 1001), (5, 6, 7), (1, 100003)])
@pytest.mark.parametrize("p", [0.0, 0.3, 1.0])
def test_dropout_is_exact_in_its_mask(kind, shape, p):
    dt = TYPES[kind]
    x, r, dy = (t.to(dt) for t in make(sum(shape), shape, shape, shape))
    seed, offset = 0x123456789ABCDEF, 77
    for res in (None, r):
        xs = x.cuda().requires_grad_()
        rs = res.cuda().requires_grad_() if res is not None else None
        y = head.dropout(xs, p, seed, offset, residual=rs)
        assert ho.worst(y, *ho.dropout(x, p, seed, offset, res)) <= 1.0
        grads = torch.autograd.grad(y, (xs,) if res is None else (xs, rs), dy.cuda())
        assert ho.worst(grads[0], *ho.dropout(dy, p, seed, offset, None)) <= 1.0
        if res is not None:
            assert torch.equal(grads[1].cpu(), dy)


@pytest.mark.parametrize("kind", list(TYPES))
def test_dropout_depends_on_the_position_not_on_the_strides(kind):
    dt = TYPES[kind]
    x, r = (t.to(dt) for t in make(4, (67, 50), (67, 50)))
    want = head.dropout(x.cuda(), 0.4, 9, 2, residual=r.cuda())
    pad = torch.full((67, 61), float("nan"), dtype=dt, device="cuda")
    pad[:, 5:55] = x.cuda()
    odd = torch.empty(67 * 50 + 1, dtype=dt, device="cuda")
    odd[1:] = r.reshape(-1).cuda()
    for xs in (pad[:, 5:55], x.t().contiguous().cuda().t()):
        for rs in (r.cuda(), odd[1:].view(67, 50), r.t().contiguous().cuda().t()):
            assert torch.equal(head.dropout(xs, 0.4, 9, 2, residual=rs), want)
    row = head.dropout(x[:1].cuda().expand(67, 50), 0.4, 9, 2)
    assert ho.worst(row, *ho.dropout(x[:1].expand(67, 50).contiguous(), 0.4, 9, 2, None)) <= 1.0


def test_dropout_keeps_infinities_and_nan_of_dropped_places_out():
    x = torch.full((64, 64), math.nan)
    y = head.dropout(x.cuda(), 0.5, 1, 0).cpu()
    keep = torch.from_numpy(ho.keep_mask(4096, 0.5, 1, 0)).view(64, 64)
    assert torch.isnan(y[keep]).all() and (y[~keep] == 0).all()
    assert (head.dropout(x.cuda(), 1.0, 1, 0) == 0).all()


def test_dropout_takes_its_seed_from_the_device():
    x, = make(6, (100, 30))
    xs = x.cuda().requires_grad_()
    rng = torch.tensor([-5, 12], dtype=torch.int64, device="cuda")
    y = head.dropout(xs, 0.25, rng)
    assert torch.equal(y, head.dropout(xs, 0.25, -5, 12))
    dx, = torch.autograd.grad(y, xs, torch.ones_like(y))
    assert torch.equal(dx != 0, torch.from_numpy(ho.keep_mask(3000, 0.25, -5, 12)).view(100, 30).cuda())
    y = head.dropout(xs, 0.25, rng)
    rng += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, xs, torch.ones_like(y))


# ---- linear + cross entropy ------------------------------------------------------------------------------------------------

def loss_case(seed, T, V, D, dt, bias, pad=True):
    g = torch.Generator().manual_seed(seed)
    x, w, b = (torch.randn(*s, generator=g) for s in ((T, D), (V, D), (V,)))
    target = torch.randint(0, V, (T,), generator=g)
    if pad and T > 2:
        target[torch.rand(T, generator=g) < 0.2] = -100
    return x.to(dt), (w * 2 / math.sqrt(D)).to(dt), b.to(dt) if bias else None, target


def run_loss(x, w, target, b, eps, reduction, dloss, ignore=-100):
    leaves = [t.cuda().requires_grad_() if t is not None else None for t in (x, w, b)]
    loss = head.linear_cross_entropy(leaves[0], leaves[1], target.cuda(), leaves[2], ignore_index=ignore, label_smoothing=eps,
                                     reduction=reduction)
    grads = torch.autograd.grad(loss, [t for t in leaves if t is not None], dloss.cuda())
    return {"loss": loss, **dict(zip(("dx", "dw", "db"), grads))}


LOSS_SIZES = [(1, 1, 1), (1, 2, 8), (2, 3, 5), (256, 3, 256), (1, 5000, 64), (16, 1031, 200), (17, 4100, 96), (64, 64, 64),
              (65, 130, 67), (130, 257, 72), (300, 777, 101), (513, 1024, 128)]


@pytest.mark.parametrize("T,V,D", LOSS_SIZES)
@pytest.mark.parametrize("kind", list(TYPES))
def test_linear_cross_entropy_and_its_gradients(kind, T, V, D):
    i = LOSS_SIZES.index((T, V, D))
    reduction = ("mean", "sum", "none")[i % 3]
    eps = 0.1 if i % 2 else 0.0
    x, w, b, target = loss_case(T + V + D, T, V, D, TYPES[kind], bias=i % 4 != 3)
    scale = 256.0 if kind == "f16" else 1.0              # half precision trains with a scaled loss
    dloss = torch.rand(T, generator=torch.Generator().manual_seed(i)) * scale / T if reduction == "none" else \
        torch.tensor(scale if reduction == "mean" else scale / T)
    got = run_loss(x, w, target, b, eps, reduction, dloss)
    assert got["loss"].dtype == torch.float32
    check(got, ho.cross_entropy(x, w, target, b, -100, eps, reduction, dloss))


@pytest.mark.parametrize("kind", list(TYPES))
def test_linear_cross_entropy_over_several_pieces_of_the_vocabulary(kind):
    """Sizes at which the [T, V] logits pass the largest piece: 2100 x 70000 in 32 bits are 588 MB."""
    T, V, D = 2100, 70000, 16
    dt = TYPES[kind]
    x, w, b, target = loss_case(1, T, V, D, dt, True)
    dloss = torch.tensor(1024.0 if kind == "f16" else 1.0)
    got = run_loss(x, w, target, b, 0.1, "mean", dloss)
    rows = [0, 1, 63, 64, 1000, 2098, 2099]
    count = (target != -100).sum().item()
    part = ho.cross_entropy(x[rows], w, target[rows], b, -100, 0.1, "sum", dloss / count)
    check({"dx": got["dx"][rows]}, {"dx": part["dx"]})
    # everything else against plain 64-bit products on the device
    X, W = x.cuda().double(), w.cuda().double()
    z = X @ W.t() + b.cuda().double()
    live = (target != -100).cuda()
    logp = torch.log_softmax(z, 1)
    wanted = torch.full_like(z, 0.1 / V)
    wanted[torch.arange(T, device="cuda")[live], target.cuda()[live]] += 0.9
    wanted[~live] = 0
    loss = -(wanted * logp).sum() / count
    assert abs(got["loss"].item() - loss.item()) < 2e-3        # (V / 32 + ...) units of 2^-24, the bound of a row's loss
    dz = (logp.exp() * live[:, None] - wanted) * (dloss.item() / count)
    u = ho.half_step(dt) + 2.0 ** -9 * (kind == "bf16")
    for name, ref, mag in (("dw", dz.t() @ X, dz.abs().t() @ X.abs()), ("db", dz.sum(0), dz.abs().sum(0))):
        err = (got[name].double() - ref).abs()
        # dz rounded once (h), its probability off by the logits' and lse's errors (below 2e-3), the result rounded (h)
        assert bool((err <= (2 * u + 2e-3) * mag + ho.tiny(dt)).all()), name


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_ignored_rows_and_bad_labels(kind, reduction):
    dt = TYPES[kind]
    x, w, b, target = loss_case(12, 70, 50, 24, dt, True, pad=False)
    target[5:9] = 7                                       # the ignored label may be a class
    x[5], x[6], x[7] = math.nan, math.inf, torch.finfo(dt).max
    dloss = torch.rand(70) if reduction == "none" else torch.tensor(1.0)
    got = run_loss(x, w, target, b, 0.0, reduction, dloss, ignore=7)
    check(got, ho.cross_entropy(x, w, target, b, 7, 0.0, reduction, dloss))
    assert (got["dx"][target == 7] == 0).all()
    target[20], target[21] = 50, -1                       # not a class, not ignored: NaN, and no gradient
    got = run_loss(x, w, target, b, 0.0, reduction, dloss, ignore=7)
    check(got, ho.cross_entropy(x, w, target, b, 7, 0.0, reduction, dloss))
    assert (got["dx"][20:22] == 0).all()


def test_a_batch_of_ignored_rows():
    x, w, b, target = loss_case(12, 9, 50, 24, torch.float32, True)
    target[:] = -100
    got = run_loss(x, w, target, b, 0.0, "mean", torch.tensor(1.0))
    assert math.isnan(got["loss"].item()) and not got["dx"].any() and not got["dw"].any() and not got["db"].any()
    got = run_loss(x, w, target, b, 0.0, "none", torch.ones(9))
    assert not got["loss"].any() and not got["dw"].any()


@pytest.mark.parametrize("kind", list(TYPES))
def test_masked_classes(kind):
    """A bias of -inf takes a class out; the type's lowest value nearly does; a label on a masked class costs inf."""
    dt = TYPES[kind]
    V = 600
    x, w, b, target = loss_case(15, 40, V, 32, dt, True, pad=False)
    b[:256], b[300:302], b[V - 1] = -math.inf, torch.finfo(dt).min, -math.inf
    target = 256 + target % 40
    dloss = torch.ones(40) * (64.0 if kind == "f16" else 1.0)
    got = run_loss(x, w, target, b, 0.0, "none", dloss)
    want = ho.cross_entropy(x, w, target, b, -100, 0.0, "none", dloss)
    # a logit at the type's lowest value is exact enough to be nothing: its own magnitude is no error of the row
    b2 = b.clone()
    b2[300:302] = -1000.0 if kind != "f16" else -60000.0
    want2 = ho.cross_entropy(x, w, target, b.masked_fill(b == torch.finfo(dt).min, -math.inf), -100, 0.0, "none", dloss)
    for k in want:
        want[k] = (want2[k][0], want2[k][1])
    check(got, want)
    assert (got["db"][:256] == 0).all() and (got["dw"][:256] == 0).all()
    target[3] = 0
    got = run_loss(x, w, target, b, 0.0, "none", dloss)
    assert got["loss"][3].item() == math.inf and torch.isfinite(got["loss"][4:]).all()
    b[:] = -math.inf                                      # nothing left at all
    assert torch.isnan(head.linear_cross_entropy(x.cuda(), w.cuda(), target.cuda(), b.cuda(), reduction="none")).all()


@pytest.mark.parametrize("kind", list(TYPES))
def test_large_logits_and_a_sure_row(kind):
    x, w, b, target = loss_case(19, 33, 300, 16, TYPES[kind], False, pad=False)
    x = x * 40
    dloss = torch.tensor(1.0)
    check(run_loss(x, w, target, b, 0.0, "mean", dloss), ho.cross_entropy(x, w, target, b, -100, 0.0, "mean", dloss))


@pytest.mark.parametrize("kind", list(TYPES))
def test_linear_cross_entropy_takes_any_strides(kind):
    dt = TYPES[kind]
    x, w, b, target = loss_case(31, 60, 90, 40, dt, True)
    want = ho.cross_entropy(x, w, target, b, -100, 0.0, "none", torch.ones(60))
    xs = torch.full((60, 47), math.nan, dtype=dt, device="cuda")
    xs[:, 1:41] = x.cuda()
    xs = xs[:, 1:41].detach().requires_grad_()
    ws = w.t().contiguous().cuda().t().requires_grad_()
    bs = torch.stack([b, b]).t().contiguous().cuda()[:, 0].detach().requires_grad_()
    ts = torch.stack([target, target]).t().contiguous().cuda()[:, 0]
    loss = head.linear_cross_entropy(xs, ws, ts.int(), bs, reduction="none")
    dx, dw, db = torch.autograd.grad(loss, (xs, ws, bs), torch.ones((), device="cuda").expand(60))
    check({"loss": loss, "dx": dx, "dw": dw, "db": db}, want)
    loss = head.linear_cross_entropy(x.cuda().view(3, 20, 40), w.cuda(), target.cuda().view(3, 20), b.cuda(), reduction="none")
    assert loss.shape == (3, 20)
    check({"loss": loss.reshape(-1)}, {"loss": want["loss"]})


# ---- beyond 32 bits --------------------------------------------------------------------------------------------------------

def test_dropout_beyond_32_bits_of_elements():
    n, tail = 2 ** 32 + 4104, 5000
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = head.dropout(x.view(8, n // 8), 0.25, 3, 1).view(-1)
    keep = ho.keep_mask_at(n - tail, tail, 0.25, 3, 1)
    assert torch.equal(y[-tail:].cpu() != 0, torch.from_numpy(keep))
    assert torch.equal(y[:tail].cpu() != 0, torch.from_numpy(ho.keep_mask(tail, 0.25, 3, 1)))
    share = sum((c != 0).sum().item() for c in y.split(2 ** 28)) / n
    assert abs(share - 0.75) < 5 * (0.25 * 0.75 / n) ** 0.5


def test_linear_beyond_32_bits_of_elements():
    """2 100 000 rows of 2056: the last ones lie behind 4 G elements, and the weight's gradient runs over all rows."""
    M, N, K, tail = 2_100_000, 4, 2056, 300
    dt = torch.bfloat16
    xt, w, b, _, dyt = linear_case(77, tail, N, K, dt, None, True, False)
    x = torch.zeros(M, K, dtype=dt, device="cuda")
    x[-tail:] = xt.cuda()
    dy = torch.zeros(M, N, dtype=dt, device="cuda")
    dy[-tail:] = dyt.cuda()
    xs, ws, bs = x.requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
    y = head.linear(xs, ws, bs, activation="silu")
    dx, dw, db = torch.autograd.grad(y, (xs, ws, bs), dy)
    want = ho.linear(xt, w, b, "silu", None, dyt)
    check({"y": y[-tail:], "dx": dx[-tail:], "dw": dw, "db": db}, want)
    assert not dx[:1000].any() and torch.equal(y[:1000], y[1000:2000])


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_linear_cross_entropy_beyond_32_bits_of_logits(kind):
    """40 000 rows by 131 072 classes: 5.2 G logits, in several runs of rows (forward) and pieces of the vocabulary."""
    T, V, D = 40000, 131072, 16
    dt = TYPES[kind]
    x, w, b, target = loss_case(5, T, V, D, dt, True)
    rows = [0, 1, 255, 256, 4095, 4096, 8191, 8192, 8193, 16383, 16384, 32767, 32768, T - 2, T - 1]
    dloss = torch.zeros(T)
    dloss[rows] = torch.rand(len(rows)) + 0.5
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    loss = head.linear_cross_entropy(leaves[0], leaves[1], target.cuda(), leaves[2], label_smoothing=0.1, reduction="none")
    dx, dw, db = torch.autograd.grad(loss, leaves, dloss.cuda())
    want = ho.cross_entropy(x[rows], w, target[rows], b, -100, 0.1, "none", dloss[rows])
    # the sums over the rows have T terms, all but those of `rows` exact zeros
    check({"loss": loss[rows], "dx": dx[rows], "dw": dw, "db": db}, want)
    others = torch.ones(T, dtype=torch.bool)
    others[rows] = False
    assert not dx[others.cuda()].any()


# ---- against differences, together, captured --------------------------------------------------------------------------------

def test_gradients_against_differences():
    """Directional derivatives by central differences of step 2^-6 in float32.  The loss is a mean of rows whose logits move
    by at most 1 per unit of the direction: the third derivative is at most 4, the truncation h^2 / 6 * 4 = 1.7e-4; the two
    losses (below 8) are off by at most 40 units of 2^-24 each: 40 * 8 * 2^-24 / 2^-6 = 1.3e-3 at worst."""
    x, w, b, target = loss_case(41, 48, 37, 20, torch.float32, True)
    x, w, b, target = x.cuda(), w.cuda(), b.cuda(), target.cuda()
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    loss = head.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], label_smoothing=0.1)
    grads = torch.autograd.grad(loss, leaves)
    h = 2.0 ** -6
    for i in range(3):
        d = torch.randn_like(leaves[i])
        moved = d @ w.t() if i == 0 else x @ d.t() if i == 1 else d.expand(48, 37)
        d = d / moved.abs().max()
        at = []
        for s in (h, -h):
            args = [x, w, b]
            args[i] = args[i] + s * d
            at.append(head.linear_cross_entropy(args[0], args[1], target, args[2], label_smoothing=0.1).item())
        slope = (grads[i].double() * d.double()).sum().item()
        assert abs((at[0] - at[1]) / (2 * h) - slope) < 1.5e-3, i
    # the smooth activations: sum of y over a direction of the output; |act'''| <= 3, moved by at most 1 a unit: truncation
    # 48 * 30 * h^2 / 6 * 3 spread over random signs - a tenth of it - against slopes of some tens
    x, w, b, r, dy = (t.cuda() if t is not None else None for t in linear_case(43, 48, 30, 20, torch.float32, None, True, False))
    for act in ("gelu", "gelu_tanh", "silu"):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(head.linear(*leaves, activation=act), leaves, dy)
        for i in range(3):
            d = torch.randn_like(leaves[i])
            moved = d @ w.t() if i == 0 else x @ d.t() if i == 1 else d.expand(48, 30)
            d = d / moved.abs().max()
            at = []
            for s in (h, -h):
                args = [x, w, b]
                args[i] = args[i] + s * d
                at.append((head.linear(*args, activation=act).double() * dy.double()).sum().item())
            slope = (grads[i].double() * d.double()).sum().item()
            assert abs((at[0] - at[1]) / (2 * h) - slope) < 0.02 + 1e-3 * abs(slope), (act, i)


def head_step(x, params, target, rng):
    """linear -> dropout with its residual -> linear_cross_entropy, as a training step uses them."""
    w1, b1, w2, b2, w3, b3 = params
    h1 = head.linear(x, w1, b1, activation="relu")
    h2 = head.linear(h1, w2, b2, activation="gelu")
    h3 = head.dropout(h2, 0.3, rng, residual=h1)
    loss = head.linear_cross_entropy(h3, w3, target, b3, label_smoothing=0.05)
    return loss, torch.autograd.grad(loss, params)


def head_params(dt, D, H, V, seed):
    p = make(seed, (H, D), (H,), (H, H), (H,), (V, H), (V,))
    return [(t / math.sqrt(t.shape[-1]) if t.dim() == 2 else 0.1 * t).to(dt).cuda().requires_grad_() for t in p]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_the_operators_together(kind):
    """A head's step against the same step in 64 bits.  Three layers of rounding, each of h relative to its values and
    amplified by norms near 1: 16 h of a tensor's norm (and what float32 sums leave, 1e-5) bounds it."""
    dt = TYPES[kind]
    params = head_params(dt, 96, 128, 333, 51)
    x, = make(52, (200, 96))
    x = x.to(dt).cuda()
    target = torch.randint(0, 333, (200,), generator=torch.Generator().manual_seed(1)).cuda()
    target[::9] = -100
    rng = torch.tensor([77, 3], dtype=torch.int64, device="cuda")
    loss, grads = head_step(x, params, target, rng)
    P = [p.detach().cpu().double().requires_grad_() for p in params]
    keep = torch.from_numpy(ho.keep_mask(200 * 128, 0.3, 77, 3)).view(200, 128).double()
    X = x.cpu().double()
    h1 = torch.relu(X @ P[0].t() + P[1])
    h2 = torch.nn.functional.gelu(h1 @ P[2].t() + P[3])
    h3 = h1 + keep * h2 / 0.7
    want = torch.nn.functional.cross_entropy(h3 @ P[4].t() + P[5], target.cpu(), label_smoothing=0.05)
    wg = torch.autograd.grad(want, P)
    tol = 16 * ho.half_step(dt) + 1e-5
    assert abs(loss.item() - want.item()) <= tol * abs(want.item())
    for g, v in zip(grads, wg):
        assert (g.cpu().double() - v).norm() <= tol * v.norm()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_results_do_not_change_from_run_to_run(kind):
    dt = TYPES[kind]
    params = head_params(dt, 96, 128, 333, 61)
    x = make(62, (300, 96))[0].to(dt).cuda()
    target = torch.randint(0, 333, (300,), generator=torch.Generator().manual_seed(2)).cuda()
    rng = torch.tensor([5, 5], dtype=torch.int64, device="cuda")
    loss, grads = head_step(x, params, target, rng)
    for _ in range(3):
        again, more = head_step(x, params, target, rng)
        assert torch.equal(loss, again) and all(torch.equal(a, b) for a, b in zip(grads, more))


def test_two_captured_steps_replayed_between_eager_work():
    """Two graphs of the same step on different inputs, replayed in turn, with a new mask each time and eager work and
    synchronizations in between; every replay against the eager result."""
    dt = torch.bfloat16
    params = head_params(dt, 64, 128, 200, 71)
    target = torch.randint(0, 200, (96,), generator=torch.Generator().manual_seed(3)).cuda()
    xs = [make(s, (96, 64))[0].to(dt).cuda() for s in (72, 73)]
    rngs = [torch.tensor([7, i], dtype=torch.int64, device="cuda") for i in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        head_step(xs[0], params, target, rngs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x, rng in zip(xs, rngs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss, grads = head_step(x, params, target, rng)
        graphs.append(g)
        outs.append((loss, grads))
    for step in range(4):
        for i in range(2):
            xs[i].copy_(make(100 + 2 * step + i, (96, 64))[0].to(dt))
            rngs[i].add_(11)
        for i in range(2):
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            loss, grads = head_step(xs[i], params, target, rngs[i])
            assert torch.equal(loss, outs[i][0]), (step, i)
            assert all(torch.equal(a, b) for a, b in zip(grads, outs[i][1])), (step, i)


def test_calls_on_two_streams_at_once():
    dt = torch.bfloat16
    params = head_params(dt, 256, 512, 3000, 81)
    target = torch.randint(0, 3000, (512,), generator=torch.Generator().manual_seed(4)).cuda()
    xs = [make(s, (512, 256))[0].to(dt).cuda() for s in (82, 83)]
    rng = torch.tensor([1, 2], dtype=torch.int64, device="cuda")
    want = [head_step(x, params, target, rng) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(3):
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(head_step(x, params, target, rng))
    torch.cuda.synchronize()
    for i, (loss, grads) in enumerate(got):
        assert torch.equal(loss, want[i % 2][0])
        assert all(torch.equal(a, b) for a, b in zip(grads, want[i % 2][1]))


def test_refusals_on_the_device():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(6, 8, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad, err in ((lambda: head.linear(x, w.bfloat16()), TypeError), (lambda: head.linear(x, w[:, :5]), ValueError),
                     (lambda: head.linear(x.double(), w.double()), TypeError), (lambda: head.linear(x, w.cpu()), RuntimeError),
                     (lambda: head.linear(x, w, torch.zeros(5, device="cuda")), ValueError),
                     (lambda: head.linear(x, w, residual=torch.zeros(4, 5, device="cuda")), ValueError),
                     (lambda: head.dropout(x, 1.5, 0), ValueError), (lambda: head.dropout(x, float("nan"), 0), ValueError),
                     (lambda: head.dropout(x, 0.5, torch.zeros(2, device="cuda")), ValueError),
                     (lambda: head.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64, device="cuda"), 1), ValueError),
                     (lambda: head.dropout(x, 0.5, 0, residual=x[:2]), ValueError),
                     (lambda: head.linear_cross_entropy(x, w, t[:3]), ValueError),
                     (lambda: head.linear_cross_entropy(x, w, t.float()), TypeError),
                     (lambda: head.linear_cross_entropy(x, w, t.cpu()), RuntimeError),
                     (lambda: head.linear_cross_entropy(x, w, t, label_smoothing=2.0), ValueError)):
        with pytest.raises(err):
            bad()
    y = head.linear(x.requires_grad_(), w)
    dx, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):                     # differentiable once
        torch.autograd.grad(dx.sum() + 0 * y.sum(), w.requires_grad_())


def calls_of(x, w, b, target):
    return (lambda: head.linear(x, w, b, activation="silu"), lambda: head.dropout(x, 0.25, 5),
            lambda: head.linear_cross_entropy(x, w, target, b))


def test_a_captured_backward_with_an_eager_graph_alive_raises():
    x, w, b = (t.cuda().requires_grad_() for t in make(90, (32, 24), (40, 24), (40,)))
    target = torch.randint(0, 40, (32,), generator=torch.Generator().manual_seed(9)).cuda()
    for call in calls_of(x, w, b, target):
        want, = torch.autograd.grad(call().sum(), x)                       # its graph ends here
        kept = call()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            y = call()
            with pytest.raises(RuntimeError, match="eager graph"):
                torch.autograd.grad(y, x, torch.ones_like(y))
        del kept, y, g
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            y = call()
            dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        for _ in range(3):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(dx, want)
        del y, g


def test_eager_steps_on_other_streams_than_their_leaves():
    """An eager backward pass whose leaves have a graph on another stream: the engine waits, nothing is refused."""
    x, w, b = (t.cuda().requires_grad_() for t in make(91, (64, 24), (40, 24), (40,)))
    target = torch.randint(0, 40, (64,), generator=torch.Generator().manual_seed(9)).cuda()
    for call in calls_of(x, w, b, target):
        kept = call()
        want, = torch.autograd.grad(call().sum(), x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got, = torch.autograd.grad(call().sum(), x)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and kept.shape == call().shape


def test_forward_mode_is_refused():
    x, w, b = (t.cuda() for t in make(92, (4, 24), (40, 24), (40,)))
    target = torch.zeros(4, dtype=torch.int64, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls_of(dual, w, b, target):
            with pytest.raises(RuntimeError):
                call()


def test_gradients_of_some_inputs_of_a_call():
    """Each subset of the inputs that need gradients gives those inputs the same ones."""
    x, w, b, r = (t.cuda() for t in make(93, (48, 24), (40, 24), (40,), (48, 40)))
    target = torch.randint(0, 40, (48,), generator=torch.Generator().manual_seed(9)).cuda()
    ops = (lambda x, w, b, r: head.linear(x, w, b, "gelu", r), lambda x, w, b, r: head.linear_cross_entropy(x, w, target, b),
           lambda x, w, b, r: head.dropout(r, 0.25, 5, residual=x @ w.t()))
    for op, uses in zip(ops, ("xwbr", "xwb", "xwr")):
        full = {n: t.clone().requires_grad_() for n, t in zip("xwbr", (x, w, b, r))}
        want = dict(zip(uses, torch.autograd.grad(op(**full).sum(), [full[n] for n in uses])))
        for mask in range(1, 2 ** len(uses)):
            chosen = [n for i, n in enumerate(uses) if mask >> i & 1]
            some = {n: t.clone().requires_grad_(n in chosen) for n, t in zip("xwbr", (x, w, b, r))}
            for n, grad in zip(chosen, torch.autograd.grad(op(**some).sum(), [some[n] for n in chosen])):
                assert torch.equal(grad, want[n]), (uses, chosen, n)


def test_limits_raise_the_librarys_error():
    from pointnetgpd_amd._lib import PngpdError
    w = torch.zeros(1, 1, device="cuda").expand(2 ** 21 + 1, 4)
    with pytest.raises(PngpdError) as e:
        head.linear(torch.zeros(2, 4, device="cuda"), w)
    assert e.value.code != 0 and "pngpd_linear_forward" in str(e.value)


# many tiles, few rows, a cut contraction, few columns
KEPT = [("f32", 333, 5003, 700), ("f32", 1023, 1000, 1000), ("f32", 5, 30011, 2000), ("f32", 40, 2002, 4096), ("bf16", 8000, 40, 4104),
        ("f16", 2000, 2001, 4104), ("bf16", 517, 8001, 4100)]


@pytest.mark.parametrize("kind,T,V,D", KEPT)
def test_logits_kept_for_the_backward_pass(kind, T, V, D):
    """Sizes whose logits are kept: padding rows that hold NaN, a bad label, a masked class, odd sizes."""
    from pointnetgpd_amd import _lib
    dt = TYPES[kind]
    assert _lib.load().pngpd_linear_cross_entropy_kept_bytes(list(TYPES).index(kind), T, V, D) > 0
    i = KEPT.index((kind, T, V, D))
    reduction = ("mean", "sum", "none")[i % 3]
    x, w, b, target = loss_case(T + V, T, V, D, dt, bias=i % 4 != 1)
    target[0], target[1] = 3, -100
    x[target == -100] = float("nan")
    if b is not None:
        b[7] = float("-inf")
        target[target == 7] = 8
    if reduction == "none":
        target[2] = V
    scale = 256.0 if kind == "f16" else 1.0
    dloss = torch.rand(T, generator=torch.Generator().manual_seed(i)) * scale / T if reduction == "none" else \
        torch.tensor(scale if reduction == "mean" else scale / T)
    clean = torch.where(torch.isnan(x), torch.zeros((), dtype=dt), x)
    got = run_loss(x, w, target, b, 0.0, reduction, dloss)
    check(got, ho.cross_entropy(clean, w, target, b, -100, 0.0, reduction, dloss))


def test_kept_logits_serve_two_backward_passes():
    x, w, b = (t.cuda().requires_grad_() for t in make(95, (300, 1024), (3001, 1024), (3001,)))
    target = torch.randint(0, 3001, (300,), generator=torch.Generator().manual_seed(9)).cuda()
    loss = head.linear_cross_entropy(x, w, target, b, label_smoothing=0.1)
    first = torch.autograd.grad(loss, (x, w, b), retain_graph=True)
    other = torch.autograd.grad(head.linear_cross_entropy(x * 2, w, target, b), (x, w, b))      # another call in between
    again = torch.autograd.grad(loss, (x, w, b))
    assert all(torch.equal(p, q) for p, q in zip(first, again)) and not torch.equal(first[0], other[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, (x, w, b))
    loss = head.linear_cross_entropy(x, w, target, b)
    with torch.no_grad():
        b.add_(1)                                              # the kept logits are of the bias as it was
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, (x, w, b))


def test_a_step_captured_over_two_streams():
    """A capture that forks: the loss on a stream of its own, with float32 logits that are kept; replayed between eager work."""
    x, w, v, b = (t.cuda().requires_grad_() for t in make(96, (300, 64), (1024, 64), (3001, 1024), (3001,)))
    target = torch.randint(0, 3001, (300,), generator=torch.Generator().manual_seed(9)).cuda()

    def step(main, side):
        h = head.linear(x, w, activation="relu")
        side.wait_stream(main)
        with torch.cuda.stream(side):
            loss = head.linear_cross_entropy(h, v, target, b)
        main.wait_stream(side)
        return [loss.detach(), *torch.autograd.grad(loss, (x, w, v, b))]

    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    main.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(main):
        step(main, side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=main):
        got = step(main, side)
    for i in range(3):
        with torch.no_grad():
            x.mul_(1.25)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(main):
            want = step(main, side)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), i


def test_one_tensor_in_two_places():
    """The same tensor as input, weight and residual: its gradients add up."""
    x, = make(97, (40, 40))
    a = x.cuda().requires_grad_()
    dx, = torch.autograd.grad(head.linear(a, a, residual=a).sum(), a)
    parts = [x.clone().cuda().requires_grad_() for _ in range(3)]
    want = torch.autograd.grad(head.linear(parts[0], parts[1], residual=parts[2]).sum(), parts)
    assert (dx - sum(t.double() for t in want)).abs().max().item() <= 2 * 2 ** -23 * sum(t.abs() for t in want).max().item()
    target = torch.arange(40, device="cuda")
    dx, = torch.autograd.grad(head.linear_cross_entropy(a, a, target, a[0]), a)
    assert torch.isfinite(dx).all()


def test_threads_call_at_once():
    """Threads of one process, each on a stream of its own, forward and backward at the same time."""
    import threading
    cases = []
    for i in range(4):
        x, w, b = (t.cuda().requires_grad_() for t in make(100 + i, (200 + i, 64), (500, 64), (500,)))
        cases.append((x, w, b, torch.randint(0, 500, (200 + i,), generator=torch.Generator().manual_seed(i)).cuda()))
    want = [torch.autograd.grad(head.linear_cross_entropy(head.dropout(x, 0.2, 3), w, t, b), (x, w, b)) for x, w, b, t in cases]
    torch.cuda.synchronize()
    got, streams = [None] * 4, [torch.cuda.Stream() for _ in range(4)]

    def run(i):
        x, w, b, t = cases[i]
        with torch.cuda.stream(streams[i]):
            for _ in range(10):
                got[i] = torch.autograd.grad(head.linear_cross_entropy(head.dropout(x, 0.2, 3), w, t, b), (x, w, b))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for a, c in zip(got, want) for p, q in zip(a, c))


FEW = [(1, 1, 7), (1000, 8, 513), (70, 7, 1001), (5000, 2, 64), (33, 4, 4096), (256, 3, 256), (2049, 5, 2056), (17, 8, 30000)]


@pytest.mark.parametrize("T,V,D", FEW)
@pytest.mark.parametrize("kind", list(TYPES))
def test_few_classes(kind, T, V, D):
    """At most eight classes: padding rows that hold NaN, a bad label, masked classes, label smoothing, odd sizes."""
    dt = TYPES[kind]
    i = FEW.index((T, V, D))
    reduction, eps = ("mean", "sum", "none")[i % 3], 0.1 if i % 2 else 0.0
    x, w, b, target = loss_case(T + V + D, T, V, D, dt, bias=i != 4)
    scale = 256.0 if kind == "f16" else 1.0
    if T > 20:
        target[:2], target[3] = 0, -100
        x[target == -100] = float("nan")
        if reduction == "none":
            target[2] = V
        if i == 2:
            eps, b[3] = 0.0, float("-inf")
            target[target == 3] = 2
    dloss = torch.rand(T, generator=torch.Generator().manual_seed(i)) * scale / T if reduction == "none" else \
        torch.tensor(scale if reduction == "mean" else scale / T)
    clean = torch.where(torch.isnan(x), torch.zeros((), dtype=dt), x)
    got = run_loss(x, w, target, b, eps, reduction, dloss)
    check(got, ho.cross_entropy(clean, w, target, b, -100, eps, reduction, dloss))
    assert (got["dx"][(target < 0) | (target >= V)] == 0).all()


@pytest.mark.parametrize("kind", list(TYPES))
def test_few_classes_of_any_strides(kind):
    dt = TYPES[kind]
    x, w, b, target = loss_case(41, 60, 6, 72, dt, True)
    dloss = torch.tensor(64.0 if kind == "f16" else 1.0)
    want = run_loss(x, w, target, b, 0.05, "mean", dloss)
    X, W = torch.zeros(60, 101, dtype=dt).cuda(), torch.zeros(72, 6, dtype=dt).cuda()
    X[:, 3:75], W[:] = x.cuda(), w.t().cuda()
    B = torch.zeros(12, dtype=dt).cuda()
    B[::2] = b.cuda()
    leaves = [X[:, 3:75].requires_grad_(), W.t().requires_grad_(), B[::2].requires_grad_()]
    loss = head.linear_cross_entropy(leaves[0], leaves[1], target.cuda(), leaves[2], label_smoothing=0.05)
    grads = torch.autograd.grad(loss, leaves, dloss.cuda())
    check({"loss": loss, **dict(zip(("dx", "dw", "db"), grads))}, ho.cross_entropy(x, w, target, b, -100, 0.05, "mean", dloss))
    assert torch.equal(loss, want["loss"]) and all(torch.equal(p, want[k]) for k, p in zip(("dx", "dw", "db"), grads))
    some = torch.autograd.grad(head.linear_cross_entropy(x.cuda(), w.cuda(), target.cuda(), leaves[2], label_smoothing=0.05), leaves[2],
                               dloss.cuda())
    assert torch.equal(some[0], grads[2])


def test_few_classes_without_kept_logits():
    """The C entries without the memory that carries the logits: the general products' gradients."""
    from pointnetgpd_amd import _lib
    lib = _lib.load()
    T, V, D = 300, 3, 128
    x, w, b, target = loss_case(43, T, V, D, torch.float32, True)
    dev = [t.cuda() for t in (x, w, b, target)]
    loss, lse = torch.empty(1, device="cuda"), torch.empty(T, device="cuda")
    out = [torch.empty(s, device="cuda") for s in ((T, D), (V, D), (V,))]
    ws = torch.empty(max(lib.pngpd_linear_cross_entropy_workspace_bytes(0, T, V, D, k, 1) for k in (0, 1)), dtype=torch.uint8, device="cuda")
    dloss = torch.ones(1, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    args = (0, T, V, D, dev[0].data_ptr(), D, dev[1].data_ptr(), D, dev[2].data_ptr(), dev[3].data_ptr(), -100, 0.1, 1)
    assert lib.pngpd_linear_cross_entropy_forward(*args, loss.data_ptr(), lse.data_ptr(), None, ws.data_ptr(), ws.numel(), stream) == 0
    assert lib.pngpd_linear_cross_entropy_backward(*args, lse.data_ptr(), None, dloss.data_ptr(), *(t.data_ptr() for t in out),
                                                   ws.data_ptr(), ws.numel(), stream) == 0
    want = ho.cross_entropy(x, w, target, b, -100, 0.1, "mean", torch.tensor(1.0))
    check({"loss": loss[0], "dx": out[0], "dw": out[1], "db": out[2]}, want)


def shifted(t, by, gap):
    """The same values `by` elements behind an aligned address, rows `gap` elements apart behind their end."""
    flat = torch.zeros(by + t.shape[0] * (t.shape[1] + gap), dtype=t.dtype, device="cuda")
    view = flat[by:].view(t.shape[0], t.shape[1] + gap)[:, :t.shape[1]]
    view.copy_(t.cuda())
    return view


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M", [1, 3, 70])
@pytest.mark.parametrize("by,gap", [(1, 0), (3, 1), (0, 5), (2, 6)])
def test_rows_that_start_at_any_element(kind, M, by, gap):
    """Inputs, weight, residual, bias and incoming gradient away from 16-byte addresses: the same results, bit for bit."""
    dt = TYPES[kind]
    x, w, b, r, dy = linear_case(7, M, 88, 120, dt, "silu", True, True)
    bias = torch.zeros(88 + by, dtype=dt, device="cuda")
    bias[by:] = b.cuda()
    target = torch.arange(M, device="cuda") % 88

    def run(x, w, b, r, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = head.linear(leaves[0], leaves[1], leaves[2], "silu", leaves[3])
        d = head.dropout(leaves[3], 0.3, 5, 1, residual=dy)
        loss = head.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], reduction="sum")
        few = head.linear_cross_entropy(leaves[0], leaves[1][:5], target % 5, leaves[2][:5], reduction="sum")
        with torch.no_grad():
            plain = head.linear(x, w, b, "silu", r)
        return [y, d, plain, *torch.autograd.grad(y, leaves, dy), *torch.autograd.grad(d, leaves[3], dy),
                *torch.autograd.grad(loss, leaves[:3]), *torch.autograd.grad(few, leaves[:3])]

    want = run(*(t.cuda() for t in (x, w, b, r, dy)))
    got = run(shifted(x, by, gap), shifted(w, by, gap), bias[by:], shifted(r, by, gap), shifted(dy, by, gap))
    for i, (p, q) in enumerate(zip(got, want)):
        assert torch.equal(p, q), i


def test_a_captured_head_on_an_eager_feature():
    """Gradients of the head's own parameters alone: the eager graph behind the feature is not reached, and not refused."""
    x, w0, w, b = (t.cuda().requires_grad_() for t in make(98, (32, 24), (40, 24), (50, 40), (50,)))
    target = torch.randint(0, 50, (32,), generator=torch.Generator().manual_seed(9)).cuda()
    feature = head.linear(x, w0)
    want = torch.autograd.grad(head.linear_cross_entropy(feature, w, target, b), (w, b))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(head.linear_cross_entropy(feature, w, target, b), (w, b))
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("T,V,D", [(300, 2048, 64), (40, 1100, 4096), (600, 2100, 2048)])      # a whole, a cut contraction, kept logits
@pytest.mark.parametrize("kind", list(TYPES))
def test_runs_of_classes_masked_by_finite_values(kind, T, V, D):
    """Aligned runs of 64, 128 and 512 classes under a large finite bias: nothing of them is left in 32 bits (exp(-8000) = 0), so
    the results are those of a bias of -inf."""
    dt = TYPES[kind]
    x, w, b, target = loss_case(T + V, T, V, D, dt, True)
    masked = torch.zeros(V, dtype=torch.bool)
    masked[:64] = masked[192:320] = masked[512:1024] = True
    free = (~masked).nonzero()[:, 0]
    target = torch.where(target == -100, target, free[target % len(free)])
    dloss = torch.tensor(64.0 if kind == "f16" else 1.0)
    want = ho.cross_entropy(x, w, target, b.masked_fill(masked, -math.inf), -100, 0.0, "mean", dloss)
    for low in (-1e4, torch.finfo(dt).min) if kind == "f16" else (-1e4, -1e10, -1e30, torch.finfo(dt).min):
        got = run_loss(x, w, target, b.masked_fill(masked, low), 0.0, "mean", dloss)
        check(got, want)
        assert not got["dw"][masked.cuda()].any() and not got["db"][masked.cuda()].any()


@pytest.mark.parametrize("shift", [3e4, -3e4, 1e10, -1e10, 1e30, -1e30])
@pytest.mark.parametrize("T,V,D", [(300, 2048, 64), (40, 1100, 4096), (600, 2100, 2048)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_rows_whose_log_sum_is_large(kind, T, V, D, shift):
    """Every class under the same large bias: what 32 bits leave of the probabilities stays in [0, 1], and nothing overflows."""
    dt = TYPES[kind]
    if abs(shift) > torch.finfo(dt).max:
        return
    x, w, _, target = loss_case(T + V, T, V, D, dt, False)
    b = torch.full((V,), shift, dtype=dt)
    got = run_loss(x, w, target, b, 0.0, "sum", torch.tensor(1.0))
    check(got, ho.cross_entropy(x, w, target, b, -100, 0.0, "sum", torch.tensor(1.0)))
    count = torch.bincount(target[target >= 0], minlength=V).double()
    db, h = got["db"].double().cpu(), ho.half_step(dt)
    # sum of p - [label] over the rows that count, p in [0, 1], each rounded once, the sum once (its 32-bit errors are smaller)
    assert ((db >= -count * (1 + h) ** 2 * 1.001) & (db <= (count.sum() - count) * (1 + h) ** 2 * 1.001 + 1e-30)).all()


def test_forward_mode_is_refused_whatever_the_gradient_mode():
    """no_grad leaves forward-mode differentiation on: a result without its tangent would read as a derivative of zero."""
    x, w, b = (t.cuda() for t in make(92, (4, 24), (40, 24), (40,)))
    target = torch.zeros(4, dtype=torch.int64, device="cuda")
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        duals = [fw.make_dual(t, torch.ones_like(t)) for t in (x, w, b)]
        dual_r = fw.make_dual(torch.zeros(4, 40, device="cuda"), torch.ones(4, 40, device="cuda"))
        for mode in (torch.no_grad, torch.enable_grad):
            with mode():
                for i in range(3):
                    args = [duals[j] if j == i else t for j, t in enumerate((x, w, b))]
                    for call in (lambda: head.linear(*args), lambda: head.linear_cross_entropy(args[0], args[1], target, args[2])):
                        with pytest.raises(RuntimeError, match="forward-mode"):
                            call()
                for call in (lambda: head.dropout(duals[0], 0.25, 5), lambda: head.dropout(x, 0.25, 5, residual=duals[0]),
                             lambda: head.linear(x, w, residual=dual_r)):
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        call()
        with torch.inference_mode():                          # torch itself has no tangents there
            assert head.linear(duals[0], w).shape == (4, 40)
        x2 = fw.unpack_dual(duals[0]).primal
        assert head.linear(x2, w).shape == (4, 40)
    assert head.linear(x, w).shape == (4, 40)


# a whole and a cut contraction, kept logits, several pieces of the vocabulary
WEIGHTED = [(1500, 700, 80), (40, 1100, 4096), (600, 2100, 2048), (2100, 70000, 16)]


@pytest.mark.parametrize("T,V,D", WEIGHTED)
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_rows_of_one_weight_are_the_sum_of_that_weight(kind, T, V, D):
    """(loss * mask).sum() / n over the losses of the rows: the same gradients as the sum's, bit for bit.  The weight (not a power of
    two) stays out of the 16-bit logits' gradients, where it would round the labels' p - 1 the same way in every row."""
    dt = TYPES[kind]
    x, w, b, target = loss_case(T + V, T, V, D, dt, True)
    for g in (1.0 / 3891, 0.75, -1.0 / 3, 300.0):
        want = run_loss(x, w, target, b, 0.1, "sum", torch.tensor(g))
        got = run_loss(x, w, target, b, 0.1, "none", torch.full((T,), g))
        for k in ("dx", "dw", "db"):
            assert torch.equal(got[k], want[k]), (g, k)


@pytest.mark.parametrize("kind", list(TYPES))
def test_weights_of_rows_far_apart(kind):
    """Rows whose incoming gradients differ by up to 2^30, zeros, infinities and NaN among them."""
    dt = TYPES[kind]
    x, w, b, target = loss_case(21, 90, 150, 40, dt, True, pad=False)
    dloss = torch.rand(90, generator=torch.Generator().manual_seed(2)) * 2.0 ** -(torch.arange(90) % 31).float()
    dloss[::7] = 0.0
    dloss[5] = -dloss[5]
    got = run_loss(x, w, target, b, 0.0, "none", dloss)
    check(got, ho.cross_entropy(x, w, target, b, -100, 0.0, "none", dloss))
    assert not got["dx"][::7].any()
    dloss[3], dloss[4], target[6], dloss[6] = math.inf, math.nan, -100, math.nan
    got = run_loss(x, w, target, b, 0.0, "none", dloss)
    rest = [i for i in range(90) if i not in (3, 4)]
    assert torch.isnan(got["dx"][4]).all() and not torch.isfinite(got["dx"][3]).any() and torch.isfinite(got["dx"][rest]).all()
    assert not got["dx"][6].any()


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("eps", [0.1, 0.3])
def test_labels_of_smoothed_targets_are_not_rounded_one_way(eps, reduction):
    """1 - eps has no exact bfloat16: were it in every row's gradient, the weight's gradient would be off by one factor (0.0017 for
    0.1, 0.0011 for 0.3), which the projection on the exact gradient shows.  Its elements carry two roundings of at most h each,
    random in sign: the projection of N = 65536 of them deviates by at most 2 h / sqrt N (Gaussian values: sqrt(3) for their fourth
    moment, 1 / sqrt(3) for a rounding's deviation), taken six times; the label's p - (1 - eps) may lose p besides, below 2^-11."""
    T, V, D = 8192, 4096, 16
    g = torch.Generator().manual_seed(33)
    x, w = torch.randn(T, D, generator=g).bfloat16(), (torch.randn(V, D, generator=g) * 0.02).bfloat16()
    target = torch.arange(T) % V
    dloss = torch.tensor(1.0) if reduction == "mean" else torch.full((T,), 1.0 / T)
    got = run_loss(x, w, target, None, eps, reduction, dloss)["dw"].double()
    X, W, y = x.cuda().double(), w.cuda().double(), target.cuda()
    p = torch.softmax(X @ W.t(), 1)
    assert p.max() < 2.0 ** -11
    p -= eps / V
    p[torch.arange(T, device="cuda"), y] -= 1 - eps
    want = p.t() @ X / T
    off = ((got - want) * want).sum() / want.square().sum()
    assert abs(off.item()) <= 6 * 2 * ho.half_step(torch.bfloat16) / (V * D) ** 0.5 + 2.0 ** -11


@pytest.mark.parametrize("eps", [0.5, 0.999, 1.0])
@pytest.mark.parametrize("kind", list(TYPES))
def test_strong_smoothing(kind, eps):
    x, w, b, target = loss_case(37, 70, 90, 40, TYPES[kind], True)
    dloss = torch.tensor(64.0 if kind == "f16" else 1.0)
    check(run_loss(x, w, target, b, eps, "mean", dloss), ho.cross_entropy(x, w, target, b, -100, eps, "mean", dloss))


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("T,V,D", WEIGHTED[:3] + [(77, 9, 40), (4, 3000, 4096), (5000, 40, 24)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_bias_gradient_of_the_loss_is_rounded_once(kind, T, V, D, reduction):
    """Sums of the logits' gradients before these are rounded: off by what 32 bits leave, as for float32 operands, and one rounding
    of the result."""
    dt = TYPES[kind]
    x, w, b, target = loss_case(T + V, T, V, D, dt, True)
    scale = 256.0 if kind == "f16" else 1.0
    dloss = torch.tensor(scale) if reduction == "mean" else torch.rand(T, generator=torch.Generator().manual_seed(T)) * scale / T
    got = run_loss(x, w, target, b, 0.1, reduction, dloss)
    v, e = ho.cross_entropy(x.float(), w.float(), target, b.float(), -100, 0.1, reduction, dloss)["db"]
    check({"db": got["db"]}, {"db": (v, e + ho.half_step(dt) * (v.abs() + e) + ho.tiny(dt))})
    # alone, without the other two
    bs = b.cuda().requires_grad_()
    loss = head.linear_cross_entropy(x.cuda(), w.cuda(), target.cuda(), bs, label_smoothing=0.1, reduction=reduction)
    alone, = torch.autograd.grad(loss, bs, dloss.cuda())
    assert torch.equal(alone, got["db"])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T,V,D", [(5000, 3, 200), (5000, 8, 513), (20, 4, 2056)])
def test_few_classes_stay_inside_the_workspace_they_ask_for(kind, T, V, D):
    """The C entries with exactly the memory that the size functions name, marks behind it; x away from 16-byte addresses."""
    from pointnetgpd_amd import _lib
    lib, dt, t = _lib.load(), TYPES[kind], list(TYPES).index(kind)
    x, w, b, target = loss_case(T + V, T, V, D, dt, True)
    X, W, B, Y = shifted(x, 1, 3), shifted(w, 3, 0), b.cuda(), target.cuda()
    loss, lse = torch.empty(1, device="cuda"), torch.empty(T, device="cuda")
    out = [torch.empty(s, dtype=dt, device="cuda") for s in ((T, D), (V, D), (V,))]
    dloss = torch.full((1,), 64.0 if kind == "f16" else 1.0, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream

    def room(n):
        return torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device="cuda")

    size = lib.pngpd_linear_cross_entropy_workspace_bytes
    nk, nf, nb = lib.pngpd_linear_cross_entropy_kept_bytes(t, T, V, D), size(t, T, V, D, 0, 0), size(t, T, V, D, 2, 0)
    kept, ws, wsb = room(nk), room(nf), room(nb)
    args = (t, T, V, D, X.data_ptr(), X.stride(0), W.data_ptr(), W.stride(0), B.data_ptr(), Y.data_ptr(), -100, 0.1, 1)
    assert lib.pngpd_linear_cross_entropy_forward(*args, loss.data_ptr(), lse.data_ptr(), kept.data_ptr(), ws.data_ptr(), nf, stream) == 0
    assert lib.pngpd_linear_cross_entropy_backward(*args, lse.data_ptr(), kept.data_ptr(), dloss.data_ptr(), *(o.data_ptr() for o in out),
                                                   wsb.data_ptr(), nb, stream) == 0
    check({"loss": loss[0], "dx": out[0], "dw": out[1], "db": out[2]},
          ho.cross_entropy(x, w, target, b, -100, 0.1, "mean", dloss.cpu()[0]))
    for buffer, n in ((kept, nk), (ws, nf), (wsb, nb)):
        assert (buffer[n:] == 0xA5).all()


def test_few_classes_take_no_copy_of_a_large_input():
    x = torch.randn(100000, 1025, device="cuda")[:, 1:].requires_grad_()      # rows away from 16-byte addresses
    w, y = torch.randn(3, 1024, device="cuda").requires_grad_(), torch.arange(100000, device="cuda") % 3
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = head.linear_cross_entropy(x, w, y)
    torch.autograd.grad(loss, (x, w))
    assert torch.cuda.max_memory_allocated() - before < 100000 * 1024 * 4 + (32 << 20)      # x's gradient, and little else


def test_dropout_of_one_dimension_beyond_31_bits():
    """A one-dimensional tensor, and a column, of 2^31 + 9 elements drop what the same elements of another shape do."""
    n, tail = 2 ** 31 + 9, 5001
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    keep = torch.cat([torch.from_numpy(ho.keep_mask(tail, 0.25, 3, 1)), torch.from_numpy(ho.keep_mask_at(n - tail, tail, 0.25, 3, 1))])
    for view in (x, x.view(n, 1), x.view(1, n)):
        y = head.dropout(view, 0.25, 3, 1)
        assert y.shape == view.shape
        y = y.view(-1)
        assert torch.equal(torch.cat([y[:tail], y[-tail:]]).cpu() != 0, keep)
        del y


def test_a_head_behind_the_trunk():
    """PointNetfeat in training mode, then linear, dropout and linear_cross_entropy, one backward pass through both: the head's
    gradients against 64 bits on the feature as it is, the trunk's against the trunk's own backward pass of the feature's gradient."""
    from pointnetgpd_amd import synth
    from pointnetgpd_amd.pointnet import PointNetfeat
    B, P, H, V = 12, 64, 96, 5
    sd = {k[len("feat."):]: v for k, v in synth.torch_state_dict(3, 2, 0.02).items() if k.startswith("feat.")}
    points = torch.from_numpy(synth.candidate_points(5, B, P, "gripper")).cuda()
    target = (torch.arange(B) % V).cuda()

    def trunk():
        m = PointNetfeat(P, 3)
        m.load_state_dict(sd)
        return m.cuda().train()

    params = [t.cuda().requires_grad_() for t in make(6, (H, 1024), (H,), (H, H), (H,), (V, H), (V,), scale=0.05)]
    m = trunk()
    feat, trans = m(points)
    feat.retain_grad()
    h0 = head.linear(feat, params[0], params[1])
    h1 = head.linear(h0, params[2], params[3], activation="gelu")
    h = head.dropout(h1, 0.3, 11, 2, residual=h0)
    loss = head.linear_cross_entropy(h, params[4], target, params[5], label_smoothing=0.1)
    (loss + 0.001 * trans.square().sum()).backward()

    P64 = [p.detach().cpu().double().requires_grad_() for p in params]
    F64 = feat.detach().cpu().double().requires_grad_()
    keep = torch.from_numpy(ho.keep_mask(B * H, 0.3, 11, 2)).view(B, H).double()
    a0 = F64 @ P64[0].t() + P64[1]
    a1 = torch.nn.functional.gelu(a0 @ P64[2].t() + P64[3])
    want = torch.nn.functional.cross_entropy((a0 + keep * a1 / 0.7) @ P64[4].t() + P64[5], target.cpu(), label_smoothing=0.1)
    want.backward()
    # three layers of 32-bit sums over at most 1024 terms, random in sign: 64 units a layer, and their functions
    tol = 4 * 64 * ho.U * 3
    assert abs(loss.item() - want.item()) <= tol * abs(want.item())
    for got, ref in zip(params + [feat], P64 + [F64]):
        assert (got.grad.cpu().double() - ref.grad).norm() <= tol * ref.grad.norm()

    twin = trunk()
    again, trans2 = twin(points)
    assert torch.equal(again, feat)
    torch.autograd.backward([again, trans2], [feat.grad, 0.002 * trans2.detach()])
    for (name, p), q in zip(m.named_parameters(), twin.parameters()):
        assert torch.equal(p.grad, q.grad), name


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_negative_tails_of_the_activations(act):
    """Relative to the value, down to z = -12, in units of 2^-24.  The exponential's argument a is rounded three times (its constant
    and two products; gelu_tanh's fma besides), which the result sees as 4 |a| ln 2 <= 4 |ln of the factor|; besides at most 12 for
    the fit, the instructions' own steps and the last products.  Factors below 2^-126 may be 0."""
    z = -torch.linspace(0.0, 12.0, 4801)[1:, None]
    Z = z.double()
    if act == "gelu":
        gate, expo = 0.5 * torch.special.erfc(-Z / math.sqrt(2)), Z * Z / 2
    elif act == "silu":
        gate, expo = torch.sigmoid(Z), Z.abs()
    else:
        u = math.sqrt(2 / math.pi) * (Z + 0.044715 * Z ** 3)
        gate, expo = torch.sigmoid(2 * u), 2 * u.abs()
    want = Z * gate
    bound = (12 + 4 * expo) * ho.U * want.abs() + 2 * 2.0 ** -126 * Z.abs()
    one = torch.ones(1, 1, device="cuda")
    assert ho.worst(head.linear(z.cuda(), one, activation=act), want, bound) <= 1.0


@pytest.mark.parametrize("T,V,D", [(4096, 12, 24), (4097, 12, 24), (16384, 12, 16), (16385, 12, 16), (300001, 9, 8), (300001, 3, 8)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("kind", list(TYPES))
def test_losses_and_weights_of_many_rows(kind, reduction, T, V, D):
    """Rows whose count, weights and losses are formed by one workgroup and by many; labels and weights that differ from run to
    run of the rows, the largest weight in the last one."""
    dt = TYPES[kind]
    x, w, b, target = loss_case(T, T, V, D, dt, True)
    target[T // 2:T // 2 + 1500] = -100
    scale = 2.0 ** 14 if kind == "f16" else 1.0
    dloss = torch.tensor(scale) if reduction == "mean" else torch.rand(T, generator=torch.Generator().manual_seed(T)) * scale / T
    if reduction == "none":
        dloss[T - 1], target[T - 1] = 3 * scale / T, 1
    got = run_loss(x, w, target, b, 0.1, reduction, dloss)
    check(got, ho.cross_entropy(x, w, target, b, -100, 0.1, reduction, dloss))


@pytest.mark.parametrize("kind", list(TYPES))
def test_a_caller_may_refuse_kept_logits(kind):
    """keep_logits=False: nothing of the logits' size lives between the passes, and the gradients are within the same bounds."""
    dt = TYPES[kind]
    T, V, D = 1000, 6000, 1536
    x, w, b, target = loss_case(61, T, V, D, dt, True)
    dloss = torch.tensor(64.0 if kind == "f16" else 1.0)
    want = ho.cross_entropy(x, w, target, b, -100, 0.1, "mean", dloss)
    held = {}
    for keep in (True, False):
        leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
        y = target.cuda()
        before = torch.cuda.memory_allocated()
        loss = head.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], label_smoothing=0.1, keep_logits=keep)
        held[keep] = torch.cuda.memory_allocated() - before
        check({"loss": loss, **dict(zip(("dx", "dw", "db"), torch.autograd.grad(loss, leaves, dloss.cuda())))}, want)
    assert held[True] >= T * V * 4 and held[False] < 1 << 20
    few = [t.cuda().requires_grad_() for t in (x, w[:5], b[:5])]
    grads = [torch.autograd.grad(head.linear_cross_entropy(*few[:2], target.cuda() % 5, few[2], keep_logits=keep), few) for keep in (True, False)]
    assert all(torch.equal(p, q) for p, q in zip(*grads))


@pytest.mark.parametrize("grad", [math.inf, math.nan])
@pytest.mark.parametrize("T,V", [(70, 50), (70, 5), (5000, 50)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_ignored_rows_under_an_infinite_gradient(kind, T, V, grad):
    """A loss scale that overflowed: every gradient shows it but those of the rows that have none."""
    x, w, b, target = loss_case(71, T, V, 24, TYPES[kind], True)
    target[1], target[2], target[3] = -100, 2, V
    for reduction in ("mean", "sum"):
        got = run_loss(x, w, target, b, 0.0, reduction, torch.tensor(grad))
        none = ((target < 0) | (target >= V)).cuda()
        assert not got["dx"][none].any() and not torch.isfinite(got["dx"][~none]).any(1).all()
        assert not torch.isfinite(got["dw"]).all() and not torch.isfinite(got["db"]).all()
