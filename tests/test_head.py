"""CPU: refusals of the classification-head operators, and their 64-bit restatement against torch's own functions."""
import ctypes

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import head_oracle as ho
from pointnetgpd_amd import _lib, crop, head

ERR_INVALID, ERR_SHAPE, ERR_WORKSPACE = 1, 2, 5


def test_no_cpu_fallback():
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        head.linear(x, w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        head.dropout(x, 0.5, 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        head.linear_cross_entropy(x, w, torch.zeros(2, dtype=torch.int64))


def test_wrong_names_are_refused_before_anything_else():
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    with pytest.raises(ValueError, match="activation"):
        head.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="reduction"):
        head.linear_cross_entropy(x, w, torch.zeros(2, dtype=torch.int64), reduction="batchmean")
    with pytest.raises(TypeError, match="tensor"):
        head.linear([1.0], w)


# every call below fails its checks: nothing is launched and no GPU is needed
def _linear(lib, type=0, M=2, N=3, K=4, x=16, ldx=4, w=16, ldw=4, act=0, r=0, ldr=3, y=16, ws=0, nbytes=0):
    return lib.pngpd_linear_forward(type, M, N, K, x, ldx, w, ldw, None, act, r, ldr, y, None, ws, nbytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(type=3), ERR_INVALID), (dict(type=-1), ERR_INVALID), (dict(M=-1), ERR_SHAPE), (dict(N=0), ERR_SHAPE),
    (dict(K=0), ERR_SHAPE), (dict(M=2 ** 31), ERR_SHAPE), (dict(x=None), ERR_INVALID), (dict(w=None), ERR_INVALID),
    (dict(y=None), ERR_INVALID), (dict(act=5), ERR_INVALID), (dict(ldx=3), ERR_SHAPE), (dict(ldw=3), ERR_SHAPE),
    (dict(r=16, ldr=2), ERR_SHAPE), (dict(K=2 ** 21 + 1, ldx=2 ** 22, ldw=2 ** 22), ERR_SHAPE), (dict(N=2 ** 21 + 1), ERR_SHAPE),
    (dict(M=6, K=5, ldx=5, ldw=5), ERR_INVALID)])      # rows that have to be copied, and no workspace
def test_linear_forward_refuses(change, code):
    lib = _lib.load()
    assert _linear(lib, **change) == code
    assert b"pngpd_linear_forward" in lib.pngpd_last_error()


@pytest.mark.parametrize("change,code", [
    (dict(type=7), ERR_INVALID), (dict(N=0), ERR_SHAPE), (dict(dy=None), ERR_INVALID), (dict(z=None), ERR_INVALID),
    (dict(w=None), ERR_INVALID), (dict(x=None), ERR_INVALID), (dict(ld_dy=2), ERR_SHAPE), (dict(ws=None), ERR_INVALID),
    (dict(nbytes=8), ERR_WORKSPACE), (dict(ws=24), ERR_INVALID)])
def test_linear_backward_refuses(change, code):
    lib = _lib.load()
    a = dict(type=0, M=2, N=3, K=4, dy=16, ld_dy=3, z=16, x=16, w=16, act=1, ws=4096, nbytes=1 << 20)
    a.update(change)
    rc = lib.pngpd_linear_backward(a["type"], a["M"], a["N"], a["K"], a["dy"], a["ld_dy"], a["z"], a["x"], 4, a["w"], 4, a["act"],
                                   16, 16, 16, a["ws"], a["nbytes"], None)
    assert rc == code and b"pngpd_linear_backward" in lib.pngpd_last_error()


@pytest.mark.parametrize("change,code", [
    (dict(type=9), ERR_INVALID), (dict(rows=-1), ERR_SHAPE), (dict(cols=0), ERR_SHAPE), (dict(p=1.5), ERR_INVALID),
    (dict(p=-0.1), ERR_INVALID), (dict(p=float("nan")), ERR_INVALID), (dict(x=None), ERR_INVALID), (dict(y=None), ERR_INVALID),
    (dict(ldx=3), ERR_SHAPE)])
def test_dropout_refuses(change, code):
    lib = _lib.load()
    a = dict(type=0, rows=2, cols=4, x=16, ldx=4, y=16, p=0.5)
    a.update(change)
    rc = lib.pngpd_dropout(a["type"], a["rows"], a["cols"], a["x"], a["ldx"], None, 4, a["y"], a["p"], 1, 0, None, None)
    assert rc == code and b"pngpd_dropout" in lib.pngpd_last_error()


@pytest.mark.parametrize("change,code", [
    (dict(type=-2), ERR_INVALID), (dict(T=-1), ERR_SHAPE), (dict(V=0), ERR_SHAPE), (dict(D=0), ERR_SHAPE),
    (dict(x=None), ERR_INVALID), (dict(w=None), ERR_INVALID), (dict(target=None), ERR_INVALID), (dict(eps=1.5), ERR_INVALID),
    (dict(eps=float("nan")), ERR_INVALID), (dict(reduction=3), ERR_INVALID), (dict(ldw=3), ERR_SHAPE),
    (dict(lse=None), ERR_INVALID), (dict(out=None), ERR_INVALID), (dict(V=2 ** 24 + 1), ERR_SHAPE), (dict(D=2 ** 21 + 1, ldw=2 ** 22), ERR_SHAPE), (dict(ws=None), ERR_INVALID), (dict(nbytes=64), ERR_WORKSPACE), (dict(kept=24), ERR_INVALID)])
def test_linear_cross_entropy_refuses(change, code):
    lib = _lib.load()
    a = dict(type=0, T=2, V=5, D=4, x=16, w=16, ldw=4, target=16, eps=0.0, reduction=1, lse=16, out=16, kept=None, ws=4096, nbytes=1 << 20)
    a.update(change)
    args = (a["type"], a["T"], a["V"], a["D"], a["x"], 4, a["w"], a["ldw"], None, a["target"], -100, a["eps"], a["reduction"])
    assert lib.pngpd_linear_cross_entropy_forward(*args, a["out"], a["lse"], a["kept"], a["ws"], a["nbytes"], None) == code
    assert b"pngpd_linear_cross_entropy_forward" in lib.pngpd_last_error()
    assert lib.pngpd_linear_cross_entropy_backward(*args, a["lse"], a["kept"], a["out"], 16, 16, 16, a["ws"], a["nbytes"], None) == code
    assert b"pngpd_linear_cross_entropy_backward" in lib.pngpd_last_error()


def test_workspace_sizes_are_bounded_and_grow_with_no_logits():
    lib = _lib.load()
    whole = 8192 * 131072 * 4
    assert 0 < lib.pngpd_linear_cross_entropy_workspace_bytes(1, 8192, 131072, 1024, 0, 1) < whole // 8
    assert 0 < lib.pngpd_linear_cross_entropy_workspace_bytes(1, 8192, 131072, 1024, 1, 1) < whole // 8
    assert lib.pngpd_linear_workspace_bytes(5, 1, 1, 1, 0, 1) == 0
    kept = lib.pngpd_linear_cross_entropy_kept_bytes
    assert kept(0, 1023, 10007, 1000) == 1023 * 10008 * 4      # rows of whole 16-byte chunks
    assert kept(1, 8192, 131072, 1024) == kept(2, 1024, 8192, 128) == kept(0, 4096, 131072, 1024) == 0
    assert kept(0, 256, 3, 256) == 256 + 256 * 4 * 4 and kept(1, 77, 8, 99) == 256 + 77 * 8 * 4      # few classes
    assert kept(0, 2 ** 30, 8, 2) == kept(2, 256, 9, 256) == 0
    assert kept(0, 1024, 8192, 16) == kept(0, 0, 8192, 1024) == kept(7, 1024, 8192, 1024) == 0


def test_a_missing_binding_is_an_error(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_head", None)
    monkeypatch.setattr(_lib, "HEAD_PATH", str(tmp_path / "_head.so"))
    with pytest.raises(ImportError, match="not found"):
        _lib.load_head()


# ---- the restatement itself -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("name", [None, "relu", "gelu", "gelu_tanh", "silu"])
def test_restated_linear_is_torchs(name):
    g = torch.Generator().manual_seed(3)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_() for s in ((7, 5), (6, 5), (6,)))
    r, dy = torch.randn(7, 6, generator=g, dtype=torch.float64), torch.randn(7, 6, generator=g, dtype=torch.float64)
    fn = {None: lambda v: v, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda v: F.gelu(v, approximate="tanh"),
          "silu": F.silu}[name]
    y = fn(F.linear(x, w, b)) + r
    grads = torch.autograd.grad(y, (x, w, b), dy)
    out = ho.linear(x.detach(), w.detach(), b.detach(), name, r, dy)
    for key, want in zip(("y", "dx", "dw", "db"), (y.detach(), *grads)):
        torch.testing.assert_close(out[key][0], want, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("eps", [0.0, 0.2])
def test_restated_cross_entropy_is_torchs(reduction, eps):
    g = torch.Generator().manual_seed(4)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_() for s in ((9, 5), (11, 5), (11,)))
    target = torch.tensor([0, 10, -100, 3, 3, -100, 7, 1, 2])
    loss = F.cross_entropy(F.linear(x, w, b), target, label_smoothing=eps, reduction=reduction)
    dloss = torch.rand(loss.shape, generator=g, dtype=torch.float64)
    grads = torch.autograd.grad(loss, (x, w, b), dloss)
    out = ho.cross_entropy(x.detach(), w.detach(), target, b.detach(), -100, eps, reduction, dloss)
    for key, want in zip(("loss", "dx", "dw", "db"), (loss.detach(), *grads)):
        torch.testing.assert_close(out[key][0], want, rtol=1e-12, atol=1e-12)


def test_keep_mask_uses_the_selection_generators_hash_and_keeps_its_share():
    v = np.array([0, 1, 2 ** 63, 2 ** 64 - 1], dtype=np.uint64)
    np.testing.assert_array_equal(ho.mix64(v), crop._mix64(v))
    n = 1 << 20
    for p in (0.0, 0.1, 0.5, 1.0):
        kept = ho.keep_mask(n, p, 11, 5).mean()
        assert abs(kept - (1 - p)) <= 5 * (p * (1 - p) / n) ** 0.5
    a, b = ho.keep_mask(n, 0.5, 11, 5), ho.keep_mask(n, 0.5, 11, 6)
    assert abs((a == b).mean() - 0.5) < 5 * 0.5 / n ** 0.5          # another offset: an independent mask
    assert abs((a[1:] == a[:-1]).mean() - 0.5) < 5 * 0.5 / n ** 0.5


def test_a_planted_mistake_exceeds_the_bounds():
    g = torch.Generator().manual_seed(8)
    x, w = torch.randn(33, 40, generator=g).bfloat16(), torch.randn(21, 40, generator=g).bfloat16()
    y, bound = ho.linear(x, w, None, "silu", None, None)["y"]
    assert ho.worst(y.bfloat16(), y, bound) <= 1.0
    wrong = ho.linear(x[:, :-1], w[:, :-1], None, "silu", None, None)["y"][0]      # the last product left out
    assert ho.worst(wrong.bfloat16(), y, bound) > 10.0
    t = torch.randint(0, 21, (33,), generator=g)
    loss, lb = ho.cross_entropy(x, w, t, None, -100, 0.0, "none", None)["loss"]
    other = ho.cross_entropy(x, w, (t + 1) % 21, None, -100, 0.0, "none", None)["loss"][0]
    assert ho.worst(loss.float(), loss, lb) <= 1.0 and ho.worst(other.float(), loss, lb) > 10.0


def test_forward_mode_is_refused_before_anything_is_launched():
    """A tangent raises in the binding itself, with gradients enabled or not (no_grad leaves forward-mode on in torch)."""
    m, fw = _lib.load_head(), torch.autograd.forward_ad
    x, w, b, t = torch.ones(2, 4), torch.ones(3, 4), torch.ones(3), torch.zeros(2, dtype=torch.int64)
    with fw.dual_level():
        for mode in (torch.no_grad, torch.enable_grad):
            with mode():
                dual = [fw.make_dual(v, torch.ones_like(v)) for v in (x, w, b)]
                for i in range(3):
                    a = [dual[j] if j == i else v for j, v in enumerate((x, w, b))]
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        m.linear(a[0], a[1], a[2], None, 0)
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        m.linear_cross_entropy(a[0], a[1], t, a[2], -100, 0.0, 1, True)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    m.linear(x, w, None, fw.make_dual(torch.ones(2, 3), torch.ones(2, 3)), 0)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    m.dropout(dual[0], None, 0.5, 1, 0, None)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    m.dropout(x, dual[0], 0.5, 1, 0, None)


@pytest.mark.parametrize("type", [0, 1, 2])
def test_few_classes_ask_for_the_memory_they_use(type):
    """At most eight classes: the rows' losses forward, parts of the gradients backward; no copy of x, aligned or not."""
    lib = _lib.load()
    size = lib.pngpd_linear_cross_entropy_workspace_bytes
    for T, V, D in ((192000, 3, 1024), (2 ** 20, 8, 1024), (8192, 3, 4096), (1, 1, 1)):
        parts = 256 * V * (D + 1) * 4 + 255
        for aligned in (0, 1):
            assert size(type, T, V, D, 0, aligned) <= T * 4 + 256 * 16 + 255
            assert size(type, T, V, D, 2, aligned) <= parts < size(type, T, V, D, 1, aligned) + parts
    assert size(type, 192000, 3, 1024, 1, 1) > 192000 * 1024 * 2          # without kept logits the general products run
    assert size(type, 1024, 9, 64, 2, 1) == size(type, 1024, 9, 64, 1, 1)
    # the entries ask for as much
    need = size(type, 8192, 3, 4096, 2, 1)
    args = (type, 8192, 3, 4096, 16, 4096, 16, 4096, None, 16, -100, 0.0, 1)
    assert lib.pngpd_linear_cross_entropy_backward(*args, 16, 16, 16, 16, 16, 16, 4096, need - 1, None) == ERR_WORKSPACE
    assert lib.pngpd_linear_cross_entropy_forward(*args, 16, 16, 16, 4096, size(type, 8192, 3, 4096, 0, 1) - 1, None) == ERR_WORKSPACE


@pytest.mark.parametrize("rows,cols", [(2 ** 21, 2 ** 21 + 1), (1, 2 ** 40 + 1), (2 ** 42 + 1, 1), (2 ** 62, 4)])
def test_dropout_refuses_what_passes_its_own_limits(rows, cols):
    """2^42 elements, 2^40 a row: neither the rows nor a row end at 2^31."""
    lib = _lib.load()
    assert lib.pngpd_dropout(0, rows, cols, 16, cols, None, cols, 16, 0.5, 1, 0, None, None) == ERR_SHAPE
    assert b"2^42" in lib.pngpd_last_error()


@pytest.mark.parametrize("rows,cols", [(1, 2 ** 31 + 9), (2 ** 31 + 9, 1), (2 ** 32, 2 ** 10)])
def test_dropout_takes_more_than_31_bits_of_rows_or_columns(rows, cols):
    """The sizes pass; what is refused is the missing pointer, which is looked at behind them."""
    lib = _lib.load()
    assert lib.pngpd_dropout(0, rows, cols, None, cols, None, cols, None, 0.5, 1, 0, None, None) == ERR_INVALID
    assert b"NULL" in lib.pngpd_last_error()


def test_a_binding_for_another_torch_is_an_error(monkeypatch, tmp_path):
    """The binding is compiled against one version of torch's C++ interface; another's is built again, and not loaded."""
    from pointnetgpd_amd import build
    assert build.built_for(_lib.HEAD_PATH, torch.__version__) and not build.built_for(_lib.HEAD_PATH, torch.__version__ + "1")
    other = tmp_path / "_head.so"
    other.write_bytes(open(_lib.HEAD_PATH, "rb").read().replace(build._mark(torch.__version__).encode(), b"x" * len(build._mark(torch.__version__))))
    monkeypatch.setattr(_lib, "_head", None)
    monkeypatch.setattr(_lib, "HEAD_PATH", str(other))
    with pytest.raises(ImportError, match="not built for this torch"):
        _lib.load_head()
    commands = []
    monkeypatch.setattr(build, "HEAD_PATH", str(other))
    monkeypatch.setattr(build, "_run", commands.append)
    build.build_head()
    assert len(commands) == 1 and any(build._mark(torch.__version__) in word for word in commands[0])
    monkeypatch.setattr(build, "HEAD_PATH", _lib.__file__.replace("_lib.py", "_head.so"))
    commands.clear()
    monkeypatch.setattr(build, "_newer", lambda target, deps: False)
    build.build_head()
    assert not commands


def test_a_host_without_torchs_headers_builds_the_rest(monkeypatch):
    from pointnetgpd_amd import build
    done = []
    for name in ("build_library", "build_example", "build_probe", "build_oracle_c"):
        monkeypatch.setattr(build, name, lambda force=False, name=name: done.append(name))

    def no_headers(force=False):
        raise OSError("torch/extension.h")

    monkeypatch.setattr(build, "build_head", no_headers)
    with pytest.raises(OSError):
        build.build_all()
    assert sorted(done) == ["build_example", "build_library", "build_oracle_c", "build_probe"]


def test_more_tiles_than_a_launch_holds_are_refused():
    """2^23 tiles of 128 x 128 (float32) or 256 x 256: an error that says so, not the runtime's."""
    lib = _lib.load()
    for type, M, N in ((0, 2 ** 30, 1), (0, 2 ** 20, 2 ** 17), (1, 2 ** 31 - 1, 1), (2, 2 ** 22, 2 ** 17)):
        assert _linear(lib, type=type, M=M, N=N, ldr=N) == ERR_SHAPE
        assert b"tiles" in lib.pngpd_last_error()
        rc = lib.pngpd_linear_backward(type, M, 4, N, 16, 4, None, 16, N, 16, N, 0, 16, None, None, None, 0, None)
        assert rc == ERR_SHAPE and b"tiles" in lib.pngpd_last_error()
    # one row less passes the sizes: the missing workspace is refused next
    assert _linear(lib, M=2 ** 30 - 128, N=1, K=5, ldx=5, ldw=5) == ERR_INVALID
    rc = lib.pngpd_linear_backward(0, 8, 2 ** 21, 2 ** 21, 16, 2 ** 21, None, 16, 2 ** 21, 16, 2 ** 21, 0, None, 16, None, None, 0, None)
    assert rc == ERR_SHAPE and b"tiles" in lib.pngpd_last_error()
    args = (0, 2 ** 30, 9, 4, 16, 4, 16, 4, None, 16, -100, 0.0, 1)
    assert lib.pngpd_linear_cross_entropy_backward(*args, 16, None, 16, 16, 16, None, 4096, 1 << 60, None) == ERR_SHAPE
    assert b"tiles" in lib.pngpd_last_error()
