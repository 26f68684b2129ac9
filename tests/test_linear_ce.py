"""Cross entropy of a linear projection in pieces of the vocabulary against its definition in 64 bits.

Bounds.  A logit is an fp32 sum of D products of 16-bit values: off by at most D * 2^-23 * sum |x w| =: d (the tensor
cores may truncate, hence a whole step).  A loss is off by at most 2 d plus a few roundings of its terms and the hardware
exponential and logarithm (2^-21 relative to 1 each).  P is off by P * (2 d + 2^-20), then rounded to 16 bits (half a
step, or half the smallest step of fp16 at its factor of 2^15); the gradients are sums of such errors times |w| or |x|,
the fp32 sums of their terms, and the final rounding.
"""
import os
import subprocess
import sys

import pytest
import torch

from metaseq_b200.ops import _lib
from metaseq_b200.ops import autograd as ag
from metaseq_b200.ops import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
IGN = 1


def _inputs(n, V, D, dtype, device, seed=0, ignored=0.0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, D, generator=g).to(dtype)
    w = (torch.randn(V, D, generator=g) * (spread / D ** 0.5)).to(dtype)
    t = torch.randint(0, V, (n,), generator=g)
    if V > IGN + 1:
        t[t == IGN] = 0  # nothing is ignored by chance
    t[torch.rand(n, generator=g) < ignored] = IGN
    return x.to(device), w.to(device), t.to(device)


class _Oracle:
    def __init__(self, x, w, t, g=1.0):
        dtype = x.dtype
        eps = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
        x, w, t = x.detach().cpu().double(), w.detach().cpu().double(), t.cpu()
        keep = t != IGN
        D = x.shape[1]
        x = torch.where(keep[:, None], x, torch.zeros_like(x))
        z = x @ w.t()
        d = (x.abs() @ w.abs().t()).amax(1) * (D + 8) * 2.0 ** -23
        lse = torch.logsumexp(z, 1)
        hit = z.gather(1, t.clamp(0, len(w) - 1)[:, None]).squeeze(1)
        self.loss = (lse - hit) * keep
        self.loss_off = (2 * d + 2.0 ** -20 + (lse.abs() + hit.abs()) * 2.0 ** -22) * keep
        p = torch.exp(z - lse[:, None])
        p_off = p * (2 * d[:, None] + 2.0 ** -19)
        p.scatter_add_(1, t.clamp(0, len(w) - 1)[:, None], -torch.ones(len(t), 1, dtype=torch.float64))
        low = 2.0 ** -25 / 32768 if dtype == torch.float16 else 0.0
        p_off = (p_off + (p.abs() + p_off) * eps + low) * keep[:, None]
        p = p * keep[:, None]
        sums = lambda k: (k + 8) * 2.0 ** -23  # noqa: E731
        self.dx, self.dw = g * (p @ w), g * (p.t() @ x)
        self.dx_off = g * (p_off @ w.abs() + (p.abs() @ w.abs()) * sums(len(w)))
        self.dw_off = g * (p_off.t() @ x.abs() + (p.abs().t() @ x.abs()) * sums(len(x)))


def _near(got, want, off):
    fi = torch.finfo(got.dtype)
    off = off + (want.abs() + off) * fi.eps / 2 + fi.smallest_normal * fi.eps
    err = (got.detach().cpu().double() - want).abs()
    assert (err <= off).all(), float((err / off.clamp(min=1e-300)).max())


def _status_ok(device):
    if device == "cuda":
        assert _lib.check_status("cuda") == 0


SIZES = [(1, 1, 8), (1, 2, 64), (3, 257, 72), (37, 1021, 64), (128, 256, 128), (129, 511, 136), (257, 1000, 8), (300, 1283, 520),
         (513, 300, 328)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ignored", [0.0, 0.5])
@pytest.mark.parametrize("n,V,D", SIZES)
def test_loss_and_gradients(device, dtype, ignored, n, V, D):
    x, w, t = _inputs(n, V, D, dtype, device, n + V, ignored)
    want = _Oracle(x, w, t, 0.5)
    rows = F.linear_cross_entropy(x, w, t, IGN)
    assert rows.dtype == torch.float32 and rows.shape == t.shape
    _near(rows, want.loss, want.loss_off)
    x.requires_grad_(), w.requires_grad_()
    loss = ag.linear_cross_entropy_sum(x, w, t, IGN)
    _near(loss, want.loss.sum(), want.loss_off.sum() + want.loss.abs().sum() * (n + 8) * 2.0 ** -24)
    dx, dw = torch.autograd.grad(loss * 0.5, (x, w))
    _status_ok(device)
    assert dx.dtype == dtype and dw.dtype == dtype
    _near(dx, want.dx, want.dx_off)
    _near(dw, want.dw, want.dw_off)
    assert (dx.cpu()[t.cpu() == IGN] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_one_gradient_only_and_leading_dimensions(device):
    x, w, t = _inputs(60, 300, 64, torch.bfloat16, device, 4, 0.2)
    want = _Oracle(x, w, t)
    xs, ts = x.view(5, 12, 64), t.view(5, 12)
    for need_x, need_w in ((True, False), (False, True)):
        a, b = xs.detach().clone().requires_grad_(need_x), w.detach().clone().requires_grad_(need_w)
        ag.linear_cross_entropy_sum(a, b, ts, IGN).backward()
        if need_x:
            _near(a.grad.view(60, 64), want.dx, want.dx_off)
        if need_w:
            _near(b.grad, want.dw, want.dw_off)
    assert F.linear_cross_entropy(xs, w, ts, IGN).shape == (5, 12)
    with torch.no_grad():
        assert not ag.linear_cross_entropy_sum(xs, w.requires_grad_(), ts, IGN).requires_grad


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [0, 5, 300])
def test_nothing_to_learn_from(device, n):
    x = torch.full((n, 64), float("nan"), dtype=torch.half, device=device, requires_grad=True)
    w = torch.randn(100, 64, device=device).half().requires_grad_()
    t = torch.full((n,), IGN, device=device)
    loss = ag.linear_cross_entropy_sum(x, w, t, IGN)
    loss.backward()
    assert loss.item() == 0 and (x.grad == 0).all() and x.grad.shape == x.shape and (w.grad == 0).all()
    _status_ok(device)


@pytest.mark.parametrize("device", DEVICES)
def test_what_stands_in_ignored_rows_reaches_nothing(device):
    x, w, t = _inputs(300, 513, 64, torch.bfloat16, device, 6, 0.4)
    results = []
    for fill in (0.0, float("nan"), float("inf")):
        a = torch.where((t == IGN)[:, None], torch.full_like(x, fill), x).requires_grad_()
        b = w.detach().clone().requires_grad_()
        loss = ag.linear_cross_entropy_sum(a, b, t, IGN)
        loss.backward()
        results.append((loss.detach(), a.grad, b.grad))
    for other in results[1:]:
        for got, first in zip(other, results[0]):
            assert torch.equal(got, first)
    want = _Oracle(x, w, t)
    _near(results[0][2], want.dw, want.dw_off)


@pytest.mark.parametrize("device", DEVICES)
def test_targets_outside_the_vocabulary_and_values_that_are_not_finite(device):
    x, w, t = _inputs(40, 70, 64, torch.half, device, 8)
    t[3], t[9] = 70, -100
    rows = F.linear_cross_entropy(x, w, t, IGN)
    bad = torch.zeros(40, dtype=torch.bool)
    bad[3] = bad[9] = True
    assert torch.equal(torch.isnan(rows).cpu(), bad)
    x, w, t = _inputs(40, 70, 64, torch.half, device, 8)
    clean = F.linear_cross_entropy(x, w, t, IGN)
    x[7, 5] = float("nan")
    rows = F.linear_cross_entropy(x, w, t, IGN)
    assert torch.isnan(rows[7]) and torch.equal(rows[:7], clean[:7]) and torch.equal(rows[8:], clean[8:])


@pytest.mark.parametrize("device", DEVICES)
def test_large_logits(device):
    """A confident model: logits of a few hundred, losses next to zero and far from it."""
    x, w, t = _inputs(100, 300, 64, torch.bfloat16, device, 9, spread=100.0)
    t[:50] = (x[:50].float() @ w.float().t()).argmax(1)
    want = _Oracle(x, w, t)
    assert float(want.loss.max()) > 100 and float(want.loss.min()) < 1e-3
    _near(F.linear_cross_entropy(x, w, t, IGN), want.loss, want.loss_off)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.half, torch.float32])
def test_weight_gradient_into_a_buffer(device, dtype):
    """A parameter that carries a view of a flat gradient buffer: filled first, added to afterwards; also of 32 bits."""
    x, w, t = _inputs(200, 330, 64, torch.half, device, 10, 0.1)
    want = _Oracle(x, w, t)
    w = torch.nn.Parameter(w)
    buffer = torch.full((2, 330 * 64), float("nan"), dtype=dtype, device=device)
    w._grad_view, w._grad_filled = buffer[1].view(330, 64), False
    ag.linear_cross_entropy_sum(x, w, t, IGN).backward()
    assert w.grad is None and w._grad_filled
    _near(w._grad_view, want.dw, want.dw_off + want.dw.abs() * 2.0 ** -11 + 2.0 ** -25)
    ag.linear_cross_entropy_sum(x, w, t, IGN).backward()
    _near(w._grad_view, 2 * want.dw, 2 * want.dw_off + 2 * want.dw.abs() * 2.0 ** -11 + 2.0 ** -24)
    assert torch.isnan(buffer[0]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_strided_operands(device):
    x, w, t = _inputs(70, 130, 64, torch.bfloat16, device, 11)
    want = _Oracle(x, w, t)
    wide_x = torch.zeros(70, 96, dtype=x.dtype, device=device)
    wide_w = torch.zeros(130, 80, dtype=x.dtype, device=device)
    wide_x[:, 8:72], wide_w[:, 16:80] = x, w
    odd_x = torch.zeros(70, 67, dtype=x.dtype, device=device)
    odd_x[:, 3:] = x
    for a in (wide_x[:, 8:72], odd_x[:, 3:], x.t().contiguous().t()):
        a = a.detach().requires_grad_()
        b = wide_w[:, 16:80].detach().requires_grad_()
        ag.linear_cross_entropy_sum(a, b, t, IGN).backward()
        _near(a.grad, want.dx, want.dx_off)
        _near(b.grad, want.dw, want.dw_off)


def test_fp32_and_gradients_by_differences():
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(6, 5, generator=g), torch.randn(9, 5, generator=g)
    t = torch.tensor([0, 8, IGN, 3, 3, IGN])
    x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(ag.linear_cross_entropy_sum(x, w, t, IGN), (x, w))
    h = 1e-4

    def loss(a, b):
        z = a.double() @ b.double().t()
        keep = t != IGN
        return (torch.logsumexp(z, 1) - z.gather(1, t[:, None]).squeeze(1))[keep].sum()

    for p, d in ((x, dx), (w, dw)):
        for i in range(p.numel()):
            up, down = p.detach().double().clone(), p.detach().double().clone()
            up.view(-1)[i] += h
            down.view(-1)[i] -= h
            pair = (up, w.detach()), (down, w.detach())
            if p is w:
                pair = (x.detach(), up), (x.detach(), down)
            num = (loss(*pair[0]) - loss(*pair[1])) / (2 * h)
            # the third derivative of a log-sum-exp is at most |x|^3: h^2 / 6 of it, next to fp32's own error
            assert abs(float(num) - float(d.view(-1)[i])) < 30 * h * h + 1e-5


def test_refusals():
    x, w, t = _inputs(4, 10, 8, torch.float32, "cpu")
    for args, text in [((x, w[:, :7], t), "do not multiply"), ((x, w, t[:3]), "does not go with"), ((x, w, t.int()), "int64"),
                       ((x.half(), w, t), "one floating type"), ((x, w[:0], t), "no elements"), ((x, w.to("meta"), t), "different devices")]:
        with pytest.raises(ValueError, match=text):
            F.linear_cross_entropy(*args, IGN)
    _, _, saved = F.linear_cross_entropy_fwd(x, w, t, IGN)
    with pytest.raises(ValueError, match="accumulate needs"):
        F.linear_cross_entropy_bwd(saved, w, t, torch.ones(()), IGN, accumulate=True)
    with pytest.raises(ValueError, match="dw_out is"):
        F.linear_cross_entropy_bwd(saved, w, t, torch.ones(()), IGN, dw_out=torch.zeros(9, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,D", [(2000, 50257, 72), (5000, 33000, 128), (70, 50272, 768), (9000, 30011, 64)])
def test_several_pieces_and_long_vocabularies(n, V, D):
    x, w, t = _inputs(n, V, D, torch.bfloat16, "cuda", 12, 0.1)
    xg, wg = x.requires_grad_(), w.requires_grad_()
    loss = ag.linear_cross_entropy_sum(xg, wg, t, IGN)
    dx, dw = torch.autograd.grad(loss, (xg, wg))
    _status_ok("cuda")
    rows = torch.randperm(n)[:64].cuda()
    sub = _Oracle(x[rows], w, t[rows])
    _near(dx[rows], sub.dx, sub.dx_off)
    # columns of dw: the exact column from all rows, in 64 bits on the device
    keep = t != IGN
    xd, wd = x.detach().double() * keep[:, None], w.detach().double()
    z = xd @ wd.t()
    lse = torch.logsumexp(z, 1)
    cols = torch.cat([torch.randperm(V)[:50], torch.tensor([0, V - 1])]).cuda()
    q = (torch.exp(z[:, cols] - lse[:, None]) - (t[:, None] == cols).double()) * keep[:, None]
    want = (q.t() @ xd).cpu()
    d = (x.detach().abs().double() @ wd.abs()[cols].t()).amax() * (D + 8) * 2.0 ** -23
    p_off = (q.abs() + (t[:, None] == cols).double()) * (2 * d + 2.0 ** -19) + q.abs() * 2.0 ** -8
    off = (p_off.t() @ xd.abs() + (q.abs().t() @ xd.abs()) * (n + 8) * 2.0 ** -23).cpu()
    _near(dw[cols], want, off)
    total = ((lse - z.gather(1, t[:, None]).squeeze(1)) * keep).sum().cpu()
    _near(loss, total, total * (n + 64) * 2.0 ** -24 + n * 4e-6)


@pytest.mark.gpu
def test_graph_replay_with_other_inputs_and_two_streams():
    x, w, t = _inputs(500, 1300, 128, torch.bfloat16, "cuda", 13, 0.2)

    def both(a, b, c):
        loss, total, saved = F.linear_cross_entropy_fwd(a, b, c, IGN)
        dx, dw = F.linear_cross_entropy_bwd(saved, b, c, torch.ones((), device="cuda"), IGN)
        return loss, total, dx, dw

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(x, w, t)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(x, w, t)
    for seed, ignored in ((14, 0.0), (15, 0.9)):
        x2, w2, t2 = _inputs(500, 1300, 128, torch.bfloat16, "cuda", seed, ignored)
        x.copy_(x2), w.copy_(w2), t.copy_(t2)
        graph.replay()
        for got, want in zip(out, both(x2, w2, t2)):
            assert torch.equal(got, want)
    # two calls at once, on two streams
    a, b = _inputs(500, 1300, 128, torch.bfloat16, "cuda", 16), _inputs(700, 900, 64, torch.half, "cuda", 17)
    want_a, want_b = both(*a), both(*b)
    torch.cuda.synchronize()
    for _ in range(3):
        got_a = both(*a)
        with torch.cuda.stream(side):
            got_b = both(*b)
        torch.cuda.synchronize()
        assert all(map(torch.equal, got_a, want_a)) and all(map(torch.equal, got_b, want_b))
    _status_ok("cuda")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [1, 60])
def test_operands_at_odd_addresses(device, n):
    """Contiguous views at an odd element offset (``contiguous()`` gives them back as they are), and a single row of a wider
    matrix, which counts as contiguous whatever its row stride."""
    x, w, t = _inputs(n, 130, 64, torch.bfloat16, device, 21)
    want = _Oracle(x, w, t)

    def shifted(a, by):
        return torch.zeros(a.numel() + by, dtype=a.dtype, device=device)[by:].view(a.shape).copy_(a)

    def one_of_many(a):
        return torch.zeros(3, 67, dtype=a.dtype, device=device)[:1, :64].copy_(a)

    views = [shifted(x, 1), shifted(x, 4)] + ([one_of_many(x)] if n == 1 else [])
    for a in views:
        assert a.is_contiguous()
        for b in (w, shifted(w, 3)):
            _near(F.linear_cross_entropy(a, b, t, IGN), want.loss, want.loss_off)
            a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
            ag.linear_cross_entropy_sum(a, b, t, IGN).backward()
            _near(a.grad, want.dx, want.dx_off)
            _near(b.grad, want.dw, want.dw_off)
    _status_ok(device)


@pytest.mark.gpu
def test_weight_gradient_added_to_an_odd_buffer_is_rounded_once():
    """A buffer of the weight's type that the kernel cannot write (not 16-byte aligned) gets the bits that an aligned one gets."""
    x, w, t = _inputs(120, 330, 64, torch.bfloat16, "cuda", 22, 0.1)
    _, _, saved = F.linear_cross_entropy_fwd(x, w, t, IGN)
    g = torch.ones((), device="cuda")
    old = torch.randn(330, 64, device="cuda").bfloat16()
    for accumulate in (False, True):
        aligned = old.clone()
        F.linear_cross_entropy_bwd(saved, w, t, g, IGN, dw_out=aligned, accumulate=accumulate)
        for odd in (torch.zeros(330 * 64 + 1, dtype=old.dtype, device="cuda")[1:].view(330, 64), torch.zeros(330, 67, dtype=old.dtype, device="cuda")[:, 1:65]):
            odd.copy_(old)
            _, dw = F.linear_cross_entropy_bwd(saved, w, t, g, IGN, need_dx=False, dw_out=odd, accumulate=accumulate)
            assert dw is odd and torch.equal(odd, aligned)
    _status_ok("cuda")


def test_workspace_queries_answer_without_a_device():
    """The size of the scratch depends on the device: without one the query says so and does not end the process."""
    if not _lib.kernels_built():
        pytest.skip("library not built")
    code = ("from metaseq_b200.ops import _lib; lib = _lib.kernels(); "
            "print(lib.msq_lce_saved_bytes(100, 200, 64), lib.msq_lce_fwd_bytes(100, 200, 64), lib.msq_lce_bwd_bytes(100, 200, 64, 1, 1))")
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env={**os.environ, "CUDA_VISIBLE_DEVICES": ""})
    assert run.returncode == 0, run.stderr
    saved, fwd, bwd = map(int, run.stdout.split())
    assert saved > 2 * 100 * 64 and fwd > 0 and bwd == -1


def test_failed_launches_are_reported():
    """Without a device no kernel starts: the first launch of a call says so (what follows reads what it leaves)."""
    if not _lib.kernels_built():
        pytest.skip("library not built")
    code = ("import torch; from metaseq_b200.ops import _lib; lib = _lib.kernels(); b = torch.zeros(1 << 16); p = b.data_ptr() + 63 & ~63; "
            "print(lib.msq_lce_fwd(p, 64, p, 64, p, 4, 8, 64, 1, p, p, p, p, 1, None, None), "
            "lib.msq_lce_bwd(p, 64, p, 4, 8, 64, 1, p, p, p, 64, p, 64, 0, p, 1, None, None))")
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env={**os.environ, "CUDA_VISIBLE_DEVICES": ""})
    assert run.returncode == 0, run.stderr
    assert run.stdout.split() == ["-11", "-10"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,V,D", [(513, 300, 328), (700, 129, 72), (1500, 600, 64)])
def test_weight_gradient_in_parts_is_added_to_a_buffer(dtype, n, V, D):
    """Sizes whose rows are cut into parts: fp32 slabs, joined into the buffer when it is filled and when it is added to."""
    lib = _lib.kernels()
    assert lib.msq_lce_bwd_bytes(n, V, D, 0, 1) > lib.msq_lce_bwd_bytes(n, V, D, 0, 0)  # the slabs
    x, w, t = _inputs(n, V, D, dtype, "cuda", 23, 0.1)
    want = _Oracle(x, w, t)
    w = torch.nn.Parameter(w)
    half = torch.finfo(dtype).eps / 2
    wide = torch.full((V, D + 16), 3.0, dtype=dtype, device="cuda")  # rows that lie apart
    for view in (torch.full((V, D), float("nan"), dtype=dtype, device="cuda"), wide[:, 8:8 + D]):
        w._grad_view, w._grad_filled = view, False
        for k in (1, 2, 3):  # micro-batches: every sum is rounded to the buffer's type
            ag.linear_cross_entropy_sum(x, w, t, IGN).backward()
            assert w.grad is None
            _near(view, k * want.dw, k * (1 + 4 * half) * want.dw_off + half * want.dw.abs() * sum(range(1, k)))
    assert (wide[:, :8] == 3.0).all() and (wide[:, 8 + D:] == 3.0).all()
    _status_ok("cuda")


@pytest.mark.gpu
def test_equal_inputs_give_equal_bits():
    """Pieces and parts are added in a fixed order."""
    for n, V, D in ((513, 300, 328), (2000, 30011, 136), (37, 1021, 64)):
        x, w, t = _inputs(n, V, D, torch.bfloat16, "cuda", 24, 0.2)
        results = []
        for _ in range(4):
            loss, total, saved = F.linear_cross_entropy_fwd(x, w, t, IGN)
            results.append((loss, total, *F.linear_cross_entropy_bwd(saved, w, t, torch.ones((), device="cuda"), IGN)))
        for other in results[1:]:
            assert all(map(torch.equal, other, results[0]))
    _status_ok("cuda")
