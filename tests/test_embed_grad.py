"""Embedding gradient by sorted tokens against its definition in 64 bits, on the CPU and on the GPU.

Bound of an element: the fp32 sum of its k terms and the product with the scale are off by at most
(k + 2) * 2^-24 * (|old| + scale * sum |dy|), and the one rounding to the table's type by half a step of the result.
"""
import pytest
import torch

from metaseq_b200.ops import _lib
from metaseq_b200.ops import autograd as ag
from metaseq_b200.ops import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _oracle(tokens, dy, rows, scale, pad, start, old):
    """(result, bound of the error before rounding) in 64 bits."""
    tok = tokens.reshape(-1).cpu()
    d = dy.reshape(-1, dy.shape[-1]).cpu().double()
    want = torch.zeros(rows, d.shape[1], dtype=torch.float64) if old is None else old.cpu().double()
    mass = want.abs()
    terms = torch.zeros(rows, 1, dtype=torch.float64)
    keep = (tok != pad) & (tok >= start) & (tok < start + rows)
    idx = tok[keep] - start
    want = want.index_add(0, idx, d[keep] * scale)
    mass = mass.index_add(0, idx, d[keep].abs() * abs(scale))
    terms = terms.index_add(0, idx, torch.ones(len(idx), 1, dtype=torch.float64))
    return want, mass * (terms + 2) * 2.0 ** -24


def _check(got, want, bound):
    eps = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2  # half a step below the normal range
    off = (got.cpu().double() - want).abs()
    assert (off <= bound * 1.01 + eps * (want.abs() + bound) + tiny).all(), float((off - bound - eps * want.abs()).max())


def _tokens(kind, n, rows, start, g):
    if kind == "uniform":
        return torch.randint(start, start + rows, (n,), generator=g)
    if kind == "frequent":  # a few tokens make up most of the batch: runs that cross many pieces
        t = torch.randint(start, start + rows, (n,), generator=g)
        t[torch.rand(n, generator=g) < 0.8] = start + rows // 2
        return t
    if kind == "one":
        return torch.full((n,), start + rows - 1)
    if kind == "outside":  # half of them belong to other partitions, on either side
        return torch.randint(start - rows, start + 2 * rows, (n,), generator=g)
    if kind == "ascending":
        return start + torch.arange(n) % rows
    raise ValueError(kind)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["uniform", "frequent", "one", "outside", "ascending"])
@pytest.mark.parametrize("n,rows,D", [(1, 1, 8), (7, 3, 8), (33, 130, 264), (257, 511, 520), (1000, 513, 64), (5003, 2050, 136)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_against_the_definition(device, dtype, kind, n, rows, D, accumulate):
    g = torch.Generator().manual_seed(n * 31 + D)
    start, pad = 100, 100 + rows // 3 if rows > 1 else -5
    tokens = _tokens(kind, n, rows, start, g).to(device)
    dy = torch.randn(n, D, generator=g).to(dtype).to(device)
    old = torch.randn(rows, D, generator=g).to(dtype).to(device) if accumulate else None
    want, bound = _oracle(tokens, dy, rows, 1.5, pad, start, old)
    out = old.clone() if accumulate else None
    got = F.embed_grad_sorted(tokens, dy, rows, 1.5, pad, start, out=out, accumulate=accumulate)
    assert got.dtype == dtype and (out is None or got is out)
    _check(got, want, bound)
    if accumulate:
        named = torch.zeros(rows, dtype=torch.bool)
        t = tokens.cpu()
        named[t[(t != pad) & (t >= start) & (t < start + rows)] - start] = True
        assert torch.equal(got.cpu()[~named], old.cpu()[~named])


@pytest.mark.parametrize("device", DEVICES)
def test_no_tokens_at_all(device):
    tokens = torch.empty(0, 5, dtype=torch.long, device=device)
    dy = torch.empty(0, 5, 16, dtype=torch.bfloat16, device=device)
    assert torch.equal(F.embed_grad_sorted(tokens, dy, 9).float().cpu(), torch.zeros(9, 16))
    out = torch.ones(9, 16, dtype=torch.bfloat16, device=device)
    assert (F.embed_grad_sorted(tokens, dy, 9, out=out, accumulate=True) == 1).all()
    # a batch of padding: nothing is added, and what stands in the padded rows does not matter
    tokens = torch.full((4,), 3, device=device)
    dy = torch.full((4, 16), float("nan"), dtype=torch.bfloat16, device=device)
    assert (F.embed_grad_sorted(tokens, dy, 9, pad_idx=3) == 0).all()
    assert (F.embed_grad_sorted(tokens, dy, 9, pad_idx=3, out=out, accumulate=True) == 1).all()


@pytest.mark.parametrize("device", DEVICES)
def test_strided_operands(device):
    g = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, 40, (6, 11), generator=g).to(device)
    wide = torch.randn(6, 11, 48, generator=g).half().to(device)
    dy = wide[..., 8:40]  # rows 48 apart, 16-byte aligned
    store = torch.zeros(40, 64, dtype=torch.half, device=device)
    want, bound = _oracle(tokens, dy, 40, 1.0, -1, 0, store[:, 16:48])
    _check(F.embed_grad_sorted(tokens, dy, 40, out=store[:, 16:48], accumulate=True), want, bound)
    assert (store[:, :16] == 0).all() and (store[:, 48:] == 0).all()
    odd = wide[..., 3:35]  # not aligned
    want, bound = _oracle(tokens, odd, 40, 1.0, -1, 0, None)
    _check(F.embed_grad_sorted(tokens, odd, 40), want, bound)
    broadcast = torch.ones((), dtype=torch.half, device=device).expand(6, 11, 32)  # the gradient of a sum
    want, bound = _oracle(tokens, broadcast, 40, 1.0, -1, 0, None)
    _check(F.embed_grad_sorted(tokens, broadcast, 40), want, bound)
    _check(F.embed_grad_sorted(tokens.t(), broadcast.transpose(0, 1), 40), want, bound)


def test_refusals():
    tokens, dy = torch.zeros(4, dtype=torch.long), torch.zeros(4, 8)
    with pytest.raises(ValueError, match="int64"):
        F.embed_grad_sorted(tokens.int(), dy, 3)
    with pytest.raises(ValueError, match="does not extend"):
        F.embed_grad_sorted(tokens, dy[:3], 3)
    with pytest.raises(ValueError, match="accumulate needs"):
        F.embed_grad_sorted(tokens, dy, 3, accumulate=True)
    with pytest.raises(ValueError, match="the table is"):
        F.embed_grad_sorted(tokens, dy, 3, out=torch.zeros(4, 8))
    with pytest.raises(ValueError, match="no elements"):
        F.embed_grad_sorted(tokens, dy, 0)
    with pytest.raises(ValueError, match="different devices"):
        F.embed_grad_sorted(tokens, dy.to("meta"), 3)
    with pytest.raises(ValueError, match=r"2\^31"):
        F.embed_grad_sorted(tokens, dy, 1 << 31)


def test_embedding_backward_takes_other_shapes_of_positions():
    """Positions given flat, and 32-bit tokens on the CPU, as the lookup takes them."""
    w = torch.randn(9, 8).requires_grad_()
    p = torch.randn(12, 8).requires_grad_()
    tokens, positions = torch.randint(0, 9, (2, 6)), torch.arange(12)
    ag.embedding(tokens.int(), positions, w, p, 1.0, -1).sum().backward()
    assert torch.equal(p.grad, torch.ones_like(p))
    assert torch.equal(w.grad[:, 0], torch.bincount(tokens.reshape(-1), minlength=9).float())


@pytest.mark.parametrize("device", DEVICES)
def test_embedding_backward_uses_it_for_tokens_and_positions(device):
    torch.manual_seed(0)
    dt = torch.bfloat16
    tok_w = torch.randn(50, 24, device=device, dtype=dt).requires_grad_()
    pos_w = torch.randn(20, 24, device=device, dtype=dt).requires_grad_()
    tokens = torch.randint(0, 50, (3, 17), device=device)
    tokens[:, -4:] = 1
    positions = torch.arange(17, device=device).expand(3, 17) + 2
    positions = torch.where(tokens == 1, torch.ones_like(positions), positions)
    y = ag.embedding(tokens, positions, tok_w, pos_w, 2.0, 1)
    up = torch.randn(y.shape, device=device).to(dt)
    y.backward(up)
    want, bound = _oracle(tokens, up, 50, 2.0, 1, 0, None)
    _check(tok_w.grad, want, bound)
    want, bound = _oracle(positions, up, 20, 1.0, 1, 0, None)
    _check(pos_w.grad, want, bound)


@pytest.mark.gpu
def test_equal_inputs_give_equal_bits_and_graph_replay():
    torch.manual_seed(1)
    tokens = torch.randint(0, 300, (4096,), device="cuda")
    tokens[::3] = 7
    dy = torch.randn(4096, 512, device="cuda", dtype=torch.bfloat16)
    first = F.embed_grad_sorted(tokens, dy, 300)
    for _ in range(5):
        assert torch.equal(F.embed_grad_sorted(tokens, dy, 300), first)
    out = torch.empty_like(first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        F.embed_grad_sorted(tokens, dy, 300, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        F.embed_grad_sorted(tokens, dy, 300, out=out)
    tokens.copy_(torch.randint(0, 300, (4096,), device="cuda"))
    out.fill_(float("nan"))
    graph.replay()
    assert torch.equal(out, F.embed_grad_sorted(tokens, dy, 300))


@pytest.mark.gpu
@pytest.mark.parametrize("n,rows,D", [(70001, 50272, 128), (20000, 300000, 8), (3, 1 << 20, 8), (40000, 2, 2048), (3000, 5000011, 8), (9001, 50272, 72)])
def test_large_batches_and_tables(n, rows, D):
    g = torch.Generator(device="cuda").manual_seed(n)
    tokens = torch.randint(0, rows, (n,), generator=g, device="cuda")
    dy = torch.randn(n, D, generator=g, device="cuda").half()
    want, bound = _oracle(tokens, dy, rows, 1.0, -1, 0, None)
    _check(F.embed_grad_sorted(tokens, dy, rows), want, bound)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_one_row_of_a_wider_matrix(device, accumulate):
    """A single row counts as contiguous whatever its row stride."""
    dy = torch.randn(3, 67, device=device).half()[:1, :64]
    old = torch.randn(9, 64, device=device).half() if accumulate else None
    tokens = torch.tensor([4], device=device)
    want, bound = _oracle(tokens, dy, 9, 1.5, -1, 0, old)
    _check(F.embed_grad_sorted(tokens, dy, 9, 1.5, out=old, accumulate=accumulate), want, bound)
    if accumulate:  # a table of one row
        out = torch.randn(3, 67, device=device).half()[:1, :64]
        want, bound = _oracle(tokens - 4, dy, 1, 1.0, -1, 0, out)
        _check(F.embed_grad_sorted(tokens - 4, dy, 1, out=out, accumulate=True), want, bound)


def _captured(call):
    """A graph of ``call``, which is run once before on another stream."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph


@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype,other", [(torch.half, torch.float32), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16),
                                         (torch.half, torch.bfloat16)])
def test_tables_of_another_type_use_the_kernel(dtype, other, accumulate):
    """Gradients and table of different types: the kernel works in fp32 (its launches are counted, and a captured call repeats)."""
    g = torch.Generator().manual_seed(8)
    tokens = torch.randint(0, 60, (700,), generator=g).cuda()
    dy = torch.randn(700, 40, generator=g).to(dtype).cuda()
    old = torch.randn(60, 40, generator=g).to(other).cuda()
    old[7] = -0.0
    tokens[tokens == 7] = 8
    want, bound = _oracle(tokens, dy, 60, 1.5, 3, 0, old if accumulate else None)
    out, before = old.clone(), _lib.launch_count()
    assert F.embed_grad_sorted(tokens, dy, 60, 1.5, 3, out=out, accumulate=accumulate) is out
    assert _lib.launch_count() > before
    _check(out, want, bound + want.abs() * 2.0 ** -24)  # the fp32 result is rounded before the table's type is
    if accumulate:
        assert torch.equal(out[7], old[7]) and torch.signbit(out[7]).all() and torch.equal(out[3], old[3])
    eager = out.clone()
    graph = _captured(lambda: F.embed_grad_sorted(tokens, dy, 60, 1.5, 3, out=out, accumulate=accumulate))
    out.copy_(old)
    graph.replay()
    assert torch.equal(out, eager)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 2, 12, 100, 777])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("n", [9, 900])
def test_widths_and_addresses_the_kernel_does_not_take_are_copied(dtype, D, accumulate, n):
    """Widths that are no multiple of eight, and tables at odd addresses: copied to and from a layout that the kernel takes."""
    g = torch.Generator().manual_seed(D)
    tokens = torch.randint(0, 50, (n,), generator=g).cuda()
    tokens[tokens == 20] = 21
    dy = torch.randn(n, D, generator=g).to(dtype).cuda()
    space = torch.randn(50 * D + 3, generator=g).to(dtype).cuda()
    old = space[1:1 + 50 * D].view(50, D).clone()
    want, bound = _oracle(tokens, dy, 50, 0.5, 3, 0, old if accumulate else None)
    before = _lib.launch_count()
    if not accumulate:
        got = F.embed_grad_sorted(tokens, dy, 50, 0.5, 3)
        assert got.shape == (50, D) and got.is_contiguous()
        _check(got, want, bound)
    edges = space[[0, -2, -1]].clone()
    out = space[1:1 + 50 * D].view(50, D)
    F.embed_grad_sorted(tokens, dy, 50, 0.5, 3, out=out, accumulate=accumulate)
    assert _lib.launch_count() > before
    _check(out, want, bound)
    assert torch.equal(space[[0, -2, -1]], edges)
    if accumulate:
        assert torch.equal(out[20], old[20]) and torch.equal(out[3], old[3])
    wide = torch.full((50, D + 5), 2.0, dtype=dtype, device="cuda")  # rows that lie apart
    wide[:, :D] = old
    F.embed_grad_sorted(tokens, dy, 50, 0.5, 3, out=wide[:, :D], accumulate=accumulate)
    assert torch.equal(wide[:, :D], out) and (wide[:, D:] == 2.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [12, 16])
def test_embedding_backward_is_captured_at_every_width(D):
    w = torch.nn.Parameter(torch.randn(60, D, device="cuda").half())
    w._grad_view, w._grad_filled = torch.zeros(60 * D + 1, dtype=torch.half, device="cuda")[1:].view(60, D), False
    tokens, up = torch.randint(0, 60, (5, 70), device="cuda"), torch.randn(5, 70, D, device="cuda").half()

    def step():
        w._grad_filled = False
        ag.embedding(tokens, None, w, None, 1.0, 3).backward(up)

    graph = _captured(step)
    tokens.copy_(torch.randint(0, 60, (5, 70), device="cuda"))
    graph.replay()
    want, bound = _oracle(tokens, up, 60, 1.0, 3, 0, None)
    _check(w._grad_view, want, bound)


@pytest.mark.parametrize("accumulate", [False, True])
def test_tensor_form_has_no_shape_that_depends_on_the_tokens(accumulate):
    """On the meta device there are no values: an operation whose result's shape hangs on them raises."""
    tokens = torch.zeros(6, 5, dtype=torch.long, device="meta")
    dy = torch.zeros(6, 5, 12, dtype=torch.half, device="meta")
    out = torch.zeros(9, 12, dtype=torch.half, device="meta") if accumulate else None
    assert F.embed_grad_sorted(tokens, dy, 9, out=out, accumulate=accumulate).shape == (9, 12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_tensor_form_leaves_other_rows_as_they_are(dtype):
    out = torch.full((4, 3), -0.0, dtype=dtype)
    out[1] = 1.0 / 3.0
    old = out.clone()
    dy = torch.full((3, 3), float("nan"), dtype=dtype)
    dy[0] = 2.0
    F.embed_grad_sorted(torch.tensor([2, 7, 3]), dy, 4, pad_idx=3, out=out, accumulate=True)
    assert torch.equal(out[[0, 1, 3]], old[[0, 1, 3]]) and torch.signbit(out[[0, 3]]).all() and (out[2] == 2.0).all()


@pytest.mark.gpu
def test_tensor_form_is_captured():
    tokens = torch.randint(0, 60, (300,), device="cuda")
    dy = torch.randn(300, 12, device="cuda").half()
    out = torch.ones(60, 12, device="cuda").half()

    def step():
        F.set_backend("torch")
        try:
            F.embed_grad_sorted(tokens, dy, 60, 1.0, 3, out=out, accumulate=True)
        finally:
            F.set_backend("auto")

    graph = _captured(step)
    out.fill_(1.0)
    graph.replay()
    want, bound = _oracle(tokens, dy, 60, 1.0, 3, 0, torch.ones(60, 12))
    _check(out, want, bound)


@pytest.mark.gpu
def test_fp32_embedding_runs_without_the_library(monkeypatch):
    """Without the built library 32-bit tensors take tensor operations, in both directions; 16-bit ones are refused."""
    monkeypatch.setattr(_lib, "kernels_built", lambda: False)
    w = torch.randn(20, 16, device="cuda").requires_grad_()
    tokens = torch.randint(0, 20, (3, 7), device="cuda")
    up = torch.randn(3, 7, 16, device="cuda")
    ag.embedding(tokens, None, w, None, 2.0, 1).backward(up)
    want, bound = _oracle(tokens, up, 20, 2.0, 1, 0, None)
    _check(w.grad, want, bound)
    with pytest.raises(RuntimeError, match="not built"):
        F.embed_grad_sorted(tokens, up.half(), 20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n,rows,D", [(torch.float32, 3000, 30011, 1000), (torch.float32, 700, 20011, 1032), (torch.bfloat16, 5000, 50272, 776),
                                            (torch.float16, 300, 41003, 1544), (torch.bfloat16, 70001, 60007, 520)])
@pytest.mark.parametrize("kind", ["uniform", "frequent"])
def test_new_tables_larger_than_what_is_cleared_beside_the_sort(dtype, n, rows, D, kind):
    """Tables over 40 MB of wide rows: the rows behind that are cleared unless a token names them."""
    assert rows * D * dtype.itemsize > 40 << 20
    tokens = _tokens(kind, n, rows, 0, torch.Generator().manual_seed(n))
    tokens[:3] = torch.tensor([0, rows - 1, rows - 2])
    tokens = tokens.cuda()
    dy = torch.randn(n, D, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda").to(dtype)
    out = torch.full((rows, D), float("nan"), dtype=dtype, device="cuda")
    F.embed_grad_sorted(tokens, dy, rows, 1.5, 1, out=out)
    keep = tokens != 1
    named, place = torch.unique(tokens[keep], return_inverse=True)
    want, bound = _oracle(place, dy[keep], len(named), 1.5, -1, 0, None)
    _check(out[named], want, bound)
    out[named] = 0
    assert (out == 0).all()


@pytest.mark.gpu
def test_pairs_at_odd_addresses():
    """16-bit tensors at an odd element offset: the kernels that read or write two values at once are not given them."""
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 40, (300,), generator=g).cuda()
    space = torch.randn(300 * 12 + 1, generator=g).half().cuda()
    dy = space[1:].view(300, 12)
    assert dy.is_contiguous() and dy.data_ptr() % 4 == 2
    want, bound = _oracle(tokens, dy, 40, 1.5, 3, 0, None)
    table, _ = F.embed_bwd(tokens, None, dy, 40, 0, 1.5, 3, need_pos=False)
    _check(table, want, bound)
    for accumulate in (False, True):
        room = torch.ones(40 * 12 + 2, dtype=torch.half, device="cuda")
        F.fold_fp32_into(table, room[1:-1].view(40, 12), accumulate)
        assert torch.equal(room[1:-1].view(40, 12), (table + float(accumulate)).half()) and room[0] == 1 and room[-1] == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [12, 100, 18])
@pytest.mark.parametrize("views", [False, True])
def test_embedding_backward_of_even_widths_scatters(monkeypatch, dtype, D, views):
    """16-bit rows of an even width that is no multiple of eight: the kernel that scatters with atomics, for both tables."""
    calls, scatter = [], F.embed_bwd
    monkeypatch.setattr(F, "embed_bwd", lambda *a, **k: calls.append(1) or scatter(*a, **k))
    g = torch.Generator().manual_seed(D)
    tok_w, pos_w = (torch.nn.Parameter(torch.randn(k, D, generator=g).to(dtype).cuda()) for k in (50, 30))
    tokens = torch.randint(0, 50, (4, 25), generator=g).cuda()
    tokens[2, 9:] = 1
    positions = torch.where(tokens == 1, 1, torch.arange(25, device="cuda") + 2)
    up = torch.randn(4, 25, D, generator=g).to(dtype).cuda()
    if views:
        for w in (tok_w, pos_w):
            w._grad_view, w._grad_filled = torch.full(w.shape, float("nan"), dtype=dtype, device="cuda"), False
    before = _lib.launch_count()
    ag.embedding(tokens, positions, tok_w, pos_w, 2.0, 1).backward(up)
    assert calls == [1] and _lib.launch_count() > before
    for w, index, scale in ((tok_w, tokens, 2.0), (pos_w, positions, 1.0)):
        want, bound = _oracle(index, up, len(w), scale, 1, 0, None)
        _check(w._grad_view if views else w.grad, want, bound)
        assert not views or w.grad is None
    if not views:
        tok_w.grad = None
        ag.embedding(tokens, positions[:1], tok_w, None, 2.0, 1).backward(up)  # no position table: the numbers are not looked at
        want, bound = _oracle(tokens, up, 50, 2.0, 1, 0, None)
        _check(tok_w.grad, want, bound)
