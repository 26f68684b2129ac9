"""AdamW with 8-bit moments: the storage form, the update against its formula in 64 bits, the restatement against the
kernel bit by bit, and the optimizer on top of it."""
import math

import pytest
import torch

from metaseq_b200.ops import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
PAIRS = [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
         (torch.float32, torch.bfloat16), (torch.float32, torch.float16), (torch.float16, torch.float32), (torch.bfloat16, torch.float32)]
HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)
E4M3 = torch.arange(0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).double()  # 0 .. 448 in order


def _items(sizes, pdt, gdt, device, seed, flat=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        p = torch.randn(n, generator=g).to(pdt)
        grad = (torch.randn(n, generator=g) * 10 ** (4 * torch.rand(n, generator=g) - 5)).to(gdt)
        m, ms, r, rs = F.adamw8_state(p)
        m = (torch.randn(n, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        r = (torch.randn(n, generator=g).abs() * 100).clamp(2.0 ** -9, 448).to(torch.float8_e4m3fn)
        ms = torch.exp2(torch.randint(-20, -10, ms.shape, generator=g).float())
        rs = torch.exp2(torch.randint(-20, -10, rs.shape, generator=g).float())
        out.append(tuple(t.to(device) for t in (p, grad, m, ms, r, rs)))
    return out


def _oracle(item, step, gmul=1.0):
    """(p, m, r) after the step in 64 bits, and the sum of the magnitudes that p is made of."""
    p, g, m, ms, r, rs = (t.cpu() for t in item)
    h = HYPER
    g = g.double() * gmul
    m = F.adamw8_decode(m, ms).double() * h["beta1"] + (1 - h["beta1"]) * g
    r = torch.sqrt(F.adamw8_decode(r, rs).double() ** 2 * h["beta2"] + (1 - h["beta2"]) * g * g)
    size = h["lr"] * math.sqrt(1 - h["beta2"] ** step) / (1 - h["beta1"] ** step)
    move = size * m / (r + h["eps"])
    return p.double() * (1 - h["lr"] * h["weight_decay"]) - move, m, r, p.double().abs() + move.abs()


def _check_codes(code, scale, value, root):
    """Scales are the smallest power of two that fits, codes one of the two neighbours of the value."""
    code, scale, value = code.cpu(), scale.cpu().double(), value.abs()
    n = value.numel()
    pad = torch.cat([value, value.new_zeros(-n % 256)]).view(-1, 256)
    top = pad.amax(1)
    assert (torch.log2(scale) == torch.log2(scale).round()).all()
    slack = 1 + 1e-6  # the fp32 value may lie on the other side of a power of two
    live = top > 448 * 2.0 ** -110
    assert (top <= 448 * scale * slack)[live].all() and (top * 2 * slack > 448 * scale)[live].all()
    stored = (code.view(torch.uint8).view(-1) & 0x7F).long()
    assert (stored < 0x7F).all()
    mag = value / scale.repeat_interleave(256)[:n]
    below = (torch.searchsorted(E4M3, mag.clamp(max=448.0), right=True) - 1).clamp(0, 0x7E)
    near = 1e-6 * mag + 1e-9
    ok = (stored == below) | ((stored == below + 1) & (mag > E4M3[below] - near)) | ((stored == below - 1) & (mag <= E4M3[below] + near))
    if root:
        ok &= (stored > 0) | (value == 0)
    assert ok.all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("pdt,gdt", PAIRS)
@pytest.mark.parametrize("sizes", [[1], [255, 256, 257], [7, 4096, 1, 0, 1025, 3], [70001]])
def test_update_against_the_formula(device, pdt, gdt, sizes):
    items = _items(sizes, pdt, gdt, device, 3)
    ctrl = torch.tensor([0.5, 0.0, 0.0, 1.0], device=device)
    wants = [_oracle(it, 7, 0.5) for it in items]
    F.adamw8_step_multi(items, **HYPER, step=7, seed=11, ctrl=ctrl)
    for (p, _, m, ms, r, rs), (wp, wm, wr, mass) in zip(items, wants):
        # a dozen roundings to fp32 of 2^-24, the root's and the quotient's approximations (4 * 2^-24 each), all relative to p
        # or to the step, then half a step of p's type
        eps = torch.finfo(pdt).eps / 2
        bound = 20 * 2.0 ** -24 * mass + eps * wp.abs() * 1.001 + torch.finfo(pdt).smallest_normal * eps
        assert ((p.cpu().double() - wp).abs() <= bound).all()
        if p.numel():
            _check_codes(m, ms, wm, False)
            _check_codes(r, rs, wr, True)
            sign = (m.cpu().view(torch.uint8) > 0x7F)
            assert ((wm.abs() < 1e-12) | (sign == (wm < 0))).all()  # cancelled to nothing: either sign


@pytest.mark.gpu
@pytest.mark.parametrize("pdt,gdt", PAIRS)
@pytest.mark.parametrize("step", [1, 3])
def test_kernel_and_restatement_agree(pdt, gdt, step):
    """On one device (PyTorch's CPU operators fuse some products into the sums that follow, its CUDA operators round every
    operation, as the kernel does): scales and codes are equal bit by bit, the parameters but for the kernel's quotient,
    which is off by four units of 2^-24 and rounded once less."""
    sizes = [5, 256, 1000, 33333, 2, 512] + [110] * 300  # over 256 tensors: two launches
    here, there = _items(sizes, pdt, gdt, "cuda", 5), _items(sizes, pdt, gdt, "cuda", 5)
    F.adamw8_step_multi(here, **HYPER, step=step, seed=(step << 40) + 5)
    F.set_backend("torch")
    try:
        F.adamw8_step_multi(there, **HYPER, step=step, seed=(step << 40) + 5)
    finally:
        F.set_backend("auto")
    for a, b in zip(here, there):
        for k in (2, 3, 4, 5):
            assert torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8))
    again = _items(sizes, pdt, gdt, "cuda", 5)
    F.adamw8_step_multi(again, **HYPER, step=step, seed=(step << 40) + 5)
    for a, b in zip(here, again):  # equal calls, equal bits
        for x, y in zip(a, b):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.gpu
def test_views_that_are_not_aligned():
    base = _items([4099], torch.bfloat16, torch.bfloat16, "cuda", 9)[0]
    want = [t.clone() for t in base]
    F.adamw8_step_multi([tuple(want)], **HYPER, step=2, seed=1)
    p, g, m, ms, r, rs = base
    room = [torch.zeros(4099 + 8, dtype=t.dtype, device="cuda") for t in (p, g)] + [
        torch.zeros(4099 + 8, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    shifted = []
    for t, space, off in zip((p, g, m, r), room, (1, 3, 5, 7)):
        v = space[off:off + 4099]
        v.view(torch.uint8).copy_(t.view(torch.uint8)) if t.dtype == torch.float8_e4m3fn else v.copy_(t)
        shifted.append(v)
    item = (shifted[0], shifted[1], shifted[2], ms, shifted[3], rs)
    F.adamw8_step_multi([item], **HYPER, step=2, seed=1)
    assert torch.equal(item[0], want[0]) and torch.equal(item[3], want[3]) and torch.equal(item[5], want[5])
    for a, b in ((item[2], want[2]), (item[4], want[4])):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert (room[0][:1] == 0).all() and (room[0][4100:] == 0).all()  # the neighbours are not touched


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("size", [1e15, 1e7, 3e4, 1e-9, 1e-17])
def test_scales_of_every_size(device, size):
    """Gradients from far above to far below one: scales on both sides of 2^6, where storing takes another path."""
    g = torch.Generator().manual_seed(4)
    p = torch.randn(1500, generator=g)
    item = tuple(t.to(device) for t in (p, torch.randn(1500, generator=g) * size, *F.adamw8_state(p)))
    for step in (1, 2):
        _, wm, wr, _ = _oracle(item, step)
        F.adamw8_step_multi([item], **HYPER, step=step, seed=step)
        _check_codes(item[2], item[3], wm, False)
        _check_codes(item[4], item[5], wr, True)


@pytest.mark.parametrize("device", DEVICES)
def test_skip_flag_and_values_that_are_not_finite(device):
    items = _items([600], torch.float32, torch.float32, device, 2)
    snap = [t.clone() for t in items[0]]
    F.adamw8_step_multi(items, **HYPER, step=1, seed=1, ctrl=torch.tensor([1.0, 1.0, 0.0, 1.0], device=device))
    for x, y in zip(items[0], snap):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    items[0][1][5], items[0][1][300] = float("nan"), float("inf")
    F.adamw8_step_multi(items, **HYPER, step=1, seed=1)
    p, _, m, ms, r, rs = (t.cpu() for t in items[0])
    mv, rv = F.adamw8_decode(m, ms), F.adamw8_decode(r, rs)
    bad = torch.zeros(600, dtype=torch.bool)
    bad[5] = bad[300] = True
    assert torch.equal(torch.isnan(mv), bad) and torch.equal(torch.isnan(rv), bad)
    assert torch.isnan(p[5]) and torch.isnan(p[300]) and torch.isfinite(p[~bad]).all()
    assert torch.isfinite(ms).all() and torch.isfinite(rs).all()


@pytest.mark.parametrize("device", DEVICES)
def test_rounding_is_unbiased_and_stays_on_the_grid(device):
    n = 256 * 400
    x = torch.full((n,), 1.0 + 1 / 32, device=device)  # a quarter of the way from 1.0 to 1.125 in every block
    x[::256] = 448.0
    low, high = F._adamw8_draws(400, 0, 99, torch.device(device))
    code, scale = F._adamw8_round(x.view(400, 256), low, False)
    got = F.adamw8_decode(code.view(-1).view(torch.float8_e4m3fn), scale)
    keep = torch.ones(n, dtype=torch.bool, device=device)
    keep[::256] = False
    share = ((got[keep] - 1.0) / 0.125).mean().item()
    k = int(keep.sum())
    assert abs(share - 0.25) < 5 * math.sqrt(0.25 * 0.75 / k)  # five standard deviations of the mean of k draws
    # what is on the grid stays on it, whatever the draw
    again, s2 = F._adamw8_round(got.view(400, 256), high, False)
    assert torch.equal(again, code) and torch.equal(s2, scale)
    nearest, s3 = F.adamw8_encode(x)
    assert (F.adamw8_decode(nearest, s3)[keep] == 1.0).all()
    tiny = torch.full((256,), 1e-30, device=device)
    tiny[0] = 1.0
    assert (F.adamw8_decode(*F.adamw8_encode(tiny, root=True)) > 0).all()


def test_refusals():
    ok = _items([300], torch.float32, torch.float32, "cpu", 1)[0]
    p, g, m, ms, r, rs = ok
    step = lambda *item, **kw: F.adamw8_step_multi([item], **{**HYPER, "step": 1, "seed": 0, **kw})  # noqa: E731
    for bad, text in [((p.long(), g, m, ms, r, rs), "share one type"), ((p.half(), g.bfloat16(), m, ms, r, rs), "share one type"),
                      ((p, g, m.float(), ms, r, rs), "float8"), ((p, g, m, ms.half(), r, rs), "fp32"),
                      ((p, g[:-1], m, ms, r, rs), "differ in size"), ((p, g, m, ms[:1], r, rs), "one scale per block"),
                      ((p, g[::2], m, ms, r, rs), "contiguous"), ((p, g, m, ms, r), "items are"),
                      ((p, g.to("meta"), m, ms, r, rs), "different devices")]:
        with pytest.raises(ValueError, match=text):
            step(*bad)
    with pytest.raises(ValueError, match="twice"):
        F.adamw8_step_multi([ok, ok], **HYPER, step=1, seed=0)
    empty = _items([0, 0, 5], torch.float32, torch.float32, "cpu", 1)
    F.adamw8_step_multi(empty, **HYPER, step=1, seed=0)  # tensors without elements share an address
    with pytest.raises(ValueError, match="first step"):
        step(*ok, step=0)
    with pytest.raises(ValueError, match="seed"):
        step(*ok, seed=-1)
    with pytest.raises(ValueError, match="control block"):
        step(*ok, ctrl=torch.zeros(4, dtype=torch.float64))
    F.adamw8_step_multi([], **HYPER, step=1, seed=0)


@pytest.mark.gpu
@pytest.mark.parametrize("pdt,gdt", PAIRS)
def test_long_lists_turn_the_ring(pdt, gdt):
    """Lists whose warps take more blocks one after the other than the ring of copies has stages (46,000 blocks: six a warp
    and more), with odd tails: scales and codes equal the restatement's bit by bit."""
    sizes = [11_900_123, 7, 70_001]
    g = torch.Generator(device="cuda").manual_seed(6)
    here = []
    for n in sizes:
        blocks = -(-n // 256)
        p = torch.randn(n, generator=g, device="cuda").to(pdt)
        grad = (torch.randn(n, generator=g, device="cuda") * 10 ** (4 * torch.rand(n, generator=g, device="cuda") - 5)).to(gdt)
        m = (torch.randn(n, generator=g, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        r = (torch.randn(n, generator=g, device="cuda").abs() * 100).clamp(2.0 ** -9, 448).to(torch.float8_e4m3fn)
        scales = [torch.exp2(torch.randint(-20, -10, (blocks,), generator=g, device="cuda").float()) for _ in range(2)]
        here.append((p, grad, m, scales[0], r, scales[1]))
    there = [tuple(t.clone() for t in item) for item in here]
    F.adamw8_step_multi(here, **HYPER, step=3, seed=77)
    F.set_backend("torch")
    try:
        F.adamw8_step_multi(there, **HYPER, step=3, seed=77)
    finally:
        F.set_backend("auto")
    _same_update(here, there, pdt)


def _same_update(here, there, pdt):
    """The parameters differ by the kernel's quotient (2^-22 of the step) and by five roundings of 2^-24 of the old value, the
    step and the new value; the step is at most the new value and the old one, which is below 6: 2^-20 of both together, and
    a whole step of p's type where the two lie on either side of a border."""
    for a, b in zip(here, there):
        for k in (2, 3, 4, 5):
            assert torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8))
        p, q = a[0].double(), b[0].double()
        assert ((p == q) | ((p - q).abs() <= (q.abs() + 8.0) * 2.0 ** -20 + torch.finfo(pdt).eps * q.abs())).all()


@pytest.mark.gpu
def test_element_numbers_beyond_32_bits(monkeypatch):
    """The draws of a list that passes 2^32 elements inside a tensor, in the middle of a warp's run of blocks: windows around the
    border, at the start and at the end equal the restatement, which is given the windows' first element numbers."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 26 GB")
    lead, n = 5 * 256, (1 << 32) + 300_000
    zeros = lambda k, dt: torch.zeros(k, dtype=torch.uint8, device="cuda").view(dt)  # noqa: E731
    p, g, m, r = zeros(2 * n, torch.bfloat16), zeros(2 * n, torch.bfloat16), zeros(n, torch.float8_e4m3fn), zeros(n, torch.float8_e4m3fn)
    ms, rs = torch.ones(-(-n // 256), device="cuda"), torch.ones(-(-n // 256), device="cuda")
    border = ((1 << 32) - lead) // 256  # block of the tensor at which the element number passes 2^32
    windows = [(0, 40), (border - 700, border + 700), (len(ms) - 300, len(ms))]
    gen = torch.Generator(device="cuda").manual_seed(2)
    for b0, b1 in windows:
        a, b = b0 * 256, min(b1 * 256, n)
        p[a:b] = torch.randn(b - a, generator=gen, device="cuda").bfloat16()
        g[a:b] = (torch.randn(b - a, generator=gen, device="cuda") * 1e-3).bfloat16()
        m[a:b] = (torch.randn(b - a, generator=gen, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        r[a:b] = (torch.randn(b - a, generator=gen, device="cuda").abs() * 100).clamp(2.0 ** -9, 448).to(torch.float8_e4m3fn)
        ms[b0:b1], rs[b0:b1] = 2.0 ** -14, 2.0 ** -15
    cut = lambda b0, b1: tuple(t[b0 * 256:min(b1 * 256, n)] for t in (p, g, m)) + (ms[b0:b1], r[b0 * 256:min(b1 * 256, n)], rs[b0:b1])  # noqa: E731
    wants = [tuple(t.clone() for t in cut(b0, b1)) for b0, b1 in windows]
    first = torch.zeros(lead, dtype=torch.bfloat16, device="cuda")
    F.adamw8_step_multi([(first, torch.zeros_like(first), *F.adamw8_state(first)), (p, g, m, ms, r, rs)], **HYPER, step=2, seed=(9 << 33) + 1)
    draws = F._adamw8_draws
    F.set_backend("torch")
    try:
        for (b0, b1), want in zip(windows, wants):
            monkeypatch.setattr(F, "_adamw8_draws", lambda blocks, at, seed, device: draws(blocks, at + 5 + b0, seed, device))
            F.adamw8_step_multi([want], **HYPER, step=2, seed=(9 << 33) + 1)
    finally:
        F.set_backend("auto")
    _same_update([cut(b0, b1) for b0, b1 in windows], wants, torch.bfloat16)
