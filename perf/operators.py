"""Timed cases of three training operators: the token-embedding gradient by sorted tokens, the softmax cross entropy of a
linear projection in pieces of the vocabulary (the logits are never kept), and the AdamW step over many tensors with
moments held in 8 bits.

``run`` computes each operator either in plain 32-bit tensor operations (``own`` false) or through the framework's entry
points (``own`` true); ``exact`` restates the definition in 64 bits.
"""
import torch

own = False

PAD = 1  # the dictionary's padding index: the ignored target and the token without a gradient
VOCAB = 50272  # dictionary size of the training configurations (padded to a multiple of 8)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
BLOCK = 256  # values that share one scale in the 8-bit moments


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # Embedding gradient of a full training batch (8 sequences of 2048 tokens, model width 2048) into a new table.
        dict(name="embed_grad_batch", op="embed_grad", rows=16384, vocab=VOCAB, dim=2048, dtype="bf16", accumulate=False, pad=0.0),
        # Tied embeddings: the output projection's gradient is in the 16-bit buffer already, the lookup's is added to it.
        dict(name="embed_grad_tied", op="embed_grad", rows=8192, vocab=VOCAB, dim=768, dtype="fp16", accumulate=True, pad=0.0),
        # One short sequence added to a large table: latency.
        dict(name="embed_grad_short", op="embed_grad", rows=131, vocab=VOCAB, dim=768, dtype="bf16", accumulate=True, pad=0.0),
        # A padded fine-tuning batch, 32-bit table, odd vocabulary and row count.
        dict(name="embed_grad_padded_fp32", op="embed_grad", rows=6007, vocab=10007, dim=1000, dtype="fp32", accumulate=False, pad=0.4),
        # Loss and both gradients of a full training batch, the widest product here.
        dict(name="linear_ce_batch", op="linear_ce", rows=16384, vocab=VOCAB, dim=2048, dtype="fp16", ignored=0.0, train=True),
        # Fine-tuning: the targets of the prompts are ignored (well over a third of the rows), smaller model.
        dict(name="linear_ce_prompts", op="linear_ce", rows=4096, vocab=VOCAB, dim=768, dtype="bf16", ignored=0.4, train=True),
        # A small model on a few tokens, odd vocabulary and row count: latency.
        dict(name="linear_ce_few", op="linear_ce", rows=37, vocab=1021, dim=64, dtype="bf16", ignored=0.1, train=True),
        # Validation: the loss of every token, no gradient.
        dict(name="linear_ce_scoring", op="linear_ce", rows=4099, vocab=50257, dim=1024, dtype="bf16", ignored=0.02, train=False),
        # Flat shards of eight decoder layers of width 2048 (12 d^2 + 13 d parameters each), 16-bit parameters.
        dict(name="adamw8_shards", op="adamw8", count=8, size=50358272, odd=False, dtype="bf16", grad="bf16"),
        # The unflattened parameter list of a 12-layer model: matrices next to biases.
        dict(name="adamw8_list", op="adamw8", count=144, size=590592, odd=True, dtype="fp16", grad="fp16"),
        # Norms and biases only: latency.
        dict(name="adamw8_biases", op="adamw8", count=12, size=769, odd=True, dtype="bf16", grad="bf16"),
        # 32-bit master parameters with 16-bit gradients, odd sizes.
        dict(name="adamw8_master", op="adamw8", count=9, size=2100001, odd=True, dtype="fp32", grad="bf16"),
    ]


def _log_int(rng, lo, hi):
    """A whole number whose logarithm is spread evenly."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["embed_grad", "linear_ce", "adamw8"])
    if op == "embed_grad":
        return dict(op=op, rows=_log_int(rng, 1, 16384), vocab=_log_int(rng, 64, VOCAB), dim=8 * _log_int(rng, 8, 256),
                    dtype=rng.choice(["fp16", "bf16", "fp32"]), accumulate=rng.random() < 0.5, pad=round(rng.choice([0.0, 0.5]) * rng.random(), 3))
    if op == "linear_ce":
        return dict(op=op, rows=_log_int(rng, 1, 16384), vocab=_log_int(rng, 64, VOCAB), dim=8 * _log_int(rng, 8, 256),
                    dtype=rng.choice(["fp16", "bf16"]), ignored=round(rng.choice([0.0, 0.6]) * rng.random(), 3), train=rng.random() < 0.75)
    count = _log_int(rng, 1, 200)
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    return dict(op=op, count=count, size=_log_int(rng, 1, 100_000_000 // count), odd=rng.random() < 0.5, dtype=dtype,
                grad=rng.choice(["bf16", "fp32"]) if dtype == "fp32" else dtype)


def _sizes(case):
    """Element counts of the AdamW case's tensors: matrices, and with ``odd`` every third a vector and none even."""
    if not case["odd"]:
        return [case["size"]] * case["count"]
    return [max(1, (case["size"] >> (i % 3 * 4)) // 2 * 2 - 1) for i in range(case["count"])]


def _offsets(case):
    """First block of every tensor in the padded flat layout, and the number of blocks."""
    first, at = [], 0
    for n in _sizes(case):
        first.append(at)
        at += (n + BLOCK - 1) // BLOCK
    return first, at


# -------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _tokens(g, n, vocab):
    """Frequent tokens have small numbers and the frequency falls with the rank, as in a BPE dictionary."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return (torch.exp(u * torch.log(torch.tensor(float(vocab), dtype=torch.float64, device="cuda"))).long() - 1).clamp_(0, vocab - 1)


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "embed_grad":
        n, v, d, dt = case["rows"], case["vocab"], case["dim"], DTYPES[case["dtype"]]
        tokens = _tokens(g, n, v)
        tokens[torch.rand(n, generator=g, device="cuda") < case["pad"]] = PAD
        s = {"op": "embed_grad", "tokens": tokens, "dy": torch.randn(n, d, generator=g, device="cuda").to(dt), "vocab": v, "scale": d ** 0.5, "grad": None}
        if case["accumulate"]:
            s["grad"] = torch.randn(v, d, generator=g, device="cuda").to(dt)
        return s
    if case["op"] == "linear_ce":
        n, v, d, dt = case["rows"], case["vocab"], case["dim"], DTYPES[case["dtype"]]
        x = torch.randn(n, d, generator=g, device="cuda").to(dt)  # the final layer norm's output
        w = (torch.randn(v, d, generator=g, device="cuda") * (2.0 / d ** 0.5)).to(dt)
        target = _tokens(g, n, v)
        target[torch.rand(n, generator=g, device="cuda") < case["ignored"]] = PAD
        return {"op": "linear_ce", "x": x.requires_grad_(case["train"]), "w": w.requires_grad_(case["train"]), "target": target, "train": case["train"],
                "upstream": torch.tensor(0.5, device="cuda")}
    dt, gt = DTYPES[case["dtype"]], DTYPES[case["grad"]]
    first, blocks = _offsets(case)
    sizes = _sizes(case)
    n = blocks * BLOCK
    live = torch.zeros(blocks, BLOCK, device="cuda", dtype=torch.bool)
    for f, k in zip(first, sizes):
        live.view(-1)[f * BLOCK:f * BLOCK + k] = True
    size = torch.exp(torch.randn(blocks, 1, generator=g, device="cuda") - 7.0)  # gradients differ in size from block to block
    mask = live.float()
    grad = (torch.randn(blocks, BLOCK, generator=g, device="cuda") * size * mask).to(gt).view(n)
    p = (torch.randn(blocks, BLOCK, generator=g, device="cuda") * 0.02 * mask).to(dt).view(n)
    # moments of a run under way: codes over the whole range, scales next to the gradients'
    m8 = (torch.randn(blocks, BLOCK, generator=g, device="cuda") * 100.0 * mask).clamp_(-448, 448).to(torch.float8_e4m3fn).view(n)
    r8 = (torch.randn(blocks, BLOCK, generator=g, device="cuda").abs() * 120.0 * mask).clamp_(0, 448).to(torch.float8_e4m3fn).view(n)
    scale = torch.exp2(torch.floor(torch.log2(size.view(-1))) - 7.0)
    s = {"op": "adamw8", "p": p, "g": grad, "m8": m8, "ms": scale.clone(), "r8": r8, "rs": scale.clone(), "seed": int(seed) * 7919 + 100, "step": 100,
         "ctrl": torch.tensor([0.25, 0.0, 1.0, 1.0], device="cuda")}
    s["items"] = []
    for f, k in zip(first, sizes):
        a, b, nb = f * BLOCK, f * BLOCK + k, (k + BLOCK - 1) // BLOCK
        s["items"].append((p[a:b], grad[a:b], m8[a:b], s["ms"][f:f + nb], r8[a:b], s["rs"][f:f + nb]))
    return s


HYPER = dict(lr=2e-4, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)


# ----------------------------------------------------------------------------------------------------------- plain forms
def _embed_grad_plain(s):
    keep = s["tokens"] != PAD
    table = torch.zeros(s["vocab"], s["dy"].shape[1], device="cuda")
    table.index_add_(0, s["tokens"], s["dy"].float() * (s["scale"] * keep)[:, None])
    if s["grad"] is None:
        return {"grad": table.to(s["dy"].dtype)}
    s["grad"].copy_(s["grad"].float() + table)
    return {"grad": s["grad"]}


def _linear_ce_plain(s):
    x, w, t = s["x"].detach().float(), s["w"].detach().float(), s["target"]
    keep = t != PAD
    logits = x @ w.t()
    top = logits.amax(dim=1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(dim=1, keepdim=True)
    loss = (top + torch.log(total) - logits.gather(1, t[:, None])).squeeze(1) * keep
    if not s["train"]:
        return {"loss": loss}
    del logits
    prob = e.div_(total)
    prob.scatter_add_(1, t[:, None], torch.full_like(total, -1.0))
    prob *= (keep * s["upstream"])[:, None]
    return {"loss": loss.sum(), "dx": (prob @ w).to(s["x"].dtype), "dw": (prob.t() @ x).to(s["w"].dtype)}


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random16(seed, n):
    """Two 16-bit random numbers for every element number: a hash of the number and the seed (an input)."""
    i = torch.arange(n, device="cuda", dtype=torch.int64)
    bits = _mix((i & 0xFFFFFFFF) ^ (seed & 0xFFFFFFFF) ^ _mix((i >> 32) ^ ((seed >> 32) & 0xFFFFFFFF)))
    return (bits & 0xFFFF).int(), (bits >> 16).int()


def _pow2_scale(top):
    """Per block the smallest power of two that brings the largest magnitude to at most 448, the top of e4m3."""
    k = ((top.view(torch.int32) + 0x1FFFFF) >> 23) - (127 + 8)
    return ((k.clamp(-110, 110) + 127) << 23).view(torch.float32)


def _to_8bit(mag, rnd, at_least_one):
    """e4m3 codes of magnitudes in [0, 448], rounded up with the probability of the remainder (16 random bits)."""
    normal = ((mag.view(torch.int32) + (rnd << 4)) >> 20) - (120 << 3)
    small = torch.floor(mag * 512.0 + rnd.float() * (1.0 / 65536.0)).int()
    code = torch.where(mag < 0.015625, small, normal).clamp(max=0x7E)
    return torch.where((code == 0) & (mag > 0), torch.ones_like(code), code) if at_least_one else code


def _adamw8_plain(s):
    h, n = HYPER, s["p"].numel()
    bc1, bc2 = 1.0 - h["beta1"] ** s["step"], 1.0 - h["beta2"] ** s["step"]
    step_size = h["lr"] * bc2 ** 0.5 / bc1
    g = s["g"].float().view(-1, BLOCK) * s["ctrl"][0]
    m = s["m8"].float().view(-1, BLOCK) * s["ms"][:, None]
    r = s["r8"].float().view(-1, BLOCK) * s["rs"][:, None]
    m = m * h["beta1"] + g * (1.0 - h["beta1"])
    v = (r * r) * h["beta2"] + (g * g) * (1.0 - h["beta2"])
    r = torch.sqrt(v)
    p = s["p"].float().view(-1, BLOCK)
    p = p - p * (h["lr"] * h["weight_decay"])
    p = p - (m / (r + h["eps"])) * step_size
    s["p"].copy_(p.view(-1))
    low, high = (x.view(-1, BLOCK) for x in _random16(s["seed"], n))
    ms, rs = _pow2_scale(m.abs().amax(1)), _pow2_scale(r.amax(1))
    code = _to_8bit(m.abs() / ms[:, None], low, False) | ((m < 0).int() << 7)
    s["m8"].view(torch.uint8).copy_(code.to(torch.uint8).view(-1))
    s["r8"].view(torch.uint8).copy_(_to_8bit(r / rs[:, None], high, True).to(torch.uint8).view(-1))
    s["ms"].copy_(ms)
    s["rs"].copy_(rs)
    return {k: s[k] for k in ("p", "m8", "ms", "r8", "rs")}


# ------------------------------------------------------------------------------------------------------------------- run
def run(state):
    if not own:
        return {"embed_grad": _embed_grad_plain, "linear_ce": _linear_ce_plain, "adamw8": _adamw8_plain}[state["op"]](state)
    from metaseq_b200.ops import autograd, functional

    s = state
    if s["op"] == "embed_grad":
        return {"grad": functional.embed_grad_sorted(s["tokens"], s["dy"], s["vocab"], scale=s["scale"], pad_idx=PAD, out=s["grad"],
                                                     accumulate=s["grad"] is not None)}
    if s["op"] == "linear_ce":
        if not s["train"]:
            return {"loss": functional.linear_cross_entropy(s["x"], s["w"], s["target"], PAD)}
        loss = autograd.linear_cross_entropy_sum(s["x"], s["w"], s["target"], PAD)
        dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]), grad_outputs=s["upstream"])
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    functional.adamw8_step_multi(s["items"], **HYPER, step=s["step"], seed=s["seed"], ctrl=s["ctrl"])
    return {k: s[k] for k in ("p", "m8", "ms", "r8", "rs")}


def work(case):
    """The least that must be moved and computed: every input read once, every output written once."""
    if case["op"] == "embed_grad":
        b, n, v, d = SIZE[case["dtype"]], case["rows"], case["vocab"], case["dim"]
        kept = max(1, round(n * (1 - case["pad"])))
        table = 2.0 * _expected_distinct(kept, v) * d * b if case["accumulate"] else v * d * b  # added to, or written as a whole
        return {"bytes": 8 * n + kept * d * b + table, "flops": 2.0 * kept * d}
    if case["op"] == "linear_ce":
        b, v, d = SIZE[case["dtype"]], case["vocab"], case["dim"]
        n = max(1, round(case["rows"] * (1 - case["ignored"])))
        move = (n * d + v * d) * b + 12 * case["rows"]
        if not case["train"]:
            return {"bytes": move, "flops": 2.0 * n * v * d + 4.0 * n * v}
        return {"bytes": move + (case["rows"] * d + v * d) * b, "flops": 6.0 * n * v * d + 6.0 * n * v}
    total = sum(_sizes(case))
    _, blocks = _offsets(case)
    return {"bytes": total * (2 * SIZE[case["dtype"]] + SIZE[case["grad"]] + 4) + 16 * blocks, "flops": 40.0 * total}


def _expected_distinct(n, vocab):
    """Expected number of different tokens among ``n`` of the distribution in ``_tokens`` (probability log(1 + 1/k) / log V)."""
    k = torch.arange(1, vocab + 1, dtype=torch.float64)
    p = torch.log1p(1.0 / k) / torch.log(torch.tensor(float(vocab), dtype=torch.float64))
    return float((1.0 - torch.exp(n * torch.log1p(-p.clamp(max=1 - 1e-12)))).sum())


# ----------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed_grad":
        base = s["grad"].double() if s["grad"] is not None else torch.zeros(s["vocab"], s["dy"].shape[1], dtype=torch.float64, device="cuda")
        rows = (s["tokens"] != PAD).nonzero().squeeze(1)
        return {"grad": base.index_put((s["tokens"][rows],), s["dy"][rows].double() * s["scale"], accumulate=True)}
    if case["op"] == "linear_ce":
        x, w, t = s["x"].detach().double(), s["w"].detach().double(), s["target"]
        losses, dx, dw = torch.zeros(len(t), dtype=torch.float64, device="cuda"), torch.zeros_like(x), torch.zeros_like(w)
        for rows in (t != PAD).nonzero().squeeze(1).split(2048):  # in blocks of rows: [tokens, vocabulary] in 64 bits is large
            z = torch.einsum("nd,vd->nv", x[rows], w)
            lse = torch.logsumexp(z, dim=1)
            losses[rows] = lse - z[torch.arange(len(rows), device="cuda"), t[rows]]
            if case["train"]:
                q = torch.softmax(z, dim=1)
                q[torch.arange(len(rows), device="cuda"), t[rows]] -= 1.0
                q *= float(s["upstream"])
                dx[rows] = torch.einsum("nv,vd->nd", q, w)
                dw += torch.einsum("nv,nd->vd", q, x[rows])
        return {"loss": losses} if not case["train"] else {"loss": losses.sum(), "dx": dx, "dw": dw}
    h = HYPER
    value = torch.cat([torch.arange(8) * 2.0 ** -9, ((8 + torch.arange(8)) * 2.0 ** torch.arange(-9, 6)[:, None]).reshape(-1)]).double().cuda()
    code = lambda c: value[(c.view(torch.uint8).long() & 0x7F).clamp(max=126)] * torch.where(c.view(torch.uint8) > 127, -1.0, 1.0)  # noqa: E731
    g = s["g"].double() * float(s["ctrl"][0])
    m = h["beta1"] * code(s["m8"]) * s["ms"].double().repeat_interleave(BLOCK) + (1 - h["beta1"]) * g
    r = torch.sqrt(h["beta2"] * (code(s["r8"]) * s["rs"].double().repeat_interleave(BLOCK)) ** 2 + (1 - h["beta2"]) * g * g)
    step = h["lr"] * (1 - h["beta2"] ** s["step"]) ** 0.5 / (1 - h["beta1"] ** s["step"])
    p = s["p"].double() * (1 - h["lr"] * h["weight_decay"]) - step * m / (r + h["eps"])
    # The codes come from a draw between two neighbours and the scales from a comparison with a power of two: a value next
    # to a border may fall on its other side in 64 bits, so these outputs have no value of their own there.
    return {"p": p, "m8": None, "ms": None, "r8": None, "rs": None}
