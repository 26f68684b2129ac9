"""The three vocabulary-sized operators together, as a training step with tied embeddings uses them: lookup, loss without
logits, one gradient for the shared table, AdamW with 8-bit moments.  And the options that switch them on."""
import copy
import math

import pytest
import torch

from metaseq_b200 import options, tasks
from metaseq_b200.checkpoint import flat_shards
from metaseq_b200.cli.train import build_model_and_criterion
from metaseq_b200.dataclass.utils import convert_namespace_to_config
from metaseq_b200.ops import _lib
from metaseq_b200.ops import autograd as ag
from metaseq_b200.ops import functional as F
from metaseq_b200.optim.adam import Adam
from metaseq_b200.trainer import Trainer

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
PAD = 1


def _step_inputs(device, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(515, 72, generator=g) * 0.3).to(dtype)
    tokens = torch.randint(2, 515, (3, 41), generator=g)
    tokens[0, 30:] = PAD
    target = torch.roll(tokens, -1, 1)
    target[:, -1] = PAD
    target[1, :20] = PAD
    return w.to(device), tokens.to(device), target.to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("views", [False, True])
def test_gradient_of_a_tied_table(device, dtype, views):
    w, tokens, target = _step_inputs(device, dtype)
    ref = w.detach().cpu().double().requires_grad_()
    pad_free = torch.where(tokens.cpu() == PAD, torch.full_like(tokens.cpu(), 0), tokens.cpu())
    # the lookup of padding carries no gradient; its targets are ignored or roll in from kept tokens, so detach it
    x = ref[pad_free]
    x = torch.where((tokens.cpu() == PAD)[..., None], ref.detach()[tokens.cpu()], x)
    keep = target.cpu() != PAD
    z = torch.tanh(x * 1.5)[keep] @ ref.t()
    want_loss = (torch.logsumexp(z, 1) - z.gather(1, target.cpu()[keep][:, None]).squeeze(1)).sum()
    want_loss.backward()
    param = torch.nn.Parameter(w)
    if views:
        param._grad_view, param._grad_filled = torch.full_like(w, float("nan")), False
    x = torch.tanh(ag.embedding(tokens, None, param, None, 1.5, PAD))
    loss = ag.linear_cross_entropy_sum(x, param, target, PAD)
    loss.backward()
    got = param._grad_view if views else param.grad
    assert not views or param.grad is None
    # roundings to 16 bits on the way: the lookup, tanh, P, dx, the gradient through tanh, dy, and two of the sum: eight
    # half steps of the sum of the magnitudes that make an element up
    eps = torch.finfo(dtype).eps / 2
    loss, want_loss = loss.detach(), want_loss.detach()
    assert abs(float(loss) - float(want_loss)) <= 8 * eps * float(want_loss)
    norm = (got.cpu().double() - ref.grad).norm() / ref.grad.norm()
    assert norm <= 8 * eps, float(norm)
    if device == "cuda":
        assert _lib.check_status("cuda") == 0


@pytest.mark.gpu
def test_whole_step_in_a_graph_equals_the_eager_step():
    """Lookup, loss, gradient and update captured together and replayed on new tokens."""
    w, tokens, target = _step_inputs("cuda", torch.bfloat16)
    up = torch.ones((), device="cuda")

    def step(table, grad, state, tok, tgt):
        x = F.embed_fwd(tok, None, table, None, 1.0)
        _, total, saved = F.linear_cross_entropy_fwd(x, table, tgt, PAD)
        dx, _ = F.linear_cross_entropy_bwd(saved, table, tgt, up, PAD, dw_out=grad)
        F.embed_grad_sorted(tok, dx, table.shape[0], 1.0, PAD, out=grad, accumulate=True)
        F.adamw8_step_multi([(table, grad, *state)], lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=1, seed=5)
        return total

    def fresh():
        return w.clone(), torch.empty_like(w), F.adamw8_state(w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*fresh(), tokens, target)
    torch.cuda.current_stream().wait_stream(side)
    captured = fresh()
    tok, tgt = tokens.clone(), target.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total = step(*captured, tok, tgt)
    for t, v in zip((captured[0], *captured[2]), (w, *F.adamw8_state(w))):
        t.view(torch.uint8).copy_(v.view(torch.uint8))
    _, t2, g2 = _step_inputs("cuda", torch.bfloat16, seed=7)
    tok.copy_(t2), tgt.copy_(g2)
    graph.replay()
    eager = fresh()
    want = step(*eager, t2, g2)
    assert torch.equal(total, want)
    for a, b in zip((captured[0], captured[1], *captured[2]), (eager[0], eager[1], *eager[2])):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert _lib.check_status("cuda") == 0


# ------------------------------------------------------------------------------------------------------- optimizer
def _params(device, dtype=torch.float32):
    g = torch.Generator().manual_seed(1)
    return [torch.nn.Parameter(torch.randn(*s, generator=g).to(dtype).to(device)) for s in ((40, 33), (300,), (1,))]


def _train(params, opt, steps, start=0):
    for k in range(start, start + steps):
        for i, p in enumerate(params):
            g = torch.Generator().manual_seed(1000 * k + i)
            p.grad = (torch.randn(p.shape, generator=g) * 0.1 + 0.05).to(p.dtype).to(p.device)
        opt.step()


@pytest.mark.parametrize("device", DEVICES)
def test_optimizer_follows_the_fp32_moments(device):
    """Every stored moment lies within one code of itself: a step of 2^-3 of the value at most, so after k steps the two
    directions m / r differ by no more than the codes' spread; with the same gradients and signs the parameters keep within
    a third of the distance they have moved."""
    a, b = _params(device), _params(device)
    start = [p.detach().clone() for p in a]
    kw = dict(lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)
    _train(a, Adam(a, **kw), 20)
    _train(b, opt := Adam(b, use_fp8_stats=True, **kw), 20)
    for p, q, s in zip(a, b, start):
        assert (p - q).norm() <= (p - s).norm() / 3
        st = opt.state[q]
        assert set(st) == {"step", *Adam.EIGHT_BIT} and st["step"] == 20
        assert st["exp_avg_8"].dtype == torch.float8_e4m3fn and st["exp_avg_8"].numel() == q.numel()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_resumed_run_continues_exactly(device, dtype):
    kw = dict(lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1, use_fp8_stats=True)
    a = _params(device, dtype)
    opt = Adam(a, **kw)
    _train(a, opt, 3)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    other = Adam(b, **kw)
    other.load_state_dict(opt.state_dict())
    _train(a, opt, 3, 3)
    _train(b, other, 3, 3)
    for p, q in zip(a, b):
        assert torch.equal(p, q)


@pytest.mark.parametrize("form", ["fp32", "fp16", "fp8"])
@pytest.mark.parametrize("target", ["fp32", "fp8"])
def test_states_of_every_form_are_taken_over(form, target):
    """A run that changes how the moments are held continues from their values.  A stored value is off by half a code, 2^-4
    of itself, or by half the smallest code of its block, 2^-10 of a scale that is at most 2^-7 of the largest value.  So in
    the next step m is off by dm = 0.9 (|m|/16 + max|m| 2^-17), the root by dr at most likewise, and the step by no more
    than size * (dm + |m'| dr / r') / (r' - dr)."""
    forms = {"fp32": {}, "fp16": {"use_fp16_stats": True}, "fp8": {"use_fp8_stats": True}}
    if form == "fp16" and target == "fp32":
        pytest.skip("fp16 moments carry a scale that an fp32 run does not read")
    kw = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8)
    a = _params("cpu")
    opt = Adam(a, **kw, **forms[form])
    _train(a, opt, 4)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    other = Adam(b, **kw, **forms[target])
    other.load_state_dict(copy.deepcopy(opt.state_dict()))  # loaded fp32 tensors are not copied
    before = []
    for p in a:
        st = opt.state[p]
        if form == "fp8":
            m, v = F.adamw8_decode(st["exp_avg_8"], st["exp_avg_8_scale"]), F.adamw8_decode(st["exp_avg_sq_root_8"], st["exp_avg_sq_root_8_scale"]) ** 2
        else:
            m, v = (st[k].float() * st.get(k + "_scale", 1.0) for k in ("exp_avg", "exp_avg_sq"))
        before.append((m.view(p.shape).clone(), v.view(p.shape).clone()))
    _train(b, other, 1, 4)
    size = 1e-2 * math.sqrt(1 - 0.95 ** 5) / (1 - 0.9 ** 5)
    for p, q, (m, v) in zip(a, b, before):
        off = lambda x: x.abs() / 16 + x.abs().max() * 2.0 ** -17  # noqa: E731
        g = q.grad
        m1, r1 = 0.9 * m + 0.1 * g, (0.95 * v + 0.05 * g * g).sqrt()
        want = p - size * m1 / (r1 + 1e-8)
        dr = off(v.sqrt()).clamp(max=r1 * 0.9)
        bound = size * (0.9 * off(m) + m1.abs() * dr / r1) / (r1 - dr)
        assert ((q - want).abs() <= bound + 1e-6 * (p.abs() + 1)).all()


def test_refused_combinations():
    p = _params("cpu")
    with pytest.raises(ValueError, match="8 bits or in fp16"):
        Adam(p, use_fp8_stats=True, use_fp16_stats=True)
    with pytest.raises(ValueError, match="PyTorch-ops form"):
        Adam(p, use_fp8_stats=True, use_kernels=False)


def test_resharding_joins_eight_bit_moments():
    n = 1000
    g = torch.Generator().manual_seed(3)
    m, v = torch.randn(n, generator=g), torch.rand(n, generator=g)
    states = []
    for k in range(2):
        part = slice(500 * k, 500 * k + 500)
        a, b = F.adamw8_encode(m[part]), F.adamw8_encode(v[part].sqrt(), root=True)
        entry = dict(zip(Adam.EIGHT_BIT, a + b), step=7)
        states.append({"model": {"flat_param_0": torch.zeros(500)}, "last_optimizer_state": {"state": {0: entry}, "param_groups": []},
                       "shard_metadata": {"param_metadata": [{"fsdp_path": "", "params": {"flat_param_0": {
                           "names": ["w"], "shapes": [(n,)], "numels": [n], "padding": 0}}}]}})
    whole = flat_shards.reshard_optimizer_state(states, 0, 1)["state"][0]
    assert set(whole) == {"exp_avg", "exp_avg_sq", "step"} and whole["step"] == 7
    assert ((whole["exp_avg"] - m).abs() <= m.abs() / 16 + 1e-4).all()  # half a step of e4m3: 2^-4
    assert ((whole["exp_avg_sq"].sqrt() - v.sqrt()).abs() <= v.sqrt() / 16 + 1e-4).all()


# ----------------------------------------------------------------------------------------------------------- training
BASE = ["--task", "dummy_lm", "--dict-size", "124", "--tokens-per-sample", "16", "--batch-size", "2", "--arch",
        "transformer_lm_megatron", "--decoder-layers", "2", "--decoder-embed-dim", "32", "--decoder-ffn-embed-dim", "64",
        "--decoder-attention-heads", "2", "--decoder-learned-pos", "--share-decoder-input-output-embed", "--dropout", "0.0",
        "--attention-dropout", "0.0", "--optimizer", "adam", "--lr", "1e-2", "--clip-norm", "1.0", "--distributed-world-size",
        "1", "--disable-validation", "--log-format", "none", "--lr-scheduler", "polynomial_decay", "--total-num-update", "100",
        "--warmup-updates", "1"]


def _trainer(save_dir, extra):
    argv = BASE + ["--save-dir", str(save_dir), *extra]
    cfg = convert_namespace_to_config(options.parse_args_and_arch(options.get_training_parser(), input_args=argv))
    torch.manual_seed(1)
    task = tasks.setup_task(cfg.task)
    model, criterion = build_model_and_criterion(cfg, task)
    trainer = Trainer(cfg, task, model, criterion)
    task.load_dataset("train")
    return trainer, task.dataset("train").collater([0, 1])


def _losses(save_dir, extra, updates=4):
    trainer, batch = _trainer(save_dir, extra)
    logs = [trainer.train_step([batch]) for _ in range(updates)]
    valid = trainer.valid_step(batch)
    return [float(log["loss"]) for log in logs if log is not None], float(valid["loss"]), trainer


@pytest.mark.parametrize("criterion", ["cross_entropy", "vocab_parallel_cross_entropy"])
@pytest.mark.parametrize("extra", [[], ["--ddp-backend", "fully_sharded"], ["--memory-efficient-fp16", "--fp16-init-scale", "4"]])
def test_logits_free_training_equals_training_with_logits(tmp_path, criterion, extra):
    flags = ["--cpu", "--criterion", criterion, *extra]
    plain, plain_valid, _ = _losses(tmp_path / "a", flags)
    free, free_valid, _ = _losses(tmp_path / "b", flags + ["--logits-free"])
    half = bool(extra) and "fp16" in extra[0]
    # fp16: logits are rounded to 16 bits on one side only; a loss of about 7 moves by a few of their half steps (2^-9 at 4)
    tol = 2e-2 if half else 1e-4
    assert free == pytest.approx(plain, abs=tol) and free_valid == pytest.approx(plain_valid, abs=tol)


@pytest.mark.parametrize("extra", [["--cpu"], ["--cpu", "--memory-efficient-fp16", "--fp16-init-scale", "4"],
                                   pytest.param(["--memory-efficient-fp16", "--fp16-init-scale", "4"], marks=pytest.mark.gpu),
                                   pytest.param(["--memory-efficient-fp16", "--fp16-init-scale", "4", "--ddp-backend",
                                                 "fully_sharded"], marks=pytest.mark.gpu)])
def test_training_with_all_three(tmp_path, extra):
    losses, valid, trainer = _losses(tmp_path, extra + ["--criterion", "vocab_parallel_cross_entropy", "--logits-free",
                                                        "--fp8-adam-stats"], updates=6)
    assert len(losses) >= 4 and all(map(math.isfinite, losses)) and math.isfinite(valid)
    states = trainer.optimizer.optimizer.state.values()
    assert states and all("exp_avg_8" in s for s in states)


@pytest.mark.parametrize("extra", [["--cpu"], ["--cpu", "--memory-efficient-fp16", "--fp16-init-scale", "4"], ["--cpu", "--fp16",
                                   "--fp16-init-scale", "4"],
                                   pytest.param(["--memory-efficient-fp16", "--fp16-init-scale", "4"], marks=pytest.mark.gpu)])
def test_checkpointed_run_resumes_with_eight_bit_moments(tmp_path, extra):
    flags = extra + ["--criterion", "cross_entropy", "--logits-free", "--fp8-adam-stats"]
    trainer, batch = _trainer(tmp_path, flags)
    for _ in range(3):
        trainer.train_step([batch])
    path = str(tmp_path / "resume.pt")
    trainer.save_checkpoint(path, {"train_iterator": {"epoch": 1}})
    want = [float(trainer.train_step([batch])["loss"]) for _ in range(3)]
    other, batch = _trainer(tmp_path / "b", flags)
    other.load_checkpoint(path)
    states = list(other.optimizer.optimizer.state.values())
    assert states and all(s["exp_avg_8"].dtype == torch.float8_e4m3fn for s in states)
    got = [float(other.train_step([batch])["loss"]) for _ in range(3)]
    assert got == want


def test_logits_free_needs_the_whole_vocabulary(monkeypatch, tmp_path):
    from metaseq_b200.parallel import mpu

    monkeypatch.setattr(mpu, "get_tensor_model_parallel_world_size", lambda: 2)
    from metaseq_b200.criterions.vocab_parallel_cross_entropy import VocabParallelCrossEntropyCriterion

    with pytest.raises(ValueError, match="whole vocabulary"):
        VocabParallelCrossEntropyCriterion(type("T", (), {"target_dictionary": None})(), logits_free=True)


def _nodes_of(call):
    """Launches of a call: the nodes of the graph that it is captured into (the calls below launch nothing but kernels)."""
    import ctypes

    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    count = ctypes.c_size_t(0)
    get = ctypes.CDLL("libcudart.so.12").cudaGraphGetNodes
    assert get(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(count)) == 0
    return count.value


@pytest.mark.gpu
def test_launch_counter_counts_what_is_launched():
    w, tokens, target = _step_inputs("cuda", torch.bfloat16)
    big = torch.randn(20000, 72, device="cuda").bfloat16()
    few, many = torch.randint(0, 500, (100,), device="cuda"), torch.randint(0, 500, (600,), device="cuda")
    dy = torch.randn(600, 72, device="cuda").bfloat16()
    table = torch.zeros(500, 72, device="cuda").bfloat16()
    x = torch.randn(600, 72, device="cuda").bfloat16()
    t = torch.randint(0, 20000, (600,), device="cuda")
    small_t = t % 515
    one = torch.ones((), device="cuda")
    _, _, saved = F.linear_cross_entropy_fwd(x, big, t, PAD)
    _, _, small = F.linear_cross_entropy_fwd(x, w, small_t, PAD)
    items = [(torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda"), *F.adamw8_state(torch.zeros(300, device="cuda"))) for _ in range(300)]
    hyper = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, step=1, seed=1)
    calls = {
        "few tokens, new table": lambda: F.embed_grad_sorted(few, dy[:100], 500),
        "few tokens, added": lambda: F.embed_grad_sorted(few, dy[:100], 500, out=table, accumulate=True),
        "many tokens": lambda: F.embed_grad_sorted(many, dy, 500),
        "loss": lambda: F.linear_cross_entropy(x, big, t, PAD),
        "both gradients": lambda: F.linear_cross_entropy_bwd(saved, big, t, one, PAD),
        "dx": lambda: F.linear_cross_entropy_bwd(saved, big, t, one, PAD, need_dw=False),
        "dw": lambda: F.linear_cross_entropy_bwd(small, w, small_t, one, PAD, need_dx=False),
        "list of 300": lambda: F.adamw8_step_multi(items, **hyper),
        "list of 5": lambda: F.adamw8_step_multi(items[:5], **hyper),
    }
    for name, call in calls.items():
        call()
        before = _lib.launch_count()
        nodes = _nodes_of(call)
        assert _lib.launch_count() - before == nodes, name
    assert _lib.check_status("cuda") == 0
