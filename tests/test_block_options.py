"""The encoder with norms after its blocks, gated and scaled residuals, scaled / partial / interleaved rotary positions, and AdamW moments
in 8 bits: together, as a run uses them."""
import copy
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from nanoplm_b200.config.loaders import load_model_config, load_pretrain_config
from nanoplm_b200.config.schema import ModelConfig
from nanoplm_b200.data.tokenizer import ProtTokenizer
from nanoplm_b200.models.encoder import ProtEncoderMLM, RotaryPlan
from nanoplm_b200.ops import functional as ops
from nanoplm_b200.parallel.engine import AdamWHyper, ShardedEngine

GEOM = dict(hidden_size=64, intermediate_size=128, num_hidden_layers=3, num_attention_heads=2, max_position_embeddings=128)
YARN = {"type": "yarn", "factor": 2.0, "original_max_position": 64}
OPTIONS = [
    dict(sandwich_norm=True),
    dict(sandwich_norm=True, residual_gate="channel", residual_scale=True, norm_type="rmsnorm"),
    dict(sandwich_norm=True, residual_gate="token", residual_scale=True, rope_scaling=YARN, rotary_fraction=0.5,
         rope_interleaved=True),
    dict(rope_scaling=YARN),
    dict(rope_interleaved=True),
    dict(sandwich_norm=True, conv_kernel_size=3,
         moe={"num_experts": 4, "top_k": 2, "expert_intermediate_size": 32, "every_n_layers": 2}),
]


def _model(seed=0, geom=GEOM, **kw):
    torch.manual_seed(seed)
    m = ProtEncoderMLM(ModelConfig(**geom, **kw), ProtTokenizer())
    with torch.no_grad():
        for n, p in m.named_parameters():
            if n.endswith(("Wo.weight", "gate_proj.weight")) or "experts_Wo" in n:
                p.normal_(0, 0.05)
            elif n.endswith((".gate", ".scale", "norm_weight")):
                p.add_(0.1 * torch.randn_like(p))
    return m


def _batch(seed=0, lens=(25, 1, 64, 30)):
    g = torch.Generator().manual_seed(seed)
    n = sum(lens)
    ids = torch.randint(4, 24, (n,), generator=g)
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)
    labels = torch.full((n,), -100)
    labels[::3] = ids[::3]
    return ids, cu, labels


# ------------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("kw", OPTIONS)
def test_options_give_every_parameter_a_gradient(kw):
    m = _model(**kw)
    ids, cu, labels = _batch()
    out = m(input_ids=ids, cu_seqlens=cu, labels=labels)
    out["loss"].backward()
    missing = [n for n, p in m.named_parameters() if p.grad is None or not torch.isfinite(p.grad).all()]
    assert not missing, missing


def test_layer_by_layer_is_what_the_joined_layers_give():
    """A watched layer or norm runs its own calls; the results are those of the joined ones."""
    m = _model(**OPTIONS[2])
    ids, cu, labels = _batch()
    want = m(input_ids=ids, cu_seqlens=cu, labels=labels)["loss"]
    seen = []
    hooks = [m.model.layers[1].register_forward_hook(lambda *a: seen.append("layer")),
             m.model.layers[2].attn_norm.register_forward_hook(lambda *a: seen.append("attn_norm")),
             m.model.layers[0].mlp_norm.register_forward_hook(lambda *a: seen.append("mlp_norm"))]
    got = m(input_ids=ids, cu_seqlens=cu, labels=labels)["loss"]
    for h in hooks:
        h.remove()
    assert sorted(seen) == ["attn_norm", "layer", "mlp_norm"] and torch.allclose(got, want, atol=1e-6)


@pytest.mark.parametrize("gate", ["none", "channel", "token"])
def test_first_gradients_of_a_fresh_model_are_alike(gate):
    """A projection of zeros behind whose block a norm stands gets first gradients 1 / sqrt(eps) = 316 times as large as one whose outputs
    have a deviation of one. As the models start, no output projection's gradient is eight times another kind's largest."""
    torch.manual_seed(0)
    m = ProtEncoderMLM(ModelConfig(**dict(GEOM, hidden_size=128, num_hidden_layers=4), sandwich_norm=True, residual_gate=gate,
                                   moe={"num_experts": 4, "top_k": 2, "expert_intermediate_size": 64, "every_n_layers": 2}), ProtTokenizer())
    ids, cu, labels = _batch(lens=(100, 128, 90))
    m(input_ids=ids, cu_seqlens=cu, labels=labels)["loss"].backward()
    size = {n: float(p.grad.norm()) for n, p in m.named_parameters()}
    experts = [v for n, v in size.items() if n.endswith("experts_Wo")]
    dense = [v for n, v in size.items() if n.endswith("Wo.weight")]
    assert len(experts) == 2 and len(dense) == 6
    assert max(experts) <= 8 * max(dense) and max(dense) <= 8 * max(experts), (experts, dense)


def test_a_layer_follows_its_formula():
    m = _model(**OPTIONS[1])
    layer, rope = m.model.layers[1], m.model.rope("cpu")["sliding_attention"]
    ids, cu, _ = _batch()
    from nanoplm_b200.models.encoder import BatchContext, position_ids_from_cu_seqlens
    ctx = BatchContext(cu, position_ids_from_cu_seqlens(cu, len(ids)), len(ids))
    x = torch.randn(len(ids), 64)
    got, aux = layer(x, ctx, 64, rope)
    norm = lambda t, w: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-5) * w
    y = x
    for join, block, pre in ((layer.attn_join, lambda t: layer.attn(t, ctx, 64, rope), layer.attn_norm),
                             (layer.mlp_join, layer.mlp, layer.mlp_norm)):
        y = join.scale * y + join.gate * norm(block(norm(y, pre.weight)), join.norm_weight)
    assert aux is None and torch.allclose(got, y, rtol=1e-5, atol=1e-5)


def test_yarn_ends_its_ramp_where_the_configuration_says():
    whole = ops.rotary_frequencies(32, 160000.0, dict(YARN, truncate=True))[0]
    plan = _model(rope_scaling=dict(YARN, truncate=True), rope_interleaved=True).model.rope("cpu")["full_attention"]
    assert torch.equal(plan.frequencies, whole) and not torch.equal(whole, ops.rotary_frequencies(32, 160000.0, YARN)[0])


def test_plain_models_keep_their_tables_and_parameters():
    m = _model()
    rope = m.model.rope("cpu")["full_attention"]
    want = ops.rope_tables(128, 32, 160000.0, "cpu")
    assert all(torch.equal(a, b) for a, b in zip(rope, want))
    assert not any("join" in n for n in m.state_dict())
    scaled = _model(rope_scaling=YARN).model.rope("cpu")["full_attention"]
    w, factor = ops.rotary_frequencies(32, 160000.0, YARN)
    a = torch.arange(128).double()[:, None] * w
    assert torch.allclose(scaled[0].double(), factor * a.cos(), atol=1e-6) and torch.allclose(scaled[1].double(), factor * a.sin(), atol=1e-6)
    plan = _model(rotary_fraction=0.4).model.rope("cpu")["full_attention"]
    assert type(plan) is RotaryPlan and plan.frequencies.numel() == 6 and plan.factor == 1.0


@pytest.mark.parametrize("bad", [dict(residual_gate="other", sandwich_norm=True), dict(residual_gate="channel"), dict(residual_scale=True),
                                 dict(sandwich_norm=True, mhc_streams=2), dict(sandwich_norm=True, norm_bias=True),
                                 dict(rotary_fraction=0.0), dict(rotary_fraction=1.5), dict(rotary_fraction=0.01),
                                 dict(rope_scaling={"type": "other", "factor": 2}), dict(rope_scaling={"type": "linear"}),
                                 dict(rope_scaling={"type": "linear", "factor": 0.5}), dict(rope_scaling={"type": "yarn", "factor": 2}),
                                 dict(rope_scaling={"type": "ntk", "factor": 2, "base": 3}), dict(rope_scaling=dict(YARN, truncate="no")),
                                 dict(rope_scaling={"type": "linear", "factor": 2, "truncate": True})])
def test_configurations_that_are_refused(bad):
    with pytest.raises(ValueError):
        ModelConfig(**GEOM, **bad)


def test_options_load_from_yaml_sections():
    section = dict(hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=2, vocab_size=32,
                   mlp_activation="swiglu", mlp_dropout=0.0, mlp_bias=False, attention_bias=False, attention_dropout=0.0,
                   classifier_activation="gelu", max_position_embeddings=64, rope_scaling=YARN, rotary_fraction="0.5",
                   sandwich_norm="true", residual_gate="token")
    cfg = load_model_config(section)
    assert cfg.sandwich_norm is True and cfg.rotary_channels == 16 and cfg.rope_scaling == YARN
    assert load_pretrain_config({"dataset_dir": "x", "optimizer_state_bits": "8"}).optimizer_state_bits == 8
    assert load_pretrain_config({"dataset_dir": "x"}).optimizer_state_bits == 32


def _engine(model, device="cpu", bits=8, **kw):
    return ShardedEngine(model, AdamWHyper(lr=3e-3, weight_decay=0.05, beta2=0.98), torch.device(device), state_bits=bits, **kw)


def _steps(model, engine, n, first=0, device="cpu"):
    losses = []
    for i in range(first, first + n):
        ids, cu, labels = (t.to(device) for t in _batch(i))
        loss = model(input_ids=ids, cu_seqlens=cu, labels=labels)["loss"]
        loss.backward()
        engine.step(3e-3)
        losses.append(loss.item())
    return losses


def test_8bit_engine_resumes_as_it_would_have_gone_on():
    """Its checkpoint, in torch's fp32 layout, brings the same codes back, and the next steps are the same to the bit."""
    a = _model(**OPTIONS[2])
    ea = _engine(a)
    _steps(a, ea, 3)
    sd, model_sd = ea.optimizer_state_dict(), ea.full_state_dict_model()
    b = _model(seed=1, **OPTIONS[2])
    eb = _engine(b)
    eb.load_model_state_dict(model_sd)
    eb.load_optimizer_state_dict(sd)
    shard = _engine(c := _model(seed=2, **OPTIONS[2]))
    shard.load_shard_state(ea.shard_state())
    assert eb.step_count == shard.step_count == 3
    for e in (eb, shard):
        for x, y in zip(sum(ea.moments.values(), []), sum(e.moments.values(), [])):
            assert torch.equal(x, y)
    want = _steps(a, ea, 2, first=3)
    assert _steps(b, eb, 2, first=3) == want and _steps(c, shard, 2, first=3) == want
    assert torch.equal(ea.master, eb.master) and torch.equal(ea.master, shard.master)


def test_8bit_engine_stays_near_the_fp32_one():
    """First step: the update is lr g / |g| whatever the moments are kept in, and the weights are equal up to fp32."""
    a, b = _model(), _model()
    ea, eb = _engine(a), _engine(b, bits=32)
    la, lb = _steps(a, ea, 1), _steps(b, eb, 1)
    assert la == lb and torch.allclose(ea.master, eb.master, rtol=1e-5, atol=1e-6)
    assert ea.moments.nbytes() < 8 * ea.master.numel() / 2      # (small tensors are whole blocks)


def test_state_bits_are_checked():
    with pytest.raises(ValueError):
        _engine(_model(), bits=16)
    from nanoplm_b200.config.schema import PretrainingConfig
    from nanoplm_b200.runtime.pretrain import check_state_bits
    for bad in (dict(optimizer_state_bits=16), dict(optimizer_state_bits=8, optimizer="muon"),
                dict(optimizer_state_bits=8, expert_parallel_size=2), dict(optimizer_state_bits=8, shard_params=True)):
        with pytest.raises(ValueError):
            check_state_bits(PretrainingConfig(dataset_dir="x", **bad), distributed=True)
    assert check_state_bits(PretrainingConfig(dataset_dir="x"), True) == 32
    assert check_state_bits(PretrainingConfig(dataset_dir="x", optimizer_state_bits=8), True) == 8
    assert check_state_bits(PretrainingConfig(dataset_dir="x", optimizer_state_bits=8, shard_params=True), False) == 8


def _rank(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.set_num_threads(1)
    m = _model()
    e = _engine(m)
    sd0 = None
    for i in range(3):
        ids, cu, labels = _batch(10 * i + rank)
        m(input_ids=ids, cu_seqlens=cu, labels=labels)["loss"].backward()
        e.step(3e-3)
    sd0 = e.optimizer_state_dict()
    full = e.full_state_dict_model()
    # the gathered checkpoint in a single engine, and back into this one
    e.load_optimizer_state_dict(sd0)
    sd1 = e.optimizer_state_dict()
    same = all(torch.equal(sd0["state"][k]["exp_avg_sq"], sd1["state"][k]["exp_avg_sq"]) for k in sd0["state"])
    q.put((rank, same, float(sum(t.double().sum() for t in full.values())), [float(v["exp_avg"].double().sum()) for v in sd0["state"].values()]))
    dist.destroy_process_group()


def test_8bit_engine_on_two_ranks():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = sorted(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(timeout=60)
    assert all(same for _, same, _, _ in got) and got[0][2:] == got[1][2:]


def _spawned(target, *args, world=2):
    """What the ranks of a gloo group put into their queue as (rank, ...), by rank."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=target, args=(r, world, port, q, *args)) for r in range(world)]
    for p in procs:
        p.start()
    got = sorted((q.get(timeout=120) for _ in procs), key=lambda g: g[0])
    for p in procs:
        p.join(timeout=60)
    return got


def _warned_rank(rank, world, port, q):
    import logging
    from nanoplm_b200.utils.logging import logger
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.set_num_threads(1)
    said = []
    handler = logging.Handler(logging.WARNING)
    handler.emit = lambda record: said.append(record.getMessage())
    logger.addHandler(handler)
    counts = []
    for kw in (dict(bits=8, fused_comm=True), dict(bits=8), dict(bits=32, fused_comm=True)):
        said.clear()
        _engine(_model(), **kw)
        counts.append(sum("fused_comm" in m and "optimizer_state_bits" in m for m in said))
    q.put((rank, counts))
    dist.destroy_process_group()


def test_8bit_engine_says_that_fused_comm_is_off():
    """Once, by the first rank, where both were asked for and there are ranks to move anything between."""
    assert _spawned(_warned_rank) == [(0, [1, 0, 0]), (1, [0, 0, 0])]


def _snapshot(e):
    """{parameter: (master weights, first moments, second moments)} of all ranks, fp64 (collective)."""
    parts = [e._gather_full(t).double().cpu() for t in (e.master, *e._moments_flat())]
    return {s.name: tuple(t[s.offset:s.offset + s.numel] for t in parts) for s in e.slots}


def _gradients(e, step, ranks):
    """One flat gradient over all slots: layers and elements of different sizes, the sum of the ranks'."""
    total = 0
    for r in ranks:
        g = torch.Generator().manual_seed(1000 * step + r)
        flat = torch.zeros(e.total)
        for s in e.slots:
            size = torch.exp(2 * torch.randn(1, generator=g)) * torch.exp(torch.randn(s.numel, generator=g))
            flat[s.offset:s.offset + s.numel] = 0.05 * size * torch.randn(s.numel, generator=g)
        total = total + flat
    return total


def _follows_adamw(e, before, after, grad, t, lr, world):
    """One 8-bit step against the formula in 64 bits, from the moments that were kept before it. The gradient's scale (a norm of fp32 squares)
    and the moments are good to 2^-18 of their terms, the weights to a few roundings more. A moment is kept as one of the two codes
    around it, an eighth of its octave apart, or, below a block's smallest code, as that or as zero: 1.125 x 2^-15 of the octave of the block's
    largest in first moments, and 2^-31 in second ones, where the largest may have been rounded up into the next octave."""
    h = e.hyper
    g_all = grad.double() / world
    g_all = g_all * min(1.0, h.max_grad_norm / (float(g_all.norm()) + 1e-6))
    assert [s.name for s in e.slots] == list(before) and any(s.decay for s in e.slots) and not all(s.decay for s in e.slots)
    for s in e.slots:
        (p0, m0, v0), (p1, m1, v1), g = before[s.name], after[s.name], g_all[s.offset:s.offset + s.numel]
        m, v = h.beta1 * m0 + (1 - h.beta1) * g, h.beta2 * v0 + (1 - h.beta2) * g ** 2
        terms = h.beta1 * m0.abs() + (1 - h.beta1) * g.abs()
        denom = (v / (1 - h.beta2 ** t)).sqrt() + h.eps
        p = p0 * (1 - lr * h.weight_decay * s.decay) - lr / (1 - h.beta1 ** t) * m / denom
        assert ((p1 - p).abs() <= 2.0 ** -22 * p0.abs() + 2.0 ** -17 * lr / (1 - h.beta1 ** t) * terms / denom + 1e-30).all(), (s.name, t)
        assert ((m1 - m).abs() <= m.abs() / 8 + 2.0 ** -18 * terms + 2.0 ** -14 * m.abs().max()).all(), (s.name, t)
        assert ((v1 - v).abs() <= v * (1 / 8 + 2.0 ** -17) + 2.0 ** -30 * v.max()).all() and (v1[v > 0] > 0).all(), (s.name, t)


def _check_steps(e, steps, rank=0, world=1):
    lr = 3e-3
    before = _snapshot(e)
    for t in range(1, steps + 1):
        e.main_grad.copy_(_gradients(e, t, [rank]))
        e.step(lr)
        after = _snapshot(e)
        _follows_adamw(e, before, after, _gradients(e, t, range(world)), t, lr, world)
        before = after


def test_8bit_engine_follows_the_formula_step_by_step():
    _check_steps(_engine(_model()), 30)


def _checked_rank(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.set_num_threads(1)
    e = _engine(_model())
    crosses = [s.name for s in e.slots if s.offset < e.shard < s.offset + s.numel]
    error = ""
    try:
        _check_steps(e, 8, rank, world)
    except AssertionError as exc:
        error = str(exc) or "no"
    q.put((rank, len(crosses), error))
    dist.barrier()
    dist.destroy_process_group()


def test_8bit_engine_on_two_ranks_follows_the_formula():
    """With the ranks' gradients summed, and a tensor that lies on both of them."""
    assert _spawned(_checked_rank) == [(0, 1, ""), (1, 1, "")]


# ------------------------------------------------------------------------------------------- GPU
BIG = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, max_position_embeddings=256)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", OPTIONS)
def test_encoder_on_the_kernels_follows_the_cpu(kw, cuda_status):
    """Loss and gradients of a bf16 run on the kernels against the fp32 restatement, within what the suite allows bf16 encoders."""
    if "moe" in kw:
        kw = dict(kw, moe=dict(kw["moe"], expert_intermediate_size=128))
    cpu = _model(geom=BIG, **kw)
    with torch.no_grad():       # routing by near ties differs between the precisions
        for n, p in cpu.named_parameters():
            if "router" in n:
                p.mul_(8)
    gpu = copy.deepcopy(cpu)
    engine = ShardedEngine(gpu, AdamWHyper(lr=1e-3), torch.device("cuda:0"))
    ids, cu, labels = _batch(3, lens=(200, 1, 64, 129, 256))
    a = cpu(input_ids=ids, cu_seqlens=cu, labels=labels)["loss"]
    a.backward()
    b = gpu(input_ids=ids.cuda(), cu_seqlens=cu.cuda(), labels=labels.cuda())["loss"]
    b.backward()
    engine.collect_autograd_grads()
    assert abs(a.item() - b.item()) < 3e-2
    by_name = dict(cpu.named_parameters())
    for s in engine.slots:
        if "moe" in kw and ("mlp." in s.name or "router" in s.name):
            continue            # (tokens near a tie go to other experts)
        want = by_name[s.name].grad
        got = engine.main_grad[s.offset:s.offset + s.numel].view(s.shape).cpu()
        assert (got - want).norm() <= 0.08 * want.norm() + 1e-6, s.name


@pytest.mark.gpu
def test_training_with_all_options_on_the_gpu(cuda_status):
    """Rotary, sandwich norms and the 8-bit step together: finite losses, codes that a checkpoint brings back, and the same steps."""
    kw = OPTIONS[2]
    a = _model(geom=BIG, **kw)
    b = copy.deepcopy(a)
    ea, eb = _engine(a, "cuda:0"), _engine(b, "cuda:0")
    from nanoplm_b200.ops import kernels as K
    K.set_attention_deterministic(True)
    try:
        losses = _steps(a, ea, 4, device="cuda:0")
        assert all(x == x and abs(x) < 1e4 for x in losses)
        eb.load_model_state_dict(ea.full_state_dict_model())
        eb.load_optimizer_state_dict(ea.optimizer_state_dict())
        for x, y in zip(sum(ea.moments.values(), []), sum(eb.moments.values(), [])):
            assert torch.equal(x, y)
        _steps(a, ea, 1, first=4, device="cuda:0")
        _steps(b, eb, 1, first=4, device="cuda:0")
    finally:
        K.set_attention_deterministic(False)
    # (embedding and loss-head gradients are sums in any order, and a rounding near its threshold may go the other way)
    assert (ea.master - eb.master).norm() <= 1e-3 * (ea.master).norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_8bit_engine_follows_the_formula_on_the_gpu(dtype, cuda_status):
    e = _engine(_model(geom=BIG), "cuda:0", compute_dtype=dtype)
    _check_steps(e, 12)
    assert torch.equal(e.flat_params, e._gather_full(e.master).to(dtype))


@pytest.mark.gpu
def test_gradients_of_the_packed_rotation(cuda_status):
    T, H, D = 50, 4, 64
    w, factor = ops.rotary_frequencies(32, 1e4, YARN, "cuda")
    pos = torch.randint(0, 500, (T,), device="cuda", dtype=torch.int32)
    x = torch.randn(T, 3 * H * D, device="cuda", requires_grad=True)
    y = ops.rotary_qkv(x * 1.0, H, D, positions=pos, frequencies=w, factor=factor, interleaved=True)
    d = torch.randn_like(y)
    kept = d.clone()
    g, = torch.autograd.grad(y, x, d)
    assert torch.equal(d, kept)
    xc = x.detach().cpu().requires_grad_(True)
    yc = ops.rotary_qkv(xc * 1.0, H, D, positions=pos.cpu(), frequencies=w.cpu(), factor=factor, interleaved=True)
    gc, = torch.autograd.grad(yc, xc, d.cpu())
    assert torch.allclose(y.cpu(), yc, atol=1e-5) and torch.allclose(g.cpu(), gc, atol=1e-5)
    assert torch.equal(y[:, 2 * H * D:], x[:, 2 * H * D:]) and torch.equal(g[:, 2 * H * D:], d[:, 2 * H * D:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,D,n,interleaved", [(4, 64, 16, False), (3, 64, 25, True), (5, 37, 7, False), (2, 80, 40, True), (1, 512, 1, False)])
def test_packed_rotation_is_the_rotation_of_its_parts(dtype, H, D, n, interleaved, cuda_status):
    """In place, with the bits of `rotary` on q and k apart, both ways; values and their gradients pass as they are."""
    T = 131
    w, factor = ops.rotary_frequencies(2 * n, 1e4, None, "cuda")
    how = dict(positions=torch.randint(0, 3000, (T,), device="cuda", dtype=torch.int32), frequencies=w, factor=1.3, interleaved=interleaved)
    x = torch.randn(T, 3 * H * D, device="cuda").to(dtype).requires_grad_(True)
    given = x * 1.0
    at = given.data_ptr()
    y = ops.rotary_qkv(given, H, D, **how)
    assert y.data_ptr() == at
    d = torch.randn(T, 3 * H * D, device="cuda").to(dtype)
    g, = torch.autograd.grad(y, x, d)
    q, k, v = (t.detach().contiguous().requires_grad_(True) for t in x.view(T, 3, H, D).unbind(1))
    parts = [t.contiguous() for t in d.view(T, 3, H, D).unbind(1)]
    out = ops.rotary(q, k, **how)
    back = torch.autograd.grad(out, (q, k), parts[:2])
    assert torch.equal(y.view(T, 3, H, D), torch.stack((*out, v), 1)) and torch.equal(g.view(T, 3, H, D), torch.stack((*back, parts[2]), 1))
