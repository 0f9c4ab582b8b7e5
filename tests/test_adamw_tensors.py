"""One AdamW step over a list of tensors with moments in fp32 or 8 bits: the restatement on the CPU, and the kernel against it."""
import math

import pytest
import torch

from nanoplm_b200.ops import kernels as K
from nanoplm_b200.ops import moments as M

BF, F32 = torch.bfloat16, torch.float32
SIZES = [(3,), (256,), (257,), (40, 64), (1,), (0,), (33, 33), (8192 + 256 + 5,), (64, 256)]


def _hyper(t, lr=1e-2, b1=0.9, b2=0.999, wd=0.1, gs=0.5, most=1.0, device="cpu"):
    return torch.tensor([lr, b1, b2, 1e-8, wd, 1 - b1 ** t, 1 - b2 ** t, gs, most], device=device)


def _set(shapes, p_type, g_type, shift=0, seed=0):
    """(params, grads, copies or None) on the CPU; with shift inside larger buffers at odd addresses."""
    gen = torch.Generator().manual_seed(seed)

    def make(dtype, scale):
        out = []
        for s in shapes:
            n = math.prod(s)
            buf = torch.zeros(n + shift, dtype=dtype)
            buf[shift:] = (scale * torch.randn(n, generator=gen) * torch.exp(2 * torch.randn(n, generator=gen))).to(dtype)
            out.append(buf[shift:].view(s))
        return out
    params = make(p_type, 0.1)
    return params, make(g_type, 0.01), [torch.zeros_like(p, dtype=BF) for p in params] if p_type == F32 else None


# ------------------------------------------------------------------------------------------- CPU
def test_fp32_moments_follow_torch():
    params, grads, copies = _set([(5, 7), (300,)], F32, F32)
    ref = [p.clone().requires_grad_(True) for p in params]
    opt = torch.optim.AdamW([{"params": ref[:1], "weight_decay": 0.1}, {"params": ref[1:], "weight_decay": 0.0}], lr=1e-2)
    st = M.TensorMoments([p.numel() for p in params], "cpu")
    for t in range(1, 8):
        for r, g in zip(ref, grads):
            r.grad = g * 0.5
        opt.step()
        st.step(params, grads, _hyper(t, most=0.0), copies=copies, decay=[True, False])
    for p, r, c in zip(params, ref, copies):
        assert torch.allclose(p, r, rtol=1e-5, atol=1e-6) and torch.equal(c, p.to(BF))


def test_codes_are_neighbours_and_come_back():
    x = torch.randn(4 * M.BLOCK) * torch.exp(4 * torch.randn(4 * M.BLOCK))
    x[5] = 0.0
    for values, signed, octaves in ((x, True, 15), (x.square(), False, 31)):
        for r in (0, 0x80000, 0xfffff):
            codes, e = M.encode(values, r, signed)
            back = M.decode(codes, e, signed)
            assert back[5] == 0
            big = values.abs() > values.abs().view(-1, M.BLOCK).amax(1).repeat_interleave(M.BLOCK) * 2.0 ** -(octaves - 1)
            # 3 bits of mantissa: neighbours are an eighth of the octave apart, the nearest half of that
            step = torch.exp2(torch.floor(torch.log2(values.abs().clamp(min=1e-30)))) / 8
            assert ((back - values).abs()[big] <= (step * (0.5 if r == 0x80000 else 1) * (1 + 1e-6))[big]).all()
            again, e2 = M.encode(back, 0x80000, signed)
            assert torch.equal(M.decode(again, e2, signed), back)
            assert signed or (back[values > 0] > 0).all()


def test_rounding_keeps_the_mean():
    """The mean of n independent roundings of x is off x by at most 5 of its deviations: a value that is kept as a or b, d apart,
    has a deviation of at most d / 2."""
    n = 4096
    for signed, value in ((True, 1.03), (True, -0.9999), (False, 0.7), (True, 2.0 ** -17 * 1.3), (True, -(2.0 ** -16))):
        x = torch.full((n * M.BLOCK // 256, 256), value)
        x[:, 0] = 1.5 if abs(value) < 1 else value          # the largest of every block
        r = M.random_bits(x.numel(), torch.tensor([12345])) & 0xfffff
        codes, e = M.encode(x.view(-1), r, signed)
        back = M.decode(codes, e, signed).view(-1, 256)[:, 1:].double()
        d = float(back.max() - back.min())
        assert abs(float(back.mean()) - value) <= 5 * max(d, 1e-12) / 2 / back.numel() ** 0.5 + abs(value) * 2e-6
        assert len(back.unique()) <= 2


def test_slow_average_is_followed():
    """A second moment that moves by 0.1 % a step reaches its gradient's square, which rounding to the nearest code would not let
    it do: after 4 000 steps the fp32 average is at 98 % of it."""
    st = M.TensorMoments([512], "cpu", 8)
    p, g = torch.zeros(512), torch.full((512,), 0.1)
    for t in range(1, 4001):
        st.step([p], [g], _hyper(t, most=0.0, gs=1.0), rng=torch.tensor([t * 7919]))
    v = st.values()[1][0]
    assert float(v.mean()) == pytest.approx(0.01 * (1 - 0.999 ** 4000), rel=0.05)


@pytest.mark.parametrize("bits", [8, 32])
def test_states_load_what_they_gave(bits):
    shapes = [(300,), (5, 5), (700,)]
    params, grads, _ = _set(shapes, F32, F32)
    st = M.TensorMoments([p.numel() for p in params], "cpu", bits)
    for t in (1, 2, 3):
        st.step(params, grads, _hyper(t), rng=torch.tensor([t]))
    m, v = st.values()
    other = M.TensorMoments([p.numel() for p in params], "cpu", bits)
    other.load([t.clone() for t in m], [t.clone() for t in v])
    assert all(torch.equal(a, b) for a, b in zip(m + v, sum(other.values(), [])))
    assert st.nbytes() == (6 if bits == 8 else 6) * 256 * (2 if bits == 8 else 8) + (12 if bits == 8 else 0)


def test_refusals():
    params, grads, copies = _set([(300,), (8,)], F32, F32)
    st = M.TensorMoments([300, 8], "cpu", 8)
    rng, hyper = torch.tensor([1]), _hyper(1)
    ok = dict(params=params, grads=grads, hyper=hyper, rng=rng, copies=copies, decay=None, sumsq=None)
    step = lambda **k: (lambda a: st.step(a.pop("params"), a.pop("grads"), a.pop("hyper"), **a))(ok | k)
    step()
    for bad in (dict(params=params[:1], grads=grads[:1], copies=copies[:1]), dict(grads=grads[:1]), dict(copies=copies[:1]),
                dict(decay=[True]), dict(rng=None), dict(rng=torch.tensor([1.0])), dict(hyper=hyper[:8]), dict(hyper=hyper.double()),
                dict(grads=[grads[0], grads[1].to(BF)]), dict(grads=[g.double() for g in grads]), dict(copies=grads),
                dict(grads=[grads[0][:299], grads[1]]), dict(sumsq=torch.zeros(2)), dict(params=[p.half() for p in params])):
        with pytest.raises(ValueError):
            step(**bad)
    with pytest.raises(ValueError):     # bf16 copies of bf16 params
        step(params=[p.to(BF) for p in params])
    with pytest.raises(ValueError):     # the same tensor twice
        M.TensorMoments([8, 8], "cpu").step([params[1]] * 2, [grads[1]] * 2, hyper)
    two = [torch.zeros(8), torch.zeros(8)]
    with pytest.raises(ValueError, match="twice"):     # the same copy twice, of which one would be lost
        M.TensorMoments([8, 8], "cpu").step(two, [grads[1]] * 2, hyper, copies=[copies[1]] * 2)
    M.TensorMoments([8, 8, 0, 0], "cpu").step(two + [torch.zeros(0)] * 2, [grads[1]] * 2 + [torch.zeros(0)] * 2, hyper,
                                              copies=[copies[1], copies[1].clone()] + [torch.zeros(0, dtype=BF)] * 2)
    with pytest.raises(ValueError):     # not contiguous
        M.TensorMoments([16], "cpu").step([torch.zeros(4, 4).t()[:, :]], [torch.zeros(4, 4)], hyper)
    with pytest.raises(ValueError):
        M.TensorMoments([8], "cpu", 16)
    with pytest.raises(ValueError):
        st.load([torch.zeros(300)], [torch.zeros(300)])
    with pytest.raises(ValueError):     # too few blocks
        K.check_step(params, grads, None, None, torch.zeros(512), torch.zeros(512), None, hyper, None, None)
    with pytest.raises(ValueError):     # codes without their scales
        K.check_step(params, grads, None, None, torch.zeros(768, dtype=torch.uint8), torch.zeros(768, dtype=torch.uint8), None, hyper, rng, None)


# ------------------------------------------------------------------------------------------- GPU
def _both(shapes, p_type, g_type, bits, shift=0, steps=3, clip=True, decay=None):
    """The same steps on the CPU and on the GPU: ([params, copies, m, v, scales] of each)."""
    params, grads, copies = _set(shapes, p_type, g_type, shift)
    dev = lambda ts: None if ts is None else [torch.cat((torch.zeros(shift, dtype=t.dtype), t.reshape(-1))).cuda()[shift:].view(t.shape) for t in ts]
    gp, gg, gc = dev(params), dev(grads), dev(copies)
    sizes = [p.numel() for p in params]
    a, b = M.TensorMoments(sizes, "cpu", bits), M.TensorMoments(sizes, "cuda", bits)
    sumsq = torch.stack([g.float().square().sum() for g in grads]).sum().reshape(1) if clip else None
    for t in range(1, steps + 1):
        rng = torch.tensor([t * 2 ** 33 + 17 * t])
        a.step(params, grads, _hyper(t), rng=rng, copies=copies, decay=decay, sumsq=sumsq)
        b.step(gp, gg, _hyper(t, device="cuda"), rng=rng.cuda(), copies=gc, decay=decay, sumsq=None if sumsq is None else sumsq.cuda())
    return (params, copies, a), (gp, gc, b)


def _same(cpu, gpu, p_type):
    (p, c, a), (gp, gc, b) = cpu, gpu
    assert torch.equal(a.m, b.m.cpu()) and torch.equal(a.v, b.v.cpu())
    assert a.scales is None or torch.equal(a.scales, b.scales.cpu())
    for x, y in zip(p, gp):
        x, y = x.double(), y.cpu().double()
        # each of three steps: the quotient is good to 2^-20 of at most 10 lr (m / sqrt v is at most 1 / sqrt(1 - b2)), the
        # sum to a step of the weight's type, which may be rounded the other way
        tol = 3 * (0.01 * 32 * 2.0 ** -20 + 2 * torch.finfo(p_type).eps / 2 * x.abs())
        assert ((x - y).abs() <= tol).all()
    for x, y in zip(gp, gc or ()):
        assert torch.equal(x.to(BF), y)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("p_type,g_type", [(F32, F32), (F32, BF), (BF, BF), (BF, F32)])
@pytest.mark.parametrize("shift", [0, 1])
def test_kernel_has_the_bits_of_the_restatement(bits, p_type, g_type, shift, cuda_status):
    if p_type == BF:        # a weight that is rounded the other way changes no moment: gradients are given
        cpu, gpu = _both(SIZES, p_type, g_type, bits, shift, decay=[i % 2 == 0 for i in range(len(SIZES))])
    else:
        cpu, gpu = _both(SIZES, p_type, g_type, bits, shift, clip=shift == 0)
    _same(cpu, gpu, p_type)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e-15, 1.0, 1e12, 1e17])
def test_codes_of_extreme_and_of_far_apart_gradients(size, cuda_status):
    """Gradients over 40 octaves inside a block, so that most moments are below code 1, or zero, at sizes at which squares leave fp32's
    normal range on either side."""
    torch.manual_seed(3)
    g = size * torch.randn(4096) * torch.exp2(-40 * torch.rand(4096))
    g[::7] = 0.0
    a, b = M.TensorMoments([4096], "cpu", 8), M.TensorMoments([4096], "cuda", 8)
    p, q = torch.randn(4096), None
    q = p.cuda()
    for t in (1, 2, 3):
        rng = torch.tensor([t * 12345678901])
        a.step([p], [g], _hyper(t, gs=1.0, most=0.0), rng=rng)
        b.step([q], [g.cuda()], _hyper(t, gs=1.0, most=0.0, device="cuda"), rng=rng.cuda())
        assert torch.equal(a.scales, b.scales.cpu()) and torch.equal(a.m, b.m.cpu()) and torch.equal(a.v, b.v.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("exponent", [1, 2, 14, 15, 16, 17, 30, 31, 32, 33, 150, 235, 236, 237, 238, 251, 252, 253, 254])
@pytest.mark.parametrize("second", [False, True])
def test_codes_at_the_ends_of_the_exponents(exponent, second, cuda_status):
    """Blocks whose largest moment has a given exponent field, with elements in every octave down to fp32's smallest numbers, and again
    with all of them in the block's two lowest octaves: the restatement's bits, where the kernel's two ways of coding meet and
    where a block reaches below the normal range. With beta 0 a moment is its gradient, or the gradient's square."""
    gen = torch.Generator().manual_seed(exponent)
    n, below = 4096, 31 if second else 15
    lowest = max(exponent - below, 0)
    fields = torch.cat((torch.randint(0, exponent + 1, (n,), generator=gen), torch.randint(max(lowest - 1, 0), min(lowest + 2, exponent + 1), (n,), generator=gen)))
    patterns = (fields << 23) + torch.randint(0, 2 ** 23, (2 * n,), generator=gen)
    patterns[::256] = (exponent << 23) + 12345                  # the largest of the block, which no rounding takes beyond its exponent
    patterns = torch.minimum(patterns, patterns[::256].repeat_interleave(256))
    x = patterns.to(torch.int32).view(F32)
    g = x.double().sqrt().float() if second else x * torch.where(torch.rand(2 * n, generator=gen) < 0.5, -1.0, 1.0)
    a, b = M.TensorMoments([2 * n], "cpu", 8), M.TensorMoments([2 * n], "cuda", 8)
    for t in (1, 2, 3):
        how, rng = dict(lr=0.0, b1=0.0, b2=0.0, gs=1.0, most=0.0), torch.tensor([t * 98765432109])
        a.step([torch.zeros(2 * n)], [g], _hyper(t, **how), rng=rng)
        b.step([torch.zeros(2 * n, device="cuda")], [g.cuda()], _hyper(t, device="cuda", **how), rng=rng.cuda())
        assert set(a.scales[int(second)].tolist()) == set(b.scales[int(second)].tolist()) == {exponent}
        assert torch.equal(a.v if second else a.m, (b.v if second else b.m).cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("step", [1, 100])
@pytest.mark.parametrize("eps", [1e-18, 1e-15, 1e-13, 1e-11, 1e-10, 1e-8])
def test_second_moments_below_the_normal_range_beside_epsilon(eps, step, cuda_status):
    """The update of weights of zero from moments down to fp32's smallest numbers, against the formula in 64 bits from the step's own
    moments. Rounded: the root by 2^-23, the correction's root, its reciprocal and the product with it 3 x 2^-24, the sum 2^-24, its
    reciprocal 2^-23, the learning rate over its correction, and two products 3 x 2^-24: below 2^-20 of the update."""
    n = 4096
    v = torch.exp2(-149 + 40 * torch.rand(n)).clamp(min=2.0 ** -149)
    m = torch.randn(n).abs() * 2.0 ** -60 + 2.0 ** -61
    st = M.TensorMoments([n], "cuda")
    st.load([m], [v])
    p, hyper = torch.zeros(n, device="cuda"), _hyper(step, gs=1.0, most=0.0, device="cuda")
    hyper[3] = eps
    st.step([p], [torch.zeros_like(p)], hyper)
    lr, b1, b2, eps32, wd, bc1, bc2, _, _ = hyper.double()
    want = -lr / bc1 * st.m.double() / ((st.v.double() / bc2).sqrt() + eps32)
    assert ((p.double() - want).abs() <= 2.0 ** -20 * want.abs()).all(), float(((p.double() - want) / want).abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("p_type,g_type", [(F32, F32), (F32, BF), (BF, BF), (BF, F32)])
@pytest.mark.parametrize("shifts", [(1, 1, 1), (1, 0, 0), (0, 1, 1), (2, 3, 1), (3, 2, 2), (5, 4, 7)])
def test_tensors_at_any_address_beside_others(bits, p_type, g_type, shifts, cuda_status):
    """Weights, gradients and copies that start at addresses of their own, between numbers that are none: the bits of the same step on
    16 bytes, and the neighbours as they were."""
    shapes = [(256,), (255,), (20000 + 7,), (1,), (40, 64), (8192,)]
    params, grads, copies = _set(shapes, p_type, g_type)
    whole = [[t.cuda() for t in ts] if ts else None for ts in (params, grads, copies)]
    bufs, cut = [], []
    for ts, at in zip((params, grads, copies), shifts):
        bufs.append([torch.full((t.numel() + 16,), float("nan"), dtype=t.dtype, device="cuda") for t in ts] if ts else None)
        cut.append([b[at:at + t.numel()].copy_(t.cuda().view(-1)).view(t.shape) for b, t in zip(bufs[-1], ts)] if ts else None)
    sizes = [t.numel() for t in params]
    a, b = M.TensorMoments(sizes, "cuda", bits), M.TensorMoments(sizes, "cuda", bits)
    for t in (1, 2):
        rng = torch.tensor([t * 7 ** 11], device="cuda")
        for st, (p, g, c) in ((a, whole), (b, cut)):
            st.step(p, g, _hyper(t, device="cuda"), rng=rng, copies=c)
    assert torch.equal(a.m, b.m) and torch.equal(a.v, b.v) and (bits == 32 or torch.equal(a.scales, b.scales))
    for x, y, buf in zip(whole, cut, bufs):
        for s, t, around in zip(x or (), y or (), buf or ()):
            assert torch.equal(s, t)
            assert int(around.isnan().sum()) == 16


@pytest.mark.gpu
def test_more_tensors_than_a_launch_takes(cuda_status):
    shapes = [(1 + 37 * i % 900,) for i in range(301)]
    _same(*_both(shapes, F32, F32, 8, steps=1), F32)


@pytest.mark.gpu
def test_nothing_behind_a_tensor_is_written(cuda_status):
    """Views of one buffer with a gap behind each keep their gaps."""
    buf = torch.randn(4, 700, device="cuda")
    before = buf.clone()
    params = [buf[i, :n] for i, n in enumerate((1, 255, 513, 690))]
    grads = [torch.randn_like(p) for p in params]
    st = M.TensorMoments([p.numel() for p in params], "cuda", 8)
    st.step(params, grads, _hyper(1, device="cuda"), rng=torch.tensor([3], device="cuda"))
    for i, p in enumerate(params):
        assert torch.equal(buf[i, p.numel():], before[i, p.numel():]) and not torch.equal(p, before[i, :p.numel()])
        assert not M.decode(st.m.cpu(), st.scales[0].cpu(), True).view(-1)[sum(-(-q.numel() // 256) for q in params[:i]) * 256 + p.numel():][:-p.numel() % 256].any()


@pytest.mark.gpu
def test_captured_step_reads_its_numbers_at_replay(cuda_status):
    shapes = [(700,), (64, 64)]
    params, grads, copies = ([t.cuda() for t in ts] for ts in _set(shapes, F32, F32))
    eager = [[t.clone() for t in ts] for ts in (params, grads, copies)]
    sizes = [p.numel() for p in params]
    a, b = M.TensorMoments(sizes, "cuda", 8), M.TensorMoments(sizes, "cuda", 8)
    hyper, rng = _hyper(1, device="cuda"), torch.tensor([1], device="cuda")
    graph = torch.cuda.CUDAGraph()
    a.step(params, grads, hyper, rng=rng, copies=copies)       # (loads the library)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a.step(params, grads, hyper, rng=rng, copies=copies)
    b.step(*eager[:2], _hyper(1, device="cuda"), rng=torch.tensor([1], device="cuda"), copies=eager[2])
    for t in (2, 3, 4):
        hyper.copy_(_hyper(t, lr=1e-2 * t))
        rng.fill_(t * 99)
        graph.replay()
        b.step(*eager[:2], _hyper(t, lr=1e-2 * t, device="cuda"), rng=torch.tensor([t * 99], device="cuda"), copies=eager[2])
    assert all(torch.equal(x, y) for x, y in zip(params + copies + [a.m, a.v, a.scales], eager[0] + eager[2] + [b.m, b.v, b.scales]))


@pytest.mark.gpu
def test_values_and_codes(cuda_status):
    (_, _, a), (_, _, b) = _both([(5000,), (77,)], F32, F32, 8)
    for dtype in (F32, BF):
        m, v = K.moment_values(b.m, b.v, b.scales, dtype)
        assert torch.equal(m.cpu().float(), M.decode(a.m, a.scales[0], True))
        assert torch.equal(v.cpu().float(), M.decode(a.v, a.scales[1], False))
    m, v = K.moment_values(b.m, b.v, b.scales)
    again = K.moment_values(*K.moment_codes(m, v))
    assert torch.equal(again[0], m) and torch.equal(again[1], v)
    x, y = torch.randn(1024), torch.rand(1024) * torch.exp(9 * torch.randn(1024))
    codes = K.moment_codes(x.cuda(), y.cuda())
    for got, values, row, signed in ((codes[0], x, 0, True), (codes[1], y, 1, False)):
        c, e = M.encode(values, 0x80000, signed)
        assert torch.equal(got.cpu(), c) and torch.equal(codes[2][row].cpu(), e)


@pytest.mark.gpu
def test_tensor_past_32_bit_places(cuda_status):
    """2^32 + 700 elements: the blocks on both sides of place 2^32 and the last ones against a restatement of theirs alone, the random
    numbers of their places among it."""
    n, tail = 2 ** 32 + 700, 256 * 6
    p, g = torch.zeros(n, dtype=BF, device="cuda"), torch.zeros(n, dtype=BF, device="cuda")
    st = M.TensorMoments([n], "cuda", 8)
    first = 2 ** 32 - 256 * 3
    gen = torch.Generator().manual_seed(1)
    p[first:] = torch.randn(n - first, generator=gen).to(BF).cuda()
    g[first:] = torch.randn(n - first, generator=gen).to(BF).cuda()
    want_p, grad = p[first:].cpu(), g[first:].cpu()
    rng = torch.tensor([77])
    st.step([p], [g], _hyper(1, most=0.0, device="cuda"), rng=rng.cuda())
    m = torch.zeros(tail)
    m[:n - first] = grad.float() * 0.5 * (1 - _hyper(1)[1])
    v = torch.zeros(tail)
    v[:n - first] = (grad.float() * 0.5) ** 2 * (1 - _hyper(1)[2])
    key = M._mix((rng & M._LOW32) ^ M._mix(rng >> 32))
    at = torch.arange(first, first + tail)
    r = M._mix((at & M._LOW32) ^ M._mix((key + (at >> 32)) & M._LOW32))
    for codes, row, values, bits, signed in ((st.m, 0, m, r & 0xfffff, True), (st.v, 1, v, r >> 12, False)):
        c, e = M.encode(values, bits, signed)
        assert torch.equal(codes[first:first + tail].cpu(), c)
        assert torch.equal(st.scales[row, first // 256:first // 256 + 6].cpu(), e)
        assert not codes[:first].any()
    new = want_p.float() * (1 - 0.01 * 0.1) - 0.01 * torch.sign(grad.float())
    assert ((p[first:].cpu().float() - new).abs() <= 2 ** -8 * new.abs() + 1e-4).all()


@pytest.mark.gpu
def test_no_tensors(cuda_status):
    M.TensorMoments([], "cuda", 8).step([], [], _hyper(1, device="cuda"), rng=torch.tensor([1], device="cuda"))
    m, v = K.moment_values(*(torch.zeros(0, dtype=torch.uint8, device="cuda") for _ in range(2)), torch.zeros(2, 0, dtype=torch.uint8, device="cuda"))
    assert m.numel() == v.numel() == 0
