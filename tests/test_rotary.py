"""Rotary positions in their general form: layouts, parts of a head, head counts, strides, far positions, scaled frequencies,
gradients; against a complex rotation in 64 bits."""
import math

import pytest
import torch

from nanoplm_b200.ops import functional as ops
from nanoplm_b200.ops import kernels as K

BF = torch.bfloat16


def _exact(x, pos, w, factor=1.0, interleaved=False, sign=1.0):
    """x [..., H, D] in 64 bits with its first 2 len(w) channels turned, and the sum of the magnitudes that meet in each value."""
    n = len(w)
    a = sign * pos.double()[..., None] * w
    t = torch.polar(torch.full_like(a, factor), a)[..., None, :]
    re, im = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    z = torch.complex(y[..., re].clone(), y[..., im].clone()) * t
    size[..., re] = size[..., im] = factor * (y[..., re].abs() + y[..., im].abs())
    y[..., re], y[..., im] = z.real, z.imag
    return y, size


def _close(got, x, pos, w, **how):
    """Within half a step of the type, which below its smallest normal number is that number's (fp16: 2^-14 eps / 2 = 2^-25, half of the
    subnormal numbers' distance 2^-24), and the fp32 errors before it: of an angle in turns, 2^-26 from the cast of the part behind
    the comma and 2^-50 of the turns before it (products of rounded fp64 numbers, here and in the 64-bit form), i.e.
    2 pi times that; of sincospi and factor 2^-22, of the two products and their sum 2^-23."""
    want, size = _exact(x, pos, w, **how)
    turns = float(pos.abs().max()) * float(w.max()) / (2 * math.pi) if pos.numel() else 0.0
    info = torch.finfo(got.dtype)
    tol = info.eps / 2 * want.abs().clamp(min=info.smallest_normal) + size * (2 * math.pi * (2.0 ** -26 + turns * 2.0 ** -50) + 2.0 ** -21)
    n = len(w)
    assert torch.equal(got[..., 2 * n:], x[..., 2 * n:])
    assert ((got.double() - want).abs() <= tol + 1e-30).all(), ((got.double() - want).abs() - tol).max()


def _w(n, device="cpu", theta=10000.0):
    return ops.rotary_frequencies(2 * n, theta, device=device)[0]


# ------------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,n", [(64, 32), (10, 3), (2, 1)])
def test_restatement(D, n, interleaved):
    q, k, pos, w = torch.randn(7, 3, D), torch.randn(7, 1, D), torch.randint(0, 9000, (7,)), _w(n)
    a, b = ops.rotary(q, k, positions=pos, frequencies=w, factor=1.25, interleaved=interleaved)
    _close(a, q, pos, w, factor=1.25, interleaved=interleaved)
    _close(b, k, pos, w, factor=1.25, interleaved=interleaved)
    assert torch.equal(ops.rotary(q, positions=pos, frequencies=w, factor=1.25, interleaved=interleaved), a)


@pytest.mark.parametrize("interleaved", [False, True])
def test_64_bit_heads_are_turned_in_64_bits(interleaved):
    """To the last bits: cos, sin and the factor with them 3 roundings, the two products and their sum 3."""
    q, pos, w = torch.randn(7, 3, 10, dtype=torch.float64, requires_grad=True), torch.randint(0, 9000, (7,)), _w(4)
    how = dict(factor=1.25, interleaved=interleaved)
    got = ops.rotary(q, positions=pos, frequencies=w, **how)
    want, size = _exact(q.detach(), pos, w, **how)
    assert got.dtype == torch.float64 and ((got - want).abs() <= 16 * 2.0 ** -53 * size).all()
    assert torch.autograd.gradcheck(lambda t: ops.rotary(t, positions=pos, frequencies=w, **how), [q])


def test_plain_frequencies_are_those_of_the_tables():
    cos, sin = ops.rope_tables(100, 64, 10000.0, "cpu")
    w, factor = ops.rotary_frequencies(64, 10000.0)
    a = torch.arange(100).double()[:, None] * w
    assert factor == 1.0 and (a.cos() - cos).abs().max() < 1e-5 and (a.sin() - sin).abs().max() < 1e-5


def test_scaled_frequencies():
    n, s = 32, 8.0
    w = _w(n)
    linear, f = ops.rotary_frequencies(64, 10000.0, {"type": "linear", "factor": s})
    assert torch.allclose(linear, w / s, rtol=1e-12) and f == 1.0
    ntk, f = ops.rotary_frequencies(64, 10000.0, {"type": "ntk", "factor": s})
    assert torch.allclose(ntk[0], w[0]) and torch.allclose(ntk[-1], w[-1] / s, rtol=1e-9) and f == 1.0
    scaling = {"type": "yarn", "factor": s, "original_max_position": 1024}
    yarn, f = ops.rotary_frequencies(64, 10000.0, scaling)
    turns = 1024 * w / (2 * math.pi)
    assert torch.allclose(yarn[turns >= 32], w[turns >= 32], rtol=1e-12)
    assert torch.allclose(yarn[turns <= 1], w[turns <= 1] / s, rtol=1e-12)
    assert bool((yarn <= w * (1 + 1e-12)).all() and (yarn >= w / s * (1 - 1e-12)).all())
    assert f == pytest.approx(0.1 * math.log(s) + 1)
    assert ops.rotary_frequencies(64, 10000.0, dict(scaling, attention_factor=1.0))[1] == 1.0


@pytest.mark.parametrize("rotated,theta,s,first", [(64, 1e4, 4.0, 1024), (128, 1e4, 8.0, 4096), (32, 1.6e5, 2.0, 64), (2, 1e4, 2.0, 64)])
def test_yarn_with_whole_pairs_at_the_ends_of_its_ramp(rotated, theta, s, first):
    """`truncate`: the blend goes linearly from the pair below the one that turns beta_fast times to the pair above the one that turns beta_slow
    times, both within the head; without it from the fractional places themselves. Pair by pair, and the two differ."""
    scaling = {"type": "yarn", "factor": s, "original_max_position": first}
    place = lambda turns: rotated * math.log(first / (turns * 2 * math.pi)) / (2 * math.log(theta))
    found = {}
    for truncate in (False, True):
        got, f = ops.rotary_frequencies(rotated, theta, dict(scaling, truncate=truncate))
        low, high = place(32.0), place(1.0)
        if truncate:
            low, high = max(math.floor(low), 0), min(math.ceil(high), rotated - 1)
        for i in range(rotated // 2):
            w = theta ** (-2 * i / rotated)
            slowed = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            assert float(got[i]) == pytest.approx(w / s * slowed + w * (1 - slowed), rel=1e-12), i
        assert f == pytest.approx(0.1 * math.log(s) + 1)
        found[truncate] = got
    assert torch.equal(found[False], ops.rotary_frequencies(rotated, theta, scaling)[0])
    assert rotated == 2 or (found[True] / found[False] - 1).abs().max() > 0.01


@pytest.mark.parametrize("args", [(3, 1e4), (0, 1e4), (4, 1e4, {"type": "other", "factor": 2}), (4, 1e4, {"type": "linear", "factor": 0.5}),
                                  (4, 1e4, {"type": "yarn", "factor": 2, "original_max_position": 8, "beta_fast": 1})])
def test_frequencies_that_are_refused(args):
    with pytest.raises(ValueError):
        ops.rotary_frequencies(*args)


def test_refusals():
    q, k, pos, w = torch.randn(5, 2, 8), torch.randn(5, 1, 8), torch.arange(5), _w(2)
    bad = [dict(q=q[0]), dict(k=k[:4]), dict(k=k[..., :6]), dict(k=k.double()), dict(k=k[None]), dict(q=q[:, :0]),
           dict(positions=pos.float()), dict(positions=pos[:4]), dict(positions=pos[None, :4]), dict(frequencies=w.float()),
           dict(frequencies=_w(5)), dict(frequencies=w[:0]), dict(frequencies=_w(4)[::2])]
    for change in bad:
        a = dict(q=q, k=k, positions=pos, frequencies=w) | change
        with pytest.raises(ValueError):
            ops.rotary(a["q"], a["k"], positions=a["positions"], frequencies=a["frequencies"])
    with pytest.raises(ValueError):         # the kernel's wrapper takes no CPU tensors
        K.rotary(q, k, pos, w)
    with pytest.raises(ValueError):
        K.rotary(q[:, :1].expand(5, 2, 8), None, pos, w, inplace=True)
    with pytest.raises(ValueError):
        K.rotary(q.transpose(1, 2), None, pos, w)
    for out in ((q,), (q[:4], k), (q.double(), k), (q, None)):
        with pytest.raises(ValueError):
            K.rotary(q, k, pos, w, out=out if len(out) == 2 else (out[0], k[:, :, :6]))
    with pytest.raises(ValueError):         # one memory for both
        K.rotary(q, q, pos, w, inplace=True)


# ------------------------------------------------------------------------------------------- GPU
SHAPES = [  # tokens, query heads, key heads, width, pairs
    (1, 1, 1, 2, 1), (1, 8, 8, 64, 32), (3, 5, 0, 70, 17), (129, 4, 1, 128, 16), (77, 3, 3, 80, 40), (250, 12, 2, 64, 31),
    (33, 2, 1, 512, 256), (19, 70, 3, 6, 1), (11, 1, 1, 511, 255), (4097, 2, 2, 32, 12),
    (300, 6, 2, 64, 25), (1, 4, 4, 128, 1), (900, 5, 0, 80, 21), (40, 48, 12, 96, 47), (64, 3, 2, 8, 3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,Hk,D,n", SHAPES)
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_and_gradient(T, H, Hk, D, n, dtype, interleaved, cuda_status):
    g = lambda *s: torch.randn(*s, device="cuda").to(dtype)
    packed = g(T, (H + 2 * Hk) * D)                       # heads inside a projection's row
    q = packed[:, :H * D].view(T, H, D).requires_grad_(True)
    k = packed[:, H * D:(H + Hk) * D].view(T, Hk, D).requires_grad_(True) if Hk else None
    pos = torch.randint(0, 3000, (T,), device="cuda", dtype=torch.int32)
    w = _w(n, "cuda")
    out = ops.rotary(q, k, positions=pos, frequencies=w, factor=1.2, interleaved=interleaved)
    both = (q, k) if Hk else (q,)
    out = out if Hk else (out,)
    grads = [g(*t.shape) for t in both]
    back = torch.autograd.grad(out, both, grads)
    how = dict(factor=1.2, interleaved=interleaved)
    for x, y, d, dx in zip(both, out, grads, back):
        _close(y.detach(), x.detach(), pos, w, **how)
        _close(dx, d, pos, w, sign=-1.0, **how)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("first", [-5, 10 ** 6, 2 ** 31 - 40])
def test_far_positions(dtype, first, cuda_status):
    q, w = torch.randn(40, 2, 64, device="cuda"), _w(32, "cuda")
    pos = torch.arange(first, first + 40, device="cuda").clamp(max=2 ** 31 - 1).to(dtype)
    _close(ops.rotary(q, positions=pos, frequencies=w), q, pos, w)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1])
def test_batches_orders_and_addresses(shift, cuda_status):
    """[B, S, H, D] views of a [B, H, S, D] tensor, at an odd address, positions of each sequence or for all."""
    B, S, H, D = 3, 37, 4, 64
    flat = torch.randn(shift + B * H * S * D, device="cuda").to(BF)
    q = flat[shift:].view(B, H, S, D).transpose(1, 2)
    k = torch.randn(B, S, 1, D, device="cuda").to(BF).expand(B, S, 2, D)
    w = _w(16, "cuda")
    for pos in (torch.randint(0, 999, (B, S), device="cuda"), torch.randint(0, 999, (S, B), device="cuda").t(),
                torch.randint(0, 999, (2 * S,), device="cuda")[::2]):
        a, b = ops.rotary(q, k, positions=pos, frequencies=w, interleaved=True)
        for got, x in ((a, q), (b, k)):
            assert got.is_contiguous()
            _close(got, x, pos.expand(B, S), w, interleaved=True)


@pytest.mark.gpu
def test_in_place_leaves_the_rest(cuda_status):
    T, H, Hk, D, n = 130, 6, 2, 64, 24
    packed = torch.randn(T, (H + 2 * Hk) * D, device="cuda").to(BF)
    before = packed.clone()
    parts = lambda p: (p[:, :H * D].view(T, H, D), p[:, H * D:(H + Hk) * D].view(T, Hk, D))
    pos, w = torch.arange(T, device="cuda"), _w(n, "cuda")
    q, k = parts(packed)
    K.rotary(q, k, pos, w, inplace=True)
    for got, x in zip(parts(packed), parts(before)):
        _close(got, x, pos, w)
    assert torch.equal(packed[:, (H + Hk) * D:], before[:, (H + Hk) * D:])


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,D,n,row,at", [(4, 4, 75, 25, 904, 0), (4, 2, 75, 37, 900, 4), (2, 4, 75, 3, 1000, 8), (8, 8, 33, 10, 1000, 0), (6, 2, 34, 1, 600, 2),
                                            (3, 1, 64, 25, 520, 8), (2, 2, 80, 20, 480, 16), (1, 1, 10, 5, 24, 4), (16, 16, 128, 31, 6200, 8)])
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_heads_that_lie_side_by_side(H, Hk, D, n, row, at, dtype, interleaved, cuda_status):
    """Pairs narrower than 16 bytes in heads that move in pieces of 4, 8 or 16 bytes, in rows of tokens with something before, between and
    behind them, which stays as it is where the heads are turned in place."""
    T = 211
    first = torch.randn(T, row, device="cuda").to(dtype)
    pos, w = torch.randint(0, 3000, (T,), device="cuda"), _w(n, "cuda")
    cut = lambda t: (t[:, at:at + H * D].view(T, H, D), t[:, row - Hk * D:].view(T, Hk, D))
    a, b = K.rotary(*cut(first), pos, w, factor=1.2, interleaved=interleaved)
    for got, t in zip((a, b), cut(first)):
        _close(got, t, pos, w, factor=1.2, interleaved=interleaved)
    here = first.clone()
    K.rotary(*cut(here), pos, w, factor=1.2, interleaved=interleaved, out=cut(here))
    assert all(torch.equal(s, t) for s, t in zip(cut(here), (a, b)))
    for t in (here, first):
        for part in cut(t):
            part.zero_()
    assert torch.equal(here, first)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [24, 25])
def test_given_outputs_of_other_strides(n, cuda_status):
    """Outputs inside wider rows, and one that starts where the input does but with other strides."""
    T, H, D = 70, 3, 64
    pos, w = torch.arange(T, device="cuda"), _w(n, "cuda")
    q, k = torch.randn(T, H, D, device="cuda"), torch.randn(T, 1, D, device="cuda")
    wide = torch.full((T, (H + 2) * D), 7.0, device="cuda")
    a, b = wide[:, :H * D].view(T, H, D), wide[:, H * D:(H + 1) * D].view(T, 1, D)
    got = K.rotary(q, k, pos, w, out=(a, b))
    assert got[0] is a and got[1] is b
    _close(a, q, pos, w)
    _close(b, k, pos, w)
    assert (wide[:, (H + 1) * D:] == 7.0).all()
    one = torch.randn(1, 2 * D, device="cuda")
    x, y = one.view(1, 2, D)[:, :1], one.as_strided((1, 1, D), (D, 5 * D, 1))        # one token, one head: the same elements
    before = x.clone()
    K.rotary(x, None, pos[:1] + 3, w, out=(y, None))
    _close(y, before, pos[:1] + 3, w)


@pytest.mark.gpu
def test_no_tokens_and_unused_outputs(cuda_status):
    w = _w(4, "cuda")
    q = torch.randn(0, 2, 8, device="cuda", requires_grad=True)
    y = ops.rotary(q, positions=torch.zeros(0, device="cuda", dtype=torch.int32), frequencies=w)
    assert y.shape == q.shape and torch.autograd.grad(y.sum(), q)[0].shape == q.shape
    q, k = (torch.randn(5, h, 8, device="cuda", requires_grad=True) for h in (2, 1))
    pos = torch.arange(5, device="cuda")
    a, b = ops.rotary(q, k, positions=pos, frequencies=w)
    d = torch.randn_like(b)
    dk, = torch.autograd.grad(b, k, d, retain_graph=True)
    _close(dk, d, pos, w, sign=-1.0)
    dq, none = torch.autograd.grad(a, (q, k), torch.ones_like(a), allow_unused=True, create_graph=False)
    assert none is None
    _close(dq, torch.ones_like(a), pos, w, sign=-1.0)


@pytest.mark.gpu
def test_gradient_of_the_gradient_and_differences(cuda_status):
    """The rotation is linear: <d, R x> = <R' d, x> exactly, and the gradient with respect to d is the rotation again."""
    w, pos = _w(8, "cuda"), torch.arange(9, device="cuda")
    x = torch.randn(9, 3, 20, device="cuda", requires_grad=True)
    d = torch.randn(9, 3, 20, device="cuda", requires_grad=True)
    y = ops.rotary(x, positions=pos, frequencies=w, factor=0.7)
    dx, = torch.autograd.grad(y, x, d, create_graph=True)
    assert ((y.double() * d.double()).sum() - (x.double() * dx.double()).sum()).abs() < 1e-5 * x.numel() ** 0.5
    back, = torch.autograd.grad(dx, d, x.detach())
    _close(back, x.detach(), pos, w, factor=0.7)


@pytest.mark.gpu
def test_captured_and_on_another_stream(cuda_status):
    """A replay reads the positions and values that are there then; another stream gives the same bits."""
    w = _w(32, "cuda")
    q, pos = torch.randn(300, 4, 64, device="cuda").to(BF), torch.arange(300, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want, _ = K.rotary(q, None, pos, w)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = K.rotary(q, None, pos, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    pos += 1000
    graph.replay()
    _close(got, q, pos, w)
    # tokens past 32-bit offsets: rows far apart in a large buffer
    big = torch.empty(3 * 2 ** 30 + 512, dtype=BF, device="cuda")
    far = big.as_strided((4, 2, 64), (2 ** 30, 64, 1))
    far.copy_(torch.randn(4, 2, 64))
    _close(K.rotary(far, None, pos[:4], w)[0], far, pos[:4], w)


@pytest.mark.gpu
@pytest.mark.parametrize("D,n", [(64, 25), (75, 25), (66, 10)])
def test_narrow_pairs_past_32_bit_offsets(D, n, cuda_status):
    """Tokens 2^30 elements apart, and tokens within 31 bits of one another."""
    pos, w = torch.randint(0, 3000, (4,), device="cuda"), _w(n, "cuda")
    big = torch.empty(3 * 2 ** 30 + 2 * D, dtype=BF, device="cuda")
    for apart in (2 ** 30, 2 ** 28 + 2):
        far = big.as_strided((4, 2, D), (apart, D, 1))
        far.copy_(torch.randn(4, 2, D))
        got = K.rotary(far, None, pos, w)[0]
        _close(got, far, pos, w)
        assert torch.equal(got, K.rotary(far.contiguous(), None, pos, w)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("D,n", [(64, 25), (75, 30), (34, 10)])
def test_narrow_pairs_in_batches(D, n, cuda_status):
    """[B, S, H, D]: batches behind one another, in another order, between others, and one for all; positions of their own or for all."""
    B, S, H = 3, 53, 4
    w = _w(n, "cuda")
    full = torch.randn(2 * B, S, H, D, device="cuda").to(BF)
    orders = (full[:B], full[::2], torch.randn(B, H, S, D, device="cuda").to(BF).transpose(1, 2), full[:1].expand(B, S, H, D),
              torch.randn(S, B, H, D, device="cuda").to(BF).transpose(0, 1), full[:B, :, 1:3])
    for q in orders:
        for pos in (torch.randint(0, 999, (B, S), device="cuda"), torch.randint(0, 999, (S,), device="cuda")):
            a, b = K.rotary(q, full[B:, :, :2], pos, w)
            _close(a, q, pos.expand(B, S), w)
            _close(b, full[B:, :, :2], pos.expand(B, S), w)
