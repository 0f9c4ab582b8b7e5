"""Norm of a block's output, gate, residual scale, sum and the next norm in one operator, forward and backward, against the
formulas in 64 bits."""
import pytest
import torch

from nanoplm_b200.ops import functional as ops
from nanoplm_b200.ops import kernels as K

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-5


def _unit(v, rms):
    if not rms:
        v = v - v.mean(-1, keepdim=True)
    return v / (v.square().mean(-1, keepdim=True) + EPS).sqrt()


def _formula(x, f, post, nxt, gate, sigmoid, scale, rms):
    n = _unit(f, rms)
    n = n if post is None else n * post
    if gate is not None:
        n = n * (torch.sigmoid(gate) if sigmoid else gate)
    y = n + (x if scale is None else scale * x)
    h = _unit(y, rms)
    return y, h if nxt is None else h * nxt


def _inputs(T, C, dtype, gate, scaled, weighted, device, w_type=None):
    rnd = lambda *s: torch.randn(*s, device=device)
    w_type = w_type or dtype
    p = {"x": (2 * rnd(T, C)).to(dtype), "f": (0.5 * rnd(T, C) + 0.1).to(dtype), "post": None, "nxt": None, "gate": None, "scale": None}
    if weighted:
        p["post"], p["nxt"] = (1 + 0.2 * rnd(C)).to(w_type), (1 + 0.2 * rnd(C)).to(w_type)
    if gate == "channel":
        p["gate"] = (0.4 + 0.2 * rnd(C)).to(w_type)
    elif gate != "none":
        p["gate"] = rnd(T, C).to(dtype)
    if scaled:
        p["scale"] = (1 + 0.2 * rnd(C)).to(w_type)
    return {k: v if v is None else v.requires_grad_(True) for k, v in p.items()}


def _call(p, sigmoid, rms, **more):
    return ops.sandwich_norm(p["x"], p["f"], p["post"], p["nxt"], gate=p["gate"], sigmoid=sigmoid, scale=p["scale"], eps=EPS,
                             rms=rms, **more)


def _check(p, sigmoid, rms, use=("y", "h")):
    """Outputs and gradients. fp32 errors: every value of a row is a chain of some 40 operations on numbers no larger than the
    row's largest times 1 / std, and its two means are sums of depth log C + C / (8 threads): 256 units of 2^-24 of the
    row's largest. A sum over T rows adds those of its terms and T units more of the sum of their magnitudes."""
    names = [k for k in p if p[k] is not None]
    y, h = _call(p, sigmoid, rms, with_next="h" in use)
    ref = {k: (None if v is None else v.detach().double().requires_grad_(True)) for k, v in p.items()}
    ye, he = _formula(ref["x"], ref["f"], ref["post"], ref["nxt"], ref["gate"], sigmoid, ref["scale"], rms)
    out = {"y": (y, ye), "h": (h, he)}
    ds = {k: torch.randn_like(ye).to(p["x"].dtype) for k in use}
    u = 2.0 ** -24
    for k in use:
        got, want = out[k]
        assert got.dtype == p["x"].dtype and got.is_contiguous()
        if want.numel():
            std = (ye.var(-1, unbiased=False, keepdim=True) + EPS).sqrt() if k == "h" else 1.0
            tol = torch.finfo(got.dtype).eps / 2 * want.abs() + 256 * u * (ye.abs().amax(-1, keepdim=True) / std + 1)
            assert ((got.double() - want).abs() <= tol).all(), k
    back = torch.autograd.grad([out[k][0] for k in use], [p[k] for k in names], [ds[k] for k in use], allow_unused=True)
    want = torch.autograd.grad([out[k][1] for k in use], [ref[k] for k in names], [ds[k].double() for k in use], allow_unused=True)
    T, C = p["x"].shape
    for k, a, b in zip(names, back, want):
        if b is None:       # the next norm is not used
            assert k == "nxt" and (a is None or not a.any())
            continue
        assert a.dtype == p[k].dtype and a.shape == p[k].shape, k
        if not a.numel():
            continue
        step = torch.finfo(a.dtype).eps / 2
        if p[k].dim() == 2:
            tol = step * b.abs() + 1024 * u * (b.abs().amax(-1, keepdim=True) + 1)
        else:               # magnitudes of the terms: at most those of dy, dh times those of unit rows and x, some tens
            tol = step * b.abs() + (1024 + T) * u * T ** 0.5 * 16 + (1024 + T) * u * b.abs()
        assert ((a.double() - b).abs() <= tol).all(), (k, float(((a.double() - b).abs() - tol).max()))
    return back


# ------------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("gate,sigmoid", [("none", False), ("channel", False), ("token", False), ("token", True)])
@pytest.mark.parametrize("rms", [False, True])
def test_restatement(gate, sigmoid, rms):
    _check(_inputs(5, 24, F32, gate, True, True, "cpu"), sigmoid, rms)


@pytest.mark.parametrize("gate,sigmoid", [("none", False), ("channel", False), ("token", True)])
@pytest.mark.parametrize("rms", [False, True])
def test_64_bit_rows_are_computed_in_64_bits(gate, sigmoid, rms):
    """Outputs to the last bits (rows of 9 numbers: some 40 roundings of 2^-53 of numbers below 100), gradients against differences."""
    p = _inputs(4, 9, torch.float64, gate, True, True, "cpu")
    y, h = _call(p, sigmoid, rms)
    for got, want in zip((y, h), _formula(p["x"], p["f"], p["post"], p["nxt"], p["gate"], sigmoid, p["scale"], rms)):
        assert got.dtype == torch.float64 and ((got - want).abs() <= 40 * 2.0 ** -53 * 100).all()
    names = [k for k in p if p[k] is not None]
    assert torch.autograd.gradcheck(lambda *a: _call(p | dict(zip(names, a)), sigmoid, rms), [p[k] for k in names])


def test_refusals():
    p = _inputs(4, 8, F32, "token", True, True, "cpu")
    x = p["x"]
    for bad in (dict(x=x[0]), dict(f=x[:3]), dict(f=x.to(BF)), dict(gate=x[:, :1]), dict(gate=x.to(BF)), dict(post=x[0, :7]),
                dict(post=p["post"].to(F16)), dict(nxt=p["nxt"].to(BF), post=p["post"].to(BF)), dict(scale=torch.ones(16)[::2]),
                dict(gate=p["post"], sigmoid=True), dict(gate=None, sigmoid=True)):
        a = p | {"sigmoid": False} | bad
        with pytest.raises(ValueError):
            ops.sandwich_norm(a["x"], a["f"], a["post"], a["nxt"], gate=a["gate"], scale=a["scale"], sigmoid=a["sigmoid"])
    with pytest.raises(ValueError):
        K.sandwich_fwd(x, p["f"], None, None)       # no CPU tensors
    with pytest.raises(ValueError):
        K.sandwich_fwd(x.double(), p["f"].double(), None, None)
    with pytest.raises(ValueError):
        K.sandwich_bwd(None, None, x, x, torch.empty(4, 4), None, None)
    with pytest.raises(ValueError):
        K.sandwich_bwd(x, None, x, x, torch.empty(3, 4), None, None)


@pytest.mark.parametrize("tied", [("post", "nxt"), ("gate", "scale"), ("post", "nxt", "gate", "scale")])
def test_one_weight_in_several_places_has_one_running_sum(tied, monkeypatch):
    """Column sums of one kernel never go to the same memory: a parameter that is, say, post and next gets one of them added to its
    running gradient by the kernel, and the others behind it."""
    T, C, given = 6, 8, []

    def fwd(x, f, post, nxt, gate, scale, eps, rms, sigmoid, with_next, stats):
        y, h = _formula(x, f, post, nxt, gate, sigmoid, scale, rms)
        return y, h, torch.zeros(T, 4)

    def bwd(dy, dh, x, f, stats, post, nxt, gate, scale, rms, sigmoid, sums, add):
        given.append([s.data_ptr() for s in sums if s is not None])
        v = [t.detach().clone().requires_grad_(True) for t in (nxt, post, scale, gate)]
        with torch.enable_grad():
            out = _formula(x, f, v[1], v[0], v[3], sigmoid, v[2], rms)
            grads = torch.autograd.grad(out, v, (dy, dh))
        for s, a, g in zip(sums, add, grads):
            s.copy_(s + g if a else g)
        return torch.zeros_like(x), torch.zeros_like(f), None
    monkeypatch.setattr(K, "sandwich_fwd", fwd)
    monkeypatch.setattr(K, "sandwich_bwd", bwd)
    p = _inputs(T, C, F32, "channel", True, True, "cpu")
    dy, dh = torch.randn(T, C), torch.randn(T, C)
    call = lambda q: ops._SandwichFn.apply(q["x"], q["f"], q["post"], q["nxt"], q["gate"], q["scale"], EPS, False, False, True)
    for name in tied:
        p[name] = p[tied[0]]
    apart = {k: p[k].detach().clone().requires_grad_(True) for k in p}
    want = sum(torch.autograd.grad(call(apart), [apart[k] for k in tied], (dy, dh)))
    p[tied[0]].main_grad = torch.full((C,), 3.0)
    torch.autograd.backward(call(p), (dy, dh))
    assert len(set(given[-1])) == len(given[-1]) == 4 and p[tied[0]].grad is None
    assert torch.allclose(p[tied[0]].main_grad - 3.0, want, rtol=1e-5, atol=1e-5)


def test_sums_that_share_memory_are_refused():
    x, st, buf = torch.randn(4, 8), torch.empty(4, 4), torch.zeros(20)
    a, b = buf[:8], buf[8:16]
    with pytest.raises(ValueError, match="CUDA"):       # apart, and for the next check to refuse
        K.sandwich_bwd(x, None, x, x, st, None, None, sums=(a, b, None, buf[16:].view(BF)), add=(True, True, False, False))
    for sums in ((a, a, None, None), (None, a, None, buf[4:12]), (a, None, buf[7:15], None), (a, b, None, buf[:4].view(BF)[:8])):
        with pytest.raises(ValueError, match="share"):
            K.sandwich_bwd(x, None, x, x, st, None, None, sums=sums, add=(False,) * 4)
    for sums, add in (((a[:7], None, None, None), (False,) * 4), ((buf[::2][:8], None, None, None), (False,) * 4),
                      ((a.to(BF), None, None, None), (True, False, False, False))):
        with pytest.raises(ValueError):
            K.sandwich_bwd(x, None, x, x, st, None, None, sums=sums, add=add)


# ------------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("T,C", [(1, 1), (1, 8), (2, 3), (33, 7), (150, 16), (1, 24), (301, 17), (700, 32), (37, 66), (500, 100), (149, 128),
                                 (3, 250), (37, 256), (5, 264), (700, 512), (130, 768), (9, 1111), (1300, 1024),
                                 (33, 2048), (3, 3001), (5, 4096)])
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("gate,sigmoid,scaled", [("none", False, False), ("channel", False, True), ("token", False, False),
                                                 ("token", True, True)])
def test_outputs_and_gradients(T, C, dtype, gate, sigmoid, scaled, cuda_status):
    _check(_inputs(T, C, dtype, gate, scaled, True, "cuda"), sigmoid, rms=(T + C) % 2 == 0 or C == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("use", [("y",), ("h",), ("y", "h")])
def test_outputs_that_are_not_used(rms, use, cuda_status):
    _check(_inputs(50, 320, BF, "channel", True, True, "cuda"), False, rms, use)


@pytest.mark.gpu
def test_no_weights_and_fp32_weights(cuda_status):
    _check(_inputs(50, 320, BF, "none", False, False, "cuda"), False, False)
    _check(_inputs(50, 320, BF, "channel", True, True, "cuda", F32), False, False)
    _check(_inputs(50, 321, F16, "token", True, True, "cuda", F32), True, True)


@pytest.mark.gpu
def test_no_rows(cuda_status):
    back = _check(_inputs(0, 64, BF, "channel", True, True, "cuda"), False, False)
    assert all(not b.any() for b in back)


@pytest.mark.gpu
@pytest.mark.parametrize("C,shift", [(256, 0), (256, 1), (100, 0)])
def test_strides_and_addresses(C, shift, cuda_status):
    """Rows inside wider rows, at odd addresses, transposed, and gradients that share one row or are transposed."""
    T = 40
    p = _inputs(T, C, BF, "token", True, True, "cuda")
    wide = torch.randn(T, 2 * C + 24, device="cuda").to(BF)
    p["x"] = wide[:, shift:C + shift].detach().requires_grad_(True)
    p["f"] = torch.randn(C, T, device="cuda").to(BF).t().detach().requires_grad_(True)
    p["gate"] = wide[:, C + 16 + shift:2 * C + 16 + shift].detach().requires_grad_(True)
    _check(p, True, False)
    y, h = _call(p, True, False)
    dy, dh = torch.randn(C, device="cuda").to(BF).expand(T, C), torch.randn(C, T, device="cuda").to(BF).t()
    a = torch.autograd.grad((y, h), (p["x"], p["f"], p["gate"], p["post"]), (dy, dh), retain_graph=True)
    b = torch.autograd.grad((y, h), (p["x"], p["f"], p["gate"], p["post"]), (dy.contiguous(), dh.contiguous()))
    for s, t in zip(a, b):
        if shift == 0 and C % 8 == 0:
            assert torch.equal(s, t)
        else:
            assert torch.allclose(s.float(), t.float(), rtol=2 ** -7, atol=1e-5)


@pytest.mark.gpu
def test_the_same_bits_every_run_and_on_another_stream(cuda_status):
    p = _inputs(3000, 512, BF, "channel", True, True, "cuda")
    names = list(p)
    dy, dh = (torch.randn(3000, 512, device="cuda").to(BF) for _ in range(2))

    def run():
        y, h = _call(p, False, False)
        return (y, h) + torch.autograd.grad((y, h), [p[k] for k in names], (dy, dh))
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.gpu
def test_gradients_against_differences(cuda_status):
    """Directional derivatives of the 64-bit formula by central differences (step 1e-5: errors below 1e-8 here) against the
    kernel's fp32 gradients, whose sum over 4 000 products is good to some 2^-24 of the sum of their magnitudes a row."""
    p = _inputs(20, 200, F32, "token", True, True, "cuda")
    names = [k for k in p if p[k] is not None]
    y, h = _call(p, True, False)
    dy, dh = torch.randn_like(y), torch.randn_like(h)
    back = torch.autograd.grad((y, h), [p[k] for k in names], (dy, dh))
    for k, g in zip(names, back):
        d = torch.randn_like(p[k]).double()

        def value(t):
            q = {n: (v.detach().double() + (t * d if n == k else 0)) for n, v in p.items()}
            a, b = _formula(q["x"], q["f"], q["post"], q["nxt"], q["gate"], True, q["scale"], False)
            return ((a * dy).sum() + (b * dh).sum()).item()
        want = (value(1e-5) - value(-1e-5)) / 2e-5
        got = (g.double() * d).sum().item()
        assert abs(got - want) <= 1e-6 * (g.double() * d).abs().sum().item() + 1e-5, k


@pytest.mark.gpu
def test_running_gradients_are_added_to(cuda_status):
    p = _inputs(300, 256, BF, "channel", True, True, "cuda")
    names = ("post", "nxt", "gate", "scale")
    dy, dh = (torch.randn(300, 256, device="cuda").to(BF) for _ in range(2))
    plain = {}
    y, h = _call(p, False, False)
    for k, g in zip(names, torch.autograd.grad((y, h), [p[k] for k in names], (dy, dh))):
        plain[k] = g
    for k in names:
        p[k].main_grad = torch.full((256,), 3.0, device="cuda")
    torch.autograd.backward(_call(p, False, False), (dy, dh))
    for k in names:
        assert p[k].grad is None
        assert torch.allclose(p[k].main_grad - 3.0, plain[k].float(), rtol=2 ** -7, atol=1e-4), k


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [("post", "nxt"), ("gate", "scale")])
def test_running_gradient_of_a_weight_in_two_places(tied, cuda_status):
    """Every time the sum of the gradients of two weights apart. Both are sums of T terms in fp32 here (the kernel's partial sums, the
    same in either call), and what is compared are the roundings of three additions to numbers of at most 3 + both gradients."""
    T, C = 700, 512
    p = _inputs(T, C, F32, "channel", True, True, "cuda")
    p[tied[1]] = p[tied[0]]
    apart = {k: v.detach().clone().requires_grad_(True) for k, v in p.items()}
    dy, dh = torch.randn(T, C, device="cuda"), torch.randn(T, C, device="cuda")
    a, b = torch.autograd.grad(_call(apart, False, False), [apart[k] for k in tied], (dy, dh))
    main = p[tied[0]].main_grad = torch.empty(C, device="cuda")
    for _ in range(100):
        main.fill_(3.0)
        torch.autograd.backward(_call(p, False, False), (dy, dh))
        assert p[tied[0]].grad is None
        assert ((main - 3.0 - (a + b)).abs() <= 4 * 2.0 ** -24 * (3.0 + a.abs() + b.abs())).all()


@pytest.mark.gpu
def test_captured_passes_do_not_share_their_scratch(cuda_status):
    T, C = 900, 256
    sets = [[torch.randn(T, C, device="cuda").to(BF) for _ in range(4)] for _ in range(2)]
    w = torch.ones(C, device="cuda").to(BF)
    out, graphs = [], []

    def one(x, f, dy, dh):
        y, h, st = K.sandwich_fwd(x, f, w, w)
        s = [torch.empty(C, device="cuda") for _ in range(2)]
        return [y, h, *K.sandwich_bwd(dy, dh, x, f, st, w, w, sums=(*s, None, None))[:2], *s]
    want = [one(*s) for s in sets]
    torch.cuda.synchronize()
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.append(one(*s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, want):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,C,width,first", [
    (BF, 1001, 1005, 2), (F16, 1001, 1005, 1), (BF, 1001, 1004, 0), (BF, 1002, 1006, 2), (F16, 1002, 1007, 0), (BF, 129, 131, 4),
    (BF, 4095, 4097, 0), (F32, 1001, 1003, 1), (F32, 130, 133, 3), (F32, 17, 21, 1), (F32, 4001, 4003, 2), (BF, 6, 14, 2), (BF, 66, 70, 0)])
@pytest.mark.parametrize("gate,sigmoid", [("channel", False), ("token", True)])
def test_rows_beside_numbers_that_are_none(dtype, C, width, first, gate, sigmoid, cuda_status):
    """Rows of any width, stride and place in wider ones whose other channels are NaN: nothing of them shows in any result. Enough
    rows that blocks have several groups and groups several steps, an odd number of them."""
    T = 1501
    p = _inputs(T, C, dtype, gate, True, True, "cuda")
    for name in ("x", "f") + (("gate",) if gate == "token" else ()):
        around = torch.full((T + 2, width), float("nan"), device="cuda", dtype=dtype)
        rows = around.view(-1)[first:first + T * width].view(T, width)[:, :C]
        p[name] = rows.copy_(p[name].detach()).requires_grad_(True)
    _check(p, sigmoid, rms=C % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [256, 40, 33])
def test_rows_past_32_bit_offsets(C, cuda_status):
    """Rows 2^30 elements apart in one buffer, outputs and gradients against those of the same rows put together."""
    big = torch.zeros(3 * 2 ** 30 + C, dtype=BF, device="cuda")
    far = big.as_strided((4, C), (2 ** 30, 1))
    far.copy_(torch.randn(4, C))
    near = far.contiguous()
    f, dy = torch.randn(4, C, device="cuda").to(BF), torch.randn(4, C, device="cuda").to(BF)
    a = K.sandwich_fwd(far, f, None, None, gate=far, sigmoid=True)
    b = K.sandwich_fwd(near, f, None, None, gate=near, sigmoid=True)
    x = K.sandwich_bwd(far, dy, far, f, a[2], None, None, gate=far, sigmoid=True)
    y = K.sandwich_bwd(near, dy, near, f, b[2], None, None, gate=near, sigmoid=True)
    for s, t in zip(a + x, b + y):
        assert torch.allclose(s.float(), t.float(), rtol=2 ** -7, atol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,C,apart", [(BF, 1001, 2 ** 30 + 1), (F16, 1002, 2 ** 30 + 6), (F32, 131, 2 ** 29 + 3)])
def test_rows_by_words_past_32_bit_offsets(dtype, C, apart, cuda_status):
    """Rows that lie between words or 16 bytes, far from one another: the results of the same rows put together."""
    big = torch.zeros(3 * apart + C, dtype=dtype, device="cuda")
    far = big.as_strided((4, C), (apart, 1))
    far.copy_(torch.randn(4, C))
    near = far.contiguous()
    f, dy = torch.randn(4, C, device="cuda").to(dtype), torch.randn(4, C, device="cuda").to(dtype)
    a = K.sandwich_fwd(far, f, None, None, gate=far, sigmoid=True)
    b = K.sandwich_fwd(near, f, None, None, gate=near, sigmoid=True)
    x = K.sandwich_bwd(dy, far, far, f, a[2], None, None, gate=far, sigmoid=True)
    y = K.sandwich_bwd(dy, near, near, f, b[2], None, None, gate=near, sigmoid=True)
    for s, t in zip(a + x, b + y):
        assert torch.equal(s, t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,C", [(BF, 17), (F32, 17), (F16, 40), (BF, 100), (F32, 100), (BF, 256), (F32, 264), (BF, 1001), (F16, 1002),
                                     (F32, 1111), (BF, 2048)])
@pytest.mark.parametrize("rms", [False, True])
def test_infinities_and_nan_stay_in_their_rows(dtype, C, rms, cuda_status):
    """Rows with numbers that are none or infinite come out where the formula has such numbers, and all other rows have the bits of a call
    without them, forward and backward; an infinite gate behind a sigmoid is zero or one."""
    T, inf, nan = 333, float("inf"), float("nan")
    p = _inputs(T, C, dtype, "token", True, True, "cuda")
    clean = {k: v.detach().clone().requires_grad_(True) for k, v in p.items()}
    at = {3: ("f", inf), 4: ("f", nan), 50: ("x", inf), 51: ("x", nan), 100: ("gate", nan), 101: ("f", -inf), 331: ("x", -inf), 332: ("f", nan),
          0: ("f", nan), 150: ("gate", inf), 151: ("gate", -inf)}
    with torch.no_grad():
        for row, (name, value) in at.items():
            p[name][row, (7 * row) % C] = value
    dy, dh = (torch.randn(T, C, device="cuda").to(dtype) for _ in range(2))
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[list(at)] = False

    def run(q):
        out = _call(q, True, rms)
        return out + torch.autograd.grad(out, [q[k] for k in ("x", "f", "gate")], (dy, dh))
    got = run(p)
    assert all(torch.equal(a[rest], b[rest]) for a, b in zip(got, run(clean)))
    d = {k: v.detach().double() for k, v in p.items()}
    want = _formula(d["x"], d["f"], d["post"], d["nxt"], d["gate"], True, d["scale"], rms)
    for a, b in zip(got, want):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf())
    for row in (150, 151):
        assert all(a[row].isfinite().all() for a in got)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [100, 256, 264, 1111])
def test_gates_far_from_zero(C, cuda_status):
    """fp32 rows of ones and minus ones, whose norm is 1 / sqrt(1 + eps) and whose block input is zero: y is the sigmoid alone, and the
    gate's gradient its slope. Rounded, in units of 2^-24: the mean of the squares (a sum of equal terms) log2 C + 8, its reciprocal
    root 4, the exponential 4, its sum with one 1, the division 1, the products of y 2 and of the gradient 4: below 32 units of either."""
    T = 64
    f = torch.where(torch.rand(T, C, device="cuda") < 0.5, -1.0, 1.0)
    gate = (170 * torch.rand(T, C, device="cuda") - 85).requires_grad_(True)
    y, _ = ops.sandwich_norm(torch.zeros_like(f), f, gate=gate, sigmoid=True, eps=EPS, rms=True, with_next=False)
    dg, = torch.autograd.grad(y, gate, torch.ones_like(y))
    n, v = f.double() / (1 + EPS) ** 0.5, gate.detach().double()
    for got, want in ((y, n * torch.sigmoid(v)), (dg, n * torch.sigmoid(v) * torch.sigmoid(-v))):
        assert ((got.double() - want).abs() <= 32 * 2.0 ** -24 * want.abs()).all(), float(((got.double() - want) / want).abs().max())
    for v, at in ((-float("inf"), 0.0), (float("inf"), 1.0), (-200.0, 0.0), (200.0, 1.0)):
        gate = torch.full((T, C), v, device="cuda", requires_grad=True)
        y, _ = ops.sandwich_norm(torch.zeros_like(f), f, gate=gate, sigmoid=True, eps=EPS, rms=True, with_next=False)
        dg, = torch.autograd.grad(y, gate, torch.ones_like(y))
        assert (y.abs() <= at).all() and (y.abs() >= at * 0.9999).all() and not dg.any()


@pytest.mark.gpu
def test_rows_without_variance_and_large_means(cuda_status):
    """Constant rows are zeros behind a LayerNorm, and a mean a thousand times the deviation costs no more than the cast did."""
    T, C = 6, 384
    x, f = torch.randn(T, C, device="cuda"), torch.randn(T, C, device="cuda")
    f[0] = 3.0
    f[1] = 0.0
    f[2] += 1000.0
    y, h = ops.sandwich_norm(x, f)
    assert torch.equal(y[:2], x[:2])
    ye, he = _formula(x.double(), f.double(), None, None, None, False, None, False)
    # the mean of the third row is known to 2^-24 of 1000, in units of its deviation 1
    assert (y.double() - ye).abs().max() <= 16 * 1000 * 2.0 ** -24 and (h.double() - he).abs().max() <= 16 * 1000 * 2.0 ** -24
