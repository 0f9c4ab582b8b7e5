"""Thin tensor-level wrappers over the C ABI of the sm_100a kernels (no autograd here).

Every function takes CUDA tensors, checks shapes / dtypes / contiguity, launches on the current
stream and returns output tensors. ``nanoplm_b200.ops.functional`` builds differentiable ops on top.
"""
from __future__ import annotations

from contextlib import nullcontext
from ctypes import c_float, c_int, c_longlong
from functools import lru_cache
from struct import Struct

import torch

from . import _lib
from ._lib import check_rc, count_launch, lib, ptr, raw_stream, status_word, stream_ptr, typed

EPI_STORE, EPI_ADD, EPI_ATOMIC_F32, EPI_GELU, EPI_STORE_F32, EPI_SWIGLU, EPI_ROPE, EPI_RELU = 0, 1, 2, 3, 4, 5, 6, 7
# acc = dL/dh of h = silu(gate) * value; aux = the [value | gate] pre-activations (2N wide);
# out = their gradient (2N wide)
EPI_SWIGLU_BWD, EPI_STORE_DELTA = 8, 9

_BF16 = torch.bfloat16


def _chk(t: torch.Tensor, dtype, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")


def _dp(t: torch.Tensor | None):
    """Device address for a `typed` call; None is the null pointer."""
    return None if t is None else t.data_ptr()


def _address(t: torch.Tensor | None) -> int:
    """Device address for a packed call; 0 for None."""
    return 0 if t is None else t.data_ptr()


def _like(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and uninitialised, of t's shape, type and device (a third of the time of torch.empty with those)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _is_tracing() -> bool:
    return torch._C._is_tracing()


ROW_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_NULL = nullcontext()


def _device_of(first: torch.Tensor, *rest):
    """A context in which the first tensor's device is the current one; ValueError where another tensor is elsewhere."""
    if not first.is_cuda:
        raise ValueError("the tensors must be on a CUDA device")
    index = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != index:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")
    return _NULL if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def _rowmajor(t: torch.Tensor, name: str) -> int:
    """Returns the row stride of a 2-D tensor whose last dim is contiguous."""
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be 2-D with a contiguous last dim")
    return t.stride(0)


# --------------------------------------------------------------------------- GEMM
import os as _os

_GEMM_PAIR_DEFAULT = [{"1": True, "0": False}.get(_os.environ.get("NPLM_GEMM_PAIR", ""))]


def set_gemm_pair_default(enabled: bool | None) -> None:
    """Default of gemm(pair=None): run qualifying GEMMs on CTA pairs (cta_group::2). True / False: all / none; None (the
    initial value): those with bf16 outputs for which `pair_pays`. The fp32 weight gradients run at the same rate
    either way (384 / 377 us for 4096 x 1024 over 55 424 tokens) and stay on single CTAs."""
    _GEMM_PAIR_DEFAULT[0] = None if enabled is None else bool(enabled)


def pair_pays(M: int, N: int, K: int, epi: int) -> bool:
    """Whether a bf16-output GEMM on 256-wide tiles runs on CTA pairs by default: the rule of `gemm_pair_pays` in
    csrc/entry_points.h, which states the measurements on both sides of its lines."""
    tiles = (M + 127) // 128 * ((N + 255) // 256)
    if epi in (EPI_SWIGLU_BWD, EPI_STORE_DELTA):
        return True
    if epi == EPI_ROPE:
        return tiles > 740 if K >= 1024 else K >= 768 and tiles > 2600
    return tiles > 148 if K >= 768 else tiles * K > (190000 if epi == EPI_SWIGLU else 400000)


def tile_width(M: int, N: int, epi: int) -> int:
    """Default tile width of a GEMM: the rule of `gemm_tile_width` in csrc/entry_points.h, which states the measurements on
    both sides of its lines."""
    if epi in (EPI_SWIGLU_BWD, EPI_STORE_DELTA, EPI_ATOMIC_F32, EPI_STORE_F32):
        return 256 if N >= 256 or epi in (EPI_SWIGLU_BWD, EPI_STORE_DELTA) else 128
    rows = (M + 127) // 128
    if epi != EPI_SWIGLU and rows * ((N + 63) // 64) <= 148:
        return 64
    return 128 if (N < 256 and epi != EPI_SWIGLU) or rows * ((N + 127) // 128) <= 148 else 256


def gemm(a: torch.Tensor, b: torch.Tensor, *, a_mn: bool = False, b_mn: bool = False,
         epi: int = EPI_STORE, out: torch.Tensor | None = None, aux: torch.Tensor | None = None,
         splits: int = 1, bn: int | None = None, max_ctas: int = 0,
         direct_epilogue: bool = False, rope: tuple | None = None, pair: bool | None = None) -> torch.Tensor:
    """C[M,N] (+)= op(A) op(B)^T on tcgen05 tensor cores.

    a: [M,K] (a_mn=False) or [K,M] (a_mn=True); b: [N,K] (b_mn=False) or [K,N] (b_mn=True).
    epi: EPI_STORE / EPI_ADD (aux = residual) / EPI_ATOMIC_F32 (out fp32, accumulated in place) /
    EPI_GELU / EPI_RELU (aux = optional pre-activation output) / EPI_STORE_F32 / EPI_SWIGLU (out is N/2 wide,
    aux = optional [M,N] pre-activation output). bf16 outputs leave through shared memory and
    TMA stores; direct_epilogue=True selects per-thread global stores instead.
    EPI_ROPE: rope = (pos int32 [M], cos fp32 [P,32], sin fp32 [P,32], rope_cols): rotary embedding
    (head_dim 64) on every 64-wide head that starts below column rope_cols.
    pair: run on CTA pairs (tcgen05 cta_group::2, two SMs per 256 x 256 tile). None = the package
    default (`set_gemm_pair_default`); only 256-wide tiles without max_ctas qualify.
    """
    _chk(a, _BF16, "a")
    _chk(b, _BF16, "b")
    ag = getattr(b, "_ag", None)
    if ag is not None and ag.stale:
        # a row-sharded weight whose other row blocks are out of date (parameter-sharded data
        # parallelism): the first forward GEMM of the step gathers them from the peers inside the
        # kernel; any other consumer triggers an explicit gather
        if (not a_mn and not b_mn and splits == 1 and max_ctas == 0 and not direct_epilogue
                and epi in (EPI_STORE, EPI_ADD, EPI_GELU, EPI_RELU, EPI_SWIGLU, EPI_ROPE)):
            res = gemm_ag(a, b, ag.ptrs, ag.rank, ag.world, ag.flags, epi=epi, out=out, aux=aux, rope=rope)
            ag.stale = False
            return res
        ag.gather_now(b)
    lda, ldb = _rowmajor(a, "a"), _rowmajor(b, "b")
    if a_mn:
        K, M = a.shape
    else:
        M, K = a.shape
    if b_mn:
        Kb, N = b.shape
    else:
        N, Kb = b.shape
    if K != Kb:
        raise ValueError(f"inner dims differ: {K} vs {Kb}")
    out_cols = N // 2 if epi == EPI_SWIGLU else (2 * N if epi == EPI_SWIGLU_BWD else N)
    f32_out = epi in (EPI_ATOMIC_F32, EPI_STORE_F32)
    if out is None:
        if epi == EPI_ATOMIC_F32:
            raise ValueError("EPI_ATOMIC_F32 needs an fp32 accumulator passed as out")
        out = torch.empty((M, out_cols), dtype=torch.float32 if f32_out else _BF16, device=a.device)
    _chk(out, torch.float32 if f32_out else _BF16, "out")
    if tuple(out.shape) != (M, out_cols):
        raise ValueError(f"out has shape {tuple(out.shape)}, expected {(M, out_cols)}")
    ldc = _rowmajor(out, "out")
    ldr = 0
    if aux is not None:
        _chk(aux, _BF16, "aux")
        ldr = _rowmajor(aux, "aux")
        aux_cols = 2 * N if epi == EPI_SWIGLU_BWD else N
        if tuple(aux.shape) != (M, aux_cols):
            raise ValueError(f"aux has shape {tuple(aux.shape)}, expected {(M, aux_cols)}")
    elif epi == EPI_ADD:
        raise ValueError("EPI_ADD needs the residual passed as aux")
    elif epi == EPI_SWIGLU_BWD:
        raise ValueError("EPI_SWIGLU_BWD needs the pre-activations passed as aux")
    if bn is None:
        if pair is None and _GEMM_PAIR_DEFAULT[0] is None and max_ctas == 0 and not direct_epilogue and not a_mn:
            bn = tile_width(M, N, epi)
        else:
            bn = 256 if (N >= 256 or epi in (EPI_SWIGLU, EPI_SWIGLU_BWD)) else 128
    r_pos = r_cos = r_sin = None
    r_cols = 0
    if epi == EPI_ROPE:
        if rope is None:
            raise ValueError("EPI_ROPE needs rope=(pos, cos, sin, rope_cols)")
        r_pos, r_cos, r_sin, r_cols = rope
        _chk(r_pos, torch.int32, "rope pos")
        _chk(r_cos, torch.float32, "rope cos")
        if r_pos.numel() != M or r_cos.shape[-1] != 32:
            raise ValueError("rope tables must be [P, 32] and pos must have one entry per row")
    if pair is None:
        pair = _GEMM_PAIR_DEFAULT[0]
        if pair is None:
            pair = not f32_out and bn == 256 and pair_pays(M, N, K, epi)
    aux_p = aux.data_ptr() if aux is not None else None
    rope_p = (r_pos.data_ptr(), r_cos.data_ptr(), r_sin.data_ptr()) if r_pos is not None else (None, None, None)
    if pair and bn == 256 and max_ctas == 0 and not (a_mn and not b_mn):
        rc = typed("gemm_tcgen05", "nplm_gemm_bf16_pair", "pppp" + "i" * 12 + "pppipp")(
            a.data_ptr(), b.data_ptr(), out.data_ptr(), aux_p, M, N, K, lda, ldb, ldc, ldr, a_mn, b_mn, epi, splits,
            direct_epilogue, *rope_p, r_cols, status_word(a.device).data_ptr(), raw_stream())
        check_rc(rc, "gemm_bf16_pair")
        count_launch()
        return out
    rc = typed("gemm_tcgen05", "nplm_gemm_bf16", "pppp" + "i" * 14 + "pppipp")(
        a.data_ptr(), b.data_ptr(), out.data_ptr(), aux_p, M, N, K, lda, ldb, ldc, ldr, a_mn, b_mn, epi, splits, bn,
        max_ctas, direct_epilogue, *rope_p, r_cols, status_word(a.device).data_ptr(), raw_stream())
    check_rc(rc, "gemm_bf16")
    count_launch()
    return out


def gemm_ag(a: torch.Tensor, b_full: torch.Tensor, b_ptrs, rank: int, world: int, flags: torch.Tensor, *,
            epi: int = EPI_STORE, out: torch.Tensor | None = None, aux: torch.Tensor | None = None,
            bn: int | None = None, rope: tuple | None = None) -> torch.Tensor:
    """All-gather fused into the GEMM: C = A B^T with B [N,K] row-sharded over `world` ranks.

    b_full is this rank's full-size weight buffer in peer-mapped (symmetric) memory, of which only
    rows [rank*N/world, (rank+1)*N/world) are valid on entry; b_ptrs is the ctypes array of all ranks'
    buffer addresses. The kernel pulls the other shards over NVLink while the tensor cores work on
    the local shard's tiles; afterwards b_full holds the whole matrix. flags: uint32/int32 [8].
    The caller orders the call after the peers' shard writes and before their next update.
    """
    _chk(a, _BF16, "a")
    _chk(b_full, _BF16, "b")
    M, K = a.shape
    N, Kb = b_full.shape
    if K != Kb:
        raise ValueError(f"inner dims differ: {K} vs {Kb}")
    if N % world:
        raise ValueError("rows of B must divide evenly over the ranks")
    rows = N // world
    unit = rows * 2 if epi == EPI_SWIGLU else rows     # a SwiGLU tile reads bn / 2 value rows and bn / 2 gate rows
    if bn is None:
        bn = 256 if unit % 256 == 0 else 128
    if unit % bn:
        raise ValueError(f"shard height {rows} does not hold whole {bn}-wide tiles")
    if epi == EPI_SWIGLU and (world % 2 or (N // 2) % rows):
        raise ValueError("SwiGLU with a row-sharded weight needs an even number of ranks")
    if out is None:
        out = torch.empty((M, N // 2 if epi == EPI_SWIGLU else N), dtype=_BF16, device=a.device)
    ldr = 0
    if aux is not None:
        ldr = _rowmajor(aux, "aux")
    r_pos, r_cos, r_sin, r_cols = rope if rope is not None else (None, None, None, 0)
    if epi == EPI_ROPE and rope is None:
        raise ValueError("EPI_ROPE needs rope=(pos, cos, sin, rope_cols)")
    rc = lib("gemm_tcgen05").nplm_gemm_bf16_ag_rope(
        ptr(a), b_ptrs, ptr(out), ptr(aux), c_int(M), c_int(N), c_int(K), c_int(_rowmajor(a, "a")),
        c_int(_rowmajor(b_full, "b")), c_int(_rowmajor(out, "out")), c_int(ldr), c_int(epi), c_int(bn),
        c_int(rank), c_int(world), ptr(flags), ptr(r_pos), ptr(r_cos), ptr(r_sin), c_int(r_cols),
        ptr(status_word(a.device)), stream_ptr())
    check_rc(rc, "gemm_bf16_ag")
    count_launch()
    return out


def gemm_stack(a: torch.Tensor, b: torch.Tensor, *, b_mn: bool = False, alpha: float = 1.0, r: torch.Tensor | None = None,
               beta: float = 0.0, symmetric: bool = False) -> torch.Tensor:
    """alpha a_i op(b_i) + beta r_i for stacks a [B, m, k], b [B, n, k] (or [B, k, n] with b_mn), r [B, m, n], all bf16
    and contiguous, with one rounding; m a multiple of 256, k and n of 64. symmetric: the results are symmetric (and
    square), and only the tiles on and below the diagonal are computed."""
    B, m, k = a.shape
    n = b.shape[2] if b_mn else b.shape[1]
    if tuple(b.shape) != ((B, k, n) if b_mn else (B, n, k)) or (r is not None and tuple(r.shape) != (B, m, n)):
        raise ValueError(f"shapes do not match: {tuple(a.shape)}, {tuple(b.shape)}, {None if r is None else tuple(r.shape)}")
    for t, name in ((a, "a"), (b, "b"), (r, "r")):
        if t is not None:
            _chk(t, _BF16, name)
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
    out = torch.empty((B, m, n), dtype=_BF16, device=a.device)
    rc = typed("gemm_tcgen05", "nplm_gemm_bf16_stack", "pppp" + "i" * 9 + "ffipp")(
        a.data_ptr(), b.data_ptr(), out.data_ptr(), _dp(r), B, m, n, k, k, b.shape[2], n, n, b_mn, alpha, beta, symmetric,
        status_word(a.device).data_ptr(), raw_stream())
    check_rc(rc, "gemm_bf16_stack")
    count_launch()
    return out


def wgrad_splits(n_out: int, k_in: int, tokens: int, bn: int = 256, sms: int = 148) -> int:
    """Split-K factor for a weight-gradient GEMM [n_out, k_in] reduced over `tokens`.

    A work item of kb 64-token blocks costs kb + 25 block times (pipeline fill, epilogue, and what its additions take from
    the others); the factor with the least waves * cost wins. Graph-timed us, unsplit / this rule's factor: 55 424 tokens, 3072
    x 1024 (96 tiles) 286 / 239 in 3, 1024 x 1024 (32 tiles) 279 / 88 in 4, 4096 x 1024 (128 tiles) 324 unsplit, 332
    in 2; 17 024 tokens, 512 x 512 (8 tiles) 81 / 13.1 in 16, 64 x 768 80 / 11.1 in 16; 1 000 tokens, 1024 x 1024 11.9 / 8.6 in
    4. Of ten outputs at five token counts (1 000 to 55 424) it picks the best factor of 1 to 16 or one within 2 %, but
    for 3072 x 1024 at 4 352 tokens (28.2 unsplit, 25.1 in 3)."""
    tiles = ((n_out + 127) // 128) * ((k_in + bn - 1) // bn)
    kb = (tokens + 63) // 64
    best, best_cost = 1, None
    for s in range(1, 17):
        if s > 1 and kb // s < 4:
            break
        cost = -(-tiles * s // sms) * (-(-kb // s) + 25)
        if best_cost is None or cost < 0.98 * best_cost:
            best, best_cost = s, cost
    return best


_default_splits = lru_cache(maxsize=1024)(wgrad_splits)


def weight_grad_splits(n_out: int, k_in: int, tokens: int) -> int:
    """Split factor of a weight gradient in a backward pass: `wgrad_splits`, and 1 under
    `set_attention_deterministic` (several work items add to a tile in any order, one gives the same bits every run)."""
    return 1 if _FA_DETERMINISTIC[0] else _default_splits(n_out, k_in, tokens)


# --------------------------------------------------------------------------- norms
def norm_fwd(x: torch.Tensor, w: torch.Tensor | None, eps: float, rms: bool = False,
             ids: torch.Tensor | None = None, stats: bool = True):
    """LayerNorm (no bias) / RMSNorm over the last dim. With ids, rows are table[ids] (embedding).

    Returns (y, mean, rstd); mean is None for RMSNorm, both are with stats=False (no backward pass to come).
    """
    _chk(x, _BF16, "x")
    C = x.shape[-1]
    if ids is not None:
        _chk(ids, torch.int32, "ids")
        T = ids.numel()
    else:
        T = x.numel() // C
    x2 = x.reshape(-1, C)
    if not x2.is_contiguous():
        x2 = x2.contiguous()
    y = torch.empty((T, C), dtype=_BF16, device=x.device)
    mean = None if rms or not stats else torch.empty(T, dtype=torch.float32, device=x.device)
    rstd = torch.empty(T, dtype=torch.float32, device=x.device) if stats else None
    rc = typed("elementwise", "nplm_norm_fwd", "ppppppiifip")(
        x2.data_ptr(), _dp(ids), _dp(w), y.data_ptr(), _dp(mean), _dp(rstd), T, C, eps, rms, raw_stream())
    check_rc(rc, "norm_fwd")
    count_launch()
    return y, mean, rstd


def norm_bwd(dy, x, w, mean, rstd, *, rms=False, dres=None, dw=None, ids=None, dtable=None):
    """Backward of norm_fwd. dw (fp32 [C]) and dtable (fp32 [V,C]) are accumulated in place.

    Returns dx (None in embedding mode)."""
    C = dy.shape[-1]
    T = dy.numel() // C
    dy2 = dy.reshape(T, C)
    if not dy2.is_contiguous():
        dy2 = dy2.contiguous()
    dx = None if ids is not None else torch.empty((T, C), dtype=_BF16, device=dy.device)
    V = x.shape[0] if ids is not None else 0
    if ids is not None and dtable is not None and V <= 200:
        scratch = torch.empty(V * (C + 1), dtype=torch.float32, device=dy.device)
        rc = typed("elementwise", "nplm_embed_bwd", "ppppppppp" + "iiiip")(
            dy2.data_ptr(), x.data_ptr(), ids.data_ptr(), _dp(w), _dp(mean), rstd.data_ptr(), _dp(dw), dtable.data_ptr(),
            scratch.data_ptr(), T, C, V, rms, raw_stream())
        check_rc(rc, "embed_bwd")
        count_launch(2)
        return None
    rc = typed("elementwise", "nplm_norm_bwd", "pppppppppp" + "iiiip")(
        dy2.data_ptr(), x.data_ptr(), _dp(ids), _dp(w), _dp(mean), _dp(rstd), _dp(dres), _dp(dx), _dp(dw),
        _dp(dtable), T, C, V, rms, raw_stream())
    check_rc(rc, "norm_bwd")
    count_launch()
    return dx


GATE_NONE, GATE_CHANNEL, GATE_TOKEN, GATE_SIGMOID = 0, 1, 2, 3
SANDWICH_MAX_C = 4096
_SANDWICH = Struct("=15q4q6q9if")       # SandwichCall of csrc/sandwich_norm.cu


def check_sandwich(x, f, gate, post, nxt, scale, sigmoid) -> tuple[int, bool]:
    """Checks the arguments of a sandwich norm; (gate mode, whether the [C] weights are fp32 beside other rows)."""
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be [T, C], got {tuple(x.shape)}")
    C = x.shape[1]
    if f.shape != x.shape or f.dtype != x.dtype:
        raise ValueError(f"f must be {tuple(x.shape)} {x.dtype}, got {tuple(f.shape)} {f.dtype}")
    mode = GATE_NONE
    vectors = [("post", post), ("next", nxt), ("scale", scale)]
    if gate is not None and gate.dim() == 1:
        if sigmoid:
            raise ValueError("a gate per channel is a weight: sigmoid is for gates of tokens")
        mode = GATE_CHANNEL
        vectors.append(("gate", gate))
    elif gate is not None:
        if gate.shape != x.shape or gate.dtype != x.dtype:
            raise ValueError(f"gate must be [{C}] or {tuple(x.shape)} {x.dtype}, got {tuple(gate.shape)} {gate.dtype}")
        mode = GATE_SIGMOID if sigmoid else GATE_TOKEN
    kinds = set()
    for name, v in vectors:
        if v is not None:
            if tuple(v.shape) != (C,) or not v.is_contiguous():
                raise ValueError(f"{name} must be a contiguous [{C}], got {tuple(v.shape)}")
            kinds.add(v.dtype)
    if len(kinds) > 1 or not kinds <= {x.dtype, torch.float32}:
        raise ValueError(f"the [C] weights must all be {x.dtype} or all fp32, got {sorted(map(str, kinds))}")
    return mode, bool(kinds) and kinds != {x.dtype}


def _sandwich_rows(x, *rows):
    if x.dtype not in ROW_TYPES or x.shape[1] > SANDWICH_MAX_C:
        raise ValueError(f"x must be bf16, fp16 or fp32 with up to {SANDWICH_MAX_C} channels, got {x.dtype} {tuple(x.shape)}")
    for t in (x, *rows):
        if t is not None and t.dim() == 2 and t.stride(1) != 1 and t.shape[1] > 1 and t.numel():
            raise ValueError("rows must have a contiguous last dim")


def sandwich_fwd(x, f, post, nxt, gate=None, scale=None, eps: float = 1e-5, rms: bool = False, sigmoid: bool = False,
                 with_next: bool = True, stats: bool = True):
    """y = scale x + g norm(f) post, h = norm(y) nxt for rows of up to 4 096 channels: (y, h, stats), h None without
    `with_next`. gate: None, [C], or like x (with `sigmoid` through one). post, nxt, scale: [C] or None, all of x's type
    or all fp32. stats: fp32 [T, 4] for `sandwich_bwd`."""
    mode, param32 = check_sandwich(x, f, gate, post, nxt, scale, sigmoid)
    _sandwich_rows(x, f, gate)
    T, C = x.shape
    with _device_of(x, f, gate, post, nxt, scale):
        y = _like(x)
        h = _like(x) if with_next else None
        st = x.new_empty((T, 4), dtype=torch.float32) if stats else None
        if T:
            call = _SANDWICH.pack(x.data_ptr(), f.data_ptr(), _address(gate), _address(post), _address(nxt), _address(scale), 0, 0,
                                  y.data_ptr(), _address(h), 0, 0, 0, _address(st), 0, 0, 0, 0, 0, x.stride(0), f.stride(0),
                                  gate.stride(0) if mode >= GATE_TOKEN else 0, 0, 0, T, 0, 0, 0, 0, C, rms, mode,
                                  ROW_TYPES[x.dtype], param32, eps)
            check_rc(typed("sandwich_norm", "nplm_sandwich_fwd", "pp")(call, raw_stream()), "sandwich_fwd")
            count_launch()
    return y, h, st


_SUM_KINDS = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}


def _sum_kinds(sums, add, C: int) -> list[int]:
    """Checks where column sums go; what each is there (`ColumnSums` of csrc/sandwich_norm.cu). A block of the kernel reads and writes
    each of them, so no two may share memory."""
    kinds, spans = [], []
    for s, a in zip(sums, add):
        if s is None:
            kinds.append(0)
            continue
        if s.numel() != C or not s.is_contiguous() or s.dtype not in _SUM_KINDS or (a and s.dtype != torch.float32):
            raise ValueError(f"sums must be contiguous [{C}] tensors, fp32 where added to")
        kinds.append(4 if a else _SUM_KINDS[s.dtype])
        at = s.data_ptr()
        spans.append((at, at + C * s.element_size()))
    spans.sort()
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError("sums share memory")
    return kinds


def sandwich_bwd(dy, dh, x, f, stats, post, nxt, gate=None, scale=None, rms: bool = False, sigmoid: bool = False,
                 sums=(None, None, None, None), add=(False, False, False, False)):
    """Gradients of `sandwich_fwd` from dy and dh (one of them may be None): (dx, df, dgate of a gate of tokens or None).
    sums: [C] tensors for the gradients of nxt, post, scale and a gate per channel, None where unwanted; written, or
    with `add` (fp32 only) added to. No two of them may share memory."""
    mode, param32 = check_sandwich(x, f, gate, post, nxt, scale, sigmoid)
    _sandwich_rows(x, f, gate, dy, dh)
    (T, C), kind = x.shape, ROW_TYPES[x.dtype]
    if dy is None and dh is None:
        raise ValueError("dy or dh is needed")
    for name, d in (("dy", dy), ("dh", dh)):
        if d is not None and (d.shape != x.shape or d.dtype != x.dtype):
            raise ValueError(f"{name} must be {tuple(x.shape)} {x.dtype}, got {tuple(d.shape)} {d.dtype}")
    if stats.dtype != torch.float32 or tuple(stats.shape) != (T, 4) or not stats.is_contiguous():
        raise ValueError(f"stats must be the fp32 [{T}, 4] of the forward pass")
    kinds = _sum_kinds(sums, add, C)
    with _device_of(x, f, gate, post, nxt, scale, dy, dh, stats, *sums):
        dx, df = _like(x), _like(x)
        dg = _like(x) if mode >= GATE_TOKEN else None
        partial = None
        if any(kinds) and T:
            blocks = typed("sandwich_norm", "nplm_sandwich_bwd_blocks", "li")(T, C)
            partial = x.new_empty((4, blocks, C), dtype=torch.float32)
        rs = lambda t: 0 if t is None else t.stride(0)
        call = _SANDWICH.pack(x.data_ptr(), f.data_ptr(), _address(gate), _address(post), _address(nxt), _address(scale),
                              _address(dy), _address(dh), 0, 0, dx.data_ptr(), df.data_ptr(), _address(dg), stats.data_ptr(),
                              _address(partial), *map(_address, sums), x.stride(0), f.stride(0),
                              gate.stride(0) if mode >= GATE_TOKEN else 0, rs(dy), rs(dh), T, *kinds, C, rms, mode, kind, param32,
                              0.0)
        rc = typed("sandwich_norm", "nplm_sandwich_bwd", "pp")(call, raw_stream())
        check_rc(rc, "sandwich_bwd")
        count_launch((T > 0) + any(kinds))
    return dx, df, dg


# --------------------------------------------------------------------------- rope / swiglu / act
def rope_(qkv: torch.Tensor, pos: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, H: int,
          D: int, backward: bool = False) -> torch.Tensor:
    """In-place rotary embedding on the q and k parts of qkv [T, 3*H*D]."""
    _chk(qkv, _BF16, "qkv")
    _chk(pos, torch.int32, "pos")
    T = qkv.shape[0]
    rc = lib("elementwise").nplm_rope(ptr(qkv), ptr(pos), ptr(cos), ptr(sin), c_int(T), c_int(H),
                                      c_int(D), c_int(int(backward)), stream_ptr())
    check_rc(rc, "rope")
    count_launch()
    return qkv


ROTARY_MAX_WIDTH = 512
_ROTARY = Struct("=4q12q3q3q8if4x")       # RotaryCall of csrc/rotary.cu


def check_rotary(q, k, positions, frequencies):
    """Checks the arguments of a rotation: (batch, tokens, heads, width, heads of k, number of channels that rotate), strides of the
    batch, tokens and heads of q, of k, and of the batch and tokens of the positions."""
    shape, st = q.shape, q.stride()
    if len(shape) == 3:
        (S, H, D), B, qs = shape, 1, (0, st[0], st[1])
    elif len(shape) == 4:
        (B, S, H, D), qs = shape, st[:3]
    else:
        raise ValueError(f"q must be [tokens, heads, width] or [batch, tokens, heads, width], got {tuple(shape)}")
    Hk, ks = 0, (0, 0, 0)
    if k is not None:
        kshape, kst = k.shape, k.stride()
        if len(kshape) != len(shape) or kshape[:-2] != shape[:-2] or kshape[-1] != D:
            raise ValueError(f"q {tuple(shape)} and k {tuple(kshape)} differ in tokens or width")
        if k.dtype != q.dtype:
            raise ValueError(f"k must be {q.dtype}, got {k.dtype}")
        Hk, ks = kshape[-2], (0, kst[0], kst[1]) if len(shape) == 3 else kst[:3]
    if not 1 <= H <= 65536 or (k is not None and not 1 <= Hk <= 65536):
        raise ValueError(f"1 to 65536 heads are taken: got {H} and {Hk}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    pshape = positions.shape
    if len(pshape) == 1 and pshape[0] == S:
        ps = (0, positions.stride(0))
    elif len(shape) == 4 and pshape == shape[:2]:
        ps = positions.stride()
    else:
        raise ValueError(f"positions {tuple(pshape)} do not fit q {tuple(shape)}")
    R = 2 * frequencies.numel()
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or not 2 <= R <= D or not frequencies.is_contiguous():
        raise ValueError(f"frequencies must be a contiguous fp64 vector of 1 to {D // 2} pairs, got "
                         f"{tuple(frequencies.shape)} {frequencies.dtype}")
    return (B, S, H, D, Hk, R), qs, ks, ps


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, frequencies: torch.Tensor, factor: float = 1.0,
           interleaved: bool = False, transposed: bool = False, inplace: bool = False, out: tuple | None = None):
    """Rotary positions on q [T, H, D] or [B, S, H, D] and, in the same launch, k with as many tokens, any number of heads and
    the same width: (q', k'), contiguous, or `out` (tensors like q and k, of any strides, that share no memory with each other,
    nor with q and k unless they are those), or with `inplace` q and k themselves.

    bf16, fp16 or fp32; the last dimension contiguous, the others of any stride. positions: int32 or int64, [T], [B, S], or [S]
    for all of a batch. frequencies: fp64 [R / 2], radians a position for each pair of the first R channels of a head; the
    others pass. Pairs are (i, i + R / 2), or (2 i, 2 i + 1) with `interleaved`. factor multiplies cos and sin. transposed:
    the gradient's rotation, backwards and with the same factor."""
    (B, S, H, D, Hk, R), qs, ks, ps = check_rotary(q, k, positions, frequencies)
    kind = ROW_TYPES.get(q.dtype)
    if kind is None or D > ROTARY_MAX_WIDTH:
        raise ValueError(f"q must be bf16, fp16 or fp32 with heads of up to {ROTARY_MAX_WIDTH} channels, got {q.dtype}, {D}")
    if inplace:
        out = (q, k)
    qo, ko = out or (None, None)
    if out is not None and ((ko is None) != (k is None) or qo.shape != q.shape or qo.dtype != q.dtype
                            or (k is not None and (ko.shape != k.shape or ko.dtype != k.dtype))):
        raise ValueError("out must be like q and k")
    for t, name in ((q, "q"), (k, "k"), (qo, "out"), (ko, "out")):
        if t is not None and t.stride(-1) != 1 and t.numel():
            raise ValueError(f"{name} must have a contiguous last dim")
    for t in (qo, ko):
        if t is not None and any(st == 0 and n > 1 for st, n in zip(t.stride(), t.shape)):
            raise ValueError("what is written has elements that share memory")
    if qo is not None and ko is not None and qo.data_ptr() == ko.data_ptr() and qo.numel() and ko.numel():
        raise ValueError("q and k are written to the same memory")
    with _device_of(q, k, positions, frequencies, qo, ko):
        if out is not None:
            heads = lambda t: (0, 0, 0) if t is None else (0, *t.stride()[:2]) if t.dim() == 3 else t.stride()[:3]
            qos, kos = heads(qo), heads(ko)
        else:
            qo, qos = _like(q), (S * H * D, H * D, D)
            ko, kos = (None, (0, 0, 0)) if k is None else (_like(k), (S * Hk * D, Hk * D, D))
        if B * S:
            call = _ROTARY.pack(q.data_ptr(), qo.data_ptr(), _address(k), _address(ko), *qs, *qos, *ks, *kos,
                                positions.data_ptr(), *ps, frequencies.data_ptr(), B, S, H, Hk,
                                positions.dtype == torch.int64, transposed, D, R, kind, interleaved, factor)
            check_rc(typed("rotary", "nplm_rotary_qk", "pp")(call, raw_stream()), "rotary")
            count_launch()
    return qo, ko


def swiglu_fwd(pre: torch.Tensor) -> torch.Tensor:
    T, two_i = pre.shape
    out = torch.empty((T, two_i // 2), dtype=_BF16, device=pre.device)
    rc = lib("elementwise").nplm_swiglu_fwd(ptr(pre), ptr(out), c_longlong(T), c_int(two_i // 2),
                                            stream_ptr())
    check_rc(rc, "swiglu_fwd")
    count_launch()
    return out


def swiglu_bwd(pre: torch.Tensor, dout: torch.Tensor) -> torch.Tensor:
    T, two_i = pre.shape
    dpre = torch.empty_like(pre)
    rc = lib("elementwise").nplm_swiglu_bwd(ptr(pre), ptr(dout), ptr(dpre), c_longlong(T),
                                            c_int(two_i // 2), stream_ptr())
    check_rc(rc, "swiglu_bwd")
    count_launch()
    return dpre


_ACT = {"gelu": 0, "relu": 1, "silu": 2}


def act_fwd(pre: torch.Tensor, act: str) -> torch.Tensor:
    out = torch.empty_like(pre)
    rc = lib("elementwise").nplm_act_fwd(ptr(pre), ptr(out), c_longlong(pre.numel()),
                                         c_int(_ACT[act]), stream_ptr())
    check_rc(rc, "act_fwd")
    count_launch()
    return out


def act_bwd(pre: torch.Tensor, dout: torch.Tensor, act: str) -> torch.Tensor:
    dpre = torch.empty_like(pre)
    rc = lib("elementwise").nplm_act_bwd(ptr(pre), ptr(dout), ptr(dpre), c_longlong(pre.numel()),
                                         c_int(_ACT[act]), stream_ptr())
    check_rc(rc, "act_bwd")
    count_launch()
    return dpre


def gather_rows(src: torch.Tensor, idx: torch.Tensor) -> torch.Tensor:
    n, C = idx.numel(), src.shape[1]
    dst = torch.empty((n, C), dtype=_BF16, device=src.device)
    rc = lib("elementwise").nplm_gather_rows(ptr(src), ptr(idx), ptr(dst), c_int(n), c_int(C),
                                             stream_ptr())
    check_rc(rc, "gather_rows")
    count_launch()
    return dst


def scatter_rows_(dst: torch.Tensor, idx: torch.Tensor, src: torch.Tensor) -> torch.Tensor:
    n, C = idx.numel(), src.shape[1]
    rc = lib("elementwise").nplm_scatter_rows(ptr(src), ptr(idx), ptr(dst), c_int(n), c_int(C),
                                              stream_ptr())
    check_rc(rc, "scatter_rows")
    count_launch()
    return dst


_UNPAD_MASKS = {torch.bool: 1, torch.uint8: 1, torch.int8: 1, torch.int32: 4, torch.int64: 8}


def unpad_takes(ids: torch.Tensor, mask: torch.Tensor) -> bool:
    """Whether `unpad` takes a padded batch: [B, S] integers on one GPU, contiguous, not empty."""
    return (ids.is_cuda and mask.is_cuda and ids.device == mask.device and ids.dim() == 2 and ids.shape == mask.shape
            and ids.numel() > 0 and ids.dtype in (torch.int32, torch.int64) and mask.dtype in _UNPAD_MASKS
            and ids.is_contiguous() and mask.is_contiguous() and not _is_tracing())


def unpad(ids: torch.Tensor, mask: torch.Tensor):
    """(flat ids, indices int64 into the B * S positions, positions int32, cu_seqlens int32 [B + 1]) of the tokens that the
    mask keeps. Waits for the device once, for their number."""
    B, S = ids.shape
    mb = _UNPAD_MASKS[mask.dtype]
    work = torch.empty(2 * B + 1, dtype=torch.int32, device=ids.device)
    cu, counts = work[:B + 1], work[B + 1:]
    rc = typed("elementwise", "nplm_unpad_count", "piiippp")(mask.data_ptr(), mb, B, S, counts.data_ptr(), cu.data_ptr(),
                                                             raw_stream())
    check_rc(rc, "unpad_count")
    T = int(cu[-1])
    flat = torch.empty(T, dtype=ids.dtype, device=ids.device)
    index = torch.empty(T, dtype=torch.int64, device=ids.device)
    pos = torch.empty(T, dtype=torch.int32, device=ids.device)
    rc = typed("elementwise", "nplm_unpad_fill", "pipipiipppp")(
        mask.data_ptr(), mb, ids.data_ptr(), ids.element_size(), cu.data_ptr(), B, S, index.data_ptr(), flat.data_ptr(),
        pos.data_ptr(), raw_stream())
    check_rc(rc, "unpad_fill")
    count_launch(3)
    return flat, index, pos, cu


def segment_mean(x: torch.Tensor, cu: torch.Tensor, drop_last: int = 0) -> torch.Tensor:
    """fp32 [B, C]: mean of x's rows cu[b] .. cu[b + 1] - drop_last (x bf16 [T, C] contiguous, cu int32 [B + 1])."""
    _chk(x, _BF16, "x")
    _chk(cu, torch.int32, "cu")
    if x.dim() != 2 or not x.is_contiguous() or not cu.is_contiguous():
        raise ValueError("x must be a contiguous [T, C] tensor and cu contiguous")
    B, C = cu.numel() - 1, x.shape[1]
    out = torch.empty((B, C), dtype=torch.float32, device=x.device)
    rc = lib("elementwise").nplm_segment_mean(ptr(x), ptr(cu), ptr(out), c_int(B), c_int(C), c_int(int(drop_last)),
                                              stream_ptr())
    check_rc(rc, "segment_mean")
    count_launch()
    return out


# --------------------------------------------------------------------------- cross entropy
def ce_count(labels):
    """(1 / number of labels >= 0, at least one; 0), fp32 [1] each: what `ce_fwd` takes as inv_count and loss."""
    _chk(labels, torch.int32, "labels")
    both = torch.empty(8, dtype=torch.float32, device=labels.device)
    inv, loss = both[:1], both[4:5]
    rc = typed("elementwise", "nplm_ce_count", "pippp")(labels.data_ptr(), labels.numel(), inv.data_ptr(), loss.data_ptr(),
                                                        raw_stream())
    check_rc(rc, "ce_count")
    count_launch()
    return inv, loss


def ce_fwd(h, W, bias, labels, inv_count, want_logits=False, loss=None):
    n, C = h.shape
    V = W.shape[0]
    dlogits = torch.empty((n, 32), dtype=torch.float32, device=h.device)
    logits = torch.empty((n, V), dtype=torch.float32, device=h.device) if want_logits else None
    if loss is None:
        loss = torch.zeros(1, dtype=torch.float32, device=h.device)
    rc = typed("elementwise", "nplm_ce_fwd", "ppppppppiiip")(
        h.data_ptr(), W.data_ptr(), _dp(bias), labels.data_ptr(), inv_count.data_ptr(), dlogits.data_ptr(), _dp(logits),
        loss.data_ptr(), n, C, V, raw_stream())
    check_rc(rc, "ce_fwd")
    count_launch()
    return loss, dlogits, logits


def ce_bwd(h, W, dlogits, gscale, dW, dbias):
    n, C = h.shape
    V = W.shape[0]
    dh = torch.empty_like(h)
    rc = typed("elementwise", "nplm_ce_bwd", "pppppppiiip")(
        h.data_ptr(), W.data_ptr(), dlogits.data_ptr(), gscale.data_ptr(), dh.data_ptr(), dW.data_ptr(), _dp(dbias), n, C, V,
        raw_stream())
    check_rc(rc, "ce_bwd")
    count_launch()
    return dh


# --------------------------------------------------------------------------- optimizer
def sumsq_(x: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    rc = lib("elementwise").nplm_sumsq(ptr(x), c_longlong(x.numel()), ptr(out), stream_ptr())
    check_rc(rc, "sumsq")
    count_launch()
    return out


def adamw_(p, m, v, g, p_bf16, hyper, sumsq, zero_grad=True) -> None:
    rc = lib("elementwise").nplm_adamw(ptr(p), ptr(m), ptr(v), ptr(g), ptr(p_bf16), ptr(hyper),
                                       ptr(sumsq), c_longlong(p.numel()), c_int(int(zero_grad)),
                                       stream_ptr())
    check_rc(rc, "adamw")
    count_launch()


def muon_momentum_(g, m, offsets, numel: int, upd, usq, sumsq, grad_scale: float, max_norm: float,
                   mu: float, nesterov: bool) -> None:
    """Momentum update of the matrices at flat `offsets` (int64, device) of g / m (fp32 flat
    buffers); writes the bf16 Newton-Schulz input `upd` [n, numel] and adds its squared Frobenius
    norms to `usq` [n]."""
    rc = lib("elementwise").nplm_muon_momentum(
        ptr(g), ptr(m), ptr(offsets), c_int(offsets.numel()), c_longlong(numel), ptr(upd), ptr(usq),
        ptr(sumsq), c_float(grad_scale), c_float(max_norm), c_float(mu), c_int(int(nesterov)), stream_ptr())
    check_rc(rc, "muon_momentum")
    count_launch()


def transpose_scale(x: torch.Tensor, scale: torch.Tensor | None = None) -> torch.Tensor:
    """[B, C, R] = x[B, R, C] transposed, times scale[b] (bf16 [B]) where given; x bf16 contiguous, R and C multiples
    of 64."""
    _chk(x, _BF16, "x")
    B, R, C = x.shape
    if not x.is_contiguous() or (scale is not None and (scale.dtype != _BF16 or scale.numel() != B
                                                        or not scale.is_contiguous())):
        raise ValueError("x must be contiguous and scale a contiguous bf16 [B]")
    y = torch.empty((B, C, R), dtype=_BF16, device=x.device)
    rc = lib("elementwise").nplm_transpose_scale(ptr(x), ptr(scale), ptr(y), c_int(B), c_int(R), c_int(C), stream_ptr())
    check_rc(rc, "transpose_scale")
    count_launch()
    return y


def muon_apply_(p, p_bf16, offsets, numel: int, O, lr: float, wd: float, cautious: bool) -> None:
    """p[offsets[i] : +numel] -= lr * (wd-term + O[i]) for the bf16 stack O [n, numel]; also
    writes the bf16 copy of the parameters."""
    rc = lib("elementwise").nplm_muon_apply(
        ptr(p), ptr(p_bf16), ptr(offsets), c_int(offsets.numel()), c_longlong(numel), ptr(O),
        c_float(lr), c_float(wd), c_int(int(cautious)), stream_ptr())
    check_rc(rc, "muon_apply")
    count_launch()


def adamw_slots_(p, m, v, g, p_bf16, offsets, numels, decay, max_numel: int, sumsq, grad_scale: float,
                 max_norm: float, lr: float, beta1: float, beta2: float, eps: float, wd: float,
                 bc1: float, bc2: float) -> None:
    """AdamW on the tensors listed in (offsets, numels, decay) of one flat buffer, one launch."""
    rc = lib("elementwise").nplm_adamw_slots(
        ptr(p), ptr(m), ptr(v), ptr(g), ptr(p_bf16), ptr(offsets), ptr(numels), ptr(decay),
        c_int(offsets.numel()), c_longlong(max_numel), ptr(sumsq), c_float(grad_scale), c_float(max_norm),
        c_float(lr), c_float(beta1), c_float(beta2), c_float(eps), c_float(wd), c_float(bc1), c_float(bc2),
        stream_ptr())
    check_rc(rc, "adamw_slots")
    count_launch()


_STEP_TYPES = (torch.float32, torch.bfloat16)
MOMENT_BLOCK = 256      # elements of a tensor that share the offset of their 8-bit moments


def moment_blocks(numels) -> int:
    """Blocks that the moments of tensors of these sizes take: every tensor starts one."""
    return sum(-(-n // MOMENT_BLOCK) for n in numels)


def check_moments(m: torch.Tensor, v: torch.Tensor, scales: torch.Tensor | None) -> tuple[int, int]:
    """(bits, blocks) of moments: fp32 without scales, or uint8 with scales uint8 [2, blocks]."""
    bits = {torch.float32: 32, torch.uint8: 8}.get(m.dtype)
    if bits is None or v.dtype != m.dtype or (bits == 8) != (scales is not None):
        raise ValueError(f"moments must be fp32, or uint8 with scales: got {m.dtype}, {v.dtype}"
                         f"{'' if scales is None else ' and scales'}")
    blocks = m.numel() // MOMENT_BLOCK
    if m.numel() != blocks * MOMENT_BLOCK or v.numel() != m.numel() or not (m.is_contiguous() and v.is_contiguous()):
        raise ValueError(f"moments must be contiguous, equally large and whole blocks of {MOMENT_BLOCK}")
    if scales is not None and (tuple(scales.shape) != (2, blocks) or scales.dtype != torch.uint8
                               or not scales.is_contiguous()):
        raise ValueError(f"scales must be a contiguous uint8 [2, {blocks}], got {tuple(scales.shape)} {scales.dtype}")
    return bits, blocks


def check_step(params, grads, copies, decay, m, v, scales, hyper, rng, sumsq) -> tuple[int, int, list[int]]:
    """Checks the arguments of an AdamW step over tensors; (bits, blocks, sizes)."""
    bits, blocks = check_moments(m, v, scales)
    n, tensor = len(params), torch.Tensor
    if len(grads) != n or (copies is not None and len(copies) != n) or (decay is not None and len(decay) != n):
        raise ValueError("params, grads, copies and decay must be equally long")
    sizes = list(map(tensor.numel, params))
    if sizes != list(map(tensor.numel, grads)) or (copies is not None and sizes != list(map(tensor.numel, copies))):
        raise ValueError("params, grads and copies must have the same sizes")
    if moment_blocks(sizes) > blocks:
        raise ValueError(f"the moments hold {blocks} blocks of {MOMENT_BLOCK}, the tensors take {moment_blocks(sizes)}")
    home = m.get_device()
    for name, ts, allowed in (("params", params, _STEP_TYPES), ("grads", grads, _STEP_TYPES), ("copies", copies, (_BF16,))):
        if ts:
            kinds = {t.dtype for t in ts}
            if len(kinds) != 1 or not kinds.issubset(allowed):
                raise ValueError(f"{name} must all be one of {allowed}, got {sorted(map(str, kinds))}")
            if not all(map(tensor.is_contiguous, ts)):
                raise ValueError(f"{name} must be contiguous")
            if set(map(tensor.get_device, ts)) != {home}:
                raise ValueError(f"{name} and the moments are on different devices")
    if copies is not None and n and params[0].dtype != torch.float32:
        raise ValueError("bf16 copies are of fp32 params")
    for written in (params, copies):
        if written is not None and len(set(map(tensor.data_ptr, written))) != n:       # (tensors without elements have none)
            starts = [p.data_ptr() for p, k in zip(written, sizes) if k]
            if len(set(starts)) != len(starts):
                raise ValueError("a tensor is listed twice")
    if hyper.dtype != torch.float32 or hyper.numel() != 9 or not hyper.is_contiguous():
        raise ValueError("hyper must be 9 contiguous fp32 numbers")
    if sumsq is not None and (sumsq.dtype != torch.float32 or sumsq.numel() != 1):
        raise ValueError("sumsq must be one fp32 number")
    if bits == 8 and (rng is None or rng.dtype != torch.int64 or rng.numel() != 1):
        raise ValueError("8-bit moments need rng, one int64 number")
    for t in (v, scales, hyper, rng, sumsq):
        if t is not None and t.get_device() != home:
            raise ValueError(f"tensors on different devices: {m.device} and {t.device}")
    return bits, blocks, sizes


def adamw_tensors_(params, grads, exp_avg, exp_avg_sq, hyper, *, scales=None, rng=None, copies=None, decay=None,
                   sumsq=None) -> None:
    """One AdamW step (the update of `adamw_`) over a list of tensors, 128 to a launch.

    params, grads: lists of contiguous tensors, fp32 or bf16 each. copies: bf16 copies of fp32 params, written too. No two tensors that
    are written may share memory (one that is listed twice is refused).
    decay: which tensors the weight decay acts on (None: all). exp_avg, exp_avg_sq: fp32 [blocks * 256] in the order of the
    tensors, each starting a block; or their 8-bit codes, uint8, with scales uint8 [2, blocks] (see `moment_values`) and rng,
    an int64 number that must be another one each step: codes are rounded stochastically.
    hyper: fp32 [9] lr, beta1, beta2, eps, weight decay, bias corrections 1 and 2, gradient scale, largest norm; with sumsq, the
    sum of the gradients' squares, gradients are clipped to the largest norm. hyper, rng and sumsq are read on the
    device, by a captured step at each replay. The codes of moments that are not finite are unspecified."""
    bits, blocks, sizes = check_step(params, grads, copies, decay, exp_avg, exp_avg_sq, scales, hyper, rng, sumsq)
    n, pointer = len(params), torch.Tensor.data_ptr
    if not n:
        return
    if exp_avg.data_ptr() % 16 or exp_avg_sq.data_ptr() % 16:
        raise ValueError("moments must start on 16 bytes")
    first, at = [], 0
    for k in sizes:
        first.append(at)
        at += -(-k // MOMENT_BLOCK)
    table = Struct(f"={n}q")
    with _device_of(exp_avg):
        rc = typed("adamw_tensors", "nplm_adamw_tensors", "ppppppiiiippplpppp")(
            table.pack(*map(pointer, params)), table.pack(*map(pointer, grads)),
            None if copies is None else table.pack(*map(pointer, copies)), table.pack(*sizes), table.pack(*first),
            bytes([1] * n) if decay is None else bytes(map(bool, decay)), n, 2 if params[0].dtype == torch.float32 else 0,
            2 if grads[0].dtype == torch.float32 else 0, bits, exp_avg.data_ptr(), exp_avg_sq.data_ptr(), _dp(scales), blocks,
            hyper.data_ptr(), _dp(sumsq), _dp(rng), raw_stream())
        check_rc(rc, "adamw_tensors")
    count_launch(-(-(n - sizes.count(0)) // 128))


def moment_values(exp_avg, exp_avg_sq, scales, dtype=torch.float32):
    """What the codes of 8-bit moments stand for: (first, second) moments [blocks * 256], fp32 or bf16, both exact."""
    _, blocks = check_moments(exp_avg, exp_avg_sq, scales)
    if exp_avg.dtype != torch.uint8 or dtype not in (torch.float32, _BF16):
        raise ValueError("8-bit moments as fp32 or bf16")
    with _device_of(exp_avg, exp_avg_sq, scales):
        m = torch.empty(blocks * MOMENT_BLOCK, dtype=dtype, device=exp_avg.device)
        v = torch.empty_like(m)
        rc = typed("adamw_tensors", "nplm_moment_values", "ppplppip")(
            exp_avg.data_ptr(), exp_avg_sq.data_ptr(), scales.data_ptr(), blocks, m.data_ptr(), v.data_ptr(),
            2 if dtype == torch.float32 else 0, raw_stream())
        check_rc(rc, "moment_values")
        count_launch(blocks > 0)
    return m, v


def moment_codes(m: torch.Tensor, v: torch.Tensor):
    """(codes of the first moments, of the second, scales) of fp32 [blocks * 256] moments, rounded to the nearest code: what
    `moment_values` gave comes back as it was."""
    _, blocks = check_moments(m, v, None)
    with _device_of(m, v):
        mc, vc = (torch.empty(m.numel(), dtype=torch.uint8, device=m.device) for _ in range(2))
        scales = torch.empty((2, blocks), dtype=torch.uint8, device=m.device)
        if m.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("moments must start on 16 bytes")
        rc = typed("adamw_tensors", "nplm_moment_codes", "ppppplp")(
            m.data_ptr(), v.data_ptr(), mc.data_ptr(), vc.data_ptr(), scales.data_ptr(), blocks, raw_stream())
        check_rc(rc, "moment_codes")
        count_launch(blocks > 0)
    return mc, vc, scales


def cast_f32_bf16_(src: torch.Tensor, dst: torch.Tensor) -> None:
    rc = lib("elementwise").nplm_cast_f32_bf16(ptr(src), ptr(dst), c_longlong(src.numel()),
                                               stream_ptr())
    check_rc(rc, "cast")
    count_launch()


def masked_mse(s, t, valid, inv_count, want_grad=True, rows=None):
    """rows (int64 [T], contiguous): row r of s is compared with row rows[r] of t."""
    T, C = s.shape
    ds = torch.empty_like(s) if want_grad else None
    loss = torch.zeros(1, dtype=torch.float32, device=s.device)
    rc = lib("elementwise").nplm_masked_mse(ptr(s), ptr(t), ptr(valid), ptr(rows), ptr(inv_count), ptr(ds),
                                            ptr(loss), c_int(T), c_int(C), stream_ptr())
    check_rc(rc, "masked_mse")
    count_launch()
    return loss, ds


# --------------------------------------------------------------------------- attention
def seq_bounds(cu_seqlens: torch.Tensor, T: int):
    _chk(cu_seqlens, torch.int32, "cu_seqlens")
    s = torch.empty(T, dtype=torch.int32, device=cu_seqlens.device)
    e = torch.empty(T, dtype=torch.int32, device=cu_seqlens.device)
    rc = lib("attention").nplm_seq_bounds(ptr(cu_seqlens), c_int(cu_seqlens.numel() - 1), ptr(s),
                                          ptr(e), c_int(T), stream_ptr())
    check_rc(rc, "seq_bounds")
    count_launch()
    return s, e


_FA_IMPL = [_os.environ.get("NPLM_FA_IMPL", "ws")]


def set_attention_impl(name: str) -> None:
    """"ws": the persistent warp-specialised kernels (attention_ws.cu, default);
    "single": the one-role-per-CTA kernels of attention.cu."""
    if name not in ("ws", "single"):
        raise ValueError("attention impl must be 'ws' or 'single'")
    _FA_IMPL[0] = name


def fa_fwd(qkv, seq_start, seq_end, H, D, window, scale, impl: str | None = None, max_ctas: int = 0):
    _chk(qkv, _BF16, "qkv")
    T = qkv.shape[0]
    out = torch.empty((T, H * D), dtype=_BF16, device=qkv.device)
    lse = torch.empty((H, T), dtype=torch.float32, device=qkv.device)
    if (impl or _FA_IMPL[0]) == "ws":
        rc = typed("attention_ws", "nplm_fa_fwd_ws", "pppppiiiifipp")(
            qkv.data_ptr(), out.data_ptr(), lse.data_ptr(), seq_start.data_ptr(), seq_end.data_ptr(), T, H, D, window,
            scale, max_ctas, status_word(qkv.device).data_ptr(), raw_stream())
    else:
        rc = lib("attention").nplm_fa_fwd(ptr(qkv), ptr(out), ptr(lse), ptr(seq_start), ptr(seq_end),
                                          c_int(T), c_int(H), c_int(D), c_int(window), c_float(scale),
                                          ptr(status_word(qkv.device)), stream_ptr())
    check_rc(rc, "fa_fwd")
    count_launch()
    return out, lse


def gemm_dgrad_delta(dy: torch.Tensor, w: torch.Tensor, o: torch.Tensor, delta: torch.Tensor) -> torch.Tensor:
    """dO = dy @ w (w [K, N] read MN-major) in bf16 and, from the same epilogue,
    delta[h, t] = sum over head h's 64 columns of dO[t] * o[t] (fp32 [N / 64, T])."""
    _chk(dy, _BF16, "dy")
    _chk(w, _BF16, "w")
    _chk(o, _BF16, "o")
    _chk(delta, torch.float32, "delta")
    M, Kd = dy.shape
    if w.shape[0] != Kd:
        raise ValueError("inner dims differ")
    N = w.shape[1]
    if N % 64 or tuple(o.shape) != (M, N) or tuple(delta.shape) != (N // 64, M) or not delta.is_contiguous():
        raise ValueError("o must be [M, N], delta [N / 64, M] contiguous, N a multiple of 64")
    out = torch.empty((M, N), dtype=_BF16, device=dy.device)
    rc = typed("gemm_tcgen05", "nplm_gemm_bf16_delta", "pppppp" + "iiiiiiii" + "pp")(
        dy.data_ptr(), w.data_ptr(), out.data_ptr(), o.data_ptr(), delta.data_ptr(), 0, M, N, Kd, _rowmajor(dy, "dy"),
        _rowmajor(w, "w"), N, _rowmajor(o, "o"), 1, status_word(dy.device).data_ptr(), raw_stream())
    check_rc(rc, "gemm_bf16_delta")
    count_launch()
    return out


_FA_DETERMINISTIC = [_os.environ.get("NPLM_FA_DETERMINISTIC", "0") not in ("", "0")]


def set_attention_deterministic(flag: bool) -> None:
    """True: the warp-specialised backward pass forms dQ in a second, query-stationary launch instead
    of fp32 atomics, so two runs on the same inputs give the same bits (about 1.4x the time). The weight gradients
    of linear layers (bf16 and e4m3), which by default are summed by several work items in any order, then come
    from one work item a tile."""
    _FA_DETERMINISTIC[0] = bool(flag)


def fa_bwd(qkv, out, dout, lse, seq_start, seq_end, H, D, window, scale, dq_acc=None, delta=None,
           rope: tuple | None = None, delta_ready: bool = False, impl: str | None = None, max_ctas: int = 0,
           deterministic: bool | None = None):
    """rope = (pos, cos, sin): q / k in qkv were rotated before the forward pass; dQ / dK are rotated
    back inside the kernels. delta_ready: `delta` [H, T] already holds rowsum(dO * O) (see
    gemm_dgrad_delta); the kernel that computes it from out and dout is skipped. deterministic (default:
    `set_attention_deterministic`): no atomics, bitwise reproducible (warp-specialised kernels only)."""
    T = qkv.shape[0]
    dqkv = torch.empty_like(qkv)
    use_ws = (impl or _FA_IMPL[0]) == "ws"
    det = use_ws and (_FA_DETERMINISTIC[0] if deterministic is None else deterministic)
    if dq_acc is None and not det:
        dq_acc = torch.empty((T, H * D), dtype=torch.float32, device=qkv.device)
    if delta is None:
        delta = torch.empty((H, T), dtype=torch.float32, device=qkv.device)
    if not dout.is_contiguous():
        dout = dout.contiguous()
    r_pos, r_cos, r_sin = rope if rope is not None else (None, None, None)
    if delta_ready:
        out = None
    if use_ws:
        rc = typed("attention_ws", "nplm_fa_bwd_ws_mode", "ppppppppp" + "iiiif" + "pppii" + "pp")(
            qkv.data_ptr(), _dp(out), dout.data_ptr(), lse.data_ptr(), dqkv.data_ptr(), _dp(dq_acc), delta.data_ptr(),
            seq_start.data_ptr(), seq_end.data_ptr(), T, H, D, window, scale, _dp(r_pos), _dp(r_cos), _dp(r_sin),
            max_ctas, 3 if det else -1, status_word(qkv.device).data_ptr(), raw_stream())
    else:
        rc = lib("attention").nplm_fa_bwd_rope(ptr(qkv), ptr(out), ptr(dout), ptr(lse), ptr(dqkv),
                                               ptr(dq_acc), ptr(delta), ptr(seq_start), ptr(seq_end),
                                               c_int(T), c_int(H), c_int(D), c_int(window), c_float(scale),
                                               ptr(r_pos), ptr(r_cos), ptr(r_sin),
                                               ptr(status_word(qkv.device)), stream_ptr())
    check_rc(rc, "fa_bwd")
    count_launch(3 if delta_ready else 4)
    return dqkv


def fa_bias_fwd(qkv: torch.Tensor, seq_start: torch.Tensor, seq_end: torch.Tensor, bias: torch.Tensor,
                H: int, D: int, scale: float = 1.0) -> torch.Tensor:
    """Inference attention with a relative-position bias (T5-style teacher).

    qkv bf16 [T, 3*H*D] (q | k | v, head-major), seq_start / seq_end int32 [T] (key range of every
    token), bias fp32 [H, 2*S-1] indexed by key - query + S - 1. Returns bf16 [T, H*D]."""
    _chk(qkv, _BF16, "qkv")
    _chk(seq_start, torch.int32, "seq_start")
    _chk(seq_end, torch.int32, "seq_end")
    _chk(bias, torch.float32, "bias")
    T = qkv.shape[0]
    S = (bias.shape[1] + 1) // 2
    out = torch.empty((T, H * D), dtype=_BF16, device=qkv.device)
    rc = lib("attention_bias").nplm_fa_bias_fwd(ptr(qkv), ptr(out), ptr(seq_start), ptr(seq_end),
                                                ptr(bias.contiguous()), c_int(T), c_int(H), c_int(D), c_int(S),
                                                c_float(scale), ptr(status_word(qkv.device)), stream_ptr())
    check_rc(rc, "fa_bias_fwd")
    count_launch()
    return out


def check_status() -> None:
    _lib.check_status()


# --------------------------------------------------------------------------- conv / mHC
def dwconv(x, w, bias, seq_start, seq_end, flip=False, skip=False):
    """With skip x plus the convolution, both bf16."""
    T, C = x.shape
    KS = w.shape[1]
    y = torch.empty_like(x)
    rc = lib("extras").nplm_dwconv(ptr(x), ptr(w), ptr(bias), ptr(seq_start), ptr(seq_end), ptr(y), c_int(T),
                                   c_int(C), c_int(KS), c_int(int(flip)), c_int(int(skip)), stream_ptr())
    check_rc(rc, "dwconv")
    count_launch()
    return y


def dwconv_bwd_w(x, dy, seq_start, seq_end, dw, dbias):
    T, C = x.shape
    KS = dw.shape[1]
    rc = lib("extras").nplm_dwconv_bwd_w(ptr(x), ptr(dy), ptr(seq_start), ptr(seq_end), ptr(dw), ptr(dbias),
                                         c_int(T), c_int(C), c_int(KS), stream_ptr())
    check_rc(rc, "dwconv_bwd_w")
    count_launch()


def mhc_read(X, alpha):
    T, n, C = X.shape
    h = torch.empty((T, C), dtype=_BF16, device=X.device)
    rc = lib("extras").nplm_mhc_read(ptr(X), ptr(alpha), ptr(h), c_int(T), c_int(n), c_int(C), stream_ptr())
    check_rc(rc, "mhc_read")
    count_launch()
    return h


def mhc_write(X, y, R, beta, mean: bool = False):
    """With mean also the mean over the written streams [T, C]."""
    T, n, C = X.shape
    Xn = torch.empty_like(X)
    z = torch.empty((T, C), dtype=_BF16, device=X.device) if mean else None
    rc = lib("extras").nplm_mhc_write(ptr(X), ptr(y), ptr(R), ptr(beta), ptr(Xn), ptr(z), c_int(T), c_int(n), c_int(C),
                                      stream_ptr())
    check_rc(rc, "mhc_write")
    count_launch()
    return (Xn, z) if mean else Xn


def mhc_mean(X):
    """Mean over the streams: X [T, n, C] bf16 -> [T, C]."""
    T, n, C = X.shape
    z = torch.empty((T, C), dtype=_BF16, device=X.device)
    rc = lib("extras").nplm_mhc_mean(ptr(X), ptr(z), c_int(T), c_int(n), c_int(C), stream_ptr())
    check_rc(rc, "mhc_mean")
    count_launch()
    return z


def mhc_dx_combine(g, alpha, dh, dz, shape):
    """dX = g + alpha[:, :, None] * dh[:, None, :] + dz[:, None, :] / n in one pass (any of the three
    terms may be None); shape = (T, n, C)."""
    T, n, C = shape
    ref = next(t for t in (g, dh, dz) if t is not None)
    dX = torch.empty((T, n, C), dtype=_BF16, device=ref.device)
    rc = lib("extras").nplm_mhc_dx_combine(ptr(g), ptr(alpha), ptr(dh), ptr(dz), ptr(dX), c_int(T), c_int(n),
                                           c_int(C), stream_ptr())
    check_rc(rc, "mhc_dx_combine")
    count_launch()
    return dX


def mhc_bwd(X, y, R, alpha, beta, dXn, dh, want_dx: bool = True, dz=None):
    """Backward of write (dXn given) and / or read (dh given). Returns (dX, dy, dR, dalpha, dbeta);
    want_dx=False skips the dX output (only the coefficient gradients are computed). With dz the backward of write alone,
    of the gradient mhc_dx_combine(dXn, alpha, dh, dz)."""
    T, n, C = X.shape
    dev = X.device
    dX = torch.empty_like(X) if want_dx else None
    dy = torch.empty((T, C), dtype=_BF16, device=dev) if dXn is not None else None
    dR = torch.empty((T, n, n), dtype=torch.float32, device=dev) if dXn is not None else None
    dbeta = torch.empty((T, n), dtype=torch.float32, device=dev) if dXn is not None else None
    dalpha = torch.empty((T, n), dtype=torch.float32, device=dev) if dh is not None and dz is None else None
    rc = lib("extras").nplm_mhc_bwd(ptr(X), ptr(y), ptr(R), ptr(alpha), ptr(beta), ptr(dXn), ptr(dh), ptr(dz), ptr(dX),
                                    ptr(dy), ptr(dR), ptr(dalpha), ptr(dbeta), c_int(T), c_int(n), c_int(C),
                                    stream_ptr())
    check_rc(rc, "mhc_bwd")
    count_launch()
    return dX, dy, dR, dalpha, dbeta


# --------------------------------------------------------------------------- device-side MLM masking
def _coef_bf16(*params) -> int:
    """1 when the parameters are all bf16, 0 when all fp32."""
    kinds = {p.dtype for p in params}
    if kinds not in ({_BF16}, {torch.float32}) or not all(p.is_contiguous() for p in params):
        raise ValueError("the static parameters must be contiguous and of one type, fp32 or bf16")
    return int(kinds == {_BF16})


def mhc_coef_fwd(pre, a, b, r, s, iters: int, n: int):
    """Raw coefficient projections pre bf16 [T, 2n+n*n] -> (alpha [T,n], beta [T,n], R [T,n,n]) fp32.
    a, b [n], r [n,n], s [3]: static parts and dynamic scales, all fp32 or all bf16, contiguous."""
    _chk(pre, _BF16, "pre")
    T = pre.shape[0]
    dev = pre.device
    alpha = torch.empty((T, n), dtype=torch.float32, device=dev)
    beta = torch.empty((T, n), dtype=torch.float32, device=dev)
    R = torch.empty((T, n, n), dtype=torch.float32, device=dev)
    rc = lib("extras").nplm_mhc_coef_fwd(ptr(pre), ptr(a), ptr(b), ptr(r), ptr(s), c_int(_coef_bf16(a, b, r, s)), c_int(iters), c_int(T),
                                         c_int(n), ptr(alpha), ptr(beta), ptr(R), stream_ptr())
    check_rc(rc, "mhc_coef_fwd")
    count_launch()
    return alpha, beta, R


def mhc_coef_bwd(pre, a, b, r, s, iters: int, n: int, dalpha, dbeta, dR, da, db, dr, ds):
    """Backward of mhc_coef_fwd. Returns dpre (bf16); da, db, dr, ds (fp32) are accumulated in place."""
    T = pre.shape[0]
    dpre = torch.empty_like(pre)
    rc = lib("extras").nplm_mhc_coef_bwd(ptr(pre), ptr(a), ptr(b), ptr(r), ptr(s), c_int(_coef_bf16(a, b, r, s)), c_int(iters), c_int(T),
                                         c_int(n), ptr(dalpha), ptr(dbeta), ptr(dR), ptr(dpre), ptr(da), ptr(db),
                                         ptr(dr), ptr(ds), stream_ptr())
    check_rc(rc, "mhc_coef_bwd")
    count_launch()
    return dpre


def mlm_mask(ids: torch.Tensor, n_real: int, special_ids, mask_id: int, pool: torch.Tensor, p_sel: float,
             p_mask: float, p_rand: float, seed: int, step: int):
    """Philox masking of flat int64 ids on the device. Returns (corrupted ids, labels)."""
    from ctypes import c_ulonglong
    _chk(ids, torch.int64, "ids")
    _chk(pool, torch.int32, "pool")
    bits = 0
    for s in special_ids:
        bits |= 1 << int(s)
    out, labels = torch.empty_like(ids), torch.empty_like(ids)
    rc = lib("extras").nplm_mlm_mask(ptr(ids), ptr(out), ptr(labels), c_int(ids.numel()), c_int(int(n_real)),
                                     c_ulonglong(bits), c_int(mask_id), ptr(pool), c_int(pool.numel()),
                                     c_float(p_sel), c_float(p_mask), c_float(p_rand), c_ulonglong(seed),
                                     c_ulonglong(step), stream_ptr())
    check_rc(rc, "mlm_mask")
    count_launch()
    return out, labels
