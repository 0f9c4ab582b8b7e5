"""Moments of AdamW over a list of tensors, in fp32 or in 8 bits, and the step that updates them.

On a GPU the step is one kernel launch (`kernels.adamw_tensors_`, whose source explains the 8-bit codes); on a CPU it is the
fp32 restatement below, which has the kernel's moments and codes bit for bit.

The reference keeps fp32 moments (torch.optim.AdamW, src/nanoplm/pretraining/pure_pipeline.py:107-147) and has no 8-bit ones.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import kernels as K

BLOCK = K.MOMENT_BLOCK
_LOW32 = 0xffffffff


# ------------------------------------------------------------------------------------ restatement
def _mix(x: torch.Tensor) -> torch.Tensor:
    x = ((x ^ (x >> 16)) * 0x7feb352d) & _LOW32
    x = ((x ^ (x >> 15)) * 0x846ca68b) & _LOW32
    return x ^ (x >> 16)


def random_bits(n: int, rng: torch.Tensor) -> torch.Tensor:
    """32 random bits (int64) for each of n elements: a function of the step's number and the element's place."""
    key = _mix((rng & _LOW32) ^ _mix((rng >> 32) & _LOW32))
    at = torch.arange(n, device=rng.device)
    return _mix((at & _LOW32) ^ _mix((key + (at >> 32)) & _LOW32))


def _offsets(exponents: torch.Tensor, signed: bool) -> torch.Tensor:
    return (exponents.to(torch.int32) - (15 if signed else 31)).clamp(min=0)[:, None] << 3


def encode(x: torch.Tensor, r, signed: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, exponents) of fp32 values [blocks * 256]; r: random numbers of 20 bits, or one number for all."""
    bits = x.abs().view(torch.int32).view(-1, BLOCK)
    e = (bits.amax(1) + 0xfffff) >> 23
    base = _offsets(e, signed)
    r = torch.as_tensor(r, device=x.device).to(torch.int32)
    r = r.view(-1, BLOCK) if r.dim() else r
    code = ((bits + r) >> 20) - base
    least = (base + 1) << 20
    if signed:
        up = r.float() * (least.view(torch.float32) * 2.0 ** -20) < x.abs().view(-1, BLOCK)
        code = torch.where(bits < least, up.to(torch.int32), code)
        code = torch.where((code > 0) & torch.signbit(x).view(-1, BLOCK), code + 128, code)
    else:
        code = torch.where(bits < least, 1, code)
    code = torch.where(bits == 0, 0, code)
    return code.to(torch.uint8).view(-1), e.to(torch.uint8)


def decode(codes: torch.Tensor, exponents: torch.Tensor, signed: bool) -> torch.Tensor:
    code = codes.view(-1, BLOCK).to(torch.int32)
    low = code & 127 if signed else code
    x = torch.where(low == 0, 0, (low + _offsets(exponents, signed)) << 20).view(torch.float32)
    return (torch.where(code >= 128, -x, x) if signed else x).view(-1)


def _step_cpu(params, grads, m, v, hyper, scales, rng, copies, decay, sumsq) -> None:
    lr, b1, b2, eps, wd, bc1, bc2, gs, most = hyper
    factor = gs
    if sumsq is not None and float(most) > 0:
        factor = gs * torch.fmin(most / (sumsq.reshape(()).sqrt() * gs + 1e-6), torch.ones(()))
    eight = scales is not None
    mv, vv = (decode(m, scales[0], True), decode(v, scales[1], False)) if eight else (m, v)
    at = 0
    for i, (p, g) in enumerate(zip(params, grads)):
        n = p.numel()
        g = g.reshape(-1).float() * factor
        a, b = mv[at:at + n], vv[at:at + n]
        a.copy_(a * b1 + g * (1 - b1))
        b.copy_(b * b2 + (g * g) * (1 - b2))
        keep = 1 - lr * wd if decay is None or decay[i] else 1.0
        new = p.reshape(-1).float() * keep - lr / bc1 * (a / (b.sqrt() / bc2.sqrt() + eps))
        p.view(-1).copy_(new)
        if copies is not None:
            copies[i].view(-1).copy_(new)
        at += -(-n // BLOCK) * BLOCK
    if eight:
        r = random_bits(mv.numel(), rng)
        for values, codes, row, bits, signed in ((mv, m, 0, r & 0xfffff, True), (vv, v, 1, r >> 12, False)):
            c, e = encode(values, bits, signed)
            codes.copy_(c)
            scales[row].copy_(e)


# --------------------------------------------------------------------------------------- moments
class TensorMoments:
    """First and second moments of a list of tensors of the given sizes, every tensor in blocks of its own.

    bits 32: fp32, 8 bytes an element. bits 8: 2 bytes an element and 2 a block of 256."""

    def __init__(self, numels: Sequence[int], device, bits: int = 32):
        if bits not in (8, 32):
            raise ValueError(f"moments have 8 or 32 bits, got {bits}")
        self.numels, self.bits = list(numels), bits
        self.device = torch.device(device)
        blocks = K.moment_blocks(self.numels)
        dtype = torch.uint8 if bits == 8 else torch.float32
        self.m = torch.zeros(blocks * BLOCK, dtype=dtype, device=self.device)
        self.v = torch.zeros_like(self.m)
        self.scales = torch.zeros(2, blocks, dtype=torch.uint8, device=self.device) if bits == 8 else None
        self._at = []
        at = 0
        for n in self.numels:
            self._at.append(at)
            at += -(-n // BLOCK) * BLOCK

    def step(self, params, grads, hyper, *, rng=None, copies=None, decay=None, sumsq=None) -> None:
        """One AdamW step: see `kernels.adamw_tensors_`."""
        if [p.numel() for p in params] != self.numels:
            raise ValueError("the tensors are not those that these moments were made for")
        if self.device.type == "cuda":
            K.adamw_tensors_(params, grads, self.m, self.v, hyper, scales=self.scales, rng=rng, copies=copies, decay=decay,
                             sumsq=sumsq)
        else:
            K.check_step(params, grads, copies, decay, self.m, self.v, self.scales, hyper, rng, sumsq)
            with torch.no_grad():
                _step_cpu(params, grads, self.m, self.v, hyper, self.scales, rng, copies, decay, sumsq)

    def values(self) -> tuple[list[torch.Tensor], list[torch.Tensor]]:
        """fp32 first and second moments of every tensor, flat (for checkpoints). Those of 32 bits are the moments themselves,
        which the next step changes."""
        if self.bits == 32:
            m, v = self.m, self.v
        elif self.device.type == "cuda":
            m, v = K.moment_values(self.m, self.v, self.scales)
        else:
            m, v = decode(self.m, self.scales[0], True), decode(self.v, self.scales[1], False)
        cut = lambda t: [t[a:a + n] for a, n in zip(self._at, self.numels)]
        return cut(m), cut(v)

    def load(self, m: Sequence[torch.Tensor], v: Sequence[torch.Tensor]) -> None:
        """Takes fp32 moments; those that `values` gave come back as they were."""
        if [t.numel() for t in m] != self.numels or [t.numel() for t in v] != self.numels:
            raise ValueError("the moments are of tensors of other sizes")
        flat = torch.zeros(2, self.m.numel(), dtype=torch.float32, device=self.device)
        for row, ts in zip(flat, (m, v)):
            for a, n, t in zip(self._at, self.numels, ts):
                row[a:a + n] = t.reshape(-1).to(self.device, torch.float32)
        if self.bits == 32:
            self.m.copy_(flat[0])
            self.v.copy_(flat[1])
        elif self.device.type == "cuda":
            mc, vc, scales = K.moment_codes(flat[0], flat[1])
            self.m.copy_(mc)
            self.v.copy_(vc)
            self.scales.copy_(scales)
        else:
            for row, codes, values, signed in ((0, self.m, flat[0], True), (1, self.v, flat[1], False)):
                c, e = encode(values, 0x80000, signed)
                codes.copy_(c)
                self.scales[row].copy_(e)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.m, self.v, self.scales) if t is not None)
