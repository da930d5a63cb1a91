"""The 8-bit and clipping operators in 64 bits, written from their definitions,
and how far a result in fewer bits may be from them."""
import math

import torch

TINY = 2.0 ** -126
U32 = 2.0 ** -24      # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def codes_and_scale(x):
    """quantize_rows: (codes int8, scale fp32), to be met exactly."""
    v = x.detach().cpu().double()
    top = v.abs().amax(-1) if v.shape[-1] else torch.zeros(v.shape[:-1]).double()
    scale = torch.maximum((top / 127).float(), torch.full_like(top, TINY).float())
    bad = ~torch.isfinite(top)
    # exact quotients of 24-bit numbers are either on a border of two codes or
    # 2^-32 of their size away from it, so 53 bits round as exact ones do
    codes = torch.round(v / scale.double()[..., None])
    codes[bad] = 0
    scale[bad] = math.nan
    return codes.to(torch.int8), scale


def product(xq, sx, wq, sw, bias, act):
    """int8_matmul: (result, bound on the error of fp32 arithmetic)."""
    xq, sx, wq, sw = (t.detach().cpu().double() for t in (xq, sx, wq, sw))
    bias = torch.zeros_like(sw) if bias is None else bias.detach().cpu().double()
    if xq.dim() == 1:  # one row without an axis of rows
        y, err = product(xq[None], sx[None], wq, sw, bias, act)
        return y[0], err[0]
    p = (xq @ wq.transpose(-1, -2)) * sx[..., None] * sw[..., None, :]
    y = p + bias[..., None, :]
    # roundings: the sum's conversion and two products (of p), one addition (of
    # y); the second order goes into the 4th unit; 2^-148: subnormal products
    err = 4 * U32 * p.abs() + U32 * y.abs() + 2.0 ** -148
    if act == "relu":
        return y.clamp_min(0), err
    if act == "tanh":  # its slope is at most 1; the function itself: 2 steps
        return y.tanh(), err + 4 * U32
    return y, err


def check_product(got, want, err, dtype):
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    top = torch.finfo(dtype).max
    over = want.abs() > top * (1 + half_step(dtype))
    assert bool((got[over].abs() >= top).all())
    fine = ~want.isnan() & ~over
    least = torch.finfo(dtype).smallest_normal * half_step(dtype)
    most = err + half_step(dtype) * (want.abs() + err) + least
    off = (got - want).abs()
    assert bool((off <= most)[fine].all()), float((off / most)[fine].max())


def clipped(tensors, max_norm):
    """clip_by_global_norm: (values in 64 bits, norm in 64 bits)."""
    cpu = [t.detach().cpu().double() for t in tensors]
    norm = math.sqrt(math.fsum(float((t * t).sum()) for t in cpu))
    c = max_norm / norm if norm > max_norm else 1.0
    return [t * c for t in cpu], norm


def check_clipped(got, norm, want, want_norm):
    # the norm: one rounding to fp32 (64-bit sums lose less than that keeps)
    assert abs(float(norm) - want_norm) <= 2 * U32 * want_norm
    for g, w in zip(got, want):
        # roundings: the factor, its product in fp32, the result's own
        h = half_step(g.dtype)
        most = (2.1 * U32 + h) * w.abs() + torch.finfo(g.dtype).smallest_normal * h
        off = (g.detach().cpu().double() - w).abs()
        assert g.shape == w.shape and bool((off <= most).all())
