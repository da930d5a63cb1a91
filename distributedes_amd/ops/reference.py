"""Pure-torch reference twins of every HIP kernel.

These are (a) the CPU execution path, (b) the eager-GPU self-baseline the
hand kernels are measured against, and (c) the oracles for kernel parity
tests.  Member-chunked so the GPU eager path never materializes pop x dim
index tensors beyond `chunk` rows.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from ..core import noise as noise_mod

_MAX_COLS = 131072     # int32 sums of 127 * 127 stay in range
_ELEMS = (torch.float32, torch.bfloat16, torch.float16)
_ACTS = ("none", "relu", "tanh")


def _want(ok, message):
    if not ok:
        raise ValueError(message)


def _want_no_grad(**tensors):
    for name, t in tensors.items():
        _want(t is None or not (t.requires_grad and torch.is_grad_enabled()),
              f"{name} requires a gradient, and this operator has none")
        _want(t is None or forward_ad.unpack_dual(t).tangent is None,
              f"{name} carries a forward-mode gradient, and this operator has "
              "none")


def _want_plain(*out):
    _want(not any(o.is_neg() for o in out), "out must not be a negated view")


def _span(t):
    """The bytes that a tensor spans: [begin, end)."""
    if t.numel() == 0:
        return t.data_ptr(), t.data_ptr()
    last = sum((n - 1) * step for n, step in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlap(a, b):
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1 and a0 < a1 and b0 < b1


def _rows_apart(t):
    """Whether a tensor that is written holds its rows apart from one another,
    by two strides and with a last stride of 1."""
    cols = t.shape[-1]
    if 0 in t.shape[:-1]:                    # no rows
        return True
    if cols > 1 and t.stride(-1) != 1:
        return False
    groups = []                              # (size, step), inside out
    for n, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if groups and step == groups[-1][0] * groups[-1][1]:
            groups[-1] = (groups[-1][0] * n, groups[-1][1])
        else:
            groups.append((n, step))
    room = cols
    for n, step in sorted((g for g in groups if g[0] > 1), key=lambda g: g[1]):
        if step < room:
            return False
        room += step * (n - 1)
    return len(groups) <= 2


def _want_apart(tensors, out):
    """A write may meet no other write, and no read but that of its own tensor,
    in place."""
    uses = []
    for i, (t, o) in enumerate(zip(tensors, out)):
        if o.numel():
            uses.append((*_span(o), i, True))
            if _span(t) != _span(o):
                uses.append((*_span(t), i, False))
    written = read = 0
    for begin, end, i, write in sorted(uses):
        _want(begin >= written and (not write or begin >= read),
              f"out[{i}] overlaps another tensor")
        if write:
            written = max(written, end)
        else:
            read = max(read, end)


def _want_product(x, wq, sw, bias, activation, out_dtype, out):
    _want_no_grad(x=x, sw=sw, bias=bias, out=out)
    _want(wq.dtype == torch.int8, "wq must be int8")
    _want(wq.dim() in (2, 3),
          "wq must be [channels, cols] or [members, channels, cols]")
    _want(wq.dim() == 2 or x.dim() == 3,
          "members' weights need x of [members, tokens, cols]")
    _want(x.shape[-1] == wq.shape[-1], "x and wq differ in cols")
    _want(wq.dim() == 2 or x.shape[0] == wq.shape[0],
          "x and wq differ in members")
    _want(x.shape[-1] <= _MAX_COLS, f"rows of at most {_MAX_COLS} values")
    _want(sw.dtype == torch.float32 and sw.shape == wq.shape[:-1],
          "sw must be float32 of wq's shape without its last dimension")
    _want(bias is None or (bias.dtype == torch.float32
                           and bias.shape == sw.shape),
          "bias must be float32 of sw's shape")
    _want(activation in _ACTS, "activation must be none, relu or tanh")
    _want(out_dtype in _ELEMS, "out_dtype must be float32, bfloat16 or float16")
    _want(out is None or (out.dtype == out_dtype and out.is_contiguous()
                          and out.shape == (*x.shape[:-1], wq.shape[-2])),
          "out must be contiguous, of out_dtype and of the result's shape")
    if out is not None:
        _want_plain(out)
    _want(out is None or not any(_overlap(out, t) for t in (x, wq, sw, bias)
                                 if t is not None),
          "out overlaps an argument")


class TorchOps:
    name = "torch_ref"

    # --- K1 ---------------------------------------------------------------
    def fill_table(self, size: int, seed: int, device,
                   dtype=torch.float32) -> torch.Tensor:
        t = noise_mod.fill_noise_table_cpu(size, seed)
        return t.to(dtype).to(device)

    # --- K2: theta_i = theta + sigma * sign_i * table[off_i : off_i+D] ----
    def perturb(self, theta: torch.Tensor, table: torch.Tensor,
                offsets: torch.Tensor, signs: torch.Tensor, sigma: float,
                sigma_vec: torch.Tensor = None, out_dtype=torch.float32,
                chunk: int = 256) -> torch.Tensor:
        """offsets [P] int64 (device), signs [P] fp32 -> [P, D] out_dtype.
        sigma_vec [D] (CEM) overrides scalar sigma per-coordinate."""
        P = offsets.shape[0]
        D = theta.shape[0]
        out = torch.empty(P, D, dtype=out_dtype, device=theta.device)
        ar = torch.arange(D, device=theta.device)
        for s in range(0, P, chunk):
            e = min(s + chunk, P)
            idx = offsets[s:e].unsqueeze(1) + ar
            eps = table[idx].to(torch.float32)              # [c, D]
            eps.mul_(signs[s:e].unsqueeze(1))
            if sigma_vec is not None:
                eps.mul_(sigma_vec)
            else:
                eps.mul_(sigma)
            out[s:e] = (theta + eps).to(out_dtype)
        return out

    # --- K10: partial weighted noise sum (the ES "backward") --------------
    def weighted_noise_sum(self, table: torch.Tensor, offsets: torch.Tensor,
                           signs: torch.Tensor, weights: torch.Tensor,
                           dim: int, want_sq: bool = False, chunk: int = 256):
        """returns sum_i w_i * s_i * eps_i  [D] fp32 (and optionally
        sum_i w_i * eps_i^2 for the CEM variance refit)."""
        dev = table.device
        acc = torch.zeros(dim, dtype=torch.float32, device=dev)
        acc_sq = torch.zeros(dim, dtype=torch.float32, device=dev) if want_sq else None
        ar = torch.arange(dim, device=dev)
        P = offsets.shape[0]
        for s in range(0, P, chunk):
            e = min(s + chunk, P)
            idx = offsets[s:e].unsqueeze(1) + ar
            eps = table[idx].to(torch.float32)              # [c, D]
            w = weights[s:e].unsqueeze(1)
            acc += (eps * (w * signs[s:e].unsqueeze(1))).sum(dim=0)
            if want_sq:
                acc_sq += (eps * eps * w).sum(dim=0)
        return (acc, acc_sq) if want_sq else acc

    # --- 8-bit rows and products (see ops/hip.py for the definitions) ------
    def quantize_rows(self, x, out=None):
        _want(x.dtype in _ELEMS, "x must be float32, bfloat16 or float16")
        _want(x.dim() >= 1, "x must have at least one dimension")
        _want(x.shape[-1] <= _MAX_COLS, f"rows of at most {_MAX_COLS} values")
        _want_no_grad(x=x)
        if out is not None:
            _want_no_grad(out=out[1])
            _want_plain(*out)
            _want(out[0].dtype == torch.int8 and out[0].shape == x.shape,
                  "out[0] must be int8 of x's shape")
            _want(out[1].dtype == torch.float32
                  and out[1].shape == x.shape[:-1] and out[1].is_contiguous(),
                  "out[1] must be contiguous float32 of x's shape without its "
                  "last dimension")
            _want(_rows_apart(out[0]),
                  "out[0] must hold its rows apart, by two strides and with a "
                  "last stride of 1")
            _want(not (_overlap(out[0], x) or _overlap(out[1], x)
                       or _overlap(*out)), "out overlaps x or itself")
        v = x.detach().to(torch.float64)
        top = (v.abs().amax(dim=-1) if x.shape[-1]
               else v.new_zeros(x.shape[:-1]))
        scale = (top / 127).to(torch.float32).clamp_min(2.0 ** -126)
        bad = ~torch.isfinite(top)
        scale = torch.where(bad, torch.full_like(scale, float("nan")), scale)
        codes = (v / scale.to(torch.float64).unsqueeze(-1)).round()
        codes = codes.masked_fill(bad.unsqueeze(-1), 0).to(torch.int8)
        if out is None:
            return codes, scale
        out[0].copy_(codes)
        out[1].copy_(scale)
        return out

    def int8_matmul(self, xq, sx, wq, sw, bias=None, activation="none",
                    out_dtype=torch.float32, out=None):
        _want(xq.dtype == torch.int8, "xq must be int8")
        _want(xq.dim() >= 1, "xq must have at least one dimension")
        _want(sx.dtype == torch.float32 and sx.shape == xq.shape[:-1],
              "sx must be float32 of xq's shape without its last dimension")
        _want_no_grad(sx=sx)
        _want_product(xq, wq, sw, bias, activation, out_dtype, out)
        _want(out is None or not _overlap(out, sx), "out overlaps an argument")
        if xq.dim() == 1:                    # one row, no axis of rows
            y = self.int8_matmul(xq[None], sx[None], wq, sw, bias, activation,
                                 out_dtype)[0]
            return y if out is None else out.copy_(y)
        # whole numbers below 2^53: the sums are exact in any order
        y = xq.to(torch.float64) @ wq.to(torch.float64).transpose(-1, -2)
        # 64 bits: sum * sx may leave fp32's range where the result does not
        y = y * sx.to(torch.float64).unsqueeze(-1)
        y = y * sw.to(torch.float64).unsqueeze(-2)
        if bias is not None:
            y = y + bias.to(torch.float64).unsqueeze(-2)
        y = y.to(torch.float32)
        if activation == "relu":
            y = y.clamp_min(0)
        elif activation == "tanh":
            y = y.tanh()
        return y.to(out_dtype) if out is None else out.copy_(y)

    def int8_linear(self, x, wq, sw, bias=None, activation="none",
                    out_dtype=torch.float32, out=None):
        _want(out is None or not _overlap(out, x), "out overlaps an argument")
        return self.int8_matmul(*self.quantize_rows(x), wq, sw, bias,
                                activation, out_dtype, out)

    # --- gradient norm ----------------------------------------------------
    def global_norm(self, tensors):
        return self._norm64(tensors).to(torch.float32)

    @staticmethod
    def _norm64(tensors):
        _want(len(tensors) > 0, "no tensors")
        for t in tensors:
            _want(t.dtype in _ELEMS,
                  "tensors must be float32, bfloat16 or float16")
            _want_no_grad(tensors=t)
        return torch.stack([t.to(torch.float64).square().sum()
                            for t in tensors]).sum().sqrt()

    def clip_by_global_norm(self, tensors, max_norm, out=None):
        norm = self._norm64(tensors)
        _want(max_norm >= 0, "max_norm must be at least 0")
        if out is not None:
            _want(len(out) == len(tensors), "out must hold as many tensors")
            for o, t in zip(out, tensors):
                _want_no_grad(out=o)
                _want_plain(o)
                _want(o.dtype == t.dtype and o.shape == t.shape
                      and o.is_contiguous(),
                      "out must be contiguous, of its tensor's type and shape")
            _want_apart(tensors, out)
        c = torch.where(norm > max_norm, max_norm / norm,
                        torch.ones_like(norm))
        clipped = [(t.to(torch.float64) * c).to(t.dtype) for t in tensors]
        if out is not None:
            for o, t in zip(out, clipped):
                o.copy_(t)
            clipped = list(out)
        return clipped, norm.to(torch.float32)
