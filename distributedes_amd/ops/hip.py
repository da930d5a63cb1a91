"""HIP kernel backend: loads the in-tree gfx950 extensions.

The extensions are built IN-TREE (setup.py build_ext --inplace -> _hip_ops.so
and _hip_ops2.so next to this file) so the .so ship with the repo snapshot to
GPU boxes.
On a GPU box, ops FAIL LOUDLY if the extension is missing — no silent
eager fallback (the engine enforces this in _make_ops).
"""
from __future__ import annotations

import importlib

import torch

_ext = None
_ext2 = None
_err = None
_err2 = None


def _import(name):
    """(module, None) or (None, why not)."""
    try:
        return importlib.import_module("." + name, __package__), None
    except ImportError as e:
        try:
            return importlib.import_module(name), None
        except ImportError:
            return None, e


def _load():
    global _ext, _ext2, _err, _err2
    if _ext is None and _err is None:
        _ext, _err = _import("_hip_ops")
        # 8-bit rows and products, gradient norm: whoever calls none of them
        # does without it
        _ext2, _err2 = _import("_hip_ops2")
    return _ext


def hip_available() -> bool:
    return _load() is not None


def load_error():
    _load()
    return _err


class HipOps:
    """Same surface as ops.reference.TorchOps, backed by CDNA4 HIP kernels."""

    name = "hip"

    def __init__(self):
        self.ext = _load()
        if self.ext is None:
            raise RuntimeError(f"HIP extension not built: {_err}")

    @property
    def ext2(self):
        if _ext2 is None:
            raise RuntimeError("HIP extension for 8-bit rows and gradient "
                               f"norms (_hip_ops2) not built: {_err2}")
        return _ext2

    # K1
    def fill_table(self, size: int, seed: int, device,
                   dtype=torch.float32) -> torch.Tensor:
        t = torch.empty(size, dtype=dtype, device=device)
        self.ext.noise_fill(t, seed)
        return t

    # K2
    def perturb(self, theta, table, offsets, signs, sigma,
                sigma_vec=None, out_dtype=torch.float32, chunk=None,
                pad_rows: bool = False, out=None):
        """pad_rows: allocate [P, pad16(D)] so every member row is 16B-aligned
        for the vectorized policy-forward kernels (pad tail is unwritten).
        out: reuse a persistent buffer (stable pointer for hipGraph replay)."""
        P = offsets.shape[0]
        D = theta.shape[0]
        stride = (D + 7) & ~7 if pad_rows else D
        if out is None or out.shape != (P, stride) or out.dtype != out_dtype:
            out = torch.empty(P, stride, dtype=out_dtype, device=theta.device)
        self.ext.perturb(out, theta, table, offsets, signs, float(sigma),
                         sigma_vec if sigma_vec is not None else
                         torch.empty(0, device=theta.device))
        return out

    # K10
    def weighted_noise_sum(self, table, offsets, signs, weights, dim,
                           want_sq=False, chunk=None):
        acc = torch.zeros(dim, dtype=torch.float32, device=table.device)
        acc_sq = (torch.zeros(dim, dtype=torch.float32, device=table.device)
                  if want_sq else torch.empty(0, device=table.device))
        self.ext.weighted_noise_sum(acc, acc_sq, table, offsets, signs,
                                    weights, bool(want_sq))
        return (acc, acc_sq) if want_sq else acc

    # --- 8-bit rows and products -----------------------------------------
    # No gradient passes through these: the framework estimates its gradients
    # from forward passes.  An argument that requires one, or carries one of
    # forward mode, is refused.  A write to `out` counts as a write for autograd.
    # `out` overlaps no argument, unless said otherwise.

    def quantize_rows(self, x, out=None):
        """x [..., K] (fp32/bf16/fp16, K <= 131072) -> (codes [..., K] int8,
        scale [...] fp32), with x ~ codes * scale: one scale a row,
        max(fp32(max|x| / 127), 2^-126), and codes the whole numbers nearest
        to x / scale, ties to even.  A row that holds a NaN or an infinity
        gets scale NaN and codes 0.

        Fresh codes have rows that begin at multiples of 16 bytes, or of 128
        where that adds 1/16 at most.
        out: (codes, scale) to write to; the codes' rows may lie anywhere
        apart from one another (bytes between them are left as they were)."""
        q, s = out if out is not None else (None, None)
        return self.ext2.quantize_rows(x, q, s)

    def int8_matmul(self, xq, sx, wq, sw, bias=None, activation="none",
                    out_dtype=torch.float32, out=None):
        """act(sum_k xq[m, k] wq[n, k] * sx[m] * sw[n] + bias[n]): codes in
        [-127, 127] and scales on both sides, as quantize_rows gives them; sums
        are exact in int32, and their scaling stays in range wherever the result
        does.

        One policy: xq [..., K] with wq [N, K] -> [..., N].  Members with
        weights of their own: xq [B, M, K] with wq [B, N, K] -> [B, M, N].
        sx, sw, bias: fp32, shaped like the rows they belong to.
        activation: none | relu | tanh.  out_dtype: fp32 | bf16 | fp16.
        out: a contiguous tensor to write to."""
        return self.ext2.int8_matmul(xq, sx, wq, sw, bias, activation,
                                     out_dtype, out)

    def int8_linear(self, x, wq, sw, bias=None, activation="none",
                    out_dtype=torch.float32, out=None):
        """int8_matmul of quantize_rows(x): x fp32/bf16/fp16."""
        return self.ext2.int8_linear(x, wq, sw, bias, activation, out_dtype,
                                     out)

    # --- gradient norm ----------------------------------------------------
    def global_norm(self, tensors):
        """sqrt of the sum of squares over all tensors (fp32/bf16/fp16, mixed
        as they come), summed in fp64 -> fp32 scalar tensor."""
        return self.ext2.global_norm(tensors)

    def clip_by_global_norm(self, tensors, max_norm, out=None):
        """-> ([t * c for t in tensors], norm), with c = max_norm / norm (fp64)
        where norm > max_norm, else 1; the norm stays on the GPU.  A NaN norm
        leaves the values as they are, an infinite one gives c = 0.
        out: contiguous tensors to write to (the tensors themselves clip in
        place)."""
        clipped, norm = self.ext2.clip_by_global_norm(tensors, max_norm, out)
        return (clipped if out is None else list(out)), norm
