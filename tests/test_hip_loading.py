"""The two HIP extensions load apart: without the one of the 8-bit rows and
gradient norms everything else is there, and its operators say what is missing."""
import sys

import pytest
import torch

from distributedes_amd import preset
from distributedes_amd.core import engine
from distributedes_amd.ops import hip


@pytest.fixture
def without_second(monkeypatch):
    if not hip.hip_available():
        pytest.skip("extension not built")
    for name in ("_ext", "_ext2", "_err", "_err2"):
        monkeypatch.setattr(hip, name, None, raising=False)
    for name in ("distributedes_amd.ops._hip_ops2", "_hip_ops2"):
        monkeypatch.setitem(sys.modules, name, None)   # an ImportError
    import distributedes_amd.ops as package
    monkeypatch.delattr(package, "_hip_ops2", raising=False)


def test_the_first_extension_stands_alone(without_second):
    assert hip.hip_available() and hip.load_error() is None
    ops = hip.HipOps()
    assert ops.ext is not None
    w = torch.zeros(5, 4, dtype=torch.int8), torch.ones(5)
    for call in (lambda: ops.quantize_rows(torch.zeros(3, 4)),
                 lambda: ops.int8_linear(torch.zeros(3, 4), *w),
                 lambda: ops.int8_matmul(w[0], w[1], *w),
                 lambda: ops.global_norm([torch.zeros(3)]),
                 lambda: ops.clip_by_global_norm([torch.zeros(3)], 1.0)):
        with pytest.raises(RuntimeError, match="_hip_ops2"):
            call()


@pytest.mark.parametrize("kw", [dict(precision="int8"),
                                dict(max_grad_norm=0.5)])
def test_training_that_needs_the_second_does_not_begin(without_second,
                                                       monkeypatch, kw):
    monkeypatch.setattr(engine, "_make_ops", lambda *a: hip.HipOps())
    cfg = preset("cartpole_es", pop=8, device="cpu", noise_table_size=1 << 16,
                 **kw)
    with pytest.raises(RuntimeError, match="_hip_ops2"):
        engine.TrainState(cfg)
