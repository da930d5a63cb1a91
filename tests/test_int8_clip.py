"""8-bit rows and products, gradient norm and clipping, on the CPU: the torch
twins against 64 bits, and what both backends refuse."""
import math

import pytest
import torch

import oracle64 as oracle
from distributedes_amd.ops.reference import TorchOps

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ref():
    return TorchOps()


@pytest.fixture(scope="module", params=["torch_ref", "hip"])
def any_ops(request):
    if request.param == "torch_ref":
        return TorchOps()
    from distributedes_amd.ops.hip import HipOps, hip_available
    if not hip_available():
        pytest.skip("extension not built")
    return HipOps()   # with CPU tensors: refusals come before the device's


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (0, 4), (4, 0), (2, 7, 33),
                                   (16,)])
def test_quantize_rows_is_exact(ref, dtype, shape):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(shape, generator=g).to(dtype)
    q, s = ref.quantize_rows(x)
    wq, ws = oracle.codes_and_scale(x)
    assert torch.equal(q, wq) and torch.equal(s, ws)
    assert q.shape == x.shape and s.shape == x.shape[:-1]
    # half a step of the scale is the most that a value may be off
    off = (q.double() * s.double().unsqueeze(-1) - x.double()).abs()
    assert bool((off <= s.double().unsqueeze(-1) * (0.5 + 1e-12)).all())


def test_quantize_rows_borders_and_unusable_rows(ref):
    x = torch.tensor([[127.0, 0.5, 1.5, -0.5, -1.5, 2.5],
                      [0.0, -0.0, 0.0, 0.0, 0.0, 0.0],
                      [1.0, math.nan, 0.0, 0.0, 0.0, 0.0],
                      [1.0, -math.inf, 0.0, 0.0, 0.0, 0.0],
                      [3e38, -3e38, 1e38, 0.0, 0.0, 1.0],
                      [1e-45, 0.0, 1e-40, 0.0, 0.0, 0.0]])
    q, s = ref.quantize_rows(x)
    assert q[0].tolist() == [127, 0, 2, 0, -2, 2]      # ties to even
    assert q[1].tolist() == [0] * 6 and float(s[1]) == 2.0 ** -126
    assert s[2].isnan() and s[3].isnan() and not q[2:4].any()
    assert q[4].tolist() == [127, -127, 42, 0, 0, 0] and s[4].isfinite()
    assert float(s[5]) == 2.0 ** -126 and not q[5].any()


@pytest.mark.parametrize("act", ["none", "relu", "tanh"])
@pytest.mark.parametrize("members", [0, 3])
@pytest.mark.parametrize("out", DTYPES)
def test_products_against_64_bits(ref, act, members, out):
    g = torch.Generator().manual_seed(5)
    lead = (members,) if members else ()
    x = torch.randn(*lead, 7, 33, generator=g)
    wq, sw = ref.quantize_rows(torch.randn(*lead, 9, 33, generator=g))
    b = torch.randn(*lead, 9, generator=g)
    xq, sx = ref.quantize_rows(x)
    want, err = oracle.product(xq, sx, wq, sw, b, act)
    got = ref.int8_matmul(xq, sx, wq, sw, b, act, out)
    oracle.check_product(got, want, err, out)
    assert torch.equal(got, ref.int8_linear(x, wq, sw, b, act, out))
    if not members:                       # one row without an axis of rows
        one = ref.int8_linear(x[2], wq, sw, b, act, out)
        assert torch.equal(one, got[2])


@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9, math.inf])
def test_clip_against_64_bits(ref, max_norm):
    g = torch.Generator().manual_seed(7)
    ts = [torch.randn(5, 3, generator=g), torch.randn(0),
          torch.randn(17, generator=g).bfloat16(),
          torch.randn((), generator=g).half()]
    got, norm = ref.clip_by_global_norm(ts, max_norm)
    oracle.check_clipped(got, norm, *oracle.clipped(ts, max_norm))
    assert float(ref.global_norm(ts)) == float(norm)


def test_clip_of_extreme_values(ref):
    big = [torch.full((4,), 3e38), torch.full((4,), -3e38)]
    got, norm = ref.clip_by_global_norm(big, 1.0)
    assert norm.isinf() and torch.allclose(got[0], torch.full((4,), 8 ** -0.5))
    small = [torch.full((4,), 1e-30)]
    assert float(ref.global_norm(small)) == pytest.approx(2e-30, rel=1e-6)
    bad = [torch.tensor([1.0, math.nan]), torch.tensor([2.0])]
    got, norm = ref.clip_by_global_norm(bad, 1.0)
    assert norm.isnan() and float(got[1]) == 2.0       # left as it is


def _w(n=5, k=4, lead=()):
    return torch.zeros(*lead, n, k, dtype=torch.int8), torch.ones(*lead, n)


@pytest.mark.parametrize("call", [
    lambda o: o.quantize_rows(torch.zeros(3, 4, dtype=torch.float64)),
    lambda o: o.quantize_rows(torch.zeros(3, 4, dtype=torch.int32)),
    lambda o: o.quantize_rows(torch.zeros(())),
    lambda o: o.quantize_rows(torch.zeros(1, 131073)),
    lambda o: o.quantize_rows(torch.zeros(2, 4), out=(
        torch.zeros(2, 5, dtype=torch.int8), torch.zeros(2))),
    lambda o: o.quantize_rows(torch.zeros(2, 4), out=(
        torch.zeros(2, 4, dtype=torch.uint8), torch.zeros(2))),
    lambda o: o.quantize_rows(torch.zeros(2, 4), out=(
        torch.zeros(2, 4, dtype=torch.int8), torch.zeros(3))),
    lambda o: o.int8_linear(torch.zeros(3, 4, dtype=torch.float64), *_w()),
    lambda o: o.int8_linear(torch.zeros(3, 5), *_w()),
    lambda o: o.int8_linear(torch.zeros(3, 4), *_w(lead=(2,))),
    lambda o: o.int8_linear(torch.zeros(3, 1, 4), *_w(lead=(2,))),
    lambda o: o.int8_linear(torch.zeros(3, 4), _w()[0].float(), _w()[1]),
    lambda o: o.int8_linear(torch.zeros(3, 4), _w()[0][0], torch.ones(())),
    lambda o: o.int8_linear(torch.zeros(3, 4), _w()[0], torch.ones(4)),
    lambda o: o.int8_linear(torch.zeros(3, 4), _w()[0], _w()[1].double()),
    lambda o: o.int8_linear(torch.zeros(3, 4), *_w(), bias=torch.zeros(4)),
    lambda o: o.int8_linear(torch.zeros(3, 4), *_w(),
                            bias=torch.zeros(5).half()),
    lambda o: o.int8_linear(torch.zeros(3, 4), *_w(), activation="gelu"),
    lambda o: o.int8_linear(torch.zeros(3, 4), *_w(),
                            out_dtype=torch.float64),
    lambda o: o.int8_linear(torch.zeros(3, 4), *_w(), out=torch.zeros(3, 4)),
    lambda o: o.int8_linear(torch.zeros(3, 4), *_w(),
                            out=torch.zeros(3, 5).half()),
    lambda o: o.int8_linear(torch.zeros(3, 4), *_w(),
                            out=torch.zeros(5, 3).t()),
    lambda o: o.int8_matmul(torch.zeros(3, 4), torch.ones(3), *_w()),
    lambda o: o.int8_matmul(torch.zeros(3, 4, dtype=torch.int8),
                            torch.ones(4), *_w()),
    lambda o: o.int8_matmul(torch.zeros(3, 4, dtype=torch.int8),
                            torch.ones(3).half(), *_w()),
    lambda o: o.int8_matmul(torch.zeros(3, 131073, dtype=torch.int8),
                            torch.ones(3), *_w(k=131073)),
    lambda o: o.global_norm([]),
    lambda o: o.global_norm([torch.zeros(3, dtype=torch.int32)]),
    lambda o: o.clip_by_global_norm([], 1.0),
    lambda o: o.clip_by_global_norm([torch.zeros(3).double()], 1.0),
    lambda o: o.clip_by_global_norm([torch.zeros(3)], -1.0),
    lambda o: o.clip_by_global_norm([torch.zeros(3)], math.nan),
    lambda o: o.clip_by_global_norm([torch.zeros(3)], 1.0, out=[]),
    lambda o: o.clip_by_global_norm([torch.zeros(3)], 1.0,
                                    out=[torch.zeros(4)]),
    lambda o: o.clip_by_global_norm([torch.zeros(3)], 1.0,
                                    out=[torch.zeros(3).half()]),
])
def test_refused(any_ops, call):
    with pytest.raises(ValueError):
        call(any_ops)


def _overlapping():
    buf = torch.zeros(8)
    codes = torch.zeros(64, dtype=torch.int8)
    return [
        # a write that meets another tensor's read or write, or its own read
        lambda o: o.clip_by_global_norm([buf[:4], buf[4:]], 1.0,
                                        out=[buf[4:], torch.zeros(4)]),
        lambda o: o.clip_by_global_norm([buf[:4], buf[4:]], 1.0,
                                        out=[torch.zeros(8)[:4], buf[2:6]]),
        lambda o: o.clip_by_global_norm([buf[:4]], 1.0, out=[buf[1:5]]),
        lambda o: o.clip_by_global_norm([buf[:4], buf[:4]], 1.0,
                                        out=[buf[:4], buf[:4]]),
        lambda o: o.clip_by_global_norm([buf[:4], buf[:4]], 1.0,
                                        out=[buf[:4], torch.zeros(4)]),
        lambda o: o.clip_by_global_norm([buf.view(2, 4).t()], 1.0,
                                        out=[buf.view(2, 4).t()]),
        # rows that run into one another, or hold their values apart
        lambda o: o.quantize_rows(torch.zeros(4, 8), out=(
            codes.as_strided((4, 8), (4, 1)), torch.zeros(4))),
        lambda o: o.quantize_rows(torch.zeros(4, 8), out=(
            codes.as_strided((4, 8), (0, 1)), torch.zeros(4))),
        lambda o: o.quantize_rows(torch.zeros(2, 2, 8), out=(
            codes.as_strided((2, 2, 8), (8, 8, 1)), torch.zeros(2, 2))),
        lambda o: o.quantize_rows(torch.zeros(4, 8), out=(
            codes.as_strided((4, 8), (1, 4)), torch.zeros(4))),
        lambda o: o.quantize_rows(torch.zeros(2, 2, 2, 4), out=(
            codes.as_strided((2, 2, 2, 4), (32, 12, 4, 1)),
            torch.zeros(2, 2, 2))),
        lambda o: o.quantize_rows(buf.view(2, 4), out=(
            buf.view(torch.int8)[:8].view(2, 4), torch.zeros(2))),
        # a gradient that would be lost
        lambda o: o.int8_linear(torch.zeros(3, 4, requires_grad=True), *_w()),
        lambda o: o.quantize_rows(torch.zeros(3, 4, requires_grad=True)),
        lambda o: o.int8_linear(torch.zeros(3, 4), *_w(),
                                bias=torch.zeros(5, requires_grad=True)),
        lambda o: o.global_norm([torch.zeros(3, requires_grad=True)]),
        # results over an argument
        lambda o: o.int8_linear(buf[:4].view(1, 4),
                                torch.zeros(4, 4, dtype=torch.int8),
                                torch.ones(4), out=buf[2:6].view(1, 4)),
    ]


@pytest.mark.parametrize("i", range(17))
def test_refused_by_the_kernels(i):
    from distributedes_amd.ops.hip import HipOps, hip_available
    if not hip_available():
        pytest.skip("extension not built")
    with pytest.raises(ValueError):
        _overlapping()[i](HipOps())


def test_cpu_tensors_are_refused_by_the_kernels():
    from distributedes_amd.ops.hip import HipOps, hip_available
    if not hip_available():
        pytest.skip("extension not built")
    ops = HipOps()
    for call in (lambda: ops.quantize_rows(torch.zeros(2, 3)),
                 lambda: ops.int8_linear(torch.zeros(3, 4), *_w()),
                 lambda: ops.global_norm([torch.zeros(3)]),
                 lambda: ops.clip_by_global_norm([torch.zeros(3)], 1.0)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_every_refusal_is_listed():
    assert len(_overlapping()) == 17


def test_scales_that_require_a_gradient_are_not_written():
    from distributedes_amd.ops.hip import HipOps, hip_available
    if not hip_available():
        pytest.skip("extension not built")
    out = (torch.empty(3, 4, dtype=torch.int8),
           torch.zeros(3, requires_grad=True))
    with pytest.raises(ValueError, match="gradient"):
        HipOps().quantize_rows(torch.zeros(3, 4), out=out)


@pytest.mark.parametrize("members", [0, 3])
def test_products_of_large_rows(ref, members):
    """Sums times the token's scale leave fp32's range, results do not."""
    g = torch.Generator().manual_seed(5)
    lead = (members,) if members else ()
    x = torch.randn(*lead, 7, 3000, generator=g) * 1e36
    x[..., 0, :] = 1e36
    x[..., -1, :] = 1e-3
    wq, sw = ref.quantize_rows(torch.randn(*lead, 9, 3000, generator=g) * 1e-8)
    wq[..., 0, :] = 127
    b = torch.randn(*lead, 9, generator=g)
    xq, sx = ref.quantize_rows(x)
    assert 127.0 * 127.0 * 3000 * float(sx.max()) > 3.4e38
    want, err = oracle.product(xq, sx, wq, sw, b, "none")
    assert bool((want.abs() < 3e38).all())
    oracle.check_product(ref.int8_matmul(xq, sx, wq, sw, b), want, err,
                         torch.float32)


def _leaf(*shape):
    return torch.ones(*shape, requires_grad=True)


@pytest.mark.parametrize("call", [
    lambda o: o.quantize_rows(_leaf(3, 4)),
    lambda o: o.quantize_rows(torch.zeros(3, 4), out=(
        torch.empty(3, 4, dtype=torch.int8), _leaf(3))),
    lambda o: o.int8_linear(_leaf(3, 4), *_w()),
    lambda o: o.int8_linear(torch.zeros(3, 4), _w()[0], _leaf(5)),
    lambda o: o.int8_linear(torch.zeros(3, 4), *_w(), bias=_leaf(5)),
    lambda o: o.int8_linear(torch.zeros(3, 4), *_w(), out=_leaf(3, 5)),
    lambda o: o.int8_matmul(torch.zeros(3, 4, dtype=torch.int8), _leaf(3),
                            *_w()),
    lambda o: o.global_norm([torch.zeros(3), _leaf(3)]),
    lambda o: o.clip_by_global_norm([_leaf(3)], 1.0),
    lambda o: o.clip_by_global_norm([torch.zeros(3)], 1.0, out=[_leaf(3)]),
])
def test_gradients_are_refused_alike(any_ops, call):
    with pytest.raises(ValueError, match="gradient"):
        call(any_ops)
    if any_ops.name != "hip":                  # without one nothing is lost
        with torch.no_grad():
            call(any_ops)


@pytest.mark.parametrize("i", range(17))
def test_refused_by_the_twin(ref, i):
    with pytest.raises(ValueError):
        _overlapping()[i](ref)


@pytest.mark.parametrize("call", [
    lambda o: o.clip_by_global_norm([torch.zeros(2, 4)], 1.0,
                                    out=[torch.zeros(4, 2).t()]),
    lambda o: o.quantize_rows(torch.zeros(3, 4), out=(
        torch.empty(3, 4, dtype=torch.int8), torch.zeros(6)[::2])),
    lambda o: (lambda y: o.int8_matmul(
        torch.zeros(4, 4, dtype=torch.int8), y.view(-1)[2:6],
        *_w(4), out=y))(torch.zeros(4, 4)),
])
def test_outputs_refused_alike(any_ops, call):
    with pytest.raises(ValueError):
        call(any_ops)


def test_nothing_is_written_where_one_output_is_refused(ref):
    good, bad = torch.full((3,), 9.0), torch.zeros(4)
    with pytest.raises(ValueError):
        ref.clip_by_global_norm([torch.ones(3)] * 2, 1.0, out=[good, bad])
    assert bool((good == 9).all())


def test_the_twin_takes_what_lies_apart(ref):
    """In place, side by side, rows between bytes that stay."""
    buf = torch.arange(1.0, 9.0)
    ts = [buf[:3], buf[3:3], buf[3:]]
    want, norm = oracle.clipped(ts, 1.0)
    got, n = ref.clip_by_global_norm(ts, 1.0, out=ts)
    oracle.check_clipped(got, n, want, norm)
    x = torch.randn(2, 3, 4, generator=torch.Generator().manual_seed(1))
    store = torch.full((64,), 99, dtype=torch.int8)
    for shape in ((24, 8, 1), (4, 8, 1), (30, 4, 1)):
        q, s = store.as_strided((2, 3, 4), shape, 1), torch.empty(2, 3)
        ref.quantize_rows(x, out=(q, s))
        wq, ws = oracle.codes_and_scale(x)
        assert torch.equal(q, wq) and torch.equal(s, ws)
        q.fill_(99)
        assert bool((store == 99).all())


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_gradients_are_refused_alike(any_ops, grad):
    import torch.autograd.forward_ad as forward_ad
    z = torch.zeros
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = lambda *s: forward_ad.make_dual(z(*s), torch.ones(*s))
        for call in (
                lambda: any_ops.quantize_rows(dual(3, 4)),
                lambda: any_ops.quantize_rows(z(3, 4), out=(
                    z(3, 4, dtype=torch.int8), dual(3))),
                lambda: any_ops.int8_linear(dual(3, 4), *_w()),
                lambda: any_ops.int8_linear(z(3, 4), _w()[0], dual(5)),
                lambda: any_ops.int8_linear(z(3, 4), *_w(), bias=dual(5)),
                lambda: any_ops.int8_linear(z(3, 4), *_w(), out=dual(3, 5)),
                lambda: any_ops.int8_matmul(z(3, 4, dtype=torch.int8),
                                            dual(3), *_w()),
                lambda: any_ops.global_norm([dual(3)]),
                lambda: any_ops.clip_by_global_norm([z(3), dual(3)], 1.0),
                lambda: any_ops.clip_by_global_norm([z(3)], 1.0,
                                                    out=[dual(3)])):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


def _negated(t):
    """A view of -t's memory that torch negates when it reads it."""
    view = torch.complex(torch.zeros_like(t, dtype=torch.float32),
                         -t.float()).conj().imag
    assert view.is_neg()
    return view


@pytest.mark.parametrize("call", [
    lambda o: o.quantize_rows(torch.zeros(3, 1), out=(
        torch.empty(3, 1, dtype=torch.int8), _negated(torch.ones(1)).expand(3))),
    lambda o: o.int8_linear(torch.zeros(1, 4), *_w(1),
                            out=_negated(torch.zeros(1, 1))),
    lambda o: o.clip_by_global_norm([torch.zeros(1)], 1.0,
                                    out=[_negated(torch.zeros(1))]),
])
def test_negated_views_are_not_written(any_ops, call):
    with pytest.raises(ValueError):
        call(any_ops)
