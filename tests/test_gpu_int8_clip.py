"""8-bit rows and products, gradient norm and clipping: the HIP kernels against
64 bits at the sizes, strides and values where they can go wrong."""
import math

import pytest
import torch

import oracle64 as oracle

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs MI355X", allow_module_level=True)

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    from distributedes_amd.ops.hip import HipOps, hip_available, load_error
    assert hip_available(), load_error()
    return HipOps()


def _rand(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _check_codes(x, q, s):
    wq, ws = oracle.codes_and_scale(x)
    assert torch.equal(q.cpu(), wq)
    assert torch.equal(s.cpu().nan_to_num(7.0), ws.nan_to_num(7.0))


# ------------------------------------------------------------------ rows ---
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [
    (1, 1), (5, 1), (3, 2), (1000, 4), (7, 15), (9, 16), (33, 17), (64, 64),
    (65, 63), (5, 127), (11, 128), (3, 255), (6, 376), (4, 512), (2, 513),
    (3, 1023), (3, 1024), (2, 1025), (2, 2049), (2, 3136), (3, 4097),
    (2, 8193), (1, 16384), (1, 16385), (1, 40001), (2, 131072), (0, 8),
    (8, 0), (600, 300), (513, 1100), (520, 4100), (515, 20003), (512, 33000)])
def test_quantize_rows_sizes(ops, dtype, rows, cols):
    x = _rand(rows, cols, seed=rows + cols, dtype=dtype)
    _check_codes(x, *ops.quantize_rows(x))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows_borders(ops, dtype):
    """Values on and next to the border of two codes."""
    k = torch.arange(-126, 127, device="cuda").float() + 0.5
    rows = []
    for top in (127.0, 254.0, 1016.0):        # scales 1, 2, 8: ties are exact
        v = (k * (top / 127)).to(dtype)
        rows.append(torch.cat([v, torch.tensor([top], device="cuda").to(dtype)]))
    x = torch.stack(rows)
    _check_codes(x, *ops.quantize_rows(x))
    y = _rand(64, 1, seed=1).abs() + 0.5      # scales with every bit in use
    v = (y / 127) * k[None, :]
    for z in (v, torch.nextafter(v, v.new_tensor(math.inf)),
              torch.nextafter(v, v.new_tensor(-math.inf))):
        z = torch.cat([z, y], 1).to(dtype)
        _check_codes(z, *ops.quantize_rows(z))


@pytest.mark.parametrize("cols", [3, 70, 700, 9000])
def test_quantize_rows_extreme_values(ops, cols):
    x = _rand(12, cols, seed=2)
    x[0] = 0
    x[1] = -0.0
    x[2, cols // 2] = math.nan
    x[3, cols - 1] = math.inf
    x[4, 0] = -math.inf
    x[5] *= 3e37
    x[6] *= 1e-38
    x[7] *= 1e-44
    x[8, :-1] = 0
    x[9] = 3.4028234e38
    x[10] = 1.1754944e-38
    x[11] *= 1e-35
    _check_codes(x, *ops.quantize_rows(x))


def test_quantize_rows_strides_and_out(ops):
    pop = _rand(6, 1003, seed=3)               # members' flat rows, odd step
    for off, n, k in ((0, 9, 33), (7, 5, 64), (1, 16, 16), (3, 1, 1000)):
        x = pop[:, off:off + n * k].unflatten(1, (n, k))
        _check_codes(x, *ops.quantize_rows(x))
        # codes side by side, between bytes that have to stay
        buf = torch.full((6, n * (k + 3) + 5), 99, dtype=torch.int8,
                         device="cuda")
        q = buf[:, 1:1 + n * (k + 3)].unflatten(1, (n, k + 3))[..., :k]
        s = torch.empty(6, n, device="cuda")
        got = ops.quantize_rows(x, out=(q, s))
        assert got[0].data_ptr() == q.data_ptr()
        _check_codes(x, q, s)
        q.fill_(99)
        assert bool((buf == 99).all())
    t = _rand(40, 24, seed=4).t()              # last stride is not 1
    _check_codes(t, *ops.quantize_rows(t))
    e = _rand(1, 50, seed=5).expand(7, 50)
    _check_codes(e, *ops.quantize_rows(e))
    f = _rand(3, 4, 5, 37, seed=6).transpose(0, 2)   # three strides
    _check_codes(f, *ops.quantize_rows(f))
    # x in two groups, out in one, and the other way round
    y = _rand(4, 6, 40, seed=7)[:, :5, :]
    q = torch.empty(4, 5, 40, dtype=torch.int8, device="cuda")
    _check_codes(y, *ops.quantize_rows(y, out=(q, torch.empty(4, 5,
                                                              device="cuda"))))
    z = _rand(4, 5, 40, seed=8)
    q = torch.empty(4, 9, 40, dtype=torch.int8, device="cuda")[:, 2:7]
    _check_codes(z, *ops.quantize_rows(z, out=(q, torch.empty(4, 5,
                                                              device="cuda"))))


def test_quantize_rows_behind_32_bits(ops):
    x = torch.zeros(1100, 2_000_003, dtype=torch.bfloat16, device="cuda")
    v = x[:, 11:11 + 48].unflatten(1, (3, 16))
    v[:] = _rand(1100, 3, 16, seed=9).bfloat16()
    _check_codes(v, *ops.quantize_rows(v))


# --------------------------------------------------------------- products ---
def _weights(ops, n, k, lead=(), seed=1):
    return ops.quantize_rows(_rand(*lead, n, k, seed=seed) / max(1, k) ** 0.5)


def _check_both(ops, x, wq, sw, bias, act, out_dtype):
    q, s = oracle.codes_and_scale(x)
    want, err = oracle.product(q, s, wq, sw, bias, act)
    got = ops.int8_linear(x, wq, sw, bias, act, out_dtype)
    assert got.dtype == out_dtype
    oracle.check_product(got, want, err, out_dtype)
    xq, sx = ops.quantize_rows(x)
    same = ops.int8_matmul(xq, sx, wq, sw, bias, act, out_dtype)
    assert torch.equal(same.nan_to_num(7.0), got.nan_to_num(7.0))
    return got


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 2, 64), (1, 64, 4), (2, 3, 5), (1, 17, 256), (1, 512, 3136),
    (15, 16, 17), (16, 16, 64), (17, 15, 63), (16, 512, 3136), (33, 65, 129),
    (48, 31, 200), (63, 64, 65), (64, 129, 376), (65, 127, 64), (100, 70, 31),
    (127, 257, 130), (128, 128, 128), (129, 256, 192), (200, 500, 1000),
    (255, 64, 4097), (256, 256, 256), (257, 255, 257), (300, 1, 300),
    (1000, 512, 3136), (1025, 513, 513), (3, 4096, 4096), (70, 40, 20000),
    (5, 6, 131072), (600, 260, 0), (3, 5, 0), (4000, 4500, 0), (0, 4, 4), (4, 0, 4), (2500, 1, 1),
    (1, 3000, 77)])
def test_product_sizes(ops, m, n, k):
    x = _rand(m, k, seed=m + n + k)
    wq, sw = _weights(ops, n, k)
    bias = _rand(n, seed=2)
    _check_both(ops, x, wq, sw, bias, "none", torch.float32)


@pytest.mark.parametrize("m,n,k", [
    (4099, 4090, 300), (4096, 4096, 128), (8190, 2049, 77), (5, 900, 9000),
    (4099, 2050, 515), (2048, 4096, 64), (16400, 250, 129), (16390, 64, 385),
    (513, 4097, 256), (700, 1500, 1)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_product_large_tiles(ops, m, n, k, out):
    """Results enough for each size of tile, edges in both directions."""
    x = _rand(m, k, seed=m + n + k)
    wq, sw = _weights(ops, n, k)
    bias = _rand(n, seed=2)
    act = "tanh" if out == torch.float32 and k < 100 else "relu"
    _check_both(ops, x, wq, sw, bias, act, out)


def _sampled(ops, b, m, n, k, packed=False, seed=1):
    """Many members, a few of them against 64 bits."""
    step = k if packed else (k + 15) // 16 * 16
    store = torch.randint(-127, 128, (b * n * step,), dtype=torch.int8,
                          device="cuda",
                          generator=torch.Generator("cuda").manual_seed(seed))
    wq = store.view(b, n, step)[:, :, :k]
    sw, bias = torch.rand(b, n, device="cuda") / 127, _rand(b, n, seed=3)
    x = _rand(b, m, k, seed=4)
    at = sorted({0, 1, b // 3, b // 2, b - 2, b - 1})
    q, s = oracle.codes_and_scale(x[at])
    want, err = oracle.product(q, s, wq[at], sw[at], bias[at], "none")
    got = ops.int8_linear(x, wq, sw, bias)
    oracle.check_product(got[at], want, err, torch.float32)
    xq, sx = ops.quantize_rows(x)
    assert torch.equal(ops.int8_matmul(xq, sx, wq, sw, bias), got)


@pytest.mark.parametrize("m", [1, 3])
@pytest.mark.parametrize("b,n,k,packed", [
    (9000, 100, 376, False), (9000, 100, 375, True), (9000, 101, 384, False),
    (900, 100, 3136, False), (900, 101, 3137, True), (900, 100, 3200, False),
    (300, 70, 2000, False), (1000, 200, 250, True), (3000, 210, 60, False),
    (9000, 300, 16, False), (9000, 300, 13, True), (20000, 110, 33, True)])
def test_member_products_as_streams(ops, b, m, n, k, packed):
    """Weights of 33 MB to 400 MB: every way of the stream of weights."""
    _sampled(ops, b, m, n, k, packed)


@pytest.mark.parametrize("b,m,n,k,packed", [
    (1000, 16, 130, 376, False), (1000, 5, 130, 375, True),
    (700, 20, 130, 376, False), (700, 31, 129, 375, True),
    (100, 40, 129, 375, True), (60, 70, 300, 500, False),
    (20, 300, 500, 129, True)])
def test_member_products_of_more_tokens(ops, b, m, n, k, packed):
    _sampled(ops, b, m, n, k, packed)


@pytest.mark.parametrize("b,m,n,k", [
    (1, 1, 1, 1), (16, 1, 64, 64), (16, 1, 64, 4), (5, 1, 2, 64),
    (7, 1, 17, 256), (3, 1, 256, 376), (2, 2, 512, 3136), (3, 16, 33, 65),
    (4, 17, 40, 100), (2, 65, 130, 70), (3, 130, 129, 257), (2, 300, 300, 300),
    (0, 1, 4, 4), (4, 1, 6, 0), (3, 40, 6, 0), (300, 1, 3, 3), (2, 5, 6, 70000), (70000, 1, 1, 3)])
def test_member_product_sizes(ops, b, m, n, k):
    x = _rand(b, m, k, seed=b + m + n + k)
    wq, sw = _weights(ops, n, k, (b,))
    bias = _rand(b, n, seed=2)
    _check_both(ops, x, wq, sw, bias, "none", torch.float32)


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "relu", "tanh"])
@pytest.mark.parametrize("lead,m", [((), 1), ((), 70), ((), 300), ((5,), 1),
                                    ((2,), 40)])
def test_product_types_and_activations(ops, out, dtype, act, lead, m):
    x = _rand(*lead, m, 72, seed=3, dtype=dtype)
    wq, sw = _weights(ops, 50, 72, lead)
    bias = _rand(*lead, 50, seed=4)
    _check_both(ops, x, wq, sw, bias, act, out)
    _check_both(ops, x, wq, sw, None, act, out)


@pytest.mark.parametrize("m", [1, 20, 200, 600, 7000])
def test_product_largest_sums(ops, m):
    """Codes of 127 throughout: 131072 * 127^2 is just inside 32 bits."""
    k = 131072
    x = torch.ones(m, k, device="cuda")
    x[-1] = -1
    wq = torch.full((3, k), 127, dtype=torch.int8, device="cuda")
    sw = torch.ones(3, device="cuda")
    got = ops.int8_linear(x, wq, sw)
    want = 127.0 * k * torch.ones(m, 3, device="cuda")
    want[-1] *= -1
    torch.testing.assert_close(got, want, rtol=4 * oracle.U32, atol=0)


@pytest.mark.parametrize("m,n,k", [(1, 40, 33), (9, 33, 65), (70, 70, 70),
                                   (300, 200, 131), (300, 300, 256)])
def test_product_strides(ops, m, n, k):
    """Rows at odd addresses and steps, the last byte at its storage's end."""
    wf, sw = _weights(ops, n, k, seed=5)
    xf, sx = _weights(ops, m, k, seed=6)
    bias = _rand(n, seed=7)
    want, err = oracle.product(xf, sx, wf, sw, bias, "none")

    def laid(t, off, step):
        buf = torch.full((off + (t.shape[0] - 1) * step + k,), 77,
                         dtype=torch.int8, device="cuda")
        v = buf.as_strided(t.shape, (step, 1), off)
        v.copy_(t)
        return v

    for off, step in ((0, k), (1, k), (3, k + 5), (16, (k + 15) // 16 * 16),
                      (0, (k + 127) // 64 * 64)):
        for xo, xs in ((0, k), (5, k + 1), (32, (k + 15) // 16 * 16)):
            got = ops.int8_matmul(laid(xf, xo, xs), sx, laid(wf, off, step),
                                  sw, bias)
            oracle.check_product(got, want, err, torch.float32)
    t = wf.t().contiguous().t()                # last stride is not 1
    got = ops.int8_matmul(xf.t().contiguous().t(), sx, t, sw, bias)
    oracle.check_product(got, want, err, torch.float32)


def test_product_broadcast_and_more_dimensions(ops):
    wq, sw = _weights(ops, 30, 48)
    bias = _rand(30, seed=1)
    x = _rand(4, 3, 48, seed=2)
    got = _check_both(ops, x, wq, sw, bias, "none", torch.float32)
    assert got.shape == (4, 3, 30)
    one = _check_both(ops, x[0, 0], wq, sw, bias, "none", torch.float32)
    assert torch.equal(one, got[0, 0])
    # one policy's weights expanded to members: the same results
    many = _check_both(ops, x, wq.expand(4, 30, 48), sw.expand(4, 30),
                       bias.expand(4, 30), "none", torch.float32)
    assert torch.equal(many, got)
    # one observation expanded to all members
    _check_both(ops, x[:1].expand(4, 3, 48), wq.expand(4, 30, 48),
                sw.expand(4, 30), None, "tanh", torch.float32)
    # steps between members, tokens and channels
    big = _rand(4, 6, 96, seed=3)[:, ::2, 5:53]
    _check_both(ops, big, wq, sw, bias, "relu", torch.bfloat16)
    wb, sb = _weights(ops, 60, 48, (8,))
    _check_both(ops, x, wb[::2, ::2], sb[::2, ::2], None, "none",
                torch.float32)


def test_product_unusable_and_empty_rows(ops):
    for m in (4, 100, 400):
        x = _rand(m, 40, seed=m)
        x[0] = 0
        x[1, 3] = math.nan
        x[2, 39] = math.inf
        wq, sw = _weights(ops, 20, 40)
        sw[4] = 0
        sw[5] = math.inf
        bias = _rand(20, seed=1)
        bias[7] = math.nan
        q, s = oracle.codes_and_scale(x)
        for act in ("none", "relu", "tanh"):
            got = ops.int8_linear(x, wq, sw, bias, act)
            assert got[1:3].isnan().all()              # they show
            keep = [c for c in range(20) if c not in (5, 7)]
            want, err = oracle.product(q, s, wq[keep], sw[keep], bias[keep],
                                       act)
            oracle.check_product(got[:, keep], want, err, torch.float32)
            assert got[:, 7].isnan().all()


def test_product_out_leaves_its_surroundings(ops):
    for m, n in ((1, 5), (30, 19), (130, 70), (300, 301)):
        buf = torch.full((m * n + 64,), 123.0, device="cuda")
        out = buf[32:32 + m * n].view(m, n)
        x = _rand(m, 50, seed=m)
        wq, sw = _weights(ops, n, 50)
        got = ops.int8_linear(x, wq, sw, out=out)
        assert got.data_ptr() == out.data_ptr()
        q, s = oracle.codes_and_scale(x)
        oracle.check_product(got, *oracle.product(q, s, wq, sw, None, "none"),
                             torch.float32)
        assert bool((buf[:32] == 123).all()) and bool((buf[-32:] == 123).all())


def test_product_behind_32_bits(ops):
    """Weights of more than 2^31 bytes: the last members are found."""
    b, n, k = 1100, 1000, 2048
    wq = torch.zeros(b, n, k, dtype=torch.int8, device="cuda")
    wq[-3:] = torch.randint(-127, 128, (3, n, k), device="cuda").to(torch.int8)
    sw = torch.rand(b, n, device="cuda")
    for m in (1, 20):
        x = _rand(b, m, k, seed=1)
        got = ops.int8_linear(x, wq, sw)
        q, s = oracle.codes_and_scale(x[-3:])
        want, err = oracle.product(q, s, wq[-3:], sw[-3:], None, "none")
        oracle.check_product(got[-3:], want, err, torch.float32)
        assert not got[:-3].any()


def test_product_larger_than_a_launch_is_refused(ops):
    n = 70_000_000                # members of 64 threads: more than 2^32
    wq = torch.ones(1, 1, 1, dtype=torch.int8, device="cuda").expand(n, 1, 1)
    sw = torch.ones(1, 1, device="cuda").expand(n, 1)
    x = torch.ones(1, 1, 1, device="cuda").expand(n, 1, 1)
    with pytest.raises(ValueError, match="too large"):
        ops.int8_linear(x, wq, sw)
    got = ops.int8_linear(x[:60_000_000], wq[:60_000_000], sw[:60_000_000])
    assert bool((got == 1).all())


def test_no_gradient_mode_is_no_refusal(ops):
    x = _rand(3, 8, seed=1).requires_grad_()
    wq, sw = _weights(ops, 4, 8)
    with torch.no_grad():
        got = ops.int8_linear(x, wq, sw)
    assert not got.requires_grad
    with pytest.raises(ValueError):
        ops.int8_linear(x, wq, sw)


def test_product_same_bits_every_time(ops):
    for m, n, k in ((1, 700, 5000), (40, 64, 9000), (500, 300, 2000)):
        x, (wq, sw) = _rand(m, k, seed=1), _weights(ops, n, k)
        first = ops.int8_linear(x, wq, sw)
        for _ in range(3):
            assert torch.equal(ops.int8_linear(x, wq, sw), first)


# -------------------------------------------------------------- clipping ---
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [
    (1,), (0, 3), (5, 1, 0), (256, 64, 4096, 64, 128, 2), (4095, 4096, 4097),
    (8191, 8192, 8193, 1), (100_003,), (1_693_362,), (3,) * 300,
    (70_001,) * 130, (20_000_001, 7)])
@pytest.mark.parametrize("share", [0.3, 5.0])
def test_clip_sizes(ops, dtype, sizes, share):
    ts = [_rand(n, seed=i, dtype=dtype) for i, n in enumerate(sizes)]
    most = share * math.sqrt(max(1, sum(sizes)))
    got, norm = ops.clip_by_global_norm(ts, most)
    oracle.check_clipped(got, norm, *oracle.clipped(ts, most))
    assert torch.equal(ops.global_norm(ts), norm)
    if share > 1:
        assert all(torch.equal(g, t) for g, t in zip(got, ts))
    again, norm2 = ops.clip_by_global_norm(ts, most)
    assert torch.equal(norm, norm2)
    assert all(torch.equal(a, b) for a, b in zip(again, got))


def test_clip_in_place_mixed_and_misaligned(ops):
    theta = _rand(30_000, seed=1)
    half = _rand(9_999, seed=2, dtype=torch.bfloat16)
    ts = [theta[1:8], theta[8:8], theta[11:20_000], half[1:], half[:1],
          theta[20_001:].view(3, -1), _rand(33, 65, seed=3, dtype=torch.float16),
          _rand(1, seed=4)[0]]
    kept = [t.clone() for t in ts]
    rest = [theta[0].item(), theta[8:11].clone(), theta[20_000].item()]
    want, norm64 = oracle.clipped(kept, 2.5)
    got, norm = ops.clip_by_global_norm(ts, 2.5, out=ts)
    assert all(g.data_ptr() == t.data_ptr() for g, t in zip(got, ts))
    oracle.check_clipped(ts, norm, want, norm64)
    assert theta[0].item() == rest[0] and theta[20_000].item() == rest[2]
    assert torch.equal(theta[8:11], rest[1])
    for shift in range(4):                     # in and out shifted apart
        src = _rand(5_000, seed=5)[shift:]
        dst = torch.full((5_100,), 9.0, device="cuda")
        out = dst[3 + 2 * shift:3 + 2 * shift + src.numel()]
        got, norm = ops.clip_by_global_norm([src], 1.0, out=[out])
        oracle.check_clipped([out], norm, *oracle.clipped([src], 1.0))
        assert bool((dst[:3 + 2 * shift] == 9).all())
        assert bool((dst[3 + 2 * shift + src.numel():] == 9).all())
    t = _rand(50, 60, seed=6).t()              # read by its strides
    got, norm = ops.clip_by_global_norm([t], 1.0)
    oracle.check_clipped(got, norm, *oracle.clipped([t], 1.0))
    # the same tensor twice counts twice
    got, norm = ops.clip_by_global_norm([t, t], 1.0)
    oracle.check_clipped(got, norm, *oracle.clipped([t, t], 1.0))


@pytest.mark.parametrize("n", [3, 100_000])
def test_clip_extreme_values(ops, n):
    big = torch.full((n,), 3e38, device="cuda")
    got, norm = ops.clip_by_global_norm([big, -big], 1.0)
    assert norm.isinf()                        # of 64 bits, not of the squares
    want = torch.full((n,), (2 * n) ** -0.5)
    torch.testing.assert_close(got[0].cpu(), want, rtol=1e-6, atol=0)
    small = torch.full((n,), 1e-42, device="cuda")
    want = float(small[0]) * math.sqrt(n)
    assert abs(float(ops.global_norm([small])) - want) <= 1e-6 * want + 1e-45
    for bad in (math.nan, math.inf):
        t = _rand(n, seed=1)
        t[n // 2] = bad
        u = _rand(n, seed=2)
        got, norm = ops.clip_by_global_norm([u, t], 1.0)
        if math.isnan(bad):
            assert norm.isnan() and torch.equal(got[0], u)
        else:
            assert norm.isinf() and not got[0].any() and got[1].isnan().any()
    z = torch.zeros(n, device="cuda")
    for most in (0.0, 1.0):
        got, norm = ops.clip_by_global_norm([z], most)
        assert float(norm) == 0 and not got[0].any()
    got, norm = ops.clip_by_global_norm([_rand(n, seed=3)], 0.0)
    assert not got[0].any() and float(norm) > 0


def test_clip_of_nothing(ops):
    e = torch.empty(0, device="cuda")
    for ts in ([e], [e, e.view(0, 3)], [e] * 120):
        got, norm = ops.clip_by_global_norm(ts, 0.0, out=ts)
        assert float(norm) == 0 and len(got) == len(ts)
        assert float(ops.global_norm(ts)) == 0


def test_clip_behind_32_bits(ops):
    n = (1 << 31) + 5001
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t[-3:] = 2.0
    t[0] = 2.0
    got, norm = ops.clip_by_global_norm([t], 1.0, out=[t])
    assert float(norm) == 4.0
    assert got[0][[0, -3, -2, -1]].tolist() == [0.5] * 4 and float(t[1]) == 0


# ------------------------------------------------- streams, graphs, devices ---
def _step(ops, x, layers, grads, most):
    """One member step and its bounded gradient, as a program chains them."""
    for i, (wq, sw, b) in enumerate(layers):
        x = ops.int8_linear(x, wq, sw, b,
                            "tanh" if i + 1 < len(layers) else "none")
    clipped, norm = ops.clip_by_global_norm(grads, most)
    return [x, norm, *clipped]


def _chain(ops, lead, m, seed):
    sizes = (376, 256, 256, 17)
    layers = [(*_weights(ops, o, i, lead, seed + i), _rand(*lead, o, seed=i))
              for i, o in zip(sizes, sizes[1:])]
    x = _rand(*lead, m, 376, seed=seed)
    grads = [_rand(n, seed=seed + n) for n in (96256, 256, 65536, 256, 4352, 17)]
    return x, layers, grads


@pytest.mark.parametrize("lead,m", [((9,), 1), ((), 16), ((), 300),
                                    ((), 70000)])
def test_captured_and_replayed(ops, lead, m):
    """Two graphs and eager calls in turn: each replay gives what an eager call
    on the inputs of that moment gives."""
    graphs = []
    for seed in (1, 2):
        x, layers, grads = _chain(ops, lead, m, seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(ops, x, layers, grads, 3.0)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(ops, x, layers, grads, 3.0)
        graphs.append((g, x, layers, grads, out))
    for turn in range(4):
        for g, x, layers, grads, out in graphs:
            x.copy_(_rand(*x.shape, seed=50 + turn))
            grads[0].mul_(1.5)
            g.replay()
            want = _step(ops, x, layers, grads, 3.0)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once(ops):
    chains = [_chain(ops, (), 200, s) for s in (3, 4)]
    want = [_step(ops, *c, 3.0) for c in chains]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in chains]
    for _ in range(5):
        got = []
        for s, c in zip(streams, chains):
            with torch.cuda.stream(s):
                got.append(_step(ops, *c, 3.0))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_mixed_places_are_refused(ops):
    x, (wq, sw) = _rand(3, 8, seed=1), _weights(ops, 4, 8)
    with pytest.raises(ValueError):
        ops.int8_linear(x, wq.cpu(), sw)
    with pytest.raises(ValueError):
        ops.int8_linear(x, wq, sw, sw.cpu())
    with pytest.raises(ValueError):
        ops.clip_by_global_norm([x, x.cpu()], 1.0)


@pytest.mark.parametrize("m,n,k", [
    (8191, 1023, 2900), (16385, 510, 1290), (8190, 511, 700), (4095, 1000, 1900),
    (8192, 512, 128), (8192, 512, 256), (8192, 512, 257), (8192, 512, 384),
    (20001, 1020, 300), (4090, 500, 640), (4090, 500, 200), (2040, 500, 600),
    (8190, 2040, 2000), (8190, 1022, 1100)])
@pytest.mark.parametrize("out", [torch.float32, torch.float16])
def test_product_tiles_by_turns(ops, m, n, k, out):
    """Each size of tile with fewer stages than its ring and with many, a whole
    last stage and a part of one, one turn and several."""
    x = _rand(m, k, seed=m + n + k)
    wq, sw = _weights(ops, n, k)
    _check_both(ops, x, wq, sw, _rand(n, seed=2), "relu", out)


@pytest.mark.parametrize("b,m,n,k", [
    (40, 250, 500, 1000), (300, 250, 250, 900), (16, 500, 500, 2000),
    (17, 500, 500, 2000), (30, 500, 500, 2000)])
def test_member_product_tiles_by_turns(ops, b, m, n, k):
    _sampled(ops, b, m, n, k)


@pytest.mark.parametrize("m,n,k", [(2040, 500, 601), (4090, 500, 641),
                                   (8190, 511, 701), (8191, 1023, 2901),
                                   (8190, 2040, 2001)])
def test_captured_tiles_of_odd_rows(ops, m, n, k):
    """Codes whose rows lie at odd addresses are copied inside the graph; two
    graphs take turns with eager calls."""
    g = torch.Generator("cuda").manual_seed(m)
    codes = lambda r: torch.randint(-127, 128, (r, k), dtype=torch.int8,
                                    device="cuda", generator=g)
    wq, sw, sx = codes(n), torch.rand(n, device="cuda"), torch.rand(m, device="cuda")
    xs = [codes(m), codes(m)]
    ops.int8_matmul(xs[0], sx, wq, sw)
    graphs = []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.int8_matmul(x, sx, wq, sw)
        graphs.append((graph, out))
    for _ in range(3):
        for x, (graph, out) in zip(xs, graphs):
            x.copy_(codes(m))
            graph.replay()
            want = ops.int8_matmul(x, sx, wq, sw)
            torch.cuda.synchronize()
            assert torch.equal(out, want)


# ------------------------------------------------------ rows of no values ---
def _valueless(dtype):
    """Rows of no values in layouts that dense tensors do not have."""
    z = lambda *s: torch.zeros(*s, dtype=dtype, device="cuda")
    return [z(3, 4, 5)[:, :2, :0], z(30, 40, 5)[:, :20, :0],
            z(5, 9, 2)[::2, ::2, :0], z(2, 3, 4, 0).permute(2, 1, 0, 3),
            z(7, 3)[::2, :0], z(600, 4, 2)[:, :2, :0]]


@pytest.mark.parametrize("i", range(6))
@pytest.mark.parametrize("act", ["none", "tanh"])
def test_product_of_no_values_in_any_layout(ops, i, act):
    sw, bias = _rand(6, seed=1), _rand(6, seed=2)
    wq = torch.zeros(6, 0, dtype=torch.int8, device="cuda")
    x, xq = _valueless(torch.float32)[i], _valueless(torch.int8)[i]
    want = (bias.tanh() if act == "tanh" else bias).expand(*x.shape[:-1], 6)
    out = torch.full(want.shape, 99.0, device="cuda")
    ops.int8_linear(x, wq, sw, bias, act, out=out)
    # the bias as it is, or its tanh: two steps of 32 bits
    torch.testing.assert_close(out, want, rtol=4 * oracle.U32, atol=0)
    out.fill_(99.0)
    ops.int8_matmul(xq, torch.ones(x.shape[:-1], device="cuda"), wq, sw, bias,
                    act, out=out)
    torch.testing.assert_close(out, want, rtol=4 * oracle.U32, atol=0)


@pytest.mark.parametrize("i", range(6))
def test_quantize_rows_of_no_values_in_any_layout(ops, i):
    x = _valueless(torch.float32)[i]
    q, s = ops.quantize_rows(x)
    assert q.shape == x.shape and q.dtype == torch.int8
    assert s.shape == x.shape[:-1] and bool((s == 2.0 ** -126).all())
    s = torch.zeros(x.shape[:-1], device="cuda")
    ops.quantize_rows(x, out=(torch.empty(x.shape, dtype=torch.int8,
                                          device="cuda"), s))
    assert bool((s == 2.0 ** -126).all())
    none = torch.zeros(4, 0, 6, 8, device="cuda").permute(2, 1, 0, 3)
    q, s = ops.quantize_rows(none)             # no rows, by three strides
    assert q.shape == none.shape and s.shape == none.shape[:-1]


@pytest.mark.parametrize("lead,m", [((), 1), ((), 4), ((), 20), ((), 600),
                                    ((3,), 2), ((3,), 20)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_scales_count_where_rows_have_no_values(ops, lead, m, bad):
    """0 * NaN and 0 * inf: the token's results are NaN, as the twin's are."""
    wq = torch.zeros(*lead, 6, 0, dtype=torch.int8, device="cuda")
    sw, bias = _rand(*lead, 6, seed=1).abs(), _rand(*lead, 6, seed=2)
    sx = torch.ones(*lead, m, device="cuda")
    sx[..., -1] = bad
    xq = torch.zeros(*lead, m, 0, dtype=torch.int8, device="cuda")
    got = ops.int8_matmul(xq, sx, wq, sw, bias)
    assert got[..., -1, :].isnan().all()
    assert torch.equal(got[..., :-1, :],
                       bias[..., None, :].expand(*lead, m - 1, 6))


# ------------------------------------------------------------ large scales ---
@pytest.mark.parametrize("lead,m,n,k", [
    ((), 2, 40, 3136), ((), 3, 40, 500), ((), 16, 70, 700), ((), 16, 70, 100),
    ((), 700, 700, 300), ((), 2100, 2100, 200), ((5,), 2, 40, 64),
    ((5,), 20, 40, 64)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["none", "tanh"])
def test_product_of_large_rows(ops, lead, m, n, k, out, act):
    """Rows of 1e36 with weights of 1e-8: sums times the token's scale leave
    fp32's range, results do not.  Other tokens of the batch keep their bits."""
    x = _rand(*lead, m, k, seed=1)
    wq, sw = ops.quantize_rows(_rand(*lead, n, k, seed=2) * 1e-8)
    bias = _rand(*lead, n, seed=3)
    alone = ops.int8_linear(x, wq, sw, bias, act, out)
    x[..., ::2, :] *= 1e36
    x[..., 0, :] = 1e36
    wq[..., 0, :] = 127
    q, s = oracle.codes_and_scale(x)
    want, err = oracle.product(q, s, wq, sw, bias, act)
    got = _check_both(ops, x, wq, sw, bias, act, out)
    oracle.check_product(got, want, err, out)
    # the first product is that of codes alone, so that no product is finite
    # by chance: its sum times the scale is beyond 32 bits
    assert 127.0 * 127.0 * k * float(s.max()) > 3.4e38
    assert torch.equal(got[..., 1::2, 1:], alone[..., 1::2, 1:])


@pytest.mark.parametrize("m,n", [(2, 4), (16, 4), (600, 700), (2100, 2100)])
def test_product_of_large_scales_on_both_sides(ops, m, n):
    """A sum of 0 gives the bias, any other one is beyond the range."""
    xq = torch.full((m, 64), 127, dtype=torch.int8, device="cuda")
    wq = torch.full((n, 64), 127, dtype=torch.int8, device="cuda")
    wq[::2, ::2] = -127
    sx, sw = (torch.full((r,), 2.0 ** 100, device="cuda") for r in (m, n))
    sw[3] = math.nan
    sx[1] = -sx[1]
    bias = _rand(n, seed=1)
    got = ops.int8_matmul(xq, sx, wq, sw, bias)
    assert torch.equal(got[:, ::2], bias[::2].expand(m, len(bias[::2])))
    assert got[:, 3].isnan().all()
    assert bool((got[1, 1] == -math.inf) & (got[0, 1] == math.inf))
    sw[1] = 2.0 ** -126                        # 64 * 127^2 * 2^-26
    got = ops.int8_matmul(xq, sx, wq, sw)
    assert bool((got[::2, 1] == 127.0 ** 2 * 2.0 ** -20).all())


# ---------------------------------------------------------------- autograd ---
def test_writes_count_as_writes(ops):
    """Version counters, as torch's own in-place operators keep them."""
    x, (wq, sw) = _rand(3, 8, seed=1), _weights(ops, 4, 8)
    q, s = ops.quantize_rows(x)
    y, g, e = _rand(3, 4), _rand(5), torch.empty(0, 4, device="cuda")
    for call, written in (
            (lambda: ops.quantize_rows(x, out=(q, s)), (q, s)),
            (lambda: ops.int8_linear(x, wq, sw, out=y), (y,)),
            (lambda: ops.int8_matmul(q, s, wq, sw, out=y), (y,)),
            (lambda: ops.int8_linear(x[:0], wq, sw, out=e), (e,)),
            (lambda: ops.clip_by_global_norm([g, y], 1.0, out=[g, y]), (g, y)),
            (lambda: ops.clip_by_global_norm([g], 9.0, out=[g]), (g,))):
        before = [t._version for t in (x, q, s, y, g, e, wq, sw)]
        call()
        for t, v in zip((x, q, s, y, g, e, wq, sw), before):
            assert t._version == v + any(t is w for w in written)


def test_a_saved_tensor_that_is_written_is_noticed(ops):
    leaf = _rand(5, seed=2).requires_grad_()
    for write in (lambda t: ops.clip_by_global_norm([t], 0.1, out=[t]),
                  lambda t: ops.int8_linear(
                      _rand(1, 8), *_weights(ops, 5, 8), out=t[None])):
        saved = _rand(5, seed=3)
        loss = (leaf * saved).sum()
        write(saved)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    with torch.inference_mode():
        t = _rand(5, seed=4)
        ops.clip_by_global_norm([t], 0.1, out=[t])      # has no counter
    with pytest.raises(RuntimeError, match="nference"):
        ops.clip_by_global_norm([t], 0.1, out=[t])


# ----------------------------------------------------------- negated views ---
def _negated(t):
    """t as a view of -t's memory that torch negates when it reads it; its last
    stride is 2."""
    view = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert view.is_neg() and torch.equal(view, t)
    return view


def test_negated_views_are_read_as_their_values(ops):
    x = _rand(5, 1, seed=1)                # rows of one value: any last stride
    v = _negated(x)
    _check_codes(x, *ops.quantize_rows(v))
    wq, sw = _weights(ops, 4, 1)
    bias = _rand(4, seed=2)
    assert torch.equal(ops.int8_linear(v, wq, sw, bias),
                       ops.int8_linear(x, wq, sw, bias))
    xq, sx = ops.quantize_rows(x)
    want = ops.int8_matmul(xq, sx, wq, sw, bias)
    one = slice(0, 1)                      # a vector of one value: contiguous
    assert torch.equal(want[:, one], ops.int8_matmul(
        xq, sx, wq[one], _negated(sw[one]), _negated(bias[one])))
    assert torch.equal(want[one], ops.int8_matmul(xq[one], _negated(sx[one]),
                                                  wq, sw, bias))
    t = _rand(1, seed=3)
    for norm in (0.1, 9.0):
        got, n = ops.clip_by_global_norm([_negated(t), x], norm)
        oracle.check_clipped(got, n, *oracle.clipped([t, x], norm))
    assert torch.equal(ops.global_norm([_negated(t), _negated(x)]), n)


@pytest.mark.parametrize("shape,perm", [
    ((3, 0, 0, 17), (0, 1, 2, 3)), ((0, 0, 5, 8), (2, 0, 1, 3)),
    ((4, 0, 6, 8), (2, 1, 0, 3)), ((3, 0, 0, 2, 0), (3, 1, 0, 2, 4)),
    ((0, 9, 4), (0, 2, 1))])
def test_no_rows_in_any_layout(ops, shape, perm):
    x = torch.zeros(shape, device="cuda").permute(perm)
    q, s = ops.quantize_rows(x)
    assert q.shape == x.shape and s.shape == x.shape[:-1]
    out = (torch.zeros(shape, dtype=torch.int8, device="cuda").permute(perm), s)
    assert ops.quantize_rows(x, out=out)[0].shape == x.shape
    wq, sw = _weights(ops, 5, max(1, x.shape[-1]))
    wq = wq[:, :x.shape[-1]]
    assert ops.int8_linear(x, wq, sw).shape == (*x.shape[:-1], 5)
    assert ops.int8_matmul(q, s, wq, sw).shape == (*x.shape[:-1], 5)
