"""8-bit row quantisation, the norm in front of it and the 8-bit product, against plain formulas in 64 bits on the CPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
STEP32 = 2.0 ** -24     # half a step of a 32-bit float, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference_rows(r, weight):
    """(q, largest p) of rows r (CPU): the 32-bit product with the weight, the integers in 64 bits."""
    p = r.float() if weight is None else r.float() * weight.float()
    top = p.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, torch.round(p.double() * 127 / top.double()), 0.0)
    return q.to(torch.int8), top[..., 0].double()


def sum_error(cols):
    """Relative error of a sum of squares: a thread adds at most 32 + cols / 1024 rounded products one after the other,
    each addition and product is off by half a step, five shuffles join a warp, the rest is in 64 bits."""
    return (2 * (32 + cols / 1024) + 5) * STEP32


def check_norm(x, res, weight, eps, out):
    x, w = x.cpu(), weight.cpu()
    total = x if res is None else (x.float() + res.cpu().float()).to(x.dtype)
    q, top = reference_rows(total, w)
    rms = torch.sqrt(total.double().square().mean(-1) + eps)
    assert torch.equal(out[0].cpu(), q)
    expect = top / 127 / rms
    # the scale: the sum's error halved by the root, one rounding
    assert ((out[1].cpu().double() - expect).abs() <= expect * (sum_error(x.shape[-1]) / 2 + 2 * STEP32) + 2.0 ** -149).all()
    if res is not None:
        assert torch.equal(out[2].cpu(), total)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (1, 4096), (5, 512), (300, 64), (700, 257), (33, 2048), (2, 33000), (4, 40000), (400, 1000), (500, 255), (50, 2047), (9, 4095), (3, 60001)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_matches_the_formula(cuda_device, dtype, rows, cols, with_residual):
    from geo_b200 import functional as F

    g = torch.Generator().manual_seed(rows * 7 + cols)
    x = (torch.randn(rows, cols, generator=g) * 2).to(dtype).to(cuda_device)
    res = (torch.randn(rows, cols, generator=g) * 3).to(dtype).to(cuda_device) if with_residual else None
    for wtype in TYPES:
        w = (1 + 0.3 * torch.randn(cols, generator=g)).to(wtype).to(cuda_device)
        check_norm(x, res, w, 1e-5, F.rms_norm_int8(x, w, res, 1e-5))


def test_norm_borders_and_ties(cuda_device):
    """Values at and next to the borders between two integers: k + 1/2 in units of the row's largest value / 127."""
    from geo_b200 import functional as F

    k = torch.arange(-127, 127).float()
    half = torch.cat([torch.tensor([127.0]), k + 0.5])                     # exact ties
    rows = [half, half * 3, torch.nextafter(half, torch.full_like(half, 1e9)), torch.nextafter(half, torch.full_like(half, -1e9)), half / 7]
    x = torch.stack(rows).clone()
    x[2:4, 0] = 127.0
    x = torch.cat([x, x * 2.0 ** -120, x * 2.0 ** 100, x * 2.0 ** -149])   # the last: below the normal range
    for weight in (torch.ones(x.shape[1]), torch.full((x.shape[1],), 1 / 3)):
        q, top = reference_rows(x, weight)
        assert torch.equal(F.rms_norm_int8(x.to(cuda_device), weight.to(cuda_device), eps=0.0)[0].cpu(), q)
    q, top = reference_rows(x, None)
    got, scale = F.quantize_int8(x.to(cuda_device))
    assert torch.equal(got.cpu(), q)
    assert ((scale.cpu().double() - top / 127).abs() <= top / 127 * STEP32 + 2.0 ** -150).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_extreme_rows(cuda_device, dtype):
    from geo_b200 import functional as F

    big = 6e4 if dtype == torch.float16 else 3e38
    x = torch.zeros(7, 40, dtype=dtype)
    x[1] = big                     # squares leave the range of 32 bits
    x[2, 3] = float("inf")
    x[3, 5] = float("nan")
    x[4] = torch.finfo(dtype).tiny
    x[5, ::2] = -big
    x[6, 0] = 1.0
    w = torch.ones(40)
    q, scale = F.rms_norm_int8(x.to(cuda_device), w.to(cuda_device), eps=1e-12)
    q, scale = q.cpu(), scale.cpu()
    assert (q[0] == 0).all() and scale[0] == 0
    assert (q[1] == 127).all() and abs(float(scale[1]) * 127 - 1) < 1e-5
    for bad in (2, 3):
        assert (q[bad] == 0).all() and scale[bad].isnan()
    rows = [0, 1, 4, 5, 6]
    check_norm(x[rows], None, w, 1e-12, (q[rows], scale[rows]))
    q, scale = F.quantize_int8(x.to(cuda_device))
    expect, top = reference_rows(x[rows], None)
    assert torch.equal(q.cpu()[rows], expect) and scale.cpu()[2:4].isnan().all()
    # a product that leaves the range, though the row does not
    q, scale = F.rms_norm_int8(x[1:2].to(cuda_device), (w * 1e38).to(cuda_device))
    assert (q == 0).all() and scale.isnan().all()
    # with eps = 0 a row of zeros stays a row of zeros
    q, scale = F.rms_norm_int8(x[:1].to(cuda_device), w.to(cuda_device), eps=0.0)
    assert (q == 0).all() and (scale == 0).all()


@pytest.mark.parametrize("value", [1.7e17, 1.05e17, 6e16, 1e18, 3e-16, 1e-18, 3e-20])
@pytest.mark.parametrize("cols", [16384, 16383, 40000, 300])
def test_norm_at_the_ends_of_the_sum(cuda_device, value, cols):
    """Rows whose squares fit 32 bits one by one and warp by warp, but not together, or nearly vanish."""
    from geo_b200 import functional as F

    x = torch.full((3, cols), value)
    x[1, ::2] *= -0.5
    w = torch.ones(cols)
    check_norm(x.to(cuda_device), None, w, 0.0, F.rms_norm_int8(x.to(cuda_device), w.to(cuda_device), eps=0.0))


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_strides_and_shapes(cuda_device, dtype):
    from geo_b200 import functional as F

    g = torch.Generator().manual_seed(3)
    base = torch.randn(6, 5, 200, generator=g).to(dtype).to(cuda_device)
    w = torch.rand(96, generator=g).to(cuda_device)
    for x in (base[..., :96], base[..., 1:97], base[:, 2, 8:104], base.transpose(1, 2)[:, :96].transpose(1, 2), base[0, 0, 3:99],
              base[0, :1, :96].expand(4, 96), base.permute(0, 2, 1)[:, 4:100].permute(0, 2, 1)):
        res = torch.randn(x.shape, generator=g).to(dtype).to(cuda_device)
        q, scale, total = F.rms_norm_int8(x, w, res, 1e-5)
        assert q.shape == x.shape and scale.shape == x.shape[:-1] and total.shape == x.shape
        check_norm(x, res, w, 1e-5, (q, scale, total))
        q, scale = F.quantize_int8(x)
        assert torch.equal(q.cpu(), reference_rows(x.cpu(), None)[0]) and (q.dim() < 2 or q.stride(-2) % 16 == 0)
        y = F.dequantize_int8(q, scale, dtype)
        exact = q.cpu().double() * scale.cpu().double()[..., None]
        assert y.shape == x.shape and ((y.cpu().double() - exact).abs() <= exact.abs() * (half_step(dtype) + STEP32) + 2.0 ** -25).all()
    for empty in (base[:0, 0, :96], base[:, :0, :96]):
        q, scale = F.rms_norm_int8(empty, w)
        assert q.shape == empty.shape and scale.shape == empty.shape[:-1]
        assert F.dequantize_int8(q, scale).shape == empty.shape


def test_quantised_rows_do_not_depend_on_their_neighbours(cuda_device):
    """One row gives the same integers and scale alone, in a small and in a large batch (other launch shapes)."""
    from geo_b200 import functional as F

    g = torch.Generator().manual_seed(4)
    w = torch.rand(1024, generator=g).to(cuda_device)
    x = torch.randn(1000, 1024, generator=g).to(cuda_device)
    q, scale = F.rms_norm_int8(x, w)
    for rows in (1, 40):
        q1, s1 = F.rms_norm_int8(x[:rows], w)
        assert torch.equal(q1, q[:rows])
        assert ((s1 - scale[:rows]).abs() <= scale[:rows] * sum_error(1024)).all()


def int8_rows(g, rows, cols, device, low=-128):
    t = torch.empty((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=device)[:, :cols]
    return t.copy_(torch.randint(low, 128, (rows, cols), generator=g, dtype=torch.int8))


def check_product(x, xs, w, ws, bias, out):
    s = x.cpu().double() @ w.cpu().double().T                             # exact: below 2^31
    y = s * xs.cpu().double()[:, None] * ws.cpu().double()
    b = torch.zeros(1).double() if bias is None else bias.cpu().double()
    # integer to float, two products and the addition: half a step each; then one rounding to the output's type
    bound = (4 * y.abs() + b.abs()) * STEP32 + (y + b).abs() * half_step(out.dtype) * (1 + 2.0 ** -10) + 2.0 ** -25
    assert ((out.cpu().double() - (y + b)).abs() <= bound).all()


PRODUCT_SIZES = [(1, 1, 1), (1, 16, 16), (1, 4096, 1024), (2, 33, 65), (7, 100, 2047), (8, 64, 64), (9, 129, 333), (17, 64, 4097),
                 (32, 48, 128), (33, 257, 100), (65, 130, 1000), (100, 10, 512), (128, 128, 128), (129, 127, 255), (256, 512, 512),
                 (300, 1001, 130), (513, 511, 640), (1000, 64, 33), (64, 2048, 2048), (700, 900, 1),
                 (100, 19000, 64), (129, 9500, 70), (257, 9600, 130), (1000, 5000, 300), (2000, 2100, 1024), (300, 20000, 16),
                 (200, 300, 4000), (50, 500, 8000), (400, 900, 6000), (450, 401, 9001), (600, 701, 3001), (1100, 1501, 700)]


@pytest.mark.parametrize("m, n, k", PRODUCT_SIZES)
def test_product_matches_the_formula(cuda_device, m, n, k):
    from geo_b200 import _lib, functional as F

    g = torch.Generator().manual_seed(m + 3 * n + 5 * k)
    x, w = int8_rows(g, m, k, cuda_device), int8_rows(g, n, k, cuda_device)
    xs, ws = (torch.rand(m, generator=g) * 0.1).to(cuda_device), (torch.rand(n, generator=g) * 0.1).to(cuda_device)
    bias = torch.randn(n, generator=g).to(cuda_device)
    for dtype in TYPES:
        for b in (None, bias):
            scale = xs * 1e-3 if dtype == torch.float16 else xs           # inside the range of 16 bits
            check_product(x, scale, w, ws, b, F.linear_int8(x, scale, w, ws, b, dtype))
    assert _lib.device_error_count() == 0


def test_product_of_the_longest_sums_is_exact(cuda_device):
    """k = 131071 rows of -128: 2^14 k, the largest sum that 32 bits are promised for."""
    from geo_b200 import functional as F

    k = 131071
    for m in (1, 40, 200):
        x, w = torch.full((m, k), -128, dtype=torch.int8, device=cuda_device), torch.full((3, k), -128, dtype=torch.int8, device=cuda_device)
        w[1] = 127
        out = F.linear_int8(x, torch.ones(m, device=cuda_device), w, torch.ones(3, device=cuda_device))
        expect = torch.tensor([16384.0 * k, -16256.0 * k, 16384.0 * k], dtype=torch.float64).float()   # one rounding to 32 bits
        assert torch.equal(out.cpu(), expect.expand(m, 3))


@pytest.mark.parametrize("m", [3, 70, 300])
def test_product_strides_shapes_and_poisoned_rows(cuda_device, m):
    from geo_b200 import functional as F

    g = torch.Generator().manual_seed(m)
    base_x = torch.randint(-127, 128, (m, 400), generator=g, dtype=torch.int8).to(cuda_device)
    base_w = torch.randint(-127, 128, (150, 400), generator=g, dtype=torch.int8).to(cuda_device)
    xs, ws = torch.rand(m, generator=g).to(cuda_device), torch.rand(150, generator=g).to(cuda_device)
    for x, w in ((base_x[:, :200], base_w[:, 16:216]), (base_x[:, 1:202], base_w[:, 3:204]), (base_x[:, ::2], base_w[:, 1::2]),
                 (base_x[:1].expand(m, 400), base_w), (base_x.t().contiguous().t(), base_w)):
        check_product(x, xs, w, ws, None, F.linear_int8(x, xs, w, ws))
    x3 = base_x[:, :64].reshape(1, m, 64).expand(2, m, 64)
    out = F.linear_int8(x3, xs.expand(2, m), base_w[:, :64], ws, dtype=torch.bfloat16)
    assert out.shape == (2, m, 150)
    check_product(base_x[:, :64], xs, base_w[:, :64], ws, None, out[1])
    assert F.linear_int8(base_x[0], xs[0], base_w, ws).shape == (150,)
    assert F.linear_int8(base_x[:0], xs[:0], base_w, ws).shape == (0, 150)
    xs[1] = float("nan")
    out = F.linear_int8(base_x, xs, base_w, ws)
    assert out[1].isnan().all() and out[[0, 2]].isfinite().all()


def test_product_writes_its_rows_only(cuda_device):
    """Through the C ABI into a wider output: the columns beside and the rows behind stay as they were."""
    import ctypes

    from geo_b200 import _lib

    g = torch.Generator().manual_seed(11)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for m, n, k in ((5, 37, 48), (40, 37, 100), (200, 300, 130)):
        x, w = int8_rows(g, m, k, cuda_device), int8_rows(g, n, k, cuda_device)
        xs, ws = torch.ones(m, device=cuda_device), torch.ones(n, device=cuda_device)
        out = torch.full((m + 3, n + 5), -7.0, device=cuda_device)
        _lib.check(_lib.lib().geo_sc_linear_int8(m, n, k, x.data_ptr(), x.stride(0), xs.data_ptr(), w.data_ptr(), w.stride(0),
                                                 ws.data_ptr(), None, 0, out.data_ptr(), n + 5, stream), "geo_sc_linear_int8")
        check_product(x, xs, w, ws, None, out[:m, :n])
        assert (out[m:] == -7).all() and (out[:, n:] == -7).all()


def test_offsets_past_32_bits(cuda_device):
    """More than 2^31 values in rows, integers and outputs: the last rows are right."""
    from geo_b200 import functional as F

    for cols in (16400, 16401):
        x = torch.zeros(131100, cols, dtype=torch.bfloat16, device=cuda_device)
        g = torch.Generator().manual_seed(cols)
        x[-3:] = torch.randn(3, cols, generator=g).bfloat16().to(cuda_device)
        q, scale = F.quantize_int8(x)
        expect, _ = reference_rows(x[-3:].cpu(), None)
        assert torch.equal(q[-3:].cpu(), expect) and (q[:2] == 0).all()
        y = F.dequantize_int8(q, scale, torch.bfloat16)
        exact = q[-3:].cpu().double() * scale[-3:].cpu().double()[:, None]
        assert ((y[-3:].cpu().double() - exact).abs() <= exact.abs() * (2.0 ** -8 + 2.0 ** -20)).all()
        del x, y
    m, n = 70000, 33001
    x, w = int8_rows(g, m, 32, cuda_device), int8_rows(g, n, 32, cuda_device)
    xs, ws = torch.rand(m, generator=g).to(cuda_device), torch.rand(n, generator=g).to(cuda_device)
    out = F.linear_int8(x, xs, w, ws, dtype=torch.bfloat16)
    check_product(x[-300:], xs[-300:], w, ws, None, out[-300:])
    check_product(x[:7], xs[:7], w, ws, None, out[:7])


def test_layers_chain_and_capture(cuda_device):
    """norm -> 8-bit layer -> residual -> norm -> 8-bit layer, eagerly, on another stream and replayed from a graph."""
    from geo_b200 import layers

    torch.manual_seed(5)
    norm1, norm2 = torch.nn.RMSNorm(72, eps=1e-5).to(cuda_device), torch.nn.RMSNorm(72).to(cuda_device)
    lin1, lin2 = torch.nn.Linear(72, 72).to(cuda_device), torch.nn.Linear(72, 20, bias=False).to(cuda_device)
    with torch.no_grad():
        norm1.weight.uniform_(0.5, 1.5)
        n1, n2 = layers.RMSNorm_Int8.from_float(norm1), layers.RMSNorm_Int8.from_float(norm2)
        l1, l2 = layers.Linear_Int8.from_float(lin1), layers.Linear_Int8.from_float(lin2)
        assert n2.eps == torch.finfo(torch.float32).eps

        def chain(x):
            h = l1(n1(x))
            q, scale, total = n2(h, residual=x)
            return l2((q, scale)), total

        x = torch.randn(50, 72, device=cuda_device)
        out, total = chain(x)
        ref_h = lin1(norm1(x))
        ref = lin2(norm2(ref_h + x))
        # quantisation of two operands, 1/254 of a row's largest value each: a bound on the outputs' rms error
        assert (out - ref).square().mean().sqrt() < 0.02 * ref.square().mean().sqrt() * 3
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = chain(x)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(again[0], out) and torch.equal(again[1], total)
        graph = torch.cuda.CUDAGraph()
        static = x.clone()
        with torch.cuda.graph(graph):
            captured = chain(static)
        x2 = torch.randn(50, 72, device=cuda_device)
        static.copy_(x2)
        graph.replay()
        expect = chain(x2)
        assert torch.equal(captured[0], expect[0]) and torch.equal(captured[1], expect[1])
        # float rows are quantised by the layer itself; the state travels
        l3 = layers.Linear_Int8(72, 72).to(cuda_device)
        l3.load_state_dict(l1.state_dict())
        for dtype in TYPES:
            y = l3(x.to(dtype).view(5, 10, 72))
            assert y.shape == (5, 10, 72) and y.dtype == dtype and torch.equal(y, l1(x.to(dtype)).view(5, 10, 72))
    with pytest.raises(RuntimeError):
        l1(torch.randn(2, 72, device=cuda_device, requires_grad=True))
