"""8-bit operators: the scale's error over long rows and at the ends of its range, layers that are cast."""
import pytest
import torch

from test_int8_gpu import STEP32, TYPES, check_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_layers_of_a_cast_model(cuda_device, dtype):
    """A model that is cast for evaluation gives the products that it gave before: scales and bias stay in 32 bits."""
    from geo_b200 import layers

    torch.manual_seed(2)
    linear = torch.nn.Linear(40, 24).to(cuda_device)
    with torch.no_grad():
        layer = layers.Linear_Int8.from_float(linear)
        model = torch.nn.Sequential(layer)
        x = torch.randn(6, 40, device=cuda_device).bfloat16()
        expect = model(x)
        assert torch.equal(model.to(dtype)(x), expect)
        assert torch.equal(model.cpu().to(cuda_device)(x), expect)


# Error of a row's scale, whatever its length: a thread adds at most 32 rounded products one after the other, what lies
# past those in parts of at most 16 products which are joined in 64 bits (one rounding back, one addition), five shuffles
# join a warp and five the warps: 32 + 2 + 10 half steps of the sum, halved by the root; the mean's division and the
# addition of eps, halved as well, the root, and two divisions.
SCALE_ERROR = (44 / 2 + 2 / 2 + 3) * STEP32


@pytest.mark.parametrize("cols", [40000, 60001, (1 << 20) - 4, (1 << 26) - 4, (1 << 26) - 1])
@pytest.mark.parametrize("with_residual", [False, True])
def test_error_of_the_scale_does_not_grow_with_the_row(cuda_device, cols, with_residual):
    """Squares of 1 + 2^-9: a sum of many in 32 bits loses the 2^-9 of each as soon as it is large."""
    from geo_b200 import functional as F

    value = (1 + 2.0 ** -9) ** 0.5
    x = torch.full((1, cols), value, device=cuda_device)
    x[0, 7] = 3.0
    res = torch.zeros(1, cols, device=cuda_device) if with_residual else None
    q, scale = F.rms_norm_int8(x, torch.ones(cols, device=cuda_device), res, eps=0.0)[:2]
    single = float(x[0, 0])
    expect = 3 / 127 / (((cols - 1) * single * single + 9) / cols) ** 0.5
    assert abs(float(scale) - expect) <= SCALE_ERROR * expect
    assert q[0, 7] == 127 and (q[0, 8:] == round(127 * single / 3)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("unit", [1.0, 2.0 ** -14, 2.0 ** -45])
@pytest.mark.parametrize("cols", [4, 5, 64, 1000, 4096])
def test_scale_near_the_end_of_its_range(cuda_device, dtype, cols, unit):
    """A weight so large that max|p| / rms leaves the range of 32 bits although the scale, 1/127 of it, does not."""
    from geo_b200 import functional as F

    x = torch.zeros(3, cols, dtype=dtype, device=cuda_device)
    x[0, 0], x[1, cols - 1], x[2, 1] = unit, -0.5 * unit, 0.75 * unit
    x[2, 2] = 0.25 * unit
    if dtype == torch.float16 and unit < 2.0 ** -14:
        x[:, 0] = 2.0 ** -24         # the type's smallest value
    w = torch.full((cols,), 3e38, device=cuda_device)
    q, scale = F.rms_norm_int8(x, w, eps=0.0)
    assert scale.isfinite().all()
    check_norm(x, None, w, 0.0, (q, scale))


@pytest.mark.parametrize("bias", [False, True])
def test_layer_from_a_stochastic_layer(cuda_device, bias):
    """The integers of a Linear_Or are those of its full-precision weight, not of the one that its last forward has quantised."""
    from geo_b200 import functional as F
    from geo_b200 import layers

    torch.manual_seed(3)
    sc = layers.Linear_Or(32, 12, bias=bias).to(cuda_device)
    kept = sc.weight_org.clone()
    sc(torch.rand(4, 32, device=cuda_device))
    assert not torch.equal(sc.weight, kept)
    with torch.no_grad():
        layer = layers.Linear_Int8.from_float(sc)
        q, scale = F.quantize_int8(kept)
        assert torch.equal(layer.weight_q[:, :32], q) and torch.equal(layer.weight_scale, scale)
        x = torch.randn(5, 32, device=cuda_device)
        xq, xs = F.quantize_int8(x)
        assert torch.equal(layer(x), F.linear_int8(xq, xs, q, scale, sc.bias))
