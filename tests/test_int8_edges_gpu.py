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
