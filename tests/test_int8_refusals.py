"""What the 8-bit operators and the distillation loss refuse, without a GPU: argument checks come before the device is
looked at, and the C entry points check before they launch."""
import ctypes

import pytest
import torch

from geo_b200 import _lib, functional as F, layers, ops, train


def i8(*shape):
    return torch.zeros(*shape, dtype=torch.int8)


@pytest.mark.parametrize("call, error", [
    (lambda: F.rms_norm_int8(torch.zeros(2, 8, dtype=torch.float64), torch.ones(8)), TypeError),
    (lambda: F.rms_norm_int8(torch.zeros(2, 8), torch.ones(7)), ValueError),
    (lambda: F.rms_norm_int8(torch.zeros(2, 8), torch.ones(8), eps=-1.0), ValueError),
    (lambda: F.rms_norm_int8(torch.zeros(2, 8), torch.ones(8), eps=float("nan")), ValueError),
    (lambda: F.rms_norm_int8(torch.zeros(2, 8), torch.ones(8), residual=torch.zeros(2, 8).bfloat16()), ValueError),
    (lambda: F.rms_norm_int8(torch.zeros(2, 8), torch.ones(8), residual=torch.zeros(1, 8)), ValueError),
    (lambda: F.rms_norm_int8(torch.zeros(2, 0), torch.ones(0)), ValueError),
    (lambda: F.rms_norm_int8(torch.zeros(2, 8, requires_grad=True), torch.ones(8)), RuntimeError),
    (lambda: F.rms_norm_int8(torch.zeros(2, 8), torch.ones(8)), RuntimeError),          # no CPU path
    (lambda: F.quantize_int8(torch.zeros(2, 8, dtype=torch.int32)), TypeError),
    (lambda: F.quantize_int8(torch.tensor(1.0)), ValueError),
    (lambda: F.quantize_int8(torch.zeros(2, 8)), RuntimeError),
    (lambda: F.dequantize_int8(torch.zeros(2, 8), torch.ones(2)), TypeError),
    (lambda: F.dequantize_int8(i8(2, 8), torch.ones(3)), ValueError),
    (lambda: F.dequantize_int8(i8(2, 8), torch.ones(2), torch.int32), TypeError),
    (lambda: F.linear_int8(i8(2, 8), torch.ones(2), i8(3, 9), torch.ones(3)), ValueError),
    (lambda: F.linear_int8(i8(2, 8), torch.ones(3), i8(3, 8), torch.ones(3)), ValueError),
    (lambda: F.linear_int8(i8(2, 8), torch.ones(2), i8(3, 8), torch.ones(3), bias=torch.ones(2)), ValueError),
    (lambda: F.linear_int8(i8(2, 8), torch.ones(2), i8(3, 8), torch.ones(3).half()), TypeError),
    (lambda: F.linear_int8(torch.zeros(2, 8), torch.ones(2), i8(3, 8), torch.ones(3)), TypeError),
    (lambda: F.linear_int8(i8(1, 131072), torch.ones(1), i8(1, 131072), torch.ones(1)), ValueError),
    (lambda: F.linear_int8(i8(2, 8), torch.ones(2), i8(0, 8), torch.ones(0)), ValueError),
    (lambda: F.linear_int8(i8(2, 8), torch.ones(2), i8(3, 8), torch.ones(3)), RuntimeError),
    (lambda: F.distillation_loss(torch.zeros(2, 8), torch.zeros(2, 3), torch.zeros(2, 3)), TypeError),
    (lambda: F.distillation_loss(torch.zeros(2, 8), torch.zeros(2, 3).long(), torch.zeros(2, 4)), ValueError),
    (lambda: F.distillation_loss(torch.zeros(2, 8), torch.zeros(3, 3).long(), torch.zeros(3, 3)), ValueError),
    (lambda: F.distillation_loss(torch.zeros(2, 8), torch.zeros(2, 513).long(), torch.zeros(2, 513)), ValueError),
    (lambda: F.distillation_loss(torch.zeros(2, 8), torch.zeros(2, 3).long(), torch.zeros(2, 3), temperature=0.0), ValueError),
    (lambda: F.distillation_loss(torch.zeros(2, 8), torch.zeros(2, 3).long(), torch.zeros(2, 3), reduction="mean"), ValueError),
    (lambda: F.distillation_loss(torch.zeros(2, 8), torch.zeros(2, 3).long(), torch.zeros(2, 3), weight=torch.ones(3)), ValueError),
    (lambda: F.distillation_loss(torch.zeros(2, 8), torch.zeros(2, 3).long(), torch.zeros(2, 3), scale=float("inf")), ValueError),
    (lambda: F.distillation_loss(torch.zeros(2, 8), torch.zeros(2, 3).long(), torch.zeros(2, 3, requires_grad=True)), ValueError),
    (lambda: F.distillation_loss(torch.zeros(2, 8), torch.zeros(2, 3).long(), torch.zeros(2, 3)), RuntimeError),
])
def test_python_entry_points_refuse(call, error):
    with pytest.raises(error):
        call()


def test_c_entry_points_refuse_before_they_launch():
    """Status codes of the C ABI for arguments that no kernel may see (the pointers are never followed)."""
    L, p = _lib.lib(), ctypes.c_void_p(4096)
    odd = ctypes.c_void_p(4097)
    SHAPE, NULL, LARGE, UNSUPPORTED = -3, -1, -6, -9
    assert L.geo_sc_linear_int8(1, 1, 131072, p, 131072, p, p, 131072, p, None, 0, p, 1, None) == LARGE
    assert L.geo_sc_linear_int8(1, 1, 0, p, 16, p, p, 16, p, None, 0, p, 1, None) == SHAPE
    assert L.geo_sc_linear_int8(1, 1, 16, odd, 16, p, p, 16, p, None, 0, p, 1, None) == UNSUPPORTED
    assert L.geo_sc_linear_int8(1, 1, 16, p, 17, p, p, 16, p, None, 0, p, 1, None) == UNSUPPORTED
    assert L.geo_sc_linear_int8(1, 1, 16, p, 16, p, p, 16, p, None, 3, p, 1, None) == UNSUPPORTED
    assert L.geo_sc_linear_int8(1, 2, 16, p, 16, p, p, 16, p, None, 0, p, 1, None) == SHAPE
    assert L.geo_sc_linear_int8(1, 1, 16, p, 16, None, p, 16, p, None, 0, p, 1, None) == NULL
    assert L.geo_sc_linear_int8(0, 1, 16, None, 16, None, None, 16, None, None, 0, None, 1, None) == 0
    assert L.geo_sc_quantize_int8(1, 0, 0, p, 0, p, 0, p, None) == SHAPE
    assert L.geo_sc_quantize_int8(1, 8, 0, None, 8, p, 16, p, None) == NULL
    assert L.geo_sc_quantize_int8(1, 8, 0, p, 8, p, 4, p, None) == SHAPE
    assert L.geo_sc_rms_norm_int8(1, 8, 0, p, 8, p, 8, p, 0, 1e-6, None, p, 16, p, None) == NULL
    assert L.geo_sc_rms_norm_int8(1, 8, 0, p, 8, None, 0, p, 7, 1e-6, None, p, 16, p, None) == UNSUPPORTED
    assert L.geo_sc_rms_norm_int8(1, 8, 0, p, 8, None, 0, p, 0, float("nan"), None, p, 16, p, None) == SHAPE
    assert L.geo_sc_rms_norm_int8(1 << 40, 8, 0, p, 8, None, 0, p, 0, 1e-6, None, p, 16, p, None) == LARGE
    assert L.geo_sc_dequantize_int8(1, 8, p, 16, None, 0, p, None) == NULL
    forward = L.geo_sc_distill_forward
    assert forward(1, 8, 513, 0, p, 8, p, 64, p, 0, None, 1.0, 1.0, 1, p, p, p, None, None) == LARGE
    assert forward(1, 8, 3, 0, p, 8, p, 16, p, 0, None, 1.0, 1.0, 1, p, p, p, None, None) == UNSUPPORTED
    assert forward(1, 8, 3, 0, p, 8, p, 64, p, 0, None, 0.0, 1.0, 1, p, p, p, None, None) == SHAPE
    assert forward(1, 8, 3, 0, p, 8, p, 64, p, 0, None, 1.0, 1.0, 1, p, p, None, None, None) == NULL
    assert L.geo_sc_distill_backward(1, 8, 3, 0, p, 8, p, 64, p, 0, None, 1.0, 1.0, 1, p, None, 0, p, None) == NULL
    assert L.geo_sc_distill_backward(0, 8, 3, 0, None, 8, None, 64, None, 0, None, 1.0, 1.0, 1, None, None, 0, None, None) == 0


def test_training_step_and_its_teacher_come_together():
    model = torch.nn.Linear(4, 4)
    with pytest.raises(ValueError):
        train.TrainStep(model, distillation=layers.DistillationLoss(reduction="none"))
    with pytest.raises(ValueError):
        train.TrainStep(model, distillation=layers.DistillationLoss())(torch.zeros(2, 4), torch.zeros(2).long())
    with pytest.raises(ValueError):
        train.TrainStep(model)(torch.zeros(2, 4), torch.zeros(2).long(), teacher=(torch.zeros(2, 1).long(), torch.zeros(2, 1)))


def test_rows_for_the_product_are_padded():
    assert layers.Linear_Int8(17, 5).weight_q.shape == (5, 32)
    assert layers.Linear_Int8(32, 5).weight_q.shape == (5, 32)


def test_launch_count_is_one_number():
    stats = ops._Stats()
    ops._lib.rows()
    stats.reset()
    stats.launches += 3
    assert stats.launches == 3
    stats.reset()
    assert stats.launches == 0
