"""8-bit operators: the scale's error over long rows and at the ends of its range, layers that are cast."""
import pytest
import torch

from test_int8_gpu import STEP32, TYPES, check_norm

pytestmark = pytest.mark.gpu
