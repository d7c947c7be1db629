"""8-bit operators and the distillation loss: what can be said of their calls without a GPU."""
import pytest
import torch

from geo_b200 import functional as F, layers, train


def i8(*shape):
    return torch.zeros(*shape, dtype=torch.int8)
