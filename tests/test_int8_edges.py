"""8-bit operators and the distillation loss: what can be said of their calls without a GPU."""
import pytest
import torch

from geo_b200 import functional as F, layers, train


def i8(*shape):
    return torch.zeros(*shape, dtype=torch.int8)


def test_kernels_launched_ahead_read_by_plain_loads():
    """A kernel that is launched while the one in front of it still writes reads nothing through the read-only path, which is
    promised only for memory that nobody writes as long as the kernel lives (nor may such a load be kept behind the wait)."""
    import os
    import re

    csrc = os.path.join(os.path.dirname(os.path.abspath(layers.__file__)), "csrc")
    ahead = []
    for name in sorted(os.listdir(csrc)):
        with open(os.path.join(csrc, name)) as f:
            code = re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)
        if "launch_behind(" in code:
            ahead.append(name)
            assert not re.search(r"\b__ldg\b|ld\.global\.nc|\b__restrict__\b", code), name
    assert {"sc_norm_int8.cu", "sc_linear_int8.cu", "sc_linear_int8_tc.cu", "sc_distill.cu"} <= set(ahead)


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.float16), lambda m: m.double(),
                                  lambda m: torch.nn.Sequential(m).to(torch.bfloat16)[0]])
def test_cast_layers_keep_their_scales(cast):
    """Scales and bias of the 8-bit layer are part of its arithmetic, not of the model's element type."""
    layer = layers.Linear_Int8(17, 5)
    layer.weight_scale.copy_(torch.rand(5) + 1 / 3)
    layer.bias.copy_(torch.rand(5) + 1 / 3)
    scale, bias = layer.weight_scale.clone(), layer.bias.clone()
    layer = cast(layer)
    assert layer.weight_q.dtype == torch.int8
    assert torch.equal(layer.weight_scale, scale) and torch.equal(layer.bias, bias)
    assert set(layer.state_dict()) == {"weight_q", "weight_scale", "bias"}
    with pytest.raises(RuntimeError, match="CUDA tensors only"):     # refused for the device, not for a type
        layer((i8(2, 17), torch.ones(2)))
    assert cast(layers.Linear_Int8(17, 5, bias=False)).bias is None


@pytest.mark.parametrize("call", [
    lambda dual: F.rms_norm_int8(dual(2, 8), torch.ones(8)),
    lambda dual: F.rms_norm_int8(torch.zeros(2, 8), dual(8)),
    lambda dual: F.rms_norm_int8(torch.zeros(2, 8), torch.ones(8), residual=dual(2, 8)),
    lambda dual: F.quantize_int8(dual(2, 8)),
    lambda dual: F.dequantize_int8(i8(2, 8), dual(2)),
    lambda dual: F.linear_int8(i8(2, 8), dual(2), i8(3, 8), torch.ones(3)),
    lambda dual: F.linear_int8(i8(2, 8), torch.ones(2), i8(3, 8), dual(3)),
    lambda dual: F.linear_int8(i8(2, 8), torch.ones(2), i8(3, 8), torch.ones(3), bias=dual(3)),
])
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(call, grad):
    """Forward-mode derivatives are not dropped without a word, under no_grad (which does not concern them) neither."""
    import torch.autograd.forward_ad as ad

    with ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(RuntimeError, match="evaluation only"):
            call(lambda *shape: ad.make_dual(torch.ones(*shape), torch.ones(*shape)))


def test_replayed_step_refuses_a_teacher_of_another_form():
    """A captured step copies the teacher's entries into its own: what does not correspond is named, not left out."""
    class Replay:
        def replay(self):
            raise AssertionError("replayed")

    step = train.TrainStep(torch.nn.Linear(4, 4), graph=True, distillation=layers.DistillationLoss())
    entries = (torch.zeros(2, 3).long(), torch.zeros(2, 3), torch.ones(2))      # with a weight per row
    step._graph, step._static = Replay(), (torch.zeros(2, 4), torch.zeros(2).long(), entries, None, None)
    for teacher in (entries[:2], entries[:1], (*entries, torch.ones(2))):
        with pytest.raises(ValueError):
            step(torch.zeros(2, 4), torch.zeros(2).long(), teacher=teacher)


def test_scale_of_a_sum_that_leaves_the_range_is_refused():
    """The kernels take the scale times the number of rows; past 32 bits the loss would be infinite."""
    entries = torch.zeros(4096, 1).long(), torch.zeros(4096, 1)
    with pytest.raises(ValueError):
        F.distillation_loss(torch.zeros(4096, 8), *entries, reduction="sum", scale=1e36)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        F.distillation_loss(torch.zeros(4096, 8), *entries, reduction="batchmean", scale=1e36)


def test_no_thread_block_leaves_with_copies_or_instructions_in_flight():
    """What a wait that runs out leaves behind is waited for (with a bound) after the roles of all warps, whichever of them
    gave up, and before tensor memory is freed."""
    import os
    import re

    with open(os.path.join(os.path.dirname(os.path.abspath(layers.__file__)), "csrc", "sc_linear_int8_tc.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    kernel = code[code.index("linear_int8_tc_kernel(") : code.index("EncodeTiledFn encode_fn")]
    roles, end = kernel[: kernel.rindex("mbar_arrive_leader")], kernel[kernel.rindex("mbar_arrive_leader") :]
    assert "mbar_drain" not in roles
    order = [end.index(step) for step in ("__syncthreads();", "store_remote(smem_u32(other)", "tile_sync<CTAS == 2 || SPLIT>();", "if (abort_flag || ",
                                          "mbar_drain(full_bar", "umma_commit<CTAS>(drain_bar)", "mbar_drain(drain_bar", "tile_sync<CTAS == 2>();",
                                          "tmem_free<CTAS>")]
    assert order == sorted(order)


def test_a_warp_that_reads_tensor_memory_stops_as_a_whole():
    """The reads are instructions of a whole warp: its lanes, which look at the barrier and the flag one by one, agree first."""
    import os
    import re

    with open(os.path.join(os.path.dirname(os.path.abspath(layers.__file__)), "csrc", "sc_linear_int8_tc.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert re.findall(r"if \(!(.*?)mbar_wait\(accf_bar", code) == ["__all_sync(0xffffffffu, "]


def test_c_entry_points_refuse_stats_between_boundaries():
    """The rows' statistics are read and written 8 bytes at a time (the pointers are never followed)."""
    import ctypes

    from geo_b200 import _lib

    L, p, between, UNSUPPORTED = _lib.lib(), ctypes.c_void_p(4096), ctypes.c_void_p(4100), -9
    assert L.geo_sc_distill_forward(1, 8, 3, 0, p, 8, p, 64, p, 0, None, 1.0, 1.0, 1, p, between, p, None, None) == UNSUPPORTED
    assert L.geo_sc_distill_backward(1, 8, 3, 0, p, 8, p, 64, p, 0, None, 1.0, 1.0, 1, between, p, 0, p, None) == UNSUPPORTED
