"""Distillation loss: rows at the far end of the exponent, and gradients across the border of a captured graph."""
import math

import pytest
import torch

from test_distill_gpu import check, make, reference

pytestmark = pytest.mark.gpu


def far_rows(dtype, vocab, T, device):
    """Rows whose logits are past 2^30 in the exponent z log2(e) / T, with entries on logits that are not the largest."""
    top = {1e-6: 1000.0, 5e-5: 60000.0, 1.0: 2e9}[T]
    logits, indices, teacher = make(5, vocab, 4, dtype, vocab, device)
    with torch.no_grad():
        logits[0, :4] = torch.tensor([top, top * 0.75, 3.0, 4.0], device=device)
        indices[0], teacher[0] = torch.tensor([0, 1, -1, -1], device=device), 0.0
        logits[1] = -top                      # the largest is negative, and twice there
        logits[1, 2:4] = -top * 0.8
        indices[1], teacher[1] = torch.tensor([3, 1, vocab - 1, 2], device=device), 0.5
        logits[2, vocab - 1] = top            # one entry, and it is not the largest logit
        indices[2] = torch.tensor([0, -1, -1, -1], device=device)
        logits[3, 1] = top
        logits[3, 2] = -math.inf              # an entry that the student rules out, without a share
        indices[3], teacher[3] = torch.tensor([1, 2, 0, 0], device=device), torch.tensor([0.0, -math.inf, 1.0, 1.0], device=device)
    return logits, indices, teacher


FAR = [(torch.float32, 1e-6), (torch.float32, 1.0), (torch.bfloat16, 1e-6), (torch.bfloat16, 1.0), (torch.float16, 1e-6), (torch.float16, 5e-5)]


@pytest.mark.parametrize("dtype, T", FAR)
@pytest.mark.parametrize("vocab", [5, 41, 3000, 90001, 300001])
def test_entries_below_the_largest_logit_far_out(cuda_device, dtype, T, vocab):
    """The loss of an entry that is not the row's largest logit is finite, however far its probability lies below the range."""
    logits, indices, teacher = far_rows(dtype, vocab, T, cuda_device)
    loss, _ = check(logits, indices, teacher, T)
    assert loss.isfinite().all() and (loss[:3] > 0).all()
    check(logits, indices, teacher, T, up=torch.tensor([1.0, -2.0, 0.5, 1.0, 3.0], device=cuda_device))
    check(logits, indices, teacher, T, reduction="batchmean")
    check(logits, indices, teacher, T, reduction="sum", up=torch.tensor(-3.0, device=cuda_device))


def test_far_rows_by_hand(cuda_device):
    from geo_b200 import functional as F

    entries, equal = torch.tensor([[0, 1]], device=cuda_device), torch.zeros(1, 2, device=cuda_device)
    loss = F.distillation_loss(torch.tensor([[1000.0, 999.0, 3.0, 4.0]], device=cuda_device), entries, equal, 1e-6)
    # p = 1/2 twice, log q = 0 and -1e6: T^2 (log(1/2) + 1e6 / 2)
    assert abs(float(loss) - 1e-12 * (5e5 - math.log(2))) <= 5e-7 * 2.0 ** -20
    loss = F.distillation_loss(torch.tensor([[2e9, 1e9, 0.0, 1.0]], device=cuda_device), entries, equal)
    assert abs(float(loss) - 5e8) <= 5e8 * 2.0 ** -20
    # the two ends of the type, further apart than the type reaches: T (6e38 / 2)
    loss = F.distillation_loss(torch.tensor([[3e38, -3e38, 0.0, 1.0]], device=cuda_device), entries, equal, 1e-3)
    assert abs(float(loss) - 3e35) <= 3e35 * 2.0 ** -20
    # a student that rules the second entry out
    loss = F.distillation_loss(torch.tensor([[2e9, -math.inf, 0.0, 1.0]], device=cuda_device), entries, equal)
    assert float(loss) == math.inf


@pytest.mark.parametrize("dtype, T", FAR)
@pytest.mark.parametrize("vocab", [41, 3000, 90001, 300001])
def test_nan_among_far_rows(cuda_device, dtype, T, vocab):
    """A NaN logit makes its row's loss and gradient NaN, as it does in every other row."""
    from geo_b200 import functional as F

    logits, indices, teacher = far_rows(dtype, vocab, T, cuda_device)
    with torch.no_grad():
        logits[0, vocab - 2] = math.nan      # no entry
        logits[1, 3] = math.nan              # an entry
    for reduction, up in (("none", torch.ones(5, device=cuda_device)), ("batchmean", None)):
        loss = F.distillation_loss(logits, indices, teacher, T, reduction=reduction)
        (grad,) = torch.autograd.grad(loss, logits, up)
        assert grad[:2].isnan().all() and grad[2:].isfinite().all()
        assert loss.isnan().tolist() == ([True, True, False, False, False] if reduction == "none" else True)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", ["logits", "teacher", "weight"])
def test_tangents_are_refused(cuda_device, which, grad):
    import torch.autograd.forward_ad as ad

    from geo_b200 import functional as F

    logits, indices, teacher = make(4, 20, 3, torch.float32, 1, cuda_device)
    given = {"logits": logits.detach(), "teacher": teacher, "weight": torch.ones(4, device=cuda_device)}
    with ad.dual_level(), torch.set_grad_enabled(grad):
        given[which] = ad.make_dual(given[which], torch.ones_like(given[which]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            F.distillation_loss(given["logits"], indices, given["teacher"], weight=given["weight"])


def test_backward_captured_after_an_eager_forward(cuda_device):
    """The gradient that an eager forward pass has written is not what a captured backward pass hands over: the graph
    writes its own at every replay, whatever the upstream gradient was before or was done with the last one's memory."""
    from geo_b200 import functional as F

    source, indices, teacher = make(7, 3001, 12, torch.float32, 5, cuda_device)
    expect = torch.autograd.grad(F.distillation_loss(source, indices, teacher, 2.0), source)[0]
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        logits = source.detach().clone().requires_grad_(True)
        up = torch.ones((), device=cuda_device)
        loss = F.distillation_loss(logits, indices, teacher, 2.0)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            (grad,) = torch.autograd.grad(loss, logits, up, retain_graph=True)
        for factor in (2.0, 1.0, -1.0, 1.0):
            up.fill_(factor)
            graph.replay()
            assert torch.equal(grad, expect * factor)
        grad.zero_()
        graph.replay()
        assert torch.equal(grad, expect)
        # the eager pass's own gradient is still to be had
        assert torch.equal(torch.autograd.grad(loss, logits, up)[0], expect)
    torch.cuda.current_stream().wait_stream(stream)


@pytest.mark.parametrize("vocab, top", [(10, 3), (10, 9), (3000, 12), (40000, 40)])
def test_c_entry_points_row_by_row(cuda_device, vocab, top):
    """What the C ABI offers beside the front end's calls: the gradient with a loss per row, and a backward pass over it that
    leaves the rows alone whose upstream gradient is 1."""
    import ctypes

    from geo_b200 import _lib

    L, rows, T = _lib.lib(), 9, 2.0
    logits, indices, teacher = make(rows, vocab, top, torch.float32, 4, cuda_device)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    loss, stats = torch.empty(rows, device=cuda_device), torch.empty(rows, 2, device=cuda_device)
    grad = torch.empty(rows, vocab, device=cuda_device)
    _lib.check(L.geo_sc_distill_forward(rows, vocab, top, 0, logits.data_ptr(), vocab, indices.data_ptr(), 64, teacher.data_ptr(), 0, None, T, 1.5, 0,
                                        loss.data_ptr(), stats.data_ptr(), None, grad.data_ptr(), stream), "geo_sc_distill_forward")
    row, expect, row_bound, bound = reference(logits, indices, teacher, T, None, 1.5, torch.ones(rows))
    assert ((loss.cpu().double() - row).abs() <= row_bound).all() and ((grad.cpu().double() - expect).abs() <= bound).all()
    up = torch.tensor([1.0, 2.0, 1.0, -1.0, 0.0, 1.0, 1.0, 0.5, 1.0], device=cuda_device)
    grad[up == 1] = -7.0     # not to be touched
    _lib.check(L.geo_sc_distill_backward(rows, vocab, top, 0, logits.data_ptr(), vocab, indices.data_ptr(), 64, teacher.data_ptr(), 0, None, T, 1.5, 0,
                                         stats.data_ptr(), up.data_ptr(), 1, grad.data_ptr(), stream), "geo_sc_distill_backward")
    _, expect, _, bound = reference(logits, indices, teacher, T, None, 1.5, up)
    assert (grad[up == 1] == -7).all()
    rest = (up != 1).cpu()
    assert ((grad.cpu().double() - expect).abs() <= bound)[rest].all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_walks_over_many_small_rows(cuda_device, dtype):
    """More rows than are resident in a pass that may have nothing to do."""
    logits, indices, teacher = make(20000, 10, 4, dtype, 6, cuda_device)
    check(logits, indices, teacher, 2.0, reduction="batchmean", up=torch.tensor(2.5, device=cuda_device))
    check(logits, indices, teacher, 2.0, reduction="batchmean")


def test_the_largest_vocabulary(cuda_device):
    """2^31 - 1 equal logits that start off a 16-byte boundary: the step past the last one stays in range."""
    from geo_b200 import functional as F

    vocab = 2 ** 31 - 1
    logits = torch.zeros(vocab + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(1, vocab).requires_grad_(True)
    indices = torch.tensor([[5, vocab - 1, 2 ** 30]], device=cuda_device)
    teacher = torch.zeros(1, 3, device=cuda_device)
    loss = F.distillation_loss(logits, indices, teacher, reduction="none")
    assert abs(float(loss.detach()) - (31 * math.log(2) - math.log(3))) <= 22 * 2.0 ** -15
    (grad,) = torch.autograd.grad(loss, logits, torch.ones(1, device=cuda_device))
    assert (grad[0, indices[0]].double() + 1 / 3).abs().max() <= 2.0 ** -8
    assert int((grad == 2.0 ** -31).sum()) == vocab - 3      # 1 / vocab in 16 bits
    del grad
    loss = F.distillation_loss(logits, indices, teacher, weight=torch.zeros(1, device=cuda_device), reduction="none")
    (grad,) = torch.autograd.grad(loss, logits, torch.ones(1, device=cuda_device))
    assert float(loss.detach()) == 0 and int(torch.count_nonzero(grad)) == 0
