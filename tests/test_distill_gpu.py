"""Distillation loss and its gradient against the formulas in 64 bits on the CPU."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(logits, indices, teacher, T, weight, scale, up):
    """(row losses, gradient, bound of the losses' error, bound of the gradient's) in 64 bits; `up` per row.

    Bounds: an exponential's argument is off by some half steps of itself (product, constant; 2^-22 |a| with |a| below 64
    in what carries a sum: 2^-16), ex2 by 2^-22, a sum of up to 2^17 terms by 2^-17 (at most 512 terms one after the
    other in a thread, then joined): 2^-15 covers q, p and their logarithms' absolute error."""
    z, w = logits.detach().cpu().double(), (torch.ones(logits.shape[0]) if weight is None else weight.cpu()).double()
    idx, t = indices.cpu().long(), teacher.cpu().double() / T
    t = torch.where(idx >= 0, t, -math.inf)
    live = (t > -math.inf).any(-1) & (w != 0)
    logp = torch.log_softmax(torch.where(live[:, None], t, 0.0), -1)
    p = torch.where(live[:, None], logp.exp(), 0.0)
    logq = torch.log_softmax(torch.where(live[:, None], z, 0.0) / T, -1)
    at = idx.clamp(min=0)
    lq = logq.gather(-1, at)
    terms = torch.where(p > 0, p * (logp - lq), 0.0)
    row = torch.where(live, scale * w * T * T * terms.sum(-1), 0.0)
    row_bound = (scale * w * T * T).abs() * torch.where(p > 0, p * (logp.abs() + lq.abs() + 1), 0.0).sum(-1) * 2.0 ** -15
    dense = torch.zeros_like(z).scatter_add_(-1, at, torch.where(idx >= 0, p, 0.0))
    a = (scale * w * T * up.cpu().double() * live)[:, None]
    q = logq.exp()
    grad = torch.where(live[:, None], a * (q - dense), 0.0)
    grad_bound = a.abs() * (q + dense) * 2.0 ** -15 + grad.abs() * torch.finfo(logits.dtype).eps / 2 * (1 + 2.0 ** -8)
    grad_bound = grad_bound + (2.0 ** -25 if logits.dtype == torch.float16 else 2.0 ** -134)
    return row, grad, row_bound, torch.where(live[:, None], grad_bound, 0.0)


def make(rows, vocab, top, dtype, seed, device, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(rows, vocab, generator=g) * spread).to(dtype).to(device).requires_grad_(True)
    indices = torch.stack([torch.randperm(vocab, generator=g)[:top] for _ in range(rows)]).to(device)
    teacher = (torch.randn(rows, top, generator=g) * 2).to(dtype).to(device)
    return logits, indices, teacher


def check(logits, indices, teacher, T=1.0, weight=None, scale=1.0, up=None, reduction="none"):
    from geo_b200 import functional as F

    rows = logits.shape[0]
    loss = F.distillation_loss(logits, indices, teacher, T, weight, reduction, scale)
    per_row = scale / rows if reduction == "batchmean" else scale
    if up is None:
        up = torch.ones(rows if reduction == "none" else (), device=logits.device)
    (grad,) = torch.autograd.grad(loss, logits, up)
    row, g, row_bound, g_bound = reference(logits, indices, teacher, T, weight, per_row, up.expand(rows))
    if reduction == "none":
        assert ((loss.detach().cpu().double() - row).abs() <= row_bound).all()
    else:
        assert abs(float(loss.detach()) - float(row.sum())) <= float(row_bound.sum()) + abs(float(row.sum())) * 2.0 ** -22
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    assert ((grad.cpu().double() - g).abs() <= g_bound).all()
    return loss.detach(), grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, vocab, top", [(1, 1, 1), (256, 10, 3), (5, 2, 2), (9, 100, 100), (33, 1000, 17), (3, 1024, 512), (3, 1025, 40),
                                              (400, 1500, 8), (7, 4099, 64), (2, 33333, 100), (1, 131071, 256), (200, 8192, 31),
                                              (600, 33333, 9), (3, 300001, 20)])
def test_loss_and_gradient_match_the_formula(cuda_device, dtype, rows, vocab, top):
    logits, indices, teacher = make(rows, vocab, top, dtype, rows + vocab, cuda_device)
    g = torch.Generator().manual_seed(1)
    weight = (torch.rand(rows, generator=g) + 0.2).to(cuda_device)
    check(logits, indices, teacher, 2.0, weight, up=torch.randn(rows, generator=g).to(cuda_device))
    check(logits, indices.int(), teacher.float(), 0.7, reduction="batchmean")
    check(logits, indices, teacher, 4.0, scale=3.0, reduction="sum")
    # another upstream gradient than 1 for a scalar loss: the gradient is written anew
    check(logits, indices, teacher, 1.5, weight, up=torch.tensor(-2.5, device=cuda_device), reduction="batchmean")


@pytest.mark.parametrize("vocab", [50, 5000])
def test_padding_empty_rows_and_weights(cuda_device, vocab):
    logits, indices, teacher = make(12, vocab, 9, torch.float32, vocab, cuda_device)
    with torch.no_grad():
        logits[7] = float("nan")         # a row that has no part: its logits are not looked at
        logits[8] = float("inf")
    indices[0, 4:] = -1
    indices[1, :8] = -5
    indices[7] = -1
    indices[9] = -1
    teacher[2, 3] = -math.inf
    teacher[3, 1:] = -math.inf
    teacher[4] = -math.inf
    weight = torch.ones(12, device=cuda_device)
    weight[8] = 0
    weight[5] = -0.5
    loss, grad = check(logits, indices, teacher, 2.0, weight)
    for empty in (4, 7, 8, 9):
        assert loss[empty] == 0 and (grad[empty] == 0).all()
    check(logits, indices, teacher, 2.0, weight, reduction="batchmean")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 3000])
def test_masked_logits(cuda_device, dtype, vocab):
    """Logits of -inf and of the type's lowest value; a row where nothing else is left."""
    logits, indices, teacher = make(6, vocab, 5, dtype, 3, cuda_device)
    with torch.no_grad():
        keep = torch.zeros(6, vocab, dtype=torch.bool, device=cuda_device).scatter_(1, indices, True)
        logits.masked_fill_(~keep & (torch.arange(6, device=cuda_device)[:, None] < 2), -math.inf)
        logits.masked_fill_(~keep & (torch.arange(6, device=cuda_device)[:, None] == 2), torch.finfo(dtype).min)
        logits[4, : vocab // 2] = -math.inf
        indices[4, 0], indices[4, 1:] = vocab - 1, -1
    check(logits, indices, teacher, 0.5)
    with torch.no_grad():
        logits[5] = -math.inf            # no distribution
        logits[3, indices[3, 0]] = -math.inf
    from geo_b200 import functional as F

    loss = F.distillation_loss(logits, indices, teacher, reduction="none")
    (grad,) = torch.autograd.grad(loss.sum(), logits)
    assert loss[5].isnan() and grad[5].isnan().all()
    assert loss[3] == math.inf and grad[3].isfinite().all() and grad[3, indices[3, 0]] < 0
    assert loss[[0, 1, 2, 4]].isfinite().all() and grad[[0, 1, 2, 4]].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [41, 3000, 90001, 300001])
def test_rows_at_the_ends_of_the_type(cuda_device, dtype, vocab):
    """Rows masked by the type's lowest value throughout, or in part by -inf, and rows around the largest value: whatever
    the temperature, logits that are equal have equal probabilities and the others none."""
    logits, indices, teacher = make(4, vocab, 5, dtype, 3, cuda_device)
    with torch.no_grad():
        low = torch.finfo(dtype).min
        logits[0] = low
        logits[1] = -math.inf
        logits[1, : vocab // 3] = low
        indices[1] = torch.arange(5, device=cuda_device)
        logits[2] = 0
        logits[2, 3] = -low
        logits[2, vocab - 2] = -low
        indices[2], teacher[2, 1:] = 3, -math.inf
    for T in (0.5, 1.0, 3.0):
        check(logits, indices, teacher, T)
        check(logits, indices, teacher, T, reduction="batchmean", up=torch.tensor(3.0, device=cuda_device))


@pytest.mark.parametrize("vocab", [30, 2500])
def test_bad_entries_poison_their_row_only(cuda_device, vocab):
    from geo_b200 import functional as F

    logits, indices, teacher = make(6, vocab, 4, torch.float32, 8, cuda_device)
    clean = F.distillation_loss(logits, indices, teacher, reduction="none")
    (clean_grad,) = torch.autograd.grad(clean.sum(), logits)
    indices[0, 2] = vocab
    indices[1, 0] = 2 ** 40
    teacher[2, 1] = float("nan")
    teacher[3, 1] = math.inf
    loss = F.distillation_loss(logits, indices, teacher, reduction="none")
    (grad,) = torch.autograd.grad(loss.sum(), logits)
    assert loss[:4].isnan().all() and grad[:4].isnan().all()
    assert torch.equal(loss[4:], clean[4:]) and torch.equal(grad[4:], clean_grad[4:])
    mean = F.distillation_loss(logits[4:], indices[4:], teacher[4:])
    assert abs(float(mean) - float(clean[4:].double().mean())) <= 1e-6 * abs(float(mean))


@pytest.mark.parametrize("vocab, top", [(20, 12), (1200, 12), (1200, 33), (1200, 512), (50000, 300)])
def test_one_index_several_times(cuda_device, vocab, top):
    logits, indices, teacher = make(5, vocab, top, torch.float32, 9, cuda_device)
    indices[:, 3] = indices[:, 0]
    indices[:, 7] = indices[:, 0]
    indices[:, 11] = indices[:, 5]
    indices[2] = indices[2, 0]
    first = check(logits, indices, teacher, 2.0)
    again = check(logits, indices, teacher, 2.0)
    assert torch.equal(first[1], again[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(cuda_device, dtype):
    from geo_b200 import functional as F

    base, indices, teacher = make(24, 2000, 6, dtype, 4, cuda_device)
    base = base.detach()
    indices = indices % 1400
    for view in (base[:, :1501], base[:, 1:1502], base[::2, 5:1506], base.t().contiguous().t()[:, :1501], base[:1, :1501].expand(24, 1501)):
        rows = view.shape[0]
        z = view.detach().requires_grad_(True)
        check(z, indices[:rows], teacher[:rows], 2.0)
    z = base[:, :1501].unflatten(0, (4, 6)).detach().requires_grad_(True)
    loss = F.distillation_loss(z, indices.view(4, 6, 6), teacher.view(4, 6, 6), 2.0, reduction="none")
    flat = F.distillation_loss(base[:, :1501], indices, teacher, 2.0, reduction="none")
    assert loss.shape == (4, 6) and torch.equal(loss.detach().view(24), flat)
    assert F.distillation_loss(z[0, 0], indices[0], teacher[0], reduction="none").shape == ()
    empty = base[:0].detach().requires_grad_(True)
    loss = F.distillation_loss(empty, indices[:0], teacher[:0])
    loss.backward()
    assert float(loss) == 0 and empty.grad.shape == (0, 2000)
    assert F.distillation_loss(empty, indices[:0], teacher[:0], reduction="none").shape == (0,)


def test_offsets_past_32_bits(cuda_device):
    """66000 rows of 33000 logits are more than 2^31 values: the last rows as a call of their own gives them."""
    from geo_b200 import functional as F

    rows, vocab, last = 66000, 33000, 5
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=cuda_device)
    g = torch.Generator().manual_seed(6)
    logits[-last:] = torch.randn(last, vocab, generator=g).bfloat16().to(cuda_device)
    logits.requires_grad_(True)
    indices = torch.randint(0, vocab, (rows, 4), generator=g).to(cuda_device)
    teacher = torch.randn(rows, 4, generator=g).to(cuda_device)
    small = logits.detach()[-last:].clone().requires_grad_(True)
    expect = F.distillation_loss(small, indices[-last:], teacher[-last:], 2.0, reduction="none")
    (expect_grad,) = torch.autograd.grad(expect.sum(), small)
    loss = F.distillation_loss(logits, indices, teacher, 2.0, reduction="none")
    (grad,) = torch.autograd.grad(loss.sum(), logits)
    # another team may hold the rows there: the same values but for the order of a sum
    assert (loss[-last:] - expect).abs().max() <= 2.0 ** -18 * expect.abs().max()
    assert (grad[-last:].float() - expect_grad.float()).abs().max() <= 2.0 ** -8 * expect_grad.float().abs().max()
    scalar = F.distillation_loss(logits, indices, teacher, 2.0, reduction="sum")
    (grad,) = torch.autograd.grad(scalar, logits)
    assert (grad[-last:].float() - expect_grad.float()).abs().max() <= 2.0 ** -8 * expect_grad.float().abs().max()


def test_gradient_against_differences(cuda_device):
    """Central differences of the loss itself along random directions of size 1: the third derivative of T^2 logsumexp(z / T)
    is at most (2 / T)^3 T^2 / 4 for |d| <= 1, so h = 1/16 leaves h^2 / 6 of that; the loss is off by 2^-20 of about 8."""
    from geo_b200 import functional as F

    T, h = 2.0, 1 / 16
    logits, indices, teacher = make(64, 12, 4, torch.float32, 12, cuda_device, spread=1.0)
    loss = F.distillation_loss(logits, indices, teacher, T, reduction="none")
    (grad,) = torch.autograd.grad(loss.sum(), logits)
    g = torch.Generator().manual_seed(2)
    for _ in range(4):
        d = (torch.rand(64, 12, generator=g) * 2 - 1).to(cuda_device)
        with torch.no_grad():
            up = F.distillation_loss(logits + h * d, indices, teacher, T, reduction="none").double()
            down = F.distillation_loss(logits - h * d, indices, teacher, T, reduction="none").double()
        bound = h * h / 6 * (2 / T) ** 3 * T * T / 4 + 8 * 2.0 ** -20 / h
        assert ((up - down) / (2 * h) - (grad.double() * d.double()).sum(-1)).abs().max() <= bound


def test_second_backward_and_accumulation(cuda_device):
    """The gradient that the forward pass has written is handed over once; a second pass over the same graph writes its own."""
    from geo_b200 import functional as F

    logits, indices, teacher = make(40, 3001, 16, torch.bfloat16, 21, cuda_device)
    loss = F.distillation_loss(logits, indices, teacher, 2.0)
    (first,) = torch.autograd.grad(loss, logits, retain_graph=True)
    kept = first.clone()
    (second,) = torch.autograd.grad(loss, logits, torch.tensor(2.0, device=cuda_device), retain_graph=True)
    (third,) = torch.autograd.grad(loss, logits)
    assert torch.equal(first, kept) and torch.equal(third, first)
    assert torch.equal(second, (first.float() * 2).bfloat16())
    (F.distillation_loss(logits, indices, teacher, 2.0) + F.distillation_loss(logits, indices, teacher, 2.0)).backward()
    assert torch.equal(logits.grad, (kept.float() * 2).bfloat16())
    with torch.no_grad():
        assert not F.distillation_loss(logits, indices, teacher).requires_grad


def test_differentiable_once(cuda_device):
    from geo_b200 import functional as F

    logits, indices, teacher = make(4, 30, 5, torch.float32, 2, cuda_device)
    (grad,) = torch.autograd.grad(F.distillation_loss(logits, indices, teacher), logits, create_graph=True)
    (plain,) = torch.autograd.grad(F.distillation_loss(logits, indices, teacher), logits)
    assert torch.equal(grad, plain)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_captured_and_on_another_stream(cuda_device):
    from geo_b200 import functional as F

    logits, indices, teacher = make(10, 5000, 20, torch.float32, 31, cuda_device)
    other = make(10, 5000, 20, torch.float32, 32, cuda_device)

    def step(z):
        loss = F.distillation_loss(z, indices, teacher, 2.0)
        return loss, torch.autograd.grad(loss * 1.0, z)[0], torch.autograd.grad(F.distillation_loss(z, indices, teacher, 2.0, scale=2.0), z)[0]

    eager = step(logits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = step(logits)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, aside))
    static = logits.detach().clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static)
    for source in (other[0], logits):
        with torch.no_grad():
            static.copy_(source)
        graph.replay()
        graph.replay()
        expect = step(source)
        assert all(torch.equal(a, b) for a, b in zip(captured, expect))


def test_kernels_in_a_row_wait_for_each_other(cuda_device):
    """Chains of all operators, one after the other into memory that is reused, against the same with the device waited for
    after every call; eagerly and replayed."""
    from geo_b200 import _lib
    from geo_b200 import functional as F

    g = torch.Generator().manual_seed(17)
    cases = []
    for m, n, k, dtype in ((1, 512, 2048, torch.bfloat16), (40, 1001, 513, torch.float32), (300, 10, 4096, torch.float16), (1500, 4096, 64, torch.float32),
                           (3, 4096, 4096, torch.bfloat16), (700, 600, 1100, torch.float16)):
        cases.append((torch.randn(m, k, generator=g).to(dtype).to(cuda_device), torch.randn(n, k, generator=g).to(cuda_device),
                      torch.rand(k, generator=g).to(cuda_device), torch.randint(-1, n, (m, 8), generator=g).to(cuda_device),
                      torch.randn(m, 8, generator=g).to(cuda_device)))

    def chain(case, wait=lambda: None):
        x, w, norm, indices, teacher = case
        out = []
        for step in (lambda: F.quantize_int8(w), lambda: F.rms_norm_int8(x, norm, residual=x),
                     lambda: (F.linear_int8(*out[2:4], *out[:2]).requires_grad_(True),),
                     lambda: (F.dequantize_int8(*out[2:4], x.dtype),),
                     lambda: torch.autograd.grad(F.distillation_loss(out[5], indices, teacher, 2.0), out[5]),
                     lambda: torch.autograd.grad(F.distillation_loss(out[5], indices, teacher, reduction="none").sum(), out[5])):
            out.extend(step())
            wait()
        return [t.detach() for t in out]

    expect = [chain(case, torch.cuda.synchronize) for case in cases]
    for i in [0, 3, 1, 5, 2, 4] * 10:
        assert all(torch.equal(a, b) for a, b in zip(chain(cases[i]), expect[i]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [chain(case) for case in cases]
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got, want in zip(captured, expect) for a, b in zip(got, want))
    assert _lib.device_error_count() == 0


@pytest.mark.parametrize("graph", [False, True])
def test_training_against_a_fixed_point_teacher(cuda_device, graph):
    """A teacher on 8-bit integers (norm, linear layers) scores a batch, its top logits train the stochastic-computing
    network through TrainStep; the student's gradients are those of the two losses added."""
    from geo_b200 import layers, network, train

    torch.manual_seed(0)
    with torch.no_grad():
        norm = layers.RMSNorm_Int8(32 * 32).to(cuda_device)
        hidden = layers.Linear_Int8.from_float(torch.nn.Linear(32 * 32, 64).to(cuda_device))
        head = layers.Linear_Int8.from_float(torch.nn.Linear(64, 10).to(cuda_device))
        x = torch.rand(16, 3, 32, 32, device=cuda_device)
        y = torch.randint(0, 10, (16,), device=cuda_device)
        scores = head(torch.relu(hidden(norm(x[:, 0].flatten(1)))))
        values, indices = torch.topk(scores, 4)
    distill = layers.DistillationLoss(temperature=3.0, scale=0.5)
    models = []
    for _ in range(2):
        torch.manual_seed(1)
        models.append(network.CONV_tiny_add_partial().to(cuda_device))
    step = train.TrainStep(models[0], lr=0.01, graph=graph, distillation=distill)
    loss, out = step(x.clone(), y, teacher=(indices, values))
    # the same step from its parts, the distillation's gradient by elementary operations
    parts = train.TrainStep(models[1], lr=0.01)
    models[1].train()
    logits = models[1](x.clone())
    p = torch.softmax(values / 3.0, -1)
    logq = torch.log_softmax(logits / 3.0, -1).gather(-1, indices)
    kl = (p * (p.log() - logq)).sum(-1).mean() * 9.0 * 0.5
    expect = (torch.nn.functional.cross_entropy(logits, y) + kl) * train.SCALE_FACTOR
    expect.backward()
    parts._update()
    assert torch.equal(out, logits.detach())
    assert abs(float(loss) - float(expect)) <= 1e-4 * abs(float(expect))
    for a, b in zip(models[0].parameters(), models[1].parameters()):
        assert (a - b).abs().max() <= 1e-5
