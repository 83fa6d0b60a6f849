"""Distillation and cross entropy, forward and backward, against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

_TYPES = [torch.float16, torch.bfloat16, torch.float32]
_INF = float("inf")


def _formula(z, tid, tlog, labels, temperature, weight, ignore=-100):
    """Losses and gradients in 64 bits, with the rules for absent entries, labels and empty rows."""
    z = z.double()
    n, V = z.shape
    loss, grad = torch.zeros(n, dtype=torch.float64, device=z.device), torch.zeros_like(z)
    empty = (z == -_INF).all(-1)
    rows = torch.arange(n, device=z.device)
    if labels is not None and weight != 1:
        y = labels.reshape(-1).long()
        real = (y != ignore) & (y >= 0) & (y < V) & ~empty
        y = torch.where(real, y, 0)
        log_s = torch.log_softmax(z, -1)
        loss += torch.where(real, -(1 - weight) * log_s[rows, y], 0)
        g = log_s.exp()
        g[rows, y] -= 1
        grad += torch.where(real[:, None], (1 - weight) * g, 0)
    if tid is not None and weight != 0:
        tid, t = tid.reshape(n, -1).long(), tlog.reshape(n, -1).double()
        there = (tid >= 0) & (tid < V)
        t = torch.where(there, t, -_INF)
        some = (t > -_INF).any(-1) & ~empty
        p = torch.where(some[:, None], torch.softmax(t / temperature, -1), 0)
        p = torch.where(there, p, 0)
        log_q = torch.log_softmax(z / temperature, -1)
        cross = torch.where(p > 0, p * log_q.gather(1, torch.where(there, tid, 0)), 0)
        loss += torch.where(some, weight * temperature ** 2 * (torch.special.xlogy(p, p) - cross).sum(-1), 0)
        g = log_q.exp().scatter_add(1, torch.where(there, tid, 0), -p)
        grad += torch.where(some[:, None], weight * temperature * g, 0)
    return loss, grad


def _span(x):
    """Distance of the smallest from the largest value of every row (without masked ones), and log of the width and one."""
    x = x.reshape(-1, x.shape[-1]).double()
    there = x.isfinite() & (x > -1000)
    high, low = torch.where(there, x, -_INF).max(-1)[0], torch.where(there, x, _INF).min(-1)[0]
    return torch.where(there.any(-1), high - low, 0) + math.log(x.shape[-1]) + 1


def _check(z, tid, tlog, labels, temperature, weight, scale=3.0, per_row=True):
    """All three forms against the formula.

    Losses: fp32 sums of V positive terms in a tree of partial sums, exponentials good to 2^-21 and logarithms to 2^-20
    of the loss's terms, whose largest is T^2 a (or 1 - a) times the distance of a logit from the largest (<= `span`).
    Gradients: fp32 values of at most g (1 + T) with relative errors of 2^-18 (the exponent of up to `span` / T in fp32),
    rounded to the type."""
    from terapipe_b200.ops import functional as F
    n, V = z.shape
    g = torch.Generator(device="cuda").manual_seed(n + V)
    gl = torch.rand(n, device="cuda", generator=g) if per_row else None
    loss64, grad64 = _formula(z, tid, tlog, labels, temperature, weight)
    grad64 = grad64 * scale * (gl.double()[:, None] if per_row else 1.0)
    span, span_t = _span(z), 0.0 if tlog is None else _span(tlog)
    size = (1 - weight) * span + weight * temperature ** 2 * (span + span_t) / min(1.0, temperature)      # per row
    eps = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[z.dtype]
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}[z.dtype]
    how = {} if tid is None else {"temperature": temperature, "teacher_weight": weight}
    fwd, bwd, both = ((F.cross_entropy_fwd, F.cross_entropy_bwd, F.cross_entropy_fwd_bwd) if tid is None else
                      (F.distill_fwd, F.distill_bwd, F.distill_fwd_bwd))
    teacher = () if tid is None else (tid, tlog)
    before = z.clone()
    loss_a, stats = fwd(z, *teacher, labels, **how)
    grad_a = bwd(z, stats, *teacher, labels, **how, grad_loss=gl, grad_scale=scale)
    loss_b, grad_b = both(z, *teacher, labels, **how, grad_loss=gl, grad_scale=scale)
    assert torch.equal(z, before)
    inplace = z.clone() if z.is_contiguous() else z
    loss_c, grad_c = both(inplace, *teacher, labels, **how, grad_loss=gl, grad_scale=scale, dlogits=inplace)
    assert grad_c is inplace
    row = (gl.double() if per_row else torch.ones(n, device="cuda", dtype=torch.float64))[:, None] * scale
    for loss in (loss_a, loss_b, loss_c):
        assert torch.equal(loss.double().isinf(), loss64.isinf())
        ok = loss64.isfinite()
        assert ((loss.double() - loss64)[ok].abs() <= (2.0 ** -20 * size)[ok]).all()
    for grad in (grad_a, grad_b, grad_c):
        err = (grad.double() - grad64).abs()
        assert (err <= eps * grad64.abs() + tiny + row * (1 + temperature) * (1 + span[:, None] / temperature / 16) * 2.0 ** -20).all()
    # nothing may leak into rows without a term
    nothing = grad64.abs().sum(-1) == 0
    assert (grad_b[nothing] == 0).all() and (loss_b[loss64 == 0] == 0).all()
    return loss_b, grad_b


def _logits(n, V, dtype, g, std=3.0):
    return (torch.randn(n, V, device="cuda", generator=g) * std).to(dtype)


def _teacher(n, V, K, g, dtype=torch.float32, ids=torch.int64):
    tid = torch.stack([torch.randperm(V, device="cuda", generator=g)[:K] for _ in range(n)])
    return tid.to(ids), (torch.randn(n, K, device="cuda", generator=g) * 2 + 3).to(dtype)


# V: one, fewer than a granule, around one and several rounds of a block, rows on every 2-byte offset, longer than what a
# block holds of a row
_SIZES = [(1, 1), (3, 5), (5, 129), (130, 1000), (3, 4099), (300, 8192), (17, 32001), (9, 50257), (2, 131072), (1, 300007)]


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("n,V", _SIZES)
def test_cross_entropy(n, V, dtype):
    g = torch.Generator(device="cuda").manual_seed(V)
    z = _logits(n, V, dtype, g)
    labels = torch.randint(0, V, (n,), device="cuda", generator=g)
    labels[n // 2] = -100
    if n > 2:
        labels[0], labels[1] = V + 3, V - 1
    _check(z, None, None, labels.int() if n % 2 else labels, 1.0, 0.0)


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("n,V", _SIZES)
@pytest.mark.parametrize("temperature,weight", [(1.0, 1.0), (2.0, 0.5), (1.0, 0.3), (0.7, 1.0), (3.3, 0.9)])
def test_distillation(n, V, temperature, weight, dtype):
    g = torch.Generator(device="cuda").manual_seed(V + n)
    z = _logits(n, V, dtype, g)
    K = min(V, 1 + n * 7 % 97)
    tid, tlog = _teacher(n, V, K, g, _TYPES[n % 3], torch.int32 if V % 2 else torch.int64)
    labels = torch.randint(0, V, (n,), device="cuda", generator=g)
    labels[-1] = tid[-1, 0]                       # the teacher's first choice
    if n > 2:
        labels[0] = -100                          # the teacher's term only
        tid[1] = -1                               # the label's term only
        tid[2, K // 2:], tlog[2, K // 2:] = V, float("nan")     # fewer entries
        labels[1] = 0
    if n > 4:
        labels[3], tid[3] = -100, -7              # neither
        z[3] = float("nan")
    _check(z if n <= 4 else torch.where(torch.arange(n, device="cuda")[:, None] == 3, 0, z), tid, tlog, labels, temperature,
           weight)
    if n > 4:
        # a row without a term is zero whatever its logits are
        from terapipe_b200.ops import functional as F
        loss, grad = F.distill_fwd_bwd(z, tid, tlog, labels, temperature=temperature, teacher_weight=weight)
        assert loss[3] == 0 and (grad[3] == 0).all() and not loss.isnan().any()


@pytest.mark.parametrize("K", [1, 2, 31, 33, 256, 1000, 1024])
def test_entries(K):
    """Any number of entries; the same id more than once adds up."""
    g = torch.Generator(device="cuda").manual_seed(K)
    z = _logits(6, 2048, torch.bfloat16, g)
    tid, tlog = _teacher(6, 2048, K, g)
    labels = tid[:, -1].clone()
    _check(z, tid, tlog, labels, 2.0, 0.5)
    tid[1] = int(tid[1, 0])                        # one id only
    tid[2, K // 2:] = int(tid[2, 0])
    tid[3] = torch.randint(0, 7, (K,), device="cuda", generator=g)
    labels[3] = 2
    _check(z, tid, tlog, labels, 2.0, 0.5)
    _check(z, tid, tlog, None, 1.5, 1.0)


@pytest.mark.parametrize("dtype", _TYPES)
def test_masked_logits(dtype):
    """-inf and the type's lowest value in masked columns, rows with one column or none left, large offsets."""
    g = torch.Generator(device="cuda").manual_seed(5)
    V = 3001
    z = _logits(8, V, dtype, g)
    tid, tlog = _teacher(8, V, 16, g)
    labels = torch.randint(0, V - 60, (8,), device="cuda", generator=g)
    tid = torch.where(tid >= V - 50, tid - 100, tid)
    z[0:3, V - 50:] = -_INF
    z[3, V - 50:] = -65504.0
    z[4] = -_INF
    z[4, labels[4]] = 2.0                         # one column left, the label's
    tid[4], tlog[4] = labels[4], 0.0
    z[5] = -_INF                                  # none
    z[6] = z[6] / 4 + 500.0 if dtype != torch.bfloat16 else z[6] + 256.0
    tlog[7] = -65504.0                            # all alike: a uniform teacher
    tlog[6, 3:] = -_INF
    for temperature, weight in ((1.0, 1.0), (2.0, 0.5), (1.0, 0.5)):
        _check(z, tid, tlog, labels, temperature, weight)
    _check(z, None, None, labels, 1.0, 0.0)
    tlog[2] = -_INF                               # a teacher with no probability anywhere: as no teacher
    z[1, labels[1]] = -_INF                       # an impossible label: an infinite loss, finite gradients
    z[0, tid[0, 2]] = -_INF
    _check(z, tid, tlog, labels, 2.0, 0.5)


def test_nan_and_inf_are_not_hidden():
    from terapipe_b200.ops import functional as F
    z = torch.zeros(4, 5000, device="cuda")
    z[0, 4321], z[1, 17], z[2] = float("nan"), _INF, float("nan")
    labels = torch.tensor([1, 2, 3, 4], device="cuda")
    loss, grad = F.cross_entropy_fwd_bwd(z, labels)
    assert loss[:3].isnan().all() and grad[0].isnan().all() and grad[2].isnan().all() and not loss[3].isnan()
    assert F.cross_entropy_fwd(z, labels)[0][:3].isnan().all()


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("offset,ld,ld_out", [(0, 4104, 4104), (1, 4105, 4105), (3, 4200, 4111), (8, 4128, 4100)])
def test_strided_tensors(offset, ld, ld_out, dtype):
    """Rows of wider matrices, gradients on another alignment than the logits, sequence-first views of batch-first arrays."""
    from terapipe_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(ld)
    B, L, V, K = 3, 7, 4091, 20
    z = torch.empty(L * B, ld, device="cuda", dtype=dtype)[:, offset:offset + V]
    z.copy_(_logits(L * B, V, dtype, g))
    out = torch.full((L * B, ld_out), 9.0, device="cuda", dtype=dtype)
    labels = torch.randint(0, V, (B, L), device="cuda", generator=g).t()
    tid, tlog = _teacher(L * B, V, K, g)
    tid = torch.cat([tid.view(L, B, K).transpose(0, 1), tid.new_zeros(B, L, 3)], -1)[..., :K].transpose(0, 1)
    tlog = tlog.view(L, B, K).transpose(0, 1).contiguous().transpose(0, 1)
    loss64, grad64 = _formula(z, tid, tlog, labels, 2.0, 0.5)
    loss, grad = F.distill_fwd_bwd(z, tid, tlog, labels, temperature=2.0, teacher_weight=0.5, dlogits=out[:, :V])
    eps = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[dtype]
    assert ((loss.double() - loss64).abs() <= 2.0 ** -20 * 100).all()
    assert ((grad.double() - grad64).abs() <= eps * grad64.abs() + 2.0 ** -18).all()
    assert torch.equal(out[:, :V], grad) and (out[:, V:] == 9.0).all()
    loss2, stats = F.distill_fwd(z, tid, tlog, labels, temperature=2.0, teacher_weight=0.5)
    out[:, :V] = 9.0
    grad2 = F.distill_bwd(z, stats, tid, tlog, labels, temperature=2.0, teacher_weight=0.5, dlogits=out[:, :V])
    assert ((grad2.double() - grad64).abs() <= eps * grad64.abs() + 2.0 ** -18).all()
    assert (out[:, V:] == 9.0).all() and ((loss2.double() - loss64).abs() <= 2.0 ** -20 * 100).all()
    # a [L, B, V] view is as good as its rows
    if offset == 0:
        loss3, _ = F.distill_fwd(z.view(L, B, V), tid, tlog, labels, temperature=2.0, teacher_weight=0.5)
        assert torch.equal(loss3, loss2)


def test_gradient_against_differences():
    """Central differences of the kernel's own fp32 losses: a step of 2^-5 leaves an error of (2^-5)^2 / 6 of a third
    derivative below 1, and 2^-20 * size / 2^-5 of the losses' rounding."""
    from terapipe_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(3)
    V, h = 40, 2.0 ** -5
    z = _logits(1, V, torch.float32, g, 1.0)
    tid, tlog = _teacher(1, V, 5, g)
    labels = tid[:, 1]
    how = {"temperature": 2.0, "teacher_weight": 0.5}
    _, grad = F.distill_fwd_bwd(z, tid, tlog, labels, **how)
    step = torch.eye(V, device="cuda") * h
    rep = (tid.expand(V, 5).contiguous(), tlog.expand(V, 5).contiguous(), labels.expand(V).contiguous())
    up, _ = F.distill_fwd(z + step, *rep, **how)
    down, _ = F.distill_fwd(z - step, *rep, **how)
    assert ((up - down) / (2 * h) - grad[0]).abs().max() < h * h / 6 + 2.0 ** -20 * 40 / h


def test_repeats_are_bit_identical_and_graphs_replay():
    from terapipe_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(8)
    z = _logits(200, 20011, torch.bfloat16, g)
    tid, tlog = _teacher(200, 20011, 40, g)
    labels = torch.randint(0, 20011, (200,), device="cuda", generator=g)
    out, loss = torch.empty_like(z), torch.empty(200, device="cuda")
    how = {"temperature": 2.0, "teacher_weight": 0.5, "loss": loss, "dlogits": out}
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        F.distill_fwd_bwd(z, tid, tlog, labels, **how)
    s.synchronize()
    first = (loss.clone(), out.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        F.distill_fwd_bwd(z, tid, tlog, labels, **how)
    for _ in range(3):
        out.zero_(), loss.zero_()
        graph.replay()
        assert torch.equal(loss, first[0]) and torch.equal(out, first[1])


def test_no_rows_and_no_columns():
    from terapipe_b200.ops import functional as F
    z = torch.empty(0, 50, device="cuda", dtype=torch.float16)
    loss, grad = F.cross_entropy_fwd_bwd(z, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert loss.shape == (0,) and grad.shape == (0, 50)
    z = torch.empty(3, 0, device="cuda", dtype=torch.float16)
    loss, grad = F.cross_entropy_fwd_bwd(z, torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert (loss == 0).all() and grad.shape == (3, 0)
    # no entries at all, and labels left out
    z = torch.randn(3, 64, device="cuda")
    none = torch.empty(3, 0, dtype=torch.int64, device="cuda"), torch.empty(3, 0, device="cuda")
    loss, grad = F.distill_fwd_bwd(z, *none)
    assert (loss == 0).all() and (grad == 0).all()


def test_labels_beside_a_teacher_without_entries():
    """No room for entries at all: the label's term alone, at a temperature of 1."""
    g = torch.Generator(device="cuda").manual_seed(6)
    z, labels = _logits(20, 3001, torch.float16, g), torch.randint(0, 3001, (20,), device="cuda", generator=g)
    none = torch.empty(20, 0, dtype=torch.int64, device="cuda"), torch.empty(20, 0, device="cuda")
    from terapipe_b200.ops import functional as F
    how = {"temperature": 2.0, "teacher_weight": 0.25}
    loss64, grad64 = _formula(z, None, None, labels, 1.0, 0.25)
    loss, grad = F.distill_fwd_bwd(z, *none, labels, **how)
    loss2, stats = F.distill_fwd(z, *none, labels, **how)
    grad2 = F.distill_bwd(z, stats, *none, labels, **how)
    for a, b in ((loss, grad), (loss2, grad2)):
        assert ((a.double() - loss64).abs() <= 2.0 ** -20 * 40).all()
        assert ((b.double() - grad64).abs() <= 2.0 ** -11 * grad64.abs() + 2.0 ** -18).all()


def test_rows_beyond_32_bit_offsets():
    """The last rows of a matrix of more than 2^32 elements."""
    from terapipe_b200.ops import functional as F
    n, V = 34000, 131072
    z = torch.empty(n, V, device="cuda", dtype=torch.bfloat16)
    z[:2] = 0.0
    last = z[n - 130:]
    g = torch.Generator(device="cuda").manual_seed(2)
    last.copy_(_logits(130, V, torch.bfloat16, g))
    labels = torch.full((n,), -100, device="cuda")
    labels[n - 130:] = torch.randint(0, V, (130,), device="cuda", generator=g)
    loss, grad = F.cross_entropy_fwd_bwd(z, labels, dlogits=z)
    g = torch.Generator(device="cuda").manual_seed(2)
    loss64, grad64 = _formula(_logits(130, V, torch.bfloat16, g), None, None, labels[n - 130:], 1.0, 0.0)
    assert (loss[:n - 130] == 0).all() and ((loss[n - 130:].double() - loss64).abs() <= 2.0 ** -20 * 50).all()
    assert ((grad[n - 130:].double() - grad64).abs() <= 2.0 ** -8 * grad64.abs() + 2.0 ** -18).all()
    assert (grad[:2] == 0).all()


def test_refusals():
    from terapipe_b200.ops import functional as F
    from terapipe_b200.ops.lib import KernelError
    z, y = torch.zeros(6, 64, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda")
    tid, tlog = torch.zeros(6, 4, dtype=torch.int64, device="cuda"), torch.zeros(6, 4, device="cuda")
    wide = torch.zeros(6, 1025, dtype=torch.int64, device="cuda")
    _, stats = F.cross_entropy_fwd(z, y)
    for bad in (lambda: F.cross_entropy_fwd(z.double(), y), lambda: F.cross_entropy_fwd(z, y.float()),
                lambda: F.cross_entropy_fwd(z, y[:5]), lambda: F.cross_entropy_fwd(z.t(), y),
                lambda: F.cross_entropy_fwd(z, y.cpu()), lambda: F.cross_entropy_fwd(z.cpu(), y),
                lambda: F.cross_entropy_fwd(z, y, loss=torch.empty(6, device="cuda", dtype=torch.float16)),
                lambda: F.cross_entropy_fwd(z, y, loss=torch.empty(5, device="cuda")),
                lambda: F.cross_entropy_bwd(z, None, y), lambda: F.cross_entropy_bwd(z, stats[:5], y),
                lambda: F.cross_entropy_bwd(z, stats, y, dlogits=z.half()),
                lambda: F.cross_entropy_bwd(z, stats, y, dlogits=z[:, :32]),
                lambda: F.cross_entropy_bwd(z, stats, y, grad_loss=torch.ones(5, device="cuda")),
                lambda: F.cross_entropy_bwd(z, stats, y, grad_loss=torch.ones(6, device="cuda", dtype=torch.float16)),
                lambda: F.cross_entropy_fwd_bwd(z[:4], y[:4], dlogits=z[1:5]),
                lambda: F.cross_entropy_fwd_bwd(z, y, dlogits=torch.empty(1, 64, device="cuda").expand(6, 64)),
                lambda: F.distill_fwd(z, tid, tlog[:, :3]), lambda: F.distill_fwd(z, tid.float(), tlog),
                lambda: F.distill_fwd(z, tid, tlog.double()), lambda: F.distill_fwd(z, tid[:5], tlog[:5]),
                lambda: F.distill_fwd(z, tid.t().contiguous().t(), tlog), lambda: F.distill_fwd(z, wide, wide.float()),
                lambda: F.distill_fwd(z, tid, tlog, temperature=0.0),
                lambda: F.distill_fwd(z, tid, tlog, temperature=float("nan")),
                lambda: F.distill_fwd(z, tid, tlog, teacher_weight=1.5)):
        with pytest.raises(KernelError):
            bad()
