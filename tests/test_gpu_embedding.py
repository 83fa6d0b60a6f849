"""Embedding lookup and its gradient against sums in 64 bits: types, strides, shards, absent and frequent tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# values are multiples of 2^-4 up to 1 and scales powers of two: sums of 2^20 of them are exact in fp32, whatever the
# order, so results are compared bit by bit
_TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _values(*shape, dtype, g):
    return (torch.randint(-16, 17, shape, device="cuda", generator=g) / 16).to(dtype)


def _ids(n, rows, how, g):
    if how == "one":
        return torch.full((n,), rows // 2, device="cuda")
    if how == "distinct":
        return torch.randperm(max(n, rows), device="cuda", generator=g)[:n] % rows
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    return ((rows + 1.0) ** u - 1).long().clamp_(0, rows - 1)      # a few tokens make up most


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("n,rows,H", [(1, 1, 1), (1, 50, 768), (7, 33, 5), (129, 1000, 264), (1000, 77, 1000), (33, 9, 4099)])
def test_lookup(n, rows, H, dtype):
    from terapipe_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(n + H)
    w, ids = _values(rows, H, dtype=dtype, g=g), _ids(n, rows, "text", g)
    assert torch.equal(F.embedding_fwd(ids, w), w[ids])
    ids = ids - rows // 3                     # a shard's: some ids lie below it
    ids[n // 2] = rows + 5                    # and above
    in_ = (ids >= 2) & (ids < rows + 2)
    want = torch.where(in_[:, None], w[(ids - 2).clamp(0, rows - 1)] * 4, 0)
    assert torch.equal(F.embedding_fwd(ids.int(), w, scale=4.0, first_row=2), want.to(dtype))


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("H,offset", [(64, 0), (63, 1), (64, 1), (72, 8)])
def test_lookup_of_strided_tensors(H, offset, dtype):
    """Transposed ids, rows of wider matrices, addresses on no 16-byte boundary."""
    from terapipe_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(H)
    w = _values(40, H + 24, dtype=dtype, g=g)[:, offset:offset + H]
    ids = torch.randint(0, 40, (5, 13, 2), device="cuda", generator=g)[:, :, 1].t()     # [13, 5], no stride of one
    out = torch.full((65, H + 16), 7.0, device="cuda", dtype=dtype)
    F.embedding_fwd(ids, w, out[:, offset:offset + H])
    assert torch.equal(out[:, offset:offset + H], w[ids.reshape(-1)])
    out[:, offset:offset + H] = 7.0
    assert (out == 7.0).all()
    assert F.embedding_fwd(ids, w).shape == (13, 5, H)


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("how", ["text", "one", "distinct"])
@pytest.mark.parametrize("n,rows,H", [(1, 1, 8), (2, 600, 40), (31, 5, 256), (33, 1000, 264), (256, 300, 1600), (257, 40, 520),
                                      (1025, 7000, 768), (5000, 511, 136), (5001, 70000, 64), (20011, 513, 128)])
def test_gradient(n, rows, H, how, dtype):
    from terapipe_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    ids, dy = _ids(n, rows, how, g), _values(n, H, dtype=dtype, g=g)
    want = torch.zeros(rows, H, device="cuda", dtype=torch.float64).index_add_(0, ids, dy.double())
    dw = torch.full((rows, H), float("nan"), device="cuda")
    F.embedding_bwd(ids, dy, dw, accumulate=False)
    assert torch.equal(dw.double(), want)
    F.embedding_bwd(ids.int(), dy, dw, scale=0.5)          # adds
    assert torch.equal(dw.double(), 1.5 * want)


@pytest.mark.parametrize("n,rows,H,offset", [(300, 50, 64, 0), (300, 50, 63, 1), (5000, 900, 72, 4), (4097, 900, 1001, 3),
                                             (40, 90, 264, 2)])
@pytest.mark.parametrize("dtype", _TYPES)
def test_gradient_of_a_shard(n, rows, H, offset, dtype):
    """Ids of other shards and the padding token add nothing, whatever their rows hold; strided tensors; rows of other
    columns stay."""
    from terapipe_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(n)
    ids = torch.randint(-3, 3 * rows, (4, n // 4 + 1), device="cuda", generator=g)
    ids[1, 3] = rows + 1
    flat = ids.t().reshape(-1)
    n = flat.numel()
    dy = _values(n, H + 8, dtype=dtype, g=g)[:, offset:offset + H]
    in_ = (flat >= rows) & (flat < 2 * rows) & (flat != rows + 1)
    dy[~in_] = float("nan")
    want = torch.zeros(rows, H, device="cuda", dtype=torch.float64).index_add_(0, flat[in_] - rows, dy[in_].double())
    for accumulate in (False, True):
        whole = torch.full((rows, H + 12), 3.0, device="cuda")
        dw = whole[:, offset:offset + H]
        F.embedding_bwd(ids.t(), dy, dw, first_row=rows, padding_id=rows + 1, accumulate=accumulate)
        assert torch.equal(dw.double(), want + 3.0 * accumulate)
        dw.fill_(3.0)
        assert (whole == 3.0).all()


def test_gradient_of_no_tokens():
    from terapipe_b200.ops import functional as F
    ids, dy = torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, 40, device="cuda", dtype=torch.bfloat16)
    dw = torch.ones(30, 40, device="cuda")
    F.embedding_bwd(ids, dy, dw)
    assert (dw == 1).all()
    F.embedding_bwd(ids, dy, dw, accumulate=False)
    assert (dw == 0).all()
    assert F.embedding_fwd(ids, dy).shape == (0, 40)
    # tokens, but none of this shard's
    ids = torch.arange(100, 164, device="cuda")
    F.embedding_bwd(ids, torch.ones(64, 40, device="cuda"), dw.fill_(2.0))
    assert (dw == 2).all()
    F.embedding_bwd(ids, torch.ones(64, 40, device="cuda"), dw, accumulate=False)
    assert (dw == 0).all()


@pytest.mark.parametrize("n", [100, 3000, 40000])
def test_gradient_does_not_depend_on_timing(n):
    """fp32 sums of values that round: the same bits every time, and as near to the sums in 64 bits as fp32 sums of that
    many terms are (half a unit of 2^-24 a term of a sum in any order)."""
    from terapipe_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(n)
    ids, dy = _ids(n, 2000, "text", g), torch.randn(n, 520, device="cuda", generator=g)
    first = F.embedding_bwd(ids, dy, torch.empty(2000, 520, device="cuda"), accumulate=False)
    for _ in range(5):
        assert torch.equal(first, F.embedding_bwd(ids, dy, torch.empty(2000, 520, device="cuda"), accumulate=False))
    want = torch.zeros(2000, 520, device="cuda", dtype=torch.float64).index_add_(0, ids, dy.double())
    size = torch.zeros(2000, 520, device="cuda", dtype=torch.float64).index_add_(0, ids, dy.double().abs())
    count = torch.bincount(ids, minlength=2000)[:, None]
    assert ((first.double() - want).abs() <= size * count * 2.0 ** -24).all()


def test_on_another_stream_and_in_a_graph():
    from terapipe_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(1)
    ids, w = _ids(600, 300, "text", g), _values(300, 128, dtype=torch.bfloat16, g=g)
    dy, dw = torch.empty(600, 128, device="cuda", dtype=torch.bfloat16), torch.empty(300, 128, device="cuda")
    ws = torch.empty(F.embedding_bwd_workspace_bytes(600, 300, 128), dtype=torch.uint8, device="cuda")

    def both():
        F.embedding_fwd(ids, w, dy, scale=2.0)
        F.embedding_bwd(ids, dy, dw, accumulate=False, workspace=ws)

    def want():
        d = (w[ids] * 2).double()
        return torch.zeros(300, 128, device="cuda", dtype=torch.float64).index_add_(0, ids, d)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    s.synchronize()
    assert torch.equal(dw.double(), want())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    ids.copy_(_ids(600, 300, "distinct", g))
    graph.replay()
    assert torch.equal(dw.double(), want())


def test_refusals():
    from terapipe_b200.ops import functional as F
    from terapipe_b200.ops.lib import KernelError
    ids, w = torch.zeros(6, dtype=torch.int64, device="cuda"), torch.zeros(9, 16, device="cuda")
    dy = torch.zeros(6, 16, device="cuda")
    for bad in (lambda: F.embedding_fwd(ids.float(), w), lambda: F.embedding_fwd(ids, w.double()),
                lambda: F.embedding_fwd(ids, w.t()), lambda: F.embedding_fwd(ids, w, torch.empty(5, 16, device="cuda")),
                lambda: F.embedding_fwd(ids, w, torch.empty(6, 16, device="cuda", dtype=torch.float16)),
                lambda: F.embedding_fwd(ids, w, torch.empty(1, 16, device="cuda").expand(6, 16)),
                lambda: F.embedding_fwd(ids.cpu(), w), lambda: F.embedding_fwd(ids, w.cpu()),
                lambda: F.embedding_bwd(ids, dy, w.half()), lambda: F.embedding_bwd(ids[:5], dy, w),
                lambda: F.embedding_bwd(ids, dy[:, :8], w), lambda: F.embedding_bwd(ids, dy.cpu(), w),
                lambda: F.embedding_bwd(ids, dy, w[:1].expand(9, 16)),
                lambda: F.embedding_bwd(ids, dy, w, workspace=torch.empty(16, device="cuda")),
                lambda: F.embedding_bwd(ids.view(1, 2, 3).transpose(0, 2), dy.view(3, 2, 1, 16).transpose(0, 1), w)):
        with pytest.raises(KernelError):
            bad()
