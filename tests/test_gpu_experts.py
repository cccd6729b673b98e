"""The operators around a GPU's experts against plain implementations in 64 bits.

Tolerances count roundings: half a step of a type (u = finfo.eps / 2) for each output that is rounded to it, 2^-24 for each
fp32 operation on the longest chain behind it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, device="cuda", generator=_gen(seed)).to(dtype)


def _close(got, want, bound, what=""):
    """|got - want| <= bound everywhere (a bound of the values' shape, or a number)."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan()), what
    off = (got - want).abs() - bound
    worst = off.nan_to_num(nan=-1.0).max().item() if off.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3g} over the bound"


# --------------------------------------------------------------------------------------
# rows with block scales
# --------------------------------------------------------------------------------------

def _e4m3(v):
    """Nearest e4m3 value of |v| <= 448, ties to even, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))) / 8
    return torch.round(v / step) * step


def _check_quantised(q, scale, y, rel):
    """q and scale against y [rows, cols] in 64 bits, which the kernel knows to within a factor of 1 +- rel."""
    rows, cols = y.shape
    blocks = -(-cols // 128)
    assert q.dtype == torch.float8_e4m3fn and q.shape == (rows, cols) and q.is_contiguous()
    assert scale.dtype == torch.float32 and scale.shape == (rows, blocks) and scale.is_contiguous()
    padded = torch.nn.functional.pad(y, (0, blocks * 128 - cols)).view(rows, blocks, 128)
    want = padded.abs().amax(2).clamp(min=1e-30) / 448
    _close(scale, want, (rel + 2 * U32) * want, "scale")
    v = (padded / want[:, :, None]).view(rows, -1)[:, :cols]
    # the kernel's quotient is v to within twice that and the roundings of reciprocal, product and scale
    slack = 2 * rel + 6 * U32
    low, high = _e4m3((v.abs() * (1 - slack))), _e4m3((v.abs() * (1 + slack)).clamp(max=448))
    got = q.double()
    assert bool(((got.abs() >= low) & (got.abs() <= high)).all())
    assert bool((got * v >= 0).all())


def _norm_rel(cols):
    # sum of squares: a lane's chain of cols / 32 terms at most (cols / 512 from 1024 columns on), ten steps to add up the
    # lanes; the root halves that; the sum of x and residual, the mean, the reciprocal root (two steps), two products
    return (max(cols / 512, min(cols, 2048) / 32) / 2 + 16) * U32


def _norm_case(rows, cols, dtype, residual, normed, weight_dtype=None, seed=1):
    x = _randn(rows, cols, dtype=dtype, seed=seed)
    w = (1 + 0.2 * _randn(cols, seed=seed + 1)).to(weight_dtype or dtype)
    r = (3 * _randn(rows, cols, seed=seed + 2)).to(dtype) if residual else None
    return x, w, r, normed


def _check_norm(x, w, r, got, eps=1e-6):
    rows, cols = x.shape
    h = x.double() + (r.double() if r is not None else 0)
    # y * (1 + rel): fp32 addition is off by U32 |h|
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * w.double()
    rel = _norm_rel(cols)
    _check_quantised(got.q, got.scale, y, rel)
    if r is None:
        assert got.total is None
    else:
        assert got.total.dtype == x.dtype
        _close(got.total, h, (_u(x.dtype) + U32) * h.abs() + 2.0 ** -25, "total")
    if got.normed is not None:
        assert got.normed.dtype == x.dtype
        _close(got.normed, y, (_u(x.dtype) + rel) * y.abs() + 2.0 ** -25, "normed")  # (2^-25: half of fp16's least step)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 8), (9, 127), (8, 128), (17, 129), (4, 513), (33, 1000), (2, 1024),
                                       (3, 1032), (1, 2880), (7, 4097), (130, 4096), (1, 7168), (3, 8200), (2, 16392), (2, 32768),
                                       (1, 32767)])
def test_rms_norm_fp8(rows, cols, dtype):
    from amd_distributed_2025_b200.ops.fp8_rows import rms_norm_fp8

    for residual, normed in ((False, False), (True, True)):
        x, w, r, normed = _norm_case(rows, cols, dtype, residual, normed)
        got = rms_norm_fp8(x, w, 1e-6, residual=r, normed=normed)
        assert (got.normed is not None) == normed
        _check_norm(x, w, r, got)


def test_rms_norm_fp8_weight_in_fp32_strides_and_alignment():
    from amd_distributed_2025_b200.ops.fp8_rows import rms_norm_fp8

    x, w, r, _ = _norm_case(6, 512, torch.bfloat16, True, True, torch.float32)
    _check_norm(x, w, r, rms_norm_fp8(x, w, residual=r, normed=True))
    wide, other = _randn(6, 2000, dtype=torch.float16, seed=3), _randn(6, 1001, dtype=torch.float16, seed=4)
    w16 = w.half()
    for lo in (0, 8, 1, 4):  # columns of a wider matrix: whole vectors, and not
        x, r = wide[:, lo:lo + 512], other[:, lo:lo + 512]
        _check_norm(x, w16, r, rms_norm_fp8(x, w16, residual=r))
    x = _randn(512, 6, dtype=torch.float16, seed=5).t()  # rows that are not contiguous
    _check_norm(x, w16, None, rms_norm_fp8(x, w16))
    x = _randn(1, 512, dtype=torch.float16, seed=6).expand(6, 512)  # the same row six times
    _check_norm(x, w16, None, rms_norm_fp8(x, w16, normed=True))
    shifted = torch.empty(513, dtype=torch.float16, device="cuda")[1:].copy_(w16)
    _check_norm(wide[:, :512], shifted, None, rms_norm_fp8(wide[:, :512], shifted))


@pytest.mark.parametrize("dtype", DTYPES)
def test_fp8_rows_at_every_alignment(dtype):
    """Rows and weights that begin 0, 8, 16, .. bytes and single elements behind a 32-byte border, with distances to match."""
    from amd_distributed_2025_b200.ops.fp8_rows import rms_norm_fp8, silu_mul_fp8

    step = 8 // torch.tensor([], dtype=dtype).element_size()
    for cols in (256, 264, 2048):
        wide, other = _randn(5, cols + 80, dtype=dtype, seed=1), _randn(5, 2 * cols + 96, dtype=dtype, seed=2)
        long = 1 + 0.1 * _randn(cols + 80, seed=3)
        for lo in (0, step, 2 * step, 3 * step, 4 * step, 1):
            x, r = wide[:, lo:lo + cols], other[:, lo:lo + cols]
            for w in (long.to(dtype)[lo:lo + cols], long[lo:lo + cols]):
                _check_norm(x, w, r, rms_norm_fp8(x, w, residual=r, normed=True))
            x = other[:, lo:lo + 2 * cols]
            _check_silu(x, silu_mul_fp8(x))


@pytest.mark.parametrize("cols", [1024, 1500, 4100])
def test_rms_norm_fp8_total_in_place(cols):
    from amd_distributed_2025_b200.ops.fp8_rows import rms_norm_fp8

    x, w, r, _ = _norm_case(40, cols, torch.bfloat16, True, False)
    want = rms_norm_fp8(x, w, residual=r)
    kept = r.clone()
    got = rms_norm_fp8(x, w, residual=kept, total_out=kept)
    assert got.total is kept or got.total.data_ptr() == kept.data_ptr()
    assert torch.equal(kept, want.total) and torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8))
    kept = x.clone()
    got = rms_norm_fp8(kept, w, residual=r, total_out=kept)
    assert torch.equal(kept, want.total) and torch.equal(got.scale, want.scale)
    room = torch.full((40, cols + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    rms_norm_fp8(x, w, residual=r, total_out=room[:, 8:8 + cols])
    assert torch.equal(room[:, 8:8 + cols], want.total)
    assert bool((room[:, :8] == 7).all()) and bool((room[:, 8 + cols:] == 7).all())
    both = torch.zeros(41, cols, dtype=torch.bfloat16, device="cuda")
    for bad in (lambda: rms_norm_fp8(both[:40], w, residual=r, total_out=both[1:]),
                lambda: rms_norm_fp8(r, w, residual=both[:40], total_out=both[1:]),
                lambda: rms_norm_fp8(both[:1].expand(40, cols), w, residual=r, total_out=both[:40])):
        with pytest.raises(RuntimeError, match="overlap"):
            bad()
    side = torch.zeros(40, 2 * cols + 8, dtype=torch.bfloat16, device="cuda")  # the sum beside its residual
    side[:, :cols] = r
    rms_norm_fp8(x, w, residual=side[:, :cols], total_out=side[:, cols + 8:])
    assert torch.equal(side[:, cols + 8:], want.total) and torch.equal(side[:, :cols], r)


def test_rms_norm_fp8_zeros_infinities_and_nan():
    from amd_distributed_2025_b200.ops.fp8_rows import rms_norm_fp8

    x = _randn(6, 300, dtype=torch.bfloat16, seed=8)
    w = torch.ones(300, dtype=torch.bfloat16, device="cuda")
    x[0] = 0
    x[1, 128:] = 0
    x[2, 5] = float("nan")
    x[3, 200] = float("inf")
    x[4, :] = 1e-30
    got = rms_norm_fp8(x, w)
    assert bool((got.q[0].float() == 0).all()) and bool((got.q[1, 128:].float() == 0).all())
    assert bool(got.scale[0].isfinite().all()) and bool((got.scale[0] > 0).all())
    assert bool(got.q[2].float().isnan().all()) and bool(got.scale[2].isnan().all())  # the whole row's norm is NaN
    # one infinity: its own block is NaN, and the others are zero (everything over infinity)
    assert bool(got.q[3, 128:256].float().isnan().all()) and bool((got.q[3, :128].float() == 0).all())
    assert bool(got.q[4].float().isfinite().all())
    _check_norm(x[5:], w, None, rms_norm_fp8(x[5:], w))
    assert torch.equal(got.q[5].view(torch.uint8), rms_norm_fp8(x[5:], w).q[0].view(torch.uint8))
    empty = rms_norm_fp8(x[:0], w, residual=x[:0], normed=True)
    assert empty.q.shape == (0, 300) and empty.scale.shape == (0, 3) and empty.total.shape == empty.normed.shape == (0, 300)


def _check_silu(x, got):
    cols = x.shape[1] // 2
    g, u = x[:, :cols].double(), x[:, cols:].double()
    y = g / (1 + torch.exp(-g)) * u
    # exp to two steps, and a step for each unit of the exponent that is rounded before it; sum, quotient (two steps), product
    rel = (x[:, :cols].abs().max().double().item() * 1.5 + 8) * U32 if x.numel() else 0.0
    _check_quantised(got[0], got[1], y, rel)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 8), (3, 127), (9, 128), (2, 130), (33, 360), (7, 1000), (130, 2048), (1, 2880),
                                       (3, 8192), (2, 8191)])
def test_silu_mul_fp8(rows, cols, dtype):
    from amd_distributed_2025_b200.ops.fp8_rows import silu_mul_fp8

    x = _randn(rows, 2 * cols, dtype=dtype, seed=rows + cols) * 2
    _check_silu(x, silu_mul_fp8(x))


def test_silu_mul_fp8_strides_and_special_values():
    from amd_distributed_2025_b200.ops.fp8_rows import silu_mul_fp8

    wide = _randn(9, 3000, dtype=torch.bfloat16, seed=4)
    for lo in (0, 8, 3):
        x = wide[:, lo:lo + 1024]
        _check_silu(x, silu_mul_fp8(x))
    x = _randn(1024, 5, dtype=torch.float16, seed=4).t()
    _check_silu(x, silu_mul_fp8(x))
    x = torch.zeros(4, 512, device="cuda")
    x[:, 256:] = 1.0
    x[0, 3] = float("nan")
    x[1, :256] = -200.0  # exp overflows: the gate is -0, not NaN
    x[2, 7] = float("inf")
    q, scale = silu_mul_fp8(x)
    assert bool(q[0, :128].float().isnan().all()) and bool((q[0, 128:].float() == 0).all())
    assert bool((q[1].float() == 0).all())
    assert bool(scale[2, 0].isinf()) and bool(q[2, 7].float().isnan()) and bool((q[2, 128:].float() == 0).all())
    assert bool((q[3].float() == 0).all())
    q, scale = silu_mul_fp8(x[:0])
    assert q.shape == (0, 256) and scale.shape == (0, 2)


# --------------------------------------------------------------------------------------
# tokens sorted by expert
# --------------------------------------------------------------------------------------

def _ids(tokens, k, experts, seed, kind="uniform", dtype=torch.int32):
    g = _gen(seed)
    if kind == "uniform":
        ids = torch.randint(0, experts, (tokens, k), device="cuda", generator=g)
    elif kind == "one":  # everything at one expert
        ids = torch.full((tokens, k), experts // 2, device="cuda")
    elif kind == "none":
        ids = torch.full((tokens, k), -1, device="cuda")
    else:  # skewed, one entry in five without an expert: -1, the first id that is too large, and far off
        ids = (torch.rand(tokens, k, device="cuda", generator=g) ** 3 * experts).long()
        bad = torch.tensor([-1, experts, -2 ** 31, 2 ** 31 - 1], device="cuda")
        pick = torch.randint(0, 4, (tokens, k), device="cuda", generator=g)
        ids = torch.where(torch.rand(tokens, k, device="cuda", generator=g) < 0.2, bad[pick], ids)
    return ids.to(dtype)


def _order_of(ids, experts):
    flat = ids.reshape(-1).long()
    flat = torch.where((flat >= 0) & (flat < experts), flat, experts)
    at = torch.argsort(flat, stable=True)
    row_of = torch.empty_like(at)
    row_of[at] = torch.arange(at.numel(), device=at.device)
    row_of[flat == experts] = -1
    ends = torch.bincount(flat, minlength=experts + 1)[:experts].cumsum(0)
    return torch.cat([ends.new_zeros(1), ends]).int(), row_of.reshape(ids.shape).int()


def _check_sort(x, ids, experts, got, scale=None):
    offsets, row_of = _order_of(ids, experts)
    assert torch.equal(got.order.offsets, offsets) and torch.equal(got.order.row_of, row_of)
    for source, rows in ((x, got.rows), (scale, got.scale)):
        if source is None:
            assert rows is None
            continue
        assert rows.dtype == source.dtype and rows.shape == (ids.numel(), source.shape[1])
        raw = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[source.element_size()]
        want = torch.zeros(rows.shape, dtype=raw, device="cuda")
        t = torch.arange(ids.shape[0], device="cuda")[:, None].expand_as(ids)
        has = row_of >= 0
        want[row_of[has].long()] = source.contiguous().view(raw)[t[has]]
        assert torch.equal(rows.view(raw), want)


@pytest.mark.parametrize("kind", ["uniform", "skewed", "one", "none"])
@pytest.mark.parametrize("tokens,k,experts,hidden,dtype", [
    (1, 1, 1, 8, torch.float16), (1, 8, 256, 7168, torch.bfloat16), (11, 2, 8, 6144, torch.float16), (32, 2, 16, 250, torch.float32),
    (101, 4, 128, 2880, torch.float16), (37, 32, 33, 71, torch.bfloat16), (300, 3, 8192, 64, torch.float32),
    (2047, 8, 128, 512, torch.bfloat16), (16384, 1, 5, 16, torch.float16), (2049, 8, 256, 136, torch.bfloat16),
    (5000, 7, 64, 33, torch.float16), (40000, 4, 300, 8, torch.float32), (9000, 2, 8192, 24, torch.float16)])
def test_sort_tokens(tokens, k, experts, hidden, dtype, kind):
    from amd_distributed_2025_b200.ops.moe_sort import sort_tokens

    x = _randn(tokens, hidden, dtype=dtype, seed=tokens)
    for wide in (torch.int32, torch.int64):
        ids = _ids(tokens, k, experts, 3, kind, wide)
        _check_sort(x, ids, experts, sort_tokens(x, ids, experts))


@pytest.mark.parametrize("tokens,k,experts,hidden", [(1, 8, 64, 7168), (101, 4, 128, 2880), (4096, 8, 64, 1111), (3, 2, 8, 130),
                                                         (70, 3, 8, 12800), (5000, 8, 64, 8512)])
def test_sort_tokens_e4m3_rows_with_scales(tokens, k, experts, hidden):
    from amd_distributed_2025_b200.ops.moe_sort import sort_tokens

    x = (50 * _randn(tokens, hidden, seed=2)).to(torch.float8_e4m3fn)
    scale = _randn(tokens, -(-hidden // 128), seed=3)
    ids = _ids(tokens, k, experts, 4, "skewed")
    _check_sort(x, ids, experts, sort_tokens(x, ids, experts, scale=scale), scale)
    _check_sort(x, ids, experts, sort_tokens(x, ids, experts))
    wide = _randn(scale.shape[1], tokens, seed=5).t()  # scales column by column
    _check_sort(x, ids, experts, sort_tokens(x, ids, experts, scale=wide), wide)


@pytest.mark.parametrize("kind", ["uniform", "skewed", "one", "none"])
@pytest.mark.parametrize("tokens,k,experts,hidden,stride", [(2000, 20, 8192, 4112, 4112), (1100, 32, 3, 4096, 5120), (33001, 1, 5, 4224, 4224),
                                                            (6000, 7, 64, 20000, 20016), (5000, 8, 65, 4100, 4100), (5000, 7, 200, 24592, 24592)])
def test_sort_tokens_long_rows(tokens, k, experts, hidden, stride, kind):
    """More entries than one launch takes, rows of a page and more: e4m3 with scales, then bf16 without."""
    from amd_distributed_2025_b200.ops.moe_sort import sort_tokens

    x = _randn(tokens, stride, seed=tokens).to(torch.float8_e4m3fn)[:, :hidden]
    scale = torch.rand(tokens, -(-hidden // 128), device="cuda", generator=_gen(2))
    for wide in (torch.int32, torch.int64):
        ids = _ids(tokens, k, experts, 3, kind, wide)
        _check_sort(x, ids, experts, sort_tokens(x, ids, experts, scale=scale), scale)
    if hidden % 2 == 0 and stride % 2 == 0:
        half = x.contiguous().view(torch.bfloat16)
        _check_sort(half, ids, experts, sort_tokens(half, ids, experts))


def test_sort_tokens_strides_alignment_and_wide_ids():
    from amd_distributed_2025_b200.ops.moe_sort import sort_tokens

    big = _randn(50, 700, dtype=torch.bfloat16, seed=1)
    ids = _ids(50, 4, 16, 2)
    for lo, n in ((0, 512), (8, 512), (1, 512), (2, 130), (3, 65)):
        x = big[:, lo:lo + n]
        _check_sort(x, ids, 16, sort_tokens(x, ids, 16))
    x = big[:1, :512].expand(50, 512)
    _check_sort(x, ids, 16, sort_tokens(x, ids, 16))
    x = _randn(512, 50, dtype=torch.bfloat16, seed=1).t()
    _check_sort(x, ids, 16, sort_tokens(x, ids, 16))
    columns = _ids(4, 50, 16, 2).t()  # ids that are not contiguous
    _check_sort(big, columns, 16, sort_tokens(big, columns, 16))
    far = ids.long() + (torch.arange(50, device="cuda")[:, None] % 2) * 2 ** 32  # in range once the upper half is lost
    _check_sort(big, far, 16, sort_tokens(big, far, 16))
    none = sort_tokens(big[:0], ids[:0], 16)
    assert none.rows.shape == (0, 700) and none.order.offsets.tolist() == [0] * 17 and none.order.row_of.shape == (0, 4)


def _unsort64(rows, row_of, weights):
    has = row_of >= 0
    got = rows.double()[row_of.clamp(min=0).long()] * has[:, :, None]
    got = torch.where(has[:, :, None], got, torch.zeros((), dtype=torch.float64, device="cuda"))
    w = weights.double()[:, :, None] if weights is not None else 1.0
    w = torch.where(has[:, :, None], w, torch.zeros((), dtype=torch.float64, device="cuda"))
    return got, w


def _check_unsort(rows, row_of, weights, out):
    got, w = _unsort64(rows, row_of, weights)
    want, size = (got * w).sum(1), (got * w).abs().sum(1)
    assert out.dtype == rows.dtype
    _close(out, want, _u(rows.dtype) * want.abs() + (row_of.shape[1] + 2) * U32 * size * 2 + 2.0 ** -25, "out")


def _check_backward(grad, rows, row_of, weights, got):
    d_rows, d_weights = got
    y, w = _unsort64(rows, row_of, weights)
    has = row_of >= 0
    g = grad.double()[:, None, :]
    want = torch.zeros(rows.shape, dtype=torch.float64, device="cuda")
    want[row_of[has].long()] = (g * w).expand(-1, row_of.shape[1], -1)[has]
    if d_rows is not None:
        assert d_rows.dtype == rows.dtype
        _close(d_rows, want, (_u(rows.dtype) + U32) * want.abs() + 2.0 ** -25, "rows")
    if weights is None:
        assert d_weights is None
    elif d_weights is not None:
        dot, size = (g * y).sum(2), (g * y).abs().sum(2)
        # a lane's chain of hidden / 32 terms at most, then the lanes and warps
        _close(d_weights, dot, (rows.shape[1] / 32 + 24) * U32 * size, "weights")


UNSORT = [(1, 1, 1, 8), (1, 8, 256, 7168), (11, 2, 8, 6144), (128, 8, 256, 512), (32, 2, 16, 250), (37, 32, 33, 71), (101, 5, 128, 2880),
          (2047, 4, 16, 136), (300, 3, 64, 1), (9, 6, 4, 8200)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,experts,hidden", UNSORT)
def test_unsort_tokens_and_gradients(tokens, k, experts, hidden, dtype):
    from amd_distributed_2025_b200.ops import moe_sort

    for kind in ("uniform", "skewed", "none"):
        offsets, row_of = _order_of(_ids(tokens, k, experts, 5, kind), experts)
        order = moe_sort.ExpertOrder(offsets, row_of)
        rows = _randn(tokens * k, hidden, dtype=dtype, seed=6)
        weights = torch.rand(tokens, k, device="cuda", generator=_gen(7))
        _check_unsort(rows, row_of, weights, moe_sort.unsort_tokens(rows, order, weights))
        _check_unsort(rows, row_of, None, moe_sort.unsort_tokens(rows, order))
        grad = _randn(tokens, hidden, dtype=dtype, seed=8)
        _check_backward(grad, rows, row_of, weights, moe_sort.unsort_tokens_backward(grad, rows, order, weights))
        _check_backward(grad, rows, row_of, None, moe_sort.unsort_tokens_backward(grad, rows, order))
        _check_unsort(rows, row_of, None, moe_sort.sort_tokens_backward(rows, order))


def test_unsort_tokens_ignores_what_has_no_row():
    """NaN and infinities in weights without a row and in rows behind the last expert's reach nothing; where they count they show."""
    from amd_distributed_2025_b200.ops import moe_sort

    ids = _ids(200, 4, 16, 9, "skewed")
    offsets, row_of = _order_of(ids, 16)
    order = moe_sort.ExpertOrder(offsets, row_of)
    end = int(offsets[-1])
    assert end < ids.numel()
    for hidden in (264, 33):
        rows = _randn(ids.numel(), hidden, dtype=torch.bfloat16, seed=1)
        weights = torch.rand(200, 4, device="cuda", generator=_gen(2))
        grad = _randn(200, hidden, dtype=torch.bfloat16, seed=3)
        want = moe_sort.unsort_tokens(rows, order, weights)
        want_rows, want_weights = moe_sort.unsort_tokens_backward(grad, rows, order, weights)
        rows[end:] = float("nan")
        weights[row_of < 0] = float("inf")
        assert torch.equal(moe_sort.unsort_tokens(rows, order, weights), want)
        d_rows, d_weights = moe_sort.unsort_tokens_backward(grad, rows, order, weights)
        assert torch.equal(d_rows, want_rows) and torch.equal(d_weights, want_weights)
        assert bool((d_rows[end:] == 0).all()) and bool((d_weights[row_of < 0] == 0).all())
        empty = (row_of < 0).all(1)
        assert bool((want[empty] == 0).all())
        rows[0] = float("nan")
        t = (row_of == 0).any(1)
        out = moe_sort.unsort_tokens(rows, order, weights)
        assert bool(out[t].isnan().all()) and not bool(out[~t].isnan().any())
    # places that are no rows at all are skipped, whatever they say
    wild = row_of.clone()
    wild[0, 0], wild[1, 1], wild[2, 2] = 2 ** 31 - 1, -2 ** 31, ids.numel()
    rows = _randn(ids.numel(), 64, dtype=torch.float32, seed=1)
    tame = torch.where((wild < 0) | (wild >= ids.numel()), -1, wild)
    assert torch.equal(moe_sort.unsort_tokens(rows, moe_sort.ExpertOrder(offsets, wild)),
                       moe_sort.unsort_tokens(rows, moe_sort.ExpertOrder(offsets, tame)))


def test_unsort_tokens_strides_alignment_and_empty():
    from amd_distributed_2025_b200.ops import moe_sort

    offsets, row_of = _order_of(_ids(30, 4, 8, 1), 8)
    order = moe_sort.ExpertOrder(offsets, row_of)
    big, grads = _randn(120, 800, dtype=torch.float16, seed=1), _randn(30, 900, dtype=torch.float16, seed=2)
    weights = torch.rand(4, 30, device="cuda", generator=_gen(2)).t()  # not contiguous
    for lo, n in ((0, 512), (8, 512), (3, 512), (0, 77)):
        rows, grad = big[:, lo:lo + n], grads[:, lo:lo + n]
        _check_unsort(rows, row_of, weights, moe_sort.unsort_tokens(rows, order, weights))
        _check_backward(grad, rows, row_of, weights, moe_sort.unsort_tokens_backward(grad, rows, order, weights))
    one = grads[:1, :512].expand(30, 512)
    _check_backward(one, big[:, :512], row_of, weights, moe_sort.unsort_tokens_backward(one, big[:, :512], order, weights))
    same = torch.ones((), device="cuda", dtype=torch.float16).expand(30, 512)
    _check_backward(same, big[:, :512], row_of, weights, moe_sort.unsort_tokens_backward(same, big[:, :512], order, weights))
    none = moe_sort.ExpertOrder(torch.zeros(9, dtype=torch.int32, device="cuda"), row_of[:0])
    assert moe_sort.unsort_tokens(big[:0], none, weights[:0]).shape == (0, 800)
    d_rows, d_weights = moe_sort.unsort_tokens_backward(grads[:0, :800], big[:0], none, weights[:0])
    assert d_rows.shape == (0, 800) and d_weights.shape == (0, 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sort_and_unsort_through_autograd(dtype):
    """Leaves through sort, an expert's scale, unsort: gradients of the formula, in 64 bits by autograd itself."""
    from amd_distributed_2025_b200.ops import moe_sort

    tokens, k, experts, hidden = 60, 3, 8, 72
    ids = _ids(tokens, k, experts, 3, "skewed", torch.int64)
    x = _randn(tokens, hidden, dtype=dtype, seed=1).requires_grad_()
    weights = torch.rand(tokens, k, device="cuda", generator=_gen(2)).to(dtype).requires_grad_()
    grad = _randn(tokens, hidden, dtype=dtype, seed=4)
    got = moe_sort.sort_tokens(x, ids, experts)
    assert not got.order.offsets.requires_grad and not got.order.row_of.requires_grad
    out = moe_sort.unsort_tokens(got.rows, got.order, weights)
    out.backward(grad)
    xd, wd = x.detach().double().requires_grad_(), weights.detach().double().requires_grad_()
    has = (ids >= 0) & (ids < experts)
    want = (xd[:, None, :] * (wd * has)[:, :, None]).sum(1)
    want.backward(grad.double())
    u = _u(dtype)
    size = (wd * has).abs().sum(1, keepdim=True)
    _close(out, want, ((u + 8 * U32) * size * xd.abs()).detach() + 2.0 ** -25)
    # k rows of w * grad, rounded each, added and rounded again
    _close(x.grad, xd.grad, ((2 * u + 8 * U32) * size * grad.double().abs()).detach() + 4 * 2.0 ** -25)
    dot = (xd.detach().abs() * grad.double().abs()).sum(1, keepdim=True)
    _close(weights.grad, wd.grad, u * wd.grad.abs() + (hidden / 32 + 24) * U32 * dot + 2.0 ** -25)
    # against differences, in fp32: the output is linear in x and in the weights
    if dtype == torch.float32:
        for leaf in (x, weights):
            step = _randn(*leaf.shape, seed=9)
            moved = {id(leaf): leaf.detach() + step}
            xs, ws = moved.get(id(x), x.detach()), moved.get(id(weights), weights.detach())
            rows = moe_sort.sort_tokens(xs, ids, experts)
            far = moe_sort.unsort_tokens(rows.rows, rows.order, ws)
            change = ((far.double() - out.detach().double()) * grad.double()).sum().item()
            assert abs(change - (leaf.grad.double() * step.double()).sum().item()) < 1e-4 * grad.numel() ** 0.5


def test_sort_autograd_broadcast_gradients_and_unused_outputs():
    from amd_distributed_2025_b200.ops import moe_sort

    ids = _ids(20, 2, 4, 3)
    x = _randn(20, 48, seed=1).requires_grad_()
    got = moe_sort.sort_tokens(x, ids, 4)
    got.rows.sum().backward()  # an expanded gradient
    assert torch.equal(x.grad, torch.full_like(x, 2.0))
    base = _randn(1, 48, seed=1).requires_grad_()
    moe_sort.sort_tokens(base.expand(20, 48), ids, 4).rows.sum().backward()  # a broadcast input: its rows' gradients add up
    assert torch.equal(base.grad, torch.full_like(base, 40.0))
    weights = torch.ones(20, 2, device="cuda", requires_grad=True)
    order = got.order
    rows = _randn(40, 48, seed=2)
    moe_sort.unsort_tokens(rows, order, weights).sum().backward()  # only the weights want one
    _close(weights.grad, rows.double()[order.row_of.long()].sum(2), 48 * U32 * rows.abs().max().item() * 48)
    with torch.no_grad():
        assert not moe_sort.sort_tokens(x, ids, 4).rows.requires_grad


def test_sort_and_unsort_captured_and_replayed():
    """A training step in a graph: new inputs, the same buffers; twice in one graph, each with results of its own."""
    from amd_distributed_2025_b200.ops import moe_sort

    for tokens, hidden in ((64, 128), (5000, 128), (9000, 128), (9000, 1100)):  # one launch, two, and three
        x = _randn(tokens, hidden, seed=1).requires_grad_()
        weights = torch.rand(tokens, 4, device="cuda").requires_grad_()
        ids = _ids(tokens, 4, 16, 2, "skewed")
        grad = _randn(tokens, hidden, seed=3)

        def step():
            got = moe_sort.sort_tokens(x, ids, 16)
            out = moe_sort.unsort_tokens(got.rows * 2, got.order, weights)
            return (out.detach(), *torch.autograd.grad(out, (x, weights), grad))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            first, second = step(), step()
        for seed in (5, 6):
            with torch.no_grad():
                x.copy_(_randn(tokens, hidden, seed=seed))
                ids.copy_(_ids(tokens, 4, 16, seed, "skewed"))
            graph.replay()
            want = step()
            for a, b, c in zip(want, first, second):
                assert torch.equal(a, b) and torch.equal(a, c)


def test_capture_beside_an_eager_graph_of_the_same_leaf_is_refused():
    from amd_distributed_2025_b200.ops import moe_sort

    ids = _ids(16, 2, 4, 2)
    x = _randn(16, 64, seed=1).requires_grad_()
    alive = (x * 2).sum()  # its graph holds x's accumulation node, of the eager stream
    refused = []
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for leaf in (x, x * 1):
            try:
                moe_sort.sort_tokens(leaf, ids, 4)
            except RuntimeError as e:
                refused.append(str(e))
    assert len(refused) == 2 and all("eager graph" in r for r in refused)
    del alive, leaf  # (x * 1 holds the node too)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(moe_sort.sort_tokens(x, ids, 4).rows.sum(), x)
    graph.replay()
    assert torch.equal(got[0], torch.full_like(x, 2.0))


def test_expert_operators_on_streams_of_their_own():
    """Two streams at once, again and again: nothing is shared between calls."""
    from amd_distributed_2025_b200.ops import fp8_rows, moe_sort

    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    cases = []
    for s, (tokens, seed) in enumerate(((6000, 1), (700, 2))):
        x = _randn(tokens, 512, dtype=torch.bfloat16, seed=seed)
        ids = _ids(tokens, 4, 32, seed)
        cases.append((x, ids, moe_sort.sort_tokens(x, ids, 32), fp8_rows.rms_norm_fp8(x, x[0], residual=x)))
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for stream, (x, ids, _, _) in zip(streams, cases):
            with torch.cuda.stream(stream):
                got.append((moe_sort.sort_tokens(x, ids, 32), fp8_rows.rms_norm_fp8(x, x[0], residual=x)))
    torch.cuda.synchronize()
    for i, (rows, normed) in enumerate(got):
        want_rows, want_normed = cases[i % 2][2:]
        assert torch.equal(rows.rows, want_rows.rows) and torch.equal(rows.order.row_of, want_rows.order.row_of)
        assert torch.equal(normed.q.view(torch.uint8), want_normed.q.view(torch.uint8)) and torch.equal(normed.total, want_normed.total)


def test_long_and_short_rows_sorted_on_two_streams_at_once():
    """More entries than one launch takes: the launches of one call lie between those of the other."""
    from amd_distributed_2025_b200.ops.moe_sort import sort_tokens

    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    cases = [(_randn(9000, hidden, dtype=torch.bfloat16, seed=hidden), _ids(9000, 4, experts, hidden, "skewed"), experts)
             for hidden, experts in ((2056, 300), (256, 64))]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for stream, case in zip(streams, cases):
            with torch.cuda.stream(stream):
                got.append(sort_tokens(*case))
    torch.cuda.synchronize()
    for i, rows in enumerate(got):
        _check_sort(*cases[i % 2], rows)


# --------------------------------------------------------------------------------------
# the experts' products
# --------------------------------------------------------------------------------------

def _grouped_inputs(counts, n, k, seed=1):
    rows, experts, kb = sum(counts), len(counts), -(-k // 128)
    g = _gen(seed)
    a = (60 * torch.randn(max(rows, 1), k, device="cuda", generator=g)).to(torch.float8_e4m3fn)[:rows]
    b = (60 * torch.randn(experts, n, k, device="cuda", generator=g)).to(torch.float8_e4m3fn)
    a_scale = 0.01 + 0.02 * torch.rand(rows, kb, device="cuda", generator=g)
    b_scale = 0.01 + 0.02 * torch.rand(experts, -(-n // 128), kb, device="cuda", generator=g)
    offsets = torch.tensor([0] + counts).cumsum(0).int().cuda()
    return a, b, a_scale, b_scale, offsets


def _grouped64(a, b, a_scale, b_scale, offsets):
    """The product in 64 bits, and the sum of its terms' sizes."""
    k, n = a.shape[1], b.shape[1]
    ad = a.double() * a_scale.double().repeat_interleave(128, 1)[:, :k]
    want = torch.zeros(a.shape[0], n, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    ends = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        bd = b[e].double() * b_scale[e].double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        want[lo:hi] = ad[lo:hi] @ bd.T
        size[lo:hi] = ad[lo:hi].abs() @ bd.abs().T
    return want, size


def _check_grouped(inputs, out):
    want, size = _grouped64(*inputs)
    assert out.dtype == torch.bfloat16 and out.shape == want.shape
    # Products of a block of 128 are added up in the tensor cores in fp32 or a little less (23 bits at least are kept
    # of the largest term: 2^-22 of the sum of sizes for 128 of them is more than it takes), then two fp32 roundings a block.
    kb = inputs[2].shape[1]
    _close(out, want, _u(torch.bfloat16) * want.abs() + (128 * 2.0 ** -22 + (2 * kb + 2) * U32) * size)


GROUPED = [
    ([1], 128, 128), ([1], 1, 16), ([0, 1], 256, 256), ([3, 0, 0, 5, 1], 130, 272), ([32] * 8, 384, 512), ([33, 31, 64, 65, 0, 1], 257, 1024),
    ([4] * 256, 256, 640), ([0] * 100 + [7] + [0] * 155, 512, 2880), ([256], 512, 512), ([257, 255, 300, 129, 1], 264, 400),
    ([1000, 0, 500, 3], 1000, 896), ([70] * 9, 200, 1152), ([97, 200, 10, 0, 96], 640, 384), ([1] * 1024, 64, 128),
    ([5000, 20, 1], 300, 256), ([511, 513], 2048, 1536),
    ([100] * 7, 320, 1152), ([65, 128, 1, 129, 96, 33, 97, 127], 400, 400), ([0, 0, 350, 0, 1], 513, 272), ([70], 64, 144),
    ([127, 70] * 40, 256, 896), ([900] + [1] * 8, 264, 640),
    ([2400, 100, 4700], 600, 128), ([700] + [0] * 14 + [9], 600, 384), ([4353], 513, 144),
]


@pytest.mark.parametrize("counts,n,k", GROUPED, ids=[f"{len(c)}x{sum(c)}-{n}-{k}" for c, n, k in GROUPED])
def test_fp8_grouped_gemm(counts, n, k):
    from amd_distributed_2025_b200.ops import fp8_gemm as f

    inputs = _grouped_inputs(counts, n, k)
    out = f.fp8_grouped_gemm(*inputs)
    f.check()
    _check_grouped(inputs, out)
    assert torch.equal(out, f.fp8_grouped_gemm(*inputs))
    given = torch.full_like(out, 5.0)
    assert f.fp8_grouped_gemm(*inputs, c=given) is given and torch.equal(given, out)


def test_fp8_grouped_gemm_keeps_its_sums_in_registers():
    from amd_distributed_2025_b200.ops import _ext

    ext = _ext.load()
    assert [ext.fp8_grouped_local_bytes(tile) for tile in (64, 256)] == [0, 0]
    assert ext.fp8_grouped_tile(64 * 8 + 7, 8) == 64 and ext.fp8_grouped_tile(65 * 8, 8) == 256


def test_fp8_grouped_gemm_matches_fp8_gemm():
    """One expert is fp8_gemm (the same sums in the same order, but the two scales are multiplied first in both)."""
    from amd_distributed_2025_b200.ops.fp8_gemm import fp8_gemm, fp8_grouped_gemm

    a, b, a_scale, b_scale, offsets = inputs = _grouped_inputs([300], 384, 1024)
    got, one = fp8_grouped_gemm(*inputs), fp8_gemm(a, b[0], a_scale, b_scale[0])
    _check_grouped(inputs, got)
    _check_grouped(inputs, one)


def test_fp8_grouped_gemm_rows_of_no_expert():
    from amd_distributed_2025_b200.ops import fp8_gemm as f
    from amd_distributed_2025_b200.ops.fp8_gemm import fp8_grouped_gemm
    from amd_distributed_2025_b200.utils.status import StatusError

    for n in (264, 129):
        a, b, a_scale, b_scale, offsets = _grouped_inputs([40, 0, 30, 50], n, 256)
        want = fp8_grouped_gemm(a, b, a_scale, b_scale, offsets)
        fewer = offsets.clamp(max=70)  # the last expert's rows belong to nobody: whatever lies there is not looked at
        a.view(torch.uint8)[70:] = 0x7F  # NaN
        a_scale[70:] = float("nan")
        out = fp8_grouped_gemm(a, b, a_scale, b_scale, fewer)
        assert torch.equal(out[:70], want[:70]) and bool((out[70:] == 0).all())
        given = torch.full_like(out, 7.0)
        fp8_grouped_gemm(a, b, a_scale, b_scale, fewer, c=given)
        assert torch.equal(given[:70], want[:70]) and bool((given[70:] == 7).all())
        none = torch.zeros_like(offsets)
        assert bool((fp8_grouped_gemm(a, b, a_scale, b_scale, none) == 0).all())
        # offsets that are no order at all: more rows than there are is refused, fewer stay inside the matrices
        wild = torch.tensor([-5, 2 ** 31 - 1, -2 ** 31, 90, 400], dtype=torch.int32, device="cuda")
        f.fp8_grouped_gemm(a, b, a_scale, b_scale, wild)
        with pytest.raises(StatusError, match="bad_index"):
            f.check()
        f.fp8_grouped_gemm(a, b, a_scale, b_scale, torch.tensor([-5, 40, 10, 5, 60], dtype=torch.int32, device="cuda"))
        f.check()
        assert torch.equal(fp8_grouped_gemm(a, b, a_scale, b_scale, fewer)[:70], want[:70])
    empty = _grouped_inputs([0, 0], 64, 128)
    assert fp8_grouped_gemm(*empty).shape == (0, 64)


def test_fp8_grouped_gemm_strides_alignment_and_nan():
    from amd_distributed_2025_b200.ops.fp8_gemm import fp8_grouped_gemm

    a, b, a_scale, b_scale, offsets = _grouped_inputs([100, 3, 60], 200, 512)
    want = fp8_grouped_gemm(a, b, a_scale, b_scale, offsets)
    _check_grouped((a, b, a_scale, b_scale, offsets), want)
    columns = a_scale.t().contiguous().t()
    turned = b_scale.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(fp8_grouped_gemm(a, b, columns, turned, offsets), want)
    wide = torch.zeros(163, 528, dtype=torch.uint8, device="cuda")
    wide[:, 16:] = a.view(torch.uint8)
    assert torch.equal(fp8_grouped_gemm(wide.view(torch.float8_e4m3fn)[:, 16:], b, a_scale, b_scale, offsets), want)
    shifted = torch.zeros(a.numel() + 1, dtype=torch.uint8, device="cuda")
    shifted[1:] = a.view(torch.uint8).flatten()
    assert torch.equal(fp8_grouped_gemm(shifted[1:].view(torch.float8_e4m3fn).view(163, 512), b, a_scale, b_scale, offsets), want)
    room = torch.zeros(163 * 200 + 1, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(fp8_grouped_gemm(a, b, a_scale, b_scale, offsets, c=room[1:].view(163, 200)), want)
    flat = a_scale.clone()
    flat = torch.cat([flat.new_zeros(1), flat.flatten()])[1:].view(163, 4)  # four scales of a row that are no aligned piece
    assert torch.equal(fp8_grouped_gemm(a, b, flat, b_scale, offsets), want)
    a.view(torch.uint8)[101, 5] = 0x7F  # NaN stays in its row ...
    a_scale[7, 2] = float("inf")
    b.view(torch.uint8)[2, 9, 4] = 0x7F  # ... and in its column of its expert
    out = fp8_grouped_gemm(a, b, a_scale, b_scale, offsets)
    touched = torch.zeros_like(out, dtype=torch.bool)
    touched[101], touched[7], touched[103:, 9] = True, True, True
    assert bool(out[101].isnan().all()) and bool(out[103:, 9].isnan().all()) and not bool(out[7].isfinite().any())
    assert torch.equal(out[~touched], want[~touched])
    with pytest.raises(RuntimeError, match="overlap|memory location"):
        both = torch.zeros(163 * 512, dtype=torch.uint8, device="cuda")
        fp8_grouped_gemm(both.view(torch.float8_e4m3fn).view(163, 512), b, a_scale, b_scale, offsets,
                         c=both[:163 * 400].view(torch.bfloat16).view(163, 200))


def test_fp8_grouped_gemm_expired_wait_leaves_a_record():
    from amd_distributed_2025_b200.ops import _ext, fp8_gemm as f
    from amd_distributed_2025_b200.utils.status import StatusError

    inputs = _grouped_inputs([5, 6], 128, 256)
    want = f.fp8_grouped_gemm(*inputs)
    _ext.load().fp8_wait_selftest(0, 1_000_000)  # a barrier nobody arrives on, 1 ms
    torch.cuda.synchronize()
    with pytest.raises(StatusError):
        f.fp8_grouped_gemm(*inputs)
    assert torch.equal(f.fp8_grouped_gemm(*inputs), want)


def test_experts_of_a_layer_together():
    """norm -> sort -> gate and up -> activation -> down -> unsort, as a layer calls them, eager and in a graph, against
    fp32 with the same quantised rows."""
    from amd_distributed_2025_b200.ops import fp8_rows, moe_sort
    from amd_distributed_2025_b200.ops.fp8_gemm import check, fp8_grouped_gemm

    tokens, k, experts, hidden, inner = 150, 4, 16, 512, 384
    g = _gen(3)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).bfloat16()
    residual = torch.randn(tokens, hidden, device="cuda", generator=g).bfloat16()
    weight = torch.ones(hidden, device="cuda", dtype=torch.bfloat16)
    _, up, _, up_scale, _ = _grouped_inputs([1] * experts, 2 * inner, hidden, 5)
    _, down, _, down_scale, _ = _grouped_inputs([1] * experts, hidden, inner, 6)
    up_scale, down_scale = up_scale * 0.02, down_scale * 0.02
    ids = _ids(tokens, k, experts, 4, "skewed")
    routing = torch.rand(tokens, k, device="cuda", generator=g)

    def layer():
        normed = fp8_rows.rms_norm_fp8(x, weight, residual=residual)
        rows = moe_sort.sort_tokens(normed.q, ids, experts, scale=normed.scale)
        inside = fp8_grouped_gemm(rows.rows, up, rows.scale, up_scale, rows.order.offsets)
        q, scale = fp8_rows.silu_mul_fp8(inside)
        y = fp8_grouped_gemm(q, down, scale, down_scale, rows.order.offsets)
        return normed, rows, inside, q, scale, y, moe_sort.unsort_tokens(y, rows.order, routing)

    normed, rows, inside, q, scale, y, out = layer()
    check()
    end = int(rows.order.offsets[-1])
    assert 0 < end < tokens * k
    # each step on the one before it
    _check_norm(x, weight, residual, normed)
    _check_sort(normed.q, ids, experts, rows_of := moe_sort.SortedTokens(rows.rows, rows.scale, rows.order), normed.scale)
    _check_grouped((rows_of.rows, up, rows.scale, up_scale, rows.order.offsets), inside)
    _check_silu(inside, (q, scale))
    _check_grouped((q, down, scale, down_scale, rows.order.offsets), y)
    _check_unsort(y, rows.order.row_of, routing, out)
    assert bool((out[(rows.order.row_of < 0).all(1)] == 0).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer()[-1]
    for seed in (7, 8):
        x.copy_(_randn(tokens, hidden, dtype=torch.bfloat16, seed=seed))
        ids.copy_(_ids(tokens, k, experts, seed, "skewed"))
        graph.replay()
        assert torch.equal(captured, layer()[-1])
    check()


# --------------------------------------------------------------------------------------
# more than 2^31 elements, and calls at the same time
# --------------------------------------------------------------------------------------

def test_rows_beyond_32_bit_offsets():
    """4.6 GB of rows: their first and last ones, and those about 2^31 elements and 2^32 bytes."""
    from amd_distributed_2025_b200.ops import fp8_rows, moe_sort

    tokens, k, experts, hidden = 35000, 8, 64, 8192
    entries = tokens * k
    assert entries * hidden > 2 ** 31
    x = _randn(tokens, hidden, dtype=torch.bfloat16, seed=1)
    ids = _ids(tokens, k, experts, 2)
    got = moe_sort.sort_tokens(x, ids, experts)
    offsets, row_of = _order_of(ids, experts)
    assert torch.equal(got.order.offsets, offsets) and torch.equal(got.order.row_of, row_of)
    for j in range(k):
        assert torch.equal(got.rows[row_of[:, j].long()], x)
    some = torch.cat([torch.arange(0, 40), torch.arange(tokens - 40, tokens)]).cuda()
    edge = 2 ** 31 // hidden
    last = torch.cat([torch.arange(0, 40), torch.arange(edge - 20, edge + 20), torch.arange(entries - 40, entries)]).cuda()
    weights = torch.rand(tokens, k, device="cuda", generator=_gen(3))
    _check_unsort(got.rows, row_of[some], weights[some], moe_sort.unsort_tokens(got.rows, got.order, weights)[some])
    grad_rows, grad_weights = moe_sort.unsort_tokens_backward(x, got.rows, got.order, weights)
    at = torch.empty(entries, dtype=torch.long, device="cuda")  # the entry of a row
    at[row_of.reshape(-1).long()] = torch.arange(entries, device="cuda")
    want = x[at[last] // k].double() * weights.reshape(-1)[at[last]].double()[:, None]
    _close(grad_rows[last], want, (_u(torch.bfloat16) + U32) * want.abs())
    dot = (x[some].double()[:, None] * got.rows[row_of[some].long()].double()).sum(2)
    size = (x[some].double()[:, None] * got.rows[row_of[some].long()].double()).abs().sum(2)
    _close(grad_weights[some], dot, (hidden + 2) * U32 * size)
    del grad_rows
    w = torch.ones(hidden, dtype=torch.bfloat16, device="cuda")
    normed = fp8_rows.rms_norm_fp8(got.rows, w, residual=got.rows)
    _check_norm(got.rows[last], w, got.rows[last], fp8_rows.NormedRows(normed.q[last], normed.scale[last], normed.total[last], None))
    del normed
    wide = got.rows.view(entries // 2, 2 * hidden)
    last = last[last < entries // 2]
    last = torch.cat([last, torch.arange(entries // 2 - 40, entries // 2, device="cuda")])
    q, scale = fp8_rows.silu_mul_fp8(wide)
    _check_silu(wide[last], (q[last], scale[last]))


def test_fp8_grouped_gemm_beyond_32_bit_offsets():
    from amd_distributed_2025_b200.ops.fp8_gemm import check, fp8_grouped_gemm

    rows, n, k = 140000, 16384, 16
    assert rows * n > 2 ** 31
    a, b, a_scale, b_scale, offsets = _grouped_inputs([100, 130900, 9000], n, k)
    out = fp8_grouped_gemm(a, b, a_scale, b_scale, offsets)
    check()
    assert int(offsets[-1]) == rows
    edge = 2 ** 31 // n
    for lo, hi, e in ((0, 100, 0), (edge - 40, edge, 2), (edge, edge + 40, 2), (rows - 40, rows, 2), (130900, 131000, 1)):
        own = torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda")
        assert int(offsets[e]) <= lo and hi <= int(offsets[e + 1])
        _check_grouped((a[lo:hi], b[e:e + 1], a_scale[lo:hi], b_scale[e:e + 1], own), out[lo:hi])


def test_expert_products_on_two_streams_at_once():
    """Both kernels (few rows an expert, many), which hold all of an SM's tensor memory, beside one another and fp8_gemm."""
    from amd_distributed_2025_b200.ops.fp8_gemm import check, fp8_gemm, fp8_grouped_gemm

    few, many = _grouped_inputs([5] * 40, 1024, 2048), _grouped_inputs([700, 30, 1500], 1024, 1024, 2)
    one = (many[0], many[1][0], many[2], many[3][0])
    want = fp8_grouped_gemm(*few), fp8_grouped_gemm(*many), fp8_gemm(*one)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(20):
        for stream, call in zip(streams, (lambda: fp8_grouped_gemm(*few), lambda: fp8_grouped_gemm(*many), lambda: fp8_gemm(*one))):
            with torch.cuda.stream(stream):
                got.append(call())
    torch.cuda.synchronize()
    check()
    for i, c in enumerate(got):
        assert torch.equal(c, want[i % 3])


# --------------------------------------------------------------------------------------
# block scales to the last bit
# --------------------------------------------------------------------------------------

def _check_quotients(q, scale, y):
    """y is the kernel's own fp32 matrix: scales are to a step of it, a product with 1/448 (rounded, both), and values are its
    quotients by them, rounded as a division is and then to e4m3."""
    rows, cols = y.shape
    blocks = -(-cols // 128)
    padded = torch.nn.functional.pad(y, (0, blocks * 128 - cols)).view(rows, blocks, 128)
    want = padded.double().abs().amax(2).clamp(min=1e-30) / 448
    _close(scale, want, (2 * U32 + U32 ** 2) * want, "scale")
    values = (padded / scale[:, :, None]).view(rows, -1)[:, :cols].to(torch.float8_e4m3fn)
    assert torch.equal(q.view(torch.uint8), values.contiguous().view(torch.uint8))


@pytest.mark.parametrize("cols", [2048, 264, 1001])
def test_fp8_values_are_quotients_by_their_scale(cols):
    """Values between two e4m3 numbers too: whole numbers times one factor have many of those."""
    from amd_distributed_2025_b200.ops.fp8_rows import rms_norm_fp8, silu_mul_fp8

    rows = 3000
    whole = torch.randint(-448, 449, (rows, cols), device="cuda", generator=_gen(1)).float()
    for x, w in ((whole, torch.exp2(torch.randint(-3, 4, (cols,), device="cuda", generator=_gen(2)).float())),
                 (_randn(rows, cols, seed=3), 1 + 0.2 * _randn(cols, seed=4))):
        got = rms_norm_fp8(x, w, normed=True)  # (fp32: the normed rows are what was quantised)
        _check_quotients(got.q, got.scale, got.normed)
        for dtype in DTYPES:  # 32 / (1 + exp(-32)) is 32, so the products are known
            values = x.to(dtype)
            _check_quotients(*silu_mul_fp8(torch.cat([torch.full_like(values, 32.0), values], 1)), values.float() * 32)


@pytest.mark.parametrize("cols", [2048, 264, 1001])
def test_fp8_blocks_at_both_ends_of_the_range(cols):
    """Largest values from 2^126, whose reciprocal is no normal number, up to the largest finite one, and small ones."""
    from amd_distributed_2025_b200.ops.fp8_rows import rms_norm_fp8, silu_mul_fp8

    rows = 64
    top = torch.finfo(torch.float32).max
    y = torch.rand(rows, cols, device="cuda", generator=_gen(1)) * 2 - 1
    sizes = torch.logspace(-37.9, 38.5, rows, device="cuda", dtype=torch.float64)
    sizes[-8:] = torch.tensor([2.0 ** 126, 1.1 * 2.0 ** 126, 2.0 ** 127, 1.9 * 2.0 ** 127, top, 1e38, 2e38, 3e38], dtype=torch.float64)
    y = (y.double() * sizes[:, None]).float()
    y[:, ::200] = sizes.float().clamp(max=top)[:, None]
    values = y / 32
    products = values * 32
    assert bool(products.isfinite().all())
    _check_quotients(*silu_mul_fp8(torch.cat([torch.full_like(values, 32.0), values], 1)), products)
    got = rms_norm_fp8(_randn(rows, cols, seed=5), torch.full((cols,), 5e37, device="cuda"), normed=True)
    assert bool(got.normed.isfinite().all()) and bool((got.normed.abs().amax(1) > 2.0 ** 126).any())
    _check_quotients(got.q, got.scale, got.normed)


def test_fp8_zeros_keep_their_signs():
    from amd_distributed_2025_b200.ops.fp8_rows import silu_mul_fp8

    values = torch.zeros(2, 512, device="cuda")
    values[:, ::2] = -0.0
    values[1, 5], values[1, 200] = 1.0, float("inf")
    _check_quotients(*silu_mul_fp8(torch.cat([torch.full_like(values, 32.0), values], 1)[:1]), values[:1] * 32)
    q, scale = silu_mul_fp8(torch.cat([torch.full_like(values, 32.0), values], 1))
    raw = q[1].view(torch.uint8)
    assert raw[4] == 0x80 and raw[7] == 0 and raw[5] == 0x7E and bool(scale[1, 1].isinf())
    assert raw[202] == 0x80 and raw[201] == 0 and bool(q[1, 200].float().isnan())  # over infinity: zeros


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_silu_mul_fp8_gates_whose_exponential_is_near_the_end_of_the_range(dtype):
    """exp(-gate) from 2^115 to 2^128, times values so large that the product counts."""
    from amd_distributed_2025_b200.ops.fp8_rows import silu_mul_fp8

    for cols in (256, 250):
        gates = torch.linspace(-88.5, -80, 17, device="cuda").to(dtype)[:, None].expand(17, cols)
        values = ((torch.rand(17, cols, device="cuda", generator=_gen(1)) * 2 - 1) * 3e38).to(dtype)
        x = torch.cat([gates, values], 1)
        g, u = gates.double(), values.double()
        y = g / (1 + torch.exp(-g)) * u
        assert bool((y.abs().amax(1) > 1e-2).all())
        # as _check_silu; below 2^-126 the exponential has at least 21 bits
        _check_quantised(*silu_mul_fp8(x), y, (88.5 * 1.5 + 8) * U32 + 2.0 ** -21)


@pytest.mark.parametrize("cols", [1032, 1040, 1152, 1408, 2816, 2880, 2888, 8976])
def test_silu_mul_fp8_rows_whose_last_round_leaves_part_of_a_warp_idle(cols):
    """Rows of a few units more than whole rounds of a team: its warps stay together, and nothing behind a row is written."""
    from amd_distributed_2025_b200.ops.fp8_rows import silu_mul_fp8

    for rows in (1, 3, 333):
        for dtype in DTYPES:
            values = _randn(rows, cols, dtype=dtype, seed=rows)
            q, scale = silu_mul_fp8(torch.cat([torch.full_like(values, 32.0), values], 1))
            _check_quotients(q, scale, values.float() * 32)


@pytest.mark.parametrize("counts,lo,hi", [([40, 0, 30, 50], 1, 3), ([40, 0, 30, 50], 2, 4), ([700, 300, 5], 1, 2), ([3, 2, 90], 2, 3), ([0, 9], 0, 1)])
def test_fp8_grouped_gemm_some_of_the_experts(counts, lo, hi):
    """A slice of the experts and of their offsets: rows in front of the first and behind the last are zero, whatever the
    memory held, and those of a given c stay."""
    from amd_distributed_2025_b200.ops.fp8_gemm import check, fp8_grouped_gemm

    for n in (264, 129):
        a, b, a_scale, b_scale, offsets = _grouped_inputs(counts, n, 256)
        want = fp8_grouped_gemm(a, b, a_scale, b_scale, offsets)
        first, last = offsets[lo].item(), offsets[hi].item()
        own = torch.zeros(a.shape[0], dtype=torch.bool, device="cuda")
        own[first:last] = True
        stale = [torch.full_like(want, float("nan")) for _ in range(4)]
        torch.cuda.synchronize()
        del stale  # (its memory is handed out again)
        out = fp8_grouped_gemm(a, b[lo:hi], a_scale, b_scale[lo:hi], offsets[lo:hi + 1])
        check()
        assert torch.equal(out[own], want[own]) and bool((out[~own] == 0).all())
        given = torch.full_like(want, 7.0)
        fp8_grouped_gemm(a, b[lo:hi], a_scale, b_scale[lo:hi], offsets[lo:hi + 1], c=given)
        assert torch.equal(given[own], want[own]) and bool((given[~own] == 7).all())


def test_fp8_grouped_gemm_offsets_that_fall_give_no_row_to_two_experts():
    from amd_distributed_2025_b200.ops.fp8_gemm import check, fp8_grouped_gemm
    from amd_distributed_2025_b200.utils.status import StatusError

    for falling in ([10, 60, 20, 90, 80, 120], [0, 50, 40, 30, 20, 70], [0, 100, 90, 5, 60, 70], [-5, 40, 10, 5, 60, 300], [300, 0, 0, 0, 0, 0],
                    [100, 90, 2 ** 31 - 1, -2 ** 31, 5, 290], [0] * 700 + [40, 20, 60, 1]):
        experts = len(falling) - 1
        for rows in (300, 5000) if experts < 100 else (300,):  # both kernels
            a, b, a_scale, b_scale, _ = _grouped_inputs([rows] + [0] * (experts - 1), 136, 144)
            offsets = torch.tensor(falling, dtype=torch.int32, device="cuda")
            cut = [min(max(v, 0), rows) for v in falling]
            if sum(max(there - here, 0) for here, there in zip(cut, cut[1:])) > rows:  # more rows than there are
                fp8_grouped_gemm(a, b, a_scale, b_scale, offsets)
                with pytest.raises(StatusError, match="bad_index"):
                    check()
                continue
            rising = offsets.clamp(0, rows).cummax(0).values.int()
            got = fp8_grouped_gemm(a, b, a_scale, b_scale, offsets)
            check()
            assert torch.equal(got, fp8_grouped_gemm(a, b, a_scale, b_scale, rising))
            _check_grouped((a, b, a_scale, b_scale, rising), got)
            given = torch.full_like(got, 7.0)
            fp8_grouped_gemm(a, b, a_scale, b_scale, offsets, c=given)
            assert torch.equal(given[rising[0]:rising[-1]], got[rising[0]:rising[-1]])
            assert bool((given[:rising[0]] == 7).all()) and bool((given[rising[-1]:] == 7).all())


def test_outputs_in_place_count_as_changes():
    """What autograd has saved and total_out or c then overwrites is noticed by the backward pass, as with torch's own operations."""
    from amd_distributed_2025_b200.ops.fp8_gemm import fp8_grouped_gemm
    from amd_distributed_2025_b200.ops.fp8_rows import rms_norm_fp8

    x, w = _randn(4, 256, seed=1), _randn(256, seed=2)
    inputs = _grouped_inputs([3, 5], 256, 128)

    def saved(values):
        scale = torch.ones(256, device="cuda", requires_grad=True)
        return (scale * values).sum()

    residual = _randn(4, 256, seed=3)
    c = torch.ones(8, 256, dtype=torch.bfloat16, device="cuda")
    for target, write in ((residual, lambda: rms_norm_fp8(x, w, residual=residual, total_out=residual)),
                          (x, lambda: rms_norm_fp8(x, w, residual=residual, total_out=x)),
                          (residual, lambda: rms_norm_fp8(x[:2], w, residual=x[2:], total_out=residual[1:3])),  # a view
                          (c, lambda: fp8_grouped_gemm(*inputs, c=c))):
        loss = saved(target)
        with torch.no_grad():
            write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        saved(target).backward()
    loss = saved(x)  # nothing of it is written
    fresh = rms_norm_fp8(x, w, residual=residual)
    loss.backward()
    with torch.inference_mode():  # (tensors that count no changes)
        out = torch.empty(4, 256, device="cuda")
        assert torch.equal(rms_norm_fp8(x, w, residual=residual, total_out=out).total, fresh.total)
        inside = torch.empty_like(c)
        assert torch.equal(fp8_grouped_gemm(*inputs, c=inside), c)


def test_unsort_keeps_rows_for_the_weights_gradient_only():
    """The rows' own gradient does not need them: they are free to go when the weights want none."""
    from amd_distributed_2025_b200.ops import moe_sort

    ids = _ids(40, 3, 8, 1, "skewed")
    order = moe_sort.ExpertOrder(*_order_of(ids, 8))
    grad = _randn(40, 72, seed=3)
    routing = torch.rand(40, 3, device="cuda", generator=_gen(2))
    for dtype in DTYPES:
        leaf = _randn(120, 72, dtype=dtype, seed=1).requires_grad_()
        for weights in (None, routing, routing.half(), routing.clone().requires_grad_()):
            kept = []

            def pack(t):
                kept.append(t.data_ptr())
                return t

            rows = leaf * 1
            with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
                out = moe_sort.unsort_tokens(rows, order, weights)
            wanted = weights is not None and weights.requires_grad
            assert (rows.data_ptr() in kept) == wanted
            out.backward(grad.to(dtype))
            w32 = None if weights is None else weights.detach().float()
            want = moe_sort.unsort_tokens_backward(grad.to(dtype), rows.detach(), order, w32)
            assert torch.equal(leaf.grad, want[0])
            if wanted:
                assert torch.equal(weights.grad, want[1])
            leaf.grad = None
        only = routing.clone().requires_grad_()  # and the weights alone
        moe_sort.unsort_tokens(leaf.detach(), order, only).backward(grad.to(dtype))
        assert torch.equal(only.grad, moe_sort.unsort_tokens_backward(grad.to(dtype), leaf.detach(), order, routing)[1])
    none = moe_sort.ExpertOrder(torch.zeros(9, dtype=torch.int32, device="cuda"), order.row_of[:0])
    empty = torch.empty(0, 72, device="cuda", requires_grad=True)
    moe_sort.unsort_tokens(empty, none).sum().backward()
    assert empty.grad.shape == (0, 72)


def test_unsort_without_gradient_is_captured_whatever_the_weights_type():
    """No backward pass follows, so an eager graph of the rows and weights is no reason to refuse."""
    from amd_distributed_2025_b200.ops import moe_sort

    ids = _ids(16, 2, 4, 2)
    order = moe_sort.ExpertOrder(*_order_of(ids, 4))
    rows = _randn(32, 64, seed=1).requires_grad_()
    for dtype in (torch.float32, torch.bfloat16, torch.float16, torch.float64):
        weights = torch.rand(16, 2, device="cuda", generator=_gen(3)).to(dtype).requires_grad_()
        alive = (weights * 2).sum() + rows.sum()
        with torch.no_grad():
            want = moe_sort.unsort_tokens(rows, order, weights)
            assert not want.requires_grad
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = moe_sort.unsort_tokens(rows, order, weights)
        graph.replay()
        assert torch.equal(got, want) and torch.equal(want, moe_sort.unsort_tokens(rows.detach(), order, weights.detach().float()))
        refused = []
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):  # with a gradient it is still refused
            try:
                moe_sort.unsort_tokens(rows, order, weights)
            except RuntimeError as e:
                refused.append(str(e))
        assert len(refused) == 1 and "eager graph" in refused[0]
        del alive


def test_rms_norm_fp8_rows_whose_squares_leave_the_range():
    """fp32 holds no sum of them: such a row is normed to zeros, and its neighbours are not touched."""
    from amd_distributed_2025_b200.ops.fp8_rows import rms_norm_fp8

    x = _randn(4, 264, seed=1)
    w = torch.ones(264, device="cuda")
    x[1] *= 1e25
    got = rms_norm_fp8(x, w, normed=True)
    assert bool((got.normed[1] == 0).all()) and bool((got.q[1].float() == 0).all()) and bool((got.scale[1] == got.scale[1].amin()).all())
    for row in (0, 2, 3):
        _check_norm(x[row:row + 1], w, None, rms_norm_fp8(x[row:row + 1], w))
        assert torch.equal(got.q[row].view(torch.uint8), rms_norm_fp8(x[row:row + 1], w).q[0].view(torch.uint8))
