"""Calls of the operators around a GPU's experts that are refused before anything is launched (no GPU needed)."""
import pytest
import torch

from amd_distributed_2025_b200.ops import fp8_rows, moe_sort
from amd_distributed_2025_b200.ops.moe_sort import ExpertOrder

F = torch.zeros


def _refused(match, call):
    with pytest.raises((RuntimeError, ValueError, TypeError), match=match):
        call()


def test_rms_norm_fp8_refusals():
    x, w = F(4, 256), F(256)
    f = fp8_rows.rms_norm_fp8
    _refused("matrix", lambda: f(F(256), w))
    _refused("matrix", lambda: f(F(2, 2, 256), w))
    _refused("unsupported dtype", lambda: f(x.double(), w.double()))
    _refused("unsupported dtype", lambda: f(x.to(torch.float8_e4m3fn), w))
    _refused("weight must be a vector", lambda: f(x, F(255)))
    _refused("weight must be a vector", lambda: f(x, F(1, 256)))
    _refused("weight must have x's type", lambda: f(x, w.half()))
    _refused("columns", lambda: f(F(2, 0), F(0)))
    _refused("columns", lambda: f(F(1, 32769), F(32769)))
    _refused("eps", lambda: f(x, w, -1.0))
    _refused("eps", lambda: f(x, w, float("nan")))
    _refused("residual must", lambda: f(x, w, residual=F(4, 255)))
    _refused("residual must", lambda: f(x, w, residual=x.half()))
    _refused("there is no residual", lambda: f(x, w, total_out=x))
    _refused("total_out must have x's", lambda: f(x, w, residual=x, total_out=F(3, 256)))
    _refused("total_out must have contiguous rows", lambda: f(x, w, residual=x, total_out=F(256, 4).t()))
    _refused("total_out must have contiguous rows", lambda: f(x, w, residual=x, total_out=F(1, 256).expand(4, 256)))
    _refused("no_grad", lambda: f(x.clone().requires_grad_(), w))
    _refused("no_grad", lambda: f(x, w.clone().requires_grad_()))
    _refused("no_grad", lambda: f(x, w, residual=x.clone().requires_grad_()))
    _refused("CUDA", lambda: f(x, w))
    with torch.no_grad():  # a parameter is fine there
        _refused("CUDA", lambda: f(x, w.clone().requires_grad_()))
    _refused("expected a torch.Tensor", lambda: f(None, w))


def test_silu_mul_fp8_refusals():
    f = fp8_rows.silu_mul_fp8
    _refused("matrix", lambda: f(F(256)))
    _refused("even number", lambda: f(F(4, 255)))
    _refused("even number", lambda: f(F(4, 0)))
    _refused("unsupported dtype", lambda: f(F(4, 256, dtype=torch.int32)))
    _refused("no_grad", lambda: f(F(4, 256).requires_grad_()))
    _refused("CUDA", lambda: f(F(4, 256)))


def test_sort_tokens_refusals():
    x, ids = F(4, 64), F(4, 2, dtype=torch.int32)
    f = moe_sort.sort_tokens
    _refused("x must be a matrix", lambda: f(F(4), ids, 8))
    _refused("x must be a matrix", lambda: f(F(4, 0), ids, 8))
    _refused("unsupported dtype", lambda: f(x.double(), ids, 8))
    _refused("indices must be", lambda: f(x, ids[:3], 8))
    _refused("indices must be", lambda: f(x, ids[0], 8))
    _refused("int32 or int64", lambda: f(x, ids.to(torch.int16), 8))
    _refused("int32 or int64", lambda: f(x, ids.float(), 8))
    _refused("1 to 32 experts", lambda: f(x, F(4, 0, dtype=torch.int32), 8))
    _refused("1 to 32 experts", lambda: f(x, F(4, 33, dtype=torch.int32), 64))
    _refused("num_experts", lambda: f(x, ids, 0))
    _refused("num_experts", lambda: f(x, ids, 8193))
    _refused("2\\^30", lambda: f(F(1, 1).expand(1 << 29, 1), F(1, 1, dtype=torch.int32).expand(1 << 29, 4), 8))
    _refused("scale must be", lambda: f(x, ids, 8, scale=F(3, 1)))
    _refused("scale must be", lambda: f(x, ids, 8, scale=F(4, 1).half()))
    _refused("no gradient", lambda: f(x.clone().requires_grad_(), ids, 8, scale=F(4, 1)))
    _refused("no gradient", lambda: f(x.to(torch.float8_e4m3fn).requires_grad_(), ids, 8))
    _refused("CUDA", lambda: f(x, ids, 8))


def test_unsort_tokens_refusals():
    order = ExpertOrder(F(9, dtype=torch.int32), F(4, 2, dtype=torch.int32))
    rows, w = F(8, 64), F(4, 2)
    f = moe_sort.unsort_tokens
    _refused("rows must be a matrix", lambda: f(F(8), order, w))
    _refused("unsupported dtype", lambda: f(rows.to(torch.float8_e4m3fn), order, w))
    _refused("a row for each", lambda: f(F(7, 64), order, w))
    _refused("a row for each", lambda: f(F(9, 64), order, w))
    _refused("weights must be", lambda: f(rows, order, F(4, 3)))
    _refused("weights must be", lambda: f(rows, order, F(8)))
    _refused("floating type", lambda: f(rows, order, F(4, 2, dtype=torch.int32)))
    _refused("row_of must be", lambda: f(rows, ExpertOrder(order.offsets, order.row_of.long()), w))
    _refused("row_of must be", lambda: f(rows, ExpertOrder(order.offsets, order.row_of[0]), w))
    _refused("CUDA", lambda: f(rows, order, w))
    b = moe_sort.unsort_tokens_backward
    grad = F(4, 64)
    _refused("gradient must be", lambda: b(F(4, 63), rows, order, w))
    _refused("gradient must be", lambda: b(grad.half(), rows, order, w))
    _refused("a row for each", lambda: b(grad, F(9, 64), order, w))
    _refused("offsets must be", lambda: b(grad, rows, ExpertOrder(order.offsets.long(), order.row_of), w))
    _refused("offsets must be", lambda: b(grad, rows, ExpertOrder(order.offsets[:1], order.row_of), w))
    _refused("weights must be", lambda: b(grad, rows, order, F(4, 3)))
    _refused("CUDA", lambda: b(grad, rows, order, w))
    _refused("a row for each", lambda: moe_sort.sort_tokens_backward(F(7, 64), order))


def test_fp8_grouped_gemm_refusals():
    from amd_distributed_2025_b200.ops.fp8_gemm import fp8_grouped_gemm as f

    fp8 = torch.float8_e4m3fn
    a, b = F(4, 256).to(fp8), F(3, 130, 256).to(fp8)
    sa, sb, off = F(4, 2), F(3, 2, 2), F(4, dtype=torch.int32)
    _refused("equal K", lambda: f(a, b[0], sa, sb, off))
    _refused("equal K", lambda: f(a[:, :128], b, sa, sb, off))
    _refused("float8_e4m3fn", lambda: f(F(4, 256), b, sa, sb, off))
    _refused("float8_e4m3fn", lambda: f(a, b.to(torch.float8_e5m2), sa, sb, off))
    _refused("1 to 1024 experts", lambda: f(a, b[:0], sa, sb[:0], off[:1]))
    _refused("1 to 1024 experts", lambda: f(a, F(1025, 1, 256).to(fp8), sa, F(1025, 1, 2), F(1026, dtype=torch.int32)))
    _refused("multiple of 16", lambda: f(a[:, :24], b[:, :, :24], sa[:, :1], sb[:, :, :1], off))
    _refused("multiple of 16", lambda: f(a[:, :0], b[:, :, :0], sa[:, :0], sb[:, :, :0], off))
    _refused("N must not", lambda: f(a, b[:, :0], sa, sb[:, :0], off))
    _refused("a_scale must", lambda: f(a, b, F(4, 3), sb, off))
    _refused("a_scale must", lambda: f(a, b, sa.double(), sb, off))
    _refused("b_scale must", lambda: f(a, b, sa, F(3, 1, 2), off))
    _refused("b_scale must", lambda: f(a, b, sa, F(2, 2), off))
    _refused("offsets must", lambda: f(a, b, sa, sb, off[:3]))
    _refused("offsets must", lambda: f(a, b, sa, sb, off.long()))
    _refused("c must", lambda: f(a, b, sa, sb, off, F(4, 130)))
    _refused("c must", lambda: f(a, b, sa, sb, off, F(130, 4, dtype=torch.bfloat16).t()))
    _refused("timeout_ms", lambda: f(a, b, sa, sb, off, timeout_ms=0))
    _refused("CUDA", lambda: f(a, b, sa, sb, off))


def test_grouped_product_leaves_no_room_for_a_cta_that_waits_for_tensor_memory():
    """Its CTAs hold all of an SM's tensor memory: none of the GEMM kernels' may fit beside one by shared memory."""
    from amd_distributed_2025_b200.ops import _ext

    ext = _ext.load()
    others = [ext.gemm_tile_share(rows, bn, splits, pair)[0] for rows in range(8, 129, 8) for bn in range(32, 257, 32)
              for pair in (False, True) for splits in range(1, (8 if pair else 16) + 1)]
    others += [ext.gemm_pair_share(bn, 1)[0] for bn in range(32, 257, 32)] + [ext.gemm_pair_share(256, 2)[0]]
    others += [ext.gemm_rs_share(bn, pair)[0] for bn, pair in ((64, False), (128, False), (256, False), (128, True), (192, True), (256, True))]
    others += [ext.fp8_gemm_share(bn, splits)[0] for bn in (64, 128) for splits in range(1, 9)]
    own = [ext.fp8_grouped_share(tile, experts) for tile in (64, 256) for experts in (1, 7, 256, 1000, 1024)]
    sm, reserved = 228 * 1024, 1024
    for smem, columns in own:
        assert columns == 512 and smem <= 232448
        assert smem + reserved + min(others + [s for s, _ in own]) + reserved > sm


def test_scales_that_want_a_gradient_are_refused():
    """Neither operator has one: e4m3 rows cannot have a gradient themselves, but their scales can want one."""
    from amd_distributed_2025_b200.ops.fp8_gemm import fp8_grouped_gemm

    fp8 = torch.float8_e4m3fn
    ids = F(4, 2, dtype=torch.int32)
    for x in (F(4, 256).to(fp8), F(4, 256)):
        _refused("scale requires a gradient", lambda: moe_sort.sort_tokens(x, ids, 8, scale=F(4, 2).requires_grad_()))
        _refused("scale requires a gradient", lambda: moe_sort.sort_tokens(x, ids, 8, scale=F(4, 2).requires_grad_() * 2))
        with torch.no_grad():
            _refused("CUDA", lambda: moe_sort.sort_tokens(x, ids, 8, scale=F(4, 2).requires_grad_()))
    off = F(4, dtype=torch.int32)
    names = ("a", "b", "a_scale", "b_scale", "c")
    for i, name in enumerate(names):
        given = [F(4, 256).to(fp8), F(3, 130, 256).to(fp8), F(4, 2), F(3, 2, 2), F(4, 130, dtype=torch.bfloat16)]
        given[i].requires_grad_()
        a, b, a_scale, b_scale, c = given
        _refused(f"^{name} requires a gradient", lambda: fp8_grouped_gemm(a, b, a_scale, b_scale, off, c))
        with torch.no_grad():
            _refused("CUDA", lambda: fp8_grouped_gemm(a, b, a_scale, b_scale, off, c))


def test_forward_mode_tangents_are_refused():
    """No operator here has a forward derivative, and a result without a tangent would count as one of zero."""
    import torch.autograd.forward_ad as fwd

    from amd_distributed_2025_b200.ops.fp8_gemm import fp8_grouped_gemm

    fp8 = torch.float8_e4m3fn
    ids, off = F(4, 2, dtype=torch.int32), F(4, dtype=torch.int32)
    order = ExpertOrder(F(9, dtype=torch.int32), ids)
    x, w, rows, routing = F(4, 256), F(256), F(8, 64), F(4, 2)
    a, b, sa, sb = F(4, 256).to(fp8), F(3, 130, 256).to(fp8), F(4, 2), F(3, 2, 2)
    with fwd.dual_level():
        def d(t, grad=False):
            return fwd.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))

        calls = [
            ("x", lambda: fp8_rows.rms_norm_fp8(d(x), w)),
            ("weight", lambda: fp8_rows.rms_norm_fp8(x, d(w))),
            ("residual", lambda: fp8_rows.rms_norm_fp8(x, w, residual=d(x))),
            ("total_out", lambda: fp8_rows.rms_norm_fp8(x, w, residual=x, total_out=d(x))),
            ("x", lambda: fp8_rows.silu_mul_fp8(d(x))),
            ("x", lambda: moe_sort.sort_tokens(d(x), ids, 8)),
            ("x", lambda: moe_sort.sort_tokens(d(x, True), ids, 8)),
            ("scale", lambda: moe_sort.sort_tokens(x, ids, 8, scale=d(F(4, 2)))),
            ("rows", lambda: moe_sort.unsort_tokens(d(rows), order, routing)),
            ("weights", lambda: moe_sort.unsort_tokens(rows, order, d(routing))),
            ("weights", lambda: moe_sort.unsort_tokens(rows, order, d(routing.half()))),
            ("rows", lambda: moe_sort.unsort_tokens(d(rows, True), order, routing)),
            ("the gradient", lambda: moe_sort.unsort_tokens_backward(d(F(4, 64)), rows, order, routing)),
            ("rows", lambda: moe_sort.unsort_tokens_backward(F(4, 64), d(rows), order, routing)),
            ("weights", lambda: moe_sort.unsort_tokens_backward(F(4, 64), rows, order, d(routing))),
            ("rows", lambda: moe_sort.sort_tokens_backward(d(rows), order)),
            ("a_scale", lambda: fp8_grouped_gemm(a, b, d(sa), sb, off)),
            ("b_scale", lambda: fp8_grouped_gemm(a, b, sa, d(sb), off)),
            ("c", lambda: fp8_grouped_gemm(a, b, sa, sb, off, d(F(4, 130, dtype=torch.bfloat16)))),
        ]
        for name, call in calls:
            _refused(f"^{name} has a forward-mode tangent", call)
            with torch.no_grad():
                _refused(f"^{name} has a forward-mode tangent", call)
    _refused("CUDA", lambda: moe_sort.sort_tokens(x, ids, 8))


def test_outputs_that_share_memory_with_inputs():
    """Refused unless they are the very same rows, or columns of one wider matrix that do not meet."""
    from amd_distributed_2025_b200.ops.fp8_gemm import fp8_grouped_gemm

    w = F(8)
    f = fp8_rows.rms_norm_fp8

    def norm(x, residual, total, weight=w):
        return lambda: f(x, weight, residual=residual, total_out=total)

    flat = F(1000)
    # one row, whatever the distance to a next one says (0 divides nothing)
    for one, other in ((0, 0), (8, 0), (0, 8), (8, 100), (3, 5)):
        x, total = flat.as_strided((1, 8), (one, 1), 4), flat.as_strided((1, 8), (other, 1), 0)
        _refused("total_out and x overlap", norm(x, F(1, 8), total))
        _refused("total_out and residual overlap", norm(F(1, 8), x, total))
        same = flat.as_strided((1, 8), (one, 1), 0)
        _refused("CUDA", norm(same, F(1, 8), total))
        _refused("CUDA", norm(F(1, 8), same, total))
        _refused("CUDA", norm(flat.as_strided((1, 8), (one, 1), 8), F(1, 8), total))
    wide = flat.view(20, 50)
    total = wide[:, 10:18]
    for lo, fine in ((0, True), (2, True), (3, False), (10, True), (17, False), (18, True), (42, True)):
        _refused("CUDA" if fine else "overlap", norm(wide[:, lo:lo + 8], F(20, 8), total))
        _refused("CUDA" if fine else "overlap", norm(F(20, 8), wide[:, lo:lo + 8], total))
    _refused("overlap", norm(wide[:1, 10:18].expand(20, 8), F(20, 8), total))  # one row of it, read again and again
    _refused("CUDA", norm(wide[:1, 20:28].expand(20, 8), F(20, 8), total))
    _refused("overlap", norm(flat[4:164].view(20, 8), F(20, 8), total))
    # the weight in the sum's rows, and between them
    _refused("total_out and weight overlap", norm(F(20, 8), F(20, 8), total, wide[3, 10:18]))
    _refused("total_out and weight overlap", norm(F(20, 8), F(20, 8), total, wide[3, 4:12]))
    _refused("total_out and weight overlap", norm(F(20, 8), F(20, 8), total, wide[:8, 10]))
    _refused("CUDA", norm(F(20, 8), F(20, 8), total, wide[3, 20:28]))
    _refused("CUDA", norm(F(20, 8), F(20, 8), total, flat[:8]))
    _refused("CUDA", norm(F(0, 8), F(0, 8), wide[:0, :8]))
    # a product's result and inputs whose strides leave room in between
    fp8 = torch.float8_e4m3fn
    a, b, sb, off = F(4, 256).to(fp8), F(3, 130, 256).to(fp8), F(3, 2, 2), F(4, dtype=torch.int32)
    room = F(4000)
    c = room[:260].view(torch.bfloat16).view(4, 130)
    _refused("c and a_scale overlap", lambda: fp8_grouped_gemm(a, b, room.as_strided((4, 2), (100, 2), 10), sb, off, c))
    _refused("c and b_scale overlap", lambda: fp8_grouped_gemm(a, b, F(4, 2), room.as_strided((3, 2, 2), (1000, 100, 10), 9), off, c))
    _refused("c and a overlap", lambda: fp8_grouped_gemm(room.view(fp8).view(4, 4000)[:, :256], b, F(4, 2), sb, off, c))
    raw = F(25000)
    inside = raw[10:270].view(torch.bfloat16).view(4, 130)
    _refused("c and b overlap", lambda: fp8_grouped_gemm(a, raw.view(fp8)[:99840].view(3, 130, 256), F(4, 2), sb, off, inside))
    _refused("c and offsets overlap", lambda: fp8_grouped_gemm(a, b, F(4, 2), sb, room[255:259].view(torch.int32), c))
    _refused("CUDA", lambda: fp8_grouped_gemm(a, b, room.as_strided((4, 2), (100, 2), 260), sb, room[800:804].view(torch.int32), c))
