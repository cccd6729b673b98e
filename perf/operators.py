"""The operators around the experts of one GPU: their plain forms, the calls of the framework, and what is measured.

* ``sort``         ``ops.moe_sort.sort_tokens``: tokens sorted by expert (rows packed expert by expert);
* ``unsort``       ``ops.moe_sort.unsort_tokens``: the weighted sum of a token's rows, back in token order;
* ``sort_grad``    ``ops.moe_sort.sort_tokens_backward``;
* ``unsort_grad``  ``ops.moe_sort.unsort_tokens_backward``;
* ``norm``         ``ops.fp8_rows.rms_norm_fp8``: root-mean-square norm with the residual's addition, e4m3 out;
* ``silu_mul``     ``ops.fp8_rows.silu_mul_fp8``: gated activation between two products, e4m3 out;
* ``grouped``      ``ops.fp8_gemm.fp8_grouped_gemm``: the experts' products on sorted rows.

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` makes what a program
holds before the call, ``run`` is one call (in elementary torch operations, or where ``own`` is true through the
framework), ``work`` the bytes and operations the call cannot do without and ``exact`` the result in 64 bits.
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
TINY = 1e-30  # the smallest maximum that a block's scale is made from
EPS = 1e-6

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32, "e4m3": torch.float8_e4m3fn}
_SIZES = {"float16": 2, "bfloat16": 2, "float32": 4, "e4m3": 1}

# Bounds of drawn cases: bytes of the sorted rows, values of a quantised matrix, bytes of the experts' weights, 2 R N K.
_MAX_ROW_BYTES = 8192 * 8 * 7168
_MAX_VALUES = 16384 * 4096
_MAX_WEIGHT_BYTES = 256 * 2048 * 7168
_MAX_FLOPS = 2 * 24576 * 4096 * 4096


def _routed(name, op, tokens, topk, experts, hidden, dtype, routing="uniform", dropped=0.0):
    return {"name": name, "op": op, "tokens": tokens, "topk": topk, "experts": experts, "hidden": hidden, "dtype": dtype,
            "routing": routing, "dropped": dropped}


def listed():
    return [
        # A dozen tokens of the smallest decode step (configs/all2all.yml): launches and host time are all there is.
        _routed("sort_decode_fp16", "sort", 11, 2, 8, 6144, "float16"),
        # Prefill of an fp8 model with many experts, skewed routing: quantised rows move together with their scales.
        _routed("sort_prefill_e4m3", "sort", 8192, 8, 256, 7168, "e4m3", routing="zipf"),
        # Headline decode step (configs/headline.yml): the way back to the tokens.
        _routed("unsort_decode_bf16", "unsort", 128, 8, 256, 7168, "bfloat16"),
        # An odd batch of the benchmark list's rows where one entry in ten has no expert here (experts of other ranks).
        _routed("unsort_prefill_fp16", "unsort", 2047, 4, 128, 2880, "float16", dropped=0.1),
        # Training, the headline prefill's sizes (configs/headline.yml): gradients of rows and routing weights.
        _routed("unsort_grad_bf16", "unsort_grad", 4096, 6, 64, 4096, "bfloat16", routing="zipf"),
        # Training in full precision, an odd batch of narrow rows: the gradient of the tokens.
        _routed("sort_grad_fp32", "sort_grad", 3001, 2, 16, 1000, "float32", dropped=0.05),
        # Serving, a handful of tokens (one decode step of a small batch) of a wide model.
        {"name": "norm_decode_bf16", "op": "norm", "rows": 8, "cols": 7168, "dtype": "bfloat16", "residual": True, "normed": False},
        # Prefill; the router wants the normed rows in bf16 as well.
        {"name": "norm_prefill_bf16", "op": "norm", "rows": 16384, "cols": 4096, "dtype": "bfloat16", "residual": True,
         "normed": True},
        # Between the experts' products: one token of eight experts, and a prefill batch of ragged length.
        {"name": "silu_mul_decode_bf16", "op": "silu_mul", "rows": 8, "cols": 2048, "dtype": "bfloat16"},
        {"name": "silu_mul_prefill_bf16", "op": "silu_mul", "rows": 32761, "cols": 2048, "dtype": "bfloat16"},
        # Headline decode step: four tokens for each of 256 experts, whose weights have to stream once.
        {"name": "grouped_decode", "op": "grouped", "rows": 1024, "experts": 256, "n": 2048, "k": 7168, "routing": "uniform"},
        # Headline prefill: 4096 tokens of six experts each, skewed over 64.
        {"name": "grouped_prefill", "op": "grouped", "rows": 24576, "experts": 64, "n": 4096, "k": 4096, "routing": "zipf"},
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread evenly over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return min(hi, max(-(-lo // step) * step, int(v) // step * step))


def draw(rng):
    op = rng.choice(["sort", "unsort", "sort_grad", "unsort_grad", "norm", "silu_mul", "grouped", "grouped"])
    if op in ("sort", "unsort", "sort_grad", "unsort_grad"):
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"] + (["e4m3", "e4m3"] if op == "sort" else []))
        hidden = _log_int(rng, 128, 7168, rng.choice([8, 8, 1]))  # rows of whole 16-byte vectors, and others
        topk = rng.randint(1, 8)
        most = min(16384, _MAX_ROW_BYTES // (topk * hidden * _SIZES[dtype]))
        return {"op": op, "tokens": _log_int(rng, 1, most), "topk": topk, "experts": _log_int(rng, 8, 256), "hidden": hidden,
                "dtype": dtype, "routing": rng.choice(["uniform", "zipf"]), "dropped": rng.choice([0.0, 0.0, 0.1, 0.5])}
    if op in ("norm", "silu_mul"):
        cols = _log_int(rng, 128, 16384 if op == "norm" else 8192, rng.choice([128, 8, 1]))
        case = {"op": op, "rows": _log_int(rng, 1, min(65536, _MAX_VALUES // cols)), "cols": cols,
                "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}
        if op == "norm":
            case.update(residual=rng.random() < 0.7, normed=rng.random() < 0.4)
        return case
    experts = _log_int(rng, 1, 256)
    k = _log_int(rng, 256, 8192, 16)
    n = min(_log_int(rng, 128, 8192, rng.choice([128, 8, 1])), _MAX_WEIGHT_BYTES // (experts * k))
    return {"op": op, "rows": _log_int(rng, 1, min(65536, _MAX_FLOPS // (2 * n * k))), "experts": experts, "n": n, "k": k,
            "routing": rng.choice(["uniform", "zipf"])}


# --------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------

def _popularity(experts, routing):
    p = [1.0 / (e + 1) ** 1.2 if routing == "zipf" else 1.0 for e in range(experts)]
    return [v / sum(p) for v in p]


def _indices(case, gen):
    """Distinct experts of a token (Gumbel top-k); an entry in `dropped` has none: -1."""
    logp = torch.tensor(_popularity(case["experts"], case["routing"]), device="cuda").log()
    u = torch.rand(case["tokens"], case["experts"], device="cuda", generator=gen).clamp_(1e-12, 1 - 1e-7)
    ids = (logp - (-u.log()).log()).topk(case["topk"], dim=1).indices.to(torch.int32)
    if case["dropped"]:
        ids[torch.rand(ids.shape, device="cuda", generator=gen) < case["dropped"]] = -1
    return ids


def _order(ids, experts):
    """(offsets [E + 1], row_of [T, k]) of the entries sorted by expert, stable."""
    flat = ids.reshape(-1).long()
    flat = torch.where((flat >= 0) & (flat < experts), flat, experts)
    at = torch.argsort(flat, stable=True)
    row_of = torch.empty_like(at)
    row_of[at] = torch.arange(at.numel(), device=at.device)
    row_of[flat == experts] = -1
    ends = torch.bincount(flat, minlength=experts + 1)[:experts].cumsum(0)
    offsets = torch.cat([ends.new_zeros(1), ends])
    return offsets.to(torch.int32), row_of.reshape(ids.shape).to(torch.int32)


def _randn(shape, dtype, gen, scale=1.0):
    """Normal values, made in slices so that the full-precision copy stays small."""
    out = torch.empty(shape, dtype=_DTYPES[dtype], device="cuda")
    flat = out.view(-1)
    for lo in range(0, flat.numel(), 1 << 27):
        part = flat[lo:lo + (1 << 27)]
        part.copy_(torch.randn(part.numel(), device="cuda", generator=gen) * scale)
    return out


def prepare(case, seed):
    op = case["op"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if op in ("sort", "unsort", "sort_grad", "unsort_grad"):
        tokens, topk, hidden, dtype = case["tokens"], case["topk"], case["hidden"], case["dtype"]
        ids = _indices(case, gen)
        state = {"op": op, "experts": case["experts"], "indices": ids, "scale": None}
        if op == "sort":
            state["x"] = _randn((tokens, hidden), dtype, gen, 60.0 if dtype == "e4m3" else 1.0)
            if dtype == "e4m3":
                state["scale"] = torch.rand(tokens, -(-hidden // BLOCK), device="cuda", generator=gen) * 0.01 + 0.001
            return state
        state["offsets"], state["row_of"] = _order(ids, case["experts"])
        if op != "sort_grad":
            state["rows"] = _randn((tokens * topk, hidden), dtype, gen)
            state["weights"] = torch.softmax(torch.randn(tokens, topk, device="cuda", generator=gen), 1)
        if op == "sort_grad":
            state["grad"] = _randn((tokens * topk, hidden), dtype, gen)
        if op == "unsort_grad":
            state["grad"] = _randn((tokens, hidden), dtype, gen)
        return state
    if op == "norm":
        shape = (case["rows"], case["cols"])
        return {"op": op, "x": _randn(shape, case["dtype"], gen), "normed": case["normed"],
                "residual": _randn(shape, case["dtype"], gen, 4.0) if case["residual"] else None,
                "weight": (1 + 0.2 * torch.randn(case["cols"], device="cuda", generator=gen)).to(_DTYPES[case["dtype"]])}
    if op == "silu_mul":
        return {"op": op, "x": _randn((case["rows"], 2 * case["cols"]), case["dtype"], gen, 2.0)}
    experts, rows, n, k = case["experts"], case["rows"], case["n"], case["k"]
    p = torch.tensor(_popularity(experts, case["routing"]), device="cuda")
    counts = torch.bincount(torch.multinomial(p, rows, replacement=True, generator=gen), minlength=experts)
    ends = counts.cumsum(0)
    kb = -(-k // BLOCK)
    return {"op": op, "offsets": torch.cat([ends.new_zeros(1), ends]).to(torch.int32), "ends": [0] + ends.tolist(),
            "a": _randn((rows, k), "e4m3", gen, 60.0), "b": _randn((experts, n, k), "e4m3", gen, 60.0),
            "a_scale": torch.rand(rows, kb, device="cuda", generator=gen) * 0.02 + 0.01,
            "b_scale": torch.rand(experts, -(-n // BLOCK), kb, device="cuda", generator=gen) * 0.0004 + 0.0002}


# --------------------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------------------

def _run_own(s):
    op = s["op"]
    if op == "grouped":
        from amd_distributed_2025_b200.ops.fp8_gemm import fp8_grouped_gemm

        return fp8_grouped_gemm(s["a"], s["b"], s["a_scale"], s["b_scale"], s["offsets"])
    if op in ("norm", "silu_mul"):
        from amd_distributed_2025_b200.ops import fp8_rows

        if op == "silu_mul":
            q, scale = fp8_rows.silu_mul_fp8(s["x"])
            return {"q": q, "scale": scale}
        got = fp8_rows.rms_norm_fp8(s["x"], s["weight"], EPS, residual=s["residual"], normed=s["normed"])
        return {"q": got.q, "scale": got.scale, "total": got.total, "normed": got.normed}
    from amd_distributed_2025_b200.ops import moe_sort

    if op == "sort":
        got = moe_sort.sort_tokens(s["x"], s["indices"], s["experts"], scale=s["scale"])
        return {"rows": got.rows, "scale": got.scale, "offsets": got.order.offsets, "row_of": got.order.row_of}
    order = moe_sort.ExpertOrder(s["offsets"], s["row_of"])
    if op == "unsort":
        return moe_sort.unsort_tokens(s["rows"], order, s["weights"])
    if op == "sort_grad":
        return moe_sort.sort_tokens_backward(s["grad"], order)
    return list(moe_sort.unsort_tokens_backward(s["grad"], s["rows"], order, s["weights"]))


# --------------------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------------------

def _quantised(y):
    """e4m3 values and a scale for each row and 128 columns of a fp32 matrix."""
    rows, cols = y.shape
    blocks = -(-cols // BLOCK)
    if cols % BLOCK:
        y = torch.nn.functional.pad(y, (0, blocks * BLOCK - cols))
    y = y.view(rows, blocks, BLOCK)
    scale = y.abs().amax(2).clamp(min=TINY) / E4M3_MAX
    q = (y / scale[:, :, None]).to(torch.float8_e4m3fn).view(rows, blocks * BLOCK)
    return q[:, :cols].contiguous(), scale


def _scattered(values, row_of, rows):
    """values [T, k, ...] at their rows; zeros in rows that no entry has."""
    out = torch.zeros((rows + 1,) + values.shape[2:], dtype=values.dtype, device=values.device)
    out[torch.where(row_of < 0, rows, row_of).long()] = values
    return out[:rows]


def _gathered(rows, row_of):
    """rows [R, H] of each entry, [T, k, H] in fp32; zeros for an entry without one."""
    got = rows[row_of.clamp(min=0).long()].float()
    return got.masked_fill_((row_of < 0)[:, :, None], 0.0)


def _run_plain(s):
    op = s["op"]
    if op == "sort":
        x, ids = s["x"], s["indices"]
        offsets, row_of = _order(ids, s["experts"])
        rows = _scattered(x.view(torch.uint8)[:, None, :].expand(-1, ids.shape[1], -1), row_of, ids.numel()).view(x.dtype)
        scale = s["scale"]
        if scale is not None:
            scale = _scattered(scale[:, None, :].expand(-1, ids.shape[1], -1), row_of, ids.numel())
        return {"rows": rows, "scale": scale, "offsets": offsets, "row_of": row_of}
    if op == "unsort":
        return (_gathered(s["rows"], s["row_of"]) * s["weights"][:, :, None]).sum(1).to(s["rows"].dtype)
    if op == "sort_grad":
        return _gathered(s["grad"], s["row_of"]).sum(1).to(s["grad"].dtype)
    if op == "unsort_grad":
        grad = s["grad"].float()[:, None, :]
        rows = _scattered((grad * s["weights"][:, :, None]).to(s["rows"].dtype), s["row_of"], s["rows"].shape[0])
        return [rows, (_gathered(s["rows"], s["row_of"]) * grad).sum(2)]
    if op == "norm":
        x = s["x"]
        h = x.float() if s["residual"] is None else x.float() + s["residual"].float()
        y = h * (h.square().mean(1, keepdim=True) + EPS).rsqrt() * s["weight"].float()
        q, scale = _quantised(y)
        return {"q": q, "scale": scale, "total": None if s["residual"] is None else h.to(x.dtype),
                "normed": y.to(x.dtype) if s["normed"] else None}
    if op == "silu_mul":
        gate, up = s["x"].float().chunk(2, 1)
        q, scale = _quantised(gate * torch.sigmoid(gate) * up)
        return {"q": q, "scale": scale}
    a, b, k = s["a"], s["b"], s["a"].shape[1]
    full = a.float() * s["a_scale"].repeat_interleave(BLOCK, 1)[:, :k]
    out = torch.empty((a.shape[0], b.shape[1]), dtype=torch.bfloat16, device=a.device)
    for e, (lo, hi) in enumerate(zip(s["ends"], s["ends"][1:])):  # an expert's rows, times its own weight
        if lo < hi:
            scale = s["b_scale"][e].repeat_interleave(BLOCK, 0)[:b.shape[1]].repeat_interleave(BLOCK, 1)[:, :k]
            out[lo:hi] = full[lo:hi] @ (b[e].float() * scale).T
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("sort", "unsort", "sort_grad", "unsort_grad"):
        size = _SIZES[case["dtype"]]
        entries = case["tokens"] * case["topk"]
        row = case["hidden"] * size
        kept = int(entries * (1 - case["dropped"]))
        if op == "sort":
            if case["dtype"] == "e4m3":
                row += 4 * -(-case["hidden"] // BLOCK)
            # ids in and rows' places out; tokens in; rows out, those without an entry as zeros
            return {"bytes": 8 * entries + 4 * case["experts"] + (case["tokens"] + entries) * row, "flops": 0}
        if op == "unsort":
            return {"bytes": 8 * entries + (case["tokens"] + kept) * row, "flops": 2 * kept * case["hidden"]}
        if op == "sort_grad":
            return {"bytes": 4 * entries + (case["tokens"] + kept) * row, "flops": kept * case["hidden"]}
        return {"bytes": 12 * entries + (case["tokens"] + kept + entries) * row, "flops": 3 * kept * case["hidden"]}
    if op in ("norm", "silu_mul"):
        rows, cols, size = case["rows"], case["cols"], _SIZES[case["dtype"]]
        scales = 4 * rows * -(-cols // BLOCK)
        if op == "silu_mul":
            return {"bytes": rows * cols * (2 * size + 1) + scales, "flops": 8 * rows * cols}
        passes = 1 + 2 * case["residual"] + case["normed"]
        return {"bytes": rows * cols * (passes * size + 1) + cols * size + scales, "flops": 8 * rows * cols}
    rows, experts, n, k = case["rows"], case["experts"], case["n"], case["k"]
    kb = -(-k // BLOCK)
    touched = sum(1 - (1 - p) ** rows for p in _popularity(experts, case["routing"]))  # experts that have rows, on average
    weights = touched * (n * k + 4 * kb * -(-n // BLOCK))
    return {"bytes": weights + rows * (k + 4 * kb + 2 * n) + 4 * experts, "flops": 2 * rows * n * k}


# --------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------

_E4M3_STEPS = 8  # values to a power of two


def _exact_e4m3(v):
    """The e4m3 value next to each of v (|v| <= 448), ties to the even one, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))) / _E4M3_STEPS
    return torch.round(v / step) * step


def _exact_blocks(y):
    q = torch.empty_like(y)
    scale = y.new_empty(y.shape[0], -(-y.shape[1] // BLOCK))
    for c in range(scale.shape[1]):
        part = y[:, c * BLOCK:(c + 1) * BLOCK]
        scale[:, c] = part.abs().amax(1).clamp(min=TINY) / E4M3_MAX
        q[:, c * BLOCK:(c + 1) * BLOCK] = _exact_e4m3((part / scale[:, c:c + 1]).clamp(-E4M3_MAX, E4M3_MAX))
    return q, scale


def _exact_positions(ids, experts):
    """Row of each entry, from counts: entries of lower experts, and earlier ones of the same."""
    flat = ids.reshape(-1).long()
    rows = torch.full_like(flat, -1)
    start = 0
    for e in range(experts):
        mine = flat == e
        n = int(mine.sum())
        rows[mine] = torch.arange(start, start + n, device=flat.device)
        start += n
    return rows.reshape(ids.shape)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("sort", "unsort", "sort_grad", "unsort_grad"):
        places = _exact_positions(s["indices"], case["experts"])
        tokens, topk = places.shape
        if op == "sort":
            rows = torch.zeros(tokens * topk, case["hidden"], dtype=torch.float64, device="cuda")
            scale = None if s["scale"] is None else torch.zeros(tokens * topk, s["scale"].shape[1], dtype=torch.float64, device="cuda")
            for j in range(topk):
                has = places[:, j] >= 0
                rows[places[has, j]] = s["x"].to(torch.float64)[has]
                if scale is not None:
                    scale[places[has, j]] = s["scale"].double()[has]
            return {"rows": rows, "scale": scale, "offsets": None, "row_of": None}
        if op in ("unsort", "sort_grad"):
            source = s["rows"] if op == "unsort" else s["grad"]
            out = torch.zeros(tokens, case["hidden"], dtype=torch.float64, device="cuda")
            for j in range(topk):
                has = places[:, j] >= 0
                w = s["weights"][has, j].double() if op == "unsort" else 1.0
                out[has] += source[places[has, j]].double() * (w[:, None] if op == "unsort" else 1.0)
            return out
        rows = torch.zeros(tokens * topk, case["hidden"], dtype=torch.float64, device="cuda")
        weights = torch.zeros(tokens, topk, dtype=torch.float64, device="cuda")
        for j in range(topk):
            has = places[:, j] >= 0
            g = s["grad"][has].double()
            rows[places[has, j]] = g * s["weights"][has, j].double()[:, None]
            weights[has, j] = (g * s["rows"][places[has, j]].double()).sum(1)
        return [rows, weights]
    if op == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = h + s["residual"].double()
        y = h / torch.sqrt((h * h).sum(1, keepdim=True) / case["cols"] + EPS) * s["weight"].double()
        q, scale = _exact_blocks(y)
        return {"q": q, "scale": scale, "total": h if s["residual"] is not None else None, "normed": y if case["normed"] else None}
    if op == "silu_mul":
        gate, up = s["x"][:, :case["cols"]].double(), s["x"][:, case["cols"]:].double()
        q, scale = _exact_blocks(gate / (1 + torch.exp(-gate)) * up)
        return {"q": q, "scale": scale}
    if 2.0 * case["rows"] * case["n"] * case["k"] > 3e12:
        return None
    out = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        lo, hi = s["ends"][e], s["ends"][e + 1]
        if lo == hi:
            continue
        total = torch.zeros(hi - lo, case["n"], dtype=torch.float64, device="cuda")
        columns = torch.arange(case["n"], device="cuda") // BLOCK
        for kb in range(s["a_scale"].shape[1]):
            sl = slice(kb * BLOCK, min((kb + 1) * BLOCK, case["k"]))
            part = s["a"][lo:hi, sl].double() @ s["b"][e][:, sl].double().T
            total += part * s["a_scale"][lo:hi, kb, None].double() * s["b_scale"][e][columns, kb].double()
        out[lo:hi] = total
    return out
