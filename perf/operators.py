"""Workloads of the operators around expert products over the caller's own tensors.

The operators: sorting a router's picks into one run of rows per expert (group_rows), the
ragged products of those runs with 16-bit expert weights in both directions (grouped_mm,
grouped_mm_dx, grouped_mm_dw), quantising to e4m3 with one scale per block of 128
(fp8_quantize), and products of such operands, dense (fp8_mm) and ragged (fp8_grouped_mm).
`run` computes them either in a plain form (elementary torch operations in 32 bits, rounded
once at the end) or, with `own` set, through this repository's entry points; `exact`
computes the definition in 64 bits.
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
# the smallest scale: the smallest normal float, so that a code times its scale never loses bits
SCALE_MIN = 2.0 ** -126
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def _grouped(name, op, tokens, top_k, experts, n, k, dtype, out, world=1, skew=0.0):
    return {"name": name, "op": op, "tokens": tokens, "top_k": top_k, "experts": experts, "n": n, "k": k, "dtype": dtype,
            "out": out, "world": world, "skew": skew}


def listed():
    """Widths, expert counts and token counts are those of this repository's layer configurations."""
    return [
        # a decode step of 16 sequences, 8 of 128 experts each
        {"name": "group-decode", "op": "group", "tokens": 16, "top_k": 8, "experts": 128, "world": 1, "skew": 0.0},
        # a long prompt batch on one of two expert-parallel ranks: about half of the picks are masked
        {"name": "group-prefill-ep", "op": "group", "tokens": 16384, "top_k": 8, "experts": 128, "world": 2, "skew": 0.0},
        # activations of one decode step
        {"name": "quant-decode", "op": "quantize", "matrices": 1, "rows": 16, "cols": 2048, "block_rows": 1, "dtype": "bf16"},
        # expert activations of a prompt; the last block of a row has 64 columns
        {"name": "quant-prefill", "op": "quantize", "matrices": 1, "rows": 16384, "cols": 2880, "block_rows": 1,
         "dtype": "bf16"},
        # a shared expert's fused gate and up matrix, one token
        {"name": "fp8-dense-token", "op": "fp8_mm", "rows": 1, "n": 2816, "k": 2048, "out": "bf16"},
        # the dense first layer's gate matrix over a prompt
        {"name": "fp8-dense-prompt", "op": "fp8_mm", "rows": 2048, "n": 10944, "k": 2048, "out": "bf16"},
        # routed experts, 16 sequences decoding
        _grouped("fp8-experts-decode", "fp8_grouped", 16, 6, 64, 2816, 2048, "e4m3", "bf16"),
        # routed experts over a prompt, widths that end in half a block
        _grouped("fp8-experts-prompt", "fp8_grouped", 4096, 4, 128, 5760, 2880, "e4m3", "bf16"),
        # one token through eight bf16 experts
        _grouped("mm-token", "mm", 1, 8, 128, 1536, 2048, "bf16", "bf16"),
        # a prompt on one of two expert-parallel ranks, fp32 rows for the combine; rows behind the last group stay
        _grouped("mm-prompt-ep", "mm", 4096, 8, 128, 1536, 2048, "f16", "f32", world=2),
        # a small training step with skewed expert loads, fp32 weight gradients
        _grouped("backward-small", "mm_backward", 512, 6, 64, 2816, 2048, "f16", "f32", skew=1.2),
        # a training step of a wide layer
        _grouped("backward-wide", "mm_backward", 4096, 4, 32, 5760, 2880, "bf16", "bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _width(rng, lo, hi, align):
    # widths of matrices are nearly always a multiple of the vector length; one in eight is odd
    return _log(rng, lo, hi // 4) | 1 if rng.random() < 0.125 else max(align, _log(rng, lo, hi) // align * align)


MOST_FLOPS = {"fp8_mm": 2 * 2048 * 10944 * 2048, "fp8_grouped": 2 * 16384 * 5760 * 2880, "mm": 2 * 16384 * 1536 * 2048,
              "mm_backward": 4 * 16384 * 5760 * 2880}
MOST_WEIGHTS = {"fp8_mm": 10944 * 2880, "fp8_grouped": 128 * 5760 * 2880, "mm": 128 * 1536 * 2048,
                "mm_backward": 32 * 5760 * 2880}


def draw(rng):
    op = rng.choice(["group", "quantize", "fp8_mm", "fp8_grouped", "mm", "mm_backward"])
    if op == "group":
        experts = rng.choice([8, 32, 60, 64, 128, 256])
        return {"op": op, "tokens": _log(rng, 1, 16384), "top_k": rng.randint(1, 8), "experts": experts,
                "world": rng.choice([1, 1, 2, 4]), "skew": rng.choice([0.0, 0.0, 1.2])}
    if op == "quantize":
        block_rows = rng.choice([1, 1, BLOCK])
        rows, cols = _log(rng, 1, 16384), _width(rng, 64, 10944, 16)
        matrices = 1 if block_rows == 1 else rng.randint(1, 8)
        while matrices * rows * cols > 16384 * 2880:
            rows = max(1, rows // 2)
        return {"op": op, "matrices": matrices, "rows": rows, "cols": cols, "block_rows": block_rows,
                "dtype": rng.choice(["f32", "bf16", "bf16", "f16"])}
    if op == "fp8_mm":
        c = {"op": op, "rows": _log(rng, 1, 4096), "n": _log(rng, 64, 10944), "k": _width(rng, 64, 10944, 16),
             "out": rng.choice(["f32", "bf16", "f16"])}
        while c["n"] * c["k"] > MOST_WEIGHTS[op] or 2 * c["rows"] * c["n"] * c["k"] > MOST_FLOPS[op]:
            c["rows"] = max(1, c["rows"] // 2)
            c["n"] = max(64, c["n"] // 2)
        return c
    experts = rng.choice([8, 16, 32, 60, 64, 128])
    c = {"op": op, "tokens": _log(rng, 1, 4096), "top_k": rng.randint(1, 8), "experts": experts,
         "n": _width(rng, 64, 5760, 8), "k": _width(rng, 64, 2880, 16),
         "dtype": "e4m3" if op == "fp8_grouped" else rng.choice(["bf16", "f16"]), "out": rng.choice(["f32", "bf16", "f16"]),
         "world": rng.choice([1, 1, 2]), "skew": rng.choice([0.0, 0.0, 1.2])}
    cost = 4 if op == "mm_backward" else 2
    # the plain form pads every group to the longest one, which skewed loads make up to ten times the mean
    pad = 4 if c["skew"] else 1
    while cost * pad * c["tokens"] * c["top_k"] * c["n"] * c["k"] > MOST_FLOPS[op] or experts * c["n"] * c["k"] > MOST_WEIGHTS[op]:
        c["tokens"] = max(1, c["tokens"] * 3 // 4)
        c["n"] = max(64, c["n"] * 3 // 4 // 8 * 8)
    return c


# ---- inputs --------------------------------------------------------------------------------


def _route(case, gen):
    """Picks [tokens, top_k] of a router over world * experts experts (distinct in a row); those of the
    other ranks are -1.  skew: experts' popularity follows a power law of that exponent."""
    total = case["experts"] * case["world"]
    score = torch.randn(case["tokens"], total, generator=gen, device="cuda")
    if case["skew"]:
        rank = torch.argsort(torch.rand(total, generator=gen, device="cuda"))
        score = score - case["skew"] * torch.log(rank + 1.0)
    ids = torch.topk(score, case["top_k"], dim=1).indices.to(torch.int32)
    return torch.where(ids < case["experts"], ids, -1).contiguous()


def _offsets(ids, experts):
    flat = ids.flatten()
    counts = torch.bincount(torch.where(flat < 0, experts, flat).long(), minlength=experts + 1)[:experts]
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)


def _codes(gen, shape, sigma):
    """e4m3 codes of Gaussian blocks scaled to their largest entry."""
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0, sigma, generator=gen) \
        .clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _scales(gen, shape, mean):
    return mean * torch.exp(0.3 * torch.randn(shape, generator=gen, device="cuda"))


def _blocks(v):
    return -(-v // BLOCK)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"op": op, "case": case}
    if op == "group":
        s["ids"] = _route(case, gen)
        return s
    if op == "quantize":
        shape = (case["rows"], case["cols"]) if case["matrices"] == 1 else (case["matrices"], case["rows"], case["cols"])
        x = torch.randn(shape, generator=gen, device="cuda")
        x = x * torch.exp(torch.randn(shape[:-1] + (1,), generator=gen, device="cuda"))  # rows of unlike size
        x[..., 1::509] *= 20.0  # a few outlier channels, as activations have
        s["x"] = x.to(DTYPES[case["dtype"]])
        return s
    n, k = case["n"], case["k"]
    if op == "fp8_mm":
        rows = case["rows"]
        s["x"], s["xs"] = _codes(gen, (rows, k), 166.0), _scales(gen, (_blocks(k), rows), 6e-3).t()
        s["w"], s["ws"] = _codes(gen, (n, k), 112.0), _scales(gen, (_blocks(n), _blocks(k)), 2e-4)
        return s
    experts = case["experts"]
    ids = _route(case, gen)
    rows = ids.numel()
    s["offsets"] = _offsets(ids, experts)
    s["cap"] = max(1, int((s["offsets"][1:] - s["offsets"][:-1]).max()))  # longest group: the plain form pads to it
    if op == "fp8_grouped":
        s["x"], s["xs"] = _codes(gen, (rows, k), 166.0), _scales(gen, (_blocks(k), rows), 6e-3).t()
        s["w"], s["ws"] = _codes(gen, (experts, n, k), 112.0), _scales(gen, (experts, _blocks(n), _blocks(k)), 2e-4)
        s["y"] = torch.zeros(rows, n, dtype=DTYPES[case["out"]], device="cuda")
        return s
    dt = DTYPES[case["dtype"]]
    s["w"] = torch.empty(experts, n, k, dtype=dt, device="cuda").normal_(0, 0.02, generator=gen)
    s["x"] = torch.empty(rows, k, dtype=dt, device="cuda").normal_(0, 1.0, generator=gen)
    if op == "mm":
        s["y"] = torch.zeros(rows, n, dtype=DTYPES[case["out"]], device="cuda")
    else:
        s["dy"] = torch.empty(rows, n, dtype=dt, device="cuda").normal_(0, 1.0, generator=gen)
        s["dx"] = torch.zeros(rows, k, dtype=dt, device="cuda")
    return s


# ---- plain forms ---------------------------------------------------------------------------


def _plain_group(ids, experts):
    k = ids.shape[1]
    flat = ids.flatten().long()
    key = torch.where(flat < 0, experts, flat)
    ordered, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(ordered, torch.arange(experts + 1, device=ids.device))
    row_token = torch.where(ordered < experts, order // k, 0)
    row_of_job = torch.empty_like(order)
    row_of_job[order] = torch.arange(order.numel(), device=ids.device)
    row_of_job = torch.where(flat < 0, -1, row_of_job).view(ids.shape)
    return offsets.to(torch.int32), row_token.to(torch.int32), row_of_job.to(torch.int32)


def _plain_quantize(x, block_rows):
    m = x.float().reshape(-1, x.shape[-2], x.shape[-1])
    count, rows, cols = m.shape
    br, bc = -(-rows // block_rows), _blocks(cols)
    m = torch.nn.functional.pad(m, (0, bc * BLOCK - cols, 0, br * block_rows - rows))
    m = m.view(count, br, block_rows, bc, BLOCK)
    amax = m.abs().amax(dim=(2, 4))
    scale = torch.clamp(amax / E4M3_MAX, min=SCALE_MIN)
    q = (m / scale[:, :, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    q = q.view(count, br * block_rows, bc * BLOCK)[:, :rows, :cols].reshape(x.shape)
    return q, scale.view(x.shape[:-2] + (br, bc))


def _rows_dequant(q, scales):
    return q.float() * scales.repeat_interleave(BLOCK, dim=1)[:, :q.shape[1]]


def _weights_dequant(q, scales):
    s = scales.repeat_interleave(BLOCK, dim=-2).repeat_interleave(BLOCK, dim=-1)
    return q.float() * s[..., :q.shape[-2], :q.shape[-1]]


def _expert_of_row(offsets, rows):
    """Each row's expert (the number of experts behind the last group) and its place in the group."""
    r = torch.arange(rows, device=offsets.device)
    e = torch.searchsorted(offsets[1:].contiguous(), r.to(torch.int32), right=True)
    return e, r - offsets[e.clamp(max=offsets.numel() - 1)]


def _padded(x, slot, experts, cap):
    buf = x.new_zeros(experts * cap + 1, x.shape[1])
    buf[slot] = x
    return buf[:-1].view(experts, cap, x.shape[1])


def _slots(offsets, rows, experts, cap):
    e, place = _expert_of_row(offsets, rows)
    return torch.where(e < experts, e * cap + place, experts * cap), e < experts


def _from_padded(y, slot, valid, before):
    flat = y.reshape(-1, y.shape[2])
    rows = flat[slot.clamp(max=flat.shape[0] - 1)].to(before.dtype)
    return torch.where(valid[:, None], rows, before)


def _plain_mm(x, w, dequant, offsets, cap, before):
    """Rows of each group times that expert's transposed weights, in 32 bits."""
    rows, experts = x.shape[0], offsets.numel() - 1
    slot, valid = _slots(offsets, rows, experts, cap)
    if rows <= 16:  # few rows: gather each row's matrix
        e = (slot // cap).clamp(max=experts - 1)
        y = torch.matmul(dequant(w, e), x[:, :, None])[:, :, 0]
        return torch.where(valid[:, None], y.to(before.dtype), before)
    return _from_padded(torch.bmm(_padded(x, slot, experts, cap), dequant(w, None).transpose(1, 2)), slot, valid, before)


def _pick(t, e):
    return t if e is None else t[e]


def run(s):
    case, op = s["case"], s["op"]
    if own:
        from __graft_entry__ import load_package
        u = load_package().umsx
        if op == "group":
            return u.group_rows(s["ids"], case["experts"])
        if op == "quantize":
            return u.fp8_quantize(s["x"], block_rows=case["block_rows"])
        if op == "fp8_mm":
            return u.fp8_mm(s["x"], s["xs"], s["w"], s["ws"], out_dtype=DTYPES[case["out"]])
        if op == "fp8_grouped":
            return u.fp8_grouped_mm(s["x"], s["xs"], s["w"], s["ws"], s["offsets"], out=s["y"])
        if op == "mm":
            return u.grouped_mm(s["x"], s["w"], s["offsets"], out=s["y"])
        return (u.grouped_mm_dx(s["dy"], s["w"], s["offsets"], out=s["dx"]),
                u.grouped_mm_dw(s["dy"], s["x"], s["offsets"], out_dtype=DTYPES[case["out"]]))
    if op == "group":
        return _plain_group(s["ids"], case["experts"])
    if op == "quantize":
        return _plain_quantize(s["x"], case["block_rows"])
    if op == "fp8_mm":
        y = torch.matmul(_rows_dequant(s["x"], s["xs"]), _weights_dequant(s["w"], s["ws"]).t())
        return y.to(DTYPES[case["out"]])
    if op == "fp8_grouped":
        return _plain_mm(_rows_dequant(s["x"], s["xs"]), (s["w"], s["ws"]),
                         lambda w, e: _weights_dequant(_pick(w[0].view(torch.uint8), e).view(torch.float8_e4m3fn), _pick(w[1], e)),
                         s["offsets"], s["cap"], s["y"])
    if op == "mm":
        return _plain_mm(s["x"].float(), s["w"], lambda w, e: _pick(w, e).float(), s["offsets"], s["cap"], s["y"])
    rows, experts, cap = s["x"].shape[0], case["experts"], s["cap"]
    slot, valid = _slots(s["offsets"], rows, experts, cap)
    dy = _padded(s["dy"].float(), slot, experts, cap)
    dx = _from_padded(torch.bmm(dy, s["w"].float()), slot, valid, s["dx"])
    dw = torch.bmm(dy.transpose(1, 2), _padded(s["x"].float(), slot, experts, cap))
    return dx, dw.to(DTYPES[case["out"]])


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "group":
        jobs = case["tokens"] * case["top_k"]
        return {"bytes": 4 * (3 * jobs + case["experts"] + 1), "flops": jobs}
    if op == "quantize":
        values = case["matrices"] * case["rows"] * case["cols"]
        scales = case["matrices"] * -(-case["rows"] // case["block_rows"]) * _blocks(case["cols"])
        return {"bytes": values * (SIZES[case["dtype"]] + 1) + 4 * scales, "flops": 2 * values}
    n, k = case["n"], case["k"]
    if op == "fp8_mm":
        rows = case["rows"]
        return {"bytes": rows * k + 4 * rows * _blocks(k) + n * k + 4 * _blocks(n) * _blocks(k) + rows * n * SIZES[case["out"]],
                "flops": 2 * rows * n * k}
    rows = max(1, case["tokens"] * case["top_k"] // case["world"])
    # experts that some row chose, for picks that are spread evenly
    total = case["experts"] * case["world"]
    used = max(1, int(case["experts"] * (1 - (1 - case["top_k"] / total) ** case["tokens"])))
    if op == "fp8_grouped":
        return {"bytes": rows * (k + 4 * _blocks(k)) + used * (n * k + 4 * _blocks(n) * _blocks(k)) + rows * n * SIZES[case["out"]],
                "flops": 2 * rows * n * k}
    if op == "mm":
        return {"bytes": 2 * rows * k + 2 * used * n * k + rows * n * SIZES[case["out"]], "flops": 2 * rows * n * k}
    return {"bytes": 2 * rows * (n + 2 * k) + 2 * used * n * k + case["experts"] * n * k * SIZES[case["out"]],
            "flops": 4 * rows * n * k}


# ---- the definition in 64 bits ------------------------------------------------------------------


def _e4m3_round(v):
    """Nearest e4m3 value (3 bits behind the leading one, steps of 2^-9 below 2^-6, at most 448), ties to even."""
    a = v.abs()
    exponent = torch.floor(torch.log2(torch.clamp(a, min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return torch.sign(v) * torch.clamp(torch.round(a / step) * step, max=448.0)


def _exact_quantize(x, block_rows):
    count, rows, cols = (1,) * (3 - x.dim()) + tuple(x.shape)
    m = x.double().reshape(count, rows, cols)
    q = torch.empty_like(m)
    scales = torch.empty(count, -(-rows // block_rows), _blocks(cols), dtype=torch.float64, device=x.device)
    for j in range(_blocks(cols)):
        at = slice(j * BLOCK, min(cols, (j + 1) * BLOCK))
        if block_rows == 1:
            sc = torch.clamp(m[:, :, at].abs().amax(2) / 448.0, min=2.0 ** -126)
            scales[:, :, j], each = sc, sc[:, :, None]
            q[:, :, at] = _e4m3_round(m[:, :, at] / each)
            continue
        for i in range(-(-rows // block_rows)):
            part = m[:, i * block_rows:(i + 1) * block_rows, at]
            sc = torch.clamp(part.abs().amax((1, 2)) / 448.0, min=2.0 ** -126)
            scales[:, i, j] = sc
            q[:, i * block_rows:(i + 1) * block_rows, at] = _e4m3_round(part / sc[:, None, None])
    return q.reshape(x.shape), scales.reshape(x.shape[:-2] + scales.shape[-2:])


def _exact_dequant(q, scales):
    """One matrix: entry (i, j) times the scale of its block; rows have blocks of one or of 128."""
    i = torch.arange(q.shape[0], device=q.device)
    i = i if scales.shape[0] == q.shape[0] else i // BLOCK
    j = torch.arange(q.shape[1], device=q.device) // BLOCK
    return q.to(torch.float64) * scales.double()[i][:, j]


def exact(case, seed):
    op = case["op"]
    if op == "group":
        return None  # whole numbers: the plain form is exact
    s = prepare(case, seed)
    if op == "quantize":
        return _exact_quantize(s["x"], case["block_rows"])
    if op == "fp8_mm":
        xd = s["x"].to(torch.float64) * s["xs"].double()[:, torch.arange(case["k"], device="cuda") // BLOCK]
        i, j = torch.arange(case["n"], device="cuda") // BLOCK, torch.arange(case["k"], device="cuda") // BLOCK
        return xd @ (s["w"].to(torch.float64) * s["ws"].double()[i][:, j]).T
    ends = s["offsets"].tolist()
    if op in ("fp8_grouped", "mm"):
        y = s["y"].double()
        j = torch.arange(case["k"], device="cuda") // BLOCK
        for e in range(case["experts"]):
            a, b = ends[e], ends[e + 1]
            if a == b:
                continue
            if op == "mm":
                y[a:b] = s["x"][a:b].double() @ s["w"][e].double().T
            else:
                xd = s["x"][a:b].to(torch.float64) * s["xs"][a:b].double()[:, j]
                i = torch.arange(case["n"], device="cuda") // BLOCK
                y[a:b] = xd @ (s["w"][e].to(torch.float64) * s["ws"][e].double()[i][:, j]).T
        return y
    dx = s["dx"].double()
    dw = torch.zeros(case["experts"], case["n"], case["k"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        a, b = ends[e], ends[e + 1]
        dy = s["dy"][a:b].double()
        dx[a:b] = dy @ s["w"][e].double()
        dw[e] = dy.T @ s["x"][a:b].double()
    return dx, dw
