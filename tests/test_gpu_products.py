"""Row grouping, ragged 16-bit products with their gradients, and block-scaled e4m3 products against plain
64-bit forms (needs a B200).

Tolerances, element by element: a sum of C products accumulated in fp32 in any order is off by at most
C * 2^-23 * sum|a b| (one ulp for every addition, truncated or rounded; products of 16- and 8-bit operands are exact in
fp32), the scales of an e4m3 product add three more roundings per block, and the result is rounded once to the
output's type: eps / 2 of the value, or half the smallest subnormal step.
"""
import pytest

from tests.helpers import U

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
SUB = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(gen, *shape, dtype=BF16):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _close(got, want, size, terms, what):
    """got (rounded) against want and size = sum|a b| (both fp64)."""
    half = torch.finfo(got.dtype).eps / 2
    acc = (terms + 8) * 2.0 ** -23 * size
    tol = acc + half * (want.abs() + acc) + SUB[got.dtype]
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol)[bad].max())} x tolerance"


def _offsets(counts, start=0):
    return torch.tensor([start] + [start + sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int32, device="cuda")


def _spans(offsets):
    o = offsets.tolist()
    return list(enumerate(zip(o[:-1], o[1:])))


# group sizes, rows before the first and behind the last group
RAGGED = [
    ([1], 0, 0),
    ([0, 3, 0, 1, 0], 0, 0),
    ([0, 0, 0], 0, 5),
    ([7, 9, 16, 17, 1], 2, 3),
    ([1] * 8 + [0] * 120, 0, 0),
    ([33, 0, 129, 64, 255, 256, 257, 1], 0, 70),
    ([700, 13], 1, 0),
]
# n, k: tensor-core sizes, sizes that end inside a tile, odd ones that only the general kernel takes
WIDTHS = [(128, 64), (256, 256), (384, 512), (72, 200), (136, 1032), (17, 33), (1, 1), (1000, 8), (8, 136), (130, 128)]


def _case(counts, before, behind, n, k, dtype, seed, pad=0):
    """x, dy, w, offsets; rows outside the groups hold NaN, which must reach nothing.  pad: columns between rows."""
    g = _gen(seed)
    rows = before + sum(counts) + behind
    x = torch.full((rows, k + pad), float("nan"), dtype=dtype, device="cuda")[:, :k]
    dy = torch.full((rows, n + pad), float("nan"), dtype=dtype, device="cuda")[:, :n]
    a, b = before, before + sum(counts)
    x[a:b] = _rand(g, b - a, k, dtype=dtype)
    dy[a:b] = _rand(g, b - a, n, dtype=dtype)
    w = torch.empty(len(counts), n, k + pad, dtype=dtype, device="cuda")[:, :, :k]
    w.copy_(_rand(g, len(counts), n, k, dtype=dtype))
    return x, dy, w, _offsets(counts, before)


def _check_all(counts, before, behind, n, k, dtype, out, seed, pad=0):
    x, dy, w, off = _case(counts, before, behind, n, k, dtype, seed, pad)
    rows = x.shape[0]
    y = torch.full((rows, n), 7.0, dtype=out, device="cuda")
    dx = torch.full((rows, k), -3.0, dtype=out, device="cuda")
    dw = torch.full((len(counts), n, k), float("nan"), dtype=out, device="cuda")
    assert U.grouped_mm(x, w, off, out=y) is y
    assert U.grouped_mm_dx(dy, w, off, out=dx) is dx
    assert U.grouped_mm_dw(dy, x, off, out=dw) is dw
    a, b = before, before + sum(counts)
    for t, keep in ((y, 7.0), (dx, -3.0)):
        assert torch.all(t[:a] == keep) and torch.all(t[b:] == keep), "rows outside the groups were written"
    for e, (i, j) in _spans(off):
        xe, dye, we = x[i:j].double(), dy[i:j].double(), w[e].double()
        _close(y[i:j], xe @ we.T, xe.abs() @ we.abs().T, k, f"y of expert {e}")
        _close(dx[i:j], dye @ we, dye.abs() @ we.abs(), n, f"dx of expert {e}")
        _close(dw[e], dye.T @ xe, dye.abs().T @ xe.abs(), j - i, f"dw of expert {e}")


@pytest.mark.parametrize("n,k", WIDTHS)
@pytest.mark.parametrize("ragged", range(len(RAGGED)))
def test_products_and_gradients(ragged, n, k):
    dtype = BF16 if (ragged + n) % 2 else F16
    out = (F32, dtype, BF16)[(ragged + k) % 3]
    _check_all(*RAGGED[ragged], n, k, dtype, out, seed=100 * ragged + n)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_types_and_strides(dtype, out, pad):
    _check_all([40, 0, 5, 300], 1, 2, 192, 320, dtype, out, seed=7, pad=pad)


def test_wide_outputs_and_many_experts():
    """1024 experts, most of them empty; and an n above any tile count of one wave."""
    counts = [0] * 1024
    for e in range(0, 1024, 37):
        counts[e] = 1 + e % 5
    _check_all(counts, 0, 0, 64, 64, BF16, BF16, seed=3)
    _check_all([65, 3], 0, 0, 20000, 64, BF16, F32, seed=4)


def test_gradients_against_differences():
    """dx and dw are the derivatives of sum(y * dy): directional differences of the 64-bit product of nudged operands."""
    x, dy, w, off = _case([5, 0, 12], 0, 0, 40, 24, BF16, seed=11)
    dx, dw = U.grouped_mm_dx(dy, w, off, out_dtype=F32).double(), U.grouped_mm_dw(dy, x, off).double()

    def loss(xd, wd):
        return sum((xd[i:j] @ wd[e].T * dy[i:j].double()).sum() for e, (i, j) in _spans(off))

    g = _gen(5)
    vx, vw = torch.randn(x.shape, generator=g, device="cuda").double(), torch.randn(w.shape, generator=g, device="cuda").double()
    xd, wd, h = x.double(), w.double(), 2.0 ** -10
    # the loss is linear in each operand: central differences are exact but for fp64 rounding
    want_x = (loss(xd + h * vx, wd) - loss(xd - h * vx, wd)) / (2 * h)
    want_w = (loss(xd, wd + h * vw) - loss(xd, wd - h * vw)) / (2 * h)
    # each gradient entry is off by at most (terms + 8) 2^-23 sum|a b| + half an ulp
    ax = sum((dy[i:j].double().abs() @ w[e].double().abs() * vx[i:j].abs()).sum() for e, (i, j) in _spans(off))
    aw = sum((dy[i:j].double().abs().T @ x[i:j].double().abs() * vw[e].abs()).sum() for e, (i, j) in _spans(off))
    assert abs((dx * vx).sum() - want_x) <= 50 * 2.0 ** -23 * ax
    assert abs((dw * vw).sum() - want_w) <= 50 * 2.0 ** -23 * aw


def test_non_finite_values_stay_in_their_rows():
    x, dy, w, off = _case([20, 300, 7], 0, 0, 128, 256, BF16, seed=2)
    clean = U.grouped_mm(x, w, off)
    x2 = x.clone()
    x2[25, 3], x2[319, 0] = float("nan"), float("inf")
    y = U.grouped_mm(x2, w, off)
    rows = [r for r in range(x.shape[0]) if r not in (25, 319)]
    assert torch.equal(y[rows], clean[rows]) and torch.isnan(y[25]).all() and not torch.isfinite(y[319]).any()
    dw, dw2 = U.grouped_mm_dw(dy, x, off), U.grouped_mm_dw(dy, x2, off)
    assert torch.equal(dw[0], dw2[0]) and torch.equal(dw[2], dw2[2])
    assert torch.isnan(dw2[1][:, 3]).all() and torch.equal(dw[1][:, 4:], dw2[1][:, 4:])
    w2 = w.clone()
    w2[1] = float("nan")
    y = U.grouped_mm(x, w2, off)
    assert torch.equal(y[:20], clean[:20]) and torch.equal(y[320:], clean[320:]) and torch.isnan(y[20:320]).all()


def test_bad_offsets_stay_inside_the_matrices():
    """Offsets outside 0..rows are clamped, descending ones give empty groups: nothing outside is touched."""
    x, dy, w, _ = _case([30, 30], 0, 0, 64, 64, BF16, seed=9)
    for o in ([0, 30, 1000], [-50, 30, 60], [60, 20, 60], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]):
        off = torch.tensor(o, dtype=torch.int32, device="cuda")
        y = torch.zeros(62, 64, dtype=F32, device="cuda")
        U.grouped_mm(x, w, off, out=y[1:61])
        U.grouped_mm_dw(dy, x, off)
        U.grouped_mm_dx(dy, w, off)
        torch.cuda.synchronize()
        assert not y[0].any() and not y[61].any()


# ---- e4m3 ------------------------------------------------------------------------------------------


def _round_e4m3(v):
    a = v.abs()
    step = torch.exp2(torch.floor(torch.log2(torch.clamp(a, min=2.0 ** -6))) - 3)
    return torch.sign(v) * torch.clamp(torch.round(a / step) * step, max=448.0)


def _blocks(v):
    return -(-v // 128)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1), (3, 128), (5, 130), (128, 64), (129, 257), (300, 2880), (2, 131, 200), (3, 1, 77)])
def test_quantize(dtype, block_rows, shape):
    g = _gen(shape[-1])
    x = (torch.randn(shape, generator=g, device="cuda") * torch.exp(3 * torch.randn(shape[:-1] + (1,), generator=g, device="cuda")))
    x = x.to(dtype)
    x[..., 0] = 0
    q, s = U.fp8_quantize(x, block_rows)
    assert q.dtype == E4M3 and q.shape == x.shape and s.shape == shape[:-2] + (-(-shape[-2] // block_rows), _blocks(shape[-1]))
    rows, cols = shape[-2:]
    x3, q3, s3 = x.float().reshape(-1, rows, cols), q.float().reshape(-1, rows, cols), s.reshape((-1,) + s.shape[-2:])
    for i in range(s.shape[-2]):
        for j in range(s.shape[-1]):
            xb = x3[:, i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128]
            # the fp32 divisions, as documented: a 64-bit quotient of fp32 values rounds to fp32 as theirs does
            # (torch divides an fp32 CUDA tensor by a number through its reciprocal, which is one ulp off)
            fine = torch.isfinite(xb)  # some rows overflow fp16
            want = torch.clamp(torch.where(fine, xb, 0).abs().amax((1, 2)).double() / 448.0, min=2.0 ** -126).float()
            assert torch.equal(s3[:, i, j], want)
            qb = q3[:, i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128]
            exact = _round_e4m3((torch.where(fine, xb, 0).double() / want.double()[:, None, None]).float().double()).float()
            assert torch.equal(torch.isnan(qb), ~fine) and torch.equal(torch.where(fine, qb, 0), exact)
        if i >= 8:
            break


def test_quantize_edges():
    """Zeros, subnormals, the largest floats, and non-finite values beside finite ones."""
    x = torch.zeros(6, 256, device="cuda")
    x[1, :128] = 1e-45
    x[2] = torch.finfo(F32).max
    x[3, 5], x[3, 6], x[3, 7], x[3, 8] = float("inf"), float("nan"), -float("inf"), 2.0
    x[4, 200] = -448.0
    x[5] = 2.0 ** -126
    q, s = U.fp8_quantize(x)
    assert torch.isfinite(s).all() and (s >= 2.0 ** -126).all()
    assert not q[0].float().any() and not q[1].float().any()
    assert (q[2].float() == 448).all()
    assert torch.isnan(q[3, 5:8].float()).all() and q[3, 8].float() == 448 and not q[3, 9:].float().any()
    assert s[4, 1] == 1 and q[4, 200].float() == -448
    assert (q[5].float() == 1).all()


def test_quantize_strides_and_given_outputs():
    g = _gen(1)
    big = torch.randn(70, 3 * 400, generator=g, device="cuda", dtype=F32).to(BF16)
    x = big[3:53, 405:405 + 300]  # rows that start at odd offsets
    q0, s0 = U.fp8_quantize(x.contiguous())
    store = torch.full((52, 320), 99, dtype=torch.uint8, device="cuda")
    q = store[1:51, 7:307].view(E4M3)
    scales = torch.zeros(50, 5, device="cuda")[:, 1:4]
    U.fp8_quantize(x, q=q, scales=scales)
    assert torch.equal(q.float(), q0.float()) and torch.equal(scales, s0)
    assert (store[0] == 99).all() and (store[51] == 99).all() and (store[:, :7] == 99).all() and (store[:, 307:] == 99).all()


def _fp8_case(counts, before, behind, n, k, seed, pad=0):
    g = _gen(seed)
    rows, e = before + sum(counts) + behind, len(counts)
    x = torch.full((rows, k + pad), 0x7F, dtype=torch.uint8, device="cuda")[:, :k].view(E4M3)  # NaN outside the groups
    a, b = before, before + sum(counts)
    x[a:b] = (100 * torch.randn(b - a, k, generator=g, device="cuda")).clamp(-448, 448).to(E4M3)
    w = torch.empty(e, n, k + pad, dtype=torch.uint8, device="cuda")[:, :, :k].view(E4M3)
    w.copy_((100 * torch.randn(e, n, k, generator=g, device="cuda")).clamp(-448, 448).to(E4M3))
    xs = torch.exp(torch.randn(_blocks(k), rows, generator=g, device="cuda")).t() * 0.01
    ws = torch.exp(torch.randn(e, _blocks(n), _blocks(k), generator=g, device="cuda")) * 0.001
    return x, xs, w, ws, _offsets(counts, before)


def _fp8_want(x, xs, w, ws):
    j = torch.arange(x.shape[1], device="cuda") // 128
    i = torch.arange(w.shape[0], device="cuda") // 128
    xd, wd = x.to(F32).double() * xs.double()[:, j], w.to(F32).double() * ws.double()[i][:, j]
    return xd @ wd.T, xd.abs() @ wd.abs().T


FP8_WIDTHS = [(128, 128), (256, 512), (384, 64), (72, 208), (136, 1040), (17, 33), (1, 1), (1000, 16), (130, 2880), (2816, 144)]


@pytest.mark.parametrize("n,k", FP8_WIDTHS)
@pytest.mark.parametrize("ragged", range(len(RAGGED)))
def test_fp8_grouped(ragged, n, k):
    counts, before, behind = RAGGED[ragged]
    x, xs, w, ws, off = _fp8_case(counts, before, behind, n, k, seed=10 * ragged + n)
    out = (BF16, F32, F16)[(ragged + n) % 3]
    y = torch.full((x.shape[0], n), 5.0, dtype=out, device="cuda")
    assert U.fp8_grouped_mm(x, xs, w, ws, off, out=y) is y
    a, b = before, before + sum(counts)
    assert (y[:a] == 5).all() and (y[b:] == 5).all()
    for e, (i, j) in _spans(off):
        want, size = _fp8_want(x[i:j], xs[i:j], w[e], ws[e])
        _close(y[i:j], want, size, k, f"expert {e}")


@pytest.mark.parametrize("rows", [0, 1, 2, 8, 9, 31, 64, 200, 1025])
@pytest.mark.parametrize("n,k", [(128, 128), (700, 1056), (24, 129), (2816, 2048)])
@pytest.mark.parametrize("pad", [0, 16])
def test_fp8_dense(rows, n, k, pad):
    x, xs, w, ws, _ = _fp8_case([rows], 0, 0, n, k, seed=rows + n, pad=pad)
    for scales in (xs, xs.contiguous()):  # either layout of the rows' scales
        for out in (F32, BF16):
            y = U.fp8_mm(x, scales, w[0], ws[0], out_dtype=out)
            assert y.shape == (rows, n) and y.dtype == out
            if rows:
                want, size = _fp8_want(x, xs, w[0], ws[0])
                _close(y, want, size, k, "y")


def test_fp8_non_finite_codes_stay_in_their_rows():
    x, xs, w, ws, off = _fp8_case([20, 300, 7], 0, 0, 128, 256, seed=2)
    clean = U.fp8_grouped_mm(x, xs, w, ws, off)
    bad = x.view(torch.uint8).clone()
    bad[25, 3] = 0x7F
    y = U.fp8_grouped_mm(bad.view(E4M3), xs, w, ws, off)
    rows = [r for r in range(x.shape[0]) if r != 25]
    assert torch.equal(y[rows], clean[rows]) and torch.isnan(y[25]).all()


# ---- grouping -----------------------------------------------------------------------------------------


def _group_want(ids, experts):
    flat = ids.flatten().long().cpu()
    key = torch.where((flat < 0) | (flat >= experts), experts, flat)
    order = torch.argsort(key, stable=True)
    off = torch.zeros(experts + 1, dtype=torch.int64)
    off[1:] = torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0)
    rows = int(off[-1])
    token = order // ids.shape[1]
    token[rows:] = 0
    job = torch.full((flat.numel(),), -1, dtype=torch.int64)
    job[order[:rows]] = torch.arange(rows)
    return off, token, job.view(ids.shape)


@pytest.mark.parametrize("tokens,top_k,experts", [(0, 4, 8), (1, 1, 1), (1, 8, 128), (5, 3, 7), (16, 8, 128), (128, 8, 60),
                                                  (129, 8, 60), (1000, 1, 1024), (4096, 8, 1024), (513, 6, 64), (70000, 8, 256)])
@pytest.mark.parametrize("kind", ["even", "masked", "one", "none"])
def test_group_rows(tokens, top_k, experts, kind):
    g = _gen(tokens + experts)
    ids = torch.randint(0, experts, (tokens, top_k), generator=g, device="cuda", dtype=torch.int32)
    if kind == "masked":
        ids = torch.where(torch.rand(ids.shape, generator=g, device="cuda") < 0.6, -1, ids)
        if tokens > 3:
            ids[1, 0], ids[2, 0], ids[3, 0] = experts, 2 ** 31 - 1, -2 ** 31
    elif kind == "one":
        ids[:] = experts - 1
    elif kind == "none":
        ids[:] = -1
    got = U.group_rows(ids, experts)
    for name, a, b in zip(("offsets", "row_token", "row_of_job"), got, _group_want(ids, experts)):
        assert a.dtype == torch.int32
        assert torch.equal(a.cpu().long(), b), name


@pytest.mark.parametrize("jobs", [512, 513, 1536, 1537, 2048, 4095, 4096, 4097, 65536, 65537, 1048577])
@pytest.mark.parametrize("experts", [7, 255, 256, 1024])
def test_group_rows_around_its_launch_shapes(jobs, experts):
    g = _gen(jobs + experts)
    ids = torch.randint(-1, experts, (jobs, 1), generator=g, device="cuda", dtype=torch.int32)
    got = U.group_rows(ids, experts)
    for name, a, b in zip(("offsets", "row_token", "row_of_job"), got, _group_want(ids, experts)):
        assert torch.equal(a.cpu().long(), b), name


# ---- use -------------------------------------------------------------------------------------------------


def test_refusals():
    x, dy, w, off = _case([3, 4], 0, 0, 64, 32, BF16, seed=1)
    xq, xs, wq, ws, _ = _fp8_case([3, 4], 0, 0, 64, 32, seed=1)
    bad = [
        lambda: U.grouped_mm(x.float(), w, off), lambda: U.grouped_mm(x, w.half(), off), lambda: U.grouped_mm(x[:, :16], w, off),
        lambda: U.grouped_mm(x, w, off[:2]), lambda: U.grouped_mm(x, w, off.long()), lambda: U.grouped_mm(x, w, off.cpu()),
        lambda: U.grouped_mm(x.t(), w, off), lambda: U.grouped_mm(x, w.transpose(1, 2), off),
        lambda: U.grouped_mm(x, w, off, out_dtype=torch.float64), lambda: U.grouped_mm(x, w, off, out=torch.empty(7, 63, device="cuda")),
        lambda: U.grouped_mm(x, w, off, out=torch.empty(7, 64)), lambda: U.grouped_mm(x[:1].expand(7, 32), w, off),
        lambda: U.grouped_mm(x, w[:1].expand(2, 64, 32), off),
        lambda: U.grouped_mm_dx(x, w, off), lambda: U.grouped_mm_dw(dy[:3], x, off), lambda: U.grouped_mm_dw(dy, x, off[0]),
        lambda: U.grouped_mm_dw(dy, x.half(), off), lambda: U.grouped_mm_dw(dy, x, off[:1]),
        lambda: U.fp8_mm(x, xs, wq[0], ws[0]), lambda: U.fp8_mm(xq, xs.double(), wq[0], ws[0]), lambda: U.fp8_mm(xq, xs[:3], wq[0], ws[0]),
        lambda: U.fp8_mm(xq, xs, wq, ws), lambda: U.fp8_grouped_mm(xq, xs, wq, ws, None), lambda: U.fp8_grouped_mm(xq, xs, wq, ws[:1], off),
        lambda: U.fp8_quantize(x[0]), lambda: U.fp8_quantize(x, 64), lambda: U.fp8_quantize(x.t()), lambda: U.fp8_quantize(xq),
        lambda: U.fp8_quantize(x, q=xq[:3]), lambda: U.fp8_quantize(x, scales=xs[:3]),
        lambda: U.group_rows(off, 4), lambda: U.group_rows(off[None].long(), 4), lambda: U.group_rows(off[None], 0),
        lambda: U.group_rows(off[None], 2000), lambda: U.group_rows(torch.zeros(4, 4, dtype=torch.int32, device="cuda").t()[:, :2], 4),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(U.UmsxError) as e:
            call()
        assert e.value.status == U.EINVAL, i


def _expert_layer(x, ids, weights, gate_up, down, experts):
    """An expert layer as a user builds it from the e4m3 operators; returns its output [tokens, width] in fp32."""
    off, row_token, row_of_job = U.group_rows(ids, experts)
    xq, xs = U.fp8_quantize(x)
    xs_rows = xs.t()[:, row_token].t()
    h = U.fp8_grouped_mm(xq.view(torch.uint8)[row_token].view(E4M3), xs_rows, *gate_up, off)
    gate, up = h.float().chunk(2, dim=1)
    a = (torch.nn.functional.silu(gate) * up).to(BF16)
    y = U.fp8_grouped_mm(*U.fp8_quantize(a), *down, off, out_dtype=F32)
    jobs = y[row_of_job.clamp(min=0)]
    jobs = torch.where((row_of_job < 0)[..., None], 0.0, jobs)
    return U.combine(jobs, weights)


def test_expert_layer_of_e4m3_weights():
    """Router, grouping, quantiser, both products and the combine in a row, as they are used; against the same layer in
    64 bits on the operands' exact values.  The activations are rounded to bf16 once and to e4m3 twice on the way, which
    the 64-bit layer repeats, so that what is left is the accumulation and rounding of each step."""
    T, H, I, E, K = 37, 256, 192, 8, 2
    g = _gen(21)
    x = _rand(g, T, H)
    rw = torch.randn(E, H, generator=g, device="cuda") * 0.1
    ids, weights, _ = U.route_static(x, rw, None, E, K, U.ROUTE_SOFTMAX_TOPK_NORM)
    ids[5, 1] = -1
    gu = U.fp8_quantize(torch.randn(E, 2 * I, H, generator=g, device="cuda") * 0.05, 128)
    dn = U.fp8_quantize(torch.randn(E, H, I, generator=g, device="cuda") * 0.05, 128)
    got = _expert_layer(x, ids, weights, gu, dn, E)
    xq, xs = U.fp8_quantize(x)
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    tol = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for t in range(T):
        for r in range(K):
            e = int(ids[t, r])
            if e < 0:
                continue
            h, _ = _fp8_want(xq[t:t + 1], xs[t:t + 1], gu[0][e], gu[1][e])
            a = (torch.nn.functional.silu(h[:, :I]) * h[:, I:])
            y, size = _fp8_want(*U.fp8_quantize(a.to(BF16).contiguous()), dn[0][e], dn[1][e])
            wt = float(weights[t, r])
            want[t] += wt * y[0]
            # h is rounded to bf16 on the way (2^-8 of gate and of up; silu's slope is at most 1.1 and |silu| <= |gate|,
            # so a is off by at most 3.2 * 2^-8 of itself plus the rounding of a, 2^-8), and a code may then land one
            # step off, 2^-3 of the value: every term of y is off by at most 2^-3 + 5 * 2^-8 of itself.
            tol[t] += wt * size[0] * (2.0 ** -3 + 5 * 2.0 ** -8)
    off = (got.double() - want).abs()
    assert (off <= tol).all()
    assert (got.double() - want).norm() <= 0.05 * want.norm()


def test_layer_of_16_bit_weights_with_gradients():
    """Grouping, forward and both gradients in a row: the chain rule through two products, against autograd in 64 bits."""
    T, H, I, E, K = 50, 128, 96, 6, 2
    g = _gen(4)
    ids = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:K] for t in range(T)]).int().cuda()
    ids[3, 0] = -1
    off, row_token, row_of_job = U.group_rows(ids, E)
    x = _rand(g, T, H)
    w1, w2 = _rand(g, E, I, H) * 0.125, _rand(g, E, H, I) * 0.125
    xr = x[row_token]
    h = U.grouped_mm(xr, w1, off, out_dtype=F32)
    hb = h.to(BF16)
    y = U.grouped_mm(hb, w2, off, out_dtype=F32)
    dy = _rand(g, T * K, H)
    dh = U.grouped_mm_dx(dy, w2, off)
    dw2 = U.grouped_mm_dw(dy, hb, off)
    dw1 = U.grouped_mm_dw(dh, xr, off)
    n = int(off[-1])
    for e, (i, j) in _spans(off):
        xe, he, dye, dhe = (t[i:j].double() for t in (xr, hb, dy, dh))
        _close(h[i:j], xe @ w1[e].double().T, xe.abs() @ w1[e].double().abs().T, H, "h")
        _close(y[i:j], he @ w2[e].double().T, he.abs() @ w2[e].double().abs().T, I, "y")
        _close(dh[i:j], dye @ w2[e].double(), dye.abs() @ w2[e].double().abs(), H, "dh")
        _close(dw2[e], dye.T @ he, dye.abs().T @ he.abs(), j - i, "dw2")
        _close(dw1[e], dhe.T @ xe, dhe.abs().T @ xe.abs(), j - i, "dw1")
    assert n == T * K - 1


# Either side of what decides between the kernels: 1024 rows, 2^17 outputs (features in steps of 16), 4 and 8 rows an expert,
# 16-byte strides; long contractions of few tiles.
@pytest.mark.parametrize("counts,n,k", [([1024], 128, 64), ([1025], 128, 64), ([512], 256, 96), ([513], 256, 96), ([511], 241, 96),
                                        ([57], 640, 4096), ([4] * 9, 48, 160), ([5] * 9, 48, 160), ([8, 9, 0, 7], 512, 2080),
                                        ([9, 9, 0, 9], 512, 2080), ([300, 0, 3], 136, 1040), ([7, 500], 17, 1041)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_around_the_choice_of_kernel(counts, n, k, out):
    _check_all(counts, 2, 3, n, k, BF16, out, seed=n + k)
    x, xs, w, ws, off = _fp8_case(counts, 2, 3, n, k, seed=n + k)
    y = torch.full((x.shape[0], n), 5.0, dtype=out, device="cuda")
    U.fp8_grouped_mm(x, xs, w, ws, off, out=y)
    assert (y[:2] == 5).all() and (y[-3:] == 5).all()
    for e, (i, j) in _spans(off):
        want, size = _fp8_want(x[i:j], xs[i:j], w[e], ws[e])
        _close(y[i:j], want, size, k, f"expert {e}")


# Operands that begin and end at any element of an allocation's first and last words, in every direction.
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 5), (63, 65), (129, 131), (257, 64)])
def test_operands_at_the_ends_of_their_memory(shift, n, k):
    counts = [3, 0, 66]
    x, dy, w, off = _case(counts, 0, 0, n, k, BF16, seed=n * k)

    def moved(t):  # the last bytes of their storage, `shift` elements from its start
        buf = torch.full((t.numel() + shift,), float("nan"), dtype=t.dtype, device="cuda")
        buf[shift:] = t.flatten()
        return buf[shift:].view(t.shape)

    xm, dym, wm = moved(x), moved(dy), moved(w)
    for e, (i, j) in _spans(off):
        _close(U.grouped_mm(xm, wm, off, out_dtype=F32)[i:j], x[i:j].double() @ w[e].double().T,
               x[i:j].double().abs() @ w[e].double().abs().T, k, f"expert {e}")
        _close(U.grouped_mm_dw(dym, xm, off)[e], dy[i:j].double().T @ x[i:j].double(),
               dy[i:j].double().abs().T @ x[i:j].double().abs(), j - i, f"dw {e}")
        _close(U.grouped_mm_dx(dym, wm, off, out_dtype=F32)[i:j], dy[i:j].double() @ w[e].double(),
               dy[i:j].double().abs() @ w[e].double().abs(), n, f"dx {e}")


def test_operand_and_output_in_one_buffer():
    """Columns of one buffer lie beside one another and are allowed; the same memory is refused, and left as it was."""
    x, dy, w, off = _case([70, 5, 33], 0, 2, 96, 96, BF16, seed=8)
    rows = x.shape[0]

    def same(a, b):  # bit by bit: x has rows of NaN
        return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))

    buf = torch.zeros(rows, 192, dtype=BF16, device="cuda")
    buf[:, :96] = x
    want = torch.zeros_like(dy)
    U.grouped_mm(x, w, off, out=want)
    U.grouped_mm(buf[:, :96], w, off, out=buf[:, 96:])
    assert same(buf[:, :96], x) and same(buf[:, 96:], want)
    for out in (buf[:, :96], buf[:, 8:104]):
        with pytest.raises(U.UmsxError, match="overlaps"):
            U.grouped_mm(buf[:, :96], w, off, out=out)
    assert same(buf[:, :96], x) and same(buf[:, 96:], want)


def test_the_legacy_stream_by_its_number():
    x, dy, w, off = _case([20, 3], 0, 0, 64, 64, F16, seed=9)
    want = U.grouped_mm(x, w, off)
    torch.cuda.synchronize()
    got = U.grouped_mm(x, w, off, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_same_bits_twice_and_on_another_stream():
    x, dy, w, off = _case([300, 0, 41, 77], 0, 3, 256, 384, BF16, seed=6)
    xq, xs, wq, ws, _ = _fp8_case([300, 0, 41, 77], 0, 3, 256, 384, seed=6)

    def run(stream=None):
        y = torch.zeros(x.shape[0], 256, dtype=F32, device="cuda")
        z = torch.zeros_like(y)
        dx = torch.zeros(x.shape[0], 384, dtype=F32, device="cuda")
        torch.cuda.synchronize()
        return (U.grouped_mm(x, w, off, out=y, stream=stream), U.grouped_mm_dx(dy, w, off, out=dx, stream=stream),
                U.grouped_mm_dw(dy, x, off, stream=stream), U.fp8_grouped_mm(xq, xs, wq, ws, off, out=z, stream=stream))

    first = run()
    side, side2 = torch.cuda.Stream(), torch.cuda.Stream()
    a, b = run(side), run(side2)  # two calls at once
    torch.cuda.synchronize()
    for p, q, r in zip(first, a, b):
        assert torch.equal(p, q) and torch.equal(p, r)


def test_captured_and_replayed():
    """All operators in one graph, replayed on new inputs and new group sizes in the same buffers."""
    E, n, k, T, K = 6, 192, 256, 40, 2
    g = _gen(8)
    ids = torch.randint(0, E, (T, K), generator=g, device="cuda", dtype=torch.int32)
    x, w = _rand(g, T, k), _rand(g, E, n, k)
    dy = _rand(g, T * K, n)
    wq, ws = U.fp8_quantize(w, 128)

    def step():
        off, tok, job = U.group_rows(ids, E)
        xr = x[tok]
        y = U.grouped_mm(xr, w, off, out_dtype=F32)
        dx = U.grouped_mm_dx(dy, w, off)
        dw = U.grouped_mm_dw(dy, xr, off)
        xq, xs = U.fp8_quantize(xr)
        z = U.fp8_grouped_mm(xq, xs, wq, ws, off)
        return [off, tok, job, y, dx, dw, z]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2, 3):
        g2 = _gen(seed)
        ids.copy_(torch.randint(0, E if seed < 3 else 1, (T, K), generator=g2, device="cuda", dtype=torch.int32))
        x.copy_(_rand(g2, T, k))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("tokens", [400, 20000])
def test_captured_and_replayed_at_length(tokens):
    """The same for the prompt's kernels (tcgen05, clusters of sixteen)."""
    E, n, k, K = 7, 264, 128, 2
    g = _gen(18)
    ids = torch.randint(0, E, (tokens, K), generator=g, device="cuda", dtype=torch.int32)
    x, w = _rand(g, tokens, k), _rand(g, E, n, k)
    wq, ws = U.fp8_quantize(w, 128)

    def step():
        off, tok, job = U.group_rows(ids, E)
        xr = x[tok]
        y = U.grouped_mm(xr, w, off)
        dx = U.grouped_mm_dx(y, w, off)
        dw = U.grouped_mm_dw(y, xr, off)
        return [off, tok, job, y, dx, dw, U.fp8_grouped_mm(*U.fp8_quantize(xr), wq, ws, off)]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2):
        ids.copy_(torch.randint(0, E, (tokens, K), generator=_gen(seed), device="cuda", dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_two_threads_at_once():
    """Calls of two host threads on streams of their own give what they give alone."""
    import threading
    cases = [_case([200, 3, 90], 0, 0, 256, 512, BF16, seed=s) for s in (1, 2)]

    def work(c, stream=None):
        x, dy, w, off = c
        return [U.grouped_mm(x, w, off, stream=stream), U.grouped_mm_dx(dy, w, off, stream=stream),
                U.grouped_mm_dw(dy, x, off, stream=stream), *U.fp8_quantize(x, stream=stream)]

    alone = [work(c) for c in cases]
    torch.cuda.synchronize()
    got = [None, None]

    def run(i):
        s = torch.cuda.Stream()
        for _ in range(20):
            got[i] = work(cases[i], s)
        s.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, got):
        for p, q in zip(a, b):
            assert torch.equal(p.float(), q.float())


def test_given_stream_orders_new_outputs():
    """Outputs that a call makes for a given stream (a torch stream or its number) are that stream's."""
    x, dy, w, off = _case([300, 41], 0, 0, 256, 384, BF16, seed=6)
    want = U.grouped_mm(x, w, off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for s in (side, side.cuda_stream):
        y = U.grouped_mm(x, w, off, stream=s)
        z = U.grouped_mm_dx(y, w, off, stream=s)
        side.synchronize()
        assert torch.equal(y, want) and torch.equal(z, U.grouped_mm_dx(want, w, off))


@pytest.mark.parametrize("n,k", [(256, 2048), (136, 4096), (96, 8200)])
def test_long_contractions_in_fp32(n, k):
    """fp32 outputs of the tensor cores add 512 of the contraction at a time, 16 to an addition: each of the at most 32
    truncated additions of a part costs up to an ulp (2^-23 of the part's sum of magnitudes), the parts are added with
    rounding."""
    x, dy, w, off = _case([200, 60], 0, 0, n, k, BF16, seed=k)
    y, parts = U.grouped_mm(x, w, off, out_dtype=F32), -(-k // 512)
    for e, (i, j) in _spans(off):
        xe, we = x[i:j].double(), w[e].double()
        size = xe.abs() @ we.abs().T
        off_by = (y[i:j].double() - xe @ we.T).abs()
        assert (off_by <= (33 * 2.0 ** -23 + parts * 2.0 ** -24) * size).all()


def test_every_row_to_one_of_many_experts():
    """Few rows an expert on average, all of them with one: the choice of a kernel goes by the average."""
    for rows in (33, 200):
        counts = [0] * 64
        counts[37] = rows
        _check_all(counts, 0, 0, 272, 160, BF16, BF16, seed=rows)
        x, xs, w, ws, off = _fp8_case(counts, 0, 0, 272, 160, seed=rows)
        want, size = _fp8_want(x, xs, w[37], ws[37])
        _close(U.fp8_grouped_mm(x, xs, w, ws, off, out_dtype=F32), want, size, 160, "y")


@pytest.mark.parametrize("rows", [1, 17, 1024, 1025])
def test_one_expert_is_the_dense_product(rows):
    x, xs, w, ws, off = _fp8_case([rows], 0, 0, 200, 256, seed=rows)
    assert torch.equal(U.fp8_grouped_mm(x, xs, w, ws, off), U.fp8_mm(x, xs, w[0], ws[0]))


def test_status_is_clear_after_use():
    x, dy, w, off = _case([300, 41], 0, 0, 256, 384, BF16, seed=6)
    U.grouped_mm(x, w, off)
    U.products_status()


def test_launches_are_counted():
    x, dy, w, off = _case([3], 0, 0, 64, 64, BF16, seed=1)
    before = U.kernel_launches()
    U.grouped_mm(x, w, off)
    U.fp8_quantize(x)
    assert U.kernel_launches() >= before + 2


# ---- bounded waits ---------------------------------------------------------------------------------------


def _tcgen05_calls():
    """Calls that run on the tcgen05 kernels (more than 1024 rows, aligned), name -> (function, reads of its result)."""
    counts = [700, 0, 10, 413]
    x, dy, w, off = _case(counts, 0, 0, 256, 512, BF16, seed=31)
    xs16, dys16, _, off16 = _case([64, 1056], 0, 0, 256, 512, BF16, seed=32)
    xt, dyt, _, offt = _case([10, 1100], 0, 0, 256, 512, BF16, seed=33)  # the first tile's only stage ends raggedly
    xq, xs, wq, ws, offq = _fp8_case(counts, 0, 0, 256, 512, seed=34)
    return {"forward": lambda: U.grouped_mm(x, w, off), "forward in fp32": lambda: U.grouped_mm(x, w, off, out_dtype=F32),
            "dx": lambda: U.grouped_mm_dx(dy, w, off), "dw": lambda: U.grouped_mm_dw(dys16, xs16, off16),
            "dw of ragged groups": lambda: U.grouped_mm_dw(dyt, xt, offt), "e4m3": lambda: U.fp8_grouped_mm(xq, xs, wq, ws, offq)}


@pytest.mark.parametrize("call", ["forward", "forward in fp32", "dx", "dw", "dw of ragged groups", "e4m3"])
@pytest.mark.parametrize("cta", [0, 1])
def test_a_wait_that_runs_out_is_reported(call, cta):
    """A CTA's first copies never start, so that the waits behind them run out (a millisecond here): the kernel ends, the
    status says so once, and the next call gives its usual bits.  CTA 1 is the second of a pair in the 16-bit products."""
    fn = _tcgen05_calls()[call]
    want = fn()
    U.products_status()
    U.products_inject_fault(cta, wait_limit_cycles=2_000_000)
    fn()
    with pytest.raises(U.UmsxError) as e:
        U.products_status()
    assert e.value.status == U.ETIMEOUT
    U.products_status()
    assert torch.equal(fn(), want)
    U.products_status()


def test_a_fault_beyond_the_grid_injects_nothing():
    for fn in _tcgen05_calls().values():
        want = fn()
        U.products_inject_fault(1 << 20, wait_limit_cycles=200_000_000)
        assert torch.equal(fn(), want)
        U.products_status()


# ---- long contractions -----------------------------------------------------------------------------------
#
# Operands between 0.5 and 1.5, so that a partial sum grows steadily and what an addition cuts off does not average out.
# A tensor-core addition of 16 products to a sum may cut each of the products and the result off, at one and a half units in the
# last place at worst.  Over the 32 additions of a part of 512 the sum grows linearly, 16.5 times the part's own size in all:
# at most 25 units (2^-23) of it.  The parts are added with rounding, half a unit each, and the result is rounded once to its
# type.  One accumulator for the whole contraction loses about 0.3 units an addition on average.


def _grows(gen, *shape, dtype=BF16):
    return (torch.rand(shape, generator=gen, device="cuda") + 0.5).to(dtype)


def _long_close(got, want, part, parts, what):
    """want: fp64, of positive terms.  part: of the contraction in one accumulator; parts: roundings of fp32 sums."""
    half = torch.finfo(got.dtype).eps / 2
    tol = (25 * (part / 512) * 2.0 ** -23 + parts * 2.0 ** -24 + half) * want * (1 + half)
    off = (got.double() - want).abs()
    assert (off <= tol).all(), f"{what}: {float((off / want).max()):.3g} of the value off"


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_contractions_of_any_alignment(dtype):
    """The kernel for odd widths, fp32 out: 65,537 of the contraction in every direction; and the last of them in 16 bits, where an
    accumulator takes 4,096."""
    g, c = _gen(51), 65537
    off = _offsets([70])
    x, w = _grows(g, 70, c, dtype=dtype), _grows(g, 1, 65, c, dtype=dtype)
    _long_close(U.grouped_mm(x, w, off, out_dtype=F32), x.double() @ w[0].double().T, 512, 129, "y")
    dy, w = _grows(g, 70, c, dtype=dtype), _grows(g, 1, c, 65, dtype=dtype)
    _long_close(U.grouped_mm_dx(dy, w, off, out_dtype=F32), dy.double() @ w[0].double(), 512, 129, "dx")
    dy, x, off = _grows(g, c, 67, dtype=dtype), _grows(g, c, 65, dtype=dtype), _offsets([c])
    _long_close(U.grouped_mm_dw(dy, x, off)[0], dy.double().T @ x.double(), 512, 129, "dw")
    x = x * 2.0 ** -6  # the sum stays an f16
    _long_close(U.grouped_mm_dw(dy, x, off, out_dtype=dtype)[0], dy.double().T @ x.double(), 4096, 17, "dw in 16 bits")


@pytest.mark.parametrize("rows", [2, 8, 60])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_contractions_of_few_rows(rows, dtype):
    """The streaming kernel, fp32 out: eight warps share 65,536 of the contraction and add at most 256 in one accumulator."""
    g, c = _gen(52), 65536
    x, w = _grows(g, rows, c, dtype=dtype), _grows(g, 1, 48, c, dtype=dtype)
    y = U.grouped_mm(x, w, _offsets([rows]), out_dtype=F32)
    _long_close(y, x.double() @ w[0].double().T, 256, c // (8 * 128) + 8, "y")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_contractions_of_16_bit_outputs(dtype):
    """The tcgen05 kernel with 16-bit outputs: 4,096 of the contraction in one accumulator, in every direction."""
    g, c = _gen(53), 1 << 20
    dy, x, off = _grows(g, c, 64, dtype=dtype), _grows(g, c, 64, dtype=dtype) * 2.0 ** -8, _offsets([c])
    _long_close(U.grouped_mm_dw(dy, x, off, out_dtype=dtype)[0], dy.double().T @ x.double(), 4096, c // 4096, "dw")
    c, off = 1 << 17, _offsets([1100])
    x, w = _grows(g, 1100, c, dtype=dtype) * 2.0 ** -6, _grows(g, 1, 128, c, dtype=dtype)
    _long_close(U.grouped_mm(x, w, off), x.double() @ w[0].double().T, 4096, c // 4096, "y")
    dy, w = _grows(g, 1100, c, dtype=dtype) * 2.0 ** -6, _grows(g, 1, c, 128, dtype=dtype)
    _long_close(U.grouped_mm_dx(dy, w, off), dy.double() @ w[0].double(), 4096, c // 4096, "dx")


def test_a_ragged_end_far_ahead_is_waited_for():
    """A weight gradient whose groups end at multiples of 16 rows but for the last: the warp that zeroes a ragged end waits for it
    from the start, for several times the limit of 0.1 ms (200,000 cycles), to which no other wait comes near."""
    counts = [64] * 1023 + [30]
    x, dy, _, off = _case(counts, 0, 0, 1024, 1024, BF16, seed=41)
    want = U.grouped_mm_dw(dy, x, off)
    U.products_status()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    U.products_inject_fault(1 << 20, wait_limit_cycles=200_000)
    start.record()
    got = U.grouped_mm_dw(dy, x, off)
    end.record()
    U.products_status()
    assert torch.equal(got, want)
    assert start.elapsed_time(end) > 0.3, "the call was too short to show anything"


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_contractions_in_fp32_on_tcgen05(dtype):
    """The tcgen05 kernel with fp32 outputs (more than 1024 rows, or a gradient): 512 of the contraction in one accumulator."""
    g, c = _gen(54), 1 << 16
    off = _offsets([700, 400])
    x, w = _grows(g, 1100, c, dtype=dtype), _grows(g, 2, 128, c, dtype=dtype)
    y = U.grouped_mm(x, w, off, out_dtype=F32)
    dy, v = _grows(g, 1100, c, dtype=dtype), _grows(g, 2, c, 128, dtype=dtype)
    dx = U.grouped_mm_dx(dy, v, off, out_dtype=F32)
    for e, (i, j) in _spans(off):
        _long_close(y[i:j], x[i:j].double() @ w[e].double().T, 512, c // 512, "y")
        _long_close(dx[i:j], dy[i:j].double() @ v[e].double(), 512, c // 512, "dx")
    dy, x, off = _grows(g, 2 * c, 72, dtype=dtype), _grows(g, 2 * c, 136, dtype=dtype), _offsets([c - 37, c + 37])
    dw = U.grouped_mm_dw(dy, x, off)
    for e, (i, j) in _spans(off):
        _long_close(dw[e], dy[i:j].double().T @ x[i:j].double(), 512, c // 512 + 1, "dw")


# ---- the prompt's kernels: more than 1024 rows, aligned ------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("pad", [0, 8])
def test_types_and_strides_of_prompts(dtype, out, pad):
    _check_all([640, 0, 5, 500], 1, 2, 192, 320, dtype, out, seed=17, pad=pad)


def test_non_finite_values_stay_in_their_rows_of_prompts():
    """One row of a tile of 256 with a NaN or an infinity, and an expert of NaN between two others, in all three directions."""
    counts = [600, 700, 7]
    x, dy, w, off = _case(counts, 0, 0, 128, 256, BF16, seed=12)
    clean, clean_dx, clean_dw = U.grouped_mm(x, w, off), U.grouped_mm_dx(dy, w, off), U.grouped_mm_dw(dy, x, off)
    x2, dy2 = x.clone(), dy.clone()
    x2[605, 3], x2[1299, 0] = float("nan"), float("inf")
    dy2[605, 5], dy2[1299, 0] = float("nan"), float("inf")
    y, dx = U.grouped_mm(x2, w, off), U.grouped_mm_dx(dy2, w, off)
    rows = [r for r in range(x.shape[0]) if r not in (605, 1299)]
    for got, want in ((y, clean), (dx, clean_dx)):
        assert torch.equal(got[rows], want[rows]) and torch.isnan(got[605]).all() and not torch.isfinite(got[1299]).any()
    dw = U.grouped_mm_dw(dy, x2, off)
    assert torch.equal(dw[0], clean_dw[0]) and torch.equal(dw[2], clean_dw[2])
    assert torch.isnan(dw[1][:, 3]).all() and torch.equal(dw[1][:, 4:], clean_dw[1][:, 4:])
    w2 = w.clone()
    w2[1] = float("nan")
    for got, want in ((U.grouped_mm(x, w2, off), clean), (U.grouped_mm_dx(dy, w2, off), clean_dx)):
        assert torch.equal(got[:600], want[:600]) and torch.equal(got[1300:], want[1300:]) and torch.isnan(got[600:1300]).all()


def test_fp8_non_finite_codes_stay_in_their_rows_of_prompts():
    x, xs, w, ws, off = _fp8_case([600, 700, 7], 0, 0, 128, 256, seed=12)
    clean = U.fp8_grouped_mm(x, xs, w, ws, off)
    bad = x.view(torch.uint8).clone()
    bad[605, 3], bad[1299, 200] = 0x7F, 0xFF
    y = U.fp8_grouped_mm(bad.view(E4M3), xs, w, ws, off)
    rows = [r for r in range(x.shape[0]) if r not in (605, 1299)]
    assert torch.equal(y[rows], clean[rows]) and torch.isnan(y[605]).all() and torch.isnan(y[1299]).all()
    bad = w.view(torch.uint8).clone()
    bad[1] = 0x7F
    y = U.fp8_grouped_mm(x, xs, bad.view(E4M3), ws, off)
    assert torch.equal(y[:600], clean[:600]) and torch.equal(y[1300:], clean[1300:]) and torch.isnan(y[600:1300]).all()


def test_same_bits_twice_and_on_other_streams_of_prompts():
    counts = [900, 0, 341, 77]
    x, dy, w, off = _case(counts, 0, 3, 256, 1024, BF16, seed=16)
    xq, xs, wq, ws, _ = _fp8_case(counts, 0, 3, 256, 1024, seed=16)

    def run(stream=None):
        y = torch.zeros(x.shape[0], 256, dtype=F32, device="cuda")
        z = torch.zeros_like(y)
        torch.cuda.synchronize()
        return (U.grouped_mm(x, w, off, out=y, stream=stream), U.fp8_grouped_mm(xq, xs, wq, ws, off, out=z, stream=stream))

    first = run()
    side, side2 = torch.cuda.Stream(), torch.cuda.Stream()
    a, b = run(side), run(side2)  # two calls at once
    torch.cuda.synchronize()
    for p, q, r in zip(first, a, b):
        assert torch.equal(p, q) and torch.equal(p, r)


def test_given_stream_orders_new_outputs_of_prompts():
    x, dy, w, off = _case([700, 441], 0, 0, 256, 384, BF16, seed=26)
    want = U.grouped_mm(x, w, off)
    want_dx = U.grouped_mm_dx(want, w, off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for s in (side, side.cuda_stream):
        y = U.grouped_mm(x, w, off, stream=s)
        z = U.grouped_mm_dx(y, w, off, stream=s)
        side.synchronize()
        assert torch.equal(y, want) and torch.equal(z, want_dx)


def test_status_is_clear_after_prompts():
    for fn in _tcgen05_calls().values():
        fn()
        U.products_status()


def test_scales_of_any_nested_layout():
    """Blocks of columns first, rows first, matrices innermost, with gaps; a broadcast one is refused and nothing is written."""
    x = _rand(_gen(61), 3, 20, 300)
    q0, s0 = U.fp8_quantize(x)
    for order in ((0, 1, 2), (0, 2, 1), (1, 2, 0), (2, 1, 0)):
        shape = [s0.shape[i] for i in order]
        store = torch.zeros([2 * n for n in shape], device="cuda")
        view = store[:shape[0], :shape[1], :shape[2]].permute([order.index(i) for i in range(3)])
        q, s = U.fp8_quantize(x, scales=view)
        assert torch.equal(s, s0) and torch.equal(q.float(), q0.float())
    shared = torch.zeros(1, 1, 1, device="cuda")
    with pytest.raises(U.UmsxError, match="one address"):
        U.fp8_quantize(x, scales=shared.expand(3, 20, 3))
    torch.cuda.synchronize()
    assert not shared.any()
    U.fp8_quantize(x[0, :1, :100], scales=torch.zeros(1, device="cuda").expand(1, 1))  # one block: no stride counts


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_tiny_blocks(dtype, block_rows):
    """Block maxima from 2^-110 to 2^-70, on both sides of where the quotient's residual stops being exact, values down to
    2^-22 of them: scales and codes as the formula gives them with one rounding each."""
    g = _gen(71)
    top = torch.arange(-110, -69, device="cuda").repeat_interleave(128).double()
    x = torch.exp2(top[:, None] - 22 * torch.rand(top.numel(), 128, generator=g, device="cuda").double())
    x = (x * torch.where(torch.rand(x.shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)).to(dtype)
    q, s = U.fp8_quantize(x, block_rows)
    amax = x.double().abs().view(-1, block_rows, 128).amax((1, 2))
    want = torch.clamp(amax / 448.0, min=2.0 ** -126).float()
    assert torch.equal(s[:, 0], want)
    quotient = (x.double() / want.double().repeat_interleave(block_rows)[:, None]).float()
    assert torch.equal(q.float(), _round_e4m3(quotient.double()).float())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("top", [1.0, 2.0 ** -14, 0.0])
def test_quantize_keeps_the_sign_of_zero(dtype, block_rows, top):
    """x / scale of a zero has the zero's sign, and so has a quotient that rounds to zero; in a block of zeros too."""
    x = torch.zeros(128, 256, device="cuda", dtype=dtype)
    x[:, 1::2] = -0.0
    x[:, 0] = x[:, 128] = top
    x[:, 2], x[:, 3] = top * 2.0 ** -10 / 448, -top * 2.0 ** -11 / 448  # half the smallest code, but for x's own rounding; less
    q, s = U.fp8_quantize(x, block_rows)
    value = _round_e4m3((x.double().abs() / max(top / 448, 2.0 ** -126)).float().double()).to(E4M3).view(torch.uint8)
    sign = torch.where(torch.signbit(x.float()), 0x80, 0).to(torch.uint8)
    assert torch.equal(q.view(torch.uint8), value | sign)


# ---- autograd --------------------------------------------------------------------------------------------


def test_a_gradient_that_would_be_lost_is_warned_about():
    import warnings
    x, dy, w, off = _case([3, 4], 0, 0, 64, 32, BF16, seed=1)
    xq, xs, wq, ws, _ = _fp8_case([3, 4], 0, 0, 64, 32, seed=1)
    need = [t.clone().requires_grad_() for t in (x, w, dy, xs)]
    calls = [lambda: U.grouped_mm(need[0], w, off), lambda: U.grouped_mm(x, need[1], off), lambda: U.grouped_mm_dx(need[2], w, off),
             lambda: U.grouped_mm_dw(need[2], x, off), lambda: U.fp8_quantize(need[0])[0],
             lambda: U.fp8_grouped_mm(xq, need[3], wq, ws, off), lambda: U.fp8_mm(xq, need[3], wq[0], ws[0])]
    for call in calls:
        with pytest.warns(UserWarning, match="autograd"):
            got = call()
        assert not got.requires_grad
        with warnings.catch_warnings(), torch.no_grad():
            warnings.simplefilter("error")
            assert torch.equal(call().float(), got.float())
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        U.grouped_mm(x, w, off)


class _GroupedMM(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, off):
        ctx.save_for_backward(x, w, off)
        return U.grouped_mm(x, w, off, out=x.new_zeros(x.shape[0], w.shape[1]))

    @staticmethod
    def backward(ctx, dy):
        x, w, off = ctx.saved_tensors
        dy = dy.contiguous()
        return U.grouped_mm_dx(dy, w, off, out=torch.zeros_like(x)), U.grouped_mm_dw(dy, x, off, out_dtype=w.dtype), None


def test_products_joined_in_an_autograd_function():
    import warnings
    x, dy, w, off = _case([30, 0, 41], 0, 0, 64, 96, BF16, seed=81)
    x = torch.cat([x, _rand(_gen(82), 5, 96)])  # five rows of no group
    dy = torch.cat([dy, _rand(_gen(83), 5, 64)])
    x.requires_grad_(), w.requires_grad_()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        y = _GroupedMM.apply(x, w, off)
        y.backward(dy)
    assert not y[71:].any() and not x.grad[71:].any()
    x, w, dx, dw = x.detach().double(), w.detach().double(), x.grad, w.grad
    for e, (i, j) in _spans(off):
        dye = dy[i:j].double()
        _close(y[i:j].detach(), x[i:j] @ w[e].T, x[i:j].abs() @ w[e].abs().T, 96, "y")
        _close(dx[i:j], dye @ w[e], dye.abs() @ w[e].abs(), 64, "dx")
        _close(dw[e], dye.T @ x[i:j], dye.abs().T @ x[i:j].abs(), j - i, "dw")


def test_an_error_is_reported_by_its_own_call_only():
    """A call that fails in the CUDA runtime (a status query, which synchronises, on a stream that is being captured) leaves
    nothing that a later, sound one reports."""
    rt = pytest.importorskip("cuda.bindings.runtime")
    x, dy, w, off = _case([3, 4], 0, 0, 64, 32, BF16, seed=1)
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    xb, rw = _rand(_gen(2), 4, 64), torch.zeros(8, 64, device="cuda")
    calls = [lambda: U.grouped_mm(x, w, off), lambda: U.grouped_mm_dx(dy, w, off), lambda: U.fp8_quantize(x),
             lambda: U.group_rows(ids, 4), lambda: U.route_static(xb, rw, None, 8, 2, U.ROUTE_SOFTMAX_TOPK_NORM)]
    for call in calls:
        call()
        side = torch.cuda.Stream()
        assert int(rt.cudaStreamBeginCapture(side.cuda_stream, rt.cudaStreamCaptureMode.cudaStreamCaptureModeThreadLocal)[0]) == 0
        with pytest.raises(U.UmsxError) as e:
            U.products_status(side)
        assert e.value.status == U.EDEVICE
        rt.cudaStreamEndCapture(side.cuda_stream)  # the capture is void
        call()
    torch.cuda.synchronize()
    U.products_status()


# ---- odd widths in padded buffers -------------------------------------------------------------------------


@pytest.mark.parametrize("counts", [[640, 0, 5, 500], [3, 0, 7, 1], [70, 9]])
@pytest.mark.parametrize("out", [F32, F16])
def test_odd_widths_with_aligned_rows(counts, out):
    """Rows that start at multiples of 16 bytes but end between them: the tensor cores' kernels take them, and NaN in the padding
    reaches nothing.  Outputs are columns of a wider buffer too, whose padding stays as it was."""
    for n, k in ((193, 321), (33, 65), (17, 129)):
        x, dy, w, off = _case(counts, 1, 2, n, k, F16, seed=n, pad=7)  # rows of n + 7 and k + 7
        w._base[:, :, k:] = float("nan")
        rows = x.shape[0]
        stores = [torch.full(s, 9.0, dtype=out, device="cuda") for s in ((rows, n + 7), (rows, k + 7), (len(counts), n, k + 7))]
        y, dx, dw = stores[0][:, :n], stores[1][:, :k], stores[2][:, :, :k]
        U.grouped_mm(x, w, off, out=y)
        U.grouped_mm_dx(dy, w, off, out=dx)
        U.grouped_mm_dw(dy, x, off, out=dw)
        assert (stores[0][:, n:] == 9).all() and (stores[1][:, k:] == 9).all() and (stores[2][:, :, k:] == 9).all()
        a, b = 1, 1 + sum(counts)
        for t in stores[:2]:
            assert (t[:a] == 9).all() and (t[b:] == 9).all()
        for e, (i, j) in _spans(off):
            xe, dye, we = x[i:j].double(), dy[i:j].double(), w[e].double()
            _close(y[i:j], xe @ we.T, xe.abs() @ we.abs().T, k, "y")
            _close(dx[i:j], dye @ we, dye.abs() @ we.abs(), n, "dx")
            _close(dw[e], dye.T @ xe, dye.abs().T @ xe.abs(), j - i, "dw")


@pytest.mark.parametrize("counts", [[640, 0, 5, 500], [3, 0, 7, 1], [70, 9]])
@pytest.mark.parametrize("out", [F32, BF16])
def test_fp8_odd_widths_with_aligned_rows(counts, out):
    for n, k in ((193, 321), (130, 129), (17, 145)):
        x, xs, w, ws, off = _fp8_case(counts, 1, 2, n, k, seed=n, pad=-k % 16)
        torch.as_strided(w.view(torch.uint8), (len(counts), n, k + -k % 16), w.stride())[:, :, k:] = 0x7F  # NaN
        store = torch.full((x.shape[0], n + 7), 9.0, dtype=out, device="cuda")
        U.fp8_grouped_mm(x, xs, w, ws, off, out=store[:, :n])
        assert (store[:, n:] == 9).all() and (store[:1] == 9).all() and (store[-2:] == 9).all()
        for e, (i, j) in _spans(off):
            want, size = _fp8_want(x[i:j], xs[i:j], w[e], ws[e])
            _close(store[i:j, :n], want, size, k, f"expert {e}")


def test_quantize_takes_one_matrix_for_all():
    """A matrix that is broadcast over the first dimension is read in place."""
    x = _rand(_gen(91), 1, 30, 200)
    q0, s0 = U.fp8_quantize(x[0], 128)
    q, s = U.fp8_quantize(x.expand(3, 30, 200), 128)
    for i in range(3):
        assert torch.equal(q[i].float(), q0.float()) and torch.equal(s[i], s0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_ties_go_to_the_even_code(dtype, block_rows):
    """Every midpoint of two neighbouring e4m3 values, beside a 448 that makes the scale one, and the same times 2^-5."""
    value = torch.arange(127, dtype=torch.uint8, device="cuda").view(E4M3).float()
    x = torch.zeros(4, 128, device="cuda")
    x[:, 0] = 448.0
    x[0, 1:127] = (value[:-1] + value[1:]) / 2
    x[1, 1:127] = -x[0, 1:127]
    x[2:] = x[:2] * 2.0 ** -5
    code = torch.arange(126, dtype=torch.uint8, device="cuda")
    even = code + (code & 1)
    for rows in ((0, 2), (2, 4)):
        xr = x[rows[0]:rows[1]].to(dtype)
        assert torch.equal(xr.float(), x[rows[0]:rows[1]])  # exact in every type
        q, s = U.fp8_quantize(xr, block_rows)
        assert (s == xr[0, 0].float() / 448).all()
        q = q.view(torch.uint8)
        assert torch.equal(q[0, 1:127], even) and torch.equal(q[1, 1:127], even | 0x80)


@pytest.mark.parametrize("rows,n,k,pad", [(1100, 128, 1 << 16, 0), (8, 128, 1 << 16, 0), (60, 128, 1 << 16, 0), (70, 65, (1 << 16) + 1, 2)])
def test_long_contractions_of_e4m3(rows, n, k, pad):
    """e4m3 in fp32 on the tcgen05 kernel, the streaming one (one and two tiles of eight rows) and that for any alignment: a block
    of 128 in one accumulator, then a product of two scales and one multiply-add for each block, each rounded once."""
    g = _gen(95)
    x = torch.empty(rows, k + pad, dtype=torch.uint8, device="cuda")[:, :k].view(E4M3)
    x.copy_((torch.rand(rows, k, generator=g, device="cuda") + 0.5).to(E4M3))
    w = torch.empty(n, k + pad, dtype=torch.uint8, device="cuda")[:, :k].view(E4M3)
    w.copy_((torch.rand(n, k, generator=g, device="cuda") + 0.5).to(E4M3))
    xs, ws = _grows(g, _blocks(k), rows, dtype=F32).t(), _grows(g, _blocks(n), _blocks(k), dtype=F32)
    want, _ = _fp8_want(x, xs, w, ws)
    _long_close(U.fp8_mm(x, xs, w, ws, out_dtype=F32), want, 128, _blocks(k) + 8 + 1, "y")
