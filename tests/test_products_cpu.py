"""Refusals of the products over caller-owned weights, before any device call (CPU only)."""
import ctypes

import numpy as np
import pytest

from tests.helpers import U

torch = pytest.importorskip("torch")

# An address that no check dereferences on the host: every call below is refused before a launch.
P = ctypes.c_void_p(256)
NULL = None


def _mm(**over):
    a = dict(x=P, ldx=64, w=P, ldw=64, w_stride=64 * 32, offsets=P, experts=4, rows=10, n=32, k=64, dtype=U.DTYPE_BF16,
             out=P, ldo=32, out_dtype=U.DTYPE_F32, stream=NULL)
    a.update(over)
    return U.lib().umsx_grouped_mm(*a.values())


def _dx(**over):
    a = dict(dy=P, lddy=32, w=P, ldw=64, w_stride=64 * 32, offsets=P, experts=4, rows=10, n=32, k=64, dtype=U.DTYPE_F16,
             dx=P, lddx=64, out_dtype=U.DTYPE_F16, stream=NULL)
    a.update(over)
    return U.lib().umsx_grouped_mm_dx(*a.values())


def _dw(**over):
    a = dict(dy=P, lddy=32, x=P, ldx=64, offsets=P, experts=4, rows=10, n=32, k=64, dtype=U.DTYPE_BF16, dw=P, lddw=64,
             dw_stride=64 * 32, out_dtype=U.DTYPE_F32, stream=NULL)
    a.update(over)
    return U.lib().umsx_grouped_mm_dw(*a.values())


def _fp8(**over):
    a = dict(x=P, ldx=64, xs=P, xs_row=1, xs_blk=10, w=P, ldw=64, w_stride=64 * 32, ws=P, ws_row=1, ws_blk=1, ws_stride=1,
             offsets=P, experts=4, rows=10, n=32, k=64, out=P, ldo=32, out_dtype=U.DTYPE_BF16, stream=NULL)
    a.update(over)
    return U.lib().umsx_fp8_grouped_mm(*a.values())


def _quant(**over):
    a = dict(x=P, ldx=64, x_stride=640, x_dtype=U.DTYPE_BF16, matrices=2, rows=10, cols=64, block_rows=1, q=P, ldq=64,
             q_stride=640, scales=P, s_row=1, s_blk=10, s_stride=10, stream=NULL)
    a.update(over)
    return U.lib().umsx_fp8_quantize(*a.values())


def _group(**over):
    a = dict(ids=P, tokens=4, top_k=2, experts=8, offsets=P, row_token=P, row_of_job=P, stream=NULL)
    a.update(over)
    return U.lib().umsx_group_rows(*a.values())


COMMON = [dict(experts=0), dict(experts=1025), dict(rows=-1), dict(rows=0x7fffffff), dict(n=0), dict(k=0), dict(k=1 << 25),
          dict(n=1 << 25), dict(out_dtype=U.DTYPE_E4M3), dict(out_dtype=-1)]


@pytest.mark.parametrize("call,over", [(c, o) for c in (_mm, _dx, _dw, _fp8) for o in COMMON] + [
    (_mm, dict(dtype=U.DTYPE_F32)), (_mm, dict(dtype=U.DTYPE_E4M3)), (_mm, dict(ldx=63)), (_mm, dict(ldw=63)),
    (_mm, dict(ldo=31)), (_mm, dict(w_stride=64 * 32 - 1)), (_mm, dict(x=NULL)), (_mm, dict(w=NULL)),
    (_mm, dict(offsets=NULL)), (_mm, dict(out=NULL)),
    (_dx, dict(dtype=U.DTYPE_F32)), (_dx, dict(lddy=31)), (_dx, dict(lddx=63)), (_dx, dict(dy=NULL)), (_dx, dict(w=NULL)),
    (_dx, dict(offsets=NULL)), (_dx, dict(dx=NULL)), (_dx, dict(w_stride=0)),
    (_dw, dict(dtype=9)), (_dw, dict(lddy=31)), (_dw, dict(ldx=63)), (_dw, dict(lddw=63)), (_dw, dict(dw_stride=5)),
    (_dw, dict(dy=NULL)), (_dw, dict(x=NULL)), (_dw, dict(offsets=NULL)), (_dw, dict(dw=NULL)),
    (_fp8, dict(ldx=63)), (_fp8, dict(xs_row=-1)), (_fp8, dict(ws_blk=-1)), (_fp8, dict(offsets=NULL)),
    (_fp8, dict(xs=NULL)), (_fp8, dict(ws=NULL)), (_fp8, dict(x=NULL)), (_fp8, dict(w=NULL)), (_fp8, dict(out=NULL)),
    (_fp8, dict(w_stride=7)),
    (_quant, dict(x_dtype=U.DTYPE_E4M3)), (_quant, dict(block_rows=64)), (_quant, dict(block_rows=0)),
    (_quant, dict(cols=0)), (_quant, dict(rows=-1)), (_quant, dict(matrices=-1)), (_quant, dict(ldx=63)),
    (_quant, dict(ldq=63)), (_quant, dict(q_stride=100)), (_quant, dict(s_row=-1)), (_quant, dict(x=NULL)),
    (_quant, dict(q=NULL)), (_quant, dict(scales=NULL)),
    (_group, dict(tokens=-1)), (_group, dict(top_k=0)), (_group, dict(experts=0)), (_group, dict(experts=1025)),
    (_group, dict(tokens=1 << 30, top_k=2)), (_group, dict(ids=NULL)), (_group, dict(offsets=NULL)),
    (_group, dict(row_token=NULL)), (_group, dict(row_of_job=NULL)),
])
def test_entry_points_refuse_bad_arguments(call, over):
    assert call(**over) == U.EINVAL
    assert U.lib().umsx_last_error()


def test_no_rows_is_no_work():
    """Without rows there is nothing to write, and no device is needed to say so."""
    assert _mm(rows=0, x=NULL, out=NULL) == U.OK
    assert _dx(rows=0, dy=NULL, dx=NULL) == U.OK
    assert _fp8(rows=0, x=NULL, xs=NULL, out=NULL) == U.OK
    assert _quant(rows=0, x=NULL, q=NULL, scales=NULL) == U.OK
    assert _quant(matrices=0) == U.OK


def test_python_refuses_host_tensors():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(2, 32, 64, dtype=torch.bfloat16)
    off = torch.tensor([0, 2, 4], dtype=torch.int32)
    f8 = torch.zeros(4, 64, dtype=torch.float8_e4m3fn)
    for call in (lambda: U.grouped_mm(x, w, off), lambda: U.grouped_mm_dx(x, w, off), lambda: U.grouped_mm_dw(x, x, off),
                 lambda: U.fp8_quantize(x), lambda: U.fp8_mm(f8, x, f8, x), lambda: U.group_rows(off[None], 4)):
        with pytest.raises(U.UmsxError) as e:
            call()
        assert e.value.status == U.EINVAL and "CUDA" in str(e.value)


def test_e4m3_rounding_rule():
    """The quantiser's definition in numpy on the whole e4m3 grid: every representable value keeps itself, and
    halfway points go to the even code (the rule that the GPU tests hold the kernel to)."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    grid = np.unique(codes[np.isfinite(codes)])
    assert grid.max() == 448.0 and len(grid) == 253
    mid = (grid[:-1] + grid[1:]) / 2
    near = torch.from_numpy(mid.astype(np.float32)).to(torch.float8_e4m3fn).float().numpy()
    assert np.all((near == grid[:-1]) | (near == grid[1:]))


def _at(byte):
    return ctypes.c_void_p(byte)


BASE = 1 << 20
# x [10][64], w [4][32][64], dy [10][32] and their results far from one another; what the overlapping calls move.
FAR = {_mm: dict(x=_at(BASE), w=_at(2 * BASE), offsets=_at(3 * BASE), out=_at(4 * BASE)),
       _dx: dict(dy=_at(BASE), w=_at(2 * BASE), offsets=_at(3 * BASE), dx=_at(4 * BASE)),
       _dw: dict(dy=_at(BASE), x=_at(2 * BASE), offsets=_at(3 * BASE), dw=_at(4 * BASE)),
       _fp8: dict(x=_at(BASE), xs=_at(2 * BASE), w=_at(3 * BASE), ws=_at(4 * BASE), offsets=_at(5 * BASE), out=_at(6 * BASE)),
       _quant: dict(x=_at(BASE), q=_at(2 * BASE), scales=_at(3 * BASE)),
       _group: dict(ids=_at(BASE), offsets=_at(2 * BASE), row_token=_at(3 * BASE), row_of_job=_at(4 * BASE))}


@pytest.mark.parametrize("call,over", [
    (_mm, dict(out=_at(BASE))), (_mm, dict(out=_at(BASE + 10 * 64 * 2 - 2))), (_mm, dict(out=_at(2 * BASE + 4 * 32 * 64 * 2 - 2))),
    (_mm, dict(out=_at(BASE - 10 * 32 * 4 + 4))), (_mm, dict(out=_at(3 * BASE + 16))),
    (_mm, dict(ldx=96, out=_at(BASE + 126), ldo=96, out_dtype=U.DTYPE_BF16)),  # columns 63.. beside columns ..63
    (_mm, dict(ldx=96, out=_at(BASE + 128), ldo=48)),                          # equal strides in bytes, the rows are 128 wide
    (_mm, dict(ldx=128, out=_at(BASE + 128), ldo=100, out_dtype=U.DTYPE_BF16)),
    (_dx, dict(dx=_at(BASE))), (_dx, dict(dx=_at(2 * BASE + 64))), (_dx, dict(dx=_at(3 * BASE))),
    (_dw, dict(dw=_at(BASE))), (_dw, dict(dw=_at(2 * BASE + 8))), (_dw, dict(dw=_at(3 * BASE + 4))),
    (_fp8, dict(out=_at(BASE + 639))), (_fp8, dict(out=_at(2 * BASE))), (_fp8, dict(out=_at(3 * BASE))),
    (_fp8, dict(out=_at(4 * BASE))), (_fp8, dict(out=_at(5 * BASE))),
    (_quant, dict(q=_at(BASE))), (_quant, dict(scales=_at(BASE + 4))), (_quant, dict(scales=_at(2 * BASE + 4))),
    (_group, dict(row_of_job=_at(BASE))), (_group, dict(row_token=_at(BASE + 28))), (_group, dict(offsets=_at(BASE))),
    (_group, dict(row_token=_at(4 * BASE))), (_group, dict(row_of_job=_at(2 * BASE + 4)))])
def test_overlapping_outputs_are_refused(call, over):
    assert call(**{**FAR[call], **over}) == U.EINVAL
    assert b"overlaps" in U.lib().umsx_last_error()


@pytest.mark.parametrize("call,over", [
    (_mm, dict(x=_at(BASE + 1))), (_mm, dict(w=_at(2 * BASE + 1))), (_mm, dict(out=_at(4 * BASE + 2))),
    (_mm, dict(offsets=_at(3 * BASE + 2))), (_dx, dict(dy=_at(BASE + 1))), (_dx, dict(dx=_at(4 * BASE + 1))),
    (_dw, dict(x=_at(2 * BASE + 1))), (_dw, dict(dw=_at(4 * BASE + 2))), (_fp8, dict(xs=_at(2 * BASE + 2))),
    (_fp8, dict(ws=_at(4 * BASE + 1))), (_fp8, dict(out=_at(6 * BASE + 1))), (_quant, dict(x=_at(BASE + 1))),
    (_quant, dict(scales=_at(3 * BASE + 2))), (_group, dict(ids=_at(BASE + 2))), (_group, dict(row_token=_at(3 * BASE + 1)))])
def test_buffers_between_elements_are_refused(call, over):
    assert call(**{**FAR[call], **over}) == U.EINVAL
    assert b"aligned" in U.lib().umsx_last_error()


@pytest.mark.parametrize("cta,limit", [(-1, 1000), (0, 0), (0, -5), (0, 2_000_000_001)])
def test_bad_fault_injections_are_refused(cta, limit):
    assert U.lib().umsx_products_inject_fault(cta, limit) == U.EINVAL


@pytest.mark.parametrize("call", [_mm, _dx, _dw, _fp8])
@pytest.mark.parametrize("rows", [2 ** 31 - 511, 2 ** 31 - 256, 2 ** 31 - 16, 2 ** 32])
def test_rows_that_the_index_arithmetic_does_not_hold_are_refused(call, rows):
    """A row index plus a tile of 256 rows, or a step of 128 of the contraction, has to fit into 32 bits."""
    assert call(rows=rows) == U.EINVAL
    assert b"rows must be" in U.lib().umsx_last_error()


def test_e4m3_ties_go_to_the_even_code():
    """Halfway between two neighbours of the grid the code with an even last bit is taken, on either side of zero."""
    codes = torch.arange(256, dtype=torch.uint8)
    value = codes.view(torch.float8_e4m3fn).float().numpy()
    for sign in (0, 0x80):
        for c in range(126):  # 0x7F is NaN
            mid = np.float32((value[sign + c] + value[sign + c + 1]) / 2)
            got = int(torch.tensor([mid]).to(torch.float8_e4m3fn).view(torch.uint8)[0])
            assert got == sign + c + (c & 1), (sign, c)


@pytest.mark.parametrize("over", [dict(s_row=0), dict(s_row=1, s_blk=9, cols=200, ldx=200, ldq=200, x_stride=2000, q_stride=2000),
                                  dict(s_stride=0), dict(s_stride=9), dict(s_row=2, s_stride=18), dict(block_rows=128, s_stride=0),
                                  dict(s_row=0, s_blk=0, s_stride=0, rows=1, matrices=1, cols=129, ldx=129, ldq=129)])
def test_scales_that_share_an_address_are_refused(over):
    """matrices 2 x 10 rows x 64 columns unless given otherwise: each block's scale needs an address of its own."""
    assert _quant(**{**FAR[_quant], **over}) == U.EINVAL
    assert b"one address" in U.lib().umsx_last_error()
