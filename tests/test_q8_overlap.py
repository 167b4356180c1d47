"""Outputs of the calls on 8-bit rows that share bytes with an input, or with one another: refused on the host, before
anything is launched and before any pointer is read; neighbours that share none are not (no GPU needed)."""
import pytest

from test_q8_args import AT, FAR, INVALID, dequantize, linear, quantize, rmsnorm

# the calls' spans: 4 rows of 64, pitch 64.  quantize: x at AT (512 bytes), codes at FAR (256), scale at 2 FAR (16);
# rmsnorm: x at AT (1,024), res at 2 AT (512), w at 3 AT (256), sum at 4 AT (1,024), codes at FAR, scale at 2 FAR;
# dequantize: codes at AT, scale at 2 AT, out at FAR (512)
MEET = [
    (quantize, [dict(scale=AT), dict(scale=AT + 508), dict(scale=AT - 12), dict(scale=FAR), dict(scale=FAR + 252),
                dict(codes=AT + 511), dict(codes=AT - 255)]),
    (rmsnorm, [dict(scale=AT), dict(scale=AT + 1020), dict(scale=2 * AT), dict(scale=2 * AT + 508), dict(scale=3 * AT),
               dict(scale=3 * AT + 252), dict(scale=3 * AT - 12), dict(scale=4 * AT), dict(scale=4 * AT + 1020),
               dict(scale=FAR + 4), dict(codes=3 * AT), dict(codes=3 * AT + 255), dict(codes=3 * AT - 255),
               dict(sum=3 * AT), dict(sum=3 * AT + 252), dict(sum=3 * AT - 1020), dict(sum=3 * AT - 252, lds=128),
               dict(w=4 * AT + 600), dict(res=None, scale=AT + 4), dict(res=None, sum=3 * AT + 4)]),
    (dequantize, [dict(out=2 * AT), dict(out=2 * AT + 14), dict(out=2 * AT - 510)]),
]


@pytest.mark.parametrize("call,over", [(c, o) for c, all_ in MEET for o in all_])
def test_shared_bytes_are_refused(call, over):
    assert call(**over) == INVALID


# What shares no byte passes these checks: each of the calls is refused by a check behind them (a launch of more
# workgroups than there may be), so none reaches the GPU.
ROWS, BIG = 2 ** 34, 2 ** 40
NEAR = [
    (quantize, dict(M=ROWS, codes=BIG * 8, scale=BIG * 16)),
    (rmsnorm, dict(M=ROWS, x=BIG * 8, res=BIG * 16, sum=BIG * 32, codes=BIG * 64, scale=BIG * 72, w=BIG * 80)),
    # the weight between two of the sum's rows, and the sum over x
    (rmsnorm, dict(M=ROWS, x=BIG * 8, ldx=256, res=BIG * 128, sum=BIG * 8, lds=256, codes=BIG * 64, scale=BIG * 72,
                   w=BIG * 8 + 256)),
    (rmsnorm, dict(M=ROWS, x=BIG * 8, ldx=256, res=BIG * 128, sum=BIG * 8, lds=256, codes=BIG * 64, scale=BIG * 72,
                   w=BIG * 8 + 768)),
    (dequantize, dict(M=ROWS, K=2000, ldc=2000, ldo=2000, codes=BIG, scale=BIG * 128, out=BIG * 256)),
]


@pytest.mark.parametrize("call,over", NEAR)
def test_neighbours_are_not(call, over):
    from versenext_amd import _lib
    assert call(**over) == _lib.VNX_ERR_UNSUPPORTED


def test_weight_across_a_row_of_the_sum():
    over = dict(M=ROWS, x=BIG * 8, ldx=256, res=BIG * 128, sum=BIG * 8, lds=256, codes=BIG * 64, scale=BIG * 72)
    for at in (BIG * 8 + 252, BIG * 8 + 772, BIG * 8 + 1024 * (ROWS - 1) + 252):
        assert rmsnorm(**over, w=at) == INVALID
    assert linear(y=2 * AT) == INVALID
