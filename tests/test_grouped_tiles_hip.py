"""The tiles that the grouped linear takes for large layers (csrc/grouped.hip,
launch_rows and weight_tile), against the 64-bit form: every depth of their
buffers from one step of the contraction to five, a short last step, uneven
groups, an empty one, and rows of no group."""
import pytest
import torch

import token_util as tu
from test_grouped_hip import check, gen
from xrdslam_amd import _lib
from xrdslam_amd.engine import grouped

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
HALF = [torch.bfloat16, torch.float16]


def uneven(m, groups, tail, seed):
    """starts of `groups` groups over m - tail rows, the third (if any) empty"""
    cuts = torch.randint(0, m - tail + 1, (groups - 1, ), generator=gen(seed))
    starts = [0, *cuts.sort().values.tolist(), m - tail]
    if groups > 2:
        starts[3] = starts[2]
    return starts


def layer(m, groups, n_in, n_out, dtype, bias, tail=37):
    g = gen(m + n_in + n_out)
    x = torch.randn(m, n_in, generator=g).to(dtype).to(DEV)
    w = torch.randn(groups, n_out, n_in, generator=g) / n_in**0.5
    b = torch.randn(groups, n_out, generator=g).to(dtype).to(DEV) \
        if bias else None
    dy = torch.randn(m, n_out, generator=g).to(dtype).to(DEV)
    return x, w.to(dtype).to(DEV), uneven(m, groups, tail, m + n_in), b, dy


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('n_in', [64, 128, 192, 200, 264])
def test_wide_result_16_bit(n_in, dtype):
    """128 x 256 products of 1 to 5 steps in three buffers; without a bias (and
    264 columns) the 256 x 256 weight gradient"""
    m, groups, n_out = 4001, 16, 3848
    # the conditions of launch_rows and weight_tile
    assert m // groups > 96 and (m // 128 + groups) * -(-n_out // 128) >= 1024
    wide = -(-n_in // 256) * -(-n_out // 256) * groups >= 512
    assert wide == (n_in == 264)
    check(*layer(m, groups, n_in, n_out, dtype, False), False)


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('n_out', [64, 128, 192, 200, 264])
def test_wide_input_gradient_16_bit(n_out, dtype):
    """128 x 128 input gradients of 1 to 5 steps, the right operand turned"""
    m, groups, n_in = 4001, 16, 3848
    assert (m // 128 + groups) * -(-n_in // 128) >= 1024
    check(*layer(m, groups, n_in, n_out, dtype, False), False)


@pytest.mark.parametrize('dtype', HALF)
def test_wide_layer_with_bias_and_relu_16_bit(dtype):
    check(*layer(4001, 16, 264, 3848, dtype, True), True)


@pytest.mark.parametrize('dtype', HALF)
def test_weight_gradient_of_few_rows_in_wide_tiles(dtype):
    """groups shorter than a step, and of exactly one and two: 256 x 256"""
    groups, n_in, n_out = 16, 520, 2600
    assert -(-n_in // 256) * -(-n_out // 256) * groups >= 512
    sizes = [0, 1, 63, 64, 65, 127, 128, 129, 192, 8, 16, 0, 256, 5, 40, 320]
    starts = [0]
    for s in sizes:
        starts.append(starts[-1] + s)
    m = starts[-1] + 3
    x, w, _, _, dy = layer(m, groups, n_in, n_out, dtype, False)
    check(x, w, starts, None, dy, False)


@pytest.mark.parametrize('bias', [False, True])
@pytest.mark.parametrize('m,n_in,n_out', [(2100, 136, 132), (5003, 260, 200)])
def test_large_weight_gradient_f32(m, n_in, n_out, bias):
    """128 x 128 tiles, groups cut into pieces and joined"""
    groups = 2
    assert m // groups >= 1024 and n_in > 128 and n_out > 128
    x, w, _, b, dy = layer(m, groups, n_in, n_out, torch.float32, bias)
    check(x, w, [0, m // 3, m - 9], b, dy, False)


def test_starts_at_the_ends_of_their_type():
    """nothing outside the rows is read or written, rows between the first and
    the last start that are in range keep their group"""
    x = torch.randn(100, 16, device=DEV)
    w = torch.randn(3, 8, 16, device=DEV)
    top, low = 2**31 - 1, -2**31
    for starts, spans in (([0, 40, 100, top], [(0, 40), (40, 100), (100, 100)]),
                          ([low, 30, top, top], [(0, 30), (30, 100), (100, 100)]),
                          ([low, low, low, top], [(0, 0), (0, 0), (0, 100)])):
        st = torch.tensor(starts, dtype=torch.int32, device=DEV)
        guard = torch.full((300, 8), 7.0, device=DEV)
        lib = _lib.lib()
        _lib.check(lib.xrd_grouped_fwd(
            0, 100, 3, 16, 8, x.data_ptr(), 16, w.data_ptr(), None,
            st.data_ptr(), 0, guard[100:].data_ptr(),
            _lib.stream_ptr(x.device)))
        assert (guard[:100] == 7).all() and (guard[200:] == 7).all()
        plain = [spans[0][0], *(b for _, b in spans)]
        want, terms = tu.linear64(x, w, plain, None)
        tu.within(guard[100:200], want, terms, 2 * 18, 'y')
        tu.within(grouped.linear(x, w, st), want, terms, 2 * 18, 'y')
