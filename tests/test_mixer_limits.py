"""Borders of the token mixers' host arithmetic: no GPU."""
import ctypes
import random

import pytest

from test_mixer_arguments import decay_args, decay_grad_args, grad_args, window_args


def deal_bounds(dh, total, slots, pairs, least=4):
    lo, hi = ctypes.c_int32(), ctypes.c_int32()
    dh.lib.dragon_window_deal_bounds(float(total), slots, pairs, least, ctypes.byref(lo), ctypes.byref(hi))
    return lo.value, hi.value


def parts(steps, longest):
    return sum(max(-(-s // longest), 1) for s in steps)


@pytest.mark.parametrize("pairs", (1, 2, 3, 60, 256, 500, 505, 508, 510, 511, 512))
@pytest.mark.parametrize("most", (1, 100, 70000, 1 << 22, 1 << 25))
def test_the_parts_fit_the_slots_at_the_upper_bound(dh, pairs, most):
    """512 slots; a tile has up to 2^25 steps (2^30 keys, 32 at a time).  With one slot to spare all / (slots - pairs) is the
    sum of all steps, up to 2^34."""
    rng = random.Random(pairs * 31 + most)
    for steps in ([most] * pairs, [rng.randint(0, most) for _ in range(pairs)], [most] + [0] * (pairs - 1)):
        lo, hi = deal_bounds(dh, sum(steps), 512, pairs)
        assert 4 <= lo <= hi
        assert parts(steps, hi) <= 512
        assert lo == 4 or parts(steps, lo - 1) > 512        # what lies below lo does not fit


# A launch has fewer than 2^32 threads along x.  Just inside and just outside, kernel by kernel:
# N, head, kv_head, QL, VL, d, window, sinks of the forward pass
FORWARD = [((1 << 24) - 1, 1, 1, 1, 1, 4, 0, 0), ((1 << 22) - 1, 8, 1, 8, 1, 4, 0, 0)]                 # 16 and 64 rows a key / value head
FORWARD_BEYOND = [(1 << 24, 1, 1, 1, 1, 4, 0, 0), (1 << 23, 2, 2, 1, 1, 64, 0, 0), (1 << 22, 8, 1, 8, 1, 4, 0, 0)]
# and of the gradient: rows over 8, tiles of 512 threads, key tiles
BACKWARD = [((1 << 20) - 1, 1, 1, 127, 1, 4, 0, 0), (1 << 22, 2, 1, 1, 1, 4, 0, 0), (1, 1, 1, 1, (1 << 30) - 1000, 4, 0, 0)]
BACKWARD_BEYOND = [(1 << 20, 1, 1, 128, 1, 4, 0, 0), (1 << 24, 1, 1, 1, 1, 4, 0, 0), (1 << 23, 1, 1, 1, 1, 4, 0, 0),
                   (1 << 23, 1, 1, 1, 129, 4, 0, 0)]


def window_sizes(c):
    return dict(zip(("N", "head", "kv_head", "QL", "VL"), c), dK4=c[5], dV4=c[5], window=c[6], sinks=c[7])


@pytest.mark.parametrize("case", FORWARD, ids=str)
def test_window_sizes_that_a_launch_takes(dh, case):
    assert dh.Cuda_attention.window_bufsize(**window_sizes(case)) >= 0


@pytest.mark.parametrize("case", FORWARD_BEYOND, ids=str)
def test_window_sizes_beyond_a_launch(dh, case):
    with pytest.raises(dh.CudaException):
        dh.Cuda_attention.window_bufsize(**window_sizes(case))
    with pytest.raises(dh.CudaException):
        dh.Cuda_attention.window_forward(**window_args(**window_sizes(case)))


@pytest.mark.parametrize("case", BACKWARD, ids=str)
def test_window_gradient_sizes_that_a_launch_takes(dh, case):
    assert dh.Cuda_attention.window_backward_bufsize(**window_sizes(case)) > 0


@pytest.mark.parametrize("case", BACKWARD_BEYOND, ids=str)
def test_window_gradient_sizes_beyond_a_launch(dh, case):
    with pytest.raises(dh.CudaException):
        dh.Cuda_attention.window_backward_bufsize(**window_sizes(case))
    with pytest.raises(dh.CudaException):
        dh.Cuda_attention.window_backward(**grad_args(**window_sizes(case)))


# N, head, L, dk, dv: a wavefront for 32 columns, or four for 64 of the single tokens'
DECAY = [((1 << 24) - 1, 1, 1, 4, 4), ((1 << 23) - 1, 1, 1, 4, 128), ((1 << 24) - 1, 1, 13, 4, 128), ((1 << 25) - 1, 1, 13, 128, 4)]
DECAY_BEYOND = [(1 << 24, 1, 1, 4, 4), (1 << 23, 1, 12, 4, 128), (1 << 24, 1, 13, 4, 128), (1 << 22, 4, 13, 128, 100)]
DECAY_BACKWARD = [((1 << 24) - 1, 1, 1, 4, 128), ((1 << 25) - 1, 1, 1, 4, 4)]
DECAY_BACKWARD_BEYOND = [(1 << 24, 1, 1, 4, 128), (1 << 24, 1, 13, 128, 4), (1 << 22, 4, 1, 100, 4)]


def decay_sizes(c):
    return dict(zip(("N", "head", "L", "dK4", "dV4"), c))


@pytest.mark.parametrize("case", DECAY, ids=str)
def test_decay_sizes_that_a_launch_takes(dh, case):
    assert dh.Cuda_linear_attention.bufsize(**decay_sizes(case)) == 0


@pytest.mark.parametrize("case", DECAY_BEYOND, ids=str)
def test_decay_sizes_beyond_a_launch(dh, case):
    with pytest.raises(dh.CudaException):
        dh.Cuda_linear_attention.bufsize(**decay_sizes(case))
    with pytest.raises(dh.CudaException):
        dh.Cuda_linear_attention.forward(**decay_args(**decay_sizes(case)))


@pytest.mark.parametrize("case", DECAY_BACKWARD, ids=str)
def test_decay_gradient_sizes_that_a_launch_takes(dh, case):
    assert dh.Cuda_linear_attention.backward_bufsize(**decay_sizes(case)) == 0


@pytest.mark.parametrize("case", DECAY_BACKWARD_BEYOND, ids=str)
def test_decay_gradient_sizes_beyond_a_launch(dh, case):
    with pytest.raises(dh.CudaException):
        dh.Cuda_linear_attention.backward_bufsize(**decay_sizes(case))
    with pytest.raises(dh.CudaException):
        dh.Cuda_linear_attention.backward(**decay_grad_args(**decay_sizes(case)))


@pytest.mark.parametrize("dk, dv", [(128, 64), (128, 32), (68, 4), (128, 128), (4, 128)])
def test_a_sequence_is_not_cut_where_the_whole_walks_fill_the_chip(dh, dk, dv):
    """Two workgroups a compute unit where a head dimension is above 64: with 500 pairs there is no room for segments."""
    assert dh.Cuda_linear_attention.bufsize(N=500, head=1, L=4096, dK4=dk, dV4=dv) == 0
    assert dh.Cuda_linear_attention.backward_bufsize(N=500, head=1, L=4096, dK4=dk, dV4=dv) == 0
    assert dh.Cuda_linear_attention.bufsize(N=100, head=1, L=4096, dK4=dk, dV4=dv) > 0
