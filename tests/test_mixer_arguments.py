"""What the entries of the token mixers refuse, and the sizes of their work buffers: host checks, no GPU."""
import pytest

P = 1 << 20          # an aligned address that is never followed: every call here is refused before a launch


def window_args(**kw):
    a = dict(streams=[0], length=1, dQ=P, dK=P, dV=P, dY=P, dLse=P, dQLens=0, dVLens=0, dBuf=P, buf_size=1 << 40, N=1, head=4,
             kv_head=2, QL=64, VL=64, dK4=64, dV4=64, head_inner=0, scale=0.125, window=16, sinks=2)
    a.update(kw)
    return a


def grad_args(**kw):
    a = window_args()
    for x in ("dDeltaY", "dDeltaQ", "dDeltaK", "dDeltaV"):
        a[x] = P
    a.update(kw)
    return a


BAD_SIZES = [dict(N=0), dict(N=-1), dict(head=0), dict(kv_head=0), dict(kv_head=3), dict(kv_head=8), dict(QL=0), dict(VL=0),
             dict(dK4=0), dict(dK4=62), dict(dK4=132), dict(dV4=0), dict(dV4=2), dict(dV4=260), dict(window=-1), dict(sinks=-1),
             dict(QL=1 << 29, VL=(1 << 30) + 1), dict(head=1 << 16, kv_head=1 << 16)]
BAD_WINDOW = BAD_SIZES + [dict(dQ=0), dict(dK=0), dict(dV=0), dict(dY=0), dict(dQ=P + 4), dict(dK=P + 8), dict(dV=P + 4),
                          dict(dY=P + 4), dict(dLse=P + 2), dict(dQLens=P + 1), dict(dVLens=P + 3), dict(scale=float("nan")),
                          dict(scale=float("inf")), dict(length=0), dict(length=11)]


@pytest.mark.parametrize("bad", BAD_WINDOW, ids=str)
def test_window_refusals(dh, bad):
    with pytest.raises(dh.CudaException):
        dh.Cuda_attention.window_forward(**window_args(**bad))
    with pytest.raises(dh.CudaException):
        dh.Cuda_attention.window_backward(**grad_args(**bad))


@pytest.mark.parametrize("bad", [dict(dLse=0), dict(dBuf=0), dict(dBuf=P + 8), dict(buf_size=0)] +
                         [{x: v} for x in ("dDeltaY", "dDeltaQ", "dDeltaK", "dDeltaV") for v in (0, P + 4)], ids=str)
def test_window_gradient_refusals(dh, bad):
    with pytest.raises(dh.CudaException):
        dh.Cuda_attention.window_backward(**grad_args(**bad))


def test_window_buffers(dh):
    A = dh.Cuda_attention
    names = ("N", "head", "kv_head", "QL", "VL", "dK4", "dV4", "window", "sinks")
    for bad in BAD_SIZES:
        sizes = {k: v for k, v in window_args(**bad).items() if k in names}
        for f in (A.window_bufsize, A.window_backward_bufsize):
            with pytest.raises(dh.CudaException):
                f(**sizes)
    assert A.window_bufsize(64, 32, 32, 512, 512, 64, 64, 0, 0) == 0         # enough workgroups: nothing is cut
    need = A.window_bufsize(1, 4, 1, 1, 100000, 128, 128, 0, 0)              # one token on a long cache: cut
    assert need > 0
    call = dict(N=1, head=4, kv_head=1, QL=1, VL=100000, dK4=128, dV4=128, window=0, sinks=0)
    for short in (dict(dBuf=0), dict(buf_size=need - 1), dict(dBuf=P + 4)):
        with pytest.raises(dh.CudaException):
            A.window_forward(**window_args(**call, **short))


def decay_args(**kw):
    a = dict(streams=[0], length=1, dQ=P, dK=P, dV=P, dDecay=P, dState=0, dY=P, dStateOut=0, dLens=0, dBuf=P, buf_size=1 << 40,
             N=1, head=2, L=300, dK4=64, dV4=64, head_inner=0, scale=0.125)
    a.update(kw)
    return a


def decay_grad_args(**kw):
    a = decay_args()
    del a["dY"], a["dStateOut"]
    for x in ("dDeltaY", "dDeltaQ", "dDeltaK", "dDeltaV"):
        a[x] = P
    a.update(dDeltaStateOut=0, dDeltaState=0)
    a.update(kw)
    return a


BAD_DECAY_SIZES = [dict(N=0), dict(head=0), dict(L=0), dict(L=-5), dict(L=1 << 30), dict(dK4=0), dict(dK4=30), dict(dK4=132), dict(dV4=0), dict(dV4=6),
                   dict(dV4=132), dict(head=1 << 18), dict(N=1 << 16, head=1 << 15, L=200)]
BAD_DECAY = BAD_DECAY_SIZES + [dict(dQ=0), dict(dK=0), dict(dV=0), dict(dDecay=0), dict(dQ=P + 4), dict(dK=P + 4), dict(dV=P + 8),
                               dict(dDecay=P + 2), dict(dState=P + 4), dict(dLens=P + 1), dict(scale=float("-inf")), dict(length=0),
                               dict(length=11), dict(dBuf=0), dict(dBuf=P + 4), dict(buf_size=100)]


@pytest.mark.parametrize("bad", BAD_DECAY, ids=str)
def test_decay_refusals(dh, bad):
    L = dh.Cuda_linear_attention
    with pytest.raises(dh.CudaException):
        L.forward(**decay_args(**bad))
    with pytest.raises(dh.CudaException):
        L.backward(**decay_grad_args(**bad))


@pytest.mark.parametrize("bad", [dict(dY=0), dict(dY=P + 4), dict(dStateOut=P + 8)], ids=str)
def test_decay_forward_refusals(dh, bad):
    with pytest.raises(dh.CudaException):
        dh.Cuda_linear_attention.forward(**decay_args(**bad))


@pytest.mark.parametrize("bad", [{x: P + 4} for x in ("dDeltaState", "dDeltaStateOut")] +
                         [{x: v} for x in ("dDeltaY", "dDeltaQ", "dDeltaK", "dDeltaV") for v in (0, P + 4)], ids=str)
def test_decay_gradient_refusals(dh, bad):
    with pytest.raises(dh.CudaException):
        dh.Cuda_linear_attention.backward(**decay_grad_args(**bad))


def test_decay_buffers(dh):
    L = dh.Cuda_linear_attention
    names = ("N", "head", "L", "dK4", "dV4")
    for bad in BAD_DECAY_SIZES:
        sizes = {k: v for k, v in decay_args(**bad).items() if k in names}
        for f in (L.bufsize, L.backward_bufsize):
            with pytest.raises(dh.CudaException):
                f(**sizes)
    assert L.bufsize(64, 16, 1, 128, 128) == 0                   # single tokens need none
    assert L.bufsize(1, 1, 4096, 64, 64) > 0 and L.backward_bufsize(1, 1, 4096, 64, 64) > L.bufsize(1, 1, 4096, 64, 64)
