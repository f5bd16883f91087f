"""Refusals of svd_rmsnorm, svd_linear_act and svd_attn_diff (no GPU needed): the C entries return SVD_EINVAL before any device work, the Python launchers raise."""
import ctypes

import pytest
import torch

EINVAL, OK = -1, 0
BUF = (ctypes.c_char * 8192)()
A = ctypes.addressof(BUF) + (-ctypes.addressof(BUF)) % 64          # a 64-byte aligned host address, never dereferenced
BF16, F16, F32, F8 = 0, 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    from streamingt2v_amd.lib import lib as l
    return l


def norm(lib, X=A, ldx=64, R=None, ldr=0, gamma=A, eps=1e-6, Y=A, ldy=64, ys=None, S=None, lds=0, rows=4, ch=64, flags=0, dt=F16):
    return lib.svd_rmsnorm(X, ldx, R, ldr, gamma, eps, Y, ldy, ys, S, lds, rows, ch, flags, dt, None)


@pytest.mark.parametrize("bad", [
    dict(X=None), dict(Y=None), dict(ldx=63), dict(ldy=63), dict(rows=-1), dict(ch=0), dict(eps=-1e-6), dict(eps=float("nan")), dict(dt=F32), dict(dt=F8), dict(dt=-1), dict(flags=8),
    dict(R=A, ldr=63), dict(S=A, lds=64), dict(R=A, ldr=64, S=A, lds=63), dict(flags=2), dict(flags=4), dict(X=A + 1), dict(X=A + 2, flags=1), dict(Y=A + 1), dict(gamma=A + 2),
    dict(flags=4, ys=A + 2), dict(R=A + 2, ldr=64, flags=2), dict(R=A, ldr=64, S=A + 1, lds=64)], ids=str)
def test_rmsnorm_refuses(lib, bad):
    assert norm(lib, **bad) == EINVAL


def test_rmsnorm_no_rows(lib):
    assert norm(lib, rows=0) == OK


def linear(lib, X=A, ldx=64, W=A, ldw=64, xs=None, ws=None, bias=None, R=None, ldr=0, Y=A, ldy=32, M=4, N=32, K=64, act=0, flags=0, scratch=None, sb=0, it=F16, dt=F16):
    return lib.svd_linear_act(X, ldx, W, ldw, xs, ws, bias, R, ldr, Y, ldy, M, N, K, act, flags, scratch, sb, it, dt, None)


@pytest.mark.parametrize("bad", [
    dict(X=None), dict(W=None), dict(Y=None), dict(ldx=63), dict(ldw=63), dict(ldy=31), dict(R=A, ldr=31), dict(M=-1), dict(N=0), dict(K=0), dict(M=2 ** 31), dict(act=-1), dict(act=5),
    dict(flags=4), dict(flags=1), dict(it=BF16), dict(it=F32), dict(dt=F32, it=F32), dict(dt=F8, it=F8), dict(xs=A), dict(ws=A), dict(it=F8, xs=A + 2), dict(bias=A + 1), dict(X=A + 1),
    dict(W=A + 1), dict(Y=A + 1), dict(Y=A + 2, flags=2), dict(R=A + 2, ldr=32, flags=1)], ids=str)
def test_linear_refuses(lib, bad):
    assert linear(lib, **bad) == EINVAL


def test_linear_scratch_size(lib):
    f = lib.svd_linear_act_ws_bytes
    assert f(-1, 1, 1, 0, F16, 1) == EINVAL and f(1, 0, 1, 0, F16, 1) == EINVAL and f(1, 1, 0, 0, F16, 1) == EINVAL
    assert f(0, 64, 64, 0, F16, 0) == 0 and f(1, 5120, 1280, 0, F8, 0) == 0 and f(64, 64, 64, 0, F16, 0) == 0
    for m, n, k, it, fl in [(28800, 1280, 5120, BF16, 0), (2304, 1280, 5120, F8, 0), (2304, 1280, 5120, F8, 2), (1100, 1040, 4096, F16, 0)]:
        need = f(m, n, k, fl, it, 1)
        assert 0 < need <= 1 << 29 and need % 16 == 0
        big = dict(M=m, N=n, K=k, ldx=k, ldw=k, ldy=n, it=it, flags=fl, dt=BF16 if it != F16 else F16)
        assert linear(lib, **big) == EINVAL and linear(lib, scratch=A, sb=need - 1, **big) == EINVAL and linear(lib, scratch=A + 8, sb=need, **big) == EINVAL
        copies = f(m, n, k, fl, it, 0)
        assert copies == need + (m + n) * k * (1 if it == F8 else 2)
        assert linear(lib, scratch=A, sb=copies - 1, **dict(big, ldx=k + 1)) == EINVAL          # unaligned rows need room for aligned copies
    far = dict(M=1100, N=1040, K=1 << 23, ldx=1 << 23, ldw=1 << 23, ldy=1040)
    assert linear(lib, scratch=A, sb=1 << 60, **far) == EINVAL                                  # rows that no tile can address


def test_linear_no_rows(lib):
    assert linear(lib, M=0) == OK


def attn(lib, Q=A, qs=(1024, 256, 128), K=A, ks=(1024, 128, 128), V=A, vs=(1024, 128, 128), O=A, os=(1024, 256, 128), lam=A, li=0.2, gamma=None, eps=1e-5, k_len=None, q_start=None,
         B=2, nq=3, nk=8, H=2, KV=1, causal=0, ws=A, wsb=1 << 40, dt=F16):
    return lib.svd_attn_diff(Q, *qs, K, *ks, V, *vs, O, *os, lam, li, gamma, eps, k_len, q_start, B, nq, nk, H, KV, causal, ws, wsb, dt, None)


@pytest.mark.parametrize("bad", [
    dict(Q=None), dict(K=None), dict(V=None), dict(O=None), dict(lam=None), dict(qs=(1024, 252, 128)), dict(ks=(1020, 128, 128)), dict(vs=(1024, 128, 124)), dict(os=(1024, 257, 128)),
    dict(Q=A + 8), dict(K=A + 2), dict(V=A + 8), dict(O=A + 8), dict(lam=A + 2), dict(gamma=A + 1), dict(k_len=A + 2), dict(q_start=A), dict(q_start=A + 2, causal=1), dict(B=-1), dict(nq=-1),
    dict(nk=-1), dict(H=0), dict(KV=0), dict(H=3, KV=2), dict(eps=-1.0), dict(eps=float("nan")), dict(dt=F32), dict(dt=F8), dict(wsb=-1)], ids=str)
def test_attn_refuses(lib, bad):
    assert attn(lib, **bad) == EINVAL


def test_attn_nothing_to_do(lib):
    assert attn(lib, B=0) == OK and attn(lib, nq=0) == OK


def test_attn_scratch_size(lib):
    f = lib.svd_attn_diff_ws_bytes
    assert f(1, 1, 1, 3, 2) == EINVAL and f(-1, 1, 1, 1, 1) == EINVAL and f(1, 1, 1, 0, 1) == EINVAL
    assert f(0, 1, 1, 1, 1) == 0 and f(1, 0, 1, 1, 1) == 0 and f(1, 1, 0, 1, 1) == 0
    for B, nq, nk, H, KV in [(1, 1, 100, 8, 8), (8, 1, 32768, 16, 4), (1, 1, 10 ** 6, 1, 1), (4, 4000, 4000, 8, 8), (2 ** 15, 25, 25, 10, 10)]:
        n = f(B, nq, nk, H, KV)
        assert 0 <= n <= 1 << 31 and n % 16 == 0
        if n:
            assert attn(lib, B=B, nq=nq, nk=nk, H=H, KV=KV, wsb=n - 1) == EINVAL and attn(lib, B=B, nq=nq, nk=nk, H=H, KV=KV, ws=None, wsb=n) == EINVAL


def test_sizes_that_32_bit_positions_cannot_walk(lib):
    """The kernels step over channels, bytes of K and keys in 32-bit numbers; sizes whose last step would pass 2^31 are refused."""
    big = 2 ** 31 - 1
    for ch in (big, big - 254):
        assert norm(lib, ch=ch, ldx=big, ldy=big) == EINVAL
    for k in (2 ** 30 - 257, 2 ** 30 - 4096):
        assert linear(lib, K=k, ldx=big, ldw=big) == EINVAL and lib.svd_linear_act_ws_bytes(4, 32, k, 0, F16, 1) == EINVAL
    for n in (big, big - 255, 0x7fff0001):
        assert attn(lib, nk=n, ks=(0, 0, 0), vs=(0, 0, 0)) == EINVAL


def test_launchers_refuse_host_tensors():
    """There is no CPU form: the launchers say so instead of handing host addresses to a kernel."""
    from streamingt2v_amd import ops
    x = torch.zeros(4, 128, dtype=torch.float16)
    with pytest.raises(AssertionError):
        ops.rmsnorm(x)
    with pytest.raises(AssertionError):
        ops.linear_act(x, x)
    q = x.view(1, 4, 1, 128)
    with pytest.raises(AssertionError):
        ops.attn_diff(q, q, q, torch.zeros(4, 64), 0.2)


class _Gpu(torch.Tensor):
    """A host tensor that says it is on a GPU: reaches the launchers' argument checks, and none of the calls below gets past them."""
    is_cuda = True


def _g(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Gpu)


@pytest.fixture()
def nolaunch(monkeypatch):
    from streamingt2v_amd import ops

    def no(*a):
        raise RuntimeError("got past the checks")
    monkeypatch.setattr(torch.cuda, "current_device", no)
    return ops


f32 = torch.float32


@pytest.mark.parametrize("make", [
    lambda o: o.rmsnorm(_g(4, 128, 2)), lambda o: o.rmsnorm(_g(4, 128, dtype=torch.int32)), lambda o: o.rmsnorm(_g(4, 128), _g(127, dtype=f32)), lambda o: o.rmsnorm(_g(4, 128), _g(128)),
    lambda o: o.rmsnorm(_g(4, 128), _g(256, dtype=f32)[::2]), lambda o: o.rmsnorm(_g(4, 128), residual=_g(3, 128)), lambda o: o.rmsnorm(_g(4, 128), residual=_g(4, 128, dtype=torch.bfloat16)),
    lambda o: o.rmsnorm(_g(4, 128), out_sum=_g(4, 128)), lambda o: o.rmsnorm(_g(4, 128), residual=_g(4, 128), out_sum=_g(4, 128, dtype=f32)), lambda o: o.rmsnorm(_g(4, 128), out=_g(4, 64)),
    lambda o: o.rmsnorm(_g(4, 128), out=_g(4, 128), f8=True),
    lambda o: o.linear_act(_g(4, 128), _g(8, 64)), lambda o: o.linear_act(_g(4, 128), _g(8, 128, dtype=torch.bfloat16)), lambda o: o.linear_act(_g(4, 128, dtype=f32), _g(8, 128, dtype=f32)),
    lambda o: o.linear_act(_g(4, 128), _g(8, 128), act="tanh"), lambda o: o.linear_act(_g(4, 128), _g(8, 128), bias=_g(8)), lambda o: o.linear_act(_g(4, 128), _g(8, 128), bias=_g(9, dtype=f32)),
    lambda o: o.linear_act(_g(4, 128), _g(8, 128), x_scale=_g(4, dtype=f32)), lambda o: o.linear_act(_g(4, 128), _g(8, 128), residual=_g(4, 9)),
    lambda o: o.linear_act(_g(4, 128), _g(8, 128), out_dtype=torch.bfloat16), lambda o: o.linear_act(_g(4, 128), _g(8, 128), out=_g(4, 8, dtype=f32), out_dtype=torch.float16),
    lambda o: o.linear_act(_g(4, 0), _g(8, 0)), lambda o: o.linear_act(_g(4, 128), _g(0, 128)),
    lambda o: o.linear_act(_g(4, 128, dtype=torch.float8_e4m3fn), _g(8, 128, dtype=torch.float8_e4m3fn), x_scale=_g(8, dtype=f32)),
    lambda o: o.attn_diff(_g(1, 4, 1, 64), _g(1, 4, 1, 64), _g(1, 4, 1, 64), _g(4, 64, dtype=f32), 0.2), lambda o: o.attn_diff(_g(1, 4, 3, 128), _g(1, 4, 2, 128), _g(1, 4, 2, 128), _g(4, 64, dtype=f32), 0.2),
    lambda o: o.attn_diff(_g(1, 4, 2, 128), _g(1, 4, 2, 128), _g(1, 5, 2, 128), _g(4, 64, dtype=f32), 0.2), lambda o: o.attn_diff(_g(2, 4, 2, 128), _g(1, 4, 2, 128), _g(1, 4, 2, 128), _g(4, 64, dtype=f32), 0.2),
    lambda o: o.attn_diff(*[_g(1, 4, 2, 128, dtype=f32)] * 3, _g(4, 64, dtype=f32), 0.2), lambda o: o.attn_diff(*[_g(1, 4, 2, 128)] * 3, _g(4, 64), 0.2),
    lambda o: o.attn_diff(*[_g(1, 4, 2, 128)] * 3, _g(4, 32, dtype=f32), 0.2), lambda o: o.attn_diff(*[_g(1, 4, 2, 128)] * 3, _g(4, 64, dtype=f32), 0.2, gamma=_g(64, dtype=f32)),
    lambda o: o.attn_diff(*[_g(1, 4, 2, 128)] * 3, _g(4, 64, dtype=f32), 0.2, k_len=_g(1, dtype=torch.int64)),
    lambda o: o.attn_diff(*[_g(1, 4, 2, 128)] * 3, _g(4, 64, dtype=f32), 0.2, k_len=_g(2, dtype=torch.int32)),
    lambda o: o.attn_diff(*[_g(1, 4, 2, 128)] * 3, _g(4, 64, dtype=f32), 0.2, q_start=_g(1, dtype=torch.int32)),
    lambda o: o.attn_diff(*[_g(1, 4, 2, 128)] * 3, _g(4, 64, dtype=f32), 0.2, out=_g(1, 4, 2, 128, dtype=torch.bfloat16)),
])
def test_launchers_refuse(nolaunch, make):
    with pytest.raises(AssertionError):
        make(nolaunch)
