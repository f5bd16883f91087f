"""Refusals of svd_attn_diff and the block's launchers at the edge of what a call can hold (no GPU needed)."""
import pytest
import torch

from tests.test_block_ops_args import EINVAL, _g, attn, f32, lib, nolaunch  # noqa: F401


def test_attn_more_threads_than_a_launch_has(lib):
    """2^26 waves are 2^32 threads, which no launch has: refused like any other size, not handed to the driver."""
    for B in (2 ** 26, 2 ** 26 + 1, 2 ** 30):
        assert attn(lib, B=B, nq=1, nk=25, H=1, KV=1, qs=(0, 0, 0), ks=(0, 0, 0), vs=(0, 0, 0), os=(0, 0, 0)) == EINVAL
    assert attn(lib, B=2 ** 24, nq=65, nk=25, H=1, KV=1, qs=(0, 0, 0), ks=(0, 0, 0), vs=(0, 0, 0), os=(0, 0, 0)) == EINVAL          # 2^24 workgroups of 256


@pytest.mark.parametrize("call", [
    lambda o, b: o.linear_act(b[:, :16], _g(16, 16), out=b[:, :16]), lambda o, b: o.linear_act(_g(16, 16), b[:, :16], out=b[:, :16]), lambda o, b: o.linear_act(b[:, :16], _g(16, 16), out=b[:, 8:24]),
    lambda o, b: o.linear_act(b[:, 8:24], _g(16, 16), out=b[:, :16]), lambda o, b: o.linear_act(b[:4, :16], _g(16, 16), out=b.view(48, 16)[2:6]), lambda o, b: o.linear_act(b[3:4, :16], _g(16, 16), out=b[3:4, 15:31]),
    lambda o, b: o.attn_diff(*[_g(1, 4, 2, 128), q := _g(1, 4, 2, 128), _g(1, 4, 2, 128)], _g(4, 64, dtype=f32), 0.2, out=q),
    lambda o, b: o.attn_diff(*[_g(1, 4, 2, 128), _g(1, 4, 2, 128), q := _g(1, 4, 2, 128)], _g(4, 64, dtype=f32), 0.2, out=q)])
def test_destinations_on_an_operand_are_refused(nolaunch, call):
    """A result written over an operand that other workgroups still read would be neither."""
    with pytest.raises(AssertionError):
        call(nolaunch, _g(16, 48))


@pytest.mark.parametrize("call", [
    lambda o, b: o.linear_act(b[:, :16], b[:, 16:32], out=b[:, 32:]), lambda o, b: o.linear_act(b[:, 32:], b[:, 16:32], out=b[:, :16]), lambda o, b: o.linear_act(b[:8, :16], _g(48, 16), out=b[8:]),
    lambda o, b: o.linear_act(b[3:4, :16], _g(16, 16), out=b[3:4, 16:32]), lambda o, b: o.linear_act(_g(16, 16), _g(48, 16), residual=b, out=b),
    lambda o, b: o.attn_diff(q := _g(1, 4, 2, 128), _g(1, 4, 2, 128), _g(1, 4, 2, 128), _g(4, 64, dtype=f32), 0.2, out=q)])
def test_destinations_beside_the_operands_are_not(nolaunch, call):
    with pytest.raises(RuntimeError, match="got past the checks"):
        call(nolaunch, _g(16, 48))
