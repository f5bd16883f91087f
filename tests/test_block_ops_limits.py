"""Refusals of svd_attn_diff and the block's launchers at the edge of what a call can hold (no GPU needed)."""
import pytest  # noqa: F401

from tests.test_block_ops_args import EINVAL, attn, lib  # noqa: F401

def test_attn_more_threads_than_a_launch_has(lib):
    """2^26 waves are 2^32 threads, which no launch has: refused like any other size, not handed to the driver."""
    for B in (2 ** 26, 2 ** 26 + 1, 2 ** 30):
        assert attn(lib, B=B, nq=1, nk=25, H=1, KV=1, qs=(0, 0, 0), ks=(0, 0, 0), vs=(0, 0, 0), os=(0, 0, 0)) == EINVAL
    assert attn(lib, B=2 ** 24, nq=65, nk=25, H=1, KV=1, qs=(0, 0, 0), ks=(0, 0, 0), vs=(0, 0, 0), os=(0, 0, 0)) == EINVAL          # 2^24 workgroups of 256
