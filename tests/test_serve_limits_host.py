"""Sizes of the batched decode operators that a launch cannot hold (2^32 threads) are refused on the host."""
from test_serve_host import NOT_INIT, UNSUPPORTED, append, cache, linear


def test_linear_q4_channels():
    most = (1 << 30) - 1024
    for M in (1, 5, 9, 17):
        assert linear(M=M, N=most, K=32, group=32) == NOT_INIT
        assert linear(M=M, N=most + 1, K=32, group=32) == UNSUPPORTED
        assert linear(M=M, N=1 << 30, K=32, group=32) == UNSUPPORTED


def test_append_tokens():
    assert append(cache(), tokens=(1 << 31) - 1) == NOT_INIT  # in several launches
    assert append(cache(), tokens=1 << 31) == UNSUPPORTED
