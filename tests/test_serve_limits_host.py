"""Sizes of the batched decode operators that a launch cannot hold (2^32 threads) are refused on the host."""
from test_serve_host import NOT_INIT, UNSUPPORTED, append, cache


def test_append_tokens():
    assert append(cache(), tokens=(1 << 31) - 1) == NOT_INIT  # in several launches
    assert append(cache(), tokens=1 << 31) == UNSUPPORTED
