"""What attention over full-width pages refuses of buffers and sizes that its kernels could not keep
apart or count. Every call stops at its checks: no kernel is launched."""

import ctypes

import pytest

from everserve_amd import kernels

AT = 1 << 20  # an address that is never dereferenced


@pytest.fixture(scope="module")
def lib():
    return kernels.open_library(kernels.library_path())


def attend(lib, q=AT, out=1 << 24, tokens=3, qs=(256, 64), bs=16, width=1, max_len=0, groups=0,
           prefix_width=0, max_prefix=0, work=None, size=0):
    """Three single queries of four heads of 64 on two; one part a row, so no workspace is needed.
    Returns the message of the refusal."""
    p = ctypes.c_void_p
    rc = lib.evs_attend(p(q), (ctypes.c_int64 * 2)(*qs), 0, p(out), None, tokens, 4, p(1 << 28), 9,
                        bs, 2, 64, (ctypes.c_int64 * 5)(2048, 128, 64, 18432, 1), p(1 << 16), width,
                        width, p(1 << 17), None, tokens, 1, max_len, p(1 << 18), prefix_width,
                        prefix_width, p(1 << 18), p(1 << 18), groups, max_prefix, None, 0.125, work,
                        size, None)
    assert rc == 1
    return lib.evs_last_error().decode()


SIZE = 3 * 4 * 64 * 2  # bytes of the output


@pytest.mark.parametrize("out,qs", [
    (AT, (256, 64)),
    (AT + SIZE - 16, (256, 64)), (AT - SIZE + 16, (256, 64)),  # the last row, and the first
    (AT + 512, (256, 64)),  # a later token of the same tensor
    (AT + 2 * 4096 + 3 * 128, (2048, 64)),  # the last row of queries that lie apart
    (AT + 2 * 4096 + 4 * 128 - 16, (2048, 64)),
    (AT - SIZE + 16, (2048, 64)),
    (AT + 3 * 4096 - 128, (64, 2048)),  # head by head: from the gap into the last head
    (AT + 16, (0, 64)),  # one row for all tokens
    (AT + 16, (0, 0)),
    (AT - 2 * 512 + 16, (-256, 64)),  # the tokens backwards
    (AT - 3 * 128, (256, -64)),
])
def test_an_output_among_the_queries_is_refused(lib, out, qs):
    assert "must not be the queries" in attend(lib, out=out, qs=qs)


@pytest.mark.parametrize("width,prefix_width,bs", [
    (1 << 10, 1 << 10, 1 << 20), (2047, 1, 1 << 20), (2047, 2047, 1 << 20), (1, (1 << 31) - 1, 1),
    ((1 << 31) - 1, (1 << 31) - 1, (1 << 31) - 1), (1 << 30, 1, 1 << 30)])
@pytest.mark.parametrize("groups", [0, 1])
def test_prefixes_and_own_tokens_that_32_bits_do_not_count_are_refused(lib, width, prefix_width, bs,
                                                                       groups):
    """A long chunk takes its prefix and its own tokens as one context, numbered in 32 bits; parts
    of the tables' whole room are dealt where a caller gives no bound."""
    for bounds in (dict(), dict(max_len=1, max_prefix=1)):
        said = attend(lib, width=width, prefix_width=prefix_width, bs=bs, groups=groups, **bounds)
        assert "2^31 tokens" in said


@pytest.mark.parametrize("width,prefix_width,bs", [(1 << 10, 1023, 1 << 20), (2046, 1, 1 << 20),
                                                   (1 << 20, 0, 1 << 12), (1 << 10, (1 << 20) - 1, 1 << 10)])
def test_room_just_below_and_wide_tables_without_prefixes_are_not(lib, width, prefix_width, bs):
    groups = 1 if prefix_width else 0
    assert "workspace" in attend(lib, width=width, prefix_width=prefix_width, bs=bs, groups=groups)
