"""lz_call: the strides that follow the words are checked to their whole length. No GPU
needed: every call is refused before any CUDA call."""
import struct

import pytest


@pytest.fixture(scope="module")
def lib(built_lib):
    from lizard_cuda import _lib
    return _lib.load()


def test_strides_have_to_lie_within_the_words(lib):
    p = 0x1000

    def call(at, at_prev, n):
        """32 arguments, then room for strides, n words in all; every last dimension has
        stride 2, which the entry refuses once the words are accepted."""
        args = [p, p, p, 0, at, p, p, 0, 0, p, p, at_prev, p, p, 0, 0, p, p, p, p, 4, p, p, 1 << 30,
                2, 8, 2, 4, 4, 64, 64, 0]
        assert len(args) == 32
        words = args + [2] * (80 - len(args))  # readable past n
        return lib.lz_call(2, struct.pack("80q", *words), n), lib.lz_last_error_string()

    assert call(32, 44, 52) == (1, b"lz_swa_decode_block: the last dimension must be contiguous")
    # q, k and v have 12 strides
    for at in (41, 42, 43, 44, 45, 52):
        rc, msg = call(at, 32, 52)
        assert rc == 1 and b"does not fit" in msg, at
    rc, msg = call(40, 32, 52)
    assert rc == 1 and b"contiguous" in msg
    # the block before has 8
    for at in (45, 52):
        rc, msg = call(32, at, 52)
        assert rc == 1 and b"does not fit" in msg, at
