"""CPU checks of the decoder's ends at the limits of their 32-bit indices: the C entry points
refuse what lies past them before any launch."""

import os

import pytest

SHAPE, ARG = -1, -3


def _lib():
    import _nsa_lib
    if not os.path.exists(_nsa_lib.LIB_PATH):
        pytest.skip("libnsa_hip.so not built")
    return _nsa_lib.load()


@pytest.mark.parametrize("T", [0x7ffffff1, 1 << 31, 1 << 32, (1 << 32) + 3, 1 << 62])
def test_embed_sequences_past_32_bits(T):
    """Positions i % T are formed in 32 bits: T = 2^32 would divide by 0, 2^32 + 3 give i % 3."""
    lib = _lib()

    def fwd(T, pos=None, pw=16):
        return lib.nsa_embed_fwd(None, pos, None, pw, None, 4, T, 10, 3, 8, 1.0, 0, 0, 0, None)
    assert fwd(T) == SHAPE
    assert fwd(0x7ffffff0) == ARG                     # the longest that is taken: refused for its null tokens
    assert fwd(T, pos=16) == ARG and fwd(T, pw=None) == ARG   # T is not looked at with positions given, or without a table
    assert lib.nsa_embed_bwd(None, 16, 16, None, 0, T, T, 10, 8, 1.0, 0, 0, None) == SHAPE
