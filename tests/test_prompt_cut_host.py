"""The cut that a call of a prompt's attention takes, on the host: by its arguments alone."""

import ctypes

import pytest

from test_latent_prompt_host import _prompt


def waves(**over):
    from sgl_amd_mono.moe import _lib

    return _lib.testing_lib().mkmoe_host_prompt_waves(ctypes.byref(_prompt(**over)))


@pytest.mark.parametrize("over,want", [
    (dict(seqs=1, tokens=193, max_context=893, max_pages=56), 4),
    (dict(seqs=1, tokens=2048, max_context=2048, max_pages=128), 4),
    (dict(seqs=1, tokens=2049, max_context=2049, max_pages=129), 8),  # more new tokens
    (dict(seqs=2, tokens=4097, max_context=32768, max_pages=2048), 4),  # 2048 in the mean
    (dict(seqs=1, tokens=193, max_context=65536, max_pages=2048), 4),  # a table of 32768 tokens
    (dict(seqs=1, tokens=193, max_context=65536, max_pages=2049), 8),
    (dict(seqs=1, tokens=193, max_context=32768, max_pages=8192), 4),  # a context of as many
    (dict(seqs=2, tokens=194, max_context=65536, max_pages=8192), 4),  # each
    (dict(seqs=2, tokens=194, max_context=65538, max_pages=8192), 8),
    # where 4 waves' work passes 32 bits 8 are taken, and neither where theirs does
    (dict(seqs=512, tokens=512, heads=128, max_context=500000, max_pages=1 << 16), 4),
    (dict(seqs=512, tokens=512, heads=128, max_context=600000, max_pages=1 << 16), 8),
    (dict(seqs=512, tokens=512, heads=128, max_context=1100000, max_pages=1 << 17), 0),
])  # fmt: skip
def test_cuts(over, want):
    assert waves(**over) == want
