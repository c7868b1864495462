"""Which calls of attention_kv8_shared are attention_kv8's, and with what bound (host only)."""

import pytest

from quashkv_amd import _native as N


def _plain(B, rows, width, Hq=32, H=8, d=128, pt=256, groups=1):
    return N.lib().qkv_kv8_attention_shared_plain(B, groups, rows, Hq, H, d, width, pt)


@pytest.mark.parametrize("B,rows,width,bound", [
    (4, 4, 4, 8), (16, 16, 8, 8), (16, 33, 8, 33), (16, 128, 8, 128),   # up to 192 MB of tokens
    (16, 129, 8, 0),                                # more than 32 rows of a kv head a request
    (64, 64, 64, 0), (4, 4, 1000, 0),               # longer ones
    (30, 1200, 1 << 23, 1200),                      # tables of more places than a plan counts
    (0, 4, 4, 0), (4, 0, 4, 0), (16001, 16001, 1, 0), (4, 1 << 23, 4, 0), (-1, 4, 4, 0),
])
def test_plain(B, rows, width, bound):
    assert _plain(B, rows, width) == bound


def test_refused_sizes_are_not_handed_over():
    assert _plain(4, 4, 4, groups=2049) == _plain(4, 4, 4, groups=-1) == 0
    assert _plain(4, 4, 4, H=0) == _plain(4, 4, 4, Hq=4) == 0
