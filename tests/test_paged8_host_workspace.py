"""CPU tests of the 8-bit attention's workspace: its size follows the bound of the longest
request that the call is given, and a smaller one is refused before any launch."""

import pytest

from quashkv_amd import _native as N

X = 4096          # an address that no refused call touches


def _size(B, rows, max_q, Hq=32, H=8, d=128):
    return N.lib().qkv_kv8_attention_workspace_bytes(B, rows, Hq, H, d, max_q)


def test_size_follows_the_bound():
    # 4 query heads a kv head: up to 8 rows a request are one kernel's, more need both
    small = _size(1, 100, 1)
    assert _size(1, 100, 0) == _size(1, 100, 8) == small
    assert _size(1, 100, 9) > small + (1 << 20)
    assert _size(1, 100, 9) == _size(1, 100, 100) == _size(1, 100, 1 << 40)
    # a bound above the rows counts as them
    assert _size(4, 8, 1 << 40) == _size(4, 8, 8) == _size(4, 8, 1)


@pytest.mark.parametrize("q_start", [X, None])
@pytest.mark.parametrize("B,rows,max_q", [(1, 100, 1), (1, 100, 100), (2, 100, 1000), (5, 5, 1),
                                          (100, 1000, 3), (100, 1000, 10)])
def test_smaller_workspaces_are_refused(q_start, B, rows, max_q):
    need = _size(B, rows, max_q)
    for have in (0, 256, need - 256, need - 1):
        st = N.lib().qkv_kv8_attention(X, N.QKV_BF16, 4096, 128, rows, X, X, X, X, 0, 4, 64, X, 2,
                                       q_start, None, X, B, 32, 8, 128, max_q, 0.1, 1, X,
                                       N.QKV_BF16, X, have, None)
        assert st == N.QKV_E_INVALID and "workspace" in N.lib().qkv_last_error().decode(), have
