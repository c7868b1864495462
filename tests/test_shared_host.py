"""CPU tests of shared pages and rotary positions: the entry points refuse bad arguments before
any launch, the classes theirs before any kernel, and frequencies and turns are their formulas."""

import math
from fractions import Fraction

import pytest
import torch

import quashkv_amd as Q
from quashkv_amd import _native as N
from quashkv_amd import paged8 as P8
from quashkv_amd import rotary as rot

CPU = torch.device("cpu")
X = 4096          # an address that no refused call touches


def _refused(status, text, kind=N.QKV_E_INVALID):
    assert status == kind, status
    assert text in N.lib().qkv_last_error().decode()


def _fork(B=2, width=4, forks=1, pool=8, pt=64, ptr=X, shares=X):
    return N.lib().qkv_page_fork(ptr, ptr, B, width, ptr, ptr, None, forks, ptr, pool, ptr, shares,
                                 pt, ptr, ptr, ptr, ptr, None)


def _release(B=2, width=4, pool=8, pt=64, ptr=X, shares=X):
    return N.lib().qkv_page_release_shared(ptr, ptr, B, ptr, width, ptr, pool, ptr, shares, pt,
                                           None)


def _compact(B=2, width=4, pool=8, pt=64, ptr=X):
    return N.lib().qkv_page_compact(ptr, ptr, B, width, ptr, pool, ptr, None, pt, ptr, ptr, ptr,
                                    ptr, None)


@pytest.mark.parametrize("call", [_fork, _release, _compact])
def test_page_refusals(call):
    _refused(call(B=16001), "requests")
    _refused(call(B=-1), "requests")
    _refused(call(width=0), "pages_per_seq")
    _refused(call(pool=0), "num_pages")
    _refused(call(pt=96), "page_tokens")
    _refused(call(ptr=None), "null pointer")


def test_more_page_refusals():
    _refused(_fork(forks=16001), "forks")
    _refused(_fork(forks=-1), "forks")
    _refused(_fork(shares=None), "null pointer")
    _refused(_release(shares=None), "null pointer")
    _refused(_compact(pool=(1 << 20) + 1), "pages")
    assert _fork(forks=0, ptr=None) == N.QKV_OK and _release(B=0, ptr=None) == N.QKV_OK


def _copy(n=1, H=2, d=64, fmt=0, kpool=X, pool=4, pt=64, ptr=X):
    return N.lib().qkv_kv8_copy_pages(ptr, X, None, n, None, H, d, fmt, kpool, X, X, X, pool, pt,
                                      None)


def test_copy_refusals():
    _refused(_copy(n=-1), "number of pages")
    _refused(_copy(d=80), "head_dim", N.QKV_E_UNSUPPORTED)
    _refused(_copy(fmt=2), "code format")
    _refused(_copy(H=0), "kv heads")
    _refused(_copy(pool=0), "num_pages")
    _refused(_copy(pt=32), "page_tokens")
    _refused(_copy(kpool=X + 8), "16-byte aligned")
    _refused(_copy(ptr=None), "null pointer")
    assert _copy(n=0, ptr=None) == N.QKV_OK


def _rotary(dt=N.QKV_BF16, q=X, Hq=4, k=X, Hk=2, rows=3, d=64, R=64, pos=X):
    return N.lib().qkv_rotary(dt, q, 256, 64, Hq, k, 128, 64, Hk, rows, d, R, pos, X, 1.0, 0, 0, X,
                              256, 64, X, 128, 64, None)


def test_rotary_refusals():
    _refused(_rotary(dt=7), "element type")
    for R in (0, 3, 66, -2):
        _refused(_rotary(R=R), "even number")
    _refused(_rotary(d=1024, R=514), "even number")
    _refused(_rotary(Hq=-1), "heads")
    _refused(_rotary(Hq=1 << 25), "heads")
    _refused(_rotary(rows=-1), "rows")
    _refused(_rotary(rows=1 << 31), "rows")
    _refused(_rotary(q=None), "null pointer")
    _refused(_rotary(k=None), "null pointer")
    _refused(_rotary(pos=None), "null pointer")
    assert _rotary(rows=0) == N.QKV_OK and _rotary(Hq=0, Hk=0, q=None, k=None) == N.QKV_OK


def _size(B, groups, rows, Hq=32, H=8, d=128):
    return N.lib().qkv_kv8_attention_shared_workspace_bytes(B, groups, rows, Hq, H, d)


def _attend(dt=N.QKV_F32, rows=4, fmt=0, pool=4, pt=64, width=2, q_start=X, q_lens=X, B=2, groups=1,
            Hq=4, H=2, d=64, odt=N.QKV_F32, ws=X, ws_bytes=1 << 40, q=X, kpool=X, group_start=X):
    return N.lib().qkv_kv8_attention_shared(
        q, dt, 256, 64, rows, kpool, X, X, X, fmt, pool, pt, X, width, group_start, X, groups, 0,
        q_start, q_lens, X, B, Hq, H, d, 0.1, 1, X, odt, ws, ws_bytes, None)


def test_attention_refusals():
    _refused(_attend(dt=5), "element type")
    _refused(_attend(odt=5), "element type")
    _refused(_attend(d=80), "head_dim", N.QKV_E_UNSUPPORTED)
    _refused(_attend(Hq=5), "multiple of kv heads")
    _refused(_attend(Hq=0), "multiple of kv heads")
    _refused(_attend(H=0), "kv heads")
    _refused(_attend(pool=0), "num_pages")
    _refused(_attend(pt=65), "page_tokens")
    _refused(_attend(width=0), "pages_per_seq")
    _refused(_attend(B=-1), "batch")
    _refused(_attend(B=16001), "batch")
    _refused(_attend(groups=-1), "groups")
    _refused(_attend(groups=2049), "groups")
    _refused(_attend(group_start=None), "null pointer")
    _refused(_attend(rows=-1), "rows")
    _refused(_attend(rows=1 << 26), "rows")
    _refused(_attend(rows=16000, B=16000, Hq=600, H=600), "too large")
    _refused(_attend(rows=5, q_start=None, q_lens=None), "without q_start")
    _refused(_attend(q_start=None), "q_lens needs q_start")
    _refused(_attend(q=None), "null pointer")
    _refused(_attend(kpool=X + 4), "16-byte aligned")
    _refused(_attend(ws=X + 16), "workspace")
    _refused(_attend(ws=None), "workspace")
    _refused(_attend(ws_bytes=_size(2, 1, 4, 4, 2, 64) - 1), "workspace")
    assert _attend(rows=0) == N.QKV_OK and _attend(B=0) == N.QKV_OK


def test_workspace():
    size = [_size(*a) for a in ((1, 0, 1), (64, 1, 64), (64, 64, 64), (8, 1, 2400), (16000, 2000, 16000))]
    assert min(size) > 0 and all(s % 256 == 0 for s in size)
    assert size[1] < 32 << 20 and max(size) < 1 << 31


# ------------------------------------------------------------- Python refusals

def test_functions_want_a_gpu_and_shapes():
    st = P8.PagedKV8Store(2, 1, 64, 4, CPU, page_tokens=64, sharing=True)
    one = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: st.fork(one, one), lambda: st.compact(), lambda: st.release(),
                 lambda: P8.copy_pages(one, one, **st.pools()),
                 lambda: rot.rotary(torch.zeros(1, 2, 8), None, one,
                                    torch.zeros(4, dtype=torch.long))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="sharing"):
        P8.PagedKV8Store(2, 1, 64, 4, CPU, page_tokens=64).fork(one, one)
    with pytest.raises(ValueError, match="shrink"):
        st.shrink(5)
    with pytest.raises(ValueError, match="shrink"):
        st.shrink(0)
    st.free_count.fill_(1)
    with pytest.raises(ValueError, match="3 of them in use"):
        st.shrink(2)
    assert st.num_pages == 4
    st.grow(6)
    assert st.shares.tolist() == [0] * 6
    st.to(CPU)
    assert P8.PagedKV8Store(1, 1, 64, 2, CPU).shares is None


# ------------------------------------------------------------- frequencies

def test_frequencies():
    w = Q.rotary_frequencies(8, 10000.0)
    assert w == [10000.0 ** (-i / 4) for i in range(4)]
    assert Q.rotary_frequencies(8, 10000.0, "linear", 4.0) == [x / 4 for x in w]
    n = Q.rotary_frequencies(8, 10000.0, "ntk", 4.0)
    assert n[0] == 1.0 and math.isclose(n[-1], w[-1] / 4, rel_tol=1e-12)
    # within 4096 tokens the pairs make 652, 65, 6.5 and 0.65 turns
    r = Q.rotary_frequencies(8, 10000.0, "ramp", 4.0, original=4096, low=1.0, high=32.0)
    keep = (4096 * w[2] / (2 * math.pi) - 1) / 31
    assert r[:2] == w[:2] and r[3] == w[3] / 4
    assert math.isclose(r[2], w[2] * (keep + (1 - keep) / 4), rel_tol=1e-12)
    for kw in (dict(dim=7), dict(dim=0), dict(base=0.0), dict(factor=0.0), dict(scaling="other"),
               dict(scaling="ramp", low=4.0, high=4.0), dict(scaling="ntk", dim=2),
               dict(original=0)):
        with pytest.raises(ValueError):
            Q.rotary_frequencies(**{**dict(dim=8), **kw})


def test_turns_are_the_nearest():
    """2^64 w / 2 pi, rounded, modulo a turn: against pi's continued fraction bounds."""
    pi = Fraction(31415926535897932384626433832795028841971693993751, 10 ** 49)
    ws = [1.0, 0.75, 10000.0 ** -0.3, 1e-9, 0.0, -0.5, 7.0, 100.25]
    for w, t in zip(ws, Q.rotary_turns(ws).tolist()):
        exact = Fraction(w) / (2 * pi) * 2 ** 64
        off = (t - exact) % 2 ** 64
        assert min(off, 2 ** 64 - off) <= Fraction(1, 2) + Fraction(1, 10 ** 20), w
    # tensors as models hold them
    x = torch.tensor([[1.0, 0.3]], dtype=torch.float32)
    assert Q.rotary_turns(x).tolist() == Q.rotary_turns([1.0, float(x[0, 1])]).tolist()
    for bad in (float("nan"), float("inf")):
        with pytest.raises((ValueError, OverflowError)):
            Q.rotary_turns([bad])
