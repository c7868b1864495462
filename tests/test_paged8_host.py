"""CPU tests of the 8-bit paged cache: the entry points refuse bad arguments
before any launch, and the classes theirs before any kernel."""

import pytest
import torch

from quashkv_amd import _native as N
from quashkv_amd import paged8 as P8
from quashkv_amd.integrations.vllm_backend import QuashKVPageConfig, QuashKVPageManager

CPU = torch.device("cpu")
X = 4096          # an address that no refused call touches


def _refused(status, text, kind=N.QKV_E_INVALID):
    assert status == kind, status
    assert text in N.lib().qkv_last_error().decode()


def _plan(B=2, width=4, pool=8, pt=64, rows=4, ptr=X):
    return N.lib().qkv_page_plan(ptr, ptr, B, ptr, width, ptr, pool, ptr, pt, rows, ptr, ptr, ptr,
                                 ptr, ptr, ptr, ptr, None)


def test_plan_refusals():
    _refused(_plan(B=16001), "requests")
    _refused(_plan(B=-1), "requests")
    _refused(_plan(width=0), "pages_per_seq")
    _refused(_plan(pool=0), "num_pages")
    _refused(_plan(pt=96), "page_tokens")
    _refused(_plan(rows=-1), "rows")
    _refused(_plan(rows=1 << 31), "rows")
    _refused(_plan(ptr=None), "null pointer")
    L = N.lib()
    _refused(L.qkv_page_release(X, X, 2, X, 0, X, 8, X, 64, None), "pages_per_seq")
    _refused(L.qkv_page_release(X, X, 2, X, 4, X, 8, X, 32, None), "page_tokens")
    _refused(L.qkv_page_release(X, X, 2, X, 4, X, 8, None, 64, None), "null pointer")
    assert L.qkv_page_release(None, None, 0, None, 4, None, 8, None, 64, None) == N.QKV_OK


def _append(dt=N.QKV_F32, rows=3, H=2, d=64, fmt=0, kpool=X, pool=4, pt=64, slots=X):
    return N.lib().qkv_kv8_append(dt, X, 64, 64, X, 64, 64, slots, rows, H, d, fmt, kpool, X, X, X,
                                  pool, pt, None)


def _read(rows=3, H=2, d=64, fmt=0, kpool=X, pool=4, pt=64, dt=N.QKV_F32):
    return N.lib().qkv_kv8_read(X, rows, H, d, fmt, kpool, X, X, X, pool, pt, X, X, dt, None)


def test_append_and_read_refusals():
    for call in (_append, _read):
        _refused(call(dt=9), "dtype")
        _refused(call(d=80), "head_dim", N.QKV_E_UNSUPPORTED)
        _refused(call(fmt=2), "code format")
        _refused(call(H=0), "kv heads")
        _refused(call(pool=0), "num_pages")
        _refused(call(pt=16), "page_tokens")
        _refused(call(rows=-1), "rows")
        _refused(call(rows=1 << 31), "rows")
        _refused(call(kpool=X + 8), "16-byte aligned")
        _refused(call(kpool=None), "null pointer")
        assert call(rows=0) == N.QKV_OK
    _refused(_append(slots=None), "null pointer")


def _attend(dt=N.QKV_F32, rows=4, fmt=0, pool=4, pt=64, width=2, q_start=X, q_lens=X, B=2, Hq=4,
            H=2, d=64, max_q=2, odt=N.QKV_F32, ws=X, ws_bytes=1 << 40, q=X, kpool=X):
    return N.lib().qkv_kv8_attention(q, dt, 256, 64, rows, kpool, X, X, X, fmt, pool, pt, X, width,
                                     q_start, q_lens, X, B, Hq, H, d, max_q, 0.1, 1, X, odt, ws,
                                     ws_bytes, None)


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
    _refused(_attend(rows=-1), "rows")
    _refused(_attend(rows=5, q_start=None, q_lens=None), "without q_start")
    _refused(_attend(q_start=None), "q_lens needs q_start")
    _refused(_attend(q=None), "null pointer")
    _refused(_attend(kpool=X + 4), "16-byte aligned")
    _refused(_attend(ws_bytes=0), "workspace")
    _refused(_attend(ws=X + 16), "workspace")
    _refused(_attend(ws=None), "workspace")
    assert _attend(rows=0) == N.QKV_OK and _attend(B=0) == N.QKV_OK


def test_workspace_grows_with_the_batch():
    L = N.lib()
    size = [L.qkv_kv8_attention_workspace_bytes(B, B * Q, 32, 8, 128, Q)
            for B, Q in ((1, 1), (1, 2048), (64, 1), (64, 200))]
    assert min(size) > 0 and all(s % 256 == 0 for s in size)
    assert max(size) < 1 << 28


def test_classes():
    for kw in (dict(d=80), dict(page_tokens=100), dict(code="int4"), dict(num_pages=0), dict(B=0)):
        with pytest.raises(ValueError):
            P8.PagedKV8Store(**{**dict(B=1, H=1, d=64, num_pages=2, device=CPU), **kw})
    for kw in (dict(head_dim=80), dict(page_tokens=100), dict(code="x")):
        with pytest.raises(ValueError):
            P8.PagedKV8Engine(device=CPU, **kw)
    st = P8.PagedKV8Store(2, 3, 64, 5, CPU, page_tokens=128, pages_per_seq=4, code="fp8")
    assert st.kpool.shape == (5, 3, 128, 64) and st.vpool.shape == (5, 3, 8, 64, 16)
    assert st.kpool.dtype == torch.float8_e4m3fn and st.free.tolist() == [4, 3, 2, 1, 0]
    st.grow(7, 6)
    assert st.num_pages == 7 and st.pages_per_seq == 6 and st.free_count.item() == 7
    assert sorted(st.free.tolist()) == list(range(7)) and st.free.tolist()[-1] == 0
    x = torch.zeros(1, 3, 64)
    for call in (lambda: st.plan(torch.zeros(2, dtype=torch.int32), 1),
                 lambda: P8.append_kv8(x, x, torch.zeros(1, dtype=torch.long), **st.pools()),
                 lambda: st.read(torch.zeros(1, dtype=torch.long)),
                 lambda: P8.attention_kv8(x, **st.pools(), table=st.table, kv_lens=st.lens),
                 lambda: st.release()):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_page_manager_of_8_bits():
    cfg = QuashKVPageConfig(key_bits=8, value_bits=8)
    pm = QuashKVPageManager(2, 128, cfg, CPU)
    assert pm.paged and isinstance(pm.engine, P8.PagedKV8Engine) and pm.total_tokens == 0
    assert pm.compression_ratio() == 1.0
    with pytest.raises(ValueError, match="No compressed"):
        pm.attention(torch.zeros(1, 2, 1, 128))
    with pytest.raises(RuntimeError, match="GPU"):
        pm.compress_and_store(torch.zeros(1, 2, 4, 128), torch.zeros(1, 2, 4, 128))
    with pytest.raises(ValueError):
        QuashKVPageManager(2, 80, cfg, CPU)
    with pytest.raises(ValueError):
        QuashKVPageManager(2, 128, QuashKVPageConfig(key_bits=8, value_bits=3), CPU)
