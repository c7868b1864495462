"""The 8-bit paged cache at its edges (quashkv_amd.paged8): blocks of zero values, queries
of NaN, scales near the largest fp32, row offsets behind the buffer, bounds of the longest
request that are too small.  Definitions and bounds are tests/kv8_reference.py's."""

import math

import pytest
import torch

from quashkv_amd import _native as N
from quashkv_amd import paged8 as P8
from tests import kv8_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
# a weight's half step: f16 pairs, or one f16 for 16-bit results
WEIGHT = {F32: 2.0 ** -22, F16: 2.0 ** -11, BF16: 2.0 ** -11}


@pytest.fixture(autouse=True, scope="module")
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    N.lib()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _held(k, v, code="int8", pt=256, width=None):
    """One request's tokens (T, H, d) in a store, and what the cache holds of them
    (float64, on the CPU)."""
    T, H, d = k.shape
    pages = -(-T // pt)
    st = P8.PagedKV8Store(1, H, d, pages, DEV, page_tokens=pt, pages_per_seq=width or pages,
                          code=code)
    st.append(k.to(DEV), v.to(DEV), st.plan(i32([T]), T))
    cache = R.Cache(1, H, d, code)
    cache.append(0, k, v)
    return st, cache.values(0, 0), cache.values(0, 1)


def _check(st, kd, vd, q, out_dtype=F32, causal=False, scale=None, **kw):
    """q (Q, Hq, d) against the definition."""
    T, _, d = kd.shape
    sc = 1 / math.sqrt(d) if scale is None else scale
    x = P8.attention_kv8(q.to(DEV), **st.pools(), table=st.table, kv_lens=st.lens, scale=sc,
                         causal=causal, out_dtype=out_dtype, **kw).cpu().double()
    o, tol = R.attend(q.double(), kd, vd, sc, T - q.shape[0] if causal else None, 2.0 ** -22,
                      WEIGHT[out_dtype], HALF[out_dtype])
    assert torch.isfinite(x).all()
    bad = (x - o).abs() > tol + 2.0 ** -149
    assert not bad.any(), ((x - o).abs().max().item(), o.abs().max().item())
    return x


# ------------------------------------- bounds of the longest request that are too small

@pytest.mark.parametrize("T", [200, 3000])                 # whole, and cut into pieces
@pytest.mark.parametrize("Q", [1, 9, 100])
def test_uniform_rows_whatever_the_hint(T, Q):
    """Without q_start the hint picks kernels and workspace alike: the results are right, and
    no byte behind the workspace that the hint asks for is written."""
    B, H, G, d = 2, 2, 4, 128
    gen = torch.Generator().manual_seed(T + Q)
    st = P8.PagedKV8Store(B, H, d, 2 * -(-T // 64), DEV, page_tokens=64)
    x = torch.randn(2, B * T, H, d, generator=gen).to(BF16)
    st.append(*x.to(DEV), st.plan(i32([T, T]), B * T))
    q = torch.randn(B * Q, H * G, d, generator=gen)
    refs = []
    for b in range(B):
        cache = R.Cache(1, H, d, "int8")
        cache.append(0, x[0, b * T:(b + 1) * T], x[1, b * T:(b + 1) * T])
        refs.append(R.attend(q[b * Q:(b + 1) * Q].double(), cache.values(0, 0), cache.values(0, 1),
                             1 / math.sqrt(d), T - Q, 2.0 ** -22, 2.0 ** -22, HALF[F32]))
    for hint in (None, 0, 1, Q, 1000):
        longest = Q if hint is None else min(Q, hint)
        nbytes = P8.attention_kv8_workspace_bytes(B, B * Q, H * G, H, d, longest)
        space = torch.full((nbytes + (32 << 20),), 0x5a, dtype=torch.uint8, device=DEV)
        for ws in (None, space[:nbytes]):
            out = P8.attention_kv8(q.to(DEV), **st.pools(), table=st.table, kv_lens=st.lens,
                                   causal=True, max_q_len=hint, workspace=ws).cpu().double()
            for b, (o, tol) in enumerate(refs):
                assert ((out[b * Q:(b + 1) * Q] - o).abs() <= tol).all(), (hint, b)
        assert (space[nbytes:] == 0x5a).all(), hint
    with pytest.raises(ValueError, match="workspace"):
        P8.attention_kv8(q.to(DEV), **st.pools(), table=st.table, kv_lens=st.lens, max_q_len=1,
                         workspace=space[:256])
# -------------------------------------------------------- blocks of zero values

# tokens whose values are 0, of T
ZEROS = {"first": (0, 64), "middle": (320, 352), "last": (-16, None), "most": (16, -16),
         "half": (0, 2048)}


@pytest.mark.parametrize("T", [700, 4100])                 # whole, and cut into pieces
@pytest.mark.parametrize("Q", [1, 40])                     # both kernels
@pytest.mark.parametrize("size", [1e-3, 1e-6, 1e-9, 2.0 ** -92, 1e30])
def test_zero_blocks_beside_values_of_any_size(T, Q, size):
    gen = torch.Generator().manual_seed(T + Q)
    k = torch.randn(T, 1, 64, generator=gen)
    q = torch.randn(Q, 2, 64, generator=gen)
    for name, (a, b) in ZEROS.items():
        v = torch.randn(T, 1, 64, generator=gen) * size
        v[a:b if b is None or b < T else T // 2] = 0
        st, kd, vd = _held(k, v, pt=64, width=80)
        for out_dtype in (F32, BF16):
            x = _check(st, kd, vd, q, out_dtype, causal=Q > 1)
            assert x.any(), name


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("T", [300, 3000])
@pytest.mark.parametrize("Q", [1, 40])
def test_zero_blocks_that_take_most_of_the_weight(code, T, Q):
    """Sink tokens: values 0, scores far above the others'."""
    gen = torch.Generator().manual_seed(T)
    d = 128
    way = torch.randn(1, 1, d, generator=gen)
    way /= way.norm()
    for sink in ((0, 16), (160, 176), (T - 16 - T % 16, T - T % 16)):
        for lead in (3.0, 20.0, 60.0):                     # of the scores, natural units
            k = torch.randn(T, 1, d, generator=gen)
            k -= (k * way).sum(-1, keepdim=True) * way
            k[sink[0]:sink[1]] = way * lead
            q = way * math.sqrt(d) + 0.1 * torch.randn(Q, 4, d, generator=gen)
            for size in (1.0, 1e-5):
                v = torch.randn(T, 1, d, generator=gen) * size
                v[sink[0]:sink[1]] = 0
                st, kd, vd = _held(k, v, code, pt=64, width=80)
                _check(st, kd, vd, q)


def test_zero_values_alone():
    """Nothing but zeros: exactly 0, also where their codes are not."""
    gen = torch.Generator().manual_seed(1)
    for T in (100, 3000):
        k = torch.randn(T, 1, 64, generator=gen)
        v = torch.randn(T, 1, 64, generator=gen)
        st, _, _ = _held(k, 0 * v, pt=64, width=80)
        full, kd, vd = _held(k, v, pt=64, width=80)
        for Q in (1, 40):
            q = torch.randn(Q, 4, 64, generator=gen)
            x = P8.attention_kv8(q.to(DEV), **st.pools(), table=st.table, kv_lens=st.lens)
            assert not x.any()
        # a scale of 0 makes any codes' values 0
        full.vscale[:, :, 1] = 0
        vd = vd.clone()
        for t0 in range(16, T, 64):
            vd[t0:t0 + 16] = 0
        for Q in (1, 40):
            _check(full, kd, vd, torch.randn(Q, 4, 64, generator=gen))


# ------------------------------------------------------------- queries of NaN

@pytest.mark.parametrize("zero", [False, True])            # values
@pytest.mark.parametrize("T", [150, 5000])                 # whole, and cut into pieces
@pytest.mark.parametrize("Q", [4, 40])
def test_nan_query_stays_nan(T, Q, zero):
    """A query of NaN gives NaN in its row alone, whatever the cache's length."""
    gen = torch.Generator().manual_seed(T)
    k, v = torch.randn(2, T, 1, 64, generator=gen)
    st, kd, vd = _held(k, v * (not zero), pt=64, width=80)
    q = torch.randn(Q, 4, 64, generator=gen)
    q[1, 2, 5] = float("nan")
    q[3, 0] = float("nan")
    same = torch.ones(Q, 4, dtype=torch.bool)
    same[1, 2] = same[3, 0] = False
    o, tol = R.attend(torch.where(same[..., None], q, torch.zeros(())).double(), kd, vd, 0.125,
                      T - Q, 2.0 ** -22, 2.0 ** -22, HALF[F32])
    x = P8.attention_kv8(q.to(DEV), **st.pools(), table=st.table, kv_lens=st.lens,
                         causal=True).cpu().double()
    assert ((x - o).abs() <= tol)[same].all()
    assert x[1, 2].isnan().all() and x[3, 0].isnan().all()
    y = P8.attention_kv8(q.to(DEV).to(BF16), **st.pools(), table=st.table, kv_lens=st.lens,
                         causal=True, out_dtype=BF16).cpu()
    assert torch.equal(y.isnan().all(-1), ~same) and torch.equal(y.isnan().any(-1), ~same)


# ------------------------------------------------------ scales at fp32's upper end

@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("Q", [1, 40])
def test_values_near_the_largest_fp32(code, Q):
    """Scales up to 2^121, whose inverse times the weights' sum's factor is no normal fp32.
    (What the cache holds is read back: the definition's append clamps at 3e38.)"""
    gen = torch.Generator().manual_seed(Q)
    T, d = 640, 64
    way = torch.zeros(d)
    way[0] = 1.0
    k = torch.randn(T, 1, d, generator=gen) * (1 - way)
    v = torch.randn(T, 1, d, generator=gen).clamp(-1, 1) * 3.3e38
    k[5] = way * 40
    q = torch.randn(Q, 4, d, generator=gen)
    for lead in (0.0, 1.0, 3.0):       # of token 5's score: 5 to 15 above the others
        st, _, _ = _held(k, v, code, pt=64)
        assert st.vscale.max() > 2.0 ** (120 if code == "int8" else 118)
        slots = st.table[0].long().repeat_interleave(64) * 64 + torch.arange(T, device=DEV) % 64
        kd, vd = (x.cpu().double() for x in st.read(slots))
        _check(st, kd, vd, q + lead * way)


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("Q", [1, 40])
def test_one_token_gives_its_values(code, Q):
    """One token's weight cancels: what is left of roundings are the f16 pair's (2^-22), those
    of log2 and 1 / scale, the sum, its inverse and the products (2^-23 each at most, six of
    them): within 2^-20 of the value, at scales from 2^-99 to 2^121."""
    gen = torch.Generator().manual_seed(7)
    H, d = 512, 64
    size = torch.exp2(torch.cat([torch.linspace(-92, 127.9, H // 2),
                                 torch.linspace(122, 127.9, H // 2)]).double()).float()
    k = torch.randn(1, H, d, generator=gen)
    v = torch.randn(1, H, d, generator=gen).clamp(-1, 1) * size[:, None]
    st, _, _ = _held(k, v, code, pt=64)
    _, vd = st.read(st.table[0].long() * 64)
    x = P8.attention_kv8(torch.randn(Q, H, d, generator=gen).to(DEV), **st.pools(), table=st.table,
                         kv_lens=st.lens)
    vd = vd.double()
    assert ((x.double() - vd).abs() <= 2.0 ** -20 * vd.abs()).all()


# ------------------------------------------------------ rows behind the buffer

@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("start,rows,lens", [
    ([0, 50, 90, 400], 100, [300, 200, 500]),              # the last request's rows end early
    ([0, 60, 260, 2000, 2300], 200, [90, 2500, 40, 10]),   # and one begins behind the last row
    ([0, 1, 2, 90], 3, [70, 300, 200]),                    # one row each
])
def test_rows_end_with_the_buffer(start, rows, lens, causal):
    """Without q_lens a request's rows run to the next one's first, as far as there are any."""
    B, H, G, d = len(lens), 1, 4, 64
    gen = torch.Generator().manual_seed(rows)
    for width in (16, 80):                                 # whole tiles, and cut ones
        if max(lens) > 64 * width:
            continue
        st = P8.PagedKV8Store(B, H, d, sum(-(-t // 64) for t in lens), DEV, page_tokens=64,
                              pages_per_seq=width)
        x = torch.randn(2, sum(lens), H, d, generator=gen)
        st.append(*x.to(DEV), st.plan(i32(lens), sum(lens)))
        q = torch.randn(rows, H * G, d, generator=gen)
        out = P8.attention_kv8(q.to(DEV), **st.pools(), table=st.table, kv_lens=st.lens,
                               q_start=i32(start), causal=causal).cpu().double()
        at = 0
        for b, T in enumerate(lens):
            cache = R.Cache(1, H, d, "int8")
            cache.append(0, x[0, at:at + T], x[1, at:at + T])
            at += T
            a, e = min(start[b], rows), min(start[b + 1], rows)
            if a == e:
                continue
            n = start[b + 1] - start[b]
            # the definition of all n rows, of which the first are there
            full = torch.zeros(n, H * G, d)
            full[:e - a] = q[a:e]
            o, tol = R.attend(full[:e - a].double(), cache.values(0, 0), cache.values(0, 1),
                              1 / math.sqrt(d), T - n if causal else None, 2.0 ** -22,
                              2.0 ** -22, HALF[F32])
            assert ((out[a:e] - o).abs() <= tol).all(), (b, width)


# ---------------------------------------------------------------- bf16 results

def test_bf16_decode_results_are_rounded_once():
    """Decode weights hold 22 bits for bf16 results too: a result is the fp32 one, rounded."""
    gen = torch.Generator().manual_seed(3)
    for T in (100, 4000):
        st, _, _ = _held(*torch.randn(2, T, 2, 128, generator=gen))
        q = torch.randn(2, 8, 128, generator=gen).to(DEV).to(BF16)
        args = dict(**st.pools(), table=st.table, kv_lens=st.lens)
        x = P8.attention_kv8(q, **args)
        assert torch.equal(P8.attention_kv8(q, **args, out_dtype=BF16), x.to(BF16))


# ---------------------------------------------------------- types and page sizes

@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("pt", [512, 1024])
def test_pages_and_types(code, pt):
    """Pages of 512 and 1024 tokens; fp16 results hold their weights in 22 bits, fp32 queries
    give bf16 results; what the cache holds, read in fp16."""
    gen = torch.Generator().manual_seed(pt)
    T, H, d = 1500, 2, 96
    k, v = torch.randn(2, T, H, d, generator=gen)
    st, kd, vd = _held(k, v, code, pt)
    slots = st.table[0].cpu().long()[torch.arange(T) // pt] * pt + torch.arange(T) % pt
    order = torch.randperm(T, generator=gen)
    for dt in (F16, BF16):
        for x, ref in zip(st.read(slots[order].to(DEV), out_dtype=dt), (kd, vd)):
            assert torch.equal(x.cpu(), ref[order].float().to(dt))
    for Q in (1, 40):
        q = torch.randn(Q, 4 * H, d, generator=gen)
        _check(st, kd, vd, q, BF16, causal=True)
        _check(st, kd, vd, q.half(), F16, causal=True)
        x = P8.attention_kv8(q.half().to(DEV), **st.pools(), table=st.table, kv_lens=st.lens,
                             out_dtype=F16).cpu().double()
        o, tol = R.attend(q.half().double(), kd, vd, 1 / math.sqrt(d), None, 2.0 ** -22, 2.0 ** -22,
                          HALF[F16])
        assert ((x - o).abs() <= tol + 2.0 ** -25).all()


# ------------------------------------------------------------- a refused append

def test_refused_append_is_made_up_for():
    """A plan stands whether its append was taken or not: the rows follow with the same plan."""
    st = P8.PagedKV8Store(2, 1, 64, 6, DEV, page_tokens=64)
    cache = [R.Cache(1, 1, 64, "int8") for _ in range(2)]
    gen = torch.Generator().manual_seed(1)
    for n in ([70, 5], [1, 1], [20, 64]):
        x = torch.randn(2, sum(n), 1, 64, generator=gen)
        plan = st.plan(i32(n), sum(n))
        for k in (x[0, :, :, :32], x[0, 1:], x[0].double()):
            with pytest.raises(ValueError):
                st.append(k.to(DEV), x[1].to(DEV), plan)
        st.append(*x.to(DEV), plan)
        for b, part in enumerate(x.split(n, 1)):
            cache[b].append(0, *part)
    for b, T in enumerate([91, 70]):
        t = torch.arange(T)
        slots = st.table[b].cpu().long()[t // 64] * 64 + t % 64
        for half, y in enumerate(st.read(slots.to(DEV))):
            assert torch.equal(y.cpu(), cache[b].values(0, half).float())
