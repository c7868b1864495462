"""The 8-bit paged cache on the GPU (quashkv_amd.paged8) against its definitions
(tests/kv8_reference.py): plans exactly, codes and scales exactly, attention within
bounds derived there; and a serving loop of plan, append, attention, release as a
program runs it, eager and captured."""

import math
import random

import pytest
import torch

from quashkv_amd import _native as N
from quashkv_amd import paged8 as P8
from quashkv_amd.integrations.vllm_backend import QuashKVPageConfig, QuashKVPageManager
from tests import kv8_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


@pytest.fixture(autouse=True, scope="module")
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    N.lib()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------- plans

def _plan_case(lens, new, pt, rows, width=None, spare=None, seed=0):
    rng = random.Random(seed)
    held = [-(-t // pt) for t in lens]
    want = [-(-(t + max(n, 0)) // pt) for t, n in zip(lens, new)]
    width = width or max(max(want), max(held), 1)
    spare = sum(w - h for w, h in zip(want, held)) if spare is None else spare
    pool = sum(held) + spare + 3
    ids = list(range(pool))
    rng.shuffle(ids)
    table = [[-7] * width for _ in lens]
    for b, h in enumerate(held):
        for p in range(h):
            table[b][p] = ids.pop()
    free = ids + [-5] * (pool - len(ids))
    return table, free, spare, pool


def _check_plan(lens, new, pt, rows, width=None, spare=None, seed=0):
    table, free, count, _ = _plan_case(lens, new, pt, rows, width, spare, seed)
    tab = i32(table)
    ref = R.plan(table, lens, new, free, count, rows, pt)
    plan = P8.plan_pages(tab, i32(lens), i32(new), i32(free), i32([count]), rows, pt)
    got = (plan.q_start, plan.q_lens, plan.kv_lens, plan.slots, plan.positions)
    for name, x, y in zip(("q_start", "q_lens", "kv_lens", "slots", "positions"), got, ref):
        assert x.tolist() == y, name
    assert plan.free_count.item() == ref[5]
    assert tab.tolist() == ref[6]
    return plan


@pytest.mark.parametrize("lens,new,pt,rows", [
    ([0], [1], 64, 1),
    ([63, 64, 65, 0], [1, 1, 1, 1], 64, 4),
    ([5, 0, 200], [0, 0, 0], 64, 0),
    ([5, 0, 200], [0, 7, 0], 128, 10),
    ([1000, 1, 64], [300, 0, 2000], 256, 2305),
    ([0, 2047, 2048, 4096], [2048, 1, 2049, 3], 2048, 5000),
])
def test_plan_small(lens, new, pt, rows):
    _check_plan(lens, new, pt, rows)


def test_plan_refusals():
    # rows end behind the buffer: that request and the ones behind it get nothing
    p = _check_plan([10, 10, 10], [5, 6, 7], 64, 12)
    assert p.q_lens.tolist() == [5, 6, 0]
    # pages end behind the table
    p = _check_plan([64, 60, 0], [65, 4, 1], 64, 100, width=2)
    assert p.q_lens.tolist() == [0, 4, 1]
    # the pool runs out: no page for requests 1 and 2, request 3 needs none
    p = _check_plan([0, 64, 64, 10], [64, 65, 1, 1], 64, 200, spare=1)
    assert p.q_lens.tolist() == [64, 0, 0, 1]
    # negative counts are none; a batch of nothing
    _check_plan([3, 4], [-2, 5], 64, 8)
    _check_plan([0, 0], [0, 0], 64, 3, spare=0)


@pytest.mark.parametrize("B,rows,seed", [(1, 5000, 1), (7, 300, 2), (130, 4096, 3), (300, 9000, 4),
                                         (2049, 2049, 5), (5000, 20000, 6), (1024, 1024, 7)])
def test_plan_random(B, rows, seed):
    rng = random.Random(seed)
    lens = [rng.choice([0, 1, 63, 64, rng.randrange(700)]) for _ in range(B)]
    new = [rng.choice([0, 1, 1, rng.randrange(1 + 2 * rows // B)]) for _ in range(B)]
    _check_plan(lens, new, 64, rows, spare=rng.choice([None, B // 2]), seed=seed)


def test_plan_longest_request():
    """A request holds up to 2^31 - 64 tokens: one that would pass them is not served."""
    pt, width = 2048, 1 << 20
    table = torch.zeros(2, width, dtype=torch.int32, device=DEV)
    lens, new = i32([2 ** 31 - 70, 2 ** 31 - 70]), i32([7, 6])
    plan = P8.plan_pages(table, lens, new, i32([5, 6]), i32([2]), 13, pt)
    assert plan.q_lens.tolist() == [0, 6] and plan.free_count.item() == 2
    assert plan.kv_lens.tolist() == [2 ** 31 - 70, 2 ** 31 - 64]
    assert plan.positions.tolist() == [0] * 7 + list(range(2 ** 31 - 70, 2 ** 31 - 64))


def test_plan_no_requests():
    plan = P8.plan_pages(torch.zeros(0, 4, dtype=torch.int32, device=DEV), i32([]), i32([]),
                         i32([0, 1]), i32([2]), 5, 64)
    assert plan.slots.tolist() == [-1] * 5 and plan.positions.tolist() == [0] * 5
    assert plan.free_count.item() == 2 and plan.q_start.tolist() == [0]


def test_release_and_take_again():
    pt = 64
    st = P8.PagedKV8Store(4, 1, 64, 20, DEV, page_tokens=pt, pages_per_seq=6)
    rng = random.Random(3)
    lens = [0] * 4
    for step in range(30):
        new = [rng.choice([0, 1, 40, 90]) for _ in range(4)]
        plan = st.plan(i32(new), 400)
        got = plan.q_lens.tolist()
        for b in range(4):
            assert got[b] in (0, new[b])
            lens[b] += got[b]
        done = [rng.random() < 0.3 for _ in range(4)]
        st.release(torch.tensor(done, dtype=torch.bool, device=DEV))
        lens = [0 if f else n for f, n in zip(done, lens)]
        assert st.lens.tolist() == lens
        count = st.free_count.item()
        held = [st.table[b, p].item() for b in range(4) for p in range(-(-lens[b] // pt))]
        # every page is free or held, once
        assert sorted(held + st.free[:count].tolist()) == list(range(20)), step


# ------------------------------------------------- append and read

def _raw(store, slots):
    """(keys, values) codes' values and scales at slots, by indexing on the CPU."""
    n, nb = store.pt, store.pt // 16
    dt = R.CODE[store.code]
    k = store.kpool.view(torch.int8).cpu()
    v = store.vpool.view(torch.int8).cpu()
    page, o = slots // n, slots % n
    kc = k[page, :, o].view(dt).double()
    vc = v[page, :, o // 16, :, o % 16].contiguous().view(dt).double()
    return kc, vc, store.kscale.cpu()[page, :, o // 16], store.vscale.cpu()[page, :, o // 16]


def _slots(store, b, T):
    t = torch.arange(T)
    return store.table[b].cpu().long()[t // store.pt] * store.pt + t % store.pt


def _same(store, cache, lens):
    for b, T in enumerate(lens):
        if T == 0:
            continue
        slots = _slots(store, b, T)
        kc, vc, ks, vs = _raw(store, slots)
        for half, (c, s) in enumerate(((kc, ks), (vc, vs))):
            assert torch.equal(c, cache.val[b][half]), (b, half)
            assert torch.equal(s, cache.scale[b][half].repeat_interleave(16, 0)[:T]), (b, half)
        for dt in (F32, BF16):
            k, v = store.read(slots.to(DEV), out_dtype=dt)
            for half, x in enumerate((k, v)):
                assert torch.equal(x.cpu(), cache.values(b, half).float().to(dt)), (b, half, dt)


def _rows_of(gen, rows, H, d, dtype, loud=1.0):
    """Rows cut out of one projection's output (strided), with outlier channels."""
    x = torch.randn(rows, (2 * H + 1) * d, generator=gen) * loud
    x[:, ::17] *= 6
    x = x.to(dtype).to(DEV)
    return (x[:, :H * d].unflatten(1, (H, d)), x[:, H * d:2 * H * d].unflatten(1, (H, d)))


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("d,H,dtype,pt", [(128, 8, BF16, 256), (96, 3, F16, 64), (64, 1, F32, 128),
                                          (64, 5, BF16, 64), (128, 2, F32, 2048)])
def test_append_exact(code, d, H, dtype, pt):
    gen = torch.Generator().manual_seed(d + H)
    B = 4
    st = P8.PagedKV8Store(B, H, d, 40 if pt < 2048 else 6, DEV, page_tokens=pt, code=code)
    cache, lens = R.Cache(B, H, d, code), [0] * B
    # ragged steps: whole blocks, single tokens, runs across blocks and pages, none;
    # the loudness grows and falls, so scales stand and grow
    for step, (new, loud) in enumerate([([16, 1, 70, 0], 1.0), ([1, 1, 1, 1], 0.1),
                                        ([3, 40, 0, 130], 5.0), ([1, 1, 1, 1], 30.0),
                                        ([15, 7, 64, 17], 1e-3), ([1, 2, 3, 4], 200.0)]):
        rows = sum(new) + 3
        plan = st.plan(i32(new), rows)
        k, v = _rows_of(gen, rows, H, d, dtype, loud)
        st.append(k, v, plan)
        at = 0
        for b, n in enumerate(new):
            if n:
                cache.append(b, k[at:at + n], v[at:at + n])
            at += n
            lens[b] += n
        _same(st, cache, lens)


@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_append_special_values(code):
    """Zeros, tiny and huge values, infinities, NaN, values on the border of two codes."""
    H, d = 1, 64
    top = R.TOP[code]
    x = torch.zeros(16 * 9, H, d)
    x[16:32, 0, 0] = 1e-45                                   # a scale at the floor
    x[32:48] = torch.randn(16, H, d, generator=torch.Generator().manual_seed(1)) * 1e37
    x[48, 0, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")])
    x[48, 0, 3:5] = torch.tensor([1.0, -2.0])
    x[64, 0, 0] = float("inf")                               # nothing finite but 0
    x[80:96] = (torch.arange(16 * d).view(16, 1, d) % 255 - 127) / 2.0   # halves: ties
    x[80, 0, 0] = top
    x[96:112] = torch.randn(16, H, d, generator=torch.Generator().manual_seed(2)) * 2.0 ** -130
    x[112:128] = torch.linspace(-top, top, 16 * d).view(16, 1, d)
    x[128:144, 0, ::2] = -0.0
    st = P8.PagedKV8Store(1, H, d, 3, DEV, page_tokens=64, code=code)
    cache = R.Cache(1, H, d, code)
    plan = st.plan(i32([144]), 144)
    st.append(x.to(DEV), x.flip(0).contiguous().to(DEV), plan)
    cache.append(0, x, x.flip(0))
    _same(st, cache, [144])


def test_append_border_codes():
    """fp32 values next to the border of two codes: the product's rounding does not decide."""
    g = torch.Generator().manual_seed(5)
    H, d = 2, 128
    x = torch.randn(64, H, d, generator=g)
    for code in ("int8", "fp8"):
        s = R.scale_of(x.view(4, 16, H, d).abs().amax((1, 3)), code)
        per = s.repeat_interleave(16, 0)[..., None]
        y = x.double() / per.double()
        half = (y.floor() + 0.5 if code == "int8" else R.nearest(y, code) * (1 + 2.0 ** -4)) * per
        near = half.float()
        near = torch.where(torch.rand(near.shape, generator=g) < 0.5, near,
                           torch.nextafter(near, near * 2))
        keep = near.abs() < x.view(4, 16, H, d).abs().amax((1, 3)).repeat_interleave(16, 0)[..., None]
        z = torch.where(keep & (torch.rand(near.shape, generator=g) < 0.9), near, x)
        z = torch.where(x.abs() >= x.view(4, 16, H, d).abs().amax((1, 3)).repeat_interleave(
            16, 0)[..., None], x, z)
        st = P8.PagedKV8Store(1, H, d, 1, DEV, page_tokens=64, code=code)
        cache = R.Cache(1, H, d, code)
        st.append(z.to(DEV), z.to(DEV), st.plan(i32([64]), 64))
        cache.append(0, z, z)
        _same(st, cache, [64])


@pytest.mark.parametrize("code,dtype,d", [("int8", BF16, 96), ("fp8", F16, 64), ("int8", F32, 128)])
def test_append_unaligned_and_read_in_any_order(code, dtype, d):
    """Rows at odd addresses and strides; slots read back out of order, twice, or not there."""
    H, T = 3, 150
    gen = torch.Generator().manual_seed(d)
    wide = torch.randn(T, 2 * H * d + 5, generator=gen).to(dtype).to(DEV)
    k = wide[:, 1:1 + H * d].unflatten(1, (H, d))
    v = wide[:, 2 + H * d:2 + 2 * H * d].unflatten(1, (H, d))
    st = P8.PagedKV8Store(1, H, d, 4, DEV, page_tokens=64, code=code)
    cache = R.Cache(1, H, d, code)
    for a, b in ((0, 70), (70, 71), (71, T)):
        st.append(k[a:b], v[a:b], st.plan(i32([b - a]), b - a))
        cache.append(0, k[a:b], v[a:b])
    _same(st, cache, [T])
    # a head_dim that is not the last axis in memory
    st2 = P8.PagedKV8Store(1, H, d, 4, DEV, page_tokens=64, code=code)
    kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    for a, b in ((0, 70), (70, 71), (71, T)):
        st2.append(kt[a:b], vt[a:b], st2.plan(i32([b - a]), b - a))
    for a, b in zip(st.pools().values(), st2.pools().values()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    order = torch.randint(0, T, (6000,), generator=gen)
    slots = _slots(st, 0, T)[order]
    slots[::50] = -1
    for n in (1, 40, 700, 6000):
        ks, vs = st.read(slots[:n].to(DEV))
        for half, x in enumerate((ks, vs)):
            want = cache.values(0, half)[order[:n]].float()
            want[::50] = 0
            assert torch.equal(x.cpu(), want), (n, half)


def test_append_chunks_of_all_sizes():
    """The rules that deal rows to waves: the same cache from one call and from many."""
    H, d, T = 2, 64, 4500
    x = torch.randn(2, T, H, d, device=DEV)
    ref = P8.PagedKV8Store(3, H, d, 80, DEV, page_tokens=64, pages_per_seq=80)
    split = [1500, 17, T - 1517]
    ref.append(x[0], x[1], ref.plan(i32(split), T))
    st = P8.PagedKV8Store(3, H, d, 80, DEV, page_tokens=64, pages_per_seq=80)
    plan = st.plan(i32(split), T)
    for rows in (13, 600):                       # cut at block ends: a block's rows stay together
        st.kscale.zero_()
        st.vscale.zero_()
        at = 0
        while at < T:
            end = min(T, at + rows)
            while end < T and plan.slots[end].item() % 16:
                end += 1
            P8.append_kv8(x[0, at:end], x[1, at:end], plan.slots[at:end].contiguous(),
                          **st.pools())
            at = end
        for a, b in zip(ref.pools().values(), st.pools().values()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), rows


def test_append_skips_bad_slots_and_keeps_the_rest():
    st = P8.PagedKV8Store(1, 2, 64, 2, DEV, page_tokens=64)
    before = [t.view(torch.uint8).clone() for t in st.pools().values()]
    x = torch.randn(4, 2, 64, device=DEV)
    bad = torch.tensor([-1, 128, 1 << 40, -(1 << 40)], device=DEV)
    P8.append_kv8(x, x, bad, **st.pools())
    for a, b in zip(before, st.pools().values()):
        assert torch.equal(a, b.view(torch.uint8))
    k, v = st.read(bad)
    assert not k.any() and not v.any()
    # a run in the middle of a page touches its own blocks alone
    P8.append_kv8(x, x, torch.tensor([70, 71, -1, 96], device=DEV), **st.pools())
    k = st.kpool.cpu()
    touched = k.view(2 * 2 * 64, 64).abs().sum(-1).nonzero().view(-1).tolist()
    assert touched == sorted([(2 + h) * 64 + o for h in range(2) for o in (6, 7, 32)])
    assert (st.kscale > 0).cpu().nonzero().tolist() == [[1, h, b] for h in range(2) for b in (0, 2)]


# --------------------------------------------------------------- attention

def _filled(B, H, d, lens, code, pt, dtype=BF16, seed=0, loud=1.0, pages=None):
    gen = torch.Generator().manual_seed(seed)
    pages = pages or sum(-(-t // pt) for t in lens) + 1
    st = P8.PagedKV8Store(B, H, d, pages, DEV, page_tokens=pt, code=code)
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    st.free.copy_(i32(order))
    # what lies behind the cached tokens is garbage, NaN codes among it
    for t in (st.kpool, st.vpool):
        t.view(torch.uint8).fill_(0x7f)
    st.kscale.fill_(float("nan"))
    st.vscale.fill_(float("inf"))
    cache = R.Cache(B, H, d, code)
    rows = max(sum(lens), 1)
    k, v = _rows_of(gen, rows, H, d, dtype, loud)
    st.append(k, v, st.plan(i32(lens), rows))
    at = 0
    for b, n in enumerate(lens):
        if n:
            cache.append(b, k[at:at + n], v[at:at + n])
        at += n
    return st, cache


def _check_attention(st, cache, lens, q_lens, G, q_dtype, out_dtype, causal=True, scale=None,
                     seed=0, gaps=(), loud=1.0, max_q_len=None):
    """Ragged queries (gaps: requests whose rows are there but not served)."""
    gen = torch.Generator().manual_seed(seed + 100)
    B, H, d = st.B, st.H, st.d
    start = [0]
    for n in q_lens:
        start.append(start[-1] + n)
    rows = start[-1] + 2
    served = [0 if b in gaps else n for b, n in enumerate(q_lens)]
    wide = (torch.randn(rows, H * G + 1, d, generator=gen) * loud).to(q_dtype).to(DEV)
    q = wide[:, :H * G]                                     # rows and heads strided
    out = torch.full((rows, H * G, d), 7.0, dtype=out_dtype, device=DEV)
    got = P8.attention_kv8(q, **st.pools(), table=st.table, kv_lens=i32(lens),
                           q_start=i32(start), q_lens=i32(served), causal=causal, scale=scale,
                           max_q_len=max_q_len, out=out)
    assert got is out
    out = out.cpu()
    qc = q.cpu()
    sc = 1.0 / math.sqrt(d) if scale is None else scale
    # weights and fp32 queries reach the product in fp16 pairs (22 bits); 16-bit results
    # take weights of 11 bits
    w = 2.0 ** -22 if out_dtype == F32 else 2.0 ** -11
    for b in range(B):
        rows_b = slice(start[b], start[b] + served[b])
        o, tol = R.attend(qc[rows_b].double(), cache.values(b, 0)[:lens[b]],
                          cache.values(b, 1)[:lens[b]], sc,
                          lens[b] - served[b] if causal else None, 2.0 ** -22, w,
                          HALF[out_dtype])
        x = out[rows_b].double()
        assert torch.isfinite(x).all(), b
        bad = (x - o).abs() > tol
        assert not bad.any(), (b, (x - o).abs().max().item(), tol[bad].min().item())
        assert (out[start[b] + served[b]:start[b + 1]] == 7.0).all(), b
    assert (out[start[-1]:] == 7.0).all()


CASES = [
    # lens, q_lens, G, d, H, code, pt
    ([1], [1], 1, 128, 1, "int8", 64),
    ([512], [1], 4, 128, 8, "int8", 256),
    ([0, 1, 2, 63, 64, 65], [1] * 6, 2, 64, 2, "int8", 64),
    ([700, 33, 1500], [1, 1, 1], 7, 64, 2, "fp8", 128),
    ([100, 17, 300], [3, 2, 4], 5, 96, 3, "fp8", 64),
    ([130, 5, 0, 90], [130, 5, 0, 31], 4, 128, 2, "int8", 64),
    ([300, 290, 40], [40, 1, 40], 8, 64, 1, "int8", 64),
    ([10, 40], [25, 41], 3, 96, 1, "int8", 64),           # more queries than tokens
    ([257, 256, 255, 129], [257, 1, 100, 64], 2, 128, 1, "fp8", 256),
]


@pytest.mark.parametrize("q_dtype,out_dtype", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attention(case, q_dtype, out_dtype):
    lens, q_lens, G, d, H, code, pt = case
    st, cache = _filled(len(lens), H, d, lens, code, pt)
    _check_attention(st, cache, lens, q_lens, G, q_dtype, out_dtype)


@pytest.mark.parametrize("case", CASES[3:8], ids=[str(i) for i in range(3, 8)])
def test_attention_not_causal(case):
    lens, q_lens, G, d, H, code, pt = case
    st, cache = _filled(len(lens), H, d, lens, code, pt, dtype=F32, seed=4)
    _check_attention(st, cache, lens, q_lens, G, F32, F32, causal=False, scale=0.2)


def test_attention_gaps_and_hints():
    """Requests that are not served keep their rows; a wrong bound of the longest
    request changes nothing."""
    lens, q_lens = [300, 20, 500, 64], [90, 1, 4, 33]
    st, cache = _filled(4, 2, 128, lens, "int8", 64, seed=5)
    for hint in (None, 1, 90, 1000):
        _check_attention(st, cache, lens, q_lens, 4, BF16, F32, gaps=(1, 3), max_q_len=hint)
        _check_attention(st, cache, lens, q_lens, 4, BF16, BF16, gaps=(0,), max_q_len=hint)


@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_attention_scales_of_any_size(code):
    """Block scales that differ by many powers of two, large scores, tiny values."""
    for loud, seed in ((1e-12, 1), (40.0, 2), (1e12, 3)):
        lens, q_lens = [200, 77], [1, 40]
        st, cache = _filled(2, 1, 64, lens, code, 64, dtype=F32, seed=seed, loud=loud)
        _check_attention(st, cache, lens, q_lens, 4, F32, F32, scale=0.5 / loud)
    gen = torch.Generator().manual_seed(9)
    T, H, d = 240, 1, 64
    st = P8.PagedKV8Store(1, H, d, 4, DEV, page_tokens=64, code=code)
    cache = R.Cache(1, H, d, code)
    k = torch.randn(T, H, d, generator=gen)
    v = torch.randn(T, H, d, generator=gen) * torch.exp2(
        torch.randint(-30, 30, (T // 16, 1, 1), generator=gen).float()).repeat_interleave(16, 0)
    v[32:48] = 0
    k[64:80] = 0
    st.append(k.to(DEV), v.to(DEV), st.plan(i32([T]), T))
    cache.append(0, k, v)
    _check_attention(st, cache, [T], [1], 4, F32, F32)
    _check_attention(st, cache, [T], [70], 2, F32, F32)


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("size", [2.0 ** -92, 2.0 ** 118])
def test_attention_values_at_the_scales_ends(code, size):
    """All values near the smallest scale, or near the largest fp32: the weights' sum holds."""
    gen = torch.Generator().manual_seed(11)
    T, H, d = 20000, 1, 64
    st = P8.PagedKV8Store(1, H, d, 80, DEV, code=code)
    k = torch.randn(T, H, d, generator=gen)
    v = torch.randn(T, H, d, generator=gen) * size
    st.append(k.to(DEV), v.to(DEV), st.plan(i32([T]), T))
    kd, vd = (x.cpu().double() for x in st.read(_slots(st, 0, T).to(DEV)))
    for Q in (1, 30):
        q = torch.randn(Q, 4, d, generator=gen)
        x = P8.attention_kv8(q.to(DEV), **st.pools(), table=st.table, kv_lens=st.lens)
        o, tol = R.attend(q.double(), kd, vd, 0.125, None, 2.0 ** -22, 2.0 ** -22, HALF[F32])
        assert ((x.cpu().double() - o).abs() <= tol + 2.0 ** -149).all(), Q


def test_attention_uniform_rows():
    """Without q_start: rows split evenly, the same result as with it."""
    st, cache = _filled(3, 2, 128, [90, 5, 200], "int8", 64, seed=6)
    lens = i32([90, 5, 200])
    for Q in (1, 4, 5, 60):
        q = torch.randn(3 * Q, 8, 128, device=DEV)
        a = P8.attention_kv8(q, **st.pools(), table=st.table, kv_lens=lens, causal=True)
        b = P8.attention_kv8(q, **st.pools(), table=st.table, kv_lens=lens, causal=True,
                             q_start=i32([0, Q, 2 * Q, 3 * Q]))
        assert torch.equal(a, b), Q


def test_attention_bad_pages_are_left_out():
    """Table entries that name no page: their tokens carry no weight."""
    st, cache = _filled(1, 1, 64, [192], "int8", 64, seed=7)
    st.table[0, 1] = st.num_pages + 5
    q = torch.randn(40, 4, 64, device=DEV)
    keep = torch.cat([torch.arange(64), torch.arange(128, 192)])
    k, v = cache.values(0, 0)[keep], cache.values(0, 1)[keep]
    for Q in (1, 40):
        x = P8.attention_kv8(q[:Q], **st.pools(), table=st.table, kv_lens=i32([192]))
        o, tol = R.attend(q[:Q].cpu().double(), k, v, 0.125, None, 2.0 ** -22, 2.0 ** -22,
                          HALF[F32])
        assert ((x.cpu().double() - o).abs() <= tol).all(), Q
    st.table[0, :3] = -1
    for Q in (1, 40):
        x = P8.attention_kv8(q[:Q], **st.pools(), table=st.table, kv_lens=i32([192]))
        assert not x.any(), Q


@pytest.mark.parametrize("q_dtype", [F32, F16, BF16])
def test_attention_unaligned(q_dtype):
    """Queries and results at odd addresses, queries with odd row strides."""
    st, cache = _filled(2, 2, 64, [100, 300], "int8", 64, seed=8)
    for q_lens in ([1, 2], [40, 1]):
        rows = sum(q_lens)
        wide = torch.randn(rows, 8 * 64 + 3, device=DEV).to(q_dtype)
        q = wide[:, 1:1 + 8 * 64].unflatten(1, (8, 64))
        out = torch.zeros(rows * 8 * 64 + 1, dtype=q_dtype, device=DEV)[1:].view(rows, 8, 64)
        args = dict(**st.pools(), table=st.table, kv_lens=i32([100, 300]),
                    q_start=i32([0, q_lens[0], rows]), causal=True)
        P8.attention_kv8(q, **args, out=out)
        ref = P8.attention_kv8(q.contiguous(), **args, out_dtype=q_dtype)
        assert torch.equal(out, ref)
        # a transposed head_dim is taken too
        t = q.transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(P8.attention_kv8(t, **args, out_dtype=q_dtype), ref)


@pytest.mark.parametrize("B,pt", [(65, 64), (300, 64), (600, 128)])
def test_attention_of_many_requests(B, pt):
    """More requests than a wave has lanes, some empty, some not served, some cut."""
    rng = random.Random(B)
    lens = [rng.choice([0, 1, 17, 64, rng.randrange(200)]) for _ in range(B)]
    lens[B // 2], lens[B - 1] = 3000, 1700
    q_lens = [rng.choice([0, 1, 1, 1, 2]) for _ in range(B)]
    st, cache = _filled(B, 1, 64, lens, "int8", pt, seed=B)
    gaps = tuple(b for b in range(B) if rng.random() < 0.1)
    _check_attention(st, cache, lens, q_lens, 4, BF16, F32, gaps=gaps, max_q_len=2)
    for b in range(0, B, 9):
        q_lens[b] = rng.choice([9, 33, 50])
    _check_attention(st, cache, lens, q_lens, 4, BF16, F32, gaps=gaps)


def test_attention_of_the_most_requests():
    """16,000 requests give, bit by bit, what 64 at a time give (nothing is cut)."""
    B, pt, G, d = 16000, 64, 2, 64
    gen = torch.Generator(DEV).manual_seed(1)
    st = P8.PagedKV8Store(B, 1, d, B, DEV, page_tokens=pt, pages_per_seq=1)
    for t in (st.kpool, st.vpool):
        t.copy_(torch.randint(-127, 128, t.shape, generator=gen, device=DEV, dtype=torch.int8))
    for t in (st.kscale, st.vscale):
        t.uniform_(0.001, 0.1, generator=gen)
    st.table.copy_(torch.randperm(B, generator=gen, device=DEV).view(B, 1))
    kv = torch.randint(0, pt + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
    for wide in (False, True):
        n = torch.randint(0, 3, (B,), generator=gen, device=DEV, dtype=torch.int32)
        if wide:
            n[::50] = 40
        start = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
        start[1:] = n.cumsum(0)
        at = start.tolist()
        q = torch.randn(at[-1], G, d, generator=gen, device=DEV).to(BF16)
        args = dict(**st.pools(), causal=True, out_dtype=BF16)
        out = P8.attention_kv8(q, table=st.table, kv_lens=kv, q_start=start, **args)
        for b in range(0, B, 64):
            part = P8.attention_kv8(q[at[b]:at[b + 64]], table=st.table[b:b + 64],
                                    kv_lens=kv[b:b + 64], q_start=start[b:b + 65] - at[b], **args)
            assert torch.equal(out[at[b]:at[b + 64]], part), (wide, b)
    with pytest.raises(ValueError, match="16000"):
        P8.attention_kv8(q, table=st.table.new_zeros(B + 1, 1), kv_lens=kv.new_zeros(B + 1),
                         q_start=start.new_zeros(B + 2), **args)


@pytest.mark.parametrize("Q", [1, 40])
def test_attention_of_the_longest_request(Q):
    """2^31 - 64 tokens, all but the first and the last page's on no page of the pool."""
    pt, n = 2048, 4096 - 64
    st, cache = _filled(1, 1, 64, [n], "int8", pt, seed=14)
    first, last = st.table[0, :2].tolist()
    table = torch.full((1, 1 << 20), -1, dtype=torch.int32, device=DEV)
    table[0, 0], table[0, -1] = first, last
    q = torch.randn(Q, 1, 64, generator=torch.Generator().manual_seed(3)).to(BF16)
    args = dict(**st.pools(), table=table, out_dtype=BF16)
    x = P8.attention_kv8(q.to(DEV), kv_lens=i32([2 ** 31 - 64]), **args)
    o, tol = R.attend(q.double(), cache.values(0, 0)[:n], cache.values(0, 1)[:n], 0.125, None,
                      2.0 ** -22, 2.0 ** -11, HALF[BF16])
    assert ((x.cpu().double() - o).abs() <= tol).all()
    # lengths past that count as it
    assert torch.equal(P8.attention_kv8(q.to(DEV), kv_lens=i32([2 ** 31 - 1]), **args), x)


@pytest.mark.parametrize("H,G,Q", [(1, 1, 1), (3, 11, 1), (5, 16, 2), (1, 32, 1), (1, 71, 1),
                                   (16, 1, 40), (7, 3, 200)])
def test_attention_head_layouts(H, G, Q):
    """Cut requests at odd head counts and wide groups."""
    lens = [2500, 1100]
    st, cache = _filled(2, H, 64, lens, "fp8", 256, seed=H)
    _check_attention(st, cache, lens, [Q, min(Q, 3)], G, F16, F32)


@pytest.mark.parametrize("lens,q_lens,G", [([1500] * 4, [400] * 4, 7),
                                           ([3000, 40, 1100], [30, 40, 90], 16)])
def test_attention_of_cut_chunks(lens, q_lens, G):
    """Long tiles of a few chunks: as many pieces as the card holds at once, joined."""
    st, cache = _filled(len(lens), 1, 64, lens, "int8", 256, seed=21)
    _check_attention(st, cache, lens, q_lens, G, BF16, F32)


def test_attention_of_nothing():
    """Requests that hold no token, short and long: zeros, and rows of no request stay."""
    st = P8.PagedKV8Store(3, 2, 96, 4, DEV, page_tokens=64)
    st.kscale.fill_(float("nan"))
    st.vscale.fill_(float("nan"))
    for q_lens in ([1, 0, 2], [40, 1, 70], [0, 0, 0]):
        rows = sum(q_lens) + 3
        start = [0, q_lens[0], q_lens[0] + q_lens[1], sum(q_lens)]
        q = torch.randn(rows, 6, 96, device=DEV, dtype=F16)
        out = torch.full((rows, 6, 96), 3.0, device=DEV)
        P8.attention_kv8(q, **st.pools(), table=st.table, kv_lens=st.lens, q_start=i32(start),
                         causal=True, out=out)
        assert not out[:sum(q_lens)].any() and (out[sum(q_lens):] == 3.0).all()
        # the result that the call makes itself: zeros there too
        assert not P8.attention_kv8(q, **st.pools(), table=st.table, kv_lens=st.lens,
                                    q_start=i32(start), causal=True).any()


def test_attention_lengths_off_the_table():
    """Lengths below 0 count as 0, lengths behind the table as its tokens."""
    st, cache = _filled(2, 1, 64, [128, 64], "int8", 64, seed=9)
    table = st.table[:, :2].contiguous()
    for Q in (1, 40):
        q = torch.randn(2 * Q, 4, 64, device=DEV)
        x = P8.attention_kv8(q, **st.pools(), table=table, kv_lens=i32([1000, -5]))
        y = P8.attention_kv8(q, **st.pools(), table=table, kv_lens=i32([128, 0]))
        assert torch.equal(x, y) and not x[Q:].any() and x[:Q].any()


@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_attention_scales_behind_the_tokens(code):
    """Scales of blocks behind the cached tokens may be anything: subnormal ones too, whose
    inverse is infinite."""
    lens = [70, 1, 130]
    st, cache = _filled(3, 2, 64, lens, code, 256, seed=12)
    unset = st.vscale.isinf()                 # _filled's mark of what no append wrote
    assert unset.view(-1, 4).any(1).logical_and(~unset.view(-1, 4).all(1)).any()
    for Q in (1, 40):
        q = torch.randn(3 * Q, 4, 64, device=DEV)
        args = dict(**st.pools(), table=st.table, kv_lens=i32(lens))
        ref = P8.attention_kv8(q, **args)
        assert ref.isfinite().all() and ref.view(3, -1).any(1).all()
        for x in (2.0 ** -149, 2.0 ** -130, -1.0, 3e38, float("nan")):
            st.vscale[unset] = x
            st.kscale[unset] = x
            assert torch.equal(P8.attention_kv8(q, **args), ref), x
        st.vscale[unset] = float("inf")


def test_attention_nan_stays_in_its_row():
    """A query of NaN or infinities leaves the other queries as they are."""
    st, cache = _filled(1, 1, 64, [150], "int8", 64, seed=10)
    for Q in (4, 40):
        q = torch.randn(Q, 4, 64, device=DEV)
        args = dict(**st.pools(), table=st.table, kv_lens=i32([150]), causal=True)
        ref = P8.attention_kv8(q, **args)
        bad = q.clone()
        bad[1, 2, 5], bad[2, 0, 0] = float("nan"), float("inf")
        x = P8.attention_kv8(bad, **args)
        same = torch.ones(Q, 4, dtype=torch.bool)
        same[1, 2] = same[2, 0] = False
        assert torch.equal(x[same], ref[same]) and x[1, 2].isnan().all()


def test_offsets_past_32_bits():
    """A request in the last pages of pools of more than 4 GiB."""
    H, d, pt = 8, 128, 2048
    pages = (5 << 30) // (H * d * pt)
    st = P8.PagedKV8Store(2, H, d, pages, DEV, page_tokens=pt, pages_per_seq=2)
    # handed out first: the pool's last two pages, then its first two
    st.free[-4:] = i32([0, 1, pages - 2, pages - 1])
    x = torch.randn(2, 2100, H, d, device=DEV, dtype=BF16)
    st.append(x[0], x[1], st.plan(i32([2100, 0]), 2100))
    st.append(x[0], x[1], st.plan(i32([0, 2100]), 2100))
    assert st.table[:, :2].tolist() == [[pages - 1, pages - 2], [1, 0]]
    for a, b in zip(st.read(_slots(st, 0, 2100).to(DEV)), st.read(_slots(st, 1, 2100).to(DEV))):
        assert torch.equal(a, b) and a.any()
    for Q in (1, 100):
        q = torch.randn(Q, 4 * H, d, device=DEV, dtype=BF16)
        out = P8.attention_kv8(torch.cat([q, q]), **st.pools(), table=st.table, kv_lens=st.lens,
                               causal=True)
        assert torch.equal(out[:Q], out[Q:]) and out.any()


def test_attention_long_against_itself():
    """A long cache, cut into many pieces, against one softmax over all of it."""
    T, H, d = 40000, 2, 128
    gen = torch.Generator(device=DEV).manual_seed(3)
    st = P8.PagedKV8Store(1, H, d, 160, DEV)
    for t0 in range(0, T, 10000):
        x = torch.randn(2, 10000, H, d, generator=gen, device=DEV)
        st.append(x[0], x[1], st.plan(i32([10000]), 10000))
    k, v = st.read(_slots(st, 0, T).to(DEV))
    for Q, dt in ((1, F32), (3, F32), (50, F32)):
        q = torch.randn(Q, 4 * H, d, generator=gen, device=DEV)
        x = P8.attention_kv8(q, **st.pools(), table=st.table, kv_lens=st.lens, causal=True)
        o, tol = R.attend(q.cpu().double(), k.cpu().double(), v.cpu().double(),
                          1 / math.sqrt(d), T - Q, 2.0 ** -22, 2.0 ** -22, HALF[F32])
        assert ((x.cpu().double() - o).abs() <= tol).all(), Q


# ----------------------------------------------------- as a program uses it

def _run_steps(st, steps, G, seed):
    """A serving loop; the outputs of all steps and the cache that they built."""
    gen = torch.Generator().manual_seed(seed)
    B, H, d = st.B, st.H, st.d
    cache, lens, outs = R.Cache(B, H, d, st.code), [0] * B, []
    for new, done in steps:
        rows = sum(new) + 1
        qkv = torch.randn(rows, (G + 2) * H * d, generator=gen).to(BF16).to(DEV)
        q = qkv[:, :G * H * d].unflatten(1, (G * H, d))
        k = qkv[:, G * H * d:(G + 1) * H * d].unflatten(1, (H, d))
        v = qkv[:, (G + 1) * H * d:].unflatten(1, (H, d))
        plan = st.plan(i32(new), rows, max_q_len=max(new))
        st.append(k, v, plan)
        out = st.attention(q, plan, out_dtype=BF16)
        at = 0
        for b, n in enumerate(new):
            if n:
                cache.append(b, k[at:at + n], v[at:at + n])
                lens[b] += n
                o, tol = R.attend(q[at:at + n].cpu().double(), cache.values(b, 0),
                                  cache.values(b, 1), 1 / math.sqrt(d), lens[b] - n, 2.0 ** -22,
                                  2.0 ** -11, HALF[BF16])
                err = (out[at:at + n].cpu().double() - o).abs()
                assert (err <= tol).all(), (new, b)
            at += n
        outs.append(out)
        if any(done):
            st.release(torch.tensor(done, dtype=torch.bool, device=DEV))
            for b, f in enumerate(done):
                if f:
                    cache.val[b] = [x[:0] for x in cache.val[b]]
                    cache.scale[b] = [x[:0] for x in cache.scale[b]]
                    lens[b] = 0
    return outs


STEPS = [([40, 0, 7, 100], [0] * 4), ([1, 60, 1, 1], [0, 0, 1, 0]), ([1, 1, 33, 1], [0] * 4),
         ([1, 1, 1, 1], [1, 0, 0, 1]), ([20, 1, 1, 64], [0] * 4), ([1, 1, 1, 1], [0] * 4)]


@pytest.mark.parametrize("code,d,H,G", [("int8", 128, 2, 4), ("fp8", 64, 1, 7)])
def test_serving_loop(code, d, H, G):
    st = P8.PagedKV8Store(4, H, d, 9, DEV, page_tokens=64, code=code)
    _run_steps(st, STEPS, G, 11)


def test_serving_loop_on_another_stream():
    st = P8.PagedKV8Store(4, 2, 128, 9, DEV, page_tokens=64)
    a = _run_steps(st, STEPS, 4, 12)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        st = P8.PagedKV8Store(4, 2, 128, 9, DEV, page_tokens=64)
        b = _run_steps(st, STEPS, 4, 12)
    s.synchronize()
    for x, y, (new, _) in zip(a, b, STEPS):
        assert torch.equal(x[:sum(new)], y[:sum(new)])


def test_two_calls_at_once():
    """Attention on two streams at the same time: each as alone."""
    st, _ = _filled(3, 2, 128, [2000, 700, 1200], "int8", 64, seed=12)
    qs = [torch.randn(3, 8, 128, device=DEV, dtype=BF16), torch.randn(150, 8, 128, device=DEV)]
    args = dict(**st.pools(), table=st.table, kv_lens=i32([2000, 700, 1200]), causal=True)
    alone = [P8.attention_kv8(q, **args) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(P8.attention_kv8(qs[i], **args))
    torch.cuda.synchronize()
    for ref, outs in zip(alone, got):
        for x in outs:
            assert torch.equal(x, ref)


def test_captured_step():
    """A decode step as a graph: plan, append and attention replayed, against eager steps."""
    B, H, G, d, steps = 5, 2, 4, 128, 40
    def store():
        st = P8.PagedKV8Store(B, H, d, 12, DEV, page_tokens=64)
        gen = torch.Generator().manual_seed(1)
        lens = [50, 1, 64, 0, 130]
        rows = sum(lens)
        x = torch.randn(2, rows, H, d, generator=gen).to(DEV)
        st.append(x[0], x[1], st.plan(i32(lens), rows))
        return st
    eager, st = store(), store()
    new = torch.ones(B, dtype=torch.int32, device=DEV)
    q = torch.zeros(B, G * H, d, dtype=BF16, device=DEV)
    k, v = (torch.zeros(B, H, d, dtype=BF16, device=DEV) for _ in range(2))
    out = torch.zeros(B, G * H, d, dtype=BF16, device=DEV)
    # a first plan, which the captured step writes again, taken back
    plan = st.plan(new, B, max_q_len=1)
    st.lens.sub_(plan.q_lens)
    st.free_count.copy_(eager.free_count)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        P8.attention_kv8(q, **st.pools(), table=st.table, kv_lens=st.lens, max_q_len=1)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st.plan(new, B, max_q_len=1, out=plan)
        st.append(k, v, plan)
        st.attention(q, plan, out_dtype=BF16, out=out)
    gen = torch.Generator().manual_seed(2)
    for i in range(steps):
        x = torch.randn(3, B, G * H, d, generator=gen).to(BF16).to(DEV)
        if i % 3 == 1:
            new.copy_(i32([1, 0, 1, 1, 0]))      # some requests pause
        else:
            new.fill_(1)
        q.copy_(x[0])
        k.copy_(x[1, :, :H])
        v.copy_(x[2, :, :H])
        last = out.clone()
        g.replay()
        p = eager.plan(new, B, max_q_len=1)
        eager.append(x[1, :, :H], x[2, :, :H], p)
        # the same rows are served; a row that is not keeps the last step's values
        ref = eager.attention(x[0], p, out_dtype=BF16, out=last)
        torch.cuda.synchronize()
        assert torch.equal(eager.lens, st.lens) and torch.equal(eager.free_count, st.free_count)
        assert torch.equal(p.slots, plan.slots), i
        assert torch.equal(ref, out), i
    for a, b in zip(eager.pools().values(), st.pools().values()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_refusals():
    st = P8.PagedKV8Store(2, 2, 64, 4, DEV, page_tokens=64)
    pools = st.pools()
    x = torch.zeros(3, 2, 64, device=DEV)
    slots = torch.arange(3, device=DEV)
    q = torch.zeros(4, 4, 64, device=DEV)
    att = dict(table=st.table, kv_lens=st.lens)
    bad = [
        lambda: P8.plan_pages(st.table, st.lens.long(), st.lens, st.free, st.free_count, 1, 64),
        lambda: P8.plan_pages(st.table, st.lens, st.lens[:1], st.free, st.free_count, 1, 64),
        lambda: P8.plan_pages(st.table, st.lens, st.lens, st.free, st.free_count, 1, 96),
        lambda: P8.plan_pages(st.table, st.lens, st.lens, st.free, st.free_count, -1, 64),
        lambda: P8.plan_pages(st.table[:, ::2], st.lens, st.lens, st.free, st.free_count, 1, 64),
        lambda: st.plan(st.lens, 2, out=P8.PagePlan.empty(2, 2, DEV)),
        lambda: st.plan(st.lens, 2, out=st.plan(st.lens, 3)),
        lambda: P8.release_pages(st.table, st.lens, st.lens, st.free, st.free_count, 64),
        lambda: P8.append_kv8(x, x.half(), slots, **pools),
        lambda: P8.append_kv8(x[:, :1], x[:, :1], slots, **pools),
        lambda: P8.append_kv8(x, x, slots[:2], **pools),
        lambda: P8.append_kv8(x, x, slots.int(), **pools),
        lambda: P8.append_kv8(x.double(), x.double(), slots, **pools),
        lambda: P8.append_kv8(x, x, slots, **{**pools, "vscale": st.vscale[:1]}),
        lambda: P8.append_kv8(x, x, slots, **{**pools, "vpool": st.vpool.view(torch.uint8)}),
        lambda: P8.read_kv8(slots, **pools, out_dtype=torch.int8),
        lambda: P8.attention_kv8(q[:, :3], **pools, **att),
        lambda: P8.attention_kv8(q[:3], **pools, **att),
        lambda: P8.attention_kv8(q, **pools, **att, q_lens=st.lens),
        lambda: P8.attention_kv8(q, **pools, **att, q_start=st.lens),
        lambda: P8.attention_kv8(q, **pools, **att, out=torch.zeros(4, 4, 32, device=DEV)),
        lambda: P8.attention_kv8(q.double(), **pools, **att),
        lambda: P8.attention_kv8(q, **pools, table=st.table.long(), kv_lens=st.lens),
        lambda: P8.attention_kv8(q, **pools, **att, workspace=torch.zeros(0, dtype=torch.uint8,
                                                                          device=DEV)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(RuntimeError, match="GPU"):
        P8.append_kv8(x.cpu(), x, slots, **pools)
    # nothing to do is no error
    st.append(x[:0], x[:0], st.plan(i32([0, 0]), 0))
    assert st.read(slots[:0])[0].shape == (0, 2, 64)
    assert P8.attention_kv8(q[:0], **pools, **att).shape == (0, 4, 64)


@pytest.mark.parametrize("B", [6, 80])
def test_captured_chunks(B):
    """A batch of chunks and decode rows, cut requests among them, captured and replayed."""
    rng = random.Random(B)
    lens = [rng.randrange(1, 400) for _ in range(B)]
    lens[1], lens[B - 2] = 2500, 1800
    q_lens = [1 if b % 3 else min(lens[b], 60) for b in range(B)]
    st, _ = _filled(B, 2, 64, lens, "int8", 64, seed=B)
    start = [0]
    for n in q_lens:
        start.append(start[-1] + n)
    q = torch.zeros(start[-1], 8, 64, dtype=BF16, device=DEV)
    out = torch.zeros(start[-1], 8, 64, device=DEV)
    kv = i32(lens)
    args = dict(**st.pools(), table=st.table, kv_lens=kv, q_start=i32(start), causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        P8.attention_kv8(q, **args, out=out)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        P8.attention_kv8(q, **args, out=out)
    gen = torch.Generator(device=DEV).manual_seed(B)
    for i in range(6):
        q.copy_(torch.randn(q.shape, generator=gen, device=DEV))
        if i % 2:                               # shorter: other cuts, the same graph
            kv.copy_(i32([max(n, t // 2) for n, t in zip(q_lens, lens)]))
        else:
            kv.copy_(i32(lens))
        g.replay()
        torch.cuda.synchronize()
        ref = P8.attention_kv8(q, **args)
        assert torch.equal(out, ref), i
        assert ref.any()


def test_grow_keeps_the_cache():
    st = P8.PagedKV8Store(2, 1, 64, 2, DEV, page_tokens=64, pages_per_seq=1)
    cache = R.Cache(2, 1, 64, "int8")
    gen = torch.Generator().manual_seed(8)
    lens = [0, 0]
    for step in range(5):
        if step == 2:
            st.grow(7, 3)
        n = [30, 25] if step != 2 else [40, 0]
        x = torch.randn(2, sum(n), 1, 64, generator=gen).to(DEV)
        plan = st.plan(i32(n), sum(n))
        assert plan.q_lens.tolist() == n, step
        st.append(x[0], x[1], plan)
        cache.append(0, x[0, :n[0]], x[1, :n[0]])
        if n[1]:
            cache.append(1, x[0, n[0]:], x[1, n[0]:])
        lens = [a + b for a, b in zip(lens, n)]
    _same(st, cache, lens)


def test_engine_and_page_manager():
    """The engine interface, and a page manager of 8-bit layers, against plain attention."""
    gen = torch.Generator().manual_seed(4)
    B, H, G, d = 3, 2, 4, 128
    pm = QuashKVPageManager(H, d, QuashKVPageConfig(key_bits=8, value_bits=8),
                            torch.device(DEV))
    assert isinstance(pm.engine, P8.PagedKV8Engine)
    cache, T = R.Cache(B, H, d, "int8"), 0
    for S, dt in ((300, F32), (1, BF16), (1, F16), (250, torch.float64)):
        k, v = (torch.randn(B, H, S, d, generator=gen).to(dt).to(DEV) for _ in range(2))
        pm.compress_and_store(k, v)
        T += S
        for b in range(B):
            cache.append(b, k[b].transpose(0, 1), v[b].transpose(0, 1))
        assert pm.total_tokens == T
        for Q in (1, 33):
            q = torch.randn(B, H * G, Q, d, generator=gen).to(DEV)
            out = pm.attention(q).cpu().double()
            for b in range(B):
                o, tol = R.attend(q[b].cpu().double().transpose(0, 1), cache.values(b, 0),
                                  cache.values(b, 1), 1 / math.sqrt(d), None, 2.0 ** -22,
                                  2.0 ** -22, HALF[F32])
                assert ((out[b].transpose(0, 1) - o).abs() <= tol).all(), (S, Q, b)
    assert 1.9 < pm.compression_ratio() < 2.0
    assert pm.engine.actual_memory_bytes() == B * H * 2 * (T * d + 4 * -(-T // 16))
    with pytest.raises(ValueError, match="codebook"):
        pm.get_compressed_blocks()
    pages = pm.engine.store.num_pages
    pm.clear()
    with pytest.raises(ValueError, match="No compressed"):
        pm.attention(torch.randn(B, H, 1, d, device=DEV))
    assert pm.total_tokens == 0 and pm.engine.store.free_count.item() == pages
    k = torch.randn(1, H, 5, d, device=DEV)                  # another batch after clear()
    pm.compress_and_store(k, k)
    assert pm.attention(torch.randn(1, H, 1, d, device=DEV)).shape == (1, H, 1, d)
