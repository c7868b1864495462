"""Attention of groups that share a prefix (attention_kv8_shared) on the GPU: within the bounds
of tests/kv8_reference.py over forked requests' pages, and a serving loop of forks, plans, rotary
positions, appends, attention and releases as a program runs it, eager and captured."""

import math
import random

import pytest
import torch

import quashkv_amd as Q
from quashkv_amd import _native as N
from quashkv_amd import paged8 as P8
from quashkv_amd import rotary as rot
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


def shared(*args, **kw):
    """The call, sharing wherever two requests of a group see the prefix."""
    return P8.attention_kv8_shared(*args, always=True, **kw)


def _forked(groups, own, H, d, code, pt, seed=0, loud=1.0, fork=True):
    """A store of requests in groups: groups [(prefix, requests)], own[b] tokens behind the
    prefix; and their tokens.  The prefix is appended once, to the group's first request
    (through a template that is released), and forked.  What lies behind the tokens is garbage.
    fork=False: the prefix is appended to every request, pages shared by none."""
    gen = torch.Generator().manual_seed(seed)
    B = len(own)
    n = len(groups)
    prefix = [p for p, m in groups for _ in range(m)]
    prefix += [0] * (B - len(prefix))
    top = max(p + o for p, o in zip(prefix, own))
    pages = sum(-(-(p + o) // pt) + 1 for p, o in zip(prefix, own)) + sum(
        -(-p // pt) for p, _ in groups) + 2
    st = P8.PagedKV8Store(B + n, H, d, pages, DEV, page_tokens=pt, pages_per_seq=-(-top // pt) + 1,
                          code=code, sharing=True)
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    st.free.copy_(i32(order))
    for t in (st.kpool, st.vpool):
        t.view(torch.uint8).fill_(0x7f)
    st.kscale.fill_(float("nan"))
    st.vscale.fill_(float("inf"))
    cache = R.Cache(B + n, H, d, code)

    def bring(new):
        rows = max(sum(new), 1)
        k, v = ((torch.randn(rows, H, d, generator=gen) * loud).to(BF16).to(DEV) for _ in range(2))
        plan = st.plan(i32(new), rows)
        assert plan.q_lens.tolist() == new
        st.append(k, v, plan)
        at = 0
        for b, m in enumerate(new):
            if m:
                cache.append(b, k[at:at + m], v[at:at + m])
            at += m

    bring([0] * B + [p for p, _ in groups])
    src = [B + g for g, (_, m) in enumerate(groups) for _ in range(m)]
    assert st.fork(i32(src), i32(range(len(src)))).tolist() == [groups[s - B][0] for s in src]
    for b, s in enumerate(src):
        for half in (0, 1):
            cache.val[b][half] = cache.val[s][half].clone()
            cache.scale[b][half] = cache.scale[s][half].clone()
    done = torch.zeros(B + n, dtype=torch.bool, device=DEV)
    done[B:] = True
    st.release(done)
    bring(list(own) + [0] * n)
    return st, cache, [p + o for p, o in zip(prefix, own)]


def _starts(groups):
    s = [0]
    for _, m in groups:
        s.append(s[-1] + m)
    return s


def _check(st, cache, lens, groups, q_lens, G, q_dtype, out_dtype, causal=True, scale=None, seed=0,
           gaps=(), start=None, prefix=None, loud=1.0, guard=False, always=True):
    gen = torch.Generator().manual_seed(seed + 100)
    B, H, d = len(lens), st.H, st.d
    q_start = [0]
    for n in q_lens:
        q_start.append(q_start[-1] + n)
    rows = q_start[-1] + 2
    served = [0 if b in gaps else n for b, n in enumerate(q_lens)]
    wide = (torch.randn(rows, H * G + 1, d, generator=gen) * loud).to(q_dtype).to(DEV)
    q = wide[:, :H * G]
    out = torch.full((rows, H * G, d), 7.0, dtype=out_dtype, device=DEV)
    start = _starts(groups) if start is None else start
    prefix = [p for p, _ in groups] if prefix is None else prefix
    ws = None
    if guard:
        need = P8.attention_kv8_shared_workspace_bytes(B, len(prefix), rows, H * G, H, d)
        whole = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
        ws = whole[:need]
    got = P8.attention_kv8_shared(
        q, **st.pools(), table=st.table[:B], kv_lens=i32(lens), group_start=i32(start),
        prefix_lens=i32(prefix), q_start=i32(q_start), q_lens=i32(served), causal=causal,
        scale=scale, out=out, workspace=ws, always=always)
    assert got is out
    if guard:
        assert (whole[need:] == 0xA5).all()
    x, qc = out.cpu(), q.cpu()
    sc = 1.0 / math.sqrt(d) if scale is None else scale
    w = 2.0 ** -22 if out_dtype == F32 else 2.0 ** -11
    for b in range(B):
        rows_b = slice(q_start[b], q_start[b] + served[b])
        o, tol = R.attend(qc[rows_b].double(), cache.values(b, 0)[:lens[b]],
                          cache.values(b, 1)[:lens[b]], sc,
                          lens[b] - served[b] if causal else None, 2.0 ** -22, w, HALF[out_dtype])
        y = x[rows_b].double()
        assert torch.isfinite(y).all(), b
        bad = (y - o).abs() > tol
        assert not bad.any(), (b, (y - o).abs().max().item(), tol[bad].min().item())
        assert (x[q_start[b] + served[b]:q_start[b + 1]] == 7.0).all(), b
    assert (x[q_start[-1]:] == 7.0).all()
    return out


CASES = [
    # groups [(prefix, requests)], own tokens, q_lens, G, H, d, code, pt
    ([(128, 2)], [1, 1], [1, 1], 1, 1, 64, "int8", 64),
    ([(512, 4)], [1, 30, 64, 7], [1] * 4, 1, 8, 128, "int8", 256),
    ([(300, 9)], [3, 1, 17, 16, 1, 90, 2, 5, 1], [1] * 9, 4, 2, 128, "int8", 64),   # 36 rows: tall
    ([(1000, 3), (70, 2)], [5, 6, 7, 8, 9, 200], [1] * 6, 7, 2, 64, "fp8", 128),
    ([(200, 2), (64, 2), (63, 2), (130, 1)], [9] * 7 + [33], [1, 2, 3, 1, 1, 2, 4, 1], 3, 3, 96, "fp8", 64),
    ([(700, 3)], [150, 40, 130], [150, 40, 129], 2, 2, 128, "int8", 256),           # questions
    ([(330, 5)], [20, 70, 3, 40, 64], [20, 1, 3, 40, 64], 8, 1, 64, "int8", 64),
    ([(2500, 2)], [12, 1], [5, 1], 4, 1, 96, "int8", 1024),                         # cut prefix
    ([(256, 40)], [1] * 40, [1] * 40, 4, 2, 64, "fp8", 64),
]


@pytest.mark.parametrize("q_dtype,out_dtype", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attention(case, q_dtype, out_dtype):
    groups, own, q_lens, G, H, d, code, pt = case
    st, cache, lens = _forked(groups, own, H, d, code, pt)
    _check(st, cache, lens, groups, q_lens, G, q_dtype, out_dtype, guard=True)


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attention_by_the_rule(case):
    """Small calls, which go to the plain attention."""
    groups, own, q_lens, G, H, d, code, pt = case
    st, cache, lens = _forked(groups, own, H, d, code, pt, seed=2)
    _check(st, cache, lens, groups, q_lens, G, F16, F32, guard=True, always=False)


@pytest.mark.parametrize("groups,own,q_lens,G", [
    # behind a table too wide to count as small: groups that share and ones for which that does
    # not pay (short prefixes, two requests, requests of many rows), in one batch
    ([(1300, 6), (70, 5), (600, 2), (640, 3)], [5, 30, 1, 64, 7, 8, 9, 1, 1, 2, 3, 4, 5, 150, 130, 140],
     [1] * 13 + [150, 130, 140], 4),
    ([(900, 3), (900, 3)], [300, 280, 260, 60, 50, 40], [290, 270, 260, 41, 40, 40], 2),
])
def test_attention_by_the_rule_of_groups(groups, own, q_lens, G):
    st, cache, lens = _forked(groups, own, 2, 128, "int8", 64, seed=3)
    wide = torch.zeros(st.B, 40000, dtype=torch.int32, device=DEV)
    wide[:, :st.pages_per_seq] = st.table
    st.table = wide
    _check(st, cache, lens, groups, q_lens, G, BF16, F32, guard=True, always=False)
    _check(st, cache, lens, groups, q_lens, G, BF16, BF16, causal=False, always=False)


@pytest.mark.parametrize("case", CASES[2:8], ids=[str(i) for i in range(2, 8)])
def test_attention_not_causal(case):
    groups, own, q_lens, G, H, d, code, pt = case
    st, cache, lens = _forked(groups, own, H, d, code, pt, seed=4)
    _check(st, cache, lens, groups, q_lens, G, F32, F32, causal=False, scale=0.2)


def test_requests_that_do_not_see_the_prefix():
    """Chunks that begin inside the prefix, requests shorter than it, idle ones and ones without
    rows in this step: alone, wherever in the group they are."""
    groups, own = [(320, 6)], [4, 10, 100, 20, 5, 6]
    st, cache, lens = _forked(groups, own, 2, 64, "int8", 64, seed=5)
    # request 0 is idle, 1 holds a part of the prefix, 3's chunk begins inside the prefix
    lens = [0, 200, 420, 340, 325, 326]
    for q_lens in ([0, 1, 2, 100, 1, 1], [3, 1, 0, 340, 5, 1], [0, 0, 1, 1, 0, 0], [1, 1, 0, 0, 0, 1]):
        for causal in (True, False):
            _check(st, cache, lens, groups, q_lens, 3, F32, F32, causal=causal)
    _check(st, cache, lens, groups, [1, 1, 2, 30, 9, 1], 3, BF16, BF16, gaps=(2, 4))


def test_groups_at_the_ends_of_a_batch():
    """Requests before the first group and behind the last; empty groups; no group at all;
    prefixes of nothing, of less than is shared, and lengths that are no numbers of tokens."""
    groups, own = [(0, 2), (200, 3), (130, 2)], [40, 100, 5, 6, 7, 8, 9, 50]
    st, cache, lens = _forked(groups, own, 1, 128, "int8", 64, seed=6)
    ones = [1] * 8
    for start, prefix in (([2, 5, 7], [200, 130]), ([2, 2, 5, 5, 7, 7], [9, 200, 50, 130, 8]),
                          ([5, 7], [130]), ([2, 5], [128]), ([3, 5], [191]), ([0], []), ([8], []),
                          ([0, 2, 5, 7], [0, 64, -5])):
        _check(st, cache, lens, groups, ones, 4, F32, F32, start=start, prefix=prefix)


@pytest.mark.parametrize("groups,own", [
    ([(64, 0), (128, 2), (192, 0), (64, 0), (200, 3), (64, 0)], [1, 20, 3, 70, 5]),
    ([(128, 1)] * 30 + [(64, 2)] * 17 + [(64, 0)] * 17, [1 + i % 7 for i in range(64)]),
    ([(64, 0)] * 40 + [(128, 3), (64, 0), (192, 4)] + [(64, 0)] * 30, [4, 3, 2, 1, 90, 1, 2]),
])
def test_empty_groups(groups, own):
    """Groups without requests among the others and behind the last, up to 64 of both and more."""
    st, cache, lens = _forked(groups, own, 1, 64, "int8", 64)
    _check(st, cache, lens, groups, [1] * len(own), 2, F32, F32, guard=True)


def test_attention_is_the_plain_one():
    """Against attention_kv8 on the same tables, long prefixes cut into many parts."""
    B, H, G, d, prefix = 24, 2, 4, 128, 20000
    st = P8.PagedKV8Store(B, H, d, 700, DEV, page_tokens=64, pages_per_seq=340, sharing=True)
    gen = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(prefix, H, d, generator=gen, device=DEV).to(BF16) for _ in range(2))
    st.append(k, v, st.plan(i32([prefix] + [0] * (B - 1)), prefix))
    st.fork(i32([0] * (B - 1)), i32(range(1, B)))
    for Q in (1, 11):
        k, v = (torch.randn(B * Q, H, d, generator=gen, device=DEV) for _ in range(2))
        q = torch.randn(B * Q, H * G, d, generator=gen, device=DEV)
        plan = st.plan(i32([Q] * B), B * Q)
        st.append(k, v, plan)
        x = st.attention(q, plan, groups=(i32([0, B]), i32([prefix])))
        y = st.attention(q, plan)
        # both hold fp32 scores and sums over T tokens and 22-bit weights of values up to 5
        T = prefix + 12
        bound = 2 * 2 * 5 * (2.0 ** -20 + (4 * math.sqrt(T) + 8) * 2.0 ** -24 + 2.0 ** -22)
        assert float((x - y).abs().max()) <= bound, Q


@pytest.mark.parametrize("H,G,Q", [(1, 1, 1), (5, 3, 2), (32, 1, 1), (3, 16, 1), (2, 33, 3), (1, 71, 2),
                                   (300, 1, 1), (260, 2, 7)])
def test_head_layouts(H, G, Q):
    groups, own = [(192, 3)], [Q, Q + 5, 40]
    st, cache, lens = _forked(groups, own, H, 64, "int8", 64, seed=H)
    _check(st, cache, lens, groups, [Q] * 3, G, BF16, F32, guard=True)


def test_uniform_rows_and_outputs_made_here():
    groups, own = [(256, 4)], [9, 20, 33, 64]
    st, cache, lens = _forked(groups, own, 2, 64, "fp8", 64, seed=7)
    for Q in (1, 8):
        q = torch.randn(4 * Q, 6, 64, generator=torch.Generator().manual_seed(Q)).to(DEV)
        x = shared(q, **st.pools(), table=st.table[:4], kv_lens=i32(lens),
                                    group_start=i32([0, 4]), prefix_lens=i32([256]), causal=True)
        for b in range(4):
            o, tol = R.attend(q[b * Q:b * Q + Q].cpu().double(), cache.values(b, 0),
                              cache.values(b, 1), 0.125, lens[b] - Q, 2.0 ** -22, 2.0 ** -22,
                              HALF[F32])
            assert ((x[b * Q:b * Q + Q].cpu().double() - o).abs() <= tol).all(), (Q, b)
    # rows of no request are 0 in an output that the call makes
    y = shared(q, **st.pools(), table=st.table[:4], kv_lens=i32(lens),
                                group_start=i32([0, 4]), prefix_lens=i32([256]),
                                q_start=i32([0, 1, 2, 3, 4]), q_lens=i32([1, 0, 1, 1]))
    assert not y[1].any() and not y[4:].any() and y[0].any()


@pytest.mark.parametrize("q_dtype", [F32, F16, BF16])
def test_unaligned_queries(q_dtype):
    groups, own = [(128, 5)], [3, 4, 70, 1, 9]
    st, cache, lens = _forked(groups, own, 1, 96, "int8", 64, seed=8)
    for G, Q in ((2, 1), (7, 3)):
        base = torch.randn(5 * Q * G * 96 + 1, generator=torch.Generator().manual_seed(G)).to(q_dtype).to(DEV)
        q = base[1:].view(5 * Q, G, 96)
        args = dict(**st.pools(), table=st.table[:5], kv_lens=i32([n + 3 - 3 for n in lens]),
                    group_start=i32([0, 5]), prefix_lens=i32([128]))
        x = shared(q, **args)
        assert torch.equal(x, shared(q.clone(), **args))
        z = q.permute(2, 1, 0).contiguous().permute(2, 1, 0)      # heads innermost
        assert torch.equal(x, shared(z, **args))


def test_bad_pages_are_left_out():
    """Entries of the prefix, and of a request's own tokens, that name no page."""
    groups, own = [(256, 3)], [64, 70, 1]
    st, cache, lens = _forked(groups, own, 1, 64, "int8", 64, seed=9)
    st.table[0, 1] = st.num_pages
    st.table[1, 4] = -1
    keep = [torch.cat([torch.arange(64), torch.arange(128, 320)]),
            torch.cat([torch.arange(64), torch.arange(128, 256), torch.arange(320, 326)]),
            torch.cat([torch.arange(64), torch.arange(128, 257)])]
    for Q in (1, 20):
        q = torch.randn(3 * Q, 4, 64, generator=torch.Generator().manual_seed(Q)).to(DEV)
        x = shared(q, **st.pools(), table=st.table[:3], kv_lens=i32(lens),
                                    group_start=i32([0, 3]), prefix_lens=i32([256]))
        for b in range(3):
            o, tol = R.attend(q[b * Q:b * Q + Q].cpu().double(), cache.values(b, 0)[keep[b]],
                              cache.values(b, 1)[keep[b]], 0.125, None, 2.0 ** -22, 2.0 ** -22,
                              HALF[F32])
            assert ((x[b * Q:b * Q + Q].cpu().double() - o).abs() <= tol).all(), (Q, b)


def test_nan_stays_in_its_row():
    """The other rows stay within their bounds.  (Not the same bits: rows of a tile rescale
    their sums together, by a power that is rounded, when one of them needs it.)"""
    groups, own = [(192, 12)], [5] * 12
    st, cache, lens = _forked(groups, own, 2, 64, "int8", 64, seed=10)
    q = torch.randn(12, 8, 64, device=DEV)
    q[4, 3, 7] = float("nan")
    y = shared(q, **st.pools(), table=st.table[:12], kv_lens=i32(lens),
                                group_start=i32([0, 12]), prefix_lens=i32([192])).cpu()
    assert torch.isnan(y[4, 3]).all()
    for b in range(12):
        x = torch.nan_to_num(q[b:b + 1].cpu()).double()
        o, tol = R.attend(x, cache.values(b, 0), cache.values(b, 1), 0.125, None, 2.0 ** -22,
                          2.0 ** -22, HALF[F32])
        for h in range(8):
            if (b, h) != (4, 3):
                assert ((y[b, h].double() - o[0, h]).abs() <= tol[0, h]).all(), (b, h)


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1.0, 1e30])
def test_value_scales_and_blocks_of_zeros(size):
    """A prefix of zero values before own ones of any size, and the other way round."""
    for zero_first in (True, False):
        B, H, d = 3, 1, 64
        st = P8.PagedKV8Store(B, H, d, 20, DEV, page_tokens=64, pages_per_seq=6, sharing=True)
        gen = torch.Generator().manual_seed(2)
        k, v = torch.randn(2, 128, H, d, generator=gen)
        k2, v2 = torch.randn(2, 3 * 20, H, d, generator=gen)
        v, v2 = (v * 0, v2 * size) if zero_first else (v * size, v2 * 0)
        st.append(k.to(DEV), v.to(DEV), st.plan(i32([128, 0, 0]), 128))
        st.fork(i32([0, 0]), i32([1, 2]))
        plan = st.plan(i32([20] * 3), 60)
        st.append(k2.to(DEV), v2.to(DEV), plan)
        cache = R.Cache(B, H, d, "int8")
        for b in range(B):
            cache.append(b, k, v)
            cache.append(b, k2[20 * b:20 * b + 20], v2[20 * b:20 * b + 20])
        for G in (2, 40):
            q = torch.randn(B, G, d, generator=gen)
            x = shared(q.to(DEV), **st.pools(), table=st.table, kv_lens=st.lens,
                                        group_start=i32([0, 3]), prefix_lens=i32([128]))
            for b in range(B):
                o, tol = R.attend(q[b:b + 1].double(), cache.values(b, 0), cache.values(b, 1),
                                  0.125, None, 2.0 ** -22, 2.0 ** -22, HALF[F32])
                assert ((x[b:b + 1].cpu().double() - o).abs() <= tol).all(), (zero_first, G, b)


@pytest.mark.parametrize("B,m", [(1030, 5), (4100, 2), (2000, 2000)])
def test_many_requests(B, m):
    """More requests, and groups, than the plan's workgroup has threads: against attention_kv8."""
    H, d, pt = 1, 64, 64
    n = min(B // m, 2048)
    gen = torch.Generator(device=DEV).manual_seed(B)
    rng = random.Random(B)
    whole, P = 2, 2 * n + 2 * B
    table = torch.zeros(B, 5, dtype=torch.int32)
    order = torch.randperm(P, generator=torch.Generator().manual_seed(1)).int()
    for b in range(B):
        g = b // m
        first = order[2 * g:2 * g + 2] if g < n else order[2 * n + 2 * b - 2:2 * n + 2 * b]
        table[b, :2] = first
        table[b, 2:4] = order[2 * n + 2 * b:2 * n + 2 * b + 2]
    pools = dict(kpool=torch.randint(-127, 128, (P, H, pt, d), generator=gen, device=DEV).to(torch.int8),
                 vpool=torch.randint(-127, 128, (P, H, pt // 16, d, 16), generator=gen, device=DEV).to(torch.int8),
                 kscale=0.01 * torch.rand(P, H, pt // 16, generator=gen, device=DEV) + 1e-4,
                 vscale=0.01 * torch.rand(P, H, pt // 16, generator=gen, device=DEV) + 1e-4)
    lens = i32([rng.choice([0, 128, 129, 200, 256, 60]) for _ in range(B)])
    q_lens = [rng.choice([0, 1, 1, 1, 2]) for _ in range(B)]
    start = [0]
    for x in q_lens:
        start.append(start[-1] + x)
    q = torch.randn(start[-1], 2, d, generator=gen, device=DEV)
    args = dict(q=q, **pools, table=table.to(DEV), kv_lens=lens, q_start=i32(start),
                q_lens=i32(q_lens), causal=True)
    x = shared(**args, group_start=i32([m * g for g in range(n + 1)]),
                                prefix_lens=i32([whole * pt] * n))
    y = P8.attention_kv8(**args)
    # 256 tokens, values up to 1.3: as in test_attention_is_the_plain_one
    assert float((x - y).abs().max()) <= 4 * 1.3 * (2.0 ** -18 + 72 * 2.0 ** -24)


@pytest.mark.parametrize("B,m,H,G,d", [(65, 65, 1, 1, 64), (90, 4, 4, 9, 96), (250, 250, 4, 2, 128),
                                       (300, 5, 4, 9, 64), (520, 40, 8, 4, 128), (700, 7, 4, 16, 64),
                                       (1000, 1000, 2, 1, 96), (1000, 45, 2, 3, 64)])
def test_many_tiles(B, m, H, G, d):
    """Batches beyond a wave's lanes, one item a thread of the plan, with 4, 2 or 1 waves for each tile of
    requests' own tokens: against attention_kv8."""
    pt = 64
    n = min(B // m, 2048)
    gen = torch.Generator(device=DEV).manual_seed(B)
    rng = random.Random(B)
    whole, P = 2, 2 * n + 2 * B
    table = torch.zeros(B, 5, dtype=torch.int32)
    order = torch.randperm(P, generator=torch.Generator().manual_seed(1)).int()
    for b in range(B):
        g = b // m
        first = order[2 * g:2 * g + 2] if g < n else order[2 * n + 2 * b - 2:2 * n + 2 * b]
        table[b, :2] = first
        table[b, 2:4] = order[2 * n + 2 * b:2 * n + 2 * b + 2]
    pools = dict(kpool=torch.randint(-127, 128, (P, H, pt, d), generator=gen, device=DEV).to(torch.int8),
                 vpool=torch.randint(-127, 128, (P, H, pt // 16, d, 16), generator=gen, device=DEV).to(torch.int8),
                 kscale=0.01 * torch.rand(P, H, pt // 16, generator=gen, device=DEV) + 1e-4,
                 vscale=0.01 * torch.rand(P, H, pt // 16, generator=gen, device=DEV) + 1e-4)
    lens = i32([rng.choice([0, 128, 129, 200, 256, 60]) for _ in range(B)])
    q_lens = [rng.choice([0, 1, 1, 1, 2]) for _ in range(B)]
    start = [0]
    for x in q_lens:
        start.append(start[-1] + x)
    q = torch.randn(start[-1], H * G, d, generator=gen, device=DEV)
    args = dict(q=q, **pools, table=table.to(DEV), kv_lens=lens, q_start=i32(start),
                q_lens=i32(q_lens), causal=True)
    x = shared(**args, group_start=i32([m * g for g in range(n + 1)]),
                                prefix_lens=i32([whole * pt] * n))
    y = P8.attention_kv8(**args)
    # as in test_many_requests
    assert float((x - y).abs().max()) <= 4 * 1.3 * (2.0 ** -18 + 72 * 2.0 ** -24)


def test_attention_of_nothing():
    st = P8.PagedKV8Store(2, 1, 64, 4, DEV, page_tokens=64)
    args = dict(**st.pools(), table=st.table, kv_lens=st.lens, group_start=i32([0, 2]),
                prefix_lens=i32([64]))
    x = shared(torch.ones(2, 3, 64, device=DEV), **args)
    assert not x.any()
    x = shared(torch.ones(0, 3, 64, device=DEV), **args, q_start=i32([0, 0, 0]))
    assert x.shape == (0, 3, 64)


def test_unsound_arrays_stay_in_bounds():
    """Starts that do not ascend, groups and rows beyond the batch: results of no meaning, the
    guard behind the workspace and the rows beyond the output untouched."""
    B, H, d = 6, 1, 64
    groups, own = [(128, 6)], [5] * 6
    st, cache, lens = _forked(groups, own, H, d, "int8", 64, seed=11)
    q = torch.randn(12, 40, d, device=DEV)
    whole = torch.full((14, 40, d), 7.0, device=DEV)
    need = P8.attention_kv8_shared_workspace_bytes(B, 2, 12, 40, H, d)
    box = torch.full((need + 65536,), 0xA5, dtype=torch.uint8, device=DEV)
    for start, q_start, q_lens in (([4, 2, 9], [0, 2, 4, 6, 8, 10, 12], None),
                                   ([-3, 3, 1 << 30], [0, 2, 4, 6, 8, 10, 12], None),
                                   ([0, 3, 6], [5, 1, 9, -4, 30, 2, 0], None),
                                   ([0, 3, 6], [0, 0, 0, 0, 0, 0, 12], [12] * 6),
                                   ([0, 6, 6], [0, 2, 4, 6, 8, 10, 1 << 30], [1 << 30] * 6)):
        shared(q, **st.pools(), table=st.table[:B],
                                kv_lens=i32(lens), group_start=i32(start),
                                prefix_lens=i32([128, 128]), q_start=i32(q_start),
                                q_lens=None if q_lens is None else i32(q_lens), out=whole[:12],
                                workspace=box[:need])
        assert (box[need:] == 0xA5).all() and (whole[12:] == 7.0).all(), (start, q_start)


def test_offsets_past_32_bits():
    """A prefix and own tokens in pages beyond 2^32 bytes of a pool."""
    P, H, d, pt = 18000, 8, 128, 256
    st = P8.PagedKV8Store(2, H, d, P, DEV, page_tokens=pt, pages_per_seq=4, sharing=True)
    st.free.copy_(torch.arange(P, dtype=torch.int32, device=DEV))     # the highest first
    gen = torch.Generator().manual_seed(3)
    k, v = torch.randn(2, 300, H, d, generator=gen)
    st.append(k.to(DEV), v.to(DEV), st.plan(i32([300, 0]), 300))
    st.fork(i32([0]), i32([1]))
    cache = R.Cache(2, H, d, "int8")
    for b in range(2):
        cache.append(b, k, v)
    assert int(st.table[:, :2].min()) >= P - 3
    _check(st, cache, [300, 300], [(300, 2)], [1, 1], 2, BF16, F32)


# ------------------------------------------------------------------- steps

def _serve(st, G, steps, seed, turns, share, out_dtype=F32):
    """n-best sampling: prompts, forks, decode steps of plan, rotary, append and attention,
    releases; yields each step's results."""
    rng = random.Random(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, H, d = st.B, st.H, st.d
    prompt = 150
    prefix = 0
    for step in range(steps):
        if step % 12 == 0:
            st.release()
            new = [prompt] + [0] * (B - 1)
        else:
            new = [1 if rng.random() < 0.9 else 0 for _ in range(B)]
        rows = sum(new) + 3
        q = torch.randn(rows, H * G, d, generator=gen, device=DEV)
        k, v = (torch.randn(rows, H, d, generator=gen, device=DEV) for _ in range(2))
        plan = st.plan(i32(new), rows)
        q, k = rot.rotary(q, k, plan.positions, turns)
        st.append(k, v, plan)
        out = torch.zeros(rows, H * G, d, dtype=out_dtype, device=DEV)
        if share:
            shared(q, **st.pools(), table=st.table, kv_lens=plan.kv_lens, group_start=i32([0, B]),
                   prefix_lens=i32([prefix]), q_start=plan.q_start, q_lens=plan.q_lens, causal=True,
                   out=out)
            yield out
        else:
            groups = (i32([0, B]), i32([prefix])) if step % 2 else None
            yield st.attention(q, plan, out_dtype=out_dtype, out=out, groups=groups)
        if step % 12 == 0:
            assert st.fork(i32([0] * (B - 1)), i32(range(1, B))).tolist() == [prompt] * (B - 1)
            prefix = prompt
        if step % 5 == 4:
            st.compact()
        if step % 12 == 11:
            prefix = 0


def test_serving_loop():
    """Shared and plain attention over the same steps, and a store whose requests each hold the
    prompt themselves."""
    turns = Q.rotary_turns(Q.rotary_frequencies(64), DEV)
    make = lambda: P8.PagedKV8Store(6, 2, 64, 40, DEV, page_tokens=64, pages_per_seq=5, sharing=True)
    a, b = make(), make()
    for x, y in zip(_serve(a, 4, 40, 1, turns, True), _serve(b, 4, 40, 1, turns, False)):
        # values up to 5, at most 170 tokens (see test_attention_is_the_plain_one)
        assert float((x - y).abs().max()) <= 4 * 5 * (2.0 ** -19 + 60 * 2.0 ** -24)
    for x, y in zip(a.pools().values(), b.pools().values()):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert a.free_count.item() == b.free_count.item()


def test_two_calls_at_once():
    """Two streams, each with its own workspace, beside each other."""
    turns = Q.rotary_turns(Q.rotary_frequencies(64), DEV)
    make = lambda: P8.PagedKV8Store(6, 2, 64, 40, DEV, page_tokens=64, pages_per_seq=5, sharing=True)
    want = [x.clone() for x in _serve(make(), 4, 12, 3, turns, True)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    runs = [_serve(make(), 4, 12, 3, turns, True) for _ in streams]
    got = [[], []]
    for _ in want:
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(next(runs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, y) for x, y in zip(got[i], want)), i


def test_captured_step():
    """A fork, a decode step and a release as one graph, replayed against eager steps: the state
    moves on as theirs does."""
    B, H, G, d = 5, 2, 4, 128
    turns = Q.rotary_turns(Q.rotary_frequencies(d), DEV)

    def store():
        st = P8.PagedKV8Store(B, H, d, 30, DEV, page_tokens=64, pages_per_seq=6, sharing=True)
        x = torch.randn(2, 200, H, d, generator=torch.Generator().manual_seed(1)).to(DEV)
        st.append(x[0], x[1], st.plan(i32([200] + [0] * (B - 1)), 200))
        return st

    src, dst = i32([0, 0, 0]), i32([1, 2, 4])
    new = torch.ones(B, dtype=torch.int32, device=DEV)
    done = torch.tensor([False, True, False, False, True], device=DEV)
    groups = (i32([0, B]), i32([200]))
    q = torch.zeros(B, H * G, d, dtype=BF16, device=DEV)
    k, v = (torch.zeros(B, H, d, dtype=BF16, device=DEV) for _ in range(2))
    out = torch.zeros(B, H * G, d, dtype=BF16, device=DEV)

    def step(st, plan, out):
        granted = st.fork(src, dst)
        plan = st.plan(new, B, max_q_len=1, out=plan)
        a, b = rot.rotary(q, k, plan.positions, turns)
        st.append(b, v, plan)
        shared(a, **st.pools(), table=st.table, kv_lens=plan.kv_lens, group_start=groups[0],
               prefix_lens=groups[1], q_start=plan.q_start, q_lens=plan.q_lens, causal=True, out=out)
        st.release(done)
        st.compact()
        return granted, plan

    eager, st, warm = store(), store(), store()
    _, plan = step(warm, None, out.clone())          # (what a first call sets up)
    plan = st.plan(torch.zeros_like(new), B, max_q_len=1)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        granted, _ = step(st, plan, out)
    gen = torch.Generator().manual_seed(2)
    ref = out.clone()
    ep = eager.plan(torch.zeros_like(new), B, max_q_len=1)
    for i in range(12):
        x = torch.randn(3, B, H * G, d, generator=gen).to(BF16).to(DEV)
        q.copy_(x[0])
        k.copy_(x[1, :, :H])
        v.copy_(x[2, :, :H])
        g.replay()
        got, _ = step(eager, ep, ref)
        torch.cuda.synchronize()
        assert torch.equal(got, granted) and torch.equal(ref, out), i
        for name in ("table", "lens", "free", "free_count", "shares", "kscale", "vscale"):
            assert torch.equal(getattr(eager, name), getattr(st, name)), (i, name)
        for a, b in zip(eager.pools().values(), st.pools().values()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i


def test_refusals():
    st = P8.PagedKV8Store(3, 1, 64, 4, DEV, page_tokens=64)
    q = torch.zeros(3, 2, 64, device=DEV)
    ok = dict(q=q, **st.pools(), table=st.table, kv_lens=st.lens, group_start=i32([0, 3]),
              prefix_lens=i32([0]))
    P8.attention_kv8_shared(**ok)
    for bad in (dict(group_start=i32([0])), dict(group_start=i32([0, 3]).long()),
                dict(prefix_lens=i32([[0]])), dict(prefix_lens=i32([0]).float()),
                dict(q=q[:2]), dict(q=q[:, :, :32]), dict(kv_lens=st.lens.long()),
                dict(q_lens=i32([1, 1, 1])), dict(out=torch.zeros(3, 2, 32, device=DEV)),
                dict(workspace=torch.zeros(64, dtype=torch.uint8, device=DEV)),
                dict(workspace=torch.zeros(1 << 24, device=DEV)), dict(q=q.double()),
                dict(group_start=i32([0] * 2050), prefix_lens=i32([0] * 2049))):
        with pytest.raises(ValueError):
            P8.attention_kv8_shared(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="GPU"):
        P8.attention_kv8_shared(**{**ok, "prefix_lens": torch.zeros(1, dtype=torch.int32)})
