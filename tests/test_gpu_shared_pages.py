"""Shared pages of the 8-bit cache on the GPU -- forks, releases by the last holder, compaction,
page copies -- against their definitions (tests/shared_reference.py), exactly; and rotary
positions within bounds derived there."""

import random

import pytest
import torch

import quashkv_amd as Q
from quashkv_amd import _native as N
from quashkv_amd import paged8 as P8
from quashkv_amd import rotary as rot
from tests import shared_reference as S

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


class Books:
    """Page tables on both sides: lists, and tensors on the device."""

    def __init__(self, lens, pt, spare, width=None, seed=0):
        rng = random.Random(seed)
        need = [S.held(n, pt) for n in lens]
        width = width or max(need + [1])
        P = sum(need) + spare
        ids = list(range(P))
        rng.shuffle(ids)
        table = [[rng.choice([-3, 0, P + 9]) for _ in range(width)] for _ in lens]
        for b, n in enumerate(need):
            for c in range(n):
                table[b][c] = ids.pop()
        self.pt, self.P, self.count = pt, P, len(ids)
        self.table, self.lens, self.shares = table, list(lens), [0] * P
        self.free = ids + [-5] * (P - len(ids))
        self.d = dict(table=i32(table).view(len(lens), width), lens=i32(lens), free=i32(self.free),
                      free_count=i32([self.count]), shares=i32(self.shares))

    def same(self, **want):
        for k, x in want.items():
            setattr(self, k, x)
        for k in ("table", "lens", "free", "shares"):
            assert self.d[k].tolist() == getattr(self, k), k
        assert self.d["free_count"].item() == self.count

    def fork(self, src, dst, tokens=None):
        ref = S.fork(self.table, self.lens, src, dst, tokens, self.free, self.count, self.shares,
                     self.pt)
        d = self.d
        p = P8.fork_pages(d["table"], d["lens"], i32(src), i32(dst),
                          None if tokens is None else i32(tokens), d["free"], d["free_count"],
                          d["shares"], self.pt)
        for k in ("granted", "src_pages", "dst_pages", "copy_tokens"):
            assert getattr(p, k).tolist() == ref[k], k
        self.same(**{k: ref[k] for k in ("table", "lens", "shares", "count")})
        return ref["granted"]

    def release(self, done):
        ref = S.release(self.table, self.lens, done, self.free, self.count, self.shares, self.pt)
        d = self.d
        P8.release_pages(d["table"], d["lens"], torch.tensor(done, dtype=torch.bool, device=DEV),
                         d["free"], d["free_count"], self.pt, shares=d["shares"])
        self.same(**ref)

    def compact(self, shares=True):
        ref = S.compact(self.table, self.lens, self.free, self.count, self.shares, self.pt)
        d = self.d
        p = P8.compact_pages(d["table"], d["lens"], d["free"], d["free_count"], self.pt,
                             shares=d["shares"] if shares else None)
        for k in ("src_pages", "dst_pages", "remap"):
            assert getattr(p, k).tolist() == ref[k], k
        assert p.moves.item() == ref["moves"]
        if not shares:
            ref["shares"] = self.shares
        self.same(**{k: ref[k] for k in ("table", "free", "count", "shares")})

    def sound(self):
        """Every page is free once, or held by one more than its shares."""
        n = [0] * self.P
        for b, t in enumerate(self.lens):
            for p in self.table[b][:S.held(t, self.pt)]:
                n[p] += 1
        for p in self.free[:self.count]:
            assert n[p] == 0
            n[p] = -1
        assert all(x == -1 or x == s + 1 for x, s in zip(n, self.shares))
        assert all(s == 0 for x, s in zip(n, self.shares) if x == -1)


# ------------------------------------------------------------------- forks

def test_fork_small():
    b = Books([200, 0, 64, 0, 0, 0, 7], 64, 4)
    assert b.fork([0, 2, 6], [1, 3, 4]) == [200, 64, 7]       # parts, whole pages alone, no whole page
    assert b.fork([1], [5], [130]) == [130]                   # of a fork, behind a part of it
    b.sound()


@pytest.mark.parametrize("copies", [1, 3])
def test_fork_refusals(copies):
    """(three times the calls: more forks than one workgroup takes with their tables)"""
    b = Books([200, 0, 64, 0, 0, 0, 7] + [0] * 20, 64, 9)
    src = [0, 0, -1, 7 + 20, 0, 3, 2, 0, 5] * copies
    dst = [2, 0, 1, 1, 7 + 20, 4, 3, 3, -9] * copies
    got = b.fork(src, dst)
    # held by tokens; itself; no request (four); of an empty request; granted; named before
    assert got[:9] == [-1, -1, -1, -1, -1, 0, 64, -1, -1] and set(got[9:]) <= {-1}
    b.sound()


def test_fork_tokens():
    b = Books([100, 0, 0, 0, 0, 0], 64, 8)
    assert b.fork([0] * 5, [1, 2, 3, 4, 5], [0, -4, 63, 64, 1000]) == [0, 0, 63, 64, 100]
    b.sound()


@pytest.mark.parametrize("spare", [0, 1, 3])
def test_fork_out_of_pages(spare):
    # forks 0, 2, 3 and 4 need a page each, fork 1 needs none
    b = Books([70, 128, 0, 0, 0, 0, 0], 64, spare)
    got = b.fork([0, 1, 0, 0, 0], [2, 3, 4, 5, 6])
    assert got == [70 if spare > 0 else -1, 128] + [70 if spare > k else -1 for k in (1, 2, 3)]
    b.sound()


def test_fork_longer_lengths_than_the_table():
    b = Books([64, 0], 64, 2)
    b.lens[0] = 200
    b.d["lens"][0] = 200
    assert b.fork([0], [1]) == [64]


@pytest.mark.parametrize("B,F,pt,seed", [(40, 7, 64, 0), (40, 30, 128, 1), (700, 600, 64, 2),
                                         (3000, 2500, 256, 3), (16000, 16000, 64, 4)])
def test_fork_and_release_random(B, F, pt, seed):
    rng = random.Random(seed)
    lens = [rng.choice([0, 0, 1, pt, rng.randrange(6 * pt)]) for _ in range(B)]
    b = Books(lens, pt, B // 3, width=7, seed=seed)
    src = [rng.randrange(-1, B + 1) for _ in range(F)]
    dst = [rng.randrange(B) for _ in range(F)]
    b.fork(src, dst, [rng.choice([0, 1, 10 ** 6, rng.randrange(6 * pt)]) for _ in range(F)])
    b.sound()
    for share in (0.3, 0.0, 0.7, 1.0):
        b.release([rng.random() < share for _ in range(B)])
        b.sound()
    assert b.count == b.P


def test_release_order_and_many_holders():
    """A page of many holders goes back with the last, at the place of the last entry."""
    b = Books([150] + [0] * 20, 64, 25)
    b.fork([0] * 20, list(range(1, 21)))
    b.release([False] + [True] * 19 + [False])
    assert b.shares[b.table[0][0]] == 1
    b.release([True] + [False] * 19 + [True])
    b.sound()
    assert b.count == b.P


def test_release_of_unsound_tables():
    """A page named too often is given back once; entries that name no page are left out."""
    b = Books([192, 128], 64, 3)
    b.table[0][1] = b.table[0][0]
    b.table[1][0] = -1
    b.table[1][1] = b.P + 3
    b.d["table"].copy_(i32(b.table))
    b.release([True, True])
    assert b.count == 3 + 2


def test_release_is_the_plain_one_where_nothing_is_shared():
    x, y = Books([300, 0, 65, 64], 64, 5, seed=3), Books([300, 0, 65, 64], 64, 5, seed=3)
    done = torch.tensor([True, True, False, True], device=DEV)
    for b, shares in ((x, x.d["shares"]), (y, None)):
        P8.release_pages(b.d["table"], b.d["lens"], done, b.d["free"], b.d["free_count"], 64,
                         shares=shares)
    for k in x.d:
        assert torch.equal(x.d[k], y.d[k]), k


# ------------------------------------------------------------------- compaction

@pytest.mark.parametrize("B,pt,spare,seed", [(1, 64, 0, 0), (1, 64, 1, 1), (5, 64, 31, 2),
                                             (40, 128, 20, 3), (40, 64, 400, 4),
                                             (900, 64, 5000, 5)])
def test_compact(B, pt, spare, seed):
    rng = random.Random(seed)
    lens = [rng.choice([0, 1, pt, rng.randrange(6 * pt)]) for _ in range(B)]
    lens[0] = 3 * pt - 1
    b = Books(lens, pt, spare, seed=seed)
    empty = [i for i, n in enumerate(lens) if n == 0]
    b.fork([0] * len(empty), empty)
    b.release([rng.random() < 0.4 for _ in lens])
    b.compact()
    b.sound()
    assert all(p < b.P - b.count for i, t in enumerate(b.lens)
               for p in b.table[i][:S.held(t, pt)])
    b.compact()                       # nothing to move
    b.fork([0], [1] if B > 1 else [0])
    b.release([True] * B)
    b.compact()
    assert b.free == list(range(b.P - 1, -1, -1))


def test_compact_without_shares_or_requests():
    b = Books([100, 300, 20], 64, 9, seed=8)
    b.release([False, True, False])
    b.compact(shares=False)
    b.sound()
    p = P8.compact_pages(torch.zeros(0, 3, dtype=torch.int32, device=DEV), i32([]), i32([2, 0]),
                         i32([1]), 64)       # a pool of two pages, page 2 of them none
    assert p.moves.item() == 0 and p.remap.tolist() == [0, 1]
    one = i32([0])
    P8.compact_pages(i32([[0]]), i32([5]), one, i32([0]), 64)


@pytest.mark.parametrize("P", [600_000, 1 << 20])
def test_compact_of_a_large_pool(P):
    gen = torch.Generator().manual_seed(1)
    order = torch.randperm(P, generator=gen).int()
    used = P // 3
    table = order[:used].view(1, used).to(DEV)
    free = torch.zeros(P, dtype=torch.int32)
    free[:P - used] = order[used:]
    p = P8.compact_pages(table, i32([used * 64]), free.to(DEV), i32([P - used]), 64)
    src = order[:used][order[:used] >= used].sort().values
    dst = order[used:][order[used:] < used].sort().values
    n = src.numel()
    assert p.moves.item() == n == dst.numel()
    assert torch.equal(p.src_pages[:n].cpu(), src) and torch.equal(p.dst_pages[:n].cpu(), dst)
    want = order[:used].clone()
    to = torch.arange(P, dtype=torch.int32)
    to[src.long()] = dst
    assert torch.equal(table[0].cpu(), to[want.long()]) and torch.equal(p.remap.cpu(), to)


# ------------------------------------------------------------------- copies

def _pools(P, H, d, pt, code="int8", seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    def byte(*shape):
        x = torch.randint(0, 256, shape, generator=gen, device=DEV, dtype=torch.int16)
        return x.to(torch.uint8).view(P8.CODE_DTYPES[code])
    return dict(kpool=byte(P, H, pt, d), vpool=byte(P, H, pt // 16, d, 16),
                kscale=torch.rand(P, H, pt // 16, generator=gen, device=DEV),
                vscale=torch.rand(P, H, pt // 16, generator=gen, device=DEV))


def _copied(pools, pairs, pt):
    """The pools after copies (source, target, tokens), as bytes."""
    out = {k: (v if v.element_size() == 4 else v.view(torch.uint8)).clone()
           for k, v in pools.items()}
    for s, t, n in pairs:
        b = -(-n // 16)
        for k, x in out.items():
            m = 16 * b if k == "kpool" else b
            x[t, :, :m] = x[s, :, :m]
    return out


def _equal(pools, want):
    for k, v in pools.items():
        assert torch.equal(v if v.element_size() == 4 else v.view(torch.uint8), want[k]), k


@pytest.mark.parametrize("d,H,pt,code", [(64, 1, 64, "int8"), (96, 3, 128, "fp8"),
                                         (128, 8, 256, "int8"), (96, 2, 2048, "int8"),
                                         (128, 1, 2048, "fp8")])
def test_copy_pages(d, H, pt, code):
    pools = _pools(12, H, d, pt, code)
    src, dst = [3, 0, -1, 5, 12, 7, 8], [4, 1, 2, -1, 6, 9, 10]
    tokens = [1, pt, 5, 5, 5, pt // 2 + 3, 0]
    want = _copied(pools, [(3, 4, 1), (0, 1, pt), (7, 9, pt // 2 + 3)], pt)
    P8.copy_pages(i32(src), i32(dst), **pools, tokens=i32(tokens))
    _equal(pools, want)
    # whole pages, the first of them
    want = _copied(pools, [(3, 4, pt), (0, 1, pt)], pt)
    P8.copy_pages(i32(src), i32(dst), **pools, count=i32([3]))
    _equal(pools, want)
    for n in (0, -2):
        P8.copy_pages(i32(src), i32(dst), **pools, count=i32([n]))
    _equal(pools, want)
    # more than there are, token counts off the page
    want = _copied(pools, [(1, 11, pt)], pt)
    P8.copy_pages(i32([1, 2]), i32([11, 3]), **pools, tokens=i32([10 ** 9, -7]), count=i32([99]))
    _equal(pools, want)
    P8.copy_pages(i32([]), i32([]), **pools)
    _equal(pools, want)


def test_copy_of_the_largest_token_counts():
    pools = _pools(6, 2, 64, 128)
    want = _copied(pools, [(0, 3, 128)], 128)
    P8.copy_pages(i32([0, 1]), i32([3, 4]), **pools, tokens=i32([2 ** 31 - 1, -2 ** 31]))
    _equal(pools, want)


def test_copy_many_pages():
    pools = _pools(3000, 2, 64, 64)
    order = torch.randperm(3000, generator=torch.Generator().manual_seed(2)).int()
    src, dst = order[:1500], order[1500:]
    P8.copy_pages(src.to(DEV), dst.to(DEV), **pools)
    for v in pools.values():
        assert torch.equal(v.view(torch.uint8)[src.long()], v.view(torch.uint8)[dst.long()])


def test_copy_past_32_bits():
    """Pages beyond 2^32 bytes of a pool."""
    P, H, d, pt = 18000, 8, 128, 256
    pools = dict(kpool=torch.zeros(P, H, pt, d, dtype=torch.int8, device=DEV),
                 vpool=torch.zeros(P, H, pt // 16, d, 16, dtype=torch.int8, device=DEV),
                 kscale=torch.zeros(P, H, pt // 16, device=DEV),
                 vscale=torch.zeros(P, H, pt // 16, device=DEV))
    for i, v in enumerate(pools.values()):
        v[P - 1] = 5 + i
    P8.copy_pages(i32([P - 1]), i32([P - 2]), **pools)
    P8.copy_pages(i32([P - 2]), i32([0]), **pools, tokens=i32([pt - 20]))
    for i, (k, v) in enumerate(pools.items()):
        m = (pt - 20 + 15) // 16 * (16 if k == "kpool" else 1)
        assert (v[P - 2] == 5 + i).all() and (v[0, :, :m] == 5 + i).all() and not v[0, :, m:].any()
        assert not v[1].any() and not v[P - 3].any()


# ------------------------------------------------------------------- the store

def test_store_forks_compacts_and_shrinks():
    """Every request's tokens stay what they were through forks, appends behind them, releases,
    compactions, shrinking and growing."""
    rng = random.Random(5)
    B, H, d, pt = 12, 2, 64, 64
    st = P8.PagedKV8Store(B, H, d, 40, DEV, page_tokens=pt, pages_per_seq=8, sharing=True)
    gen = torch.Generator(device=DEV).manual_seed(1)
    held = [None] * B                 # (keys, values) as read back after the append

    def slots(b):
        n = int(st.lens[b])
        t = torch.arange(n, device=DEV)
        return st.table[b].long()[t // pt] * pt + t % pt

    for step in range(60):
        new = [rng.choice([0, 0, 1, 5, 40]) for _ in range(B)]
        rows = sum(new) + 1
        plan = st.plan(i32(new), rows)
        k, v = (torch.randn(rows, H, d, generator=gen, device=DEV) for _ in range(2))
        st.append(k, v, plan)
        for b, n in enumerate(plan.q_lens.tolist()):
            x = st.read(slots(b))
            if held[b] is not None and n >= 0:
                # whole blocks never change; the open one may be quantised anew
                whole = held[b][0].shape[0] // 16 * 16
                for a, c in zip(x, held[b]):
                    assert torch.equal(a[:whole], c[:whole]), (step, b)
            held[b] = x
        src, dst = [rng.randrange(B) for _ in range(3)], [rng.randrange(B) for _ in range(3)]
        tokens = [rng.randrange(400) for _ in range(3)] if step % 2 else None
        got = st.fork(i32(src), i32(dst), None if tokens is None else i32(tokens)).tolist()
        old = list(held)
        for s, t, n in zip(src, dst, got):
            if n >= 0:
                held[t] = tuple(x[:n] for x in old[s])
        if step % 3 == 0:
            done = [rng.random() < 0.25 for _ in range(B)]
            st.release(torch.tensor(done, device=DEV))
            held = [tuple(x[:0] for x in h) if f else h for f, h in zip(done, held)]
        if step % 7 == 3:
            st.compact()
        if step == 30:
            used = st.num_pages - st.free_count.item()
            st.shrink(max(used, 1))
            assert st.num_pages == st.kpool.shape[0] == st.free.numel() == st.shares.numel()
            st.grow(45)
        for b in range(B):
            assert held[b][0].shape[0] == int(st.lens[b]), (step, b)
            for a, c in zip(st.read(slots(b)), held[b]):
                assert torch.equal(a, c), (step, b)
    st.release()
    assert st.free_count.item() == st.num_pages and not st.shares.any()


def test_store_shrinks_fp8():
    st = P8.PagedKV8Store(3, 1, 96, 20, DEV, page_tokens=64, code="fp8")
    x = torch.randn(2, 400, 1, 96, device=DEV)
    st.append(x[0], x[1], st.plan(i32([200, 130, 70]), 400))
    st.release(torch.tensor([True, False, False], device=DEV))
    t = torch.arange(130, device=DEV)
    def read():
        return st.read(st.table[1].long()[t // 64] * 64 + t % 64)
    before = read()
    with pytest.raises(ValueError):
        st.shrink(4)
    st.shrink(5)
    assert st.free_count.item() == 0 and st.num_pages == 5
    for a, b in zip(before, read()):
        assert torch.equal(a, b)


# ------------------------------------------------------------------- rotary

def _check_rotary(x, pos, turns, got, factor=1.0, interleaved=False, inverse=False):
    y, tol = S.turned(x.cpu(), pos.tolist(), turns.tolist(), factor, interleaved, inverse)
    tol = tol + HALF[x.dtype] * y.abs()
    err = (got.cpu().double() - y).abs()
    assert (err <= tol).all(), (err - tol).max().item()
    R = 2 * turns.numel()
    assert torch.equal(got[..., R:], x[..., R:])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,Hq,Hk,d,R,interleaved", [
    (1, 1, 1, 128, 128, False), (7, 4, 2, 64, 64, True), (33, 5, 1, 96, 40, False),
    (33, 5, 1, 96, 40, True), (100, 3, 3, 128, 64, False), (5, 2, 1, 80, 16, True),
    (9, 3, 1, 70, 34, False), (9, 1, 2, 7, 6, True), (1300, 8, 2, 64, 64, False),
    (20, 2, 2, 512, 512, False), (9, 3, 2, 512, 500, False), (11, 2, 0, 2048, 70, False),
    (3, 2, 1, 2056, 512, True), (700, 20, 4, 128, 100, False), (700, 20, 4, 128, 90, True)])
def test_rotary(rows, Hq, Hk, d, R, interleaved, dtype):
    gen = torch.Generator().manual_seed(rows)
    # cut out of a projection's output: rows and heads strided
    wide = torch.randn(rows, Hq + Hk + 1, d, generator=gen).to(dtype).to(DEV)
    q, k = wide[:, :Hq], wide[:, Hq:Hq + Hk]
    pos = torch.randint(0, 1 << 20, (rows,), generator=gen).int().to(DEV)
    turns = Q.rotary_turns(Q.rotary_frequencies(R), DEV)
    a, b = rot.rotary(q, k, pos, turns, 1.25, interleaved=interleaved)
    assert a.is_contiguous() and a.dtype is dtype
    _check_rotary(q, pos, turns, a, 1.25, interleaved)
    _check_rotary(k, pos, turns, b, 1.25, interleaved)
    back, none = rot.rotary(q, None, pos, turns, interleaved=interleaved, inverse=True)
    assert none is None
    _check_rotary(q, pos, turns, back, 1.0, interleaved, True)


def test_rotary_positions_of_any_size():
    """Positions at both ends of int32, where 32-bit angles are off by turns."""
    pos = i32([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, 131071, 3])
    turns = Q.rotary_turns([1.0, 0.3, 3.14159, 1e-6, 0.0, 6.3, -0.7, 1e-4], DEV)
    x = torch.randn(8, 2, 16, device=DEV)
    y, _ = rot.rotary(x, None, pos, turns)
    _check_rotary(x, pos, turns, y)
    assert torch.equal(y[0], x[0])       # position 0 turns nothing


@pytest.mark.parametrize("d,R,off", [(64, 64, 0), (64, 48, 0), (64, 64, 1), (66, 60, 3)])
def test_rotary_in_place_and_unaligned(d, R, off):
    gen = torch.Generator().manual_seed(3)
    for dtype in (BF16, F32):
        base = torch.randn(11 * 6 * d + off, generator=gen).to(dtype).to(DEV)
        x = base[off:].view(11, 6, d)
        pos = torch.arange(11, dtype=torch.int32, device=DEV) * 7
        turns = Q.rotary_turns(Q.rotary_frequencies(R), DEV)
        was = x.clone()
        a, b = rot.rotary(x[:, :4], x[:, 4:5], pos, turns, q_out=x[:, :4], k_out=x[:, 4:5])
        assert a.data_ptr() == x.data_ptr()
        _check_rotary(was[:, :4], pos, turns, x[:, :4])
        _check_rotary(was[:, 4:5], pos, turns, x[:, 4:5])
        assert torch.equal(x[:, 5], was[:, 5]) and torch.equal(base[:off], base[:off])
        # into other memory with its own strides, a transposed input
        out = torch.zeros(11, 9, d, dtype=dtype, device=DEV)
        z = was.permute(2, 1, 0).contiguous().permute(2, 1, 0)
        rot.rotary(z[:, :4], None, pos, turns, q_out=out[:, 2:6])
        _check_rotary(was[:, :4], pos, turns, out[:, 2:6])
        assert not out[:, :2].any() and not out[:, 6:].any()


def test_rotary_gradient_is_the_inverse_map():
    """<g, f(x)> = <f'(g), x>, and f' is what differences of f give (f is linear)."""
    gen = torch.Generator().manual_seed(4)
    x, g = (torch.randn(6, 3, 32, generator=gen).to(DEV) for _ in range(2))
    pos = i32([0, 5, 900, 131072, 77, 2])
    turns = Q.rotary_turns(Q.rotary_frequencies(24), DEV)
    for pairs in (False, True):
        f, _ = rot.rotary(x, None, pos, turns, 0.8, interleaved=pairs)
        b, _ = rot.rotary(g, None, pos, turns, 0.8, interleaved=pairs, inverse=True)
        _check_rotary(g, pos, turns, b, 0.8, pairs, True)
        left, right = (g.double() * f.double()).sum(), (b.double() * x.double()).sum()
        # each of the 576 products is off by at most 11 2^-24 of |g| (|x1| + |x2|)
        bound = 2 * 11 * 2.0 ** -24 * float(g.abs().double().max() * 2 * x.abs().double().sum())
        assert abs(float(left - right)) <= bound
        for r, h, c in ((1, 0, 3), (3, 2, 20), (4, 1, 30)):
            e = torch.zeros_like(x)
            e[r, h, c] = 1.0
            fe, _ = rot.rotary(x + e, None, pos, turns, 0.8, interleaved=pairs)
            slope = (g.double() * (fe.double() - f.double())).sum()
            # both results, and the sum x + e, are off by roundings of values up to |x| + 1
            bound = 4 * 11 * 2.0 ** -24 * float((x.abs() + e).max() * 2 * g.abs()[r, h].sum())
            assert abs(float(slope - b[r, h, c].double())) <= bound + 11 * 2.0 ** -24 * 4


def test_rotary_of_nothing_and_special_values():
    turns = Q.rotary_turns(Q.rotary_frequencies(16), DEV)
    a, b = rot.rotary(torch.zeros(0, 4, 16, device=DEV), torch.zeros(0, 2, 16, device=DEV), i32([]),
                      turns)
    assert a.shape == (0, 4, 16) and b.shape == (0, 2, 16)
    x = torch.randn(2, 2, 16, device=DEV)
    x[0, 0, 3], x[0, 1, 1] = float("nan"), float("inf")
    y, _ = rot.rotary(x, None, i32([5, 6]), turns)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[0, 0, [3, 11]] = want[0, 1, [1, 9]] = True
    assert torch.equal(bad, want)


def test_rotary_of_more_rows_than_a_launch():
    """A launch of 256 threads for 8 rows ends below 2^27 of them."""
    part, rows = 1000, (1 << 27) + 1005
    turns = Q.rotary_turns(Q.rotary_frequencies(2), DEV)
    x = torch.randn(part, 1, 2, device=DEV).to(F16)
    pos = torch.arange(part, dtype=torch.int32, device=DEV)
    want, _ = rot.rotary(x, None, pos, turns)
    _check_rotary(x, pos, turns, want)
    n = -(-rows // part)
    xs = x.repeat(n, 1, 1)[:rows]
    got, _ = rot.rotary(xs, None, pos.repeat(n)[:rows], turns)
    assert torch.equal(got, want.repeat(n, 1, 1)[:rows])


def test_rotary_outputs_that_overlap():
    turns = Q.rotary_turns(Q.rotary_frequencies(32), DEV)
    x = torch.randn(4, 3, 32, device=DEV)
    pos = torch.arange(4, dtype=torch.int32, device=DEV)
    for bad in (x[:1].expand(4, 3, 32), x[:, :1].expand(4, 3, 32),
                torch.zeros(400, device=DEV).as_strided((4, 3, 32), (40, 32, 1)),
                torch.zeros(400, device=DEV).as_strided((4, 3, 32), (32, 31, 1))):
        with pytest.raises(ValueError, match="overlap"):
            rot.rotary(x, None, pos, turns, q_out=bad)
        with pytest.raises(ValueError, match="overlap"):
            rot.rotary(x, x.clone(), pos, turns, k_out=bad)
    y = torch.zeros(3, 4, 40, device=DEV)[:, :, :32].transpose(0, 1)   # head-major: disjoint
    rot.rotary(x, None, pos, turns, q_out=y)
    assert torch.equal(y, rot.rotary(x, None, pos, turns)[0])


def test_rotary_of_shared_rows():
    """Rows and heads with a stride of 0 are inputs like others."""
    turns = Q.rotary_turns(Q.rotary_frequencies(32), DEV)
    x = torch.randn(1, 1, 32, device=DEV).expand(40, 3, 32)
    pos = torch.arange(40, dtype=torch.int32, device=DEV)
    y, _ = rot.rotary(x, None, pos, turns)
    _check_rotary(x, pos, turns, y)


def test_python_refusals():
    st = P8.PagedKV8Store(3, 1, 64, 6, DEV, page_tokens=64, sharing=True)
    one, long = i32([0]), torch.zeros(1, dtype=torch.long, device=DEV)
    x = torch.zeros(2, 3, 16, device=DEV)
    pos, turns = i32([0, 1]), Q.rotary_turns([1.0] * 8, DEV)
    books = (st.table, st.lens)
    for call in (
            lambda: st.fork(long, one), lambda: st.fork(one, i32([1, 2])),
            lambda: st.fork(one, one, i32([1, 2])), lambda: st.fork(one.view(1, 1), one),
            lambda: P8.fork_pages(*books, one, one, None, st.free, st.free_count, st.shares[:3], 64),
            lambda: P8.fork_pages(*books, one, one, None, st.free, st.free_count, st.shares, 63),
            lambda: P8.compact_pages(*books, st.free, st.lens, 64),
            lambda: P8.compact_pages(st.table[0], st.lens, st.free, st.free_count, 64),
            lambda: P8.copy_pages(one, i32([1, 2]), **st.pools()),
            lambda: P8.copy_pages(one, one, **st.pools(), count=i32([1, 2])),
            lambda: P8.copy_pages(one, one, **st.pools(), tokens=long),
            lambda: P8.release_pages(*books, st.lens, st.free, st.free_count, 64, shares=st.shares),
            lambda: rot.rotary(x[0], None, pos, turns), lambda: rot.rotary(x, x[:1], pos, turns),
            lambda: rot.rotary(x, x.half(), pos, turns), lambda: rot.rotary(x, None, pos[:1], turns),
            lambda: rot.rotary(x, None, pos.long(), turns),
            lambda: rot.rotary(x, None, pos, turns.int()),
            lambda: rot.rotary(x, None, pos, Q.rotary_turns([1.0] * 9, DEV)),
            lambda: rot.rotary(x, None, pos, turns[:0]),
            lambda: rot.rotary(x.double(), None, pos, turns),
            lambda: rot.rotary(x, None, pos, turns, q_out=x[:1]),
            lambda: rot.rotary(x, None, pos, turns, q_out=x.half()),
            lambda: rot.rotary(x, None, pos, turns, k_out=x),
            lambda: rot.rotary(x, None, pos, turns, q_out=x.permute(2, 1, 0).contiguous().permute(2, 1, 0))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="GPU"):
        rot.rotary(x, None, pos.cpu(), turns)
