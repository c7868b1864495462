"""The bits that softmax weights reach the value product with in attention_kv8_shared: sharing
a prefix takes none from a request, whoever else is in its group.

Keys are zero, so that a weight is its block's value scale.  In each step of 64 tokens two blocks of
16 have scale s and two a smaller one, t, whose codes in coordinate 0 cancel: m t + n s = 0.  The result
there is 0 but for the weights' roundings, so that no rounding of the result hides them: s meets
an f16 as the power of two that the largest weight is, t not, and weights of 11 bits leave
up to 2^-12 of the values, where the bound is about 2^-16 of them."""

import pytest
import torch

from quashkv_amd import _native as N
from quashkv_amd import paged8 as P8
from tests import kv8_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
# codes m of the larger and n of the smaller scale, a kv head each: 128 |m / n| lies a third of an
# f16's step or more from the nearest one
CODES = {"int8": [(50, -127), (74, -121), (99, -127), (73, -121)],
         "fp8": [(-240.0, 416.0), (176.0, -288.0), (288.0, -448.0), (256.0, -352.0)]}


@pytest.fixture(autouse=True, scope="module")
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    N.lib()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_codes_are_off_an_f16():
    for code, pairs in CODES.items():
        for m, n in pairs:
            w = 128 * abs(m / n)
            step = 2.0 ** (torch.tensor(w).log2().floor().item() - 10)
            assert abs(w / step - round(w / step)) > 0.3, (code, m, n)


def _cancelling(code, d, B, prefix, seed):
    """Pools and a table of B requests behind one prefix, a page of 64 own tokens each, of
    which they hold 16; values in 64 bits of a request's tokens, which are every request's."""
    H, pt = 4, 64
    pages = prefix // pt + 1
    gen = torch.Generator().manual_seed(seed)
    top = 127 if code == "int8" else 448
    v = torch.randint(-top, top + 1, (pages, H, pt // 16, d, 16), generator=gen).float()
    s = torch.empty(pages, H, pt // 16)
    for h, (m, n) in enumerate(CODES[code]):
        s[:, h, 0::2] = 0.01
        s[:, h, 1::2] = (torch.tensor(0.01, dtype=F32).double() * abs(m / n)).float()
        v[:, h, 0::2, 0], v[:, h, 1::2, 0] = m, n
    # own tokens: one block, of zeros in coordinate 0
    s[-1], v[-1, :, :, 0] = 0.003, 0
    codes = v.to(P8.CODE_DTYPES[code])
    v = codes.double() * s[:, :, :, None, None].double()
    v = v.permute(0, 2, 4, 1, 3).reshape(pages * pt, H, d)[:prefix + 16]
    u8 = lambda x: x.view(torch.uint8).to(DEV).view(x.dtype)
    pools = dict(kpool=u8(torch.zeros(pages, H, pt, d, dtype=torch.int8).view(codes.dtype)),
                 kscale=torch.zeros(pages, H, pt // 16, device=DEV),
                 vpool=u8(codes), vscale=s.to(DEV))
    return pools, i32([list(range(pages))] * B), v


def _check(code, d, q_dtype, out_dtype, q_lens, groups, G=4, prefix=256, seed=0, exact=None):
    B, H = len(q_lens), 4
    pools, table, v = _cancelling(code, d, B, prefix, seed)
    T = v.shape[0]
    start = [0]
    for n in q_lens:
        start.append(start[-1] + n)
    q = torch.randn(start[-1], H * G, d, generator=torch.Generator().manual_seed(seed + 1)).to(q_dtype)
    out = P8.attention_kv8_shared(
        q.to(DEV), **pools, table=table, kv_lens=i32([T] * B), group_start=i32(groups),
        prefix_lens=i32([prefix] * (len(groups) - 1)), q_start=i32(start), out_dtype=out_dtype,
        always=True).cpu().double()
    o, tol = R.attend(q[:1].double(), torch.zeros_like(v), v, d ** -0.5, None, 2.0 ** -22,
                      2.0 ** -22, HALF[out_dtype])           # (every row's: weights ignore queries)
    assert float(o[..., 0].abs().max()) < 2.0 ** -22
    for b in range(B) if exact is None else exact:
        bad = (out[start[b]:start[b + 1]] - o).abs() > tol
        assert not bad.any(), (b, float((out[start[b]:start[b + 1]] - o)[..., 0].abs().max()),
                               float(tol[..., 0].max()))


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("q_dtype,out_dtype", [(BF16, BF16), (F16, BF16), (BF16, F16), (F32, BF16)])
def test_decode_rows(code, d, q_dtype, out_dtype):
    """A few requests of a row each, and so many that their rows are a tall tile."""
    for B in (3, 12, 40):
        _check(code, d, q_dtype, out_dtype, [1] * B, [0, B], seed=B)


@pytest.mark.parametrize("B,groups", [(90, [0, 90]), (100, [0, 40, 41, 99]), (1100, [0, 1000])])
def test_decode_rows_of_many_requests(B, groups):
    _check("int8", 64, BF16, BF16, [1] * B, groups, seed=B)


@pytest.mark.parametrize("more", [0, 70])
@pytest.mark.parametrize("at", [0, 2, 4])
def test_decode_rows_beside_a_chunk(at, more):
    """A request of many rows in the group takes no bits from the others."""
    q_lens = [1, 3, 1, 8]
    q_lens.insert(at, 40)
    q_lens += [1] * more
    _check("int8", 128, BF16, BF16, q_lens, [0, len(q_lens)], seed=at,
           exact=[b for b in range(len(q_lens)) if b != at])


def test_chunks_of_fp16_results():
    """Where attention_kv8 keeps 22 bits for any number of rows."""
    _check("int8", 64, F16, F16, [40, 70, 33], [0, 3])
    _check("fp8", 96, BF16, F32, [40, 70, 33], [0, 3])
    _check("fp8", 128, F32, BF16, [40, 70, 33], [0, 3])
