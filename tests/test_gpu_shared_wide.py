"""attention_kv8_shared under tables of room for more tokens than its plan counts places for: the
call is attention_kv8's, and refused where it has to share."""

import pytest
import torch

from quashkv_amd import _native as N
from quashkv_amd import paged8 as P8

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(autouse=True, scope="module")
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    N.lib()


@pytest.mark.parametrize("q_lens,causal", [([40] * 30, True), ([1] * 29 + [1200], True),
                                           ([0] * 10 + [60] * 20, False)])
def test_wide_tables(q_lens, causal):
    """30 requests, each with a row of 2^20 table entries (2^31 tokens)."""
    B, H, G, d, pt, W = 30, 2, 4, 64, 2048, 1 << 20
    gen = torch.Generator(device=DEV).manual_seed(1)
    P = 2 + B
    pools = dict(
        kpool=torch.randint(-127, 128, (P, H, pt, d), generator=gen, device=DEV).to(torch.int8),
        vpool=torch.randint(-127, 128, (P, H, pt // 16, d, 16), generator=gen, device=DEV).to(torch.int8),
        kscale=0.01 * torch.rand(P, H, pt // 16, generator=gen, device=DEV) + 1e-4,
        vscale=0.01 * torch.rand(P, H, pt // 16, generator=gen, device=DEV) + 1e-4)
    table = torch.zeros(B, W, dtype=torch.int32, device=DEV)
    table[:, 1] = 1
    table[:, 2] = torch.arange(2, 2 + B, device=DEV)
    start = torch.tensor([0] + q_lens, device=DEV).cumsum(0).int()
    rows = sum(q_lens)
    lens = torch.arange(4096 + 1200, 4096 + 1200 + B, dtype=torch.int32, device=DEV)
    q = torch.randn(rows + 2, H * G, d, generator=gen, device=DEV)
    args = dict(q=q, **pools, table=table, kv_lens=lens, q_start=start, causal=causal,
                q_lens=torch.tensor(q_lens, dtype=torch.int32, device=DEV))
    groups = dict(group_start=torch.tensor([0, B], dtype=torch.int32, device=DEV),
                  prefix_lens=torch.tensor([4096], dtype=torch.int32, device=DEV))
    x = P8.attention_kv8_shared(**args, **groups)
    y = P8.attention_kv8(**args)
    assert torch.equal(x, y) and not x[rows:].any() and x[:rows].abs().amax() > 0
    with pytest.raises(ValueError, match="too large"):
        P8.attention_kv8_shared(**args, **groups, always=True)
    # as wide as the requests are: within 22-bit weights and fp32 sums over 5300 tokens, values up to 1.3
    z = P8.attention_kv8_shared(**{**args, "table": table[:, :3].contiguous()}, **groups, always=True)
    assert float((x - z).abs().max()) <= 4 * 1.3 * (2.0 ** -18 + 300 * 2.0 ** -24)


@pytest.mark.parametrize("rows,max_q_len,told", [(16, 1, 1), (40, 1, 1), (40, 0, 0), (40, 39, 39),
                                                 (40, None, 40), (40, 64, 40), (16, None, 8)])
def test_small_calls_are_told_the_longest(monkeypatch, rows, max_q_len, told):
    """A decode batch with padding rows: what a plan knows of the longest request's rows reaches
    attention_kv8, which else goes by a guess."""
    B, H, G, d = 16, 2, 4, 64
    st = P8.PagedKV8Store(B, H, d, 64, DEV, page_tokens=64, pages_per_seq=4)
    gen = torch.Generator(device=DEV).manual_seed(2)
    k, v = torch.randn(2, B * 70, H, d, generator=gen, device=DEV)
    st.append(k, v, st.plan(torch.full((B,), 70, dtype=torch.int32, device=DEV), B * 70))
    plan = st.plan(torch.zeros(B, dtype=torch.int32, device=DEV), rows, max_q_len=max_q_len)
    plan.q_start.copy_(torch.arange(B + 1, device=DEV))
    plan.q_lens.fill_(1)
    q = torch.randn(rows, H * G, d, generator=gen, device=DEV)
    groups = tuple(torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, B], [64]))
    calls = []
    real = P8._call
    monkeypatch.setattr(P8, "_call", lambda dev, fn, *a: (calls.append((fn.__name__, a)), real(dev, fn, *a)))
    x = st.attention(q, plan, groups=groups)
    monkeypatch.undo()
    (name, args), = calls
    guess = N.lib().qkv_kv8_attention_shared_plain(B, 1, rows, H * G, H, d, 4, 64)
    if told < guess:
        assert name == "qkv_kv8_attention" and args[21] == told
    else:
        assert name == "qkv_kv8_attention_shared" and told == guess
    y = P8.attention_kv8(q, **st.pools(), table=st.table, kv_lens=plan.kv_lens, q_start=plan.q_start,
                         q_lens=plan.q_lens, causal=True, max_q_len=told)
    assert torch.equal(x, y)
    with pytest.raises(ValueError, match="workspace"):
        P8.attention_kv8_shared(q, **st.pools(), table=st.table, kv_lens=plan.kv_lens,
                                group_start=groups[0], prefix_lens=groups[1], q_start=plan.q_start,
                                max_q_len=1,
                                workspace=torch.zeros(64, dtype=torch.uint8, device=DEV))
