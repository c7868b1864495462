"""Timed cases of the 8-bit paged cache: page plans, appends, attention.

The operators, and what a program holds of them:

* ``plan_pages``: block tables and slot maps of a batch of requests, built on
  the GPU from their lengths;
* ``append_kv8`` / ``read_kv8``: keys and values quantised to 8 bits (int8 or
  float8_e4m3fn) with one fp32 scale per block of 16 tokens and head, and back;
* ``attention_kv8``: attention of a ragged batch of queries over that cache.

``own`` picks what ``run`` calls: the framework's operators, or the plain forms
below (elementary torch operations in 32 bits).  ``exact`` is the same result
in 64 bits from the definition.

Pools: pages of ``pt`` tokens with all H kv heads; ``kpool`` (P, H, pt, d),
``vpool`` (P, H, pt / 16, d, 16), ``kscale`` / ``vscale`` (P, H, pt / 16).
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"int8": (torch.int8, 127.0), "fp8": (torch.float8_e4m3fn, 448.0)}
BLOCK = 16
FLOOR = 2.0 ** -100
FINITE = torch.finfo(torch.float32).max


# ---------------------------------------------------------------- cases

def plan(name, B, rows, new, longest, pt=256, spare=1.25):
    return dict(name=name, kind="plan", B=B, rows=rows, new=new, longest=longest, pt=pt,
                spare=spare)


def append(name, B, rows, H, d, new, longest, dtype="bf16", fmt="int8", pt=256, out="bf16"):
    return dict(name=name, kind="append", B=B, rows=rows, H=H, d=d, new=new, longest=longest,
                dtype=dtype, fmt=fmt, pt=pt, out=out)


def attend(name, B, Hq, Hkv, d, T, Q=1, ragged=False, causal=True, dtype="bf16", out="bf16",
           fmt="int8", pt=256):
    return dict(name=name, kind="attend", B=B, Hq=Hq, Hkv=Hkv, d=d, T=T, Q=Q, ragged=ragged,
                causal=causal, dtype=dtype, out=out, fmt=fmt, pt=pt)


def listed():
    return [
        # a decode step of 64 requests: one new token each, few of them open a page
        plan("plan_decode", 64, 64, "one", 8192),
        # a step that admits prompts of many lengths beside running requests; the pool runs short
        plan("plan_admit", 384, 32768, "ragged", 4096, pt=64, spare=0.9),
        # a decode step's token of 64 requests into a Llama-3-8B layer's cache
        append("append_token", 64, 64, 8, 128, "one", 2048),
        # the prompts of 24 requests, odd lengths, into the same layer
        append("append_prompt", 24, 24001, 8, 128, "ragged", 1000),
        # a chunk at head_dim 96 into an 8-bit float cache, fp16 in, read back in fp32
        append("append_chunk", 5, 2003, 3, 96, "ragged", 300, dtype="fp16", fmt="fp8", pt=64,
               out="fp32"),
        # the README's quickstart shape: one fp32 query over a 512-token context
        attend("attend_quickstart", 1, 8, 8, 128, 512, dtype="fp32", out="fp32"),
        # a Llama-3-8B layer serving 32 sequences of 8k tokens
        attend("attend_serving", 32, 32, 8, 128, 8192),
        # requests of very different lengths, head_dim 96, 8-bit float codes
        attend("attend_ragged", 40, 24, 8, 96, 9001, ragged=True, dtype="fp16", out="fp16",
               fmt="fp8", pt=64),
        # one 128k-token document
        attend("attend_long", 1, 32, 8, 128, 131072),
        # the prompt pass of a Llama-3-8B layer: 2048 causal queries
        attend("attend_prompt", 1, 32, 8, 128, 2048, Q=2048),
        # chunks of longer prompts beside decoding requests, head_dim 64, 7 query heads per kv head
        attend("attend_mixed", 12, 14, 2, 64, 1501, Q=301, ragged=True, dtype="fp16", out="fp32",
               pt=128),
        # a whole decode step of one Qwen2.5-0.5B layer: plan, append, attention, 16 requests
        dict(name="step_decode", kind="step", B=16, Hq=14, Hkv=2, d=64, T=2048, dtype="bf16",
             out="bf16", fmt="int8", pt=256),
    ]


def _lu(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "append", "decode", "decode", "decode", "prefill",
                       "prefill", "mixed", "step"])
    d = rng.choice([64, 96, 128, 128])
    H = rng.choice([1, 2, 3, 4, 8])
    G = rng.choice([1, 2, 3, 4, 4, 7, 8])
    fmt = rng.choice(["int8", "int8", "fp8"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    pt = rng.choice([64, 128, 256, 256, 1024])
    if kind == "plan":
        B = _lu(rng, 1, 2000)
        new = rng.choice(["one", "ragged"])
        rows = B if new == "one" else max(B, _lu(rng, 16, 32768))
        return plan("", B, rows, new, _lu(rng, 16, 8192), pt, rng.choice([0.7, 1.1, 1.5]))
    if kind == "append":
        B = _lu(rng, 1, 128)
        new = rng.choice(["one", "ragged"])
        rows = B if new == "one" else max(B, _lu(rng, 16, 24000))
        return append("", B, rows, H, d, new, _lu(rng, 16, 1000), dtype, fmt, pt,
                      rng.choice(["bf16", "fp32"]))
    out = rng.choice([dtype, "fp32"])
    if kind == "decode":
        T = _lu(rng, 1, 100000)
        B = max(1, min(_lu(rng, 1, 128), 2000000 // (H * T)))
        return attend("", B, H * G, H, d, T, Q=min(T, rng.choice([1, 1, 1, 2, 4])),
                      ragged=rng.random() < 0.5, dtype=dtype, out=out, fmt=fmt, pt=pt)
    if kind == "prefill":
        Q = _lu(rng, 16, 2048)
        T = Q if rng.random() < 0.5 else Q + _lu(rng, 16, 4096)
        T = min(T, max(Q, (1 << 26) // (H * G * Q)))
        Q = min(Q, (1 << 26) // (H * G * T))
        B = max(1, min(rng.choice([1, 1, 2, 4]), (1 << 26) // (H * G * Q * T)))
        return attend("", B, H * G, H, d, T, Q=Q, causal=rng.random() < 0.8, dtype=dtype, out=out,
                      fmt=fmt, pt=pt)
    if kind == "mixed":
        Q = _lu(rng, 16, 512)
        T = Q + _lu(rng, 16, 2048)
        B = max(2, min(_lu(rng, 2, 24), (1 << 26) // (H * G * Q * T)))
        return attend("", B, H * G, H, d, T, Q=Q, ragged=True, dtype=dtype, out=out, fmt=fmt,
                      pt=pt)
    T = _lu(rng, 16, 8192)
    return dict(kind="step", B=max(1, min(_lu(rng, 1, 64), (1 << 20) // (H * T))), Hq=H * G, Hkv=H,
                d=d, T=T, dtype=dtype, out=out, fmt=fmt, pt=pt)


# --------------------------------------------------- sizes (host)

def _ceil(a, b):
    return -(-a // b)


def _pages_of(tokens, pt):
    return (tokens + pt - 1) // pt


def _split(total, parts, g):
    """`parts` whole numbers that sum to `total`, of very different sizes."""
    w = torch.rand(parts, generator=g).double() ** 3 + 1e-3
    n = (w / w.sum() * total).floor().long()
    n[0] += total - int(n.sum())
    return n


def _lengths(case, g):
    """(cached tokens before the call, new tokens) of each request."""
    B, kind = case["B"], case["kind"]
    if kind in ("plan", "append"):
        lens = torch.randint(0, case["longest"] + 1, (B,), generator=g)
        if case["new"] == "one":
            return lens, torch.ones(B, dtype=torch.long)
        # a part of the requests takes no tokens in this step; the last rows are padding
        new = _split(case["rows"] - case["rows"] // 50, B, g)
        new[1:][torch.rand(B - 1, generator=g) < 0.1] = 0
        return lens, new
    if kind == "step":
        return torch.full((B,), case["T"] - 1, dtype=torch.long), torch.ones(B, dtype=torch.long)
    T, Q = case["T"], case["Q"]
    if not case["ragged"]:
        return torch.full((B,), T - Q, dtype=torch.long), torch.full((B,), Q, dtype=torch.long)
    kv = (T * torch.rand(B, generator=g).double() ** 2).long() + 1
    kv[0] = T
    if Q > 8:   # every third request is a chunk of a prompt, the others decode
        new = torch.ones(B, dtype=torch.long)
        new[::3] = torch.minimum((Q * (0.3 + 0.7 * torch.rand(B, generator=g))).long() + 1,
                                 kv)[::3]
        new[0] = Q
    else:
        new = torch.full((B,), Q, dtype=torch.long)
    new = torch.minimum(new, kv)
    return kv - new, new


def _pages(case, lens, new, g):
    """(pool pages, table width, table, free list, free count) with the cached
    tokens' pages placed at random."""
    pt, B = case["pt"], case["B"]
    held, want = _pages_of(lens, pt), _pages_of(lens + new, pt)
    width = int(want.max()) + 1
    ask = int((want - held).sum())
    spare = max(1, int(case.get("spare", 1.0) * ask))
    P = int(held.sum()) + spare
    order = torch.randperm(P, generator=g).int()
    table = torch.zeros(B, width, dtype=torch.int32)
    at = 0
    for b in range(B):
        n = int(held[b])
        table[b, :n] = order[at:at + n]
        at += n
    free = torch.zeros(P, dtype=torch.int32)
    free[:spare] = order[at:]
    return P, table, free, torch.tensor([spare], dtype=torch.int32)


def _sizes(case, seed):
    """The requests' lengths are the case's, the places of their pages the seed's."""
    lens, new = _lengths(case, torch.Generator().manual_seed(17))
    return (lens, new) + _pages(case, lens, new, torch.Generator().manual_seed(seed))


# --------------------------------------------------------------- plain forms

def _codes_of(y, fmt):
    """The 8-bit codes (as int8 bytes) nearest to y (float64), ties to even."""
    if fmt == "int8":
        return y.round().clamp(-127, 127).to(torch.int8)
    y = y.clamp(-448, 448)
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 4).clamp(min=-9))
    return ((y / step).round() * step).to(torch.float8_e4m3fn).view(torch.int8)


def _values(codes, fmt, dtype=torch.float32):
    """The numbers that int8 bytes stand for, before the scale."""
    return codes.to(dtype) if fmt == "int8" else codes.view(torch.float8_e4m3fn).to(dtype)


def _scale_of(amax, fmt):
    s = (amax * (1.0 / CODES[fmt][1])).clamp(min=FLOOR)
    return torch.where(amax > 0, s, torch.zeros_like(s))


def _inverse(s):
    """fp32 1 / s, 0 where s is."""
    r = (1.0 / s.double()).float()
    return torch.where(s > 0, r, torch.zeros_like(r))


def _new_codes(x, inv, fmt):
    """Codes of fp32 values x at inverse scales inv: the product is exact in 64 bits."""
    return _codes_of(x.double() * inv.double(), fmt)


def _plain_plan(st):
    table, pt, rows = st["table"], st["pt"], st["rows"]
    lens, new = st["lens"].long(), st["new"].long().clamp(min=0)
    B, width = table.shape
    ends = torch.cumsum(new, 0)
    q_start = torch.cat([ends.new_zeros(1), ends])
    held, want = _pages_of(lens, pt), _pages_of(lens + new, pt)
    fits = (ends <= rows) & (want <= width)
    ask = torch.where(fits, want - held, torch.zeros_like(held))
    top = torch.cumsum(ask, 0)
    count = st["free_count"].long()
    ok = fits & ((ask == 0) | (top <= count))
    q_lens = torch.where(ok, new, torch.zeros_like(new))
    take = torch.where(ok, ask, torch.zeros_like(ask))
    col = torch.arange(width, device=table.device)
    fresh = (col >= held[:, None]) & (col < (held + take)[:, None])
    at = count - 1 - (top - ask)[:, None] - (col - held[:, None])
    table.copy_(torch.where(fresh, st["free"][at.clamp(0, st["free"].numel() - 1)], table))
    r = torch.arange(rows, device=table.device)
    b = torch.searchsorted(ends, r, right=True).clamp(max=B - 1)
    i = r - q_start[b]
    live = (r < ends[-1]) & (i < q_lens[b])
    t = torch.where(live, lens[b] + i, torch.zeros_like(i))
    slots = torch.where(live, table[b, t // pt].long() * pt + t % pt, torch.full_like(t, -1))
    return {"q_start": q_start.int(), "q_lens": q_lens.int(), "kv_lens": (lens + q_lens).int(),
            "slots": slots, "positions": t.int(), "free_count": (count - take.sum()).int(),
            "table": table}


def _blocks(slots, pt):
    """(page, token in the page, block of the page, token of the block) of slots >= 0."""
    page, o = slots // pt, slots % pt
    return page, o, o // BLOCK, o % BLOCK


def _plain_append(st, x, slots, pool, scale, transposed):
    """x (N, H, d) into the pool at slots.  st["part"]: the first rows of the requests whose
    first new token falls into a block that holds tokens already."""
    fmt, pt = st["fmt"], st["pt"]
    codes = pool.view(torch.int8)
    H = x.shape[1]
    nb = pt // BLOCK
    h = torch.arange(H, device=x.device)
    k = torch.arange(BLOCK, device=x.device)
    x, slots1 = x[st["live_rows"]].float(), slots[st["part"]]
    page, o, blk, j = _blocks(slots[st["live_rows"]], pt)
    page1, _, blk1, j1 = _blocks(slots1, pt)
    # (page, head, block) of every row, and of the blocks that hold tokens
    at = (page[:, None] * H + h) * nb + blk[:, None]
    at1 = (page1[:, None] * H + h) * nb + blk1[:, None]
    size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    top = torch.zeros(scale.numel(), device=x.device)
    top.scatter_reduce_(0, at.reshape(-1), size.reshape(-1), "amax")
    old = torch.zeros(scale.numel(), device=x.device)
    old1 = scale.view(-1)[at1]
    old[at1.reshape(-1)] = old1.reshape(-1)
    s = torch.maximum(old, _scale_of(top, fmt))
    inv = _inverse(s)
    # earlier tokens of those blocks at the new scale, where it grew
    if transposed:
        place = (page1[:, None], h, blk1[:, None])
        was = codes[place].transpose(-1, -2)                                    # (n, H, 16, d)
    else:
        place = (page1[:, None, None], h[:, None], blk1[:, None, None] * BLOCK + k)
        was = codes[place]
    again = _new_codes(_values(was, fmt) * old1[..., None, None], inv[at1][..., None, None], fmt)
    grew = (s[at1] > old1)[..., None] & (k < j1[:, None, None])
    now = torch.where(grew[..., None], again, was)
    codes[place] = now.transpose(-1, -2) if transposed else now
    # the new tokens
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x.clamp(-FINITE, FINITE))
    new = _new_codes(x, inv[at][..., None], fmt)
    if transposed:
        codes[page[:, None], h, blk[:, None], :, j[:, None]] = new
    else:
        codes[page[:, None], h, o[:, None]] = new
    scale.view(-1)[at.reshape(-1)] = s[at.reshape(-1)]


def _plain_read(st, slots, pool, scale, transposed, dtype):
    page, o, blk, j = _blocks(slots.clamp(min=0), st["pt"])
    codes = pool.view(torch.int8)
    h = torch.arange(pool.shape[1], device=pool.device)
    if transposed:
        c = codes[page[:, None], h, blk[:, None], :, j[:, None]]
    else:
        c = codes[page[:, None], h, o[:, None]]
    x = _values(c, st["fmt"]) * scale[page[:, None], h, blk[:, None]][..., None]
    return torch.where((slots >= 0)[:, None, None], x, torch.zeros_like(x)).to(dtype)


def _dense(st, table, dtype):
    """The cache as (B, H, T, d) keys and values, T = the longest request's pages."""
    fmt, pt = st["fmt"], st["pt"]
    pages = table[:, :_ceil(st["T"], pt)].long()
    B, W = pages.shape
    _, H, _, d = st["kpool"].shape
    kc = _values(st["kpool"].view(torch.int8)[pages], fmt, dtype)             # (B, W, H, pt, d)
    kc = kc.view(B, W, H, pt // BLOCK, BLOCK, d) * st["kscale"][pages].to(dtype)[..., None, None]
    vc = _values(st["vpool"].view(torch.int8)[pages], fmt, dtype)             # (B, W, H, nb, d, 16)
    vc = (vc * st["vscale"][pages].to(dtype)[..., None, None]).transpose(-1, -2)
    k = kc.permute(0, 2, 1, 3, 4, 5).reshape(B, H, W * pt, d)
    v = vc.permute(0, 2, 1, 3, 4, 5).reshape(B, H, W * pt, d)
    return k, v


def _plain_attend(st, q, table, q_start, q_lens, kv_lens, out):
    N, Hq, d = q.shape
    k, v = _dense(st, table, torch.float32)
    B, H, T, _ = k.shape
    G, Q = Hq // H, st["Q"]
    i = torch.arange(Q, device=q.device)
    row = (q_start[:B].long()[:, None] + i).clamp(max=N - 1)                  # (B, Q)
    live = i < q_lens.long()[:, None]
    x = q[row].float().view(B, Q, H, G, d).permute(0, 2, 3, 1, 4).reshape(B, H, G * Q, d)
    s = torch.matmul(x, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(d))
    s = s.view(B, H, G, Q, T)
    t = torch.arange(T, device=q.device)
    last = kv_lens.long()[:, None] - 1 + torch.zeros_like(row)
    if st["causal"]:
        last = kv_lens.long()[:, None] - q_lens.long()[:, None] + i
    seen = (t <= last[..., None])[:, None, None]                              # (B, 1, 1, Q, T)
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(p.view(B, H, G * Q, T), v).view(B, H, G, Q, d)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, Q, Hq, d).to(out.dtype)
    # rows that no request asks for keep what they hold
    flat = torch.where(live, row, torch.full_like(row, N))
    wide = torch.cat([out, out.new_zeros(1, Hq, d)])
    wide[flat.reshape(-1)] = o.reshape(B * Q, Hq, d)
    out.copy_(wide[:N])
    return out


# ------------------------------------------------------------- prepare / run

def _fill(gen, P, H, pt, d, fmt, loud):
    """A pool's codes and scales from random tokens: quantised block by block."""
    nb = pt // BLOCK
    x = torch.randn(P, H, nb, BLOCK, d, generator=gen, device="cuda")
    x = x * (1 + 4 * (torch.rand(d, generator=gen, device="cuda") < 0.03) * loud)
    x = x * torch.exp(0.3 * torch.randn(P, H, nb, 1, 1, generator=gen, device="cuda"))
    s = _scale_of(x.abs().amax((-1, -2)), fmt)
    y = x * _inverse(s)[..., None, None]
    if fmt == "int8":
        return y.round().clamp(-127, 127).to(torch.int8), s
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), s


def _pools(case, P, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    H = case.get("Hkv", case.get("H"))
    d, pt, fmt = case["d"], case["pt"], case["fmt"]
    k, ks = _fill(gen, P, H, pt, d, fmt, 1)
    v, vs = _fill(gen, P, H, pt, d, fmt, 0)
    k = k.view(P, H, pt, d)
    v = v.view(torch.int8).transpose(-1, -2).contiguous().view(CODES[fmt][0])
    return dict(kpool=k, kscale=ks, vpool=v, vscale=vs)


def _rows(gen, n, H, d, dtype, parts=1):
    """n rows of `parts` tensors (n, H, d), cut out of one projection's output."""
    x = torch.randn(n, parts * H * d, generator=gen, device="cuda").to(dtype)
    return [x[:, i * H * d:(i + 1) * H * d].unflatten(1, (H, d)) for i in range(parts)]


def _placed(table, free, count, lens, new, pt):
    """The table after the plan, on the host, where every request is granted."""
    table = table.clone()
    top = int(count)
    for b in range(len(lens)):
        held, want = _ceil(int(lens[b]), pt), _ceil(int(lens[b] + new[b]), pt)
        for p in range(held, want):
            top -= 1
            table[b, p] = free[top]
    return table


def _slot_map(table, lens, new, pt, rows):
    slots = torch.full((rows,), -1, dtype=torch.long)
    at = 0
    for b in range(len(lens)):
        n = int(new[b])
        t = int(lens[b]) + torch.arange(n)
        slots[at:at + n] = table[b].long()[t // pt] * pt + t % pt
        at += n
    return slots


def prepare(case, seed):
    kind, pt = case["kind"], case["pt"]
    lens, new, P, table, free, count = _sizes(case, seed)
    B = case["B"]
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    dev = "cuda"
    st = dict(kind=kind, pt=pt, table=table.to(dev), free=free.to(dev), free_count=count.to(dev),
              lens=lens.int().to(dev), new=new.int().to(dev))
    if kind == "plan":
        st["rows"] = case["rows"]
        return st
    st["fmt"] = case["fmt"]
    st.update(_pools(case, P, seed + 2))
    q_start = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(new, 0)])
    st["q_start"] = q_start.int().to(dev)
    dtype = DTYPES[case["dtype"]]
    if kind == "append":
        rows = case["rows"]
        after = _placed(table, free, count, lens, new, pt)
        slots = _slot_map(after, lens, new, pt, rows)
        st["slots"] = slots.to(dev)
        st["live_rows"] = torch.nonzero(slots >= 0).view(-1).to(dev)
        st["part"] = q_start[:-1][(new > 0) & (lens % BLOCK > 0)].to(dev)
        st["k"], st["v"] = _rows(gen, rows, case["H"], case["d"], dtype, 2)
        # a request's block that the call finds half full is read back with the new tokens
        edge = lens - lens % BLOCK
        back = [after[b].long()[t // pt] * pt + t % pt for b in range(B) if new[b] > 0
                for t in [torch.arange(int(edge[b]), int(lens[b] + new[b]))]]
        st["back"] = torch.cat(back).to(dev)
        st["out_dtype"] = DTYPES[case["out"]]
        return st
    N = int(new.sum())
    kv = lens + new
    st["T"], st["Q"], st["causal"] = int(kv.max()), int(new.max()), case.get("causal", True)
    st["out_dtype"] = DTYPES[case["out"]]
    Hq, H, d = case["Hq"], case["Hkv"], case["d"]
    st["out"] = torch.zeros(N, Hq, d, dtype=st["out_dtype"], device=dev)
    if kind == "step":
        st["rows"] = N
        x = torch.randn(N, (Hq + 2 * H) * d, generator=gen, device=dev).to(dtype)
        st["q"] = x[:, :Hq * d].unflatten(1, (Hq, d))
        st["k"] = x[:, Hq * d:(Hq + H) * d].unflatten(1, (H, d))
        st["v"] = x[:, (Hq + H) * d:].unflatten(1, (H, d))
        st["part"] = q_start[:-1][lens % BLOCK > 0].to(dev)
        st["live_rows"] = torch.arange(N, device=dev)
        return st
    st["table"] = _placed(table, free, count, lens, new, pt).to(dev)
    st["kv_lens"] = kv.int().to(dev)
    st["q_lens"] = new.int().to(dev)
    st["q"] = torch.randn(N, Hq, d, generator=gen, device=dev).to(dtype)
    return st


def run(st):
    kind = st["kind"]
    if own:
        from quashkv_amd import paged8
        pools = {k: st[k] for k in ("kpool", "kscale", "vpool", "vscale")} if kind != "plan" else {}
        if kind in ("plan", "step"):
            p = paged8.plan_pages(st["table"], st["lens"], st["new"], st["free"],
                                  st["free_count"], st["rows"], st["pt"])
        if kind == "plan":
            return {"q_start": p.q_start, "q_lens": p.q_lens, "kv_lens": p.kv_lens,
                    "slots": p.slots, "positions": p.positions, "free_count": p.free_count,
                    "table": st["table"]}
        if kind == "append":
            paged8.append_kv8(st["k"], st["v"], st["slots"], **pools)
            k, v = paged8.read_kv8(st["back"], **pools, out_dtype=st["out_dtype"])
            return {"k": k, "v": v, "kscale": st["kscale"], "vscale": st["vscale"]}
        if kind == "step":
            paged8.append_kv8(st["k"], st["v"], p.slots, **pools)
            out = paged8.attention_kv8(st["q"], **pools, table=st["table"], kv_lens=p.kv_lens,
                                       q_start=p.q_start, q_lens=p.q_lens, causal=True,
                                       max_q_len=st["Q"], out=st["out"])
            return {"out": out, "slots": p.slots, "kv_lens": p.kv_lens,
                    "free_count": p.free_count, "kscale": st["kscale"], "vscale": st["vscale"]}
        return paged8.attention_kv8(st["q"], **pools, table=st["table"], kv_lens=st["kv_lens"],
                                    q_start=st["q_start"], q_lens=st["q_lens"],
                                    causal=st["causal"], max_q_len=st["Q"], out=st["out"])
    if kind == "plan":
        return _plain_plan(st)
    if kind == "append":
        _plain_append(st, st["k"], st["slots"], st["kpool"], st["kscale"], False)
        _plain_append(st, st["v"], st["slots"], st["vpool"], st["vscale"], True)
        return {"k": _plain_read(st, st["back"], st["kpool"], st["kscale"], False, st["out_dtype"]),
                "v": _plain_read(st, st["back"], st["vpool"], st["vscale"], True, st["out_dtype"]),
                "kscale": st["kscale"], "vscale": st["vscale"]}
    if kind == "step":
        p = _plain_plan(st)
        _plain_append(st, st["k"], p["slots"], st["kpool"], st["kscale"], False)
        _plain_append(st, st["v"], p["slots"], st["vpool"], st["vscale"], True)
        out = _plain_attend(st, st["q"], st["table"], p["q_start"], p["q_lens"], p["kv_lens"],
                            st["out"])
        return {"out": out, "slots": p["slots"], "kv_lens": p["kv_lens"],
                "free_count": p["free_count"], "kscale": st["kscale"], "vscale": st["vscale"]}
    return _plain_attend(st, st["q"], st["table"], st["q_start"], st["q_lens"], st["kv_lens"],
                         st["out"])


# ---------------------------------------------------------------------- work

def work(case):
    lens, new, P, table, free, count = _sizes(case, 0)
    n, B = int(new.sum()), case["B"]
    if case["kind"] == "plan":
        pages = int((_pages_of(lens + new, case["pt"]) - _pages_of(lens, case["pt"])).sum())
        # lengths in and out, a slot and a position a row, the pages touched
        return {"bytes": 20 * B + 12 * case["rows"] + 8 * pages + 8, "flops": 0}
    d = case["d"]
    H = case.get("Hkv", case.get("H"))
    es = 4 if case["dtype"] == "fp32" else 2
    os_ = 4 if case["out"] == "fp32" else 2
    blocks = int(((lens + new + BLOCK - 1) // BLOCK - lens // BLOCK)[new > 0].sum())
    held = int((lens % BLOCK)[new > 0].sum())
    put = 2 * H * (n * d * (es + 1) + 4 * blocks) + 8 * n
    if case["kind"] == "append":
        # both halves in and their codes and scales out; the values of the blocks read back
        return {"bytes": put + 2 * H * ((n + held) * d * (1 + os_) + 4 * blocks) + 8 * (n + held),
                "flops": 0}
    kv = lens + new
    Hq = case["Hq"]
    seen = kv * new
    if case.get("causal", True):
        seen = (lens + 1 + kv) * new // 2
    cache = int((2 * H * d * kv + 2 * 4 * H * ((kv + BLOCK - 1) // BLOCK)).sum())
    w = {"bytes": cache + n * Hq * d * (es + os_) + 4 * table.numel(),
         "flops": 4 * d * Hq * int(seen.sum())}
    if case["kind"] == "step":
        w["bytes"] += put
    return w


# --------------------------------------------------------------------- exact

def _exact_quant(x, s, fmt):
    """The values (64 bits) that x stands for at fp32 scales s, from the definition."""
    top = CODES[fmt][1]
    inv = torch.where(s > 0, (1.0 / s.double()).float().double(), torch.zeros_like(s).double())
    y = (x.double() * inv).clamp(-top, top)
    if fmt == "int8":
        return torch.round(y) * s.double()
    # spacing of e4m3 numbers: 2^(e - 3) in [2^e, 2^(e + 1)), e >= -6
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30)))
    e = torch.where(y.abs() < torch.exp2(e), e - 1, e)
    e = torch.where(y.abs() >= torch.exp2(e + 1), e + 1, e).clamp(min=-6)
    return torch.round(y * torch.exp2(3 - e)) * torch.exp2(e - 3) * s.double()


def _exact_scale(a, fmt):
    s = (a.double() * float(torch.tensor(1.0 / CODES[fmt][1]))).float().clamp(min=FLOOR)
    return torch.where(a > 0, s, torch.zeros_like(s))


def _tokens(pool, scale, table_row, t0, t1, pt, fmt, transposed):
    """Tokens [t0, t1) of a request as (t1 - t0, H, d): the values in 64 bits, and fp32 scales."""
    t = torch.arange(t0, t1, device=pool.device)
    page = table_row.long()[t // pt]
    o = t % pt
    raw = pool.view(torch.int8)
    c = raw[page, :, o // BLOCK, :, o % BLOCK] if transposed else raw[page, :, o]
    c = c.double() if fmt == "int8" else c.view(torch.float8_e4m3fn).double()
    s = scale[page, :, o // BLOCK]
    return c, s


def _exact_append(x, lens, new, pool, scale, transposed, fmt, table, pt):
    """Per request: the values (64 bits) of the tokens from its first touched block on, and
    the scales, which are updated in `scale`."""
    out, at = [], 0
    scale = scale.clone()
    for b in range(len(lens)):
        n, t0 = int(new[b]), int(lens[b])
        if n == 0:
            continue
        rows = x[at:at + n].float()
        at += n
        edge = t0 - t0 % BLOCK
        if t0 > edge:
            c, s = _tokens(pool, scale, table[b], edge, t0, pt, fmt, transposed)
            c = (c * s.double()[..., None]).float()
            first = s[0]
        else:
            c, first = rows[:0], torch.zeros(rows.shape[1], device=rows.device)
        full = torch.cat([c, rows])
        total = t0 + n - edge
        nblk = _ceil(total, BLOCK)
        pad = torch.zeros(nblk * BLOCK, *rows.shape[1:], device=rows.device)
        pad[t0 - edge:total] = rows.abs()
        s = _exact_scale(pad.view(nblk, BLOCK, *rows.shape[1:]).amax((1, 3)), fmt)   # (nblk, H)
        s[0] = torch.maximum(s[0], first)
        per = s.repeat_interleave(BLOCK, 0)[:total]
        val = _exact_quant(full, per[..., None], fmt)
        kept = (s[0] == first) & (first > 0)          # the scale stands: the codes stay
        if t0 > edge:
            val[:t0 - edge] = torch.where(kept[None, :, None], c.double(), val[:t0 - edge])
        blk = edge // BLOCK + torch.arange(nblk, device=rows.device)
        scale[table[b].long()[blk * BLOCK // pt], :, blk % (pt // BLOCK)] = s
        out.append(val)
    return torch.cat(out), scale


def _exact_attend(q, case, table, lens, new, pools, causal):
    pt, fmt, at = case["pt"], case["fmt"], 0
    Hq, H, d = case["Hq"], case["Hkv"], case["d"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b in range(len(lens)):
        n, T = int(new[b]), int(lens[b] + new[b])
        k, ks = _tokens(pools["kpool"], pools["kscale"], table[b], 0, T, pt, fmt, False)
        v, vs = _tokens(pools["vpool"], pools["vscale"], table[b], 0, T, pt, fmt, True)
        k = (k * ks.double()[..., None]).permute(1, 2, 0).contiguous()          # (H, d, T)
        v = (v * vs.double()[..., None]).transpose(0, 1).contiguous()           # (H, T, d)
        x = q[at:at + n].double().view(n, H, Hq // H, d).permute(1, 2, 0, 3)
        step = max(1, (1 << 27) // (T * Hq))
        for i in range(0, n, step):
            e = min(n, i + step)
            s = torch.matmul(x[:, :, i:e].reshape(H, -1, d), k) / math.sqrt(d)
            s = s.view(H, Hq // H, e - i, T)
            if causal:
                pos = T - n + torch.arange(i, e, device=q.device)
                s = s.masked_fill(torch.arange(T, device=q.device) > pos[:, None], -math.inf)
            o = torch.matmul(torch.softmax(s, -1).view(H, -1, T), v).view(H, Hq // H, e - i, d)
            out[at + i:at + e] = o.permute(2, 0, 1, 3).reshape(e - i, Hq, d)
        at += n
    return out


def exact(case, seed):
    lens, new, P, table, free, count = _sizes(case, seed)
    pt = case["pt"]
    if case["kind"] == "plan":
        B, width, top, rows = case["B"], table.shape[1], int(count), case["rows"]
        start, got, slots, pos, short = [0], [], [-1] * rows, [0] * rows, False
        asked = 0
        for b in range(B):
            n, t0, r0 = int(new[b]), int(lens[b]), start[-1]
            start.append(r0 + n)
            ask = _ceil(t0 + n, pt) - _ceil(t0, pt)
            ok = r0 + n <= rows and _ceil(t0 + n, pt) <= width
            if ok:
                asked += ask
                ok = ask == 0 or asked <= int(count)
            got.append(n if ok else 0)
            for i in range(n if ok else 0):
                t = t0 + i
                if t % pt == 0:
                    top -= 1
                    table[b, t // pt] = free[top]
                slots[r0 + i], pos[r0 + i] = int(table[b, t // pt]) * pt + t % pt, t
        got = torch.tensor(got)
        return {"q_start": torch.tensor(start).int(), "q_lens": got.int(),
                "kv_lens": (lens + got).int(), "slots": torch.tensor(slots),
                "positions": torch.tensor(pos).int(),
                "free_count": torch.tensor([top]).int(), "table": table}
    st = prepare(case, seed)
    after = _placed(table, free, count, lens, new, pt).to("cuda")
    pools = {k: st[k] for k in ("kpool", "kscale", "vpool", "vscale")}
    fmt = case["fmt"]
    if case["kind"] == "append":
        k, ks = _exact_append(st["k"], lens, new, st["kpool"], st["kscale"], False, fmt, after, pt)
        v, vs = _exact_append(st["v"], lens, new, st["vpool"], st["vscale"], True, fmt, after, pt)
        return {"k": k, "v": v, "kscale": ks.double(), "vscale": vs.double()}
    if case["kind"] == "step":
        # the plain append's codes are exact: only the attention is computed apart
        slots = _slot_map(after.cpu(), lens, new, pt, st["rows"]).to("cuda")
        _plain_append(st, st["k"], slots, st["kpool"], st["kscale"], False)
        _plain_append(st, st["v"], slots, st["vpool"], st["vscale"], True)
    out = _exact_attend(st["q"], case, after, lens, new, pools, case.get("causal", True))
    if case["kind"] == "attend":
        return out
    return {"out": out, "slots": slots, "kv_lens": (lens + new).int(),
            "free_count": (count - (_pages_of(lens + new, pt) - _pages_of(lens, pt)).sum()).int(),
            "kscale": st["kscale"].double(), "vscale": st["vscale"].double()}
