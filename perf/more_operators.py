"""Timed cases of shared pages in the 8-bit paged cache: forks, compaction, rotary
positions, attention over a prefix that requests share.

The operators, and what a program holds of them:

* ``fork_pages`` / ``copy_pages`` / ``release_pages``: requests that go on from another's
  tokens; whole pages are shared, the page in part filled is copied, and a page is free
  again when its last holder is done (``shares``: holders beyond the first);
* ``compact_pages``: the pages in use move to the lowest places of the pool;
* ``rotary``: query and key rows turned by their positions;
* ``attention_kv8_shared``: attention of a batch in groups whose requests share a prefix.

``own`` picks what ``run`` calls: the framework's operators, or the plain forms below
(elementary torch operations in 32 bits; angles in 64).  ``exact`` is the same result in
64 bits from the definition.

Pools: pages of ``pt`` tokens with all H kv heads; ``kpool`` (P, H, pt, d), ``vpool``
(P, H, pt / 16, d, 16), ``kscale`` / ``vscale`` (P, H, pt / 16).
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"int8": (torch.int8, 127.0), "fp8": (torch.float8_e4m3fn, 448.0)}
BLOCK = 16
FLOOR = 2.0 ** -100
FINITE = torch.finfo(torch.float32).max
TWO_PI = 62831853071795864769252867665590057683943387987502116419498891846  # 2 pi 10^64


# ---------------------------------------------------------------- cases

def fork(name, templates, forks, longest, H, d, fmt="int8", pt=256, spare=1.2):
    return dict(name=name, kind="fork", templates=templates, forks=forks, longest=longest, H=H,
                d=d, fmt=fmt, pt=pt, spare=spare)


def compact(name, B, longest, H, d, empty, fmt="int8", pt=256):
    return dict(name=name, kind="compact", B=B, longest=longest, H=H, d=d, empty=empty, fmt=fmt,
                pt=pt)


def rotary(name, rows, Hq, Hkv, d, R, layout="half", far=8192, scaled=False, dtype="bf16"):
    return dict(name=name, kind="rotary", rows=rows, Hq=Hq, Hkv=Hkv, d=d, R=R, layout=layout,
                far=far, scaled=scaled, dtype=dtype)


def shared(name, B, groups, Hq, Hkv, d, prefix, T, Q=1, ragged=True, causal=True, dtype="bf16",
           out="bf16", fmt="int8", pt=256):
    return dict(name=name, kind="shared", B=B, groups=groups, Hq=Hq, Hkv=Hkv, d=d, prefix=prefix,
                T=T, Q=Q, ragged=ragged, causal=causal, dtype=dtype, out=out, fmt=fmt, pt=pt)


def listed():
    return [
        # four continuations of one prompt, a few thousand tokens long
        fork("fork_few", 1, 4, 3001, 8, 128),
        # requests admitted behind a server's 16 system prompts, 8-bit float codes
        fork("fork_many", 16, 384, 4000, 3, 96, fmt="fp8", pt=128),
        # a pool of a small model's layer after an hour of requests of all lengths
        compact("compact_small", 40, 3000, 2, 64, 0.5, pt=64),
        # a Llama-3-8B layer's pool before it gives a part of its memory back
        compact("compact_pool", 64, 9000, 8, 128, 0.4),
        # a decode step of 64 requests of a Llama-3-8B layer
        rotary("rotary_token", 64, 32, 8, 128, 128),
        # the prompt pass of the same layer
        rotary("rotary_prompt", 8192, 32, 8, 128, 128),
        # interleaved pairs, part of the head, scaled for long contexts, odd sizes, fp32
        rotary("rotary_part", 3001, 5, 1, 96, 40, "pairs", 1000000, True, "fp32"),
        # four fp32 continuations of the README's quickstart context
        shared("shared_few", 4, 1, 8, 8, 128, 512, 24, dtype="fp32", out="fp32"),
        # a Llama-3-8B layer serving 64 requests behind one system prompt of 8k tokens
        shared("shared_serving", 64, 1, 32, 8, 128, 8192, 500),
        # six prompts' requests and some of no group, head_dim 96, 8-bit float codes
        shared("shared_groups", 60, 6, 24, 8, 96, 5003, 700, dtype="fp16", out="fp16",
               fmt="fp8", pt=64),
        # questions of some hundred tokens about one document, head_dim 64, 7 query heads a kv head
        shared("shared_questions", 8, 1, 14, 2, 64, 16001, 301, Q=301, out="fp32", pt=128),
        # a whole decode step of one Qwen2.5-0.5B layer behind a shared prompt: plan, positions,
        # append, attention, 16 requests
        dict(shared("step_shared", 16, 1, 14, 2, 64, 1800, 260), kind="step"),
    ]


def _lu(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["fork", "fork", "compact", "rotary", "rotary", "decode", "decode", "groups",
                       "groups", "prompts", "prompts", "step"])
    d = rng.choice([64, 96, 128, 128])
    H = rng.choice([1, 2, 3, 4, 8])
    G = rng.choice([1, 2, 3, 4, 4, 7, 8])
    fmt = rng.choice(["int8", "int8", "fp8"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    out = rng.choice([dtype, "fp32"])
    pt = rng.choice([64, 128, 256, 256, 1024])
    if kind == "fork":
        K = _lu(rng, 1, 24)
        return fork("", K, _lu(rng, 1, 600), _lu(rng, 3, 4000), H, d, fmt, rng.choice([64, 128, 256]),
                    rng.choice([0.6, 1.2, 1.5]))
    if kind == "compact":
        T = _lu(rng, 16, 9000)
        B = max(1, min(_lu(rng, 1, 300), 2000000 // (T * H)))
        return compact("", B, T, H, d, rng.choice([0.1, 0.3, 0.4]), fmt, pt)
    if kind == "rotary":
        rows = max(1, min(_lu(rng, 1, 8192), (1 << 25) // (d * H * (G + 1))))
        R = rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)])
        return rotary("", rows, H * G, H, d, R, rng.choice(["half", "pairs"]), _lu(rng, 16, 1 << 20),
                      rng.random() < 0.4, dtype)
    if kind == "decode":
        P = _lu(rng, 40, 32000)
        T = _lu(rng, 1, 1000)
        B = max(2, min(_lu(rng, 2, 128), 4000000 // (H * (P + T))))
        return shared("", B, 1, H * G, H, d, P, T, Q=min(T, rng.choice([1, 1, 1, 3])),
                      ragged=rng.random() < 0.6, dtype=dtype, out=out, fmt=fmt, pt=pt)
    if kind == "groups":
        P = _lu(rng, 40, 8000)
        T = _lu(rng, 1, 1000)
        B = max(6, min(_lu(rng, 6, 100), 4000000 // (H * (P + T))))
        return shared("", B, rng.randint(2, max(2, B // 4)), H * G, H, d, P, T, dtype=dtype,
                      out=out, fmt=fmt, pt=pt, causal=rng.random() < 0.7)
    if kind == "prompts":
        Q = _lu(rng, 9, 400)
        T = Q + _lu(rng, 1, 400)
        B = _lu(rng, 2, 12)
        P = max(40, min(_lu(rng, 40, 16000), (1 << 29) // (H * G * Q * B) - T))
        return shared("", B, rng.choice([1, 1, 2]), H * G, H, d, P, T, Q=Q, dtype=dtype, out=out,
                      fmt=fmt, pt=pt, causal=rng.random() < 0.8)
    P = _lu(rng, 40, 8000)
    return dict(shared("", max(2, min(_lu(rng, 2, 64), 2000000 // (H * P))), 1, H * G, H, d, P,
                       _lu(rng, 2, 500), dtype=dtype, out=dtype, fmt=fmt, pt=pt), kind="step")


# --------------------------------------------------- sizes (host)

def _ceil(a, b):
    return -(-a // b)


def _batch(case):
    """(group starts, prefix lengths, cached tokens before the call, new tokens) of a batch.
    The last request of a batch with several groups is in none; where the batch is ragged some
    requests are idle."""
    g = torch.Generator().manual_seed(17)
    B, n, P, T, Q = (case[k] for k in ("B", "groups", "prefix", "T", "Q"))
    cuts = (torch.randperm(B - 1, generator=g)[:n - 1] + 1).sort().values.tolist() if n > 1 else []
    start = [0] + cuts + [B]
    if n > 1:
        start[-1] = max(B - 1, start[-2])
    prefix = (P * torch.rand(n, generator=g)).long() + 1
    prefix[0] = P
    mine = torch.full((B,), T)
    new = torch.full((B,), Q)
    if case["ragged"]:
        mine = (T * torch.rand(B, generator=g).double() ** 2).long() + 1
        mine[0] = T
        if Q > 8:
            new = (Q * (0.3 + 0.7 * torch.rand(B, generator=g))).long() + 1
            new[0] = Q
    new = torch.minimum(new, torch.tensor(Q))
    mine = torch.maximum(mine, new)
    kv = mine.clone()
    for i in range(n):
        kv[start[i]:start[i + 1]] += prefix[i]
    if case["ragged"] and case["kind"] != "step":
        kv[7::16] = 0
        new[7::16] = 0
    if case["kind"] == "step":
        new[:] = 1
    return start, prefix.tolist(), kv - new, new


def _placed(case, seed):
    """The batch with its pages at random places of the pool: dict(P, table, free, count, copies),
    copies (from page, to page, blocks): pages in part filled by the prefix, of which every
    request has one of its own."""
    start, prefix, lens, new = _batch(case)
    pt, kv = case["pt"], lens + new
    held = lens if case["kind"] == "step" else kv
    need = int(((held + pt - 1) // pt).sum()) + sum(_ceil(p, pt) for p in prefix) + case["B"] + 3
    order = torch.randperm(need, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.zeros(case["B"], int(((kv + pt - 1) // pt).max()) + 1, dtype=torch.int32)
    at, copies = 0, []
    group = [(start[i], start[i + 1], prefix[i]) for i in range(len(prefix))]
    for b0, b1, p in group + [(b, b + 1, 0) for b in range(start[-1], case["B"])]:
        whole, part = p // pt, p % pt
        first = None
        common = order[at:at + whole]
        at += whole
        for b in range(b0, b1):
            if kv[b] == 0:
                continue
            n = _ceil(int(held[b]), pt) - whole
            table[b, :whole] = common
            table[b, whole:whole + n] = order[at:at + n]
            at += n
            if part and n > 0:
                if first is None:
                    first = b
                else:
                    copies.append((int(table[first, whole]), int(table[b, whole]),
                                   _ceil(part, BLOCK)))
    return dict(P=need, table=table, free=order.clone().roll(-at), count=need - at, copies=copies,
                start=start, prefix=prefix, lens=lens, new=new)


def _books(case, seed):
    """Page tables of the fork and compact cases (host): dict of int32 tensors and P."""
    g = torch.Generator().manual_seed(seed)
    fixed = torch.Generator().manual_seed(17)
    pt = case["pt"]
    if case["kind"] == "fork":
        K, F = case["templates"], case["forks"]
        B = K + F
        lens = torch.zeros(B, dtype=torch.int32)
        lens[:K] = (case["longest"] * (0.3 + 0.7 * torch.rand(K, generator=fixed))).int() + 1
        lens[0] = case["longest"]
        src = torch.randint(0, K, (F,), generator=fixed).int()
        dst = (K + torch.randperm(F, generator=fixed)).int()
        # most go on behind the whole prompt, some behind a part of it
        tokens = lens[src.long()].clone()
        part = torch.rand(F, generator=fixed) < 0.2
        tokens[part] = (tokens[part] * torch.rand(F, generator=fixed)[part]).int()
        if F > 20:   # calls that are refused: a request that holds tokens, one named before
            dst[5], dst[9], src[11] = 0, dst[8], B
        held = (lens + pt - 1) // pt
        P = int(held.sum()) + max(1, int(case["spare"] * int((tokens % pt > 0).sum())))
        width = int(held.max()) + 2
        more = dict(src=src, dst=dst, tokens=tokens)
        shares = torch.zeros(P, dtype=torch.int32)
    else:
        B = case["B"]
        lens = (case["longest"] * torch.rand(B, generator=fixed).double() ** 1.5).int() + 1
        lens[0] = case["longest"]
        held = (lens + pt - 1) // pt
        P = max(2, int(int(held.sum()) / (1 - case["empty"])))
        width = int(held.max()) + 1
        more = {}
        shares = torch.zeros(P, dtype=torch.int32)
    order = torch.randperm(P, generator=g).int()
    table = torch.zeros(B, width, dtype=torch.int32)
    at = 0
    for b in range(B):
        n = int(held[b])
        table[b, :n] = order[at:at + n]
        if case["kind"] == "compact" and b % 3 == 1:    # shares its first pages with the one before
            both = min(n, int(held[b - 1])) // 2
            table[b, :both] = table[b - 1, :both]
            shares[table[b, :both].long()] += 1
            table[b, both:n] = order[at:at + n - both]
            n -= both
        at += n
    count = P - at
    free = torch.zeros(P, dtype=torch.int32)
    free[:count] = order[at:]
    return dict(P=P, table=table, lens=lens, free=free,
                free_count=torch.tensor([count], dtype=torch.int32), shares=shares, **more)


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


def _scatter(size, at, keep, values, fill, like):
    """A tensor of `size` values `fill` with `values` at `at` where `keep`."""
    out = torch.full((size + 1,), fill, dtype=like.dtype, device=like.device)
    out[torch.where(keep, at, torch.full_like(at, size)).long()] = values.to(like.dtype)
    return out[:size]


def _plain_fork(st, book):
    table, lens, shares = book["table"], book["lens"], book["shares"]
    src, dst, pt = st["src"].long(), st["dst"].long(), st["pt"]
    B, W = table.shape
    F = src.numel()
    valid = (src >= 0) & (src < B) & (dst >= 0) & (dst < B) & (src != dst)
    i = torch.arange(F, device=src.device)
    s, t = src.clamp(0, B - 1), dst.clamp(0, B - 1)
    first = torch.full((B + 1,), F, device=src.device)
    first.scatter_reduce_(0, torch.where(valid, t, torch.full_like(t, B)), i, "amin")
    valid &= (lens[t] == 0) & (first[t] == i)
    n = torch.minimum(st["tokens"].long().clamp(min=0), lens[s].long().clamp(0, W * pt))
    ask = (valid & (n % pt > 0)).long()
    top = torch.cumsum(ask, 0)
    count = book["free_count"].long()
    ok = valid & ((ask == 0) | (top <= count))
    part = ok & (ask > 0)
    fresh = book["free"][(count - top).clamp(0, book["free"].numel() - 1)]
    whole = torch.where(ok, n // pt, torch.zeros_like(n))
    col = torch.arange(W, device=src.device)
    mine = col < whole[:, None]
    rows = table[s]
    P = shares.numel()
    page = torch.where(mine, rows, torch.full_like(rows, P)).long()
    more = torch.zeros(P + 1, dtype=torch.int32, device=src.device)
    more.index_add_(0, page.reshape(-1), torch.ones_like(page, dtype=torch.int32).reshape(-1))
    shares += more[:P]
    from_page = rows.gather(1, (n // pt).clamp(max=W - 1)[:, None])[:, 0]
    to = torch.where(mine, rows, table[t])
    to = torch.where((col == whole[:, None]) & part[:, None], fresh[:, None], to)
    wide = torch.cat([table, table[:1]])
    wide[torch.where(ok, t, torch.full_like(t, B))] = to
    table.copy_(wide[:B])
    full = torch.cat([lens, lens[:1]])
    full[torch.where(ok, t, torch.full_like(t, B))] = n.int()
    lens.copy_(full[:B])
    book["free_count"].sub_(part.sum().int())
    none = torch.full_like(fresh, -1)
    return {"granted": torch.where(ok, n, torch.full_like(n, -1)).int(),
            "src_pages": torch.where(part, from_page, none),
            "dst_pages": torch.where(part, fresh, none),
            "copy_tokens": torch.where(part, n % pt, torch.zeros_like(n)).int()}


def _plain_copy(st, src, dst, tokens):
    ok = dst >= 0
    src, dst = src[ok].long(), dst[ok].long()
    nb = st["pt"] // BLOCK
    blocks = torch.full_like(dst, nb) if tokens is None else (tokens[ok].long() + BLOCK - 1) // BLOCK
    keep = torch.arange(nb, device=dst.device) < blocks[:, None]              # (moves, nb)
    for name in ("kpool", "vpool", "kscale", "vscale"):
        pool = st[name]
        flat = pool if pool.element_size() == 4 else pool.view(torch.int8)
        flat = flat.view(flat.shape[0], flat.shape[1], nb, -1)
        flat[dst] = torch.where(keep[:, None, :, None], flat[src], flat[dst])


def _plain_release(st, book, done):
    table, lens, shares, free = (book[k] for k in ("table", "lens", "shares", "free"))
    B, W = table.shape
    P, pt = shares.numel(), st["pt"]
    held = torch.where(done, (lens.clamp(min=0) + pt - 1) // pt, torch.zeros_like(lens))
    mine = (torch.arange(W, device=lens.device) < held[:, None]) & (table >= 0) & (table < P)
    page = torch.where(mine, table, torch.full_like(table, P)).long().reshape(-1)
    e = torch.arange(B * W, device=lens.device)
    gone = torch.zeros(P + 1, dtype=torch.int32, device=lens.device)
    gone.index_add_(0, page, torch.ones_like(page, dtype=torch.int32))
    last = torch.full((P + 1,), -1, device=lens.device)
    last.scatter_reduce_(0, page, e, "amax")
    left = shares - gone[:P]
    out = torch.cat([left < 0, left.new_zeros(1, dtype=torch.bool)])[page] & (last[page] == e)
    out &= mine.reshape(-1)
    at = book["free_count"].long() + torch.cumsum(out.long(), 0) - 1
    wide = torch.cat([free, free[:1]])
    wide[torch.where(out, at, torch.full_like(at, P)).clamp(max=P)] = table.reshape(-1)
    free.copy_(wide[:P])
    book["free_count"].copy_((book["free_count"] + out.sum()).clamp(max=P))
    shares.copy_(left.clamp(min=0))
    lens.copy_(torch.where(done, torch.zeros_like(lens), lens))


def _plain_compact(st, book):
    table, lens, shares, free = (book[k] for k in ("table", "lens", "shares", "free"))
    P, pt = shares.numel(), st["pt"]
    ids = torch.arange(P, device=lens.device)
    live = ids < book["free_count"]
    used = _scatter(P, free, live, torch.zeros_like(free), 1, ids) > 0
    U = used.sum()
    mover, hole = used & (ids >= U), ~used & (ids < U)
    half = P // 2
    src = _scatter(half, torch.cumsum(mover.long(), 0) - 1, mover, ids, -1, table)
    dst = _scatter(half, torch.cumsum(hole.long(), 0) - 1, hole, ids, -1, table)
    moved = src >= 0
    remap = torch.cat([ids, ids[:1]]).int()
    remap[torch.where(moved, src, torch.full_like(src, P)).long()] = dst
    remap = remap[:P]
    held = (lens.clamp(min=0) + pt - 1) // pt
    mine = (torch.arange(table.shape[1], device=lens.device) < held[:, None]) & (table >= 0)
    mine &= table < P
    table.copy_(torch.where(mine, remap[table.clamp(0, P - 1).long()], table))
    now = _scatter(P, remap, used, shares, 0, shares)
    shares.copy_(torch.where(used | (ids < U), now, shares))
    free.copy_(torch.where(live, (P - 1 - ids).int(), free))
    return {"src_pages": src, "dst_pages": dst, "moves": moved.sum().int().view(1), "remap": remap}


def _plain_rotary(x, st):
    """x (rows, H, d) turned by its rows' positions, in its own type."""
    R = st["R"]
    a = st["positions"].double()[:, None] * st["inv_freq"]
    cos = (torch.cos(a) * st["factor"]).float()[:, None]
    sin = (torch.sin(a) * st["factor"]).float()[:, None]
    y = x.float()
    if st["layout"] == "half":
        u, v = y[..., :R // 2], y[..., R // 2:R]
        turned = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
    else:
        u, v = y[..., :R:2], y[..., 1:R:2]
        turned = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
    return torch.cat([turned, y[..., R:]], -1).to(x.dtype)


def _plain_plan(st):
    """plan_pages where every request is served."""
    table, pt, rows = st["table"], st["pt"], st["rows"]
    lens, new = st["lens"].long(), st["new"].long()
    B, W = table.shape
    ends = torch.cumsum(new, 0)
    held, want = (lens + pt - 1) // pt, (lens + new + pt - 1) // pt
    top = torch.cumsum(want - held, 0)
    count = st["free_count"].long()
    col = torch.arange(W, device=table.device)
    fresh = (col >= held[:, None]) & (col < want[:, None])
    at = count - 1 - (top - want + held)[:, None] - (col - held[:, None])
    table.copy_(torch.where(fresh, st["free"][at.clamp(0, st["free"].numel() - 1)], table))
    r = torch.arange(rows, device=table.device)
    b = torch.searchsorted(ends, r, right=True)
    t = lens[b] + r - (ends - new)[b]
    return {"kv_lens": (lens + new).int(), "positions": t.int(),
            "slots": table[b, t // pt].long() * pt + t % pt,
            "q_start": torch.cat([ends.new_zeros(1), ends]).int()}


def _plain_append(st, x, slots, pool, scale, transposed):
    """One row x (B, H, d) a request into the pool, behind the tokens that its block holds."""
    fmt, pt = st["fmt"], st["pt"]
    codes = pool.view(torch.int8)
    H = x.shape[1]
    h = torch.arange(H, device=x.device)
    k = torch.arange(BLOCK, device=x.device)
    page, o = slots // pt, slots % pt
    blk, j = o // BLOCK, o % BLOCK
    x = x.float()
    old = torch.where((j > 0)[:, None], scale[page[:, None], h, blk[:, None]], 0.0)
    s = torch.maximum(old, _scale_of(x.abs().amax(-1), fmt))
    inv = _inverse(s)
    if transposed:
        place = (page[:, None], h, blk[:, None])
        was = codes[place].transpose(-1, -2)                                    # (B, H, 16, d)
    else:
        place = (page[:, None, None], h[:, None], blk[:, None, None] * BLOCK + k)
        was = codes[place]
    again = _values(was, fmt) * old[..., None, None]
    again = _codes_of(again.double() * inv.double()[..., None, None], fmt)
    grew = (s > old)[..., None] & (k < j[:, None, None])
    now = torch.where(grew[..., None], again, was)
    fresh = _codes_of(x.double() * inv.double()[..., None], fmt)
    now = torch.where((k == j[:, None, None])[..., None], fresh[:, :, None], now)
    codes[place] = now.transpose(-1, -2) if transposed else now
    scale[page[:, None], h, blk[:, None]] = s


def _dense(st, table):
    """The cache as (B, H, T, d) keys and values, T = the longest request's pages."""
    fmt, pt = st["fmt"], st["pt"]
    pages = table[:, :_ceil(st["T"], pt)].long()
    B, W = pages.shape
    _, H, _, d = st["kpool"].shape
    k = _values(st["kpool"].view(torch.int8)[pages], fmt).view(B, W, H, pt // BLOCK, BLOCK, d)
    k = k * st["kscale"][pages][..., None, None]                              # (B, W, H, nb, 16, d)
    v = _values(st["vpool"].view(torch.int8)[pages], fmt) * st["vscale"][pages][..., None, None]
    v = v.transpose(-1, -2)
    return (k.permute(0, 2, 1, 3, 4, 5).reshape(B, H, W * pt, d),
            v.permute(0, 2, 1, 3, 4, 5).reshape(B, H, W * pt, d))


def _plain_attend(st, q, table, q_start, q_lens, kv_lens, out):
    N, Hq, d = q.shape
    k, v = _dense(st, table)
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


BOOK = ("table", "lens", "free", "free_count", "shares")


def _views(flat, shapes):
    """The parts of a flat int32 tensor, in BOOK's order."""
    sizes = [math.prod(s) for s in shapes]
    return {k: x.view(s) for k, x, s in zip(BOOK, flat.split(sizes), shapes)}


def _frequencies(case):
    """(angles per position in radians (64 bits), the factor of sine and cosine): a base of
    10000; scaled: the long waves eight times as long, the short ones as they are."""
    R = case["R"]
    w = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    if not case["scaled"]:
        return w, 1.0
    turns = 4096 * w / (2 * math.pi)          # within the original context
    keep = ((turns - 1) / 31).clamp(0, 1)
    return w * (keep + (1 - keep) / 8), 0.1 * math.log(8) + 1


def _turns(w):
    """Angles per position as turns in units of 2^-64, rounded."""
    pairs = [x.as_integer_ratio() for x in w.tolist()]
    whole = [(2 * n * 10 ** 64 * 2 ** 64 + d * TWO_PI) // (2 * d * TWO_PI) % 2 ** 64
             for n, d in pairs]
    return torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in whole])


def _spin(case, dev):
    w, factor = _frequencies(case)
    return dict(inv_freq=w.to(dev), turns=_turns(w).to(dev), factor=factor, R=case["R"],
                layout=case["layout"])


def prepare(case, seed):
    kind = case["kind"]
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    dev = "cuda"
    if kind == "rotary":
        rows, Hq, H, d = (case[k] for k in ("rows", "Hq", "Hkv", "d"))
        x = torch.randn(rows, (Hq + 2 * H) * d, generator=gen, device=dev).to(DTYPES[case["dtype"]])
        # runs of positions, as of chunks of prompts, or of decoding requests
        pos = torch.randint(0, case["far"], (rows,), generator=gen, device=dev)
        run_ = torch.arange(rows, device=dev) % 37
        pos = torch.where(pos % 3 > 0, (pos // 37 * 37 + run_).clamp(max=case["far"] - 1), pos)
        return dict(kind=kind, q=x[:, :Hq * d].unflatten(1, (Hq, d)),
                    k=x[:, Hq * d:(Hq + H) * d].unflatten(1, (H, d)), positions=pos.int(),
                    **_spin(case, dev))
    if kind in ("fork", "compact"):
        books = _books(case, seed)
        st = dict(kind=kind, pt=case["pt"], fmt=case["fmt"])
        st["shapes"] = [tuple(books[k].shape) for k in BOOK]
        st["book"] = torch.cat([books[k].reshape(-1) for k in BOOK]).to(dev)
        for k in ("src", "dst", "tokens"):
            if k in books:
                st[k] = books[k].to(dev)
        if kind == "fork":
            st["done"] = torch.arange(books["lens"].numel(), device=dev) >= case["templates"]
        st.update(_pools(case, books["P"], seed + 2))
        return st
    b = _placed(case, seed)
    lens, new = b["lens"], b["new"]
    st = dict(kind=kind, pt=case["pt"], fmt=case["fmt"], causal=case["causal"],
              table=b["table"].to(dev), T=int((lens + new).max()), Q=int(new.max()))
    st.update(_pools(case, b["P"], seed + 2))
    for s, t, n in b["copies"]:
        for name in ("kpool", "vpool", "kscale", "vscale"):
            x = st[name] if st[name].element_size() == 4 else st[name].view(torch.int8)
            m = n * BLOCK if name == "kpool" else n
            x[t, :, :m] = x[s, :, :m]
    st["group_start"] = torch.tensor(b["start"], dtype=torch.int32, device=dev)
    st["prefix_lens"] = torch.tensor(b["prefix"], dtype=torch.int32, device=dev)
    N, Hq, H, d = int(new.sum()), case["Hq"], case["Hkv"], case["d"]
    dtype = DTYPES[case["dtype"]]
    st["out"] = torch.zeros(N, Hq, d, dtype=DTYPES[case["out"]], device=dev)
    if kind == "step":
        st.update(rows=N, lens=lens.int().to(dev), new=new.int().to(dev), free=b["free"].to(dev),
                  free_count=torch.tensor([b["count"]], dtype=torch.int32, device=dev))
        x = torch.randn(N, (Hq + 2 * H) * d, generator=gen, device=dev).to(dtype)
        st["q"] = x[:, :Hq * d].unflatten(1, (Hq, d))
        st["k"] = x[:, Hq * d:(Hq + H) * d].unflatten(1, (H, d))
        st["v"] = x[:, (Hq + H) * d:].unflatten(1, (H, d))
        st.update(_spin(dict(R=d, layout="half", scaled=False), dev))
        return st
    st["q_start"] = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(new, 0)]).int().to(dev)
    st["q_lens"], st["kv_lens"] = new.int().to(dev), (lens + new).int().to(dev)
    st["q"] = torch.randn(N, Hq, d, generator=gen, device=dev).to(dtype)
    return st


def _held(st):
    """The pools as a fork or a compaction leaves them: their codes are copied, not computed."""
    return {"kcodes": st["kpool"].view(torch.int8), "vcodes": st["vpool"].view(torch.int8),
            "kscale": st["kscale"], "vscale": st["vscale"]}


def run(st):
    kind = st["kind"]
    if kind in ("fork", "compact"):
        # (the tables before are kept, as by a program that may step back)
        book = _views(st["book"].clone(), st["shapes"])
    if own:
        from quashkv_amd import paged8
        from quashkv_amd import rotary as rot
        pools = {k: st[k] for k in ("kpool", "kscale", "vpool", "vscale") if k in st}
        if kind == "rotary":
            q, k = rot.rotary(st["q"], st["k"], st["positions"], st["turns"], st["factor"],
                              interleaved=st["layout"] == "pairs")
            return {"q": q, "k": k}
        if kind == "fork":
            p = paged8.fork_pages(book["table"], book["lens"], st["src"], st["dst"], st["tokens"],
                                  book["free"], book["free_count"], book["shares"], st["pt"])
            paged8.copy_pages(p.src_pages, p.dst_pages, **pools, tokens=p.copy_tokens)
            paged8.release_pages(book["table"], book["lens"], st["done"], book["free"],
                                 book["free_count"], st["pt"], shares=book["shares"])
            return {"granted": p.granted, "src_pages": p.src_pages, "dst_pages": p.dst_pages,
                    "copy_tokens": p.copy_tokens, **book, **_held(st)}
        if kind == "compact":
            p = paged8.compact_pages(book["table"], book["lens"], book["free"], book["free_count"],
                                     st["pt"], shares=book["shares"])
            paged8.copy_pages(p.src_pages, p.dst_pages, **pools, count=p.moves)
            return {"src_pages": p.src_pages, "dst_pages": p.dst_pages, "moves": p.moves,
                    "remap": p.remap, **book, **_held(st)}
        if kind == "step":
            p = paged8.plan_pages(st["table"], st["lens"], st["new"], st["free"],
                                  st["free_count"], st["rows"], st["pt"])
            q, k = rot.rotary(st["q"], st["k"], p.positions, st["turns"], st["factor"])
            paged8.append_kv8(k, st["v"], p.slots, **pools)
            out = paged8.attention_kv8_shared(
                q, **pools, table=st["table"], kv_lens=p.kv_lens, group_start=st["group_start"],
                prefix_lens=st["prefix_lens"], q_start=p.q_start, q_lens=p.q_lens, causal=True,
                out=st["out"])
            return {"out": out, "slots": p.slots, "positions": p.positions, "kv_lens": p.kv_lens,
                    "kscale": st["kscale"], "vscale": st["vscale"]}
        return paged8.attention_kv8_shared(
            st["q"], **pools, table=st["table"], kv_lens=st["kv_lens"],
            group_start=st["group_start"], prefix_lens=st["prefix_lens"], q_start=st["q_start"],
            q_lens=st["q_lens"], causal=st["causal"], out=st["out"])
    if kind == "rotary":
        return {"q": _plain_rotary(st["q"], st), "k": _plain_rotary(st["k"], st)}
    if kind == "fork":
        p = _plain_fork(st, book)
        _plain_copy(st, p["src_pages"], p["dst_pages"], p["copy_tokens"])
        _plain_release(st, book, st["done"])
        return {**p, **book, **_held(st)}
    if kind == "compact":
        p = _plain_compact(st, book)
        _plain_copy(st, p["src_pages"], p["dst_pages"], None)
        return {**p, **book, **_held(st)}
    if kind == "step":
        p = _plain_plan(st)
        turn = dict(st, positions=p["positions"])
        q, k = _plain_rotary(st["q"], turn), _plain_rotary(st["k"], turn)
        _plain_append(st, k, p["slots"], st["kpool"], st["kscale"], False)
        _plain_append(st, st["v"], p["slots"], st["vpool"], st["vscale"], True)
        out = _plain_attend(st, q, st["table"], p["q_start"], st["new"], p["kv_lens"], st["out"])
        return {"out": out, "slots": p["slots"], "positions": p["positions"],
                "kv_lens": p["kv_lens"], "kscale": st["kscale"], "vscale": st["vscale"]}
    return _plain_attend(st, st["q"], st["table"], st["q_start"], st["q_lens"], st["kv_lens"],
                         st["out"])


# ---------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    if kind == "rotary":
        n = case["rows"] * (case["Hq"] + case["Hkv"])
        return {"bytes": 2 * size[case["dtype"]] * n * case["d"] + 4 * case["rows"],
                "flops": 3 * n * case["R"]}
    d, pt = case["d"], case["pt"]
    if kind in ("fork", "compact"):
        book = _books(case, 0)
        _, pairs, counts = _exact_books(case, book)
        block = 2 * case["H"] * (BLOCK * d + 4)
        blocks = sum(_ceil(n, BLOCK) for _, _, n in pairs)
        entries = int(((book["lens"] + pt - 1) // pt).sum())
        small = 12 * case["forks"] + 24 * counts if kind == "fork" else 8 * entries + 8 * book["P"]
        return {"bytes": 2 * block * blocks + small, "flops": 0}
    start, prefix, lens, new = _batch(case)
    Hq, H = case["Hq"], case["Hkv"]
    kv, n = lens + new, int(new.sum())
    tokens = int(kv.sum())
    for i, p in enumerate(prefix):
        live = int((kv[start[i]:start[i + 1]] > 0).sum())
        tokens -= max(0, live - 1) * p
    seen = kv * new
    if case["causal"]:
        seen = (lens + 1 + kv) * new // 2
    w = {"bytes": 2 * H * tokens * d + H * tokens // 2
         + n * Hq * d * (size[case["dtype"]] + size[case["out"]]),
         "flops": 4 * d * Hq * int(seen.sum())}
    if kind == "step":    # rows turned (query and key, in and out), and both halves in the cache
        e = size[case["dtype"]]
        w["bytes"] += n * d * (2 * e * (Hq + H) + H * (2 * e + 2)) + 16 * n * H + 12 * n
    return w


# --------------------------------------------------------------------- exact

def _exact_books(case, book):
    """(outputs, pages copied as (from, to, tokens), entries touched), request by request."""
    pt, P = case["pt"], book["P"]
    table, lens = book["table"].tolist(), book["lens"].tolist()
    shares, count = book["shares"].tolist(), int(book["free_count"])
    free = book["free"].tolist()
    B = len(lens)
    pairs, touched = [], 0
    if case["kind"] == "fork":
        src, dst, tokens = (book[k].tolist() for k in ("src", "dst", "tokens"))
        before, named = list(lens), set()
        rows = [list(r) for r in table]
        top = count
        asked, got = 0, []
        res = {"granted": [], "src_pages": [], "dst_pages": [], "copy_tokens": []}
        for s, t, n in zip(src, dst, tokens):
            ok = 0 <= s < B and 0 <= t < B and s != t
            if ok:
                ok = t not in named and before[t] == 0
                named.add(t)
            n = min(max(n, 0), before[s]) if ok else 0
            if ok and n % pt:
                asked += 1
                ok = asked <= count
            new = (-1, -1, 0)
            if ok:
                whole = n // pt
                for c in range(whole):
                    rows[t][c] = table[s][c]
                    shares[table[s][c]] += 1
                if n % pt:
                    top -= 1
                    rows[t][whole] = free[top]
                    new = (table[s][whole], free[top], n % pt)
                    pairs.append(new)
                lens[t] = n
                got.append(t)
                touched += _ceil(n, pt)
            res["granted"].append(n if ok else -1)
            for k, x in zip(("src_pages", "dst_pages", "copy_tokens"), new):
                res[k].append(x)
        # and back: the forked requests are done
        left = top
        held = [(b, c) for b in range(case["templates"], B) for c in range(_ceil(lens[b], pt))]
        last = {rows[b][c]: (b, c) for b, c in held}
        over = dict.fromkeys(last, 0)
        for b, c in held:
            over[rows[b][c]] += 1
        for b, c in held:
            p = rows[b][c]
            if last[p] == (b, c):
                shares[p] -= over[p]
                if shares[p] < 0:
                    shares[p] = 0
                    free[left] = p
                    left += 1
        lens[case["templates"]:] = [0] * case["forks"]
        res.update(table=rows, lens=lens, free=free, free_count=[left], shares=shares)
        return res, pairs, touched
    spare = set(free[:count])
    U = P - count
    movers = [p for p in range(U, P) if p not in spare]
    holes = [p for p in range(U) if p in spare]
    to = dict(zip(movers, holes))
    for b in range(B):
        for c in range(_ceil(lens[b], pt)):
            table[b][c] = to.get(table[b][c], table[b][c])
    for s, t in to.items():
        shares[t], shares[s] = shares[s], 0
    pad = [-1] * (P // 2 - len(movers))
    res = {"src_pages": movers + pad, "dst_pages": holes + pad, "moves": [len(movers)],
           "remap": [to.get(p, p) for p in range(P)], "table": table, "lens": lens,
           "free": [P - 1 - i for i in range(count)] + free[count:], "free_count": [count],
           "shares": shares}
    return res, [(s, t, pt) for s, t in to.items()], B


def _exact_quant(x, s, fmt):
    """The values (64 bits) that x stands for at fp32 scales s, from the definition."""
    top = CODES[fmt][1]
    inv = torch.where(s > 0, (1.0 / s.double()).float().double(), torch.zeros_like(s).double())
    y = (x.double() * inv).clamp(-top, top)
    if fmt == "int8":
        return torch.round(y) * s.double()
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30)))
    e = torch.where(y.abs() < torch.exp2(e), e - 1, e)
    e = torch.where(y.abs() >= torch.exp2(e + 1), e + 1, e).clamp(min=-6)
    return torch.round(y * torch.exp2(3 - e)) * torch.exp2(e - 3) * s.double()


def _tokens(pool, scale, row, T, pt, fmt, transposed):
    """The first T tokens of a request as (T, H, d): the codes' values in 64 bits, and scales."""
    t = torch.arange(T, device=pool.device)
    page, o = row.long()[t // pt], t % pt
    raw = pool.view(torch.int8)
    c = raw[page, :, o // BLOCK, :, o % BLOCK] if transposed else raw[page, :, o]
    c = c.double() if fmt == "int8" else c.view(torch.float8_e4m3fn).double()
    return c, scale[page, :, o // BLOCK]


def _exact_attend(q, case, n, T, k, v, causal):
    """One request's rows q (n, Hq, d) over k, v (T, H, d) in 64 bits."""
    Hq, H, d = case["Hq"], case["Hkv"], case["d"]
    k = k.permute(1, 2, 0).contiguous()                                       # (H, d, T)
    v = v.transpose(0, 1).contiguous()                                        # (H, T, d)
    x = q.double().view(n, H, Hq // H, d).permute(1, 2, 0, 3)
    out = torch.zeros(n, Hq, d, dtype=torch.float64, device=q.device)
    step = max(1, (1 << 27) // (T * Hq))
    for i in range(0, n, step):
        e = min(n, i + step)
        s = torch.matmul(x[:, :, i:e].reshape(H, -1, d), k) / math.sqrt(d)
        s = s.view(H, Hq // H, e - i, T)
        if causal:
            pos = T - n + torch.arange(i, e, device=q.device)
            s = s.masked_fill(torch.arange(T, device=q.device) > pos[:, None], -math.inf)
        o = torch.matmul(torch.softmax(s, -1).view(H, -1, T), v).view(H, Hq // H, e - i, d)
        out[i:e] = o.permute(2, 0, 1, 3).reshape(e - i, Hq, d)
    return out


def _exact_turn(x, positions, w, factor, layout):
    """x (rows, H, d) as complex numbers times factor e^(i position w), in 64 bits."""
    x, n = x.double(), w.numel()
    head, tail = x[..., :2 * n], x[..., 2 * n:]
    pairs = head.unflatten(-1, (2, n)).transpose(-1, -2) if layout == "half" else \
        head.unflatten(-1, (n, 2))
    z = torch.view_as_complex(pairs.contiguous())
    a = (positions.double()[:, None] * w)[:, None]
    z = torch.view_as_real(z * torch.polar(torch.full_like(a, factor), a))
    z = z.transpose(-1, -2) if layout == "half" else z
    return torch.cat([z.flatten(-2), tail], -1)


def exact(case, seed):
    kind = case["kind"]
    st = prepare(case, seed)
    if kind == "rotary":
        turn = (st["positions"], st["inv_freq"], st["factor"], st["layout"])
        return {"q": _exact_turn(st["q"], *turn), "k": _exact_turn(st["k"], *turn)}
    if kind in ("fork", "compact"):
        book = _books(case, seed)
        res, pairs, _ = _exact_books(case, book)
        res = {k: torch.tensor(x, dtype=torch.int32) for k, x in res.items()}
        for s, t, n in pairs:
            b = _ceil(n, BLOCK)
            st["kpool"].view(torch.int8)[t, :, :b * BLOCK] = \
                st["kpool"].view(torch.int8)[s, :, :b * BLOCK]
            st["vpool"].view(torch.int8)[t, :, :b] = st["vpool"].view(torch.int8)[s, :, :b]
            st["kscale"][t, :, :b] = st["kscale"][s, :, :b]
            st["vscale"][t, :, :b] = st["vscale"][s, :, :b]
        held = _held(st)
        return {**res, **held, "kscale": held["kscale"].double(), "vscale": held["vscale"].double()}
    b = _placed(case, seed)
    lens, new = b["lens"], b["new"]
    table, fmt, pt = b["table"].to("cuda"), case["fmt"], case["pt"]
    q, top = st["q"], b["count"]
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    scales = [st["kscale"].clone(), st["vscale"].clone()]
    slots, at = [], 0
    if kind == "step":
        q = _exact_turn(q, lens.to("cuda"), st["inv_freq"], 1.0, "half").to(q.dtype)
        kt = _exact_turn(st["k"], lens.to("cuda"), st["inv_freq"], 1.0, "half").to(q.dtype)
    for r in range(case["B"]):
        n, t0 = int(new[r]), int(lens[r])
        T = t0 + n
        if n == 0:
            continue
        if kind == "step" and t0 % pt == 0:
            top -= 1
            table[r, t0 // pt] = int(b["free"][top])
        kv = []
        for half, (p, s) in enumerate((("kpool", "kscale"), ("vpool", "vscale"))):
            c, sc = _tokens(st[p], scales[half], table[r], T, pt, fmt, half == 1)
            x = c * sc.double()[..., None]
            if kind == "step":
                row = (kt if half == 0 else st["v"])[at].float()             # (H, d)
                page, blk = int(table[r, t0 // pt]), t0 % pt // BLOCK
                j = t0 % BLOCK
                old = scales[half][page, :, blk] if j else torch.zeros_like(sc[0])
                a = row.abs().amax(-1).double() * float(torch.tensor(1.0 / CODES[fmt][1]))
                s_new = a.float().clamp(min=FLOOR) * (a > 0)
                s_new = torch.maximum(old, s_new)
                if j:
                    again = _exact_quant(x[T - 1 - j:T - 1].float(), s_new[None, :, None], fmt)
                    x[T - 1 - j:T - 1] = torch.where((s_new > old)[None, :, None], again,
                                                     x[T - 1 - j:T - 1])
                x[T - 1] = _exact_quant(row, s_new[:, None], fmt)
                scales[half][page, :, blk] = s_new
            kv.append(x)
        slots.append(int(table[r, (T - 1) // pt]) * pt + (T - 1) % pt)
        out[at:at + n] = _exact_attend(q[at:at + n], case, n, T, *kv, case["causal"])
        at += n
    if kind == "shared":
        return out
    return {"out": out, "slots": torch.tensor(slots), "positions": lens.int(),
            "kv_lens": (lens + new).int(), "kscale": scales[0].double(),
            "vscale": scales[1].double()}
