"""Shared pages of the 8-bit cache from their definitions: forks, releases and compactions by
loops over requests and pages, and rotary positions with integer turns."""

import math

import torch


def held(n, pt):
    return -(-max(n, 0) // pt)


def fork(table, lens, src, dst, tokens, free, count, shares, pt):
    """Lists in; dict of the tensors after the call and of the plan."""
    table, lens, shares = [list(r) for r in table], list(lens), list(shares)
    before, was = [list(r) for r in table], list(lens)
    B, width = len(lens), len(table[0])
    named, asked, taken = set(), 0, 0
    got, sp, dp, ct = [], [], [], []
    for i, (s, t) in enumerate(zip(src, dst)):
        n = -1
        if 0 <= s < B and 0 <= t < B and s != t:
            if was[t] <= 0 and t not in named:
                has = min(max(was[s], 0), width * pt)
                n = has if tokens is None else min(max(tokens[i], 0), has)
            named.add(t)
        part = n > 0 and n % pt != 0
        if part:
            asked += 1
            if asked > count:
                n, part = -1, False
        row = (-1, -1, 0)
        if n >= 0:
            lens[t] = n
            for c in range(n // pt):
                p = before[s][c]
                table[t][c] = p
                if 0 <= p < len(shares):
                    shares[p] += 1
            if part:
                taken += 1
                table[t][n // pt] = free[count - taken]
                row = (before[s][n // pt], free[count - taken], n % pt)
        got.append(n)
        for x, y in zip((sp, dp, ct), row):
            x.append(y)
    return dict(table=table, lens=lens, shares=shares, count=count - taken, granted=got,
                src_pages=sp, dst_pages=dp, copy_tokens=ct)


def release(table, lens, done, free, count, shares, pt):
    lens, free, shares = list(lens), list(free), list(shares)
    entries = []
    for b, f in enumerate(done):
        if f:
            entries += [p for p in table[b][:held(lens[b], pt)] if 0 <= p < len(shares)]
            lens[b] = 0
    last = {p: i for i, p in enumerate(entries)}
    for p in entries:
        shares[p] -= 1
    for i, p in enumerate(entries):
        if last[p] == i and shares[p] < 0:
            shares[p] = 0
            if count < len(free):
                free[count] = p
                count += 1
    return dict(lens=lens, free=free, count=count, shares=shares)


def compact(table, lens, free, count, shares, pt):
    P = len(free)
    spare = set(free[:count])
    U = P - len(spare)
    movers = [p for p in range(U, P) if p not in spare]
    to = dict(zip(movers, [p for p in range(U) if p in spare]))
    table, shares, free = [list(r) for r in table], list(shares), list(free)
    for b, n in enumerate(lens):
        for c in range(min(held(n, pt), len(table[b]))):
            table[b][c] = to.get(table[b][c], table[b][c])
    for s, t in to.items():
        shares[t], shares[s] = shares[s], 0
    free[:P - U] = [P - 1 - i for i in range(P - U)]
    pad = [-1] * (P // 2 - len(movers))
    return dict(table=table, free=free, count=P - U, shares=shares, moves=len(movers),
                src_pages=movers + pad, dst_pages=list(to.values()) + pad,
                remap=[to.get(p, p) for p in range(P)])


def turned(x, positions, turns, factor, interleaved, inverse=False):
    """x (rows, H, d) turned, in 64 bits, and what a kernel may be off before the result's
    rounding.

    The remainder of position * turn is a whole number of 2^-64 turns, whose nearest fp32 in
    half turns is off by half a step of [1/2, 1), 2^-25: pi 2^-25 radians.  Sine and cosine are
    fp32's, off by at most 4 steps, 2^-22; the factor's product, the two products and their
    sum round once each, 2^-24 of at most |x1| + |x2|.  Together (1.6 + 4 + 4) 2^-24, taken as
    10, of factor (|x1| + |x2|)."""
    n = len(turns)
    rest = [[(int(p) * int(t)) % 2 ** 64 / 2 ** 64 for t in turns] for p in positions]
    a = torch.tensor(rest, dtype=torch.float64) * (2 * math.pi) * (-1 if inverse else 1)
    a = a.view(len(positions), 1, n)
    x = x.double()
    y = x.clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else \
        (slice(0, n), slice(n, 2 * n))
    u, v = x[..., first], x[..., second]
    y[..., first] = factor * (u * torch.cos(a) - v * torch.sin(a))
    y[..., second] = factor * (v * torch.cos(a) + u * torch.sin(a))
    tol = torch.zeros_like(y)
    tol[..., first] = tol[..., second] = 10 * 2.0 ** -24 * abs(factor) * (u.abs() + v.abs())
    return y, tol
