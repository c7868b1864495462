"""The 8-bit paged cache's operators from their definitions: plans by a loop
over the requests, codes and attention in 64 bits on the CPU."""

import math

import torch

TOP = {"int8": 127.0, "fp8": 448.0}
CODE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


def plan(table, lens, new, free, count, rows, pt):
    """Lists in; (q_start, q_lens, kv_lens, slots, positions, free count, table)."""
    table = [list(r) for r in table]
    width, top, asked = len(table[0]), count, 0
    start, got, kv = [0], [], []
    slots, pos = [-1] * rows, [0] * rows
    for b, (t0, n) in enumerate(zip(lens, new)):
        n, r0 = max(n, 0), start[-1]
        start.append(r0 + n)
        held, want = -(-t0 // pt), -(-(t0 + n) // pt)
        ok = r0 + n <= rows and want <= width
        if ok:
            asked += want - held
            ok = want == held or asked <= count
        for i in range(n if ok else 0):
            t = t0 + i
            if t % pt == 0:
                top -= 1
                table[b][t // pt] = free[top]
            slots[r0 + i], pos[r0 + i] = table[b][t // pt] * pt + t % pt, t
        got.append(n if ok else 0)
        kv.append(t0 + got[-1])
    return start, got, kv, slots, pos, top, table


def scale_of(a, code):
    """fp32 scales of blocks whose largest value is a (fp32)."""
    s = (a * torch.tensor(1.0 / TOP[code])).clamp(min=2.0 ** -100)
    return torch.where(a > 0, s, torch.zeros_like(s))


def e4m3_grid():
    """The 127 finite e4m3 magnitudes, ascending (from the format: 4 exponent bits, bias 7)."""
    return torch.tensor([(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** (max(e, 1) - 7)
                         for e in range(16) for m in range(8)][:127], dtype=torch.float64)


def nearest(y, code):
    """The values that codes stand for, nearest to y (float64), ties to the even code."""
    if code == "int8":
        return y.round().clamp(-127, 127)
    g = e4m3_grid()
    a = y.abs().clamp(max=448)
    hi = torch.searchsorted(g, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up = (g[hi] - a) < (a - g[lo])
    tie = (g[hi] - a) == (a - g[lo])
    i = torch.where(up | (tie & (hi % 2 == 0)), hi, lo)
    i = torch.where(g[hi] == a, hi, i)
    return torch.where(y < 0, -g[i], g[i])


def quantise(x, s, code):
    """x fp32 -> nearest code's value (float64, without the scale); s fp32 broadcasts."""
    inv = torch.where(s > 0, (1.0 / s.double()).float().double(), torch.zeros_like(s).double())
    y = torch.where(torch.isnan(x), torch.zeros_like(x), x.clamp(-3e38, 3e38)).double() * inv
    y = torch.where(torch.isinf(x), torch.sign(x).double() * TOP[code] * (s > 0), y)
    return nearest(y, code)


class Cache:
    """Tokens of each request as (codes' values, block scales), appended in runs."""

    def __init__(self, B, H, d, code):
        self.code, self.H, self.d = code, H, d
        self.val = [[torch.zeros(0, H, d, dtype=torch.float64) for _ in range(2)] for _ in range(B)]
        self.scale = [[torch.zeros(0, H) for _ in range(2)] for _ in range(B)]

    def append(self, b, k, v):
        """k, v (S, H, d) of any float type."""
        for half, x in enumerate((k, v)):
            x, val, sc = x.float().cpu(), self.val[b][half], self.scale[b][half]
            while x.shape[0]:
                j = val.shape[0] % 16
                part, x = x[:16 - j], x[16 - j:]
                fin = torch.where(torch.isfinite(part), part.abs(), torch.zeros(()))
                s = scale_of(fin.amax((0, 2)), self.code)                     # (H,)
                if j:
                    old = sc[-1]
                    grew = s > old
                    s = torch.where(grew, s, old)
                    was = val[-j:]
                    again = quantise((was * old.double()[None, :, None]).float(),
                                     s[None, :, None], self.code)
                    val = torch.cat([val[:-j], torch.where(grew[None, :, None], again, was)])
                    sc = sc[:-1]
                val = torch.cat([val, quantise(part, s[None, :, None], self.code)])
                sc = torch.cat([sc, s[None]])
            self.val[b][half], self.scale[b][half] = val, sc

    def values(self, b, half):
        """(T, H, d) float64."""
        T = self.val[b][half].shape[0]
        s = self.scale[b][half].double().repeat_interleave(16, 0)[:T]
        return self.val[b][half] * s[..., None]


def attend(q, k, v, scale, first, q_half_step, weight_half_step, out_half_step):
    """One request: q (Q, Hq, d), k / v (T, H, d) float64; query i sees tokens
    [0, first + i] (causal) or, with first None, all.  Returns the result (Q, Hq, d)
    in 64 bits and what a kernel may be off:

    * a score s = scale sum q k carries d fp32 roundings of partial sums of at most
      A = scale sum |q k| (taken as 4 sqrt(d) of them in one direction), the rounding of
      q to the product's type, and those of its scaling and of the exponent's argument:
        ds = A (4 sqrt(d) + 4) 2^-24 + A q_half_step + (|s| + 16) 2^-22;
    * a weight p carries ds and its own rounding; the sums over T tokens 4 sqrt(T) + 8
      fp32 roundings; numerator and denominator each, so twice:
        |d out| <= 2 sum p |v| (ds + weight_half_step + (4 sqrt(T) + 8) 2^-24);
    * a weight p vs meets an f16 with the largest weight at 2^7 or more: below 2^-14 the
      steps of an f16 do not shrink, and half a step, 2^-25, is 2^-32 of the largest
      weight.  Times a code it is at most 2^-32 p_max max |v|, for each of T tokens:
        |d out| <= T 2^-32 max |v|;
    * the result is rounded once to its type: out_half_step |out|."""
    Q, Hq, d = q.shape
    T, H, _ = k.shape
    out = torch.zeros(Q, Hq, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i in range(Q):
        n = T if first is None else min(T, first + i + 1)
        if n <= 0:
            continue
        for h in range(H):
            qs = q[i, h * (Hq // H):(h + 1) * (Hq // H)].double()                # (G, d)
            s = qs @ k[:n, h].T * scale
            A = float((qs.abs() @ k[:n, h].abs().T * abs(scale)).max())
            p = torch.softmax(s, -1)
            o, e = p @ v[:n, h], p @ v[:n, h].abs()
            ds = (A * (4 * math.sqrt(d) + 4) * 2.0 ** -24 + A * q_half_step
                  + (float(s.abs().max()) + 16) * 2.0 ** -22)
            out[i, h * (Hq // H):(h + 1) * (Hq // H)] = o
            tol[i, h * (Hq // H):(h + 1) * (Hq // H)] = (
                2 * e * (ds + weight_half_step + (4 * math.sqrt(n) + 8) * 2.0 ** -24)
                + n * 2.0 ** -32 * v[:n, h].abs().max() + out_half_step * o.abs())
    return out, tol
