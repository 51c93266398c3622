"""Plain 64-bit forms of the per-request operators, on CPU tensors, and the bounds of their
rounding that the tests allow."""
import math

import torch


def adapter(x, W, A, B, scale, offsets, ids, ranks=None, bias=None, substitute=False, out=None):
    """(y, allowance): the product in float64 and, per element, a bound of the rounding errors
    of float32 accumulation in any order with the operands' own dtype (before the result is
    rounded to it); rows of no request are out's, with allowance 0."""
    T, N = x.shape[0], W.shape[1] if substitute else W.shape[0]
    K, R = x.shape[1], A.shape[1]
    y = torch.zeros(T, N, dtype=torch.float64) if out is None else out.double().clone()
    tol = torch.zeros(T, N, dtype=torch.float64)
    xd, Wd = x.double(), W.double() if substitute else W.double().t()
    for q in range(len(ids)):
        a, b = int(offsets[q]), int(offsets[q + 1])
        a, b = max(0, min(a, T)), max(0, min(b, T))
        if b <= a:
            continue
        v = xd[a:b] @ Wd
        s = xd[a:b].abs() @ Wd.abs()
        low = torch.zeros_like(s)
        if bias is not None and not substitute:
            v = v + bias.double()
            s = s + bias.double().abs()
        e = int(ids[q])
        if 0 <= e < A.shape[0]:
            r = R if ranks is None else max(0, min(R, int(ranks[e])))
            P, Q = (B[e, :, :r].double(), A[e, :r].double()) if substitute else \
                (A[e, :r].double().t(), B[e, :, :r].double().t())
            sc = float(scale[e])
            v = v + sc * ((xd[a:b] @ P) @ Q)
            low = abs(sc) * ((xd[a:b].abs() @ P.abs()) @ Q.abs())
        y[a:b] = v
        # Each product and each addition of a chain of n terms rounds (or truncates) by at most
        # 2^-23 of a partial sum, which is at most the sum of magnitudes: (n + 8) 2^-23 s for
        # the shared part (n = K), the same twice over for the chained low-rank part (K, then R).
        # float32 as 3xTF32: hi + lo keeps 2^-22 of an operand and lo * lo, at most 2^-22 of the
        # product, is left out: 2^-20 s in all, for two chained products 2^-19.
        # The low-rank intermediate is held as two bfloat16 (float16) numbers: 2^-16 of it.
        tol[a:b] = (K + 8) * 2.0**-23 * s + (K + R + 16) * 2.0**-23 * low
        if x.dtype == torch.float32:
            tol[a:b] += 2.0**-20 * s + 2.0**-19 * low
        else:
            tol[a:b] += 2.0**-16 * low
    return y, tol


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, want, tol, what=""):
    """got (a tensor of its dtype) is want (float64) within tol and one rounding to the dtype."""
    g = got.double().cpu()
    h = half_step(got.dtype)
    tiny = torch.finfo(got.dtype).tiny
    lim = tol + h * (want.abs() + tol) + tiny * h
    bad = ~((g - want).abs() <= lim) & ~(g == want)
    bad &= ~(g.isnan() & want.isnan())
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, the worst by "
                           f"{float(((g - want).abs() / lim)[bad].max()):.3g} allowances at "
                           f"{bad.nonzero()[0].tolist()}: {g[bad][0]} for {want[bad][0]}")


def rules(x, n, tokens=None, token_offsets=None, prompt_len=None, repetition=None, frequency=None, presence=None,
          bias_ids=None, bias_values=None, bias_offsets=None, allowed=None, allowed_row=None, dtype=torch.float64):
    """The rules on x [rows, n], answer by answer as they are defined, in `dtype`."""
    out = x.to(dtype).clone()
    rows = x.shape[0]
    for r in range(rows):
        count, seen = {}, set()
        if tokens is not None:
            a, b = (max(0, min(len(tokens), int(token_offsets[r + i]))) for i in (0, 1))
            given = 0 if prompt_len is None else max(0, int(prompt_len[r]))
            for i in range(a, max(a, b)):
                j = int(tokens[i])
                if 0 <= j < n:
                    seen.add(j)
                    if i - a >= given:
                        count[j] = count.get(j, 0) + 1
        bias = {}
        if bias_ids is not None:
            a, b = (max(0, min(len(bias_ids), int(bias_offsets[r + i]))) for i in (0, 1))
            for i in range(a, max(a, b)):
                j = int(bias_ids[i])
                if 0 <= j < n:
                    bias[j] = bias_values[i].to(dtype)
        one = torch.ones((), dtype=dtype)
        rep = one if repetition is None else repetition[r].to(dtype)
        freq = one * 0 if frequency is None else frequency[r].to(dtype)
        pres = one * 0 if presence is None else presence[r].to(dtype)
        for j in seen:
            v = out[r, j]
            v = v / rep if v > 0 else v * rep
            if count.get(j):
                v = v - freq * count[j]
                v = v - pres
            out[r, j] = v
        for j, bv in bias.items():
            out[r, j] = out[r, j] + bv
        if allowed is not None:
            m = r if allowed_row is None else int(allowed_row[r])
            if 0 <= m < allowed.shape[0]:
                w = (allowed[m].long() & 0xFFFFFFFF)
                j = torch.arange(n)
                free = ((w[j // 32] >> (j % 32)) & 1).bool()
                out[r][~free] = -math.inf
    return out


def margin(l, u, labels, n, dtype=torch.float32, **kw):
    """(margin, rival) in `dtype` from the definition."""
    lo, hi = rules(l, n, dtype=dtype, **kw), rules(u, n, dtype=dtype, **kw)
    lo[lo.isnan()] = -math.inf
    free = rules(torch.zeros_like(u), n, allowed=kw.get("allowed"), allowed_row=kw.get("allowed_row")) == 0
    m, rival = [], []
    for r in range(l.shape[0]):
        j = int(labels[r])
        mine = lo[r, j] if 0 <= j < n else torch.full((), -math.inf, dtype=dtype)
        h = hi[r].clone()
        h[h.isnan() & free[r]] = math.inf
        h[~free[r]] = -math.inf
        if 0 <= j < n:
            h[j] = -math.inf
        best = h.max()
        d = mine - best
        m.append(torch.full((), -math.inf, dtype=dtype) if d.isnan() else d)
        rival.append(-1 if best == -math.inf else int((h == best).nonzero()[0]))
    return torch.stack(m) if m else torch.zeros(0, dtype=dtype), torch.tensor(rival, dtype=torch.int32)


def pack(free):
    """[m, n] truth values as [m, ceil(n / 32)] int32 words."""
    m, n = free.shape
    words = (n + 31) // 32
    bits = torch.zeros(m, words * 32, dtype=torch.int64)
    bits[:, :n] = free.long()
    w = (bits.view(m, words, 32) << torch.arange(32)).sum(dim=2)
    return torch.where(w >= 2**31, w - 2**32, w).to(torch.int32)
