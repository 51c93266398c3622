"""The operators for many variants of one network in a batch, as cases to be timed and compared.

Every request (a region under certification, a sequence being answered) may carry its own
low-rank adapter beside the shared weights of a layer, and its own rules for the answer: the
tokens it has seen with their penalties, its biases, and the set it may answer from.

  adapter     y = x W^T + b + s_e (x A_e^T) B_e^T      the layer on rows of many requests
  substitute  y = x W + s_e (x B_e) A_e                coefficient rows over the layer's outputs
                                                       taken to its inputs (its input gradient)
  logits      the rules applied to rows of logits
  margin      the rules applied to lower and upper bounds of logits: how far the label's lower
              bound stays above the best upper bound among the other answers, and which that is

With `own` false the cases run in plain torch operations, else through cfgpu.
"""
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SZ = {"f32": 4, "bf16": 2, "f16": 2}


def _ops():
    root = os.path.join(os.getcwd(), "constraintflow-gpu_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from cfgpu import ops
    return ops


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one request answering, one token: the latency of a layer with an adapter
        dict(name="adapter_token", op="adapter", dtype="bf16", rows=1, requests=1, k=4096, n=4096, rank=16,
             adapters=8, even=True, bias=False),
        # sixty-four requests answering together, one token each, an adapter for nearly each
        dict(name="adapter_tokens", op="adapter", dtype="bf16", rows=64, requests=64, k=4096, n=4096, rank=16,
             adapters=48, even=True, bias=False),
        # prompts of ragged lengths through a wide projection
        dict(name="adapter_prompts", op="adapter", dtype="bf16", rows=4001, requests=7, k=4096, n=11008, rank=64,
             adapters=12, even=False, bias=True),
        # odd sizes that no vector load or tile divides, as a certifier's float32 rows have them
        dict(name="adapter_odd", op="adapter", dtype="f32", rows=517, requests=11, k=1021, n=777, rank=6,
             adapters=5, even=False, bias=True),
        # a 784-(200x9)-10 network's first layer under 256 regions of 200 coefficient rows
        dict(name="substitute_regions", op="substitute", dtype="f32", rows=256 * 200, requests=256, k=200, n=784,
             rank=8, adapters=32, even=True, bias=False),
        # the same direction over long sequences: the gradient with respect to the layer's input
        dict(name="substitute_long", op="substitute", dtype="bf16", rows=8192, requests=16, k=4096, n=4096, rank=32,
             adapters=16, even=False, bias=False),
        # one request's logits
        dict(name="logits_token", op="logits", dtype="f32", rows=1, n=131072, history=4096, biases=64),
        # a serving batch
        dict(name="logits_batch", op="logits", dtype="bf16", rows=256, n=131072, history=2048, biases=64),
        # long histories over an odd number of answers
        dict(name="logits_long", op="logits", dtype="f16", rows=33, n=100003, history=32768, biases=300),
        # 256 regions of a ten-class network
        dict(name="margin_classes", op="margin", dtype="f32", rows=256, n=10, history=0, biases=3),
        # bounds of a vocabulary's logits
        dict(name="margin_tokens", op="margin", dtype="f32", rows=128, n=131072, history=1024, biases=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["adapter", "adapter", "substitute", "substitute", "logits", "logits", "margin"])
    if op in ("adapter", "substitute"):
        dtype = rng.choice(["bf16", "bf16", "f32"])
        rows = _log(rng, 1, 8192)
        k, n = _log(rng, 64, 8192), _log(rng, 64, 8192)
        if rng.random() < 0.7:        # most layers are a multiple of 16 wide
            k, n = max(64, k // 16 * 16), max(64, n // 16 * 16)
        limit = 2.0e10 if dtype == "f32" else 1.3e11
        while rows * k * n > limit:
            rows = max(1, rows // 2 - rng.randrange(2))
        style = rng.choice(["tokens", "ragged", "ragged", "even"])
        requests = rows if style == "tokens" and rows <= 256 else max(1, min(rows, _log(rng, 1, 64)))
        even = style != "ragged"
        if even:
            rows = rows // requests * requests
        return dict(op=op, dtype=dtype, rows=rows, requests=requests, k=k, n=n,
                    rank=rng.choice([1, 4, 5, 8, 16, 16, 24, 32, 64, 128]), adapters=_log(rng, 1, 32), even=even,
                    bias=op == "adapter" and rng.random() < 0.5)
    rows = _log(rng, 1, 256)
    n = _log(rng, 10, 262144)
    if op == "margin":
        rows = max(1, min(rows, 128 * 131072 // n))
    rows = max(1, min(rows, 256 * 131072 // n))
    history = rng.choice([0, _log(rng, 1, 64), _log(rng, 64, 32768)])
    history = min(history, max(1, 256 * 2048 // rows))
    return dict(op=op, dtype="f32" if op == "margin" else rng.choice(["f32", "bf16", "f16"]), rows=rows, n=n,
                history=history, biases=rng.choice([0, 3, 64, 300]))


# ------------------------------------------------------------------------------ inputs
def _gen(seed, device="cpu"):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed))
    return g


def _adapter_inputs(case, seed):
    dev = torch.device("cuda")
    gd, gh = _gen(seed, dev), _gen(seed)
    dt = _DT[case["dtype"]]
    T, Q, R, E = case["rows"], case["requests"], case["rank"], case["adapters"]
    sub = case["op"] == "substitute"
    n_out, n_in = (case["k"], case["n"]) if sub else (case["n"], case["k"])

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gd, device=dev) * std).to(dt)

    x = normal(T, case["k"])
    W = normal(n_out, n_in, std=case["k"] ** -0.5)
    A = normal(E, R, n_in, std=(R if sub else n_in) ** -0.5)
    B = normal(E, n_out, R, std=0.3 * (n_out if sub else R) ** -0.5)
    if case["even"]:
        cuts = [T * q // Q for q in range(Q + 1)]
    else:
        share = torch.rand(Q, generator=gh).pow(2) + 0.02
        ends = (share.cumsum(0) / share.sum() * T).round().long().tolist()
        cuts = [0] + ends[:-1] + [T]
    ids = torch.randint(0, E, (Q,), generator=gh)
    if Q > 1:                      # a request without an adapter of its own
        ids[int(torch.randint(0, Q, (1,), generator=gh))] = -1
    ranks = torch.where(torch.rand(E, generator=gh) < 0.25, torch.full((E,), (R + 1) // 2), torch.full((E,), R))
    scale = torch.rand(E, generator=gh) * 1.5 + 0.5
    bias = normal(n_out, std=0.1) if case["bias"] else None
    return dict(x=x, W=W, A=A, B=B, scale=scale.to(dev), ranks=ranks.to(dev, torch.int32),
                offsets=torch.tensor(cuts, dtype=torch.int64, device=dev), ids=ids.to(dev, torch.int32), bias=bias,
                cuts=cuts, ids_host=ids.tolist(), ranks_host=ranks.tolist(), scale_host=scale.tolist())


def _rule_inputs(case, seed):
    dev = torch.device("cuda")
    gh, gd = _gen(seed), _gen(seed, dev)
    rows, n = case["rows"], case["n"]
    H = case["history"]
    s = {}
    if H:
        lens = (torch.rand(rows, generator=gh) * H).long()
        lens[0] = H                                 # the longest one is always there
        prompt = (lens.float() * torch.rand(rows, generator=gh)).int()
        total = int(lens.sum())
        # word frequencies: a few answers come back again and again
        toks = (n * torch.rand(total, generator=gd, device=dev).double().pow(3)).long().clamp_(max=n - 1)
        s["tokens"] = toks.to(torch.int32)
        s["token_offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(dev)
        s["prompt_len"] = prompt.to(dev)
        s["token_total"] = total
        s["repetition"] = (1.0 + 0.5 * torch.rand(rows, generator=gh)).to(dev)
        s["frequency"] = (0.3 * torch.rand(rows, generator=gh)).to(dev)
        s["presence"] = (0.6 * torch.rand(rows, generator=gh)).to(dev)
    if case["biases"]:
        lens = (torch.rand(rows, generator=gh) * (case["biases"] + 1)).long()
        total = int(lens.sum())
        s["bias_ids"] = torch.randint(0, n, (total,), generator=gh).to(dev, torch.int32)
        s["bias_values"] = (torch.randn(total, generator=gh) * 2).to(dev)
        s["bias_offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(dev)
        s["bias_total"] = total
    masks = max(1, rows // 4)
    s["free"] = torch.rand(masks, (n + 31) // 32 * 32, generator=gd, device=dev) < 0.5
    row = torch.randint(0, masks, (rows,), generator=gh)
    row[torch.rand(rows, generator=gh) < 0.5] = -1      # half of the requests have no grammar
    s["allowed_row"] = row.to(dev, torch.int32)
    return s


def _pack(free):
    """[m, 32 w] truth values as [m, w] words, the first in the lowest bit."""
    bits = free.view(free.shape[0], -1, 32).long() << torch.arange(32, device=free.device)
    words = bits.sum(dim=2)
    return torch.where(words >= 2**31, words - 2**32, words).to(torch.int32)


_RULES = ("tokens", "token_offsets", "prompt_len", "repetition", "frequency", "presence", "bias_ids", "bias_values",
          "bias_offsets", "allowed", "allowed_row")


def prepare(case, seed):
    dev = torch.device("cuda")
    if case["op"] in ("adapter", "substitute"):
        s = _adapter_inputs(case, seed)
        s["sub"] = case["op"] == "substitute"
        if own:
            ops = _ops()
            s["layer"] = ops.AdapterLayer(s["W"], s["A"], s["B"], s["scale"], ranks=s["ranks"], bias=s["bias"])
            s["out"] = torch.empty(case["rows"], case["n"], dtype=_DT[case["dtype"]], device=dev)
    else:
        s = _rule_inputs(case, seed)
        g = _gen(seed + 1, dev)
        rows, n = case["rows"], case["n"]
        x = torch.randn(rows, n, generator=g, device=dev) * 3.0
        if case["op"] == "logits":
            s["x"] = x.to(_DT[case["dtype"]])
        else:
            r = torch.rand(rows, n, generator=g, device=dev) * 0.2
            labels = x.argmax(dim=1)
            s["l"], s["u"], s["labels"] = x - r, x + r, labels
            # the certified answer is one that the rules allow
            s["free"][s["allowed_row"].long().clamp(min=0), labels] = True
        s["allowed"] = _pack(s.pop("free"))
        if own:
            s["rules"] = _ops().AnswerRules(rows, n, **{k: s.get(k) for k in _RULES})
            if case["op"] == "logits":
                s["out"] = torch.empty_like(s["x"])
    s["op"], s["rows"], s["n"] = case["op"], case["rows"], case["n"]
    return s


# -------------------------------------------------------------------------- plain forms
def _plain_adapter(s):
    x, W = s["x"].float(), s["W"].float()
    y = x @ W if s["sub"] else x @ W.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    for q, e in enumerate(s["ids_host"]):
        a, b = s["cuts"][q], s["cuts"][q + 1]
        if e < 0 or a == b:
            continue
        r = s["ranks_host"][e]
        A, B = s["A"][e, :r].float(), s["B"][e, :, :r].float()
        if s["sub"]:
            y[a:b] += s["scale_host"][e] * ((x[a:b] @ B) @ A)
        else:
            y[a:b] += s["scale_host"][e] * ((x[a:b] @ A.t()) @ B.t())
    return y.to(s["x"].dtype)


def _row_ids(offsets, total):
    lens = offsets[1:] - offsets[:-1]
    return torch.repeat_interleave(torch.arange(lens.numel(), device=offsets.device), lens, output_size=total)


def _plain_rules(s, x):
    """The rules on x [rows, n] float32."""
    rows, n = s["rows"], s["n"]
    dev = x.device
    if s.get("tokens") is not None:
        row = _row_ids(s["token_offsets"], s["token_total"])
        at = torch.arange(s["token_total"], device=dev) - s["token_offsets"][row]
        answered = (at >= s["prompt_len"][row]).int()
        flat = row * n + s["tokens"].long()
        count = torch.zeros(rows * n, dtype=torch.int32, device=dev).index_add_(0, flat, answered).view(rows, n)
        seen = torch.zeros(rows * n, dtype=torch.int32, device=dev)
        seen = seen.index_add_(0, flat, torch.ones_like(answered)).view(rows, n) > 0
        rep = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = x - s["frequency"][:, None] * count
        x = x - s["presence"][:, None] * (count > 0)
    if s.get("bias_ids") is not None:
        row = _row_ids(s["bias_offsets"], s["bias_total"])
        flat = row * n + s["bias_ids"].long()
        last = torch.zeros(rows * n, dtype=torch.int64, device=dev)
        last = last.scatter_reduce_(0, flat, torch.arange(1, s["bias_total"] + 1, device=dev), "amax")
        values = torch.cat([torch.zeros(1, device=dev), s["bias_values"]])
        x = x + values[last].view(rows, n)
    col = torch.arange(n, device=dev)
    word = s["allowed"][:, col // 32]
    free = ((word >> (col % 32)) & 1) != 0
    free = torch.cat([free, torch.ones(1, n, dtype=torch.bool, device=dev)])
    return torch.where(free[s["allowed_row"].long()], x, torch.full((), -math.inf, device=dev))


def _plain_margin(s):
    lo, hi = _plain_rules(s, s["l"]), _plain_rules(s, s["u"])
    mine = lo.gather(1, s["labels"][:, None])[:, 0]
    hi = hi.scatter(1, s["labels"][:, None], -math.inf)
    best = hi.max(dim=1).values
    col = torch.arange(s["n"], device=hi.device)
    rival = torch.where(hi == best[:, None], col, s["n"]).min(dim=1).values
    rival = torch.where(best == -math.inf, -1, rival)
    margin = mine - best
    # an infinite bound less itself says nothing
    return torch.where(margin.isnan(), -math.inf, margin), rival.to(torch.int32)


def run(state):
    s = state
    if not own:
        if s["op"] == "logits":
            return _plain_rules(s, s["x"].float()).to(s["x"].dtype)
        return _plain_margin(s) if s["op"] == "margin" else _plain_adapter(s)
    ops = _ops()
    if s["op"] == "logits":
        return ops.edit_logits(s["x"], s["rules"], out=s["out"])
    if s["op"] == "margin":
        return ops.answer_margin(s["l"], s["u"], s["labels"], s["rules"])
    return ops.adapter_matmul(s["x"], s["layer"], s["offsets"], s["ids"], substitute=s["sub"], out=s["out"])


# -------------------------------------------------------------------------- what it takes
def work(case):
    if case["op"] in ("adapter", "substitute"):
        T, Q, K, N, R = (case[k] for k in ("rows", "requests", "k", "n", "rank"))
        used = min(Q, case["adapters"])
        size = _SZ[case["dtype"]]
        return {"bytes": size * (T * K + K * N + T * N + used * R * (K + N)) + 16 * Q,
                "flops": 2.0 * T * (K * N + R * (K + N))}
    rows, n = case["rows"], case["n"]
    extra = rows * (case["history"] // 2 * 4 + case["biases"] // 2 * 8) + rows // 2 * n // 8
    if case["op"] == "logits":
        return {"bytes": 2 * _SZ[case["dtype"]] * rows * n + extra, "flops": 4.0 * rows * n}
    return {"bytes": 4 * rows * n + 16 * rows + extra, "flops": 5.0 * rows * n}


# ------------------------------------------------------------------------- in 64 bits
def _exact_adapter(s):
    out = []
    W, x = s["W"].double(), s["x"].double()
    merged = {}
    for q, e in enumerate(s["ids_host"]):
        if e not in merged:
            M = W
            if e >= 0:
                r = s["ranks_host"][e]
                M = W + float(s["scale"][e]) * (s["B"][e].double()[:, :r] @ s["A"][e].double()[:r])
            merged = {e: M}             # one merged weight at a time
        M = merged[e]
        rows = x[s["cuts"][q]:s["cuts"][q + 1]]
        out.append(rows.matmul(M if s["sub"] else M.t()))
    y = torch.cat(out)
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_rules(s, x):
    """Row by row from the definition, x [rows, n] float64."""
    out = x.clone()
    n = s["n"]
    col = torch.arange(n, device=x.device)
    toff = s["token_offsets"].tolist() if s.get("tokens") is not None else None
    boff = s["bias_offsets"].tolist() if s.get("bias_ids") is not None else None
    plen = s["prompt_len"].tolist() if toff else None
    for r in range(s["rows"]):
        v = out[r]
        if toff:
            hist = s["tokens"][toff[r]:toff[r + 1]].long()
            count = torch.bincount(hist[plen[r]:], minlength=n).double()
            seen = torch.bincount(hist, minlength=n) != 0
            rep = s["repetition"][r].double()
            v = torch.where(seen & (v > 0), v / rep, torch.where(seen, v * rep, v))
            v = v - s["frequency"][r].double() * count - s["presence"][r].double() * (count != 0).double()
        if boff:
            ids = s["bias_ids"][boff[r]:boff[r + 1]].tolist()
            vals = s["bias_values"][boff[r]:boff[r + 1]].tolist()
            given = dict(zip(ids, vals))         # the last entry of an id counts
            if given:
                at = torch.tensor(list(given), device=x.device)
                v = v.index_add(0, at, torch.tensor(list(given.values()), dtype=torch.float64, device=x.device))
        m = int(s["allowed_row"][r])
        if m >= 0:
            bits = s["allowed"][m].long() & 0xFFFFFFFF
            v = v.masked_fill(torch.div(bits[col >> 5], 2 ** (col & 31), rounding_mode="floor") % 2 == 0, -math.inf)
        out[r] = v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("adapter", "substitute"):
        return _exact_adapter(s)
    if s["op"] == "logits":
        return _exact_rules(s, s["x"].double())
    lo, hi = _exact_rules(s, s["l"].double()), _exact_rules(s, s["u"].double())
    at = torch.arange(s["rows"], device=lo.device)
    mine = lo[at, s["labels"]]
    hi[at, s["labels"]] = -math.inf
    margin = mine - hi.amax(dim=1)
    return margin.masked_fill(margin.isnan(), -math.inf), None
