"""Per-request adapters and answer rules on the GPU against plain 64-bit forms."""
import math

import pytest
import torch

import variants_oracle as V

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ops():
    from cfgpu import ops as o
    return o


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def make(T, K, N, R, E, Q, dtype, sub, seed=0, style="ragged", ranks=False, bias=False):
    g = gen(seed)
    n_out, n_in = (K, N) if sub else (N, K)
    t = dict(x=torch.randn(T, K, generator=g).to(dtype),
             W=(torch.randn(n_out, n_in, generator=g) * K**-0.5).to(dtype),
             A=(torch.randn(E, R, n_in, generator=g) * (R if sub else K)**-0.5).to(dtype),
             B=(torch.randn(E, n_out, R, generator=g) * (K if sub else max(R, 1))**-0.5).to(dtype),
             scale=torch.rand(E, generator=g) + 0.5)
    if style == "tokens":
        cuts = [T * q // max(Q, 1) for q in range(Q + 1)]
    else:
        cuts = [0] + sorted(torch.randint(0, T + 1, (max(Q - 1, 0),), generator=g).tolist()) + [T] * min(Q, 1)
    t["offsets"] = torch.tensor(cuts, dtype=torch.int64)
    t["ids"] = torch.randint(-1, max(E, 1), (Q,), generator=g).to(torch.int32)
    t["ranks"] = torch.randint(0, R + 1, (E,), generator=g).to(torch.int32) if ranks else None
    t["bias"] = torch.randn(n_out, generator=g).to(dtype) if bias else None
    return t


def layer(t, dev="cuda"):
    d = {k: None if t[k] is None else t[k].to(dev) for k in ("W", "A", "B", "scale", "ranks", "bias")}
    return ops().AdapterLayer(d["W"], d["A"], d["B"], d["scale"], ranks=d["ranks"], bias=d["bias"])


def oracle(t, sub, out=None):
    return V.adapter(t["x"], t["W"], t["A"], t["B"], t["scale"], t["offsets"], t["ids"], t["ranks"], t["bias"], sub,
                     out)


def compare(t, sub, what=""):
    y, tol = oracle(t, sub)
    got = ops().adapter_matmul(t["x"].cuda(), layer(t), t["offsets"].cuda(), t["ids"].cuda(), substitute=sub)
    V.check(got, y, tol, what)
    return got


SHAPES = [
    # T, K, N, R, E, Q, style
    (1, 64, 64, 8, 2, 1, "tokens"),
    (1, 1, 1, 1, 1, 1, "tokens"),
    (7, 33, 65, 3, 2, 3, "ragged"),
    (64, 256, 384, 16, 8, 64, "tokens"),
    (129, 128, 257, 16, 4, 5, "ragged"),
    (130, 136, 264, 24, 4, 2, "ragged"),
    (200, 200, 784, 8, 3, 2, "tokens"),
    (300, 192, 512, 64, 4, 3, "ragged"),
    (513, 320, 320, 128, 3, 4, "ragged"),
    (300, 72, 200, 130, 2, 1, "tokens"),
    (640, 64, 128, 16, 6, 40, "ragged"),
    (257, 40, 48, 200, 2, 9, "ragged"),
]


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:6])))
def test_adapter_matmul(shape, dtype, sub):
    T, K, N, R, E, Q, style = shape
    compare(make(T, K, N, R, E, Q, dtype, sub, seed=T + K, style=style, ranks=True, bias=True), sub)
    compare(make(T, K, N, R, E, Q, dtype, sub, seed=T + K + 1, style=style), sub)


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adapter_large(dtype, sub):
    """Several tiles in each direction, requests that span tiles."""
    compare(make(1100, 520, 1096, 32, 5, 6, dtype, sub, seed=5, ranks=True, bias=True), sub)


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_of_no_request_are_left(dtype, sub):
    t = make(150, 96, 144, 16, 3, 4, dtype, sub, seed=2)
    t["offsets"] = torch.tensor([5, 5, 40, 41, 139])
    before = torch.randn(150, 144, generator=gen(9)).to(dtype)
    y, tol = oracle(t, sub, out=before)
    out = before.cuda()
    got = ops().adapter_matmul(t["x"].cuda(), layer(t), t["offsets"].cuda(), t["ids"].cuda(), substitute=sub, out=out)
    assert got is out
    V.check(got, y, tol)
    assert torch.equal(got[:5].cpu(), before[:5]) and torch.equal(got[139:].cpu(), before[139:])
    fresh = ops().adapter_matmul(t["x"].cuda(), layer(t), t["offsets"].cuda(), t["ids"].cuda(), substitute=sub)
    assert (fresh[:5] == 0).all() and (fresh[139:] == 0).all()


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Q", [3, 60])
def test_another_request_cannot_reach_a_row(dtype, sub, Q):
    """An adapter of infinities and NaN, and NaN rows of its request, stay with that request."""
    t = make(180, 128, 192, 16, 4, Q, dtype, sub, seed=11, style="tokens")
    t["ids"] = (torch.arange(Q) % 3).to(torch.int32)
    bad = dict(t)
    bad["A"], bad["B"], bad["x"] = t["A"].clone(), t["B"].clone(), t["x"].clone()
    bad["A"][1], bad["B"][1] = math.inf, math.nan
    for q in range(Q):
        if q % 3 == 1:
            bad["x"][t["offsets"][q]:t["offsets"][q + 1]] = math.nan
    good = compare(t, sub)
    got = ops().adapter_matmul(bad["x"].cuda(), layer(bad), t["offsets"].cuda(), t["ids"].cuda(), substitute=sub)
    for q in range(Q):
        a, b = int(t["offsets"][q]), int(t["offsets"][q + 1])
        if q % 3 == 1:
            assert got[a:b].isnan().all()
        else:
            assert torch.equal(got[a:b], good[a:b])


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_unused_ranks_and_foreign_ids(dtype, sub):
    t = make(100, 64, 80, 16, 4, 5, dtype, sub, seed=3)
    t["ranks"] = torch.tensor([16, 5, 0, 99], dtype=torch.int32)
    t["ids"] = torch.tensor([1, 2, 4, -7, 3], dtype=torch.int32)
    t["A"][1, 5:], t["B"][1, :, 5:] = math.nan, math.inf
    t["A"][2], t["B"][2] = math.nan, math.nan
    compare(t, sub)


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_float16_range_of_the_intermediate(dtype, sub):
    """x A^T far above float16's largest value, the result well within it."""
    t = make(160, 128, 160, 8, 2, 2, dtype, sub, seed=4)
    a, b = ("B", "A") if sub else ("A", "B")
    t[a] = t[a] * 200
    t[b] = t[b] * 2.0**-12
    t["x"] = t["x"] * 100
    t["W"] = t["W"] * 0.1
    compare(t, sub)


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (0, 1), (5, 3)])
def test_strides_and_alignment(dtype, sub, pad, shift):
    t = make(140, 128, 144, 16, 3, 4, dtype, sub, seed=6, ranks=True)
    y, tol = oracle(t, sub)

    def strided(a):
        flat = torch.full((a[..., 0].numel() * (a.shape[-1] + pad) + shift,), math.nan, dtype=a.dtype, device="cuda")
        v = flat[shift:].view(*a.shape[:-1], a.shape[-1] + pad)[..., :a.shape[-1]]
        v.copy_(a)
        return v
    L = ops().AdapterLayer(strided(t["W"]), strided(t["A"]), strided(t["B"]), t["scale"].cuda(), t["ranks"].cuda())
    out = strided(torch.zeros(140, 144, dtype=dtype))
    ops().adapter_matmul(strided(t["x"]), L, t["offsets"].cuda(), t["ids"].cuda(), substitute=sub, out=out)
    V.check(out, y, tol)
    # a transposed x is laid out first
    got = ops().adapter_matmul(t["x"].t().contiguous().cuda().t(), L, t["offsets"].cuda(), t["ids"].cuda(),
                               substitute=sub)
    V.check(got, y, tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_adapters_no_rank_no_rows(dtype):
    o = ops()
    t = make(50, 64, 72, 0, 3, 2, dtype, False, bias=True)
    compare(t, False)
    t = make(50, 64, 72, 4, 0, 2, dtype, False)
    compare(t, False)
    t = make(50, 64, 72, 4, 2, 2, dtype, False)
    L = layer(t)
    empty = o.adapter_matmul(torch.zeros(0, 64, dtype=dtype).cuda(), L, torch.zeros(3, dtype=torch.int64).cuda(),
                             t["ids"].cuda())
    assert tuple(empty.shape) == (0, 72)
    none = o.adapter_matmul(t["x"].cuda(), L, torch.zeros(1, dtype=torch.int64).cuda(), t["ids"][:0].cuda())
    assert (none == 0).all()


def test_same_call_same_bits():
    t = make(300, 512, 256, 16, 4, 7, BF16, False)
    L, x, off, ids = layer(t), t["x"].cuda(), t["offsets"].cuda(), t["ids"].cuda()
    first = ops().adapter_matmul(x, L, off, ids)
    for _ in range(5):
        assert torch.equal(ops().adapter_matmul(x, L, off, ids), first)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,Q", [(8, 8), (400, 3)])
def test_adapter_streams_and_graphs(dtype, T, Q):
    """Two captured graphs and an eager call on another stream, inputs exchanged in place."""
    o = ops()
    t = make(T, 256, 320, 16, 4, Q, dtype, False, seed=1, style="tokens")
    u = make(T, 256, 320, 16, 4, Q, dtype, False, seed=2, style="tokens")
    L, M = layer(t), layer(u)
    off = t["offsets"].cuda()
    xs, ids = [t["x"].cuda(), u["x"].cuda()], [t["ids"].cuda(), u["ids"].cuda()]
    want = [oracle(t, False), oracle(u, False)]
    o.adapter_matmul(xs[0], L, off, ids[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i, lay in enumerate((L, M)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(o.adapter_matmul(xs[i], lay, off, ids[i]))
        graphs.append(g)
    side = torch.cuda.Stream()
    for rep in range(3):
        with torch.cuda.stream(side):
            eager = o.adapter_matmul(xs[0], L, off, ids[0])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            V.check(outs[i], *want[i])
        V.check(eager, *want[0])
    # other adapters and rows in the same buffers
    ids[0].copy_(u["ids"])
    t["ids"] = u["ids"]
    t["x"] = u["x"]
    xs[0].copy_(u["x"])
    graphs[0].replay()
    torch.cuda.synchronize()
    V.check(outs[0], *oracle(t, False))


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_adapter_few_rows_many_columns(dtype, sub):
    """Less than a tile of rows through enough columns for the wide tiles, aligned and not."""
    compare(make(40, 72, 20008, 16, 3, 4, dtype, sub, seed=41, ranks=True), sub)
    compare(make(5, 72, 17001, 5, 3, 2, dtype, sub, seed=42, ranks=True), sub)


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17])
def test_adapter_few_rows(dtype, sub, T):
    """A few rows of a layer wide enough that its contraction is shared, aligned and not."""
    for K, N, R, Q in ((2048, 264, 16, T), (1027, 131, 5, 2), (72, 1000, 8, 1)):
        t = make(T, K, N, R, 3, Q, dtype, sub, seed=T + K, style="tokens", ranks=True, bias=True)
        compare(t, sub)
        t["offsets"] = torch.clamp(t["offsets"] - 1, min=0)      # the last row is no request's
        before = torch.randn(T, N, generator=gen(T)).to(dtype)
        y, tol = oracle(t, sub, out=before)
        got = ops().adapter_matmul(t["x"].cuda(), layer(t), t["offsets"].cuda(), t["ids"].cuda(), substitute=sub,
                                   out=before.cuda())
        V.check(got, y, tol)


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_a_contraction_over_nothing(dtype, sub):
    o = ops()
    n_out, n_in = (0, 24) if sub else (24, 0)
    z = lambda *s: torch.zeros(*s, dtype=dtype, device="cuda")
    bias = None if sub else torch.randn(24, generator=gen(0)).to(dtype).cuda()
    L = o.AdapterLayer(z(n_out, n_in), z(2, 4, n_in), z(2, n_out, 4), torch.ones(2, device="cuda"), bias=bias)
    got = o.adapter_matmul(z(33, 0), L, torch.tensor([0, 20, 33]).cuda(), torch.tensor([0, 1]).int().cuda(),
                           substitute=sub)
    assert torch.equal(got, z(33, 24) if sub else bias.expand(33, 24))


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("K,N,R", [(65, 130, 7), (200, 131, 16), (67, 264, 16), (129, 136, 24)])
@pytest.mark.parametrize("T,Q", [(3, 3), (40, 40), (300, 4), (2500, 30)])
def test_adapter_unaligned_sizes(dtype, sub, K, N, R, T, Q):
    compare(make(T, K, N, R, 4, Q, dtype, sub, seed=T + K, style="tokens" if Q == T else "ragged", ranks=True,
                 bias=True), sub)


# ------------------------------------------------------------------------ answer rules
def make_rules(rows, n, seed=0, hist=20, biases=5, masks=2, penalties=True, prompt=True):
    g = gen(seed)
    kw = {}
    if hist is not None:
        lens = torch.randint(0, hist + 1, (rows,), generator=g)
        total = int(lens.sum())
        # ids off both ends of the answers as well
        kw["tokens"] = torch.randint(-2, n + 2, (total,), generator=g).to(torch.int32)
        kw["token_offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
        if prompt:
            kw["prompt_len"] = torch.randint(-1, hist + 2, (rows,), generator=g).to(torch.int32)
        if penalties:
            kw["repetition"] = torch.rand(rows, generator=g) + 0.6
            kw["frequency"] = torch.rand(rows, generator=g)
            kw["presence"] = torch.rand(rows, generator=g) - 0.3
    if biases is not None:
        lens = torch.randint(0, biases + 1, (rows,), generator=g)
        total = int(lens.sum())
        kw["bias_ids"] = torch.randint(-1, n + 1, (total,), generator=g).to(torch.int32)
        kw["bias_values"] = torch.randn(total, generator=g)
        kw["bias_offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    if masks:
        kw["allowed"] = V.pack(torch.rand(masks, n, generator=g) < 0.6)
        kw["allowed_row"] = torch.randint(-1, masks + 1, (rows,), generator=g).to(torch.int32)
    return kw


def on_gpu(kw):
    return {k: v.cuda() for k, v in kw.items()}


def same(got, want):
    """Equal values, NaN in the same places."""
    g, w = got.cpu(), want
    assert torch.equal(g.isnan(), w.isnan())
    assert torch.equal(g.nan_to_num(nan=0.0), w.nan_to_num(nan=0.0)), (g - w).abs().max()


RULES = [
    # rows, n, hist, biases, masks
    (1, 1, 3, 1, 1), (3, 10, None, 3, 2), (5, 10, 20, None, None), (4, 33, 8, 40, 2), (2, 1000, 300, 30, 1),
    (7, 2049, 50, 20, 3), (3, 9001, 700, 9, 2), (1, 40000, 2000, 100, 1), (2, 20011, 0, 0, 0), (40, 517, 30, 6, 5),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", RULES, ids=lambda c: "x".join(map(str, c)))
def test_edit_logits(case, dtype):
    """Every step is one float32 operation rounded to nearest, so the float32 form gives the
    same bits; the 64-bit form agrees within the roundings of its (at most five) steps."""
    rows, n, hist, biases, masks = case
    kw = make_rules(rows, n, seed=rows + n, hist=hist, biases=biases, masks=masks)
    x = (torch.randn(rows, n, generator=gen(n)) * 4).to(dtype)
    got = ops().edit_logits(x.cuda(), ops().AnswerRules(rows, n, **on_gpu(kw)))
    assert got.dtype == dtype
    same(got.float(), V.rules(x.float(), n, dtype=F32, **kw).to(dtype).float())
    want = V.rules(x, n, **kw)
    size = x.double().abs() * 2 + 30.0          # |v| after any step: |x| / 0.6 + the penalties and the bias
    fin = want.isfinite()
    lim = 6 * V.half_step(F32) * size + V.half_step(dtype) * want.abs()
    assert ((got.double().cpu() - want).abs()[fin] <= lim[fin]).all()
    # in place
    y = x.cuda()
    assert ops().edit_logits(y, ops().AnswerRules(rows, n, **on_gpu(kw)), out=y) is y
    assert torch.equal(y.nan_to_num(), got.nan_to_num())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_edit_logits_strange_values(dtype):
    """Infinities, NaN and the type's extremes, masked and not; a row whose mask leaves nothing."""
    n = 96
    lo, hi = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.tensor([[-math.inf, math.inf, math.nan, lo, hi, 0.0, -0.0, 1.0] * 12] * 4).to(dtype)
    free = torch.ones(2, n, dtype=torch.bool)
    free[0] = False
    free[1, ::3] = False
    hist = torch.arange(0, n, 2, dtype=torch.int32).repeat(4)
    kw = dict(tokens=hist, token_offsets=torch.arange(5) * 48, repetition=torch.tensor([2.0, 0.5, 1.0, 3.0]),
              frequency=torch.full((4,), 0.25), presence=torch.zeros(4), allowed=V.pack(free),
              allowed_row=torch.tensor([0, 1, -1, 2], dtype=torch.int32))
    got = ops().edit_logits(x.cuda(), ops().AnswerRules(4, n, **on_gpu(kw)))
    assert (got[0] == -math.inf).all()
    same(got.float(), V.rules(x.float(), n, dtype=F32, **kw).to(dtype).float())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("pad,shift,opad,oshift", [(0, 1, 0, 0), (3, 2, 3, 2), (5, 0, 2, 7), (8, 0, 16, 0)])
def test_edit_logits_strides(dtype, pad, shift, opad, oshift):
    rows, n = 6, 3001
    kw = make_rules(rows, n, seed=4, hist=200, biases=30)
    x = torch.randn(rows, n, generator=gen(1)).to(dtype)

    def strided(pad, shift):
        flat = torch.full((rows * (n + pad) + shift + 8,), 7.0, dtype=dtype, device="cuda")
        return flat, flat[shift:shift + rows * (n + pad)].view(rows, n + pad)[:, :n]
    _, xin = strided(pad, shift)
    xin.copy_(x)
    flat, out = strided(opad, oshift)
    ops().edit_logits(xin, ops().AnswerRules(rows, n, **on_gpu(kw)), out=out)
    same(out.float(), V.rules(x.float(), n, dtype=F32, **kw).to(dtype).float())
    keep = torch.ones_like(flat, dtype=torch.bool)
    keep[oshift:oshift + rows * (n + opad)].view(rows, n + opad)[:, :n] = False
    assert (flat[keep] == 7.0).all()          # nothing is written between or behind the rows
    # one row of logits for every row of rules
    got = ops().edit_logits(xin[:1].expand(rows, n), ops().AnswerRules(rows, n, **on_gpu(kw)))
    same(got.float(), V.rules(x[:1].expand(rows, n).float(), n, dtype=F32, **kw).to(dtype).float())


def test_long_history_and_many_rows():
    rows, n = 3, 70000
    kw = make_rules(rows, n, seed=8, hist=40000, biases=3000, masks=2)
    x = torch.randn(rows, n, generator=gen(1))
    got = ops().edit_logits(x.cuda(), ops().AnswerRules(rows, n, **on_gpu(kw)))
    same(got, V.rules(x, n, dtype=F32, **kw))
    rows, n = 3000, 12
    kw = make_rules(rows, n, seed=9, hist=6, biases=2, masks=7)
    x = torch.randn(rows, n, generator=gen(2))
    got = ops().edit_logits(x.cuda(), ops().AnswerRules(rows, n, **on_gpu(kw)))
    same(got, V.rules(x, n, dtype=F32, **kw))


def one_history(n, lens, biases, seed, tops=()):
    """A row for each of `lens` tokens; `tops`: (row, answer, times) answered beyond the random ones."""
    g = gen(seed)
    rows = [torch.randint(0, n, (m,), generator=g) for m in lens]
    for r, j, times in tops:
        rows[r] = torch.cat([rows[r], torch.full((times,), j, dtype=torch.int64)])
    count = torch.tensor([0] + [len(r) for r in rows])
    R = len(rows)
    ids = [torch.randint(0, n, (b,), generator=g) for b in biases]
    return dict(tokens=torch.cat(rows).to(torch.int32), token_offsets=count.cumsum(0),
                repetition=torch.rand(R, generator=g) + 0.6, frequency=torch.rand(R, generator=g) * 0.01,
                presence=torch.rand(R, generator=g), bias_ids=torch.cat(ids).to(torch.int32),
                bias_values=torch.randn(sum(biases), generator=g),
                bias_offsets=torch.tensor([0] + list(biases)).cumsum(0))


HISTORIES = [
    # at the most that a row's own small table holds, and one more; repeated and distinct answers
    (5000, [2800, 2801, 2700, 2700, 0, 0], [0, 0, 100, 101, 2800, 2801], ()),
    (2900, [1536, 1537, 1036, 1036, 1, 0, 0], [0, 0, 500, 501, 1536, 1537, 1], ()),
    # more biases than are compared one by one; one answer more often than 15 bits count
    (9001, [10, 4000, 5000], [1025, 1024, 1500], ()),
    (40000, [100, 5000, 0], [3, 2, 0], ((0, 77, 32767), (1, 39999, 32768), (2, 5, 70000))),
    (70001, [4096, 4097], [0, 9], ((0, 0, 40000), (1, 1, 32769), (1, 70000, 32769))),
]


@pytest.mark.parametrize("case", range(len(HISTORIES)))
def test_histories_at_the_tables_limits(case):
    n, lens, biases, tops = HISTORIES[case]
    rows = len(lens)
    kw = one_history(n, lens, biases, case, tops)
    x = torch.randn(rows, n, generator=gen(case)) * 3
    rules = ops().AnswerRules(rows, n, **on_gpu(kw))
    same(ops().edit_logits(x.cuda(), rules), V.rules(x, n, dtype=F32, **kw))
    labels = kw["tokens"][kw["token_offsets"][:-1].clamp(max=len(kw["tokens"]) - 1)].long()
    m, j = V.margin(x - 0.5, x + 0.5, labels, n, **kw)
    gm, gj = ops().answer_margin((x - 0.5).cuda(), (x + 0.5).cuda(), labels.cuda(), rules)
    same(gm, m)
    assert torch.equal(gj.cpu(), j)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens", [[0] * 64, [3] + [0] * 63, [9000] + [0] * 63], ids=["none", "one", "long"])
def test_the_result_may_be_used_at_once(dtype, lens):
    """Rows without a history end at once; what follows on the stream still finds the whole result,
    and nothing is written after it."""
    n = 100003
    kw = one_history(n, lens, [0] * 64, 3)
    x = torch.randn(64, n, generator=gen(1)).to(dtype)
    want = V.rules(x[:1].float(), n, dtype=F32, tokens=kw["tokens"], token_offsets=kw["token_offsets"][:2],
                   **{k: kw[k][:1] for k in ("repetition", "frequency", "presence")}).to(dtype)
    xd, rules, out = x.cuda(), ops().AnswerRules(64, n, **on_gpu(kw)), torch.empty(64, n, dtype=dtype, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            ops().edit_logits(xd, rules, out=out)
            got = out.clone()
            out.zero_()
            assert torch.equal(got[1:], xd[1:])
            same(got[:1].float(), want.float())
            assert not out.any()


def test_offsets_are_held_within_their_lists():
    n = 50
    kw = dict(tokens=torch.arange(10, dtype=torch.int32), token_offsets=torch.tensor([-5, 4, 2, 1 << 40]),
              repetition=torch.full((3,), 2.0), bias_ids=torch.arange(4, dtype=torch.int32),
              bias_values=torch.ones(4), bias_offsets=torch.tensor([-1, 1, 1 << 35, 3]))
    x = torch.randn(3, n, generator=gen(0))
    got = ops().edit_logits(x.cuda(), ops().AnswerRules(3, n, **on_gpu(kw)))
    same(got, V.rules(x, n, dtype=F32, **kw))


@pytest.mark.parametrize("case", RULES, ids=lambda c: "x".join(map(str, c)))
def test_answer_margin(case):
    rows, n, hist, biases, masks = case
    kw = make_rules(rows, n, seed=rows + 2 * n, hist=hist, biases=biases, masks=masks)
    g = gen(n + 1)
    x = torch.randn(rows, n, generator=g) * 3
    r = torch.rand(rows, n, generator=g)
    labels = torch.randint(0, n, (rows,), generator=g)
    m, j = V.margin(x - r, x + r, labels, n, **kw)
    gm, gj = ops().answer_margin((x - r).cuda(), (x + r).cuda(), labels.cuda(),
                                 ops().AnswerRules(rows, n, **on_gpu(kw)))
    same(gm, m)
    assert torch.equal(gj.cpu(), j)
    m64, _ = V.margin(x - r, x + r, labels, n, dtype=torch.float64, **kw)
    fin = m64.isfinite()
    assert ((gm.cpu().double() - m64)[fin].abs() <= 14 * V.half_step(F32) * 60.0).all()


def test_answer_margin_edges():
    inf, nan = math.inf, math.nan
    n = 5
    l = torch.tensor([[3.0, 0, 0, 0, 0], [nan, 0, 0, 0, 0], [3, 0, 0, 0, 0], [inf, 0, 0, 0, 0], [-inf, 0, 0, 0, 0],
                      [3, 0, 0, 0, 0], [3, 0, 0, 0, 0], [3, 0, 0, 0, 0], [-inf, 0, 0, 0, 0]])
    u = torch.tensor([[9.0, 1, 2, 2, 1], [9, 1, 2, 2, 1], [9, 1, nan, 2, 1], [inf, inf, 2, 2, 1],
                      [9, -inf, -inf, -inf, -inf], [9, 1, 2, 2, 1], [9, 1, 2, 2, 1], [9, 1, 2, 2, 1], [9, 1, 2, 2, 1]])
    labels = torch.tensor([0, 0, 0, 0, 0, -1, 5, 0, 0])
    free = torch.ones(9, n, dtype=torch.bool)
    free[7, 1:] = False
    free[8] = False
    kw = dict(allowed=V.pack(free))
    m, j = V.margin(l, u, labels, n, **kw)
    assert m.tolist() == [1.0, -inf, -inf, -inf, -inf, -inf, -inf, inf, -inf]
    assert j.tolist() == [2, 2, 2, 1, -1, 0, 0, -1, -1]
    gm, gj = ops().answer_margin(l.cuda(), u.cuda(), labels.cuda(), ops().AnswerRules(9, n, **on_gpu(kw)))
    same(gm, m)
    assert torch.equal(gj.cpu(), j)


def test_equal_bounds_name_the_lowest_rival():
    rows, n = 3, 30000
    u = torch.zeros(rows, n)
    labels = torch.tensor([0, 5, 29999])
    gm, gj = ops().answer_margin(u.cuda(), u.cuda(), labels.cuda(), ops().AnswerRules(rows, n))
    assert gm.tolist() == [0.0] * 3 and gj.tolist() == [1, 0, 0]


def test_margin_bounds_every_point():
    """The edit of any logits within the bounds leaves the label ahead by the margin at least:
    float32 edits are monotone, and a float32 difference of them is too."""
    rows, n = 8, 200
    kw = make_rules(rows, n, seed=3, hist=60, biases=20, masks=3)
    g = gen(1)
    x = torch.randn(rows, n, generator=g) * 3
    r = torch.rand(rows, n, generator=g)
    rules = ops().AnswerRules(rows, n, **on_gpu(kw))
    lo, hi = (x - r), (x + r)
    labels = torch.randint(0, n, (rows,), generator=g)
    gm, _ = ops().answer_margin(lo.cuda(), hi.cuda(), labels.cuda(), rules)
    for seed in range(20):
        z = torch.maximum(lo, torch.minimum(hi, lo + (hi - lo) * torch.rand(rows, n, generator=gen(seed))))
        v = ops().edit_logits(z.cuda(), rules).cpu()
        mine = v.gather(1, labels[:, None])[:, 0]
        best = v.scatter(1, labels[:, None], -math.inf).max(dim=1).values
        d = mine - best
        assert (d >= gm.cpu())[~d.isnan()].all()


def test_rules_in_a_graph():
    rows, n = 4, 5000
    kw = make_rules(rows, n, seed=6, hist=100, biases=10, masks=2)
    dev = on_gpu(kw)
    rules = ops().AnswerRules(rows, n, **dev)
    x = torch.randn(rows, n, generator=gen(0))
    xd, labels = x.cuda(), torch.zeros(rows, dtype=torch.int64).cuda()
    ops().edit_logits(xd, rules)
    ops().answer_margin(xd, xd, labels, rules)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops().edit_logits(xd, rules)
        m, j = ops().answer_margin(xd, xd, labels, rules)
    other = make_rules(rows, n, seed=7, hist=100, biases=10, masks=2)
    for k in ("repetition", "frequency", "presence", "allowed", "allowed_row"):
        dev[k].copy_(other[k])
        kw[k] = other[k]
    x = torch.randn(rows, n, generator=gen(5))
    xd.copy_(x)
    g.replay()
    torch.cuda.synchronize()
    same(y, V.rules(x, n, dtype=F32, **kw))
    wm, wj = V.margin(x, x, torch.zeros(rows, dtype=torch.int64), n, **kw)
    same(m, wm)
    assert torch.equal(j.cpu(), wj)


def test_adapters_then_rules():
    """A batch of requests answering: adapted projection, rules, and the certified margin of the
    answers under a bound of the projection's inputs, on one stream without a synchronisation."""
    o = ops()
    T, K, n = 24, 96, 130
    t = make(T, K, n, 8, 3, 6, F32, False, seed=21)
    kw = make_rules(T, n, seed=22, hist=30, biases=5, masks=3)
    rules = o.AnswerRules(T, n, **on_gpu(kw))
    y = o.adapter_matmul(t["x"].cuda(), layer(t), t["offsets"].cuda(), t["ids"].cuda())
    v = o.edit_logits(y, rules)
    best = v.argmax(dim=1)
    m, rival = o.answer_margin(y, y, best, rules)
    want, tol = oracle(t, False)
    V.check(y, want, tol)
    same(v, V.rules(y.cpu(), n, dtype=F32, **kw))
    wm, wj = V.margin(y.cpu(), y.cpu(), best.cpu(), n, **kw)
    same(m, wm)
    assert torch.equal(rival.cpu(), wj)
    ok = (v.gather(1, best[:, None])[:, 0] > -math.inf).cpu()
    assert (m.cpu()[ok] >= 0).all()


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("rows", [256, 1000, 1024, 1100, 1281])
def test_requests_at_the_tiles_bounds(sub, rows):
    """Requests that begin and end at, before and behind the bounds of row tiles; ranks that go row by
    row beside those that do not; NaN stays with its request."""
    K, N, R = 136, 5000, 48
    cuts = [c for c in (0, 128, 200, 256, 300, 512, 640, 700, 704, 768, 900, 1024, 1050, 1152, 1200) if c < rows] + [rows]
    t = make(rows, K, N, R, 7, len(cuts) - 1, BF16, sub, seed=71)
    t["offsets"] = torch.tensor(cuts)
    t["ids"] = torch.tensor([0, 1, 1, 2, 2, -1, 3, 4, 3, 5, 5, 3, 0, 4, 4, 4][:len(cuts) - 1], dtype=torch.int32)
    t["ranks"] = torch.tensor([48, 32, 16, 48, 5, 0, 48], dtype=torch.int32)
    compare(t, sub)
    want, tol = oracle(t, sub)
    for e in (0, 2, 3):
        u = dict(t, A=t["A"].clone(), B=t["B"].clone())
        u["A"][e] = math.nan
        u["B"][e, 3] = math.inf
        got = ops().adapter_matmul(u["x"].cuda(), layer(u), u["offsets"].cuda(), u["ids"].cuda(), substitute=sub)
        for q, i in enumerate(t["ids"].tolist()):
            if i != e:
                V.check(got[cuts[q]:cuts[q + 1]], want[cuts[q]:cuts[q + 1]], tol[cuts[q]:cuts[q + 1]], f"{e} {q}")
            else:
                assert got[cuts[q]:cuts[q + 1]].isnan().all()
    # the first and last rows are no request's
    t["offsets"] = torch.tensor([c + 1 for c in cuts[:-1]] + [rows - 2])
    before = torch.randn(rows, N, generator=gen(3)).to(BF16)
    y, tol = oracle(t, sub, out=before)
    V.check(ops().adapter_matmul(t["x"].cuda(), layer(t), t["offsets"].cuda(), t["ids"].cuda(), substitute=sub,
                                 out=before.cuda()), y, tol)
    ops().adapter_check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_beside_their_results(dtype):
    """x and y as columns of one buffer, logits and result too."""
    t = make(37, 40, 56, 8, 3, 4, dtype, False, seed=51)
    buf = torch.full((37, 120), 7.0, dtype=dtype, device="cuda")
    buf[:, 8:48] = t["x"].cuda()
    out = buf[:, 48:104]
    out.zero_()
    ops().adapter_matmul(buf[:, 8:48], layer(t), t["offsets"].cuda(), t["ids"].cuda(), out=out)
    V.check(out, *oracle(t, False))
    assert (buf[:, :8] == 7).all() and (buf[:, 104:] == 7).all()
    kw = make_rules(37, 50, seed=52, hist=9, biases=3, masks=2)
    x = torch.randn(37, 50, generator=gen(2)).to(dtype)
    buf[:, 1:51] = x.cuda()
    ops().edit_logits(buf[:, 1:51], ops().AnswerRules(37, 50, **on_gpu(kw)), out=buf[:, 51:101])
    same(buf[:, 51:101].float(), V.rules(x.float(), 50, dtype=F32, **kw).to(dtype).float())
    assert (buf[:, :1] == 7).all() and torch.equal(buf[:, 1:51].cpu(), x)


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,Q", [(3, 2), (40, 2), (300, 200)])
def test_broadcast_operands(dtype, sub, T, Q):
    """One row of x for all rows, and one adapter's tensors under every id."""
    t = make(T, 64, 72, 8, 3, Q, dtype, sub, seed=61)
    t["x"] = t["x"][:1].expand(T, 64)
    t["A"], t["B"] = t["A"][:1].expand(3, -1, -1), t["B"][:1].expand(3, -1, -1)
    d = {k: t[k].cuda() for k in ("W", "scale", "offsets", "ids")}
    A, B = t["A"][:1].contiguous().cuda().expand(3, -1, -1), t["B"][:1].contiguous().cuda().expand(3, -1, -1)
    x = t["x"][:1].contiguous().cuda().expand(T, 64)
    L = ops().AdapterLayer(d["W"], A, B, d["scale"])
    V.check(ops().adapter_matmul(x, L, d["offsets"], d["ids"], substitute=sub), *oracle(t, sub))
    ops().adapter_check()


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_adapter_grid_of_wide_tiles(dtype, sub):
    """Enough tiles that every SM walks over several, the last ones ragged in both directions."""
    compare(make(4000, 72, 5208, 32, 5, 9, dtype, sub, seed=31, ranks=True, bias=True), sub)
    compare(make(8000, 136, 2056, 72, 3, 60, dtype, sub, seed=32), sub)


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,N", [(4, 96), (300, 96), (300, 9000)])
def test_an_infinity_stays_with_its_row(dtype, sub, T, N):
    t = make(T, 64, N, 8, 3, 3, dtype, sub, seed=85, style="tokens")
    want, tol = oracle(t, sub)
    x = t["x"].clone()
    x[T // 2, 7] = math.inf
    got = ops().adapter_matmul(x.cuda(), layer(t), t["offsets"].cuda(), t["ids"].cuda(), substitute=sub)
    assert not got[T // 2].isfinite().any()
    keep = torch.arange(T) != T // 2
    V.check(got[keep.cuda()], want[keep], tol[keep])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_results_of_more_than_2_31_elements(dtype):
    """The rows at the far end of a large result are those of a call with these rows alone."""
    T, K, N, tail = 33001, 64, 66000, 150
    t = make(T, K, N, 8, 3, 5, dtype, False, seed=81, style="tokens")
    L = layer(t)
    y = ops().adapter_matmul(t["x"].cuda(), L, t["offsets"].cuda(), t["ids"].cuda())
    u = dict(t, x=t["x"][-tail:], offsets=(t["offsets"] - (T - tail)).clamp(min=0))
    V.check(y[-tail:], *oracle(u, False))
    del y
    rows, n = 16500, 131072
    kw = make_rules(2, n, seed=82, hist=50, biases=9, masks=1)
    at = [0, rows - 1]                         # the rules of the first and the last row
    for k in ("token_offsets", "bias_offsets"):
        kw[k] = torch.cat([kw[k][:1], kw[k][1:2].expand(rows - 1), kw[k][2:]])
    for k in ("prompt_len", "repetition", "frequency", "presence", "allowed_row"):
        full = torch.full((rows,), -1 if k == "allowed_row" else 1, dtype=kw[k].dtype)
        full[at] = kw[k]
        kw[k] = full
    x = torch.zeros(rows, n, dtype=dtype, device="cuda")
    ends = (torch.randn(2, n, generator=gen(1)) * 3).to(dtype)
    x[at] = ends.cuda()
    rules = ops().AnswerRules(rows, n, **on_gpu(kw))
    got = ops().edit_logits(x, rules)
    small = {k: v[at] if k in ("prompt_len", "repetition", "frequency", "presence", "allowed_row") else v
             for k, v in kw.items()}
    for k in ("token_offsets", "bias_offsets"):
        small[k] = torch.stack([kw[k][0], kw[k][1], kw[k][-1]])
    same(got[at].float(), V.rules(ends.float(), n, dtype=F32, **small).to(dtype).float())
    assert not got[1:-1].any()
    if dtype is F32:
        labels = torch.full((rows,), 7)
        m, j = ops().answer_margin(x, x, labels.cuda(), rules)
        wm, wj = V.margin(ends, ends, labels[:2], n, **small)
        same(m[at], wm)
        assert torch.equal(j[at].cpu(), wj)
        assert not m[1:-1].any() and not j[1:-1].any()


def test_rules_on_two_streams_at_once():
    rows, n = 40, 60000
    xs, want, rules = [], [], []
    for i in range(2):
        kw = make_rules(rows, n, seed=90 + i, hist=3000 * (i + 1), biases=40, masks=3)
        x = torch.randn(rows, n, generator=gen(i)) * 3
        labels = x.argmax(dim=1)
        xs.append((x.cuda(), labels.cuda()))
        rules.append(ops().AnswerRules(rows, n, **on_gpu(kw)))
        want.append((V.rules(x, n, dtype=F32, **kw), *V.margin(x, x, labels, n, **kw)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, labels = xs[i]
                got[i] = (ops().edit_logits(x, rules[i]), *ops().answer_margin(x, x, labels, rules[i]))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            same(g[0], w[0])
            same(g[1], w[1])
            assert torch.equal(g[2].cpu(), w[2])


@pytest.mark.parametrize("adapted", [False, True])
@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("K", [1027, 4096])
def test_float32_precision_of_long_contractions(K, sub, adapted):
    """The error of whole results, which the bounds of single values above do not hold to what
    emptying the accumulator gives.  Relative to the root mean square of y, for independent terms:

    * a chunk of 64 columns is 24 additions that truncate, each by half of 2^-23 of its partial sum on
      average; partial sums grow as a root, so the 24 make at most 2/3 * 24 * 2^-24 of the chunk's, and the
      chunks' together at most that of y's;
    * hi + lo keeps 22 bits of each operand and lo * lo is left out: 2^-22 of a product;
    * the chunks' sums are added with rounding: 2^-25 * sqrt(K / 64) at K = 4096, less than 2^-22.

    16 * 2^-24 + 2 * 2^-22 in all (1.4e-6), twice for the chained low-rank part.  Without
    chunks the first term would be K / 64 times that, one TF32 product would be off by 2^-11."""
    T, N, R, Q = 1100, 384, 32, 3
    t = make(T, K, N, R, 2, Q, F32, sub, seed=K)
    if not adapted:
        t["ids"] = torch.full((Q,), -1, dtype=torch.int32)
    d = {k: t[k].cuda() for k in ("x", "W", "A", "B")}
    got = ops().adapter_matmul(d["x"], layer(t), t["offsets"].cuda(), t["ids"].cuda(), substitute=sub)
    d = {k: v.double() for k, v in d.items()}
    base = d["x"] @ (d["W"] if sub else d["W"].t())
    low = torch.zeros_like(base)
    for q, e in enumerate(t["ids"].tolist()):
        a, b = int(t["offsets"][q]), int(t["offsets"][q + 1])
        if e >= 0:
            P, O = (d["B"][e], d["A"][e]) if sub else (d["A"][e].t(), d["B"][e].t())
            low[a:b] = float(t["scale"][e]) * (d["x"][a:b] @ P) @ O

    def rms(z):
        return float(z.square().mean().sqrt())
    off = got.double() - base - low
    allowed = (16 * 2.0**-24 + 2 * 2.0**-22) * (rms(base) + 2 * rms(low))
    assert rms(off) <= allowed, (rms(off) / allowed, rms(off) / rms(base + low))
    towards_zero = float((off * (base + low).sign()).mean())
    assert abs(towards_zero) <= allowed, (towards_zero / allowed)
