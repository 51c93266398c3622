"""Certifying adapted variants of one network in one batch, and answers under rules."""
import math

import numpy as np
import pytest
import torch

import variants_oracle as V

pytestmark = pytest.mark.gpu
E, RANK = 3, 4


def dev():
    return torch.device("cuda:0")


def make(wid=0, B=6, seed=0, adapted=(0, 2, 4)):
    """The 784-50x3-10 network (or the residual one) with adapters in some linear layers."""
    from cfgpu import nets
    wl = nets.workload(wid)
    X = nets.centres(wl, B)
    y = nets.labels(wl, X)
    l0, u0 = nets.input_box(X, wl.eps, wl.dataset)
    g = torch.Generator()
    g.manual_seed(seed)
    linear = [i for i, L in enumerate(wl.layers) if L.kind == "linear"]
    adapters = {}
    for i in linear:
        if adapted is None or i in adapted:
            n_out, n_in = wl.layers[i].W.shape
            adapters[i] = (torch.randn(E, RANK, n_in, generator=g) * n_in**-0.5,
                           torch.randn(E, n_out, RANK, generator=g) * 0.3, torch.rand(E, generator=g) + 0.5)
    ids = (torch.arange(B) % (E + 1) - 1).to(torch.int32)
    return wl, y, l0, u0, adapters, ids


def merged(wl, adapters, e):
    """The layers of variant e, its adapters added to the weights (in float64, rounded once)."""
    import copy
    layers = []
    for i, L in enumerate(wl.layers):
        L = copy.copy(L)
        if e >= 0 and i in adapters:
            A, B, s = adapters[i]
            L.W = (torch.as_tensor(L.W).double() + float(s[e]) * B[e].double() @ A[e].double()).float().numpy()
        layers.append(L)
    return layers


def points(layers, z):
    """The network's values at points z [n, n0], float64, layer by layer."""
    vals = []
    for i, L in enumerate(layers):
        parents = getattr(L, "parents", None) or (i - 1,)
        ins = [z if p < 0 else vals[p] for p in parents]
        if L.kind == "linear":
            vals.append(ins[0] @ torch.as_tensor(L.W).double().t() + torch.as_tensor(L.b).double())
        elif L.kind == "relu":
            vals.append(ins[0].clamp(min=0))
        elif L.kind == "add":
            vals.append(ins[0] + ins[1])
        else:
            vals.append(torch.cat(ins, dim=1))
    return vals


def engine(wl, adapters, layers=None):
    from cfgpu.engine import DeepPolyEngine
    return DeepPolyEngine(layers or wl.layers, wl.input_size, dev(), adapters=adapters)


@pytest.mark.parametrize("graphs", [True, False])
def test_each_region_is_bounded_for_its_variant(graphs):
    """The bounds equal those of a network with the adapter merged into its weights, which
    replays the same ReLU decisions: 8e-5 of the layer's largest bound (the measured float32
    disagreement of two implementations with equal decisions) plus 1e-5 of the value."""
    from cfgpu import nets
    wl, y, l0, u0, adapters, ids = make()
    B = l0.shape[0]
    spec = nets.spec_weight(y).to(dev())
    eng = engine(wl, adapters)
    eng.graphs = graphs
    for turn in range(2):                     # a second batch through the same captured pass
        lb, ub, sl, su = eng.run(l0.to(dev()), u0.to(dev()), spec, want_state=True, adapter_ids=ids.to(dev()))
        sl, su = sl.clone(), su.clone()
        for e in range(-1, E):
            m = engine(wl, None, merged(wl, adapters, e))
            _, _, ml, mu = m.run(l0.to(dev()), u0.to(dev()), spec, want_state=True, replay=(sl, su))
            rows = [b for b in range(B) if int(ids[b]) == e]
            at = wl.input_size
            for L in list(wl.layers) + [None]:
                n = 9 if L is None else L.n_out
                for got, want in ((sl, ml), (su, mu)):
                    g, w = got[rows, at:at + n].double(), want[rows, at:at + n].double()
                    S = torch.maximum(ml[rows, at:at + n].abs(), mu[rows, at:at + n].abs()).double().amax()
                    assert ((g - w).abs() <= 1e-5 * w.abs() + 8e-5 * S).all(), (e, at, float((g - w).abs().max() / S))
                at += n
        assert torch.equal(lb.float(), sl[:, -9:]) and torch.equal(ub.float(), su[:, -9:])
        ids = ids.roll(1)


@pytest.mark.parametrize("wid", [0, 5, 6])
def test_bounds_hold_at_points(wid):
    """Chain, residual and concat networks: the variant's own values lie within its bounds."""
    from cfgpu import nets
    wl, y, l0, u0, adapters, ids = make(wid, adapted=None)
    spec = nets.spec_weight(y)
    _, _, sl, su = engine(wl, adapters).run(l0.to(dev()), u0.to(dev()), spec.to(dev()), want_state=True,
                                            adapter_ids=ids.to(dev()))
    sl, su = sl.cpu().double(), su.cpu().double()
    g = torch.Generator()
    g.manual_seed(1)
    for b in range(l0.shape[0]):
        layers = merged(wl, adapters, int(ids[b]))
        z = l0[b].double() + (u0[b] - l0[b]).double() * torch.rand(40, l0.shape[1], generator=g).round().double()
        vals = points(layers, z)
        v = torch.cat(vals + [vals[-1] @ spec[b].double().t()], dim=1)
        lo, up = sl[b, wl.input_size:], su[b, wl.input_size:]
        slack = 1e-4 * torch.maximum(lo.abs(), up.abs()).max()
        assert (v >= lo - slack).all() and (v <= up + slack).all()


def test_without_ids_the_network_itself_runs():
    from cfgpu import nets
    wl, y, l0, u0, adapters, ids = make()
    spec = nets.spec_weight(y).to(dev())
    a = engine(wl, adapters).run(l0.to(dev()), u0.to(dev()), spec)
    b = engine(wl, None).run(l0.to(dev()), u0.to(dev()), spec)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def rules_for(B, n, seed, repetition):
    import test_gpu_variants as T
    from cfgpu import ops
    kw = T.make_rules(B, n, seed=seed, hist=4, biases=3, masks=2)
    if not repetition:
        kw.pop("repetition")
    return kw, ops.AnswerRules(B, n, **T.on_gpu(kw))


@pytest.mark.parametrize("repetition", [False, True])
@pytest.mark.parametrize("adapted", [False, True])
def test_answer_under_rules(repetition, adapted):
    """At points of a region the edited logits leave the label ahead of every other answer by
    the margin at least (up to the float32 error of the bounds)."""
    wl, y, l0, u0, adapters, ids = make()
    B, n = l0.shape[0], 10
    eng = engine(wl, adapters)
    kw, rules = rules_for(B, n, 3, repetition)
    where = ids.to(dev()) if adapted else None
    margin, rival = eng.answer(l0.to(dev()), u0.to(dev()), y.to(dev()), rules, adapter_ids=where)
    margin, rival = margin.cpu().double(), rival.cpu()
    g = torch.Generator()
    g.manual_seed(2)
    for b in range(B):
        layers = merged(wl, adapters, int(ids[b]) if adapted else -1)
        z = l0[b].double() + (u0[b] - l0[b]).double() * torch.rand(60, l0.shape[1], generator=g).round().double()
        logits = points(layers, z)[-1]
        one = {k: (v[b:b + 1] if k in ("prompt_len", "repetition", "frequency", "presence", "allowed_row") else
                   v[b:b + 2] if k.endswith("offsets") else v) for k, v in kw.items()}
        v = torch.cat([V.rules(p[None], n, **one) for p in logits])
        mine = v[:, int(y[b])]
        others = v.clone()
        others[:, int(y[b])] = -math.inf
        gap = (mine - others.max(dim=1).values)
        gap[gap.isnan()] = -math.inf
        assert (gap >= margin[b] - 1e-4 * logits.abs().max()).all(), b
        if margin[b] > -math.inf and int(rival[b]) >= 0:
            assert others[0, int(rival[b])] > -math.inf


def test_answer_without_edits_is_the_property():
    """No rules at all: the margin is the least of the property's lower bounds."""
    from cfgpu import nets, ops
    wl, y, l0, u0, adapters, ids = make()
    eng = engine(wl, adapters)
    lb, _ = eng.run(l0.to(dev()), u0.to(dev()), nets.spec_weight(y).to(dev()), adapter_ids=ids.to(dev()))
    margin, _ = eng.answer(l0.to(dev()), u0.to(dev()), y.to(dev()), ops.AnswerRules(l0.shape[0], 10),
                           adapter_ids=ids.to(dev()))
    assert torch.equal(margin.double(), lb.min(dim=1).values)


def test_refusals():
    from cfgpu import nets, ops
    from cfgpu.engine import DeepPolyEngine
    wl, y, l0, u0, adapters, ids = make()
    spec = nets.spec_weight(y).to(dev())
    for kw in (dict(certifier="ibp"), dict(stop_depth=1), dict(relu_strict=True)):
        with pytest.raises(NotImplementedError):
            DeepPolyEngine(wl.layers, wl.input_size, dev(), adapters=adapters, **kw)
    with pytest.raises(NotImplementedError, match="only linear"):
        engine(wl, {1: adapters[0]})
    with pytest.raises(ValueError, match="same number"):
        engine(wl, {0: adapters[0], 2: tuple(t[:1] for t in adapters[2])})
    with pytest.raises(Exception, match="SHAPE MISMATCH"):
        engine(wl, {0: adapters[2]})
    eng = engine(wl, adapters)
    box = (l0.to(dev()), u0.to(dev()))
    with pytest.raises(Exception, match="SHAPE MISMATCH"):
        eng.run(*box, spec, adapter_ids=ids.long().to(dev()))
    with pytest.raises(Exception, match="SHAPE MISMATCH"):
        eng.run(*box, spec, adapter_ids=ids[:2].to(dev()))
    with pytest.raises(ValueError, match="without adapters"):
        engine(wl, None).run(*box, spec, adapter_ids=ids.to(dev()))
    with pytest.raises(Exception, match="SHAPE MISMATCH"):
        eng.answer(*box, y.to(dev()), ops.AnswerRules(2, 10))
    with pytest.raises(Exception, match="SHAPE MISMATCH"):
        eng.answer(*box, y.int().to(dev()), ops.AnswerRules(6, 10))


def constant_network(logits):
    """A network whose logits are `logits`, whatever its input: bounds without any slack."""
    from cfgpu.engine import DeepPolyEngine

    class Layer:
        kind, W, b = "linear", torch.zeros(len(logits), 4), logits
    return DeepPolyEngine([Layer()], 4, dev(), n_spec=len(logits) - 1)


def certified(logits, labels, **kw):
    """(margin, the logits as edited) for len(labels) regions of the constant network."""
    from cfgpu import ops
    B, n = len(labels), len(logits)
    rules = ops.AnswerRules(B, n, **{k: v.to(dev()) for k, v in kw.items()})
    box = torch.zeros(B, 4, device=dev()), torch.ones(B, 4, device=dev())
    margin, _ = constant_network(logits).answer(*box, labels.to(dev()), rules)
    return margin.cpu(), ops.edit_logits(logits.expand(B, n).contiguous().to(dev()), rules).cpu()


def test_the_margin_is_of_the_rounded_rule():
    """16777216 + 0.5 is a tie in float32, which 0 + 0.5 against 0 is not."""
    margin, edited = certified(torch.full((2,), 16777216.0), torch.tensor([0]),
                               bias_ids=torch.tensor([0], dtype=torch.int32), bias_values=torch.tensor([0.5]),
                               bias_offsets=torch.tensor([0, 1]))
    assert edited[0, 0] == edited[0, 1] and float(margin[0]) <= 0


@pytest.mark.parametrize("size", [2.0**25, 2.0**12, 1.0])
def test_certified_answers_win_after_rounding(size):
    """Logits a few float32 steps apart and edits of a few steps: a margin above 0 means that the
    label's edited logit is above all others.  The margin is at most 4 * 2^-21 of the magnitudes
    (two answers' allowance of 2^-21 and its rounding, twice for good measure) below the real one."""
    g = torch.Generator()
    g.manual_seed(7)
    B, n = 400, 5
    step = size * 2.0**-23
    for turn in range(4):
        logits = (size + step * torch.randint(-3, 4, (n,), generator=g)).float()
        labels = torch.randint(0, n, (B,), generator=g)
        kw = dict(tokens=torch.randint(0, n, (3 * B,), generator=g).to(torch.int32),
                  token_offsets=torch.arange(0, 3 * B + 1, 3),
                  prompt_len=torch.randint(0, 3, (B,), generator=g).to(torch.int32),
                  frequency=step * torch.randn(B, generator=g), presence=step * torch.randn(B, generator=g),
                  bias_ids=torch.randint(0, n, (2 * B,), generator=g).to(torch.int32),
                  bias_values=(10.0**turn) * step * torch.randn(2 * B, generator=g),
                  bias_offsets=torch.arange(0, 2 * B + 1, 2))
        margin, edited = certified(logits, labels, **kw)
        others = edited.scatter(1, labels[:, None], -math.inf).max(dim=1).values
        mine = edited.gather(1, labels[:, None])[:, 0]
        assert (mine > others)[margin > 0].all()
        real = V.rules(logits.expand(B, n), n, **kw)
        gap = real.gather(1, labels[:, None])[:, 0] - real.scatter(1, labels[:, None], -math.inf).max(dim=1).values
        far = logits.abs().max().double() + 2 * (real - logits.double()).abs().max() + 40 * step * 10.0**turn
        assert (margin.double() <= gap + 2.0**-20 * far).all() and (margin.double() >= gap - 2.0**-19 * far).all()


def test_bans_by_infinite_biases_and_by_sets():
    """An answer with a bias of -inf is out, one with +inf bars any certificate, sets need no
    allowance: the margin is then the difference of the logits itself."""
    logits = torch.tensor([3.0, 5.0, 4.0, 1.0])
    labels = torch.tensor([0, 0, 0])
    margin, _ = certified(logits, labels, bias_ids=torch.tensor([1, 2, 1], dtype=torch.int32),
                          bias_values=torch.tensor([-math.inf, -math.inf, math.inf]),
                          bias_offsets=torch.tensor([0, 2, 2, 3]))
    assert margin.tolist() == [2.0, -2.0, -math.inf]
    margin, _ = certified(logits, labels, allowed=V.pack(torch.tensor([[True, False, False, True]] * 3)))
    assert margin.tolist() == [2.0] * 3


def test_a_device_without_an_index_is_the_current_one():
    from cfgpu import nets, ops
    from cfgpu.engine import DeepPolyEngine
    wl, y, l0, u0, adapters, ids = make()
    eng = DeepPolyEngine(wl.layers, wl.input_size, "cuda", adapters=adapters)
    assert eng.device == torch.device("cuda", torch.cuda.current_device())
    box = l0.cuda(), u0.cuda()
    got = eng.run(*box, nets.spec_weight(y).cuda(), adapter_ids=ids.cuda())
    want = engine(wl, adapters).run(*box, nets.spec_weight(y).cuda(), adapter_ids=ids.cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    eng.answer(*box, y.cuda(), ops.AnswerRules(l0.shape[0], 10), adapter_ids=ids.cuda())


@pytest.mark.parametrize("want_state", [False, True])
def test_calls_on_two_streams(want_state):
    """Calls of one engine on streams of their own, neither waited for: each has its own inputs' bounds."""
    from cfgpu import nets
    wl, y, l0, u0, adapters, ids = make(B=48)
    eng = engine(wl, adapters)
    spec, ids = nets.spec_weight(y).to(dev()), ids.to(dev())
    inputs = []
    for k in range(2):
        inputs.append(((l0 - 0.1 * k).to(dev()), (u0 + 0.1 * k).to(dev()), spec, want_state))
    want = [[t.clone() for t in eng.run(*a, adapter_ids=ids.roll(k))] for k, a in enumerate(inputs)]
    assert not torch.equal(want[0][0], want[1][0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    rolled = [ids.roll(k) for k in range(2)]
    torch.cuda.synchronize()
    for turn in range(10):
        got = []
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got.append(eng.run(*inputs[k], adapter_ids=rolled[k]))
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(g, w) for g, w in zip(got[k], want[k])), (turn, k)


def test_dense_weights_of_the_variants():
    """The weights that a traversal starts from: the shared ones bit for bit without an adapter (also
    where unused adapters hold NaN), else within the float32 roundings of R products, their sums, the
    scale and the last addition: (R + 3) 2^-24 of the magnitudes, doubled for second-order terms."""
    from cfgpu import general, ops
    g = torch.Generator()
    g.manual_seed(5)
    n_out, n_in, R = 37, 53, 6
    W, A, B = (torch.randn(*s, generator=g) for s in ((n_out, n_in), (4, R, n_in), (4, n_out, R)))
    scale, ranks = torch.rand(4, generator=g) + 0.5, torch.tensor([R, 2, 0, 99], dtype=torch.int32)
    A[1, 2:], B[1, :, 2:], A[2], B[2] = math.nan, math.inf, math.nan, math.nan
    ids = torch.tensor([0, -1, 1, 2, 3, 4, -7, 0], dtype=torch.int32)
    layer = ops.AdapterLayer(*(t.to(dev()) for t in (W, A, B, scale, ranks)))
    D = general._Adapted(layer, ids.to(dev())).dense().cpu()
    assert tuple(D.shape) == (8, n_out, n_in)
    for b, e in enumerate(ids.tolist()):
        r = min(R, int(ranks[e])) if 0 <= e < 4 else 0
        if r == 0:
            assert torch.equal(D[b], W)
            continue
        low = float(scale[e]) * B[e, :, :r].double() @ A[e, :r].double()
        size = float(scale[e]) * B[e, :, :r].double().abs() @ A[e, :r].double().abs() + W.double().abs()
        assert ((D[b].double() - W.double() - low).abs() <= 2 * (R + 3) * 2.0**-24 * size).all()
    bad = [t.clone() for t in (A, B, scale)]
    bad[0][0], bad[1][0], bad[2][0] = math.nan, math.inf, math.nan      # the one that ids below 0 clamp to
    layer = ops.AdapterLayer(W.to(dev()), *(t.to(dev()) for t in bad))
    none = general._Adapted(layer, torch.tensor([-1, 9], dtype=torch.int32, device=dev())).dense().cpu()
    assert torch.equal(none[0], W) and torch.equal(none[1], W)


def test_without_an_adapter_the_first_bounds_are_the_networks():
    """Regions of no adapter, beside others: the first layer's bounds are those of the same traversal
    of the network itself, bit for bit."""
    from cfgpu import general, nets
    wl, y, l0, u0, adapters, ids = make(adapted=(0,))
    eng = engine(wl, adapters)
    box, spec = (l0.to(dev()), u0.to(dev())), nets.spec_weight(y).to(dev())
    some, _ = general.run(eng._general, *box, spec, "deeppoly", eng._adapters, ids.to(dev()))
    plain, _ = general.run(eng._general, *box, spec, "deeppoly")
    rows = ids == -1
    assert rows.any()
    for got, want in zip(some[0], plain[0]):
        assert torch.equal(got.cpu()[rows], want.cpu()[rows])


@pytest.mark.parametrize("graphs", [True, False])
def test_adapters_are_exchanged_by_writing_into_them(graphs):
    """Tensors on the engine's device are read at every call, also by a captured pass."""
    from cfgpu import nets
    wl, y, l0, u0, adapters, ids = make()
    box, spec, ids = (l0.to(dev()), u0.to(dev())), nets.spec_weight(y).to(dev()), ids.to(dev())
    held = {i: tuple(t.to(dev()) for t in a) for i, a in adapters.items()}
    eng = engine(wl, held)
    eng.graphs = graphs
    before = eng.run(*box, spec, adapter_ids=ids)[0].clone()
    other = make(seed=1)[4]
    for i, a in held.items():
        for t, n in zip(a, other[i]):
            t.copy_(n)
    fresh = engine(wl, other)
    fresh.graphs = graphs
    after = eng.run(*box, spec, adapter_ids=ids)[0]
    assert torch.equal(after, fresh.run(*box, spec, adapter_ids=ids)[0]) and not torch.equal(after, before)


@pytest.mark.parametrize("certifier", ["deeppoly", "crown", "zono", "ibp", "crownibp"])
def test_answers_of_every_certifier(certifier):
    """Biases and sets on the bounds of each certifier: the margin is the property's plus the edits
    (whole numbers), less the allowance of 2^-21 of the magnitudes and their rounding, here 2^-17 of
    them; and the values at points of a region keep it, up to the float32 error of the bounds.  Not
    so CROWN's: its program takes one branch for a whole layer, and its property's bounds do not
    hold at points either."""
    from cfgpu import nets, ops
    from cfgpu.engine import DeepPolyEngine
    wl, y, l0, u0, _, _ = make()
    B, n = l0.shape[0], 10
    u0 = l0 + (u0 - l0) * 0.05
    eng = DeepPolyEngine(wl.layers, wl.input_size, dev(), certifier=certifier)
    box = l0.to(dev()), u0.to(dev())
    kw, _ = rules_for(B, n, 3, False)
    kw = {k: kw[k] for k in ("bias_ids", "bias_values", "bias_offsets", "allowed", "allowed_row")}
    kw["bias_values"] = kw["bias_values"].round()
    margin = eng.answer(*box, y.to(dev()), ops.AnswerRules(B, n, **{k: v.to(dev()) for k, v in kw.items()}))[0].cpu()
    lb = eng.run(*box, nets.spec_weight(y).to(dev()))[0].cpu()
    g = torch.Generator()
    g.manual_seed(3)
    edits = V.rules(torch.zeros(B, n), n, **kw)
    for b in range(B):
        z = l0[b].double() + (u0[b] - l0[b]).double() * torch.rand(40, l0.shape[1], generator=g).double()
        logits = points(wl.layers, z)[-1]
        label = int(y[b])
        v = logits + edits[b]
        others = v.clone()
        others[:, label] = -math.inf
        gap = v[:, label] - others.max(dim=1).values
        gap[gap.isnan()] = -math.inf
        size = logits.abs().max() + lb[b].abs().max() + edits[b][edits[b] > -math.inf].abs().sum()
        if certifier != "crown":
            assert (gap >= margin[b].double() - 1e-4 * size).all(), b
        others = [j for j in range(n) if j != label]
        want = min(float(lb[b, i] + edits[b, label] - edits[b, j]) if edits[b, label] > -math.inf else -math.inf
                   for i, j in enumerate(others) if edits[b, j] > -math.inf)
        if want == -math.inf:
            assert margin[b] == -math.inf
        else:
            assert abs(float(margin[b]) - want) <= 2.0**-17 * float(size + 1), (b, float(margin[b]), want)


@pytest.mark.parametrize("before", [True, False])
def test_run_and_answer_in_a_callers_graph(before):
    """Captured by the caller, with and without an eager call before it, and replayed on other inputs."""
    from cfgpu import nets, ops
    wl, y, l0, u0, adapters, ids = make()
    eng, other = engine(wl, adapters), engine(wl, adapters)
    box, spec, ids, y = (l0.to(dev()), u0.to(dev())), nets.spec_weight(y).to(dev()), ids.to(dev()), y.to(dev())
    kw, rules = rules_for(l0.shape[0], 10, 3, False)
    warm = engine(wl, adapters)                    # kernels' first uses
    warm.run(*box, spec, adapter_ids=ids)
    warm.answer(*box, y, rules, adapter_ids=ids)
    if before:
        eng.run(*box, spec, adapter_ids=ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lb, ub = eng.run(*box, spec, adapter_ids=ids)
        margin, rival = eng.answer(*box, y, rules, adapter_ids=ids)
    for turn in range(2):
        if turn:
            box[0].sub_(0.01)
            ids.copy_(ids.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        want = other.run(*box, spec, adapter_ids=ids)
        assert torch.equal(lb, want[0]) and torch.equal(ub, want[1])
        m, j = other.answer(*box, y, rules, adapter_ids=ids)
        assert torch.equal(margin, m) and torch.equal(rival, j)
    again = eng.run(*box, spec, adapter_ids=ids)   # the engine's own pass still is one
    assert torch.equal(again[0], lb) and eng.graphs
