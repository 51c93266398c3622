"""Failure detection of the adapter product without a GPU fault: bounded device waits that run out.

With a short poll limit (CF_WAIT_POLLS) and one arrival withheld (CF_FAULT=adapter_withhold_stage:
the barrier of each CTA's first stage of operands expects an arrival that nothing makes), the loads
of a later step wait for that stage and give up, the MMAs wait for the loads, the epilogue for the
MMAs.  Copies and MMAs in flight are awaited before shared memory and tensor memory are released,
adapter_check reports the site, and the next call, without the fault, gives the usual bits.
"""
import re

import pytest
import torch

from test_gpu_variants import BF16, F16, F32, layer, make, ops

pytestmark = pytest.mark.gpu

# the bounded waits of k_adapter_tile, k_adapter_wide and k_adapter_f32
TILE, WIDE, F32_SITES = {11, 21, 41}, {81, 83, 84, 86}, {51, 61, 62, 71}

# more steps of the contraction than stages in every CTA
CASES = [
    # dtype, T, K, N, sites of v's kernel and of the product's
    (BF16, 200, 1024, 256, TILE), (F16, 200, 1024, 256, TILE),
    (BF16, 1024, 512, 1280, TILE | WIDE), (F16, 1024, 512, 2304, TILE | WIDE),
    (F32, 1100, 128, 520, F32_SITES),
]


def withhold(monkeypatch):
    monkeypatch.setenv("CF_WAIT_POLLS", "65536")
    monkeypatch.setenv("CF_FAULT", "adapter_withhold_stage")


def restore(monkeypatch):
    monkeypatch.delenv("CF_FAULT")
    monkeypatch.delenv("CF_WAIT_POLLS")


def gave_up(call):
    """The site at which a bounded wait gave up, as `call` reports it."""
    from cfgpu import _lib
    with pytest.raises(_lib.CfError) as e:
        call()
    m = re.search(r"gave up \(site (\d+)\)", str(e.value))
    assert m and e.value.status == _lib.CF_ERR_TIMEOUT, e.value
    return int(m.group(1))


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[1:4])) + str(c[0])[5:])
def test_a_stage_that_is_never_released(monkeypatch, case, sub):
    dtype, T, K, N, sites = case
    t = make(T, K, N, 16, 3, 3, dtype, sub, seed=8)
    args = t["x"].cuda(), layer(t), t["offsets"].cuda(), t["ids"].cuda(), sub
    good = ops().adapter_matmul(*args)
    ops().adapter_check()
    withhold(monkeypatch)
    ops().adapter_matmul(*args)
    assert gave_up(ops().adapter_check) in sites
    restore(monkeypatch)
    ops().adapter_check()                      # reported once
    assert torch.equal(ops().adapter_matmul(*args), good)
    ops().adapter_check()


def test_later_waits_do_not_give_up_on_an_earlier_one(monkeypatch):
    """Until it is reported, a wait that gave up is a record only: a later call whose epilogue waits
    through a contraction of 2^20 gives the usual bits."""
    K = 1 << 20
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x, W = (torch.randn(128, K, generator=g, device="cuda").bfloat16() for _ in range(2))
    L = ops().AdapterLayer(W, W.new_empty(1, 0, K), W.new_empty(1, 128, 0), torch.ones(1, device="cuda"))
    rest = torch.tensor([0, 128]).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    good = ops().adapter_matmul(x, L, *rest)
    t = make(200, 1024, 256, 16, 3, 3, BF16, False, seed=8)
    withhold(monkeypatch)
    ops().adapter_matmul(t["x"].cuda(), layer(t), t["offsets"].cuda(), t["ids"].cuda())
    torch.cuda.synchronize()
    restore(monkeypatch)
    for _ in range(3):
        assert torch.equal(ops().adapter_matmul(x, L, *rest), good)
    assert gave_up(ops().adapter_check) in TILE
    ops().adapter_check()


def test_the_engine_reports_a_wait_that_gave_up(monkeypatch):
    """run and answer with check_device raise, and succeed on the next call.  64 regions: 3200 rows
    through 50 x 784 weights are more tiles than CTAs, so some need a stage twice."""
    from cfgpu import nets
    from test_gpu_variants_engine import dev, engine, make as network
    wl, y, l0, u0, adapters, ids = network(B=64)
    eng = engine(wl, adapters)
    eng.graphs = False                                  # a captured pass keeps the launches it was made of
    box, spec = (l0.to(dev()), u0.to(dev())), nets.spec_weight(y).to(dev())
    kw = dict(adapter_ids=ids.to(dev()), check_device=True)
    rules = ops().AnswerRules(64, 10)
    lb, ub = eng.run(*box, spec, **kw)
    margin, _ = eng.answer(*box, y.to(dev()), rules, **kw)
    withhold(monkeypatch)
    assert gave_up(lambda: eng.run(*box, spec, **kw)) in F32_SITES
    assert gave_up(lambda: eng.run(*box, spec, want_state=True, **kw)) in F32_SITES
    assert gave_up(lambda: eng.answer(*box, y.to(dev()), rules, **kw)) in F32_SITES
    restore(monkeypatch)
    again = eng.run(*box, spec, **kw)
    assert torch.equal(again[0], lb) and torch.equal(again[1], ub)
    assert torch.equal(eng.answer(*box, y.to(dev()), rules, **kw)[0], margin)
