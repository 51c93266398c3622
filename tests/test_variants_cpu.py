"""Per-request adapters and answer rules without a GPU: refusals before any launch, and the
64-bit forms that the GPU tests compare with, against independent statements of them."""
import ctypes
import math

import pytest
import torch

import variants_oracle as V
from cfgpu import _lib, ops


def c_layer(**kw):
    d = dict(dtype=_lib.CF_BF16, n_adapters=2, rank=4, reserved=0, n_out=32, n_in=16, W_dev=256, w_rs=16, bias_dev=None,
             A_dev=256, a_es=64, a_rs=16, B_dev=256, b_es=128, b_rs=4, scale_dev=256, ranks_dev=None)
    d.update(kw)
    return _lib.CfAdapterLayer(**d)


def call(L, substitute=0, T=8, x=256, x_rs=16, q=2, off=256, ids=256, y=4096, y_rs=32, ws=1 << 16, wsb=None):
    if wsb is None:
        wsb = _lib.lib.cf_adapter_workspace_bytes(ctypes.byref(L), substitute, T, x, x_rs, q)
    return _lib.lib.cf_adapter_matmul(ctypes.byref(L), substitute, T, x, x_rs, q, off, ids, y, y_rs, ws, wsb, None)


@pytest.mark.parametrize("layer,args,status", [
    (dict(dtype=_lib.CF_BOOL), {}, "UNSUPPORTED"), (dict(dtype=9), {}, "UNSUPPORTED"),
    (dict(n_out=-1), {}, "SHAPE"), (dict(rank=-1), {}, "SHAPE"), (dict(w_rs=15), {}, "SHAPE"),
    (dict(a_rs=15), {}, "SHAPE"), (dict(b_rs=3), {}, "SHAPE"), (dict(W_dev=257), {}, "SHAPE"),
    (dict(W_dev=None), {}, "NULL"), (dict(A_dev=None), {}, "NULL"), (dict(B_dev=None), {}, "NULL"),
    (dict(scale_dev=None), {}, "NULL"),
    ({}, dict(T=-1), "SHAPE"), ({}, dict(q=-1), "SHAPE"), ({}, dict(y_rs=31), "SHAPE"), ({}, dict(x_rs=-1), "SHAPE"),
    ({}, dict(x=None), "NULL"), ({}, dict(y=None), "NULL"), ({}, dict(off=None), "NULL"), ({}, dict(ids=None), "NULL"),
    ({}, dict(wsb=0), "WORKSPACE"), ({}, dict(ws=None), "WORKSPACE"), ({}, dict(ws=(1 << 16) + 8), "WORKSPACE"),
])
def test_adapter_refusals(layer, args, status):
    st = call(c_layer(**layer), **args)
    assert st == getattr(_lib, f"CF_ERR_{status}"), _lib.lib.cf_last_error()
    assert _lib.lib.cf_last_error()


def test_nothing_to_do_is_no_error():
    assert call(c_layer(), T=0) == _lib.CF_OK
    assert call(c_layer(), q=0) == _lib.CF_OK
    assert call(c_layer(n_out=0)) == _lib.CF_OK


def test_adapter_fault_injection(monkeypatch):
    monkeypatch.setenv("CF_FAULT", "adapter_matmul")
    assert call(c_layer()) == _lib.CF_ERR_INJECTED


def c_rules(**kw):
    d = dict(rows=2, n=10)
    d.update(kw)
    return _lib.CfAnswerRules(**d)


@pytest.mark.parametrize("rules,status", [
    (dict(rows=-1), "SHAPE"), (dict(n=1 << 31), "SHAPE"), (dict(n_tokens=1 << 31), "SHAPE"),
    (dict(tokens_dev=256), "NULL"), (dict(token_offsets_dev=256), "NULL"), (dict(repetition_dev=256), "NULL"),
    (dict(bias_ids_dev=256, bias_offsets_dev=256), "NULL"), (dict(allowed_row_dev=256), "NULL"),
    (dict(allowed_dev=256, n_masks=1, allowed_words=1), "SHAPE"),
    (dict(allowed_dev=256, n_masks=2, allowed_words=0), "SHAPE"),
])
def test_rules_refusals(rules, status):
    R = c_rules(**rules)
    want = getattr(_lib, f"CF_ERR_{status}")
    assert _lib.lib.cf_edit_logits(ctypes.byref(R), _lib.CF_F32, 256, 10, 4096, 10, None) == want
    assert _lib.lib.cf_answer_margin(ctypes.byref(R), 256, 10, 256, 10, 256, 256, 256, None) == want


def test_edit_and_margin_refusals():
    R = c_rules()
    ref = ctypes.byref(R)
    e, m = _lib.lib.cf_edit_logits, _lib.lib.cf_answer_margin
    assert e(None, _lib.CF_F32, 256, 10, 4096, 10, None) == _lib.CF_ERR_NULL
    assert e(ref, _lib.CF_BOOL, 256, 10, 4096, 10, None) == _lib.CF_ERR_UNSUPPORTED
    assert e(ref, _lib.CF_F32, None, 10, 4096, 10, None) == _lib.CF_ERR_NULL
    assert e(ref, _lib.CF_F32, 256, 10, 4096, 9, None) == _lib.CF_ERR_SHAPE
    assert e(ref, _lib.CF_F32, 258, 10, 4096, 10, None) == _lib.CF_ERR_SHAPE
    assert m(ref, 256, 10, 256, 10, None, 256, 256, None) == _lib.CF_ERR_NULL
    assert m(ref, 256, -1, 256, 10, 256, 256, 256, None) == _lib.CF_ERR_SHAPE
    assert m(ctypes.byref(c_rules(n=0)), 256, 0, 256, 0, 256, 256, 256, None) == _lib.CF_ERR_SHAPE
    assert e(ctypes.byref(c_rules(n=0)), _lib.CF_F32, None, 0, None, 0, None) == _lib.CF_OK


def test_overlapping_rows_are_refused():
    S = _lib.CF_ERR_SHAPE
    # y within x, x within y, one element of both, for rows at one stride and at two
    for x, x_rs, y, y_rs in ((256, 16, 256, 32), (256, 16, 300, 32), (512, 16, 256, 32), (256, 48, 258, 48),
                             (256, 48, 256 + 30, 48), (256, 0, 286, 32), (256, 47, 256 + 32, 47)):
        assert call(c_layer(), x=x, x_rs=x_rs, y=y, y_rs=y_rs) == S, (x, x_rs, y, y_rs)
    e, ref = _lib.lib.cf_edit_logits, ctypes.byref(c_rules())
    for x, x_rs, y, y_rs in ((256, 10, 260, 10), (300, 10, 256, 10), (256, 0, 256, 10), (256, 12, 256, 10),
                             (256, 19, 296, 19)):
        assert e(ref, _lib.CF_F32, x, x_rs, y, y_rs, None) == S, (x, x_rs, y, y_rs)
    assert b"overlap" in _lib.lib.cf_last_error()


def test_rules_fault_injection(monkeypatch):
    ref = ctypes.byref(c_rules())
    monkeypatch.setenv("CF_FAULT", "edit_logits")
    assert _lib.lib.cf_edit_logits(ref, _lib.CF_F32, 256, 10, 4096, 10, None) == _lib.CF_ERR_INJECTED
    monkeypatch.setenv("CF_FAULT", "answer_margin")
    assert _lib.lib.cf_answer_margin(ref, 256, 10, 256, 10, 256, 256, 256, None) == _lib.CF_ERR_INJECTED


def test_cpu_tensors_are_refused():
    W, A, B = torch.zeros(4, 4), torch.zeros(1, 2, 4), torch.zeros(1, 4, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.AdapterLayer(W, A, B, torch.ones(1))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.AnswerRules(1, 4, allowed=torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.edit_logits(torch.zeros(1, 4), ops.AnswerRules(1, 4))
    with pytest.raises(NotImplementedError):
        ops.edit_logits(torch.zeros(1, 4, dtype=torch.float64), ops.AnswerRules(1, 4))


# ------------------------------------------------------------------------- the 64-bit forms
def test_oracle_adapter_is_the_merged_weight():
    g = torch.Generator()
    g.manual_seed(0)
    W, A, B = (torch.randn(*s, generator=g) for s in ((6, 5), (2, 3, 5), (2, 6, 3)))
    scale = torch.tensor([0.5, 2.0])
    for sub in (False, True):
        x = torch.randn(4, 6 if sub else 5, generator=g)
        y, tol = V.adapter(x, W, A, B, scale, [0, 1, 3, 4], [1, -1, 0], substitute=sub)
        for row, e in ((0, 1), (1, None), (2, None), (3, 0)):
            M = W.double() if e is None else W.double() + scale[e].double() * B[e].double() @ A[e].double()
            want = x[row].double() @ (M if sub else M.t())
            assert torch.allclose(y[row], want, rtol=1e-12, atol=1e-12)
        assert (tol > 0).all()
        with pytest.raises(AssertionError):
            V.check((y * 1.001).to(torch.float32), y, tol)


def test_oracle_substitute_is_the_input_gradient():
    """x W + s (x B) A is the gradient of <x, layer(z)> with respect to z: by differences, which
    are exact up to rounding for a linear layer."""
    g = torch.Generator()
    g.manual_seed(1)
    W, A, B = (torch.randn(*s, generator=g) for s in ((6, 5), (1, 3, 5), (1, 6, 3)))
    x, z = torch.randn(1, 6, generator=g), torch.randn(1, 5, generator=g)
    scale = torch.tensor([0.7])
    grad, _ = V.adapter(x, W, A, B, scale, [0, 1], [0], substitute=True)

    def value(z):
        return (x.double() * V.adapter(z, W, A, B, scale, [0, 1], [0])[0]).sum()
    for k in range(5):
        d = torch.zeros(1, 5, dtype=torch.float64)
        d[0, k] = 0.25
        diff = (value(z.double() + d) - value(z.double() - d)) / 0.5
        assert abs(float(diff - grad[0, k])) < 1e-12


def test_oracle_rules_by_hand():
    n = 4
    x = torch.tensor([[2.0, -2.0, 1.0, 5.0]])
    kw = dict(tokens=torch.tensor([0, 1, 1, 2], dtype=torch.int32), token_offsets=torch.tensor([0, 4]),
              prompt_len=torch.tensor([1], dtype=torch.int32), repetition=torch.tensor([2.0]),
              frequency=torch.tensor([0.5]), presence=torch.tensor([0.25]),
              bias_ids=torch.tensor([3, 3], dtype=torch.int32), bias_values=torch.tensor([9.0, 1.0]),
              bias_offsets=torch.tensor([0, 2]), allowed=V.pack(torch.tensor([[True, True, False, True]])))
    assert V.rules(x, n, **kw).tolist() == [[1.0, -4.0 - 1.0 - 0.25, -math.inf, 6.0]]
    m, j = V.margin(x, x, torch.tensor([3]), n, **kw)
    assert m.tolist() == [5.0] and j.tolist() == [0]


@pytest.mark.parametrize("sets", [0, 1, 3])
def test_a_row_without_a_set_of_its_own_is_refused(sets):
    """Without allowed_row, row r has set r: fewer sets than rows would leave rows without their mask."""
    with pytest.raises(Exception, match="SHAPE MISMATCH"):
        ops.AnswerRules(2, 4, allowed=torch.zeros(sets, 1, dtype=torch.int32))


def test_widths_that_an_int_cannot_step_past_are_refused():
    """The kernels step an int through the contraction, up to 2^16 past its end."""
    most = 2**31 - 2**16 - 1
    for n in (most + 1, 2**31 - 300, 2**31 - 256, 2**31 - 255, 2**31):
        assert call(c_layer(n_in=n, w_rs=n, a_rs=n, a_es=4 * n), x_rs=n, ws=1 << 40, wsb=1 << 50) == _lib.CF_ERR_SHAPE
        assert call(c_layer(n_out=n, b_es=4 * n), y=1 << 50, y_rs=n, ws=1 << 40, wsb=1 << 50) == _lib.CF_ERR_SHAPE
    # within the limits: the next check is the one that answers
    assert call(c_layer(n_in=most, w_rs=most, a_rs=most, a_es=4 * most), x_rs=most, y=1 << 50, wsb=0) == \
        _lib.CF_ERR_WORKSPACE


def test_unaligned_lists_are_refused():
    """A misaligned address would end the context."""
    S = _lib.CF_ERR_SHAPE
    for at in (257, 258, 260):
        assert call(c_layer(), off=at) == S
    for at in (257, 258):
        assert call(c_layer(), ids=at) == S
        assert call(c_layer(scale_dev=at)) == S
        assert call(c_layer(ranks_dev=at)) == S
    full = dict(tokens_dev=256, token_offsets_dev=256, prompt_len_dev=256, repetition_dev=256, frequency_dev=256,
                presence_dev=256, bias_ids_dev=256, bias_values_dev=256, bias_offsets_dev=256, allowed_dev=256,
                allowed_row_dev=256, n_tokens=4, n_biases=4, n_masks=1, allowed_words=1)
    for k in full:
        if k.endswith("_dev"):
            R = ctypes.byref(c_rules(**{**full, k: 260 if k.endswith("offsets_dev") else 258}))
            assert _lib.lib.cf_edit_logits(R, _lib.CF_F32, 256, 10, 4096, 10, None) == S, k
            assert _lib.lib.cf_answer_margin(R, 256, 10, 256, 10, 256, 256, 256, None) == S, k
    R = ctypes.byref(c_rules())
    for labels, margin, rival in ((260, 256, 256), (256, 258, 256), (256, 256, 257)):
        assert _lib.lib.cf_answer_margin(R, 256, 10, 256, 10, labels, margin, rival, None) == S


@pytest.mark.parametrize("substitute", [0, 1])
def test_ranks_beyond_a_grid_are_refused(substitute):
    rank = 65535 * 8 + 1
    L = c_layer(rank=rank, a_es=16 * rank, b_es=32 * rank, b_rs=rank)
    assert call(L, substitute, x_rs=32, ws=1 << 40, wsb=1 << 50, y=1 << 50) == _lib.CF_ERR_SHAPE
    assert b"rank" in _lib.lib.cf_last_error()
