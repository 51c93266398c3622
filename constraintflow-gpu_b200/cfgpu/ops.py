"""Tensor-level wrappers over libcfgpu's block kernels (cf_ew_binary, cf_ew_unary,
cf_ew_where, cf_ew_clamp, cf_ew_any, cf_bmm, cf_conv_*), used by the gbcsr mirror
(constraintflow.gbcsr) and by the general traversal (cfgpu.general), and over the
operators for many variants of one network in a batch (cf_adapter_matmul,
cf_edit_logits, cf_answer_margin).

Operands are CUDA tensors, possibly broadcast views (zero strides); results are new
contiguous tensors.  PyTorch only allocates the memory and supplies the stream.
"""
import ctypes
import operator

import torch

from cfgpu import _lib

_OPS = {operator.add: "add", operator.sub: "sub", operator.mul: "mul", operator.truediv: "truediv",
        operator.ge: "ge", operator.gt: "gt", operator.le: "le", operator.lt: "lt", operator.eq: "eq",
        operator.ne: "ne", operator.and_: "and_", operator.or_: "or_"}
COMPARISONS = (operator.lt, operator.le, operator.eq, operator.ne, operator.gt, operator.ge, operator.and_,
               operator.or_)


# libcfgpu launches made through these wrappers (each wrapper launches one kernel); the
# engine uses it to count the launches a captured CUDA graph replays
LAUNCHES = [0]


def device():
    if not torch.cuda.is_available():
        raise RuntimeError("the gbcsr ops run on a CUDA device only (libcfgpu); no CPU fallback")
    return torch.device("cuda", torch.cuda.current_device())


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _dt(t):
    return _lib.CF_BOOL if t.dtype == torch.bool else _lib.CF_F32


def _geo(t):
    return _lib.i64_array(list(t.shape)), _lib.i64_array(list(t.stride()))


def as_block_tensor(x, dtype=None):
    """A block payload on the device: bool stays bool, every other dtype becomes float32."""
    t = torch.as_tensor(x)
    if dtype is None:
        dtype = torch.bool if t.dtype == torch.bool else torch.float32
    return t.to(device=device(), dtype=dtype)


def scalar_view(value, shape, dtype):
    """A fill value broadcast to `shape` without materialising it (all strides zero)."""
    t = torch.full((), value, dtype=dtype, device=device())   # a fill kernel: no host copy
    return t.expand(*shape) if len(shape) else t


def binary(op, a, b, out_dtype):
    assert a.shape == b.shape, (a.shape, b.shape)
    out = torch.empty(a.shape, dtype=out_dtype, device=a.device)
    if out.numel() == 0:
        return out
    shp, sa = _geo(a)
    _, sb = _geo(b)
    LAUNCHES[0] += 1
    st = _lib.lib.cf_ew_binary(_lib.OPS[_OPS[op]], a.dim(), shp, a.data_ptr(), _dt(a), sa, b.data_ptr(), _dt(b), sb,
                               out.data_ptr(), _dt(out), _stream())
    _lib.check(st, "cf_ew_binary")
    return out


def unary(name, a, out_dtype):
    out = torch.empty(a.shape, dtype=out_dtype, device=a.device)
    if out.numel() == 0:
        return out
    shp, sa = _geo(a)
    LAUNCHES[0] += 1
    st = _lib.lib.cf_ew_unary(_lib.UOPS[name], a.dim(), shp, a.data_ptr(), _dt(a), sa, out.data_ptr(), _dt(out),
                              _stream())
    _lib.check(st, "cf_ew_unary")
    return out


def where(c, y, z):
    out = torch.empty(c.shape, dtype=torch.float32, device=c.device)
    if out.numel() == 0:
        return out
    shp, sc = _geo(c)
    _, sy = _geo(y)
    _, sz = _geo(z)
    LAUNCHES[0] += 1
    st = _lib.lib.cf_ew_where(c.dim(), shp, c.data_ptr(), sc, y.data_ptr(), sy, z.data_ptr(), sz, out.data_ptr(),
                              _lib.CF_F32, _stream())
    _lib.check(st, "cf_ew_where")
    return out


def clamp(a, const, min_true):
    out = torch.empty(a.shape, dtype=torch.float32, device=a.device)
    if out.numel() == 0:
        return out
    shp, sa = _geo(a)
    LAUNCHES[0] += 1
    st = _lib.lib.cf_ew_clamp(a.dim(), shp, a.data_ptr(), sa, float(const), 1 if min_true else 0, out.data_ptr(),
                              _stream())
    _lib.check(st, "cf_ew_clamp")
    return out


def any_nonzero(a):
    if a.numel() == 0:
        return False
    flag = torch.zeros(1, dtype=torch.int32, device=a.device)
    shp, sa = _geo(a)
    LAUNCHES[0] += 1
    st = _lib.lib.cf_ew_any(a.dim(), shp, a.data_ptr(), _dt(a), sa, flag.data_ptr(), _stream())
    _lib.check(st, "cf_ew_any")
    return bool(flag.item())


def signscale(A, p, q, pc, qc):
    """out = A * (A >= 0 ? p : q) column-wise per batch, dc = sum_n A * (A >= 0 ? pc : qc).

    A [nb, M, N] with unit column stride; p, q, pc, qc [nb, N] contiguous (pc / qc may be
    None: 0).  Returns (out [nb, M, N], dc [nb, M])."""
    nb, M, N = A.shape
    if A.stride(2) != 1:
        A = A.contiguous()
    out = torch.empty(nb, M, N, dtype=torch.float32, device=A.device)
    dc = torch.empty(nb, M, dtype=torch.float32, device=A.device)
    vs = [v.contiguous() if v is not None else None for v in (p, q, pc, qc)]
    LAUNCHES[0] += 1
    st = _lib.lib.cf_signscale(nb, M, N, A.data_ptr(), A.stride(0), A.stride(1), vs[0].data_ptr(), vs[1].data_ptr(),
                               vs[2].data_ptr() if vs[2] is not None else None,
                               vs[3].data_ptr() if vs[3] is not None else None, N, out.data_ptr(), dc.data_ptr(),
                               _stream())
    _lib.check(st, "cf_signscale")
    return out, dc


def bmm(A, B, C=None, accumulate=False):
    """C[b] (+)= A[b] @ B[b]; A [nb, M, K], B [nb, K, N] strided views."""
    nb, M, K = A.shape
    N = B.shape[2]
    if C is None:
        C = torch.empty(nb, M, N, dtype=torch.float32, device=A.device)
    LAUNCHES[0] += 1
    st = _lib.lib.cf_bmm(nb, M, N, K, A.data_ptr(), A.stride(0), A.stride(1), A.stride(2), B.data_ptr(),
                         B.stride(0), B.stride(1), B.stride(2), C.data_ptr(), 1 if accumulate else 0, _stream())
    _lib.check(st, "cf_bmm")
    return C


# ---------------------------------------------------------------- gbcsr conv blocks
def conv_geom(K, C, ox, oy, ix, iy, kx, ky, sx, sy, px, py):
    """The geometry of a conv block (cf_conv_geom)."""
    return _lib.CfConvGeom(*[int(v) for v in (K, C, ox, oy, ix, iy, kx, ky, sx, sy, px, py)])


def conv_densify(g, nb, P, p_bs, p_ks, p_ps):
    """[nb, K*ox*oy, C*ix*iy]: the matrix a conv block stands for (cf_conv_densify)."""
    out = torch.empty(nb, g.K * g.ox * g.oy, g.C * g.ix * g.iy, dtype=torch.float32, device=P.device)
    LAUNCHES[0] += 1
    _lib.check(_lib.lib.cf_conv_densify(ctypes.byref(g), nb, P.data_ptr(), p_bs, p_ks, p_ps, out.data_ptr(),
                                        _stream()), "cf_conv_densify")
    return out


def conv_apply(g, nb, per_b, P, pstr, X, xstr, out, ostr):
    """out = M x for nb*per_b images (cf_conv_apply); pstr = (p_bs, p_ks, p_ps),
    xstr = (x_bs, x_ss, x_es), ostr = (o_bs, o_ss, o_rs) in elements."""
    LAUNCHES[0] += 1
    _lib.check(_lib.lib.cf_conv_apply(ctypes.byref(g), nb, per_b, P.data_ptr(), *pstr, X.data_ptr(), *xstr,
                                      out.data_ptr(), *ostr, _stream()), "cf_conv_apply")
    return out


def conv_scale(g, nb, P, pstr, X, x_bs, x_es):
    """[nb, K*ox*oy, C*kx*ky]: patch values times the input values under them (cf_conv_scale)."""
    out = torch.empty(nb, g.K * g.ox * g.oy, g.C * g.kx * g.ky, dtype=torch.float32, device=P.device)
    LAUNCHES[0] += 1
    _lib.check(_lib.lib.cf_conv_scale(ctypes.byref(g), nb, P.data_ptr(), *pstr, X.data_ptr(), x_bs, x_es,
                                      out.data_ptr(), _stream()), "cf_conv_scale")
    return out


def conv_transpose(g, nb, per_b, Y, ystr, W, OH, OW, out, ostr):
    """Transposed convolution of nb*per_b rows (cf_conv_transpose)."""
    LAUNCHES[0] += 1
    _lib.check(_lib.lib.cf_conv_transpose(ctypes.byref(g), nb, per_b, Y.data_ptr(), *ystr, W.data_ptr(), OH, OW,
                                          out.data_ptr(), *ostr, _stream()), "cf_conv_transpose")
    return out


# ------------------------------------------------- many variants of one network in a batch
_DTYPES = {torch.float32: _lib.CF_F32, torch.bfloat16: _lib.CF_BF16, torch.float16: _lib.CF_F16}


def _expect(name, t, dtype, shape, dev, strided=False):
    """Refuse a tensor that is not `dtype` on `dev` of `shape` (None: any size), its last
    dimension contiguous (strided) or all of them."""
    if t.dtype is dtype and t.device == dev:
        got = t.shape
        if got == shape or (len(got) == len(shape) and all(w is None or g == w for g, w in zip(got, shape))):
            if t.is_contiguous() or (strided and (t.stride(-1) == 1 or got[-1] <= 1)):
                return
    raise Exception(f"SHAPE MISMATCH: {name} must be {dtype} {tuple('any' if w is None else w for w in shape)} on "
                    f"{dev}{', its rows contiguous' if strided else ', contiguous'}; got {t.dtype} "
                    f"{tuple(t.shape)} with strides {t.stride()} on {t.device}")


def _cuda(name, t):
    if not t.is_cuda:
        raise RuntimeError(f"{name} is on {t.device}: libcfgpu runs on CUDA tensors only (no CPU fallback)")
    return t.device


def _ptr(t):
    return None if t is None else t.data_ptr()


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _plain(t, dtype, gpu, shape):
    """A contiguous tensor as expected; anything else goes through _expect, which says why not."""
    return t.dtype is dtype and t.get_device() == gpu and t.shape == shape and t.is_contiguous()


def _launch(gpu, fn, *args):
    """fn(*args, stream): a libcfgpu call on the current stream of that GPU, made the current device
    where it is not."""
    if gpu == torch._C._cuda_getDevice():
        return fn(*args, torch._C._cuda_getCurrentRawStream(gpu))
    with torch.cuda.device(gpu):
        return fn(*args, torch._C._cuda_getCurrentRawStream(gpu))


class AdapterLayer:
    """An affine layer with low-rank adapters, one of them for each request of a batch.

    W [n_out, n_in] (and bias [n_out]) are shared; adapter e adds scale[e] * B[e] @ A[e] to W,
    with A [n_adapters, rank, n_in], B [n_adapters, n_out, rank], scale [n_adapters] float32 and,
    optionally, ranks [n_adapters] int32, each adapter's own rank (what A and B hold beyond it
    is not used).  W, bias, A and B are of one dtype (float32, bfloat16, float16), on one GPU.
    The tensors are kept and read at every call: an adapter is exchanged by writing into them."""

    def __init__(self, W, A, B, scale, ranks=None, bias=None):
        dev = _cuda("W", W)
        dt = W.dtype
        if dt not in _DTYPES:
            raise NotImplementedError(f"adapters over {dt} weights (float32, bfloat16 and float16 are supported)")
        if W.dim() != 2 or A.dim() != 3:
            raise Exception(f"SHAPE MISMATCH: W {tuple(W.shape)} and A {tuple(A.shape)} are not [n_out, n_in] and "
                            "[n_adapters, rank, n_in]")
        self.n_out, self.n_in = int(W.shape[0]), int(W.shape[1])
        self.n_adapters, self.rank = int(A.shape[0]), int(A.shape[1])
        _expect("W", W, dt, (None, None), dev, strided=True)
        _expect("A", A, dt, (None, None, self.n_in), dev, strided=True)
        _expect("B", B, dt, (self.n_adapters, self.n_out, self.rank), dev, strided=True)
        _expect("scale", scale, torch.float32, (self.n_adapters,), dev)
        if ranks is not None:
            _expect("ranks", ranks, torch.int32, (self.n_adapters,), dev)
        if bias is not None:
            _expect("bias", bias, dt, (self.n_out,), dev)
        self.device, self.dtype, self.gpu = dev, dt, dev.index
        self.size = W.element_size()
        self._need = {}           # workspace bytes by sizes and alignment
        self._keep = (W, A, B, scale, ranks, bias)

        def strides(t):
            rs = t.stride(1) if t.shape[1] > 1 else t.shape[2]
            return (t.stride(0) if t.shape[0] > 1 else 0), max(rs, 0)
        a_es, a_rs = strides(A)
        b_es, b_rs = strides(B)
        self.c = _lib.CfAdapterLayer(_DTYPES[dt], self.n_adapters, self.rank, 0, self.n_out, self.n_in, W.data_ptr(),
                                     _row_stride(W), _ptr(bias), A.data_ptr(), a_es, a_rs, B.data_ptr(), b_es, b_rs,
                                     scale.data_ptr(), _ptr(ranks))
        self._ref = ctypes.byref(self.c)


def adapter_matmul(x, layer, offsets, ids, substitute=False, out=None):
    """Rows of many requests through `layer` (an AdapterLayer), each with its request's adapter.

    x [T, n_in] -> x @ W.T + bias + scale_e * (x @ A_e.T) @ B_e.T  [T, n_out]; or, with
    substitute, coefficient rows over the layer's outputs taken to its inputs (also the
    gradient with respect to the layer's input): x [T, n_out] -> x @ W + scale_e * (x @ B_e) @ A_e.
    offsets [n_requests + 1] int64: the rows of request q are offsets[q] .. offsets[q+1]-1;
    ids [n_requests] int32: its adapter, any value outside 0 .. n_adapters-1 none.  Both are
    read on the device, without a synchronisation.  Rows of no request are left as they were in
    `out`, and are 0 in a new result (filled first: a launch and a write more than with `out`).  `out`
    must not overlap x.  What meets an infinity comes out as an infinity or NaN, in rows of that
    request only.  No gradient is recorded: substitute gives the input's, those of the weights and
    adapters are the caller's products."""
    dev, gpu, dt = layer.device, layer.gpu, layer.dtype
    K, N = (layer.n_out, layer.n_in) if substitute else (layer.n_in, layer.n_out)
    if x.dim() == 2 and x.stride(1) != 1:
        x = x.contiguous()
    T, Q = x.shape[0], ids.shape[0]
    rs, out_rs = K, N
    if not _plain(x, dt, gpu, (T, K)):
        _expect("x", x, dt, (None, K), dev, strided=True)
        rs = _row_stride(x)
    if not _plain(offsets, torch.int64, gpu, (Q + 1,)):
        _expect("offsets", offsets, torch.int64, (Q + 1,), dev)
    if not _plain(ids, torch.int32, gpu, (Q,)):
        _expect("ids", ids, torch.int32, (None,), dev)
    if out is None:
        out = torch.zeros(T, N, dtype=dt, device=dev)
    elif not _plain(out, dt, gpu, (T, N)):
        _expect("out", out, dt, (T, N), dev, strided=True)
        out_rs = _row_stride(out)
    xp = x.data_ptr()
    key = (substitute, T, Q, xp % 16, rs)
    need = layer._need.get(key)
    if need is None:
        if len(layer._need) >= 4096:
            layer._need.clear()
        need = layer._need[key] = _lib.lib.cf_adapter_workspace_bytes(layer._ref, 1 if substitute else 0, T, xp, rs, Q)
    ws = x.new_empty(need // layer.size)
    LAUNCHES[0] += 1 + (need > 0)        # the adapters' part has a launch of its own
    st = _launch(gpu, _lib.lib.cf_adapter_matmul, layer._ref, 1 if substitute else 0, T, xp, rs, Q,
                 offsets.data_ptr(), ids.data_ptr(), out.data_ptr(), out_rs, ws.data_ptr(), need)
    if st:
        _lib.check(st, "cf_adapter_matmul")
    return out


def adapter_check(device=None):
    """Wait for the current stream and raise if a bounded device-side wait of an adapter_matmul
    on `device` gave up since the last check (its rows are not valid then)."""
    with torch.cuda.device(device):
        _lib.check(_lib.lib.cf_adapter_check(_stream()), "cf_adapter_check")


class AnswerRules:
    """The rule by which each of `rows` rows' answer is taken from its n logits.

    tokens [n_tokens] int32 with token_offsets [rows + 1] int64: the rows' histories, the first
    prompt_len [rows] int32 (default 0) tokens of each given, the rest answered; repetition,
    frequency, presence [rows] float32: the penalties (a repetition factor > 0);
    bias_ids [n_biases] int32, bias_values float32, bias_offsets [rows + 1] int64: biases, of an
    id given more than once the last; allowed [n_masks, words >= ceil(n / 32)] int32: sets of
    allowed answers, bit j % 32 of word j / 32 for answer j; allowed_row [rows] int32: the rows'
    sets, any value outside 0 .. n_masks-1 none (default: row r has set r).  The tensors are
    kept and read at every call.

        v = x;  j in the history: v = v / repetition if v > 0 else v * repetition
        answered c > 0 times:     v = v - frequency * c;  v = v - presence
        j has a bias:             v = v + bias;      j is not allowed: v = -inf
    """

    def __init__(self, rows, n, tokens=None, token_offsets=None, prompt_len=None, repetition=None, frequency=None,
                 presence=None, bias_ids=None, bias_values=None, bias_offsets=None, allowed=None, allowed_row=None):
        self.rows, self.n = int(rows), int(n)
        self.shape = (self.rows, self.n)
        given = dict(tokens=tokens, token_offsets=token_offsets, prompt_len=prompt_len, repetition=repetition,
                     frequency=frequency, presence=presence, bias_ids=bias_ids, bias_values=bias_values,
                     bias_offsets=bias_offsets, allowed=allowed, allowed_row=allowed_row)
        if allowed is not None and allowed_row is None and allowed.shape[:1] != (self.rows,):
            raise Exception(f"SHAPE MISMATCH: {tuple(allowed.shape)} sets for {self.rows} rows without allowed_row")
        first = next(((k, t) for k, t in given.items() if t is not None), None)
        self.device = _cuda(*first) if first else None
        i32, i64, f32 = torch.int32, torch.int64, torch.float32
        shapes = dict(tokens=(i32, (None,)), token_offsets=(i64, (self.rows + 1,)), prompt_len=(i32, (self.rows,)),
                      repetition=(f32, (self.rows,)), frequency=(f32, (self.rows,)), presence=(f32, (self.rows,)),
                      bias_ids=(i32, (None,)), bias_values=(f32, (None,)), bias_offsets=(i64, (self.rows + 1,)),
                      allowed=(i32, (None, None)), allowed_row=(i32, (self.rows,)))
        for k, t in given.items():
            if t is not None:
                _expect(k, t, shapes[k][0], shapes[k][1], self.device)
        if bias_ids is not None and bias_values is not None and bias_ids.shape != bias_values.shape:
            raise Exception(f"SHAPE MISMATCH: {tuple(bias_ids.shape)} bias ids, {tuple(bias_values.shape)} values")
        self._keep = given
        # an empty list has no storage of its own: nothing is in it, offsets and all
        if tokens is not None and tokens.numel() == 0:
            given = {k: None if k in ("tokens", "token_offsets", "prompt_len", "repetition", "frequency", "presence")
                     else t for k, t in given.items()}
        if allowed is not None and allowed.shape[0] == 0:
            given = {k: None if k.startswith("allowed") else t for k, t in given.items()}
        if bias_ids is not None and bias_ids.numel() == 0:
            given = {k: None if k.startswith("bias_") else t for k, t in given.items()}
        count = {k: 0 if given[k] is None else int(given[k].shape[0]) for k in ("tokens", "bias_ids", "allowed")}
        self.c = _lib.CfAnswerRules(self.rows, self.n, count["tokens"], count["bias_ids"],
                                    0 if allowed is None else int(allowed.shape[1]), count["allowed"], 0,
                                    *[_ptr(t) for t in given.values()])
        self._ref = ctypes.byref(self.c)
        self.launches = 1 + (count["tokens"] + count["bias_ids"] > 0)   # the stream, the edits

    def constants(self, device):
        """[rows, n] float32: a quarter of the sum of the magnitudes of what the penalties and the
        biases add to each logit, 0 where nothing is added, infinite only where a constant is."""
        k = self._keep

        def quarter(t, sign):
            return None if t is None else torch.where(t == 0, 0.0, sign * (0.25 * t.abs() + 1e-38))
        added = AnswerRules(self.rows, self.n, k["tokens"], k["token_offsets"], k["prompt_len"],
                            frequency=quarter(k["frequency"], -1.0), presence=quarter(k["presence"], -1.0),
                            bias_ids=k["bias_ids"], bias_values=quarter(k["bias_values"], 1.0),
                            bias_offsets=k["bias_offsets"])
        return edit_logits(torch.zeros(self.rows, self.n, dtype=torch.float32, device=device), added)


def _rules_rows(name, t, rules, dtype, gpu):
    """(t, its row stride) as rows for the rules: [rows, n] of `dtype` on `gpu`, its last dimension
    contiguous."""
    if rules.device is not None and gpu != rules.device.index:
        raise Exception(f"SHAPE MISMATCH: {name} is on GPU {gpu}, the rules are on {rules.device}")
    if _plain(t, dtype, gpu, rules.shape):
        return t, rules.n
    if t.dim() == 2 and t.stride(1) != 1:
        t = t.contiguous()
    _expect(name, t, dtype, rules.shape, torch.device("cuda", gpu), strided=True)
    return t, _row_stride(t)


def edit_logits(logits, rules, out=None):
    """The rules applied to logits [rows, n] (float32, bfloat16, float16), in float32, rounded
    once to the logits' dtype; `out` may be the logits themselves.  No gradient is recorded."""
    dt = logits.dtype
    if dt not in _DTYPES:
        raise NotImplementedError(f"logits of {dt} (float32, bfloat16 and float16 are supported)")
    gpu = _cuda("logits", logits).index
    x, rs = _rules_rows("logits", logits, rules, dt, gpu)
    out_rs = rules.n
    if out is None:
        out = torch.empty(rules.rows, rules.n, dtype=dt, device=x.device)
    elif not _plain(out, dt, gpu, rules.shape):
        _expect("out", out, dt, rules.shape, x.device, strided=True)
        out_rs = _row_stride(out)
    LAUNCHES[0] += rules.launches
    st = _launch(gpu, _lib.lib.cf_edit_logits, rules._ref, _DTYPES[dt], x.data_ptr(), rs, out.data_ptr(), out_rs)
    if st:
        _lib.check(st, "cf_edit_logits")
    return out


def answer_margin(l, u, labels, rules):
    """How far labels [rows] (int64) are certified under the rules: l, u [rows, n] float32
    bounds of the logits.  Returns margin [rows] float32, the label's edited lower bound less
    the best edited upper bound among the other answers (> 0: the answer is the label), and
    rival [rows] int32, that other answer (the lowest on equal bounds, -1: none is left).
    A label that is not allowed has margin -inf; a bound that is NaN bounds nothing."""
    dev = _cuda("l", l)
    gpu = dev.index
    l, l_rs = _rules_rows("l", l, rules, torch.float32, gpu)
    u, u_rs = _rules_rows("u", u, rules, torch.float32, gpu)
    if not _plain(labels, torch.int64, gpu, (rules.rows,)):
        _expect("labels", labels, torch.int64, (rules.rows,), dev)
    margin, rival = l.new_empty(rules.rows), l.new_empty(rules.rows, dtype=torch.int32)
    LAUNCHES[0] += 1
    st = _launch(gpu, _lib.lib.cf_answer_margin, rules._ref, l.data_ptr(), l_rs, u.data_ptr(), u_rs,
                 labels.data_ptr(), margin.data_ptr(), rival.data_ptr())
    if st:
        _lib.check(st, "cf_answer_margin")
    return margin, rival
