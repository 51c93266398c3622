"""Host side of the DeepPoly network driver: network upload + one call into libcfgpu.

``DeepPolyEngine`` mirrors what ``Flow(abs_elem, deeppoly(), network).flow()``
(constraintflow/lib/flow_sparse.py:27-228) computes.  For a chain network it runs the
whole layer loop inside ``cf_deeppoly_run``: one C-ABI call per batch of regions, all
work stream-ordered on the current torch stream.  Networks with Add / Concat layers (and
CROWN's all-crossing branch) run the general traversal of cfgpu.general over libcfgpu's
block kernels.  Torch only provides device memory and the stream handle.
"""
import ctypes
import math

import torch

from . import _lib
from ._lib import lib, check, CfLayer, CfNetwork

N_CLASSES = 10


class DeepPolyEngine:
    """A network resident on one GPU, ready to certify batches of input regions.

    layers: sequence of objects with ``kind`` in {'linear','conv','relu','add','concat'}
    and, for affine layers, ``W`` / ``b`` arrays (Linear W [out, in]; Conv W [Cout, Cin,
    k, k]) plus ``in_shape`` / ``out_shape`` / ``stride`` / ``pad`` for conv layers;
    optional ``parents`` (layer-list indices, -1 = the network input; default the previous
    layer), listed in the reference reader's order (every parent before its children).
    certifier: 'deeppoly' (deeppoly.cf, deeppoly_efficient.cf), 'crown' (crown.cf, whose
    ReLU branch is decided over the whole batch: a CROWN run always takes the batch in
    one workspace chunk and checks the device status; when a layer takes the all-crossing
    branch the bounds are recomputed by the general traversal of cfgpu.general), 'zono'
    (zono.cf, DeepZ: forward zonotope pass, linear chains), 'ibp' (ibp.cf: interval
    bounds) or 'crownibp' (crownibp.cf: interval bounds below the property, DeepPoly's
    ReLU relaxation from them, one backsubstitution of the property rows; chains).
    stop_depth: the custom-stop DeepPoly programs (deeppoly_custom_stop.cf, custom_stops/)
    with get_start = stop_depth: the traversal bounding a neuron of list layer m stops below
    layer m - stop_depth and concretises there with those neurons' own bounds (linear chains;
    None: every traversal reaches the input).  relu_strict: the lower ReLU slope is 1 where
    l + u > 0 (the relu_n of those programs and of zid.cf) instead of l + u >= 0; deeppoly
    and crownibp.
    adapters: {index of a linear layer: (A [E, rank, n_in], B [E, n_out, rank], scale [E][,
    ranks [E]])}: variants of the network that share its weights, W + scale[e] * B[e] @ A[e] in
    those layers (the same E everywhere).  run(..., adapter_ids=[B] int32) certifies every
    region for its own variant, in one batch; DeepPoly, through the general traversal.
    """

    def __init__(self, layers, input_size, device="cuda", n_spec=N_CLASSES - 1, certifier="deeppoly",
                 stop_depth=None, relu_strict=False, adapters=None):
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("DeepPolyEngine runs on a CUDA device only (no CPU fallback)")
        if self.device.index is None:          # tensors are on a device with an index
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.input_size = int(input_size)
        self.n_spec = int(n_spec)
        relax = {"deeppoly": _lib.CF_RELAX_DEEPPOLY, "crown": _lib.CF_RELAX_CROWN, "zono": _lib.CF_RELAX_ZONO,
                 "ibp": _lib.CF_RELAX_IBP, "crownibp": _lib.CF_RELAX_CROWNIBP}
        if certifier not in relax:
            raise NotImplementedError(f"certifier {certifier!r} (the driver runs deeppoly, crown, zono, ibp and "
                                      "crownibp)")
        self.certifier = certifier
        self.stop_depth = None
        self._keep = []
        self._general = []        # (kind, W, b, parents) device tensors for cfgpu.general
        widths = []
        descs = []
        self.chain = True
        for i, L in enumerate(layers):
            parents = tuple(int(p) for p in getattr(L, "parents", None) or (i - 1,))
            if any(not -1 <= p < i for p in parents):
                raise ValueError(f"layer {i}: parents {parents} must precede it in the list")
            pw = [self.input_size if p < 0 else widths[p] for p in parents]
            self.chain &= parents == (i - 1,)
            d = CfLayer()
            if L.kind in ("relu", "add", "concat"):
                if L.kind != "relu":
                    self.chain = False
                    if len(parents) != 2:
                        raise ValueError(f"layer {i}: {L.kind} takes two parents, got {parents}")
                    if L.kind == "add" and pw[0] != pw[1]:
                        raise ValueError(f"layer {i}: add of widths {pw}")
                d.kind = _lib.CF_LAYER_RELU
                d.n_in = d.n_out = sum(pw) if L.kind == "concat" else pw[0]
                self._general.append((L.kind, None, None, parents))
            else:
                W = torch.as_tensor(L.W, dtype=torch.float32).to(self.device).contiguous()
                b = torch.as_tensor(L.b, dtype=torch.float32).to(self.device).contiguous()
                self._keep += [W, b]
                d.W_dev, d.b_dev = W.data_ptr(), b.data_ptr()
                if L.kind == "linear":
                    d.kind = _lib.CF_LAYER_LINEAR
                    d.n_out, d.n_in = int(W.shape[0]), int(W.shape[1])
                elif L.kind == "conv":
                    d.kind = _lib.CF_LAYER_CONV
                    d.cout, d.cin, d.kh, d.kw = (int(x) for x in W.shape)
                    _, d.ih, d.iw = (int(x) for x in L.in_shape)
                    _, d.oh, d.ow = (int(x) for x in L.out_shape)
                    d.stride, d.pad = int(L.stride), int(L.pad)
                    d.n_in = d.cin * d.ih * d.iw
                    d.n_out = d.cout * d.oh * d.ow
                else:
                    raise NotImplementedError(f"layer kind {L.kind}")
                geom = ((d.cin, d.ih, d.iw, d.cout, d.oh, d.ow, d.stride, d.pad) if L.kind == "conv" else None)
                self._general.append((L.kind, W, b, parents, geom))
                if d.n_in != pw[0]:
                    raise ValueError(f"layer {i}: {L.kind} reads {d.n_in} neurons, its parent has {pw[0]}")
            widths.append(int(d.n_out))
            descs.append(d)
        self.n_last = widths[-1] if widths else self.input_size
        self.kinds = [g[0] for g in self._general]
        if self.chain:
            self._layers = (CfLayer * len(descs))(*descs)
            if stop_depth is not None and (certifier != "deeppoly" or int(stop_depth) < 0 or
                                           any(g[0] == "conv" for g in self._general)):
                raise NotImplementedError("a custom stop depth applies to the DeepPoly traversal of linear chains")
            self.stop_depth = None if stop_depth is None else int(stop_depth)
            code = relax[certifier]
            if relu_strict:
                strict = {"deeppoly": _lib.CF_RELAX_DEEPPOLY_STRICT, "crownibp": _lib.CF_RELAX_CROWNIBP_STRICT}
                if certifier not in strict:
                    raise NotImplementedError("the strict lower-slope test applies to DeepPoly's relaxation "
                                              "(deeppoly, crownibp)")
                code = strict[certifier]
            self.net = CfNetwork(len(descs), self._layers, self.input_size, self.n_spec, code,
                                 0 if stop_depth is None else int(stop_depth) + 1)
            self.N = int(lib.cf_network_neurons(ctypes.byref(self.net)))
            if self.N < 0:
                check(_lib.CF_ERR_SHAPE, "network description")
        else:
            # Add / Concat: polyexps mix layers; the general traversal runs the whole network
            if certifier not in ("deeppoly", "crown"):
                raise NotImplementedError(f"{certifier} on a network with Add / Concat layers (the forward "
                                          "drivers run chain networks)")
            if stop_depth is not None or relu_strict:
                raise NotImplementedError("a custom stop depth or strict ReLU test on a network with Add / Concat "
                                          "layers")
            self.net = None
            self.N = self.input_size + sum(widths) + self.n_spec
        self._adapters = self._adapter_layers(adapters, certifier, stop_depth, relu_strict) if adapters else {}
        self._ws = None
        self.graphs = True           # CUDA-graph replay of the general traversal (DeepPoly)
        self._graph_cache = {}
        self.replayed_launches = 0   # libcfgpu kernels replayed by those graphs

    def _adapter_layers(self, adapters, certifier, stop_depth, relu_strict):
        from . import ops
        if certifier != "deeppoly" or stop_depth is not None or relu_strict:
            raise NotImplementedError("adapters apply to the plain DeepPoly traversal")
        made = {}
        for idx, given in adapters.items():
            if not 0 <= idx < len(self._general) or self._general[idx][0] != "linear":
                raise NotImplementedError(f"adapters of layer {idx}: only linear layers carry them")
            A, B, scale, ranks = tuple(given) + (None,) * (4 - len(given))
            A, B, scale = (torch.as_tensor(t, dtype=torch.float32).to(self.device).contiguous() for t in (A, B, scale))
            if ranks is not None:
                ranks = torch.as_tensor(ranks, dtype=torch.int32).to(self.device).contiguous()
            made[idx] = ops.AdapterLayer(self._general[idx][1], A, B, scale, ranks)
        if len({layer.n_adapters for layer in made.values()}) > 1:
            raise ValueError("every adapted layer needs the same number of adapters")
        return made

    def workspace_bytes(self, chunk):
        if self.net is None:
            raise ValueError("the fused driver's workspace applies to chain networks only")
        return int(lib.cf_deeppoly_workspace_bytes(ctypes.byref(self.net), int(chunk)))

    def _workspace(self, B, budget_bytes):
        need_full = self.workspace_bytes(max(1, B))
        # CROWN needs the whole batch in one chunk; DeepPoly regions are independent
        need = need_full if self.certifier == "crown" else min(need_full, max(self.workspace_bytes(1), budget_bytes))
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        return self._ws

    # device bytes the fused driver's workspace may take; DeepPoly regions beyond what fits
    # run in further chunks of the same call
    workspace_budget = 8 << 30

    def run(self, l0, u0, spec_W, want_state=False, workspace_budget=None, out=None, check_device=False,
            replay=None, adapter_ids=None):
        """Bounds for B regions.

        l0, u0: [B, n_input] float32 device tensors (normalised input box);
        spec_W: [B, n_spec, n_last] float32 device tensor (property matrix).
        Returns (lb, ub) float64 [B, n_spec] and, if want_state, (state_l, state_u)
        float32 [B, N] with every neuron's bounds in the reference's neuron order.
        check_device=True synchronises and raises if a bounded device wait gave up (with adapter_ids: in
        any adapter_matmul on this device since the last check).
        replay=(dec_l, dec_u): [B, N] float32 device tensors (state layout) from which every
        ReLU branch decision is taken (cf_deeppoly_run_replay; DeepPoly chains only).
        """
        B = int(l0.shape[0])
        for t, shp in ((l0, (B, self.input_size)), (u0, (B, self.input_size)),
                       (spec_W, (B, self.n_spec, self.n_last))):
            if tuple(t.shape) != shp or t.dtype != torch.float32 or not t.is_contiguous() or t.device != self.device:
                raise Exception(f"SHAPE MISMATCH: expected contiguous float32 {shp} on {self.device}, "
                                f"got {tuple(t.shape)} {t.dtype} on {t.device}")
        if out is None:
            lb = torch.empty(B, self.n_spec, dtype=torch.float64, device=self.device)
            ub = torch.empty_like(lb)
        else:
            lb, ub = out
        sl = su = None
        if want_state:
            sl = torch.empty(B, self.N, dtype=torch.float32, device=self.device)
            su = torch.empty_like(sl)
        if adapter_ids is not None:
            if not self._adapters:
                raise ValueError("adapter_ids on an engine without adapters")
            if replay is not None:
                raise NotImplementedError("decision replay of adapted networks")
            if tuple(adapter_ids.shape) != (B,) or adapter_ids.dtype != torch.int32 or \
                    adapter_ids.device != self.device or not adapter_ids.is_contiguous():
                raise Exception(f"SHAPE MISMATCH: adapter_ids must be contiguous int32 {(B,)} on {self.device}")
        if self.net is None or adapter_ids is not None:
            self._general_run(l0, u0, spec_W, lb, ub, sl, su, adapter_ids)
            if check_device and adapter_ids is not None:
                from . import ops
                ops.adapter_check(self.device)
            if want_state:
                return lb, ub, sl, su
            return lb, ub
        ws = self._workspace(B, self.workspace_budget if workspace_budget is None else workspace_budget)
        stream = torch.cuda.current_stream(self.device).cuda_stream
        if replay is not None:
            dl, du = replay
            for t in (dl, du):
                if tuple(t.shape) != (B, self.N) or t.dtype != torch.float32 or not t.is_contiguous() or \
                        t.device != self.device:
                    raise Exception(f"SHAPE MISMATCH: replay bounds must be contiguous float32 {(B, self.N)}")
            st = lib.cf_deeppoly_run_replay(ctypes.byref(self.net), B, l0.data_ptr(), u0.data_ptr(),
                                            spec_W.data_ptr(), dl.data_ptr(), du.data_ptr(),
                                            sl.data_ptr() if sl is not None else None,
                                            su.data_ptr() if su is not None else None,
                                            lb.data_ptr(), ub.data_ptr(), ws.data_ptr(), ws.numel(), stream)
            check(st, "cf_deeppoly_run_replay")
        else:
            st = lib.cf_deeppoly_run(ctypes.byref(self.net), B, l0.data_ptr(), u0.data_ptr(), spec_W.data_ptr(),
                                     sl.data_ptr() if sl is not None else None,
                                     su.data_ptr() if su is not None else None,
                                     lb.data_ptr(), ub.data_ptr(), ws.data_ptr(), ws.numel(), stream)
            check(st, "cf_deeppoly_run")
        if self.certifier == "crown":
            st = lib.cf_deeppoly_check(ws.data_ptr(), stream)
            if st == _lib.CF_ERR_UNSUPPORTED:
                # a ReLU layer took the all-crossing branch: its polyexps mix layers
                self._general_run(l0, u0, spec_W, lb, ub, sl, su)
            else:
                check(st, "device status")
        elif check_device:
            check(lib.cf_deeppoly_check(ws.data_ptr(), stream), "device status")
        if want_state:
            return lb, ub, sl, su
        return lb, ub

    def _general_run(self, l0, u0, spec_W, lb, ub, state_l, state_u, adapter_ids=None):
        """Bounds through the general lowest-layer-first traversal (cfgpu.general) into lb, ub
        and, where they are not None, state_l, state_u.

        DeepPoly's traversal takes no data-dependent decision on the host, so for a given
        batch size its launches are captured once in a CUDA graph and replayed (the inputs
        are copied into the graph's buffers, which a call on another stream waits for); a call
        that is itself captured issues the launches into that graph.  CROWN decides its ReLU
        branches on the host and runs eagerly."""
        from . import general
        if self.certifier == "deeppoly" and self.graphs and not torch.cuda.is_current_stream_capturing():
            key = (int(l0.shape[0]), adapter_ids is not None)
            g = self._graph_cache.get(key)
            if g is None:
                g = self._capture(l0, u0, spec_W, adapter_ids, key)
            if g is not None:
                stream = torch.cuda.current_stream(self.device)
                stream.wait_event(g["done"])
                g["l0"].copy_(l0)
                g["u0"].copy_(u0)
                g["W"].copy_(spec_W)
                if adapter_ids is not None:
                    g["ids"].copy_(adapter_ids)
                g["graph"].replay()
                self.replayed_launches += g["launches"]
                lb.copy_(g["sl"][:, -self.n_spec:])
                ub.copy_(g["su"][:, -self.n_spec:])
                if state_l is not None:
                    state_l.copy_(g["sl"])
                    state_u.copy_(g["su"])
                g["done"].record(stream)
                return
        adapters = self._adapters if adapter_ids is not None else None
        bounds, _ = general.run(self._general, l0, u0, spec_W, self.certifier, adapters, adapter_ids)
        lb.copy_(bounds[-1][0])
        ub.copy_(bounds[-1][1])
        if state_l is not None:
            sl, su = general.state(l0, u0, bounds)
            state_l.copy_(sl)
            state_u.copy_(su)

    def _capture(self, l0, u0, spec_W, adapter_ids, key):
        from . import general
        static = {"l0": l0.clone(), "u0": u0.clone(), "W": spec_W.clone(),
                  "ids": None if adapter_ids is None else adapter_ids.clone(), "done": torch.cuda.Event()}
        variant = (self._adapters if adapter_ids is not None else None, static["ids"])
        try:
            side = torch.cuda.Stream(self.device)
            side.wait_stream(torch.cuda.current_stream(self.device))
            with torch.cuda.stream(side):      # warm-up outside the capture
                general.run(self._general, static["l0"], static["u0"], static["W"], "deeppoly", *variant)
            torch.cuda.current_stream(self.device).wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            from . import ops
            n0 = ops.LAUNCHES[0]
            with torch.cuda.graph(graph):
                bounds, _ = general.run(self._general, static["l0"], static["u0"], static["W"], "deeppoly", *variant)
                static["sl"], static["su"] = general.state(static["l0"], static["u0"], bounds)
        except RuntimeError:
            self.graphs = False                  # capture refused: run eagerly from now on
            return None
        static["graph"] = graph
        static["launches"] = ops.LAUNCHES[0] - n0
        self._graph_cache[key] = static
        return static

    def input_spec(self, X, y, eps, dataset):
        """Device input box and property matrix from device centres X [B,C,H,W] and labels y [B].

        Same arithmetic as constraintflow/lib/spec.py:21-72 (clip, normalise, e_label - e_k).
        """
        from .nets import MNIST_MEAN, MNIST_STD, CIFAR_MEAN, CIFAR_STD
        B = int(X.shape[0])
        C = int(X.shape[1])
        HW = int(X[0, 0].numel())
        mean, std = (MNIST_MEAN, MNIST_STD) if dataset == "mnist" else (CIFAR_MEAN, CIFAR_STD)
        if len(mean) == 1:
            mean, std = mean * C, std * C
        l0 = torch.empty(B, C * HW, dtype=torch.float32, device=self.device)
        u0 = torch.empty_like(l0)
        W = torch.empty(B, self.n_spec, self.n_spec + 1, dtype=torch.float32, device=self.device)
        stream = torch.cuda.current_stream(self.device).cuda_stream
        check(lib.cf_input_box(B, C, HW, X.data_ptr(), float(eps), _lib.f32_array(mean), _lib.f32_array(std),
                               l0.data_ptr(), u0.data_ptr(), stream), "cf_input_box")
        check(lib.cf_spec_matrix(B, self.n_spec + 1, y.data_ptr(), W.data_ptr(), stream), "cf_spec_matrix")
        return l0, u0, W

    def certify(self, X, y, eps, dataset, out=None):
        """Whole pipeline on device tensors: input box, property, certifier -> (lb, ub) float64."""
        l0, u0, W = self.input_spec(X, y, eps, dataset)
        lb, ub = self.run(l0, u0, W, out=out)
        return lb, ub

    def answer(self, l0, u0, labels, rules, adapter_ids=None, check_device=False):
        """Whether each region's answer under `rules` (ops.AnswerRules over the network's last
        layer) is its label: (margin [B] float32, rival [B] int32), margin > 0 certifies it
        (ops.answer_margin): ops.edit_logits of any float32 logits within the bounds then leaves
        the label above every other answer.  Without a repetition factor the rules add constants
        to a logit, and the margin is taken from the property rows' bounds of y[label] - y[j], less
        what the additions to logits of that size may round by; with one, from the bounds of the
        logits themselves.  labels [B] int64 device tensor of answers in 0 .. n_last-1.  The property
        rows take B (n_last - 1) n_last floats.  A margin proves as much as the certifier's bounds do:
        CROWN's and DeepZ's programs are not sound in every case.  check_device as in run: without
        it a margin may come from bounds that a device wait gave up on."""
        from . import ops
        B, n = int(l0.shape[0]), self.n_last
        if (rules.rows, rules.n) != (B, n) or self.n_spec != n - 1:
            raise Exception(f"SHAPE MISMATCH: rules for {rules.rows} rows of {rules.n} answers and {self.n_spec} "
                            f"property rows; {B} regions of {n} answers")
        if tuple(labels.shape) != (B,) or labels.dtype != torch.int64 or labels.device != self.device or \
                not labels.is_contiguous():
            raise Exception(f"SHAPE MISMATCH: labels must be contiguous int64 {(B,)} on {self.device}")
        W = torch.empty(B, n - 1, n, dtype=torch.float32, device=self.device)
        stream = torch.cuda.current_stream(self.device).cuda_stream
        check(lib.cf_spec_matrix(B, n, labels.data_ptr(), W.data_ptr(), stream), "cf_spec_matrix")
        edits = rules.launches > 1
        if not edits:
            lb, _ = self.run(l0, u0, W, adapter_ids=adapter_ids, check_device=check_device)
        else:
            lb, _, sl, su = self.run(l0, u0, W, want_state=True, adapter_ids=adapter_ids,
                                     check_device=check_device)
            at = self.N - self.n_spec - n
            l, u = sl[:, at:at + n], su[:, at:at + n]
            if rules.c.repetition_dev:
                return ops.answer_margin(l, u, labels, rules)
        # y[j] - y[label] <= -lb: upper bounds of the other answers relative to the label's 0
        row = torch.arange(n - 1, device=self.device)
        col = row + (row >= labels[:, None])
        low = lb.float()
        low = torch.where(low > lb, torch.nextafter(low, low.new_full((), -math.inf)), low)
        lo = torch.zeros(B, n, dtype=torch.float32, device=self.device)
        up = torch.zeros_like(lo).scatter_(1, col, ops.unary("neg", low, torch.float32))
        if edits:
            # Up to three additions round the edited logit, each by 2^-24 of at most |logit| + constants;
            # the same three, and the sum below, the edited difference: 8 * 2^-24 of all of them for both.
            # An infinite constant makes the logit infinite and rounds nothing.
            K = rules.constants(self.device)
            far = torch.maximum(l.abs(), u.abs()) + up.abs() + 4.0 * K
            slack = torch.where((K > 0) & (K < math.inf), 2.0**-21 * far, torch.zeros_like(K))
            lo, up = lo - slack, up + slack
        return ops.answer_margin(lo, up, labels, rules)


def profile_enable(on=True):
    check(lib.cf_profile_enable(1 if on else 0))


def profile_collect():
    st = _lib.CfProfileStats()
    check(lib.cf_profile_collect(ctypes.byref(st)), "cf_profile_collect")
    return dict(kernel_launches=st.kernel_launches, step_launches=st.step_launches, step_ms=st.step_ms,
                step_flops=st.step_flops, step_bytes=st.step_bytes, mem_launches=st.mem_launches,
                mem_ms=st.mem_ms, mem_bytes=st.mem_bytes)
