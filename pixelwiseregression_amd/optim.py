"""The Muon optimizer on one flat fp32 parameter buffer: beside AdamW and SGD (`pwr_adamw_step` / `pwr_sgd_step`, train.py:139-142) the third
choice of ``TrainStep(opt=...)``.

    opt = Muon.for_model(model, lr=2e-3)          # or Muon(flat, shapes, ...)
    opt.step(model.flat_grad())

Matrices -- the conv kernels, one row per output channel -- take the orthogonalised momentum (``ops.orthogonalize``) scaled to the rms an AdamW
update has (``update_rms``, so one learning rate serves both); every other parameter takes an AdamW step.  All parameters of a network go through the
same few launches (eighteen; more where some of them are long), whatever their number and shapes.  A step that is captured into a graph keeps the
learning rate and the step number it was captured with.
"""
import ctypes

import torch

from . import _lib
from .ops import NS_COEFFICIENTS, _check_range, _on, _written


class _Param(ctypes.Structure):
    _fields_ = [("offset", ctypes.c_longlong), ("rows", ctypes.c_int), ("cols", ctypes.c_int)]


class Muon:
    """flat: the parameters, updated in place.  shapes: theirs, in their order in ``flat``.  buf, v: the state (momentum and first moments; second
    moments) where it exists already; ``steps`` counts the steps taken (AdamW's bias correction).  Gradients are all-reduced by the caller, if at all:
    equal gradients give equal updates on every rank, bit for bit."""

    def __init__(self, flat, shapes, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.0, update_rms=0.2, ns_steps=5,
                 coefficients=NS_COEFFICIENTS, eps=1e-7, beta1=0.9, beta2=0.999, adam_eps=1e-8, buf=None, v=None):
        shapes = [tuple(int(n) for n in s) for s in shapes]
        sizes = [int(torch.Size(s).numel()) for s in shapes]
        if sum(sizes) != flat.numel():
            raise ValueError("the shapes hold %d parameters, the buffer %d" % (sum(sizes), flat.numel()))
        self.flat = flat
        self._check(flat, "flat")
        if not 1 <= int(ns_steps) <= 64 or not float(eps) >= 0.0:
            raise ValueError("ns_steps must be 1 .. 64 and eps not negative, got %d, %g" % (ns_steps, eps))
        coefficients = tuple(float(c) for c in coefficients)
        if len(coefficients) != 3:
            raise ValueError("coefficients are (a, b, c)")
        self.lr, self.momentum, self.nesterov, self.weight_decay, self.update_rms = lr, momentum, nesterov, weight_decay, update_rms
        self.ns_steps, self.coefficients, self.eps = int(ns_steps), coefficients, eps
        self.beta1, self.beta2, self.adam_eps = beta1, beta2, adam_eps
        self.buf = torch.zeros_like(flat) if buf is None else self._check(buf, "buf")
        self.v = torch.zeros_like(flat) if v is None else self._check(v, "v")
        self.steps = 0
        params, at = [], 0
        for s, n in zip(shapes, sizes):
            if n:
                rows = s[0] if len(s) > 1 else 1
                if n >= 2 ** 31:
                    raise ValueError("a parameter of %d elements (2^31 at most)" % n)
                params.append((at, rows, n // rows))
            at += n
        if any(min(rows, cols) > 1 for _, rows, cols in params):
            _check_range(self.ns_steps, *self.coefficients)
        self._plan = self._ws = None
        if not params:
            return
        l = _lib.lib()
        arr = (_Param * len(params))(*params)
        need = l.pwr_muon_plan_bytes(arr, len(params))
        if need == 0:
            raise ValueError("a matrix is larger than the step takes (2^20 a side)")
        self._plan = ctypes.create_string_buffer(need)
        _lib.check(l.pwr_muon_plan(arr, len(params), self._plan), "pwr_muon_plan")
        self._plan_dev = torch.frombuffer(bytearray(self._plan.raw), dtype=torch.uint8).to(flat.device)
        self._ws = torch.empty(max(1, l.pwr_muon_workspace_bytes(self._plan)), device=flat.device, dtype=torch.uint8)

    @classmethod
    def for_model(cls, model, **kw):
        return cls(model.flat_parameters(), [shape for (_, shape) in model._offsets.values()], **kw)

    def _check(self, t, what):
        if not t.is_cuda:
            raise _lib.PwrError("Muon runs on the GPU only (%s is a %s tensor); there is no CPU fallback" % (what, t.device))
        if t.dtype != torch.float32 or t.dim() != 1 or not t.is_contiguous() or t.numel() != self.flat.numel() or t.device != self.flat.device:
            raise ValueError("%s must be a contiguous float32 vector of %d elements on %s" % (what, self.flat.numel(), self.flat.device))
        return t

    def step(self, grad, grad_scale=1.0):
        """One step with the flat gradient ``grad`` (multiplied by ``grad_scale`` first: 1 / world size after a SUM all-reduce)."""
        self._check(grad, "grad")
        self.steps += 1
        if self._plan is None:
            return
        a, b, c = self.coefficients
        with _on(self.flat.device):
            _lib.check(_lib.lib().pwr_muon_step(
                self._plan, self._plan_dev.data_ptr(), self.flat.data_ptr(), grad.data_ptr(), self.buf.data_ptr(), self.v.data_ptr(), self.lr,
                self.momentum, 1 if self.nesterov else 0, self.weight_decay, self.update_rms, self.ns_steps, a, b, c, self.eps, self.beta1, self.beta2,
                self.adam_eps, self.steps, grad_scale, self._ws.data_ptr(), self._ws.numel(), _lib.stream_ptr(self.flat.device)), "pwr_muon_step")
        _written(self.flat, self.buf, self.v)

    def state_dict(self):
        return {"buf": self.buf.clone(), "v": self.v.clone(), "steps": self.steps}

    def load_state_dict(self, state):
        if state["buf"].numel() != self.flat.numel() or state["v"].numel() != self.flat.numel():
            raise ValueError("the state of another parameter buffer")
        self.buf.copy_(state["buf"])
        self.v.copy_(state["v"])
        self.steps = int(state["steps"])
