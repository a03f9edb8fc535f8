"""torch.autograd bindings of individual HIP kernels (through the C ABI of include/pwr.h).

Only device tensors are accepted: there is no CPU implementation behind these ops by design.
"""
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib

HEATMAP_METHODS = {"softmax": 0, "sum": 1}


def _require_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise _lib.PwrError("pixelwiseregression_amd ops run on the GPU only (got a %s tensor); "
                                "there is no CPU fallback" % t.device)


def decode_forward(z, D, L, m, w, method):
    """Fused soft-argmax decoder forward (model.py:79-97 + 123-132). Returns (p, uvd)."""
    _require_cuda(z, D, L, m, w)
    B, J, P, P2 = z.shape
    assert P == P2 and D.shape == z.shape and L.shape == (B, 1, P, P) and m.shape == (B, 1, P, P)
    z, D, L, m = (t.contiguous().float() for t in (z, D, L, m))
    wv = w.contiguous().float().view(-1) if w is not None else None
    p = torch.empty_like(z)
    uvd = torch.empty(B, J, 3, device=z.device, dtype=torch.float32)
    l = _lib.lib()
    _lib.check(l.pwr_decode_fwd(_lib.ptr(z), _lib.ptr(D), _lib.ptr(L), _lib.ptr(m), _lib.ptr(wv), _lib.ptr(p),
                                _lib.ptr(uvd), B, J, P, HEATMAP_METHODS[method], _lib.stream_ptr(z.device)),
               "pwr_decode_fwd")
    return p, uvd


def decode_backward(p, z, D, L, m, w, uvd, gH, gD, gU, method):
    """Closed-form decoder backward. Returns (gz, gD_total, gw or None)."""
    _require_cuda(p, z, D, L, m, gU)
    B, J, P, _ = z.shape
    gz = torch.empty_like(z)
    gDo = torch.empty_like(z)
    wv = w.contiguous().float().view(-1) if w is not None else None
    gw_part = torch.empty(B * J, device=z.device, dtype=torch.float32) if w is not None else None
    gH = gH.contiguous().float() if gH is not None else None
    gD = gD.contiguous().float() if gD is not None else None
    gU = gU.contiguous().float()
    l = _lib.lib()
    s = _lib.stream_ptr(z.device)
    _lib.check(l.pwr_decode_bwd(_lib.ptr(p), _lib.ptr(z), _lib.ptr(D), _lib.ptr(L), _lib.ptr(m), _lib.ptr(wv),
                                _lib.ptr(uvd), _lib.ptr(gH), _lib.ptr(gD), _lib.ptr(gU), _lib.ptr(gz), _lib.ptr(gDo),
                                _lib.ptr(gw_part), B, J, P, HEATMAP_METHODS[method], s), "pwr_decode_bwd")
    gw = None
    if w is not None:
        gw = torch.empty(J, device=z.device, dtype=torch.float32)
        _lib.check(l.pwr_decode_gw_reduce(_lib.ptr(gw_part), _lib.ptr(gw), B, J, 0, s), "pwr_decode_gw_reduce")
        gw = gw.view_as(w)
    return gz, gDo, gw


class DecodeFn(torch.autograd.Function):
    """p, uvd = decode(z, D, L, m, w).  D's own gradient path (depth-map loss) stays in autograd;
    this node adds the decoder's contribution gd * p * m^2 / S."""

    @staticmethod
    def forward(ctx, z, D, L, m, w, method):
        z, D, L, m = (t.contiguous().float() for t in (z, D, L, m))
        p, uvd = decode_forward(z, D, L, m, w, method)
        ctx.method = method
        ctx.save_for_backward(p, z, D, L, m, w if w is not None else torch.empty(0, device=z.device), uvd)
        ctx.has_w = w is not None
        return p, uvd

    @staticmethod
    def backward(ctx, gp, guvd):
        p, z, D, L, m, w, uvd = ctx.saved_tensors
        w = w if ctx.has_w else None
        if guvd is None:
            guvd = torch.zeros_like(uvd)
        gz, gD, gw = decode_backward(p, z, D, L, m, w, uvd, gp, None, guvd, ctx.method)
        return gz, gD, None, None, gw, None


def decode(z, D, L, m, w, method="softmax"):
    return DecodeFn.apply(z, D, L, m, w, method)


class _on:
    """Launches go to the tensors' device, whichever is current."""

    def __init__(self, device):
        self.device = device if device.index not in (None, torch.cuda.current_device()) else None

    def __enter__(self):
        if self.device is not None:
            self.before = torch.cuda.current_device()
            torch.cuda.set_device(self.device)

    def __exit__(self, *a):
        if self.device is not None:
            torch.cuda.set_device(self.before)


_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_INT = 2 ** 31 - 1
_LONGEST_ROW = 2 ** 31 - 2 ** 14


def _dtype_tag(t, what):
    if t.dtype not in _DTYPES:
        raise ValueError("%s must be float32 or bfloat16, got %s" % (what, t.dtype))
    return _DTYPES[t.dtype]


def _tangents(*ts):
    """Whether one of them carries a forward-mode tangent (requires_grad says nothing of those)."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None for t in ts)


def _same_device(t, *others):
    for o in others:
        if o is not None and o.device != t.device:
            raise ValueError("tensors on %s and %s" % (t.device, o.device))


class LogLikelihood(NamedTuple):
    """What ``log_likelihood`` returns; ``top_logp`` / ``top_index`` are None without ``topk``."""
    logp: torch.Tensor
    entropy: torch.Tensor
    top_logp: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


def _plain(t, dtype):
    """t itself where it is what a kernel reads (a call of these small operators costs its Python), else a copy that is."""
    if t.dtype is dtype and t.is_contiguous():
        return t
    return t.detach().to(dtype).contiguous()


class _Rows:
    """The arguments of log_likelihood as the kernels take them: rows of V values, `ld` apart."""

    __slots__ = ("z", "ld", "index", "w", "mask", "mask_rows", "lead", "J", "rows", "V", "dtype")

    def __init__(self, z, index, w, mask):
        shape, dim = z.shape, z.dim()
        if not 2 <= dim <= 4:
            raise ValueError("z must be [N, V], [B, J, V] or [B, J, H, W], got %s" % (tuple(shape),))
        self.dtype = _dtype_tag(z, "z")
        self.lead = lead = tuple(shape[:1]) if dim == 2 else tuple(shape[:2])
        self.J = J = shape[1] if dim > 2 else 1
        self.rows, self.V = (lead[0] * J if dim > 2 else lead[0]), shape[-1] * shape[-2] if dim == 4 else shape[-1]
        if self.V < 1:
            raise ValueError("a row of no values")
        if J < 1:
            raise ValueError("no joints")
        if self.V > _LONGEST_ROW or J > _INT:            # (they cross the C ABI as int, which would cut them)
            raise ValueError("rows of %d values (2^31 - 2^14 at most), %d joints (2^31 - 1)" % (self.V, J))
        v = z.flatten(2) if dim == 4 else z
        if not v.is_contiguous():
            if (self.V > 1 and v.stride(-1) != 1) or (v.dim() == 3 and v.shape[0] > 1 and J > 1 and v.stride(0) != J * v.stride(1)):
                v = v.contiguous()
        self.z = v
        self.ld = v.stride(1) if v.dim() == 3 and J > 1 else v.stride(0)
        dev = z.device
        self.index = index
        if index is not None:
            if index.shape != lead or index.dtype not in _WHOLE:
                raise ValueError("index must be whole numbers of shape %s, got %s %s" % (lead, index.dtype, tuple(index.shape)))
            self.index = _plain(index, torch.int64)
            if index.device != dev:
                _same_device(z, index)
        self.w = w
        if w is not None:
            if w.numel() != J or not w.is_floating_point():
                raise ValueError("w must hold one number per joint (%d), got %s" % (J, tuple(w.shape)))
            self.w = _plain(w, torch.float32)
            if w.device != dev:
                _same_device(z, w)
        self.mask_rows = 1
        self.mask = mask
        if mask is not None:
            if dim == 4 and mask.dim() == 4 and mask.shape[2:] != shape[2:]:       # (as many pixels in other rows are no mask of these)
                raise ValueError("mask must be %s a map, got %s" % (tuple(shape[2:]), tuple(mask.shape)))
            m = mask.flatten(2) if dim == 4 and mask.dim() == 4 else mask
            if m.dtype is torch.float64:
                m = m != 0                                                         # (what float32 would round to 0 is allowed)
            if dim > 2 and m.shape == (lead[0], 1, self.V):
                self.mask_rows = J
            elif m.shape != lead + (self.V,):
                raise ValueError("mask must be %s or one per sample %s, got %s" % (lead + (self.V,), (lead[0], 1, self.V), tuple(mask.shape)))
            self.mask = _plain(m, torch.float32)
            if mask.device != dev:
                _same_device(z, mask)


_WHOLE = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _likelihood_forward(r, topk, stats):
    z, dev, lead = r.z, r.z.device, r.lead
    # (each result its own tensor: views of one buffer could not be changed in place, and would share a version)
    logp = torch.empty(lead, device=dev, dtype=torch.float32) if r.index is not None else None
    entropy = torch.empty(lead, device=dev, dtype=torch.float32) if logp is None else torch.empty_like(logp)
    top_logp = torch.empty(lead + (topk,), device=dev, dtype=torch.float32) if topk else None
    top_index = torch.empty(lead + (topk,), device=dev, dtype=torch.int64) if topk else None
    st = torch.empty((r.rows, 2), device=dev, dtype=torch.float32) if stats else None
    l = _lib.lib()
    need = l.pwr_likelihood_workspace_bytes(r.rows, r.V, topk) if r.V > 4096 else 0
    ws = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
    with _on(dev):
        _lib.check(l.pwr_likelihood_fwd(z.data_ptr(), r.ld, _ptr(r.w), r.J, _ptr(r.mask), r.mask_rows, _ptr(r.index), _ptr(logp), entropy.data_ptr(),
                                        _ptr(st), _ptr(top_logp), _ptr(top_index), r.rows, r.V, topk, r.dtype, _ptr(ws), need, _lib.stream_ptr(dev)),
                   "pwr_likelihood_fwd")
    return logp, entropy, top_logp, top_index, st


def _likelihood_backward(r, z, w, index, mask, stats, entropy, glogp, gentropy, need_w):
    """(r: the numbers; the tensors as r had them)"""
    dev = z.device
    gz = torch.empty(z.shape, device=dev, dtype=z.dtype)
    gw = torch.empty(r.J, device=dev, dtype=torch.float32) if need_w else None
    glogp, gentropy = (_plain(g, torch.float32) if g is not None else None for g in (glogp, gentropy))
    l = _lib.lib()
    need = l.pwr_likelihood_bwd_workspace_bytes(r.rows, r.V) if need_w else 0
    ws = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
    with _on(dev):
        _lib.check(l.pwr_likelihood_bwd(z.data_ptr(), r.ld, _ptr(w), r.J, _ptr(mask), r.mask_rows, _ptr(index), stats.data_ptr(),
                                        entropy.data_ptr(), _ptr(glogp), _ptr(gentropy), gz.data_ptr(), _ptr(gw), r.rows, r.V, r.dtype, _ptr(ws), need,
                                        _lib.stream_ptr(dev)), "pwr_likelihood_bwd")
    return gz, gw


class LogLikelihoodFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, w, index, mask, topk):
        r = _Rows(z, index, w, mask)
        logp, entropy, top_logp, top_index, stats = _likelihood_forward(r, topk, True)
        # The inputs, so that a change of one before the backward pass is noticed, and what the kernels read in their place: all of it saved, none held by
        # ctx, so that the backward pass frees it, whoever keeps a result.
        own = [t for t, given in ((r.z, z), (r.w, w), (r.index, index), (r.mask, mask)) if t is not given]
        if own:
            ctx.own = (r.z is not z, r.w is not w, r.index is not index, r.mask is not mask)
        ctx.save_for_backward(z, w, index, mask, stats, entropy, *own)
        r.z = r.w = r.index = r.mask = None
        ctx.r = r
        ctx.set_materialize_grads(False)
        if topk:
            ctx.mark_non_differentiable(top_logp, top_index)
        return logp, entropy, top_logp, top_index

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, glogp, gentropy, _, __):
        z, w, index, mask, stats, entropy, *own = ctx.saved_tensors
        if glogp is None and gentropy is None:
            return None, None, None, None, None
        need_z, need_w = ctx.needs_input_grad[:2]
        read = [z, w, index, mask]
        if own:
            read = [own.pop(0) if apart else t for t, apart in zip(read, ctx.own)]
        gz, gw = _likelihood_backward(ctx.r, *read, stats, entropy, glogp, gentropy, need_w)
        if gw is not None and (gw.shape != w.shape or gw.dtype != w.dtype):
            gw = gw.view(w.shape).to(w.dtype)
        return (gz if gz.shape == z.shape else gz.view(z.shape)) if need_z else None, gw, None, None, None


def log_likelihood(z, index, w=None, mask=None, topk=0):
    """Log likelihood of the pixel ``index`` under every heat map ``softmax(w z)`` -- the distribution ``decode`` reads its joint from
    (model.py:83-85) --, the map's entropy and its ``topk`` most likely pixels: a loss for the maps, and the confidence and the alternatives of a
    prediction.

    z: logits ``[B, J, H, W]``, ``[B, J, V]`` or ``[N, V]``, float32 or bfloat16.  index: ``[B, J]`` (``[N]``) whole numbers, -1 where no pixel is
    given (log likelihood 0, no gradient); a pixel outside its map gives NaN; None: no ``logp``.  w: one number per joint.  mask: ``[B, 1, H, W]``
    (one per sample) or one per map; 0 = not allowed, whatever z holds there.  A map has 2^31 - 2^14 pixels at most.  topk <= 32 (less for maps of over
    2^21 pixels): equal values go by the lowest index; what does not exist (masked, -inf, beyond the map) is ``(-inf, -1)``.  A map without an allowed
    pixel: -inf, entropy 0, zero gradient.

    Returns ``LogLikelihood(logp, entropy, top_logp, top_index)``, float32 (int64 the last); gradients of ``logp`` and ``entropy`` reach z and w
    (reverse mode; a forward-mode tangent is refused).
    In a captured graph: ``likelihood_gradients``, or forward and backward with no other autograd graph of the same leaves alive."""
    _require_cuda(z, index, w, mask)
    topk = int(topk)
    if not 0 <= topk <= 32:
        raise ValueError("topk must be 0 .. 32, got %d" % topk)
    if _tangents(z, w):
        raise NotImplementedError("log_likelihood has no forward-mode derivative")
    if torch.is_grad_enabled() and (z.requires_grad or (w is not None and w.requires_grad)):
        return LogLikelihood(*LogLikelihoodFn.apply(z, w, index, mask, topk))
    return LogLikelihood(*_likelihood_forward(_Rows(z, index, w, mask), topk, False)[:4])


def likelihood_gradients(z, index, w, glogp, gentropy, mask=None):
    """``log_likelihood(z, index, w, mask)`` and, without an autograd graph, the gradients of ``sum(glogp logp) + sum(gentropy entropy)`` with
    respect to z and w (float32 ``[J]``).  Returns ``(LogLikelihood, gz, gw)``; gw is None without w."""
    _require_cuda(z, index, w, glogp, gentropy, mask)
    if _tangents(z, w, glogp, gentropy):
        raise NotImplementedError("likelihood_gradients has no forward-mode derivative")
    with torch.no_grad():
        r = _Rows(z, index, w, mask)
        for g in (glogp, gentropy):
            if g is not None and tuple(g.shape) != r.lead:
                raise ValueError("an upstream gradient must be %s, got %s" % (r.lead, tuple(g.shape)))
        _same_device(z, glogp, gentropy)
        logp, entropy, _, _, stats = _likelihood_forward(r, 0, True)
        gz, gw = _likelihood_backward(r, r.z, r.w, r.index, r.mask, stats, entropy, glogp, gentropy, w is not None)
    return LogLikelihood(logp, entropy, None, None), gz.view(z.shape), gw


def heatmap_pixels(uvd, P):
    """The pixel (row-major index of a P x P map) nearest to each normalised joint ``uvd[..., :2]``, -1 where it lies outside: the inverse of the
    decoder's grid, u = (column - P // 2) / (P - 1) (utils.py:24-35)."""
    uv = torch.floor(uvd[..., :2].double() * (P - 1) + (P // 2) + 0.5)
    inside = ((uv >= 0) & (uv <= P - 1)).all(-1)          # (false for NaN)
    uv = torch.where(inside[..., None], uv, torch.zeros_like(uv)).long()
    return torch.where(inside, uv[..., 1] * P + uv[..., 0], torch.full_like(uv[..., 0], -1))


NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _overlap(s, t):
    """Whether the spans of memory of two tensors meet."""
    def span(u):
        return u.data_ptr(), u.data_ptr() + (1 + sum((n - 1) * k for n, k in zip(u.shape, u.stride()))) * u.element_size()
    (a, b), (c, d) = span(s), span(t)
    return s.numel() > 0 and t.numel() > 0 and s.device == t.device and a < d and c < b


def _check_range(steps, a, b, c):
    if _lib.lib().pwr_orthogonalize_range(steps, a, b, c) != 0:
        raise ValueError("coefficients (%g, %g, %g): in %d steps some matrix reaches entries of 16 and more, which the products cannot hold" % (a, b, c, steps))


def _written(*ts):
    """A kernel has written to them: a gradient that saved one before notices, as after an in-place operation."""
    torch.autograd.graph.increment_version([t for t in ts if not t.is_inference()])


def orthogonalize(x, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7, out=None):
    """The matrices ``x`` (``[..., rows, cols]``, float32 or bfloat16) made nearly orthogonal by ``steps`` Newton-Schulz products:
    ``X = x / (|x| + eps)``, then ``X = a X + (b A + c A A) X`` with ``A = X X^T`` (of the shorter side).  With the default coefficients every singular
    value above about 1e-3 of the norm ends up between 0.7 and 1.2.

    Precision, in norm.  Float32: that of float32 products, for entries of ``x / (|x| + eps)`` above 6e-5; smaller ones are kept to 2^-37, so a row of
    1e-5 times the others' size comes out right to 1e-4 of itself, and a matrix whose norm is 4e-4 eps to 4e-6.  Bfloat16: the products take 11 bits of
    each entry, and the result is off by 2.0 - 2.5e-3 where rounding it alone costs 1.7e-3; ``orthogonalize(x.float()).to(x.dtype)`` has float32 products.

    Other coefficients are taken as far as no entry of X, A or ``b A + c A A`` can reach 16 (``a I`` included): ValueError where some matrix would.

    Not differentiable (it is what an optimizer does to a gradient): a tensor that requires a gradient, or carries a forward-mode tangent, is refused."""
    _require_cuda(x, out)
    tag = _dtype_tag(x, "x")
    if x.dim() < 2:
        raise ValueError("x must be a matrix or a batch of them, got %s" % (tuple(x.shape),))
    if (torch.is_grad_enabled() and x.requires_grad) or _tangents(x, out):
        raise NotImplementedError("orthogonalize has no gradient: detach x")
    a, b, c = (float(t) for t in coefficients)
    steps = int(steps)
    if not 1 <= steps <= 64 or not float(eps) >= 0.0:
        raise ValueError("steps must be 1 .. 64 and eps not negative, got %d, %g" % (steps, eps))
    _check_range(steps, a, b, c)
    rows, cols = x.shape[-2:]
    if x.numel() and (max(rows, cols) > 2 ** 20 or rows * cols > _INT):      # (before they cross the C ABI as int, which would cut them)
        raise ValueError("matrices of %d x %d are larger than orthogonalize takes (2^20 a side, 2^31 - 1 entries)" % (rows, cols))
    given = out is not None
    if not given:
        out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    elif torch.is_grad_enabled() and out.requires_grad:
        raise NotImplementedError("orthogonalize has no gradient: detach out")
    elif out.shape != x.shape or out.dtype != x.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous %s tensor of shape %s" % (x.dtype, tuple(x.shape)))
    elif _overlap(x, out) and not (out.data_ptr() == x.data_ptr() and x.is_contiguous()):
        raise ValueError("out shares memory with x: it has to be x itself, contiguous, or apart from it")
    _same_device(x, out)
    if x.numel() == 0:
        return out
    v = x if x.dim() == 3 else x.reshape(-1, rows, cols)
    if (cols > 1 and v.stride(2) != 1) or (v is not x and v.data_ptr() != x.data_ptr()):
        v = v.contiguous()
    l = _lib.lib()
    need = l.pwr_orthogonalize_workspace_bytes(rows, cols, v.shape[0])
    ws = torch.empty(need, device=x.device, dtype=torch.uint8)
    with _on(x.device):
        _lib.check(l.pwr_orthogonalize(v.data_ptr(), v.stride(0), v.stride(1), out.data_ptr(), rows, cols, v.shape[0], tag, steps, a, b, c, float(eps),
                                       ws.data_ptr(), need, _lib.stream_ptr(x.device)), "pwr_orthogonalize")
    if given:
        _written(out)
    return out
