"""Operator-level mirror of the reference's native seam `models/StyleGAN2/op` (op/__init__.py:1-2):
`FusedLeakyReLU`, `fused_leaky_relu`, `upfirdn2d` — same names, arguments and autograd behaviour,
backed by the C ABI (wgs_bias_act / wgs_upfirdn2d) instead of the JIT-built CUDA extension.

Beside it, the operators that close a training step: `label_logprobs` (log-probabilities of given labels, entropy, top alternatives, and
their gradient), `orthogonalise` (orthogonal factor of an update) and `muon_step` (momentum, orthogonalisation, weight update).
"""
import collections
import contextlib
import ctypes
import struct

import torch
from torch import nn

from . import _lib as L


def fused_bias_act(x, bias=None, ref=None, act=3, grad=0, alpha=0.2, scale=2 ** 0.5):
    """fused.fused_bias_act(input, bias, refer, act, grad, alpha, scale) -> Tensor
    (models/StyleGAN2/op/fused_bias_act.cpp:11-21): bias indexed on dim 1, output allocated here."""
    x = x.contiguous()
    y = torch.empty_like(x)
    step_b = 1
    for s in x.shape[2:]:
        step_b *= s
    has_b = bias is not None and bias.numel() > 0
    has_r = ref is not None and ref.numel() > 0
    # hold every (possibly re-laid-out) operand in a local until the launch has been issued
    bias_c = bias.contiguous() if has_b else None
    ref_c = ref.contiguous() if has_r else None
    L.check(L.lib().wgs_bias_act(L.ptr(x), L.ptr(bias_c), L.ptr(ref_c), L.ptr(y), act, grad,
                                 L.c_float(alpha), L.c_float(scale), L.c_int64(x.numel()), step_b,
                                 bias.numel() if has_b else 1, L.stream()), 'wgs_bias_act')
    return y


class _FusedLeakyReLU(torch.autograd.Function):
    """FusedLeakyReLUFunction (op/fused_act.py:51-70): backward gated on the saved OUTPUT."""

    @staticmethod
    def forward(ctx, x, bias, negative_slope, scale):
        out = fused_bias_act(x, bias, None, 3, 0, negative_slope, scale)
        ctx.save_for_backward(out)
        ctx.cfg = (negative_slope, scale)
        return out

    @staticmethod
    def backward(ctx, gout):
        out, = ctx.saved_tensors
        negative_slope, scale = ctx.cfg
        gin = fused_bias_act(gout, None, out, 3, 1, negative_slope, scale)
        dims = [0] + list(range(2, gin.ndim))
        return gin, gin.sum(dims), None, None


def fused_leaky_relu(x, bias, negative_slope=0.2, scale=2 ** 0.5):
    return _FusedLeakyReLU.apply(x, bias, negative_slope, scale)


class FusedLeakyReLU(nn.Module):
    def __init__(self, channel, negative_slope=0.2, scale=2 ** 0.5):
        super().__init__()
        self.bias = nn.Parameter(torch.zeros(channel))
        self.negative_slope = negative_slope
        self.scale = scale

    def forward(self, x):
        return fused_leaky_relu(x, self.bias, self.negative_slope, self.scale)


def upfirdn2d_mhwc(x, kernel, up_x, up_y, down_x, down_y, pad_x0, pad_x1, pad_y0, pad_y1):
    """upfirdn2d_op.upfirdn2d(input[major,h,w,minor], kernel, ...) (op/upfirdn2d.cpp:12-23)."""
    x = x.contiguous()
    major, in_h, in_w, minor = x.shape
    kh, kw = kernel.shape
    out_h = (in_h * up_y + pad_y0 + pad_y1 - kh) // down_y + 1
    out_w = (in_w * up_x + pad_x0 + pad_x1 - kw) // down_x + 1
    y = torch.empty(major, out_h, out_w, minor, dtype=x.dtype, device=x.device)
    kernel_c = kernel.contiguous()
    L.check(L.lib().wgs_upfirdn2d(L.ptr(x), L.ptr(kernel_c), L.ptr(y), major, in_h, in_w, minor, kh, kw,
                                  up_x, up_y, down_x, down_y, pad_x0, pad_x1, pad_y0, pad_y1, L.stream()),
            'wgs_upfirdn2d')
    return y


class _UpFirDn2d(torch.autograd.Function):
    """UpFirDn2d (op/upfirdn2d.py:87-141): backward = the same op with up<->down swapped, the flipped
    kernel and the g_pad of :110-115."""

    @staticmethod
    def forward(ctx, x, kernel, up, down, pad):
        up_x, up_y = up
        down_x, down_y = down
        px0, px1, py0, py1 = pad
        kh, kw = kernel.shape
        b, c, in_h, in_w = x.shape
        out = upfirdn2d_mhwc(x.reshape(-1, in_h, in_w, 1), kernel, up_x, up_y, down_x, down_y, px0, px1, py0, py1)
        out_h, out_w = out.shape[1], out.shape[2]
        ctx.save_for_backward(torch.flip(kernel, [0, 1]))
        ctx.cfg = (up, down, (b, c, in_h, in_w), (out_h, out_w),
                   (kw - px0 - 1, in_w * up_x - out_w * down_x + px0 - up_x + 1,
                    kh - py0 - 1, in_h * up_y - out_h * down_y + py0 - up_y + 1))
        return out.view(b, c, out_h, out_w)

    @staticmethod
    def backward(ctx, gout):
        gkernel, = ctx.saved_tensors
        (up_x, up_y), (down_x, down_y), in_size, (out_h, out_w), (gx0, gx1, gy0, gy1) = ctx.cfg
        gin = upfirdn2d_mhwc(gout.reshape(-1, out_h, out_w, 1), gkernel, down_x, down_y, up_x, up_y, gx0, gx1, gy0, gy1)
        return gin.view(in_size), None, None, None, None


def upfirdn2d(x, kernel, up=1, down=1, pad=(0, 0)):
    return _UpFirDn2d.apply(x, kernel, (up, up), (down, down), (pad[0], pad[1], pad[0], pad[1]))


# ---- operators of the training objective -------------------------------------------------------------------------------------------
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # WGS_F32 / WGS_BF16 / WGS_F16
_HERE = contextlib.nullcontext()


def _on(device):
    """Context in which launches go to `device`'s current stream, whatever the current device is."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


LabelLogprobs = collections.namedtuple('LabelLogprobs', 'logp entropy top_logp top_index')
TOP_MAX = 64


def _rows_of(x):
    """(x viewed or copied as [rows, V] with adjacent scores and rows that do not overlap, row stride in elements)."""
    V = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(-1, V)
    if (V > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < V):
        x = x.contiguous()
    return x, (x.stride(0) if x.shape[0] > 1 else V)


_P, _I, _I64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
_logprob_calls = None


def _logprobs():
    """(workspace, forward, backward) entry points with their argument types: plain integers go in without a conversion object each."""
    global _logprob_calls
    if _logprob_calls is None:
        lib = L.lib()
        ws, fwd, bwd = lib.wgs_label_logprobs_ws_bytes, lib.wgs_label_logprobs_fwd, lib.wgs_label_logprobs_bwd
        ws.argtypes = [_I64, _I64, _I]
        fwd.argtypes = [_P, _I, _I64, _I64, _I64, _P, _I64, _I, _P, _P, _P, _P, _P, _P, _I64, _P]
        bwd.argtypes = [_P, _I, _I64, _I64, _I64, _P, _I64, _P, _P, _I, _P, _P, _P, _P, _P, _I64, _P]
        _logprob_calls = ws, fwd, bwd
    return _logprob_calls


def _upstream(g):
    return g if g is None or (g.dtype == torch.float32 and g.is_contiguous()) else g.to(torch.float32).contiguous()


class _LabelLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, top, ignore_index):
        dev, V = logits.device, logits.shape[-1]
        x, stride = _rows_of(logits)
        rows = x.shape[0]
        code = _DTYPES[x.dtype]
        lead = logits.shape[:-1]
        ws_bytes, fwd, _ = _logprobs()
        with _on(dev):
            logp = torch.empty(lead, device=dev)
            entropy = torch.empty(lead, device=dev)
            stat = torch.empty(rows, 2, device=dev)
            top_logp = torch.empty(lead + (top,), device=dev)
            top_index = torch.empty(lead + (top,), dtype=torch.int64, device=dev)
            need = ws_bytes(rows, V, top)
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
            L.check(fwd(x.data_ptr(), code, rows, V, stride, labels.data_ptr(), ignore_index, top, logp.data_ptr(), entropy.data_ptr(), stat.data_ptr(),
                        top_logp.data_ptr(), top_index.data_ptr(), ws.data_ptr() if need else None, need, L.stream_id()), 'wgs_label_logprobs_fwd')
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_index)
        # (a copy made of a strided input is saved in its place)
        ctx.save_for_backward(x if x.data_ptr() != logits.data_ptr() else logits, labels, stat, entropy, top_index)
        ctx.cfg = (top, ignore_index, logits.shape)
        return logp, entropy, top_logp, top_index

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logp, g_entropy, g_top, _):
        logits, labels, stat, entropy, top_index = ctx.saved_tensors
        top, ignore_index, shape = ctx.cfg
        dev, V = logits.device, shape[-1]
        x, stride = _rows_of(logits)
        rows, size = x.shape[0], x.element_size()
        with _on(dev):
            g_logp, g_entropy, g_top = _upstream(g_logp), _upstream(g_entropy), _upstream(g_top)
            # rows of the gradient start at the same place of a 16-byte block as those of the logits: whole-vector reads and writes
            first = x.data_ptr() % 16 // size
            gstride = V + (stride - V) % (16 // size) if rows > 1 else V
            if first == 0 and gstride == V:
                grad = torch.empty(shape, dtype=x.dtype, device=dev)
            else:
                grad = torch.empty(first + rows * gstride, dtype=x.dtype, device=dev)[first:].view(rows, gstride)[:, :V]
            L.check(_logprobs()[2](x.data_ptr(), _DTYPES[x.dtype], rows, V, stride, labels.data_ptr(), ignore_index, stat.data_ptr(), entropy.data_ptr(),
                                   top, top_index.data_ptr(), None if g_logp is None else g_logp.data_ptr(),
                                   None if g_entropy is None else g_entropy.data_ptr(), None if g_top is None else g_top.data_ptr(),
                                   grad.data_ptr(), gstride, L.stream_id()), 'wgs_label_logprobs_bwd')
        return (grad if grad.shape == shape else grad.reshape(shape)), None, None, None


def label_logprobs(logits, labels, top=0, ignore_index=-100):
    """Log-probability of each row's label under softmax(logits), the entropy of the row, and its `top` most likely classes.

    logits [..., V] (float32 / bfloat16 / float16, any strides), labels [...] int64.  Rows with adjacent scores that are equally far apart are read in
    place; others are copied first, a slice of positions logits[:, :-1] of [B, S, V] too (its rows have two strides).
    -> LabelLogprobs(logp [...], entropy [...], top_logp [..., top], top_index [..., top]): float32, int64 indices, equal scores in the order
    of their indices.  A label equal to ignore_index has logp 0 and passes no gradient; one that is no class otherwise gives NaN.  Rows of
    nothing but -inf: logp -inf, entropy 0, gradient 0; rows with a NaN or +inf: NaN, top_index -1.  top <= 64.
    Differentiable in logp, entropy and top_logp (the loss and the statistics of lib/trainer.py:245-258 are made of them).  Both directions can be captured
    into a graph; as with any operator of PyTorch, no eager graph of the same leaves may be alive while their backward is captured."""
    if not logits.is_cuda:
        raise L.WgsError("logits must be a GPU tensor (the HIP path has no CPU fallback)")
    if logits.dtype not in _DTYPES:
        raise L.WgsError("logits must be float32, bfloat16 or float16, got %s" % logits.dtype)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise L.WgsError("logits must have at least one class, got shape %s" % (tuple(logits.shape),))
    if labels.dtype != torch.int64 or labels.device != logits.device or labels.shape != logits.shape[:-1]:
        raise L.WgsError("labels must be int64 of shape %s on %s, got %s %s on %s" % (
            tuple(logits.shape[:-1]), logits.device, labels.dtype, tuple(labels.shape), labels.device))
    if not 0 <= top <= min(TOP_MAX, logits.shape[-1]):
        raise L.WgsError("top must be 0 .. %d (and at most the number of classes), got %d" % (TOP_MAX, top))
    return LabelLogprobs(*_LabelLogprobsFn.apply(logits, labels.contiguous(), int(top), int(ignore_index)))


NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)      # the quintic whose iterates take singular values of (0, 1] to about 1 in five steps
_MATRIX = struct.Struct('=3Q4q3i2fi')            # wgs_matrix of include/wgs.h


def _run_matrices(entries, ws_bytes, call, dtype, device, steps):
    """entries: packed wgs_matrix fields of every matrix; call(mats, count, dtype code, workspace, its bytes)."""
    n = len(entries)
    mats = ctypes.create_string_buffer(_MATRIX.size * n)
    for i, e in enumerate(entries):
        _MATRIX.pack_into(mats, i * _MATRIX.size, *e)
    code = _DTYPES[dtype]
    with _on(device):
        need = ws_bytes(mats, n, code, steps)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        call(mats, n, code, L.rawptr(ws), L.c_int64(need))


def _as_rows(x):
    """[batch, M, N] view (or copy) of x [..., M, N] with adjacent elements in a row."""
    M, N = x.shape[-2:]
    y = x if x.dim() == 3 else x.reshape(-1, M, N)
    b, r, c = y.stride()
    if (N > 1 and c != 1) or (M > 1 and r < N) or (y.shape[0] > 1 and b < 0):
        y = y.contiguous()
    return y


def _strides(y):
    """(batch stride, row stride) of a [batch, M, N] tensor, as the kernels want them where a dimension has one entry."""
    _, M, N = y.shape
    r = y.stride(1) if M > 1 else N
    return (y.stride(0) if y.shape[0] > 1 else M * r), r


def _joined(n):
    """wgs_matrix.joined of an argument: None goes by the result's type."""
    if n is None:
        return 0
    if not 1 <= int(n) <= 16:
        raise L.WgsError("joined must be None or 1 .. 16, got %s" % (n,))
    return int(n)


def _check_matrix(x, what, device=None, dtype=None):
    if not x.is_cuda:
        raise L.WgsError("%s must be a GPU tensor (the HIP path has no CPU fallback)" % what)
    if x.dtype not in _DTYPES:
        raise L.WgsError("%s must be float32, bfloat16 or float16, got %s" % (what, x.dtype))
    if x.dim() < 2 or x.shape[-1] < 1 or x.shape[-2] < 1:
        raise L.WgsError("%s must be [..., M, N] with M, N >= 1, got shape %s" % (what, tuple(x.shape)))
    if device is not None and (x.device != device or x.dtype != dtype):
        raise L.WgsError("%s: the tensors of a call must share device and type, got %s on %s beside %s on %s" % (what, x.dtype, x.device, dtype, device))


def orthogonalise(x, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7, joined=None):
    """Orthogonal factor of x [..., M, N] by the quintic Newton-Schulz iteration: X / (|X|_F + eps), then `steps` times
    X <- (a + b A + c A A) X, A = X X^T (on the transposed matrix where M > N).  With the default coefficients singular values go to about 1
    (0.7 .. 1.2) and singular vectors stay.

    x: float32 / bfloat16 / float16, any strides; or a list of such matrices, of any sizes, which then share the launches.  Returns a new tensor
    (list) of the same type.  Operands of the products are fp16 hi + lo pairs (22 bits) whatever the type, sums fp32.  A matrix of zeros
    gives zeros, one with a NaN or infinity NaN throughout.  Not differentiable: an update rule's operator, for use without gradients.

    joined: the most iterations that run on the smaller side's matrices alone between two products with the longer side.  None takes 5 for bfloat16,
    3 for float16, 1 for float32 and for matrices (all those of a call) of over 128 rows that are square to a sixteenth.  Up to 3 come as close to the
    exact iterate as 32-bit products do (within 1.4 times their distance); 5 are faster on wide matrices and put a bfloat16 result up to 11 % further from
    it than its rounding does, where one direction outweighs the rest.  Matrices whose smaller side is at most 16 (and the longer one at most 4096 in float32,
    1024 in 16 bits) are computed in 64 bits and rounded once."""
    many = isinstance(x, (list, tuple))
    xs = list(x) if many else [x]
    joined = _joined(joined)
    if not xs:
        return []
    for t in xs:
        _check_matrix(t, 'x', xs[0].device, xs[0].dtype)
        if t.requires_grad and torch.is_grad_enabled():
            raise L.WgsError("orthogonalise has no gradient: call it under torch.no_grad() or on a detached tensor")
    entries, outs, keep = [], [], []
    for t in xs:
        swap = t.stride(-1) != 1 and t.stride(-2) == 1 and t.shape[-1] > 1       # columns adjacent: orthogonalise the transposed view
        y = _as_rows(t.mT if swap else t)
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
        keep.append(y)
        bs, rs = _strides(y)
        b, M, N = y.shape
        if b:
            entries.append((y.data_ptr(), out.data_ptr(), 0, bs, M * N, rs, N, M, N, b, 0.0, 0.0, joined))
        out = out.view(t.shape[:-2] + (M, N))
        outs.append(out.mT if swap else out)
    if entries:
        lib = L.lib()
        a, b, c = (L.c_float(v) for v in coefficients)

        def call(mats, n, code, ws, need):
            L.check(lib.wgs_orthogonalise(mats, n, code, int(steps), a, b, c, L.c_float(eps), ws, need, L.stream()), 'wgs_orthogonalise')
        if not 1 <= int(steps) <= 16:
            raise L.WgsError("steps must be 1 .. 16, got %s" % (steps,))
        _run_matrices(entries, lib.wgs_orthogonalise_ws_bytes, call, xs[0].dtype, xs[0].device, int(steps))
    return outs if many else outs[0]


def _matrix_view(t):
    """A weight as a dense matrix [first dimension, the rest] in MEMORY order of the rest (2-D: as it is): a convolution's [Co, Ci, kh, kw] in
    either layout.  A column permutation commutes with the orthogonalisation, so the order does not matter as long as the weight, its gradient and
    its momentum have the same.  None: no such view."""
    if t.dim() == 2:
        return t
    if t.dim() > 2 and t.is_contiguous():
        return t.view(t.shape[0], -1)
    if t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last):
        return t.permute(0, 2, 3, 1).reshape(t.shape[0], -1)
    return None


def _layout(t):
    """Strides of the dimensions that have more than one entry."""
    return [s for s, n in zip(t.stride(), t.shape) if n > 1]


class MuonUpdate:
    """The step of `muon_step` on tensors that stay where they are: checked and described once, then `step(lr)` any number of times.

    It keeps the tensors themselves (and so their memory), not results: every call reads the gradients and updates momenta and weights in place,
    on the current stream of their device; its workspace comes from torch's allocator, call by call.  A step is refused once a tensor has other memory,
    or once a gradient that was its param's .grad is so no longer (zero_grad(set_to_none=True) and the next backward make a new one)."""

    def __init__(self, params, grads, momenta, momentum=0.95, nesterov=True, weight_decay=0.0, scale=None, grad_scale=1.0, steps=5,
                 coefficients=NS_COEFFICIENTS, eps=1e-7, joined=None):
        joined = _joined(joined)
        if not (len(params) == len(grads) == len(momenta)):
            raise L.WgsError("muon_step: %d params, %d grads, %d momenta" % (len(params), len(grads), len(momenta)))
        if not 0.0 <= momentum < 1.0:
            raise L.WgsError("momentum must be in [0, 1), got %s" % (momentum,))
        if not 1 <= int(steps) <= 16:
            raise L.WgsError("steps must be 1 .. 16, got %s" % (steps,))
        if isinstance(scale, str) and scale != 'rms':
            raise L.WgsError("scale must be None, a number or 'rms', got %r" % (scale,))
        self.tensors = (list(params), list(grads), list(momenta))
        self.weight_decay, self.grad_scale, self.steps = weight_decay, grad_scale, int(steps)
        self.args = (L.c_float(momentum), int(bool(nesterov)))
        self.rest = tuple(L.c_float(v) for v in coefficients) + (L.c_float(eps),)
        self.n = len(params)
        if not self.n:
            return
        self.device, self.dtype = dev, dtype = params[0].device, params[0].dtype
        self.mats = ctypes.create_string_buffer(_MATRIX.size * self.n)
        self.factors, spans = [], []
        for k, (w, g, m) in enumerate(zip(params, grads, momenta)):
            _check_matrix(w, 'param', dev, dtype)
            _check_matrix(g, 'grad', dev, dtype)
            if m.dtype != torch.float32 or m.device != dev or m.shape != w.shape or g.shape != w.shape:
                raise L.WgsError("a momentum must be float32 of its param's shape on its device, got %s %s on %s and grad %s for param %s" % (
                    m.dtype, tuple(m.shape), m.device, tuple(g.shape), tuple(w.shape)))
            if w.dim() != 2 and not (_layout(w) == _layout(m) == _layout(g)):
                raise L.WgsError("a convolution weight, its gradient and its momentum must have the same layout, got strides %s %s %s" % (
                    w.stride(), g.stride(), m.stride()))
            w2, g2, m2 = _matrix_view(w), _matrix_view(g), _matrix_view(m)
            if w2 is None or g2 is None or m2 is None:
                raise L.WgsError("muon_step takes matrices and dense convolution weights, got shape %s strides %s" % (tuple(w.shape), w.stride()))
            M, N = w2.shape
            if not m2.is_contiguous():
                raise L.WgsError("momentum must be contiguous")
            for t, what in ((w2, 'param'), (g2, 'grad')):
                if (N > 1 and t.stride(1) != 1) or (M > 1 and t.stride(0) < N):
                    raise L.WgsError("%s: the elements of a row must be adjacent, got strides %s" % (what, t.stride()))
            gr, wr = (g2.stride(0), w2.stride(0)) if M > 1 else (N, N)
            size = w2.element_size()
            spans.append((m2.data_ptr(), 1, 4 * M * N, 4 * M * N, True))
            for t, r, written in ((w2, wr, True), (g2, gr, False)):
                spans.append((t.data_ptr(), 1, size * M * N, size * M * N, written) if r == N else (t.data_ptr(), M, size * N, size * r, written))
            self.factors.append(max(1.0, M / N) ** 0.5 if scale is None else 0.2 * max(M, N) ** 0.5 if scale == 'rms' else float(scale))
            _MATRIX.pack_into(self.mats, k * _MATRIX.size, g2.data_ptr(), w2.data_ptr(), m2.data_ptr(), 0, 0, gr, wr, M, N, 1, 0.0, 1.0, joined)
        _check_apart(spans)
        self.code = _DTYPES[dtype]
        self.need = L.lib().wgs_muon_step_ws_bytes(self.mats, self.n, self.code, self.steps)
        self.places = self._places()
        self.own = [(w, g) for w, g in zip(params, grads) if w.is_leaf and w.grad is g]
        self.lr = None

    def _places(self):
        return [t.data_ptr() for ts in self.tensors for t in ts]

    @torch.no_grad()
    def step(self, lr):
        if not self.n:
            return
        if self._places() != self.places:
            raise L.WgsError("MuonUpdate: a tensor has been given other memory since it was described: make a new one")
        if any(w.grad is not g for w, g in self.own):
            raise L.WgsError("MuonUpdate: a param's .grad is another tensor than the one described: make a new one, or keep the gradients "
                             "(zero_grad(set_to_none=False))")
        lr = float(lr)                          # (a tensor may change in place)
        if lr != self.lr:
            decay = 1.0 - lr * self.weight_decay
            for k, f in enumerate(self.factors):
                _STEP_DECAY.pack_into(self.mats, k * _MATRIX.size + _STEP_DECAY_AT, lr * f, decay)
            self.lr = lr
        with _on(self.device):
            ws = torch.empty(self.need, dtype=torch.uint8, device=self.device)
            L.check(L.lib().wgs_muon_step(self.mats, self.n, self.code, self.args[0], self.args[1], L.c_float(self.grad_scale), self.steps, *self.rest,
                                          L.rawptr(ws), L.c_int64(self.need), L.stream()), 'wgs_muon_step')
        # (a graph that saved a weight before the step may not use it after)
        torch.autograd.graph.increment_version(self.tensors[0] + self.tensors[2])


_STEP_DECAY, _STEP_DECAY_AT = struct.Struct('=2f'), struct.calcsize('=3Q4q3i')


def _check_apart(spans):
    """What a step writes may overlap neither what else it writes nor the gradients: spans (start, rows, bytes of a row, bytes between rows,
    written).  Rows of one may lie between the rows of another."""
    live = []                                   # spans that reach behind the start of the one at hand
    for span in sorted((a, a + (rows - 1) * step + size, rows, size, step, written) for a, rows, size, step, written in spans):
        live = [s for s in live if s[1] > span[0]]
        for other in live:
            if (span[5] or other[5]) and _rows_meet(other, span):
                raise L.WgsError("muon_step: a param or momentum is given twice, or overlaps another tensor of the call")
        live.append(span)


def _rows_meet(p, q):
    """Whether a row of p and one of q share a byte; (start, end, rows, bytes of a row, bytes between rows, ..), ascending rows apart from each other."""
    if p[2] > q[2]:
        p, q = q, p
    a, _, rows, size, step = p[:5]
    b, end, _, qsize, qstep = q[:5]
    if step == qstep and rows > 1:
        # row i of p against row i + k of q: the same for all i, so the two k around the first row's place decide, where such rows exist
        k = (a - b) // step
        return any(max(0, -n) < min(rows, q[2] - n) and b + n * step < a + size and a < b + n * step + qsize for n in (k, k + 1))
    for i in range(max(0, -((a + size - 1 - b) // step)), rows):
        first = a + i * step
        if first >= end:
            return False
        if first + size > b:
            last = min(q[2] - 1, (first + size - 1 - b) // qstep)       # q's last row that begins before this one ends: the others end earlier
            if b + last * qstep + qsize > first:
                return True
    return False


def muon_step(params, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, scale=None, grad_scale=1.0, steps=5,
              coefficients=NS_COEFFICIENTS, eps=1e-7, joined=None):
    """One update of many matrices in place, in the launches of one (instead of torch.optim.Adam's, lib/trainer.py:153-156, for these weights):

        momentum buffer  m <- momentum m + g,        u = g + momentum m (nesterov) or m       (g = grad_scale * gradient)
        weight           W <- (1 - lr weight_decay) W - lr f O,   O = orthogonalise(u)
        f = sqrt(max(1, M / N)) where scale is None, 0.2 sqrt(max(M, N)) for 'rms' (steps of the size of Adam's), or the number given

    params, grads: matrices [M, N] (rows may be strided, elements of a row adjacent), or convolution weights [Co, Ci, kh, kw], contiguous or
    channels-last, taken as [Co, Ci kh kw]; float32, bfloat16 or float16, one type a call.  momenta: float32 of the same shape and order,
    contiguous.  What is written may overlap nothing else of the call (rows of one tensor may lie between another's).  The stored momentum
    and the whole update are fp32; weights are rounded once.  steps, coefficients, eps, joined: as for `orthogonalise`."""
    MuonUpdate(params, grads, momenta, momentum, nesterov, weight_decay, scale, grad_scale, steps, coefficients, eps, joined).step(lr)
