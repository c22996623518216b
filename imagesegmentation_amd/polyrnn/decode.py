"""Softmax cross-entropy, argmax, sampling, log-probabilities and distillation over the vertex class grid, on the libisg
kernels (isg_softmax_xent_fwd / _bwd, isg_argmax_rows, isg_sample_rows, isg_token_logprobs_*, isg_distill_*)."""
import typing

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _lib
from ..ops import dtype_code, pixel_stride


def _rows(logits):
    cols = logits.shape[-1]
    z = logits.reshape(-1, cols)
    if z.dtype not in (torch.float32, torch.bfloat16):
        z = z.float()
    return z.contiguous(), z.shape[0], cols


class _XentRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, weights, argmax_out=None):
        z, rows, cols = _rows(logits)
        lab = labels.reshape(-1).to(torch.int32).contiguous()
        w = weights.reshape(-1).to(torch.float32).contiguous() if weights is not None else None
        loss = torch.empty([rows], dtype=torch.float32, device=z.device)
        lse = torch.empty([rows], dtype=torch.float32, device=z.device)
        rc = _lib.lib().isg_softmax_xent_fwd(_lib.ptr(z), _lib.ptr(lab), _lib.ptr(w), rows, cols, dtype_code(z.dtype),
                                             _lib.ptr(loss), _lib.ptr(lse), _lib.ptr(argmax_out),
                                             _lib.current_stream())
        _lib.check(rc, "isg_softmax_xent_fwd")
        ctx.save_for_backward(z, lab, lse, w)
        ctx.shape, ctx.in_dtype = logits.shape, logits.dtype
        return loss.reshape(logits.shape[:-1])

    @staticmethod
    def backward(ctx, dloss):
        z, lab, lse, w = ctx.saved_tensors
        rows, cols = z.shape
        scale = dloss.reshape(-1).to(torch.float32)
        if w is not None:
            scale = scale * w
        scale = scale.contiguous()
        dz = torch.empty_like(z)
        rc = _lib.lib().isg_softmax_xent_bwd(_lib.ptr(z), _lib.ptr(lab), _lib.ptr(lse), _lib.ptr(scale), 1.0, rows,
                                             cols, dtype_code(z.dtype), _lib.ptr(dz), _lib.current_stream())
        _lib.check(rc, "isg_softmax_xent_bwd")
        return dz.reshape(ctx.shape).to(ctx.in_dtype), None, None, None


class _SequenceLoss(torch.autograd.Function):
    """Mean cross-entropy over every step of every sequence together with the step's masked metrics (reference
    polyrnn/Model.py:44-54, 98-100) in two launches - the per-row pass and one summary launch that finishes the
    mean and the quotients on the device - and a backward pass of one launch."""

    @staticmethod
    def forward(ctx, logits, targets, durations, prediction_size):
        z, rows, cols = _rows(logits)
        B, T = targets.shape[0], targets.shape[1]
        tg = targets.to(torch.int32).contiguous()
        dur = durations.to(torch.int32).contiguous()
        dev = z.device
        loss_rows = torch.empty([rows], dtype=torch.float32, device=dev)
        lse = torch.empty([rows], dtype=torch.float32, device=dev)
        pred = torch.empty([rows], dtype=torch.int32, device=dev)
        lab = torch.empty([rows], dtype=torch.int32, device=dev)
        rc = _lib.lib().isg_sequence_xent_fwd(_lib.ptr(z), _lib.ptr(tg), rows, cols, int(prediction_size),
                                              dtype_code(z.dtype), _lib.ptr(loss_rows), _lib.ptr(lse), _lib.ptr(pred),
                                              _lib.ptr(lab), _lib.current_stream())
        _lib.check(rc, "isg_sequence_xent_fwd")
        out6 = torch.empty([6], dtype=torch.float64, device=dev)
        mean = torch.empty([], dtype=torch.float32, device=dev)
        rc = _lib.lib().isg_sequence_summary(_lib.ptr(pred), _lib.ptr(tg), _lib.ptr(dur), _lib.ptr(loss_rows), B, T,
                                             int(prediction_size), _lib.ptr(out6), _lib.ptr(mean), _lib.current_stream())
        _lib.check(rc, "isg_sequence_summary")
        ctx.save_for_backward(z, lab, lse)
        ctx.shape, ctx.in_dtype = logits.shape, logits.dtype
        ctx.mark_non_differentiable(out6)
        ctx.set_materialize_grads(False)  # (else a zero gradient for out6 is filled in on every backward pass)
        return mean, out6

    @staticmethod
    def backward(ctx, dmean, _):
        z, lab, lse = ctx.saved_tensors
        rows, cols = z.shape
        if dmean is None:
            return None, None, None, None
        up = dmean.to(torch.float32).contiguous()
        dz = torch.empty_like(z)
        rc = _lib.lib().isg_softmax_xent_mean_bwd(_lib.ptr(z), _lib.ptr(lab), _lib.ptr(lse), _lib.ptr(up), rows, cols,
                                                  dtype_code(z.dtype), _lib.ptr(dz), _lib.current_stream())
        _lib.check(rc, "isg_softmax_xent_mean_bwd")
        return dz.reshape(ctx.shape).to(ctx.in_dtype), None, None, None


def sequence_loss(logits, targets, durations, prediction_size):
    """(mean loss, float64 [6] = correct, error sum, error max, live steps, accuracy, mean error); logits [B,T,K],
    targets int [B,T,2] as (x, y) (class = x * prediction_size + y), durations int [B]."""
    return _SequenceLoss.apply(logits, targets, durations, prediction_size)


def softmax_xent_rows(logits, labels, weights=None, argmax_out=None):
    """Per-row sparse softmax cross-entropy (optionally times a per-row weight).  ``argmax_out``
    (int32, one per row) receives the first-maximum class of each row from the same pass."""
    return _XentRows.apply(logits, labels, weights, argmax_out)


def softmax_xent_mean(logits, labels, weights=None, argmax_out=None):
    """mean over every row (reference polyrnn/Model.py:98-100)."""
    return softmax_xent_rows(logits, labels, weights, argmax_out).mean()


def sequence_metrics(pred, targets, durations, prediction_size):
    """Masked accuracy / mean L2 error / max L2 error of reference polyrnn/Model.py:44-54 from ONE kernel:
    pred int32 [B, T] argmax classes, targets int [B, T, 2] (x, y), durations int [B].
    Returns a float64 device tensor [4] = (correct, error sum, error max, number of live steps)."""
    B, T = targets.shape[0], targets.shape[1]
    pred = pred.reshape(-1).to(torch.int32).contiguous()
    tg = targets.to(torch.int32).contiguous()
    dur = durations.to(torch.int32).contiguous()
    out = torch.empty([4], dtype=torch.float64, device=pred.device)
    rc = _lib.lib().isg_sequence_metrics(_lib.ptr(pred), _lib.ptr(tg), _lib.ptr(dur), B, T, int(prediction_size),
                                         _lib.ptr(out), _lib.current_stream())
    _lib.check(rc, "isg_sequence_metrics")
    return out


def argmax_rows(logits):
    """int64 argmax over the last axis, first maximum wins (tf.argmax)."""
    z, rows, cols = _rows(logits)
    out = torch.empty([rows], dtype=torch.int32, device=z.device)
    rc = _lib.lib().isg_argmax_rows(_lib.ptr(z), rows, cols, dtype_code(z.dtype), _lib.ptr(out), _lib.current_stream())
    _lib.check(rc, "isg_argmax_rows")
    return out.to(torch.int64).reshape(logits.shape[:-1])


def prediction_max(logits, prediction_size):
    """[..., 2] = (argmax // P, argmax % P), i.e. (x, y) (reference polyrnn/Model.py:91-94)."""
    a = argmax_rows(logits)
    return torch.stack([a // prediction_size, a % prediction_size], dim=-1)


def sample_rows(logits, seed, row_offset=0):
    """One categorical sample per row of softmax(logits) (tf.multinomial's role)."""
    z, rows, cols = _rows(logits)
    out = torch.empty([rows], dtype=torch.int32, device=z.device)
    rc = _lib.lib().isg_sample_rows(_lib.ptr(z), rows, cols, dtype_code(z.dtype), int(seed), int(row_offset),
                                    _lib.ptr(out), _lib.current_stream())
    _lib.check(rc, "isg_sample_rows")
    return out.to(torch.int64).reshape(logits.shape[:-1])


def sample_actions(logits, seed, grid_side, row_offset=0, row_offset_dev=None, out=None):
    """One categorical sample per row, delivered as the action (x, y) = (class // P, class % P), int32
    [rows, 2], from one launch (reference polyrl/ReinforceOverfitExperiment.py:101-105).
    ``row_offset_dev`` (uint64/int64 device scalar) is added to ``row_offset`` on the device."""
    z, rows, cols = _rows(logits)
    if out is None:
        out = torch.empty([rows, 2], dtype=torch.int32, device=z.device)
    rc = _lib.lib().isg_sample_actions(_lib.ptr(z), rows, cols, dtype_code(z.dtype), int(seed), int(row_offset),
                                       _lib.ptr(row_offset_dev), int(grid_side), _lib.ptr(out), _lib.current_stream())
    _lib.check(rc, "isg_sample_actions")
    return out


# ---- log-probabilities, entropy, alternatives ------------------------------------------------------------------------
TOP_MAX = 64             # ISG_TOP_MAX
DISTILL_MAX = 1024       # ISG_DISTILL_MAX
CLASSES_MAX = 1 << 20    # ISG_CLASSES_MAX
ROWS_MAX = (1 << 31) - 1  # the entry points' int


class TokenLogprobs(typing.NamedTuple):
    """What ``token_logprobs`` returns; ``logprobs`` is None without tokens, the ``top_*`` are None with top = 0."""
    logprobs: typing.Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprobs: typing.Optional[torch.Tensor]
    top_classes: typing.Optional[torch.Tensor]


def _refuse_tangent(t, what):
    """The kernels read a tensor's values only.  (A dual tensor need not require a gradient, so nothing else would notice.)"""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError("%s: forward-mode derivatives are not implemented" % what)


def _class_rows(logits, what):
    """(logits, rows, classes, elements from row to row) as the kernels read them: float32 or bfloat16, a row's classes
    adjacent, rows evenly spaced - in place where the tensor is that (a column slice of padded logits, every other step of a batch), a
    copy otherwise."""
    if not torch.is_tensor(logits) or logits.dim() < 1 or not logits.is_floating_point():
        raise TypeError("%s: logits must be a floating-point tensor of at least one axis" % what)
    cols = logits.shape[-1]
    if not 1 <= cols <= CLASSES_MAX:
        raise ValueError("%s: %d classes (1 to %d)" % (what, cols, CLASSES_MAX))
    rows = logits.numel() // cols
    if rows > ROWS_MAX:  # (an int argument would keep its lower 32 bits without a word)
        raise ValueError("%s: %d rows (at most %d)" % (what, rows, ROWS_MAX))
    _refuse_tangent(logits, what)
    if not logits.is_cuda:
        raise RuntimeError("%s: logits must live on the GPU: libisg has no CPU path" % what)
    z = logits if logits.dtype in (torch.float32, torch.bfloat16) else logits.float()
    if z.is_contiguous():
        return z, rows, cols, cols
    stride = pixel_stride(z) if z.dim() > 1 else None
    if stride is None or stride < cols:
        return z.contiguous(), rows, cols, cols
    return z, rows, cols, stride


def _row_argument(t, shape, kinds, device, what):
    """A per-row tensor of one of the ``kinds`` in the rows' shape, contiguous."""
    if not torch.is_tensor(t) or t.dtype not in kinds:
        raise TypeError("%s must be a tensor of %s" % (what, " or ".join(str(k).replace("torch.", "") for k in kinds)))
    if t.shape != shape:
        raise ValueError("%s must have the shape %s, not %s" % (what, tuple(shape), tuple(t.shape)))
    if t.device != device:
        raise ValueError("%s lives on %s, the logits on %s" % (what, t.device, device))
    return t.contiguous()


def _temperature(value, what):
    value = float(value)
    if not 1e-30 <= value <= 1e30:
        raise ValueError("%s: temperature %g (positive and finite)" % (what, value))
    return value


def _launch(function, device, args):
    """A launch on the current stream of the device, which is made the current one where it is not."""
    if device == torch._C._cuda_getDevice():
        rc = function(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = function(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        _lib.check(rc, function.__name__)


_ONE_UNIT_CLASSES = 2048  # rows up to here take no workspace
_ROW_CLASSES = (torch.int32, torch.int64)
_ROW_MASKS = (torch.bool, torch.uint8)


def _logprobs_forward(z, geometry, tokens, live, top, temperature, keep):
    rows, cols, stride = geometry
    lib, dev, f32 = _lib.lib(), z.device, torch.float32
    entropy = torch.empty([rows], dtype=f32, device=dev)
    logp = top_logp = top_cls = stats = space = None
    if tokens is not None:
        logp = torch.empty_like(entropy)
    if top:
        top_logp = torch.empty([rows, top], dtype=f32, device=dev)
        top_cls = torch.empty([rows, top], dtype=torch.int32, device=dev)
    if keep:
        stats = torch.empty([rows, 4], dtype=f32, device=dev)
    if cols > _ONE_UNIT_CLASSES:
        space = torch.empty([lib.isg_token_logprobs_workspace_bytes(rows, cols, top)], dtype=torch.uint8, device=dev)
    _launch(lib.isg_token_logprobs_fwd, dev.index, (
        z.data_ptr(), stride, _address(tokens), tokens.element_size() if tokens is not None else 4, _address(live), rows,
        cols, dtype_code(z.dtype), temperature, top, _address(logp), entropy.data_ptr(), _address(top_logp),
        _address(top_cls), _address(stats), _address(space)))
    return logp, entropy, top_logp, top_cls, stats


def _address(t):
    return None if t is None else t.data_ptr()


# Backward passes run on autograd's own thread, where every line of Python costs two to three times what it does in the
# caller's: sizes and types are put together in the forward pass, and their checks are the forward's.  The tensors are
# asked for their addresses here: saved-tensor hooks (checkpoints, copies in host memory) may hand back others.
def _saved_rows(z, cols, what):
    """The logits the forward pass saved, the elements from row to row, and the (dense) tensor for their gradient."""
    if z.is_contiguous():
        return z, cols, torch.empty_like(z)
    dense = torch.empty(z.shape, dtype=z.dtype, device=z.device)
    z, _, _, stride = _class_rows(z, what)
    return z, stride, dense


def _float_gradient(g, what):
    if g is None:
        return None
    _refuse_tangent(g, what)
    if g.dtype == torch.float32 and g.is_contiguous():
        return g
    return g.to(torch.float32).contiguous()


def _first_derivative_only(function):
    """As ``once_differentiable``, at no cost where no graph of the backward pass is asked for."""
    guarded = once_differentiable(function)

    def backward(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else function(ctx, *grads)
    return backward


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, geometry, tokens, live, top, temperature):
        logp, entropy, top_logp, top_cls, stats = _logprobs_forward(z, geometry, tokens, live, top, temperature, True)
        ctx.save_for_backward(z, tokens, top_cls, stats)
        ctx.last = (geometry[0], geometry[1], dtype_code(z.dtype), temperature, top)
        if top_cls is not None:
            ctx.mark_non_differentiable(top_cls)
        ctx.set_materialize_grads(False)
        return logp, entropy, top_logp, top_cls

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dlogp, dentropy, dtop, _):
        if dlogp is None and dentropy is None and dtop is None:
            return None, None, None, None, None, None
        z, tokens, top_cls, stats = ctx.saved_tensors
        what = "token_logprobs"
        z, stride, dz = _saved_rows(z, ctx.last[1], what)
        dlogp, dentropy, dtop = _float_gradient(dlogp, what), _float_gradient(dentropy, what), _float_gradient(dtop, what)
        _launch(_lib.lib().isg_token_logprobs_bwd, dz.get_device(), (
            z.data_ptr(), stride, _address(tokens), tokens.element_size() if tokens is not None else 4, _address(top_cls),
            stats.data_ptr(), _address(dlogp), _address(dentropy), _address(dtop), *ctx.last, dz.data_ptr()))
        return dz, None, None, None, None, None


def token_logprobs(logits, tokens=None, top=0, temperature=1.0, live=None):
    """Log-probabilities of given classes, entropies and the most probable classes of softmax(logits / temperature),
    from one pass over the logits (isg_token_logprobs_fwd); differentiable in the logits through everything but the
    classes (isg_token_logprobs_bwd; first derivatives only, in reverse mode).

    logits [..., K] (float32 and bfloat16 as they are, also with rows evenly apart; others through float32; fewer than
    2^31 rows), tokens int32 or int64 [...] or None, top = how many of the largest logits to report (0 to 64, at most
    K; equal logits lowest class first), live bool or uint8 [...] or None: rows without it are not read and give zeros
    (class -1) and no gradient - steps past a sequence's duration.  Logits of -inf are classes without probability.

    Returns ``TokenLogprobs``: logprobs float32 [...] (NaN for a class outside [0, K)), entropy float32 [...],
    top_logprobs float32 [..., top], top_classes int32 [..., top].  Near 0 they are good to some 1e-7 absolutely: where
    all other classes together have less than 6e-8, a class's log-probability is 0."""
    if not torch.is_tensor(logits) or logits.dim() < 1:
        raise TypeError("token_logprobs: logits must be a floating-point tensor of at least one axis")
    lead = logits.shape[:-1]
    top = int(top)
    if not 0 <= top <= min(TOP_MAX, logits.shape[-1]):
        raise ValueError("token_logprobs: top %d of %d classes (0 to %d)" % (top, logits.shape[-1], TOP_MAX))
    temperature = _temperature(temperature, "token_logprobs")
    if tokens is not None:
        tokens = _row_argument(tokens, lead, _ROW_CLASSES, logits.device, "token_logprobs: tokens")
    if live is not None:
        live = _row_argument(live, lead, _ROW_MASKS, logits.device, "token_logprobs: live")
    z, *geometry = _class_rows(logits, "token_logprobs")
    if z.requires_grad and torch.is_grad_enabled():
        logp, entropy, top_logp, top_cls = _TokenLogprobs.apply(z, geometry, tokens, live, top, temperature)
    else:
        logp, entropy, top_logp, top_cls, _ = _logprobs_forward(z, geometry, tokens, live, top, temperature, False)
    if len(lead) != 1:
        logp = logp.reshape(lead) if logp is not None else None
        entropy = entropy.reshape(lead)
        if top:
            top_logp, top_cls = top_logp.reshape(lead + (top,)), top_cls.reshape(lead + (top,))
    return TokenLogprobs(logp, entropy, top_logp, top_cls)


# ---- distillation -----------------------------------------------------------------------------------------------------
def _distill_forward(z, geometry, values, classes, live, temperature, tail, keep):
    rows, cols, stride = geometry
    lib, dev, f32 = _lib.lib(), z.device, torch.float32
    loss = torch.empty([rows], dtype=f32, device=dev)
    stats = torch.empty([rows, 8], dtype=f32, device=dev) if keep else None
    space = None
    if cols > _ONE_UNIT_CLASSES:
        space = torch.empty([lib.isg_distill_workspace_bytes(rows, cols)], dtype=torch.uint8, device=dev)
    _launch(lib.isg_distill_fwd, dev.index, (
        z.data_ptr(), stride, values.data_ptr(), classes.data_ptr(), classes.element_size(), _address(live), rows, cols,
        values.shape[-1], dtype_code(z.dtype), temperature, tail, loss.data_ptr(), _address(stats), _address(space)))
    return loss, stats


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, geometry, values, classes, live, temperature, tail):
        loss, stats = _distill_forward(z, geometry, values, classes, live, temperature, tail, True)
        ctx.save_for_backward(z, values, classes, stats)
        ctx.last = (geometry[0], geometry[1], values.shape[-1], dtype_code(z.dtype), temperature, tail)
        return loss

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dloss):
        z, values, classes, stats = ctx.saved_tensors
        z, stride, dz = _saved_rows(z, ctx.last[1], "distill_rows")
        dloss = _float_gradient(dloss, "distill_rows")
        _launch(_lib.lib().isg_distill_bwd, dz.get_device(), (
            z.data_ptr(), stride, values.data_ptr(), classes.data_ptr(), classes.element_size(), stats.data_ptr(),
            dloss.data_ptr(), *ctx.last, dz.data_ptr()))
        return dz, None, None, None, None, None, None


def distill_rows(logits, teacher_values, teacher_classes, temperature=1.0, tail=False, live=None):
    """Per-row divergence of softmax(logits / temperature) from a teacher's k most probable classes (isg_distill_fwd /
    isg_distill_bwd), float32 [...], differentiable in the logits (first derivatives only, in reverse mode):
    sum_j q_j (log q_j - log p_j).  The teacher takes no gradient and no tangent.

    logits [..., K] as ``token_logprobs`` takes them; teacher_values float [..., k] and teacher_classes int32 or int64
    [..., k], k from 1 to 1024: what ``token_logprobs(teacher_logits, top=k, temperature=temperature)`` returns.  A
    negative class is no entry; a class outside the row makes the row NaN.

    tail=False: q = softmax(teacher_values / temperature) over the entries (the teacher's logits); tail=True: the values
    are log-probabilities at this temperature and the mass they leave is one more class, set against the student's mass
    outside the entries (where no class is left outside, up to 1e-5 of remaining mass counts as rounding, more gives an
    infinite loss).  live: as in ``token_logprobs``.  (A loss that mixes temperatures multiplies by temperature^2
    to keep the gradients' size; that factor is the caller's.)"""
    if not torch.is_tensor(logits) or logits.dim() < 1:
        raise TypeError("distill_rows: logits must be a floating-point tensor of at least one axis")
    lead = logits.shape[:-1]
    temperature = _temperature(temperature, "distill_rows")
    if not torch.is_tensor(teacher_values) or not teacher_values.is_floating_point():
        raise TypeError("distill_rows: teacher_values must be a floating-point tensor")
    k = teacher_values.shape[-1] if teacher_values.dim() else 0
    if not 1 <= k <= DISTILL_MAX:
        raise ValueError("distill_rows: %d classes of the teacher (1 to %d)" % (k, DISTILL_MAX))
    values = teacher_values.detach() if teacher_values.requires_grad else teacher_values
    if values.dtype != torch.float32:
        values = values.float()
    shape = lead + (k,)
    values = _row_argument(values, shape, (torch.float32,), logits.device, "distill_rows: teacher_values")
    classes = _row_argument(teacher_classes, shape, _ROW_CLASSES, logits.device, "distill_rows: teacher_classes")
    if live is not None:
        live = _row_argument(live, lead, _ROW_MASKS, logits.device, "distill_rows: live")
    z, *geometry = _class_rows(logits, "distill_rows")
    if z.requires_grad and torch.is_grad_enabled():
        loss = _Distill.apply(z, geometry, values, classes, live, temperature, int(bool(tail)))
    else:
        loss, _ = _distill_forward(z, geometry, values, classes, live, temperature, int(bool(tail)), False)
    return loss if len(lead) == 1 else loss.reshape(lead)


def distill_mean(logits, teacher_values, teacher_classes, temperature=1.0, tail=False, live=None):
    """``distill_rows`` averaged over the live rows (over every row without ``live``); 0 when none is live."""
    loss = distill_rows(logits, teacher_values, teacher_classes, temperature, tail, live)
    if live is None:
        return loss.mean()
    return loss.sum() / torch.count_nonzero(live).clamp(min=1)


def decode_begin(true_vertices, num_true, hist, steps):
    """isg_decode_begin: what the decode loop starts from, one launch (reference polyrnn/Model.py:218-230).
    true_vertices int32 [B, vmax, 2], num_true int32 [B] -> (close_xy [B,2], first history points [B,hist,2], the
    loop's own copy of them, required [B] = 1, durations [B] = 0, predicted [B,steps,2] = 0), all int32."""
    B, vmax = true_vertices.shape[0], true_vertices.shape[1]
    dev = true_vertices.device
    assert true_vertices.dtype == torch.int32 and num_true.dtype == torch.int32
    new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=dev)
    close, pts0, pts = new(B, 2), new(B, hist, 2), new(B, hist, 2)
    required, durations, predicted = new(B), new(B), new(B, steps, 2)
    rc = _lib.lib().isg_decode_begin(_lib.ptr(true_vertices.contiguous()), _lib.ptr(num_true.contiguous()), B, vmax,
                                     int(hist), int(steps), _lib.ptr(close), _lib.ptr(pts0) if hist else None,
                                     _lib.ptr(pts) if hist else None, _lib.ptr(required), _lib.ptr(durations),
                                     _lib.ptr(predicted), _lib.current_stream())
    _lib.check(rc, "isg_decode_begin")
    return close, pts0, pts, required, durations, predicted


def decode_polygons(predicted, durations, first_points, scale, prepend_history, slice_by_duration, vmax):
    """isg_decode_polygons: the decoded polygons as the rasteriser takes them (reference polyrnn/Model.py:252-260):
    (polygons int32 [B, vmax, 2], counts int32 [B])."""
    B, T = predicted.shape[0], predicted.shape[1]
    hist = first_points.shape[1]
    vp = torch.empty([B, vmax, 2], dtype=torch.int32, device=predicted.device)
    count = torch.empty([B], dtype=torch.int32, device=predicted.device)
    rc = _lib.lib().isg_decode_polygons(_lib.ptr(predicted), _lib.ptr(durations), _lib.ptr(first_points) if hist else None,
                                        B, T, hist, int(bool(prepend_history)), int(bool(slice_by_duration)), int(scale),
                                        int(vmax), _lib.ptr(vp), _lib.ptr(count), _lib.current_stream())
    _lib.check(rc, "isg_decode_polygons")
    return vp, count


def column_sums(x, out=None):
    """isg_column_sums: float32 [cols] = sum over the rows of x [rows, cols] (float32 or bfloat16), a fixed order of
    additions - the dense head's bias gradient over all (sample, step) rows (a library reduction over a tall matrix
    takes 0.27 ms for 20,480 x 785, this 0.02).  ``out``: where to write (float32 [cols], contiguous)."""
    rows, cols = x.shape
    x = x.contiguous()
    if out is None:
        out = torch.empty([cols], dtype=torch.float32, device=x.device)
    assert out.dtype == torch.float32 and out.is_contiguous() and out.numel() == cols
    ws = torch.empty([_lib.lib().isg_column_sums_workspace_bytes(int(cols)) // 4], dtype=torch.float32, device=x.device)
    rc = _lib.lib().isg_column_sums(_lib.ptr(x), int(rows), int(cols), dtype_code(x.dtype), _lib.ptr(out), _lib.ptr(ws),
                                    _lib.current_stream())
    _lib.check(rc, "isg_column_sums")
    return out


def dense_few_rows(flat, w, b, slices=None):
    """flat [M, K] @ w [K, N] + b in the operands' type for few rows against a long reduction axis (a decode or
    rollout step's head): one library GEMM has M N / tile output tiles for 256 CUs, so the reduction axis is cut
    into ``slices`` batched GEMMs with float results, summed with the bias by one launch (isg_sum_slices_bias).
    None when the shape does not call for it (the caller's plain GEMM then)."""
    M, K = flat.shape
    N = b.numel()  # (w may carry zero columns beyond the bias's classes: a copy padded to a multiple of 8)
    if slices is None:  # (measured at K = 12,544, N = 785: 16 rows 26 -> 19 us, 2,048 rows 125 -> 82 us)
        slices = 8 if M <= 256 else 4
    # (the rows may lie apart - one step's outputs inside a sequence's kept outputs -, each contiguous in itself)
    if not (flat.is_cuda and flat.dtype == torch.bfloat16 and w.dtype == flat.dtype and flat.stride(1) == 1 and
            (M == 1 or (flat.stride(0) >= K and flat.stride(0) % 8 == 0)) and flat.data_ptr() % 16 == 0 and
            w.is_contiguous() and M * N <= (1 << 21) and K % (slices * 8) == 0 and K // slices >= 512):
        return None
    try:
        part = torch.bmm(flat.unflatten(1, (slices, K // slices)).transpose(0, 1),
                         w.view(slices, K // slices, w.shape[1]), out_dtype=torch.float32)
    except TypeError:  # (a torch without float32 results from a bf16 batched GEMM)
        return None
    return sum_slices_bias(part, b)


def sum_slices_bias(part, b):
    """part float32 [slices, M, Np] summed over the slices + b [N], N <= Np (the first N columns are kept), in b's type
    (float32 or bf16), in one launch."""
    slices, M, Np = part.shape
    N = b.numel()
    assert part.dtype == torch.float32 and part.is_contiguous() and N <= Np
    out = torch.empty([M, N], dtype=b.dtype, device=part.device)
    rc = _lib.lib().isg_sum_slices_bias_padded(_lib.ptr(part), slices, M, N, Np, _lib.ptr(b.contiguous()),
                                               dtype_code(out.dtype), _lib.ptr(out), _lib.current_stream())
    _lib.check(rc, "isg_sum_slices_bias_padded")
    return out


def rows_dot(flat, w, b=None):
    """flat [M, K] . w [K] (or [K, 1]) + b as float32 [M], operands bf16 (isg_rows_dot): a dense layer with one output
    column.  None when the operands do not fit (the caller's library GEMM then)."""
    M, K = flat.shape
    if not (flat.is_cuda and flat.dtype == torch.bfloat16 and w.dtype == flat.dtype and flat.is_contiguous() and
            w.is_contiguous() and w.numel() == K and K % 8 == 0 and (b is None or b.dtype == flat.dtype) and
            flat.data_ptr() % 16 == 0 and w.data_ptr() % 16 == 0):
        return None
    out = torch.empty([M], dtype=torch.float32, device=flat.device)
    rc = _lib.lib().isg_rows_dot(_lib.ptr(flat), _lib.ptr(w), _lib.ptr(b), M, K, dtype_code(flat.dtype), _lib.ptr(out),
                                 _lib.current_stream())
    _lib.check(rc, "isg_rows_dot")
    return out


def decode_step(logits, grid_side, end_token, close_xy, required, durations, predicted, step, history_points):
    """isg_decode_step: argmax of every row, then the decode loop's bookkeeping (stop rule, predicted polygon,
    history points of the next step) on the device.  logits [B, K]; all other tensors int32 and updated in
    place: close_xy [B,2], required [B], durations [B], predicted [B,T,2], history_points [B,hist,2]."""
    z, rows, cols = _rows(logits)
    hist = history_points.shape[1]
    for t in (close_xy, required, durations, predicted, history_points):
        assert t.dtype == torch.int32 and t.is_contiguous()
    rc = _lib.lib().isg_decode_step(_lib.ptr(z), rows, cols, dtype_code(z.dtype), int(grid_side), int(bool(end_token)),
                                    _lib.ptr(close_xy), _lib.ptr(required), _lib.ptr(durations), _lib.ptr(predicted),
                                    predicted.shape[1], int(step), _lib.ptr(history_points) if hist else None, hist,
                                    _lib.current_stream())
    _lib.check(rc, "isg_decode_step")
