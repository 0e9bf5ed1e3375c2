"""speech_amd.logits -- operators on output rows (csrc/constrain.hip, top_logits.hip, distill.hip; include/speech_amd.h,
section 9).  A row is the logits of one token over V classes, in float32, bfloat16 or float16; sums are held in 32 bits.

  constrain / pick   what a decoder is allowed to answer: penalties for repeated tokens, biases, a grammar's mask -- the
                     constrained logits, or the token they leave and its log-probability
  top_logits         what a teacher leaves of its rows: the k largest logits and the log-sum-exp of the others
  DistillLoss        a student's loss on that, with its gradient; hard targets mixed in on request

Every call runs on the device of its logits, on that device's current stream; all other tensors must live there too.
Arguments that a call cannot take raise SpeechAmdError.  V <= 1048576, k <= 128, histories and bias lists <= 65535 entries."""
import ctypes
import math

import torch

from . import _lib
from ._lib import SpeechAmdError, check
from .ops import is_unit_gradient

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
VOCAB_MAX, LIST_MAX, TOP_MAX = 1048576, 65535, 128


def _rows_of(x, name="logits"):
    """(ld_outer, ld_inner, n_inner, rows) of a (..., V) tensor without copying it: one or two steps between rows."""
    if not torch.is_tensor(x):
        raise SpeechAmdError("%s must be a tensor" % name)
    if x.dtype not in _DTYPES:
        raise SpeechAmdError("%s must be float32, bfloat16 or float16, not %s" % (name, x.dtype))
    if x.dim() < 2 or x.shape[-1] < 1 or x.shape[-1] > VOCAB_MAX:
        raise SpeechAmdError("%s must be (..., V) with 1 <= V <= %d, got %s" % (name, VOCAB_MAX, tuple(x.shape)))
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        raise SpeechAmdError("%s must have a last stride of 1, got strides %s" % (name, x.stride()))
    _lib.require_cuda(x, name)
    if x.dim() == 2:
        return x.stride(0), 0, 1, x.shape[0]
    if x.numel() == 0:
        return x.shape[-1], 0, 1, 0
    merged = []
    for n, s in zip(x.shape[:-1], x.stride()[:-1]):
        if n == 1:
            continue
        if merged and merged[-1][1] == n * s:
            merged[-1] = (merged[-1][0] * n, s)
        else:
            merged.append((n, s))
    if len(merged) > 2:
        raise SpeechAmdError("%s of strides %s has more than two steps between rows: make it contiguous" % (name, x.stride()))
    rows = 1
    for n in x.shape[:-1]:
        rows *= n
    if not merged:
        return x.shape[-1], 0, 1, rows
    if len(merged) == 1:
        return merged[0][1], 0, 1, rows
    return merged[0][1], merged[1][1], merged[1][0], rows


def _tensor(t, name, dtype, shape, device):
    """The device pointer of a packed tensor of exactly this type, shape and device."""
    if not torch.is_tensor(t) or t.dtype != dtype or t.shape != shape:
        raise SpeechAmdError("%s must be a %s tensor of shape %s" % (name, dtype, tuple(shape)))
    if t.device != device:
        raise SpeechAmdError("%s must be on %s like the logits, not %s" % (name, device, t.device))
    if not t.is_contiguous():
        raise SpeechAmdError("%s must be contiguous" % name)
    return t.data_ptr()


_device_now = torch._C._cuda_getDevice                # (what torch.cuda.current_device() / current_stream() end up calling:
_stream_now = torch._C._cuda_getCurrentRawStream      # a token's call is shorter than the objects those two build)


def _launch(name, x, *args):
    """Library entry `name` on the device of x and that device's current stream."""
    fn, index = getattr(_lib.lib(), name), x.get_device()
    if _device_now() == index:
        status = fn(*args, _stream_now(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _stream_now(index))
    if status != 0:
        check(status, name)


def pack_mask(allowed):
    """A (states, V) bool tensor (True: the token may follow) -> the (states, ceil(V / 32)) int32 words constrain reads."""
    if not torch.is_tensor(allowed) or allowed.dtype != torch.bool or allowed.dim() != 2 or allowed.shape[1] < 1:
        raise SpeechAmdError("a mask is packed from a (states, V) bool tensor")
    n, v = allowed.shape
    bits = torch.nn.functional.pad(allowed, (0, -v % 32)).view(n, (v + 31) // 32, 32).to(torch.int64)
    words = (bits << torch.arange(32, device=allowed.device)).sum(2)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _list(t, name, rows, device, dtype):
    if not torch.is_tensor(t) or t.dtype != dtype or t.dim() != 2 or t.shape[0] != rows or t.shape[1] > LIST_MAX:
        raise SpeechAmdError("%s must be a (%d, n) %s tensor with n <= %d" % (name, rows, dtype, LIST_MAX))
    if t.device != device:
        raise SpeechAmdError("%s must be on %s like the logits, not %s" % (name, device, t.device))
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise SpeechAmdError("%s must have a last stride of 1" % name)
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else t.shape[1], t.shape[1]


def _penalty(value, name, rows, device, neutral):
    """(device pointer or None, the value for every row)."""
    if value is None:
        return None, neutral
    if torch.is_tensor(value):
        return _tensor(value, name, torch.float32, (rows,), device), neutral
    value = float(value)
    if not math.isfinite(value) or (name == "repetition" and value <= 0):
        raise SpeechAmdError("%s must be finite%s, got %r" % (name, " and positive" if name == "repetition" else "", value))
    return None, value


def _constraints(rows, V, dev, history, lengths, repetition, presence, frequency, bias_ids, bias_values, mask, states, decoding=False):
    """The arguments of `constrain`, checked, as the library reads them.  decoding: the decode itself keeps the history."""
    c = _lib.saConstraints()
    if history is not None:
        c.history, c.history_ld, c.history_len = _list(history, "history", rows, dev, torch.int64)
        if lengths is not None:
            c.lengths = _tensor(lengths, "lengths", torch.int32, (rows,), dev)
    elif lengths is not None:
        raise SpeechAmdError("lengths without a history")
    c.repetition, c.repetition_all = _penalty(repetition, "repetition", rows, dev, 1.0)
    c.presence, c.presence_all = _penalty(presence, "presence", rows, dev, 0.0)
    c.frequency, c.frequency_all = _penalty(frequency, "frequency", rows, dev, 0.0)
    if history is None and not decoding and not (repetition is None and presence is None and frequency is None):
        raise SpeechAmdError("penalties for repeated tokens need a history")
    if (bias_ids is None) != (bias_values is None):
        raise SpeechAmdError("bias_ids and bias_values come together")
    if bias_ids is not None:
        c.bias_ids, c.bias_ld, c.n_bias = _list(bias_ids, "bias_ids", rows, dev, torch.int64)
        c.bias_values, ld, n = _list(bias_values, "bias_values", rows, dev, torch.float32)
        if n != c.n_bias or ld != c.bias_ld:
            raise SpeechAmdError("bias_ids and bias_values must have the same shape and strides")
    if mask is not None:
        words = (V + 31) // 32
        if not torch.is_tensor(mask) or mask.dtype != torch.int32 or mask.dim() != 2 or mask.shape[0] < min(rows, 1) or mask.shape[1] < words:
            raise SpeechAmdError("mask must be a (states, >= %d) int32 tensor (see pack_mask)" % words)
        if mask.device != dev or (mask.stride(1) != 1 and mask.shape[1] > 1):
            raise SpeechAmdError("mask must be on %s with a last stride of 1" % dev)
        c.mask, c.n_states = mask.data_ptr(), mask.shape[0]
        c.mask_ld = mask.stride(0) if mask.shape[0] > 1 else mask.shape[1]
        if c.mask_ld < words:
            raise SpeechAmdError("the rows of mask overlap")
        if states is not None:
            c.states = _tensor(states, "states", torch.int32, (rows,), dev)
        elif mask.shape[0] != rows:
            raise SpeechAmdError("without states the mask needs a row for each of the %d requests, got %d" % (rows, mask.shape[0]))
    elif states is not None:
        raise SpeechAmdError("states without a mask")
    return c


def decoding_constraints(rows, V, dev, repetition=None, presence=None, frequency=None, bias_ids=None, bias_values=None,
                         mask=None, states=None, next_states=None):
    """What a constrained decode takes (Seq2Seq.infer(constraints=...)): the arguments of `constrain` without a history -- the
    tokens of the decode are that --, and the grammar's transitions: after token v a request in state s goes on in
    next_states[s, v] ((states, V) int32; it stays without them).  Requests start in `states`, or all in state 0; a state
    outside the mask is unmasked from then on.  Returns (saConstraints, penalties, states, pointer of next_states)."""
    if mask is not None and states is None:
        states = torch.zeros(rows, dtype=torch.int32, device=dev)
    c = _constraints(rows, V, dev, None, None, repetition, presence, frequency, bias_ids, bias_values, mask, states, decoding=True)
    following = None
    if next_states is not None:
        if mask is None:
            raise SpeechAmdError("next_states without a mask")
        following = _tensor(next_states, "next_states", torch.int32, (mask.shape[0], V), dev)
    penalties = not (repetition is None and presence is None and frequency is None)
    if states is not None:
        states = states.clone()  # the decode moves its own copy on
    return c, penalties, states, following


def _matrix(logits):
    ld, _, _, rows = _rows_of(logits)
    if logits.dim() != 2 or rows > 0x7fffffff:
        raise SpeechAmdError("logits must be (requests, V), got %s" % (tuple(logits.shape),))
    return ld, rows, logits.shape[1]


def _overlap(x, ldx, y, ldy, rows, V):
    """Whether two (rows, V) matrices of one type share elements without being the same matrix."""
    off = (y.data_ptr() - x.data_ptr()) // x.element_size()
    if rows == 0 or (off == 0 and (ldx == ldy or rows == 1)):
        return False
    if off >= (rows - 1) * ldx + V or -off >= (rows - 1) * ldy + V:
        return False
    return rows == 1 or ldx != ldy or off % ldx < V or -off % ldx < V  # (columns of one matrix may lie beside each other)


def constrain(logits, history=None, lengths=None, repetition=None, presence=None, frequency=None, bias_ids=None,
              bias_values=None, mask=None, states=None, out=None):
    """The logits (requests, V) of each request's next token under its constraints, in the logits' type.

    history (requests, n) int64, lengths (requests,) int32: the tokens so far (n of them without lengths); entries that are no
    class count nowhere.  A token that stands there c > 0 times has its logit x divided by `repetition` where x > 0 and
    multiplied by it elsewhere, then lowered by c * frequency and by presence (numbers, or one float32 per request).
    bias_ids int64, bias_values float32, both (requests, n): added to those tokens; the last entry of a token counts, ids that
    are no class are skipped.
    mask (states, ceil(V / 32)) int32 (pack_mask), states (requests,) int32: a token whose bit is clear in the request's row
    becomes -inf; a state outside the mask leaves its request unmasked; without states request b reads row b.
    out: a tensor like the logits to write to (the logits themselves, too); nothing else may overlap it.  Not differentiable."""
    ld, rows, V = _matrix(logits)
    dev = logits.device
    c = _constraints(rows, V, dev, history, lengths, repetition, presence, frequency, bias_ids, bias_values, mask, states)
    if out is None:
        out = torch.empty_like(logits) if logits.is_contiguous() else torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    else:
        ldo, _, _, _ = _rows_of(out, "out")
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev or (rows > 1 and ldo < V):
            raise SpeechAmdError("out must be like the logits, without overlapping rows")
        if _overlap(logits, ld, out, ldo, rows, V):
            raise SpeechAmdError("out must be the logits themselves or share nothing with them")
        if out.requires_grad and torch.is_grad_enabled():
            raise SpeechAmdError("constrain writes to out without recording it: out must not require a gradient")
    torch.autograd.graph.increment_version(out)  # (written behind autograd's back: whoever saved it must see that)
    _launch("sa_logits_constrain", logits, logits.data_ptr(), ld, _DTYPES[logits.dtype], out.data_ptr(), out.stride(0), rows, V,
            ctypes.byref(c))
    return out


def pick(logits, history=None, lengths=None, repetition=None, presence=None, frequency=None, bias_ids=None,
         bias_values=None, mask=None, states=None):
    """The most likely token of every request under the constraints of `constrain`: (tokens (requests,) int64, its
    log-probability (requests,) float32).  Ties go to the lowest token, NaN counts as the largest value; a request that has no
    token left gets -1 and -inf.  The constrained logits are not written anywhere."""
    ld, rows, V = _matrix(logits)
    dev = logits.device
    c = _constraints(rows, V, dev, history, lengths, repetition, presence, frequency, bias_ids, bias_values, mask, states)
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    code = _DTYPES[logits.dtype]
    nbytes = _lib.lib().sa_logits_pick_workspace_bytes(rows, V, code)
    # a workspace of the call's own: two streams, or two captured graphs, never share one
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _launch("sa_logits_pick", logits, logits.data_ptr(), ld, code, rows, V, ctypes.byref(c), tokens.data_ptr(), logp.data_ptr(),
            ws.data_ptr() if nbytes else None, nbytes)
    return tokens, logp


def _temperature(t):
    t = float(t)
    if not 1e-6 <= t <= 1e6:  # (beyond it T^2 or logits / T leave float32)
        raise SpeechAmdError("temperature must be within 1e-6 .. 1e6, got %r" % t)
    return t


def top_logits(logits, k, temperature=1.0):
    """The k largest logits of every row of (..., V): (values (..., k) float32, ids (..., k) int64, rest (...) float32).
    Descending; ties go to the lowest id; NaN counts as the largest value.  rest = log sum exp(logits / temperature) over the
    other V - k classes (-inf when there are none): with it DistillLoss knows how much of the teacher the list leaves out.
    Not differentiable."""
    ld_outer, ld_inner, n_inner, rows = _rows_of(logits)
    V, k, t = logits.shape[-1], int(k), _temperature(temperature)
    if not 1 <= k <= min(V, TOP_MAX):
        raise SpeechAmdError("k must be 1 .. min(V, %d), got %d for V = %d" % (TOP_MAX, k, V))
    shape, dev = tuple(logits.shape[:-1]), logits.device
    values = torch.empty(shape + (k,), dtype=torch.float32, device=dev)
    ids = torch.empty(shape + (k,), dtype=torch.int64, device=dev)
    rest = torch.empty(shape, dtype=torch.float32, device=dev)
    code = _DTYPES[logits.dtype]
    nbytes = _lib.lib().sa_top_logits_workspace_bytes(rows, V, k, code)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _launch("sa_top_logits", logits, logits.data_ptr(), ld_outer, ld_inner, n_inner, code, rows, V, k, t, values.data_ptr(),
            ids.data_ptr(), rest.data_ptr(), ws.data_ptr() if nbytes else None, nbytes)
    return values, ids, rest


def _versions(tensors):
    """How often each has been written to (a tensor made in inference mode does not count that)."""
    try:
        return [t._version for t in tensors]
    except RuntimeError:
        return [None if t.is_inference() else t._version for t in tensors]


class DistillFunction(torch.autograd.Function):
    """The summed loss (1,) of DistillLoss.  The gradient is produced in the forward pass; autograd's factor is applied by the
    kernel, in 32 bits and before the one rounding to the logits' type."""

    @staticmethod
    def forward(ctx, logits, values, ids, rest, targets, weights, temperature, alpha, scale):
        x = logits.detach()
        ld_outer, ld_inner, n_inner, rows = _rows_of(x)
        V, dev, lead, k = x.shape[-1], x.device, tuple(x.shape[:-1]), values.shape[-1]
        args = (_tensor(values, "values", torch.float32, lead + (k,), dev), _tensor(ids, "ids", torch.int64, lead + (k,), dev),
                None if rest is None else _tensor(rest, "rest", torch.float32, lead, dev), k,
                None if targets is None else _tensor(targets, "targets", torch.int64, lead, dev),
                None if weights is None else _tensor(weights, "weights", torch.float32, lead, dev), temperature, alpha, scale)
        loss = torch.empty(1, dtype=torch.float32, device=dev)
        loss_rows = torch.empty(rows, dtype=torch.float32, device=dev)
        dx = None
        if ctx.needs_input_grad[0]:
            dx = torch.empty_like(x)
            if dx.stride() != x.stride():  # rows with gaps, or shared: the gradient is packed, and the logits with it
                x = x.contiguous()
                dx = torch.empty_like(x)
                ld_outer, ld_inner, n_inner, rows = _rows_of(x)
        _launch("sa_distill_loss", x, x.data_ptr(), None if dx is None else dx.data_ptr(), ld_outer, ld_inner, n_inner,
                _DTYPES[x.dtype], rows, V, *args, None, 0, loss_rows.data_ptr(), loss.data_ptr())
        if dx is not None:
            # (the logits are freed by the walk; the lists are plain attributes with the versions that save_for_backward would keep:
            # six of its records cost more than the launches)
            ctx.save_for_backward(x)
            lists = (values, ids, rest, targets, weights)
            given = [t for t in lists if t is not None]
            ctx.again = (lists, given, _versions(given), ld_outer, ld_inner, n_inner, rows, V, k, temperature, alpha, scale)
            ctx.dx = dx
        return loss

    @staticmethod
    def backward(ctx, go):
        if torch.is_grad_enabled():
            raise SpeechAmdError("the distillation loss is differentiable once: its gradient is no function of the logits to autograd")
        # the first walk takes the buffer of the forward pass along: it is handed out once and never written again
        dx, ctx.dx = ctx.dx, None
        if dx is not None and is_unit_gradient(go):
            return dx, None, None, None, None, None, None, None, None
        x, = ctx.saved_tensors
        lists, given, versions, ld_outer, ld_inner, n_inner, rows, V, k, temperature, alpha, scale = ctx.again
        if _versions(given) != versions:
            raise RuntimeError("the teacher's list, targets or weights of a distillation loss were changed in place after its forward pass")
        fresh = dx is None
        if fresh:
            dx = torch.empty_like(x)
        values, ids, rest, targets, weights = [None if t is None else t.data_ptr() for t in lists]
        # (go: one float32, the type and shape of the loss)
        _launch("sa_distill_loss", x, x.data_ptr(), dx.data_ptr(), ld_outer, ld_inner, n_inner, _DTYPES[x.dtype], rows, V, values, ids,
                rest, k, targets, weights, temperature, alpha, scale, go.data_ptr(), 0 if fresh else 1, None, None)
        return dx, None, None, None, None, None, None, None, None


class DistillLoss(torch.nn.Module):
    """Distillation from a teacher's top logits (top_logits):

        loss = sum over rows of weights * (alpha T^2 soft + (1 - alpha) hard) / denom

    soft = KL(q || p) between the teacher's list and softmax(logits / T): with `rest` the list and, as one more class, everything
    outside it; without `rest` the teacher renormalised over its list.  hard = cross-entropy with `targets` (needed for
    alpha < 1).  denom: the number of rows by default (a data-parallel rank passes the GLOBAL number).

    forward(logits (..., V), values (..., k) float32, ids (..., k) int64, rest=None (...) float32, targets=None (...) int64,
    weights=None (...) float32) -> (1,) float32.  An id that is no class is absent from the list (padding), a target that is none
    gives no hard term, a row of weight 0 is not read and has a gradient of 0 whatever it holds; NaN or +inf in another row's list or
    rest makes the loss NaN.  Only the logits get a gradient, in their own type; it is differentiable once."""

    def __init__(self, temperature=1.0, alpha=1.0, denom=None):
        super().__init__()
        self.temperature, self.alpha, self.denom = _temperature(temperature), float(alpha), denom
        if not 0.0 <= self.alpha <= 1.0:
            raise SpeechAmdError("alpha must be within 0 .. 1, got %r" % alpha)
        if denom is not None and not 1e-30 <= float(denom) <= 1e30:
            raise SpeechAmdError("denom must be within 1e-30 .. 1e30, got %r" % denom)

    def forward(self, logits, values, ids, rest=None, targets=None, weights=None):
        if not torch.is_tensor(values) or values.dim() < 1 or not 1 <= values.shape[-1] <= TOP_MAX:
            raise SpeechAmdError("values must be a (..., k) tensor with 1 <= k <= %d" % TOP_MAX)
        if self.alpha < 1.0 and targets is None:
            raise SpeechAmdError("alpha < 1 mixes in hard targets: targets are needed")
        if not torch.is_tensor(logits) or logits.dim() < 1:
            raise SpeechAmdError("logits must be a (..., V) tensor")
        denom = float(self.denom) if self.denom else float(max(1, logits.numel() // max(1, logits.shape[-1])))
        return DistillFunction.apply(logits, values, ids, rest, targets, weights, self.temperature, self.alpha, 1.0 / denom)
