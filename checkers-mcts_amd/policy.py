"""What a policy says about given actions: log probabilities, entropy and top alternatives of rows of logits, with their gradient
(csrc/ckr_logprobs.hip), and the moves a network would consider in given positions.

The reference reads its policy as one dense masked softmax (Checkers.predict, Checkers.py:425-438; `rules.mask_renorm`); it has no
counterpart of these.  All tensors live on a `cuda` (HIP) device; there is no CPU fallback.
"""
import ctypes as C
import functools
from collections import namedtuple

import torch
from torch.autograd import forward_ad

from . import _lib, rules

ACTIONS = 512                       # of the Checkers policy: 64 layer + 8 x + y (Checkers.py:434)
MOST = 64                           # given actions and alternatives of a row (CKR_LOGPROBS_MOST)
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MASK_NONE, MASK_BYTES, MASK_LEGAL = 0, 1, 2

ActionLogprobs = namedtuple("ActionLogprobs", "logp entropy top_action top_logp")
RankedMoves = namedtuple("RankedMoves", "action logp entropy value")


class LogprobsArgs(C.Structure):
    """ckr_logprobs_args (include/ckr.h)."""
    _fields_ = [(n, C.c_void_p) for n in ("logits", "actions", "mask", "logp", "entropy", "top_action", "top_logp", "stats",
                                          "g_logp", "g_entropy", "grad", "scratch")] + \
        [(n, C.c_int64) for n in ("n", "v", "row_stride", "mask_stride", "grad_stride", "scratch_bytes")] + \
        [(n, C.c_int32) for n in ("dtype", "mask_kind", "action_bytes", "n_given", "top")] + [("inv_temperature", C.c_float)]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _given(actions, n):
    """Given actions a row."""
    return 0 if actions is None or n == 0 else actions.numel() // n


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(n, v, top, dtype):
    """ckr_logprobs_scratch: a function of the sizes alone."""
    bytes_ = _lib.load().ckr_logprobs_scratch(C.byref(LogprobsArgs(n=n, v=v, top=top, dtype=dtype, inv_temperature=1.0, logits=16)))
    if bytes_ < 0:
        _lib.check(int(bytes_))
    return bytes_


def _call(fn, args, device):
    """Launch on the current stream of `device`."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(C.byref(args), _lib.raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(C.byref(args), _lib.raw_stream(index))
    if rc:
        _lib.check(rc)


def _forward(x, actions, mask, mask_kind, top, inv_temperature, want_stats):
    """x [n, v] (last dimension dense), actions dense, k a row, or None, mask [n or 1, ...] or None; logp has the actions' shape."""
    (n, v), dev, f32 = x.shape, x.device, torch.float32
    empty = torch.empty
    logp = None if actions is None else empty(actions.shape, dtype=f32, device=dev)
    entropy = empty(n, dtype=f32, device=dev)
    top_action = top_logp = None
    if top:
        top_action, top_logp = empty((n, top), dtype=torch.int64, device=dev), empty((n, top), dtype=f32, device=dev)
    stats = empty((n, 4), dtype=f32, device=dev) if want_stats else None
    need = _scratch_bytes(n, v, top, DTYPES[x.dtype])
    scratch = empty(need, dtype=torch.uint8, device=dev) if need else None
    a = LogprobsArgs(x.data_ptr(), _ptr(actions), _ptr(mask), _ptr(logp), entropy.data_ptr(), _ptr(top_action), _ptr(top_logp), _ptr(stats),
                     None, None, None, _ptr(scratch), n, v, x.stride(0) if n > 1 else v, mask.stride(0) if mask is not None and mask.shape[0] > 1 else 0, 0, need,
                     DTYPES[x.dtype], mask_kind, 0 if actions is None else actions.element_size(), _given(actions, n), top, inv_temperature)
    _call(_lib.load().ckr_logprobs_forward, a, dev)
    return logp, entropy, top_action, top_logp, stats, a


def _f32(g):
    """An output's gradient as the kernel reads it (sums and means hand expanded ones down, an imaginary part's may be a view of the
    negative of its memory)."""
    return g if g is None or (g.dtype is torch.float32 and g.is_contiguous() and not g.is_neg()) else g.float().contiguous().resolve_neg()


def _kind(t):
    return None if t is None else (t.dtype, t.shape, t.device)


def _came_back(t, kind):
    """A saved tensor as the kernel reads it: hooks may hand another one back."""
    if _kind(t) != kind:
        raise RuntimeError("action_logprobs: a saved tensor came back with another type, shape or device")
    return t if t is None or t.dim() < 2 or t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


class _Logprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, actions, mask, mask_kind, top, inv_temperature):
        logp, entropy, top_action, top_logp, stats, ctx.args = _forward(x, actions, mask, mask_kind, top, inv_temperature, True)
        ctx.save_for_backward(x, actions, mask, stats)
        ctx.kinds = [_kind(t) for t in (x, actions, mask, stats)]
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_action, top_logp)
        return logp, entropy, top_action, top_logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logp, g_entropy, _action, _top):
        if g_logp is None and g_entropy is None:
            return (None,) * 6
        x, actions, mask, stats = map(_came_back, ctx.saved_tensors, ctx.kinds)
        actions, stats = actions if actions is None else actions.contiguous(), stats.contiguous()
        grad = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        g_logp, g_entropy = _f32(g_logp), _f32(g_entropy)
        # the forward's arguments, with the tensors as they come back (hooks may have moved them); a copy, as passes over one graph may run at
        # the same time
        a = LogprobsArgs.from_buffer_copy(ctx.args)
        a.logits, a.stats, a.grad, a.grad_stride, a.top = x.data_ptr(), stats.data_ptr(), grad.data_ptr(), x.shape[1], 0
        a.row_stride = x.stride(0) if x.shape[0] > 1 else x.shape[1]
        a.g_logp, a.g_entropy, a.actions, a.mask, a.scratch = _ptr(g_logp), _ptr(g_entropy), _ptr(actions), _ptr(mask), None
        a.n_given = 0 if g_logp is None else _given(actions, x.shape[0])
        if mask is not None:
            a.mask_stride = mask.stride(0) if mask.shape[0] > 1 else 0
        _call(_lib.load().ckr_logprobs_backward, a, x.device)
        return (grad,) + (None,) * 5


def _check_derivatives(logits):
    """Refuses what would get outputs without knowing how they came about: kernels leave no trace in torch's records, and autograd takes part
    in reverse mode alone."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(logits).tangent is not None:
        raise ValueError("action_logprobs has no forward-mode derivative")
    recorded = torch.jit.is_tracing()
    if not recorded and torch._C._len_torch_dispatch_stack():
        from torch.fx.experimental.proxy_tensor import get_proxy_mode
        recorded = get_proxy_mode() is not None
    if recorded:
        raise ValueError("action_logprobs cannot be recorded by torch.jit.trace or make_fx")


def _check_mask(mask, lead, v, device):
    """-> (mask with one row or a row per row of logits, kind)."""
    if not isinstance(mask, torch.Tensor) or mask.device != device:
        raise ValueError("mask must be a tensor on %s" % device)
    if mask.dtype == torch.int32:
        width, kind = 8, MASK_LEGAL
        if v != ACTIONS:
            raise ValueError("legal-move words (int32 [..., 8]) belong to logits of %d actions, not %d" % (ACTIONS, v))
    elif mask.dtype in (torch.bool, torch.uint8):
        width, kind = v, MASK_BYTES
    else:
        raise ValueError("mask must be a bool tensor [..., %d] (True: allowed) or the int32 [..., 8] legal-move words of rules.movegen" % v)
    if mask.dim() < 1 or mask.shape[-1] != width:
        raise ValueError("the mask's last dimension must be %d, got %s" % (width, list(mask.shape)))
    if mask.dim() == 2 and len(lead) == 1 and mask.shape[0] == lead[0]:
        pass
    elif mask.shape[:-1].numel() == 1:
        mask = mask.reshape(1, width)
    else:
        try:
            mask = mask.expand(lead + (width,)).reshape(-1, width)
        except RuntimeError:
            raise ValueError("a mask of shape %s does not fit logits of shape %s" % (list(mask.shape), list(lead + (v,)))) from None
    return mask if mask.stride(1) == 1 or width == 1 else mask.contiguous(), kind


def action_logprobs(logits, actions=None, mask=None, top=0, temperature=1.0):
    """Log probabilities of given actions, the entropy and the top alternatives of softmax(logits / temperature).

    logits    [..., V] float32, bfloat16 or float16 on the GPU, V from 1 to 2^30.  Rows may lie apart (any row stride, also 0) and start
              anywhere; a last dimension that is not dense is copied once.
    actions   int64 or int32, [...] (one given action a row) or [..., K] with K <= 64; a negative action is none (log p 0, no
              gradient); one >= V gives NaN, and a NaN gradient in its row.
    mask      the actions that count: bool [..., V], [V] or broadcastable (True: allowed), or the int32 [..., 8] legal-move words of
              `rules.movegen` (V = 512).  A logit of -inf is masked too; what is masked may hold anything, NaN included.
    temperature  1e-6 to 1e6.
    top       up to 64 alternatives: the most likely allowed actions, ties to the lower action.

    Returns ActionLogprobs(logp, entropy, top_action, top_logp), float32 and int64 (None for what was not asked).  A masked action has log p
    -inf.  A row without an allowed action: log p -inf, entropy 0, gradient 0.  Where there are fewer than `top` alternatives: action
    -1, log p -inf.  NaN or +inf among the allowed logits make the row's numbers NaN and its alternatives -1.

    Differentiable (once, in reverse mode) in logits through logp and entropy; the alternatives are not.  A masked given action of a row with others keeps
    its part in the gradient, - g p_j, as the formula has it."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dtype not in DTYPES or logits.dim() < 1:
        raise ValueError("logits must be a cuda float32, bfloat16 or float16 tensor [..., V]")
    _check_derivatives(logits)
    lead, v = logits.shape[:-1], logits.shape[-1]
    if v < 1 or v > 1 << 30:
        raise ValueError("logits must have 1 to 2^30 actions a row, got %d" % v)
    if isinstance(top, bool) or not isinstance(top, int) or not 0 <= top <= MOST:
        raise ValueError("top must be an int from 0 to %d" % MOST)
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError("temperature must be from 1e-6 to 1e6, got %r" % temperature)
    x = logits if logits.dim() == 2 else logits.reshape(-1, v)
    if x.stride(1) != 1 and v > 1:
        x = x.contiguous()
    shape = None
    if actions is not None:
        if not isinstance(actions, torch.Tensor) or actions.device != logits.device or actions.dtype not in (torch.int64, torch.int32):
            raise ValueError("actions must be an int64 or int32 tensor on %s" % logits.device)
        shape = actions.shape
        if shape != lead and (len(shape) != len(lead) + 1 or shape[:-1] != lead or not 1 <= shape[-1] <= MOST):
            raise ValueError("actions must have the shape %s or %s + [1 .. %d], got %s" % (list(lead), list(lead), MOST, list(shape)))
        actions = actions.contiguous()
    mask_kind = MASK_NONE
    if mask is not None:
        mask, mask_kind = _check_mask(mask, lead, v, logits.device)
    if x.requires_grad and torch.is_grad_enabled():
        logp, entropy, top_action, top_logp = _Logprobs.apply(x, actions, mask, mask_kind, top, 1.0 / temperature)
    else:
        logp, entropy, top_action, top_logp = _forward(x, actions, mask, mask_kind, top, 1.0 / temperature, False)[:4]
    if len(lead) != 1:
        entropy = entropy.reshape(lead)
        if top:
            top_action, top_logp = top_action.reshape(lead + (top,)), top_logp.reshape(lead + (top,))
    return ActionLogprobs(logp, entropy, top_action, top_logp)


def legal_from_features(x):
    """Network input [N, 8, 8, 14] -> bool [N, 512]: the legal actions its planes 6-13 hold (Checkers.py:431-432)."""
    return (x[..., 6:14] != 0).permute(0, 3, 1, 2).reshape(x.shape[0], ACTIONS)


@torch.no_grad()
def rank_moves(net, boards, top=5, temperature=1.0):
    """The moves that a network (net.PolicyValueNet, on the GPU, eval mode) considers in positions [N, 4] (rules.boards_to_device), best
    first: RankedMoves(action int64 [N, top], logp [N, top], entropy [N], value [N]).  Probabilities are over the legal moves
    (what `rules.mask_renorm` normalises to); action -1 where a position has fewer."""
    mask, _ = rules.movegen(boards)
    x = rules.features(boards).to(next(net.parameters()).dtype)
    logits, value = net.logits(x.permute(0, 3, 1, 2))
    out = action_logprobs(logits, mask=mask, top=top, temperature=temperature)
    return RankedMoves(out.top_action, out.top_logp, out.entropy, value)
