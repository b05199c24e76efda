"""Operators of a policy row on the GPU: `score` (log-probabilities of given moves, entropy, best alternatives) and
`loss` (the trainer's loss, reference src/train.py: KLDivLoss(batchmean) + MSELoss), both differentiable.

The HIP kernels (csrc/az_policy.hip, reached through the C ABI) run on torch's current stream of the tensors' device;
they allocate through torch, wait for nothing and can be captured into a graph.  Only legal moves count where `board`
or `legal` names them; what stands in the other cells (infinities, NaN) is not looked at, and a row in which nothing
is legal (a full board) is empty: log-probability -inf, entropy 0, no alternatives, no gradient.

A forward and backward pass that are captured together need nothing from outside.  As with every torch operator, do
not capture a backward pass while an eager graph of the same leaves is alive (its gradient accumulators belong to the
eager stream): drop the eager loss first, or differentiate with `torch.autograd.grad`."""
import functools
from collections import namedtuple

import torch
from torch.autograd import forward_ad as _forward

from . import engine as _E

MAX_MOVES, MAX_TOP = 64, 32  # AZ_POLICY_MAX_MOVES, AZ_POLICY_MAX_TOP
MAX_ACTIONS = 1 << 24
SHORT_MAX = 1024  # rows up to here are held in registers
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # AZ_F32, AZ_BF16, AZ_F16

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)
_tracing = getattr(torch._C, "_get_tracing_state", None) or (lambda: torch.jit.is_tracing() or None)

Score = namedtuple("Score", "logp entropy top_moves top_logp")


def _refuse(what):
    raise ValueError(what)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(name, device, *args):
    """An entry point on the current stream of `device` (an index); raises what it refuses."""
    entry = getattr(_E.load_library(), name)
    stream = _raw_stream(device)  # (torch.cuda.current_stream: 3 us more a call)
    if torch.cuda.current_device() == device:
        rc = entry(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = entry(*args, stream)
    if rc != 0:
        raise RuntimeError(f"{name} failed (code {rc})")


@functools.lru_cache(1024)
def _score_sizes(n, actions, top):
    """(mask words a row, bytes of workspace) of a score."""
    L = _E.load_library()
    return L.az_policy_mask_words(actions), L.az_policy_score_work(n, actions, top)


@functools.lru_cache(1024)
def _loss_work(n, actions):
    return _E.load_library().az_policy_loss_work(n, actions)


def _once():
    if torch.is_grad_enabled():  # a backward pass that builds a graph of itself
        raise RuntimeError("the policy operators can be differentiated once (no create_graph)")


def _untraced(what):
    if _tracing() is not None:  # a trace would hold the addresses of this call's tensors, or none of its work
        raise RuntimeError(f"{what} cannot be traced")


def _without_tangents(*tensors):
    for t in tensors:
        if torch.is_tensor(t) and _forward.unpack_dual(t).tangent is not None:
            raise RuntimeError("the policy operators have no forward-mode derivative")


def _on_one_gpu(logits, *others):
    device = logits.get_device()
    if device < 0:
        _refuse("logits must be on a GPU (there is no CPU path)")
    for t in others:
        if t is not None and t.get_device() != device:
            _refuse("all tensors must be on the GPU of the logits")
    return device


def _rows(logits, board, legal):
    """Checks a batch of rows; returns what the kernels are handed (logits and masks with unit inner stride) and the entry
    points' leading arguments."""
    if not torch.is_tensor(logits) or logits.dim() != 2:
        _refuse("logits must be a tensor [rows, actions]")
    kind = TYPES.get(logits.dtype)
    if kind is None:
        _refuse(f"logits must be float32, bfloat16 or float16, not {logits.dtype}")
    n, actions = logits.shape
    if not 1 <= actions <= MAX_ACTIONS or n > 0x7FFFFFFF:
        _refuse(f"{n} rows of {actions} actions: at least 1 action and at most {MAX_ACTIONS} are supported")
    ld, step = logits.stride()
    if (actions > 1 and step != 1) or (n > 1 and ld < actions):
        logits, ld = logits.contiguous(), actions
    if n <= 1:
        ld = actions
    at_board = at_legal = None
    ld_legal = 0
    if board is not None:
        if legal is not None:
            _refuse("give the legal moves by board or by legal, not both")
        shape = board.shape
        if board.dtype != torch.float32 or len(shape) != 4 or shape[0] != n or shape[1] != 2 or shape[2] != shape[3] \
                or shape[2] * shape[2] != actions:
            _refuse(f"board must be float32 [{n}, 2, S, S] with S * S = {actions}")
        board = board.contiguous()
        at_board = board.data_ptr()
    elif legal is not None:
        if legal.dtype not in (torch.bool, torch.uint8) or tuple(legal.shape) not in ((n, actions), (actions,), (1, actions)):
            _refuse(f"legal must be bool or uint8, [{n}, {actions}] or [{actions}]")
        legal = legal.expand(n, actions)
        ld_legal, step = legal.stride()
        if (actions > 1 and step != 1) or (n > 1 and 0 != ld_legal < actions):
            legal, ld_legal = legal.contiguous(), actions
        if n <= 1:
            ld_legal = actions
        at_legal = legal.data_ptr()
    return logits, board, legal, (n, actions, logits.data_ptr(), kind, ld, at_board, at_legal, ld_legal)


def _keep(ctx, rows, device, logits, board, legal, *others):
    """Saves tensors for the backward pass (the others dense)."""
    ctx.rows, ctx.device = rows, device
    ctx.kept = [None if t is None else (t.data_ptr(), t.shape, t.dtype) for t in others]
    ctx.save_for_backward(logits, board, legal, *others)


def _kept(ctx):
    """What _keep saved: the entry points' leading arguments, and the tensors.  A saved-tensor hook may have moved a tensor or
    laid it out otherwise; one that hands back other sizes or types, or a tensor on another device, is refused."""
    logits, board, legal, *others = ctx.saved_tensors
    rows = ctx.rows
    if not (logits.data_ptr() == rows[2] and _ptr(board) == rows[5] and _ptr(legal) == rows[6] and
            (rows[0] <= 1 or (logits.stride(0) == rows[4] and (legal is None or legal.stride(0) == rows[7])))):
        logits, board, legal, rows = _rows(logits, board, legal)
        if (rows[0], rows[1], rows[3]) != (ctx.rows[0], ctx.rows[1], ctx.rows[3]) or _on_one_gpu(logits, board, legal) != ctx.device:
            raise RuntimeError("a saved-tensor hook handed back other logits or masks")
    for i, (t, was) in enumerate(zip(others, ctx.kept)):
        if t is not None and (t.data_ptr() != was[0] or not t.is_contiguous()):
            if t.shape != was[1] or t.dtype != was[2] or t.get_device() != ctx.device:
                raise RuntimeError(f"a saved-tensor hook handed back {t.dtype} {tuple(t.shape)} on {t.device} for {was[2]} {tuple(was[1])}")
            others[i] = t.contiguous()
    return rows, logits, board, legal, *others


def _score_forward(logits, moves, board, legal, top, rows, device, keep):
    n, actions = rows[:2]
    new = logits.new_empty
    logp = None if moves is None else new(moves.shape, dtype=torch.float32)
    m = 0 if moves is None else 1 if moves.dim() == 1 else moves.shape[1]
    entropy = new((n,), dtype=torch.float32)
    top_logp, top_moves = (new((n, top), dtype=torch.float32), new((n, top), dtype=torch.int32)) if top else (None, None)
    words, size = _score_sizes(n, actions, top)
    stats = new((n, 2), dtype=torch.float32) if keep else None
    bits = new((n, words), dtype=torch.int64) if keep and words and (board is not None or legal is not None) else None
    work = new((size,), dtype=torch.uint8) if size else None
    _call("az_policy_score", device, *rows, _ptr(moves), 0 if moves is None else moves.element_size(),
          m, top, _ptr(logp), entropy.data_ptr(), _ptr(top_logp), _ptr(top_moves), _ptr(stats), _ptr(bits), _ptr(work))
    return logp, entropy, top_moves, top_logp, stats, bits


class _ScoreFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, moves, board, legal, top, rows, device):
        logp, entropy, top_moves, top_logp, stats, bits = _score_forward(logits, moves, board, legal, top, rows, device, True)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_moves, top_logp)
        _keep(ctx, rows, device, logits, board, legal, moves, entropy, stats, bits)
        return logp, entropy, top_moves, top_logp

    @staticmethod
    def backward(ctx, g_logp, g_entropy, _moves, _logp):
        _once()
        rows, logits, board, legal, moves, entropy, stats, bits = _kept(ctx)
        if g_logp is None and g_entropy is None:
            return (None,) * 7
        d = logits.new_empty(logits.shape)
        m = 0 if moves is None or g_logp is None else 1 if moves.dim() == 1 else moves.shape[1]
        g_logp = None if g_logp is None else g_logp.contiguous()
        g_entropy = None if g_entropy is None else g_entropy.contiguous()
        _call("az_policy_score_grad", ctx.device, *rows, _ptr(bits), _ptr(moves),
              0 if moves is None else moves.element_size(), m, _ptr(g_logp), _ptr(g_entropy), entropy.data_ptr(),
              stats.data_ptr(), d.data_ptr())
        return d, None, None, None, None, None, None


def score(logits, moves=None, *, board=None, legal=None, top=0):
    """What a policy answers: Score(logp, entropy, top_moves, top_logp) for logits [n, actions] (log-probabilities are
    logits too; float32, bfloat16 or float16).

    moves     int32 or int64 [n] or [n, m], m <= 64: logp (float32, same shape) holds their log-probabilities; a negative
              move stands for none (0), an illegal one gives -inf, one past the last action NaN.  None: logp is None
    board     float32 [n, 2, S, S]: a cell is legal where both planes are 0;  legal  bool or uint8 [n, actions] or
              [actions].  Neither: every action counts
    top       the `top` <= 32 best legal moves, best first and equal logits by lowest index, as int32 top_moves
              (-1 where no legal move is left) and float32 top_logp (-inf there).  0: both are None
    entropy   float32 [n], of the distribution over the legal moves

    logp and entropy are differentiable for logits (once, in reverse mode); the alternatives are not."""
    _untraced("policy.score")
    if _forward._current_level >= 0:  # (within a dual_level; no other call pays for the look)
        _without_tangents(logits)
    logits, board, legal, rows = _rows(logits, board, legal)
    n = rows[0]
    if moves is not None:
        if moves.dtype not in (torch.int32, torch.int64) or moves.dim() not in (1, 2) or moves.shape[0] != n:
            _refuse(f"moves must be int32 or int64, [{n}] or [{n}, m]")
        if moves.dim() == 2 and not 1 <= moves.shape[1] <= MAX_MOVES:
            _refuse(f"at most {MAX_MOVES} moves per row (and at least one)")
        moves = moves.contiguous()
    if not isinstance(top, int) or not 0 <= top <= MAX_TOP:
        _refuse(f"top must be 0..{MAX_TOP}")
    device = _on_one_gpu(logits, board, legal, moves)
    if logits.requires_grad and torch.is_grad_enabled():
        return Score(*_ScoreFunction.apply(logits, moves, board, legal, top, rows, device))
    return Score(*_score_forward(logits, moves, board, legal, top, rows, device, False)[:4])


def _loss_call(rows, device, value, pi, r, scale, only_if_scaled, total, parts, d_logits, d_value):
    work = None if total is None and rows[1] <= SHORT_MAX else pi.new_empty((_loss_work(rows[0], rows[1]),), dtype=torch.uint8)
    _call("az_policy_loss", device, *rows, value.data_ptr(), int(value.dtype == torch.float32), pi.data_ptr(), r.data_ptr(),
          _ptr(scale), only_if_scaled, _ptr(total), _ptr(parts), _ptr(d_logits), _ptr(d_value), _ptr(work))


class _LossFunction(torch.autograd.Function):
    """The gradients are written in the forward pass, which has the row at hand.  The backward pass hands them out as they
    are when the upstream gradient is 1 (decided on the device) and otherwise computes them again with that factor, so
    that a loss scale acts before the rounding to 16 bits."""

    @staticmethod
    def forward(ctx, logits, value, pi, r, board, legal, want_parts, rows, device):
        total = pi.new_empty(())
        parts = pi.new_empty((2,)) if want_parts else None
        need_l, need_v = ctx.needs_input_grad[:2]
        d_logits = logits.new_empty(logits.shape) if need_l else None
        d_value = value.new_empty(value.shape) if need_v else None
        _loss_call(rows, device, value, pi, r, None, 0, total, parts, d_logits, d_value)
        ctx.set_materialize_grads(False)
        _keep(ctx, rows, device, logits, board, legal, value, pi, r)
        ctx.ready = d_logits, d_value
        if want_parts:
            ctx.mark_non_differentiable(parts)
        return total, parts

    @staticmethod
    def backward(ctx, g, _parts):
        _once()
        rows, logits, board, legal, value, pi, r = _kept(ctx)
        ready, ctx.ready = ctx.ready, None  # given away once: a second backward pass computes its own
        if ready is None:
            need_l, need_v = ctx.needs_input_grad[:2]
            d_logits = logits.new_empty(logits.shape) if need_l else None
            d_value = value.new_empty(value.shape) if need_v else None
        else:
            d_logits, d_value = ready
        _loss_call(rows, ctx.device, value, pi, r, g.contiguous(), int(ready is not None), None, None, d_logits, d_value)
        return d_logits, d_value, None, None, None, None, None, None, None


def loss(logits, value, pi, r, *, board=None, legal=None, parts=False):
    """The loss of n training records as a float32 scalar:

        1/n sum_i sum_j pi_ij (log pi_ij - log p_ij)  +  1/n sum_i (value_i - r_i)^2

    logits  [n, actions] float32, bfloat16 or float16, p their softmax over the legal moves (see `score` for board and
            legal; the reference trains without a mask);  value  n values of any shape, float32 or the logits' type
    pi      float32 [n, actions], targets (rows need not sum to 1; masked cells are not looked at, a target on a legal cell
            at -inf makes the loss infinite);  r  float32, n results

    Differentiable (once, in reverse mode) for logits and value.  parts=True returns (total, policy part, value part), the
    parts without gradient.  Zero records give 0."""
    _untraced("policy.loss")
    if _forward._current_level >= 0:
        _without_tangents(logits, value, pi, r)
    logits, board, legal, rows = _rows(logits, board, legal)
    n, actions = rows[:2]
    if value.dtype not in (torch.float32, logits.dtype) or value.numel() != n:
        _refuse(f"value must hold {n} values of float32 or the logits' type")
    if pi.dtype != torch.float32 or tuple(pi.shape) != (n, actions):
        _refuse(f"pi must be float32 [{n}, {actions}]")
    if r.dtype != torch.float32 or r.numel() != n:
        _refuse(f"r must hold {n} float32 results")
    if pi.requires_grad or r.requires_grad:
        _refuse("pi and r have no gradient: detach them")
    device = _on_one_gpu(logits, board, legal, value, pi, r)
    if n == 0:
        zero = logits.sum(dtype=torch.float32) + value.sum(dtype=torch.float32)
        return (zero, zero.detach(), zero.detach()) if parts else zero
    if not torch.is_grad_enabled():
        logits, value = logits.detach(), value.detach()  # no gradients are computed that nobody can ask for
    total, two = _LossFunction.apply(logits, value.contiguous(), pi.contiguous(), r.contiguous(), board, legal, bool(parts),
                                     rows, device)
    return (total, two[0], two[1]) if parts else total
