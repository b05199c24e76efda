"""Operators of a policy row on the GPU: `score` (log-probabilities of given moves, entropy, best alternatives) and
`loss` (the trainer's loss, reference src/train.py: KLDivLoss(batchmean) + MSELoss), both differentiable.

The HIP kernels (csrc/az_policy.hip, reached through the C ABI) run on torch's current stream of the tensors' device;
they allocate through torch, wait for nothing and can be captured into a graph.  Only legal moves count where `board`
or `legal` names them; what stands in the other cells (infinities, NaN) is not looked at, and a row in which nothing
is legal (a full board) is empty: log-probability -inf, entropy 0, no alternatives, no gradient.

A forward and backward pass that are captured together need nothing from outside.  As with every torch operator, do
not capture a backward pass while an eager graph of the same leaves is alive (its gradient accumulators belong to the
eager stream): drop the eager loss first, or differentiate with `torch.autograd.grad`."""
from collections import namedtuple

import torch

from . import engine as _E

MAX_MOVES, MAX_TOP = 64, 32  # AZ_POLICY_MAX_MOVES, AZ_POLICY_MAX_TOP
MAX_ACTIONS = 1 << 24
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # AZ_F32, AZ_BF16, AZ_F16

Score = namedtuple("Score", "logp entropy top_moves top_logp")


def _refuse(what):
    raise ValueError(what)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(name, device, *args):
    entry = getattr(_E.load_library(), name)
    stream = torch._C._cuda_getCurrentRawStream(device.index)  # (torch.cuda.current_stream: 3 us more a call)
    if torch.cuda.current_device() == device.index:
        rc = entry(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = entry(*args, stream)
    if rc != 0:
        raise RuntimeError(f"{name} failed (code {rc})")


def _once():
    if torch.is_grad_enabled():  # a backward pass that builds a graph of itself
        raise RuntimeError("the policy operators can be differentiated once (no create_graph)")


def _on_one_gpu(**tensors):
    device = tensors["logits"].device
    for what, t in tensors.items():
        if t is not None and (not t.is_cuda or t.device != device):
            _refuse(f"{what} must be on the GPU of the logits (there is no CPU path)")


def _rows(logits, board, legal):
    """Checks a batch of rows; returns what the kernels are handed: logits and masks with unit inner stride."""
    if not torch.is_tensor(logits) or logits.dim() != 2:
        _refuse("logits must be a tensor [rows, actions]")
    if logits.dtype not in TYPES:
        _refuse(f"logits must be float32, bfloat16 or float16, not {logits.dtype}")
    n, actions = logits.shape
    if not 1 <= actions <= MAX_ACTIONS or n > 0x7FFFFFFF:
        _refuse(f"{n} rows of {actions} actions: at least 1 action and at most {MAX_ACTIONS} are supported")
    if board is not None and legal is not None:
        _refuse("give the legal moves by board or by legal, not both")
    if board is not None:
        if board.dtype != torch.float32 or board.dim() != 4 or board.shape[0] != n or board.shape[1] != 2 \
                or board.shape[2] != board.shape[3] or board.shape[2] * board.shape[3] != actions:
            _refuse(f"board must be float32 [{n}, 2, S, S] with S * S = {actions}")
        board = board.contiguous()
    if legal is not None:
        if legal.dtype not in (torch.bool, torch.uint8) or tuple(legal.shape) not in ((n, actions), (actions,), (1, actions)):
            _refuse(f"legal must be bool or uint8, [{n}, {actions}] or [{actions}]")
        legal = legal.expand(n, actions)
        if (actions > 1 and legal.stride(1) != 1) or (n > 1 and legal.stride(0) != 0 and legal.stride(0) < actions):
            legal = legal.contiguous()
    if (actions > 1 and logits.stride(1) != 1) or (n > 1 and logits.stride(0) < actions):
        logits = logits.contiguous()
    return logits, board, legal


def _row_args(logits, board, legal):
    n, actions = logits.shape
    ld = logits.stride(0) if n > 1 else actions
    ld_legal = 0 if legal is None else legal.stride(0) if n > 1 else actions
    return (n, actions, logits.data_ptr(), TYPES[logits.dtype], ld, _ptr(board), _ptr(legal), ld_legal)


def _score_forward(logits, moves, board, legal, top, keep):
    n, actions = logits.shape
    dev = logits.device
    new = lambda shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=dev)  # noqa: E731
    logp = None if moves is None else new(moves.shape)
    m = 0 if moves is None else 1 if moves.dim() == 1 else moves.shape[1]
    entropy = new(n)
    top_logp, top_moves = (new((n, top)), new((n, top), torch.int32)) if top else (None, None)
    stats = new((n, 2)) if keep else None
    L = _E.load_library()
    words = L.az_policy_mask_words(actions) if keep and (board is not None or legal is not None) else 0
    bits = new((n, words), torch.int64) if words else None
    bytes_ = L.az_policy_score_work(n, actions, top)
    work = new(bytes_, torch.uint8) if bytes_ else None
    _call("az_policy_score", dev, *_row_args(logits, board, legal), _ptr(moves), 0 if moves is None else moves.element_size(),
          m, top, _ptr(logp), entropy.data_ptr(), _ptr(top_logp), _ptr(top_moves), _ptr(stats), _ptr(bits), _ptr(work))
    return logp, entropy, top_moves, top_logp, stats, bits


class _ScoreFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, moves, board, legal, top):
        logp, entropy, top_moves, top_logp, stats, bits = _score_forward(logits, moves, board, legal, top, True)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in (top_moves, top_logp) if t is not None])
        ctx.save_for_backward(logits, moves, board, legal, entropy, stats, bits)
        return logp, entropy, top_moves, top_logp

    @staticmethod
    def backward(ctx, g_logp, g_entropy, _moves, _logp):
        _once()
        logits, moves, board, legal, entropy, stats, bits = ctx.saved_tensors
        if g_logp is None and g_entropy is None:
            return None, None, None, None, None
        d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        m = 0 if moves is None or g_logp is None else 1 if moves.dim() == 1 else moves.shape[1]
        g_logp = None if g_logp is None else g_logp.contiguous()
        g_entropy = None if g_entropy is None else g_entropy.contiguous()
        _call("az_policy_score_grad", logits.device, *_row_args(logits, board, legal), _ptr(bits), _ptr(moves),
              0 if moves is None else moves.element_size(), m, _ptr(g_logp), _ptr(g_entropy), entropy.data_ptr(),
              stats.data_ptr(), d.data_ptr())
        return d, None, None, None, None


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

    logp and entropy are differentiable for logits (once); the alternatives are not."""
    logits, board, legal = _rows(logits, board, legal)
    n = logits.shape[0]
    if moves is not None:
        if moves.dtype not in (torch.int32, torch.int64) or moves.dim() not in (1, 2) or moves.shape[0] != n:
            _refuse(f"moves must be int32 or int64, [{n}] or [{n}, m]")
        if moves.dim() == 2 and not 1 <= moves.shape[1] <= MAX_MOVES:
            _refuse(f"at most {MAX_MOVES} moves per row (and at least one)")
        moves = moves.contiguous()
    if not isinstance(top, int) or not 0 <= top <= MAX_TOP:
        _refuse(f"top must be 0..{MAX_TOP}")
    _on_one_gpu(logits=logits, board=board, legal=legal, moves=moves)
    if torch.is_grad_enabled() and logits.requires_grad:
        return Score(*_ScoreFunction.apply(logits, moves, board, legal, top))
    return Score(*_score_forward(logits, moves, board, legal, top, False)[:4])


def _loss_call(logits, value, pi, r, board, legal, scale, only_if_scaled, total, parts, d_logits, d_value):
    n, actions = logits.shape
    work = torch.empty(_E.load_library().az_policy_loss_work(n, actions), dtype=torch.uint8, device=logits.device)
    _call("az_policy_loss", logits.device, *_row_args(logits, board, legal), value.data_ptr(),
          int(value.dtype == torch.float32), pi.data_ptr(), r.data_ptr(), _ptr(scale), int(only_if_scaled), _ptr(total),
          _ptr(parts), _ptr(d_logits), _ptr(d_value), work.data_ptr())


class _LossFunction(torch.autograd.Function):
    """The gradients are written in the forward pass, which has the row at hand.  The backward pass hands them out as they
    are when the upstream gradient is 1 (decided on the device) and otherwise computes them again with that factor, so
    that a loss scale acts before the rounding to 16 bits."""

    @staticmethod
    def buffers(ctx, *inputs):
        return [torch.empty(t.shape, dtype=t.dtype, device=t.device) if need else None
                for t, need in zip(inputs, ctx.needs_input_grad)]

    @staticmethod
    def forward(ctx, logits, value, pi, r, board, legal, want_parts):
        total = torch.empty((), dtype=torch.float32, device=logits.device)
        parts = torch.empty(2, dtype=torch.float32, device=logits.device) if want_parts else None
        d_logits, d_value = _LossFunction.buffers(ctx, logits, value)
        _loss_call(logits, value, pi, r, board, legal, None, False, total, parts, d_logits, d_value)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, value, pi, r, board, legal)
        ctx.ready = (d_logits, d_value)
        if want_parts:
            ctx.mark_non_differentiable(parts)
        return total, parts

    @staticmethod
    def backward(ctx, g, _parts):
        _once()
        logits, value, pi, r, board, legal = ctx.saved_tensors
        ready, ctx.ready = ctx.ready, None  # given away once: a second backward pass computes its own
        d_logits, d_value = ready or _LossFunction.buffers(ctx, logits, value)
        _loss_call(logits, value, pi, r, board, legal, g.contiguous(), ready is not None, None, None,
                   d_logits, d_value)
        return d_logits, d_value, None, None, None, None, None


def loss(logits, value, pi, r, *, board=None, legal=None, parts=False):
    """The loss of n training records as a float32 scalar:

        1/n sum_i sum_j pi_ij (log pi_ij - log p_ij)  +  1/n sum_i (value_i - r_i)^2

    logits  [n, actions] float32, bfloat16 or float16, p their softmax over the legal moves (see `score` for board and
            legal; the reference trains without a mask);  value  n values of any shape, float32 or the logits' type
    pi      float32 [n, actions], targets (rows need not sum to 1; masked cells are not looked at);  r  float32, n results

    Differentiable (once) for logits and value.  parts=True returns (total, policy part, value part), the parts without
    gradient.  Zero records give 0."""
    logits, board, legal = _rows(logits, board, legal)
    n, actions = logits.shape
    if value.dtype not in (torch.float32, logits.dtype) or value.numel() != n:
        _refuse(f"value must hold {n} values of float32 or the logits' type")
    if pi.dtype != torch.float32 or tuple(pi.shape) != (n, actions):
        _refuse(f"pi must be float32 [{n}, {actions}]")
    if r.dtype != torch.float32 or r.numel() != n:
        _refuse(f"r must hold {n} float32 results")
    if pi.requires_grad or r.requires_grad:
        _refuse("pi and r have no gradient: detach them")
    _on_one_gpu(logits=logits, board=board, legal=legal, value=value, pi=pi, r=r)
    if n == 0:
        zero = logits.sum(dtype=torch.float32) + value.sum(dtype=torch.float32)
        return (zero, zero.detach(), zero.detach()) if parts else zero
    total, two = _LossFunction.apply(logits, value.contiguous(), pi.contiguous(), r.contiguous(), board, legal, bool(parts))
    return (total, two[0], two[1]) if parts else total
