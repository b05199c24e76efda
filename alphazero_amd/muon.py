"""Orthogonalised weight updates on the GPU: `orthogonalise` (Newton-Schulz steps on matrices of updates) and `Muon`, the
optimiser that applies them to a network's weight matrices (K. Jordan et al., "Muon: An optimizer for hidden layers in neural
networks", 2024: the coefficients, the momentum and the factor for weights with more rows than columns).

The HIP kernels (csrc/az_muon.hip, reached through the C ABI) run on torch's current stream of the tensors' device; they
allocate through torch, wait for nothing and can be captured into a graph."""
import ctypes as C
import functools

import torch

from . import engine as _E
from .policy import TYPES, _call, _ptr, _refuse, _untraced

MAX_DIM, MAX_CELLS, MAX_STEPS = 32768, 1 << 28, 10  # AZ_MUON_MAX_*


@functools.lru_cache(1024)
def _work(count, rows, cols):
    return _E.load_library().az_muon_work(count, rows, cols)


def _check(rows, cols, dtype, steps):
    if dtype not in TYPES:
        _refuse(f"updates must be float32, bfloat16 or float16, not {dtype}")
    if rows > MAX_DIM or cols > MAX_DIM or rows * cols > MAX_CELLS:
        _refuse(f"an update of {rows} x {cols}: at most {MAX_DIM} rows or columns and {MAX_CELLS} cells are supported")
    if not isinstance(steps, int) or not 1 <= steps <= MAX_STEPS:
        _refuse(f"steps must be 1..{MAX_STEPS}")


def _on_gpu(tensors):
    if any(not t.is_cuda for t in tensors):
        _refuse("weights and updates must be on a GPU (there is no CPU path)")


def _run(inputs, outputs, rows, cols, ld, dtype, device, steps):
    """inputs, outputs: device addresses of matrices of one shape on GPU `device` (an index), rows `ld` (outputs: cols)
    elements apart."""
    count = len(inputs)
    addresses = C.c_void_p * count
    size = _work(count, rows, cols)
    work = torch.empty(size, dtype=torch.uint8, device=torch.device("cuda", device)) if size else None
    _call("az_muon_orthogonalise", device, count, rows, cols, addresses(*inputs), ld, addresses(*outputs), cols,
          TYPES[dtype], steps, _ptr(work))


def _rows_apart(x):
    """x [..., rows, cols] with unit column stride and rows that do not overlap, copied only if it has none."""
    rows, cols = x.shape[-2:]
    if (cols > 1 and x.stride(-1) != 1) or (rows > 1 and x.stride(-2) < cols):
        x = x.contiguous()
    return x, x.stride(-2) if rows > 1 else cols


def orthogonalise(updates, steps=5):
    """Moves the singular values of each update towards 1 and keeps its singular vectors: X = G / |G|, then `steps` times
    X <- a X + (b A + c A^2) X with A = X X' and (a, b, c) = (3.4445, -4.7750, 2.0315).

    updates   float32, bfloat16 or float16: a matrix [rows, cols], a batch [count, rows, cols], or a list of tensors of two
              or more dimensions, each taken as [first, all others] (a convolution's weights: output channels by the rest).
    steps     1..10
    Returns new tensors of the same shapes and types (a list for a list), without gradient; a matrix of zeros stays zero.
    Whatever the type, the steps are computed with products of float32 precision, relative to the whole matrix, and rounded
    once at the end.  Numbers below 2^-39 of |G| are not kept: a row of 1e-5 |G| comes out with five digits, one of 1e-7 |G|
    with three, one of 1e-11 |G| as zero."""
    _untraced("muon.orthogonalise")
    if torch.is_tensor(updates):
        if updates.dim() not in (2, 3):
            _refuse("updates must be a matrix, a batch of matrices or a list of tensors")
        rows, cols = updates.shape[-2:]
        _check(rows, cols, updates.dtype, steps)
        _on_gpu([updates])
        out = updates.new_empty(updates.shape)
        if out.numel():
            x, ld = _rows_apart(updates.detach())
            size = x.element_size()
            count = x.shape[0] if x.dim() == 3 else 1
            step = x.stride(0) * size if x.dim() == 3 else 0
            a, b, c = x.data_ptr(), out.data_ptr(), rows * cols * size
            _run([a + i * step for i in range(count)], range(b, b + count * c, c), rows, cols, ld, x.dtype, x.get_device(), steps)
        return out
    updates = list(updates)
    groups = {}
    outs = []
    for t in updates:
        if not torch.is_tensor(t) or t.dim() < 2:
            _refuse("an update must be a tensor of two or more dimensions")
        _check(t.shape[0], t[0].numel() if t.shape[0] else 0, t.dtype, steps)
    _on_gpu(updates)
    for i, t in enumerate(updates):
        outs.append(torch.empty(t.shape, dtype=t.dtype, device=t.device))
        if t.numel():
            x, ld = _rows_apart(t.detach().flatten(1))
            groups.setdefault((x.shape[0], x.shape[1], ld, x.dtype, x.get_device()), []).append((x, outs[i]))
    for (rows, cols, ld, dtype, device), members in groups.items():
        _run([x.data_ptr() for x, _ in members], [o.data_ptr() for _, o in members], rows, cols, ld, dtype, device, steps)
    return outs


def _check_options(group, read=True):
    """read=False: a learning rate that is a tensor is not looked at (that would wait for the GPU)."""
    lr, decay = group["lr"], group["weight_decay"]
    if (read or not torch.is_tensor(lr)) and not lr >= 0 or not decay >= 0 or not 0 <= group["momentum"] < 1:
        _refuse("lr and weight_decay must not be negative, momentum must be in [0, 1)")
    if not isinstance(group["steps"], int) or not 1 <= group["steps"] <= MAX_STEPS:
        _refuse(f"steps must be 1..{MAX_STEPS}")


class Muon(torch.optim.Optimizer):
    """Momentum with orthogonalised updates, for weights of two or more dimensions (convolutions and dense layers; give
    biases and batch-norm parameters to another optimiser, `weights_of` tells them apart):

        m <- momentum m + g,   u = g + momentum m (nesterov) or m,
        w <- w (1 - lr weight_decay) - lr sqrt(max(1, rows / cols)) orthogonalise(u)

    Whatever the weights' type, m and u are float32 and a step is rounded into the weight once: in 16 bits a momentum of 0.999
    would not decay at all, and one of 0.95 would stop at gradients below 6e-7."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5):
        options = dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps)
        _check_options(options)
        super().__init__(params, options)

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            _check_options(self.param_groups[-1])
            for p in self.param_groups[-1]["params"]:
                if p.dim() < 2:
                    _refuse("Muon takes weights of two or more dimensions")
                _check(p.shape[0], p[0].numel() if p.shape[0] else 0, p.dtype, self.param_groups[-1]["steps"])
        except ValueError:
            self.param_groups.pop()
            raise

    @staticmethod
    def weights_of(module):
        """(weights for Muon, the other parameters) of a module, e.g. model.PolicyValueNet."""
        params = list(module.parameters())
        return [p for p in params if p.dim() >= 2], [p for p in params if p.dim() < 2]

    def load_state_dict(self, state_dict):
        loaded = []
        hook = self.register_load_state_dict_pre_hook(lambda _, state: loaded.append(state))  # (as other hooks leave it)
        try:
            super().load_state_dict(state_dict)
        finally:
            hook.remove()
        # the base class gives what it loads the weight's type: m again, in float32
        numbers = [i for group in loaded[-1]["param_groups"] for i in group["params"]]
        for i, p in zip(numbers, (p for group in self.param_groups for p in group["params"])):
            m = loaded[-1]["state"].get(i, {}).get("momentum")
            if m is not None:
                self.state[p]["momentum"] = m.detach().to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = [(group, [p for p in group["params"] if p.grad is not None and p.numel()]) for group in self.param_groups]
        for group, params in groups:  # what is refused is refused before anything has changed
            _check_options(group, read=False)
            for p in params:
                if p.grad.layout != torch.strided:
                    _refuse("Muon takes no sparse gradients")
                if p.dtype not in TYPES:
                    _refuse(f"weights must be float32, bfloat16 or float16, not {p.dtype}")
            _on_gpu(params)
        for group, params in groups:
            if not params:
                continue
            grads = [p.grad.float() for p in params]  # (float32 ones are these themselves, and so are the weights below)
            for p, g in zip(params, grads):
                if "momentum" not in self.state[p]:
                    self.state[p]["momentum"] = torch.zeros_like(g)
            moments = [self.state[p]["momentum"] for p in params]
            mu = group["momentum"]
            torch._foreach_mul_(moments, mu)
            torch._foreach_add_(moments, grads)
            updates = torch._foreach_add(grads, moments, alpha=mu) if group["nesterov"] else moments
            updates = orthogonalise(updates, group["steps"])
            weights = [p.float() for p in params]
            if group["weight_decay"]:
                torch._foreach_mul_(weights, 1 - group["lr"] * group["weight_decay"])
            factors = [-group["lr"] * max(1.0, p.shape[0] * p.shape[0] / p.numel()) ** 0.5 for p in params]
            torch._foreach_mul_(updates, factors)
            torch._foreach_add_(weights, updates)
            for p, w in zip(params, weights):
                if w is not p:
                    p.copy_(w)
        return loss
