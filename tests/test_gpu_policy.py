"""The policy-row operators (alphazero_amd.policy) against their definitions in 64 bits, over sizes on both sides of every
width the kernels have, masks that leave rows empty, and strides.

Tolerances (u = 2^-24, half a step of float32).  An exponential e^d carries |d| u (the difference) + 1.5 |d| u (the scaled
exponent) + 2 u; a row's sum adds one u per addition in a lane (A / 64 cells) and 12 across the wavefront and the
chunks, so log S is off by at most (2.5 D + 16 + A / 64) u with D = sum p |d| <= H + log S, and log p = d - log S by
that plus 2 (|d| + log S) u.  H and the gradients are sums of p times those.  A result of 16 bits adds half a step of
its type (and half of float16's smallest step)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# one lane, both sides of each register width, the board sizes, the last short row, long rows with ragged chunks
SIZES = [1, 2, 25, 63, 64, 65, 169, 225, 256, 257, 361, 400, 513, 700, 1024, 1025, 4099, 50021]


def _inputs(rows, actions, dtype, mask, seed):
    g = torch.Generator().manual_seed(seed)
    x = (3 * torch.randn(rows, actions, generator=g)).to(dtype)
    if actions > 3:
        x[:, actions // 2] = x[:, 1]  # equal logits far apart
    legal = torch.rand(rows, actions, generator=g) > torch.rand(rows, 1, generator=g)
    legal[0] = False                  # an empty row
    if rows > 1:
        legal[1] = False
        legal[1, actions - 1] = True  # one legal cell, the last
    if mask == "none":
        legal[:] = True
    x = torch.where(legal, x, torch.tensor([math.inf, math.nan, -math.inf, torch.finfo(dtype).min], dtype=dtype)[
        torch.randint(0, 4, (rows, actions), generator=g)])  # masked places hold anything
    return x, legal


def _mask_args(mask, legal, seed):
    if mask == "none":
        return {}
    if mask == "legal":
        return {"legal": legal.cuda()}
    side = math.isqrt(legal.shape[1])
    who = torch.rand(legal.shape, generator=torch.Generator().manual_seed(seed)) < 0.5
    return {"board": torch.stack([~legal & who, ~legal & ~who], 1).float().view(-1, 2, side, side).cuda()}


def _exact(x, legal):
    """log p (-inf where masked or -inf), p, M, log S, in float64."""
    x = torch.where(legal, x.double(), -math.inf)
    M = x.max(1, keepdim=True).values
    d = torch.where(x == -math.inf, -math.inf, x - M)
    S = d.exp().sum(1, keepdim=True)
    logS = torch.where(S > 0, S.log(), 0.0)
    return d - logS, torch.where(S > 0, d.exp() / S, 0.0), d, logS


def _sum_tol(p, d, logS, actions):  # error of log S
    D = torch.where(p > 0, p * d.abs(), 0.0).sum(1, keepdim=True)
    return (2.5 * D + 16 + actions / 64) * U


def _ok(got, want, tol, what):
    got, want, tol = got.detach().cpu().double(), want.double(), torch.as_tensor(tol, dtype=torch.float64).expand(want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs())
    bad = ~(off <= tol)
    assert not bad.any(), (what, bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist(), tol[bad][:4].tolist())


CASES = [(a, TYPES[i % 3], m) for i, a in enumerate(SIZES) for m in ("none", "legal")] + \
        [(a, t, "board") for a in (25, 169, 225, 361, 400, 1089) for t in TYPES]


@pytest.mark.parametrize("actions,dtype,mask", CASES)
def test_score_and_its_gradient(actions, dtype, mask):
    from alphazero_amd import policy

    rows = 37 if actions < 10000 else 5
    x, legal = _inputs(rows, actions, dtype, mask, actions)
    kw = _mask_args(mask, legal, 1)
    g = torch.Generator().manual_seed(7)
    m, top = 3, 8
    moves = torch.randint(0, actions, (rows, m), generator=g, dtype=torch.int64)
    moves[:, 2] = moves[:, 0]          # the same move twice
    moves[-1, 1] = -1                  # none
    if rows > 2:
        moves[2, 0] = actions + 5      # past the end
    xg = x.cuda().requires_grad_()
    s = policy.score(xg, moves.cuda(), top=top, **kw)
    logp, p, d, logS = _exact(x, legal)
    inside = (moves >= 0) & (moves < actions)
    at = moves.clamp(0, actions - 1)
    want = torch.where(inside, logp.gather(1, at), torch.where(moves < 0, 0.0, math.nan))
    tS = _sum_tol(p, d, logS, actions)
    dm = torch.where(d.gather(1, at) == -math.inf, 0.0, d.gather(1, at).abs())
    _ok(s.logp, want, tS + 3 * (dm + logS) * U, "logp")
    plogp = torch.where(p > 0, p * logp, 0.0)
    H = -plogp.sum(1, keepdim=True)
    pd = torch.where(p > 0, p * d.abs(), 0.0)
    tH = 2 * tS + (pd.abs() * (2.5 * torch.where(p > 0, d.abs(), 0.0) + 20 + actions / 64)).sum(1, keepdim=True) * U + 2 * (H.abs() + logS) * U
    _ok(s.entropy, H.squeeze(1), tH.squeeze(1), "entropy")
    # alternatives: by value, then by lowest index
    for i in range(rows):
        row = torch.where(legal[i], x[i].double(), -math.inf).numpy()
        order = [j for j in np.lexsort((np.arange(actions), -row)) if row[j] > -np.inf][:top]
        assert s.top_moves[i].tolist() == order + [-1] * (top - len(order)), i
        wanted = torch.full((top,), -math.inf, dtype=torch.float64)
        wanted[:len(order)] = logp[i, order]
        _ok(s.top_logp[i], wanted, torch.nn.functional.pad(tS[i] + 3 * (d[i, order].abs() + logS[i]) * U, (0, top - len(order))), "top_logp")
    # gradient
    gl, gh = torch.randn(rows, m, generator=g), torch.randn(rows, generator=g)
    dx, = torch.autograd.grad((s.logp, s.entropy), xg, (gl.cuda(), gh.cuda()))
    assert dx.dtype == dtype and dx.shape == x.shape
    use = torch.where(inside & (logp.gather(1, at) > -math.inf), gl.double(), 0.0)
    G, aG = use.sum(1, keepdim=True), use.abs().sum(1, keepdim=True)
    k = torch.where(p > 0, p * (logp + H), 0.0)
    wx = -p * G - gh.double().unsqueeze(1) * k
    wx.scatter_add_(1, at, use)
    lp = torch.where(p > 0, logp.abs(), 0.0)
    rel = (6 * lp + 8) * U + 2 * tS  # error of p, relative
    tol = p * rel * aG + gh.abs().double().unsqueeze(1) * (k.abs() * (rel + 4 * U) + p * (tS + tH + 4 * (lp + H) * U)) + 8 * U * aG
    tol = tol + (wx.abs() + tol) * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype == torch.float16 else 0)
    _ok(dx, wx, tol, "d_logits")
    assert (dx.cpu()[~legal] == 0).all()


@pytest.mark.parametrize("rows", [1, 3, 4, 5, 9000])
def test_rows_left_over_and_more_rows_than_the_grid(rows):
    from alphazero_amd import policy

    x = torch.randn(rows, 25, generator=torch.Generator().manual_seed(rows)).cuda()
    s = policy.score(x, torch.full((rows,), 3, dtype=torch.int32, device="cuda"), top=1)
    want = torch.log_softmax(x.double(), 1)
    _ok(s.logp, want[:, 3].cpu(), 60 * U, "logp")
    assert torch.equal(s.top_moves[:, 0].long(), x.argmax(1))


def test_strides_broadcast_masks_and_empty_batches():
    from alphazero_amd import policy

    base = torch.randn(20, 300, generator=torch.Generator().manual_seed(0)).cuda()
    legal = torch.rand(225, device="cuda") < 0.5
    mv = torch.arange(20, device="cuda", dtype=torch.int32)
    dense = base[:, 40:265].contiguous()
    want = policy.score(dense, mv, legal=legal.expand(20, 225).contiguous(), top=4)
    for x in (base[:, 40:265], dense.t().contiguous().t(), torch.stack([dense, dense], 2)[:, :, 0]):
        for lg in (legal, legal.unsqueeze(0), legal.expand(20, 225), legal.to(torch.uint8) * 7):
            got = policy.score(x, mv, legal=lg, top=4)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = policy.score(dense[:1].expand(20, 225), mv, legal=legal)
    assert torch.equal(one.entropy, want.entropy[:1].expand(20))
    # strided rows through the gradient, moves as a strided int64 column
    x1, x2 = base.clone().requires_grad_(), dense.clone().requires_grad_()
    m64 = torch.stack([mv, mv], 1).long()[:, 1]
    policy.score(x1[:, 40:265], m64, legal=legal).logp[legal[mv.long()]].sum().backward()
    policy.score(x2, mv, legal=legal).logp[legal[mv.long()]].sum().backward()
    assert torch.equal(x1.grad[:, 40:265], x2.grad) and not x1.grad[:, :40].any()
    empty = policy.score(base[:0], mv[:0], top=2)
    assert empty.logp.shape == (0,) and empty.top_moves.shape == (0, 2)
    e = torch.empty(0, 9, device="cuda", requires_grad=True)
    policy.loss(e, e[:, 0], e.detach(), e.detach()[:, 0]).backward()
    assert e.grad.shape == (0, 9)


def test_special_values():
    from alphazero_amd import policy

    inf, nan = math.inf, math.nan
    low = torch.finfo(torch.float32).min
    x = torch.tensor([[-inf, -inf, -inf], [low, low, low], [nan, 0, 1], [inf, 0, 1], [-inf, 5, -inf], [3e38, -3e38, 0],
                      [nan, nan, nan]], device="cuda")
    mv = torch.tensor([0, 1, 1, 1, 1, 0, 2], device="cuda")
    x.requires_grad_()
    s = policy.score(x, mv, top=2)
    assert s.top_moves.tolist() == [[-1, -1], [0, 1], [2, 1], [0, 2], [1, -1], [0, 2], [-1, -1]]
    lp, h = s.logp.tolist(), s.entropy.tolist()
    assert lp[0] == -inf and abs(lp[1] + math.log(3)) < 1e-6 and lp[4] == 0 and lp[5] == 0
    assert h[0] == 0 and abs(h[1] - math.log(3)) < 1e-6 and h[4] == 0 and h[5] == 0
    assert all(math.isnan(lp[i]) and math.isnan(h[i]) for i in (2, 6)) and math.isnan(h[3])
    (g,) = torch.autograd.grad(s.logp[[0, 1, 4, 5]].sum() + s.entropy[[0, 1, 4, 5]].sum(), x)
    assert torch.isfinite(g[[0, 1, 4, 5]]).all() and not g[0].any() and not g[4].any()
    # a NaN that is masked is not looked at
    legal = torch.tensor([False, True, True], device="cuda")
    t = policy.score(x.detach()[2:3], mv[2:3], legal=legal)
    assert abs(t.logp.item() + math.log1p(math.e)) < 1e-6


def test_values_at_the_ends_of_the_range_in_long_rows():
    # differences that leave float32's range, between chunks and between steps of a chunk
    from alphazero_amd import policy

    x = torch.full((2, 70000), -3e38, device="cuda")
    x[0, 69999] = 3e38
    x[1, 5], x[1, 40000], x[1, 3000] = 3e38, 3e38, -math.inf
    pi = torch.zeros(2, 70000, device="cuda")
    pi[0, 69999], pi[1, 5], pi[1, 40000] = 1.0, 0.5, 0.5
    s = policy.score(x, torch.tensor([[69999, 0], [5, 3000]], device="cuda"), top=3)
    assert s.top_moves.tolist() == [[69999, 0, 1], [5, 40000, 0]]
    assert s.logp[0, 0] == 0 and s.logp[0, 1] == -math.inf and s.logp[1, 1] == -math.inf
    assert abs(s.logp[1, 0].item() + math.log(2)) < 1e-6 and s.entropy[0] == 0 and abs(s.entropy[1].item() - math.log(2)) < 1e-6
    x.requires_grad_()
    v = torch.zeros(2, device="cuda")
    total = policy.loss(x, v, pi, v)
    d, = torch.autograd.grad(total, x)
    assert abs(total.item()) < 1e-6 and not d.any()


def _loss_inputs(rows, actions, dtype, mask, seed):
    x, legal = _inputs(rows, actions, dtype, mask, seed)
    g = torch.Generator().manual_seed(seed + 1)
    pi = torch.rand(rows, actions, generator=g) ** 8
    pi[torch.rand(rows, actions, generator=g) < 0.5] = 0
    pi = pi / pi.sum(1, keepdim=True).clamp(min=1e-6)
    pi[~legal] = math.nan
    v = torch.tanh(torch.randn(rows, generator=g))
    r = torch.where(torch.rand(rows, generator=g) < 0.5, 1.0, -1.0)
    return x, legal, pi, v, r


@pytest.mark.parametrize("actions,dtype,mask", CASES)
@pytest.mark.parametrize("scale", [1.0, 1024.0])
def test_loss_and_its_gradients(actions, dtype, mask, scale):
    from alphazero_amd import policy

    rows = 37 if actions < 10000 else 5
    x, legal, pi, v, r = _loss_inputs(rows, actions, dtype, mask, actions)
    v = v.to(dtype) if actions % 2 else v
    kw = _mask_args(mask, legal, 1)
    xg, vg = x.cuda().requires_grad_(), v.cuda().view(rows, 1, 1, 1).requires_grad_()
    total, part_p, part_v = policy.loss(xg, vg, pi.cuda(), r.cuda(), parts=True, **kw)
    dx, dv = torch.autograd.grad(total * scale, (xg, vg))
    assert dx.dtype == dtype and dv.dtype == v.dtype and dv.shape == vg.shape
    logp, p, d, logS = _exact(x, legal)
    q = torch.where(legal & (x != -math.inf), pi.double(), 0.0)
    terms = torch.where(q > 0, q * (torch.log(q) - logp), 0.0)
    tS = _sum_tol(p, d, logS, actions)
    # each term: pi times the errors of log pi (2 u and u relative) and of log p, and the sum's additions
    mag = torch.where(q > 0, q * (torch.log(q).abs() + logp.abs() + 1), 0.0)
    dd = torch.where(q > 0, d.abs(), 0.0)
    tol = ((q * (tS + 3 * (dd + logS) * U)) + mag * (8 + actions / 64) * U).sum(1)
    want_p, want_v = terms.sum() / rows, ((v.double() - r.double()) ** 2).sum() / rows
    _ok(part_p, want_p, tol.sum() / rows + want_p.abs() * U, "policy part")
    _ok(part_v, want_v, 4 * U * want_v, "value part")
    _ok(total, want_p + want_v, tol.sum() / rows + 6 * U * (want_p.abs() + want_v), "total")
    W = q.sum(1, keepdim=True)
    f = scale / rows
    wx = torch.where(legal & (x != -math.inf), (p * W - q) * f, 0.0)
    lp = torch.where(p > 0, d.abs(), 0.0)
    t = (p * W * ((4 * lp + 24 + actions / 32) * U + tS) + 4 * U * (p * W + q)) * f
    t = t + (wx.abs() + t) * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype == torch.float16 else 0)
    _ok(dx, wx, t, "d_logits")
    wv = 2 * (v.double() - r.double()) * f
    _ok(dv.view(rows), wv, wv.abs() * (torch.finfo(v.dtype).eps / 2 + 6 * U) + (2.0 ** -25 if v.dtype == torch.float16 else 0), "d_value")


def test_loss_backward_twice_with_other_factors():
    # the forward pass's gradients are handed out once; later passes compute their own
    from alphazero_amd import policy

    x, legal, pi, v, r = (t.cuda() for t in _loss_inputs(50, 225, torch.float16, "none", 3))
    x.requires_grad_()
    v.requires_grad_()
    total = policy.loss(x, v, pi, r)
    first = torch.autograd.grad(total, (x, v), retain_graph=True)
    kept = [t.clone() for t in first]
    again = torch.autograd.grad(total, (x, v), retain_graph=True)
    big = torch.autograd.grad(total, (x, v), torch.tensor(4096.0, device="cuda"), retain_graph=True)
    only, = torch.autograd.grad(policy.loss(x.detach(), v, pi, r) * 1.0, v)
    assert all(torch.equal(a, b) for a, b in zip(first, kept)) and all(torch.equal(a, b) for a, b in zip(again, kept))
    assert torch.equal(only, kept[1])
    # float16 keeps more of the small gradients when the factor acts before the rounding
    exact = (torch.softmax(x.detach().double(), 1) - pi) / 50
    off = lambda g, f: ((g.double() / f - exact).norm() / exact.norm()).item()  # noqa: E731
    assert off(big[0], 4096.0) < 2.0 ** -11 < off(torch.full_like(big[0], 0), 1.0)
    assert off(big[0], 4096.0) <= off(kept[0], 1.0)


def test_gradients_against_differences():
    from alphazero_amd import policy

    x, legal, pi, v, r = _loss_inputs(4, 30, torch.float32, "legal", 11)
    pi = torch.where(legal, pi, 0.0)
    mv = torch.tensor([[1, 2], [29, 29], [5, -1], [7, 7]])
    w, h = torch.randn(4, 2), torch.randn(4)
    x = torch.where(legal, x, 0.0)

    def both(x):
        logp, p, _, _ = _exact(x, legal)
        hit = torch.where(mv >= 0, logp.gather(1, mv.clamp(min=0)), 0.0)
        hit = torch.where(hit == -math.inf, 0.0, hit)
        H = -torch.where(p > 0, p * logp, 0.0).sum(1)
        kl = torch.where(pi > 0, pi * (torch.log(pi.double()) - logp), 0.0).sum() / 4
        return (hit * w).sum() + (H * h).sum() + kl

    xg = x.cuda().requires_grad_()
    s = policy.score(xg, mv.cuda(), legal=legal.cuda())
    logp = torch.where(s.logp == -math.inf, 0.0, s.logp)
    f = (logp * w.cuda()).sum() + (s.entropy * h.cuda()).sum() + policy.loss(xg, r.cuda(), pi.cuda(), r.cuda(), legal=legal.cuda())
    got, = torch.autograd.grad(f, xg)
    step = 1e-4
    for i in range(4):
        for j in range(0, 30, 3):
            e = torch.zeros(4, 30, dtype=torch.float64)
            e[i, j] = step
            diff = (both(x.double() + e) - both(x.double() - e)) / (2 * step)
            # central differences are off by step^2 / 6 times a third derivative of at most a few tens; float32 by 100 u
            assert abs(got[i, j].item() - diff.item()) < 1e-6 + 100 * U * (1 + abs(diff.item())), (i, j)


def test_streams_and_graph_replay():
    # a captured forward and backward pass, replayed on new contents between eager passes, gives the eager results
    from alphazero_amd import policy

    g = torch.Generator(device="cuda").manual_seed(5)
    n, a = 300, 225
    x = torch.randn(n, a, generator=g, device="cuda").requires_grad_()
    v = torch.randn(n, generator=g, device="cuda").requires_grad_()
    pi = torch.softmax(torch.randn(n, a, generator=g, device="cuda"), 1)
    r = torch.randn(n, generator=g, device="cuda")
    long_x = torch.randn(3, 5000, generator=g, device="cuda").requires_grad_()
    mv = torch.randint(0, a, (n,), generator=g, device="cuda")

    def work():
        total = policy.loss(x, v, pi, r)
        s = policy.score(x, mv, top=3)
        l = policy.score(long_x, mv[:3], top=3)
        gx, gv, gl = torch.autograd.grad((total, s.logp.sum(), s.entropy.sum(), l.entropy.sum()), (x, v, long_x))
        return [total.detach(), s.logp.detach(), s.top_moves, l.top_logp, gx, gv, gl]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [t.clone() for t in work()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(work(), on_side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for k in range(3):
        with torch.no_grad():
            x.mul_(0.5).add_(k)
            pi.copy_(pi.flip(1))
            long_x.add_(torch.randn(3, 5000, generator=g, device="cuda"))
        want = [t.clone() for t in work()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), k


def test_evaluators_score_positions():
    from alphazero_amd import policy
    from alphazero_amd.evaluator import FusedNetEvaluator, TorchEvaluator
    from alphazero_amd.model import PolicyValueNet

    torch.manual_seed(0)
    net = PolicyValueNet(15).eval()
    boards = torch.zeros(6, 2, 225)
    for i in range(6):
        at = torch.randperm(225, generator=torch.Generator().manual_seed(i))[:12 * i]
        boards[i, 0, at[::2]] = 1
        boards[i, 1, at[1::2]] = 1
    boards = boards.view(6, 2, 15, 15).cuda()
    mv = torch.arange(6, device="cuda")
    for ev in (FusedNetEvaluator(net, 15), TorchEvaluator(net)):
        value, s = ev.score(boards, mv, top=5)
        v2, logp = ev(boards)
        assert torch.equal(value, v2)
        free = boards.sum(1).flatten(1) == 0
        want = torch.log_softmax(logp.double().masked_fill(~free, -math.inf), 1)
        _ok(s.logp, want.gather(1, mv.unsqueeze(1)).squeeze(1).cpu(), 200 * U, "logp")
        best = want.sort(dim=1, descending=True, stable=True)
        _ok(s.top_logp, best.values[:, :5].cpu(), 200 * U, "top_logp")
        assert free.gather(1, s.top_moves.long()).all()
    # the network's own loss: its heads through policy.loss, gradients in every parameter
    net = net.cuda().train()
    pi = torch.softmax(torch.randn(6, 225, device="cuda"), 1)
    r = torch.tensor([1.0, -1, 1, -1, 1, 1e-3], device="cuda")
    total = net.loss(boards, pi, r)
    total.backward()
    value, logits = net.heads(boards)
    want = torch.nn.functional.kl_div(torch.log_softmax(logits, 1), pi, reduction="batchmean") + \
        torch.nn.functional.mse_loss(value.view(-1), r)
    assert abs(total.item() - want.item()) < 1e-4 * abs(want.item())
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in net.parameters())


def test_nothing_is_computed_for_gradients_without_grad_mode_and_only_once():
    from alphazero_amd import policy

    x, legal, pi, v, r = (t.cuda() for t in _loss_inputs(20, 225, torch.float32, "none", 9))
    x.requires_grad_()
    mv = torch.arange(20, device="cuda")
    with torch.no_grad():
        total, part_p, part_v = policy.loss(x, v, pi, r, parts=True)
        s = policy.score(x, mv)
    assert not total.requires_grad and not s.logp.requires_grad
    with_grad = policy.loss(x, v, pi, r)
    assert torch.equal(with_grad.detach(), total)
    assert abs((part_p + part_v - total).item()) <= 4 * U * abs(total.item())
    for f in (with_grad, policy.score(x, mv).logp.sum()):
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(f, x, create_graph=True)


def test_saved_tensors_moved_by_a_hook():
    # activation offloading hands other tensors to the backward pass than the forward pass was given
    from alphazero_amd import policy

    x, legal, pi, v, r = (t.cuda() for t in _loss_inputs(30, 225, torch.float32, "legal", 4))
    x = torch.where(legal, x, 0.0)
    wide = torch.zeros(30, 300, device="cuda")
    wide[:, 10:235] = x
    mv = torch.arange(30, device="cuda")

    def grads(leaf, rows):
        s = policy.score(rows, mv, legal=legal)
        total = policy.loss(rows, v, pi, r, legal=legal)
        return lambda: torch.autograd.grad(total + (s.entropy * 0.1).sum(), leaf)[0]

    a = x.clone().requires_grad_()
    want = grads(a, a)()
    b = wide.clone().requires_grad_()
    with torch.autograd.graph.save_on_cpu():
        later = grads(b, b[:, 10:235])
    junk = [torch.full((30, 300), math.nan, device="cuda") for _ in range(8)]
    assert torch.equal(later()[:, 10:235], want)
    del junk


def test_two_streams_at_once():
    from alphazero_amd import policy

    g = torch.Generator(device="cuda").manual_seed(2)
    xs = [torch.randn(4000, 361, generator=g, device="cuda"), torch.randn(40, 30000, generator=g, device="cuda")]
    mv = [torch.randint(0, t.shape[1], (t.shape[0],), generator=g, device="cuda") for t in xs]
    want = [policy.score(t, m, top=8) for t, m in zip(xs, mv)]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            got.append(policy.score(xs[k % 2], mv[k % 2], top=8))
    torch.cuda.synchronize()
    for k, s in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(s, want[k % 2])), k


@pytest.mark.parametrize("actions", [5, 225, 1024, 1500, 70000])
@pytest.mark.parametrize("dtype", TYPES)
def test_loss_where_a_legal_move_has_no_probability(actions, dtype):
    # A legal cell at -inf has log-probability -inf: a target there makes the loss infinite (as torch's own kl_div), none
    # adds nothing.  Its gradient is p sum pi - pi with p = 0.  A cell that is not legal is not looked at at all.
    from alphazero_amd import policy

    rows, last = 6, actions - 1
    g = torch.Generator().manual_seed(actions)
    x = torch.randn(rows, actions, generator=g)
    pi = torch.rand(rows, actions, generator=g)
    pi /= pi.sum(1, keepdim=True)
    legal = torch.ones(rows, actions, dtype=torch.bool)
    x[0, last] = -math.inf                                 # a target that cannot be reached
    x[1, 1], pi[1, 1] = -math.inf, 0.0                     # the same without a target
    legal[2, last], x[2, last], pi[2, last] = False, -math.inf, 0.5
    x[3] = -math.inf                                       # every legal cell
    x[4], pi[4] = -math.inf, 0.0
    legal[5] = False                                       # a full board
    x = x.to(dtype)
    xg = x.cuda().requires_grad_()
    v = torch.zeros(rows, device="cuda")
    parts = [policy.loss(xg[i:i + 1], v[:1], pi[i:i + 1].cuda(), v[:1], legal=legal[i:i + 1].cuda(), parts=True)[1].item()
             for i in range(rows)]
    total = policy.loss(xg, v, pi.cuda(), v, legal=legal.cuda())
    dx, = torch.autograd.grad(total, xg)
    logp, p, d, logS = _exact(x, legal)
    q = torch.where(legal, pi.double(), 0.0)
    terms = torch.where(q > 0, q * (torch.log(q) - logp), 0.0)
    tS = _sum_tol(p, d, logS, actions)
    dd = torch.where((q > 0) & legal & (d > -math.inf), d.abs(), 0.0)
    mag = torch.where(q > 0, q * (torch.log(q).abs() + dd + logS + 1), 0.0)
    tol = (q * (tS + 3 * (dd + logS) * U) + mag * (8 + actions / 64) * U).sum(1)
    _ok(torch.tensor(parts), terms.sum(1), tol + terms.sum(1).nan_to_num(posinf=0.0).abs() * U, "parts")
    assert [math.isinf(t) for t in parts] == [True, False, False, True, False, False] and total.item() == math.inf
    assert parts[4] == 0 and parts[5] == 0
    W = q.sum(1, keepdim=True)
    wx = torch.where(legal, p * W - q, 0.0) / rows
    t = (p * W * ((4 * dd + 24 + actions / 32) * U + tS) + 4 * U * (p * W + q)) / rows
    t = t + (wx.abs() + t) * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype == torch.float16 else 0)
    _ok(dx, wx, t, "d_logits")
    assert not dx[5].any() and dx[2, last] == 0


@pytest.mark.parametrize("actions", [9, 225, 3000])
def test_loss_of_the_smallest_targets(actions):
    # subnormal float32 targets (a softmax far from its peak) count for what they are
    from alphazero_amd import policy

    g = torch.Generator().manual_seed(actions)
    x = torch.randn(3, actions, generator=g)
    pi = torch.softmax(torch.randn(3, actions, generator=g), 1)
    tiny = torch.tensor([2.0 ** -149, 1e-42, 1e-39, 2.0 ** -126])
    pi[0, :4] = tiny                                       # among ordinary ones
    pi[1] = tiny[torch.randint(0, 4, (actions,), generator=g)]  # and alone
    v = torch.zeros(3, device="cuda")
    parts = torch.stack([policy.loss(x[i:i + 1].cuda(), v[:1], pi[i:i + 1].cuda(), v[:1], parts=True)[1] for i in range(3)])
    logp, p, d, logS = _exact(x, torch.ones_like(x, dtype=torch.bool))
    q = pi.double()
    terms = q * (torch.log(q) - logp)
    tS = _sum_tol(p, d, logS, actions)
    mag = q * (torch.log(q).abs() + logp.abs() + 1)
    tol = (q * (tS + 3 * (d.abs() + logS) * U) + mag * (8 + actions / 64) * U).sum(1) + 2 * actions * 2.0 ** -149
    _ok(parts, terms.sum(1), tol + terms.sum(1).abs() * U, "parts")


def test_more_long_rows_than_a_launch_has_workgroups():
    # 2^24 workgroups of 256 threads are one thread too many for a launch; the rows around the seams are the ones that differ
    from alphazero_amd import policy

    n, a = (1 << 24) + 5, 1025
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 180 << 30:
        pytest.skip("180 GiB of free GPU memory needed")
    g = torch.Generator().manual_seed(6)
    at = torch.tensor([0, 1, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, (1 << 24) - 1, 1 << 24, n - 1])
    some = torch.randn(len(at), a, generator=g).half()
    moves = torch.zeros(n, dtype=torch.int32, device="cuda")
    moves[at.cuda()] = torch.arange(1, 9, dtype=torch.int32, device="cuda") * 100
    x = torch.zeros(n, a, dtype=torch.float16, device="cuda")
    x[at.cuda()] = some.cuda()
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[at.cuda()] = False
    x.requires_grad_()
    s = policy.score(x, moves, top=2)
    logp, p, d, logS = _exact(some, torch.ones_like(some, dtype=torch.bool))
    tS = _sum_tol(p, d, logS, a).squeeze(1)
    mine = (torch.arange(8), torch.arange(1, 9) * 100)
    _ok(s.logp[at.cuda()], logp[mine], tS + 3 * (d[mine].abs() + logS.squeeze(1)) * U, "logp")
    assert torch.equal(s.top_moves[at.cuda(), 0].cpu().long(), some.argmax(1))
    assert ((s.logp[rest] + math.log(a)).abs() <= 40 * U).all() and ((s.entropy[rest] - math.log(a)).abs() <= 80 * U).all()
    assert (s.top_moves[rest] == torch.tensor([0, 1], device="cuda")).all()
    dx, = torch.autograd.grad(s.logp, x, torch.ones(n, device="cuda"))
    want = -p
    want[mine] += 1
    _ok(dx[at.cuda()], want, want.abs() * (2.0 ** -11 + 60 * U) + 60 * U * p + 2.0 ** -25, "d_logits")
    ends = dx[rest][:: 1 << 18]
    assert ((ends[:, 0].float() - 1024 / 1025).abs() <= 2.0 ** -11).all() and ((ends[:, 1:].float() + 1 / 1025).abs() <= 2.0 ** -21).all()
    del dx, ends, s
    x = x.detach()
    pi = torch.zeros(n, a, device="cuda")
    pi[at.cuda(), moves[at.cuda()].long()] = 1.0
    v = torch.zeros(n, device="cuda")
    got = policy.loss(x, v, pi, v).double() * n
    off = (got.cpu() + logp[mine].sum()).abs()
    assert off <= (tS + 3 * (d[mine].abs() + logS.squeeze(1)) * U).sum() + 4 * U * logp[mine].sum().abs()
    del x, pi
    torch.cuda.empty_cache()


@pytest.mark.parametrize("actions", [225, 1089])
@pytest.mark.parametrize("mask", ["none", "legal", "board"])
def test_saved_tensors_laid_out_otherwise_by_a_hook(actions, mask):
    # a hook may hand back the same numbers with other strides; other types, sizes or devices are refused before a kernel runs
    from alphazero_amd import policy

    x, legal, pi, v, r = _loss_inputs(30, actions, torch.float32, mask, 4)
    kw = _mask_args(mask, legal, 1)
    x = torch.where(legal, x, 0.0).cuda().requires_grad_()
    pi, v, r = pi.cuda(), v.cuda().requires_grad_(), r.cuda()
    mv = torch.arange(30, device="cuda")

    def grads(unpack):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            s = policy.score(x, mv, **kw)
            total = policy.loss(x, v, pi, r, **kw)
        return [torch.autograd.grad(total, (x, v), torch.tensor(3.0, device="cuda")), torch.autograd.grad((s.entropy, s.logp), x, (r, v.detach()))]

    want = grads(lambda t: t)
    got = grads(lambda t: torch.stack([t, t], -1)[..., 0])
    assert all(torch.equal(p, q) for a, b in zip(want, got) for p, q in zip(a, b))
    for bad in (lambda t: t.cpu(), lambda t: t[:-1].clone(), lambda t: t.double() if t.is_floating_point() else t.short()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, bad):
            s = policy.score(x, mv, **kw)
            total = policy.loss(x, v, pi, r, **kw)
        for f in (total, s.entropy.sum()):
            with pytest.raises((RuntimeError, ValueError)):
                torch.autograd.grad(f, x)
    kept = x.data_ptr()
    for change in (lambda t: t.double() if t.dtype == torch.float32 and t.data_ptr() != kept else t,  # all but the logits
                   lambda t: t.cpu() if t.data_ptr() != kept else t):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            s = policy.score(x, mv, **kw)
            total = policy.loss(x, v, pi, r, **kw)
        for f in (total, s.entropy.sum()):
            with pytest.raises((RuntimeError, ValueError), match="hook|board|GPU of the logits"):
                torch.autograd.grad(f, x)


@pytest.mark.parametrize("actions", [225, 5000])
def test_c_entry_does_nothing_unless_scaled(actions):
    # every output stays as it was where the factor is 1, the loss too; with another factor all of them are written
    from alphazero_amd import engine as E

    L = E.load_library()
    x, legal, pi, v, r = (t.cuda() for t in _loss_inputs(9, actions, torch.float32, "none", 5))
    work = torch.empty(L.az_policy_loss_work(9, actions), dtype=torch.uint8, device="cuda").fill_(77)

    def call(scale, only, out):
        at = torch.tensor(scale, device="cuda")
        rc = L.az_policy_loss(9, actions, x.data_ptr(), 0, actions, None, None, 0, v.data_ptr(), 1, pi.data_ptr(), r.data_ptr(), at.data_ptr(),
                              only, *[t.data_ptr() for t in out], work.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        return [t.clone() for t in out]

    fresh = lambda: [torch.full(s, 7.0, device="cuda") for s in ((1,), (2,), (9, actions), (9,))]  # noqa: E731
    assert all((t == 7).all() for t in call(1.0, 1, fresh()))
    want = call(3.0, 0, fresh())
    assert all(torch.equal(a, b) for a, b in zip(call(3.0, 1, fresh()), want))
    plain = call(1.0, 0, fresh())
    assert torch.equal(plain[0], want[0]) and torch.equal(plain[1], want[1])  # (the factor is the gradients')


@pytest.mark.parametrize("actions,dtype", [(1 << 24, torch.float32), ((1 << 24) - 1, torch.float16)])
def test_the_longest_rows(actions, dtype):
    from alphazero_amd import policy

    g = torch.Generator(device="cuda").manual_seed(actions)
    x = (2 * torch.randn(2, actions, generator=g, device="cuda")).to(dtype)
    legal = torch.rand(actions, generator=g, device="cuda") < 0.7
    legal[-1] = True
    x[0, -1] = 30
    moves = torch.tensor([[actions - 1, 12345], [actions - 1, 12345]], device="cuda")
    x.requires_grad_()
    s = policy.score(x, moves, legal=legal, top=32)
    at = legal.nonzero().squeeze(1)
    xd = x.detach()[:, at].double()
    M = xd.max(1, keepdim=True).values
    logS = (xd - M).exp().sum(1, keepdim=True).log()
    p = (xd - M - logS).exp()
    tS = ((2.5 * (p * (xd - M).abs()).sum(1, keepdim=True) + 16 + actions / 64 / 256) * U).cpu()  # (256 chunks)
    got = x.detach().gather(1, moves).double()
    want = torch.where(legal[moves], got - M - logS, -math.inf)
    _ok(s.logp, want.cpu(), tS + 3 * ((got - M).abs() + logS).cpu() * U, "logp")
    ranked = xd.sort(dim=1, descending=True, stable=True)
    assert torch.equal(s.top_moves.long(), at[ranked.indices[:, :32]])
    H = -(p * (xd - M - logS)).sum(1)
    assert ((s.entropy - H).abs().cpu() <= 4 * tS.squeeze(1) * (1 + H.cpu())).all()
    dx, = torch.autograd.grad(s.logp[:, 0].sum(), x)
    want = torch.zeros_like(x, dtype=torch.float64)
    want[:, at] = -p
    want[:, -1] += 1
    tol = want.abs() * (torch.finfo(dtype).eps / 2 + 200 * U) + 4 * U + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert ((dx - want).abs() <= tol).all() and not dx[:, ~legal].any()


def test_evaluators_score_batches_of_none_and_strided_boards():
    from alphazero_amd.evaluator import FusedNetEvaluator, TorchEvaluator
    from alphazero_amd.model import PolicyValueNet

    torch.manual_seed(0)
    net = PolicyValueNet(9).eval()
    wide = torch.zeros(5, 2, 9, 12, device="cuda")
    wide[2, 1, 4, 5] = wide[3, 0, 0, 0] = 1
    boards, mv = wide[..., :9], torch.arange(5, device="cuda")
    for ev in (FusedNetEvaluator(net, 9), TorchEvaluator(net), TorchEvaluator(net, torch.device("cuda"))):
        value, s = ev.score(boards, mv, top=3)
        v2, want = ev.score(boards.contiguous(), mv, top=3)
        assert (value - v2).abs().max() < 1e-5 and (s.logp - want.logp).abs().max() < 1e-4
        value, s = ev.score(boards[:0].contiguous(), mv[:0], top=2)
        assert value.shape == (0,) and s.logp.shape == (0,) and s.top_moves.shape == (0, 2)


def test_under_checkpointing_and_inference_mode():
    from torch.utils.checkpoint import checkpoint

    from alphazero_amd import policy

    x, legal, pi, v, r = (t.cuda() for t in _loss_inputs(30, 225, torch.float32, "legal", 8))
    x = torch.where(legal, x, 0.0)
    w = (torch.eye(225, device="cuda") * 2).requires_grad_()
    mv = torch.arange(30, device="cuda")

    def f(w):
        rows = x @ w
        s = policy.score(rows, mv, legal=legal, top=2)
        return policy.loss(rows, v, pi, r, legal=legal) * 3 + s.entropy.sum()

    want, = torch.autograd.grad(f(w), w)
    for reentrant in (False, True):
        w.grad = None
        checkpoint(f, w, use_reentrant=reentrant).backward()
        assert torch.equal(w.grad, want)
    with torch.inference_mode():
        total = f(w)
    assert torch.equal(total, f(w).detach()) and not total.requires_grad
