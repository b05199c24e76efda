"""Refusals of the policy-row operators (alphazero_amd.policy and its C ABI): bad arguments raise before anything
reaches the GPU, so they are checked without one."""
import pytest
import torch

from alphazero_amd import engine as E
from alphazero_amd import policy

X = torch.zeros(4, 9)
PI, V, R = torch.zeros(4, 9), torch.zeros(4), torch.zeros(4)


@pytest.mark.parametrize("args,kw,text", [
    ((X[0],), {}, r"\[rows, actions\]"),
    ((X.double(),), {}, "float32, bfloat16 or float16"),
    ((X[:, :0],), {}, "at least 1 action"),
    ((X,), dict(board=torch.zeros(4, 2, 3, 3), legal=torch.ones(4, 9, dtype=torch.bool)), "not both"),
    ((X,), dict(board=torch.zeros(4, 2, 3, 3, dtype=torch.int8)), "board must be float32"),
    ((X,), dict(board=torch.zeros(4, 2, 4, 4)), "board must be float32"),
    ((X,), dict(board=torch.zeros(3, 2, 3, 3)), "board must be float32"),
    ((X,), dict(legal=torch.ones(4, 9)), "legal must be bool"),
    ((X,), dict(legal=torch.ones(4, 8, dtype=torch.bool)), "legal must be bool"),
    ((X, torch.zeros(4)), {}, "moves must be int32 or int64"),
    ((X, torch.zeros(3, dtype=torch.int32)), {}, "moves must be int32 or int64"),
    ((X, torch.zeros(4, 65, dtype=torch.int32)), {}, "at most 64 moves"),
    ((X, torch.zeros(4, 0, dtype=torch.int32)), {}, "at most 64 moves"),
    ((X,), dict(top=33), "top must be"),
    ((X,), dict(top=-1), "top must be"),
    ((X,), dict(top=1.0), "top must be"),
    ((X,), {}, "no CPU path"),
])
def test_score_refuses(args, kw, text):
    with pytest.raises(ValueError, match=text):
        policy.score(*args, **kw)


@pytest.mark.parametrize("args,text", [
    ((X, V[:3], PI, R), "value must hold 4"),
    ((X, V.double(), PI, R), "value must hold 4"),
    ((X, V.half(), PI, R), "value must hold 4"),
    ((X, V, PI[:, :8], R), "pi must be float32"),
    ((X, V, PI.half(), R), "pi must be float32"),
    ((X, V, PI, R[:2]), "r must hold 4"),
    ((X, V, PI, R.double()), "r must hold 4"),
    ((X, V, PI.clone().requires_grad_(), R), "detach"),
    ((X, V, PI, R), "no CPU path"),
])
def test_loss_refuses(args, text):
    with pytest.raises(ValueError, match=text):
        policy.loss(*args)


def test_c_entries_refuse():
    L = E.load_library()
    p = 0x1000  # never looked at: the sizes are refused first
    score = lambda n=1, a=9, dt=0, ld=9, board=None, legal=None, ldl=0, moves=p, mb=4, m=1, top=1: L.az_policy_score(  # noqa: E731
        n, a, p, dt, ld, board, legal, ldl, moves, mb, m, top, p, p, p, p, None, None, None, None)
    assert score(n=0) == 0
    for bad in (dict(n=-1), dict(a=0), dict(a=(1 << 24) + 1, ld=1 << 25), dict(dt=3), dict(dt=-1), dict(ld=8), dict(m=65),
                dict(m=-1), dict(top=33), dict(mb=2), dict(moves=None), dict(board=p, legal=p), dict(legal=p, ldl=8),
                dict(a=2000, ld=2000)):  # (a long row without a workspace)
        assert score(**bad) == E.ERR_ARG, bad
    assert L.az_policy_score_grad(1, 9, p, 0, 9, None, None, 0, None, p, 4, 1, p, p, None, p, p, None) == E.ERR_ARG
    assert L.az_policy_score_grad(1, 2000, p, 0, 2000, None, None, 0, p, p, 4, 1, p, None, None, p, p, None) == E.ERR_ARG
    loss = lambda n=1, scale=None, only=0, work=p: L.az_policy_loss(  # noqa: E731
        n, 9, p, 0, 9, None, None, 0, p, 1, p, p, scale, only, p, None, p, p, work, None)
    for bad in (dict(n=0), dict(only=1), dict(work=None)):
        assert loss(**bad) == E.ERR_ARG, bad
    assert L.az_policy_score_work(4, 400, 8) == 0 and L.az_policy_score_work(4, 4000, 8) > 0
    assert L.az_policy_score_work(-1, 400, 8) == -1 and L.az_policy_loss_work(1, 0) == -1
    assert [L.az_policy_mask_words(a) for a in (0, 1, 64, 65, 1024, 1025)] == [0, 1, 1, 2, 16, 0]


def test_forward_mode_derivatives_are_refused():
    # a tangent would be lost without a word, with and without grad mode
    import torch.autograd.forward_ad as fw

    with fw.dual_level():
        x, v, pi, r = (fw.make_dual(t, torch.ones_like(t)) for t in (X, V, PI, R))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    policy.score(x)
                for args in ((x, V, PI, R), (X, v, PI, R), (X, V, pi, R), (X, V, PI, r)):
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        policy.loss(*args)
        with pytest.raises(ValueError, match="no CPU path"):  # (nothing to lose)
            policy.score(X)


def test_traces_are_refused():
    # a trace keeps addresses, not tensors: its result on other inputs would be the first call's, or freed memory's
    from alphazero_amd import muon

    for f, args in ((policy.score, (X,)), (policy.loss, (X, V, PI, R)), (muon.orthogonalise, (X,))):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, args)


def test_c_entries_refuse_workspaces_off_their_alignment():
    import ctypes as C

    L = E.load_library()
    p, one = 0x1000, (C.c_void_p * 1)(0x1000)  # never looked at
    for off in (1, 4, 8):
        assert L.az_policy_score(1, 2000, p, 0, 2000, None, None, 0, None, 4, 0, 1, None, p, p, p, None, None, p + off, None) == E.ERR_ARG
        assert L.az_policy_loss(1, 9, p, 0, 9, None, None, 0, p, 1, p, p, None, 0, p, None, p, p, p + off, None) == E.ERR_ARG
        assert L.az_muon_orthogonalise(1, 100, 100, one, 100, one, 100, 0, 5, p + off, None) == E.ERR_ARG


def test_evaluators_refuse_boards_they_are_not_made_for():
    # the fused kernel reads n boards of its own size at an address on the GPU, whatever stands there
    from alphazero_amd.evaluator import FusedNetEvaluator, TorchEvaluator
    from alphazero_amd.model import PolicyValueNet

    net = PolicyValueNet(7).eval()
    good = torch.zeros(3, 2, 7, 7)
    for ev in (FusedNetEvaluator(net, 7, torch.device("cpu")), TorchEvaluator(net, torch.device("cpu"))):
        for bad in (good.double(), good.to(torch.uint8), good[:, :1], good[0], good[:, :, :6], good.tolist()):
            with pytest.raises(ValueError, match="boards must be float32"):
                ev.score(bad)
        with pytest.raises(ValueError, match="no CPU path"):
            ev.score(good)
    with pytest.raises(ValueError, match=r"\[n, 2, 7, 7\]"):
        FusedNetEvaluator(net, 7, torch.device("cpu")).score(torch.zeros(3, 2, 6, 6))
