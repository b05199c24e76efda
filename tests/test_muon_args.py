"""Refusals of the orthogonalised updates (alphazero_amd.muon and its C ABI), checked without a GPU."""
import ctypes as C

import pytest
import torch

from alphazero_amd import engine as E
from alphazero_amd import muon

G = torch.zeros(4, 9)


@pytest.mark.parametrize("updates,steps,text", [
    (G[0], 5, "a matrix, a batch"),
    (G.view(1, 1, 4, 9), 5, "a matrix, a batch"),
    (G.double(), 5, "float32, bfloat16 or float16"),
    ([G, G.double()], 5, "float32, bfloat16 or float16"),
    ([G, G[0]], 5, "two or more dimensions"),
    ([G, 3], 5, "two or more dimensions"),
    (G, 0, "steps must be"),
    (G, 21, "steps must be"),
    (G, 2.0, "steps must be"),
    (torch.empty(1, 1).expand(32769, 1), 5, "at most 32768"),
    (torch.empty(1, 1).expand(20000, 20000), 5, "cells"),
    (G, 5, "no CPU path"),
    ([G], 5, "no CPU path"),
])
def test_refuses(updates, steps, text):
    with pytest.raises(ValueError, match=text):
        muon.orthogonalise(updates, steps)


def test_c_entry_refuses():
    L = E.load_library()
    one = (C.c_void_p * 1)(0x1000)  # never looked at: the sizes are refused first
    none = (C.c_void_p * 1)(None)
    call = lambda count=1, rows=4, cols=9, a=one, lda=9, b=one, ldb=9, dt=0, steps=5, work=0x1000: \
        L.az_muon_orthogonalise(count, rows, cols, a, lda, b, ldb, dt, steps, work, None)  # noqa: E731
    assert call(count=0) == 0
    for bad in (dict(count=-1), dict(rows=0), dict(cols=0), dict(rows=32769), dict(rows=20000, cols=20000, lda=20000, ldb=20000),
                dict(a=None), dict(b=None), dict(a=none), dict(b=none), dict(lda=8), dict(ldb=8), dict(dt=3), dict(steps=0),
                dict(steps=21), dict(rows=100, cols=100, lda=100, ldb=100, work=None)):
        assert call(**bad) == E.ERR_ARG, bad
    assert L.az_muon_work(1, 100, 144) > 0 and L.az_muon_work(1, 16, 144) == 0 and L.az_muon_work(0, 16, 144) == 0 and L.az_muon_work(1, 0, 5) == -1


def test_optimiser_refuses():
    p = torch.nn.Parameter(torch.zeros(3, 3))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(steps=0)):
        with pytest.raises(ValueError):
            muon.Muon([p], **kw)
    with pytest.raises(ValueError, match="two or more"):
        muon.Muon([torch.nn.Parameter(torch.zeros(3))])


def test_optimiser_refuses_later_groups():
    opt = muon.Muon([torch.nn.Parameter(torch.zeros(3, 3))])
    for group in (dict(params=[torch.nn.Parameter(torch.zeros(3))]), dict(params=[torch.nn.Parameter(torch.zeros(2, 2))], steps=0),
                  dict(params=[torch.nn.Parameter(torch.zeros(2, 2, dtype=torch.float64))])):
        with pytest.raises(ValueError):
            opt.add_param_group(group)
        assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2, 5))], lr=0.1))
    assert len(opt.param_groups) == 2


def test_workspace_grows_with_the_batch_and_ends():
    L = E.load_library()
    one, many = L.az_muon_work(1, 100, 400), L.az_muon_work(200, 100, 400)
    assert one < 18 << 20 and many > 200 * 3 * 100 * 400 * 4  # (16 MiB of sums of shared tiles) one launch for all
    for shape in ((100, 400), (1000, 1000), (70, 20000)):
        assert L.az_muon_work(100000, *shape) <= (1 << 30) + 4096
    assert L.az_muon_work(3, 16384, 16384) > 0


def test_steps_end_where_the_precision_does():
    for steps in (11, 20):
        with pytest.raises(ValueError, match="steps must be 1..10"):
            muon.orthogonalise(G, steps)
        with pytest.raises(ValueError, match="steps must be 1..10"):
            muon.Muon([torch.nn.Parameter(torch.zeros(3, 3))], steps=steps)
        one = (C.c_void_p * 1)(0x1000)
        assert E.load_library().az_muon_orthogonalise(1, 4, 9, one, 9, one, 9, 0, steps, None, None) == E.ERR_ARG


def test_optimiser_checks_the_options_of_every_group():
    opt = muon.Muon([torch.nn.Parameter(torch.zeros(3, 3))])
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-0.1), dict(steps=0), dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2, 2))], **bad))
        with pytest.raises(ValueError):
            muon.Muon([dict(params=[torch.nn.Parameter(torch.zeros(2, 2))], **bad)])
        assert len(opt.param_groups) == 1


def test_a_refused_step_changes_nothing():
    # no path on the CPU, an option changed to one that is refused, gradients of a kind that is not taken
    def weight(grad=None):
        p = torch.nn.Parameter(torch.ones(3, 3))
        p.grad = torch.ones(3, 3) if grad is None else grad
        return p

    ok, late = weight(), weight()
    opt = muon.Muon([dict(params=[ok]), dict(params=[late])], lr=0.1, weight_decay=0.1)
    for i, change in ((0, {}), (1, dict(steps=11)), (1, dict(momentum=1.0)), (1, dict(lr=-1.0))):
        kept = dict(opt.param_groups[i])
        opt.param_groups[i].update(change)
        with pytest.raises(ValueError):
            opt.step()
        opt.param_groups[i].update(kept)
        assert not opt.state[ok] and not opt.state[late]
        assert torch.equal(ok.detach(), torch.ones(3, 3)) and torch.equal(late.detach(), torch.ones(3, 3))
    with pytest.raises(ValueError, match="sparse"):
        muon.Muon([weight(torch.ones(3, 3).to_sparse())]).step()
