"""Orthogonalised updates (alphazero_amd.muon) against the definition in 64 bits.

Tolerance: with u = 2^-24 a product of m x n matrices held in 22 bits (hi + lo, and the lo lo products left out) is off by
at most about 8 u of its operands' sizes, entry errors of random sign; a step multiplies what an earlier one left by at
most a = 3.4445, so the result's error is at most sum_{k < steps} a^k 8 u sqrt(terms that add up) of the input's
size.  The input's size is |X_0|_F = 1 and errors of random sign spread over its m directions, so relative to the
result's norm (about sqrt(rank)) the bound used is  a^(steps-1) * 1.41 * 32 u / sqrt(rank of the result)  plus 64 u for
the later steps' own roundings; a result of 16 bits adds half a step of its type relative to its norm."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ABC = (3.4445, -4.7750, 2.0315)


def _exact(g, steps=5):
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if tall else x
    norm = x.square().sum((-1, -2), keepdim=True).sqrt()
    x = torch.where(norm > 0, x / norm, 0.0)
    a, b, c = ABC
    for _ in range(steps):
        A = x @ x.transpose(-1, -2)
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.transpose(-1, -2) if tall else x


def _check(got, g, steps=5):
    want = _exact(g.cpu(), steps)
    assert got.shape == g.shape and got.dtype == g.dtype
    off = (got.cpu().double() - want).flatten(-2).norm(dim=-1)
    size = want.flatten(-2).norm(dim=-1)
    tol = ABC[0] ** (steps - 1) * 1.41 * 32 * U + size * (64 * U + (torch.finfo(g.dtype).eps / 2 if g.dtype != torch.float32 else 0))
    assert (off <= tol).all(), (off, tol, size)


def _updates(shape, seed, scale=1e-3, rank=None):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    m, n = shape[-2:]
    if rank is None:
        return rnd(*shape) * scale
    return (rnd(*shape[:-1], rank) @ rnd(*shape[:-2], rank, n)) * scale


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3), (16, 18), (16, 144), (144, 16), (31, 33), (32, 32), (33, 31), (63, 65), (64, 64), (64, 576),
          (65, 63), (128, 100), (129, 127), (130, 1000), (200, 64), (256, 2304), (333, 1201), (512, 40), (640, 640), (17, 4100)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_against_the_definition(shape, dtype):
    from alphazero_amd import muon

    g = _updates(shape, 1, 1e-2).to(dtype).cuda()
    _check(muon.orthogonalise(g), g)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 10])
@pytest.mark.parametrize("shape", [(16, 144), (100, 300), (300, 100)])
def test_numbers_of_steps(steps, shape):
    from alphazero_amd import muon

    g = _updates(shape, steps).cuda()
    _check(muon.orthogonalise(g, steps), g, min(steps, 7)) if steps <= 7 else None
    if steps == 10:  # the singular values of a well conditioned update stay in the band that the polynomial maps to itself
        s = torch.linalg.svdvals(muon.orthogonalise(g, 10).double().cpu())
        assert 0.6 < s.min() and s.max() < 1.25


@pytest.mark.parametrize("shape,dtype", [((2, 2048, 2100), torch.float32), ((1, 2050, 2300), torch.float32), ((2300, 2100), torch.bfloat16),
                                         ((1, 2600, 2500), torch.float16)])
def test_large_tiles_that_workgroups_share(shape, dtype):
    # a few tiles more than there are CUs (symmetric, two products at once, the last product in each type), and a few less
    from alphazero_amd import muon

    g = _updates(shape, 17).to(dtype).cuda()
    out = muon.orthogonalise(g, 4)
    assert torch.equal(out, muon.orthogonalise(g, 4))
    x = g.double()  # (the definition on the GPU, in 64 bits)
    x = x.transpose(-1, -2).contiguous() if x.shape[-2] > x.shape[-1] else x
    x = x / x.square().sum((-1, -2), keepdim=True).sqrt()
    for _ in range(4):
        A = x @ x.transpose(-1, -2).contiguous()
        x = ABC[0] * x + (ABC[1] * A + ABC[2] * (A @ A)) @ x
    x = x.transpose(-1, -2) if shape[-2] > shape[-1] else x
    off, size = (out.double() - x).flatten(-2).norm(dim=-1), x.flatten(-2).norm(dim=-1)
    tol = ABC[0] ** 3 * 1.41 * 32 * U + size * (64 * U + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0))
    assert (off <= tol).all(), (off, tol)


@pytest.mark.parametrize("shape", [(3, 64, 2304), (4608, 20), (300, 4000), (2, 129, 3000), (300, 33, 800), (2, 1500, 40), (1, 1050, 1400)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_gram_sums_and_large_tiles(shape, dtype):
    # K shared by several workgroups, with Q at once up to 64 rows, more matrices than CUs; tiles of 128
    from alphazero_amd import muon

    g = _updates(shape, 4).to(dtype).cuda()
    got = muon.orthogonalise(g)
    _check(got, g)
    assert torch.equal(got, muon.orthogonalise(g))


@pytest.mark.parametrize("count", [1, 2, 7, 63, 64, 65, 130])
def test_batches(count):
    from alphazero_amd import muon

    g = _updates((count, 16, 40), count).cuda()
    got = muon.orthogonalise(g)
    _check(got, g)
    assert torch.equal(got[count // 2], muon.orthogonalise(g[count // 2]))  # a matrix's result is its own


@pytest.mark.parametrize("shape", [(3, 130, 200), (2, 20, 50), (1, 700, 500)])
def test_low_rank_sizes_and_zeros(shape):
    from alphazero_amd import muon

    for scale in (1e-30, 1e-3, 1e25):
        g = _updates(shape, 3, 1.0, rank=4).cuda() * scale
        _check(muon.orthogonalise(g), g)
    g[0] = 0
    got = muon.orthogonalise(g)
    assert not got[0].any() and torch.isfinite(got).all()
    if shape[0] > 1:
        for bad in (math.nan, math.inf):
            g[1, 3, 5] = bad
            got = muon.orthogonalise(g)
            assert got[1].isnan().all() and not got[0].any()
            assert shape[0] < 3 or torch.isfinite(got[2]).all()


@pytest.mark.parametrize("shape", [(8, 16, 144), (8, 30, 600), (8, 64, 576), (2, 64, 4000), (2, 128, 1024), (1, 500, 2048),
                                   # whole tiles and stages, so that no padding hides a missing product: few and many workgroups
                                   (32, 192, 768), (300, 64, 1024), (3, 128, 256), (200, 128, 512), (5, 256, 1056), (1, 512, 2048),
                                   (1, 128, 8192), (8, 512, 1024), (2, 1024, 4096), (6, 384, 1536)])
def test_every_number_of_wide_matrices_has_float32_precision(shape):
    # The singular values of a wide random matrix lie close together, so no direction's error outgrows the others: five
    # steps of at most 8 u each (the bound above) and as much again for their mutual growth are 80 u.  One number of X or Q
    # kept to 11 bits instead of 22 would show: 2^-12 / sqrt(m n) of X, of many more where several are.
    from alphazero_amd import muon

    g = _updates(shape, 21)
    off = muon.orthogonalise(g.cuda()).cpu().double() - _exact(g)
    assert (off.flatten(-2).norm(dim=-1) <= 80 * U * _exact(g).flatten(-2).norm(dim=-1)).all()


@pytest.mark.parametrize("shape", [(5, 9), (48, 100), (100, 200)])
def test_the_smallest_numbers(shape):
    # subnormal float32 numbers: whole multiples of 2^-149
    from alphazero_amd import muon

    gen = torch.Generator().manual_seed(8)
    g = torch.ldexp(torch.randint(-300, 301, shape, generator=gen).float(), torch.tensor(-120)) * 2.0 ** -29
    assert 0 < g.abs().max() < 2.0 ** -126
    _check(muon.orthogonalise(g.cuda()), g)


def test_strides_lists_and_empty():
    from alphazero_amd import muon

    base = _updates((6, 50, 90), 5).cuda()
    want = muon.orthogonalise(base[:, 3:43, 7:80].contiguous())
    assert torch.equal(muon.orthogonalise(base[:, 3:43, 7:80]), want)
    assert torch.equal(muon.orthogonalise(base[::2, 3:43, 7:80]), want[::2])
    turned = base[:, 3:43, 7:80].transpose(1, 2).contiguous().transpose(1, 2)  # unit stride along the rows
    assert torch.equal(muon.orthogonalise(turned), want)
    assert torch.equal(muon.orthogonalise(base[:1, 3:43, 7:80].expand(4, 40, 73)), want[:1].expand(4, 40, 73))
    conv = _updates((16, 16 * 9), 6).cuda().view(16, 16, 3, 3)
    first = _updates((16, 2 * 9), 7).cuda().view(16, 2, 3, 3)
    dense = _updates((30, 20), 8).cuda().bfloat16()
    wide = base[0, :, :77]
    got = muon.orthogonalise([conv, first, dense, conv * 2, wide, torch.empty(0, 4, device="cuda")])
    assert [t.shape for t in got] == [conv.shape, first.shape, dense.shape, conv.shape, wide.shape, (0, 4)]
    for g, t in ((conv, got[0]), (first, got[1]), (dense, got[2]), (wide, got[4])):
        assert torch.equal(t.flatten(1), muon.orthogonalise(g.flatten(1)))
        _check(t.flatten(1), g.flatten(1))
    assert torch.equal(got[3], got[0])  # a factor of two does not change a single bit
    assert muon.orthogonalise([]) == [] and muon.orthogonalise(base[:0]).shape == (0, 50, 90)
    x = base[0].clone().requires_grad_()
    assert not muon.orthogonalise(x).requires_grad


def test_many_separate_tensors_and_odd_alignment():
    # more tensors than one launch's table of addresses holds, none of them evenly spaced; rows that start at any element
    from alphazero_amd import muon

    store = _updates((1, 400000), 12).cuda().flatten()
    at, many = 0, []
    for i in range(70):
        many.append(store[at:at + 64 * 70].view(64, 70))
        at += 64 * 70 + i % 5 + 1
    got = muon.orthogonalise(many)
    for i in (0, 1, 33, 63, 64, 69):
        _check(got[i], many[i])
        assert torch.equal(got[i], muon.orthogonalise(many[i]))
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        flat = store[:200003].to(dtype)
        for rows, cols, off in ((64, 129, 1), (129, 64, 3), (32, 65, 1), (130, 201, 1), (201, 130, 3)):
            g = flat[off:off + rows * (cols + 2)].view(rows, cols + 2)[:, 1:cols + 1]
            _check(muon.orthogonalise(g), g)


def test_in_place_through_the_c_entry():
    import ctypes as C

    from alphazero_amd import engine as E
    from alphazero_amd import muon

    L = E.load_library()
    for shape in ((3, 20, 50), (2, 100, 130)):
        g = _updates(shape, 14).cuda()
        want = muon.orthogonalise(g)
        work = torch.empty(max(1, L.az_muon_work(*shape)), dtype=torch.uint8, device="cuda")
        at = (C.c_void_p * shape[0])(*[t.data_ptr() for t in g])
        rc = L.az_muon_orthogonalise(*shape, at, shape[2], at, shape[2], 0, 5, work.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(g, want)


def test_two_streams_at_once():
    from alphazero_amd import muon

    gs = [_updates((2, 130, 300), 15).cuda(), _updates((9, 40, 300), 16).cuda()]
    want = [muon.orthogonalise(g) for g in gs]
    streams = [torch.cuda.Stream() for _ in gs]
    torch.cuda.synchronize()
    got = []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            got.append(muon.orthogonalise(gs[k % 2]))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[k % 2]) for k, t in enumerate(got))


def test_streams_and_graph_replay():
    from alphazero_amd import muon

    g = _updates((3, 100, 260), 9).cuda()
    small = _updates((5, 16, 144), 10).cuda()
    work = lambda: (muon.orthogonalise(g), muon.orthogonalise(small))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(work(), on_side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for k in range(3):
        g.add_(torch.randn_like(g) * 1e-3)
        small.mul_(1.5).add_(1e-4)
        want = [t.clone() for t in work()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_optimiser_step_by_step():
    from alphazero_amd import muon

    torch.manual_seed(0)
    w = [torch.nn.Parameter(torch.randn(16, 4, 3, 3, device="cuda")), torch.nn.Parameter(torch.randn(40, 10, device="cuda"))]
    opt = muon.Muon(w, lr=0.1, momentum=0.9, weight_decay=0.01)
    want = [p.detach().double().cpu() for p in w]
    moments = [torch.zeros_like(p) for p in want]
    for _ in range(3):
        grads = [torch.randn_like(p) for p in w]
        for p, g in zip(w, grads):
            p.grad = g
        opt.step()
        for i, g in enumerate(grads):
            g = g.double().cpu()
            moments[i] = 0.9 * moments[i] + g
            u = _exact((g + 0.9 * moments[i]).flatten(1)).view(g.shape)
            want[i] = want[i] * (1 - 0.1 * 0.01) - 0.1 * max(1.0, g.shape[0] / g[0].numel()) ** 0.5 * u
    for p, t in zip(w, want):
        assert (p.detach().cpu().double() - t).norm() < 1e-5 * t.norm()
    empty = torch.nn.Parameter(torch.zeros(3, 0, device="cuda"))
    empty.grad = torch.zeros_like(empty)
    muon.Muon([empty]).step()
    with pytest.raises(ValueError, match="two or more"):
        muon.Muon([torch.nn.Parameter(torch.zeros(4))])


def test_records_to_update_together():
    # what a training program does: records -> symmetries and duplicates -> network -> loss -> gradients -> update
    from alphazero_amd import augment, muon
    from alphazero_amd.model import PolicyValueNet

    gen = torch.Generator(device="cuda").manual_seed(3)
    n, S = 40, 7
    board = torch.zeros(n, 2, S * S, device="cuda")
    for i in range(n):
        at = torch.randperm(S * S, generator=gen, device="cuda")[:2 * (i % 9)]
        board[i, 0, at[::2]] = 1
        board[i, 1, at[1::2]] = 1
    board = board.view(n, 2, S, S)
    pi = torch.rand(n, S * S, generator=gen, device="cuda") * (board.sum(1).flatten(1) == 0)
    pi = pi / pi.sum(1, keepdim=True)
    r = torch.where(torch.rand(n, generator=gen, device="cuda") < 0.5, 1.0, -1.0)
    more = augment.rotations_device(board, pi, r)
    board, pi, r = augment.unique_device(*[torch.cat(t) for t in zip((board, pi, r), more)])
    torch.manual_seed(1)
    net = PolicyValueNet(S).cuda()
    weights, others = muon.Muon.weights_of(net)
    assert len(weights) == 10 and all(p.dim() == 4 for p in weights)
    opts = [muon.Muon(weights, lr=0.02), torch.optim.SGD(others, lr=0.02)]
    before = [p.detach().clone() for p in weights]
    net.loss(board, pi, r, mask_illegal=True).backward()
    # the gradients of the masked loss, written with torch's own operators
    grads = [p.grad.clone() for p in net.parameters()]
    net.zero_grad()
    value, logits = net.heads(board)
    logp = torch.log_softmax(logits.masked_fill(board.sum(1).flatten(1) > 0, -1e30), 1)
    (torch.nn.functional.kl_div(logp, pi, reduction="batchmean") + torch.nn.functional.mse_loss(value.view(-1), r)).backward()
    for p, g in zip(net.parameters(), grads):
        assert (p.grad - g).norm() <= 1e-3 * p.grad.norm() + 1e-6
        p.grad = g
    for opt in opts:
        opt.step()
    for p, b in zip(weights, before):
        u = _exact((1.95 * p.grad).flatten(1).cpu()).view(p.shape)  # first step: m = g, u = g + 0.95 g
        want = b.cpu().double() - 0.02 * max(1.0, p.shape[0] / p[0].numel()) ** 0.5 * u
        assert (p.detach().cpu().double() - want).norm() < 1e-5 * want.norm()


# widths from 1.5 times the height on, more than 64 rows: tiles of 64 (Gram matrices shared and not) and of 128
@pytest.mark.parametrize("shape", [(256, 2304), (512, 1024), (70, 130), (333, 1201), (1500, 130), (12, 256, 768)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank,floor", [(1, None), (4, None), (1, 0.0), (4, 0.0), (32, 0.0), (64, 0.02)])
def test_low_rank_updates_in_16_bits(shape, dtype, rank, floor):
    # Gradients of a batch smaller than the layer: most directions hold nothing, or only noise, and every step multiplies
    # what a rounded product leaves in them by a.  Same bound as above: products of float32 precision, one rounding.
    from alphazero_amd import muon

    g = _updates(shape, 31, 1.0, rank=rank)
    if floor is None:  # small whole numbers: exactly of that rank in every type
        gen = torch.Generator().manual_seed(33)
        g = (torch.randint(-2, 3, (*shape[:-1], rank), generator=gen) @ torch.randint(-2, 3, (*shape[:-2], rank, shape[-1]), generator=gen)).float()
    elif floor:
        g = g + floor * math.sqrt(rank) * _updates(shape, 32, 1.0)
    g = g.to(dtype).cuda()
    for steps in (3, 4, 5, 6, 7):
        _check(muon.orthogonalise(g, steps), g, steps)


@pytest.mark.parametrize("shape", [(30, 600), (64, 576), (2, 60, 200), (130, 1000), (256, 2304), (2, 400, 2000), (2, 1024, 4096)])
@pytest.mark.parametrize("rows", ["one", "half", "spread"])
def test_updates_with_rows_of_very_different_size(shape, rows):
    # A nearly dead channel.  Numbers of X stop at 2^-39 (an error of 2^-40 each), of A at 2^-38, of Q at 2^-34 (2^-35 each,
    # with A's 2^-39 times b and c: at most 2^-34), so a step adds to each row at most 2^-40 sqrt(n) + 2^-34 |X|, and
    # later steps multiply that by at most a each: sqrt(m) (...) a^(steps - 1) sum_k a^-k, the sum being below 1.41.  To that
    # come 16 u a step for the products (8 u, and as much again for the errors' mutual growth).
    from alphazero_amd import muon

    m, n = shape[-2:]
    for s in (1e-3, 1e-5, 1e-7, 1e-9, 1e-11):
        g = _updates(shape, 41, 1.0)
        if rows == "one":
            g[..., m // 3, :] *= s
        elif rows == "half":
            g[..., ::2, :] *= s
        else:
            g *= s ** (torch.arange(m) / m).unsqueeze(1)
        for steps in (1, 5, 10) if m < 400 else (5, 10):
            x = g.double().cuda()  # (the definition on the GPU, in 64 bits)
            x = x / x.square().sum((-1, -2), keepdim=True).sqrt()
            for _ in range(steps):
                A = x @ x.transpose(-1, -2).contiguous()
                x = ABC[0] * x + (ABC[1] * A + ABC[2] * (A @ A)) @ x
            off = (muon.orthogonalise(g.cuda(), steps).double() - x).flatten(-2).norm(dim=-1)
            size = x.flatten(-2).norm(dim=-1)
            tol = 16 * steps * U * size + 1.41 * ABC[0] ** (steps - 1) * m ** 0.5 * (2.0 ** -40 * n ** 0.5 + 2.0 ** -34 * size)
            assert (off <= tol).all(), (s, steps, off, tol)


@pytest.mark.parametrize("dtype,momentum,quiet,size", [(torch.float16, 0.95, 16, 6e-7), (torch.bfloat16, 0.999, 250, 1e-7), (torch.float32, 0.95, 16, 1e-7)])
def test_momentum_of_16_bit_weights_decays(dtype, momentum, quiet, size):
    # A gradient, a number of steps without one, another gradient: how much of the first is left decides the direction.  In 16
    # bits 0.95 m rounds back to m below 6e-7 (float16), and 0.999 m everywhere (bfloat16).
    from alphazero_amd import muon

    gen = torch.Generator().manual_seed(51)
    first, second = [(torch.randn(24, 60, generator=gen) * size).to(dtype) for _ in range(2)]
    w = torch.nn.Parameter(torch.zeros(24, 60, dtype=dtype, device="cuda"))
    opt = muon.Muon([w], lr=0.02, momentum=momentum)
    m, none = torch.zeros(24, 60, dtype=torch.float64), torch.zeros_like(first)
    for g in [first] + [none] * quiet + [second]:
        w.grad = g.cuda()
        w.data.zero_()
        opt.step()
        m = momentum * m + g.double()
    u = _exact(g.double() + momentum * m)
    want = -0.02 * u
    # the last step alone: the update's own error (float32 products, momentum in float32: quiet u), half a step of the weight
    off = (w.detach().cpu().double() - want).norm()
    assert off <= 0.02 * ABC[0] ** 4 * 1.41 * (32 + 2 * quiet) * U + torch.finfo(dtype).eps / 2 * want.norm()


TYPES_16 = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES_16)
def test_weights_of_16_bits_step_by_step(dtype):
    # several weights of both kinds in one optimiser: each step is computed in float32 and rounded into the weight once
    from alphazero_amd import muon

    gen = torch.Generator().manual_seed(52)
    shapes = [(16, 4, 3, 3), (40, 10), (130, 300)]
    w = [torch.nn.Parameter(torch.randn(*s, generator=gen).to(t).cuda()) for s in shapes for t in (dtype, torch.float32)]
    opt = muon.Muon(w, lr=0.05, momentum=0.9, weight_decay=0.02)
    moments = [torch.zeros(p.shape, dtype=torch.float64) for p in w]
    for _ in range(3):
        for i, p in enumerate(w):
            g = (torch.randn(p.shape, generator=gen) * 1e-3).to(p.dtype)
            p.grad = g.cuda()
            moments[i] = 0.9 * moments[i] + g.double()
        before = [p.detach().cpu().double() for p in w]
        opt.step()
        for i, (p, b) in enumerate(zip(w, before)):
            u = _exact((p.grad.cpu().double() + 0.9 * moments[i]).flatten(1)).view(p.shape)
            want = b * (1 - 0.05 * 0.02) - 0.05 * max(1.0, p.shape[0] / p[0].numel()) ** 0.5 * u
            off = (p.detach().cpu().double() - want).abs()
            # 1e-5 of the step for the update (as above), 3 u for decay, product and sum, half a step of the weight
            assert (off <= 1e-5 * 0.05 * u.norm() + want.abs() * (torch.finfo(p.dtype).eps / 2 + 3 * U) +
                    (2.0 ** -25 if p.dtype == torch.float16 else 0)).all()
        assert all(opt.state[p]["momentum"].dtype == torch.float32 for p in w)


@pytest.mark.parametrize("dtype", [torch.float32] + TYPES_16)
def test_optimiser_goes_on_from_its_saved_state(dtype):
    import io

    from alphazero_amd import muon

    gen = torch.Generator().manual_seed(53)
    grads = [(torch.randn(20, 50, generator=gen) * 1e-6).to(dtype).cuda() for _ in range(6)]

    def steps(w, opt, some):
        for g in some:
            w.grad = g.clone()
            opt.step()

    a = torch.nn.Parameter(torch.zeros(20, 50, dtype=dtype, device="cuda"))
    one = muon.Muon([a], lr=0.1, momentum=0.9)
    steps(a, one, grads[:3])
    b = torch.nn.Parameter(a.detach().clone())
    two = muon.Muon([b], lr=0.5)
    file = io.BytesIO()
    torch.save(one.state_dict(), file)
    file.seek(0)
    two.load_state_dict(torch.load(file, weights_only=True, map_location="cpu"))
    assert two.param_groups[0]["momentum"] == 0.9 and two.state[b]["momentum"].dtype == torch.float32
    assert torch.equal(two.state[b]["momentum"], one.state[a]["momentum"])
    steps(a, one, grads[3:])
    steps(b, two, grads[3:])
    assert torch.equal(a, b) and two.state[b]["momentum"].data_ptr() != one.state[a]["momentum"].data_ptr()


@pytest.mark.parametrize("shape,steps", [((32768, 1), 5), ((1, 32768), 5), ((33, 32768), 5), ((32768, 70), 5), ((16384, 16384), 1), ((8192, 32768), 1)])
def test_the_largest_sizes(shape, steps):
    from alphazero_amd import muon

    g = torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    out = muon.orthogonalise(g, steps)
    x = g.double()  # (the definition on the GPU, in 64 bits)
    x = x.t().contiguous() if shape[0] > shape[1] else x
    x = x / x.square().sum().sqrt()
    for _ in range(steps):
        A = x @ x.t().contiguous()
        x = ABC[0] * x + (ABC[1] * A + ABC[2] * (A @ A)) @ x
    x = x.t() if shape[0] > shape[1] else x
    size = x.norm()
    assert (out.double() - x).norm() <= ABC[0] ** (steps - 1) * 1.41 * 32 * U + size * 64 * U
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(1280, 3328), (1300, 3400), (1536, 2816), (2432, 1792), (1150, 3700), (1280, 3968)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_last_tiles_shared_from_a_smaller_k_on(shape, dtype):
    # 260 to 310 large tiles for 256 CUs, on both sides of the rule
    from alphazero_amd import muon

    g = _updates(shape, 61).to(dtype).cuda()
    out = muon.orthogonalise(g, 3)
    assert torch.equal(out, muon.orthogonalise(g, 3))
    x = g.double()  # (the definition on the GPU, in 64 bits)
    x = x.t().contiguous() if shape[0] > shape[1] else x
    x = x / x.square().sum().sqrt()
    for _ in range(3):
        A = x @ x.t().contiguous()
        x = ABC[0] * x + (ABC[1] * A + ABC[2] * (A @ A)) @ x
    x = x.t() if shape[0] > shape[1] else x
    size = x.norm()
    assert (out.double() - x).norm() <= ABC[0] ** 2 * 1.41 * 32 * U + size * (64 * U + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0))


def test_a_captured_step():
    # forward pass, backward pass and update of weights of both kinds in one graph, between eager steps of a twin
    from alphazero_amd import muon

    torch.manual_seed(5)
    shapes = [(24, 30), (100, 140)]
    x = torch.ones((), device="cuda")

    def program():
        gen = torch.Generator().manual_seed(54)
        w = [torch.nn.Parameter((torch.randn(*s, generator=gen) * 0.1).to(t).cuda()) for s in shapes for t in (torch.float32, torch.bfloat16)]
        opt = muon.Muon(w, lr=0.05, weight_decay=0.01)

        ones = [torch.ones(p.shape, device="cuda") for p in w]

        def step():
            for p, g in zip(w, torch.autograd.grad([torch.tanh(p.float() * x) for p in w], w, ones)):
                p.grad.copy_(g)
            opt.step()

        for p in w:
            p.grad = torch.zeros_like(p)
        return w, step

    (a, eager), (b, captured) = program(), program()
    eager(), captured()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured()
    for k in range(4):
        x.add_(0.1 * k)
        eager()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), k
