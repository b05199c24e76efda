"""The policy-learning operators of the framework as measured calls.

Three operators, used together by a program that trains the policy/value network on self-play records and
reads its answers:

  score        log-probabilities of given moves, the entropy and the best alternatives of a policy row,
               over the legal moves of a position, with the gradient for the logits
  loss         the trainer's loss (KL divergence of the policy head from the visit distribution, averaged over
               the batch, plus the mean squared error of the value head) with the gradients for both heads
  orthogonalise   Newton-Schulz orthogonalisation of weight updates (the Muon optimiser's step)

`own = False` computes them in elementary torch operations in 32 bits, `own = True` through alphazero_amd.
"""
import math

import torch

own = False

NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315  # coefficients of one Newton-Schulz step
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one position, asked for its best five moves: a front end shows what the network thinks
        {"name": "score_one", "op": "score", "rows": 1, "side": 15, "type": "f32", "mask": "board", "top": 5, "grad": False},
        # a step of 8192 trees of 15x15: the played move's log-probability and eight alternatives per position
        {"name": "score_step", "op": "score", "rows": 8192, "side": 15, "type": "f32", "mask": "board", "top": 8, "grad": False},
        # policy-gradient style training on 19x19 records in bf16, legal moves as a bool mask, with the backward pass
        {"name": "score_train", "op": "score", "rows": 32768, "side": 19, "type": "bf16", "mask": "legal", "top": 0, "grad": True},
        # few long rows (a large action set of another module's policy head), odd length
        {"name": "score_long", "op": "score", "rows": 96, "actions": 50021, "type": "f16", "mask": "none", "top": 16, "grad": False},
        # a small training batch at the reference's board size
        {"name": "loss_small", "op": "loss", "rows": 128, "side": 13, "type": "f32", "mask": "none"},
        # 20x20 in bf16 with illegal moves masked
        {"name": "loss_masked", "op": "loss", "rows": 65536, "side": 20, "type": "bf16", "mask": "legal"},
        # 32768 records of 15x15 with their seven symmetries in one batch
        {"name": "loss_large", "op": "loss", "rows": 262144, "side": 15, "type": "f32", "mask": "none"},
        # the 16 -> 16 layers of the reference network (16 x 16 * 3 * 3 weights, seven of them)
        {"name": "muon_net", "op": "muon", "count": 7, "m": 16, "n": 144, "type": "f32"},
        # a 64-channel tower of 16 layers
        {"name": "muon_tower", "op": "muon", "count": 16, "m": 64, "n": 576, "type": "f32"},
        # a 256-channel tower of 12 layers, bf16 updates
        {"name": "muon_wide", "op": "muon", "count": 12, "m": 256, "n": 2304, "type": "bf16"},
        # dense layers of odd sizes, taller than wide
        {"name": "muon_ragged", "op": "muon", "count": 5, "m": 1201, "n": 333, "type": "f32"},
        # two large dense layers
        {"name": "muon_large", "op": "muon", "count": 2, "m": 2048, "n": 4096, "type": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "score", "loss", "muon", "muon"])
    if op == "muon":
        while True:
            c = {"op": op, "count": _log(rng, 1, 16), "m": _log(rng, 8, 2048), "n": _log(rng, 8, 4608),
                 "type": rng.choice(["f32", "f32", "bf16"])}
            lo, hi = min(c["m"], c["n"]), max(c["m"], c["n"])
            if c["count"] * lo * lo * (2 * hi + lo) <= 2 * 2048 * 2048 * (2 * 4096 + 2048) and c["count"] * lo * hi <= 2 * 2048 * 4096:
                return c
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "loss":
        return {"op": op, "rows": _log(rng, 1, 140000), "side": rng.randint(5, 20), "type": kind,
                "mask": rng.choice(["none", "board", "legal"])}
    if rng.random() < 0.3:
        actions = _log(rng, 1, 100000)
        return {"op": op, "rows": _log(rng, 1, max(1, 5_000_000 // actions)), "actions": actions, "type": kind,
                "mask": rng.choice(["none", "legal"]), "top": rng.choice([0, 1, 5, 16]), "grad": rng.random() < 0.5}
    return {"op": op, "rows": _log(rng, 1, 32768), "side": rng.randint(5, 20), "type": kind,
            "mask": rng.choice(["none", "board", "legal"]), "top": rng.choice([0, 1, 5, 8]), "grad": rng.random() < 0.5}


def _actions(case):
    return case["actions"] if "actions" in case else case["side"] ** 2


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    uni = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    dtype = TYPES[case["type"]]
    if case["op"] == "muon":
        # gradients of a layer: a few strong directions over a noise floor, small in size
        c, m, n = case["count"], case["m"], case["n"]
        r = max(1, min(m, n) // 8)
        strong = torch.matmul(rnd(c, m, r), rnd(c, r, n)) / math.sqrt(r)
        return {"case": case, "updates": ((strong + 0.5 * rnd(c, m, n)) * 1e-3).to(dtype)}
    rows, actions = case["rows"], _actions(case)
    s = {"case": case, "logits": (2.5 * rnd(rows, actions)).to(dtype), "board": None, "legal": None}
    # positions between the empty and the nearly full board; now and then a full one (nothing is legal)
    density = 0.9 * uni(rows, 1) ** 2
    density[uni(rows, 1) > 0.98] = 1.0
    taken = uni(rows, actions) < density
    if case["mask"] == "board":
        first = uni(rows, actions) < 0.5
        planes = torch.stack([taken & first, taken & ~first], dim=1)
        s["board"] = planes.to(torch.float32).view(rows, 2, case["side"], case["side"])
    elif case["mask"] == "legal":
        s["legal"] = ~taken
    if case["op"] == "score":
        s["moves"] = torch.randint(0, actions, (rows,), generator=g, device="cuda", dtype=torch.int32)
        if case["mask"] != "none":  # mostly a legal move: the highest of a random order of the row
            s["moves"] = torch.where(taken, -1.0, uni(rows, actions)).argmax(1).to(torch.int32)
        s["top"] = case["top"]
        if case["grad"]:
            s["logits"].requires_grad_()
            s["d_logp"], s["d_entropy"] = rnd(rows) / rows, torch.full((rows,), 0.01 / rows, device="cuda")
        return s
    # visit distributions: about 800 searches over the moves the network likes, most cells never visited
    v = torch.where(taken if case["mask"] != "none" else torch.zeros_like(taken), -math.inf, 3.0 * rnd(rows, actions))
    visits = torch.floor(800 * torch.softmax(v, dim=1).nan_to_num(0.0))
    s["pi"] = visits / visits.sum(1, keepdim=True).clamp(min=1.0)
    s["value"] = torch.tanh(rnd(rows)).to(dtype)
    s["r"] = torch.where(uni(rows) < 0.5, 1.0, -1.0)
    s["logits"].requires_grad_()
    s["value"].requires_grad_()
    return s


# ---------------------------------------------------------------- plain forms

def _legal(s):
    if s["board"] is not None:
        b = s["board"].flatten(2)
        return (b[:, 0] == 0) & (b[:, 1] == 0)
    return s["legal"]


def _log_probs(s):
    """Masked logits, log-probabilities (-inf at illegal moves and in rows without a legal one) and probabilities."""
    x = s["logits"].detach().float()
    legal = _legal(s)
    if legal is not None:
        x = torch.where(legal, x, -math.inf)
    top = x.max(dim=1, keepdim=True).values
    d = torch.where(x == -math.inf, -math.inf, x - top)
    e = torch.exp(d)
    total = e.sum(dim=1, keepdim=True)
    logp = d - torch.log(total).clamp(min=0.0)
    return x, logp, e / total.clamp(min=1.0)


def _plain_score(s):
    x, logp, p = _log_probs(s)
    moves = s["moves"].long().unsqueeze(1)
    out = {"logp": logp.gather(1, moves).squeeze(1)}
    plogp = torch.where(p > 0, p * logp, 0.0)
    out["entropy"] = -plogp.sum(dim=1)
    k = s["top"]
    if k:
        # keys that order by value, then by lowest index
        bits = (x + 0.0).view(torch.int32)
        order = bits ^ ((bits >> 31) & 0x7FFFFFFF)
        index = torch.arange(x.shape[1], device=x.device)
        keys = (order.long() << 32) | (0x7FFFFFFF - index)
        kept = min(k, x.shape[1])
        at = 0x7FFFFFFF - (torch.topk(keys, kept, dim=1).values & 0xFFFFFFFF)
        found = logp.gather(1, at)
        at = torch.where(found == -math.inf, -1, at).int()
        out["top_moves"] = torch.nn.functional.pad(at, (0, k - kept), value=-1)
        out["top_logp"] = torch.nn.functional.pad(found, (0, k - kept), value=-math.inf)
    if s["case"]["grad"]:
        g, h = s["d_logp"].unsqueeze(1), s["d_entropy"].unsqueeze(1)
        g = torch.where(out["logp"].unsqueeze(1) == -math.inf, 0.0, g)
        d = -p * g - h * torch.where(p > 0, p * (logp + out["entropy"].unsqueeze(1)), 0.0)
        d.scatter_add_(1, moves, g)
        out["d_logits"] = d.to(s["logits"].dtype)
    return out


def _plain_loss(s):
    x, logp, p = _log_probs(s)
    n = x.shape[0]
    pi = torch.where(x == -math.inf, 0.0, s["pi"])
    kl = torch.where(pi == 0, 0.0, pi * (torch.log(pi) - logp)).sum(dim=1).double().sum() / n
    miss = s["value"].detach().float() - s["r"]
    loss = kl + miss.double().square().sum() / n
    d_logits = (p * pi.sum(dim=1, keepdim=True) - pi) / n
    d_value = miss * (2.0 / n)
    return {"loss": loss.float(), "d_logits": d_logits.to(s["logits"].dtype), "d_value": d_value.to(s["value"].dtype)}


def _ns_step(x):
    gram = torch.matmul(x, x.transpose(1, 2))
    return torch.baddbmm(x, torch.baddbmm(gram, gram, gram, beta=NS_B, alpha=NS_C), x, beta=NS_A)


def _plain_orthogonalise(s):
    x = s["updates"].float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    x = x / x.double().square().sum(dim=(1, 2), keepdim=True).sqrt().clamp(min=1e-30).float()
    x = _ns_step(_ns_step(_ns_step(_ns_step(_ns_step(x)))))
    if tall:
        x = x.transpose(1, 2).contiguous()
    return {"update": x.to(s["updates"].dtype)}


# ---------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        if op == "muon":
            from alphazero_amd import muon

            return {"update": muon.orthogonalise(state["updates"])}
        from alphazero_amd import policy

        if op == "score":
            s = policy.score(state["logits"], state["moves"], board=state["board"], legal=state["legal"], top=state["top"])
            out = {"logp": s.logp.detach(), "entropy": s.entropy.detach()}
            if state["top"]:
                out["top_moves"], out["top_logp"] = s.top_moves, s.top_logp
            if state["case"]["grad"]:
                out["d_logits"], = torch.autograd.grad((s.logp, s.entropy), state["logits"], (state["d_logp"], state["d_entropy"]))
            return out
        loss = policy.loss(state["logits"], state["value"], state["pi"], state["r"], board=state["board"], legal=state["legal"])
        d_logits, d_value = torch.autograd.grad(loss, (state["logits"], state["value"]))
        return {"loss": loss.detach(), "d_logits": d_logits, "d_value": d_value}
    return {"score": _plain_score, "loss": _plain_loss, "muon": _plain_orthogonalise}[op](state)


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    if case["op"] == "muon":
        lo, hi = min(case["m"], case["n"]), max(case["m"], case["n"])
        # five steps of a Gram matrix (symmetric: half of its products), its square (half) and the product with x
        flops = 5.0 * (lo * lo * hi + lo ** 3 + 2.0 * lo * lo * hi)
        return {"bytes": 2.0 * case["count"] * lo * hi * size, "flops": case["count"] * flops}
    rows, cells = case["rows"], case["rows"] * _actions(case)
    mask = {"none": 0, "board": 8, "legal": 1}[case["mask"]]
    if case["op"] == "score":
        nbytes = cells * (size + mask) + rows * (4 + 4 + 4 + 8 * case["top"])
        if case["grad"]:
            nbytes += cells * size + rows * 8
        return {"bytes": float(nbytes), "flops": cells * (12.0 if case["grad"] else 6.0)}
    return {"bytes": float(cells * (2 * size + 4 + mask) + rows * (2 * size + 4)), "flops": 12.0 * cells}


# ---------------------------------------------------------------- in 64 bits, from the definitions

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "muon":
        # sigma -> p(p(p(p(p(sigma))))) on the singular values of the scaled update: with G = U S V', the result is
        # U f(S) V' = U (f(S) / S) U' G, the left vectors from the eigenvectors of G G'
        g = s["updates"].double()
        tall = case["m"] > case["n"]
        g = g.transpose(1, 2).contiguous() if tall else g
        g = g / torch.linalg.vector_norm(g, dim=(1, 2), keepdim=True).clamp(min=1e-30)
        if min(case["m"], case["n"]) <= 512:
            lam, u = torch.linalg.eigh(torch.matmul(g, g.transpose(1, 2)).cpu())
            lam, u = lam.clamp(min=0.0).to(g.device), u.to(g.device)
            gain, sq = torch.ones_like(lam), lam
            for _ in range(5):
                q = NS_A + NS_B * sq + NS_C * sq * sq
                gain, sq = gain * q, sq * q * q
            out = torch.matmul(u * gain.unsqueeze(1), torch.matmul(u.transpose(1, 2).contiguous(), g))
        else:  # the same polynomial of G G' without its eigenvectors: products of commuting factors
            gram = torch.matmul(g, g.transpose(1, 2).contiguous())
            eye = torch.eye(gram.shape[1], dtype=gram.dtype, device=gram.device)
            total = eye.expand_as(gram)
            for _ in range(5):
                q = NS_A * eye + torch.matmul(NS_B * eye + NS_C * gram, gram)
                total, gram = torch.matmul(q, total), torch.matmul(q, torch.matmul(q, gram))
            out = torch.matmul(total, g)
        return {"update": out.transpose(1, 2).contiguous() if tall else out}

    x = s["logits"].detach().double().requires_grad_()
    if s["board"] is not None:
        open_ = (s["board"].sum(dim=1) == 0).flatten(1)
    else:
        open_ = s["legal"] if s["legal"] is not None else torch.ones_like(x, dtype=torch.bool)
    some = open_.any(dim=1, keepdim=True)
    # rows without a legal move: computed on a stand-in row, then left out
    use = open_ | ~some
    logp = torch.log_softmax(x.masked_fill(~use, -math.inf), dim=1)
    finite = logp.masked_fill(~use, 0.0)
    live = some.squeeze(1)
    if case["op"] == "score":
        moves = s["moves"].long()
        hit = open_.gather(1, moves.unsqueeze(1)).squeeze(1)
        mine = finite.gather(1, moves.unsqueeze(1)).squeeze(1)
        entropy = -(finite.exp() * finite * use).sum(dim=1)
        out = {"logp": mine.detach().masked_fill(~hit, -math.inf), "entropy": entropy.detach().masked_fill(~live, 0.0)}
        if case["top"]:
            k = min(case["top"], x.shape[1])
            ranked = logp.detach().masked_fill(~open_, -math.inf).topk(k, dim=1).values
            out["top_moves"] = None
            out["top_logp"] = torch.nn.functional.pad(ranked, (0, case["top"] - k), value=-math.inf)
        if case["grad"]:
            upstream = (mine * s["d_logp"].double())[hit & live].sum() + (entropy * s["d_entropy"].double())[live].sum()
            out["d_logits"], = torch.autograd.grad(upstream, x)
        return out
    v = s["value"].detach().double().requires_grad_()
    pi = s["pi"].double() * open_
    loss = ((torch.xlogy(pi, pi) - pi * finite).sum() + (v - s["r"].double()).square().sum()) / case["rows"]
    d_logits, d_value = torch.autograd.grad(loss, (x, v))
    return {"loss": loss.detach(), "d_logits": d_logits, "d_value": d_value}
