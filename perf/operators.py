"""What the operators of a training iteration around the optimizer step are measured on.

Operators:

``rotate``    ``rotate_qk``: queries and keys turned by their positions, on one axis or several (time, height, width).
``norm``      ``norm_rotate_qk``: the root-mean-square norm of every head's query and key and the rotation in one pass;
              forward alone, or with the gradients of both and of the norms' weights.
``top``       ``top_logits``: the k largest logits of every row, their places and the row's log-sum-exp (what a teacher leaves
              behind for its student).
``distill``   ``distill_loss``: the loss of a student's logits against a teacher's top logits and the labels; every row's loss
              alone, or their mean with the gradient at a loss scale.

With ``own`` false everything is computed in plain torch operations in 32 bits.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # One new token of one sequence, grouped heads: what a decoding step pays before its attention; latency.
        dict(name="rotate_one_token", op="rotate", train=False, dtype="bf16", batch=1, seq=1, heads=16, kv_heads=4, dim=128,
             rotary=128, axes=1, interleaved=False, packed=True, start=20000),
        # A long text prompt, neighbouring pairs, half of the dimensions rotated; q and k lie in one projection's output.
        dict(name="rotate_prompt", op="rotate", train=False, dtype="fp16", batch=1, seq=16384, heads=25, kv_heads=25, dim=64,
             rotary=32, axes=1, interleaved=True, packed=True, start=0),
        # Frames of a video (time, height, width), a training batch: out and back.
        dict(name="rotate_video_train", op="rotate", train=True, dtype="bf16", batch=2, seq=6000, heads=16, kv_heads=16, dim=128,
             rotary=128, axes=3, interleaved=False, packed=False, start=0),
        # A batch of sequences that each add one token.
        dict(name="norm_new_tokens", op="norm", train=False, dtype="fp16", batch=32, seq=1, heads=32, kv_heads=8, dim=128,
             rotary=128, axes=1, interleaved=False, packed=True, start=100000),
        # 8 sequences of 128 tokens with BERT-base's heads: the training batch of the package's own engine case.
        dict(name="norm_bert_base_train", op="norm", train=True, dtype="fp16", batch=8, seq=128, heads=12, kv_heads=12, dim=64,
             rotary=64, axes=1, interleaved=False, packed=True, start=0),
        # A large training batch with grouped heads and three axes.
        dict(name="norm_video_train", op="norm", train=True, dtype="bf16", batch=1, seq=16383, heads=32, kv_heads=8, dim=128,
             rotary=128, axes=3, interleaved=False, packed=True, start=0),
        # A small teacher batch over BERT's vocabulary.
        dict(name="top_bert_vocab", op="top", dtype="fp16", rows=128, vocab=30522, k=32, temperature=1.0),
        # A teacher's batch of 8192 tokens over GPT-2's vocabulary (odd, so rows start at any alignment).
        dict(name="top_gpt2_vocab", op="top", dtype="fp16", rows=8192, vocab=50257, k=64, temperature=2.0),
        # Logits in 32 bits over a vocabulary beyond what one workgroup can keep, and a long list.
        dict(name="top_fp32_long", op="top", dtype="fp32", rows=500, vocab=200000, k=200, temperature=1.0),
        # A small student: 64 tokens, a small vocabulary, every list short of some entries.
        dict(name="distill_small_train", op="distill", train=True, dtype="fp16", rows=64, vocab=8192, k=8, rest=False,
             temperature=1.0, label_weight=0.0, ignored=0.0, scale=2.0**12),
        # A student's batch of 8192 tokens over GPT-2's vocabulary: lists of 64 with the rest of the teacher's mass, labels, padding.
        dict(name="distill_gpt2_train", op="distill", train=True, dtype="fp16", rows=8192, vocab=50257, k=64, rest=True,
             temperature=2.0, label_weight=0.25, ignored=0.1, scale=2.0**16),
        # Every token's loss alone, on held-out tokens.
        dict(name="distill_bert_vocab_loss", op="distill", train=False, dtype="bf16", rows=4096, vocab=30522, k=32, rest=True,
             temperature=1.0, label_weight=0.0, ignored=0.2, scale=1.0),
    ]


# ------------------------------------------------------------------------------------------------------ drawn cases


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "norm", "norm", "top", "distill", "distill"])
    case = dict(op=op, dtype=rng.choice(["fp16", "fp16", "bf16", "fp32"]))
    if op in ("rotate", "norm"):
        dim = rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 3, 4, 8, 12, 16])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 5])
        batch = rng.choice([1, 1, 2, 3, 8])
        width = (heads + kv_heads) * dim * (2 if case["dtype"] == "fp32" else 1)
        seq = max(1, min(_log_int(rng, 1, 16384), 16383 * 40 * 128 // (width * batch)))
        case.update(train=rng.random() < 0.5, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim,
                    rotary=rng.choice([dim, dim, dim // 2]), axes=rng.choice([1, 1, 3]), interleaved=rng.random() < 0.3,
                    packed=rng.random() < 0.6, start=rng.choice([0, 0, rng.randint(0, 1000000)]))
        return case
    vocab = _log_int(rng, 1000, 200000)
    wide = 2 if case["dtype"] == "fp32" else 1
    rows = max(1, min(_log_int(rng, 1, 8192), 8192 * 50257 // (vocab * wide)))
    case.update(rows=rows, vocab=vocab, k=_log_int(rng, 1, 256), temperature=rng.choice([1.0, 1.0, 2.0, 4.0, 0.7]))
    if op == "distill":
        case.update(train=rng.random() < 0.7, rest=rng.random() < 0.5, label_weight=rng.choice([0.0, 0.0, 0.25, 1.0]),
                    ignored=rng.choice([0.0, 0.1, 0.5]), scale=2.0 ** (int(math.log2(rows)) + rng.choice([0, 3])))
    return case


# ----------------------------------------------------------------------------------------------------------- inputs


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _normal(gen, shape, std, dtype):
    """Normal numbers, made in parts so that the 32-bit ones never stand there whole."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for lo in range(0, flat.numel(), 1 << 27):
        part = flat[lo : lo + (1 << 27)]
        part.copy_(torch.empty(part.numel(), device="cuda").normal_(0, std, generator=gen))
    return out


def _sections(case):
    """Pairs of each axis: a quarter for time, the rest shared by height and width."""
    pairs = case["rotary"] // 2
    if case["axes"] == 1:
        return None
    time = pairs // 4
    return (time, (pairs - time) // 2, pairs - time - (pairs - time) // 2)


def _heads_inputs(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    b, s, h, hk, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dim"]
    if case["packed"]:
        qkv = _normal(gen, (b, s, (h + 2 * hk) * d), 1.0, dtype)
        q = qkv[..., : h * d].view(b, s, h, d)
        k = qkv[..., h * d : (h + hk) * d].view(b, s, hk, d)
    else:
        q, k = _normal(gen, (b, s, h, d), 1.0, dtype), _normal(gen, (b, s, hk, d), 1.0, dtype)
    if case["axes"] == 1:
        positions = case["start"] + torch.arange(s, device="cuda").expand(b, s)
        if s == 1:  # sequences of different lengths
            positions = torch.randint(case["start"] // 2, case["start"] + 1, (b, 1), device="cuda", generator=gen)
    else:  # frames of 25 by 40 patches
        place = torch.arange(s, device="cuda").expand(b, s)
        positions = case["start"] + torch.stack([place // 1000, place % 1000 // 40, place % 40])
    out = dict(q=q, k=k, positions=positions)
    if case["op"] == "norm":
        out["q_weight"] = (1 + 0.1 * torch.randn(d, device="cuda", generator=gen)).to(dtype)
        out["k_weight"] = (1 + 0.1 * torch.randn(d, device="cuda", generator=gen)).to(dtype)
    if case["train"]:
        out["q_grad"], out["k_grad"] = _normal(gen, (b, s, h, d), 0.1, dtype), _normal(gen, (b, s, hk, d), 0.1, dtype)
    return out


def _logits(gen, case):
    """Rows in which a few tokens hold most of the mass."""
    return _normal(gen, (case["rows"], case["vocab"]), 3.0, DTYPES[case["dtype"]])


def _distill_inputs(case, seed):
    """A student's logits, and the list that a teacher near it leaves: its values are the student's own with noise on them."""
    gen = _generator(seed)
    n, v, k, t = case["rows"], case["vocab"], min(case["k"], case["vocab"]), case["temperature"]
    logits = _logits(gen, case)
    ids = torch.empty(n, k, dtype=torch.int32, device="cuda")
    values = torch.empty(n, k, dtype=logits.dtype, device="cuda")
    lse = torch.empty(n, device="cuda")
    step = max(1, (1 << 26) // v)
    for lo in range(0, n, step):
        part = logits[lo : lo + step].float()
        part += torch.empty_like(part).normal_(0, 0.5, generator=gen)
        part = part.to(logits.dtype)
        top = part.topk(k, dim=-1)
        values[lo : lo + step], ids[lo : lo + step] = top.values, top.indices.int()
        lse[lo : lo + step] = (part.float() / t).logsumexp(-1)
    if not case["rest"]:  # lists of different lengths: the places behind a list's end hold -1
        length = torch.randint(1, k + 1, (n, 1), device="cuda", generator=gen)
        ids = torch.where(torch.arange(k, device="cuda") < length, ids, -1)
    labels = torch.randint(v, (n,), device="cuda", generator=gen)
    labels[torch.rand(n, device="cuda", generator=gen) < case["ignored"]] = -100
    return dict(logits=logits, ids=ids, values=values, lse=lse if case["rest"] else None, labels=labels,
                scale=torch.tensor(case["scale"], device="cuda"))


def _inputs(case, seed):
    if case["op"] in ("rotate", "norm"):
        return _heads_inputs(case, seed)
    if case["op"] == "top":
        return dict(logits=_logits(_generator(seed), case))
    return _distill_inputs(case, seed)


BASE, EPS = 1000000.0, 1e-6


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case["op"] in ("rotate", "norm"):
        if own:
            from patrickstar_amd import RotaryPlan

            state["plan"] = RotaryPlan(case["rotary"], BASE, sections=_sections(case), interleaved=case["interleaved"], device="cuda")
        else:
            state["steps"], state["axis"] = _plain_steps(case)
    if own and case.get("train"):
        for name in ("q", "k", "q_weight", "k_weight", "logits"):
            if name in state:
                state[name] = state[name].detach().requires_grad_()
    return state


# -------------------------------------------------------------------------------------------------- the plain forms


def _plain_steps(case):
    """How far one position turns every pair, in units of 2**-64 of a turn, and the pair's axis."""
    steps = []
    for i in range(case["rotary"] // 2):
        step = int(BASE ** (-2.0 * i / case["rotary"]) / (2 * math.pi) * 2.0**64)
        steps.append(step - (1 << 64) if step >= 1 << 63 else step)
    sections = _sections(case) or (case["rotary"] // 2,)
    axis = [a for a, count in enumerate(sections) for _ in range(count)]
    return torch.tensor(steps, device="cuda"), torch.tensor(axis, device="cuda")


def _plain_cos_sin(state):
    positions = state["positions"]
    if state["case"]["axes"] == 1:
        positions = positions.unsqueeze(0)
    at = positions[state["axis"]].movedim(0, -1)  # batch, seq, pair
    phase = (at * state["steps"]) >> 32  # of a turn, modulo one turn: whole numbers that wrap around
    angle = phase.float() * (2 * math.pi / 2.0**32)
    return angle.cos().unsqueeze(-2), angle.sin().unsqueeze(-2)


def _plain_turn(case, x, cos, sin):
    r = case["rotary"]
    out = x.clone()
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        out[..., 0:r:2], out[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., : r // 2], x[..., r // 2 : r]
        out[..., : r // 2], out[..., r // 2 : r] = a * cos - b * sin, b * cos + a * sin
    return out


def _plain_heads(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    cos, sin = _plain_cos_sin(state)
    out = []
    normed = {}
    for name in ("q", "k"):
        x = state[name].float()
        if case["op"] == "norm":
            r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
            normed[name] = (x, r)
            x = x * r * state[name + "_weight"].float()
        out.append(_plain_turn(case, x, cos, sin).to(dtype))
    if not case["train"]:
        return out
    weights = []
    for name in ("q", "k"):
        g = _plain_turn(case, state[name + "_grad"].float(), cos, -sin)
        if case["op"] == "norm":
            x, r = normed[name]
            weights.append((g * x * r).sum((0, 1, 2)).to(dtype))
            g = g * state[name + "_weight"].float()
            g = r * g - x * (r * r * r * (x * g).mean(-1, keepdim=True))
        out.append(g.to(dtype))
    return out + weights


def _plain_top(state):
    case = state["case"]
    logits = state["logits"]
    x = logits.float()
    values, places = x.sort(dim=-1, descending=True, stable=True)
    k = min(case["k"], case["vocab"])
    x = x / case["temperature"]
    top = x.amax(-1, keepdim=True)
    lse = (x - top).exp().sum(-1).log() + top.squeeze(-1)
    return values[:, :k].to(logits.dtype), places[:, :k].int(), lse


def _plain_distill(state):
    case = state["case"]
    t, a = case["temperature"], case["label_weight"]
    z = state["logits"].float()
    counted = state["labels"] != -100
    there = state["ids"] >= 0
    places = state["ids"].clamp(min=0).long()
    x = z / t
    x = x - x.amax(-1, keepdim=True)
    total = x.exp().sum(-1, keepdim=True)
    log_q = x - total.log()
    q = log_q.exp()
    values = state["values"].float() / t
    if case["rest"]:
        p = (values - state["lse"][:, None]).exp()
        rest = (1 - p.sum(-1)).clamp(min=0)
        off = torch.ones_like(q).scatter_(-1, places, 0.0)
        q_rest = (q * off).sum(-1)
    else:
        values = values.masked_fill(~there, -math.inf)
        p = (values - values.amax(-1, keepdim=True)).exp()
        p = p / p.sum(-1, keepdim=True)
    term = torch.where(p > 0, p * (p.log() - log_q.gather(-1, places)), 0.0)
    loss = term.sum(-1)
    if case["rest"]:
        loss = loss + torch.where(rest > 0, rest * (rest.log() - q_rest.log()), 0.0)
    loss = loss * ((1 - a) * t * t)
    if a:
        y = z - z.amax(-1, keepdim=True)
        log_y = y - y.exp().sum(-1, keepdim=True).log()
        labels = state["labels"].clamp(min=0)[:, None]
        loss = loss - a * log_y.gather(-1, labels).squeeze(-1)
    share = counted / counted.sum().clamp(min=1)
    loss = loss.masked_fill(~counted, 0.0)
    if not case["train"]:
        return [loss]
    loss = (loss * share).sum()
    grad = q
    if case["rest"]:
        grad = q * torch.where(off > 0, (1 - rest / q_rest)[:, None], 1.0)
    grad = grad.scatter_add(-1, places, -p) * ((1 - a) * t)
    if a:
        grad = grad + a * log_y.exp().scatter_add(-1, labels, torch.full_like(labels, -1, dtype=torch.float))
    return [loss, (grad * (share * state["scale"])[:, None]).to(state["logits"].dtype)]


# -------------------------------------------------------------------------------------------------------------- run


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"rotate": _plain_heads, "norm": _plain_heads, "top": _plain_top, "distill": _plain_distill}[op](state)
    import patrickstar_amd as ps

    if op == "top":
        return ps.top_logits(state["logits"], min(case["k"], case["vocab"]), temperature=case["temperature"])
    if op == "distill":
        loss = ps.distill_loss(state["logits"], state["ids"], state["values"], teacher_lse=state["lse"], labels=state["labels"],
                               label_weight=case["label_weight"], temperature=case["temperature"],
                               reduction="mean" if case["train"] else "none", grad_scale=state["scale"] if case["train"] else None)
        if not case["train"]:
            return [loss]
        return [loss.detach(), *torch.autograd.grad(loss, state["logits"], state["scale"])]
    if op == "rotate":
        weights = []
        out = ps.rotate_qk(state["q"], state["k"], state["positions"], state["plan"])
    else:
        weights = [state["q_weight"], state["k_weight"]]
        out = ps.norm_rotate_qk(state["q"], state["k"], *weights, state["positions"], state["plan"], eps=EPS)
    if not case["train"]:
        return list(out)
    grads = torch.autograd.grad(out, [state["q"], state["k"]] + weights, [state["q_grad"], state["k_grad"]])
    return [x.detach() for x in out] + list(grads)


# --------------------------------------------------------------------------------------------- what a pass must move


def work(case):
    """Bytes: every input read once, every output written once.  Flops: 6 per element for a rotation, 5 for a norm, twice
    that and 6 for its gradient; 4 per logit for a softmax, 4 more for a gradient."""
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("rotate", "norm"):
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        per = 6 if case["op"] == "rotate" else 11
        reads = n * size
        if case["train"]:  # a rotation's gradient is a rotation of the gradient
            return {"bytes": 4 * reads + 8 * tokens * case["axes"], "flops": (2 * per if case["op"] == "rotate" else 3 * per) * n}
        return {"bytes": 2 * reads + 8 * tokens * case["axes"], "flops": per * n}
    n = case["rows"] * case["vocab"]
    k = min(case["k"], case["vocab"])
    if case["op"] == "top":
        return {"bytes": n * size + case["rows"] * (k * (size + 4) + 4), "flops": 5 * n}
    both = 2 if case["train"] else 1
    passes = 2 if 0 < case["label_weight"] < 1 and case["temperature"] != 1 else 1
    return {"bytes": both * n * size + case["rows"] * (k * (size + 4) + 16), "flops": 4 * both * passes * n}


# ----------------------------------------------------------------------------- the operators' definition, in 64 bits


def _exact_heads(case, given):
    r, pairs = case["rotary"], case["rotary"] // 2
    freq = BASE ** (-2.0 * torch.arange(pairs, dtype=torch.float64, device="cuda") / r)
    sections = _sections(case) or (pairs,)
    positions = given["positions"] if case["axes"] > 1 else given["positions"][None]
    angles = torch.cat([positions[i][..., None].double() * part for i, part in enumerate(freq.split(sections))], -1)
    turn = torch.polar(torch.ones_like(angles), angles).unsqueeze(-2)  # unit complex numbers: batch, seq, 1, pair

    def turned(x, turn):
        head, tail = x[..., :r], x[..., r:]
        if case["interleaved"]:
            z = torch.view_as_complex(head.reshape(*head.shape[:-1], pairs, 2)) * turn
            head = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(head[..., :pairs], head[..., pairs:]) * turn
            head = torch.cat([z.real, z.imag], -1)
        return torch.cat([head, tail], -1)

    forward, backward, weights = [], [], []
    for name in ("q", "k"):
        x = given[name].double()
        if case["op"] == "rotate":
            forward.append(turned(x, turn))
            if case["train"]:
                backward.append(turned(given[name + "_grad"].double(), turn.conj()))
            continue
        w = given[name + "_weight"].double()
        rms = torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS)
        unit = x / rms
        forward.append(turned(unit * w, turn))
        if case["train"]:
            g = turned(given[name + "_grad"].double(), turn.conj())
            weights.append((g * unit).flatten(0, 2).sum(0))
            g = g * w
            backward.append((g - unit * (g * unit).sum(-1, keepdim=True) / case["dim"]) / rms)
    return forward + backward + weights


def _exact_top(case, given):
    logits = given["logits"]
    n, v = logits.shape
    k = min(case["k"], v)
    lse = torch.empty(n, dtype=torch.float64, device="cuda")
    places = torch.empty(n, k, dtype=torch.int32, device="cuda")
    index = torch.arange(v, device="cuda")
    step = max(1, (1 << 26) // v)
    for lo in range(0, n, step):
        part = logits[lo : lo + step].float()
        lse[lo : lo + step] = torch.logsumexp(part.double() / case["temperature"], -1)
        # whole numbers in the order of the values (zeros of both signs alike), lower places in front of higher ones
        bits = (part + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        places[lo : lo + step] = (order * (1 << 24) - index).topk(k, dim=-1).indices.int()
    return logits.gather(-1, places.long()), places, lse


def _exact_distill(case, given):
    t, a = case["temperature"], case["label_weight"]
    logits, labels = given["logits"], given["labels"]
    n, v = logits.shape
    count = max(1, int((labels != -100).sum()))
    rows = torch.empty(n, dtype=torch.float64, device="cuda")
    grad = torch.empty(n, v, dtype=torch.float64, device="cuda") if case["train"] else None
    step = max(1, (1 << 26) // v)
    for lo in range(0, n, step):
        z = logits[lo : lo + step].double()
        ids = given["ids"][lo : lo + step].long()
        values = given["values"][lo : lo + step].double() / t
        label = labels[lo : lo + step]
        counted = (label != -100).double()
        # the teacher's probabilities over the whole vocabulary, and a column more for places without a token
        full = torch.zeros(z.shape[0], v + 1, dtype=torch.float64, device="cuda")
        on_list = torch.zeros_like(full)
        slot = torch.where(ids < 0, v, ids)
        on_list.scatter_(1, slot, 1.0)
        full.scatter_(1, slot, torch.exp(values - given["lse"][lo : lo + step, None].double()) if case["rest"] else torch.exp(values))
        full, on_list = full[:, :v], on_list[:, :v]
        q = torch.softmax(z / t, -1)
        log_q = torch.log_softmax(z / t, -1)
        if not case["rest"]:
            full = full / full.sum(1, keepdim=True)
        kl = (torch.xlogy(full, full) - full * log_q).sum(1)
        g = q - full
        if case["rest"]:
            p_rest = (1 - full.sum(1)).clamp(min=0)
            q_rest = (q * (1 - on_list)).sum(1)
            kl = kl + torch.xlogy(p_rest, p_rest) - torch.xlogy(p_rest, q_rest)
            g = g - (1 - on_list) * q * (p_rest / q_rest)[:, None]
        row = (1 - a) * t * t * kl
        g = (1 - a) * t * g
        if a:
            at = label.clamp(min=0)[:, None]
            row = row - a * torch.log_softmax(z, -1).gather(1, at)[:, 0]
            hard = torch.softmax(z, -1)
            hard.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float64))
            g = g + a * hard
        rows[lo : lo + step] = row * counted
        if grad is not None:
            grad[lo : lo + step] = g * (counted * (case["scale"] / count))[:, None]
    return [rows.sum() / count, grad] if case["train"] else [rows]


def exact(case, seed):
    given = _inputs(case, seed)
    if case["op"] == "top":
        return _exact_top(case, given)
    return _exact_distill(case, given) if case["op"] == "distill" else _exact_heads(case, given)
