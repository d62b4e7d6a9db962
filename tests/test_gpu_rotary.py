"""Rotations and norms of queries and keys against their formulas in 64 bits, forward and backward.

Tolerances.  One rounding to the type at the end: half a unit in the last place of the result (``HALF_ULP``).  In front of it
32-bit arithmetic: cosines and sines within 2e-7 (their polynomials 2e-9, their evaluation and the angle's rounding to 24 bits one
or two last places each), and up to eight roundings of a term, so 2**-20 of the sum of the terms' magnitudes holds all of it.  A sum of n
terms in 32 bits, in whatever order, adds n * 2**-24 of the sum of their magnitudes, n being how many one lane adds up before the tree."""
import math

import pytest
import torch

import patrickstar_amd as ps
from patrickstar_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["compiled", "general"], autouse=True)
def way(request, monkeypatch):
    """Both ways to the library: the binding's calls, and the Python ones that take over where a call is not of the ordinary form."""
    lib = _lib.load()
    assert lib.ops is not None
    if request.param == "general":
        monkeypatch.setattr(lib, "ops", None)

HALF_ULP = {torch.half: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float: 2.0**-24}
TINY = {torch.half: 2.0**-25, torch.bfloat16: 0.0, torch.float: 0.0}  # half of the smallest number below the normal ones
DTYPES = list(HALF_ULP)


def angles(positions, plan):
    """[..., pairs] in 64 bits, reduced in whole numbers: positions of any size."""
    steps = [s % (1 << 64) for s in plan.steps]
    flat = positions.cpu().reshape(plan.axes, -1).tolist()
    rows = []
    for token in range(len(flat[0])):
        rows.append([(flat[a][token] * s) % (1 << 64) / 2.0**64 * 2 * math.pi for a, s in zip(plan.axis_of_pair, steps)])
    return torch.tensor(rows, dtype=torch.float64, device=positions.device)


def turned(x, angle, plan):
    r, p = plan.rotary_dim, plan.rotary_dim // 2
    c, s = angle.cos(), angle.sin()
    out = x.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if plan.interleaved else (slice(0, p), slice(p, r))
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    return out


def magnitude(x, plan):
    """|a| + |b| of every element's pair."""
    r, p = plan.rotary_dim, plan.rotary_dim // 2
    out = x.abs().clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if plan.interleaved else (slice(0, p), slice(p, r))
    both = x[..., first].abs() + x[..., second].abs()
    out[..., first], out[..., second] = both, both
    return out


def close(got, want, size, what, slack=2.0**-20):
    dtype = got.dtype
    off = (got.double() - want).abs()
    allowed = HALF_ULP[dtype] * want.abs() + slack * size + TINY[dtype]
    allowed = allowed * (1 + 2.0**-10)
    bad = ~(off <= allowed)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} are off, by up to {float((off / allowed.clamp(min=1e-300)).max()):.3g} times the allowed"


def made(shape, dtype, seed, std=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, device="cuda").normal_(0, std, generator=gen).to(dtype)


# batch, tokens, heads, kv_heads, dim, rotary, interleaved, sections, cycled, packed
SHAPES = [
    (1, 1, 1, 1, 64, 64, False, None, False, False),
    (1, 1, 16, 4, 128, 128, False, None, False, True),
    (2, 7, 12, 12, 64, 64, False, None, False, True),
    (3, 5, 4, 1, 128, 64, False, None, False, False),
    (1, 33, 5, 5, 80, 80, False, (10, 14, 16), False, True),
    (2, 9, 3, 2, 72, 36, True, (6, 6, 6), True, False),
    (2, 6, 8, 2, 256, 256, True, (32, 48, 48), False, True),
    (1, 4, 2, 1, 512, 512, False, None, False, False),
    (1, 4, 2, 1, 512, 6, True, (1, 2), False, False),
    (1, 3, 3, 1, 37, 22, False, None, False, True),
    (1, 3, 2, 2, 7, 2, True, None, False, False),
    (1, 2, 1, 1, 511, 510, False, None, False, False),
    (2, 3, 2, 1, 96, 48, True, (0, 24), False, True),
    (5, 130, 2, 1, 32, 32, False, (4, 6, 6), True, False),
]


def inputs(shape, dtype, start=1000, seed=0):
    b, s, h, hk, d, r, interleaved, sections, cycled, packed = shape
    plan = ps.RotaryPlan(r, 10000.0, sections=sections, cycled=cycled, interleaved=interleaved)
    if packed:  # one projection's output, with something in front so that the addresses are odd
        qkv = made((b, s, (h + 2 * hk) * d + 3), dtype, seed)[..., 3:]
        q, k = qkv[..., : h * d].unflatten(-1, (h, d)), qkv[..., h * d : (h + hk) * d].unflatten(-1, (hk, d))
    else:
        q, k = made((b, s, h, d), dtype, seed), made((b, s, hk, d), dtype, seed + 1)
    lead = (b, s) if plan.axes == 1 else (plan.axes, b, s)
    gen = torch.Generator(device="cuda").manual_seed(seed + 2)
    positions = torch.randint(0, start + 1, lead, device="cuda", generator=gen)
    return q, k, positions, plan


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_rotation(shape, dtype):
    q, k, positions, plan = inputs(shape, dtype)
    out = ps.rotate_qk(q, k, positions, plan)
    angle = angles(positions, plan).view(*q.shape[:2], 1, -1)
    for got, x, name in zip(out, (q, k), "qk"):
        assert got.shape == x.shape and got.dtype == dtype and got.is_contiguous()
        close(got, turned(x.double(), angle, plan), magnitude(x.double(), plan), name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_rotation_backward(shape, dtype):
    q, k, positions, plan = inputs(shape, dtype)
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    gq, gk = made(q.shape, dtype, 7), made(k.shape, dtype, 8)
    grads = torch.autograd.grad(ps.rotate_qk(q, k, positions, plan), (q, k), (gq, gk))
    angle = -angles(positions, plan).view(*q.shape[:2], 1, -1)
    for got, g, name in zip(grads, (gq, gk), "qk"):
        close(got, turned(g.double(), angle, plan), magnitude(g.double(), plan), name)


def norm_forward(x, w, angle, plan, eps):
    r = 1.0 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    y = x * r if w is None else x * r * w
    return turned(y, angle, plan), y, r


WEIGHTS = ["own", "fp32", "none"]


@pytest.mark.parametrize("weights", WEIGHTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_and_rotation_forward_and_backward(shape, dtype, weights):
    eps = 1e-5
    q, k, positions, plan = inputs(shape, dtype, seed=3)
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    d = q.shape[-1]
    wq = wk = None
    if weights != "none":
        wq, wk = ((1 + made((d,), torch.float, n, 0.2)).to(torch.float if weights == "fp32" else dtype).requires_grad_() for n in (4, 5))
    out = ps.norm_rotate_qk(q, k, wq, wk, positions, plan, eps)
    gq, gk = made(q.shape, dtype, 7, 0.1), made(k.shape, dtype, 8, 0.1)
    wanted = [t for t in (q, k, wq, wk) if t is not None]
    grads = dict(zip(("q", "k", "wq", "wk"), torch.autograd.grad(out, wanted, (gq, gk))))
    angle = angles(positions, plan).view(*q.shape[:2], 1, -1)
    for got, x, w, g, name in zip(out, (q, k), (wq, wk), (gq, gk), "qk"):
        x64, g64 = x.detach().double(), g.double()
        w64 = None if w is None else w.detach().double()
        want, y, r = norm_forward(x64, w64, angle, plan, eps)
        close(got.detach(), want, magnitude(y, plan), name)
        dy = turned(g64, -angle, plan)
        size = magnitude(g64, plan)
        ww = torch.ones((), dtype=torch.float64, device="cuda") if w64 is None else w64
        mean = (x64 * ww * dy).mean(-1, keepdim=True)
        dx = r * (ww * dy - x64 * r * r * mean)
        spread = r * (ww.abs() * size + x64.abs() * r * r * (x64 * ww * size).abs().mean(-1, keepdim=True))
        close(grads[name], dx, spread, "d" + name)
        if w is not None:
            term = dy * x64 * r
            sizes = (size * (x64 * r).abs()).sum((0, 1, 2))
            n = x.shape[0] * x.shape[1] * x.shape[2]
            close(grads["w" + name], term.sum((0, 1, 2)), sizes, "dw" + name, slack=2.0**-20 + min(n, 256) * 2.0**-24)


def test_gradients_against_differences():
    """Along a direction, the loss's difference quotient in 64 bits of the operator's own fp32 outputs.  Step 2**-7: the third
    derivative's part is of the order of 2**-14, the outputs' rounding 2**-24 / 2**-7 = 2**-17 of their size."""
    shape = (2, 5, 4, 2, 64, 48, False, (6, 9, 9), False, False)
    q, k, positions, plan = inputs(shape, torch.float, seed=11)
    wq, wk = 1 + made((64,), torch.float, 12, 0.2), 1 + made((64,), torch.float, 13, 0.2)
    given = [t.requires_grad_() for t in (q, k, wq, wk)]
    g = [made(q.shape, torch.float, 14), made(k.shape, torch.float, 15)]
    grads = torch.autograd.grad(ps.norm_rotate_qk(*given, positions, plan), given, g)
    h = 2.0**-7
    for i, t in enumerate(given):
        v = made(t.shape, torch.float, 20 + i)
        value = []
        with torch.no_grad():
            for sign in (1, -1):
                moved = [x if j != i else x + sign * h * v for j, x in enumerate(given)]
                value.append(sum((o.double() * gg.double()).sum() for o, gg in zip(ps.norm_rotate_qk(*moved, positions, plan), g)))
        quotient = float(value[0] - value[1]) / (2 * h)
        along = float((grads[i].double() * v.double()).sum())
        assert abs(quotient - along) <= 2e-3 * float(grads[i].double().norm() * v.double().norm()) ** 1.0, i


@pytest.mark.parametrize("start", [2**20 + 1, 2**31 + 5, 2**53 + 1, -(2**40) - 3])
@pytest.mark.parametrize("base", [10000.0, 5e6])
def test_positions_of_any_size_are_exact(start, base):
    plan = ps.RotaryPlan(64, base)
    q = made((9, 2, 64), torch.float, 1)
    positions = start + torch.arange(9, device="cuda")
    got, none = ps.rotate_qk(q, None, positions, plan)
    assert none is None
    close(got, turned(q.double(), angles(positions, plan).view(9, 1, -1), plan), magnitude(q.double(), plan), "q")


def test_int32_positions_and_expansion_give_the_same_bits():
    q, k, positions, plan = inputs((3, 6, 4, 2, 64, 64, False, (8, 12, 12), False, False), torch.half)
    positions = positions[:, :1]  # one row for all batches
    want = ps.rotate_qk(q, k, positions.expand(3, 3, 6).contiguous(), plan)
    for other in (positions, positions[:, 0], positions.int(), positions.expand(3, 3, 6), positions.transpose(1, 2).contiguous().transpose(1, 2)):
        for a, b in zip(ps.rotate_qk(q, k, other, plan), want):
            assert torch.equal(a, b)


def test_layouts_give_the_same_bits():
    """Heads in front of tokens, a head's elements apart, a batch that is one tensor seen again, three dimensions."""
    q, k, positions, plan = inputs((3, 6, 4, 2, 64, 64, False, None, False, False), torch.bfloat16)
    w = 1 + made((64,), torch.bfloat16, 5, 0.2)
    want = ps.norm_rotate_qk(q, k, w, w, positions, plan)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k)]
    apart = [torch.stack([x, x], -1)[..., 0] for x in (q, k)]
    for a, b in (heads_first, apart):
        for got, x in zip(ps.norm_rotate_qk(a, b, w, w, positions, plan), want):
            assert torch.equal(got, x)
    one = ps.norm_rotate_qk(q[:1].expand(3, -1, -1, -1), k[:1].expand(3, -1, -1, -1), w, w, positions[:1].expand(3, -1), plan)
    flat = ps.norm_rotate_qk(q[0], k[0], w, w, positions[0], plan)
    for a, b, x in zip(one, flat, want):
        assert all(torch.equal(a[i], x[0]) for i in range(3)) and torch.equal(b, x[0])


def test_gradients_that_are_broadcast_or_strided():
    q, k, positions, plan = inputs((2, 6, 4, 2, 64, 64, False, None, False, False), torch.half)
    w = (1 + made((64,), torch.half, 5, 0.2)).requires_grad_()
    q, k = q.requires_grad_(), k.requires_grad_()
    out = ps.norm_rotate_qk(q, k, w, w, positions, plan)
    ones = torch.ones((), dtype=torch.half, device="cuda")
    want = torch.autograd.grad(out, (q, k, w), [torch.ones_like(x) for x in out], retain_graph=True)
    got = torch.autograd.grad(out, (q, k, w), [ones.expand(x.shape) for x in out], retain_graph=True)
    turned_round = torch.autograd.grad(out, (q, k, w), [torch.ones_like(x).transpose(1, 3).contiguous().transpose(1, 3) for x in out])
    for a, b, c in zip(got, want, turned_round):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_an_output_that_goes_nowhere():
    q, k, positions, plan = inputs((2, 6, 4, 2, 64, 64, False, None, False, False), torch.float)
    wq, wk = ((1 + made((64,), torch.float, n, 0.2)).requires_grad_() for n in (4, 5))
    q, k = q.requires_grad_(), k.requires_grad_()
    g = made(q.shape, torch.float, 6)
    both = torch.autograd.grad(ps.norm_rotate_qk(q, k, wq, wk, positions, plan), (q, wq), (g, torch.zeros_like(k)))
    out = ps.norm_rotate_qk(q, k, wq, wk, positions, plan)[0]
    alone = torch.autograd.grad(out, (q, k, wq, wk), g, allow_unused=True)
    assert alone[1] is None and alone[3] is None
    assert torch.equal(alone[0], both[0])
    angle = angles(positions, plan).view(2, 6, 1, -1)
    term = turned(g.double(), -angle, plan) * q.detach().double() / (q.detach().double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
    for weight_grad in (alone[2], both[1]):  # (the heads are dealt to the lanes in another way: not the same bits)
        close(weight_grad, term.sum((0, 1, 2)), (magnitude(g.double(), plan) * 6).sum((0, 1, 2)), "dwq", slack=2.0**-18)
    turned_q = torch.autograd.grad(ps.rotate_qk(q, k, positions, plan)[1], (q, k), torch.ones_like(k), allow_unused=True)
    assert turned_q[0] is None and turned_q[1].shape == k.shape


def test_rows_of_zeros_infinities_and_nan_stay_their_own():
    q, k, positions, plan = inputs((1, 8, 4, 2, 64, 64, False, None, False, False), torch.half, seed=9)
    w = 1 + made((64,), torch.half, 5, 0.2)
    clean = ps.norm_rotate_qk(q, k, w, w, positions, plan)
    q = q.clone()
    q[0, 1, 2] = 0
    q[0, 2, 0, 5] = float("inf")
    q[0, 3, 3, 7] = float("nan")
    got = ps.norm_rotate_qk(q, k, w, w, positions, plan)
    assert (got[0][0, 1, 2] == 0).all()
    assert got[0][0, 2, 0].isnan().any() and got[0][0, 3, 3].isnan().all()
    untouched = torch.ones(8, 4, dtype=torch.bool, device="cuda")
    untouched[1, 2] = untouched[2, 0] = untouched[3, 3] = False
    assert torch.equal(got[0][0][untouched], clean[0][0][untouched]) and torch.equal(got[1], clean[1])
    x = torch.zeros(1, 1, 64, dtype=torch.float, device="cuda", requires_grad=True)
    out, _ = ps.norm_rotate_qk(x, None, None, None, positions[0, :1], plan)
    (g,) = torch.autograd.grad(out, x, torch.ones_like(x))
    assert g.isfinite().all()


def test_a_gradient_is_not_differentiated_in_silence():
    q, k, positions, plan = inputs((2, 6, 4, 2, 64, 64, False, None, False, False), torch.float)
    w = torch.ones(64, device="cuda", requires_grad=True)
    q = q.requires_grad_()
    for out in (ps.rotate_qk(q, k, positions, plan)[0], ps.norm_rotate_qk(q, k, w, w, positions, plan)[0]):
        (g,) = torch.autograd.grad(out.square().sum(), q, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate"):
            g.sum().backward()


def test_no_tokens_and_no_heads():
    plan = ps.RotaryPlan(64)
    w = torch.ones(64, device="cuda", requires_grad=True)
    q = torch.empty(0, 4, 64, device="cuda", requires_grad=True)
    out = ps.norm_rotate_qk(q, None, w, None, torch.empty(0, dtype=torch.int64, device="cuda"), plan)[0]
    gq, gw = torch.autograd.grad(out, (q, w), out.detach())
    assert out.shape == q.shape and gq.shape == q.shape and (gw == 0).all()
    x = torch.empty(5, 0, 64, device="cuda")
    y = made((5, 2, 64), torch.float, 3)
    a, b = ps.rotate_qk(x, y, torch.arange(5, device="cuda"), plan)
    assert a.shape == x.shape and torch.equal(b, ps.rotate_qk(y, None, torch.arange(5, device="cuda"), plan)[0])


def test_weight_gradients_do_not_change_from_call_to_call():
    q, k, positions, plan = inputs((4, 700, 6, 2, 64, 64, False, None, False, False), torch.half, seed=2)
    wq, wk = ((1 + made((64,), torch.half, n, 0.2)).requires_grad_() for n in (4, 5))
    first = None
    for _ in range(4):
        out = ps.norm_rotate_qk(q, k, wq, wk, positions, plan)
        grads = torch.autograd.grad(out, (wq, wk), [torch.ones_like(x) for x in out])
        first = first or grads
        assert all(torch.equal(a, b) for a, b in zip(grads, first))


def test_on_another_stream_and_in_a_graph():
    q, k, positions, plan = inputs((1, 32, 8, 2, 128, 128, False, None, False, True), torch.half)
    w = 1 + made((128,), torch.half, 5, 0.2)
    want = ps.norm_rotate_qk(q, k, w, w, positions, plan)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ps.norm_rotate_qk(q, k, w, w, positions, plan)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ps.norm_rotate_qk(q, k, w, w, positions, plan)
    for n in range(3):
        q.copy_(made(q.shape, torch.half, 30 + n))
        positions.add_(17)
        graph.replay()
        want = ps.norm_rotate_qk(q, k, w, w, positions, plan)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    plan = ps.RotaryPlan(64)
    q, k = made((5, 4, 64), torch.half, 1), made((5, 2, 64), torch.half, 2)
    at = torch.arange(5, device="cuda")
    w = torch.ones(64, dtype=torch.half, device="cuda")
    for error, call in [
        (TypeError, lambda: ps.rotate_qk(q, k, at, None)),
        (RuntimeError, lambda: ps.rotate_qk(q.cpu(), k, at, plan)),
        (RuntimeError, lambda: ps.rotate_qk(q, k, at.cpu(), plan)),
        (RuntimeError, lambda: ps.rotate_qk(q, k, at, ps.RotaryPlan(64, device="cpu"))),
        (TypeError, lambda: ps.rotate_qk(q.double(), k, at, plan)),
        (TypeError, lambda: ps.rotate_qk(q, k.float(), at, plan)),
        (TypeError, lambda: ps.rotate_qk(q, k, at.float(), plan)),
        (ValueError, lambda: ps.rotate_qk(q[0], k[0], at, plan)),
        (ValueError, lambda: ps.rotate_qk(q, k[:4], at, plan)),
        (ValueError, lambda: ps.rotate_qk(q, k[..., :32], at, plan)),
        (ValueError, lambda: ps.rotate_qk(q, k, at[:4], plan)),
        (ValueError, lambda: ps.rotate_qk(q, k, at, ps.RotaryPlan(64, sections=(16, 16)))),
        (ValueError, lambda: ps.rotate_qk(q, k, at, ps.RotaryPlan(128))),
        (ValueError, lambda: ps.rotate_qk(made((5, 1, 520), torch.half, 1), None, at, plan)),
        (ValueError, lambda: ps.norm_rotate_qk(q, k, w, w, at, plan, eps=-1.0)),
        (ValueError, lambda: ps.norm_rotate_qk(q, k, w[:32], w, at, plan)),
        (TypeError, lambda: ps.norm_rotate_qk(q, k, w.bfloat16(), w, at, plan)),
        (TypeError, lambda: ps.norm_rotate_qk(q, k, w.float(), w, at, plan)),
        (RuntimeError, lambda: ps.norm_rotate_qk(q, k, w.cpu(), w, at, plan)),
        (ValueError, lambda: ps.norm_rotate_qk(q, None, w, w, at, plan)),
    ]:
        with pytest.raises(error):
            call()


def test_more_than_two_to_the_31_elements():
    tokens, heads, dim = 140001, 120, 128
    plan = ps.RotaryPlan(dim)
    q = torch.empty(tokens, heads, dim, dtype=torch.half, device="cuda")
    q[-3:] = made((3, heads, dim), torch.half, 1)
    q[:-3] = 1.0
    at = torch.arange(tokens, device="cuda")
    w = 1 + made((dim,), torch.half, 5, 0.2)
    for whole, part in (
        (ps.rotate_qk(q, None, at, plan)[0], ps.rotate_qk(q[-3:], None, at[-3:], plan)[0]),
        (ps.norm_rotate_qk(q, None, w, None, at, plan)[0], ps.norm_rotate_qk(q[-3:], None, w, None, at[-3:], plan)[0]),
    ):
        assert whole.numel() > 2**31 and torch.equal(whole[-3:], part)
