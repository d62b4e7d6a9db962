"""What of the operators needs no GPU: plans, descriptors, refusals at the C entry points."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

import patrickstar_amd as ps
from patrickstar_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def header():
    return re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ps_ops.h")).read(), flags=re.S)


def test_every_declared_operator_is_exported_and_bound():
    declared = set(re.findall(r"\b(ps_[a-z0-9_]+)\s*\(", header()))
    assert declared == set(_lib.OP_SIGNATURES)
    lib = _lib.load()
    assert all(hasattr(lib, name) for name in declared)


def test_descriptors_have_the_headers_layout(tmp_path):
    structs = ("ps_heads_call", "ps_top_call", "ps_distill_call")
    lines = []
    for s in structs:
        lines.append(f'printf("{s} %zu\\n", sizeof({s}));')
        lines += [f'printf("{s}.{f[0]} %zu\\n", offsetof({s}, {f[0]}));' for f in getattr(_lib, s)._fields_]
    source = tmp_path / "layout.c"
    source.write_text('#include <stdio.h>\n#include "ps_ops.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Wextra", "-pedantic", "-Werror", "-I", os.path.join(ROOT, "include"), str(source), "-o",
                           str(tmp_path / "layout")])
    for line in subprocess.check_output([str(tmp_path / "layout")], text=True).splitlines():
        name, size = line.split()
        if "." in name:
            s, field = name.split(".")
            assert getattr(getattr(_lib, s), field).offset == int(size), name
        else:
            assert ctypes.sizeof(getattr(_lib, name)) == int(size), name


def test_plan_steps_are_fractions_of_a_turn():
    plan = ps.RotaryPlan(64, 10000.0, device="cpu")
    for i, step in enumerate(plan.steps):
        turns = 10000.0 ** (-2.0 * i / 64) / (2 * math.pi)
        assert abs(step / 2.0**64 - turns) <= 2.0**-53
    assert plan.axes == 1 and plan.axis_of_pair == [0] * 32
    assert plan.table.tolist() == [[s, 0] for s in plan.steps] and plan.table.dtype == torch.int64
    # faster than a turn a position, the other way round, half a turn: all modulo one turn, as signed numbers
    plan = ps.RotaryPlan(8, inv_freq=[7.0, -1.0, math.pi, 0.0], device="cpu")
    for step, f in zip(plan.steps, (7.0, -1.0, math.pi, 0.0)):
        assert -(1 << 63) <= step < 1 << 63
        off = (step / 2.0**64 - f / (2 * math.pi)) % 1.0
        assert min(off, 1 - off) <= 2.0**-51


def test_plan_axes():
    plan = ps.RotaryPlan(16, sections=(2, 3, 3), device="cpu")
    assert plan.axis_of_pair == [0, 0, 1, 1, 1, 2, 2, 2] and plan.axes == 3
    plan = ps.RotaryPlan(16, sections=(2, 3, 3), cycled=True, device="cpu")
    assert plan.axis_of_pair == [0, 1, 2, 0, 1, 2, 1, 2]
    plan = ps.RotaryPlan(16, sections=(5, 0, 3), cycled=True, device="cpu")
    assert plan.axis_of_pair == [0, 2, 0, 2, 0, 2, 0, 0]


@pytest.mark.parametrize("arguments", [
    dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=-2), dict(rotary_dim=2.0), dict(rotary_dim=True), dict(rotary_dim=514),
    dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, base=math.inf), dict(rotary_dim=8, base=math.nan),
    dict(rotary_dim=8, inv_freq=[1.0] * 3), dict(rotary_dim=8, inv_freq=[1.0, 1.0, 1.0, math.inf]),
    dict(rotary_dim=8, sections=()), dict(rotary_dim=8, sections=(1, 2)), dict(rotary_dim=8, sections=(5, -1)),
])
def test_plan_refusals(arguments):
    with pytest.raises(ValueError):
        ps.RotaryPlan(device="cpu", **arguments)


def test_tensors_off_the_gpu_are_refused():
    plan = ps.RotaryPlan(8, device="cpu")
    x, at = torch.zeros(2, 1, 8), torch.arange(2)
    w = torch.ones(8)
    for call in (lambda: ps.rotate_qk(x, x, at, plan), lambda: ps.norm_rotate_qk(x, x, w, w, at, plan), lambda: ps.top_logits(x, 2),
                 lambda: ps.distill_loss(x, torch.zeros(2, 1, 3, dtype=torch.int32), torch.zeros(2, 1, 3))):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call()


def heads_call(**changes):
    """A call that passes every check (its addresses are never used: a call that is refused launches nothing)."""
    c = _lib.ps_heads_call()
    for field, value in dict(batch=1, tokens=4, dim=64, rotary=64, axes=1, dtype=_lib.PS_F16, weight_dtype=_lib.PS_F16, position_bytes=8,
                             eps=1e-6, positions=1 << 20, plan=1 << 20).items():
        setattr(c, field, value)
    c.heads[0] = 2
    c.x[0] = c.out[0] = c.grad[0] = 1 << 20
    for field, value in changes.items():
        if isinstance(value, tuple):
            getattr(c, field)[value[0]] = value[1]
        else:
            setattr(c, field, value)
    return c


@pytest.mark.parametrize("changes", [
    dict(dtype=3), dict(dtype=-1), dict(weight_dtype=_lib.PS_BF16), dict(position_bytes=2), dict(dim=0), dict(dim=513), dict(rotary=7), dict(rotary=66),
    dict(rotary=-2), dict(axes=0), dict(batch=-1), dict(tokens=-1), dict(heads=(0, -1)), dict(heads=(1, 1 << 21)), dict(batch=1 << 20, tokens=1 << 20),
    dict(batch=1 << 62, tokens=8), dict(eps=-1.0), dict(eps=math.nan), dict(x=(0, None)), dict(out=(0, None)), dict(positions=None), dict(plan=None),
    dict(heads=(1, 1)), dict(weight_grad=(0, 1 << 20)), dict(x=(0, (1 << 20) + 1)), dict(out=(0, (1 << 20) + 1)), dict(x=(0, (1 << 20) + 2), dtype=_lib.PS_F32, weight_dtype=_lib.PS_F32),
])
def test_heads_calls_that_are_refused(changes):
    lib = _lib.load()
    c = heads_call(**changes)
    assert lib.ps_rotate_heads(_lib.address(c), None) == _lib.PS_ERR_BAD_ARG
    assert lib.ps_last_error()
    assert lib.ps_norm_rotate_heads_workspace_bytes(_lib.address(c)) == 0
    assert lib.ps_norm_rotate_heads_backward(_lib.address(c), None, 0, None) == _lib.PS_ERR_BAD_ARG


def test_a_workspace_that_is_too_small_is_refused():
    lib = _lib.load()
    c = heads_call(weight=(0, 1 << 20), weight_grad=(0, 1 << 20))
    size = lib.ps_norm_rotate_heads_workspace_bytes(_lib.address(c))
    assert size > 0
    for at, given in ((1 << 20, size - 1), (None, size), ((1 << 20) + 4, size)):
        assert lib.ps_norm_rotate_heads_backward(_lib.address(c), at, given, None) == _lib.PS_ERR_BAD_ARG
        assert b"workspace" in lib.ps_last_error()
    assert lib.ps_norm_rotate_heads_backward(_lib.address(heads_call(grad=(0, None))), None, 0, None) == _lib.PS_ERR_BAD_ARG


def test_calls_without_work_launch_nothing():
    lib = _lib.load()
    for c in (heads_call(tokens=0), heads_call(batch=0), heads_call(heads=(0, 0))):
        assert lib.ps_rotate_heads(_lib.address(c), None) == 0
    top = _lib.ps_top_call()
    top.vocab, top.k, top.temperature = 10, 3, 1.0
    assert lib.ps_top_logits(_lib.address(top), None) == 0


def top_call(**changes):
    c = _lib.ps_top_call()
    fields = dict(rows=2, vocab=100, row_stride=100, k=5, dtype=_lib.PS_F16, temperature=1.0)
    fields.update({name: 1 << 20 for name in ("logits", "values", "ids", "lse")})
    for field, value in {**fields, **changes}.items():
        setattr(c, field, value)
    return c


@pytest.mark.parametrize("changes", [
    dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(k=0), dict(k=101), dict(k=1025, vocab=5000), dict(dtype=9), dict(temperature=0.0),
    dict(temperature=math.nan), dict(temperature=math.inf), dict(logits=None), dict(logits=(1 << 20) + 1), dict(values=None), dict(ids=None), dict(lse=None),
])
def test_top_calls_that_are_refused(changes):
    lib = _lib.load()
    assert lib.ps_top_logits(_lib.address(top_call(**changes)), None) == _lib.PS_ERR_BAD_ARG
    assert lib.ps_last_error()


def distill_call(**changes):
    c = _lib.ps_distill_call()
    fields = dict(rows=2, vocab=100, row_stride=100, k=5, ids_stride=5, values_stride=5, dtype=_lib.PS_F16, values_dtype=_lib.PS_F16, ids_bytes=4,
                  temperature=1.0)
    fields.update({name: 1 << 20 for name in ("logits", "ids", "values", "row_loss", "stats", "denominator", "grad", "upstream")})
    for field, value in {**fields, **changes}.items():
        setattr(c, field, value)
    return c


@pytest.mark.parametrize("changes", [
    dict(rows=-1), dict(vocab=0), dict(vocab=400001), dict(k=0), dict(k=1025), dict(dtype=4), dict(values_dtype=-1), dict(ids_bytes=2),
    dict(labels=1 << 20, labels_bytes=1), dict(temperature=-1.0), dict(label_weight=-0.1), dict(label_weight=1.1), dict(label_weight=math.nan),
    dict(label_weight=0.5), dict(logits=None), dict(logits=(1 << 20) + 1), dict(ids=None), dict(values=None), dict(mean=1, denominator=None),
])
def test_distill_calls_that_are_refused(changes):
    lib = _lib.load()
    c = distill_call(**changes)
    assert lib.ps_distill_loss(_lib.address(c), None) == _lib.PS_ERR_BAD_ARG
    assert lib.ps_last_error()
    assert lib.ps_distill_loss_backward(_lib.address(c), None) == _lib.PS_ERR_BAD_ARG


def test_distill_calls_that_lack_what_one_direction_needs():
    lib = _lib.load()
    assert lib.ps_distill_loss(_lib.address(distill_call(row_loss=None)), None) == _lib.PS_ERR_BAD_ARG
    for name in ("grad", "stats", "upstream"):
        assert lib.ps_distill_loss_backward(_lib.address(distill_call(**{name: None})), None) == _lib.PS_ERR_BAD_ARG
    for call in (lib.ps_rotate_heads, lib.ps_top_logits, lib.ps_distill_loss, lib.ps_distill_loss_backward):
        assert call(None, None) == _lib.PS_ERR_BAD_ARG
