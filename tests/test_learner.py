"""The learner layers without a GPU: the 64-bit definitions' gradients against differences, and what the entry points
refuse before they touch a device."""
from __future__ import annotations

import copy
import os
import pickle
import subprocess

import pytest

import turbinator_c_b200 as tb
from tests import learner_reference as ref

torch = pytest.importorskip("torch")


def _f64(gen, *shape):
    return torch.randn(shape, generator=gen, dtype=torch.float64)


def _directional(f, x, d, step=1e-6):
    return (f(x + step * d) - f(x - step * d)) / (2 * step)


@pytest.mark.parametrize("act", ("none", "silu", "gelu", "relu"))
def test_group_norm_gradient_is_the_difference(act):
    gen = torch.Generator().manual_seed(2)
    x, dy, gamma, beta = _f64(gen, 2, 5, 12), _f64(gen, 2, 5, 12), _f64(gen, 12), _f64(gen, 12)
    _, mean, rstd = ref.group_norm(x, gamma, beta, 3, 1e-5, act)
    (dx, dgamma, dbeta), _ = ref.group_norm_backward(x, gamma, beta, mean, rstd, dy, 3, act)
    loss = lambda x, g, b: (ref.group_norm(x, g, b, 3, 1e-5, act)[0] * dy).sum()  # noqa: E731
    d, dg, db = _f64(gen, 2, 5, 12), _f64(gen, 12), _f64(gen, 12)
    assert torch.allclose((dx * d).sum(), _directional(lambda v: loss(v, gamma, beta), x, d), rtol=1e-6, atol=1e-7)
    assert torch.allclose((dgamma * dg).sum(), _directional(lambda v: loss(x, v, beta), gamma, dg), rtol=1e-6, atol=1e-7)
    assert torch.allclose((dbeta * db).sum(), _directional(lambda v: loss(x, gamma, v), beta, db), rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("resets,ragged", [(False, False), (True, False), (False, True), (True, True)])
def test_recurrence_gradient_is_the_difference(resets, ragged):
    gen = torch.Generator().manual_seed(3)
    b, t, d = 3, 21, 4
    v = {n: _f64(gen, b, t, d) for n in ("x", "rec", "inp")}
    v["decay"], v["state"] = _f64(gen, d) - 2, _f64(gen, b, d)
    dh, dstate = _f64(gen, b, t, d), _f64(gen, b, d)
    reset = (torch.rand((b, t), generator=gen) < 0.15).to(torch.uint8) if resets else None
    lengths = torch.tensor([0, 7, 21]) if ragged else None
    live = torch.arange(t)[None] < (lengths[:, None] if ragged else t)
    dh = dh * live[..., None]

    def run(w, back=False):
        return ref.recurrence(w["x"], w["rec"], w["inp"], w["decay"], 8.0, reset, lengths, w["state"],
                              dh if back else None, dstate)

    got = run(v, True)
    names = {"x": "dx", "rec": "drec", "inp": "dinp", "decay": "ddecay", "state": "dstate"}
    for n, grad in names.items():
        way = _f64(gen, *v[n].shape)
        loss = lambda w: (lambda o: (o["h"][0] * dh).sum() + (o["state"][0] * dstate).sum())(run({**v, n: w}))  # noqa: E731,B023
        assert torch.allclose((got[grad][0] * way).sum(), _directional(loss, v[n], way), rtol=1e-6, atol=1e-7), n


@pytest.mark.parametrize("kind", ("softmax", "sigmoid"))
@pytest.mark.parametrize("renormalise", (False, True))
def test_route_weights_gradient_is_the_difference(kind, renormalise):
    gen = torch.Generator().manual_seed(4)
    logits, dw = _f64(gen, 6, 9), _f64(gen, 6, 3)
    ids = ref.route(logits, None, kind, 3)[0]
    ids[0, 2] = -1
    l64 = logits.clone().requires_grad_(True)
    grad = torch.autograd.grad(ref.route_weights(l64, ids, kind, renormalise, 1.5), l64, dw)[0]
    way = _f64(gen, 6, 9)
    loss = lambda w: (ref.route_weights(w, ids, kind, renormalise, 1.5) * dw).sum()  # noqa: E731
    assert torch.allclose((grad * way).sum(), _directional(loss, logits, way), rtol=1e-6, atol=1e-8)


FAKE = 0x10000  # never dereferenced: every call below is refused first


def _norm(**change):
    return tb.GroupNormDesc(**{**dict(samples=2, positions=3, channels=8, groups=2, type=1, activation=2,
                                      epsilon=1e-5), **change})


@pytest.mark.parametrize("change", [
    dict(samples=0), dict(positions=0), dict(channels=0), dict(groups=0), dict(groups=3), dict(type=3),
    dict(activation=4), dict(activation=-1), dict(epsilon=-1.0), dict(epsilon=float("nan")),
    dict(x_position_stride=7), dict(y_position_stride=7), dict(dx_position_stride=7), dict(samples=2 ** 40), dict(positions=2 ** 62),
    dict(channels=2 ** 33, groups=1)])
def test_group_norm_refuses_descriptors(change):
    d = _norm(**change)
    assert tb.tb_cuda_group_norm_workspace(d) == 0
    assert tb.tb_cuda_group_norm_device(d, FAKE, FAKE, FAKE, 2 * FAKE, FAKE, FAKE, FAKE) == 0
    assert tb.tb_cuda_group_norm_backward_device(d, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2 * FAKE, FAKE, FAKE, FAKE) == 0


def test_group_norm_refuses_pointers():
    good = [FAKE, FAKE, FAKE, 2 * FAKE, FAKE, FAKE, FAKE]  # x gamma beta y mean rstd workspace
    for i, bad in [(0, None), (3, None), (4, None), (5, None), (0, FAKE + 1), (1, FAKE + 2),
                   (2, FAKE + 1), (3, FAKE + 1), (4, FAKE + 2), (5, FAKE + 2), (6, FAKE + 4)]:
        args = list(good)
        args[i] = bad
        assert tb.tb_cuda_group_norm_device(_norm(), *args) == 0, (i, bad)
    assert tb.tb_cuda_group_norm_device(_norm(y_position_stride=16), FAKE, None, None, FAKE, None, None, FAKE) == 0
    good = [FAKE] * 6 + [2 * FAKE] + [FAKE] * 3  # x gamma beta mean rstd dy dx dgamma dbeta workspace
    for i, bad in [(0, None), (3, None), (4, None), (5, None), (6, None), (0, FAKE + 1), (5, FAKE + 1),
                   (6, FAKE + 1), (7, FAKE + 2), (8, FAKE + 2), (9, FAKE + 8), (9, None)]:
        args = list(good)
        args[i] = bad
        assert tb.tb_cuda_group_norm_backward_device(_norm(), *args) == 0, (i, bad)
    assert tb.tb_cuda_group_norm_backward_device(_norm(dx_position_stride=16), FAKE, None, None, FAKE, FAKE, 2 * FAKE,
                                                 FAKE, None, None, FAKE) == 0
    assert tb.load_library().tb_cuda_group_norm_device(None, *good[:7], None) == 0


def _rec(**change):
    return tb.GatedRecurrenceDesc(**{**dict(sequences=2, steps=40, channels=8, type=1, decay_scale=8.0), **change})


@pytest.mark.parametrize("change", [
    dict(sequences=0), dict(steps=0), dict(channels=0), dict(type=-1), dict(decay_scale=-0.5),
    dict(decay_scale=float("nan")), dict(in_step_stride=7), dict(out_step_stride=7), dict(grad_step_stride=7),
    dict(steps=2 ** 31), dict(sequences=2 ** 30), dict(sequences=2 ** 20, channels=2 ** 20)])
def test_recurrence_refuses_descriptors(change):
    d = _rec(**change)
    assert tb.tb_cuda_gated_recurrence_workspace(d) == 0
    assert tb.tb_cuda_gated_recurrence_device(d, *[FAKE] * 7, 2 * FAKE, FAKE, FAKE, FAKE) == 0
    assert tb.tb_cuda_gated_recurrence_backward_device(d, *[FAKE] * 9, 2 * FAKE, 3 * FAKE, 4 * FAKE, FAKE, FAKE, FAKE) == 0


def test_recurrence_refuses_pointers():
    # x rec inp decay reset lengths state_in h state_out checkpoints workspace
    good = [FAKE] * 7 + [2 * FAKE] + [FAKE] * 3
    for i, bad in [(0, None), (1, None), (2, None), (3, None), (7, None), (7, FAKE), (10, FAKE + 4), (0, FAKE + 1),
                   (3, FAKE + 2), (5, FAKE + 2), (6, FAKE + 1), (8, FAKE + 2), (9, FAKE + 2)]:
        args = list(good)
        args[i] = bad
        assert tb.tb_cuda_gated_recurrence_device(_rec(), *args) == 0, (i, bad)
    # x rec inp decay reset lengths checkpoints dh dstate_out dx drec dinp ddecay dstate_in workspace
    good = [FAKE] * 9 + [2 * FAKE, 3 * FAKE, 4 * FAKE] + [FAKE] * 3
    for i, bad in [(0, None), (3, None), (6, None), (7, None), (9, None), (10, None), (11, None), (9, FAKE),
                   (10, 2 * FAKE), (11, FAKE), (14, FAKE + 8), (12, FAKE + 2), (13, FAKE + 2), (7, FAKE + 1)]:
        args = list(good)
        args[i] = bad
        assert tb.tb_cuda_gated_recurrence_backward_device(_rec(), *args) == 0, (i, bad)


def _rt(**change):
    return tb.ExpertRouteDesc(**{**dict(tokens=4, experts=8, top_k=2, groups=2, top_groups=1, group_best=2, type=0,
                                        score=1, renormalise=1, weight_scale=1.0), **change})


@pytest.mark.parametrize("change", [
    dict(tokens=0), dict(experts=0), dict(experts=1026), dict(top_k=0), dict(top_k=9), dict(groups=0),
    dict(groups=3), dict(top_groups=0), dict(top_groups=3), dict(group_best=0), dict(group_best=3), dict(type=9),
    dict(score=2), dict(weight_scale=float("nan")), dict(logits_stride=7), dict(tokens=2 ** 30),
    dict(experts=64, top_k=33)])
def test_route_refuses_descriptors(change):
    d = _rt(**change)
    assert tb.tb_cuda_route_experts_workspace(d) == 0
    assert tb.tb_cuda_route_experts_device(d, *[FAKE] * 8) == 0
    assert tb.tb_cuda_route_experts_backward_device(d, FAKE, FAKE, FAKE, 2 * FAKE) == 0


def test_route_refuses_pointers():
    # logits bias ids weights offsets order position workspace
    for i, bad in [(0, None), (2, None), (3, None), (4, None), (5, None), (6, None), (7, None), (0, FAKE + 2),
                   (1, FAKE + 2), (2, FAKE + 1), (3, FAKE + 2), (4, FAKE + 2), (5, FAKE + 2), (6, FAKE + 2),
                   (7, FAKE + 4)]:
        args = [FAKE] * 8
        args[i] = bad
        assert tb.tb_cuda_route_experts_device(_rt(), *args) == 0, (i, bad)
    for i, bad in [(0, None), (1, None), (2, None), (3, None), (3, FAKE), (3, FAKE + 2), (2, FAKE + 2)]:
        args = [FAKE, FAKE, FAKE, 2 * FAKE]
        args[i] = bad
        assert tb.tb_cuda_route_experts_backward_device(_rt(), *args) == 0, (i, bad)


def _cb(**change):
    return tb.ExpertCombineDesc(**{**dict(tokens=4, rows=8, width=16, top_k=2, type=1), **change})


@pytest.mark.parametrize("change", [
    dict(tokens=0), dict(rows=0), dict(width=0), dict(top_k=0), dict(top_k=33), dict(type=3), dict(rows_stride=15),
    dict(out_stride=15), dict(tokens=2 ** 31), dict(rows=2 ** 31), dict(width=2 ** 60)])
def test_combine_refuses_descriptors(change):
    d = _cb(**change)
    assert tb.tb_cuda_combine_experts_device(d, FAKE, FAKE, FAKE, 2 * FAKE) == 0
    assert tb.tb_cuda_combine_experts_backward_device(d, FAKE, FAKE, FAKE, FAKE, 2 * FAKE, FAKE) == 0


def test_combine_refuses_pointers():
    for i, bad in [(0, None), (1, None), (3, None), (3, FAKE), (0, FAKE + 1), (1, FAKE + 2), (2, FAKE + 2),
                   (3, FAKE + 1)]:
        args = [FAKE, FAKE, FAKE, 2 * FAKE]
        args[i] = bad
        assert tb.tb_cuda_combine_experts_device(_cb(), *args) == 0, (i, bad)
    for i, bad in [(0, None), (1, None), (3, None), (4, None), (4, FAKE), (5, FAKE + 2), (3, FAKE + 1)]:
        args = [FAKE, FAKE, FAKE, FAKE, 2 * FAKE, FAKE]
        args[i] = bad
        assert tb.tb_cuda_combine_experts_backward_device(_cb(), *args) == 0, (i, bad)


def test_descriptors_take_their_fields_only():
    with pytest.raises(TypeError):
        tb.GroupNormDesc(sample=3)


def test_shared_memory_limits_only_grow(tmp_path):
    """Of two threads that first ask for different sizes, the smaller one does not take away what the larger one has."""
    here = os.path.dirname(os.path.abspath(__file__))
    exe = str(tmp_path / "shared_limit")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I",
                    os.path.join(os.path.dirname(here), "turbinator_c_b200", "csrc"),
                    os.path.join(here, "shared_limit.cpp"), "-o", exe], check=True, timeout=120)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout


@pytest.mark.parametrize("over", (0, 1))
def test_recurrence_limit_of_steps(over):
    """The kernels count steps in 31 bits, and the last round of warps goes up to 64 steps past the end."""
    d = _rec(sequences=1, channels=1, steps=2 ** 31 - 256 + over)
    assert (tb.tb_cuda_gated_recurrence_workspace(d) == 0) == bool(over)


def test_copied_descriptors_stand_for_themselves():
    """A copy of a descriptor that is changed afterwards is what its calls read, and it outlives the original."""
    first = _norm(samples=2, positions=4096)
    need = tb.tb_cuda_group_norm_workspace(first)
    fresh = _norm(samples=500, positions=4096)
    for many in (copy.copy(first), copy.deepcopy(first), pickle.loads(pickle.dumps(first)),
                 type(first).from_buffer_copy(bytes(first)), (type(first) * 2)(first, first)[1]):
        many.samples = 500
        assert tb.tb_cuda_group_norm_workspace(many) == tb.tb_cuda_group_norm_workspace(fresh) != need
        many.samples = 0
        assert tb.tb_cuda_group_norm_workspace(many) == 0
    assert tb.tb_cuda_group_norm_workspace(first) == need
