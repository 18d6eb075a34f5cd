"""Refusals of the learner layers on a GPU, where a call that is not refused returns 1: every output at the address of
an input or of another output, but for the pairs that the header states."""
from __future__ import annotations

import itertools

import pytest

import turbinator_c_b200 as tb

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

CALLS = {
    # function, descriptor, arguments (outputs in capitals), pairs that may share an address
    "norm": (tb.tb_cuda_group_norm_device,
             tb.GroupNormDesc(samples=2, positions=64, channels=32, groups=4, type=0, activation=2, epsilon=1e-5),
             "x gamma beta Y MEAN RSTD WORK", [("x", "Y")]),
    "norm_backward": (tb.tb_cuda_group_norm_backward_device,
                      tb.GroupNormDesc(samples=2, positions=64, channels=32, groups=4, type=0, activation=2, epsilon=1e-5),
                      "x gamma beta mean rstd dy DX DGAMMA DBETA WORK", [("x", "DX"), ("dy", "DX")]),
    "recurrence": (tb.tb_cuda_gated_recurrence_device,
                   tb.GatedRecurrenceDesc(sequences=2, steps=200, channels=32, type=0, decay_scale=8.0),
                   "x rec inp decay reset lengths state H STATE SAVED WORK", [("state", "STATE")]),
    "recurrence_step": (tb.tb_cuda_gated_recurrence_device,
                        tb.GatedRecurrenceDesc(sequences=4, steps=1, channels=32, type=0, decay_scale=8.0),
                        "x rec inp decay reset lengths state H STATE SAVED WORK", [("state", "STATE")]),
    "recurrence_backward": (tb.tb_cuda_gated_recurrence_backward_device,
                            tb.GatedRecurrenceDesc(sequences=2, steps=200, channels=32, type=0, decay_scale=8.0),
                            "x rec inp decay reset lengths saved dh dstate DX DREC DINP DDECAY DSTATE WORK",
                            [("dstate", "DSTATE")]),
    "route": (tb.tb_cuda_route_experts_device,
              tb.ExpertRouteDesc(tokens=50, experts=16, top_k=2, groups=1, top_groups=1, group_best=1, type=0, score=1,
                                 renormalise=1, weight_scale=1.0),
              "logits bias IDS WEIGHTS OFFSETS ORDER POSITION WORK", []),
    "route_backward": (tb.tb_cuda_route_experts_backward_device,
                       tb.ExpertRouteDesc(tokens=50, experts=16, top_k=2, groups=1, top_groups=1, group_best=1, type=0,
                                          score=1, renormalise=1, weight_scale=1.0),
                       "logits ids dweights DLOGITS", []),
    "combine": (tb.tb_cuda_combine_experts_device, tb.ExpertCombineDesc(tokens=20, rows=40, width=32, top_k=2, type=0),
                "rows position weights OUT", []),
    "combine_backward": (tb.tb_cuda_combine_experts_backward_device,
                         tb.ExpertCombineDesc(tokens=20, rows=40, width=32, top_k=2, type=0),
                         "rows position weights dout DROWS DWEIGHTS", []),
}


@pytest.mark.parametrize("name", CALLS)
def test_outputs_on_inputs_are_refused(name):
    call, desc, names, stated = CALLS[name]
    names = names.split()
    # every buffer is as large as the largest need, and zeros are valid as flags, lengths, ids and positions alike
    buffers = {n: torch.zeros(1 << 18, device="cuda") for n in names}
    for n in ("position",):
        if n in buffers:
            buffers[n].view(torch.int32)[:40] = torch.arange(40, dtype=torch.int32, device="cuda")

    def run(**change):
        return call(desc, *[{**buffers, **change}[n] for n in names])

    assert run() == 1
    torch.cuda.synchronize()
    for n, other in itertools.permutations(names, 2):
        if not n.isupper() or (other, n) in stated:
            continue
        before = [b.clone() for b in buffers.values()]
        assert run(**{n: buffers[other]}) == 0, (n, other)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(before, buffers.values())), (n, other)
    for other, n in stated:
        assert run(**{n: buffers[other]}) == 1, (n, other)
    torch.cuda.synchronize()
