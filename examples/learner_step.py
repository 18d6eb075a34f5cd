"""The learner layers as a learner uses them, on the library's own input tensors.

A small actor over aircraft trajectories: ``tb_cuda_prepare_actor_inputs_device`` turns observations, missions and
cameras into proprio and luma; a camera stem (convolution, group norm + SiLU), a gated recurrence over each aircraft's
trajectory with resets at episode ends, and a trunk of routed experts predict the next step's proprio.

    python examples/learner_step.py            # trains for some steps, then acts step by step from kept states

The ``torch.autograd.Function`` wrappers below are all that a PyTorch program needs around the C entry points; matrix
products and the convolution are PyTorch's.  They make descriptors, workspaces and outputs anew in each call, which a
program that counts microseconds, as one that acts does, makes once and keeps: a step of 64 aircraft is 2 us of the
GPU's time and more than ten times that of the host's in this form."""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import turbinator_c_b200 as tb  # noqa: E402

TYPE = {torch.float32: tb.TB_TYPE_F32, torch.bfloat16: tb.TB_TYPE_BF16, torch.float16: tb.TB_TYPE_F16}


def _call(ok: int) -> None:
    if ok != 1:
        raise RuntimeError("the learner call was refused")


def _finish() -> None:
    """Waits for the stream; an error if a kernel's wait for its own copies ran out since the last time."""
    if tb.tb_cuda_synchronize(torch.cuda.current_stream()) != 1:
        raise RuntimeError("a kernel gave up waiting: the results since the last check are not valid")


def _scratch(need: int) -> torch.Tensor:
    return torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")


class GroupNormAct(torch.autograd.Function):
    """x [samples, positions, channels] -> silu(group norm)."""

    @staticmethod
    def forward(ctx, x, gamma, beta, groups):
        n, p, c = x.shape
        desc = tb.GroupNormDesc(samples=n, positions=p, channels=c, groups=groups, type=TYPE[x.dtype],
                                activation=tb.TB_ACT_SILU, epsilon=1e-5)
        work = _scratch(tb.tb_cuda_group_norm_workspace(desc))
        y, mean, rstd = torch.empty_like(x), *torch.empty((2, n, groups), device="cuda")
        _call(tb.tb_cuda_group_norm_device(desc, x, gamma, beta, y, mean, rstd, work, torch.cuda.current_stream()))
        ctx.save_for_backward(x, gamma, beta, mean, rstd)
        ctx.desc = desc
        return y

    @staticmethod
    def backward(ctx, dy):
        x, gamma, beta, mean, rstd = ctx.saved_tensors
        dy, dx = dy.contiguous(), torch.empty_like(x)
        dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(beta)
        work = _scratch(tb.tb_cuda_group_norm_workspace(ctx.desc))
        _call(tb.tb_cuda_group_norm_backward_device(ctx.desc, x, gamma, beta, mean, rstd, dy, dx, dgamma, dbeta, work,
                                                    torch.cuda.current_stream()))
        return dx, dgamma, dbeta, None


class GatedRecurrence(torch.autograd.Function):
    """xgg [sequences, steps, 3 * channels]: x and both gates, thirds of one projection -> h, last state."""

    @staticmethod
    def forward(ctx, xgg, decay, state, reset):
        b, t, d = xgg.shape[0], xgg.shape[1], xgg.shape[2] // 3
        desc = tb.GatedRecurrenceDesc(sequences=b, steps=t, channels=d, type=TYPE[xgg.dtype], decay_scale=8.0,
                                      in_sequence_stride=t * 3 * d, in_step_stride=3 * d,
                                      grad_sequence_stride=t * 3 * d, grad_step_stride=3 * d)
        work = _scratch(tb.tb_cuda_gated_recurrence_workspace(desc))
        h, last = torch.empty((b, t, d), dtype=xgg.dtype, device="cuda"), torch.empty_like(state)
        saved = torch.empty((b, -(-t // tb.RECURRENCE_CHECKPOINT), d), device="cuda")
        _call(tb.tb_cuda_gated_recurrence_device(desc, xgg, xgg[..., d:], xgg[..., 2 * d:], decay, reset, None, state,
                                                 h, last, saved, work, torch.cuda.current_stream()))
        ctx.save_for_backward(xgg, decay, reset, saved)
        ctx.desc = desc
        return h, last

    @staticmethod
    def backward(ctx, dh, dlast):
        xgg, decay, reset, saved = ctx.saved_tensors
        d = xgg.shape[2] // 3
        dh, dlast, dxgg = dh.contiguous(), dlast.contiguous(), torch.empty_like(xgg)
        ddecay, dstate = torch.empty_like(decay), torch.empty_like(dlast)
        work = _scratch(tb.tb_cuda_gated_recurrence_workspace(ctx.desc))
        _call(tb.tb_cuda_gated_recurrence_backward_device(
            ctx.desc, xgg, xgg[..., d:], xgg[..., 2 * d:], decay, reset, None, saved, dh, dlast, dxgg, dxgg[..., d:],
            dxgg[..., 2 * d:], ddecay, dstate, work, torch.cuda.current_stream()))
        return dxgg, ddecay, dstate, None


class RouteExperts(torch.autograd.Function):
    """logits [tokens, experts] -> weights, ids, offsets, order, position (the last four without a gradient)."""

    @staticmethod
    def forward(ctx, logits, bias, top_k):
        t, e = logits.shape
        desc = tb.ExpertRouteDesc(tokens=t, experts=e, top_k=top_k, groups=1, top_groups=1, group_best=1,
                                  type=TYPE[logits.dtype], score=tb.TB_SCORE_SIGMOID, renormalise=1, weight_scale=1.0)
        whole = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
        ids, offsets, order, position = whole(t, top_k), whole(e + 1), whole(t * top_k), whole(t, top_k)
        weights = torch.empty((t, top_k), device="cuda")
        work = _scratch(tb.tb_cuda_route_experts_workspace(desc))
        _call(tb.tb_cuda_route_experts_device(desc, logits, bias, ids, weights, offsets, order, position, work,
                                              torch.cuda.current_stream()))
        ctx.save_for_backward(logits, ids)
        ctx.desc = desc
        ctx.mark_non_differentiable(ids, offsets, order, position)
        return weights, ids, offsets, order, position

    @staticmethod
    def backward(ctx, dweights, *_):
        logits, ids = ctx.saved_tensors
        dlogits = torch.empty_like(logits)
        _call(tb.tb_cuda_route_experts_backward_device(ctx.desc, logits, ids, dweights.contiguous(), dlogits,
                                                       torch.cuda.current_stream()))
        return dlogits, None, None


def _combine_desc(tokens, top_k, rows, width, dtype):
    return tb.ExpertCombineDesc(tokens=tokens, top_k=top_k, rows=rows, width=width, type=TYPE[dtype])


class HandOut(torch.autograd.Function):
    """x [tokens, width] -> its rows in the experts' order; the gradient sums a token's rows."""

    @staticmethod
    def forward(ctx, x, order, position):
        ctx.save_for_backward(position)
        return x[order.long() // position.shape[1]]

    @staticmethod
    def backward(ctx, drows):
        (position,) = ctx.saved_tensors
        t, k = position.shape
        drows = drows.contiguous()
        dx = torch.empty((t, drows.shape[1]), dtype=drows.dtype, device="cuda")
        _call(tb.tb_cuda_combine_experts_device(_combine_desc(t, k, *drows.shape, drows.dtype), drows, position, None, dx,
                                                torch.cuda.current_stream()))
        return dx, None, None


class Combine(torch.autograd.Function):
    """The experts' rows back to their tokens, weighted."""

    @staticmethod
    def forward(ctx, rows, position, weights):
        t, k = position.shape
        rows = rows.contiguous()
        desc = _combine_desc(t, k, *rows.shape, rows.dtype)
        out = torch.empty((t, rows.shape[1]), dtype=rows.dtype, device="cuda")
        _call(tb.tb_cuda_combine_experts_device(desc, rows, position, weights, out, torch.cuda.current_stream()))
        ctx.save_for_backward(rows, position, weights)
        ctx.desc = desc
        return out

    @staticmethod
    def backward(ctx, dout):
        rows, position, weights = ctx.saved_tensors
        drows, dweights = torch.empty_like(rows), torch.empty_like(weights)
        _call(tb.tb_cuda_combine_experts_backward_device(ctx.desc, rows, position, weights, dout.contiguous(), drows,
                                                         dweights, torch.cuda.current_stream()))
        return drows, None, dweights


class Actor(torch.nn.Module):
    def __init__(self, width=128, experts=8, top_k=2, stem=32, dtype=torch.bfloat16, seed=0):
        super().__init__()
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        new = lambda *s, scale=1.0: torch.nn.Parameter(  # noqa: E731
            (torch.randn(s, generator=gen, device="cuda") * scale).to(dtype))
        self.width, self.experts, self.top_k, self.stem = width, experts, top_k, stem
        self.kernel = new(stem, 1, 8, 8, scale=0.125)
        self.gamma = torch.nn.Parameter(torch.ones(stem, device="cuda"))
        self.beta = torch.nn.Parameter(torch.zeros(stem, device="cuda"))
        self.gates = new(91 + 4 * stem, 3 * width, scale=0.06)
        self.decay = torch.nn.Parameter(torch.linspace(-5.0, -3.0, width, device="cuda"))
        self.router = new(width, experts, scale=0.1)
        self.register_buffer("balance", torch.zeros(experts, device="cuda"))
        self.up, self.down = new(experts, width, 2 * width, scale=0.09), new(experts, 2 * width, width, scale=0.06)
        self.head = new(width, 91, scale=0.05)

    def forward(self, proprio, luma, state, reset):
        """proprio [aircraft, steps, 91], luma [.., 4, 64, 64] -> prediction, last state, experts' loads."""
        b, t = proprio.shape[:2]
        dtype = self.gates.dtype
        views = luma.reshape(b * t * 4, 1, 64, 64).to(dtype)
        maps = torch.nn.functional.conv2d(views, self.kernel, stride=4, padding=2)  # [.., stem, 16, 16]
        maps = maps.permute(0, 2, 3, 1).reshape(b * t * 4, 256, self.stem).contiguous()
        seen = GroupNormAct.apply(maps, self.gamma, self.beta, 8).mean(1).reshape(b, t, 4 * self.stem)
        xgg = torch.cat([proprio.to(dtype), seen], 2) @ self.gates
        h, state = GatedRecurrence.apply(xgg, self.decay, state, reset)
        tokens = h.reshape(b * t, self.width)
        weights, _, offsets, order, position = RouteExperts.apply(tokens @ self.router, self.balance, self.top_k)
        rows = HandOut.apply(tokens, order, position)
        ends = offsets.tolist()  # each expert's rows: a program on the hot path keeps them on the GPU
        done = [torch.nn.functional.silu(rows[a:z] @ self.up[e]) @ self.down[e]
                for e, (a, z) in enumerate(zip(ends, ends[1:]))]
        out = tokens + Combine.apply(torch.cat(done), position, weights)
        return (out @ self.head).reshape(b, t, 91), state, offsets.diff()


def trajectories(aircraft: int, steps: int, seed: int = 0):
    """Learner inputs of synthetic observations, a slow mixture of four of them for each aircraft so that there is
    something to predict; and the flags of episodes' first steps."""
    n = 4 * aircraft
    obs, mission, cams, _ = tb.generate(seed, 0, n)
    dev = [torch.from_numpy(v).cuda() for v in (obs, mission, cams)]
    widths = (91, 49, 24, 15, 6 * 2048, 16384)
    proprio, missions, tactical, prior, lidar, luma = (torch.empty((n, w), device="cuda") for w in widths)
    _call(tb.tb_cuda_prepare_actor_inputs_device(*dev, proprio, missions, tactical, prior, lidar, luma, n,
                                                 torch.cuda.current_stream()))
    phase = torch.arange(steps, device="cuda")[None, :, None] * 0.2 + torch.arange(4, device="cuda") * 1.57
    mix = (phase + torch.arange(aircraft, device="cuda")[:, None, None]).cos() * 0.5
    proprio = torch.einsum("bts,bsp->btp", mix, proprio.reshape(aircraft, 4, -1))
    luma = torch.einsum("bts,bsp->btp", mix, luma.reshape(aircraft, 4, -1)).reshape(aircraft, steps, 4, 64, 64)
    reset = (torch.arange(steps, device="cuda") % 13 == 0).to(torch.uint8).repeat(aircraft, 1)
    return proprio, luma, reset


def train(actor: Actor, aircraft=16, steps=33, updates=40, rate=2e-3, seed=0):
    """Predicts each step's successor; returns the losses."""
    proprio, luma, reset = trajectories(aircraft, steps + 1, seed)
    first = torch.zeros((aircraft, actor.width), device="cuda")
    optimiser = torch.optim.Adam(actor.parameters(), lr=rate)
    losses = []
    for _ in range(updates):
        guess, _, loads = actor(proprio[:, :-1], luma[:, :-1], first, reset[:, :-1].contiguous())
        loss = (guess.float() - proprio[:, 1:]).square().mean()
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        actor.balance += 0.001 * torch.sign(loads.float().mean() - loads)  # the busy experts' scores go down
        _finish()
        losses.append(loss.item())
    return losses


@torch.no_grad()
def act(actor: Actor, proprio, luma, reset):
    """The same forward pass one step at a time, each aircraft's state kept between the calls."""
    state = torch.zeros((proprio.shape[0], actor.width), device="cuda")
    out = []
    for t in range(proprio.shape[1]):
        guess, state, _ = actor(proprio[:, t:t + 1], luma[:, t:t + 1], state, reset[:, t:t + 1].contiguous())
        out.append(guess)
    _finish()
    return torch.cat(out, 1)


def main() -> None:
    actor = Actor()
    losses = train(actor)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} over {len(losses)} updates")
    proprio, luma, reset = trajectories(4, 20, seed=1)
    with torch.no_grad():
        whole = actor(proprio, luma, torch.zeros((4, actor.width), device="cuda"), reset)[0]
    stepped = act(actor, proprio, luma, reset)
    off = (whole - stepped).float().square().mean(2).sqrt()  # per step
    print(f"acting step by step differs from the whole trajectory by {float(off.median()):.2g} (median of the steps; "
          f"{float(off.max()):.2g} at most, where bf16 rounding decides between two experts) "
          f"of {float(whole.float().square().mean().sqrt()):.2g}")


if __name__ == "__main__":
    main()
