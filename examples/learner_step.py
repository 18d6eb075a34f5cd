"""The learner layers as a learner uses them, on the library's own input tensors.

A small actor over aircraft trajectories: ``tb_cuda_prepare_actor_inputs_device`` turns observations, missions and
cameras into proprio and luma; a camera stem (convolution, group norm + SiLU), a gated recurrence over each aircraft's
trajectory with resets at episode ends, and a trunk of routed experts predict the next step's proprio.  The experts'
matrices are updated by orthogonalised momentum, everything else by Adam; for acting they may be held in 8 bits.

    python examples/learner_step.py            # trains for some steps, then acts step by step from kept states

The ``torch.autograd.Function`` wrappers below, each differentiable once, are all that a PyTorch program needs around
the C entry points; the convolution and the products of dense layers are PyTorch's.  They make descriptors, workspaces
and outputs anew in each call, which a program that counts microseconds, as one that acts does, makes once and keeps: a
step of 64 aircraft is 2 us of the GPU's time and more than ten times that of the host's in this form."""
from __future__ import annotations

import os
import sys

import torch
from torch.autograd.function import once_differentiable

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
    @once_differentiable
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
    @once_differentiable
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
    @once_differentiable
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
        desc = _combine_desc(*position.shape, order.shape[0], x.shape[1], x.dtype)
        rows = torch.empty((order.shape[0], x.shape[1]), dtype=x.dtype, device="cuda")
        _call(tb.tb_cuda_hand_out_experts_device(desc, x.contiguous(), order, None, rows, torch.cuda.current_stream()))
        ctx.save_for_backward(position)
        ctx.desc = desc
        return rows

    @staticmethod
    @once_differentiable
    def backward(ctx, drows):
        (position,) = ctx.saved_tensors
        drows = drows.contiguous()
        dx = torch.empty((position.shape[0], drows.shape[1]), dtype=drows.dtype, device="cuda")
        _call(tb.tb_cuda_hand_out_experts_backward_device(ctx.desc, None, position, None, drows, dx, None,
                                                          torch.cuda.current_stream()))
        return dx, None, None


def _fit_together(rows, weight, offsets, n):
    """The C entry points see addresses only: what a tensor says of itself is checked here."""
    if rows.ndim != 2 or weight.ndim != 3 or rows.shape[1] != n:
        raise ValueError(f"rows {tuple(rows.shape)} and weights {tuple(weight.shape)} do not go together")
    if offsets.dtype != torch.int32 or offsets.shape != (weight.shape[0] + 1,) or not offsets.is_contiguous():
        raise ValueError("offsets are one more 32-bit whole number than there are experts")
    if not rows.device == weight.device == offsets.device:
        raise ValueError("rows, weights and offsets lie on different devices")


class Product(torch.autograd.Function):
    """rows [rows, in] of the experts' runs, weights [experts, in, out] of the same type -> [rows, out]; offsets stay on
    the GPU.  Weights that lie [experts, out, in] (a transposed view) are multiplied as they lie, others copied."""

    @staticmethod
    def forward(ctx, rows, weight, offsets):
        e, n, m = weight.shape
        _fit_together(rows, weight, offsets, n)
        if rows.dtype != weight.dtype:
            raise TypeError(f"rows of {rows.dtype} and weights of {weight.dtype}")
        rows = rows.contiguous()
        turned = not weight.is_contiguous() and weight.transpose(1, 2).is_contiguous()
        weight = weight if turned else weight.contiguous()
        desc = tb.ExpertProductDesc(rows=rows.shape[0], experts=e, in_width=n, out_width=m, type=TYPE[rows.dtype],
                                    weight_order=tb.TB_WEIGHT_OUT_IN if turned else tb.TB_WEIGHT_IN_OUT)
        out = torch.empty((rows.shape[0], m), dtype=rows.dtype, device="cuda")
        work = _scratch(tb.tb_cuda_experts_product_workspace(desc))
        _call(tb.tb_cuda_experts_product_device(desc, rows, weight, offsets, out, work, torch.cuda.current_stream()))
        ctx.save_for_backward(rows, weight, offsets)
        ctx.desc = desc
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        rows, weight, offsets = ctx.saved_tensors
        drows, dweight = torch.empty_like(rows), torch.empty_like(weight)  # which keeps the weights' order
        work = _scratch(tb.tb_cuda_experts_product_workspace(ctx.desc))
        _call(tb.tb_cuda_experts_product_backward_device(ctx.desc, rows, weight, offsets, dout.contiguous(), drows, dweight, work,
                                                         torch.cuda.current_stream()))
        return drows, dweight, None


def quantised(x):
    """Rows of x [.., width] in 8 bits, and their scales."""
    x = x.contiguous()
    q, scale = torch.empty(x.shape, dtype=torch.int8, device="cuda"), torch.empty(x.shape[:-1], device="cuda")
    desc = tb.QuantiseDesc(rows=scale.numel(), width=x.shape[-1], type=TYPE[x.dtype])
    _call(tb.tb_cuda_quantise_rows_device(desc, x, q, scale, torch.cuda.current_stream()))
    return q, scale


def product_8_bit(rows, weight, weight_scale, offsets):
    """rows [rows, in] of the experts' runs by weights [experts, out, in] of 8 bits."""
    e, m, n = weight.shape
    _fit_together(rows, weight, offsets, n)
    if weight.dtype != torch.int8 or weight_scale.dtype != torch.float32 or weight_scale.shape != (e, m):
        raise TypeError("weights of 8 bits with an f32 scale for each output channel")
    weight, weight_scale = weight.contiguous(), weight_scale.contiguous()
    q, scale = quantised(rows)
    desc = tb.ExpertProductI8Desc(rows=rows.shape[0], experts=e, in_width=n, out_width=m, type=TYPE[rows.dtype])
    out = torch.empty((rows.shape[0], m), dtype=rows.dtype, device="cuda")
    work = _scratch(tb.tb_cuda_experts_product_i8_workspace(desc))
    _call(tb.tb_cuda_experts_product_i8_device(desc, q, scale, weight, weight_scale, offsets, out, work,
                                               torch.cuda.current_stream()))
    return out


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
    @once_differentiable
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
        self.held = None  # the experts in 8 bits, for acting

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
        silu = torch.nn.functional.silu
        if self.held:
            done = product_8_bit(silu(product_8_bit(rows, *self.held[0], offsets)), *self.held[1], offsets)
        else:
            done = Product.apply(silu(Product.apply(rows, self.up, offsets)), self.down, offsets)
        out = tokens + Combine.apply(done, position, weights)
        return (out @ self.head).reshape(b, t, 91), state, offsets.diff()


    @torch.no_grad()
    def hold_experts_in_8_bits(self):
        """For acting: a scale for each output channel, whose weights become a row."""
        self.held = [quantised(w.transpose(1, 2)) for w in (self.up, self.down)]


class OrthogonalMomentum:
    """Momentum of stacks of matrices, orthogonalised before it is applied: every direction moves alike."""

    def __init__(self, parameters, rate=0.02, momentum=0.95):
        self.parameters, self.rate, self.momentum = list(parameters), rate, momentum
        self.kept = [torch.zeros_like(p) for p in self.parameters]

    @torch.no_grad()
    def step(self):
        for p, kept in zip(self.parameters, self.kept):
            kept.mul_(self.momentum).add_(p.grad)
            b, m, n = p.shape
            desc = tb.OrthogonaliseDesc(matrices=b, rows=m, columns=n, type=TYPE[p.dtype], steps=5, a=3.4445, b=-4.7750,
                                        c=2.0315, epsilon=1e-7, scale=max(1.0, n / m) ** 0.5)
            g = p.grad.add(kept, alpha=self.momentum).contiguous()  # however the parameter lies
            update, work = torch.empty_like(g), _scratch(tb.tb_cuda_orthogonalise_workspace(desc))
            _call(tb.tb_cuda_orthogonalise_device(desc, g, update, work, torch.cuda.current_stream()))
            p.add_(update, alpha=-self.rate)


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


def train(actor: Actor, aircraft=16, steps=33, updates=40, rate=2e-3, seed=0, orthogonal=False):
    """Predicts each step's successor; returns the losses.  orthogonal: the experts' matrices by orthogonalised momentum."""
    proprio, luma, reset = trajectories(aircraft, steps + 1, seed)
    first = torch.zeros((aircraft, actor.width), device="cuda")
    experts = [actor.up, actor.down] if orthogonal else []
    optimiser = torch.optim.Adam([p for p in actor.parameters() if not any(p is e for e in experts)], lr=rate)
    of_experts = OrthogonalMomentum(experts, rate=5 * rate)
    losses = []
    for _ in range(updates):
        guess, _, loads = actor(proprio[:, :-1], luma[:, :-1], first, reset[:, :-1].contiguous())
        loss = (guess.float() - proprio[:, 1:]).square().mean()
        actor.zero_grad()
        loss.backward()
        optimiser.step()
        of_experts.step()
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
    losses = train(actor, orthogonal=True)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} over {len(losses)} updates")
    proprio, luma, reset = trajectories(4, 20, seed=1)
    with torch.no_grad():
        whole = actor(proprio, luma, torch.zeros((4, actor.width), device="cuda"), reset)[0]
    stepped = act(actor, proprio, luma, reset)
    off = (whole - stepped).float().square().mean(2).sqrt()  # per step
    print(f"acting step by step differs from the whole trajectory by {float(off.median()):.2g} (median of the steps; "
          f"{float(off.max()):.2g} at most, where bf16 rounding decides between two experts) "
          f"of {float(whole.float().square().mean().sqrt()):.2g}")
    actor.hold_experts_in_8_bits()
    off = (act(actor, proprio, luma, reset) - stepped).float().square().mean(2).sqrt()
    print(f"with the experts in 8 bits by {float(off.median()):.2g} (median of the steps)")


if __name__ == "__main__":
    main()
