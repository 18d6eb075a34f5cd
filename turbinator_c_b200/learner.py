"""Learner layers -- Python view of ``include/turbinator/training/cuda_learner.h``.

Group norm with an activation, the gated linear recurrence, routing to experts,
handing tokens out to them, the experts' products and their combine, each
forward and backward, the products in 8-bit integers and the orthogonalised
update, under the names of the C functions.  A descriptor is made once and kept; the calls take device tensors
(or pointers), run on ``stream`` and return 1, or 0 on a rejected argument or a
launch error, like the other device entry points.  The caller owns outputs and
workspaces; nothing is allocated here.
"""
from __future__ import annotations

import ctypes as _c

from . import _ptr, _stream_handle, load_library

_address = _c.addressof

TB_TYPE_F32, TB_TYPE_BF16, TB_TYPE_F16 = range(3)
TB_ACT_NONE, TB_ACT_RELU, TB_ACT_SILU, TB_ACT_GELU = range(4)
TB_SCORE_SOFTMAX, TB_SCORE_SIGMOID = range(2)
TB_WEIGHT_IN_OUT, TB_WEIGHT_OUT_IN = range(2)

#: Steps between two saved states of the recurrence (TB_RECURRENCE_CHECKPOINT).
RECURRENCE_CHECKPOINT = 16


class _Desc(_c.Structure):
    """A descriptor of the C ABI: fields by keyword, the rest zero (strides: dense)."""

    def __init__(self, **fields):
        unknown = set(fields) - {name for name, _ in self._fields_}
        if unknown:
            raise TypeError(f"{type(self).__name__} has no field {sorted(unknown)}")
        super().__init__(**fields)

    @property
    def address(self) -> int:
        """Where this descriptor lies: asked for at each call, since a copy lies elsewhere."""
        return _address(self)


class GroupNormDesc(_Desc):
    """Mirror of ``tb_group_norm_desc``."""

    _fields_ = [(n, _c.c_size_t) for n in
                ("samples", "positions", "channels", "groups", "x_sample_stride", "x_position_stride",
                 "y_sample_stride", "y_position_stride", "dx_sample_stride", "dx_position_stride")] + [
        ("type", _c.c_int), ("activation", _c.c_int), ("epsilon", _c.c_float)]


class GatedRecurrenceDesc(_Desc):
    """Mirror of ``tb_gated_recurrence_desc``."""

    _fields_ = [(n, _c.c_size_t) for n in
                ("sequences", "steps", "channels", "in_sequence_stride", "in_step_stride", "out_sequence_stride",
                 "out_step_stride", "grad_sequence_stride", "grad_step_stride")] + [
        ("type", _c.c_int), ("decay_scale", _c.c_float)]


class ExpertRouteDesc(_Desc):
    """Mirror of ``tb_expert_route_desc``."""

    _fields_ = [(n, _c.c_size_t) for n in ("tokens", "experts", "logits_stride")] + [
        (n, _c.c_int) for n in ("top_k", "groups", "top_groups", "group_best", "type", "score", "renormalise")] + [
        ("weight_scale", _c.c_float)]


class ExpertCombineDesc(_Desc):
    """Mirror of ``tb_expert_combine_desc``."""

    _fields_ = [(n, _c.c_size_t) for n in ("tokens", "rows", "width", "rows_stride", "out_stride")] + [
        ("top_k", _c.c_int), ("type", _c.c_int)]


class ExpertProductDesc(_Desc):
    """Mirror of ``tb_expert_product_desc``."""

    _fields_ = [(n, _c.c_size_t) for n in
                ("rows", "experts", "in_width", "out_width", "in_stride", "din_stride", "out_stride",
                 "weight_expert_stride", "weight_row_stride")] + [("weight_order", _c.c_int), ("type", _c.c_int)]


class QuantiseDesc(_Desc):
    """Mirror of ``tb_quantise_desc``."""

    _fields_ = [(n, _c.c_size_t) for n in ("rows", "width", "x_stride", "q_stride")] + [("type", _c.c_int)]


class ExpertProductI8Desc(_Desc):
    """Mirror of ``tb_expert_product_i8_desc``."""

    _fields_ = [(n, _c.c_size_t) for n in
                ("rows", "experts", "in_width", "out_width", "in_stride", "out_stride", "weight_expert_stride",
                 "weight_row_stride")] + [("type", _c.c_int)]


class OrthogonaliseDesc(_Desc):
    """Mirror of ``tb_orthogonalise_desc``."""

    _fields_ = [(n, _c.c_size_t) for n in
                ("matrices", "rows", "columns", "in_matrix_stride", "in_row_stride", "out_matrix_stride",
                 "out_row_stride")] + [("type", _c.c_int), ("steps", _c.c_int)] + [
        (n, _c.c_float) for n in ("a", "b", "c", "epsilon", "scale")]


def tb_cuda_group_norm_workspace(desc: GroupNormDesc) -> int:
    return load_library().tb_cuda_group_norm_workspace(_address(desc))


def tb_cuda_group_norm_device(desc: GroupNormDesc, x, gamma, beta, y, mean, rstd, workspace, stream=None) -> int:
    return load_library().tb_cuda_group_norm_device(
        _address(desc), _ptr(x), _ptr(gamma), _ptr(beta), _ptr(y), _ptr(mean), _ptr(rstd), _ptr(workspace),
        _stream_handle(stream))


def tb_cuda_group_norm_backward_device(desc: GroupNormDesc, x, gamma, beta, mean, rstd, dy, dx, dgamma, dbeta,
                                       workspace, stream=None) -> int:
    return load_library().tb_cuda_group_norm_backward_device(
        _address(desc), _ptr(x), _ptr(gamma), _ptr(beta), _ptr(mean), _ptr(rstd), _ptr(dy), _ptr(dx), _ptr(dgamma),
        _ptr(dbeta), _ptr(workspace), _stream_handle(stream))


def tb_cuda_gated_recurrence_workspace(desc: GatedRecurrenceDesc) -> int:
    return load_library().tb_cuda_gated_recurrence_workspace(_address(desc))


def tb_cuda_gated_recurrence_device(desc: GatedRecurrenceDesc, x, recurrence_gate, input_gate, decay, reset, lengths,
                                    state_in, h, state_out, checkpoints, workspace, stream=None) -> int:
    return load_library().tb_cuda_gated_recurrence_device(
        _address(desc), _ptr(x), _ptr(recurrence_gate), _ptr(input_gate), _ptr(decay), _ptr(reset), _ptr(lengths),
        _ptr(state_in), _ptr(h), _ptr(state_out), _ptr(checkpoints), _ptr(workspace), _stream_handle(stream))


def tb_cuda_gated_recurrence_backward_device(desc: GatedRecurrenceDesc, x, recurrence_gate, input_gate, decay, reset,
                                             lengths, checkpoints, dh, dstate_out, dx, drecurrence_gate,
                                             dinput_gate, ddecay, dstate_in, workspace, stream=None) -> int:
    return load_library().tb_cuda_gated_recurrence_backward_device(
        _address(desc), _ptr(x), _ptr(recurrence_gate), _ptr(input_gate), _ptr(decay), _ptr(reset), _ptr(lengths),
        _ptr(checkpoints), _ptr(dh), _ptr(dstate_out), _ptr(dx), _ptr(drecurrence_gate), _ptr(dinput_gate),
        _ptr(ddecay), _ptr(dstate_in), _ptr(workspace), _stream_handle(stream))


def tb_cuda_route_experts_workspace(desc: ExpertRouteDesc) -> int:
    return load_library().tb_cuda_route_experts_workspace(_address(desc))


def tb_cuda_route_experts_device(desc: ExpertRouteDesc, logits, bias, ids, weights, offsets, order, position,
                                 workspace, stream=None) -> int:
    return load_library().tb_cuda_route_experts_device(
        _address(desc), _ptr(logits), _ptr(bias), _ptr(ids), _ptr(weights), _ptr(offsets), _ptr(order), _ptr(position),
        _ptr(workspace), _stream_handle(stream))


def tb_cuda_route_experts_backward_device(desc: ExpertRouteDesc, logits, ids, dweights, dlogits, stream=None) -> int:
    return load_library().tb_cuda_route_experts_backward_device(
        _address(desc), _ptr(logits), _ptr(ids), _ptr(dweights), _ptr(dlogits), _stream_handle(stream))


def tb_cuda_combine_experts_device(desc: ExpertCombineDesc, rows, position, weights, out, stream=None) -> int:
    return load_library().tb_cuda_combine_experts_device(
        _address(desc), _ptr(rows), _ptr(position), _ptr(weights), _ptr(out), _stream_handle(stream))


def tb_cuda_combine_experts_backward_device(desc: ExpertCombineDesc, rows, position, weights, dout, drows, dweights,
                                            stream=None) -> int:
    return load_library().tb_cuda_combine_experts_backward_device(
        _address(desc), _ptr(rows), _ptr(position), _ptr(weights), _ptr(dout), _ptr(drows), _ptr(dweights),
        _stream_handle(stream))


def tb_cuda_hand_out_experts_device(desc: ExpertCombineDesc, x, order, weights, rows, stream=None) -> int:
    return load_library().tb_cuda_hand_out_experts_device(
        _address(desc), _ptr(x), _ptr(order), _ptr(weights), _ptr(rows), _stream_handle(stream))


def tb_cuda_hand_out_experts_backward_device(desc: ExpertCombineDesc, x, position, weights, drows, dx, dweights,
                                             stream=None) -> int:
    return load_library().tb_cuda_hand_out_experts_backward_device(
        _address(desc), _ptr(x), _ptr(position), _ptr(weights), _ptr(drows), _ptr(dx), _ptr(dweights),
        _stream_handle(stream))


def tb_cuda_experts_product_workspace(desc: ExpertProductDesc) -> int:
    return load_library().tb_cuda_experts_product_workspace(_address(desc))


def tb_cuda_experts_product_device(desc: ExpertProductDesc, x, weight, offsets, y, workspace, stream=None) -> int:
    return load_library().tb_cuda_experts_product_device(
        _address(desc), _ptr(x), _ptr(weight), _ptr(offsets), _ptr(y), _ptr(workspace), _stream_handle(stream))


def tb_cuda_experts_product_backward_device(desc: ExpertProductDesc, x, weight, offsets, dy, dx, dweight, workspace,
                                            stream=None) -> int:
    return load_library().tb_cuda_experts_product_backward_device(
        _address(desc), _ptr(x), _ptr(weight), _ptr(offsets), _ptr(dy), _ptr(dx), _ptr(dweight), _ptr(workspace),
        _stream_handle(stream))


def tb_cuda_quantise_rows_device(desc: QuantiseDesc, x, q, scale, stream=None) -> int:
    return load_library().tb_cuda_quantise_rows_device(
        _address(desc), _ptr(x), _ptr(q), _ptr(scale), _stream_handle(stream))


def tb_cuda_experts_product_i8_workspace(desc: ExpertProductI8Desc) -> int:
    return load_library().tb_cuda_experts_product_i8_workspace(_address(desc))


def tb_cuda_experts_product_i8_device(desc: ExpertProductI8Desc, q, q_scale, weight, weight_scale, offsets, y, workspace,
                                      stream=None) -> int:
    return load_library().tb_cuda_experts_product_i8_device(
        _address(desc), _ptr(q), _ptr(q_scale), _ptr(weight), _ptr(weight_scale), _ptr(offsets), _ptr(y),
        _ptr(workspace), _stream_handle(stream))


def tb_cuda_orthogonalise_workspace(desc: OrthogonaliseDesc) -> int:
    return load_library().tb_cuda_orthogonalise_workspace(_address(desc))


def tb_cuda_orthogonalise_device(desc: OrthogonaliseDesc, g, out, workspace, stream=None) -> int:
    return load_library().tb_cuda_orthogonalise_device(
        _address(desc), _ptr(g), _ptr(out), _ptr(workspace), _stream_handle(stream))
