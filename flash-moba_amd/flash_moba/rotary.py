"""Rotary positions with several axes for the q and k of every attention here (no counterpart in the reference, whose callers
turn q and k themselves): flash_moba_rotary_func, forward and backward by the kernel of csrc/rotary.hip."""
from typing import List, Tuple

import torch

from flash_moba import flash_moba_hip as flash_moba_gpu


@torch.library.custom_op("flash_moba::_rotary", mutates_args=(), device_types="cuda")
def _rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, sections: List[int], base: float, rotary_dim: int,
            interleaved: bool, inverse: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    return flash_moba_gpu.host_module().rotary_raw(q, k, positions, sections, base, rotary_dim, interleaved, inverse)


@torch.library.register_fake("flash_moba::_rotary")
def _rotary_fake(q, k, positions, sections, base, rotary_dim, interleaved, inverse):
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _rotary_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[2])
    ctx.form = inputs[3:]


def _rotary_backward(ctx, dq, dk):
    sections, base, rotary_dim, interleaved, inverse = ctx.form
    dq, dk = torch.ops.flash_moba._rotary(dq, dk, ctx.saved_tensors[0], sections, base, rotary_dim, interleaved, not inverse)
    return dq, dk, None, None, None, None, None, None


torch.library.register_autograd("flash_moba::_rotary", _rotary_backward, setup_context=_rotary_setup)


def rotary_form(q, positions, sections, rotary_dim):
    """The defaults: one axis, all features, all pairs on the only axis."""
    if positions.dim() == 1:
        positions = positions[None]
    if rotary_dim is None:
        rotary_dim = q.shape[-1]
    if sections is None:
        if positions.shape[0] != 1:
            raise RuntimeError("positions of several axes need sections")
        sections = (rotary_dim // 2,)
    return positions, sections, rotary_dim


def flash_moba_rotary_func(q, k, positions, sections=None, base=10000.0, rotary_dim=None, interleaved=False):
    """Rotary positions with several axes on packed q and k, with autograd.

    q: (tokens, num_heads, head_size), k: (tokens, num_heads_k, head_size), fp16/bf16, any strides (q and k of one fused
    projection are read where they lie); positions: (tokens,) or (axes, tokens), int32 or int64, one to four axes (text: one;
    images and video: time, height, width).  The first `rotary_dim` features of a head (default: all; a multiple of 8) are
    rotary_dim / 2 pairs, pair j = features (j, j + rotary_dim / 2), or (2 j, 2 j + 1) with interleaved=True.  `sections` says how
    many consecutive pairs follow each axis (default: all follow the only axis).  Pair j is turned by
    positions[its axis] * base ** (-2 j / rotary_dim), formed in 64 bits; the features behind rotary_dim stay as they are.

    Returns (q, k), turned, as new contiguous tensors.
    """
    positions, sections, rotary_dim = rotary_form(q, positions, sections, rotary_dim)
    if not torch.compiler.is_compiling():  # plain eager calls: one native call (None: not of its form)
        turned = flash_moba_gpu.host_module().rotary(q, k, positions, sections, base, rotary_dim, interleaved)
        if turned is not None:
            return turned
    return torch.ops.flash_moba._rotary(q, k, positions, list(sections), float(base), rotary_dim, interleaved, False)
