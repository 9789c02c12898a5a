"""Several experts per token: routing to the k best, rows to their experts and back (torch tensors over the C ABI).

    router = TopKRouter(expert_count, top_k, score="sigmoid", bias=bias, groups=8, top_groups=4)
    gate, weight = router.select(logits)                              # the gate's projection of the tokens, [T, E]
    pos, count, offset = count_experts(gate, expert_count)
    routed, row_of = scatter_topk(x, pos, offset, top_k)              # rows in expert order, for experts of your own
    out = combine_topk(results, weight, row_of=row_of)

`MoELayer.forward_topk(x, gate, weight)` runs a layer's own experts in the place of the last three lines.  The reference routes
every token to one expert (top-k is a TODO there).

All functions work on torch's current stream of the tensors' device, and allocate what they return unless they are given it.
They are for inference: what they return carries no gradient.
"""
from __future__ import annotations

import ctypes

from . import capi

__all__ = ["TopKRouter", "count_experts", "scatter_topk", "combine_topk"]


def binding():
    """The extension module that checks tensors, makes outputs and calls the library (csrc/binding.cc)."""
    global _binding
    if _binding is None:
        import torch  # noqa: F401  its libraries come before the module's

        from . import _binding as module

        _binding = module
    return _binding


_binding = None


def launch(device: int, name: str, *args) -> None:
    """Calls a C entry point whose last argument is the stream, on `device` and torch's current stream there."""
    import torch

    from .plugin import _current_stream

    fn = getattr(capi.lib(), name)
    if torch.cuda.current_device() == device:
        capi.check(fn(*args, _current_stream(torch, device)))
    else:
        with torch.cuda.device(device):
            capi.check(fn(*args, _current_stream(torch, device)))


def check_array(t, shape, dtype, device, what: str) -> None:
    """A contiguous tensor of this shape and type on this device."""
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {str(dtype)[6:]} tensor of shape {list(shape)} on {device}")


class TopKRouter:
    """The choice of a token's k experts from its gating logits (infmoe_expert_select_topk).

    score        "softmax" or "sigmoid" of the logits
    bias         float32 CUDA tensor [expert_count] added to the scores for the choice alone (load balance), or None;
                 read at every call, so it may be updated in place
    groups, top_groups, group_best
                 with groups > 1, only the experts of the top_groups best groups are chosen from; a group counts with the sum
                 of its two best experts (group_best=2) or with its best one (1)
    renormalise  the weights of a token's experts sum to `scale`
    """

    def __init__(self, expert_count: int, top_k: int, score: str = "softmax", bias=None, groups: int = 1, top_groups: int = 1,
                 group_best: int = 1, renormalise: bool = True, scale: float = 1.0) -> None:
        import torch

        if score not in capi.SCORES:
            raise ValueError(f"score must be one of {sorted(capi.SCORES)}")
        if bias is not None and not (bias.is_cuda and bias.dtype == torch.float32 and tuple(bias.shape) == (expert_count,) and
                                     bias.is_contiguous()):
            raise ValueError(f"bias must be a contiguous float32 CUDA tensor of shape [{expert_count}]")
        self.expert_count, self.top_k, self.bias = int(expert_count), int(top_k), bias
        self._cfg = capi.TopKConfig(expert_count, top_k, capi.SCORES[score], groups, top_groups, group_best, int(renormalise),
                                    scale)
        self._select = binding().select_topk
        # what a configuration can be refused for, now and not at the first call: no tokens, no device work
        capi.check(capi.lib().infmoe_expert_select_topk(ctypes.byref(self._cfg), 0, None, capi.DTYPE_F32, expert_count, None, None, None,
                                                        None, None))

    def select(self, logits, gate=None, weight=None, status=None):
        """logits: float32, float16 or bfloat16 CUDA tensor [..., expert_count] -> (gate int32, weight float32), [..., top_k].

        Experts with a logit of NaN or of the type's lowest value or less (-inf) are not chosen; places that stay empty hold
        gate -1 and weight 0.  More than 16 experts to a token cost several times what 16 do.

        status (int32 [1], may be None): bit 0 is set when a token has no expert at all."""
        return self._select(self._cfg, logits, self.bias, gate, weight, status)


def count_experts(gate, expert_count: int, status=None):
    """gate: int32 CUDA tensor of expert indices, one per slot -> (pos, count, offset) of the slots in expert order
    (infmoe_expert_count).  Slots with an index outside [0, expert_count) come last, offset[expert_count] is where they begin;
    status (int32 [1], may be None): bit 1 is set when there are any."""
    import torch

    if not gate.is_cuda or gate.dtype != torch.int32 or not gate.is_contiguous():
        raise ValueError("gate must be a contiguous int32 CUDA tensor")
    pos = torch.empty(gate.numel(), dtype=torch.int32, device=gate.device)
    count = torch.empty(expert_count, dtype=torch.int32, device=gate.device)
    offset = torch.empty(expert_count + 1, dtype=torch.int32, device=gate.device)
    if status is not None:
        check_array(status, (1,), torch.int32, gate.device, "status")
    launch(gate.get_device(), "infmoe_expert_count", gate.numel(), expert_count, gate.data_ptr(), pos.data_ptr(),
           count.data_ptr(), offset.data_ptr(), status.data_ptr() if status is not None else None)
    return pos, count, offset


def scatter_topk(x, pos, offset, top_k: int, out=None, row_of=None):
    """x [..., D] -> (rows in expert order [T * top_k, D], row of every slot [T, top_k], -1 for slots without an expert).

    pos and offset are count_experts' of the slots; rows behind the last expert's are left as they are in `out`."""
    return binding().scatter_topk(x, pos, offset, top_k, out, row_of)


def combine_topk(rows, weight, row_of=None, gate=None, residual=None, out=None):
    """out[t] = sum_s weight[t, s] * rows[row_of[t, s]] (+ (1 - sum_s weight[t, s]) * residual[t]).

    rows [n, D]; weight float32 [..., top_k]; row_of int32 like weight (None: slot (t, s) is row t * top_k + s); gate int32
    like weight or None: slots with a negative gate are left out, like slots whose row lies outside [0, n).  residual, out:
    [..., D] like weight's leading dimensions; out may be residual."""
    return binding().combine_topk(rows, weight, row_of, gate, residual, out)
