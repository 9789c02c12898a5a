"""Low-rank adapters of many requests at once, beside a projection they share (torch tensors over the C ABI).

    adapters = Adapters(a, b, scale)                 # a [n, r, d_in], b [n, d_out, r]
    plan = adapters.plan(adapter_of_token)           # once per batch: int32 [T], -1 = none
    out = adapters.apply(x, y, plan)                 # y + scale * b (a x), row by row with the row's adapter

A plan holds for every projection of the batch whose set has as many adapters.  `MoELayer.forward(x, adapters=..., plan=...)`
adds the adapters of a layer's requests to its output.  For inference: results carry no gradient.
"""
from __future__ import annotations

import ctypes

from . import capi
from .plugin import _current_stream
from .topk import binding, check_array, launch

__all__ = ["Adapters", "AdapterPlan"]


class AdapterPlan:
    """A batch's tokens grouped by adapter (infmoe_adapter_plan)."""

    def __init__(self, adapter_of_token, adapter_count: int) -> None:
        import torch

        if not adapter_of_token.is_cuda or adapter_of_token.dtype != torch.int32 or not adapter_of_token.is_contiguous():
            raise ValueError("adapter_of_token must be a contiguous int32 CUDA tensor")
        self.tokens, self.adapter_count, self.device = adapter_of_token.numel(), int(adapter_count), adapter_of_token.device
        need = ctypes.c_size_t()
        capi.check(capi.lib().infmoe_adapter_plan_bytes(self.tokens, self.adapter_count, ctypes.byref(need)))
        self.buffer = torch.empty(need.value, dtype=torch.uint8, device=self.device)
        self._home = _current_stream(torch, adapter_of_token.get_device())      # that the buffer was allocated on
        launch(adapter_of_token.get_device(), "infmoe_adapter_plan", self.tokens, self.adapter_count,
               adapter_of_token.data_ptr(), self.buffer.data_ptr(), need.value)


class Adapters:
    """A set of low-rank adapters of one projection (infmoe_adapter_set).

    a [n, r, d_in] and b [n, d_out, r]: contiguous CUDA tensors, float32, float16 or bfloat16 (the type of x and y too); they
    are used in place, not copied, and may be updated, or their data replaced by others of the same shape, between calls.  scale: a number, or a float32 tensor [n].  rank: int32 tensor [n], of which adapter i uses
    only the first rank[i] rows of a[i] and columns of b[i]; None: all r."""

    def __init__(self, a, b, scale=1.0, rank=None) -> None:
        import torch

        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or a.dtype != b.dtype or \
                a.device != b.device or not a.is_cuda or not a.is_contiguous() or not b.is_contiguous():
            raise ValueError("a [n, r, d_in] and b [n, d_out, r] must be contiguous CUDA tensors of one type and device")
        n, r, d_in = a.shape
        self.dtype, self.device = a.dtype, a.device
        self.adapter_count, self.rank, self.d_in, self.d_out = n, r, d_in, b.shape[1]
        self._home = None                            # the stream that a scale made here was allocated on
        if isinstance(scale, (int, float)):
            if scale == 1:
                scale = None
            else:
                # copied from the host, so that it is there for calls on any stream (a capture cannot wait for that)
                at = a.device if torch.cuda.is_current_stream_capturing() else "cpu"
                scale = torch.full((n,), float(scale), dtype=torch.float32, device=at).to(a.device)
                self._home = _current_stream(torch, a.get_device())
        if scale is not None:
            check_array(scale, (n,), torch.float32, a.device, "scale")
        if rank is not None:
            check_array(rank, (n,), torch.int32, a.device, "rank")
        self._tensors = (a, b, scale, rank)
        codes = {torch.float32: capi.DTYPE_F32, torch.float16: capi.DTYPE_F16, torch.bfloat16: capi.DTYPE_BF16}
        if a.dtype not in codes:
            raise ValueError(f"adapters of {a.dtype} are not supported: use float32, float16 or bfloat16")
        held = capi.AdapterSet(n, r, d_in, self.d_out, codes[a.dtype], a.data_ptr(), b.data_ptr(),
                               scale.data_ptr() if scale is not None else None, rank.data_ptr() if rank is not None else None)
        self._apply, self._set = binding().apply_adapters, bytes(held)
        # what a set can be refused for, now and not at the first call
        capi.check(capi.lib().infmoe_adapter_workspace_bytes(ctypes.byref(held), 0, ctypes.byref(ctypes.c_size_t())))

    def plan(self, adapter_of_token) -> AdapterPlan:
        """adapter_of_token: int32 CUDA tensor, one index per token; an index outside [0, n) means none."""
        return AdapterPlan(adapter_of_token, self.adapter_count)

    def apply(self, x, y, plan: AdapterPlan, out=None, status=None):
        """x [..., d_in], y [..., d_out] -> y plus each row's adapter of x.  out may be y (in place), not x.

        status (int32 [1], may be None): bit 2 is set when a bounded wait inside a kernel ran out.  The result is then not complete,
        and without a status nothing says so.  A plan may be used, and given up, on other streams than that it was made on, once
        they have waited for it."""
        return self._apply(self._set, *self._tensors, x, y, plan.buffer, plan.tokens, plan.adapter_count, out, status, self._home,
                           plan._home)
