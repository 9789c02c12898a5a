"""B200-native MoE layer behind InfMoE's plugin interface.

Public surface (same names as the reference's python/infmoe/__init__.py:6-10):
MoELayerConfig, MoELayerPlugin and the helpers of utils; plus MoELayer, the object create_plugin returns, and what the
reference has no counterpart for: several experts per token (topk) and low-rank adapters of requests (adapters).
"""
from .adapters import AdapterPlan, Adapters
from .config import MoELayerConfig
from .plugin import MoELayer, MoELayerPlugin
from .topk import TopKRouter, combine_topk, count_experts, scatter_topk
from .utils import HostDeviceMem, allocate_buffers, create_layer_from_plugin, do_inference

__version__ = '0.0.1'
__all__ = ["MoELayerConfig", "MoELayerPlugin", "MoELayer", "HostDeviceMem", "allocate_buffers", "do_inference",
           "create_layer_from_plugin", "TopKRouter", "count_experts", "scatter_topk", "combine_topk", "Adapters",
           "AdapterPlan"]
