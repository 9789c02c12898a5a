"""What the operators for several experts per token and for adapters refuse, before any device work."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

from infmoe_b200 import Adapters, TopKRouter, capi, combine_topk, count_experts, scatter_topk
from tests import topk_ref

GOOD = dict(expert_count=16, top_k=4, score=1, group_count=4, top_groups=2, group_best=2, renormalise=1, scale=1.0)
SOME = 1 << 20      # an address that no refused call looks at


def _select(T=3, logits=SOME, dtype=0, ld=16, gate=SOME, weight=SOME, cfg=None, **kw):
    c = capi.TopKConfig(**{**GOOD, **kw})
    ref = ctypes.byref(c) if cfg is None else cfg
    return capi.lib().infmoe_expert_select_topk(ref, T, logits, dtype, ld, None, gate, weight, None, None)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(T=1 << 31), dict(logits=None), dict(gate=None), dict(weight=None),
                                 dict(dtype=3), dict(dtype=-1), dict(ld=15), dict(expert_count=0), dict(expert_count=18, ld=18),
                                 dict(top_k=0), dict(top_k=9), dict(group_count=0), dict(group_count=32, ld=32),
                                 dict(top_groups=0), dict(top_groups=5), dict(group_best=0), dict(group_best=3), dict(score=2)],
                         ids=str)
def test_select_refuses_bad_arguments(bad):
    assert _select(**bad) == 1 and "expert_select_topk" in capi.last_error()


def test_select_refuses_what_no_kernel_has_lanes_for():
    big = dict(group_count=1, top_groups=1, top_k=1)
    assert _select(T=0, expert_count=1024, ld=1024, **big) == 0
    assert _select(T=0, expert_count=1025, ld=1025, **big) == 6
    assert _select(T=0, expert_count=64, ld=64, group_count=1, top_groups=1, top_k=33) == 6
    assert _select(T=0, expert_count=66, ld=66, group_count=33, top_groups=1, top_k=1) == 6
    assert _select(T=0, expert_count=17 * 33, ld=17 * 33, group_count=17, top_groups=1, top_k=1) == 6
    assert _select(T=0) == 0
    assert capi.lib().infmoe_expert_select_topk(None, 0, None, 0, 1, None, None, None, None, None) == 1


@pytest.mark.parametrize("at,value,status", [(0, -1, 1), (1, 0, 1), (2, 0, 1), (3, 7, 1), (4, None, 1), (5, 7, 1), (6, None, 1),
                                             (7, None, 1), (8, None, 1), (0, 1 << 30, 6)])
def test_scatter_refuses_bad_arguments(at, value, status):
    args = [3, 2, 8, 0, SOME, 8, SOME, SOME, SOME, SOME, None]
    args[at] = value
    assert capi.lib().infmoe_expert_scatter_topk(*args) == status


@pytest.mark.parametrize("at,value,status", [(0, -1, 1), (1, 0, 1), (2, -8, 1), (3, 9, 1), (4, None, 1), (5, -1, 1), (6, None, 1),
                                             (10, None, 1), (10, SOME, 1), (0, 1 << 30, 6)])
def test_combine_refuses_bad_arguments(at, value, status):
    args = [3, 2, 8, 0, SOME, 6, SOME, None, None, None, 2 * SOME, None]
    args[at] = value
    assert capi.lib().infmoe_expert_combine_topk(*args) == status


def _apply(T=4, x=SOME, ldx=32, y=2 * SOME, ldy=48, out=3 * SOME, ldo=48, plan=4 * SOME, ws=5 * SOME, ws_bytes=1 << 20, **kw):
    s = capi.AdapterSet(**{**dict(adapter_count=3, rank=8, d_in=32, d_out=48, dtype=2, d_a=SOME, d_b=SOME), **kw})
    return capi.lib().infmoe_adapter_apply(ctypes.byref(s), T, x, ldx, y, ldy, out, ldo, plan, ws, ws_bytes, None, None)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(x=None), dict(y=None), dict(out=None), dict(plan=None), dict(plan=8),
                                 dict(ldx=31), dict(ldy=47), dict(ldo=47), dict(out=SOME), dict(out=2 * SOME, ldo=64),
                                 dict(adapter_count=0), dict(rank=0), dict(d_in=0), dict(d_out=-1), dict(dtype=5),
                                 dict(d_a=None), dict(d_b=None), dict(ws=None), dict(ws=8), dict(ws_bytes=100)], ids=str)
def test_apply_refuses_bad_arguments(bad):
    assert _apply(**bad) == 1 and "adapter_apply" in capi.last_error()


def test_apply_refuses_what_is_too_large():
    assert _apply(rank=capi.ADAPTER_MAX_RANK + 1) == 6
    assert _apply(adapter_count=100000) == 6
    assert _apply(T=1 << 31) == 6
    assert _apply(T=0, rank=capi.ADAPTER_MAX_RANK) == 0


def test_plan_refuses_bad_arguments():
    lib, n = capi.lib(), ctypes.c_size_t()
    assert lib.infmoe_adapter_plan_bytes(100, 7, ctypes.byref(n)) == 0
    need = n.value
    assert need >= 4 * 100 + 4 * 8 + 16 * 8
    assert lib.infmoe_adapter_plan_bytes(100, 7, None) == 1
    assert lib.infmoe_adapter_plan_bytes(-1, 7, ctypes.byref(n)) == 1
    assert lib.infmoe_adapter_plan_bytes(100, 0, ctypes.byref(n)) == 1
    assert lib.infmoe_adapter_plan_bytes(100, 100000, ctypes.byref(n)) == 6
    assert lib.infmoe_adapter_plan(100, 7, SOME, SOME, need - 1, None) == 1 and str(need) in capi.last_error()
    assert lib.infmoe_adapter_plan(100, 7, SOME, SOME + 4, need, None) == 1
    assert lib.infmoe_adapter_plan(100, 7, None, SOME, need, None) == 1
    assert lib.infmoe_adapter_plan(100, 7, SOME, None, need, None) == 1
    assert lib.infmoe_adapter_plan(0, 7, None, None, 0, None) == 0


def test_forward_topk_refuses_bad_arguments():
    from tests.test_capi_host import _layer

    layer, lib, n = _layer(), capi.lib(), ctypes.c_size_t()
    assert lib.infmoe_layer_topk_workspace_bytes(layer._h, 10, 2, ctypes.byref(n)) == 0
    need = n.value
    assert need > layer.get_workspace_size(20) + 2 * 20 * 8 * 4
    assert lib.infmoe_layer_topk_workspace_bytes(layer._h, 10, 0, ctypes.byref(n)) == 1
    assert lib.infmoe_layer_topk_workspace_bytes(layer._h, -1, 2, ctypes.byref(n)) == 1
    assert lib.infmoe_layer_topk_workspace_bytes(layer._h, 1 << 30, 2, ctypes.byref(n)) == 6
    assert lib.infmoe_layer_topk_workspace_bytes(layer._h, 10, 2, None) == 1
    good = [layer._h, SOME, SOME, SOME, 10, 2, 2 * SOME, 3 * SOME, need, None]
    for at, value, status in [(0, None, 1), (1, None, 1), (2, None, 1), (3, None, 1), (4, -1, 1), (5, 0, 1), (6, None, 1),
                              (6, SOME, 1), (7, None, 1), (8, need - 1, 1), (4, 1 << 40, 6)]:
        args = list(good)
        args[at] = value
        assert lib.infmoe_layer_forward_topk(*args) == status, (at, value)
    assert lib.infmoe_layer_forward_topk(*[0 if i == 4 else v for i, v in enumerate(good)]) == 0
    layer.terminate()


def test_python_refuses_tensors_off_the_device_and_bad_configurations():
    f = torch.zeros
    with pytest.raises(ValueError):
        TopKRouter(8, 2, score="tanh")
    with pytest.raises(ValueError):
        TopKRouter(8, 2, bias=f(8))                              # not on a GPU
    with pytest.raises(capi.InfMoEError):
        TopKRouter(8, 9)
    with pytest.raises(capi.InfMoEError):
        TopKRouter(9, 2, groups=2)
    with pytest.raises(ValueError):
        TopKRouter(8, 2).select(f(3, 8))
    with pytest.raises(ValueError):
        count_experts(f(6, dtype=torch.int32), 3)
    with pytest.raises(ValueError):
        scatter_topk(f(3, 8), f(6, dtype=torch.int32), f(4, dtype=torch.int32), 2)
    with pytest.raises(ValueError):
        combine_topk(f(6, 8), f(3, 2))
    with pytest.raises(ValueError):
        Adapters(f(2, 4, 8), f(2, 16, 4))


def test_reference_choices_by_hand():
    """The tests' own reference on rows whose answers are plain."""
    l = np.array([[1.0, 3.0, 2.0, 3.0], [-np.inf, np.nan, 0.0, -np.inf], [-np.inf] * 4])
    gate, w = topk_ref.select(l, topk_ref.LOWEST["float32"], 2, "softmax")
    assert gate.tolist() == [[1, 3], [2, -1], [-1, -1]]
    np.testing.assert_allclose(w, [[0.5, 0.5], [1, 0], [0, 0]])
    gate, w = topk_ref.select(l[:1], -1e38, 1, "sigmoid", np.array([9.0, 0, 0, 0]), renormalise=False)
    assert gate.tolist() == [[0]] and abs(w[0, 0] - 1 / (1 + np.exp(-1))) < 1e-15
    gate, _ = topk_ref.select(np.array([[5.0, -9, 2, 2.5]]), -1e38, 1, "sigmoid", None, 2, 1, 2)
    assert gate.tolist() == [[3]]                                # 0.993 + 0.0001 against 0.881 + 0.924


def test_rows_longer_than_a_grid_can_count_are_refused():
    lib = capi.lib()
    assert lib.infmoe_expert_scatter_topk(3, 2, 1 << 25, 0, SOME, 1 << 25, SOME, SOME, SOME, SOME, None) == 6
    assert lib.infmoe_expert_combine_topk(3, 2, 1 << 25, 0, SOME, 6, SOME, None, None, None, 2 * SOME, None) == 6
    assert _apply(d_in=(1 << 24) + 1, ldx=1 << 25) == 6
    assert _apply(d_out=(1 << 24) + 1, ldy=1 << 25, ldo=1 << 25) == 6


def _body(source, kernel):
    text = re.sub(r"//[^\n]*", "", source)
    at = text.index("{", text.index(f"{kernel}(const ApplyArgs p)"))
    depth, i = 0, at
    while True:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
        if depth == 0:
            return text[at:i]


def test_adapters_second_kernel_may_start_early():
    """It reads, before its own wait, what was there before the first one's, which therefore triggers behind its wait; and the first
    one, where it takes tensor memory, has it before it triggers: blocks that hold some must not keep others from theirs."""
    with open(os.path.join(os.path.dirname(capi.LIB_PATH), "csrc", "adapters.cu")) as f:
        source = f.read()
    for kernel in ("adapter_down_kernel", "adapter_down_tc_kernel"):
        body = _body(source, kernel)
        assert body.index("pdl_wait()") < body.index("pdl_trigger()"), kernel
    for kernel in ("adapter_down_tc_kernel", "adapter_up_tc_kernel"):
        body = _body(source, kernel)
        assert body.index("tmem_alloc(") < body.rindex("pdl_trigger()"), kernel
    for kernel in ("adapter_up_kernel", "adapter_up_tc_kernel"):        # shares of A x, and every store to memory
        body = _body(source, kernel)
        first_wait = body.index("pdl_wait()")
        assert body.index("p.sums") > first_wait and body.index("out_base + (long long)") > first_wait, kernel
        assert "mbar_wait" not in body[:first_wait]


@pytest.mark.parametrize("n", [1, 7, 1000])
def test_plans_of_more_rows_than_32_bits_count_are_refused(n):
    """A plan's tiles have room for up to 128 rows each: whole tiles, and one that is not full for every adapter and for none."""
    lib, need = capi.lib(), ctypes.c_size_t()
    most = ((1 << 31) // 128 - (n + 1)) * 128 - 1                    # tokens whose tiles have room for 2^31 - 128 rows
    assert lib.infmoe_adapter_plan_bytes(most, n, ctypes.byref(need)) == 0 and need.value > 12 * most
    for T in (most + 1, (1 << 31) - 1):
        assert lib.infmoe_adapter_plan_bytes(T, n, ctypes.byref(need)) == 6 and "plan" in capi.last_error()
        assert lib.infmoe_adapter_plan(T, n, SOME, SOME, 1 << 60, None) == 6
        assert _apply(T=T, adapter_count=n, ws_bytes=1 << 60) == 6
        s = capi.AdapterSet(adapter_count=n, rank=8, d_in=32, d_out=48, dtype=2, d_a=SOME, d_b=SOME)
        assert lib.infmoe_adapter_workspace_bytes(ctypes.byref(s), T, ctypes.byref(need)) == 6


def test_workspace_grows_with_what_a_call_uses():
    """One share of A x for every place of the tiles in large batches, eight at most in small ones; enough for every smaller batch."""
    lib, need = capi.lib(), ctypes.c_size_t()
    for dtype, rank, padded, n in ((0, 128, 128, 8), (2, 128, 128, 8), (1, 33, 64, 3), (2, 16, 16, 64), (0, 20, 32, 1000), (1, 20, 32, 1)):
        s = capi.AdapterSet(adapter_count=n, rank=rank, d_in=4096, d_out=4096, dtype=dtype, d_a=SOME, d_b=SOME)
        before = 0
        for T in sorted({1, 5, 16, 17, 100, 777, 2047, 2048, 4095, 4096, 32 * n - 1, 32 * n, 32 * n + 1, 131072, 1 << 20}):
            assert lib.infmoe_adapter_workspace_bytes(ctypes.byref(s), T, ctypes.byref(need)) == 0
            assert need.value >= max(before, 4 * padded * T)
            before = need.value
        assert need.value <= 4 * padded * (T + 128 * (n + 1))


def test_binding_is_built_for_the_torch_that_is_there(monkeypatch, tmp_path):
    import importlib.util
    import subprocess

    from infmoe_b200 import build

    made = []

    def compile_(cmd, **kw):
        made.append(cmd)
        with open(build.BINDING, "w") as f:
            f.write("")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "BINDING", str(tmp_path / "_binding.so"))
    monkeypatch.setattr(build, "BINDING_STAMP", str(tmp_path / "_binding.made_for"))
    monkeypatch.setattr(build.subprocess, "run", compile_)
    for _ in range(2):
        build._build_binding(False)
    assert len(made) == 1
    text = build._text
    monkeypatch.setattr(build, "_text", lambda path: "0.0" if path.endswith("version.py") else text(path))
    for _ in range(2):
        build._build_binding(False)
    assert len(made) == 2
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: None)
    build._build_binding(False)                                      # the libraries alone: no error
    assert len(made) == 2


def _depth(body, at):
    return body.count("{", 0, at) - body.count("}", 0, at)


def _touches_results_behind_its_wait(body):
    """The shares of A x and every store to memory come behind the one wait that is in no branch; in a branch, behind the branch's."""
    waits = [m.start() for m in re.finditer(r"pdl_wait\(\)", body)]
    main = [w for w in waits if _depth(body, w) == 1]
    if len(main) != 1:
        return False
    uses = [m.start() for m in re.finditer(r"p\.sums|\*reinterpret_cast<uint4\*>\(out|\bdst\[|\bout_base\[|out_base \+", body)]
    assert len(uses) >= 3 and "copy_rows<T>" in body
    branch = body.rindex("{", 0, body.index("copy_rows<T>"))
    return min(uses) > main[0] and any(branch < w < body.index("copy_rows<T>") for w in waits)


@pytest.mark.parametrize("kernel", ["adapter_up_kernel", "adapter_up_tc_kernel"])
def test_adapters_second_kernel_waits_for_the_first_ones_results(kernel):
    with open(os.path.join(os.path.dirname(capi.LIB_PATH), "csrc", "adapters.cu")) as f:
        body = _body(f.read(), kernel)
    assert _touches_results_behind_its_wait(body)
    waits = [m.start() for m in re.finditer(r"pdl_wait\(\);", body)]
    assert len(waits) == 3                       # an empty tile's, a tile's without adapter, the others'
    for w in waits[1:]:
        assert not _touches_results_behind_its_wait(body[:w] + body[w + len("pdl_wait();"):])
