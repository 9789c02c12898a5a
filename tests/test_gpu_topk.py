"""Routing to the k best experts, and rows to k experts and back, against 64-bit references (tests/topk_ref.py)."""
import numpy as np
import pytest
import torch

from infmoe_b200 import MoELayer, TopKRouter, capi, combine_topk, count_experts, scatter_topk, synth
from tests import topk_ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# Weights, in half units of the last place (2^-24) for logits within 16 of each other: expf's argument 16 and its value 4, the
# sigmoid's sum 1 and its 4 again from the exponential inside, quotient 1; the same once more for the sum of up to 32 of them,
# which adds 5; quotient and scale 2.
WEIGHT_TOL = (2 * 26 + 5 + 2) * 2.0 ** -24


def lowest(dtype):
    return topk_ref.LOWEST[str(dtype)[6:]]


def check_select(logits, k, score, bias=None, groups=1, top_groups=1, group_best=1, renormalise=True, scale=1.0):
    router = TopKRouter(logits.shape[-1], k, score=score, bias=bias, groups=groups, top_groups=top_groups,
                        group_best=group_best, renormalise=renormalise, scale=scale)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    gate, weight = router.select(logits, status=status)
    flat = logits.reshape(-1, logits.shape[-1])
    want, w = topk_ref.select(flat.double().cpu().numpy(), lowest(logits.dtype), k, score,
                              None if bias is None else bias.double().cpu().numpy(), groups, top_groups, group_best,
                              renormalise, scale)
    assert gate.shape == (*logits.shape[:-1], k) and weight.shape == gate.shape
    np.testing.assert_array_equal(gate.reshape(-1, k).cpu().numpy(), want)
    np.testing.assert_allclose(weight.reshape(-1, k).cpu().numpy(), w, rtol=WEIGHT_TOL, atol=1e-37)
    assert int(status) == int((want[:, 0] < 0).any())
    return gate, weight


def logits_of(T, E, dtype, seed=0, spread=1.5):
    rng = np.random.default_rng(seed)
    return torch.from_numpy(np.clip(rng.standard_normal((T, E)) * spread, -8, 8)).cuda().to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 2, 2), (5, 7, 3), (33, 8, 2), (100, 31, 5), (64, 32, 8), (63, 33, 33 - 1),
                                   (200, 64, 2), (50, 100, 10), (77, 128, 8), (40, 129, 8), (300, 256, 8), (9, 257, 4),
                                   (20, 512, 16), (10, 513, 6), (6, 1000, 32), (5, 1024, 8)])
def test_select(T, E, k, score, dtype):
    l = logits_of(T, E, TYPES[dtype], T + E)
    bias = torch.from_numpy(np.random.default_rng(E).standard_normal(E).astype(np.float32) * 0.1).cuda()
    check_select(l, k, score)
    check_select(l, k, score, renormalise=False, scale=2.5)
    check_select(l, k, score, bias=bias)
    check_select(l, k, score, bias=10 * bias - 0.5, renormalise=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score,bias", [("softmax", False), ("softmax", True), ("sigmoid", False), ("sigmoid", True)])
@pytest.mark.parametrize("T,E,k,groups,top_groups", [(1, 4, 2, 2, 1), (70, 64, 6, 8, 3), (90, 128, 8, 8, 4), (50, 256, 8, 8, 4),
                                                     (30, 60, 6, 5, 3), (30, 60, 12, 30, 6), (20, 32, 8, 32, 9), (20, 96, 4, 3, 2),
                                                     (20, 160, 6, 8, 3), (7, 512, 8, 16, 16), (7, 544, 8, 17, 4),
                                                     (9, 1024, 12, 32, 3), (40, 100, 5, 2, 1)])
@pytest.mark.parametrize("group_best", [1, 2])
def test_select_in_groups(T, E, k, groups, top_groups, group_best, score, bias, dtype):
    l = logits_of(T, E, TYPES[dtype], T * E + groups)
    b = torch.from_numpy(np.random.default_rng(E).standard_normal(E).astype(np.float32) * 0.1).cuda() if bias else None
    check_select(l, k, score, b, groups, top_groups, group_best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", TYPES)
def test_select_ties_go_to_the_lowest_index(dtype, score):
    rng = np.random.default_rng(3)
    l = torch.from_numpy(rng.integers(-2, 3, size=(300, 100)).astype(np.float32)).cuda().to(TYPES[dtype])
    check_select(l, 10, score)
    check_select(l, 10, score, bias=torch.zeros(100, device="cuda"))
    check_select(l, 10, score, None, 10, 3, 1)
    for best in (1, 2):
        check_select(l, 10, score, torch.full((100,), 0.25, device="cuda"), 5, 2, best)
    check_select(torch.zeros(4, 64, device="cuda", dtype=TYPES[dtype]), 8, score, None, 8, 2, 2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,groups,top_groups", [(2, 1, 1), (24, 4, 2), (60, 5, 3), (100, 10, 3), (256, 8, 4), (513, 1, 1), (1024, 32, 3)])
def test_select_zeros_of_both_signs_are_ties(E, groups, top_groups, dtype, score):
    """A logit masked by a product with zero is +0 or -0: one value.  16 experts are chosen in 32 bits, 17 in 64."""
    rng = np.random.default_rng(E)
    l = np.where(rng.random((60, E)) < 0.8, np.copysign(0.0, rng.standard_normal((60, E))), -1.0)
    l[0], l[0, -1] = -0.0, 0.0
    l[1:20] = np.where(rng.random((19, E)) < 0.2, 1.0, l[1:20])
    l = torch.from_numpy(l).cuda().to(TYPES[dtype])
    assert torch.signbit(l[0, 0]) and not torch.signbit(l[0, -1])
    size = E // groups
    for k in (1, 2, 16, 17):
        for best in (1, 2):
            if k <= E and best == 1:
                check_select(l, k, score)
                check_select(l, k, score, torch.full((E,), -0.0, device="cuda"))
            if groups > 1 and k <= top_groups * size:
                check_select(l, k, score, None, groups, top_groups, best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_select_where_32_bits_do_not_tell_apart(score):
    """Scores plus bias that differ by less than a 32-bit sum shows: the choice is that of 64 bits."""
    rng = np.random.default_rng(5)
    T, E = 400, 96
    l = rng.standard_normal((T, E)).astype(np.float32)
    s = 1 / (1 + np.exp(-l[0].astype(np.float64)))
    if score == "softmax":
        s = np.exp(l[0].astype(np.float64))
        s /= s.sum()
    bias = (0.5 - s).astype(np.float32)                 # every sum of row 0 within rounding of 0.5
    l[1:] = l[0] + rng.integers(-2, 3, size=(T - 1, E)).astype(np.float32) * np.float32(2.0 ** -23)
    dl, db = torch.from_numpy(l).cuda(), torch.from_numpy(bias).cuda()
    check_select(dl, 8, score, db)
    check_select(dl, 8, score, db, 8, 3, 2)
    check_select(dl, 8, score, db, 8, 3, 1)
    check_select(dl, 4, score, None, 8, 3, 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score,bias", [("softmax", False), ("softmax", True), ("sigmoid", False), ("sigmoid", True)])
@pytest.mark.parametrize("E,groups,top_groups", [(20, 1, 1), (31, 1, 1), (96, 8, 6), (160, 8, 5), (256, 8, 4), (270, 30, 20), (513, 1, 1),
                                                 (544, 17, 4), (1000, 1, 1), (1024, 32, 3)])
def test_select_alone_as_among_others(E, groups, top_groups, score, bias, dtype):
    """More than 16 experts to a token are always chosen in 64 bits: a token's choice does not depend on those beside it."""
    t = TYPES[dtype]
    rng = np.random.default_rng(E + groups)
    l = logits_of(48, E, t, E)
    l[1] = -np.inf
    l[2, : E // 2] = torch.finfo(t).min
    l[3, ::2] = np.nan
    l[4] = l[4, 0].item()                                # all alike
    l[5, E // 3] = np.inf
    l[6, 3:] = -np.inf                                   # fewer than k
    l[7] = torch.from_numpy(rng.integers(0, 3, size=E)).to(t).cuda()
    b = torch.from_numpy(np.round(rng.standard_normal(E), 1).astype(np.float32) * 0.1).cuda() if bias else None
    if bias:
        b[0], b[E - 1] = -np.inf, np.nan
    for best in (1, 2) if groups > 1 else (1,):
        for renormalise in (True, False):
            gate, weight = check_select(l, 20, score, b, groups, top_groups, best, renormalise)
            for i in range(9):
                one = check_select(l[i:i + 1], 20, score, b, groups, top_groups, best, renormalise)
                assert torch.equal(one[0][0], gate[i]) and torch.equal(one[1][0], weight[i])
                two = check_select(l[i:i + 2], 20, score, b, groups, top_groups, best, renormalise)
                assert torch.equal(two[0], gate[i:i + 2]) and torch.equal(two[1], weight[i:i + 2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_select_masks(score, dtype):
    t = TYPES[dtype]
    l = logits_of(60, 48, t, 11)
    l[0] = -np.inf
    l[1] = torch.finfo(t).min
    l[2] = np.nan
    l[3, 1:] = -np.inf                                  # one left
    l[4, :46] = torch.finfo(t).min                      # two left, fewer than k
    l[5, 10:20] = np.nan
    l[6, 5] = np.inf
    l[7, [5, 40]] = np.inf
    l[8:20, 12:24] = -np.inf                            # a whole group of four
    l[20:30, ::2] = -np.inf
    l[30] = torch.finfo(t).min
    l[30, [3, 30]] = torch.tensor([torch.finfo(t).min / 2, torch.finfo(t).max]).to(t).cuda()
    bias = torch.zeros(48, device="cuda")
    bias[7], bias[9], bias[30] = -np.inf, np.nan, 0.3
    for b in (None, bias):
        check_select(l, 5, score, b)
        check_select(l, 5, score, b, renormalise=False)
        for best in (1, 2):
            check_select(l, 5, score, b, 4, 2, best)
            check_select(l, 5, score, b, 16, 2, best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_select_weights_where_all_scores_are_tiny(score):
    """Renormalised weights come from the chosen logits and do not vanish with their scores."""
    l = logits_of(20, 40, torch.float32, 2)
    l[:, :20] -= 200
    l[:, 20:] = -np.inf
    gate, weight = check_select(l, 6, score)
    assert torch.allclose(weight.sum(1), torch.ones(20, device="cuda"), rtol=1e-6)


def test_select_strides_shapes_and_given_outputs():
    wide = logits_of(50, 200, torch.bfloat16, 4)
    check_select(wide[:, 3:67], 4, "softmax")           # rows apart, and not aligned
    check_select(wide[::2, 8:72], 4, "sigmoid")
    check_select(wide.view(5, 10, 200), 4, "softmax")
    check_select(wide[7], 4, "softmax")                 # one row
    router = TopKRouter(64, 4)
    gate = torch.full((52, 4), -7, dtype=torch.int32, device="cuda")
    weight = torch.full((52, 4), -7.0, device="cuda")
    router.select(wide[:, :64], gate[:50], weight[:50])
    assert (gate[50:] == -7).all() and (weight[50:] == -7).all() and (gate[:50] >= 0).all()
    empty = router.select(wide[:0, :64])
    assert empty[0].shape == (0, 4) and empty[1].shape == (0, 4)
    with pytest.raises(ValueError):
        router.select(wide[:1, :64].expand(4, 64))      # rows on top of one another
    with pytest.raises(ValueError):
        router.select(wide[:, :64].double())
    with pytest.raises(ValueError):
        router.select(wide[:, :63])
    with pytest.raises(ValueError):
        router.select(wide[:, :64], gate=gate)
    with pytest.raises(ValueError):
        router.select(wide.t()[:64].t()[:, :64].t().contiguous().t())


def test_select_bias_is_read_at_every_call():
    l = logits_of(30, 16, torch.float32, 9)
    bias = torch.zeros(16, device="cuda")
    router = TopKRouter(16, 1, score="sigmoid", bias=bias)
    first = router.select(l)[0].clone()
    bias[3] = 2.0
    assert (router.select(l)[0] == 3).all() and not (first == 3).all()


def test_select_refuses_a_bias_that_was_replaced():
    l = logits_of(30, 16, torch.float32, 9)
    router = TopKRouter(16, 1, score="sigmoid", bias=torch.zeros(16, device="cuda"))
    for bias in (torch.zeros(15, device="cuda"), torch.zeros(16, dtype=torch.bfloat16, device="cuda"),
                 torch.zeros(32, device="cuda")[::2], torch.zeros(16)):
        router.bias = bias
        with pytest.raises(ValueError, match="bias"):
            router.select(l)


def choice_of_all(l, k, score, bias, groups, top_groups, group_best, renormalise):
    """topk_ref.select for many rows at once, in 64 bits on the GPU."""
    T, E = l.shape
    ok = l > torch.finfo(l.dtype).min
    d = torch.where(ok, l.double(), -torch.inf)
    p = torch.softmax(d, 1).nan_to_num(0) if score == "softmax" else torch.where(ok, torch.sigmoid(d), 0.0)
    c = torch.where(ok, p + bias.double(), -torch.inf) if bias is not None else d
    if groups > 1:
        best = torch.where(ok, c if bias is not None or group_best == 1 else p, -torch.inf).view(T, groups, -1).topk(min(2, E // groups), 2).values
        value = best[:, :, 0]
        if group_best == 2 and best.shape[2] == 2:
            value = value + torch.where(best[:, :, 1] > -torch.inf, best[:, :, 1], 0.0)
        order = value.sort(dim=1, descending=True, stable=True).indices
        out = torch.zeros(T, groups, dtype=torch.bool, device="cuda").scatter(1, order[:, top_groups:], True)
        c = c.masked_fill(out.repeat_interleave(E // groups, 1), -torch.inf)
    value, gate = c.sort(dim=1, descending=True, stable=True)
    gate, none = gate[:, :k], value[:, :k] == -torch.inf
    w = p.gather(1, gate).masked_fill(none, 0.0)
    if renormalise:
        w = (w / w.sum(1, keepdim=True)).nan_to_num(0)
    return gate.masked_fill(none, -1).to(torch.int32), w


@pytest.mark.parametrize("dtype,score,E,k,groups,top_groups,group_best,bias,renormalise", [
    ("f32", "softmax", 24, 4, 1, 1, 1, False, True), ("bf16", "softmax", 64, 2, 1, 1, 1, False, False),
    ("f16", "sigmoid", 120, 6, 5, 3, 2, True, True), ("f32", "sigmoid", 256, 8, 8, 4, 2, True, True),
    ("f32", "softmax", 256, 20, 8, 4, 1, False, True), ("bf16", "softmax", 512, 16, 1, 1, 1, True, False),
    ("f32", "sigmoid", 1000, 7, 1, 1, 1, True, True)])
@pytest.mark.parametrize("T", [10000, 160000])
def test_select_of_many_tokens(T, dtype, score, E, k, groups, top_groups, group_best, bias, renormalise):
    """A warp's second token comes after 2368 to 4736 of them, a block's second 32 turns after 75776 to 151552."""
    l = logits_of(T, E, TYPES[dtype], E)
    l[::97] = -torch.inf
    l[1::101, E // 2:] = torch.nan
    b = torch.from_numpy(np.random.default_rng(E).standard_normal(E).astype(np.float32) * 0.1).cuda() if bias else None
    router = TopKRouter(E, k, score=score, bias=b, groups=groups, top_groups=top_groups, group_best=group_best, renormalise=renormalise)
    gate, weight = router.select(l)
    for t0 in range(0, T, 20000):
        want, w = choice_of_all(l[t0:t0 + 20000], k, score, b, groups, top_groups, group_best, renormalise)
        assert torch.equal(gate[t0:t0 + 20000], want)
        torch.testing.assert_close(weight[t0:t0 + 20000].double(), w, rtol=WEIGHT_TOL, atol=1e-37)


def slots_of(T, k, E, none=0.1, seed=0):
    rng = np.random.default_rng(seed)
    gate = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32) if T else np.zeros((0, k), np.int32)
    gate[rng.random((T, k)) < none] = -1
    return torch.from_numpy(gate).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,D,E", [(1, 1, 1, 1), (1, 8, 64, 8), (3, 2, 8, 4), (17, 3, 510, 7), (5, 8, 4096, 64), (64, 4, 100, 9),
                                     (130, 6, 36, 60), (33, 2, 4097, 5), (300, 8, 256, 128), (2, 4, 10240, 32)])
def test_rows_to_their_experts_and_back(T, k, D, E, dtype):
    rng = np.random.default_rng(T * D)
    t = TYPES[dtype]
    x = torch.from_numpy(rng.standard_normal((T, D))).cuda().to(t)
    gate = slots_of(T, k, E)
    pos, count, offset = count_experts(gate, E)
    out = torch.full((T * k, D), 7.0, device="cuda", dtype=t)
    routed, row_of = scatter_topk(x, pos, offset, k, out=out)
    n = int(offset[-1])
    g = gate.flatten().cpu().numpy()
    order = np.argsort(np.where(g < 0, E, g), kind="stable")
    assert n == int((g >= 0).sum())
    want_row = np.full(T * k, -1)
    want_row[order[:n]] = np.arange(n)
    np.testing.assert_array_equal(row_of.cpu().numpy().ravel(), want_row)
    assert torch.equal(routed[:n], x[torch.from_numpy(order[:n] // k).cuda()])
    assert (out[n:] == 7).all()                                     # rows behind the last are left as they were

    y = torch.from_numpy(rng.standard_normal((T * k, D))).cuda().to(t)
    y[n:] = np.nan                                                  # nobody reads them
    weight = torch.from_numpy(rng.random((T, k)).astype(np.float32)).cuda()
    for residual in (None, x):
        got = combine_topk(y, weight, row_of=row_of, residual=residual)
        check_combined(got, y, weight, row_of.cpu().numpy(), residual)


@pytest.mark.parametrize("dtype,T,k,D", [("f32", 700, 4, 1024), ("f32", 3000, 3, 1001), ("bf16", 3000, 3, 1001), ("f16", 2500, 2, 1002),
                                         ("bf16", 300001, 3, 5), ("f32", 250000, 3, 3), ("f16", 150000, 8, 8), ("f32", 5, 2, 300004)])
def test_many_rows_to_their_experts(dtype, T, k, D):
    """More than 8 MB of them: four rows to a thread, by 16, 4 and 2 bytes, long rows and short ones."""
    t, E = TYPES[dtype], 60
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, D, device="cuda", generator=g).to(t)
    gate = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
    gate[torch.rand(T, device="cuda", generator=g) < 0.1] = -1
    pos, _, offset = count_experts(gate, E)
    routed, row_of = scatter_topk(x, pos, offset, k, out=torch.full((T * k, D), 7.0, device="cuda", dtype=t))
    flat = gate.flatten().long()
    order = torch.where(flat < 0, E, flat).sort(stable=True).indices
    n = int((flat >= 0).sum())
    want_row = torch.full((T * k,), -1, dtype=torch.int32, device="cuda")
    want_row[order[:n]] = torch.arange(n, dtype=torch.int32, device="cuda")
    assert int(offset[-1]) == n and torch.equal(row_of.flatten(), want_row)
    assert torch.equal(routed[:n], x[order[:n] // k]) and (routed[n:] == 7).all()


def check_combined(got, y, weight, row_of, residual):
    d = lambda v: None if v is None else v.double().cpu().numpy()  # noqa: E731
    want, size = topk_ref.combine(d(y), d(weight), row_of, d(residual))
    k = weight.shape[1]
    eps = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[y.dtype]
    # k + 1 fused multiply-adds and, in the rest, k subtractions, each half a unit in 32 bits; the stored type's half unit
    # (FP16: also half of its smallest step)
    tol = (2 * k + 2) * 2.0 ** -24 * size + eps * np.abs(want) + (2.0 ** -25 if y.dtype == torch.float16 else 0)
    err = np.abs(d(got) - want)
    assert (err <= tol * (1 + 2.0 ** -8)).all(), (err / np.maximum(tol, 1e-300)).max()


@pytest.mark.parametrize("dtype", TYPES)
def test_combine_in_slot_order_and_with_gates(dtype):
    rng = np.random.default_rng(8)
    T, k, D = 40, 5, 72
    t = TYPES[dtype]
    y = torch.from_numpy(rng.standard_normal((T * k, D))).cuda().to(t)
    x = torch.from_numpy(rng.standard_normal((T, D))).cuda().to(t)
    weight = torch.from_numpy(rng.random((T, k)).astype(np.float32)).cuda()
    gate = slots_of(T, k, 9, 0.3)
    gate[0] = -1                                                    # a token without any expert
    y.view(T, k, D)[gate < 0] = np.nan
    rows = np.where(gate.cpu().numpy() >= 0, np.arange(T * k).reshape(T, k), -1)
    for residual in (None, x):
        got = combine_topk(y, weight, gate=gate, residual=residual)
        check_combined(got, y, weight, rows, residual)
        assert torch.equal(got[0], x[0] if residual is not None else torch.zeros_like(x[0]))
    inplace = x.clone()
    want = combine_topk(y, weight, gate=gate, residual=x)
    assert torch.equal(combine_topk(y, weight, gate=gate, residual=inplace, out=inplace), want)
    # rows outside [0, n), the same row twice
    odd = torch.from_numpy(rng.integers(-3, 23, size=(T, k)).astype(np.int32)).cuda()
    few = torch.nan_to_num(y[:20])
    check_combined(combine_topk(few, weight, row_of=odd), few, weight, odd.cpu().numpy(), None)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_unaligned_tensors(dtype):
    t = TYPES[dtype]
    rng = np.random.default_rng(1)
    T, k, D, E = 21, 3, 64, 6
    gate = slots_of(T, k, E)
    pos, _, offset = count_experts(gate, E)
    base = torch.from_numpy(rng.standard_normal((T, D + 3))).cuda().to(t)
    for x in (base[:, :D], base[:, 1:D + 1], base[:, 3:]):
        routed, row_of = scatter_topk(x, pos, offset, k)
        again, row_of2 = scatter_topk(x.contiguous(), pos, offset, k)
        n = int(offset[-1])
        assert torch.equal(routed[:n], again[:n]) and torch.equal(row_of, row_of2)
    flat = torch.from_numpy(rng.standard_normal(T * k * D + 1)).cuda().to(t)
    weight = torch.rand(T, k, device="cuda")
    rows = flat[1:].view(T * k, D)                                  # starts between two 16-byte boundaries
    assert torch.equal(combine_topk(rows, weight, row_of=row_of), combine_topk(rows.clone(), weight, row_of=row_of))


def test_rows_past_32_bits():
    """Offsets of elements beyond 2^32: rows at the far end of large tensors."""
    D, n = 4096, (1 << 20) + 64
    y = torch.zeros(n, D, dtype=torch.float16, device="cuda")       # 8.6 GB
    y[-3:] = torch.arange(3, device="cuda", dtype=torch.float16)[:, None] + 1
    weight = torch.ones(1, 3, device="cuda")
    row_of = torch.tensor([[n - 3, n - 1, n - 2]], dtype=torch.int32, device="cuda")
    assert (combine_topk(y, weight, row_of=row_of) == 6).all()
    pos = torch.tensor([n - 1, 0], dtype=torch.int32, device="cuda")
    pos = torch.cat([pos, torch.arange(1, n - 1, dtype=torch.int32, device="cuda")])
    routed, row_of = scatter_topk(y, pos, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), 1)
    assert (routed[0] == 3).all() and (routed[1] == 0).all() and int(row_of[n - 1]) == 0 and int(row_of[5]) == -1


def small_layer(E=6, D=64, F=128, variant="default", **kw):
    w = synth.scaled(synth.WORKLOADS["tiny_default"], variant=variant, expert_count=E, embedding_size=D, hidden_size=F)
    x, cent, ln = synth.gen_inputs(synth.scaled(w, batch=1, seq_len=70))
    experts = [synth.gen_expert_numpy(w, e) for e in range(E)]
    layer = MoELayer.create(E, D, F, 2, cent, None, kw.get("sublayer", "T5_FF"), variant, ln)
    for e, ex in enumerate(experts):
        # a pass can be captured when the experts came as device tensors: no upload to wait for
        layer.set_expert(e, *([torch.from_numpy(v).cuda() for v in ex] if kw.get("on_device") else ex))
    return layer, experts, x


def reference_pass(oracle, x, gate, weight, experts):
    out = x.astype(np.float64)
    for s in range(gate.shape[1]):
        for e in range(len(experts)):
            rows = np.flatnonzero(gate[:, s] == e)
            if len(rows):
                out[rows] += weight[rows, s, None].astype(np.float64) * (oracle.expert_ffn_f64(x[rows], *experts[e]) - x[rows])
    return out


@pytest.mark.parametrize("E,D,F,k,T", [(6, 64, 128, 2, 70), (6, 64, 128, 1, 1), (9, 256, 512, 4, 70), (4, 66, 130, 3, 33),
                                       (5, 100, 60, 2, 17)])
@pytest.mark.parametrize("mode", ["resident", "streamed"])
def test_layer_with_several_experts_per_token(oracle, E, D, F, k, T, mode):
    layer, experts, x = small_layer(E, D, F)
    layer.set_residency(1 if mode == "resident" else 0)
    x = x[:T]
    dx = torch.from_numpy(x).cuda()
    gate, weight = TopKRouter(E, k, score="sigmoid", renormalise=k > 2).select(logits_of(T, E, torch.float32, E))
    if T > 5:
        gate[2, 0], gate[3], gate[4, 0] = -1, -1, E + 3
    out = layer.forward_topk(dx, gate, weight)
    layer.sync_status()
    want = reference_pass(oracle, x, gate.cpu().numpy(), weight.cpu().numpy(), experts)
    assert oracle.rel_l2(out.cpu().numpy(), want) <= 1e-5
    if T > 5:
        assert torch.equal(out[3], dx[3])
    layer.terminate()


def test_layer_of_identity_experts():
    layer, _, x = small_layer(4, 32, 64, sublayer="Identity")
    dx = torch.from_numpy(x).cuda()
    gate, weight = TopKRouter(4, 3).select(logits_of(70, 4, torch.float32))
    assert torch.allclose(layer.forward_topk(dx, gate, weight), dx, rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("mode", ["enqueue_first", "topk_first"])
def test_last_routing_is_that_of_the_last_enqueue(mode):
    layer, _, x = small_layer(4, 32, 64)
    dx = torch.from_numpy(x).cuda()
    gate, weight = TopKRouter(4, 2).select(logits_of(70, 4, torch.float32))
    if mode == "topk_first":
        layer.forward_topk(dx, gate, weight)
        with pytest.raises(capi.InfMoEError):
            layer.last_routing()
    layer.forward(dx)
    before = layer.last_routing()
    layer.forward_topk(dx, gate, weight)
    assert layer.last_routing() == before and gate.data_ptr() not in before
    layer.sync_status()
    layer.terminate()


def test_router_rows_and_experts_together(oracle):
    """Router -> dispatch -> rows to experts -> experts of the caller -> rows back, against the layer's own pass and 64 bits."""
    E, D, F, k, T = 8, 128, 256, 3, 70
    layer, experts, x = small_layer(E, D, F)
    dx = torch.from_numpy(x).cuda()
    bias = torch.linspace(-0.2, 0.2, E, device="cuda")
    logits = logits_of(T, E, torch.bfloat16, 21)
    logits[11] = -np.inf
    gate, weight = TopKRouter(E, k, score="sigmoid", bias=bias, groups=4, top_groups=2, group_best=2, scale=1.5).select(logits)
    pos, count, offset = count_experts(gate, E)
    routed, row_of = scatter_topk(dx, pos, offset, k)
    n = int(offset[-1])
    assert n == 3 * 69
    results = torch.empty_like(routed)
    owner = torch.repeat_interleave(torch.arange(E, dtype=torch.int32, device="cuda"), count)
    results[:n] = layer.expert_forward(routed[:n].contiguous(), owner)
    out = combine_topk(results, weight, row_of=row_of, residual=dx)
    want = reference_pass(oracle, x, gate.cpu().numpy(), weight.cpu().numpy(), experts)
    assert oracle.rel_l2(out.cpu().numpy(), want) <= 1e-5
    assert oracle.rel_l2(layer.forward_topk(dx, gate, weight).cpu().numpy(), want) <= 1e-5
    assert torch.equal(out[11], dx[11])
    layer.terminate()


def test_captured_and_replayed(oracle):
    layer, experts, x = small_layer(8, 64, 128, on_device=True)
    T, E, k = 70, 8, 2
    dx = torch.from_numpy(x).cuda()
    logits = logits_of(T, E, torch.float32, 5)
    router = TopKRouter(E, k)

    def step():
        gate, weight = router.select(logits)
        pos, _, offset = count_experts(gate, E)
        routed, row_of = scatter_topk(dx, pos, offset, k)
        return gate, weight, layer.forward_topk(dx, gate, weight), combine_topk(routed, weight, row_of=row_of)

    step()
    torch.cuda.synchronize()
    graphs, answers = [], []
    for _ in range(2):                                              # two graphs with memory of their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            answers.append(step())
        graphs.append(g)
    for seed in (6, 7):
        logits.copy_(logits_of(T, E, torch.float32, seed))
        dx.copy_(torch.from_numpy(np.random.default_rng(seed).standard_normal(x.shape).astype(np.float32)))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        eager = step()
        for got in answers:
            for u, v in zip(got, eager):
                assert torch.equal(u, v)
    del graphs
    layer.terminate()


def test_on_another_stream():
    logits = logits_of(500, 64, torch.float32, 1)
    router = TopKRouter(64, 8)
    want = router.select(logits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big * 1e-2                                  # the stream is busy while the inputs change behind it
        logits2 = (logits * 2).contiguous()
        got = router.select(logits2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0])                             # doubling the logits keeps their order
