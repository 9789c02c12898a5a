"""Low-rank adapters of many requests beside a shared projection, against a 64-bit reference (tests/topk_ref.py)."""
import numpy as np
import pytest
import torch

from infmoe_b200 import AdapterPlan, Adapters, synth
from tests import topk_ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def whole(rng, shape, most, dtype):
    return torch.from_numpy(rng.integers(-most, most + 1, size=shape).astype(np.float32)).cuda().to(dtype)


def owners(rng, T, n, requests, none=0.15):
    """Requests one behind the other, some of them with an index that means no adapter."""
    ends = np.sort(rng.integers(0, T + 1, size=requests - 1)) if requests < T else np.arange(1, T)
    which = rng.integers(0, n, size=requests).astype(np.int32)
    which[rng.random(requests) < none] = rng.choice([-1, n, n + 5, -9])
    return which[np.searchsorted(ends, np.arange(T), side="right")]


def reference(x, y, a, b, scale, rank, at):
    d = lambda v: None if v is None else v.double().cpu().numpy()  # noqa: E731
    n = a.shape[0]
    s = np.full(n, float(scale)) if isinstance(scale, (int, float)) else d(scale)
    return topk_ref.adapters(d(x), d(y), d(a), d(b), s, None if rank is None else rank.cpu().numpy(), at)


def check_exact(got, want, dtype):
    """Sums of whole numbers, exact in 32 bits whatever their order: only the last rounding is left."""
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(dtype)), \
        np.abs(got.double().cpu().numpy() - torch.from_numpy(want).to(dtype).double().numpy()).max()


# Whole numbers: |A x| <= 4 d_in in whole numbers, |B v| below 2^24; rounding to the type is the last step alone.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,n,r,d_in,d_out,requests", [
    (1, 1, 1, 1, 1, 1), (1, 1, 16, 64, 64, 1), (1, 3, 8, 4096, 4096, 1), (2, 2, 3, 7, 5, 2), (16, 4, 16, 256, 512, 16),
    (17, 2, 8, 100, 36, 3), (63, 5, 24, 510, 130, 7), (64, 1, 64, 1024, 256, 1), (65, 1, 33, 128, 1000, 1),
    (130, 3, 128, 520, 264, 3), (200, 9, 4, 1000, 2724, 31), (300, 40, 17, 72, 80, 100), (64, 64, 16, 2048, 2048, 64),
    (700, 2, 48, 1028, 516, 4), (37, 1000, 8, 64, 64, 37), (513, 6, 10, 96, 4100, 9), (5, 2, 127, 33, 2050, 2),
    (256, 2, 65, 192, 130, 2), (20, 3, 16, 10240, 64, 5)])
def test_whole_numbers(T, n, r, d_in, d_out, requests, dtype):
    rng = np.random.default_rng(T * 7 + r)
    t = TYPES[dtype]
    x, a = whole(rng, (T, d_in), 2, t), whole(rng, (n, r, d_in), 2, t)
    b, y = whole(rng, (n, d_out, r), 1, t), whole(rng, (T, d_out), 50, t)
    at = owners(rng, T, n, requests)
    scale = torch.from_numpy(2.0 ** rng.integers(-3, 1, size=n).astype(np.float32)).cuda()
    adapters = Adapters(a, b, scale=scale)
    plan = adapters.plan(torch.from_numpy(at).cuda())
    want = reference(x, y, a, b, scale, None, at)
    check_exact(adapters.apply(x, y, plan), want, t)
    inplace = y.clone()
    assert adapters.apply(x, inplace, plan, out=inplace) is inplace
    check_exact(inplace, want, t)
    rank = torch.from_numpy(rng.integers(-1, r + 3, size=n).astype(np.int32)).cuda()
    check_exact(Adapters(a, b, scale, rank).apply(x, y, plan), reference(x, y, a, b, scale, rank, at), t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,n,r,d_in,d_out", [(50, 3, 16, 4096, 1024), (300, 7, 64, 1000, 700), (9, 9, 8, 512, 10240),
                                              (1, 1, 128, 2050, 2050)])
def test_against_64_bits(T, n, r, d_in, d_out, dtype):
    """The products in at least 32 bits.  The error of a sum of d_in rounded products, taken as a random walk of half units, is
    sqrt(d_in) 2^-24 of its terms' 2-norm, which for terms of one size is that of the sum times 2^-24 sqrt(d_in); eight times
    that (a chain of adds that truncates is twice as bad, and so is a walk at four sigma) covers A x, and B v with r for d_in.
    With v kept in two parts of 8 bits each its own rounding is 2^-17, so 16-bit types get that too, and the stored half unit."""
    rng = np.random.default_rng(r)
    t = TYPES[dtype]
    f = lambda *s: torch.from_numpy(rng.standard_normal(s)).cuda()  # noqa: E731
    x, y = f(T, d_in).to(t), torch.zeros(T, d_out, device="cuda", dtype=t)
    a, b = (f(n, r, d_in) / d_in ** 0.5).to(t), (f(n, d_out, r) / r ** 0.5).to(t)
    at = rng.integers(0, n, size=T).astype(np.int32)
    adapters = Adapters(a, b, scale=0.75)
    got = adapters.apply(x, y, adapters.plan(torch.from_numpy(at).cuda())).double().cpu().numpy()
    want = reference(x, y, a, b, 0.75, None, at)
    eps = {"f32": 2.0 ** -24, "f16": 2.0 ** -11 + 2.0 ** -17, "bf16": 2.0 ** -8 + 2.0 ** -17}[dtype]
    tol = 8 * 2.0 ** -24 * (d_in ** 0.5 + r ** 0.5) + eps
    assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_apart_and_unaligned(dtype):
    rng = np.random.default_rng(4)
    t = TYPES[dtype]
    T, n, r, d_in, d_out = 90, 3, 16, 128, 256
    xs, ys = whole(rng, (T, d_in + 9), 2, t), whole(rng, (T, d_out + 9), 50, t)
    a, b = whole(rng, (n, r, d_in), 2, t), whole(rng, (n, d_out, r), 1, t)
    at = owners(rng, T, n, 5)
    adapters = Adapters(a, b)
    plan = adapters.plan(torch.from_numpy(at).cuda())
    for i, j in ((0, 0), (1, 0), (0, 3), (8, 8)):
        x, y = xs[:, i:i + d_in], ys[:, j:j + d_out]
        want = reference(x, y, a, b, 1, None, at)
        check_exact(adapters.apply(x, y, plan), want, t)
        outs = torch.full((T + 2, d_out + 5), 9.0, device="cuda", dtype=t)
        adapters.apply(x, y, plan, out=outs[:T, 2:2 + d_out])
        check_exact(outs[:T, 2:2 + d_out], want, t)
        assert (outs[T:] == 9).all() and (outs[:, :2] == 9).all() and (outs[:, 2 + d_out:] == 9).all()
        keep = ys.clone()
        adapters.apply(x, keep[:, j:j + d_out], plan, out=keep[:, j:j + d_out])
        check_exact(keep[:, j:j + d_out], want, t)
        assert torch.equal(keep[:, :j], ys[:, :j]) and torch.equal(keep[:, j + d_out:], ys[:, j + d_out:])


def test_weights_that_start_between_boundaries():
    rng = np.random.default_rng(6)
    n, r, d_in, d_out, T = 2, 8, 64, 72, 40
    fa, fb = whole(rng, (n * r * d_in + 1,), 2, torch.bfloat16), whole(rng, (n * r * d_out + 1,), 1, torch.bfloat16)
    a, b = fa[1:].view(n, r, d_in), fb[1:].view(n, d_out, r)
    x, y = whole(rng, (T, d_in), 2, torch.bfloat16), whole(rng, (T, d_out), 9, torch.bfloat16)
    at = owners(rng, T, n, 4)
    adapters = Adapters(a, b)
    check_exact(adapters.apply(x, y, adapters.plan(torch.from_numpy(at).cuda())), reference(x, y, a, b, 1, None, at),
                torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES)
def test_nobody_elses_numbers(dtype):
    """Rows of tokens without an adapter pass as they are, with what they hold; infinities and NaN stay in their own rows and in
    the adapters that nobody uses, and so does what lies past an adapter's rank."""
    rng = np.random.default_rng(9)
    t = TYPES[dtype]
    T, n, r, d_in, d_out = 80, 4, 16, 200, 136
    x, y = whole(rng, (T, d_in), 2, t), whole(rng, (T, d_out), 50, t)
    a, b = whole(rng, (n, r, d_in), 2, t), whole(rng, (n, d_out, r), 1, t)
    at = np.array([0, 1, -1, 3] * 20, np.int32)
    at[5] = -1
    rank = torch.tensor([16, 5, 16, 16], dtype=torch.int32, device="cuda")
    want = reference(x, y, a, b, 1, rank, at)
    a[2], b[2] = np.nan, np.inf                                     # nobody's adapter
    a[1, 5:], b[1, :, 5:] = np.nan, np.nan                          # past its rank
    x[2], x[6], x[10] = np.nan, np.inf, torch.finfo(t).max          # of tokens without an adapter
    y[2], y[6] = np.nan, -np.inf
    x[4, 3] = np.nan                                                # a token of adapter 0
    adapters = Adapters(a, b, rank=rank)
    got = adapters.apply(x, y, adapters.plan(torch.from_numpy(at).cuda()))
    rest = np.setdiff1d(np.arange(T), [2, 4, 6])
    check_exact(got[rest], want[rest], t)
    assert torch.isnan(got[2]).all() and (got[6] == -np.inf).all() and torch.isnan(got[4]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_large_and_small_inner_values(dtype):
    """A x far above and below what 16 bits hold, brought back by B and the scale."""
    rng = np.random.default_rng(12)
    t = TYPES[dtype]
    T, r, d_in, d_out = 33, 16, 512, 64
    for up, down in ((2.0 ** 7, 2.0 ** -12), (2.0 ** -10, 2.0 ** 8)):
        x, a = whole(rng, (T, d_in), 2, t) * up, whole(rng, (1, r, d_in), 2, t) * up
        b, y = whole(rng, (1, d_out, r), 1, t) * down, torch.zeros(T, d_out, device="cuda", dtype=t)
        at = np.zeros(T, np.int32)
        scale = torch.full((1,), up ** -2, device="cuda")
        adapters = Adapters(a, b, scale=scale)
        check_exact(adapters.apply(x, y, adapters.plan(torch.from_numpy(at).cuda())),
                    reference(x, y, a, b, scale, None, at), t)


def test_plans():
    rng = np.random.default_rng(2)
    x, y = whole(rng, (200, 64), 2, torch.float32), whole(rng, (200, 64), 9, torch.float32)
    a, b = whole(rng, (5, 8, 64), 2, torch.float32), whole(rng, (5, 64, 8), 1, torch.float32)
    adapters = Adapters(a, b)
    for at in (np.full(200, -1), np.full(200, 4), np.arange(200) % 5, np.arange(200) % 6 - 1):
        at = at.astype(np.int32)
        plan = AdapterPlan(torch.from_numpy(at).cuda(), 5)
        check_exact(adapters.apply(x, y, plan), reference(x, y, a, b, 1, None, at), torch.float32)
    empty = adapters.plan(torch.empty(0, dtype=torch.int32, device="cuda"))
    assert adapters.apply(x[:0], y[:0], empty).shape == (0, 64)
    with pytest.raises(ValueError):
        adapters.apply(x[:199], y[:199], plan)                      # another batch's plan
    with pytest.raises(ValueError):
        Adapters(a[:4].contiguous(), b[:4].contiguous()).apply(x, y, plan)
    with pytest.raises(ValueError):
        adapters.apply(x.double(), y, plan)
    with pytest.raises(ValueError):
        adapters.apply(x, y, plan, out=y[:199])
    with pytest.raises(ValueError):
        adapters.plan(torch.zeros(5, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        Adapters(a, b.half())
    with pytest.raises(ValueError):
        Adapters(a, b, scale=torch.ones(4, device="cuda"))


def test_same_bits_every_time():
    """No order that a run leaves open."""
    rng = np.random.default_rng(3)
    f = lambda *s: torch.from_numpy(rng.standard_normal(s)).cuda().to(torch.bfloat16)  # noqa: E731
    n, r, d_in, d_out, T = 4, 16, 1024, 1024, 300
    x, y, a, b = f(T, d_in), f(T, d_out), f(n, r, d_in), f(n, d_out, r)
    at = torch.from_numpy(owners(rng, T, n, 12)).cuda()
    adapters = Adapters(a, b)
    first = adapters.apply(x, y, adapters.plan(at))
    for _ in range(3):
        assert torch.equal(adapters.apply(x, y, adapters.plan(at)), first)


def test_layer_with_adapters_and_captured():
    from tests.test_gpu_topk import small_layer

    layer, _, xs = small_layer(4, 64, 128, variant="cpm_2", on_device=True)
    rng = np.random.default_rng(1)
    x = torch.from_numpy(xs).cuda()
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32) * 0.1).cuda()  # noqa: E731
    adapters = Adapters(f(3, 8, 64), f(3, 64, 8), scale=2.0)
    at = torch.from_numpy(owners(rng, 70, 3, 6)).cuda()
    plan = adapters.plan(at)
    plain = layer.forward(x)
    want = adapters.apply(x, plain, plan)
    got = layer.forward(x, adapters=adapters, plan=plan)
    assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = torch.empty_like(x)
    side.wait_stream(torch.cuda.current_stream())
    layer.forward(x, stream=side.cuda_stream, out=other, adapters=adapters, plan=plan)
    torch.cuda.synchronize()
    assert torch.equal(other, want)
    with pytest.raises(ValueError):
        layer.forward(x, adapters=adapters)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p = adapters.plan(at)
        out = layer.forward(x, adapters=adapters, plan=p)
    x.mul_(0.5)
    at.copy_(torch.from_numpy(owners(np.random.default_rng(5), 70, 3, 9)).cuda())
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, layer.forward(x, adapters=adapters, plan=adapters.plan(at)))
    del g
    layer.terminate()


# Many tokens to an adapter and wide ranks in 16 bits take the kernels on tiles of 128 rows: from 2048 tokens on (rank over 32) or 4096
# (over 16), 32 tokens to an adapter; both sides of these lines, tiles that end anywhere, rows of every alignment.
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,n,r,d_in,d_out,requests", [
    (2047, 1, 64, 64, 64, 1), (2048, 1, 64, 256, 512, 1), (2048, 64, 33, 136, 72, 64), (2048, 65, 33, 136, 72, 64),
    (2100, 3, 40, 130, 76, 9), (2500, 60, 100, 520, 264, 70), (4095, 2, 32, 64, 200, 5), (4096, 2, 32, 64, 200, 5),
    (4096, 2, 17, 72, 1000, 5), (4096, 2, 16, 72, 1000, 5), (4500, 7, 128, 1000, 130, 40), (2300, 2, 64, 63, 65, 5),
    (2049, 1, 128, 8, 4100, 2), (3000, 4, 65, 2056, 64, 2900)])
def test_whole_numbers_of_many_tokens(T, n, r, d_in, d_out, requests, dtype):
    test_whole_numbers(T, n, r, d_in, d_out, requests, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_many_tokens_rows_apart_and_unaligned(dtype):
    rng = np.random.default_rng(14)
    t = TYPES[dtype]
    T, n, r, d_in, d_out = 2200, 3, 48, 96, 160
    xs, ys = whole(rng, (T, d_in + 9), 2, t), whole(rng, (T, d_out + 9), 50, t)
    a, b = whole(rng, (n, r, d_in), 2, t), whole(rng, (n, d_out, r), 1, t)
    at = owners(rng, T, n, 20)
    adapters = Adapters(a, b)
    plan = adapters.plan(torch.from_numpy(at).cuda())
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for i, j in ((0, 0), (1, 0), (0, 3), (8, 8)):
        x, y = xs[:, i:i + d_in], ys[:, j:j + d_out]
        want = reference(x, y, a, b, 1, None, at)
        outs = torch.full((T + 2, d_out + 5), 9.0, device="cuda", dtype=t)
        adapters.apply(x, y, plan, out=outs[:T, 2:2 + d_out], status=status)
        check_exact(outs[:T, 2:2 + d_out], want, t)
        assert (outs[T:] == 9).all() and (outs[:, :2] == 9).all() and (outs[:, 2 + d_out:] == 9).all()
        keep = ys.clone()
        adapters.apply(x, keep[:, j:j + d_out], plan, out=keep[:, j:j + d_out])
        check_exact(keep[:, j:j + d_out], want, t)
        assert torch.equal(keep[:, :j], ys[:, :j]) and torch.equal(keep[:, j + d_out:], ys[:, j + d_out:])
    assert int(status) == 0


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_many_tokens_nobody_elses_numbers(dtype):
    """test_nobody_elses_numbers on tiles of 128 rows."""
    rng = np.random.default_rng(19)
    t = TYPES[dtype]
    T, n, r, d_in, d_out = 2400, 4, 64, 200, 136
    x, y = whole(rng, (T, d_in), 2, t), whole(rng, (T, d_out), 50, t)
    a, b = whole(rng, (n, r, d_in), 2, t), whole(rng, (n, d_out, r), 1, t)
    at = np.array([0, 1, -1, 3] * 600, np.int32)
    rank = torch.tensor([64, 21, 64, 37], dtype=torch.int32, device="cuda")
    want = reference(x, y, a, b, 1, rank, at)
    a[2], b[2] = np.nan, np.inf                                     # nobody's adapter
    a[1, 21:], b[1, :, 21:] = np.nan, np.nan                        # past its rank
    a[3, 37:], b[3, :, 37:] = np.inf, -np.inf
    x[2], x[6], x[10] = np.nan, np.inf, torch.finfo(t).max          # of tokens without an adapter
    y[2], y[6] = np.nan, -np.inf
    x[4, 3] = np.nan                                                # a token of adapter 0
    adapters = Adapters(a, b, rank=rank)
    got = adapters.apply(x, y, adapters.plan(torch.from_numpy(at).cuda()))
    rest = np.setdiff1d(np.arange(T), [2, 4, 6])
    check_exact(got[rest], want[rest], t)
    assert torch.isnan(got[2]).all() and (got[6] == -np.inf).all() and torch.isnan(got[4]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_many_tokens_against_64_bits(dtype):
    test_against_64_bits(2200, 3, 64, 1000, 300, dtype)
    test_against_64_bits(2200, 3, 128, 4096, 72, dtype)


def test_many_tokens_on_two_streams_with_one_plan():
    """A plan serves calls that run at once; each has its workspace."""
    rng = np.random.default_rng(23)
    t = torch.bfloat16
    T, n, r, d = 3000, 3, 64, 512
    at = owners(rng, T, n, 12)
    sets = [Adapters(whole(rng, (n, r, d), 2, t), whole(rng, (n, d, r), 1, t)) for _ in range(2)]
    xs, ys = [whole(rng, (T, d), 2, t) for _ in range(2)], [whole(rng, (T, d), 50, t) for _ in range(2)]
    plan = sets[0].plan(torch.from_numpy(at).cuda())
    want = [s.apply(x, y, plan).clone() for s, x, y in zip(sets, xs, ys)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(sets[i].apply(xs[i], ys[i], plan))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_many_tokens_captured_behind_a_layer():
    """The layer's last kernel, then the adapters' kernels, which start early, twice over in one graph."""
    from tests.test_gpu_topk import small_layer

    layer, _, _ = small_layer(4, 64, 128, on_device=True)
    rng = np.random.default_rng(29)
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32) * 0.1).cuda()  # noqa: E731
    x = f(2500, 64)
    sets = [Adapters(f(2, 40, 64).bfloat16(), f(2, 64, 40).bfloat16()) for _ in range(2)]
    at = torch.from_numpy(owners(rng, 2500, 2, 6)).cuda()

    def step():
        h, plan = layer.forward(x).bfloat16(), sets[0].plan(at)
        for s in sets:
            h = s.apply(h, h, plan)
        return h

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in (1, 2):
        x.copy_(torch.from_numpy(np.random.default_rng(seed).standard_normal((2500, 64)).astype(np.float32)))
        at.copy_(torch.from_numpy(owners(np.random.default_rng(seed), 2500, 2, 9)).cuda())
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())
    del g
    layer.terminate()


def test_rows_past_32_bits():
    """Elements of x, y and out beyond 2^32 of their tensors."""
    T, ld, d, r = (1 << 20) + 50, 4104, 64, 16
    t = torch.bfloat16
    rng = np.random.default_rng(31)
    x = torch.zeros(T, ld, dtype=t, device="cuda")                  # 8.6 GB
    x[-70:, :d] = whole(rng, (70, d), 2, t)
    y = torch.zeros(T, d, dtype=t, device="cuda")
    y[-70:] = whole(rng, (70, d), 50, t)
    a, b = whole(rng, (2, r, d), 2, t), whole(rng, (2, d, r), 1, t)
    at = np.full(T, -1, np.int32)
    at[-70:] = owners(rng, 70, 2, 7)
    adapters = Adapters(a, b)
    plan = adapters.plan(torch.from_numpy(at).cuda())
    got = adapters.apply(x[:, :d], y, plan)
    check_exact(got[-70:], reference(x[-70:, :d], y[-70:], a, b, 1, None, at[-70:]), t)
    assert not got[:-70].any()
    into = x[:, 2000:2000 + d]                                      # rows apart on the way out too
    adapters.apply(x[:, :d], y, plan, out=into)
    assert torch.equal(into, got)


@pytest.mark.parametrize("which", ["default", "side"])
def test_layer_with_adapters_on_a_given_stream(which):
    """The adapters run on the stream that the layer was given; 0 is the handle of the default one."""
    from tests.test_gpu_topk import small_layer

    layer, _, xs = small_layer(4, 64, 128, on_device=True)
    rng = np.random.default_rng(1)
    x = torch.from_numpy(xs).cuda()
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32) * 0.1).cuda()  # noqa: E731
    adapters = Adapters(f(3, 8, 64), f(3, 64, 8), scale=2.0)
    plan = adapters.plan(torch.from_numpy(owners(rng, 70, 3, 6)).cuda())
    want = adapters.apply(x, layer.forward(x), plan)
    stream = torch.cuda.default_stream() if which == "default" else torch.cuda.Stream()
    assert (stream.cuda_stream == 0) == (which == "default")
    seen = []

    class Recorded:
        def apply(self, *args, **kw):
            seen.append(torch.cuda.current_stream(x.device).cuda_stream)
            return adapters.apply(*args, **kw)

    torch.cuda.synchronize()
    for _ in range(3):
        out = torch.full_like(x, 7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(20_000_000)           # about 10 ms: adapters on another stream would not wait for the layer's pass
        got = layer.forward(x, stream=stream.cuda_stream, out=out, adapters=Recorded(), plan=plan)
        assert got is out
        stream.synchronize()
        assert torch.equal(out, want)
    assert seen == [stream.cuda_stream] * 3
    layer.terminate()


# FP32 products are made of two parts of 11 bits to each number.  Of a number u in [1, 2) the first part leaves at most 2^-11, in
# steps of 2^-23, and the second keeps 11 bits of that: at most 2^-23 of u is lost.  The product of the second parts, at most 2^-22, is
# left out.  So a product of two is off by (2 + 1 + 1) 2^-23, and by one more for a sum in 32 bits that is cut off and not rounded; A x
# and B v are one such product each where d_in and the rank are one.
FP32_PRODUCTS_TOL = 10 * 2.0 ** -23 * (1 + 2.0 ** -8)


def one_by_one(x, a, b, at):
    """Adapters with one product to A x and one to B v: what they give and what 64 bits do."""
    t = lambda v: torch.from_numpy(v.astype(np.float32)).cuda()  # noqa: E731
    adapters = Adapters(t(a).view(-1, 1, 1), t(b).unsqueeze(2))
    y = torch.zeros(len(x), b.shape[1], device="cuda")
    got = adapters.apply(t(x).view(-1, 1), y, adapters.plan(torch.from_numpy(at).cuda()))
    with np.errstate(invalid="ignore"):
        return got.double().cpu().numpy(), (x * a[at])[:, None] * b[at]


def test_fp32_products():
    """Numbers whose last 13 bits are as large as they can be are what a first part that is cut off serves worst."""
    rng = np.random.default_rng(17)
    f = lambda *s: 1 + rng.integers(0, 8, s) * 2.0 ** -10 + (2.0 ** 13 - 1 - rng.integers(0, 64, s)) * 2.0 ** -23  # noqa: E731
    at = rng.integers(0, 64, size=600).astype(np.int32)
    for x, a, b in ((f(600), f(64), f(64, 100)), (f(600), np.ones(64), f(64, 100)),
                    *((1 + (rng.integers(0, 1 << 23, s) * 2.0 ** -23) for s in (600, 64, (64, 100))) for _ in range(4))):
        sign = rng.choice([-1.0, 1.0], size=64)
        got, want = one_by_one(x, a * sign, b, at)
        off = (got - want) / want
        assert np.abs(off).max() <= FP32_PRODUCTS_TOL, np.abs(off).max() * 2 ** 23
        # cutting off after each product shrinks by up to two units of 2^-23 in the mean; nothing else has a side
        assert abs(off.mean()) <= 2 * 2.0 ** -23, off.mean() * 2 ** 23


def test_fp32_infinities_and_the_largest_numbers():
    """What the formula makes of them: an infinity stays one where the other factor is exact in few bits, and is NaN only where it
    meets a zero or its opposite."""
    big = np.float64(np.finfo(np.float32).max)
    x = np.array([np.inf, -np.inf, np.nan, big, -big, big * (1 - 2.0 ** -12), 1.0, 3.0, 0.0, 1 + 2.0 ** -23] * 4).astype(np.float32).astype(np.float64)
    a = np.array([1.0, 2.0 ** -20, -0.75, 2.0 ** -20 * (1 + 2.0 ** -12 + 2.0 ** -23)])
    b = np.array([[1.0, -2.0, 0.5, 1 / 3, 0.0, 2.0 ** -30]] * 4).astype(np.float32).astype(np.float64)
    at = np.repeat(np.arange(4), 10).astype(np.int32)
    got, want = one_by_one(x, a, b, at)
    some = np.abs(want) <= big
    beyond = ~some & ~np.isnan(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(got[beyond], np.sign(want[beyond]) * np.inf)
    assert (np.abs(got[some] - want[some]) <= FP32_PRODUCTS_TOL * np.abs(want[some])).all()
    # infinite weights
    got, want = one_by_one(np.array([1.0, -2.0, 0.0]), np.array([np.inf]), np.array([[1.0, -1.0]]), np.zeros(3, np.int32))
    assert (got[:2] == want[:2]).all() and np.isnan(got[2]).all()
    got, want = one_by_one(np.array([1.0, -2.0, 0.0]), np.array([1.0]), np.array([[np.inf, -np.inf, 4.0]]), np.zeros(3, np.int32))
    np.testing.assert_array_equal(got, np.where(np.isnan(want), np.nan, want))


@pytest.mark.parametrize("r", [3, 16, 24, 64, 128])
def test_fp32_rows_beside_infinities_keep_their_bits(r):
    """A row's result does not depend on what the other rows of its tile hold, nor on what lies in memory past the tile and the rank."""
    rng = np.random.default_rng(r)
    T, n, d_in, d_out = 61, 2, 300, 140
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    x, y, a, b = f(T, d_in), f(T, d_out), f(n, r, d_in), f(n, d_out, r)
    at = owners(rng, T, n, 4)
    adapters = Adapters(a, b)
    plan = adapters.plan(torch.from_numpy(at).cuda())
    want = adapters.apply(x, y, plan)
    odd = x.clone()
    odd[3::7, 5], odd[4::7, 200], odd[5::7, 299] = np.inf, torch.finfo(torch.float32).max, np.nan
    got = adapters.apply(odd, y, plan)
    same = np.array([t % 7 not in (3, 4, 5) or not 0 <= at[t] < n for t in range(T)])
    assert torch.equal(got[same], want[same]) and not torch.isfinite(got[5::7][(at[5::7] >= 0) & (at[5::7] < n)]).any()
    # an infinite column of one adapter's A x, B's row of one column of out
    a[0, r // 2, 7] = np.inf
    b[1, 100] = np.nan
    got = adapters.apply(x, y, plan)
    two = at == 1
    keep = np.arange(d_out) != 100
    assert torch.equal(got[two][:, keep], want[two][:, keep]) and torch.isnan(got[two][:, 100]).all()
    assert not torch.isfinite(got[at == 0]).any()


def test_weights_whose_data_was_replaced():
    """Parameters get other memory when a model is converted, moved or loaded anew: a call reads what they hold then."""
    rng = np.random.default_rng(41)
    n, r, d_in, d_out, T = 3, 8, 64, 72, 40
    new = lambda: (whole(rng, (n, r, d_in), 2, torch.float32), whole(rng, (n, d_out, r), 1, torch.float32),  # noqa: E731
                   torch.from_numpy(2.0 ** rng.integers(-3, 1, size=n).astype(np.float32)).cuda(),
                   torch.from_numpy(rng.integers(0, r + 1, size=n).astype(np.int32)).cuda())
    held = new()
    x, y = whole(rng, (T, d_in), 2, torch.float32), whole(rng, (T, d_out), 9, torch.float32)
    at = owners(rng, T, n, 4)
    adapters = Adapters(*held)
    plan = adapters.plan(torch.from_numpy(at).cuda())
    kept = [t.data for t in held]                                   # the first memory stays valid
    for _ in range(2):
        check_exact(adapters.apply(x, y, plan), reference(x, y, *held, at), torch.float32)
        for t, other in zip(held, new()):
            t.data = other
    assert [t.data_ptr() for t in held] != [t.data_ptr() for t in kept]
    for i, other in enumerate((held[0][:, :4].contiguous(), held[1].half(), held[2][:2].contiguous(), held[3].float())):
        good, held[i].data = held[i].data, other
        with pytest.raises(ValueError, match="must be a contiguous"):
            adapters.apply(x, y, plan)
        held[i].data = good


@pytest.mark.parametrize("dtype,T,n,r,d", [("f32", 1, 1, 16, 2048), ("f32", 600, 3, 128, 512), ("f32", 9000, 2, 40, 64), ("bf16", 64, 64, 16, 2048),
                                           ("bf16", 2048, 1, 64, 1024), ("f16", 4100, 3, 17, 512), ("bf16", 40000, 2, 64, 256)])
def test_workspace_of_the_size_asked_for(dtype, T, n, r, d):
    """A call writes nothing behind it, and its results are right with no byte more."""
    import ctypes

    from infmoe_b200 import capi
    rng = np.random.default_rng(T)
    t = TYPES[dtype]
    x, y, a, b = whole(rng, (T, d), 2, t), whole(rng, (T, d), 50, t), whole(rng, (n, r, d), 2, t), whole(rng, (n, d, r), 1, t)
    at = owners(rng, T, n, min(T, 9))
    plan = Adapters(a, b).plan(torch.from_numpy(at).cuda())
    code = {"f32": capi.DTYPE_F32, "f16": capi.DTYPE_F16, "bf16": capi.DTYPE_BF16}[dtype]
    held, need = capi.AdapterSet(n, r, d, d, code, a.data_ptr(), b.data_ptr(), None, None), ctypes.c_size_t()
    capi.check(capi.lib().infmoe_adapter_workspace_bytes(ctypes.byref(held), T, ctypes.byref(need)))
    ws = torch.full((need.value + (16 << 20),), 77, dtype=torch.uint8, device="cuda")
    out, status = torch.empty_like(y), torch.zeros(1, dtype=torch.int32, device="cuda")
    capi.check(capi.lib().infmoe_adapter_apply(ctypes.byref(held), T, x.data_ptr(), d, y.data_ptr(), d, out.data_ptr(), d,
                                               plan.buffer.data_ptr(), ws.data_ptr(), need.value, status.data_ptr(),
                                               torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert int(status) == 0 and (ws[need.value:] == 77).all()
    rows = np.unique(np.concatenate([np.arange(min(T, 300)), np.arange(max(0, T - 300), T)]))
    check_exact(out[rows], reference(x[rows], y[rows], a, b, 1, None, at[rows]), t)


def test_plan_given_up_while_another_stream_still_needs_it():
    """What a plan and a set allocate themselves stays theirs until the calls on other streams that read it are done."""
    rng = np.random.default_rng(43)
    n, r, d, T = 3, 8, 64, 500
    x, y, a, b = whole(rng, (T, d), 2, torch.float32), whole(rng, (T, d), 9, torch.float32), whole(rng, (n, r, d), 2, torch.float32), \
        whole(rng, (n, d, r), 1, torch.float32)
    at = owners(rng, T, n, 7)
    dat = torch.from_numpy(at).cuda()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            adapters = Adapters(a, b, scale=0.5)
            plan = adapters.plan(dat)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda._sleep(40_000_000)                               # about 20 ms
        got = adapters.apply(x, y, plan)
        size = plan.buffer.numel()
        del plan, adapters
        with torch.cuda.stream(side):                               # zeros: a plan of no rows, a scale of zero
            taken = [torch.zeros(size, dtype=torch.uint8, device="cuda"), torch.zeros(n, device="cuda")]
        side.synchronize()
        check_exact(got, reference(x, y, a, b, 0.5, None, at), torch.float32)
        del taken


def test_scale_is_there_when_the_set_is():
    """A number for a scale becomes a tensor on the device, of which other streams know nothing."""
    rng = np.random.default_rng(47)
    r, d, T = 8, 64, 64
    x, y = whole(rng, (T, d), 2, torch.float32), whole(rng, (T, d), 9, torch.float32)
    a, b = whole(rng, (3, r, d), 2, torch.float32), whole(rng, (3, d, r), 1, torch.float32)
    at = owners(rng, T, 3, 7)
    plan = AdapterPlan(torch.from_numpy(at).cuda(), 3)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for scale in (0.5, 0.25, 4.0):
        before = torch.full((3,), 3.0, device="cuda")
        torch.cuda.synchronize()
        del before                                                  # its memory is the next scale's
        torch.cuda._sleep(40_000_000)
        adapters = Adapters(a, b, scale=scale)
        with torch.cuda.stream(side):
            got = adapters.apply(x, y, plan)
        side.synchronize()
        check_exact(got, reference(x, y, a, b, scale, None, at), torch.float32)
        torch.cuda.synchronize()


def test_captured_with_a_plan_made_before():
    """The stream of a capture is another one than the plan's; a set may be made within it."""
    rng = np.random.default_rng(53)
    T, n, r, d = 90, 3, 8, 64
    x, y, a, b = whole(rng, (T, d), 2, torch.float32), whole(rng, (T, d), 9, torch.float32), whole(rng, (n, r, d), 2, torch.float32), \
        whole(rng, (n, d, r), 1, torch.float32)
    at = owners(rng, T, n, 5)
    first = Adapters(a, b, scale=0.5)
    plan = first.plan(torch.from_numpy(at).cuda())
    first.apply(x, y, plan)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        second = Adapters(a, b, scale=2.0)
        out = second.apply(x, first.apply(x, y, plan), plan)
    for _ in range(2):
        x.copy_(whole(rng, (T, d), 2, torch.float32))
        g.replay()
        torch.cuda.synchronize()
        check_exact(out, reference(x, y, a, b, 2.5, None, at), torch.float32)
    del g, first, second, plan
    assert torch.equal(torch.zeros(4096, device="cuda"), torch.zeros(4096, device="cuda"))   # the allocator's work goes on
