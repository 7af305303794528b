"""The global norm of many tensors and clipping to it (gncde_global_norm, gncde_clip_by_global_norm) against 64 bits.

Tolerances: squares and sums are held in 64 bits (errors below 2^-40 here), so the norm carries its rounding to fp32
(2^-24) and the scale one division and one product more (2^-23 and 2^-24 of the value), then the type's own half step."""
import math

import pytest
import torch

from gncde import _lib, engine, train

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def tensors(sizes, dtypes=(torch.float32,), seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=g, device="cuda") * scale).to(dtypes[i % len(dtypes)])
            for i, n in enumerate(sizes)]


def norm64(ts):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))


def check(ts, max_norm=1.0):
    n = norm64(ts)
    m = max((float(t.abs().max()) for t in ts if t.numel()), default=0.0)
    keep = [t.clone() for t in ts]
    st = engine.global_norm(ts).double()
    assert abs(float(st[0]) - n) <= 2 * U * n and float(st[1]) == m
    out, st2 = engine.clip_by_global_norm(ts, max_norm)
    assert torch.equal(st2.double(), st)
    for t, k, o in zip(ts, keep, out):
        assert torch.equal(t, k) and o.dtype == t.dtype and o.shape == t.shape
        if float(st[0]) < max_norm:
            assert torch.equal(o, t)
        else:
            w = t.double() * (max_norm / n)
            assert bool(((o.double() - w).abs() <= (6 * U + HALF[t.dtype] * (1 + 6 * U)) * w.abs() + TINY[t.dtype]).all())
    same, _ = engine.clip_by_global_norm(ts, max_norm, out=ts)
    for o, t in zip(out, ts):
        assert torch.equal(o, t)
    return out


@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float16,),
                                    (torch.float32, torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("sizes", [(1,), (1, 1, 1), (3, 1000, 17), (4096, 4095, 4097, 8191), (0, 5, 0), (0,),
                                   (100003, 1, 2_000_001), tuple(range(1, 300))])
def test_sizes_and_types(sizes, dtypes):
    check(tensors(sizes, dtypes))


def test_large_chunks_and_more_than_one_table():
    check(tensors([150_001] * 260 + [9_000_001], (torch.bfloat16, torch.float32)))


@pytest.mark.parametrize("max_norm", [1e-6, 0.5, 1e3, 1e6])
def test_clips_only_past_the_norm(max_norm):
    check(tensors((1000, 77), scale=0.1), max_norm)


def test_addresses_off_the_vector():
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        flat = tensors((60000,), (dt,))[0]
        cuts = [0, 1, 4, 7, 5000, 5003, 21001, 60000]
        check([flat[a:b] for a, b in zip(cuts, cuts[1:])])


def test_outputs_elsewhere_aligned():
    t = tensors((5001, 333), (torch.bfloat16,))
    buf = torch.zeros(6000, dtype=torch.bfloat16, device="cuda")
    out = [buf[1:5002], buf[5003:5336]]
    engine.clip_by_global_norm(t, 1.0, out=out)
    want, _ = engine.clip_by_global_norm(t, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert float(buf[0]) == 0 and float(buf[5002]) == 0 and bool((buf[5336:] == 0).all())


def test_shapes_and_strides():
    t = torch.randn(30, 50, device="cuda")
    a = engine.global_norm([t.t(), torch.randn((), device="cuda") * 0])
    assert abs(float(a[0]) - norm64([t])) <= 2 * U * norm64([t])
    out, _ = engine.clip_by_global_norm([t.t()], 1.0)
    assert out[0].shape == (50, 30) and out[0].is_contiguous()
    assert torch.equal(out[0], engine.clip_by_global_norm([t], 1.0)[0][0].t())
    with pytest.raises(_lib.GncdeError, match="contiguous"):
        engine.clip_by_global_norm([t.t()], 1.0, out=[t.t()])


def test_far_values():
    """Squares that fp32 could not hold, at both ends."""
    for scale in (1e30, 1e-30):
        ts = [torch.full((1000,), scale, device="cuda"), torch.full((24,), scale, device="cuda", dtype=torch.bfloat16)]
        n = norm64(ts)
        st = engine.global_norm(ts)
        assert abs(float(st[0]) - n) <= 2 * U * n
    big = [torch.full((4,), 3e38, device="cuda")]
    out, st = engine.clip_by_global_norm(big, 1.0)
    assert math.isinf(float(st[0])) and bool((out[0] == 0).all())


def test_nan_and_inf():
    for bad in (float("nan"), float("inf"), -float("inf")):
        ts = tensors((700, 5000, 3))
        ts[1][4321] = bad
        out, st = engine.clip_by_global_norm(ts, 1.0)
        if math.isnan(bad):
            assert math.isnan(float(st[0])) and math.isnan(float(st[1]))
            assert all(bool(torch.isnan(o).all()) for o in out)
        else:
            assert math.isinf(float(st[0])) and math.isinf(float(st[1]))
            assert math.isnan(float(out[1][4321]))
            out[1][4321] = 0
            assert all(bool((o == 0).all()) for o in out)


def test_zeros():
    out = check([torch.zeros(100, device="cuda"), torch.zeros(7, device="cuda", dtype=torch.bfloat16)])
    assert all(bool((o == 0).all()) for o in out)


def test_the_same_tensor_twice():
    t = tensors((500,))
    n = norm64(t + t)
    assert abs(float(engine.global_norm(t + t)[0]) - n) <= 2 * U * n
    with pytest.raises(_lib.GncdeError, match="share"):
        engine.clip_by_global_norm(t + t, 1.0, out=t + t)


def test_compiled_and_python_calls_agree(monkeypatch):
    class NotPlain:
        tensor_list = staticmethod(lambda *a: None)

    ts = tensors((700, 1, 90001), (torch.float32, torch.bfloat16, torch.float16))
    want = [engine.global_norm(ts)] + list(engine.clip_by_global_norm(ts, 0.7))
    monkeypatch.setattr(engine, "_fast", NotPlain)
    got = [engine.global_norm(ts)] + list(engine.clip_by_global_norm(ts, 0.7))
    assert torch.equal(want[0], got[0]) and torch.equal(want[2], got[2])
    assert all(torch.equal(a, b) for a, b in zip(want[1], got[1]))
    place = [t.clone() for t in ts]
    out, _ = engine.clip_by_global_norm(place, 0.7, out=place)
    assert out is not None and all(torch.equal(a, b) for a, b in zip(place, want[1]))
    with pytest.raises(_lib.GncdeError, match="share"):
        engine.clip_by_global_norm(ts + ts, 1.0, out=ts + ts)


def test_tuples_and_generators():
    ts = tensors((100, 200))
    want = engine.global_norm(ts)
    assert torch.equal(engine.global_norm(tuple(ts)), want) and torch.equal(engine.global_norm(t for t in ts), want)
    out, st = engine.clip_by_global_norm(tuple(ts), 1.0)
    assert torch.equal(st, want) and all(torch.equal(a, b) for a, b in zip(out, engine.clip_by_global_norm(ts, 1.0)[0]))


def test_streams_and_replays():
    ts = tensors((70001, 33, 5), (torch.float32, torch.bfloat16))
    want, st = engine.clip_by_global_norm(ts, 1.0)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for s in (s1, s2, s1):
        with torch.cuda.stream(s):
            got.append(engine.clip_by_global_norm(ts, 1.0))
    torch.cuda.synchronize()
    for o, a in got:
        assert torch.equal(a, st) and all(torch.equal(x, y) for x, y in zip(o, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, stats = engine.clip_by_global_norm(ts, 1.0)
    for k in range(3):
        for t in ts:
            t.copy_(torch.randn(t.shape, device="cuda").to(t.dtype) * (k + 1))
        g.replay()
        torch.cuda.synchronize()
        want, st = engine.clip_by_global_norm(ts, 1.0)
        assert torch.equal(stats, st) and all(torch.equal(x, y) for x, y in zip(out, want))


@pytest.mark.parametrize("kind", ["sgd", "adamw"])
def test_clipped_optimiser(kind):
    """One step equals clipping by hand and the optimiser's own step; parameters may be of mixed types."""
    def params():
        g = torch.Generator().manual_seed(3)
        return [torch.nn.Parameter(torch.randn(s, generator=g).to("cuda", dt)) for s, dt in
                (((20, 30), torch.float32), ((30,), torch.float32), ((8, 8), torch.bfloat16), ((1,), torch.float32))]
    make = {"sgd": lambda ps: torch.optim.SGD(ps, lr=0.1), "adamw": lambda ps: torch.optim.AdamW(ps, lr=0.1)}[kind]
    a, b = params(), params()
    opt, ref = train.ClippedOptimiser(make(a), 0.5), make(b)
    flat = torch.randn(20 * 30 + 30 + 64 + 1, device="cuda")
    stats = opt.step(flat.clone())
    off = 0
    for p in b:
        p.grad = flat[off:off + p.numel()].view_as(p).to(p.dtype)
        off += p.numel()
    before = [p.detach().clone() for p in b]
    engine.clip_by_global_norm([p.grad for p in b], 0.5, out=[p.grad for p in b])
    ref.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    assert float(stats[2]) == max(float((q.detach() - z).abs().max()) for q, z in zip(b, before))
    opt.zero_grad()
    assert all(p.grad is None for p in a) and bool((opt.flat_grad() == 0).all()) and bool((opt.clip() == 0).all())


def test_optimiser_without_clipping_and_refusals():
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    opt = train.ClippedOptimiser(torch.optim.SGD([p], lr=1.0), None)
    stats = opt.step(torch.full((4,), 2.0, device="cuda"))
    assert float(stats[0]) == 4.0 and float(stats[1]) == 2.0 and float(stats[2]) == 2.0 and bool((p == -1).all())
    with pytest.raises(ValueError, match="max_norm"):
        train.ClippedOptimiser(torch.optim.SGD([p], lr=1.0), 0.0)
    with pytest.raises(ValueError, match="GPU"):
        train.ClippedOptimiser(torch.optim.SGD([torch.nn.Parameter(torch.ones(2))], lr=1.0))
