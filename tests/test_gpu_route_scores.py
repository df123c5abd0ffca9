"""Context.route_scores / Layer.route_scores (osm_route_scores,
osm_moe_route_scores) against the definition in 64 bits.

The picks have to be equal.  Weights: a score in fp32 is an exponential (2 ulp)
of a rounded difference d (|d| half-ulps), a sum of at most E / 32 + 5 rounded
additions and a division; renormalised weights hold that twice.  So a weight
may be off by (|d| + E / 32 + 16) 2^-24 of itself, twice with renormalisation.
"""
import numpy as np
import pytest

from gpu_util import MoeFixture, require_cuda

pytestmark = pytest.mark.gpu

LOWEST = {"fp32": float(np.finfo(np.float32).min), "bf16": -3.3895313892515355e38, "fp16": -65504.0}


@pytest.fixture(scope="module")
def torch():
    return require_cuda()


@pytest.fixture(scope="module")
def ctx(torch):
    import osm_b200 as osm

    c = osm.Context(0, max_tokens=64)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    return c


def _dtype(torch, name):
    return {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[name]


def define(l, k, score="softmax", bias=None, groups=1, keep=1, pair=False, renorm=True, scale=1.0,
           lowest=LOWEST["fp32"]):
    """One row, straight from the definition: (ids, weights, mass)."""
    l = np.asarray(l, np.float64)
    E = len(l)
    if np.isnan(l).any() or (l == np.inf).any():
        return [0] * k, np.zeros(k), 0.0
    there = l > lowest
    if score == "softmax":
        e = np.where(there, np.exp(np.where(there, l, 0) - (l[there].max() if there.any() else 0)), 0.0)
        s = e / e.sum() if there.any() else e
    else:
        s = np.where(there, 1 / (1 + np.exp(-np.where(there, l, 0))), 0.0)
    c = s + (0 if bias is None else np.asarray(bias, np.float64))
    # without a bias the scores' order is the logits', also where 64 bits saturate
    key = [(c[e], l[e] if bias is None else 0.0) for e in range(E)]
    free = [e for e in range(E) if there[e]]
    if groups > 1:
        n = E // groups

        def value(g):
            best = sorted((e for e in range(g * n, g * n + n) if there[e]), key=lambda e: key[e], reverse=True)
            if not best:
                return (-np.inf, -np.inf)
            if pair:
                return (sum(c[e] for e in best[:2]), 0.0)
            return key[best[0]]

        order = sorted(range(groups), key=lambda g: (-value(g)[0], -value(g)[1], g))
        kept = set(order[:keep])
        free = [e for e in free if e // n in kept]
    picks = sorted(free, key=lambda e: (-key[e][0], -key[e][1], e))[:k]
    w = [s[e] for e in picks]
    picks += [e for e in range(E) if e not in set(picks)][:k - len(picks)]
    w = np.array(w + [0.0] * (k - len(w)))
    mass = w.sum()
    if renorm:
        w = w / mass if mass > 0 else w * 0
    return picks, w * scale, mass


def run(torch, ctx, logits, k, mass=True, **kw):
    import osm_b200 as osm

    T, E = logits.shape
    bias = kw.pop("bias", None)
    b = None if bias is None else torch.as_tensor(np.asarray(bias, np.float32)).cuda()
    r = osm.Routing(E, k, bias=b, score=kw.get("score", "softmax"), groups=kw.get("groups", 1),
                    top_groups=kw.get("keep", 1), group_score="top2" if kw.get("pair") else "max",
                    renormalize=kw.get("renorm", True), scale=kw.get("scale", 1.0))
    ids = torch.full((T + 2, k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((T + 2, k), -7.0, device="cuda")
    m = torch.full((T + 2,), -7.0, device="cuda") if mass else None
    ctx.route_scores(logits, r, ids, w, mass=m)
    torch.cuda.synchronize()
    assert (ids[T:] == -7).all() and (w[T:] == -7).all()  # rows behind the last one stay
    if mass:
        assert (m[T:] == -7).all()
    return ids[:T].cpu().numpy(), w[:T].cpu().numpy(), m[:T].cpu().numpy() if mass else None


def check(torch, ctx, logits, k, rows=None, **kw):
    name = {torch.float32: "fp32", torch.bfloat16: "bf16", torch.float16: "fp16"}[logits.dtype]
    ids, w, mass = run(torch, ctx, logits, k, **dict(kw))
    l = logits.float().cpu().numpy().astype(np.float64)
    E = l.shape[1]
    for t in range(l.shape[0]) if rows is None else rows:
        ri, rw, rm = define(l[t], k, lowest=LOWEST[name], **kw)
        assert ids[t].tolist() == list(ri), (t, ids[t], ri)
        fin = l[t][np.isfinite(l[t]) & (l[t] > LOWEST[name])]
        d = float(fin.max() - fin.min()) if fin.size else 0.0
        tol = (min(d, 104.0) + E / 32 + 16) * 2.0 ** -24 * (2 if kw.get("renorm", True) else 1)
        np.testing.assert_allclose(w[t], rw, rtol=tol, atol=1e-37)
        np.testing.assert_allclose(mass[t], rm, rtol=tol, atol=1e-37)


def _logits(torch, T, E, dtype, seed, pad=0, masked=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    l = (1.5 * torch.randn(T, E, device="cuda", generator=g)).to(_dtype(torch, dtype))
    if masked:
        l[:, torch.randperm(E, device="cuda", generator=g)[:masked]] = -float("inf")
    if pad:
        wide = torch.full((T, E + pad), float("nan"), device="cuda", dtype=l.dtype)
        wide[:, :E] = l
        l = wide[:, :E]
    return l


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,E,k,opt", [
    (1, 512, 10, {}),
    (5, 1, 1, {}),
    (3, 7, 7, dict(score="sigmoid")),
    (33, 33, 5, dict(renorm=False, scale=2.5)),
    (6, 1024, 32, {}),
    (6, 1023, 31, dict(score="sigmoid", bias=0.1)),
    (9, 64, 32, dict(bias=0.05)),
    (17, 256, 8, dict(score="sigmoid", bias=0.1, groups=8, keep=4, pair=True, scale=2.5)),
    (17, 160, 6, dict(groups=8, keep=3, renorm=False, scale=16.0)),
    (9, 60, 9, dict(groups=3, keep=1, pair=True, score="sigmoid")),
    (9, 60, 6, dict(groups=20, keep=2, pair=True, bias=0.1)),
    (9, 32, 3, dict(groups=32, keep=5, pair=True, bias=0.1, score="sigmoid")),
    (5, 1020, 12, dict(groups=17, keep=4, pair=True, bias=0.1)),
    (9, 96, 12, dict(groups=6, keep=6, pair=True)),
])
def test_matches_definition(torch, ctx, T, E, k, opt, dtype):
    opt = dict(opt)
    if "bias" in opt:
        opt["bias"] = opt["bias"] * np.random.RandomState(E).randn(E).astype(np.float32)
    ctx.status()
    check(torch, ctx, _logits(torch, T, E, dtype, 3 * E + T), k, **opt)
    assert ctx.status()[0] == 0


@pytest.mark.parametrize("pad", [1, 3, 8])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strided_rows_do_not_read_the_padding(torch, ctx, dtype, pad):
    check(torch, ctx, _logits(torch, 21, 256, dtype, 5, pad=pad), 8, score="sigmoid")
    # a first element that is not aligned to a vector
    l = _logits(torch, 7, 129, dtype, 6)[:, 1:]
    check(torch, ctx, l, 8)
    assert ctx.status()[0] == 0


@pytest.mark.parametrize("T", [129, 2000])
def test_many_rows(torch, ctx, T):
    b = 0.1 * np.random.RandomState(1).randn(256).astype(np.float32)
    check(torch, ctx, _logits(torch, T, 256, "bf16", 8), 8, score="sigmoid", bias=b, groups=8, keep=4, pair=True)
    check(torch, ctx, _logits(torch, T, 512, "fp32", 9), 10)


def test_ties_go_to_the_lower_index(torch, ctx):
    for E in (5, 64, 512, 1000):
        k = min(E, 32)
        for opt in ({}, dict(score="sigmoid"), dict(bias=np.full(E, 0.25, np.float32))):
            ids, w, _ = run(torch, ctx, torch.zeros(3, E, device="cuda"), k, **opt)
            assert (ids == np.arange(k)).all()
            np.testing.assert_allclose(w, 1 / k, rtol=1e-6)
    # a few equal logits in 16 bits, everywhere
    l = torch.randint(0, 4, (40, 256), device="cuda", generator=torch.Generator("cuda").manual_seed(2)).bfloat16()
    check(torch, ctx, l, 12)
    check(torch, ctx, l, 8, groups=8, keep=3, pair=True, score="sigmoid")
    check(torch, ctx, l, 8, groups=4, keep=2, bias=np.random.RandomState(0).choice([0, 0.5], 256).astype(np.float32))
    assert ctx.status()[0] == 0


def test_choices_that_32_bits_cannot_tell_apart(torch, ctx):
    """Each bias is 1 - score rounded to fp32: all choices are 1 within 2^-24,
    and their order is that of the 64-bit sums."""
    rs = np.random.RandomState(4)
    for E, k, opt in ((64, 8, {}), (256, 8, dict(groups=8, keep=3, pair=True)), (256, 16, dict(groups=8, keep=2)),
                      (512, 32, {}), (1024, 10, dict(groups=32, keep=7, pair=True))):
        l = (1.5 * rs.randn(E)).astype(np.float32)
        s = 1 / (1 + np.exp(-l.astype(np.float64)))
        bias = (1 - s).astype(np.float32)
        check(torch, ctx, torch.from_numpy(np.tile(l, (3, 1))).cuda(), k, score="sigmoid", bias=bias, **opt)
        s = np.exp(l.astype(np.float64) - l.max())
        s /= s.sum()
        bias = (s.max() - s).astype(np.float32)
        check(torch, ctx, torch.from_numpy(np.tile(l, (2, 1))).cuda(), k, bias=bias, **opt)


def test_masked_experts(torch, ctx):
    for dtype in ("fp32", "bf16", "fp16"):
        check(torch, ctx, _logits(torch, 9, 128, dtype, 11, masked=16), 8)
        check(torch, ctx, _logits(torch, 9, 128, dtype, 12, masked=100), 8, score="sigmoid", groups=8, keep=4,
              pair=True, bias=np.random.RandomState(3).randn(128).astype(np.float32))
        l = _logits(torch, 6, 64, dtype, 13)
        l[:, ::2] = LOWEST[dtype]  # the type's lowest value masks as -infinity does
        check(torch, ctx, l, 8, bias=np.linspace(1, 0, 64).astype(np.float32))
        # fewer experts than picks: the lowest-numbered others with weight 0
        l = _logits(torch, 4, 64, dtype, 14, masked=59)
        check(torch, ctx, l, 8)
        check(torch, ctx, l, 8, score="sigmoid", groups=4, keep=2, pair=True)
    assert ctx.status()[0] == 0


def test_rows_with_nothing_left(torch, ctx):
    l = _logits(torch, 6, 96, "fp32", 15)
    l[1] = -float("inf")
    l[4] = LOWEST["fp32"]
    for opt in ({}, dict(score="sigmoid", bias=np.ones(96, np.float32)), dict(groups=4, keep=2, pair=True)):
        ctx.status()
        check(torch, ctx, l, 5, **opt)
        assert ctx.status()[0] == 2  # zero mass
        ids, w, mass = run(torch, ctx, l, 5, **opt)
        assert ids[1].tolist() == [0, 1, 2, 3, 4] and (w[1] == 0).all() and mass[1] == 0
    ctx.status()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_non_finite_rows(torch, ctx, value):
    l = _logits(torch, 5, 200, "fp32", 16)
    l[2, 199] = value
    ctx.status()
    check(torch, ctx, l, 6, score="sigmoid")
    assert ctx.status()[0] == 1
    check(torch, ctx, l.half(), 6, groups=8, keep=2)
    assert ctx.status()[0] == 1


def test_extreme_logits(torch, ctx):
    l = torch.zeros(4, 64, device="cuda")
    l[0] = torch.linspace(-3e38, 3e38, 64)
    l[1] = torch.linspace(-120, -90, 64)   # sigmoids below fp32's range: the ratios still count
    l[2] = torch.linspace(30, 60, 64)      # sigmoids that round to 1
    l[3] = torch.linspace(-700, -600, 64)
    ctx.status()
    check(torch, ctx, l, 8, renorm=False)
    ids, w, mass = run(torch, ctx, l, 8, score="sigmoid")
    for t in range(4):
        ri, rw, _ = define(l[t].cpu().numpy(), 8, score="sigmoid")
        assert ids[t].tolist() == ri
        np.testing.assert_allclose(w[t], rw, rtol=1e-5)


def test_zero_scale_and_no_mass_output(torch, ctx):
    l = _logits(torch, 3, 40, "fp32", 17)
    ids, w, _ = run(torch, ctx, l, 4, mass=False, scale=0.0)
    assert (w == 0).all()
    assert ids[0].tolist() == define(l[0].cpu().numpy(), 4)[0]


def test_rows_far_apart(torch, ctx):
    """Row offsets past 2^31 elements."""
    stride, E = (1 << 30) + 8, 128
    buf = torch.empty(2 * stride + E, dtype=torch.bfloat16, device="cuda")
    l = buf.as_strided((3, E), (stride, 1))
    l.copy_(_logits(torch, 3, E, "bf16", 18))
    check(torch, ctx, l, 8)


def test_other_stream_and_graph(torch, ctx):
    import osm_b200 as osm

    l = _logits(torch, 50, 256, "fp32", 19)
    r = osm.Routing(256, 8, score="sigmoid", groups=8, top_groups=4, group_score="top2")
    ids = torch.zeros(50, 8, dtype=torch.int32, device="cuda")
    w = torch.zeros(50, 8, device="cuda")
    c = osm.Context(0, max_tokens=4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c.set_stream(s.cuda_stream)
    c.route_scores(l, r, ids, w)
    s.synchronize()
    want, ww = ids.clone(), w.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        c.route_scores(l, r, ids, w)
    other = _logits(torch, 50, 256, "fp32", 20)
    keep = l.clone()
    l.copy_(other)
    g.replay()
    torch.cuda.synchronize()
    assert not torch.equal(ids, want)
    l.copy_(keep)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(ids, want) and torch.equal(w, ww)


def test_refusals(torch, ctx):
    import osm_b200 as osm

    l = torch.zeros(2, 64, device="cuda")
    ids = torch.zeros(2, 8, dtype=torch.int32, device="cuda")
    w = torch.zeros(2, 8, device="cuda")
    bad = [dict(experts=64, top_k=0), dict(experts=64, top_k=33), dict(experts=64, top_k=8, groups=5),
           dict(experts=64, top_k=8, groups=0, top_groups=0), dict(experts=64, top_k=8, groups=8, top_groups=9),
           dict(experts=64, top_k=8, groups=8, top_groups=0), dict(experts=64, top_k=9, groups=8, top_groups=1),
           dict(experts=64, top_k=8, groups=64, top_groups=8), dict(experts=64, top_k=8, scale=float("nan"))]
    for b in bad:
        with pytest.raises((osm.OsmError, ValueError)):
            ctx.route_scores(l, osm.Routing(**b), ids, w)
    r = osm.Routing(64, 8)
    with pytest.raises(osm.OsmError):
        ctx.route_scores(l, r, ids, w, tokens=0)
    for args in ((l[:, :63], r, ids, w), (l.double(), r, ids, w), (l, r, ids.long(), w), (l, r, ids[:1], w),
                 (l.t(), r, ids, w), (l.cpu(), r, ids, w), (l, r, ids, w.half())):
        with pytest.raises(ValueError):
            ctx.route_scores(*args)
    lib = osm.lib()
    assert lib.osm_route_scores(ctx.h, r.ref, l.data_ptr(), 0, 63, 2, ids.data_ptr(), w.data_ptr(), None) == -1
    assert lib.osm_route_scores(ctx.h, r.ref, l.data_ptr() + 2, 0, 0, 1, ids.data_ptr(), w.data_ptr(), None) == -1
    assert lib.osm_route_scores(ctx.h, r.ref, l.data_ptr(), 3, 0, 2, ids.data_ptr(), w.data_ptr(), None) == -1
    assert lib.osm_route_scores(ctx.h, None, l.data_ptr(), 0, 0, 2, ids.data_ptr(), w.data_ptr(), None) == -1
    assert lib.osm_route_scores(ctx.h, r.ref, l.data_ptr(), 0, 0, 2, None, w.data_ptr(), None) == -1


@pytest.mark.parametrize("tokens", [1, 2, 7, 40])
def test_layer_routes_and_runs_its_experts(torch, port, tokens):
    """A grouped sigmoid router in front of the layer's experts: the picks are
    those of the reference's logits, and the sublayer's output is the picks'
    weighted experts (plus the shared expert), as the oracle computes it."""
    import osm_b200 as osm

    H, E, I, K = 512, 32, 256, 4
    f = MoeFixture(torch, H, E, I, K, seed=31, max_tokens=64)
    x = port.gen_normal(31, 8, 1.0, tokens * H).reshape(tokens, H)
    xd = torch.from_numpy(x).cuda()
    bias = 0.05 * torch.randn(E, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    r = osm.Routing(E, K, score="sigmoid", bias=bias, groups=4, top_groups=2, group_score="top2", scale=1.5)
    ids = torch.zeros(tokens, K, dtype=torch.int32, device="cuda")
    w = torch.zeros(tokens, K, device="cuda")
    mass = torch.zeros(tokens, device="cuda")
    f.layer.route_scores(xd, tokens, r, ids, w, mass=mass)
    logits = torch.zeros(tokens, E, device="cuda")
    f.layer.route_qwen_top_k_logits(xd, tokens, logits)
    out = torch.zeros(tokens, H, device="cuda")
    f.layer.run_experts(xd, tokens, ids, w, out)
    torch.cuda.synchronize()
    assert f.ctx.status()[0] == 0
    gi, gw, got = ids.cpu().numpy(), w.cpu().numpy(), out.cpu().numpy()
    shared = f.shared_f32()
    for t in range(tokens):
        l = logits[t].cpu().numpy()
        ri, rw, rm = define(l, K, score="sigmoid", bias=bias.cpu().numpy(), groups=4, keep=2, pair=True, scale=1.5)
        assert gi[t].tolist() == ri
        np.testing.assert_allclose(gw[t], rw, rtol=1e-5)
        np.testing.assert_allclose(mass[t].item(), rm, rtol=1e-5)
        ref = np.zeros(H, np.float64)
        ex = f.experts(ri)
        for e, we in zip(ri, rw):
            g, u, d = ex[e]
            ref += we * port.matvec(d, port.swiglu(port.matvec(g, x[t]), port.matvec(u, x[t])))
        g, u, d = shared
        gate = 1 / (1 + np.exp(-float(f.sg.astype(np.float64) @ x[t])))
        ref += gate * port.matvec(d, port.swiglu(port.matvec(g, x[t]), port.matvec(u, x[t])))
        assert np.abs(got[t] - ref).max() <= 1e-4 * np.abs(ref).max()


def test_layer_refusals_and_non_finite_rows(torch, port):
    import osm_b200 as osm

    f = MoeFixture(torch, 256, 32, 64, 4, seed=33)
    x = torch.randn(4, 256, device="cuda")
    ids = torch.zeros(4, 4, dtype=torch.int32, device="cuda")
    w = torch.zeros(4, 4, device="cuda")
    for r in (osm.Routing(16, 4), osm.Routing(32, 2)):
        with pytest.raises(osm.OsmError):
            f.layer.route_scores(x, 4, r, ids, w)
    with pytest.raises((osm.OsmError, ValueError)):
        f.layer.route_scores(x, 5, osm.Routing(32, 4), ids, w)
    x[1, 7] = float("nan")
    f.ctx.status()
    f.layer.route_scores(x, 4, osm.Routing(32, 4, score="sigmoid"), ids, w)
    assert f.ctx.status()[0] == 1
    assert (w[1] == 0).all() and (w[0] > 0).all()
