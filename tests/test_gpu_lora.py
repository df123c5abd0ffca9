"""Context.q4_gemv_lora (osm_q4_gemv_lora) against the definition in 64 bits.

Tolerance, per value y[t][o].  With c = bias + 8 scale of each group,
  S = sum_g sum_k (|scale| |q - 8| + |c|) |x_k|,  C = sum_g |c| sum_k |x_k|,
  L = |gain| sum_j |B_oj| sum_k |A_jk| |x_k|
the sum is taken as scale (q - 8) x + c (sum of x per group):
  half a step of y's type times |y| (one rounding at the end);
  every kind of row: operands to 2^-22 of themselves, a group's sum of x to
  10 half-ulps, steps of 16 products that each lose at most 2^-23 of the sum of
  magnitudes, twice over K / 16 steps and three times over K / 1024:
  (K / 8 + K / 256 + 16) 2^-23 (S + L), plus rank 2^-23 L;
  16-bit rows: c and the group sums once to fp16, the low-rank products to 16
  bits: 2^-11 C + 2^-15 L on top.
"""
import ctypes

import numpy as np
import pytest

from gpu_util import require_cuda

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return require_cuda()


@pytest.fixture(scope="module")
def ctx(torch):
    import osm_b200 as osm

    c = osm.Context(0, max_tokens=4)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    return c


class Case:
    def __init__(self, torch, T, K, N, rank=16, n=4, dtype="fp32", half=None, seed=0, ranks=False, xpad=0, ypad=0,
                 runs=None):
        g = torch.Generator(device="cuda").manual_seed(seed + 1000 * T + K + N)
        f = dict(device="cuda", generator=g)
        self.T, self.K, self.N, self.rank, self.n = T, K, N, rank, n
        dt = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
        half = {"bf16": torch.bfloat16, "fp16": torch.float16, None: torch.float16 if dtype == "fp16" else
                torch.bfloat16}[half]
        self.dt = dt
        self.packed = torch.randint(-2**31, 2**31, (N, K // 8), dtype=torch.int32, **f)
        sc = 0.008 * (0.5 + torch.rand(N, K // 64, **f))
        self.scales = sc.bfloat16()
        self.biases = (-7.5 * sc + 0.002 * torch.randn(N, K // 64, **f)).bfloat16()
        xw = torch.full((T, K + xpad), float("nan"), device="cuda", dtype=dt)
        xw[:, :K] = torch.randn(T, K, **f).to(dt)
        self.x = xw[:, :K]
        self.a = (torch.randn(n, rank, K, **f) / K ** 0.5).to(half)
        self.b = (0.1 * torch.randn(n, N, rank, **f)).to(half)
        self.gain = 0.5 + torch.rand(n, **f)
        self.ranks = torch.randint(0, rank + 1, (n,), dtype=torch.int32, **f) if ranks else None
        if runs is None:
            self.adapter = torch.randint(-1, n, (T,), dtype=torch.int32, **f)
        else:
            self.adapter = torch.repeat_interleave(torch.arange(T // runs + 1, device="cuda") % n, runs)[:T].int()
        self.yw = torch.full((T + 2, N + ypad), -7.0, device="cuda", dtype=dt)
        self.y = self.yw[:T, :N]

    def run(self, ctx, lora=True):
        import osm_b200 as osm

        table = osm.Lora(self.a, self.b, scale=self.gain, ranks=self.ranks) if lora else None
        ctx.q4_gemv_lora(self.packed, self.scales, self.biases, self.N, self.K, self.x, self.T, self.y, lora=table,
                         adapter=self.adapter if lora else None)
        return self.y

    def weight(self, torch):
        q = torch.stack([(self.packed.long() >> (4 * i)) & 15 for i in range(8)], 2).reshape(self.N, self.K).double()
        return (q * self.scales.double().repeat_interleave(64, 1)
                + self.biases.double().repeat_interleave(64, 1))

    def reference(self, torch, lora=True):
        """(y, (S, C), L) in 64 bits."""
        w, x = self.weight(torch), self.x.double()
        L = torch.zeros(self.T, self.N, dtype=torch.float64, device="cuda")
        c = (self.biases.double() + 8 * self.scales.double()).repeat_interleave(64, 1)
        y, C = x @ w.T, x.abs() @ c.abs().T
        S = x.abs() @ (w - c).abs().T + C
        for i in range(self.n if lora else 0):
            rows = (self.adapter == i).nonzero()[:, 0]
            r = self.rank if self.ranks is None else int(self.ranks[i].clamp(max=self.rank))
            a, b, g = self.a[i, :r].double(), self.b[i, :, :r].double(), float(self.gain[i])
            y[rows] += g * ((x[rows] @ a.T) @ b.T)
            L[rows] += abs(g) * ((x[rows].abs() @ a.abs().T) @ b.abs().T)
        return y, (S, C), L

    def tolerance(self, torch, y, SC, L):
        S, C = SC
        step = torch.finfo(self.dt).eps / 2
        tol = (step * y.abs() + (self.K / 8 + self.K / 256 + 16) * 2.0 ** -23 * (S + L) + self.rank * 2.0 ** -23 * L
               + 1e-30)
        if self.dt != torch.float32:
            tol = tol + 2.0 ** -11 * C + 2.0 ** -15 * L
        return tol

    def check(self, torch, ctx, lora=True):
        self.run(ctx, lora)
        torch.cuda.synchronize()
        y, S, L = self.reference(torch, lora)
        off = (self.y.double() - y).abs() / self.tolerance(torch, y, S, L)
        assert float(off.max()) <= 1.0, float(off.max())  # NaN fails too
        assert (self.yw[self.T:] == -7).all() and (self.yw[:, self.N:] == -7).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,K,N", [(1, 64, 1), (1, 2048, 512), (2, 512, 2048), (3, 128, 77), (8, 2048, 768),
                                   (15, 64, 130), (16, 256, 128), (17, 320, 129), (33, 2048, 512), (64, 768, 2048),
                                   (100, 1984, 333), (129, 512, 200), (257, 128, 640), (300, 2048, 128)])
def test_matches_definition(torch, ctx, T, K, N, dtype):
    ctx.status()
    Case(torch, T, K, N, dtype=dtype).check(torch, ctx)
    assert ctx.status()[0] == 0


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("half", ["bf16", "fp16"])
@pytest.mark.parametrize("T,rank", [(1, 1), (1, 128), (5, 7), (40, 16), (40, 33), (140, 64), (140, 128), (150, 3)])
def test_ranks_and_types(torch, ctx, T, rank, half, dtype):
    Case(torch, T, 256, 200, rank=rank, n=5, dtype=dtype, half=half, ranks=rank > 1, seed=rank).check(torch, ctx)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,K,N,rank,n", [(1, 4096, 24, 127, 2), (2, 2048, 300, 128, 3), (4, 2048, 40, 100, 3),
                                          (4, 4096, 64, 128, 2), (5, 64, 1, 1, 1), (20, 512, 64, 127, 3),
                                          (100, 2048, 48, 128, 5), (128, 1024, 640, 128, 4), (255, 704, 777, 20, 64),
                                          (256, 2048, 2048, 8, 9)])
def test_large_ranks_and_batches(torch, ctx, T, K, N, rank, n, dtype):
    Case(torch, T, K, N, rank=rank, n=n, dtype=dtype, seed=rank, ranks=rank == 20).check(torch, ctx)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T", [2, 20, 300])
def test_rows_near_the_largest_value(torch, ctx, T, dtype):
    """Sums of a group of x, or of (q - 8) x, that pass the range of fp32 while y does not."""
    c = Case(torch, T, 128, 64, dtype=dtype)
    c.scales, c.biases = c.scales * 2.0 ** -14, c.biases * 2.0 ** -14
    c.x.copy_(1e38 + 2e38 * torch.rand(T, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(T)))
    c.check(torch, ctx, lora=False)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T", [1, 12, 31, 200])
def test_without_adapters(torch, ctx, T, dtype):
    Case(torch, T, 512, 300, dtype=dtype).check(torch, ctx, lora=False)
    c = Case(torch, T, 512, 300, dtype=dtype)
    c.adapter.fill_(-1)  # a table, but no token uses it
    c.check(torch, ctx)


@pytest.mark.parametrize("T,n,runs", [(512, 40, None), (300, 300, None), (1000, 3, 125), (1024, 7, 200), (2100, 64, 33), (4100, 9, 700),
                                      (4111, 40, 17)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_many_tokens_and_adapters(torch, ctx, T, n, runs, dtype):
    Case(torch, T, 512, 384, n=n, rank=16, dtype=dtype, runs=runs).check(torch, ctx)


@pytest.mark.parametrize("xpad,ypad", [(1, 1), (3, 5), (8, 8), (0, 1), (2, 0)])
@pytest.mark.parametrize("dtype,T", [("fp32", 3), ("fp32", 70), ("bf16", 3), ("bf16", 70), ("fp16", 290)])
def test_strides(torch, ctx, T, dtype, xpad, ypad):
    Case(torch, T, 320, 136, dtype=dtype, xpad=xpad, ypad=ypad).check(torch, ctx)


@pytest.mark.parametrize("dtype,T", [("fp32", 2), ("bf16", 2), ("fp32", 66), ("bf16", 66)])
def test_unaligned_tables(torch, ctx, T, dtype):
    """Every table one element (one word) past a 16-byte boundary, adapters with gaps between them."""
    c = Case(torch, T, 256, 72, rank=5, dtype=dtype, ranks=True)
    for name in ("packed", "scales", "biases", "gain", "ranks", "adapter"):
        v = getattr(c, name)
        buf = torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")
        buf[1:] = v.reshape(-1)
        setattr(c, name, buf[1:].view(v.shape))
    for name in ("a", "b"):
        v = getattr(c, name)
        m = v[0].numel()
        buf = torch.full((1 + c.n * (m + 3),), float("nan"), dtype=v.dtype, device="cuda")
        w = buf[1:].as_strided(v.shape, (m + 3, v.shape[2], 1))
        w.copy_(v)
        setattr(c, name, w)
    x = torch.empty(T * 256 + 1, dtype=c.dt, device="cuda")[1:].view(T, 256)
    x.copy_(c.x)
    c.x = x
    c.check(torch, ctx)


@pytest.mark.parametrize("dtype,T", [("fp32", 4), ("bf16", 4), ("fp32", 90), ("bf16", 90), ("fp16", 260)])
def test_rows_and_adapters_do_not_meet(torch, ctx, T, dtype):
    """Non-finite values in one adapter or one token's row stay there."""
    c = Case(torch, T, 256, 160, n=4, dtype=dtype)
    c.adapter = (torch.arange(T, device="cuda") % 4).int()
    c.run(ctx)
    good = c.y.clone()
    c.a[2, 3, 5] = float("nan")
    c.b[1, 7, 2] = float("inf")
    c.b[1, 9, 0] = float("nan")
    c.x[0, 1] = float("nan")
    c.x[3, 9] = float("inf")
    c.run(ctx)
    torch.cuda.synchronize()
    ad = c.adapter
    clean = (ad != 2) & (ad != 1)
    clean[0] = clean[3] = False
    assert torch.equal(c.y[clean], good[clean])
    one = ad == 1
    cols = torch.ones(160, dtype=torch.bool, device="cuda")
    cols[7] = cols[9] = False
    assert torch.equal(c.y[one][:, cols], good[one][:, cols])
    assert not torch.isfinite(c.y[one][:, ~cols].float()).any()
    assert torch.isnan(c.y[(ad == 2)]).all()
    assert not torch.isfinite(c.y[0].float()).any() and not torch.isfinite(c.y[3].float()).any()


@pytest.mark.parametrize("T", [5, 80])
def test_rows_behind_an_adapters_rank_are_not_used(torch, ctx, T):
    c = Case(torch, T, 128, 96, rank=24, n=3, ranks=True, dtype="bf16")
    c.ranks.copy_(torch.tensor([0, 9, 24]))
    c.a[0] = c.b[0] = float("nan")
    c.a[1, 9:] = float("nan")
    c.b[1, :, 9:] = float("inf")
    c.check(torch, ctx)
    c.ranks[2] = 1000  # more than the table holds: all of them
    c.check(torch, ctx)


@pytest.mark.parametrize("T", [3, 70])
def test_index_past_the_table(torch, ctx, T):
    c = Case(torch, T, 128, 64, n=2)
    c.adapter[1] = -2**31
    ctx.status()
    c.check(torch, ctx)
    assert ctx.status()[0] == 0
    c.adapter[0] = 2
    c.adapter[2] = 2**31 - 1
    c.check(torch, ctx)  # the reference takes neither as an adapter
    assert ctx.status()[0] == 256


@pytest.mark.parametrize("T", [2, 60])
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_scales_of_every_size(torch, ctx, T, dtype):
    """Rows of x and of W from 1e-30 to 1e+30 (fp16 rows: what fp16 holds)."""
    c = Case(torch, T, 256, 64, dtype=dtype)
    row = torch.logspace(-15, 15, 64, device="cuda")[:, None]
    c.scales, c.biases = (c.scales.float() * row).bfloat16(), (c.biases.float() * row).bfloat16()
    c.b = (c.b.float() * row).to(c.b.dtype) if dtype == "fp32" else torch.zeros_like(c.b)
    if dtype == "fp32":
        c.x.mul_(torch.logspace(-12, 12, T, device="cuda")[:, None])
        c.x[:, ::7] *= 1e-4
        c.check(torch, ctx)
    else:
        c.x.mul_(1e-3)
        c.y.zero_()
        c.run(ctx)
        torch.cuda.synchronize()
        y, S, L = c.reference(torch)
        fits = (y.abs() < 6e4) & (y.abs() > 1e-3)
        off = (c.y.double() - y).abs() / c.tolerance(torch, y, S, L)
        assert float(off[fits].max()) <= 1.0
    # zero rows give zeros
    c.x.zero_()
    c.run(ctx)
    torch.cuda.synchronize()
    assert (c.y == 0).all()


def test_rows_far_apart(torch, ctx):
    """Row offsets of x and y past 2^31 elements."""
    c = Case(torch, 3, 128, 64, dtype="bf16")
    stride = (1 << 30) + 8
    x = torch.empty(2 * stride + 128, dtype=torch.bfloat16, device="cuda").as_strided((3, 128), (stride, 1))
    x.copy_(c.x)
    y = torch.empty(2 * stride + 64, dtype=torch.bfloat16, device="cuda").as_strided((3, 64), (stride, 1))
    want = c.run(ctx).clone()
    c.x, c.y = x, y
    c.run(ctx)
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_streams_growth_and_graphs(torch):
    """Calls on two streams, a workspace that grows between them, and two
    graphs replayed at the same time on two streams."""
    import osm_b200 as osm

    c = osm.Context(0, max_tokens=4)
    cases = [Case(torch, T, 512, 256, dtype=d, seed=i) for i, (T, d) in
             enumerate([(3, "fp32"), (200, "fp32"), (90, "bf16"), (700, "fp32")])]
    torch.cuda.synchronize()
    c.set_stream(0)
    want = []
    for k in cases:
        want.append(k.run(c).clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in cases:
        k.yw.fill_(-7)
    torch.cuda.synchronize()
    for _ in range(5):
        for i, k in enumerate(cases):
            c.set_stream(streams[i % 2].cuda_stream)
            k.run(c)
    torch.cuda.synchronize()
    for k, w in zip(cases, want):
        assert torch.equal(k.y, w)
    graphs = []
    for pair in ((0, 3), (1, 2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.set_stream(torch.cuda.current_stream().cuda_stream)
            for i in pair:
                cases[i].run(c)
        graphs.append(g)
    for k in cases:
        k.yw.fill_(-7)
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for k, w in zip(cases, want):
        assert torch.equal(k.y, w)
    # other inputs in the same buffers
    cases[1].x.mul_(0.5)
    cases[1].adapter.copy_(cases[1].adapter.flip(0))
    graphs[1].replay()
    torch.cuda.synchronize()
    y, S, L = cases[1].reference(torch)
    assert float(((cases[1].y.double() - y).abs() / cases[1].tolerance(torch, y, S, L)).max()) <= 1
    del graphs
    c.close()


def test_same_inputs_same_bits(torch, ctx):
    for T in (1, 40, 600):
        c = Case(torch, T, 1024, 512, n=9)
        first = c.run(ctx).clone()
        for _ in range(3):
            c.yw.fill_(-7)
            assert torch.equal(c.run(ctx), first)


def test_refusals(torch, ctx):
    import osm_b200 as osm
    from osm_b200 import _lib

    c = Case(torch, 2, 128, 64)
    t = osm.Lora(c.a, c.b)

    def call(**kw):
        v = dict(packed=c.packed, s=c.scales, b=c.biases, N=64, K=128, x=c.x, T=2, y=c.y, lora=t, adapter=c.adapter)
        v.update(kw)
        ctx.q4_gemv_lora(v["packed"], v["s"], v["b"], v["N"], v["K"], v["x"], v["T"], v["y"], lora=v["lora"],
                         adapter=v["adapter"])

    call()
    for kw in (dict(T=0), dict(lora=None)):
        with pytest.raises(osm.OsmError):
            call(**kw)
    for kw in (dict(T=3), dict(x=c.x.double()), dict(x=c.x.bfloat16()), dict(x=c.x.t()), dict(x=c.x.cpu()),
               dict(adapter=c.adapter.long()), dict(adapter=None), dict(N=32), dict(K=64), dict(adapter=c.adapter[:1])):
        with pytest.raises(ValueError):
            call(**kw)
    for a, b in ((c.a.float(), c.b.float()), (c.a, c.b.half()), (c.a, c.b[:, :, :8]), (c.a.cpu(), c.b.cpu()),
                 (c.a.transpose(1, 2), c.b)):
        with pytest.raises(ValueError):
            osm.Lora(a, b)
    lib = osm.lib()

    def raw(N=64, K=128, group=64, x=c.x.data_ptr(), ty=0, xs=0, T=2, lora=t.ref, ad=c.adapter.data_ptr(),
            y=c.y.data_ptr(), ys=0):
        return lib.osm_q4_gemv_lora(ctx.h, c.packed.data_ptr(), c.scales.data_ptr(), c.biases.data_ptr(), N, K, group,
                                    x, ty, xs, T, lora, ad, y, ys)

    assert raw() == 0
    torch.cuda.synchronize()
    for kw in (dict(group=32), dict(K=96), dict(K=0), dict(N=0), dict(ty=3), dict(xs=127), dict(ys=63), dict(x=None),
               dict(y=None), dict(ad=None), dict(x=c.x.data_ptr() + 2), dict(y=c.x.data_ptr()),
               dict(y=c.x.data_ptr() + 128 * 4 + 64), dict(ad=c.adapter.data_ptr() + 1), dict(T=1 << 25)):
        assert raw(**kw) == -1, kw
    for field, value in (("rank", 0), ("rank", 129), ("count", 0), ("type", 0), ("a_dev", None), ("a_stride", 5),
                         ("b_dev", t.desc.b_dev + 1)):
        d = _lib.LoraDesc.from_buffer_copy(t.desc)
        setattr(d, field, value)
        assert raw(lora=ctypes.byref(d)) == -1, field
    assert lib.osm_q4_gemv_lora(None, None, None, None, 1, 64, 64, None, 0, 0, 1, None, None, None, 0) == -1


def test_shared_expert_with_adapters(torch):
    """The shared expert of a sublayer with an adapter on each of its three
    projections, beside a grouped router and the layer's routed experts."""
    import osm_b200 as osm

    H, I, T = 512, 256, 20
    c = osm.Context(0, max_tokens=32)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    gate, up = Case(torch, T, H, I, seed=1), Case(torch, T, H, I, seed=2)
    down = Case(torch, T, I, H, seed=3)
    up.x, up.adapter, down.adapter = gate.x, gate.adapter, gate.adapter
    g, u = gate.run(c), up.run(c)
    h = torch.empty(T, I, device="cuda")
    c.swiglu(g.contiguous(), u.contiguous(), h)
    down.x = h
    y = down.run(c)
    torch.cuda.synchronize()
    rg, ru = gate.reference(torch)[0], up.reference(torch)[0]
    down.x = rg / (1 + torch.exp(-rg)) * ru
    ref = down.reference(torch)[0]
    assert float((y.double() - ref).abs().max()) <= 1e-4 * float(ref.abs().max())
