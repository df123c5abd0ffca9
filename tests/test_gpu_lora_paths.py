"""Context.q4_gemv_lora on its prompt path (more than 256 tokens, or more than
1e9 products), where operands are prepared and the adapters are further steps
of one sum: row types unlike the adapters', ranks that fill no whole piece,
ranges of a tile's tokens and of a CTA's share of K.

Cases, the definition in 64 bits and the tolerance of fp32 rows are those of
test_gpu_lora."""
import pytest

from test_gpu_lora import Case, ctx, torch  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def tolerance(torch, c, y, S, L):  # noqa: F811
    """That of test_gpu_lora without its term 2^-11 C for 16-bit rows.

    Per group: c = bias + 8 scale is hi + lo of fp16, within 2^-24 of itself; the
    sum of x is taken in fp32 (10 half-ulps, 2^-24 each, of the sum of magnitudes)
    and held as hi + lo, 2^-24; the product of the two lo parts is left out, 2^-24:
    under 16 2^-23 C together.  Steps of 16: K / 16 of the products, 3 K / 1024 of
    the biases' columns, rounded up to a stage of 4: under K / 8 + K / 256 + 4, each
    with a loss of 2^-23 of the sum of magnitudes at most.  v is held in 16 bits for
    16-bit rows, 2^-15 L as there; y of fp16 is rounded to a multiple of 2^-24 at
    the least."""
    S = S[0]
    tol = (torch.finfo(c.dt).eps / 2 * y.abs() + (c.K / 8 + c.K / 256 + 20) * 2.0 ** -23 * (S + L)
           + c.rank * 2.0 ** -23 * L + 1e-30)
    if c.dt != torch.float32:
        tol = tol + 2.0 ** -15 * L
    if c.dt == torch.float16:
        tol = tol + 2.0 ** -25
    return tol


def check(torch, ctx, c, lora=True):  # noqa: F811
    c.run(ctx, lora)
    torch.cuda.synchronize()
    y, S, L = c.reference(torch, lora)
    off = (c.y.double() - y).abs() / tolerance(torch, c, y, S, L)
    assert float(off.max()) <= 1.0, float(off.max())  # NaN fails too
    assert (c.yw[c.T:] == -7).all() and (c.yw[:, c.N:] == -7).all()


# Tiles of 96 to 128 fp32 tokens take the three planes of v in two passes, and
# fp16 adapters their low part in further ones; a CTA's share of K is 17, 17, 13
# and 9 stages here, so that the last of these passes would open a partial sum.
@pytest.mark.parametrize("T,K,N", [(512, 2048, 2048), (1000, 2048, 768), (4096, 704, 2048), (2000, 448, 2048)])
@pytest.mark.parametrize("rank,n", [(16, 4), (40, 7)])
def test_fp32_rows_with_fp16_adapters(torch, ctx, T, K, N, rank, n):  # noqa: F811
    Case(torch, T, K, N, rank=rank, n=n, dtype="fp32", half="fp16").check(torch, ctx)


def one_sided(torch, T, K, N, dtype, kind, seed=0):
    """Weights whose part scale (q - 8) and whose part bias + 8 scale nearly
    cancel (codes mostly 0 without a bias, or mostly 15 with -15 scale), and rows
    of x with a mean, so that y is small beside the two."""
    c = Case(torch, T, K, N, dtype=dtype, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + T)
    f = dict(device="cuda", generator=g)
    if kind != "middle":
        few = torch.rand(N, K, **f) < 0.02
        q = torch.where(few, torch.randint(0, 16, (N, K), **f), 0 if kind == "low" else 15)
        word = torch.zeros(N, K // 8, dtype=torch.int64, device="cuda")
        for i in range(8):
            word |= q[:, i::8] << (4 * i)
        c.packed = torch.where(word >= 2**31, word - 2**32, word).int()
        c.biases = (0.0 if kind == "low" else -15.0) * c.scales
    c.x.copy_(1 + 0.25 * torch.randn(T, K, **f))
    return c


@pytest.mark.parametrize("kind", ["low", "high", "middle"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,K,N", [(3, 512, 96), (40, 512, 96), (300, 512, 96), (300, 1408, 2048), (1100, 64, 200),
                                   (4200, 2048, 130)])
def test_parts_that_cancel(torch, ctx, T, K, N, dtype, kind):  # noqa: F811
    """No operand of the two parts has fewer than 22 bits, whatever the rows' type."""
    c = one_sided(torch, T, K, N, dtype, kind, seed=K)
    check(torch, ctx, c)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_workspace_is_bounded(torch, dtype):  # noqa: F811
    """Rounds of launches hold the workspace at 256 MB beside what the weights
    take, also where v (rank 128) is more than x (64 values).  Rows on both sides
    of a round's end are right."""
    import osm_b200 as osm

    T, N = 700_001, 8
    case = Case(torch, T, 64, N, rank=128, n=3, dtype=dtype)
    ctx = osm.Context(0, max_tokens=4)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    small = Case(torch, 300, 64, N, rank=128, n=3, dtype=dtype)
    small.run(ctx)   # what the first call sets up
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    case.run(ctx)
    torch.cuda.synchronize()
    assert free - torch.cuda.mem_get_info()[0] <= (256 + 32) << 20
    check(torch, ctx, case)
    ctx.close()


def test_streams_that_come_and_go(torch):  # noqa: F811
    """Streams destroyed right behind their calls, whose handles the next ones may
    have again: each call has its own workspace while it runs, and what the calls
    of 60 streams take is not more than those in flight need."""
    import ctypes

    import osm_b200 as osm

    rt = torch.cuda.cudart()
    ctx = osm.Context(0, max_tokens=4)
    cases = [Case(torch, T, K, 512, n=n, rank=r, dtype=d, seed=i) for i, (T, K, n, r, d) in
             enumerate([(1500, 1024, 9, 24, "fp32"), (90, 512, 40, 16, "bf16"), (700, 2048, 5, 64, "fp16"),
                        (3, 4096, 3, 100, "fp32")])]
    want = []
    ctx.set_stream(0)
    for c in cases:
        want.append(c.run(ctx).clone())
    torch.cuda.synchronize()

    def generation():
        for c in cases:
            c.yw.fill_(-7)
        torch.cuda.synchronize()
        for c in cases:
            s = ctypes.c_void_p()
            assert int(rt.cudaStreamCreate(ctypes.addressof(s))) == 0
            ctx.set_stream(s.value)
            for _ in range(3):
                c.run(ctx)
            assert int(rt.cudaStreamDestroy(s.value)) == 0
        torch.cuda.synchronize()
        for c, w in zip(cases, want):
            assert torch.equal(c.y, w)

    for _ in range(5):
        generation()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(10):
        generation()
    assert free - torch.cuda.mem_get_info()[0] <= 64 << 20
    ctx.set_stream(0)
    ctx.close()


# Shares of K of 1 to 16 stages in all remainders of 4 (a partial sum of fp32
# rows), on 1, 2, 4 and 8 CTAs a tile, tiles of 16 to 240 tokens whose last one
# holds 12 to 172; below and above 4096 tokens, where another kernel computes v.
SIZES = [(300, 64, 72, 7, 3), (300, 192, 72, 33, 3), (300, 256, 136, 128, 4), (300, 832, 300, 65, 5),
         (300, 2048, 72, 1, 3), (1100, 320, 200, 33, 6), (1100, 1088, 640, 7, 4), (1100, 2112, 72, 128, 3),
         (1100, 128, 1500, 65, 9), (4200, 192, 136, 128, 6), (4200, 448, 72, 7, 40), (4200, 64, 130, 65, 3),
         (4200, 704, 1024, 33, 5), (700, 896, 2048, 16, 3), (2500, 704, 1500, 24, 7)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("half", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,N,rank,n", SIZES)
def test_ranks_and_types(torch, ctx, T, K, N, rank, n, half, dtype):  # noqa: F811
    """Every type of row beside every type of adapter, ranks that end inside a
    piece of 16 and inside the pieces of one pass over A, adapters of rank 0."""
    ctx.status()
    check(torch, ctx, Case(torch, T, K, N, rank=rank, n=n, dtype=dtype, half=half, ranks=rank > 1, seed=rank))
    assert ctx.status()[0] == 0


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,K,N", [(300, 512, 200), (1100, 192, 130), (4200, 448, 136)])
def test_without_adapters(torch, ctx, T, K, N, dtype):  # noqa: F811
    check(torch, ctx, Case(torch, T, K, N, dtype=dtype), lora=False)
    c = Case(torch, T, K, N, dtype=dtype)
    c.adapter.fill_(-1)  # a table, but no token uses it
    check(torch, ctx, c)


@pytest.mark.parametrize("what", ["tables", "adapters", "x"])
@pytest.mark.parametrize("dtype,half", [("fp32", "bf16"), ("fp32", "fp16"), ("bf16", "bf16"), ("bf16", "fp16"),
                                        ("fp16", "fp16")])
@pytest.mark.parametrize("T", [300, 1100, 4200])
def test_unaligned(torch, ctx, T, dtype, half, what):  # noqa: F811
    """One element (one word) past a 16-byte boundary: W's tables and the lists, A
    and B with gaps between adapters, or the rows of x, with NaN in the gaps."""
    c = Case(torch, T, 320, 136, rank=21, n=5, dtype=dtype, half=half, ranks=True)
    if what == "tables":
        for name in ("packed", "scales", "biases", "gain", "ranks", "adapter"):
            v = getattr(c, name)
            buf = torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")
            buf[1:] = v.reshape(-1)
            setattr(c, name, buf[1:].view(v.shape))
    elif what == "adapters":
        for name in ("a", "b"):
            v = getattr(c, name)
            m = v[0].numel()
            buf = torch.full((1 + c.n * (m + 3),), float("nan"), dtype=v.dtype, device="cuda")
            w = buf[1:].as_strided(v.shape, (m + 3, v.shape[2], 1))
            w.copy_(v)
            setattr(c, name, w)
    else:
        buf = torch.full((1 + T * 323,), float("nan"), dtype=c.dt, device="cuda")
        x = buf[1:].as_strided((T, 320), (323, 1))
        x.copy_(c.x)
        c.x = x
    check(torch, ctx, c)


@pytest.mark.parametrize("xpad,ypad", [(1, 1), (8, 8), (0, 1), (3, 0)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T", [300, 4200])
def test_strides(torch, ctx, T, dtype, xpad, ypad):  # noqa: F811
    check(torch, ctx, Case(torch, T, 320, 136, dtype=dtype, xpad=xpad, ypad=ypad))


@pytest.mark.parametrize("half", ["bf16", "fp16"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T", [1100, 4200])
def test_rows_and_adapters_do_not_meet(torch, ctx, T, dtype, half):  # noqa: F811
    """Non-finite values in one adapter or one token's row stay there."""
    c = Case(torch, T, 256, 160, n=4, rank=20, dtype=dtype, half=half)
    c.adapter = (torch.arange(T, device="cuda") % 4).int()
    c.run(ctx)
    good = c.y.clone()
    c.a[2, 17, 5] = float("nan")
    c.b[1, 7, 2] = float("inf")
    c.b[1, 9, 19] = float("nan")
    c.x[0, 1] = float("nan")
    c.x[T - 1, 9] = float("inf")
    c.run(ctx)
    torch.cuda.synchronize()
    ad = c.adapter
    clean = (ad != 2) & (ad != 1)
    clean[0] = clean[T - 1] = False
    assert torch.equal(c.y[clean], good[clean])
    one = ad == 1
    one[T - 1] = False
    cols = torch.ones(160, dtype=torch.bool, device="cuda")
    cols[7] = cols[9] = False
    assert torch.equal(c.y[one][:, cols], good[one][:, cols])
    assert not torch.isfinite(c.y[one][:, ~cols].float()).any()
    assert torch.isnan(c.y[(ad == 2)]).all()
    assert not torch.isfinite(c.y[0].float()).any() and not torch.isfinite(c.y[T - 1].float()).any()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T", [300, 4200])
def test_rows_behind_an_adapters_rank_are_not_used(torch, ctx, T, dtype):  # noqa: F811
    c = Case(torch, T, 128, 96, rank=72, n=4, ranks=True, dtype=dtype)
    c.ranks.copy_(torch.tensor([0, 9, 72, 33]))
    c.a[0] = c.b[0] = float("nan")
    c.a[1, 9:], c.a[3, 33:] = float("nan"), float("inf")
    c.b[1, :, 9:], c.b[3, :, 33:] = float("inf"), float("nan")
    check(torch, ctx, c)


@pytest.mark.parametrize("T", [300, 4200])
def test_index_past_the_table(torch, ctx, T):  # noqa: F811
    c = Case(torch, T, 128, 64, n=2)
    c.adapter[1] = -2**31
    ctx.status()
    check(torch, ctx, c)
    assert ctx.status()[0] == 0
    c.adapter[0] = 2
    c.adapter[T - 1] = 2**31 - 1
    check(torch, ctx, c)  # the reference takes neither as an adapter
    assert ctx.status()[0] == 256


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T", [300, 1100, 4200])
def test_scales_of_every_size(torch, ctx, T, dtype):  # noqa: F811
    """Rows of x and of W from 1e-27 to 1e+27, zero rows among them."""
    c = Case(torch, T, 256, 64, dtype=dtype)
    row = torch.logspace(-15, 15, 64, device="cuda")[:, None]
    c.scales, c.biases = (c.scales.float() * row).bfloat16(), (c.biases.float() * row).bfloat16()
    c.b = (c.b.float() * row).to(c.b.dtype)
    c.x.mul_(torch.logspace(-12, 12, T, device="cuda")[:, None].to(c.dt))
    c.x[:, ::7] *= 1e-4
    c.x[::5] = 0
    check(torch, ctx, c)
    assert (c.y[::5] == 0).all()


@pytest.mark.parametrize("T", [300, 1100])
def test_sublayer_of_many_requests(torch, T):  # noqa: F811
    """A sublayer as a server of many requests runs it: a grouped sigmoid router
    with a balance bias in front of the layer's routed experts, and beside them a
    dense branch of three Q4 projections with an adapter per request (gate, up,
    SwiGLU, down), whose output is the experts' residual; everything captured into
    one graph and replayed with other inputs."""
    import osm_b200 as osm
    from gpu_util import MoeFixture

    H, E, I, k = 512, 32, 256, 4
    f = MoeFixture(torch, H, E, I, k, seed=31, max_tokens=T)
    gate, up = (Case(torch, T, H, I, n=6, seed=s, dtype="fp32", half="fp16") for s in (1, 2))
    down = Case(torch, T, I, H, n=6, seed=3, dtype="fp32", half="fp16")
    up.x, up.adapter, down.adapter = gate.x, gate.adapter, gate.adapter
    bias = 0.05 * torch.randn(E, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    r = osm.Routing(E, k, score="sigmoid", bias=bias, groups=4, top_groups=2, group_score="top2", scale=1.5)
    ids = torch.zeros(T, k, dtype=torch.int32, device="cuda")
    w = torch.zeros(T, k, device="cuda")
    x, h = gate.x, torch.empty(T, I, device="cuda")
    dense, out, logits = (torch.empty(T, n, device="cuda") for n in (H, H, E))
    down.x, down.y = h, dense

    def step():
        f.layer.route_scores(x, T, r, ids, w)
        g, u = gate.run(f.ctx), up.run(f.ctx)
        f.ctx.swiglu(g, u, h)
        down.run(f.ctx)
        f.layer.run_experts(x, T, ids, w, out, residual=dense)

    def verify():
        torch.cuda.synchronize()
        assert f.ctx.status()[0] == 0
        gy, uy = gate.reference(torch)[0], up.reference(torch)[0]
        down.x = gy / (1 + torch.exp(-gy)) * uy
        dy = down.reference(torch)[0]
        down.x = h
        f.layer.route_qwen_top_k_logits(x, T, logits)
        torch.cuda.synchronize()
        s = torch.sigmoid(logits.double())
        c = (s + bias.double()).view(T, 4, E // 4)
        value = c.sort(2, descending=True).values[:, :, :2].sum(2)
        kept = torch.zeros(T, 4, dtype=torch.bool, device="cuda").scatter_(1, value.topk(2, 1).indices, True)
        pick = c.masked_fill(~kept[:, :, None], -9).view(T, E).topk(k, 1).indices
        assert torch.equal(ids.long(), pick)
        sw = s.gather(1, pick)
        sw = 1.5 * sw / sw.sum(1, keepdim=True)
        assert torch.allclose(w.double(), sw, rtol=1e-5)
        mats = {e: [torch.from_numpy(m).double().cuda() for m in v] for e, v in f.experts(range(E)).items()}

        def run(m):
            gx = x.double() @ m[0].T
            return (gx / (1 + torch.exp(-gx)) * (x.double() @ m[1].T)) @ m[2].T

        shared = run([torch.from_numpy(m).double().cuda() for m in f.shared_f32()])
        ref = dy + torch.sigmoid(x.double() @ torch.from_numpy(f.sg).double().cuda())[:, None] * shared
        for e in range(E):
            ref += run(mats[e]) * (sw * (pick == e)).sum(1, keepdim=True)
        off = (out.double() - ref).abs().amax(1) / ref.abs().amax(1)
        assert float(off.max()) <= 1e-4, float(off.max())

    step()
    verify()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f.ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        step()
    f.ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    x.copy_(torch.randn(T, H, device="cuda", generator=torch.Generator("cuda").manual_seed(T)))
    gate.adapter.copy_(gate.adapter.flip(0))
    out.fill_(-7)
    graph.replay()
    verify()


def test_context_destroyed_behind_its_calls(torch):  # noqa: F811
    """A context may go while the calls of several streams still run."""
    import osm_b200 as osm

    cases = [Case(torch, T, 2048, 1024, n=9, rank=64, dtype=d, seed=i) for i, (T, d) in
             enumerate([(6000, "fp32"), (5000, "bf16"), (900, "fp16")])]
    want = []
    first = osm.Context(0, max_tokens=4)
    for c in cases:
        first.set_stream(torch.cuda.current_stream().cuda_stream)
        want.append(c.run(first).clone())
    torch.cuda.synchronize()
    first.close()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        for c in cases:
            c.yw.fill_(-7)
        torch.cuda.synchronize()
        ctx = osm.Context(0, max_tokens=4)
        for c, s in zip(cases, streams):
            ctx.set_stream(s.cuda_stream)
            for _ in range(10):
                c.run(ctx)
        ctx.reset_stream()
        ctx.close()
        torch.cuda.synchronize()
        for c, w in zip(cases, want):
            assert torch.equal(c.y, w)


FIRST_CALL = """
import sys
sys.path[:0] = {paths!r}
import torch
import osm_b200 as osm
from test_gpu_lora import Case
ctx = osm.Context(0, max_tokens=4)
cases = [Case(torch, T, K, 256, n=5, rank=40, dtype=d, half=h, seed=i) for i, (T, K, d, h) in enumerate(
    [(3, 8192, "fp32", "bf16"), (4, 512, "fp32", "fp16"), (90, 512, "fp32", "fp16"), (200, 768, "bf16", "bf16"),
     (700, 512, "fp32", "fp16"), (4200, 320, "bf16", "fp16")])]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    for c in cases:
        c.run(ctx)
for c in cases:
    c.yw.fill_(-7)
g.replay()
torch.cuda.synchronize()
got = [c.y.clone() for c in cases]
ctx.set_stream(torch.cuda.current_stream().cuda_stream)
for c, y in zip(cases, got):
    c.check(torch, ctx)
    assert torch.equal(c.y, y)
print("PASS")
"""


def test_first_calls_of_a_process_are_captured(torch):  # noqa: F811
    """Kernels that were never launched before, and ask for their shared memory at
    their first launch, may have it under capture."""
    import subprocess
    import sys

    paths = [p for p in sys.path if p]
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(paths=paths)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "PASS" in r.stdout, (r.stdout[-2000:], r.stderr[-2000:])
