"""Context.q4_gemv_lora on its prompt path (more than 256 tokens, or more than
1e9 products), where operands are prepared and the adapters are further steps
of one sum: row types unlike the adapters', ranks that fill no whole piece,
ranges of a tile's tokens and of a CTA's share of K.

Cases, the definition in 64 bits and the tolerance of fp32 rows are those of
test_gpu_lora."""
import pytest

from test_gpu_lora import Case, ctx, torch  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


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
    """No operand of the two parts has fewer than 22 bits, whatever the rows'
    type: the tolerance of test_gpu_lora without its term 2^-11 C.

    Per group: c = bias + 8 scale is hi + lo of fp16, within 2^-24 of itself; the
    sum of x is taken in fp32 (10 half-ulps, 2^-24 each, of the sum of magnitudes)
    and held as hi + lo, 2^-24; the product of the two lo parts is left out, 2^-24:
    under 16 2^-23 C together.  Steps of 16: K / 16 of the products, 3 K / 1024 of
    the biases' columns, rounded up to a stage of 4: under K / 8 + K / 256 + 4, each
    with a loss of 2^-23 of the sum of magnitudes at most.  v is held in 16 bits for
    16-bit rows, 2^-15 L as there; y of fp16 is rounded to a multiple of 2^-24 at
    the least."""
    c = one_sided(torch, T, K, N, dtype, kind, seed=K)
    c.run(ctx)
    torch.cuda.synchronize()
    y, (S, C), L = c.reference(torch)
    tol = (torch.finfo(c.dt).eps / 2 * y.abs() + (K / 8 + K / 256 + 20) * 2.0 ** -23 * (S + L) + c.rank * 2.0 ** -23 * L
           + 1e-30)
    if dtype != "fp32":
        tol = tol + 2.0 ** -15 * L
    if dtype == "fp16":
        tol = tol + 2.0 ** -25
    off = (c.y.double() - y).abs() / tol
    assert float(off.max()) <= 1.0, float(off.max())


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
    y, S, L = case.reference(torch)
    assert float(((case.y.double() - y).abs() / case.tolerance(torch, y, S, L)).max()) <= 1.0
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
