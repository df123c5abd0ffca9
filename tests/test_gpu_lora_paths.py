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
