"""Context.route_scores where a balance bias picks experts whose scores are at or
below what fp32 holds: renormalised weights are still those of 64 bits.

Tolerance as in test_gpu_route_scores: (|d| + E / 32 + 16) 2^-24 of a weight,
twice with renormalisation, |d| being at most 104; 1e-37 absolutely."""
import numpy as np
import pytest

from test_gpu_route_scores import ctx, define, run, torch  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 2)])
@pytest.mark.parametrize("score,logits", [
    ("sigmoid", (-55.5, -86.5, -90.75)),            # 8e-25, 3e-38, 4e-40: two below fp32's normal values
    ("sigmoid", (-33.0, -132.0, -100.0)), ("sigmoid", (-68.0, -69.0, -103.0)), ("sigmoid", (-2.0, -3.0, -95.0)),
    ("softmax", (-11.0, -5.0, -35.5)), ("softmax", (28.5, -30.25, 23.75)), ("softmax", (70.0, -25.0, -30.0))])
def test_renormalised_weights_of_small_scores(torch, ctx, score, logits, groups, keep, renorm):  # noqa: F811
    E, k = 64, 3
    at = [3, 9, 35]                                 # in groups 0 and 2
    l = -120 + 10 * torch.rand(5, E, device="cuda", generator=torch.Generator("cuda").manual_seed(E))
    l[:, 1] = 75.0                                  # the largest: softmax scores are relative to it
    l[:, at] = torch.tensor(logits, device="cuda")
    bias = np.zeros(E, np.float32)
    bias[at] = [4.0, 3.0, 2.0]
    ids, w, mass = run(torch, ctx, l, k, score=score, bias=bias, groups=groups, keep=keep, renorm=renorm)
    tol = (104 + E / 32 + 16) * 2.0 ** -24 * (2 if renorm else 1)
    for t in range(5):
        ri, rw, rm = define(l[t].cpu().numpy(), k, score=score, bias=bias, groups=groups, keep=keep, renorm=renorm)
        assert ids[t].tolist() == list(ri) == at
        np.testing.assert_allclose(w[t], rw, rtol=tol, atol=1e-37)
        np.testing.assert_allclose(mass[t], rm, rtol=tol, atol=1e-37)
