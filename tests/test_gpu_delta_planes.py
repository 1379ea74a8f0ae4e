"""Products of fp32 accuracy on the bf16 matrix instructions, at values where a sum of three bf16 ones loses most."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [1 + 2.0 ** -7 - 2.0 ** -23, 1 + 2.0 ** -8 - 2.0 ** -23, 1 + 2.0 ** -8 + 2.0 ** -16 - 2.0 ** -23, 2 - 2.0 ** -23, 1 + 2.0 ** -7 + 2.0 ** -15 - 2.0 ** -23])
@pytest.mark.parametrize("negative", [False, True])
def test_products_lose_no_more_than_half_a_step(value, negative):
    """One key, kept from the first row on, and queries of all rows: 32 times the value squared, within a chunk and behind it.

    What is left out is below 2^-24 of the whole.  Behind it come two products one after another (the scores, or the state as an operand; and what they multiply, which is 1), of each of which one
    addition is to the whole sum and off by at most a step (2^-23): 5 x 2^-24 in all."""
    from genn_amd.sequence import GatedDeltaRule
    n, K = 70, 32
    q, k, v = torch.full((n, K), -value if negative else value), torch.zeros(n, K), torch.zeros(n, 1)
    beta, g, out = torch.zeros(n, 1), torch.zeros(n, 1).cuda(), torch.zeros(n, 1).cuda()
    k[0], v[0], beta[0] = value, 1.0, 1.0
    op = GatedDeltaRule(1, n, 1, K, 1, scale=1.0)
    op.bind(q=q.cuda(), k=k.cuda(), v=v.cuda(), g=g, beta=beta.cuda(), out=out)
    op.run()
    want = K * float(q[0, 0].double()) * float(k[0, 0].double())
    off = (out.cpu().double() / want - 1) * 2.0 ** 24
    assert (off.abs() <= 5).all(), (float(off[:32].abs().max()), float(off[32:].abs().max()))
