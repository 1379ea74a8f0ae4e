"""Sizes that take other instances of the kernels than the small tests do."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, slots", [("bfloat16", False), ("float32", True)])
def test_tokens_whose_states_pass_the_caches_by(dtype, slots):
    """States of more than 256 MiB in one call, which are read and written around the caches."""
    from genn_amd.sequence import GatedDeltaRule
    T = {"float32": torch.float32, "bfloat16": torch.bfloat16}[dtype]
    S, H, G, K, V = 150, 32, 16, 128, 128
    gen = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    q, k, v, g, beta = r(S, G * K).to(T), r(S, G * K).to(T), r(S, H * V).to(T), -torch.exp(r(S, H) - 2), torch.sigmoid(r(S, H))
    places = S + 2 if slots else S
    pool, out = r(places, H, K, V), torch.zeros(S, H * V, dtype=T, device="cuda")
    assert S * H * K * V * 4 > 256 << 20
    before = pool.clone()
    where = torch.randperm(places, generator=gen, device="cuda")[:S]
    op = GatedDeltaRule(S, 1, H, K, V, key_heads=G, dtype=dtype, normalise=True)
    op.bind(q=q, k=k, v=v, g=g, beta=beta, out=out, initial_state=pool, final_state=pool, slots=where.to(torch.int32) if slots else None)
    op.run()
    torch.cuda.synchronize()
    if not slots:
        where = torch.arange(S, device="cuda")
    unit = lambda x: (x.double().view(S, G, K) / torch.sqrt((x.double().view(S, G, K) ** 2).sum(-1, keepdim=True) + 1e-6)).repeat_interleave(H // G, 1)  # noqa: E731
    # a sum over 128 keys, a product and a rounding of each element: 128 + 8 operations of half a step of fp32 each, of the lengths of a state's column and a value
    step = (K + 8) * 2.0 ** -24
    for n in range(0, S, 30):
        part = slice(n, n + 30)
        hq, hk, w = unit(q)[part], unit(k)[part], where[part]
        s = torch.exp(g[part].double())[..., None, None] * before[w].double()
        value = v[part].double().view(-1, H, V)
        u = beta[part].double()[..., None] * (value - (s * hk[..., None]).sum(2))
        column = s.norm(dim=2) + value.abs()
        s = s + hk[..., None] * u[..., None, :]
        assert ((pool[w].double() - s).abs() <= 2.0 ** -24 * s.abs() + step * column[:, :, None, :]).all()
        want = (K ** -0.5 * (s * hq[..., None]).sum(2)).view(-1, H * V)
        assert ((out[part].double() - want).abs() <= torch.finfo(T).eps / 2 * want.abs() + step * 2 * column.reshape(-1, H * V)).all()
    others = torch.ones(places, dtype=torch.bool, device="cuda")
    others[where] = False
    assert torch.equal(pool[others], before[others])
