"""CPU: the bounds that attention over the 4-bit cache is held to are met by an output that is rounded once, and by none that lost something."""
import pytest
import torch

from tests import kv4_bounds
from tests import kv4_reference as ref


def case(L, new, heads, nkv, hd, qscale, seed):
    g = torch.Generator().manual_seed(seed)
    x = lambda t, h, s: (torch.randn(t, h, hd, generator=g) * s).bfloat16()  # noqa: E731
    return x(new, heads, qscale), ref.values(x(L, nkv, 1.3).float()), ref.values(x(L, nkv, 1.0).float())


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("L,new,heads,nkv,hd,qscale", [(30, 3, 8, 2, 64, 1.5), (200, 1, 16, 1, 80, 1.5), (1000, 4, 4, 1, 128, 1.5), (5000, 1, 4, 1, 128, 1.0), (33000, 1, 4, 1, 128, 0.3),
                                                       (33000, 1, 5, 1, 64, 0.3), (700, 40, 4, 2, 64, 1.5)])
def test_what_the_bounds_let_pass(L, new, heads, nkv, hd, qscale, many):
    q, K, V = case(L, new, heads, nkv, hd, qscale, L + hd)
    cached, scale = L - new, hd ** -0.5
    limits = kv4_bounds.bounds(q, K, V, cached, scale, many=many)
    exact = ref.attention(q, K, V, cached, scale)
    assert (limits[0] - exact).abs().max() <= 1e-12
    worst, whole = kv4_bounds.check(exact.bfloat16(), *limits)
    assert whole >= 0.1                                    # the bounds are not far above what one rounding takes
    wrong = [torch.zeros_like(exact), ref.attention(q, K, V, cached, scale * 1.03), ref.attention(q, K, V.roll(1, 0), cached, scale), exact * 1.004]
    if L >= 128:
        for page in {0, (L // 64) // 2, L // 64 - 2}:      # without a page, and with one twice
            keep = torch.ones(L, dtype=torch.bool)
            keep[64 * page:64 * page + 64] = False
            twice = torch.cat([K[:64 * page + 64], K[64 * page:]]), torch.cat([V[:64 * page + 64], V[64 * page:]])
            wrong += [ref.attention(q, K[keep], V[keep], cached - 64, scale), ref.attention(q, *twice, cached + 64, scale)]
    for i, out in enumerate(wrong):
        with pytest.raises(AssertionError):
            kv4_bounds.check(out.bfloat16(), *limits)
            pytest.fail(f"output {i} was let pass")
