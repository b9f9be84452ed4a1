"""More tokens than one launch has workgroups for."""
import pytest
import torch

from deepseekrpc_amd import tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_than_2_to_the_24_tokens(dtype):
    """Every token as if alone: small calls over the same rows, at the borders
    of launches and in the end, and the whole against its own inverse."""
    n, kv, dim = (1 << 24) + 77, 1, 4
    g = torch.Generator(device="cuda").manual_seed(3)
    packed = torch.randn(n, 3, dim, generator=g, device="cuda").to(dtype)
    q, k, v = packed[:, :1], packed[:, 1:2], packed[:, 2:]
    pos = torch.randint(0, 1 << 20, (n,), generator=g, device="cuda", dtype=torch.int32)
    slots = torch.arange(n, device="cuda", dtype=torch.int32).flip(0)
    slots[5], slots[(1 << 23) + 5], slots[n - 2] = -1, n + 1000, -9
    freqs, _ = tree.rotary_frequencies(dim)
    kc, vc = (torch.zeros(n // 1024 + 1, 1024, kv, dim, device="cuda", dtype=dtype) for _ in range(2))
    res = tree.rotary(q, k, pos, freqs, v=v, slots=slots, k_cache=kc, v_cache=vc, k_out=torch.empty_like(k))
    for lo in (0, (1 << 23) - 30, (1 << 24) - 30, n - 60):
        part = slice(lo, lo + 60)
        small = tree.rotary(q[part], k[part], pos[part], freqs)
        assert torch.equal(res.q[part], small.q) and torch.equal(res.k[part], small.k)
    bad = torch.zeros(n, dtype=torch.int32, device="cuda")
    bad[n - 2] = tree.E_BLOCK
    bad[(1 << 23) + 5] = tree.E_BLOCK if n + 1000 >= kc.shape[0] * 1024 else 0
    assert torch.equal(res.status, bad)
    there = (slots >= 0) & (bad == 0)
    assert torch.equal(kc.view(-1, kv, dim)[slots[there].long()], res.k[there])
    assert torch.equal(vc.view(-1, kv, dim)[slots[there].long()], v[there])
    back = tree.rotary(res.q, None, pos, freqs, inverse=True).q
    # Two rotations, each a rounding of the value to its type and of two products and a sum in float32.
    u = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-24
    assert float((back - q).abs().max()) <= (4 * u + 32 * 2.0**-24) * float(q.abs().max())
