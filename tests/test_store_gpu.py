"""The store into e4m3 caches whose rows are whole 8 bytes and no whole 16: checks and tolerances of the store of other
sizes."""
import pytest
import torch

from ako4x_b200 import qk_norm_rope, rope
from test_rope_gpu import _qkv
from test_rope_gpu import test_store as store

pytestmark = pytest.mark.gpu
BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.mark.parametrize("layout", ["tokens", "heads", "pairs"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,ps", [(70, 4, 3, 72, 72, 16), (33, 2, 2, 104, 40, 7), (300, 3, 2, 136, 64, 16), (5, 8, 8, 8, 8, 1),
                                                        (700, 1, 2, 24, 8, 32), (9, 2, 3, 248, 248, 5), (6000, 1, 1, 56, 20, 16)])
def test_rows_of_8_bytes(built_lib, tokens, hq, hk, dim, rotary, ps, dtype, layout):
    store(built_lib, tokens, hq, hk, dim, rotary, ps, dtype, E4M3, layout)


def test_a_cache_inside_another(built_lib):
    """Data and strides on 8 bytes; what lies between the rows stays."""
    q, k, v = _qkv(20, 2, 3, 64, BF16, 1)
    f, _ = rope.frequencies(64)
    pos, slots = torch.arange(20).cuda(), torch.arange(20).flip(0).cuda()
    sc = [torch.ones(3, 8, 3, device="cuda") for _ in range(4)]
    flat = [torch.zeros(3, 8, 3, 64, device="cuda").to(E4M3) for _ in range(2)]
    wide = [torch.ones(3, 8, 3, 88, device="cuda").to(E4M3) for _ in range(2)]
    qk_norm_rope.run_to_cache(q, k, v, None, None, pos, f, slots, flat[0], flat[1], sc[0], sc[1])
    inside = [x[..., 8:72] for x in wide]
    assert inside[0].data_ptr() % 16 == 8
    qk_norm_rope.run_to_cache(q, k, v, None, None, pos, f, slots, inside[0], inside[1], sc[2], sc[3])
    for a, b, c in zip(flat, inside, wide):
        rows = slots // 8, slots % 8
        assert torch.equal(a[rows].view(torch.uint8), b[rows].view(torch.uint8))
        assert (c[..., :8].float() == 1).all() and (c[..., 72:].float() == 1).all()
    assert torch.equal(sc[0], sc[2]) and torch.equal(sc[1], sc[3])
