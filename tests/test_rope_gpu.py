"""Rotary positions and head norms against the formulas in 64 bits.

Tolerances: a result is rounded once, by at most eps / 2 of its value (bf16 2^-8 / 2 is written as
finfo.eps / 2 = 2^-8 for bf16, 2^-11 for fp16), and half the smallest step where fp16 runs out of exponents (2^-25). Before that everything is fp32: the angle (reduced in fp64, then
2^-25 of a turn, 1.9e-7), sine and cosine (2 units of 2^-24), two products and a sum make less than 2^-21 of the magnitudes that
are added; the norm adds the sum of dim squares (its rounding grows with the 8 + 5 steps that one element sees, halved by
the root), rsqrt (2 units) and two products, less than 2^-20. Both are doubled: 2^-20 and 2^-19 of the magnitudes."""
import pytest
import torch

import oracle
from ako4x_b200 import qk_norm_rope, rope

pytestmark = pytest.mark.gpu
BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _check(out, ref, size, rel, what):
    ref = ref.to(out.device)
    tol = torch.finfo(out.dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -8) + rel * size.to(out.device) + 2.0 ** -25
    err = (out.double() - ref).abs()
    assert (err <= tol).all(), f"{what}: {int((err > tol).sum())} of {err.numel()}, worst {float((err / tol).max()):.3g} tolerances"


def _qkv(tokens, hq, hk, dim, dtype, seed, fused=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, (hq + 2 * hk) * dim, generator=g).to(dtype).cuda()
    q, k, v = x.split([hq * dim, hk * dim, hk * dim], dim=1)
    q, k, v = q.view(tokens, hq, dim), k.view(tokens, hk, dim), v.view(tokens, hk, dim)
    return (q, k, v) if fused else (q.contiguous(), k.contiguous(), v.contiguous())


def _positions(tokens, seed, far=1 << 20):
    g = torch.Generator().manual_seed(seed)
    pos = torch.randint(0, far, (tokens,), generator=g)
    pos[0] = 0
    return pos


SHAPES = [  # tokens, q heads, k heads, dim, rotary
    (1, 32, 8, 128, 128), (5, 16, 1, 64, 64), (37, 7, 7, 80, 20), (64, 4, 2, 256, 64), (3, 1, 1, 8, 8), (9, 12, 3, 96, 48),
    (2, 5, 1, 192, 96), (130, 3, 1, 72, 72), (11, 2, 1, 104, 2), (700, 40, 8, 128, 64), (6000, 2, 1, 64, 32), (4, 9, 2, 248, 248),
    (17, 6, 6, 136, 0), (33, 1, 1, 128, 100),
    # rotated parts of an odd number of eights: pieces of half the size, in rows of one, two and four to a warp
    (33, 5, 2, 80, 40), (21, 4, 2, 96, 24), (6000, 2, 1, 64, 40), (13, 3, 1, 256, 200), (1, 1, 0, 24, 24), (10, 2, 2, 64, 26)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary", SHAPES)
def test_rope(built_lib, tokens, hq, hk, dim, rotary, interleaved, dtype):
    q, k, _ = _qkv(tokens, hq, hk, dim, dtype, tokens + dim)
    f = torch.empty(0) if rotary == 0 else rope.frequencies(rotary, device="cpu")[0]
    pos = _positions(tokens, dim + rotary)
    qo, ko = rope.run(q, k, pos.int().cuda(), f.cuda(), interleaved, 1.25)
    assert qo.is_contiguous() and qo.shape == q.shape and ko.shape == k.shape and qo.dtype == dtype
    for x, y, what in ((q, qo, "q"), (k, ko, "k")):
        ref, size = oracle.paged.rotate(x.cpu(), pos, f, interleaved, 1.25)
        _check(y, ref, size, 2.0 ** -20, what)
        assert torch.equal(y[..., rotary:], x[..., rotary:])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary", SHAPES)
def test_norm(built_lib, tokens, hq, hk, dim, rotary, interleaved, dtype):
    q, k, _ = _qkv(tokens, hq, hk, dim, dtype, tokens + dim)
    g = torch.Generator().manual_seed(dim)
    w = [(1 + 0.3 * torch.randn(dim, generator=g)).to(dtype if tokens % 2 else torch.float32) for _ in range(2)]
    f = torch.empty(0) if rotary == 0 else rope.frequencies(rotary, device="cpu")[0]
    pos = _positions(tokens, dim + rotary)
    outs = qk_norm_rope.run(q, k, w[0].cuda(), w[1].cuda(), pos.cuda(), f.cuda(), 1e-5, interleaved, 0.9)
    for x, y, wi, what in zip((q, k), outs, w, "qk"):
        ref, size = oracle.paged.rotate(oracle.paged.head_norm(x.cpu(), wi, 1e-5), pos, f, interleaved, 0.9)
        _check(y, ref, size, 2.0 ** -19, what)


def test_far_positions_are_as_exact_as_near_ones(built_lib):
    pos = torch.tensor([0, 1, 2 ** 20 - 1, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 40 + 12345, -7, -(2 ** 33)])
    q, _, _ = _qkv(len(pos), 2, 1, 64, FP16, 1)
    f, _ = rope.frequencies(64, device="cpu")
    # the first frequency is 1, the last ones small: at 2^40 radians fp64 itself is good to 2^-13
    keep = pos.abs() < 2 ** 34
    y, none = rope.run(q, None, pos.cuda(), f.cuda())
    assert none is None
    ref, size = oracle.paged.rotate(q.cpu(), pos, f)
    # what fp64 loses of the angles on either side: two roundings of up to 2^34 radians
    _check(y[keep.cuda()], ref[keep], size[keep], 2.0 ** -20 + 2 * 2.0 ** 34 * 2.0 ** -53, "far")


def test_strides_and_misaligned_views(built_lib):
    f, _ = rope.frequencies(64, device="cpu")
    pos = _positions(9, 2)
    base = torch.randn(9, 6, 130, generator=torch.Generator().manual_seed(7)).to(BF16).cuda()
    views = [base[:, :, :128], base[:, :, 1:129], base[:, ::2, 2:130], base[:, 1:2, :128].expand(9, 4, 128),
             base[:, :, :128].transpose(0, 1).contiguous().transpose(0, 1), base.flip(0)[:, :, :128]]
    for q in views:
        y, _ = rope.run(q, None, pos.cuda(), f.cuda())
        z, _ = rope.run(q.contiguous(), None, pos.cuda(), f.cuda())
        assert torch.equal(y, z)
    wide = torch.arange(18).cuda()[::2]                      # positions with a stride
    assert torch.equal(rope.run(views[0], None, wide, f.cuda())[0], rope.run(views[0], None, wide.contiguous(), f.cuda())[0])


def test_nothing_to_do(built_lib):
    f, _ = rope.frequencies(64, device="cuda")
    q = torch.zeros(0, 4, 64, dtype=BF16, device="cuda")
    y, z = rope.run(q, q[:, :1], torch.zeros(0, dtype=torch.int32, device="cuda"), f)
    assert y.shape == q.shape and z.shape == (0, 1, 64)
    q = torch.randn(3, 4, 64, device="cuda").to(BF16)
    y, z = rope.run(q, q[:, :0], torch.arange(3, device="cuda"), f)
    assert z.shape == (3, 0, 64) and torch.equal(y, rope.run(q, None, torch.arange(3, device="cuda"), f)[0])


def test_values_that_are_not_finite_stay_in_their_pairs(built_lib):
    q = torch.ones(2, 3, 64, dtype=BF16)
    q[0, 0, 5], q[0, 1, 40], q[1, 2, 63] = float("inf"), float("nan"), float("-inf")
    f, _ = rope.frequencies(32, device="cpu")
    for interleaved in (False, True):
        y, _ = rope.run(q.cuda(), None, torch.tensor([3, 9]).cuda(), f.cuda(), interleaved)
        ref, _ = oracle.paged.rotate(q, torch.tensor([3, 9]), f, interleaved)
        fin = torch.isfinite(ref)
        assert torch.equal(torch.isfinite(y.cpu()), fin)
        assert torch.equal(torch.isnan(y.cpu()), torch.isnan(ref))


CACHES = [(1, 32, 8, 128, 128, 16), (70, 8, 2, 64, 64, 1), (33, 6, 3, 80, 20, 7), (300, 16, 4, 256, 64, 64), (6, 2, 1, 96, 96, 24),
          (45, 4, 2, 80, 40, 16), (12, 3, 2, 256, 24, 5), (700, 1, 1, 64, 8, 32)]


def _cache(pages, ps, hk, dim, kind, layout):
    """Caches with something in them: pages of tokens, pages of heads, or keys and values side by side."""
    if layout == "tokens":
        c = [torch.zeros(pages, ps, hk, dim, device="cuda") for _ in range(2)]
    elif layout == "heads":
        c = [torch.zeros(pages, hk, ps, dim, device="cuda").transpose(1, 2) for _ in range(2)]
    else:
        c = list(torch.zeros(pages, 2, ps, hk, dim, device="cuda").unbind(1))
    return [(x + 3).to(kind) if layout == "tokens" else torch.empty_like(x, dtype=kind).copy_(torch.full_like(x, 3.0)) if layout == "heads"
            else x for x in c] if layout != "pairs" else list(torch.full((pages, 2, ps, hk, dim), 3.0, device="cuda").to(kind).unbind(1))


@pytest.mark.parametrize("layout", ["tokens", "heads", "pairs"])
@pytest.mark.parametrize("dtype,kind", [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, E4M3)])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,ps", CACHES)
def test_store(built_lib, tokens, hq, hk, dim, rotary, ps, dtype, kind, layout):
    q, k, v = _qkv(tokens, hq, hk, dim, dtype, tokens)
    if tokens > 4:
        v[3] = 0                                             # rows of zeros: scale 1
        k[4, 0, 1], v[4, 0, 2] = 1000.0, -3000.0
    g = torch.Generator().manual_seed(dim)
    w = [(1 + 0.3 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2)]
    f, _ = rope.frequencies(rotary, device="cpu")
    pos = _positions(tokens, ps, 50000)
    pages = tokens // ps + 2
    slots = torch.randperm(pages * ps, generator=g)[:tokens]
    if tokens > 4:
        slots[1], slots[2] = -1, pages * ps                  # padding, and a slot behind the cache
    kc, vc = _cache(pages, ps, hk, dim, kind, layout)
    ks = vs = None
    if kind == E4M3:
        ks, vs = torch.full((pages, ps, hk), 5.0, device="cuda"), torch.full((hk, pages, ps), 5.0, device="cuda").permute(1, 2, 0)
    qo = qk_norm_rope.run_to_cache(q, k, v, w[0].cuda(), w[1].cuda(), pos.int().cuda(), f.cuda(), slots.int().cuda(), kc, vc, ks, vs)
    qr, kr = qk_norm_rope.run(q, k, w[0].cuda(), w[1].cuda(), pos.cuda(), f.cuda())
    assert torch.equal(qo, qr)
    ref, size = oracle.paged.rotate(oracle.paged.head_norm(k.cpu(), w[1]), pos, f)
    stored = (slots >= 0) & (slots < pages * ps)
    at = slots[stored]
    page, slot = (at // ps).cuda(), (at % ps).cuda()
    untouched = torch.ones(pages, ps, dtype=torch.bool, device="cuda")
    untouched[page, slot] = False
    for c in (kc, vc):
        assert (c.float()[untouched] == 3.0).all()           # slots that no token has are as they were
    if kind != E4M3:
        assert torch.equal(kc[page, slot], kr[stored.cuda()]) and torch.equal(vc[page, slot], v[stored.cuda()])
        return
    for s in (ks, vs):
        assert (s[untouched] == 5.0).all()
    # the values: the library's rule, bit for bit
    vq, vsc = oracle.paged.quantize_rows(v.cpu()[stored])
    assert torch.equal(vs[page, slot].cpu(), vsc) and torch.equal(vc[page, slot].cpu().view(torch.uint8), vq.view(torch.uint8))
    # the keys: from fp32 values that are 2^-19 of their magnitudes off; the scale is its largest one / 448, the values
    # half a step off (2^-4 of themselves, 2^-10 of the scale below the normal ones)
    ref, size = ref[stored], size[stored]
    top = ref.abs().amax(-1)
    sc = ks[page, slot].cpu().double()
    assert ((sc * 448 - top).abs() <= 2.0 ** -19 * size.amax(-1) + 2.0 ** -22 * top).all()
    got = kc[page, slot].cpu().double() * sc[..., None]
    tol = 2.0 ** -4 * ref.abs() + 2.0 ** -10 * sc[..., None] + 2.0 ** -18 * size
    assert ((got - ref).abs() <= tol).all()


def test_store_without_norms_and_with_nan(built_lib):
    q, k, v = _qkv(4, 4, 2, 64, BF16, 11)
    k[2, 1, 7] = float("nan")
    f, _ = rope.frequencies(64)
    pos, slots = torch.arange(4).cuda(), torch.tensor([5, 0, 2, 7]).cuda()
    kc, vc = torch.zeros(2, 4, 2, 64, dtype=BF16, device="cuda"), torch.zeros(2, 4, 2, 64, dtype=BF16, device="cuda")
    qo = qk_norm_rope.run_to_cache(q, k, v, None, None, pos, f, slots, kc, vc)
    qr, kr = rope.run(q, k, pos, f)
    assert torch.equal(qo, qr)
    assert torch.equal(kc.view(8, 2, 64)[slots].view(torch.int16), kr.view(torch.int16))
    assert torch.equal(vc.view(8, 2, 64)[slots], v)
    ke, ve, ks, vs = kc.to(E4M3), vc.to(E4M3), torch.zeros(2, 4, 2, device="cuda"), torch.zeros(2, 4, 2, device="cuda")
    qk_norm_rope.run_to_cache(q, k, v, None, None, pos, f, slots, ke, ve, ks, vs)
    bad = torch.isnan(ks.view(8, 2))
    assert bad[2, 1] and int(bad.sum()) == 1                 # a row with a NaN, and no other, has a scale of NaN


def test_weights_and_tables_that_are_views(built_lib):
    q, k, _ = _qkv(7, 4, 2, 64, BF16, 12)
    f, _ = rope.frequencies(64)
    pos = torch.arange(7).cuda()
    base = (1 + 0.1 * torch.randn(200, generator=torch.Generator().manual_seed(1))).to(BF16).cuda()
    for w in (base[1:65], base[3:131:2], base.float()[1:65]):
        a = qk_norm_rope.run(q, k, w, w, pos, f)
        b = qk_norm_rope.run(q, k, w.clone(), w.clone(), pos, f)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    odd = torch.zeros(33, device="cuda")
    odd[1:] = f
    assert torch.equal(rope.run(q, None, pos, odd[1:])[0], rope.run(q, None, pos, f)[0])


@pytest.mark.parametrize("tokens", [5919, 5920, 5921, 11843, 23700])
@pytest.mark.parametrize("interleaved", [False, True])
def test_tokens_side_by_side(built_lib, tokens, interleaved):
    """Around the sizes at which a warp takes one, two, four and eight tokens; the last warp not full."""
    for hq, hk, dim, rotary in ((3, 1, 64, 64), (1, 1, 48, 20), (2, 1, 128, 64), (1, 0, 16, 16)):
        q, k, _ = _qkv(tokens, hq, max(hk, 1), dim, BF16, tokens)
        k = k[:, :hk]
        f, _ = rope.frequencies(rotary)
        pos = _positions(tokens, dim, 100000).cuda()
        y, z = rope.run(q, k, pos, f, interleaved)
        for at in range(0, tokens, 3000):                    # pieces too short for that
            a, b = rope.run(q[at:at + 3000], k[at:at + 3000], pos[at:at + 3000], f, interleaved)
            assert torch.equal(y[at:at + 3000], a) and torch.equal(z[at:at + 3000], b)


def test_captured_and_replayed(built_lib):
    q, k, v = _qkv(20, 8, 2, 128, BF16, 5)
    w = torch.ones(128, dtype=BF16, device="cuda")
    f, _ = rope.frequencies(128)
    pos, slots = torch.arange(20).cuda(), torch.arange(20).cuda()
    kc, vc = (torch.zeros(2, 16, 2, 128, dtype=BF16, device="cuda") for _ in range(2))
    call = lambda: qk_norm_rope.run_to_cache(q, k, v, w, w, pos, f, slots, kc, vc)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    q.normal_()
    k.normal_()
    pos.add_(100)
    slots.add_(7)
    kc.zero_()
    graph.replay()
    torch.cuda.synchronize()
    held = kc.clone()
    kc.zero_()
    assert torch.equal(out, call()) and torch.equal(held, kc)


def test_side_stream(built_lib):
    q, k, _ = _qkv(300, 8, 2, 64, FP16, 6)
    f, _ = rope.frequencies(64)
    pos = torch.arange(300).cuda()
    want = rope.run(q, k, pos, f)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rope.run(q, k, pos, f)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
