"""Attention of one new token over a paged cache where weights, scales and values differ by many powers of two,
against the formula in 64 bits.

Tolerances as in the tests of ordinary values: the output's own rounding (half a step, finfo.eps / 2 of its value), and,
relative to the weighted mean magnitude of the values, 2^-15 for the two pieces of a weight, n / 16 + 64 roundings of
fp32 for the sums, dim 2^-24 A for a score of magnitude A, 2^-21 for exp2. Queries in bf16 meet e4m3 keys in fp16, a
head's largest element at 2^14 to 2^15: the smallest step of fp16, 2^-24, is then 2^-38 of it at most, so that every element of q is off by
half of that, 2^-39 of the largest, and a score by that times the sum of its key's magnitudes. None of them has an absolute part but the end of
the output's type: 2^-25 in fp16, 2^-134 in bf16."""
import pytest
import torch

import oracle
from ako4x_b200 import paged_decode
from test_paged_decode_gpu import make, on_gpu

pytestmark = pytest.mark.gpu
BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def check(a, o, lse, **more):
    ro, rlse, size, score = oracle.paged.paged_decode(**{**a, **more})
    dim, n = a["q"].shape[2], max(int(x) for x in a["seq_lens"])
    rel = (n / 16 + 64) * 2.0 ** -24 + dim * 2.0 ** -24 * score + 2.0 ** -21
    if a["k_cache"].dtype == E4M3 and o.dtype == BF16:
        key = (a["k_cache"].double().abs().sum(-1) * a["k_scale"].double()).max()
        rel = rel + 2.0 ** -39 * a["q"].double().abs().amax(-1) * key * a["sm_scale"]
    end = 2.0 ** -25 if o.dtype == FP16 else 2.0 ** -134
    tol = torch.finfo(o.dtype).eps / 2 * (1 + 2.0 ** -8) * ro.abs() + (rel + 2.0 ** -15)[..., None] * size + end
    o = o.cpu().double()
    if end == 2.0 ** -25:                                    # 65520 and more are infinite in fp16: half a step above its last value
        beyond = ro.abs() >= 65520 + tol
        assert torch.equal(o[beyond], ro[beyond].sign() * float("inf"))
        o = torch.where(beyond, ro, o)
    err = (o - ro).abs()
    assert (err <= tol).all(), f"o: {int((~(err <= tol)).sum())} of {err.numel()}, worst {float((err / tol).max()):.3g} tolerances"
    off, lim = (lse.cpu().double() - rlse).abs(), rel * 1.4427 + 2.0 ** -23 * (rlse.abs() + 1)
    assert (off <= lim).all(), f"lse: worst {float((off / lim).max()):.3g} tolerances"


def run_check(a, **more):
    o, lse = paged_decode.run(**on_gpu(a), **more)
    check(a, o, lse, **more)
    return o, lse


def at(a, b, t):
    ps = a["k_cache"].shape[1]
    return int(a["block_table"][b, t // ps]), t % ps


LAYOUTS = [  # lengths, KV heads, group, dim, page size: shares and merge, a CTA for a sequence, the warps of a CTA for one
    ([3000, 40], 2, 4, 128, 16), ([64, 33, 17] * 30, 4, 8, 64, 16), ([100], 1, 4, 128, 16), ([700, 31], 1, 20, 64, 7),
    ([500], 2, 3, 256, 16), ([90, 200], 1, 9, 256, 5)]


@pytest.mark.parametrize("scale", [1e-5, 1e-7, 1e-9, 1e-11, 2e-13])
@pytest.mark.parametrize("lens,hk,group,dim,ps", LAYOUTS)
def test_a_row_of_zeros_among_small_values(built_lib, lens, hk, group, dim, ps, scale):
    """The store gives a row of zeros the scale 1, whatever the other rows have."""
    a = make(lens, hk, group, dim, BF16, E4M3, ps, seed=dim)
    a["v_scale"] = a["v_scale"] * 50 * scale
    for b, n in enumerate(lens):
        where = at(a, b, n // 2)
        a["v_cache"][where], a["v_scale"][where] = 0, 1.0
    run_check(a)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("octaves", [20, 30, 60])
@pytest.mark.parametrize("lens,hk,group,dim,ps", LAYOUTS)
def test_one_scale_far_above_the_others(built_lib, lens, hk, group, dim, ps, octaves, dtype):
    """Of a key that is large in one feature alone, and hardly weighs anything."""
    a = make(lens, hk, group, dim, dtype, E4M3, ps, seed=dim + octaves)
    a["q"] = a["q"].abs()
    for b, n in enumerate(lens):
        where = at(a, b, n // 3)
        a["v_cache"][where] = 0
        a["v_cache"][where][..., 5] = 1.5
        a["v_scale"][where] = 2.0 ** (octaves - 6)
        a["k_cache"][where] = -448.0
        a["k_scale"][where] = 30 / (448 * dim ** 0.5 * 0.8)     # some 30 below the others, 2^-43
    run_check(a)


@pytest.mark.parametrize("lens,hk,group,dim,ps", LAYOUTS)
def test_scales_of_all_sizes(built_lib, lens, hk, group, dim, ps):
    """Values of neighbouring keys, each in features of its own, differ by up to 2^60."""
    a = make(lens, hk, group, dim, BF16, E4M3, ps, seed=dim + 1)
    g = torch.Generator().manual_seed(dim)
    a["v_scale"] = 2.0 ** (torch.rand(a["v_scale"].shape, generator=g) * 60 - 45)
    pages, ps, hk, dim = a["v_cache"].shape
    mine = torch.randint(0, 8, (pages, ps, hk, 1), generator=g) == torch.arange(dim) % 8
    a["v_cache"] = (a["v_cache"].float() * mine).to(E4M3)
    run_check(a)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens,hk,group,dim,ps", LAYOUTS)
def test_a_key_of_zeros_far_above_the_others(built_lib, lens, hk, group, dim, ps, dtype):
    """One key takes all the weight and has no value: what is left of the others is the answer, feature by feature."""
    a = make(lens, hk, group, dim, dtype, E4M3, ps, seed=dim + 2)
    a["q"] = a["q"].abs()
    # what fp16 can hold of it, and all sizes in bf16
    a["v_scale"] = a["v_scale"] * (2.0 ** 40 if dtype == FP16 else 2.0 ** -10)
    for b, n in enumerate(lens):
        where = at(a, b, n - 1)
        a["v_cache"][where], a["k_cache"][where] = 0, 448.0
        a["k_scale"][where] = 30 / (448 * dim ** 0.5 * 0.8)
    run_check(a)


@pytest.mark.parametrize("lens,hk,group,dim,ps", LAYOUTS)
def test_values_near_the_end_of_bf16(built_lib, lens, hk, group, dim, ps):
    """No sum of weights and values is above 2^126: 700 times 448 times 2^107."""
    a = make([min(n, 700) for n in lens], hk, group, dim, BF16, E4M3, ps, seed=dim + 3)
    a["v_scale"] = a["v_scale"] * 50 * 2.0 ** 107
    run_check(a)


@pytest.mark.parametrize("octaves", [10, 20, 28])
@pytest.mark.parametrize("lens,hk,group,dim,ps", LAYOUTS)
def test_a_feature_of_q_far_above_the_others(built_lib, lens, hk, group, dim, ps, octaves):
    """That no key has: the scores come from the others."""
    a = make(lens, hk, group, dim, BF16, E4M3, ps, seed=dim + octaves + 1)
    a["q"][..., 7] = 2.0 ** octaves
    a["k_cache"][..., 7] = 0
    run_check(a)


@pytest.mark.parametrize("power", [-119, -110, -60, 60, 124])
@pytest.mark.parametrize("lens,hk,group,dim,ps", LAYOUTS)
def test_queries_of_any_size(built_lib, lens, hk, group, dim, ps, power):
    """Against scales of the keys that make ordinary scores of them."""
    a = make(lens, hk, group, dim, BF16, E4M3, ps, seed=dim + 5)
    a["q"] = (a["q"].float().clamp(-7, 7) * 2.0 ** power).to(BF16)
    a["k_scale"] = a["k_scale"] * 2.0 ** -power
    run_check(a)


# ---- 16-bit caches ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("nats", [16, 24, 27, 29, 33])
@pytest.mark.parametrize("lens,hk,group,dim,ps", LAYOUTS)
def test_a_key_without_a_value_far_above_the_others(built_lib, lens, hk, group, dim, ps, nats, dtype):
    """One key takes all the weight, its value is zero, and the others have the largest values that the type holds."""
    a = make(lens, hk, group, dim, dtype, dtype, ps, seed=dim + nats)
    a["q"] = a["q"].abs()
    big = 60000.0 if dtype == FP16 else 1e30
    a["v_cache"] = (a["v_cache"].float().sign() * big).to(dtype)
    a["v_cache"][..., ::2] = big                             # no signs that cancel in every other feature
    mean = a["q"].float().mean() * dim ** 0.5                # of a score with ones
    for b, n in enumerate(lens):
        where = at(a, b, n - 1)
        a["v_cache"][where], a["k_cache"][where] = 0, float(nats / mean)
    run_check(a)


@pytest.mark.parametrize("dtype,kind", [(BF16, BF16), (FP16, FP16)])
@pytest.mark.parametrize("nats", [20, 30, 45, 60])
@pytest.mark.parametrize("lens,hk,group,dim,ps", LAYOUTS)
def test_an_infinite_value_far_below_the_others(built_lib, lens, hk, group, dim, ps, nats, dtype, kind):
    """It counts, however little its key weighs."""
    a = make(lens, hk, group, dim, dtype, kind, ps, seed=dim + nats)
    a["q"] = a["q"].abs()
    a["k_cache"] = (a["k_cache"].float() * 0.25).to(kind)
    mean = a["q"].float().mean() * dim ** 0.5
    for b, n in enumerate(lens):
        where = at(a, b, n // 2)
        a["k_cache"][where] = -float(nats / mean)
        a["v_cache"][where][..., 3], a["v_cache"][where][..., 8] = float("inf"), float("-inf")
    o, lse = paged_decode.run(**on_gpu(a))
    ro, rlse, *_ = oracle.paged.paged_decode(**a)
    assert (ro[..., 3] == float("inf")).all() and (ro[..., 8] == float("-inf")).all()
    o = o.cpu().double()
    assert torch.equal(o[..., 3], ro[..., 3]) and torch.equal(o[..., 8], ro[..., 8])
    assert int(torch.isfinite(o).sum()) == o.numel() // dim * (dim - 2)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens,hk,group,dim,ps", LAYOUTS)
def test_a_key_that_scores_minus_infinity_weighs_zero(built_lib, lens, hk, group, dim, ps, dtype):
    """A finite value of it is left out; 0 times another one is NaN, in its feature."""
    a = make(lens, hk, group, dim, dtype, dtype, ps, seed=dim + 4)
    a["q"] = a["q"].abs() + 0.125
    for b, n in enumerate(lens):
        a["k_cache"][at(a, b, n // 2)] = float("-inf")
    want = run_check(a)
    for b, n in enumerate(lens):
        a["v_cache"][at(a, b, n // 2)][..., 3], a["v_cache"][at(a, b, n // 2)][..., 8] = float("inf"), float("nan")
    o, lse = paged_decode.run(**on_gpu(a))
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[..., 3] = bad[..., 8] = True
    assert torch.equal(torch.isnan(o), bad) and torch.equal(lse, want[1])
    assert torch.equal(o[~bad], want[0][~bad])
