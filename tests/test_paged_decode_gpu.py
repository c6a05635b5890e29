"""Attention of one new token over a paged cache against the formula in 64 bits.

Tolerances. The output is rounded once (finfo.eps / 2 of its value, fp16 at least 2^-25). Before that,
relative to the weighted mean magnitude of the values: the two pieces of a weight hold 2^-15 of it, the sums of n keys
are rounded n / 16 times by 2^-24 and some thirty times more at joints, a score that is the sum of dim products of magnitude A
in all is off by dim 2^-24 A at most, and so, relatively, is its weight; exp2 adds 2^-21. The log-sum has the same
errors but that of the pieces, in base 2, and its own rounding."""
import pytest
import torch

import oracle
from ako4x_b200 import paged_decode

pytestmark = pytest.mark.gpu
BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def make(lens, hk, group, dim, dtype, kind, ps, seed=0, spread=1.0, extra=3, layout="tokens"):
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // ps) for n in lens]
    pages = sum(held) + extra
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((len(lens), max(held + [1])), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    a = dict(q=(torch.randn(len(lens), hk * group, dim, generator=g) * spread).to(dtype))
    shape = (pages, ps, hk, dim) if layout == "tokens" else (pages, hk, ps, dim)
    for name in ("k_cache", "v_cache"):
        x = torch.randn(shape, generator=g)
        x = (x * 100).clamp(-448, 448).to(E4M3) if kind == E4M3 else x.to(kind)
        a[name] = x if layout == "tokens" else x.transpose(1, 2)
    a.update(block_table=table, seq_lens=torch.tensor(lens, dtype=torch.int32), sm_scale=dim ** -0.5)
    if kind == E4M3:
        a.update(k_scale=torch.rand(pages, ps, hk, generator=g) * 0.02, v_scale=torch.rand(pages, ps, hk, generator=g) * 0.02)
    return a


def on_gpu(a):
    return {k: v.cuda() if torch.is_tensor(v) else v for k, v in a.items()}


def check(a, o, lse, **more):
    ro, rlse, size, score = oracle.paged.paged_decode(**{**a, **more})
    dim, n = a["q"].shape[2], max([int(x) for x in a["seq_lens"]] + [1])
    o, lse = o.cpu(), lse.cpu()
    assert o.dtype == a["q"].dtype and lse.dtype == torch.float32
    rel = (n / 16 + 64) * 2.0 ** -24 + dim * 2.0 ** -24 * score + 2.0 ** -21
    tol = torch.finfo(o.dtype).eps / 2 * (1 + 2.0 ** -8) * ro.abs() + (rel + 2.0 ** -15)[..., None] * size + 2.0 ** -25
    err = (o.double() - ro).abs()
    assert (err <= tol).all(), f"o: {int((err > tol).sum())} of {err.numel()}, worst {float((err / tol).max()):.3g} tolerances"
    empty = torch.isinf(rlse)
    assert torch.equal(torch.isinf(lse), empty) and torch.equal(lse[empty].double(), rlse[empty])
    off = (lse.double() - rlse).abs()[~empty]
    lim = (rel * 1.4427 + 2.0 ** -23 * (rlse.abs() + 1))[~empty]
    assert (off <= lim).all(), f"lse: worst {float((off / lim).max()):.3g} tolerances"


def run_check(a, **more):
    o, lse = paged_decode.run(**on_gpu(a), **more)
    check(a, o, lse, **more)
    return o, lse


TYPES = [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, E4M3)]
RAGGED = [1, 15, 16, 17, 0, 33, 100, 547]


@pytest.mark.parametrize("dtype,kind", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hk,group", [(8, 4), (1, 1), (1, 8), (2, 3), (3, 7), (2, 16), (1, 20), (5, 2)])
def test_heads_sizes_types(built_lib, hk, group, dim, dtype, kind):
    run_check(make(RAGGED, hk, group, dim, dtype, kind, 16, seed=hk * group + dim))


@pytest.mark.parametrize("dtype,kind", TYPES)
@pytest.mark.parametrize("hk,group,dim", [(8, 4, 128), (4, 9, 64), (2, 5, 256)])
@pytest.mark.parametrize("batch,longest,window", [(1, 31, 0), (9, 65, 0), (130, 65, 0), (1, 255, 0), (30, 257, 0), (9, 512, 0), (1, 513, 0),
                                                  (24, 300, 130), (1, 700, 130)])
def test_short_tables_of_several_heads(built_lib, batch, longest, window, hk, group, dim, dtype, kind):
    """The warps of a CTA share a pair's tiles, take a pair each, or split the batch into shares, by what the table can hold."""
    lens = [longest - (i * 37) % (longest + 1) for i in range(batch)]
    run_check(make(lens, hk, group, dim, dtype, kind, 16 if batch % 2 else 5, seed=longest + batch), **({"window": window} if window else {}))


@pytest.mark.parametrize("dtype,kind", TYPES)
@pytest.mark.parametrize("ps", [1, 2, 7, 16, 24, 64, 100])
def test_page_sizes_end_inside_a_tile(built_lib, ps, dtype, kind):
    run_check(make([1, ps, ps + 1, 3 * ps - 1, 200, 16, 15], 2, 4, 128, dtype, kind, ps, seed=ps))


@pytest.mark.parametrize("dtype,kind", TYPES)
@pytest.mark.parametrize("lens", [[1], [16], [2100], [8192], [5000, 3], [40] * 300, [1] * 500, [3000] + [5] * 250 + [0] * 30, [0, 0], [0]])
def test_lengths(built_lib, lens, dtype, kind):
    run_check(make(lens, 2, 4, 64, dtype, kind, 16, seed=len(lens) + sum(lens)))


@pytest.mark.parametrize("dtype,kind", TYPES)
@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 1000, 5000])
def test_window(built_lib, window, dtype, kind):
    run_check(make([1, 15, 16, 17, 0, 33, 100, 547, 2500], 2, 4, 64, dtype, kind, 16, seed=window), window=window)


@pytest.mark.parametrize("dtype,kind", TYPES)
def test_strides(built_lib, dtype, kind):
    """Pages of whole heads, keys and values side by side, a slice of the heads, scales turned, a q and a table that
    are views."""
    a = make([100, 33, 0, 260], 4, 4, 64, dtype, kind, 16, seed=9, layout="heads")
    o, lse = run_check(a)
    d = on_gpu(a)
    both = torch.empty((d["k_cache"].shape[0], 2) + d["k_cache"].shape[1:], dtype=kind, device="cuda")
    both[:, 0].copy_(d["k_cache"])
    both[:, 1].copy_(d["v_cache"])
    d["k_cache"], d["v_cache"] = both[:, 0], both[:, 1]
    if kind == E4M3:
        d["k_scale"] = d["k_scale"].permute(2, 1, 0).contiguous().permute(2, 1, 0)
    wide = torch.zeros(4, 16, 128, dtype=dtype, device="cuda")
    wide[..., 32:96] = d["q"]
    d["q"] = wide[..., 32:96]
    table = torch.full((d["block_table"].shape[1], 4), -1, dtype=torch.int32, device="cuda")
    table.copy_(d["block_table"].T)
    d["block_table"] = table.T
    o2, lse2 = paged_decode.run(**d)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    part = {**d, "k_cache": d["k_cache"][:, :, 1:3], "v_cache": d["v_cache"][:, :, 1:3], "q": d["q"][:, 4:12]}
    if kind == E4M3:
        part.update(k_scale=d["k_scale"][:, :, 1:3], v_scale=d["v_scale"][:, :, 1:3])
    o3, lse3 = paged_decode.run(**part)
    assert torch.allclose(o3.float(), o2[:, 4:12].float(), rtol=torch.finfo(dtype).eps * 2, atol=1e-5)


@pytest.mark.parametrize("dtype,kind", TYPES)
def test_bad_pages_are_not_visible(built_lib, dtype, kind):
    a = make([100, 64, 40, 500], 2, 4, 128, dtype, kind, 16, seed=12)
    pages = a["k_cache"].shape[0]
    a["block_table"][0, 2] = -1
    a["block_table"][0, 0] = pages
    a["block_table"][1, :] = -5                     # none left: o = 0, lse = -inf
    a["block_table"][3, -1] = 2 ** 31 - 1
    run_check(a)
    a["seq_lens"][2] = 10 ** 9                      # longer than the table: what the table has
    a["seq_lens"][0] = -3
    d = on_gpu(a)
    o, lse = paged_decode.run(**d)
    clipped = dict(a, seq_lens=a["seq_lens"].clamp(0, a["block_table"].shape[1] * 16))
    check(clipped, o, lse)


@pytest.mark.parametrize("dtype,kind", TYPES)
def test_what_lies_behind_the_end_does_not_matter(built_lib, dtype, kind):
    """NaN and infinities in the slots behind a sequence, in free pages and in front of a window."""
    a = make([5, 100, 33, 700], 2, 4, 64, dtype, kind, 16, seed=13)
    want = run_check(a, window=50)
    seen = torch.zeros(a["k_cache"].shape[:2], dtype=torch.bool)
    for b, n in enumerate(a["seq_lens"].tolist()):
        for t in range(max(0, n - 50), n):
            seen[a["block_table"][b, t // 16], t % 16] = True
    for name, bad in (("k_cache", float("nan")), ("v_cache", float("nan")), ("v_cache", float("inf")), ("k_cache", float("-inf"))):
        c = a[name].float()
        c[~seen] = bad
        b = dict(a)
        b[name] = c.to(kind)
        if kind == E4M3:
            for s in ("k_scale", "v_scale"):
                b[s] = a[s].clone()
                b[s][~seen] = bad
        o, lse = paged_decode.run(**on_gpu(b), window=50)
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_infinite_values_and_scores(built_lib, dtype):
    a = make([40, 3, 200], 1, 4, 64, dtype, dtype, 16, seed=14)
    at = lambda b, t: (int(a["block_table"][b, t // 16]), t % 16, 0)  # noqa: E731
    a["v_cache"][at(0, 39)][5] = float("inf")
    a["v_cache"][at(2, 0)][6] = float("-inf")
    a["v_cache"][at(2, 7)][9] = float("nan")
    o, lse = paged_decode.run(**on_gpu(a))
    ro, rlse, *_ = oracle.paged.paged_decode(**a)
    o = o.cpu()
    assert torch.equal(torch.isnan(o), torch.isnan(ro)) and torch.equal(torch.isinf(o), torch.isinf(ro))
    assert torch.equal(o[torch.isinf(ro)].double(), ro[torch.isinf(ro)])
    # keys that score minus infinity weigh nothing, whatever their values are; with all of them so there is nothing
    a = make([40, 3, 200], 1, 4, 64, dtype, dtype, 16, seed=15)
    a["q"].abs_()
    for b, ts in ((0, range(0, 40, 3)), (1, range(3)), (2, range(0, 100))):
        for t in ts:
            a["k_cache"][at(b, t)] = float("-inf")
    run_check(a)


def test_e4m3_codes(built_lib):
    """Every code, subnormals and NaN too, as a key and as a value."""
    codes = torch.arange(256, dtype=torch.uint8).view(E4M3)
    a = make([1] * 256, 1, 1, 64, BF16, E4M3, 1, seed=16, extra=0)
    a["k_scale"].fill_(1.0)
    a["v_scale"].fill_(1.0)
    for b in range(256):
        page = a["block_table"][b, 0]
        a["v_cache"][page, 0, 0] = codes.roll(b)[:64].float().nan_to_num(0.0).to(E4M3)
        a["k_cache"][page, 0, 0] = codes.roll(-b)[:64].float().nan_to_num(0.0).to(E4M3)
    run_check(a)
    o, _ = paged_decode.run(**on_gpu(a))
    for b in range(256):                                     # one key: the output is its value
        assert torch.equal(o[b, 0].cpu(), a["v_cache"][a["block_table"][b, 0], 0, 0].to(BF16))
    a["v_cache"][a["block_table"][7, 0], 0, 0, 3] = float("nan")
    a["k_cache"][a["block_table"][9, 0], 0, 0, 3] = float("nan")
    o, lse = paged_decode.run(**on_gpu(a))
    assert torch.isnan(o[7, 0, 3]) and int(torch.isnan(o[7]).sum()) == 1
    assert torch.isnan(o[9]).all() and torch.isnan(lse[9]).all() and int(torch.isnan(lse).sum()) == 1


@pytest.mark.parametrize("dtype,kind", TYPES)
def test_one_key_above_a_long_tail(built_lib, dtype, kind):
    """One key that scores 17 above thousands of others which together weigh something: weights far below the
    smallest that 16 bits next to 1 hold."""
    a = make([8000], 1, 2, 64, dtype, kind, 16, seed=17)
    a["q"].fill_(1.0)
    k = torch.zeros(a["k_cache"].shape)
    k[int(a["block_table"][0, 0]), 0, 0] = 2.25              # 64 * 2.25 / 8 = 18 in the exponent
    a["k_cache"] = k.to(kind)
    if kind == E4M3:
        a["k_scale"].fill_(1.0)
    run_check(a)


def test_large_offsets(built_lib):
    """A cache of more than 2^32 bytes, its last pages used."""
    pages, ps, hk, dim = 40000, 64, 8, 64
    k = torch.zeros(pages, 2, ps, hk, dim, dtype=BF16, device="cuda")     # 5.2 GB
    assert k.numel() * 2 > 2 ** 32
    a = make([150, 64], 8, 2, 64, BF16, BF16, 64, seed=18, extra=0)
    d = on_gpu(a)
    n = a["k_cache"].shape[0]
    k[pages - n:, 0] = d["k_cache"]
    k[pages - n:, 1] = d["v_cache"]
    d["block_table"] = torch.where(d["block_table"] >= 0, d["block_table"] + (pages - n), d["block_table"])
    d["k_cache"], d["v_cache"] = k[:, 0], k[:, 1]
    o, lse = paged_decode.run(**d)
    check(a, o, lse)


def test_repeats_to_the_bit_and_captures(built_lib):
    a = make([3000, 17, 0, 900, 8000], 2, 4, 128, BF16, BF16, 16, seed=19)
    d = on_gpu(a)
    o, lse = paged_decode.run(**d)
    for _ in range(3):
        o2, lse2 = paged_decode.run(**d)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go, glse = paged_decode.run(**d)
    d["q"].normal_()
    d["seq_lens"].copy_(torch.tensor([10, 17, 0, 40, 7999], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    o, lse = paged_decode.run(**d)
    assert torch.equal(go, o) and torch.equal(glse, lse)


def test_two_graphs_of_one_pool(built_lib):
    """Two captured calls that may share a workspace, replayed in turn on one stream."""
    a, b = (on_gpu(make([2000, 300], 2, 4, 64, BF16, BF16, 16, seed=20 + i)) for i in range(2))
    want = [paged_decode.run(**x) for x in (a, b)]
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for x in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(paged_decode.run(**x))
        pool = graph.pool()
        graphs.append(graph)
    for i in (1, 0):
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])


def test_a_query_that_is_not_aligned(built_lib):
    a = make([100, 33], 2, 4, 64, BF16, BF16, 16, seed=23)
    d = on_gpu(a)
    o, lse = paged_decode.run(**d)
    flat = torch.zeros(a["q"].numel() + 3, dtype=BF16, device="cuda")
    flat[3:] = d["q"].flatten()
    d["q"] = flat[3:].view(a["q"].shape)
    assert d["q"].data_ptr() % 16 != 0
    o2, lse2 = paged_decode.run(**d)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_no_cache_no_table_no_batch(built_lib):
    q = torch.randn(3, 4, 64, device="cuda").to(BF16)
    none = torch.zeros(0, 16, 2, 64, dtype=BF16, device="cuda")
    some = torch.randn(4, 16, 2, 64, device="cuda").to(BF16)
    table, lens = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.full((3,), 20, dtype=torch.int32, device="cuda")
    for k, t in ((none, table), (some, table[:, :0]), (none, table[:, :0])):
        o, lse = paged_decode.run(q, k, k, t, lens, 0.1)
        assert (o == 0).all() and torch.isinf(lse).all()
    o, lse = paged_decode.run(q[:0], some, some, table[:0], lens[:0], 0.1)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_many_heads(built_lib):
    """More pairs of KV heads and query blocks than CTAs are resident."""
    run_check(make([17, 40], 48, 17, 64, FP16, FP16, 16, seed=24))
    run_check(make([100], 1, 300, 64, BF16, E4M3, 7, seed=25))


def test_two_host_threads_two_streams(built_lib):
    import threading
    cases = [make([900, 64, 1200, 0], 2, 4, 128, BF16, kind, 16, seed=26) for kind in (BF16, E4M3)]
    dev = [on_gpu(a) for a in cases]
    torch.cuda.synchronize()
    results, errors = [None, None], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    out = paged_decode.run(**dev[i])
            s.synchronize()
            results[i] = out
        except Exception as e:  # surfaced in the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, out in zip(cases, results):
        check(a, *out)


def test_agrees_with_gqa_decode(built_lib):
    from ako4x_b200 import gqa_decode, workloads as W
    w = W.make_gqa_decode(5, shape_id=7, device="cuda", lens=[300, 1, 17, 2000, 64], extra_pages=9)
    lens = (w["kv_indptr"][1:] - w["kv_indptr"][:-1]).int()
    table = torch.full((5, int(lens.max())), -1, dtype=torch.int32, device="cuda")
    for b in range(5):
        table[b, :lens[b]] = w["kv_indices"][w["kv_indptr"][b]:w["kv_indptr"][b + 1]]
    ro, rlse = gqa_decode.run(w["q"], w["k_cache"], w["v_cache"], w["kv_indptr"], w["kv_indices"], w["sm_scale"])
    o, lse = paged_decode.run(w["q"], w["k_cache"], w["v_cache"], table, lens, w["sm_scale"])
    assert torch.allclose(lse, rlse, atol=1e-4)
    assert torch.allclose(o.float(), ro.float(), rtol=2.0 ** -7, atol=1e-4)     # a bf16 step each
