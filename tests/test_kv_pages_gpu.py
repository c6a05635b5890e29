"""The pages of a cache against a bookkeeping that takes one entry after the other; and a run of the
operators around a paged cache together."""
import pytest
import torch

import oracle
from ako4x_b200 import kv_pages, paged_decode, qk_norm_rope, rope

pytestmark = pytest.mark.gpu


def _caches(pages, ps, g):
    """Pages of several sizes and layouts: 16-bit rows, scales, single bytes, keys and values side by side."""
    both = torch.randn(pages, 2, ps, 2, 8, generator=g)
    return [torch.randn(pages, ps, 2, 64, generator=g).to(torch.bfloat16), torch.rand(pages, ps, 3, generator=g),
            torch.randint(0, 256, (pages, 37), generator=g, dtype=torch.uint8), both[:, 0], both[:, 1],
            torch.randn(pages, 3, ps, 16, generator=g).transpose(1, 2), torch.randn(pages, 5000, generator=g)]


class Pair:
    """The same state on the CPU (the oracle's) and on the GPU."""

    def __init__(self, rows, max_pages, pages, ps, seed):
        self.g = torch.Generator().manual_seed(seed)
        self.cpu = oracle.paged.Pages(rows, max_pages, pages, ps)
        self.caches = _caches(pages, ps, self.g)
        both = self.caches[3]._base.cuda()
        self.gpu_caches = [both[:, 0] if i == 3 else both[:, 1] if i == 4 else c.cuda() for i, c in enumerate(self.caches)]
        self.t, self.n, self.r = self.cpu.table.cuda(), self.cpu.lens.cuda(), self.cpu.refs.cuda()
        self.ps = ps

    def ints(self, lo, hi, n):
        return torch.randint(lo, hi, (n,), generator=self.g).int()

    def same(self):
        assert torch.equal(self.t.cpu(), self.cpu.table) and torch.equal(self.n.cpu(), self.cpu.lens)
        assert torch.equal(self.r.cpu(), self.cpu.refs)
        for a, b in zip(self.gpu_caches, self.caches):
            assert torch.equal(a.cpu(), b)

    def extend(self, rows, add):
        ok = kv_pages.extend(self.t, self.n, self.r, rows.cuda(), add.cuda(), self.ps)
        assert ok.tolist() == self.cpu.extend(rows.tolist(), add.tolist())

    def fork(self, parents, children):
        ok = kv_pages.fork(self.gpu_caches, self.t, self.n, self.r, parents.cuda(), children.cuda(), self.ps)
        assert ok.tolist() == self.cpu.fork(self.caches, parents.tolist(), children.tolist())

    def free(self, rows):
        kv_pages.free(self.t, self.n, self.r, rows.cuda(), self.ps)
        self.cpu.free(rows.tolist())

    def compact(self):
        page_map = kv_pages.compact(self.gpu_caches, self.t, self.r)
        assert torch.equal(page_map.cpu(), self.cpu.compact(self.caches))


@pytest.mark.parametrize("rows,max_pages,pages,ps", [(12, 5, 20, 4), (40, 9, 150, 16), (7, 3, 9, 1), (300, 4, 700, 3), (3, 2, 1, 5)])
def test_any_sequence_of_requests(built_lib, rows, max_pages, pages, ps):
    """Rows out of range, listed twice, too long, more than there are pages, empty parents, full children."""
    s = Pair(rows, max_pages, pages, ps, seed=rows + pages)
    for step in range(60):
        what = int(s.ints(0, 5, 1))
        n = int(s.ints(1, max(2, rows // 2), 1))
        if what <= 1:
            s.extend(s.ints(-1, rows + 1, n), s.ints(-1, max_pages * ps + 2, n))
        elif what == 2:
            s.fork(s.ints(-1, rows + 1, n), s.ints(-1, rows + 1, n))
        elif what == 3:
            s.free(s.ints(-1, rows + 1, n))
        else:
            s.compact()
        if step % 10 == 9 or step < 4:
            s.same()
    s.same()


def test_many_requests_and_many_pages(built_lib):
    """More requests than a planning CTA has threads, more pages than one of its steps or one tile of a compaction."""
    rows, pages = 3000, 40000
    s = Pair(rows, 24, pages, 2, seed=1)
    s.extend(torch.randperm(rows, generator=s.g).int(), s.ints(0, 40, rows))
    s.free(s.ints(0, rows, 1300))
    s.extend(s.ints(0, rows, 2500), s.ints(0, 9, 2500))
    s.same()
    empty = torch.nonzero(s.cpu.lens == 0).flatten().int()
    s.fork(s.ints(0, rows, len(empty)), empty)
    s.same()
    s.free(s.ints(0, rows, 2000))
    s.compact()
    s.same()


def test_pages_run_out_in_the_order_of_the_request(built_lib):
    s = Pair(6, 10, 10, 4, seed=2)
    s.extend(torch.tensor([0, 1, 2, 3], dtype=torch.int32), torch.tensor([16, 21, 4, 0], dtype=torch.int32))   # 4 + 6 pages of 10, then none
    assert s.cpu.lens.tolist() == [16, 21, 0, 0, 0, 0]
    s.fork(torch.tensor([0, 1, 0], dtype=torch.int32), torch.tensor([2, 3, 4], dtype=torch.int32))   # 1 needs a page and gets none
    assert s.cpu.lens.tolist() == [16, 21, 16, 0, 16, 0]
    s.same()


def test_nothing_to_do(built_lib):
    s = Pair(4, 3, 8, 4, seed=3)
    none = torch.empty(0, dtype=torch.int32)
    s.extend(none, none)
    s.fork(none, none)
    s.free(none)
    s.compact()
    assert kv_pages.copy(s.gpu_caches, none.cuda(), none.cuda()).tolist() == [True]
    s.same()
    t, n, r = (torch.zeros(k, dtype=torch.int32, device="cuda") for k in ((0, 3), (0,), (0,)))
    assert kv_pages.extend(t, n, r, none.cuda(), none.cuda(), 4).numel() == 0
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert kv_pages.extend(t, n, r, zero, zero, 4).tolist() == [False]
    assert kv_pages.compact([], t, r).numel() == 0


@pytest.mark.parametrize("pages,n", [(50, 20), (3000, 1400), (9, 1)])
def test_copy(built_lib, pages, n):
    g = torch.Generator().manual_seed(n)
    cpu = _caches(pages, 4, g)
    gpu = [c.cuda() for c in cpu]
    order = torch.randperm(pages, generator=g).int()
    src, dst = order[torch.randint(0, n, (n,), generator=g)], order[n:2 * n]      # a source may be named often
    src, dst = torch.cat([src, torch.tensor([-1, 3, pages, 5])]).int(), torch.cat([dst, torch.tensor([4, -2, 5, pages])]).int()
    own = order[0].view(1)                                                        # a page onto itself
    assert kv_pages.copy(gpu, torch.cat([src, own]).cuda(), torch.cat([dst, own]).cuda()).tolist() == [True]
    for a, b in zip(cpu, gpu):
        c = a.clone()
        c[dst[:n].long()] = a[src[:n].long()]
        assert torch.equal(b.cpu(), c)


@pytest.mark.parametrize("src,dst", [([0, 1], [5, 5]), ([0, 5], [5, 6]), ([5, 0], [6, 5]), ([0, 1], [1, 0]), ([0, 0, 3], [1, 2, 1])])
def test_copy_refuses_a_list_that_depends_on_the_order(built_lib, src, dst):
    gpu = [torch.randn(8, 100, device="cuda")]
    before = gpu[0].clone()
    many = torch.arange(1000, 1000, dtype=torch.int32)
    assert kv_pages.copy(gpu, torch.tensor(src + many.tolist(), dtype=torch.int32).cuda(), torch.tensor(dst + many.tolist(), dtype=torch.int32).cuda()).tolist() == [False]
    assert torch.equal(gpu[0], before)


def test_more_caches_than_a_launch_takes(built_lib):
    g = torch.Generator().manual_seed(8)
    cpu = [torch.randn(40, 3 + i, generator=g) for i in range(150)]
    gpu = [c.cuda() for c in cpu]
    s = oracle.paged.Pages(10, 4, 40, 4)
    t, n, r = s.table.cuda(), s.lens.cuda(), s.refs.cuda()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    assert kv_pages.extend(t, n, r, i32(0, 1, 2), i32(14, 9, 3), 4).tolist() == s.extend([0, 1, 2], [14, 9, 3])
    assert kv_pages.fork(gpu, t, n, r, i32(0, 1, 2), i32(5, 6, 7), 4).tolist() == s.fork(cpu, [0, 1, 2], [5, 6, 7])
    kv_pages.free(t, n, r, i32(0, 1), 4)
    s.free([0, 1])
    assert torch.equal(kv_pages.compact(gpu, t, r).cpu(), s.compact(cpu))
    assert torch.equal(t.cpu(), s.table) and torch.equal(r.cpu(), s.refs)
    assert kv_pages.copy(gpu, i32(0, 1), i32(38, 39)).tolist() == [True]
    for a, b in zip(cpu, gpu):
        a[38], a[39] = a[0].clone(), a[1].clone()
        assert torch.equal(a, b.cpu())


def test_a_cache_of_one_number_per_page_and_one_page(built_lib):
    a, b = torch.arange(9., device="cuda"), torch.randn(9, 4, 6, device="cuda").transpose(1, 2)
    want = b.clone()
    want[7] = want[2]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    assert kv_pages.copy([a, b], i32(2), i32(7)).tolist() == [True]
    assert a[7] == 2 and torch.equal(b, want)
    one = torch.randn(1, 3, 5, device="cuda")
    table, lens, refs = torch.full((2, 1), -1, dtype=torch.int32).cuda(), i32(0, 0), i32(0)
    assert kv_pages.extend(table, lens, refs, i32(1), i32(3), 4).tolist() == [True]
    assert kv_pages.fork([one], table, lens, refs, i32(1), i32(0), 4).tolist() == [False]   # no second page
    assert kv_pages.compact([one], table, refs).tolist() == [0] and lens.tolist() == [0, 3]


@pytest.mark.parametrize("pages", [4096, 4097, 8192, 9000])
def test_compaction_at_the_edges_of_its_tiles(built_lib, pages):
    """Everything in use, nothing in use, all in front, all behind."""
    cache = torch.arange(pages, dtype=torch.float32, device="cuda").view(pages, 1).repeat(1, 4)
    for used in (range(0), range(pages), range(pages // 2), range(pages // 2, pages), range(0, pages, 2), range(pages - 1, pages)):
        refs = torch.zeros(pages, dtype=torch.int32)
        refs[list(used)] = 1
        s = oracle.paged.Pages(3, (len(used) + 2) // 3 + 1, pages, 1)
        s.refs = refs.clone()
        ids = torch.tensor(list(used), dtype=torch.int32)
        s.table.view(-1)[:len(used)] = ids[torch.randperm(len(used), generator=torch.Generator().manual_seed(1))]
        t, r, c = s.table.cuda(), refs.cuda(), cache.clone()
        before = c[t[t >= 0].long(), 0]
        mine = c.cpu()
        page_map = kv_pages.compact([c], t, r)
        assert torch.equal(page_map.cpu(), s.compact([mine]))
        assert torch.equal(t.cpu(), s.table) and torch.equal(r.cpu(), s.refs) and torch.equal(c.cpu(), mine)
        assert torch.equal(c[t[t >= 0].long(), 0], before)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float8_e4m3fn])
def test_a_serving_run(built_lib, kind):
    """Prompts come in, one is forked, tokens are added to all, a prompt leaves, the pool is compacted: after every step
    attention of the rows agrees with plain tensors of their keys and values."""
    g = torch.Generator().manual_seed(21)
    hq, hk, dim, ps, rows, max_pages, pages = 8, 2, 64, 8, 6, 8, 40
    fp8 = kind == torch.float8_e4m3fn
    kc, vc = (torch.zeros(pages, ps, hk, dim, device="cuda").to(kind) for _ in range(2))
    ks, vs = (torch.ones(pages, ps, hk, device="cuda") if fp8 else None for _ in range(2))
    caches = [kc, vc] + ([ks, vs] if fp8 else [])
    table = torch.full((rows, max_pages), -1, dtype=torch.int32, device="cuda")
    lens, refs = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(pages, dtype=torch.int32, device="cuda")
    w = (1 + 0.2 * torch.randn(2, dim, generator=g)).to(torch.bfloat16).cuda()
    f, factor = rope.frequencies(dim, scaling="yarn", factor=4.0, original_length=64)
    held = {r: (torch.zeros(0, hk, dim, dtype=torch.float64), torch.zeros(0, hk, dim, dtype=torch.float64)) for r in range(rows)}
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731

    def add(row_list, counts):
        before = lens.tolist()
        assert all(kv_pages.extend(table, lens, refs, i32(*row_list), i32(*counts), ps).tolist())
        row = torch.tensor(row_list).repeat_interleave(torch.tensor(counts)).cuda()
        pos = torch.cat([torch.arange(before[r], before[r] + c) for r, c in zip(row_list, counts)]).cuda()
        slots = table[row, pos // ps] * ps + pos % ps
        qkv = torch.randn(len(pos), (hq + 2 * hk) * dim, generator=g).to(torch.bfloat16).cuda()
        q, k, v = (x.view(len(pos), -1, dim) for x in qkv.split([hq * dim, hk * dim, hk * dim], dim=1))
        qo = qk_norm_rope.run_to_cache(q, k, v, w[0], w[1], pos, f, slots, kc, vc, ks, vs, 1e-6, True, factor)
        rk, _ = oracle.paged.rotate(oracle.paged.head_norm(k.cpu(), w[1].cpu()), pos.cpu(), f.cpu(), True, factor)
        for r in row_list:
            mine = (row == r).cpu()
            held[r] = (torch.cat([held[r][0], rk[mine]]), torch.cat([held[r][1], v.cpu().double()[mine]]))
        last = torch.tensor([int(torch.nonzero(row == r).max()) for r in row_list])
        attend(row_list, qo[last.cuda()])

    def attend(row_list, q):
        o, lse = paged_decode.run(q, kc, vc, table[row_list], lens[row_list], dim ** -0.5, ks, vs)
        for i, r in enumerate(row_list):
            k, v = (x.repeat_interleave(hq // hk, dim=1) for x in held[r])
            s = torch.einsum("hd,lhd->hl", q[i].cpu().double(), k) * dim ** -0.5
            ref = torch.einsum("hl,lhd->hd", torch.softmax(s, -1), v)
            # keys and values are rounded to 2^-9 (bf16) or 2^-4 and half a step below the normal ones (e4m3) of themselves:
            # a score of magnitude A in all moves by that much of A, the weights by twice as much at most, the values by the rest
            unit = 2.0 ** -4 if fp8 else 2.0 ** -8
            A = torch.einsum("hd,lhd->hl", q[i].cpu().double().abs(), k.abs()).amax(-1) * dim ** -0.5
            tol = (2 * unit * A + 2 * unit)[:, None] * v.abs().amax(0)
            assert ((o[i].cpu().double() - ref).abs() <= tol).all()
            assert torch.isfinite(lse[i]).all()
        return o

    add([0, 2, 3], [13, 24, 1])
    add([0, 2, 3], [1, 1, 1])
    assert kv_pages.fork(caches, table, lens, refs, i32(0, 2, 0), i32(4, 1, 5), ps).tolist() == [True] * 3
    for child, parent in ((4, 0), (1, 2), (5, 0)):
        held[child] = held[parent]
    add([0, 1, 2, 3, 4, 5], [1, 1, 1, 1, 1, 1])           # the copies go their own ways
    add([4, 5], [9, 2])
    kv_pages.free(table, lens, refs, i32(0, 2), ps)
    held[0] = held[2] = (torch.zeros(0, hk, dim, dtype=torch.float64), torch.zeros(0, hk, dim, dtype=torch.float64))
    q = torch.randn(4, hq, dim, generator=g).to(torch.bfloat16).cuda()
    before = attend([1, 3, 4, 5], q)
    kv_pages.compact(caches, table, refs)
    used = int((refs > 0).sum())
    assert (refs[:used] > 0).all() and int(table.max()) < used
    assert torch.equal(attend([1, 3, 4, 5], q), before)   # the same keys in other places
    add([0, 1], [30, 1])
    counts = torch.bincount(table[table >= 0].long(), minlength=pages)
    assert torch.equal(counts.int(), refs)


def test_a_captured_step(built_lib):
    """Free, extend and fork in a graph: replayed on a state, they do what the calls do."""
    pages, ps = 64, 4
    cache = torch.randn(pages, 300, device="cuda")
    table = torch.full((8, 6), -1, dtype=torch.int32, device="cuda")
    lens, refs = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(pages, dtype=torch.int32, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    rows, add, parents, children, out = i32(0, 1, 2), i32(5, 9, 3), i32(0, 1), i32(4, 5), i32(0, 1, 4, 5)

    def step():
        kv_pages.free(table, lens, refs, out, ps)
        a = kv_pages.extend(table, lens, refs, rows, add, ps)
        b = kv_pages.fork([cache], table, lens, refs, parents, children, ps)
        return a, b

    def state():
        return [x.clone() for x in (table, lens, refs, cache)]

    step()
    torch.cuda.synchronize()
    start = state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oks = step()
    for x, y in zip((table, lens, refs, cache), start):
        assert torch.equal(x, y)                          # capturing does nothing
    add.copy_(i32(1, 20, 4))
    graph.replay()
    torch.cuda.synchronize()
    got, got_ok = state(), [x.clone() for x in oks]
    for x, y in zip((table, lens, refs, cache), start):
        x.copy_(y)
    want_ok = step()
    for x, y in zip(got, state()):
        assert torch.equal(x, y)
    assert all(torch.equal(x, y) for x, y in zip(got_ok, want_ok))
