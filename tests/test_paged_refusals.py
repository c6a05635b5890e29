"""Refusals of the operators around a paged cache, the frequencies, and the oracle's own rules: nothing here
reaches a GPU. Every call is refused before a launch: by the checks of shapes and types, or, with good
ones, because the tensors are on the CPU."""
import ctypes
import math

import pytest
import torch

import oracle
from ako4x_b200 import _cabi, kv_pages, paged_decode, qk_norm_rope, rope

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
OK, EINVAL, ESHAPE, EWORKSPACE = 0, -1, -2, -4


def _refused(call, text):
    with pytest.raises(_cabi.Ako4xError, match=text):
        call()


# ---- rows ---------------------------------------------------------------------------------------

def _rows(tokens=3, hq=4, hk=2, dim=64, dtype=BF16):
    q, k = torch.zeros(tokens, hq, dim, dtype=dtype), torch.zeros(tokens, hk, dim, dtype=dtype)
    return q, k, torch.arange(tokens, dtype=torch.int32), torch.ones(dim // 2)


def test_rope_refusals(built_lib):
    q, k, pos, f = _rows()
    _refused(lambda: rope.run(q, k, pos, f), "CUDA")
    _refused(lambda: rope.run(q, None, pos, f), "CUDA")
    _refused(lambda: rope.run(q[0], k, pos, f), "tokens, heads, dim")
    _refused(lambda: rope.run(q, k[:2], pos, f), "same tokens")
    _refused(lambda: rope.run(q, k[..., :32], pos, f), "same tokens and dim")
    _refused(lambda: rope.run(q.float(), k.float(), pos, f), "bf16 or fp16")
    _refused(lambda: rope.run(q, k.half(), pos, f), "one type")
    _refused(lambda: rope.run(q, k, pos.float(), f), "positions")
    _refused(lambda: rope.run(q, k, pos[:2], f), "positions")
    _refused(lambda: rope.run(q, k, pos, f.double()), "inv_freq")
    _refused(lambda: rope.run(q, k, pos, torch.ones(33)), "rotary_dim <= dim")
    odd = torch.zeros(3, 4, 60, dtype=BF16)
    _refused(lambda: rope.run(odd, None, pos, f[:8]), "multiple of 8")
    wide = torch.zeros(3, 4, 264, dtype=BF16)
    _refused(lambda: rope.run(wide, None, pos, f[:8]), "multiple of 8")
    with pytest.raises(TypeError):
        rope.run(q, 3, pos, f)


def test_norm_refusals(built_lib):
    q, k, pos, f = _rows()
    w = torch.ones(64, dtype=BF16)
    _refused(lambda: qk_norm_rope.run(q, k, w, w, pos, f), "CUDA")
    _refused(lambda: qk_norm_rope.run(q, k, w[:32], w, pos, f), "weights")
    _refused(lambda: qk_norm_rope.run(q, k, w.half(), w, pos, f), "weights")
    _refused(lambda: qk_norm_rope.run(q, k, w, w.float(), pos, f), "one type")


def test_cache_refusals(built_lib):
    q, k, pos, f = _rows()
    w, slots = torch.ones(64, dtype=BF16), torch.arange(3, dtype=torch.int32)
    kc, vc = torch.zeros(2, 16, 2, 64, dtype=BF16), torch.zeros(2, 16, 2, 64, dtype=BF16)
    sc = torch.ones(2, 16, 2)

    def call(q=q, k=k, v=k, slots=slots, kc=kc, vc=vc, ks=None, vs=None):
        return lambda: qk_norm_rope.run_to_cache(q, k, v, w, w, pos, f, slots, kc, vc, ks, vs)

    _refused(call(), "CUDA")
    _refused(call(v=q), "same heads")
    _refused(call(slots=slots.float()), "slot_mapping")
    _refused(call(slots=slots[:2]), "slot_mapping")
    _refused(call(kc=kc.half(), vc=vc.half()), "rows' type or e4m3")
    _refused(call(kc=kc[:, :, :1], vc=vc[:, :, :1]), "k's heads")
    _refused(call(vc=vc[:1]), "caches")
    _refused(call(kc=kc.to(E4M3), vc=vc.to(E4M3)), "scales")
    _refused(call(ks=sc, vs=sc), "scales")
    _refused(call(kc=kc.to(E4M3), vc=vc.to(E4M3), ks=sc.half(), vs=sc), "scales")
    _refused(call(kc=kc.to(E4M3), vc=vc.to(E4M3), ks=sc[:, :8], vs=sc), "scales")
    strided = torch.zeros(2, 16, 2, 68, dtype=BF16)[..., :64]    # rows 136 bytes apart
    _refused(call(kc=strided), "16 bytes")
    turned = torch.zeros(2, 16, 64, 2, dtype=BF16).transpose(2, 3)
    _refused(call(vc=turned), "contiguous last dimension")


def test_nothing_is_copied_before_the_devices_are_checked(built_lib):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            ops.append(str(func))
            return func(*args, **(kwargs or {}))

    q, k, _, _ = _rows(dim=64)
    pos, f, w = torch.arange(6, dtype=torch.int32)[::2], torch.ones(64)[::2], torch.ones(128, dtype=BF16)[::2]
    off = torch.ones(65, dtype=BF16)[1:]
    slots, kc = torch.arange(3, dtype=torch.int32), torch.zeros(2, 16, 2, 64, dtype=BF16)
    for call in (lambda: rope.run(q, k, pos, f), lambda: qk_norm_rope.run(q, k, w, off, pos, f),
                 lambda: qk_norm_rope.run_to_cache(q, k, k, off, w, pos, f, slots, kc, kc)):
        ops = []
        with Seen():
            _refused(call, "CUDA")
        assert ops == []


@pytest.mark.parametrize("dim", [8, 24, 72, 104, 136, 248])
def test_e4m3_caches_of_rows_of_8_bytes(built_lib, dim):
    """Rows of any multiple of 8 are stored; decode reads 16 bytes at once."""
    q, k, pos, f = _rows(dim=dim)
    w, slots = torch.ones(dim, dtype=BF16), torch.arange(3, dtype=torch.int32)
    c, sc = torch.zeros(2, 16, 2, dim).to(E4M3), torch.ones(2, 16, 2)
    _refused(lambda: qk_norm_rope.run_to_cache(q, k, k, w, w, pos, f, slots, c, c, sc, sc), "CUDA")
    odd = torch.zeros(2, 16, 2, dim + 4).to(E4M3)[..., :dim]
    _refused(lambda: qk_norm_rope.run_to_cache(q, k, k, w, w, pos, f, slots, odd, c, sc, sc), "8 bytes")
    apart = torch.zeros(2, 16, 2, 72).to(E4M3)[..., :64]
    _refused(lambda: paged_decode.run(torch.zeros(2, 8, 64, dtype=BF16), apart, apart, torch.zeros(2, 3, dtype=torch.int32),
                                      torch.ones(2, dtype=torch.int32), 0.1, sc, sc), "16 bytes")


def test_rows_c_status(built_lib):
    L = _cabi.lib()
    raw = ctypes.create_string_buffer(4096)
    x = (ctypes.addressof(raw) + 255) & ~255
    rows = _cabi.HeadRows(x, 128, 64, 2)
    off = _cabi.HeadRows(x + 2, 128, 64, 2)
    odd = _cabi.HeadRows(x, 132, 66, 2)
    ref = ctypes.byref

    def call(q=rows, out=x, tokens=4, dim=64, rotary=64, dtype=0, freq=x):
        return L.ako4x_rope(ref(q), None, x, 0, freq, rotary, 0, 1.0, out, None, tokens, dim, dtype, None)

    assert call(tokens=0) == OK
    assert call(tokens=-1) == EINVAL
    assert call(dim=60) == ESHAPE and call(dim=264) == ESHAPE
    assert call(rotary=66) == ESHAPE and call(rotary=3) == ESHAPE
    assert call(dtype=2) == ESHAPE
    assert call(q=off) == EINVAL and call(q=odd) == EINVAL and call(out=x + 8) == EINVAL and call(out=None) == EINVAL
    assert call(freq=None) == EINVAL


def test_norm_c_status(built_lib):
    L = _cabi.lib()
    raw = ctypes.create_string_buffer(4096)
    x = (ctypes.addressof(raw) + 255) & ~255
    rows = _cabi.HeadRows(x, 128, 64, 2)
    ref = ctypes.byref

    def call(qw=x, kw=x, out=x, tokens=4):
        return L.ako4x_qk_norm_rope(ref(rows), ref(rows), qw, kw, 0, 1e-6, x, 0, x, 64, 0, 1.0, x, out, tokens, 64, 0, None)

    assert call(tokens=0) == OK
    assert call(qw=None) == EINVAL and call(kw=None) == EINVAL and call(out=None) == EINVAL
    assert call(qw=x + 2) == EINVAL and call(kw=x + 8) == EINVAL

    def store(kc, cdtype=0, slots=x, pages=8, qw=x):
        return L.ako4x_qk_norm_rope_cache(ref(rows), ref(rows), ref(rows), qw, x, 0, 1e-6, x, 0, x, 64, 0, 1.0, x, slots, 0, ref(kc),
                                          ref(kc), cdtype, pages, 16, 4, 64, 0, None)

    good = _cabi.KvCache(x, None, 2048, 128, 64, 0, 0, 0)
    assert store(good, slots=None) == EINVAL and store(good, pages=-1) == EINVAL and store(good, cdtype=1) == ESHAPE
    assert store(good, qw=x + 2) == EINVAL
    assert store(_cabi.KvCache(x + 8, None, 2048, 128, 64, 0, 0, 0)) == EINVAL
    assert store(_cabi.KvCache(x, None, 2048, 132, 66, 0, 0, 0)) == EINVAL
    assert store(good, cdtype=2) == EINVAL                  # e4m3 without scales


def test_frequencies():
    f, m = rope.frequencies(64, base=10000.0, device="cpu")
    i = torch.arange(32, dtype=torch.float64)
    assert m == 1.0 and torch.equal(f, (10000.0 ** (-i / 32)).float())
    g, m = rope.frequencies(64, scaling="linear", factor=4.0, device="cpu")
    assert m == 1.0 and torch.equal(g, (10000.0 ** (-i / 32) / 4).float())
    h, m = rope.frequencies(64, scaling="ntk", factor=4.0, device="cpu")
    assert h[0] == 1.0 and math.isclose(h[-1], f[-1] / 4, rel_tol=1e-6)
    y, m = rope.frequencies(64, scaling="yarn", factor=40.0, original_length=4096, device="cpu")
    assert math.isclose(m, 0.1 * math.log(40.0) + 1)
    turns = 4096 * f.double() / (2 * math.pi)
    assert torch.equal(y[turns > 33], f[turns > 33])
    assert torch.allclose(y[turns < 0.7], f[turns < 0.7] / 40, rtol=1e-6)
    assert (y <= f).all() and (y >= f / 40 * (1 - 1e-6)).all() and (y[1:] < y[:-1]).all()
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=64, scaling="other"),
                dict(rotary_dim=64, scaling="yarn", factor=4.0), dict(rotary_dim=64, factor=0.0),
                dict(rotary_dim=2, scaling="ntk", factor=2.0)):
        with pytest.raises(_cabi.Ako4xError):
            rope.frequencies(device="cpu", **bad)


@pytest.mark.parametrize("length,slow,fast,dim,base", [(6, 1.0, 32.0, 64, 1e4), (512, 100.0, 100.0, 64, 1e4), (4096, 1.0, 32.0, 8, 1e6), (4096, 1.0, 1.0, 128, 1e4),
                                                       (1, 1.0, 32.0, 2, 1e4), (10 ** 9, 1.0, 32.0, 64, 1e4)])
def test_yarn_keeps_and_divides_as_it_says(length, slow, fast, dim, base):
    f, _ = rope.frequencies(dim, base=base, device="cpu")
    y, _ = rope.frequencies(dim, base=base, scaling="yarn", factor=8.0, original_length=length, beta_fast=fast, beta_slow=slow, device="cpu")
    turns = length * f.double() / (2 * math.pi)
    assert torch.equal(y[turns > fast], f[turns > fast])
    assert torch.allclose(y[turns < slow], f[turns < slow] / 8, rtol=1e-6)
    assert (y <= f).all() and (y >= f / 8 * (1 - 1e-6)).all()


def test_yarn_refusals():
    for bad in (dict(beta_fast=0.5), dict(beta_slow=0.0), dict(beta_slow=-1.0), dict(beta_fast=float("nan"))):
        with pytest.raises(_cabi.Ako4xError, match="beta"):
            rope.frequencies(64, scaling="yarn", factor=4.0, original_length=4096, device="cpu", **bad)


def test_the_oracles_rotation_is_one():
    """Lengths stay, and a rotation back by the negative positions undoes it."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 2, 32, generator=g, dtype=torch.float64)
    f, _ = rope.frequencies(24, device="cpu")
    pos = torch.tensor([0, 1, 77, 4095, 900001])
    for interleaved in (False, True):
        y, size = oracle.paged.rotate(x, pos, f, interleaved)
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1)) and (size >= y.abs() * (1 - 1e-12)).all()
        back, _ = oracle.paged.rotate(y, -pos, f, interleaved)
        assert torch.allclose(back, x, atol=1e-9)


# ---- decode -------------------------------------------------------------------------------------

def test_decode_refusals(built_lib):
    q = torch.zeros(2, 8, 128, dtype=BF16)
    kc, vc = torch.zeros(4, 16, 2, 128, dtype=BF16), torch.zeros(4, 16, 2, 128, dtype=BF16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)

    def call(q=q, kc=kc, vc=vc, table=table, lens=lens, ks=None, vs=None, window=0):
        return lambda: paged_decode.run(q, kc, vc, table, lens, 0.1, ks, vs, window)

    _refused(call(), "CUDA")
    _refused(call(q=q[..., :96]), "64, 128 or 256")
    _refused(call(q=q.float()), "bf16 or fp16")
    _refused(call(q=q.half()), "rows' type or e4m3")
    _refused(call(q=q[:, :7]), "multiple")
    _refused(call(q=q[:, :0]), "multiple")
    _refused(call(vc=vc[:3]), "caches")
    _refused(call(kc=kc[..., :64]), "caches")
    _refused(call(table=table.long()), "block_table")
    _refused(call(table=table[:1]), "block_table")
    _refused(call(lens=lens[:1]), "seq_lens")
    _refused(call(window=-1), "window")
    _refused(call(kc=kc.to(E4M3), vc=vc.to(E4M3)), "scales")
    _refused(call(kc=torch.zeros(4, 16, 2, 132, dtype=BF16)[..., :128]), "16 bytes")


def test_decode_c_status(built_lib):
    L = _cabi.lib()
    raw = ctypes.create_string_buffer(4096)
    x = (ctypes.addressof(raw) + 255) & ~255
    ref = ctypes.byref
    cache = _cabi.KvCache(x, None, 4096, 256, 128, 0, 0, 0)
    off = _cabi.KvCache(x + 8, None, 4096, 256, 128, 0, 0, 0)

    def call(batch=2, hq=4, hk=2, dim=128, pages=8, dtype=0, cdtype=0, k=cache, ws=None, nbytes=0, window=0):
        return L.ako4x_paged_decode(x, ref(k), ref(cache), x, x, 0.1, window, x, x, batch, hq, hk, dim, pages, 16, 400, dtype, cdtype,
                                    ws, nbytes, None)

    assert call(batch=0) == OK
    assert call(batch=-1) == EINVAL and call(pages=-1) == EINVAL
    assert call(dim=96) == ESHAPE and call(hq=5) == ESHAPE and call(hk=0) == ESHAPE and call(cdtype=1) == ESHAPE
    assert call(window=-1) == ESHAPE
    assert call(k=off) == EINVAL
    assert call(cdtype=2) == EINVAL                         # e4m3 without scales
    assert call() == EWORKSPACE and call(ws=x, nbytes=16) == EWORKSPACE
    need = L.ako4x_paged_decode_workspace_bytes(2, 4, 2, 128, 400, 16, 0)
    assert need > 0 and call(ws=x + 8, nbytes=need) == EINVAL
    assert L.ako4x_paged_decode_workspace_bytes(2, 5, 2, 128, 4, 16, 0) == 0


def test_decode_plans_of_any_window(built_lib):
    """A window that no sequence reaches plans like none; a table of more tokens than are read like one of those."""
    L = _cabi.lib()
    need = lambda pages, ps, window, batch=1: L.ako4x_paged_decode_workspace_bytes(batch, 32, 8, 128, pages, ps, window)  # noqa: E731
    assert need(8192, 16, 0) > 0
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 62, 2 ** 63 - 17, 2 ** 63 - 16, 2 ** 63 - 1):
        assert need(8192, 16, window) == need(8192, 16, 0)
    assert need(8192, 16, 1000) == need(-(-1016 // 16), 16, 0)
    most = 2 ** 31 - 2
    assert need(most, most, 0, 64) == need(2 ** 20, 2 ** 11, 0, 64) > 0


def test_the_oracle_skips_bad_pages_and_empty_rows():
    g = torch.Generator().manual_seed(4)
    q = torch.randn(3, 2, 64, generator=g)
    k, v = torch.randn(4, 2, 1, 64, generator=g), torch.randn(4, 2, 1, 64, generator=g)
    table = torch.tensor([[1, -1, 2], [9, 9, 9], [0, 1, 2]], dtype=torch.int32)
    lens = torch.tensor([5, 6, 0], dtype=torch.int32)
    o, lse, *_ = oracle.paged.paged_decode(q, k, v, table, lens, 0.3)
    assert (o[1:] == 0).all() and torch.isinf(lse[1:]).all()
    keys = torch.cat([k[1], k[2][:1]])[:, 0].double()
    vals = torch.cat([v[1], v[2][:1]])[:, 0].double()
    p = torch.softmax(q[0].double() @ keys.T * 0.3, -1)
    assert torch.allclose(o[0], p @ vals)


# ---- pages --------------------------------------------------------------------------------------

def test_pages_refusals(built_lib):
    table, lens, refs = torch.full((4, 3), -1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)
    rows = torch.zeros(2, dtype=torch.int32)
    caches = [torch.zeros(8, 16, 2, 64, dtype=BF16)]
    _refused(lambda: kv_pages.extend(table, lens, refs, rows, rows, 16), "CUDA")
    _refused(lambda: kv_pages.free(table, lens, refs, rows, 16), "CUDA")
    _refused(lambda: kv_pages.fork(caches, table, lens, refs, rows, rows, 16), "CUDA")
    _refused(lambda: kv_pages.copy(caches, rows, rows), "CUDA")
    _refused(lambda: kv_pages.compact(caches, table, refs), "CUDA")
    _refused(lambda: kv_pages.extend(table.long(), lens, refs, rows, rows, 16), "int32 and contiguous")
    _refused(lambda: kv_pages.extend(table.T, lens, refs, rows, rows, 16), "contiguous")
    _refused(lambda: kv_pages.extend(table, lens[:3], refs, rows, rows, 16), "seq_lens")
    _refused(lambda: kv_pages.extend(table, lens, refs, rows, rows[:1], 16), "rows and add")
    _refused(lambda: kv_pages.extend(table, lens, refs, rows.long(), rows.long(), 16), "int32")
    _refused(lambda: kv_pages.extend(table, lens, refs, rows, rows, 0), "page_size")
    _refused(lambda: kv_pages.copy([], rows, rows), "no caches")
    _refused(lambda: kv_pages.copy(caches + [torch.zeros(7, 4)], rows, rows), "first dimension")
    _refused(lambda: kv_pages.fork([torch.zeros(7, 4)], table, lens, refs, rows, rows, 16), "first dimension")
    _refused(lambda: kv_pages.compact([torch.zeros(4, 8).T], table, refs), "one piece")
    _refused(lambda: kv_pages.copy([torch.zeros(1, 4).expand(8, 4)], rows, rows), "one piece")
    _refused(lambda: kv_pages.copy([torch.zeros(8, 3, 4).transpose(1, 2), torch.zeros(8), torch.zeros(8, 0)], rows, rows), "CUDA")
    _refused(lambda: kv_pages.copy([torch.zeros(8, 3, 4)[:, :, ::2]], rows, rows), "one piece")
    _refused(lambda: kv_pages.copy([torch.zeros(8, 1, 4).expand(8, 2, 4)], rows, rows), "one piece")
    with pytest.raises(TypeError):
        kv_pages.copy(3, rows, rows)


def test_pages_c_status(built_lib):
    L = _cabi.lib()
    raw = ctypes.create_string_buffer(4096)
    x = (ctypes.addressof(raw) + 255) & ~255
    one = (ctypes.c_void_p * 1)(x)
    size, stride, short = (ctypes.c_int64 * 1)(512), (ctypes.c_int64 * 1)(512), (ctypes.c_int64 * 1)(256)
    assert L.ako4x_kv_pages_extend(x, x, x, x, x, x, 0, 4, 4, 4, 16, None, 0, None) == OK
    assert L.ako4x_kv_pages_extend(x, x, x, x, x, x, 2, 4, 4, 4, 0, None, 0, None) == EINVAL
    assert L.ako4x_kv_pages_extend(x, x, x, x, x, x, 2, 4, 4, 4, 16, None, 0, None) == EWORKSPACE
    assert L.ako4x_kv_pages_extend(x + 1, x, x, x, x, x, 2, 4, 4, 4, 16, x, 4096, None) == EINVAL
    assert L.ako4x_kv_pages_free(x, x, x, x, 0, 4, 4, 4, 16, None) == OK
    assert L.ako4x_kv_pages_free(x, x, x, None, 1, 4, 4, 4, 16, None) == EINVAL
    assert L.ako4x_kv_pages_fork(one, size, short, 1, x, x, x, x, x, x, 2, 4, 4, 4, 16, x, 4096, None) == EINVAL
    assert L.ako4x_kv_pages_fork(one, size, stride, 1, x, x, x, x, x, x, 2, 4, 4, 4, 16, x, 16, None) == EWORKSPACE
    assert L.ako4x_kv_pages_copy(one, size, stride, 1, x, x, None, 2, 4, x, 4096, None) == EINVAL
    assert L.ako4x_kv_pages_copy(one, size, stride, 1, x, x, x, 5000, 4, None, 0, None) == EWORKSPACE
    assert L.ako4x_kv_pages_compact(one, size, stride, 1, x, x, x, 4, 4, 0, None, 0, None) == OK
    assert L.ako4x_kv_pages_compact(one, size, stride, 1, x, x, x, 4, 4, 4, None, 0, None) == EWORKSPACE
    assert L.ako4x_kv_pages_compact(one, size, stride, 1, x, x, x, -4, 4, 4, x, 4096, None) == EINVAL


def test_the_oracles_pages_keep_count():
    """Every count is the number of table entries that name the page, whatever is asked."""
    g = torch.Generator().manual_seed(5)
    s = oracle.paged.Pages(12, 5, 20, 4)
    draw = lambda n, hi: torch.randint(-1, hi, (n,), generator=g).tolist()  # noqa: E731
    for _ in range(200):
        what = int(torch.randint(0, 4, (1,), generator=g))
        if what == 0:
            s.extend(draw(3, 13), draw(3, 9))
        elif what == 1:
            s.fork([], draw(2, 12), draw(2, 13))
        elif what == 2:
            s.free(draw(2, 13))
        else:
            s.compact([])
            n = int((s.refs > 0).sum())
            assert (s.refs[:n] > 0).all() and (s.refs[n:] == 0).all()
        counts = torch.bincount(s.table[s.table >= 0].flatten().long(), minlength=20)
        assert torch.equal(counts.int(), s.refs)
