"""The serving step that the documentation shows, run as it stands."""
import re
import textwrap
from pathlib import Path

import pytest
import torch

import oracle
from ako4x_b200 import kv_pages

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
E4M3 = torch.float8_e4m3fn


def documented_step():
    blocks = [b for f in sorted(ROOT.glob("*.md")) for b in re.findall(r"```python\n(.*?)```", f.read_text(), re.S)]
    (step,) = [textwrap.dedent(b) for b in blocks if "kv_pages.extend(" in b]
    return step


@pytest.mark.parametrize("pages", [5, 4, 3])
def test_a_pool_that_runs_out(built_lib, pages):
    """Two rows that share two full pages want a token each, with a page left for one of them or none: what was there
    stays, and the row that got a page gets its token."""
    step = documented_step()
    hq, hk, dim, ps = 8, 2, 128, 4
    g = torch.Generator().manual_seed(pages)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    table = torch.full((5, 4), -1, dtype=torch.int32, device="cuda")
    lens, refs = i32(0, 0, 0, 0, 0), torch.zeros(pages, dtype=torch.int32, device="cuda")
    caches = [torch.randn(pages, ps, hk, dim, generator=g).to(E4M3).cuda() for _ in range(2)]
    scales = [torch.rand(pages, ps, hk, generator=g).cuda() for _ in range(2)]
    assert kv_pages.extend(table, lens, refs, i32(0, 2), i32(2 * ps, 1), ps).tolist() == [True] * 2
    assert kv_pages.fork(caches + scales, table, lens, refs, i32(0), i32(1), ps).tolist() == [True]
    free = pages - 3
    before = [x.clone() for x in caches + scales]
    names = dict(table=table, lens=lens, refs=refs, rows=i32(0, 1), ones=i32(1, 1), page_size=ps, dim=dim,
                 k_cache=caches[0], v_cache=caches[1], k_scale=scales[0], v_scale=scales[1],
                 q_weight=torch.ones(dim, dtype=torch.bfloat16, device="cuda"), k_weight=torch.ones(dim, dtype=torch.bfloat16, device="cuda"),
                 parents=i32(0), children=i32(3), done=i32(2))
    for name, heads in (("q", hq), ("k", hk), ("v", hk)):
        names[name] = torch.randn(2, heads, dim, generator=g).to(torch.bfloat16).cuda()
    v = names["v"].cpu()
    exec(step, names)
    got = [i < free for i in range(2)]
    assert names["ok"].tolist() == got and lens[:2].tolist() == [2 * ps + x for x in got]
    taken = [int(table[i, 2]) for i in range(2) if got[i]]
    for x, y in zip(caches + scales, before):                # the pages that were in use
        assert torch.equal(x[:3].float(), y[:3].float())
    for i, page in enumerate(taken):
        codes, scale = oracle.paged.quantize_rows(v[i])
        assert torch.equal(caches[1][page, 0].cpu().view(torch.uint8), codes.view(torch.uint8)) and torch.equal(scales[1][page, 0].cpu(), scale)
    assert torch.isfinite(names["o"].float()).all() and names["o"].shape == (2, hq, dim)
