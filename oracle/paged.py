"""CPU oracle (test infrastructure) of the operators around a paged cache, in 64 bits, written from
their formulas; the reference has no counterpart of them.

The functions of rows also return, per element, the sum of the magnitudes that went into it, and
``paged_decode`` the mean magnitude of the values and of the products in a score: what a tolerance in fp32
has to be taken relative to."""
import torch

E4M3_MAX = 448.0


def rotate(x, positions, inv_freq, interleaved=False, attention_factor=1.0):
    """x [tokens, heads, dim] -> (rotated, sum of the magnitudes), fp64."""
    x = x.double()
    half = inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.double()[None, :]
    c, s = (angle.cos() * attention_factor)[:, None], (angle.sin() * attention_factor)[:, None]
    y, size = x.clone(), x.abs()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        ci, si = c[..., i], s[..., i]
        y[..., a] = x[..., a] * ci - x[..., b] * si
        y[..., b] = x[..., b] * ci + x[..., a] * si
        size[..., a] = (x[..., a] * ci).abs() + (x[..., b] * si).abs()
        size[..., b] = (x[..., b] * ci).abs() + (x[..., a] * si).abs()
    return y, size


def head_norm(x, weight, eps=1e-6):
    x = x.double()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()


def quantize_rows(x):
    """Rows of fp32 values -> (e4m3, fp32 scale per row) by the library's rule."""
    x = x.float()
    top = x.abs().amax(-1)
    scale = torch.where(top > 1e-10, top / E4M3_MAX, torch.ones_like(top))
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def paged_decode(q, k_cache, v_cache, block_table, seq_lens, sm_scale, k_scale=None, v_scale=None, window=0):
    """(o, lse, mean magnitude of the values [batch, heads, dim], largest sum of a score's magnitudes [batch,
    heads]), fp64. Keys whose score is minus infinity weigh nothing."""
    batch, hq, dim = q.shape
    pages, page_size, hk, _ = k_cache.shape
    o = torch.zeros(batch, hq, dim, dtype=torch.float64)
    lse = torch.full((batch, hq), float("-inf"), dtype=torch.float64)
    size, score_size = torch.zeros_like(o), torch.zeros_like(lse)
    for b in range(batch):
        n = min(max(int(seq_lens[b]), 0), block_table.shape[1] * page_size)
        seen = []
        for t in range(max(0, n - window) if window else 0, n):
            page = int(block_table[b, t // page_size])
            if 0 <= page < pages:
                seen.append((page, t % page_size))
        if not seen:
            continue
        page, slot = torch.tensor(seen).T
        for h in range(hq):
            kv = h // (hq // hk)
            k, v = k_cache[page, slot, kv].double(), v_cache[page, slot, kv].double()
            if k_scale is not None:
                k, v = k * k_scale[page, slot, kv].double()[:, None], v * v_scale[page, slot, kv].double()[:, None]
            s = k @ q[b, h].double() * sm_scale
            live = s != float("-inf")
            if not live.any():
                continue
            s, v = s[live], v[live]
            p = torch.exp(s - s.max())
            o[b, h] = (p[:, None] * v).sum(0) / p.sum()
            lse[b, h] = (s.max() + torch.log(p.sum())) / torch.log(torch.tensor(2.0, dtype=torch.float64))
            size[b, h] = (p[:, None] * v.abs()).sum(0) / p.sum()
            score_size[b, h] = (k.abs() @ q[b, h].double().abs()).max() * abs(sm_scale)
    return o, lse, size, score_size


class Pages:
    """The pages' bookkeeping, one entry after the other. ``table`` [rows, max_pages], ``lens``, ``refs``."""

    def __init__(self, rows, max_pages, pages, page_size):
        self.table = torch.full((rows, max_pages), -1, dtype=torch.int32)
        self.lens = torch.zeros(rows, dtype=torch.int32)
        self.refs = torch.zeros(pages, dtype=torch.int32)
        self.page_size = page_size

    def held(self, tokens):
        return -(-tokens // self.page_size)

    def extend(self, rows, add):
        fresh, taken, seen, ok = [p for p, r in enumerate(self.refs.tolist()) if r == 0], 0, set(), []
        for row, n in zip(rows, add):
            good = 0 <= row < len(self.lens) and row not in seen and n >= 0
            if 0 <= row < len(self.lens):
                seen.add(row)
            if good:
                old, now = self.held(int(self.lens[row])), self.held(int(self.lens[row]) + n)
                good = now <= self.table.shape[1]
            if good:
                mine = fresh[taken:taken + now - old]
                taken += now - old
                good = len(mine) == now - old
            if good:
                for j, page in enumerate(mine):
                    self.table[row, old + j] = page
                    self.refs[page] = 1
                self.lens[row] += n
            ok.append(good)
        return ok

    def free(self, rows):
        for row in rows:
            if 0 <= row < len(self.lens):
                for j in range(self.held(int(self.lens[row]))):
                    self.refs[self.table[row, j]] -= 1
                    self.table[row, j] = -1
                self.lens[row] = 0

    def fork(self, caches, parents, children):
        fresh, taken, seen, ok = [p for p, r in enumerate(self.refs.tolist()) if r == 0], 0, set(), []
        lens = self.lens.clone()
        for parent, child in zip(parents, children):
            rows = len(self.lens)
            good = 0 <= parent < rows and 0 <= child < rows and child not in seen and int(lens[child]) == 0
            if 0 <= child < rows:
                seen.add(child)
            if good:
                n = int(lens[parent])
                full, part = divmod(n, self.page_size)
                if part:
                    taken += 1
                    good = taken <= len(fresh)
            if good:
                for j in range(full):
                    self.table[child, j] = self.table[parent, j]
                    self.refs[self.table[parent, j]] += 1
                if part:
                    page = fresh[taken - 1]
                    self.table[child, full] = page
                    self.refs[page] = 1
                    for c in caches:
                        c[page] = c[int(self.table[parent, full])]
                self.lens[child] = n
            ok.append(good)
        return ok

    def compact(self, caches):
        used = [p for p, r in enumerate(self.refs.tolist()) if r > 0]
        page_map = torch.full_like(self.refs, -1)
        for p in used:
            page_map[p] = p
        holes = [p for p in range(len(used)) if int(self.refs[p]) <= 0]
        for src, dst in zip([p for p in reversed(used) if p >= len(used)], holes):
            page_map[src] = dst
            self.refs[dst], self.refs[src] = int(self.refs[src]), 0
            for c in caches:
                c[dst] = c[src]
        for i, page in enumerate(self.table.flatten().tolist()):
            if 0 <= page < len(self.refs) and int(page_map[page]) >= 0:
                self.table.view(-1)[i] = page_map[page]
        return page_map
