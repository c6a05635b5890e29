"""The operators that take new tokens into and through a paged key-value cache, as cases that can be
timed and compared: rotary positions, the norms of queries and keys with the rotation in the same pass
(and with keys and values stored into the cache), the pages of the cache, and attention of one new token
over it.

With ``own`` false, ``run`` computes an operator in its plain form, elementary torch operations in 32
bits (angles in 64) rounded once at the end; with ``own`` true it makes the calls that a user of the
library makes. ``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
LOG2E = 1.4426950408889634
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "fp16": 2, "e4m3": 1}


def listed():
    return [
        # One token of one user through a layer with 32 query and 8 key heads: a single short launch.
        {"name": "rope_t1", "op": "rope", "tokens": 1, "q_heads": 32, "k_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "dtype": "bf16", "max_position": 8192},
        # A prefill step of latent attention: the 64 rotary features of 16 query heads and of the one shared
        # key, pairs side by side, positions far into a long context.
        {"name": "rope_t8192_interleaved", "op": "rope", "tokens": 8192, "q_heads": 16, "k_heads": 1, "dim": 64,
         "rotary": 64, "interleaved": True, "dtype": "bf16", "max_position": 131072},
        # A decode step of 64 users: norms, rotation and the store into an 8-bit cache.
        {"name": "norm_t64_e4m3", "op": "norm", "tokens": 64, "q_heads": 32, "k_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "dtype": "bf16", "cache": "e4m3", "page_size": 16, "max_position": 8192},
        # A prefill step of 8192 tokens into a 16-bit cache.
        {"name": "norm_t8192", "op": "norm", "tokens": 8192, "q_heads": 32, "k_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "dtype": "bf16", "cache": "bf16", "page_size": 64, "max_position": 32768},
        # An odd number of tokens with wide heads of which a quarter is rotated, in fp16, kept by the caller.
        {"name": "norm_t969_partial", "op": "norm", "tokens": 969, "q_heads": 20, "k_heads": 4, "dim": 256, "rotary": 64,
         "interleaved": False, "dtype": "fp16", "cache": "none", "page_size": 16, "max_position": 1000000},
        # One user's chat at a few hundred tokens of context: the smallest attention call.
        {"name": "decode_b1", "op": "decode", "batch": 1, "max_len": 547, "kv_heads": 8, "group": 4, "dim": 128,
         "dtype": "bf16", "cache": "bf16", "page_size": 16, "window": 0},
        # A serving batch with ragged contexts up to 8192 tokens.
        {"name": "decode_b64", "op": "decode", "batch": 64, "max_len": 8192, "kv_heads": 8, "group": 4, "dim": 128,
         "dtype": "bf16", "cache": "bf16", "page_size": 16, "window": 0},
        # Twice the batch in an 8-bit cache: the largest case.
        {"name": "decode_b128_e4m3", "op": "decode", "batch": 128, "max_len": 8192, "kv_heads": 8, "group": 4, "dim": 128,
         "dtype": "bf16", "cache": "e4m3", "page_size": 64, "window": 0},
        # Three long documents, one wide key head for all of seven query heads, fp16.
        {"name": "decode_b3_long", "op": "decode", "batch": 3, "max_len": 131072, "kv_heads": 1, "group": 7, "dim": 256,
         "dtype": "fp16", "cache": "fp16", "page_size": 32, "window": 0},
        # A scheduling step: old requests leave, new ones enter, some of them are forked for a second answer.
        {"name": "pages_step", "op": "pages", "what": "step", "pages": 4096, "rows": 256, "max_len": 1024, "count": 16,
         "caches": 4, "kv_heads": 8, "dim": 128, "page_size": 16, "dtype": "bf16"},
        # Pages of eight layers copied for another holder.
        {"name": "pages_copy", "op": "pages", "what": "copy", "pages": 2048, "rows": 64, "max_len": 256, "count": 201,
         "caches": 16, "kv_heads": 8, "dim": 128, "page_size": 16, "dtype": "bf16"},
        # A pool of which half is in use, moved together: eight layers, half a gigabyte read and written.
        {"name": "pages_compact", "op": "pages", "what": "compact", "pages": 2048, "rows": 128, "max_len": 256, "count": 0,
         "caches": 16, "kv_heads": 8, "dim": 128, "page_size": 16, "dtype": "bf16"},
    ]


# ---- drawn cases --------------------------------------------------------------------------------

def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 5, 8, 16])
    return kv, kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])


def _draw(rng):
    op = rng.choice(["rope", "norm", "norm", "decode", "decode", "decode", "pages"])
    if op in ("rope", "norm"):
        kv, q = _heads(rng)
        dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
        c = {"op": op, "tokens": _log_int(rng, 1, 16384), "q_heads": q, "k_heads": kv, "dim": dim,
             "rotary": rng.choice([dim, dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.4,
             "dtype": rng.choice(["bf16", "bf16", "fp16"]), "max_position": _log_int(rng, 256, 1000000)}
        if op == "norm":
            c["cache"] = rng.choice(["none", c["dtype"], "e4m3"])
            c["page_size"] = rng.choice([1, 8, 16, 24, 64])
        return c
    if op == "decode":
        kv, q = _heads(rng)
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        return {"op": op, "batch": _log_int(rng, 1, 256), "max_len": _log_int(rng, 1, 65536), "kv_heads": kv,
                "group": q // kv, "dim": rng.choice([64, 128, 128, 256]), "dtype": dtype,
                "cache": rng.choice([dtype, "e4m3"]), "page_size": rng.choice([1, 7, 16, 32, 64]),
                "window": rng.choice([0, 0, 0, 128, 1000])}
    pages = _log_int(rng, 64, 8192)
    what = rng.choice(["step", "copy", "compact"])
    page_size = rng.choice([4, 16, 16, 64])
    return {"op": op, "what": what, "pages": pages, "rows": _log_int(rng, 4, 512), "max_len": page_size * _log_int(rng, 2, 64),
            "count": _log_int(rng, 1, max(1, pages // 4)), "caches": 2 * rng.randint(1, 8), "kv_heads": rng.choice([1, 2, 8]),
            "dim": rng.choice([64, 128]), "page_size": page_size, "dtype": rng.choice(["bf16", "e4m3"])}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def _padded(case):
    """Keys of the batch when every sequence is as long as the longest: what a plain form gathers."""
    return case["batch"] * case["max_len"] * case["kv_heads"] * case["dim"] if case["op"] == "decode" else 0


def draw(rng):
    largest = max(_cost(c) for c in listed())
    padded = max(_padded(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= largest and _padded(case) <= padded and _pool_bytes(case) <= 1 << 30:
            return case


# ---- what belongs to a case, whatever the seed --------------------------------------------------

def _of_case(case, what):
    return random.Random(" ".join([what] + ["%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"]))


def _lens(case):
    r = _of_case(case, "lens")
    return [r.randint(max(1, case["max_len"] // 64), case["max_len"]) for _ in range(case["batch"])]


def _visible(case):
    w = case["window"]
    return [min(n, w) if w else n for n in _lens(case)]


def _page_bytes(case):
    return case["page_size"] * case["kv_heads"] * case["dim"] * BYTES[case["dtype"]]


def _pool_bytes(case):
    return case["pages"] * case["caches"] * _page_bytes(case) if case["op"] == "pages" else 0


def _pool(case):
    """Lengths of the rows that hold something (half of the pool at most, the last `count` rows of a
    step are left empty) and what a step asks for."""
    r = _of_case(case, "pool")
    rows, ps = case["rows"], case["page_size"]
    lens, left = [0] * rows, case["pages"] // 2
    count = min(case["count"], max(1, rows // 4)) if case["what"] == "step" else 0
    for i in range(rows - 2 * count):
        n = r.randint(1, case["max_len"])
        if -(-n // ps) > left:
            break
        lens[i] = n
        left -= -(-n // ps)
    add = [r.randint(1, case["max_len"]) for _ in range(count)]
    parents = [r.randrange(rows - count) for _ in range(count)]
    return lens, add, parents, count


def work(case):
    op = case["op"]
    if op in ("rope", "norm"):
        t, q, k, d, b = case["tokens"], case["q_heads"], case["k_heads"], case["dim"], BYTES[case["dtype"]]
        cache = case.get("cache", "none")
        read = t * (q + k) * d * b + 4 * t + case["rotary"] * 2
        wrote = t * q * d * b
        if cache == "none":
            wrote += t * k * d * b
        else:
            read += t * k * d * b + 4 * t
            wrote += 2 * t * k * (d * BYTES[cache] + (4 if cache == "e4m3" else 0))
        return {"bytes": read + wrote, "flops": t * (q + k) * d * (7 if op == "norm" else 3)}
    if op == "decode":
        seen, b = sum(_visible(case)), case["batch"]
        heads = case["kv_heads"] * case["group"]
        per_key = case["kv_heads"] * 2 * (case["dim"] * BYTES[case["cache"]] + (4 if case["cache"] == "e4m3" else 0))
        return {"bytes": seen * per_key + 4 * seen // case["page_size"] + b * heads * (4 * case["dim"] + 4),
                "flops": 4 * seen * heads * case["dim"]}
    lens, add, parents, count = _pool(case)
    ps = case["page_size"]
    used = sum(-(-n // ps) for n in lens)
    table = case["rows"] * -(-case["max_len"] // ps) * 4
    if case["what"] == "copy":
        moved = min(case["count"], case["pages"] // 2)
        return {"bytes": 2 * moved * case["caches"] * _page_bytes(case) + 8 * moved, "flops": 0}
    if case["what"] == "compact":
        moved = used * (1 - used / case["pages"])   # pages lie anywhere in the pool
        return {"bytes": 2 * moved * case["caches"] * _page_bytes(case) + 3 * table + 8 * case["pages"], "flops": 0}
    all_lens = lens[: case["rows"] - 2 * count] + add
    moved = sum(all_lens[p] % ps != 0 for p in parents)
    return {"bytes": 2 * moved * case["caches"] * _page_bytes(case) + 4 * case["pages"] + 12 * count * -(-case["max_len"] // ps),
            "flops": 0}


# ---- inputs -------------------------------------------------------------------------------------

def _randn(shape, g, dtype, scale=1.0):
    """Normal values; one fp32 piece of a large tensor at a time."""
    out = torch.empty(shape, device=DEVICE, dtype=dtype)
    flat = out.view(-1)
    step = 1 << 28
    for at in range(0, flat.numel(), step):
        n = min(step, flat.numel() - at)
        x = torch.randn(n, generator=g, device=DEVICE).mul_(scale)
        flat[at:at + n] = (x.clamp_(-E4M3_MAX, E4M3_MAX) if dtype == torch.float8_e4m3fn else x).to(dtype)
    return out


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _prepare_rows(case, g):
    t, hq, hk, d = case["tokens"], case["q_heads"], case["k_heads"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    # queries, keys and values come out of one projection: views into its rows
    qkv = _randn((t, (hq + 2 * hk) * d), g, dtype)
    s = {"op": case["op"], "q": qkv[:, :hq * d].view(t, hq, d), "k": qkv[:, hq * d:(hq + hk) * d].view(t, hk, d),
         "interleaved": case["interleaved"], "attention_factor": 1.0}
    half = case["rotary"] // 2
    s["inv_freq"] = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).float().to(DEVICE)
    # runs of neighbouring tokens, each from a place of its own
    start = torch.randint(0, max(1, case["max_position"] - 512), (t // 512 + 1,), generator=g, device=DEVICE)
    s["positions"] = (start.repeat_interleave(512)[:t] + torch.arange(t, device=DEVICE) % 512).to(torch.int32)
    if case["op"] == "rope":
        return s
    s["q_weight"] = (1.0 + 0.1 * torch.randn(d, generator=g, device=DEVICE)).to(dtype)
    s["k_weight"] = (1.0 + 0.1 * torch.randn(d, generator=g, device=DEVICE)).to(dtype)
    s["eps"] = 1e-6
    s["cache"] = case["cache"]
    if case["cache"] == "none":
        return s
    s["v"] = qkv[:, (hq + hk) * d:].view(t, hk, d)
    ps = case["page_size"]
    pages = -(-t // ps) + 3
    order = torch.randperm(pages, generator=g, device=DEVICE)
    token = torch.arange(t, device=DEVICE)
    s["slot_mapping"] = (order[token // ps] * ps + token % ps).to(torch.int32)
    kind = DTYPES[case["cache"]]
    s["k_cache"] = torch.zeros((pages, ps, hk, d), device=DEVICE, dtype=kind)
    s["v_cache"] = torch.zeros((pages, ps, hk, d), device=DEVICE, dtype=kind)
    s["k_scale"] = s["v_scale"] = None
    if case["cache"] == "e4m3":
        s["k_scale"] = torch.ones((pages, ps, hk), device=DEVICE)
        s["v_scale"] = torch.ones((pages, ps, hk), device=DEVICE)
    return s


def _prepare_decode(case, g):
    b, hk, d, ps = case["batch"], case["kv_heads"], case["dim"], case["page_size"]
    lens = _lens(case)
    held = [-(-n // ps) for n in lens]
    pages = sum(held) + 5
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((b, max(held)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    dtype, kind = DTYPES[case["dtype"]], DTYPES[case["cache"]]
    s = {"op": "decode", "q": _randn((b, hk * case["group"], d), g, dtype), "block_table": table, "seq_lens": _ints(lens),
         "sm_scale": d ** -0.5, "window": case["window"], "k_scale": None, "v_scale": None}
    shape = (pages, ps, hk, d)
    if case["cache"] == "e4m3":
        s["k_cache"], s["v_cache"] = _randn(shape, g, kind, 150.0), _randn(shape, g, kind, 150.0)
        s["k_scale"] = torch.rand(shape[:3], generator=g, device=DEVICE).mul_(0.008).add_(0.002)
        s["v_scale"] = torch.rand(shape[:3], generator=g, device=DEVICE).mul_(0.008).add_(0.002)
    else:
        s["k_cache"], s["v_cache"] = _randn(shape, g, kind), _randn(shape, g, kind)
    return s


def _prepare_pages(case, g):
    ps, rows, pages = case["page_size"], case["rows"], case["pages"]
    lens, add, parents, count = _pool(case)
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((rows, -(-case["max_len"] // ps)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(lens):
        held = -(-n // ps)
        table[i, :held] = order[at:at + held]
        at += held
    refs = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
    refs[order[:at].long()] = 1
    stack = torch.empty((case["caches"], pages, ps, case["kv_heads"], case["dim"]), dtype=DTYPES[case["dtype"]], device=DEVICE)
    bits = stack.view(torch.uint8).view(-1)
    for i in range(0, bits.numel(), 1 << 28):   # any byte below 0x78 is part of a finite value
        n = min(1 << 28, bits.numel() - i)
        bits[i:i + n] = torch.randint(0, 0x78, (n,), generator=g, device=DEVICE, dtype=torch.uint8)
    # the caches come back as bytes: copies are equal or wrong
    s = {"op": "pages", "what": case["what"], "stack": stack, "bits": stack.view(torch.uint8), "caches": list(stack.unbind(0)), "page_size": ps,
         "block_table": table, "seq_lens": _ints(lens), "ref_counts": refs}
    if case["what"] == "copy":
        n = min(case["count"], pages // 2)
        s["src"], s["dst"] = order[:n].contiguous(), order[pages - n:].contiguous()
    if case["what"] == "step":
        s["new_rows"] = _ints(list(range(rows - 2 * count, rows - count)))
        s["children"] = _ints(list(range(rows - count, rows)))
        s["leaving"] = torch.cat([s["new_rows"], s["children"]])
        s["add"], s["parents"] = _ints(add), _ints(parents)
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    if case["op"] == "decode":
        return _prepare_decode(case, g)
    if case["op"] == "pages":
        return _prepare_pages(case, g)
    return _prepare_rows(case, g)


# ---- plain forms --------------------------------------------------------------------------------

def _plain_rotate(x, s):
    """x fp32 [tokens, heads, dim]."""
    half = s["inv_freq"].numel()
    turn = s["positions"].double()[:, None] * s["inv_freq"].double()[None, :]
    cos = (torch.cos(turn) * s["attention_factor"]).float()[:, None, :]
    sin = (torch.sin(turn) * s["attention_factor"]).float()[:, None, :]
    if s["interleaved"]:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([y, x[..., 2 * half:]], dim=-1)


def _plain_norm(x, w, eps):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.float()


def _plain_store(x, slots, cache, scale):
    """x fp32 [tokens, heads, dim] into the slots of a cache."""
    page, slot = slots.long() // cache.shape[1], slots.long() % cache.shape[1]
    if scale is not None:
        top = x.abs().amax(-1)
        sc = torch.where(top > 1e-10, top / E4M3_MAX, torch.ones_like(top))
        scale[page, slot] = sc
        x = x / sc[..., None]
    cache[page, slot] = x.to(cache.dtype)


def _plain_rows(s):
    dtype = s["q"].dtype
    if s["op"] == "rope":
        return _plain_rotate(s["q"].float(), s).to(dtype), _plain_rotate(s["k"].float(), s).to(dtype)
    q = _plain_rotate(_plain_norm(s["q"], s["q_weight"], s["eps"]), s).to(dtype)
    k = _plain_rotate(_plain_norm(s["k"], s["k_weight"], s["eps"]), s)
    if s["cache"] == "none":
        return q, k.to(dtype)
    _plain_store(k, s["slot_mapping"], s["k_cache"], s["k_scale"])
    _plain_store(s["v"].float(), s["slot_mapping"], s["v_cache"], s["v_scale"])
    return q, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _plain_gather(cache, scale, table):
    x = cache[table].float()
    if scale is not None:
        x = x * scale[table][..., None]
    return x.flatten(1, 2)   # [batch, keys, heads, dim]


def _plain_decode(s):
    q, (_, ps, hk, d) = s["q"], s["k_cache"].shape
    b, hq, _ = q.shape
    table = s["block_table"].long().clamp(min=0)
    k = _plain_gather(s["k_cache"], s["k_scale"], table)
    at, n = torch.arange(k.shape[1], device=q.device), s["seq_lens"][:, None]
    seen = at < n
    if s["window"]:
        seen = seen & (at >= n - s["window"])
    score = torch.einsum("bhgd,blhd->bhgl", q.float().view(b, hk, hq // hk, d), k) * s["sm_scale"]
    del k
    score = score.masked_fill(~seen[:, None, None, :], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = _plain_gather(s["v_cache"], s["v_scale"], table)
    o = torch.einsum("bhgl,blhd->bhgd", p, v)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + torch.log(total)).squeeze(-1) * LOG2E
    return o.reshape(b, hq, d).to(q.dtype), lse.reshape(b, hq)


def _plain_fresh(refs, need, valid):
    """The lowest free pages in the order of the request: (who gets them, all pages with the free ones in
    front, how many are taken before each)."""
    need = torch.where(valid, need, torch.zeros_like(need))
    upto = need.cumsum(0)
    ok = valid & ((need == 0) | (upto <= (refs == 0).sum()))
    return ok, torch.argsort((refs != 0).int(), stable=True), upto - need


def _plain_free(s, rows):
    table, lens, refs, ps = s["block_table"], s["seq_lens"], s["ref_counts"], s["page_size"]
    rows = rows.long()
    mine = table[rows]
    held = torch.arange(table.shape[1], device=table.device) < ((lens[rows] + ps - 1) // ps)[:, None]
    refs.scatter_add_(0, mine.clamp(min=0).flatten().long(), -held.flatten().int())
    table[rows] = torch.where(held, torch.full_like(mine, -1), mine)
    lens[rows] = torch.zeros_like(rows, dtype=torch.int32)


def _plain_extend(s, rows, add):
    table, lens, refs, ps = s["block_table"], s["seq_lens"], s["ref_counts"], s["page_size"]
    rows = rows.long()
    n = lens[rows]
    old, new = (n + ps - 1) // ps, (n + add + ps - 1) // ps
    ok, order, before = _plain_fresh(refs, new - old, new <= table.shape[1])
    at = torch.arange(table.shape[1], device=table.device)[None, :]
    fill = ok[:, None] & (at >= old[:, None]) & (at < new[:, None])
    page = order[(before[:, None] + at - old[:, None]).clamp(0, refs.numel() - 1)]
    refs.scatter_add_(0, page.flatten(), fill.flatten().int())
    table[rows] = torch.where(fill, page.int(), table[rows])
    lens[rows] = torch.where(ok, n + add, n)
    return ok


def _plain_fork(s, parents, children):
    table, lens, refs, ps = s["block_table"], s["seq_lens"], s["ref_counts"], s["page_size"]
    parents, children = parents.long(), children.long()
    n = lens[parents]
    full, part = n // ps, n % ps != 0
    ok, order, before = _plain_fresh(refs, part.int(), lens[children] == 0)
    page = order[before.clamp(max=refs.numel() - 1)]
    theirs = table[parents]
    at = torch.arange(table.shape[1], device=table.device)[None, :]
    shared = ok[:, None] & (at < full[:, None])
    fresh = (ok & part)[:, None] & (at == full[:, None])
    refs.scatter_add_(0, theirs.clamp(min=0).flatten().long(), shared.flatten().int())
    refs.scatter_add_(0, page, (ok & part).int())
    mine = torch.where(shared, theirs, torch.full_like(theirs, -1))
    table[children] = torch.where(fresh, page.int()[:, None], mine)
    lens[children] = torch.where(ok, n, torch.zeros_like(n))
    last = theirs.gather(1, full.long().clamp(max=table.shape[1] - 1)[:, None])[:, 0].long()
    copied = ok & part
    s["stack"][:, page[copied]] = s["stack"][:, last[copied]]
    return ok


def _plain_pages(s):
    if s["what"] == "copy":
        s["stack"][:, s["dst"].long()] = s["stack"][:, s["src"].long()]
        return s["bits"]
    if s["what"] == "step":
        _plain_free(s, s["leaving"])
        entered = _plain_extend(s, s["new_rows"], s["add"])
        forked = _plain_fork(s, s["parents"], s["children"])
        return entered, forked, s["block_table"], s["seq_lens"], s["ref_counts"], s["bits"]
    table, refs = s["block_table"].clone(), s["ref_counts"].clone()
    ids = torch.arange(refs.numel(), device=refs.device, dtype=torch.int32)
    used = refs > 0
    count = used.sum()
    src = torch.nonzero(used & (ids >= count)).flatten().flip(0)   # the highest page into the lowest hole
    dst = torch.nonzero(~used & (ids < count)).flatten()
    page_map = torch.where(used, ids, torch.full_like(ids, -1))
    page_map[src] = dst.int()
    s["stack"][:, dst] = s["stack"][:, src]
    to = page_map[table.clamp(min=0).long()]
    table = torch.where((table >= 0) & (to >= 0), to, table)
    refs[dst] = refs[src]
    refs[src] = 0
    return page_map, table, refs, s["bits"]


# ---- the library's operators --------------------------------------------------------------------

def _own_rows(s):
    from ako4x_b200 import qk_norm_rope, rope
    if s["op"] == "rope":
        return rope.run(s["q"], s["k"], s["positions"], s["inv_freq"], s["interleaved"], s["attention_factor"])
    if s["cache"] == "none":
        return qk_norm_rope.run(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"], s["eps"],
                                s["interleaved"], s["attention_factor"])
    q = qk_norm_rope.run_to_cache(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"],
                                  s["slot_mapping"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["eps"],
                                  s["interleaved"], s["attention_factor"])
    return q, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _own_decode(s):
    from ako4x_b200 import paged_decode
    return paged_decode.run(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"], s["sm_scale"],
                            s["k_scale"], s["v_scale"], s["window"])


def _own_pages(s):
    from ako4x_b200 import kv_pages
    if s["what"] == "copy":
        kv_pages.copy(s["caches"], s["src"], s["dst"])
        return s["bits"]
    table, lens, refs, ps = s["block_table"], s["seq_lens"], s["ref_counts"], s["page_size"]
    if s["what"] == "step":
        kv_pages.free(table, lens, refs, s["leaving"], ps)
        entered = kv_pages.extend(table, lens, refs, s["new_rows"], s["add"], ps)
        forked = kv_pages.fork(s["caches"], table, lens, refs, s["parents"], s["children"], ps)
        return entered, forked, table, lens, refs, s["bits"]
    table, refs = table.clone(), refs.clone()
    page_map = kv_pages.compact(s["caches"], table, refs)
    return page_map, table, refs, s["bits"]


def run(state):
    op = state["op"]
    if own:
        return _own_decode(state) if op == "decode" else _own_pages(state) if op == "pages" else _own_rows(state)
    return _plain_decode(state) if op == "decode" else _plain_pages(state) if op == "pages" else _plain_rows(state)


# ---- the definitions in 64 bits -----------------------------------------------------------------

def _exact_head_rows(x, weight, s):
    """Norm (where there is a weight) and rotation as a multiplication of complex numbers."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + s["eps"]).sqrt() * weight.double()
    half = s["inv_freq"].numel()
    angle = torch.outer(s["positions"].double(), s["inv_freq"].double())
    wheel = torch.polar(torch.full_like(angle, s["attention_factor"]), angle)[:, None, :]
    first = slice(0, 2 * half, 2) if s["interleaved"] else slice(0, half)
    second = slice(1, 2 * half, 2) if s["interleaved"] else slice(half, 2 * half)
    y = x.clone()
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * wheel
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_store(x, slots, cache, scale):
    """The cache after the store: in 8 bits the quotients before they are rounded."""
    flat = cache.double().flatten(0, 1)
    if scale is None:
        flat[slots.long()] = x
        return flat.view(cache.shape), None
    top = x.abs().max(-1).values
    sc = torch.where(top > 1e-10, top / E4M3_MAX, 1.0)
    flat[slots.long()] = x / sc.unsqueeze(-1)
    scales = scale.double().flatten(0, 1)
    scales[slots.long()] = sc
    return flat.view(cache.shape), scales.view(scale.shape)


def _exact_decode(s):
    q, (_, ps, hk, d) = s["q"].double(), s["k_cache"].shape
    b, hq, _ = q.shape
    o = torch.zeros((b, hq, d), dtype=torch.float64, device=q.device)
    lse = torch.full((b, hq), float("-inf"), dtype=torch.float64, device=q.device)
    for i, n in enumerate(s["seq_lens"].tolist()):
        at = torch.arange(max(0, n - s["window"]) if s["window"] else 0, n, device=q.device)
        page, slot = s["block_table"][i].long()[at // ps], at % ps
        for h in range(hk):
            k, v = s["k_cache"][page, slot, h].double(), s["v_cache"][page, slot, h].double()
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][page, slot, h].double()[:, None], v * s["v_scale"][page, slot, h].double()[:, None]
            rows = slice(h * (hq // hk), (h + 1) * (hq // hk))
            score = q[i, rows] @ k.T * s["sm_scale"]
            lse[i, rows] = torch.logsumexp(score, -1) / math.log(2.0)
            o[i, rows] = torch.softmax(score, -1) @ v
    return o, lse


def exact(case, seed):
    if case["op"] == "pages":   # whole numbers and copies
        return None
    s = prepare(case, seed)
    if case["op"] == "decode":
        return _exact_decode(s)
    if case["op"] == "rope":
        return _exact_head_rows(s["q"], None, s), _exact_head_rows(s["k"], None, s)
    q, k = _exact_head_rows(s["q"], s["q_weight"], s), _exact_head_rows(s["k"], s["k_weight"], s)
    if s["cache"] == "none":
        return q, k
    k_cache, k_scale = _exact_store(k, s["slot_mapping"], s["k_cache"], s["k_scale"])
    v_cache, v_scale = _exact_store(s["v"].double(), s["slot_mapping"], s["v_cache"], s["v_scale"])
    return q, k_cache, v_cache, k_scale, v_scale
