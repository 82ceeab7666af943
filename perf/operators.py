"""The paged-attention operators of the decoder layer's attention half, as they are measured.

Five kinds of case: ``rope`` (multi-axis rotary positions, per-head norm and the write of keys and
values into the cache's pages), ``decode`` (attention of one new token a sequence over the paged
cache), ``prefill`` (attention of several new tokens a sequence), ``fork`` (a beam step's page
bookkeeping: free, fork, grow) and ``compact`` (live pages moved to the front of the pool).

The plain forms use elementary torch operations in 32 bits (rotary angles in 64), rounded once.
"""
from __future__ import annotations

import importlib.util
import math
import os
import sys

import torch

own = False

BF16 = torch.bfloat16


def _package():
    """The framework's package (its folder name has hyphens)."""
    name = "paris_moe_b200"
    if name not in sys.modules:
        d = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                         "paris-hackathon-2026-inference_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ---- the cases -----------------------------------------------------------------------------


def listed():
    return [
        # A decode step's 64 tokens: 16 query and 2 key/value heads of 256, 64 rotary dims in
        # three interleaved axes, q/k norms: the call between projection and attention.
        dict(name="rope_decode_64", op="rope", tokens=64, seqs=64, hq=16, hkv=2, d=256, rot=64,
             axes=3, interleaved=True, norm=True, page=64, ctx=700),
        # A prefill batch of 8192 tokens (32 prompts of 256), the same layer.
        dict(name="rope_prefill_8192", op="rope", tokens=8192, seqs=32, hq=16, hkv=2, d=256,
             rot=64, axes=3, interleaved=True, norm=True, page=64, ctx=0),
        # One chat session early on: latency of the smallest call.
        dict(name="decode_b1_short", op="decode", seqs=1, max_len=333, hq=16, hkv=2, d=256,
             page=16, window=0, sinks=0),
        # A full decode batch over ragged contexts up to 16k: the serving steady state.
        dict(name="decode_b64_16k", op="decode", seqs=64, max_len=16384, hq=16, hkv=2, d=256,
             page=64, window=0, sinks=0),
        # A few very long documents in small pages under a wide window with 4 sinks, 5 query
        # heads a group: few rows, so the work is split over the cache's length.
        dict(name="decode_b3_window", op="decode", seqs=3, max_len=100001, hq=40, hkv=8, d=128,
             page=16, window=30000, sinks=4),
        # One long prompt in one go.
        dict(name="prefill_8192", op="prefill", seqs=1, new=8192, ctx=0, hq=16, hkv=2, d=256,
             page=64, window=0, sinks=0),
        # Chunks of prompts on top of long cached contexts, under a window with sinks.
        dict(name="prefill_chunk_window", op="prefill", seqs=3, new=1021, ctx=9000, hq=32, hkv=8,
             d=128, page=16, window=2000, sinks=16),
        # Drafted tokens of 16 sequences checked in one pass: a handful of rows each.
        dict(name="prefill_verify", op="prefill", seqs=16, new=5, ctx=900, hq=16, hkv=2, d=256,
             page=64, window=0, sinks=0),
        # A beam step of 2 prompts into 8 branches, small cache.
        dict(name="fork_small", op="fork", parents=2, children=4, max_len=300, add=1, layers=2,
             hkv=2, d=128, page=16),
        # 32 prompts, each forked into 8 samples, all attention layers of a 40-layer hybrid model.
        dict(name="fork_large", op="fork", parents=32, children=8, max_len=2000, add=64, layers=10,
             hkv=2, d=256, page=16),
        # A pool of 10 layers, half of it live, packed before it is shrunk.
        dict(name="compact_large", op="compact", seqs=64, max_len=2048, layers=10, hkv=2, d=256,
             page=64),
        # A small pool, as a quiet server packs it.
        dict(name="compact_small", op="compact", seqs=5, max_len=400, layers=2, hkv=2, d=128,
             page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "decode", "decode", "prefill", "prefill", "fork", "compact"])
    d = rng.choice([64, 128, 256])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8, 16])
    page = rng.choice([16, 32, 64, 128])
    if op == "rope":
        seqs = _log(rng, 1, 64)
        c = dict(op=op, tokens=seqs if rng.random() < 0.4 else max(seqs, _log(rng, 1, 8192)),
                 seqs=seqs, hq=min(hq, 32), hkv=hkv, d=d, rot=rng.choice([d // 4, d // 2, d]),
                 axes=rng.choice([1, 3, 4]), interleaved=rng.random() < 0.5,
                 norm=rng.random() < 0.5, page=page, ctx=_log(rng, 1, 3000) - 1)
    elif op in ("decode", "prefill"):
        window = rng.choice([0, 0, _log(rng, 16, 5000)])
        c = dict(op=op, seqs=_log(rng, 1, 64) if op == "decode" else _log(rng, 1, 32),
                 hq=hq, hkv=hkv, d=d, page=page, window=window,
                 sinks=rng.choice([0, 4, _log(rng, 1, 200)]) if window else 0)
        if op == "decode":
            c["max_len"] = _log(rng, 1, 100000)
        else:
            c["new"], c["ctx"] = _log(rng, 1, 8192), _log(rng, 1, 12000) - 1
    elif op == "fork":
        c = dict(op=op, parents=_log(rng, 1, 32), children=rng.randint(1, 8),
                 max_len=_log(rng, 1, 2000), add=_log(rng, 1, 100), layers=rng.randint(1, 10),
                 hkv=min(hkv, 2), d=d, page=rng.choice([16, 32]))
    else:
        c = dict(op=op, seqs=_log(rng, 1, 64), max_len=_log(rng, 16, 2048),
                 layers=rng.randint(1, 10), hkv=min(hkv, 2), d=d, page=page)
    most = {x["op"]: x for x in sorted(listed(), key=lambda x: work(x)["bytes"] + work(x)["flops"])}
    while not _fits(c, most[op]):
        for key in ("max_len", "new", "ctx", "tokens", "seqs", "parents"):
            if c.get(key, 0) > 1:
                c[key] = max(1, int(c[key] * 0.7))
        if op == "rope":
            c["tokens"] = max(c["tokens"], c["seqs"])
    return c


def _fits(c, most):
    a, b = work(c), work(most)
    if a["bytes"] > max(b["bytes"], 1 << 20) or a["flops"] > max(b["flops"], 1 << 20):
        return False
    # what the plain forms hold: padded keys, or all pairs of rows and keys
    if c["op"] == "decode":
        return c["seqs"] * c["max_len"] * c["hkv"] * c["d"] <= 1 << 29
    if c["op"] == "prefill":
        return c["seqs"] * c["hq"] * c["new"] * (c["new"] + c["ctx"] + c["page"]) <= 1.1e9
    return True


def _ragged(n, most, least=1):
    """n lengths between `least` and `most`, spread evenly and out of order; the first is `most`."""
    return [most] + [least + int((most - least) * ((i * 0.6180339887498949) % 1.0))
                     for i in range(1, n)]


def _seq_lens(c):
    """(new tokens, cached length with them) of each sequence."""
    if c["op"] == "decode":
        kv = _ragged(c["seqs"], c["max_len"])
        return [1] * c["seqs"], kv
    if c["op"] == "prefill":
        new = _ragged(c["seqs"], c["new"])
        return new, [n + x for n, x in zip(new, _ragged(c["seqs"], c["ctx"], c["ctx"] // 2))]
    base, more = divmod(c["tokens"], c["seqs"])
    new = [base + (1 if i < more else 0) for i in range(c["seqs"])]
    return new, [n + x for n, x in zip(new, _ragged(c["seqs"], c["ctx"], c["ctx"] // 2))]


def _visible(p, window, sinks):
    """Keys that the token at index p sees."""
    lo = max(0, p + 1 - window) if window else 0
    return p + 1 - lo + min(sinks, lo)


def _sections(c):
    half, a = c["rot"] // 2, c["axes"]
    rest = [half // a] * (a - 1)
    return [half - sum(rest)] + rest


def work(case):
    c = case
    if c["op"] == "rope":
        t = c["tokens"]
        return {"bytes": 2.0 * 2 * t * (c["hq"] + 2 * c["hkv"]) * c["d"] + 8 * t * c["axes"],
                "flops": 6.0 * t * (c["hq"] + c["hkv"]) * c["rot"] / 2}
    if c["op"] in ("decode", "prefill"):
        new, kv = _seq_lens(c)
        pairs = read = 0
        for n, l in zip(new, kv):
            if not c["window"]:
                pairs += n * l - n * (n - 1) // 2
                read += l
            else:
                pairs += sum(_visible(p, c["window"], c["sinks"]) for p in range(l - n, l))
                lo = max(0, l - n + 1 - c["window"])
                read += l - lo + min(c["sinks"], lo)
        return {"bytes": 4.0 * read * c["hkv"] * c["d"] + 4.0 * sum(new) * c["hq"] * c["d"],
                "flops": 4.0 * pairs * c["hq"] * c["d"]}
    row = 2.0 * 2 * c["layers"] * c["hkv"] * c["d"]   # bytes of one token in all layers
    if c["op"] == "fork":
        lens = _ragged(c["parents"], c["max_len"])
        tail = sum(n % c["page"] for n in lens) * c["children"]
        entries = sum(-(-n // c["page"]) + -(-(n + c["add"]) // c["page"]) for n in lens)
        return {"bytes": 2 * row * tail + 8.0 * entries * c["children"], "flops": 0.0}
    _, _, moved, entries = _fragmented(c)
    return {"bytes": 2 * row * c["page"] * len(moved) + 8.0 * entries, "flops": 0.0}


# ---- inputs --------------------------------------------------------------------------------


def _randn(shape, gen):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(BF16)


def _pool(shape, gen):
    """A pool filled with normal values (a block of them, repeated by page with other scales)."""
    n = shape[0]
    block = _randn((min(n, 256), *shape[1:]), gen)
    if n <= 256:
        return block
    out = torch.empty(shape, dtype=BF16, device="cuda")
    order = torch.randint(0, 256, (n,), generator=gen, device="cuda")
    torch.index_select(block, 0, order, out=out)
    size = (n,) + (1,) * (len(shape) - 1)
    return out.mul_(0.5 + torch.rand(size, generator=gen, device="cuda").to(BF16))


def _paged(c, kv, gen, layers=2):
    """A pool of `layers` layers with every sequence's pages at random places, and its tables.
    Entries behind a sequence's last page are -1."""
    need = [-(-n // c["page"]) for n in kv]
    total, width = sum(need), max(max(need), 1)
    n_pages = total + 1 + total // 8
    shape = (n_pages, layers, 2, c["hkv"], c["page"], c["d"])
    pages = _pool(shape, gen)
    order = torch.randperm(n_pages, generator=gen, device="cuda")[:total].int()
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    table[at] = order
    lens = torch.tensor(kv, dtype=torch.int32, device="cuda")
    return pages, table, lens


def _prefix(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _parent_tables(c):
    """Tables of the parents, pages in order; children slots follow, empty."""
    lens = _ragged(c["parents"], c["max_len"])
    slots = c["parents"] * (1 + c["children"])
    width = -(-(c["max_len"] + c["add"]) // c["page"])
    own_pages = sum(-(-n // c["page"]) for n in lens)
    fresh = sum(-(-(n + c["add"]) // c["page"]) - n // c["page"] for n in lens) * c["children"]
    return lens, slots, width, own_pages, own_pages + fresh + 7


def _fragmented(c):
    """Sequences of a pool in which every other one has been freed: (lengths, their page
    numbers, pages that compaction moves, table entries)."""
    lens = _ragged(2 * c["seqs"], c["max_len"])
    at, mine = 0, []
    for i, n in enumerate(lens):
        k = -(-n // c["page"])
        if i % 2:
            mine.append(list(range(at, at + k)))
        at += k
    live = sum(len(m) for m in mine)
    moved = [p for m in mine for p in m if p >= live]
    return lens[1::2], mine, moved, live


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    st = {"case": c}
    if c["op"] in ("rope", "decode", "prefill"):
        new, kv = _seq_lens(c)
        pages, table, lens = _paged(c, kv, gen)
        st |= dict(pages=pages, k=pages[:, 1, 0], v=pages[:, 1, 1], table=table, lens=lens,
                   cu=_prefix(new))
        tokens = sum(new)
        if c["op"] != "rope":
            st["q"] = _randn((tokens, c["hq"], c["d"]), gen)
            st["scale"] = c["d"] ** -0.5
            st["new"], st["most"] = new, max(new)
            return st
        width = (c["hq"] + 2 * c["hkv"]) * c["d"]
        qkv = _randn((tokens, width), gen)     # the fused projection's output
        cut = (c["hq"] * c["d"], c["hkv"] * c["d"], c["hkv"] * c["d"])
        q, k, v = torch.split(qkv, cut, dim=1)
        st |= dict(q_in=q.view(tokens, c["hq"], c["d"]), k_in=k.view(tokens, c["hkv"], c["d"]),
                   v_in=v.view(tokens, c["hkv"], c["d"]))
        # text positions far into a session; every third token lies in an image's grid
        text = torch.arange(tokens, device="cuda") + 90000 + int(seed) % 1000
        grid = torch.randint(0, 64, (c["axes"], tokens), generator=gen, device="cuda")
        grid[0] = 0
        st["positions"] = torch.where(torch.arange(tokens, device="cuda") % 3 == 0,
                                      text[None] + grid, text[None]).contiguous()
        i = torch.arange(c["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / c["rot"]
        st["inv_freq"] = (1e7 ** -i).float()
        st["sections"] = _sections(c)
        st["one"] = c["tokens"] == c["seqs"]
        w = _randn((2, c["d"]), gen) * 0.1
        st["wq"], st["wk"] = (w[0], w[1]) if c["norm"] else (None, None)
        return st
    if c["op"] == "fork":
        lens, slots, width, held, n_pages = _parent_tables(c)
        pages = _pool((n_pages, c["layers"], 2, c["hkv"], c["page"], c["d"]), gen)
        order = torch.randperm(n_pages, generator=gen, device="cuda")[:held].int()
        refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        refs[order.long()] = 1
        tables = torch.full((slots, width), -1, dtype=torch.int32, device="cuda")
        need = torch.tensor([-(-n // c["page"]) for n in lens], device="cuda")
        tables[:c["parents"]][torch.arange(width, device="cuda")[None] < need[:, None]] = order
        all_lens = torch.zeros(slots, dtype=torch.int32, device="cuda")
        all_lens[:c["parents"]] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        src = torch.arange(c["parents"], device="cuda").repeat_interleave(c["children"]).int()
        dst = torch.randperm(slots - c["parents"], generator=gen, device="cuda").int()
        st |= dict(pages=pages, refs=refs, tables=tables, lens=all_lens, src=src,
                   dst=dst + c["parents"], keep=all_lens[src.long()].clone(),
                   add=torch.full((slots - c["parents"],), c["add"], dtype=torch.int32,
                                  device="cuda"))
    else:
        lens, mine, moved, live = _fragmented(c)
        n_pages = sum(-(-n // c["page"]) for n in _ragged(2 * c["seqs"], c["max_len"])) + 3
        pages = _pool((n_pages, c["layers"], 2, c["hkv"], c["page"], c["d"]), gen)
        width = -(-c["max_len"] // c["page"])
        rows = torch.tensor([m + [-1] * (width - len(m)) for m in mine], dtype=torch.int32)
        order = torch.randperm(len(mine), generator=torch.Generator().manual_seed(int(seed)))
        tables = rows[order].cuda()
        refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        refs[tables[tables >= 0].long()] = 1
        lens = torch.tensor(lens, dtype=torch.int32)[order].cuda()
        # the bookkeeping as it is before packing: a pass starts from it each time
        st |= dict(pages=pages, refs=refs, tables=tables, lens=lens, refs_before=refs.clone(),
                   tables_before=tables.clone())
    return st


# ---- one pass ------------------------------------------------------------------------------


def run(state):
    c = state["case"]
    return {"rope": _rope, "decode": _decode, "prefill": _prefill, "fork": _fork,
            "compact": _compact}[c["op"]](state, c)


def _rope(st, c):
    cu = None if st["one"] else st["cu"]
    if own:
        q = _package().rope_append(st["q_in"], st["k_in"], st["v_in"], st["positions"],
                                   st["inv_freq"], st["sections"], c["interleaved"], st["k"],
                                   st["v"], st["table"], st["lens"], cu_q=cu, w_qnorm=st["wq"],
                                   w_knorm=st["wk"], eps=1e-6)
        return {"q": q, "k_pages": st["k"], "v_pages": st["v"]}
    half = c["rot"] // 2
    i = torch.arange(half, device="cuda")
    sec = torch.tensor(st["sections"], device="cuda")
    if c["interleaved"]:
        axis = i % c["axes"]
        axis = torch.where(i < sec[axis] * c["axes"], axis, 0)
    else:
        axis = torch.bucketize(i, sec.cumsum(0), right=True)
    angle = st["positions"][axis].double() * st["inv_freq"].double()[:, None]
    cos, sin = angle.cos().T.float()[:, None], angle.sin().T.float()[:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (1 + w.float())
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1).to(BF16)

    q, k = turned(st["q_in"], st["wq"]), turned(st["k_in"], st["wk"])
    cu, t = st["cu"], torch.arange(c["tokens"], device="cuda")
    b = torch.searchsorted(cu[1:].long(), t, right=True)
    at = st["lens"][b].long() - cu[b + 1] + t
    page = st["table"][b, at // c["page"]].long()
    st["k"][page, :, at % c["page"]] = k
    st["v"][page, :, at % c["page"]] = st["v_in"]
    return {"q": q, "k_pages": st["k"], "v_pages": st["v"]}


def _attend(q, k_pages, v_pages, table, at, c, scale):
    """q [B,N,Hq,D] at key indexes `at` [B,N] (-1: no token) over each row's gathered pages."""
    b, n, hq, d = q.shape
    hkv, width = c["hkv"], table.shape[1] * c["page"]
    idx = table.clamp(min=0).long()
    k = k_pages[idx].transpose(1, 2).reshape(b, hkv, 1, width, d).float()
    q = q.view(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).float()
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    del k
    j = torch.arange(width, device="cuda")
    see = j <= at[..., None]
    if c["window"]:
        see &= (j > at[..., None] - c["window"]) | (j < c["sinks"])
    see = see[:, None, None]
    s.masked_fill_(~see, -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    v = v_pages[idx].transpose(1, 2).reshape(b, hkv, 1, width, d).float()
    o = torch.matmul(s, v) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d).to(BF16)


def _decode(st, c):
    if own:
        return _package().attn_decode(st["q"], st["k"], st["v"], st["table"], st["lens"],
                                      st["scale"], c["window"], c["sinks"])
    at = st["lens"].long()[:, None] - 1
    return _attend(st["q"][:, None], st["k"], st["v"], st["table"], at, c, st["scale"])[:, 0]


def _prefill(st, c):
    if own:
        return _package().attn_prefill(st["q"], st["k"], st["v"], st["table"], st["lens"],
                                       st["cu"], st["scale"], c["window"], c["sinks"])
    cu = st["cu"].long()
    new = cu[1:] - cu[:-1]
    i = torch.arange(st["most"], device="cuda")
    there = i < new[:, None]
    row = torch.where(there, cu[:-1, None] + i, 0)
    at = torch.where(there, st["lens"].long()[:, None] - new[:, None] + i, -1)
    o = _attend(st["q"][row], st["k"], st["v"], st["table"], at, c, st["scale"])
    return o[there]


def _grow_plain(st, slots, add, page):
    slots = slots.long()
    old = st["lens"][slots].long()
    need = (old + add + page - 1) // page - (old + page - 1) // page
    free = torch.nonzero(st["refs"] == 0)[:, 0]
    end = need.cumsum(0)
    ok = end <= free.numel()
    got = torch.where(ok, need, 0)
    picked = free[:int(got.sum())]
    st["refs"][picked] = 1
    at = torch.repeat_interleave(torch.arange(len(slots), device="cuda"), got)
    nth = torch.arange(len(picked), device="cuda") - (end - need)[at]
    st["tables"][slots[at], (old[at] + page - 1) // page + nth] = picked.int()
    st["lens"][slots] = torch.where(ok, old + add, old).int()
    return ok.int()


def _fork(st, c):
    page = c["page"]
    if own:
        pm, held = _package(), (st["refs"], st["tables"], st["lens"])
        pm.pages_free(*held, st["dst"], page)
        ok = pm.pages_fork(st["pages"], *held, st["src"], st["dst"], st["keep"])
        grown = pm.pages_grow(*held, st["dst"], st["add"], page)
    else:
        dst, src = st["dst"].long(), st["src"].long()
        rows = st["tables"][dst]
        st["refs"].index_add_(0, rows[rows >= 0].long(), torch.full_like(rows[rows >= 0], -1))
        st["tables"][dst] = -1
        # children share the parent's full pages and copy the partly filled one
        keep = st["keep"].long()
        full, part = keep // page, keep % page
        col = torch.arange(st["tables"].shape[1], device="cuda")
        rows = torch.where(col < full[:, None], st["tables"][src], -1)
        shared = rows[rows >= 0]
        tail = st["tables"][src, full.clamp(max=len(col) - 1)].long()
        free = torch.nonzero(st["refs"] == 0)[:, 0]
        end = (part > 0).long().cumsum(0)
        ok = (end <= free.numel()).int()      # the pool has room for every child
        st["refs"].index_add_(0, shared.long(), torch.ones_like(shared))
        has = part > 0
        fresh = free[end[has] - 1]
        st["refs"][fresh] = 1
        rows[has, full[has]] = fresh.int()
        st["tables"][dst] = rows
        st["lens"][dst] = st["keep"]
        within = torch.arange(page, device="cuda") < part[has][:, None]
        which, slot = torch.nonzero(within, as_tuple=True)
        st["pages"][fresh[which], :, :, :, slot] = st["pages"][tail[has][which], :, :, :, slot]
        grown = _grow_plain(st, dst, st["add"], page)
    return {"ok": ok, "grown": grown, "pages": st["pages"], "refs": st["refs"],
            "tables": st["tables"], "lens": st["lens"]}


def _compact(st, c):
    st["refs"].copy_(st["refs_before"])
    st["tables"].copy_(st["tables_before"])
    if own:
        live, remap = _package().pages_compact(st["pages"], st["refs"], st["tables"])
    else:
        used = st["refs"] > 0
        live = used.sum().int().reshape(1)
        n = int(live)
        holes = torch.nonzero(~used[:n])[:, 0]
        movers = torch.nonzero(used[n:])[:, 0] + n
        remap = torch.where(used, torch.arange(len(used), device="cuda"), -1).int()
        remap[movers] = holes.int()
        st["pages"][holes] = st["pages"][movers]
        st["refs"][holes] = st["refs"][movers]
        st["refs"][movers] = 0
        t = st["tables"]
        t.copy_(torch.where(t >= 0, remap[t.clamp(min=0).long()], t))
    return {"live": live, "remap": remap, "pages": st["pages"], "refs": st["refs"],
            "tables": st["tables"]}


# ---- in 64 bits ----------------------------------------------------------------------------


def exact(case, seed):
    """What run() returns, from the definitions in 64 bits, sequence by sequence."""
    c, st = case, prepare(case, seed)
    if c["op"] == "rope":
        half, a = c["rot"] // 2, c["axes"]
        sec, angle = st["sections"], []
        for i in range(half):
            if c["interleaved"]:
                x = i % a if i < a * sec[i % a] else 0
            else:
                x = next(k for k in range(a) if i < sum(sec[:k + 1]))
            angle.append(st["positions"][x].double() * float(st["inv_freq"][i]))
        z = torch.polar(torch.ones_like(angle[0]), angle[0])[:, None].repeat(1, half)
        for i in range(half):
            z[:, i] = torch.polar(torch.ones_like(angle[i]), angle[i])

        def turn(x, w):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * (w.double() + 1)
            y = x.clone()
            pair = torch.complex(x[..., :half], x[..., half:2 * half]) * z[:, None]
            y[..., :half], y[..., half:2 * half] = pair.real, pair.imag
            return y

        q, k = turn(st["q_in"], st["wq"]), turn(st["k_in"], st["wk"])
        kp, vp = st["k"].double(), st["v"].double()
        new, kv = _seq_lens(c)
        t = 0
        for b, (n, l) in enumerate(zip(new, kv)):
            at = torch.arange(l - n, l, device="cuda")
            page = st["table"][b].long()[at // c["page"]]
            kp[page, :, at % c["page"]] = k[t:t + n]
            vp[page, :, at % c["page"]] = st["v_in"][t:t + n].double()
            t += n
        return {"q": q, "k_pages": kp, "v_pages": vp}
    if c["op"] in ("decode", "prefill"):
        new, kv = _seq_lens(c)
        g, out, t = c["hq"] // c["hkv"], [], 0
        for b, (n, l) in enumerate(zip(new, kv)):
            idx = st["table"][b, :-(-l // c["page"])].long()
            p = torch.arange(l - n, l, device="cuda")[:, None]
            j = torch.arange(l, device="cuda")[None]
            hide = j > p
            if c["window"]:
                hide = hide | ((j <= p - c["window"]) & (j >= c["sinks"]))
            heads = []
            for h in range(c["hq"]):
                k = st["k"][idx, h // g].reshape(-1, c["d"])[:l].double()
                v = st["v"][idx, h // g].reshape(-1, c["d"])[:l].double()
                s = st["q"][t:t + n, h].double() @ k.T * st["scale"]
                heads.append(torch.softmax(s.masked_fill(hide, -math.inf), 1) @ v)
            out.append(torch.stack(heads, 1))
            t += n
        return torch.cat(out)
    return None
