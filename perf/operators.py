"""The operators of a paged key-value cache, as one generates text with a trained model: what they compute, on what sizes, and
in what time they could.

* `attend`  attention of one new token per sequence over its pages, the token's own key and value written into its slot on the
            way; with statistics the softmax weights that every cached key gets are added to its accumulated mass.
* `mass`    the attention mass of a prompt's keys: the column sums of its causal softmax map, from the log-sum-exp that the
            attention forward has saved.
* `append`  a prompt's keys and values (and masses and positions) into the pages of its sequences.
* `evict`   every head of every sequence keeps the `keep` keys that are recent or have the largest mass: the survivors from
            behind slot `keep` move into the slots of the keys that go.  In place, or into other pages.

Sizes are those of the framework's configurations (160M: 12 heads of 64; 410M: 16 heads of 64; 840M: 12 heads of 128), or
generic ones with grouped key heads.  A sequence's slot s lies in page `tables[b, s // page]` at row s % page; page 0 belongs
to nobody and fills the tables' ends.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _attend(name, batch, kv_heads, group, hd, length, spread, page, dtype, stats=False, alibi=False):
    return {"name": name, "kind": "attend", "batch": batch, "kv_heads": kv_heads, "group": group, "hd": hd,
            "length": length, "spread": spread, "page": page, "dtype": dtype, "stats": stats, "alibi": alibi}


def _mass(name, batch, kv_heads, group, hd, length, spread, dtype, alibi=False):
    return {"name": name, "kind": "mass", "batch": batch, "kv_heads": kv_heads, "group": group, "hd": hd,
            "length": length, "spread": spread, "dtype": dtype, "alibi": alibi}


def _append(name, batch, kv_heads, hd, length, spread, page, dtype, stats=False):
    return {"name": name, "kind": "append", "batch": batch, "kv_heads": kv_heads, "hd": hd, "length": length,
            "spread": spread, "page": page, "dtype": dtype, "stats": stats}


def _evict(name, batch, kv_heads, hd, length, spread, keep, recent, page, dtype, in_place):
    return {"name": name, "kind": "evict", "batch": batch, "kv_heads": kv_heads, "hd": hd, "length": length,
            "spread": spread, "keep": keep, "recent": recent, "page": page, "dtype": dtype, "in_place": in_place}


def listed():
    return [
        # one user, the 160M model, some hundred tokens in: the call costs its latency
        _attend("attend_160m_one", 1, 12, 1, 64, 700, False, 64, "fp16"),
        # a batch of users of the 410M model with ALiBi at all ages, masses kept for eviction
        _attend("attend_410m_alibi", 24, 16, 1, 64, 2048, True, 64, "fp16", stats=True, alibi=True),
        # two long documents on the 840M model's heads, a length that ends inside a page
        _attend("attend_long", 2, 12, 1, 128, 49157, False, 128, "bf16"),
        # a serving batch with eight query heads on each key head and small pages
        _attend("attend_grouped", 64, 8, 8, 128, 8192, True, 32, "bf16", stats=True),
        # three short prompts of odd lengths
        _mass("mass_short", 3, 12, 1, 64, 331, True, "fp16"),
        # the prompts of the 410M configuration with ALiBi
        _mass("mass_410m", 4, 16, 1, 64, 2048, False, "fp16", alibi=True),
        # one long prompt with three query heads on each key head
        _mass("mass_long", 1, 4, 3, 128, 8192, False, "bf16"),
        # the prompts of the 160M configuration into the cache
        _append("append_160m", 2, 12, 64, 1024, False, 64, "fp16"),
        # prompts of many lengths into small pages, with masses and positions
        _append("append_grouped", 16, 8, 128, 4096, True, 32, "bf16", stats=True),
        # what a generation loop does every 64 tokens: back to the budget, in place
        _evict("evict_step", 8, 12, 64, 1088, False, 1024, 128, 64, "fp16", True),
        # prompts of the 410M configuration cut to a quarter, into pages of their own
        _evict("evict_410m", 16, 16, 64, 2048, True, 512, 64, 64, "fp16", False),
        # long documents cut to a quarter, in place
        _evict("evict_long", 4, 8, 128, 32768, False, 8192, 1024, 128, "bf16", True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _odd_one_out(n):
    """No size is 3 * 1024, which is another model's."""
    return n + 1 if n == 3 << 10 else n


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "mass", "mass", "append", "evict", "evict"])
    dtype, hd, page = rng.choice(["fp16", "bf16"]), rng.choice([32, 64, 64, 128, 128]), rng.choice([16, 32, 48, 64, 128])
    spread = rng.random() < 0.6
    if kind == "attend":
        length = _odd_one_out(_log(rng, 1, 49157))
        kv_heads, group = rng.randint(1, 16), rng.choice([1, 1, 1, 2, 3, 4, 7, 8, 16])
        most = max(1, min(128, 1_000_000_000 // (length * kv_heads * hd * 4), 40_000_000 // (length * kv_heads)))
        return _attend("", _log(rng, 1, most), kv_heads, group, hd, length, spread, page, dtype,
                       rng.random() < 0.5, rng.random() < 0.4)
    if kind == "mass":
        length = _odd_one_out(_log(rng, 1, 8192))
        kv_heads, group = rng.randint(1, 16), rng.choice([1, 1, 1, 2, 3])
        kv_heads = max(1, min(kv_heads, 12 * 8192 * 8192 // (length * length * group)))
        most = max(1, min(32, 12 * 8192 * 8192 // (length * length * kv_heads * group)))
        return _mass("", _log(rng, 1, most), kv_heads, group, hd, length, spread, dtype, rng.random() < 0.4)
    if kind == "append":
        length, kv_heads = _odd_one_out(_log(rng, 1, 8192)), rng.randint(1, 16)
        most = max(1, min(64, 30_000_000 // (length * kv_heads * hd)))
        return _append("", _log(rng, 1, most), kv_heads, hd, length, spread, page, dtype, rng.random() < 0.5)
    length, kv_heads = _odd_one_out(_log(rng, 2, 32768)), rng.randint(1, 16)
    keep = _odd_one_out(max(1, int(length * rng.uniform(0.1, 1.0))))
    most = max(1, min(32, 60_000_000 // (length * kv_heads * hd)))
    return _evict("", _log(rng, 1, most), kv_heads, hd, length, spread, keep, rng.randint(0, keep), page, dtype,
                  rng.random() < 0.5)


def _lengths(case):
    """The sequences' lengths, in no order of meaning: all the same, or evenly from one up to the largest."""
    b, n = case["batch"], case["length"]
    if not case["spread"] or b == 1:
        return [n] * b
    return [1 + (n - 1) * i // (b - 1) for i in range(b)]


def work(case):
    """Every key row that counts is read (and written) once; what a pass has to move beside them is its rows' statistics, its
    queries and its outputs."""
    lengths, hd, kv = _lengths(case), case["hd"], case["kv_heads"]
    rows = sum(lengths) * kv
    if case["kind"] == "attend":
        q = case["batch"] * kv * case["group"] * hd
        pages = sum(-(-n // case["page"]) for n in lengths)
        stats = rows * (8 if case["stats"] else 0) + rows * (4 if case["stats"] and case["alibi"] else 0)
        new = case["batch"] * kv * hd * 2
        return {"bytes": 2 * (2 * rows * hd + 2 * q + new) + stats + 4 * pages, "flops": 4 * rows * case["group"] * hd}
    if case["kind"] == "mass":
        heads = kv * case["group"]
        pairs = sum(n * (n + 1) // 2 for n in lengths) * heads
        return {"bytes": sum(lengths) * heads * (2 * hd + 4) + rows * 2 * hd + 4 * case["batch"] * kv * case["length"],
                "flops": 2 * pairs * hd}
    if case["kind"] == "append":
        return {"bytes": 2 * rows * 4 * hd + rows * (12 if case["stats"] else 0), "flops": 0}
    kept = sum(min(n, case["keep"]) for n in lengths) * kv
    # in place the rows that move are, on the whole, the survivors' share of what lies behind slot `keep`
    moved = kept if not case["in_place"] else sum(
        min(n, case["keep"]) * max(0, n - case["keep"]) // n for n in lengths) * kv
    return {"bytes": rows * 8 + kept * 8 + moved * 8 * hd, "flops": 0}


class _Draws:
    """Seeded values on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, scale=1.0):
        out = torch.empty(shape, device="cuda", dtype=dtype)
        return out.normal_(0.0, scale, generator=self.gen)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")


def _tables(draws, lengths, page):
    """Tables of the pages that sequences of these lengths need, in an order that has come about over time."""
    need = [-(-n // page) for n in lengths]
    ids = draws.order(sum(need)) + 1
    at = torch.arange(max(need), device="cuda")
    need = torch.tensor(need, device="cuda")
    first = torch.cumsum(need, 0) - need
    table = ids[(first[:, None] + at).clamp(max=ids.numel() - 1)]
    return torch.where(at < need[:, None], table, 0).to(torch.int32), ids.numel() + 1


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], device="cuda")


def _masses(draws, *shape):
    """Accumulated attention has a long tail; keys that have just come have none."""
    w = torch.exp(2.0 * draws.normal(*shape))
    return torch.where(draws.uniform(*shape) < 0.05, 0.0, w)


def prepare(case, seed):
    draws, dtype = _Draws(seed), DTYPES[case["dtype"]]
    b, kv, hd, n = case["batch"], case["kv_heads"], case["hd"], case["length"]
    lengths = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[draws.order(b)]
    s = {"case": case, "lengths": lengths}
    if case["kind"] in ("mass", "append"):
        group = case.get("group", 1)
        # the views of one projection's output, as the model has them
        width = (group + 2) * kv * hd
        qkv = draws.normal(b, n, width, dtype=dtype)
        q, k, v = (x.view(b, n, -1, hd).transpose(1, 2) for x in qkv.split([group * kv * hd, kv * hd, kv * hd], dim=2))
        s.update(k=k, v=v)
        if case["kind"] == "mass":
            q.mul_(2.0)
            s.update(q=q, slopes=_slopes(kv * group) if case["alibi"] else None)
            s["lse"] = torch.stack([_prompt_scores(q[i:i + 1], k[i:i + 1], s["slopes"]).logsumexp(-1)[0] for i in range(b)])
            return s
    stats = case.get("stats", True)
    s["tables"], pages = _tables(draws, lengths.tolist(), case["page"])
    shape = (pages, kv, case["page"])
    s["k_pages"], s["v_pages"] = draws.normal(*shape, hd, dtype=dtype), draws.normal(*shape, hd, dtype=dtype)
    s["mass"] = _masses(draws, *shape) if stats else None
    s["positions"] = None
    if stats:
        # after evictions the slots of a head are in no order of position, and those that went leave gaps
        slots = torch.arange(s["tables"].shape[1] * case["page"], device="cuda").expand(b, kv, -1)
        rows, valid = _rows(s["tables"], kv, case["page"], slots), slots < lengths[:, None, None]
        order = draws.uniform(*slots.shape).masked_fill(~valid, 2.0).argsort(-1)
        s["positions"] = torch.zeros(shape, device="cuda", dtype=torch.int32)
        _write(s["positions"], rows, 2 * order + draws.order(2)[0], valid)
        s["next"] = 2 * lengths + 2
    if case["kind"] == "attend":
        # the last of the `length` keys is the new token's
        s["before"] = lengths - 1
        s["q"] = draws.normal(b, kv * case["group"], hd, dtype=dtype, scale=2.0)
        s["k"], s["v"] = draws.normal(b, kv, hd, dtype=dtype), draws.normal(b, kv, hd, dtype=dtype)
        s["slopes"] = _slopes(kv * case["group"]) if case["alibi"] else None
        if stats:
            s["mass_out"] = torch.zeros_like(s["mass"])
    if case["kind"] == "append":
        s["before"] = torch.zeros_like(lengths)
        s["key_mass"] = _masses(draws, b, kv, n) if stats else None
    if case["kind"] == "evict":
        keep = [min(x, case["keep"]) for x in lengths.tolist()]
        s["out_tables"], pages = (None, 0) if case["in_place"] else _tables(draws, keep, case["page"])
        # the statistics go into buffers of their own, so that every pass finds the same ones
        out = shape if case["in_place"] else (pages, kv, case["page"])
        s["out"] = (s["k_pages"] if case["in_place"] else torch.zeros(*out, hd, device="cuda", dtype=dtype),
                    s["v_pages"] if case["in_place"] else torch.zeros(*out, hd, device="cuda", dtype=dtype),
                    torch.zeros(out, device="cuda"), torch.zeros(out, device="cuda", dtype=torch.int32))
    return s


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state)
    return _PLAIN[kind](state)


# ------------------------------------------------------------------------------------------------- the framework's calls


def _attend_own(s):
    from tritonformer_b200 import kvcache
    out = kvcache.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["before"], s["k"], s["v"],
                                  attn_bias=s["slopes"], query_positions=s.get("next"), mass=s["mass"],
                                  positions=s["positions"], mass_out=s.get("mass_out"))
    return _attend_outputs(s, out)


def _mass_own(s):
    from tritonformer_b200 import kvcache
    return kvcache.prompt_mass(s["q"], s["k"], s["lse"], s["lengths"], attn_bias=s["slopes"])


def _append_own(s):
    from tritonformer_b200 import kvcache
    kvcache.cache_append(s["k_pages"], s["v_pages"], s["tables"], s["before"], s["k"], s["v"], s["lengths"],
                         mass=s["mass"], positions=s["positions"], key_mass=s["key_mass"])
    return [x for x in (s["k_pages"], s["v_pages"], s["mass"], s["positions"]) if x is not None]


def _evict_own(s):
    from tritonformer_b200 import kvcache
    c = s["case"]
    left = kvcache.cache_evict(s["k_pages"], s["v_pages"], s["mass"], s["positions"], s["tables"], s["lengths"], c["keep"],
                               c["recent"], next_positions=s["next"], out=s["out"], out_tables=s["out_tables"])
    return [left, *s["out"]]


_OWN = {"attend": _attend_own, "mass": _mass_own, "append": _append_own, "evict": _evict_own}


def _attend_outputs(s, out):
    got = [out, s["k_pages"], s["v_pages"]]
    return got + [s["mass_out"], s["positions"]] if s["mass"] is not None else got


# ------------------------------------------------------------------------------------------------------- the plain forms


def _rows(tables, kv, page, slots):
    """Rows in the flattened pages of `slots` (batch, kv heads, n) of every sequence and head."""
    b = torch.arange(tables.shape[0], device="cuda")[:, None, None]
    head = torch.arange(kv, device="cuda")[None, :, None]
    return (tables.long()[b, (slots // page).clamp(max=tables.shape[1] - 1)] * kv + head) * page + slots % page


def _write(pages, rows, values, valid):
    """values into the rows of the flattened pages, where valid; elsewhere the row keeps what it has."""
    flat = pages.view(-1, pages.shape[-1]) if values.dim() > rows.dim() else pages.view(-1)
    mask = valid[..., None] if values.dim() > rows.dim() else valid
    flat[rows] = torch.where(mask, values.to(flat.dtype), flat[rows])


def _attend_plain(s):
    c, tables = s["case"], s["tables"]
    b, kv, group, hd, page = c["batch"], c["kv_heads"], c["group"], c["hd"], c["page"]
    slot = s["before"].long()[:, None, None].expand(b, kv, 1)
    new = _rows(tables, kv, page, slot)
    always = torch.ones_like(new, dtype=torch.bool)
    _write(s["k_pages"], new, s["k"][:, :, None], always)
    _write(s["v_pages"], new, s["v"][:, :, None], always)
    if s["mass"] is not None:
        _write(s["positions"], new, s["next"][:, None, None].expand(b, kv, 1), always)
    n = tables.shape[1] * page
    slots = torch.arange(n, device="cuda").expand(b, kv, n)
    rows, valid = _rows(tables, kv, page, slots), slots <= slot
    k, v = (x.view(-1, hd)[rows].float() for x in (s["k_pages"], s["v_pages"]))
    q = s["q"].float().view(b, kv, group, hd)
    scores = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(hd)
    if c["alibi"]:
        at = slots if s["positions"] is None else s["positions"].view(-1)[rows]
        here = s["before"][:, None, None] if s["positions"] is None else s["next"][:, None, None]
        scores = scores - s["slopes"].view(1, kv, group, 1) * (here - at).float()[:, :, None]
    scores = scores.masked_fill(~valid[:, :, None], float("-inf"))
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = e / e.sum(-1, keepdim=True)
    out = torch.matmul(weights, v).view(b, kv * group, hd).to(s["q"].dtype)
    if s["mass"] is not None:
        had = s["mass"].view(-1)[rows].masked_fill(slots == slot, 0.0)  # a new key has none
        _write(s["mass_out"], rows, had + weights.sum(2), valid)
    return _attend_outputs(s, out)


def _prompt_scores(q, k, slopes):
    """(b, heads, n, n) scaled scores with ALiBi, -inf above the diagonal, in 32 bits."""
    n, hd = k.shape[2:]
    q, k = q.float(), k.float().repeat_interleave(q.shape[1] // k.shape[1], 1)
    scores = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(hd)
    at = torch.arange(n, device="cuda")
    back = at[:, None] - at
    if slopes is not None:
        scores = scores - slopes[:, None, None] * back.float()
    return scores.masked_fill(back < 0, float("-inf"))


def _mass_plain(s):
    c = s["case"]
    weights = torch.exp(_prompt_scores(s["q"], s["k"], s["slopes"]) - s["lse"][..., None])
    queries = torch.arange(c["length"], device="cuda") < s["lengths"][:, None]
    weights = torch.where(queries[:, None, :, None], weights, 0.0)
    return weights.sum(2).view(c["batch"], c["kv_heads"], c["group"], c["length"]).sum(2)


def _append_plain(s):
    c = s["case"]
    slots = torch.arange(c["length"], device="cuda").expand(c["batch"], c["kv_heads"], c["length"])
    valid = slots < s["lengths"][:, None, None]
    rows = _rows(s["tables"], c["kv_heads"], c["page"], s["before"].long()[:, None, None] + slots)
    _write(s["k_pages"], rows, s["k"], valid)
    _write(s["v_pages"], rows, s["v"], valid)
    if c["stats"]:
        _write(s["mass"], rows, s["key_mass"], valid)
        _write(s["positions"], rows, s["before"][:, None, None] + slots, valid)
    return [x for x in (s["k_pages"], s["v_pages"], s["mass"], s["positions"]) if x is not None]


def _evict_plain(s):
    c, tables = s["case"], s["tables"]
    kv, page, keep = c["kv_heads"], c["page"], c["keep"]
    n = tables.shape[1] * page
    slots = torch.arange(n, device="cuda").expand(c["batch"], kv, n)
    rows, valid = _rows(tables, kv, page, slots), slots < s["lengths"][:, None, None]
    recent = s["positions"].view(-1)[rows] >= (s["next"] - c["recent"])[:, None, None]
    worth = torch.where(recent, float("inf"), s["mass"].view(-1)[rows]).masked_fill(~valid, -1.0)
    order = worth.argsort(dim=-1, descending=True, stable=True)
    kept = torch.empty_like(order).scatter_(2, order, slots) < keep
    kept = kept & valid
    to, front = slots[..., :keep], kept[..., :keep]
    hole, valid = valid[..., :keep] & ~front, valid[..., :keep]
    src = to
    if n > keep:
        behind = (~kept[..., keep:]).to(torch.int8).argsort(dim=-1, stable=True)  # the survivors' slots first, in their order
        nth = (hole.long().cumsum(-1) - 1).clamp(min=0, max=n - keep - 1)
        src = torch.where(hole, keep + behind.gather(2, nth), to)
    src = _rows(tables, kv, page, src)
    dst = _rows(tables if s["out_tables"] is None else s["out_tables"], kv, page, to)
    dst = torch.where(valid, dst, 0)
    for pages, out in zip((s["k_pages"], s["v_pages"], s["mass"], s["positions"]), s["out"]):
        flat = pages.view(-1, c["hd"]) if pages.dim() == 4 else pages.view(-1)
        _write(out, dst, flat[src], valid)
    return [s["lengths"].clamp(max=keep), *s["out"]]


_PLAIN = {"attend": _attend_plain, "mass": _mass_plain, "append": _append_plain, "evict": _evict_plain}


# ------------------------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](case, s)


def _place(s, b, slot):
    """(page, row) of a slot, or of a tensor of slots, of sequence b."""
    page = s["case"]["page"]
    return s["tables"][b].long()[slot // page], slot % page


def _attend_exact(c, s):
    group, hd = c["group"], c["hd"]
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    total = s["mass_out"].double() if s["mass"] is not None else None
    for b, last in enumerate(s["before"].tolist()):
        p, r = _place(s, b, torch.tensor(last, device="cuda"))
        s["k_pages"][p, :, r], s["v_pages"][p, :, r] = s["k"][b], s["v"][b]
        if total is not None:
            s["positions"][p, :, r], s["mass"][p, :, r] = s["next"][b], 0.0
        slots = torch.arange(last + 1, device="cuda")
        p, r = _place(s, b, slots)
        for h in range(c["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            scores = s["q"][b, heads].double() @ s["k_pages"][p, h, r].double().T / math.sqrt(hd)
            if c["alibi"]:
                back = last - slots if s["positions"] is None else s["next"][b] - s["positions"][p, h, r]
                scores -= s["slopes"][heads].double()[:, None] * back
            weights = torch.softmax(scores, -1)
            out[b, heads] = weights @ s["v_pages"][p, h, r].double()
            if total is not None:
                total[p, h, r] = s["mass"][p, h, r].double() + weights.sum(0)
    got = [out, s["k_pages"], s["v_pages"]]
    return got + [total, s["positions"]] if total is not None else got


def _mass_exact(c, s):
    out = torch.zeros(c["batch"], c["kv_heads"], c["length"], device="cuda", dtype=torch.float64)
    for b, n in enumerate(s["lengths"].tolist()):
        back = torch.arange(n, device="cuda")[:, None] - torch.arange(n, device="cuda")
        for h in range(c["kv_heads"] * c["group"]):
            kv = h // c["group"]
            e = s["q"][b, h, :n].double() @ s["k"][b, kv, :n].double().T / math.sqrt(c["hd"]) - s["lse"][b, h, :n, None]
            if c["alibi"]:
                e -= s["slopes"][h].double() * back
            out[b, kv, :n] += torch.where(back >= 0, e, -math.inf).exp_().sum(0)
    return out


def _append_exact(c, s):
    for b, n in enumerate(s["lengths"].tolist()):
        p, r = _place(s, b, torch.arange(n, device="cuda"))
        for h in range(c["kv_heads"]):
            s["k_pages"][p, h, r], s["v_pages"][p, h, r] = s["k"][b, h, :n], s["v"][b, h, :n]
            if c["stats"]:
                s["mass"][p, h, r] = s["key_mass"][b, h, :n]
                s["positions"][p, h, r] = torch.arange(n, device="cuda", dtype=torch.int32)
    return [x for x in (s["k_pages"], s["v_pages"], s["mass"], s["positions"]) if x is not None]


def _evict_exact(c, s):
    keep, left = c["keep"], []
    for b, n in enumerate(s["lengths"].tolist()):
        m = min(n, keep)
        left.append(m)
        p, r = _place(s, b, torch.arange(n, device="cuda"))
        masses, at = s["mass"][p, :, r].T.tolist(), s["positions"][p, :, r].T.tolist()
        oldest = int(s["next"][b]) - c["recent"]
        maps = []
        for worth, where in zip(masses, at):
            best = sorted(range(n), key=lambda i: (where[i] < oldest, 0.0 if where[i] >= oldest else -worth[i], i))[:m]
            stay, spare = set(best), iter(sorted(i for i in best if i >= m))
            maps.append([i if i in stay else next(spare) for i in range(m)])
        src = torch.tensor(maps, device="cuda")
        heads = torch.arange(c["kv_heads"], device="cuda")[:, None]
        table = s["tables"] if s["out_tables"] is None else s["out_tables"]
        to = torch.arange(m, device="cuda")
        p, r = table[b].long()[to // c["page"]], to % c["page"]
        rows = [x[p_, heads, r_] for p_, r_ in [_place(s, b, src)]
                for x in (s["k_pages"], s["v_pages"], s["mass"], s["positions"])]
        for out, values in zip(s["out"], rows):
            out[p[None], heads, r[None]] = values
    return [torch.tensor(left, device="cuda", dtype=torch.int32), *s["out"]]


_EXACT = {"attend": _attend_exact, "mass": _mass_exact, "append": _append_exact, "evict": _evict_exact}
