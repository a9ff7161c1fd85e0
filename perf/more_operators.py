"""The operators of generating text at a quarter of the bytes: what they compute, on what sizes, and in what time they could.

* `sample`  one token per sequence from its logits and a given uniform number, with temperature, top-k, top-p and min-p.
* `linear`  y = act(x W + bias) + addend with W in 4 bits and a scale for each group of rows of a column: single tokens, batches of
            them, and prompts.
* `attend`  attention of one token per sequence over a paged cache whose keys and values are held in 4 bits.
* `append`  keys and values into the pages of such a cache, and back as what the cache now holds.

Sizes are those of the framework's configurations (160M: 12 heads of 64; 410M: hidden size 1024, 16 heads of 64, 50304 tokens; 840M:
1536 and 6144, 12 heads of 128; 1.4B: 2048 and 8192 with linear biases), or generic ones with grouped key heads.

Four bits.  A value is its scale times a code from -7 to 7: the scale is the largest magnitude of the group over 7, rounded to the
16-bit type, the code the nearest whole number to value / scale (ties to even).  A nibble holds the code plus 8.
  Cache: a row of head_dim values has one scale.  The 32-bit word w of a row holds dims 8 w .. 8 w + 7, dim 8 w + 2 n + e at bits
  4 n + 16 e.  `scales` (pages, heads, page, 2) has a row's scales of key and value.
  Weights (K, N), codes (N / 16, K / 64, 32, 4) words: the word (strip, unit, 4 r + j, t) holds columns 16 strip + r and
  16 strip + r + 8 at rows 64 unit + 32 (t / 2) + 8 j + 4 (t % 2) + 0..3; row offset 2 p + e of column half c lies at bits
  4 (c + 2 p) + 16 e.  `scales` (N / 16, groups, 8, 2): of columns r and r + 8.  Behind the last row or column: code and scale 0.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _sample(name, batch, vocab, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False, banned=0.0):
    return {"name": name, "kind": "sample", "batch": batch, "vocab": vocab, "dtype": dtype, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed, "banned": banned}


def _linear(name, rows, k, n, group, dtype, bias=False, relu=False, addend=False):
    return {"name": name, "kind": "linear", "rows": rows, "k": k, "n": n, "group": group, "dtype": dtype, "bias": bias,
            "relu": relu, "addend": addend}


def _attend(name, batch, kv_heads, group, hd, length, spread, page, dtype, alibi=False):
    return {"name": name, "kind": "attend", "batch": batch, "kv_heads": kv_heads, "group": group, "hd": hd, "length": length,
            "spread": spread, "page": page, "dtype": dtype, "alibi": alibi}


def _append(name, batch, kv_heads, hd, length, spread, page, dtype):
    return {"name": name, "kind": "append", "batch": batch, "kv_heads": kv_heads, "hd": hd, "length": length, "spread": spread,
            "page": page, "dtype": dtype}


def listed():
    return [
        # one user's next token: the call costs its latency
        _sample("sample_one", 1, 50304, "fp16", 0.8, 40, 0.95),
        # a serving batch in which every user has settings of their own
        _sample("sample_mixed", 128, 50304, "fp16", mixed=True),
        # a larger vocabulary of an odd size, a third of it ruled out by a grammar
        _sample("sample_wide", 16, 131071, "bf16", 1.0, 0, 0.9, 0.02, banned=0.33),
        # one user, the output projection of the 410M model with its residual
        _linear("linear_one", 1, 1024, 1024, 64, "fp16", addend=True),
        # four users, the 410M model's head
        _linear("linear_head", 4, 1024, 50304, 64, "fp16"),
        # a batch of users, the first MLP product of the 1.4B model
        _linear("linear_batch", 24, 2048, 8192, 32, "bf16", bias=True, relu=True),
        # a prompt of a thousand tokens through the first MLP product of the 840M model
        _linear("linear_prompt", 1000, 1536, 6144, 128, "fp16", relu=True),
        # one user, the 160M model, some hundred tokens in
        _attend("attend_one", 1, 12, 1, 64, 700, False, 64, "fp16"),
        # a batch of users of the 410M model with ALiBi at all ages
        _attend("attend_alibi", 24, 16, 1, 64, 2048, True, 64, "fp16", alibi=True),
        # a serving batch of long documents with four query heads on each key head and small pages
        _attend("attend_grouped", 32, 8, 4, 128, 16384, True, 32, "bf16"),
        # the keys of one step of a batch
        _append("append_step", 32, 16, 64, 1, False, 64, "fp16"),
        # prompts of many lengths into small pages
        _append("append_prompts", 16, 8, 128, 4096, True, 32, "bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind, dtype = rng.choice(["sample", "sample", "linear", "linear", "linear", "attend", "attend", "append"]), rng.choice(["fp16", "bf16"])
    if kind == "sample":
        dtype, vocab = rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"]), _log(rng, 100, 131072)
        batch = _log(rng, 1, max(1, min(128, 6_400_000 // vocab)))
        if rng.random() < 0.4:
            return _sample("", batch, vocab, dtype, mixed=True, banned=rng.choice([0.0, 0.2]))
        return _sample("", batch, vocab, dtype, rng.choice([1.0, 0.7, 1.3, 0.0]), rng.choice([0, 0, 1, 40, 200, _log(rng, 1, 5000)]),
                       rng.choice([1.0, 1.0, 0.95, 0.9, 0.5]), rng.choice([0.0, 0.0, 0.05]), banned=rng.choice([0.0, 0.0, 0.3, 0.9]))
    if kind == "linear":
        n = _log(rng, 9, 50304)
        k = _log(rng, 17, min(8192, 51_000_000 // n))
        rows = _log(rng, 1, max(1, min(1024, 9_000_000_000 // (k * n))))
        return _linear("", rows, k, n, rng.choice([32, 64, 64, 128]), dtype, rng.random() < 0.4, rng.random() < 0.4, rng.random() < 0.4)
    hd, page, spread = rng.choice([32, 64, 64, 128, 128]), rng.choice([16, 24, 32, 64, 128]), rng.random() < 0.6
    if kind == "attend":
        length = _log(rng, 1, 16384)
        kv_heads, group = rng.randint(1, 16), rng.choice([1, 1, 1, 2, 3, 4, 8, 16])
        most = max(1, min(128, 260_000_000 // (length * kv_heads * hd)))
        return _attend("", _log(rng, 1, most), kv_heads, group, hd, length, spread, page, dtype, rng.random() < 0.4)
    length, kv_heads = _log(rng, 1, 8192), rng.randint(1, 16)
    most = max(1, min(64, 30_000_000 // (length * kv_heads * hd)))
    return _append("", _log(rng, 1, most), kv_heads, hd, length, spread, page, dtype)


def _lengths(case):
    """The sequences' lengths, in no order of meaning: all the same, or evenly from one up to the largest."""
    b, n = case["batch"], case["length"]
    if not case["spread"] or b == 1:
        return [n] * b
    return [1 + (n - 1) * i // (b - 1) for i in range(b)]


def work(case):
    """Logits, packed weights, packed rows and their scales are read once, inputs too; outputs are written once."""
    if case["kind"] == "sample":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["batch"] * (case["vocab"] * size + 12 + (16 if case["mixed"] else 0)), "flops": case["batch"] * case["vocab"]}
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        scales = -(-k // case["group"]) * n
        return {"bytes": k * n // 2 + 2 * (scales + m * k + m * n * (2 if case["addend"] else 1) + (n if case["bias"] else 0)),
                "flops": 2 * m * k * n}
    lengths, hd, kv = _lengths(case), case["hd"], case["kv_heads"]
    rows = sum(lengths) * kv
    if case["kind"] == "attend":
        q = case["batch"] * kv * case["group"] * hd
        pages = sum(-(-n // case["page"]) for n in lengths)
        return {"bytes": rows * (hd + 4) + 4 * q + 4 * pages, "flops": 4 * rows * case["group"] * hd}
    return {"bytes": rows * (4 * hd + hd + 4) + case["batch"] * kv * case["length"] * 4 * hd, "flops": 0}


class _Draws:
    """Seeded values on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, scale=1.0):
        out = torch.empty(shape, device="cuda", dtype=dtype)
        return out.normal_(0.0, scale, generator=self.gen)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def whole(self, low, high, *shape):
        return torch.randint(low, high, shape, generator=self.gen, device="cuda")

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")


def _quantize(x):
    """(codes from -7 to 7 as int8, scales in x's type) of the groups along the last dimension."""
    scales = (x.abs().amax(-1, keepdim=True).float() / 7).to(x.dtype)
    codes = torch.where(scales > 0, x.float() / scales.float(), 0.0).round_().clamp_(-7, 7)
    return codes.to(torch.int8), scales.squeeze(-1)


def _pack_rows(codes):
    """Rows of the cache, (.., hd) codes into (.., hd / 2) bytes."""
    c = (codes + 8).to(torch.uint8).view(*codes.shape[:-1], -1, 2, 2, 2)  # (word, n / 2, n % 2, e)
    c = c.movedim(-1, -3)                                                 # (word, e, n / 2, n % 2): a byte has two n
    return (c[..., 0] | c[..., 1] << 4).reshape(*codes.shape[:-1], -1)


def _unpack_rows(packed):
    """The codes of rows of the cache, in 32 bits."""
    c = torch.stack((packed & 15, packed >> 4), -1).view(*packed.shape[:-1], -1, 2, 2, 2)  # (word, e, n / 2, n % 2)
    return c.movedim(-3, -1).reshape(*packed.shape[:-1], -1).float() - 8


def _pack_weight(codes, scales):
    """(K, N) codes and (groups, N) scales in the layout of the operator."""
    k, n = codes.shape
    strips, units = -(-n // 16), -(-k // 64)
    c = torch.full((units * 64, strips * 16), 8, device="cuda", dtype=torch.int32)
    c[:k, :n] = codes.int() + 8
    # unit, t / 2, j, t % 2, p, e; strip, column half, r
    c = c.view(units, 2, 4, 2, 2, 2, strips, 2, 8).permute(6, 0, 8, 2, 1, 3, 5, 4, 7).reshape(strips, units, 32, 4, 2, 4)  # .., e, c + 2 p
    shift = torch.arange(8, device="cuda", dtype=torch.int32).view(2, 4) * 4
    words = (c << shift).sum((-1, -2), dtype=torch.int32)
    out = torch.zeros((scales.shape[0], strips * 16), device="cuda", dtype=scales.dtype)
    out[:, :n] = scales
    return words, out.view(-1, strips, 2, 8).permute(1, 0, 3, 2).contiguous()


def _groups(k, group):
    """Groups of a column: the rows are padded to whole units of 64."""
    return -(-(-(-k // 64) * 64) // group)


def _tables(draws, lengths, page):
    """Tables of the pages that sequences of these lengths need, in an order that has come about over time."""
    need = [-(-n // page) for n in lengths]
    ids = draws.order(sum(need)) + 1
    at = torch.arange(max(need), device="cuda")
    need = torch.tensor(need, device="cuda")
    first = torch.cumsum(need, 0) - need
    table = ids[(first[:, None] + at).clamp(max=ids.numel() - 1)]
    return torch.where(at < need[:, None], table, 0).to(torch.int32), ids.numel() + 1


def prepare(case, seed):
    draws, dtype = _Draws(seed), DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "sample":
        return _prepare_sample(case, draws, dtype, s)
    if case["kind"] == "linear":
        m, k, n, group = case["rows"], case["k"], case["n"], case["group"]
        groups = _groups(k, group)
        w = torch.zeros((groups * group, n), device="cuda", dtype=dtype)
        w[:k] = draws.normal(k, n, dtype=dtype, scale=0.02)
        codes, s["w_scales"] = _quantize(w.view(groups, group, n).transpose(1, 2))
        codes = codes.transpose(1, 2).reshape(-1, n)[:k]
        s["codes"], s["scales"] = _pack_weight(codes, s.pop("w_scales"))
        s["x"] = draws.normal(m, k, dtype=dtype)
        s["bias"] = draws.normal(n, dtype=dtype, scale=0.1) if case["bias"] else None
        s["addend"] = draws.normal(m, n, dtype=dtype) if case["addend"] else None
        return s
    b, kv, hd, n = case["batch"], case["kv_heads"], case["hd"], case["length"]
    s["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[draws.order(b)]
    s["tables"], pages = _tables(draws, s["lengths"].tolist(), case["page"])
    shape = (pages, kv, case["page"])
    if case["kind"] == "append":
        # the views of one projection's output, as the model has them
        qkv = draws.normal(b, n, 3 * kv * hd, dtype=dtype)
        s["k"], s["v"] = (x.view(b, n, kv, hd).transpose(1, 2) for x in qkv.split(kv * hd, dim=2)[1:])
        s["before"] = torch.zeros_like(s["lengths"])
        s["k_pages"], s["v_pages"] = (torch.zeros((*shape, hd // 2), device="cuda", dtype=torch.uint8) for _ in range(2))
        s["scales"] = torch.zeros((*shape, 2), device="cuda", dtype=dtype)
        return s
    (k, k_scales), (v, v_scales) = (_quantize(draws.normal(*shape, hd, dtype=dtype)) for _ in range(2))
    s["k_pages"], s["v_pages"], s["scales"] = _pack_rows(k), _pack_rows(v), torch.stack((k_scales, v_scales), -1)
    heads = kv * case["group"]
    s["q"] = draws.normal(b, heads, hd, dtype=dtype, scale=2.0)
    s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], device="cuda") if case["alibi"] else None
    return s


def _prepare_sample(c, draws, dtype, s):
    b, vocab = c["batch"], c["vocab"]
    # a long bell of unlikely tokens, and some that fit; how sure the model is differs from token to token
    logits = draws.normal(b, vocab) * (1.0 + 2.0 * draws.uniform(b, 1))
    likely = draws.whole(0, vocab, b, 48)
    logits.scatter_add_(1, likely, 8.0 * draws.uniform(b, 48))
    if c["banned"]:
        logits.masked_fill_(draws.uniform(b, vocab) < c["banned"], float("-inf"))
    s["logits"], s["uniforms"] = logits.to(dtype), draws.uniform(b)
    for key in ("temperature", "top_k", "top_p", "min_p"):
        s[key] = c[key]
    if c["mixed"]:
        pick = lambda *choices: torch.tensor(choices, device="cuda")[draws.whole(0, len(choices), b)]  # noqa: E731
        s["temperature"] = 0.5 + draws.uniform(b)
        s["temperature"][draws.uniform(b) < 0.1] = 0.0
        s["top_k"] = pick(0, 0, 1, 20, 50, 400).to(torch.int32)
        s["top_p"], s["min_p"] = pick(1.0, 0.95, 0.9, 0.7), pick(0.0, 0.0, 0.02, 0.1)
    return s


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state)
    return _PLAIN[kind](state)


# ------------------------------------------------------------------------------------------------- the framework's calls


def _sample_own(s):
    from tritonformer_b200 import sample_tokens
    return sample_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


def _linear_own(s):
    from tritonformer_b200 import Int4Weight, linear_int4
    c = s["case"]
    return linear_int4(s["x"], Int4Weight(s["codes"], s["scales"], c["k"], c["n"], c["group"]), s["bias"], c["relu"], s["addend"])


def _attend_own(s):
    from tritonformer_b200 import paged_attention
    return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lengths"], attn_bias=s["slopes"], scales=s["scales"])


def _append_own(s):
    from tritonformer_b200 import cache_append
    return cache_append(s["k_pages"], s["v_pages"], s["tables"], s["before"], s["k"], s["v"], s["lengths"], scales=s["scales"],
                        stored=True)


_OWN = {"sample": _sample_own, "linear": _linear_own, "attend": _attend_own, "append": _append_own}


# ------------------------------------------------------------------------------------------------------- the plain forms


def _column(value, like):
    """A setting as a (batch, 1) column in 64 bits."""
    return (value if isinstance(value, torch.Tensor) else torch.full((like.shape[0],), value, device="cuda")).double()[:, None]


def _sample_plain(s):
    x = s["logits"].double().nan_to_num(nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
    temperature, top_k, top_p, min_p = (_column(s[key], x) for key in ("temperature", "top_k", "top_p", "min_p"))
    # settings that are given as numbers are 32-bit ones
    temperature, top_p, min_p = temperature.float().double(), top_p.float().double(), min_p.float().double()
    greedy = temperature == 0
    top_k = torch.where(greedy, 1.0, torch.where(top_k == 0, float("inf"), top_k))
    top = x.amax(1, keepdim=True)
    w = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(greedy, 1.0, temperature)))
    order = x.argsort(dim=1, descending=True, stable=True)
    ranked = w.gather(1, order)
    ranked = torch.where(torch.arange(x.shape[1], device="cuda") < top_k, ranked, 0.0)
    upto = ranked.cumsum(1)
    inside = (upto - ranked < top_p * upto[:, -1:]) | (top_p >= 1)
    ranked = torch.where(inside & (ranked >= min_p), ranked, 0.0)
    upto = torch.zeros_like(w).scatter_(1, order, ranked).cumsum(1)
    token = (upto > s["uniforms"].double()[:, None] * upto[:, -1:]).to(torch.uint8).argmax(1)
    return torch.where(top[:, 0] == float("-inf"), -1, token)


def _linear_plain(s):
    c = s["case"]
    k, n, group = c["k"], c["n"], c["group"]
    strips, units = s["codes"].shape[:2]
    shift = torch.arange(8, device="cuda", dtype=torch.int32).view(2, 2, 2) * 4  # e, p, column half
    codes = ((s["codes"].view(strips, units, 8, 4, 2, 2, 1, 1, 1) >> shift) & 15).permute(1, 4, 3, 5, 7, 6, 0, 8, 2)
    codes = codes.reshape(units * 64, strips * 16)[:k].float() - 8
    scales = s["scales"].permute(1, 0, 3, 2).reshape(-1, strips * 16).float().repeat_interleave(group, 0)[:k]
    y = torch.matmul(s["x"].float(), (codes * scales)[:, :n])
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if c["relu"]:
        y = torch.where(y > 0, y, 0.0)
    if s["addend"] is not None:
        y = y + s["addend"].float()
    return y.to(s["x"].dtype)


def _rows(tables, kv, page, slots):
    """Rows in the flattened pages of `slots` (batch, kv heads, n) of every sequence and head."""
    b = torch.arange(tables.shape[0], device="cuda")[:, None, None]
    head = torch.arange(kv, device="cuda")[None, :, None]
    return (tables.long()[b, (slots // page).clamp(max=tables.shape[1] - 1)] * kv + head) * page + slots % page


def _attend_plain(s):
    c, tables = s["case"], s["tables"]
    b, kv, group, hd = c["batch"], c["kv_heads"], c["group"], c["hd"]
    n = tables.shape[1] * c["page"]
    slots = torch.arange(n, device="cuda").expand(b, kv, n)
    rows, lengths = _rows(tables, kv, c["page"], slots), s["lengths"].long()[:, None, None]
    scales = s["scales"].view(-1, 2)[rows].float()
    q = s["q"].float().view(b, kv, group, hd)
    scores = torch.matmul(q, _unpack_rows(s["k_pages"].view(-1, hd // 2)[rows]).transpose(2, 3)) * scales[:, :, None, :, 0] / math.sqrt(hd)
    if c["alibi"]:
        scores = scores - s["slopes"].view(1, kv, group, 1) * (lengths - 1 - slots).float()[:, :, None]
    scores = scores.masked_fill((slots >= lengths)[:, :, None], float("-inf"))
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = e / e.sum(-1, keepdim=True) * scales[:, :, None, :, 1]
    return torch.matmul(weights, _unpack_rows(s["v_pages"].view(-1, hd // 2)[rows])).view(b, kv * group, hd).to(s["q"].dtype)


def _append_plain(s):
    c, hd = s["case"], s["case"]["hd"]
    slots = torch.arange(c["length"], device="cuda").expand(c["batch"], c["kv_heads"], c["length"])
    valid = slots < s["lengths"][:, None, None]
    rows = _rows(s["tables"], c["kv_heads"], c["page"], s["before"].long()[:, None, None] + slots)
    (k, k_scales), (v, v_scales) = _quantize(s["k"]), _quantize(s["v"])
    for pages, values in ((s["k_pages"].view(-1, hd // 2), _pack_rows(k)), (s["v_pages"].view(-1, hd // 2), _pack_rows(v)),
                          (s["scales"].view(-1, 2), torch.stack((k_scales, v_scales), -1))):
        pages[rows] = torch.where(valid[..., None], values, pages[rows])
    return [torch.where(valid[..., None], codes.float() * scales.float()[..., None], 0.0).to(x.dtype)
            for x, codes, scales in ((s["k"], k, k_scales), (s["v"], v, v_scales))]


_PLAIN = {"sample": _sample_plain, "linear": _linear_plain, "attend": _attend_plain, "append": _append_plain}


# ------------------------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](case, s)


def _sample_exact(c, s):
    tokens = []
    settings = [[float(torch.tensor(v, dtype=torch.float32)) for v in (x.tolist() if isinstance(x, torch.Tensor) else [x] * c["batch"])]
                for x in (s["temperature"], s["top_k"], s["top_p"], s["min_p"])]
    for x, u, t, k, p, least in zip(s["logits"].double().cpu(), s["uniforms"].tolist(), *settings):
        best, order = torch.sort(x, descending=True, stable=True)
        count = len(best)
        if best[0] == -math.inf:
            tokens.append(-1)
            continue
        if t == 0:
            tokens.append(int(order[0]))
            continue
        if k:
            count = min(count, int(k))
        w = ((best[:count] - best[0]) / t).exp()
        if p < 1:
            ahead = torch.cat((torch.zeros(1, dtype=torch.float64), w.cumsum(0)[:-1]))
            count = max(1, int((ahead < p * w.sum()).sum()))
        count = min(count, int((w >= least).sum()))
        chosen, back = torch.sort(order[:count])
        line = w[:count][back].cumsum(0)
        tokens.append(int(chosen[int(torch.searchsorted(line, u * float(line[-1]), right=True))]))
    return torch.tensor(tokens, device="cuda")


def _linear_exact(c, s):
    k, n = c["k"], c["n"]
    w = torch.zeros((s["codes"].shape[1] * 64, s["codes"].shape[0] * 16), device="cuda", dtype=torch.float64)
    words = s["codes"].view(s["codes"].shape[0], -1, 8, 4, 4).long()  # strip, unit, r, j, t
    row, column = torch.arange(words.shape[1], device="cuda") * 64, torch.arange(words.shape[0], device="cuda") * 16
    for t in range(4):
        for j in range(4):
            for bit in range(8):
                at = row + 32 * (t // 2) + 8 * j + 4 * (t % 2) + 2 * (bit % 4 // 2) + bit // 4
                columns = (column[:, None] + torch.arange(8, device="cuda") + 8 * (bit % 2)).flatten()
                w[at[:, None], columns] = ((words[:, :, :, j, t] >> 4 * bit) & 15).double().sub(8).transpose(0, 1).reshape(len(row), -1)
    scale = s["scales"].double()  # strip, group, r, half
    for g in range(scale.shape[1]):
        w[g * c["group"]:(g + 1) * c["group"]] *= scale[:, g].transpose(1, 2).reshape(-1)
    y = s["x"].double() @ w[:k, :n]
    if s["bias"] is not None:
        y += s["bias"].double()
    if c["relu"]:
        y.clamp_(min=0)
    if s["addend"] is not None:
        y += s["addend"].double()
    return y


def _values(packed, scales):
    """Rows of the cache as 64-bit values, word by word."""
    words = packed.contiguous().view(torch.int32).long()
    out = torch.empty((*packed.shape[:-1], packed.shape[-1] * 2), device="cuda", dtype=torch.float64)
    for dim in range(8):
        out[..., dim::8] = ((words >> (4 * (dim // 2) + 16 * (dim % 2))) & 15).double() - 8
    return out * scales.double()[..., None]


def _attend_exact(c, s):
    group, hd = c["group"], c["hd"]
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    for b, n in enumerate(s["lengths"].tolist()):
        slots = torch.arange(n, device="cuda")
        p, r = s["tables"][b].long()[slots // c["page"]], slots % c["page"]
        for h in range(c["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            scales = s["scales"][p, h, r]
            scores = s["q"][b, heads].double() @ _values(s["k_pages"][p, h, r], scales[:, 0]).T / math.sqrt(hd)
            if c["alibi"]:
                scores -= s["slopes"][heads].double()[:, None] * (n - 1 - slots)
            out[b, heads] = torch.softmax(scores, -1) @ _values(s["v_pages"][p, h, r], scales[:, 1])
    return out


def _append_exact(c, s):
    out = []
    for x in (s["k"], s["v"]):
        scale = (x.double().abs().amax(-1, keepdim=True) / 7).to(x.dtype).double()
        y = (x.double() / scale.clamp(min=1e-30)).round() * scale
        for b, n in enumerate(s["lengths"].tolist()):
            y[b, :, n:] = 0
        out.append(y)
    return out


_EXACT = {"sample": _sample_exact, "linear": _linear_exact, "attend": _attend_exact, "append": _append_exact}
