"""Generating text with a trained `Transformer`: prompts into a paged key-value cache, then one token per sequence and step.

    gen = Generator(model, batch=8, max_tokens=2048)                  # or budget=512: at most 512 + 64 keys a head
    tokens = gen.generate(prompts, lengths, new_tokens=100)           # (8, 100), greedy
    logits = gen.prefill(prompts, lengths); logits = gen.step(tokens) # or token by token

The prompts' attention is the training forward; their keys and values (and with a budget their attention masses) go into the
cache's pages.  Everything runs in the model's own type, also inside an autocast region, on the layers' weights: forward hooks
on a layer or a projection are not called.  A step writes each sequence's new key and value and attends over its pages in one call
per layer.  With a budget every head of every layer keeps the `recent` last keys and those that have got most attention, after
the prompt and then every `interval` tokens.  The reference has no counterpart: it trains only.

A model without ALiBi has a learned position for each token; with it, the slopes come from its table, also where the model was
moved to bf16 after the table was made in fp16.  A captured step (`graph=True`) reads the weights where they were in memory;
if they lie elsewhere when the next prompts come, it is captured again.  They must not move between a prompt and its steps.
"""
import torch

from .attention import _Bias, _resolve_bias
from .embedding import Embedding
from .fused import LinearResidual, MLPResidual, QKVProjection
from .kvcache import PagedKVCache, cache_append, cache_evict, prompt_attention, prompt_mass
from .transformer import get_slopes


def _prompt_lengths(lengths, batch, tokens, device):
    """(lengths as int32 on the device, each from 1 to `tokens`; which of them were not, or None where the host has looked)."""
    if lengths is None:
        return torch.full((batch,), tokens, dtype=torch.int32, device=device), None
    lengths = torch.as_tensor(lengths)
    assert lengths.shape == (batch,) and not lengths.is_floating_point() and lengths.dtype != torch.bool, \
        "lengths are a number of tokens for each prompt"
    if lengths.is_cuda:
        counts = lengths.to(device).clamp(1, tokens)
        return counts.to(torch.int32), counts != lengths.to(device)
    assert batch == 0 or (int(lengths.min()) >= 1 and int(lengths.max()) <= tokens), \
        f"a prompt has from 1 to {tokens} tokens, the columns that there are"
    return lengths.to(device=device, dtype=torch.int32), None


def _bias_of(table, heads):
    bias = _resolve_bias(table, heads, 0, table.dtype)
    if bias.table is None or table.dtype is not torch.bfloat16:
        return bias
    # A model that was moved to bf16 has an ALiBi table that was rounded twice (to fp16 as it was made: slopes, distances and
    # products), and so is no table of bf16 slopes.  The slopes themselves are what it stands for.
    slopes = torch.tensor(get_slopes(heads), dtype=torch.float16).float().to(table.device)
    at = torch.arange(table.shape[1], device=table.device)
    back = (at[:, None] - at).clamp(min=0).float()
    for h in range(heads):
        want = back * slopes[h]
        if not bool(((table[h].float() + want).abs() <= (2.0 ** -8 + 2.0 ** -9) * want)[back > 0].all()):
            return bias
    return _Bias(slopes=slopes)


class Generator:
    """State of `batch` sequences on one model.  `max_tokens`: prompt and generated tokens of a sequence together.  All tensors are
    made here, so steps can be captured in a CUDA graph (`graph=True`)."""

    def __init__(self, model, batch, max_tokens, page=64, budget=None, recent=None, interval=64, graph=False):
        config = model.config
        weight = model.embed_tokens.weight
        assert weight.is_cuda and weight.dtype in (torch.float16, torch.bfloat16), "Generator expects a CUDA fp16/bf16 model"
        assert max_tokens <= config.max_position_embeddings, "more tokens than the model has positions"
        assert budget is None or (budget >= 1 and interval >= 1), "the budget and the interval are at least 1"
        self.model, self.batch, self.max_tokens, self.page = model, batch, max_tokens, page
        self.heads = config.num_attention_heads
        self.head_dim = config.hidden_size // config.num_attention_heads
        self.budget, self.interval = budget, interval
        self.recent = min(budget, 32 if recent is None else recent) if budget is not None else 0
        slots = max_tokens if budget is None else min(max_tokens, budget + interval)
        self.width = -(-slots // page)
        device = weight.device
        # every sequence owns its pages, the same ones in every layer's pool
        self.tables = torch.arange(batch * self.width, dtype=torch.int32, device=device).view(batch, self.width)
        self.caches = [PagedKVCache(batch * self.width, self.heads, self.head_dim, page, weight.dtype, device, budget is not None)
                       for _ in model.layer_list]
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)  # keys in the cache
        self.next = torch.zeros(batch, dtype=torch.int32, device=device)     # position of the token that comes next
        self.tokens = torch.zeros(batch, dtype=torch.int64, device=device)
        self.logits = torch.zeros((batch, config.vocab_size), dtype=weight.dtype, device=device)
        self.longest = self.position = 0  # upper bounds of `lengths` and `next` that the host knows
        self.want_graph, self.graph = graph, None
        self.weights = None  # where the captured step reads them
        self.bias = None, None, None  # the model's table, its version, and what _bias_of found

    def _bias(self):
        """The model's bias in the operators' form; a table that is new here is looked over, which waits for the host."""
        table = self.model.attn_bias
        version = None if table is None else table._version
        if self.bias[0] is not table or self.bias[1] != version:
            self.bias = table, version, None if table is None else _bias_of(table, self.heads)
            self.graph = None  # a captured step reads the slopes that it was captured with
        return self.bias[2]

    def _block(self, layer, x, attend):
        """One layer on (batch, tokens, hidden) without gradients; `attend` maps q, k, v to the context."""
        att, mlp = layer.attention, layer.mlp
        normed = layer.input_layernorm(x)
        q, k, v = QKVProjection.apply(normed, att.q_proj.weight, att.k_proj.weight, att.v_proj.weight)
        x = LinearResidual.apply(attend(q, k, v), att.out_proj.weight, None, x)
        normed = layer.post_attention_layernorm(x)
        return MLPResidual.apply(normed, mlp.dense_h_to_4h.weight, mlp.dense_h_to_4h.bias, mlp.dense_4h_to_h.weight,
                                 mlp.dense_4h_to_h.bias, x)

    @torch.no_grad()
    @torch.autocast("cuda", enabled=False)
    def prefill(self, prompts, lengths=None):
        """Starts the sequences: prompts (batch, T) int64, the first lengths[b] of each (all by default); what follows those may be
        any number.  Returns the logits (batch, vocab) of the tokens that follow.  Lengths are from 1 to T; those that are on the
        GPU are not waited for, but taken as the nearest ones that are, and `_lib.check_status()` says so."""
        b, t = prompts.shape
        assert b == self.batch and 1 <= t <= self.max_tokens, "prompts are (batch, up to max_tokens) token ids"
        device = self.tables.device
        counts, bad = _prompt_lengths(lengths, b, t, device)
        if self.graph is not None and self.weights != self._addresses():
            self.graph = None
        padded = -(-t // 64) * 64  # the training attention takes whole tiles of 64
        positions = self.model.embed_positions.weight if self.model.embed_positions is not None else None
        ids = torch.zeros((b, padded), dtype=torch.int64, device=device)
        behind = torch.arange(t, device=device) >= counts[:, None]
        ids[:, :t] = prompts.to(device).masked_fill(behind, 0)  # padding may be no token at all
        known = min(padded, self.model.config.max_position_embeddings)
        x = Embedding.apply(ids[:, :known], self.model.embed_tokens.weight, positions)
        if known < padded:  # rows behind the model's last position, which no other row sees
            x = torch.nn.functional.pad(x, (0, 0, 0, padded - known))
        start = torch.zeros_like(counts)
        # a prompt that is longer than what its sequence has pages for passes through pages of its own
        room = self.width * self.page
        through, tables = None, self.tables
        if t > room:
            width = -(-t // self.page)
            through = PagedKVCache(b * width, self.heads, self.head_dim, self.page, x.dtype, device)
            tables = torch.arange(b * width, dtype=torch.int32, device=device).view(b, width)
        left = counts
        for layer, cache in zip(self.model.layer_list, self.caches):
            into = through or cache

            def attend(q, k, v):
                q, k, v = (layer.attention._heads(y) for y in (q, k, v))
                out, lse = prompt_attention(q, k, v, self._bias())
                masses = prompt_mass(q, k, lse, counts, self._bias()) if self.budget is not None else None
                into.append(tables, start, k, v, counts, masses)
                return out.transpose(1, 2).reshape(b, padded, -1)

            x = self._block(layer, x, attend)
            if self.budget is not None and t > self.budget:
                if through is None:
                    left = cache.evict(tables, counts, self.budget, self.recent, counts)
                else:
                    left = cache_evict(through.k, through.v, through.mass, through.positions, tables, counts, self.budget,
                                       self.recent, counts, out=(cache.k, cache.v, cache.mass, cache.positions),
                                       out_tables=self.tables)
        last = x[torch.arange(b, device=device), counts.long() - 1]
        self.lengths.copy_(left)
        self.next.copy_(counts)
        self.longest = t if self.budget is None else min(t, self.budget)
        self.position = t
        logits = self._logits(last)
        if bad is not None:  # once the work is done, because the matrix products stop while there is a report
            none = torch.zeros((b, self.heads, 1, self.head_dim), dtype=x.dtype, device=device)
            cache_append(self.caches[0].k, self.caches[0].v, self.tables, start, none, none, torch.where(bad, -1, 0).to(torch.int32))
        return logits

    def _logits(self, x):
        return self.model.logits_out(self.model.final_layernorm(x.unsqueeze(1))).squeeze(1)

    def _forward(self):
        model = self.model
        position = None if model.embed_positions is None else model.embed_positions.weight[self.next.long()]
        x = Embedding.apply(self.tokens[None], model.embed_tokens.weight, position).transpose(0, 1)  # (batch, 1, hidden)
        for layer, cache in zip(model.layer_list, self.caches):

            def attend(q, k, v):
                q, k, v = (y.view(self.batch, self.heads, self.head_dim) for y in (q, k, v))
                out = cache.attend(q, self.tables, self.lengths, k, v, self._bias(), self.next)
                return out.view(self.batch, 1, -1)

            x = self._block(layer, x, attend)
        self.logits.copy_(self._logits(x.squeeze(1)))
        self.lengths += 1
        self.next += 1

    @torch.no_grad()
    @torch.autocast("cuda", enabled=False)
    def step(self, tokens):
        """Appends one token per sequence, (batch,) int64.  Returns the logits (batch, vocab) of those that follow, in a buffer
        that the next step writes again."""
        assert self.position < self.max_tokens, "the sequences have max_tokens tokens"
        if self.longest == self.width * self.page or (self.budget is not None and self.longest >= self.budget + self.interval):
            self._evict()
        self.tokens.copy_(tokens)
        self._bias()
        if self.want_graph and self.graph is None:
            self._capture()
        if self.graph is not None:
            self.graph.replay()
        else:
            self._forward()
        self.longest += 1
        self.position += 1
        return self.logits

    def _evict(self):
        assert self.budget is not None, "the cache is full"
        for cache in self.caches:
            left = cache.evict(self.tables, self.lengths, self.budget, self.recent, self.next)
        self.lengths.copy_(left)
        self.longest = min(self.longest, self.budget)

    def _addresses(self):
        return [p.data_ptr() for p in self.model.parameters()]

    def _capture(self):
        # a step ahead of the capture makes the workspaces; the sequences then go back to where they were
        before = self.lengths.clone(), self.next.clone()
        masses = [c.mass.clone() if c.mass is not None else None for c in self.caches]

        def back():
            self.lengths.copy_(before[0])
            self.next.copy_(before[1])
            for c, m in zip(self.caches, masses):
                if m is not None:
                    c.mass.copy_(m)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self._forward()
            back()
        torch.cuda.current_stream().wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=side):
            self._forward()
        self.weights = self._addresses()

    def generate(self, prompts, lengths=None, new_tokens=1, choose=None):
        """(batch, new_tokens) token ids that follow the prompts; `choose` maps logits to tokens (the largest by default)."""
        choose = choose or (lambda logits: logits.argmax(-1))
        logits, out = self.prefill(prompts, lengths), []
        for i in range(new_tokens):
            out.append(choose(logits))
            if i + 1 < new_tokens:
                logits = self.step(out[-1])
        return torch.stack(out, 1) if out else prompts[:, :0]
