"""A paged key-value cache: what generating text with a trained model needs of attention (the reference trains only).

The keys and values of a layer lie in a pool of pages, (pages, heads, page, head_dim).  Slot s of sequence b is row s % page of
page `tables[b, s // page]`; what a table holds beyond the slots in use does not matter.  `tables` (batch, pages of a sequence)
and `lengths` (batch,) are int32 tensors on the GPU, so no call waits for the host and all of them can be captured in a CUDA
graph, which has its own scratch and may be replayed beside other calls and graphs.  For eviction every (page, head, slot) has two statistics: the attention that its key has got so far (`mass`, fp32), and
the position of its token (`positions`, int32), because a key that moves to another slot keeps its distance for ALiBi.

  * `paged_attention`   one new token per sequence: writes its key and value, attends to all keys, adds to the masses
  * `prompt_attention`  a prompt's causal attention, with the log-sum-exp of its rows
  * `prompt_mass`       the masses that the prompt gives its own keys, from that
  * `cache_append`      a prompt's keys and values (masses, positions) into the pages
  * `cache_evict`       each head keeps `keep` keys: the recent ones, then those of the largest mass

The query heads may be a multiple of the cache's heads (query head h uses key head h // group).  head_dim is 32, 64 or 128, the
type fp16 or bf16.  `attn_bias` is None, the (heads,) ALiBi slopes, or the model's (heads, T, T) ALiBi table, from which only
the slopes and the rounding are taken.  None of these has a gradient.  A page id or a length that does not fit the cache reads
and writes nothing out of bounds and shows in `_lib.check_status()`.
"""
import torch

from . import _host
from .attention import _resolve_bias, attention_forward


def _slopes(attn_bias, heads):
    bias = _resolve_bias(attn_bias, heads, 0, getattr(attn_bias, "dtype", None))
    assert bias.table is None, "the cache takes ALiBi slopes or an ALiBi table, no other bias"
    return bias


def paged_attention(query, k_pages, v_pages, tables, lengths, key=None, value=None, attn_bias=None, query_positions=None,
                    mass=None, positions=None, mass_out=None):
    """Attention of one query per sequence, (batch, heads, head_dim), over the lengths[b] keys in its pages; with `key` and
    `value` (batch, cache heads, head_dim) over those and the new key, which is written into slot lengths[b] (`lengths` itself
    stays).  A sequence without keys gets zeros.  With `mass` every key's weights, summed over the query heads of its head, are
    added to it, in place or into `mass_out` (no page may then be part of two sequences); the call then takes 4 bytes of scratch per
    query head and slot of the tables, whatever the lengths are.  With `positions` the new key's entry is set.  The query's
    position is query_positions[b], or the number of the last slot."""
    bias = _slopes(attn_bias, query.shape[1])
    return _host.paged_attention(query, k_pages, v_pages, tables, lengths, key, value, bias.slopes, int(bias.rounded),
                                 query_positions, mass, positions, mass_out)


def prompt_attention(query, key, value, attn_bias=None):
    """(causal attention, fp32 log-sum-exp of its rows) of a prompt: q, k, v as `fast_causal_attention` takes them."""
    out, lse, _ = attention_forward(query, key, value, _resolve_bias(attn_bias, query.shape[1], query.shape[2], query.dtype))
    return out, lse


def prompt_mass(query, key, lse, counts=None, attn_bias=None):
    """(batch, cache heads, T) fp32: what each key of a prompt gets of the causal attention of its first counts[b] tokens, summed
    over the queries and over the query heads of its head.  query (batch, heads, T, head_dim), key (batch, cache heads, T,
    head_dim), lse (batch, heads, T) of the scaled and biased scores; any T.  What lies behind a prompt's end may be anything."""
    bias = _slopes(attn_bias, query.shape[1])
    return _host.prompt_mass(query, key, lse, counts, bias.slopes, int(bias.rounded))


def cache_append(k_pages, v_pages, tables, lengths, key, value, counts=None, mass=None, positions=None, key_mass=None,
                 first_positions=None):
    """Writes the first counts[b] (None: all) of the keys and values (batch, cache heads, T, head_dim) into the slots from
    lengths[b] on (`lengths` itself stays).  `mass` gets `key_mass` (batch, cache heads, T), or zeros; `positions`
    first_positions[b] + t, or the slots' numbers."""
    _host.cache_append(k_pages, v_pages, tables, lengths, key, value, counts, mass, positions, key_mass, first_positions)


def cache_evict(k_pages, v_pages, mass, positions, tables, lengths, keep, recent=0, next_positions=None, out=None,
                out_tables=None):
    """Every head of every sequence that has more than `keep` keys keeps the `keep` of the largest mass, ties to the lower slot,
    where a key whose position is at least next_positions[b] - recent (positions and next_positions None: the slot's number and
    the length) counts as one of infinite mass.  Keys before slot `keep` that stay do not move; those from behind fill the free slots.
    Returns the new lengths.  In place, unless `out` = (k_pages, v_pages, mass, positions) of other buffers is given, and where
    their pages are others, `out_tables`; in place, no page may be part of two sequences."""
    k_out, v_out, mass_out, positions_out = (None,) * 4 if out is None else out
    return _host.cache_evict(k_pages, v_pages, mass, positions, tables, lengths, next_positions, k_out, v_out, mass_out,
                             positions_out, out_tables, int(keep), int(recent))


class PagedKVCache:
    """The pages of one layer and their statistics.  `statistics=False` leaves out what only eviction (and, where keys have been
    evicted, ALiBi) needs."""

    def __init__(self, pages, heads, head_dim, page=64, dtype=torch.float16, device="cuda", statistics=True):
        self.k = torch.zeros((pages, heads, page, head_dim), device=device, dtype=dtype)
        self.v = torch.zeros_like(self.k)
        self.mass = torch.zeros((pages, heads, page), device=device) if statistics else None
        self.positions = torch.zeros((pages, heads, page), device=device, dtype=torch.int32) if statistics else None

    def attend(self, query, tables, lengths, key=None, value=None, attn_bias=None, query_positions=None):
        return paged_attention(query, self.k, self.v, tables, lengths, key, value, attn_bias, query_positions, self.mass,
                               self.positions)

    def append(self, tables, lengths, key, value, counts=None, key_mass=None, first_positions=None):
        cache_append(self.k, self.v, tables, lengths, key, value, counts, self.mass, self.positions, key_mass, first_positions)

    def evict(self, tables, lengths, keep, recent=0, next_positions=None):
        return cache_evict(self.k, self.v, self.mass, self.positions, tables, lengths, keep, recent, next_positions)
