"""Generation from the paged cache against the model's own forward pass on the whole sequence.

Tolerance: the bound of the whole-model comparisons (2e-2 of the logits' norm); both sides round their activations to 16 bits
in other places."""
import pytest
import torch

import tritonformer_b200._lib as L
from tritonformer_b200.generate import Generator
from tritonformer_b200.transformer import Transformer, TransformerConfig
from util import norm_rel

pytestmark = pytest.mark.gpu


def _model(head_dim=64, heads=4, layers=2, alibi=False, bias=False, dtype=torch.float16, positions=512):
    torch.manual_seed(0)
    d = head_dim * heads
    config = TransformerConfig(vocab_size=1000, hidden_size=d, max_position_embeddings=positions, num_attention_heads=heads,
                               head_dim=head_dim, ffn_dim=4 * d, num_hidden_layers=layers, use_linear_bias=bias, attn_bias=alibi)
    model = Transformer(config, device="cuda")
    with torch.no_grad():
        model.logits_out.weight.normal_(0.0, 0.02)
        model.embed_tokens.weight.normal_(0.0, 1.0)
        for layer in model.layer_list:  # attention that is not uniform
            layer.attention.q_proj.weight.normal_(0.0, 0.1)
            layer.attention.k_proj.weight.normal_(0.0, 0.1)
    if dtype is torch.bfloat16:
        table = model.attn_bias
        model = model.to(dtype)
        if table is not None:
            model.attn_bias = table
    return model.fuse_projection_weights()


def _teacher(model, ids, prompt, generator, lengths=None):
    """Logits of every position from the last prompt token on, token by token."""
    out = [generator.prefill(ids[:, :prompt], lengths).clone()]
    for t in range(prompt, ids.shape[1]):
        out.append(generator.step(ids[:, t]).clone())
    return torch.stack(out, 1)


@pytest.mark.parametrize("head_dim,alibi,bias,dtype", [(64, False, False, torch.float16), (64, True, True, torch.float16),
                                                       (128, True, False, torch.bfloat16), (32, False, True, torch.bfloat16)])
@pytest.mark.parametrize("page,prompt", [(64, 100), (16, 1), (24, 64)])
def test_steps_match_the_whole_sequence(page, prompt, head_dim, alibi, bias, dtype):
    model = _model(head_dim, 4, 2, alibi, bias, dtype)
    ids = torch.randint(0, 1000, (3, 128), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    with torch.no_grad():
        want = model(ids, None)[:, prompt - 1:]
    got = _teacher(model, ids, prompt, Generator(model, 3, 128, page))
    assert norm_rel(got, want) < 2e-2
    L.check_status()


def test_a_budget_that_is_never_reached_changes_nothing():
    model = _model(alibi=True)
    ids = torch.randint(0, 1000, (2, 96), device="cuda")
    plain = _teacher(model, ids, 50, Generator(model, 2, 96))
    kept = _teacher(model, ids, 50, Generator(model, 2, 96, budget=96))
    assert torch.equal(plain, kept)


def test_inside_an_autocast_region():
    model = _model(dtype=torch.float16)
    ids = torch.randint(0, 1000, (1, 70), device="cuda")
    plain = _teacher(model, ids, 60, Generator(model, 1, 128, budget=64))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(plain, _teacher(model, ids, 60, Generator(model, 1, 128, budget=64)))


def test_prompts_of_different_lengths():
    """A sequence's logits do not depend on what it shares the batch with."""
    model = _model()
    g = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.randint(0, 1000, (3, 100), device="cuda", generator=g)
    new = torch.randint(0, 1000, (3, 5), device="cuda", generator=g)
    lengths = [100, 1, 37]
    gen = Generator(model, 3, 128)
    first = gen.prefill(ids, lengths)
    steps = [gen.step(new[:, i]).clone() for i in range(5)]
    for b, n in enumerate(lengths):
        whole = torch.zeros((1, 128), dtype=torch.int64, device="cuda")
        whole[0, :n], whole[0, n:n + 5] = ids[b, :n], new[b]
        with torch.no_grad():
            want = model(whole, None)[0, n - 1:n + 5]
        got = torch.stack([first[b]] + [s[b] for s in steps])
        assert norm_rel(got, want) < 2e-2, b


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("alibi", [False, True])
def test_eviction_keeps_the_budget_and_the_recent_keys(alibi, graph):
    """The prompt passes through pages of its own (160 tokens, 48 slots); then every 16 tokens."""
    model = _model(alibi=alibi)
    ids = torch.randint(0, 1000, (2, 300), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    gen = Generator(model, 2, 300, page=16, budget=32, recent=8, interval=16, graph=graph)
    gen.prefill(ids[:, :160], [160, 20])
    assert gen.lengths.tolist() == [32, 20]
    for t in range(160, 300):
        logits = gen.step(ids[:, t])
        assert logits.isfinite().all()
        here = gen.next.tolist()
        for cache in gen.caches:
            for b, n in enumerate(gen.lengths.tolist()):
                assert n <= 48
                slots = torch.arange(n, device="cuda")
                pages = gen.tables[b].long()[slots // 16]
                positions = cache.positions[pages, :, slots % 16].T  # (heads, n)
                assert (positions.sort(-1).values.diff() > 0).all()  # no key twice
                kept = set(range(max(0, here[b] - 8), here[b]))
                assert all(kept <= set(p.tolist()) for p in positions)
                assert cache.mass[pages, :, slots % 16].min() > 0  # every key has been attended to
    L.check_status()


def test_a_short_memory_matches_the_attention_it_leaves():
    """One layer, budget of recent keys only: each step attends to the keys that the cache holds, whatever slots they lie in."""
    model = _model(layers=1, alibi=True)
    ids = torch.randint(0, 1000, (1, 200), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    gen = Generator(model, 1, 200, page=16, budget=24, recent=24, interval=8)
    gen.prefill(ids[:, :100])
    layer = model.layer_list[0]
    with torch.no_grad():
        hidden = torch.nn.functional.embedding(ids, model.embed_tokens.weight)
        normed = layer.input_layernorm(hidden)
        k = layer.attention.k_proj(normed).view(200, 4, 64)
        v = layer.attention.v_proj(normed).view(200, 4, 64)
        for t in range(100, 140):
            gen.step(ids[:, t])
            n = int(gen.lengths[0])
            slots = torch.arange(n, device="cuda")
            pages = gen.tables[0].long()[slots // 16]
            positions = gen.caches[0].positions[pages, :, slots % 16].long()  # (n, heads)
            heads = torch.arange(4, device="cuda")
            # keys and values lie where their positions say
            assert (gen.caches[0].k[pages, :, slots % 16] - k[positions, heads]).abs().max() <= 2e-2
            assert (gen.caches[0].v[pages, :, slots % 16] - v[positions, heads]).abs().max() <= 2e-2
            assert positions.min() >= t + 1 - 32  # the last 24, and up to 8 since


@pytest.mark.parametrize("alibi", [False, True])
def test_graph_and_greedy(alibi):
    model = _model(alibi=alibi)
    ids = torch.randint(0, 1000, (2, 40), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    eager = Generator(model, 2, 128).generate(ids, None, 30)
    graph = Generator(model, 2, 128, graph=True)
    assert torch.equal(eager, graph.generate(ids, None, 30))
    assert torch.equal(eager, graph.generate(ids, None, 30))  # started again on the captured step
    assert eager.shape == (2, 30)


def test_refusals():
    model = _model(layers=1)
    with pytest.raises(AssertionError, match="positions"):
        Generator(model, 1, 513)
    with pytest.raises(AssertionError, match="budget"):
        Generator(model, 1, 128, budget=0)
    gen = Generator(model, 1, 70)
    with pytest.raises(AssertionError, match="prompts"):
        gen.prefill(torch.zeros((2, 4), dtype=torch.int64, device="cuda"))
    gen.prefill(torch.zeros((1, 69), dtype=torch.int64, device="cuda"))
    gen.step(torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(AssertionError, match="max_tokens"):
        gen.step(torch.zeros(1, dtype=torch.int64, device="cuda"))
    L.check_status()
