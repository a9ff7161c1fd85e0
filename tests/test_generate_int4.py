"""Generation with weights and cache in 4 bits, and drawn tokens.

Tolerances.  With packed weights: the model with the weights that they stand for, at the bound of the whole-model comparisons (2e-2 of the
logits' norm).  With a cache in 4 bits two ways through the same tokens differ by 16-bit roundings, some 2e-3 of a key; a code changes where that
crosses the border between two, for some 1 in 100 values, by a step (a third of a typical value): a tenth of a third of the values' norm, halved for
what averaging over keys takes off: 2e-2, and the 2e-2 of the roundings themselves."""
import copy

import pytest
import torch

import tritonformer_b200._lib as L
from test_generate import _model, _teacher
from tritonformer_b200 import linear_int4, quantize_int4, sample_tokens
from tritonformer_b200.generate import Generator
from tritonformer_b200.kvcache import PagedKVCache
from util import norm_rel

gpu = pytest.mark.gpu
pytestmark = gpu


def _dequantized(model, group):
    """The model with the weights that its packed ones stand for."""
    other = copy.deepcopy(model)
    with torch.no_grad():
        for layer in other.layer_list:
            att, mlp = layer.attention, layer.mlp
            for lin in (att.q_proj, att.k_proj, att.v_proj, att.out_proj, mlp.dense_h_to_4h, mlp.dense_4h_to_h):
                lin.weight.copy_(quantize_int4(lin.weight, group).dequantize())
        other.logits_out.weight.copy_(quantize_int4(other.logits_out.weight, group).dequantize())
    return other


@pytest.mark.parametrize("head_dim,alibi,bias,dtype,group", [(64, False, False, torch.float16, 64), (64, True, True, torch.float16, 32),
                                                             (128, True, False, torch.bfloat16, 128), (32, False, True, torch.bfloat16, 64)])
def test_packed_weights_are_the_model_with_what_they_stand_for(head_dim, alibi, bias, dtype, group):
    model = _model(head_dim, 4, 2, alibi, bias, dtype)
    ids = torch.randint(0, 1000, (3, 110), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    with torch.no_grad():
        want = _dequantized(model, group)(torch.nn.functional.pad(ids, (0, 18)), None)[:, 99:110]
    got = _teacher(model, ids, 100, Generator(model, 3, 128, weight_bits=4, weight_group=group))
    assert norm_rel(got, want) < 2e-2
    L.check_status()


@pytest.mark.parametrize("head_dim,alibi,dtype", [(64, False, torch.float16), (64, True, torch.float16), (128, True, torch.bfloat16),
                                                  (32, False, torch.bfloat16)])
@pytest.mark.parametrize("page", [64, 24])
def test_a_prompt_is_its_tokens_one_by_one(page, head_dim, alibi, dtype):
    model = _model(head_dim, 4, 2, alibi, False, dtype)
    ids = torch.randint(0, 1000, (2, 100), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    make = lambda: Generator(model, 2, 128, page, cache_bits=4)  # noqa: E731
    steps = _teacher(model, ids, 1, make())
    for n in (33, 64, 100):
        assert norm_rel(make().prefill(ids[:, :n]), steps[:, n - 1]) < 4e-2
    # and the 16-bit cache's are near: a fourteenth of the largest value is at most half a step
    plain = _teacher(model, ids, 1, Generator(model, 2, 128, page))
    assert 0 < norm_rel(steps, plain) < 0.5
    L.check_status()


def test_everything_in_four_bits_in_a_graph():
    model = _model(alibi=True)
    ids = torch.randint(0, 1000, (3, 90), device="cuda")
    lengths = [90, 1, 40]
    eager, graph = (Generator(model, 3, 128, weight_bits=4, cache_bits=4, graph=g) for g in (False, True))
    a, b = eager.prefill(ids, lengths).clone(), graph.prefill(ids, lengths).clone()
    assert torch.equal(a, b)
    for t in range(20):
        assert torch.equal(eager.step(ids[:, t]), graph.step(ids[:, t]))
    # packed again after the weights have changed
    with torch.no_grad():
        model.logits_out.weight.mul_(2.0)
    before = graph.prefill(ids, lengths).clone()
    graph.pack_weights()
    assert norm_rel(graph.prefill(ids, lengths), 2 * before) < 1e-2 and graph.graph is None
    graph.step(ids[:, 0])


def test_drawn_tokens_are_those_of_the_operator():
    model = _model()
    ids = torch.randint(0, 1000, (4, 30), device="cuda")
    u = torch.rand((4, 12), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    settings = {"temperature": 0.9, "top_k": 50, "top_p": 0.9, "min_p": 0.01}
    got = Generator(model, 4, 64, weight_bits=4, cache_bits=4).generate(ids, None, 12, uniforms=u, **settings)
    gen, want = Generator(model, 4, 64, weight_bits=4, cache_bits=4), []
    logits = gen.prefill(ids)
    for i in range(12):
        want.append(sample_tokens(logits, u[:, i], **settings))
        logits = gen.step(want[-1]) if i < 11 else None
    assert torch.equal(got, torch.stack(want, 1))
    seeded = [Generator(model, 4, 64).generate(ids, None, 8, temperature=1.3, generator=torch.Generator(device="cuda").manual_seed(s))
              for s in (5, 5, 6)]
    assert torch.equal(seeded[0], seeded[1]) and not torch.equal(seeded[0], seeded[2])
    greedy = Generator(model, 4, 64)
    assert torch.equal(greedy.generate(ids, None, 8), greedy.generate(ids, None, 8, temperature=0.0))
    each = torch.tensor([0.0, 1.0, 0.5, 2.0], device="cuda")
    assert torch.equal(greedy.generate(ids, None, 8, temperature=each)[0], greedy.generate(ids, None, 8)[0])


def test_refusals():
    model = _model()
    ids = torch.randint(0, 1000, (2, 10), device="cuda")
    gen = Generator(model, 2, 64)
    for call, text in ((lambda: Generator(model, 2, 64, cache_bits=4, budget=32), "evicted"), (lambda: Generator(model, 2, 64, weight_bits=8), "16 or 4"),
                       (lambda: Generator(model, 2, 64, cache_bits=2), "16 or 4"), (lambda: Generator(model, 2, 64, weight_bits=4, weight_group=16), "32, 64"),
                       (lambda: gen.generate(ids, None, 2, top_k=5), "temperature"), (lambda: gen.generate(ids, None, 2, uniforms=ids.float()), "temperature"),
                       (lambda: gen.generate(ids, None, 2, choose=lambda x: x.argmax(-1), temperature=1.0), "chosen"),
                       (lambda: gen.generate(ids, None, 2, temperature=1.0, uniforms=torch.zeros((2, 3), device="cuda")), "uniforms"),
                       (lambda: gen.generate(ids, None, 2, temperature=-1.0), "temperature")):
        with pytest.raises(AssertionError, match=text):
            call()


def test_a_length_that_does_not_fit_is_reported():
    model = _model()
    ids = torch.randint(0, 1000, (2, 20), device="cuda")
    gen = Generator(model, 2, 64, cache_bits=4)
    gen.prefill(ids, torch.tensor([20, 25], device="cuda"))
    with pytest.raises(RuntimeError, match="length"):
        L.check_status()
    assert L.device_status(reset=True) == 0x7201


def test_two_streams_and_two_graphs_at_once():
    """The operators' calls share no state: what runs beside them, eagerly or from graphs, changes nothing."""
    g = torch.Generator(device="cuda").manual_seed(3)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda").half()  # noqa: E731
    cache = PagedKVCache(64, 4, 64, 64, torch.float16, "cuda", False, 4)
    tables = torch.arange(64, dtype=torch.int32, device="cuda").view(4, 16)
    lengths = torch.tensor([1000, 3, 0, 512], dtype=torch.int32, device="cuda")
    cache.append(tables, torch.zeros_like(lengths), randn(4, 4, 1000, 64), randn(4, 4, 1000, 64), lengths)
    weight = quantize_int4(randn(200, 130))
    sides = [(randn(40, 50304), torch.rand(40, generator=g, device="cuda"), {"top_p": 0.9}, randn(4, 4, 64), randn(1, 200)),
             (randn(30, 30000), torch.rand(30, generator=g, device="cuda"), {"top_k": 300}, randn(4, 12, 64), randn(100, 200))]

    def run(logits, u, settings, q, x):
        return sample_tokens(logits, u, **settings), cache.attend(q, tables, lengths), linear_int4(x, weight)

    want = [run(*side) for side in sides]
    streams = [torch.cuda.Stream() for _ in sides]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for stream, side in zip(streams, sides):
            with torch.cuda.stream(stream):
                got.append(run(*side))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    graphs, got = [], []
    for side in sides:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(run(*side))
    for _ in range(20):
        for out in got:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    L.check_status()
