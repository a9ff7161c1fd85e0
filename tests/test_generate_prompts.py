"""Prompts as they come: lengths that do not fit, padding of any kind, models in other types."""
import pytest
import torch

import tritonformer_b200._lib as L
from test_generate import _model, _teacher
from tritonformer_b200.generate import Generator, _prompt_lengths
from util import norm_rel

gpu = pytest.mark.gpu


@pytest.mark.parametrize("bad", [[0, 5], [5, 9], [-1, 5], [5], [5, 5, 5], [1.0, 2.0], [True, True], [[5, 5]]])
def test_lengths_that_the_host_refuses(bad):
    for lengths in (bad, torch.tensor(bad)):
        with pytest.raises(AssertionError, match="tokens"):
            _prompt_lengths(lengths, 2, 8, "cpu")


def test_lengths_that_the_host_takes():
    for lengths in ([1, 8], (1, 8), torch.tensor([1, 8]), torch.tensor([1, 8], dtype=torch.int16)):
        counts, bad = _prompt_lengths(lengths, 2, 8, "cpu")
        assert counts.tolist() == [1, 8] and counts.dtype is torch.int32 and bad is None
    assert _prompt_lengths(None, 2, 8, "cpu")[0].tolist() == [8, 8]


@gpu
@pytest.mark.parametrize("budget", [None, 20])
def test_lengths_on_the_gpu_that_do_not_fit(budget):
    """They are taken as the nearest that do, here where the model has no position behind the prompt's padding; it is reported."""
    model = _model(layers=1, positions=64)
    ids = torch.randint(0, 1000, (4, 50), device="cuda")
    gen = Generator(model, 4, 64, budget=budget)
    want = gen.prefill(ids, [1, 50, 50, 7])
    assert L.device_status() == 0
    got = gen.prefill(ids, torch.tensor([0, 64, 2 ** 40, 7], device="cuda"))
    assert L.device_status(reset=True) == 0x7201
    assert torch.equal(want, got)
    assert gen.next.tolist() == [1, 50, 50, 7]
    for value in (torch.tensor([1, 50, 50, 7], device="cuda"), torch.tensor([1, 50, 50, 7], device="cuda", dtype=torch.int16)):
        assert torch.equal(want, gen.prefill(ids, value)) and L.device_status() == 0
    for _ in range(14):
        logits = gen.step(ids[:, 0])
    assert logits.isfinite().all() and gen.next.tolist() == [15, 64, 64, 21]
    L.check_status()


@gpu
@pytest.mark.parametrize("pad", [-1, -100, 1 << 40])
def test_padding_may_be_any_number(pad):
    model = _model(layers=1)
    ids = torch.randint(0, 1000, (3, 70), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    lengths = [70, 33, 1]
    for at in (lengths, torch.tensor(lengths, device="cuda")):
        gen = Generator(model, 3, 128, budget=24)
        want = gen.prefill(ids, lengths)
        padded = ids.clone()
        for b, n in enumerate(lengths):
            padded[b, n:] = pad
        assert torch.equal(want, gen.prefill(padded, at)) and L.device_status() == 0
        assert torch.equal(want, gen.prefill(padded.cpu(), at)) and L.device_status() == 0


@gpu
@pytest.mark.parametrize("heads", [4, 12])
@pytest.mark.parametrize("budget", [None, 128])
def test_alibi_models_moved_to_bf16(heads, budget):
    """Their table was made in fp16 and rounded again; the logits are the model's own."""
    model = _model(heads=heads, alibi=True).to(torch.bfloat16).fuse_projection_weights()
    assert model.attn_bias.dtype is torch.bfloat16
    ids = torch.randint(0, 1000, (2, 128), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    with torch.no_grad():
        want = model(ids, None)[:, 99:]
    got = _teacher(model, ids, 100, Generator(model, 2, 128, budget=budget))
    assert norm_rel(got, want) < 2e-2  # as in test_generate.py
    graph = _teacher(model, ids, 100, Generator(model, 2, 128, budget=budget, graph=True))
    assert torch.equal(got, graph)
    L.check_status()


@gpu
def test_a_bias_that_is_not_alibi_is_refused():
    model = _model(heads=12, alibi=True)
    model.attn_bias = model.attn_bias * 1.05
    ids = torch.randint(0, 1000, (1, 10), device="cuda")
    gen = Generator(model, 1, 64)
    with pytest.raises(AssertionError, match="no other bias"):
        gen.prefill(ids)
        gen.step(ids[:, 0])


@gpu
@pytest.mark.parametrize("alibi", [False, True])
def test_prompts_up_to_the_last_position(alibi):
    """Whole tiles of 64 may be more than the model's positions: 100 of them here."""
    model = _model(layers=2, alibi=alibi, positions=100)
    ids = torch.randint(0, 1000, (2, 100), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    steps = _teacher(model, ids, 60, Generator(model, 2, 100))
    for t in (65, 99, 100):
        for budget in (None, 100):
            got = Generator(model, 2, 100, budget=budget).prefill(ids[:, :t])
            assert norm_rel(got, steps[:, t - 60]) < 2e-2  # as in test_generate.py
    L.check_status()


@gpu
def test_a_captured_step_follows_the_models_bias():
    """A table of other slopes, in another tensor and in the same one; the step that was captured before has gone."""
    model = _model(alibi=True)
    ids = torch.randint(0, 1000, (2, 60), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    gen = Generator(model, 2, 128, graph=True)
    seen = []
    for change in (lambda: None, lambda: setattr(model, "attn_bias", model.attn_bias * 0.25), lambda: model.attn_bias.mul_(8)):
        change()
        want = _teacher(model, ids, 40, Generator(model, 2, 128))
        assert torch.equal(want, _teacher(model, ids, 40, gen))
        assert all(not torch.equal(want, x) for x in seen)
        seen.append(want)
    graph = gen.graph
    _teacher(model, ids, 40, gen)
    assert gen.graph is graph  # nothing has changed
    L.check_status()


@gpu
def test_a_captured_step_follows_the_models_weights():
    """Weights that are written to in place, and weights that have moved."""
    model = _model()
    ids = torch.randint(0, 1000, (2, 60), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    gen = Generator(model, 2, 128, graph=True)
    _teacher(model, ids, 40, gen)
    graph = gen.graph
    with torch.no_grad():
        model.layer_list[0].attention.v_proj.weight.mul_(0.5)
    want = _teacher(model, ids, 40, Generator(model, 2, 128))
    assert torch.equal(want, _teacher(model, ids, 40, gen)) and gen.graph is graph
    model.fuse_projection_weights()
    with torch.no_grad():
        model.layer_list[1].attention.v_proj.weight.mul_(0.5)
    want = _teacher(model, ids, 40, Generator(model, 2, 128))
    assert torch.equal(want, _teacher(model, ids, 40, gen)) and gen.graph is not graph
    L.check_status()
