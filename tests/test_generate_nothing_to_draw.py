"""Generation where a sequence has no token that could be drawn: it alone is concerned."""
import pytest
import torch

import tritonformer_b200._lib as L
from test_generate import _model
from tritonformer_b200.generate import Generator

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("bits", [16, 4])
def test_the_other_sequences_go_on(bits, graph):
    model = _model()
    ids = torch.randint(8, 1000, (3, 40), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    u = torch.rand((3, 6), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    with torch.no_grad():
        model.embed_tokens.weight[7] = float("nan")
    gen = Generator(model, 3, 64, weight_bits=bits, cache_bits=bits, graph=graph)
    want = gen.generate(ids, None, 6, temperature=0.9, top_k=30, uniforms=u)
    assert (want >= 0).all()
    ids[1, 39] = 7  # its last token's logits are NaN, and through its key those of all that follow
    for generator in (gen, Generator(model, 3, 64, weight_bits=bits, cache_bits=bits, graph=graph)):
        for settings in ({"temperature": 0.9, "top_k": 30}, {"temperature": 0.9, "top_k": torch.full((3,), 30, dtype=torch.int32, device="cuda")}):
            got = generator.generate(ids, None, 6, uniforms=u, **settings)
            assert (got[1] == -1).all() and torch.equal(got[[0, 2]], want[[0, 2]])
            assert L.device_status() == 0
    ids[1, 39] = 8
    assert (gen.generate(ids, None, 6, temperature=0.9, top_k=30, uniforms=u) >= 0).all()
