"""A served decoder's refusals leave its cache as it was."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = dict(hidden_size=512, intermediate_size=1536, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
             vocab_size=1000, tie_word_embeddings=False, max_position_embeddings=512)


@pytest.fixture(scope="module")
def model(dev):
    from transformers import LlamaConfig
    from quipsharp_amd.adapters import attach_adapters
    from quipsharp_amd.decode import random_quantized_model
    m = random_quantized_model(LlamaConfig(**SIZES, head_dim=128), dev, seed=5)
    g = torch.Generator().manual_seed(6)
    for bank in attach_adapters(m, 2, 8).values():
        bank.load(0, torch.randn(8, bank.down.shape[2], generator=g).to(dev) * 0.05, torch.randn(bank.up.shape[1], 8, generator=g).to(dev) * 0.3)
    return m


def test_a_refused_call_leaves_the_cache(model, dev):
    """After refusals a decoder goes on as one that had none."""
    from quipsharp_amd.decode import PagedDecoder
    one, two = (PagedDecoder(model, 2, 64, 16) for _ in range(2))
    ids = torch.randint(0, 1000, (20,), generator=torch.Generator().manual_seed(7)).to(dev)
    which = torch.tensor([0, -1], dtype=torch.int32, device=dev)
    one.which.copy_(which), two.which.copy_(which)
    assert torch.equal(one.prompt(ids[:12], [7, 5]), two.prompt(ids[:12], [7, 5]))
    books = lambda: [t.clone() for t in (two.cache.table, two.cache.lengths, two.cache.refs, two.cache.over, two.cache.missing)]  # noqa: E731
    before, bank = books(), model.model.layers[1].mlp.up_proj.adapters

    def refused(error, message):
        for call in (lambda: two.prompt(ids[:3], [2, 1]), lambda: two.score(ids[:3], [2, 1]), lambda: two.step(ids[:2]),
                     lambda: two.step(ids[:2], torch.tensor([1, 0], dtype=torch.int32, device=dev))):
            with pytest.raises(error, match=message):
                call()
        assert all(torch.equal(a, b) for a, b in zip(before, books()))

    two.which = two.which.long()
    refused(ValueError, "which must be")
    two.which = which.clone()
    up = bank.up
    try:
        bank.up = up.half()
        refused(TypeError, "adapters 1 are")
    finally:
        bank.up = up
    with pytest.raises(ValueError, match="for 2 rows"):
        two.step(ids[:3])
    assert all(torch.equal(a, b) for a, b in zip(before, books())) and torch.equal(two.which, which)
    assert torch.equal(one.prompt(ids[12:16], [1, 3]), two.prompt(ids[12:16], [1, 3]))
    assert torch.equal(one.step(ids[16:18]), two.step(ids[16:18]))
