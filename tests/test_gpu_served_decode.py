"""A served decoder's step as a whole: adapters beside its quantized linears,
rotary positions into its paged cache, log probabilities of its tokens
(quipsharp_amd/decode.py), on tiny models against transformers' forward of the
whole sequence, whose linears are given the adapters' products in 32 bits.
Logits are compared in the 2-norm, to 2 % as for the other decoders: the
quantized linears round their activations to fp16."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

VOCAB = 1000
SIZES = dict(hidden_size=512, intermediate_size=1536, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
             vocab_size=VOCAB, tie_word_embeddings=False, max_position_embeddings=512)


def config(kind):
    from transformers import LlamaConfig, Qwen2Config, Qwen3Config
    if kind == "llama":
        return LlamaConfig(**SIZES, head_dim=128, rope_parameters=dict(
            rope_type="llama3", rope_theta=500000.0, factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
            original_max_position_embeddings=64))
    if kind == "llama64":
        return LlamaConfig(**dict(SIZES, num_attention_heads=8), head_dim=64)
    if kind == "qwen2":
        return Qwen2Config(**SIZES, rope_parameters=dict(rope_type="yarn", rope_theta=1e6, factor=4.0,
                                                         original_max_position_embeddings=128))
    return Qwen3Config(**SIZES, head_dim=128)


@pytest.fixture(scope="module", params=["llama", "llama64", "qwen2", "qwen3"])
def model(dev, request):
    from quipsharp_amd.adapters import attach_adapters
    from quipsharp_amd.checkpoint import QuantizedLinear
    from quipsharp_amd.decode import random_quantized_model
    m = random_quantized_model(config(request.param), dev, seed=3)
    g = torch.Generator().manual_seed(4)
    for mod in m.modules():
        if isinstance(mod, QuantizedLinear) and mod.bias is not None:
            mod.bias.copy_(torch.randn(mod.bias.shape, generator=g) * 0.5)
    for name, bank in attach_adapters(m, 3, 12, names=("q_proj", "v_proj", "o_proj", "gate_proj", "down_proj")).items():
        for i, r in enumerate((12, 4)):  # the third stays empty
            down = torch.randn(r, bank.down.shape[2], generator=g) * bank.down.shape[2] ** -0.5
            bank.load(i, down.to(dev), (torch.randn(bank.up.shape[1], r, generator=g) * 0.3).to(dev), 1.0 + i)
    return m


def ids_of(n, seed, dev):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).to(dev)


def whole(model, ids, adapter):
    """Logits of every position, every linear with its adapter."""
    from quipsharp_amd.checkpoint import QuantizedLinear
    hooks = []

    def beside(mod, args, out):
        b = mod.adapters
        x = args[0].float()
        return (out.float() + b.scale[adapter] * ((x @ b.down[adapter].float().t()) @ b.up[adapter].float().t())).to(out.dtype)

    if adapter >= 0:
        hooks = [m.register_forward_hook(beside) for m in model.modules()
                 if isinstance(m, QuantizedLinear) and getattr(m, "adapters", None) is not None]
    try:
        with torch.no_grad():
            return model(input_ids=ids[None], use_cache=False).logits[0].float()
    finally:
        for h in hooks:
            h.remove()


def near(got, want):
    assert ((got.float() - want).norm() / want.norm()).item() < 2e-2


def test_prompts_and_steps(model, dev):
    """Rows with two adapters, an empty one and none: prompts of different lengths, a second turn, single tokens, and an
    adapter that a row changes to."""
    from quipsharp_amd.decode import PagedDecoder
    dec = PagedDecoder(model, 4, 128, page=16)
    which = [0, 1, -1, 2]
    dec.which.copy_(torch.tensor(which, dtype=torch.int32))
    rows = [ids_of(n, n, dev) for n in (33, 17, 5, 70)]
    got = dec.prompt(torch.cat(rows), [len(r) for r in rows])
    for r in range(4):
        near(got[r], whole(model, rows[r], which[r])[-1])
    assert (whole(model, rows[0], 0)[-1] - whole(model, rows[0], -1)[-1]).norm() > 0.2 * whole(model, rows[0], -1)[-1].norm()
    more = [ids_of(n, 50 + n, dev) for n in (0, 24, 1, 0)]
    got = dec.prompt(torch.cat(more), [len(r) for r in more])
    rows = [torch.cat(t) for t in zip(rows, more)]
    for r, x in ((1, got[0]), (2, got[1])):
        near(x, whole(model, rows[r], which[r])[-1])
    for step in range(3):
        new = ids_of(4, 100 + step, dev)
        got = dec.step(new)
        rows = [torch.cat([t, new[r:r + 1]]) for r, t in enumerate(rows)]
        for r in range(4):
            near(got[r], whole(model, rows[r], which[r])[-1])


def test_forked_rows_keep_their_adapters(model, dev):
    from quipsharp_amd.decode import PagedDecoder
    dec = PagedDecoder(model, 4, 64, page=16)
    dec.which.copy_(torch.tensor([0, 1, -1, -1], dtype=torch.int32))
    first = [ids_of(21, 7, dev), ids_of(16, 8, dev)]
    dec.prompt(torch.cat(first), [21, 16, 0, 0])
    rows, which = first + [first[0][:0]] * 2, [0, 1, -1, -1]
    for step, parents in enumerate(([1, 0, 1, 0], [3, 3, 2, 0])):
        new = ids_of(4, 60 + step, dev)
        got = dec.step(new, torch.tensor(parents, dtype=torch.int32, device=dev))
        rows = [torch.cat([rows[p], new[i:i + 1]]) for i, p in enumerate(parents)]
        which = [which[p] for p in parents]
        assert dec.which.tolist() == which
        for r in range(4):
            near(got[r], whole(model, rows[r], which[r])[-1])
    dec.step(ids_of(4, 70, dev), torch.tensor([0, -1, 9, 1], dtype=torch.int32, device=dev))
    assert dec.which.tolist() == [which[0], -1, -1, which[1]]


def test_scores_of_prompts(model, dev):
    """Every token's log probability, entropy, rank and alternatives are those of its own logits, row by row."""
    from quipsharp_amd.decode import PagedDecoder
    dec = PagedDecoder(model, 3, 128, page=16)
    which = [0, -1, 1]
    dec.which.copy_(torch.tensor(which, dtype=torch.int32))
    rows = [ids_of(n, 20 + n, dev) for n in (40, 1, 27)]
    got = dec.score(torch.cat(rows), [len(r) for r in rows], top=4, rows=32)
    assert [tuple(t.shape) for t in got] == [(68,), (68,), (68,), (68, 4), (68, 4)]
    at = 0
    for r, ids in enumerate(rows):
        n = len(ids)
        logits = whole(model, ids, which[r])
        logp = torch.log_softmax(logits.double(), 1)
        lp, H, rank, best, tokens = (t[at:at + n] for t in got)
        # a log probability is off by at most twice what its logits are
        off = 2 * 0.02 * logits.norm(dim=1)
        assert ((lp[:-1] - logp[:-1].gather(1, ids[1:, None])[:, 0]).abs() <= off[:-1]).all()
        assert lp[-1] == 0 and rank[-1] == -1 and (rank[:-1] >= 0).all()
        entropy = -(logp.exp() * logp).sum(1)
        assert ((H - entropy).abs() <= off * (1 + entropy)).all()
        assert ((best - logp.gather(1, tokens.long())).abs() <= off[:, None]).all()
        assert (best[:, 1:] <= best[:, :-1]).all()
        at += n


def test_greedy_decode_with_scores(model, dev):
    """Replayed steps give the eager ones' tokens and scores; each token is the best alternative, and the scores are the
    sequences' log probabilities."""
    from quipsharp_amd.decode import greedy_decode_paged
    prompts, which, new = [ids_of(n, 30 + n, dev) for n in (19, 40, 3)], [1, -1, 0], 12
    got = greedy_decode_paged(model, prompts, new, which=which, top=3, page=16)
    eager = greedy_decode_paged(model, prompts, new, which=which, top=3, use_graph=False, page=16)
    assert all(torch.equal(a, b) for a, b in zip(got, eager))
    tokens, logp, entropy, best, alternatives = got
    assert torch.equal(best[:, :, 0], logp) and (best[:, :, 1:] <= best[:, :, :-1]).all()
    top = best.gather(2, (alternatives == tokens[:, :, None]).int().argmax(2, keepdim=True))[:, :, 0]
    assert torch.equal(top, logp)
    for r, p in enumerate(prompts):
        logits = whole(model, torch.cat([p, tokens[r]]), which[r])[len(p) - 1:-1]
        want = torch.log_softmax(logits.double(), 1).gather(1, tokens[r][:, None])[:, 0]
        assert ((logp[r] - want).abs() <= 2 * 0.02 * logits.norm(dim=1)).all()


def test_rows_adapters_given_as_a_new_tensor(model, dev):
    """A step takes the ``which`` that the decoder has then, a tensor of its own among them, and a refused prompt leaves
    nothing behind."""
    from quipsharp_amd.decode import PagedDecoder
    one, two = (PagedDecoder(model, 2, 64, 16) for _ in range(2))
    ids, counts = ids_of(12, 20, dev), [7, 5]
    one.prompt(ids, counts), two.prompt(ids, counts)
    one.which.copy_(torch.tensor([1, 0], dtype=torch.int32))
    two.which = torch.tensor([1, 0], dtype=torch.int32, device=dev)
    assert torch.equal(one.step(ids[:2]), two.step(ids[:2]))
    two.which = two.which.long()
    with pytest.raises(ValueError, match="which must be"):
        two.prompt(ids[:3], [2, 1])
    two.which = one.which
    two.cache.lengths.copy_(one.cache.lengths)
    assert torch.equal(one.step(ids[2:4]), two.step(ids[2:4]))


@pytest.mark.parametrize("window", [0, 24])
def test_a_captured_step_follows_the_rows_adapters(model, dev, window):
    """Replays, with other adapters and parents from one to the next and eager work between, give what an eager
    decoder's steps give."""
    from quipsharp_amd.decode import PagedDecoder
    captured, eager = (PagedDecoder(model, 3, 96, page=16, window=window, sinks=4 if window else 0) for _ in range(2))
    prompts = [ids_of(n, 80 + n, dev) for n in (30, 17, 5)]
    ids, parents = torch.zeros(3, dtype=torch.long, device=dev), torch.arange(3, dtype=torch.int32, device=dev)
    for dec in (captured, eager):
        dec.which.copy_(torch.tensor([0, -1, 1], dtype=torch.int32))
        dec.prompt(torch.cat(prompts), [len(p) for p in prompts])
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            dec.step(ids, parents)  # loads what the first call loads
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = captured.step(ids, parents)
    for step, (which, order) in enumerate((([0, -1, 1], [0, 1, 2]), ([1, 1, -1], [2, 1, 0]), ([2, 0, 0], [0, 0, 1]), (None, [0, 1, 2]))):
        ids.copy_(ids_of(3, 90 + step, dev))
        parents.copy_(torch.tensor(order, dtype=torch.int32))
        if which is not None:
            for dec in (captured, eager):
                dec.which.copy_(torch.tensor(which, dtype=torch.int32))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, eager.step(ids, parents))
        assert torch.equal(captured.which, eager.which)


def test_beam_search_with_adapters(model, dev):
    """Beams of one request keep its adapters; one beam is greedy decode."""
    from quipsharp_amd.decode import beam_decode, greedy_decode_paged
    prompts, which = [ids_of(19, 9, dev), ids_of(33, 10, dev)], [0, 1]
    tokens, scores, _, _ = beam_decode(model, prompts, 3, 8, page=16, which=which)
    for r, p in enumerate(prompts):
        for b in range(3):
            logits = whole(model, torch.cat([p, tokens[r, b]]), which[r])[len(p) - 1:-1]
            logp = torch.log_softmax(logits.double(), 1).gather(1, tokens[r, b][:, None]).sum()
            assert (scores[r, b] - logp).abs().item() <= 2 * 8 * 0.02 * logits.norm(dim=1).max().item()
    one = beam_decode(model, prompts[:1], 1, 8, page=16, which=which[:1])
    greedy = greedy_decode_paged(model, prompts[:1], 8, which=which[:1], page=16)
    assert torch.equal(one[0][0], greedy[0])
    assert torch.allclose(one[1][0, 0].double(), greedy[1][0].double().sum(), rtol=0, atol=8 * 5e-6)


def test_perplexity(model, dev):
    from quipsharp_amd.decode import perplexity
    ids = ids_of(95, 11, dev)
    total, count = 0.0, 0
    for part in ids.split(40):
        logits = whole(model, part, -1)[:-1].double()
        total -= torch.log_softmax(logits, 1).gather(1, part[1:, None]).sum().item()
        count += len(part) - 1
    assert math.isclose(perplexity(model, ids, 40), math.exp(total / count), rel_tol=1e-4)
    with pytest.raises(ValueError, match="no token has one before it"):
        perplexity(model, ids[:1])


def test_other_models_are_refused(dev):
    from transformers import MistralConfig
    from quipsharp_amd.decode import PagedDecoder, random_quantized_model
    m = random_quantized_model(MistralConfig(**SIZES, head_dim=128), dev, seed=1)
    with pytest.raises(ValueError, match="not mistral"):
        PagedDecoder(m, 1, 64)
    m = random_quantized_model(config("llama"), dev, seed=1)
    m.config.rope_parameters = dict(rope_type="longrope", rope_theta=1e4)
    with pytest.raises(NotImplementedError, match="longrope"):
        PagedDecoder(m, 1, 64)
