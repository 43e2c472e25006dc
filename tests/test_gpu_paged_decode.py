"""The paged decoder and the beam search (quipsharp_amd/decode.py) on a tiny
Qwen3-shaped model, against transformers' forward of the whole sequence.
Logits are compared in the 2-norm, to 2 % as for the static decoder: the
quantized linears round their activations to fp16."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(dev):
    from transformers import Qwen3Config
    from quipsharp_amd.decode import random_quantized_model
    cfg = Qwen3Config(hidden_size=512, intermediate_size=1536, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128, vocab_size=1000, tie_word_embeddings=False,
                      max_position_embeddings=512)
    return random_quantized_model(cfg, dev, seed=2)


def ids_of(n, seed, dev):
    return torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(seed)).to(dev)


def whole(model, ids, window=0, sinks=0):
    """Logits of every position, with the positions that a window hides masked."""
    n = len(ids)
    i, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
    see = (j <= i) & ((j > i - window) | (j < sinks)) if window else j <= i
    mask = torch.zeros(n, n).masked_fill(~see, torch.finfo(torch.bfloat16).min).bfloat16().to(ids.device)
    with torch.no_grad():
        return model(input_ids=ids[None], attention_mask=mask[None, None], use_cache=False).logits[0].float()


def near(got, want):
    assert ((got.float() - want).norm() / want.norm()).item() < 2e-2


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_rows_of_different_lengths(model, dev, window, sinks):
    """Prompts of different lengths at once, a second turn of one row and the first of another while the third waits,
    then single tokens for all."""
    from quipsharp_amd.decode import PagedDecoder
    dec = PagedDecoder(model, 3, 128, page=16, window=window, sinks=sinks)
    rows = [ids_of(33, 1, dev), ids_of(17, 2, dev), ids_of(0, 3, dev)]
    got = dec.prompt(torch.cat(rows), [33, 17, 0])
    for r in range(2):
        near(got[r], whole(model, rows[r], window, sinks)[-1])
    more = [ids_of(0, 4, dev), ids_of(24, 5, dev), ids_of(5, 6, dev)]
    got = dec.prompt(torch.cat(more), [0, 24, 5])
    rows = [torch.cat(t) for t in zip(rows, more)]
    for r, g in ((1, got[0]), (2, got[1])):
        near(g, whole(model, rows[r], window, sinks)[-1])
    for step in range(20):
        new = ids_of(3, 100 + step, dev)
        got = dec.step(new)
        rows = [torch.cat([t, new[r:r + 1]]) for r, t in enumerate(rows)]
        if step % 6 == 0 or step == 19:
            for r in range(3):
                near(got[r], whole(model, rows[r], window, sinks)[-1])
    assert dec.cache.short.item() == 0 and dec.cache.lengths.tolist() == [len(t) for t in rows]
    if window:
        # pages that no later token sees are free again
        for r, t in enumerate(rows):
            n = len(t)
            held = {c for c in range(-(-n // 16)) if c * 16 < sinks or (c + 1) * 16 > n - window + 1}
            assert {c for c, p in enumerate(dec.cache.table[r].tolist()) if p >= 0} == held


def test_forked_rows(model, dev):
    """Rows that go on from others' pages."""
    from quipsharp_amd.decode import PagedDecoder
    dec = PagedDecoder(model, 4, 64, page=16)
    first = [ids_of(21, 7, dev), ids_of(16, 8, dev)]
    dec.prompt(torch.cat(first), [21, 16, 0, 0])
    rows = first + [first[0][:0]] * 2
    for step, parents in enumerate(([0, 0, 1, 1], [1, 0, 0, 3], [2, 2, 2, 0], [0, 1, 2, 3])):
        new = ids_of(4, 50 + step, dev)
        got = dec.step(new, torch.tensor(parents, dtype=torch.int32, device=dev))
        rows = [torch.cat([rows[p], new[i:i + 1]]) for i, p in enumerate(parents)]
        for r in range(4):
            near(got[r], whole(model, rows[r])[-1])


def test_beam_search(model, dev):
    """Replayed steps give the eager ones' tokens, scores are the sequences' log probabilities, and a beam that ended
    goes on with the end."""
    from quipsharp_amd.decode import beam_decode
    prompts = [ids_of(19, 9, dev), ids_of(40, 10, dev), ids_of(16, 11, dev)]
    new = 20
    tokens, scores, _, _ = beam_decode(model, prompts, 4, new, page=16)
    eager = beam_decode(model, prompts, 4, new, use_graph=False, page=16)
    assert torch.equal(tokens, eager[0]) and torch.equal(scores, eager[1])
    assert (scores[:, 1:] <= scores[:, :-1]).all()
    for r, p in enumerate(prompts):
        assert len({tuple(t.tolist()) for t in tokens[r]}) == 4
        for b in range(4):
            ids = torch.cat([p, tokens[r, b]])
            logits = whole(model, ids)[len(p) - 1:-1]
            logp = torch.log_softmax(logits.double(), 1).gather(1, tokens[r, b][:, None]).sum()
            # a log probability is off by at most twice what its logits are
            assert (scores[r, b] - logp).abs().item() <= 2 * new * 0.02 * logits.abs().max().item()
    eos = tokens[0, 0, 3].item()
    ended, _, _, _ = beam_decode(model, prompts, 4, new, eos=eos, page=16)
    for t in ended.view(-1, new):
        at = (t == eos).nonzero()
        if len(at):
            assert (t[at[0, 0]:] == eos).all()


def test_one_beam_is_greedy(model, dev):
    from quipsharp_amd.decode import PagedDecoder, beam_decode
    p = ids_of(30, 12, dev)
    tokens, _, _, _ = beam_decode(model, [p], 1, 12, page=16)
    dec = PagedDecoder(model, 1, 48, page=16)
    last = dec.prompt(p, [30]).argmax(-1)
    for i in range(12):
        assert tokens[0, 0, i] == last[0]
        last = dec.step(last).argmax(-1)


def test_the_last_page_of_a_row_is_whole(model, dev):
    """max_len ends inside a page: the positions up to the page's end work like the others, and a step beyond them is
    counted."""
    from quipsharp_amd.decode import PagedDecoder
    dec = PagedDecoder(model, 2, 20, page=16)
    rows = [ids_of(17, 13, dev), ids_of(9, 14, dev)]
    dec.prompt(torch.cat(rows), [17, 9])
    for step in range(15):
        new = ids_of(2, 200 + step, dev)
        got = dec.step(new)
        rows = [torch.cat([t, new[r:r + 1]]) for r, t in enumerate(rows)]
        for r in range(2):
            near(got[r], whole(model, rows[r])[-1])
    assert dec.cache.short.item() == 0 and dec.cache.lengths.tolist() == [32, 24]
    dec.step(ids_of(2, 300, dev))
    assert dec.cache.short.item() == 1


def test_a_short_cache_is_told(model, dev):
    """A prompt that gets no room raises; a step that gets none is told by the next check or prompt, also where later
    steps had all that they asked for."""
    from quipsharp_amd.decode import PagedDecoder
    with pytest.raises(RuntimeError, match="short of 2 pages"):
        PagedDecoder(model, 2, 64, page=16, pages=3).prompt(ids_of(50, 15, dev), [33, 17])
    with pytest.raises(RuntimeError, match="short of 1 pages"):
        PagedDecoder(model, 2, 32, page=16).prompt(ids_of(50, 15, dev), [33, 17])
    dec = PagedDecoder(model, 2, 64, page=16, pages=3)
    dec.prompt(ids_of(31, 16, dev), [16, 15])
    dec.cache.check()
    for step in range(2):  # row 1 fills its page, then wants one that row 0 took
        dec.step(ids_of(2, 400 + step, dev))
    dec.cache.free(torch.tensor([True, False], device=dev))
    dec.cache.advance(0)
    assert dec.cache.short.item() == 0 and dec.cache.missing.item() == 1
    with pytest.raises(RuntimeError, match="short of 1 pages"):
        dec.cache.check()
    with pytest.raises(RuntimeError, match="short of 1 pages"):
        dec.prompt(ids_of(3, 17, dev), [0, 3])
    dec.cache.missing.zero_()
    dec.prompt(ids_of(3, 17, dev), [0, 3])


@pytest.mark.parametrize("use_graph", [False, True])
def test_beam_search_tells_a_shortage_of_any_step(model, dev, use_graph, monkeypatch):
    """The first step has no page for the second beam's copy; the others ask for none."""
    from quipsharp_amd import decode

    class Fewer(decode.PagedDecoder):
        def __init__(self, model, rows, max_len, page, pages):
            super().__init__(model, rows, max_len, page, 2)

    monkeypatch.setattr(decode, "PagedDecoder", Fewer)
    with pytest.raises(RuntimeError, match="short of"):
        decode.beam_decode(model, [ids_of(19, 18, dev)], 2, 8, use_graph=use_graph, page=16)
