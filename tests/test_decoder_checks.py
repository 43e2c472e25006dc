"""What the paged decoder refuses, on the host: of its rows' adapters before the
cache has room for tokens that no layer will write, and of models."""
import pytest
import torch

from quipsharp_amd.adapters import attach_adapters
from quipsharp_amd.checkpoint import QuantizedLinear
from quipsharp_amd.decode import PagedDecoder

BF, HF, I32 = torch.bfloat16, torch.float16, torch.int32
SIZES = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
             vocab_size=100, max_position_embeddings=128)


def llama(dtype=BF, kind="llama", **more):
    from transformers import AutoModelForCausalLM, LlamaConfig, Qwen2Config, Qwen3Config
    config = {"llama": LlamaConfig, "qwen2": Qwen2Config, "qwen3": Qwen3Config}[kind](**dict(SIZES, **more))
    model = AutoModelForCausalLM.from_config(config, dtype=dtype)
    for layer in model.model.layers:
        for part in (layer.self_attn, layer.mlp):
            for name, lin in list(part.named_children()):
                if isinstance(lin, torch.nn.Linear):
                    setattr(part, name, QuantizedLinear(lin.in_features, lin.out_features, 8, "rht"))
    return model


@pytest.fixture
def decoder(monkeypatch):
    """A decoder of two rows on the CPU whose cache notes that it was advanced."""
    model = llama()
    attach_adapters(model, 3, 8)
    dec = PagedDecoder(model, 2, 64, 16)
    dec.advanced = []
    monkeypatch.setattr(dec.cache, "advance", lambda *a: dec.advanced.append(a))
    return dec


def last_bank(dec):
    return dec.layers[-1].mlp.down_proj.adapters


def strided(dec):
    bank = last_bank(dec)
    bank.down = torch.zeros(3, 8, 2 * bank.down.shape[2], dtype=BF)[:, :, ::2]


SPOILED = [
    (lambda d: setattr(d, "which", d.which.long()), ValueError, "which must be"),
    (lambda d: setattr(d, "which", torch.zeros(3, dtype=I32)), ValueError, "which must be"),
    (lambda d: setattr(d, "which", torch.zeros(2, dtype=I32, device="meta")), ValueError, "which is on"),
    (lambda d: setattr(last_bank(d), "up", last_bank(d).up.half()), TypeError, "adapters 0 are"),
    (lambda d: setattr(last_bank(d), "down", last_bank(d).down[:, :, :128]), ValueError, "512 inputs"),
    (lambda d: setattr(last_bank(d), "scale", last_bank(d).scale[:2]), ValueError, "adapters"),
    (lambda d: setattr(last_bank(d), "scale", last_bank(d).scale.double()), ValueError, r"scales\[0\] must be"),
    (strided, ValueError, "stride 1"),
    (lambda d: attach_adapters(d.model, 5, 8, names=("v_proj",)), ValueError, "5 adapters beside 3"),
    (lambda d: attach_adapters(d.model, 3, 8, names=("gate_proj",), dtype=HF), TypeError, "adapters 0 are"),
]


@pytest.mark.parametrize("spoil,error,message", SPOILED)
def test_adapters_are_refused_before_the_cache_grows(decoder, spoil, error, message):
    spoil(decoder)
    ids = torch.arange(4)
    for call in (lambda: decoder.prompt(ids, [3, 1]), lambda: decoder.score(ids, [3, 1]), lambda: decoder.step(ids[:2])):
        with pytest.raises(error, match=message):
            call()
    assert not decoder.advanced


def test_ranks_and_alignment_are_refused_before_the_cache_grows(decoder):
    bank = last_bank(decoder)
    down, up = bank.down, bank.up
    n, far = down.shape[2], (1 << 24) + 8
    for bank.down, bank.up in ((down[:, :4].contiguous(), up[:, :, :4].contiguous()),
                               (torch.zeros(3 * 8 * n + 4, dtype=BF)[4:].view(3, 8, n), up),
                               (down[:, :1].expand(3, 8, n), up),
                               (torch.empty(7 * far + n, dtype=BF).as_strided((3, 8, n), (0, far, 1)), up)):
        with pytest.raises(ValueError, match="multiple of 8"):
            decoder.step(torch.arange(2))
    bank.down, bank.up = torch.zeros(3, 8, n + 8, dtype=BF)[:, :, :n], up  # rows of a wider tensor are fine
    decoder._check_beside(2)
    with pytest.raises(ValueError, match="524289 tokens"):
        decoder._check_beside((1 << 19) + 1)
    assert not decoder.advanced


def test_other_ids_are_refused_before_the_cache_grows(decoder):
    with pytest.raises(ValueError, match="for 2 rows"):
        decoder.step(torch.arange(3))
    decoder.model.half()
    with pytest.raises(TypeError, match="bf16 models"):
        decoder.step(torch.arange(2))
    assert not decoder.advanced


def test_what_a_score_does_not_give_is_refused_before_the_cache_grows(decoder):
    ids = torch.arange(4)
    for more in (dict(top=65), dict(top=-1), dict(rows=0), dict(rows=-5)):
        with pytest.raises(ValueError, match="alternatives"):
            decoder.score(ids, [3, 1], **more)
    for bad in (ids.float(), ids.to("meta"), ids.short()):
        for call in (lambda: decoder.prompt(bad, [3, 1]), lambda: decoder.score(bad, [3, 1]), lambda: decoder.step(bad[:2])):
            with pytest.raises(ValueError, match="ids must be"):
                call()
    assert not decoder.advanced
    decoder.model.lm_head = torch.nn.Linear(256, 40, dtype=BF)
    with pytest.raises(ValueError, match="41 alternatives"):
        decoder.score(ids, [3, 1], top=41)
    assert not decoder.advanced


@pytest.mark.parametrize("which", [[1], [0, 1, 2], [[0, 1]], 1, [0.5, 1.0], [True, False]])
def test_adapters_of_each_prompt(which):
    """One number for every prompt: one alone is not taken for all of them."""
    from quipsharp_amd.decode import beam_decode, greedy_decode_paged
    prompts = [torch.arange(3), torch.arange(5)]
    for call in (lambda: greedy_decode_paged(None, prompts, 2, which=which), lambda: beam_decode(None, prompts, 1, 2, which=which)):
        with pytest.raises(ValueError, match="for each of 2 prompts"):
            call()
    from quipsharp_amd.decode import _each_prompts
    assert _each_prompts(None, 2).tolist() == [-1, -1] and _each_prompts(torch.tensor([3, 1 << 40]), 2).tolist() == [3, 2 ** 31 - 1]


# ---------------------------------------------------------------------------
# models
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["llama", "qwen2", "qwen3"])
def test_other_activations_are_refused(kind):
    """The step's kernel computes SiLU, the prompt the model's own activation: one that differs would be right in the
    prompt and wrong in every step."""
    heads = dict(head_dim=128) if kind == "qwen3" else {}
    with pytest.raises(ValueError, match="the model has 'relu'"):
        PagedDecoder(llama(kind=kind, hidden_act="relu", **heads), 2, 64, 16)
    for act in ("silu", "swish"):
        assert PagedDecoder(llama(kind=kind, hidden_act=act, **heads), 2, 64, 16).fused_ok == (kind == "qwen3")


def test_static_steps_of_other_activations_run_the_models_own():
    from quipsharp_amd.decode import StaticDecoder
    for act, fused in (("silu", True), ("relu", False)):
        dec = StaticDecoder(llama(kind="qwen3", head_dim=128, hidden_act=act), 1, 32)
        took = []
        dec._decode_step = lambda *a: took.append("kernels")
        dec._prompt_step = lambda *a: took.append("modules")
        dec.step(torch.zeros(1, 1, dtype=torch.long), torch.zeros(1, dtype=torch.long))
        assert took == ["kernels" if fused else "modules"]


@pytest.mark.parametrize("kind", ["llama", "qwen2"])
def test_heads_that_turn_in_part_are_refused(kind):
    """transformers' modules of these models turn whole heads whatever partial_rotary_factor says (the default
    frequencies) or fail (scaled ones)."""
    whole = dict(rope_type="default", rope_theta=1e4)
    assert len(PagedDecoder(llama(kind=kind, rope_parameters=whole), 2, 64, 16).frequencies) == 32
    with pytest.raises(ValueError, match="32 elements of 64"):
        PagedDecoder(llama(kind=kind, rope_parameters=dict(whole, partial_rotary_factor=0.5)), 2, 64, 16)


def test_the_static_decoder_refuses_what_it_does_not_run():
    """Layers without q/k norms, and adapters, which it would leave out, attached before or after it is made."""
    from quipsharp_amd.decode import StaticDecoder
    with pytest.raises(ValueError, match="not llama"):
        StaticDecoder(llama(), 1, 32)
    model = llama(kind="qwen3", head_dim=128)
    dec, ids, pos = StaticDecoder(model, 1, 32), torch.zeros(1, 3, dtype=torch.long), torch.arange(3)
    dec._decode_step = dec._prompt_step = lambda *a: "ran"
    assert dec.step(ids, pos) == dec.step(ids[:, :1], pos[:1]) == "ran"
    banks = attach_adapters(model, 2, 8, names=("down_proj",))
    for n in (3, 1):
        with pytest.raises(ValueError, match="runs no adapters"):
            dec.step(ids[:, :n], pos[:n])
    for layer in model.model.layers:
        layer.mlp.down_proj.adapters = None
    assert len(banks) == 2 and dec.step(ids, pos) == "ran"
