"""What the operators around a served step's linears refuse, on the host, and the
frequencies of rotary positions: adapters, rotary positions with the cache
write, log probabilities of given tokens."""
import ctypes
import math

import pytest
import torch

from quipsharp_amd import _lib
from quipsharp_amd.adapters import Adapters, add_adapters, attach_adapters
from quipsharp_amd.logprobs import token_logprobs
from quipsharp_amd.rope import append_rotated, rope_frequencies

BF, HF, I32 = torch.bfloat16, torch.float16, torch.int32
P = ctypes.c_void_p(4096)


# ---------------------------------------------------------------------------
# adapters
# ---------------------------------------------------------------------------

def beside(**over):
    a = dict(ys=[torch.zeros(3, 40, dtype=BF)], x=torch.zeros(3, 64, dtype=BF), which=torch.zeros(3, dtype=I32),
             downs=[torch.zeros(2, 8, 64, dtype=BF)], ups=[torch.zeros(2, 40, 8, dtype=BF)], scales=[torch.zeros(2)])
    a.update(over)
    return a


@pytest.mark.parametrize("over,error,message", [
    (dict(x=torch.zeros(3, 64)), TypeError, "unsupported dtype"),
    (dict(x=torch.zeros(3, 1, 64, dtype=BF)), ValueError, "x must be"),
    (dict(x=torch.zeros(3, 128, dtype=BF)[:, ::2]), ValueError, "lie together"),
    (dict(which=torch.zeros(3, dtype=torch.int64)), ValueError, "which must be"),
    (dict(which=torch.zeros(4, dtype=I32)), ValueError, "which must be"),
    (dict(which=torch.zeros(3, dtype=I32, device="meta")), ValueError, "which is on"),
    (dict(ys=[torch.zeros(2, 40, dtype=BF)]), ValueError, r"ys\[0\] must be"),
    (dict(ys=[torch.zeros(3, 41, dtype=BF)]), ValueError, "41 outputs"),
    (dict(ys=[torch.zeros(3, 40, dtype=HF)]), TypeError, r"ys\[0\] is"),
    (dict(ys=[torch.zeros(3, 40, dtype=BF)] * 2), ValueError, "2 outputs for 1"),
    (dict(ys=[], downs=[], ups=[], scales=[]), ValueError, "1 to 4 linears"),
    (dict(downs=[torch.zeros(2, 8, 32, dtype=BF)]), ValueError, "64 inputs"),
    (dict(ups=[torch.zeros(3, 40, 8, dtype=BF)]), ValueError, "adapters 0"),
    (dict(ups=[torch.zeros(2, 40, 16, dtype=BF)]), ValueError, "adapters 0"),
    (dict(downs=[torch.zeros(2, 8, 64, dtype=HF)]), TypeError, "adapters 0 are"),
    (dict(ups=[torch.zeros(2, 8, 40, dtype=BF).transpose(1, 2)]), ValueError, "stride 1"),
    (dict(scales=[torch.zeros(3)]), ValueError, r"scales\[0\] must be"),
    (dict(scales=[torch.zeros(2, dtype=BF)]), ValueError, r"scales\[0\] must be"),
    (dict(scales=[torch.zeros(2, device="meta")]), ValueError, "adapters 0 are on"),
    (dict(outs=[torch.zeros(3, 41, dtype=BF)]), ValueError, r"outs\[0\] must be"),
    (dict(outs=[]), ValueError, "0 outs"),
    (dict(), RuntimeError, "runs on the GPU"),
])
def test_adapters_refuse(over, error, message):
    with pytest.raises(error, match=message):
        add_adapters(**beside(**over))


def test_adapters_refuse_what_does_not_go_together():
    a = beside()
    two = {k: v * 2 for k, v in a.items() if isinstance(v, list)}
    two["downs"] = [a["downs"][0], torch.zeros(3, 8, 64, dtype=BF)]
    two["ups"] = [a["ups"][0], torch.zeros(3, 40, 8, dtype=BF)]
    with pytest.raises(ValueError, match="3 adapters beside 2"):
        add_adapters(**beside(**two))
    out = torch.zeros(3, 40, dtype=BF)
    with pytest.raises(ValueError, match="of its own"):
        add_adapters(**beside(ys=a["ys"] * 2, downs=a["downs"] * 2, ups=a["ups"] * 2, scales=a["scales"] * 2, outs=[out, out]))
    with pytest.raises(ValueError, match="no adapters"):
        add_adapters(**beside(downs=[torch.zeros(0, 8, 64, dtype=BF)], ups=[torch.zeros(0, 40, 8, dtype=BF)], scales=[torch.zeros(0)]))


def test_bank_refuses():
    for bad in (dict(rank=129), dict(rank=0), dict(in_features=60), dict(count=0), dict(out_features=0)):
        with pytest.raises(ValueError, match="adapters of rank"):
            Adapters(**dict(dict(count=2, rank=8, in_features=64, out_features=40, device="cpu"), **bad))
    with pytest.raises(TypeError, match="unsupported dtype"):
        Adapters(2, 8, 64, 40, dtype=torch.float32, device="cpu")
    bank = Adapters(2, 8, 64, 40, device="cpu")
    with pytest.raises(ValueError, match="for adapters of rank 8"):
        bank.load(0, torch.zeros(9, 64), torch.zeros(40, 9))
    with pytest.raises(ValueError, match="for adapters of rank 8"):
        bank.load(0, torch.zeros(8, 64), torch.zeros(41, 8))
    with pytest.raises(IndexError, match="adapter 2 of 2"):
        bank.load(2, torch.zeros(8, 64), torch.zeros(40, 8))
    bank.load(1, torch.ones(3, 64), torch.ones(40, 3), 2.0)
    assert bank.down[1].sum() == 192 and bank.up[1].sum() == 120 and bank.scale.tolist() == [0.0, 2.0]
    bank.clear(1)
    assert not bank.down.any() and not bank.up.any() and not bank.scale.any()


def test_bank_takes_its_own_values():
    bank = Adapters(2, 8, 64, 40, device="cpu")
    bank.load(0, torch.randn(8, 64), torch.randn(40, 8))
    down, up = bank.down[0].clone(), bank.up[0].clone()
    bank.load(0, bank.down[0, 2:5], bank.up[0, :, 2:5], 3.0)
    assert torch.equal(bank.down[0, :3], down[2:5]) and torch.equal(bank.up[0, :, :3], up[:, 2:5])
    assert not bank.down[0, 3:].any() and not bank.up[0, :, 3:].any() and bank.scale[0] == 3.0


def test_adapters_beside_other_linears_are_refused():
    with pytest.raises(ValueError, match="lm_head"):
        attach_adapters(torch.nn.Module(), 2, 8, names=("q_proj", "lm_head"))


@pytest.mark.parametrize("y,out,message", [
    ((4096, 12288), (12288, 8192), "the output of linear 0 is linear 1's y or output"),
    ((4096, 12288), (8192, 4096), "the output of linear 1 is linear 0's y"),
    ((4096, 12288), (8192, 8192), "the output of linear 0 is linear 1's y or output"),
    ((8192, 12288), (4096, 16384), "the output of linear 0 is x"),
])
def test_adapters_c_refuse_outputs_that_are_read(y, out, message):
    L = _lib.lib()
    jobs = (_lib.AdapterJob * 2)(*[_lib.AdapterJob(down=4096, up=4096, scale=4096, down_adapter=512, down_row=64, up_adapter=320,
                                                   up_row=8, rank=8, m=40, y=a, ldy=40, out=b, ldo=40) for a, b in zip(y, out)])
    assert L.qs_adapters_add(P, 2, 64, 3, 64, P, 2, 2, jobs, P, 1 << 20, None) == 1
    assert message in L.qs_last_error().decode()


def adapters_c(L, **over):
    a = dict(x=P, dtype=2, ldx=64, tokens=3, n=64, which=P, adapters=2, count=1, ws=P, bytes=1 << 20, stream=None)
    j = dict(down=4096, up=4096, scale=4096, down_adapter=512, down_row=64, up_adapter=320, up_row=8, rank=8, m=40,
             y=4096, ldy=40, out=8192, ldo=40)
    for k, v in over.items():
        (j if k in j else a)[k] = v
    jobs = (_lib.AdapterJob * 4)(*[_lib.AdapterJob(**j)] * 4)
    return L.qs_adapters_add(a["x"], a["dtype"], a["ldx"], a["tokens"], a["n"], a["which"], a["adapters"], a["count"], jobs,
                             a["ws"], a["bytes"], a["stream"])


@pytest.mark.parametrize("over,code,message", [
    (dict(x=None), 1, "null"), (dict(which=None), 1, "null"), (dict(dtype=0), 1, "dtype 0"), (dict(count=5), 1, "5 linears"),
    (dict(count=0), 1, "0 linears"), (dict(n=60), 1, "rows of 60"), (dict(ldx=56), 1, "56 apart"), (dict(ldx=68), 1, "68 apart"),
    (dict(adapters=0), 1, "0 adapters"), (dict(x=ctypes.c_void_p(4104)), 1, "16-byte aligned"),
    (dict(tokens=(1 << 19) + 1), 3, "524289 rows"), (dict(ldx=(1 << 24) + 8), 3, "16777224 apart"), (dict(down_row=(1 << 24) + 8), 3, "rows 16777224 and 8 apart"), (dict(down=None), 1, "linear 0: null"), (dict(scale=None), 1, "linear 0: null"),
    (dict(rank=12), 1, "rank 12"), (dict(rank=136), 1, "rank 136"), (dict(rank=0), 1, "rank 0"), (dict(m=0), 1, "0 outputs"),
    (dict(ldy=39), 1, "39 and 40 apart"), (dict(ldo=39), 1, "40 and 39 apart"), (dict(down_row=56), 1, "rows 56"),
    (dict(up_row=12), 1, "and 12 apart"), (dict(down=4104), 1, "weights must be"), (dict(y=4097), 1, "aligned to their"),
    (dict(out=4096, ldo=48), 1, "share memory"), (dict(ws=None), 1, "workspace"), (dict(bytes=16), 1, "workspace of 16"),
])
def test_adapters_c_refusals(over, code, message):
    L = _lib.lib()
    assert adapters_c(L, **over) == code and message in L.qs_last_error().decode()


def test_adapters_workspace():
    L = _lib.lib()
    need = lambda *a: L.qs_adapters_workspace_bytes(*a[:4], _lib.int_array(a[4]))  # noqa: E731
    assert need(0, 64, 2, 1, [8]) == need(3, 64, 2, 1, [0]) == need(3, 64, 2, 1, [129]) == need(3, 64, 2, 5, [8] * 5) == 0
    assert need(3, 64, 2, 1, [8]) == 3 * 8 * 4 and need(3, 64, 2, 2, [8, 24]) == 3 * 32 * 4
    assert adapters_c(L, tokens=0, x=None) == 0


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

def rotated(**over):
    a = dict(q=torch.zeros(2, 4, 64, dtype=BF), k=torch.zeros(2, 2, 64, dtype=BF), v=torch.zeros(2, 2, 64, dtype=BF),
             k_pages=torch.zeros(3, 2, 16, 64, dtype=BF), v_pages=torch.zeros(3, 2, 16, 64, dtype=BF),
             table=torch.zeros(2, 3, dtype=I32), lengths=torch.zeros(2, dtype=I32),
             frequencies=torch.ones(32, dtype=torch.float64))
    a.update(over)
    return a


@pytest.mark.parametrize("over,error,message", [
    (dict(q=torch.zeros(2, 4, 32, dtype=BF)), ValueError, "q must be"),
    (dict(q=torch.zeros(3, 4, 64, dtype=BF)), ValueError, "q must be"),
    (dict(q=torch.zeros(2, 4, 64, dtype=HF)), TypeError, "q is"),
    (dict(k=torch.zeros(3, 2, 64, dtype=BF)), ValueError, "k must be"),
    (dict(v=torch.zeros(2, 3, 64, dtype=BF)), ValueError, "2 and 3 heads"),
    (dict(q=torch.zeros(2, 4, 128, dtype=BF)[:, :, ::2]), ValueError, "stride 1"),
    (dict(k_pages=torch.zeros(3, 2, 16, 64), v_pages=torch.zeros(3, 2, 16, 64)), TypeError, "cache dtype"),
    (dict(table=torch.zeros(2, 3)), ValueError, "table must be"),
    (dict(lengths=torch.zeros(3, dtype=I32)), ValueError, "lengths must be"),
    (dict(starts=torch.zeros(2, dtype=I32)), ValueError, "starts must be"),
    (dict(over=torch.zeros(3, dtype=I32)), ValueError, "over must be"),
    (dict(frequencies=torch.ones(32)), ValueError, "float64"),
    (dict(frequencies=torch.ones(4, 8, dtype=torch.float64)), ValueError, "float64"),
    (dict(frequencies=torch.ones(33, dtype=torch.float64)), ValueError, "33 pairs"),
    (dict(frequencies=torch.ones(0, dtype=torch.float64)), ValueError, "0 pairs"),
    (dict(frequencies=torch.ones(32, dtype=torch.float64, device="meta")), ValueError, "frequencies is on"),
    (dict(layout="pairs"), ValueError, "layout"),
    (dict(out=torch.zeros(2, 4, 64)), ValueError, "out must be"),
    (dict(out=torch.zeros(2, 8, 64, dtype=BF)[:, ::2]), ValueError, "lie together"),
    (dict(), RuntimeError, "runs on the GPU"),
])
def test_rotation_refuses(over, error, message):
    with pytest.raises(error, match=message):
        append_rotated(**rotated(**over))


def rotated_c(L, **over):
    pool = dict(k=4096, v=4096, k_page=2048, k_head=1024, k_pos=64, v_page=2048, v_head=1024, v_pos=64, pages=3, page=16,
                table=4096, table_ld=3, cols=3, lengths=4096)
    a = dict(q=P, k_new=P, v_new=P, dtype=2, tokens=2, rows=2, heads=4, kv_heads=2, dim=64, q_token=256, q_head=64,
             k_token=128, v_token=128, starts=None, over=None, frequencies=P, pairs=32, interleaved=0, factor=1.0, out=P,
             out_token=256)
    for key, v in over.items():
        (pool if key in pool else a)[key] = v
    return L.qs_page_append_rotated(a["q"], a["k_new"], a["v_new"], a["dtype"], a["tokens"], a["rows"], a["heads"],
                                    a["kv_heads"], a["dim"], a["q_token"], a["q_head"], a["k_token"], 64, a["v_token"], 64,
                                    a["starts"], _lib.PagePool(**pool), a["over"], a["frequencies"], a["pairs"],
                                    a["interleaved"], a["factor"], a["out"], a["out_token"], None)


@pytest.mark.parametrize("over,code,message", [
    (dict(q=None), 1, "null"), (dict(frequencies=None), 1, "null"), (dict(lengths=None), 1, "null"), (dict(dtype=0), 1, "dtype 0"),
    (dict(tokens=3), 1, "3 tokens of 2 rows"), (dict(heads=0), 1, "0 and 2 heads"), (dict(dim=60), 1, "heads of 60"),
    (dict(pairs=33), 1, "33 pairs"), (dict(pairs=0), 1, "0 pairs"), (dict(dim=1024, pairs=257, q_token=4096, out_token=4096), 1, "257 pairs"),
    (dict(pages=0), 1, "0 pages"), (dict(table_ld=2), 1, "table of 3"), (dict(cols=1 << 28, table_ld=1 << 28), 1, "table of"),
    (dict(q_token=252), 1, "252"), (dict(k_pos=68), 1, "68"), (dict(out_token=192), 1, "192 apart"),
    (dict(q=ctypes.c_void_p(4104)), 1, "16-byte"), (dict(v=4104), 1, "16-byte"), (dict(frequencies=ctypes.c_void_p(4100)), 1, "8-byte"),
    (dict(heads=60000, dim=512, q_token=60000 * 512, out_token=60000 * 512), 3, "60004 heads of 512"),
])
def test_rotation_c_refusals(over, code, message):
    L = _lib.lib()
    assert rotated_c(L, **over) == code and message in L.qs_last_error().decode()


def test_no_tokens_do_nothing():
    assert rotated_c(_lib.lib(), tokens=0, q=None) == 0 and rotated_c(_lib.lib(), rows=0, q=None) == 0


@pytest.mark.parametrize("kind,scaling", [
    ("default", {}), ("linear", dict(factor=4.0)),
    ("llama3", dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)),
    ("yarn", dict(factor=4.0, original_max_position_embeddings=32768)),
    ("yarn", dict(factor=16.0, original_max_position_embeddings=4096, beta_fast=16, beta_slow=2, attention_factor=1.25)),
    ("yarn", dict(factor=40.0, original_max_position_embeddings=4096, mscale=1.0, mscale_all_dim=0.5)),
    ("yarn", dict(factor=40.0, original_max_position_embeddings=4096, truncate=False)),
])
@pytest.mark.parametrize("dim,base", [(128, 500000.0), (64, 10000.0)])
def test_frequencies_are_transformers(kind, scaling, dim, base):
    """Against transformers' own, which are in 32 bits: 2^-20 of each, and where two are blended the ramp between them,
    which is off by a difference's, a quotient's and a difference's rounding, 3 2^-24 of up to 1, against a blend of 1 /
    factor at least: factor 2^-22."""
    from transformers import LlamaConfig
    from transformers.models.llama.modeling_llama import LlamaRotaryEmbedding
    cfg = LlamaConfig(hidden_size=dim * 2, num_attention_heads=2, head_dim=dim, max_position_embeddings=131072,
                      rope_parameters=dict(rope_type=kind, rope_theta=base, **scaling))
    want = LlamaRotaryEmbedding(cfg)
    w, factor = rope_frequencies(dim, base, dict(rope_type=kind, **scaling), "cpu")
    blend = scaling["factor"] * 2.0 ** -22 if kind in ("llama3", "yarn") else 0.0
    assert w.dtype == torch.float64 and torch.allclose(w.float(), want.inv_freq.float(), rtol=2.0 ** -20 + blend, atol=0)
    assert math.isclose(factor, want.attention_scaling, rel_tol=1e-6)


def test_frequencies_of_a_raised_base():
    """The slowest pair turns factor times slower, the fastest as before."""
    w, _ = rope_frequencies(128, 10000.0, None, "cpu")
    n, factor = rope_frequencies(128, 10000.0, dict(type="ntk", factor=4.0), "cpu")
    assert factor == 1.0 and n[0] == w[0] == 1 and math.isclose(w[-1] / n[-1], 4.0, rel_tol=1e-12)


def test_frequencies_refuse():
    for dim in (0, 7):
        with pytest.raises(ValueError, match="even number"):
            rope_frequencies(dim, device="cpu")
    with pytest.raises(NotImplementedError, match="longrope"):
        rope_frequencies(64, scaling=dict(rope_type="longrope"), device="cpu")
    for scaling in (dict(rope_type="linear"), dict(rope_type="yarn", factor=4.0), dict(rope_type="linear", factor=0.0),
                    dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192, low_freq_factor=1.0)):
        with pytest.raises(ValueError, match="scaling takes"):
            rope_frequencies(64, scaling=scaling, device="cpu")
    with pytest.raises(ValueError, match="must be the lower"):
        rope_frequencies(64, scaling=dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192,
                                          low_freq_factor=4.0, high_freq_factor=4.0), device="cpu")
    for base in (0.0, 1.0):
        with pytest.raises(ValueError, match="above 1"):
            rope_frequencies(64, base, device="cpu")
    assert rope_frequencies(64, scaling=dict(rope_type="default", factor=None), device="cpu")[1] == 1.0


def test_greedy_decode_refuses():
    from quipsharp_amd.decode import greedy_decode_paged
    for prompts, new in (([], 3), ([torch.zeros(2), torch.zeros(0)], 3), ([torch.zeros(2)], 0)):
        with pytest.raises(ValueError, match="every prompt has a token"):
            greedy_decode_paged(None, prompts, new)


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("args,error,message", [
    ((torch.zeros(2, 3, 4), torch.zeros(2, dtype=I32)), ValueError, "logits must be"),
    ((torch.zeros(2, 4, dtype=torch.float64), torch.zeros(2, dtype=I32)), TypeError, "unsupported dtype"),
    ((torch.zeros(2, 8)[:, ::2], torch.zeros(2, dtype=I32)), ValueError, "stride 1"),
    ((torch.zeros(1, 8).expand(3, 8), torch.zeros(3, dtype=I32)), ValueError, "overlap"),
    ((torch.zeros(2, 4), torch.zeros(2)), ValueError, "tokens must be"),
    ((torch.zeros(2, 4), torch.zeros(3, dtype=I32)), ValueError, "tokens must be"),
    ((torch.zeros(2, 4), torch.zeros(4, dtype=I32)[::2]), ValueError, "tokens must be"),
    ((torch.zeros(2, 4), torch.zeros(2, dtype=I32, device="meta")), ValueError, "tokens is on"),
    ((torch.zeros(2, 4), torch.zeros(2, dtype=I32), 5), ValueError, "5 alternatives"),
    ((torch.zeros(2, 400), torch.zeros(2, dtype=I32), 65), ValueError, "65 alternatives"),
    ((torch.zeros(2, 4), torch.zeros(2, dtype=I32), -1), ValueError, "-1 alternatives"),
    ((torch.zeros(2, 4), torch.zeros(2, dtype=I32)), RuntimeError, "runs on the GPU"),
])
def test_logprobs_refuse(args, error, message):
    with pytest.raises(error, match=message):
        token_logprobs(*args)


def scores_c(L, **over):
    a = dict(logits=P, dtype=0, ld=50, rows=2, vocab=50, tokens=P, token_bytes=8, top=5, logp=P, entropy=P, ranks=P, best=P,
             ids=P, ws=P, bytes=1 << 20)
    a.update(over)
    return L.qs_token_logprobs(*a.values(), None)


@pytest.mark.parametrize("over,code,message", [
    (dict(logits=None), 1, "null"), (dict(tokens=None), 1, "null"), (dict(best=None), 1, "null"), (dict(dtype=3), 1, "dtype 3"),
    (dict(token_bytes=2), 1, "2 bytes"), (dict(ld=49), 1, "49 apart"), (dict(top=51), 1, "51 alternatives"),
    (dict(top=-1), 1, "-1 alternatives"), (dict(vocab=0, ld=0), 1, "of 0 tokens"), (dict(top=65, vocab=100, ld=100), 3, "at most 64"),
    (dict(vocab=(1 << 24) + 1, ld=1 << 25), 3, "2^24"), (dict(logits=ctypes.c_void_p(4098)), 1, "aligned"),
    (dict(tokens=ctypes.c_void_p(4100)), 1, "aligned"), (dict(vocab=50000, ld=50000, bytes=64), 1, "workspace of 64"),
    (dict(vocab=50000, ld=50000, ws=None), 1, "workspace"),
])
def test_logprobs_c_refusals(over, code, message):
    L = _lib.lib()
    assert scores_c(L, **over) == code and message in L.qs_last_error().decode()


def test_logprobs_workspace():
    L = _lib.lib()
    need = L.qs_token_logprobs_workspace_bytes
    assert need(0, 50, 0, 0) == need(1, 0, 0, 0) == need(1, 50, 0, 65) == need(1, 50, 0, 51) == 0
    assert need(5000, 50000, 0, 20) == 0  # a work-group for each row
    assert need(1, 151936, 2, 20) > need(1, 151936, 2, 0) > 0
    assert scores_c(L, rows=0, logits=None) == 0


# ---------------------------------------------------------------------------

def test_gradients_are_refused():
    """An input that requires a gradient is refused where one would be recorded, and taken where none is."""
    grad = lambda *shape, dtype=BF: torch.zeros(*shape, dtype=dtype, requires_grad=True)  # noqa: E731
    calls = [lambda: add_adapters(**beside(x=grad(3, 64))), lambda: add_adapters(**beside(ys=[grad(3, 40)])),
             lambda: add_adapters(**beside(downs=[grad(2, 8, 64)])), lambda: add_adapters(**beside(ups=[grad(2, 40, 8)])),
             lambda: add_adapters(**beside(scales=[grad(2, dtype=torch.float32)])),
             lambda: append_rotated(**rotated(q=grad(2, 4, 64))), lambda: append_rotated(**rotated(k=grad(2, 2, 64))),
             lambda: append_rotated(**rotated(v=grad(2, 2, 64))), lambda: append_rotated(**rotated(v_pages=grad(3, 2, 16, 64))),
             lambda: token_logprobs(grad(2, 50, dtype=torch.float32), torch.zeros(2, dtype=I32))]
    for call in calls:
        with pytest.raises(RuntimeError, match="has no gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="runs on the GPU"):
            call()
