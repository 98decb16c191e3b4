# SPDX-License-Identifier: Apache-2.0
"""Generation over the paged cache: the same tokens and states as the dense cache, conversations, page accounting, and the
operators run together step by step."""

import paged_oracle as po
import pytest
import torch

from arctictraining_b200.models import CausalLM
from arctictraining_b200.models import PagedKVCache
from arctictraining_b200.models import load_arch_config
from arctictraining_b200.models.generation import generate


def _model(name, dtype=torch.float32, device="cpu", **overrides):
    cfg = load_arch_config(name, overrides)
    if name == "tiny-deepseek-v2":
        from arctictraining_b200.models.deepseek import DeepseekV2ForCausalLM as cls
    else:
        cls = CausalLM
    m = cls(cfg, dtype=dtype, device=device)
    m.init_weights(seed=3)
    return m.eval()


def _prompt(model, batch, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(8, model.config["vocab_size"], (batch, n), generator=g).to(next(model.parameters()).device)


@pytest.mark.parametrize("length", [5, 23])  # on the paged kernels from the start, and through the read-back
@pytest.mark.parametrize("name", ["tiny-llama", "tiny-qwen3", "tiny-deepseek-v2"])
def test_same_tokens_as_the_dense_cache(name, length):
    m = _model(name)
    ids = _prompt(m, 3, length)
    want, want_h = generate(m, ids, 9, do_sample=False)
    cache = PagedKVCache.for_model(m.config, 3, length + 9, page=8, dtype=torch.float32)
    got, got_h = generate(m, ids, 9, do_sample=False, cache=cache)
    assert torch.equal(got, want) and cache.lengths == [length + 8] * 3
    torch.testing.assert_close(got_h, want_h, atol=2e-5, rtol=1e-4)


@pytest.mark.parametrize("second", [1, 4, 140])
@pytest.mark.parametrize("name", ["tiny-llama", "tiny-deepseek-v2"])
def test_a_conversation_continues_in_the_cache(name, second):
    """A second prompt behind the first answer: the states are those of a plain forward over the whole text."""
    m = _model(name)
    cache = PagedKVCache.for_model(m.config, 2, 200, page=16, dtype=torch.float32)
    first, _ = generate(m, _prompt(m, 2, 20), 6, do_sample=False, cache=cache)
    more = torch.cat([first[:, -1:], _prompt(m, 2, second, seed=5)], dim=1)
    answer, hidden = generate(m, more, 4, do_sample=False, cache=cache)
    text = torch.cat([first[:, :-1], answer], dim=1)
    with torch.no_grad():
        full = m(input_ids=text[:, :-1], hidden_only=True).hidden_states
    torch.testing.assert_close(hidden, full[:, first.shape[1] - 1 :], atol=2e-5, rtol=1e-4)


def test_sliding_window_layers():
    m = _model("tiny-llama", sliding_window=6, use_sliding_window=True)
    cache = PagedKVCache.for_model(m.config, 2, 40, page=4, dtype=torch.float32)
    ids, hidden = generate(m, _prompt(m, 2, 19), 5, do_sample=False, cache=cache)
    with torch.no_grad():
        full = m(input_ids=ids[:, :-1], hidden_only=True).hidden_states
    torch.testing.assert_close(hidden, full, atol=2e-5, rtol=1e-4)


def test_8_bit_cache_stays_near_the_plain_one():
    """e4m3 rows are off by 2^-4 of an element at most, typically 2^-6: states of a two-layer model with weights of 0.02 move
    by much less than that."""
    m = _model("tiny-llama")
    ids = _prompt(m, 2, 30)
    _, want = generate(m, ids, 1, do_sample=False)
    _, got = generate(m, ids, 1, do_sample=False, cache=PagedKVCache.for_model(m.config, 2, 32, e4m3=True, dtype=torch.float32))
    off = float((got - want).norm() / want.norm())
    assert 0 < off < 2.0**-4


def test_pages_are_handed_out_and_given_back():
    c = PagedKVCache(1, 2, 16, batch=3, max_length=40, page=8, num_pages=9, dtype=torch.float32)
    c.reserve(17)
    ids = sorted(p for row in c.page_table.tolist() for p in row if p >= 0)
    assert ids == list(range(9))
    c.advance(17)
    c.reserve(7)  # up to 24 positions: no new page
    with pytest.raises(RuntimeError):
        c.reserve(8)
    with pytest.raises(ValueError):
        c.reserve(24)
    before = c.page_table.clone()
    c.release(1)
    assert c.lengths == [17, 0, 17] and c.starts.tolist() == [17, 0, 17]
    assert c.page_table[1].tolist() == [-1] * 5 and torch.equal(c.page_table[0], before[0])
    c.reserve(8)  # one more page for each of the others and one for the empty sequence: the three that came back
    with pytest.raises(RuntimeError):
        c.reserve(16)
    with pytest.raises(ValueError):
        PagedKVCache(1, 2, 16, batch=0, max_length=40)
    with pytest.raises(ValueError):
        PagedKVCache(1, 2, 16, batch=1, max_length=40, latent=True)


def test_generate_refuses_a_cache_of_another_batch_or_too_short():
    m = _model("tiny-llama")
    with pytest.raises(ValueError):
        generate(m, _prompt(m, 2, 4), 3, cache=PagedKVCache.for_model(m.config, 3, 40, dtype=torch.float32))
    with pytest.raises(ValueError):
        generate(m, _prompt(m, 2, 4), 9, cache=PagedKVCache.for_model(m.config, 2, 8, dtype=torch.float32))


@pytest.mark.parametrize("kind", ["paged", "paged_e4m3"])
def test_speculator_trainer_generates_with_it(tiny_recipe, tmp_path, kind):
    from test_speculator_cpu import _spec_trainer

    tr = _spec_trainer(tiny_recipe, tmp_path, exit_iteration=1, gen_kv_cache=kind)
    prompts = torch.randint(8, 1000, (3, 9), generator=torch.Generator().manual_seed(0))
    got, hidden = tr.generate(prompts, 7, do_sample=False)
    assert got.shape == (3, 16) and hidden.shape[:2] == (3, 15)
    if kind == "paged":
        assert torch.equal(got, tr.generate_continuations(prompts, 7))


def _steps(device, dtype, e4m3, latent):
    """Prompt and single tokens through append and attention as a model does it; every step against the oracle on what the
    cache then holds."""
    B, hq, hkv, D, page = 3, 8, 1 if latent else 2, 96 if latent else 64, 16
    R = 64
    g = torch.Generator().manual_seed(1)

    def normal(*shape):
        return torch.randn(*shape, generator=g).to(dtype).to(device)

    cache = PagedKVCache(1, hkv, D, B, 64, page=page, e4m3=e4m3, latent=latent, dtype=dtype, device=device)
    w = normal(R)
    for S in (13, 1, 1, 4, 1):
        cache.reserve(S)
        rot = D - R if latent else D
        ang = cache.positions(S).unsqueeze(-1).float() * torch.logspace(0, -3, rot // 2, device=device)
        cos, sin = ang.cos(), ang.sin()
        su = po.Setup.__new__(po.Setup)
        su.B, su.S, su.Hkv, su.D, su.page, su.dtype, su.e4m3, su.P = B, S, hkv, D, page, dtype, e4m3, cache.num_pages
        su.table_list, su.starts_list, su.counts_list = cache.page_table.tolist(), list(cache.lengths), [S] * B
        su.k_pages, su.k_scale, su.v_pages, su.v_scale = cache.k_pages[0], cache.k_scale[0], cache.v_pages[0], cache.v_scale[0]
        p_type = torch.float32 if dtype == torch.float32 else torch.float16 if e4m3 else dtype
        if latent:
            q_pe = cache.append_latent(0, normal(B, S, hq, rot), normal(B, S, D), w, 1e-6, cos, sin)
            q = normal(B, S, hq, R)
            got = cache.attend_latent(0, q, q_pe, 0.1)
            want, tol = po.attention(su, torch.cat([q, q_pe], -1), 0.1, latent=R, p_type=p_type)
        else:
            q = cache.append(0, normal(B, S, hq, D), normal(B, S, hkv, D), normal(B, S, hkv, D), cos, sin)
            got = cache.attend(0, q)
            want, tol = po.attention(su, q, D**-0.5, p_type=p_type)
        po.check_attention(got, want, tol, f"{S} tokens at {cache.lengths}")
        cache.advance(S)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("dtype,e4m3", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True)], ids=str)
def test_steps(dtype, e4m3, latent):
    _steps("cpu", dtype, e4m3, latent)


@pytest.mark.gpu
@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("dtype,e4m3", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, True)],
                         ids=str)
def test_steps_on_the_gpu(dtype, e4m3, latent):
    _steps("cuda", dtype, e4m3, latent)


@pytest.mark.gpu
@pytest.mark.parametrize("name,length", [("tiny-llama", 9), ("tiny-llama", 40), ("tiny-deepseek-v2", 9), ("tiny-deepseek-v2", 40)])
def test_generation_on_the_gpu(name, length):
    """bf16 states of a generation are those of a plain forward over its tokens: two or three layers of about ten roundings of
    2^-9 each, whose errors add up to at most 3 * 10 * 2^-9 = 6 %."""
    from arctictraining_b200.ops import LAUNCH_COUNTER

    sizes = dict(hidden_size=256, head_dim=64) if name == "tiny-llama" else dict(kv_lora_rank=64, qk_rope_head_dim=32, qk_nope_head_dim=32,
                                                                                 v_head_dim=32, head_dim=32)
    m = _model(name, torch.bfloat16, "cuda", **sizes)
    cache = PagedKVCache.for_model(m.config, 2, 80, dtype=torch.bfloat16, device="cuda")
    before = LAUNCH_COUNTER["native"]
    ids, hidden = generate(m, _prompt(m, 2, length), 12, do_sample=False, cache=cache)
    assert LAUNCH_COUNTER["native"] - before >= 12 * 2 * m.config["num_hidden_layers"]
    with torch.no_grad():
        full = m(input_ids=ids[:, :-1], hidden_only=True).hidden_states
    assert float((hidden.float() - full.float()).norm() / full.float().norm()) < 0.06
