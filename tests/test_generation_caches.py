# SPDX-License-Identifier: Apache-2.0
"""The two caches of ``generate`` where they can go wrong: layers that share keys and values, sliding windows on the
dense cache, positions that nobody reserved, and a device wait that ran out."""

import sys
from pathlib import Path

import pytest
import torch
from test_paged_generation import _model
from test_paged_generation import _prompt

from arctictraining_b200.models import PagedKVCache
from arctictraining_b200.models import load_arch_config
from arctictraining_b200.models.generation import generate

SWIFTKV = Path(__file__).resolve().parent.parent / "projects" / "swiftkv" / "train.py"


def _swiftkv_model(name, **overrides):
    from arctictraining_b200.config.trainer import load_user_module_from_path
    from arctictraining_b200.registry import get_registered_trainer

    load_user_module_from_path(SWIFTKV)
    project = sys.modules[get_registered_trainer("swiftkv").__module__]
    cls = project.MLASwiftKVForCausalLM if name == "tiny-deepseek-v2" else project.SwiftKVForCausalLM
    m = cls(load_arch_config(name, {"num_hidden_layers": 3, "num_key_value_layers": 1, "key_value_group_size": 1, **overrides}),
            dtype=torch.float32)
    g = torch.Generator().manual_seed(3)
    for p_name, p in m.named_parameters():
        with torch.no_grad():
            p.copy_(torch.ones_like(p) if "norm" in p_name else torch.randn(p.shape, generator=g) * 0.05)
    m.swiftkv(True)
    return m.eval()


def _same_as_a_plain_forward(m, ids, hidden):
    with torch.no_grad():
        full = m(input_ids=ids[:, :-1], hidden_only=True).hidden_states
    torch.testing.assert_close(hidden, full, atol=2e-5, rtol=1e-4)


@pytest.mark.parametrize("name", ["tiny-llama", "tiny-deepseek-v2"])
def test_layers_that_share_keys_and_values_on_the_dense_cache(name):
    """The states of every fed position are those of a plain forward over the same tokens."""
    m = _swiftkv_model(name)
    _same_as_a_plain_forward(m, *generate(m, _prompt(m, 2, 7), 6, do_sample=False))


@pytest.mark.parametrize("name", ["tiny-llama", "tiny-deepseek-v2"])
def test_layers_that_share_keys_and_values_refuse_the_paged_cache(name):
    m = _swiftkv_model(name)
    with pytest.raises(NotImplementedError):
        generate(m, _prompt(m, 2, 7), 6, do_sample=False, cache=PagedKVCache.for_model(m.config, 2, 20, dtype=torch.float32))


@pytest.mark.parametrize("length", [1, 4, 19])
def test_sliding_window_layers_on_the_dense_cache(length):
    m = _model("tiny-llama", sliding_window=6, use_sliding_window=True)
    want, _ = generate(m, _prompt(m, 2, length), 12, do_sample=False,
                       cache=PagedKVCache.for_model(m.config, 2, 40, page=4, dtype=torch.float32))
    ids, hidden = generate(m, _prompt(m, 2, length), 12, do_sample=False)
    _same_as_a_plain_forward(m, ids, hidden)
    assert torch.equal(ids, want)


def test_sliding_window_layers_that_share_keys_and_values():
    m = _swiftkv_model("tiny-llama", sliding_window=6, use_sliding_window=True)
    _same_as_a_plain_forward(m, *generate(m, _prompt(m, 2, 7), 6, do_sample=False))


def _layer_inputs(c, S):
    return [torch.zeros(c.batch, S, 2, 16)] * 3 + [torch.ones(c.batch, S, 8), torch.zeros(c.batch, S, 8)]


def test_positions_that_nobody_reserved_are_refused():
    c = PagedKVCache(1, 2, 16, batch=2, max_length=40, page=8, dtype=torch.float32)
    latent = PagedKVCache(1, 1, 48, batch=2, max_length=40, page=8, latent=True, dtype=torch.float32)
    with pytest.raises(ValueError):
        c.append(0, *_layer_inputs(c, 1))
    with pytest.raises(ValueError):
        latent.append_latent(0, torch.zeros(2, 1, 2, 16), torch.zeros(2, 1, 48), torch.ones(32), 1e-6, torch.ones(2, 1, 8), torch.zeros(2, 1, 8))
    with pytest.raises(ValueError):
        c.advance(1)
    assert c.lengths == [0, 0]
    c.reserve(3)  # a page of eight each
    c.append(0, *_layer_inputs(c, 8))
    with pytest.raises(ValueError):
        c.append(0, *_layer_inputs(c, 9))
    with pytest.raises(ValueError):
        c.advance(30)
    c.advance(8)
    assert c.lengths == [8, 8] and c.starts.tolist() == [8, 8]
    with pytest.raises(ValueError):
        c.append(0, *_layer_inputs(c, 1))
    c.reserve(1)
    c.append(0, *_layer_inputs(c, 1))
    c.release(1)  # its next position has no page, as on a fresh cache
    with pytest.raises(ValueError):
        c.append(0, *_layer_inputs(c, 1))
    c.reserve(1)
    c.append(0, *_layer_inputs(c, 1))
    c.advance(1)
    assert c.lengths == [9, 1]


def test_no_position_beyond_the_largest_length():
    c = PagedKVCache(1, 2, 16, batch=2, max_length=21, page=8, dtype=torch.float32)  # three pages each hold 24
    c.reserve(21)
    with pytest.raises(ValueError):
        c.append(0, *_layer_inputs(c, 22))
    c.append(0, *_layer_inputs(c, 21))
    c.advance(21)
    with pytest.raises(ValueError):
        c.advance(1)


@pytest.mark.parametrize("cached", [True, False])
def test_a_device_wait_that_ran_out_is_raised_at_the_end(monkeypatch, cached):
    """The error words of the device, here the host's stand-in for them, are read once per generation."""
    from arctictraining_b200.comm import errors
    from arctictraining_b200.exceptions import KernelWaitError

    m = _model("tiny-llama")
    reads = []
    monkeypatch.setattr(errors, "read_error_words", lambda like: reads.append(like) or (0x3101, 0))
    cache = PagedKVCache.for_model(m.config, 2, 20, dtype=torch.float32) if cached else None
    if cached:
        with pytest.raises(KernelWaitError):
            generate(m, _prompt(m, 2, 4), 3, do_sample=False, cache=cache)
        assert len(reads) == 1
        monkeypatch.setattr(errors, "read_error_words", lambda like: (0, 0))
        cache.release(0)
        cache.release(1)
    assert generate(m, _prompt(m, 2, 4), 3, do_sample=False, cache=cache)[0].shape == (2, 7)
    assert len(reads) == int(cached)


def _gpu_model(name, **overrides):
    sizes = dict(hidden_size=256, head_dim=64) if name == "tiny-llama" else dict(kv_lora_rank=64, qk_rope_head_dim=32, qk_nope_head_dim=32,
                                                                                 v_head_dim=32, head_dim=32)
    return _model(name, torch.bfloat16, "cuda", **sizes, **overrides)


def _off(m, text, hidden, first=0):
    with torch.no_grad():
        full = m(input_ids=text[:, :-1], hidden_only=True).hidden_states[:, first:]
    return float((hidden.float() - full.float()).norm() / full.float().norm())


# Two or three layers of about ten bf16 roundings of 2^-9 each add up to 3 * 10 * 2^-9 = 6 % at most; an 8-bit row's elements are off by
# 2^-4 at most, and what attention makes of them by no more in models with weights of 0.02.
@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("second", [1, 4, 140])
@pytest.mark.parametrize("name,window", [("tiny-llama", None), ("tiny-llama", 6), ("tiny-deepseek-v2", None)])
def test_a_conversation_on_the_gpu(name, window, second, e4m3):
    """A prompt, its answer, a second prompt of one, few and many tokens, and a second answer, in one cache."""
    m = _gpu_model(name, **(dict(sliding_window=window, use_sliding_window=True) if window else {}))
    limit = 0.06 + (2.0**-4 if e4m3 else 0.0)
    cache = PagedKVCache.for_model(m.config, 2, 200, page=16, e4m3=e4m3, dtype=torch.bfloat16, device="cuda")
    first, hidden = generate(m, _prompt(m, 2, 20), 6, do_sample=False, cache=cache)
    assert _off(m, first, hidden) < limit
    more = torch.cat([first[:, -1:], _prompt(m, 2, second, seed=5)], dim=1)
    answer, hidden = generate(m, more, 4, do_sample=False, cache=cache)
    assert _off(m, torch.cat([first[:, :-1], answer], dim=1), hidden, first.shape[1] - 1) < limit
