# SPDX-License-Identifier: Apache-2.0
"""The two caches of ``generate`` where they can go wrong: layers that share keys and values, sliding windows on the
dense cache."""

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
