# SPDX-License-Identifier: Apache-2.0
"""The paged-cache operators' reference implementations against the 64-bit oracle, and what they refuse."""

import paged_cases as pc
import pytest
import torch

from arctictraining_b200 import ops

TYPES = [(pc.F32, False), (pc.BF, False), (pc.F32, True), (pc.BF, True)]


@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
@pytest.mark.parametrize("name", [n for n in pc.ATTENTION if n != "long"])
def test_attention(name, dtype, e4m3):
    pc.attention_case(pc.ATTENTION[name], dtype, e4m3, "cpu")


@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
@pytest.mark.parametrize("name", ["one-token-cache", "ragged", "draft", "twenty-heads", "small-widths", "counts-missing"])
def test_latent_attention(name, dtype, e4m3):
    pc.latent_case(pc.LATENT[name], dtype, e4m3, "cpu")


@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
@pytest.mark.parametrize("name", ["one-token-cache", "ragged", "counts", "missing-pages", "negative-start", "page-of-one", "chunk"])
def test_append(name, dtype, e4m3):
    pc.append_case(pc.ATTENTION[name], dtype, e4m3, "cpu")


@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
@pytest.mark.parametrize("name", ["one-token-cache", "draft", "small-widths", "counts-missing"])
def test_latent_append(name, dtype, e4m3):
    pc.latent_append_case(pc.LATENT[name], dtype, e4m3, "cpu")


@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
@pytest.mark.parametrize("name", ["one-token-cache", "ragged", "missing-pages", "group-of-five-odd-page"])
def test_read(name, dtype, e4m3):
    pc.read_case(pc.ATTENTION[name], dtype, e4m3, "cpu", values=name != "ragged")


@pytest.mark.parametrize("window", [None, 2])
@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
def test_hidden_values_that_are_not_finite(dtype, e4m3, window):
    pc.not_finite_case(dtype, e4m3, "cpu", window=window)


@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
def test_hidden_latents_that_are_not_finite(dtype, e4m3):
    pc.not_finite_case(dtype, e4m3, "cpu", latent=True)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0])
def test_scales_of_any_sign(scale):
    pc.attention_case(pc.ATTENTION["draft-window"], pc.BF, False, "cpu", scale)
    pc.latent_case(pc.LATENT["draft"], pc.BF, True, "cpu", scale)


@pytest.mark.parametrize("dtype", [pc.F32, pc.BF], ids=str)
@pytest.mark.parametrize("name", list(pc.refusals("cpu", pc.F32)))
def test_refusals(name, dtype):
    with pytest.raises(ValueError):
        pc.refusals("cpu", dtype)[name]()


@pytest.mark.parametrize("shape", [(0, 1, 4, 2), (2, 0, 4, 2), (2, 1, 0, 2)])
def test_empty_calls(shape):
    B, S, hq, hkv = shape
    pages = torch.zeros(3, hkv, 16, 32)
    table, starts = torch.zeros(B, 2, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    q = torch.zeros(B, S, hq, 32)
    assert ops.paged_attention(q, pages, pages, table, starts).shape == q.shape
    kv, cos = torch.zeros(B, S, hkv, 32), torch.zeros(B, S, 16)
    assert ops.paged_kv_append(q, kv, kv, cos, cos, pages, pages.clone(), table, starts).shape == q.shape
    assert ops.paged_kv_read(pages, None, table, starts, 0)[0].shape == (B, 0, hkv, 32)


def test_no_pages():
    pages, table, starts = torch.zeros(0, 2, 16, 32), torch.zeros(2, 3, dtype=torch.int32), torch.tensor([4, 9], dtype=torch.int32)
    q = torch.ones(2, 1, 4, 32)
    assert torch.equal(ops.paged_attention(q, pages, pages, table, starts), torch.zeros_like(q))
    assert torch.equal(ops.paged_attention(q, torch.ones(2, 2, 16, 32), torch.ones(2, 2, 16, 32), table[:, :0], starts), torch.zeros_like(q))
    assert torch.equal(ops.paged_kv_read(pages, None, table, starts, 5)[0], torch.zeros(2, 5, 2, 32))


def test_rows_of_zeros_and_of_nan_in_an_8_bit_cache():
    """A row of zeros is read back as zeros; one with a NaN or an infinity as NaN; its neighbours are not touched."""
    pages, scale = torch.zeros(1, 1, 4, 16).to(torch.float8_e4m3fn), torch.zeros(1, 1, 4)
    x = torch.stack([torch.zeros(16), torch.full((16,), 3.0), torch.ones(16), torch.ones(16)]).view(1, 4, 1, 16)
    x[0, 2, 0, 5], x[0, 3, 0, 7] = float("nan"), float("inf")
    table, starts = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    one, zero = torch.ones(1, 4, 8), torch.zeros(1, 4, 8)
    ops.paged_kv_append(x, x, x, one, zero, pages, pages.clone(), table, starts, None, scale, scale.clone())
    got, _ = ops.paged_kv_read(pages, None, table, starts + 4, 4, scale, None, torch.float32)
    assert torch.equal(got[0, 0], torch.zeros(1, 16))
    torch.testing.assert_close(got[0, 1], torch.full((1, 16), 3.0), rtol=2.0**-22, atol=0)
    assert torch.isnan(got[0, 2]).all() and torch.isnan(got[0, 3]).all()
