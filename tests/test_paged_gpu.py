# SPDX-License-Identifier: Apache-2.0
"""The paged-cache kernels against the 64-bit oracle: types, head layouts, lengths, page sizes, masks, strides, streams and
captured graphs."""

import paged_cases as pc
import paged_oracle as po
import pytest
import torch

from arctictraining_b200 import ops

pytestmark = pytest.mark.gpu
TYPES = [(pc.BF, False), (pc.HF, False), (pc.BF, True), (pc.HF, True), (pc.F32, False)]


@pytest.mark.parametrize("name", list(pc.refusals("cpu", pc.F32)))
def test_refusals(name):
    with pytest.raises(ValueError):
        pc.refusals("cuda", pc.BF)[name]()


def test_refusal_of_mixed_devices():
    c = pc.ATTENTION["one-token-cache"]
    su, cpu = pc.set_up(c, pc.BF, False, "cuda"), pc.set_up(c, pc.BF, False, "cpu")
    q = su.normal(1, 1, 4, 64)
    for args in ((q, cpu.k_pages, cpu.v_pages, su.table, su.starts), (q, su.k_pages, su.v_pages, cpu.table, su.starts),
                 (q, su.k_pages, su.v_pages, su.table, cpu.starts), (q.cpu(), su.k_pages, su.v_pages, su.table, su.starts)):
        with pytest.raises(ValueError):
            ops.paged_attention(*args)


@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
@pytest.mark.parametrize("name", ["one-token-cache", "one-sequence", "ragged", "counts", "missing-pages", "negative-start", "page-of-one",
                                  "chunk", "wide-head", "narrow-head", "head-of-80", "many-heads"])
def test_append(name, dtype, e4m3):
    pc.append_case(pc.ATTENTION[name], dtype, e4m3, "cuda")


@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
@pytest.mark.parametrize("name", list(pc.LATENT))
def test_latent_append(name, dtype, e4m3):
    pc.latent_append_case(pc.LATENT[name], dtype, e4m3, "cuda")


@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
@pytest.mark.parametrize("name", ["one-token-cache", "ragged", "counts", "missing-pages", "group-of-five-odd-page", "page-of-one",
                                  "wide-head", "narrow-head", "head-of-80"])
def test_read(name, dtype, e4m3):
    pc.read_case(pc.ATTENTION[name], dtype, e4m3, "cuda", values=name != "ragged")


@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
@pytest.mark.parametrize("name", list(pc.ATTENTION))
def test_attention(name, dtype, e4m3):
    pc.attention_case(pc.ATTENTION[name], dtype, e4m3, "cuda")


@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
@pytest.mark.parametrize("name", list(pc.LATENT))
def test_latent_attention(name, dtype, e4m3):
    pc.latent_case(pc.LATENT[name], dtype, e4m3, "cuda")


@pytest.mark.parametrize("shape", [(0, 1, 4, 2), (2, 0, 4, 2), (2, 1, 0, 2)])
def test_empty_calls(shape):
    B, S, hq, hkv = shape
    pages = torch.zeros(3, hkv, 16, 32, device="cuda", dtype=pc.BF)
    table, starts = torch.zeros(B, 2, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    q = torch.zeros(B, S, hq, 32, device="cuda", dtype=pc.BF)
    assert ops.paged_attention(q, pages, pages, table, starts).shape == q.shape
    kv, cos = torch.zeros(B, S, hkv, 32, device="cuda", dtype=pc.BF), torch.zeros(B, S, 16, device="cuda")
    assert ops.paged_kv_append(q, kv, kv, cos, cos, pages, pages.clone(), table, starts).shape == q.shape
    assert ops.paged_kv_read(pages, None, table, starts, 0)[0].shape == (B, 0, hkv, 32)


def test_no_pages():
    pages, table = torch.zeros(0, 2, 16, 32, device="cuda", dtype=pc.BF), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    starts, q = torch.tensor([4, 9], dtype=torch.int32, device="cuda"), torch.ones(2, 1, 4, 32, device="cuda", dtype=pc.BF)
    assert torch.equal(ops.paged_attention(q, pages, pages, table, starts), torch.zeros_like(q))
    full = torch.ones(2, 2, 16, 32, device="cuda", dtype=pc.BF)
    assert torch.equal(ops.paged_attention(q, full, full, table[:, :0], starts), torch.zeros_like(q))
    assert torch.equal(ops.paged_kv_read(pages, None, table, starts, 5)[0], torch.zeros(2, 5, 2, 32, device="cuda", dtype=pc.BF))
