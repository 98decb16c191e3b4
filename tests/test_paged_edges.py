# SPDX-License-Identifier: Apache-2.0
"""Edges of the paged-cache operators: the bytes of an append."""

import paged_cases as pc
import pytest
import torch

from arctictraining_b200 import ops

HALF = [(pc.BF, False), (pc.HF, False), (pc.BF, True), (pc.HF, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,e4m3", HALF, ids=str)
def test_append_writes_the_bytes_of_the_reference(dtype, e4m3):
    """Products and sums of the rotation are rounded one by one in both, and so is the quantisation: the same bytes."""
    c = dict(starts=[3, 60, 0, 131], S=70, hq=6, hkv=4, d=128, page=16, counts=[70, 1, 0, 64])
    one, two = (pc.set_up(c, dtype, e4m3, device) for device in ("cuda", "cpu"))
    q, k, v = (one.normal(4, 70, h, 128) for h in (6, 4, 4))
    cos, sin = one.angles(128)

    def call(su, *x):
        out = ops.paged_kv_append(*x, su.k_pages, su.v_pages, su.table, su.starts, su.counts, su.k_scale, su.v_scale)
        raw = [su.k_pages.view(torch.uint8), su.v_pages.view(torch.uint8)]
        return [out] + raw + ([su.k_scale.view(torch.int32), su.v_scale.view(torch.int32)] if e4m3 else [])

    for a, b in zip(call(one, q, k, v, cos, sin), call(two, *(t.cpu() for t in (q, k, v, cos, sin)))):
        assert torch.equal(a.cpu(), b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [pc.BF, pc.HF], ids=str)
def test_latent_append_rotates_like_the_reference(dtype):
    """The rotary part (of a plain cache) and the queries, bit for bit; the norm's sum has another order."""
    c = dict(starts=[3, 60], S=40, page=16)
    one, two = (pc.set_up(c, dtype, False, device, values=False, d=576, hkv=1) for device in ("cuda", "cpu"))
    q_pe, kv_a, w = one.normal(2, 40, 5, 64), one.normal(2, 40, 576), one.normal(512)
    cos, sin = one.angles(64)
    got = []
    for su, x in ((one, (q_pe, kv_a, w, 1e-6, cos, sin)), (two, (q_pe.cpu(), kv_a.cpu(), w.cpu(), 1e-6, cos.cpu(), sin.cpu()))):
        q = ops.paged_latent_append(*x, su.k_pages, su.table, su.starts)
        got.append((q.cpu(), su.k_pages[..., 512:].cpu().contiguous().view(torch.int16)))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
