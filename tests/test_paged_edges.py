# SPDX-License-Identifier: Apache-2.0
"""Edges of the paged-cache operators: the bytes of an append, scales of zero, scales of attention that
are no numbers, long windows, heads or positions of one with any stride, more
sequences than a block has threads."""

import paged_cases as pc
import paged_oracle as po
import pytest
import torch

from arctictraining_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
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


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads,latent", [(8, False), (16, True), (64, True), (128, True)])
@pytest.mark.parametrize("log2_score,byte,scale", [(-127, -64.0, 2.0**-6), (-200, -1.0, 1.0), (-100, -128.0, 2.0**12), (-126, -256.0, 2.0**-20),
                                                   (-1, -64.0, 2.0**-120)])
def test_keys_with_a_scale_of_zero(device, heads, latent, log2_score, byte, scale):
    """A row of zeros with a scale of zero (a position of a zero-filled cache) has score 0; the others are far below it.  Their
    weight is 2^log2_score each; weights below 2^-126 may be lost, others are off by the usual roundings."""
    D, n = (576 if latent else 64), 40
    hkv = 1 if latent else 2
    pages = torch.full((3, hkv, 16, D), byte, device=device).to(torch.float8_e4m3fn)
    scales = torch.full((3, hkv, 16), scale, device=device)
    pages.view(torch.uint8)[1, :, 5] = 0
    scales[1, :, 5] = 0.0
    table, starts = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=device), torch.tensor([n - 1], dtype=torch.int32, device=device)
    q = torch.ones(1, 1, heads, D, device=device, dtype=pc.BF)
    by = log2_score * 0.6931471805599453 / (D * byte * scale)  # the scores are D byte scale
    if latent:
        got = ops.paged_latent_attention(q[..., :512], q[..., 512:], pages, table, starts, None, scales, by)
    else:
        got = ops.paged_attention(q, pages, pages, table, starts, None, scales, scales, by)
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    weight = 2.0**log2_score
    want = (n - 1) * weight * byte * scale / (1 + (n - 1) * weight)
    # the exponent |log2_score| is a product of two fp32 roundings and a sum of D equal products (D roundings at most): it is off by
    # (D + 8) 2^-24 of itself at most, and the weight by 0.7 times that; its sums with a scale's logarithm and a maximum, all below
    # 256, add four roundings of 2^-17; probabilities are rounded to fp16, the result to bf16.
    slack = 0.7 * abs(log2_score) * (D + 8) * 2.0**-24 + 2.0**-15 + 2.0**-11 + 2.0**-8
    lost = (n - 1) * 2.0**-126 * abs(byte) * scale if log2_score < -125 else 0.0
    assert bool(((got - want).abs() <= abs(want) * slack + lost + 2.0**-126).all()), (got.min(), got.max(), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 1e39])
def test_a_scale_that_is_no_number_is_refused(device, scale):
    dtype = pc.BF
    su, lat = pc.set_up(pc.ATTENTION["draft"], dtype, False, device), pc.set_up(pc.LATENT["draft"], dtype, False, device, values=False, d=576)
    with pytest.raises(ValueError):
        ops.paged_attention(su.normal(3, 5, 8, 64), su.k_pages, su.v_pages, su.table, su.starts, scale=scale)
    with pytest.raises(ValueError):
        ops.paged_latent_attention(lat.normal(3, 3, 16, 512), lat.normal(3, 3, 16, 64), lat.k_pages, lat.table, lat.starts, scale=scale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("window", [2**31 - 1, 2**31, 10**15])
def test_a_window_longer_than_any_sequence(device, window):
    su = pc.set_up(pc.ATTENTION["draft"], pc.BF, False, device)
    q = su.normal(3, 5, 8, 64)
    args = (q, su.k_pages, su.v_pages, su.table, su.starts)
    assert torch.equal(ops.paged_attention(*args, window=window), ops.paged_attention(*args))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("e4m3", [False, True])
def test_dimensions_of_one_may_have_any_stride(device, e4m3):
    """One head, or pages of one position, as views of tensors whose dimensions have another order: the same rows."""
    for c in (dict(starts=[20, 70], S=2, hq=4, hkv=1, d=64, page=16), dict(starts=[20, 7], S=2, hq=4, hkv=3, d=64, page=1)):
        su = pc.set_up(c, pc.BF, e4m3, device)
        q = su.normal(2, 2, 3 * su.Hkv, 64)
        k, v = su.normal(2, 2, su.Hkv, 64), su.normal(2, 2, su.Hkv, 64)
        cos, sin = su.angles(64)

        def turned(t):
            return None if t is None else t.transpose(1, 2).clone(memory_format=torch.contiguous_format).transpose(1, 2)

        def calls(kp, vp, ks, vs):
            a = ops.paged_kv_append(q, k, v, cos, sin, kp, vp, su.table, su.starts, None, ks, vs)
            return [a, ops.paged_attention(q, kp, vp, su.table, su.starts, None, ks, vs),
                    *ops.paged_kv_read(kp, vp, su.table, su.starts, 30, ks, vs)]

        mine = [turned(t) for t in (su.k_pages, su.v_pages, su.k_scale, su.v_scale)]
        for a, b in zip(calls(*mine), calls(su.k_pages, su.v_pages, su.k_scale, su.v_scale)):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [None, 16, 40])
@pytest.mark.parametrize("batch", [129, 384, 1000])
def test_more_sequences_than_a_block_has_threads(batch, heads):
    """The division of the work gives a thread several sequences then, some of them with one position only."""
    lengths = [(i * 37) % 90 for i in range(batch)]
    su = pc.set_up(dict(starts=lengths, S=1, page=16, hkv=1 if heads else 2), pc.BF, False, "cuda", values=heads is None, d=576 if heads else 64)
    q, q_pe = su.normal(batch, 1, heads or 8, 512 if heads else 64), su.normal(batch, 1, heads or 8, 64)
    if heads:
        got = ops.paged_latent_attention(q, q_pe, su.k_pages, su.table, su.starts, None, None, 0.07)
        want, tol = po.attention(su, torch.cat((q, q_pe), -1), 0.07, latent=512, p_type=pc.BF)
    else:
        got = ops.paged_attention(q, su.k_pages, su.v_pages, su.table, su.starts)
        want, tol = po.attention(su, q, 64**-0.5, p_type=pc.BF)
    po.check_attention(got, want, tol, "many sequences")
