# SPDX-License-Identifier: Apache-2.0
"""Cases and checks of the paged-cache operators that the CPU (reference) and the GPU (kernels) tests share."""

import paged_oracle as po
import torch

from arctictraining_b200 import ops

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32

# starts, new tokens, query heads, cache heads, dim, page, counts, window, missing pages (sequence, place, id)
ATTENTION = {
    "one-token-cache": dict(starts=[0], S=1, hq=4, hkv=4, d=64, page=16),
    "one-sequence": dict(starts=[776], S=1, hq=32, hkv=8, d=128, page=64),
    "ragged": dict(starts=[0, 15, 16, 17, 333, 64, 1], S=1, hq=14, hkv=2, d=128, page=16),
    "group-of-seven": dict(starts=[130, 95], S=1, hq=7, hkv=1, d=128, page=32),
    "group-of-five-odd-page": dict(starts=[101, 7], S=1, hq=10, hkv=2, d=64, page=24),
    "page-of-one": dict(starts=[37, 5], S=1, hq=4, hkv=1, d=64, page=1),
    "long-page": dict(starts=[700, 900], S=1, hq=4, hkv=2, d=64, page=1000),
    "draft": dict(starts=[0, 40, 257], S=5, hq=8, hkv=2, d=64, page=16),
    "draft-window": dict(starts=[0, 40, 257, 1023], S=5, hq=8, hkv=2, d=128, page=32, window=48),
    "window-of-one": dict(starts=[9, 100], S=3, hq=4, hkv=2, d=64, page=16, window=1),
    "counts": dict(starts=[3, 60, 0, 31], S=6, hq=8, hkv=4, d=128, page=16, counts=[6, 2, 0, 1]),
    "missing-pages": dict(starts=[100, 70, 40], S=2, hq=8, hkv=2, d=64, page=16,
                          lose=((0, 1, -1), (0, 3, 10**6), (1, 4, -5), (2, 0, -1), (2, 1, -1), (2, 2, 10**9))),
    "negative-start": dict(starts=[-3, 20], S=2, hq=4, hkv=2, d=64, page=16),
    "chunk": dict(starts=[0, 70, 200], S=40, hq=12, hkv=2, d=128, page=16),
    "wide-head": dict(starts=[300, 31], S=2, hq=8, hkv=4, d=256, page=32),
    "narrow-head": dict(starts=[300, 31], S=1, hq=8, hkv=4, d=16, page=32),
    "head-of-80": dict(starts=[200, 31], S=2, hq=8, hkv=4, d=80, page=32),
    "many-heads": dict(starts=[150], S=3, hq=64, hkv=1, d=128, page=64),
    "long": dict(starts=[9000, 4097], S=1, hq=8, hkv=1, d=128, page=64),
}
LATENT = {
    "one-token-cache": dict(starts=[0], S=1, h=16, R=512, rope=64, page=16),
    "one-sequence": dict(starts=[1500], S=1, h=16, R=512, rope=64, page=64),
    "ragged": dict(starts=[0, 15, 16, 700, 63, 64], S=1, h=16, R=512, rope=64, page=32),
    "draft": dict(starts=[0, 77, 300], S=3, h=16, R=512, rope=64, page=16),
    "many-heads": dict(starts=[100, 333], S=1, h=128, R=512, rope=64, page=64),
    "many-heads-draft": dict(starts=[5, 90], S=2, h=128, R=512, rope=64, page=64),
    "twenty-heads": dict(starts=[200, 10], S=3, h=20, R=512, rope=64, page=48),
    "sixty-four-heads-draft": dict(starts=[200, 31, 0], S=3, h=64, R=512, rope=64, page=48),
    "hundred-heads": dict(starts=[400, 64], S=2, h=100, R=512, rope=64, page=64, counts=[2, 1]),
    "two-hundred-heads-missing": dict(starts=[130, 63], S=1, h=200, R=512, rope=64, page=16, lose=((0, 2, -1), (1, 0, 10**8), (0, 8, -3))),
    "many-heads-long": dict(starts=[5000, 33, 1777], S=1, h=128, R=512, rope=64, page=64),
    "many-heads-page-of-one": dict(starts=[45], S=1, h=64, R=512, rope=64, page=1),
    "many-heads-negative-start": dict(starts=[-2, 31], S=2, h=128, R=512, rope=64, page=16),
    "small-widths": dict(starts=[90, 3], S=2, h=6, R=48, rope=16, page=16),
    "counts-missing": dict(starts=[60, 20, 0], S=4, h=16, R=512, rope=64, page=16, counts=[2, 4, 0], lose=((1, 0, -1), (0, 1, 10**7))),
}


def set_up(c, dtype, e4m3, device, values=True, d=None, hkv=None, seed=0):
    return po.Setup(c["starts"], c["S"], hkv or c.get("hkv", 1), d or c.get("d"), c["page"], dtype, e4m3, counts=c.get("counts"),
                    lose=c.get("lose", ()), device=device, values=values, seed=seed)


def p_type(dtype, e4m3):
    """What probabilities are rounded to: the model's type, fp16 for an 8-bit cache."""
    return F32 if dtype == F32 else HF if e4m3 else dtype


def attention_case(c, dtype, e4m3, device, scale=None):
    su = set_up(c, dtype, e4m3, device)
    q = su.normal(su.B, su.S, c["hq"], su.D) * 2
    scale = su.D**-0.5 if scale is None else scale
    got = ops.paged_attention(q, su.k_pages, su.v_pages, su.table, su.starts, su.counts, su.k_scale, su.v_scale, scale, c.get("window"))
    assert got.dtype == dtype and got.shape == q.shape
    want, tol = po.attention(su, q, scale, c.get("window"), p_type=p_type(dtype, e4m3))
    po.check_attention(got, want, tol, "attention")


def latent_case(c, dtype, e4m3, device, scale=192**-0.5):
    su = set_up(c, dtype, e4m3, device, values=False, d=c["R"] + c["rope"])
    q, q_pe = su.normal(su.B, su.S, c["h"], c["R"]), su.normal(su.B, su.S, c["h"], c["rope"])
    got = ops.paged_latent_attention(q, q_pe, su.k_pages, su.table, su.starts, su.counts, su.k_scale, scale)
    assert got.dtype == dtype and got.shape == q.shape
    want, tol = po.attention(su, torch.cat((q, q_pe), -1), scale, latent=c["R"], p_type=p_type(dtype, e4m3))
    po.check_attention(got, want, tol, "latent attention")


def append_case(c, dtype, e4m3, device):
    su = set_up(c, dtype, e4m3, device)
    width = (c["hq"] + 2 * su.Hkv) * su.D
    q, k, v = su.normal(su.B, su.S, width).split([c["hq"] * su.D, su.Hkv * su.D, su.Hkv * su.D], -1)  # strided views
    q, k, v = q.unflatten(-1, (-1, su.D)), k.unflatten(-1, (-1, su.D)), v.unflatten(-1, (-1, su.D))
    cos, sin = su.angles(su.D)
    before = [t.clone() if t is not None else None for t in (su.k_pages, su.k_scale, su.v_pages, su.v_scale)]
    q0 = q.clone()
    got = ops.paged_kv_append(q, k, v, cos, sin, su.k_pages, su.v_pages, su.table, su.starts, su.counts, su.k_scale, su.v_scale)
    assert got.dtype == dtype and got.shape == q.shape and torch.equal(q, q0)
    po.check_rounded(got, *po.rotate(q, cos, sin), "queries")
    po.check_written(su, su.k_pages, su.k_scale, before[0], before[1], *po.rotate(k, cos, sin), "keys")
    vd = v.cpu().double()
    po.check_written(su, su.v_pages, su.v_scale, before[2], before[3], vd, torch.zeros_like(vd), "values")


def latent_append_case(c, dtype, e4m3, device):
    su = set_up(c, dtype, e4m3, device, values=False, d=c["R"] + c["rope"])
    R, eps = c["R"], 1e-6
    q_pe = su.normal(su.B, su.S, c["h"], 32 + c["rope"])[..., 32:]  # the rotary part of whole query heads
    kv_a = su.normal(su.B, su.S, su.D) * 3
    w = su.normal(R)
    cos, sin = su.angles(c["rope"])
    before = (su.k_pages.clone(), su.k_scale.clone() if e4m3 else None)
    got = ops.paged_latent_append(q_pe, kv_a, w, eps, cos, sin, su.k_pages, su.table, su.starts, su.counts, su.k_scale)
    assert got.dtype == dtype and got.shape == q_pe.shape
    po.check_rounded(got, *po.rotate(q_pe, cos, sin), "queries")
    a = kv_a.cpu().double()
    lat = a[..., :R] / (a[..., :R].pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.cpu().double()
    k_pe, slack = po.rotate(a[..., R:].unsqueeze(2), cos, sin)
    rows = torch.cat((lat.unsqueeze(2), k_pe), -1)
    # norm: a sum of R squares (R + 4 roundings, halved by the root), a reciprocal root good to 2^-21, two products
    slack = torch.cat((lat.abs().unsqueeze(2) * ((R + 4) * 2.0**-25 + 2.0**-20), slack), -1)
    po.check_written(su, su.k_pages, su.k_scale, before[0], before[1], rows, slack, "latent rows")


def read_case(c, dtype, e4m3, device, values=True):
    su = set_up(c, dtype, e4m3, device, values=values)
    for n in (su.W * su.page + 5, max(1, max(su.starts_list) // 2), 1):
        lengths = torch.tensor([s + x for s, x in zip(su.starts_list, su.counts_list)], dtype=torch.int32, device=device)
        k, v = ops.paged_kv_read(su.k_pages, su.v_pages, su.table, lengths, n, su.k_scale, su.v_scale, dtype)
        assert (v is None) == (not values)
        for got, pages, scale in ((k, su.k_pages, su.k_scale), (v, su.v_pages, su.v_scale)):
            if got is None:
                continue
            whole = po.values(pages, scale)
            want = torch.zeros(su.B, n, su.Hkv, su.D, dtype=torch.float64)
            for b in range(su.B):
                for p, pid, off in po.places(su.table_list[b], 0, int(lengths[b]), su.P, su.page):
                    if p < n:
                        want[b, p] = whole[pid, :, off]
            if e4m3:
                po.check_rounded(got, want, want.abs() * 2.0**-24, "read")
            else:
                po.check_close(got, want, torch.zeros_like(want), "read")


def refusals(device, dtype):
    """Calls that are refused with a ValueError: (name, function)."""
    c = dict(starts=[5, 9], S=2, hq=4, hkv=2, d=32, page=16)
    su, s8 = set_up(c, dtype, False, device), set_up(c, dtype, True, device)
    q, k, v = su.normal(2, 2, 4, 32), su.normal(2, 2, 2, 32), su.normal(2, 2, 2, 32)
    cos, sin = su.angles(32)
    lat = set_up(c, dtype, False, device, values=False, d=48, hkv=1)
    ql, qp, a, w = su.normal(2, 2, 4, 32), su.normal(2, 2, 4, 16), su.normal(2, 2, 48), su.normal(32)
    lc, ls = su.angles(16)
    other = HF if dtype != HF else BF

    def att(**kw):
        x = dict(q=q, k=su.k_pages, v=su.v_pages, t=su.table, s=su.starts, c=None, ks=None, vs=None, scale=None, w=None) | kw
        return lambda: ops.paged_attention(x["q"], x["k"], x["v"], x["t"], x["s"], x["c"], x["ks"], x["vs"], x["scale"], x["w"])

    def app(**kw):
        x = dict(q=q, k=k, v=v, cos=cos, sin=sin, kp=su.k_pages, vp=su.v_pages, t=su.table, s=su.starts, c=None, ks=None, vs=None) | kw
        return lambda: ops.paged_kv_append(*x.values())

    def lap(**kw):
        x = dict(q=qp, a=a, w=w, e=1e-6, cos=lc, sin=ls, p=lat.k_pages, t=lat.table, s=lat.starts, c=None, sc=None) | kw
        return lambda: ops.paged_latent_append(*x.values())

    def lat_att(**kw):
        x = dict(q=ql, p=qp, k=lat.k_pages, t=lat.table, s=lat.starts, c=None, sc=None, scale=0.1) | kw
        return lambda: ops.paged_latent_attention(*x.values())

    def read(**kw):
        x = dict(k=su.k_pages, v=su.v_pages, t=su.table, s=su.starts, n=8, ks=None, vs=None, d=None) | kw
        return lambda: ops.paged_kv_read(*x.values())

    grad = q.clone().requires_grad_(True)
    return {
        "attention: query of 3 dims": att(q=q[0]),
        "attention: other dim": att(q=su.normal(2, 2, 4, 16)),
        "attention: heads no multiple": att(q=su.normal(2, 2, 3, 32)),
        "attention: other batch": att(q=q[:1]),
        "attention: other type": att(k=su.k_pages.to(other), v=su.v_pages.to(other)),
        "attention: types differ": att(v=su.v_pages.to(other)),
        "attention: pages transposed": att(k=su.k_pages.transpose(1, 2).contiguous().transpose(1, 2)),
        "attention: pages of 3 dims": att(k=su.k_pages[0], v=su.v_pages[0]),
        "attention: page of none": att(k=su.k_pages[:, :, :0], v=su.v_pages[:, :, :0]),
        "attention: values further apart": att(v=torch.cat([su.v_pages, su.v_pages], 1)[:, :2]),
        "attention: values of other shape": att(v=su.v_pages[1:]),
        "attention: scales of a plain cache": att(ks=s8.k_scale, vs=s8.v_scale),
        "attention: no scales": att(k=s8.k_pages, v=s8.v_pages),
        "attention: one scale": att(k=s8.k_pages, v=s8.v_pages, ks=s8.k_scale),
        "attention: scales of other shape": att(k=s8.k_pages, v=s8.v_pages, ks=s8.k_scale[:, :1], vs=s8.v_scale),
        "attention: scales of other type": att(k=s8.k_pages, v=s8.v_pages, ks=s8.k_scale.double(), vs=s8.v_scale),
        "attention: table of longs": att(t=su.table.long()),
        "attention: table of other batch": att(t=su.table[:1]),
        "attention: table in columns": att(t=torch.cat([su.table, su.table], 1).t().contiguous().t()),
        "attention: starts of longs": att(s=su.starts.long()),
        "attention: starts strided": att(s=torch.stack([su.starts, su.starts], 1)[:, 0]),
        "attention: counts of other length": att(c=su.starts[:1]),
        "attention: window of none": att(w=0),
        "attention: window below none": att(w=-4),
        "attention: gradient": att(q=grad),
        "append: other shapes": app(k=k[:, :1]),
        "append: values of other shape": app(v=su.normal(2, 2, 1, 32)),
        "append: types differ": app(k=k.to(other)),
        "append: cos of half width": app(cos=cos[..., :8], sin=sin[..., :8]),
        "append: cos of 16 bits": app(cos=cos.to(dtype) if dtype != F32 else cos.double()),
        "append: other heads": app(k=su.normal(2, 2, 4, 32), v=su.normal(2, 2, 4, 32)),
        "append: no scales": app(kp=s8.k_pages, vp=s8.v_pages),
        "append: other type": app(kp=su.k_pages.to(other), vp=su.v_pages.to(other)),
        "append: gradient": app(q=grad),
        "latent append: other width": lap(a=su.normal(2, 2, 64)),
        "latent append: weight of 2 dims": lap(w=w.view(2, 16)),
        "latent append: weight of other type": lap(w=w.to(other)),
        "latent append: cache of heads": lap(p=su.k_pages),
        "latent append: cos of other width": lap(cos=cos, sin=sin),
        "latent append: gradient": lap(a=a.clone().requires_grad_(True)),
        "latent attention: other heads": lat_att(p=qp[:, :, :2]),
        "latent attention: types differ": lat_att(p=qp.to(other)),
        "latent attention: cache of other width": lat_att(k=su.k_pages),
        "latent attention: no scale": lat_att(scale=None),
        "latent attention: gradient": lat_att(q=ql.clone().requires_grad_(True)),
        "read: below none": read(n=-1),
        "read: other type": read(d=other),
        "read: no scales": read(k=s8.k_pages, v=s8.v_pages),
        "read: lengths of longs": read(s=su.starts.long()),
        "read: table of 1 dim": read(t=su.table[0]),
    }


def not_finite_case(dtype, e4m3, device, latent=False, window=None, heads=8):
    """A draft whose third token has a NaN key, an infinite value and a NaN value in some places: earlier queries (and, with a
    window, later ones that no longer see it) must not notice.  e4m3 rows hold a NaN scale instead."""
    c = dict(starts=[20, 70], S=5, hq=heads, hkv=1 if latent else 2, page=16)
    D, R = (576, 512) if latent else (64, None)
    su = set_up(c, dtype, e4m3, device, values=not latent, d=D)
    for b in range(2):
        p = su.starts_list[b] + 2
        pid, off = su.table_list[b][p // 16], p % 16
        if e4m3:
            (su.k_scale if latent else su.v_scale)[pid, 0, off] = float("nan")
        else:
            pages = su.k_pages if latent else su.v_pages
            pages[pid, 0, off, 3] = float("inf")
            pages[pid, 0, off, 8] = float("nan")
            if not latent:
                su.k_pages[pid, 1, off, 5] = float("nan")
    scale = 0.1
    if latent:
        q, q_pe = su.normal(2, 5, heads, R), su.normal(2, 5, heads, D - R)
        got = ops.paged_latent_attention(q, q_pe, su.k_pages, su.table, su.starts, None, su.k_scale, scale)
        want, tol = po.attention(su, torch.cat((q, q_pe), -1), scale, latent=R, p_type=p_type(dtype, e4m3))
    else:
        q = su.normal(2, 5, heads, D)
        got = ops.paged_attention(q, su.k_pages, su.v_pages, su.table, su.starts, None, su.k_scale, su.v_scale, scale, window)
        want, tol = po.attention(su, q, scale, window, p_type=p_type(dtype, e4m3))
    assert torch.isfinite(want[:, :2]).all() and not torch.isfinite(want[:, 2]).all()
    if window == 2:
        assert torch.isfinite(want[:, 4]).all()
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got))
    po.check_close(torch.where(fine, got, 0.0), torch.where(fine, want, 0.0),
                   torch.where(fine, tol * 1.01 + want.abs() * po.step(dtype) * 1.02 + po.floor(dtype), 0.0), "not finite")


def one_bad_query_case(dtype, e4m3, device, heads, latent):
    """A query with a NaN gets NaN; all others get what they get without it, bit for bit."""
    c = dict(starts=[300, 40], S=2, hq=heads, hkv=1 if latent else 2, page=16)
    su = set_up(c, dtype, e4m3, device, values=not latent, d=576 if latent else 128)
    q, q_pe = su.normal(2, 2, heads, 512 if latent else 128), su.normal(2, 2, heads, 64)

    def call():
        if latent:
            return ops.paged_latent_attention(q, q_pe, su.k_pages, su.table, su.starts, None, su.k_scale, 0.1)
        return ops.paged_attention(q, su.k_pages, su.v_pages, su.table, su.starts, None, su.k_scale, su.v_scale)

    want = call()
    q[0, 1, 3, 7] = float("nan")
    got = call()
    assert torch.isnan(got[0, 1, 3]).all()
    got[0, 1, 3] = want[0, 1, 3]
    assert torch.equal(got, want) and torch.isfinite(want).all()
