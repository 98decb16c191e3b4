# SPDX-License-Identifier: Apache-2.0
"""The paged-cache operators in 64 bits, position by position, with the largest error that a correct implementation in 32
bits with one final rounding may have.  Used by the CPU and the GPU tests."""

import torch

E4M3 = torch.float8_e4m3fn
TINY = 2.0**-100


def step(dtype):
    """Half a rounding step, relative (fp32: the unit of its own arithmetic)."""
    return torch.finfo(dtype).eps / 2


def floor(dtype):
    """Half a step below the smallest normal number."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def quantise(x):
    x = x.float()
    scale = x.abs().amax(-1).clamp(min=TINY) / 448.0
    return (x / scale.unsqueeze(-1)).clamp(-448, 448).to(E4M3), scale


def values(pages, scale):
    v = pages.cpu().double() if scale is None else pages.cpu().view(torch.uint8).view(E4M3).double()
    return v if scale is None else v * scale.cpu().double().unsqueeze(-1)


def places(table, start, n, P, page):
    """[(position, page, offset)] of positions start .. start + n that lie on a page that exists."""
    out = []
    for p in range(max(0, start), start + n):
        if p < len(table) * page and 0 <= table[p // page] < P:
            out.append((p, table[p // page], p % page))
    return out


class Setup:
    """A pool of pages whose unused places hold NaN, sequences of given lengths on shuffled pages, and the new tokens."""

    def __init__(self, starts, S, Hkv, D, page, dtype, e4m3=False, counts=None, seed=0, device="cpu", values=True, spare=2, lose=()):
        g = torch.Generator().manual_seed(seed)
        self.B, self.S, self.Hkv, self.D, self.page, self.dtype, self.e4m3 = len(starts), S, Hkv, D, page, dtype, e4m3
        self.g = g
        W = max(1, max((max(s, 0) + S + page - 1) // page for s in starts))
        P = self.B * W + spare
        table = torch.randperm(P, generator=g)[: self.B * W].view(self.B, W).to(torch.int32)
        for b, w, pid in lose:  # pages that are not there
            table[b, w] = pid
        self.P, self.W = P, W
        self.table_list = table.tolist()
        self.starts_list = list(starts)
        self.counts_list = list(counts) if counts is not None else [S] * self.B
        pools = []
        for _ in range(2 if values else 1):
            x = torch.randn(P, Hkv, page, D, generator=g)
            used = torch.zeros(P, page, dtype=torch.bool)
            for b in range(self.B):
                for _, pid, off in places(self.table_list[b], 0, self.starts_list[b] + min(S, max(0, self.counts_list[b])), P, page):
                    used[pid, off] = True
            hide = ~used.view(P, 1, page)
            if e4m3:
                q, sc = quantise(x * torch.exp2(torch.randint(-3, 4, (P, Hkv, page, 1), generator=g).float()))
                q.view(torch.uint8)[hide.expand(P, Hkv, page)] = 0x7F  # NaN
                sc[hide.expand(P, Hkv, page)] = float("nan")
                pools.append((q.to(device), sc.to(device)))
            else:
                x = x.to(dtype)
                x[hide.expand(P, Hkv, page)] = float("nan")
                pools.append((x.to(device), None))
        self.k_pages, self.k_scale = pools[0]
        self.v_pages, self.v_scale = pools[1] if values else (None, None)
        self.table = table.to(device)
        self.starts = torch.tensor(starts, dtype=torch.int32, device=device)
        self.counts = torch.tensor(counts, dtype=torch.int32, device=device) if counts is not None else None
        self.device = device

    def normal(self, *shape, dtype=None):
        return torch.randn(*shape, generator=self.g).to(dtype or self.dtype).to(self.device)

    def angles(self, width):
        ang = torch.rand(self.B, self.S, width // 2, generator=self.g) * 6.28
        return ang.cos().to(self.device), ang.sin().to(self.device)


def rotate(x, cos, sin):
    x, c, s = x.cpu().double(), cos.cpu().double().unsqueeze(2), sin.cpu().double().unsqueeze(2)
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    mag = torch.cat((a.abs() + b.abs(), a.abs() + b.abs()), -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1), mag * 2.0**-22  # three roundings of 2^-24 on sums of these magnitudes


def check_close(got, want, tol, what=""):
    got = got.cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    bad = (got - want).abs() > tol
    bad &= ~torch.isnan(want)
    if bad.any():
        i = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: got {got[i]}, want {want[i]}, may differ by {tol[i]}")


def check_rounded(got, want, slack, what=""):
    """One rounding to got's type, and ``slack`` of 32-bit arithmetic before it."""
    check_close(got, want, want.abs() * step(got.dtype) * (1 + 2.0**-10) + slack * 1.01 + floor(got.dtype), what)


def check_written(su, pages, scale, before, before_scale, rows, slack, what=""):
    """``rows [B, S, H, D]`` are in their places, and every other place is as it was, bit for bit."""
    raw, old = pages.cpu().view(torch.uint8 if su.e4m3 else su.dtype).clone(), before.cpu().view(torch.uint8 if su.e4m3 else su.dtype).clone()
    got = values(pages, scale)
    for b in range(su.B):
        for p, pid, off in places(su.table_list[b], su.starts_list[b], min(su.S, su.counts_list[b]) if su.starts_list[b] >= 0 else 0, su.P, su.page):
            want, sl = rows[b, p - su.starts_list[b]], slack[b, p - su.starts_list[b]]
            if su.e4m3:
                top = want.abs().amax(-1).clamp(min=TINY) / 448.0
                off_by = (scale.cpu()[pid, :, off].double() - top).abs()
                # the scale: the largest element's own error and one division
                assert bool((off_by <= top * 2.0**-22 + sl.amax(-1) / 448.0).all()), what
                tol = want.abs() * (step(E4M3) * 1.001) + top.unsqueeze(-1) * 2.0**-10 * 1.001 + sl * 1.2
                check_close(got[pid, :, off], want, tol, what)
                before_scale[pid, :, off] = scale[pid, :, off]
            else:
                check_rounded(pages.cpu()[pid, :, off], want, sl, what)
            old[pid, :, off] = raw[pid, :, off]
    as_int = torch.uint8 if su.e4m3 else {2: torch.int16, 4: torch.int32}[raw.element_size()]
    assert torch.equal(raw.view(as_int), old.view(as_int)), f"{what}: places of no new token changed"
    if scale is not None:
        assert torch.equal(scale.cpu().view(torch.int32), before_scale.cpu().view(torch.int32)), f"{what}: scales of no new token changed"


def attention(su, q, scale, window=None, latent=None, p_type=None):
    """(result, largest error) of queries ``q [B, S, Hq, D]``; ``latent``: width of the value part of a joint row.

    A probability is rounded once to ``p_type`` (half a step, relative; below its normal range half a step absolute of the
    largest, with an 8-bit cache's scales inside) and weighs |v|; a score's error of d changes it by a factor e^d; a score is
    a sum of D products in 32 bits (D + 8 roundings of its magnitudes) and goes through an exponential good to 2^-21."""
    k = values(su.k_pages, su.k_scale)
    v = k[..., :latent] if latent else values(su.v_pages, su.v_scale)
    q = q.cpu().double()
    B, S, Hq, D = q.shape
    G = Hq // su.Hkv
    out = torch.zeros(B, S, Hq, v.shape[-1], dtype=torch.float64)
    tol = torch.zeros_like(out)
    p_type = p_type or su.dtype
    for b in range(B):
        count = min(S, max(0, su.counts_list[b]))
        held = places(su.table_list[b], 0, su.starts_list[b] + count, su.P, su.page)
        for j in range(count):
            p = su.starts_list[b] + j
            seen = [(pid, off) for at, pid, off in held if at <= p and (window is None or at > p - window)]
            if not seen:
                continue
            pid, off = torch.tensor([s[0] for s in seen]), torch.tensor([s[1] for s in seen])
            for h in range(su.Hkv):
                qq, kk, vv = q[b, j, h * G : (h + 1) * G], k[pid, h, off], v[pid, h, off]
                s = qq @ kk.T * scale
                pr = torch.softmax(s, -1)
                d = ((qq.abs() @ kk.abs().T) * abs(scale) * (D + 8) + s.abs() * 8).amax(-1, keepdim=True) * 2.0**-24 + 2.0**-21
                mass = pr @ vv.abs()
                out[b, j, h * G : (h + 1) * G] = pr @ vv
                small = 0.0
                if p_type != torch.float32:
                    sc = (su.v_scale if not latent else su.k_scale).cpu().double()[pid, h, off] if su.e4m3 else torch.ones(len(seen), dtype=torch.float64)
                    top = (pr * sc).amax(-1, keepdim=True) * floor(p_type) * 2
                    small = top * (vv.abs() / sc.unsqueeze(-1)).sum(0)
                tol[b, j, h * G : (h + 1) * G] = mass * (step(p_type) + 3 * d + (len(seen) + 8) * 2.0**-24) + small
    return out, tol


def check_attention(got, want, tol, what=""):
    check_close(got, want, tol * 1.01 + want.abs() * step(got.dtype) * (1 + 2.0**-6) + floor(got.dtype), what)
