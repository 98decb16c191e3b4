# SPDX-License-Identifier: Apache-2.0
"""Cases of the paged generation cache: appending rotated keys and values (plain and 8-bit), the latent form of the same,
reading a cache back, and attention of new tokens over it.

Where ``own`` is false the operators are computed from elementary torch operations in 32 bits; where it is true the
calls of ``arctictraining_b200.ops`` are made.  ``exact`` restates each operator in 64 bits, sequence by sequence."""

import math

import torch

own = False

E4M3_MAX = 448.0
TINY = 2.0**-100  # a row whose largest value is below this is quantised as if it were this

# ------------------------------------------------------------------------------------------------ cases
# op: append / latent_append / read / attention / latent_attention.  length: the longest sequence; "ragged" sequences
# have lengths between `shortest` and it.  new: tokens of this call per sequence.  cache: "same" (the type of the
# inputs) or "e4m3" (8 bits with one scale per token and head).


def listed():
    return [
        # one sequence, one new token: the call that an interactive decoding step makes in every layer
        dict(name="append-one", op="append", batch=1, new=1, hq=32, hkv=8, dim=128, page=64, length=900, shortest=900,
             dtype="bfloat16", cache="same"),
        # prompts of unequal length, padded to one batch, written into an 8-bit cache
        dict(name="append-prompts-e4m3", op="append", batch=12, new=1511, hq=28, hkv=4, dim=128, page=32, length=1511,
             shortest=190, dtype="bfloat16", cache="e4m3"),
        # a decoding step of a batch over an 8-bit latent cache
        dict(name="latent-append-step-e4m3", op="latent_append", batch=96, new=1, hq=16, hkv=1, dim=576, page=64,
             length=2900, shortest=40, dtype="bfloat16", cache="e4m3"),
        # a batch of prompts into a latent cache
        dict(name="latent-append-prompts", op="latent_append", batch=8, new=2048, hq=16, hkv=1, dim=576, page=64,
             length=2048, shortest=700, dtype="bfloat16", cache="same"),
        # the cached part of a conversation read back before its next prompt
        dict(name="read-chat", op="read", batch=2, new=0, hq=0, hkv=8, dim=128, page=16, length=2333, shortest=1200,
             dtype="bfloat16", cache="same"),
        # an 8-bit latent cache read back for a batch of long documents
        dict(name="read-latent-e4m3", op="read", batch=16, new=0, hq=0, hkv=1, dim=576, page=64, length=16000,
             shortest=5000, dtype="bfloat16", cache="e4m3"),
        # one sequence, short context: latency counts
        dict(name="attention-one", op="attention", batch=1, new=1, hq=32, hkv=8, dim=128, page=64, length=777,
             shortest=777, dtype="bfloat16", cache="same", window=0),
        # a decoding batch whose sequences have very different lengths; seven query heads share a key head
        dict(name="attention-ragged", op="attention", batch=64, new=1, hq=28, hkv=4, dim=128, page=16, length=6100,
             shortest=17, dtype="bfloat16", cache="same", window=0),
        # few sequences over very long 8-bit caches
        dict(name="attention-long-e4m3", op="attention", batch=4, new=1, hq=64, hkv=8, dim=128, page=64, length=131000,
             shortest=60000, dtype="bfloat16", cache="e4m3", window=0),
        # a draft of five tokens verified at once, in layers with a sliding window
        dict(name="attention-draft-window", op="attention", batch=24, new=5, hq=32, hkv=8, dim=64, page=32, length=9001,
             shortest=100, dtype="float16", cache="same", window=4096),
        # absorbed latent attention, 16 heads, one sequence
        dict(name="latent-attention-one", op="latent_attention", batch=1, new=1, hq=16, hkv=1, dim=576, page=64,
             length=4003, shortest=4003, dtype="bfloat16", cache="same"),
        # absorbed latent attention, 128 heads, a decoding batch
        dict(name="latent-attention-batch", op="latent_attention", batch=32, new=1, hq=128, hkv=1, dim=576, page=64,
             length=5000, shortest=600, dtype="bfloat16", cache="same"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "latent_append", "read", "attention", "attention", "attention", "latent_attention"])
    latent = op.startswith("latent") or (op == "read" and rng.random() < 0.4)
    if latent:
        hkv, dim, hq = 1, 576, rng.choice([16, 16, 16, 32, 64, 128])
    else:
        hkv, dim = rng.choice([1, 2, 4, 4, 8, 8]), rng.choice([64, 128, 128, 128, 256])
        hq = hkv * rng.choice([1, 2, 4, 4, 5, 7, 8])
    case = dict(op=op, hq=0 if op == "read" else hq, hkv=hkv, dim=dim, page=rng.choice([16, 16, 32, 64, 64, 128, 48]),
                dtype=rng.choice(["bfloat16", "bfloat16", "bfloat16", "float16"]), cache=rng.choice(["same", "same", "e4m3"]))
    batch = _log_int(rng, 1, 96)
    if op in ("append", "latent_append"):
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, min(2048, 16000 // batch)))
        length = new + (_log_int(rng, 1, max(1, min(4000, 64000 // batch))) if rng.random() < 0.5 or new == 1 else 0)
    elif op == "read":
        new, length = 0, _log_int(rng, 1, min(16000, 256000 // batch))
    else:
        new = 1 if rng.random() < 0.7 else rng.randint(2, 8)
        tokens = 400000 if op == "attention" else (64000 if hq > 32 else 160000)
        length = _log_int(rng, new, max(new, min(131000, tokens // batch // (1 if op == "attention" else new))))
    case.update(batch=batch, new=new, length=length, shortest=_log_int(rng, max(1, new), length) if batch > 1 and op not in ("append", "latent_append")
                else (max(1, length // 8) if batch > 1 else length))
    if op == "attention":
        case["window"] = 0 if rng.random() < 0.75 else _log_int(rng, 16, 8192)
    return case


def _lengths(case):
    """Tokens of every sequence after the call, spread evenly over the range in a fixed shuffled order: a case's work does not
    depend on the seed."""
    b, lo, hi = case["batch"], case["shortest"], case["length"]
    if b == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * 7 + 3) % b if math.gcd(7, b) == 1 else i) // (b - 1) for i in range(b)]


def _counts(case):
    """(cached before the call, new tokens) of every sequence."""
    new = case["new"]
    out = []
    for n in _lengths(case):
        c = min(new, n)
        out.append((n - c, c))
    return out


def _width(case):
    return -(-(max(max(s for s, _ in _counts(case)) + case["new"], case["length"])) // case["page"])


# ------------------------------------------------------------------------------------------------ inputs
def _quantise(x):
    """Rows of fp32 values as (e4m3, scale): scale = largest magnitude / 448."""
    scale = x.abs().amax(-1).clamp(min=TINY) / E4M3_MAX
    return (x * (1.0 / scale).unsqueeze(-1)).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _pages(shape, dtype, cache, gen):
    """A cache in use: every page holds keys (or values) of some sequence."""
    P, H, page, D = shape
    if cache == "same":
        return torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=gen), None
    values = torch.empty(shape, device="cuda", dtype=torch.float8_e4m3fn)
    scale = torch.empty(shape[:3], device="cuda")
    step = max(1, (1 << 27) // (H * page * D))
    for p in range(0, P, step):
        x = torch.empty((min(step, P - p), H, page, D), device="cuda").normal_(generator=gen)
        values[p : p + step], scale[p : p + step] = _quantise(x)
    return values, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=None):
        return torch.empty(shape, device="cuda", dtype=dtype or dt).normal_(generator=gen)

    dt = getattr(torch, case["dtype"])
    B, S, Hq, Hkv, D, page, op = (case[k] for k in ("batch", "new", "hq", "hkv", "dim", "page", "op"))
    counts = _counts(case)
    width = _width(case)
    n_pages = B * width + 3
    st = dict(op=op, dtype=dt, case=case)
    st["table"] = torch.randperm(n_pages, device="cuda", generator=gen)[: B * width].view(B, width).to(torch.int32)
    st["starts"] = torch.tensor([s for s, _ in counts], device="cuda", dtype=torch.int32)
    st["counts"] = torch.tensor([c for _, c in counts], device="cuda", dtype=torch.int32) if any(c != S for _, c in counts) else None
    st["k_pages"], st["k_scale"] = _pages((n_pages, Hkv, page, D), dt, case["cache"], gen)
    if op in ("append", "attention") or (op == "read" and D != 576):
        st["v_pages"], st["v_scale"] = _pages((n_pages, Hkv, page, D), dt, case["cache"], gen)
    else:
        st["v_pages"] = st["v_scale"] = None
    if op in ("append", "latent_append"):
        rot = D if op == "append" else 64
        pos = st["starts"].double().view(B, 1, 1) + torch.arange(S, device="cuda").view(1, S, 1)
        ang = pos * (10000.0 ** (-torch.arange(0, rot, 2, device="cuda").double() / rot))
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
    if op == "append":  # the projection's output, split into heads: strided views of one tensor
        qkv = normal(B, S, (Hq + 2 * Hkv) * D)
        q, k, v = qkv.split([Hq * D, Hkv * D, Hkv * D], dim=-1)
        st["q"], st["k"], st["v"] = q.view(B, S, Hq, D), k.view(B, S, Hkv, D), v.view(B, S, Hkv, D)
    elif op == "latent_append":
        st["q_pe"] = normal(B, S, Hq, 192)[..., 128:]
        st["kv_a"] = normal(B, S, D)
        st["weight"], st["eps"] = (1.0 + 0.1 * normal(512, dtype=torch.float32)).to(dt), 1e-6
    elif op == "attention":
        st["q"] = normal(B, S, Hq, D) * 2.5
        st["scale"] = D**-0.5
    elif op == "latent_attention":
        st["q"], st["q_pe"] = normal(B, S, Hq, 512) * 0.6, normal(B, S, Hq, 64) * 0.6
        st["scale"] = 192**-0.5
    elif op == "read":
        st["lengths"] = torch.tensor([s + c for s, c in counts], device="cuda", dtype=torch.int32)
        st["max_length"] = case["length"]
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half].float(), x[..., half:].float()
    c, s = cos.unsqueeze(2), sin.unsqueeze(2)
    return torch.cat((a * c - b * s, b * c + a * s), dim=-1)


def _write(pages, scales, rows, st):
    """rows [B, S, H, D] in fp32 to their places; tokens behind a sequence's count leave the cache as it is."""
    B, S = rows.shape[:2]
    page = pages.shape[2]
    pos = st["starts"].long().view(B, 1) + torch.arange(S, device="cuda")
    pid = torch.gather(st["table"].long(), 1, pos // page)
    off = pos % page
    keep = torch.ones((B, S), device="cuda", dtype=torch.bool)
    if st["counts"] is not None:
        keep = torch.arange(S, device="cuda") < st["counts"].view(B, 1)
    if scales is None:
        pages[pid, :, off] = torch.where(keep.view(B, S, 1, 1), rows.to(pages.dtype), pages[pid, :, off])
    else:
        values, sc = _quantise(rows)
        raw = pages.view(torch.uint8)
        raw[pid, :, off] = torch.where(keep.view(B, S, 1, 1), values.view(torch.uint8), raw[pid, :, off])
        scales[pid, :, off] = torch.where(keep.view(B, S, 1), sc, scales[pid, :, off])


def _gather(pages, scales, table):
    """A cache as fp32 [B, H, positions, D]."""
    x = (pages if scales is None else pages.view(torch.uint8))[table.long()]
    x = x.float() if scales is None else x.view(torch.float8_e4m3fn).float()
    if scales is not None:
        x = x * scales[table.long()].unsqueeze(-1)
    B, W, H, page, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, W * page, D)


def _attend(q, k, v, st, scale, window):
    """q [B, S, Hq, D], k / v [B, Hkv, L, ...] in fp32."""
    B, S, Hq, _ = q.shape
    Hkv, L = k.shape[1:3]
    G = Hq // Hkv
    qf = q.float().view(B, S, Hkv, G, -1).permute(0, 2, 1, 3, 4).reshape(B, Hkv, S * G, -1)
    at = torch.arange(L, device="cuda").view(1, 1, L)
    j = torch.arange(S, device="cuda").view(1, S, 1)
    mine = st["starts"].long().view(B, 1, 1) + j
    seen = at <= mine
    if window:
        seen = seen & (at > mine - window)
    if st["counts"] is not None:
        seen = seen & (j < st["counts"].view(B, 1, 1))
    seen = seen.view(B, 1, S, 1, L).expand(B, 1, S, G, L).reshape(B, 1, S * G, L)
    scores = (torch.matmul(qf, k.transpose(-1, -2)) * scale).masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return o.view(B, Hkv, S, G, -1).permute(0, 2, 1, 3, 4).reshape(B, S, Hq, -1).to(q.dtype)


def _run_plain(st):
    op = st["op"]
    if op == "append":
        _write(st["k_pages"], st["k_scale"], _rotate(st["k"], st["cos"], st["sin"]), st)
        _write(st["v_pages"], st["v_scale"], st["v"].float(), st)
        return _rotate(st["q"], st["cos"], st["sin"]).to(st["dtype"])
    if op == "latent_append":
        a = st["kv_a"].float()
        latent, k_pe = a[..., :512], a[..., 512:]
        latent = latent * torch.rsqrt(latent.square().mean(-1, keepdim=True) + st["eps"]) * st["weight"].float()
        row = torch.cat((latent.unsqueeze(2), _rotate(k_pe.unsqueeze(2), st["cos"], st["sin"])), dim=-1)
        _write(st["k_pages"], st["k_scale"], row, st)
        return _rotate(st["q_pe"], st["cos"], st["sin"]).to(st["dtype"])
    if op == "read":
        n = st["max_length"]
        keep = torch.arange(n, device="cuda").view(1, n) < st["lengths"].view(-1, 1)
        got = []
        for pages, scales in ((st["k_pages"], st["k_scale"]), (st["v_pages"], st["v_scale"])):
            if pages is not None:
                x = _gather(pages, scales, st["table"])[:, :, :n].transpose(1, 2)
                got.append(torch.where(keep.view(*keep.shape, 1, 1), x, torch.zeros_like(x)).to(st["dtype"]))
        return got
    k = _gather(st["k_pages"], st["k_scale"], st["table"])
    if op == "attention":
        return _attend(st["q"], k, _gather(st["v_pages"], st["v_scale"], st["table"]), st, st["scale"], st["case"]["window"])
    return _attend(torch.cat((st["q"], st["q_pe"]), dim=-1), k, k[..., :512], st, st["scale"], 0)


def _run_own(st):
    from arctictraining_b200 import ops

    op = st["op"]
    if op == "append":
        return ops.paged_kv_append(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["k_pages"], st["v_pages"], st["table"],
                                   st["starts"], st["counts"], st["k_scale"], st["v_scale"])
    if op == "latent_append":
        return ops.paged_latent_append(st["q_pe"], st["kv_a"], st["weight"], st["eps"], st["cos"], st["sin"], st["k_pages"],
                                       st["table"], st["starts"], st["counts"], st["k_scale"])
    if op == "read":
        k, v = ops.paged_kv_read(st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["max_length"], st["k_scale"],
                                 st["v_scale"], st["dtype"])
        return [k] if v is None else [k, v]
    if op == "attention":
        return ops.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["starts"], st["counts"], st["k_scale"],
                                   st["v_scale"], st["scale"], st["case"]["window"] or None)
    return ops.paged_latent_attention(st["q"], st["q_pe"], st["k_pages"], st["table"], st["starts"], st["counts"], st["k_scale"],
                                      st["scale"])


def run(st):
    out = _run_own(st) if own else _run_plain(st)
    if st["op"] in ("append", "latent_append"):
        got = {"q": out, "k_pages": st["k_pages"]}
        if st["v_pages"] is not None:
            got["v_pages"] = st["v_pages"]
        if st["k_scale"] is not None:
            got["k_scale"] = st["k_scale"]
            if st["v_scale"] is not None:
                got["v_scale"] = st["v_scale"]
        return got
    return out


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    """Bytes: every new token's inputs and outputs once, every cached row that some query sees once.  FLOPs: two per
    multiply-add of the two products of attention."""
    el = 2
    D, Hq, Hkv, op = case["dim"], case["hq"], case["hkv"], case["op"]
    row = Hkv * (D * el if case["cache"] == "same" else D + 4)
    counts = _counts(case)
    table = 4 * sum(-(-(s + c) // case["page"]) for s, c in counts)
    total = sum(c for _, c in counts)
    B, S = case["batch"], case["new"]
    if op == "append":
        # every query of the padded batch is rotated; keys and values of the real tokens are read and written
        per = B * S * (Hq * D * el * 2 + D * 4)
        return {"bytes": per + total * (2 * Hkv * D * el + 2 * row), "flops": 3.0 * (B * S * Hq * D + total * Hkv * D)}
    if op == "latent_append":
        per = B * S * (Hq * 64 * el * 2 + 64 * 4)
        return {"bytes": per + total * (D * el + row), "flops": 3.0 * B * S * Hq * 64 + 6.0 * total * D}
    if op == "read":
        two = 1 if D == 576 else 2
        tokens = sum(s + c for s, c in counts)
        return {"bytes": two * (tokens * row + B * case["length"] * Hkv * D * el) + table, "flops": float(two * tokens * Hkv * D)}
    window = case.get("window") or 0
    seen_rows = pairs = 0
    for s, c in counts:
        first = max(0, s + 1 - window) if window else 0
        seen_rows += (s + c - first) if c else 0
        for j in range(c):
            pairs += min(s + j + 1, window) if window else s + j + 1
    if op == "attention":
        return {"bytes": B * S * Hq * D * el * 2 + 2 * seen_rows * row + table, "flops": 4.0 * pairs * Hq * D}
    return {"bytes": B * S * Hq * (576 + 512) * el + seen_rows * row + table, "flops": 2.0 * pairs * Hq * (576 + 512)}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def _exact_row_values(pages, scales, page_ids, head, n):
    x = (pages if scales is None else pages.view(torch.uint8))[page_ids, head]
    x = x.double() if scales is None else x.view(torch.float8_e4m3fn).double() * scales[page_ids, head].double().unsqueeze(-1)
    return x.reshape(-1, x.shape[-1])[:n]


def _exact_turn(x, cos, sin):
    x = x.double()
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(cos.double(), sin.double()).unsqueeze(-2)
    return torch.cat((z.real, z.imag), dim=-1)


def exact(case, seed):
    st = prepare(case, seed)
    op, page = case["op"], case["page"]
    counts = _counts(case)
    if op in ("append", "latent_append"):
        if op == "append":
            news = {"k": _exact_turn(st["k"], st["cos"], st["sin"]), "v": st["v"].double()}
            out = {"q": _exact_turn(st["q"], st["cos"], st["sin"])}
        else:
            a = st["kv_a"].double()
            lat = a[..., :512] / (a[..., :512].pow(2).sum(-1, keepdim=True) / 512 + st["eps"]).sqrt() * st["weight"].double()
            news = {"k": torch.cat((lat.unsqueeze(2), _exact_turn(a[..., 512:].unsqueeze(2), st["cos"], st["sin"])), -1)}
            out = {"q": _exact_turn(st["q_pe"], st["cos"], st["sin"])}
        for name, rows in news.items():
            pages, scales = st[name + "_pages"], st[name + "_scale"]
            whole = pages.double()
            whole_scale = None if scales is None else scales.double()
            for b, (s, c) in enumerate(counts):
                at = torch.arange(s, s + c, device="cuda")
                pid, off = st["table"][b].long()[at // page], at % page
                r = rows[b, :c]
                if scales is not None:
                    sc = r.abs().amax(-1).clamp(min=TINY) / E4M3_MAX
                    whole_scale[pid, :, off] = sc
                    r = r / sc.unsqueeze(-1)
                whole[pid, :, off] = r
            out[name + "_pages"] = whole
            if scales is not None:
                out[name + "_scale"] = whole_scale
        return out
    if op == "read":
        got = []
        for pages, scales in ((st["k_pages"], st["k_scale"]), (st["v_pages"], st["v_scale"])):
            if pages is None:
                continue
            x = torch.zeros((case["batch"], case["length"], case["hkv"], case["dim"]), device="cuda", dtype=torch.float64)
            for b, (s, c) in enumerate(counts):
                for h in range(case["hkv"]):
                    x[b, : s + c, h] = _exact_row_values(pages, scales, st["table"][b].long(), h, s + c)
            got.append(x)
        return got
    q = st["q"].double() if op == "attention" else torch.cat((st["q"], st["q_pe"]), -1).double()
    G, dv = case["hq"] // case["hkv"], case["dim"] if op == "attention" else 512
    window = case.get("window") or 0
    out = torch.zeros((case["batch"], case["new"], case["hq"], dv), device="cuda", dtype=torch.float64)
    for b, (s, c) in enumerate(counts):
        for h in range(case["hkv"]):
            k = _exact_row_values(st["k_pages"], st["k_scale"], st["table"][b].long(), h, s + c)
            v = _exact_row_values(st["v_pages"], st["v_scale"], st["table"][b].long(), h, s + c) if op == "attention" else k[:, :512]
            for j in range(c):
                lo = max(0, s + j + 1 - window) if window else 0
                logits = q[b, j, h * G : (h + 1) * G] @ k[lo : s + j + 1].T * st["scale"]
                out[b, j, h * G : (h + 1) * G] = torch.softmax(logits, -1) @ v[lo : s + j + 1]
    return out
