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


@pytest.mark.parametrize("window", [None, 2])
@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
def test_hidden_values_that_are_not_finite(dtype, e4m3, window):
    pc.not_finite_case(dtype, e4m3, "cuda", window=window)


@pytest.mark.parametrize("heads", [8, 64])
@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
def test_hidden_latents_that_are_not_finite(dtype, e4m3, heads):
    pc.not_finite_case(dtype, e4m3, "cuda", latent=True, heads=heads)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0])
@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
def test_scales_of_any_sign(dtype, e4m3, scale):
    pc.attention_case(pc.ATTENTION["draft-window"], dtype, e4m3, "cuda", scale)
    pc.latent_case(pc.LATENT["draft"], dtype, e4m3, "cuda", scale)
    pc.latent_case(pc.LATENT["sixty-four-heads-draft"], dtype, e4m3, "cuda", scale)


@pytest.mark.parametrize("heads,latent", [(8, False), (8, True), (40, True)])
@pytest.mark.parametrize("dtype,e4m3", TYPES, ids=str)
def test_one_bad_query(dtype, e4m3, heads, latent):
    pc.one_bad_query_case(dtype, e4m3, "cuda", heads, latent)


def test_counts_beyond_the_call_and_below_none():
    """A count is limited to the call's tokens and to none."""
    su, q = _attention_inputs([50, 60, 70], S=3)
    args = (q, su.k_pages, su.v_pages, su.table, su.starts)
    want = ops.paged_attention(*args)
    counts = torch.tensor([3, 9, -4], dtype=torch.int32, device="cuda")
    got = ops.paged_attention(*args, counts)
    assert torch.equal(got[:2], want[:2]) and torch.equal(got[2], torch.zeros_like(got[2]))


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


def _attention_inputs(starts, S=1, hq=16, hkv=4, d=128, e4m3=False, seed=0):
    su = pc.set_up(dict(starts=starts, S=S, page=16), pc.BF, e4m3, "cuda", d=d, hkv=hkv, seed=seed)
    return su, su.normal(su.B, S, hq, d)


def _latent_inputs(starts, h, S=1, e4m3=False, seed=0):
    su = pc.set_up(dict(starts=starts, S=S, page=64), pc.BF, e4m3, "cuda", values=False, d=576, seed=seed)
    q, q_pe = su.normal(su.B, S, h, 512), su.normal(su.B, S, h, 64)
    return lambda: ops.paged_latent_attention(q, q_pe, su.k_pages, su.table, su.starts, None, su.k_scale, 0.07)


@pytest.mark.parametrize("e4m3", [False, True])
def test_same_bits_every_time(e4m3):
    """Also with another call between, whose workspace may be the same memory, and without any wait."""
    su, q = _attention_inputs([5000, 17, 1234, 900], e4m3=e4m3)
    other, oq = _attention_inputs([700, 2500, 9, 40, 41], e4m3=e4m3, seed=5)

    def of(s, x):
        return lambda: ops.paged_attention(x, s.k_pages, s.v_pages, s.table, s.starts, None, s.k_scale, s.v_scale)

    calls = [of(su, q), of(other, oq)] + [_latent_inputs([3000, 17, 800], h, e4m3=e4m3, seed=h) for h in (16, 40, 128)]
    first = []
    for f in calls:
        first.append(f())
        torch.cuda.synchronize()
    got = [(i, calls[i]()) for _ in range(6) for i in (0, 1, 2, 4, 3, 0, 4, 1)]
    for i, x in got:
        assert torch.equal(x.view(torch.int16), first[i].view(torch.int16)), i


@pytest.mark.parametrize("h", [16, 128])
def test_latent_attention_captured_and_on_two_streams(h):
    calls = [_latent_inputs([2500, 3], h, seed=1), _latent_inputs([900, 1700, 64], h, seed=2)]
    want = [f() for f in calls]
    graphs, outs = [], []
    for f in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(f())
        graphs.append(graph)
    for _ in range(3):
        for x in outs:
            x.zero_()
        for graph in graphs:
            graph.replay()
        assert all(torch.equal(x, w) for x, w in zip(outs, want))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    assert torch.ops.atb200.read_and_clear_error_flag(want[0]) == 0


def test_a_captured_generation_step():
    """Append and attention of a decoding step in one graph, replayed while the cache grows: lengths are read on the device."""
    from arctictraining_b200.models import PagedKVCache

    def normal(*shape):
        return torch.randn(*shape, device="cuda").to(pc.BF)

    torch.manual_seed(0)
    caches = [PagedKVCache(1, 2, 128, 3, 200, page=32, device="cuda") for _ in range(2)]
    q, k, v, pos = normal(3, 1, 8, 128), normal(3, 1, 2, 128), normal(3, 1, 2, 128), torch.zeros(3, 1, 64, device="cuda")
    for c in caches:
        c.reserve(200)
        c.k_pages[0].fill_(float("nan"))
        c.v_pages[0].fill_(float("nan"))

    def step(c):
        return c.attend(0, c.append(0, q, k, v, pos.cos(), pos.sin()))

    step(caches[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    for i in range(150):
        for x in (q, k, v):
            x.normal_()
        pos.fill_(0.1 * i)
        graph.replay()
        assert torch.equal(out, step(caches[1])), i
        for c in caches:
            c.advance(1)


def test_two_captured_graphs_replayed_in_turn():
    """Each graph has a workspace of its own, and reads the lengths and pages of the moment it is replayed."""
    sets = [_attention_inputs([3000, 40], seed=1), _attention_inputs([700, 2500, 9], seed=2)]

    def call(i):
        su, q = sets[i]
        return ops.paged_attention(q, su.k_pages, su.v_pages, su.table, su.starts)

    want = [call(0), call(1)]
    graphs, outs = [], []
    for i in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call(i)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(i)
        graphs.append(graph)
        outs.append(out)
    for _ in range(3):
        for i in range(2):
            outs[i].zero_()
        graphs[0].replay()
        graphs[1].replay()
        for i in range(2):
            assert torch.equal(outs[i], want[i])
    su, q = sets[0]
    su.starts.fill_(39)
    graphs[0].replay()
    assert torch.equal(outs[0], call(0)) and not torch.equal(outs[0], want[0])


def test_two_streams_at_once():
    sets = [_attention_inputs([4000, 300], seed=3), _attention_inputs([2000, 3000, 1], seed=4)]
    want = [ops.paged_attention(q, su.k_pages, su.v_pages, su.table, su.starts) for su, q in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, (su, q) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.paged_attention(q, su.k_pages, su.v_pages, su.table, su.starts))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_a_strided_query_and_pages_of_one_tensor():
    """Queries as a view of a projection output, misaligned queries, and keys and values that share one allocation."""
    su, q = _attention_inputs([333, 90])
    want = ops.paged_attention(q, su.k_pages, su.v_pages, su.table, su.starts)
    wide = torch.randn(2, 1, 40 * 128, device="cuda").to(pc.BF)
    wide[..., : 16 * 128] = q.reshape(2, 1, -1)
    view = wide[..., : 16 * 128].unflatten(-1, (16, 128))
    odd = torch.empty(q.numel() + 1, device="cuda", dtype=pc.BF)[1:].view(q.shape).copy_(q)
    both = torch.stack([su.k_pages, su.v_pages], 1)
    table = torch.cat([su.table, torch.full_like(su.table, -7)], 1)[:, : su.W]
    for args in ((view, su.k_pages, su.v_pages, su.table), (odd, su.k_pages, su.v_pages, su.table), (q, both[:, 0], both[:, 1], table)):
        assert torch.equal(ops.paged_attention(*args, su.starts), want)


def test_pages_shared_by_sequences():
    """Two sequences with a common prefix read the same pages."""
    su, q = _attention_inputs([100, 100])
    table = su.table.clone()
    table[1, :5] = table[0, :5]
    got = ops.paged_attention(q, su.k_pages, su.v_pages, table, su.starts)
    su.table_list = table.tolist()
    po.check_attention(got, *po.attention(su, q, 128**-0.5, p_type=pc.BF))


def test_a_cache_of_more_than_2_31_elements():
    """Offsets past 2^31 elements (and 2^32 bytes): the last page of a large pool."""
    n = (2**31 + 2**20) // (2 * 64 * 128)
    pages = torch.zeros(n, 2, 64, 128, device="cuda", dtype=pc.BF)
    pages[-1].normal_()
    table = torch.tensor([[n - 1]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([63], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 1, 8, 128, device="cuda").to(pc.BF)
    small = pages[-1:].clone()
    assert torch.equal(ops.paged_attention(q, pages, pages, table, starts),
                       ops.paged_attention(q, small, small, torch.zeros_like(table), starts))
    got, _ = ops.paged_kv_read(pages, None, table, starts, 63)
    assert torch.equal(got[0], small[0, :, :63].transpose(0, 1))
    kv, cos, sin = torch.randn(1, 1, 2, 128, device="cuda").to(pc.BF), torch.ones(1, 1, 64, device="cuda"), torch.zeros(1, 1, 64, device="cuda")
    ops.paged_kv_append(q, kv, kv, cos, sin, pages, pages, table, starts - 3)
    assert torch.equal(pages[-1, :, 60], kv[0, 0])
