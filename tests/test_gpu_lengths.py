"""Lengths of the cache that shrink, grow unseen by the host, or are only bounded there (run on a B200: ``-m gpu``)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def rows(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


def make(layout, lens, page=16, blocks=200, capacity=None):
    import entmaxkv_b200 as E
    kw = dict(block_table=True, num_blocks=blocks) if layout == "pool" else {}
    c = E.PagedKVCache(page, capacity=capacity, **kw)
    k, v = rows(len(lens), 2, max(lens), 128, seed=1), rows(len(lens), 2, max(lens), 128, seed=2)
    c.initialize(k, v, seq_lens=lens)
    return c


def eager(cache, mode, q, k, v):
    import entmaxkv_b200 as E
    out = torch.zeros_like(q)
    if mode == "topk":
        E.sparse_attention_decode_paged(q, cache, k, v, out, 64, alpha=1.5, niter=10)
    else:
        E.sparse_attention_decode_gaussian_aware_entmax(q, cache, k, v, out, alpha=1.5, append_cache=True)
    return out


@pytest.mark.parametrize("layout", ["dense", "pool"])
@pytest.mark.parametrize("mode", ["topk", "gaussian"])
@pytest.mark.parametrize("pinned", [False, True])
def test_captured_steps_after_a_release(layout, mode, pinned):
    """A released sequence starts again through captured steps: the first capture, replays, and the capture that follows
    when the cache has to grow give what eager steps give."""
    from entmaxkv_b200.graph import DecodeStepGraph
    lens = [70, 90]
    one, two = make(layout, lens, capacity=96), make(layout, lens, capacity=96)
    kw = dict(token_budget=64) if mode == "topk" else {}
    graph = DecodeStepGraph(one, 4, mode, alpha=1.5, niter=10 if mode == "topk" else 2, **kw)
    for c in (one, two):
        c.release([0])
    for step in range(40):
        if step == 25:
            for c in (one, two):
                c.release([1])
        q, k, v = (rows(2, n, 1, 128, seed=10 * step + n) for n in (4, 2, 2))
        k, v = k, v * 0.5
        if pinned:
            io = graph.pinned_io()
            for name, t in (("q", q), ("k_new", k), ("v_new", v)):
                io[name].copy_(t)
            graph.step_pinned()
            torch.cuda.synchronize()
            got = io["out"].cuda()
        else:
            got = graph.step(q, k, v).clone()
        want = eager(two, mode, q, k, v)
        # the wider table of a grown cache may take another kernel: equal up to two roundings to bf16
        assert (got.float() - want.float()).abs().max() <= 2 * 2.0 ** -8 * max(want.abs().max().item(), 1e-3), step
        assert one.host_seq_lens == two.host_seq_lens and torch.equal(one.seq_lens, two.seq_lens), step
    assert one.seq_lens.tolist() == [40, 15] and one.device_status() == 0
    for b, n in enumerate(one.host_seq_lens):
        for name in ("k_cache", "v_cache"):
            assert torch.equal(getattr(one, name)[b, :, :n], getattr(two, name)[b, :, :n])
    # every sequence holds tokens again: an eager step without an append is not refused
    import entmaxkv_b200 as E
    E.sparse_attention_decode_paged(q, one, None, None, torch.zeros_like(q), 64, append_cache=False)


def test_a_capture_alone_gives_no_sequence_a_token():
    import entmaxkv_b200 as E
    cache = make("dense", [40, 40])
    k = rows(2, 2, 1, 128, seed=3)
    cache.release([1])
    for call in (lambda: cache.append(k, k), lambda: cache.extend(k, k)):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            call()
        q = rows(2, 4, 1, 128, seed=4)
        with pytest.raises(ValueError):
            E.sparse_attention_decode_paged(q, cache, None, None, torch.zeros_like(q), 64, append_cache=False)
    graph.replay()
    assert cache.sync_lengths() == [41, 1]
    E.sparse_attention_decode_paged(q, cache, None, None, torch.zeros_like(q), 64, append_cache=False)


@pytest.mark.parametrize("layout", ["dense", "pool"])
def test_the_loop_runs_as_long_as_its_tokens_fit(layout):
    """Eight drafts a step of which one or two are accepted, counts on the device only: 60 steps would bound the lengths by
    500, the tokens fit in 160."""
    cache = make(layout, [40, 33], blocks=20, capacity=160)
    lens = [40, 33]
    buffers = cache._meta.data_ptr()
    for step in range(60):
        k = rows(2, 2, 8, 128, seed=step)
        take = [1 + step % 2, 1]
        cache.extend(k, k, counts=torch.tensor(take, dtype=torch.int32, device="cuda"))
        lens = [n + m for n, m in zip(lens, take)]
        assert all(h >= n for h, n in zip(cache.host_seq_lens, lens))
        assert torch.equal(cache.k_cache[0, :, lens[0] - 1], k[0, :, take[0] - 1])
    assert cache._meta.data_ptr() == buffers and cache.capacity == 160
    assert cache.sync_lengths() == lens and cache.device_status() == 0


@pytest.mark.parametrize("layout", ["dense", "pool"])
@pytest.mark.parametrize("counts,start,lens", [([5, 2], None, [43, 35]), ([-1, 3], None, [40, 36]), ([1, 1], [99, 3], [41, 4]),
                                               ([1, 1], [-2, 3], [1, 4])])
def test_what_is_clipped_shows_in_the_status(layout, counts, start, lens):
    cache = make(layout, [40, 33])
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k = rows(2, 2, 3, 128, seed=5)
    cache.extend(k, k, counts=i32(counts), start=i32(start))
    assert cache.device_status() == 4 and cache.sync_lengths() == lens


def captured(call):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph


@pytest.mark.parametrize("layout", ["dense", "pool"])
@pytest.mark.parametrize("what", ["extend", "tree"])
def test_buffers_of_captured_calls_are_not_replaced_unasked(layout, what):
    """An eager call that has no room raises while a graph holds the buffers; the graph's replays stay right; after
    reserve() the cache grows by itself again."""
    import entmaxkv_b200 as E
    cache = make(layout, [60, 33], capacity=80)
    k = rows(2, 2, 4, 128, seed=6)
    counts = torch.tensor([2, 1], dtype=torch.int32, device="cuda")
    q, mask = rows(2, 4, 4, 128, seed=7), torch.ones(4, 4, dtype=torch.bool, device="cuda").tril()
    out = torch.zeros_like(q)
    tree = lambda to: E.tree_attention_decode(q, cache, k, k, mask, to)  # noqa: E731
    tree(out)
    graph = captured((lambda: cache.extend(k, k, counts=counts)) if what == "extend" else lambda: tree(out))
    buffers = cache._meta.data_ptr()
    many = rows(2, 2, 30, 128, seed=8)
    with pytest.raises(RuntimeError, match="captured calls hold"):
        cache.extend(many, many)
    assert cache._meta.data_ptr() == buffers and cache.seq_lens.tolist() == [60, 33]
    graph.replay()
    if what == "extend":
        assert cache.sync_lengths() == [62, 34]
        assert torch.equal(cache.k_cache[0, :, 60:62], k[0, :, :2]) and torch.equal(cache.k_cache[1, :, 33], k[1, :, 0])
    else:
        want = torch.zeros_like(out)
        tree(want)
        assert (out == want).float().mean() > 0.99
    cache.reserve(100)                               # whoever asks for it knows that the graph is gone
    cache.extend(many, many)
    many = rows(2, 2, 4000, 128, seed=9)
    if layout == "dense":
        cache.extend(many, many)
    assert cache.device_status() == 0


def test_a_capture_cannot_grow_the_cache():
    cache = make("dense", [60, 33], capacity=64)
    many = rows(2, 2, 30, 128, seed=8)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="reserve"):
        with torch.cuda.graph(graph):
            cache.extend(many, many)
    cache.extend(many, many)
    assert cache.sync_lengths() == [90, 63]


@pytest.mark.parametrize("layout", ["dense", "blocks", "pool"])
def test_reserve_keeps_rows_that_replays_added(layout):
    """The host counts no replays: the rows that they wrote must come along when the buffers grow."""
    import entmaxkv_b200 as E
    if layout == "blocks":
        cache = E.PagedKVCache(16, capacity=96, block_table=True, block_order="random")
        cache.initialize(rows(2, 2, 40, 128, seed=1), rows(2, 2, 40, 128, seed=2), seq_lens=[40, 33])
    else:
        cache = make(layout, [40, 33], capacity=96)
    k, counts = rows(2, 2, 4, 128, seed=6), torch.tensor([4, 3], dtype=torch.int32, device="cuda")
    graph = captured(lambda: cache.extend(k, k, counts=counts))
    for _ in range(10):
        graph.replay()
    cache.reserve(500)
    assert cache.sync_lengths() == [80, 63] and cache.capacity >= 500
    for b, (n0, n) in enumerate(((40, 4), (33, 3))):
        for view in (cache.k_cache, cache.v_cache):
            assert torch.equal(view[b, :, n0:n0 + 10 * n], k[b, :, :n].repeat(1, 10, 1))
    assert cache.device_status() == 0


def test_lists_of_lengths_and_releases_do_not_go_into_captures():
    cache = make("dense", [40, 33])
    k = rows(2, 2, 4, 128, seed=6)
    for call, error in ((lambda: cache.extend(k, k, counts=[1, 2]), ValueError),
                        (lambda: cache.extend(k, k, start=[1, 2]), ValueError), (lambda: cache.release([0]), RuntimeError)):
        torch.cuda.synchronize()
        with pytest.raises(error, match="captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    assert cache.seq_lens.tolist() == [40, 33] and cache.host_seq_lens == [40, 33] and not cache._may_be_empty


def test_a_maximum_below_what_is_known_is_refused():
    cache = make("dense", [40, 33])
    k = rows(2, 2, 4, 128, seed=6)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for change in (dict(counts=[1, 2], max_seq_len=40), dict(max_seq_len=43), dict(counts=i32(0, 0), max_seq_len=39),
                   dict(counts=[4, 0], start=[40, 0], max_seq_len=43)):
        with pytest.raises(ValueError, match="max_seq_len"):
            cache.extend(k, k, **change)
    assert cache.host_seq_lens == [40, 33] and cache.seq_lens.tolist() == [40, 33]
    cache.extend(k, k, counts=[1, 2], max_seq_len=41)
    cache.extend(k, k, counts=i32(1, 0), start=i32(5, 6), max_seq_len=6)
    assert cache.sync_lengths() == [6, 6]


def test_a_rewind_among_rows_that_replays_added():
    """The host counts one call of a captured extend, three replays wrote: a start between the two is no mistake, one
    beyond the tokens is."""
    cache = make("dense", [40, 33], capacity=96)
    k = rows(2, 2, 4, 128, seed=6)
    graph = captured(lambda: cache.extend(k, k))
    for _ in range(3):
        graph.replay()
    with pytest.raises(ValueError, match="beyond"):
        cache.extend(k, k, start=[53, 40])
    for _ in range(3):
        graph.replay()                                                   # 64 and 57 tokens, 52 and 45 of them known
    cache.extend(k, k, start=[61, 50], counts=[2, 0])
    assert cache.host_seq_lens == [63, 50] == cache.seq_lens.tolist() and cache.device_status() == 0
    assert torch.equal(cache.k_cache[0, :, 61:63], k[0, :, :2])
