"""Rows written into the cache, block tables from lengths, and the shared pool (run on a B200: ``-m gpu``)."""

import random

import pytest
import torch

pytestmark = pytest.mark.gpu

from tests import _spec_oracle as O

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def rows(*shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def same_cache(cache, k, v, lens, page):
    """``cache`` equals one built from scratch out of k, v [B, H, S, D] with these lengths, bit for bit."""
    import entmaxkv_b200 as E
    assert cache.seq_lens.tolist() == lens and cache.device_status() == 0
    for b, n in enumerate(lens):
        if n == 0:
            continue
        want = E.PagedKVCache(page)
        want.initialize(k[b:b + 1, :, :n].cuda(), v[b:b + 1, :, :n].cuda())
        assert torch.equal(cache.k_cache[b, :, :n], want.k_cache[0]), b
        assert torch.equal(cache.v_cache[b, :, :n], want.v_cache[0]), b
        for name in ("k_min", "k_max", "k_mean", "k_std"):
            assert torch.equal(getattr(cache, name)[b, :, :-(-n // page)], getattr(want, name)[0]), (b, name)


def make_cache(page, layout, k, v, lens, blocks=0):
    import entmaxkv_b200 as E
    kw = dict(dense={}, blocks=dict(block_table=True, block_order="random"),
              pool=dict(block_table=True, block_order="random", num_blocks=blocks))[layout]
    c = E.PagedKVCache(page, capacity=max(k.shape[2], 64), **kw)
    c.initialize(k.cuda(), v.cuda(), seq_lens=lens)
    return c


@pytest.mark.parametrize("layout", ["dense", "blocks", "pool"])
@pytest.mark.parametrize("page,dt,D", [(16, "bf16", 128), (8, "fp16", 64), (24, "fp32", 64), (1, "bf16", 64)])
def test_extend_equals_a_cache_built_at_once(layout, page, dt, D):
    B, H, dtype = 3, 2, DT[dt]
    lens = [5, 1, 2 * page]
    k, v = rows(B, H, 60, D, dtype=dtype, seed=1), rows(B, H, 60, D, dtype=dtype, seed=2)
    cache = make_cache(page, layout, k, v, lens, blocks=3 * (-(-400 // page)) + 3)
    mine_k, mine_v = k.clone(), v.clone()
    grown = torch.zeros(B, H, 400, D, dtype=dtype), torch.zeros(B, H, 400, D, dtype=dtype)
    for x, y in zip(grown, (mine_k, mine_v)):
        x[:, :, :60] = y
    for step, (T, counts, path) in enumerate([(1, None, False), (7, [7, 0, 3], False), (9, [2, 9, 4], True),
                                              (100, [100, 1, 37], False), (5, [0, 0, 0], True), (33, None, False)]):
        new = rows(B, T, 2 * H, D, dtype=dtype, seed=10 + step).transpose(1, 2)
        index = torch.stack([torch.randperm(T, generator=torch.Generator().manual_seed(b)) for b in range(B)])
        take = counts or [T] * B
        for b in range(B):
            i = index[b, :take[b]] if path else torch.arange(take[b])
            grown[0][b, :, lens[b]:lens[b] + take[b]] = new[b, :H, i]
            grown[1][b, :, lens[b]:lens[b] + take[b]] = new[b, H:, i]
        on_device = step % 2 and counts is not None
        given = torch.tensor(counts, dtype=torch.int32, device="cuda") if on_device else counts
        n = new.cuda()
        cache.extend(n[:, :H], n[:, H:], counts=given, index=index.to(torch.int32).cuda() if path else None)
        lens = [a + c for a, c in zip(lens, take)]
        assert all(h >= n for h, n in zip(cache.host_seq_lens, lens))
        assert cache.sync_lengths() == lens
        same_cache(cache, *grown, lens, page)


@pytest.mark.parametrize("layout", ["dense", "pool"])
@pytest.mark.parametrize("on_device", [False, True])
def test_rewinding(layout, on_device):
    """A smaller start drops what lies behind it, rows and statistics, with and without new rows."""
    page, lens = 16, [50, 17, 33]
    k, v = rows(3, 2, 64, 64, dtype=torch.float16, seed=3), rows(3, 2, 64, 64, dtype=torch.float16, seed=4)
    cache = make_cache(page, layout, k, v, lens, blocks=12)
    new = rows(3, 2, 6, 64, dtype=torch.float16, seed=5)
    give = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda") if on_device else x  # noqa: E731
    start, counts = [20, 17, 0], [6, 0, 2]
    cache.extend(new.cuda(), new.cuda(), counts=give(counts), start=give(start), max_seq_len=60)
    lens = [26, 17, 2]
    for b in range(3):
        k[b, :, start[b]:lens[b]] = new[b, :, :counts[b]]
        v[b, :, start[b]:lens[b]] = new[b, :, :counts[b]]
    same_cache(cache, k, v, lens, page)
    cache.extend(new[:, :, :0].cuda(), new[:, :, :0].cuda(), start=give([9, 16, 2]))      # a rewind alone
    lens = [9, 16, 2]
    same_cache(cache, k, v, lens, page)
    assert cache.sync_lengths() == lens
    if layout == "pool":
        held = sorted(int(x) for b, n in enumerate(lens) for x in cache._table[b, :-(-n // page)])
        free = sorted(cache._free[len(held):].tolist())
        assert sorted(held + free) == list(range(12)), "every block is held once or free"


def test_extend_values_out_of_range_are_clipped_and_reported():
    k = rows(2, 1, 32, 64, dtype=torch.float16, seed=6)
    new = rows(2, 1, 3, 64, dtype=torch.float16, seed=7).cuda()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for change in (dict(counts=i32(5, 2)), dict(counts=i32(-1, 3)), dict(start=i32(99, 3)),
                   dict(index=i32(0, 1, 2, 7, -3, 0).view(2, 3))):
        cache = make_cache(16, "dense", k, k, [32, 20])
        cache.extend(new, new, **change)
        assert cache.device_status() == 4
        assert all(0 <= n <= 35 for n in cache.sync_lengths())


def test_what_is_not_written_takes_no_block():
    """Counts beyond the rows given, and pages beyond the table: the pool's top stays where the lengths say, so no block is
    ever held twice."""
    import entmaxkv_b200 as E
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k = rows(3, 1, 8, 64, dtype=torch.float16, seed=40)
    cache = make_cache(4, "pool", k, k, [4, 4, 8], blocks=30)
    big = torch.zeros(3, 1, 40, 64, dtype=torch.float16)
    big[:, :, :8] = k
    lens = [4, 4, 8]
    for step, (given, take) in enumerate([([90, 2, 1], [2, 2, 1]), ([2, 70, -5], [2, 2, 0]), ([1, 2, 2], [1, 2, 2]),
                                          ([2, 2, 2], [2, 2, 2])]):
        new = rows(3, 1, 2, 64, dtype=torch.float16, seed=41 + step)
        cache.extend(new.cuda(), new.cuda(), counts=i32(*given))
        for b in range(3):
            big[b, :, lens[b]:lens[b] + take[b]] = new[b, :, :take[b]]
        lens = [n + m for n, m in zip(lens, take)]
        assert cache.sync_lengths() == lens
        held = [int(x) for b, n in enumerate(lens) for x in cache._table[b, :-(-n // 4)]]
        assert len(set(held)) == len(held) and min(held) >= 0
        for b, n in enumerate(lens):
            assert torch.equal(cache.k_cache[b, :, :n].cpu(), big[b, :, :n])
    # a table too narrow for one sequence: the next one's pages follow without a gap
    table, status = torch.full((2, 2), -1, dtype=torch.int32, device="cuda"), i32(0)
    slots = torch.zeros(20, dtype=torch.int64, device="cuda")
    E.plan_block_tables(i32(0, 0), i32(13, 6), table, i32(5, 6, 7, 8, 9), 4, slots=slots, status=status)
    assert table.tolist() == [[5, 6], [7, 8]] and int(status) == 2
    assert slots.tolist() == [20, 21, 22, 23, 24, 25, 26, 27, -1, -1, -1, -1, -1, 28, 29, 30, 31, 32, 33, -1]


def test_extend_refusals():
    import entmaxkv_b200 as E
    k = rows(2, 2, 32, 64, dtype=torch.float16, seed=8)
    cache = make_cache(16, "dense", k, k, [32, 20])
    new = rows(2, 2, 3, 64, dtype=torch.float16, seed=9).cuda()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    bad = [dict(k_new=new[:1], v_new=new[:1]), dict(v_new=new[:, :, :2]), dict(k_new=new.float()), dict(v_new=new.cpu()),
           dict(counts=[1]), dict(counts=[4, 0]), dict(counts=[-1, 0]), dict(counts=i32(1, 1).long()),
           dict(counts=i32(1, 1, 1)), dict(start=[33, 0]), dict(start=[0, -1]), dict(index=i32(0, 1, 2)),
           dict(index=i32(0, 1, 2, 0, 1, 2).view(2, 3).long()), dict(max_seq_len=-1)]
    for change in bad:
        with pytest.raises(ValueError):
            cache.extend(**{**dict(k_new=new, v_new=new), **change})
    with pytest.raises(RuntimeError):
        E.PagedKVCache(16).extend(new, new)
    assert cache.seq_lens.tolist() == [32, 20] and cache.host_seq_lens == [32, 20]


def test_extend_replays_from_a_graph():
    k = rows(2, 2, 40, 128, dtype=torch.bfloat16, seed=10)
    v = rows(2, 2, 40, 128, dtype=torch.bfloat16, seed=11)
    for layout in ("dense", "pool"):
        cache = make_cache(16, layout, k, v, [40, 7], blocks=40)
        cache.reserve(400)
        new = torch.zeros(2, 2, 4, 128, dtype=torch.bfloat16, device="cuda")
        counts = torch.zeros(2, dtype=torch.int32, device="cuda")
        graph = torch.cuda.CUDAGraph()
        cache.extend(new, new, counts=counts)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            cache.extend(new, new, counts=counts)
        big_k, big_v, lens = torch.zeros(2, 2, 100, 128).bfloat16(), torch.zeros(2, 2, 100, 128).bfloat16(), [40, 7]
        big_k[:, :, :40], big_v[:, :, :40] = k, v
        for step, take in enumerate([[4, 1], [0, 4], [3, 3], [4, 4]]):
            x = rows(2, 2, 4, 128, dtype=torch.bfloat16, seed=20 + step)
            new.copy_(x)
            counts.copy_(torch.tensor(take))
            graph.replay()
            for b in range(2):
                big_k[b, :, lens[b]:lens[b] + take[b]] = x[b, :, :take[b]]
                big_v[b, :, lens[b]:lens[b] + take[b]] = x[b, :, :take[b]]
            lens = [a + c for a, c in zip(lens, take)]
        cache.sync_lengths()
        same_cache(cache, big_k, big_v, lens, 16)


# ---- block tables --------------------------------------------------------------------------------------------------

def random_plan(rng, B, page, n_free=None):
    seq = [rng.choice([0, 1, page, rng.randrange(0, 6 * page)]) for _ in range(B)]
    new = [rng.choice([0, 1, page, rng.randrange(0, 5 * page)]) for _ in range(B)]
    held = sum(-(-s // page) for s in seq)
    need = sum(-(-(s + m) // page) for s, m in zip(seq, new))
    n = max(held, need - rng.choice([0, 0, 3])) if n_free is None else n_free
    order = list(range(n))
    rng.shuffle(order)
    width = max([-(-(s + m) // page) for s, m in zip(seq, new)] + [1])
    table, at = [[-7] * width for _ in range(B)], 0
    for b in range(B):
        for p in range(-(-seq[b] // page)):
            table[b][p] = order[at]
            at += 1
    return seq, new, table, order


@pytest.mark.parametrize("B,page", [(1, 16), (2, 1), (33, 16), (512, 8), (513, 24), (3000, 16)])
def test_plan_and_release_against_loops(B, page):
    import entmaxkv_b200 as E
    rng = random.Random(B * 100 + page)
    for _ in range(3):
        seq, new, table, order = random_plan(rng, B, page)
        cu = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        n_slots = sum(new) + rng.choice([0, 5]) or 1
        wide = torch.full((B, len(table[0]) + 3), 55, dtype=torch.int32, device="cuda")
        t = wide[:, :len(table[0])]                                    # rows further apart than they are long
        t.copy_(cu(table))
        slots = torch.zeros(n_slots, dtype=torch.int64, device="cuda")
        positions = torch.zeros(n_slots, dtype=torch.int32, device="cuda")
        starts = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        free = cu(order)
        ref = O.plan(seq, new, table, order, page, n_slots)
        for _ in range(2):                                             # a plan can be made twice
            got = E.plan_block_tables(cu(seq), cu(new), t, free, page, slots=slots, positions=positions,
                                      row_starts=starts, status=status)
            assert got[0].tolist() == ref[0] and got[1].tolist() == ref[1]
            assert got[2].tolist() == ref[2] and got[3].tolist() == ref[3]
        short = sum(-(-(s + m) // page) for s, m in zip(seq, new)) > len(order)
        assert int(status) == (2 if short else 0) and free.tolist() == order
        assert (wide[:, len(table[0]):] == 55).all()
        if short:
            continue
        total = [s + m for s, m in zip(seq, new)]
        keep = [rng.choice([0, n, rng.randrange(0, n + 1), n + 9]) for n in total]
        lens = cu(total)
        E.release_block_tables(lens, cu(keep), t, free, page)
        want = O.release(total, keep, ref[0], order, page)
        used = sum(-(-k // page) for k in want[2])
        assert lens.tolist() == want[2]
        for b in range(B):                 # only a sequence's pages matter
            n = -(-total[b] // page)
            assert t[b, :n].tolist() == want[0][b][:n]
        assert free.tolist()[used:] == want[1][used:]
        held = [int(x) for b in range(B) for x in want[0][b][:-(-want[2][b] // page)]]
        assert sorted(held + free.tolist()[used:]) == sorted(order), "every block is held once or free"


def test_plan_with_an_int_and_without_outputs():
    import entmaxkv_b200 as E
    seq = torch.tensor([15, 16, 0], dtype=torch.int32, device="cuda")
    table = torch.tensor([[4, -1, -1], [2, -1, -1], [-1, -1, -1]], dtype=torch.int32, device="cuda")
    free = torch.tensor([2, 4, 0, 3, 1], dtype=torch.int32, device="cuda")
    E.plan_block_tables(seq, 1, table, free, 16)
    assert table.tolist() == [[4, -1, -1], [2, 0, -1], [3, -1, -1]]
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    E.plan_block_tables(seq, 1, table, free, 16, slots=slots)
    assert slots.tolist() == [4 * 16 + 15, 0 * 16 + 0, 3 * 16, -1]
    E.release_block_tables(seq, 0, table, free, 16)
    assert seq.tolist() == [0, 0, 0] and sorted(free.tolist()) == [0, 1, 2, 3, 4]
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    starts = torch.ones(1, dtype=torch.int32, device="cuda")
    E.plan_block_tables(none, none, torch.zeros(0, 4, dtype=torch.int32, device="cuda"), free, 16, row_starts=starts)
    assert starts.tolist() == [0]


def test_plan_survives_lengths_that_make_no_sense():
    """Negative and enormous lengths on the device: nothing outside the buffers is touched, the status says so."""
    import entmaxkv_b200 as E
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    guard = torch.full((64,), 77, dtype=torch.int32, device="cuda")
    table, status = guard[16:32].view(2, 8), i32(0)
    slots = torch.zeros(6, dtype=torch.int64, device="cuda")
    E.plan_block_tables(i32(-5, 2**31 - 1), i32(3, 2**31 - 1), table, i32(0, 1, 2, 3), 4, slots=slots, status=status)
    E.release_block_tables(i32(2**31 - 1, 8), i32(-3, 4), table, i32(0, 1, 2, 3), 4, status=status)
    torch.cuda.synchronize()
    assert (guard[:16] == 77).all() and (guard[32:] == 77).all() and int(status) & 2


def test_block_table_refusals():
    import entmaxkv_b200 as E
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    good = dict(seq_lens=i32(1, 2), new_lens=i32(1, 1), block_table=i32(0, 1, 2, 3).view(2, 2), free_blocks=i32(0, 1, 2),
                page_size=16)
    E.plan_block_tables(**good)
    z64, z32 = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    bad = [dict(seq_lens=good["seq_lens"].long()), dict(seq_lens=good["seq_lens"].cpu()), dict(new_lens=i32(1)),
           dict(new_lens=-1), dict(new_lens=1.5), dict(new_lens=True), dict(block_table=i32(0, 1)),
           dict(block_table=good["block_table"].t()), dict(block_table=i32(0, 1).view(1, 2).expand(2, 2)),
           dict(free_blocks=good["free_blocks"].long()), dict(page_size=0), dict(slots=z32), dict(positions=z64),
           dict(slots=z64, positions=z32), dict(row_starts=z32[:2]), dict(status=z64)]
    for change in bad:
        with pytest.raises(ValueError):
            E.plan_block_tables(**{**good, **change})
    big = torch.zeros(16385, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        E.plan_block_tables(big, 1, big.view(-1, 1), big, 16)


def test_the_shared_pool_runs_dry_and_recovers():
    import entmaxkv_b200 as E
    k = rows(3, 2, 32, 64, dtype=torch.float16, seed=30)
    with pytest.raises(RuntimeError):
        make_cache(16, "pool", k, k, [32, 32, 32], blocks=5)
    with pytest.raises(ValueError):
        E.PagedKVCache(16, num_blocks=4)
    cache = make_cache(16, "pool", k, k, [32, 32, 20], blocks=6)
    one = rows(3, 2, 1, 64, dtype=torch.float16, seed=31)
    with pytest.raises(RuntimeError):
        cache.append(one.cuda(), one.cuda())           # two sequences need a page each
    assert cache.seq_lens.tolist() == [32, 32, 20] and cache.device_status() == 0
    cache.release([1])
    with pytest.raises(ValueError):
        E.sparse_attention_decode_paged(one.cuda(), cache, None, None, one.cuda(), 64, append_cache=False)
    cache.append(one.cuda(), one.cuda())
    lens = [33, 1, 21]
    big = torch.zeros(3, 2, 64, 64, dtype=torch.float16)
    big[:, :, :32] = k
    for b in range(3):
        big[b, :, lens[b] - 1] = one[b, :, 0]
    same_cache(cache, big, big, lens, 16)
    # through a device count the host cannot know: what has no block is dropped and reported
    cache._make_room = lambda lens: None
    more = rows(3, 2, 64, 64, dtype=torch.float16, seed=32).cuda()
    cache.extend(more, more, counts=torch.tensor([40, 0, 40], dtype=torch.int32, device="cuda"), max_seq_len=80)
    assert cache.sync_lengths()[1] == 1 and cache.device_status() & 3
    held = sum(-(-n // 16) for n in cache.host_seq_lens)
    assert held == 6


@pytest.mark.parametrize("mode", ["topk", "gaussian"])
def test_decode_steps_on_a_shared_pool_equal_the_dense_cache(mode):
    import entmaxkv_b200 as E
    from entmaxkv_b200.graph import DecodeStepGraph
    from tests import _harness as H
    B, Hq, Hkv, D, lens, P = 2, 8, 2, 128, [700, 333], 16
    inp = H.to_cuda(H.cpu_inputs(B, Hq, Hkv, D, 700, torch.bfloat16, seed=77, needle_pages=(3, 11)))
    dense, pool = (make_cache(P, layout, inp["k"], inp["v"], lens, blocks=100) for layout in ("dense", "pool"))
    g = torch.Generator().manual_seed(5)
    graph = None
    for step in range(P + 4):
        kn, vn, q = (torch.randn(B, n, 1, D, generator=g).bfloat16().cuda() for n in (Hkv, Hkv, Hq))
        outs = []
        for c in (dense, pool):
            out = torch.zeros_like(q)
            if c is pool and step >= 4:
                graph = graph or DecodeStepGraph(pool, Hq, mode, token_budget=256, alpha=1.5, niter=2)
                out = graph.step(q, kn, vn).clone()
            elif mode == "topk":
                E.sparse_attention_decode_paged(q, c, kn, vn, out, 256, alpha=1.5, niter=2)
            else:
                E.sparse_attention_decode_gaussian_aware_entmax(q, c, kn, vn, out, alpha=1.5, append_cache=True)
            outs.append(out)
        assert torch.equal(*outs), step
    assert pool.device_status() == 0
