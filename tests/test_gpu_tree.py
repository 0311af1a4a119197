"""Entmax attention of a tree of drafted tokens over the cache (run on a B200: ``-m gpu``), against 64-bit loops."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from tests import _spec_oracle as O

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def random_tree(B, T, g):
    """Every token sees itself and what its parent sees; parents are random earlier tokens or the root."""
    mask = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for t in range(T):
            p = int(torch.randint(-1, t, (1,), generator=g)) if t else -1
            if p >= 0:
                mask[b, t] = mask[b, p]
            mask[b, t, t] = True
    return mask


def make(B, Hq, Hkv, D, lens, T, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    S = max(lens)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(k=r(B, Hkv, S, D).to(dtype), v=r(B, Hkv, S, D).to(dtype), q=(scale * r(B, Hq, T, D)).to(dtype),
                kd=r(B, Hkv, T, D).to(dtype), vd=r(B, Hkv, T, D).to(dtype), mask=random_tree(B, T, g))


def cache_of(x, lens, page, layout):
    import entmaxkv_b200 as E
    kw = dict(dense={}, blocks=dict(block_table=True, block_order="random"),
              pool=dict(block_table=True, block_order="random", num_blocks=sum(-(-n // page) for n in lens) + 3))[layout]
    c = E.PagedKVCache(page, **kw)
    c.initialize(x["k"].cuda(), x["v"].cuda(), seq_lens=lens)
    return c


def run(x, cache, alpha, draft_lens=None, fill=7.0):
    import entmaxkv_b200 as E
    out = torch.full(x["q"].shape, fill, dtype=x["q"].dtype, device="cuda")
    tau = torch.full(x["q"].shape[:3], fill, dtype=torch.float32, device="cuda")
    live = None if draft_lens is None else torch.tensor(draft_lens, dtype=torch.int32, device="cuda")
    got = E.tree_attention_decode(x["q"].cuda(), cache, x["kd"].cuda(), x["vd"].cuda(), x["mask"].cuda(), out,
                                  draft_lens=live, alpha=alpha, taus_out=tau)
    assert got is out
    torch.cuda.synchronize()
    assert cache.device_status() == 0
    return out.cpu(), tau.cpu()


def check(x, lens, out, tau, alpha, draft_lens=None, fill=7.0):
    out0, tau0 = torch.full(x["q"].shape, fill), torch.full(x["q"].shape[:3], fill)
    ref, ref_tau, tol, tau_tol = O.tree_attention(x["q"], x["k"], x["v"], lens, x["kd"], x["vd"], x["mask"], draft_lens,
                                                  alpha, out0, tau0)
    half_step = torch.finfo(out.dtype).eps / 2
    tol = tol * (1 + half_step) + half_step * ref.abs() + torch.finfo(out.dtype).tiny
    bad = ~((out.double() - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} outputs off, worst {((out.double() - ref).abs() / tol).max()} of the bound"
    fine = torch.isfinite(ref_tau)
    assert torch.equal(tau.isinf(), ~fine)
    bad = ~((tau.double() - ref_tau).abs() <= tau_tol) & fine
    assert not bad.any(), f"{int(bad.sum())} thresholds off"


CASES = [
    # B, Hq, Hkv, D, lengths, T, page, dtype, alpha, layout, draft_lens
    (1, 2, 2, 64, [1], 1, 16, "fp16", 1.5, "dense", None),
    (1, 4, 1, 128, [2], 3, 16, "bf16", 1.5, "dense", None),
    (2, 4, 2, 64, [127, 128], 5, 16, "bf16", 2.0, "blocks", [5, 2]),
    (1, 8, 1, 128, [129], 4, 8, "bf16", 1.5, "pool", None),
    (3, 8, 2, 128, [700, 1, 513], 8, 16, "bf16", 1.5, "pool", [8, 3, 0]),
    (1, 4, 4, 128, [1500], 7, 24, "fp16", 1.5, "blocks", None),
    (1, 3, 3, 64, [2049], 2, 16, "bf16", 4 / 3, "dense", None),
    (1, 2, 1, 128, [300], 6, 16, "bf16", 3.0, "dense", None),
    (2, 4, 2, 128, [1000, 999], 6, 16, "fp32", 1.5, "dense", [6, 1]),
    (1, 2, 2, 64, [260], 3, 16, "fp32", 2.0, "pool", None),
    (1, 8, 1, 64, [1100], 17, 16, "fp16", 1.5, "dense", [16]),      # 136 rows per KV head: more than one tile of rows
    (1, 16, 2, 128, [900], 33, 16, "bf16", 2.0, "pool", None),      # 264 rows per KV head
    (1, 1, 1, 128, [400], 70, 16, "bf16", 1.5, "dense", None),
    (70, 1, 1, 64, [1 + 7 * i % 200 for i in range(70)], 2, 16, "fp16", 1.5, "dense", None),
]


# long enough for the sample and the candidate lists; row counts on both sides of a copy, a tile and a block of rows;
# page sizes that are no multiple of eight, or do not divide a tile
LONG = [
    (1, 1, 1, 64, [9001], 1, 16, "bf16", 1.5, "dense", None),
    (2, 4, 2, 128, [12289, 1], 9, 16, "bf16", 1.5, "pool", [9, 4]),
    (1, 16, 1, 64, [8400], 2, 12, "fp16", 1.5, "pool", None),
    (1, 8, 1, 128, [10007], 5, 1, "bf16", 2.0, "blocks", None),
    (1, 5, 1, 128, [9500], 13, 200, "fp16", 1.5, "blocks", None),
    (3, 4, 1, 64, [8193, 130, 20000], 20, 24, "bf16", 1.5, "pool", [20, 0, 11]),
    (1, 8, 1, 64, [8300], 33, 16, "fp16", 2.0, "dense", None),      # 264 rows: two blocks of rows
    (1, 4, 1, 128, [9100], 40, 16, "bf16", 1.5, "dense", None),     # 160 rows: two tiles of rows
    (1, 2, 1, 64, [9000], 3, 16, "bf16", 4 / 3, "dense", None),
    (1, 2, 1, 64, [9000], 3, 16, "fp16", 2.5, "pool", None),
    (2, 32, 32, 64, [2600, 2500], 1, 16, "fp16", 1.5, "dense", None),   # short sequences, many heads
    (40, 2, 2, 64, [2000 + 31 * i for i in range(40)], 2, 16, "bf16", 1.5, "dense", None),
]


@pytest.mark.parametrize("case", LONG, ids=[f"long{i}" for i in range(len(LONG))])
def test_long_sequences_against_64_bits(case):
    test_tree_attention_against_64_bits(case)


def test_long_flat_scores():
    """Every key a candidate of every row: the lists are full, and one block works on a row's lists in memory."""
    for alpha, seed in ((1.5, 31), (2.0, 32)):
        lens = [9100]
        x = make(1, 4, 1, 64, lens, 2, torch.bfloat16, seed=seed, scale=1e-3)
        out, tau = run(x, cache_of(x, lens, 16, "pool"), alpha)
        check(x, lens, out, tau, alpha)


def test_long_sequences_with_what_must_not_matter_and_what_must_show():
    lens, T = [9000, 8700], 4
    x = make(2, 4, 1, 64, lens, T, torch.float16, seed=33)
    want = run(x, cache_of(x, lens, 16, "dense"), 1.5)
    for _ in range(3):
        got = run(x, cache_of(x, lens, 16, "pool"), 1.5)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    y = {n: t.clone() for n, t in x.items()}
    y["k"][1, :, 8700:], y["v"][1, :, 8700:] = math.nan, math.nan
    got = run(y, cache_of(y, lens, 16, "dense"), 1.5)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    y["k"][0, 0, 5000, 3] = math.nan
    got = run(y, cache_of(y, lens, 16, "dense"), 1.5)
    assert got[0][0].isnan().all() and torch.equal(got[0][1], want[0][1])


def test_many_rows_share_the_scratch_in_turns():
    """More rows than the scratch holds at a time: the same bits as sequence by sequence."""
    import entmaxkv_b200 as E
    B, Hq, Hkv, D, S, T = 2, 64, 8, 64, 131072, 56
    g = torch.Generator(device="cuda").manual_seed(34)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    k, v, q, kd, vd = r(B, Hkv, S, D), r(B, Hkv, S, D), r(B, Hq, T, D), r(B, Hkv, T, D), r(B, Hkv, T, D)
    mask = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
    outs = []
    for rows in (slice(0, 2), slice(0, 1), slice(1, 2)):
        c = E.PagedKVCache(16, capacity=S)
        c.initialize(k[rows], v[rows])
        out = torch.zeros_like(q[rows])
        E.tree_attention_decode(q[rows], c, kd[rows], vd[rows], mask, out)
        outs.append(out)
    # which scores a launch samples, and how it cuts the tiles, is another in each case: equal up to the summation order
    both, each = outs[0].float(), torch.cat(outs[1:]).float()
    assert (both - each).abs().max() <= 2 * 2.0 ** -8 * each.abs().max()
    assert (both == each).float().mean() > 0.99


@pytest.mark.parametrize("case", CASES, ids=[f"case{i}" for i in range(len(CASES))])
def test_tree_attention_against_64_bits(case):
    B, Hq, Hkv, D, lens, T, page, dt, alpha, layout, drafts = case
    x = make(B, Hq, Hkv, D, lens, T, DT[dt], seed=900 + sum(lens) + T)
    out, tau = run(x, cache_of(x, lens, page, layout), alpha, drafts)
    check(x, lens, out, tau, alpha, drafts)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("alpha", [1.5, 2.0])
def test_flat_scores_give_every_key_a_weight(dt, alpha):
    """Small queries: the support is the whole cache, more than the finish kernel keeps on chip."""
    lens = [5003]
    x = make(1, 4, 2, 64, lens, 3, DT[dt], seed=11, scale=1e-3)
    out, tau = run(x, cache_of(x, lens, 16, "pool"), alpha)
    check(x, lens, out, tau, alpha)


def test_equal_scores_share_the_weight():
    """All keys equal: n equal scores, tau = z - n^-(alpha-1), the mean of the values."""
    lens = [4000]
    x = make(1, 2, 1, 128, lens, 2, torch.bfloat16, seed=12)
    x["k"][:] = x["k"][:, :, :1]
    x["kd"][:] = x["k"][:, :, :1]
    out, tau = run(x, cache_of(x, lens, 16, "dense"), 1.5)
    check(x, lens, out, tau, 1.5)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_masked_places_do_not_matter(dt):
    """NaN and infinities in drafted rows that nobody sees, and behind a sequence's end, change no bit."""
    lens, T = [200, 77], 6
    x = make(2, 4, 2, 64, lens, T, DT[dt], seed=13)
    x["mask"] = torch.tril(torch.ones(T, T, dtype=torch.bool))
    x["mask"][:, 2] = False
    want = run(x, cache_of(x, lens, 16, "dense"), 1.5, [5, 6])
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(DT[dt]).min):
        y = {n: t.clone() for n, t in x.items()}
        y["kd"][:, :, 2], y["vd"][:, :, 2] = bad, bad
        y["kd"][0, :, 5], y["vd"][0, :, 5], y["q"][0, :, 5] = bad, bad, bad
        y["k"][1, :, 77:], y["v"][1, :, 77:] = bad, bad
        got = run(y, cache_of(y, lens, 16, "dense"), 1.5, [5, 6])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_row_that_sees_nothing_and_a_sequence_without_tokens():
    """An empty mask row over an emptied sequence: zeros and tau = +inf; the other rows see their drafts alone."""
    x = make(2, 4, 2, 128, [40, 40], 4, torch.bfloat16, seed=14)
    x["mask"][:, 2] = False
    for layout in ("dense", "pool"):
        c = cache_of(x, [40, 40], 16, layout)
        c.release([0])
        out, tau = run(x, c, 1.5)
        assert (out[0, :, 2] == 0).all() and torch.isposinf(tau[0, :, 2]).all()
        check(x, [0, 40], out, tau, 1.5)


def test_a_nan_or_infinite_score_shows():
    x = make(1, 2, 1, 64, [50], 3, torch.bfloat16, seed=15)
    x["mask"] = torch.eye(3, dtype=torch.bool)
    want, _ = run(x, cache_of(x, [50], 16, "dense"), 1.5)
    x["kd"][0, 0, 1, 5] = math.nan
    out, tau = run(x, cache_of(x, [50], 16, "dense"), 1.5)
    assert out[:, :, 1].isnan().all() and tau[:, :, 1].isnan().all()
    assert torch.equal(out[:, :, [0, 2]], want[:, :, [0, 2]])
    x["kd"][0, 0, 1, 5] = 0
    x["k"][0, 0, 33, 0] = math.nan
    out, tau = run(x, cache_of(x, [50], 16, "dense"), 1.5)
    assert out.isnan().all() and tau.isnan().all()


def test_strided_inputs_outputs_and_one_mask_for_all():
    import entmaxkv_b200 as E
    B, Hq, Hkv, D, T, lens = 2, 8, 2, 64, 5, [333, 90]
    x = make(B, Hq, Hkv, D, lens, T, torch.float16, seed=16)
    x["mask"] = torch.tril(torch.ones(T, T, dtype=torch.bool))
    cache = cache_of(x, lens, 16, "dense")
    want, _ = run(x, cache, 1.5)
    # rows of a fused projection; the output goes into a [B, T, H, D] buffer; a misaligned query is copied
    fused = torch.cat([x["q"], x["kd"], x["vd"]], dim=1).transpose(1, 2).contiguous().cuda()
    q, kd, vd = (t.transpose(1, 2) for t in fused.split([Hq, Hkv, Hkv], dim=2))
    shifted = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape).copy_(q)
    wide = torch.zeros(T + 3, T + 5, dtype=torch.bool, device="cuda")
    wide[:T, :T] = x["mask"].cuda()
    for query in (q, shifted):
        out = torch.zeros(B, T, Hq, D, dtype=q.dtype, device="cuda").transpose(1, 2)
        E.tree_attention_decode(query, cache, kd, vd, wide[:T, :T], out)
        assert torch.equal(out.cpu(), want)


def test_layouts_give_the_same_bits_and_runs_repeat():
    lens = [900, 2500, 64]
    x = make(3, 8, 2, 128, lens, 6, torch.bfloat16, seed=17)
    dense = cache_of(x, lens, 16, "dense")
    want = run(x, dense, 1.5)
    for _ in range(3):
        got = run(x, dense, 1.5)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for layout in ("blocks", "pool"):
        got = run(x, cache_of(x, lens, 16, layout), 1.5)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("lens", [[600, 300], [9000, 8500]])
def test_two_graphs_on_one_cache_and_a_growing_sequence(lens):
    """Captured calls keep their scratch to themselves and follow the lengths on the device."""
    import entmaxkv_b200 as E
    x = make(2, 4, 2, 128, lens, 4, torch.bfloat16, seed=18)
    y = make(2, 4, 2, 128, lens, 9, torch.bfloat16, seed=19)
    cache = cache_of(x, lens, 16, "dense")
    graphs = []
    for z in (x, y):
        d = {n: z[n].cuda() for n in ("q", "kd", "vd", "mask")}
        out = torch.zeros_like(d["q"])
        call = lambda d=d, out=out: E.tree_attention_decode(d["q"], cache, d["kd"], d["vd"], d["mask"], out)  # noqa: E731
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append((graph, out, d))
    for step in range(3):
        kv = torch.randn(2, 2, 1, 128, generator=torch.Generator().manual_seed(step)).to(torch.bfloat16).cuda()
        cache.append(kv, kv)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s, (graph, _, _) in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        for _, out, d in graphs:
            want = torch.zeros_like(out)
            E.tree_attention_decode(d["q"], cache, d["kd"], d["vd"], d["mask"], want)
            # the captured call is sized by the capacity: it may take the keys in another order
            assert (out.float() - want.float()).abs().max() <= 2 * 2.0 ** -8 * want.float().abs().max()
            assert (out == want).float().mean() > 0.99


def test_refusals():
    import entmaxkv_b200 as E
    x = {n: t.cuda() for n, t in make(2, 4, 2, 64, [50, 50], 3, torch.float16, seed=20).items()}
    cache = cache_of({n: t.cpu() for n, t in x.items()}, [50, 50], 16, "dense")
    out = torch.zeros_like(x["q"])
    good = dict(q=x["q"], kv_cache=cache, k_draft=x["kd"], v_draft=x["vd"], tree_mask=x["mask"], out=out)
    E.tree_attention_decode(**good)
    bad = [dict(alpha=1.0), dict(alpha=math.nan), dict(alpha=math.inf), dict(out=x["q"]), dict(q=x["q"][:, :3]), dict(q=x["q"].float()), dict(q=x["q"].cpu()),
           dict(k_draft=x["kd"][:, :, :2]), dict(v_draft=x["vd"].float()), dict(tree_mask=x["mask"].int()),
           dict(tree_mask=x["mask"][:1]), dict(tree_mask=x["mask"].transpose(-1, -2)), dict(out=out[:, :, :2]),
           dict(out=out.float()), dict(out=out[:, :1].expand_as(out)),
           dict(draft_lens=torch.ones(2, dtype=torch.int64, device="cuda")),
           dict(draft_lens=torch.ones(3, dtype=torch.int32, device="cuda")),
           dict(taus_out=torch.zeros(2, 4, 3, dtype=torch.float16, device="cuda")),
           dict(taus_out=torch.zeros(2, 3, 4, device="cuda").transpose(1, 2))]
    for change in bad:
        with pytest.raises(ValueError):
            E.tree_attention_decode(**{**good, **change})
    with pytest.raises(RuntimeError):
        E.tree_attention_decode(**{**good, "kv_cache": E.PagedKVCache(16)})
    z = torch.zeros(2, 4, 300, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        E.tree_attention_decode(z, cache, z[:, :2], z[:, :2], torch.ones(300, 300, dtype=torch.bool, device="cuda"), z)
    empty = torch.zeros(2, 4, 0, 64, dtype=torch.float16, device="cuda")
    nothing = torch.zeros(0, 0, dtype=torch.bool, device="cuda")
    assert E.tree_attention_decode(empty, cache, empty[:, :2], empty[:, :2], nothing, empty) is empty
