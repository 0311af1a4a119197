"""Tree attention where scores, lengths or row counts are extreme (run on a B200: ``-m gpu``)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from tests import test_gpu_tree as G

#: B, Hq, Hkv, T, lengths, dtype: a block per row and a warp per row, all scores written out and candidate lists, and a row
#: per warp with more lists than a warp takes, on both ways of scoring
ROUTES = {
    "few_short": (1, 4, 1, 4, [300], "bf16"),
    "many_short": (1, 32, 1, 32, [300], "fp16"),
    "few_long": (1, 4, 1, 4, [9000], "bf16"),
    "many_long": (1, 32, 1, 32, [9000], "fp16"),
    "many_lists": (32, 8, 1, 4, [20000] + [1] * 31, "bf16"),
    "few_fp32": (1, 4, 1, 4, [3000], "fp32"),
    "many_fp32": (1, 32, 1, 32, [300], "fp32"),
    "many_lists_fp32": (4, 8, 1, 32, [20000, 1, 1, 1], "fp32"),
}


@pytest.mark.parametrize("where", ["first_tile", "second_tile", "draft"])
@pytest.mark.parametrize("route", ROUTES)
def test_an_infinite_score_makes_its_row_nan_on_every_route(route, where):
    """Key element 0 is +inf: rows whose query is positive there score +inf, the others -inf, and those must not notice.
    The first tile is always in the sample, the second one never."""
    B, Hq, Hkv, T, lens, dt = ROUTES[route]
    x = G.make(B, Hq, Hkv, 64, lens, T, G.DT[dt], seed=51)
    x["mask"] = torch.ones(T, T, dtype=torch.bool).tril()
    up = torch.arange(T) % 2 == 0
    x["q"][..., 0] = torch.where(up, 1.0, -1.0).to(G.DT[dt])
    place = {"first_tile": ("k", 5), "second_tile": ("k", 130), "draft": ("kd", 0)}[where]
    x[place[0]][0, 0, place[1], 0] = 3e4              # far under the threshold of the rows with a negative query
    want, want_tau = G.run(x, G.cache_of(x, lens, 16, "dense"), 1.5)
    assert torch.isfinite(want_tau).all()
    x[place[0]][0, 0, place[1], 0] = math.inf
    out, tau = G.run(x, G.cache_of(x, lens, 16, "dense"), 1.5)
    hit = torch.zeros(B, Hq, T, dtype=torch.bool)
    hit[0] = up
    assert out[hit].isnan().all() and tau[hit].isnan().all()
    assert torch.equal(out[~hit], want[~hit]) and torch.equal(tau[~hit], want_tau[~hit])


#: rows per KV head and sequences: a block per row, a warp per row
SHAPES = {"few": (1, 4, 1, 2), "many": (2, 32, 2, 16)}
PLACES = [(dt, n, shape) for dt in ("bf16", "fp16", "fp32") for n in (40, 4000, 20000) for shape in SHAPES
          if not (dt == "fp32" and n == 20000 and shape == "many")] + [("bf16", 100000, "few")]


def level_scores(dt, n, shape, alpha, score):
    """Every key and draft scores `score` (exactly: every product and sum is a small multiple of a power of two)."""
    B, Hq, Hkv, T = SHAPES[shape]
    x = G.make(B, Hq, Hkv, 64, [1] * B, T, G.DT[dt], seed=52)
    x["k"] = torch.ones(B, Hkv, n, 64, dtype=G.DT[dt])
    x["v"] = torch.ones(B, Hkv, n, 64, dtype=G.DT[dt])
    x["kd"], x["vd"] = torch.ones_like(x["kd"]), torch.ones_like(x["vd"])
    x["q"] = torch.full_like(x["q"], score / 8 / (alpha - 1))
    x["mask"] = torch.eye(T, dtype=torch.bool)
    return x


@pytest.mark.parametrize("alpha", [1 + 2.0 ** -11, 1.125, 1.5, 2.0, 3.0, 5.0])
@pytest.mark.parametrize("dt,n,shape", PLACES)
def test_weights_of_equal_scores_sum_to_one(dt, n, shape, alpha):
    """n + 1 equal scores of 8 and values of one: the output is the sum of the weights.  The solver leaves it within
    1e-6 of one; up to n / 4 additions one after another are off by 2^-24 of the sum each, then one rounding."""
    x = level_scores(dt, n, shape, alpha, 8.0)
    out, tau = G.run(x, G.cache_of(x, [n] * SHAPES[shape][0], 16, "dense"), alpha)
    tol = 1e-6 + (n / 4 + 64) * 2.0 ** -24 + torch.finfo(out.dtype).eps / 2
    assert (out.double() - 1).abs().max() <= tol
    # the threshold is rounded to fp32 once: half a step below 8 is 2^-22
    assert (tau.double() - (8 - (n + 1) ** -(alpha - 1))).abs().max() <= 2.0 ** -22 + 1e-6


@pytest.mark.parametrize("alpha", [1.5, 2.0, 2.5, 3.0])
@pytest.mark.parametrize("dt,n,shape", PLACES)
def test_many_equal_scores_just_above_the_threshold(dt, n, shape, alpha):
    """The drafted key scores about 0.875 more than n equal ones, whose weights together have what it leaves of one."""
    x = level_scores(dt, n, shape, alpha, 8.0)
    x["kd"] = x["kd"] * 1.109375                # exact in every type: 8 * 1.109375 = 8.875
    out, _ = G.run(x, G.cache_of(x, [n] * SHAPES[shape][0], 16, "dense"), alpha)
    tol = 1e-6 + (n / 4 + 64) * 2.0 ** -24 + torch.finfo(out.dtype).eps / 2
    assert (out.double() - 1).abs().max() <= tol


@pytest.mark.parametrize("n", [300, 9000])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_scores_past_what_fp32_counts(dt, shape, n):
    """Scores of 2^25 and more, where score - 1 is the score again: the largest key has all the weight, two of them half."""
    B, Hq, Hkv, T = SHAPES[shape]
    x = G.make(B, Hq, Hkv, 64, [n] * B, T, G.DT[dt], seed=53)
    x["q"] = torch.zeros_like(x["q"])
    x["q"][..., 0] = 2.0 ** 15
    x["k"][..., 0], x["kd"][..., 0] = 2.0 ** 14, 2.0 ** 14
    x["k"][:, :, 200, 0] = 1.5 * 2.0 ** 14
    group = Hq // Hkv
    one, _ = G.run(x, G.cache_of(x, [n] * B, 16, "dense"), 1.5)
    assert torch.equal(one, x["v"][:, :, 200].repeat_interleave(group, 1)[:, :, None].expand_as(one))
    x["k"][:, :, 7, 0] = 1.5 * 2.0 ** 14
    two, _ = G.run(x, G.cache_of(x, [n] * B, 16, "dense"), 1.5)
    mean = (x["v"][:, :, 200].double() + x["v"][:, :, 7].double()).repeat_interleave(group, 1)[:, :, None] / 2
    # weights of sqrt(1/2) squared, 2^-22 of each value, and the rounding
    assert ((two.double() - mean).abs() <= 2.0 ** -21 + (mean.abs() + 2.0 ** -21) * torch.finfo(two.dtype).eps / 2).all()


def test_rows_of_one_group_take_turns():
    """2048 rows of one KV head over 524,288 tokens: their scratch would be 8.6 GB, so the rows take turns.  The same as
    half of the query heads at a time, which fit; a tree that ends inside the second turn leaves the rest as it was."""
    import entmaxkv_b200 as E
    S, T, Hq, D = 524288, 256, 8, 64
    g = torch.Generator(device="cuda").manual_seed(54)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    q, kd, vd = r(1, Hq, T, D), r(1, 1, T, D), r(1, 1, T, D)
    cache = E.PagedKVCache(16, capacity=S)
    cache.initialize(r(1, 1, S, D), r(1, 1, S, D))
    mask = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
    live = torch.tensor([201], dtype=torch.int32, device="cuda")
    outs = []
    for heads in (slice(0, 8), slice(0, 4), slice(4, 8)):
        out, tau = torch.full_like(q[:, heads], 7.0), torch.full(q[:, heads].shape[:3], 7.0, device="cuda")
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        E.tree_attention_decode(q[:, heads], cache, kd, vd, mask, out, draft_lens=live, taus_out=tau)
        assert torch.cuda.max_memory_allocated() - before <= (6 << 30) + (1 << 20)
        outs.append((out, tau))
    torch.cuda.synchronize()
    assert cache.device_status() == 0
    whole, half = outs[0], [torch.cat(x, dim=1) for x in zip(*outs[1:])]
    assert (whole[0][:, :, 201:] == 7).all() and (whole[1][:, :, 201:] == 7).all()
    # the pieces of the tile sequence differ, and with them the order of the sums: one bf16 step, and rarely that
    assert (whole[0].float() - half[0].float()).abs().max() <= 2 * 2.0 ** -8 * half[0][:, :, :201].float().abs().max()
    assert (whole[0] == half[0]).float().mean() > 0.99
    assert (whole[1] - half[1]).abs().max() <= 1e-5


@pytest.mark.parametrize("n", [300, 9000])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_a_page_without_a_block_counts_as_zeros_and_is_reported(dt, n):
    """Table entries outside the pool, which a caller of the C entry point may hand in: the copies and the loads check them."""
    x = G.make(1, 4, 2, 64, [n], 3, G.DT[dt], seed=55)
    cache = G.cache_of(x, [n], 16, "blocks")
    for page, block in ((2, -1), (7, 10 ** 6), (n // 16, 2 ** 31 - 1)):
        cache._table[0, page] = block
        for t in (x["k"], x["v"]):
            t[:, :, 16 * page:16 * page + 16] = 0
    want = G.run(x, G.cache_of(x, [n], 16, "blocks"), 1.5)
    import entmaxkv_b200 as E
    out, tau = torch.zeros_like(x["q"]).cuda(), torch.zeros(x["q"].shape[:3], device="cuda")
    E.tree_attention_decode(x["q"].cuda(), cache, x["kd"].cuda(), x["vd"].cuda(), x["mask"].cuda(), out, taus_out=tau)
    assert torch.equal(out.cpu(), want[0]) and torch.equal(tau.cpu(), want[1])
    assert cache.device_status() == 1
