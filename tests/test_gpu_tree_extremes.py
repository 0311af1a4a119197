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
