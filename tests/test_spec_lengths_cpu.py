"""Host side of the speculative step, without a GPU: sizes of the scratch, and lengths that the host only bounds."""

import ctypes as C

import pytest
import torch

from tests.test_spec_cpu import desc, fake, lib  # noqa: F401  (lib: a fixture)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("table", [False, True])
@pytest.mark.parametrize("q_heads,tokens,most", [(8, 256, 1 << 20), (64, 256, 131072), (32, 200, 100003), (512, 256, 1 << 16),
                                                 (1, 1, 1 << 24), (16, 256, (1 << 22) + 5)])
def test_scratch_of_one_group_is_bounded(lib, dtype, table, q_heads, tokens, most):  # noqa: F811
    """More rows of a single KV head than 6 GiB hold at 8 bytes per row and token: they take turns."""
    buf, p = fake()
    cap = (most + 15) // 16 * 16
    d = desc(p, batch=1, kv_heads=1, capacity=cap, page_capacity=cap // 16, kv_stride_h=64 * cap, kv_stride_b=64 * cap,
             dtype=dtype)
    if table:
        d.block_table, d.bt_stride, d.kv_stride_block, d.num_blocks = p, cap // 16, 64 * 16, cap // 16
    size = lib.ekv_tree_workspace_bytes(C.byref(d), q_heads, tokens, most)
    assert 0 < size <= (6 << 30) + 256
    if q_heads * tokens * most * 8 < 5 << 30:
        assert size >= q_heads * tokens * most * 4          # what fits is not cut: a score takes four bytes at least


def host_cache(lens, capacity=64, page=16, **kw):
    """A cache whose buffers lie on the CPU: what the host decides before a launch can be tried without a GPU."""
    import entmaxkv_b200 as E
    c = E.PagedKVCache(page, **kw)
    c._allocate(len(lens), 2, 64, capacity, torch.bfloat16, "cpu")
    c._host_lens, c.seq_lens = list(lens), torch.tensor(lens, dtype=torch.int32)
    c._ctl = torch.zeros(16 + len(lens), dtype=torch.int32)
    return c


def test_selection_helpers_refuse_sequences_without_tokens():
    cache = host_cache([20, 0])
    cache._may_be_empty = True
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no token"):
        cache.estimate_page_criticality(q, exclude_last_page=True)
    with pytest.raises(ValueError, match="no token"):
        cache.select_gaussian_aware(q)


@pytest.mark.parametrize("layout", ["dense", "pool"])
@pytest.mark.parametrize("unseen", ["counts on the device", "replays"])
def test_a_bound_that_leaves_no_room_is_made_exact_first(layout, unseen, monkeypatch):
    """Every call may add eight tokens and adds one: neither is the cache copied into a larger one, nor does the pool seem
    used up, until the tokens are there."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    kw = dict(block_table=True, num_blocks=8) if layout == "pool" else {}
    cache = host_cache([20, 3], capacity=64, **kw)
    cache._grows_in_graphs = unseen == "replays"
    grown = []
    cache.reserve = grown.append
    for step in range(30):
        cache._lens_exact = unseen == "replays"
        cache._host_lens = cache._room_for(lambda lens: [n + 8 for n in lens])
        cache.seq_lens += 1
        assert all(h >= n for h, n in zip(cache.host_seq_lens, cache.seq_lens.tolist())) and not grown, step
    cache.seq_lens += 30
    cache._lens_exact = False
    if layout == "pool":
        with pytest.raises(RuntimeError, match="may not suffice"):
            cache._room_for(lambda lens: [n + 8 for n in lens])
    cache.num_blocks = None
    cache._room_for(lambda lens: [n + 8 for n in lens])
    assert len(grown) == 1
