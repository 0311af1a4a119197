"""CPU-side checks of the speculative-decoding operators: what is refused on the host before anything is launched, and the
64-bit forms that the GPU tests compare with."""

import ctypes as C

import numpy as np
import pytest
import torch

from tests import _spec_oracle as O


@pytest.fixture(scope="module")
def lib():
    from entmaxkv_b200 import _lib
    from entmaxkv_b200.build import build_library
    build_library()
    return _lib.load()


def fake(n=256):
    buf = (C.c_char * (n + 16))()
    return buf, C.addressof(buf) + (-C.addressof(buf)) % 16


def desc(base, **change):
    from entmaxkv_b200 import _lib
    d = _lib.CacheDesc()
    d.k = d.v = d.k_min = d.k_max = d.k_mean = d.k_std = d.seq_lens = base
    d.kv_stride_b, d.kv_stride_h = 64 * 160, 64 * 160
    d.meta_stride_b, d.meta_stride_h = 64 * 10, 64 * 10
    d.batch, d.kv_heads, d.head_dim, d.page_size, d.capacity, d.page_capacity, d.dtype = 2, 1, 64, 16, 160, 10, 1
    for name, value in change.items():
        setattr(d, name, value)
    return d


S3 = C.c_int64 * 3


def test_norm_rope_arguments(lib):
    buf, p = fake()
    st = S3(64, 64, 64)
    good = [1, 1, 1, 1, 1, 64, p, st, p, st, p, st, p, st, p, 0, 0, 0, p, 8, 0, None, None, 0, 1, 1e-6, None]
    def call(**change):
        args = list(good)
        for i, v in change.items():
            args[int(i[1:])] = v
        return lib.ekv_qk_norm_rope(*args)
    assert call(a0=7) == -1 and call(a5=96) == -1
    assert call(a1=-1) == -2 and call(a3=0) == -2 and call(a4=-1) == -2
    assert call(a6=None) == -2 and call(a7=None) == -2 and call(a12=None) == -2 and call(a14=None) == -2
    assert call(a6=p + 2) == -2 and call(a7=S3(64, 3, 64)) == -2 and call(a13=S3(64, 64, 1)) == -2
    assert call(a19=12) == -2 and call(a19=40) == -2 and call(a18=None) == -2
    assert call(a25=-1.0) == -2 and call(a25=float("nan")) == -2
    assert call(a1=0) == 0 and call(a2=0) == 0                       # nothing to do


def test_block_table_arguments(lib):
    buf, p = fake()
    assert lib.ekv_plan_block_tables(p, p, 0, -1, 16, p, 4, 4, p, 4, None, None, 0, None, None, None) == -2
    assert lib.ekv_plan_block_tables(p, p, 0, 16385, 16, p, 4, 4, p, 4, None, None, 0, None, None, None) == -2
    assert lib.ekv_plan_block_tables(p, p, 0, 2, 0, p, 4, 4, p, 4, None, None, 0, None, None, None) == -2
    assert lib.ekv_plan_block_tables(None, p, 0, 2, 16, p, 4, 4, p, 4, None, None, 0, None, None, None) == -2
    assert lib.ekv_plan_block_tables(p, p, 0, 2, 16, None, 4, 4, p, 4, None, None, 0, None, None, None) == -2
    assert lib.ekv_plan_block_tables(p, p, 0, 2, 16, p, 3, 4, p, 4, None, None, 0, None, None, None) == -2
    assert lib.ekv_plan_block_tables(p, p, 0, 2, 16, p, 4, 4, None, 4, None, None, 0, None, None, None) == -2
    assert lib.ekv_plan_block_tables(None, None, 0, 0, 16, None, 0, 0, None, 0, None, None, 0, None, None, None) == 0
    assert lib.ekv_release_blocks(p, p, 0, 2, 16, p, 3, 4, p, 4, None, None) == -2
    assert lib.ekv_release_blocks(None, None, 0, 0, 16, None, 0, 0, None, 0, None, None) == 0


def test_extend_arguments(lib):
    buf, p = fake()
    def call(d=None, k=p, v=p, sb=64, sh=64, st=64, tokens=1, counters=p, status=p):
        return lib.ekv_extend(C.byref(d or desc(p)), k, v, sb, sh, st, tokens, None, None, 0, None, counters, status, None)
    assert call(k=None) == -2 and call(v=None) == -2 and call(tokens=0) == -2
    assert call(counters=None) == -2 and call(status=None) == -2
    assert call(k=p + 2) == -2 and call(st=3) == -2 and call(sh=1) == -2 and call(sb=5) == -2
    assert call(desc(p, k_mean=None)) == -2 and call(desc(p, dtype=9)) == -1 and call(desc(p, head_dim=96)) == -1


def test_tree_arguments(lib):
    buf, p = fake()
    d = desc(p)
    size = lib.ekv_tree_workspace_bytes(C.byref(d), 4, 3, 160)
    assert size > 4 * 3 * 2 * 160 * 8
    assert lib.ekv_tree_workspace_bytes(C.byref(d), 4, 3, 0) > 0
    for q_heads, tokens, most in ((0, 3, 160), (4, 0, 160), (4, 257, 160), (4, 3, 161), (4, 3, -1)):
        assert lib.ekv_tree_workspace_bytes(C.byref(d), q_heads, tokens, most) == 0
    assert lib.ekv_tree_workspace_bytes(C.byref(desc(p, kv_heads=3)), 4, 3, 160) == 0
    # the scratch of many rows over a long cache is bounded: the rest takes turns
    big = desc(p, batch=64, kv_heads=8, capacity=1 << 17, page_capacity=1 << 13, kv_stride_h=64 << 17, kv_stride_b=64 << 20)
    assert lib.ekv_tree_workspace_bytes(C.byref(big), 64, 64, 1 << 17) <= (6 << 30) + 256
    st = S3(64, 64, 64)
    def call(d=d, q=p, qs=st, heads=4, tokens=3, k=p, v=p, mask=p, most=160, alpha=1.5, out=p, os_=st, ws=p, n=size):
        return lib.ekv_tree_decode(C.byref(d), q, qs, heads, tokens, k, st, v, st, mask, 0, 3, None, most, alpha, out, os_,
                                   None, ws, n, None, None)
    assert call(q=None) == -2 and call(k=None) == -2 and call(mask=None) == -2 and call(out=None) == -2
    assert call(ws=None) == -2 and call(qs=None) == -2 and call(os_=None) == -2
    assert call(q=p + 2) == -2 and call(qs=S3(64, 4, 64)) == -2
    assert call(tokens=300) == -2 and call(heads=0) == -2 and call(most=161) == -2
    assert call(alpha=1.0) == -4 and call(alpha=float("nan")) == -4 and call(alpha=float("inf")) == -4
    assert call(n=size // 2) == -3


def test_python_entry_points_refuse_cpu_tensors():
    import entmaxkv_b200 as E
    x = torch.zeros(1, 1, 2, 64)
    with pytest.raises(ValueError):
        E.qk_norm_rope(x, x, torch.zeros(2, dtype=torch.int32), torch.ones(8))
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        E.plan_block_tables(i, 1, i.view(2, 1), i, 16)
    with pytest.raises(ValueError):
        E.release_block_tables(i, 1, i.view(2, 1), i, 16)
    with pytest.raises(RuntimeError):
        E.tree_attention_decode(x, E.PagedKVCache(16), x, x, torch.ones(2, 2, dtype=torch.bool), x)
    with pytest.raises(RuntimeError):
        E.PagedKVCache(16).extend(x, x)
    with pytest.raises(RuntimeError):
        E.PagedKVCache(16).release([0])
    with pytest.raises(ValueError):
        E.PagedKVCache(16, block_table=True, num_blocks=0)


def test_the_class_bound_lies_under_the_threshold():
    """What the score pass relies on: the threshold of some of the scores is never above that of all of them."""
    g = np.random.default_rng(5)
    for alpha in (4 / 3, 1.5, 2.0, 3.0):
        for _ in range(20):
            z = g.normal(size=300) * g.choice([0.1, 0.5, 2.0])
            tau = O.entmax_weights(z, alpha)[1]
            classes = z[:256].reshape(32, 8).max(1)
            assert O.entmax_weights(classes, alpha)[1] <= tau + 1e-12
            assert z.max() - 1 <= tau + 1e-12


def test_oracle_weights_sum_to_one_and_plan_releases_what_it_took():
    z = np.random.default_rng(6).normal(size=50)
    for alpha in (1.5, 2.0, 2.5):
        w, tau = O.entmax_weights(z, alpha)
        assert abs(w.sum() - 1) < 1e-9 and (w[z <= tau] == 0).all()
    table, slots, positions, starts = O.plan([3, 0], [2, 5], [[7, -1], [-1, -1]], [7, 4, 5, 6], 4, 9)
    assert table == [[7, 4], [5, 6]] and starts == [0, 2, 7] and positions == [3, 4, 0, 1, 2, 3, 4, -1, -1]
    assert slots == [31, 16, 20, 21, 22, 23, 24, -1, -1]
    table, free, kept = O.release([5, 5], [0, 4], table, [7, 4, 5, 6], 4)
    assert kept == [0, 4] and table == [[-1, -1], [5, -1]] and sorted(free[1:] + [5]) == [4, 5, 6, 7]
