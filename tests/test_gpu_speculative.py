"""The speculative-decoding operators together, as a decode loop uses them (run on a B200: ``-m gpu``).

Per step: the drafted rows' queries and keys are normed and rotated at their positions in the tree, attend to the cache
and to their ancestors, and the accepted path is written into the cache.  The yardstick is the same model run one token at
a time through the existing top-k step with a budget that covers the cache (dense entmax attention).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE = 8, 2, 64, 16


def rows(n, seed, B):
    """The fused projection of n tokens per sequence."""
    return torch.randn(B, n, HQ + 2 * HKV, D, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


def split(x):
    return (t.transpose(1, 2) for t in x.split([HQ, HKV, HKV], dim=2))


@pytest.mark.parametrize("layout", ["dense", "pool"])
def test_accepted_paths_equal_one_token_at_a_time(layout):
    import entmaxkv_b200 as E
    B, lens = 2, [37, 130]
    inv = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float32, device="cuda") / (D // 2))
    wq, wk = (torch.linspace(0.5, 1.5, D, device="cuda").bfloat16() for _ in range(2))
    prompt = rows(max(lens), 1, B)
    kw = dict(block_table=True, num_blocks=60) if layout == "pool" else {}
    tree, plain = E.PagedKVCache(PAGE, **kw), E.PagedKVCache(PAGE)
    for c in (tree, plain):
        q, k, v = split(prompt)
        _, k = E.qk_norm_rope(q, k, torch.arange(max(lens), device="cuda"), inv, wq, wk)
        # the prompt in two chunks: the first by initialize, the second by extend
        c.initialize(k[:, :, :30], v[:, :, :30].contiguous(), seq_lens=[30, 30])
        c.extend(k[:, :, 30:], v[:, :, 30:], counts=[n - 30 for n in lens])
    # a tree of seven tokens: 0 - 1 - 2, 0 - 3 - 4 - 5, 6
    parent = [-1, 0, 1, 0, 3, 4, -1]
    mask, depth = torch.zeros(7, 7, dtype=torch.bool), []
    for t, p in enumerate(parent):
        if p >= 0:
            mask[t] = mask[p]
        mask[t, t] = True
        depth.append(int(mask[t].sum()) - 1)
    depth = torch.tensor(depth, device="cuda")
    paths = [[0, 3, 4, 5], [0, 1], [6], []]
    for step in range(4):
        draft = rows(7, 100 + step, B)
        q, k, v = split(draft)
        positions = tree.seq_lens[:, None] + depth
        q, k = E.qk_norm_rope(q, k, positions, inv, wq, wk)
        out = torch.zeros_like(q)
        E.tree_attention_decode(q, tree, k, v, mask.cuda(), out)
        accepted = [paths[(step + b) % 4] for b in range(B)]
        # one token at a time, along each sequence's accepted path
        longest = max(map(len, accepted))
        for i in range(longest):
            index = [p[i] if i < len(p) else 0 for p in accepted]
            one = torch.stack([draft[b, j] for b, j in enumerate(index)])[:, None]
            q1, k1, v1 = split(one)
            q1, k1 = E.qk_norm_rope(q1, k1, plain.seq_lens[:, None], inv, wq, wk)
            before = plain.seq_lens.clone()
            got = torch.zeros_like(q1)
            E.sparse_attention_decode_paged(q1, plain, k1, v1, got, 1 << 20, alpha=1.5, niter=12)
            for b, p in enumerate(accepted):
                if i < len(p):
                    want = out[b, :, p[i]].float()
                    # two roundings of the output to bf16 (half a step each, 2^-8), and the scores' own differences
                    assert (got[b, :, 0].float() - want).abs().max() <= (2 * 2.0 ** -8 + 2.0 ** -10) * want.abs().max()
            taken = torch.tensor([int(i < len(p)) for p in accepted], dtype=torch.int32, device="cuda")
            plain.extend(k1[:, :, :0], v1[:, :, :0], start=before + taken)        # those that had no token step back
        counts = torch.tensor([len(p) for p in accepted], dtype=torch.int32, device="cuda")
        index = torch.tensor([p + [0] * (7 - len(p)) for p in accepted], dtype=torch.int32, device="cuda")
        tree.extend(k, v, counts=counts, index=index)
        assert tree.sync_lengths() == plain.sync_lengths()
        for b, n in enumerate(tree.host_seq_lens):
            assert torch.equal(tree.k_cache[b, :, :n], plain.k_cache[b, :, :n])
            for name in ("k_min", "k_max", "k_mean", "k_std"):
                pages = -(-n // PAGE)
                assert torch.equal(getattr(tree, name)[b, :, :pages], getattr(plain, name)[b, :, :pages]), name
    assert tree.device_status() == 0 and plain.device_status() == 0


def test_operators_on_a_stream_of_their_own():
    """Everything on a side stream, while the default stream is busy with other memory."""
    import entmaxkv_b200 as E
    x = rows(40, 5, 1)
    results = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            q, k, v = split(x)
            q, k = E.qk_norm_rope(q, k, torch.arange(40, device="cuda"), torch.ones(8, device="cuda"))
            c = E.PagedKVCache(PAGE, block_table=True, num_blocks=6)
            c.initialize(k[:, :, :33].contiguous(), v[:, :, :33].contiguous())
            c.extend(k[:, :, 33:36], v[:, :, 33:36])
            out = torch.zeros(1, HQ, 4, D, dtype=torch.bfloat16, device="cuda")
            E.tree_attention_decode(q[:, :, 36:], c, k[:, :, 36:], v[:, :, 36:],
                                    torch.ones(4, 4, dtype=torch.bool, device="cuda").tril(), out)
        results.append((out, c.k_cache, stream))
    for _, _, stream in results:
        stream.synchronize()
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
