"""Per-head norm with the position rotation (run on a B200: ``-m gpu``), against the definition in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from tests import _spec_oracle as O

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}

CASES = [
    # B, T, Hq, Hkv, D, dtype, rotated elements, interleaved, eps, weights ("own", "fp32", None), first position
    (1, 1, 32, 8, 128, "bf16", 128, False, 1e-6, "own", 0),
    (3, 7, 5, 1, 64, "fp16", 64, False, 1e-5, "fp32", 1000),
    (2, 33, 8, 2, 128, "bf16", 64, True, 1e-6, None, 131071),
    (1, 5, 1, 1, 64, "fp32", 32, False, 1e-6, "own", 1048000),
    (2, 3, 3, 3, 128, "fp32", 128, True, 1e-6, "own", 16777300),     # past what fp32 counts
    (1, 400, 40, 8, 128, "fp16", 16, False, None, None, 5),
    (2, 2, 4, 2, 64, "bf16", 0, False, 1e-6, "own", 3),              # no rotation
    (1, 9, 2, 2, 128, "bf16", 128, False, 1e-6, "own", -4),
]


@pytest.mark.parametrize("case", CASES, ids=[f"case{i}" for i in range(len(CASES))])
@pytest.mark.parametrize("fused", [False, True])
def test_norm_rope_against_64_bits(case, fused):
    import entmaxkv_b200 as E
    B, T, Hq, Hkv, D, dt, rd, inter, eps, weights, pos0 = case
    dtype = DT[dt]
    g = torch.Generator().manual_seed(40 + T + D)
    x = (1.7 * torch.randn(B, T, Hq + 2 * Hkv, D, generator=g)).to(dtype)
    q, k = x[:, :, :Hq].transpose(1, 2), x[:, :, Hq:Hq + Hkv].transpose(1, 2)
    pos = torch.arange(pos0, pos0 + T)
    pos = pos.to(torch.int32) if T % 2 else pos[None] + 3 * torch.arange(B)[:, None]
    inv = (10000.0 ** (-torch.arange(rd // 2, dtype=torch.float64) / max(rd // 2, 1))).float()
    wt = None if weights is None else dtype if weights == "own" else torch.float32
    qw, kw = (None if wt is None else (1 + 0.3 * torch.randn(D, generator=g)).to(wt) for _ in range(2))
    cu = lambda t: None if t is None else t.cuda()  # noqa: E731
    xc = x.cuda()
    qc, kc = xc[:, :, :Hq].transpose(1, 2), xc[:, :, Hq:Hq + Hkv].transpose(1, 2)
    if not fused:
        qc, kc = qc.contiguous(), kc.contiguous()
    got = E.qk_norm_rope(qc, kc, pos.cuda(), inv.cuda(), cu(qw), cu(kw), eps, interleaved=inter)
    for a, src, w in ((got[0], q, qw), (got[1], k, kw)):
        ref = O.norm_rope(src, pos, inv, w, eps, inter)
        size = O.norm_rope(src, pos, inv * 0, w, eps, inter).abs()
        # of a pair (a, b): the norm is off by (D / 16 + 8) 2^-24 at most (sum in lanes and a tree, root, division,
        # weight), each coefficient by 6 2^-24 (its argument, the sine), the rotation adds two roundings
        pair = size.clone()
        half = rd // 2
        if inter:
            pair[..., :rd] = size[..., :rd] + size[..., :rd].unflatten(-1, (half, 2)).flip(-1).flatten(-2)
        elif rd:
            pair[..., :rd] = size[..., :rd] + size[..., :rd].unflatten(-1, (2, half)).flip(-2).flatten(-2)
        tol = pair * (D / 16 + 8 + 6 + 2) * 2.0 ** -24
        half_step = torch.finfo(dtype).eps / 2
        tol = tol * (1 + half_step) + half_step * ref.abs() + torch.finfo(dtype).tiny
        err = (a.cpu().double() - ref).abs()
        assert bool((err <= tol).all()), f"worst {float((err / tol).max())} of the bound"
    # in place, the same bits
    q2, k2 = qc.clone(), kc.clone()
    r = E.qk_norm_rope(q2, k2, pos.cuda(), inv.cuda(), cu(qw), cu(kw), eps, interleaved=inter, q_out=q2, k_out=k2)
    assert r[0] is q2 and torch.equal(q2, got[0]) and torch.equal(k2, got[1])


def test_outside_the_rotated_part_infinities_stay():
    import entmaxkv_b200 as E
    q = torch.ones(1, 1, 2, 64, device="cuda")
    q[..., 40] = math.inf
    out, _ = E.qk_norm_rope(q, q.clone(), torch.tensor([3, 4], device="cuda"), torch.ones(16, device="cuda"), eps=None)
    assert torch.isposinf(out[..., 40]).all() and torch.isfinite(out[..., :40]).all()


def test_odd_strides_are_copied_and_outputs_keep_their_neighbours():
    import entmaxkv_b200 as E
    g = torch.Generator().manual_seed(3)
    base = torch.randn(2, 4, 6, 65, generator=g).to(torch.bfloat16).cuda()
    q, k = base[:, :3, :, 1:], base[:, 3:, :, :64]                      # rows that start anywhere
    pos, inv = torch.arange(6, device="cuda"), torch.ones(8, device="cuda")
    want = E.qk_norm_rope(q.contiguous(), k.contiguous(), pos, inv)
    room = torch.full((2, 6, 4, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    got = E.qk_norm_rope(q, k, pos, inv, q_out=room[:, :, :3].transpose(1, 2))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and (room[:, :, 3] == 9).all()
    empty = torch.zeros(2, 3, 0, 64, dtype=torch.bfloat16, device="cuda")
    assert E.qk_norm_rope(empty, empty, torch.zeros(0, dtype=torch.int32, device="cuda"), inv)[0].shape == empty.shape


def test_refusals():
    import entmaxkv_b200 as E
    q, k = torch.zeros(2, 4, 3, 64, device="cuda"), torch.zeros(2, 2, 3, 64, device="cuda")
    good = dict(q=q, k=k, positions=torch.zeros(2, 3, dtype=torch.int32, device="cuda"),
                inv_freq=torch.ones(16, device="cuda"))
    E.qk_norm_rope(**good)
    w = torch.ones(64, device="cuda")
    bad = [dict(q=q.cpu()), dict(q=q[0]), dict(k=k[:1]), dict(k=k.half()), dict(q=q[..., :32], k=k[..., :32]),
           dict(q=q.double(), k=k.double()), dict(positions=torch.zeros(2, 3, device="cuda")),
           dict(positions=torch.zeros(3, 2, dtype=torch.int32, device="cuda")),
           dict(inv_freq=torch.ones(40, device="cuda")), dict(inv_freq=torch.ones(12, device="cuda")),
           dict(inv_freq=torch.ones(16, dtype=torch.float64, device="cuda")), dict(q_weight=w[:32]),
           dict(q_weight=w.half()), dict(q_weight=w, eps=None), dict(eps=-1.0), dict(eps=math.nan),
           dict(q_out=torch.zeros(2, 4, 3, 64, dtype=torch.half, device="cuda")), dict(k_out=q),
           dict(q_out=torch.zeros(2, 4, 64, 3, device="cuda").transpose(-1, -2)),
           dict(q_out=torch.zeros(2, 1, 3, 64, device="cuda").expand(2, 4, 3, 64))]
    for change in bad:
        with pytest.raises(ValueError):
            E.qk_norm_rope(**{**good, **change})
