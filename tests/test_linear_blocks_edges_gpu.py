"""The block-scaled and grouped products where their inputs leave the ordinary range, on every tile form
that the sizes choose: gates far below zero, scales whose product leaves FP32, non-finite values and
partial boxes on pairs of SMs, streams that join, a quantiser past 2^31 elements."""
import pytest

torch = pytest.importorskip("torch")

import tsfm_b200 as tb  # noqa: E402
from test_linear_blocks_gpu import E4M3, Case, gen  # noqa: E402

pytestmark = pytest.mark.gpu

# (M, N, K, groups' rows or None): E4M3 with few rows, on 64 columns, K shared by 8 CTAs, on 128 columns,
# on pairs of SMs; grouped with few rows (up to 8 and more), on 64, 128 and 256 columns.
FORMS = {
    "few": (5, 1024, 256, None), "64": (60, 1024, 256, None), "shared": (3, 512, 4096, None),
    "128": (3000, 1024, 256, None), "256": (8000, 2048, 1024, None),
    "g_few": (11, 512, 256, [4, 0, 7]), "g_few32": (40, 512, 256, [1] * 20 + [20]),
    "g_few_many": (60, 512, 256, [2, 1] * 20),
    "g_64": (200, 512, 256, [150, 0, 50]), "g_128": (3000, 1024, 256, [1000, 0, 1990, 10]),
    "g_256": (9000, 2048, 1024, [4000, 1, 0, 4999]),
}


@pytest.mark.parametrize("kind", ["e4m3", torch.bfloat16], ids=str)
@pytest.mark.parametrize("form", FORMS)
def test_gate_far_below_zero(form, kind):
    # One column of x is 1, the rest 0: u and g are single operands, exact but for the scale. Against
    # g u / (1 + e^-u): the exponential's argument is rounded, off by |u| log2(e) <= 126 half steps of
    # 2^-24 and as much by the constant's own rounding for u above -87, so with ln 2 and the approximate
    # exponential and reciprocal, the products and the two formulas' further steps under 72 of 2^-23.
    # Below -87 the reciprocal is flushed to zero, where silu is under 2^-119.
    M, N, K, counts = FORMS[form]
    if kind != "e4m3" and counts is None:
        counts = [M // 2, 0, M - M // 2]
    c = Case(M, N, K, kind, counts=counts, seed=21)
    G = c.groups
    c.x.zero_()
    c.x[:, 0] = 1.0
    r = gen(M + N)
    for su, sg in ((0.7, 1.0), (1.0, 2.0 ** 30), (2.0 ** 20, 1.0), (2.0 ** 60, 2.0 ** 40), (2.0 ** 90, 1.0), (2.0 ** 100, 2.0 ** 100),
                   (float("inf"), 3.0)):
        c.w.zero_()
        if kind == "e4m3":
            codes = torch.randint(0x20, 0x7F, (G, N), generator=r, device="cuda", dtype=torch.uint8)  # 2^-4 .. 448
            codes |= torch.randint(0, 2, (G, N), generator=r, device="cuda", dtype=torch.uint8) << 7
            c.w[:, :, 0] = codes.view(E4M3)
            c.xs.fill_(1.0)
            c.ws.fill_(1.0)
            c.ws[:, 0::2, 0] = sg
            c.ws[:, 1::2, 0] = su
            v = codes.view(E4M3).float().view(G, N // 256, 2, 128)
            g, u = v[:, :, 0] * sg, v[:, :, 1] * su
        else:
            v = 60 * torch.randn(G, N // 256, 2, 128, generator=r, device="cuda")
            v[v == 0] = 1.0
            g, u = (v[:, :, 0] * sg).to(kind), (v[:, :, 1] * su).to(kind)
            c.w[:, :, 0] = torch.stack((g, u), 2).view(G, N)
        g, u = g.double().view(G, N // 2), u.double().view(G, N // 2)
        ref = g * (u / (1 + torch.exp(-u)))
        assert not (su == float("inf")) or torch.isnan(ref).any()
        e = torch.bucketize(torch.arange(M, device="cuda"), c.off[1:].long(), right=True).clamp(max=G - 1)
        ref, tol = ref[e], (72 * 2.0 ** -23 * ref.abs() + g.abs() * 2.0 ** -119)[e]
        for dtype in (torch.bfloat16, torch.float16) if su < 1 else (torch.bfloat16,):
            if kind != "e4m3" and dtype != kind:
                continue
            for pad in (0, 4):
                y = torch.full((M, N // 2 + pad), 5.0, device="cuda", dtype=dtype)
                tb.check(c.call(y, act=3))
                torch.cuda.synchronize()
                out = y[:, :N // 2].double()
                lim = tol + torch.finfo(dtype).eps / 2 * (ref.abs() + tol) + torch.finfo(dtype).smallest_normal
                want = ref.to(dtype).double()  # past F16's largest number: infinite
                bad = ~((out - ref).abs() <= lim) & ~(out == want) & ~(torch.isnan(out) & torch.isnan(ref))
                bad &= c.used[:, None]
                assert not bad.any(), (su, sg, dtype, pad, int(bad.sum()), out[bad][:4].tolist(), ref[bad][:4].tolist())


@pytest.mark.parametrize("form", FORMS)
def test_scales_whose_product_leaves_fp32(form):
    # y = sum_b xs ws S_b for scales of which the product of two is past FP32 (blocks 1 of K: 2^140) or below
    # its normal numbers (blocks 2: 2^-140, 2^-150): rows of x whose codes are zero in the blocks of the
    # first kind keep the others' sum; rows of one subnormal code there reach 2^122; rows that have codes in
    # the blocks of the second kind alone reach 2^-115. Tolerance: that of Case, with one more rounding.
    M, N, _, counts = FORMS[form]
    K = 4096 if form == "shared" else 700
    c = Case(M, N, K, "e4m3", counts=counts, seed=22)
    kb, G = -(-K // 128), c.groups
    r = gen(M * 3 + N)
    blk = torch.arange(K, device="cuda") // 128 % 4
    row = torch.arange(M, device="cuda") % 3
    cx = c.x[:, :K].view(torch.uint8)
    cw = c.w[:, :, :K].view(torch.uint8)
    cw[:, :, blk == 1] = torch.randint(1, 4, (G, N, int((blk == 1).sum())), generator=r, device="cuda", dtype=torch.uint8)
    cx[:, blk == 1] = 0
    tiny = torch.zeros(M, K, dtype=torch.bool, device="cuda")
    tiny[row == 1, 130] = True
    cx[tiny] = 1
    cx[(row == 2)[:, None] & (blk != 2)[None]] = 0
    xs = c.xs[:, :kb]
    ws = c.ws[:, :, :kb]
    kind = torch.arange(kb, device="cuda") % 4
    xs.copy_(1 + torch.rand(M, kb, generator=r, device="cuda"))
    ws.copy_((1 + torch.rand(G, ws.shape[1], kb, generator=r, device="cuda")))
    ws[:, 0::2] *= -1
    xs[:, kind == 1] *= 2.0 ** 100
    ws[:, :, kind == 1] *= 2.0 ** 40
    xs[0::2, kind == 2] *= 2.0 ** -100
    xs[1::2, kind == 2] *= 2.0 ** -110
    ws[:, :, kind == 2] *= 2.0 ** -40
    xd = c.x[:, :K].double() * xs.double().repeat_interleave(128, 1)[:, :K]
    unit = (K + 3 * kb + 8) * 2.0 ** -23
    for e in range(G):
        lo, hi = (0, M) if counts is None else (int(c.off[e]), int(c.off[e + 1]))
        wd = c.w[e, :, :K].double() * ws[e].double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
        c.ref[lo:hi] = xd[lo:hi] @ wd.T
        c.tol[lo:hi] = unit * (xd[lo:hi].abs() @ wd.abs().T)
    assert c.ref[c.used & (row == 1)].abs().min() > 2.0 ** 110 and c.ref[c.used & (row == 2)].abs().max() < 2.0 ** -110
    for dtype in (torch.float32, torch.bfloat16):
        y = torch.full((M, N), 5.0, device="cuda", dtype=dtype)
        tb.check(c.call(y))
        torch.cuda.synchronize()
        out = y.double()
        # the smallest numbers: every sum of a block rounds once more to a multiple of 2^-149
        lim = c.tol + torch.finfo(dtype).eps / 2 * (c.ref.abs() + c.tol) + (kb + 1) * 2.0 ** -149
        if dtype == torch.bfloat16:
            lim = lim + 2.0 ** -134
        bad = ~((out - c.ref).abs() <= lim) & c.used[:, None]
        assert not bad.any(), (dtype, int(bad.sum()), [int((bad[row == i]).sum()) for i in range(3)],
                               out[bad][:4].tolist(), c.ref[bad][:4].tolist())


@pytest.mark.parametrize("M,N,K", [(8000, 1000, 768), (9001, 1001, 392), (7000, 1300, 768)])
def test_partial_boxes_leave_the_padding(M, N, K):
    # 16-bit outputs of 256 x 256 tiles leave in boxes of 64 columns x 32 rows: the last ones are clipped to
    # N columns (odd ones too) and M rows, the padding of a row is left as it was
    assert N % 64
    c = Case(M, N, K, "e4m3", bias=True, seed=24)
    for dtype in (torch.bfloat16, torch.float16):
        c.check(dtype, pad=-N % 8)
        c.check(dtype, act=1, pad=-N % 8 + 24)
        c.check(dtype, pad=-N % 8 + 8, shift=8)
    g = Case(M, N, K, "e4m3", counts=[M // 2, 0, 3, M - M // 2 - 10], first=4, bias=True, seed=25)
    g.check(torch.bfloat16, pad=-N % 8 + 24)
