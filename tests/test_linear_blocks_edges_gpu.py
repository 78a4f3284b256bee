"""The block-scaled and grouped products where their inputs leave the ordinary range, on every tile form
that the sizes choose: gates far below zero, scales whose product leaves FP32, non-finite values and
partial boxes on pairs of SMs, streams that join, a quantiser past 2^31 elements."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import tsfm_b200 as tb  # noqa: E402
from test_linear_blocks_gpu import E4M3, Case, gen, ptr, quantize  # noqa: E402

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


@pytest.mark.parametrize("act", [0, 1, 3])
@pytest.mark.parametrize("kind", ["e4m3", torch.bfloat16], ids=str)
def test_nonfinite_values_on_pairs_of_sms(kind, act):
    # rows and columns of NaN and infinities on 256 x 256 tiles: through the boxes (16-bit y), and past them
    counts = [4000, 0, 3500, 1500]
    M, N, K = sum(counts), 2048, 1024
    c = Case(M, N, K, kind, counts=counts, seed=23)
    if act == 3:
        k = 0.5 / float(c.ref.std())
        (c.xs if kind == "e4m3" else c.x).mul_(k)
    cols = N // 2 if act == 3 else N
    dtypes = (torch.bfloat16,) if act == 3 else (torch.bfloat16, torch.float32)
    clean = {}
    for dtype in dtypes:
        for pad in (0, 4):
            clean[dtype, pad] = torch.zeros(M, cols + pad, device="cuda", dtype=dtype)
            tb.check(c.call(clean[dtype, pad], act=act))
    c.x[45, 7] = float("nan")
    if kind == "e4m3":
        c.xs[7777, 1] = float("inf")
    else:
        c.x[7777, 200] = float("inf")
    c.w[2, 20, 3] = float("nan")        # gated: g of column 20; else column 20
    c.w[2, 256 + 128 + 71, 9] = float("nan")  # gated: u of column 128 + 71
    hit = torch.zeros(cols, dtype=torch.bool, device="cuda")
    hit[[20, 199] if act == 3 else [20, 455]] = True
    keep = torch.ones(M, cols, dtype=torch.bool, device="cuda")
    keep[45] = keep[7777] = False
    keep[4000:7500, hit] = False
    for (dtype, pad), want in clean.items():
        y = torch.zeros_like(want)
        tb.check(c.call(y, act=act))
        torch.cuda.synchronize()
        assert torch.equal(y[:, :cols][keep], want[:, :cols][keep])
        if act == 1:  # a NaN becomes 0
            assert (y[45] == 0).all() and (y[4000:7500, :cols][:, hit] == 0).all()
            assert not (torch.isfinite(y[7777, :cols]) & (y[7777, :cols] != 0)).any()
        else:
            assert torch.isnan(y[45, :cols]).all() and torch.isnan(y[4000:7500, :cols][:, hit]).all()
            assert not (torch.isfinite(y[7777, :cols]) & (y[7777, :cols] != 0)).any()


def test_streams_that_join():
    # A product whose operands come from kernels of two streams that meet by an event, eager and captured, and
    # whose output a third call overwrites at once.
    M, N, K = 2500, 1024, 768
    g = gen(26)
    x = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    w = torch.randn(N, K, generator=g, device="cuda").bfloat16()
    xq, xs = torch.zeros(M, K, dtype=torch.uint8, device="cuda"), torch.zeros(M, K // 128, device="cuda")
    wq, ws = torch.zeros(N, K, dtype=torch.uint8, device="cuda"), torch.zeros(N // 128, K // 128, device="cuda")
    y, copy = torch.zeros(M, N, device="cuda"), torch.zeros(M, N, device="cuda")
    side = torch.cuda.Stream()

    def steps(pause):
        main = torch.cuda.current_stream()
        xq.zero_(), xs.zero_(), wq.zero_(), ws.zero_(), y.zero_()
        side.wait_stream(main)
        pause()
        tb.check(tb.lib.tsfm_kernel_quantize_e4m3(ptr(w), 2, N, K, K, 128, ptr(wq), K, ptr(ws), K // 128, side.cuda_stream))
        tb.check(tb.lib.tsfm_kernel_quantize_e4m3(ptr(x), 2, M, K, K, 1, ptr(xq), K, ptr(xs), K // 128, main.cuda_stream))
        main.wait_stream(side)
        pause()
        tb.check(tb.lib.tsfm_kernel_linear_e4m3(ptr(xq), ptr(xs), K // 128, ptr(wq), ptr(ws), K // 128, None, ptr(y), 0, 0, 0,
                                                M, N, K, K, K, N, main.cuda_stream))
        side.wait_stream(main)
        with torch.cuda.stream(side):
            copy.copy_(y)
        main.wait_stream(side)
        pause()
        tb.check(tb.lib.tsfm_kernel_linear_e4m3(ptr(xq), ptr(xs), K // 128, ptr(wq), ptr(ws), K // 128, None, ptr(y), 0, 1, 0,
                                                M, N, K, K, K, N, main.cuda_stream))

    steps(torch.cuda.synchronize)
    torch.cuda.synchronize()
    want = y.clone(), copy.clone()
    assert want[1].abs().max() > 0 and torch.equal(want[0], 2 * want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps(lambda: None)
    for how in (lambda: steps(lambda: None), graph.replay) * 5:
        y.fill_(-1.0), copy.fill_(-1.0)
        how()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(copy, want[1])


@pytest.mark.parametrize("kind", ["e4m3", torch.bfloat16], ids=str)
def test_large_grouped_products_repeat_themselves(kind):
    # 32768 rows over 24 of 32 groups, gated: the same bits from every call, alone and in a row
    g = gen(27)
    counts = (torch.rand(32, generator=g, device="cuda") ** 2 * (torch.arange(32, device="cuda") % 4 != 1)).cpu().numpy()
    counts = np.floor(counts / counts.sum() * 32768).astype(int)
    counts[0] += 32768 - counts.sum()
    c = Case(32768, 4096, 1024, kind, counts=counts.tolist(), seed=28)
    k = 0.5 / float(c.ref.std())
    (c.xs if kind == "e4m3" else c.x).mul_(k)
    want = torch.zeros(32768, 2048, device="cuda", dtype=torch.bfloat16)
    tb.check(c.call(want, act=3))
    torch.cuda.synchronize()
    ys = [torch.zeros_like(want) for _ in range(8)]
    for y in ys:
        tb.check(c.call(y, act=3))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in ys)


def test_quantize_past_32_bits():
    # more than 2^31 elements: the last rows and scales
    rows, cols = 1050000, 2056
    x = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    tail = torch.randn(200, cols, generator=gen(29), device="cuda").bfloat16()
    x[-200:] = tail
    for block_rows in (1, 128):
        q, s = quantize(x, block_rows)
        first = rows - 200 - (rows - 200) % block_rows  # of the last 200 rows' blocks
        part = x[first:].clone()
        qw, sw = quantize(part, block_rows)
        assert torch.equal(q[first:], qw) and torch.equal(s[first // block_rows:], sw)
        assert qw[-1].any() and (q[:first] == 0).all() and (s[:first // block_rows] == 2.0 ** -126).all()
        del q, s
    del x
    torch.cuda.empty_cache()
