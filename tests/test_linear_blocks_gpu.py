"""The E4M3 quantiser, the block-scaled 8-bit product and the products grouped by expert against
float64 on the GPU, through the C ABI: odd sizes, one row, empty and ragged groups, padded strides,
non-finite values, rows that belong to no group, streams and graphs.

Tolerances. The operands are exact in float64. A product is a sum of K terms added in FP32 in some
order, with at most two more FP32 operations per 128 (scales): each operation is off by at most
2^-23 (a truncating adder) of a partial sum that sum|x w| bounds, so |error| <= (K + 2 K / 128 + 8)
2^-23 sum|x w|, plus half a step of the output type."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import tsfm_b200 as tb  # noqa: E402
from helpers import e4m3_bits  # noqa: E402

pytestmark = pytest.mark.gpu

CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
E4M3 = torch.float8_e4m3fn


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def up(n, m):
    return -(-n // m) * m


# ---- quantiser --------------------------------------------------------------------------------

def block_scales(x, block_rows):
    """numpy restatement: per block, the smallest power of two with amax / s <= 448, >= 2^-126."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    out = np.empty((-(-rows // block_rows), -(-cols // 128)), np.float32)
    for i in range(out.shape[0]):
        for j in range(out.shape[1]):
            a = np.abs(x[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128])
            if not np.isfinite(a).all():
                out[i, j] = np.nan
                continue
            e = -126
            while a.max() > 448.0 * 2.0 ** e:
                e += 1
            out[i, j] = 2.0 ** e
    return out


def quantize(x, block_rows, ldq=None, ld_scale=None):
    rows, cols = x.shape
    kb = -(-cols // 128)
    q = torch.full((rows, ldq or cols), 0x55, device="cuda", dtype=torch.uint8)
    s = torch.full((-(-rows // block_rows), ld_scale or kb), -7.0, device="cuda")
    tb.check(tb.lib.tsfm_kernel_quantize_e4m3(ptr(x), CODE[x.dtype], rows, cols, x.stride(0), block_rows, ptr(q),
                                              q.stride(0), ptr(s), s.stride(0), stream()))
    torch.cuda.synchronize()
    return q, s


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 768), (3, 127), (5, 128), (130, 129), (257, 300), (128, 1024)])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_quantize_bit_for_bit(rows, cols, block_rows, dtype):
    g = gen(rows * 1000 + cols)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x = x * torch.exp(2 * torch.randn(rows, 1, generator=g, device="cuda"))
    x[rows // 2, : cols // 2] = 0
    x = x.to(dtype)
    # a row stride longer than the row, unaligned for odd columns; padding left alone
    wide = torch.zeros(rows, cols + 5, device="cuda", dtype=dtype)
    wide[:, :cols] = x
    kb = -(-cols // 128)
    for src in (x, wide[:, :cols]):
        q, s = quantize(src, block_rows, ldq=cols + 3, ld_scale=kb + 1)
        want = block_scales(x.float().cpu(), block_rows)
        assert np.array_equal(s[:, :kb].cpu().numpy(), want)
        spread = np.repeat(np.repeat(want, block_rows, 0)[:rows], 128, 1)[:, :cols]
        assert np.array_equal(q[:, :cols].cpu().numpy(), e4m3_bits(x.float().cpu().numpy() / spread))
        assert (q[:, cols:] == 0x55).all() and (s[:, kb:] == -7.0).all()


def test_quantize_extremes():
    x = torch.zeros(9, 256, device="cuda")
    x[1, 3] = float("inf")
    x[2, 200] = float("nan")
    x[3, 0] = -float("inf")
    x[4, 0] = torch.finfo(torch.float32).max
    x[5, :128] = 2.0 ** -149  # subnormal
    x[6, 0], x[6, 1] = 448.0, 3.0
    x[7, 0], x[7, 1] = 449.0, 3.0
    x[8, 0] = -(2.0 ** -126) * 448
    q, s = quantize(x, 1)
    s = s.cpu().numpy()
    assert np.isnan(s[1, 0]) and np.isnan(s[2, 1]) and np.isnan(s[3, 0])
    assert (q[1, :128] & 0x7F == 0x7F).all() and (q[2, 128:] & 0x7F == 0x7F).all()
    assert s[1, 1] == s[0, 0] == np.float32(2.0 ** -126) and (q[0] == 0).all()
    assert s[4, 0] == 2.0 ** 120 and q[4, 0].item() == 0x78  # 2^128 - 2^104 at 2^120: rounds to 256
    assert s[5, 0] == np.float32(2.0 ** -126) and (q[5, :128] == 0).all()
    assert s[6, 0] == 1.0 and q[6, 0].item() == 0x7E and s[7, 0] == 2.0 and q[7, 0].item() == 0x76
    assert s[8, 0] == np.float32(2.0 ** -126) and q[8, 0].item() == 0xFE
    qt, st = quantize(x, 128)
    assert torch.isnan(st).all() and (qt & 0x7F == 0x7F).all()


# ---- products ---------------------------------------------------------------------------------

class Case:
    """Operands of one product and its float64 result."""

    def __init__(self, M, N, K, kind, counts=None, first=0, bias=False, seed=0, scale_jitter=True):
        g = gen(seed + 31 * M + 7 * N + K)
        self.M, self.N, self.K, self.kind, self.counts = M, N, K, kind, counts
        G = self.groups = 1 if counts is None else len(counts)
        x = torch.randn(M, K, generator=g, device="cuda") * torch.exp(torch.randn(M, 1, generator=g, device="cuda"))
        w = torch.randn(G, N, K, generator=g, device="cuda") * 0.1
        kb, nb = -(-K // 128), -(-N // 128)
        if kind == "e4m3":
            ld = up(K, 16)
            self.x = torch.full((M, ld), float("nan"), device="cuda").to(E4M3)  # NaN in the padding
            self.w = torch.full((G, N, ld), float("nan"), device="cuda").to(E4M3)
            self.x[:, :K] = (x * 30).clamp(-448, 448).to(E4M3)
            self.w[:, :, :K] = (w * 300).clamp(-448, 448).to(E4M3)
            # scales that are no powers of two, negative ones among them, in padded rows
            self.xs = torch.randn(M, kb + 1, generator=g, device="cuda")
            self.ws = torch.randn(G, nb, kb + 2, generator=g, device="cuda")
            xd = self.x[:, :K].double() * self.xs[:, :kb].double().repeat_interleave(128, 1)[:, :K]
            wd = self.w[:, :, :K].double() * self.ws[:, :, :kb].double().repeat_interleave(128, 1)[:, :N].repeat_interleave(
                128, 2)[:, :, :K]
        else:
            ld = up(K, 8)
            self.x = torch.full((M, ld), float("nan"), device="cuda", dtype=kind)
            self.w = torch.full((G, N, ld), float("nan"), device="cuda", dtype=kind)
            self.x[:, :K], self.w[:, :, :K] = x.to(kind), w.to(kind)
            xd, wd = self.x[:, :K].double(), self.w[:, :, :K].double()
        self.bias = torch.randn(G, N, generator=g, device="cuda") if bias else None
        off = np.cumsum([first] + list(counts or [M]))
        self.off = torch.tensor(off, dtype=torch.int32, device="cuda")
        self.ref = torch.zeros(M, N, dtype=torch.float64, device="cuda")
        self.tol = torch.zeros_like(self.ref)
        self.used = torch.zeros(M, dtype=torch.bool, device="cuda")
        unit = (K + 2 * kb + 8) * 2.0 ** -23
        for e in range(G):
            lo, hi = int(off[e]), int(off[e + 1])
            self.used[lo:hi] = True
            self.ref[lo:hi] = xd[lo:hi] @ wd[e].T
            mag = xd[lo:hi].abs() @ wd[e].abs().T
            if bias:
                self.ref[lo:hi] += self.bias[e].double()
                mag = mag + self.bias[e].abs().double()
            self.tol[lo:hi] = unit * mag

    def call(self, y, accumulate=0, act=0, st=None, off=None):
        x, w, b = self.x, self.w, ptr(self.bias)
        st = stream() if st is None else st
        tail = (self.M, self.N, self.K, x.stride(0), w.stride(1))
        if self.kind != "e4m3":
            return tb.lib.tsfm_kernel_linear_grouped(
                ptr(x), CODE[x.dtype], ptr(w), CODE[w.dtype], b, ptr(y), CODE[y.dtype], accumulate, act,
                ptr(self.off if off is None else off), self.groups, *tail, w.stride(0), y.stride(0), st)
        scales = (ptr(self.xs), self.xs.stride(0), ptr(w), ptr(self.ws), self.ws.stride(1))
        if self.counts is None:
            return tb.lib.tsfm_kernel_linear_e4m3(ptr(x), *scales, b, ptr(y), CODE[y.dtype], accumulate, act, *tail,
                                                  y.stride(0), st)
        return tb.lib.tsfm_kernel_linear_grouped_e4m3(
            ptr(x), *scales, self.ws.stride(0), b, ptr(y), CODE[y.dtype], accumulate, act,
            ptr(self.off if off is None else off), self.groups, *tail, w.stride(0), y.stride(0), st)

    def check(self, dtype=torch.float32, act=0, accumulate=0, pad=0, shift=0):
        """One call; `pad` extra columns per row and `shift` elements before the first (alignment)."""
        cols = self.N // 2 if act == 3 else self.N
        flat = torch.full((self.M * (cols + pad) + shift,), -5.0, device="cuda", dtype=dtype)
        y = flat[shift:].view(self.M, cols + pad)
        before = y.clone()
        tb.check(self.call(y, accumulate, act))
        torch.cuda.synchronize()
        ref, tol = self.ref, self.tol
        if accumulate:
            ref, tol = ref - 5.0, tol + 5.0 * 2.0 ** -23
        if act == 1:
            ref = ref.clamp(min=0)
        if act == 3:
            # g silu(u): |silu| <= |u|, |silu'| < 1.1; exp and division within 64 units of 2^-23
            # for |u| < 40, and the product rounds once.
            p, t = ref.view(self.M, -1, 2, 128), tol.view(self.M, -1, 2, 128)
            gg, u = p[:, :, 0], p[:, :, 1]
            ref = gg * torch.nn.functional.silu(u)
            tol = (t[:, :, 0] * (u.abs() + t[:, :, 1]) + 1.1 * t[:, :, 1] * gg.abs() + 66 * 2.0 ** -23 * ref.abs())
            ref, tol = ref.reshape(self.M, cols), tol.reshape(self.M, cols)
            tol = tol + 1e-30
        out = y[:, :cols].double()
        tol = tol + torch.finfo(dtype).eps / 2 * (ref.abs() + tol) + torch.finfo(dtype).smallest_normal
        # At and past 65504 + 16 (half a step above its largest number) F16 rounds to infinity: a sum
        # surely past it is infinite, one surely below it finite, one within its tolerance of it either.
        edge = 65520.0 if dtype == torch.float16 else float("inf")
        over = ref.abs() - tol >= edge
        bad = torch.where(over, out != torch.copysign(torch.full_like(ref, float("inf")), ref),
                          ~((out - ref).abs() <= tol) & ~(torch.isinf(out) & (ref.abs() + tol >= edge)))
        bad &= self.used[:, None]
        assert not bad.any(), (int(bad.sum()), (out - ref).abs()[self.used].max().item())
        assert torch.equal(y[~self.used], before[~self.used])
        assert torch.equal(y[:, cols:], before[:, cols:])
        assert (flat[:shift] == -5.0).all()


DENSE = [(1, 64, 64), (1, 768, 768), (2, 1000, 1032), (7, 1, 1), (33, 129, 127), (77, 65, 129), (128, 256, 128),
         (129, 257, 130), (300, 336, 1000), (640, 2304, 768), (1000, 192, 384)]


@pytest.mark.parametrize("M,N,K", DENSE)
def test_linear_e4m3(M, N, K):
    Case(M, N, K, "e4m3", bias=True).check(torch.float32)
    c = Case(M, N, K, "e4m3", seed=1)
    c.check(torch.bfloat16, act=1)
    c.check(torch.float16, pad=8)


# Tile widths by the size of the product: 64 columns with K shared by 2 to 8 CTAs of a cluster (long K,
# few tiles; rows and columns that end inside a tile, a K that its CTAs share unevenly), 128 columns,
# and 256 x 256 on pairs of SMs, with full and ragged edges.
WIDTHS = [(1, 1024, 4096), (3, 500, 8200), (130, 1000, 2050), (200, 70, 2176), (256, 512, 6000), (2048, 768, 768),
          (2100, 1030, 520), (6000, 2500, 2100), (4096, 4096, 1024), (9000, 2304, 392)]


@pytest.mark.parametrize("M,N,K", WIDTHS)
def test_linear_e4m3_tile_widths(M, N, K):
    c = Case(M, N, K, "e4m3", bias=True, seed=3)
    c.check(torch.float32)
    c.check(torch.float16, act=1)
    c.check(torch.bfloat16, pad=8)    # rows of 16-byte multiples
    c.check(torch.bfloat16, pad=3, shift=1)
    c.check(accumulate=1, act=1)


@pytest.mark.parametrize("M,N,K", [(2, 512, 4096), (300, 512, 2048), (8000, 2048, 1024)])
def test_linear_e4m3_gated_tile_widths(M, N, K):
    c = Case(M, N, K, "e4m3", seed=4)
    k = 0.5 / float(c.ref.std())
    c.xs *= k
    c.ref, c.tol = c.ref * k, 1.1 * c.tol * k
    c.check(torch.bfloat16, act=3)
    c.check(torch.float16, act=3, pad=2)


@pytest.mark.parametrize("kind", ["e4m3", torch.bfloat16, torch.float16], ids=str)
def test_grouped_wide_tiles(kind):
    # groups of many rows on 256 x 256 tiles, some of few, some that end one row into a tile
    counts = [3000, 0, 257, 2048, 1, 1500, 255, 4097]
    c = Case(sum(counts) + 7, 1100, 1030, kind, counts=counts, first=5, bias=True)
    c.check(torch.bfloat16, act=1)
    c.check(torch.float32, pad=4)
    c.check(torch.float16, pad=1, shift=1)
    c.check(torch.float32, accumulate=1)
    g = Case(sum(counts), 1024, 640, kind, counts=counts)
    if kind == "e4m3":
        k = 0.5 / float(g.ref.std())
        g.xs *= k
        g.ref, g.tol = g.ref * k, 1.1 * g.tol * k
    g.check(torch.float16 if kind == "e4m3" else kind, act=3)


# Few rows per group: W's rows as the matrix instruction's, 32 rows of x its columns. Tiles of all four
# units and of one to three (N 100, 129), K of one block, a ragged quad of blocks and many quads, groups
# of up to 8 rows, of more, and of more than one tile. Two-byte operands take this way with more tiles
# than SMs only (groups x N / 128 > 148: the last three).
FEW = [([1], 64, 64), ([1, 0, 2, 0, 0, 1], 100, 200), ([8, 0, 9, 1, 0, 0, 0], 129, 640), ([0] * 20 + [33, 0, 70], 384, 1300),
       ([2, 1] * 20, 512, 520), ([0, 1, 3, 0] * 16, 1000, 72), ([1] * 60 + [40, 31, 32], 400, 2056)]


@pytest.mark.parametrize("kind", ["e4m3", torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("counts,N,K", FEW, ids=[f"{sum(c)}r{len(c)}g{N}" for c, N, K in FEW])
def test_grouped_few_rows(kind, counts, N, K):
    c = Case(sum(counts) + 3, N, K, kind, counts=counts, first=1, bias=True, seed=5)
    c.check(torch.float32)
    c.check(torch.bfloat16, act=1)
    c.check(torch.float16, pad=3, shift=1)
    c.check(accumulate=1, act=1)


@pytest.mark.parametrize("kind", ["e4m3", torch.bfloat16, torch.float16], ids=str)
def test_grouped_few_rows_gated(kind):
    for counts, N, K in (([1, 0, 7], 256, 100), ([1, 2] * 40 + [39], 512, 700)):
        c = Case(sum(counts) + 2, N, K, kind, counts=counts, first=2, seed=6)
        if kind == "e4m3":
            k = 0.5 / float(c.ref[c.used].std())
            c.xs *= k
            c.ref, c.tol = c.ref * k, 1.1 * c.tol * k  # the scales round again
        c.check(torch.float16 if kind == "e4m3" else kind, act=3)
        c.check(torch.bfloat16, act=3, pad=1)


@pytest.mark.parametrize("M,N,K", [(1, 33, 1), (3, 300, 1024), (8, 5000, 130), (8, 2304, 768)])
def test_linear_e4m3_few_rows(M, N, K):
    c = Case(M, N, K, "e4m3", bias=True, seed=7)
    c.check(torch.float32, pad=5)
    c.check(torch.bfloat16, act=1)
    g = Case(M, up(N, 256), K, "e4m3", seed=8)
    if K > 1:
        k = 0.5 / float(g.ref.std())
        g.xs *= k
        g.ref, g.tol = g.ref * k, 1.1 * g.tol * k
    g.check(torch.float16, act=3)


def test_few_rows_bad_offsets_stay_inside():
    # negative, falling and far offsets: read as the clamped, nondecreasing ones
    M = 20
    c = Case(M, 96, 200, "e4m3", counts=[6, 0, 14, 0])
    off = torch.tensor([-50, 6, 4, 2 ** 31 - 1, 3], dtype=torch.int32, device="cuda")
    a, b = torch.full((M + 64, 96), 3.0, device="cuda"), torch.full((M + 64, 96), 3.0, device="cuda")
    tb.check(c.call(a))
    tb.check(c.call(b, off=off))
    torch.cuda.synchronize()
    assert torch.equal(a, b) and (a[:M] != 3.0).any() and (b[M:] == 3.0).all()


def test_few_rows_nonfinite_values():
    # a row of NaN beside others of its tile, an infinite scale, a weight block of NaN scale: only what
    # they belong to shows them
    c = Case(12, 256, 512, "e4m3", counts=[5, 0, 7], seed=9)
    c.x[2, 7] = float("nan")
    c.xs[6, 1] = float("inf")
    c.ws[2, 1, 0] = float("nan")  # columns 128.. of the last group
    y = torch.zeros(12, 256, device="cuda")
    tb.check(c.call(y))
    torch.cuda.synchronize()
    ok = ((y.double() - c.ref).abs() <= c.tol + (c.ref.abs() + c.tol) * 2.0 ** -24)
    assert torch.isnan(y[2]).all() and not torch.isfinite(y[6]).any()
    assert torch.isnan(y[5:, 128:]).all()
    assert ok[[0, 1, 3, 4]].all() and ok[[5, 7, 8, 9, 10, 11]][:, :128].all()



def test_linear_e4m3_offsets_past_32_bits():
    # y of more than 2^31 elements and x of more than 2^31 bytes: the last rows and columns
    M, N, K = 140000, 16384, 16400
    g = gen(9)
    x = torch.zeros(M, K, device="cuda", dtype=torch.uint8)
    w = torch.zeros(N, K, device="cuda", dtype=torch.uint8)
    x[-3:] = 0x38  # 1.0
    w[-2:] = 0x40  # 2.0
    kb, nb = -(-K // 128), N // 128
    xs, ws = torch.ones(M, kb, device="cuda"), torch.full((nb, kb), 0.5, device="cuda")
    y = torch.full((M, N), 7.0, device="cuda", dtype=torch.bfloat16)
    tb.check(tb.lib.tsfm_kernel_linear_e4m3(ptr(x), ptr(xs), kb, ptr(w), ptr(ws), kb, None, ptr(y), 2, 0, 0, M, N, K, K, K,
                                            N, stream()))
    torch.cuda.synchronize()
    # 16400 ones times 2 times 0.5, rounded to bf16
    assert (y[-3:, -2:] == torch.tensor(16400.0).bfloat16().item()).all()
    assert (y[-3:, :-2] == 0).all() and (y[:-3] == 0).all()
    del x, w, y, xs, ws, g
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M,N,K", [(1, 256, 100), (50, 512, 768), (300, 1024, 320), (2000, 2048, 1024)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_linear_e4m3_gated(M, N, K, dtype):
    c = Case(M, N, K, "e4m3")
    # bring the sums near one, where the gate bends
    k = 0.5 / c.ref.std()
    c.xs *= float(k)
    c.ref, c.tol = c.ref * float(k), 1.1 * c.tol * float(k)  # the scales round again
    c.check(dtype, act=3)


@pytest.mark.parametrize("M,N,K", [(1, 96, 200), (200, 300, 400), (1500, 512, 256)])
def test_linear_e4m3_accumulate_and_strides(M, N, K):
    c = Case(M, N, K, "e4m3", bias=True)
    c.check(accumulate=1)
    c.check(accumulate=1, act=1)
    c.check(accumulate=1, pad=3)          # rows that are not 16-byte aligned
    c.check(torch.bfloat16, pad=1)
    c.check(torch.float16, pad=8, shift=1)


COUNTS = [
    [5], [0, 0, 3], [1, 1, 1, 1], [0, 130, 0, 7, 64, 0], [128, 256, 1], [33, 0, 0, 0, 95, 127, 129],
    [0] * 40 + [3] + [0] * 60 + [200, 1], [300, 5, 700, 0, 1000],
]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}g{sum(c)}")
@pytest.mark.parametrize("kind", ["e4m3", torch.bfloat16, torch.float16], ids=str)
def test_grouped(counts, kind):
    for N, K, first, tail in ((72, 200, 0, 0), (384, 264, 3, 5)):
        c = Case(sum(counts) + first + tail, N, K, kind, counts=counts, first=first, bias=True)
        c.check(torch.float32)
        c.check(torch.bfloat16, act=1, pad=4)
        c.check(torch.float32, accumulate=1)
    Case(sum(counts), 512, 128, kind, counts=counts).check(torch.float16 if kind == "e4m3" else kind, pad=8)


@pytest.mark.parametrize("kind", ["e4m3", torch.bfloat16], ids=str)
def test_grouped_gated(kind):
    counts = [3, 0, 200, 129, 1]
    c = Case(sum(counts) + 4, 768, 320, kind, counts=counts, first=2)
    k = 0.5 / float(c.ref[c.used].std())
    if kind == "e4m3":
        c.xs *= k
        c.ref, c.tol = c.ref * k, 1.1 * c.tol * k
        c.check(torch.bfloat16, act=3)
    else:
        c.check(kind, act=3)


@pytest.mark.parametrize("kind", ["e4m3", torch.float16], ids=str)
def test_grouped_many_groups(kind):
    # 1024 groups, most of them empty, and one group of everything
    counts = [0] * 1024
    for i in (0, 1, 31, 32, 500, 1022, 1023):
        counts[i] = 1 + i % 37
    Case(sum(counts), 64, 64, kind, counts=counts).check()
    Case(777, 64, 64, kind, counts=[777]).check()


def test_grouped_without_rows():
    c = Case(9, 64, 64, torch.float16, counts=[0, 0, 0], first=4)
    c.check()


@pytest.mark.parametrize("kind", ["e4m3", torch.bfloat16], ids=str)
def test_bad_offsets_stay_inside(kind):
    # negative, falling and far offsets: read as the clamped, nondecreasing ones
    M = 300
    c = Case(M, 96, 128, kind, counts=[100, 0, 200, 0])
    off = torch.tensor([-50, 100, 40, 2 ** 31 - 1, 17], dtype=torch.int32, device="cuda")
    a, b = torch.full((M + 64, 96), 3.0, device="cuda"), torch.full((M + 64, 96), 3.0, device="cuda")
    tb.check(c.call(a))
    tb.check(c.call(b, off=off))
    torch.cuda.synchronize()
    assert torch.equal(a, b) and (b[M:] == 3.0).all()


@pytest.mark.parametrize("kind", ["e4m3", torch.float16], ids=str)
def test_nonfinite_values_stay_in_their_rows(kind):
    counts = [40, 0, 100, 20]
    c = Case(160, 128, 256, kind, counts=counts)
    clean = torch.zeros(160, 128, device="cuda")
    tb.check(c.call(clean))
    c.x[45, 7] = float("nan")
    if kind == "e4m3":
        c.xs[139, 1] = float("inf")
    else:
        c.x[139, 200] = float("inf")
    y = torch.zeros_like(clean)
    tb.check(c.call(y))
    torch.cuda.synchronize()
    keep = torch.ones(160, dtype=torch.bool, device="cuda")
    keep[[45, 139]] = False
    assert torch.equal(y[keep], clean[keep])
    assert torch.isnan(y[45]).all() and not torch.isfinite(y[139]).any()


@pytest.mark.parametrize("kind", ["e4m3", torch.bfloat16], ids=str)
def test_streams_graphs_and_repeats(kind):
    counts = [100, 3, 0, 400]
    c = Case(503, 320, 384, kind, counts=counts, bias=True)
    want = torch.zeros(503, 320, device="cuda")
    tb.check(c.call(want))
    torch.cuda.synchronize()
    # two calls at once on two streams
    ss = [torch.cuda.Stream() for _ in range(2)]
    ys = [torch.zeros_like(want) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, y in zip(ss, ys):
            tb.check(c.call(y, st=s.cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in ys)
    # captured, and replayed with other offsets and rows in the same buffers
    y = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        tb.check(c.call(y))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    c.off.copy_(torch.tensor([10, 10, 400, 401, 500], dtype=torch.int32))
    want2 = torch.full_like(want, 2.0)
    tb.check(c.call(want2))
    y.fill_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want2) and (y[:10] == 2.0).all() and (y[500:] == 2.0).all()


def test_feed_forward_chain():
    """A mixture layer's feed-forward as it is used: rows sorted by expert, quantised, through the
    gated up product, quantised again, through the down product, against float64 on the same codes."""
    counts, K, F, N = [70, 0, 300, 1, 129], 256, 512, 192
    M, G = sum(counts), len(counts)
    g = gen(5)
    x = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    up_w = torch.randn(G * 2 * F, K, generator=g, device="cuda") * K ** -0.5
    down_w = torch.randn(G * 256, F, generator=g, device="cuda") * F ** -0.5  # N = 192 rows of 256 used
    uq, us = quantize(up_w, 128)
    dq, ds = quantize(down_w, 128)
    off = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device="cuda")
    xq, xs = quantize(x, 1)
    h = torch.zeros(M, F, device="cuda", dtype=torch.bfloat16)
    tb.check(tb.lib.tsfm_kernel_linear_grouped_e4m3(
        ptr(xq), ptr(xs), xs.stride(0), ptr(uq), ptr(us), us.stride(0), us.stride(0) * (2 * F // 128), None, ptr(h), 2, 0, 3,
        ptr(off), G, M, 2 * F, K, K, K, 2 * F * K, F, stream()))
    hq, hs = quantize(h, 1)
    y = torch.zeros(M, N, device="cuda")
    tb.check(tb.lib.tsfm_kernel_linear_grouped_e4m3(
        ptr(hq), ptr(hs), hs.stride(0), ptr(dq), ptr(ds), ds.stride(0), ds.stride(0) * 2, None, ptr(y), 0, 0, 0,
        ptr(off), G, M, N, F, F, F, 256 * F, N, stream()))
    torch.cuda.synchronize()

    def val(q, s, br):
        s = s.double().repeat_interleave(br, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, : q.shape[1]]
        return q.view(E4M3).double() * s
    xv, uv, dv, hv = val(xq, xs, 1), val(uq, us, 128), val(dq, ds, 128), val(hq, hs, 1)
    for e in range(G):
        lo, hi = int(off[e]), int(off[e + 1])
        p = (xv[lo:hi] @ uv[e * 2 * F:(e + 1) * 2 * F].T).view(hi - lo, F // 128, 2, 128)
        want = (p[:, :, 0] * torch.nn.functional.silu(p[:, :, 1])).reshape(hi - lo, F)
        # bf16's half step, and FP32 sums of 256 terms whose magnitudes stay below 64
        assert ((h[lo:hi].double() - want).abs() <= 2.0 ** -8 * want.abs() + 300 * 2.0 ** -23 * 64).all()
        w = dv[e * 256:e * 256 + N]
        tol = 540 * 2.0 ** -23 * (hv[lo:hi].abs() @ w.abs().T) + 1e-30
        assert ((y[lo:hi].double() - hv[lo:hi] @ w.T).abs() <= tol).all()
    # quantising is off by at most half an E4M3 step of the block's grid
    assert ((xv - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * xs.double().repeat_interleave(128, 1)).all()


@pytest.mark.parametrize("M", [5, 60, 400, 3000])
def test_gated_nan_stays_in_its_column(M):
    # one weight of g and one of u are NaN: their output columns are, the ones beside them not; and u far
    # below zero, where the gate's exponential leaves FP32
    N, K = 1024, 256
    c = Case(M, N, K, "e4m3", seed=11)
    k = 0.5 / float(c.ref.std())
    c.xs *= k
    c.ref, c.tol = c.ref * k, 1.1 * c.tol * k
    c.check(torch.bfloat16, act=3)
    y0 = torch.zeros(M, N // 2, device="cuda", dtype=torch.bfloat16)
    y1 = torch.zeros_like(y0)
    tb.check(c.call(y0, act=3))
    torch.cuda.synchronize()
    c.w[0, 20, 3] = float("nan")            # g of column 20
    c.w[0, 256 + 128 + 71, 9] = float("nan")  # u of column 128 + 71
    tb.check(c.call(y1, act=3))
    torch.cuda.synchronize()
    hit = torch.zeros(N // 2, dtype=torch.bool, device="cuda")
    hit[[20, 199]] = True
    assert torch.isnan(y1[:, hit]).all() and torch.equal(y1[:, ~hit], y0[:, ~hit])
    # u = -3e4 in column 5 (one weight row of -448, an x of 448 in its place): g silu(u) is 0 to within
    # 3e4 * 2^-60 of |g|
    d = Case(M, N, K, "e4m3", seed=12)
    d.x.zero_()
    d.x[:, 0] = 448.0
    d.w.zero_()
    d.w[0, :128, 0] = 1.0
    d.w[0, 128:256, 0] = 1.0
    d.w[0, 128 + 5, 0] = -448.0
    d.xs.fill_(1 / 448.0)
    d.ws.fill_(1.0)
    d.ws[0, 1, 0] = 70.0  # u = 70, and -31360 in column 5; g = 1
    tb.check(d.call(y1, act=3))
    torch.cuda.synchronize()
    assert (y1[:, :5] == 70.0).all() and (y1[:, 6:128] == 70.0).all() and (y1[:, 128:] == 0).all()
    assert (y1[:, 5].float().abs() <= 31360 * 2.0 ** -60).all()


@pytest.mark.parametrize("M", [5, 300, 3000])
def test_back_to_back_calls_see_their_predecessors(M):
    # Calls that read what the call before wrote and overwrite what it read, without a pause between
    # them, eager and captured, against the same calls one at a time.
    G, D = 4, 512
    g = gen(M)
    wq, ws = quantize(torch.randn(G * D, D, generator=g, device="cuda") * 1.4 * D ** -0.5, 128)
    w16 = (torch.randn(G, D, D, generator=g, device="cuda") * 1.4 * D ** -0.5).bfloat16()
    off = torch.tensor([0, M // 3, M // 3, M - 1, M], dtype=torch.int32, device="cuda")
    h0 = torch.randn(M, D, generator=g, device="cuda").bfloat16()
    bias = torch.randn(G, D, generator=g, device="cuda")
    q, s = torch.zeros(M, D, dtype=torch.uint8, device="cuda"), torch.zeros(M, D // 128, device="cuda")
    h, total = torch.zeros_like(h0), torch.zeros(M, D, device="cuda")

    def steps(pause):
        st = stream()
        for i in range(6):
            tb.check(tb.lib.tsfm_kernel_quantize_e4m3(ptr(h), CODE[h.dtype], M, D, D, 1, ptr(q), D, ptr(s), D // 128, st))
            pause()
            tb.check(tb.lib.tsfm_kernel_linear_grouped_e4m3(
                ptr(q), ptr(s), D // 128, ptr(wq), ptr(ws), D // 128, (D // 128) ** 2, ptr(bias), ptr(h), CODE[h.dtype], 0, 1,
                ptr(off), G, M, D, D, D, D, D * D, D, st))
            pause()
            tb.check(tb.lib.tsfm_kernel_linear_grouped(
                ptr(h), CODE[h.dtype], ptr(w16), CODE[w16.dtype], None, ptr(total), CODE[total.dtype], 1, 0, ptr(off), G, M, D,
                D, D, D, D * D, D, st))
            pause()
            tb.check(tb.lib.tsfm_kernel_linear_e4m3(ptr(q), ptr(s), D // 128, ptr(wq), ptr(ws), D // 128, None, ptr(h),
                                                    CODE[h.dtype], 0, 0, M, D, D, D, D, D, st))
            pause()

    def run(how):
        h.copy_(h0)
        total.zero_()
        how()
        torch.cuda.synchronize()
        return h.clone(), total.clone(), q.clone(), s.clone()

    want = run(lambda: steps(torch.cuda.synchronize))
    assert torch.isfinite(want[1]).all() and want[1].abs().max() > 0
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        steps(lambda: None)
    for _ in range(10):
        for got in (run(lambda: steps(lambda: None)), run(graph.replay)):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
