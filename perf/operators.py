"""Workloads of the 8-bit block-scaled and the grouped products: what a caller hands over, the plain
form of each operator in elementary torch operations, and the calls into tsfm_b200.

Operators (`op` of a case):
  quantize        x [rows, cols] -> E4M3 values and one FP32 scale per block of block_rows x 128
  linear_e4m3     y = act((xq sx) (wq sw)^T + bias) on such operands
  grouped         y[r] = act(x[r] W[e]^T + bias[e]) for the rows r of expert e, 16-bit operands
  grouped_e4m3    the same on block-scaled 8-bit operands
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
E4M3 = torch.float8_e4m3fn
ACTS = {"none": 0, "relu": 1, "gated": 3}

_library = None


def _tb():
    """The package of this repository, on first use."""
    global _library
    if _library is None:
        path = os.path.join(os.getcwd(), "tsfm-zig_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import tsfm_b200
        _library = tsfm_b200
    return _library


# ---- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # One series' token before its first product, and a forecast batch's activations
        # (64 series of 577 tokens).
        dict(name="quantize_token", op="quantize", rows=1, cols=768, x="bf16", block_rows=1),
        dict(name="quantize_activations", op="quantize", rows=36928, cols=2048, x="bf16", block_rows=1),
        # A checkpoint's FP32 feed-forward matrix, laid out once per load.
        dict(name="quantize_weight", op="quantize", rows=4096, cols=1024, x="f32", block_rows=128),
        # One token through a QKV product, a ragged handful of rows, a batch of 128 series of 577
        # tokens, and the gated feed-forward of 64 series of 130 tokens.
        dict(name="linear_one_row", op="linear_e4m3", M=1, N=2304, K=768, y="bf16", act="none", bias=True),
        dict(name="linear_ragged", op="linear_e4m3", M=77, N=1000, K=1032, y="f32", act="relu", bias=True),
        dict(name="linear_batch", op="linear_e4m3", M=73856, N=2304, K=768, y="f16", act="none", bias=False),
        dict(name="linear_gated", op="linear_e4m3", M=8320, N=8192, K=1024, y="bf16", act="gated", bias=False),
        # Sixteen tokens that each went to two of 32 experts; a batch over 8 domain heads; the
        # gated half of a mixture layer over a long batch.
        dict(name="grouped_tokens", op="grouped", M=32, N=2048, K=1024, groups=32, x="bf16", y="bf16", act="none",
             bias=True, tail=0),
        dict(name="grouped_heads", op="grouped", M=5000, N=672, K=768, groups=8, x="f16", y="f32", act="none",
             bias=True, tail=8),
        dict(name="grouped_layer", op="grouped", M=32768, N=4096, K=1024, groups=32, x="bf16", y="bf16",
             act="gated", bias=False, tail=0),
        dict(name="grouped_e4m3_tokens", op="grouped_e4m3", M=32, N=2048, K=1024, groups=32, x="e4m3", y="bf16",
             act="none", bias=True, tail=0),
        dict(name="grouped_e4m3_layer", op="grouped_e4m3", M=32768, N=4096, K=1024, groups=32, x="e4m3", y="bf16",
             act="gated", bias=False, tail=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "linear_e4m3", "linear_e4m3", "grouped", "grouped_e4m3"])
    if op == "quantize":
        block = rng.choice([1, 1, 128])
        cols = _log(rng, 64, 8192)
        return dict(op=op, rows=_log(rng, 1, min(36928, 75_000_000 // cols)), cols=cols,
                    x=rng.choice(["bf16", "f16", "f32"]), block_rows=block)
    act = rng.choice(["none", "none", "relu", "gated"])
    K = _log(rng, 64, 4096)
    N = 256 * _log(rng, 1, 32) if act == "gated" else _log(rng, 64, 8192)
    y = rng.choice(["bf16", "f16"] if act == "gated" else ["bf16", "f16", "f32"])
    M = _log(rng, 1, max(1, min(73856, 100_000_000_000 // (N * K))))
    case = dict(op=op, M=M, N=N, K=K, y=y, act=act, bias=act != "gated" and rng.random() < 0.5)
    if op != "linear_e4m3":
        case["groups"] = min(_log(rng, 1, 64), max(1, 200_000_000 // (N * K)))
        case["M"] = min(M, 32768)
        case["x"] = rng.choice(["bf16", "f16"]) if op == "grouped" else "e4m3"
        case["tail"] = rng.choice([0, 0, case["M"] // 10])
    return case


# ---- inputs -----------------------------------------------------------------------------------

def _active(case):
    """Experts with rows."""
    return min(case["M"] - case["tail"], -(-3 * case["groups"] // 4))


def _up(n, m):
    return -(-n // m) * m


def _activations(gen, rows, cols):
    """Normal values with a few loud columns and rows of their own size, as a residual stream has."""
    dev = "cuda"
    x = torch.randn(rows, cols, generator=gen, device=dev)
    col = torch.exp(0.5 * torch.randn(cols, generator=gen, device=dev))
    row = torch.exp(0.3 * torch.randn(rows, 1, generator=gen, device=dev))
    return x * col * row


def _spread(v, block_rows, rows, cols):
    """Block scales laid out over the elements of a [..., rows, cols] matrix."""
    r = torch.arange(rows, device=v.device) // block_rows
    c = torch.arange(cols, device=v.device) // 128
    return v[..., r, :][..., c]


def _block_scale(x, block_rows):
    """The scale of each block: the smallest power of two with |x| / scale <= 448."""
    rows, cols = x.shape[-2:]
    pad = torch.nn.functional.pad(x.abs(), (0, _up(cols, 128) - cols, 0, _up(rows, block_rows) - rows))
    amax = pad.unflatten(-1, (-1, 128)).unflatten(-3, (-1, block_rows)).amax((-1, -3))
    mant, expo = torch.frexp(amax)  # amax = mant * 2^expo, mant in [0.5, 1)
    expo = expo - torch.where(mant <= 0.875, 9, 8).to(expo.dtype)
    scale = torch.ldexp(torch.ones_like(amax), expo.clamp(min=-126))
    scale = torch.where(amax == 0, torch.full_like(amax, 2.0 ** -126), scale)
    return torch.where(torch.isfinite(amax), scale, torch.full_like(amax, float("nan")))


def _round_e4m3(v):
    """Round to nearest even on the E4M3 grid (3 mantissa bits, exponents from -6, subnormals 2^-9)."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp(min=-9))
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _quantized(x, block_rows):
    """Operands of a product: E4M3 codes in rows padded to 16 bytes, and scales."""
    scale = _block_scale(x, block_rows)
    q = _round_e4m3(x / _spread(scale, block_rows, *x.shape[-2:]))
    buf = torch.zeros(*x.shape[:-1], _up(x.shape[-1], 16), device=x.device, dtype=E4M3)
    buf[..., :x.shape[-1]] = q.to(E4M3)
    return buf, scale


def _padded(x, dtype):
    """16-bit operands in rows padded to 16 bytes."""
    buf = torch.zeros(*x.shape[:-1], _up(x.shape[-1], 8), device=x.device, dtype=dtype)
    buf[..., :x.shape[-1]] = x.to(dtype)
    return buf


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    dev = "cuda"
    st = {"case": dict(case)}
    if case["op"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        st["x"] = _activations(gen, rows, cols).to(DTYPES[case["x"]])
        st["q"] = torch.empty(rows, cols, device=dev, dtype=E4M3)
        st["scale"] = torch.empty(-(-rows // case["block_rows"]), -(-cols // 128), device=dev)
        return st
    M, N, K = case["M"], case["N"], case["K"]
    groups = case.get("groups", 1)
    x = _activations(gen, M, K)
    w = torch.randn(groups, N, K, generator=gen, device=dev) * K ** -0.5
    if case["op"] == "grouped":
        st["x"], st["w"] = _padded(x, DTYPES[case["x"]]), _padded(w, DTYPES[case["x"]])
    else:
        st["x"], st["xs"] = _quantized(x, 1)
        st["w"], st["ws"] = _quantized(w, 128)
    st["bias"] = torch.randn(groups, N, generator=gen, device=dev) if case["bias"] else None
    st["y"] = torch.zeros(M, N // 2 if case["act"] == "gated" else N, device=dev, dtype=DTYPES[case["y"]])
    if case["op"] != "linear_e4m3":
        # Rows per expert: uneven, a quarter of the experts (in no order) without any; the last `tail`
        # rows belong to none.
        used, active = M - case["tail"], _active(case)
        share = torch.rand(active, generator=gen, device=dev) ** 2 + 1e-3
        which = torch.multinomial(share, used, replacement=True, generator=gen)
        which[:active] = torch.arange(active, device=dev)  # one row at least
        expert = torch.randperm(groups, generator=gen, device=dev)[which]
        counts = torch.bincount(expert, minlength=groups)
        st["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        st["most"] = int(counts.max())  # the plan of the plain form: rows of the fullest expert
    return st


# ---- plain forms ------------------------------------------------------------------------------

def _plain_quantize(x, block_rows):
    x = x.float()
    scale = _block_scale(x, block_rows)
    return (x / _spread(scale, block_rows, *x.shape)).to(E4M3), scale


def _activate(y, act):
    if act == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if act == "gated":  # 256-column blocks [g (128) | u (128)]: g * u / (1 + e^-u)
        p = y.unflatten(-1, (-1, 2, 128))
        g, u = p[..., 0, :], p[..., 1, :]
        return (g * (u / (1 + torch.exp(-u)))).flatten(-2)
    return y


def _operands(st):
    case = st["case"]
    x, w = st["x"][:, :case["K"]].float(), st["w"][..., :case["K"]].float()
    if case["op"] != "grouped":
        x = x * _spread(st["xs"], 1, *x.shape[-2:])
        w = w * _spread(st["ws"], 128, *w.shape[-2:])
    return x, w


def _plain_linear(st):
    case = st["case"]
    x, w = _operands(st)
    y = x @ w[0].T
    if st["bias"] is not None:
        y = y + st["bias"][0]
    return _activate(y, case["act"]).to(st["y"].dtype)


def _plain_grouped(st):
    case = st["case"]
    x, w = _operands(st)
    off = st["offsets"].long()
    # Every expert's rows padded to the fullest one's, one batched product, and back.
    place = torch.arange(st["most"], device=x.device)
    row = off[:-1, None] + place
    have = row < off[1:, None]
    row = torch.where(have, row, torch.zeros_like(row))
    y = torch.bmm(x[row], w.transpose(1, 2))
    if st["bias"] is not None:
        y = y + st["bias"][:, None]
    out = st["y"].clone()
    out[row[have]] = _activate(y, case["act"]).to(out.dtype)[have]
    return out


# ---- one pass ---------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_pass(st):
    tb, case = _tb(), st["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "quantize":
        x, q, s = st["x"], st["q"], st["scale"]
        tb.check(tb.lib.tsfm_kernel_quantize_e4m3(_ptr(x), CODES[case["x"]], case["rows"], case["cols"], x.stride(0),
                                                  case["block_rows"], _ptr(q), q.stride(0), _ptr(s), s.stride(0),
                                                  stream))
        return {"q": q, "scale": s}
    x, w, y, bias = st["x"], st["w"], st["y"], st["bias"]
    M, N, K = case["M"], case["N"], case["K"]
    act = ACTS[case["act"]]
    if case["op"] == "linear_e4m3":
        tb.check(tb.lib.tsfm_kernel_linear_e4m3(
            _ptr(x), _ptr(st["xs"]), st["xs"].stride(0), _ptr(w), _ptr(st["ws"]), st["ws"].stride(1), _ptr(bias),
            _ptr(y), CODES[case["y"]], 0, act, M, N, K, x.stride(0), w.stride(1), y.stride(0), stream))
    elif case["op"] == "grouped":
        tb.check(tb.lib.tsfm_kernel_linear_grouped(
            _ptr(x), CODES[case["x"]], _ptr(w), CODES[case["x"]], _ptr(bias), _ptr(y), CODES[case["y"]], 0, act,
            _ptr(st["offsets"]), case["groups"], M, N, K, x.stride(0), w.stride(1), w.stride(0), y.stride(0), stream))
    else:
        tb.check(tb.lib.tsfm_kernel_linear_grouped_e4m3(
            _ptr(x), _ptr(st["xs"]), st["xs"].stride(0), _ptr(w), _ptr(st["ws"]), st["ws"].stride(1),
            st["ws"].stride(0), _ptr(bias), _ptr(y), CODES[case["y"]], 0, act, _ptr(st["offsets"]), case["groups"],
            M, N, K, x.stride(0), w.stride(1), w.stride(0), y.stride(0), stream))
    return {"y": y}


def run(state):
    if own:
        return _own_pass(state)
    case = state["case"]
    if case["op"] == "quantize":
        q, scale = _plain_quantize(state["x"], case["block_rows"])
        return {"q": q, "scale": scale}
    return {"y": _plain_linear(state) if case["op"] == "linear_e4m3" else _plain_grouped(state)}


# ---- what a pass cannot do without ------------------------------------------------------------

_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}


def work(case):
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        blocks = -(-case["rows"] // case["block_rows"]) * -(-case["cols"] // 128)
        return {"bytes": n * (_SIZE[case["x"]] + 1) + 4 * blocks, "flops": 2 * n}
    M, N, K = case["M"] - case.get("tail", 0), case["N"], case["K"]
    groups = _active(case) if "groups" in case else 1
    size = _SIZE[case.get("x", "e4m3")]
    scales = 0 if size > 1 else 4 * -(-K // 128) * (M + groups * -(-N // 128))
    cols = N // 2 if case["act"] == "gated" else N
    offsets = 4 * (case["groups"] + 1) if "groups" in case else 0
    bias = 4 * groups * N if case["bias"] else 0
    return {"bytes": size * K * (M + groups * N) + scales + bias + offsets + _SIZE[case["y"]] * M * cols,
            "flops": 2 * M * N * K}


# ---- the definition in 64 bits ----------------------------------------------------------------

def _exact_codes(x, block_rows):
    """Scales and E4M3 values block by block in double precision: the scale from a logarithm with its
    neighbours tried, the value from the distance to the two grid points around it."""
    rows, cols = x.shape
    big = torch.zeros(_up(rows, block_rows), _up(cols, 128), dtype=torch.float64, device=x.device)
    big[:rows, :cols] = x.double()
    tiles = big.reshape(big.shape[0] // block_rows, block_rows, big.shape[1] // 128, 128)
    amax = tiles.abs().amax((1, 3), keepdim=True)
    guess = torch.floor(torch.log2(amax.clamp(min=2.0 ** -140) / 448.0)) - 1
    for _ in range(3):
        guess = torch.where(amax > 448.0 * torch.exp2(guess), guess + 1, guess)
    scale = torch.exp2(guess.clamp(min=-126.0))
    v = (tiles / scale)
    grid = torch.arange(0, 127, device=x.device)  # codes of the non-negative finite values, in order
    m, e = (grid % 8).double(), (grid // 8).double()
    grid = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e - 10))
    a = v.abs().clamp(max=448.0).contiguous()
    hi = torch.searchsorted(grid, a.reshape(-1)).reshape(a.shape).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    q = torch.copysign(grid[code], v).reshape(big.shape)[:rows, :cols]
    return q, scale[:, 0, :, 0]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "quantize":
        q, scale = _exact_codes(st["x"], case["block_rows"])
        return {"q": q, "scale": scale}
    M, N, K = case["M"], case["N"], case["K"]
    x, w = st["x"][:, :K].double(), st["w"][:, :, :K].double()
    if "xs" in st:
        x = x * st["xs"].double().repeat_interleave(128, 1)[:, :K]
        w = w * st["ws"].double().repeat_interleave(128, 1)[:, :N].repeat_interleave(128, 2)[:, :, :K]
    off = st["offsets"].tolist() if "offsets" in st else [0, M]
    out = torch.zeros(M, st["y"].shape[1], dtype=torch.float64, device="cuda")
    for e in range(len(off) - 1):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        y = torch.einsum("mk,nk->mn", x[lo:hi], w[e])
        if st["bias"] is not None:
            y += st["bias"][e].double()
        if case["act"] == "relu":
            y.clamp_(min=0)
        elif case["act"] == "gated":
            t = y.reshape(hi - lo, N // 256, 256)
            y = (t[..., :128] * t[..., 128:] * torch.sigmoid(t[..., 128:])).reshape(hi - lo, N // 2)
        out[lo:hi] = y
    return {"y": out}
