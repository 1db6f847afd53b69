"""MXFP4 activations times MXFP4 weights on the GPU, against plain arithmetic in
64 bits.

Tolerances of a product: a block's sum is exact; a matrix instruction adds four
of them and the sum so far, each aligned to the largest, so it loses at most
half a step of fp32 for each of the five; K is split over up to eight waves, whose sums add
one rounding each, the bias one, and the output rounds once, by half a step of
its type.  All relative to the sum of magnitudes."""
import ctypes
import math

import pytest
import torch

from ftmoe import _native as nat
from ftmoe import quant
from ftmoe.kernel.fused_mxfp4_linear import fused_mxfp4_linear
from ftmoe.kernel.fused_w4a4_linear import fused_w4a4_expert_forward, fused_w4a4_linear
from ftmoe.kernel.fused_w4a4_moe import fused_w4a4_moe
from ftmoe.kernel.mxfp4_linear import dequantize_mxfp4_blocks
from ftmoe.kernel.w4a4_linear import quantize_mxfp4, w4a4_grouped_linear, w4a4_linear
from ftmoe.moe.token_sort import combine_tokens, sort_tokens

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
U = 2.0 ** -24
LUT = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the smallest step of a type's subnormals."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def roundings(K):
    return 5 * (K // 128 + 1) + 8 + 1


def far(got, ref, bound, dtype):
    """Whether |got - ref| exceeds the bound.  From half a step over the type's largest value
    on the right rounding is an infinity."""
    top = torch.finfo(dtype).max * (1 + half_step(dtype) / 2)
    over = (ref.abs() + bound >= top) & got.isinf() & (got.sign() == ref.sign())
    return ~((got.double() - ref).abs() <= bound) & ~over


def close(got, ref, mag, dtype, n):
    """|got - ref| within n fp32 roundings of `mag` and one of the output type."""
    assert got.shape == ref.shape and got.dtype == dtype
    err = (got.double() - ref).abs()
    bound = n * U * mag * (1 + half_step(dtype)) + half_step(dtype) * ref.abs() + tiny(dtype)
    bad = far(got, ref, bound, dtype)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} out of tolerance, worst {float((err - bound).max()):.3e}"


def two_to(n):
    return torch.ldexp(torch.ones_like(n, dtype=torch.float64).cpu(), n.cpu().to(torch.float64)).to(n.device)


def values(blocks, scales):
    """What blocks and scales stand for, in 64 bits."""
    lut = LUT.to(blocks.device)
    v = torch.stack((lut[(blocks & 15).long()], lut[(blocks >> 4).long()]), dim=-1).flatten(-2)
    table = torch.tensor([math.ldexp(1.0, i - 127) for i in range(255)] + [math.nan], dtype=torch.float64)
    return (v * table.to(blocks.device)[scales.long()].unsqueeze(-1)).flatten(-2)


def operand(shape, seed, dev, spread=6):
    """Random codes [..., K/32, 16] (every byte) and scales around 1."""
    g = torch.Generator(device=dev).manual_seed(seed)
    *lead, K = shape
    b = torch.randint(0, 256, (*lead, K // 32, 16), generator=g, device=dev, dtype=torch.int32).to(torch.uint8)
    s = torch.randint(127 - spread, 128 + spread, (*lead, K // 32), generator=g, device=dev, dtype=torch.int32)
    return b, s.to(torch.uint8)


def product(x, w, bias=None):
    """(x @ w.T + bias, magnitude) in 64 bits, from values."""
    y, mag = x @ w.t(), x.abs() @ w.abs().t()
    return (y, mag) if bias is None else (y + bias.double(), mag + bias.double().abs())


def act(name, g, u, alpha=1.702, limit=7.0):
    if name == "silu":
        return g * torch.sigmoid(g) * u
    if name == "gelu":
        return 0.5 * g * (1 + torch.erf(g / math.sqrt(2))) * u
    if name == "relu":
        return g.clamp_min(0) * u
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return (u + 1) * g * torch.sigmoid(alpha * g)


def gated_close(got, gu, mag, name, dtype, n, **kw):
    """act(gate) * up of sums that may be off by n roundings of mag: the largest change at the
    corners of that box, 16 roundings of fp32 for the activation (of gelu relative to g u: its
    1 + erf cancels; of swiglu_oai to g (u + 1) with its 1 not cancelled), one of the output.  Where
    1 + exp(-g) exceeds 2^126 its reciprocal is below fp32's normal numbers and becomes 0, so the
    result is off by less than 2^-126 of its factors."""
    e = n * U * mag
    (g, u), (eg, eu) = gu.chunk(2, dim=1), e.chunk(2, dim=1)
    ref = act(name, g, u, **kw)
    off = torch.zeros_like(ref)
    for a in (-1, 1):
        for b in (-1, 1):
            off = torch.maximum(off, (act(name, g + a * eg, u + b * eu, **kw) - ref).abs())
    size = ref.abs() + ((g * u).abs() if name == "gelu" else g.abs() if name == "swiglu_oai" else 0)
    bound = 2 * off + 16 * U * size + half_step(dtype) * ref.abs() + tiny(dtype) + g.abs() * (u.abs() + 1) * 2.0 ** -126
    bad = far(got, ref, bound, dtype)
    assert got.dtype == dtype and not bad.any(), f"{int(bad.sum())} of {bad.numel()} out of tolerance"


# ------------------------------------------------------------------ quantiser
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 64), (5, 96), (7, 2880), (300, 512), (2, 8192), (1, 16384), (129, 1056)])
def test_quantiser(gpu, dtype, rows, K):
    g = torch.Generator().manual_seed(rows * 31 + K)
    x = torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g).float())
    x = x.to(dtype)
    b, s = quantize_mxfp4(x.to(gpu))
    rb, rs = quant.quantize_mxfp4_blocks(x)
    assert b.shape == (rows, K // 32, 16) and torch.equal(s.cpu(), rs) and torch.equal(b.cpu(), rb)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_borders(gpu, dtype):
    """Every border between two codes, its neighbours in the type, both signs, under several
    scales; the largest of the block is 6 of the scale."""
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0])
    rows = []
    for e in (-8, -3, 0, 5, 12) if dtype == torch.float16 else (-40, -3, 0, 9, 100):
        for part in (borders[:8], borders[8:]):
            v = (part * 2.0 ** e).to(dtype)
            up = torch.nextafter(v, torch.full_like(v, math.inf)) if dtype == torch.float32 else (v.view(torch.int16) + 1).view(dtype)
            down = torch.where(v > 0, (v.view(torch.int32 if dtype == torch.float32 else torch.int16) - 1).view(dtype), v)
            row = torch.cat([v, up, down, -v, -down])
            row = row[row.abs().float() <= 6.0 * 2.0 ** e][:31]
            rows.append(torch.cat([row, row.new_zeros(31 - row.numel()), torch.tensor([6.0 * 2.0 ** e]).to(dtype)]))
            rows.append(-rows[-1])
    x = torch.stack(rows)
    b, s = quantize_mxfp4(x.to(gpu))
    rb, rs = quant.quantize_mxfp4_blocks(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(b.cpu(), rb)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_scales(gpu, dtype):
    """The block's largest at, before and after 6 2^e, zeros, and values below 1e-12."""
    tops = []
    for e in range(-12, 12):
        t = torch.tensor(6.0 * 2.0 ** e).to(dtype)
        i = t.view(torch.int32 if dtype == torch.float32 else torch.int16)
        tops += [t, (i - 1).view(dtype), (i + 1).view(dtype)]
    x = torch.zeros(len(tops), 32, dtype=dtype)
    x[:, 5] = torch.stack(tops)
    x[:, 6] = -x[:, 5] / 3
    x = torch.cat([x, torch.zeros(1, 32, dtype=dtype), torch.full((1, 32), 1e-13).to(dtype), torch.full((1, 32), -0.0).to(dtype)])
    b, s = quantize_mxfp4(x.to(gpu))
    # the least e with top <= 6 * 2^e, in whole numbers
    top = x.abs().amax(dim=1).double().clamp_min(float(torch.tensor(1e-12)))
    m, e = torch.frexp(top)
    want = torch.where(m <= 0.75, e - 3, e - 2) + 127
    assert torch.equal(s.cpu()[:, 0].int(), want.int())
    if dtype != torch.float32:  # (fp32: log2 rounds next to a power of two)
        rb, rs = quant.quantize_mxfp4_blocks(x)
        assert torch.equal(s.cpu(), rs) and torch.equal(b.cpu(), rb)


@pytest.mark.parametrize("e", [-40, -8, -1, 0, 1, 10, 40, 100])
def test_quantiser_fp32_above_the_largest_code(gpu, e):
    """fp32 maxima next to 6 2^e: the scale by whole numbers; the bytes of the torch function but in the few
    steps above, where its logarithm may round to e."""
    steps = torch.arange(-40, 41, dtype=torch.int32)
    x = torch.zeros(len(steps), 32)
    x[:, 5] = (torch.tensor(6.0 * 2.0 ** e).view(torch.int32) + steps).view(torch.float32)
    x[:, 9] = -x[:, 5] / 3
    b, s = (t.cpu() for t in quantize_mxfp4(x.to(gpu)))
    assert torch.equal(s[:, 0].int(), torch.where(steps > 0, e + 1, e).int() + 127)
    rb, rs = quant.quantize_mxfp4_blocks(x)
    same = (steps <= 0) | (steps > 33)
    assert torch.equal(s[same], rs[same]) and torch.equal(b[same], rb[same])
    assert (rs[~same] <= s[~same]).all()


def test_quantiser_fp32_next_to_ties(gpu):
    """fp32 has values one step over a border, which go up."""
    v = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    x = torch.cat([v, torch.nextafter(v, v + 1), torch.nextafter(v, v - 1), torch.zeros(10), torch.tensor([6.0])])[None]
    b, s = quantize_mxfp4(x.to(gpu))
    got = values(b, s)[0].cpu()
    low = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0]).double()
    high = torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]).double()
    assert torch.equal(got[:7], low) and torch.equal(got[7:14], high) and torch.equal(got[14:21], low)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_not_finite(gpu, dtype):
    x = torch.randn(6, 96, generator=torch.Generator().manual_seed(1)).to(dtype)
    clean_b, clean_s = quantize_mxfp4(x.to(gpu))
    x[1, 40], x[2, 0], x[4, 95] = math.inf, math.nan, -math.inf
    b, s = quantize_mxfp4(x.to(gpu))
    hit = torch.zeros(6, 3, dtype=torch.bool)
    hit[1, 1] = hit[2, 0] = hit[4, 2] = True
    hit = hit.to(gpu)
    assert (s[hit] == 255).all() and (b[hit] == 0).all()
    assert torch.equal(s[~hit], clean_s[~hit]) and torch.equal(b[~hit], clean_b[~hit])
    assert torch.equal(dequantize_mxfp4_blocks(b, s, out_dtype=torch.float32).isnan(), hit.repeat_interleave(32, dim=1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_layouts(gpu, dtype):
    """Rows apart, rows over one another, columns apart, odd addresses, more dimensions."""
    base = torch.randn(40, 600, generator=torch.Generator().manual_seed(3)).to(dtype).to(gpu)
    flat = base.reshape(-1)
    for x in (base[:, :512], base[:, 1:65], base[::3, 8:520], base.t()[:64, :32], base[:1].expand(5, 600)[:, :96],
              flat[1:1 + 64 * 5].view(5, 64), base[:, :96].reshape(4, 10, 96), base[0, :64]):
        b, s = quantize_mxfp4(x)
        rb, rs = quant.quantize_mxfp4_blocks(x.cpu())
        assert b.shape == (*x.shape[:-1], x.shape[-1] // 32, 16)
        assert torch.equal(s.cpu(), rs) and torch.equal(b.cpu(), rb), (x.shape, x.stride())
    for x in (base[:0, :64], base[:0, :64].reshape(0, 2, 32)):
        b, s = quantize_mxfp4(x)
        assert b.numel() == 0 and s.numel() == 0
    for bad in (base[:, :0], base[:, :33], base[0, 0]):
        with pytest.raises(ValueError):
            quantize_mxfp4(bad)
    with pytest.raises(TypeError):
        quantize_mxfp4(base[:, :64].double())


# ------------------------------------------------------------------ dense products
SHAPES = [(1, 1, 32), (1, 16, 64), (1, 1536, 2048), (2, 33, 96), (3, 100, 256), (4, 4096, 4096), (5, 24, 128),
          (15, 130, 1056), (16, 2048, 768), (17, 64, 512), (31, 4100, 512), (33, 4096, 2880), (64, 1024, 1024),
          (65, 200, 320), (100, 4096, 4096), (128, 256, 256), (200, 999, 736), (256, 8192, 640), (333, 5760, 2880),
          (513, 1024, 4096), (1000, 4097, 160), (1025, 2304, 1408), (2048, 4096, 1024), (20, 5760, 352),
          (90, 5800, 288), (150, 5760, 288), (1100, 11990, 288)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(gpu, M, N, K):
    x, xs = operand((M, K), M + K, gpu)
    w, ws = operand((N, K), N, gpu)
    out_dtype = DTYPES[(M + N) % 3]
    bias = None if M % 2 else torch.randn(N, device=gpu).to(DTYPES[N % 3])
    y, mag = product(values(x, xs), values(w, ws), bias)
    got = w4a4_linear(x, xs, w, ws, bias=bias, out_dtype=out_dtype)
    close(got, y, mag, out_dtype, roundings(K))
    assert torch.equal(got, w4a4_linear(x, xs, w, ws, bias=bias, out_dtype=out_dtype))  # no order that changes


@pytest.mark.parametrize("M,N,K", [(1, 64, 8192), (7, 48, 11008), (40, 64, 16384), (3, 32, 65536), (20, 40, 131072),
                                   (300, 300, 32768), (256, 4096, 11008)])
def test_linear_long_k(gpu, M, N, K):
    x, xs = operand((M, K), K, gpu)
    w, ws = operand((N, K), N, gpu)
    y, mag = product(values(x, xs), values(w, ws))
    close(w4a4_linear(x, xs, w, ws, out_dtype=torch.float32), y, mag, torch.float32, roundings(K))


@pytest.mark.parametrize("M", [1, 9, 40, 300])
def test_linear_far_scales(gpu, M):
    """Scale bytes far apart, whose smallest products vanish beside the largest."""
    x, xs = operand((M, 384), 5, gpu, spread=50)
    w, ws = operand((72, 384), 6, gpu, spread=50)
    y, mag = product(values(x, xs), values(w, ws))
    close(w4a4_linear(x, xs, w, ws, out_dtype=torch.float32), y, mag, torch.float32, roundings(384))


@pytest.mark.parametrize("M", [1, 4, 20, 70, 400])
@pytest.mark.parametrize("K", [64, 416, 1024])
def test_linear_edge_scales(gpu, M, K):
    """The scale 255 is NaN in its row or column alone; 0 and 254 are powers of two; what
    lies behind the last block of a row is not read into it."""
    x, xs = operand((M, K), 1, gpu)
    w, ws = operand((50, K), 2, gpu)
    ws[9, 1], xs[:, 1] = 0, 130
    ws[11, 0] = 254
    xs[0, -1] = 255
    ws[7, 0] = 255
    vx, vw = values(x, xs), values(w, ws)
    got = w4a4_linear(x, xs, w, ws, out_dtype=torch.float32)
    nan = torch.zeros(M, 50, dtype=torch.bool, device=gpu)
    nan[0], nan[:, 7] = True, True
    assert torch.equal(got.isnan(), nan)
    y, mag = product(vx.nan_to_num(), vw.nan_to_num())
    keep = ~nan
    keep[:, 11] = False  # 2^127 times a sum: may be infinite
    close(got[keep], y[keep], mag[keep], torch.float32, roundings(K))


@pytest.mark.parametrize("M", [1, 4, 20, 70, 400])
@pytest.mark.parametrize("K", [64, 416, 1024])
def test_linear_largest_scales(gpu, M, K):
    """The value of a product with the scales 253 and 254, the largest that are numbers, in the weight, in
    x, and where the other operand's block brings the product back into fp32's range."""
    x, xs = operand((M, K), 1, gpu)
    w, ws = operand((50, K), 2, gpu)
    xs[:, 0] = 40          # 2^-87: the first block's products are small ...
    ws[11, 0], ws[12, 0] = 254, 253  # ... but for these, of 2^40 and 2^39
    xs[M // 2, 1] = 254
    ws[:, 1] = 30
    vx, vw = values(x, xs), values(w, ws)
    y, mag = product(vx, vw)
    assert mag.max() < 2.0 ** 100 and (mag[:, 11] > 2.0 ** 30).all() and (mag[M // 2] > 2.0 ** 20).all()
    close(w4a4_linear(x, xs, w, ws, out_dtype=torch.float32), y, mag, torch.float32, roundings(K))
    offsets = torch.tensor([0, M], dtype=torch.int32, device=gpu)
    got = w4a4_grouped_linear(x, xs, offsets, w[None], ws[None], out_dtype=torch.float32)
    close(got, y, mag, torch.float32, roundings(K))


@pytest.mark.parametrize("name", ["silu", "gelu", "relu", "swiglu_oai"])
@pytest.mark.parametrize("M,N,K", [(1, 2, 32), (1, 128, 256), (3, 30, 96), (4, 1536, 2048), (16, 66, 512), (33, 200, 640),
                                   (64, 512, 256), (129, 1030, 352), (300, 4096, 512), (700, 2880, 1024),
                                   (2050, 4100, 288), (1100, 12010, 256)])
def test_linear_gated(gpu, name, M, N, K):
    x, xs = operand((M, K), M, gpu, spread=2)
    w, ws = operand((N, K), N, gpu, spread=2)
    ws -= 8
    dtype = DTYPES[(M + K // 32) % 3]
    bias = torch.randn(N, device=gpu) if M % 2 else None
    gu, mag = product(values(x, xs), values(w, ws), bias)
    got = w4a4_linear(x, xs, w, ws, bias=bias, activation=name, out_dtype=dtype)
    assert got.shape == (M, N // 2)
    gated_close(got, gu, mag, name, dtype, roundings(K))


def test_linear_gated_nan_and_limits(gpu):
    x, xs = operand((6, 64), 1, gpu)
    w, ws = operand((64, 64), 2, gpu)
    xs[2, 1] = 255
    for name in ("silu", "gelu", "relu", "swiglu_oai"):
        got = w4a4_linear(x, xs, w, ws, activation=name, out_dtype=torch.float32)
        assert got[2].isnan().all() and not got[[0, 1, 3, 4, 5]].isnan().any()
    keep = [0, 1, 3, 4, 5]
    gu, mag = product(values(x, xs)[keep], values(w, ws))
    got = w4a4_linear(x, xs, w, ws, activation="swiglu_oai", swiglu_alpha=0.7, swiglu_limit=3.0, out_dtype=torch.float32)
    gated_close(got[keep], gu, mag, "swiglu_oai", torch.float32, roundings(64), alpha=0.7, limit=3.0)


def test_linear_layouts(gpu):
    """Operands from odd addresses, rows apart, and empty ones."""
    x, xs = operand((9, 128), 1, gpu)
    w, ws = operand((20, 128), 2, gpu)
    want = w4a4_linear(x, xs, w, ws)
    ox = torch.cat([torch.zeros(1, dtype=torch.uint8, device=gpu), x.flatten()])[1:].view(x.shape)
    osx = torch.cat([torch.zeros(3, dtype=torch.uint8, device=gpu), xs.flatten()])[3:].view(xs.shape)
    osw = torch.cat([torch.zeros(1, dtype=torch.uint8, device=gpu), ws.flatten()])[1:].view(ws.shape)
    assert torch.equal(w4a4_linear(ox, osx, w, osw), want)
    wide, wides = torch.cat([x, x], dim=1), torch.cat([xs, xs], dim=1)
    assert torch.equal(w4a4_linear(wide[:, 4:], wides[:, 4:], w, ws), want)
    assert w4a4_linear(x[:0], xs[:0], w, ws).shape == (0, 20)
    with pytest.raises(ValueError, match="K="):
        w4a4_linear(x[:, :2], xs[:, :2], w, ws)
    with pytest.raises(ValueError, match="bias"):
        w4a4_linear(x, xs, w, ws, bias=torch.zeros(19, device=gpu))
    with pytest.raises(ValueError, match="even number"):
        w4a4_linear(x, xs, w[:19], ws[:19], activation="silu")
    with pytest.raises(ValueError, match="activation"):
        w4a4_linear(x, xs, w, ws, activation="tanh")
    with pytest.raises(TypeError):
        w4a4_linear(x, xs, w, ws, out_dtype=torch.float64)


# ------------------------------------------------------------------ quantiser and product
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1536, 2048), (1, 7, 32), (2, 100, 96), (3, 4096, 4096), (4, 64, 8192), (6, 50, 1056),
                                   (8, 66, 2048), (9, 66, 1024), (16, 48, 416), (17, 300, 11008), (70, 256, 512), (300, 520, 352)])
def test_fused_linear(gpu, dtype, M, N, K):
    """The bits of the quantiser and the product in two calls' definition."""
    g = torch.Generator(device=gpu).manual_seed(M + N)
    x = (torch.randn(M, K, generator=g, device=gpu) * torch.exp2(torch.randn(M, 1, generator=g, device=gpu) * 3)).to(dtype)
    w, ws = operand((N, K), N, gpu)
    bias = torch.randn(N, generator=g, device=gpu) if N % 2 == 0 else None
    b, s = quantize_mxfp4(x)
    y, mag = product(values(b, s), values(w, ws), bias)
    close(fused_w4a4_linear(x, w, ws, bias=bias), y, mag, dtype, roundings(K))
    close(fused_w4a4_linear(x, w, ws, bias=bias, out_dtype=torch.float32), y, mag, torch.float32, roundings(K))
    wide = torch.cat([x, x, x], dim=1)[:, K:2 * K]  # rows apart
    assert torch.equal(fused_w4a4_linear(wide, w, ws, bias=bias), fused_w4a4_linear(x, w, ws, bias=bias))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 80, 288), (1, 80, 2048), (1, 33, 16384), (3, 130, 800), (3, 48, 5440), (5, 80, 1056),
                                   (5, 40, 3232), (7, 48, 1024), (7, 100, 2336)])
def test_fused_linear_odd_tokens(gpu, dtype, M, N, K):
    """The one-launch product of an odd number of tokens, whose scales end in the middle of 16
    bytes of LDS, with K over two to four waves of one to sixteen steps."""
    assert M <= 8 and M * K <= 16384 and K >= 256
    g = torch.Generator(device=gpu).manual_seed(K + M)
    x = torch.randn(M, K, generator=g, device=gpu).to(dtype)
    w, ws = operand((N, K), N + K, gpu)
    y, mag = product(values(*quantize_mxfp4(x)), values(w, ws))
    got = fused_w4a4_linear(x, w, ws, out_dtype=torch.float32)
    close(got, y, mag, torch.float32, roundings(K))
    for m in range(M):  # a token's result does not depend on how many there are
        assert torch.equal(fused_w4a4_linear(x[m:m + 1], w, ws, out_dtype=torch.float32), got[m:m + 1])


@pytest.mark.parametrize("M", [1, 3, 12, 100])
def test_fused_linear_not_finite(gpu, M):
    x = torch.randn(M, 256, device=gpu)
    w, ws = operand((70, 256), 3, gpu)
    want = fused_w4a4_linear(x, w, ws)
    bad = x.clone()
    bad[0, 40] = math.inf
    got = fused_w4a4_linear(bad, w, ws)
    assert got[0].isnan().all() and torch.equal(got[1:], want[1:])
    odd = torch.randn(M * 256 + 1, device=gpu)[1:].view(M, 256)  # not on a 16-byte border
    b, s = quantize_mxfp4(odd)
    y, mag = product(values(b, s), values(w, ws))
    close(fused_w4a4_linear(odd, w, ws), y, mag, torch.float32, roundings(256))


def test_beside_the_wide_activations(gpu):
    """Values that the format holds exactly: the result of fused_mxfp4_linear."""
    w, ws = operand((64, 512), 4, gpu, spread=2)
    x = values(*operand((5, 512), 9, gpu, spread=2)).to(torch.bfloat16)
    x[:, ::32] = x[:, ::32].sign() * 6 * 2.0 ** torch.floor(torch.log2(x.reshape(5, -1, 32).abs().amax(-1).float())).to(x.dtype)
    b, s = quantize_mxfp4(x)
    again = dequantize_mxfp4_blocks(b, s)
    a = fused_w4a4_linear(again, w, ws, out_dtype=torch.float32)
    c = fused_mxfp4_linear(again, w, ws, out_dtype=torch.float32)
    mag = again.double().abs() @ values(w, ws).abs().t()
    assert bool(((a - c).double().abs() <= 2 * 512 * U * mag).all())


# ------------------------------------------------------------------ grouped
def grouped_reference(x, offsets, w, index=None, bias=None):
    """Rows in 64 bits: (product, magnitude, rows that have a result)."""
    off = offsets.cpu().clamp(0, x.shape[0] if index is None else index.shape[0]).tolist()
    rows = x.shape[0] if index is None else index.shape[0]
    y = torch.zeros(rows, w.shape[1], dtype=torch.float64, device=x.device)
    mag, live = y.clone(), torch.zeros(rows, dtype=torch.bool, device=x.device)
    for e in range(w.shape[0]):
        lo, hi = off[e], off[e + 1]
        if hi <= lo:
            continue
        src = torch.arange(lo, hi, device=x.device) if index is None else index[lo:hi].long()
        ok = (src >= 0) & (src < x.shape[0])
        r = torch.arange(lo, hi, device=x.device)[ok]
        y[r], mag[r] = product(x[src[ok]], w[e], None if bias is None else bias[e])
        live[r] = True
    return y, mag, live


@pytest.mark.parametrize("sizes,N,K", [
    ([0, 1, 0], 33, 64), ([3, 0, 5, 1, 17], 48, 96), ([1] * 12, 1536, 2048), ([16, 15, 33, 0, 64], 130, 416),
    ([40, 7, 90, 128, 129], 520, 352), ([100] * 9, 2048, 768), ([300, 500, 1, 0, 223], 768, 1056),
    ([70] * 40, 600, 512), ([190] * 12, 1024, 256), ([0, 0, 700], 5760, 2880), ([1, 0, 9, 0, 0, 0], 77, 320),
    ([3, 9, 0, 5, 17, 1], 70, 416), ([6] * 20, 640, 256), ([1, 2, 0, 3], 48, 32768), ([5, 8, 6], 34, 16384)])
@pytest.mark.parametrize("through", [False, True])
def test_grouped(gpu, sizes, N, K, through):
    E, P = len(sizes), sum(sizes)
    offsets = torch.tensor([0] + sizes).cumsum(0).to(torch.int32).to(gpu)
    dtype = DTYPES[(P + through) % 3]
    T = max(1, P // 3) if through else P
    x, xs = operand((T, K), P, gpu)
    w, ws = operand((E, N, K), N, gpu)
    bias = torch.randn(E, N, device=gpu) if E % 2 else None
    index = None
    if through:
        index = torch.randint(0, T, (P,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
        index[P // 2] = -1
        index[P - 1] = T
        index = index.to(gpu)
    y, mag, live = grouped_reference(values(x, xs), offsets, values(w, ws), index, bias)
    got = w4a4_grouped_linear(x, xs, offsets, w, ws, row_index=index, bias=bias, out_dtype=dtype)
    assert (got[~live] == 0).all()
    close(got[live], y[live], mag[live], dtype, roundings(K))
    if N % 2 == 0:
        got = w4a4_grouped_linear(x, xs, offsets, w, ws - 8, row_index=index, bias=bias, activation="silu", out_dtype=dtype)
        y, mag, live = grouped_reference(values(x, xs), offsets, values(w, ws - 8), index, bias)
        assert (got[~live] == 0).all()
        gated_close(got[live], y[live], mag[live], "silu", dtype, roundings(K))


@pytest.mark.parametrize("rows", [20, 400])
def test_grouped_rows_of_no_expert(gpu, rows):
    """Offsets that start late, end early, or are out of range: zeros, and nothing else is written."""
    x, xs = operand((rows, 128), 1, gpu)
    w, ws = operand((3, 96, 128), 2, gpu)
    for off in ([2, 5, 5, rows - 3], [0, 0, 0, 0], [-4, 6, 9, rows + 70], [rows, rows, rows, rows], [0, rows, rows, rows]):
        offsets = torch.tensor(off, dtype=torch.int32, device=gpu)
        y, mag, live = grouped_reference(values(x, xs), offsets, values(w, ws))
        got = w4a4_grouped_linear(x, xs, offsets, w, ws, out_dtype=torch.float32)
        assert (got[~live] == 0).all()
        close(got[live], y[live], mag[live], torch.float32, roundings(128))


def test_grouped_refusals(gpu):
    x, xs = operand((4, 64), 1, gpu)
    w, ws = operand((3, 32, 64), 2, gpu)
    off = torch.tensor([0, 1, 2, 4], dtype=torch.int32, device=gpu)
    with pytest.raises(TypeError, match="offsets"):
        w4a4_grouped_linear(x, xs, off.long(), w, ws)
    with pytest.raises(ValueError, match="entries"):
        w4a4_grouped_linear(x, xs, off[:3], w, ws)
    with pytest.raises(ValueError, match="one dimension"):
        w4a4_grouped_linear(x, xs, off, w, ws, row_index=torch.zeros(4, 2, dtype=torch.int32, device=gpu)[:, 0])
    with pytest.raises(ValueError):
        w4a4_grouped_linear(x, xs, off, w[0], ws[0])
    assert w4a4_grouped_linear(x[:0], xs[:0], torch.zeros_like(off), w, ws).shape == (0, 32)
    index = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
    assert (w4a4_grouped_linear(x[:0], xs[:0], off, w, ws, row_index=index) == 0).all()


# ------------------------------------------------------------------ the expert layer
def quantised(h):
    """(scale exponents, values of the codes) of h in 64 bits."""
    b = h.reshape(*h.shape[:-1], -1, 32)
    m, e = torch.frexp(b.abs().amax(-1).clamp_min(float(torch.tensor(1e-12))))
    return torch.where(m <= 0.75, e - 3, e - 2)


def code_values(h, e):
    b = h.reshape(*h.shape[:-1], -1, 32)
    s = two_to(e).unsqueeze(-1)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=h.device)
    v = LUT[:8].to(h.device)[torch.bucketize(b.abs() / s, borders)] * s
    return (torch.sign(b) * v).reshape(h.shape)


def layer_reference(x, w1, w2, ids, wt, name, b1=None, b2=None, K=0, **kw):
    """(result, bound without the output's rounding) in 64 bits: the sums, and the codes of h that may
    fall on either side of a border for an h that is off by its own bound."""
    T, k = ids.shape
    out = torch.zeros(T, w2.shape[1], dtype=torch.float64, device=x.device)
    bound = out.clone()
    for t in range(T):
        for j in range(k):
            e = int(ids[t, j])
            if e < 0 or e >= w1.shape[0]:
                continue
            gu, mag = product(x[t:t + 1], w1[e], None if b1 is None else b1[e])
            g, u = gu.chunk(2, dim=1)
            eg, eu = (roundings(x.shape[1]) * U * mag).chunk(2, dim=1)
            h = act(name, g, u, **kw)
            off = torch.zeros_like(h)
            for a in (-1, 1):
                for b in (-1, 1):
                    off = torch.maximum(off, (act(name, g + a * eg, u + b * eu, **kw) - h).abs())
            off = 2 * off + 16 * U * (h.abs() + (g.abs() if name == "swiglu_oai" else 0)) + g.abs() * (u.abs() + 1) * 2.0 ** -126
            ex = quantised(h)
            q = code_values(h, ex)
            dq = torch.zeros_like(q)
            top = h.reshape(1, -1, 32).abs()
            grow = off.reshape(1, -1, 32)
            for s in (quantised((top + grow).reshape(h.shape)), quantised((top - grow).clamp_min(0).reshape(h.shape)), ex):
                for side in (-1, 1):
                    dq = torch.maximum(dq, (code_values(h + side * off, s) - q).abs())
            y, ymag = product(q, w2[e], None if b2 is None else b2[e])
            wgt = float(wt[t, j])
            out[t] += wgt * y[0]
            bound[t] += abs(wgt) * ((dq @ w2[e].abs().t())[0] + (roundings(w2.shape[2]) + k + 8) * U * ymag[0])
    return out, bound


def layer_close(got, ref, bound, dtype):
    err = (got.double() - ref).abs()
    limit = bound * (1 + half_step(dtype)) + half_step(dtype) * ref.abs() + tiny(dtype)
    bad = far(got, ref, limit, dtype)
    assert got.dtype == dtype and not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float((err - limit).max()):.3e}"


def layer(E, H, I, seed, dev, bias=False):
    w1, s1 = operand((E, 2 * I, H), seed, dev, spread=2)
    w2, s2 = operand((E, H, I), seed + 1, dev, spread=2)
    s1, s2 = s1 - 8, s2 - 6
    b1 = torch.randn(E, 2 * I, device=dev) * 0.3 if bias else None
    b2 = (torch.randn(E, H, device=dev) * 0.3).to(torch.bfloat16) if bias else None
    return w1, s1, w2, s2, b1, b2


def routing(T, k, E, seed, dev, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    return ids.to(dtype).to(dev), torch.softmax(torch.randn(T, k, generator=g), dim=1).to(dev)


@pytest.mark.parametrize("T,k,E,H,I,name,bias", [
    (1, 1, 1, 32, 32, "silu", False), (1, 2, 4, 64, 96, "gelu", True), (1, 8, 128, 2048, 768, "silu", False),
    (2, 3, 5, 160, 64, "relu", True), (3, 4, 32, 2880, 2880, "swiglu_oai", True), (7, 2, 16, 1024, 512, "silu", False),
    (8, 8, 64, 512, 320, "silu", True), (16, 8, 256, 256, 512, "silu", False), (17, 4, 8, 384, 160, "swiglu_oai", True),
    (16, 1, 1, 256, 128, "silu", False), (33, 6, 60, 512, 1408, "gelu", False), (150, 4, 6, 544, 288, "silu", True),
    (400, 2, 4, 256, 512, "swiglu_oai", True), (16, 1, 2, 14336, 256, "silu", True), (16, 2, 2, 2880, 1600, "silu", False),
    (15, 4, 32, 2880, 2880, "swiglu_oai", True), (16, 16, 40, 256, 256, "relu", True)])
def test_moe(gpu, T, k, E, H, I, name, bias):
    w1, s1, w2, s2, b1, b2 = layer(E, H, I, T + H, gpu, bias)
    dtype = (torch.bfloat16, torch.float16, torch.float32)[T % 3]
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(dtype).to(gpu)
    ids, wt = routing(T, k, E, 3, gpu, torch.int64 if T % 2 else torch.int32)
    if T > 2:
        ids[1, 0], ids[2, k - 1] = -1, E
    wt = wt.to((torch.float32, torch.bfloat16, torch.float16)[k % 3])
    got = fused_w4a4_moe(x, w1, s1, w2, s2, ids, wt, activation=name, w1_bias=b1, w2_bias=b2)
    ref, bound = layer_reference(values(*quantize_mxfp4(x)), values(w1, s1), values(w2, s2), ids, wt.double(), name, b1, b2)
    layer_close(got, ref, bound, dtype)
    assert torch.equal(got, fused_w4a4_moe(x, w1, s1, w2, s2, ids, wt, activation=name, w1_bias=b1, w2_bias=b2))


@pytest.mark.parametrize("T", [1, 5, 16, 90])
def test_moe_odd_routing(gpu, T):
    """No expert at all, the same expert twice, one expert for all, weights of zero."""
    w1, s1, w2, s2, b1, b2 = layer(4, 96, 64, 8, gpu, True)
    x = torch.randn(T, 96, device=gpu)
    wt = torch.rand(T, 3, device=gpu)
    v = values(*quantize_mxfp4(x)), values(w1, s1), values(w2, s2)
    for ids in (torch.full((T, 3), -1), torch.full((T, 3), 2), torch.tensor([[1, 3, 1]]).repeat(T, 1),
                torch.tensor([[9, 0, -7]]).repeat(T, 1)):
        ids = ids.to(torch.int32).to(gpu)
        got = fused_w4a4_moe(x, w1, s1, w2, s2, ids, wt, w1_bias=b1, w2_bias=b2)
        ref, bound = layer_reference(*v, ids, wt, "silu", b1, b2)
        layer_close(got, ref, bound, torch.float32)
    zero = fused_w4a4_moe(x, w1, s1, w2, s2, ids, torch.zeros_like(wt), w1_bias=b1, w2_bias=b2)
    assert (zero == 0).all()


@pytest.mark.parametrize("T", [2, 60])
def test_moe_not_finite(gpu, T):
    """A token with an infinity has NaN results, no other token's change; a NaN weight of a pair without
    an expert is not read."""
    w1, s1, w2, s2, _, _ = layer(4, 96, 64, 8, gpu)
    x = torch.randn(T, 96, device=gpu)
    ids, wt = routing(T, 2, 4, 5, gpu)
    want = fused_w4a4_moe(x, w1, s1, w2, s2, ids, wt)
    bad = x.clone()
    bad[1, 7] = math.inf
    got = fused_w4a4_moe(bad, w1, s1, w2, s2, ids, wt)
    assert got[1].isnan().all() and torch.equal(got[0], want[0]) and torch.equal(got[2:], want[2:])
    ids[0, 1] = -1
    one = fused_w4a4_moe(x, w1, s1, w2, s2, ids, wt)
    wt[0, 1] = math.nan
    assert torch.equal(fused_w4a4_moe(x, w1, s1, w2, s2, ids, wt), one)


@pytest.mark.parametrize("T", [1, 6, 100])
def test_moe_is_its_parts(gpu, T):
    """Sort, quantise, gate_up, quantise, down and combine called one by one."""
    w1, s1, w2, s2, b1, b2 = layer(8, 256, 160, 2, gpu, True)
    x = torch.randn(T, 256, device=gpu).to(torch.bfloat16)
    ids, wt = routing(T, 2, 8, 1, gpu)
    sort = sort_tokens(ids, 8)
    q, s = quantize_mxfp4(x)
    h = w4a4_grouped_linear(q, s, sort.offsets, w1, s1, row_index=sort.token_of_row, bias=b1, activation="silu",
                            out_dtype=torch.float32)
    hq, hs = quantize_mxfp4(h)
    y = w4a4_grouped_linear(hq, hs, sort.offsets, w2, s2, bias=b2, out_dtype=torch.float32)
    parts = combine_tokens(y, wt, sort, out_dtype=torch.bfloat16)
    got = fused_w4a4_moe(x, w1, s1, w2, s2, ids, wt, w1_bias=b1, w2_bias=b2)
    ref, bound = layer_reference(values(q, s), values(w1, s1), values(w2, s2), ids, wt, "silu", b1, b2)
    layer_close(parts, ref, bound, torch.bfloat16)
    layer_close(got, ref, bound, torch.bfloat16)


@pytest.mark.parametrize("M", [1, 5, 40, 200])
def test_expert_forward(gpu, M):
    w1, s1, w2, s2, _, _ = layer(1, 160, 96, 4, gpu)
    x = torch.randn(M, 160, device=gpu).to(torch.bfloat16)
    got = fused_w4a4_expert_forward(x, w1[0], s1[0], w2[0], s2[0], intermediate=96)
    ids, wt = torch.zeros(M, 1, dtype=torch.int32, device=gpu), torch.ones(M, 1, device=gpu)
    ref, bound = layer_reference(values(*quantize_mxfp4(x)), values(w1, s1), values(w2, s2), ids, wt, "silu")
    layer_close(got, ref, bound, torch.bfloat16)
    with pytest.raises(ValueError, match="rows"):
        fused_w4a4_expert_forward(x, w1[0], s1[0], w2[0], s2[0], intermediate=95)


@pytest.mark.parametrize("T", [3, 16, 40])
def test_moe_layouts(gpu, T):
    """Tokens with rows apart, from a border of 2 bytes, and tables that are not contiguous."""
    w1, s1, w2, s2, b1, b2 = layer(8, 256, 256, 9, gpu, True)
    wide = torch.randn(T, 3 * 256, device=gpu).to(torch.bfloat16)
    ids, wt = routing(T, 3, 8, 2, gpu)
    for x in (wide[:, 256:512], wide[:, 1:257], wide.t().contiguous().t()[:, :256]):
        want = fused_w4a4_moe(x.contiguous(), w1, s1, w2, s2, ids, wt, w1_bias=b1, w2_bias=b2)
        got = fused_w4a4_moe(x, w1, s1, w2, s2, ids.t().contiguous().t(), wt.t().contiguous().t(), w1_bias=b1, w2_bias=b2)
        if x.data_ptr() % 16 == 0:
            assert torch.equal(got, want)
        ref, bound = layer_reference(values(*quantize_mxfp4(x)), values(w1, s1), values(w2, s2), ids, wt, "silu", b1, b2)
        layer_close(got, ref, bound, torch.bfloat16)


# A layer of few tokens in two kernels: hidden and inter from 256 on, up to 16 tokens
def two_kernels(x, w1, s1, w2, s2, ids, wt, name="silu", b1=None, b2=None):
    """fused_w4a4_moe, and that its call is of two kernels: they leave the sort's tables, with which the workspace
    begins, as they were."""
    (T, H), k, (E, I2) = x.shape, ids.shape[1], w1.shape[:2]
    got = fused_w4a4_moe(x, w1, s1, w2, s2, ids, wt, activation=name, w1_bias=b1, w2_bias=b2)
    L, out = nat.lib(), torch.empty_like(x)
    need = L.ftm_w4a4_moe_workspace_bytes(T, k, E, H, I2 // 2)
    ws = torch.full((need,), 0xA5, dtype=torch.uint8, device=x.device)
    dt = lambda b: 0 if b is None else nat.dtype_code(b.dtype)  # noqa: E731
    c = nat.FtmW4A4Moe(x.data_ptr(), ids.data_ptr(), wt.data_ptr(), out.data_ptr(), w1.data_ptr(), s1.data_ptr(), nat.ptr(b1),
                       w2.data_ptr(), s2.data_ptr(), nat.ptr(b2), H * x.element_size(), T, k, E, H, I2 // 2,
                       nat.dtype_code(x.dtype), nat.ID_I64 if ids.dtype == torch.int64 else nat.ID_I32, nat.dtype_code(wt.dtype),
                       dt(b1), dt(b2), {"silu": nat.ACT_SILU, "swiglu_oai": nat.ACT_SWIGLU_OAI}[name], 1.702, 7.0)
    nat.launch("ftm_w4a4_moe_forward", L.ftm_w4a4_moe_forward, x, ctypes.byref(c), ws.data_ptr(), need)
    assert (ws[:4 * (E + 1)] == 0xA5).all(), "not the two kernels"
    assert torch.equal(out.view(torch.uint8), got.view(torch.uint8))
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 5, 16])
def test_two_kernels_odd_routing(gpu, T, dtype):
    """No expert at all, one expert for all pairs (48 of 16 tokens), the same expert twice, ids far outside."""
    w1, s1, w2, s2, b1, b2 = layer(4, 288, 320, 8, gpu, True)
    g = torch.Generator().manual_seed(T)
    x, wt = torch.randn(T, 288, generator=g).to(dtype).to(gpu), torch.rand(T, 3, generator=g).to(gpu)
    v = values(*quantize_mxfp4(x)), values(w1, s1), values(w2, s2)
    for ids in (torch.full((T, 3), -1), torch.full((T, 3), 2), torch.tensor([[1, 3, 1]]).repeat(T, 1),
                torch.tensor([[9, 0, -7]]).repeat(T, 1), torch.tensor([[2 ** 32 + 1, 3, -2 ** 32]]).repeat(T, 1)):
        ids = ids.to(gpu) if ids.abs().max() > 2 ** 31 else ids.to(torch.int32).to(gpu)
        got = two_kernels(x, w1, s1, w2, s2, ids, wt, "silu", b1, b2)
        ref, bound = layer_reference(*v, ids, wt, "silu", b1, b2)
        layer_close(got, ref, bound, dtype)
        if not ((ids >= 0) & (ids < 4)).any():
            assert (got == 0).all()
        assert (two_kernels(x, w1, s1, w2, s2, ids, torch.zeros_like(wt), "silu", b1, b2) == 0).all()


@pytest.mark.parametrize("T,k,E,name", [(16, 16, 1, "silu"), (16, 16, 3, "swiglu_oai"), (4, 64, 5, "silu"), (1, 64, 2, "silu"),
                                        (16, 12, 2, "silu"), (9, 28, 40, "swiglu_oai")])
def test_two_kernels_many_pairs(gpu, T, k, E, name):
    """Up to 256 pairs, an expert's more than a workgroup takes: the pairs that begin a chunk lie in
    any lane of the ids."""
    w1, s1, w2, s2, b1, b2 = layer(E, 256, 288, T + k, gpu, True)
    g = torch.Generator().manual_seed(k)
    x = torch.randn(T, 256, generator=g).to(torch.bfloat16).to(gpu)
    ids = torch.randint(-1, E + 1, (T, k), generator=g).to(gpu) if E > 1 else torch.zeros(T, k, dtype=torch.int64, device=gpu)
    wt = torch.softmax(torch.randn(T, k, generator=g), dim=1).to(gpu)
    got = two_kernels(x, w1, s1, w2, s2, ids, wt, name, b1, b2)
    ref, bound = layer_reference(values(*quantize_mxfp4(x)), values(w1, s1), values(w2, s2), ids, wt, name, b1, b2)
    layer_close(got, ref, bound, torch.bfloat16)
    assert torch.equal(got, two_kernels(x, w1, s1, w2, s2, ids, wt, name, b1, b2))


@pytest.mark.parametrize("T", [2, 16])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_two_kernels_not_finite(gpu, T, bad):
    """A token that is not finite has NaN results, no other token's change, of the same expert neither; a NaN
    weight of a pair without an expert is not read; a NaN scale of a weight is that of its expert's tokens."""
    w1, s1, w2, s2, _, _ = layer(4, 288, 256, 8, gpu)
    x = torch.randn(T, 288, generator=torch.Generator().manual_seed(T)).to(gpu)
    ids, wt = routing(T, 2, 4, 5, gpu)
    ids[:, 0] = 2
    want = two_kernels(x, w1, s1, w2, s2, ids, wt)
    assert not want.isnan().any()
    odd = x.clone()
    odd[1, 7] = bad
    got = two_kernels(odd, w1, s1, w2, s2, ids, wt)
    assert got[1].isnan().all() and torch.equal(got[0], want[0]) and torch.equal(got[2:], want[2:])
    ids[0, 1] = -1
    one = two_kernels(x, w1, s1, w2, s2, ids, wt)
    wt[0, 1] = math.nan
    assert torch.equal(two_kernels(x, w1, s1, w2, s2, ids, wt), one)
    ids[:, 0], ids[:, 1], ids[1, 1] = 0, 1, 3
    wt[0, 1] = 0.5
    want = two_kernels(x, w1, s1, w2, s2, ids, wt)
    s2 = s2.clone()
    s2[3, 40, 1] = 255
    got = two_kernels(x, w1, s1, w2, s2, ids, wt)
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[1, 40] = True
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("T", [1, 6, 16])
def test_two_kernels_is_its_parts(gpu, T):
    """Against the operators called one by one, with experts that come twice in a token."""
    w1, s1, w2, s2, b1, b2 = layer(8, 288, 352, 2, gpu, True)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, 288, generator=g).to(torch.bfloat16).to(gpu)
    ids, wt = torch.randint(0, 8, (T, 6), generator=g).to(torch.int32).to(gpu), torch.rand(T, 6, generator=g).to(gpu)
    sort = sort_tokens(ids, 8)
    q, s = quantize_mxfp4(x)
    h = w4a4_grouped_linear(q, s, sort.offsets, w1, s1, row_index=sort.token_of_row, bias=b1, activation="silu",
                            out_dtype=torch.float32)
    hq, hs = quantize_mxfp4(h)
    y = w4a4_grouped_linear(hq, hs, sort.offsets, w2, s2, bias=b2, out_dtype=torch.float32)
    parts = combine_tokens(y, wt, sort, out_dtype=torch.bfloat16)
    got = two_kernels(x, w1, s1, w2, s2, ids, wt, "silu", b1, b2)
    ref, bound = layer_reference(values(q, s), values(w1, s1), values(w2, s2), ids, wt, "silu", b1, b2)
    layer_close(parts, ref, bound, torch.bfloat16)
    layer_close(got, ref, bound, torch.bfloat16)


@pytest.mark.parametrize("T", [1, 8, 16])
def test_two_kernels_captured_and_replayed(gpu, T):
    """In a graph, replayed over other tokens and ids (experts that come often, and no expert) between eager calls;
    then on two streams at once."""
    w1, s1, w2, s2, b1, b2 = layer(8, 256, 288, 6, gpu, True)
    run = lambda x, i, w: fused_w4a4_moe(x, w1, s1, w2, s2, i, w, w1_bias=b1, w2_bias=b2)  # noqa: E731
    sets, want = [], []
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        ids = torch.randint(-1, (8, 2, 9, 1)[seed], (T, 3), generator=g).to(torch.int32).to(gpu)
        sets.append((torch.randn(T, 256, generator=g).to(torch.bfloat16).to(gpu), ids, torch.rand(T, 3, generator=g).to(gpu)))
        want.append(two_kernels(sets[-1][0], w1, s1, w2, s2, *sets[-1][1:], "silu", b1, b2))
    x, ids, wt = (t.clone() for t in sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, ids, wt)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, ids, wt)
    for n in range(8):
        for dst, src in zip((x, ids, wt), sets[n % 4]):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[n % 4])
        assert torch.equal(run(*sets[(n + 1) % 4]), want[(n + 1) % 4])
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for n in range(16):
        with torch.cuda.stream(streams[n % 2]):
            outs.append(run(*sets[n % 4]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[n % 4]) for n, o in enumerate(outs))


def test_moe_refusals(gpu):
    w1, s1, w2, s2, _, _ = layer(2, 64, 32, 1, gpu)
    x, ids, wt = torch.randn(3, 64, device=gpu), torch.zeros(3, 1, dtype=torch.int32, device=gpu), torch.ones(3, 1, device=gpu)
    for a in ((x[:2], w1, s1, w2, s2, ids, wt), (x, w1, s1, w2, s2, ids, wt[:2]), (x[:, :32], w1, s1, w2, s2, ids, wt),
              (x, w1, s1, w2[:, :32], s2[:, :32], ids, wt), (x, w1[:1], s1[:1], w2, s2, ids, wt),
              (x, w1[:, :62], s1[:, :62], w2, s2, ids, wt), (x, w1, s1[:, :, :1], w2, s2, ids, wt),
              (x, w1, s1, w2, s2, ids[:, :0], wt[:, :0])):
        with pytest.raises(ValueError):
            fused_w4a4_moe(*a)
    with pytest.raises(TypeError):
        fused_w4a4_moe(x, w1, s1, w2, s2, ids.to(torch.int16), wt)
    assert fused_w4a4_moe(x[:0], w1, s1, w2, s2, ids[:0], wt[:0]).shape == (0, 64)


# ------------------------------------------------------------------ streams, graphs, guards
@pytest.mark.parametrize("T", [1, 8, 120])
def test_captured_and_replayed(gpu, T):
    """The layer in a graph, replayed with other inputs between eager calls; and two streams at
    once, each with its own call."""
    w1, s1, w2, s2, b1, b2 = layer(8, 256, 128, 6, gpu, True)
    run = lambda x, i, w: fused_w4a4_moe(x, w1, s1, w2, s2, i, w, w1_bias=b1, w2_bias=b2)  # noqa: E731
    sets = []
    for seed in range(4):
        ids, wt = routing(T, 2, 8, seed, gpu)
        sets.append((torch.randn(T, 256, device=gpu).to(torch.bfloat16), ids, wt))
    want = [run(*s) for s in sets]
    x, ids, wt = (t.clone() for t in sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, ids, wt)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, ids, wt)
    for n in range(8):
        for dst, src in zip((x, ids, wt), sets[n % 4]):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[n % 4])
        assert torch.equal(run(*sets[(n + 1) % 4]), want[(n + 1) % 4])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for n in range(8):
        with torch.cuda.stream(streams[n % 2]):
            outs.append(run(*sets[n % 4]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[n % 4]) for n, o in enumerate(outs))


@pytest.mark.parametrize("sizes", [[1, 0, 3], [9, 4, 6, 0], [40, 0, 70], [300, 5, 90]])
def test_products_captured_and_replayed(gpu, sizes):
    """Quantiser, dense and grouped products in one graph, replayed over other values and other
    offsets, with eager calls between the replays."""
    E, P, K, N = len(sizes), sum(sizes), 288, 130
    w, ws = operand((E, N, K), 3, gpu)
    sets = []
    for n in range(3):
        cuts = torch.tensor(sizes[n:] + sizes[:n]).cumsum(0)
        sets.append((torch.randn(P, K, device=gpu), torch.cat([torch.zeros(1), cuts]).to(torch.int32).to(gpu)))

    def run(x, offsets):
        q, s = quantize_mxfp4(x)
        return (w4a4_grouped_linear(q, s, offsets, w, ws), w4a4_linear(q, s, w[0], ws[0], activation="silu"),
                fused_w4a4_linear(x, w[1], ws[1]))

    want = [run(*a) for a in sets]
    x, offsets = (t.clone() for t in sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, offsets)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, offsets)
    for n in range(6):
        for dst, src in zip((x, offsets), sets[n % 3]):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[n % 3]))
        assert all(torch.equal(a, b) for a, b in zip(run(*sets[(n + 1) % 3]), want[(n + 1) % 3]))


def test_far_offsets(gpu):
    """Operands and results past 2^31 bytes, and rows that an index finds past 2^30."""
    M, K, N = 2 ** 21 + 5, 1024, 640
    part, parts = operand((997, K), 1, gpu)
    x, xs = part.repeat(M // 997 + 1, 1, 1)[:M], parts.repeat(M // 997 + 1, 1)[:M]
    w, ws = operand((3, N, K), 2, gpu)
    rows = torch.tensor([0, 1, 2 ** 19 + 1, 2 ** 20, 2 ** 20 + 255, M - 300, M - 2, M - 1], device=gpu)
    v = values(w, ws)
    got = w4a4_linear(x, xs, w[0], ws[0], out_dtype=torch.float32)
    y, mag = product(values(x[rows], xs[rows]), v[0])
    close(got[rows], y, mag, torch.float32, roundings(K))
    del got
    offsets = torch.tensor([0, 2 ** 19 + 1, 2 ** 20, M], dtype=torch.int32, device=gpu)
    got = w4a4_grouped_linear(x, xs, offsets, w, ws, out_dtype=torch.float32)
    for r in rows.tolist():
        e = 0 if r < 2 ** 19 + 1 else 1 if r < 2 ** 20 else 2
        y, mag = product(values(x[r:r + 1], xs[r:r + 1]), v[e])
        close(got[r:r + 1], y, mag, torch.float32, roundings(K))
    del got
    index = rows.to(torch.int32)
    offsets = torch.tensor([0, 3, 4, 8], dtype=torch.int32, device=gpu)
    y, mag, live = grouped_reference(values(x[rows], xs[rows]), offsets, v)
    close(w4a4_grouped_linear(x, xs, offsets, w, ws, row_index=index, out_dtype=torch.float32), y, mag, torch.float32, roundings(K))
    assert live.all()


@pytest.mark.parametrize("M,N,K", [(1, 50, 64), (3, 66, 288), (20, 70, 256), (70, 130, 352), (300, 300, 256)])
def test_writes_its_result_alone(gpu, M, N, K):
    """Rows and bytes around the result stay as they were."""
    x, xs = operand((M, K), 1, gpu)
    w, ws = operand((N, K), 2, gpu)
    for dtype, code, size in ((torch.float32, nat.DT_F32, 4), (torch.bfloat16, nat.DT_BF16, 2)):
        guard = torch.full((M * N + 256,), 7.0, dtype=dtype, device=gpu)
        out = guard[128:128 + M * N]
        c = nat.FtmW4A4(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), None, out.data_ptr(), None, None, M, M, 0,
                        0, N, K, 1, 0, code, -1, 0.0, 0.0)
        nat.launch("ftm_w4a4_linear", nat.lib().ftm_w4a4_linear, x, ctypes.byref(c))
        assert torch.equal(out.view(M, N), w4a4_linear(x, xs, w, ws, out_dtype=dtype))
        assert (guard[:128] == 7).all() and (guard[128 + M * N:] == 7).all()
