"""The int8 product with a scale per token and per channel on the GPU, against
plain arithmetic in 64 bits.

Tolerances: the integer sum is exact; its rounding to fp32, the token scale and
the channel scale (with the bias) are one rounding each, 2^-24 relative, and
the output rounds once, by half a step of its type."""
import ctypes
import math

import pytest
import torch

from ftmoe import _native as nat
from ftmoe import quant
from ftmoe.engine import MoeGraphRunner
from ftmoe.kernel.fused_w8a8_linear import fused_w8a8_expert_forward, fused_w8a8_linear
from ftmoe.kernel.fused_w8a8_moe import fused_w8a8_moe
from ftmoe.kernel.w8a8_linear import quantize_int8_token, w8a8_grouped_linear, w8a8_linear
from ftmoe.moe.token_sort import combine_tokens, sort_tokens

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0  # fp32: the last of the counted roundings


def tiny(dtype):
    """Half of the smallest step of a type's subnormals."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def codes(shape, seed, dev, lo=-127, hi=127):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randint(lo, hi + 1, shape, generator=g, device=dev, dtype=torch.int32).to(torch.int8)


def scales(shape, seed, dev, dtype=torch.float32):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.rand(shape, generator=g, device=dev) * 0.02 + 0.001).to(dtype)


def close(got, ref, mag, dtype, roundings=3):
    """|got - ref| within `roundings` fp32 ones of `mag` and one of the output type."""
    assert got.shape == ref.shape and got.dtype == dtype
    err = (got.double() - ref).abs()
    bound = roundings * U * mag * (1 + half_step(dtype)) + half_step(dtype) * ref.abs() + tiny(dtype)
    bad = err > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} out of tolerance, worst {float((err - bound).max()):.3e}"


def exact(q, s, w, ws, bias=None):
    """(product, magnitude) in 64 bits."""
    y = (q.double() @ w.double().t()) * s.double()[:, None] * ws.double().reshape(1, -1)
    if bias is None:
        return y, y.abs()
    return y + bias.double(), y.abs() + bias.double().abs()


# ------------------------------------------------------------------ quantiser
INV = torch.ones(()) / 127  # the fp32 nearest 1 / 127, by which the scale is defined


def exact_quantise(x):
    xc = x.cpu()
    s = xc.float().abs().amax(dim=-1).clamp_min(1e-12) * INV
    q = (xc.double() / s.double().unsqueeze(-1)).round()
    return q.to(torch.int8), s


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 7), (5, 64), (9, 100), (1, 2048), (300, 512), (7, 1024), (2, 2056),
                                    (3, 4096), (2, 8192), (2, 16384), (2, 20000), (5, 2049)])
def test_quantiser(gpu, dtype, rows, K):
    g = torch.Generator().manual_seed(rows * 31 + K)
    x = (torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-8, 8, (rows, 1), generator=g).float())).to(dtype)
    q, s = quantize_int8_token(x.to(gpu))
    rq, rs = exact_quantise(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu(), rq)


def test_quantiser_borders(gpu):
    """Quotients at and next to every border n + 1/2: scale a power of two (127 s the
    maximum), x the border and its neighbours in fp32; and the same under scales that
    are none, where the exact quotient lies on one side of the border."""
    n = torch.arange(-127, 127, dtype=torch.float64) + 0.5
    for s in (2.0 ** -3, 0.1, 0.37, 1.7e-5, 3.3e7):
        top = torch.tensor(127 * s, dtype=torch.float32)
        sc = (top * INV).double()
        b = (n * sc).float()
        x = torch.cat([top.reshape(1), b, torch.nextafter(b, torch.tensor(math.inf)),
                       torch.nextafter(b, torch.tensor(-math.inf))])[None]
        q, sg = quantize_int8_token(x.to(gpu))
        rq, rs = exact_quantise(x)
        assert torch.equal(sg.cpu(), rs) and torch.equal(q.cpu(), rq), s


def test_quantiser_is_torchs_on_the_gpu(gpu):
    """bf16 values, whose quotients often end in .5: the codes of ``quantize_int8_channel``
    on the GPU wherever its fp32 quotient is not the one that a border needs."""
    x = torch.randn(500, 512, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(gpu)
    q, s = quantize_int8_token(x)
    tq, ts = quant.quantize_int8_channel(x)
    assert torch.equal(s, ts)
    quotient = x.double() / s.double()[:, None]
    sure = ((quotient - quotient.floor()) - 0.5).abs() > 127 * U
    assert torch.equal(q[sure], tq[sure])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [64, 2048, 5000])
def test_quantiser_rows_apart(gpu, dtype, K):
    """A row with an infinity or NaN gets the scale NaN and codes 0; zeros and values
    below the smallest scale become 0; the rows beside them are what they are alone."""
    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.randn(6, K, generator=g, device=gpu).to(dtype)
    ref_q, ref_s = quantize_int8_token(x)
    bad = x.clone()
    bad[0, K // 2], bad[2, K - 1], bad[3, 0] = math.inf, math.nan, -math.inf
    bad[4] = 0
    q, s = quantize_int8_token(bad)
    for r in (0, 2, 3):
        assert torch.isnan(s[r]) and not q[r].any()
    assert not q[4].any() and s[4].item() == (torch.tensor(1e-12) * INV).item()
    for r in (1, 5):
        assert torch.equal(q[r], ref_q[r]) and s[r] == ref_s[r]


def test_quantiser_layouts(gpu):
    """Leading dimensions, rows apart, rows that are not aligned, transposed input, no rows."""
    base = torch.randn(8, 6, 200, device=gpu)
    for x in (base, base[:, 2, 4:68], base[:, 1, 3:70], base[0].t(), base[0, 0], base.to(torch.bfloat16)[:, 3, 1:130]):
        q, s = quantize_int8_token(x)
        rq, rs = exact_quantise(x)
        assert q.shape == x.shape and s.shape == x.shape[:-1]
        assert torch.equal(q.cpu(), rq) and torch.equal(s.cpu(), rs)
    q, s = quantize_int8_token(base[:0, 0])
    assert q.shape == (0, 200) and s.shape == (0,)


# ------------------------------------------------------------------ dense product
SHAPES = [(1, 16, 16), (1, 2048, 1536), (2, 64, 1), (7, 48, 33), (16, 1024, 130), (17, 1408, 512), (33, 512, 100),
          (64, 768, 2048), (65, 80, 257), (130, 2880, 64), (200, 640, 300), (256, 256, 512), (300, 1024, 1024),
          (513, 128, 640), (1000, 192, 777)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear(gpu, M, K, N, dtype):
    q, w = codes((M, K), 1, gpu, -128), codes((N, K), 2, gpu, -128)
    s, ws = scales((M,), 3, gpu), scales((N,), 4, gpu)
    got = w8a8_linear(q, s, w, ws, out_dtype=dtype)
    ref, mag = exact(q, s, w, ws)
    close(got, ref, mag, dtype)
    packed = quant.pack_int8_to_int32(w)
    assert torch.equal(w8a8_linear(q, s, packed, ws[:, None], out_dtype=dtype), got)


@pytest.mark.parametrize("M,K,N", [(3, 64, 40), (70, 272, 96), (300, 512, 600)])
@pytest.mark.parametrize("sdt", DTYPES)
@pytest.mark.parametrize("bdt", DTYPES)
def test_linear_bias_and_scale_types(gpu, M, K, N, sdt, bdt):
    q, w = codes((M, K), 5, gpu), codes((N, K), 6, gpu)
    s, ws = scales((M, 1), 7, gpu), scales((N,), 8, gpu, sdt)
    b = torch.randn(N, generator=torch.Generator().manual_seed(9)).to(gpu).to(bdt)
    ref, mag = exact(q, s[:, 0], w, ws, b)
    close(w8a8_linear(q, s, w, ws, bias=b, out_dtype=torch.float32), ref, mag, torch.float32)


@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (3, 5, 7), (20, 33, 18), (70, 1001, 40), (5, 12, 20)])
def test_linear_any_k(gpu, M, K, N):
    """K that is no multiple of 16 (and, packed, of 4 only)."""
    q, w = codes((M, K), 10, gpu), codes((N, K), 11, gpu)
    s, ws = scales((M,), 12, gpu), scales((N,), 13, gpu)
    ref, mag = exact(q, s, w, ws)
    got = w8a8_linear(q, s, w, ws, out_dtype=torch.float32)
    close(got, ref, mag, torch.float32)
    if K % 4 == 0:
        assert torch.equal(w8a8_linear(q, s, quant.pack_int8_to_int32(w), ws, out_dtype=torch.float32), got)


@pytest.mark.parametrize("M", [2, 40, 300])
def test_linear_strides(gpu, M):
    """Rows apart, rows that start off a 16-byte border, a transposed weight: the bits of
    the contiguous call."""
    K, N = 128, 96
    big = codes((M, 2 * K + 32), 14, gpu)
    w, s, ws = codes((K, N), 15, gpu).t(), scales((M, 2), 16, gpu)[:, 1], scales((N, 2), 17, gpu)[:, 0]
    for at in (0, 32, 5):
        q = big[:, at:at + K]
        ref = w8a8_linear(q.contiguous(), s.contiguous(), w.contiguous(), ws.contiguous())
        assert torch.equal(w8a8_linear(q, s, w, ws), ref)
    qt = codes((K, M), 18, gpu).t()
    assert torch.equal(w8a8_linear(qt, s, w, ws), w8a8_linear(qt.contiguous(), s, w, ws))


@pytest.mark.parametrize("M", [1, 50, 300])
def test_linear_longest_sum(gpu, M):
    """K at the limit with the largest products: the sum stays inside int32."""
    K, N = 131056, 48
    q = torch.full((M, K), -128, dtype=torch.int8, device=gpu)
    w = torch.full((N, K), -128, dtype=torch.int8, device=gpu)
    w[1::2] = 127
    s, ws = torch.ones(M, device=gpu), torch.ones(N, device=gpu)
    got = w8a8_linear(q, s, w, ws, out_dtype=torch.float32)
    want = torch.tensor([128.0 * 128 * K, -128.0 * 127 * K] * (N // 2), dtype=torch.float64, device=gpu).float()
    assert torch.equal(got, want.expand(M, N))


def test_linear_rows_do_not_depend_on_the_batch(gpu):
    """The sum is exact, so a row's bits are the same in every batch and tile."""
    K, N, M = 1024, 1536, 1200
    q, w, s, ws = codes((M, K), 20, gpu), codes((N, K), 21, gpu), scales((M,), 22, gpu), scales((N,), 23, gpu)
    full = w8a8_linear(q, s, w, ws)
    for lo, hi in ((0, 1), (5, 15), (100, 133), (300, 364), (0, 200), (600, 1112)):
        assert torch.equal(w8a8_linear(q[lo:hi], s[lo:hi], w, ws), full[lo:hi]), (lo, hi)


def test_linear_scales_of_any_size(gpu):
    """A NaN scale makes its own row NaN only; infinities and zero scales follow the formula."""
    q, w = codes((70, 64), 24, gpu), codes((32, 64), 25, gpu)
    s, ws = scales((70,), 26, gpu), scales((32,), 27, gpu)
    ref = w8a8_linear(q, s, w, ws)
    s2 = s.clone()
    s2[3], s2[40], s2[41] = math.nan, 0.0, 3e38
    got = w8a8_linear(q, s2, w, ws)
    assert torch.isnan(got[3]).all() and not got[40].any()
    keep = [i for i in range(70) if i not in (3, 40, 41)]
    assert torch.equal(got[keep], ref[keep])


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "swiglu_oai"])
@pytest.mark.parametrize("M,K,N", [(1, 64, 34), (20, 256, 96), (300, 512, 768), (40, 50, 26)])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_activation(gpu, act, M, K, N, bias):
    """h = act(gate) up.  With g and u off by 4 u of their magnitudes (3 of the product and
    one of what an order of operations may add) and the exponential by 4: silu and swiglu_oai are off by
    (4 (1 + |a g|) + 8) u relative per factor, gelu by 16 u |g| |u| absolutely, relu by
    the factors' own."""
    q, w = codes((M, K), 30, gpu), codes((N, K), 31, gpu)
    s, ws = scales((M,), 32, gpu) * 0.05, scales((N,), 33, gpu)
    b = torch.randn(N, generator=torch.Generator().manual_seed(3)).to(gpu) if bias else None
    y, mag = exact(q, s, w, ws, b)
    g, u, gm, um = y[:, :N // 2], y[:, N // 2:], mag[:, :N // 2], mag[:, N // 2:]
    if act == "silu":
        ref = g * torch.sigmoid(g) * u
        tol = (4 * gm * (1 + g.abs()) * u.abs() + 4 * um * g.abs() + 12 * (g * u).abs()) * U
    elif act == "gelu":
        ref = 0.5 * g * (1 + torch.erf(g / math.sqrt(2))) * u
        tol = (8 * gm * u.abs() + 8 * um * g.abs() + 16 * (g * u).abs()) * U
    elif act == "relu":
        ref = g.clamp_min(0) * u
        tol = (4 * gm * u.abs() + 4 * um * g.abs() + 4 * (g * u).abs()) * U
    else:
        gc, uc = g.clamp_max(7.0), u.clamp(-7.0, 7.0)
        ref = (uc + 1) * gc * torch.sigmoid(1.702 * gc)
        tol = (4 * gm * (1 + 1.702 * gc.abs()) * (uc + 1).abs() + 4 * (um + 1) * gc.abs() + 14 * (gc * (uc.abs() + 1)).abs()) * U
    got = w8a8_linear(q, s, w, ws, bias=b, activation=act, out_dtype=torch.float32)
    assert got.shape == ref.shape
    err = (got.double() - ref).abs()
    assert (err <= tol + 1e-37).all(), float((err - tol).max())


@pytest.mark.parametrize("M", [1, 5, 20, 40, 300])
@pytest.mark.parametrize("K", [256, 52])
def test_linear_row_index(gpu, M, K):
    """The C call reads rows through an index without experts too; one that names none gives zeros."""
    R, N = 70, 96
    q, s, w, ws = codes((R, K), 1, gpu), scales((R,), 2, gpu), codes((N, K), 3, gpu), scales((N,), 4, gpu)
    idx = torch.randint(0, R, (M,), generator=torch.Generator().manual_seed(M), dtype=torch.int32).to(gpu)
    idx[M // 2] = R if M > 1 else -1
    out = torch.full((M, N), 7.0, device=gpu)
    c = nat.FtmW8A8(q.data_ptr(), s.data_ptr(), w.data_ptr(), ws.data_ptr(), None, out.data_ptr(), None, idx.data_ptr(),
                    M, R, K, 0, N, K, 1, 0, nat.DT_F32, 0, nat.DT_F32, -1, 0.0, 0.0)
    nat.launch("ftm_w8a8_linear", nat.lib().ftm_w8a8_linear, q, ctypes.byref(c))
    at = idx.clamp(0, R - 1).long()
    ref = w8a8_linear(q[at], s[at], w, ws, out_dtype=torch.float32)
    ref[M // 2] = 0
    assert torch.equal(out, ref)


def test_linear_row_index_past_one_grid_dimension(gpu):
    """More tiles than workgroups that one grid dimension counts, through an index without experts."""
    R, K, N, M = 70, 16, 1, (2**24 - 1) * 64 + 100
    q, s, w, ws = codes((R, K), 1, gpu), scales((R,), 2, gpu), codes((N, K), 3, gpu), scales((N,), 4, gpu)
    idx = torch.arange(M, device=gpu, dtype=torch.int32).remainder_(R)
    idx[-1] = -1
    out = torch.full((M, N), 7.0, device=gpu, dtype=torch.bfloat16)
    c = nat.FtmW8A8(q.data_ptr(), s.data_ptr(), w.data_ptr(), ws.data_ptr(), None, out.data_ptr(), None, idx.data_ptr(),
                    M, R, K, 0, N, K, 1, 0, nat.DT_F32, 0, nat.DT_BF16, -1, 0.0, 0.0)
    nat.launch("ftm_w8a8_linear", nat.lib().ftm_w8a8_linear, q, ctypes.byref(c))
    ref = w8a8_linear(q, s, w, ws)
    assert out[-1] == 0
    for at in range(0, M - 1, 2**27):
        part = slice(at, min(at + 2**27, M - 1))
        assert torch.equal(out[part], ref[idx[part]])


def test_linear_empty_and_refused(gpu):
    q, s, w, ws = codes((4, 64), 1, gpu), scales((4,), 2, gpu), codes((32, 64), 3, gpu), scales((32,), 4, gpu)
    assert w8a8_linear(q[:0], s[:0], w, ws).shape == (0, 32)
    assert w8a8_linear(q, s, w[:0], ws[:0]).shape == (4, 0)
    for err, kw in ((TypeError, dict(x_int8=q.float())), (TypeError, dict(x_scale=s.half())),
                    (TypeError, dict(weight=w.float())), (TypeError, dict(weight_scale=ws.double())),
                    (TypeError, dict(out_dtype=torch.float64)), (TypeError, dict(bias=ws.double())),
                    (ValueError, dict(x_int8=q[:, :32])), (ValueError, dict(x_scale=s[:3])),
                    (ValueError, dict(weight_scale=ws[:5])), (ValueError, dict(bias=ws[:5])),
                    (ValueError, dict(activation="tanh")), (ValueError, dict(weight=w[None])),
                    (ValueError, dict(weight=w[:31], weight_scale=ws[:31], activation="silu")),
                    (RuntimeError, dict(weight=w.cpu()))):
        a = dict(x_int8=q, x_scale=s, weight=w, weight_scale=ws)
        a.update(kw)
        with pytest.raises(err):
            w8a8_linear(a.pop("x_int8"), a.pop("x_scale"), a.pop("weight"), a.pop("weight_scale"), **a)
    with pytest.raises(ValueError, match="131071"):
        w8a8_linear(q.repeat(1, 2049), s, w.repeat(1, 2049), ws)
    with pytest.raises(TypeError):
        quantize_int8_token(q)
    with pytest.raises(ValueError):
        quantize_int8_token(s.reshape(4, 1)[:, :0])


# ------------------------------------------------------------------ grouped product
def segments(counts, gpu, tail=0):
    off = torch.zeros(len(counts) + 1, dtype=torch.int32)
    off[1:] = torch.tensor(counts).cumsum(0)
    return off.to(gpu), int(off[-1]) + tail


GROUPS = {
    "one_row": ([0, 1, 0], 0),
    "empty_experts": ([0, 0, 5, 0, 17, 0], 3),
    "no_rows": ([0, 0, 0, 0], 9),
    "one_expert_has_all": ([0, 300, 0, 0, 0, 0, 0, 0], 0),
    "ragged": ([16, 15, 17, 1, 64, 65, 130, 33], 40),
    "many": ([(7 * i) % 5 for i in range(512)], 2),
    "full": ([64] * 9, 0),
    "large": ([400, 3, 700, 256], 130),
    "about_128": ([128, 140, 117, 96, 161, 130, 160, 129, 127], 5),
}


@pytest.mark.parametrize("name", sorted(GROUPS))
@pytest.mark.parametrize("K,N", [(64, 48), (272, 33), (256, 300), (40, 10), (384, 2100), (176, 1900), (384, 7300),
                                 (144, 7300)])
@pytest.mark.parametrize("act", [None, "silu"])
def test_grouped(gpu, name, K, N, act):
    """Every expert's rows are the dense product's bits, the rows of no expert zeros; packed
    the same."""
    counts, tail = GROUPS[name]
    N = N // 2 * 2 if act else N
    E = len(counts)
    off, P = segments(counts, gpu, tail)
    q, s = codes((P, K), 1, gpu), scales((P,), 2, gpu)
    w, ws = codes((E, N, K), 3, gpu), scales((E, N), 4, gpu)
    b = scales((E, N), 5, gpu)
    got = w8a8_grouped_linear(q, s, off, w, ws, bias=b, activation=act, out_dtype=torch.float32)
    ends = off.tolist()
    for e in range(E):
        lo, hi = ends[e], ends[e + 1]
        if hi > lo:
            ref = w8a8_linear(q[lo:hi], s[lo:hi], w[e], ws[e], bias=b[e], activation=act, out_dtype=torch.float32)
            assert torch.equal(got[lo:hi], ref), e
    assert not got[ends[-1]:].any()
    if K % 4 == 0:
        again = w8a8_grouped_linear(q, s, off, quant.pack_int8_to_int32(w), ws[..., None], bias=b, activation=act,
                                    out_dtype=torch.float32)
        assert torch.equal(again, got)


@pytest.mark.parametrize("rows_per", [1, 20, 90, 300])
def test_grouped_row_index(gpu, rows_per):
    """Rows through an index: repeated, in any order, and -1 or past the end: zeros."""
    E, K, N, M = 5, 128, 80, 37
    off, P = segments([rows_per] * E, gpu, 7)
    g = torch.Generator(device=gpu).manual_seed(7)
    idx = torch.randint(0, M, (P,), generator=g, device=gpu, dtype=torch.int32)
    idx[P // 2], idx[0] = -1, M
    q, s = codes((M, K), 1, gpu), scales((M,), 2, gpu)
    w, ws = codes((E, N, K), 3, gpu), scales((E, N), 4, gpu)
    got = w8a8_grouped_linear(q, s, off, w, ws, row_index=idx)
    at = idx.clamp(0, M - 1).long()
    ref = w8a8_grouped_linear(q[at], s[at], off, w, ws)
    ref[P // 2], ref[0] = 0, 0
    assert torch.equal(got, ref)
    empty = w8a8_grouped_linear(q[:0], s[:0], off, w, ws, row_index=idx)
    assert empty.shape == (P, N) and not empty.any()


def test_grouped_rows_without_an_expert_are_not_read(gpu):
    """NaN scales behind the last expert's rows leave zeros there and nothing elsewhere."""
    off, P = segments([3, 0, 40], gpu, 20)
    q, s = codes((P, 64), 1, gpu), scales((P,), 2, gpu)
    s[43:] = math.nan
    out = w8a8_grouped_linear(q, s, off, codes((3, 32, 64), 3, gpu), scales((3, 32), 4, gpu))
    assert not out[43:].any() and not torch.isnan(out).any()


@pytest.mark.parametrize("act", [None, "silu"])
def test_grouped_weights_past_32_bits(gpu, act):
    """The last expert's weights, scales and rows lie more than 2^32 bytes behind the first's."""
    E, N, K = 40, 8192, 16384
    w, ws = torch.empty((E, N, K), dtype=torch.int8, device=gpu), scales((E, N), 4, gpu)
    w[E - 1] = codes((N, K), 3, gpu)
    w[0] = codes((N, K), 5, gpu)
    for rows in (3, 70):  # split K, tiles
        counts = [0] * E
        counts[0] = counts[E - 1] = rows
        off, P = segments(counts, gpu)
        q, s = codes((P, K), 1, gpu), scales((P,), 2, gpu)
        got = w8a8_grouped_linear(q, s, off, w, ws, activation=act)
        for e, at in ((0, slice(0, rows)), (E - 1, slice(rows, P))):
            assert torch.equal(got[at], w8a8_linear(q[at], s[at], w[e], ws[e], activation=act))


@pytest.mark.parametrize("K,N", [(8192, 96), (8208, 40)])
def test_rows_past_32_bits(gpu, K, N):
    """Tokens of more than 2^32 bytes, dense, by expert and through an index; 2^31 results."""
    M = 2**32 // K + 1000
    x = torch.zeros((M, K), dtype=torch.float16, device=gpu)  # 2^33 bytes of values, 2^32 of codes
    last = torch.randn(300, K, generator=torch.Generator(device=gpu).manual_seed(3), device=gpu).half()
    x[-300:] = last
    q, s = quantize_int8_token(x)
    del x
    lq, ls = quantize_int8_token(last)
    assert torch.equal(q[-300:], lq) and torch.equal(s[-300:], ls)
    w, ws = codes((2, N, K), 3, gpu), scales((2, N), 4, gpu)
    ref = w8a8_linear(lq, ls, w[1], ws[1])
    assert torch.equal(w8a8_linear(q, s, w[1], ws[1])[-300:], ref)
    off = torch.tensor([0, 5, M], dtype=torch.int32, device=gpu)
    assert torch.equal(w8a8_grouped_linear(q, s, off, w, ws)[-300:], ref)
    idx = torch.arange(M - 300, M, dtype=torch.int32, device=gpu)
    off = torch.tensor([0, 0, 300], dtype=torch.int32, device=gpu)
    assert torch.equal(w8a8_grouped_linear(q, s, off, w, ws, row_index=idx), ref)


@pytest.mark.parametrize("M,K", [(2**24 + 70, 3), (2**24 + 70, 24), (2**20 + 70, 2064)])
def test_more_rows_than_one_grid_dimension(gpu, M, K):
    """A workgroup a row, or for four rows, past the threads that one dimension counts."""
    x = torch.randn(M, K, generator=torch.Generator(device=gpu).manual_seed(5), device=gpu, dtype=torch.bfloat16)
    q, s = quantize_int8_token(x)
    at = torch.cat([torch.arange(0, 9), torch.arange(2**20 - 4, 2**20 + 4), torch.arange(M - 80, M)]).to(gpu)
    rq, rs = exact_quantise(x[at])
    assert torch.equal(q[at].cpu(), rq) and torch.equal(s[at].cpu(), rs)
    for N in (2, 260) if K < 30 else (2,):  # 17.8 M items of 16 x 16 the second
        w, ws = codes((N, K), 3, gpu), scales((N,), 4, gpu)
        assert torch.equal(w8a8_linear(q, s, w, ws)[at], w8a8_linear(q[at], s[at], w, ws))


def test_rows_over_one_another(gpu):
    """Rows that share memory (expanded, overlapping), and a single row of any stride."""
    w, ws = codes((40, 64), 3, gpu), scales((40,), 4, gpu)
    one = torch.randn(1, 64, device=gpu)
    q, s = quantize_int8_token(one)
    for M in (3, 70):
        assert torch.equal(w8a8_linear(q.expand(M, 64), s.expand(M), w, ws), w8a8_linear(q.repeat(M, 1), s.repeat(M), w, ws))
        assert torch.equal(fused_w8a8_linear(one.expand(M, 64), w, ws), fused_w8a8_linear(one.repeat(M, 1), w, ws))
    flat = codes((100,), 5, gpu)
    lap = flat.as_strided((5, 64), (7, 1))
    assert torch.equal(w8a8_linear(lap, s.repeat(5), w, ws), w8a8_linear(lap.clone(), s.repeat(5), w, ws))
    odd = flat.as_strided((1, 64), (7, 1))
    assert torch.equal(w8a8_linear(odd, s, w, ws), w8a8_linear(odd.clone(), s, w, ws))


@pytest.mark.parametrize("N", [16384, 16400])
def test_results_past_32_bits(gpu, N):
    M, K = 2**32 // (2 * N) + 300, 64
    q, s = codes((M, K), 1, gpu), scales((M,), 2, gpu)
    w, ws = codes((N, K), 3, gpu), scales((N,), 4, gpu)
    got = w8a8_linear(q, s, w, ws, out_dtype=torch.bfloat16)
    for at in (slice(0, 260), slice(M - 260, M)):
        assert torch.equal(got[at], w8a8_linear(q[at], s[at], w, ws, out_dtype=torch.bfloat16))


def test_grouped_refused(gpu):
    off, P = segments([3, 4], gpu)
    q, s, w, ws = codes((P, 64), 1, gpu), scales((P,), 2, gpu), codes((2, 32, 64), 3, gpu), scales((2, 32), 4, gpu)
    for err, kw in ((TypeError, dict(offsets=off.long())), (ValueError, dict(offsets=off[:2])),
                    (ValueError, dict(offsets=off.repeat(2)[::2])), (TypeError, dict(row_index=off.long())),
                    (ValueError, dict(weight=w[0])), (ValueError, dict(weight_scale=ws[:1]))):
        a = dict(offsets=off, weight=w, weight_scale=ws)
        a.update(kw)
        with pytest.raises(err):
            w8a8_grouped_linear(q, s, a.pop("offsets"), a.pop("weight"), a.pop("weight_scale"), **a)
    with pytest.raises(ValueError, match="512"):
        w8a8_grouped_linear(q, s, torch.zeros(514, dtype=torch.int32, device=gpu), codes((513, 2, 64), 1, gpu),
                            scales((513, 2), 1, gpu))


# ------------------------------------------------------------------ together
def moe_inputs(gpu, T, E, H, I, k, dtype, seed=0, drop=False):
    g = torch.Generator(device=gpu).manual_seed(seed)
    w1, s1 = quant.quantize_int8_channel(torch.randn(E, 2 * I, H, generator=g, device=gpu) * 0.02)
    w2, s2 = quant.quantize_int8_channel(torch.randn(E, H, I, generator=g, device=gpu) * 0.02)
    x = torch.randn(T, H, generator=g, device=gpu).to(dtype)
    top, ids = torch.randn(T, E, generator=g, device=gpu).topk(k, dim=-1)
    if drop:
        ids = torch.where(ids < E // 2, ids, torch.full_like(ids, -1))
    return x, w1, s1, w2, s2, ids, torch.softmax(top, dim=-1)


def exact_moe(x, w1, s1, w2, s2, ids, tw):
    def quantise(v):
        s = (v.abs().amax(dim=1).clamp_min(1e-12).float() * INV.to(v.device)).double()
        return (v / s[:, None]).round().clamp(-127, 127) * s[:, None]

    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    v = quantise(x.double())
    for e in range(w1.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        gu = v[t] @ (w1[e].double() * s1[e].double()[:, None]).t().contiguous()
        gate, up = gu.chunk(2, dim=1)
        y = quantise(gate * torch.sigmoid(gate) * up) @ (w2[e].double() * s2[e].double()[:, None]).t().contiguous()
        out.index_add_(0, t, y * tw[t, j].double()[:, None])
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,H,I,k,drop", [(1, 8, 128, 64, 2, False), (5, 16, 256, 128, 4, True),
                                            (200, 16, 512, 96, 4, False), (600, 4, 256, 256, 2, False),
                                            (33, 60, 128, 176, 4, True)])
def test_moe(gpu, dtype, T, E, H, I, k, drop):
    """The run of sort, quantiser, products and combine against 64 bits in the 2-norm: half a
    step of the output type, and the codes of h that its fp32 error (below 2^-19 relative,
    see test_linear_activation) moves over a border: at most 127 * 2^-18 of them by one
    step, the codes' norm being at least 127 / sqrt(I) a value: sqrt(127 * 2^-18) * sqrt(I) / 127."""
    x, w1, s1, w2, s2, ids, tw = moe_inputs(gpu, T, E, H, I, k, dtype, seed=T, drop=drop)
    got = fused_w8a8_moe(x, w1, s1, w2, s2, ids, tw)
    ref = exact_moe(x, w1, s1, w2, s2, ids, tw)
    assert got.dtype == dtype and got.shape == x.shape
    tol = half_step(dtype) + math.sqrt(127 * 2.0 ** -18) * math.sqrt(I) / 127
    assert ((got.double() - ref).norm() / ref.norm()).item() <= tol
    packed = fused_w8a8_moe(x, quant.pack_int8_to_int32(w1), s1[..., None], quant.pack_int8_to_int32(w2),
                            s2[..., None], ids.int(), tw)
    assert torch.equal(packed, got)


def test_moe_is_its_operators(gpu):
    x, w1, s1, w2, s2, ids, tw = moe_inputs(gpu, 70, 12, 256, 128, 3, torch.bfloat16, drop=True)
    b1, b2 = torch.randn(12, 256, device=gpu), torch.randn(12, 256, device=gpu).bfloat16()
    sort = sort_tokens(ids, 12)
    q, s = quantize_int8_token(x)
    h = w8a8_grouped_linear(q, s, sort.offsets, w1, s1, row_index=sort.token_of_row, bias=b1, activation="gelu",
                            out_dtype=torch.float32)
    q, s = quantize_int8_token(h)
    y = w8a8_grouped_linear(q, s, sort.offsets, w2, s2, bias=b2, out_dtype=torch.float32)
    ref = combine_tokens(y, tw, sort, out_dtype=torch.bfloat16)
    assert torch.equal(fused_w8a8_moe(x, w1, s1, w2, s2, ids, tw, activation="gelu", w1_bias=b1, w2_bias=b2), ref)


def test_moe_refused_and_empty(gpu):
    x, w1, s1, w2, s2, ids, tw = moe_inputs(gpu, 6, 4, 64, 32, 2, torch.bfloat16)
    assert fused_w8a8_moe(x[:0], w1, s1, w2, s2, ids[:0], tw[:0]).shape == (0, 64)
    assert not fused_w8a8_moe(x, w1, s1, w2, s2, torch.full_like(ids, -1), tw).any()
    for kw in (dict(ids=ids[:5]), dict(tw=tw[:, :1]), dict(x=x[0])):
        a = dict(x=x, ids=ids, tw=tw)
        a.update(kw)
        with pytest.raises(ValueError):
            fused_w8a8_moe(a["x"], w1, s1, w2, s2, a["ids"], a["tw"])
    with pytest.raises(ValueError, match="activation"):
        fused_w8a8_moe(x, w1, s1, w2, s2, ids, tw, activation="tanh")


@pytest.mark.parametrize("dtype", DTYPES)
def test_expert_and_projection(gpu, dtype):
    """The fused calls are the quantiser and the product."""
    x, w1, s1, w2, s2, _, _ = moe_inputs(gpu, 40, 1, 256, 128, 1, dtype)
    q, s = quantize_int8_token(x)
    b = torch.randn(256, device=gpu).to(dtype)
    assert torch.equal(fused_w8a8_linear(x, w1[0], s1[0], bias=b), w8a8_linear(q, s, w1[0], s1[0], bias=b, out_dtype=dtype))
    h = w8a8_linear(q, s, w1[0], s1[0], activation="silu", out_dtype=torch.float32)
    ref = w8a8_linear(*quantize_int8_token(h), w2[0], s2[0], out_dtype=dtype)
    assert torch.equal(fused_w8a8_expert_forward(x, w1[0], s1[0], w2[0], s2[0], intermediate=128), ref)
    with pytest.raises(ValueError):
        fused_w8a8_expert_forward(x, w1[0], s1[0], w2[0], s2[0], intermediate=64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 2048, 1536), (1, 16, 1), (2, 176, 33), (3, 1408, 64), (4, 2048, 40), (4, 48, 300),
                                   (5, 64, 64), (1, 8192, 48), (1, 8208, 48), (2, 50, 20)])
def test_projection_of_few_tokens(gpu, dtype, M, K, N):
    """Few tokens are quantised inside the product: the bits of the two calls, rows with
    infinities and NaN, rows apart, biased and packed."""
    gen = torch.Generator(device=gpu).manual_seed(K)
    big = torch.randn(M, 2 * K, generator=gen, device=gpu).to(dtype)
    w, ws = codes((N, K), 1, gpu), scales((N,), 2, gpu)
    b = torch.randn(N, generator=gen, device=gpu)
    for x in (big[:, :K].contiguous(), big[:, K:], big[:, 1:K + 1]):
        x = x.clone() if x.is_contiguous() else x
        q, s = quantize_int8_token(x)
        ref = w8a8_linear(q, s, w, ws, bias=b, out_dtype=torch.float32)
        assert torch.equal(fused_w8a8_linear(x, w, ws, bias=b, out_dtype=torch.float32), ref)
        if K % 4 == 0:
            assert torch.equal(fused_w8a8_linear(x, quant.pack_int8_to_int32(w), ws, bias=b, out_dtype=torch.float32), ref)
    bad = big[:, :K].contiguous()
    ref = fused_w8a8_linear(bad, w, ws)
    bad[M - 1, K // 2] = math.inf
    bad[0, K - 1] = math.nan
    got = fused_w8a8_linear(bad, w, ws)
    assert torch.isnan(got[0]).all() and torch.isnan(got[M - 1]).all() and torch.equal(got[1:-1], ref[1:-1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,H,I,k", [(1, 8, 128, 64, 2), (4, 16, 1024, 512, 2), (8, 64, 176, 48, 3), (2, 300, 256, 96, 8)])
def test_moe_of_few_tokens_is_its_operators(gpu, dtype, T, E, H, I, k):
    """Up to two rows an expert: both products quantise their rows themselves."""
    x, w1, s1, w2, s2, ids, tw = moe_inputs(gpu, T, E, H, I, k, dtype, seed=3, drop=True)
    if T > 1:
        ids[1] = ids[0]  # an expert with several rows
    sort = sort_tokens(ids, E)
    q, s = quantize_int8_token(x)
    h = w8a8_grouped_linear(q, s, sort.offsets, w1, s1, row_index=sort.token_of_row, activation="silu",
                            out_dtype=torch.float32)
    y = w8a8_grouped_linear(*quantize_int8_token(h), sort.offsets, w2, s2, out_dtype=torch.float32)
    ref = combine_tokens(y, tw, sort, out_dtype=dtype)
    assert torch.equal(fused_w8a8_moe(x, w1, s1, w2, s2, ids, tw), ref)


def test_moe_in_a_graph_and_on_streams(gpu):
    """Captured and replayed over new inputs, with eager work between the replays; two
    streams at once."""
    x, w1, s1, w2, s2, ids, tw = moe_inputs(gpu, 64, 16, 256, 128, 4, torch.bfloat16)
    run = MoeGraphRunner()
    out = run.capture(lambda: fused_w8a8_moe(x, w1, s1, w2, s2, ids, tw))
    for seed in range(3):
        nx, *_, nids, ntw = moe_inputs(gpu, 64, 16, 256, 128, 4, torch.bfloat16, seed=seed + 1, drop=seed == 1)
        x.copy_(nx), ids.copy_(nids), tw.copy_(ntw)
        run.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fused_w8a8_moe(x, w1, s1, w2, s2, ids, tw)), seed
    streams = [torch.cuda.Stream(device=gpu) for _ in range(2)]
    ref = fused_w8a8_moe(x, w1, s1, w2, s2, ids, tw)
    torch.cuda.synchronize()
    got = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            got.append(fused_w8a8_moe(x, w1, s1, w2, s2, ids, tw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in got)
