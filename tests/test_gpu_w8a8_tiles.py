"""The int8 product where it takes LDS tiles (many rows, dense and by expert, plain
and through an index), against arithmetic in 64 bits.

Tolerances: the integer sum is exact; its rounding to fp32, the token scale and
the channel scale (with the bias) are one rounding each, 2^-24 relative, and
the output rounds once, by half a step of its type."""
import math

import pytest
import torch

from ftmoe import quant
from ftmoe.kernel.fused_w8a8_linear import fused_w8a8_expert_forward
from ftmoe.kernel.fused_w8a8_moe import fused_w8a8_moe
from ftmoe.kernel.w8a8_linear import w8a8_grouped_linear, w8a8_linear
from test_gpu_w8a8 import DTYPES, U, close, codes, exact, exact_moe, half_step, moe_inputs, scales

pytestmark = pytest.mark.gpu
ACTS = ("silu", "gelu", "relu", "swiglu_oai")


# ------------------------------------------------------------------ values that are not finite
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,K,N", [(3, 64, 34), (20, 256, 96), (300, 512, 768), (1000, 256, 2200), (40, 50, 26)])
def test_activation_keeps_a_nan(gpu, act, M, K, N):
    """A token with the scale NaN has NaN results under every activation (a clamp does not
    turn them into its limit), and so has a channel whose gate or up scale is NaN; all
    others are what they are without."""
    q, w = codes((M, K), 40, gpu), codes((N, K), 41, gpu)
    s, ws = scales((M,), 42, gpu) * 0.05, scales((N,), 43, gpu)
    ref = w8a8_linear(q, s, w, ws, activation=act, out_dtype=torch.float32)
    s[M // 2], ws[1], ws[N // 2 + 3] = math.nan, math.nan, math.nan
    got = w8a8_linear(q, s, w, ws, activation=act, out_dtype=torch.float32)
    bad = torch.zeros_like(ref, dtype=torch.bool)
    bad[M // 2], bad[:, 1], bad[:, 3] = True, True, True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], ref[~bad])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T", [1, 6, 300])
def test_layers_keep_a_token_that_is_not_finite(gpu, act, T):
    """A token with an infinity or NaN leaves the expert and the expert layer as NaN."""
    x, w1, s1, w2, s2, ids, tw = moe_inputs(gpu, T, 8, 128, 64, 2, torch.bfloat16)
    for v in (math.inf, math.nan):
        x[T // 2, 5] = v
        out = fused_w8a8_moe(x, w1, s1, w2, s2, ids, tw, activation=act)
        one = fused_w8a8_expert_forward(x, w1[0], s1[0], w2[0], s2[0], intermediate=64, activation=act)
        for y in (out, one):
            nan = torch.isnan(y)
            assert nan[T // 2].all() and int(nan.sum()) == y.shape[1]


# ------------------------------------------------------------------ arithmetic of the activations
def exact_act(act, g, u, gm, um):
    """(act(g) u, tolerance) in 64 bits for sums g and u of magnitudes gm and um, each off by
    at most 4 units of its magnitude (3 roundings of the product, one for an order of
    operations) and the exponential by 4: silu and swiglu_oai (4 (1 + |a g|) + 8) u relative
    per factor, gelu 16 u |g| |u| absolutely, relu the factors' own."""
    if act == "silu":
        ref = g * torch.sigmoid(g) * u
        tol = 4 * gm * (1 + g.abs()) * u.abs() + 4 * um * g.abs() + 12 * (g * u).abs()
    elif act == "gelu":
        ref = 0.5 * g * (1 + torch.erf(g / math.sqrt(2))) * u
        tol = 8 * gm * u.abs() + 8 * um * g.abs() + 16 * (g * u).abs()
    elif act == "relu":
        ref = g.clamp_min(0) * u
        tol = 4 * gm * u.abs() + 4 * um * g.abs() + 4 * (g * u).abs()
    else:
        gc, uc = g.clamp_max(7.0), u.clamp(-7.0, 7.0)
        ref = (uc + 1) * gc * torch.sigmoid(1.702 * gc)
        tol = 4 * gm * (1 + 1.702 * gc.abs()) * (uc + 1).abs() + 4 * (um + 1) * gc.abs() + 14 * (gc * (uc.abs() + 1)).abs()
    return ref, tol * U + 1e-37


def check_act(got, act, y, mag):
    n = y.shape[1] // 2
    ref, tol = exact_act(act, y[:, :n], y[:, n:], mag[:, :n], mag[:, n:])
    err = (got.double() - ref).abs()
    assert got.shape == ref.shape and (err <= tol).all(), float((err - tol).max())


# ------------------------------------------------------------------ dense tiles
# Rows and weight rows (with an activation: output channels x 2) for which the product
# takes tiles of 64, 128 and 256 tokens x 256 weight rows: the last row tile and the last
# column tile are partly filled.
DENSE = {64: (1000, 1100), 128: (1000, 5020), 256: (1000, 10140)}


@pytest.mark.parametrize("rows", sorted(DENSE))
@pytest.mark.parametrize("K", [384, 512, 400, 48])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [False, True])
def test_dense_tiles(gpu, rows, K, dtype, bias):
    """K a multiple of 128 and not, and below one step; plain and packed weights."""
    M, N = DENSE[rows]
    q, w = codes((M, K), 1, gpu, -128), codes((N, K), 2, gpu, -128)
    s, ws = scales((M,), 3, gpu), scales((N,), 4, gpu)
    b = torch.randn(N, generator=torch.Generator(device=gpu).manual_seed(5), device=gpu).to(dtype) if bias else None
    ref, mag = exact(q, s, w, ws, b)
    got = w8a8_linear(q, s, w, ws, bias=b, out_dtype=dtype)
    close(got, ref, mag, dtype)
    assert torch.equal(w8a8_linear(q, s, quant.pack_int8_to_int32(w), ws[:, None], bias=b, out_dtype=dtype), got)


@pytest.mark.parametrize("rows", sorted(DENSE))
@pytest.mark.parametrize("K", [384, 400])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [False, True])
def test_dense_tiles_with_activation(gpu, rows, K, act, bias):
    M, N = DENSE[rows]
    q, w = codes((M, K), 6, gpu), codes((N, K), 7, gpu)
    s, ws = scales((M,), 8, gpu) * 0.05, scales((N,), 9, gpu)
    b = torch.randn(N, generator=torch.Generator(device=gpu).manual_seed(5), device=gpu) if bias else None
    y, mag = exact(q, s, w, ws, b)
    got = w8a8_linear(q, s, w, ws, bias=b, activation=act, out_dtype=torch.float32)
    check_act(got, act, y, mag)
    packed = w8a8_linear(q, s, quant.pack_int8_to_int32(w), ws, bias=b, activation=act, out_dtype=torch.float32)
    assert torch.equal(packed, got)
    for dtype in DTYPES[:2]:  # (the same fp32 values, rounded once)
        assert torch.equal(w8a8_linear(q, s, w, ws, bias=b, activation=act, out_dtype=dtype), got.to(dtype))


# ------------------------------------------------------------------ tiles by expert, through an index
# Experts, mean rows of each and weight rows for which a grouped product takes tiles of 64
# tokens (weights of few rows kept out of the caches where K is a multiple of 128), 64, 128
# and 160.
GROUPED = {"64_few": (40, 20, 760), "64": (9, 64, 1500), "128": (16, 100, 4036), "160": (8, 300, 4036)}


def experts(name, gpu, head=0, tail=0):
    """Offsets with uneven experts, one of them empty, rows of no expert before and behind."""
    E, mean, N = GROUPED[name]
    counts = [mean + (-1) ** i * (i * 5 % (mean // 2)) for i in range(E)]
    counts[E // 2], counts[0] = 0, counts[0] + counts[E // 2]
    off = torch.tensor([0, *counts]).cumsum(0) + head
    return E, N, off.to(torch.int32).to(gpu), int(off[-1]) + tail


def exact_grouped(q, s, off, w, ws, bias, index, P):
    """(sums, magnitudes, rows that have any) in 64 bits."""
    N, ends = w.shape[1], off.tolist()
    y = torch.zeros(P, N, dtype=torch.float64, device=q.device)
    mag, live = torch.zeros_like(y), torch.zeros(P, dtype=torch.bool, device=q.device)
    for e in range(w.shape[0]):
        lo, hi = ends[e], ends[e + 1]
        if lo == hi:
            continue
        src = index[lo:hi].long()
        live[lo:hi] = (src >= 0) & (src < q.shape[0])
        at = src.clamp(0, q.shape[0] - 1)
        y[lo:hi], mag[lo:hi] = exact(q[at], s[at], w[e], ws[e], None if bias is None else bias[e])
    return y, mag, live


@pytest.mark.parametrize("name", sorted(GROUPED))
@pytest.mark.parametrize("K", [384, 128, 400, 48])
@pytest.mark.parametrize("act", [None, "silu", "swiglu_oai"])
@pytest.mark.parametrize("indexed", [True, False])
def test_grouped_tiles(gpu, name, K, act, indexed):
    """Rows in order or through an index that repeats rows and names none (-1, or past the last)
    in the first, a middle and the last row of the experts; rows before the first expert
    and behind the last are zeros."""
    E, N, off, P = experts(name, gpu, head=11, tail=70)
    R = 500 if indexed else P
    q, s = codes((R, K), 1, gpu, -128), scales((R,), 2, gpu) * (0.05 if act else 1.0)
    w, ws, b = codes((E, N, K), 3, gpu, -128), scales((E, N), 4, gpu), scales((E, N), 5, gpu)
    if indexed:
        index = torch.randint(0, R, (P,), generator=torch.Generator(device=gpu).manual_seed(6), device=gpu,
                              dtype=torch.int32)
        ends = off.tolist()
        for i, (lo, hi) in enumerate(zip(ends, ends[1:])):
            if hi > lo:
                index[lo], index[(lo + hi) // 2], index[hi - 1] = (-1, R, R + 7) if i % 2 else (R, -1, -5)
    else:
        index = torch.arange(P, device=gpu, dtype=torch.int32)
    y, mag, live = exact_grouped(q, s, off, w, ws, b, index, P)
    kw = dict(row_index=index if indexed else None, bias=b, activation=act)
    got = w8a8_grouped_linear(q, s, off, w, ws, out_dtype=torch.float32, **kw)
    assert not got[~live].any()
    if act is None:
        close(got[live], y[live], mag[live], torch.float32)
    else:
        check_act(got[live], act, y[live], mag[live])
    packed = quant.pack_int8_to_int32(w)
    assert torch.equal(w8a8_grouped_linear(q, s, off, packed, ws[..., None], out_dtype=torch.float32, **kw), got)
    for dtype in DTYPES[:2]:
        half = w8a8_grouped_linear(q, s, off, w, ws, out_dtype=dtype, **kw)
        assert torch.equal(half, got.to(dtype))


@pytest.mark.parametrize("K", [128, 50])
@pytest.mark.parametrize("counts", [[0, 3, 0, 1], [40, 0, 17, 300]])
def test_grouped_rows_before_the_first_expert(gpu, K, counts):
    """The kernels for few rows and for any K: rows before the first offset become zeros."""
    E, N, head = len(counts), 40, 37
    off = (torch.tensor([0, *counts]).cumsum(0) + head).to(torch.int32).to(gpu)
    P = head + sum(counts) + 5
    q, s = codes((P, K), 1, gpu), scales((P,), 2, gpu)
    w, ws = codes((E, N, K), 3, gpu), scales((E, N), 4, gpu)
    y, mag, live = exact_grouped(q, s, off, w, ws, None, torch.arange(P, device=gpu), P)
    got = w8a8_grouped_linear(q, s, off, w, ws, out_dtype=torch.float32)
    assert not got[~live].any()
    close(got, y, mag, torch.float32)


# ------------------------------------------------------------------ the expert layer on tiles
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,H,I,k,drop", [(16, 128, 1024, 512, 8, False), (2000, 32, 1024, 640, 2, False),
                                            (1500, 32, 1024, 1104, 2, False), (3200, 32, 1024, 640, 4, False),
                                            (3200, 32, 1040, 656, 4, True)])
def test_moe_on_tiles(gpu, dtype, T, E, H, I, k, drop):
    """Both products on tiles of 64 (few rows and more), 128 and 160 tokens, against 64 bits in the
    2-norm: half a step of the output type, and the codes of h that its fp32 error (below 2^-19
    relative) moves over a border: at most 127 * 2^-18 of them by one step, the codes' norm
    being at least 127 / sqrt(I) a value: sqrt(127 * 2^-18) * sqrt(I) / 127."""
    x, w1, s1, w2, s2, ids, tw = moe_inputs(gpu, T, E, H, I, k, dtype, seed=T, drop=drop)
    got = fused_w8a8_moe(x, w1, s1, w2, s2, ids, tw)
    ref = exact_moe(x, w1, s1, w2, s2, ids, tw)
    assert got.dtype == dtype and got.shape == x.shape
    tol = half_step(dtype) + math.sqrt(127 * 2.0 ** -18) * math.sqrt(I) / 127
    assert ((got.double() - ref).norm() / ref.norm()).item() <= tol
    packed = fused_w8a8_moe(x, quant.pack_int8_to_int32(w1), s1[..., None], quant.pack_int8_to_int32(w2),
                            s2[..., None], ids.int(), tw)
    assert torch.equal(packed, got)
