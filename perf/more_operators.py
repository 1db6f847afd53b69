"""MXFP4 activations times MXFP4 weights, as measurable cases.

A case is one call, or the few calls that belong together, of public entry
points:

* ``quantise`` -- ``quantize_mxfp4`` and ``dequantize_mxfp4_blocks``: activations
  to 4-bit codes with one power of two per 32 of them, and the values these stand for;
* ``linear``   -- ``fused_w4a4_linear``: tokens quantised on the way, times a
  weight of the same format;
* ``grouped``  -- ``quantize_mxfp4`` + ``w4a4_grouped_linear``: rows sorted by
  expert, each expert with its own weight, ``gate_up`` read through the sort and with
  its gated activation;
* ``moe``      -- ``fused_w4a4_moe``: the routed experts of one layer.

``own`` selects the framework's operators; without it ``run`` computes the
same in elementary torch operations.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "freetoken-intel_amd"))

own = False
DEV = "cuda"
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
ALPHA, LIMIT = 1.702, 7.0  # of the clamped gate (swiglu_oai)

# Expert layers: those of the benchmark's configurations (16 experts of 512, 128
# of 768, 256 of 512, 32 of 2880 with biases and the clamped gate), and generic ones.
LAYERS = {
    "e16": dict(E=16, H=1024, I=512, k=2, act="silu", bias=False),
    "e128": dict(E=128, H=2048, I=768, k=8, act="silu", bias=False),
    "e256": dict(E=256, H=2048, I=512, k=8, act="silu", bias=False),
    "e32": dict(E=32, H=2880, I=2880, k=4, act="swiglu_oai", bias=True),
    "e60": dict(E=60, H=2048, I=1408, k=4, act="silu", bias=False),
    "e64": dict(E=64, H=2048, I=1024, k=6, act="silu", bias=False),
}
# one projection, [K, N]: gate_up and down of those experts, and generic dense ones
LINEAR = ((2048, 1536), (768, 2048), (2048, 1024), (1024, 1024), (1408, 2048), (2880, 5760), (4096, 4096),
          (4096, 12288), (11008, 4096))


def _quantise(M, K, dtype, name=None):
    c = dict(kind="quantise", M=M, K=K, dtype=dtype)
    return dict(c, name=name) if name else c


def _linear(M, K, N, dtype, bias=False, name=None):
    c = dict(kind="linear", M=M, K=K, N=N, dtype=dtype, bias=bias)
    return dict(c, name=name) if name else c


def _grouped(layer, which, T, dtype, name=None):
    c = dict(kind="grouped", T=T, which=which, dtype=dtype, **LAYERS[layer])
    return dict(c, name=name) if name else c


def _moe(layer, T, dtype, name=None):
    c = dict(kind="moe", T=T, dtype=dtype, **LAYERS[layer])
    return dict(c, name=name) if name else c


def listed():
    return [
        # a decode batch's activations, rows of an odd number of blocks
        _quantise(64, 2880, "bf16", name="quantise_64"),
        # a prefill chunk's
        _quantise(8192, 4096, "bf16", name="quantise_8192"),
        # one decoded token through one expert-sized projection: latency
        _linear(1, 2048, 1536, "bf16", name="linear_1"),
        # a decode batch through a long down projection, in fp32
        _linear(32, 11008, 4096, "f32", name="linear_32"),
        # a short prompt of odd length, fp16, biased, rows of an odd number of blocks
        _linear(333, 2880, 5760, "f16", bias=True, name="linear_333"),
        # a prefill chunk through a dense projection
        _linear(4096, 4096, 12288, "bf16", name="linear_4096"),
        # a decode batch of 16 sequences: gate_up with its activation, most experts with a row or none
        _grouped("e128", "gate_up", 16, "bf16", name="grouped_decode_16"),
        # an odd batch in fp32: the down projection
        _grouped("e60", "down", 201, "f32", name="grouped_201"),
        # a prefill chunk: gate_up with biases and the clamped gate
        _grouped("e32", "gate_up", 2048, "bf16", name="grouped_prefill_2048"),
        # one decoded token through an expert layer
        _moe("e128", 1, "bf16", name="moe_1"),
        # a small decode batch, fp16, biases and the clamped gate
        _moe("e32", 8, "f16", name="moe_8"),
        # a prefill chunk through an expert layer
        _moe("e128", 2048, "bf16", name="moe_2048"),
    ]


def _size(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    u = rng.random()
    if u < 0.15:
        return _quantise(_size(rng, 1, 8192), 32 * _size(rng, 1, 128), rng.choice(("bf16", "f16", "f32")))
    if u < 0.45:
        K, N = rng.choice(LINEAR)
        if rng.random() < 0.3:
            K, N = 32 * _size(rng, 2, 128), _size(rng, 16, 8192)
        return _linear(_size(rng, 1, 4096), K, N, rng.choice(("bf16", "bf16", "f16", "f32")), rng.random() < 0.3)
    if u < 0.65:
        return _grouped(rng.choice(sorted(LAYERS)), rng.choice(("gate_up", "down")), _size(rng, 1, 2048),
                        rng.choice(("bf16", "f16", "f32")))
    return _moe(rng.choice(sorted(LAYERS)), _size(rng, 1, 2048), rng.choice(("bf16", "f16")))


# ------------------------------------------------------------------ inputs
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def _power(e):
    """2^e in fp32, from its bits (a power function may be an ulp off): -126 <= e <= 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _plain_codes(x):
    """Blocks of 32 along the last dimension: (codes 0..7 of |x|, whether x is negative,
    exponent e): 6 * 2^e is the least such bound of the block's largest |x| (taken as at
    least 1e-12), the code the nearest of _VALUES to |x| / 2^e, ties to the smaller."""
    b = x.float().reshape(*x.shape[:-1], -1, 32)
    m, e = torch.frexp(b.abs().amax(dim=-1).clamp_min(1e-12))  # m * 2^e, 0.5 <= m < 1; 6 = 0.75 * 2^3
    e = torch.where(m <= 0.75, e - 3, e - 2)
    scaled = b.abs() * _power(-e).unsqueeze(-1)
    return torch.bucketize(scaled, torch.tensor(_BORDERS, device=x.device)), b < 0, e


def _pack(x):
    """x as a checkpoint holds it: bytes [..., K/32, 16] of two codes (the low one first)
    and scale bytes [..., K/32]."""
    code, negative, e = _plain_codes(x)
    nibble = (code + 8 * (negative & (code > 0))).to(torch.uint8)
    return nibble[..., 0::2] | (nibble[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _weight(rnd, *shape):
    """N(0, 0.02) weights [..., N, K]."""
    return _pack(rnd(*shape) * 0.02)


def _activations(rnd, rows, K, dtype):
    """Normal values with a few channels ten times as large, as activations have them."""
    x = rnd(rows, K)
    x *= 1 + 9 * (rnd(K) > 2.3)
    return x.to(dtype)


def _routing(rnd, T, k, E):
    """Expert ids and softmax weights of T tokens over E experts of uneven popularity."""
    scores = rnd(T, E) + 0.5 * rnd(E)
    top, ids = scores.topk(k, dim=-1)
    return ids.to(torch.int32), torch.softmax(top, dim=-1)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)

    kind, dt = case["kind"], _DTYPES[case["dtype"]]
    s = dict(case)
    if kind == "quantise":
        s["x"] = _activations(rnd, case["M"], case["K"], dt)
        return s
    if kind == "linear":
        s["w"], s["ws"] = _weight(rnd, case["N"], case["K"])
        s["b"] = (rnd(case["N"]) * 0.1).to(dt) if case["bias"] else None
        s["x"] = _activations(rnd, case["M"], case["K"], dt)
        return s
    T, k, E, H, I = case["T"], case["k"], case["E"], case["H"], case["I"]
    s["ids"], s["topk_w"] = _routing(rnd, T, k, E)
    up, down = kind == "moe" or case["which"] == "gate_up", kind == "moe" or case["which"] == "down"
    s["b1"] = s["b2"] = None
    if up:
        s["w1"], s["s1"] = _weight(rnd, E, 2 * I, H)
        s["b1"] = (rnd(E, 2 * I) * 0.1).to(torch.bfloat16) if case["bias"] else None
    if down:
        s["w2"], s["s2"] = _weight(rnd, E, H, I)
        s["b2"] = (rnd(E, H) * 0.1).to(torch.bfloat16) if case["bias"] else None
    s["x"] = _activations(rnd, T, H, dt) if up else _activations(rnd, T * k, I, dt)
    # the order of this step's pairs by expert, which a program has in hand at a grouped product
    order = torch.sort(s["ids"].reshape(-1).long(), stable=True)
    s["offsets"] = torch.searchsorted(order.values, torch.arange(E + 1, device=DEV)).to(torch.int32)
    s["token_of_row"] = (order.indices // k).to(torch.int32)
    return s


# ------------------------------------------------------------------ the plain form
def _plain_values(x):
    """What the codes of x stand for, in fp32."""
    code, negative, e = _plain_codes(x)
    v = torch.tensor(_VALUES, device=x.device)[code]
    return (torch.where(negative, -v, v) * _power(e).unsqueeze(-1)).reshape(x.shape)


def _plain_unpack(blocks, scales):
    """fp32 values [..., K] of bytes and scale bytes."""
    signed = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=blocks.device)
    v = torch.stack((signed[(blocks & 15).long()], signed[(blocks >> 4).long()]), dim=-1)
    v = v.reshape(*scales.shape, 32) * _power(scales.to(torch.int32) - 127).unsqueeze(-1)
    return v.reshape(*scales.shape[:-1], -1)


def _plain_act(gu, act):
    gate, up = gu.chunk(2, dim=-1)
    if act == "silu":
        return gate / (1 + torch.exp(-gate)) * up
    gate, up = gate.clamp(max=LIMIT), up.clamp(-LIMIT, LIMIT)
    return (up + 1) * gate / (1 + torch.exp(-ALPHA * gate))


def _plain_grouped(rows, offsets, w, ws, b):
    """rows [P, K] sorted by expert -> [P, N]: the rows of the experts that have any, side
    by side in a batch of as many rows as the longest has, times their weights."""
    counts = offsets[1:] - offsets[:-1]
    hit = counts.nonzero()[:, 0]
    P, K = rows.shape
    expert = torch.repeat_interleave(torch.arange(hit.numel(), device=rows.device), counts[hit].long())
    rank = torch.arange(P, device=rows.device) - offsets[hit].long()[expert]
    batch = rows.new_zeros(hit.numel(), int(counts.max()), K)
    batch[expert, rank] = rows
    out = torch.bmm(batch, _plain_unpack(w[hit], ws[hit]).transpose(1, 2).contiguous())
    if b is not None:
        out = out + b[hit].float()[:, None, :]
    return out[expert, rank]


def _plain(s):
    kind, dt = s["kind"], _DTYPES[s["dtype"]]
    x = _plain_values(s["x"])
    if kind == "quantise":
        return x
    if kind == "linear":
        y = x @ _plain_unpack(s["w"], s["ws"]).t()
        return (y + s["b"].float() if s["b"] is not None else y).to(dt)
    token = s["token_of_row"].long()
    if kind == "grouped" and s["which"] == "down":
        return _plain_grouped(x, s["offsets"], s["w2"], s["s2"], s["b2"]).to(dt)
    if kind == "grouped":
        return _plain_act(_plain_grouped(x[token], s["offsets"], s["w1"], s["s1"], s["b1"]), s["act"]).to(dt)
    order = torch.sort(s["ids"].reshape(-1).long(), stable=True)  # a layer sorts for itself
    offsets = torch.searchsorted(order.values, torch.arange(s["E"] + 1, device=x.device))
    h = _plain_act(_plain_grouped(x[order.indices // s["k"]], offsets, s["w1"], s["s1"], s["b1"]), s["act"])
    y = _plain_grouped(_plain_values(h), offsets, s["w2"], s["s2"], s["b2"])
    back = torch.empty_like(y)
    back[order.indices] = y
    return (back.reshape(s["T"], s["k"], -1) * s["topk_w"].unsqueeze(-1)).sum(dim=1).to(dt)


# ------------------------------------------------------------------ the framework's operators
def _own(s):
    kind, dt = s["kind"], _DTYPES[s["dtype"]]
    if kind == "linear":
        from ftmoe.kernel.fused_w4a4_linear import fused_w4a4_linear

        return fused_w4a4_linear(s["x"], s["w"], s["ws"], bias=s["b"])
    if kind == "moe":
        from ftmoe.kernel.fused_w4a4_moe import fused_w4a4_moe

        return fused_w4a4_moe(s["x"], s["w1"], s["s1"], s["w2"], s["s2"], s["ids"], s["topk_w"], activation=s["act"],
                              swiglu_alpha=ALPHA, swiglu_limit=LIMIT, w1_bias=s["b1"], w2_bias=s["b2"])
    from ftmoe.kernel.w4a4_linear import quantize_mxfp4, w4a4_grouped_linear

    blocks, scales = quantize_mxfp4(s["x"])
    if kind == "quantise":
        from ftmoe.kernel.mxfp4_linear import dequantize_mxfp4_blocks

        return dequantize_mxfp4_blocks(blocks, scales, out_dtype=torch.float32)
    if s["which"] == "gate_up":
        return w4a4_grouped_linear(blocks, scales, s["offsets"], s["w1"], s["s1"], row_index=s["token_of_row"],
                                   bias=s["b1"], activation=s["act"], swiglu_alpha=ALPHA, swiglu_limit=LIMIT,
                                   out_dtype=dt)
    return w4a4_grouped_linear(blocks, scales, s["offsets"], s["w2"], s["s2"], bias=s["b2"], out_dtype=dt)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def _codes(n):
    """Bytes of n values in blocks of 32: half a byte each, and their scales."""
    return 17 * n // 32


def work(case):
    kind, b = case["kind"], _SIZE[case["dtype"]]
    if kind == "quantise":  # read, and the values written
        return {"bytes": (b + 4) * case["M"] * case["K"], "flops": 0}
    if kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": b * M * (K + N) + _codes(N * K) + (b * N if case["bias"] else 0), "flops": 2 * M * N * K}
    T, k, E, H, I = case["T"], case["k"], case["E"], case["H"], case["I"]
    P = T * k
    hit = E * (1 - (1 - k / E) ** T)  # experts with a row
    if kind == "grouped":
        up = case["which"] == "gate_up"
        N, K, out, src = (2 * I, H, I, T) if up else (H, I, H, P)
        return {"bytes": int(hit * (_codes(N * K) + (2 * N if case["bias"] else 0)) + b * (src * K + P * out)
                             + (4 * P if up else 0) + 4 * E), "flops": 2 * P * N * K}
    weights = _codes(3 * I * H) + (2 * (2 * I + H) if case["bias"] else 0)
    return {"bytes": int(hit * weights + 2 * b * T * H + 8 * P), "flops": 6 * P * I * H}


# ------------------------------------------------------------------ the definition, in 64 bits
def _two_to(n):
    """2^n in 64 bits for whole n, from a table."""
    table = torch.tensor([math.ldexp(1.0, i) for i in range(-200, 201)], dtype=torch.float64, device=n.device)
    return table[n.long() + 200]


def _exact_values(x):
    """x in 64 bits -> the values of its codes, by the distance to each of them."""
    x = x.double()
    blocks = x.reshape(-1, 32)
    top = blocks.abs().max(dim=1, keepdim=True).values
    top = torch.maximum(top, torch.full_like(top, float(torch.tensor(1e-12, dtype=torch.float32))))
    scale = _two_to(torch.floor(torch.log2(top)) - 4)  # below the one wanted
    for _ in range(4):
        scale = torch.where(top > 6 * scale, 2 * scale, scale)
    size = blocks.abs() / scale
    best, value = torch.full_like(size, math.inf), torch.zeros_like(size)
    for v in _VALUES:  # ascending: of two as near the smaller stays
        d = (size - v).abs()
        value = torch.where(d < best, torch.full_like(value, v), value)
        best = torch.minimum(best, d)
    return (torch.sign(blocks) * value * scale).reshape(x.shape)


def _exact_weight(blocks, scales):
    both = torch.cat(((blocks % 16).unsqueeze(-1), torch.div(blocks, 16, rounding_mode="floor").unsqueeze(-1)), dim=-1)
    both = both.flatten(-2).double()  # nibbles
    size = both % 8
    value = torch.where(size < 4, size / 2, torch.where(size < 6, size - 2, 2 * size - 8))
    value = torch.where(both >= 8, -value, value)
    return (value * _two_to(scales.double() - 127).unsqueeze(-1)).flatten(-2)


def _exact_experts(rows, expert, w, ws, b, E):
    """rows [P, K] in 64 bits, each with its expert -> [P, N]."""
    out = torch.zeros(rows.shape[0], w.shape[1], dtype=torch.float64, device=rows.device)
    for e in range(E):
        mine = (expert == e).nonzero()[:, 0]
        if mine.numel():
            y = rows[mine] @ _exact_weight(w[e], ws[e]).transpose(0, 1)
            out[mine] = y if b is None else y + b[e].double()
    return out


def _exact_act(gu, act):
    I = gu.shape[1] // 2
    gate, up = gu[:, :I], gu[:, I:]
    if act == "silu":
        return gate * torch.sigmoid(gate) * up
    gate = torch.minimum(gate, torch.full_like(gate, LIMIT))
    up = torch.maximum(torch.minimum(up, torch.full_like(up, LIMIT)), torch.full_like(up, -LIMIT))
    return (up + 1) * (gate * torch.sigmoid(ALPHA * gate))


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    x = _exact_values(s["x"])
    if kind == "quantise":
        return x
    if kind == "linear":
        y = x @ _exact_weight(s["w"], s["ws"]).transpose(0, 1)
        return y if s["b"] is None else y + s["b"].double()
    k, E = case["k"], case["E"]
    pairs = s["ids"].reshape(-1).long()  # in order of the tokens
    if kind == "grouped":
        expert = torch.sort(pairs, stable=True).values
        if case["which"] == "down":
            return _exact_experts(x, expert, s["w2"], s["s2"], s["b2"], E)
        gu = _exact_experts(x[s["token_of_row"].long()], expert, s["w1"], s["s1"], s["b1"], E)
        return _exact_act(gu, case["act"])
    token = torch.arange(pairs.numel(), device=x.device) // k
    h = _exact_act(_exact_experts(x[token], pairs, s["w1"], s["s1"], s["b1"], E), case["act"])
    y = _exact_experts(_exact_values(h), pairs, s["w2"], s["s2"], s["b2"], E)
    y = y * s["topk_w"].reshape(-1, 1).double()
    return torch.zeros(case["T"], case["H"], dtype=torch.float64, device=x.device).index_add_(0, token, y)
