"""The 8-bit integer expert path and the dispatch of tokens to experts, as
measurable cases.

A case is one call, or the few calls that belong together, of public entry
points:

* ``linear``   -- ``fused_w8a8_linear``: tokens quantised to int8 (one scale a
  token), an integer product with an int8 weight (one scale an output channel);
* ``grouped``  -- ``w8a8_grouped_linear``: the same product for rows sorted by
  expert, each expert with its own weight, the rows read through the sort;
* ``dispatch`` -- ``sort_tokens`` + ``gather_tokens`` (with ``grad``: and the
  gradient of the tokens);
* ``combine``  -- ``combine_tokens``: the rows back in token order, weighted and
  summed (with ``grad``: and the gradients of rows and weights);
* ``moe``      -- ``fused_w8a8_moe``: all of it, one expert layer.

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

# Expert layers: those of the benchmark's configurations (16 experts of 512, 128
# of 768, 256 of 512, 32 of 2880), and generic ones beside them.
LAYERS = {
    "e16": dict(E=16, H=1024, I=512, k=2),
    "e128": dict(E=128, H=2048, I=768, k=8),
    "e256": dict(E=256, H=2048, I=512, k=8),
    "e32": dict(E=32, H=2880, I=2880, k=4),
    "e60": dict(E=60, H=2048, I=1408, k=4),
    "e64": dict(E=64, H=2048, I=1024, k=6),
}
# one projection, [K, N]: gate_up and down of those experts, and generic dense ones
LINEAR = ((2048, 1536), (768, 2048), (2048, 1024), (1024, 1024), (1408, 2048), (2880, 5760), (4096, 4096),
          (4096, 12288), (11008, 4096))


def _linear(M, K, N, dtype, bias=False, packed=False, name=None):
    c = dict(kind="linear", M=M, K=K, N=N, dtype=dtype, bias=bias, packed=packed)
    return dict(c, name=name) if name else c


def _grouped(layer, which, T, dtype, packed=False, name=None):
    c = dict(kind="grouped", T=T, which=which, dtype=dtype, packed=packed, **LAYERS[layer])
    return dict(c, name=name) if name else c


def _moved(kind, T, k, E, H, dtype, grad=False, shards=1, name=None):
    c = dict(kind=kind, T=T, k=k, E=E, H=H, dtype=dtype, grad=grad, shards=shards)
    return dict(c, name=name) if name else c


def _moe(layer, T, dtype, packed=False, name=None):
    c = dict(kind="moe", T=T, dtype=dtype, packed=packed, **LAYERS[layer])
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoded token through one expert-sized projection: latency
        _linear(1, 2048, 1536, "bf16", name="linear_1"),
        # a short prompt of odd length, fp16, biased, the checkpoint's packed bytes
        _linear(333, 1408, 2048, "f16", bias=True, packed=True, name="linear_333"),
        # a prefill chunk through a dense projection
        _linear(4096, 4096, 12288, "bf16", name="linear_4096"),
        # a decode batch of 16 sequences: gate_up with its activation, most experts with a row or none
        _grouped("e256", "gate_up", 16, "bf16", name="grouped_decode_16"),
        # a prefill chunk: the down projection
        _grouped("e128", "down", 2048, "bf16", packed=True, name="grouped_prefill_2048"),
        # a decode batch dispatched by itself
        _moved("dispatch", 16, 8, 256, 2048, "bf16", name="dispatch_16"),
        # a prefill chunk on one of two expert shards: half of the pairs have no expert here
        _moved("dispatch", 4096, 8, 256, 2048, "bf16", shards=2, name="dispatch_4096"),
        # training: an odd batch in fp16 dispatched, and the tokens' gradient
        _moved("dispatch", 1001, 4, 32, 2880, "f16", grad=True, name="dispatch_grad_1001"),
        # a decode batch back in token order
        _moved("combine", 64, 8, 128, 2048, "bf16", name="combine_64"),
        # training: a large batch combined, and the gradients of rows and router weights
        _moved("combine", 8192, 8, 128, 2048, "bf16", grad=True, name="combine_grad_8192"),
        # a small model decoding four sequences
        _moe("e16", 4, "bf16", packed=True, name="moe_4"),
        # a prefill chunk through an expert layer
        _moe("e128", 2048, "bf16", name="moe_2048"),
    ]


def _size(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    u = rng.random()
    if u < 0.3:
        K, N = rng.choice(LINEAR)
        if rng.random() < 0.3:
            K, N = 16 * _size(rng, 4, 256), _size(rng, 16, 8192)
        return _linear(_size(rng, 1, 4096), K, N, rng.choice(("bf16", "bf16", "f16", "f32")),
                       rng.random() < 0.3, rng.random() < 0.3)
    if u < 0.5:
        return _grouped(rng.choice(sorted(LAYERS)), rng.choice(("gate_up", "down")), _size(rng, 1, 2048),
                        rng.choice(("bf16", "f16", "f32")), rng.random() < 0.5)
    if u < 0.8:
        E = _size(rng, 4, 512)
        T = _size(rng, 1, 6000)
        return _moved(rng.choice(("dispatch", "combine")), T, rng.randint(1, min(8, E)), E,
                      rng.choice((1024, 2048, 2880, _size(rng, 64, 2560))),
                      rng.choice(("bf16", "bf16", "f16") if T > 3000 else ("bf16", "f16", "f32")),
                      rng.random() < 0.5, rng.choice((1, 1, 2, 4)) if E >= 8 else 1)
    return _moe(rng.choice(sorted(LAYERS)), _size(rng, 1, 2048), rng.choice(("bf16", "f16")), rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def _quantised_weight(rnd, packed, *shape):
    """N(0, 0.02) weights ``[..., N, K]`` as int8 with one fp32 scale a row; ``packed``:
    four offset-binary bytes to an int32 word and ``[..., N, 1]`` scales, as INT8
    checkpoints hold them."""
    w = rnd(*shape) * 0.02
    s = w.abs().amax(dim=-1).clamp_min(1e-12) / 127
    q = (w / s.unsqueeze(-1)).round().clamp(-127, 127)
    if packed:
        return (q + 128).to(torch.uint8).contiguous().view(torch.int32), s.unsqueeze(-1)
    return q.to(torch.int8), s


def _routing(rnd, T, k, E, shards):
    """Expert ids and softmax weights of T tokens over E experts of uneven popularity;
    with ``shards`` the first E / shards experts are here and the others' ids are -1."""
    scores = rnd(T, E) + 0.5 * rnd(E)
    top, ids = scores.topk(k, dim=-1)
    local = E // shards
    ids = torch.where(ids < local, ids, torch.full_like(ids, -1)).to(torch.int32)
    return ids, torch.softmax(top, dim=-1), local


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)

    kind, dt = case["kind"], _DTYPES[case["dtype"]]
    s = dict(case)
    if kind == "linear":
        s["w"], s["ws"] = _quantised_weight(rnd, case["packed"], case["N"], case["K"])
        s["b"] = (rnd(case["N"]) * 0.1).to(dt) if case["bias"] else None
        s["x"] = rnd(case["M"], case["K"]).to(dt)
        return s
    T, k, E, H = case["T"], case["k"], case["E"], case["H"]
    if kind in ("dispatch", "combine"):
        s["ids"], s["topk_w"], s["E"] = _routing(rnd, T, k, E, case["shards"])
        if kind == "dispatch":
            s["x"] = rnd(T, H).to(dt)
            s["g"] = rnd(T * k, H).to(dt) if case["grad"] else None
        else:
            s["y"] = rnd(T * k, H).to(dt)
            s["g"] = rnd(T, H).to(dt) if case["grad"] else None
    else:
        s["ids"], s["topk_w"], s["E"] = _routing(rnd, T, k, E, 1)
        I = case["I"]
        if kind == "moe" or case["which"] == "gate_up":
            s["w1"], s["s1"] = _quantised_weight(rnd, case["packed"], E, 2 * I, H)
        if kind == "moe" or case["which"] == "down":
            s["w2"], s["s2"] = _quantised_weight(rnd, case["packed"], E, H, I)
        if kind == "moe":
            s["x"] = rnd(T, H).to(dt)
        elif case["which"] == "gate_up":  # the tokens, read through the sort
            s["xq"], s["xs"] = _plain_quantise(rnd(T, H).to(torch.bfloat16))
        else:  # one row for each pair
            s["xq"], s["xs"] = _plain_quantise(rnd(T * k, I).to(torch.bfloat16))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("combine", "grouped"):  # the sort of this step is in hand
        if own:
            from ftmoe.moe.token_sort import sort_tokens

            s["sort"] = sort_tokens(s["ids"], s["E"])
        else:
            s["sort"] = _plain_sort(s["ids"], s["E"])
    return s


# ------------------------------------------------------------------ the plain form
def _plain_quantise(x):
    """One fp32 scale a row, max |x| / 127; the codes are the whole numbers nearest x / scale."""
    s = x.float().abs().amax(dim=-1).clamp_min(1e-12) / 127
    q = (x.double() / s.double().unsqueeze(-1)).round().clamp(-127, 127)
    return q.to(torch.int8), s


def _plain_codes(w):
    return (w.view(torch.uint8).to(torch.int16) - 128).float() if w.dtype == torch.int32 else w.float()


def _plain_sort(ids, E):
    """Pairs in order of their expert, of their number within an expert; those without
    an expert behind them all, their row and pair numbers as complements."""
    T, k = ids.shape
    flat = ids.reshape(-1).long()
    here = (flat >= 0) & (flat < E)
    key = torch.where(here, flat, torch.full_like(flat, E))
    hot = torch.zeros(key.numel(), E + 1, dtype=torch.int32, device=key.device)
    hot[torch.arange(key.numel(), device=key.device), key] = 1
    rank = hot.cumsum(0, dtype=torch.int32).gather(1, key[:, None])[:, 0].long() - 1
    counts = hot.sum(0)
    offsets = torch.zeros(E + 2, dtype=torch.int64, device=key.device)
    offsets[1:] = counts.cumsum(0)
    row = offsets[key] + rank
    pair = torch.empty_like(row)
    pair[row] = torch.arange(key.numel(), device=key.device)
    used = torch.arange(key.numel(), device=key.device) < offsets[E]
    return dict(offsets=offsets[:E + 1].int(), row_of_pair=torch.where(here, row, ~row).reshape(T, k).int(),
                pair_of_row=torch.where(used, pair, ~pair).int(),
                token_of_row=torch.where(used, pair // k, torch.full_like(pair, -1)).int())


def _plain_gather(x, sort, k):
    out = torch.zeros(sort["pair_of_row"].numel(), x.shape[1], dtype=x.dtype, device=x.device)
    n = sort["token_of_row"].long()
    out[n >= 0] = x[n[n >= 0]]
    return out


def _plain_back(rows, sort, w=None):
    """Rows back in token order, weighted and summed, in fp32."""
    row = sort["row_of_pair"].long()
    here = row >= 0
    v = rows[row.clamp_min(0)].float()
    v = torch.where(here[..., None], v, torch.zeros_like(v))
    if w is not None:
        v = v * w.float()[..., None]
    return v.sum(dim=1)


def _plain_act(gu):
    I = gu.shape[1] // 2
    gate, up = gu[:, :I], gu[:, I:]
    return gate / (1 + torch.exp(-gate)) * up


def _plain_grouped(xq, xs, sort, w, ws, index, act):
    P, N = sort["pair_of_row"].numel(), w.shape[1]
    out = torch.zeros(P, N // 2 if act else N, dtype=torch.float32, device=xq.device)
    ends = sort["offsets"].tolist()
    for e in range(len(ends) - 1):
        lo, hi = ends[e], ends[e + 1]
        if hi == lo:
            continue
        src = sort["token_of_row"][lo:hi].long() if index else slice(lo, hi)
        v = (xq[src].float() @ _plain_codes(w[e]).t()) * xs[src][:, None] * ws[e].reshape(1, -1).float()
        out[lo:hi] = _plain_act(v) if act else v
    return out


def _plain(s):
    kind, dt = s["kind"], _DTYPES[s["dtype"]]
    if kind == "linear":
        q, xs = _plain_quantise(s["x"])
        y = (q.float() @ _plain_codes(s["w"]).t()) * xs[:, None] * s["ws"].reshape(1, -1).float()
        return (y + s["b"].float() if s["b"] is not None else y).to(dt)
    if kind == "dispatch":
        sort = _plain_sort(s["ids"], s["E"])
        out = [sort["offsets"], sort["row_of_pair"], sort["pair_of_row"], sort["token_of_row"],
               _plain_gather(s["x"], sort, s["k"])]
        return out + [_plain_back(s["g"], sort).to(dt)] if s["grad"] else out
    if kind == "combine":
        sort, w = s["sort"], s["topk_w"]
        out = _plain_back(s["y"], sort, w).to(dt)
        if not s["grad"]:
            return out
        row = sort["row_of_pair"].long()
        here, gf = row >= 0, s["g"].float()
        gy = torch.zeros(s["y"].shape, dtype=dt, device=row.device)
        gy[row[here]] = (gf[:, None, :] * w[..., None])[here].to(dt)
        gw = (s["y"][row.clamp_min(0)].float() * gf[:, None, :]).sum(dim=2)
        return [out, gy, torch.where(here, gw, torch.zeros_like(gw))]
    if kind == "grouped":
        up = s["which"] == "gate_up"
        w, ws = (s["w1"], s["s1"]) if up else (s["w2"], s["s2"])
        return _plain_grouped(s["xq"], s["xs"], s["sort"], w, ws, up, up).to(dt)
    sort = _plain_sort(s["ids"], s["E"])
    xq, xs = _plain_quantise(s["x"])
    hq, hs = _plain_quantise(_plain_grouped(xq, xs, sort, s["w1"], s["s1"], True, True))
    y = _plain_grouped(hq, hs, sort, s["w2"], s["s2"], False, False)
    return _plain_back(y, sort, s["topk_w"]).to(dt)


# ------------------------------------------------------------------ the framework's operators
def _own(s):
    kind = s["kind"]
    if kind == "linear":
        from ftmoe.kernel.fused_w8a8_linear import fused_w8a8_linear

        return fused_w8a8_linear(s["x"], s["w"], s["ws"], bias=s["b"])
    if kind == "grouped":
        from ftmoe.kernel.w8a8_linear import w8a8_grouped_linear

        sort, dt = s["sort"], _DTYPES[s["dtype"]]
        if s["which"] == "gate_up":
            return w8a8_grouped_linear(s["xq"], s["xs"], sort.offsets, s["w1"], s["s1"], row_index=sort.token_of_row,
                                       activation="silu", out_dtype=dt)
        return w8a8_grouped_linear(s["xq"], s["xs"], sort.offsets, s["w2"], s["s2"], out_dtype=dt)
    if kind == "moe":
        from ftmoe.kernel.fused_w8a8_moe import fused_w8a8_moe

        return fused_w8a8_moe(s["x"], s["w1"], s["s1"], s["w2"], s["s2"], s["ids"], s["topk_w"], activation="silu")
    from ftmoe.moe.token_sort import combine_tokens, gather_tokens, sort_tokens

    if kind == "dispatch":
        sort = sort_tokens(s["ids"], s["E"])
        x = s["x"].detach().requires_grad_(s["grad"])
        rows = gather_tokens(x, sort)
        out = [sort.offsets, sort.row_of_pair, sort.pair_of_row, sort.token_of_row, rows.detach()]
        return out + list(torch.autograd.grad(rows, x, s["g"])) if s["grad"] else out
    if not s["grad"]:
        return combine_tokens(s["y"], s["topk_w"], s["sort"])
    y, w = s["y"].detach().requires_grad_(), s["topk_w"].detach().requires_grad_()
    out = combine_tokens(y, w, s["sort"])
    return [out.detach(), *torch.autograd.grad(out, (y, w), s["g"])]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, b = case["kind"], _SIZE[case["dtype"]]
    if kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": b * M * (K + N) + N * K + 4 * N + (b * N if case["bias"] else 0), "flops": 2 * M * N * K}
    T, k, E, H = case["T"], case["k"], case["E"], case["H"]
    P = T * k
    if kind in ("dispatch", "combine"):
        here = P / case["shards"]
        # tokens that have a row here, read (or written) once
        tok = T * (1 - (1 - 1 / case["shards"]) ** k)
        if kind == "dispatch":
            bytes_ = 4 * P + 12 * P + 4 * E + b * H * (tok + P)
            if case["grad"]:
                bytes_ += b * H * (here + T)
            return {"bytes": int(bytes_), "flops": int(H * here) if case["grad"] else 0}
        bytes_ = 8 * P + b * H * (here + T)
        if case["grad"]:  # the rows serve both directions
            bytes_ += b * H * (tok + P) + 4 * P
        return {"bytes": int(bytes_), "flops": int((6 if case["grad"] else 2) * H * here)}
    I = case["I"]
    hit = E * (1 - (1 - k / E) ** T)  # experts with a row
    if kind == "grouped":
        up = case["which"] == "gate_up"
        N, K, out, src = (2 * I, H, I, T) if up else (H, I, H, P)
        return {"bytes": int(hit * N * (K + 4) + src * (K + 4) + b * P * out + (4 * P if up else 0) + 4 * E),
                "flops": 2 * P * N * K}
    return {"bytes": int(hit * (3 * I * H + 4 * (2 * I + H)) + 2 * b * T * H + 8 * P), "flops": 6 * P * I * H}


# ------------------------------------------------------------------ the definition, in 64 bits
def _exact_quantise(x):
    """The scale is stored as fp32; a code is the whole number nearest x / scale."""
    x = x.double()
    s = torch.maximum(x.abs().amax(dim=1), torch.tensor(1e-12, dtype=torch.float32).double().to(x.device))
    s = (s.float() / 127.0).double()
    return torch.clamp(torch.round(x / s[:, None]), -127, 127), s


def _exact_weight(w, s):
    if w.dtype == torch.int32:
        w = torch.stack([((w >> (8 * i)) & 255) - 128 for i in range(4)], dim=-1).flatten(-2)
    return w.double() * s.reshape(-1, 1).double()


def _exact_order(ids, E):
    """Stable order of the pairs by expert, those without one last: (order, offsets)."""
    key = ids.reshape(-1).cpu().long()
    key = torch.where((key < 0) | (key >= E), E, key)
    order = torch.sort(key, stable=True).indices
    offsets = torch.searchsorted(key[order].contiguous(), torch.arange(E + 1))
    return order, offsets


def _exact_experts(rows, order, offsets, k, weight, act, through):
    """rows [., K] in 64 bits -> one output row for each sorted pair."""
    out = None
    for e in range(offsets.numel() - 1):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        if lo == hi:
            continue
        src = rows[(order[lo:hi] // k).to(rows.device)] if through else rows[lo:hi]
        y = src @ weight(e).transpose(0, 1)
        if act:
            gate, up = y.chunk(2, dim=1)
            y = gate * torch.sigmoid(gate) * up
        if out is None:
            out = torch.zeros(order.numel(), y.shape[1], dtype=torch.float64, device=y.device)
        out[lo:hi] = y
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "linear":
        q, xs = _exact_quantise(s["x"])
        y = (q * xs[:, None]) @ _exact_weight(s["w"], s["ws"]).transpose(0, 1)
        return y if s["b"] is None else y + s["b"].double()
    k, E = case["k"], s["E"]
    order, offsets = _exact_order(s["ids"], E)
    P, n = order.numel(), int(offsets[E])
    if kind in ("grouped", "moe"):
        if kind == "moe":
            q, xs = _exact_quantise(s["x"])
        else:
            q, xs = s["xq"].double(), s["xs"].double()
        v = q * xs[:, None]
        if kind == "grouped":
            up = case["which"] == "gate_up"
            w, ws = (s["w1"], s["s1"]) if up else (s["w2"], s["s2"])
            return _exact_experts(v, order, offsets, k, lambda e: _exact_weight(w[e], ws[e]), up, up)
        h = _exact_experts(v, order, offsets, k, lambda e: _exact_weight(s["w1"][e], s["s1"][e]), True, True)
        hq, hs = _exact_quantise(h)
        y = _exact_experts(hq * hs[:, None], order, offsets, k, lambda e: _exact_weight(s["w2"][e], s["s2"][e]),
                           False, False)
        y = y * s["topk_w"].reshape(-1)[order.to(y.device)].double()[:, None]
        out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device=y.device)
        return out.index_add_(0, (order // k).to(y.device), y)
    pairs = order[:n].to(DEV)  # the pairs with an expert here, in row order
    tokens = pairs // k
    if kind == "dispatch":
        row = torch.empty(P, dtype=torch.int64)
        row[order] = torch.where(torch.arange(P) < n, torch.arange(P), -1 - torch.arange(P))
        pair = torch.where(torch.arange(P) < n, order, -1 - order)
        token = torch.where(torch.arange(P) < n, order // k, -1)
        rows = torch.zeros(P, case["H"], dtype=torch.float64, device=DEV)
        rows[:n] = s["x"].double()[tokens]
        out = [offsets.int(), row.reshape(case["T"], k).int(), pair.int(), token.int(), rows]
        if case["grad"]:
            gx = torch.zeros(case["T"], case["H"], dtype=torch.float64, device=DEV)
            out.append(gx.index_add_(0, tokens, s["g"][:n].double()))
        return [o.to(DEV) for o in out]
    wt = s["topk_w"].reshape(-1)[pairs].double()
    y = s["y"][:n].double()
    out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device=DEV).index_add_(0, tokens, y * wt[:, None])
    if not case["grad"]:
        return out
    g = s["g"].double()[tokens]
    gy = torch.zeros(P, case["H"], dtype=torch.float64, device=DEV)
    gy[:n] = g * wt[:, None]
    gw = torch.zeros(P, dtype=torch.float64, device=DEV)
    gw[pairs] = (g * y).sum(dim=1)
    return [out, gy, gw.reshape(case["T"], k)]
