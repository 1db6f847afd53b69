"""Refusals of the int8 product and the token sort, on the CPU: the C entry
points check their arguments before they touch the HIP runtime, and the Python
functions take no CPU tensor."""
import ctypes
import weakref

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from ftmoe import _native as nat
from ftmoe.kernel.fused_w8a8_linear import fused_w8a8_expert_forward, fused_w8a8_linear
from ftmoe.kernel.fused_w8a8_moe import fused_w8a8_moe
from ftmoe.kernel.w8a8_linear import quantize_int8_token, w8a8_grouped_linear, w8a8_linear
from ftmoe.moe.token_sort import TokenSort, combine_tokens, gather_tokens, sort_tokens

P = 0x10000  # an aligned address that no refused call reads


def test_quantiser_arguments():
    def call(x=P, dt=nat.DT_BF16, rows=4, K=64, xs=128, q=P, qs=64, s=P):
        return nat.lib().ftm_quant_int8(x, dt, rows, K, xs, q, qs, s, None)

    assert call(dt=7) == nat.ERR_FORMAT
    assert call(rows=-1) == nat.ERR_DIM and call(K=0) == nat.ERR_DIM and call(xs=-2) == nat.ERR_DIM
    assert call(qs=63) == nat.ERR_DIM and call(rows=2**31) == nat.ERR_DIM
    assert call(rows=0, x=None, q=None, s=None) == nat.OK
    assert call(x=None) == nat.ERR_NULL and call(q=None) == nat.ERR_NULL and call(s=None) == nat.ERR_NULL
    assert call(x=P + 1) == nat.ERR_ALIGN and call(xs=129) == nat.ERR_ALIGN and call(s=P + 2) == nat.ERR_ALIGN
    assert call(dt=nat.DT_F32, x=P + 2) == nat.ERR_ALIGN


def _call(**kw):
    c = nat.FtmW8A8(P, P, P, P, None, P, None, None, 4, 4, 64, 0, 32, 64, 1, 0, nat.DT_F32, 0, nat.DT_BF16, -1, 0.0,
                    0.0)
    for k, v in kw.items():
        setattr(c, k, v)
    return nat.lib().ftm_w8a8_linear(ctypes.byref(c), None)


def test_product_arguments():
    assert nat.lib().ftm_w8a8_linear(None, None) == nat.ERR_NULL
    for k in ("x", "x_scale", "w", "w_scale", "out"):
        assert _call(**{k: None}) == nat.ERR_NULL, k
    for kw in (dict(K=0), dict(K=nat.W8A8_MAX_K + 1), dict(N=0), dict(rows=-1), dict(rows=2**31, x_rows=2**31),
               dict(x_stride=-1), dict(x_stride=63), dict(x_rows=3), dict(num_experts=0), dict(num_experts=2),
               dict(offsets=P, num_experts=513), dict(offsets=P, num_experts=2, w_stride=32 * 64 - 1),
               dict(act=nat.ACT_SILU, N=31), dict(w_packed=1, K=62), dict(row_index=P, x_rows=0), dict(w_stride=-1)):
        assert _call(**kw) == nat.ERR_DIM, kw
    for kw in (dict(w_scale_dtype=9), dict(out_dtype=9), dict(bias=P, bias_dtype=9), dict(act=4), dict(act=-2)):
        assert _call(**kw) == nat.ERR_FORMAT, kw
    assert _call(x_scale=P + 2) == nat.ERR_ALIGN
    assert _call(rows=0, x_rows=0, out=None, x=None) == nat.OK


def test_dynamic_product_arguments():
    def call(x=P, dt=nat.DT_BF16, xs=128, **kw):
        c = nat.FtmW8A8(P, P, P, P, None, P, None, None, 4, 4, 64, 0, 32, 64, 1, 0, nat.DT_F32, 0, nat.DT_BF16, -1, 0.0,
                        0.0)
        for k, v in kw.items():
            setattr(c, k, v)
        return nat.lib().ftm_w8a8_linear_dynamic(x, dt, xs, ctypes.byref(c), None)

    assert nat.lib().ftm_w8a8_linear_dynamic(P, 0, 128, None, None) == nat.ERR_NULL
    assert call(x=None) == nat.ERR_NULL and call(w=None) == nat.ERR_NULL and call(x_scale=None) == nat.ERR_NULL
    assert call(dt=7) == nat.ERR_FORMAT
    assert call(xs=-2) == nat.ERR_DIM and call(x_stride=128) == nat.ERR_DIM and call(K=0) == nat.ERR_DIM
    assert call(x=P + 1) == nat.ERR_ALIGN and call(xs=127) == nat.ERR_ALIGN
    assert call(rows=0, x_rows=0, x=None) == nat.OK


def test_moe_arguments():
    L = nat.lib()
    need = L.ftm_w8a8_moe_workspace_bytes(4, 2, 8, 64, 32)
    assert need > 0
    for a in ((0, 2, 8, 64, 32), (4, 0, 8, 64, 32), (4, 2, 513, 64, 32), (4, 2, 8, 0, 32), (4, 2, 8, 64, 0)):
        assert L.ftm_w8a8_moe_workspace_bytes(*a) == 0

    def call(ws=P, n=need, **kw):
        c = nat.FtmW8A8Moe(P, P, P, P, P, P, None, P, P, None, 128, 4, 2, 8, 64, 32, nat.DT_BF16, nat.ID_I32, nat.DT_F32,
                           0, 0, nat.DT_F32, 0, nat.DT_F32, 0, nat.ACT_SILU, 0.0, 0.0)
        for k, v in kw.items():
            setattr(c, k, v)
        return L.ftm_w8a8_moe_forward(ctypes.byref(c), ws, n, None)

    assert L.ftm_w8a8_moe_forward(None, P, need, None) == nat.ERR_NULL
    for k in ("x", "topk_ids", "topk_w", "out", "w13", "w13_scale", "w2", "w2_scale"):
        assert call(**{k: None}) == nat.ERR_NULL, k
    for kw in (dict(T=-1), dict(k=0), dict(num_experts=0), dict(num_experts=513), dict(hidden=0), dict(inter=0),
               dict(hidden=nat.W8A8_MAX_K + 1), dict(x_stride=-2), dict(T=2**30, k=2)):
        assert call(**kw) == nat.ERR_DIM, kw
    for kw in (dict(dtype=9), dict(topk_w_dtype=9), dict(act=-1), dict(act=4), dict(w13_scale_dtype=9),
               dict(w2_scale_dtype=9), dict(ids_dtype=5)):
        assert call(**kw) == nat.ERR_FORMAT, kw
    assert call(ws=None) == nat.ERR_WORKSPACE and call(n=need - 1) == nat.ERR_WORKSPACE
    assert call(ws=P + 16) == nat.ERR_ALIGN and call(x=P + 1) == nat.ERR_ALIGN
    assert call(T=0, x=None) == nat.OK


def test_sort_arguments():
    L = nat.lib()

    def call(ids=P, dt=nat.ID_I32, T=4, k=2, E=8, off=P, a=P, b=P, c=P, ws=None, n=0):
        return L.ftm_sort_tokens(ids, dt, T, k, E, off, a, b, c, ws, n, None)

    assert call(dt=2) == nat.ERR_FORMAT
    for kw in (dict(T=-1), dict(k=0), dict(E=0), dict(E=513), dict(T=2**30, k=2)):
        assert call(**kw) == nat.ERR_DIM, kw
    for k in ("ids", "off", "a", "b", "c"):
        assert call(**{k: None}) == nat.ERR_NULL, k
    need = L.ftm_sort_workspace_bytes(100000, 8, 64)
    assert need > 0 and L.ftm_sort_workspace_bytes(16, 8, 64) == 0
    assert call(T=100000, k=8, E=64) == nat.ERR_WORKSPACE
    assert call(T=100000, k=8, E=64, ws=P, n=need - 1) == nat.ERR_WORKSPACE
    assert call(T=100000, k=8, E=64, ws=P + 1, n=need) == nat.ERR_ALIGN
    assert L.ftm_sort_workspace_bytes(-1, 8, 64) == 0 and L.ftm_sort_workspace_bytes(8, 8, 513) == 0


def test_move_arguments():
    L = nat.lib()

    def gather(x=P, xs=64, eb=2, H=32, r=P, T=4, k=2, out=P):
        return L.ftm_gather_tokens(x, xs, eb, H, r, T, k, out, None)

    assert gather(eb=8) == nat.ERR_FORMAT
    for kw in (dict(T=-1), dict(k=0), dict(H=0), dict(xs=-2), dict(T=2**30, k=2)):
        assert gather(**kw) == nat.ERR_DIM, kw
    for k in ("x", "r", "out"):
        assert gather(**{k: None}) == nat.ERR_NULL, k
    assert gather(x=P + 1) == nat.ERR_ALIGN and gather(xs=65) == nat.ERR_ALIGN
    assert gather(T=0, x=None) == nat.OK

    def combine(rows=P, dt=nat.DT_BF16, rs=64, w=P, wdt=nat.DT_F32, r=P, T=4, k=2, H=32, out=P, odt=nat.DT_BF16):
        return L.ftm_combine_tokens(rows, dt, rs, w, wdt, r, T, k, H, out, odt, None)

    for kw in (dict(dt=5), dict(odt=5), dict(wdt=5), dict(odt=nat.DT_F32), dict(dt=nat.DT_F16)):
        assert combine(**kw) == nat.ERR_FORMAT, kw
    for kw in (dict(T=-1), dict(k=0), dict(H=0), dict(rs=-2)):
        assert combine(**kw) == nat.ERR_DIM, kw
    for k in ("rows", "r", "out"):
        assert combine(**{k: None}) == nat.ERR_NULL, k
    assert combine(rows=P + 1) == nat.ERR_ALIGN
    assert combine(T=0, rows=None) == nat.OK

    def grad(g=P, gdt=nat.DT_BF16, rows=P, dt=nat.DT_BF16, w=P, wdt=nat.DT_F32, r=P, T=4, k=2, H=32, gr=P, gw=P):
        return L.ftm_combine_tokens_grad(g, gdt, 64, rows, dt, 64, w, wdt, r, T, k, H, gr, gw, None)

    for kw in (dict(dt=5), dict(gdt=nat.DT_F32), dict(wdt=5)):
        assert grad(**kw) == nat.ERR_FORMAT, kw
    for k in ("g", "rows", "w", "r"):
        assert grad(**{k: None}) == nat.ERR_NULL, k
    assert grad(gr=None, gw=None, g=None) == nat.OK
    assert grad(T=-1) == nat.ERR_DIM and grad(g=P + 1) == nat.ERR_ALIGN


def test_no_cpu_fallback():
    x = torch.zeros(4, 64)
    w = torch.zeros(32, 64, dtype=torch.int8)
    s = torch.ones(32)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    sort = TokenSort(2, torch.zeros(3, dtype=torch.int32), ids, ids.reshape(-1), ids.reshape(-1))
    q, qs = torch.zeros(4, 64, dtype=torch.int8), torch.ones(4)
    for call in (lambda: quantize_int8_token(x), lambda: w8a8_linear(q, qs, w, s), lambda: fused_w8a8_linear(x, w, s),
                 lambda: w8a8_grouped_linear(q, qs, sort.offsets, w[None].expand(2, -1, -1), s[None].expand(2, -1)),
                 lambda: fused_w8a8_expert_forward(x, w, s, w[:, :16], s, intermediate=16),
                 lambda: fused_w8a8_moe(x, w[None], s[None], w[None], s[None], ids, torch.ones(4, 2)),
                 lambda: sort_tokens(ids, 2), lambda: gather_tokens(x, sort),
                 lambda: combine_tokens(torch.zeros(8, 64), None, sort)):
        with pytest.raises(RuntimeError, match="ROCm device tensor"):
            call()


# ------------------------------------------------------------------ what a call keeps and passes on
def _record_calls(monkeypatch, run):
    """The Python functions on CPU tensors, with ``run(args)`` in the place of the native call."""
    monkeypatch.setattr(nat, "require_gpu", lambda t, name: None)
    monkeypatch.setattr(nat, "launch", lambda what, fn, t, *args: run(args))


@pytest.mark.parametrize("M", [1, 40])
def test_scratch_lives_until_the_native_call_has_returned(monkeypatch, M):
    """The codes' and scales' scratch belongs to a tensor that is still held while the library
    enqueues its kernels: memory given back before could be another thread's by then."""
    made, calls = [], []
    empty = torch.empty

    def remembered(*a, **kw):
        t = empty(*a, **kw)
        made.append(weakref.ref(t))
        return t

    def run(args):
        c = args[-1]._obj
        for at, n in ((c.x, c.x_rows * c.K), (c.x_scale, 4 * c.x_rows)):
            live = [t for t in (r() for r in made) if t is not None]
            assert any(t.data_ptr() <= at and at + n <= t.data_ptr() + t.numel() * t.element_size() for t in live)
        calls.append(c.K)

    _record_calls(monkeypatch, run)
    monkeypatch.setattr(torch, "empty", remembered)
    x, w, s = torch.zeros(M, 64), torch.zeros(32, 64, dtype=torch.int8), torch.ones(32)
    fused_w8a8_linear(x, w, s)
    fused_w8a8_expert_forward(x, w, s, w[:, :16], s, intermediate=16)
    assert calls == [64, 64, 16]


def _token_order(T=4, k=2):
    ids = torch.arange(T * k, dtype=torch.int32).reshape(T, k)
    return TokenSort(2, torch.tensor([0, T * k, T * k], dtype=torch.int32), ids, ids.reshape(-1), ids.reshape(-1) // k)


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_derivatives_are_refused(monkeypatch, grad_mode):
    """A tangent is not dropped without a word (its derivative would be taken for zero): of the
    tokens, of the rows, of the weights; an input without one passes."""
    calls = []
    _record_calls(monkeypatch, calls.append)
    sort, x, rows, w = _token_order(), torch.randn(4, 8), torch.randn(8, 8), torch.rand(4, 2)
    with fwAD.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = [fwAD.make_dual(t, torch.ones_like(t)) for t in (x, rows, w)]
        for call in (lambda: gather_tokens(dual[0], sort), lambda: combine_tokens(dual[1], w, sort),
                     lambda: combine_tokens(rows, dual[2], sort), lambda: combine_tokens(dual[1], None, sort)):
            with pytest.raises(NotImplementedError, match="forward"):
                call()
        assert not calls
        gather_tokens(x, sort), combine_tokens(rows, w, sort), combine_tokens(rows, None, sort)
        assert len(calls) == 3


def test_forward_mode_derivatives_of_gradients_are_refused(monkeypatch):
    """A tangent of the upstream gradient, while the inputs have none."""
    calls = []
    _record_calls(monkeypatch, calls.append)
    sort = _token_order()
    x, rows, w = torch.randn(4, 8).requires_grad_(), torch.randn(8, 8).requires_grad_(), torch.rand(4, 2)
    for out, leaf in ((gather_tokens(x, sort), x), (combine_tokens(rows, w, sort), rows)):
        done = len(calls)
        with fwAD.dual_level():
            g = fwAD.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="forward"):
                torch.autograd.grad(out, leaf, g, retain_graph=True)
        assert len(calls) == done
        torch.autograd.grad(out, leaf, torch.ones_like(out))
        assert len(calls) == done + 1
