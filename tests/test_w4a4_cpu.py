"""Refusals of the MXFP4 x MXFP4 products, on the CPU: the C entry points check
their arguments before they touch the HIP runtime, and the Python functions
take no CPU tensor."""
import ctypes

import pytest
import torch

from ftmoe import _native as nat
from ftmoe.kernel.fused_w4a4_linear import fused_w4a4_expert_forward, fused_w4a4_linear
from ftmoe.kernel.fused_w4a4_moe import fused_w4a4_moe
from ftmoe.kernel.w4a4_linear import mxfp4_of, quantize_mxfp4, w4a4_grouped_linear, w4a4_linear

P = 0x10000  # an aligned address that no refused call reads


def test_quantiser_arguments():
    def call(x=P, dt=nat.DT_BF16, rows=4, K=64, xs=128, b=P, s=P):
        return nat.lib().ftm_quant_mxfp4(x, dt, rows, K, xs, b, s, None)

    assert call(dt=7) == nat.ERR_FORMAT
    for kw in (dict(rows=-1), dict(rows=2**31), dict(K=0), dict(K=48), dict(K=-32), dict(xs=-2)):
        assert call(**kw) == nat.ERR_DIM, kw
    assert call(rows=0, x=None, b=None, s=None) == nat.OK
    assert call(x=None) == nat.ERR_NULL and call(b=None) == nat.ERR_NULL and call(s=None) == nat.ERR_NULL
    assert call(x=P + 1) == nat.ERR_ALIGN and call(xs=129) == nat.ERR_ALIGN and call(b=P + 2) == nat.ERR_ALIGN
    assert call(dt=nat.DT_F32, x=P + 2) == nat.ERR_ALIGN


def _struct(**kw):
    c = nat.FtmW4A4(P, P, P, P, None, P, None, None, 4, 4, 0, 0, 32, 64, 1, 0, nat.DT_BF16, -1, 0.0, 0.0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_DIM = (dict(K=0), dict(K=48), dict(K=nat.W4A4_MAX_K + 32), dict(N=0), dict(rows=-1), dict(rows=2**31, x_rows=2**31),
           dict(x_rows=-1), dict(x_rows=3), dict(num_experts=0), dict(num_experts=2), dict(offsets=P, num_experts=513),
           dict(offsets=P, num_experts=2, w_stride=32 * 32 - 16, w_scale_stride=64),
           dict(offsets=P, num_experts=2, w_stride=32 * 32, w_scale_stride=63), dict(act=nat.ACT_SILU, N=31),
           dict(row_index=P), dict(offsets=P, row_index=P, x_rows=0), dict(w_stride=-1), dict(w_scale_stride=-1))
BAD_FORMAT = (dict(out_dtype=9), dict(bias=P, bias_dtype=9), dict(act=4), dict(act=-2))
BAD_ALIGN = (dict(x=P + 8), dict(w=P + 8), dict(out=P + 1), dict(bias=P + 1, bias_dtype=nat.DT_BF16), dict(offsets=P, row_index=P + 2),
             dict(offsets=P + 2), dict(offsets=P, num_experts=2, w_stride=32 * 32 + 8, w_scale_stride=64))


def test_product_arguments():
    def call(**kw):
        return nat.lib().ftm_w4a4_linear(ctypes.byref(_struct(**kw)), None)

    assert nat.lib().ftm_w4a4_linear(None, None) == nat.ERR_NULL
    for k in ("x", "x_scale", "w", "w_scale", "out"):
        assert call(**{k: None}) == nat.ERR_NULL, k
    for bad, code in ((BAD_DIM, nat.ERR_DIM), (BAD_FORMAT, nat.ERR_FORMAT), (BAD_ALIGN, nat.ERR_ALIGN)):
        for kw in bad:
            assert call(**kw) == code, kw
    assert call(rows=0, x_rows=0, out=None, x=None) == nat.OK


def test_dynamic_product_arguments():
    def call(x=P, dt=nat.DT_BF16, xs=128, **kw):
        return nat.lib().ftm_w4a4_linear_dynamic(x, dt, xs, ctypes.byref(_struct(**kw)), None)

    assert nat.lib().ftm_w4a4_linear_dynamic(P, 0, 128, None, None) == nat.ERR_NULL
    assert call(x=None) == nat.ERR_NULL and call(w=None) == nat.ERR_NULL and call(x_scale=None) == nat.ERR_NULL
    assert call(dt=7) == nat.ERR_FORMAT and call(xs=-2) == nat.ERR_DIM and call(K=0) == nat.ERR_DIM
    assert call(x=P + 1) == nat.ERR_ALIGN and call(xs=127) == nat.ERR_ALIGN
    assert call(rows=0, x_rows=0, x=None) == nat.OK


def test_moe_arguments():
    L = nat.lib()
    need = L.ftm_w4a4_moe_workspace_bytes(4, 2, 8, 64, 32)
    assert need > 0
    for a in ((0, 2, 8, 64, 32), (4, 0, 8, 64, 32), (4, 2, 513, 64, 32), (4, 2, 8, 0, 32), (4, 2, 8, 64, 0)):
        assert L.ftm_w4a4_moe_workspace_bytes(*a) == 0

    def call(ws=P, n=need, **kw):
        c = nat.FtmW4A4Moe(P, P, P, P, P, P, None, P, P, None, 128, 4, 2, 8, 64, 32, nat.DT_BF16, nat.ID_I32, nat.DT_F32,
                           0, 0, nat.ACT_SILU, 0.0, 0.0)
        for k, v in kw.items():
            setattr(c, k, v)
        return L.ftm_w4a4_moe_forward(ctypes.byref(c), ws, n, None)

    assert L.ftm_w4a4_moe_forward(None, P, need, None) == nat.ERR_NULL
    for k in ("x", "topk_ids", "topk_w", "out", "w13", "w13_scale", "w2", "w2_scale"):
        assert call(**{k: None}) == nat.ERR_NULL, k
    for kw in (dict(T=-1), dict(k=0), dict(num_experts=0), dict(num_experts=513), dict(hidden=0), dict(inter=0),
               dict(hidden=48), dict(inter=48), dict(hidden=nat.W4A4_MAX_K + 32), dict(x_stride=-2), dict(T=2**30, k=2)):
        assert call(**kw) == nat.ERR_DIM, kw
    for kw in (dict(dtype=9), dict(topk_w_dtype=9), dict(act=-1), dict(act=4), dict(ids_dtype=5),
               dict(w13_bias=P, w13_bias_dtype=9), dict(w2_bias=P, w2_bias_dtype=9)):
        assert call(**kw) == nat.ERR_FORMAT, kw
    assert call(ws=None) == nat.ERR_WORKSPACE and call(n=need - 1) == nat.ERR_WORKSPACE
    for kw in (dict(ws=P + 16), dict(x=P + 1), dict(x_stride=127), dict(w13=P + 8), dict(w2=P + 8), dict(topk_w=P + 2),
               dict(topk_ids=P + 4, ids_dtype=nat.ID_I64), dict(out=P + 1)):
        assert call(**kw) == nat.ERR_ALIGN, kw
    assert call(T=0, x=None) == nat.OK


@pytest.mark.parametrize("T,k,E,H,I", [(2048, 4, 32, 2880, 2880), (2048, 8, 128, 2048, 768), (512, 2, 16, 1024, 4096)])
def test_moe_workspace_holds_fp32_rows_once(T, k, E, H, I):
    """h is dead when the second product writes its rows, so one buffer holds both: beside it the codes and
    scales of x and h, the tables (three of the pairs, the offsets, the sort's) and borders of 256 bytes."""
    L, P = nat.lib(), T * k
    need = L.ftm_w4a4_moe_workspace_bytes(T, k, E, H, I)
    rest = T * (H // 2 + H // 32) + P * (I // 2 + I // 32) + 12 * P + 4 * (E + 1) + L.ftm_sort_workspace_bytes(T, k, E)
    assert 4 * P * max(H, I) + rest <= need <= 4 * P * max(H, I) + rest + 12 * 256


def test_no_cpu_tensors():
    x = torch.zeros(2, 64)
    b, s = torch.zeros(2, 2, 16, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    b3, s3 = b[None], s[None]
    off, ids = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32)
    for call in (lambda: quantize_mxfp4(x), lambda: w4a4_linear(b, s, b, s),
                 lambda: w4a4_grouped_linear(b, s, off, b3, s3), lambda: fused_w4a4_linear(x, b, s),
                 lambda: fused_w4a4_expert_forward(x, b, s, b, s, intermediate=1),
                 lambda: fused_w4a4_moe(x, b3, s3, b3, s3, ids, torch.ones(2, 1))):
        with pytest.raises(RuntimeError, match="device tensor"):
            call()


def test_operand_checks():
    b, s = torch.zeros(3, 2, 16, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8)
    assert mxfp4_of(b, s, 1, "w")[0].shape == b.shape
    for bad in (b.to(torch.int8), b.float()):
        with pytest.raises(TypeError, match="w_blocks must be uint8"):
            mxfp4_of(bad, s, 1, "w")
    with pytest.raises(TypeError, match="w_scales must be uint8"):
        mxfp4_of(b, s.float(), 1, "w")
    for bb, bs, lead in ((b, s, 2), (b[..., :8], s, 1), (b[:, :0], s[:, :0], 1), (b, s[:2], 1), (b, s[..., None], 1)):
        with pytest.raises(ValueError):
            mxfp4_of(bb, bs, lead, "w")
    # from an odd address on, or with rows apart: copied
    raw = torch.zeros(1 + 96, dtype=torch.uint8)
    assert mxfp4_of(raw[1:].view(3, 2, 16), s, 1, "w")[0].data_ptr() % 16 == 0
    assert mxfp4_of(torch.zeros(3, 4, 16, dtype=torch.uint8)[:, ::2], s, 1, "w")[0].is_contiguous()


@pytest.mark.parametrize("branch", [False, True])
def test_wait_states_of_two_4bit_operands(tmp_path, branch):
    """The build's check knows the shorter wait of a product of two 4-bit operands, and only of that."""
    import importlib.util
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location(
        "mfma_wait_check", os.path.join(root, "freetoken-intel_amd", "csrc", "mfma_wait_check.py"))
    check = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(check)

    def found(states, types):
        body = [f"\tv_mfma_scale_f32_16x16x128_f8f6f4 v[0:3], v[8:11], v[12:15], v[0:3], v20, v21 op_sel_hi:[0,0,0]{types}"]
        if branch:
            body += ["\ts_cbranch_scc1 .LBB0_2", "; %bb.1:", "\ts_endpgm", ".LBB0_2:"]
            states -= 1
        body += ["\ts_nop 0"] * states + ["\tv_add_f32_e32 v30, v1, v31", "\ts_endpgm"]
        path = tmp_path / "k.s"
        path.write_text("\n_Z1kPf:\n" + "\n".join(body) + "\n.Lfunc_end0:\n")
        return len(check.check(str(path)))

    assert found(8, " cbsz:4 blgp:4") == 0 and found(7, " cbsz:4 blgp:4") == 1
    for types in ("", " cbsz:4", " blgp:4"):
        assert found(12, types) == 0 and found(11, types) == 1
