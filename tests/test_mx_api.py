"""The MX operators without a GPU: what they refuse, the shapes they propagate, the plain forms the GPU tests rely on."""
import numpy as np
import pytest
import torch

import mx_plain as P
from mor_amd import _cabi, mx, wire

L = _cabi.lib()
A = 4096          # stands for device addresses that are never read: every refusal comes before a device call


def refused(rc, text):
    assert rc == -1 and text in L.mor_last_error().decode(), (rc, L.mor_last_error())


def test_product_refuses():
    ok = dict(pa=A, sa=A, fa=0, pb=A, sb=A, fb=4, out=A, m=8, n=8, k=64, ws=None, wb=0)

    def call(**kw):
        v = {**ok, **kw}
        return L.mor_mx_matmul(v["pa"], v["sa"], v["fa"], v["pb"], v["sb"], v["fb"], v["out"], v["m"], v["n"], v["k"], v["ws"], v["wb"], None)

    for p in ("pa", "sa", "pb", "sb", "out"):
        refused(call(**{p: None}), "NULL")
    for f in (2, 3, 5, -1):
        refused(call(fa=f), "formats")
        refused(call(fb=f), "formats")
    for kw in (dict(k=0), dict(k=48), dict(k=-32), dict(k=1 << 23), dict(m=0), dict(m=-1), dict(n=0), dict(m=1 << 30), dict(n=1 << 30), dict(m=1 << 31), dict(m=1 << 29, n=1 << 29)):
        refused(call(**kw), "products need")
    refused(call(pa=A + 8), "16-byte")
    refused(call(pb=A + 4), "16-byte")
    refused(call(out=A + 1), "2-byte")
    need = L.mor_mx_matmul_workspace_bytes(128, 128, 14336, 0, 0)
    assert need > 0 and need % (128 * 128 * 4) == 0
    for kw in (dict(), dict(ws=A, wb=need - 1), dict(ws=A + 4, wb=need)):
        assert call(m=128, n=128, k=14336, fb=0, **kw) == -2 and b"workspace" in L.mor_last_error()


def test_product_workspace():
    assert L.mor_mx_matmul_workspace_bytes(1, 4096, 4096, 0, 0) == 0
    assert L.mor_mx_matmul_workspace_bytes(8, 8, 33, 0, 0) == 0 and L.mor_mx_matmul_workspace_bytes(8, 8, 64, 2, 0) == 0


def test_quantisers_refuse():
    refused(L.mor_mx_quantize(A, A, A, 4, 48, 4, None), "cols")
    refused(L.mor_mx_quantize(A, A, A, 4, 64, 5, None), "format")
    refused(L.mor_mx_quantize_dual(A, A, A, A, A, 33, 64, 4, None), "rows")
    refused(L.mor_mx_quantize_dual_ragged(A, A, A, A, A, 33, 48, 4, 4, None), "cols")
    refused(L.mor_mx_quantize_dual_ragged(A, A, A, A, A, 0, 64, 4, 4, None), "positive")
    for pair in ((0, 4), (4, 1), (2, 2), (0, 1)):
        refused(L.mor_mx_quantize_dual_ragged(A, A, A, A, A, 33, 64, *pair, None), "formats")
    refused(L.mor_mx_quantize_dual_ragged(A, A, A, A, A, 1 << 30, 32, 4, 4, None), "too many tiles")
    refused(L.mor_mx_quantize_dual(A, A, A, A, A, 1 << 30, 32, 4, None), "too many tiles")
    refused(L.mor_mx_quantize_dual_ragged(A, A + 8, A, A, A, 33, 64, 4, 4, None), "aligned")
    refused(L.mor_selftest_hw_fp4(None, None), "NULL")
    assert L.mor_mx_payload_bytes(64, 128, 4) == 64 * 64


def test_swiglu_refuses():
    def call(g=A, gs=32, u=A, us=32, out=A, gc=A, gsc=A, uc=A, usc=A, rows=2, cols=32):
        return L.mor_swiglu_mx(g, gs, u, us, out, gc, gsc, uc, usc, rows, cols, None)

    for kw in (dict(g=None), dict(u=None), dict(out=None)):
        refused(call(**kw), "NULL")
    for kw in (dict(gc=None), dict(gsc=None), dict(uc=None), dict(usc=None)):
        refused(call(**kw), "all four")
    refused(call(rows=0), "positive")
    refused(call(cols=0), "positive")
    refused(call(gs=31), "strides")
    refused(call(us=0), "strides")
    refused(call(g=A + 1), "2-byte")
    refused(call(gc=A + 4), "8-byte")
    refused(call(rows=(1 << 30) - 63, cols=32), "too large")
    refused(call(rows=1 << 29, cols=96, gs=96, us=96), "too large")
    refused(call(rows=1 << 62, cols=1 << 40, gs=1 << 40, us=1 << 40), "too large")

    def back(d=A, gc=A, gsc=A, uc=A, usc=A, dg=A, du=A, rows=2, cols=32):
        return L.mor_swiglu_mx_backward(d, gc, gsc, uc, usc, dg, du, rows, cols, None)

    for name in ("d", "gc", "gsc", "uc", "usc", "dg", "du"):
        refused(back(**{name: None}), "NULL")
    refused(back(rows=-1), "positive")
    refused(back(d=A + 1), "2-byte")
    refused(back(uc=A + 2), "8-byte")


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.bfloat16, requires_grad=True)
    u8 = torch.zeros(4, 64, dtype=torch.uint8)
    for call in (lambda: mx.linear(x, w), lambda: mx.swiglu(x, x), lambda: wire.matmul_mx(u8, u8[:, :2], u8, u8[:, :2]),
                 lambda: wire.quantize_mx(x, wire.E2M1)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_python_refusals():
    with pytest.raises(RuntimeError, match="two dimensions"):
        mx.linear(torch.zeros(64), torch.zeros(32, 64))
    with pytest.raises(RuntimeError, match="one shape"):
        mx.swiglu(torch.zeros(2, 3), torch.zeros(3, 2))
    with pytest.raises(RuntimeError, match="one dimension"):
        mx.swiglu(torch.zeros(()), torch.zeros(()))


def test_fake_shapes():
    op = torch.ops.mor
    p, s = op.mx_quantize(meta(5, 96), wire.E2M1)
    assert p.shape == (5, 48) and s.shape == (5, 3) and p.dtype == s.dtype == torch.uint8
    assert op.mx_quantize(meta(5, 96), wire.E2M3)[0].shape == (5, 72)
    got = op.mx_quantize_dual(meta(33, 96), wire.E2M1, wire.E4M3)
    assert [tuple(t.shape) for t in got] == [(33, 48), (33, 3), (96, 64), (96, 2)]
    assert op.mx_dequantize(p, s, wire.E2M1).shape == (5, 96)
    out = op.mx_matmul(p, s, meta(7, 48, dtype=torch.uint8), meta(7, 3, dtype=torch.uint8), 4, 4)
    assert out.shape == (5, 7) and out.dtype == torch.bfloat16
    h, kept = op.swiglu_mx_forward(meta(3, 33), meta(3, 33), True)
    assert h.shape == (3, 33) and kept.shape == (2 * (256 + 6),) and kept.dtype == torch.uint8
    assert [tuple(t.shape) for t in op.swiglu_mx_backward(h, kept)] == [(3, 33), (3, 33)]
    y, kept = op.mx_linear_forward(meta(70, 64), meta(96, 64), wire.E2M1, True, True)
    assert y.shape == (70, 96) and kept.shape == (64 * 96 + 256 + 64 * 48 + 256,)
    assert [tuple(t.shape) for t in op.mx_linear_backward(y, kept, 64, wire.E2M1, wire.E4M3, True, True)] == [(70, 64), (96, 64)]


def test_tracing_through_the_training_operators():
    """Fake tensors go through the forward operators and their autograd nodes."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 35, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        w = torch.empty(96, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        y = mx.linear(x, w, wire.E2M1)
        h = mx.swiglu(y, y)
        assert y.shape == h.shape == (2, 35, 96) and h.requires_grad
        assert mx.linear(x.detach(), w.detach()).shape == (2, 35, 96)


def test_plain_forms():
    """The table of every format is the one torch casts to, and a round trip through packed codes is exact."""
    for fmt, dtype in ((P.E4M3, torch.float8_e4m3fn), (P.E5M2, torch.float8_e5m2)):
        codes = torch.arange(len(P.table(fmt)), dtype=torch.uint8)
        assert np.array_equal(codes.view(dtype).double().numpy(), P.table(fmt))
    assert P.table(P.E2M1).tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    x = P.to64(P.bf16(np.random.default_rng(1).standard_normal((8, 64))))
    for fmt, mode in ((P.E4M3, torch.float8_e4m3fn), (P.E5M2, torch.float8_e5m2)):
        codes, scales = P.quantize(x, fmt)
        scaled = torch.from_numpy(x.reshape(8, 2, 32) * np.exp2(127.0 - scales)[..., None]).float()
        assert np.array_equal(scaled.to(mode).view(torch.uint8).numpy().reshape(8, 64), codes)
        assert np.array_equal(P.quantized_values(P.quantized_values(x, fmt), fmt), P.quantized_values(x, fmt))
