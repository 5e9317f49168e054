"""Training operators without a GPU: what the C entry points and their Python callers refuse before any launch."""
import ctypes as C
import importlib.util
from types import SimpleNamespace

import pytest
import torch

from esm_amd import _lib as L
from esm_amd import training as T

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -4
BUF = (C.c_char * 4096)()
P = (C.addressof(BUF) + 63) // 64 * 64  # an aligned address; every call below is refused before it would be used


def refused(rc, code, text):
    assert rc == code
    assert text in L.lib().esmk_last_error().decode()


def test_layernorm_entry_points_refuse():
    lib = L.lib()
    fwd = lambda x=P, dt=L.F32, ld=64, g=P, y=P, st=P, M=4, d=64: lib.esmk_layernorm_fwd(x, dt, ld, g, None, y, st, M, d, 1e-5, None)
    refused(fwd(d=0), UNSUPPORTED, "d=0")
    refused(fwd(d=12289, ld=12289), UNSUPPORTED, "12289")
    refused(fwd(M=-1), UNSUPPORTED, "M=-1")
    refused(fwd(M=2 ** 31 - 1, d=1), UNSUPPORTED, "M=2147483647")  # a row number plus the grid's rows would pass 31 bits
    refused(fwd(dt=2), INVALID, "dtype")
    refused(fwd(ld=63), INVALID, "row stride")
    refused(fwd(st=P + 4), INVALID, "stats")
    for k in ("x", "g", "y", "st"):
        refused(fwd(**{k: None}), INVALID, "null")
    assert fwd(M=0, x=None, y=None) == 0
    bwd = lambda dy=P, ldg=64, x=P, ldx=64, dt=L.BF16, ws=P, nb=1 << 30, M=4096, d=64, dw=P: lib.esmk_layernorm_bwd(
        dy, ldg, x, ldx, dt, P, P, P, dw, P, ws, nb, M, d, None)
    refused(bwd(dy=None), INVALID, "null")
    refused(bwd(ldg=1), INVALID, "row stride")
    refused(bwd(dt=7), INVALID, "dtype")
    refused(bwd(M=2 ** 30 + 1), UNSUPPORTED, "M=1073741825")
    refused(bwd(ws=None), WORKSPACE, "workspace")
    refused(bwd(nb=lib.esmk_layernorm_bwd_workspace_bytes(4096, 64) - 1), WORKSPACE, "workspace")
    refused(lib.esmk_layernorm_bwd(P, 64, P, 64, L.BF16, P, P, None, None, None, P, 1 << 30, 4096, 64, None), INVALID, "no gradient")
    assert lib.esmk_layernorm_bwd_workspace_bytes(512, 12288) == 0 and lib.esmk_layernorm_bwd_workspace_bytes(513, 64) > 0
    assert lib.esmk_layernorm_bwd_workspace_bytes(0, 64) == 0 and lib.esmk_layernorm_bwd_workspace_bytes(4096, 64) > 0


def test_attention_entry_points_refuse():
    lib = L.lib()

    def fwd(q=P, st=(128, 64) * 4, cu=P, n=1, N=4, H=2, G=2, D=64, scale=0.125):
        return lib.esmk_attn_varlen_fwd(q, P, P, P, P, (C.c_int64 * 8)(*st), cu, n, None, N, H, G, D, scale, None)
    refused(fwd(D=32), UNSUPPORTED, "head dim 32")
    refused(fwd(G=3), INVALID, "kv heads=3")
    refused(fwd(H=0), INVALID, "heads=0")
    refused(fwd(N=-1), INVALID, "n_tokens=-1")
    refused(fwd(n=-1), INVALID, "n_segments=-1")
    for s in (0.0, -1.0, 1e-31, float("nan"), float("inf")):
        refused(fwd(scale=s), INVALID, "scale")
    refused(fwd(cu=None), INVALID, "null")
    refused(fwd(q=None), INVALID, "null")
    refused(fwd(q=P + 8), INVALID, "tensor 0")
    refused(fwd(st=(128, 64, 124, 64, 128, 64, 128, 64)), INVALID, "tensor 1")
    refused(fwd(st=(128, 64, 128, 64, 128, 60, 128, 64)), INVALID, "tensor 2")
    refused(fwd(st=(128, 64, 128, 64, 128, 64, 56, 64)), INVALID, "tensor 3")
    refused(fwd(st=(1 << 23, 64, 128, 64, 128, 64, 128, 64)), INVALID, "tensor 0")
    refused(fwd(N=2 ** 30, H=1, G=1), UNSUPPORTED, "grid")
    refused(fwd(N=2 ** 20, H=1024, G=1024), UNSUPPORTED, "grid")
    refused(fwd(N=2 ** 30 + 1), INVALID, "n_tokens")
    assert fwd(N=0, q=None) == 0

    def bwd(st=(128, 64) * 8, ws=P, nb=1 << 20, dq=P):
        return lib.esmk_attn_varlen_bwd(P, P, P, P, P, P, dq, P, P, (C.c_int64 * 16)(*st), P, 1, None, 4, 2, 2, 64, 0.125, ws, nb, None)
    refused(bwd(dq=None), INVALID, "null")
    refused(bwd(st=(128, 64) * 7 + (4, 64)), INVALID, "tensor 7")
    refused(bwd(ws=None), WORKSPACE, "32 workspace")
    refused(bwd(nb=31), WORKSPACE, "32 workspace")
    for dk, dv in ((None, P), (P, None)):
        refused(lib.esmk_attn_varlen_bwd(P, P, P, P, P, P, P, dk, dv, (C.c_int64 * 16)(*(128, 64) * 8), P, 1, None, 4, 2, 2, 64, 0.125, P, 1 << 20,
                                         None), INVALID, "together")


def test_preference_entry_points_refuse():
    lib = L.lib()

    def fwd(z=P, dt=L.F32, y=P, cu=P, n=1, e=0.0, N=4, V=8, saved=P, nb=1 << 20):
        return lib.esmk_pref_loss_fwd(z, dt, y, cu, n, P, 0.1, e, 0.0, N, V, saved, nb, P, P, None)
    refused(fwd(dt=5), INVALID, "dtype")
    refused(fwd(V=0), INVALID, "V=0")
    refused(fwd(N=-1), INVALID, "N=-1")
    refused(fwd(N=1 << 26), UNSUPPORTED, "2^26")
    refused(fwd(n=0), INVALID, "n_pairs=0")
    refused(fwd(n=1 << 23, nb=1 << 40), INVALID, "n_pairs=8388608")  # 512 threads a pair: 2^32
    refused(fwd(z=None), INVALID, "null")
    refused(fwd(cu=None), INVALID, "null")
    refused(fwd(z=P + 4), INVALID, "16-byte")
    refused(fwd(saved=P + 8), INVALID, "16-byte")
    for e in (-0.1, 1.1, float("nan")):
        refused(fwd(e=e), INVALID, "label_smoothing")
    refused(fwd(nb=4 * 16 + 16 - 1), WORKSPACE, "80 bytes")
    bwd = lambda z=P, dz=P, N=4: lib.esmk_pref_loss_bwd(z, L.F32, P, P, None, dz, N, 8, None)
    refused(bwd(dz=None), INVALID, "dlogits")
    refused(bwd(dz=P + 4), INVALID, "dlogits")
    refused(bwd(z=None), INVALID, "null")
    assert bwd(N=0, z=None, dz=None) == 0


def test_host_tensors_are_refused():
    x, w = torch.zeros(2, 8), torch.ones(8)
    q, cu = torch.zeros(4, 1, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(L.EsmkError, match="GPU only"):
        T.layer_norm(x, w)
    with pytest.raises(L.EsmkError, match="GPU only"):
        T.attention_varlen(q, q, q, cu)
    with pytest.raises(L.EsmkError, match="GPU only"):
        T.preference_loss(x, torch.zeros(2, dtype=torch.int64), cu, w)
    with pytest.raises(TypeError):
        T.layer_norm(x.half(), w)
    with pytest.raises(TypeError):
        T.attention_varlen("q", q, q, cu)


def test_rows_of_wider_tensors_are_read_in_place():
    """`_rows` copies only where the rows do not lie at one distance."""
    at = lambda t: (t.data_ptr(), t.shape)
    wide = torch.zeros(2, 5, 3, 4 * 8)
    qkv = torch.zeros(3, 7, 3 * 16)
    for t, ld in ((qkv[..., :16], 48), (qkv[..., 16:32], 48), (qkv[:, :1, :16], 7 * 48), (qkv[1:2, :, 32:], 48), (qkv[0, :, 5:21], 48),
                  (qkv[::2, :1, :16], 14 * 48), (qkv[:, ::7, 1:17], 7 * 48), (wide[..., 3:9], 32), (wide[:, :, 1, :8], 96), (wide[1, :, 2:, :8], 96),
                  (wide[:, None, :, :, 8:16], 32), (qkv[0, :, :1], 48), (qkv, 48), (qkv[0, 0], 48), (qkv[:0], 48)):
        rows, got = T._rows(t, t.shape[-1])
        assert at(rows) == at(t) and got == ld
        if t.numel():  # row r starts r * ld elements behind the first
            firsts = [rows.storage_offset() + sum(i * s for i, s in zip(index, rows.stride())) for index in torch.cartesian_prod(
                *[torch.arange(n) for n in t.shape[:-1]], torch.arange(1)).tolist()] if t.dim() > 1 else [rows.storage_offset()]
            assert [f - firsts[0] for f in firsts] == [r * ld for r in range(len(firsts))]
    for t in (qkv[:, :4, :16], wide[:, :, :2, :8], qkv[..., ::3], qkv.transpose(0, 1)[..., :16], qkv[:, :, :16].transpose(1, 2),
              qkv[:1, :, :16].expand(3, 7, 16), qkv[0, :1, :16].expand(7, 16), torch.zeros(40).as_strided((5, 8), (4, 1))):
        rows, got = T._rows(t, t.shape[-1])
        assert rows.is_contiguous() and rows.data_ptr() != t.data_ptr() and got == t.shape[-1] and torch.equal(rows, t)


def test_a_torch_without_the_raw_stream_call_is_asked_for_its_stream(monkeypatch):
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    spec = importlib.util.spec_from_file_location("esm_amd.training_again", T.__file__)
    again = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(again)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda gpu: SimpleNamespace(cuda_stream=100 + gpu))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    sent = []
    monkeypatch.setattr(L, "lib", lambda: SimpleNamespace(esmk_some_call=lambda *a: sent.append(a) or 0))
    again._call(3, "esmk_some_call", 1, 2)
    assert sent == [(1, 2, 103)]
