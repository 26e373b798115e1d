"""Host side of the text operators without a GPU: the C entry points refuse bad arguments before any
launch (the addresses below are never dereferenced), and the workspace sizes."""

from __future__ import annotations

import ctypes

import pytest
import torch

from diffucore_b200 import _lib, kernels, text
from tests.conftest import has_b200

A, BF16, F32 = 0x100000, _lib.DTYPE_BF16, _lib.DTYPE_F32
no_gpu = pytest.mark.skipif(has_b200(), reason="host-side validation only; fake addresses must never reach a GPU")


def refused(status: int, why: bytes) -> None:
    assert status != 0
    assert why in _lib.load().dc_last_error(), _lib.load().dc_last_error()


@no_gpu
def test_projection_arguments():
    lib = _lib.load()

    def linear(x=A, ldx=64, w=A, ldw=64, bias=None, res=None, ldr=0, y=A, ldy=32, z=None, ldz=0, dtype=BF16, M=40,
               N=32, K=64, act=0):
        return lib.dc_linear(x, ldx, w, ldw, bias, res, ldr, y, ldy, z, ldz, dtype, M, N, K, act, None)

    refused(linear(dtype=F32), b"bf16 or fp16")
    refused(linear(K=0), b"bad shape")
    refused(linear(M=-1), b"bad shape")
    refused(linear(act=9), b"activation")
    refused(linear(x=None), b"x is null")
    refused(linear(x=A + 2), b"16-byte")
    refused(linear(ldx=60), b"16-byte")
    refused(linear(ldw=56), b"smaller than its row")
    refused(linear(y=None), b"y is null")
    refused(linear(y=A + 1), b"aligned")
    refused(linear(ldy=31), b"leading dimension")
    refused(linear(z=A, ldz=30), b"pre-activations")
    refused(linear(z=A + 4, ldz=32), b"pre-activations")
    assert linear(M=0, x=None) == 0
    refused(linear(M=4, x=A + 1), b"aligned")               # few rows: element alignment only
    refused(linear(M=4, ldw=63), b"smaller than its row")
    refused(linear(), b"")                                  # no device here
    refused(lib.dc_gated_linear(A, 64, A, 64, A, 64, None, None, A, 32, A, None, 32, BF16, 4, 32, 64, 2, None),
            b"go together")
    refused(lib.dc_gated_linear(A, 64, A, 64, None, 64, None, None, A, 32, None, None, 0, BF16, 4, 32, 64, 2, None),
            b"w_up is null")
    refused(lib.dc_linear_dx(A, A, 32, A, 64, None, 0, A, 64, BF16, 4, 32, 64, None), b"go together")
    refused(lib.dc_linear_dx(A, None, 32, A, 64, None, 0, A, 63, BF16, 4, 32, 64, None), b"leading dimension")
    refused(lib.dc_linear_dw(A, None, 32, A, 64, A, None, 64, BF16, 0, 32, 64, None), b"no rows")
    refused(lib.dc_linear_dw(A, A, 32, A, 64, A, None, 64, BF16, 4, 32, 64, None), b"go together")


@no_gpu
def test_pointwise_norm_and_embedding_arguments():
    lib = _lib.load()
    n = ctypes.c_size_t(0)
    assert lib.dc_act_grad_workspace(100, 30, ctypes.byref(n)) == 0 and n.value % (2 * 32 * 4) == 0
    refused(lib.dc_act_grad(A, 32, None, None, 0, None, None, 0, None, None, None, 0, BF16, 4, 32, 0, None), b"nothing")
    refused(lib.dc_act_grad(A, 32, None, None, 0, A, None, 32, A, None, A, 1 << 20, BF16, 4, 32, 0, None),
            b"pre-activations")
    refused(lib.dc_act_grad(A, 32, A, None, 32, A, None, 32, A, None, A, 8, BF16, 4, 32, 0, None), b"workspace")
    refused(lib.dc_act_grad(A, 32, A, None, 32, A, None, 32, A, A, A, 1 << 20, BF16, 4, 32, 0, None), b"db1")
    refused(lib.dc_layer_norm(A, 32, A, A, _lib.DTYPE_F16, A, 32, None, None, BF16, 4, 32, 1e-5, None), b"type")
    refused(lib.dc_layer_norm(A, 32, A, A, BF16, A, 31, None, None, BF16, 4, 32, 1e-5, None), b"leading dimension")
    refused(lib.dc_layer_norm(A, 32, A, A, BF16, A, 32, A, None, BF16, 4, 32, 1e-5, None), b"go together")
    refused(lib.dc_layer_norm(A, 32, A, A, BF16, A, 32, None, None, BF16, 4, 0, 1e-5, None), b"bad shape")
    assert lib.dc_layer_norm_grad_workspace(1000, 96, ctypes.byref(n)) == 0 and n.value >= 2 * 96 * 4
    refused(lib.dc_layer_norm_grad(A, 32, A, 32, A, BF16, A, A, A, 32, A, A, A, 8, BF16, 400, 32, None), b"workspace")
    refused(lib.dc_layer_norm_grad(A, 32, A, 32, A, BF16, A, A, A, 32, None, A, None, 0, BF16, 4, 32, None), b"db")
    refused(lib.dc_embedding(A, 1, 4, A, 32, 0, 32, 1.0, A, 32, BF16, None), b"bad shape")
    refused(lib.dc_embedding(A + 4, 1, 4, A, 32, 10, 32, 1.0, A, 32, BF16, None), b"aligned")
    refused(lib.dc_embedding(A, 1, 4, A, 16, 10, 32, 1.0, A, 32, BF16, None), b"leading dimension")
    assert lib.dc_embedding_grad_workspace(5000, 1000, 64, ctypes.byref(n)) == 0
    refused(lib.dc_embedding_grad(A, 64, A, 1, 5000, 1000, 64, -1, 1.0, A, A, n.value - 1, BF16, None), b"workspace")
    refused(lib.dc_embedding_grad(A, 64, A, 1, 5000, 1000, 64, -1, 1.0, None, A, n.value, BF16, None), b"dtable")


@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (8192, (1 << 19) - 1, 8), (8193, 1000, 8), (8192, 1 << 19, 8),
                                   (1 << 20, 262143, 64), (1 << 20, 262144, 64)])
def test_embedding_workspace_holds_keys_and_partials(T, V, D):
    """Keys and indices of the sorted tokens (two pairs for the radix passes) and two fp32 partial
    rows per chunk of at most 128 sorted places."""
    n = ctypes.c_size_t(0)
    assert _lib.load().dc_embedding_grad_workspace(T, V, D, ctypes.byref(n)) == 0
    pairs = 1 if T <= 8192 and V < 1 << 19 else 2
    assert n.value >= pairs * 8 * T + -(-T // 128) * 2 * D * 4


def test_functions_refuse_cpu_tensors_and_bad_shapes():
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    for call in (lambda: text.linear(x, w), lambda: text.gated_linear(x, w, w), lambda: text.layer_norm(x),
                 lambda: text.embedding(torch.zeros(2, dtype=torch.long), w)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(ValueError, match="width"):
        text.linear(x, torch.zeros(4, 9, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="padding_idx"):
        text.embedding(torch.zeros(2, dtype=torch.long), w, padding_idx=4)


def test_matrix_operand_pads_only_what_a_tile_load_cannot_take():
    t = torch.randn(6, 24).to(torch.bfloat16)
    assert kernels.matrix_operand(t).data_ptr() == t.data_ptr()
    assert kernels.matrix_operand(t[:, :20]).data_ptr() == t.data_ptr()      # rows stay 48 bytes apart
    for v in (t[:, 1:], torch.randn(5, 21).to(torch.bfloat16), t.t(), t[:1].expand(4, 24), t[:, :1]):
        m = kernels.matrix_operand(v)
        assert torch.equal(m, v) and m.stride(0) % 8 == 0 and m.data_ptr() % 16 == 0 and m.stride(1) == 1
        assert m.stride(0) >= m.shape[1]
    one = torch.randn(3, 17).to(torch.bfloat16)[:1]
    assert kernels.matrix_operand(one).data_ptr() == one.data_ptr()          # one row: any pitch


@no_gpu
def test_pad_rows_arguments():
    lib = _lib.load()

    def pad(count=1, src=A, ld=21, rows=5, cols=21, dst=A, ldd=24):
        i64 = ctypes.c_int64 * 1
        ptr = ctypes.c_void_p * 1
        return lib.dc_pad_rows(count, ptr(src), i64(ld), i64(rows), i64(cols), ptr(dst), i64(ldd), None)

    refused(pad(count=0), b"1 to 3")
    refused(pad(count=4), b"1 to 3")
    refused(lib.dc_pad_rows(1, None, None, None, None, None, None, None), b"null array")
    refused(pad(cols=0), b"bad shape")
    refused(pad(rows=-1), b"bad shape")
    refused(pad(src=None), b"null pointer")
    refused(pad(src=A + 1), b"aligned")
    refused(pad(dst=A + 8), b"aligned")
    refused(pad(ldd=20), b"leading dimension")
    refused(pad(ldd=16), b"leading dimension")
    refused(pad(ld=-1), b"leading dimension")
    assert pad(rows=0, src=None) == 0
    refused(pad(), b"")                                     # no device here


def test_forward_mode_tangents_are_refused():
    """Before anything else, so that no path drops a tangent."""
    import torch.autograd.forward_ad as fwd
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    b, ids = torch.zeros(4, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.long)
    for reverse in (False, True):
        with fwd.dual_level():
            def dual(t):
                return fwd.make_dual(t.clone().requires_grad_(reverse), torch.ones_like(t))

            for call in (lambda: text.linear(dual(x), w), lambda: text.linear(x, dual(w)), lambda: text.linear(x, w, dual(b)),
                         lambda: text.gated_linear(x, w, dual(w)), lambda: text.layer_norm(dual(x)),
                         lambda: text.layer_norm(x, dual(x[0])), lambda: text.embedding(ids, dual(w)),
                         lambda: kernels.linear_dx(dual(x), w), lambda: kernels.linear_dw(x, dual(w))):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()


@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (300, 9, 5000), (8192, (1 << 19) - 1, 8), (8193, 1000, 8), (8192, 1 << 19, 8),
                                   (98304, 1000, 8), (98305, 600000, 2048), (1 << 20, 262143, 64), (1 << 22, 262144, 1)])
def test_embedding_workspace_is_what_the_launches_write(T, V, D):
    """The sum's partials have chunks of 8 sorted places, doubled up to 64 while there are 16 CTAs for each
    of 148 SMs; the radix passes' counts have a row per 1024 tokens, one more where they are scanned."""
    n = ctypes.c_size_t(0)
    assert _lib.load().dc_embedding_grad_workspace(T, V, D, ctypes.byref(n)) == 0
    slabs, chunk = -(-D // 1024), 8
    while chunk < 64 and -(-T // (2 * chunk)) * slabs >= 16 * 148:
        chunk *= 2
    partials = -(-T // chunk) * 2 * D * 4
    if T <= 8192 and V < 1 << 19:
        need = [T * 4, T * 4, partials]
    else:
        bits = V.bit_length()                               # keys 0 .. V
        passes = -(-bits // 9)
        tiles = -(-T // 1024)
        need = [T * 4] * 4 + [(tiles + (tiles >= 96)) * 4 << -(-bits // passes), partials]
    assert sum(need) <= n.value <= sum(need) + 256 * len(need)
