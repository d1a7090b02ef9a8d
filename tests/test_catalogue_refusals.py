"""What the catalogue head's C entry points refuse before anything is launched (no GPU needed: every call here ends on the host)."""
import ctypes

import pytest
import torch

import star_gcn_amd._lib as L
from star_gcn_amd import functional as SF
from star_gcn_amd import ops

P = ctypes.c_void_p(16)      # a pointer that is never followed


def quant(codes=P, scale=P, x=P, ldx=8, res=None, ldr=0, rows=2, dim=8, dtype=0, norm=1, eps=1e-6):
    return L.lib().sg_quant_rows_i8_hip(codes, scale, None, x, ldx, res, ldr, None, 0, rows, dim, dtype, norm, eps, None)


def gemm(C=P, ldc=8, dtype=0, A=P, lda=64, sa=P, B=P, ldb=64, sb=P, M=4, N=8, K=64, act=0, ws=None, wsn=0):
    return L.lib().sg_gemm_i8_hip(C, ldc, dtype, A, lda, sa, B, ldb, sb, None, M, N, K, act, 0.1, ws, wsn, None)


def sample(ids=P, prob=P, l=P, ld=8, dtype=0, u=P, rows=2, n=8, t=1.0, k=0, p=1.0, m=0.0, ws=P, wsn=1 << 40):
    return L.lib().sg_sample_rows_hip(ids, prob, l, ld, dtype, u, rows, n, t, k, p, m, None, None, None, None, ws, wsn, None)


def distill(loss=P, stats=P, p=P, s=P, ld=8, dtype=0, t=P, ids=P, rows=2, n=8, k=3, temp=1.0, ws=P, wsn=1 << 40):
    return L.lib().sg_distill_hip(loss, stats, p, s, ld, dtype, t, ids, rows, n, k, temp, 1.0, ws, wsn, None)


def distill_bwd(grad=P, s=P, ld=8, dtype=0, stats=P, p=P, ids=P, rows=2, n=8, k=3, temp=1.0, g=P):
    return L.lib().sg_distill_bwd_hip(grad, s, ld, dtype, stats, p, ids, rows, n, k, temp, 1.0, g, None)


NAN = float("nan")


@pytest.mark.parametrize("call,code", [
    (lambda: quant(dtype=3), -1), (lambda: quant(rows=-1), -1), (lambda: quant(dim=0), -1), (lambda: quant(dim=16385, ldx=16385), -2),
    (lambda: quant(codes=None), -1), (lambda: quant(scale=None), -1), (lambda: quant(x=None), -1), (lambda: quant(ldx=7), -1),
    (lambda: quant(res=P, ldr=7), -1), (lambda: quant(eps=-1.0), -1), (lambda: quant(eps=NAN), -1), (lambda: quant(rows=1 << 31), -1),
    (lambda: gemm(dtype=-1), -1), (lambda: gemm(act=9), -1), (lambda: gemm(M=-1), -1), (lambda: gemm(K=131072, lda=131072, ldb=131072), -2),
    (lambda: gemm(C=None), -1), (lambda: gemm(A=None), -1), (lambda: gemm(B=None), -1), (lambda: gemm(sa=None), -1), (lambda: gemm(sb=None), -1),
    (lambda: gemm(lda=63), -1), (lambda: gemm(ldb=63), -1), (lambda: gemm(ldc=7), -1), (lambda: gemm(M=1 << 30), -2),
    (lambda: sample(dtype=7), -1), (lambda: sample(rows=-1), -1), (lambda: sample(n=1 << 30, ld=1 << 30), -2), (lambda: sample(ids=None), -1),
    (lambda: sample(prob=None), -1), (lambda: sample(l=None), -1), (lambda: sample(u=None), -1), (lambda: sample(ld=7), -1),
    (lambda: sample(t=-1.0), -1), (lambda: sample(t=NAN), -1), (lambda: sample(k=-1), -1), (lambda: sample(p=-0.1), -1),
    (lambda: sample(p=NAN), -1), (lambda: sample(m=-1.0), -1),
    (lambda: distill(dtype=3), -1), (lambda: distill(rows=-1), -1), (lambda: distill(n=0), -1), (lambda: distill(k=1025), -2),
    (lambda: distill(ld=7), -1), (lambda: distill(temp=0.0), -1), (lambda: distill(temp=NAN), -1), (lambda: distill(temp=float("inf")), -1),
    (lambda: distill(loss=None), -1), (lambda: distill(s=None), -1), (lambda: distill(t=None), -1), (lambda: distill(ids=None), -1),
    (lambda: distill(p=None), -1), (lambda: distill(stats=None), -1), (lambda: distill(ws=None), -5), (lambda: distill(wsn=1), -5),
    (lambda: distill_bwd(dtype=3), -1), (lambda: distill_bwd(grad=None), -1), (lambda: distill_bwd(g=None), -1), (lambda: distill_bwd(ld=7), -1),
    (lambda: gemm(M=(1 << 30) - 1, N=1), -2), (lambda: sample(rows=1 << 23, n=20000, ld=20000), -2), (lambda: distill(rows=1 << 24), -2),
    (lambda: distill_bwd(rows=1 << 24), -2), (lambda: distill_bwd(k=1025), -2), (lambda: distill_bwd(temp=-1.0), -1), (lambda: distill_bwd(stats=None), -1), (lambda: distill_bwd(ids=None), -1),
])
def test_entry_points_refuse(call, code):
    assert call() == code
    assert L.lib().sg_last_error()


def test_split_products_and_long_rows_ask_for_their_workspace():
    lib = L.lib()
    need = lib.sg_gemm_i8_workspace_bytes(64, 64, 8192)
    assert need > 0
    assert gemm(M=64, N=64, K=8192, lda=8192, ldb=8192, ldc=64) == -5
    assert gemm(M=64, N=64, K=8192, lda=8192, ldb=8192, ldc=64, ws=P, wsn=need - 1) == -5
    assert lib.sg_gemm_i8_workspace_bytes(0, 64, 8192) == 0
    need = lib.sg_sample_rows_workspace_bytes(1, 1000000, 0)
    if need:
        assert sample(rows=1, n=1000000, ld=1000000, wsn=need - 1) == -5 and sample(rows=1, n=1000000, ld=1000000, ws=None, wsn=0) == -5


def test_nothing_to_do_needs_no_gpu():
    assert quant(rows=0) == 0 and gemm(M=0) == 0 and gemm(N=0) == 0 and sample(rows=0) == 0 and distill_bwd(rows=0) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 4)
    for call in (lambda: ops.quantize_rows(x), lambda: ops.rms_norm_i8(x), lambda: ops.sample_rows(x, x[0]),
                 lambda: ops.gemm_i8(x.char(), x[:, 0], x.char(), x[:, 0]), lambda: SF.distill_loss(x, x, x.int(), 1.0)):
        with pytest.raises(L.StarGCNError):
            call()


@pytest.mark.parametrize("temp", [1e-39, 1e-45, 2.0 ** -63.01, 2.0 ** 63.01, 3e38, -1.0, NAN])
def test_distill_refuses_temperatures_whose_square_leaves_32_bits(temp):
    assert distill(temp=temp) == -1 and distill_bwd(temp=temp) == -1
    for t in (2.0 ** -63, 2.0 ** 63):      # the ends themselves pass this check: the next one refuses the missing workspace
        assert distill(temp=t, ws=None) == -5


def test_long_rows_always_ask_for_a_workspace_and_not_for_more_than_a_batch():
    size = L.lib().sg_sample_rows_workspace_bytes
    for n in (16385, 1000000, 1 << 20, (1 << 20) + 1, (1 << 30) - 1):
        for dtype in (0, 1, 2):
            need = size(1, n, dtype)
            assert need > 0
            assert sample(rows=1, n=n, ld=n, dtype=dtype, wsn=need - 1) == -5 and sample(rows=1, n=n, ld=n, dtype=dtype, ws=None, wsn=0) == -5
    assert size(1, 16384, 0) == 0
    for rows in (16385, 69878, (1 << 23) - 1):
        assert size(rows, 20000, 0) == size(16384, 20000, 0) < 1300 << 20
