"""CPU tests of the low-bit library's boundary: exported symbols, argument checks of the C ABI (no launch is made), size
queries, refusals of the Python layer, and the oracle's formats against their definitions."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from gp_vae_amd import GpvaeError, _lib, ops
from oracle import lowbit_oracle as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_exports_are_what_the_header_declares():
    src = open(os.path.join(ROOT, "include", "gpvae_lowbit.h")).read()
    names = sorted(set(re.findall(r"\b(gpvae_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", src, flags=re.S))))
    out = subprocess.run(["nm", "-D", "--defined-only", _lib.LOWBIT_PATH], check=True, capture_output=True, text=True).stdout
    assert sorted(set(re.findall(r"\bT (\S+)$", out, flags=re.M))) == names == sorted(_lib.LOWBIT_SIGNATURES)
    lib = _lib.load_lowbit()
    assert lib.gpvae_lowbit_abi_version() == _lib.LOWBIT_ABI_VERSION == 1


def test_c_entry_points_refuse_bad_arguments_before_any_launch():
    lib = _lib.load_lowbit()
    nul, one, odd = C.c_void_p(0), C.c_void_p(16), C.c_void_p(8)
    err = lib.gpvae_lowbit_last_error
    assert lib.gpvae_quant_w4(nul, 1, 8, 8, one, 8, one, one) == -2 and b"dtype" in err()      # float64
    assert lib.gpvae_quant_w4(nul, 0, 0, 8, one, 8, one, one) == -3
    assert lib.gpvae_quant_w4(nul, 0, 8, 0, one, 8, one, one) == -4
    assert lib.gpvae_quant_w4(nul, 0, 8, 8, nul, 8, one, one) == -5
    assert lib.gpvae_quant_w4(nul, 0, 8, 8, one, 7, one, one) == -6
    assert lib.gpvae_quant_w4(nul, 0, 8, 8, one, 8, odd, one) == -7
    assert lib.gpvae_quant_w4(nul, 0, 8, 8, one, 8, one, nul) == -8 and b"gpvae_quant_w4" in err()
    assert lib.gpvae_load_w4(nul, 0, 8, 8, one, odd, one, 8) == -6
    assert lib.gpvae_load_w4(nul, 0, 8, 8, one, one, one, 7) == -8
    bad = [(dict(dt=5), -2), (dict(M=-1), -3), (dict(K=0), -4), (dict(N=-3), -5), (dict(X=nul), -6), (dict(ldx=7), -7),
           (dict(codes=odd), -8), (dict(exps=nul), -9), (dict(Y=nul), -12), (dict(ldy=8), -13)]
    for change, code in bad:
        a = dict(dt=0, M=3, K=8, N=9, X=one, ldx=8, codes=one, exps=one, Y=C.c_void_p(32), ldy=9)
        a.update(change)
        assert lib.gpvae_dense_w4(nul, a["dt"], a["M"], a["K"], a["N"], a["X"], a["ldx"], a["codes"], a["exps"], nul, 0, a["Y"],
                                  a["ldy"], one) == code, change
    bad = [(dict(dt=5), -2), (dict(M=-1), -3), (dict(K=0), -4), (dict(N=0), -5), (dict(X=nul), -6), (dict(ldx=8), -7),
           (dict(codes=odd), -8), (dict(exps=nul), -9), (dict(act=odd), -10), (dict(Y=nul), -11), (dict(ldy=7), -12)]
    for change, code in bad:
        a = dict(dt=0, M=3, K=8, N=9, X=one, ldx=9, codes=one, exps=one, act=one, Y=C.c_void_p(32), ldy=8)
        a.update(change)
        assert lib.gpvae_dense_vjp_w4(nul, a["dt"], a["M"], a["K"], a["N"], a["X"], a["ldx"], a["codes"], a["exps"], a["act"],
                                      a["Y"], a["ldy"], one) == code, change
    assert lib.gpvae_dense_w4(nul, 0, 0, 8, 8, nul, 8, nul, nul, nul, 0, nul, 8, nul) == 0           # no rows: nothing to do
    assert lib.gpvae_dense_vjp_w4(nul, 0, 0, 8, 8, nul, 8, nul, nul, nul, nul, 8, nul) == 0
    assert lib.gpvae_store_q8(nul, 0, 0, 8, nul, 8, 0, nul, 8, nul, nul) == 0
    assert lib.gpvae_load_q8(nul, 0, 0, 8, 0, nul, nul, nul, 8) == 0
    assert lib.gpvae_store_q8(nul, 0, 4, 8, one, 8, 0, C.c_void_p(32), 8, one, one) == -8             # Y without relu
    assert lib.gpvae_store_q8(nul, 0, 4, 8, one, 8, 1, C.c_void_p(32), 7, one, one) == -9
    assert lib.gpvae_store_q8(nul, 0, 4, 8, one, 8, 1, one, 9, one, one) == -9                         # in place, other ld
    assert lib.gpvae_store_q8(nul, 0, 4, 8, one, 8, 0, nul, 0, odd, one) == -10
    assert lib.gpvae_store_q8(nul, 0, 4, 8, one, 8, 0, nul, 0, one, odd) == -11
    assert lib.gpvae_load_q8(nul, 0, 4, 8, 0, one, one, one, 7) == -9
    bad = [(dict(dt=1), -2), (dict(M=-1), -3), (dict(K=0), -4), (dict(N=0), -5), (dict(codes=odd), -7), (dict(exps=nul), -8),
           (dict(dY=nul), -9), (dict(lddy=8), -10), (dict(dW=nul), -11), (dict(lddw=8), -12)]
    for change, code in bad:
        a = dict(dt=0, M=3, K=8, N=9, codes=one, exps=one, dY=one, lddy=9, dW=one, lddw=9)
        a.update(change)
        assert lib.gpvae_dense_grads_q8(nul, a["dt"], a["M"], a["K"], a["N"], 1, a["codes"], a["exps"], a["dY"], a["lddy"],
                                        a["dW"], a["lddw"], nul, one) == code, change


def test_sizes():
    lib = _lib.load_lowbit()
    assert lib.gpvae_w4_code_bytes(50, 4096) == 2 * 4096 * 16 and lib.gpvae_w4_exp_bytes(50, 4096) == 2 * 512 * 4
    assert lib.gpvae_w4_code_bytes(33, 33) == 2 * 64 * 16 and lib.gpvae_w4_code_bytes(0, 5) == 0
    assert lib.gpvae_q8_code_bytes(100, 35) == 13 * 64 * 8 and lib.gpvae_q8_exp_bytes(100, 35) == 13 * 8
    assert lib.gpvae_q8_code_bytes(0, 35) == 0


def test_python_layer_refuses():
    w = torch.zeros((1, 32, 4), dtype=torch.int32)
    e = torch.zeros((1, 4, 4), dtype=torch.uint8)
    w4 = ops.W4(w, e, 8, 9)
    with pytest.raises(GpvaeError):
        ops.W4(w, e, 33, 9)                                   # two blocks of 32 rows wanted
    with pytest.raises(GpvaeError):
        ops.W4(w.to(torch.int64), e, 8, 9)
    with pytest.raises(GpvaeError):
        ops.W4(w, e, 0, 9)
    qc, qe = torch.zeros((1, 32, 8), dtype=torch.uint8), torch.zeros((1, 4), dtype=torch.uint8)
    ops.Q8(qc, qe, 8, 9)
    with pytest.raises(GpvaeError):
        ops.Q8(qc, qe, 9, 9)
    with pytest.raises(GpvaeError):
        ops.Q8(qc.to(torch.int8), qe, 8, 9)
    X = torch.zeros((3, 8))
    for call in (lambda: ops.dense_w4(X, w4), lambda: ops.quant_w4(X), lambda: ops.store_q8(X), lambda: ops.load_w4(w4),
                 lambda: ops.dense_vjp_w4(torch.zeros((3, 9)), w4), lambda: ops.load_q8(ops.Q8(qc, qe, 8, 9)),
                 lambda: ops.dense_grads_q8(ops.Q8(qc, qe, 8, 9), torch.zeros((8, 4)))):
        with pytest.raises(GpvaeError):                        # CPU tensors: no fallback
            call()


def test_oracle_formats():
    rng = np.random.default_rng(3)
    W = rng.standard_normal((21, 13)) * 10.0 ** rng.integers(-3, 3, (21, 1))
    W[8:16, :8] = 0
    c, e = orc.quant_w4(W)
    V = orc.load_w4(c, e, 21, 13)
    assert (V[8:16, :8] == 0).all()
    for k in range(0, 21, 8):
        for n in range(0, 13, 8):
            T, Q = W[k:k + 8, n:n + 8], V[k:k + 8, n:n + 8]
            a = np.abs(T).max()
            if a:  # the tile's power of two: 3 < a 2^-e <= 6; the widest gap between values is 2 units
                assert np.abs(T - Q).max() <= a / 3 + 1e-300
    assert list(orc.e2m1_nearest(np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0, 6.0]))) == [0, 2, 2, 4, 4, 6, 6, 14, 7]
    X = rng.standard_normal((19, 37))
    for relu in (False, True):
        Y, c, e = orc.store_q8(X, relu)
        ref = np.maximum(X, 0) if relu else X
        V = orc.load_q8(c, e, 19, 37, relu)
        for m in range(0, 19, 8):
            for k in range(0, 37, 8):
                T, Q = ref[m:m + 8, k:k + 8], V[m:m + 8, k:k + 8]
                assert np.abs(T - Q).max() <= np.abs(T).max() / 127
        if relu:
            assert ((V > 0) == (X > 0)).all()


def test_workspace_queries_of_extreme_sizes():
    lib = _lib.load_lowbit()
    sizes = [-5, 0, 1, 2, 31, 33, 128, 129, 1000, 65537, 2 ** 25, 2 ** 30]
    for name in ("gpvae_dense_w4_workspace_bytes", "gpvae_dense_vjp_w4_workspace_bytes", "gpvae_dense_grads_q8_workspace_bytes"):
        fn = getattr(lib, name)
        for dt in (-1, 0, 1, 2, 3, 4):
            for m in sizes:
                for k in sizes:
                    for n in sizes:
                        w = fn(dt, m, k, n)
                        assert w >= 0, (name, dt, m, k, n)
                        if dt in (-1, 1, 4) or min(k, n) < 1 or m < (0 if "grads" in name else 1):
                            assert w == 0, (name, dt, m, k, n)


def test_gradients_refuse_rows_too_far_apart():
    fn = _lib.load_lowbit().gpvae_dense_grads_q8
    args = [None, 0, 2, 8, 2 ** 26 + 1, 0, 4096, 4096, 4096, 2 ** 26 + 1, 4096, 2 ** 26 + 1, None, 4096]
    assert fn(*args) == -5
    args[4], args[11] = 8, 8
    assert fn(*args) == -10


def test_launches_hold_fewer_than_2_32_threads_in_a_dimension():
    lib = _lib.load_lowbit()
    one, big = C.c_void_p(16), 2 ** 20
    assert lib.gpvae_store_q8(None, 2, big, big, one, big, 0, None, 0, one, one) == -3 and b"too large" in lib.gpvae_lowbit_last_error()
    assert lib.gpvae_load_q8(None, 2, big, big, 0, one, one, one, big) == -3
    assert lib.gpvae_quant_w4(None, 2, 2 ** 23, 2 ** 20, one, 2 ** 20, one, one) == -3
    assert lib.gpvae_load_w4(None, 2, 2 ** 23, 2 ** 20, one, one, one, 2 ** 20) == -3
    assert lib.gpvae_dense_grads_q8(None, 0, 1, 2 ** 30, 1, 0, one, one, one, 1, one, 1, None, one) == -4
    # many rows are taken in several launches, which share one workspace
    for fn, k, n in ((lib.gpvae_dense_w4_workspace_bytes, 640, 50), (lib.gpvae_dense_vjp_w4_workspace_bytes, 50, 640)):
        for rows in (2 ** 24, 2 ** 24 + 70, 2 ** 30):
            assert fn(0, rows, k, n) == fn(0, 2 ** 20, k, n) == 3 * 2 ** 20 * 640 * 2


def test_workspace_queries_of_sizes_the_calls_refuse():
    lib = _lib.load_lowbit()
    for big in (2 ** 30 + 1, 2 ** 31, 2 ** 32 * 128, 2 ** 38, 2 ** 40, 2 ** 62, 2 ** 63 - 1):
        for name in ("gpvae_dense_w4_workspace_bytes", "gpvae_dense_vjp_w4_workspace_bytes", "gpvae_dense_grads_q8_workspace_bytes"):
            fn = getattr(lib, name)
            for dt in (0, 2, 3):
                for at in range(3):
                    sizes = [1000, 1000, 1000]
                    sizes[at] = big
                    assert fn(dt, *sizes) == 0, (name, dt, sizes)
    assert lib.gpvae_dense_w4_workspace_bytes(0, 1000, 1000, 2 ** 25 + 1) == 0 and lib.gpvae_dense_vjp_w4_workspace_bytes(0, 1000, 1000, 2 ** 25 + 1) == 0
    assert lib.gpvae_dense_grads_q8_workspace_bytes(0, 1000, 1000, 2 ** 26 + 1) == 0
    assert lib.gpvae_dense_w4_workspace_bytes(0, 2 ** 30, 2 ** 30, 2 ** 25) > 0 and lib.gpvae_dense_vjp_w4_workspace_bytes(0, 2 ** 30, 2 ** 30, 2 ** 25) > 0
