"""Host-side argument checks of the 4-bit entry points, without a GPU."""
import ctypes as C

import numpy as np
import pytest

from mruntime_b200 import capi

BUF = np.zeros(4096, np.uint8)
P = BUF.ctypes.data
INVALID, SHAPE, DTYPE, UNSUPPORTED = 1, 2, 3, 7


def last() -> bytes:
    return capi.lib().mrt_last_error_string()


@pytest.mark.parametrize("src,dt,N,K,group,want", [
    (None, 0, 4, 128, 32, INVALID), (P, 7, 4, 128, 32, DTYPE), (P, 0, 4, 128, 16, SHAPE), (P, 0, 4, 128, 0, SHAPE),
    (P, 0, 0, 128, 32, SHAPE), (P, 0, 4, 0, 32, SHAPE), (P, 0, 4, 100, 32, SHAPE), (P, 0, 4, 96, 64, SHAPE),
    (P, 0, 1 << 31, 128, 32, SHAPE), (P, 0, -1, 128, 32, SHAPE)])
def test_upload_refuses(src, dt, N, K, group, want):
    h = C.c_void_p(1)
    assert capi.lib().mrt_weight_q4_upload(src, dt, 0, N, K, group, 0, None, C.byref(h)) == want and last()
    assert not h.value


@pytest.mark.parametrize("codes,scales,sdt,N,K,group,want", [
    (None, P, 0, 4, 128, 32, INVALID), (P, None, 0, 4, 128, 32, INVALID), (P, P, 3, 4, 128, 32, DTYPE),
    (P, P, 0, 4, 128, 48, SHAPE), (P, P, 0, 4, 130, 32, SHAPE)])
def test_import_refuses(codes, scales, sdt, N, K, group, want):
    h = C.c_void_p()
    assert capi.lib().mrt_weight_q4_import(codes, scales, sdt, None, 0, N, K, group, None, C.byref(h)) == want and last()


@pytest.mark.parametrize("pages,page,heads,D,theta,want", [
    (0, 16, 2, 64, 0.0, SHAPE), (1, 8, 2, 64, 0.0, SHAPE), (1, 0, 2, 64, 0.0, SHAPE), (1, 24, 2, 64, 0.0, SHAPE),
    (1, 16, 0, 64, 0.0, SHAPE), (1, 16, 2, 96, 0.0, UNSUPPORTED), (1, 16, 2, 256, 0.0, UNSUPPORTED),
    (1, 16, 2, 64, 0.5, INVALID), (1, 16, 2, 64, -1.0, INVALID), (1, 16, 2, 64, float("nan"), INVALID),
    (1, 16, 2, 64, float("inf"), INVALID)])
def test_cache_refuses(pages, page, heads, D, theta, want):
    h = C.c_void_p(1)
    assert capi.lib().mrt_kv_q4_create(pages, page, heads, D, theta, C.byref(h)) == want and last()
    assert not h.value


def test_null_handles():
    lib = capi.lib()
    b = capi.KvBatch(1, 1, 1, 1, P, P, P, 1)
    n = C.c_size_t()
    assert lib.mrt_gemv_q4(None, P, 1, None, 0, P, 0, 1, 1, 0, None) == INVALID
    assert lib.mrt_weight_q4_shape(None, None, None, None) == INVALID
    assert lib.mrt_weight_q4_read(None, P, 1, None) == INVALID
    assert lib.mrt_weight_q4_attach_bias(None, P, 0, 0, None) == INVALID
    assert lib.mrt_weight_q4_upload(P, 0, 0, 4, 128, 32, 0, None, None) == INVALID
    assert lib.mrt_weight_q4_import(P, P, 0, None, 0, 4, 128, 32, None, None) == INVALID
    assert lib.mrt_kv_q4_create(1, 16, 2, 64, 0.0, None) == INVALID
    assert lib.mrt_kv_q4_append(None, C.byref(b), 0, None, 0, 0, None, 0, P, 128, P, 128, None) == INVALID
    assert lib.mrt_kv_q4_read(None, C.byref(b), 0, P, 128, P, 128, None) == INVALID
    assert lib.mrt_kv_q4_attention(None, C.byref(b), 0, P, 128, 2, P, 128, 1.0, 1, P, 16, None) == INVALID
    assert lib.mrt_kv_q4_attention_workspace(None, C.byref(b), 2, C.byref(n)) == INVALID
    assert lib.mrt_weight_q4_free(None) == 0 and lib.mrt_kv_q4_free(None) == 0


def test_no_gpu_reports_cuda_error():
    import torch

    if torch.cuda.is_available():
        pytest.skip("host has a GPU")
    h = C.c_void_p()
    assert capi.lib().mrt_kv_q4_create(1, 16, 2, 64, 0.0, C.byref(h)) == 4
    assert capi.lib().mrt_weight_q4_upload(P, 0, 0, 4, 128, 32, 0, None, C.byref(h)) == 4
