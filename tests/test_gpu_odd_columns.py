"""Dense INT8 products whose rows end inside 16 bytes, into part of a wider matrix: the columns behind the result stay as they were."""
import ctypes

import numpy as np
import pytest
import torch

import oracle
from bare_metal_b200 import _lib
from bare_metal_b200 import igemm as ig
from _gpu import T, assert_clean_status, dev, options

pytestmark = pytest.mark.gpu

KERNELS = {"pairs": dict(force_bn=256, dense_pair=1), "lone 256": dict(force_bn=256, dense_pair=0), "lone 128": dict(force_bn=128),
           "lone 64": dict(force_bn=64), "lanes": dict(dense_decode=1), "chosen": {}}


def run(kind, A, W, out, N, sa, sw, zero):
    M, K = A.shape
    if kind == "f16":
        ig.w8a8_linear(A, W, out, sa, sw, M, N, K)
    elif kind == "i32":
        ig.igemm_i32(A, W, out, M, N, K, ig.BM_B_NK)
    elif kind == "tensor":
        ig.igemm_wmma(A, W, out, M, N, K, 0.01, 0.02, ig.BM_B_NK)
    else:
        ig.igemm_pipelined_cpasync_perchannel(A, W, out, M, N, K, sw, zero, ig.BM_B_NK)


def expected(kind, acc, sa, sw, zero):
    if kind == "f16":
        return oracle.dequant_w8a8_f16(acc, sa, sw)
    if kind == "i32":
        return acc
    if kind == "tensor":
        return oracle.dequant_per_tensor(acc, 0.01, 0.02)
    return (acc.astype(np.float32) - zero.astype(np.float32)) * sw


@pytest.mark.parametrize("kernel", list(KERNELS))
@pytest.mark.parametrize("kind", ["f16", "i32", "tensor", "channel"])
@pytest.mark.parametrize("M,N", [(200, 333), (33, 65), (300, 7), (2400, 1537)])          # the last: half tiles in a partly filled last wave of pairs
def test_columns_behind_the_result(M, N, kind, kernel):
    K = 144
    A, W = oracle.gen_int8((M, K), 7, 1), oracle.gen_int8((N, K), 7, 2)
    sa, sw = oracle.gen_scales(M, 7, 3), oracle.gen_scales(N, 7, 4)
    zero = np.arange(N, dtype=np.int32) * 3 - 50
    acc = oracle.igemm_nt(A, W)
    want = expected(kind, acc, sa, sw, zero)
    dtype = {"f16": torch.float16, "i32": torch.int32}.get(kind, torch.float32)
    for pitch in (-(-N // 8) * 8, -(-N // 8) * 8 + 24):
        wide = torch.full((M + 1, pitch), 7, dtype=dtype, device=dev())
        with options(**KERNELS[kernel]):
            run(kind, T(A), T(W), wide[:M, :N], N, T(sa), T(sw), T(zero))
        assert_clean_status()
        got = wide.cpu().numpy()
        assert np.array_equal(got[:M, :N], want)
        assert (got[:M, N:] == 7).all() and (got[M] == 7).all()


@pytest.mark.parametrize("kernel", ["pairs", "lone 256", "lone 128"])
@pytest.mark.parametrize("copies", [1, 3])
def test_a_slab_that_goes_to_several_matrices(copies, kernel):
    """The gathering product with destinations on this GPU: a slab of 333 columns at column 16 of each."""
    M, N, K, pitch = 200, 333, 144, 384
    A, W = oracle.gen_int8((M, K), 8, 1), oracle.gen_int8((N, K), 8, 2)
    sa, sw = oracle.gen_scales(M, 8, 3), oracle.gen_scales(N, 8, 4)
    wide = torch.full((copies, M, pitch), 7, dtype=torch.float16, device=dev())
    a, w, s, t = T(A), T(W), T(sa), T(sw)
    ptrs = (ctypes.c_void_p * copies)(*(wide[i].data_ptr() + 32 for i in range(copies)))
    with options(**KERNELS[kernel]):
        rc = _lib.load().bm_w8a8_f16_gather(a.data_ptr(), w.data_ptr(), ptrs, copies, 0, s.data_ptr(), t.data_ptr(), M, N, K, pitch, ig.BM_B_NK,
                                            torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert_clean_status()
    want = oracle.dequant_w8a8_f16(oracle.igemm_nt(A, W), sa, sw)
    for got in wide.cpu().numpy():
        assert np.array_equal(got[:, 16:16 + N].view(np.uint16), want.view(np.uint16))
        assert (got[:, :16] == 7).all() and (got[:, 16 + N:] == 7).all()
