"""Refusals of the operators beside the token loop that need no GPU: the
Python wrappers' and the C entry points' own."""
import ctypes

import numpy as np
import pytest
import torch

from mojostream_b200 import _lib
from mojostream_b200.runtime import LogitRules, Q4GroupWeight, _check_2d, _dtype_code
from rules_check import reference, words


class FakeCuda:
    """What the wrappers read of a CUDA matrix."""

    def __init__(self, shape, stride, device=0, dtype=torch.float32):
        self.is_cuda, self.dtype = True, dtype
        self.device = torch.device("cuda", device)
        self.shape, self._stride = torch.Size(shape), stride

    def stride(self):
        return self._stride


def test_matrices_with_any_row_stride():
    assert _check_2d(FakeCuda((3, 8), (8, 1)), "x", 0) == 8
    assert _check_2d(FakeCuda((3, 8), (11, 1)), "x", 0, cols=8, rows=3) == 11
    assert _check_2d(FakeCuda((1, 8), (0, 1)), "x", 0) == 8    # one row: its stride is free
    assert _check_2d(FakeCuda((3, 1), (5, 7)), "x", 0) == 5    # one column


@pytest.mark.parametrize("t,needle", [
    (torch.zeros(2, 8), "CUDA device 0"),
    (FakeCuda((2, 8), (8, 1), device=1), "CUDA device 0"),
    (FakeCuda((2, 8), (1, 2)), "adjacent"),
    (FakeCuda((2, 8), (0, 1)), "adjacent"),     # a broadcast row
    (FakeCuda((2, 8), (7, 1)), "adjacent"),     # rows that overlap
    (FakeCuda((2, 9), (9, 1)), "shape"),
    (FakeCuda((3, 8), (8, 1)), "shape"),
    (FakeCuda((2, 8, 1), (8, 1, 1)), "shape"),
])
def test_refused_matrices(t, needle):
    with pytest.raises(ValueError, match=needle):
        _check_2d(t, "x", 0, cols=8, rows=2)


def test_types():
    assert [_dtype_code(FakeCuda((1, 1), (1, 1), dtype=d), "x")
            for d in (torch.float32, torch.bfloat16, torch.float16)] == [0, 1, 2]
    with pytest.raises(ValueError, match="float64"):
        _dtype_code(FakeCuda((1, 1), (1, 1), dtype=torch.float64), "x")


@pytest.mark.parametrize("K,N,group,change,needle", [
    (128, 64, 48, {}, "group"), (96, 64, 64, {}, "group"), (128, 63, 32, {}, "N % 2"),
    (0, 64, 32, {}, "K 0"), (128, 64, 32, {"scales": np.zeros((4, 64), np.float32)}, "scales"),
    (128, 64, 32, {"scales": np.zeros((3, 64), np.float16)}, "scales"),
    (128, 64, 32, {"w_rx": np.zeros((128, 64), np.uint8)}, "w_rx"),
    (128, 64, 32, {"zeros": np.zeros((4, 64), np.int32)}, "zeros"),
    (128, 64, 32, {"zeros": np.zeros((4, 32), np.uint8)}, "zeros"),
])
def test_refused_weights(K, N, group, change, needle):
    args = {"w_rx": np.zeros((128, 32), np.uint8), "scales": np.zeros((4, 64), np.float16), "zeros": None}
    args.update(change)
    with pytest.raises(ValueError, match=needle):
        Q4GroupWeight(None, args["w_rx"], args["scales"], K, N, group, zeros=args["zeros"])


def test_rules_need_device_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        LogitRules(hist=torch.zeros(3, dtype=torch.int32), hist_off=torch.zeros(2, dtype=torch.int32))


def test_null_arguments_are_refused_without_a_device():
    L = _lib.lib()
    bad = 1  # MS_ERR_INVALID_ARG
    h = ctypes.c_void_p()
    assert L.ms_q4g_weight_create(None, None, None, 2, None, 32, 32, 32, ctypes.byref(h)) == bad
    assert L.ms_q4g_weight_destroy(None, None) == bad
    assert L.ms_q4g_weight_bytes(None) == 0
    assert L.ms_q4g_gemm(None, None, None, 1, None, 1, 0, 1, 0, None) == bad
    assert L.ms_q4g_gated(None, None, None, 0, None, 1, None, 1, 0, 1, None) == bad
    assert L.ms_logit_rules_apply(None, None, 1, None, 1, 0, 1, 1,
                                  ctypes.byref(_lib.LogitRulesDesc()), None) == bad


def test_the_rules_reference_itself():
    """A row worked by hand: rep 2, presence 1, frequency 0.5."""
    x = np.array([[4, -2, 1, 0, 3]], np.float32)
    y = reference(x, hist=np.array([0, 1, 1, 9, -1], np.int32), hist_off=np.array([0, 5]),
                  repetition=[2], presence=[1], frequency=[0.5],
                  bias_id=np.array([2, 3, 2], np.int32), bias_val=np.array([9, 1, -1], np.float32),
                  bias_off=np.array([0, 3]), mask=words(np.array([[1, 1, 1, 1, 0]], bool)))
    assert y.tolist() == [[4 / 2 - 1.5, -4 - 2, 0, 1, -np.inf]]
