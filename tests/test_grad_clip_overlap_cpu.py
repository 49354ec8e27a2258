"""Scaling refuses tensors that overlap in memory, before any CUDA call: addresses only, without a GPU."""
import ctypes

import pytest
import torch

from float8_experimental_b200 import _native as N

vp = ctypes.c_void_p
BF16, FP16, FP32 = (N.hp_code(t) for t in (torch.bfloat16, torch.float16, torch.float32))


def clip(*tensors):
    """tensors: (address, elements, type)"""
    n = len(tensors)
    p, s, c = zip(*tensors)
    return N.load().f8b200_multi_clip((vp * n)(*p), (ctypes.c_int64 * n)(*s), (ctypes.c_int * n)(*c), n, vp(256), 1.0, None)


OVERLAPS = {"the same twice": [(4096, 10, FP32), (4096, 10, FP32)], "one inside another": [(4096, 100, FP32), (4200, 2, BF16)],
            "by one element": [(4096, 10, BF16), (4114, 10, BF16)],
            "not neighbours in the list": [(8192, 4, FP32), (4096, 8, FP16), (9000, 2, FP32), (4110, 8, FP16)],
            "descending": [(8192, 10, FP32), (8188, 2, FP32)], "types of other widths": [(4096, 3, FP32), (4104, 1, BF16)]}
APART = {"touching": [(4096, 10, BF16), (4116, 10, BF16)], "descending": [(8192, 10, FP32), (8184, 2, FP32)],
         "empty inside another": [(4096, 100, FP32), (4200, 0, FP32), (8192, 1, FP32)],
         "shuffled": [(4096 + 64 * ((7 * i) % 40), 16, FP32) for i in range(40)]}


@pytest.mark.parametrize("name", OVERLAPS)
def test_overlapping_tensors_are_refused(name):
    assert clip(*OVERLAPS[name]) == N.ERR_BAD_ARG
    assert clip(*OVERLAPS[name][::-1]) == N.ERR_BAD_ARG


@pytest.mark.parametrize("name", APART)
@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up: what is not refused would be launched")
def test_tensors_that_lie_apart_pass_the_check(name):
    """They get as far as the look for a device."""
    assert clip(*APART[name]) not in (0, N.ERR_BAD_ARG)
    assert clip(*APART[name][::-1]) not in (0, N.ERR_BAD_ARG)
