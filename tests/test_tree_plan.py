"""Which attention kernel bkv_attn_tree plans for a call (host side, no GPU): the GPU tests' cases reach all three, in
every format, contiguous and paged, and a plan always covers the call within the workspace that is asked for."""
import ctypes
import random

import pytest

from bonsai_vk_amd import _lib
from tests.test_abi import call, desc
from tests.test_gpu_drafted_edges import FAR, FAR_CONTIGUOUS
from tests.test_gpu_tree import FORMATS, KERNELS


class Plan(ctypes.Structure):
    """struct TreePlan"""
    _fields_ = [(x, ctypes.c_int) for x in ("kind", "nrb", "splits", "share", "spare")] + \
               [(x, ctypes.c_size_t) for x in ("off_ml", "off_part", "total")]


def plan(nh, nkv, kf, vf, paged, pos0, n, base=0):
    f = getattr(_lib.lib(), "_ZN3bkv9plan_treeEiiiiblim")
    f.restype, f.argtypes = Plan, [ctypes.c_int] * 4 + [ctypes.c_bool, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t]
    return f(nh, nkv, kf, vf, paged, pos0, n, base)


@pytest.mark.parametrize("kf,vf", FORMATS)
@pytest.mark.parametrize("paged", [False, True])
def test_the_kernels_that_the_gpu_tests_name(kf, vf, paged):
    kinds = [plan(16, 4, kf, vf, paged, pos0, n).kind for n, pos0 in KERNELS]
    assert kinds == [0, 1, 1, 2]                   # 16, 128, 128, 256 rows a workgroup


@pytest.mark.parametrize("paged", [False, True])
def test_the_kernels_that_the_far_caches_take(paged):
    assert [plan(64, 16, 0, 0, paged, pos0, n).kind for n, pos0 in FAR] == [0, 1, 2]
    assert [plan(64, 64, 0, 0, False, pos0, n).kind for n, pos0 in FAR_CONTIGUOUS] == [0, 1, 2]


def test_plans_cover_the_call():
    r = random.Random(1)
    for _ in range(3000):
        nkv, group = r.choice([1, 2, 3, 4, 5, 8, 16, 40]), r.choice([1, 2, 3, 4, 5, 8, 16, 33])
        n, pos0 = int(2 ** r.uniform(0, 10)), int(2 ** r.uniform(0, 31)) - 1
        kf, vf, paged = r.randint(0, 1), r.randint(0, 1), bool(r.randint(0, 1))
        p = plan(nkv * group, nkv, kf, vf, paged, pos0, n)
        rows, steps = n * group, -(-(pos0 + n) // 32)
        ranges = p.splits * (4 if p.kind == 0 else 1)
        assert p.nrb == -(-rows // (16, 128, 256)[p.kind]) and 1 <= p.splits <= 128
        assert p.share * ranges + p.spare == steps and 0 <= p.spare < ranges
        d = desc(nh=nkv * group, nkv=nkv, k_fmt=kf, v_fmt=vf, n_layers=1, cap=64)
        assert p.total <= call("bkv_workspace_bytes", d, 2, 1)
