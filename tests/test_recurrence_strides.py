"""The recurrence's limit on the distance of samples, at the C entry without a GPU: what
cpab_recurrence_max_stride says is what the entry takes."""
import ctypes
import os
import subprocess
import sys

from cpab.pytorch import _native
from test_sequence_capi import HERE, ROOT, P, _refused


def test_limit_of_the_strides():
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1", CUDA_VISIBLE_DEVICES="-1")
    paths = [HERE, ROOT, os.path.join(ROOT, "fg-cpab_amd")]
    code = f"import sys; sys.path[:0] = {paths!r}; import test_recurrence_strides as t; t.check_strides()"
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def check_strides():
    lib = _native.load_library()

    def forward(dtype, T, C, stride, B=1):
        # refused for its strides, or later for the workspace or y that is not there
        st = (ctypes.c_int64 * 6)(C, stride, C, stride, C, stride)
        return lib.cpab_recurrence_forward(dtype, B, T, C, P, P, P, st, None, None, 0, None, P, None, None,
                                           0, None)
    for dtype, size in ((0, 4), (1, 2)):
        for T, C in ((2, 8), (16, 64), (40, 1024), (100000, 64), (10000, 720000), (300, 1 << 20)):
            most = lib.cpab_recurrence_max_stride(dtype, 1, T, C)
            assert most >= C
            _refused(forward(dtype, T, C, most), "y must not be NULL")
            _refused(forward(dtype, T, C, most + 1), "too far")
        # no more than the samples that there are lie in a tile, and none is 2^31 bytes away
        assert lib.cpab_recurrence_max_stride(dtype, 1, 2, 8) == ((1 << 31) // size - 1 - 8)
    # half the bytes a value, no less far
    assert lib.cpab_recurrence_max_stride(1, 1, 100000, 64) >= 2 * lib.cpab_recurrence_max_stride(0, 1, 100000, 64)
    # over one sample the stride says nothing
    for stride in (0, 1 << 31, 1 << 62):
        _refused(forward(0, 1, 8, stride), "y must not be NULL")
    assert lib.cpab_recurrence_max_stride(7, 1, 1, 1) == 0
    assert lib.cpab_recurrence_max_stride(0, -1, 1, 1) == 0
