"""An array that an AdamW step would write twice is refused at the C entry, before any HIP
call and wherever in the list it comes: two workgroups would move it at once."""
import ctypes
import os
import subprocess
import sys

from cpab.pytorch import _native
from test_sequence_capi import HERE, ROOT, _refused, _Tensor


def test_one_array_twice():
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1", CUDA_VISIBLE_DEVICES="-1")
    paths = [HERE, ROOT, os.path.join(ROOT, "fg-cpab_amd")]
    code = f"import sys; sys.path[:0] = {paths!r}; import test_adamw_capi_twice as t; t.check()"
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


NAMES = ("param", "exp_avg", "exp_avg_sq", "master", "exp_avg_scale", "exp_avg_sq_scale")


def check():
    lib = _native.load_library()

    def step(count, bits, one, two, n=8):
        # `one` and `two`: (tensor, array) that share an address
        arr = (_Tensor * count)()
        for k in range(count):
            for i, name in enumerate(NAMES + ("grad",)):
                setattr(arr[k], name, 4096 * (1 + 8 * k + i))
            arr[k].n = n
        setattr(arr[one[0]], one[1], getattr(arr[two[0]], two[1]))
        return lib.cpab_adamw_step(0, bits, count, ctypes.cast(arr, ctypes.c_void_p), 1, 1e-3, 0.9, 0.999, 1e-8,
                                   0.0, 0, None)

    for count in (2, 42, 48, 49, 700, 5000):
        for bits in (32, 8):
            for one, two in (((0, "param"), (count - 1, "param")), ((count - 1, "exp_avg"), (0, "exp_avg")),
                             ((0, "exp_avg_sq"), (0, "exp_avg")), ((1, "master"), (0, "master")),
                             ((1, "exp_avg"), (count - 1, "param"))):
                _refused(step(count, bits, one, two), "twice")
        _refused(step(count, 8, (0, "exp_avg_scale"), (1, "exp_avg_scale")), "twice")
        _refused(step(count, 8, (0, "exp_avg_sq_scale"), (0, "exp_avg_scale")), "twice")
    # arrays of no values lie anywhere
    assert step(3, 32, (0, "param"), (1, "param"), n=0) == 0
