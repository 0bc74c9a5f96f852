"""The gated delta rule's C entries without heads of values, without a GPU: what is refused,
and what is nothing to do, in a child process that sees no GPU."""
import os
import subprocess
import sys

from test_heads_capi import HERE, ODD, P, ROOT, _refused, delta_rule


def test_no_heads():
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1", CUDA_VISIBLE_DEVICES="-1")
    paths = [HERE, ROOT, os.path.join(ROOT, "fg-cpab_amd")]
    code = f"import sys; sys.path[:0] = {paths!r}; import test_heads_capi_no_heads as t; t._check()"
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def _check():
    from cpab.pytorch import _native
    lib = _native.load_library()

    def backward(gq=P, gk=P, **kw):
        args = dict(heads=0, q=None, k=None, v=None, decay=None, beta=None)
        args.update(kw)
        return lib.cpab_delta_rule_backward(delta_rule(**args), None, None, None, gq, gk, None, None, None, None, None, 0, None)
    for kw in (dict(gq=ODD), dict(gk=66)):
        _refused(backward(**kw), "aligned")
    # more values than are counted, of keys that no head reads
    for kw in (dict(B=1 << 30, T=1 << 30), dict(B=1 << 20, T=1 << 15), dict(key_heads=1 << 30)):
        _refused(backward(**kw), "too large")
        _refused(lib.cpab_delta_rule_forward(delta_rule(heads=0, **kw), P, P, None, P, 0, None), "too large")
    # nothing that is there, or nothing that is asked for
    for kw in (dict(B=0), dict(T=0), dict(key_heads=0), dict(gq=None, gk=None)):
        assert backward(**kw) == 0
    # there is something to write, and no GPU
    assert backward() != 0
    assert lib.cpab_delta_rule_forward(delta_rule(heads=0), P, P, None, None, 0, None) == 0
