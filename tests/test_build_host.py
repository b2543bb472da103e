"""CPU tests of the build: an object depends on every header that its source
includes, and kernels with counted waits may not have scratch."""

import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-sglang-fork_amd", "csrc")
SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))


def included(name, seen=None):
    seen = set() if seen is None else seen
    for h in re.findall(r'#include "([^"]+)"', open(os.path.join(CSRC, name)).read()):
        if h not in seen and os.path.exists(os.path.join(CSRC, h)):
            seen.add(h)
            included(h, seen)
    return seen


def test_objects_depend_on_their_headers(tmp_path):
    db = subprocess.run(["make", "-pn", f"OBJDIR={tmp_path}", "all"], cwd=CSRC, capture_output=True, text=True).stdout
    for src in SOURCES:
        rules = re.findall(rf"^{re.escape(str(tmp_path))}/{src[:-4]}\.o: (.*\.hip.*)$", db, re.M)
        assert rules, src
        deps = {os.path.basename(d) for rule in rules for d in rule.split()}
        assert src in deps and included(src) <= deps, (src, included(src) - deps)


@pytest.mark.parametrize("obj,kernels", [("gemm.o", ["stream_gemm_kernel", "walk_gemm_kernel"]),
                                         ("mxfp4_gemm.o", ["mxfp4_ring_kernel", "mxfp4_decode_kernel",
                                                           "mxfp4_decode_shared_kernel"])])
def test_scratch_fails_the_build(tmp_path, obj, kernels):
    """A stand-in compiler that writes an object and reports the kernels' scratch."""
    cc = tmp_path / "cc"

    def make(reports):
        lines = "".join(f"echo 'x.h:1:1: remark: Function Name: _ZN3mw8{k}EvT_ [-Rpass-analysis=kernel-resource-usage]' >&2\n"
                        f"echo 'x.h:1:1: remark:     ScratchSize [bytes/lane]: {n} [-Rpass-analysis=kernel-resource-usage]' >&2\n"
                        for k, n in reports)
        cc.write_text("#!/bin/sh\n" + lines + 'while [ "$1" != -o ]; do shift; done\ntouch "$2"\n')
        cc.chmod(0o755)
        out = tmp_path / "obj" / obj
        rc = subprocess.run(["make", f"HIPCC={cc}", f"OBJDIR={tmp_path}/obj", str(out)], cwd=CSRC, capture_output=True).returncode
        left = out.exists()
        if left:
            out.unlink()
        return rc == 0 and left

    assert make([(k, 0) for k in kernels] + [("other_kernel", 16)])
    for bad in kernels:
        assert not make([(k, 16 * (k == bad)) for k in kernels]), bad
    assert not make([("other_kernel", 0)])
