"""The Llama layer on drafted tokens (reef_b200/csrc/verify.cpp) under tensor
parallelism, its host logic on the CPU: threads as ranks over the stand-ins of
test_comm_host.py, kernels that write all they are given, AddressSanitizer.

At world 2, 4 and 8 the all-reduce plan runs, every rank issuing the same
collectives in the same order, in a workspace of the size asked for; a layer of the
all-gather plan is refused.  Needs g++ and the CUDA and NCCL headers; skipped
without them.
"""
import os

from reef_b200 import build
from tests.test_comm_host import HERE, _build_and_run


def test_verify_under_tensor_parallelism(tmp_path):
    passed = _build_and_run(tmp_path, "verify_host_test", [
        os.path.join(build.CSRC, "layer.cpp"), os.path.join(build.CSRC, "verify.cpp"),
        os.path.join(build.CSRC, "comm.cpp"), os.path.join(HERE, "host", "fake_ops.cpp"),
        os.path.join(HERE, "host", "verify_host_test.cpp")], sanitize=True)
    assert passed == {"verify world 2", "verify world 4", "verify world 8", "verify alone"}
