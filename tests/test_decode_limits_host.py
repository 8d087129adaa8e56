"""What the decoding-step operators promise beside their results, without a GPU."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fbgemm_amd", "csrc")


def test_sizes_are_asked_of_the_tensors_device():
    """The workspace's size goes by the current device: every operator makes its tensors' device that one before it calls the library."""
    text = open(os.path.join(CSRC, "torch_op_decode.cpp")).read()
    bodies = re.split(r"\n(?=[a-zA-Z].*\()", text)
    guarded = [b for b in bodies if "OptionalDeviceGuard" in b]
    assert len(guarded) == 4
    for body in guarded:
        calls = [m.start() for m in re.finditer(r"\bfbgemm_amd_\w+\(", body)]
        assert calls and body.index("OptionalDeviceGuard") < min(calls), body[:80]
