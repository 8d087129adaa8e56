"""What the decoding-step operators promise beside their results, without a GPU."""
import os
import re

import pytest

from test_decode_host import decode  # noqa: F401  (a fixture)

torch = pytest.importorskip("torch")
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fbgemm_amd", "csrc")


def test_results_over_given_tensors_can_be_traced(decode):  # noqa: F811
    x = torch.empty((2, 10), dtype=torch.bfloat16, device="meta")
    assert decode.penalize_logits(x, out=x) is x
    out = torch.empty((2, 20), dtype=torch.bfloat16, device="meta")[:, ::2]
    got = decode.penalize_logits(x, out=out)
    assert got.shape == (2, 10) and got.stride() == out.stride()
    with pytest.raises(RuntimeError):
        decode.penalize_logits(x, out=out[:, :9])


def test_sizes_are_asked_of_the_tensors_device():
    """The workspace's size goes by the current device: every operator makes its tensors' device that one before it calls the library."""
    text = open(os.path.join(CSRC, "torch_op_decode.cpp")).read()
    bodies = re.split(r"\n(?=[a-zA-Z].*\()", text)
    guarded = [b for b in bodies if "OptionalDeviceGuard" in b]
    assert len(guarded) == 4
    for body in guarded:
        calls = [m.start() for m in re.finditer(r"\bfbgemm_amd_\w+\(", body)]
        assert calls and body.index("OptionalDeviceGuard") < min(calls), body[:80]
