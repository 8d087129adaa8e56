"""Attention's and the logits' comparisons of test_decode_gpu.py once more, by a check that no NaN passes: a difference that is NaN
is not greater than a bound, so there a result of NaN where a number is wanted counts as close."""
import numpy as np
import pytest

import test_decode_gpu
from test_decode_gpu import HALF_ULP, SMALLEST, decode, np64  # noqa: F401  (decode: a fixture)
from test_decode_gpu import (  # noqa: F401  (run here again)
    test_attention_at_the_edges_of_tiles_and_pages, test_attention_beyond_32_bit_offsets, test_attention_leaves_out_blocks_that_are_not_there,
    test_attention_of_dims_between, test_attention_of_lengths_beyond_the_table_and_below_zero, test_attention_of_more_requests_than_a_workgroup_adds_up_at_once,
    test_attention_of_scores_far_apart, test_attention_of_shared_heads, test_attention_over_strided_caches, test_attention_split_over_workers,
    test_attention_with_a_window_a_cap_and_a_scale, test_logits, test_logits_in_place_and_of_strided_rows,
    test_logits_that_are_not_finite_and_rows_that_a_mask_empties, test_logits_with_parts_left_out)

pytestmark = pytest.mark.gpu


def close_and_finite(got, want, off, dtype):
    """test_decode_gpu.close, with a NaN never close to a number."""
    got = np64(got)
    fine = np.isfinite(want)
    assert (got[~fine] == want[~fine]).all()
    got, want, off = got[fine], want[fine], np.broadcast_to(off, fine.shape)[fine]
    near = np.abs(got - want) <= off + HALF_ULP[dtype] * (np.abs(want) + off) + SMALLEST[dtype]
    assert near.all(), (int((~near).sum()), got[~near][:4], want[~near][:4], off[~near][:4])


@pytest.fixture(autouse=True)
def no_nan_passes(monkeypatch):
    monkeypatch.setattr(test_decode_gpu, "close", close_and_finite)


def test_the_check_refuses_nan():
    import torch
    with pytest.raises(AssertionError):
        close_and_finite(torch.tensor([float("nan"), 1.0]), np.ones(2), 0.0, torch.float32)
