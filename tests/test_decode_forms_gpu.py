"""Forms of the decoding step's operators that a program may use and that no other file here runs: layouts, gradients, extremes."""
import pytest

from test_decode_tokens_gpu import TYPES, check_rotation

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def decode():
    from fbgemm_amd import decode as d
    return d


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 2, 33])
def test_rotation_of_heads_whose_parts_are_side_by_side(decode, tokens, dtype, interleaved):
    """A projection [tokens, heads, 3, dim], turned in place, and results put into such a buffer."""
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens)
    x = torch.randn((tokens, 8, 3, 64), device="cuda", generator=g).to(dtype)
    query, key, value = x.unbind(2)
    positions, f = torch.arange(tokens, device="cuda") * 5, decode.rotary_frequencies(64)
    want = check_rotation(decode, query, key, positions, f, interleaved=interleaved)
    held = value.clone()
    places = torch.zeros_like(x)
    got = decode.rotate_positions(query, key, positions, f, interleaved=interleaved, out=(places[:, :, 0], places[:, :, 2]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and (places[:, :, 1] == 0).all()
    decode.rotate_positions(query, key, positions, f, interleaved=interleaved, out=(query, key))
    assert torch.equal(query, want[0]) and torch.equal(key, want[1]) and torch.equal(value, held)
