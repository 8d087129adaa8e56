"""Gradients of the decoding step's operators without a GPU: which calls are followed, and which refuse to be. On meta tensors."""
import pytest

from test_decode_host import decode  # noqa: F401  (a fixture)

torch = pytest.importorskip("torch")


def tensors(**change):
    m = lambda shape, dtype, grad: torch.empty(shape, dtype=dtype, device="meta", requires_grad=grad)  # noqa: E731
    of = {"query": True, "key": True, "frequencies": False, **change}
    return (m((3, 8, 64), torch.bfloat16, of["query"]), m((3, 2, 64), torch.bfloat16, of["key"]), m((3,), torch.int64, False), m((32,), torch.float64, of["frequencies"]))


def test_a_rotation_has_a_gradient(decode):  # noqa: F811
    q, k, p, f = tensors()
    a, b = decode.rotate_positions(q, k, p, f)
    assert a.requires_grad and b.requires_grad
    (a.float().sum() + b.float().sum()).backward()
    assert q.grad.shape == q.shape and q.grad.dtype == q.dtype and k.grad.shape == k.shape
    q, k, p, f = tensors(key=False)
    a, b = decode.rotate_positions(q, k, p, f)
    assert a.requires_grad
    a.sum().backward()
    assert q.grad.shape == q.shape and k.grad is None
    q, k, p, f = tensors()
    decode.rotate_positions(q, k, p, f)[1].sum().backward()
    assert q.grad is None and k.grad.shape == k.shape
    # a gradient of the gradient
    q, k, p, f = tensors()
    a, _ = decode.rotate_positions(q, k, p, f)
    g, = torch.autograd.grad(a, q, torch.empty_like(a, requires_grad=True), create_graph=True)
    assert g.requires_grad


def test_calls_that_nothing_follows(decode):  # noqa: F811
    q, k, p, f = tensors()
    with torch.no_grad():
        assert not any(x.requires_grad for x in decode.rotate_positions(q, k, p, f))
        decode.rotate_positions(q, k, p, f, out=(torch.empty_like(q), torch.empty_like(k)))
    with torch.inference_mode():
        x = torch.empty_like(q), torch.empty_like(k)
        got = decode.rotate_positions(*x, p, f, out=x)
        assert got[0] is x[0] and decode.rotate_positions(q, k, p, f)[0].is_inference()
    q, k, p, f = tensors(query=False, key=False)
    assert not any(x.requires_grad for x in decode.rotate_positions(q, k, p, f))


def test_a_rotation_into_given_tensors_that_a_graph_follows_is_refused(decode):  # noqa: F811
    q, k, p, f = tensors()
    places = torch.empty_like(q, requires_grad=False), torch.empty_like(k, requires_grad=False)
    for query, key, out in ((q, k.detach(), places), (q.detach(), k, places), (q.detach(), k.detach(), (torch.empty_like(q, requires_grad=True), places[1])),
                            (q * 1, k * 1, (places[0], places[1]))):
        with pytest.raises(RuntimeError, match="no gradient"):
            decode.rotate_positions(query, key, p, f, out=out)
    x = torch.empty((3, 12, 64), dtype=torch.bfloat16, device="meta", requires_grad=True) * 1
    with pytest.raises(RuntimeError, match="no gradient"):
        decode.rotate_positions(x[:, :8], x[:, 8:10], p, f, out=(x[:, :8], x[:, 8:10]))
    q, k, p, f = tensors(frequencies=True)
    with pytest.raises(RuntimeError, match="frequencies"):
        decode.rotate_positions(q, k, p, f)


def test_given_tensors_that_a_graph_holds_are_known_to_have_changed(decode):  # noqa: F811
    q, k, p, f = tensors(query=False, key=False)
    fused = torch.empty((3, 12, 64), dtype=torch.bfloat16, device="meta")
    query, key = fused[:, :8], fused[:, 8:10]
    before = fused._version
    decode.rotate_positions(query, key, p, f, out=(query, key))
    assert fused._version > before and query._version == fused._version
    w = torch.empty((64, 5), dtype=torch.bfloat16, device="meta", requires_grad=True)
    y = q @ w  # which keeps the queries for the weights' gradient
    decode.rotate_positions(q, k, p, f, out=(q, k))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        before = k._version
        decode.rotate_positions(q, k, p, f, out=(q, k))
        assert k._version > before
