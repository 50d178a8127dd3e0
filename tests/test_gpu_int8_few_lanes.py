"""Up to eight lanes through wide matrices, which go to either of the two kernels by the estimates of their plans."""

import pytest
import torch

import int8_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lanes,n,k", [(8, 115672, 2272), (8, 19808, 15840), (1, 20000, 24576), (3, 10520, 70304)])
def test_linear(lanes, n, k):
    g = ref.generator(lanes + n)
    x, (w, scale) = ref.activations(g, lanes, k), ref.weights(g, n, k)
    residual = ref.activations(g, lanes, n)
    y, plus = ref.linear(x, w, scale, to_f32=True), ref.linear(x, w, scale, residual)
    want = ref.product(x, w, scale)
    ref.assert_close(y, want, want.abs() * ref.PRODUCT)
    assert torch.equal(plus, (y + residual.float()).to(torch.bfloat16))
    half = n // 2 + 3  # another plan, the same bits
    assert torch.equal(ref.linear(x, w[:half], scale[:half], to_f32=True), y[:, :half])
    assert torch.equal(ref.linear(x[:1], w, scale, to_f32=True)[0], y[0])


@pytest.mark.parametrize("lanes,n,k", [(8, 10589, 2272), (7, 10061, 2448), (4, 9863, 8304), (6, 10376, 5680)])
def test_pair(lanes, n, k):
    g = ref.generator(lanes + n)
    x, (gate, gate_scale), (up, up_scale) = ref.activations(g, lanes, k), ref.weights(g, n, k), ref.weights(g, n, k)
    gate_scale = gate_scale * 3
    y = ref.pair(x, gate, gate_scale, up, up_scale)
    want, relative = ref.silu_pair(ref.product(x, gate, gate_scale), ref.product(x, up, up_scale))
    ref.assert_close(y, want, want.abs() * relative)
    half = n // 2 + 3
    assert torch.equal(ref.pair(x, gate[:half], gate_scale[:half], up[:half], up_scale[:half]), y[:, :half])
    assert torch.equal(ref.pair(x[:1], gate, gate_scale, up, up_scale)[0], y[0])


@pytest.mark.parametrize("tokens,top_k", [(32, 16), (30, 17), (9, 56), (16, 32), (33, 16)])
def test_experts_of_many_routes_a_token(tokens, top_k):
    """Routes that the rows' quantisation groups itself and those that a launch in front does, at the border between the two."""
    g = ref.generator(tokens * top_k)
    (gate_up, gate_up_scale), (down, down_scale) = ref.weights(g, 64, 2 * 96, 256), ref.weights(g, 64, 256, 96)
    x, layer = ref.activations(g, tokens, 256), (gate_up, gate_up_scale * 3, down, down_scale)
    ids = torch.rand((tokens, 64), generator=g, device="cuda").argsort(dim=1)[:, :top_k].to(torch.int32).contiguous()
    weights = torch.rand((tokens, top_k), generator=g, device="cuda").softmax(dim=1).contiguous()
    ids[3, 2:5] = -1
    ids[5] = 63
    y = ref.experts(x, ids, weights, *layer)
    ref.assert_close(y, *ref.experts_reference(x, ids, weights, *layer))
    for token in (0, 3, 5, tokens - 1):
        some = slice(token, token + 1)
        assert torch.equal(ref.experts(x[some], ids[some], weights[some], *layer)[0], y[token])
