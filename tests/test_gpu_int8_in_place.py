"""The 8-bit integer operators onto their own inputs."""

import pytest
import torch

import int8_reference as ref
import llmoop_b200 as nb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lanes,n,k", [(1, 4096, 4096), (4, 4096, 4096), (8, 2048, 2048), (5, 3000, 3008), (3, 700, 4096), (40, 1024, 1024), (300, 512, 512)])
@pytest.mark.parametrize("form", ["bf16", "residual", "f32", "pair"])
def test_outputs_over_the_inputs(lanes, n, k, form):
    """y at x, and, where it is smaller or larger, over a part of it: what every multiprocessor reads while the first of them write."""
    g = ref.generator(lanes + n)
    w, scale = ref.weights(g, n, k)
    up, up_scale = ref.weights(g, n, k)
    width = 2 if form == "f32" else 1
    memory = torch.empty(lanes * max(k, width * n) + 64, dtype=torch.bfloat16, device="cuda")
    library = nb.library()
    buffer = ref.scratch(library.nerve_b200_op_linear_int8_scratch_bytes(lanes, k))[0]
    for offset in (0, 32):
        for _ in range(10):
            x = ref.activations(g, lanes, k)
            if form == "pair":
                want = ref.pair(x, w, scale, up, up_scale)
            else:
                want = ref.linear(x, w, scale, x[:, :n].contiguous() if form == "residual" and n <= k else None, to_f32=form == "f32")
            residual = x[:, :n].contiguous() if form == "residual" and n <= k else None
            inside = memory[: lanes * k].view(lanes, k).copy_(x)
            y = memory[offset : offset + width * lanes * n]
            y = (y.view(torch.float32) if form == "f32" else y).view(lanes, n)
            if form == "pair":
                ref.check(library.nerve_b200_op_linear_int8_silu_pair(*map(ref.pointer, (inside, w, scale, up, up_scale, y, buffer)), lanes, n, k, ref.stream()))
            else:
                ref.linear(inside, w, scale, residual, to_f32=form == "f32", y=y, buffer=buffer)
            assert torch.equal(y, want)


@pytest.mark.parametrize("tokens", [1, 5, 60, 300])
def test_experts_over_their_inputs(tokens):
    g = ref.generator(tokens)
    (gate_up, gate_up_scale), (down, down_scale) = ref.weights(g, 16, 2 * 96, 256), ref.weights(g, 16, 256, 96)
    x = ref.activations(g, tokens, 256)
    ids = torch.rand((tokens, 16), generator=g, device="cuda").argsort(dim=1)[:, :3].to(torch.int32).contiguous()
    weights = torch.rand((tokens, 3), generator=g, device="cuda")
    layer = (gate_up, gate_up_scale * 3, down, down_scale)
    want = ref.experts(x, ids, weights, *layer, x)
    for _ in range(10):
        y = x.clone()
        assert torch.equal(ref.experts(y, ids, weights, *layer, y, y=y), want)


@pytest.mark.parametrize("lanes", [1, 4])
def test_outputs_over_the_inputs_beside_other_work(lanes):
    """Multiprocessors that another stream holds: the call's CTAs start far apart."""
    g = ref.generator(lanes)
    w, scale = ref.weights(g, 4096, 4096)
    other, background = torch.randn((4096, 4096), generator=g, device="cuda").to(torch.bfloat16), torch.cuda.Stream()
    x = [ref.activations(g, lanes, 4096) for _ in range(20)]
    want = [ref.linear(one, w, scale) for one in x]
    buffer = ref.scratch(nb.library().nerve_b200_op_linear_int8_scratch_bytes(lanes, 4096))[0]
    torch.cuda.synchronize()
    with torch.cuda.stream(background):
        for _ in range(40):
            torch.mm(other, other)
    got = [ref.linear(one, w, scale, y=one, buffer=buffer) for one in x]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
