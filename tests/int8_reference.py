"""The 8-bit integer operators in 64 bits, from their definitions, with a bound on how far an implementation in 32 bits may be off."""

import ctypes

import torch

import llmoop_b200 as nb

F32 = 2.0 ** -24  # half a step of f32, bf16 and so on, relative to the value
BF16 = 2.0 ** -8
PRODUCT = 5 * F32  # a product of an exact sum: the sum as f32, amax / 127, two multiplications, one to spare


def pointer(tensor):
    return ctypes.c_void_p(None if tensor is None else tensor.data_ptr())


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def check(status):
    assert status == 0, nb.library().nerve_b200_last_error().decode()


def scratch(count):
    """That many bytes with a guard behind them, and a function that looks at the guard."""
    buffer = torch.full((count + 256,), 0x5A, dtype=torch.uint8, device="cuda")

    def intact():
        return bool((buffer[count:] == 0x5A).all())

    return buffer, intact


def linear(x, w, scale, residual=None, to_f32=False, y=None, buffer=None):
    lanes, k = x.shape
    n = w.shape[0]
    library = nb.library()
    intact = lambda: True  # noqa: E731
    if buffer is None:
        buffer, intact = scratch(library.nerve_b200_op_linear_int8_scratch_bytes(lanes, k))
    if y is None:
        y = torch.full((lanes, n), 77.0, dtype=torch.float32 if to_f32 else torch.bfloat16, device="cuda")
    check(library.nerve_b200_op_linear_int8(pointer(x), pointer(w), pointer(scale), pointer(y), pointer(residual), pointer(buffer), lanes, n, k, int(to_f32), stream()))
    assert intact()
    return y


def pair(x, gate, gate_scale, up, up_scale, buffer=None):
    lanes, k = x.shape
    n = gate.shape[0]
    library = nb.library()
    intact = lambda: True  # noqa: E731
    if buffer is None:
        buffer, intact = scratch(library.nerve_b200_op_linear_int8_scratch_bytes(lanes, k))
    y = torch.full((lanes, n), 77.0, dtype=torch.bfloat16, device="cuda")
    check(library.nerve_b200_op_linear_int8_silu_pair(pointer(x), pointer(gate), pointer(gate_scale), pointer(up), pointer(up_scale), pointer(y), pointer(buffer), lanes, n, k,
                                                      stream()))
    assert intact()
    return y


def route(logits, bias, routing, ids=None, weights=None):
    tokens = logits.shape[0]
    ids = torch.full((tokens, routing.top_k), 77, dtype=torch.int32, device="cuda") if ids is None else ids
    weights = torch.full((tokens, routing.top_k), 77.0, device="cuda") if weights is None else weights
    check(nb.library().nerve_b200_op_route_experts(pointer(logits), pointer(bias), pointer(ids), pointer(weights), tokens, int(logits.dtype == torch.float32),
                                                   ctypes.byref(routing), stream()))
    return ids, weights


def experts(x, ids, weights, gate_up, gate_up_scale, down, down_scale, residual=None, y=None, buffer=None):
    tokens, hidden = x.shape
    count, _, inter = down.shape
    sizes = (tokens, ids.shape[1], count, hidden, inter)
    library = nb.library()
    intact = lambda: True  # noqa: E731
    if buffer is None:
        buffer, intact = scratch(library.nerve_b200_op_experts_int8_scratch_bytes(*sizes))
    y = torch.full((tokens, hidden), 77.0, dtype=torch.bfloat16, device="cuda") if y is None else y
    tensors = (x, ids, weights, gate_up, gate_up_scale, down, down_scale, y, residual, buffer)
    check(library.nerve_b200_op_experts_int8(*map(pointer, tensors), *sizes, stream()))
    assert intact()
    return y


def quantised(x):
    """(whole numbers, scales) of the rows of x in 64 bits."""
    x = x.double()
    amax = x.abs().amax(dim=1, keepdim=True)
    return torch.where(amax > 0, torch.round(127 * x / amax), 0.0), amax / 127


def product(x, w, scale):
    q, a = quantised(x)
    return q @ w.double().T * a * scale.double()


def silu_pair(gate, up):
    """silu(gate) * up and its relative error where both factors are off by PRODUCT: silu turns an error of the gate into 1 + |gate| of
    it; the exponential is documented as within 2 + 1.173 |gate| steps of 2^-23, the division as within 2, two roundings more."""
    relative = PRODUCT * (2 + gate.abs()) + 2 * F32 * (2 + 1.173 * gate.abs()) + 4 * F32 + 2 * F32
    return gate * torch.sigmoid(gate) * up, relative


def assert_close(y, want, error):
    """error: how far the value may be off before it is rounded to y's type."""
    step = BF16 if y.dtype == torch.bfloat16 else F32
    off = (y.double() - want).abs()
    allowed = error * (1 + step) + want.abs() * step + 1e-36
    worst = float((off / allowed).max())
    assert worst <= 1.0, worst


def experts_reference(x, ids, weights, gate_up, gate_up_scale, down, down_scale, residual=None):
    """(y, error before the last rounding).  A quotient of an intermediate row that lies so near a tie that its error turns it may
    be one step off: as much as that step is worth is added to the error."""
    tokens, hidden = x.shape
    count, _, inter = down.shape
    y = torch.zeros((tokens, hidden), dtype=torch.float64, device=x.device)
    error, magnitude = torch.zeros_like(y), torch.zeros_like(y)
    for expert in range(count):
        token, slot = (ids == expert).nonzero(as_tuple=True)
        if len(token) == 0:
            continue
        both = product(x[token], gate_up[expert], gate_up_scale[expert])
        h, relative = silu_pair(both[:, :inter], both[:, inter:])
        amax, at = h.abs().max(dim=1, keepdim=True)
        off = relative + relative.gather(1, at) + 4 * F32  # of the quotient: its own value's, the largest one's, two operations
        quotient = torch.where(amax > 0, 127 * h / amax, 0.0)
        steps = torch.round(quotient)
        near_tie = ((quotient - torch.floor(quotient) - 0.5).abs() <= quotient.abs() * off).double()
        w, s = down[expert].double(), down_scale[expert].double() * 1.0
        factor = weights[token, slot].double()[:, None] * (amax / 127)
        part = steps @ w.T * s * factor
        slack = near_tie @ w.abs().T * s.abs() * factor.abs() + part.abs() * (PRODUCT + 2 * F32 + relative.gather(1, at))
        y.index_add_(0, token, part)
        error.index_add_(0, token, slack)
        magnitude.index_add_(0, token, part.abs())
    error += magnitude * (ids.shape[1] + 1) * F32  # the sum over the routes
    if residual is not None:
        y = y + residual.double()
        error += y.abs() * F32
    return y, error


def activations(generator, rows, width, device="cuda"):
    x = torch.randn((rows, width), generator=generator, device=device)
    x *= torch.exp(0.5 * torch.randn((1, width), generator=generator, device=device))
    return x.to(torch.bfloat16)


def weights(generator, *shape):
    w = torch.randint(-128, 128, shape, generator=generator, device="cuda", dtype=torch.int32).to(torch.int8)
    return w, torch.rand(shape[:-1], generator=generator, device="cuda") * 0.01 / shape[-1] ** 0.5 + 1e-4


def generator(seed):
    out = torch.Generator(device="cuda")
    out.manual_seed(seed)
    return out
