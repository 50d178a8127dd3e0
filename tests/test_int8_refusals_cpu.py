"""What the 8-bit integer operators and the router refuse is refused on the host, before anything is launched."""

import ctypes

import pytest

import llmoop_b200 as nb

A = 1 << 20  # a well-aligned address that is never read


def refused(name, *arguments):
    library = nb.library()
    assert getattr(library, name)(*[ctypes.c_void_p(a) if isinstance(a, int) and a >= A else a for a in arguments]) != 0
    message = library.nerve_b200_last_error().decode()
    assert name in message, message
    return message


@pytest.mark.parametrize("change,words", [
    ({"lanes": -1}, "lanes"), ({"lanes": (1 << 20) + 1}, "lanes"), ({"n": 0}, "n is 0"), ({"k": 0}, "k is 0"), ({"k": 24}, "multiple of 16"), ({"k": 131088}, "k is 131088"),
    ({"x": None}, "x is NULL"), ({"w": A + 8}, "w must start on a 16-byte"), ({"scale": A + 2}, "wscale must"), ({"y": A + 1}, "y must"), ({"to_f32": 1, "y": A + 2}, "y must"),
    ({"residual": A + 1}, "residual must"), ({"scratch": None}, "scratch is NULL"), ({"scratch": A + 4}, "scratch must"),
])
def test_linear(change, words):
    a = {"x": A, "w": A, "scale": A, "y": A, "residual": None, "scratch": A, "lanes": 4, "n": 64, "k": 64, "to_f32": 0} | change
    assert words in refused("nerve_b200_op_linear_int8", *(a[key] for key in ("x", "w", "scale", "y", "residual", "scratch", "lanes", "n", "k", "to_f32")), None)


@pytest.mark.parametrize("change,words", [
    ({"lanes": -1}, "lanes"), ({"n": 0}, "n is 0"), ({"k": 8}, "k is 8"), ({"gate": None}, "gate_w is NULL"), ({"up": A + 1}, "up_w must"), ({"up_scale": None}, "up_scale is NULL"),
    ({"y": None}, "y is NULL"), ({"scratch": None}, "scratch"),
])
def test_pair(change, words):
    a = {"x": A, "gate": A, "gate_scale": A, "up": A, "up_scale": A, "y": A, "scratch": A, "lanes": 4, "n": 64, "k": 64} | change
    assert words in refused("nerve_b200_op_linear_int8_silu_pair",
                            *(a[key] for key in ("x", "gate", "gate_scale", "up", "up_scale", "y", "scratch", "lanes", "n", "k")), None)


@pytest.mark.parametrize("change,words", [
    ({"experts": 0}, "experts"), ({"experts": 1025}, "experts"), ({"top_k": 0}, "top_k"), ({"top_k": 65, "experts": 128}, "top_k"), ({"top_k": 9}, "top_k"),
    ({"groups": 3}, "multiple of 3"), ({"groups": 33, "experts": 66}, "groups"), ({"groups": 0}, "groups"), ({"groups": 2, "chosen_groups": 3}, "chosen_groups"),
    ({"groups": 2, "chosen_groups": 1, "top_k": 5}, "top_k"), ({"groups": 8, "chosen_groups": 8, "group_scores": 2}, "group_scores"),
    ({"groups": 4, "chosen_groups": 4, "group_scores": 3}, "group_scores"), ({"tokens": -1}, "tokens"), ({"logits": None}, "logits is NULL"), ({"logits": A + 2}, "logits must"),
    ({"bias": A + 2}, "bias must"), ({"ids": None}, "ids is NULL"), ({"weights": A + 1}, "weights must"),
])
def test_route(change, words):
    routing = nb.Routing(experts=8, top_k=4)
    a = {"logits": A, "bias": None, "ids": A, "weights": A, "tokens": 2, "f32": 1}
    for key, value in change.items():
        if key in a:
            a[key] = value
        else:
            setattr(routing, key, value)
    assert words in refused("nerve_b200_op_route_experts", *(a[key] for key in ("logits", "bias", "ids", "weights", "tokens", "f32")), ctypes.byref(routing), None)


def test_route_without_a_description():
    assert "routing is NULL" in refused("nerve_b200_op_route_experts", A, None, A, A, 1, 1, None, None)


@pytest.mark.parametrize("change,words", [
    ({"tokens": -1}, "tokens"), ({"tokens": (1 << 24) // 2 + 1}, "tokens"), ({"top_k": 0}, "top_k"), ({"top_k": 65}, "top_k"), ({"experts": 0}, "experts"),
    ({"experts": 1025}, "experts"), ({"hidden": 24}, "hidden"), ({"inter": 8}, "inter"), ({"inter": 131088}, "inter"), ({"ids": None}, "ids is NULL"),
    ({"gate_up": A + 8}, "gate_up_w must"), ({"down": None}, "down_w is NULL"), ({"down_scale": A + 1}, "down_scale must"), ({"y": None}, "y is NULL"),
    ({"residual": A + 1}, "residual must"), ({"scratch": A + 8}, "scratch must"),
])
def test_experts(change, words):
    a = {key: A for key in ("x", "ids", "weights", "gate_up", "gate_up_scale", "down", "down_scale", "y", "residual", "scratch")}
    a |= {"tokens": 2, "top_k": 2, "experts": 4, "hidden": 64, "inter": 32} | change
    assert words in refused("nerve_b200_op_experts_int8", *a.values(), None)


def test_nothing_to_do_is_no_error():
    library = nb.library()
    assert library.nerve_b200_op_linear_int8(None, None, None, None, None, None, 0, 8, 16, 0, None) == 0
    assert library.nerve_b200_op_linear_int8_silu_pair(None, None, None, None, None, None, None, 0, 8, 16, None) == 0
    assert library.nerve_b200_op_route_experts(None, None, None, None, 0, 1, ctypes.byref(nb.Routing(experts=8, top_k=2)), None) == 0
    assert library.nerve_b200_op_experts_int8(None, None, None, None, None, None, None, None, None, None, 0, 2, 4, 64, 32, None) == 0


def test_scratch_sizes():
    library = nb.library()
    assert library.nerve_b200_op_linear_int8_scratch_bytes(3, 4096) >= 3 * 4096 + 12
    assert library.nerve_b200_op_linear_int8_scratch_bytes(1 << 20, 131072) > 1 << 37
    assert library.nerve_b200_op_linear_int8_scratch_bytes(3, 4097) == 0
    assert library.nerve_b200_op_linear_int8_scratch_bytes(-1, 4096) == 0
    assert library.nerve_b200_op_experts_int8_scratch_bytes(2048, 8, 128, 2048, 768) >= 2048 * 8 * (4 * 2048 + 768)
    assert library.nerve_b200_op_experts_int8_scratch_bytes(2048, 0, 128, 2048, 768) == 0


def test_scratch_bytes_are_what_the_header_says():
    up = lambda value, step: (value + step - 1) // step * step  # noqa: E731
    library = nb.library()
    for lanes in (1, 2, 8, 9, 16, 17, 100, 128, 129, 1000, 4096):
        for k in (16, 112, 128, 400, 4080, 4096, 14336, 131072):
            rows = up(lanes, 8 if lanes <= 8 else 16) if lanes <= 128 else lanes
            least = up(rows * up(k, 128), 256) + up(4 * lanes, 256)
            split = 2 * 32 * 2 * min(256, up(lanes, 32)) * 128 * 4 + 256 if lanes > 8 and k >= 4096 else 0
            assert library.nerve_b200_op_linear_int8_scratch_bytes(lanes, k) == least + split <= least + 16_800_000, (lanes, k)


FAR = [A * (16 * i + 16) for i in range(10)]  # addresses 16 MB apart


@pytest.mark.parametrize("change,words", [
    ({"residual": FAR[3], "to_f32": 1}, "y and residual overlap"),  # in place, but not of one size
    ({"residual": FAR[3] + 4 * 32 * 2 - 2}, "y and residual overlap"), ({"residual": FAR[3] - 64}, "y and residual overlap"),
    ({"scratch": FAR[0]}, "scratch and x overlap"), ({"scratch": FAR[3] - 512}, "scratch and y overlap"), ({"residual": FAR[5] + 512, "scratch": FAR[5]}, "scratch and residual overlap"),
])
def test_linear_onto_its_inputs(change, words):
    a = {"x": FAR[0], "w": FAR[1], "scale": FAR[2], "y": FAR[3], "residual": None, "scratch": FAR[4], "lanes": 4, "n": 32, "k": 64, "to_f32": 0} | change
    assert words in refused("nerve_b200_op_linear_int8", *(a[key] for key in ("x", "w", "scale", "y", "residual", "scratch", "lanes", "n", "k", "to_f32")), None)


@pytest.mark.parametrize("change,words", [({"scratch": FAR[0] - 16}, "scratch and x overlap"), ({"scratch": FAR[5]}, "scratch and y overlap")])
def test_pair_onto_its_inputs(change, words):
    a = {"x": FAR[0], "gate": FAR[1], "gate_scale": FAR[2], "up": FAR[3], "up_scale": FAR[4], "y": FAR[5], "scratch": FAR[6], "lanes": 4, "n": 64, "k": 64} | change
    assert words in refused("nerve_b200_op_linear_int8_silu_pair", *(a[key] for key in ("x", "gate", "gate_scale", "up", "up_scale", "y", "scratch", "lanes", "n", "k")), None)


@pytest.mark.parametrize("change,words", [
    ({"residual": FAR[7] + 2}, "y and residual overlap"), ({"y": FAR[1]}, "y and ids overlap"), ({"scratch": FAR[0]}, "scratch and x overlap"), ({"scratch": FAR[2]}, "scratch and weights overlap"),
    ({"scratch": FAR[7]}, "scratch and y overlap"), ({"scratch": FAR[1]}, "scratch and ids overlap"),
])
def test_experts_onto_their_inputs(change, words):
    names = ("x", "ids", "weights", "gate_up", "gate_up_scale", "down", "down_scale", "y", "residual", "scratch")
    a = dict(zip(names, FAR)) | {"residual": None} | change
    assert words in refused("nerve_b200_op_experts_int8", *(a[name] for name in names), 4, 2, 8, 64, 32, None)
