"""The 8-bit integer linears and experts and the router against 64 bits, within bounds that follow from their roundings."""

import ctypes
import math

import numpy as np
import pytest
import torch

import llmoop_b200 as nb

import int8_reference as ref

pytestmark = pytest.mark.gpu

SHAPES = [  # lanes, n, k: one lane to several tiles of 256, ragged rows and tails of K, more and fewer tiles than multiprocessors
    (1, 8, 16), (1, 1, 128), (2, 7, 32), (3, 129, 112), (8, 272, 256), (9, 96, 400), (16, 130, 1024), (17, 1031, 2032), (37, 256, 144), (64, 40, 4096), (129, 300, 512),
    (255, 64, 128), (256, 128, 128), (257, 257, 272), (300, 1030, 640), (1025, 72, 96), (1, 4096, 4096), (4, 20000, 128), (5, 1024, 14336), (520, 4096, 2048),
    (8, 20000, 2176), (16, 200, 16), (33, 20000, 272), (65, 9500, 400), (113, 4096, 1040), (128, 257, 5008), (127, 19000, 128),
]


@pytest.mark.parametrize("lanes,n,k", SHAPES)
@pytest.mark.parametrize("form", ["bf16", "residual", "f32"])
def test_linear(lanes, n, k, form):
    g = ref.generator(lanes * 7 + n * 3 + k)
    x, (w, scale) = ref.activations(g, lanes, k), ref.weights(g, n, k)
    residual = ref.activations(g, lanes, n) if form == "residual" else None
    y = ref.linear(x, w, scale, residual, to_f32=form == "f32")
    want = ref.product(x, w, scale)
    error = want.abs() * ref.PRODUCT
    if residual is not None:
        want = want + residual.double()
        error = error + want.abs() * ref.F32
    ref.assert_close(y, want, error)


@pytest.mark.parametrize("lanes,n,k", SHAPES)
def test_pair(lanes, n, k):
    g = ref.generator(lanes + n * 5 + k * 11)
    x, (gate, gate_scale), (up, up_scale) = ref.activations(g, lanes, k), ref.weights(g, n, k), ref.weights(g, n, k)
    gate_scale = gate_scale * 3
    y = ref.pair(x, gate, gate_scale, up, up_scale)
    want, relative = ref.silu_pair(ref.product(x, gate, gate_scale), ref.product(x, up, up_scale))
    ref.assert_close(y, want, want.abs() * relative)


@pytest.mark.parametrize("lanes,n,k", [(9, 24, 28672), (33, 405, 18704), (100, 1000, 16400), (128, 3, 4096), (129, 24, 9008), (143, 405, 18704), (200, 9, 20000),
                                       (300, 64, 131072), (600, 130, 16384), (1030, 1000, 20016)])
def test_few_tiles_of_many_columns(lanes, n, k):
    """Sums that several blocks add up: those of a lane alone, in whatever order they come, call after call in one buffer."""
    g = ref.generator(lanes + n)
    x, (w, scale), (up, up_scale) = ref.activations(g, lanes, k), ref.weights(g, n, k), ref.weights(g, n, k)
    residual = ref.activations(g, lanes, n)
    buffer, intact = ref.scratch(nb.library().nerve_b200_op_linear_int8_scratch_bytes(lanes, k))
    y, z, plus = ref.linear(x, w, scale, to_f32=True, buffer=buffer), ref.pair(x, w, scale, up, up_scale, buffer=buffer), ref.linear(x, w, scale, residual, buffer=buffer)
    again = [ref.linear(x, w, scale, to_f32=True, buffer=buffer) for _ in range(20)]
    assert intact() and all(torch.equal(y, other) for other in again)
    assert torch.equal(plus, (y + residual.float()).to(torch.bfloat16))
    want = ref.product(x, w, scale)
    ref.assert_close(y, want, want.abs() * ref.PRODUCT)
    for lane in (0, lanes // 2, lanes - 1):
        assert torch.equal(ref.linear(x[lane : lane + 1], w, scale, to_f32=True)[0], y[lane])
        assert torch.equal(ref.pair(x[lane : lane + 1], w, scale, up, up_scale)[0], z[lane])


@pytest.mark.parametrize("lanes", [20, 200])
def test_few_tiles_of_many_columns_in_a_graph(lanes):
    """Replays on new rows, one of them of zeros and one with a NaN, in a buffer that holds anything before the first call."""
    n, k = 70, 12304
    g = ref.generator(lanes)
    w, scale = ref.weights(g, n, k)
    x, y = ref.activations(g, lanes, k), torch.empty((lanes, n), dtype=torch.bfloat16, device="cuda")
    size = nb.library().nerve_b200_op_linear_int8_scratch_bytes(lanes, k)
    buffer = torch.randint(0, 256, (size,), dtype=torch.uint8, device="cuda")
    ref.linear(x, w, scale, x[:, :n].contiguous(), y=y, buffer=buffer)
    torch.cuda.synchronize()
    residual = ref.activations(g, lanes, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ref.linear(x, w, scale, residual, y=y, buffer=buffer)
        ref.linear(x, w, scale, y, y=y, buffer=buffer)  # onto its own outputs
    for round in range(3):
        x.copy_(ref.activations(g, lanes, k))
        x[round] = 0
        x[lanes - 1 - round, 5] = math.nan
        graph.replay()
        first = ref.linear(x, w, scale, residual)
        want = ref.linear(x, w, scale, first)
        assert torch.equal(y.nan_to_num(7e4), want.nan_to_num(7e4))
        assert bool(y[lanes - 1 - round].isnan().all()) and torch.equal(y[round], residual[round])
        torch.cuda.synchronize()


def test_the_widest_sums_are_exact():
    k = 131072
    x = torch.ones((2, k), device="cuda", dtype=torch.bfloat16)
    x[1] = -1
    w = torch.full((9, k), -128, dtype=torch.int8, device="cuda")
    w[3, 5] = 127
    y = ref.linear(x, w, torch.ones(9, device="cuda"), to_f32=True)
    total = torch.full((9,), -127.0 * 128 * k, dtype=torch.float64, device="cuda")
    total[3] += 127 * 255
    unit = torch.tensor(1 / 127, device="cuda", dtype=torch.float32)
    assert torch.equal(y, torch.stack([total.float() * unit, -total.float() * unit]))


def _whole_numbers(x):
    """What the quantisation makes of the rows of x, seen through an identity of weights."""
    k = x.shape[1]
    y = ref.linear(x, torch.eye(k, device="cuda").to(torch.int8), torch.ones(k, device="cuda"), to_f32=True)
    q, a = ref.quantised(x)
    return y, q.float() * a.float()


@pytest.mark.parametrize("exponent", [-133, -120, -95, -89, -40, 0, 60, 120])
def test_quantisation_meets_every_tie(exponent):
    """Every bf16 significand as the largest of a row, every significand and exponent that does not vanish below it."""
    largest = torch.arange(128, 256, dtype=torch.float64, device="cuda") * 2.0 ** (exponent - 7)
    others = torch.cat([torch.arange(128, 256, dtype=torch.float64, device="cuda") * 2.0 ** (exponent - 7 - down) for down in range(9)])
    others = torch.cat([others, -others])
    x = others.repeat(128, 1).clamp(-largest[:, None], largest[:, None])
    x = torch.cat([x, largest[:, None].repeat(1, 16)], dim=1)
    rounded = x.to(torch.bfloat16)
    y, want = _whole_numbers(rounded)
    assert torch.equal(y, want)


def test_rows_of_zeros_infinities_and_nan():
    g = ref.generator(3)
    x, (w, scale) = ref.activations(g, 7, 256), ref.weights(g, 40, 256)
    clean = ref.linear(x, w, scale)
    x[1] = 0
    x[2, 255] = math.inf
    x[3, 0] = -math.inf
    x[4, 17] = math.nan
    x[5] = -0.0
    residual = ref.activations(g, 7, 40)
    y = ref.linear(x, w, scale)
    assert torch.equal(y[[0, 6]], clean[[0, 6]])
    assert bool((y[[1, 5]] == 0).all()) and bool(y[2:5].isnan().all())
    assert torch.equal(ref.linear(x, w, scale, residual)[1], residual[1])
    z = ref.pair(x, w, scale, w, scale)
    assert bool((z[[1, 5]] == 0).all()) and bool(z[2:5].isnan().all()) and not bool(z[[0, 6]].isnan().any())


@pytest.mark.parametrize("lanes", [1, 5, 40, 300])
def test_a_lane_does_not_depend_on_its_company(lanes):
    g = ref.generator(lanes)
    x, (w, scale), (up, up_scale) = ref.activations(g, lanes, 1040), ref.weights(g, 520, 1040), ref.weights(g, 520, 1040)
    y, z = ref.linear(x, w, scale, to_f32=True), ref.pair(x, w, scale, up, up_scale)
    for lane in {0, lanes // 2, lanes - 1}:
        assert torch.equal(ref.linear(x[lane : lane + 1], w, scale, to_f32=True)[0], y[lane])
        assert torch.equal(ref.pair(x[lane : lane + 1], w, scale, up, up_scale)[0], z[lane])


def test_unaligned_inputs_and_what_lies_around_the_outputs():
    g = ref.generator(9)
    x, (w, scale), residual = ref.activations(g, 11, 208), ref.weights(g, 37, 208), ref.activations(g, 11, 37)
    want = ref.linear(x, w, scale, residual)
    moved = torch.empty(11 * 208 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(11, 208).copy_(x)
    beside = torch.empty(11 * 37 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(11, 37).copy_(residual)
    around = torch.full((11 * 37 + 2 * 64 + 1,), 5.0, dtype=torch.bfloat16, device="cuda")
    y = around[65 : 65 + 11 * 37].view(11, 37)
    ref.linear(moved, w, scale, beside, y=y)
    assert torch.equal(y, want) and bool((around[:65] == 5).all()) and bool((around[65 + 11 * 37 :] == 5).all())
    ref.linear(x, w, scale, residual, y=residual)  # in place
    assert torch.equal(residual, want)


def test_threads_with_streams_and_scratch_of_their_own():
    import threading

    g = ref.generator(31)
    layer, (w, scale) = _layer(g, 8, 256, 128), ref.weights(g, 700, 256)
    jobs = []
    for tokens in (1, 6, 40, 200):
        x, (ids, weights) = ref.activations(g, tokens, 256), _routes(g, tokens, 2, 8)
        jobs.append((x, ids, weights, ref.linear(x, w, scale), ref.experts(x, ids, weights, *layer)))
    torch.cuda.synchronize()
    failures = []

    def work(x, ids, weights, want, want_experts):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                outs = [(ref.linear(x, w, scale), ref.experts(x, ids, weights, *layer)) for _ in range(20)]
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, want) and torch.equal(b, want_experts) for a, b in outs)
        except BaseException as error:
            failures.append(error)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures


FIRST_CALL = """
import sys
sys.path[:0] = [".", "tests"]
import torch, int8_reference as ref, llmoop_b200 as nb
library = nb.library()
g = ref.generator(1)
w, scale = ref.weights(g, 300, 256)
for lanes in (3, 50, 400):
    x, y = ref.activations(g, lanes, 256), torch.zeros((lanes, 300), dtype=torch.bfloat16, device="cuda")
    buffer = ref.scratch(library.nerve_b200_op_linear_int8_scratch_bytes(lanes, 256))[0]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # the process's first call
        status = library.nerve_b200_op_linear_int8(*map(ref.pointer, (x, w, scale, y, None, buffer)), lanes, 300, 256, 0, ref.stream())
        assert status == 0, library.nerve_b200_last_error()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ref.linear(x, w, scale)) and bool(y.abs().max() > 0)
print("first call ok")
"""


def test_a_process_may_capture_its_first_call():
    import subprocess
    import sys
    from pathlib import Path

    result = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert result.returncode == 0 and "first call ok" in result.stdout, result.stderr[-2000:]


def test_calls_in_a_row_with_one_scratch_buffer():
    """Kernels of a call start while the ones in front drain: none may touch what an earlier call still reads."""
    g = ref.generator(5)
    xs = [ref.activations(g, 24, 2048) for _ in range(6)]
    (w, scale), (up, up_scale) = ref.weights(g, 2048, 2048), ref.weights(g, 2048, 2048)
    buffer, intact = ref.scratch(nb.library().nerve_b200_op_linear_int8_scratch_bytes(24, 2048))
    want = [(ref.linear(x, w, scale), ref.pair(x, w, scale, up, up_scale)) for x in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [(ref.linear(x, w, scale, buffer=buffer), ref.pair(x, w, scale, up, up_scale, buffer=buffer)) for x in xs]
        assert all(torch.equal(a, b) and torch.equal(c, d) for (a, c), (b, d) in zip(got, want))
    # each call's output is the next one's input
    chain, steps = xs[0], [xs[0]]
    for _ in range(8):
        steps.append(ref.linear(steps[-1], w, scale))
        torch.cuda.synchronize()
    for _ in range(8):
        chain = ref.linear(chain, w, scale, buffer=buffer)
    assert torch.equal(chain, steps[-1]) and intact()


# ---- the router


def _route_reference(logits, bias, r):
    logits = logits.double().cpu().numpy()
    tokens, count = logits.shape
    ids, weights = np.full((tokens, r.top_k), -1, dtype=np.int32), np.zeros((tokens, r.top_k))
    size = count // r.groups
    for token, row in enumerate(logits):
        able = np.flatnonzero(row > -np.inf)
        score = np.zeros(count)
        if r.sigmoid:
            with np.errstate(over="ignore"):
                score[able] = 1 / (1 + np.exp(-row[able]))
        elif len(able):
            top = row[able].max()
            terms = np.array([1.0 if value == top else math.exp(value - top) for value in row[able]])
            score[able] = terms / math.fsum(terms)
        choice = score + (0.0 if bias is None else bias.double().cpu().numpy())
        able = able[choice[able] > -np.inf]
        if r.groups > 1:
            rank = {}
            for group in {int(e) // size for e in able}:
                members = sorted((choice[e] for e in able if e // size == group), reverse=True)
                rank[group] = sum(members[: r.group_scores])
            kept = sorted(rank, key=lambda group: (-rank[group], group))[: r.chosen_groups]
            able = np.array([e for e in able if e // size in kept], dtype=int)
        order = sorted(able, key=lambda e: (-choice[e], e))[: r.top_k]
        ids[token, : len(order)] = order
        chosen = score[order] if len(order) else np.zeros(0)
        if r.renormalise and len(order):
            total = math.fsum(chosen)
            chosen = chosen / total if total > 0 else chosen * 0
        weights[token, : len(order)] = chosen * float(np.float32(r.scale))
    return torch.from_numpy(ids).cuda(), torch.from_numpy(weights).cuda()


ROUTINGS = [
    dict(experts=1, top_k=1), dict(experts=2, top_k=1, sigmoid=True), dict(experts=8, top_k=8), dict(experts=33, top_k=5), dict(experts=60, top_k=6, renormalise=False),
    dict(experts=64, top_k=6, groups=8, chosen_groups=3, group_scores=1), dict(experts=128, top_k=8), dict(experts=160, top_k=6, groups=8, chosen_groups=3, renormalise=False, scale=16.0),
    dict(experts=256, top_k=8, sigmoid=True, groups=8, chosen_groups=4, group_scores=2, scale=2.5), dict(experts=300, top_k=64, sigmoid=True), dict(experts=512, top_k=33),
    dict(experts=1024, top_k=16, groups=32, chosen_groups=9, group_scores=2), dict(experts=561, top_k=9), dict(experts=244, top_k=15, groups=4, chosen_groups=1, group_scores=2),
    dict(experts=200, top_k=15, groups=8, chosen_groups=5), dict(experts=1022, top_k=6, groups=2, chosen_groups=1, group_scores=2), dict(experts=96, top_k=12, groups=3, chosen_groups=1, group_scores=2),
]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("how", ROUTINGS, ids=lambda how: f"{how['experts']}x{how['top_k']}g{how.get('groups', 1)}")
def test_route(how, with_bias, kind):
    g = ref.generator(how["experts"] * 3 + how["top_k"])
    tokens, r = 41, nb.Routing(**how)
    logits = torch.randn((tokens, r.experts), generator=g, device="cuda") * 2
    logits[:10] = (logits[:10] * 2).round() / 2  # many equal ones
    logits.masked_fill_(torch.rand(logits.shape, generator=g, device="cuda") < torch.linspace(0, 1, tokens, device="cuda")[:, None] ** 2, -math.inf)
    logits[11] = -math.inf
    logits[12, 0] = math.nan
    logits[13] = math.nan
    logits[14] *= 50
    logits = logits if kind == "f32" else logits.to(torch.bfloat16)
    bias = torch.randn(r.experts, generator=g, device="cuda") * 0.1 if with_bias else None
    if with_bias and r.experts > 2:
        bias[1], bias[r.experts // 2] = -math.inf, math.nan
    ids, weights = ref.route(logits, bias, r)
    want_ids, want = _route_reference(logits, bias, r)
    assert torch.equal(ids, want_ids)
    # one rounding of the weight, 2^-40 for exponentials and sums in 64 bits
    assert bool(((weights.double() - want).abs() <= want.abs() * (ref.F32 + 2.0 ** -40) + 1e-44).all())


def test_route_infinite_logits_share():
    logits = torch.zeros((2, 40), device="cuda")
    logits[0, [3, 35]] = math.inf
    logits[1] = math.inf
    ids, weights = ref.route(logits, None, nb.Routing(experts=40, top_k=3, renormalise=False))
    assert ids.tolist() == [[3, 35, 0], [0, 1, 2]]
    assert torch.equal(weights[0], torch.tensor([0.5, 0.5, 0.0], device="cuda")) and torch.equal(weights[1], torch.full((3,), 1 / 40, device="cuda"))


def test_route_experts_next_to_one_another():
    """Scores that f32 cannot tell apart, told apart by the bias's order of 1e-9 and by the sigmoid's at large logits."""
    g = ref.generator(1)
    r = nb.Routing(experts=128, top_k=8, sigmoid=True)
    logits = 12 + torch.rand((64, 128), generator=g, device="cuda") * 4
    bias = torch.randn(128, generator=g, device="cuda") * 1e-7
    ids, _ = ref.route(logits, bias, r)
    assert torch.equal(ids, _route_reference(logits, bias, r)[0])


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("middle,spread", [(0.0, 1e-20), (0.0, 1e-13), (17.0, 1e-5), (19.9, 1e-4), (25.0, 1e-4), (40.0, 1.0), (-700.0, 1.0), (-760.0, 1.0)])
def test_route_scores_that_meet_in_64_bits(middle, spread, groups, sigmoid):
    """Logits that differ and whose scores do not, or hardly: the lower number first.  Two implementations of exp in 64 bits, each
    within a step of the truth, may order scores that lie within a few steps of one another either way: 1 / (1 + e) is off by at most
    a step of e's share and two roundings, four steps apart in all.  Where all scores are one number there is one answer."""
    g = ref.generator(2)
    r = nb.Routing(experts=96, top_k=6, sigmoid=sigmoid, groups=groups, chosen_groups=max(1, groups // 2), renormalise=False)
    logits = middle + spread * torch.rand((16, 96), generator=g, device="cuda")
    if not sigmoid and middle < -100:
        logits[:, 5] = 0  # the others' terms run out of exponents
    ids, weights = ref.route(logits, None, r)
    want_ids, want = _route_reference(logits, None, r)
    if spread == 1e-20 or (sigmoid and middle == 40.0) or (sigmoid and middle == -760.0):
        assert torch.equal(ids, want_ids)
    scores = logits.double()
    scores = 1 / (1 + torch.exp(-scores)) if sigmoid else torch.softmax(scores, dim=1)
    chosen, best = scores.gather(1, ids.long()), scores.gather(1, want_ids.long())
    assert bool(((chosen - best).abs() <= 4 * 2.0 ** -52 * best).all())
    assert all(len(set(row)) == 6 for row in ids.tolist())
    assert bool(((weights.double() - want).abs() <= want.abs() * (ref.F32 + 2.0 ** -40) + 1e-44).all())


@pytest.mark.parametrize("apart", [0.0, 1e-9, 1e-7, 2e-6, 2e-5, 2e-4])
@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("count,groups,chosen,group_scores", [(256, 8, 4, 2), (64, 8, 3, 1), (96, 3, 1, 2), (120, 5, 2, 2), (24, 12, 5, 2), (488, 4, 2, 2), (1024, 32, 7, 2), (70, 7, 3, 2)])
def test_route_groups_next_to_one_another(count, groups, chosen, group_scores, sigmoid, apart):
    """Groups of the same logits in other orders, told apart by the bias; some experts and whole groups closed."""
    g = ref.generator(count + groups)
    r, size = nb.Routing(experts=count, top_k=min(6, chosen * (count // groups)), sigmoid=sigmoid, groups=groups, chosen_groups=chosen, group_scores=group_scores, scale=1.5), count // groups
    one = (torch.randn((48, 1, size), generator=g, device="cuda") * 3).repeat(1, groups, 1)
    order = torch.rand((48, groups, size), generator=g, device="cuda").argsort(dim=2)
    logits = one.gather(2, order).view(48, count).contiguous()
    logits[20:30].masked_fill_(torch.rand((10, count), generator=g, device="cuda") < 0.5, -math.inf)
    logits[30:36, : 2 * size] = -math.inf
    logits[36:40] += torch.randn((4, groups, 1), generator=g, device="cuda").repeat(1, 1, size).view(4, count)  # some further away
    bias = torch.randn(count, generator=g, device="cuda") * apart
    for some in (bias, bias + 0.25, bias - 3.0, None):
        ids, weights = ref.route(logits, some, r)
        want_ids, want = _route_reference(logits, some, r)
        assert torch.equal(ids, want_ids)
        assert bool(((weights.double() - want).abs() <= want.abs() * (ref.F32 + 2.0 ** -40) + 1e-44).all())


def test_route_leaves_what_lies_behind():
    logits = torch.randn((5, 16), device="cuda")
    ids, weights = torch.full((6, 4), 9, dtype=torch.int32, device="cuda"), torch.full((6, 4), 9.0, device="cuda")
    ref.route(logits, None, nb.Routing(experts=16, top_k=4), ids, weights)
    assert bool((ids[5] == 9).all()) and bool((weights[5] == 9).all()) and bool((ids[:5] < 16).all())


# ---- the experts


def _layer(g, count, hidden, inter):
    (gate_up, gate_up_scale), (down, down_scale) = ref.weights(g, count, 2 * inter, hidden), ref.weights(g, count, hidden, inter)
    return gate_up, gate_up_scale * 3, down, down_scale


def _routes(g, tokens, top_k, count):
    ids = torch.rand((tokens, count), generator=g, device="cuda").argsort(dim=1)[:, :top_k].to(torch.int32).contiguous()
    return ids, torch.rand((tokens, top_k), generator=g, device="cuda").softmax(dim=1).contiguous()


@pytest.mark.parametrize("tokens,top_k,count,hidden,inter", [
    (1, 1, 1, 16, 16), (1, 2, 4, 64, 32), (3, 3, 8, 80, 48), (1, 8, 128, 2048, 768), (24, 8, 128, 2048, 768), (37, 2, 5, 1008, 336), (131, 6, 60, 256, 144),
    (8, 16, 128, 4096, 256), (7, 12, 16, 1024, 512), (300, 4, 8, 512, 128), (70, 1, 2, 128, 1040), (513, 2, 3, 272, 80), (65, 5, 1024, 64, 32),
    (64, 8, 16, 128, 48), (171, 3, 7, 96, 64), (9, 56, 64, 48, 32), (64, 8, 1024, 64, 48), (12, 1, 1, 4112, 80), (9, 40, 1024, 16400, 16),
])
@pytest.mark.parametrize("with_residual", [False, True])
def test_experts(tokens, top_k, count, hidden, inter, with_residual):
    g = ref.generator(tokens + top_k * 7 + count)
    x, layer, (ids, weights) = ref.activations(g, tokens, hidden), _layer(g, count, hidden, inter), _routes(g, tokens, top_k, count)
    residual = ref.activations(g, tokens, hidden) if with_residual else None
    y = ref.experts(x, ids, weights, *layer, residual)
    ref.assert_close(y, *ref.experts_reference(x, ids, weights, *layer, residual))


@pytest.mark.parametrize("tokens", [300, 100])  # routes grouped by a launch of their own, or by the rows'
def test_experts_empty_doubled_and_crowded_routes(tokens):
    g = ref.generator(8)
    x, layer, (ids, weights) = ref.activations(g, tokens, 256), _layer(g, 6, 256, 64), _routes(g, tokens, 3, 6)
    ids[:40] = 2  # one expert three times
    ids[40:60] = -1  # tokens without a route
    ids[60:70, 1] = 6  # no such expert
    ids[70:75, 0] = -(2 ** 31)
    ids[75:80, 2] = 2 ** 31 - 1
    weights[80:90] = 0
    y = ref.experts(x, ids, weights, *layer)
    want, error = ref.experts_reference(x, ids, weights, *layer)
    ref.assert_close(y, want, error)
    assert bool((y[40:60] == 0).all())
    residual = ref.activations(g, tokens, 256)
    kept = residual.clone()
    ref.experts(x, ids, weights, *layer, residual, y=residual)  # in place
    ref.assert_close(residual, want + kept.double(), error + (want + kept.double()).abs() * ref.F32)
    assert torch.equal(residual[40:60], kept[40:60])
    only = torch.full_like(ids, 4)
    ref.assert_close(ref.experts(x, only, weights, *layer), *ref.experts_reference(x, only, weights, *layer))
    none = torch.full_like(ids, -1)
    assert bool((ref.experts(x, none, weights, *layer) == 0).all())


def test_experts_rows_of_zeros_and_nan():
    g = ref.generator(4)
    x, layer, (ids, weights) = ref.activations(g, 6, 128), _layer(g, 4, 128, 64), _routes(g, 6, 2, 4)
    clean = ref.experts(x, ids, weights, *layer)
    x[1] = 0
    x[3, 100] = math.nan
    y = ref.experts(x, ids, weights, *layer)
    assert bool((y[1] == 0).all()) and bool(y[3].isnan().all()) and torch.equal(y[[0, 2, 4, 5]], clean[[0, 2, 4, 5]])


def test_a_token_does_not_depend_on_its_company_nor_on_the_run():
    g = ref.generator(12)
    x, layer, (ids, weights) = ref.activations(g, 400, 512), _layer(g, 16, 512, 256), _routes(g, 400, 4, 16)
    y = ref.experts(x, ids, weights, *layer)
    assert all(torch.equal(ref.experts(x, ids, weights, *layer), y) for _ in range(5))
    for token in (0, 123, 399):
        some = slice(token, token + 1)
        assert torch.equal(ref.experts(x[some], ids[some], weights[some], *layer)[0], y[token])


def test_experts_unaligned_rows():
    g = ref.generator(13)
    x, layer, (ids, weights) = ref.activations(g, 9, 144), _layer(g, 4, 144, 48), _routes(g, 9, 2, 4)
    residual = ref.activations(g, 9, 144)
    want = ref.experts(x, ids, weights, *layer, residual)
    new = lambda: torch.full((9 * 144 + 2,), 5.0, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    moved, beside, out = (new()[1:-1].view(9, 144) for _ in range(3))
    moved.copy_(x), beside.copy_(residual)
    assert torch.equal(ref.experts(moved, ids, weights, *layer, beside, y=out), want)


# ---- together


def test_a_sparse_expert_layer():
    """Router logits -> routes -> experts, and a shared expert added to them, as a layer runs them: against 64 bits step by step."""
    g = ref.generator(21)
    tokens, hidden, inter, count, top_k = 50, 512, 192, 32, 4
    x, layer = ref.activations(g, tokens, hidden), _layer(g, count, hidden, inter)
    (router, router_scale), bias = ref.weights(g, count, hidden), torch.randn(count, generator=g, device="cuda") * 0.02
    (gate, gate_scale), (up, up_scale), (down, down_scale) = (ref.weights(g, *shape) for shape in ((inter, hidden), (inter, hidden), (hidden, inter)))
    r = nb.Routing(experts=count, top_k=top_k, sigmoid=True, groups=4, chosen_groups=2, group_scores=2, scale=1.5)
    logits = ref.linear(x, router, router_scale, to_f32=True)
    ids, weights = ref.route(logits, bias, r)
    shared = ref.linear(ref.pair(x, gate, gate_scale, up, up_scale), down, down_scale, x)
    y = ref.experts(x, ids, weights, *layer, shared)
    want = ref.product(x, router, router_scale)
    ref.assert_close(logits, want, want.abs() * ref.PRODUCT)
    assert torch.equal(ids, _route_reference(logits, bias, r)[0])
    ref.assert_close(y, *ref.experts_reference(x, ids, weights, *layer, shared))


def test_a_captured_layer_replays_on_new_inputs_beside_another():
    g = ref.generator(22)
    tokens, hidden, inter, count, top_k = 33, 256, 96, 16, 3
    layer, r = _layer(g, count, hidden, inter), nb.Routing(experts=count, top_k=top_k)
    router, router_scale = ref.weights(g, count, hidden)
    router_scale = router_scale * 10
    library = nb.library()

    def run(state):
        ref.linear(state["x"], router, router_scale, to_f32=True, y=state["logits"], buffer=state["linear"])
        ref.route(state["logits"], None, r, state["ids"], state["weights"])
        ref.experts(state["x"], state["ids"], state["weights"], *layer, state["x"], y=state["y"], buffer=state["experts"])

    def state():
        new = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
        return {"x": new(tokens, hidden, dtype=torch.bfloat16), "logits": new(tokens, count), "ids": new(tokens, top_k, dtype=torch.int32), "weights": new(tokens, top_k),
                "y": new(tokens, hidden, dtype=torch.bfloat16), "linear": ref.scratch(library.nerve_b200_op_linear_int8_scratch_bytes(tokens, hidden))[0],
                "experts": ref.scratch(library.nerve_b200_op_experts_int8_scratch_bytes(tokens, top_k, count, hidden, inter))[0]}

    eager, captured = state(), [state(), state()]
    graphs = []
    for one in captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(one)
        graphs.append(graph)
    inputs = [ref.activations(g, tokens, hidden) for _ in range(4)]
    want = []
    for x in inputs:
        eager["x"].copy_(x)
        run(eager)
        want.append(eager["y"].clone())
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for first, second in ((0, 1), (2, 3)):
        for one, graph, stream, which in zip(captured, graphs, streams, (first, second)):
            with torch.cuda.stream(stream):
                one["x"].copy_(inputs[which])
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured[0]["y"], want[first]) and torch.equal(captured[1]["y"], want[second])
