"""The norms around a block with gate and residual scale against their 64-bit form."""
import itertools

import pytest
import torch

from oco_b200 import _lib
from tests import opref

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def moe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from oco_b200 import build, moe as m
    build.build()
    return m


def case(seed, rows, width, kind="rms", post=True, gate="row", wide=False, offset=0.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    a = dict(hidden=(n(rows, width) * 2).to(torch.float32 if wide else torch.bfloat16), block=n(rows, width).to(torch.bfloat16),
             pre_w=1 - offset + 0.1 * n(width), pre_b=0.1 * n(width) if kind == "layer" else None,
             post_w=1 - offset + 0.1 * n(width) if post else None, post_b=0.1 * n(width) if post and kind == "layer" else None,
             gate=None if gate == "none" else n(width) if gate == "channel" else n(rows, width).to(torch.bfloat16))
    return a


def run(moe, a, kind, act, offset, rs, bs, eps, hidden_out="new", norm_out="new"):
    ho = {"new": torch.empty_like(a["hidden"]), "same": a["hidden"], None: None}[hidden_out]
    no = {"new": torch.empty(a["hidden"].shape, dtype=torch.bfloat16, device="cuda"), "same": a["block"], None: None}[norm_out]
    moe.block_norm(a["hidden"], a["block"], hidden_out=ho, norm_out=no, pre_weight=a["pre_w"], pre_bias=a["pre_b"], post_weight=a["post_w"],
                   post_bias=a["post_b"], gate=a["gate"], gate_act=act, kind=kind, weight_offset=offset, residual_scale=rs, block_scale=bs, epsilon=eps)
    torch.cuda.synchronize()
    return ho, no


def near(got, want, terms, n):
    """One rounding to the type, and f32 arithmetic before it: statistics are sums of n squares over at most 1024 threads
    and trees (64 steps hold every width here) and a handful of products; 2^-17 of the terms' sizes holds it."""
    bound = HALF[got.dtype] * want.abs() + 2.0 ** -17 * terms
    worst = ((got.double() - want).abs() - bound).max().item()
    assert worst <= 0, worst


def check(moe, a, kind="rms", act="none", offset=0.0, rs=1.0, bs=1.0, eps=1e-5, **outs):
    keep = {k: (v.clone() if v is not None else None) for k, v in a.items()}
    ho, no = run(moe, a, kind, act, offset, rs, bs, eps, **outs)
    h, x = opref.block_norm(keep["hidden"], keep["block"], keep["pre_w"], keep["pre_b"], keep["post_w"], keep["post_b"], keep["gate"], act, kind, offset,
                            rs, bs, eps)
    size = h.abs().amax(1, keepdim=True) + 1
    if ho is not None:
        near(ho, h, size, h.shape[1])
    if no is not None:
        near(no, x, x.abs().amax(1, keepdim=True) + 1, h.shape[1])


@pytest.mark.parametrize("width", [8, 64, 72, 256, 264, 512, 768, 1032, 2048, 2880, 4096, 5000, 8192, 10640, 16384, 20000, 32768])
@pytest.mark.parametrize("rows", [1, 5])
def test_widths(moe, width, rows):
    check(moe, case(width + rows, rows, width))
    check(moe, case(width + rows + 1, rows, width, "layer", wide=True), "layer", "sigmoid")


@pytest.mark.parametrize("kind,post,gate,act,wide", [c for c in itertools.product(["rms", "layer"], [False, True], ["none", "channel", "row"],
                                                                                  ["none", "sigmoid", "tanh"], [False, True])])
def test_forms(moe, kind, post, gate, act, wide):
    check(moe, case(3, 9, 1040, kind, post, gate, wide, 1.0), kind, act, 1.0, 0.7, 0.22)


def test_many_rows(moe):
    check(moe, case(4, 3001, 136), "rms", "tanh")
    check(moe, case(5, 1500, 2688), "rms", "none")


@pytest.mark.parametrize("hidden_out,norm_out", [("same", "new"), ("new", "same"), ("same", "same"), (None, "new"), ("new", None)])
def test_in_place_and_single_outputs(moe, hidden_out, norm_out):
    check(moe, case(6, 21, 2880), hidden_out=hidden_out, norm_out=norm_out)


def test_without_a_block_and_without_weights(moe):
    a = case(7, 5, 512)
    x = torch.empty((5, 512), dtype=torch.bfloat16, device="cuda")
    moe.block_norm(a["hidden"], norm_out=x, residual_scale=0.5)
    near(x, opref.block_norm(a["hidden"], None, residual_scale=0.5)[1], torch.ones((5, 1), device="cuda", dtype=torch.float64) * 5, 512)


def test_gate_rows_are_shared(moe):
    """Six rows in three sequences of two: a gate row each; and one gate row for all."""
    a = case(8, 6, 128)
    for gates in (3, 1, 6):
        a["gate"] = torch.randn((gates, 128), device="cuda")
        b = dict(a, gate=a["gate"].repeat_interleave(6 // gates, 0))
        got, _ = run(moe, a, "rms", "sigmoid", 0.0, 1.0, 1.0, 1e-5)
        want, _ = run(moe, b, "rms", "sigmoid", 0.0, 1.0, 1.0, 1e-5)
        assert torch.equal(got, want)


def test_strided_rows(moe):
    a = case(9, 7, 256)
    wide = {k: torch.zeros((7, 512), dtype=torch.bfloat16, device="cuda") for k in ("hidden", "block", "gate", "ho", "no")}
    for k in ("hidden", "block", "gate"):
        wide[k][:, 128:384] = a[k]
    ho, no = run(moe, a, "rms", "tanh", 0.0, 1.0, 1.0, 1e-5)
    view = {k: v[:, 128:384] for k, v in wide.items()}
    moe.block_norm(view["hidden"], view["block"], hidden_out=view["ho"], norm_out=view["no"], pre_weight=a["pre_w"], post_weight=a["post_w"], gate=view["gate"],
                   gate_act="tanh", epsilon=1e-5)
    assert torch.equal(view["ho"], ho) and torch.equal(view["no"], no)
    assert not wide["ho"][:, :128].any() and not wide["ho"][:, 384:].any() and not wide["no"][:, :128].any()


def test_large_means_and_bad_values(moe):
    """A mean a thousand times the spread: the centred sum keeps the variance. A NaN or infinity stays in its row; zeros stay zeros."""
    a = case(10, 6, 1024, "layer", wide=True, gate="none")
    a["hidden"] += 1000.0
    check(moe, a, "layer")
    a = case(11, 6, 1024)
    a["hidden"][1, 3] = float("nan")
    a["block"][2, 5] = float("inf")
    a["hidden"][4] = 0
    a["block"][4] = 0
    ho, no = run(moe, a, "rms", "none", 0.0, 1.0, 1.0, 1e-5)
    assert no[1].isnan().all() and no[2].isnan().any()
    for r in (0, 3, 4, 5):
        assert no[r].isfinite().all() and ho[r].isfinite().all()
    assert not no[4].any() and not ho[4].any()


def test_no_rows_streams_graphs_and_refusals(moe):
    a = case(12, 8, 256)
    moe.block_norm(a["hidden"][:0], a["block"][:0], hidden_out=a["hidden"][:0])
    want = run(moe, a, "rms", "none", 0.0, 1.0, 1.0, 1e-5)
    ho, no = torch.zeros_like(a["hidden"]), torch.zeros_like(a["hidden"])
    call = lambda: moe.block_norm(a["hidden"], a["block"], hidden_out=ho, norm_out=no, pre_weight=a["pre_w"], post_weight=a["post_w"], gate=a["gate"],  # noqa: E731
                                  epsilon=1e-5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    s.synchronize()
    assert torch.equal(ho, want[0]) and torch.equal(no, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    ho.zero_(), no.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(ho, want[0]) and torch.equal(no, want[1])
    for bad in (dict(norm_out=no.float()), dict(hidden_out=ho[:4]), dict(norm_out=no, kind="mean"), dict(norm_out=no, gate=a["gate"][:3]),
                dict(norm_out=no, pre_bias=a["pre_w"], pre_weight=a["pre_w"]), dict(norm_out=no, epsilon=-1.0), dict(),
                dict(norm_out=no, pre_weight=a["pre_w"].cpu())):
        with pytest.raises(_lib.OcoError):
            moe.block_norm(a["hidden"], a["block"], **bad)
    with pytest.raises(_lib.OcoError):
        moe.block_norm(a["hidden"][:, :100].contiguous(), norm_out=no[:, :100].contiguous())       # 100 is no multiple of 8
    with pytest.raises(_lib.OcoError):
        moe.block_norm(a["hidden"][:, 4:132], norm_out=torch.empty((8, 128), dtype=torch.bfloat16, device="cuda"))   # rows start on 8 bytes


def test_expanded_rows_and_overlaps(moe):
    """An expanded gate is one gate for all rows; expanded rows and outputs that share rows with other inputs are refused."""
    a = case(31, 6, 256, gate="none")
    g = torch.randn((1, 256), device="cuda", generator=torch.Generator("cuda").manual_seed(5)).to(torch.bfloat16)
    outs = []
    for gate in (g, g[0], g.expand(6, 256), g.expand(3, 256)):
        a["gate"] = gate
        outs.append(run(moe, a, "rms", "sigmoid", 0.0, 1.0, 1.0, 1e-5))
    for ho, no in outs[1:]:
        assert torch.equal(ho, outs[0][0]) and torch.equal(no, outs[0][1])
    out = torch.empty_like(a["hidden"])
    one = a["block"][:1].expand(6, 256)
    with pytest.raises(_lib.OcoError, match="overlap"):
        moe.block_norm(a["hidden"], one, norm_out=out)
    with pytest.raises(_lib.OcoError, match="overlap"):
        moe.block_norm(one, norm_out=out)
    with pytest.raises(_lib.OcoError, match="overlap"):
        moe.block_norm(a["hidden"], a["block"], norm_out=a["hidden"])
    with pytest.raises(_lib.OcoError, match="overlap"):
        moe.block_norm(a["hidden"][1:], a["block"][1:], hidden_out=a["hidden"][:5])
    both = torch.cat((a["hidden"], a["block"]), 1)                       # interleaved rows share no element
    ho, no = torch.empty_like(both), None
    moe.block_norm(both[:, :256], both[:, 256:], hidden_out=ho[:, :256], norm_out=ho[:, 256:], epsilon=1e-5)
    a["gate"] = a["post_w"] = a["pre_w"] = None
    want = run(moe, a, "rms", "none", 0.0, 1.0, 1.0, 1e-5)
    assert torch.equal(ho[:, :256], want[0]) and torch.equal(ho[:, 256:], want[1])


@pytest.mark.parametrize("act", ["none", "sigmoid", "tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_a_bad_gate_spoils_its_row(moe, act, dtype, kind):
    """A NaN in the gate reaches its element of the residual rows and all of the row's norm; infinities are the ends of sigmoid and tanh."""
    a = case(32, 5, 520, kind, gate="row", wide=True)
    gate = a["gate"].to(dtype)
    gate[1, 7] = float("nan")
    gate[3, 500] = -float("nan")
    gate[2, 3], gate[2, 4] = float("inf"), -float("inf")
    a["gate"] = gate
    ho, no = run(moe, a, kind, act, 0.0, 1.0, 1.0, 1e-5)
    h, x = opref.block_norm(a["hidden"], a["block"], a["pre_w"], a["pre_b"], a["post_w"], a["post_b"], gate, act, kind)
    assert torch.equal(ho.isnan(), h.isnan()) and torch.equal(no.isnan(), x.isnan()) and ho[1, 7].isnan() and no[3].isnan().all()
    rows = [0, 4] if act == "none" else [0, 2, 4]
    near(ho[rows], h[rows], h[rows].abs().amax(1, keepdim=True) + 1, 520)


def test_sigmoid_gates_far_below_zero(moe):
    """f32 rows that are the gate alone: exponential and quotient (two units of 2^-23 each), their sum and two products (half
    a unit each) are within 2^-20 of the value, down to e^-85, where a cheaper exponential is off by a hundred units."""
    width = 1024
    gate = torch.linspace(-85.0, 10.0, width, device="cuda")
    hidden = torch.zeros((3, width), device="cuda")
    out = torch.empty_like(hidden)
    moe.block_norm(hidden, torch.ones((3, width), dtype=torch.bfloat16, device="cuda"), hidden_out=out, gate=gate, gate_act="sigmoid")
    want = torch.sigmoid(gate.double()).expand(3, width)
    assert ((out.double() - want).abs() <= 2.0 ** -20 * want).all(), ((out.double() - want).abs() / want).max()
