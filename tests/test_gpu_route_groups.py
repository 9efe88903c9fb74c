"""Routing with groups of experts against the 64-bit definition: ids exact, weights within their 32-bit rounding."""
import numpy as np
import pytest
import torch

from oco_b200 import _lib
from tests import opref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def moe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from oco_b200 import build, moe as m
    build.build()
    return m


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# experts, active, score, groups, top_groups, best, bias, normalize, scale
SHAPES = [
    (8, 2, "softmax", 1, 1, 1, False, True, 1.0),
    (32, 4, "sigmoid", 1, 1, 1, True, False, 2.5),
    (64, 6, "softmax", 8, 3, 1, False, True, 1.0),
    (128, 8, "softmax", 1, 1, 1, False, True, 1.0),
    (160, 6, "sigmoid", 5, 2, 2, True, True, 2.5),
    (256, 8, "sigmoid", 8, 4, 2, True, True, 2.5),
    (270, 9, "softmax", 5, 1, 2, True, True, 1.0),
    (384, 16, "sigmoid", 1, 1, 1, True, True, 1.0),
    (512, 16, "softmax", 32, 31, 2, True, False, 1.0),
    (16, 1, "sigmoid", 16, 1, 2, True, True, 1.0),      # groups of one expert
    (1, 1, "softmax", 1, 1, 1, False, True, 1.0),
    (10, 10, "sigmoid", 2, 2, 1, False, True, 1.0),     # every expert chosen
]


def make(moe, shape, hidden, rows, seed):
    E, K, score, G, TG, best, bias, normalize, scale = shape
    r = moe.RouterPlan.new(hidden, E, K, score=score, groups=G, top_groups=TG, group_best=best, normalize=normalize, scale=scale)
    r.reserve(max(rows, 1))
    g = gen(seed)
    b = torch.randn(E, device="cuda", generator=g) * 0.1 if bias else None
    w = torch.randn((E, hidden), device="cuda", generator=g) * (1.3 / max(hidden, 1) ** 0.5) if hidden else None
    r.bind(w, b)
    return r, w, b, g


def outputs(shape, rows):
    K = shape[1]
    return torch.full((rows, K), -7, dtype=torch.int32, device="cuda"), torch.full((rows, K), -7.0, device="cuda")


def expect(shape, logits, b):
    E, K, score, G, TG, best, _, normalize, scale = shape
    return opref.route(logits.cpu().numpy(), None if b is None else b.double().cpu().numpy(), E, K, score, G, TG, best, normalize, scale)


# a weight is a quotient of scores: exponential, sum and quotient in f32, each within a few units in the last place, and
# the logit's own error through the slope (at most its size times 2^-22); 2^-20 relative holds all of it
REL = 2.0 ** -20


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("rows", [1, 7, 130])
def test_select_matches_the_definition(moe, shape, rows):
    r, _, b, g = make(moe, shape, 0, rows, 1)
    logits = torch.randn((rows, shape[0]), device="cuda", generator=g) * 1.5
    ids, probs = outputs(shape, rows)
    r.select(logits, ids, probs, rows)
    r.poll()
    want, p = expect(shape, logits.double(), b)
    assert np.array_equal(ids.cpu().numpy(), want)
    np.testing.assert_allclose(probs.cpu().numpy(), p, rtol=REL, atol=0)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("hidden,rows", [(32, 3), (96, 65), (2688, 1), (2080, 9), (1024, 200), (4096, 513)])
def test_forward_matches_the_definition(moe, shape, hidden, rows):
    r, w, b, g = make(moe, shape, hidden, rows, 2)
    x = torch.randn((rows, hidden), device="cuda", generator=g).to(torch.bfloat16)
    ids, probs = outputs(shape, rows)
    logits = torch.empty((rows, shape[0]), device="cuda")
    r.forward(x, ids, probs, rows, logits=logits)
    r.poll()
    exact = x.double() @ w.double().t()
    # the product: f32 accumulation of exact products of row and weight; 2^-21 of the sum of the terms' sizes
    assert ((logits.double() - exact).abs() <= 2.0 ** -21 * (x.double().abs() @ w.double().abs().t())).all()
    want, p = expect(shape, exact, b)
    assert np.array_equal(ids.cpu().numpy(), want)
    # the logit's error enters the weight through its slope: at most 2^-21 of the terms' sizes (here below 2^5)
    np.testing.assert_allclose(probs.cpu().numpy(), p, rtol=2.0 ** -16, atol=0)


def test_equal_values_go_to_the_lower_index(moe):
    shape = (256, 8, "sigmoid", 8, 4, 2, False, True, 1.0)
    r, _, _, _ = make(moe, shape, 0, 4, 3)
    logits = torch.zeros((4, 256), device="cuda")
    logits[1, 100:] = 0.5
    logits[2] = torch.arange(256, device="cuda") // 2 * 0.25 - 20      # pairs of equal logits
    logits[3, ::2] = -0.0                                              # the two zeros are equal
    ids, probs = outputs(shape, 4)
    r.select(logits, ids, probs, 4)
    want, p = expect(shape, logits.double(), None)
    assert np.array_equal(ids.cpu().numpy(), want)
    np.testing.assert_allclose(probs.cpu().numpy(), p, rtol=REL)


def test_scores_that_32_bits_cannot_tell_apart(moe):
    """Logits near 20 have sigmoids within 2e-9 of 1: the order is decided in 64 bits."""
    shape = (64, 8, "sigmoid", 4, 2, 2, True, True, 1.0)
    r, _, b, g = make(moe, shape, 0, 50, 4)
    r.bind(None, None)
    logits = 20.0 + torch.rand((50, 64), device="cuda", generator=g)
    ids, probs = outputs(shape, 50)
    r.select(logits, ids, probs, 50)
    want, p = expect(shape, logits.double(), None)
    assert np.array_equal(ids.cpu().numpy(), want)
    np.testing.assert_allclose(probs.cpu().numpy(), p, rtol=REL)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("bias", [False, True])
def test_near_ties_of_the_product_are_decided_in_64_bits(moe, score, bias):
    """Weight rows that differ in their last bits give logits that 32-bit sums cannot order."""
    E, H, rows = 64, 1024, 40
    shape = (E, 8, score, 4, 2, 2, bias, True, 1.0)
    r, w, b, g = make(moe, shape, H, rows, 5)
    w = w[:8].repeat(8, 1)
    w *= 1.0 + (torch.rand((E, H), device="cuda", generator=g) - 0.5) * 2e-7
    if bias:
        b = b[:8].repeat(8)
    r.bind(w, b)
    x = torch.randn((rows, H), device="cuda", generator=g).to(torch.bfloat16)
    ids, probs = outputs(shape, rows)
    r.forward(x, ids, probs, rows)
    want, p = expect(shape, x.double() @ w.double().t(), b)
    assert np.array_equal(ids.cpu().numpy(), want)
    np.testing.assert_allclose(probs.cpu().numpy(), p, rtol=2.0 ** -16)


def test_ids_do_not_depend_on_the_rows_of_the_call(moe):
    shape = (256, 8, "sigmoid", 8, 4, 2, True, True, 2.5)
    r, w, b, g = make(moe, shape, 2048, 400, 6)
    x = torch.randn((400, 2048), device="cuda", generator=g).to(torch.bfloat16)
    ids, probs = outputs(shape, 400)
    r.forward(x, ids, probs, 400)
    for rows in (1, 5, 33, 100):
        i2, p2 = outputs(shape, rows)
        r.forward(x[:rows], i2, p2, rows)
        assert torch.equal(i2, ids[:rows])


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_values_that_are_not_finite(moe, score):
    """A non-finite logit: NaN weights, valid distinct ids, other rows untouched. A bias of -inf keeps an expert out."""
    shape = (32, 4, score, 4, 2, 2, True, True, 1.0)
    r, _, b, g = make(moe, shape, 0, 6, 7)
    b = b.clone()
    b[::2] = -float("inf")
    r.bind(None, b)
    logits = torch.randn((6, 32), device="cuda", generator=g)
    clean = logits.clone()
    logits[1, 5] = float("nan")
    logits[2, 6] = float("inf")
    logits[3, :] = -float("inf")
    logits[4, 1] = -3.0e38
    clean[4, 1] = -3.0e38
    ids, probs = outputs(shape, 6)
    r.select(logits, ids, probs, 6)
    ids, probs = ids.cpu().numpy(), probs.cpu().numpy()
    assert np.isnan(probs[1:4]).all() and np.isfinite(probs[[0, 4, 5]]).all()
    assert all(len(set(row)) == 4 and (row >= 0).all() and (row < 32).all() for row in ids)
    want, p = expect(shape, clean.double(), b)
    assert np.array_equal(ids[[0, 4, 5]], want[[0, 4, 5]])
    np.testing.assert_allclose(probs[[0, 4, 5]], p[[0, 4, 5]], rtol=REL)


def test_rows_of_zeros_and_of_nan(moe):
    shape = (128, 8, "sigmoid", 8, 4, 2, False, True, 1.0)
    r, w, b, g = make(moe, shape, 512, 64, 8)
    x = torch.zeros((64, 512), device="cuda", dtype=torch.bfloat16)
    x[5, 7] = float("nan")
    ids, probs = outputs(shape, 64)
    r.forward(x, ids, probs, 64)
    p = probs.cpu().numpy()
    assert np.isnan(p[5]).all() and np.all(np.delete(p, 5, 0) == 0.125)
    want, _ = expect(shape, torch.zeros((1, 128), dtype=torch.float64), None)
    assert (np.delete(ids.cpu().numpy(), 5, 0) == want).all()


def test_rows_behind_the_last_one_are_left_alone_and_no_rows_are_no_work(moe):
    shape = (64, 6, "softmax", 1, 1, 1, False, True, 1.0)
    r, w, b, g = make(moe, shape, 256, 16, 9)
    x = torch.randn((16, 256), device="cuda", generator=g).to(torch.bfloat16)
    ids, probs = outputs(shape, 16)
    r.forward(x, ids, probs, 0)
    assert r.launch_count() == 0 and (ids == -7).all()
    r.forward(x, ids, probs, 11)
    assert (ids[11:] == -7).all() and (probs[11:] == -7.0).all() and (ids[:11] >= 0).all()
    with pytest.raises(_lib.OcoError, match="rows 17 outside"):
        r.forward(torch.zeros((17, 256), device="cuda", dtype=torch.bfloat16), *outputs(shape, 17), 17)


def test_a_side_stream_and_a_replayed_graph(moe):
    shape = (256, 8, "sigmoid", 8, 4, 2, True, True, 2.5)
    r, w, b, g = make(moe, shape, 1024, 40, 10)
    x = torch.randn((40, 1024), device="cuda", generator=g).to(torch.bfloat16)
    ids, probs = outputs(shape, 40)
    r.forward(x, ids, probs, 40)
    torch.cuda.synchronize()
    i2, p2 = outputs(shape, 40)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        r.forward(x, i2, p2, 40)
    s.synchronize()
    assert torch.equal(ids, i2) and torch.equal(probs, p2)
    xs = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r.forward(xs, i2, p2, 40)
    xs.copy_(x)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(ids, i2) and torch.equal(probs, p2)


def test_refused_tensors(moe):
    shape = (64, 6, "softmax", 1, 1, 1, False, True, 1.0)
    r, w, b, g = make(moe, shape, 256, 4, 11)
    x = torch.zeros((4, 256), device="cuda", dtype=torch.bfloat16)
    ids, probs = outputs(shape, 4)
    for bad in (x.cpu(), x.float(), x[:2], torch.zeros((256, 4), device="cuda", dtype=torch.bfloat16).t()):
        with pytest.raises(_lib.OcoError, match="x"):
            r.forward(bad, ids, probs, 4)
    with pytest.raises(_lib.OcoError, match="ids"):
        r.forward(x, ids.long(), probs, 4)
    shifted = torch.zeros(4 * 256 + 1, device="cuda", dtype=torch.bfloat16)[1:]
    with pytest.raises(_lib.OcoError, match="aligned"):
        r.forward(shifted, ids, probs, 4)


@pytest.mark.parametrize("experts", [3, 40, 100, 200, 511])
@pytest.mark.parametrize("rows", [1, 4, 5, 16, 17, 129])
def test_experts_that_fill_no_tile(moe, experts, rows):
    shape = (experts, min(experts, 7), "softmax", 1, 1, 1, True, True, 1.0)
    r, w, b, g = make(moe, shape, 640, rows, 20 + rows)
    x = torch.randn((rows, 640), device="cuda", generator=g).to(torch.bfloat16)
    ids, probs = outputs(shape, rows)
    for _ in range(2):                                   # the counters of the last arrival are back at zero
        ids.fill_(-7)
        r.forward(x, ids, probs, rows)
        want, p = expect(shape, x.double() @ w.double().t(), b)
        assert np.array_equal(ids.cpu().numpy(), want)
        np.testing.assert_allclose(probs.cpu().numpy(), p, rtol=2.0 ** -16)
    r.poll()


def test_a_bias_that_is_nan_or_leaves_too_few(moe):
    """NaN and -inf biases rank last, in the order of their indexes where nothing else is left."""
    shape = (64, 6, "sigmoid", 1, 1, 1, True, True, 1.0)
    r, _, b, g = make(moe, shape, 0, 9, 30)
    b = torch.full((64,), -float("inf"), device="cuda")
    b[[9, 33, 50]] = 0.0
    r.bind(None, b)
    logits = torch.randn((9, 64), device="cuda", generator=g)
    ids, probs = outputs(shape, 9)
    r.select(logits, ids, probs, 9)
    got = ids.cpu().numpy()
    assert (np.sort(got[:, :3], 1) == [9, 33, 50]).all() and (got[:, 3:] == [0, 1, 2]).all() and np.isfinite(probs.cpu().numpy()).all()
    b[::2] = float("nan")
    b[1::2] = 0.0
    r.bind(None, b)
    r.select(logits, ids, probs, 9)
    assert (ids.cpu().numpy() % 2 == 1).all()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,K,groups,top_groups,best", [(64, 1, 1, 1, 1), (256, 1, 1, 1, 1), (256, 2, 1, 1, 1), (512, 2, 1, 1, 1), (32, 1, 1, 1, 1),
                                                         (64, 1, 4, 1, 1), (256, 2, 8, 2, 1), (512, 1, 16, 1, 1), (270, 1, 5, 1, 1), (256, 1, 8, 1, 2)])
@pytest.mark.parametrize("size", [0.0, 1e-42, 1e-38])
def test_two_equal_values_near_zero(moe, score, E, K, groups, top_groups, best, size):
    """Two logits of the same value at and near zero (+0 and -0 among them), the others below: the lower index comes first."""
    shape = (E, K, score, groups, top_groups, best, False, True, 1.0)
    rows = 96
    r, _, _, g = make(moe, shape, 0, rows, 40)
    at = torch.rand((rows, E), device="cuda", generator=g).topk(2, 1).indices
    logits = torch.full((rows, E), -1.0, device="cuda").scatter_(1, at, size)
    if size == 0.0:
        logits[torch.arange(0, rows, 2, device="cuda"), at[::2, 0]] = -0.0
    ids, probs = outputs(shape, rows)
    r.select(logits, ids, probs, rows)
    want, p = expect(shape, logits.double(), None)
    assert np.array_equal(ids.cpu().numpy(), want)
    np.testing.assert_allclose(probs.cpu().numpy(), p, rtol=REL)


@pytest.mark.parametrize("offset", [0.0, 100.0, -100.0, 300.0, -300.0])
@pytest.mark.parametrize("E,K,groups,top_groups", [(256, 8, 8, 4), (64, 4, 4, 2), (32, 4, 4, 1), (512, 16, 32, 5), (270, 9, 5, 2)])
@pytest.mark.parametrize("normalize", [True, False])
def test_a_common_offset_does_not_choose_the_groups(moe, offset, E, K, groups, top_groups, normalize):
    """Softmax without a bias, groups worth two scores: groups of the same logits in another order, one of each a step or a
    few larger, so that their worths lie within 1e-4 of each other and far logits have few bits for it."""
    shape = (E, K, "softmax", groups, top_groups, 2, False, normalize, 1.0)
    rows, size = 200, E // groups
    r, _, _, g = make(moe, shape, 0, rows, 41)
    base = torch.randn((rows, 1, size), device="cuda", generator=g).expand(rows, groups, size)
    order = torch.rand((rows, groups, size), device="cuda", generator=g).argsort(2)
    logits = torch.gather(base, 2, order) + offset
    steps = torch.randint(0, 9, (rows, groups, 1), device="cuda", generator=g)
    logits = logits + (logits == logits.amax(2, keepdim=True)) * steps * 2.0 ** -20 * max(1.0, abs(offset) / 8)
    logits = logits.reshape(rows, E).contiguous()
    ids, probs = outputs(shape, rows)
    r.select(logits, ids, probs, rows)
    want, p = expect(shape, logits.double(), None)
    assert np.array_equal(ids.cpu().numpy(), want)
    np.testing.assert_allclose(probs.cpu().numpy(), p, rtol=REL)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,K,groups,top_groups", [(64, 4, 1, 1), (256, 16, 1, 1), (512, 8, 1, 1), (256, 8, 8, 2), (32, 4, 4, 2), (270, 9, 5, 1)])
@pytest.mark.parametrize("far", [60.0, 700.0, -760.0, -1500.0])
def test_scores_that_have_run_into_their_ends(moe, score, E, K, groups, top_groups, far):
    """Without a bias the logits are what is ranked: beyond 37 a sigmoid is 1 in 64 bits too, below -745 it is 0, and so is
    a softmax's score that far under the largest. Neighbours a few steps of f32 apart keep the order of their logits."""
    shape = (E, K, score, groups, top_groups, 1, False, False, 1.0)
    rows = 64
    r, _, _, g = make(moe, shape, 0, rows, 42)
    logits = far + torch.randint(0, 40, (rows, E), device="cuda", generator=g) * 2.0 ** -14
    if far < 0:
        logits[:, 7] = 0.0                                             # the softmax's largest, and one expert with a score
    ids, probs = outputs(shape, rows)
    r.select(logits, ids, probs, rows)
    l = logits.double().cpu().numpy()
    worth = l.reshape(rows, groups, -1).max(2)
    kept = np.argsort(-worth, axis=1, kind="stable")[:, :top_groups]
    open_ = np.zeros((rows, groups), bool)
    np.put_along_axis(open_, kept, True, 1)
    want = np.argsort(-np.where(np.repeat(open_, E // groups, 1), l, -np.inf), axis=1, kind="stable")[:, :K]
    assert np.array_equal(ids.cpu().numpy(), want)
    with np.errstate(over="ignore", under="ignore"):
        s = 1.0 / (1.0 + np.exp(-l)) if score == "sigmoid" else np.exp(l - l.max(1, keepdims=True)) / np.exp(l - l.max(1, keepdims=True)).sum(1, keepdims=True)
    np.testing.assert_allclose(probs.cpu().numpy(), np.take_along_axis(s, want, 1), rtol=REL, atol=2.0 ** -126)


@pytest.mark.parametrize("shape", SHAPES[:10], ids=str)
@pytest.mark.parametrize("share", [0.05, 0.5, 0.9])
def test_masked_experts(moe, shape, share):
    """Logits of -inf among finite ones: scores of 0, finite weights, the ids of the definition; rows with one expert left."""
    E, rows = shape[0], 80
    r, _, b, g = make(moe, shape, 0, rows, 43)
    logits = torch.randn((rows, E), device="cuda", generator=g) * 1.5
    gone = torch.rand((rows, E), device="cuda", generator=g) < share
    gone[:10] = True
    gone[torch.arange(rows, device="cuda"), torch.randint(0, E, (rows,), device="cuda", generator=g)] = False
    logits = logits.masked_fill(gone, -float("inf"))
    ids, probs = outputs(shape, rows)
    r.select(logits, ids, probs, rows)
    with np.errstate(over="ignore"):
        want, p = expect(shape, logits.double(), b)
    assert np.array_equal(ids.cpu().numpy(), want)
    np.testing.assert_allclose(probs.cpu().numpy(), p, rtol=REL, atol=0)


def test_masked_experts_of_a_product(moe):
    """A weight row of -inf behind positive rows: the expert is masked, whichever kernel makes the logits."""
    for score, bias in (("sigmoid", True), ("softmax", False)):
        shape = (96, 4, score, 4, 2, 2, bias, True, 1.0)
        r, w, b, g = make(moe, shape, 256, 60, 44)
        w[[5, 40]] = -float("inf")
        w[60, 3] = -float("inf")
        r.bind(w, b)
        x = (torch.rand((60, 256), device="cuda", generator=g) + 0.1).to(torch.bfloat16)
        exact = x.double() @ w.double().t()
        with np.errstate(over="ignore"):
            want, p = expect(shape, exact, b)
        for rows in (3, 60):
            ids, probs = outputs(shape, rows)
            r.forward(x[:rows].contiguous(), ids, probs, rows)
            assert np.array_equal(ids.cpu().numpy(), want[:rows])
            np.testing.assert_allclose(probs.cpu().numpy(), p[:rows], rtol=2.0 ** -16)


@pytest.mark.parametrize("shape", [(512, 8, "sigmoid", 1, 1, 1, True, True, 1.0), (256, 8, "sigmoid", 8, 4, 2, True, True, 2.5), (128, 8, "softmax", 1, 1, 1, False, True, 1.0),
                                   (64, 4, "softmax", 8, 3, 2, False, True, 1.0), (270, 9, "softmax", 5, 2, 2, True, True, 1.0), (160, 6, "sigmoid", 5, 2, 2, False, True, 1.0)],
                         ids=str)
@pytest.mark.parametrize("H,at,size,weight", [(4096, (0, 2050), 4096.0, 1.0), (4096, (5, 4090), 45.0, 0.5), (1024, (3, 40), 2000.0, 1.0), (2080, (64, 2079), 1e6, 0.25),
                                              (256, (17, 18), 512.0, 1.0)])
def test_large_terms_that_cancel(moe, shape, H, at, size, weight):
    """Two large terms of opposite sign in every logit leave their rounding in 32-bit sums: the ids are the definition's all
    the same, at any number of rows."""
    E, rows = shape[0], 200
    r, w, b, g = make(moe, shape, H, rows, 45)
    x = torch.randn((rows, H), device="cuda", generator=g).to(torch.bfloat16)
    for k, sign in zip(at, (1.0, -1.0)):
        x[:, k] = size * sign
        w[:, k] = weight
    r.bind(w, b)
    exact = x.double() @ w.double().t()
    want, p = expect(shape, exact, b)
    logits = torch.empty((rows, E), device="cuda")
    for n in (1, 16, 17, 200):
        ids, probs = outputs(shape, n)
        r.forward(x[:n], ids, probs, n, logits=logits)
        r.poll()
        assert np.array_equal(ids.cpu().numpy(), want[:n]), n
        # logits within what the selection allows for: 45 units of 2^-24 of the norms, and the sums of up to 64 stages
        bound = 2.0 ** -24 * (45 + 2 * 64) * x[:n].double().norm(dim=1, keepdim=True) * w.double().norm(dim=1).max()
        err = (logits[:n].double() - exact[:n]).abs()
        assert (err <= bound).all()
        # a logit's error d changes a weight by at most e^(2d) where a softmax or a sum of sigmoids divides it
        np.testing.assert_allclose(probs.cpu().numpy(), p[:n], rtol=2.0 ** -16 + 3.0 * float(err.max()))


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("xs,ws", [(1e-30, 1.0), (1e20, 1e-20), (1e25, 1e-15), (1e-38, 1e10)])
def test_rows_whose_squares_leave_the_range(moe, rows, xs, ws):
    """Squares of rows below 2^-126 or beyond the range of f32: the error bound of the logits still holds."""
    for shape in ((64, 4, "sigmoid", 1, 1, 1, False, True, 1.0), (64, 4, "softmax", 8, 2, 1, False, True, 1.0)):
        r, w, b, g = make(moe, shape, 512, rows, 46)
        w = w[:16].repeat(4, 1)                                        # near ties that the product cannot tell apart
        w *= 1.0 + (torch.rand((64, 512), device="cuda", generator=g) - 0.5) * 2e-7
        w *= ws
        r.bind(w, None)
        x = (torch.randn((rows, 512), device="cuda", generator=g).to(torch.bfloat16).float() * xs).to(torch.bfloat16)
        x[1] = 0.0
        exact = x.double() @ w.double().t()
        ids, probs = outputs(shape, rows)
        r.forward(x, ids, probs, rows)
        l = exact.cpu().numpy()
        worth = l.reshape(rows, shape[3], -1).max(2)
        kept = np.argsort(-worth, axis=1, kind="stable")[:, :shape[4]]
        open_ = np.zeros((rows, shape[3]), bool)
        np.put_along_axis(open_, kept, True, 1)
        want = np.argsort(-np.where(np.repeat(open_, 64 // shape[3], 1), l, -np.inf), axis=1, kind="stable")[:, :4]
        assert np.array_equal(ids.cpu().numpy(), want)


def test_norm_of_the_weights_follows_a_new_binding(moe):
    """The error bound belongs to the weights that are bound: larger ones after smaller ones."""
    shape = (256, 8, "sigmoid", 8, 4, 2, True, True, 1.0)
    r, w, b, g = make(moe, shape, 1024, 100, 47)
    small = w * 1e-6
    x = torch.randn((100, 1024), device="cuda", generator=g).to(torch.bfloat16)
    x[:, 3], x[:, 700] = 3000.0, -3000.0
    w[:, 3] = w[:, 700] = 1.0
    ids, probs = outputs(shape, 100)
    for weights in (small, w):
        r.bind(weights, b)
        r.forward(x, ids, probs, 100)
        want, _ = expect(shape, x.double() @ weights.double().t(), b)
        assert np.array_equal(ids.cpu().numpy(), want)


@pytest.mark.parametrize("shape", [(512, 16, "softmax", 32, 7, 2, True, True, 1.0), (512, 16, "sigmoid", 1, 1, 1, False, True, 1.0), (384, 9, "softmax", 1, 1, 1, True, True, 1.0),
                                   (256, 8, "sigmoid", 8, 4, 2, True, True, 2.5), (128, 8, "softmax", 4, 2, 2, False, False, 1.0), (64, 6, "sigmoid", 16, 5, 1, False, True, 1.0),
                                   (32, 4, "softmax", 4, 2, 2, True, True, 1.0), (270, 9, "sigmoid", 5, 2, 2, False, True, 1.0)], ids=str)
@pytest.mark.parametrize("copies", ["all", "quarters", "last bits"])
def test_more_open_decisions_than_one(moe, shape, copies):
    """Experts that are copies of one another, or differ in the last bits of their weights: more than a warp's lanes are too
    near, at the border of the groups too. Rows of zeros among them. The ids are the definition's, from the product (rows on
    both sides of its forms) and from logits."""
    E, rows = shape[0], 40
    r, w, b, g = make(moe, shape, 512, rows, 48)
    few = {"all": 1, "quarters": max(1, E // 4), "last bits": max(1, E // 8)}[copies]
    w = w[:few].repeat(-(-E // few), 1)[:E].contiguous()
    if copies == "last bits":
        w *= 1.0 + (torch.rand((E, 512), device="cuda", generator=g) - 0.5) * 2e-7
    if b is not None:
        b = b[:few].repeat(-(-E // few))[:E].contiguous()
    r.bind(w, b)
    # small whole numbers: with weights that are copies the sums are equal in any order; else far apart against 64 bits
    x = torch.randint(-4, 5, (rows, 512), device="cuda", generator=g).to(torch.bfloat16)
    x[3] = x[25] = 0
    exact = x.double() @ w.double().t()
    if copies != "last bits":
        exact = exact[:, :few].repeat(1, -(-E // few))[:, :E]
    want, p = expect(shape, exact, b)
    for n in (5, 40):
        ids, probs = outputs(shape, n)
        r.forward(x[:n].contiguous(), ids, probs, n)
        r.poll()
        assert np.array_equal(ids.cpu().numpy(), want[:n]), n
        np.testing.assert_allclose(probs.cpu().numpy(), p[:n], rtol=2.0 ** -14)
    logits = exact.float()
    want, p = expect(shape, logits.double(), b)
    ids, probs = outputs(shape, rows)
    r.select(logits, ids, probs, rows)
    assert np.array_equal(ids.cpu().numpy(), want)
    # a score is the exponential of l - top, which is rounded by 2^-24 of the logits' spread (up to 30 here: 1.8e-6), and so is
    # the sum that divides it
    np.testing.assert_allclose(probs.cpu().numpy(), p, rtol=REL + 2.0 ** -23 * float(logits.max() - logits.min()))
