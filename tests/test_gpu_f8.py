"""8-bit float products with block scales (dense and routed) against their 64-bit form."""
import numpy as np
import pytest
import torch

from oco_b200 import _lib, synth
from tests import opref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from oco_b200 import build, dense, moe
    build.build()

    class Mods:
        pass
    m = Mods()
    m.moe, m.dense = moe, dense
    return m


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def bf16(g, *shape):
    return torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16)


def projection(lib, up, up_s, x, rows=None, max_rows=None):
    F, H = up.shape
    rows = x.shape[0] if rows is None else rows
    plan = lib.dense.DensePlan(lib.dense.PROJECTION, synth.FMT_F8_E4M3, H, F)
    plan.reserve(max_rows or rows)
    plan.bind(up, up_scale=up_s)
    y = torch.full((x.shape[0], F), 7.0, dtype=torch.bfloat16, device="cuda")
    plan.forward(x, y, rows)
    plan.poll()
    return plan, y


# the result: one rounding to bf16 (2^-8), and sums of exact products: f32 inside a block of 128 and over the blocks.
# 2^-14 of the terms' sizes allows the tensor cores any order and truncation of 128 terms (128 * 2^-23 = 2^-16) and the
# f32 sum of up to 64 blocks' scaled sums
def within(y, want, terms):
    assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * terms).all(), ((y.double() - want).abs() / (terms + 1e-30)).max()


@pytest.mark.parametrize("rows", [1, 2, 8, 15, 16, 17, 33, 64, 100, 128, 129, 257, 600])
@pytest.mark.parametrize("hidden,ffn", [(32, 32), (128, 128), (160, 96), (512, 384), (2880, 320), (1056, 1312)])
def test_projection(lib, rows, hidden, ffn):
    g = gen(rows * 7 + hidden)
    up, up_s = opref.weights(g, (), ffn, hidden)
    x = bf16(g, rows, hidden)
    _, y = projection(lib, up, up_s, x)
    within(y, *opref.product(*opref.quantize(x.double()), up, up_s))


@pytest.mark.parametrize("rows,hidden,ffn", [(1, 4096, 6144), (5, 8192, 512), (40, 4096, 4096), (300, 4096, 2048), (1100, 1024, 4096)])
def test_projection_larger(lib, rows, hidden, ffn):
    g = gen(5)
    up, up_s = opref.weights(g, (), ffn, hidden)
    x = bf16(g, rows, hidden)
    _, y = projection(lib, up, up_s, x)
    within(y, *opref.product(*opref.quantize(x.double()), up, up_s))


@pytest.mark.parametrize("rows", [1, 20, 70, 300])
def test_integers_are_exact(lib, rows):
    """Codes that are small whole numbers and scales of 1: every sum is exact in f32, the result is its bf16 rounding."""
    H, F = 1184, 416
    g = gen(rows)
    x = torch.randint(-8, 9, (rows, H), device="cuda", generator=g).double()
    x[:, ::128] = 448.0                                            # every block's scale is 1
    up = torch.randint(-4, 5, (F, H), device="cuda", generator=g).double()
    up_s = torch.ones((-(-F // 128), -(-H // 128)), device="cuda")
    _, y = projection(lib, up.float().to(torch.float8_e4m3fn), up_s, x.to(torch.bfloat16))
    assert torch.equal(y, (x @ up.t()).to(torch.bfloat16))


def test_rounding_of_rows_halfway_between_codes(lib):
    """Rows whose quotients lie halfway between two codes; the identity as weights shows the codes themselves."""
    H = 128
    rows = 240
    x = torch.zeros((rows, H), dtype=torch.float64)
    tops = torch.arange(128, 248).double()
    for i in range(rows):
        top = tops[i % 120] * 2.0 ** (i % 7 - 3)
        x[i, 0] = top
        mid = torch.tensor([17.0, 19.0, 21.0, 23.0, 25.0, 27.0, 29.0, 31.0]) / 16          # halfway between neighbours of a binade
        x[i, 1:9] = (mid * top / 448 * 64)
        x[i, 9:128] = torch.linspace(-1, 1, 119) * top
    x = x.to(torch.bfloat16).cuda()
    eye = torch.eye(H, device="cuda").to(torch.float8_e4m3fn)
    _, y = projection(lib, eye, torch.ones((1, 1), device="cuda"), x)
    codes, scales = opref.quantize(x.double())
    assert torch.equal(y, (codes.float() * scales.float()).to(torch.bfloat16))


def ffn_near(y, want, extra=0.0):
    """Two more roundings than a projection: activations to e4m3 (the same on both sides but where f32 and f64 lie on
    different sides of a border between codes) and bf16. Of n activations a share of about (error 2^-14) / (step 2^-3)
    = 2^-11 may land on the neighbouring code, off by at most 2^-3: 2^-3 * sqrt(2^-11) < 2^-8 of the result's norm."""
    err = (y.double() - want).norm() / want.norm()
    assert err <= 2.0 ** -8 + 2.0 ** -8 + extra, err


@pytest.mark.parametrize("rows", [1, 3, 16, 40, 129, 400])
@pytest.mark.parametrize("hidden,ffn", [(64, 32), (256, 384), (2048, 768), (416, 2080)])
def test_gated_feed_forward(lib, rows, hidden, ffn):
    g = gen(rows + ffn)
    w = dict(zip(("gate", "gate_s", "up", "up_s", "down", "down_s"),
                 (*opref.weights(g, (), ffn, hidden), *opref.weights(g, (), ffn, hidden), *opref.weights(g, (), hidden, ffn))))
    x = bf16(g, rows, hidden)
    plan = lib.dense.DensePlan(lib.dense.FFN_SILU_GATE, synth.FMT_F8_E4M3, hidden, ffn)
    plan.reserve(rows)
    plan.bind(w["up"], w["gate"], w["down"], up_scale=w["up_s"], gate_scale=w["gate_s"], down_scale=w["down_s"])
    y = torch.empty_like(x)
    plan.forward(x, y, rows)
    plan.poll()
    ffn_near(y, opref.ffn(x.double(), **w))


def expert_layer(lib, seed, H, F, E, K, max_rows):
    g = gen(seed)
    names = ("gate", "up", "down")
    w = {}
    for n in names:
        w[n], w[n + "_s"] = opref.weights(g, (E,), *((H, F) if n == "down" else (F, H)))
    plan = lib.moe.F8ExpertPlan.new(H, F, E, K)
    plan.reserve(max_rows)
    plan.bind(lib.moe.F8Experts(**{k2: w[k1] for n in names for k1, k2 in ((n, n + "_w"), (n + "_s", n + "_s"))}))
    return plan, w, g


def experts_want(w, x, ids, probs, residual):
    out = residual.double().clone()
    E = w["gate"].shape[0]
    for e in range(E):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel():
            y = opref.ffn(x[t].double(), **{n: w[n][e] for n in ("gate", "gate_s", "up", "up_s", "down", "down_s")})
            out.index_add_(0, t, y * probs[t, j].double().unsqueeze(1))
    return out


@pytest.mark.parametrize("H,F,E,K", [(64, 32, 4, 2), (256, 160, 8, 3), (2048, 768, 32, 8), (320, 256, 300, 6), (416, 96, 1, 1), (128, 128, 512, 16)])
@pytest.mark.parametrize("rows", [1, 2, 9, 64, 333])
def test_experts(lib, H, F, E, K, rows):
    plan, w, g = expert_layer(lib, rows + E, H, F, E, K, rows)
    x, res = bf16(g, rows, H), bf16(g, rows, H)
    ids = torch.topk(torch.rand((rows, E), device="cuda", generator=g), K, 1).indices.to(torch.int32)
    ids[torch.rand((rows, K), device="cuda", generator=g) < 0.15] = -1                       # routes of other shards
    probs = torch.rand((rows, K), device="cuda", generator=g)
    out = torch.empty_like(res)
    plan.forward(x, ids, probs, res, rows, out=out)
    plan.poll()
    want = experts_want(w, x, ids, probs, res)
    ffn_near(out, want, 2.0 ** -8)
    keep = (ids < 0).all(1)
    assert torch.equal(out[keep], res[keep])
    again = res.clone()
    plan.forward(x, ids, probs, again, rows)                                                  # in place
    assert torch.equal(again, out)


def test_one_expert_takes_all_and_an_expert_twice(lib):
    plan, w, g = expert_layer(lib, 3, 256, 256, 16, 4, 300)
    x, res = bf16(g, 300, 256), bf16(g, 300, 256)
    probs = torch.rand((300, 4), device="cuda", generator=g)
    for ids in (torch.full((300, 4), 5), torch.tensor([[3, 3, -1, 3]]).repeat(300, 1), torch.full((300, 4), -1), torch.full((300, 4), 16),
                torch.tensor([[0, 15, 2**31 - 1, -2**31]]).repeat(300, 1)):
        ids = ids.to(torch.int32).cuda()
        out = torch.empty_like(res)
        plan.forward(x, ids, probs, res, 300, out=out)
        ffn_near(out, experts_want(w, x, ids, probs, res), 2.0 ** -8)
        if not ((ids >= 0) & (ids < 16)).any():
            assert torch.equal(out, res)


def test_weights_of_absent_routes_are_not_read(lib):
    plan, w, g = expert_layer(lib, 4, 128, 128, 4, 2, 5)
    x, res = bf16(g, 5, 128), bf16(g, 5, 128)
    ids = torch.tensor([[0, -1]] * 5, dtype=torch.int32, device="cuda")
    probs = torch.tensor([[0.5, float("nan")]] * 5, device="cuda")
    out = torch.empty_like(res)
    plan.forward(x, ids, probs, res, 5, out=out)
    assert out.isfinite().all()


def test_rows_of_zeros_and_bad_values_stay_in_their_row(lib):
    plan, w, g = expert_layer(lib, 5, 384, 128, 4, 2, 40)
    x, res = bf16(g, 40, 384), bf16(g, 40, 384)
    ids = torch.topk(torch.rand((40, 4), device="cuda", generator=g), 2, 1).indices.to(torch.int32)
    probs = torch.rand((40, 2), device="cuda", generator=g)
    x[7] = 0
    x[9, 130] = float("nan")
    x[11, 5] = float("inf")
    x[13] = torch.finfo(torch.bfloat16).tiny / 64          # subnormal rows
    x[15] *= 1e38
    out = torch.empty_like(res)
    plan.forward(x, ids, probs, res, 40, out=out)
    assert torch.equal(out[7], res[7])
    assert out[9].isnan().all() and out[11].isnan().all()
    rows = [r for r in range(40) if r not in (9, 11, 15)]
    assert out[rows].isfinite().all()
    want = experts_want(w, x[rows], ids[rows], probs[rows], res[rows])
    ffn_near(out[rows], want, 2.0 ** -8)


def test_a_row_does_not_depend_on_its_neighbours(lib):
    """The same row alone, among few and among many: the sums run in the same order up to the parts of a split contraction."""
    plan, w, g = expert_layer(lib, 6, 512, 256, 8, 2, 500)
    x, res = bf16(g, 500, 512), bf16(g, 500, 512)
    ids = torch.topk(torch.rand((500, 8), device="cuda", generator=g), 2, 1).indices.to(torch.int32)
    probs = torch.rand((500, 2), device="cuda", generator=g)
    out = torch.empty_like(res)
    plan.forward(x, ids, probs, res, 500, out=out)
    for rows in (1, 30, 200):
        part = torch.empty_like(res)
        plan.forward(x, ids, probs, res, rows, out=part)
        ffn_near(part[:rows], out[:rows].double(), 0.0)


def test_rows_behind_the_last_one_are_left_alone(lib):
    g = gen(7)
    up, up_s = opref.weights(g, (), 96, 160)
    x = bf16(g, 50, 160)
    plan, y = projection(lib, up, up_s, x, rows=37, max_rows=64)
    assert (y[37:] == 7.0).all() and not (y[:37] == 7.0).all()
    y.fill_(7.0)
    plan.forward(x, y, 0)
    assert (y == 7.0).all() and plan.launch_count() == 0
    eplan, w, g = expert_layer(lib, 8, 160, 96, 4, 2, 64)
    out = torch.full((50, 160), 7.0, dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros((50, 2), dtype=torch.int32, device="cuda")
    probs = torch.ones((50, 2), device="cuda")
    eplan.forward(x, ids, probs, x, 37, out=out)
    assert (out[37:] == 7.0).all()
    out.fill_(7.0)
    eplan.forward(x, ids, probs, x, 0, out=out)
    assert (out == 7.0).all()


def test_streams_graphs_and_calls_in_a_row(lib):
    plan, w, g = expert_layer(lib, 9, 512, 256, 16, 4, 200)
    x, res = bf16(g, 200, 512), bf16(g, 200, 512)
    ids = torch.topk(torch.rand((200, 16), device="cuda", generator=g), 4, 1).indices.to(torch.int32)
    probs = torch.rand((200, 4), device="cuda", generator=g)
    want = {}
    for rows in (1, 8, 60, 200):
        want[rows] = torch.empty_like(res)
        plan.forward(x, ids, probs, res, rows, out=want[rows])
    torch.cuda.synchronize()
    got = {r: torch.empty_like(res) for r in want}
    for _ in range(3):                                       # back to back, nothing waits between
        for rows in (200, 1, 60, 8):
            plan.forward(x, ids, probs, res, rows, out=got[rows])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for rows in want:
        assert torch.equal(got[rows][:rows], want[rows][:rows])
    with torch.cuda.stream(s):
        plan.forward(x, ids, probs, res, 60, out=got[60])
    s.synchronize()
    assert torch.equal(got[60][:60], want[60][:60])
    graphs = []
    for rows in want:                                        # several graphs over one workspace, replayed in any order
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.forward(x, ids, probs, res, rows, out=got[rows])
        graphs.append((rows, graph))
    for rows, graph in graphs + graphs[::-1]:
        got[rows].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[rows][:rows], want[rows][:rows])


def test_refused_tensors(lib):
    plan, w, g = expert_layer(lib, 10, 128, 128, 4, 2, 8)
    x = bf16(g, 8, 128)
    ids, probs = torch.zeros((8, 2), dtype=torch.int32, device="cuda"), torch.ones((8, 2), device="cuda")
    for args in ((x.float(), ids, probs, x), (x, ids.long(), probs, x), (x, ids, probs.half(), x), (x, ids, probs, x[:4]), (x.cpu(), ids, probs, x)):
        with pytest.raises(_lib.OcoError):
            plan.forward(*args, 8)
    with pytest.raises(_lib.OcoError, match="rows"):
        big = bf16(g, 9, 128)
        plan.forward(big, ids.new_zeros((9, 2)), probs.new_ones((9, 2)), big, 9)
    with pytest.raises(_lib.OcoError, match="scales"):
        plan.bind(lib.moe.F8Experts(w["gate"], w["gate_s"][:, :, :0], w["up"], w["up_s"], w["down"], w["down_s"]))
    shifted = torch.zeros(8 * 128 + 4, dtype=torch.bfloat16, device="cuda")[4:]
    plan2 = lib.dense.DensePlan(lib.dense.PROJECTION, synth.FMT_F8_E4M3, 128, 64)
    plan2.reserve(8)
    with pytest.raises(_lib.OcoError, match="bind"):
        plan2.forward(x, x, 8)
    plan2.bind(np.zeros((64, 128), np.uint8), up_scale=np.ones((1, 1), np.float32))           # host arrays are uploaded
    y = torch.ones((8, 64), dtype=torch.bfloat16, device="cuda")
    plan2.forward(x, y, 8)
    assert not y.any()
    with pytest.raises(_lib.OcoError, match="aligned"):
        plan2.forward(shifted, y, 8)


def test_a_layer_of_the_operators(lib):
    """Norm, routing with groups, experts and the next norm, as a layer runs them, for a prefill batch and a token."""
    H, F, E, K = 512, 256, 64, 6
    plan, w, g = expert_layer(lib, 11, H, F, E, K, 150)
    router = lib.moe.RouterPlan.new(H, E, K, groups=8, top_groups=3, group_best=2, scale=2.5)
    router.reserve(150)
    rw = torch.randn((E, H), device="cuda", generator=g) * 0.05
    rb = torch.randn(E, device="cuda", generator=g) * 0.1
    router.bind(rw, rb)
    pre, post = (1 + 0.1 * torch.randn(H, device="cuda", generator=g) for _ in range(2))
    for rows in (150, 1):
        hidden, block = bf16(g, rows, H), bf16(g, rows, H)
        x, ids, probs = torch.empty_like(hidden), torch.empty((rows, K), dtype=torch.int32, device="cuda"), torch.empty((rows, K), device="cuda")
        zero = torch.zeros_like(hidden)
        h0 = hidden.clone()
        lib.moe.block_norm(hidden, block, hidden_out=hidden, norm_out=x, pre_weight=pre, post_weight=post)
        router.forward(x, ids, probs, rows)
        moe_out = torch.empty_like(hidden)
        plan.forward(x, ids, probs, zero, rows, out=moe_out)
        nxt = torch.empty_like(hidden)
        lib.moe.block_norm(hidden, moe_out, hidden_out=hidden, norm_out=nxt, pre_weight=pre, post_weight=post, residual_scale=0.5)
        plan.poll()
        # the same from the rows the operators handed on: each stage is held to its own rounding
        wid, wp = opref.route((x.double() @ rw.double().t()).cpu().numpy(), rb.double().cpu().numpy(), E, K, "sigmoid", 8, 3, 2, True, 2.5)
        assert np.array_equal(ids.cpu().numpy(), wid)
        ffn_near(moe_out, experts_want(w, x, ids, probs, zero), 2.0 ** -8)
        h1, _ = opref.block_norm(h0, block, pre, None, post)
        h2, n2 = opref.block_norm(h1.to(torch.bfloat16), moe_out, pre, None, post, residual_scale=0.5)
        assert (hidden.double() - h2).norm() <= 2.0 ** -7 * h2.norm() and (nxt.double() - n2).norm() <= 2.0 ** -7 * n2.norm()


@pytest.mark.parametrize("rows,hidden,ffn", [(1, 16384, 64), (4, 10240, 160), (1030, 288, 544), (1300, 512, 96), (2049, 160, 288)])
def test_projection_forms(lib, rows, hidden, ffn):
    """Contractions longer than a CTA rounds by itself; tiles on SM pairs with ragged rows and features."""
    g = gen(rows)
    up, up_s = opref.weights(g, (), ffn, hidden)
    x = bf16(g, rows, hidden)
    _, y = projection(lib, up, up_s, x)
    within(y, *opref.product(*opref.quantize(x.double()), up, up_s))


@pytest.mark.parametrize("rows,hidden,ffn", [(4, 16384, 96), (1100, 320, 160), (1281, 256, 416)])
def test_gated_feed_forward_forms(lib, rows, hidden, ffn):
    g = gen(rows)
    w = dict(zip(("gate", "gate_s", "up", "up_s", "down", "down_s"),
                 (*opref.weights(g, (), ffn, hidden), *opref.weights(g, (), ffn, hidden), *opref.weights(g, (), hidden, ffn))))
    x = bf16(g, rows, hidden)
    plan = lib.dense.DensePlan(lib.dense.FFN_SILU_GATE, synth.FMT_F8_E4M3, hidden, ffn)
    plan.reserve(rows)
    plan.bind(w["up"], w["gate"], w["down"], up_scale=w["up_s"], gate_scale=w["gate_s"], down_scale=w["down_s"])
    y = torch.empty_like(x)
    plan.forward(x, y, rows)
    ffn_near(y, opref.ffn(x.double(), **w))
    plan.forward(x, x, rows)                     # a feed-forward reads its rows before it writes any
    assert torch.equal(x, y)


def test_the_least_and_the_largest_blocks(lib):
    """Blocks whose largest magnitude is near either end of bf16's range take the division that leaves the range never."""
    H, F = 384, 64
    g = gen(77)
    x = bf16(g, 6, H)
    x[0, :128] *= 1e-36
    x[1, 128:256] *= 3e37
    x[2] = 0
    x[2, 300] = 1e-38
    x[3, :] = torch.finfo(torch.bfloat16).max
    up, up_s = opref.weights(g, (), F, H)
    up = (up.float() / 64).to(torch.float8_e4m3fn)
    up_s = up_s * 1e-3
    for rows in (6, 3):
        _, y = projection(lib, up, up_s, x[:rows].contiguous())
        want, terms = opref.product(*opref.quantize(x[:rows].double()), up, up_s)
        # below 2^-126 a scale has fewer bits: the smallest f32 step, 2^-149, on 448 * 448 * 128 terms
        assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * terms + 2.0 ** -149 * 448 * 448 * 128).all()


@pytest.mark.parametrize("rows", [1, 2, 3, 4])
def test_a_few_tokens_with_shared_and_absent_experts(lib, rows):
    plan, w, g = expert_layer(lib, 12, 416, 288, 6, 4, 8)
    x, res = bf16(g, rows, 416), bf16(g, rows, 416)
    probs = torch.rand((rows, 4), device="cuda", generator=g)
    for pattern in ([0, 1, 2, 3], [5, -1, 5, 6], [-1, -1, -1, -1], [-1, 2, -1, 2**31 - 1], [3, 3, 3, 3]):
        ids = torch.tensor([pattern] * rows, dtype=torch.int32, device="cuda").roll(1, 1).contiguous()
        p = probs.clone()
        p[(ids < 0) | (ids >= 6)] = float("nan")                              # never read
        out = torch.empty_like(res)
        plan.forward(x, ids, p, res, rows, out=out)
        plan.poll()
        ffn_near(out, experts_want(w, x, ids, probs, res), 2.0 ** -8)
        if not ((ids >= 0) & (ids < 6)).any():
            assert torch.equal(out, res)


@pytest.mark.parametrize("E,K,rows", [(5, 5, 1000), (130, 8, 700), (512, 16, 300)])
def test_many_routes(lib, E, K, rows):
    """More routes than one CTA orders: every route once, in any order inside its expert, absent ones nowhere."""
    H, F = 64, 64
    plan, w, g = expert_layer(lib, 13, H, F, E, K, rows)
    x, res = bf16(g, rows, H), bf16(g, rows, H)
    ids = torch.randint(-1, E, (rows, K), device="cuda", generator=g).to(torch.int32)
    probs = torch.rand((rows, K), device="cuda", generator=g)
    out = torch.empty_like(res)
    plan.forward(x, ids, probs, res, rows, out=out)
    plan.poll()
    ffn_near(out, experts_want(w, x, ids, probs, res), 2.0 ** -8)


def test_overlap_is_refused(lib):
    g = gen(14)
    up, up_s = opref.weights(g, (), 128, 128)
    x = bf16(g, 8, 128)
    plan, _ = projection(lib, up, up_s, x)
    with pytest.raises(_lib.OcoError, match="overlap"):
        plan.forward(x, x, 8)
    fresh = lib.moe.F8ExpertPlan.new(128, 128, 4, 2)
    with pytest.raises(_lib.OcoError, match="reserve"):
        fresh.forward(x, torch.zeros((8, 2), dtype=torch.int32, device="cuda"), torch.ones((8, 2), device="cuda"), x, 8)


@pytest.mark.parametrize("rows", [3, 24, 300])
def test_activations_near_the_ends_of_f32(lib, rows):
    """Activations of 1e38 and of 1e-38: their scale and quotient stay in range; down scales bring the results back."""
    H = F = 128
    g = gen(rows)
    gate, gate_s = opref.weights(g, (), F, H)
    gate_s = gate_s * 20                                    # silu(gate) is larger than one for a part of the features
    up, up_s = opref.weights(g, (), F, H)
    down, down_s = opref.weights(g, (), H, F)
    x = bf16(g, rows, H)
    for size in (1e35, 1e-35):
        scale = up_s * size
        unit = opref.ffn(x.double(), gate, gate_s, up, scale, down, down_s)
        if size > 1:                                        # up to the largest activation that f32 holds with room for the products' sums
            c, s = opref.quantize(x.double())
            a, _ = opref.product(c, s, gate, gate_s)
            u, _ = opref.product(c, s, up, scale)
            scale = scale * float(2.0 ** torch.floor(torch.log2(2.5e38 / torch.maximum(u.abs().max(), (a * torch.sigmoid(a) * u).abs().max()))))
        plan = lib.dense.DensePlan(lib.dense.FFN_SILU_GATE, synth.FMT_F8_E4M3, H, F)
        plan.reserve(rows)
        back = down_s * float(2.0 ** -torch.floor(torch.log2(unit.abs().max())))
        if size > 1:
            back = back / 2.0 ** 10
        plan.bind(up, gate, down, up_scale=scale, gate_scale=gate_s, down_scale=back)
        y = torch.empty_like(x)
        plan.forward(x, y, rows)
        plan.poll()
        ffn_near(y, opref.ffn(x.double(), gate, gate_s, up, scale, down, back))


def test_a_part_of_the_residual_is_refused(lib):
    plan, w, g = expert_layer(lib, 15, 128, 128, 4, 2, 8)
    buf, x = bf16(g, 9, 128), bf16(g, 8, 128)
    ids, probs = torch.zeros((8, 2), dtype=torch.int32, device="cuda"), torch.ones((8, 2), device="cuda")
    with pytest.raises(_lib.OcoError, match="overlap"):
        plan.forward(x, ids, probs, buf[:8], 8, out=buf[1:])
    want = torch.empty_like(x)
    plan.forward(x, ids, probs, buf[:8], 8, out=want)
    into = x.clone()
    plan.forward(into, ids, probs, buf[:8], 8, out=into)    # onto x, which has been read by then
    assert torch.equal(into, want)


@pytest.mark.parametrize("H,F", [(128, 1024), (416, 1056)])
@pytest.mark.parametrize("rows", [1, 3, 4, 40, 300, 1500])
def test_routes_are_summed_before_they_are_rounded(lib, rows, H, F):
    """Two experts whose results nearly cancel: down codes of opposite sign, but for one of each feature's. What is left is
    about 2 / sqrt(F) of either, and is off by its own rounding, 2^-8, by activations on the other side of a border
    between codes (ffn_near: 2^-8), and by the f32 sums: a block's four MMAs cut off up to 33 addends at 2^-25 of the
    largest and the sum at 2^-23, 4 * 18.5 * 2^-24, its nine blocks add 2 * 9 * 2^-24: below 2^-17 of the terms' sizes.
    Results rounded to bf16 on their way would leave 2^-8 / sqrt(3) * 0.7 * sqrt(2) * sqrt(F) / 2 = 0.037 and more."""
    g = gen(rows + F)
    w = {}
    for n, shape in (("gate", (F, H)), ("up", (F, H)), ("down", (H, F))):
        w[n], w[n + "_s"] = (t.repeat(2, 1, 1) for t in opref.weights(g, (1,), *shape))
    kept = torch.randint(0, F, (H, 1), device="cuda", generator=g)
    w["down"][1] = (w["down"][0].float() * torch.full((H, F), -1.0, device="cuda").scatter_(1, kept, 1.0)).to(torch.float8_e4m3fn)
    plan = lib.moe.F8ExpertPlan.new(H, F, 2, 2)
    plan.reserve(rows)
    plan.bind(lib.moe.F8Experts(w["gate"], w["gate_s"], w["up"], w["up_s"], w["down"], w["down_s"]))
    x, res = bf16(g, rows, H), torch.zeros((rows, H), dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([[0, 1]] * rows, dtype=torch.int32, device="cuda")
    out = torch.empty_like(res)
    plan.forward(x, ids, torch.ones((rows, 2), device="cuda"), res, rows, out=out)
    plan.poll()
    one = {n: w[n][0] for n in w}
    c, s = opref.quantize(x.double())
    gg, uu = opref.product(c, s, one["gate"], one["gate_s"])[0], opref.product(c, s, one["up"], one["up_s"])[0]
    ac, as_ = opref.quantize(gg * torch.sigmoid(gg) * uu)
    y0, terms = opref.product(ac, as_, one["down"], one["down_s"])
    y1 = opref.product(ac, as_, w["down"][1], w["down_s"][1])[0]
    want = y0 + y1
    err = (out.double() - want).norm()
    assert err <= (2.0 ** -8 + 2.0 ** -8) * want.norm() + 2.0 ** -17 * 2 * terms.norm(), err / want.norm()


@pytest.mark.parametrize("rows", [1, 3, 16, 20, 70, 300, 1100])
def test_rounding_of_activations_halfway_between_codes(lib, rows):
    """Activations that are whole numbers, halfway between two codes of their block, and the identity as the down matrix:
    every stage is exact but the rounding itself. Row r: gate 64 (its sigmoid is 1 in 32 bits), up k * (16 + 1), k * (18 + 1),
    .. and k * 448 for the largest, k small and not a power of two: codes of exactly 17, 19, .. before they are rounded."""
    H = F = 128
    k = torch.tensor([3, 5, 7, 9, 11, 13, 15], dtype=torch.float64).repeat(rows // 7 + 1)[:rows]
    x = torch.zeros((rows, H), dtype=torch.float64)
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = 448.0, 64.0, k, k                       # the scale is 1
    gate, up = torch.zeros((F, H), dtype=torch.float64), torch.zeros((F, H), dtype=torch.float64)
    gate[:, 1] = 1.0
    up[0, 2] = 448.0
    for f in range(1, F):
        m, size = 16 + 2 * (f % 8), 2.0 ** (f // 8 % 5 - 1)
        up[f, 2], up[f, 3] = m * size * (-1) ** f, size * (-1) ** f
    one = torch.ones((1, 1), device="cuda")
    as_codes = lambda t: t.float().to(torch.float8_e4m3fn).cuda()  # noqa: E731
    plan = lib.dense.DensePlan(lib.dense.FFN_SILU_GATE, synth.FMT_F8_E4M3, H, F)
    plan.reserve(rows)
    plan.bind(as_codes(up), as_codes(gate), as_codes(torch.eye(H)), up_scale=one, gate_scale=one, down_scale=one)
    y = torch.empty((rows, H), dtype=torch.bfloat16, device="cuda")
    plan.forward(x.to(torch.bfloat16).cuda(), y, rows)
    plan.poll()
    codes, scales = opref.quantize(64.0 * (x @ up.t()))
    assert torch.equal(scales[:, 0], 64.0 * k) and codes.abs().max() == 448.0
    assert torch.equal(y.double().cpu(), codes * scales)


def test_other_types_of_the_same_size(lib):
    """Every entry point of the newer operators: fp16 rows are not bf16, floats are no ids, whole numbers no weights."""
    plan, w, g = expert_layer(lib, 16, 128, 128, 4, 2, 8)
    x, ids, probs = bf16(g, 8, 128), torch.zeros((8, 2), dtype=torch.int32, device="cuda"), torch.ones((8, 2), device="cuda")
    router = lib.moe.RouterPlan.new(128, 4, 2)
    router.reserve(8)
    rw, rb = torch.zeros((4, 128), device="cuda"), torch.zeros(4, device="cuda")
    router.bind(rw, rb)
    dense, y = projection(lib, w["up"][0], w["up_s"][0], x)
    logits = torch.zeros((8, 4), device="cuda")
    out = torch.empty_like(x)
    whole = lambda t: t.to(torch.int32)  # noqa: E731
    for call in (lambda: plan.forward(x.half(), ids, probs, x, 8, out=out), lambda: plan.forward(x, ids.float(), probs, x, 8, out=out), lambda: plan.forward(x, ids, whole(probs), x, 8, out=out),
                 lambda: plan.forward(x, ids, probs, x.half(), 8, out=out), lambda: plan.forward(x, ids, probs, x, 8, out=out.half()), lambda: router.bind(whole(rw), rb), lambda: router.bind(rw, whole(rb)),
                 lambda: router.forward(x.half(), ids, probs, 8), lambda: router.forward(x, ids.float(), probs, 8), lambda: router.forward(x, ids, whole(probs), 8),
                 lambda: router.forward(x, ids, probs, 8, logits=whole(logits)), lambda: router.select(whole(logits), ids, probs, 8), lambda: router.select(logits, ids.float(), probs, 8),
                 lambda: dense.forward(x.half(), y, 8), lambda: dense.forward(x, y.half(), 8), lambda: lib.moe.block_norm(x, norm_out=out, pre_weight=whole(torch.ones(128, device="cuda")))):
        with pytest.raises(_lib.OcoError, match="is needed"):
            call()
    router.forward(x, ids.view(torch.uint32), probs, 8)


@pytest.mark.parametrize("rows", [1, 4, 40])
def test_weights_written_just_before_they_are_bound(lib, rows):
    """Codes that kernels of another stream are still making when they are bound: binding waits for them, as calls fetch
    weights ahead of the work before them."""
    H, F = 2048, 4096
    g = gen(rows)
    wide = torch.randn((F, H), device="cuda", generator=g)
    x = bf16(g, rows, H)
    one = torch.full((F // 128, H // 128), 2e-4, device="cuda")
    plan = lib.dense.DensePlan(lib.dense.PROJECTION, synth.FMT_F8_E4M3, H, F)
    plan.reserve(rows)
    y = torch.empty((rows, F), dtype=torch.bfloat16, device="cuda")
    codes = torch.zeros((F, H), dtype=torch.float8_e4m3fn, device="cuda")
    slow = torch.randn((8192, 8192), device="cuda", generator=g)
    slow_out = slow @ slow
    torch.cuda.synchronize()
    for size in (105.0, 50.0):                               # and once more after rewriting them
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(4):                               # some tens of milliseconds
                torch.mm(slow, slow, out=slow_out)
            codes.copy_((wide * size).clamp(-448, 448))
        plan.bind(codes, up_scale=one)
        plan.forward(x, y, rows)
        within(y, *opref.product(*opref.quantize(x.double()), (wide * size).clamp(-448, 448).to(torch.float8_e4m3fn), one))
