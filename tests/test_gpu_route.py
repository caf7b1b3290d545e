"""Routing to experts against a plain implementation in 64 bits.

Ids have to be equal.  Weights are rounded once, from values held in 64 bits: half a step of fp32 (2^-24 of the value),
and a hundredth of that for what 64 bits leave open."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
WEIGHT_TOL = 1.01 * 2.0 ** -24


@pytest.fixture(scope="module")
def ext():
    import int4matmul_kernels_amd as pkg
    return pkg.load_extension()


def plain(logits, top_k, scoring="softmax", bias=None, n_groups=1, topk_groups=1, group_score="max", renormalize=True, scale=1.0):
    logits = logits.double().cpu().numpy()
    bias = None if bias is None else bias.double().cpu().numpy()
    T, E = logits.shape
    weights, ids = np.zeros((T, top_k)), np.full((T, top_k), -1, np.int32)
    for t in range(T):
        row, p = logits[t], np.zeros(E)
        live = [e for e in range(E) if row[e] > -math.inf]
        if not live:
            continue
        top = max(row[e] for e in live)
        for e in live:
            if scoring == "softmax":
                p[e] = 1.0 if row[e] == top else math.exp(row[e] - top)
            else:
                p[e] = 1.0 / (1.0 + math.exp(-row[e])) if row[e] > -700 else 0.0
        if scoring == "softmax":
            p /= p.sum()
        value = p if bias is None else p + bias
        key = row if bias is None else value
        live = [e for e in live if key[e] > -math.inf]
        if n_groups > 1:
            size, score = E // n_groups, {}
            for g in range(n_groups):
                members = [e for e in live if e // size == g]
                if members:
                    score[g] = max(key[e] for e in members) if group_score == "max" else sum(sorted((value[e] for e in members), reverse=True)[:2])
            kept = sorted(score, key=lambda g: (-score[g], g))[:topk_groups]
            live = [e for e in live if e // size in kept]
        best = sorted(live, key=lambda e: (-key[e], e))[:top_k]
        w = np.array([p[e] for e in best])
        if renormalize and w.sum() > 0:
            w = w / w.sum()
        ids[t, :len(best)], weights[t, :len(best)] = best, w * scale
    return weights, ids


def check(ext, logits, top_k, **how):
    weights, ids = ext.route_experts(logits, top_k, **how)
    want_w, want_i = plain(logits.reshape(-1, logits.shape[-1]), top_k, **how)
    assert weights.dtype == torch.float32 and ids.dtype == torch.int32
    assert weights.shape == ids.shape == (*logits.shape[:-1], top_k)
    assert np.array_equal(ids.cpu().numpy().reshape(want_i.shape), want_i)
    got = weights.double().cpu().numpy().reshape(want_w.shape)
    # (below the normal numbers of fp32 half a step is 2^-150)
    assert np.all(np.abs(got - want_w) <= WEIGHT_TOL * np.abs(want_w) + 2.0 ** -150), np.abs(got - want_w).max()
    return weights, ids


def logits_of(T, E, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (1.5 * torch.randn((T, E), generator=gen, device="cuda")).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 8), (5, 8, 2), (3, 63, 63), (2, 65, 6), (17, 129, 4), (33, 256, 8), (513, 60, 4), (2, 257, 3), (3, 1000, 10), (2, 1024, 64)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_sizes(ext, T, E, k, scoring, dtype):
    logits = logits_of(T, E, dtype, T + E)
    check(ext, logits, k, scoring=scoring)
    bias = torch.linspace(-0.3, 0.3, E, device="cuda")[torch.randperm(E, device="cuda")]
    check(ext, logits, k, scoring=scoring, bias=bias, renormalize=False, scale=2.5)


@pytest.mark.parametrize("E,groups,kept,k", [(256, 8, 4, 8), (60, 6, 2, 20), (64, 64, 5, 5), (96, 4, 4, 7), (160, 5, 1, 6), (1024, 2, 1, 3), (21, 3, 2, 14), (8, 8, 8, 8)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_groups(ext, E, groups, kept, k, group_score, bias, scoring):
    logits = logits_of(37, E, torch.float16, E)
    logits[5:20] = logits[5:20].masked_fill(torch.rand((15, E), device="cuda") < 0.7, -math.inf)
    b = 0.2 * torch.randn(E, device="cuda") if bias else None
    check(ext, logits, k, scoring=scoring, bias=b, n_groups=groups, topk_groups=kept, group_score=group_score)


def test_ties_go_to_the_lowest_index(ext):
    logits = torch.zeros((4, 130), device="cuda")
    logits[1, ::2] = -0.0                                       # (equal to 0)
    logits[2] = torch.randint(-2, 3, (130,), device="cuda").float()
    logits[3, 100:] = 1.0
    _, ids = check(ext, logits, 9)
    assert ids[0].tolist() == list(range(9)) and ids[1].tolist() == list(range(9)) and ids[3].tolist() == list(range(100, 109))
    check(ext, logits, 9, bias=torch.zeros(130, device="cuda"), scoring="sigmoid")
    check(ext, logits, 9, n_groups=13, topk_groups=3, group_score="top2")
    check(ext, logits, 9, n_groups=13, topk_groups=3, bias=torch.zeros(130, device="cuda"))


@pytest.mark.parametrize("how", [dict(), dict(scoring="sigmoid"), dict(n_groups=4, topk_groups=2), dict(n_groups=4, topk_groups=2, group_score="top2"), dict(with_bias=True)])
def test_masked_and_extreme_logits(ext, how):
    how = dict(how)
    inf, E = math.inf, 24
    rows = torch.randn((12, E), device="cuda")
    rows[0] = -inf                                              # nothing left
    rows[1] = -inf
    rows[1, 17] = 0.5                                           # one expert left
    rows[2, :20] = -inf                                         # fewer than top_k
    rows[3] = math.nan
    rows[4, 3:9] = math.nan                                     # a NaN is out, the others are not harmed
    rows[5] = -65504.0                                          # the lowest value of fp16 is a number: all tie
    rows[6, :12] = -65504.0
    rows[7, 5] = inf                                            # the limit: all the weight
    rows[8, [2, 20]] = inf
    rows[9] = 65504.0
    rows[10, ::2] = torch.finfo(torch.float32).min
    rows[11] = 1e4
    if how.pop("with_bias", False):
        how["bias"] = torch.where(torch.arange(E, device="cuda") % 5 == 0, -inf, 0.1 * torch.randn(E, device="cuda"))
        how["bias"][7] = math.nan
    weights, ids = check(ext, rows, 6, **how)
    assert ids[0].tolist() == [-1] * 6 and ids[3].tolist() == [-1] * 6 and not weights[0].any() and not weights[3].any()
    check(ext, rows.half(), 6, **how)


def test_shapes_strides_and_empty(ext):
    logits = logits_of(24, 40, torch.float16, 1)
    w, i = check(ext, logits.reshape(2, 3, 4, 40), 3)
    wide = torch.zeros((24, 80), dtype=torch.float16, device="cuda")
    wide[:, ::2] = logits
    w2, i2 = ext.route_experts(wide[:, ::2], 3)
    assert torch.equal(w2.reshape(-1), w.reshape(-1)) and torch.equal(i2.reshape(-1), i.reshape(-1))
    w, i = ext.route_experts(logits[:0], 3)
    assert w.shape == (0, 3) and i.shape == (0, 3)
    one, _ = ext.route_experts(logits[0], 3)
    assert one.shape == (3,)


def test_captured_streams_and_repeats(ext):
    a, b = logits_of(300, 96, torch.float32, 2), logits_of(300, 96, torch.float32, 3)
    bias = 0.1 * torch.randn(96, device="cuda")
    held = a.clone()
    ext.route_experts(held, 6, bias=bias, n_groups=6, topk_groups=3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ext.route_experts(held, 6, bias=bias, n_groups=6, topk_groups=3)
    for x in (a, b, a, b):
        held.copy_(x)
        graph.replay()
        want = ext.route_experts(x, 6, bias=bias, n_groups=6, topk_groups=3)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ext.route_experts(a, 6, bias=bias, n_groups=6, topk_groups=3)
    torch.cuda.current_stream().wait_stream(side)
    want = ext.route_experts(a, 6, bias=bias, n_groups=6, topk_groups=3)
    assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])


def test_rows_beyond_the_last_stay(ext):
    """through the C interface: what lies behind the last row's results is left as it was"""
    from int4matmul_kernels_amd import capi
    logits = logits_of(7, 30, torch.float16, 4)
    w, i = torch.full((9, 4), 7.0, device="cuda"), torch.full((9, 4), 7, dtype=torch.int32, device="cuda")
    capi.route_experts(w[:7], i[:7], logits)
    want = ext.route_experts(logits, 4)
    assert torch.equal(w[:7], want[0]) and torch.equal(i[:7], want[1])
    assert torch.all(w[7:] == 7) and torch.all(i[7:] == 7)


def test_refusals(ext):
    logits = logits_of(4, 32, torch.float16, 5)
    for how in (dict(top_k=0), dict(top_k=33), dict(top_k=2, scoring="tanh"), dict(top_k=2, group_score="sum"), dict(top_k=2, n_groups=5),
                dict(top_k=2, n_groups=4, topk_groups=5), dict(top_k=9, n_groups=4, topk_groups=1), dict(top_k=2, n_groups=0),
                dict(top_k=2, bias=torch.zeros(31, device="cuda")), dict(top_k=2, bias=torch.zeros(32)),
                dict(top_k=2, bias=torch.zeros(32, device="cuda", dtype=torch.float16)), dict(top_k=2, scale=math.inf)):
        with pytest.raises(RuntimeError):
            ext.route_experts(logits, **how)
    with pytest.raises(RuntimeError):
        ext.route_experts(logits.double(), 2)
    with pytest.raises(RuntimeError):
        ext.route_experts(logits.cpu(), 2)
    with pytest.raises(RuntimeError):
        ext.route_experts(torch.zeros((2, 1025), device="cuda"), 2)
    asks = logits.float().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        ext.route_experts(asks, 2)
    with torch.no_grad():
        ext.route_experts(asks, 2)


def test_a_bias_that_asks_for_a_gradient_is_refused(ext):
    with pytest.raises(RuntimeError, match="no backward"):
        ext.route_experts(logits_of(4, 32, torch.float16, 5), 2, bias=torch.zeros(32, device="cuda", requires_grad=True))


def test_more_tokens_than_a_grid_has(ext):
    """2^26 and a few tokens, 64 work-items for each: more than one launch holds"""
    T, gen = 2 ** 26 + 5, torch.Generator(device="cuda").manual_seed(3)
    logits = torch.empty((T, 2), dtype=torch.float16, device="cuda").normal_(generator=gen)
    weights, ids = ext.route_experts(logits, 1, renormalize=False)
    assert torch.equal(ids[:, 0], (logits[:, 1] > logits[:, 0]).to(torch.int32))
    want = torch.sigmoid((logits[:, 1].double() - logits[:, 0].double()).abs())
    assert ((weights[:, 0].double() - want).abs() <= WEIGHT_TOL * want).all()
