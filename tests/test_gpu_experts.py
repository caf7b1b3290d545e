"""The experts' feed-forward on packed weights against a plain implementation in 64 bits on the same codes.

Tolerances.  From the exact result a kernel may be off by its roundings to fp16, each at most half a step (2^-11 relative):
two of each weight of the first product, the hidden state, two of each weight of the second product, the result: six.  They are
spread over the terms of a sum, so in the 2-norm they add as independent ones at most: sqrt(6) 2^-11 = 1.2e-3 of the result;
the activation can pass an error of the gate on with a factor of up to 1.1 (its slope), and weights whose two roundings
meet a difference q - z of less than 1 lose no more than that: 1.5e-3.  A single element can be off by more than its share,
five times the 2-norm's over the root of the mean square: 8e-3."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
REL, MOST = 1.5e-3, 8e-3
FORMATS = [(4, False), (3, False), (2, False), (4, True)]


@pytest.fixture(scope="module")
def ext():
    import int4matmul_kernels_amd as pkg
    return pkg.load_extension()


def packed(bits, sparse, n, k, s, group, gen, expo=0.0):
    """(matrix, scales, zeros, mask) of n experts and their exact weights [n, k, s] in float64"""
    from int4matmul_kernels_amd import capi
    codes = torch.randint(0, 2 ** bits, (n, k, s), dtype=torch.uint8, generator=gen, device="cuda")
    keep = None
    if sparse:
        keep = torch.zeros((n, s, k // 32, 32), dtype=torch.uint8, device="cuda")
        keep.scatter_(3, torch.rand(keep.shape, generator=gen, device="cuda").argsort(dim=3)[..., :16], 1)
        keep = keep.reshape(n, s, k)
    groups = 1 if group < 0 else -(-k // group)
    lo, hi = (0.001, 0.02) if bits == 4 else (0.004, 0.08)
    scales = torch.empty((n, groups, s), device="cuda").uniform_(lo, hi, generator=gen)
    zeros = torch.full((n, groups, s), (2 ** bits - 1) / 2, device="cuda").half()
    if expo:
        chosen = torch.rand((n, groups, s), generator=gen, device="cuda") < expo
        scales = torch.where(chosen, -scales / 2 ** (2 ** (bits - 1) - bits + 1), scales)
        zeros = torch.where(chosen, torch.zeros_like(zeros), zeros)
    scales = scales.half()
    matrix = torch.empty((n, k // 16 if sparse else k * bits // 32, s), dtype=torch.int32, device="cuda")
    mask = torch.empty((n, k // 32, s), dtype=torch.int32, device="cuda") if sparse else None
    for e in range(n):
        if sparse:
            capi.sparse_pack(matrix[e], mask[e], codes[e].t().contiguous(), keep[e])
        else:
            capi.dense_pack(bits, matrix[e], codes[e])
    rows = torch.arange(k, device="cuda") // (k if group < 0 else group)
    sc, ze, q = scales.double()[:, rows], zeros.double()[:, rows], codes.double()
    half = 2 ** (bits - 1)
    power = 2.0 ** (codes % half).double() * torch.where(codes < half, 1.0, -1.0).double()
    w = torch.where(sc >= 0, (q - ze) * sc, ze - sc * power)
    if sparse:
        w = w * keep.transpose(1, 2)
    return (matrix, scales, zeros, mask), w


def problem(bits=4, sparse=False, n=4, k=2, T=5, K=256, F=192, group=64, expo=0.0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    up, wu = packed(bits, sparse, n, K, 2 * F, group, gen, expo)
    down, wd = packed(bits, sparse, n, F, K, group, gen, expo)
    x = torch.randn((T, K), generator=gen, device="cuda").half()
    ids = torch.rand((T, n), generator=gen, device="cuda").argsort(dim=1)[:, :k].to(torch.int32).contiguous()
    weights = torch.rand((T, k), generator=gen, device="cuda")
    return dict(bits=bits, x=x, weights=weights, ids=ids, up=up, down=down, wu=wu, wd=wd, group=group)


def plain(p):
    x, F = p["x"].double(), p["wd"].shape[1]
    y = torch.zeros((x.shape[0], p["wd"].shape[2]), dtype=torch.float64, device="cuda")
    for e in range(p["wu"].shape[0]):
        token, slot = (p["ids"] == e).nonzero(as_tuple=True)
        if token.numel():
            gate, up = (x[token] @ p["wu"][e]).split(F, dim=1)
            h = gate * torch.sigmoid(gate) * up
            y.index_add_(0, token, p["weights"].double()[token, slot][:, None] * (h @ p["wd"][e]))
    return y


def forward(ext, p, **change):
    p = dict(p, **change)
    (um, us, uz, uk), (dm, ds, dz, dk) = p["up"], p["down"]
    return ext.experts_forward(p["bits"], p["x"], p["weights"], p["ids"], um, us, uz, dm, ds, dz, p["group"], uk, dk)


def close(got, want):
    assert got.dtype == torch.float16 and torch.isfinite(got).all()
    off, rms = got.double() - want, want.pow(2).mean().sqrt()
    rel = (off.norm() / want.norm()).item() if want.norm() > 0 else off.norm().item()
    most = (off.abs() / torch.maximum(rms, want.abs())).max().item() if rms > 0 else 0.0
    assert rel <= REL and most <= MOST, (rel, most)


@pytest.mark.parametrize("bits,sparse", FORMATS)
@pytest.mark.parametrize("T,n,k", [(1, 4, 2), (1, 3, 3), (5, 4, 2), (33, 4, 1), (70, 2, 2), (150, 3, 2), (600, 4, 3), (1500, 2, 1)])
def test_rows(ext, bits, sparse, T, n, k):
    p = problem(bits, sparse, n, k, T, seed=T + bits)
    close(forward(ext, p), plain(p))


@pytest.mark.parametrize("bits,sparse", FORMATS)
@pytest.mark.parametrize("K,F,group", [(64, 64, 64), (64, 64, -1), (128, 320, 128), (320, 64, 128), (1344, 448, 128), (576, 704, -1), (2048, 512, 256), (512, 1088, 1024)])
def test_features(ext, bits, sparse, K, F, group):
    for T in (3, 40, 700):
        p = problem(bits, sparse, 3, 2, T, K, F, group, seed=K + F)
        close(forward(ext, p), plain(p))


@pytest.mark.parametrize("bits,sparse", FORMATS)
@pytest.mark.parametrize("T", [2, 60, 520])
def test_exponent_mode(ext, bits, sparse, T):
    for share in (0.05, 0.6, 1.0):
        p = problem(bits, sparse, 3, 2, T, 512, 256, 64, expo=share, seed=T)
        close(forward(ext, p), plain(p))


@pytest.mark.parametrize("T", [1, 9, 300])
def test_pairs_without_an_expert(ext, T):
    p = problem(T=T, n=5, k=3, seed=T)
    ids = p["ids"].clone()
    ids[:, 1] = torch.tensor([-1, 5, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda").repeat(T)[:T]
    ids[T // 2] = -1                                            # a token without any
    weights = p["weights"].clone()
    weights[:, 1] = math.nan                                    # (not looked at)
    got = forward(ext, p, ids=ids, weights=weights)
    want = plain(dict(p, ids=torch.where((ids < 0) | (ids >= 5), -1, ids), weights=torch.nan_to_num(weights)))
    assert not got[T // 2].any()
    close(got, want)
    assert not forward(ext, p, ids=torch.full_like(ids, -1)).any()


def test_skewed_and_repeated(ext):
    """all rows at one expert; the same expert in every slot of a token; an expert that nobody asked"""
    for T in (1, 20, 900):
        p = problem(T=T, n=6, k=3, seed=7)
        for ids in (torch.full_like(p["ids"], 4), torch.where(p["ids"] < 3, 5, 0).to(torch.int32)):
            close(forward(ext, p, ids=ids), plain(dict(p, ids=ids)))


def test_more_experts_than_a_wave_has_lanes(ext):
    for T, n, k in ((1, 200, 8), (30, 130, 4), (500, 128, 8)):
        p = problem(T=T, n=n, k=k, K=128, F=64, seed=n)
        close(forward(ext, p), plain(p))


@pytest.mark.parametrize("T", [1, 6, 130, 700])
def test_infinities_and_nan_stay_where_they_are(ext, T):
    """an expert whose scales are infinite or NaN spoils its own tokens, a token its own row"""
    p = problem(T=T + 2, n=4, k=1, seed=T)
    ids = (torch.arange(T + 2, device="cuda") % 3).to(torch.int32)[:, None].contiguous()
    ids[T] = 3
    clean = forward(ext, p, ids=ids)
    (um, us, uz, uk) = p["up"]
    us = us.clone()
    us[3] = math.inf
    us[3, 0] = math.nan
    x = p["x"].clone()
    x[T + 1] = math.nan
    got = forward(ext, p, ids=ids, x=x, up=(um, us, uz, uk))
    assert torch.equal(got[:T], clean[:T])
    assert not torch.isfinite(got[T:]).any()


def test_shapes_strides_types_and_empty(ext):
    p = problem(T=12, k=2, seed=3)
    want = forward(ext, p)
    batched = {n: p[n].reshape(3, 4, -1) for n in ("x", "weights", "ids")}
    assert torch.equal(forward(ext, p, **batched).reshape(12, -1), want)
    wide = torch.zeros((12, 512), dtype=torch.float16, device="cuda")
    wide[:, ::2] = p["x"]
    apart = torch.full((12, 4), 99, dtype=torch.int32, device="cuda")
    apart[:, ::2] = p["ids"]
    assert torch.equal(forward(ext, p, x=wide[:, ::2], ids=apart[:, ::2], weights=p["weights"].t().contiguous().t()), want)
    assert torch.equal(forward(ext, p, x=p["x"].float()), want)
    assert forward(ext, p, x=p["x"][:0], ids=p["ids"][:0], weights=p["weights"][:0]).shape == (0, 256)
    one = problem(group=-1, T=4, seed=5)
    flat = [(m, s[:, 0], z[:, 0], k) for m, s, z, k in (one["up"], one["down"])]
    assert torch.equal(forward(ext, one, up=flat[0], down=flat[1]), forward(ext, one))


@pytest.mark.parametrize("T", [1, 40, 600])
def test_captured_streams_and_repeats(ext, T):
    a, b = problem(T=T, seed=1), problem(T=T, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(9)
    b["x"] = torch.randn(a["x"].shape, generator=gen, device="cuda").half()
    b["ids"] = a["ids"].flip(0).contiguous()
    held = {n: a[n].clone() for n in ("x", "ids", "weights")}
    want = {id(q): forward(ext, q) for q in (a, b)}
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(forward(ext, a, **held))
    for q in (a, b, a, b):
        for n in held:
            held[n].copy_(q[n])
        for g in graphs:
            g.replay()
        eager = forward(ext, q)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[id(q)]) and all(torch.equal(o, eager) for o in outs)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s, q in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append((forward(ext, q), want[id(q)]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in got)


def test_rows_beyond_the_last_stay_and_the_workspace_may_hold_anything(ext):
    from int4matmul_kernels_amd import capi
    for T in (1, 21, 400):
        p = problem(T=T, seed=2)
        outs = torch.full((T + 3, 256), 7.0, dtype=torch.float16, device="cuda")
        ws = capi.new_experts_workspace(T, 2, 4, 256, 192, 64)
        ws.fill_(255)
        capi.experts_forward(4, outs[:T], p["x"], p["weights"], p["ids"], p["up"], p["down"], 64, ws)
        assert torch.equal(outs[:T], forward(ext, p)) and torch.all(outs[T:] == 7)
        with pytest.raises(capi.Int4mmError) as e:
            capi.experts_forward(4, outs[:T], p["x"], p["weights"], p["ids"], p["up"], p["down"], 64, ws[:-256])
        assert e.value.code == 6


def test_offsets_beyond_32_bits(ext):
    """pairs whose results lie more than 2^32 bytes, and elements, apart"""
    T, K, F, n, k = 70000, 8192, 64, 3, 8
    p = problem(T=1, K=K, F=F, n=n, k=1, seed=4)
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((T, K), generator=gen, device="cuda").half()
    ids = torch.randint(0, n, (T, k), generator=gen, device="cuda").to(torch.int32)
    weights = torch.rand((T, k), generator=gen, device="cuda")
    got = forward(ext, p, x=x, ids=ids, weights=weights)
    for rows in (slice(0, 40), slice(T // 2, T // 2 + 40), slice(T - 40, T)):
        close(got[rows], plain(dict(p, x=x[rows], ids=ids[rows], weights=weights[rows])))


def test_a_last_share_of_one_token(ext):
    """so many pairs that they go through the workspace in shares, the last one with a token alone"""
    T, k = 4096 * 4095 + 1, 64
    p = problem(T=1, n=70, k=64, K=64, F=64, seed=6)
    x = torch.zeros((T, 64), dtype=torch.float16, device="cuda")
    ids = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    weights = torch.zeros((T, k), device="cuda")
    x[-1:], ids[-1:], weights[-1:] = p["x"], p["ids"], p["weights"]
    got = forward(ext, p, x=x, ids=ids, weights=weights)
    assert torch.equal(got[-1:], forward(ext, p)) and not got[:-1].any()
    close(got[-1:], plain(p))


def test_layer_and_router_together():
    """router, experts and the modules that hold them, as a block of a model uses them"""
    from int4matmul_kernels_amd.quant_experts import ExpertRouter, QuantExperts
    from int4matmul_kernels_amd.quant_linear import QuantLinear
    torch.manual_seed(0)
    n, K, F = 8, 256, 128
    layer = QuantExperts.from_float((torch.randn((n, K, 2 * F), device="cuda") * 0.05).half(), (torch.randn((n, F, K), device="cuda") * 0.05).half(),
                                    group_size=64)
    gate = QuantLinear.from_float((torch.randn((K, 64), device="cuda") * 0.05).half(), group_size=64)
    router = ExpertRouter(n, 2, scoring="sigmoid", bias=True, n_groups=4, topk_groups=2, group_score="top2")
    router.bias.copy_(0.1 * torch.randn(n, device="cuda"))
    for shape in ((1, 1), (3, 50), (2, 300)):
        x = torch.randn((*shape, K), device="cuda").half()
        weights, ids = router(gate(x)[..., :n])
        y = layer(x, weights, ids)
        want = torch.zeros((*shape, K), dtype=torch.float64, device="cuda")
        for e in range(n):
            m = [QuantLinear.from_packed(4, getattr(layer, f"{w}_matrix")[e], getattr(layer, f"{w}_scales")[e], getattr(layer, f"{w}_zeros")[e],
                                         64).dequantized_weight().double() for w in ("up", "down")]
            g, u = (x.double() @ m[0]).split(F, dim=-1)
            term = (g * torch.sigmoid(g) * u) @ m[1]
            want += torch.where(ids == e, weights.double(), 0.0).sum(-1, keepdim=True) * term
        close(y, want)
    copy = QuantExperts(4, n, K, F, 64)
    copy.load_state_dict(layer.state_dict())
    assert torch.equal(copy(x, weights, ids), y)
    sparse = torch.zeros((n, 2 * F, K // 32, 32), dtype=torch.bool, device="cuda")
    sparse[..., ::2] = True
    sparse = sparse.reshape(n, 2 * F, K).transpose(1, 2)
    keep = torch.zeros((n, K, F // 32, 32), dtype=torch.bool, device="cuda")
    keep[..., 16:] = True
    keep = keep.reshape(n, K, F).transpose(1, 2)
    thin = QuantExperts.from_float((torch.randn((n, K, 2 * F), device="cuda") * 0.05).half(), (torch.randn((n, F, K), device="cuda") * 0.05).half(),
                                   group_size=64, up_keep=sparse, down_keep=keep)
    assert thin.sparse and torch.isfinite(thin(x, weights, ids)).all()


@pytest.mark.parametrize("T,n,k", [(2, 5, 3), (85, 9, 3), (128, 16, 2), (257, 16, 1), (64, 256, 4), (64, 257, 4), (255, 256, 1), (86, 300, 3)])
def test_few_pairs_with_and_without_an_expert(ext, T, n, k):
    """around the sizes where the pairs are ordered in another way; ids that nobody has; all pairs at one expert"""
    p = problem(T=T, n=n, k=k, K=128, F=64, seed=T)
    ids = p["ids"].clone()
    ids[::3, 0] = n
    ids[1::5] = -1
    for which in (p["ids"], ids, torch.full_like(ids, n - 1)):
        close(forward(ext, p, ids=which), plain(dict(p, ids=torch.where(which < n, which, -1))))


def test_refusals(ext):
    p = problem(T=4)
    (um, us, uz, _), (dm, ds, dz, _) = p["up"], p["down"]
    bad = [dict(ids=p["ids"].long()), dict(weights=p["weights"].half()), dict(ids=p["ids"][:, :1]), dict(x=p["x"][:, :128]), dict(x=p["x"].cpu()),
           dict(ids=p["ids"].cpu()), dict(up=(um[:3], us, uz, None)), dict(up=(um, us[:, :1].contiguous(), uz, None)), dict(up=(um.float(), us, uz, None)),
           dict(down=(dm, ds, dz.float(), None)), dict(down=(dm[:, :-1].contiguous(), ds, dz, None)), dict(bits=3), dict(group=96), dict(group=0),
           dict(up=(um, us, uz, torch.zeros((4, 8, 384), dtype=torch.int32, device="cuda"))), dict(up=(um.transpose(1, 2), us, uz, None)),
           dict(x=p["x"].to(torch.int32)), dict(x=p["x"][0], ids=p["ids"][0], weights=p["weights"][0])]
    for change in bad:
        with pytest.raises(RuntimeError):
            forward(ext, p, **change)
    with pytest.raises(ValueError):
        forward(ext, p, bits=5)
    with pytest.raises(RuntimeError, match="no backward"):
        forward(ext, p, x=p["x"].clone().requires_grad_())


@pytest.mark.parametrize("bits,sparse", FORMATS)
@pytest.mark.parametrize("T,n", [(1, 4), (9, 4), (300, 16), (300, 4)])
@pytest.mark.parametrize("sign", [1, -1])
def test_a_single_nan_scale(ext, bits, sparse, T, n, sign):
    """one group of one column of one expert has a NaN scale, of either sign: NaN where the definition has it, all else as without"""
    p = problem(bits, sparse, n, 1, T, seed=T + bits)
    ids = p["ids"].clone()
    ids[0] = 2
    nan = torch.tensor([0x7E00 if sign > 0 else -0x200], dtype=torch.int16, device="cuda").view(torch.float16)
    F = p["wd"].shape[1]
    for which, column, rows in (("up", 5, slice(64, 128)), ("up", F + 70, slice(64, 128)), ("down", 133, slice(64, 128))):
        m, s, z, k = p[which]
        s = s.clone()
        s[2, 1, column] = nan[0]
        assert s.view(torch.int16)[2, 1, column] == nan.view(torch.int16)[0]
        exact = p["w" + which[0]].clone()
        exact[2, rows, column] = math.nan
        got = forward(ext, p, ids=ids, **{which: (m, s, z, k)})
        want = plain(dict(p, ids=ids, **{"w" + which[0]: exact}))
        assert want[0].isnan().any() and torch.equal(got.isnan(), want.isnan())
        there = ~want.isnan()
        if there.any():
            close(got[there], want[there])


@pytest.mark.parametrize("bits,sparse", FORMATS)
@pytest.mark.parametrize("T", [20, 300, 900])
def test_pairs_beyond_the_range_of_fp16(ext, bits, sparse, T):
    """h @ DOWN far above 65504, weights that bring a token's sum back: the same in a small batch and in a large one"""
    p = problem(bits, sparse, 3, 2, T, seed=T)
    (m, s, z, k), by = p["down"], 2.0 ** 18 if bits == 4 else 2.0 ** 17
    p["down"], p["wd"] = (m, (s.float() * by).half(), z, k), p["wd"] * by
    p["weights"] = p["weights"] * 2.0 ** -16 * torch.tensor([1.0, -1.0], device="cuda")
    h = dict(p, weights=torch.tensor([1.0, 0.0], device="cuda").expand(T, 2))
    assert plain(h).abs().max() > 65504
    got = forward(ext, p)
    close(got, plain(p))
    if T > 20:
        assert (got[:3].double() - forward(ext, p, x=p["x"][:3], ids=p["ids"][:3], weights=p["weights"][:3]).double()).norm() <= 2 * REL * got[:3].double().norm()


def test_the_widest_rows(ext):
    """a width where a tile of 256 rows would be 2^32 bytes of hidden states"""
    T, F, part = 300, 2 ** 23, 2 ** 17
    p, gen = problem(2, False, 1, 1, T, 64, 64, -1, seed=8), torch.Generator(device="cuda").manual_seed(8)
    p["up"], p["wu"] = packed(2, False, 1, 64, 2 * F, -1, gen)
    parts = [packed(2, False, 1, part, 64, -1, gen) for _ in range(F // part)]         # (a matrix is packed in parts of its rows)
    first = parts[0][0]
    p["down"] = (torch.cat([m for (m, _, _, _), _ in parts], dim=1), first[1], first[2], None)
    p["wd"] = torch.cat([w / s.double() * first[1].double() for (_, s, _, _), w in parts], dim=1)
    got = forward(ext, p)
    for rows in (slice(0, 3), slice(255, 258), slice(T - 3, T)):
        close(got[rows], plain(dict(p, x=p["x"][rows], ids=p["ids"][rows], weights=p["weights"][rows])))
    few = forward(ext, p, x=p["x"][:20], ids=p["ids"][:20], weights=p["weights"][:20])
    close(few[:3], plain(dict(p, x=p["x"][:3], ids=p["ids"][:3], weights=p["weights"][:3])))


def test_more_work_items_than_a_grid_has(ext):
    """1000 pairs, one of 4096 experts each, of 2^21 columns: 8.6e9 work-items if they were one launch.  (The first eight experts are asked,
    and only they are in memory.)"""
    import ctypes as C
    from int4matmul_kernels_amd import capi
    T, K, F, part = 1000, 64, 2 ** 20, 2 ** 17
    p, gen = problem(2, False, 8, 1, T, 64, 64, -1, seed=9), torch.Generator(device="cuda").manual_seed(9)
    p["up"], p["wu"] = packed(2, False, 8, 64, 2 * F, -1, gen)
    parts = [packed(2, False, 8, part, 64, -1, gen) for _ in range(F // part)]
    first = parts[0][0]
    p["down"] = (torch.cat([m for (m, _, _, _), _ in parts], dim=1), first[1], first[2], None)
    p["wd"] = torch.cat([w / s.double() * first[1].double() for (_, s, _, _), w in parts], dim=1)
    sh = capi.experts_shape(T, 1, 4096, K, F, -1)
    ws = torch.empty(capi.lib().int4mm_experts_workspace_bytes(C.byref(sh)), dtype=torch.uint8, device="cuda")
    outs = torch.empty((T, K), dtype=torch.float16, device="cuda")
    ptr = lambda t: C.c_void_p(None if t is None else t.data_ptr())
    assert capi.lib().int4mm_experts_forward(2, *map(ptr, (outs, p["x"], p["weights"], p["ids"], *p["up"], *p["down"])), C.byref(sh), ptr(ws), ws.numel(),
                                             C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    for rows in (slice(0, 4), slice(254, 258), slice(T // 2, T // 2 + 4), slice(T - 4, T)):
        close(outs[rows], plain(dict(p, x=p["x"][rows], ids=p["ids"][rows], weights=p["weights"][rows])))


@pytest.mark.parametrize("T,n", [(32767, 3), (17000, 4096)])
def test_a_share_beyond_32_bits(ext, T, n):
    """pairs' results in one share of the workspace that are more than 2^32 elements apart, through the tiles and through the blocks of few pairs (of
    whose 4096 experts the first three are asked, and only they are in memory)"""
    import ctypes as C
    from int4matmul_kernels_amd import capi
    K, F, k = 32768, 64, 8
    p, gen = problem(2, False, 3, 1, 1, K, F, 1024, seed=5), torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((T, K), generator=gen, device="cuda").half()
    ids = torch.randint(0, 3, (T, k), generator=gen, device="cuda").to(torch.int32)
    weights = torch.rand((T, k), generator=gen, device="cuda")
    sh = capi.experts_shape(T, k, n, K, F, 1024)
    size = capi.lib().int4mm_experts_workspace_bytes(C.byref(sh))
    assert T * k * K > 2 ** 32 and size > 4 * T * k * K                       # (all of them at once)
    ws, outs = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty((T, K), dtype=torch.float16, device="cuda")
    ptr = lambda t: C.c_void_p(None if t is None else t.data_ptr())
    assert capi.lib().int4mm_experts_forward(2, *map(ptr, (outs, x, weights, ids, *p["up"], *p["down"])), C.byref(sh), ptr(ws), size,
                                             C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    for rows in (slice(0, 30), slice(T // 2, T // 2 + 30), slice(T - 30, T)):
        close(outs[rows], plain(dict(p, x=x[rows], ids=ids[rows], weights=weights[rows])))
