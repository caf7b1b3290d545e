"""Low-rank adapters of many requests against a plain implementation in 64 bits.

Tolerance, element by element: half a step of the fp16 result (2^-11 of it; 2^-25 below the normal numbers), and for the sums in
fp32 and the 22 bits that are kept of x down^T an error of at most (K + rank + 64) 2^-24 + 2^-21 of the sum of the terms' absolute values."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ext():
    import int4matmul_kernels_amd as pkg
    return pkg.load_extension()


def problem(shape=(5, 3), n=4, rank=16, K=256, S=192, per_row=False, seed=0, idle=0.2):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    of = shape if per_row else shape[:1]
    ids = torch.randint(0, n, of, generator=gen, device="cuda")
    ids = torch.where(torch.rand(of, generator=gen, device="cuda") < idle, -1, ids).to(torch.int32)
    return dict(base=torch.randn((*shape, S), generator=gen, device="cuda").half(), x=torch.randn((*shape, K), generator=gen, device="cuda").half(),
                down=(torch.randn((n, rank, K), generator=gen, device="cuda") / math.sqrt(K)).half(),
                up=(torch.randn((n, rank, S), generator=gen, device="cuda") * 0.3).half(),
                scales=torch.empty(n, device="cuda").uniform_(-2.0, 2.0, generator=gen), ids=ids)


def plain(p):
    """the result and the sum of the terms' absolute values"""
    y, x, ids = p["base"].double(), p["x"].double(), p["ids"]
    size = torch.zeros_like(y)
    each = ids.reshape(*ids.shape, *[1] * (x.dim() - 1 - ids.dim())).expand(x.shape[:-1])
    for a in range(p["down"].shape[0]):
        rows = each == a
        if rows.any():
            d, u, c = p["down"][a].double(), p["up"][a].double(), p["scales"][a].double()
            y[rows] += c * (x[rows] @ d.t() @ u)
            size[rows] = c.abs() * (x[rows].abs() @ d.abs().t() @ u.abs())
    return y, size


def add(ext, p, **change):
    p = dict(p, **change)
    return ext.low_rank_add(p["base"], p["x"], p["down"], p["up"], p["scales"], p["ids"])


def close(got, p, rows=slice(None)):
    want, size = plain(p)
    K, rank = p["x"].shape[-1], p["down"].shape[1]
    off = (got.double() - want).abs()
    most = 2.0 ** -11 * want.abs() + 2.0 ** -25 + ((K + rank + 64) * 2.0 ** -24 + 2.0 ** -21) * size
    assert got.dtype == torch.float16 and (off <= most).all(), (off / most).max().item()


@pytest.mark.parametrize("rank", [1, 4, 16, 20, 32, 33, 64, 100, 128, 200, 512])
@pytest.mark.parametrize("shape,per_row", [((1, 1), False), ((7, 1), False), ((300, 1), False), ((1, 45), True), ((3, 100), False), ((1, 700), True)])
def test_ranks_and_rows(ext, rank, shape, per_row):
    p = problem(shape, 5, rank, per_row=per_row, seed=rank)
    close(add(ext, p), p)


@pytest.mark.parametrize("K,S", [(64, 64), (64, 1088), (1344, 64), (5120, 320), (2048, 1408), (448, 4160)])
@pytest.mark.parametrize("T", [1, 16, 17, 64, 256, 257, 600])
def test_features(ext, K, S, T):
    for n in (1, 3, 40):
        p = problem((T, 1), n, 24, K, S, seed=K + T)
        close(add(ext, p), p)


def test_ids_per_request_row_and_dimension(ext):
    p = problem((2, 3, 5), 4, 8, seed=1)
    for of in ((2,), (2, 3), (2, 3, 5)):
        q = dict(p, ids=torch.randint(-1, 4, of, device="cuda").to(torch.int32))
        close(add(ext, q), q)
    q = dict(p, ids=torch.randint(-1, 4, (3, 2), device="cuda").to(torch.int32).t())
    close(add(ext, q), q)


def test_rows_without_an_adapter_keep_their_base(ext):
    for T in (1, 40, 500):
        p = problem((T, 1), 3, 16, seed=T, idle=0.0)
        p["base"][:, :, 5] = math.nan
        p["base"][:, :, 6] = -65504.0
        p["base"][:, :, 7] = math.inf
        ids = torch.tensor([-1, 3, 2 ** 31 - 1, -2 ** 31, 1000], dtype=torch.int32, device="cuda").repeat(T)[:T].contiguous()
        got = add(ext, p, ids=ids)
        assert torch.equal(got.view(torch.int16), p["base"].view(torch.int16))


@pytest.mark.parametrize("T", [6, 200, 700])
def test_infinities_and_nan_stay_where_they_are(ext, T):
    """an adapter's infinities and NaN reach its own rows alone, and a row's reach that row"""
    p = problem((T, 1), 4, 16, seed=T, idle=0.0)
    p["ids"] = (torch.arange(T, device="cuda") % 3).to(torch.int32)
    p["ids"][T - 1] = 3
    clean = add(ext, p)
    q = {n: v.clone() for n, v in p.items()}
    q["down"][3] = math.nan
    q["up"][3] = math.inf
    q["x"][T - 2] = math.inf
    got = add(ext, q)
    assert torch.equal(got[:T - 2], clean[:T - 2])
    assert not torch.isfinite(got[T - 2:]).any()


def test_large_and_small_products(ext):
    """x down^T beyond fp16's range times factors that bring it back, and products below fp16's normal numbers"""
    for T in (2, 300):
        for by in (2.0 ** 10, 2.0 ** -10):
            p = problem((T, 1), 2, 16, seed=3, idle=0.0)
            p["x"] = (p["x"].float() * by).half()
            p["down"] = (p["down"].float() * by).half()
            p["up"] = (p["up"].float() / by).half()
            p["scales"] = p["scales"] / by
            p["scales"][1] = 0.0
            close(add(ext, p), p)


def test_in_place_outs_strides_types_and_empty(ext):
    p = problem((6, 40), 3, 16, seed=2)
    want = add(ext, p)
    base = p["base"].clone()
    assert ext.low_rank_add(base, p["x"], p["down"], p["up"], p["scales"], p["ids"], base).data_ptr() == base.data_ptr()
    assert torch.equal(base, want)
    outs = torch.empty_like(base)
    ext.low_rank_add(p["base"], p["x"], p["down"], p["up"], p["scales"], p["ids"], outs=outs)
    assert torch.equal(outs, want)
    wide = torch.zeros((6, 40, 512), dtype=torch.float16, device="cuda")
    wide[..., ::2] = p["x"]
    turned = p["base"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(add(ext, p, x=wide[..., ::2], base=turned), want)
    assert torch.equal(add(ext, p, x=p["x"].float()), want)
    empty = problem((0, 4), 3, 16)
    assert add(ext, empty).shape == (0, 4, 192)


def test_captured_streams_and_repeats(ext):
    for shape in ((40, 1), (4, 200)):
        a, b = problem(shape, 6, 16, seed=1), problem(shape, 6, 16, seed=2)
        b.update({n: a[n] for n in ("down", "up", "scales")})
        held = {n: a[n].clone() for n in ("base", "x", "ids")}
        want = {id(q): add(ext, q) for q in (a, b)}
        torch.cuda.synchronize()
        graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
        for g in graphs:
            with torch.cuda.graph(g):
                outs.append(add(ext, a, **held))
        for q in (a, b, a, b):
            for n in held:
                held[n].copy_(q[n])
            for g in graphs:
                g.replay()
            eager = add(ext, q)
            torch.cuda.synchronize()
            assert torch.equal(eager, want[id(q)]) and all(torch.equal(o, eager) for o in outs)
        streams, got = [torch.cuda.Stream() for _ in range(2)], []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            for s, q in zip(streams, (a, b)):
                with torch.cuda.stream(s):
                    got.append((add(ext, q), want[id(q)]))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in got)


def test_rows_beyond_the_last_stay_and_the_workspace_may_hold_anything(ext):
    from int4matmul_kernels_amd import capi
    for T in (1, 37, 400):
        p = problem((T, 1), 3, 20, seed=T)
        outs = torch.full((T + 20, 192), 7.0, dtype=torch.float16, device="cuda")
        ws = capi.new_adapters_workspace(T, 1, p["down"], p["up"])
        ws.fill_(255)
        capi.low_rank_add(outs[:T], p["base"][:, 0], p["x"][:, 0], p["down"], p["up"], p["scales"], p["ids"], 1, ws)
        assert torch.equal(outs[:T], add(ext, p)[:, 0]) and torch.all(outs[T:] == 7)
        with pytest.raises(capi.Int4mmError) as e:
            capi.low_rank_add(outs[:T], p["base"][:, 0], p["x"][:, 0], p["down"], p["up"], p["scales"], p["ids"], 1, ws[:-16])
        assert e.value.code == 6


def test_offsets_beyond_32_bits(ext):
    """rows more than 2^32 bytes, and elements, into base and outs"""
    T, S = 140000, 32768
    p = problem((1, 1), 3, 8, 64, S, seed=4, idle=0.0)
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((T, 64), generator=gen, device="cuda").half()
    base = torch.empty((T, S), dtype=torch.float16, device="cuda").normal_(generator=gen)
    ids = torch.randint(0, 3, (T,), generator=gen, device="cuda").to(torch.int32)
    got = add(ext, p, base=base, x=x, ids=ids)
    for rows in (slice(0, 20), slice(T // 2, T // 2 + 20), slice(T - 20, T)):
        close(got[rows], dict(p, base=base[rows], x=x[rows], ids=ids[rows]))


@pytest.mark.parametrize("bits,sparse", [(4, False), (2, False), (4, True)])
@pytest.mark.parametrize("shape", [(1, 1), (6, 1), (3, 70)])
def test_beside_a_packed_projection(bits, sparse, shape):
    """a layer with its adapters: the projection's own output plus each request's term, then the bias"""
    from int4matmul_kernels_amd.adapters import LowRankAdapters
    from int4matmul_kernels_amd.quant_linear import QuantLinear
    torch.manual_seed(1)
    K, S, n = 512, 320, 4
    keep = None
    if sparse:
        keep = (torch.arange(K, device="cuda") % 2 == 0)[:, None].expand(K, S).contiguous()
    layer = QuantLinear.from_float((torch.randn((K, S), device="cuda") * 0.05).half(), bits, 64, keep, torch.randn(S, device="cuda").half())
    adapters = LowRankAdapters(n, 16, K, S)
    for i in range(n):
        adapters.set_adapter(i, torch.randn((4 + 4 * i, K), device="cuda").half() * 0.05, torch.randn((S, 4 + 4 * i), device="cuda").half() * 0.1, 0.5 + i)
    x = torch.randn((*shape, K), device="cuda").half()
    ids = torch.tensor([2, -1, 0, 3, 1, 7], dtype=torch.int32, device="cuda")[:shape[0]]
    got = layer(x, adapters, ids)
    bias, layer.bias = layer.bias, None
    base = layer(x)
    q = dict(base=base, x=x, down=adapters.down, up=adapters.up, scales=adapters.scales, ids=ids)
    term = adapters(base, x, ids)
    close(term, q)
    assert torch.equal(got, term + bias)
    flat = layer(x[:, 0], adapters, ids)
    assert flat.shape == (shape[0], S)
    with pytest.raises(ValueError):
        layer(x, adapters)
    with pytest.raises(ValueError):
        layer(x, adapter_ids=ids)
    with pytest.raises(ValueError):
        adapters.set_adapter(0, torch.zeros((17, K), device="cuda"), torch.zeros((S, 17), device="cuda"))
    with pytest.raises(IndexError):
        adapters.set_adapter(4, torch.zeros((4, K), device="cuda"), torch.zeros((S, 4), device="cuda"))


def test_refusals(ext):
    p = problem((4, 2), 3, 16)
    bad = [dict(ids=p["ids"].long()), dict(ids=p["ids"][:3]), dict(ids=p["ids"].cpu()), dict(x=p["x"][..., :128]), dict(base=p["base"][..., :128]),
           dict(base=p["base"].cpu()), dict(down=p["down"].float()), dict(up=p["up"][:2]), dict(up=p["up"].transpose(1, 2)), dict(scales=p["scales"].half()),
           dict(scales=p["scales"][:2]), dict(ids=torch.zeros((4, 2, 192), dtype=torch.int32, device="cuda")), dict(x=p["x"][:, 0]),
           dict(ids=torch.tensor(0, dtype=torch.int32, device="cuda"))]
    for change in bad:
        with pytest.raises(RuntimeError):
            add(ext, p, **change)
    for outs in (p["base"][:2], p["base"].float(), p["base"].transpose(0, 1)):
        with pytest.raises(RuntimeError):
            ext.low_rank_add(p["base"], p["x"], p["down"], p["up"], p["scales"], p["ids"], outs=outs)
    both = torch.zeros(4 * 2 * 192 + 64, dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError):                           # outs over a shifted base, over x
        ext.low_rank_add(both[:-64].reshape(4, 2, 192), p["x"], p["down"], p["up"], p["scales"], p["ids"], outs=both[64:].reshape(4, 2, 192))
    square = problem((4, 2), 3, 16, 192, 192)
    with pytest.raises(RuntimeError):
        ext.low_rank_add(square["base"], square["x"], square["down"], square["up"], square["scales"], square["ids"], outs=square["x"])
    with pytest.raises(RuntimeError):
        add(ext, problem((2, 1), 2, 513))
    with pytest.raises(RuntimeError):
        add(ext, problem((2, 1), 2, 8, 96, 64))
    with pytest.raises(RuntimeError, match="no backward"):
        add(ext, p, x=p["x"].clone().requires_grad_())


@pytest.mark.parametrize("rank", [5, 40, 130])
@pytest.mark.parametrize("T,n", [(300, 3), (1100, 30), (2500, 70), (4000, 250)])
def test_many_rows_with_ids_of_their_own(ext, T, n, rank):
    """random ids, one adapter for all rows but one, adapters without a row, no adapter at all; in place too"""
    p = problem((1, T), n, rank, 128, 192, per_row=True, seed=T)
    one = torch.full_like(p["ids"], n - 1)
    one[0, T // 2] = 0
    outside = torch.tensor([-1, n, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda").repeat(T)[:T].reshape(1, T)
    mixed = torch.where(torch.arange(T, device="cuda") % 3 == 0, outside, p["ids"] // 2)
    for ids in (p["ids"], one, mixed.to(torch.int32).contiguous()):
        q = dict(p, ids=ids)
        got = add(ext, q)
        close(got, dict(q, ids=torch.where((ids < 0) | (ids >= n), -1, ids)))
        base = p["base"].clone()
        ext.low_rank_add(base, p["x"], p["down"], p["up"], p["scales"], ids, base)
        assert torch.equal(base, got)
    assert torch.equal(add(ext, p, ids=outside), p["base"])


def test_many_rows_with_ids_of_their_own_captured(ext):
    a, b = problem((900, 1), 12, 16, seed=1), problem((900, 1), 12, 16, seed=2)
    b.update({n: a[n] for n in ("down", "up", "scales")})
    held = {n: a[n].clone() for n in ("base", "x", "ids")}
    want = {id(q): add(ext, q) for q in (a, b)}
    close(want[id(a)], a)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(add(ext, a, **held))
    for q in (a, b, a, b):
        for n in held:
            held[n].copy_(q[n])
        for g in graphs:
            g.replay()
        eager = add(ext, q)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[id(q)]) and all(torch.equal(o, eager) for o in outs)


def test_rows_in_order_leave_what_lies_behind(ext):
    from int4matmul_kernels_amd import capi
    p = problem((500, 1), 9, 20, seed=7)
    outs = torch.full((520, 192), 7.0, dtype=torch.float16, device="cuda")
    ws = capi.new_adapters_workspace(500, 1, p["down"], p["up"])
    ws.fill_(255)
    capi.low_rank_add(outs[:500], p["base"][:, 0], p["x"][:, 0], p["down"], p["up"], p["scales"], p["ids"], 1, ws)
    assert torch.equal(outs[:500], add(ext, p)[:, 0]) and torch.all(outs[500:] == 7)
    with pytest.raises(capi.Int4mmError) as e:
        capi.low_rank_add(outs[:500], p["base"][:, 0], p["x"][:, 0], p["down"], p["up"], p["scales"], p["ids"], 1, ws[:-16])
    assert e.value.code == 6


def test_outs_over_scales_or_ids_is_refused(ext):
    p = problem((4, 2), 1024, 1, 64, 64)
    raw = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    outs = raw[:1024].view(torch.float16).reshape(4, 2, 64)
    scales = raw.view(torch.float32)[:1024]
    with pytest.raises(RuntimeError):
        ext.low_rank_add(p["base"], p["x"], p["down"], p["up"], scales, p["ids"], outs=outs)
    ids = raw.view(torch.int32)[:4]
    with pytest.raises(RuntimeError):
        ext.low_rank_add(p["base"], p["x"], p["down"], p["up"], p["scales"], ids, outs=outs)


@pytest.mark.parametrize("rank", [480, 481, 512])
@pytest.mark.parametrize("shape,per_row,n", [((3, 401), False, 3), ((1, 1203), True, 9), ((1, 1025), True, 1)])
def test_highest_ranks_with_many_rows(ext, rank, shape, per_row, n):
    """tiles of 32 rows whose x down^T takes more than 64 KB of LDS"""
    p = problem(shape, n, rank, 128, 320, per_row=per_row, seed=rank)
    close(add(ext, p), p)
    if rank == 512:
        held, graph = {k: v.clone() for k, v in p.items()}, torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = add(ext, held)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, add(ext, p))


@pytest.mark.parametrize("rank", [16, 20, 33, 64, 100, 200, 512])
@pytest.mark.parametrize("shape,n", [((3, 401), 4), ((5, 333), 2), ((70, 17), 9), ((2, 1024), 3)])
def test_prompts_of_many_rows(ext, rank, shape, n):
    """an id per request and more than 1024 rows: tiles of 32 rows that several requests share, idle ones among them, a last tile that is
    not full; in place too"""
    p = problem(shape, n, rank, 192, 320, seed=rank)
    p["ids"][-1] = n - 1
    p["ids"][1] = -1
    got = add(ext, p)
    close(got, p)
    assert torch.equal(got[1], p["base"][1])
    base = p["base"].clone()
    ext.low_rank_add(base, p["x"], p["down"], p["up"], p["scales"], p["ids"], base)
    assert torch.equal(base, got)


def test_outs_that_ask_for_a_gradient_are_refused(ext):
    p = problem((4, 2), 3, 16)
    outs = torch.zeros_like(p["base"]).requires_grad_()
    for o in (outs, outs * 1):
        with pytest.raises(RuntimeError, match="no backward"):
            ext.low_rank_add(p["base"], p["x"], p["down"], p["up"], p["scales"], p["ids"], outs=o)
    assert not outs.any()
    with torch.no_grad():
        ext.low_rank_add(p["base"], p["x"], p["down"], p["up"], p["scales"], p["ids"], outs=outs)
    assert torch.equal(outs, add(ext, p))


def test_outs_that_a_backward_pass_has_kept(ext):
    """writing into a tensor that autograd keeps for a gradient: the backward pass refuses, as after torch's own in-place operations"""
    p = problem((4, 2), 3, 16)
    outs, w = p["base"].clone(), torch.ones(1, dtype=torch.float16, device="cuda", requires_grad=True)
    loss = (outs * w).sum()
    ext.low_rank_add(p["base"], p["x"], p["down"], p["up"], p["scales"], p["ids"], outs=outs)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        kept = torch.empty_like(outs)
        ext.low_rank_add(p["base"], p["x"], p["down"], p["up"], p["scales"], p["ids"], outs=kept)
    assert torch.equal(kept, outs)


@pytest.mark.parametrize("dtype,apart,copies", [(torch.float16, False, 0), (torch.float32, False, 1), (torch.bfloat16, False, 1), (torch.float16, True, 1)])
def test_states_are_converted_once(dtype, apart, copies):
    """a layer with its adapters makes one fp16 copy of states that are not fp16 and contiguous"""
    from torch.utils._python_dispatch import TorchDispatchMode
    from int4matmul_kernels_amd.adapters import LowRankAdapters
    from int4matmul_kernels_amd.quant_linear import QuantLinear

    class Copies(TorchDispatchMode):
        seen = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen += func.name() in ("aten::_to_copy", "aten::clone")
            return func(*args, **(kwargs or {}))

    torch.manual_seed(2)
    layer, adapters = QuantLinear.from_float((torch.randn((128, 64), device="cuda") * 0.05).half(), 4, 64), LowRankAdapters(2, 4, 128, 64)
    adapters.set_adapter(0, torch.randn((4, 128), device="cuda").half() * 0.1, torch.randn((64, 4), device="cuda").half())
    ids = torch.tensor([0, -1, 0], dtype=torch.int32, device="cuda")
    for shape in ((3, 128), (3, 5, 128)):
        x = torch.randn((*shape[:-1], 256), device="cuda").to(dtype)[..., ::2] if apart else torch.randn(shape, device="cuda").to(dtype)
        with Copies() as mode:
            got = layer(x, adapters, ids)
        assert torch.equal(got, layer(x.half().contiguous(), adapters, ids)) and mode.seen == copies
