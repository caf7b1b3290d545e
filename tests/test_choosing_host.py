"""Products whose rows choose their weights, without a GPU: the C interface refuses bad arguments before it touches the
device, the extension tensors that are not on one, the modules what no call could serve."""
import ctypes as C

import pytest
import torch

import int4matmul_kernels_amd as pkg
from int4matmul_kernels_amd import capi
from int4matmul_kernels_amd.adapters import LowRankAdapters
from int4matmul_kernels_amd.quant_experts import ExpertRouter, QuantExperts

VP = C.c_void_p
OK = 0x1000


def test_route_arguments():
    lib = capi.lib()

    def call(weights=OK, ids=OK, logits=OK, bias=None, **change):
        fields = dict(tokens=4, experts=64, top_k=8, groups=1, topk_groups=1, scoring=0, group_score=0, renormalize=1, logits_bytes=2, scale=1.0)
        fields.update(change)
        return lib.int4mm_route_experts(VP(weights), VP(ids), VP(logits), VP(bias), C.byref(capi.RouteShape(**fields)), None)

    assert call(tokens=0) == 0 and call(tokens=0, logits=None) == 0
    for change in (dict(tokens=-1), dict(experts=0), dict(experts=1025), dict(top_k=0), dict(top_k=65, experts=128), dict(top_k=65), dict(groups=3),
                   dict(groups=0), dict(groups=128, experts=128), dict(groups=8, topk_groups=9), dict(groups=8, topk_groups=0),
                   dict(groups=16, topk_groups=1), dict(scoring=2), dict(group_score=-1), dict(logits_bytes=8), dict(scale=float("nan"))):
        assert call(**change) == 3, change
    for change in (dict(weights=None), dict(ids=None), dict(logits=None)):
        assert call(**change) == 5, change
    for change in (dict(weights=OK + 2), dict(ids=OK + 1), dict(logits=OK + 1), dict(logits=OK + 2, logits_bytes=4), dict(bias=OK + 2)):
        assert call(**change) == 8, change
    assert lib.int4mm_route_experts(VP(OK), VP(OK), VP(OK), None, None, None) == 5


def test_experts_arguments():
    lib = capi.lib()

    def call(bits=4, masks=(None, None), at=None, value=None, ws=OK, ws_bytes=1 << 40, **change):
        sh = capi.experts_shape(change.pop("tokens", 4), change.pop("top_k", 2), change.pop("experts", 8), change.pop("in_size", 256),
                                change.pop("width", 128), change.pop("group_size", 64))
        for name, v in change.items():
            setattr(sh, name, v)
        ptrs = [OK] * 12
        ptrs[7], ptrs[11] = masks
        if at is not None:
            ptrs[at] = value
        return lib.int4mm_experts_forward(bits, *map(VP, ptrs), C.byref(sh), VP(ws), ws_bytes, None)

    assert call(tokens=0) == 0
    assert call(bits=5) == 1 and call(bits=3, masks=(OK, OK)) == 2
    for change in (dict(tokens=-1), dict(top_k=0), dict(experts=0), dict(in_size=96), dict(width=96), dict(width=0), dict(up_groups=3), dict(down_groups=3),
                   dict(experts=4097), dict(tokens=1 << 31), dict(top_k=1025), dict(in_size=1 << 32), dict(in_size=1 << 16, width=1 << 15)):
        assert call(**change) == 3, change
    for g in (0, 32, 96):
        sh = capi.experts_shape(4, 2, 8, 256, 128, 64)
        sh.group_size = g
        assert lib.int4mm_experts_forward(4, *[VP(OK)] * 7, None, *[VP(OK)] * 3, None, C.byref(sh), VP(OK), 1 << 40, None) == 4, g
    for i in (0, 1, 2, 3, 4, 5, 6, 8, 9, 10):
        assert call(at=i, value=None) == 5, i
    for i in (0, 1, 4, 5, 6, 8, 9, 10):
        assert call(at=i, value=OK + 8) == 8, i
    for i in (2, 3):
        assert call(at=i, value=OK + 2) == 8, i
    assert call(masks=(OK, None)) == 5 and call(masks=(None, OK)) == 5
    assert call(ws=None) == 6 and call(ws_bytes=100) == 6 and call(ws=OK + 4) == 8
    assert lib.int4mm_experts_forward(4, *[VP(OK)] * 12, None, VP(OK), 1 << 40, None) == 5


def test_adapter_arguments():
    lib = capi.lib()

    def call(at=None, value=None, ws=OK, ws_bytes=1 << 40, **change):
        fields = dict(rows=4, rows_per_id=1, adapters=3, rank=16, in_size=256, out_size=128)
        fields.update(change)
        ptrs = [OK] * 7
        if at is not None:
            ptrs[at] = value
        return lib.int4mm_low_rank_add(*map(VP, ptrs), C.byref(capi.AdapterShape(**fields)), VP(ws), ws_bytes, None)

    assert call(rows=0) == 0
    for change in (dict(rows=-1), dict(rows=1 << 21), dict(rows_per_id=0), dict(adapters=0), dict(rank=0), dict(rank=513), dict(in_size=96), dict(out_size=96),
                   dict(in_size=0), dict(out_size=0), dict(in_size=1 << 30), dict(out_size=1 << 27), dict(adapters=1 << 31)):
        assert call(**change) == 3, change
    for i in range(7):
        assert call(at=i, value=None) == 5, i
        assert call(at=i, value=OK + 2) == 8, i
    assert call(ws=None) == 6 and call(ws_bytes=16) == 6 and call(ws=OK + 4) == 8
    assert lib.int4mm_low_rank_add(*[VP(OK)] * 7, None, VP(OK), 1 << 40, None) == 5


def test_extension_needs_a_gpu():
    ext = pkg.load_extension()
    with pytest.raises(RuntimeError):
        ext.route_experts(torch.zeros((2, 8)), 2)
    x, i, w = torch.zeros((2, 64), dtype=torch.float16), torch.zeros((2, 1), dtype=torch.int32), torch.zeros((2, 1))
    m, s = torch.zeros((1, 8, 128), dtype=torch.int32), torch.zeros((1, 1, 128), dtype=torch.float16)
    with pytest.raises(RuntimeError):
        ext.experts_forward(4, x, w, i, m, s, s, m, s, s, 64)
    a = torch.zeros((1, 4, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError):
        ext.low_rank_add(x, x, a, a, torch.zeros(1), torch.zeros(2, dtype=torch.int32))


def test_modules_refuse():
    for how in (dict(n_experts=0, top_k=1), dict(n_experts=8, top_k=9), dict(n_experts=8, top_k=2, n_groups=3), dict(n_experts=8, top_k=5, n_groups=2),
                dict(n_experts=8, top_k=2, scoring="relu"), dict(n_experts=8, top_k=2, group_score="mean"), dict(n_experts=1025, top_k=2)):
        with pytest.raises(ValueError):
            ExpertRouter(device="cpu", **how)
    for how in (dict(bits=5, n_experts=2, features=64, width=64), dict(bits=3, n_experts=2, features=64, width=64, sparse=True),
                dict(bits=4, n_experts=2, features=96, width=64), dict(bits=4, n_experts=0, features=64, width=64),
                dict(bits=4, n_experts=2, features=64, width=64, group_size=96)):
        with pytest.raises(ValueError):
            QuantExperts(device="cpu", **how)
    for how in ((0, 4, 64, 64), (2, 0, 64, 64), (2, 513, 64, 64), (2, 4, 65, 64)):
        with pytest.raises(ValueError):
            LowRankAdapters(*how, device="cpu")


def test_experts_grids():
    """a grid has fewer than 2^32 work-items: so many pairs go through in shares, and a token that is too much by itself is refused"""
    lib = capi.lib()

    def call(*shape):
        ptrs = [OK] * 12
        ptrs[7] = ptrs[11] = None
        sh = capi.experts_shape(*shape)
        return lib.int4mm_experts_forward(4, *map(VP, ptrs), C.byref(sh), VP(OK), 0, None), lib.int4mm_experts_workspace_bytes(C.byref(sh))

    # (no workspace is given: 6 is an accepted shape)
    widest = (1 << 24) - 64
    assert call(1, 64, 128, 64, widest, -1) == (3, 0) and call(7, 17, 128, 64, widest, -1) == (3, 0)
    assert call(1, 16, 128, 64, widest, -1)[0] == 6 and call(7, 16, 128, 64, widest, -1)[0] == 6
    # 1000 tokens, one of 4096 experts each, 32768 strips of columns: 256 work-items for each, 8.6e9 in one grid
    code, size = call(1000, 1, 4096, 64, 1 << 20, -1)
    assert code == 6 and size < 256 * 2 ** 21 * 1.01
    # ordinary ones are not cut: the hidden states of all pairs, their sums, and a little
    for T, k, E, K, F in ((4096, 8, 64, 2048, 1024), (8192, 2, 8, 4096, 14336), (32768, 8, 256, 7168, 2048), (2048, 4, 16, 4096, 32768)):
        code, size = call(T, k, E, K, F, 128)
        assert code == 6 and T * k * (2 * F + 4 * K) < size < 1.02 * T * k * (2 * F + 4 * K + 8) + 2 ** 20


def test_half_leaves_fp32_buffers():
    """a model turned to fp16 keeps the scales of its adapters and the bias of its router"""
    router, adapters = ExpertRouter(8, 2, bias=True, device="cpu"), LowRankAdapters(3, 4, 64, 64, device="cpu")
    router.bias.copy_(torch.linspace(-1, 1, 8) / 3)
    adapters.scales.copy_(torch.tensor([1 / 3, 1e-9, 1e9]))
    bias, scales = router.bias.clone(), adapters.scales.clone()
    model = torch.nn.Sequential(router, adapters, ExpertRouter(8, 2, device="cpu"))
    for turned in (model.half(), model.to(torch.float16), model.to("cpu", torch.float16), model.cpu()):
        assert turned is model and turned[0] is router and turned[1] is adapters
        assert router.bias.dtype == adapters.scales.dtype == torch.float32
        assert torch.equal(router.bias, bias) and torch.equal(adapters.scales, scales)
        assert adapters.down.dtype == adapters.up.dtype == torch.float16
    assert set(model.state_dict()) == {"0.bias", "1.down", "1.up", "1.scales"}
    assert model.to("meta")[1].scales.is_meta and model[0].bias.dtype == torch.float32
