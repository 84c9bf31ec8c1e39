"""Refusals of the operators around the collectives: everything that depends on arguments only is
refused before any HIP call, at the C boundary and by the tensor front end."""
import ctypes

import pytest
import torch

vp = ctypes.c_void_p


@pytest.fixture()
def abi(mccl):
    from torch_ccl_amd import capi
    L = capi.lib()
    return L, capi, lambda: L.mccl_last_error().decode()


def test_embedding_refusals(abi):
    L, capi, err = abi

    def call(table=0x10000000, rows=10, ids=0x20000000, idt=capi.I64, n=4, first=0, hidden=64, dtype=capi.BF16, out=0x30000000):
        return L.mccl_embedding(vp(table), rows, vp(ids), idt, n, first, hidden, 1.0, dtype, vp(out), None)

    assert call(dtype=capi.I32) == -3 and "bf16, f16 and f32" in err()
    assert call(dtype=99) == -3
    assert call(idt=capi.F32) == -3 and "int32 or int64" in err()
    assert call(n=0) == 0 and call(hidden=0) == 0
    assert call(ids=0) == -1 and "id pointer is null" in err()
    assert call(ids=0x20000004) == -1 and "ids not aligned" in err()
    assert call(table=0) == -1 and "null" in err()
    assert call(out=0) == -1 and "null" in err()
    assert call(out=0x30000001) == -1 and "not aligned" in err()
    assert call(table=0x10000002, dtype=capi.F32) == -1 and "not aligned" in err()
    assert call(hidden=1 << 24) == -1 and "too long" in err()
    assert call(n=1 << 31) == -1 and "too long" in err()
    assert call(out=0x10000000 + 64) == -1 and "overlaps" in err()
    assert call(out=0x20000000 - 8) == -1 and "overlaps" in err()


def test_sort_refusals(abi):
    L, capi, err = abi

    def call(ids=0x10000000, idt=capi.I64, n=4, rows=10, ws=0, wsb=0, order=0x20000000, offsets=0x30000000):
        return L.mccl_sort_ids(vp(ids), idt, n, 0, rows, vp(ws), wsb, vp(order), vp(offsets), None)

    assert call(idt=capi.I16) == -3
    assert call(n=1 << 31) == -1 and "too many ids" in err()
    assert call(rows=1 << 31) == -1 and "too many rows" in err()
    assert call(ids=0) == -1 and "null" in err()
    assert call(order=0) == -1 and "order" in err()
    assert call(order=0x20000004) == -1 and "order" in err()
    assert call(offsets=0) == -1 and "offsets" in err()
    assert L.mccl_sort_ids_workspace(100) == 0
    need = L.mccl_sort_ids_workspace(100000)
    assert need >= 100000 * 16
    assert call(n=100000) == -1 and "workspace" in err()
    assert call(n=100000, order=0x20000000, offsets=0x30000000, ws=0x40000008, wsb=need) == -1 and "workspace" in err()
    assert call(n=100000, ws=0x40000000, wsb=need - 1) == -1 and "workspace" in err()
    assert call(n=100000, ws=0x20000010, wsb=need) == -1 and "overlap" in err()
    assert call(offsets=0x20000008) == -1 and "overlap" in err()


def test_embedding_grad_refusals(abi):
    L, capi, err = abi

    def call(grad=0x10000000, order=0x20000000, offsets=0x21000000, n=4, rows=10, hidden=64, dtype=capi.BF16, out=0x30000000, odt=capi.BF16,
             ws=0, wsb=0):
        return L.mccl_embedding_grad(vp(grad), vp(order), vp(offsets), n, rows, hidden, 1.0, dtype, vp(out), odt, 0, vp(ws), wsb, None)

    assert call(dtype=capi.I32) == -3
    assert call(odt=capi.F16) == -3 and "same type or f32" in err()
    assert call(dtype=capi.F32) == -3
    assert call(rows=0) == 0 and call(hidden=0) == 0
    assert call(grad=0) == -1 and call(order=0) == -1 and call(offsets=0) == -1 and call(out=0) == -1 and "null" in err()
    assert call(grad=0x10000001) == -1 and "aligned" in err()
    assert call(order=0x20000004) == -1 and "misaligned" in err()
    assert call(n=(1 << 28) + 1) == -1 and "too long" in err()
    need = L.mccl_embedding_grad_workspace(1000, 64)
    assert need >= 16 * 2 * 64 * 4 and L.mccl_embedding_grad_workspace(64, 64) == 0
    assert call(n=1000) == -1 and "workspace" in err()
    assert call(n=1000, ws=0x40000000, wsb=need - 4) == -1 and "workspace" in err()
    assert call(out=0x10000000 + 8) == -1 and "overlaps an input" in err()
    assert call(n=1000, ws=0x30000000, wsb=need) == -1 and "overlaps the workspace" in err()


def test_router_refusals(abi):
    L, capi, err = abi

    def route(logits=0x10000000, T=4, E=16, k=2, dtype=capi.F32, ids=0x20000000, w=0x30000000):
        return L.mccl_moe_route(vp(logits), T, E, k, 1, dtype, vp(ids), vp(w), None)

    def grad(g=0x20000000, logits=0x10000000, ids=0x30000000, T=4, E=16, k=2, dtype=capi.F32, out=0x40000000):
        return L.mccl_moe_route_grad(vp(g), vp(logits), vp(ids), T, E, k, 1, dtype, vp(out), None)

    for call in (route, grad):
        assert call(dtype=capi.F64) == -3 and "bf16, f16 and f32" in err()
        assert call(E=0) == -1 and call(E=4097) == -1 and "expert count" in err()
        assert call(k=0) == -1 and call(k=17) == -1 and call(E=100, k=65) == -1 and "topk" in err()
        assert call(T=1 << 31) == -1 and "too many tokens" in err()
        assert call(T=0) == 0
        assert call(logits=0) == -1 and "null" in err()
        assert call(logits=0x10000002) == -1 and "aligned" in err()
        assert call(ids=0x20000002) == -1 and "aligned" in err()
    assert route(ids=0x10000010) == -1 and "overlap" in err()
    assert route(w=0x20000004) == -1 and "overlap" in err()
    assert grad(out=0x10000000) == -1 and "overlaps" in err()
    assert grad(out=0x30000000) == -1 and "overlaps" in err()


def test_layer_refusals(abi):
    L, capi, err = abi

    def call(x=0x10000000, w_in=0x100000000, w_out=0x200000000, ids=0x20000000, w=0x21000000, T=4, k=2, E=8, first=0, H=64, I=32,
             act=capi.ACT_SILU, dtype=capi.BF16, out=0x30000000, ws=0x40000000, wsb=1 << 24):
        return L.mccl_moe_layer(vp(x), vp(w_in), vp(w_out), vp(ids), vp(w), T, k, E, first, H, I, act, dtype, vp(out), vp(ws), wsb, None)

    assert call(dtype=capi.F32) == -3 and "bf16 and f16" in err()
    assert call(act=2) == -1 and "activation" in err()
    assert call(T=257) == -3 and "at most 256" in err()
    assert call(k=0) == -1 and call(k=65) == -1 and call(T=256, k=17) == -1 and "topk" in err()
    assert call(E=0) == -1 and call(E=5000) == -1 and "expert count" in err()
    assert call(T=0) == 0
    assert call(H=60) == -3 and call(I=12) == -3 and call(I=0) == -3 and "multiples of 8" in err()
    assert call(x=0) == -1 and call(w_in=0) == -1 and call(w_out=0) == -1 and call(ids=0) == -1 and call(w=0) == -1 and call(out=0) == -1
    assert "null" in err()
    assert call(x=0x10000008) == -1 and "16-byte aligned" in err()
    assert call(w_out=0x200000002) == -1 and "16-byte aligned" in err()
    assert call(ids=0x20000002) == -1 and "misaligned" in err()
    assert call(H=(1 << 17) + 8) == -1 and call(I=(1 << 17) + 8) == -1 and call(H=1 << 17, I=1 << 12) == -1 and "w_in above" in err()
    assert call(H=1 << 14, I=1 << 15) == -1 and "w_in above" in err()  # 2 GiB
    assert call(T=256, k=16, E=4096, H=8, I=1 << 17) == -1 and "too many rows" in err()
    for sizes in ((0, 2, 8, 64, 32), (100, 0, 8, 64, 32), (100, 8, 0, 64, 32), (100, 8, 4, 0, 32), (100, 8, 4, 64, 0)):
        assert L.mccl_moe_layer_workspace(*sizes) == 0
    assert call(T=100, k=8, E=4, H=0) == 0 and call(T=100, k=8, E=4, I=0) == -3
    need = L.mccl_moe_layer_workspace(4, 2, 8, 64, 32)
    assert need > 0 and call(ws=0) == -1 and call(wsb=need - 1) == -1 and call(ws=0x40000008) == -1 and "workspace" in err()
    assert call(out=0x10000000) == -1 and "overlaps an input" in err()
    assert call(ws=0x200000000) == -1 and "overlaps an input" in err()
    assert call(out=0x40000000) == -1 and "overlaps the workspace" in err()


def test_the_front_end_refuses_what_it_is_not_for(mccl):
    f, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        mccl.embedding(f, i)
    with pytest.raises(RuntimeError, match="bf16, f16 or f32"):
        mccl.embedding(f.double(), i)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        mccl.embedding(f, i.to(torch.int16))
    with pytest.raises(RuntimeError, match="out must be"):
        mccl.embedding(f, i, out=torch.zeros(4, 9))
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        mccl.sort_ids(i, 4)
    with pytest.raises(RuntimeError, match="negative row count"):
        mccl.sort_ids(i, -1)
    plan = (torch.arange(4), torch.tensor([0, 2, 4]))
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        mccl.embedding_grad(f, plan)
    with pytest.raises(RuntimeError, match="one row per sorted id"):
        mccl.embedding_grad(f[:3], plan)
    with pytest.raises(RuntimeError, match="accumulate needs"):
        mccl.embedding_grad(f, plan, accumulate=True)
    with pytest.raises(RuntimeError, match="order must be int64"):
        mccl.embedding_grad(f, (plan[0].int(), plan[1]))
    with pytest.raises(RuntimeError, match="out must be float32"):
        mccl.embedding_grad(f, plan, out=torch.zeros(2, 8, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        mccl.moe_route(f, 2)
    with pytest.raises(RuntimeError, match="topk must be positive"):
        mccl.moe_route(f, 0)
    with pytest.raises(RuntimeError, match="grad_weights must be float32"):
        mccl.moe_route_grad(torch.zeros(4, 3), f, torch.zeros(4, 2, dtype=torch.int32))
    x, w_in, w_out = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(3, 32, 8, dtype=torch.bfloat16), torch.zeros(3, 8, 16, dtype=torch.bfloat16)
    ids, w = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        mccl.moe_layer(x, w_in, w_out, ids, w)
    with pytest.raises(RuntimeError, match="activation must be one of gelu, silu"):
        mccl.moe_layer(x, w_in, w_out, ids, w, activation="tanh")
    with pytest.raises(RuntimeError, match="w_in must be bfloat16 of shape"):
        mccl.moe_layer(x, w_in[:, :30], w_out, ids, w)
    with pytest.raises(RuntimeError, match="weights must be float32 of shape"):
        mccl.moe_layer(x, w_in, w_out, ids, w[:, :1])
    with pytest.raises(RuntimeError, match="bf16 or f16"):
        mccl.moe_layer(x.float(), w_in, w_out, ids, w)


def test_rows_past_the_largest_id_are_refused(abi):
    """Their row numbers would wrap around to the smallest ids."""
    L, capi, err = abi
    last = (1 << 63) - 1

    def embedding(first, rows, n=4):
        return L.mccl_embedding(vp(0x10000000), rows, vp(0x20000000), capi.I64, n, first, 64, 1.0, capi.BF16, None, None)

    def sort(first, rows):
        return L.mccl_sort_ids(vp(0x10000001), capi.I64, 4, first, rows, None, 0, vp(0x20000000), vp(0x30000000), None)

    for call, fits in ((embedding, "null"), (sort, "ids not aligned")):
        for first, rows in ((last, 2), (last - 3, 5), (1, 1 << 63), (last // 2 + 2, last // 2 + 1)):
            if call is sort and rows > 0x7fffffff:
                continue
            assert call(first, rows) == -1 and "pass 2^63" in err()
        for first, rows in ((last, 1), (last - 3, 4), (last, 0), (-1, 10), (-last - 1, 10)):
            assert call(first, rows) == -1 and fits in err()  # refused for something else that comes later
