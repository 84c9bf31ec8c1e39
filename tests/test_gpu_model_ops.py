"""The operators that compute around the collectives, against plain implementations in 64 bits:
embedding and its gradient by sorted tokens, the router and its gradient, the mixture-of-experts layer
for a few tokens, and runs of them together with the collectives' own calls.

Tolerances count roundings: u = 2^-24 per fp32 operation, eps / 2 for the one rounding to the output's
type, times the sums of absolute values that the roundings act on."""
import ctypes
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
FLOATS = [torch.bfloat16, torch.float16, torch.float32]


def gen(*key):
    return torch.Generator().manual_seed(hash(tuple(int(k) for k in key)) % (1 << 31))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, want, tol, what=""):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = tuple(int(v) for v in torch.nonzero(bad)[0])
        raise AssertionError("%s: %d of %d off; first at %s: got %r want %r tolerance %r" % (
            what, int(bad.sum()), bad.numel(), i, float(got[i]), float(want[i]), float(torch.as_tensor(tol).expand_as(want)[i])))


def keys_of(ids, first, rows):
    r = ids.long() - first
    return torch.where((r >= 0) & (r < rows), r, torch.full_like(r, rows))


# ---------------------------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("n,rows,hidden,first", [(1, 1, 1, 0), (3, 7, 5, 0), (8, 100, 64, 40), (257, 50, 521, -3), (1000, 333, 4096, 5),
                                                 (33, 10, 7168, 0), (5, 3, 8 * 64 * 4 + 7, 1)])
@pytest.mark.parametrize("id_dtype", [torch.int32, torch.int64], ids=str)
def test_embedding_is_the_scaled_row_or_zero(mccl, dtype, id_dtype, n, rows, hidden, first):
    """Bit for bit: one fp32 product, one rounding.  Ids below, above and far outside the shard give zeros."""
    g = gen(n, rows, hidden, first)
    table = torch.randn(rows, hidden, generator=g).to(dtype)
    ids = torch.randint(first - 2, first + rows + 2, (n,), generator=g)
    info = torch.iinfo(id_dtype)
    for i, v in enumerate((info.min, info.max, -1)):
        if i + 1 < n:
            ids[i + 1] = v
    scale = 1.0 / 3.0
    out = mccl.embedding(table.to(DEV), ids.to(id_dtype).to(DEV), scale=scale, first_row=first)
    key = torch.tensor([int(v) - first if 0 <= int(v) - first < rows else rows for v in ids])
    padded = torch.cat([table, torch.zeros(1, hidden, dtype=dtype)])
    want = (padded[key].float() * torch.tensor(scale, dtype=torch.float32)).to(dtype)
    assert out.dtype == dtype and torch.equal(out.cpu(), want)


@pytest.mark.parametrize("src_off,dst_off", [(1, 0), (0, 3), (5, 1)])
@pytest.mark.parametrize("hidden", [8, 24, 33, 1024])
def test_embedding_at_any_alignment_leaves_the_neighbours_alone(mccl, src_off, dst_off, hidden):
    g = gen(src_off, dst_off, hidden)
    rows, n, dtype = 19, 40, torch.bfloat16
    table = torch.randn(src_off + rows * hidden, generator=g).to(dtype).to(DEV)
    buf = torch.full((dst_off + n * hidden + 40,), 7.0, dtype=dtype, device=DEV)
    t, o = table[src_off:].view(rows, hidden), buf[dst_off:dst_off + n * hidden].view(n, hidden)
    ids = torch.randint(0, rows, (n,), generator=g).to(DEV)
    mccl.embedding(t, ids, out=o)
    assert torch.equal(o, t[ids])
    assert bool((buf[:dst_off] == 7).all()) and bool((buf[dst_off + n * hidden:] == 7).all())


def test_embedding_shapes_empty_lists_and_an_empty_shard(mccl):
    table = torch.randn(6, 16, generator=gen(1)).to(DEV)
    ids = torch.tensor([[0, 5], [9, -1]], device=DEV)
    out = mccl.embedding(table, ids)
    assert out.shape == (2, 2, 16) and torch.equal(out[0], table[[0, 5]]) and not out[1].any()
    assert mccl.embedding(table, ids[:0]).shape == (0, 2, 16)
    assert not mccl.embedding(table[:0], ids).any()


def test_embedding_of_values_that_are_not_finite(mccl):
    table = torch.tensor([[float("inf"), float("-inf"), float("nan"), 3e38]] * 2, device=DEV)
    out = mccl.embedding(table, torch.tensor([1, 7], device=DEV), scale=2.0).cpu()
    assert out[0, 0] == float("inf") and out[0, 1] == float("-inf") and out[0, 2].isnan() and out[0, 3] == float("inf")
    assert not out[1].any()


def test_embedding_rows_past_4_gib(mccl):
    """Offsets that need more than 32 bits, in the table and in the output."""
    hidden = 8192
    rows = (5 << 30) // (2 * hidden)
    table = torch.zeros(rows, hidden, dtype=torch.bfloat16, device=DEV)
    marks = torch.arange(1, 9, device=DEV, dtype=torch.bfloat16)
    at = torch.tensor([0, 1, rows // 2, rows - 3, rows - 2, rows - 1, rows // 3, 5], device=DEV)
    table[at] = marks[:, None].expand(8, hidden)
    n = rows + 11
    ids = torch.full((n,), 2, device=DEV)
    ids[torch.arange(0, 8, device=DEV) * ((n - 1) // 7)] = at
    out = mccl.embedding(table, ids)
    assert torch.equal(out[torch.arange(0, 8, device=DEV) * ((n - 1) // 7), -1], marks)
    assert int((out[:, 0] != 0).sum()) == 8


# ---------------------------------------------------------------------------------------------
# sort
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [0, 1, 2, 64, 255, 256, 257, 2047, 2048, 2049, 4096, 5000, 65537, 196_608, 196_609, 1_000_003])
@pytest.mark.parametrize("rows,first", [(1, 0), (8, -2), (255, 0), (256, 1), (50_000, 10), (3_000_000, 0)])
def test_sort_ids_is_the_stable_order(mccl, n, rows, first):
    g = gen(n, rows)
    ids = torch.randint(first - 1 - rows // 8, first + rows + 2 + rows // 8, (n,), generator=g)
    if n > 100:
        ids[torch.rand(n, generator=g) < 0.3] = first + rows // 2
    order, offsets = mccl.sort_ids(ids.to(torch.int32).to(DEV) if n % 2 else ids.to(DEV), rows, first_row=first)
    key = keys_of(ids, first, rows)
    in_order, want = torch.sort(key, stable=True)
    assert torch.equal(order.cpu(), want)
    assert torch.equal(offsets.cpu(), torch.searchsorted(in_order, torch.arange(rows + 1)))


def test_sort_ids_without_rows_and_with_far_ids(mccl):
    info = torch.iinfo(torch.int64)
    ids = torch.tensor([info.max, 5, info.min, 4, 5, -1], device=DEV)
    order, offsets = mccl.sort_ids(ids, 0)
    assert order.tolist() == [0, 1, 2, 3, 4, 5] and offsets.tolist() == [0]
    order, offsets = mccl.sort_ids(ids, 2, first_row=4)
    assert order.tolist() == [3, 1, 4, 0, 2, 5] and offsets.tolist() == [0, 1, 3]
    order, offsets = mccl.sort_ids(ids, 4, first_row=info.min)  # a range at the very end of the type
    assert order.tolist() == [2, 0, 1, 3, 4, 5] and offsets.tolist() == [0, 1, 1, 1, 1]


# ---------------------------------------------------------------------------------------------
# embedding gradient
# ---------------------------------------------------------------------------------------------
def grad_reference(grad, ids, first, rows, scale):
    """(sum, tolerance of the fp32 sum): m terms, at most m roundings of partial sums of the absolute
    values, one of the scaling."""
    key = keys_of(ids, first, rows)
    inside = key < rows
    total = torch.zeros(rows, grad.shape[1], dtype=torch.float64)
    size, count = torch.zeros_like(total), torch.zeros(rows, 1, dtype=torch.float64)
    total.index_add_(0, key[inside], grad[inside].double())
    size.index_add_(0, key[inside], grad[inside].double().abs())
    count.index_add_(0, key[inside], torch.ones(int(inside.sum()), 1, dtype=torch.float64))
    s = float(torch.tensor(scale, dtype=torch.float32))
    return total * s, (count + 1) * U * size * abs(s)


@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                             (torch.float16, torch.float32), (torch.float32, torch.float32)], ids=str)
@pytest.mark.parametrize("n,rows,hidden,hot", [(0, 5, 16, 0.0), (1, 1, 1, 0.0), (64, 3, 40, 1.0), (65, 3, 40, 1.0), (128, 2, 7, 0.5),
                                               (1000, 40, 521, 0.6), (3000, 500, 264, 0.2), (700, 20, 2056, 0.3), (9000, 7, 130, 0.0),
                                               (9000, 7000, 2056, 0.1)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_grad(mccl, dtype, out_dtype, n, rows, hidden, hot, accumulate):
    """Rows without a token, with one, with more than one piece of the sorted tokens holds, and rows that
    begin and end inside a piece; added into a gradient or written over one that holds NaN."""
    g = gen(n, rows, hidden, int(accumulate))
    grad = torch.randn(n, hidden, generator=g).to(dtype)
    first, scale = 3, 1.5 if n % 2 else 1.0 / 3.0
    ids = torch.randint(first - 1, first + rows + 1, (n,), generator=g)
    ids[torch.rand(n, generator=g) < hot] = first + rows // 2
    old = torch.randn(rows, hidden, generator=g).to(out_dtype) if accumulate else torch.full((rows, hidden), float("nan"), dtype=out_dtype)
    plan = mccl.sort_ids(ids.to(DEV), rows, first_row=first)
    out = old.to(DEV)
    mccl.embedding_grad(grad.to(DEV), plan, scale=scale, out=out, accumulate=accumulate)
    want, tol = grad_reference(grad, ids, first, rows, scale)
    if accumulate:
        touched = torch.zeros(rows + 1, dtype=torch.bool)
        touched[keys_of(ids, first, rows)] = True
        assert torch.equal(out.cpu()[~touched[:-1]], old[~touched[:-1]]), "rows without a token"
        want = want + old.double()
        tol = tol + U * want.abs()
    within(out, want, tol + half_step(out_dtype) * (want.abs() + tol) + torch.finfo(out_dtype).smallest_normal * half_step(out_dtype), "grad")


def test_embedding_grad_gives_the_same_bits_every_time_and_for_any_split(mccl):
    g = gen(5)
    n, rows, hidden = 20000, 300, 200
    grad = torch.randn(n, hidden, generator=g).to(DEV)
    ids = torch.randint(0, rows, (n,), generator=g)
    ids[torch.rand(n, generator=g) < 0.4] = 17
    plan = mccl.sort_ids(ids.to(DEV), rows)
    one = mccl.embedding_grad(grad, plan)
    for _ in range(3):
        assert torch.equal(one, mccl.embedding_grad(grad, plan))


def test_embedding_grad_is_the_derivative(mccl):
    """Against central differences of a loss through the lookup itself (fp32 table, linear in it: exact
    but for roundings of the loss, 2^-24 of the sum of its terms' sizes over the step)."""
    g = gen(8)
    rows, hidden, n, scale = 9, 24, 50, 0.75
    table = torch.randn(rows, hidden, generator=g).to(DEV)
    ids = torch.randint(-1, rows + 1, (n,), generator=g).to(DEV)
    up = torch.randn(n, hidden, generator=g).to(DEV)
    grad = mccl.embedding_grad(up, mccl.sort_ids(ids, rows), scale=scale)
    step = 0.5
    for v in range(rows):
        delta = torch.randn(hidden, generator=g).to(DEV)
        sides = []
        for sign in (1, -1):
            moved = table.clone()
            moved[v] += sign * step * delta
            sides.append((mccl.embedding(moved, ids, scale=scale).double() * up.double()).sum())
        slope = float((sides[0] - sides[1]) / (2 * step))
        size = float((up.double().abs().sum(dim=1) * (ids == v)).sum() * 4 * 4) + 1.0
        assert abs(slope - float((grad[v].double() * delta.double()).sum())) <= 100 * U * size, v


def test_embedding_grad_skips_what_a_foreign_plan_points_past(mccl):
    """Indices and offsets outside the gradient are not followed."""
    grad = torch.ones(4, 8, device=DEV)
    order = torch.tensor([0, 99, -5, 3], device=DEV)
    offsets = torch.tensor([0, 2, 1 << 40], device=DEV)
    out = mccl.embedding_grad(grad, (order, offsets))
    assert out[:, 0].tolist() == [1.0, 1.0]


def test_embedding_grad_stays_inside_whatever_the_offsets_say(mccl):
    """Offsets that fall, end early or point past the end: no row of the result depends on more than the
    gradient (each is a sum of some of its rows, all ones here: at most their number)."""
    n, rows, hidden = 700, 40, 24
    grad = torch.ones(n, hidden, device=DEV)
    order = torch.randperm(n, generator=gen(3)).to(DEV)
    for seed in range(6):
        offsets = torch.randint(-50, n + 200, (rows + 1,), generator=gen(4, seed))
        if seed % 2:
            offsets = torch.sort(offsets, descending=True).values
        out = mccl.embedding_grad(grad, (order, offsets.to(DEV)), out=torch.zeros(rows, hidden, device=DEV))
        assert out.shape == (rows, hidden)
    good = mccl.embedding_grad(grad, mccl.sort_ids(torch.arange(n, device=DEV) % rows, rows))
    assert good[:, 0].sum() == n


# ---------------------------------------------------------------------------------------------
# router
# ---------------------------------------------------------------------------------------------
def route_reference(logits, topk, normalize):
    l = logits.double()
    ids = torch.argsort(torch.where(l.isnan(), torch.full_like(l, float("-inf")), -(-l)).neg(), dim=1, stable=True)[:, :topk]
    value = l.gather(1, ids)
    closed = (value == float("-inf")) | value.isnan()
    p = torch.softmax(l, dim=1)
    w = p.gather(1, ids)
    w = torch.where(closed, torch.zeros_like(w), w)
    if normalize:
        w = w / w.sum(dim=1, keepdim=True)
    w = torch.where(closed, torch.zeros_like(w), w)
    return torch.where(closed, torch.full_like(ids, -1), ids).int(), w


ROUTES = [(1, 1, 1), (7, 5, 5), (16, 64, 6), (33, 65, 3), (50, 100, 8), (200, 256, 8), (9, 257, 8), (40, 512, 4), (5, 1000, 64), (3, 4096, 10),
          (4097, 16, 2), (4099, 17, 17), (5000, 60, 6), (4500, 100, 20), (4999, 255, 8), (8191, 256, 8)]


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("tokens,experts,topk", ROUTES)
def test_route_and_its_gradient(mccl, dtype, normalize, tokens, experts, topk):
    """Choices equal, weights within: the difference to the largest logit, exp (2 u), a sum over the
    lane's share and six steps, a division.  Every third token has closed experts; ties are frequent in
    the 16-bit types."""
    g = gen(tokens, experts, topk, int(normalize))
    logits = (3.0 * torch.randn(tokens, experts, generator=g)).to(dtype)
    closed = torch.rand(tokens, experts, generator=g) < 0.4
    closed[torch.arange(tokens) % 3 != 1] = False
    closed[:, 0] = False
    logits[closed] = float("-inf")
    ids, weights = mccl.moe_route(logits.to(DEV), topk, normalize=normalize)
    want_ids, want = route_reference(logits, topk, normalize)
    assert torch.equal(ids.cpu(), want_ids)
    per_lane = max(1, 1 << max(0, math.ceil(math.log2(experts / 64))))
    span = 30.0 + per_lane + topk
    within(weights, want, (span + 20) * U * want, "weights")

    up = torch.randn(tokens, topk, generator=g)
    d = mccl.moe_route_grad(up.to(DEV), logits.to(DEV), ids, normalize=normalize)
    at = logits.double().clone().requires_grad_(True)
    # normalised: p / sum of the chosen p is the softmax of the chosen alone, whose derivative elsewhere is 0 exactly
    q = torch.softmax(at.gather(1, want_ids.long().clamp(min=0)).masked_fill(want_ids < 0, float("-inf")), dim=1) if normalize \
        else torch.softmax(at, dim=1).gather(1, want_ids.long().clamp(min=0))
    q = torch.where(want_ids >= 0, q, torch.zeros_like(q))
    (q * up.double()).sum().backward()
    chosen = torch.where(want_ids >= 0, want, torch.zeros_like(want))
    mean_size = (chosen * up.double().abs()).sum(dim=1, keepdim=True)
    own = torch.zeros(tokens, experts, dtype=torch.float64).scatter_add(1, want_ids.long().clamp(min=0), torch.where(want_ids >= 0, up.double().abs(), torch.zeros_like(want)))
    p = torch.softmax(logits.double(), dim=1) if not normalize else torch.zeros(tokens, experts, dtype=torch.float64).scatter_add(1, want_ids.long().clamp(min=0), chosen)
    tol = 2 * (span + 20) * U * p * (own + mean_size)
    within(d, at.grad, tol + half_step(dtype) * (at.grad.abs() + tol) + torch.finfo(dtype).smallest_normal * half_step(dtype), "grad")


@pytest.mark.parametrize("normalize", [True, False])
def test_route_gradient_against_differences(mccl, normalize):
    """fp32 weights of logits moved by 2^-6 either way: the third derivative's part is below
    step^2 * sum |g|, the roundings' below 40 u * sum |g| / step."""
    g = gen(77)
    tokens, experts, topk, step = 6, 40, 4, 2.0 ** -6
    logits = torch.randn(tokens, experts, generator=g)
    top = torch.argsort(logits, dim=1, descending=True)
    logits.scatter_add_(1, top[:, :topk], torch.full((tokens, topk), 0.5))  # no choice changes within the step
    up = torch.randn(tokens, topk, generator=g)
    ids, _ = mccl.moe_route(logits.to(DEV), topk, normalize=normalize)
    d = mccl.moe_route_grad(up.to(DEV), logits.to(DEV), ids, normalize=normalize).cpu().double()
    for trial in range(4):
        way = torch.randn(tokens, experts, generator=g).clamp(-2, 2)
        sides = []
        for sign in (1, -1):
            i2, w2 = mccl.moe_route((logits + sign * step * way).to(DEV), topk, normalize=normalize)
            # the same experts, perhaps in another order: the weight of each choice of ids
            at = torch.zeros(tokens, experts, dtype=torch.float64).scatter(1, i2.cpu().long(), w2.cpu().double())
            assert torch.equal(torch.sort(i2.cpu(), dim=1).values, torch.sort(ids.cpu(), dim=1).values)
            sides.append((at.gather(1, ids.cpu().long()) * up.double()).sum(dim=1))
        slope = (sides[0] - sides[1]) / (2 * step)
        size = up.double().abs().sum(dim=1)
        within(slope, (d * way.double()).sum(dim=1), 8 * step * step * size + 60 * U * size / step, "differences")


def test_route_ties_masks_and_values_that_are_not_finite(mccl):
    inf, nan = float("inf"), float("nan")
    low = torch.finfo(torch.float32).min
    rows = [
        [1.0, 1.0, 1.0, 1.0, 1.0],          # all equal: lowest indices
        [-0.0, 0.0, -0.0, -1.0, 0.0],       # -0 equals +0
        [-inf] * 5,                         # nothing open
        [-inf, -inf, 2.0, -inf, -inf],      # one open
        [low, low, low, low, low],          # the type's lowest value is a logit like any other
        [nan, 1.0, 2.0, 0.0, 0.0],          # NaN: not chosen, weights NaN
        [inf, 1.0, 2.0, 0.0, 0.0],          # +inf: chosen, weights NaN
        [low, 5.0, low, low, -inf],
    ]
    logits = torch.tensor(rows, device=DEV)
    for normalize in (True, False):
        ids, w = mccl.moe_route(logits, 3, normalize=normalize)
        assert ids.tolist() == [[0, 1, 2], [0, 1, 2], [-1] * 3, [2, -1, -1], [0, 1, 2], [2, 1, 3], [0, 2, 1], [1, 0, 2]]
        w = w.cpu()
        even = 1.0 / 3.0 if normalize else 0.2
        within(w[0], torch.full((3,), even), 4 * U, "even")
        within(w[4], torch.full((3,), even), 4 * U, "lowest")
        assert w[2].tolist() == [0, 0, 0] and w[3].tolist() == [1, 0, 0] and w[7].tolist() == [1, 0, 0]
        assert w[5].isnan().all() and w[6].isnan().all()
        d = mccl.moe_route_grad(torch.ones(8, 3, device=DEV), logits, ids, normalize=normalize).cpu()
        assert not d[2].any() and not d[3].any(), "no gradient where nothing, or only one expert, was open"
        assert torch.isfinite(d[4]).all()


def test_route_gradient_of_repeated_and_foreign_ids(mccl):
    """The same expert twice gets both gradients; ids outside are skipped."""
    logits = torch.tensor([[0.0, 1.0, 2.0, 0.5]], device=DEV)
    g = torch.tensor([[1.0, 3.0, 100.0, 50.0]], device=DEV)
    ids = torch.tensor([[2, 2, 4, -7]], dtype=torch.int32, device=DEV)
    d = mccl.moe_route_grad(g, logits, ids, normalize=False).cpu().double()[0]
    p = torch.softmax(logits.cpu().double()[0], dim=0)
    want = -p * (4 * p[2])
    want[2] += 4 * p[2]
    within(d, want, 40 * U * 4 * torch.ones(4), "repeated")


# ---------------------------------------------------------------------------------------------
# mixture-of-experts layer
# ---------------------------------------------------------------------------------------------
def act64(v, name):
    return v / (1 + torch.exp(-v)) if name == "silu" else 0.5 * v * torch.erfc(-v / math.sqrt(2.0))


def layer_reference(x, w_in, w_out, ids, weights, first, activation, dtype):
    """(out, tolerance) in 64 bits.  gate and up: hidden roundings of the fp32 sum of |w x| (the slope of
    either activation is below 1.2); h is rounded once to the layer's type; the second product has inter
    roundings, the weighted sum topk + 1, the output one half step."""
    T, H = x.shape
    E, I = w_out.shape[0], w_out.shape[2]
    out, tol = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    size = torch.zeros_like(out)
    tiny = torch.finfo(dtype).smallest_normal * half_step(dtype)
    for t in range(T):
        for k in range(ids.shape[1]):
            e = int(ids[t, k]) - first
            if not 0 <= e < E:
                continue
            a, b, xt, w = w_in[e].double(), w_out[e].double(), x[t].double(), float(weights[t, k])
            s, ds = a @ xt, (H + 1) * U * (a.abs() @ xt.abs())
            act = act64(s[:I], activation)
            h = act * s[I:]
            dh = (1.2 * ds[:I] + 8 * U * act.abs()) * (s[I:].abs() + ds[I:]) + act.abs() * ds[I:]
            dh = dh + half_step(dtype) * (h.abs() + dh) + tiny
            y, dy = b @ h, b.abs() @ dh + (I + 1) * U * (b.abs() @ (h.abs() + dh))
            out[t] += w * y
            size[t] += abs(w) * (y.abs() + dy)
            tol[t] += abs(w) * dy
    tol = tol + (ids.shape[1] + 1) * U * size
    return out, tol + half_step(dtype) * (out.abs() + tol) + tiny


def layer_inputs(g, T, k, E, local, H, I, dtype):
    x = torch.randn(T, H, generator=g).to(dtype)
    w_in = (torch.randn(local, 2 * I, H, generator=g) / math.sqrt(H)).to(dtype)
    w_out = (torch.randn(local, H, I, generator=g) / math.sqrt(I)).to(dtype)
    ids = torch.argsort(torch.rand(T, E, generator=g), dim=1)[:, :k].to(torch.int32).contiguous()
    weights = torch.softmax(torch.randn(T, k, generator=g), dim=1).contiguous()
    return x, w_in, w_out, ids, weights


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("T,k,E,local,first,H,I", [
    (1, 1, 1, 1, 0, 8, 8), (1, 8, 64, 64, 0, 256, 64), (2, 2, 4, 4, 0, 40, 24), (5, 3, 34, 34, 0, 520, 200), (16, 2, 3, 3, 0, 64, 128),
    (17, 1, 1, 1, 0, 72, 16), (31, 4, 16, 4, 8, 136, 88), (64, 2, 2, 2, 0, 32, 40), (3, 64, 70, 70, 0, 48, 16), (100, 6, 12, 5, 3, 264, 72),
    (256, 2, 4, 4, 0, 96, 56), (256, 8, 128, 128, 0, 64, 16), (256, 16, 300, 300, 0, 16, 8), (3, 2, 4, 4, 0, 4096, 72), (6, 4, 9, 9, 0, 7168, 8), (7, 2, 40, 10, 20, 1032, 328), (33, 1, 2, 1, 1, 1024, 512), (2, 1, 300, 300, 0, 16, 2056)])
def test_moe_layer(mccl, dtype, activation, T, k, E, local, first, H, I):
    g = gen(T, k, E, H, I)
    x, w_in, w_out, ids, weights = layer_inputs(g, T, k, E, local, H, I, dtype)
    if T > 2:
        ids[1] = -1                      # padding
        ids[2] = ids[2, 0]               # the same expert topk times
        x[1] = float("nan")              # what padding holds does not matter
        weights[1] = float("nan")
    out = torch.full((T, H), float("nan"), dtype=dtype, device=DEV)
    mccl.moe_layer(x.to(DEV), w_in.to(DEV), w_out.to(DEV), ids.to(DEV), weights.to(DEV), first_expert=first, activation=activation, out=out)
    want, tol = layer_reference(x, w_in, w_out, ids, weights, first, activation, dtype)
    within(out, want, tol, "layer")


def test_moe_layer_without_any_pair_is_zero_and_no_tokens_are_no_work(mccl):
    g = gen(3)
    x, w_in, w_out, ids, weights = [t.to(DEV) for t in layer_inputs(g, 4, 2, 6, 2, 64, 32, torch.bfloat16)]
    assert not mccl.moe_layer(x, w_in, w_out, torch.full_like(ids, -1), weights).any()
    assert not mccl.moe_layer(x, w_in, w_out, ids, weights, first_expert=1 << 40).any()
    assert not mccl.moe_layer(x, w_in, w_out, ids, weights, first_expert=-(1 << 62)).any()
    assert mccl.moe_layer(x[:0], w_in, w_out, ids[:0], weights[:0]).shape == (0, 64)


def test_moe_layer_keeps_other_tokens_apart_from_one_that_is_not_finite(mccl):
    """A token with infinities or NaN changes its own output alone, also where it shares an expert."""
    g = gen(4)
    x, w_in, w_out, ids, weights = layer_inputs(g, 20, 2, 3, 3, 128, 64, torch.bfloat16)
    args = [w_in.to(DEV), w_out.to(DEV), ids.to(DEV), weights.to(DEV)]
    clean = mccl.moe_layer(x.to(DEV), *args)
    x[7, 5], x[12] = float("inf"), float("nan")
    out = mccl.moe_layer(x.to(DEV), *args)
    keep = [t for t in range(20) if t not in (7, 12)]
    assert torch.equal(out[keep], clean[keep]) and not torch.isfinite(out[12].float()).any()


def test_moe_layer_weights_past_4_gib(mccl):
    """Experts behind the first 4 GiB of weights."""
    H, I, E, T = 4096, 4096, 70, 3
    w_in = torch.zeros(E, 2 * I, H, dtype=torch.bfloat16, device=DEV)
    w_out = torch.zeros(E, H, I, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(9)
    last = E - 1
    w_in[last].normal_(0, 1 / math.sqrt(H), generator=g)
    w_out[last].normal_(0, 1 / math.sqrt(I), generator=g)
    x = torch.randn(T, H, generator=gen(10)).to(torch.bfloat16)
    ids = torch.tensor([[last], [0], [last]], dtype=torch.int32)
    weights = torch.ones(T, 1)
    out = mccl.moe_layer(x.to(DEV), w_in, w_out, ids.to(DEV), weights.to(DEV))
    want, tol = layer_reference(x, w_in[last:].cpu(), w_out[last:].cpu(), ids, weights, last, "silu", torch.bfloat16)
    within(out, want, tol, "layer")


def test_moe_layer_gives_the_same_bits_every_time(mccl):
    g = gen(11)
    args = [t.to(DEV) for t in layer_inputs(g, 40, 4, 8, 8, 512, 256, torch.bfloat16)]
    one = mccl.moe_layer(*args)
    for _ in range(5):
        assert torch.equal(one, mccl.moe_layer(*args))


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
def test_route_then_layer_equals_dispatch_experts_combine(mccl):
    """One decode step both ways: moe_layer, and sort_ids + gather_rows + the experts in torch +
    moe_combine.  Both are within their tolerance of the definition."""
    g = gen(21)
    T, k, E, H, I, dtype = 24, 4, 16, 256, 96, torch.bfloat16
    x, w_in, w_out, _, _ = layer_inputs(g, T, k, E, E, H, I, dtype)
    logits = torch.randn(T, E, generator=g)
    ids, weights = mccl.moe_route(logits.to(DEV), k)
    out = mccl.moe_layer(x.to(DEV), w_in.to(DEV), w_out.to(DEV), ids, weights)
    want, tol = layer_reference(x, w_in, w_out, ids.cpu(), weights.cpu(), 0, "silu", dtype)
    within(out, want, tol, "layer")

    order, offsets = mccl.sort_ids(ids.reshape(-1), E)
    assert torch.equal(offsets.diff(), mccl.route_counts(ids.reshape(-1), E))
    sent = mccl.gather_rows(x.to(DEV), torch.div(order, k, rounding_mode="floor"))
    back = torch.empty_like(sent)
    at = offsets.tolist()
    for e in range(E):
        s = sent[at[e]:at[e + 1]].float() @ w_in[e].to(DEV).float().t().contiguous()
        h = (torch.nn.functional.silu(s[:, :I]) * s[:, I:]).to(dtype).float()
        back[at[e]:at[e + 1]] = (h @ w_out[e].to(DEV).float().t().contiguous()).to(dtype)
    row = torch.empty_like(order)
    row[order] = torch.arange(T * k, device=DEV)
    y = mccl.moe_combine([back], torch.zeros(T, k, dtype=torch.int32, device=DEV), row.view(T, k).contiguous(), weights)
    # the exchanged rows are rounded once more, to the layer's type
    within(y, want, tol + half_step(dtype) * 2 * (want.abs() + 4 * tol) + half_step(dtype) * 8, "combine")


def test_expert_parallel_ranks_add_up_to_the_layer(mccl):
    """Four ranks with a quarter of the experts each, their outputs added by reduce_n as the all_reduce
    of the group adds them: within one half step per rank of the definition."""
    g = gen(22)
    T, k, E, H, I, W, dtype = 12, 4, 16, 264, 72, 4, torch.float16
    x, w_in, w_out, ids, weights = layer_inputs(g, T, k, E, E, H, I, dtype)
    per = E // W
    parts = [mccl.moe_layer(x.to(DEV), w_in[r * per:(r + 1) * per].contiguous().to(DEV), w_out[r * per:(r + 1) * per].contiguous().to(DEV),
                            ids.to(DEV), weights.to(DEV), first_expert=r * per) for r in range(W)]
    total = mccl.reduce_n(parts)
    want, tol = layer_reference(x, w_in, w_out, ids, weights, 0, "silu", dtype)
    sizes = sum(p.cpu().double().abs() for p in parts)
    within(total, want, tol + half_step(dtype) * 2 * sizes, "sum of the ranks")


def test_vocabulary_shards_add_up_to_the_lookup_and_its_gradient(mccl):
    """Every id is in exactly one shard: the sum over the ranks is the lookup bit for bit (0 + x), and
    each rank's gradient is its rows of the whole table's."""
    g = gen(23)
    W, per, hidden, n, dtype = 4, 50, 136, 300, torch.bfloat16
    table = torch.randn(W * per, hidden, generator=g).to(dtype).to(DEV)
    ids = torch.randint(0, W * per, (n,), generator=g).to(DEV)
    shards = [table[r * per:(r + 1) * per].contiguous() for r in range(W)]
    parts = [mccl.embedding(s, ids, scale=0.5, first_row=r * per) for r, s in enumerate(shards)]
    assert torch.equal(mccl.reduce_n(parts), mccl.embedding(table, ids, scale=0.5))
    up = torch.randn(n, hidden, generator=g).to(dtype).to(DEV)
    whole = mccl.embedding_grad(up, mccl.sort_ids(ids, W * per), scale=0.5)
    for r in range(W):
        part = mccl.embedding_grad(up, mccl.sort_ids(ids, per, first_row=r * per), scale=0.5)
        within(part, whole[r * per:(r + 1) * per].cpu(), 4 * half_step(dtype) * (whole[r * per:(r + 1) * per].cpu().double().abs() + 1), "rank %d" % r)


def test_gradient_of_the_token_permute(mccl):
    """gather_rows' gradient: what autograd gives for the indexing itself, in 64 bits."""
    g = gen(24)
    T, k, hidden = 60, 4, 200
    src = torch.randn(T, hidden, generator=g, dtype=torch.float64, requires_grad=True)
    index = torch.randperm(T * k, generator=g) % T
    up = torch.randn(T * k, hidden, generator=g)
    (src[index] * up.double()).sum().backward()
    rows = mccl.gather_rows(src.detach().float().to(DEV), index.to(DEV))
    assert torch.equal(rows.cpu(), src.detach().float()[index])
    d = mccl.embedding_grad(up.to(DEV), mccl.sort_ids(index.to(DEV), T))
    size = torch.zeros(T, hidden, dtype=torch.float64).index_add_(0, index, up.double().abs())
    within(d, src.grad, (k + 1) * U * size, "permute")


def test_replayed_from_a_graph_on_a_stream_of_their_own(mccl):
    """A router, layer, lookup and gradient step recorded once and replayed with new inputs, with eager
    work in between: every replay equals the eager result bit for bit."""
    g = gen(31)
    T, k, E, H, I, V, dtype = 6, 2, 8, 128, 64, 40, torch.bfloat16
    _, w_in, w_out, _, _ = [t.to(DEV) for t in layer_inputs(g, T, k, E, E, H, I, dtype)]
    table = torch.randn(V, H, generator=g).to(dtype).to(DEV)
    ids = torch.zeros(5000, dtype=torch.int64, device=DEV)
    up = torch.zeros(5000, H, dtype=dtype, device=DEV)
    logits = torch.zeros(T, E, device=DEV)

    def step():
        x = mccl.embedding(table, ids[:T], scale=2.0)
        chosen, w = mccl.moe_route(logits, k)
        y = mccl.moe_layer(x, w_in, w_out, chosen, w)
        d = mccl.embedding_grad(up, mccl.sort_ids(ids, V), scale=2.0)
        dl = mccl.moe_route_grad(w, logits, chosen)
        return x, chosen, w, y, d, dl

    def fill(seed):
        gs = gen(seed)
        ids.copy_(torch.randint(-1, V + 1, (5000,), generator=gs))
        up.copy_(torch.randn(5000, H, generator=gs))
        logits.copy_(torch.randn(T, E, generator=gs))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        fill(1)
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
        for seed in (2, 3, 4):
            fill(seed)
            graph.replay()
            side.synchronize()
            got = [t.clone() for t in held]
            for a, b in zip(got, step()):
                assert torch.equal(a, b)
            graph.replay()
            side.synchronize()
            for a, b in zip(held, got):
                assert torch.equal(a, b)


def test_two_streams_at_once_and_results_that_wait_for_each_other(mccl):
    """Calls of different sizes on two streams at once, each with its own workspace from the allocator, give
    what they give alone."""
    g = gen(51)
    layers = [[t.to(DEV) for t in layer_inputs(g, T, 4, 16, 16, 256, 128, torch.bfloat16)] for T in (3, 40)]
    ids = [torch.randint(0, 500, (n,), generator=g).to(DEV) for n in (3000, 20000)]
    ups = [torch.randn(len(i), 136, generator=g).to(DEV) for i in ids]
    alone = [(mccl.moe_layer(*layers[k]), mccl.embedding_grad(ups[k], mccl.sort_ids(ids[k], 500))) for k in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((mccl.moe_layer(*layers[k]), mccl.embedding_grad(ups[k], mccl.sort_ids(ids[k], 500))))
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_layer_with_most_pairs_replays_from_a_graph(mccl):
    """2048 pairs over many experts: more LDS than a kernel has by default, also under capture."""
    tensors = [t.to(DEV) for t in layer_inputs(gen(53), 256, 8, 200, 200, 64, 32, torch.bfloat16)]
    alone = mccl.moe_layer(*tensors)
    out = torch.zeros_like(alone)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mccl.moe_layer(*tensors, out=out)
    for _ in range(3):
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, alone)
        assert torch.equal(mccl.moe_layer(*tensors), alone)


def test_views_that_are_not_contiguous_are_refused(mccl):
    table, ids = torch.zeros(16, 32, device=DEV), torch.zeros(8, dtype=torch.int64, device=DEV)
    for call in (lambda: mccl.embedding(table[:, ::2], ids), lambda: mccl.embedding(table, ids[::2]), lambda: mccl.sort_ids(ids[::2], 4),
                 lambda: mccl.embedding_grad(table[::2], mccl.sort_ids(ids, 4)), lambda: mccl.moe_route(table.t(), 2),
                 lambda: mccl.moe_route(table, 2, out=(torch.zeros(16, 4, dtype=torch.int32, device=DEV)[:, ::2], None))):
        with pytest.raises(RuntimeError, match="contiguous"):
            call()
    with pytest.raises(RuntimeError, match="on the GPU"):
        mccl.embedding(table, ids.cpu())
    big = torch.zeros(5000, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="workspace must be"):
        mccl.sort_ids(big, 4, workspace=torch.zeros(16, dtype=torch.uint8, device=DEV))


def test_results_go_where_the_caller_says(mccl):
    """out tensors: the same object comes back, and only it is written."""
    g = gen(52)
    x, w_in, w_out, ids, weights = [t.to(DEV) for t in layer_inputs(g, 5, 2, 4, 4, 64, 40, torch.float16)]
    out = torch.full((7, 64), 9.0, dtype=torch.float16, device=DEV)
    assert mccl.moe_layer(x, w_in, w_out, ids, weights, out=out[1:6]).data_ptr() == out[1:6].data_ptr()
    assert torch.equal(out[1:6], mccl.moe_layer(x, w_in, w_out, ids, weights)) and bool((out[0] == 9).all()) and bool((out[6] == 9).all())
    logits = torch.randn(33, 70, generator=g).to(DEV)
    held = (torch.full((35, 3), 77, dtype=torch.int32, device=DEV), torch.full((35, 3), 77.0, device=DEV))
    a, b = mccl.moe_route(logits, 3, out=(held[0][1:34], held[1][1:34]))
    want = mccl.moe_route(logits, 3)
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    for h in held:
        assert bool((h[0] == 77).all()) and bool((h[34] == 77).all())
    d = torch.full((35, 70), 5.0, device=DEV)
    mccl.moe_route_grad(b.contiguous(), logits, a.contiguous(), out=d[1:34])
    assert torch.equal(d[1:34], mccl.moe_route_grad(want[1], logits, want[0])) and bool((d[0] == 5).all()) and bool((d[34] == 5).all())


def test_workspaces_of_the_caller_are_used_and_may_be_dirty(mccl):
    from torch_ccl_amd import capi
    g = gen(41)
    x, w_in, w_out, ids, weights = [t.to(DEV) for t in layer_inputs(g, 9, 3, 8, 8, 64, 40, torch.bfloat16)]
    need = capi.lib().mccl_moe_layer_workspace(9, 3, 8, 64, 40)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=DEV)
    assert torch.equal(mccl.moe_layer(x, w_in, w_out, ids, weights, workspace=ws), mccl.moe_layer(x, w_in, w_out, ids, weights))
    tokens = torch.randint(0, 30, (4000,), generator=g).to(DEV)
    ws = torch.full((capi.lib().mccl_sort_ids_workspace(4000),), 0xFF, dtype=torch.uint8, device=DEV)
    a, b = mccl.sort_ids(tokens, 30, workspace=ws), mccl.sort_ids(tokens, 30)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    up = torch.randn(4000, 72, generator=g).to(DEV)
    ws = torch.full((capi.lib().mccl_embedding_grad_workspace(4000, 72),), 0xFF, dtype=torch.uint8, device=DEV)
    assert torch.equal(mccl.embedding_grad(up, a, workspace=ws), mccl.embedding_grad(up, b))

# ---------------------------------------------------------------------------------------------
# the layer between its two products
# ---------------------------------------------------------------------------------------------
def layer_reference_unrounded(x, w_in, w_out, ids, weights, first, activation, dtype):
    """layer_reference without a rounding of act(..) * (..) to the layer's type: what the second product
    takes holds 2^-16 of it or better (two parts of 8 bits each), next to the fp32 roundings."""
    T, H = x.shape
    E, I = w_out.shape[0], w_out.shape[2]
    out, tol, size = (torch.zeros(T, H, dtype=torch.float64) for _ in range(3))
    for t in range(T):
        for k in range(ids.shape[1]):
            e = int(ids[t, k]) - first
            if not 0 <= e < E:
                continue
            a, b, xt, w = w_in[e].double(), w_out[e].double(), x[t].double(), float(weights[t, k])
            s, ds = a @ xt, (H + 1) * U * (a.abs() @ xt.abs())
            act = act64(s[:I], activation)
            h = act * s[I:]
            dh = (1.2 * ds[:I] + 8 * U * act.abs()) * (s[I:].abs() + ds[I:]) + act.abs() * ds[I:]
            dh = dh + 2.0 ** -16 * (h.abs() + dh)
            y, dy = b @ h, b.abs() @ dh + 4 * (I + 1) * U * (b.abs() @ (h.abs() + dh))  # four products of parts each
            out[t] += w * y
            size[t] += abs(w) * (y.abs() + dy)
            tol[t] += abs(w) * dy
    tol = tol + (ids.shape[1] + 1) * U * size
    return out, tol + half_step(dtype) * (out.abs() + tol) + torch.finfo(dtype).smallest_normal * half_step(dtype)


LAYERS_BOTH_WAYS = [(1, 1, 1, 64, 64), (5, 1, 1, 40, 200), (9, 2, 3, 264, 136), (17, 1, 1, 72, 88), (40, 2, 2, 136, 264), (64, 8, 128, 64, 72), (130, 1, 1, 264, 392)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("T,k,E,H,I", LAYERS_BOTH_WAYS)
def test_moe_layer_rounds_to_its_type_once(mccl, dtype, activation, T, k, E, H, I):
    x, w_in, w_out, ids, weights = layer_inputs(gen(61, T, k, E, H, I), T, k, E, E, H, I, dtype)
    out = mccl.moe_layer(x.to(DEV), w_in.to(DEV), w_out.to(DEV), ids.to(DEV), weights.to(DEV), activation=activation)
    want, tol = layer_reference_unrounded(x, w_in, w_out, ids, weights, 0, activation, dtype)
    within(out, want, tol, "layer")


@pytest.mark.parametrize("T,k,E,H,I", LAYERS_BOTH_WAYS)
def test_moe_layer_between_its_products_has_the_range_of_fp32(mccl, T, k, E, H, I):
    """act(..) * (..) around 10^6, which f16 has no number for, and an output that it has."""
    dtype = torch.float16
    x, w_in, w_out, ids, weights = layer_inputs(gen(62, T, k, E, H, I), T, k, E, E, H, I, dtype)
    x, w_out = 2.0 ** 10 * x, (2.0 ** -10 * w_out.double()).to(dtype)
    assert torch.isfinite(x).all()
    out = mccl.moe_layer(x.to(DEV), w_in.to(DEV), w_out.to(DEV), ids.to(DEV), weights.to(DEV))
    want, tol = layer_reference_unrounded(x, w_in, w_out, ids, weights, 0, "silu", dtype)
    assert float(want.abs().max()) < 65504 / 2
    within(out, want, tol, "layer")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("T,k,E", [(3, 1, 1), (40, 2, 2)])
def test_moe_layer_of_weights_that_are_not_finite(mccl, dtype, T, k, E):
    """An infinite weight of the second product makes its row of the output infinite with the sign that the
    formula gives, a NaN makes it NaN, and the other rows stay as they are."""
    H, I = 72, 40
    x, w_in, w_out, ids, weights = layer_inputs(gen(63, T, k, E), T, k, E, E, H, I, dtype)
    args = [x.to(DEV), w_in.to(DEV), w_out.to(DEV), ids.to(DEV), weights.to(DEV)]
    clean = mccl.moe_layer(*args)
    bad = w_out.clone()
    bad[0, 5, 7], bad[0, 6, 0], bad[0, 20, I - 1] = float("inf"), float("-inf"), float("nan")
    args[2] = bad.to(DEV)
    out = mccl.moe_layer(*args).cpu()
    rows = [c for c in range(H) if c not in (5, 6, 20)]
    assert torch.equal(out[:, rows], clean.cpu()[:, rows])
    s = torch.einsum("ij,tj->ti", w_in[0].double(), x.double())
    h = act64(s[:, :I], "silu") * s[:, I:]
    for t in range(T):
        if 0 not in ids[t].tolist():
            continue
        assert out[t, 20].isnan()
        assert float(out[t, 5]) == math.copysign(math.inf, float(h[t, 7])) and float(out[t, 6]) == -math.copysign(math.inf, float(h[t, 0]))


# ---------------------------------------------------------------------------------------------
# the router's gradient of rows that are not finite
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("tokens,experts", [(5, 5), (7, 300), (4100, 16), (4100, 250)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_route_gradient_of_rows_that_are_not_finite(mccl, dtype, tokens, experts, bad):
    """The weights of a row that holds a NaN or +inf are NaN, and so is what depends on them: the chosen experts'
    gradients with normalize (zero elsewhere), every expert's without.  Other rows are not touched by it."""
    g = gen(71, tokens, experts)
    topk = 3
    logits = torch.randn(tokens, experts, generator=g).to(dtype)
    marked = torch.arange(tokens) % 4 == 1
    at = torch.randint(0, experts, (tokens,), generator=g)
    broken = logits.clone()
    broken[marked, at[marked]] = bad
    up = torch.randn(tokens, topk, generator=g).to(DEV)
    for normalize in (True, False):
        ids, w = mccl.moe_route(broken.to(DEV), topk, normalize=normalize)
        assert w[marked].isnan().all()
        d = mccl.moe_route_grad(up, broken.to(DEV), ids, normalize=normalize).cpu()
        chosen = torch.zeros(tokens, experts, dtype=torch.bool).scatter(1, ids.cpu().long(), True)
        if normalize:
            assert d[marked][chosen[marked]].isnan().all() and not d[marked][~chosen[marked]].any()
        else:
            assert d[marked].isnan().all()
        clean_ids, _ = mccl.moe_route(logits.to(DEV), topk, normalize=normalize)
        clean = mccl.moe_route_grad(up, logits.to(DEV), clean_ids, normalize=normalize).cpu()
        assert torch.equal(d[~marked], clean[~marked])


# ---------------------------------------------------------------------------------------------
# plans that are a part of another, or none that a sort gives
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("n,hidden", [(40, 24), (700, 24), (5000, 136), (5000, 7)])
@pytest.mark.parametrize("skip", [0, 3, 64, 70, 200])
def test_embedding_grad_of_a_range_of_rows_of_a_larger_plan(mccl, n, hidden, skip, accumulate):
    """One sort of the whole vocabulary, and the gradient of rows [first, first + 6) by their offsets alone: the same bits
    as those rows of the whole gradient where both cut the tokens alike, and within the sum's roundings of the
    definition.  `skip` tokens come before the range, whose first row holds most of the others."""
    g = gen(81, n, hidden, skip, int(accumulate))
    rows, first, count = 20, 9, 6
    ids = torch.full((n,), first)
    ids[torch.rand(n, generator=g) < 0.4] = first + 3
    some = torch.rand(n, generator=g) < 0.1
    ids[some] = torch.randint(first, rows, (int(some.sum()),), generator=g)
    ids[:min(skip, n)] = torch.randint(0, first, (min(skip, n),), generator=g)
    ids = ids[torch.randperm(n, generator=g)]
    up = torch.randn(n, hidden, generator=g)
    order, offsets = mccl.sort_ids(ids.to(DEV), rows)
    old = torch.randn(count, hidden, generator=g)
    out = old.to(DEV) if accumulate else torch.full((count, hidden), float("nan"), device=DEV)
    mccl.embedding_grad(up.to(DEV), (order, offsets[first:first + count + 1].contiguous()), out=out, accumulate=accumulate)
    want, tol = grad_reference(up, ids, first, count, 1.0)
    if accumulate:
        want, tol = want + old.double(), tol + U * (want + old.double()).abs()
    within(out, want, tol + 2 * U * want.abs(), "range")
    if not accumulate:
        assert torch.equal(out, mccl.embedding_grad(up.to(DEV), (order, offsets))[first:first + count])


@pytest.mark.parametrize("hidden", [24, 7, 2056])
@pytest.mark.parametrize("way", ["any", "falling", "steps back"])
def test_embedding_grad_adds_nothing_that_no_call_wrote(mccl, way, hidden):
    """Offsets that no sort gives, over a workspace full of NaN: with rows of ones every result is a number of
    gradient rows, so a whole number from 0 to n, or what was there before (zero here)."""
    from torch_ccl_amd import capi
    n, rows = 1000, 12
    grad = torch.ones(n, hidden, device=DEV)
    order = torch.randperm(n, generator=gen(82)).to(DEV)
    ws = torch.empty(capi.lib().mccl_embedding_grad_workspace(n, hidden), dtype=torch.uint8, device=DEV)
    for seed in range(40):
        g = gen(83, seed)
        offsets = torch.randint(-50, n + 100, (rows + 1,), generator=g)
        if way == "falling":
            offsets = torch.sort(offsets, descending=True).values
        elif way == "steps back":
            offsets = torch.sort(offsets).values
            i = int(torch.randint(1, rows, (1,), generator=g))
            offsets[i] -= 300
        ws.fill_(255)
        out = mccl.embedding_grad(grad, (order, offsets.to(DEV)), out=torch.zeros(rows, hidden, device=DEV), workspace=ws).cpu()
        assert torch.isfinite(out).all(), (way, seed)
        assert bool((out == out.round()).all()) and float(out.min()) >= 0 and float(out.max()) <= n, (way, seed)


def test_a_shard_at_the_end_of_the_id_type(mccl):
    info = torch.iinfo(torch.int64)
    table = torch.arange(1.0, 6.0, device=DEV)[:, None].repeat(1, 8)
    ids = torch.tensor([info.max, info.min, info.max - 3, info.min + 1, -1, 0], device=DEV)
    assert mccl.embedding(table[:4], ids, first_row=info.max - 3)[:, 0].tolist() == [4, 0, 1, 0, 0, 0]
    order, offsets = mccl.sort_ids(ids, 4, first_row=info.max - 3)
    assert order.tolist() == [2, 0, 1, 3, 4, 5] and offsets.tolist() == [0, 1, 1, 1, 2]
    with pytest.raises(RuntimeError, match="pass 2"):
        mccl.embedding(table, ids, first_row=info.max - 3)
    with pytest.raises(RuntimeError, match="pass 2"):
        mccl.sort_ids(ids, 5, first_row=info.max - 3)


# ---------------------------------------------------------------------------------------------
# autograd around the calls
# ---------------------------------------------------------------------------------------------
def calls_with_out(mccl, g):
    """(name, tensors written, the call) of every operator that writes into tensors of the caller."""
    table, ids = torch.randn(9, 16, generator=g).to(DEV), torch.randint(0, 9, (5,), generator=g).to(DEV)
    logits = torch.randn(5, 8, generator=g).to(DEV)
    x, w_in, w_out, chosen, w = [t.to(DEV) for t in layer_inputs(g, 5, 2, 8, 8, 16, 8, torch.bfloat16)]
    plan = mccl.sort_ids(ids, 9)
    outs = [torch.zeros(5, 16, device=DEV), torch.zeros(9, 16, device=DEV), torch.zeros(9, 16, device=DEV),
            (torch.zeros(5, 2, dtype=torch.int32, device=DEV), torch.zeros(5, 2, device=DEV)), torch.zeros(5, 8, device=DEV), torch.zeros_like(x)]
    up = torch.randn(5, 16, generator=g).to(DEV)
    return [("embedding", outs[:1], lambda: mccl.embedding(table, ids, out=outs[0])),
            ("embedding_grad", outs[1:2], lambda: mccl.embedding_grad(up, plan, out=outs[1])),
            ("accumulate", outs[2:3], lambda: mccl.embedding_grad(up, plan, out=outs[2], accumulate=True)),
            ("moe_route", list(outs[3]), lambda: mccl.moe_route(logits, 2, out=outs[3])),
            ("moe_route_grad", outs[4:5], lambda: mccl.moe_route_grad(w, logits, chosen, out=outs[4])),
            ("moe_layer", outs[5:6], lambda: mccl.moe_layer(x, w_in, w_out, chosen, w, out=outs[5]))]


def test_writing_into_a_tensor_that_autograd_keeps_is_noticed(mccl):
    for name, written, call in calls_with_out(mccl, gen(91)):
        before = [t._version for t in written]
        call()
        assert all(t._version > b for t, b in zip(written, before)), name
    out = torch.ones(5, 16, device=DEV)
    leaf = torch.ones(5, 16, device=DEV, requires_grad=True)
    loss = (leaf * out).sum()  # keeps out for leaf's gradient
    mccl.embedding(torch.zeros(3, 16, device=DEV), torch.zeros(5, dtype=torch.int64, device=DEV), out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_of_inference_mode_are_written_too(mccl):
    with torch.inference_mode():
        calls = calls_with_out(mccl, gen(92))
    for name, written, call in calls:
        call()
        with torch.inference_mode():
            call()
        assert all(t.is_inference() for t in written), name


def test_inputs_that_require_grad_are_told_that_they_get_none(mccl):
    import warnings
    g = gen(93)
    table, ids = torch.randn(9, 16, generator=g).to(DEV), torch.randint(0, 9, (5,), generator=g).to(DEV)
    logits, up = torch.randn(5, 8, generator=g).to(DEV), torch.randn(5, 16, generator=g).to(DEV)
    x, w_in, w_out, chosen, w = [t.to(DEV) for t in layer_inputs(g, 5, 2, 8, 8, 16, 8, torch.bfloat16)]
    plan = mccl.sort_ids(ids, 9)

    def calls(want):
        wants = lambda t, name: t.detach().requires_grad_(name == want)
        return {"table": lambda: mccl.embedding(wants(table, "table"), ids),
                "grad": lambda: mccl.embedding_grad(wants(up, "grad"), plan),
                "logits": lambda: mccl.moe_route(wants(logits, "logits"), 2)[1],
                "grad_weights": lambda: mccl.moe_route_grad(wants(w, "grad_weights"), logits, chosen),
                "x": lambda: mccl.moe_layer(wants(x, "x"), w_in, w_out, chosen, w),
                "w_in": lambda: mccl.moe_layer(x, wants(w_in, "w_in"), w_out, chosen, w),
                "w_out": lambda: mccl.moe_layer(x, w_in, wants(w_out, "w_out"), chosen, w),
                "weights": lambda: mccl.moe_layer(x, w_in, w_out, chosen, wants(w, "weights"))}

    for name in calls(None):
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            alone = calls(None)[name]()
            with torch.no_grad():
                calls(name)[name]()
            with pytest.raises(UserWarning, match="%s requires grad" % name):
                calls(name)[name]()
        with pytest.warns(UserWarning, match="no autograd node"):
            assert torch.equal(calls(name)[name](), alone), name


def test_moe_layer_on_a_rank_without_experts_is_zero(mccl):
    """Its part of the all_reduce, also into a tensor of the caller and from a graph."""
    x, w_in, w_out, ids, weights = [t.to(DEV) for t in layer_inputs(gen(94), 6, 2, 4, 4, 64, 40, torch.bfloat16)]
    none = (w_in[:0], w_out[:0])
    assert mccl.moe_layer(x, *none, ids, weights).shape == x.shape and not mccl.moe_layer(x, *none, ids, weights, first_expert=4).any()
    out = torch.full_like(x, 5.0)
    assert mccl.moe_layer(x, *none, ids, weights, out=out).data_ptr() == out.data_ptr() and not out.any()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mccl.moe_layer(x, *none, ids, weights, out=out)
    for _ in range(3):
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert not out.any()
    with pytest.raises(RuntimeError, match="w_in must be"):
        mccl.moe_layer(x, w_in, w_out[:0], ids, weights)
    with pytest.raises(RuntimeError, match="at most 256"):  # as on the ranks that hold some
        mccl.moe_layer(x[:1].repeat(257, 1), *none, ids[:1].repeat(257, 1), weights[:1].repeat(257, 1))


# ---------------------------------------------------------------------------------------------
# sizes at which a call takes another way
# ---------------------------------------------------------------------------------------------
def unevenly(g, T, k, E, hot):
    """ids [T, k]: the first `hot` tokens have expert 1 among their choices, no other token has; choices differ."""
    ids = torch.argsort(torch.rand(T, E, generator=g), dim=1)[:, :k]
    for t in range(T):
        row = [int(e) for e in ids[t] if e != 1]
        row += [e for e in range(2, E) if e not in row]
        ids[t] = torch.tensor(([1] if t < hot else []) + row)[:k] if E > 1 else 0
    return ids.to(torch.int32).contiguous()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("T,k,E,hot,H,I", [
    # through LDS: one tile and two of an expert's tokens, over 3 and 4 (and 5) chunks of 128 columns of either product,
    # turns of 128 and of 64 columns, one or more parts of inter
    (256, 1, 1, 256, 392, 520), (129, 1, 1, 129, 520, 392), (128, 1, 1, 128, 264, 640), (65, 1, 1, 65, 640, 264), (64, 1, 1, 64, 520, 520),
    (256, 2, 3, 200, 136, 264), (150, 2, 6, 67, 400, 136), (13, 1, 1, 13, 264, 1160),
    # from memory: an expert with more pairs than one list holds, more than 32, 16, 8 and 4 of them
    (256, 8, 200, 256, 72, 40), (130, 4, 60, 130, 136, 72), (100, 4, 64, 65, 72, 136), (40, 4, 30, 33, 136, 72), (40, 4, 30, 17, 72, 72),
    (20, 4, 30, 9, 136, 200), (20, 4, 30, 5, 264, 72)])
def test_moe_layer_of_uneven_experts(mccl, dtype, T, k, E, hot, H, I):
    g = gen(95, T, k, E, hot, H, I)
    x, w_in, w_out, _, weights = layer_inputs(g, T, k, E, E, H, I, dtype)
    ids = unevenly(g, T, k, E, hot)
    assert int((ids == min(1, E - 1)).sum()) == hot
    out = torch.full((T, H), float("nan"), dtype=dtype, device=DEV)
    mccl.moe_layer(x.to(DEV), w_in.to(DEV), w_out.to(DEV), ids.to(DEV), weights.to(DEV), out=out)
    want, tol = layer_reference_unrounded(x, w_in, w_out, ids, weights, 0, "silu", dtype)
    within(out, want, tol, "layer")


@pytest.mark.parametrize("T,k,E,local,first", [(1, 8, 64, 8, 16), (8, 8, 64, 8, 0), (60, 8, 64, 8, 24), (70, 8, 64, 8, 56), (256, 8, 64, 8, 8), (256, 8, 64, 1, 63)])
def test_moe_layer_on_a_shard_at_every_batch(mccl, T, k, E, local, first):
    """Most pairs are other ranks' experts; the workspace holds NaN where nothing of this rank is written."""
    from torch_ccl_amd import capi
    H, I, dtype = 136, 264, torch.bfloat16
    x, w_in, w_out, ids, weights = layer_inputs(gen(96, T, local, first), T, k, E, local, H, I, dtype)
    ws = torch.full((capi.lib().mccl_moe_layer_workspace(T, k, local, H, I),), 255, dtype=torch.uint8, device=DEV)
    out = mccl.moe_layer(x.to(DEV), w_in.to(DEV), w_out.to(DEV), ids.to(DEV), weights.to(DEV), first_expert=first, workspace=ws)
    want, tol = layer_reference_unrounded(x, w_in, w_out, ids, weights, first, "silu", dtype)
    within(out, want, tol, "layer")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_embedding_grad_gives_a_columns_bits_whatever_is_beside_it(mccl, dtype):
    """The columns of a wide row, which one wavefront takes two chunks of, alone: one chunk, spread over workgroups, or
    shorter than a vector.  The order of a column's sum depends on the offsets alone."""
    g = gen(97)
    n, rows, hidden = 3000, 6000, 4 * 512 + 8 * 64 + 24
    ids = torch.randint(0, rows, (n,), generator=g)
    ids[torch.rand(n, generator=g) < 0.3] = 1234
    ids[torch.rand(n, generator=g) < 0.1] = 7
    up = torch.randn(n, hidden, generator=g).to(dtype).to(DEV)
    plan = mccl.sort_ids(ids.to(DEV), rows)
    wide = mccl.embedding_grad(up, plan, scale=0.75)
    for first, count in ((0, 512), (0, 2048), (512, 1032), (hidden - 24, 24), (hidden - 3, 3), (77, 1), (100, 513)):
        part = mccl.embedding_grad(up[:, first:first + count].contiguous(), plan, scale=0.75)
        assert torch.equal(part, wide[:, first:first + count]), (first, count)


@pytest.mark.parametrize("T", [1, 6, 20])
@pytest.mark.parametrize("power", [40, 54, 55, 56, 58, 60, 61, 62])
def test_moe_layer_of_very_small_values(mccl, T, power):
    """gate = up = 2^-power: silu's half of that times up is 2^-(2 power + 1), exactly (exp(-gate) is 1), down to the
    smallest normal numbers of bf16; so is the output."""
    H, I = 8, 8
    x = torch.zeros(T, H, dtype=torch.bfloat16)
    x[:, 3] = 2.0 ** -power
    w_in, w_out = torch.zeros(1, 2 * I, H, dtype=torch.bfloat16), torch.zeros(1, H, I, dtype=torch.bfloat16)
    w_in[0, :, 3], w_out[0, 5, 6] = 1.0, 1.0
    ids, weights = torch.zeros(T, 1, dtype=torch.int32), torch.ones(T, 1)
    out = mccl.moe_layer(*[t.to(DEV) for t in (x, w_in, w_out, ids, weights)]).cpu().double()
    want = torch.zeros(T, H, dtype=torch.float64)
    want[:, 5] = 2.0 ** -(2 * power + 1)
    assert torch.equal(out, want)
