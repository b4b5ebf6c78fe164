"""The operators around the index against plain implementations in 64 bits.

Tolerances follow from the arithmetic, before any run: u is half a unit in the last place of the output's type (2^-24 fp32,
2^-11 fp16, 2^-8 bf16) and covers the one rounding of the result; what is computed in fp32 before it adds a multiple of 2^-24
of the sum of magnitudes.  Results of fp16 below its normal numbers are allowed half their spacing, 2^-25.
"""
import math
import time

import pytest

pytestmark = pytest.mark.gpu

ULP = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
FLOOR = {"fp32": 2.0 ** -126, "fp16": 2.0 ** -25, "bf16": 2.0 ** -126}
EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def torch():
    import torch
    torch.cuda.set_device(0)
    return torch


def dtype_of(torch, name):
    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


def generator(torch, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def laid_out(torch, x, layout):
    """The same values as a matrix of another layout."""
    n, d = x.shape
    if layout == "dense":
        return x
    if layout == "padded":      # rows further apart, by a number of elements that is odd
        room = torch.full((n, d + 7), float("nan") if x.dtype.is_floating_point else 77, dtype=x.dtype, device=x.device)
        room[:, :d] = x
        return room[:, :d]
    if layout == "shifted":     # rows that start one element into a word
        room = torch.zeros((n, d + 17), dtype=x.dtype, device=x.device)
        room[:, 1:d + 1] = x
        return room[:, 1:d + 1]
    room = torch.empty((d, n), dtype=x.dtype, device=x.device)  # columns next to one another
    room.copy_(x.t())
    return room.t()


def within(torch, got, want, bound):
    got, want = got.double(), want.double()
    same = torch.isnan(got) == torch.isnan(want)
    assert bool(same.all()), "NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fine = ~(torch.isnan(want) | inf)
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0.0, "off by %g more than allowed" % float(off.max())


# ---- lookup ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,rows,dim,layout", [
    (1, 1, 1, "dense"), (1, 5000, 1024, "dense"), (7, 3, 2, "dense"), (33, 100, 3, "padded"), (1000, 70_001, 96, "dense"),
    (257, 1000, 300, "dense"), (257, 1000, 301, "dense"), (64, 500, 1024, "shifted"), (65, 200, 1029, "dense"), (17, 90, 5000, "padded"),
    (40, 64, 128, "columns")])
def test_lookup(cp, torch, name, n, rows, dim, layout):
    gen = generator(torch, n * 31 + dim)
    table = torch.randn((rows, dim), generator=gen, device="cuda").to(dtype_of(torch, name))
    ids = torch.randint(0, rows, (n,), generator=gen, device="cuda", dtype=torch.int64)
    if n > 4:
        ids[1], ids[2], ids[4] = -1, rows, 2 ** 40
        ids[3] = rows - 1
    scale = math.sqrt(dim)
    for kind in (torch.int64, torch.int32):
        these = ids if kind == torch.int64 else torch.where(ids >= 2 ** 31, torch.full_like(ids, -2 ** 31), ids).to(kind)
        got = cp.embedding_lookup(laid_out(torch, table, layout), these, scale)
        inside = (ids >= 0) & (ids < rows)
        want = torch.where(inside[:, None], table[torch.where(inside, ids, 0)].double() * scale, 0.0)
        assert got.dtype == table.dtype and got.shape == (n, dim)
        # the scale is rounded to fp32, the product twice
        within(torch, got, want, want.abs() * (ULP[name] + 3 * EPS) + FLOOR[name])
        assert not bool(got[~inside].any())


def test_lookup_shapes_and_outputs(cp, torch):
    table = torch.randn((50, 24), device="cuda")
    ids = torch.randint(0, 50, (3, 5), device="cuda", dtype=torch.int32)
    assert torch.equal(cp.embedding_lookup(table, ids), table[ids.long()])
    room = torch.full((15, 31), 9.0, device="cuda")
    out = room[:, 2:26]
    assert cp.embedding_lookup(table, ids.view(-1), 2.0, out=out) is out
    assert torch.equal(out, table[ids.long().view(-1)] * 2) and bool((room[:, :2] == 9).all()) and bool((room[:, 26:] == 9).all())
    assert cp.embedding_lookup(table, ids[:0]).shape == (0, 5, 24)
    one = torch.randn((1, 24), device="cuda").expand(50, 24)  # a broadcast row
    assert torch.equal(cp.embedding_lookup(one, ids.view(-1)), one[:15])
    # values that are not numbers pass where they are asked for, and only there
    table[7, 3], table[8, 0], table[9] = float("nan"), float("inf"), float("nan")
    got = cp.embedding_lookup(table, torch.tensor([7, 8, -1], device="cuda"), 3.0)
    assert bool(torch.isnan(got[0, 3])) and bool(torch.isinf(got[1, 0])) and int((~torch.isfinite(got)).sum()) == 2 and not bool(got[2].any())


# ---- its gradient ----------------------------------------------------------------------------------------------------------
def ids_of(torch, gen, kind, n, rows):
    if kind == "same":
        return torch.full((n,), rows // 2, device="cuda", dtype=torch.int64)
    if kind == "none":
        return torch.full((n,), -1, device="cuda", dtype=torch.int64)
    if kind == "zipf":
        weight = 1.0 / torch.arange(1, rows + 1, device="cuda", dtype=torch.float64)
        total = torch.cumsum(weight, 0)
        ids = torch.searchsorted(total, torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * total[-1]).clamp_max_(rows - 1)
        ids = torch.randperm(rows, generator=gen, device="cuda")[ids]
    else:
        ids = torch.randint(0, rows, (n,), generator=gen, device="cuda")
    if n > 8:
        ids[torch.rand(n, generator=gen, device="cuda") < 0.05] = -1
        ids[5], ids[n - 1] = rows, rows - 1
    return ids


def grad_want(torch, ids, grad, rows, scale):
    inside = (ids >= 0) & (ids < rows)
    at = torch.where(inside, ids, rows)
    total = torch.zeros((rows + 1, grad.shape[1]), dtype=torch.float64, device="cuda")
    size = torch.zeros_like(total)
    total.index_add_(0, at, grad.double())
    size.index_add_(0, at, grad.double().abs())
    many = torch.bincount(at, minlength=rows + 1)[:rows, None]
    return total[:rows] * scale, size[:rows] * abs(scale), many


@pytest.mark.parametrize("types", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32")])
@pytest.mark.parametrize("n,rows,dim,kind,layout", [
    (0, 40, 16, "even", "dense"), (1, 1, 1, "even", "dense"), (31, 70, 5, "zipf", "dense"), (512, 3000, 300, "zipf", "dense"),
    (2048, 129, 64, "zipf", "padded"), (2048, 65, 1024, "same", "dense"), (1500, 1000, 2100, "zipf", "dense"),
    (2049, 1, 33, "even", "dense"), (2049, 4000, 8, "none", "dense"), (5000, 511, 256, "zipf", "dense"), (5000, 512, 258, "even", "shifted"),
    (4099, 100_003, 100, "zipf", "padded"), (20_000, 300_000, 24, "zipf", "dense"), (6000, 50, 1030, "same", "dense"),
    (140_000, 2000, 40, "zipf", "dense"), (3000, 700, 64, "zipf", "columns")])
def test_grad(cp, torch, types, n, rows, dim, kind, layout):
    gen = generator(torch, n + rows + dim)
    ids = ids_of(torch, gen, kind, n, rows)
    grad = torch.randn((n, dim), generator=gen, device="cuda").to(dtype_of(torch, types[0]))
    scale = 1.75
    want, size, many = grad_want(torch, ids, grad, rows, scale)
    given = laid_out(torch, grad, layout)
    got = cp.embedding_grad(ids, given, rows, scale, dtype=dtype_of(torch, types[1]))
    bound = size * EPS * (many + 2) + want.abs() * ULP[types[1]] + FLOOR[types[1]]
    assert got.shape == (rows, dim) and got.dtype == dtype_of(torch, types[1])
    within(torch, got, want, bound)
    assert not bool(got[many[:, 0] == 0].any())
    # the same bits again, from ids of 4 bytes
    again = cp.embedding_grad(ids.to(torch.int32), given, rows, scale, dtype=dtype_of(torch, types[1]))
    assert torch.equal(got, again)
    # added to what is there, the rows that no id names left alone
    room = torch.randn((rows, dim + 3), generator=gen, device="cuda").to(got.dtype)
    before = room.clone()
    out = cp.embedding_grad(ids, given, rows, scale, out=room[:, :dim], accumulate=True)
    total = want + before[:, :dim].double()
    within(torch, out, total, size * EPS * (many + 2) + (total.abs() + before[:, :dim].double().abs()) * EPS + total.abs() * ULP[types[1]] + FLOOR[types[1]])
    assert torch.equal(room[:, dim:], before[:, dim:])
    idle = many[:, 0] == 0
    assert torch.equal(room[idle], before[idle])


@pytest.mark.parametrize("types", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32")])
@pytest.mark.parametrize("n,dim", [(300, 64), (2048, 1024), (2049, 64), (9000, 1024)])
@pytest.mark.parametrize("first,more", [(0, 4), (4, 4), (4, 0), (4, 8), (2, 2), (8, 8)])
def test_grad_into_part_of_a_buffer(cp, torch, types, n, dim, first, more):
    """Rows of the output that start at any multiple of 4 to 32 bytes and at any distance: a slice of a flat buffer, columns of a
    wider one.  Whole numbers: the sums are exact, and what lies beside them stays."""
    gen = generator(torch, n + dim + 10 * first + more)
    rows = 150
    ids = ids_of(torch, gen, "zipf", n, rows)  # (the commonest id has more places than a piece)
    grad = torch.randint(-2, 3, (n, dim), generator=gen, device="cuda").to(dtype_of(torch, types[0]))
    want = grad_want(torch, ids, grad, rows, 0.5)[0]
    want = want.to(dtype_of(torch, types[1]))  # (one rounding of an exact sum)
    width = dim + more
    for accumulate in (False, True):
        flat = torch.full((first + rows * width + 40,), 1.0, dtype=want.dtype, device="cuda")
        out = flat[first:first + rows * width].view(rows, width)[:, :dim]
        assert cp.embedding_grad(ids, grad, rows, 0.5, out=out, accumulate=accumulate) is out
        expect = torch.ones_like(flat)
        inside = expect[first:first + rows * width].view(rows, width)[:, :dim]
        # (with what was there: the sum in fp32 is exact too, and rounded once)
        inside.copy_((grad_want(torch, ids, grad, rows, 0.5)[0] + 1.0).to(want.dtype) if accumulate else want)
        assert torch.equal(flat, expect)
    cp.check_operator_status()


@pytest.mark.parametrize("name", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,rows,dim", [(300, 15, 512), (300, 15, 300), (2048, 40, 96), (1000, 5, 1024), (2000, 3, 255), (5000, 200, 512), (5000, 3, 96)])
def test_grad_bits_of_other_layouts(cp, torch, name, n, rows, dim):
    """The order of a sum does not depend on where rows start: the same bits from, and to, every layout."""
    gen = generator(torch, n + dim)
    ids = ids_of(torch, gen, "even", n, rows)
    grad = torch.randn((n, dim), generator=gen, device="cuda").to(dtype_of(torch, name))
    for dtype in {torch.float32, grad.dtype}:
        want = cp.embedding_grad(ids, grad, rows, 1.75, dtype=dtype)
        for layout in ("padded", "shifted"):
            assert torch.equal(cp.embedding_grad(ids, laid_out(torch, grad, layout), rows, 1.75, dtype=dtype), want)
        for first, more in ((0, 1), (1, 8), (2, 6), (4, 4), (4, 8), (8, 8)):
            room = torch.zeros((rows, first + dim + more), dtype=dtype, device="cuda")
            assert torch.equal(cp.embedding_grad(ids, grad, rows, 1.75, out=room[:, first:first + dim]), want)


@pytest.mark.parametrize("n,rows,dim", [(1_100_007, 5000, 4), (2_200_000, 300, 3)])
def test_grad_of_many_places(cp, torch, n, rows, dim):
    gen = generator(torch, n)
    ids = ids_of(torch, gen, "zipf", n, rows)
    grad = torch.randn((n, dim), generator=gen, device="cuda")
    want, size, many = grad_want(torch, ids, grad, rows, 0.5)
    # (a chain of roundings is at most as long as the longest of thread, piece and join, and each adds less than the sizes' sum)
    within(torch, cp.embedding_grad(ids, grad, rows, 0.5), want, size * EPS * (many + 2))


# places of each id, in the order of the ids, by which runs begin and end inside pieces of 32, on their edges, and in the piece where
# the one before ended; 8,193 places and more are over 256 pieces, and so joined three times
LONG_RUNS = {
    "inside": [20, 8295, 40, 33, 8200, 31, 32, 1, 64, 65, 500, 0, 17, 9000, 3],
    "edges": [32, 8192, 64, 8224, 33, 31, 32, 96, 16_384, 0, 512, 544, 7],
    "longest": [5, 300_007, 13, 50, 270_000, 2, 1000],
    "one": [0, 2_200_000, 0],
}


@pytest.mark.parametrize("types", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp32")])
@pytest.mark.parametrize("lengths,dim", [("inside", 3), ("inside", 264), ("inside", 1024), ("edges", 40), ("edges", 262), ("longest", 8), ("longest", 72), ("one", 4)])
def test_grad_of_long_runs_exactly(cp, torch, types, lengths, dim):
    """Whole numbers whose sums stay below 2^24: fp32 sums are exact in any order, so that a piece that is lost, counted twice or
    joined to another run shows.  A tenth of the places name no row."""
    gen = generator(torch, dim)
    count = torch.tensor(LONG_RUNS[lengths], device="cuda")
    ids = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count)
    ids = torch.cat([ids, torch.full((len(ids) // 10 + 2049,), -1, device="cuda")])
    n, rows = len(ids), len(count)
    ids = ids[torch.randperm(n, generator=gen, device="cuda")]
    grad = torch.randint(-3, 8, (n, dim), generator=gen, device="cuda", dtype=torch.int8).to(dtype_of(torch, types[0]))
    assert int(count.max()) * 7 < 2 ** 24
    total = torch.stack([grad[ids == k].double().sum(0) for k in range(rows)])
    for accumulate in (False, True):
        out = torch.full((rows, dim), 3.0, dtype=dtype_of(torch, types[1]), device="cuda")
        cp.embedding_grad(ids, grad, rows, 0.5, out=out, accumulate=accumulate)
        want = (total * 0.5 + 3.0 * accumulate).to(out.dtype)
        assert torch.equal(out, want)


@pytest.mark.parametrize("n,dim,dtype", [(5, 2049, "bf16"), (70, 2050, "fp32"), (33, 16_400, "bf16"), (9, 8196, "fp32"), (9, 8192, "fp32")])
def test_quantize_rows_by_blocks(cp, torch, n, dim, dtype):
    gen = generator(torch, n + dim)
    x = torch.randn((n, dim), generator=gen, device="cuda").to(dtype_of(torch, dtype))
    x[0] = torch.where(torch.rand(dim, generator=gen, device="cuda") < 0.5, x[0].float().abs().amax() / 2, x[0].float()).to(x.dtype)  # (ties)
    x[1] *= 1e-33
    q, scale = cp.quantize_rows(x)
    top = x.float().abs().amax(1)
    want = top * (torch.ones_like(top) / torch.full_like(top, 127.0))  # (by the rounded 1 / 127)
    assert torch.equal(scale, want)
    assert torch.equal(q.float(), torch.where(want[:, None] > 0, torch.round(x.float() / want[:, None]).clamp(-127, 127), 0.0))


@pytest.mark.parametrize("n", [100, 3000])
def test_grad_of_a_broadcast_row_and_of_odd_values(cp, torch, n):
    ids = torch.arange(n, device="cuda") % 50
    row = torch.randn((1, 128), device="cuda")
    got = cp.embedding_grad(ids, row.expand(n, 128), 64)
    want = row.double() * (n // 50)
    within(torch, got[:50], want.expand(50, 128), want.abs() * EPS * (n // 50 + 2))
    grad = torch.randn((n, 128), device="cuda")
    grad[3], grad[4, 5], grad[7] = float("nan"), float("inf"), float("nan")
    ids[7] = -1  # what is masked does not count, whatever it holds
    got = cp.embedding_grad(ids, grad, 64)
    assert bool(torch.isnan(got[3]).all()) and bool(torch.isinf(got[4, 5])) and int((~torch.isfinite(got)).sum()) == 129


@pytest.mark.parametrize("n", [60, 4000])
def test_grad_against_differences(cp, torch, n):
    """The lookup is linear: <grad, E> is the difference of <lookup, G> between table + E and table - E, halved."""
    gen = generator(torch, n)
    rows, dim, scale = 200, 48, 3.0
    ids = ids_of(torch, gen, "zipf", n, rows)
    table, E = torch.randn((2, rows, dim), generator=gen, device="cuda")
    G = torch.randn((n, dim), generator=gen, device="cuda")
    slope = [(cp.embedding_lookup(t, ids, scale).double() * G.double()).sum() for t in (table + E, table - E)]
    grad = cp.embedding_grad(ids, G, rows, scale)
    # each of the n * dim terms is rounded when the table is shifted and when it is scaled
    bound = n * dim * 4 * EPS * scale * 8 * 5
    assert abs(float((slope[0] - slope[1]) / 2 - (grad.double() * E.double()).sum())) <= bound


# ---- 8-bit products --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,dim,layout", [(1, 1, "dense"), (5, 3, "padded"), (9, 100, "dense"), (64, 128, "dense"), (3, 960, "shifted"), (70, 1023, "dense"),
                                          (2, 4096, "dense"), (3, 8200, "dense"), (2, 40_001, "padded"), (30, 64, "columns")])
def test_quantize_rows(cp, torch, name, n, dim, layout):
    gen = generator(torch, n + dim)
    x = (torch.randn((n, dim), generator=gen, device="cuda") * torch.rand((n, 1), generator=gen, device="cuda") * 10).to(dtype_of(torch, name))
    if n > 4:
        x[1] = 0
        x[2, dim // 2] = float("inf")
        x[3, 0] = float("nan")
        x[4] = 2.0 ** -24
        x[4, -1] = -2.0 ** -23
    q, scale = cp.quantize_rows(laid_out(torch, x, layout))
    assert q.dtype == torch.int8 and q.shape == (n, dim) and (n == 1 or q.stride(0) % 16 == 0) and q.data_ptr() % 16 == 0
    top = x.float().abs().amax(1)
    finite = torch.isfinite(x).all(1)
    # the definition, in fp32: equal bit for bit (a division by a plain number would be a product with its reciprocal in torch)
    want = top * (torch.ones_like(top) / torch.full_like(top, 127.0))  # (by the rounded 1 / 127)
    assert torch.equal(scale[finite], want[finite]) and bool(torch.isnan(scale[~finite]).all()) and not bool(q[~finite].any())
    back = torch.where(want[:, None] > 0, torch.round(x.float() / want[:, None]), 0.0)[finite]
    assert torch.equal(q[finite].float(), back)
    zero = top == 0
    assert not bool(q[zero].any()) and not bool(scale[zero].any())


PRODUCTS = [(1, 1, 1), (1, 4096, 4096), (3, 7, 15), (16, 128, 128), (17, 129, 100), (33, 1000, 960), (61, 3001, 96), (64, 256, 257), (100, 127, 300),
            (128, 640, 4096), (129, 515, 64), (300, 700, 1000), (1, 300, 131_071), (1024, 4096, 200), (2000, 5003, 333), (513, 10_007, 128), (2, 40_000, 64),
            (4000, 3, 50)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("name,layout", [("bf16", "dense"), ("fp32", "padded"), ("fp16", "shifted"), ("fp32", "dense")])
def test_int8_matmul(cp, torch, m, n, k, name, layout):
    gen = generator(torch, m + n + k)
    a = torch.randint(-128, 128, (m, k), generator=gen, device="cuda", dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=gen, device="cuda", dtype=torch.int8)
    a[0], b[0] = 127, 127  # the largest sum that operands of quantize_rows have
    sa = torch.rand(m, generator=gen, device="cuda") / (128 * k)
    sb = torch.rand(n, generator=gen, device="cuda")
    if m > 2:
        sa[1], sa[2] = 0.0, float("nan")
    got = cp.int8_matmul(laid_out(torch, a, layout), sa, laid_out(torch, b, layout), sb, dtype=dtype_of(torch, name))
    # sums of whole numbers below 2^53 are exact in 64 bits; then the sum, and two products, are rounded to fp32
    want = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None, :]
    within(torch, got, want, want.abs() * (ULP[name] + 4 * EPS) + FLOOR[name])
    room = torch.full((m, n + 5), 3.0, dtype=got.dtype, device="cuda")
    cp.int8_matmul(a, sa, b, sb, out=room[:, 1:n + 1])
    assert torch.equal(torch.nan_to_num(room[:, 1:n + 1]), torch.nan_to_num(got)) and bool((room[:, 0] == 3).all()) and bool((room[:, n + 1:] == 3).all())


@pytest.mark.parametrize("m,n,k", [(1, 1000, 8192), (5, 777, 4100), (100, 1500, 2048), (70, 2001, 3000), (300, 20_001, 200), (1024, 9001, 400), (128, 9000, 255), (90, 30_003, 128)])
@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_int8_matmul_split_and_unaligned(cp, torch, m, n, k, name):
    test_int8_matmul(cp, torch, m, n, k, name, "dense")


def test_int8_matmul_empty_and_broadcast(cp, torch):
    a = torch.ones((4, 32), dtype=torch.int8, device="cuda")
    s = torch.ones(4, device="cuda")
    assert cp.int8_matmul(a[:0], s[:0], a, s).shape == (0, 4) and cp.int8_matmul(a, s, a[:0], s[:0]).shape == (4, 0)
    one = torch.randint(-9, 9, (1, 32), dtype=torch.int8, device="cuda")
    got = cp.int8_matmul(one.expand(4, 32), s, a, s, dtype=torch.float32)
    assert torch.equal(got, one.float().sum().expand(4, 4))
    cp.check_operator_status()


# ---- distillation ------------------------------------------------------------------------------------------------------------
def distill_want(torch, z, ids, teacher, T, weight):
    """Loss, gradient, and the magnitudes that their bounds follow from, in 64 bits."""
    n, rows = z.shape
    u = z.double() / T
    top = u.amax(1, keepdim=True)
    safe = torch.where(torch.isinf(top) & (top < 0), 0.0, top)
    e = torch.exp(u - safe)
    total = e.sum(1, keepdim=True)
    q = torch.where(total == 0, 0.0, e / total)
    logq = torch.where(total == 0, u, u - safe - torch.log(total))
    inside = (ids >= 0) & (ids < rows)
    at = torch.where(inside, ids, 0).long()
    t = torch.where(inside, teacher.double() / T, -math.inf)
    best = t.amax(1, keepdim=True) if ids.shape[1] else torch.full((n, 1), -math.inf, dtype=torch.float64, device="cuda")
    some = best > -math.inf
    p = torch.exp(t - torch.where(some, best, 0.0))
    sum_p = p.sum(1, keepdim=True)
    p = torch.where(some, p / sum_p, 0.0)
    logp = torch.where(p > 0, t - best - torch.log(sum_p), 0.0)
    terms = torch.where(p > 0, p * (logp - torch.gather(logq, 1, at)), 0.0)
    loss = T * T * terms.sum(1)
    taken = torch.zeros_like(u).scatter_add_(1, at, p)
    g = torch.where(some & (weight[:, None] != 0), weight.double()[:, None] * T * (q - taken), 0.0)
    spread = torch.where(torch.isfinite(u), (u - safe).abs(), 0.0)
    return loss, g, q, taken, spread, some[:, 0]


def distill_bounds(torch, want, T, weight, name):
    """A sum of exponentials is off by at most 2^-17 of itself: 2^-22 each, and fewer than 400 additions in a chain of one
    thread, warp, block and cluster (400 * 2^-24 < 2^-15 would be the worst of all signs; they round both ways, so the
    bound taken is 2^-16).  The exponent (z - m) log2(e) / T is rounded three times: 2^-22 of its size."""
    loss, g, q, taken, spread, some = want
    rel = 2.0 ** -16 + spread * 2.0 ** -21
    grad = weight.double().abs()[:, None] * T * (q + taken) * rel + g.abs() * ULP[name] + FLOOR[name] * (1 + T)
    far = torch.where(taken > 0, spread, 0.0).amax(1)
    return T * T * (2.0 ** -16 + (far + 10) * 2.0 ** -20), grad


DISTILL = [(1, 1, 1, 1.0), (3, 7, 2, 1.0), (5, 1000, 0, 1.0), (9, 1000, 33, 2.0), (64, 4099, 64, 0.5), (2, 8192, 100, 4.0), (16, 32_768, 64, 1.0),
           (5, 32_769, 1024, 1.0), (40, 100_003, 100, 2.0), (3, 131_072, 257, 1.0), (2, 262_144, 64, 1.0), (2, 300_007, 64, 1.0), (700, 515, 8, 1.0),
           (2, 1_000_003, 16, 1.0)]


def distill_inputs(torch, name, n, rows, top, seed):
    gen = generator(torch, seed)
    z = (torch.randn((n, rows), generator=gen, device="cuda") * 3).to(dtype_of(torch, name))
    ids = torch.randint(0, rows, (n, top), generator=gen, device="cuda")  # (an id may come twice)
    teacher = torch.randn((n, top), generator=gen, device="cuda") * 3
    weight = torch.rand(n, generator=gen, device="cuda") + 0.5
    if top > 1:
        ids[0, 1] = -1
        teacher[0, 0] = -math.inf if top > 2 else 0.0
        z[0, ids[0, 0]] = -math.inf if top > 2 else 1.0   # a masked candidate that the teacher does not want either
    if n > 2:
        ids[1] = -1                                       # an empty list, over logits that are not numbers
        z[1, 0] = float("nan")
        weight[2] = 0.0
    if n > 4:
        z[3, : rows // 2] = -math.inf                     # half of the candidates masked, the list in the other half
        ids[3] = torch.clamp(ids[3], min=rows // 2)
        z[4] = torch.finfo(z.dtype).min                   # all at the type's lowest value
    if n > 8:
        ids[5], ids[6, top // 2:], ids[7] = ids[5, 0], rows, rows - 1
        teacher[8] = -math.inf
    return z, ids, teacher, weight


@pytest.mark.parametrize("name", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,rows,top,T", DISTILL)
@pytest.mark.parametrize("layout", ["dense", "shifted"])
def test_distill(cp, torch, name, n, rows, top, T, layout):
    z, ids, teacher, weight = distill_inputs(torch, name, n, rows, top, n + rows + top)
    clean = z.clone()
    if n > 2:
        clean[1, 0] = 0.0  # (its list is empty: nothing of it counts)
    want = distill_want(torch, clean, ids, teacher, T, weight)
    loss_bound, grad_bound = distill_bounds(torch, want, T, weight, name)
    given = laid_out(torch, z, layout)
    loss = cp.distill_loss(given, ids.to(torch.int32), teacher, T)
    within(torch, loss, want[0], loss_bound)
    loss2, grad = cp.distill_loss_and_grad(given, ids, teacher, weight, T)
    within(torch, loss2, want[0], loss_bound)
    within(torch, grad, want[1], grad_bound)
    assert grad.dtype == z.dtype and not bool(grad[~want[5]].any()) and not bool(grad[weight == 0].any())
    # the same bits again, in place of the logits
    mine = given.clone() if layout == "dense" else laid_out(torch, z, layout)
    loss3, same = cp.distill_loss_and_grad(mine, ids, teacher, weight, T, out=mine)
    assert same is mine and torch.equal(same, grad) and torch.equal(loss3, loss2)


@pytest.mark.parametrize("name", ["fp32", "bf16"])
@pytest.mark.parametrize("n,rows,top,T", [(40, 300, 130, 1.0), (33, 1400, 129, 2.0), (21, 2400, 64, 1.0), (300, 33_000, 8, 1.0), (210, 70_001, 20, 2.0), (1200, 9000, 5, 1.0)])
def test_distill_by_sizes(cp, torch, name, n, rows, top, T):
    test_distill(cp, torch, name, n, rows, top, T, "dense")


def test_distill_of_masked_and_odd_rows(cp, torch):
    z = torch.zeros((5, 40), device="cuda")
    z[0] = -math.inf                 # nothing left of the student
    z[1, 3] = float("nan")
    z[2, 4] = math.inf
    z[3, 5] = -math.inf              # a candidate that the teacher wants and the student masks
    ids = torch.tensor([[5, 6]] * 5, device="cuda")
    teacher = torch.zeros((5, 2), device="cuda")
    teacher[4, 1] = float("nan")
    loss, grad = cp.distill_loss_and_grad(z, ids, teacher, temperature=2.0)
    assert bool(torch.isinf(loss[0])) and loss[0] > 0 and bool(torch.isinf(loss[3])) and loss[3] > 0
    assert bool(torch.isnan(loss[[1, 2, 4]]).all())
    want = torch.zeros(40, device="cuda")
    want[5] = want[6] = -1.0         # -T p
    assert torch.equal(grad[0], want)
    q = torch.full((40,), 2.0 / 39, dtype=torch.float64, device="cuda")
    q[5] = 0.0
    q[5:7] -= 1.0
    within(torch, grad[3], q, torch.full((40,), 2.0 ** -16, dtype=torch.float64, device="cuda"))
    assert bool(torch.isnan(grad[[1, 4]]).all(1).any())
    assert torch.equal(torch.isinf(cp.distill_loss(z, ids, teacher, 2.0)), torch.isinf(loss))


@pytest.mark.parametrize("name,n,rows,top,T", [("fp32", 5, 1_000_003, 16, 1.0), ("fp32", 40, 1_000_003, 1024, 2.0), ("bf16", 20, 1_200_005, 64, 1.0),
                                               ("fp16", 13, 2_000_000, 700, 1.0)])
@pytest.mark.parametrize("layout", ["dense", "shifted"])
def test_distill_by_several_pieces_a_block(cp, torch, name, n, rows, top, T, layout):
    """Rows longer than a cluster holds go in pieces; here a block takes up to 17 of them, so that its ring goes round many times."""
    test_distill(cp, torch, name, n, rows, top, T, layout)
    cp.check_operator_status()


# one length for each way a row can take: a warp (two sizes), small rings, large rings in one block and in clusters, pieces
@pytest.mark.parametrize("name,rows", [("fp32", 40), ("bf16", 3001), ("fp32", 1500), ("bf16", 5003), ("fp32", 4000), ("fp16", 16_384), ("bf16", 100_003),
                                       ("fp32", 300_001), ("fp32", 1_000_003), ("bf16", 1_200_005)])
@pytest.mark.parametrize("layout", ["dense", "shifted"])
def test_distill_of_odd_rows_by_sizes(cp, torch, name, rows, layout):
    """Each kind of row by itself: what is not a number shows where the formula has it, and nowhere else."""
    T = 2.0
    base = torch.zeros((6, rows), device="cuda").to(dtype_of(torch, name))
    place = rows - 7                     # (far from the list)
    base[0] = -math.inf                  # nothing left of the student
    base[1, place] = math.nan
    base[2, place] = math.inf
    base[3, 5] = -math.inf               # a candidate that the teacher wants and the student masks
    ids = torch.tensor([[5, 6]] * 6, device="cuda")
    teacher = torch.zeros((6, 2), device="cuda")
    teacher[4, 1] = math.nan
    z = laid_out(torch, base, layout)
    loss, grad = cp.distill_loss_and_grad(z, ids, teacher, temperature=T)
    alone = cp.distill_loss(z, ids, teacher, T)
    for each in (loss, alone):
        assert float(each[0]) == math.inf and float(each[3]) == math.inf
        assert bool(torch.isnan(each[[1, 2, 4]]).all()) and bool(torch.isfinite(each[5]))
        # T^2 (log 1/2 + log rows): logits all alike
        assert abs(float(each[5]) - T * T * (math.log(0.5) + math.log(rows))) <= T * T * (2.0 ** -16 + 10 * 2.0 ** -20)
    assert bool(torch.isnan(grad[[1, 2]]).all())
    there = torch.zeros(rows, dtype=torch.bool, device="cuda")
    there[5:7] = True
    assert bool(torch.isnan(grad[4, there]).all())
    want = torch.zeros((6, rows), dtype=torch.float64, device="cuda")   # T (q - p)
    want[3] = T / (rows - 1)
    want[3, 5] = 0.0
    want[4:] = T / rows
    for row in (0, 3, 5):
        want[row, there] -= T * 0.5
    fine = torch.ones((6, rows), dtype=torch.bool, device="cuda")
    fine[1:3], fine[4, there] = False, False
    bound = (want.abs() + T * 0.5 * there) * 2.0 ** -16 + want.abs() * ULP[name] + FLOOR[name] * (1 + T)
    within(torch, grad[fine], want[fine], bound[fine])
    assert not bool(grad[0, ~there].any())
    cp.check_operator_status()


@pytest.mark.parametrize("rows", [50, 9000])
def test_distill_grad_against_differences(cp, torch, rows):
    gen = generator(torch, rows)
    n, top, T, h = 6, 12, 1.5, 2.0 ** -6
    z = torch.randn((n, rows), generator=gen, device="cuda")
    ids = torch.randint(0, rows, (n, top), generator=gen, device="cuda")
    teacher = torch.randn((n, top), generator=gen, device="cuda")
    d = torch.randn((n, rows), generator=gen, device="cuda")
    d /= d.norm(dim=1, keepdim=True)
    _, grad = cp.distill_loss_and_grad(z, ids, teacher, temperature=T)
    up, down = cp.distill_loss(z + h * d, ids, teacher, T).double(), cp.distill_loss(z - h * d, ids, teacher, T).double()
    # a loss is off by at most 2^-16 T^2 (1 + 2^-4 * 20); the third derivative along a direction of length 1 is below 2 / T
    bound = 2 * T * T * 2.0 ** -16 * 2.25 / (2 * h) + h * h / 6 * 2 / T + 2.0 ** -15
    assert float(((up - down) / (2 * h) - (grad.double() * d.double()).sum(1)).abs().max()) <= bound


def test_distill_lists_of_many_lengths(cp, torch):
    """What a launch asks of the driver it asks once, not again with every length of the lists: the host takes as long for calls
    of forty lengths in turn as for forty of one.  Eleven questions take 4 us and more; 2 us a call are allowed."""
    n, rows, calls = 40, 100_003, 40
    z = torch.randn((n, rows), device="cuda").bfloat16()
    out = torch.empty_like(z)
    ids = torch.randint(0, rows, (n, calls), device="cuda")
    teacher = torch.randn((n, calls), device="cuda")
    lists = [(ids[:, :top].contiguous(), teacher[:, :top].contiguous()) for top in range(1, calls + 1)]

    def host(lists):
        torch.cuda.synchronize()
        start = time.perf_counter()
        for i, t in lists:
            cp.distill_loss_and_grad(z, i, t, out=out)
        return (time.perf_counter() - start) / calls * 1e6

    turns = [(host([lists[9]] * calls), host(lists)) for _ in range(30)][1:]  # (the shortest of each: the host does other things too)
    one, many = (min(t[k] for t in turns) for k in range(2))
    assert many <= one + 2.0, (many, one)


# ---- the whole, other streams, refusals --------------------------------------------------------------------------------------
def test_on_another_stream_and_in_a_graph(cp, torch):
    gen = generator(torch, 1)
    table = torch.randn((3000, 96), generator=gen, device="cuda")
    ids = torch.randint(0, 3000, (5000,), generator=gen, device="cuda")
    w, ws = cp.quantize_rows(torch.randn((2000, 96), generator=gen, device="cuda"))
    lists = torch.randint(0, 2000, (5000, 10), generator=gen, device="cuda")
    scores = torch.randn((5000, 10), generator=gen, device="cuda")

    def step():
        x = cp.embedding_lookup(table, ids, 2.0)
        q, s = cp.quantize_rows(x)
        z = cp.int8_matmul(q, s, w, ws, dtype=torch.float32)
        loss, dz = cp.distill_loss_and_grad(z, lists, scores)
        return loss, dz, cp.embedding_grad(ids, x, 3000)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    table.neg_()
    graph.replay()
    torch.cuda.synchronize()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    cp.check_operator_status()


def test_refusals(cp, torch):
    f = torch.zeros((4, 8), device="cuda")
    i8 = torch.zeros((4, 8), dtype=torch.int8, device="cuda")
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    lists = torch.zeros((4, 2), dtype=torch.int64, device="cuda")
    teacher = torch.zeros((4, 2), device="cuda")
    one = torch.ones(4, device="cuda")
    wide = torch.zeros((4, 1025), device="cuda")
    calls = [
        lambda: cp.embedding_lookup(f.cpu(), ids), lambda: cp.embedding_lookup(f.double(), ids), lambda: cp.embedding_lookup(f, ids.float()),
        lambda: cp.embedding_lookup(f[0], ids), lambda: cp.embedding_lookup(f, ids, out=f[:2]), lambda: cp.embedding_lookup(f, ids, out=f.half()),
        lambda: cp.embedding_lookup(f[:0], ids),
        lambda: cp.embedding_grad(ids, f[:3], 4), lambda: cp.embedding_grad(ids, f, 0), lambda: cp.embedding_grad(ids, f, 4, dtype=torch.float16),
        lambda: cp.embedding_grad(ids, f, 4, accumulate=True), lambda: cp.embedding_grad(ids, f, 5, out=f),
        lambda: cp.embedding_grad(ids, f, 4, out=torch.zeros((1, 8), device="cuda").expand(4, 8)),
        lambda: cp.quantize_rows(i8), lambda: cp.quantize_rows(f[0]),
        lambda: cp.int8_matmul(i8, one, i8[:, :4], one), lambda: cp.int8_matmul(i8, one[:3], i8, one), lambda: cp.int8_matmul(i8, one.half(), i8, one),
        lambda: cp.int8_matmul(f, one, i8, one), lambda: cp.int8_matmul(i8, one, i8, one, dtype=torch.int8),
        lambda: cp.int8_matmul(i8, one, i8, one, out=f), lambda: cp.int8_matmul(i8[:, :0], one, i8[:, :0], one),
        lambda: cp.int8_matmul(torch.zeros((1, 131_072), dtype=torch.int8, device="cuda"), one[:1], torch.zeros((1, 131_072), dtype=torch.int8, device="cuda"), one[:1]),
        lambda: cp.distill_loss(f, lists[:3], teacher[:3]), lambda: cp.distill_loss(f, lists, teacher[:, :1]), lambda: cp.distill_loss(f, lists, teacher, 0.0),
        lambda: cp.distill_loss(f, lists, teacher, math.nan), lambda: cp.distill_loss(f, wide.long(), wide), lambda: cp.distill_loss(f.double(), lists, teacher),
        lambda: cp.distill_loss_and_grad(f, lists, teacher, one[:2]), lambda: cp.distill_loss_and_grad(f, lists, teacher, out=f.half()),
    ]
    for k, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was not refused" % k)
    cp.check_operator_status()


def test_tensors_that_require_a_gradient(cp, torch):
    """No graph is recorded, so a result that would be cut off from a tensor that wants a gradient is refused, not given."""
    f = torch.randn((4, 8), device="cuda", requires_grad=True)
    g = torch.randn((4, 8), device="cuda")
    i8 = torch.ones((4, 8), dtype=torch.int8, device="cuda")
    one, wanted = torch.ones(4, device="cuda"), torch.ones(4, device="cuda", requires_grad=True)
    ids = torch.arange(4, device="cuda")
    lists = torch.zeros((4, 2), dtype=torch.int64, device="cuda")
    teacher, learned = torch.zeros((4, 2), device="cuda"), torch.zeros((4, 2), device="cuda", requires_grad=True)
    calls = [
        lambda: cp.embedding_lookup(f, ids), lambda: cp.embedding_lookup(f * 2, ids), lambda: cp.embedding_grad(ids, f, 4), lambda: cp.quantize_rows(f),
        lambda: cp.int8_matmul(i8, wanted, i8, one), lambda: cp.int8_matmul(i8, one, i8, wanted), lambda: cp.distill_loss(f, lists, teacher),
        lambda: cp.distill_loss(g, lists, learned), lambda: cp.distill_loss_and_grad(g, lists, learned), lambda: cp.distill_loss_and_grad(f, lists, learned),
        lambda: cp.distill_loss_and_grad(f, lists, teacher, wanted),
    ]
    for k, call in enumerate(calls):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
            pytest.fail("call %d was not refused" % k)
        with torch.no_grad():
            call()
    # the logits' gradient is what this call returns: it goes on from there
    base = torch.randn((30, 8), device="cuda")
    loss, grad = cp.distill_loss_and_grad(f @ base.T, lists, teacher)
    assert not loss.requires_grad and not grad.requires_grad
    logits = f @ base.T
    logits.backward(cp.distill_loss_and_grad(logits, lists, teacher)[1])
    assert torch.equal(f.grad, grad @ base)
    assert torch.equal(cp.embedding_lookup(f.detach(), ids), f.detach())


def test_outputs_count_as_changed(cp, torch):
    """What is written to a caller's tensor autograd hears of, as of torch's own operations in place: a graph that had kept its
    values refuses to go back through them, instead of going with others."""
    f = torch.randn((4, 8), device="cuda", requires_grad=True)
    lists, teacher = torch.zeros((4, 2), dtype=torch.int64, device="cuda"), torch.zeros((4, 2), device="cuda")
    base = torch.randn((30, 8), device="cuda")
    i8, one, ids = torch.ones((4, 8), dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda"), torch.arange(4, device="cuda")
    for given in (lambda t: t, lambda t: t.detach()):
        logits = torch.exp(f @ base.T)  # (its derivative is its result)
        _, grad = cp.distill_loss_and_grad(given(logits), lists, teacher, out=given(logits))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            logits.backward(grad)
    # a graph that has not kept them goes on
    want = cp.distill_loss_and_grad((f @ base.T).detach(), lists, teacher)[1] @ base
    logits = f @ base.T
    logits.backward(cp.distill_loss_and_grad(logits, lists, teacher, out=logits)[1])
    assert torch.equal(f.grad, want)
    table, grad = torch.randn((4, 8), device="cuda"), torch.randn((4, 8), device="cuda")
    for write in (lambda out: cp.embedding_lookup(table, ids, out=out), lambda out: cp.embedding_grad(ids, grad, 4, out=out),
                  lambda out: cp.embedding_grad(ids, grad, 4, out=out, accumulate=True), lambda out: cp.distill_loss_and_grad(grad, lists, teacher, out=out)):
        out = torch.zeros((4, 8), device="cuda")
        before = out._version
        write(out)
        assert out._version > before
        with pytest.raises(ValueError, match="requires a gradient"):
            write(f)  # (a leaf: torch does not change one in place either)
        with pytest.raises(ValueError, match="requires a gradient"):
            write(f * 2)
    out = torch.zeros((4, 4), device="cuda")
    before = out._version
    cp.int8_matmul(i8, one, i8, one, out=out)
    assert out._version > before
    with torch.inference_mode():  # (tensors without a count)
        out = torch.zeros((4, 8), device="cuda")
        assert torch.equal(cp.embedding_lookup(table, ids, out=out), table)


def test_lookup_into_rows_at_several_distances(cp, torch):
    """Rows of `out` lie at one distance from one another; where they do not, it is refused like other wrong arguments."""
    table, ids = torch.randn((50, 24), device="cuda"), torch.arange(15, device="cuda").view(3, 5)
    room = torch.zeros((3, 5, 31), device="cuda")
    cp.embedding_lookup(table, ids, out=room[:, :, 2:26])
    assert torch.equal(room[:, :, 2:26], table[ids]) and not bool(room[:, :, :2].any()) and not bool(room[:, :, 26:].any())
    room = torch.zeros((3, 7, 24), device="cuda")
    with pytest.raises(ValueError, match="one distance"):
        cp.embedding_lookup(table, ids, out=room[:, :5])
    assert not bool(room.any())
