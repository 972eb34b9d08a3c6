"""`glide_b200.rows` against plain implementations in 64 bits.

Tolerances, derived from the operators' definition (u = 2^-24, half a step of fp32; h = half a step of the result's type,
eps / 2; both relative). A lookup rounds its product to fp32 and to the result's type: (u + h) |value|. A sum of m fp32 terms,
whatever their order, is off by at most m u times the sum of the terms' magnitudes, each term has rounded its own product
(u) and the scale rounds once more: (m + 2) u sum|term| + h |value|. Values below the smallest normal one of fp16 round to a
step of 2^-24, half of it 2^-25, which is added for fp16."""
import ctypes as C

import numpy as np
import pytest
import torch

from glide_b200 import api, rows

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, seed):
    return torch.randn(shape, generator=_gen(seed), device="cuda").to(dtype)


def _close(got, want, tol):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} values off, the worst by {off[bad].max().item():.3g} with {tol[bad].min().item() if torch.is_tensor(tol) else tol:.3g} allowed"


def _ids(shape, n, seed, empty=0.1):
    g = _gen(seed)
    ids = torch.randint(0, n, shape, generator=g, device="cuda", dtype=torch.int32)
    return torch.where(torch.rand(shape, generator=g, device="cuda") < empty, torch.full_like(ids, -1), ids)


def _strided(shape, dtype, seed, stride, offset=0):
    """A matrix whose rows lie `stride` values apart, `offset` values into its memory; and that memory."""
    whole = _randn((shape[0] * stride + offset + shape[1],), dtype, seed)
    return whole.as_strided(shape, (stride, 1), offset), whole


def _lookup_want(table, ids, scale):
    i = ids.long().reshape(-1)
    there = (i >= 0) & (i < table.shape[0])
    want = torch.zeros((i.numel(), table.shape[1]), dtype=torch.float64, device="cuda")
    want[there] = table[i[there]].double() * scale
    return want.reshape(*ids.shape, table.shape[1])


# ---- lookup --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES + [torch.uint8])
@pytest.mark.parametrize("n,dim,shape,scale", [(1, 1, (1,), 1.0), (7, 3, (5,), 2.5), (100, 100, (13, 10), 1.0), (1000, 128, (64, 10), 11.314),
                                               (50, 33, (1000,), 1.0), (300, 960, (301,), 0.1), (17, 4096, (3, 3), 64.0), (40, 1030, (2000,), 1.0),
                                               (700, 129, (3000,), 1.0), (300, 1001, (2400, 2), 1.5), (90, 520, (5000,), 1.0)])
def test_lookup(gpu_ctx, dtype, n, dim, shape, scale):
    table = torch.randint(0, 256, (n, dim), generator=_gen(1), device="cuda", dtype=torch.uint8) if dtype == torch.uint8 else _randn((n, dim), dtype, 1)
    ids = _ids(shape, n, 2)
    got = rows.lookup_rows(gpu_ctx, table, ids, scale)
    want = _lookup_want(table, ids, float(np.float32(scale)))
    assert got.dtype == (torch.float32 if dtype == torch.uint8 else dtype)
    _close(got, want, want.abs() * (U + _half(got.dtype)) + _floor(got.dtype))
    if scale == 1.0:
        assert torch.equal(got.double(), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stride,offset", [(128, 0), (136, 8), (129, 0), (130, 2), (128, 1), (132, 4)])
def test_lookup_takes_any_stride_and_leaves_what_lies_between_the_rows(gpu_ctx, dtype, stride, offset):
    table, _ = _strided((50, 128), dtype, 3, stride, offset)
    out, whole = _strided((70, 128), dtype, 4, stride, offset)
    before = whole.clone()
    ids = _ids((70,), 50, 5)
    rows.lookup_rows(gpu_ctx, table, ids, out=out)
    assert torch.equal(out.double(), _lookup_want(table, ids, 1.0))
    mask = torch.zeros_like(whole, dtype=torch.bool)
    mask.as_strided((70, 128), (stride, 1), offset).fill_(True)
    assert torch.equal(whole[~mask], before[~mask])


def test_lookup_ids_beyond_the_table_give_zeros_whatever_the_table_holds(gpu_ctx):
    table = torch.full((5, 64), float("nan"), device="cuda")
    ids = torch.tensor([5, -1, 2 ** 31 - 1, -2 ** 31, 6], dtype=torch.int32, device="cuda")
    assert torch.equal(rows.lookup_rows(gpu_ctx, table, ids, float("inf")), torch.zeros((5, 64), device="cuda"))
    got = rows.lookup_rows(gpu_ctx, table, torch.tensor([4, -1], dtype=torch.int32, device="cuda"))
    assert got[0].isnan().all() and (got[1] == 0).all()


def test_lookup_of_no_ids_and_of_a_broadcast_table(gpu_ctx):
    assert rows.lookup_rows(gpu_ctx, torch.zeros((3, 8), device="cuda"), torch.empty((0,), dtype=torch.int32, device="cuda")).shape == (0, 8)
    assert rows.lookup_rows(gpu_ctx, torch.zeros((3, 8), device="cuda"), torch.empty((0, 10), dtype=torch.int32, device="cuda")).shape == (0, 10, 8)
    one = _randn((1, 40), torch.float32, 6)
    ids = _ids((9,), 6, 7, 0.0)
    assert torch.equal(rows.lookup_rows(gpu_ctx, one.expand(6, 40), ids), one.expand(9, 40))


def test_lookup_offsets_pass_32_bits(gpu_ctx):
    n, dim = 2_100_000, 2_048      # 4.3e9 values
    table = torch.empty((n, dim), dtype=torch.float16, device="cuda")
    ids = torch.tensor([n - 1, 0, n - 2, 1_048_576, 2_097_152], dtype=torch.int32, device="cuda")
    table[ids.long()] = _randn((5, dim), torch.float16, 8)
    assert torch.equal(rows.lookup_rows(gpu_ctx, table, ids), table[ids.long()])
    grad = _randn((5, dim), torch.float16, 9)
    rows.lookup_rows_grad(gpu_ctx, grad, ids, n, out=table)
    assert torch.equal(table[ids.long()], grad)
    untouched = torch.ones(n, dtype=torch.bool, device="cuda")
    untouched[ids.long()] = False
    for part in (slice(0, 1000), slice(1_048_000, 1_049_000), slice(n - 10_000, n)):     # each holds rows that ids name
        assert (table[part][untouched[part]] == 0).all()


def test_more_pieces_than_a_launch_counts(gpu_ctx):
    """2,200,000 rows of 1,001 fp32 values, one value a piece: more than 2^31 pieces, so the calls are made of two launches."""
    count, dim = 2_200_000, 1_001
    table = _randn((7, dim), torch.float32, 26)
    ids = torch.randint(0, 7, (count,), generator=_gen(27), device="cuda", dtype=torch.int32)
    out = rows.lookup_rows(gpu_ctx, table, ids)

    def same(got, want_ids):
        return all(torch.equal(got[a:a + 100_000], table[want_ids[a:a + 100_000].long()]) for a in range(0, count, 100_000))
    assert same(out, ids)
    d = rows.dispatch_rows(gpu_ctx, out, ids[:, None].contiguous(), 7)
    assert same(d.d_sorted, torch.repeat_interleave(torch.arange(7, device="cuda"), torch.diff(d.d_segment_start).long()))
    out.zero_()
    rows.dispatch_rows_grad(gpu_ctx, d.d_sorted, d.d_position, out=out)
    assert same(out, ids)


# ---- gradient of a lookup ---------------------------------------------------------------------------------------

def _grad_want(grad, ids, n, scale):
    """The sum and the sum of magnitudes in 64 bits, and the number of terms of each row."""
    i = ids.long().reshape(-1)
    there = (i >= 0) & (i < n)
    g = grad.reshape(i.numel(), -1).double()[there] * scale
    want = torch.zeros((n, g.shape[1]), dtype=torch.float64, device="cuda").index_add_(0, i[there], g)
    size = torch.zeros_like(want).index_add_(0, i[there], g.abs())
    return want, size, torch.bincount(i[there], minlength=n).double()[:, None]


def _grad_tol(want, size, terms, dtype):
    return (terms + 2) * U * size + want.abs() * _half(dtype) + _floor(dtype)


@pytest.mark.parametrize("dtype,out_type", [(t, t) for t in TYPES] + [(torch.float16, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("n,dim,shape,scale", [(1, 1, (1,), 1.0), (3, 7, (200,), 1.0), (1, 64, (1000,), 0.5), (1000, 128, (50, 10), 1.0), (5000, 100, (3000,), 8.0),
                                               (70_000, 33, (5000,), 1.0), (40, 520, (777,), 22.8), (5_000_000, 8, (4100,), 1.0), (2000, 2048, (33,), 1.0)])
def test_lookup_grad(gpu_ctx, dtype, out_type, n, dim, shape, scale):
    grad, ids = _randn((*shape, dim), dtype, 10), _ids(shape, n, 11)
    got = rows.lookup_rows_grad(gpu_ctx, grad, ids, n, scale, dtype=out_type)
    want, size, terms = _grad_want(grad, ids, n, float(np.float32(scale)))
    assert got.dtype == out_type
    _close(got, want, _grad_tol(want, size, terms, out_type))
    assert (got[terms[:, 0] == 0] == 0).all()
    again = rows.lookup_rows_grad(gpu_ctx, grad, ids, n, scale, dtype=out_type)
    assert torch.equal(got, again)


@pytest.mark.parametrize("runs", [[1] * 100, [31, 1, 32, 33, 64, 65], [32, 32, 32], [33], [500, 1, 1, 30, 700], [16, 32, 48, 2], [8192], [2047, 2, 2047, 4096, 1], [5, 0, 0, 91, 0]])
@pytest.mark.parametrize("dim", [4, 96, 300])
def test_lookup_grad_runs_of_every_length(gpu_ctx, runs, dim):
    """Integer values: the sums are exact, so every element of the batch is in exactly one sum."""
    ids = torch.cat([torch.full((r,), i, dtype=torch.int32) for i, r in enumerate(runs)])
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(12))].cuda()
    grad = torch.randint(-50, 50, (ids.numel(), dim), generator=_gen(13), device="cuda").float()
    want = torch.zeros((len(runs), dim), dtype=torch.float64, device="cuda").index_add_(0, ids.long(), grad.double())
    assert torch.equal(rows.lookup_rows_grad(gpu_ctx, grad, ids, len(runs)).double(), want)


@pytest.mark.parametrize("count", [1, 2, 255, 256, 257, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 8192, 8193, 70_000, 140_000])
@pytest.mark.parametrize("n", [1, 2, 255, 256, 2047, 2048, 65_536, 4_194_304, 4_194_305])
def test_lookup_grad_sorts_every_size(gpu_ctx, count, n):
    ids = _ids((count,), n, 14, 0.05)
    grad = torch.randint(-50, 50, (count, 4), generator=_gen(15), device="cuda").float()
    there = ids >= 0
    want = torch.zeros((n, 4), dtype=torch.float64, device="cuda").index_add_(0, ids[there].long(), grad[there].double())
    assert torch.equal(rows.lookup_rows_grad(gpu_ctx, grad, ids, n).double(), want)


@pytest.mark.parametrize("count,n", [(5000, 1_000_000), (200_000, 1_000_000), (5000, 5_000_000), (200_000, 5_000_000)])
def test_lookup_grad_sorts_in_a_workspace_that_earlier_calls_have_used(gpu_ctx, count, n):
    """Two and three passes, two and three launches each, one call behind the other in the same workspace with other ids: what a pass reads is
    what the pass before it has placed in the same call, not in an earlier one."""
    lib, dim, calls = gpu_ctx.lib, 2, 20
    need = lib.glide_lookup_rows_grad_workspace(n, dim, count)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    ids = [_ids((count,), n, 140 + i, 0.02) for i in range(calls)]
    grad = torch.randint(-50, 50, (count, dim), generator=_gen(139), device="cuda").float()
    out = [torch.full((n, dim), float("nan"), device="cuda") for _ in range(calls)]
    stream = torch.cuda.current_stream().cuda_stream
    for i in range(calls):
        gpu_ctx.check(lib.glide_lookup_rows_grad(gpu_ctx.handle, grad.data_ptr(), 0, dim, ids[i].data_ptr(), count, 1.0, out[i].data_ptr(), 0, n, dim, dim, 0,
                                                 scratch.data_ptr(), need, stream))
    for i in range(calls):
        there = ids[i] >= 0
        want = torch.zeros((n, dim), dtype=torch.float64, device="cuda").index_add_(0, ids[i][there].long(), grad[there].double())
        assert torch.equal(out[i].double(), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_lookup_grad_accumulates_and_leaves_other_rows(gpu_ctx, dtype):
    base = _randn((500, 72), dtype, 16)
    base[499] = float("nan")
    grad, ids = _randn((60, 72), dtype, 17), _ids((60,), 400, 18)
    out = base.clone()
    assert rows.lookup_rows_grad(gpu_ctx, grad, ids, 500, 3.0, out=out, accumulate=True) is out
    want, size, terms = _grad_want(grad, ids, 500, 3.0)
    touched = terms[:, 0] > 0
    assert torch.equal(out[~touched].view(torch.int32 if dtype == torch.float32 else torch.int16), base[~touched].view(torch.int32 if dtype == torch.float32 else torch.int16))
    want += base.double()
    _close(out[touched], want[touched], ((terms + 3) * U * (size + base.double().abs()) + want.abs() * _half(dtype) + _floor(dtype))[touched])


def _often(count, n, seed):
    """Ids of which half are one and the same (a run over many chunks of the sorted list), an eighth another, the others any."""
    ids, which = _ids((count,), n, seed, 0.05), torch.rand((count,), generator=_gen(seed + 1), device="cuda")
    return torch.where(which < 0.5, n // 2, torch.where(which < 0.625, n - 2, ids)).int()


def _bits(t):
    return t.view(torch.int32 if t.dtype == torch.float32 else torch.int16)


@pytest.mark.parametrize("dtype,out_type", [(t, t) for t in TYPES] + [(torch.float16, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("count,n", [(1024, 300), (1025, 300), (2000, 5000), (6000, 40), (6000, 70_000), (30_000, 900), (30_000, 20_011)])
@pytest.mark.parametrize("dim,stride,offset", [(1, 1, 0), (33, 40, 1), (72, 72, 0), (520, 528, 8)])
def test_lookup_grad_accumulates_many_ids(gpu_ctx, dtype, out_type, count, n, dim, stride, offset):
    """Whole numbers: exact sums, rounded once with what was there. Rows that no id names, and what lies between the rows, hold NaN and keep it."""
    ids = _often(count, n - 1, 150)
    grad = torch.randint(-3, 4, (count, dim), generator=_gen(152), device="cuda").to(dtype)
    out, whole = _strided((n, dim), out_type, 153, stride, offset)
    whole.fill_(float("nan"))
    there = ids >= 0
    named = torch.zeros(n, dtype=torch.bool, device="cuda")
    named[ids[there].long()] = True
    base = torch.randint(-60, 61, (n, dim), generator=_gen(154), device="cuda").to(out_type)
    out[named] = base[named]
    before = whole.clone()
    want = base.double().index_add_(0, ids[there].long(), 2 * grad[there].double())
    assert rows.lookup_rows_grad(gpu_ctx, grad, ids, n, 2.0, out=out, accumulate=True) is out
    assert torch.equal(out[named], want.to(out_type)[named])
    assert not named[n - 1] and out[~named].isnan().all()
    mask = torch.zeros_like(whole, dtype=torch.bool)
    mask.as_strided((n, dim), (stride, 1), offset).fill_(True)
    assert torch.equal(_bits(whole)[~mask], _bits(before)[~mask])


def test_lookup_grad_accumulates_at_every_replay(gpu_ctx):
    ids = [_often(count, 3000, 155 + count) for count in (500, 2500, 9000)]
    grad = torch.randint(-3, 4, (9000, 40), generator=_gen(160), device="cuda").float()
    out = torch.zeros((3000, 40), device="cuda")

    def step():
        for i in ids:
            rows.lookup_rows_grad(gpu_ctx, grad[:i.numel()], i, 3000, out=out, accumulate=True)
    step()
    torch.cuda.synchronize()
    once = out.clone()
    assert once.abs().max() > 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(3):
        g.replay()
    assert torch.equal(out, once * 4)
    del g


@pytest.mark.parametrize("count,n,dtype,out_type,dim,stride,offset", [
    (5000, 1_000_003, torch.float32, torch.float32, 100, 100, 0),               # two launches a pass
    (70_000, 1_000_003, torch.float32, torch.float32, 100, 100, 0),             # three, each beside 48 MB that it clears, the rest by the join
    (70_000, 1_000_003, torch.bfloat16, torch.bfloat16, 201, 201, 3),           # rows of no whole words
    (140_000, 1_200_001, torch.bfloat16, torch.float32, 72, 80, 4),             # rows apart from one another
    (140_000, 600_000, torch.float16, torch.float16, 24, 24, 0),                # all cleared beside the sort
    (70_000, 4_300_000, torch.float16, torch.float16, 40, 41, 1),               # three passes
    (140_000, 4_300_000, torch.float32, torch.float32, 4, 4, 0)])
def test_lookup_grad_clears_large_tables(gpu_ctx, count, n, dtype, out_type, dim, stride, offset):
    """Every row that no id names is cleared, by whichever launch, and what lies between the rows is left alone."""
    out, whole = _strided((n, dim), out_type, 161, stride, offset)
    whole.fill_(float("nan"))
    ids = _ids((count,), n, 162)
    grad = torch.randint(-3, 4, (count, dim), generator=_gen(163), device="cuda").to(dtype)
    rows.lookup_rows_grad(gpu_ctx, grad, ids, n, out=out)
    there = ids >= 0
    want = torch.zeros((n, dim), device="cuda").index_add_(0, ids[there].long(), grad[there].float())     # whole numbers: exact
    assert torch.equal(out, want.to(out_type))
    if stride != dim:
        mask = torch.zeros_like(whole, dtype=torch.bool)
        mask.as_strided((n, dim), (stride, 1), offset).fill_(True)
        assert whole[~mask].isnan().all()


def test_lookup_grad_clears_rows_whose_offsets_pass_32_bits(gpu_ctx):
    n, dim = 2_100_000, 2_048      # 4.3e9 values
    out = torch.full((n, dim), 7.0, dtype=torch.float16, device="cuda")
    for count in (5, 3000, 9000):
        ids = torch.cat([torch.tensor([n - 1, 0, 2_097_152, 1_048_576, n - 2], dtype=torch.int32, device="cuda"), _ids((count - 5,), n, 164)])
        grad = torch.randint(-3, 4, (count, dim), generator=_gen(165), device="cuda").half()
        rows.lookup_rows_grad(gpu_ctx, grad, ids, n, out=out)
        there = ids >= 0
        which, back = torch.unique(ids[there].long(), return_inverse=True)
        want = torch.zeros((which.numel(), dim), device="cuda").index_add_(0, back, grad[there].float())
        assert torch.equal(out[which].float(), want)
        out[which] = 0
        assert all(not out[a:a + 100_000].any() for a in range(0, n, 100_000))
        out.fill_(7.0)


def test_lookup_grad_empty_places_take_no_part_whatever_they_hold(gpu_ctx):
    grad = _randn((40, 24), torch.float32, 19)
    ids = _ids((40,), 9, 20, 0.3)
    bad = torch.where((ids < 0)[:, None], torch.full_like(grad, float("nan")), grad)
    got = rows.lookup_rows_grad(gpu_ctx, bad, ids, 9)
    assert torch.equal(got, rows.lookup_rows_grad(gpu_ctx, grad, ids, 9)) and got.isfinite().all()
    none = torch.full((40,), -1, dtype=torch.int32, device="cuda")
    assert (rows.lookup_rows_grad(gpu_ctx, bad, none, 9) == 0).all()
    assert (rows.lookup_rows_grad(gpu_ctx, grad[:0], none[:0], 9) == 0).all()
    held = torch.ones((9, 24), device="cuda")
    rows.lookup_rows_grad(gpu_ctx, grad[:0], none[:0], 9, out=held, accumulate=True)
    assert (held == 1).all()


def test_lookup_grad_of_a_broadcast_gradient_and_strided_results(gpu_ctx):
    one, ids = _randn((1, 40), torch.float32, 21), torch.arange(12, dtype=torch.int32, device="cuda") // 3
    out, whole = _strided((6, 40), torch.float32, 22, 45, 3)
    before = whole.clone()
    rows.lookup_rows_grad(gpu_ctx, one.expand(12, 40), ids, 6, out=out)
    want = torch.cat([(one * 3).expand(4, 40), torch.zeros((2, 40), device="cuda")])
    _close(out, want.double(), want.double().abs() * 5 * U)
    mask = torch.zeros_like(whole, dtype=torch.bool)
    mask.as_strided((6, 40), (45, 1), 3).fill_(True)
    assert torch.equal(whole[~mask], before[~mask])


@pytest.mark.parametrize("dtype,out_type", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("count", [40, 1500, 6000, 30_000])
@pytest.mark.parametrize("dim,stride,offset", [(100, 108, 0), (100, 100, 3), (20, 33, 1), (1, 1, 0), (1, 3, 1), (5, 5, 1), (7, 8, 0), (136, 136, 1), (264, 271, 0)])
def test_lookup_grad_clears_what_no_id_names_and_nothing_else(gpu_ctx, dtype, out_type, count, dim, stride, offset):
    """Results of every alignment, with many more rows than ids (cleared beside the sort) and with few (cleared by the join)."""
    for n in (700, 20_011):
        out, whole = _strided((n, dim), out_type, 28, stride, offset)
        whole.fill_(float("nan"))
        ids = _ids((count,), n, 29)
        grad = torch.randint(-3, 4, (count, dim), generator=_gen(30), device="cuda").to(dtype)
        rows.lookup_rows_grad(gpu_ctx, grad, ids, n, out=out)
        there = ids >= 0
        want = torch.zeros((n, dim), dtype=torch.float64, device="cuda").index_add_(0, ids[there].long(), grad[there].double())
        assert torch.equal(out, want.to(out_type))        # whole numbers: exact sums, rounded once
        mask = torch.zeros_like(whole, dtype=torch.bool)
        mask.as_strided((n, dim), (stride, 1), offset).fill_(True)
        assert whole[~mask].isnan().all()


def test_ids_of_unsigned_type(gpu_ctx):
    table = _randn((50, 24), torch.float32, 31)
    ids = _ids((30,), 50, 32)
    assert torch.equal(rows.lookup_rows(gpu_ctx, table, ids.view(torch.uint32)), rows.lookup_rows(gpu_ctx, table, ids))
    data, choice = _randn((9, 24), torch.float32, 33), _ids((9, 2), 4, 34)
    a, b = rows.dispatch_rows(gpu_ctx, data, choice, 4), rows.dispatch_rows(gpu_ctx, data, choice.view(torch.uint32), 4)
    assert b.d_map.dtype == torch.uint32 and torch.equal(a.d_position, b.d_position.view(torch.int32))
    assert torch.equal(rows.dispatch_rows_grad(gpu_ctx, b.d_sorted, b.d_position), rows.dispatch_rows_grad(gpu_ctx, a.d_sorted, a.d_position))


def test_lookup_grad_is_the_derivative_of_lookup(gpu_ctx):
    """A linear map: <lookup(X), G> = <X, grad(G)> for any X and G. The products are of values of fp32, the sums in 64 bits; each side's
    fp32 rounding is bounded as above, by (terms + 3) u of the magnitudes."""
    ids = _ids((30, 7), 90, 23)
    x, g = _randn((90, 50), torch.float32, 24), _randn((30, 7, 50), torch.float32, 25)
    left = (rows.lookup_rows(gpu_ctx, x, ids, 1.7).double() * g.double()).sum()
    got = rows.lookup_rows_grad(gpu_ctx, g, ids, 90, 1.7)
    right = (x.double() * got.double()).sum()
    _, size, terms = _grad_want(g, ids, 90, 1.7)
    assert (left - right).abs() <= ((terms + 3) * U * size * x.double().abs()).sum()


# ---- dispatch --------------------------------------------------------------------------------------------------

def _choice(count, choices, partitions, seed, empty=0.1, skew=False):
    c = _ids((count, choices), max(1, partitions // 8) if skew else partitions, seed, empty)
    return c


def _dispatch_want(choice, partitions):
    c = choice.cpu().numpy().astype(np.int64).reshape(-1)
    place = np.flatnonzero((c >= 0) & (c < partitions))
    place = place[np.lexsort((place, c[place]))]
    position = np.full(c.size, -1, np.int32)
    position[place] = np.arange(place.size, dtype=np.int32)
    which = np.full(c.size, -1, np.int32)
    which[:place.size] = place // choice.shape[1]
    start = np.concatenate([[0], np.cumsum(np.bincount(c[place], minlength=partitions))]).astype(np.int32)
    return position.reshape(choice.shape), which, start


def _check_dispatch(got, data, choice, partitions):
    position, which, start = _dispatch_want(choice, partitions)
    assert np.array_equal(got.d_segment_start.cpu().numpy(), start)
    assert np.array_equal(got.d_position.cpu().numpy(), position)
    assert np.array_equal(got.d_map.cpu().numpy(), which)
    taken = int(start[-1])
    assert torch.equal(got.d_sorted[:taken], data[torch.from_numpy(which[:taken]).long().cuda()])
    return taken


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,dim,choices,partitions", [(1, 1, 1, 1), (1, 64, 8, 64), (3, 100, 2, 5), (64, 256, 8, 256), (500, 33, 3, 7), (257, 520, 1, 1024), (2049, 12, 2, 4096),
                                                          (1000, 8, 128, 130), (5000, 40, 2, 1), (9, 4096, 4, 3), (300, 130, 6, 2048), (20_001, 6, 2, 300), (2500, 129, 3, 40), (2400, 1001, 2, 5), (3000, 2048, 2, 64)])
def test_dispatch(gpu_ctx, dtype, count, dim, choices, partitions):
    data, choice = _randn((count, dim), dtype, 30), _choice(count, choices, partitions, 31)
    keep = _randn((count * choices, dim), dtype, 32)
    out = keep.clone()
    got = rows.dispatch_rows(gpu_ctx, data, choice, partitions, out=out)
    assert got.d_sorted is out
    taken = _check_dispatch(got, data, choice, partitions)
    assert torch.equal(out[taken:], keep[taken:])          # rows behind the last place stay


@pytest.mark.parametrize("pairs", [1, 2, 31, 32, 33, 255, 256, 257, 1023, 1024, 1025, 2047, 2048, 2049, 4096, 8191, 8193, 65_537, 300_000])
@pytest.mark.parametrize("partitions", [1, 2, 33, 255, 1024, 4096])
@pytest.mark.parametrize("skew", [False, True])
def test_dispatch_sorts_every_size(gpu_ctx, pairs, partitions, skew):
    data, choice = torch.arange(pairs, device="cuda", dtype=torch.float32)[:, None].contiguous(), _choice(pairs, 1, partitions, 33, 0.05, skew)
    _check_dispatch(rows.dispatch_rows(gpu_ctx, data, choice, partitions), data, choice, partitions)


def test_dispatch_without_any_choice_and_without_rows(gpu_ctx):
    data = _randn((50, 16), torch.bfloat16, 34)
    out = torch.ones((100, 16), dtype=torch.bfloat16, device="cuda")
    got = rows.dispatch_rows(gpu_ctx, data, torch.full((50, 2), -1, dtype=torch.int32, device="cuda"), 6, out=out)
    assert (got.d_position == -1).all() and (got.d_map == -1).all() and (got.d_segment_start == 0).all() and (out == 1).all()
    got = rows.dispatch_rows(gpu_ctx, data[:0], torch.empty((0, 2), dtype=torch.int32, device="cuda"), 6)
    assert got.d_sorted.shape == (0, 16) and got.d_map.shape == (0,) and got.d_position.shape == (0, 2)
    assert (got.d_segment_start == 0).all() and got.d_segment_start.shape == (7,)


def test_dispatch_choices_out_of_range_and_the_same_partition_twice(gpu_ctx):
    data = _randn((4, 8), torch.float32, 35)
    choice = torch.tensor([[2, 2], [4, 5], [-7, 0], [2 ** 31 - 1, 3]], dtype=torch.int32, device="cuda")
    got = rows.dispatch_rows(gpu_ctx, data, choice, 4)
    assert _check_dispatch(got, data, choice, 4) == 4
    back = rows.dispatch_rows_grad(gpu_ctx, got.d_sorted, got.d_position)
    assert torch.equal(back, torch.stack([data[0] * 2, data[1] * 0, data[2], data[3]]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stride,offset", [(64, 0), (72, 8), (65, 0), (66, 2), (64, 1)])
def test_dispatch_and_back_take_any_stride(gpu_ctx, dtype, stride, offset):
    data, _ = _strided((90, 64), dtype, 36, stride, offset)
    choice = _choice(90, 2, 7, 37)
    out, whole = _strided((180, 64), dtype, 38, stride, offset)
    before = whole.clone()
    got = rows.dispatch_rows(gpu_ctx, data, choice, 7, out=out)
    taken = _check_dispatch(got, data, choice, 7)
    mask = torch.zeros_like(whole, dtype=torch.bool)
    mask.as_strided((taken, 64), (stride, 1), offset).fill_(True)
    assert torch.equal(whole[~mask], before[~mask])
    back, whole = _strided((90, 64), dtype, 39, stride, offset)
    before = whole.clone()
    rows.dispatch_rows_grad(gpu_ctx, got.d_sorted, got.d_position, out=back)
    assert torch.equal(back, data * (choice >= 0).sum(1, keepdim=True).to(dtype))      # at most twice a value: exact
    mask = torch.zeros_like(whole, dtype=torch.bool)
    mask.as_strided((90, 64), (stride, 1), offset).fill_(True)
    assert torch.equal(whole[~mask], before[~mask])


# ---- combine ---------------------------------------------------------------------------------------------------

def _combine_case(dtype, count, dim, choices, empty, seed):
    """Positions as dispatch makes them: distinct, some missing, rows behind the last that no position names."""
    choice = _choice(count, choices, max(1, choices * 2), seed, empty)
    position = torch.from_numpy(_dispatch_want(choice, max(1, choices * 2))[0]).cuda()
    return _randn((count * choices, dim), dtype, seed + 1), position, torch.rand((count, choices), generator=_gen(seed + 2), device="cuda") * 2 - 1


COMBINE = [(1, 1, 1, 0.0), (1, 64, 8, 0.0), (64, 2048, 8, 0.1), (301, 100, 2, 0.2), (77, 33, 3, 0.1), (19, 1030, 9, 0.1), (40, 12, 128, 0.5), (1000, 520, 1, 0.1), (5000, 24, 4, 0.1), (33, 130, 17, 0.0), (2500, 129, 3, 0.3),
           (2400, 1001, 2, 0.1), (2400, 1001, 5, 0.1), (2500, 520, 6, 0.6), (2400, 258, 9, 0.1), (1100, 600, 9, 0.1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("count,dim,choices,empty", COMBINE)
def test_combine(gpu_ctx, dtype, weighted, count, dim, choices, empty):
    data, position, weights = _combine_case(dtype, count, dim, choices, empty, 40)
    got = rows.combine_rows(gpu_ctx, data, position, weights if weighted else None)
    there = (position >= 0)[..., None]
    term = torch.where(there, data[position.clamp(min=0).long()].double() * (weights[..., None].double() if weighted else 1.0), 0.0)
    want = term.sum(1)
    assert got.dtype == dtype
    _close(got, want, (choices + 2) * U * term.abs().sum(1) + want.abs() * _half(dtype) + _floor(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("count,dim,choices,empty", COMBINE)
def test_combine_grad(gpu_ctx, dtype, weighted, count, dim, choices, empty):
    data, position, weights = _combine_case(dtype, count, dim, choices, empty, 43)
    grad = _randn((count, dim), dtype, 47)
    keep = _randn((count * choices, dim), dtype, 48)
    out = keep.clone()
    got, got_w = rows.combine_rows_grad(gpu_ctx, grad, data, position, weights if weighted else None, out=out)
    assert got is out and got_w.dtype == torch.float32
    there = position >= 0
    want = (grad.double()[:, None] * (weights[..., None].double() if weighted else 1.0)).expand(count, choices, dim)
    at = position[there].long()
    _close(out[at], want[there], want[there].abs() * (U + _half(dtype)) + _floor(dtype))
    rest = torch.ones(count * choices, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert torch.equal(out[rest], keep[rest])
    term = torch.where(there[..., None], data[position.clamp(min=0).long()].double() * grad.double()[:, None], 0.0)
    _close(got_w, term.sum(2), (dim + 2) * U * term.abs().sum(2) + 2.0 ** -126)
    assert (got_w[~there] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,dim,choices,empty", [(0, 40, 3, 0.0), (1, 24, 1, 1.0), (64, 512, 2, 0.4), (700, 33, 8, 0.3), (3000, 128, 2, 0.5)])
def test_combine_grad_makes_zeros_of_rows_without_a_place(gpu_ctx, dtype, count, dim, choices, empty):
    """A result that the call itself makes, in memory that held NaN before; with more sorted rows than pairs, too."""
    data, position, weights = _combine_case(dtype, count, dim, choices, empty, 56)
    grad = _randn((count, dim), dtype, 59)
    for more in (0, 5):
        data = torch.cat([data, _randn((more, dim), dtype, 58)])
        torch.full(data.shape, float("nan"), dtype=dtype, device="cuda")      # goes back to the allocator, which gives it out again
        got, _ = rows.combine_rows_grad(gpu_ctx, grad, data, position, weights)
        there = position >= 0
        at = position[there].long()
        want = torch.zeros(data.shape, dtype=torch.float64, device="cuda")
        want[at] = (grad.double()[:, None] * weights[..., None].double())[there]
        _close(got, want, want.abs() * (U + _half(dtype)) + _floor(dtype))
        rest = torch.ones(data.shape[0], dtype=torch.bool, device="cuda")
        rest[at] = False
        assert (got[rest] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,dim,choices,empty", [(16_000, 600, 4, 0.02), (9001, 1001, 8, 0.6), (50_000, 520, 2, 0.0), (70_000, 520, 1, 1.0)])
def test_combine_grad_makes_zeros_in_large_results(gpu_ctx, dtype, count, dim, choices, empty):
    """More bytes than are cleared whole, places in any order, memory that held NaN: as with a result of zeros that is handed in."""
    data, position, weights = _combine_case(dtype, count, dim, choices, empty, 68)
    place = torch.randperm(count * choices, generator=_gen(71), device="cuda").int()
    position = torch.where(position >= 0, place[position.clamp(min=0).long()], -1).contiguous()
    grad = _randn((count, dim), dtype, 72)
    assert data.numel() * data.element_size() > rows._FEW_BYTES
    want, want_w = rows.combine_rows_grad(gpu_ctx, grad, data, position, weights, out=torch.zeros_like(data))
    torch.full(data.shape, float("nan"), dtype=dtype, device="cuda")
    got, got_w = rows.combine_rows_grad(gpu_ctx, grad, data, position, weights)
    assert torch.equal(got, want) and torch.equal(got_w, want_w)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,stride,offset", [(1, 1, 1), (1, 3, 0), (5, 5, 1), (7, 8, 0), (8, 8, 0), (20, 33, 1), (100, 100, 3), (136, 136, 1), (264, 271, 0), (40_000, 40_001, 1), (70_000, 70_000, 0)])
def test_rows_without_a_place_are_cleared_and_nothing_else(gpu_ctx, dtype, dim, stride, offset):
    """None, some and all of the rows with a place, positions beyond the rows, the same position twice; in captured calls, too."""
    lib, stream = gpu_ctx.lib, torch.cuda.current_stream().cuda_stream
    for n in (1, 31, 32, 33, 255, 256, 257, 1000):
        if n * dim > 20_000_000:
            continue
        scratch = torch.full((lib.glide_clear_rows_without_place_workspace(n),), 255, dtype=torch.uint8, device="cuda")
        for share in (0.0, 0.4, 0.97, 1.0):
            named = torch.rand((n,), generator=_gen(170 + n), device="cuda") < share
            at = torch.nonzero(named).reshape(-1).int()
            position = torch.cat([at, torch.tensor([-1, n, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), at[:3]])[torch.randperm(at.numel() + 3 + at[:3].numel(), device="cuda")]
            held, whole = _strided((n, dim), dtype, 171, stride, offset)
            whole.fill_(float("nan"))
            gpu_ctx.check(lib.glide_clear_rows_without_place(gpu_ctx.handle, held.data_ptr(), rows._FLOATS[dtype], n, dim, stride, position.data_ptr(), position.numel(),
                                                             scratch.data_ptr(), scratch.numel(), stream))
            assert held[named].isnan().all() and (held[~named] == 0).all()
            mask = torch.zeros_like(whole, dtype=torch.bool)
            mask.as_strided((n, dim), (stride, 1), offset).fill_(True)
            assert whole[~mask].isnan().all()
    held = torch.ones((4, dim), dtype=dtype, device="cuda")
    gpu_ctx.check(lib.glide_clear_rows_without_place(gpu_ctx.handle, held.data_ptr(), rows._FLOATS[dtype], 4, dim, dim, None, 0, scratch.data_ptr(), scratch.numel(), stream))
    assert not held.any()


def test_clearing_rows_without_a_place_is_captured_and_its_refusals(gpu_ctx):
    lib, h = gpu_ctx.lib, gpu_ctx.handle
    held, position = torch.ones((5000, 40), device="cuda"), torch.arange(0, 5000, 2, dtype=torch.int32, device="cuda")
    scratch = torch.full((lib.glide_clear_rows_without_place_workspace(5000),), 255, dtype=torch.uint8, device="cuda")
    H, P, W, S = held.data_ptr(), position.data_ptr(), scratch.data_ptr(), scratch.numel()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        gpu_ctx.check(lib.glide_clear_rows_without_place(h, H, 0, 5000, 40, 40, P, 2500, W, S, torch.cuda.current_stream().cuda_stream))
    for shift in (0, 1):
        held.fill_(1)
        position.copy_(torch.arange(shift, 5000, 2, dtype=torch.int32, device="cuda"))
        g.replay()
        assert (held[shift::2] == 1).all() and (held[1 - shift::2] == 0).all()
    del g
    held.fill_(1)

    def clear(code, r=H, kind=0, n=5000, dim=40, stride=40, p=P, pairs=2500, w=W, wb=S):
        assert lib.glide_clear_rows_without_place(h, r, kind, n, dim, stride, p, pairs, w, wb, None) == code
        assert code == 0 or len(lib.glide_last_error(h)) > 10

    clear(0, n=0)
    for wrong in (dict(r=None), dict(p=None), dict(w=None), dict(wb=S - 1), dict(dim=0), dict(stride=39), dict(r=H + 2), dict(p=P + 1), dict(w=W + 16), dict(p=H), dict(w=H), dict(stride=1 << 60)):
        clear(-1, **wrong)
    for wrong in (dict(kind=1), dict(kind=4), dict(dim=1 << 21), dict(n=1 << 31), dict(pairs=1 << 31)):
        clear(-2, **wrong)
    torch.cuda.synchronize()
    assert (held == 1).all()


def test_combine_leaves_out_what_has_no_place_whatever_it_would_hold(gpu_ctx):
    data = _randn((6, 40), torch.float32, 50)
    data[5] = float("nan")
    weights = torch.tensor([[0.5, float("nan")], [float("inf"), float("nan")], [1.0, 0.0]], device="cuda")
    position = torch.tensor([[0, -1], [-1, 6], [1, 2]], dtype=torch.int32, device="cuda")
    data[2] = float("inf")
    got = rows.combine_rows(gpu_ctx, data, position, weights)
    assert torch.equal(got[0], data[0] * 0.5) and (got[1] == 0).all() and got[2].isnan().all()     # 0 x inf is NaN, as everywhere
    grad = torch.full((3, 40), float("nan"), device="cuda")
    keep = torch.ones((6, 40), device="cuda")
    _, got_w = rows.combine_rows_grad(gpu_ctx, grad, data, position, weights, out=keep)
    assert got_w[0, 1] == 0 and (got_w[1] == 0).all() and got_w[0, 0].isnan()
    assert keep[:3].isnan().all() and (keep[3:] == 1).all()


@pytest.mark.parametrize("count,dim,choices", [(40, 64, 2), (900, 600, 9), (3000, 96, 8)])
def test_combine_grad_without_the_gradient_of_the_weights(gpu_ctx, count, dim, choices):
    """The C entry point takes null for it (and null for the weights): the gradient of the sorted rows is the same."""
    data, position, weights = _combine_case(torch.bfloat16, count, dim, choices, 0.2, 62)
    grad = _randn((count, dim), torch.bfloat16, 66)
    for w in (weights, None):
        want, _ = rows.combine_rows_grad(gpu_ctx, grad, data, position, w)
        got = torch.zeros_like(data)
        gpu_ctx.check(gpu_ctx.lib.glide_combine_rows_grad(gpu_ctx.handle, grad.data_ptr(), 3, count, dim, dim, data.data_ptr(), data.shape[0], dim, position.data_ptr(),
                                                          choices, None if w is None else w.data_ptr(), got.data_ptr(), dim, None, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(got, want) and got.any()


def test_dispatch_and_back_where_offsets_pass_32_bits(gpu_ctx):
    count, dim, choices = 1_100_000, 2_048, 2      # 4.5e9 values sorted
    data = torch.empty((count, dim), dtype=torch.float16, device="cuda")
    data[:] = (torch.arange(count, device="cuda") % 2003 - 1001).half()[:, None]
    data[:, 5] = (torch.arange(count, device="cuda") % 1999).half()
    choice = _choice(count, choices, 3, 67)
    d = rows.dispatch_rows(gpu_ctx, data, choice, 3)
    _, which, start = _dispatch_want(choice, 3)
    taken = int(start[-1])
    assert taken * dim < 2 ** 32 < count * choices * dim
    for a in list(range(0, taken, 200_000)):
        assert torch.equal(d.d_sorted[a:min(a + 200_000, taken)], data[d.d_map[a:min(a + 200_000, taken)].long()])
    assert np.array_equal(d.d_map.cpu().numpy(), which)
    moved = torch.where(d.d_position >= 0, count * choices - 1 - d.d_position, -1)      # the same rows from the other end, beyond 2^32 values
    flipped = d.d_sorted.flip(0)
    times = (choice >= 0).sum(1, keepdim=True).half()
    for position, held in ((d.d_position, d.d_sorted), (moved, flipped)):
        back = rows.dispatch_rows_grad(gpu_ctx, held, position)
        assert all(torch.equal(back[a:a + 100_000], data[a:a + 100_000] * times[a:a + 100_000]) for a in range(0, count, 100_000))
    got, got_w = rows.combine_rows_grad(gpu_ctx, data, flipped, moved)
    got = got.flip(0)
    assert all(torch.equal(got[a:min(a + 200_000, taken)], d.d_sorted[a:min(a + 200_000, taken)]) for a in range(0, taken, 200_000))
    assert not got[taken:].any()
    size = torch.cat([(part.double() ** 2).sum(1) for part in data.split(100_000)])[:, None]
    _close(got_w, torch.where(choice >= 0, size, 0.0), (dim + 2) * U * size)


def test_combine_of_nothing(gpu_ctx):
    none = torch.empty((0, 3), dtype=torch.int32, device="cuda")
    assert rows.combine_rows(gpu_ctx, torch.zeros((5, 8), device="cuda"), none).shape == (0, 8)
    assert (rows.combine_rows(gpu_ctx, torch.zeros((0, 8), device="cuda"), torch.full((4, 3), -1, dtype=torch.int32, device="cuda")) == 0).all()
    out, w = rows.combine_rows_grad(gpu_ctx, torch.zeros((0, 8), device="cuda"), torch.zeros((5, 8), device="cuda"), none, out=torch.ones((5, 8), device="cuda"))
    assert (out == 1).all() and w.shape == (0, 3)


def test_gradients_against_differences(gpu_ctx):
    """combine(Y, w) is linear in Y and in w: a difference over a step of 1 is the derivative up to the rounding of fp32 results, of
    which each side has at most (choices + 3) u (or (dim + 3) u) of the magnitudes."""
    data, position, weights = _combine_case(torch.float32, 50, 36, 3, 0.2, 51)
    grad = _randn((50, 36), torch.float32, 55)
    g_data, g_weights = rows.combine_rows_grad(gpu_ctx, grad, data, position, weights, out=torch.zeros_like(data))
    base = rows.combine_rows(gpu_ctx, data, position, weights).double()
    size = rows.combine_rows(gpu_ctx, data.abs(), position, weights.abs()).double()
    for seed in range(3):
        d_data, d_weights = _randn(data.shape, torch.float32, 60 + seed), _randn(weights.shape, torch.float32, 70 + seed)
        moved = (data.double() + d_data.double())
        step = (moved.float().double() - data.double())                          # the step that fp32 really takes
        left = ((rows.combine_rows(gpu_ctx, moved.float(), position, weights).double() - base) * grad.double()).sum()
        right = (step * g_data.double()).sum()
        m = rows.combine_rows(gpu_ctx, moved.float().abs(), position, weights.abs()).double()
        bound = ((size + m) * 8 * U * grad.double().abs()).sum() + (step.abs() * g_data.double().abs()).sum() * 2 * U
        assert (left - right).abs() <= bound
        moved = (weights.double() + d_weights.double())
        step = (moved.float().double() - weights.double())
        left = ((rows.combine_rows(gpu_ctx, data, position, moved.float()).double() - base) * grad.double()).sum()
        there = (position >= 0).double()
        right = (step * g_weights.double()).sum()
        m = rows.combine_rows(gpu_ctx, data.abs(), position, moved.float().abs()).double()
        dots = torch.where(position[..., None] >= 0, data[position.clamp(min=0).long()].double() * grad.double()[:, None], 0.0).abs().sum(2)
        bound = ((size + m) * 8 * U * grad.double().abs()).sum() + (step.abs() * there * dots).sum() * 40 * U
        assert (left - right).abs() <= bound


# ---- together, streams, graphs -----------------------------------------------------------------------------------

def test_experts_by_the_partitions_of_an_index(gpu_ctx):
    """Rows to their two nearest k-means partitions, an expert (a matrix) for each, back with weights; and the gradients of all of it,
    against the same in 64 bits. Integer values keep the experts' products exact, so tolerances are those of the operators."""
    ctx, parts, k, dim = gpu_ctx, 12, 2, 32
    data = torch.randint(-4, 5, (700, dim), generator=_gen(80), device="cuda").float()
    centroids, _ = api.get_centroids(ctx, data, parts, 0.5, seed=3)
    choice, dist = api.bruteforce_knn(ctx, centroids, data, k)
    weights = torch.softmax(-dist, dim=1)
    experts = torch.randint(-2, 3, (parts, dim, dim), generator=_gen(81), device="cuda").float()
    d = rows.dispatch_rows(ctx, data, choice, parts)
    start = d.d_segment_start.tolist()
    assert start[-1] == 700 * k
    through = torch.empty_like(d.d_sorted)
    for e in range(parts):
        through[start[e]:start[e + 1]] = (d.d_sorted[start[e]:start[e + 1]].double() @ experts[e].double()).float()
    out = rows.combine_rows(ctx, through, d.d_position, weights)
    grad = torch.randint(-3, 4, (700, dim), generator=_gen(82), device="cuda").float()
    g_through, g_weights = rows.combine_rows_grad(ctx, grad, through, d.d_position, weights)
    g_sorted = torch.empty_like(g_through)
    for e in range(parts):
        g_sorted[start[e]:start[e + 1]] = (g_through[start[e]:start[e + 1]].double() @ experts[e].double().t()).float()
    g_data = rows.dispatch_rows_grad(ctx, g_sorted, d.d_position)

    x = data.double().requires_grad_()
    w = weights.double().requires_grad_()
    y = torch.einsum("td,tkde->tke", x, experts.double()[choice.long()])
    want = (y * w[..., None]).sum(1)
    want.backward(grad.double())
    size = (y.abs() * w[..., None]).sum(1).detach()
    _close(out, want.detach(), (k + 3) * U * size)
    _close(g_weights, w.grad, (dim + 2) * U * (y.abs() * grad.double().abs()[:, None]).sum(2).detach())
    # each of the k terms: w g rounded (u), the product with the expert rounded once to fp32 (u), the sum of k
    each = (torch.einsum("te,tkde->tkd", grad.double().abs(), experts.double().abs()[choice.long()]) * w.detach()[..., None]).sum(1)
    _close(g_data, x.grad, (k + 4) * U * each)


def test_a_search_a_lookup_and_the_gradient_of_the_rows_found(gpu_ctx):
    ctx = gpu_ctx
    table, queries = _randn((3000, 48), torch.float32, 83), _randn((40, 48), torch.float32, 84)
    ids, _ = api.bruteforce_knn(ctx, table, queries, 10)
    found = rows.lookup_rows(ctx, table, ids)
    assert torch.equal(found, table[ids.long()])
    index = api.GLIDE(ctx, 16, table, table[:4])
    assert torch.equal(index.lookup(ids), found) and torch.equal(index.lookup(ids, 2.0), found * 2)
    grad = torch.randint(-9, 10, found.shape, generator=_gen(85), device="cuda").float()
    got = rows.lookup_rows_grad(ctx, grad, ids, 3000)
    want = torch.zeros((3000, 48), device="cuda").index_add_(0, ids.long().reshape(-1), grad.reshape(-1, 48))
    assert torch.equal(got, want)


def test_an_index_looks_up_what_its_own_search_returned(gpu_ctx):
    """Arrays on the host, of ``search`` and of ``search_host``: with places that a search leaves unfilled, in any shape and order."""
    from glide_b200.params import SearchParameter
    g = torch.Generator().manual_seed(86)
    data, queries = torch.rand((500, 24), generator=g), torch.rand((9, 24), generator=g)
    index = api.GLIDE(gpu_ctx, 32, data, data[:2])
    index.load(torch.randint(0, 500, (500, 32), generator=g).numpy().astype(np.uint32), np.array([3, 77], np.uint32))
    param = SearchParameter(top_k=10, beam=32).derive(32)
    ids, _, _ = index.search(param, queries.cuda())
    host_ids, _ = index.search_host(param, queries.numpy())
    assert isinstance(ids, np.ndarray) and np.array_equal(ids, host_ids)
    ids[4, 7:] = api.INVALID
    want = torch.cat([data, torch.zeros((1, 24))])[torch.from_numpy(np.minimum(ids, 500).astype(np.int64))].cuda()
    assert torch.equal(index.lookup(ids), want) and torch.equal(index.lookup(ids, 2.0), want * 2)
    assert torch.equal(index.lookup(ids.view(np.int32)), want)
    assert torch.equal(index.lookup(ids.T[::-1, 1:]), want.transpose(0, 1).flip(0)[:, 1:])
    assert torch.equal(index.lookup(ids[0, 0].reshape(())), want[0, 0]) and index.lookup(ids[:0]).shape == (0, 10, 24)
    for bad in (ids.astype(np.int64), ids.astype(np.float32), ids.tolist()):
        with pytest.raises(TypeError):
            index.lookup(bad)


def test_calls_run_on_the_current_stream(gpu_ctx):
    """Two streams work at once, each on what its own earlier work leaves behind, without a wait on the host between."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    base = _randn((4096, 256), torch.float32, 90)
    ids = [_ids((20_000,), 4096, 91 + i) for i in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            table = base.clone()
            for _ in range(20):
                table = table * 1.0 + 1.0
            found = rows.lookup_rows(gpu_ctx, table, ids[i])
            got.append((table, found, rows.lookup_rows_grad(gpu_ctx, found, ids[i], 4096)))
    torch.cuda.synchronize()
    for i in range(2):
        table, found, grad = got[i]
        assert torch.equal(found.double(), _lookup_want(table, ids[i], 1.0))
        want, size, terms = _grad_want(found, ids[i], 4096, 1.0)
        _close(grad, want, _grad_tol(want, size, terms, torch.float32))


@pytest.mark.parametrize("shape", [1, 3, 10])       # one launch, few ids, tiles
def test_calls_are_captured_and_replayed(gpu_ctx, shape):
    """One graph of all operators, replayed on new inputs in the same tensors, gives the bits of the calls themselves; a second graph, captured
    while the first lives, does not disturb it."""
    ctx, parts = gpu_ctx, 40
    table, ids = _randn((5000, 96), torch.bfloat16, 100), _ids((700, shape), 5000, 101)
    data, choice = _randn((1500, 96), torch.bfloat16, 102), _choice(1500, 4, parts, 103)
    weights = torch.rand((1500, 4), generator=_gen(104), device="cuda")
    keep, keep2 = torch.zeros((6000, 96), dtype=torch.bfloat16, device="cuda"), torch.zeros((6000, 96), dtype=torch.bfloat16, device="cuda")

    def work():
        found = rows.lookup_rows(ctx, table, ids, 2.0)
        g_table = rows.lookup_rows_grad(ctx, found, ids, 5000, 2.0, dtype=torch.float32)
        d = rows.dispatch_rows(ctx, data, choice, parts, out=keep)
        back = rows.combine_rows(ctx, d.d_sorted, d.d_position, weights)
        g_sorted, g_weights = rows.combine_rows_grad(ctx, back, d.d_sorted, d.d_position, weights, out=keep2)
        return [found, g_table, d.d_sorted, d.d_map, d.d_position, d.d_segment_start, back, g_sorted, g_weights]

    work()
    torch.cuda.synchronize()
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(work())
        graphs.append(g)
    for seed in (110, 120):
        table.copy_(_randn(table.shape, torch.bfloat16, seed))
        ids.copy_(_ids((700, shape), 5000, seed + 1))
        data.copy_(_randn(data.shape, torch.bfloat16, seed + 2))
        choice.copy_(_choice(1500, 4, parts, seed + 3, 0.4))
        for g, r in zip(graphs, results):
            keep.zero_()
            keep2.zero_()
            g.replay()
            torch.cuda.synchronize()
            replayed = [x.clone() for x in r]
            keep.zero_()
            keep2.zero_()
            for x, y in zip(replayed, work()):
                assert torch.equal(x, y)
    del graphs, results


def test_two_threads_with_a_context_each(gpu_ctx):
    import threading
    table = _randn((30_000, 64), torch.float32, 130)
    work = []
    for i in range(2):
        ids, data, choice = _ids((9000 + i,), 30_000, 131 + i), _randn((5000, 40), torch.float32, 133 + i), _choice(5000, 2, 300, 135 + i)
        work.append((api.Context(0), torch.cuda.Stream(), ids, data, choice))
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        ctx, stream, ids, data, choice = work[i]
        with torch.cuda.stream(stream):
            for _ in range(10):
                d = rows.dispatch_rows(ctx, data, choice, 300)
                got[i] = [rows.lookup_rows_grad(ctx, rows.lookup_rows(ctx, table, ids), ids, 30_000), rows.dispatch_rows_grad(ctx, d.d_sorted, d.d_position), *d[1:]]
        stream.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for i in range(2):
        _, _, ids, data, choice = work[i]
        d = rows.dispatch_rows(gpu_ctx, data, choice, 300)
        want = [rows.lookup_rows_grad(gpu_ctx, rows.lookup_rows(gpu_ctx, table, ids), ids, 30_000), rows.dispatch_rows_grad(gpu_ctx, d.d_sorted, d.d_position), *d[1:]]
        assert all(torch.equal(x, y) for x, y in zip(got[i], want))
        work[i][0].close()


def test_the_current_device_stays(gpu_ctx):
    before = torch.cuda.current_device()
    rows.lookup_rows(gpu_ctx, torch.zeros((3, 8), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert torch.cuda.current_device() == before


# ---- refusals of the C entry points ------------------------------------------------------------------------------

def test_c_entry_points_refuse_what_they_do_not_take(gpu_ctx):
    """Arguments that the host can see to be wrong are errors with a message; nothing is launched."""
    ctx, lib, h = gpu_ctx, gpu_ctx.lib, gpu_ctx.handle
    x = torch.zeros((64, 64), device="cuda")
    y = torch.zeros((64, 64), device="cuda")
    i = torch.zeros(64 * 4, dtype=torch.int32, device="cuda")
    j, m, s = torch.zeros_like(i), torch.zeros_like(i), torch.zeros_like(i)
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    X, Y, I, J, M, S, W = (t.data_ptr() for t in (x, y, i, j, m, s, ws))
    BAD, NO = -1, -2

    def look(code, table=X, kind=0, n=64, dim=64, ts=64, ids=I, count=8, out=Y, os=64):
        assert lib.glide_lookup_rows(h, table, kind, n, dim, ts, ids, count, 1.0, out, os, None) == code
        assert code == 0 or len(lib.glide_last_error(h)) > 10

    look(0)
    look(NO, kind=4)
    look(NO, kind=-1)
    look(BAD, n=0)
    look(BAD, dim=0)
    look(NO, dim=1 << 21)
    look(BAD, n=1 << 32)
    look(NO, count=1 << 31)
    look(BAD, table=None)
    look(BAD, ids=None)
    look(BAD, out=None)
    look(BAD, os=63)
    look(BAD, out=X)
    look(BAD, out=X + 64 * 64 * 4 - 4)
    look(BAD, out=I)
    look(BAD, table=X + 2)
    look(BAD, ids=I + 2)
    look(BAD, ts=1 << 62)

    def grad(code, g=X, kind=0, gs=64, ids=I, count=8, out=Y, ok=0, n=64, dim=64, os=64, w=W, wb=1 << 20):
        assert lib.glide_lookup_rows_grad(h, g, kind, gs, ids, count, 1.0, out, ok, n, dim, os, 0, w, wb, None) == code

    grad(0)
    grad(NO, kind=1)
    grad(NO, kind=0, ok=2)
    grad(NO, kind=3, ok=2)
    grad(BAD, n=0)
    grad(BAD, g=None)
    grad(BAD, out=None)
    grad(BAD, count=2000, gs=1, wb=100)        # few ids need no workspace, these do
    grad(BAD, count=2000, gs=1, w=None)
    grad(BAD, w=W + 16)
    grad(BAD, out=X)
    grad(BAD, count=2000, gs=0, w=Y)
    grad(BAD, os=10)
    grad(BAD, n=1 << 32)

    def send(code, r=X, kind=0, count=16, dim=64, rs=64, c=I, choices=4, parts=8, out=Y, os=64, p=J, mp=M, st=S, w=W, wb=1 << 20):
        assert lib.glide_dispatch_rows(h, r, kind, count, dim, rs, c, choices, parts, out, os, p, mp, st, w, wb, None) == code

    send(0)
    send(NO, kind=1)
    send(BAD, dim=0)
    send(BAD, choices=0)
    send(BAD, parts=0)
    send(NO, choices=129)
    send(NO, parts=4097)
    send(NO, count=1 << 30)
    send(BAD, out=None)
    send(BAD, st=None)
    send(BAD, p=I)
    send(BAD, mp=J)
    send(BAD, out=X)
    send(BAD, count=10_000, wb=10)        # few pairs need no workspace, these do
    send(BAD, os=8)
    send(BAD, w=W + 8)

    def back(code, t=X, kind=0, n=64, dim=64, ts=64, p=I, count=16, choices=4, w=None, out=Y, os=64):
        assert lib.glide_combine_rows(h, t, kind, n, dim, ts, p, count, choices, w, out, os, None) == code

    back(0)
    back(NO, kind=1)
    back(BAD, dim=0)
    back(BAD, choices=0)
    back(NO, choices=200)
    back(BAD, out=X)
    back(BAD, out=I)
    back(BAD, t=None)
    back(BAD, os=5)
    back(BAD, w=I + 1)
    z = torch.zeros((64, 64), device="cuda")

    def both(code, g=X, kind=0, count=16, dim=64, gs=64, t=Y, n=64, ts=64, p=J, choices=4, w=None, gt=z.data_ptr(), gts=64, gw=S):
        assert lib.glide_combine_rows_grad(h, g, kind, count, dim, gs, t, n, ts, p, choices, w, gt, gts, gw, None) == code

    i.fill_(-1)
    j.copy_(torch.arange(256, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    both(0)
    both(NO, kind=1)
    both(BAD, gt=X)
    both(BAD, gt=Y)
    both(BAD, gw=J)
    both(BAD, g=None)
    both(BAD, gts=3)
    both(NO, choices=129)
    torch.cuda.synchronize()
    assert isinstance(C.c_int(0).value, int)


def test_refused_calls_raise_with_the_library_s_message(gpu_ctx):
    with pytest.raises(api.UnsupportedError, match="4096 partitions"):
        rows.dispatch_rows(gpu_ctx, torch.zeros((4, 8), device="cuda"), torch.zeros((4, 1), dtype=torch.int32, device="cuda"), 5000)
    with pytest.raises(api.GlideError, match="overlaps"):
        t = torch.zeros((8, 8), device="cuda")
        rows.lookup_rows(gpu_ctx, t, torch.zeros(4, dtype=torch.int32, device="cuda"), out=t[2:6])
