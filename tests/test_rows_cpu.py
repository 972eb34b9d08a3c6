"""Refusals of `glide_b200.rows` that need no GPU: every call that its documentation does not allow is an error before
the library is reached. The context is a stand-in on the CPU whose library fails the test when it is called."""
import ctypes as C

import pytest
import torch

from glide_b200 import _lib, rows


class _Lib:
    def __getattr__(self, name):
        if name.endswith("_workspace"):
            return getattr(_lib.load(), name)
        def reached(*args):
            raise AssertionError(f"{name} was reached")
        return reached


class _Context:
    torch_device = torch.device("cpu")
    lib = _Lib()
    handle = None

    def check(self, rc):
        raise AssertionError("the library was reached")


ctx = _Context()
F = torch.float32


def _ids(*shape):
    return torch.zeros(shape, dtype=torch.int32)


BAD = {
    "lookup: table of integers": lambda: rows.lookup_rows(ctx, torch.zeros((4, 8), dtype=torch.int32), _ids(2)),
    "lookup: table of doubles": lambda: rows.lookup_rows(ctx, torch.zeros((4, 8), dtype=torch.float64), _ids(2)),
    "lookup: table of one dimension": lambda: rows.lookup_rows(ctx, torch.zeros(8), _ids(2)),
    "lookup: table with rows that are not contiguous": lambda: rows.lookup_rows(ctx, torch.zeros((8, 4)).t(), _ids(2)),
    "lookup: ids of 64 bits": lambda: rows.lookup_rows(ctx, torch.zeros((4, 8)), torch.zeros(2, dtype=torch.int64)),
    "lookup: ids that are not contiguous": lambda: rows.lookup_rows(ctx, torch.zeros((4, 8)), _ids(4, 2)[:, 0]),
    "lookup: result of another shape": lambda: rows.lookup_rows(ctx, torch.zeros((4, 8)), _ids(2), out=torch.zeros((3, 8))),
    "lookup: result of another type": lambda: rows.lookup_rows(ctx, torch.zeros((4, 8)), _ids(2), out=torch.zeros((2, 8), dtype=torch.float16)),
    "lookup: result whose rows are strided": lambda: rows.lookup_rows(ctx, torch.zeros((4, 8)), _ids(2), out=torch.zeros((2, 16))[:, ::2]),
    "lookup: result that is no matrix": lambda: rows.lookup_rows(ctx, torch.zeros((4, 8)), _ids(2, 3), out=torch.zeros((3, 2, 8)).transpose(0, 1)),
    "lookup: another device": lambda: rows.lookup_rows(ctx, torch.zeros((4, 8), device="meta"), _ids(2)),
    "lookup: an array": lambda: rows.lookup_rows(ctx, torch.zeros((4, 8)).numpy(), _ids(2)),
    "grad: shape": lambda: rows.lookup_rows_grad(ctx, torch.zeros((3, 8)), _ids(2), 4),
    "grad: bytes": lambda: rows.lookup_rows_grad(ctx, torch.zeros((2, 8), dtype=torch.uint8), _ids(2), 4),
    "grad: rows that do not lie one stride apart": lambda: rows.lookup_rows_grad(ctx, torch.zeros((3, 2, 8)).transpose(0, 1), _ids(2, 3), 4),
    "grad: nothing to add to": lambda: rows.lookup_rows_grad(ctx, torch.zeros((2, 8)), _ids(2), 4, accumulate=True),
    "grad: result of another length": lambda: rows.lookup_rows_grad(ctx, torch.zeros((2, 8)), _ids(2), 4, out=torch.zeros((5, 8))),
    "grad: result of another type than asked for": lambda: rows.lookup_rows_grad(ctx, torch.zeros((2, 8)), _ids(2), 4, dtype=torch.float16, out=torch.zeros((4, 8))),
    "grad: result of integers": lambda: rows.lookup_rows_grad(ctx, torch.zeros((2, 8)), _ids(2), 4, out=torch.zeros((4, 8), dtype=torch.int32)),
    "dispatch: bytes": lambda: rows.dispatch_rows(ctx, torch.zeros((2, 8), dtype=torch.uint8), _ids(2, 1), 4),
    "dispatch: choices of other rows": lambda: rows.dispatch_rows(ctx, torch.zeros((2, 8)), _ids(3, 1), 4),
    "dispatch: choices of one dimension": lambda: rows.dispatch_rows(ctx, torch.zeros((2, 8)), _ids(2), 4),
    "dispatch: result of another length": lambda: rows.dispatch_rows(ctx, torch.zeros((2, 8)), _ids(2, 2), 4, out=torch.zeros((2, 8))),
    "combine: positions of 64 bits": lambda: rows.combine_rows(ctx, torch.zeros((4, 8)), _ids(2, 2).long()),
    "combine: positions of one dimension": lambda: rows.combine_rows(ctx, torch.zeros((4, 8)), _ids(4)),
    "combine: weights in half precision": lambda: rows.combine_rows(ctx, torch.zeros((4, 8)), _ids(2, 2), torch.zeros((2, 2), dtype=torch.float16)),
    "combine: weights of another shape": lambda: rows.combine_rows(ctx, torch.zeros((4, 8)), _ids(2, 2), torch.zeros((2, 1))),
    "combine grad: another type": lambda: rows.combine_rows_grad(ctx, torch.zeros((2, 8), dtype=torch.float16), torch.zeros((4, 8)), _ids(2, 2)),
    "combine grad: another shape": lambda: rows.combine_rows_grad(ctx, torch.zeros((3, 8)), torch.zeros((4, 8)), _ids(2, 2)),
}


@pytest.mark.parametrize("what", sorted(BAD))
def test_calls_that_are_not_allowed_are_refused(what):
    with pytest.raises((TypeError, ValueError)):
        BAD[what]()


def test_entry_points_refuse_a_null_context():
    lib = _lib.load()
    assert lib.glide_lookup_rows(None, None, 0, 1, 1, 1, None, 0, 1.0, None, 1, None) == -1
    assert lib.glide_lookup_rows_grad(None, None, 0, 1, None, 0, 1.0, None, 0, 1, 1, 1, 0, None, 0, None) == -1
    assert lib.glide_dispatch_rows(None, None, 0, 0, 1, 1, None, 1, 1, None, 1, None, None, None, None, 0, None) == -1
    assert lib.glide_combine_rows(None, None, 0, 0, 1, 1, None, 0, 1, None, None, 1, None) == -1
    assert lib.glide_combine_rows_grad(None, None, 0, 0, 1, 1, None, 0, 1, None, 1, None, None, 1, None, None) == -1


def test_workspaces_hold_what_the_calls_need():
    lib = _lib.load()
    # two copies of the sorted ids with their rows, and 2 bytes of rank: 18 bytes an id at least, for every size of table
    for n in (1, 2, 1000, 1 << 20, (1 << 32) - 1):
        for count in (1025, 2049, 1 << 20):
            assert lib.glide_lookup_rows_grad_workspace(n, 128, count) >= 18 * count
    assert lib.glide_lookup_rows_grad_workspace(100, 128, 0) == 0 and lib.glide_lookup_rows_grad_workspace(100, 128, 10) == 0   # few need none
    assert lib.glide_dispatch_rows_workspace(100_000, 8, 64) >= 2 * 800_000
    # what the calls refuse needs no workspace
    assert lib.glide_dispatch_rows_workspace(1000, 129, 64) == 0
    assert lib.glide_dispatch_rows_workspace(1000, 8, 4097) == 0
    assert lib.glide_dispatch_rows_workspace(1 << 31, 1, 64) == 0
    assert lib.glide_lookup_rows_grad_workspace(1 << 32, 128, 10) == 0
    assert isinstance(C.c_size_t(lib.glide_lookup_rows_grad_workspace((1 << 32) - 1, 1 << 20, 0x7fffffff)).value, int)


def test_the_workspace_of_a_gradient_holds_its_partial_sums():
    """Two copies of the sorted ids with their rows, a rank of 2 bytes for each, a pass's counts for every 2,048 of them, and two rows of
    fp32 sums for each chunk of at most 128; up to the largest call, whose need does not fit 32 bits by far."""
    need = _lib.load().glide_lookup_rows_grad_workspace
    for n in (1, 1000, 1 << 20, (1 << 32) - 1):
        for dim in (1, 100, 4096, 1 << 20):
            for count in (1025, 4097, 100_000, 0x7fffffff):
                bits = max(1, (n).bit_length())                       # ids 0 .. n - 1, and n for none
                passes = -(-bits // 11)
                least = 18 * count + -(-count // 2048) * 4 * (1 << -(-bits // passes)) + 2 * -(-count // 128) * dim * 4
                assert need(n, dim, count) >= least, (n, dim, count)
                assert need(n, dim, count) <= 16 * least + (1 << 20)


def test_the_workspace_for_rows_without_a_place_has_a_bit_for_each():
    lib = _lib.load()
    for n in (0, 1, 32, 33, 1 << 20, 0x7fffffff):
        assert n / 8 <= lib.glide_clear_rows_without_place_workspace(n) <= n / 8 + 512
    assert lib.glide_clear_rows_without_place_workspace(1 << 31) == 0
    assert lib.glide_clear_rows_without_place(None, None, 0, 1, 1, 1, None, 0, None, 0, None) == -1
