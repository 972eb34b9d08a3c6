"""Host threads with a context each, whose calls take the same kernels with different amounts of shared memory."""
import threading

import pytest
import torch

from glide_b200 import api

pytestmark = pytest.mark.gpu


def _at_once(calls, times):
    """Each call, `times` times in a thread of its own; the codes other than 0 that it returned."""
    codes, gate = [set() for _ in calls], threading.Barrier(len(calls))

    def run(i):
        gate.wait()
        for _ in range(times):
            codes[i].add(calls[i]())

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    return [c - {0} for c in codes]


def test_two_threads_dispatch_to_different_numbers_of_partitions(gpu_ctx):
    """A counter for each partition and warp: 64 KB for 4,096 partitions, 41 KB for 2,600."""
    lib, held, calls = gpu_ctx.lib, [], []
    for partitions in (4096, 2600):
        ctx, stream = api.Context(0), torch.cuda.Stream()
        pairs, dim = 2100, 4       # more than one launch sorts
        data = torch.arange(pairs * dim, dtype=torch.float32, device="cuda").view(pairs, dim)
        choice = (torch.arange(pairs, dtype=torch.int32, device="cuda") * 7 % partitions).contiguous()
        out, ids = torch.empty_like(data), [torch.empty(n, dtype=torch.int32, device="cuda") for n in (pairs, pairs, partitions + 1)]
        need = lib.glide_dispatch_rows_workspace(pairs, 1, partitions)
        scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
        held.append((ctx, stream, data, choice, out, ids, scratch))
        args = (ctx.handle, data.data_ptr(), 0, pairs, dim, dim, choice.data_ptr(), 1, partitions, out.data_ptr(), dim, *(t.data_ptr() for t in ids),
                scratch.data_ptr(), need, stream.cuda_stream)
        calls.append(lambda args=args: lib.glide_dispatch_rows(*args))
    torch.cuda.synchronize()
    assert _at_once(calls, 4000) == [set(), set()]
    for ctx, _, data, choice, out, _, _ in held:
        assert torch.equal(out, data[torch.sort(choice, stable=True).indices])
        ctx.close()


def test_four_threads_ask_for_different_numbers_of_neighbours(gpu_ctx):
    lib, held, calls = gpu_ctx.lib, [], []
    base = torch.randn((200, 24), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    queries = base[:2].contiguous()
    for k in (128, 1, 127, 2):
        ctx = api.Context(0)
        ids, dists = torch.empty((2, k), dtype=torch.int32, device="cuda"), torch.empty((2, k), device="cuda")
        held.append((ctx, ids, dists))
        args = (ctx.handle, base.data_ptr(), 200, queries.data_ptr(), 2, 24, k, 0, ids.data_ptr(), dists.data_ptr())
        calls.append(lambda args=args: lib.glide_bruteforce_knn(*args))
    torch.cuda.synchronize()
    assert _at_once(calls, 4000) == [set()] * 4
    for ctx, ids, _ in held:
        assert torch.equal(ids[:, 0], torch.arange(2, dtype=torch.int32, device="cuda"))
        ctx.close()
