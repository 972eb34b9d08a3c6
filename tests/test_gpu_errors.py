"""A call that a CUDA error ends reports it and leaves nothing behind: the calls after it work. The errors are the host's: memory
that cannot be had, a stream whose capture has been broken off."""
import ctypes as C

import pytest
import torch

from glide_b200 import api

pytestmark = pytest.mark.gpu


def _works(ctx):
    base = torch.arange(300, dtype=torch.float32, device="cuda")[:, None].repeat(1, 4).contiguous()
    ids, _ = api.bruteforce_knn(ctx, base, base[:5].contiguous(), 1)
    assert ids[:, 0].tolist() == [0, 1, 2, 3, 4]
    assert torch.ones(3, device="cuda").sum().item() == 3


def test_a_call_without_enough_memory(gpu_ctx):
    p = C.c_void_p()
    assert gpu_ctx.lib.glide_malloc(gpu_ctx.handle, 1 << 60, C.byref(p)) == -4
    _works(gpu_ctx)


def test_a_launch_into_a_stream_whose_capture_was_broken_off(gpu_ctx):
    cudart = C.CDLL("libcudart.so.12")       # the one that torch and the library have loaded
    table, ids, out = torch.zeros((4, 8), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros((2, 8), device="cuda")
    torch.cuda.synchronize()
    stream, graph = C.c_void_p(), C.c_void_p()
    assert cudart.cudaStreamCreateWithFlags(C.byref(stream), 1) == 0
    assert cudart.cudaStreamBeginCapture(stream, 2) == 0
    assert cudart.cudaStreamSynchronize(stream) != 0           # not allowed in a capture, which ends with it
    cudart.cudaGetLastError()
    rc = gpu_ctx.lib.glide_lookup_rows(gpu_ctx.handle, table.data_ptr(), 0, 4, 8, 8, ids.data_ptr(), 2, 1.0, out.data_ptr(), 8, stream)
    left = cudart.cudaPeekAtLastError()
    assert cudart.cudaStreamEndCapture(stream, C.byref(graph)) != 0
    cudart.cudaGetLastError()
    assert cudart.cudaStreamDestroy(stream) == 0
    assert rc == -3 and len(gpu_ctx.lib.glide_last_error(gpu_ctx.handle)) > 10 and left == 0
    _works(gpu_ctx)
