"""Workspaces of the 4-bit attention: a call takes what its kernels use."""

from __future__ import annotations

import pytest
import torch

from minisgl_amd.kernel import lib
from test_mx4_gpu import DEV, NAN, Paged, check, cumulative, i32, pool_of

pytestmark = pytest.mark.gpu
MIB = 1 << 20


def test_streamed_requests_of_many_rows_have_no_values_laid_out():
    """A chunk of 640 rows among others that are streamed from the codes in pieces: with a workspace for the partial results alone,
    or with none, and then no more memory than that."""
    extends = [80] + [3] * 19
    c = Paged(extends, [3500] + [100 * i for i in range(19)], 64, 8, 64, 16, 41)
    wide = torch.full((20, 256), -7, dtype=torch.int32)
    wide[:, : c.pt.shape[1]] = c.pt
    c.pt, ref = wide, c.ref()
    split = lib.gqa_workspace_bytes(80, 64, 8, 64)
    whole = lib.gqa_mx4_workspace_bytes(80, 64, 8, 64, 20, 4096, 20 * 4096)
    assert whole > split + 100 * MIB
    check(*c.run(workspace=torch.empty(split, dtype=torch.uint8, device=DEV)), ref)
    q, k, v, pt, cu, lens = c.q.to(DEV), pool_of(*c.k, True), pool_of(*c.v, True), c.pt.to(DEV), i32(cumulative(extends)), i32(c.lens)
    out, lse = torch.full_like(q, NAN), torch.full(q.shape[:2], NAN, device=DEV)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    lib.gqa_chunk_mx4(q, k, v, pt, cu, lens, 80, c.scale, out, lse)  # no total_keys: the table's 80k
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= split + 2 * MIB
    check(out, lse, ref)
    with pytest.raises(lib.MLAKernelError, match="workspace"):
        c.run(workspace=torch.empty(split - 1, dtype=torch.uint8, device=DEV))


def test_values_laid_out_need_the_whole_workspace():
    c = Paged([700, 1, 333, 64], [100, 900, 5, 700], 16, 4, 64, 16, 42)
    split = lib.gqa_workspace_bytes(700, 16, 4, 64)
    whole = lib.gqa_mx4_workspace_bytes(700, 16, 4, 64, 4, c.pt.shape[1] * 16, sum(c.lens))
    with pytest.raises(lib.MLAKernelError, match=f"hold {whole} bytes"):
        c.run(workspace=torch.empty(split, dtype=torch.uint8, device=DEV))
    check(*c.run(workspace=torch.empty(whole, dtype=torch.uint8, device=DEV)), c.ref())
    check(*c.run(), c.ref())
