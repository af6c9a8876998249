"""The paged cache's budget at its edges, on the GPU: caches without pages, batches
and rows of the largest kernels, wide tables, tensors written in place.  Bounds as
in test_gpu_kv_budget.py."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_kv import dev  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts", [[40, 3], [1, 1]])
def test_weights_of_a_cache_without_pages(engine, counts, dtype):
    # no key gets anything: what was there decays, the step's own keys start from zero
    c = engine.PagedKVCache.empty(0, 2, 16, 64, dtype=dtype)
    i = dict(dtype=torch.int32, device="cuda")
    tokens, past = sum(counts), [7, 20]
    positions = torch.tensor([p + t for p, n in zip(past, counts) for t in range(n)], **i)
    starts = torch.tensor([0, counts[0], tokens], **i)
    q = torch.randn(tokens, 6, 64, device="cuda").to(dtype)
    lse = torch.full((tokens, 6), -math.inf, device="cuda")
    for table in (torch.full((2, 5), -1, **i), torch.zeros(2, 5, **i)):
        mass = torch.rand(2, 2, 80, device="cuda")
        want = mass.clone()
        for r in range(2):
            want[r, :, :past[r]] *= 0.5
            want[r, :, past[r]:past[r] + counts[r]] = 0
        c.weigh(q, table, starts, positions, lse, mass, decay=0.5)
        assert torch.equal(mass, want)
