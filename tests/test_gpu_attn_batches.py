"""Attention over batches of very many sequences, most of them empty or short:
the kernels' ways of finding their work."""
import random

import pytest
import torch

from rhizome_b200 import ops
from tests.test_gpu_attn import BF, F32, cu_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1 << 20, 1 << 22])
def test_prompts_between_millions_of_empty_ones(n):
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = {0: 300, 5: 1, n // 2: 700, n - 1: 64}
    counts = torch.zeros(n, dtype=torch.int64)
    for i, m in lens.items():
        counts[i] = m
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32).cuda()
    total = int(counts.sum())
    q = torch.randn(total, 4, 128, generator=g, device="cuda").to(BF)
    k, v = (torch.randn(total, 2, 128, generator=g, device="cuda").to(BF) for _ in range(2))
    o = ops.attn_varlen_fwd(q, k, v, cu)
    assert not ops.device_status()
    assert torch.equal(o, ops.attn_varlen_fwd(q, k, v, cu_of(list(lens.values()))[1]))
