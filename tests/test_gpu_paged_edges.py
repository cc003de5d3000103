"""The paged KV cache on the GPU at the edges of what its calls allow: repeated and concurrent calls, scales of
either sign and of every size, windows without end, unmapped pages, padded batches, singleton strides."""

import math

import numpy as np
import pytest
import torch

import paged_reference as R
from test_gpu_paged import BF16, BLOCKS, CHUNKS, DEV, E4M3, F32, INT8, RAGGED, TYPES, Setup, paged  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [E4M3, INT8])
@pytest.mark.parametrize("rows", [F32, BF16])
def test_few_sequences_repeat_themselves(paged, cache, rows):
    """Queries whose heads differ by many powers of two, a few sequences of one tile: every warp's share of a
    column's largest magnitude counts, whichever warp is first. The same bits every time, and the right ones."""
    st = Setup(paged, cache, [(2100, 1), (33, 1), (700, 2)], kv_heads=4, seed=31)
    st.fill()
    size = 2.0 ** torch.randint(-18, 3, (st.rows, 8, 8, 1), generator=st.gen)
    q = (torch.randn(st.rows, 8, 8, 16, generator=st.gen) * size).view(st.rows, 8, 128).to(rows).to(DEV)
    first = st.check_attention(8, rows, q=q)
    for _ in range(200):
        assert torch.equal(st.cache.attention(st.batch, q, 1.0 / math.sqrt(128)), first)
    st.cache.check()
