"""The operators on a caller's own device memory where their work is cut in unusual ways: batches with few active sequences among many,
rows whose pages are all bad, rows that are NaN, softmax weights far below the largest, waits that run out.  The bounds are
test_gpu_ops.py's (a rounding to type t is off by at most eps(t) / 2 relative); what a test adds is derived beside it."""
import math

import pytest

import ops_reference as ref
import test_gpu_ops as ops
from mtb import capi

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda:0"
COUNTERS = 8192  # bytes of the attention workspace that every call has to leave zero


def attend(c, new, heads, ws, seed=1, q=None, decay=0.0, max_tokens=0, weights=True):
    """Attention and, with `weights`, its weights; against the 64-bit definition."""
    n = sum(new)
    if q is None:
        q = ops.normal(n, heads, c["dim"], seed=seed, dtype=c["pool"].dtype, scale=1.5)
    out, lse = torch.full_like(q, 7.0), torch.full((n, heads), 9.0, device=DEV)
    cu = ref.cu_of(new, DEV)
    old = torch.rand(c["weight"].shape, device=DEV)
    c["weight"].copy_(old)
    cache = ops.view(c, weight=c["weight"])
    capi.paged_attention(cache, cu, q, out, ws, lse=lse, max_tokens=max_tokens)
    if weights:
        capi.attention_weights(cache, cu, q, lse, decay=decay, max_tokens=max_tokens)
    torch.cuda.synchronize()
    ops.check_attention(c, new, q, out, lse, None, c["weight"] if weights else None, decay, old)
    assert not ws[:COUNTERS].any()
    return q, out, lse


# ---- few active sequences among more than 32 ------------------------------------------------------------------------


@pytest.mark.parametrize("n_seq,kv_heads,group,active", [
    (40, 8, 2, {7: (500, 1)}),                         # a step of one sequence: 8 tiles, fewer units than CTAs
    (33, 1, 4, {0: (900, 1), 32: (65, 1)}),
    (64, 2, 2, {3: (130, 8), 40: (700, 2), 63: (64, 1)}),
    (48, 1, 1, {11: (321, 16)}),
    (40, 1, 2, {5: (300, 40)}),                        # chunks
    (64, 2, 4, {1: (900, 70), 62: (257, 33)}),
    (33, 1, 4, {s: (200, 40) for s in range(33)}),     # 33 short chunks, a tile of two blocks each
    (400, 1, 1, {399: (1000, 3)}),
])
def test_sparse_batches_are_joined(n_seq, kv_heads, group, active):
    """More sequences than a warp has lanes, hardly any with tokens: every split tile is joined, and the workspace serves the next call."""
    kv, new = [(37 * s) % 90 for s in range(n_seq)], [0] * n_seq
    for s, (length, n) in active.items():
        kv[s], new[s] = length, n
    ws = ops.space()
    attend(ref.make_cache(kv, kv_heads, 64, torch.bfloat16, DEV), new, kv_heads * group, ws)
    attend(ref.make_cache([5000, 300, 2500], 2, 128, torch.bfloat16, DEV), [1, 1, 1], 4, ws)
    attend(ref.make_cache([3000, 700], 2, 128, torch.bfloat16, DEV), [200, 100], 4, ws)
