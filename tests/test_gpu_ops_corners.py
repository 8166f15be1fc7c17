"""The operators on a caller's own device memory where their work is cut in unusual ways: batches with few active sequences among many,
rows whose pages are all bad, rows that are NaN, softmax weights far below the largest, waits that run out.  The bounds are
test_gpu_ops.py's (a rounding to type t is off by at most eps(t) / 2 relative); what a test adds is derived beside it."""
import math
import time

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


@pytest.mark.parametrize("new", [1, 40])
def test_thousands_of_sequences_without_tokens_between_two(new):
    """The first and the last of 65535 sequences have tokens, and a CTA's interval holds the end of the one and the start of the other."""
    n_seq = 65535
    kv, counts = [0] * n_seq, [0] * n_seq
    kv[0], counts[0], kv[-1], counts[-1] = 70 + new, new, 20000, new
    c = ref.make_cache([kv[0], kv[-1]], 1, 64, torch.bfloat16, DEV)
    table = torch.full((n_seq, c["table"].shape[1]), -1, dtype=torch.int32, device=DEV)
    table[0], table[-1] = c["table"][0], c["table"][1]
    small = dict(c)
    c.update(table=table, kv_len=torch.tensor(kv, dtype=torch.int32, device=DEV), kv=kv)
    ws, q = ops.space(), ops.normal(2 * new, 2, 64, dtype=torch.bfloat16)
    want, want_lse = torch.zeros_like(q), torch.zeros(2 * new, 2, device=DEV)
    capi.paged_attention(ops.view(small), ref.cu_of([new, new], DEV), q, want, ops.space(), lse=want_lse)
    got, lse = attend(c, counts, 2, ws, q=q)[1:]
    assert int(c["status"]) == 0
    # The same tokens as a batch of two; cut otherwise, so roundings differ as check_attention allows each.
    assert (got.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
    assert (lse - want_lse).abs().max() <= 2.0 ** -18


# ---- weights: rows that see bad pages only, rows that are NaN --------------------------------------------------------


def weights_of(c, new, q, skip=()):
    """(the weight each slot received in 64 bits, slots that hold one): slots of pages outside the pool count as masked; rows whose
    log-sum is -inf, and (token, head) of `skip`, give nothing."""
    D, G = c["dim"], q.shape[1] // c["kv_heads"]
    want, held = torch.zeros(c["weight"].shape, dtype=torch.float64, device=DEV), torch.zeros(c["weight"].shape, dtype=torch.bool, device=DEV)
    at = 0
    for s, (n, m) in enumerate(zip(c["kv"], new)):
        page, place = ref.rows_of(c, s, n)
        good = (page >= 0) & (page < c["pool"].shape[0])
        sees = (torch.arange(n, device=DEV)[None] <= (n - m + torch.arange(m, device=DEV))[:, None]) & good[None]
        page, place, sees = page[good], place[good], sees[:, good]
        for h in range(q.shape[1] if m else 0):
            a = (q[at:at + m, h].double() @ c["k"][page, h // G, place].double().T / math.sqrt(D)).masked_fill(~sees, -math.inf)
            p = torch.softmax(a, 1).masked_fill(~sees, 0.0)  # a row without slots: NaN, all masked
            for t, head in skip:
                if head == h and at <= t < at + m:
                    p[t - at] = 0.0
            want[page, h // G, place] += p.sum(0)
        if m:
            held[page, :, place] = True
        at += m
    return want, held


def check_weights(got, want, held, old, decay, terms):
    """Each term's relative error is below 2^-17 (scores of normal values: 2 e + the log-sum's error + 2^-20 of test_gpu_ops.py, whose e is
    (D + 4) 2^-24 S with S below 40 here), and `terms` of them are added in 32 bits."""
    want = want + decay * old.double()
    assert torch.equal(got[~held], old[~held])
    off = ((got.double() - want).abs() - (2.0 ** -10 + terms * 2.0 ** -24) * want.abs() - 1e-37)[held]
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("max_tokens", [1, 0])  # the kernel for few rows, and the one for many
@pytest.mark.parametrize("new,bad", [([130], [0]), ([130, 70], [0]), ([300, 40], [0, 2]), ([200], [1]), ([64], [0])])
@pytest.mark.parametrize("before", [0, 100])
def test_weights_of_rows_that_see_bad_pages_only(new, bad, before, max_tokens):
    """A bad page's slots count as masked; rows that see no others add nothing anywhere, and nothing is written there."""
    c = ref.make_cache([n + before for n in new], 2, 64, torch.bfloat16, DEV)
    for p in bad:
        c["table"][0, p] = -1 if p else 1 << 30
    q = ops.normal(sum(new), 4, 64, dtype=torch.bfloat16, scale=1.5)
    out, lse, cu = torch.zeros_like(q), torch.zeros(sum(new), 4, device=DEV), ref.cu_of(new, DEV)
    want, held = weights_of(c, new, q)
    for decay in (0.0, 0.5):
        old = torch.rand(c["weight"].shape, device=DEV)
        c["weight"].copy_(old)
        cache = ops.view(c, weight=c["weight"])
        capi.paged_attention(cache, cu, q, out, ops.space(), lse=lse, max_tokens=max_tokens)
        capi.attention_weights(cache, cu, q, lse, decay=decay, max_tokens=max_tokens)
        torch.cuda.synchronize()
        assert int(c["status"]) == capi.BAD_PAGE
        check_weights(c["weight"], want, held, old, decay, 2 * max(new))


@pytest.mark.parametrize("max_tokens", [1, 0])
def test_weights_of_a_nan_row_stay_with_the_slots_it_sees(max_tokens):
    """A NaN query makes the weights of the slots that its row sees NaN, under its KV head; the new tokens behind it are not among them."""
    new, row = [150, 90], 20
    c = ref.make_cache([150, 190], 2, 64, torch.float16, DEV)
    q = ops.normal(sum(new), 4, 64, dtype=torch.float16, scale=1.5)
    clean, cu = q.clone(), ref.cu_of(new, DEV)
    q[row, 1, 5] = math.nan
    want, held = weights_of(c, new, clean, skip=[(row, 1)])
    page, place = ref.rows_of(c, 0, row + 1)
    out, lse, old = torch.zeros_like(q), torch.zeros(sum(new), 4, device=DEV), torch.rand(c["weight"].shape, device=DEV)
    c["weight"].copy_(old)
    cache = ops.view(c, weight=c["weight"])
    capi.paged_attention(cache, cu, q, out, ops.space(), lse=lse, max_tokens=max_tokens)
    capi.attention_weights(cache, cu, q, lse, decay=0.0, max_tokens=max_tokens)
    torch.cuda.synchronize()
    got = c["weight"].clone()
    assert bool(got[page, 0, place].isnan().all())
    got[page, 0, place] = want[page, 0, place].float()
    check_weights(got, want, held, old, 0.0, 2 * max(new))


# ---- waits that run out ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("call", ["attention", "weights"])
@pytest.mark.parametrize("new,max_tokens,n_seq", [(2, 2, 2), (150, 0, 2), (1, 1, 40)])
def test_a_wait_that_runs_out_is_reported(call, new, max_tokens, n_seq):
    """A call whose kernel hands out no work ends after two seconds with its bit set; the next one, on a zeroed workspace, is right."""
    c = ref.make_cache([300] * n_seq, 2, 64, torch.bfloat16, DEV)
    q, cu, counts = ops.normal(new * n_seq, 4, 64, dtype=torch.bfloat16), ref.cu_of([new] * n_seq, DEV), [new] * n_seq
    out, lse, ws = torch.zeros_like(q), torch.zeros(new * n_seq, 4, device=DEV), ops.space()
    cache = ops.view(c, weight=c["weight"])
    if call == "weights":
        capi.paged_attention(cache, cu, q, out, ws, lse=lse, max_tokens=max_tokens)
    torch.cuda.synchronize()
    capi.lib().mtb_debug_stall_attention(1)
    start = time.time()
    if call == "attention":
        capi.paged_attention(cache, cu, q, out, ws, lse=lse, max_tokens=max_tokens)
    else:
        capi.attention_weights(cache, cu, q, lse, decay=0.0, max_tokens=max_tokens)
    torch.cuda.synchronize()
    assert 1.0 < time.time() - start < 20.0
    assert int(c["status"]) == capi.BAD_WAIT
    c["status"].zero_()
    ws.zero_()
    attend(c, counts, 4, ws, q=q, max_tokens=max_tokens)
    assert int(c["status"]) == 0


# ---- logits: a row in several CTAs -------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129])
def test_the_choice_is_found_in_every_share_of_a_row(rows):
    """Up to 128 rows several CTAs have a row, in runs of 1024 ids: the largest value in each run in turn, equal ones in two runs, none."""
    vocab = 20 * 1024 + 7
    runs = -(-vocab // 1024)
    x = ops.normal(rows, vocab, seed=rows)
    at = torch.arange(rows, device=DEV)
    choice = torch.empty(rows, dtype=torch.int32, device=DEV)
    for run in range(runs):
        low = torch.clamp(run * 1024 + (at * 37) % 1024, max=vocab - 1)
        high = torch.clamp(low + 1024, max=vocab - 1)
        y = x.clone()
        y[at, low] = 50.0
        y[at, high] = 50.0
        y[rows // 2] = -math.inf
        capi.logits_process(y, None, choice)
        want = torch.minimum(low, high).to(torch.int32)
        want[rows // 2] = -1
        assert torch.equal(choice, want)


# ---- probabilities far below the largest -----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,kv", [(1, 4096), (8, 4096), (40, 4096), (1, 300), (150, 4096)])
def test_a_first_slot_that_takes_nearly_all(dtype, new, kv):
    """Slot 0 outweighs any other by e^14.5 and its V is 0, so that the result is made of probabilities of 2^-21: within
    check_attention's bound, which lets a probability be off by half a step of 16 bits relative to itself."""
    c = ref.make_cache([kv], 1, 64, dtype, DEV)
    page, place = ref.rows_of(c, 0, kv)
    c["k"][page, 0, place] = 0.0
    c["k"][page[0], 0, 0, 0] = 14.5  # times q's 8 and the scale of 1 / 8: the score
    c["v"][page[0], 0, 0] = 0.0
    c["v"][page[1:], 0, place[1:]] += 2.0
    q = torch.zeros(new, 2, 64, dtype=dtype, device=DEV)
    q[:, :, 0] = 8.0
    attend(c, [new], 2, ops.space(), q=q)


@pytest.mark.parametrize("kv", [9001, 20011, 27000])
def test_log_sums_do_not_depend_on_the_cut(kv):
    """Scores of 0 once and of -20 log2 units else: log(1 + (kv - 1) 2^-20), where the logarithm of a split tile has to be as exact as
    that of a whole one.  The terms are off by 2^-19 relative (the scale's product with log2 e, times 20, and the exponential); their
    sums are multiples of 2^-20 below 2 but for that, so the f32 additions lose nothing; the logarithm and its product: 2^-22 relative."""
    c = ref.make_cache([kv], 1, 64, torch.bfloat16, DEV)
    page, place = ref.rows_of(c, 0, kv)
    c["k"][page, 0, place] = 0.0
    c["k"][page[1:], 0, place[1:], 0] = -20.0
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=DEV)
    q[:, :, 0] = 1.0
    lse = torch.zeros(1, 1, device=DEV)
    capi.paged_attention(ops.view(c), ref.cu_of([1], DEV), q, torch.zeros_like(q), ops.space(), lse=lse, scale=math.log(2.0))
    tail = (kv - 1) * 2.0 ** -20
    assert abs(float(lse) - math.log1p(tail)) <= 2.0 ** -19 * tail + 2.0 ** -22 * math.log1p(tail)


# ---- what the append checks -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("cu,n", [([0, 4, 2, 6, 8], 8), ([0, 3, 3, 9, 2, 6], 6), ([0, 2, 4, 6, 99], 6), ([-1, 2, 4], 4), ([0, 6] + [5] * 300, 6)])
def test_append_and_attention_report_the_same_bounds_of_tokens(cu, n):
    """Bounds that do not ascend inside [0, n_tokens] set their bit in the append as in the attention, also where no token is
    found in the sequence that has them."""
    n_seq = len(cu) - 1
    bits = []
    bounds = torch.tensor(cu, dtype=torch.int32, device=DEV)
    q = ops.normal(n, 2, 64, dtype=torch.bfloat16)
    inv = torch.from_numpy(capi.rope_frequencies(64, 1e4)[0]).to(DEV)
    for call in ("append", "attention"):
        c = ref.make_cache([70] * n_seq, 2, 64, torch.bfloat16, DEV)
        if call == "append":
            capi.rope_append(ops.view(c), bounds, torch.zeros(n, dtype=torch.int32, device=DEV), q, q, q, inv, torch.empty_like(q))
        else:
            capi.paged_attention(ops.view(c), bounds, q, torch.empty_like(q), ops.space())
        bits.append(int(c["status"]))
    assert bits == [capi.BAD_TOKENS, capi.BAD_TOKENS]


# ---- what P's rounding leaves ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,kv_heads,group,new,kv", [(128, 8, 2, [1, 1, 1], [40, 300, 129]), (64, 2, 4, [4, 1, 2], [200, 64, 300]),
                                                       (128, 1, 16, [1], [300]), (64, 1, 1, [16, 3], [150, 33]), (128, 2, 2, [8], [300])])
def test_steps_hold_probabilities_to_more_than_16_bits(dtype, dim, kv_heads, group, new, kv):
    """At most 16 rows a KV head: P goes into the product with V with what its rounding left, so it is off by h^2, not by h.
    The scores are whole numbers times 1/8, exact: e is 2^-22 of the largest (the scale's product with log2 e, and a subtraction);
    the rest as in test_gpu_ops.py."""
    c = ref.make_cache(kv, kv_heads, dim, dtype, DEV)
    g = torch.Generator().manual_seed(dim + group)
    whole = lambda shape: torch.randint(-2, 3, shape, generator=g).to(dtype).to(DEV)
    c["k"].copy_(whole(c["k"].shape))
    q = whole((sum(new), kv_heads * group, dim))
    out = torch.zeros_like(q)
    capi.paged_attention(ops.view(c), ref.cu_of(new, DEV), q, out, ops.space(), scale=0.125, max_tokens=max(new))
    w = ref.attention(c, new, q, 0.125)
    h, e = ops.half(dtype), 2.0 ** -22 * w["size"][..., None]
    tol = h * w["out"].abs() + (h * h + 2 * e + 2.0 ** -19 + max(kv) * 2.0 ** -24) * w["spread"]
    off = (out.double() - w["out"]).abs()
    assert bool((off <= tol * 1.001 + 2.0 ** -25).all()), float((off / tol).max())  # 2^-25: half a step of fp16's smallest values


# ---- eviction by one CTA a list ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kv,heads,keep,sinks,recent,table_len,shift", [
    ([0, 1, 63, 64, 65, 100, 514, 1300], 2, 100, 4, 16, None, 1),   # books that are not 16-byte aligned
    ([700, 2000], 3, 64, 3, 7, None, 3),
    ([1300, 65], 2, 0, 0, 0, None, 2),
    ([9000, 300, 64], 2, 200, 4, 64, 1100, 0),                      # a table of more than 65536 slots
    ([41000, 40960], 1, 8192, 4, 512, 1100, 0),                     # more keys than shared memory holds, and as many
    ([70001], 1, 30000, 4, 100, None, 0),
])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_by_one_cta_a_list(kv, heads, keep, sinks, recent, table_len, shift, ties):
    c = ref.make_cache(kv, heads, 64, torch.bfloat16, DEV, table_len=table_len)
    for name in ("position", "weight"):
        room = torch.zeros(c[name].numel() + 4, dtype=c[name].dtype, device=DEV)
        c[name] = room[shift:shift + c[name].numel()].view(c[name].shape)
    ops.fill_books(c, seed=len(kv), ties=ties)
    c["weight"][:, :, 5::9] = math.nan
    ops.run_evict(c, keep, sinks, recent, alias=ties)
