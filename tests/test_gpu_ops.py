"""The operators on a caller's own device memory against their definitions in 64 bits (tests/ops_reference.py).

Tolerances, per element: a rounding to type t is off by at most h = eps(t) / 2 relative.
  rope       h |y| for the result, and 2^-21 (|a| + |b|) factor for the angle's f32 remainder (pi 2^-24), its f32 sine and
             cosine (2 ulp) and the two f32 products.
  attention  A = sum p |v|.  h |o| for the result; h A for the probabilities' rounding to 16 bits before the product with V; a score
             of D f32 products is off by at most e = (D + 4) 2^-24 S, S the largest sum of |q k| scale of the row, which scales a
             probability and the sum by e each: 2 e A; 2^-19 A for the exponential (2 ulp), the rescaling and the f32 sums, whose
             terms are all of one sign or bounded by A: n 2^-24 A for n slots.
  lse        2 e + 2^-20 (the logarithm, absolute) + 2^-22 |lse| + n 2^-24.
  weight     each term relative 2 e + the lse's error + 2^-20, n terms added in f32: n 2^-24.
"""
import math

import pytest

import ops_reference as ref
from mtb import capi

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def half(t):
    return torch.finfo(t).eps / 2


def view(c, status=True, **more):
    return capi.PagedCache(c["k"], c["v"], c["table"], c["kv_len"], status=c["status"] if status else None, **more)


def space():
    return torch.zeros(capi.ATTENTION_WORKSPACE, dtype=torch.uint8, device=DEV)


def normal(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


# ---- rotary positions and append ------------------------------------------------------------------------------------


def run_rope(c, new, H, in_type, rotary, interleaved, factor=1.0, far=0, stretch=None, pad=0, lead=0, status=True, in_place=False):
    Hk, D, t = c["kv_heads"], c["dim"], c["pool"].dtype
    n = sum(new) + pad
    rows = normal(n, lead + (H + 2 * Hk) * D, seed=3, dtype=in_type)[:, lead:]  # `lead` elements shift the alignment
    q = torch.as_strided(rows, (n, H, D), (rows.stride(0), D, 1), rows.storage_offset())
    k = torch.as_strided(rows, (n, Hk, D), (rows.stride(0), D, 1), rows.storage_offset() + H * D)
    v = torch.as_strided(rows, (n, Hk, D), (rows.stride(0), D, 1), rows.storage_offset() + (H + Hk) * D)
    pos = torch.cat([torch.arange(m, dtype=torch.int32) + far + 10 * i for i, m in enumerate(new)] + [torch.zeros(pad, dtype=torch.int32)]).to(DEV)
    inv = torch.from_numpy(capi.rope_frequencies(rotary, 1e6)[0]).to(DEV)
    out = q if in_place else torch.full((n, H, D), 7.0, dtype=t, device=DEV)
    want_q = ref.rotate(q, pos, inv, factor, interleaved)
    want_k, want_v = ref.rotate(k, pos, inv, factor, interleaved), v.double()
    reach = (2 * factor * q.double().abs().amax(), 2 * factor * k.double().abs().amax())
    old_q = q.clone()
    before = c["pool"].clone()
    c["weight"].fill_(5.0)
    c["position"].fill_(-3)
    capi.rope_append(view(c, status, position=c["position"], weight=c["weight"]), ref.cu_of(new, DEV), pos, q, k, v, inv, out,
                     interleaved=interleaved, factor=factor)
    torch.cuda.synchronize()
    h, live = half(t), sum(new)
    tol = 2.0 ** -21
    assert ((out[:live].double() - want_q[:live]).abs() <= h * want_q[:live].abs() * 1.001 + tol * reach[0]).all()
    if pad:
        assert torch.equal(out[live:], old_q[live:] if in_place else torch.full_like(out[live:], 7.0))
    want = before.clone()
    wpos, ww = torch.full_like(c["position"], -3), torch.full_like(c["weight"], 5.0)
    at = 0
    for s, (length, m) in enumerate(zip(c["kv"], new)):
        for i in range(max(0, m - max(length, 0)), m):
            slot = length - m + i
            page, place = int(c["table"][s, slot // 64]), slot % 64
            if not 0 <= page < c["pool"].shape[0]:
                continue
            got_k = c["k"][page, :, place].double()
            assert ((got_k - want_k[at + i]).abs() <= h * want_k[at + i].abs() * 1.001 + tol * reach[1]).all()
            assert torch.equal(c["v"][page, :, place], v[at + i].to(t))
            want[page, :, :Hk, place] = c["pool"][page, :, :Hk, place]
            wpos[page, :, place], ww[page, :, place] = int(pos[at + i]), 0.0
        at += m
    assert torch.equal(c["pool"], want) and torch.equal(c["position"], wpos) and torch.equal(c["weight"], ww)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("from_f32", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 96), (64, 64), (64, 2), (128, 30), (128, 0), (64, 62)])
def test_rope_append(dtype, from_f32, interleaved, dim, rotary):
    c = ref.make_cache([70, 1, 300, 64, 65, 130], 2, dim, dtype, DEV)
    run_rope(c, [70, 1, 5, 64, 65, 0], 6, torch.float32 if from_f32 else dtype, rotary, interleaved, factor=1.25, far=1 << 20, pad=3)


@pytest.mark.parametrize("lead", [1, 2, 8])
def test_rope_append_any_alignment(lead):
    c = ref.make_cache([70, 3], 3, 64, torch.bfloat16, DEV, apart=True)
    run_rope(c, [9, 3], 3, torch.bfloat16, 64, False, lead=lead)


def test_rope_append_in_place_and_many_tokens():
    c = ref.make_cache([1500, 777], 8, 128, torch.bfloat16, DEV)
    run_rope(c, [1500, 7], 16, torch.bfloat16, 128, False, in_place=True, pad=2)
    c = ref.make_cache([1500, 777], 8, 128, torch.bfloat16, DEV)
    run_rope(c, [1500, 7], 16, torch.bfloat16, 128, True, in_place=True, pad=2)


def test_rope_append_far_positions():
    """Positions up to 2^31 - 1: the angle keeps its digits."""
    c = ref.make_cache([4], 1, 64, torch.float16, DEV)
    run_rope(c, [4], 1, torch.float32, 64, False, far=2**31 - 20)


def test_rope_append_flags_and_skips_bad_places():
    c = ref.make_cache([70, 2, 100], 2, 64, torch.bfloat16, DEV)
    c["table"][0, 1] = 1 << 20
    run_rope(c, [70, 5, 3], 4, torch.bfloat16, 64, False)  # a bad page, and a sequence shorter than its new tokens
    assert int(c["status"]) == capi.BAD_PAGE | capi.BAD_LEN
    c = ref.make_cache([70, 100], 2, 64, torch.bfloat16, DEV)
    before = c["pool"].clone()
    q = normal(4, 2, 64, dtype=torch.bfloat16)
    out = torch.full_like(q, 7.0)
    f = torch.from_numpy(capi.rope_frequencies(64, 1e4)[0]).to(DEV)
    pos = torch.zeros(4, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 9, 4], dtype=torch.int32, device=DEV)  # beyond the tokens, then descending
    capi.rope_append(view(c), cu, pos, q, q, q, f, out)
    assert int(c["status"]) & capi.BAD_TOKENS and torch.equal(c["pool"], before) and bool((out == 7.0).all())


# ---- attention -------------------------------------------------------------------------------------------------------


def check_attention(c, new, q, out, lse, scale=None, weight=None, decay=0.0, old_weight=None):
    D = q.shape[2]
    scale = D ** -0.5 if scale is None else scale
    w = ref.attention(c, new, q, scale)
    live = sum(new)
    h = half(q.dtype)
    n = max(max(c["kv"]), 1)
    e = ((D + 4) * 2.0 ** -24 * w["size"])[..., None]
    tol = h * w["out"].abs() + (h + 2 * e + 2.0 ** -19 + n * 2.0 ** -24) * w["spread"]
    bad = (out[:live].double() - w["out"]).abs() > tol * 1.001
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist(), float((out[:live].double() - w["out"]).abs().max()))
    if lse is not None:
        assert torch.equal(lse[:live] == -math.inf, w["lse"] == -math.inf)
        seen = w["lse"] > -math.inf
        off = (lse[:live].double() - w["lse"]).abs()[seen]
        assert (off <= (2 * e[..., 0] + 2.0 ** -20 + n * 2.0 ** -24)[seen] + 2.0 ** -22 * w["lse"].abs()[seen]).all(), float(off.max())
    if weight is not None:
        G = q.shape[1] // c["kv_heads"]
        terms = max(new) * G
        top = float(e.max()) if e.numel() else 0.0
        lse_off = 2 * top + 2.0 ** -20 + n * 2.0 ** -24 + 2.0 ** -22 * float(w["lse"][w["lse"] > -math.inf].abs().max())
        rel = 2 * top + lse_off + 2.0 ** -20 + (terms + 2) * 2.0 ** -24
        base = decay * old_weight.double() if decay else torch.zeros_like(w["weight"])
        want, touched = old_weight.double().clone(), torch.zeros_like(weight, dtype=torch.bool)
        for s, (length, m) in enumerate(zip(c["kv"], new)):
            if m and length > 0:
                page, place = ref.rows_of(c, s, length)
                want[page, :, place] = (base + w["weight"])[page, :, place]
                touched[page, :, place] = True
        assert torch.equal(weight[~touched], old_weight[~touched])
        off = (weight.double() - want).abs()
        assert (off <= rel * w["weight"] + 2.0 ** -23 * want.abs() + 1e-37).all(), float((off / want.abs().clamp(min=1e-30)).max())


def run_attention(c, new, H, seed=1, scale=None, max_tokens=0, pad=0, q_scale=1.5, decay=None, strided=False, poison=True):
    D, t = c["dim"], c["pool"].dtype
    n = sum(new) + pad
    q = normal(n, H + (3 if strided else 0), D, seed=seed, dtype=t, scale=q_scale)[:, :H]
    out = torch.full((n, H + (2 if strided else 0), D), 7.0, dtype=t, device=DEV)[:, :H]
    lse = torch.full((n, H), 9.0, device=DEV)
    if poison:  # what no row sees may hold anything
        for s, length in enumerate(c["kv"]):
            length = max(length, 0)
            if length % 64:
                page = int(c["table"][s, length // 64])
                c["k"][page, :, length % 64:] = math.nan
                c["v"][page, :, length % 64:] = math.inf
    cu = ref.cu_of(new, DEV)
    ws = space()
    old = torch.rand(c["weight"].shape, device=DEV)
    c["weight"].copy_(old)
    cache = view(c, weight=c["weight"])
    capi.paged_attention(cache, cu, q, out, ws, lse=lse, scale=scale, max_tokens=max_tokens)
    if decay is not None:
        capi.attention_weights(cache, cu, q, lse, decay=decay, scale=scale, max_tokens=max_tokens)
    torch.cuda.synchronize()
    check_attention(c, new, q, out, lse, scale, c["weight"] if decay is not None else None, decay or 0.0, old)
    assert bool((out[sum(new):] == 7.0).all()) and bool((lse[sum(new):] == 9.0).all())
    if decay is None:
        assert torch.equal(c["weight"], old)
    return q, out, lse, ws


GROUPS = [(1, 1), (8, 2), (3, 3), (2, 4), (1, 7), (2, 8), (1, 16)]  # KV heads, query heads for each


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv_heads,group", GROUPS)
def test_attention_steps(dtype, dim, kv_heads, group):
    """One token each, over lengths around the pages' ends."""
    kv = [1, 2, 63, 64, 65, 127, 128, 129, 500, 1025]
    run_attention(ref.make_cache(kv, kv_heads, dim, dtype, DEV), [1] * len(kv), kv_heads * group, decay=0.5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv_heads,group", GROUPS)
def test_attention_chunks(dtype, dim, kv_heads, group):
    """Chunks of many sizes, fresh prompts and ones deep in a cache; some sequences without new tokens or without a cache."""
    kv, new = [5, 64, 200, 129, 0, 700, 300, 257], [5, 64, 200, 128, 0, 33, 0, 150]
    run_attention(ref.make_cache(kv, kv_heads, dim, dtype, DEV), new, kv_heads * group, decay=1.0, pad=2)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [2, 3, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257])
def test_attention_every_chunk_size(dim, new):
    run_attention(ref.make_cache([1000, new, new + 1], 2, dim, torch.bfloat16, DEV), [new, new, new], 4, decay=0.0)


@pytest.mark.parametrize("max_tokens", [1, 5, 64, 10**6])
def test_attention_hint_only_picks_the_kernel(max_tokens):
    run_attention(ref.make_cache([300, 77, 129], 2, 128, torch.float16, DEV), [200, 1, 40], 8, max_tokens=max_tokens, decay=0.0)


@pytest.mark.parametrize("group", [32, 64, 48])
def test_attention_wide_groups(group):
    run_attention(ref.make_cache([300, 77], 1, 128, torch.bfloat16, DEV), [20, 1], group, decay=0.0)
    run_attention(ref.make_cache([300, 1], 2, 64, torch.bfloat16, DEV), [1, 1], 2 * group)


def test_attention_long_step_is_split():
    run_attention(ref.make_cache([27000], 8, 128, torch.float16, DEV), [1], 16, decay=0.0)
    run_attention(ref.make_cache([20011, 3, 9000], 2, 128, torch.bfloat16, DEV), [8, 3, 1], 4, decay=0.9)


def test_attention_long_chunk_is_split():
    run_attention(ref.make_cache([9001, 700], 2, 128, torch.bfloat16, DEV), [513, 300], 4, decay=0.0)
    run_attention(ref.make_cache([8192], 1, 64, torch.float16, DEV), [8192], 2, decay=0.0)


def test_attention_many_sequences():
    kv = [(37 * i) % 401 for i in range(700)]
    new = [min(n, (i % 3)) for i, n in enumerate(kv)]
    run_attention(ref.make_cache(kv, 1, 64, torch.bfloat16, DEV), new, 2, decay=0.0)


@pytest.mark.parametrize("dim,group", [(64, 1), (128, 2), (64, 8), (128, 3)])
def test_attention_chunks_of_many_ragged_sequences(dim, group):
    """Tiles of one and of two halves, of one block and of many, in turn within a CTA's interval; the same bits each time."""
    new = [(0, 1, 5, 64, 65, 130, 257, 33)[i % 8] for i in range(61)]
    kv = [n + (53 * i * i) % 700 for i, n in enumerate(new)]
    c = ref.make_cache(kv, 3, dim, torch.bfloat16, DEV)
    first = run_attention(c, new, 3 * group, decay=0.0)[1]
    for _ in range(3):
        assert torch.equal(run_attention(c, new, 3 * group, decay=0.0)[1], first)


@pytest.mark.parametrize("new", [[3, 2, 1, 4], [300, 140, 1, 150]])
def test_attention_rows_that_see_nothing(new):
    """Sequences shorter than their new tokens: the rows before the first slot see nothing."""
    c = ref.make_cache([1, 0, 0, 130], 2, 128, torch.bfloat16, DEV, table_len=8)
    q, out, lse, _ = run_attention(c, new, 4, decay=0.0)
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    assert int(c["status"]) == capi.BAD_LEN


def test_attention_strides_and_gaps():
    c = ref.make_cache([300, 65, 400], 3, 64, torch.float16, DEV, apart=True)
    run_attention(c, [1, 1, 1], 6, strided=True, decay=0.0)
    run_attention(c, [140, 65, 2], 6, strided=True, decay=0.0)


@pytest.mark.parametrize("new", [1, 150])
def test_attention_extreme_scores(new):
    """Scores of thousands apart: one slot takes all; a scale of 0 averages; a negative one turns the order."""
    c = ref.make_cache([700], 2, 128, torch.bfloat16, DEV)
    run_attention(c, [new], 4, q_scale=60.0, decay=0.0)
    run_attention(c, [new], 4, scale=0.0, decay=0.0)
    run_attention(c, [new], 4, scale=-0.2, decay=0.0)
    # Rising scores: the running maximum grows with every page.
    grow = torch.linspace(0.01, 8.0, 704, device=DEV).view(11, 64, 1)
    for p in range(11):
        c["k"][int(c["table"][0, p])] = (grow[p] * torch.ones(2, 64, 128, device=DEV)).to(torch.bfloat16)
    q = torch.ones(new, 4, 128, dtype=torch.bfloat16, device=DEV)
    out, lse = torch.zeros_like(q), torch.zeros(new, 4, device=DEV)
    capi.paged_attention(view(c), ref.cu_of([new], DEV), q, out, space(), lse=lse)
    check_attention(c, [new], q, out, lse)
    capi.paged_attention(view(c), ref.cu_of([new], DEV), -q, out, space(), lse=lse)
    check_attention(c, [new], -q, out, lse)


@pytest.mark.parametrize("new", [1, 150])
def test_attention_nan_stays_in_its_row(new):
    """A NaN or infinite query makes its own row NaN and no other; a NaN key those that see it."""
    c = ref.make_cache([400, 300], 2, 64, torch.float16, DEV)
    q = normal(2 * new, 4, 64, dtype=torch.float16)
    clean = q.clone()
    q[0, 1, 5] = math.nan
    out, lse = torch.zeros_like(q), torch.zeros(2 * new, 4, device=DEV)
    cu = ref.cu_of([new, new], DEV)
    capi.paged_attention(view(c), cu, q, out, space(), lse=lse)
    assert bool(out[0, 1].isnan().all()) and bool(lse[0, 1].isnan())
    out[0, 1], lse[0, 1] = 0.0, 0.0
    want, want_lse = torch.zeros_like(q), torch.zeros_like(lse)
    capi.paged_attention(view(c), cu, clean, want, space(), lse=want_lse)
    want[0, 1], want_lse[0, 1] = 0.0, 0.0
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    # The last slot's key: seen by the last token of sequence 0 alone.
    page, place = ref.rows_of(c, 0, 400)
    c["k"][page[-1], 0, place[-1], 3] = math.nan
    capi.paged_attention(view(c), cu, clean, out, space(), lse=lse)
    assert bool(out[new - 1, :2].isnan().all())
    out[new - 1, :2] = want[new - 1, :2]
    out[0, 1] = 0.0
    assert torch.equal(out, want)


@pytest.mark.parametrize("new", [1, 150])
def test_attention_bad_pages_count_as_masked(new):
    c = ref.make_cache([400, 300], 2, 64, torch.float16, DEV)
    q = normal(2 * new, 4, 64, dtype=torch.float16)
    out, lse = torch.zeros_like(q), torch.zeros(2 * new, 4, device=DEV)
    cu = ref.cu_of([new, new], DEV)
    c["table"][0, 1], c["table"][1, 0] = -1, 1 << 30
    capi.paged_attention(view(c, weight=c["weight"]), cu, q, out, space(), lse=lse)
    capi.attention_weights(view(c, weight=c["weight"]), cu, q, lse, decay=0.0)
    torch.cuda.synchronize()
    assert int(c["status"]) == capi.BAD_PAGE
    for s, length in enumerate((400, 300)):
        keep = [j for j in range(length) if 0 <= int(c["table"][s, j // 64]) < c["pool"].shape[0]]
        page, place = ref.rows_of(c, s, length)
        keep = torch.tensor(keep, device=DEV)
        for i in (0, new - 1):
            for h in range(4):
                see = keep[keep <= length - new + i]
                k, v = c["k"][page[see], h // 2, place[see]].double(), c["v"][page[see], h // 2, place[see]].double()
                a = (k @ q[s * new + i, h].double()) / 8
                o = torch.softmax(a, 0) @ v
                # 16-bit roundings of the result and the probabilities, as above, with |v| at most 5.
                assert (out[s * new + i, h].double() - o).abs().max() <= half(torch.float16) * 10 + 1e-4
                assert abs(float(lse[s * new + i, h]) - float(torch.logsumexp(a, 0))) < 1e-4


def test_attention_bad_lengths_and_tokens():
    c = ref.make_cache([64, 128], 1, 64, torch.bfloat16, DEV, table_len=2)
    c["table"][0, 1] = c["table"][1, 1]
    c["kv_len"].copy_(torch.tensor([1000, -5], dtype=torch.int32))
    q = normal(2, 1, 64, dtype=torch.bfloat16)
    out, lse = torch.zeros_like(q), torch.zeros(2, 1, device=DEV)
    capi.paged_attention(view(c), ref.cu_of([1, 1], DEV), q, out, space(), lse=lse)
    assert int(c["status"]) == capi.BAD_LEN
    c["kv"] = [128, 0]
    check_attention(c, [1, 1], q, out, lse)
    c["status"].zero_()
    c["kv_len"].copy_(torch.tensor([64, 64], dtype=torch.int32))
    out.fill_(7.0)
    capi.paged_attention(view(c), torch.tensor([0, 3, 2], dtype=torch.int32, device=DEV), q, out, space(), lse=lse)
    assert int(c["status"]) == capi.BAD_TOKENS and bool((out == 7.0).all())


def test_attention_offsets_beyond_32_bits():
    """Pages more than 2^31 elements into the pool."""
    pages = (1 << 31) // (2 * 64 * 128) + 40
    pool = torch.empty(pages, 2, 1, 64, 128, dtype=torch.bfloat16, device=DEV)
    for new, kv in ((1, 300), (200, 300)):
        last = torch.arange(pages - 5, pages, device=DEV)
        pool[last] = normal(5, 2, 1, 64, 128, dtype=torch.bfloat16)
        c = {"pool": pool, "k": pool[:, 0], "v": pool[:, 1], "table": last.to(torch.int32)[None].contiguous(),
             "kv_len": torch.tensor([kv], dtype=torch.int32, device=DEV), "kv": [kv], "kv_heads": 1, "dim": 128,
             "weight": torch.zeros(pages, 1, 64, device=DEV), "status": torch.zeros(1, dtype=torch.int32, device=DEV),
             "position": torch.zeros(pages, 1, 64, dtype=torch.int32, device=DEV)}
        run_attention(c, [new], 2, decay=0.0)


@pytest.mark.parametrize("new", [1, 8, 300])
def test_attention_repeats_to_the_bit(new):
    c = ref.make_cache([5000, 300, 2500], 2, 128, torch.bfloat16, DEV)
    q, out, lse, ws = run_attention(c, [new] * 3, 4, decay=0.0)
    cache = view(c, weight=c["weight"])
    w = c["weight"].clone()
    for _ in range(5):
        again, lse2 = torch.zeros_like(out), torch.zeros_like(lse)
        capi.paged_attention(cache, ref.cu_of([new] * 3, DEV), q, again, ws, lse=lse2)
        capi.attention_weights(cache, ref.cu_of([new] * 3, DEV), q, lse2, decay=0.0)
        assert torch.equal(again, out) and torch.equal(lse2, lse) and torch.equal(c["weight"], w)


@pytest.mark.parametrize("new", [1, 300])
def test_attention_captured_streams_and_workspaces(new):
    """A captured call replays on new lengths and pages; two streams with a workspace each run at the same time."""
    c = ref.make_cache([3000, 1000], 2, 128, torch.bfloat16, DEV)
    d = ref.make_cache([1200, 2900], 2, 128, torch.bfloat16, DEV, seed=5, table_len=47)
    q = normal(2 * new, 4, 128, dtype=torch.bfloat16)
    cu = ref.cu_of([new, new], DEV)
    out, lse, ws = torch.zeros_like(q), torch.zeros(2 * new, 4, device=DEV), space()
    cache = view(c, weight=c["weight"])
    side = torch.cuda.Stream()
    capi.paged_attention(cache, cu, q, out, ws, lse=lse)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        capi.paged_attention(cache, cu, q, out, ws, lse=lse)
        capi.attention_weights(cache, cu, q, lse, decay=0.0)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    check_attention(c, [new, new], q, out, lse)
    c["kv_len"].copy_(torch.tensor([2000, 600], dtype=torch.int32))
    c["kv"] = [2000, 600]
    graph.replay()
    torch.cuda.synchronize()
    check_attention(c, [new, new], q, out, lse)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    out2, lse2, ws2 = torch.zeros_like(q), torch.zeros_like(lse), space()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(a):
            capi.paged_attention(view(c), cu, q, out, ws, lse=lse)
        with torch.cuda.stream(b):
            capi.paged_attention(view(d), cu, q, out2, ws2, lse=lse2)
    torch.cuda.synchronize()
    check_attention(c, [new, new], q, out, lse)
    check_attention(d, [new, new], q, out2, lse2)


# ---- eviction --------------------------------------------------------------------------------------------------------


def fill_books(c, seed=0, ties=False):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(0, 4, c["weight"].shape, generator=g).float() if ties else torch.randn(c["weight"].shape, generator=g).exp()
    c["weight"].copy_(w.to(DEV))
    for s, n in enumerate(c["kv"]):
        if n:
            page, place = ref.rows_of(c, s, n)
            pos = torch.stack([torch.randperm(2 * n, generator=g)[:n] for _ in range(c["kv_heads"])], 1).to(torch.int32).to(DEV)
            c["position"][page, :, place] = pos
    return c


def run_evict(c, keep, sinks, recent, alias=False):
    k, v, w, pos, lens = ref.evict(c, keep, sinks, recent)
    ws = torch.zeros(capi.cache_evict_workspace(len(c["kv"]), c["kv_heads"], c["table"].shape[1]), dtype=torch.uint8, device=DEV)
    new_len = c["kv_len"] if alias else torch.full((len(c["kv"]),), -1, dtype=torch.int32, device=DEV)
    capi.cache_evict(view(c, position=c["position"], weight=c["weight"]), keep, new_len, ws, sinks=sinks, recent=recent)
    torch.cuda.synchronize()
    assert new_len.tolist() == lens
    bits = torch.int16
    assert torch.equal(c["k"].contiguous().view(bits), k.contiguous().view(bits)) and torch.equal(c["v"].contiguous().view(bits), v.contiguous().view(bits))
    assert torch.equal(c["position"], pos)
    assert torch.equal(c["weight"].view(torch.int32), w.view(torch.int32))


@pytest.mark.parametrize("dtype,dim,heads", [(torch.float16, 128, 2), (torch.bfloat16, 64, 3), (torch.bfloat16, 128, 8)])
@pytest.mark.parametrize("keep,sinks,recent", [(64, 4, 16), (100, 0, 0), (1, 0, 1), (0, 0, 0), (200, 100, 100), (513, 0, 500), (1000, 4, 64)])
def test_evict(dtype, dim, heads, keep, sinks, recent):
    kv = [0, 1, 63, 64, 65, 100, 101, 513, 514, 1300]
    run_evict(fill_books(ref.make_cache(kv, heads, dim, dtype, DEV)), keep, sinks, recent)


@pytest.mark.parametrize("alias", [False, True])
def test_evict_ties_specials_and_aliased_lengths(alias):
    """Equal weights: the lowest slots stay.  NaN ranks below all, then -inf; -0 as 0; equal positions."""
    c = fill_books(ref.make_cache([700, 65, 2000], 2, 64, torch.bfloat16, DEV, apart=True), ties=True)
    page, place = ref.rows_of(c, 0, 700)
    special = torch.tensor([math.nan, math.inf, -math.inf, -0.0, 0.0, -1.0, 1e-42, 3.4e38], device=DEV)
    c["weight"][page[::5], 1, place[::5]] = special[torch.arange(140, device=DEV) % 8]
    c["position"][page, 0, place] = 9
    run_evict(c, 64, 3, 7, alias)


def test_evict_all_equal_and_all_nan():
    c = fill_books(ref.make_cache([500, 400], 1, 64, torch.float16, DEV))
    c["weight"].fill_(0.0)
    run_evict(c, 130, 0, 10)
    c["weight"].fill_(math.nan)
    run_evict(c, 77, 2, 5)


def test_evict_long_and_beyond_the_shared_keys():
    run_evict(fill_books(ref.make_cache([27000, 8192, 8193], 2, 64, torch.bfloat16, DEV)), 8192, 4, 512)
    run_evict(fill_books(ref.make_cache([50001], 1, 64, torch.bfloat16, DEV)), 20000, 4, 100)


def test_evict_bad_page_leaves_the_sequence():
    c = fill_books(ref.make_cache([300, 300], 2, 64, torch.float16, DEV))
    c["table"][0, 2] = -1
    before = [c[x].clone() for x in ("pool", "weight", "position")]
    ws = torch.zeros(capi.cache_evict_workspace(2, 2, 5), dtype=torch.uint8, device=DEV)
    new_len = torch.zeros(2, dtype=torch.int32, device=DEV)
    capi.cache_evict(view(c, position=c["position"], weight=c["weight"]), 100, new_len, ws)
    assert new_len.tolist() == [300, 100] and int(c["status"]) == capi.BAD_PAGE
    page, place = ref.rows_of(c, 1, 300)
    other = torch.ones(c["pool"].shape[0], dtype=torch.bool, device=DEV)
    other[page] = False
    for x, y in zip(("pool", "weight", "position"), before):
        assert torch.equal(c[x][other], y[other])


# ---- logits ----------------------------------------------------------------------------------------------------------


def run_logits(rows, vocab, dtype, hist=0, biases=0, masked=None, seed=0, lead=0, gap=0, in_place=False, parts=("repetition", "presence", "frequency")):
    g = torch.Generator().manual_seed(seed)
    base = (3 * torch.randn(rows, lead + vocab + gap, generator=g)).to(dtype).to(DEV)
    x = base[:, lead:lead + vocab]
    hl = [int(torch.randint(0, hist + 1, (1,), generator=g)) if hist else 0 for _ in range(rows)]
    ids = torch.randint(-2, vocab + 2, (sum(hl) + 1,), generator=g).to(torch.int32)
    ids[::3] = ids[0].clamp(0, vocab - 1)
    hb = torch.tensor([0] + hl[:-1]).cumsum(0).to(torch.int32)
    he = hb + torch.tensor(hl, dtype=torch.int32)
    kw, values = {}, {}
    if hist:
        kw.update(history=ids.to(DEV), hist_begin=hb.to(DEV), hist_end=he.to(DEV))
        for name in parts:
            values[name] = (1.0 if name == "repetition" else 0.0) + torch.rand(rows, generator=g)
            kw[name] = values[name].to(DEV)
    if biases:
        bi = torch.randint(-1, vocab + 1, (rows * biases,), generator=g).to(torch.int32)
        bi[1::4] = bi[0::4][: bi[1::4].numel()]  # the same id twice: the last entry counts
        bv = 4 * torch.randn(rows * biases, generator=g)
        bb = torch.arange(rows, dtype=torch.int32) * biases
        kw.update(bias_ids=bi.to(DEV), bias_values=bv.to(DEV), bias_begin=bb.to(DEV), bias_end=(bb + biases).to(DEV))
    allowed = None
    if masked is not None:
        allowed = torch.rand(rows, vocab, generator=g) >= masked
        words = -(-vocab // 32)
        bits = torch.zeros(rows, words * 32, dtype=torch.int64)
        bits[:, :vocab] = allowed
        word = (bits.view(rows, words, 32) << torch.arange(32)).sum(-1)
        kw["mask"] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32).to(DEV)
    before = x.clone()
    out = x if in_place else torch.full((rows, vocab + gap), 7.0, dtype=dtype, device=DEV)[:, :vocab]
    choice = torch.full((rows,), -9, dtype=torch.int32, device=DEV)
    capi.logits_process(x, out, choice, **kw)
    torch.cuda.synchronize()
    for r in range(rows):
        want = ref.logits(before[r], ids[int(hb[r]):int(he[r])].tolist(), *(float(values[n][r]) if n in values else None
                          for n in ("repetition", "presence", "frequency")),
                          list(zip(bi[r * biases:(r + 1) * biases].tolist(), bv[r * biases:(r + 1) * biases].tolist())) if biases else None,
                          allowed[r].tolist() if allowed is not None else None)
        got = out[r].double().cpu()
        assert torch.equal(got == -math.inf, want == -math.inf)
        ok = want > -math.inf
        # Five f32 steps on values below 2^9 (|x| < 20, times at most 2, less 2 times at most `hist` counts), then the type's rounding.
        size = 64.0 + hist
        assert ((got - want)[ok].abs() <= half(dtype) * want[ok].abs() * 1.001 + 5 * 2.0 ** -24 * size).all()
        c = int(choice[r])
        if not ok.any():
            assert c == -1
        else:
            assert want[c] >= want[ok].max() - 10 * 2.0 ** -24 * size
            if dtype != torch.float32 and not hist and not biases:  # exact values: the first of the equal ones
                assert c == int(torch.argmax(want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 31), (2, 33), (5, 1000), (2, 8192), (1, 65537), (2, 151936)])
def test_logits(dtype, rows, vocab):
    run_logits(rows, vocab, dtype)
    run_logits(rows, vocab, dtype, hist=200, biases=17, masked=0.4, seed=1, gap=5)
    run_logits(rows, vocab, dtype, hist=3000, seed=2, lead=1, parts=("repetition",))
    run_logits(rows, vocab, dtype, biases=5, masked=0.999, seed=3, in_place=True)


def test_logits_parts_alone_and_many_rows():
    for part in ("repetition", "presence", "frequency"):
        run_logits(4, 777, torch.float32, hist=50, parts=(part,))
    run_logits(300, 501, torch.bfloat16, hist=20, biases=3, masked=0.5)


@pytest.mark.parametrize("rows,vocab,hist,biases", [
    (2, 151936, 4096, 1), (2, 20011, 4097, 300), (130, 5003, 4500, 100), (130, 1000, 6100, 44), (130, 1000, 6100, 45), (3, 9999, 1, 6143),
    (3, 9999, 6145, 0), (130, 262144, 40, 3), (130, 262145, 40, 3)])
def test_logits_list_lengths_and_shares_at_their_limits(rows, vocab, hist, biases):
    """Entries beyond those that a thread holds, lists of 6144 entries and one more, a share of 262144 ids and one more."""
    run_logits(rows, vocab, torch.float16, hist=hist, biases=biases, masked=0.3, seed=rows + hist)
    run_logits(rows, vocab, torch.float16, hist=hist, biases=biases, seed=hist, in_place=True, lead=1)


def test_logits_nothing_allowed_nan_and_shared_masks():
    x = normal(4, 5000)
    x[0, 3] = math.nan
    x[1] = -math.inf
    x[2, 4999] = math.inf
    mask = torch.zeros(2, 157, dtype=torch.int32, device=DEV)
    mask[1, 0] = 0b1010
    rows = torch.tensor([1, -1, 0, 7], dtype=torch.int32, device=DEV)  # a mask row that is not there: not masked
    out, choice = torch.empty_like(x), torch.empty(4, dtype=torch.int32, device=DEV)
    capi.logits_process(x, out, choice, mask=mask, mask_row=rows)
    assert choice.tolist() == [1, -1, -1, int(x[3].argmax())]
    assert bool(out[0, 3].isnan()) and float(out[0, 1]) == float(x[0, 1]) and int((out[0] > -math.inf).sum()) == 1
    assert bool((out[2] == -math.inf).all()) and torch.equal(out[3], x[3])
    capi.logits_process(x, out, choice)
    assert choice.tolist()[1:3] == [-1, 4999] and choice[0] == int(torch.nan_to_num(x[0], nan=-9e9).argmax())
    only = torch.empty(4, dtype=torch.int32, device=DEV)
    capi.logits_process(x, None, only)
    assert torch.equal(only, choice)


def test_logits_ranges_are_cut_to_their_buffers():
    x = normal(2, 300)
    hist = torch.tensor([5, 6, 7], dtype=torch.int32, device=DEV)
    lo, hi = torch.tensor([-4, 2], dtype=torch.int32, device=DEV), torch.tensor([2, 1 << 30], dtype=torch.int32, device=DEV)
    out = torch.empty_like(x)
    p = torch.ones(2, device=DEV)
    capi.logits_process(x, out, history=hist, hist_begin=lo, hist_end=hi, presence=p, bias_ids=hist, bias_values=torch.ones(3, device=DEV),
                        bias_begin=lo, bias_end=hi)
    want = x.clone()
    assert torch.allclose(out, want, atol=1e-6)  # - 1 + 1 on the same ids
    capi.logits_process(x, out, history=hist, hist_begin=lo, hist_end=hi, presence=p)
    want[0, 5:7] -= 1
    want[1, 7] -= 1
    assert torch.equal(out, want)


def test_logits_bounds_near_the_end_of_int32():
    """A range that begins behind its list is empty, whatever lies between its begin and 2^31, beside a list that has entries."""
    x = normal(2, 300)
    ids = torch.tensor([5, 6, 7], dtype=torch.int32, device=DEV)
    far = torch.full((2,), 2**31 - 1, dtype=torch.int32, device=DEV)
    lo, hi = torch.zeros(2, dtype=torch.int32, device=DEV), torch.full((2,), 3, dtype=torch.int32, device=DEV)
    ones, p = torch.ones(3, device=DEV), torch.ones(2, device=DEV)
    out = torch.empty_like(x)
    capi.logits_process(x, out, history=ids, hist_begin=far, hist_end=far, presence=p, bias_ids=ids, bias_values=ones, bias_begin=lo, bias_end=hi)
    want = x.clone()
    want[:, 5:8] += 1
    assert torch.equal(out, want)
    capi.logits_process(x, out, history=ids, hist_begin=lo, hist_end=hi, presence=p, bias_ids=ids, bias_values=ones, bias_begin=far, bias_end=far)
    want = x.clone()
    want[:, 5:8] -= 1
    assert torch.equal(out, want)


def test_logits_repetition_is_greedy_choice_of_the_decoder(tiny_gguf):
    """With the repetition penalty alone, on the last 100 ids, the choice is mtb_greedy_choice's."""
    model = capi.Model(tiny_gguf, 0)
    dec = capi.Decoder(model, 64, capi.KV_F32, max_new=256)
    for seed in range(6):
        x = normal(1, model.vocab, seed=seed)
        hist = x[0].topk(40).indices[torch.randint(0, 40, (150,), generator=torch.Generator().manual_seed(seed)).to(DEV)].to(torch.int32)
        choice = torch.empty(1, dtype=torch.int32, device=DEV)
        capi.logits_process(x, None, choice, history=hist, hist_begin=torch.tensor([50], dtype=torch.int32, device=DEV),
                            hist_end=torch.tensor([150], dtype=torch.int32, device=DEV), repetition=torch.tensor([1.3], device=DEV))
        assert int(choice) == dec.cpu_greedy_choice(x[0].cpu().numpy(), hist.cpu().tolist(), float(torch.tensor(1.3)))
    dec.close()
    model.close()


# ---- together --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_bounded_cache_serves_a_run(dtype):
    """Prompts, then steps: rotary positions with the append, attention, its weights, eviction when a cache passes its budget,
    and the choice under penalties; after each call the 64-bit definition on the same inputs."""
    Hk, G, D, budget, V = 2, 2, 64, 192, 1000
    kv = [150, 40]
    c = ref.make_cache([320, 320], Hk, D, dtype, DEV, fill=0.0)
    c["kv"] = [0, 0]
    inv, factor = capi.rope_frequencies(D, 1e4, capi.ROPE_YARN, 4.0, 128.0)
    inv = torch.from_numpy(inv).to(DEV)
    ws = space()
    ews = torch.zeros(capi.cache_evict_workspace(2, Hk, c["table"].shape[1]), dtype=torch.uint8, device=DEV)
    cache = view(c, position=c["position"], weight=c["weight"])
    told, history = [0, 0], [[], []]
    head = normal(D * Hk * G, V, seed=9, scale=0.2)
    for step in range(40):
        new = list(kv) if step == 0 else [1 + 7 * (step % 4 == 1), 4]
        n = sum(new)
        rows = normal(n, Hk * G + 2 * Hk, D, seed=100 + step, dtype=dtype)
        pos = torch.cat([torch.arange(t, t + m, dtype=torch.int32) for t, m in zip(told, new)]).to(DEV)
        told = [t + m for t, m in zip(told, new)]
        c["kv"] = [a + m for a, m in zip(c["kv"], new)]
        c["kv_len"].copy_(torch.tensor(c["kv"], dtype=torch.int32))
        cu = ref.cu_of(new, DEV)
        q = torch.empty(n, Hk * G, D, dtype=dtype, device=DEV)
        out, lse = torch.empty_like(q), torch.empty(n, Hk * G, device=DEV)
        capi.rope_append(cache, cu, pos, rows[:, :Hk * G], rows[:, Hk * G:Hk * G + Hk], rows[:, Hk * G + Hk:], inv, q, factor=factor)
        old = c["weight"].clone()
        capi.paged_attention(cache, cu, q, out, ws, lse=lse, max_tokens=max(new))
        capi.attention_weights(cache, cu, q, lse, decay=0.97, max_tokens=max(new))
        check_attention(c, new, q, out, lse, None, c["weight"], 0.97, old)
        last = cu[1:].long() - 1
        x = out[last].flatten(1).float() @ head
        flat = torch.tensor(sum(history, []) + [0], dtype=torch.int32, device=DEV)
        lo = torch.tensor([0, len(history[0])], dtype=torch.int32, device=DEV)
        hi = torch.tensor([len(history[0]), len(history[0]) + len(history[1])], dtype=torch.int32, device=DEV)
        y, choice = torch.empty_like(x), torch.empty(2, dtype=torch.int32, device=DEV)
        capi.logits_process(x, y, choice, history=flat, hist_begin=lo, hist_end=hi, presence=torch.full((2,), 1e4, device=DEV))
        for s in range(2):
            assert int(choice[s]) not in history[s]  # a presence penalty that large forbids any repeat
            history[s].append(int(choice[s]))
        if max(c["kv"]) > budget + 16:
            run_evict(c, budget, 4, 64, alias=True)
            c["kv"] = [min(a, budget) for a in c["kv"]]
            for s in range(2):  # the first and the newest positions stayed
                page, place = ref.rows_of(c, s, c["kv"][s])
                for h in range(Hk):
                    held = set(c["position"][page, h, place].tolist())
                    assert {0, 1, 2, 3} <= held and set(range(told[s] - 64, told[s])) <= held and len(held) == c["kv"][s]
    assert told[0] > budget and int(c["status"]) == 0


def test_logits_longer_lists_than_16_bits():
    """Histories and bias lists of more than 65535 entries: counts and the last entry are still exact."""
    vocab, n = 40000, 70001
    x = normal(2, vocab, seed=4)
    g = torch.Generator().manual_seed(1)
    hist = torch.randint(0, 30, (n,), generator=g).to(torch.int32)
    hist[:1000] = torch.randint(0, vocab, (1000,), generator=g).to(torch.int32)
    ids = torch.randint(0, vocab, (n,), generator=g).to(torch.int32)
    val = torch.randn(n, generator=g)
    lo, hi = torch.tensor([0, 69000], dtype=torch.int32, device=DEV), torch.tensor([n, n], dtype=torch.int32, device=DEV)
    freq = torch.tensor([2.0 ** -10, 0.5], device=DEV)
    out, choice = torch.empty_like(x), torch.empty(2, dtype=torch.int32, device=DEV)
    capi.logits_process(x, out, choice, history=hist.to(DEV), hist_begin=lo, hist_end=hi, frequency=freq, bias_ids=ids.to(DEV),
                        bias_values=val.to(DEV), bias_begin=lo, bias_end=hi)
    for r in range(2):
        a = int(lo[r])
        count = torch.bincount(hist[a:].long(), minlength=vocab).to(DEV)
        last = torch.full((vocab,), -1, dtype=torch.int64)
        last.scatter_reduce_(0, ids[a:].long(), torch.arange(a, n), "amax")
        bias = torch.where(last >= 0, val[last.clamp(min=0)], torch.zeros(())).to(DEV)
        want = torch.where(count > 0, x[r] - freq[r] * count, x[r])  # f32 in the operator's order: equal to the bit
        want = torch.where(last.to(DEV) >= 0, want + bias, want)
        assert torch.equal(out[r], want) and int(choice[r]) == int(want.argmax())


# ---- captured together, and over the whole range --------------------------------------------------------------------


def test_a_captured_step_replays_on_what_the_host_changes():
    """Append, attention, weights, eviction and choice in one graph: replays follow lengths, pages, tokens and books."""
    Hk, G, D, V, dtype = 2, 2, 128, 3000, torch.bfloat16
    c = ref.make_cache([640, 640], Hk, D, dtype, DEV)
    c["kv"] = [500, 301]
    c["kv_len"].copy_(torch.tensor(c["kv"], dtype=torch.int32))
    fill_books(c)
    new, n = [2, 1], 3
    cu = ref.cu_of(new, DEV)
    rows, pos = normal(n, Hk * G + 2 * Hk, D, dtype=dtype), torch.tensor([1200, 1201, 900], dtype=torch.int32, device=DEV)
    inv = torch.from_numpy(capi.rope_frequencies(D, 1e6)[0]).to(DEV)
    q, lse, ws = torch.zeros(n, Hk * G, D, dtype=dtype, device=DEV), torch.zeros(n, Hk * G, device=DEV), space()
    out, x = torch.zeros_like(q), normal(2, V)
    ews = torch.zeros(capi.cache_evict_workspace(2, Hk, c["table"].shape[1]), dtype=torch.uint8, device=DEV)
    y, choice, new_len = torch.zeros_like(x), torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    hist, lo, hi = torch.tensor([5, 6, 7], dtype=torch.int32, device=DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV), torch.tensor([3, 3], dtype=torch.int32, device=DEV)
    rep = torch.tensor([1.5, 1.2], device=DEV)
    cache = view(c, position=c["position"], weight=c["weight"])

    def step():
        capi.rope_append(cache, cu, pos, rows[:, :Hk * G], rows[:, Hk * G:Hk * G + Hk], rows[:, Hk * G + Hk:], inv, q)
        capi.paged_attention(cache, cu, q, out, ws, lse=lse, max_tokens=2)
        capi.attention_weights(cache, cu, q, lse, decay=0.5, max_tokens=2)
        capi.cache_evict(cache, 300, new_len, ews, sinks=4, recent=50)
        capi.logits_process(x, y, choice, history=hist, hist_begin=lo, hist_end=hi, repetition=rep)

    state = [c[k].clone() for k in ("pool", "position", "weight")]

    def reset():
        for k, v in zip(("pool", "position", "weight"), state):
            c[k].copy_(v)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lengths in ([500, 301], [640, 299]):
        c["kv_len"].copy_(torch.tensor(lengths, dtype=torch.int32))
        x.copy_(normal(2, V, seed=lengths[0]))
        reset()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (c["pool"], c["position"], c["weight"], out, lse, new_len, y, choice)]
        reset()
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, (c["pool"], c["position"], c["weight"], out, lse, new_len, y, choice)):
            assert torch.equal(a, b)
        assert new_len.tolist() == [min(t, 300) for t in lengths]


@pytest.mark.parametrize("seed", range(12))
def test_attention_over_the_range(seed):
    import random
    r = random.Random(seed)
    Hk, D, G = r.choice([1, 2, 3, 5, 8]), r.choice([64, 128]), r.choice([1, 2, 3, 4, 5, 6, 8, 12])
    n_seq = r.choice([1, 2, 3, 7, 40])
    new = [r.choice([0, 1, 1, 2, r.randrange(1, 40), r.randrange(1, 600 // (1 + n_seq // 8))]) for _ in range(n_seq)]
    if not sum(new):
        new[0] = 1
    kv = [max(0, n + r.choice([0, 0, r.randrange(0, 300), r.randrange(0, 5000)])) for n in new]
    c = ref.make_cache(kv, Hk, D, r.choice([torch.float16, torch.bfloat16]), DEV, seed=seed, apart=r.random() < 0.3)
    run_attention(c, new, Hk * G, seed=seed, decay=r.choice([0.0, 0.7, 1.0]), pad=r.choice([0, 3]), strided=r.random() < 0.3,
                  max_tokens=r.choice([0, max(new), 1]))


@pytest.mark.parametrize("seed", range(8))
def test_evict_over_the_range(seed):
    import random
    r = random.Random(100 + seed)
    kv = [r.randrange(0, r.choice([70, 700, 9000])) for _ in range(r.choice([1, 3, 6]))]
    keep = r.randrange(0, max(kv) + 2)
    sinks = r.randrange(0, min(8, keep) + 1)
    c = fill_books(ref.make_cache(kv, r.choice([1, 2, 5]), r.choice([64, 128]), r.choice([torch.float16, torch.bfloat16]), DEV, seed=seed), seed, r.random() < 0.4)
    run_evict(c, keep, sinks, r.randrange(0, keep - sinks + 1), alias=r.random() < 0.5)


@pytest.mark.parametrize("seed", range(8))
def test_logits_over_the_range(seed):
    import random
    r = random.Random(200 + seed)
    vocab = r.choice([r.randrange(1, 100), r.randrange(100, 5000), r.randrange(5000, 200000)])
    rows = max(1, min(300, 400000 // vocab))
    run_logits(r.randrange(1, rows + 1), vocab, r.choice([torch.float32, torch.float16, torch.bfloat16]), hist=r.choice([0, 30, 7000]),
               biases=r.choice([0, 1, 400]), masked=r.choice([None, 0.5, 1.0]), seed=seed, lead=r.choice([0, 0, 1]), gap=r.choice([0, 3]),
               in_place=r.random() < 0.3)
