"""What the operators on a caller's own device memory refuse, and what needs no GPU: argument limits are checked before any
device is touched, so these calls carry made-up addresses that nothing reads."""
import ctypes as C
import math

import numpy as np
import pytest

from mtb import capi

P = 1 << 20  # an aligned address that is never read


def cache(**change):
    v = dict(k=P, v=P, type=capi.T_BF16, head_dim=128, n_kv_heads=8, n_pages=16, page_stride=2 * 8 * 64 * 128, head_stride=64 * 128,
             page_table=P, table_stride=4, n_seq=2, kv_len=P, position=P, weight=P, status=None)
    v.update(change)
    return capi.PagedCacheView(**v)


def error():
    return capi.lib().mtb_global_error().decode()


BAD_CACHES = [dict(k=None), dict(v=None), dict(page_table=None), dict(kv_len=None), dict(type=capi.T_F32), dict(type=7), dict(head_dim=96),
              dict(head_dim=0), dict(n_kv_heads=0), dict(n_pages=0), dict(table_stride=0), dict(table_stride=1 << 25), dict(n_seq=-1),
              dict(n_seq=70000), dict(k=P + 8), dict(v=P + 2), dict(head_stride=64 * 128 - 8), dict(head_stride=64 * 128 + 4),
              dict(page_stride=64), dict(page_stride=1 << 39)]


def rope(c, **change):
    v = dict(cu=P, n=3, pos=P, t=capi.T_BF16, q=P, qs=16 * 128, heads=16, k=P, ks=1024, v=P, vs=1024, f=P, rot=128, inter=0, factor=1.0,
             out=2 * P, os=16 * 128)
    v.update(change)
    return capi.lib().mtb_rope_append(C.byref(c) if c else None, v["cu"], v["n"], v["pos"], v["t"], v["q"], v["qs"], v["heads"], v["k"], v["ks"],
                                      v["v"], v["vs"], v["f"], v["rot"], v["inter"], v["factor"], v["out"], v["os"], None)


def attend(c, **change):
    v = dict(cu=P, n=3, most=1, q=P, qs=16 * 128, heads=16, scale=0.1, out=2 * P, os=16 * 128, lse=None, ws=P, size=capi.ATTENTION_WORKSPACE)
    v.update(change)
    return capi.lib().mtb_paged_attention(C.byref(c) if c else None, v["cu"], v["n"], v["most"], v["q"], v["qs"], v["heads"], v["scale"],
                                          v["out"], v["os"], v["lse"], v["ws"], v["size"], None)


def weights(c, **change):
    v = dict(cu=P, n=3, most=1, q=P, qs=16 * 128, heads=16, scale=0.1, lse=P, decay=1.0)
    v.update(change)
    return capi.lib().mtb_attention_weights(C.byref(c) if c else None, v["cu"], v["n"], v["most"], v["q"], v["qs"], v["heads"], v["scale"],
                                            v["lse"], v["decay"], None)


def evict(c, **change):
    v = dict(keep=100, sinks=4, recent=32, new=P, ws=P, size=1 << 30)
    v.update(change)
    return capi.lib().mtb_cache_evict(C.byref(c) if c else None, v["keep"], v["sinks"], v["recent"], v["new"], v["ws"], v["size"], None)


def logits(params=None, **change):
    v = dict(x=P, t=capi.T_F32, rows=2, vocab=1000, xs=1000, y=2 * P, ys=1000, choice=P)
    v.update(change)
    p = None
    if params is not None:
        p = C.byref(capi.LogitsParams(**params))
    return capi.lib().mtb_logits_process(v["x"], v["t"], v["rows"], v["vocab"], v["xs"], p, v["y"], v["ys"], v["choice"], None)


@pytest.mark.parametrize("call", [rope, attend, weights, evict])
@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_bad_cache_views_are_refused(call, bad):
    assert call(cache(**bad)) in (-1, -2) and error()


@pytest.mark.parametrize("call", [rope, attend, weights, evict])
def test_null_cache_is_refused(call):
    assert call(None) == -1 and "null cache" in error()


@pytest.mark.parametrize("call,bad", [
    (rope, dict(n=-1)), (rope, dict(heads=0)), (rope, dict(t=capi.T_F16)), (rope, dict(t=9)), (rope, dict(rot=129)), (rope, dict(rot=130)),
    (rope, dict(rot=-2)), (rope, dict(qs=100)), (rope, dict(ks=1023)), (rope, dict(vs=1)), (rope, dict(os=16 * 128 - 1)), (rope, dict(q=None)),
    (rope, dict(cu=None)), (rope, dict(pos=None)), (rope, dict(f=None)), (rope, dict(out=None)), (rope, dict(q=P + 1)), (rope, dict(f=P + 4)),
    (rope, dict(out=P, t=capi.T_F32)), (rope, dict(out=P, os=17 * 128)),
    (attend, dict(n=-1)), (attend, dict(heads=12)), (attend, dict(heads=0)), (attend, dict(heads=8 * 65, qs=8 * 65 * 128, os=8 * 65 * 128)),
    (attend, dict(q=None)), (attend, dict(q=P + 2)), (attend, dict(qs=2044)), (attend, dict(qs=2052)), (attend, dict(out=P + 8)), (attend, dict(os=2044)),
    (attend, dict(out=None)), (attend, dict(ws=None)), (attend, dict(size=100)), (attend, dict(ws=P + 16)), (attend, dict(scale=math.nan)),
    (attend, dict(scale=math.inf)), (attend, dict(cu=None)),
    (weights, dict(lse=None)), (weights, dict(decay=math.nan)), (weights, dict(heads=9)), (weights, dict(qs=2047)), (weights, dict(n=-5)),
    (evict, dict(keep=-1)), (evict, dict(sinks=-1)), (evict, dict(recent=-1)), (evict, dict(sinks=60, recent=41)), (evict, dict(new=None)),
    (evict, dict(ws=None)), (evict, dict(size=64)), (evict, dict(ws=P + 4)),
], ids=lambda x: x.__name__ if callable(x) else "-".join(f"{k}={v}" for k, v in x.items()))
def test_bad_arguments_are_refused(call, bad):
    assert call(cache(), **bad) in (-1, -2) and error()


def test_bookkeeping_is_needed_where_it_is_used():
    assert weights(cache(weight=None)) == -1
    assert evict(cache(weight=None)) == -1 and evict(cache(position=None)) == -1


@pytest.mark.parametrize("params,bad", [
    (None, dict(t=5)), (None, dict(rows=-1)), (None, dict(vocab=0)), (None, dict(xs=999)), (None, dict(ys=999)), (None, dict(y=None, choice=None)),
    (None, dict(x=None)), (None, dict(x=P + 2)), (None, dict(y=P + 1)), (None, dict(y=P, ys=1001)),
    (dict(repetition=P), {}), (dict(presence=P, history=P), {}), (dict(frequency=P, history=P, history_begin=P), {}), (dict(bias_ids=P), {}),
    (dict(bias_values=P, bias_ids=P, bias_begin=P), {}), (dict(mask=P, mask_stride=31), {}), (dict(history_len=-1), {}), (dict(bias_len=-1), {}),
])
def test_bad_logits_arguments_are_refused(params, bad):
    assert logits(params, **bad) in (-1, -2) and error()


@pytest.mark.parametrize("params,bad", [
    (None, dict(vocab=(1 << 30) + 1, xs=1 << 31, ys=1 << 31)), (None, dict(vocab=(1 << 31) - 1, xs=1 << 31, ys=1 << 31)),
    (dict(history_len=(1 << 30) + 1), {}), (dict(bias_len=1 << 40), {}), (None, dict(choice=P + 2)),
    (dict(history=P + 1, history_begin=P, history_end=P, history_len=4, repetition=P), {}), (dict(mask=P + 2, mask_stride=32, mask_rows=2), {}),
])
def test_logits_sizes_and_alignments_are_refused(params, bad):
    assert logits(params, **bad) == -2 and error()


@pytest.mark.parametrize("name", ["page_table", "kv_len", "position", "weight", "status"])
def test_misaligned_words_of_a_cache_are_refused(name):
    c = cache(**{name: P + 2})
    assert rope(c) == -2 and attend(c) == -2 and weights(c) == -2 and evict(c) == -2


def test_misaligned_words_are_refused():
    assert rope(cache(), cu=P + 2) == -2 and rope(cache(), pos=P + 1) == -2
    assert attend(cache(), cu=P + 2) == -2 and attend(cache(), lse=P + 2) == -2
    assert weights(cache(), lse=P + 2) == -2 and evict(cache(), new=P + 2) == -2


def test_workspace_size_of_impossible_caches():
    """Sizes beyond a cache's limits have no workspace (their product would not fit 64 bits)."""
    assert capi.cache_evict_workspace(65535, 256, 1 << 24) == 65535 * 256 * (256 + (1 << 24) * 256)
    for bad in ((1 << 31) - 1, 8, 10), (8, (1 << 31) - 1, 10), (65535, 257, 10), (1, 8, (1 << 24) + 1):
        assert capi.cache_evict_workspace(*bad) < 0


def test_calls_with_nothing_to_do_succeed_without_a_device():
    assert rope(cache(), n=0) == 0 and attend(cache(), n=0) == 0 and weights(cache(), n=0) == 0
    none = cache(n_seq=0, k=None, v=None, page_table=None, kv_len=None)
    assert rope(none) == 0 and attend(none) == 0 and weights(none) == 0 and evict(none) == 0
    assert logits(rows=0) == 0


def test_host_memory_is_refused():
    """An address that no device owns is an error of the call, with or without a GPU."""
    room = np.zeros(1 << 16, dtype=np.uint8)
    at = (room.ctypes.data + 255) // 256 * 256
    c = cache(k=at, v=at)
    assert rope(c) == -1 and attend(c) == -1 and weights(c) == -1 and evict(c) == -1 and logits(x=at) == -1
    assert error()


def test_workspace_size():
    size = capi.cache_evict_workspace(3, 8, 10)
    assert size >= 3 * 8 * 10 * 64 * 4
    assert evict(cache(n_seq=3, table_stride=10), size=size - 1) == -2
    assert capi.cache_evict_workspace(-1, 8, 10) < 0 and capi.cache_evict_workspace(1, 0, 10) < 0


# ---- rotary frequencies ---------------------------------------------------------------------------------------------


def test_rope_frequencies_plain_and_linear_and_ntk():
    R, base = 96, 1e6
    j = np.arange(R // 2)
    plain = base ** (-2.0 * j / R)
    # pow() of two libraries: a few half steps of 64 bits apart.
    f, c = capi.rope_frequencies(R, base)
    np.testing.assert_allclose(f, plain, rtol=1e-14)
    assert c == 1.0
    f, c = capi.rope_frequencies(R, base, capi.ROPE_LINEAR, 4.0)
    np.testing.assert_allclose(f, plain / 4, rtol=1e-14)
    f, c = capi.rope_frequencies(R, base, capi.ROPE_NTK, 4.0)
    assert f[0] == 1.0 and abs(f[-1] / (plain[-1] / 4) - 1) < 1e-12 and c == 1.0  # the slowest pair is stretched by the whole factor


def test_rope_frequencies_blends():
    R, base, L, factor = 128, 1e4, 4096.0, 8.0
    j = np.arange(R // 2)
    plain = base ** (-2.0 * j / R)
    turns = L * plain / (2 * math.pi)
    f, c = capi.rope_frequencies(R, base, capi.ROPE_BANDS, factor, L, fast=4.0, slow=1.0)
    assert c == 1.0
    np.testing.assert_allclose(f[turns > 4], plain[turns > 4], rtol=1e-14)
    np.testing.assert_allclose(f[turns < 1], plain[turns < 1] / factor, rtol=1e-14)
    mid = (turns <= 4) & (turns >= 1)
    share = (turns[mid] - 1) / 3
    np.testing.assert_allclose(f[mid], plain[mid] * share + plain[mid] / factor * (1 - share), rtol=1e-13)
    f, c = capi.rope_frequencies(R, base, capi.ROPE_YARN, factor, L)
    assert abs(c - (0.1 * math.log(factor) + 1)) < 1e-7
    low = math.floor(R * math.log(L / (32 * 2 * math.pi)) / (2 * math.log(base)))
    high = math.ceil(R * math.log(L / (2 * math.pi)) / (2 * math.log(base)))
    ramp = np.clip((j - low) / (high - low), 0, 1)
    np.testing.assert_allclose(f, plain * (1 - ramp) + plain / factor * ramp, rtol=1e-13)


@pytest.mark.parametrize("bad", [dict(rotary_dim=3), dict(rotary_dim=-2), dict(rotary_dim=130), dict(base=0.0), dict(base=math.nan),
                                 dict(kind=9), dict(kind=capi.ROPE_LINEAR, factor=0.5), dict(kind=capi.ROPE_YARN, factor=4.0),
                                 dict(kind=capi.ROPE_BANDS, factor=4.0, original_len=100.0, fast=1.0, slow=1.0)])
def test_rope_frequencies_refusals(bad):
    args = dict(rotary_dim=64, base=1e4)
    args.update(bad)
    with pytest.raises(capi.MtbError):
        capi.rope_frequencies(**args)
    assert capi.rope_frequencies(0, 1e4)[0].size == 0


# ---- the Python names ----------------------------------------------------------------------------------------------


def cpu_cache(n_seq=2):
    import torch
    pool = torch.zeros(4, 2, 2, 64, 64, dtype=torch.bfloat16)
    table = torch.zeros(n_seq, 2, dtype=torch.int32)
    return pool, table, torch.ones(n_seq, dtype=torch.int32)


def test_python_shapes_types_and_devices_are_checked():
    import torch
    pool, table, n = cpu_cache()
    ok = capi.PagedCache(pool[:, 0], pool[:, 1], table, n)
    with pytest.raises(capi.MtbError):
        capi.PagedCache(pool[:, 0].float(), pool[:, 1].float(), table, n)
    with pytest.raises(capi.MtbError):
        capi.PagedCache(pool[:, 0], pool[:, 1, :1], table, n)
    with pytest.raises(capi.MtbError):
        capi.PagedCache(pool[:, 0].transpose(2, 3), pool[:, 1].transpose(2, 3), table, n)
    with pytest.raises(capi.MtbError):
        capi.PagedCache(pool[:, 0], pool[:, 1], table.long(), n)
    with pytest.raises(capi.MtbError):
        capi.PagedCache(pool[:, 0], pool[:, 1], table.t(), n)
    with pytest.raises(capi.MtbError):
        capi.PagedCache(pool[:, 0], pool[:, 1], table, n[:1])
    with pytest.raises(capi.MtbError):
        capi.PagedCache(pool[:, 0], pool[:, 1], table, n, weight=torch.zeros(3))
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    cu, space = torch.tensor([0, 1, 3], dtype=torch.int32), torch.zeros(capi.ATTENTION_WORKSPACE, dtype=torch.uint8)
    for bad in (q[:, :, ::2], q.float(), q[0], q[:, :3]):
        with pytest.raises(capi.MtbError):
            capi.paged_attention(ok, cu, bad, q.clone(), space, stream=0)
    with pytest.raises(capi.MtbError):
        capi.paged_attention(ok, cu[:2], q, q.clone(), space, stream=0)
    with pytest.raises(capi.MtbError):  # right shapes, but not on a GPU
        capi.paged_attention(ok, cu, q, q.clone(), space, stream=0)
    f = torch.zeros(32, dtype=torch.float64)
    with pytest.raises(capi.MtbError):
        capi.rope_append(ok, cu, torch.zeros(3, dtype=torch.int32), q, q[:, :2], q[:, 2:], f.float(), q.clone(), stream=0)
    with pytest.raises(capi.MtbError):
        capi.rope_append(ok, cu, torch.zeros(2, dtype=torch.int32), q, q[:, :2], q[:, 2:], f, q.clone(), stream=0)
    x = torch.zeros(2, 100)
    one = torch.zeros(2, dtype=torch.int32)
    for bad in (dict(out=x.half()), dict(out=x[:, :50]), dict(choice=one.long()), dict(choice=one, mask=torch.zeros(2, 3, dtype=torch.int32)),
                dict(choice=one, mask=torch.zeros(1, 4, dtype=torch.int32)), dict(choice=one, repetition=torch.ones(1)),
                dict(choice=one, bias_ids=one, bias_values=torch.ones(1), bias_begin=one, bias_end=one)):
        with pytest.raises(capi.MtbError):
            capi.logits_process(x, stream=0, **bad)


def test_a_mask_row_spread_over_all_rows_is_refused():
    """A mask of stride 0 (one row for all) is no [mask rows][words] array: mask_row says which row each has."""
    import torch
    x, one = torch.zeros(2, 100), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(capi.MtbError, match="mask_stride"):
        capi.logits_process(x, choice=one, mask=torch.zeros(1, 4, dtype=torch.int32).expand(2, 4), stream=0)
    with pytest.raises(capi.MtbError, match="stride is shorter"):
        capi.logits_process(x[:1].expand(2, 100), choice=one, stream=0)
