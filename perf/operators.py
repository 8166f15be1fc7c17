"""The operators on a caller's own device memory: what is measured of them.

  rope      rotary positions of q and k, with the append of k and v to a paged cache
  attend    attention of a ragged batch's new tokens over the paged cache; with "weights" also the softmax weight that
            every cached position received
  evict     eviction from the cache by accumulated attention weight
  logits    repetition penalties, biases and grammar masks on logits, with the greedy choice

The caches have the decoder's own layout: pages of 64 positions, [page][K/V][kv_head][64][head_dim].
"""
import math

import numpy as np
import torch

own = False

PAGE = 64
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ints(text):
    return [int(x) for x in text.split()]


def listed():
    return [
        # One decode step of eight recordings: a single token each, the decoder's own head layout; all latency.
        {"name": "rope step", "op": "rope", "kv": "2049 1500 407 27000 811 64 65 4096", "new": "1 1 1 1 1 1 1 1", "heads": 16, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "stretch": 1.0, "in": "bf16", "type": "bf16"},
        # A long prompt's rows beside two shorter ones, f32 projections into an fp16 cache, a quarter of the pairs' dims unrotated, positions stretched.
        {"name": "rope prompt", "op": "rope", "kv": "22528 407 1131", "new": "8192 407 1131", "heads": 16, "kv_heads": 8,
         "dim": 128, "rotary": 96, "interleaved": True, "stretch": 4.0, "in": "f32", "type": "f16"},
        # The smallest useful call: one token over a short prompt's cache.
        {"name": "attend one short", "op": "attend", "kv": "408", "new": "1", "heads": 16, "kv_heads": 8, "dim": 128, "type": "bf16", "weights": False},
        # One token of a half-hour recording: all cache bandwidth, the long axis split.
        {"name": "attend one long", "op": "attend", "kv": "27000", "new": "1", "heads": 16, "kv_heads": 8, "dim": 128, "type": "f16", "weights": False},
        # The verify rows of a ragged group of recordings, with the weights that a bounded cache needs.
        {"name": "attend verify group", "op": "attend", "kv": "2056 27000 5000 411 13001 64 9000 18000", "new": "8 8 3 1 8 5 8 8", "heads": 16, "kv_heads": 8,
         "dim": 128, "type": "bf16", "weights": True},
        # Fresh prompts of odd lengths, a head layout with four query heads to a KV head and 64 dims.
        {"name": "attend prompts", "op": "attend", "kv": "407 1500 33 2048 1 777", "new": "407 1500 33 2048 1 777", "heads": 32, "kv_heads": 8,
         "dim": 64, "type": "bf16", "weights": False},
        # A chunk of new audio rows deep in a long recording; compute bound.
        {"name": "attend long chunk", "op": "attend", "kv": "24576", "new": "2048", "heads": 16, "kv_heads": 8, "dim": 128, "type": "bf16", "weights": True},
        # A group's caches one page over their budget: a few rows to move.
        {"name": "evict page", "op": "evict", "kv": "2112 2112 2111 2050 1024 2112 2100 2112", "kv_heads": 8, "dim": 128, "type": "f16", "keep": 2048,
         "sinks": 4, "recent": 256},
        # Half-hour recordings cut to a third: ranking and moving many rows.
        {"name": "evict long", "op": "evict", "kv": "27000 25001 22528 26111", "kv_heads": 8, "dim": 128, "type": "bf16", "keep": 8192, "sinks": 4, "recent": 512},
        # One row of the decoder's vocabulary: latency.
        {"name": "logits one", "op": "logits", "rows": 1, "vocab": 151936, "type": "f32", "history": 256, "biases": 16, "masked": 0.0},
        # The verify rows of eight recordings under a grammar, bf16 logits (many equal values).
        {"name": "logits verify", "op": "logits", "rows": 64, "vocab": 151936, "type": "bf16", "history": 1000, "biases": 32, "masked": 0.9},
        # A large serving batch with long histories.
        {"name": "logits batch", "op": "logits", "rows": 256, "vocab": 151936, "type": "f32", "history": 4096, "biases": 300, "masked": 0.5},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attend", "attend", "evict", "logits"])
    if op == "logits":
        rows = _spread(rng, 1, 200)
        return {"op": op, "rows": rows, "vocab": _spread(rng, 1000, 151936), "type": rng.choice(["f32", "bf16", "f16"]),
                "history": _spread(rng, 1, 4096), "biases": rng.choice([0, _spread(rng, 1, 300)]), "masked": rng.choice([0.0, 0.3, 0.99])}
    n_seq = rng.choice([1, 1, 2, 3, 5, 8])
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128])
    if op == "evict":
        kv = [_spread(rng, 65, 27000) for _ in range(n_seq)]
        keep = _spread(rng, 64, max(65, max(kv) - 1))
        return {"op": op, "kv": " ".join(map(str, kv)), "kv_heads": kv_heads, "dim": dim, "type": rng.choice(["f16", "bf16"]), "keep": keep,
                "sinks": rng.choice([0, 4]), "recent": rng.randrange(0, max(1, keep - 4))}
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    if op == "rope":
        new = [_spread(rng, 1, 4096) for _ in range(n_seq)]
        kv = [n + rng.choice([0, _spread(rng, 1, 20000)]) for n in new]
        return {"op": op, "kv": " ".join(map(str, kv)), "new": " ".join(map(str, new)), "heads": min(heads, 16), "kv_heads": kv_heads, "dim": dim,
                "rotary": dim if rng.random() < 0.5 else 2 * rng.randrange(1, dim // 2), "interleaved": rng.random() < 0.5,
                "stretch": rng.choice([1.0, 4.0]), "in": rng.choice(["same", "f32"]), "type": rng.choice(["f16", "bf16"])}
    if rng.random() < 0.5:  # steps: few rows over caches of any length
        new = [rng.choice([1, 1, 2, 4, 8, rng.randrange(1, 40)]) for _ in range(n_seq)]
        kv = [n + _spread(rng, 1, 26000) for n in new]
    else:  # chunks and whole prompts
        new = [_spread(rng, 16, 2000 // n_seq + 16) for _ in range(n_seq)]
        kv = [n + rng.choice([0, _spread(rng, 1, 12000)]) for n in new]
    return {"op": op, "kv": " ".join(map(str, kv)), "new": " ".join(map(str, new)), "heads": min(heads, 16), "kv_heads": kv_heads, "dim": dim,
            "type": rng.choice(["f16", "bf16"]), "weights": rng.random() < 0.4}


# ---- inputs --------------------------------------------------------------------------------------------------------


def _frequencies(rotary, stretch):
    """Inverse frequencies (64 bits) for a base of 1e6; stretched contexts blend the interpolated and the plain ones by wavelength."""
    j = np.arange(rotary // 2, dtype=np.float64)
    f = 1e6 ** (-2.0 * j / rotary)
    if stretch == 1.0:
        return f, 1.0
    turns = 8192 * f / (2 * math.pi)
    ramp = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
    return f * ramp + f / stretch * (1 - ramp), 0.1 * math.log(stretch) + 1.0


def _cache(case, g, kv, fill=True):
    """A pool with a few spare pages, and the sequences' page tables drawn over it."""
    need = [-(-n // PAGE) for n in kv]
    table_len = max(max(need), 1)
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(kv), table_len, dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    shape = (n_pages, 2, case["kv_heads"], PAGE, case["dim"])
    t = TYPES[case["type"]]
    pool = torch.randn(shape, generator=g, device=DEV, dtype=t) if fill else torch.zeros(shape, device=DEV, dtype=t)
    return {"pool": pool, "table": table, "kv_len": torch.tensor(kv, dtype=torch.int32, device=DEV)}


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op = case["op"]
    if op == "logits":
        return _prepare_logits(case, g)
    kv = _ints(case["kv"])
    s = _cache(case, g, kv, fill=op != "rope")
    s["case"] = case
    if op == "evict":
        # Accumulated softmax weights are spread over decades; positions run up, with the gaps that earlier evictions left.
        meta = (s["pool"].shape[0], case["kv_heads"], PAGE)
        s["weight"] = torch.exp(2.5 * torch.randn(meta, generator=g, device=DEV))
        s["position"] = torch.zeros(meta, dtype=torch.int32, device=DEV)
        ahead = 0
        for i, n in enumerate(kv):
            pages = s["table"][i, : -(-n // PAGE)].long()
            pos = torch.arange(pages.numel() * PAGE, device=DEV, dtype=torch.int32)
            pos = pos + (pos >= 64).to(torch.int32) * ahead
            s["position"][pages] = pos.view(-1, 1, PAGE).expand(-1, case["kv_heads"], -1)
            ahead += 1000
        s["new_len"] = torch.zeros(len(kv), dtype=torch.int32, device=DEV)
        pages = s["table"].shape[1]
        s["workspace"] = torch.zeros(len(kv) * case["kv_heads"] * (pages * 256 + 256), dtype=torch.uint8, device=DEV)
        return s
    new = _ints(case["new"])
    n_tokens, H, D = sum(new), case["heads"], case["dim"]
    starts = np.concatenate([[0], np.cumsum(new)])
    s["cu"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    s["n_tokens"], s["max_new"] = n_tokens, max(new)
    if op == "rope":
        t = TYPES[case["type"] if case["in"] == "same" else case["in"]]
        # q, k and v are views of the fused projection's rows, as a model has them.
        rows = torch.randn(n_tokens, H + 2 * case["kv_heads"], D, generator=g, device=DEV, dtype=t)
        s["q"], s["k"], s["v"] = rows[:, :H], rows[:, H:H + case["kv_heads"]], rows[:, H + case["kv_heads"]:]
        first = [n - m for n, m in zip(kv, new)]
        s["positions"] = torch.cat([torch.arange(f, f + m, dtype=torch.int32, device=DEV) for f, m in zip(first, new)])
        f, s["factor"] = _frequencies(case["rotary"], case["stretch"])
        s["inv_freq"] = torch.from_numpy(f).to(DEV)
        s["q_out"] = torch.zeros(n_tokens, H, D, dtype=TYPES[case["type"]], device=DEV)
        return s
    # Scores with a spread of about 1.5: some positions weigh hundreds of times others, as after normed q and k.
    s["q"] = (1.5 * torch.randn(n_tokens, H, D, generator=g, device=DEV)).to(TYPES[case["type"]])
    s["out"] = torch.zeros(n_tokens, H, D, dtype=TYPES[case["type"]], device=DEV)
    s["lse"] = torch.zeros(n_tokens, H, device=DEV)
    s["weight"] = torch.zeros(s["pool"].shape[0], case["kv_heads"], PAGE, device=DEV)
    s["workspace"] = torch.zeros(64 << 20, dtype=torch.uint8, device=DEV)
    return s


def _prepare_logits(case, g):
    rows, vocab, hist, nb = case["rows"], case["vocab"], case["history"], case["biases"]
    s = {"case": case}
    s["logits"] = (3.0 * torch.randn(rows, vocab, generator=g, device=DEV)).to(TYPES[case["type"]])
    # Text repeats itself: ids drawn from a skewed distribution, one buffer, a range of it for each row.
    u = torch.rand(rows, hist, generator=g, device=DEV)
    s["history"] = (u * u * u * (vocab - 1)).to(torch.int32).reshape(-1)
    at = torch.arange(rows, dtype=torch.int32, device=DEV)
    s["hist_begin"], s["hist_end"] = at * hist, at * hist + hist
    s["repetition"] = 1.0 + 0.5 * torch.rand(rows, generator=g, device=DEV)
    s["presence"] = torch.rand(rows, generator=g, device=DEV)
    s["frequency"] = torch.rand(rows, generator=g, device=DEV) * 0.25
    if nb:
        ids = torch.rand(rows, vocab, generator=g, device=DEV).topk(min(nb, vocab), dim=1).indices
        nb = ids.shape[1]
        s["bias_ids"] = ids.to(torch.int32).reshape(-1).contiguous()
        s["bias_values"] = 4.0 * torch.randn(rows * nb, generator=g, device=DEV)
        s["bias_begin"], s["bias_end"] = at * nb, at * nb + nb
    if case["masked"]:
        words = -(-vocab // 32)
        allowed = (torch.rand(rows, words, 32, generator=g, device=DEV) >= case["masked"]).to(torch.int64)
        allowed[:, 0, 0] = 1
        word = (allowed << torch.arange(32, device=DEV)).sum(-1)
        s["mask"] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
    s["out"] = torch.zeros_like(s["logits"])
    s["choice"] = torch.zeros(rows, dtype=torch.int32, device=DEV)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        return _own(op, s)
    return {"rope": _rope, "attend": _attend, "evict": _evict, "logits": _logits}[op](s)


def _capi():
    import importlib
    import os
    import sys
    at = os.path.join(os.getcwd(), "moss-transcribe.cpp_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    return importlib.import_module("mtb.capi")


_mtb = None


def _own(op, s):
    global _mtb
    if _mtb is None:
        _mtb = _capi()
    c, capi = s["case"], _mtb
    if op == "rope":
        pool = s["pool"]
        cache = capi.PagedCache(pool[:, 0], pool[:, 1], s["table"], s["kv_len"])
        capi.rope_append(cache, s["cu"], s["positions"], s["q"], s["k"], s["v"], s["inv_freq"], s["q_out"],
                         interleaved=c["interleaved"], factor=s["factor"])
        return {"q": s["q_out"], "pool": pool}
    if op == "attend":
        pool = s["pool"]
        cache = capi.PagedCache(pool[:, 0], pool[:, 1], s["table"], s["kv_len"], weight=s["weight"] if c["weights"] else None)
        capi.paged_attention(cache, s["cu"], s["q"], s["out"], s["workspace"], lse=s["lse"], max_tokens=s["max_new"])
        if not c["weights"]:
            return {"out": s["out"], "lse": s["lse"]}
        capi.attention_weights(cache, s["cu"], s["q"], s["lse"], decay=0.0, max_tokens=s["max_new"])
        return {"out": s["out"], "lse": s["lse"], "weight": s["weight"]}
    if op == "evict":
        # The bookkeeping is copied first, so that every pass ranks the same weights; the K and V rows move in place.
        pool, weight, position = s["pool"], s["weight"].clone(), s["position"].clone()
        cache = capi.PagedCache(pool[:, 0], pool[:, 1], s["table"], s["kv_len"], position=position, weight=weight)
        capi.cache_evict(cache, c["keep"], s["new_len"], s["workspace"], sinks=c["sinks"], recent=c["recent"])
        return {"pool": pool, "weight": weight, "position": position, "new_len": s["new_len"]}
    capi.logits_process(s["logits"], s["out"], s["choice"], history=s["history"], hist_begin=s["hist_begin"], hist_end=s["hist_end"],
                        repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"], bias_ids=s.get("bias_ids"),
                        bias_values=s.get("bias_values"), bias_begin=s.get("bias_begin"), bias_end=s.get("bias_end"), mask=s.get("mask"))
    return {"out": s["out"], "choice": s["choice"]}


def _token_slots(s):
    """Of each token: its sequence, and the slot it has in that sequence's cache."""
    token = torch.arange(s["n_tokens"], device=DEV)
    cu = s["cu"].long()
    seq = torch.searchsorted(cu, token, right=True) - 1
    return seq, token - cu[seq] + s["kv_len"].long()[seq] - (cu[1:] - cu[:-1])[seq]


def _rotate(x, cos, sin, rotary, interleaved):
    x = x.float()
    r = x[..., :rotary]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., : rotary // 2], r[..., rotary // 2:])
    cos, sin = cos[:, None], sin[:, None]
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., rotary:]], -1)


def _rope(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["inv_freq"][None]
    cos, sin = (torch.cos(angle) * s["factor"]).float(), (torch.sin(angle) * s["factor"]).float()
    t = s["pool"].dtype
    s["q_out"].copy_(_rotate(s["q"], cos, sin, c["rotary"], c["interleaved"]).to(t))
    k = _rotate(s["k"], cos, sin, c["rotary"], c["interleaved"]).to(t)
    seq, slot = _token_slots(s)
    page = s["table"][seq, slot // PAGE].long()
    s["pool"][page, 0, :, slot % PAGE] = k
    s["pool"][page, 1, :, slot % PAGE] = s["v"].to(t)
    return {"q": s["q_out"], "pool": s["pool"]}


def _attend(s):
    c = s["case"]
    Hk, D, n_seq = c["kv_heads"], c["dim"], s["kv_len"].numel()
    G, L, T = c["heads"] // Hk, s["table"].shape[1] * PAGE, s["max_new"]
    got = s["pool"][s["table"].long()].float()  # [seq][page][2][head][64][dim]
    got = got.permute(2, 0, 3, 1, 4, 5).reshape(2, n_seq, Hk, L, D)
    cu, kv_len = s["cu"].long(), s["kv_len"].long()
    new = cu[1:] - cu[:-1]
    i, slot = torch.arange(T, device=DEV), torch.arange(L, device=DEV)
    token = (cu[:-1, None] + i).clamp(max=s["n_tokens"] - 1)
    q = s["q"][token].float().view(n_seq, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(n_seq, Hk, G * T, D)
    live = slot[None] < kv_len[:, None]
    sees = (slot[None, None] <= (kv_len - new)[:, None, None] + i[None, :, None]) & (i[None] < new[:, None])[..., None]
    score = torch.matmul(q, got[0].transpose(2, 3)).view(n_seq, Hk, G, T, L) * (1.0 / math.sqrt(D))
    score = score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(score.sub_(top))
    total = e.sum(-1, keepdim=True)
    v = got[1].masked_fill(~live[:, None, :, None], 0.0)
    o = torch.matmul(e.view(n_seq, Hk, G * T, L), v).view(n_seq, Hk, G, T, D) / torch.where(total > 0, total, torch.ones_like(total))
    lse = torch.log(total) + top
    seq, slot_of = _token_slots(s)
    at = slot_of - (kv_len - new)[seq]
    s["out"].copy_(o[seq, :, :, at].reshape(s["n_tokens"], Hk * G, D))
    s["lse"].copy_(lse[seq, :, :, at].reshape(s["n_tokens"], Hk * G))
    if not c["weights"]:
        return {"out": s["out"], "lse": s["lse"]}
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    w = p.sum((2, 3)).view(n_seq, Hk, L // PAGE, PAGE).permute(0, 2, 1, 3)  # [seq][page][head][64]
    keep = live.view(n_seq, L // PAGE, 1, PAGE).expand_as(w)
    seq_i, page_i, head_i, slot_i = torch.nonzero(keep, as_tuple=True)
    s["weight"][s["table"][seq_i, page_i].long(), head_i, slot_i] = w[keep]
    return {"out": s["out"], "lse": s["lse"], "weight": s["weight"]}


def _evict(s):
    c = s["case"]
    Hk, n_seq, keep = c["kv_heads"], s["kv_len"].numel(), c["keep"]
    table, L = s["table"].long(), s["table"].shape[1] * PAGE
    weight, position, pool = s["weight"].clone(), s["position"].clone(), s["pool"]
    w = weight[table].permute(0, 2, 1, 3).reshape(n_seq, Hk, L)
    pos = position[table].permute(0, 2, 1, 3).reshape(n_seq, Hk, L)
    live = torch.arange(L, device=DEV)[None, None] < s["kv_len"].long()[:, None, None]
    newest = torch.where(live, pos, torch.full_like(pos, -1)).amax(-1, keepdim=True)
    guarded = (pos < c["sinks"]) | (pos > newest - c["recent"])
    rank = torch.where(torch.isnan(w), torch.full_like(w, -math.inf), w).double()
    rank = torch.where(guarded, torch.full_like(rank, 1e300), rank)
    order = torch.sort(torch.where(live, rank, torch.full_like(rank, -1e308)), dim=-1, descending=True, stable=True).indices
    stays = torch.zeros(n_seq, Hk, L, dtype=torch.bool, device=DEV)
    stays.scatter_(-1, order[..., :keep], True)
    stays &= live
    slot = torch.arange(L, device=DEV)
    hole, come = ~stays & live & (slot < keep), stays & (slot >= keep)
    full = s["kv_len"].long()[:, None, None] > keep
    hole, come = hole & full, come & full
    # Of each (sequence, head) the n-th hole takes the n-th row to come: nonzero() lists both in that order.
    si, hi, di = torch.nonzero(hole, as_tuple=True)
    _, _, fi = torch.nonzero(come, as_tuple=True)
    to, frm = table[si, di // PAGE], table[si, fi // PAGE]
    pool[to, :, hi, di % PAGE] = pool[frm, :, hi, fi % PAGE]
    weight[to, hi, di % PAGE] = weight[frm, hi, fi % PAGE]
    position[to, hi, di % PAGE] = position[frm, hi, fi % PAGE]
    s["new_len"].copy_(s["kv_len"].clamp(max=keep))
    return {"pool": pool, "weight": weight, "position": position, "new_len": s["new_len"]}


def _logits(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    v = s["logits"].float()
    hist = s["history"].view(rows, c["history"]).long()
    count = torch.zeros(rows, vocab, device=DEV).scatter_add_(1, hist, torch.ones(hist.shape, device=DEV))
    r = s["repetition"][:, None]
    punished = torch.where(v > 0, v / r, v * r) - s["frequency"][:, None] * count - s["presence"][:, None]
    v = torch.where(count > 0, punished, v)
    if "bias_ids" in s:
        ids = s["bias_ids"].view(rows, -1).long()
        v = v.scatter(1, ids, v.gather(1, ids) + s["bias_values"].view(rows, -1))
    if "mask" in s:
        bit = (s["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        v = torch.where(bit.view(rows, -1)[:, :vocab] != 0, v, torch.full_like(v, -math.inf))
    top = v.amax(1, keepdim=True)
    at = torch.arange(vocab, device=DEV, dtype=torch.int32)
    choice = torch.where(v == top, at, torch.full_like(at, vocab)).amin(1)
    s["out"].copy_(v)
    s["choice"].copy_(torch.where(top[:, 0] > -math.inf, choice, torch.full_like(choice, -1)))
    return {"out": s["out"], "choice": s["choice"]}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------


def work(case):
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": 2 * n * size + (n / 8 if case["masked"] else 0) + case["rows"] * (4 * case["history"] + 8 * case["biases"] + 16), "flops": 2 * n}
    kv, Hk, D = _ints(case["kv"]), case["kv_heads"], case["dim"]
    if case["op"] == "evict":
        total = 0.0
        for n in kv:
            if n <= case["keep"]:
                continue
            # All the newest ones, and of the others behind `keep` the share that ranks high enough (ranks do not go by place).
            recent, keep, sinks = min(case["recent"], n), case["keep"], case["sinks"]
            tail = max(0, n - keep - recent)
            moved = min(recent, n - keep) + tail * (keep - sinks - recent) / max(1, n - sinks - recent)
            total += Hk * (8 * n + moved * 2 * (4 * D + 8))
        return {"bytes": total + 8 * len(kv), "flops": 0}
    new, H = _ints(case["new"]), case["heads"]
    if case["op"] == "rope":
        size = 2 if case["in"] == "same" or case["in"] != "f32" else 4
        n = sum(new)
        return {"bytes": n * (H + 2 * Hk) * D * (size + 2) + 4 * n + 4 * case["rotary"], "flops": n * (H + Hk) * case["rotary"] * 3}
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(kv, new))
    out = {"bytes": sum(kv) * 2 * Hk * D * 2 + sum(new) * H * (2 * D * 2 + 4), "flops": pairs * H * D * 4}
    if case["weights"]:
        out["bytes"] += sum(kv) * Hk * 4
        out["flops"] += pairs * H * D * 2
    return out


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "attend": _exact_attend, "evict": _exact_evict, "logits": _exact_logits}[case["op"]](case, s)


def _slots(s, i, n):
    """Pages and places of the first n slots of sequence i."""
    j = torch.arange(n, device=DEV)
    return s["table"][i][j // PAGE].long(), j % PAGE


def _exact_rope(case, s):
    R = case["rotary"]

    def turn(x, positions):  # pairs as complex numbers, times factor * exp(i angle)
        x = x.double().clone()
        ang = positions.double()[:, None] * s["inv_freq"][None]
        z = torch.polar(torch.full_like(ang, s["factor"]), ang)[:, None]
        if case["interleaved"]:
            y = torch.view_as_complex(x[..., :R].reshape(*x.shape[:-1], R // 2, 2).contiguous()) * z
            x[..., :R] = torch.view_as_real(y).reshape(*x.shape[:-1], R)
        else:
            y = torch.complex(x[..., : R // 2], x[..., R // 2: R]) * z
            x[..., : R // 2], x[..., R // 2: R] = y.real, y.imag
        return x

    pool = s["pool"].double()
    q, k, v = turn(s["q"], s["positions"]), turn(s["k"], s["positions"]), s["v"].double()
    at = 0
    for i, (n, m) in enumerate(zip(_ints(case["kv"]), _ints(case["new"]))):
        page, place = _slots(s, i, n)
        pool[page[n - m:], 0, :, place[n - m:]] = k[at:at + m]
        pool[page[n - m:], 1, :, place[n - m:]] = v[at:at + m]
        at += m
    return {"q": q, "pool": pool}


def _exact_attend(case, s):
    G, D = case["heads"] // case["kv_heads"], case["dim"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device=DEV)
    weight = s["weight"].double()
    at = 0
    for i, (n, m) in enumerate(zip(_ints(case["kv"]), _ints(case["new"]))):
        page, place = _slots(s, i, n)
        hidden = torch.arange(n, device=DEV)[None] > torch.arange(n - m, n, device=DEV)[:, None]
        for h in range(case["kv_heads"]):
            k, v = s["pool"][page, 0, h, place].double(), s["pool"][page, 1, h, place].double()
            w = torch.zeros(n, dtype=torch.float64, device=DEV)
            for g in range(h * G, h * G + G):
                a = (s["q"][at:at + m, g].double() @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
                lse[at:at + m, g] = torch.logsumexp(a, -1)
                p = torch.softmax(a, -1)
                out[at:at + m, g] = p @ v
                w += p.sum(0)
            weight[page, h, place] = w
        at += m
    found = {"out": out, "lse": lse}
    if case["weights"]:
        found["weight"] = weight
    return found


def _exact_evict(case, s):
    pool, weight, position = s["pool"].double(), s["weight"].double(), s["position"].clone()
    keep, kv = case["keep"], _ints(case["kv"])
    for i, n in enumerate(kv):
        if n <= keep:
            continue
        page, place = _slots(s, i, n)
        for h in range(case["kv_heads"]):
            w, pos = s["weight"][page, h, place].cpu().numpy(), s["position"][page, h, place].cpu().numpy()
            safe = (pos < case["sinks"]) | (pos > pos.max() - case["recent"])
            best = np.lexsort((np.arange(n), -w.astype(np.float64), ~safe))[:keep]
            kept = np.zeros(n, dtype=bool)
            kept[best] = True
            to, frm = np.flatnonzero(~kept[:keep]), keep + np.flatnonzero(kept[keep:])
            to, frm = torch.from_numpy(to).to(DEV), torch.from_numpy(frm).to(DEV)
            pool[page[to], :, h, place[to]] = pool[page[frm], :, h, place[frm]]
            weight[page[to], h, place[to]] = weight[page[frm], h, place[frm]]
            position[page[to], h, place[to]] = position[page[frm], h, place[frm]]
    return {"pool": pool, "weight": weight, "position": position, "new_len": torch.tensor([min(n, keep) for n in kv], dtype=torch.int32)}


def _exact_logits(case, s):
    v = s["logits"].double()
    for row in range(case["rows"]):
        ids, count = torch.unique(s["history"][row * case["history"]:(row + 1) * case["history"]].long(), return_counts=True)
        x, r = v[row, ids], s["repetition"][row].double()
        x = torch.where(x > 0, x / r, x * r)
        v[row, ids] = x - s["frequency"][row].double() * count - s["presence"][row].double()
        if "bias_ids" in s:
            lo, hi = int(s["bias_begin"][row]), int(s["bias_end"][row])
            v[row, s["bias_ids"][lo:hi].long()] += s["bias_values"][lo:hi].double()
        if "mask" in s:
            words = s["mask"][row].cpu().numpy().view(np.uint32)
            bits = np.unpackbits(words.view(np.uint8), bitorder="little")[: case["vocab"]]
            v[row, torch.from_numpy(bits == 0).to(DEV)] = -math.inf
    return {"out": v, "choice": torch.argmax(v, 1).to(torch.int32)}
