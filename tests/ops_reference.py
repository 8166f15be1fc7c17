"""The operators on a caller's own device memory from their definitions in 64 bits (torch, any device), and what the tests share."""
import math

import torch

PAGE = 64


def make_cache(kv, kv_heads, dim, dtype, device, seed=0, spare=2, table_len=None, fill="normal", apart=False):
    """pool [pages][K/V][kv_heads][64][dim] with shuffled pages; `apart`: the heads and pages have gaps between them."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    need = [-(-max(n, 0) // PAGE) for n in kv]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((len(kv), table_len or max(max(need), 1)), -7, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    shape = (n_pages, 2, kv_heads + (1 if apart else 0), PAGE, dim)
    pool = torch.randn(shape, generator=g).to(dtype) if fill == "normal" else torch.full(shape, fill, dtype=dtype)
    pool = pool.to(device)
    return {"pool": pool, "k": pool[:, 0, :kv_heads], "v": pool[:, 1, :kv_heads], "table": table.to(device),
            "kv_len": torch.tensor(kv, dtype=torch.int32, device=device), "kv": list(kv), "kv_heads": kv_heads, "dim": dim,
            "position": torch.zeros(n_pages, kv_heads, PAGE, dtype=torch.int32, device=device),
            "weight": torch.zeros(n_pages, kv_heads, PAGE, device=device),
            "status": torch.zeros(1, dtype=torch.int32, device=device)}


def rows_of(c, s, n):
    """(pages, places) of the first n slots of sequence s."""
    j = torch.arange(n, device=c["table"].device)
    return c["table"][s][j // PAGE].long(), j % PAGE


def cu_of(new, device):
    return torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=device)


def attention(c, new, q, scale):
    """out, lse, A = sum p |v|, S = the largest sum of |q k| scale of a row, in 64 bits; rows that see nothing 0 and -inf."""
    H, D, Hk = q.shape[1], q.shape[2], c["kv_heads"]
    G, dev = H // Hk, q.device
    n_tok = sum(new)
    out = torch.zeros(n_tok, H, D, dtype=torch.float64, device=dev)
    spread = torch.zeros_like(out)
    lse = torch.full((n_tok, H), -math.inf, dtype=torch.float64, device=dev)
    size = torch.zeros(n_tok, H, dtype=torch.float64, device=dev)
    weight = c["weight"].double() * 0
    at = 0
    for s, (n, m) in enumerate(zip(c["kv"], new)):
        n = max(n, 0)
        if m and n:
            page, place = rows_of(c, s, n)
            sees = torch.arange(n, device=dev)[None] <= (n - m + torch.arange(m, device=dev))[:, None]
            for h in range(H):
                k, v = c["k"][page, h // G, place].double(), c["v"][page, h // G, place].double()
                qq = q[at:at + m, h].double()
                a = ((qq @ k.T) * scale).masked_fill(~sees, -math.inf)
                row = torch.logsumexp(a, 1)
                p = torch.where(sees, torch.exp(a - torch.where(row == -math.inf, 0.0, row)[:, None]), 0.0)
                out[at:at + m, h], spread[at:at + m, h], lse[at:at + m, h] = p @ v, p @ v.abs(), row
                size[at:at + m, h] = ((qq.abs() @ k.abs().T) * abs(scale)).masked_fill(~sees, 0).amax(1)
                weight[page, h // G, place] += p.sum(0)
        at += m
    return {"out": out, "lse": lse, "spread": spread, "size": size, "weight": weight}


def rotate(x, positions, inv_freq, factor, interleaved):
    """x [tokens][heads][dim] rotated, in 64 bits."""
    R = 2 * inv_freq.numel()
    ang = positions.double()[:, None] * inv_freq.double()[None]
    c, s = (torch.cos(ang) * factor)[:, None], (torch.sin(ang) * factor)[:, None]
    y = x.double().clone()
    if interleaved:
        a, b = y[..., 0:R:2].clone(), y[..., 1:R:2].clone()
        y[..., 0:R:2], y[..., 1:R:2] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., : R // 2].clone(), y[..., R // 2: R].clone()
        y[..., : R // 2], y[..., R // 2: R] = a * c - b * s, b * c + a * s
    return y


def evict(c, keep, sinks, recent):
    """Pool, weight, position and new lengths after the eviction: a new set of tensors, plain Python ranking."""
    k, v, w, pos = c["k"].clone(), c["v"].clone(), c["weight"].clone(), c["position"].clone()
    for s, n in enumerate(c["kv"]):
        if n <= keep:
            continue
        page, place = rows_of(c, s, n)
        for h in range(c["kv_heads"]):
            ww, pp = c["weight"][page, h, place].tolist(), c["position"][page, h, place].tolist()
            newest = max(pp)

            def rank(i):
                safe = pp[i] < sinks or pp[i] > newest - recent
                x = -math.inf if math.isnan(ww[i]) else ww[i]
                return (0 if safe else 1, 0.0 if safe else -x, 1 if math.isnan(ww[i]) and not safe else 0, i)

            kept = sorted(sorted(range(n), key=rank)[:keep])
            stay = set(kept)
            to = [i for i in range(keep) if i not in stay]
            frm = [i for i in kept if i >= keep]
            assert len(to) == len(frm)
            if to:
                to, frm = torch.tensor(to, device=page.device), torch.tensor(frm, device=page.device)
                for x, y in ((k, c["k"]), (v, c["v"]), (w, c["weight"]), (pos, c["position"])):
                    x[page[to], h, place[to]] = y[page[frm], h, place[frm]]
    return k, v, w, pos, [min(n, keep) for n in c["kv"]]


def logits(x, history=None, repetition=None, presence=None, frequency=None, biases=None, allowed=None):
    """One row in 64 bits: history a list of ids, biases a list of (id, value), allowed a list of booleans or None."""
    v = [float(t) for t in x.double().tolist()]
    n = len(v)
    count = {}
    for i in history or []:
        if 0 <= i < n:
            count[i] = count.get(i, 0) + 1
    for i, cnt in count.items():
        if repetition is not None:
            v[i] = v[i] / repetition if v[i] > 0 else v[i] * repetition
        if frequency is not None:
            v[i] -= frequency * cnt
        if presence is not None:
            v[i] -= presence
    last = {}
    for i, b in biases or []:
        if 0 <= i < n:
            last[i] = b
    for i, b in last.items():
        v[i] += b
    if allowed is not None:
        v = [a if ok else -math.inf for a, ok in zip(v, allowed)]
    return torch.tensor(v, dtype=torch.float64)
