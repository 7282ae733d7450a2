"""Operators over the paged MLA cache that are timed and compared: their cases, inputs, plain forms and
64-bit values.

  attend   dense attention of the newest tokens of every request over its paged ckv / kpe cache, optionally
           with the accumulated attention weight of every cached token (paged_attention)
  evict    the cached tokens of every request cut down to a budget by their accumulated attention
           weight, and moved to new pages (cache_evict)
  rotary   rotary positions with several axes on the queries and the new keys, and the new rows stored in
           the paged cache (rotary)

`own` chooses between the plain form (elementary torch operations in 32 bits) and this package's kernels.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE, CKV, KPE, INDEX_BYTES = 64, 512, 64, 132
STALE = 3          # pages of the pool that no request holds


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one user, a prompt just finished: the call is all latency
        dict(name="attend_1x1000", op="attend", batch=1, lo=1000, hi=1000, heads=16, tokens=1, weights=False),
        # the headline decode batch: 64 requests of 32768 tokens, one new token each
        dict(name="attend_64x32768", op="attend", batch=64, lo=32768, hi=32768, heads=16, tokens=1, weights=False),
        # a serving batch whose requests are of every age, the youngest a few tokens long
        dict(name="attend_48_ragged", op="attend", batch=48, lo=1, hi=16384, heads=16, tokens=1, weights=False),
        # one very long document: the only parallelism is along the cache
        dict(name="attend_1x131071", op="attend", batch=1, lo=131071, hi=131071, heads=16, tokens=1, weights=False),
        # verification of four drafted tokens per request
        dict(name="attend_16x8192_drafts", op="attend", batch=16, lo=8100, hi=8192, heads=16, tokens=4, weights=False),
        # all 128 heads on one GPU instead of 16 on each of eight
        dict(name="attend_8x8192_heads128", op="attend", batch=8, lo=7000, hi=8192, heads=128, tokens=1, weights=False),
        # decode that keeps score of every cached token: a small batch and a large one
        dict(name="weigh_4x4096", op="attend", batch=4, lo=1024, hi=4096, heads=16, tokens=1, weights=True),
        dict(name="weigh_64x16384", op="attend", batch=64, lo=12000, hi=16384, heads=16, tokens=1, weights=True),
        # a short chat cut to half; a batch of long contexts cut to a quarter, index keys included
        dict(name="evict_2x1500", op="evict", batch=2, lo=1400, hi=1500, budget=750, first=4, last=64, index=False),
        dict(name="evict_32x32768", op="evict", batch=32, lo=30000, hi=32768, budget=8192, first=64, last=512, index=True),
        # the new token of every request of a small batch (one row is padding), and a long mixed prompt
        dict(name="rotary_17", op="rotary", rows=17, heads=16, axes=1, interleaved=True, far=131072),
        dict(name="rotary_16384_image", op="rotary", rows=16384, heads=16, axes=3, interleaved=False, far=32768),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "evict", "rotary"])
    if op == "rotary":
        return dict(op=op, rows=_log(rng, 1, 16384), heads=rng.choice([5, 16, 16, 32, 128]) if rng.random() < 0.5 else 16,
                    axes=rng.choice([1, 2, 3, 4]), interleaved=rng.random() < 0.5, far=_log(rng, 256, 1 << 20))
    batch = _log(rng, 1, 64)
    longest = _log(rng, 1, min(131072, (64 * 32768) // (2 * batch)))
    lo = longest if rng.random() < 0.3 else max(1, int(longest * rng.uniform(0.01, 0.95)))
    if op == "evict":
        longest = max(longest, 64)
        budget = max(1, int(longest * rng.uniform(0.05, 1.1)))
        return dict(op=op, batch=batch, lo=min(lo, longest), hi=longest, budget=budget, first=rng.randint(0, budget // 8),
                    last=rng.randint(0, budget // 4), index=rng.random() < 0.5)
    heads, tokens = 16, 1
    kind = rng.random()
    if kind < 0.25:
        tokens = rng.randint(2, 6)
    elif kind < 0.5:
        heads = rng.choice([5, 32, 64, 128])
    longest = max(1, min(longest, (64 * 32768 * 16) // (batch * heads * tokens)))
    return dict(op=op, batch=batch, lo=min(lo, longest), hi=longest, heads=heads, tokens=tokens, weights=rng.random() < 0.3)


def _lengths(case):
    """The requests' lengths: spread over [lo, hi] on a log scale, fixed by the case."""
    rng = random.Random("%d %d %d" % (case["batch"], case["lo"], case["hi"]))
    lens = [_log(rng, case["lo"], case["hi"]) for _ in range(case["batch"])]
    lens[-1] = case["hi"]
    return lens


def work(case):
    if case["op"] == "rotary":
        row = 2 * (2 * case["heads"] * KPE + 2 * CKV + 2 * KPE) + 4 * case["axes"] + 4
        return {"bytes": case["rows"] * row, "flops": case["rows"] * (case["heads"] + 1) * KPE * 3}
    lens = _lengths(case)
    total = sum(lens)
    if case["op"] == "evict":
        kept = sum(min(n, case["budget"]) for n in lens)
        row = 2 * (CKV + KPE) + (INDEX_BYTES if case["index"] else 0)
        return {"bytes": 2 * kept * row + 4 * total + 4 * kept + 4 * case["batch"] * case["budget"], "flops": total}
    rows = case["batch"] * case["tokens"] * case["heads"]
    moved = 2 * total * (CKV + KPE) + rows * (2 * (CKV + KPE) + 2 * CKV + 4) + 4 * sum(-(-n // PAGE) for n in lens)
    if case["weights"]:
        moved += 8 * total
    return {"bytes": moved, "flops": 2 * total * case["tokens"] * case["heads"] * (2 * CKV + KPE)}


# ----------------------------------------------------------------------------------------- inputs
def _tables(need, first_page, perm):
    """Block table rows from the permuted pages, unused entries 0."""
    table = np.zeros((len(need), max(need)), dtype=np.int32)
    at = first_page
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, at


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    rng = np.random.RandomState(int(seed) % (1 << 32))

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.bfloat16)

    if case["op"] == "rotary":
        n, axes = case["rows"], case["axes"]
        pages = -(-n // PAGE) + STALE
        # text positions advance together on every axis; patches of an image hold time still
        start = int(rng.randint(0, max(1, case["far"] - n)))
        pos = np.tile(start + np.arange(n, dtype=np.int64), (axes, 1))
        if axes > 1:
            side = 1 + int(rng.randint(8, 40))
            image = (np.arange(n) // (side * side)) % 2 == 1
            at = np.arange(n) % (side * side)
            pos[0, image] -= at[image]
            pos[1, image] += at[image] // side - at[image]
            pos[-1, image] += at[image] % side - (at[image] if axes > 2 else at[image] // side)
        pos = np.clip(pos, 0, case["far"])
        slots = rng.permutation(pages * PAGE)[:n].astype(np.int32)
        if n > 8:
            slots[n // 2] = -1               # a row that pads the batch
        share = [32 // axes + (1 if i < 32 % axes else 0) for i in range(axes)]
        return {
            "op": "rotary", "q_pe": normal(n, case["heads"], KPE), "ckv": normal(n, CKV), "kpe": normal(n, KPE),
            "positions": torch.from_numpy(pos.astype(np.int32)).to(dev),
            "inv_freq": torch.from_numpy((10000.0 ** (-np.arange(32) / 32.0)).astype(np.float32)).to(dev),
            "pair_axes": [a for a, k in enumerate(share) for _ in range(k)], "interleaved": case["interleaved"],
            "slots": torch.from_numpy(slots).to(dev),
            "ckv_cache": normal(pages, PAGE, CKV), "kpe_cache": normal(pages, PAGE, KPE),
        }

    lens = _lengths(case)
    need = [-(-n // PAGE) for n in lens]
    new_need = [-(-min(n, case["budget"]) // PAGE) for n in lens] if case["op"] == "evict" else []
    pages = sum(need) + sum(new_need) + STALE
    perm = rng.permutation(pages).astype(np.int32)
    table, used = _tables(need, 0, perm)
    state = {
        "op": case["op"], "ckv_cache": normal(pages, PAGE, CKV), "kpe_cache": normal(pages, PAGE, KPE),
        "seq_lens": torch.tensor(lens, dtype=torch.int32, device=dev), "block_table": torch.from_numpy(table).to(dev),
    }
    width = table.shape[1] * PAGE
    if case["op"] == "evict":
        new_table, _ = _tables(new_need, used, perm)
        u = torch.rand(len(lens), width, generator=gen, device=dev)
        weights = (-torch.log(u + 1e-9)) ** 3          # few tokens carry most of the weight
        weights[u < 0.02] = 0                          # never looked at
        index = torch.randint(-128, 128, (pages, PAGE, 1, INDEX_BYTES), generator=gen, device=dev, dtype=torch.int8) if case["index"] else None
        state.update(token_weights=weights, new_block_table=torch.from_numpy(new_table).to(dev), budget=case["budget"],
                     first=case["first"], last=case["last"], k_index_cache=index)
        return state
    rows = len(lens) * case["tokens"]
    state.update(q_nope=normal(rows, case["heads"], CKV), q_pe=normal(rows, case["heads"], KPE), scale=1.0 / math.sqrt(192.0))
    state["token_weights"] = torch.rand(len(lens), width, generator=gen, device=dev) if case["weights"] else None
    state["new_token_weights"] = torch.zeros(len(lens), width, device=dev) if case["weights"] else None
    return state


# ---------------------------------------------------------------------------------- one pass
def run(state):
    return {"attend": _attend, "evict": _evict, "rotary": _rotary}[state["op"]](state)


def _attend(s):
    if own:
        from auto_gpu_kernel_b200 import paged_attention
        out, lse = paged_attention.run(s["q_nope"], s["q_pe"], s["ckv_cache"], s["kpe_cache"], s["seq_lens"], s["block_table"],
                                       s["scale"], token_weights=s["token_weights"], new_token_weights=s["new_token_weights"])
        return out, lse, s["new_token_weights"]
    batch, heads = s["block_table"].shape[0], s["q_nope"].shape[1]
    tokens = s["q_nope"].shape[0] // batch
    width = s["block_table"].shape[1] * PAGE
    pages = s["block_table"].long()
    c = s["ckv_cache"][pages].view(batch, width, CKV).float()
    k = s["kpe_cache"][pages].view(batch, width, KPE).float()
    qn = s["q_nope"].view(batch, tokens * heads, CKV).float()
    qp = s["q_pe"].view(batch, tokens * heads, KPE).float()
    x = (qn @ c.transpose(1, 2) + qp @ k.transpose(1, 2)) * s["scale"]
    # token i of a request sees the positions up to its own: the last one is at seq_len - 1
    at = torch.arange(width, device=x.device)
    mine = s["seq_lens"][:, None] - tokens + torch.arange(tokens, device=x.device)
    seen = (at[None, None] <= mine[:, :, None]).repeat_interleave(heads, 1)
    x = torch.where(seen, x, -math.inf)
    top = x.amax(2, keepdim=True)
    e = torch.where(seen, torch.exp(x - top), 0.0)
    total = e.sum(2, keepdim=True)
    p = torch.where(total > 0, e / total, 0.0)
    out = (p @ c).to(torch.bfloat16).view(batch * tokens, heads, CKV)
    lse = torch.where(total > 0, (top + torch.log(total)) / math.log(2.0), -math.inf).view(batch * tokens, heads)
    if s["new_token_weights"] is not None:
        held = at[None] < s["seq_lens"][:, None]
        s["new_token_weights"].copy_(torch.where(held, s["token_weights"] + p.sum(1), s["new_token_weights"]))
    return out, lse, s["new_token_weights"]


def _evict(s):
    if own:
        from auto_gpu_kernel_b200 import cache_evict
        lens, weights, kept = cache_evict.run(s["token_weights"], s["seq_lens"], s["block_table"], s["new_block_table"], s["budget"],
                                              s["ckv_cache"], s["kpe_cache"], s["k_index_cache"], keep_first=s["first"], keep_last=s["last"])
        return lens, weights, kept, s["ckv_cache"], s["kpe_cache"], s["k_index_cache"]
    w, lens, budget = s["token_weights"], s["seq_lens"], s["budget"]
    batch, width = w.shape
    at = torch.arange(width, device=w.device)[None]
    held = at < lens[:, None]
    safe = held & ((at < s["first"]) | (at >= lens[:, None] - s["last"]))
    key = torch.where(safe, math.inf, torch.where(held, w, -math.inf))
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :budget]
    new_lens = lens.clamp(max=budget)
    there = torch.arange(order.shape[1], device=w.device)[None] < new_lens[:, None]
    kept = torch.where(there, order, width).sort(1).values
    src = torch.where(there, kept, 0)
    weights = torch.where(there, w.gather(1, src), 0.0)
    new_pages = s["new_block_table"].repeat_interleave(PAGE, 1)[:, :order.shape[1]].long()
    to = new_pages * PAGE + torch.arange(new_pages.shape[1], device=w.device) % PAGE
    frm = s["block_table"].gather(1, src // PAGE).long() * PAGE + src % PAGE
    frm, to = frm[:, :to.shape[1]][there[:, :to.shape[1]]], to[there[:, :to.shape[1]]]
    s["ckv_cache"].view(-1, CKV)[to] = s["ckv_cache"].view(-1, CKV)[frm]
    s["kpe_cache"].view(-1, KPE)[to] = s["kpe_cache"].view(-1, KPE)[frm]
    if s["k_index_cache"] is not None:      # 8192 bytes of keys, then 64 scales of four bytes, in every page
        page = s["k_index_cache"].view(-1, PAGE * INDEX_BYTES)
        keys, scales = page[:, :PAGE * 128].view(-1, PAGE, 128), page[:, PAGE * 128:].view(-1, PAGE, 4)
        keys[to // PAGE, to % PAGE] = keys[frm // PAGE, frm % PAGE]
        scales[to // PAGE, to % PAGE] = scales[frm // PAGE, frm % PAGE]
    kept = torch.where(there, kept, -1).int()
    pad = budget - kept.shape[1]
    if pad > 0:                             # a budget beyond the longest request
        kept = torch.nn.functional.pad(kept, (0, pad), value=-1)
        weights = torch.nn.functional.pad(weights, (0, pad))
    return new_lens, weights, kept, s["ckv_cache"], s["kpe_cache"], s["k_index_cache"]


def _rotary(s):
    if own:
        from auto_gpu_kernel_b200 import rotary
        q = rotary.append(s["q_pe"], s["ckv"], s["kpe"], s["positions"], s["inv_freq"], s["pair_axes"], s["slots"],
                          s["ckv_cache"], s["kpe_cache"], interleaved=s["interleaved"])
        return q, s["ckv_cache"], s["kpe_cache"]
    # angles of far positions need 64 bits
    angle = (s["positions"].double()[s["pair_axes"]] * s["inv_freq"].double()[:, None]).t()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = _turn(s["q_pe"].float(), cos[:, None], sin[:, None], s["interleaved"]).to(torch.bfloat16)
    k = _turn(s["kpe"].float(), cos, sin, s["interleaved"]).to(torch.bfloat16)
    stored = s["slots"] >= 0
    to = s["slots"][stored].long()
    s["ckv_cache"].view(-1, CKV)[to] = s["ckv"][stored]
    s["kpe_cache"].view(-1, KPE)[to] = k[stored]
    return q, s["ckv_cache"], s["kpe_cache"]


def _turn(x, cos, sin, interleaved):
    """Every pair (a, b) of the last axis turned by its angle; pairs are neighbours, or half the width apart."""
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :KPE // 2], x[..., KPE // 2:])
    u, v = a * cos - b * sin, b * cos + a * sin
    return torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)


# ---------------------------------------------------------------------------- values in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        ang = np.empty((case["rows"], 32))
        pos, freq = s["positions"].cpu().numpy().astype(np.float64), s["inv_freq"].cpu().numpy().astype(np.float64)
        for i, axis in enumerate(s["pair_axes"]):
            ang[:, i] = pos[axis] * freq[i]
        z = torch.from_numpy(np.exp(1j * ang)).cuda()
        first, second = (slice(0, None, 2), slice(1, None, 2)) if case["interleaved"] else (slice(0, 32), slice(32, 64))
        turned = []
        for x, t in ((s["q_pe"].double(), z[:, None]), (s["kpe"].double(), z)):
            w = torch.complex(x[..., first], x[..., second]) * t
            y = torch.empty_like(x)
            y[..., first], y[..., second] = w.real, w.imag
            turned.append(y)
        rows = [r for r, slot in enumerate(s["slots"].tolist()) if slot >= 0]
        to = s["slots"][rows].long()
        ckv, kpe = s["ckv_cache"].double(), s["kpe_cache"].double()
        ckv.view(-1, CKV)[to] = s["ckv"][rows].double()
        kpe.view(-1, KPE)[to] = turned[1][rows]
        return turned[0], ckv, kpe
    lens = s["seq_lens"].tolist()
    table = s["block_table"].cpu().numpy().astype(np.int64)
    slots = (table[:, :, None] * PAGE + np.arange(PAGE)).reshape(len(lens), -1)
    if case["op"] == "evict":
        budget = case["budget"]
        w = s["token_weights"].cpu().numpy()
        kept = np.full((len(lens), budget), -1, dtype=np.int32)
        weights = np.zeros((len(lens), budget), dtype=np.float32)
        caches = [s["ckv_cache"].clone().view(-1, CKV), s["kpe_cache"].clone().view(-1, KPE)]
        index = s["k_index_cache"].clone().view(-1, PAGE * INDEX_BYTES) if case["index"] else None
        for b, n in enumerate(lens):
            inner = np.arange(min(case["first"], n), max(n - case["last"], min(case["first"], n)))
            always = np.setdiff1d(np.arange(n), inner)
            ranked = inner[np.argsort(-w[b, inner].astype(np.float64), kind="stable")]
            mine = np.sort(np.concatenate([always, ranked[:max(0, min(n, budget) - always.size)]]))
            kept[b, :mine.size] = mine
            weights[b, :mine.size] = w[b, mine]
            frm = torch.from_numpy(slots[b, mine]).cuda()
            j = np.arange(mine.size)
            to = torch.from_numpy(s["new_block_table"][b].cpu().numpy().astype(np.int64)[j // PAGE] * PAGE + j % PAGE).cuda()
            for cache in caches:
                cache[to] = cache[frm]
            if index is not None:
                byte = torch.arange(128, device="cuda")
                index[(to // PAGE)[:, None], (to % PAGE)[:, None] * 128 + byte] = index[(frm // PAGE)[:, None], (frm % PAGE)[:, None] * 128 + byte]
                byte = torch.arange(4, device="cuda") + PAGE * 128
                index[(to // PAGE)[:, None], (to % PAGE)[:, None] * 4 + byte] = index[(frm // PAGE)[:, None], (frm % PAGE)[:, None] * 4 + byte]
        like = [caches[0].view_as(s["ckv_cache"]), caches[1].view_as(s["kpe_cache"])]
        new_lens = np.minimum(np.asarray(lens), budget).astype(np.int32)
        return (torch.from_numpy(new_lens), torch.from_numpy(weights), torch.from_numpy(kept), *like,
                index.view_as(s["k_index_cache"]) if index is not None else None)
    tokens, heads = case["tokens"], case["heads"]
    out = torch.zeros(len(lens) * tokens, heads, CKV, dtype=torch.float64, device="cuda")
    lse = torch.full((len(lens) * tokens, heads), -math.inf, dtype=torch.float64, device="cuda")
    weights = s["new_token_weights"].double() if case["weights"] else None
    for b, n in enumerate(lens):
        rows = torch.from_numpy(slots[b, :n]).cuda()
        c = s["ckv_cache"].view(-1, CKV)[rows].double()
        key = torch.cat((c, s["kpe_cache"].view(-1, KPE)[rows].double()), 1)
        if case["weights"]:
            weights[b, :n] = s["token_weights"][b, :n].double()
        for i in range(tokens):
            seen, r = n - tokens + 1 + i, b * tokens + i
            if seen <= 0:
                continue
            q = torch.cat((s["q_nope"][r], s["q_pe"][r]), 1).double()
            x = q @ key[:seen].t() * s["scale"]
            lse[r] = torch.logsumexp(x, 1) / math.log(2.0)
            p = torch.softmax(x, 1)
            out[r] = p @ c[:seen]
            if case["weights"]:
                weights[b, :seen] += p.sum(0)
    return out, lse, weights
