"""Plain 64-bit forms of the operators over the paged caches, for the tests; they run on any device."""
import math

import torch

PAGE, CKV, KPE = 64, 512, 64


def slots_of(table_row, n):
    pos = torch.arange(n, device=table_row.device)
    return table_row.long()[pos // PAGE] * PAGE + pos % PAGE


def attend(q_nope, q_pe, ckv, kpe, seq_lens, table, scale, weights=None):
    """(out, lse, weights, spread, noise): spread[r] = sum_k p |ckv| bounds what a relative error of the softmax weights
    does to the output, noise[r] = max_k sum |q| |k| * scale what a relative error of the products does to a logit.
    Positions on a page id outside the cache are left out, as the operator does."""
    batch = table.shape[0]
    tokens, heads = q_nope.shape[0] // batch, q_nope.shape[1]
    out = torch.zeros(*q_nope.shape[:2], CKV, dtype=torch.float64, device=q_nope.device)
    spread, lse = torch.zeros_like(out), torch.full(q_nope.shape[:2], -math.inf, dtype=torch.float64, device=q_nope.device)
    noise = torch.zeros_like(lse)
    grown = None if weights is None else weights.double().clone()
    pages = ckv.shape[0]
    for b in range(batch):
        n = max(0, min(int(seq_lens[b]), table.shape[1] * PAGE))
        if n == 0:
            continue
        slot = slots_of(table[b], n)
        good = (slot >= 0) & (slot < pages * PAGE)
        slot = torch.where(good, slot, 0)
        c = torch.where(good[:, None], ckv.reshape(-1, CKV)[slot].double(), 0.0)
        k = torch.cat((c, torch.where(good[:, None], kpe.reshape(-1, KPE)[slot].double(), 0.0)), 1)
        for i in range(tokens):
            r = b * tokens + i
            seen = n - tokens + 1 + i
            if seen <= 0 or not bool(good[:seen].any()):
                continue
            q = torch.cat((q_nope[r], q_pe[r]), 1).double()
            x = torch.where(good[:seen], q @ k[:seen].t() * scale, -math.inf)
            noise[r] = (q.abs() @ k[:seen].abs().t()).amax(1) * abs(scale)
            p = torch.softmax(x, 1)
            out[r], spread[r] = p @ c[:seen], p @ c[:seen].abs()
            lse[r] = torch.logsumexp(x, 1) / math.log(2.0)
            if grown is not None:
                grown[b, :seen] += p.sum(0)
    return out, lse, grown, spread, noise


def check_attend(got_out, got_lse, want, longest, got_weights=None, old_weights=None, heads=1, label=""):
    """Bounds: a bf16 rounding of the output (2^-8 of it) and of every softmax weight (2^-8 of `spread`); the
    576-term fp32 products move a logit by at most d = 600 * 2^-23 * noise, and with it a weight by 2 d of itself
    (numerator and denominator); sums over `longest` fp32 terms add 2^-23 each."""
    out, lse, grown, spread, noise = want
    got_out, got_lse = got_out.double(), got_lse.double()
    assert torch.equal(torch.isinf(got_lse), torch.isinf(lse)), f"{label}: rows that see nothing differ"
    d = 600 * 2.0 ** -23 * noise
    c = 2 * d + 2.0 ** -23 * (longest + 600)
    bound = 2.0 ** -8 * out.abs() + (1 + 2.0 ** -8) * (2.0 ** -8 + c)[..., None] * spread + 1e-30
    err = (got_out - out).abs()
    assert (err <= bound).all(), f"{label}: output off by {(err / bound).max():.2f} of its bound"
    fine = ~torch.isinf(lse)
    err = (got_lse - lse).abs()[fine]
    bound = ((c + 2.0 ** -22) / math.log(2.0) + 2.0 ** -22 * lse.abs())[fine]
    assert (err <= bound).all(), f"{label}: lse off by {(err / bound).max():.2f} of its bound"
    if got_weights is not None:
        gain = (grown - old_weights.double()).abs()
        rows = got_out.shape[0] // grown.shape[0] * heads
        bound = gain * (float(c.max()) + 2.0 ** -20) + 2.0 ** -23 * (rows + 4) * (grown.abs() + gain) + 1e-30
        err = (got_weights.double() - grown).abs()
        assert (err <= bound).all(), f"{label}: weights off by {(err / bound).max():.2f} of their bound"


def evict_choice(weights, n, budget, first, last):
    """Kept positions, ascending."""
    n = max(0, n)
    if n <= budget:
        return list(range(n))
    w = weights.double().cpu()
    inner = range(first, n - last)
    key = {j: (float(w[j]) if w[j] > -3.0e38 else -3.0e38) for j in inner}     # -inf and NaN rank lowest
    best = sorted(inner, key=lambda j: (-key[j], j))[: budget - first - last]
    return sorted(list(range(first)) + best + list(range(n - last, n)))


def rotate(x, angle, interleaved):
    """x [..., 64] double, angle broadcastable [..., 32]."""
    first, second = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    a, b = x[..., first], x[..., second]
    y = torch.empty_like(x)
    y[..., first] = a * torch.cos(angle) - b * torch.sin(angle)
    y[..., second] = b * torch.cos(angle) + a * torch.sin(angle)
    return y
